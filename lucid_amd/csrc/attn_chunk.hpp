// Attention of many rows (a chunk of a prompt) over paged quantized keys and values.
//
// Bound by what the vector unit does for each score (an exponent, a maximum, an exponential, a sum, a scale, two roundings) and each code, and
// by the matrix products, on wavefronts that do not quite fill each other's gaps: of 8192 tokens of 16 384 (32 heads of 128 on 8, float16, 8 bits, 2400 us,
// three products where the result needs two: 1.03 PFLOP/s of the 1.16 that a large library product reaches) vector instructions take 50 % of
// the SIMDs' cycles and matrix ones 45; a wavefront issues for 42 % of its time, waits for its turn for 31 and for LDS, memory or the others of
// its block for 28.  So a code is turned into float16 once for a block's 128 or 256 rows, on its way into LDS, and a wavefront has 32 rows, whose
// accumulators, maxima and sums stay in its registers:
//
//   S^T = K Q^T    v_mfma_f32_32x32x16_f16, A: K from LDS, lane (h, n) key n of 32, columns 8h..8h+7 of 16; B: Q in registers.
//   O^T = V^T P^T  lane (h, n) has row n's probabilities of keys 4h..4h+3 and 8+4h..8+4h+3 of 16: B as they are.  A: V^T from LDS, where
//                  a column's keys lie in that order, so that a fragment is 16 consecutive bytes.
//
// 64 keys at a time, in two sets of LDS: while one is worked on, the next keys' codes are on their way to registers, and go
// into the other one after that.  Rows of LDS are swizzled by 16 bytes over all 64 banks, so that fragments do not meet in one (keys'
// rows swizzled over half of the banks cost 2 %); the writes of values, four columns apart, meet in pairs.
#pragma once
#include <type_traits>

#include "paged_attention.hpp"
#include "wave_reduce.hpp"

namespace lq {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// the value of the lane 32 further on (or back) with this one's
template <class F>
__device__ __forceinline__ float halves(float v, F f) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(x[0]), __uint_as_float(x[1]));
}

template <class T, int BITS, bool AFFINE, int DIM, int WAVES>
struct ChunkKernel {
    static constexpr bool F32 = std::is_same_v<T, float>;
    static constexpr int PARTS = F32 ? 2 : 1;  // float16 parts of a query
    // Probabilities are two float16 for float16 results as well: with one alone the error is 1.4 times that of the result's own rounding, and
    // would depend on which kernel has a row (8192 of 16 384, float16, 1893 us with one, 2400 so).
    static constexpr int P_PARTS = 2;
    static constexpr int THREADS = 64 * WAVES, R = 32 * WAVES, KEYS = 64;
    static constexpr int SLABS = DIM / 16, TILES = DIM / 32;
    static constexpr int PIECES = DIM * BITS / 128;                                 // 16-byte pieces of a key's codes
    static constexpr int KP = (KEYS * PIECES + THREADS - 1) / THREADS;               // of a thread
    static constexpr int VUNITS = 8 * DIM / 4, VP = (VUNITS + THREADS - 1) / THREADS;  // 8 keys at 4 columns
    static constexpr int K_BYTES = KEYS * DIM * 2, V_BYTES = DIM * KEYS * 2, STAGE = K_BYTES + V_BYTES + 2 * KEYS * 4;
    static constexpr int LDS_BYTES = 2 * STAGE;

    static __device__ __forceinline__ int k_at(int key, int chunk) { return key * DIM * 2 + ((chunk ^ (key & (DIM >= 128 ? 15 : 7))) << 4); }
    static __device__ __forceinline__ int v_at(int d, int chunk) { return K_BYTES + d * KEYS * 2 + ((chunk ^ ((d ^ (d >> 2)) & 7)) << 4); }

    static __device__ __forceinline__ void run(const AttnArgs& a, const T* __restrict__ q, T* __restrict__ out, char* lds) {
        const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, n = lane & 31;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int group = int(a.group.d);
        clear_other_rows(a, out, a.q_starts[0], a.q_starts[a.batch], blockIdx.x, gridDim.x);
        // heads vary fastest: blocks are dealt to the 8 XCDs in turn, and those of one head find its keys in the same L2.  Of a
        // sequence's tiles the last ones, which see the most keys, come first.
        const unsigned item = blockIdx.x / unsigned(a.kv_heads);
        const int head = int(blockIdx.x - item * unsigned(a.kv_heads));
        Tile it;
        if (!find_tile<R>(a, item, false, it)) return;
        const int rows = it.s.chunk * group, row0 = it.tile * R, at = it.s.len - it.s.chunk;
        const int last_row = min(rows, row0 + R) - 1;
        const Keys seen = keys_of(a, it.s, int(a.group(unsigned(row0))), int(a.group(unsigned(last_row))));
        const int base = seen.lo & ~(KEYS - 1), share = ((seen.hi - base + it.parts - 1) / it.parts + KEYS - 1) / KEYS * KEYS;
        const int from = min(seen.hi, base + it.part * share), to = min(seen.hi, from + share);
        // this wavefront's rows, and the keys that all of them see
        const int w0 = min(row0 + 32 * wave, last_row), w1 = min(row0 + 32 * wave + 31, last_row);
        const int token0 = int(a.group(unsigned(w0))), token1 = int(a.group(unsigned(w1)));
        const int all_lo = a.window > 0 ? max(0, at + token1 - a.window + 1) : 0;
        const int all_hi = min(to, a.causal ? min(it.s.len, at + token0 + 1) : it.s.len);

        // ---- the next keys
        const int row_bytes = a.dim * BITS / 8;
        const auto table = rows_at(a.table + size_t(it.seq) * a.width, a.width * 4);
        auto pages_of = [&](int key) {
            return int(__builtin_amdgcn_raw_buffer_load_b32(table, int(a.page_size(unsigned(key + 16 * (lane & 3)))) * 4, 0, 0));
        };
        size_t place[4];
        int ok = 0;
        auto locate = [&](int key, int pages) {
            if (a.page_size.d % KEYS == 0) {  // (all on one page)
                const unsigned page = unsigned(__builtin_amdgcn_readlane(pages, 0));
                const bool there = key < to && page < unsigned(a.pages);
                ok = there ? (1 << min(4, (to - key + 15) / 16)) - 1 : 0;
                const unsigned in_page = unsigned(key) - a.page_size(unsigned(key)) * a.page_size.d;
                place[0] = there ? (size_t(page) * unsigned(a.kv_heads) + unsigned(head)) * a.page_size.d + in_page : 0;
                const size_t step = there ? 16 : 0;
                place[1] = place[0] + step, place[2] = place[1] + step, place[3] = place[2] + step;
                return;
            }
            ok = 0;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const unsigned page = unsigned(__builtin_amdgcn_readlane(pages, t));
                const bool there = key + 16 * t < to && page < unsigned(a.pages);
                ok |= int(there) << t;
                const unsigned in_page = unsigned(key + 16 * t) - a.page_size(unsigned(key + 16 * t)) * a.page_size.d;
                place[t] = there ? (size_t(page) * unsigned(a.kv_heads) + unsigned(head)) * a.page_size.d + in_page : 0;
            }
        };
        auto place_of = [&](int t) {
            const size_t p0 = place[0], p1 = place[1], p2 = place[2], p3 = place[3];
            const size_t x = t & 1 ? p1 : p0, y = t & 1 ? p3 : p2;
            return t & 2 ? y : x;
        };
        uint4 kreg[KP];
        uint32_t vreg[VP][8];
        float kz[KP];
        f32x4 vz[VP][2];
        float ks_reg, vs_reg, vzero = 0.f;  // of key `lane`
        // Lanes of a wavefront whose pieces lie in one tile of 16 keys share a scalar base, and their offsets do not change.
        constexpr bool K_ONE = PIECES >= 4, V_ONE = DIM >= 128;
        auto request_k = [&] {
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const int u = tid + i * THREADS, key = u / PIECES, piece = u % PIECES;
                if (KEYS * PIECES % THREADS && u >= KEYS * PIECES) break;
                const int byte = piece * 16 < row_bytes ? piece * 16 : 0;
                if constexpr (K_ONE) {
                    const size_t row = place_of(__builtin_amdgcn_readfirstlane(key >> 4));
                    const auto rows = rows_at(a.k_codes + row * unsigned(row_bytes), 16 * row_bytes);
                    kreg[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rows, (key & 15) * row_bytes + byte, 0, 0));
                    if constexpr (AFFINE) kz[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows_at(a.k_zero + row, 64), (key & 15) * 4, 0, 0));
                } else {
                    const size_t row = place_of(key >> 4) + (key & 15);
                    kreg[i] = *reinterpret_cast<const uint4*>(a.k_codes + row * unsigned(row_bytes) + byte);
                    if constexpr (AFFINE) kz[i] = a.k_zero[row];
                }
            }
            const size_t row = place_of(lane >> 4) + (lane & 15);
            ks_reg = a.k_scale[row], vs_reg = a.v_scale[row];
            if constexpr (AFFINE) vzero = a.v_zero[row];
        };
        auto request_v = [&] {
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                const int u = tid + i * THREADS, chunk = u / (DIM / 4), d = u % (DIM / 4) * 4;
                if (VUNITS % THREADS && u >= VUNITS) break;
                const int byte = d < a.dim ? d * BITS / 8 : 0;
                if constexpr (V_ONE) {
                    const size_t row = place_of(__builtin_amdgcn_readfirstlane(chunk >> 1));
                    const auto rows = rows_at(a.v_codes + row * unsigned(row_bytes), 16 * row_bytes);
                    const int off = 4 * (chunk & 1) * row_bytes + byte;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int skip = ((e & 3) + 2 * (e & 4)) * row_bytes;  // keys 0..3 and 8..11 from here
                        if constexpr (BITS == 8) vreg[i][e] = __builtin_amdgcn_raw_buffer_load_b32(rows, off, skip, 0);
                        else vreg[i][e] = __builtin_amdgcn_raw_buffer_load_b16(rows, off, skip, 0);
                    }
                    if constexpr (AFFINE)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            vz[i][e] = __builtin_bit_cast(
                                f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows_at(a.v_zero + row, 64), 16 * (chunk & 1) + 32 * e, 0, 0));
                } else {
                    const size_t row = place_of(chunk >> 1) + 4 * (chunk & 1);
                    const uint8_t* p = a.v_codes + row * unsigned(row_bytes) + byte;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint8_t* pe = p + ((e & 3) + 2 * (e & 4)) * row_bytes;
                        if constexpr (BITS == 8) vreg[i][e] = *reinterpret_cast<const uint32_t*>(pe);
                        else vreg[i][e] = *reinterpret_cast<const uint16_t*>(pe);
                    }
                    if constexpr (AFFINE)
#pragma unroll
                        for (int e = 0; e < 2; ++e) vz[i][e] = *reinterpret_cast<const f32x4*>(a.v_zero + row + 8 * e);
                }
            }
        };
        Level level;  // of the keys that are settled
        // a negative scale changes the queries' signs, and of a scale of 0 all scores are 0, the masked ones still none.  What is left
        // goes with the keys' scales (the sum of a row's products with codes, times it, may be infinite where the score is not)
        const float key_factor = a.scale == 0.f ? 1.f : fabsf(a.scale * kLog2e);
        const uint32_t high = BITS == 4 ? magic() : 0;
        // what is requested becomes float16 in LDS, a part at a time: eight columns of a key, and at last the scales
        constexpr int K_EIGHTS = BITS == 8 ? 2 : 4, K_STEPS = KP * K_EIGHTS + 1;
        auto settle_k = [&](int part, int key, char* stage) {
            if (part < KP * K_EIGHTS) {
                const int i = part / K_EIGHTS, e = part % K_EIGHTS;
                const int u = tid + i * THREADS, k = u / PIECES, piece = u % PIECES;
                if (KEYS * PIECES % THREADS && u >= KEYS * PIECES) return;
                const Offsets<BITS> off = AFFINE ? Offsets<BITS>(kz[i], kz[i]) : Offsets<BITS>();
                const uint32_t w[4] = {kreg[i].x, kreg[i].y, kreg[i].z, kreg[i].w};
                Frag f;
                if constexpr (BITS == 8) {
                    f.p[0] = bytes01(w[2 * e], off.of1024), f.p[1] = bytes23(w[2 * e], off.of1024);
                    f.p[2] = bytes01(w[2 * e + 1], off.of1024), f.p[3] = bytes23(w[2 * e + 1], off.of1024);
                } else {
                    const uint32_t u1 = w[e] >> 8;
                    f.p[0] = nibbles0(w[e], high, off.of1024), f.p[1] = nibbles4(w[e], high, off.of64);
                    f.p[2] = nibbles0(u1, high, off.of1024), f.p[3] = nibbles4(u1, high, off.of64);
                }
                *reinterpret_cast<h8*>(stage + k_at(k, K_EIGHTS * piece + e)) = f.v;
                return;
            }
            // scales (all wavefronts come to the same level)
            float vs = vs_reg * (1.f / kValueUnit);
            if (AFFINE && !(fabsf(vzero) <= 2048.f)) vs = __builtin_nanf("");
            if (!((key + lane >= seen.lo) & (key + lane < to) & (ok >> (lane >> 4) & 1))) vs = level.hi;  // (its p is 0)
            level.follow(fabsf(vs), fabsf(vs));
            // (every wavefront writes them: the same)
            float* to_lds = reinterpret_cast<float*>(stage + K_BYTES + V_BYTES);
            to_lds[lane] = F32 ? ks_reg : ks_reg * key_factor;
            to_lds[KEYS + lane] = vs;
        };
        constexpr int V_STEPS = VP * 8;
        Frag vf[4];
        auto settle_v = [&](int part, char* stage) {
            const int i = part / 8, e = part % 8;
            const int u = tid + i * THREADS, chunk = u / (DIM / 4), d = u % (DIM / 4) * 4;
            if (e >= 4) {
                if (VUNITS % THREADS && u >= VUNITS) return;
                *reinterpret_cast<h8*>(stage + v_at(d + e - 4, chunk)) = vf[e - 4].v;
                return;
            }
            Offsets<BITS> off;
            if constexpr (AFFINE) {
                // (a zero point that is no number reaches every row through the matrix product: the scale has it instead)
                const float z0 = vz[i][e / 2][2 * (e % 2)], z1 = vz[i][e / 2][2 * (e % 2) + 1];
                off = Offsets<BITS>(fabsf(z0) <= 2048.f ? z0 : 0.f, fabsf(z1) <= 2048.f ? z1 : 0.f);
            }
            const uint32_t x = vreg[i][2 * e], y = vreg[i][2 * e + 1];
            if constexpr (BITS == 8) {
                const uint32_t u0 = __builtin_amdgcn_perm(y, x, 0x05010400u), u1 = __builtin_amdgcn_perm(y, x, 0x07030602u);
                vf[0].p[e] = bytes01(u0, off.of1024), vf[1].p[e] = bytes23(u0, off.of1024);
                vf[2].p[e] = bytes01(u1, off.of1024), vf[3].p[e] = bytes23(u1, off.of1024);
            } else {
                const uint32_t u0 = __builtin_amdgcn_perm(y, x, 0x05040100u), u1 = u0 >> 8;
                vf[0].p[e] = nibbles0(u0, high, off.of1024), vf[1].p[e] = nibbles4(u0, high, off.of64);
                vf[2].p[e] = nibbles0(u1, high, off.of1024), vf[3].p[e] = nibbles4(u1, high, off.of64);
            }
        };

        int pages = pages_of(from);
        // ---- queries: column n is row row0 + 32 wave + n
        h8 qf[SLABS][PARTS];
        float factor = key_factor;
        int lo, hi;
        {
            const int used = min(row0 + 32 * wave + n, last_row), token = int(a.group(unsigned(used)));
            const T* src = q + size_t(it.s.q0 + token) * a.ldq + size_t(head * group + (used - token * group)) * a.dim;
            const Keys mine = keys_of(a, it.s, token, token);
            lo = mine.lo, hi = min(mine.hi, to);
            using Raw = std::conditional_t<F32, f32x4, h8>;
            Raw raw[SLABS][PARTS];
#pragma unroll
            for (int i = 0; i < SLABS; ++i)
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const int d = 16 * i + 8 * h;
                    raw[i][p] = reinterpret_cast<const Raw*>(src + (d < a.dim ? d : 0))[p];
                    if (d >= a.dim || a.scale == 0.f) raw[i][p] = Raw{};
                }
            if (from < to) {
                locate(from, pages);
                pages = pages_of(from + KEYS);
                request_k(), request_v();
            }
            const bool minus = a.scale < 0.f;
            int up = 0;
            if constexpr (F32) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < SLABS; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(raw[i][e / 4][e % 4]));
                top = halves(top, [](float x, float y) { return fmaxf(x, y); });
                up = max(-126, min(126, 14 - __builtin_amdgcn_frexp_expf(top)));
                factor = __builtin_ldexpf(key_factor, -up);
            }
            constexpr int order[2][8] = {{0, 1, 2, 3, 4, 5, 6, 7}, {0, 4, 1, 5, 2, 6, 3, 7}};
#pragma unroll
            for (int i = 0; i < SLABS; ++i) {
                Frag f[PARTS];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n0 = order[BITS == 4][2 * e], n1 = order[BITS == 4][2 * e + 1];
                    if constexpr (F32) {
                        float u = __builtin_ldexpf(raw[i][n0 / 4][n0 % 4], up), w = __builtin_ldexpf(raw[i][n1 / 4][n1 % 4], up);
                        if (minus) u = -u, w = -w;
                        f[0].p[e] = to_h2(u, w);
                        f[1].p[e] = to_h2(u - float(f[0].p[e].x), w - float(f[0].p[e].y));
                    } else {
                        f[0].p[e] = h2{raw[i][0][n0], raw[i][0][n1]};
                        if (minus) f[0].p[e] = -f[0].p[e];
                    }
                }
#pragma unroll
                for (int p = 0; p < PARTS; ++p) qf[i][p] = f[p].v;
            }
        }
        f32x16 o[TILES] = {};
        float m = -__builtin_inff(), l = 0.f, l1 = 0.f;
        const unsigned span = unsigned(max(0, hi - lo));

        // 32 keys after 32 keys: while the matrix pipe has the next ones' scores the vector unit has these ones' exponentials, and while it has
        // these ones' values, the next ones' exponents and the codes of those behind them.  One wavefront's instructions alternate: with
        // float32 rows, three wavefronts' worth of products in one, 83 -> 70 us (3 x 333 of 2048); float16 ones, of which a SIMD's two wavefronts
        // filled each other's gaps, within 1 %.
        f32x16 x;  // exponents: scores less the row's maximum so far
        f32x16 s;  // the next scores
        Frag pf[2][P_PARTS];
        const auto scales_of = [&](const char* stage) { return reinterpret_cast<const float*>(stage + K_BYTES + V_BYTES); };
        // two keys' probabilities
        auto probabilities = [&](const char* stage, int half, int pair) {
            const int b = pair / 2, r = pair % 2;
            const f32x2 vs = *reinterpret_cast<const f32x2*>(scales_of(stage) + KEYS + 32 * half + 8 * b + 4 * h + 2 * r);
            const float e0 = __builtin_amdgcn_exp2f(x[2 * pair]), e1 = __builtin_amdgcn_exp2f(x[2 * pair + 1]);
            l += e0, l1 += e1;
            // (0 times anything is 0: a scale that is no number shows in the rows that see its key only)
            const float p0 = mul_legacy(e0, vs.x), p1 = mul_legacy(e1, vs.y);
            const h2 y = to_h2(p0, p1);
            pf[b / 2][0].p[2 * (b % 2) + r] = y;
            pf[b / 2][1].p[2 * (b % 2) + r] = to_h2(p0 - float(y.x), p1 - float(y.y));
        };
        // two keys' exponents
        auto exponents = [&](const char* stage, int half, int pair, float mm) {
            const f32x2 ks = *reinterpret_cast<const f32x2*>(scales_of(stage) + 32 * half + 8 * (pair / 2) + 4 * h + 2 * (pair % 2));
#pragma unroll
            for (int r = 0; r < 2; ++r) x[2 * pair + r] = __builtin_fmaf(s[2 * pair + r], F32 ? ks[r] * factor : ks[r], mm);
        };
        // Matrix products one by one, the next fragment read ahead of each, and behind it the vector unit's share of what is to be done
        // meanwhile: f of the parts [n step / steps, n (step + 1) / steps) of n.  A step is kept together.
        auto deal = [](int n, int step, int steps, auto f) {
#pragma unroll
            for (int i = n * step / steps; i < n * (step + 1) / steps; ++i) f(i);
        };
        constexpr int AHEAD = F32 ? 1 : 3;  // fragments: about as long as LDS takes
        auto scores = [&](const char* stage, int half, auto meanwhile) {
            constexpr int STEPS = SLABS * PARTS;
            s = f32x16{};
            h8 k[AHEAD + 1];
            auto read = [&](int i) { k[i % (AHEAD + 1)] = *reinterpret_cast<const h8*>(stage + k_at(32 * half + n, 2 * i + h)); };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) read(i);
#pragma unroll
            for (int x = 0; x < STEPS; ++x) {
                const int i = x / PARTS, p = PARTS - 1 - x % PARTS;
                if (p == PARTS - 1 && i + AHEAD < SLABS) read(i + AHEAD);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i % (AHEAD + 1)], qf[i][p], s, 0, 0, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                meanwhile(x, STEPS);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto products = [&](const char* stage, int half, auto meanwhile) {
            constexpr int STEPS = 2 * TILES * P_PARTS;
            h8 v[AHEAD + 1];
            auto read = [&](int i) { v[i % (AHEAD + 1)] = *reinterpret_cast<const h8*>(stage + v_at(32 * (i % TILES) + n, 2 * (2 * half + i / TILES) + h)); };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) read(i);
#pragma unroll
            for (int x = 0; x < STEPS; ++x) {
                const int i = x / P_PARTS, p = P_PARTS - 1 - x % P_PARTS;
                if (p == P_PARTS - 1 && i + AHEAD < 2 * TILES) read(i + AHEAD);
                o[i % TILES] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i % (AHEAD + 1)], pf[i / TILES][p].v, o[i % TILES], 0, 0, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                meanwhile(x, STEPS);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // masks keys `at` .. `at` + 31, renews the row's m where a w has grown by enough
        auto raise = [&](const char* stage, int half, int at, int ok_at, Level level) {
            if (!(at >= all_lo && at + 32 <= all_hi && ok_at == 3)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = at + 8 * (i / 4) + 4 * h + i % 4;
                    if (!((unsigned(j - lo) < span) & (ok_at >> (i / 8) & 1))) x[i] = -__builtin_inff();
                }
            }
            float top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
            // (a lane has half of the keys: only where one of the two has grown by enough do they ask each other)
            const bool first = m == -__builtin_inff();
            if (__ballot(top > kMost - level.at || (first && top > m)) || !level.even) {
                top += level.at;  // a bound of log2 of the largest w
                if (!level.even) {
                    const float* vs = scales_of(stage) + KEYS + 32 * half + 4 * h;
                    top = -__builtin_inff();
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i] + float(level_of(vs[8 * (i / 4) + i % 4])));
                }
                top = halves(top, [](float u, float w) { return fmaxf(u, w); }) - kRenewed;
                const float by = first ? top : fmaxf(top, 0.f);  // (-inf: no key seen yet)
                if (by != -__builtin_inff()) {
                    const float f = first ? 0.f : __builtin_amdgcn_exp2f(-0.5f * by);  // (its square may be too small where l is large)
                    m = first ? by : m + by;
                    l = l * f * f, l1 = l1 * f * f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] -= by;
#pragma unroll
                    for (int d = 0; d < TILES; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] *= f * f;
                }
            }
        };
        auto exponent_offset = [&] { return m == -__builtin_inff() ? 0.f : -m; };

        if (from < to) {
#pragma unroll
            for (int i = 0; i < K_STEPS; ++i) settle_k(i, from, lds);
#pragma unroll
            for (int i = 0; i < V_STEPS; ++i) settle_v(i, lds);
            int ok_now = ok;
            Level level_now = level;
            locate(from + KEYS, pages);
            pages = pages_of(from + 2 * KEYS);
            request_k(), request_v();
            __syncthreads();
            scores(lds, 0, [](int, int) {});
#pragma unroll
            for (int i = 0; i < 8; ++i) exponents(lds, 0, i, 0.f);
            raise(lds, 0, from, ok_now & 3, level_now);
            int side = 0;
            for (int key = from;; key += KEYS) {
                char* const now = lds + side * STAGE;
                char* const next = lds + (side ^ 1) * STAGE;
                scores(now, 1, [&](int step, int steps) { deal(8, step, steps, [&](int i) { probabilities(now, 0, i); }); });
                float mm = exponent_offset();
                products(now, 0, [&](int step, int steps) {
                    deal(8, step, steps, [&](int i) { exponents(now, 1, i, mm); });
                    deal(K_STEPS, step, steps, [&](int i) { settle_k(i, key + KEYS, next); });
                });
                const int ok_next = ok;
                locate(key + 2 * KEYS, pages);
                pages = pages_of(key + 3 * KEYS);
                request_k();
                raise(now, 1, key + 32, ok_now >> 2, level_now);
                __syncthreads();
                // (behind the last keys: the scores of what lies there, which nobody takes)
                scores(next, 0, [&](int step, int steps) { deal(8, step, steps, [&](int i) { probabilities(now, 1, i); }); });
                mm = exponent_offset();
                products(now, 1, [&](int step, int steps) {
                    deal(8, step, steps, [&](int i) { exponents(next, 0, i, mm); });
                    deal(V_STEPS, step, steps, [&](int i) { settle_v(i, next); });
                });
                if (key + KEYS >= to) break;
                request_v();
                raise(next, 0, key + KEYS, ok_next & 3, level);
                __syncthreads();
                ok_now = ok_next, level_now = level;
                side ^= 1;
            }
            l += l1;
        }
        l = halves(l, [](float x, float y) { return x + y; });
        const int row = row0 + 32 * wave + n;
        if (row > last_row) return;
        const float scale = kValueUnit * (it.parts == 1 ? (l == 0.f ? 0.f : 1.f / l) : 1.f);
        if (it.parts > 1) {
            if (it.first + it.parts > a.pieces) return;
            float* piece = a.partial + (size_t(it.first + it.part) * a.kv_heads + head) * kPiece<R, DIM>;
            if (h == 0) piece[R * DIM + 32 * wave + n] = m, piece[R * DIM + R + 32 * wave + n] = l;
#pragma unroll
            for (int d = 0; d < TILES; ++d)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    *reinterpret_cast<f32x4*>(piece + (32 * wave + n) * DIM + 32 * d + 8 * b + 4 * h) =
                        f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]} * scale;
            return;
        }
        const int token = int(a.group(unsigned(row)));
        T* dst = out + (size_t(it.s.q0 + token) * a.heads + size_t(head * group + row - token * group)) * a.dim;
#pragma unroll
        for (int d = 0; d < TILES; ++d)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int column = 32 * d + 8 * b + 4 * h;
                if (column >= a.dim) continue;
                const f32x4 v = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]} * scale;
                if constexpr (F32) *reinterpret_cast<f32x4*>(dst + column) = v;
                else *reinterpret_cast<uint2*>(dst + column) = uint2{as_u32(to_h2(v[0], v[1])), as_u32(to_h2(v[2], v[3]))};
            }
    }
};

template <class T, int BITS, bool AFFINE, int DIM, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DIM <= 128 ? 2 : 1) void attn_chunk_kernel(AttnArgs a, const T* __restrict__ q, T* __restrict__ out) {
    extern __shared__ __attribute__((aligned(16))) char chunk_lds[];
    ChunkKernel<T, BITS, AFFINE, DIM, WAVES>::run(a, q, out, chunk_lds);
}

// Joins the parts of a tile's keys, kJoined rows a block.
constexpr int kJoined = 16;
template <class T, int DIM, int R>
__global__ __launch_bounds__(256) void attn_parts_kernel(AttnArgs a, T* __restrict__ out) {
    Tile it;
    if (!find_tile<R>(a, blockIdx.x, true, it) || it.parts == 1 || it.first + it.parts > a.pieces) return;
    const float* first = a.partial + (size_t(it.first) * a.kv_heads + blockIdx.y) * kPiece<R, DIM>;
    // (several rows a wavefront: what finding the tile takes is worth more than one)
    for (int r = blockIdx.z * kJoined + (threadIdx.x >> 6); r < int(blockIdx.z + 1) * kJoined; r += 4)
        join_row<T, DIM, R, false>(a, out, it.s, it.tile, int(blockIdx.y), r, it.parts,
                            [&](int i) { return first + size_t(i) * a.kv_heads * kPiece<R, DIM>; });
}

template <class T, int BITS, int DIM, int WAVES>
int launch_chunk(const AttnArgs& a, const T* q, T* out, int tiles, bool join, hipStream_t st) {
    auto go = [&](auto affine) {
        using K = ChunkKernel<T, BITS, decltype(affine)::value, DIM, WAVES>;
        auto kernel = attn_chunk_kernel<T, BITS, decltype(affine)::value, DIM, WAVES>;
        static DeviceOnce once;
        const int rc = allow_dynamic_lds(once, reinterpret_cast<const void*>(kernel), K::LDS_BYTES);
        if (rc) return rc;
        kernel<<<unsigned(a.blocks) * a.kv_heads, K::THREADS, K::LDS_BYTES, st>>>(a, q, out);
        if (join) attn_parts_kernel<T, DIM, K::R><<<dim3(tiles, a.kv_heads, K::R / kJoined), 256, 0, st>>>(a, out);
        return int(LQ_OK);
    };
    return a.k_zero ? go(std::true_type{}) : go(std::false_type{});
}

template <class T, int BITS>
int launch_chunk_of(const AttnArgs& a, const T* q, T* out, bool wide, int tiles, bool join, hipStream_t st) {
    if (a.dim <= 64) return launch_chunk<T, BITS, 64, 4>(a, q, out, tiles, join, st);
    if (a.dim > 128) return launch_chunk<T, BITS, 256, 4>(a, q, out, tiles, join, st);
    return wide ? launch_chunk<T, BITS, 128, 8>(a, q, out, tiles, join, st) : launch_chunk<T, BITS, 128, 4>(a, q, out, tiles, join, st);
}

}  // namespace attn
}  // namespace lq
