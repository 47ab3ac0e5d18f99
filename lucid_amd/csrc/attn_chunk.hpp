// Attention of many rows (a chunk of a prompt) over paged quantized keys and values.
//
// Bound by the matrix pipe and, more, by what the vector unit does for each score (a scale, a maximum, an exponential, a sum, a scale, a
// rounding: some ten instructions per four cycles of a matrix product) and for each code.  So a code is turned into float16 once for a
// block's 128 rows, on its way into LDS, and a wavefront has 32 rows, whose accumulators, maxima and sums stay in its registers:
//
//   S^T = K Q^T    v_mfma_f32_32x32x16_f16, A: K from LDS, lane (h, n) key n of 32, columns 8h..8h+7 of 16; B: Q in registers.
//   O^T = V^T P^T  lane (h, n) has row n's probabilities of keys 4h..4h+3 and 8+4h..8+4h+3 of 16: B as they are.  A: V^T from LDS, where
//                  a column's keys lie in that order, so that a fragment is 16 consecutive bytes.
//
// 64 keys at a time, in two sets of LDS: while one is worked on, the next keys' codes are on their way to registers, and go
// into the other one after that.  Rows of LDS are swizzled by 16 bytes, so that neither the fragments nor the writes meet in a bank.
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

template <class T, int BITS, bool AFFINE, int DIM>
struct ChunkKernel {
    static constexpr bool F32 = std::is_same_v<T, float>;
    static constexpr int PARTS = F32 ? 2 : 1;
    static constexpr int WAVES = 4, THREADS = 64 * WAVES, R = 32 * WAVES, KEYS = 64;
    static constexpr int SLABS = DIM / 16, TILES = DIM / 32;
    static constexpr int PIECES = DIM * BITS / 128;                                 // 16-byte pieces of a key's codes
    static constexpr int KP = (KEYS * PIECES + THREADS - 1) / THREADS;               // of a thread
    static constexpr int VUNITS = 8 * DIM / 4, VP = (VUNITS + THREADS - 1) / THREADS;  // 8 keys at 4 columns
    static constexpr int K_BYTES = KEYS * DIM * 2, V_BYTES = DIM * KEYS * 2, STAGE = K_BYTES + V_BYTES + 2 * KEYS * 4;
    static constexpr int LDS_BYTES = 2 * STAGE;

    static __device__ __forceinline__ int k_at(int key, int chunk) { return key * DIM * 2 + ((chunk ^ (key & 7)) << 4); }
    static __device__ __forceinline__ int v_at(int d, int chunk) { return K_BYTES + d * KEYS * 2 + ((chunk ^ ((d ^ (d >> 2)) & 7)) << 4); }

    static __device__ __forceinline__ void run(const AttnArgs& a, const T* __restrict__ q, T* __restrict__ out, char* lds) {
        const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, n = lane & 31;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int group = int(a.group.d);
        clear_other_rows(a, out, blockIdx.x, gridDim.x);
        // heads vary fastest: blocks are dealt to the 8 XCDs in turn, and those of one head find its keys in the same L2.  Of a
        // sequence's tiles the last ones, which see the most keys, come first.
        const unsigned item = blockIdx.x / unsigned(a.kv_heads);
        const int head = int(blockIdx.x - item * unsigned(a.kv_heads));
        Tile it;
        if (!find_tile<R>(a, item / unsigned(a.parts), it)) return;
        const int part = int(item % unsigned(a.parts));
        const int rows = it.s.chunk * group, row0 = it.tile * R, at = it.s.len - it.s.chunk;
        const int last_row = min(rows, row0 + R) - 1;
        const Keys seen = keys_of(a, it.s, int(a.group(unsigned(row0))), int(a.group(unsigned(last_row))));
        const int base = seen.lo & ~(KEYS - 1), share = ((seen.hi - base + a.parts - 1) / a.parts + KEYS - 1) / KEYS * KEYS;
        const int from = min(seen.hi, base + part * share), to = min(seen.hi, from + share);
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
        auto request = [&] {
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
            const size_t row = place_of(lane >> 4) + (lane & 15);
            ks_reg = a.k_scale[row], vs_reg = a.v_scale[row];
            if constexpr (AFFINE) vzero = a.v_zero[row];
        };
        bool not_finite = false;  // among the scales of the keys that were settled last
        float unit = 0.f, per_unit = 0.f, regrow = 1.f;  // regrow: what the outputs so far are to be multiplied by
        // a negative scale changes the queries' signs, and of a scale of 0 all scores are 0, the masked ones still none.  What is left
        // goes with the keys' scales, with float32 queries, which have a factor for each row, with the scores
        const float key_factor = a.scale == 0.f ? 1.f : fabsf(a.scale * kLog2e);
        const uint32_t high = BITS == 4 ? magic() : 0;
        auto settle = [&](int key, char* stage) {
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const int u = tid + i * THREADS, k = u / PIECES, piece = u % PIECES;
                if (KEYS * PIECES % THREADS && u >= KEYS * PIECES) break;
                const Offsets<BITS> off = AFFINE ? Offsets<BITS>(kz[i], kz[i]) : Offsets<BITS>();
                const uint32_t w[4] = {kreg[i].x, kreg[i].y, kreg[i].z, kreg[i].w};
                if constexpr (BITS == 8) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        Frag f;
                        f.p[0] = bytes01(w[2 * e], off.of1024), f.p[1] = bytes23(w[2 * e], off.of1024);
                        f.p[2] = bytes01(w[2 * e + 1], off.of1024), f.p[3] = bytes23(w[2 * e + 1], off.of1024);
                        *reinterpret_cast<h8*>(stage + k_at(k, 2 * piece + e)) = f.v;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        Frag f;
                        const uint32_t u1 = w[e] >> 8;
                        f.p[0] = nibbles0(w[e], high, off.of1024), f.p[1] = nibbles4(w[e], high, off.of64);
                        f.p[2] = nibbles0(u1, high, off.of1024), f.p[3] = nibbles4(u1, high, off.of64);
                        *reinterpret_cast<h8*>(stage + k_at(k, 4 * piece + e)) = f.v;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                const int u = tid + i * THREADS, chunk = u / (DIM / 4), d = u % (DIM / 4) * 4;
                if (VUNITS % THREADS && u >= VUNITS) break;
                Frag f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    Offsets<BITS> off;
                    if constexpr (AFFINE) {
                        // (a zero point that is no number reaches every row through the matrix product: the scale has it instead)
                        const float z0 = vz[i][e / 2][2 * (e % 2)], z1 = vz[i][e / 2][2 * (e % 2) + 1];
                        off = Offsets<BITS>(fabsf(z0) <= 2048.f ? z0 : 0.f, fabsf(z1) <= 2048.f ? z1 : 0.f);
                    }
                    const uint32_t x = vreg[i][2 * e], y = vreg[i][2 * e + 1];
                    if constexpr (BITS == 8) {
                        const uint32_t u0 = __builtin_amdgcn_perm(y, x, 0x05010400u), u1 = __builtin_amdgcn_perm(y, x, 0x07030602u);
                        f[0].p[e] = bytes01(u0, off.of1024), f[1].p[e] = bytes23(u0, off.of1024);
                        f[2].p[e] = bytes01(u1, off.of1024), f[3].p[e] = bytes23(u1, off.of1024);
                    } else {
                        const uint32_t u0 = __builtin_amdgcn_perm(y, x, 0x05040100u), u1 = u0 >> 8;
                        f[0].p[e] = nibbles0(u0, high, off.of1024), f[1].p[e] = nibbles4(u0, high, off.of64);
                        f[2].p[e] = nibbles0(u1, high, off.of1024), f[3].p[e] = nibbles4(u1, high, off.of64);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<h8*>(stage + v_at(d + j, chunk)) = f[j].v;
            }
            // scales; the unit of the outputs (all wavefronts come to the same)
            float vs = vs_reg;
            if (AFFINE && !(fabsf(vzero) <= 2048.f)) vs = __builtin_nanf("");
            if (!(key + lane >= seen.lo && key + lane < to && (ok >> (lane >> 4) & 1))) vs = 0.f;
            not_finite = __ballot(!(fabsf(vs) < __builtin_inff())) != 0;
            float top = fmaxf(0.f, fabsf(vs));
            top = wave_max(top);
            regrow = 1.f;
            if (__builtin_amdgcn_readfirstlane(int(!(top <= unit) || unit == 0.f))) {
                const float next = fminf(fmaxf(__uint_as_float(__float_as_uint(top) & 0x7f800000u), 0x1p-100f), 0x1p124f) * 4.f;
                regrow = unit / next, unit = next, per_unit = kProbability / next;
            }
            if (wave == 0) {
                float* to_lds = reinterpret_cast<float*>(stage + K_BYTES + V_BYTES);
                to_lds[lane] = F32 ? ks_reg : ks_reg * key_factor, to_lds[KEYS + lane] = vs * per_unit;
            }
        };

        int key = from, pages = pages_of(from);
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
                request();
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
        float m = -__builtin_inff(), l = 0.f;

        auto work = [&](const char* stage, int ok_now, float grown, bool odd) {
            const float* scales = reinterpret_cast<const float*>(stage + K_BYTES + V_BYTES);
            // (neighbouring products go to different accumulators; the next fragments are read ahead of them)
            f32x16 s[2] = {};
            {
                h8 k[2][2];
                auto read = [&](int i) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) k[i & 1][t] = *reinterpret_cast<const h8*>(stage + k_at(32 * t + n, 2 * i + h));
                };
                read(0);
#pragma unroll
                for (int i = 0; i < SLABS; ++i) {
                    if (i + 1 < SLABS) read(i + 1);
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
                        for (int t = 0; t < 2; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i & 1][t], qf[i][p], s[t], 0, 0, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 2 * PARTS, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // s becomes the exponent: the score less the row's maximum so far
            const float mm = m == -__builtin_inff() ? 0.f : -m;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 ks = *reinterpret_cast<const f32x4*>(scales + 32 * t + 8 * b + 4 * h);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        s[t][4 * b + r] = __builtin_fmaf(F32 ? s[t][4 * b + r] * factor : s[t][4 * b + r], ks[r], mm);
                }
            // keys that some rows do not see: the exponential makes them zeros
            if (!(key >= all_lo && key + KEYS <= all_hi && ok_now == 15)) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int j = key + 32 * t + 8 * (i / 4) + 4 * h + i % 4;
                        if (!(j >= lo && j < hi && (ok_now >> (2 * t + i / 8) & 1))) s[t][i] = -__builtin_inff();
                    }
            }
            float top = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
            top = halves(top, [](float x, float y) { return fmaxf(x, y); });
            float f = grown;
            const bool first = m == -__builtin_inff();
            if (__ballot(top > kLazy || (first && top > m))) {
                const float by = first ? top : fmaxf(top, 0.f);  // (-inf: no key seen yet)
                const float e = first ? 0.f : __builtin_amdgcn_exp2f(-by);
                if (by != -__builtin_inff()) {
                    m = first ? by : m + by;
                    l *= e, f *= e;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[t][i] -= by;
                }
            }
            if (__ballot(f != 1.f)) {
#pragma unroll
                for (int d = 0; d < TILES; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= f;
            }
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 vs = *reinterpret_cast<const f32x4*>(scales + KEYS + 32 * t + 8 * b + 4 * h);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = __builtin_amdgcn_exp2f(s[t][4 * b + r]);
                        sum += p;
                        s[t][4 * b + r] = p * vs[r];
                    }
                }
            l += sum;
            // a scale that is no finite number shows in the rows that see its key, not in the others
            if (odd) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int j = key + 32 * t + 8 * (i / 4) + 4 * h + i % 4;
                        if (!(j >= lo && j < hi && (ok_now >> (2 * t + i / 8) & 1))) s[t][i] = 0.f;
                    }
            }
            Frag pf[4][PARTS];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const h2 x = to_h2(s[t][i], s[t][i + 1]);
                    Frag* to_frag = pf[2 * t + i / 8];
                    to_frag[0].p[i % 8 / 2] = x;
                    if constexpr (F32) to_frag[1].p[i % 8 / 2] = to_h2(s[t][i] - float(x.x), s[t][i + 1] - float(x.y));
                }
            h8 v[4];
            auto read = [&](int x) { v[x % 4] = *reinterpret_cast<const h8*>(stage + v_at(32 * (x % TILES) + n, 2 * (x / TILES) + h)); };
            read(0), read(1);
#pragma unroll
            for (int x = 0; x < 4 * TILES; x += 2) {
                if (x + 2 < 4 * TILES) read(x + 2), read(x + 3);
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
                    for (int y = x; y < x + 2; ++y)
                        o[y % TILES] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[y % 4], pf[y / TILES][p].v, o[y % TILES], 0, 0, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2 * PARTS, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };

        float own_unit = 0.f;
        if (from < to) {
            settle(from, lds);
            __syncthreads();
            int side = 0;
            for (; key < to; key += KEYS) {
                const int ok_now = ok;
                own_unit = unit;
                const float grown = regrow;
                const bool odd = not_finite;
                const bool more = key + KEYS < to;
                if (more) {
                    locate(key + KEYS, pages);
                    pages = pages_of(key + 2 * KEYS);
                    request();
                }
                char* stage = lds + side * STAGE;
                work(stage, ok_now, grown, odd);
                side ^= 1;
                if (more) {
                    settle(key + KEYS, lds + side * STAGE);
                    __syncthreads();
                }
            }
        }
        l = halves(l, [](float x, float y) { return x + y; });
        const int row = row0 + 32 * wave + n;
        if (row > last_row) return;
        const float scale = own_unit * (1.f / kProbability) * (a.parts == 1 ? (l == 0.f ? 0.f : 1.f / l) : 1.f);
        if (a.parts > 1) {
            float* piece = a.partial + (size_t(item) * a.kv_heads + head) * kPiece<R, DIM>;
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

template <class T, int BITS, bool AFFINE, int DIM>
__global__ __launch_bounds__(256, DIM <= 128 ? 2 : 1) void attn_chunk_kernel(AttnArgs a, const T* __restrict__ q, T* __restrict__ out) {
    extern __shared__ __attribute__((aligned(16))) char chunk_lds[];
    ChunkKernel<T, BITS, AFFINE, DIM>::run(a, q, out, chunk_lds);
}

// Joins the parts of a tile's keys.
template <class T, int DIM, int R>
__global__ __launch_bounds__(256) void attn_parts_kernel(AttnArgs a, T* __restrict__ out) {
    Tile it;
    if (!find_tile<R>(a, blockIdx.x, it)) return;
    const float* first = a.partial + (size_t(blockIdx.x) * a.parts * a.kv_heads + blockIdx.y) * kPiece<R, DIM>;
    join_row<T, DIM, R>(a, out, it.s, it.tile, int(blockIdx.y), blockIdx.z * 4 + (threadIdx.x >> 6), a.parts,
                        [&](int i) { return first + size_t(i) * a.kv_heads * kPiece<R, DIM>; });
}

template <class T, int BITS, int DIM>
int launch_chunk(const AttnArgs& a, const T* q, T* out, int tiles, hipStream_t st) {
    auto go = [&](auto affine) {
        using K = ChunkKernel<T, BITS, decltype(affine)::value, DIM>;
        auto kernel = attn_chunk_kernel<T, BITS, decltype(affine)::value, DIM>;
        static DeviceOnce once;
        const int rc = allow_dynamic_lds(once, reinterpret_cast<const void*>(kernel), K::LDS_BYTES);
        if (rc) return rc;
        kernel<<<unsigned(tiles) * a.parts * a.kv_heads, K::THREADS, K::LDS_BYTES, st>>>(a, q, out);
        if (a.parts > 1) attn_parts_kernel<T, DIM, K::R><<<dim3(tiles, a.kv_heads, K::R / 4), 256, 0, st>>>(a, out);
        return int(LQ_OK);
    };
    return a.k_zero ? go(std::true_type{}) : go(std::false_type{});
}

template <class T, int BITS>
int launch_chunk_of(const AttnArgs& a, const T* q, T* out, int tiles, hipStream_t st) {
    if (a.dim <= 64) return launch_chunk<T, BITS, 64>(a, q, out, tiles, st);
    if (a.dim <= 128) return launch_chunk<T, BITS, 128>(a, q, out, tiles, st);
    return launch_chunk<T, BITS, 256>(a, q, out, tiles, st);
}

}  // namespace attn
}  // namespace lq
