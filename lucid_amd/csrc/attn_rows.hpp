// Attention of few rows (one token, or a few, of each sequence) over paged quantized keys and values.
//
// Bound by reading the cache: every byte of it is read once per tile of 16 * QT rows, and what is done with it has to fit into the
// time that takes.  So nothing of it goes through LDS: a wavefront has 32 keys at a time, in the registers in which the matrix
// instruction v_mfma_f32_16x16x32_f16 wants them, and the four wavefronts of a block have different keys.
//
//   S^T = K Q^T    A: lane (g, c) holds key c of 16, 8 columns of each slab of 32, which are consecutive codes of its row.  Which 8 is
//                  free as long as Q's fragment has the same: 16 bytes of a row serve two slabs (8 bits) or four (4 bits).
//   O^T = V^T P^T  the accumulators of S^T are B as they are: lane (g, c) has row c's probabilities of keys 4g..4g+3 of
//                  either 16, eight slots of 32 keys.  A: the lane reads the same eight keys at DIM / 16 neighbouring columns, and a few
//                  byte permutations turn them into column tiles: tile j is columns i * DIM / 16 + j, i = 0..15.
//
// The next 32 keys are requested before these are worked on, their page numbers before that.
#pragma once
#include <type_traits>

#include "paged_attention.hpp"

namespace lq {
namespace attn {

template <class T, int BITS, bool AFFINE, int DIM, int QT>
struct RowsKernel {
    static constexpr bool F32 = std::is_same_v<T, float>;
    static constexpr int PARTS = F32 ? 2 : 1;  // float16 parts of a float32
    static constexpr int R = 16 * QT, WAVES = 4, SLABS = DIM / 32, TILES = DIM / 16;
    static constexpr int KW = DIM * BITS / 128;      // dwords of a key per lane
    static constexpr int VB = DIM / 16 * BITS / 8;   // bytes of a key of V per lane
    static constexpr int VW = VB < 4 ? 1 : VB / 4;
    static constexpr int LDS_ROW = DIM + 4;          // floats
    static constexpr int LDS_BYTES = 2 * 16 * LDS_ROW * 4;

    // 32 keys
    struct Step {
        uint32_t k[2][KW];
        uint32_t v[8][VW];
        f32x4 ks[2], vs[2], vz[2];
        float kz[2];
        int at;       // the first key
        int ok;       // bit t: the 16 keys of tile t lie on a page
    };

    // first column of slab i's eight of lanes g
    static __device__ __forceinline__ int column(int i, int g) {
        if constexpr (BITS == 8) return 64 * (i / 2) + 16 * g + 8 * (i % 2);
        else if constexpr (DIM == 64) return 16 * g + 8 * i;
        else return 128 * (i / 4) + 32 * g + 8 * (i % 4);
    }

    static __device__ __forceinline__ void run(const AttnArgs& a, const T* __restrict__ q, T* __restrict__ out, float* lds) {
        const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
        const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
        const int head = blockIdx.y, group = int(a.group.d);
        clear_other_rows(a, out, blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y);
        Item it;
        if (!find_item<R>(a, blockIdx.x, false, it)) return;
        const int rows = it.s.chunk * group, row0 = it.tile * R, at = it.s.len - it.s.chunk;
        const int last_row = min(rows, row0 + R) - 1;
        const int first_token = int(a.group(unsigned(row0))), last_token = int(a.group(unsigned(last_row)));
        const Keys seen = keys_of(a, it.s, first_token, last_token);
        // this item's keys
        const int base = seen.lo & ~31, share = ((seen.hi - base + it.parts - 1) / it.parts + kMinKeys - 1) / kMinKeys * kMinKeys;
        const int from = min(seen.hi, base + it.part * share), to = min(seen.hi, from + share);
        // keys that all rows see: between them nothing is masked
        const int all_lo = a.window > 0 ? max(0, at + last_token - a.window + 1) : 0;
        const int all_hi = a.causal ? min(it.s.len, at + first_token + 1) : it.s.len;

        // queries: column c of tile t is row row0 + 16 t + c
        h8 qf[QT][SLABS][PARTS];
        float factor[QT];
        int lo[QT], hi[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int row = row0 + 16 * t + c, used = min(row, last_row);
            const int token = int(a.group(unsigned(used))), h = head * group + (used - token * group);
            const T* src = q + size_t(it.s.q0 + token) * a.ldq + size_t(h) * a.dim;
            const Keys mine = keys_of(a, it.s, token, token);
            lo[t] = mine.lo, hi[t] = mine.hi;
            factor[t] = a.scale * kLog2e;
            float x[SLABS][8];
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < SLABS; ++i) {
                const int d = column(i, g);
                const bool there = d < a.dim && row <= last_row;
                if constexpr (F32) {
                    const float4 u = there ? *reinterpret_cast<const float4*>(src + d) : float4{0, 0, 0, 0};
                    const float4 w = there ? *reinterpret_cast<const float4*>(src + d + 4) : float4{0, 0, 0, 0};
                    x[i][0] = u.x, x[i][1] = u.y, x[i][2] = u.z, x[i][3] = u.w, x[i][4] = w.x, x[i][5] = w.y, x[i][6] = w.z, x[i][7] = w.w;
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
                } else {
                    h8 u = {};
                    if (there) u = *reinterpret_cast<const h8*>(src + d);
                    // 4-bit codes leave a dword in the order 0 4 1 5 2 6 3 7
                    if constexpr (BITS == 4) u = __builtin_shufflevector(u, u, 0, 4, 1, 5, 2, 6, 3, 7);
                    qf[t][i][0] = u;
                }
            }
            if constexpr (F32) {
                // times 2^up, so that the row's largest value is in [2^13, 2^14): low parts down to 2^-24 of it are normal numbers
                top = rows4_max(top);
                const int up = max(-126, min(126, 14 - __builtin_amdgcn_frexp_expf(top)));
                factor[t] = __builtin_ldexpf(factor[t], -up);
#pragma unroll
                for (int i = 0; i < SLABS; ++i) {
                    constexpr int order[2][8] = {{0, 1, 2, 3, 4, 5, 6, 7}, {0, 4, 1, 5, 2, 6, 3, 7}};
                    Frag f[2];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float u = __builtin_ldexpf(x[i][order[BITS == 4][2 * e]], up), w = __builtin_ldexpf(x[i][order[BITS == 4][2 * e + 1]], up);
                        f[0].p[e] = to_h2(u, w);
                        f[1].p[e] = to_h2(u - float(f[0].p[e].x), w - float(f[0].p[e].y));
                    }
                    qf[t][i][0] = f[0].v, qf[t][i][1] = f[1].v;
                }
            }
        }

        f32x4 o[QT][TILES] = {};
        float m[QT], l[QT], unit = 0.f, per_unit = 0.f;
#pragma unroll
        for (int t = 0; t < QT; ++t) m[t] = -__builtin_inff(), l[t] = 0.f;

        const int row_bytes = a.dim * BITS / 8;
        const int* table = a.table + size_t(it.seq) * a.width;
        auto pages_of = [&](int key, int (&page)[2]) {
#pragma unroll
            for (int t = 0; t < 2; ++t) page[t] = key + 16 * t < to ? table[a.page_size(unsigned(key + 16 * t))] : -1;
        };
        // lane offsets: key c's codes, and four keys' columns; lanes past the head's columns read the first ones (and meet zeros of q,
        // or make columns that nobody stores)
        unsigned k_off[(KW + 3) / 4];
#pragma unroll
        for (int i = 0; i < (KW + 3) / 4; ++i) {
            const int d = column(i * (16 / BITS), g);
            k_off[i] = unsigned(c * row_bytes + (d < a.dim ? d * BITS / 8 : 0));
        }
        const unsigned v_off = unsigned(4 * g * row_bytes + (c * TILES < a.dim ? c * VB : 0));
        auto request = [&](Step& s, int key, const int (&page)[2]) {
            s.at = key, s.ok = 0;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const bool ok = unsigned(page[t]) < unsigned(a.pages);
                s.ok |= int(ok) << t;
                const int in_page = key + 16 * t - int(a.page_size(unsigned(key + 16 * t)) * a.page_size.d);
                const size_t row = ok ? (size_t(unsigned(page[t])) * unsigned(a.kv_heads) + unsigned(head)) * a.page_size.d + unsigned(in_page) : 0;
                const uint8_t* kp = a.k_codes + row * unsigned(row_bytes);
                const uint8_t* vp = a.v_codes + row * unsigned(row_bytes);
                if constexpr (KW >= 4) {
#pragma unroll
                    for (int i = 0; i < KW / 4; ++i) {
                        const uint4 w = *reinterpret_cast<const uint4*>(kp + k_off[i]);
                        s.k[t][4 * i] = w.x, s.k[t][4 * i + 1] = w.y, s.k[t][4 * i + 2] = w.z, s.k[t][4 * i + 3] = w.w;
                    }
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(kp + k_off[0]);
                    s.k[t][0] = w.x, s.k[t][1] = w.y;
                }
                s.ks[t] = *reinterpret_cast<const f32x4*>(a.k_scale + row + 4 * g);
                s.vs[t] = *reinterpret_cast<const f32x4*>(a.v_scale + row + 4 * g);
                if constexpr (AFFINE) {
                    s.kz[t] = a.k_zero[row + c];
                    s.vz[t] = *reinterpret_cast<const f32x4*>(a.v_zero + row + 4 * g);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint8_t* p = vp + v_off + unsigned(e * row_bytes);
                    uint32_t(&w)[VW] = s.v[4 * t + e];
                    if constexpr (VB == 2) {
                        w[0] = *reinterpret_cast<const uint16_t*>(p);
                    } else if constexpr (VB == 4) {
                        w[0] = *reinterpret_cast<const uint32_t*>(p);
                    } else if constexpr (VB == 8) {
                        const uint2 u = *reinterpret_cast<const uint2*>(p);
                        w[0] = u.x, w[1] = u.y;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4*>(p);
                        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
                    }
                }
            }
        };

        auto work = [&](Step& s) {
            // scores
            f32x4 sc[QT][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Offsets<BITS> off;
                if constexpr (AFFINE) off.set(s.kz[t], s.kz[t]);
#pragma unroll
                for (int x = 0; x < QT; ++x) sc[x][t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < SLABS; ++i) {
                    Frag f;
                    if constexpr (BITS == 8) {
                        const uint32_t w0 = s.k[t][2 * i], w1 = s.k[t][2 * i + 1];
                        f.p[0] = bytes01(w0, off.of1024), f.p[1] = bytes23(w0, off.of1024);
                        f.p[2] = bytes01(w1, off.of1024), f.p[3] = bytes23(w1, off.of1024);
                    } else {
                        const uint32_t w = s.k[t][i], u = w >> 8;
                        f.p[0] = nibbles0(w, off.of1024), f.p[1] = nibbles4(w, off.of64);
                        f.p[2] = nibbles0(u, off.of1024), f.p[3] = nibbles4(u, off.of64);
                    }
#pragma unroll
                    for (int x = 0; x < QT; ++x)
#pragma unroll
                        for (int p = PARTS - 1; p >= 0; --p)
                            sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.v, qf[x][i][p], sc[x][t], 0, 0, 0);
                }
            }
            const bool whole = s.at >= all_lo && s.at + 32 <= min(all_hi, to) && s.ok == 3;
            float vs[2][4], vtop = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = s.at + 16 * t + 4 * g + r;
                    vs[t][r] = s.vs[t][r];
                    // (a zero point that is no number reaches every row through the matrix product: the scale has it for those that see it)
                    if constexpr (AFFINE)
                        if (!(fabsf(s.vz[t][r]) <= 2048.f)) vs[t][r] = __builtin_nanf(""), s.vz[t][r] = 0.f;
                    // (what no row sees may be anything)
                    if (!whole && !(key >= seen.lo && key < to && (s.ok >> t & 1))) vs[t][r] = 0.f;
                    vtop = fmaxf(vtop, fabsf(vs[t][r]));
                }
            // the unit of the outputs
            vtop = rows4_max(vtop);
            if (__builtin_amdgcn_readfirstlane(int(!(vtop <= unit) || unit == 0.f))) {
                // the next power of two and another one, so that it is seldom renewed; powers that have a reciprocal
                const float top = fminf(fmaxf(__uint_as_float(__float_as_uint(vtop) & 0x7f800000u), 0x1p-100f), 0x1p124f) * 4.f;
                const float f = unit / top;
#pragma unroll
                for (int x = 0; x < QT; ++x)
#pragma unroll
                    for (int j = 0; j < TILES; ++j) o[x][j] *= f;
                unit = top, per_unit = kProbability / top;
            }
            Frag pf[QT][PARTS];
#pragma unroll
            for (int x = 0; x < QT; ++x) {
                float top = -__builtin_inff();
                float e[2][4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        e[t][r] = sc[x][t][r] * (s.ks[t][r] * factor[x]);
                        if (!whole) {
                            const int key = s.at + 16 * t + 4 * g + r;
                            if (!(key >= lo[x] && key < min(hi[x], to) && (s.ok >> t & 1))) e[t][r] = -__builtin_inff();
                        }
                        top = fmaxf(top, e[t][r]);
                    }
                top = rows4_max(top);
                if (__ballot(top > m[x] + kLazy)) {
                    const float now = fmaxf(m[x], top), f = now == m[x] ? 1.f : __builtin_amdgcn_exp2f(m[x] - now);
                    l[x] *= f;
#pragma unroll
                    for (int j = 0; j < TILES; ++j) o[x][j] *= f;
                    m[x] = now;
                }
                const float mm = m[x] == -__builtin_inff() ? 0.f : m[x];
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = __builtin_amdgcn_exp2f(e[t][r] - mm);
                        sum += p;
                        e[t][r] = p * (vs[t][r] * per_unit);
                        if (!whole && p == 0.f) e[t][r] = 0.f;
                    }
                l[x] += sum;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float u = e[t][2 * r], w = e[t][2 * r + 1];
                        const h2 h = to_h2(u, w);
                        pf[x][0].p[2 * t + r] = h;
                        if constexpr (F32) pf[x][1].p[2 * t + r] = to_h2(u - float(h.x), w - float(h.y));
                    }
            }
            // values: slots 2 i and 2 i + 1 are keys 2 i and 2 i + 1 of the lane's eight
            Offsets<BITS> off[4];
            if constexpr (AFFINE)
#pragma unroll
                for (int i = 0; i < 4; ++i) off[i].set(s.vz[i / 2][2 * (i % 2)], s.vz[i / 2][2 * (i % 2) + 1]);
            constexpr int PER = BITS == 8 ? 4 : VB == 2 ? 4 : 8;  // column tiles of a dword
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                Frag f[PER];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t x = s.v[2 * i][w], y = s.v[2 * i + 1][w];
                    if constexpr (BITS == 8) {
                        const uint32_t u0 = __builtin_amdgcn_perm(y, x, 0x05010400u), u1 = __builtin_amdgcn_perm(y, x, 0x07030602u);
                        f[0].p[i] = bytes01(u0, off[i].of1024), f[1].p[i] = bytes23(u0, off[i].of1024);
                        f[2].p[i] = bytes01(u1, off[i].of1024), f[3].p[i] = bytes23(u1, off[i].of1024);
                    } else {
#pragma unroll
                        for (int h = 0; h < PER / 4; ++h) {
                            const uint32_t u = __builtin_amdgcn_perm(y, x, h ? 0x07060302u : 0x05040100u), n = u >> 8;
                            f[4 * h].p[i] = nibbles0(u, off[i].of1024), f[4 * h + 1].p[i] = nibbles4(u, off[i].of64);
                            f[4 * h + 2].p[i] = nibbles0(n, off[i].of1024), f[4 * h + 3].p[i] = nibbles4(n, off[i].of64);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < PER; ++j)
#pragma unroll
                    for (int x = 0; x < QT; ++x)
#pragma unroll
                        for (int p = PARTS - 1; p >= 0; --p)
                            o[x][w * PER + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[j].v, pf[x][p].v, o[x][w * PER + j], 0, 0, 0);
            }
        };

        int key = from + 32 * wave;
        if (key < to) {
            Step s0, s1;
            int page[2];
            pages_of(key, page);
            request(s0, key, page);
            pages_of(key + 128, page);
            while (true) {
                request(s1, key + 128, page);
                pages_of(key + 256, page);
                work(s0);
                key += 128;
                if (key >= to) break;
                request(s0, key + 128, page);
                pages_of(key + 256, page);
                work(s1);
                key += 128;
                if (key >= to) break;
            }
        }

        // The four wavefronts' results: rows' maxima first, then sums in the order (0 + 2) + (1 + 3).
        __shared__ float s_m[WAVES][R], s_l[WAVES][R];
#pragma unroll
        for (int x = 0; x < QT; ++x) {
            l[x] = rows4_sum(l[x]);
            if (g == 0) s_m[wave][16 * x + c] = m[x], s_l[wave][16 * x + c] = l[x];
        }
        __syncthreads();
        float top[QT], total[QT];
#pragma unroll
        for (int x = 0; x < QT; ++x) {
            const int r = 16 * x + c;
            top[x] = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            const float mm = top[x] == -__builtin_inff() ? 0.f : top[x];
            float f[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) f[w] = __builtin_amdgcn_exp2f(s_m[w][r] - mm);
            total[x] = s_l[0][r] * f[0] + s_l[2][r] * f[2] + (s_l[1][r] * f[1] + s_l[3][r] * f[3]);
            const float mine = __builtin_amdgcn_exp2f(m[x] - mm) * (unit * (1.f / kProbability));
#pragma unroll
            for (int j = 0; j < TILES; ++j) o[x][j] *= mine;
        }
        auto place = [&](int slot, int r, int j) { return lds + (slot * 16 + c) * LDS_ROW + (4 * g + r) * TILES + j; };
#pragma unroll
        for (int x = 0; x < QT; ++x)
#pragma unroll
            for (int round = 2; round >= 1; round >>= 1) {
                if (wave >= round && wave < 2 * round) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < TILES; j += 4)
                            *reinterpret_cast<f32x4*>(place(wave - round, r, j)) = f32x4{o[x][j][r], o[x][j + 1][r], o[x][j + 2][r], o[x][j + 3][r]};
                }
                __syncthreads();
                if (wave < round) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < TILES; j += 4) {
                            const f32x4 v = *reinterpret_cast<const f32x4*>(place(wave, r, j));
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[x][j + e][r] += v[e];
                        }
                }
                __syncthreads();
            }
        if (wave) return;
        float* part = a.partial + partial_at(a, int(blockIdx.x), head, R, DIM);
#pragma unroll
        for (int x = 0; x < QT; ++x) {
            const int row = row0 + 16 * x + c;
            if (row > last_row) continue;
            if (it.parts > 1) {
                if (g == 0) part[R * DIM + 16 * x + c] = top[x], part[R * DIM + R + 16 * x + c] = total[x];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < TILES; j += 4)
                        *reinterpret_cast<f32x4*>(part + (16 * x + c) * DIM + (4 * g + r) * TILES + j) =
                            f32x4{o[x][j][r], o[x][j + 1][r], o[x][j + 2][r], o[x][j + 3][r]};
                continue;
            }
            const float f = total[x] == 0.f ? 0.f : 1.f / total[x];
            const int token = int(a.group(unsigned(row)));
            T* dst = out + (size_t(it.s.q0 + token) * a.heads + size_t(head * group + row - token * group)) * a.dim;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = (4 * g + r) * TILES;
                if (d >= a.dim) continue;
#pragma unroll
                for (int j = 0; j < TILES; j += 4) {
                    const f32x4 v = f32x4{o[x][j][r], o[x][j + 1][r], o[x][j + 2][r], o[x][j + 3][r]} * f;
                    if constexpr (F32) *reinterpret_cast<f32x4*>(dst + d + j) = v;
                    else *reinterpret_cast<uint2*>(dst + d + j) = uint2{as_u32(to_h2(v[0], v[1])), as_u32(to_h2(v[2], v[3]))};
                }
            }
        }
    }
};

template <class T, int BITS, bool AFFINE, int DIM, int QT>
__global__ __launch_bounds__(256, DIM <= 128 ? 2 : 1) void attn_rows_kernel(AttnArgs a, const T* __restrict__ q, T* __restrict__ out) {
    using K = RowsKernel<T, BITS, AFFINE, DIM, QT>;
    __shared__ __attribute__((aligned(16))) float lds[K::LDS_BYTES / 4];
    K::run(a, q, out, lds);
}

// Joins the parts of the tiles that have several.
template <class T, int DIM, int R>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, T* __restrict__ out) {
    Item it;
    if (!find_item<R>(a, blockIdx.x, true, it) || it.parts == 1 || it.first + it.parts > a.items) return;
    const int head = blockIdx.y, group = int(a.group.d), rows = min(R, it.s.chunk * group - it.tile * R);
    const size_t step = partial_at(a, 1, 0, R, DIM);
    const float* part = a.partial + partial_at(a, it.first, head, R, DIM);
    for (int e = int(threadIdx.x) * 4; e < rows * DIM; e += 1024) {
        const int r = e / DIM, d = e % DIM;
        if (d >= a.dim) continue;
        float top = -__builtin_inff();
        for (int i = 0; i < it.parts; ++i) top = fmaxf(top, part[i * step + R * DIM + r]);
        const float mm = top == -__builtin_inff() ? 0.f : top;
        float total = 0.f;
        f32x4 v = {0, 0, 0, 0};
        for (int i = 0; i < it.parts; ++i) {
            const float* p = part + i * step;
            const float f = __builtin_amdgcn_exp2f(p[R * DIM + r] - mm);
            total += p[R * DIM + R + r] * f;
            v += *reinterpret_cast<const f32x4*>(p + e) * f;
        }
        v *= total == 0.f ? 0.f : 1.f / total;
        const int row = it.tile * R + r, token = int(a.group(unsigned(row)));
        T* dst = out + (size_t(it.s.q0 + token) * a.heads + size_t(head * group + row - token * group)) * a.dim + d;
        if constexpr (std::is_same_v<T, float>) *reinterpret_cast<f32x4*>(dst) = v;
        else *reinterpret_cast<uint2*>(dst) = uint2{as_u32(to_h2(v[0], v[1])), as_u32(to_h2(v[2], v[3]))};
    }
}

// grid: items (tiles for the join), heads
template <class T, int BITS, int DIM, int QT>
void launch_rows(const AttnArgs& a, const T* q, T* out, int tiles, bool join, hipStream_t st) {
    if (a.k_zero) attn_rows_kernel<T, BITS, true, DIM, QT><<<dim3(a.items, a.kv_heads), 256, 0, st>>>(a, q, out);
    else attn_rows_kernel<T, BITS, false, DIM, QT><<<dim3(a.items, a.kv_heads), 256, 0, st>>>(a, q, out);
    if (join) attn_join_kernel<T, DIM, 16 * QT><<<dim3(tiles, a.kv_heads), 256, 0, st>>>(a, out);
}

template <class T, int BITS>
void launch_rows_of(const AttnArgs& a, const T* q, T* out, int tiles, int qt, bool join, hipStream_t st) {
    auto by_dim = [&](auto n) {
        constexpr int QT = decltype(n)::value;
        if (a.dim <= 64) launch_rows<T, BITS, 64, QT>(a, q, out, tiles, join, st);
        else if (a.dim <= 128) launch_rows<T, BITS, 128, QT>(a, q, out, tiles, join, st);
        else launch_rows<T, BITS, 256, QT>(a, q, out, tiles, join, st);
    };
    qt == 1 ? by_dim(std::integral_constant<int, 1>{}) : by_dim(std::integral_constant<int, 2>{});
}

}  // namespace attn
}  // namespace lq
