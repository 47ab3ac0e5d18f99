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
#pragma once
#include <type_traits>

#include "paged_attention.hpp"

namespace lq {
namespace attn {

template <class T, int BITS, bool AFFINE, int DIM, int QT>
struct RowsKernel {
    static constexpr bool F32 = std::is_same_v<T, float>;
    static constexpr int PARTS = F32 ? 2 : 1;  // float16 parts of a float32
    // Probabilities are two float16 for float16 results as well: one alone makes the error 1.5 times that of the result's own rounding, and
    // the matrix pipe has the time.
    static constexpr int P_PARTS = 2;
    static constexpr int R = 16 * QT, WAVES = 4, SLABS = DIM / 32, TILES = DIM / 16;
    static constexpr int NT = rows_keys(BITS, DIM, QT) / 16, KEYS = 16 * NT, UNIT = KEYS * WAVES;
    static constexpr int KW = DIM * BITS / 128;      // dwords of a key per lane
    static constexpr int VB = DIM / 16 * BITS / 8;   // bytes of a key of V per lane
    static constexpr int VW = VB < 4 ? 1 : VB / 4;
    static constexpr int LDS_ROW = DIM + 4;          // floats
    static constexpr int ROWS = DIM <= 128 ? 16 : 8;  // rows that the wavefronts' results have room for at a time
    // queries take registers of every wavefront, or, where they are many, LDS
    static constexpr int FRAGS = QT * SLABS * PARTS;
    static constexpr bool Q_LDS = FRAGS >= 16;
    static constexpr int JOIN_BYTES = WAVES * ROWS * LDS_ROW * 4, Q_BYTES = Q_LDS ? FRAGS * 1024 : 0;
    static constexpr int LDS_BYTES = JOIN_BYTES > Q_BYTES ? JOIN_BYTES : Q_BYTES;

    // first column of slab i's eight of lanes g
    static __device__ __forceinline__ int column(int i, int g) {
        if constexpr (BITS == 8) return 64 * (i / 2) + 16 * g + 8 * (i % 2);
        else if constexpr (DIM == 64) return 16 * g + 8 * i;
        else return 128 * (i / 4) + 32 * g + 8 * (i % 4);
    }

    using Segs = Segments<R, UNIT>;

    static __device__ __forceinline__ void run(const AttnArgs& a, const T* __restrict__ q, T* __restrict__ out, float* lds) {
        const int first_row = a.q_starts[0], end_row = a.q_starts[a.batch];
        unsigned x, end;
        int head;
        typename Segs::Segment seg;
        {
            Segs segs(a);
            clear_other_rows(a, out, first_row, end_row, blockIdx.x, gridDim.x);
            const unsigned all = segs.total * unsigned(a.kv_heads), share = a.each ? segs.share() : 1u;
            if (all == 0 || blockIdx.x > (all - 1) / share) return;
            x = blockIdx.x * share, end = min(all, x + share);
            head = int(x / segs.total);
            seg = segs.at(x - unsigned(head) * segs.total);
            if (seg.tiles == 0) return;
        }
        while (true) {
            const unsigned n = min(seg.units - seg.unit, end - x);
            float* piece = n == seg.units ? nullptr : a.partial + (2 * size_t(blockIdx.x) + (seg.unit ? 0 : 1)) * kPiece<R, DIM>;
            segment(a, q, out, lds, seg, head, n, piece);
            x += n;
            if (x >= end) break;
            // on to the next tile, sequence (one that has tiles: there are units left) or head; behind eight sequences without, by a search
            seg.unit = 0;
            if (++seg.tile == int(seg.tiles)) {
                seg.tile = 0;
                for (int empty = 0;; ++empty) {
                    if (empty == 8) {
                        Segs segs(a);
                        if (segs.total == 0) return;
                        head = int(x / segs.total);
                        seg = segs.at(x - unsigned(head) * segs.total);
                        if (seg.tiles == 0) return;
                        break;
                    }
                    if (++seg.seq == a.batch) {
                        if (++head == a.kv_heads) return;
                        seg.seq = 0;
                    }
                    Segs::look(a, seg.seq, seg.s, seg.tiles, seg.units);
                    if (seg.tiles) break;
                }
            }
            __syncthreads();
        }
    }

    // `n` units of a segment from its unit on; piece: where the sums go, or NULL for the result
    static __device__ __forceinline__ void segment(const AttnArgs& a, const T* __restrict__ q, T* __restrict__ out, float* lds,
                                                   const typename Segs::Segment& it, int head, unsigned n, float* piece) {
        const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
        const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
        const int group = int(a.group.d);
        const int rows = it.s.chunk * group, row0 = it.tile * R, at = it.s.len - it.s.chunk;
        const int last_row = min(rows, row0 + R) - 1;
        const int first_token = int(a.group(unsigned(row0))), last_token = int(a.group(unsigned(last_row)));
        const Keys seen = keys_of(a, it.s, first_token, last_token);
        // these keys
        const int from = min(seen.hi, (seen.lo & ~31) + int(it.unit) * UNIT);
        const int to = a.each ? min(seen.hi, from + int(n) * UNIT) : seen.hi;
        // keys that all rows see: between them nothing is masked
        const int all_lo = a.window > 0 ? max(0, at + last_token - a.window + 1) : 0;
        const int all_hi = a.causal ? min(it.s.len, at + first_token + 1) : it.s.len;

        // queries: column c of tile t is row row0 + 16 t + c.  Requested ahead of the keys, turned into fragments behind those requests;
        // what lies past the head's columns or the last row is read from where there is something, and dropped.
        using Raw = std::conditional_t<F32, f32x4, h8>;
        Raw raw[QT][SLABS][PARTS];
        int lo[QT], hi[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int used = min(row0 + 16 * t + c, last_row), token = int(a.group(unsigned(used)));
            const T* src = q + size_t(it.s.q0 + token) * a.ldq + size_t(head * group + (used - token * group)) * a.dim;
            const Keys mine = keys_of(a, it.s, token, token);
            lo[t] = mine.lo, hi[t] = mine.hi;
#pragma unroll
            for (int i = 0; i < SLABS; ++i) {
                const int d = column(i, g);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) raw[t][i][p] = reinterpret_cast<const Raw*>(src + (d < a.dim ? d : 0))[p];
            }
        }

        const int row_bytes = a.dim * BITS / 8;
        const int* table = a.table + size_t(it.seq) * a.width;
        // Page numbers a step ahead, by a vector load (the compiler moves scalar loads to where they are used): lanes 0 to NT - 1 have those
        // of a step's tiles.  An index past the table reads 0, and its keys are past `to`.
        const auto table_rows = rows_at(table, a.width * 4);
        auto pages_of = [&](int key) {
            return int(__builtin_amdgcn_raw_buffer_load_b32(table_rows, int(a.page_size(unsigned(key + 16 * (lane & (NT - 1))))) * 4, 0, 0));
        };
        // lane offsets: key c's codes, and four keys' columns; lanes past the head's columns read the first ones (and meet zeros of q,
        // or make columns that nobody stores)
        int k_off[(KW + 3) / 4];
#pragma unroll
        for (int i = 0; i < (KW + 3) / 4; ++i) {
            const int d = column(i * (16 / BITS), g);
            k_off[i] = c * row_bytes + (d < a.dim ? d * BITS / 8 : 0);
        }
        const int v_off = 4 * g * row_bytes + (c * TILES < a.dim ? c * VB : 0);
        // 32 keys at a time.  One set of registers: each part is requested again as soon as its last reader has had it, codes of K
        // behind the scores, scales behind the probabilities, V behind the products.
        uint32_t kw[NT][KW], vw[4 * NT][VW];
        f32x4 ks[NT], vs4[NT], vz[NT];
        float kz[NT];
        size_t place[NT];  // rows of the cache where the tiles begin
        int ok = 0;       // bit t: tile t lies on a page
        auto locate = [&](int key, int pages) {
            ok = 0;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const unsigned page = unsigned(__builtin_amdgcn_readlane(pages, t));
                const bool there = key + 16 * t < to && page < unsigned(a.pages);
                ok |= int(there) << t;
                const unsigned in_page = unsigned(key + 16 * t) - a.page_size(unsigned(key + 16 * t)) * a.page_size.d;
                place[t] = there ? (size_t(page) * unsigned(a.kv_heads) + unsigned(head)) * a.page_size.d + in_page : 0;
            }
        };
        constexpr int ONCE = 2;  // non-temporal: 4352 keys of 64 sequences 112 -> 104 us
        auto request_k = [&] {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const auto rows = rows_at(a.k_codes + place[t] * unsigned(row_bytes), 16 * row_bytes);
#pragma unroll
                for (int i = 0; i < (KW + 3) / 4; ++i) {
                    if constexpr (KW >= 4) {
                        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(rows, k_off[i], 0, ONCE);
#pragma unroll
                        for (int e = 0; e < 4; ++e) kw[t][4 * i + e] = w[e];
                    } else {
                        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(rows, k_off[i], 0, ONCE);
                        kw[t][0] = w[0], kw[t][1] = w[1];
                    }
                }
                if constexpr (AFFINE) kz[t] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows_at(a.k_zero + place[t], 64), 4 * c, 0, 0));
            }
        };
        auto four = [&](const float* p) {
            return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows_at(p, 64), 16 * g, 0, 0));
        };
        auto request_scales = [&] {
#pragma unroll
            for (int t = 0; t < NT; ++t) ks[t] = four(a.k_scale + place[t]), vs4[t] = four(a.v_scale + place[t]);
        };
        auto request_v = [&] {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const auto rows = rows_at(a.v_codes + place[t] * unsigned(row_bytes), 16 * row_bytes);
                if constexpr (AFFINE) vz[t] = four(a.v_zero + place[t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t(&w)[VW] = vw[4 * t + e];
                    const int skip = e * row_bytes;
                    if constexpr (VB == 2) {
                        w[0] = __builtin_amdgcn_raw_buffer_load_b16(rows, v_off, skip, ONCE);
                    } else if constexpr (VB == 4) {
                        w[0] = __builtin_amdgcn_raw_buffer_load_b32(rows, v_off, skip, ONCE);
                    } else if constexpr (VB == 8) {
                        const u32x2 u = __builtin_amdgcn_raw_buffer_load_b64(rows, v_off, skip, ONCE);
                        w[0] = u[0], w[1] = u[1];
                    } else {
                        const u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(rows, v_off, skip, ONCE);
                        w[0] = u[0], w[1] = u[1], w[2] = u[2], w[3] = u[3];
                    }
                }
            }
        };

        int key = from + KEYS * wave, pages = pages_of(key);
        if (key < to) {
            locate(key, pages);
            pages = pages_of(key + UNIT);
            request_k(), request_scales(), request_v();
        }
        h8 qf[Q_LDS ? 1 : QT][SLABS][PARTS];
        h8* const q_lds = reinterpret_cast<h8*>(lds) + lane;
        float factor[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const bool used = row0 + 16 * t + c <= last_row;
            factor[t] = a.scale * kLog2e;
            int up = 0;
            if constexpr (F32) {
                // times 2^up, so that the row's largest value is in [2^13, 2^14): low parts down to 2^-24 of it are normal numbers
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < SLABS; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (!(used && column(i, g) < a.dim)) raw[t][i][e / 4][e % 4] = 0.f;
                        top = fmaxf(top, fabsf(raw[t][i][e / 4][e % 4]));
                    }
                top = rows4_max(top);
                up = max(-126, min(126, 14 - __builtin_amdgcn_frexp_expf(top)));
                factor[t] = __builtin_ldexpf(factor[t], -up);
            }
#pragma unroll
            for (int i = 0; i < SLABS; ++i) {
                Frag f[PARTS];
                // 4-bit codes leave a dword in the order 0 4 1 5 2 6 3 7
                constexpr int order[2][8] = {{0, 1, 2, 3, 4, 5, 6, 7}, {0, 4, 1, 5, 2, 6, 3, 7}};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n0 = order[BITS == 4][2 * e], n1 = order[BITS == 4][2 * e + 1];
                    if constexpr (F32) {
                        const float u = __builtin_ldexpf(raw[t][i][n0 / 4][n0 % 4], up), w = __builtin_ldexpf(raw[t][i][n1 / 4][n1 % 4], up);
                        f[0].p[e] = to_h2(u, w);
                        f[1].p[e] = to_h2(u - float(f[0].p[e].x), w - float(f[0].p[e].y));
                    } else {
                        f[0].p[e] = h2{raw[t][i][0][n0], raw[t][i][0][n1]};
                        if (!(used && column(i, g) < a.dim)) f[0].p[e] = h2{0, 0};
                    }
                }
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    if constexpr (!Q_LDS) qf[t][i][p] = f[p].v;
                    else if ((t * SLABS + i) % WAVES == wave) q_lds[((t * SLABS + i) * PARTS + p) * 64] = f[p].v;
                }
            }
        }
        if constexpr (Q_LDS) __syncthreads();

        f32x4 o[QT][TILES] = {};
        float m[QT], l[QT];
        Level level;
#pragma unroll
        for (int t = 0; t < QT; ++t) m[t] = -__builtin_inff(), l[t] = 0.f;

        const uint32_t high = BITS == 4 ? magic() : 0;
        for (; key < to; key += UNIT) {
            const int ok_now = ok;
            if constexpr (Q_LDS) asm volatile("" ::: "memory");  // (else all fragments of the queries are read ahead, into registers there are not)
            // scores
            f32x4 sc[QT][NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const Offsets<BITS> off = AFFINE ? Offsets<BITS>(kz[t], kz[t]) : Offsets<BITS>();
#pragma unroll
                for (int x = 0; x < QT; ++x) sc[x][t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < SLABS; ++i) {
                    Frag f;
                    if constexpr (BITS == 8) {
                        const uint32_t w0 = kw[t][2 * i], w1 = kw[t][2 * i + 1];
                        f.p[0] = bytes01(w0, off.of1024), f.p[1] = bytes23(w0, off.of1024);
                        f.p[2] = bytes01(w1, off.of1024), f.p[3] = bytes23(w1, off.of1024);
                    } else {
                        const uint32_t w = kw[t][i], u = w >> 8;
                        f.p[0] = nibbles0(w, high, off.of1024), f.p[1] = nibbles4(w, high, off.of64);
                        f.p[2] = nibbles0(u, high, off.of1024), f.p[3] = nibbles4(u, high, off.of64);
                    }
#pragma unroll
                    for (int x = 0; x < QT; ++x)
#pragma unroll
                        for (int p = PARTS - 1; p >= 0; --p)
                            sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.v, Q_LDS ? q_lds[((x * SLABS + i) * PARTS + p) * 64] : qf[Q_LDS ? 0 : x][i][p],
                                                                              sc[x][t], 0, 0, 0);
                }
            }
            locate(key + UNIT, pages);
            pages = pages_of(key + 2 * UNIT);
            request_k();
            const bool whole = key >= all_lo && key + KEYS <= min(all_hi, to) && ok_now == (1 << NT) - 1;
            float vs[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) vs[t][r] = vs4[t][r] * (1.f / kValueUnit);
            // what no row sees may be anything; and a zero point that is no number reaches every row through the matrix product: the scale
            // has it for those that see it
            if (!whole) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = key + 16 * t + 4 * g + r;
                        if constexpr (AFFINE)
                            if (!(fabsf(vz[t][r]) <= 2048.f)) vs[t][r] = __builtin_nanf(""), vz[t][r] = 0.f;
                        if (!((j >= seen.lo) & (j < to) & (ok_now >> t & 1))) vs[t][r] = level.hi;  // (its p is 0)
                    }
            }
            float least = __builtin_inff(), most = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) least = fminf(least, fabsf(vs[t][r])), most = fmaxf(most, fabsf(vs[t][r]));
            level.follow(least, most);
            Frag pf[QT][NT / 2][P_PARTS];
#pragma unroll
            for (int x = 0; x < QT; ++x) {
                // exponents: scores less the row's maximum so far
                const float mm = m[x] == -__builtin_inff() ? 0.f : -m[x];
                float e[NT][4];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) e[t][r] = __builtin_fmaf(sc[x][t][r], ks[t][r] * factor[x], mm);
                if (!whole) {
                    const int first = lo[x], count = max(0, min(hi[x], to) - first);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int j = key + 16 * t + 4 * g + r;
                            if (!((unsigned(j - first) < unsigned(count)) & (ok_now >> t & 1))) e[t][r] = -__builtin_inff();
                        }
                }
                float top = -__builtin_inff();
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fmaxf(top, e[t][r]);
                // (a lane has a quarter of the keys: only where one of them has grown by enough do the four ask each other)
                const bool first = m[x] == -__builtin_inff();
                if (__ballot(top > kMost - level.at || (first && top > m[x])) || !level.even) {
                    top += level.at;  // a bound of log2 of the largest w
                    if (!level.even) {
                        top = -__builtin_inff();
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int r = 0; r < 4; ++r) top = fmaxf(top, e[t][r] + float(level_of(vs[t][r])));
                    }
                    top = rows4_max(top) - kRenewed;
                    const float by = first ? top : fmaxf(top, 0.f);  // (-inf: no key seen yet)
                    if (by != -__builtin_inff()) {
                        const float f = first ? 0.f : __builtin_amdgcn_exp2f(-0.5f * by);  // (its square may be too small where l is large)
                        m[x] = first ? by : m[x] + by;
                        l[x] = l[x] * f * f;
#pragma unroll
                        for (int j = 0; j < TILES; ++j) o[x][j] *= f * f;
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int r = 0; r < 4; ++r) e[t][r] -= by;
                    }
                }
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = __builtin_amdgcn_exp2f(e[t][r]);
                        sum += p;
                        // (0 times anything is 0: a scale that is no number shows in the rows that see its key only)
                        e[t][r] = mul_legacy(p, vs[t][r]);
                    }
                l[x] += sum;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float u = e[t][2 * r], w = e[t][2 * r + 1];
                        const h2 h = to_h2(u, w);
                        pf[x][t / 2][0].p[2 * (t % 2) + r] = h;
                        pf[x][t / 2][1].p[2 * (t % 2) + r] = to_h2(u - float(h.x), w - float(h.y));
                    }
            }
            request_scales();
            // values: slots 2 i and 2 i + 1 are keys 2 i and 2 i + 1 of the lane's eight
            constexpr int PER = BITS == 8 ? 4 : VB == 2 ? 4 : 8;  // column tiles of a dword
#pragma unroll
            for (int k = 0; k < NT / 2; ++k) {
                Offsets<BITS> off[4];
                if constexpr (AFFINE)
#pragma unroll
                    for (int i = 0; i < 4; ++i) off[i] = Offsets<BITS>(vz[2 * k + i / 2][2 * (i % 2)], vz[2 * k + i / 2][2 * (i % 2) + 1]);
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    Frag f[PER];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t x = vw[8 * k + 2 * i][w], y = vw[8 * k + 2 * i + 1][w];
                        if constexpr (BITS == 8) {
                            const uint32_t u0 = __builtin_amdgcn_perm(y, x, 0x05010400u), u1 = __builtin_amdgcn_perm(y, x, 0x07030602u);
                            f[0].p[i] = bytes01(u0, off[i].of1024), f[1].p[i] = bytes23(u0, off[i].of1024);
                            f[2].p[i] = bytes01(u1, off[i].of1024), f[3].p[i] = bytes23(u1, off[i].of1024);
                        } else {
#pragma unroll
                            for (int h = 0; h < PER / 4; ++h) {
                                const uint32_t u = __builtin_amdgcn_perm(y, x, h ? 0x07060302u : 0x05040100u), n = u >> 8;
                                f[4 * h].p[i] = nibbles0(u, high, off[i].of1024), f[4 * h + 1].p[i] = nibbles4(u, high, off[i].of64);
                                f[4 * h + 2].p[i] = nibbles0(n, high, off[i].of1024), f[4 * h + 3].p[i] = nibbles4(n, high, off[i].of64);
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < PER; ++j)
#pragma unroll
                        for (int x = 0; x < QT; ++x)
#pragma unroll
                            for (int p = P_PARTS - 1; p >= 0; --p)
                                o[x][w * PER + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[j].v, pf[x][k][p].v, o[x][w * PER + j], 0, 0, 0);
                }
            }
            request_v();
        }

        // The wavefronts' results meet in LDS, ROWS rows at a time, and every thread adds up some columns of them.
        __shared__ float s_m[WAVES][R], s_l[WAVES][R];
#pragma unroll
        for (int x = 0; x < QT; ++x) {
            l[x] = rows4_sum(l[x]);
            if (g == 0) s_m[wave][16 * x + c] = m[x], s_l[wave][16 * x + c] = l[x];
        }
#pragma unroll
        for (int x = 0; x < QT; ++x)
#pragma unroll
            for (int part = 0; part < 16 / ROWS; ++part) {
                if (x + part && row0 + 16 * x + part * ROWS > last_row) break;
                if (Q_LDS || x + part) __syncthreads();  // (whoever reads what lies there is done)
                if (c / ROWS == part) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < TILES; j += 4)
                            *reinterpret_cast<f32x4*>(lds + (wave * ROWS + c % ROWS) * LDS_ROW + (4 * g + r) * TILES + j) =
                                f32x4{o[x][j][r], o[x][j + 1][r], o[x][j + 2][r], o[x][j + 3][r]};
                }
                __syncthreads();
                for (int e = int(threadIdx.x) * 4; e < ROWS * DIM; e += 1024) {
                    const int r = e / DIM, d = e % DIM, row = 16 * x + part * ROWS + r;
                    if (row0 + row > last_row) break;
                    const float top = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
                    const float mm = top == -__builtin_inff() ? 0.f : top;
                    f32x4 v = {0, 0, 0, 0};
                    float total = 0.f;
#pragma unroll
                    for (int w = 0; w < WAVES; ++w) {
                        const float f = __builtin_amdgcn_exp2f(0.5f * (s_m[w][row] - mm));  // (as above)
                        v += *reinterpret_cast<const f32x4*>(lds + (w * ROWS + r) * LDS_ROW + d) * (f * f);
                        total += s_l[w][row] * f * f;
                    }
                    v *= kValueUnit;
                    if (piece) {
                        if (d == 0) piece[R * DIM + row] = top, piece[R * DIM + R + row] = total;
                        *reinterpret_cast<f32x4*>(piece + row * DIM + d) = v;
                    } else if (d < a.dim) {
                        v *= total == 0.f ? 0.f : 1.f / total;
                        const int token = int(a.group(unsigned(row0 + row)));
                        T* dst = out + (size_t(it.s.q0 + token) * a.heads + size_t(head * group + row0 + row - token * group)) * a.dim + d;
                        if constexpr (F32) *reinterpret_cast<f32x4*>(dst) = v;
                        else *reinterpret_cast<uint2*>(dst) = uint2{as_u32(to_h2(v[0], v[1])), as_u32(to_h2(v[2], v[3]))};
                    }
                }
            }
    }
};

template <class T, int BITS, bool AFFINE, int DIM, int QT>
__global__ __launch_bounds__(256, DIM > 128 ? 1 : 2) void attn_rows_kernel(AttnArgs a, const T* __restrict__ q, T* __restrict__ out) {
    using K = RowsKernel<T, BITS, AFFINE, DIM, QT>;
    __shared__ __attribute__((aligned(16))) float lds[K::LDS_BYTES / 4];
    K::run(a, q, out, lds);
}

// Joins the pieces of the segments that several blocks have one of.
// APART: a block for each row of each segment, of which there are few; otherwise the blocks find the segments by the places where one
// share ends and the next begins, the first such place of a segment has it, four rows a block.
template <class T, int DIM, int R, int UNIT, bool APART>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, T* __restrict__ out) {
    Segments<R, UNIT> segs(a);
    if (segs.total == 0) return;
    const unsigned share = segs.share();
    unsigned x, head;  // first unit of the segment in the line of all
    typename Segments<R, UNIT>::Segment seg;
    if constexpr (APART) {
        head = blockIdx.y;
        unsigned tile = blockIdx.x;
        x = head * segs.total;
        for (segs.first = 0;; segs.first += 64) {
            if (segs.first >= a.batch) return;
            segs.load(a.batch);
            const unsigned upto = sum_upto(segs.tiles);
            const unsigned long long past = __ballot(upto > tile);
            if (past) {
                const int l = __builtin_ctzll(past);
                auto get = [&](unsigned v) { return unsigned(__builtin_amdgcn_readlane(int(v), l)); };
                seg.units = get(segs.units);
                tile -= get(upto) - get(segs.tiles);
                x += get(segs.upto) - get(segs.tiles) * seg.units + tile * seg.units;
                seg.tile = int(tile);
                seg.s = Sequence{int(get(unsigned(segs.s.q0))), int(get(unsigned(segs.s.chunk))), int(get(unsigned(segs.s.len)))};
                break;
            }
            tile -= of_last(upto), x += of_last(segs.upto);
        }
    } else {
        x = (blockIdx.x + 1) * share;
        if (x >= segs.total * unsigned(a.kv_heads)) return;
        head = x / segs.total;
        seg = segs.at(x - head * segs.total);
        if (seg.unit == 0 || seg.tiles == 0) return;
        x -= seg.unit;
    }
    const unsigned b0 = x / share, b1 = (x + seg.units - 1) / share;
    if (b0 == b1 || b1 >= unsigned(a.blocks) || (!APART && b0 != blockIdx.x)) return;
    // the first piece is the second of its block's two, the others are the first of theirs
    const auto piece = [&](int i) { return a.partial + (2 * size_t(b0 + i) + (i == 0)) * kPiece<R, DIM>; };
    const int parts = int(b1 - b0) + 1;
    if constexpr (APART) join_row<T, DIM, R, true>(a, out, seg.s, seg.tile, int(head), blockIdx.z, parts, piece);
    else join_row<T, DIM, R, false>(a, out, seg.s, seg.tile, int(head), blockIdx.z * 4 + (threadIdx.x >> 6), parts, piece);
}

template <class T, int BITS, int DIM, int QT>
void launch_rows(const AttnArgs& a, const T* q, T* out, int tiles, bool join, hipStream_t st) {
    if (a.k_zero) attn_rows_kernel<T, BITS, true, DIM, QT><<<a.blocks, 256, 0, st>>>(a, q, out);
    else attn_rows_kernel<T, BITS, false, DIM, QT><<<a.blocks, 256, 0, st>>>(a, q, out);
    if (!join) return;
    // few segments are in many pieces (one token of 131 072 keys, 64 pieces: 4.5 us, 6.3 as four rows a block), many in few
    constexpr int UNIT = 4 * rows_keys(BITS, DIM, QT);
    if (tiles * a.kv_heads <= 32) attn_join_kernel<T, DIM, 16 * QT, UNIT, true><<<dim3(tiles, a.kv_heads, 16 * QT), 256, 0, st>>>(a, out);
    else attn_join_kernel<T, DIM, 16 * QT, UNIT, false><<<dim3(a.blocks - 1, 1, 4 * QT), 256, 0, st>>>(a, out);
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
