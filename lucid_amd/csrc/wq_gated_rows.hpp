// Gated projections of few rows (wq_gated.hpp has the mathematics): bound by reading the weights.
//
// A block has 16 columns of both weights and 16 MT rows of x; its four wavefronts have windows of k of their own (64 lanes x 16 bytes: 128
// or 64 k of 16 weight rows, every fourth window a wavefront), so that each x that a wavefront loads meets both weights and nothing is
// shared until the sums are added in LDS.  One window is under way while another is multiplied.  Scales come with the codes: a
// lane has those of its own 16 bytes, which lie in one group, and where a window has several groups the others' come from the lanes that have
// them.  The sums of x of a group are a product with ones.
#pragma once
#include <type_traits>

#include "wq_gated.hpp"

namespace lq {
namespace gated {
namespace {

constexpr int kWaves = 4;

template <class T, int BITS, int SW, int MT>
__global__ __launch_bounds__(64 * kWaves) void gated_rows_kernel(Args a) {
    using G = WqGeom<BITS>;
    constexpr int CODES = G::CODES, WK = G::WK, NI = G::NI, GW = 1 << SW, SEG = WK / GW, IPS = NI / GW;
    constexpr bool F16 = std::is_same_v<T, _Float16>;
    constexpr int QUADS = F16 ? 1 : 2;  // 16-byte loads of x per fragment
    constexpr float UNIT = F16 ? 1.0f : kWqUnit<BITS>;
    __shared__ v4f s_y[kWaves][2][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * MT);
    const int windows = (a.K + WK - 1) / WK, groups = a.K >> a.gs_shift;
    const int n = n0 + ln < a.N ? n0 + ln : a.N - 1;
    const char* codes[2];
    const float *scales[2], *biases[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        codes[i] = reinterpret_cast<const char*>(a.w[i].packed) + size_t(n) * (size_t(a.K) * BITS / 8);
        scales[i] = a.w[i].scales + size_t(n) * groups;
        biases[i] = a.w[i].biases + size_t(n) * groups;
    }
    const T* x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = static_cast<const T*>(a.x) + size_t(m0 + t * 16 + ln) * a.K;
    struct Window {
        uint4 w[2];
        float s[2], b[2];
        uint4 x[MT][NI][QUADS];
    };
    auto load = [&](int w, Window& v) {
        // (past K: the row's first bytes, which meet zeros of x)
        const int k = w * WK + q * CODES, kc = k < a.K ? k : 0, g = kc >> a.gs_shift;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                int q_src, j_src;
                wq_source(SW, BITS == 4 ? i : 2 * i, q, q_src, j_src);
                const int at = w * WK + q_src * CODES + j_src * (32 / BITS);
#pragma unroll
                for (int h = 0; h < QUADS; ++h) {
                    v.x[t][i][h] = uint4{0u, 0u, 0u, 0u};
                    if (m0 + t * 16 + ln < a.M && at < a.K) __builtin_memcpy(&v.x[t][i][h], x[t] + at + h * 4, 16);
                }
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v.w[i] = *reinterpret_cast<const uint4*>(codes[i] + size_t(kc) * BITS / 8);
            v.s[i] = scales[i][g], v.b[i] = biases[i][g];
        }
    };
    v4f y[2][MT];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) y[i][t] = v4f{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](Window& v) {
        uint32_t wd[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            wd[i][0] = v.w[i].x, wd[i][1] = v.w[i].y, wd[i][2] = v.w[i].z, wd[i][3] = v.w[i].w;
            wq_exchange<SW>(wd[i]);
        }
#pragma unroll
        for (int e = 0; e < GW; ++e) {
            v4f acc[2][MT], sum[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[0][t] = acc[1][t] = sum[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ii = 0; ii < IPS; ++ii) {
                const int i = e * IPS + ii;
                if constexpr (F16) {
                    const _Float16 o = _Float16(1.f);
                    const v8h one{o, o, o, o, o, o, o, o}, cg = codes_f16<BITS>(wd[0], i), cu = codes_f16<BITS>(wd[1], i);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        const v8h f = slots_f16<BITS>(v.x[t][i][0]);
                        acc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, cg, acc[0][t], 0, 0, 0);
                        acc[1][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, cu, acc[1][t], 0, 0, 0);
                        sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, one, sum[t], 0, 0, 0);
                    }
                } else {
                    const v8bf one = __builtin_bit_cast(v8bf, uint4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
                    const v8bf cg = __builtin_bit_cast(v8bf, wq_codes<BITS>(wd[0], i)), cu = __builtin_bit_cast(v8bf, wq_codes<BITS>(wd[1], i));
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        float f[8];
                        __builtin_memcpy(f, v.x[t][i], 32);
                        uint32_t part[3][4];
#pragma unroll
                        for (int d = 0; d < 4; ++d)
                            wq_split3x2(BITS == 4 ? f[d] : f[2 * d], BITS == 4 ? f[d + 4] : f[2 * d + 1], part[0][d], part[1][d], part[2][d]);
#pragma unroll
                        for (int p = 0; p < 3; ++p) {
                            const v8bf fp = __builtin_bit_cast(v8bf, uint4{part[p][0], part[p][1], part[p][2], part[p][3]});
                            acc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp, cg, acc[0][t], 0, 0, 0);
                            acc[1][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp, cu, acc[1][t], 0, 0, 0);
                            sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp, one, sum[t], 0, 0, 0);
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // of the segment's first quarter
                const float s = SW == 0 ? v.s[i] : __shfl(v.s[i], ln + 16 * (e * (4 / GW)), 64);
                const float b = (SW == 0 ? v.b[i] : __shfl(v.b[i], ln + 16 * (e * (4 / GW)), 64)) - float(kWqCentre<BITS>) * s, us = UNIT * s;
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[i][t][r] = __builtin_fmaf(us, acc[i][t][r], __builtin_fmaf(b, sum[t][r], y[i][t][r]));
            }
        }
    };
    auto pin = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    Window v0, v1;
    int w = wave;
    if (w < windows) {
        load(w, v0);
        for (;;) {
            load(w + kWaves, v1);  // (past the last: bytes of the row that are not used)
            pin();
            multiply(v0);
            pin();
            if ((w += kWaves) >= windows) break;
            load(w + kWaves, v0);
            pin();
            multiply(v1);
            pin();
            if ((w += kWaves) >= windows) break;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) s_y[wave][i][t][lane] = y[i][t];
    __syncthreads();
    // a thread has row tid / 16 of each tile: element row % 4 of lane column + 16 (row / 4)
    const int col = threadIdx.x & 15, row = threadIdx.x >> 4, from = col + 16 * (row >> 2);
    if (n0 + col >= a.N) return;
    const float bg = a.w[0].bias ? a.w[0].bias[n0 + col] : 0.f, bu = a.w[1].bias ? a.w[1].bias[n0 + col] : 0.f;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = m0 + t * 16 + row;
        if (m >= a.M) return;
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int p = 0; p < kWaves; ++p) g += s_y[p][0][t][from][row & 3], u += s_y[p][1][t][from][row & 3];
        static_cast<T*>(a.out)[size_t(m) * a.N + n0 + col] = T(activate(a.act, g + bg) * (u + bu));
    }
}

template <class T>
int launch_rows(const Args& a, int bits, hipStream_t st) {
    return by_window(bits, 1 << a.gs_shift, [&](auto bits_c, auto sw) -> int {
        constexpr int BITS = decltype(bits_c)::value, SW = decltype(sw)::value;
        const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
        const dim3 grid(unsigned((a.N + 15) / 16), unsigned((a.M + 16 * mt - 1) / (16 * mt)));
        LQ_REQUIRE(grid.y <= 65535, LQ_ERR_SHAPE, "quantized_gated_matmul: %d rows", a.M);
        const auto kernel = mt == 1 ? gated_rows_kernel<T, BITS, SW, 1> : mt == 2 ? gated_rows_kernel<T, BITS, SW, 2> : gated_rows_kernel<T, BITS, SW, 4>;
        kernel<<<grid, 64 * kWaves, 0, st>>>(a);
        LQ_CHECK_LAUNCH("quantized_gated_matmul");
        return LQ_OK;
    });
}

}  // namespace
}  // namespace gated
}  // namespace lq
