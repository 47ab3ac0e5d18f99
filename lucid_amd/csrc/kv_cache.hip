// Quantizing a key / value cache as it is written, and reading it back.
//
// A row is one token's key or value of one head, quantized as a row of lq_quantize_rows_dynamic_i8 is
// (lucid/quantization/_qparams.py:198-215, _functional.py:164-182): lo = min(x, 0), hi = max(x, 0);
//   symmetric  s = max(max(|lo|, |hi|) / ((qmax - qmin) / 2), 1e-8), z = 0
//   affine     s = max((hi - lo) / (qmax - qmin), 1e-8), z = clip(qmin - rint(lo / s), qmin, qmax)
//   c = clip(rint(x / s) + z, qmin, qmax), stored as c - qmin; read back as (c - z) * s
// in IEEE float32.  Both directions move each byte once.
#include <type_traits>

#include "kv_cache.hpp"
#include "range_slots.hpp"

using namespace lq;

namespace {

constexpr float kKvEps = 1e-8f;

// eight consecutive values
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const h8 a = *reinterpret_cast<const h8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = float(a[i]);
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        reinterpret_cast<float4*>(p)[0] = float4{x[0], x[1], x[2], x[3]};
        reinterpret_cast<float4*>(p)[1] = float4{x[4], x[5], x[6], x[7]};
    } else {
        union { h2 h[4]; uint4 u; } y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.h[i] = to_h2(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = y.u;
    }
}

// over the LPR lanes of a row (a power of two; lanes of a row are neighbours)
template <int LPR, class F>
__device__ __forceinline__ float row_reduce(float v, F f) {
#pragma unroll
    for (int d = 1; d < LPR; d *= 2) v = f(v, __shfl_xor(v, d, 64));
    return v;
}

struct RowGrid {
    float s, z;
};

// LPR lanes have a row of `dim` values, eight each (lanes past it hold zeros, which change nothing: the range contains 0).
template <int LPR, bool SYMMETRIC>
__device__ __forceinline__ RowGrid grid_of(const float (&x)[8], int bits) {
    float lo = 0.f, hi = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (SYMMETRIC) hi = fmaxf(hi, fabsf(x[i]));
        else lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
        nan |= x[i] != x[i];
    }
    if (nan) hi = __builtin_inff(), lo = -__builtin_inff();  // (told from true infinities below)
    hi = row_reduce<LPR>(hi, [](float a, float b) { return fmaxf(a, b); });
    if constexpr (!SYMMETRIC) lo = row_reduce<LPR>(lo, [](float a, float b) { return fminf(a, b); });
    if (__builtin_expect(hi == __builtin_inff() || lo == -__builtin_inff(), 0)) {
        const float any = row_reduce<LPR>(nan ? 1.f : 0.f, [](float a, float b) { return fmaxf(a, b); });
        if (any != 0.f) hi = lo = __builtin_nanf("");
    }
    const int qmin = -(1 << (bits - 1)), qmax = -qmin - 1;
    const float half_range = float((double(qmax) - double(qmin)) / 2.0);
    RowGrid g;
    qparams_of(SYMMETRIC ? (hi != hi ? hi : 0.f) : lo, hi, SYMMETRIC, qmin, qmax, 1, kKvEps, half_range, &g.s, &g.z);
    return g;
}

// clip(rint(x / s) + z, qmin, qmax) - qmin.  The quotient without a division: with r the float32 next to 1 / s, x r is within
// two units of x / s in the last place, a step q + r (x - q s) brings it within one, and a second step gives the correctly
// rounded quotient (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990), which
// takes 1 / s and the remainders neither underflowing nor infinite: `plain` rows divide.  (A row's largest value of a symmetric grid
// lies on the border of two codes, so that a test whether the estimate will do fails in nearly every wavefront.)
__device__ __forceinline__ float quotient(float x, float s, float r, bool plain) {
    if (plain) return x / s;
    float q = x * r;
    q = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
    return __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
}

template <int BITS>
__device__ __forceinline__ void codes_of(const float (&x)[8], RowGrid g, uint32_t (&w)[BITS / 4]) {
    constexpr int QMIN = -(1 << (BITS - 1)), STEPS = (1 << BITS) - 1;
    const bool plain = !(g.s < 0x1p120f);  // infinite and NaN grids among them
    const float r = plain ? 0.f : 1.0f / g.s, z = g.z - float(QMIN);
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float c = __builtin_rintf(quotient(x[i], g.s, r, plain)) + z;
        if (plain) c = c != c ? float(-QMIN) : c;  // a NaN's code is 0
        c = fminf(fmaxf(c, 0.f), float(STEPS));
        w[i * BITS / 32] |= uint32_t(c) << (i * BITS % 32);
    }
}

struct CacheView {
    uint8_t* codes[2];  // keys, values
    float* scale[2];
    float* zero[2];  // NULL: symmetric
    unsigned slots, page_size, heads, dim;
    // row of the cache of a slot's head
    __device__ __forceinline__ size_t row(unsigned slot, unsigned head) const {
        const unsigned page = slot / page_size;
        return (size_t(page) * heads + head) * page_size + (slot - page * page_size);
    }
};

// One thread has eight values of a key row and of its value row, LPR neighbours a row.
template <class T, int BITS, int LPR, bool SYMMETRIC>
__global__ __launch_bounds__(256) void kv_cache_write_kernel(CacheView c, const T* __restrict__ k, const T* __restrict__ v, size_t ldk,
                                                             size_t ldv, const int* __restrict__ slots, size_t rows) {
    const size_t row = (size_t(blockIdx.x) * 256 + threadIdx.x) / LPR;
    const unsigned at = threadIdx.x % LPR * 8;
    if (row >= rows) return;
    const size_t token = row / c.heads;
    const unsigned head = unsigned(row - token * c.heads), slot = unsigned(slots[token]);
    if (slot >= c.slots) return;  // (negative ones too)
    const bool there = at < c.dim;
    const size_t to = c.row(slot, head);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float x[8] = {};
        if (there) load8((which ? v + token * ldv : k + token * ldk) + head * c.dim + at, x);
        const RowGrid g = grid_of<LPR, SYMMETRIC>(x, BITS);
        uint32_t w[BITS / 4];
        codes_of<BITS>(x, g, w);
        uint8_t* dst = c.codes[which] + (to * c.dim + at) * BITS / 8;
        if (there) {
            if constexpr (BITS == 8) *reinterpret_cast<uint2*>(dst) = uint2{w[0], w[1]};
            else *reinterpret_cast<uint32_t*>(dst) = w[0];
        }
        if (at == 0) {
            c.scale[which][to] = g.s;
            if constexpr (!SYMMETRIC) c.zero[which][to] = g.z;
        }
    }
}

template <class T, int BITS>
__global__ __launch_bounds__(256) void kv_cache_read_kernel(CacheView c, T* __restrict__ k, T* __restrict__ v,
                                                            const int* __restrict__ slots, size_t pieces) {
    const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= pieces) return;
    const unsigned per_row = c.dim / 8;
    const size_t row = i / per_row, token = row / c.heads;
    const unsigned at = unsigned(i - row * per_row) * 8, head = unsigned(row - token * c.heads), slot = unsigned(slots[token]);
    const bool there = slot < c.slots;
    const size_t from = there ? c.row(slot, head) : 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float x[8] = {};
        if (there) {
            const uint8_t* src = c.codes[which] + (from * c.dim + at) * BITS / 8;
            const float s = c.scale[which][from], z = float(-(1 << (BITS - 1))) - (c.zero[which] ? c.zero[which][from] : 0.f);
            uint32_t w[BITS / 4];
            if constexpr (BITS == 8) {
                const uint2 u = *reinterpret_cast<const uint2*>(src);
                w[0] = u.x, w[1] = u.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t*>(src);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float(w[e * BITS / 32] >> (e * BITS % 32) & ((1u << BITS) - 1)) + z) * s;
        }
        store8((which ? v : k) + row * c.dim + at, x);
    }
}

CacheView view_of(const lq_kv_cache* c) {
    CacheView v;
    v.codes[0] = c->k_codes, v.codes[1] = c->v_codes, v.scale[0] = c->k_scale, v.scale[1] = c->v_scale;
    v.zero[0] = c->k_zero, v.zero[1] = c->v_zero;
    v.slots = unsigned(c->num_pages) * unsigned(c->page_size), v.page_size = unsigned(c->page_size), v.heads = unsigned(c->kv_heads);
    v.dim = unsigned(c->head_dim);
    return v;
}

}  // namespace

extern "C" {

int lq_kv_cache_write(const lq_kv_cache* cache, const void* k, const void* v, int dtype, size_t ldk, size_t ldv, const int32_t* slots,
                      size_t tokens, lq_stream stream) {
    int rc = check_kv_cache(cache, "kv_cache_write");
    if (rc) return rc;
    if (tokens == 0) return LQ_OK;
    rc = check_kv_rows(k, ldk, dtype, "kv_cache_write", "k");
    if (!rc) rc = check_kv_rows(v, ldv, dtype, "kv_cache_write", "v");
    if (rc) return rc;
    const size_t width = size_t(cache->kv_heads) * cache->head_dim;
    LQ_REQUIRE(slots, LQ_ERR_VALUE, "kv_cache_write: slots is NULL");
    LQ_REQUIRE(ldk >= width && ldv >= width, LQ_ERR_SHAPE, "kv_cache_write: rows of %zu and %zu values for %zu", ldk, ldv, width);
    const size_t rows = tokens * cache->kv_heads;
    const int lanes = cache->head_dim / 8;
    LQ_REQUIRE(rows <= size_t(1) << 26, LQ_ERR_SHAPE, "kv_cache_write: %zu tokens of %d heads (at most 2^26 rows)", tokens, cache->kv_heads);
    const CacheView view = view_of(cache);
    by_type(dtype, cache->bits, [&](auto type, auto bits) {
        using T = decltype(type);
        auto launch = [&](auto lpr, auto symmetric) {
            constexpr int LPR = decltype(lpr)::value;
            kv_cache_write_kernel<T, decltype(bits)::value, LPR, decltype(symmetric)::value>
                <<<unsigned((rows * LPR + 255) / 256), 256, 0, as_stream(stream)>>>(view, static_cast<const T*>(k), static_cast<const T*>(v), ldk,
                                                                                    ldv, slots, rows);
        };
        auto by_lanes = [&](auto symmetric) {
            if (lanes <= 2) launch(std::integral_constant<int, 2>{}, symmetric);
            else if (lanes <= 4) launch(std::integral_constant<int, 4>{}, symmetric);
            else if (lanes <= 8) launch(std::integral_constant<int, 8>{}, symmetric);
            else if (lanes <= 16) launch(std::integral_constant<int, 16>{}, symmetric);
            else launch(std::integral_constant<int, 32>{}, symmetric);
        };
        cache->k_zero ? by_lanes(std::false_type{}) : by_lanes(std::true_type{});
    });
    LQ_CHECK_LAUNCH("kv_cache_write");
    return LQ_OK;
}

int lq_kv_cache_read(const lq_kv_cache* cache, const int32_t* slots, size_t tokens, void* k, void* v, int dtype, lq_stream stream) {
    int rc = check_kv_cache(cache, "kv_cache_read");
    if (rc) return rc;
    if (tokens == 0) return LQ_OK;
    rc = check_kv_rows(k, 0, dtype, "kv_cache_read", "k");
    if (!rc) rc = check_kv_rows(v, 0, dtype, "kv_cache_read", "v");
    if (rc) return rc;
    LQ_REQUIRE(slots, LQ_ERR_VALUE, "kv_cache_read: slots is NULL");
    const size_t pieces = tokens * cache->kv_heads * (cache->head_dim / 8);
    LQ_REQUIRE(pieces <= size_t(1) << 31, LQ_ERR_SHAPE, "kv_cache_read: %zu tokens of %zu values (at most 2^34 values)", tokens,
               size_t(cache->kv_heads) * cache->head_dim);
    const CacheView view = view_of(cache);
    by_type(dtype, cache->bits, [&](auto type, auto bits) {
        using T = decltype(type);
        kv_cache_read_kernel<T, decltype(bits)::value>
            <<<unsigned((pieces + 255) / 256), 256, 0, as_stream(stream)>>>(view, static_cast<T*>(k), static_cast<T*>(v), slots, pieces);
    });
    LQ_CHECK_LAUNCH("kv_cache_read");
    return LQ_OK;
}

}  // extern "C"
