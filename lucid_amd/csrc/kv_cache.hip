// Quantizing a key / value cache as it is written, and reading it back.
//
// A row is one token's key or value of one head, quantized as a row of lq_quantize_rows_dynamic_i8 is
// (lucid/quantization/_qparams.py:198-215, _functional.py:164-182): lo = min(x, 0), hi = max(x, 0);
//   symmetric  s = max(max(|lo|, |hi|) / ((qmax - qmin) / 2), 1e-8), z = 0
//   affine     s = max((hi - lo) / (qmax - qmin), 1e-8), z = clip(qmin - rint(lo / s), qmin, qmax)
//   c = clip(rint(x / s) + z, qmin, qmax), stored as c - qmin; read back as (c - z) * s
// in IEEE float32.
#include <type_traits>

#include "kv_cache.hpp"
#include "range_slots.hpp"

using namespace lq;

namespace {

constexpr float kKvEps = 1e-8f;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// eight consecutive values
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        const f4 a = __builtin_nontemporal_load(reinterpret_cast<const f4*>(p)), b = __builtin_nontemporal_load(reinterpret_cast<const f4*>(p) + 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
        const h8 a = __builtin_nontemporal_load(reinterpret_cast<const h8*>(p));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = float(a[i]);
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        __builtin_nontemporal_store(f4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f4*>(p));
        __builtin_nontemporal_store(f4{x[4], x[5], x[6], x[7]}, reinterpret_cast<f4*>(p) + 1);
    } else {
        union { h2 h[4]; h8 all; } y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.h[i] = to_h2(x[2 * i], x[2 * i + 1]);
        __builtin_nontemporal_store(y.all, reinterpret_cast<h8*>(p));
    }
}

// the larger / smaller of two, NaN if either is
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return __builtin_elementwise_minimum(a, b); }

// over the LPR lanes of a row (a power of two; lanes of a row are neighbours): lanes next to each other, pairs, quads and eights by the
// operand's own lane pattern, halves of 32 through the exchange in shared memory's network
template <int PATTERN>
__device__ __forceinline__ float lane_pattern(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), PATTERN, 0xf, 0xf, true));
}
template <int LPR, class F>
__device__ __forceinline__ float row_reduce(float v, F f) {
    v = f(v, lane_pattern<0xB1>(v));                             // 1 0 3 2
    if constexpr (LPR >= 4) v = f(v, lane_pattern<0x4E>(v));     // 2 3 0 1
    if constexpr (LPR >= 8) v = f(v, lane_pattern<0x141>(v));    // each eight mirrored
    if constexpr (LPR >= 16) v = f(v, lane_pattern<0x140>(v));   // each sixteen mirrored
    if constexpr (LPR >= 32) v = f(v, __shfl_xor(v, 16, 64));
    return v;
}

struct RowGrid {
    float s, z;
};

// LPR lanes have a row of `dim` values, eight each (lanes past it hold zeros, which change nothing: the range contains 0).
template <int LPR, bool SYMMETRIC>
__device__ __forceinline__ RowGrid grid_of(const float (&x)[8], int bits) {
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi = larger(hi, SYMMETRIC ? fabsf(x[i]) : x[i]);
        if constexpr (!SYMMETRIC) lo = smaller(lo, x[i]);
    }
    hi = row_reduce<LPR>(hi, larger);
    if constexpr (!SYMMETRIC) lo = row_reduce<LPR>(lo, smaller);
    else lo = hi != hi ? hi : 0.f;
    const int qmin = -(1 << (bits - 1)), qmax = -qmin - 1;
    const float half_range = float((double(qmax) - double(qmin)) / 2.0);
    RowGrid g;
    qparams_of(lo, hi, SYMMETRIC, qmin, qmax, 1, kKvEps, half_range, &g.s, &g.z);
    return g;
}

// clip(rint(x / s) + z, qmin, qmax) - qmin of a lane's values.  The quotient without a division: with r the float32 next to 1 / s,
// x r is within two units of x / s in the last place, a step q + r (x - q s) brings it within one, and a second step gives the
// correctly rounded quotient (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990),
// which takes 1 / s and the remainders neither underflowing nor infinite: lanes of other rows divide.  (A row's largest value of a
// symmetric grid lies on the border of two codes, so that a test whether the estimate will do fails in nearly every wavefront.)
// ONE: of a float16 value and the symmetric scale of a float16 maximum the first step gives it already, for each of the 10^9 pairs.
template <int BITS, bool ONE>
__device__ __forceinline__ void codes_of(const float (&x)[8], RowGrid g, uint32_t (&w)[BITS / 4]) {
    constexpr int QMIN = -(1 << (BITS - 1)), STEPS = (1 << BITS) - 1;
    const float r = 1.0f / g.s, z = g.z - float(QMIN);
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float q = x[i] * r;
        q = __builtin_fmaf(__builtin_fmaf(-q, g.s, x[i]), r, q);
        if constexpr (!ONE) q = __builtin_fmaf(__builtin_fmaf(-q, g.s, x[i]), r, q);
        c[i] = __builtin_rintf(q) + z;
    }
    if (__builtin_expect(!(g.s < 0x1p120f), 0)) {  // infinite and NaN grids among them
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            c[i] = __builtin_rintf(x[i] / g.s) + z;
            if (c[i] != c[i]) c[i] = float(-QMIN);  // a NaN's code is 0
        }
    }
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i * BITS / 32] |= uint32_t(fminf(fmaxf(c[i], 0.f), float(STEPS))) << (i * BITS % 32);
}

struct CacheView {
    uint8_t* codes[2];  // keys, values
    float* scale[2];
    float* zero[2];  // NULL: symmetric
    unsigned slots, heads, dim;
    FastDiv page_size{1}, by_head{1};
    // row of the cache of a slot's head
    __device__ __forceinline__ size_t row(unsigned slot, unsigned head) const {
        const unsigned page = page_size(slot);
        return (size_t(page) * heads + head) * page_size.d + (slot - page * page_size.d);
    }
};

// Both directions: a block has 256 / LPR neighbouring tokens of one head, LPR lanes a row, eight values of the key's and of the
// value's each, so that all it asks of memory is under way at once.  In the cache its rows lie together where their slots do (16
// tokens of 128 values: 2 KB of codes, 64 bytes of scales), in k and v a row is one piece.  Heads vary fastest over the blocks: those
// that run together then cover whole lines of k and v of neighbouring tokens (writing 65 536 tokens of 8 heads of 128, float16 to 8
// bits: 85 us, 96 with tokens fastest).  What streams past once (k and v, and the codes that are read back) leaves the caches to
// others: non-temporal (75 us, 73 with the shorter quotient; reading the same back 59 us instead of 74, 131 072 tokens in 4 bits 139 instead of 149).  Bound by memory:
// 403 MB at 5.5 and 6.8 TB/s, 671 MB, four fifths of them written, at 4.8; a large copy reaches 5.1.  Two tokens a lane read back
// 2 % faster at the largest size and need not be.
template <class T, int BITS, int LPR, bool SYMMETRIC>
__global__ __launch_bounds__(256) void kv_cache_write_kernel(CacheView c, const T* __restrict__ k, const T* __restrict__ v, size_t ldk,
                                                             size_t ldv, const int* __restrict__ slots, unsigned tokens) {
    const unsigned group = c.by_head(blockIdx.x), head = blockIdx.x - group * c.by_head.d;
    const unsigned token = group * (256 / LPR) + threadIdx.x / LPR, at = threadIdx.x % LPR * 8;
    if (token >= tokens) return;
    const bool there = at < c.dim;
    float x[2][8] = {};
    if (there) {
        load8(k + token * ldk + head * c.dim + at, x[0]);
        load8(v + token * ldv + head * c.dim + at, x[1]);
    }
    const unsigned slot = unsigned(slots[token]);
    if (slot >= c.slots) return;  // (negative ones too)
    const size_t to = c.row(slot, head);
    const RowGrid grids[2] = {grid_of<LPR, SYMMETRIC>(x[0], BITS), grid_of<LPR, SYMMETRIC>(x[1], BITS)};
    uint32_t words[2][BITS / 4];
    constexpr bool ONE = SYMMETRIC && std::is_same_v<T, _Float16>;
    codes_of<BITS, ONE>(x[0], grids[0], words[0]);
    codes_of<BITS, ONE>(x[1], grids[1], words[1]);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const RowGrid g = grids[which];
        const auto& w = words[which];
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

template <class T, int BITS, int LPR>
__global__ __launch_bounds__(256) void kv_cache_read_kernel(CacheView c, T* __restrict__ k, T* __restrict__ v,
                                                            const int* __restrict__ slots, unsigned tokens) {
    const unsigned group = c.by_head(blockIdx.x), head = blockIdx.x - group * c.by_head.d;
    const unsigned token = group * (256 / LPR) + threadIdx.x / LPR, at = threadIdx.x % LPR * 8;
    if (token >= tokens || at >= c.dim) return;
    const unsigned slot = unsigned(slots[token]);
    const bool there = slot < c.slots;
    const size_t from = there ? c.row(slot, head) : 0, row = size_t(token) * c.heads + head;
    uint32_t w[2][BITS / 4];
    float s[2], z[2];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const uint8_t* src = c.codes[which] + (from * c.dim + at) * BITS / 8;
        if constexpr (BITS == 8) {
            const u2 u = __builtin_nontemporal_load(reinterpret_cast<const u2*>(src));
            w[which][0] = u[0], w[which][1] = u[1];
        } else {
            w[which][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(src));
        }
        s[which] = c.scale[which][from], z[which] = c.zero[which] ? c.zero[which][from] : 0.f;
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float x[8];
        const float offset = float(-(1 << (BITS - 1))) - z[which];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = (float(w[which][e * BITS / 32] >> (e * BITS % 32) & ((1u << BITS) - 1)) + offset) * s[which];
            if (!there) x[e] = 0.f;
        }
        store8((which ? v : k) + row * c.dim + at, x);
    }
}

CacheView view_of(const lq_kv_cache* c) {
    CacheView v;
    v.codes[0] = c->k_codes, v.codes[1] = c->v_codes, v.scale[0] = c->k_scale, v.scale[1] = c->v_scale;
    v.zero[0] = c->k_zero, v.zero[1] = c->v_zero;
    v.slots = unsigned(c->num_pages) * unsigned(c->page_size), v.page_size = FastDiv(unsigned(c->page_size)), v.heads = unsigned(c->kv_heads);
    v.dim = unsigned(c->head_dim), v.by_head = FastDiv(v.heads);
    return v;
}

// f with the lanes that a row of the cache takes: a power of two
template <class F>
void by_lanes(const lq_kv_cache* c, F&& f) {
    const int lanes = c->head_dim / 8;
    if (lanes <= 2) f(std::integral_constant<int, 2>{});
    else if (lanes <= 4) f(std::integral_constant<int, 4>{});
    else if (lanes <= 8) f(std::integral_constant<int, 8>{});
    else if (lanes <= 16) f(std::integral_constant<int, 16>{});
    else f(std::integral_constant<int, 32>{});
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
    LQ_REQUIRE(tokens < size_t(1) << 26 && tokens * cache->kv_heads < size_t(1) << 26, LQ_ERR_SHAPE,
               "kv_cache_write: %zu tokens of %d heads (fewer than 2^26 rows a call)", tokens, cache->kv_heads);
    const CacheView view = view_of(cache);
    by_type(dtype, cache->bits, [&](auto type, auto bits) {
        using T = decltype(type);
        by_lanes(cache, [&](auto lpr) {
            constexpr int LPR = decltype(lpr)::value;
            const auto kernel = cache->k_zero ? kv_cache_write_kernel<T, decltype(bits)::value, LPR, false> : kv_cache_write_kernel<T, decltype(bits)::value, LPR, true>;
            kernel<<<unsigned((tokens * LPR + 255) / 256) * cache->kv_heads, 256, 0, as_stream(stream)>>>(
                view, static_cast<const T*>(k), static_cast<const T*>(v), ldk, ldv, slots, unsigned(tokens));
        });
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
    LQ_REQUIRE(tokens < size_t(1) << 26 && tokens * cache->kv_heads < size_t(1) << 26, LQ_ERR_SHAPE,
               "kv_cache_read: %zu tokens of %d heads (fewer than 2^26 rows a call)", tokens, cache->kv_heads);
    const CacheView view = view_of(cache);
    by_type(dtype, cache->bits, [&](auto type, auto bits) {
        using T = decltype(type);
        by_lanes(cache, [&](auto lpr) {
            constexpr int LPR = decltype(lpr)::value;
            kv_cache_read_kernel<T, decltype(bits)::value, LPR><<<unsigned((tokens * LPR + 255) / 256) * cache->kv_heads, 256, 0, as_stream(stream)>>>(
                view, static_cast<T*>(k), static_cast<T*>(v), slots, unsigned(tokens));
        });
    });
    LQ_CHECK_LAUNCH("kv_cache_read");
    return LQ_OK;
}

}  // extern "C"
