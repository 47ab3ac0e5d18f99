// The quantized key / value cache as its kernels see it (layout: lq_kv_cache in lucid_hip.h).
#pragma once
#include <type_traits>

#include "common.hpp"

namespace lq {

// Refuses a description that no kernel may follow: what an entry point checks before anything else.
inline int check_kv_cache(const lq_kv_cache* c, const char* name) {
    LQ_REQUIRE(c, LQ_ERR_VALUE, "%s: cache is NULL", name);
    LQ_REQUIRE(c->bits == 8 || c->bits == 4, LQ_ERR_NOT_IMPLEMENTED, "%s: codes of %d bits; 8 and 4 are built", name, c->bits);
    LQ_REQUIRE(c->num_pages >= 1 && c->kv_heads >= 1 && c->kv_heads <= 65535, LQ_ERR_SHAPE, "%s: a cache of %d pages and %d heads", name, c->num_pages, c->kv_heads);
    LQ_REQUIRE(c->page_size >= 16 && c->page_size % 16 == 0, LQ_ERR_SHAPE, "%s: pages of %d tokens; a multiple of 16 is needed", name,
               c->page_size);
    const int step = 128 / c->bits;  // (16 bytes of codes)
    LQ_REQUIRE(c->head_dim >= step && c->head_dim <= 256 && c->head_dim % step == 0, LQ_ERR_NOT_IMPLEMENTED,
               "%s: head dim %d; %d-bit codes take multiples of %d up to 256", name, c->head_dim, c->bits, step);
    LQ_REQUIRE(int64_t(c->num_pages) * c->page_size <= 0x7fffffff, LQ_ERR_SHAPE, "%s: %d pages of %d tokens are more than 2^31 - 1 slots",
               name, c->num_pages, c->page_size);
    LQ_REQUIRE(c->k_codes && c->v_codes && c->k_scale && c->v_scale && !c->k_zero == !c->v_zero, LQ_ERR_VALUE,
               "%s: the cache lacks a buffer", name);
    LQ_REQUIRE(aligned16(c->k_codes) && aligned16(c->v_codes) && aligned16(c->k_scale) && aligned16(c->v_scale) && aligned16(c->k_zero) &&
                   aligned16(c->v_zero), LQ_ERR_VALUE, "%s: the cache's buffers must be 16-byte aligned", name);
    return LQ_OK;
}

inline int check_kv_rows(const void* p, size_t ld, int dtype, const char* name, const char* what) {
    LQ_REQUIRE(dtype == LQ_F32 || dtype == LQ_F16, LQ_ERR_DTYPE, "%s: float32 and float16 are taken", name);
    LQ_REQUIRE(p, LQ_ERR_VALUE, "%s: %s is NULL", name, what);
    LQ_REQUIRE(aligned16(p) && ld % (dtype == LQ_F32 ? 4 : 8) == 0, LQ_ERR_VALUE, "%s: rows of %s must be 16-byte aligned", name, what);
    return LQ_OK;
}

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// two float32 as two float16, each rounded to nearest even (v_cvt_pk_f16_f32)
__device__ __forceinline__ h2 to_h2(float a, float b) { return __builtin_convertvector(f32x2{a, b}, h2); }

// f with a value of the type and the number of bits as constants
template <class F>
void by_type(int dtype, int bits, F&& f) {
    using B8 = std::integral_constant<int, 8>;
    using B4 = std::integral_constant<int, 4>;
    if (dtype == LQ_F32) bits == 8 ? f(float{}, B8{}) : f(float{}, B4{});
    else bits == 8 ? f(_Float16{}, B8{}) : f(_Float16{}, B4{});
}

}  // namespace lq
