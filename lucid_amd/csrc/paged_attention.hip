// Attention of new tokens over the pages of a quantized key / value cache (lq_paged_attention).
#include <type_traits>

#include "kv_cache.hpp"

using namespace lq;

namespace {

struct AttnArgs {
    const uint8_t* k_codes;
    const uint8_t* v_codes;
    const float* k_scale;
    const float* v_scale;
    const float* k_zero;
    const float* v_zero;
    const int* table;
    const int* q_starts;
    const int* kv_lens;
    size_t ldq;
    int pages, page_size, kv_heads, dim, tokens, heads, batch, width, causal, window;
    float scale;
};

// a wavefront per row and head: lane = key for the scores, then lane = column for the values
template <class T, int BITS>
__global__ __launch_bounds__(64) void paged_attention_simple_kernel(AttnArgs a, const T* __restrict__ q, T* __restrict__ out) {
    __shared__ float sq[256], sp[64];
    __shared__ int srow[64];
    const int lane = threadIdx.x, head = blockIdx.x % a.heads, row = blockIdx.x / a.heads;
    const int kv = head / (a.heads / a.kv_heads);
    int b = -1;
    for (int i = 0; i < a.batch; ++i)
        if (row >= a.q_starts[i] && row < a.q_starts[i + 1]) b = i;
    float acc[4] = {}, m = -__builtin_inff(), l = 0.f;
    if (b >= 0) {
        const int len = a.kv_lens[b] < a.width * a.page_size ? a.kv_lens[b] : a.width * a.page_size;
        const int place = len - a.q_starts[b + 1] + row;
        const int end = a.causal && place + 1 < len ? place + 1 : len;
        const int begin = a.window > 0 && place - a.window + 1 > 0 ? place - a.window + 1 : 0;
        for (int d = lane; d < a.dim; d += 64) sq[d] = float(q[size_t(row) * a.ldq + size_t(head) * a.dim + d]);
        __syncthreads();
        const float qmin = -float(1 << (BITS - 1));
        for (int j0 = begin; j0 < end; j0 += 64) {
            const int j = j0 + lane;
            int r = -1;
            float s = -__builtin_inff();
            if (j < end) {
                const int page = a.table[size_t(b) * a.width + j / a.page_size];
                if (unsigned(page) < unsigned(a.pages)) {
                    const size_t at = (size_t(page) * a.kv_heads + kv) * a.page_size + j % a.page_size;
                    r = page * a.page_size + j % a.page_size;
                    const float z = qmin - (a.k_zero ? a.k_zero[at] : 0.f);
                    float dot = 0.f;
                    for (int d = 0; d < a.dim; ++d) {
                        const size_t e = at * a.dim + d;
                        const unsigned u = BITS == 8 ? a.k_codes[e] : a.k_codes[e / 2] >> (e % 2 * 4) & 15;
                        dot = __builtin_fmaf(sq[d], float(u) + z, dot);
                    }
                    s = dot * a.k_scale[at] * a.scale;
                }
            }
            float top = s;
            for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
            const float mn = fmaxf(m, top), use = mn == -__builtin_inff() ? 0.f : mn;
            const float p = r < 0 ? 0.f : __expf(s - use), f = __expf(m - use);
            float sum = p;
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
            l = l * f + sum, m = mn;
            __syncthreads();
            sp[lane] = p, srow[lane] = r;
            __syncthreads();
            for (int i = 0; i < 4; ++i) acc[i] *= f;
            for (int t = 0; t < 64; ++t) {
                if (srow[t] < 0) continue;
                const size_t at = (size_t(srow[t] / a.page_size) * a.kv_heads + kv) * a.page_size + srow[t] % a.page_size;
                const float z = qmin - (a.v_zero ? a.v_zero[at] : 0.f), w = sp[t] * a.v_scale[at];
                for (int i = 0; i < 4; ++i) {
                    const int d = lane + 64 * i;
                    if (d >= a.dim) break;
                    const size_t e = at * a.dim + d;
                    const unsigned u = BITS == 8 ? a.v_codes[e] : a.v_codes[e / 2] >> (e % 2 * 4) & 15;
                    acc[i] = __builtin_fmaf(w, float(u) + z, acc[i]);
                }
            }
        }
    }
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < a.dim) out[(size_t(row) * a.heads + head) * a.dim + d] = T(l == 0.f ? 0.f : acc[i] / l);
    }
}

}  // namespace

extern "C" int lq_paged_attention(const lq_kv_cache* c, const void* q, size_t ldq, void* out, int dtype, int tokens, int heads, int batch,
                                  const int32_t* page_table, int table_width, const int32_t* q_starts, const int32_t* kv_lens, float scale,
                                  int causal, int window, int max_chunk, lq_stream stream) {
    int rc = check_kv_cache(c, "paged_attention");
    if (rc) return rc;
    LQ_REQUIRE(tokens >= 0 && batch >= 0 && table_width >= 0 && window >= 0 && max_chunk >= 0, LQ_ERR_VALUE,
               "paged_attention: %d tokens, %d sequences, %d pages each, window %d, chunks of %d", tokens, batch, table_width, window, max_chunk);
    LQ_REQUIRE(heads >= 1 && heads % c->kv_heads == 0, LQ_ERR_SHAPE, "paged_attention: %d query heads for %d key heads", heads, c->kv_heads);
    if (tokens == 0) return LQ_OK;
    rc = check_kv_rows(q, ldq, dtype, "paged_attention", "q");
    if (!rc) rc = check_kv_rows(out, 0, dtype, "paged_attention", "out");
    if (rc) return rc;
    LQ_REQUIRE(ldq >= size_t(heads) * c->head_dim, LQ_ERR_SHAPE, "paged_attention: q rows of %zu values for %d heads of %d", ldq, heads, c->head_dim);
    LQ_REQUIRE(q_starts && (batch == 0 || (kv_lens && (page_table || table_width == 0))), LQ_ERR_VALUE, "paged_attention: NULL pointer");
    LQ_REQUIRE(int64_t(tokens) * heads <= 1 << 25, LQ_ERR_SHAPE, "paged_attention: %d tokens of %d heads (at most 2^25 rows)", tokens, heads);
    LQ_REQUIRE(int64_t(table_width) * c->page_size <= 0x40000000, LQ_ERR_SHAPE, "paged_attention: %d pages of %d tokens (at most 2^30 keys)",
               table_width, c->page_size);
    AttnArgs a;
    a.k_codes = c->k_codes, a.v_codes = c->v_codes, a.k_scale = c->k_scale, a.v_scale = c->v_scale, a.k_zero = c->k_zero, a.v_zero = c->v_zero;
    a.table = page_table, a.q_starts = q_starts, a.kv_lens = kv_lens, a.ldq = ldq;
    a.pages = c->num_pages, a.page_size = c->page_size, a.kv_heads = c->kv_heads, a.dim = c->head_dim;
    a.tokens = tokens, a.heads = heads, a.batch = batch, a.width = table_width, a.causal = causal, a.window = window, a.scale = scale;
    auto launch = [&](auto type, auto bits) {
        using T = decltype(type);
        paged_attention_simple_kernel<T, decltype(bits)::value>
            <<<unsigned(tokens * heads), 64, 0, as_stream(stream)>>>(a, static_cast<const T*>(q), static_cast<T*>(out));
    };
    using B8 = std::integral_constant<int, 8>;
    using B4 = std::integral_constant<int, 4>;
    if (dtype == LQ_F32) c->bits == 8 ? launch(float{}, B8{}) : launch(float{}, B4{});
    else c->bits == 8 ? launch(_Float16{}, B8{}) : launch(_Float16{}, B4{});
    LQ_CHECK_LAUNCH("paged_attention");
    return LQ_OK;
}
