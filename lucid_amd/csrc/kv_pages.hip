// Moving what a quantized key / value cache holds: whole pages into other pages, and the rows that a sequence keeps to its beginning.
// Nothing is computed: codes, scales and zero points are moved as they are.
#include "kv_cache.hpp"

using namespace lq;

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The buffers of a cache, codes of keys and values first.
struct Buffers {
    char* at[6];
};

Buffers buffers_of(const lq_kv_cache* c) {
    return {{reinterpret_cast<char*>(c->k_codes), reinterpret_cast<char*>(c->v_codes), reinterpret_cast<char*>(c->k_scale),
             reinterpret_cast<char*>(c->v_scale), reinterpret_cast<char*>(c->k_zero), reinterpret_cast<char*>(c->v_zero)}};
}

// ---------------------------------------------------------------- pages
// A page is one run of bytes in each buffer: 2 runs of `codes` 16-byte units, then 2 or 4 of `numbers`.  A block moves `chunk`
// consecutive units of one page, or, of pages that are shorter, the units of `pages` of them.
constexpr unsigned kCopyChunk = 1024;

__global__ __launch_bounds__(256) void kv_copy_kernel(Buffers b, const int* __restrict__ src, const int* __restrict__ dst, unsigned n,
                                                      unsigned num_pages, unsigned codes, unsigned numbers, FastDiv units, FastDiv blocks,
                                                      unsigned pages) {
    const unsigned group = blocks(blockIdx.x), chunk = (blockIdx.x - group * blocks.d) * kCopyChunk, first = group * pages;
#pragma unroll
    for (unsigned u = 0; u < kCopyChunk; u += 256) {
        const unsigned i = chunk + u + threadIdx.x, pair = first + units(i);
        unsigned unit = i - units(i) * units.d;
        if (pair >= n || (pages == 1 ? pair != first : pair >= first + pages)) continue;
        const unsigned from = unsigned(src[pair]), to = unsigned(dst[pair]);
        if (from >= num_pages || to >= num_pages) continue;  // (negative ones too)
        unsigned which = 0, length = codes;
        if (unit >= 2 * codes) unit -= 2 * codes, which = 2, length = numbers;
        while (unit >= length) unit -= length, ++which;
        char* const base = b.at[which];
        const u4 v = __builtin_nontemporal_load(reinterpret_cast<const u4*>(base + (size_t(from) * length + unit) * 16));
        __builtin_nontemporal_store(v, reinterpret_cast<u4*>(base + (size_t(to) * length + unit) * 16));
    }
}

// ---------------------------------------------------------------- rows
struct Rows {
    Buffers b;
    const int* table;   // [batch, width]
    const int* keep;    // [n]
    const int* starts;  // [batch + 1]
    unsigned batch, width, n, num_pages, heads, units;  // units: 16-byte pieces of a row's codes
    FastDiv page_size{1};
    char* held;  // the rows in between
};

// The row of the cache of head `head` of a sequence's place, or ~0: a place beyond the table, a page that is none.
__device__ __forceinline__ size_t row_of(const Rows& r, unsigned seq, unsigned place, unsigned head) {
    const unsigned at = r.page_size(place);
    if (place > 0x7fffffffu || at >= r.width) return ~size_t(0);
    const unsigned page = unsigned(r.table[size_t(seq) * r.width + at]);
    if (page >= r.num_pages) return ~size_t(0);
    return (size_t(page) * r.heads + head) * r.page_size.d + (place - at * r.page_size.d);
}

// The sequence of entry i of the list: the last that begins at i or before, if it does not end there.
__device__ __forceinline__ int sequence_of(const Rows& r, unsigned i) {
    int lo = -1, hi = int(r.batch);  // starts[lo] <= i < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (unsigned(r.starts[mid]) <= i) lo = mid;
        else hi = mid;
    }
    return lo >= 0 && i < unsigned(r.starts[lo + 1]) ? lo : -1;
}

// A thread per unit of 16 bytes of an entry's key or value codes of one head; the first two of them have its numbers as well.
template <bool GATHER>
__global__ __launch_bounds__(256) void kv_rows_kernel(Rows r, FastDiv per_entry, FastDiv per_head) {
    const size_t t = size_t(blockIdx.x) * 256 + threadIdx.x;
    const unsigned i = unsigned(t / per_entry.d), rest = unsigned(t - size_t(i) * per_entry.d), head = per_head(rest), unit = rest - head * per_head.d;
    if (i >= r.n) return;
    const int seq = sequence_of(r, i);
    if (seq < 0) return;
    const unsigned place = unsigned(r.keep[i]), to = i - unsigned(r.starts[seq]);
    if (place == to) return;
    const size_t from_row = row_of(r, unsigned(seq), place, head), to_row = row_of(r, unsigned(seq), to, head);
    if (from_row == ~size_t(0) || to_row == ~size_t(0)) return;
    const unsigned which = unit >= r.units, u = unit - which * r.units;
    const size_t row = GATHER ? from_row : to_row;
    u4* const codes = reinterpret_cast<u4*>(r.b.at[which]) + row * r.units + u;
    // held: the codes of all entries, then the numbers
    u4* const held = reinterpret_cast<u4*>(r.held) + (size_t(i) * r.heads + head) * (2 * r.units) + unit;
    if (GATHER) *held = *codes;
    else *codes = *held;
    if (u == 0) {
        float* const numbers = reinterpret_cast<float*>(r.held + size_t(r.n) * r.heads * r.units * 32) + ((size_t(i) * r.heads + head) * 2 + which) * 2;
        float* const scale = reinterpret_cast<float*>(r.b.at[2 + which]) + row;
        if (GATHER) numbers[0] = *scale;
        else *scale = numbers[0];
        if (r.b.at[4]) {
            float* const zero = reinterpret_cast<float*>(r.b.at[4 + which]) + row;
            if (GATHER) numbers[1] = *zero;
            else *zero = numbers[1];
        }
    }
}

}  // namespace

extern "C" {

int lq_kv_cache_copy(const lq_kv_cache* cache, const int32_t* src, const int32_t* dst, size_t pages, lq_stream stream) {
    int rc = check_kv_cache(cache, "kv_cache_copy");
    if (rc) return rc;
    if (pages == 0) return LQ_OK;
    LQ_REQUIRE(src && dst, LQ_ERR_VALUE, "kv_cache_copy: a list of pages is NULL");
    const size_t rows = size_t(cache->kv_heads) * cache->page_size;
    const size_t codes = rows * cache->head_dim * cache->bits / 128, numbers = rows / 4, units = 2 * codes + (cache->k_zero ? 4 : 2) * numbers;
    LQ_REQUIRE(units < size_t(1) << 30, LQ_ERR_SHAPE, "kv_cache_copy: pages of %zu bytes", units * 16);
    const size_t blocks = (units + kCopyChunk - 1) / kCopyChunk, together = blocks == 1 ? kCopyChunk / units : 1;
    const size_t grid = (pages + together - 1) / together * blocks;
    LQ_REQUIRE(pages < size_t(1) << 31 && grid < size_t(1) << 31, LQ_ERR_SHAPE, "kv_cache_copy: %zu pages of %zu bytes", pages, units * 16);
    kv_copy_kernel<<<unsigned(grid), 256, 0, as_stream(stream)>>>(buffers_of(cache), src, dst, unsigned(pages), unsigned(cache->num_pages),
                                                                   unsigned(codes), unsigned(numbers), FastDiv(unsigned(units)),
                                                                   FastDiv(unsigned(blocks)), unsigned(together));
    LQ_CHECK_LAUNCH("kv_cache_copy");
    return LQ_OK;
}

int lq_kv_cache_compact(const lq_kv_cache* cache, const int32_t* page_table, int table_width, int batch, const int32_t* keep, size_t kept,
                        const int32_t* starts, lq_stream stream) {
    int rc = check_kv_cache(cache, "kv_cache_compact");
    if (rc) return rc;
    LQ_REQUIRE(batch >= 0 && table_width >= 0, LQ_ERR_SHAPE, "kv_cache_compact: %d sequences of %d pages", batch, table_width);
    if (kept == 0 || batch == 0 || table_width == 0) return LQ_OK;
    LQ_REQUIRE(page_table && keep && starts, LQ_ERR_VALUE, "kv_cache_compact: a list is NULL");
    LQ_REQUIRE(kept <= size_t(cache->num_pages) * cache->page_size, LQ_ERR_SHAPE, "kv_cache_compact: %zu rows kept of a cache of %zu", kept,
               size_t(cache->num_pages) * cache->page_size);
    Rows r;
    r.b = buffers_of(cache), r.table = page_table, r.keep = keep, r.starts = starts, r.batch = unsigned(batch), r.width = unsigned(table_width);
    r.n = unsigned(kept), r.num_pages = unsigned(cache->num_pages), r.heads = unsigned(cache->kv_heads);
    r.units = unsigned(cache->head_dim * cache->bits / 128), r.page_size = FastDiv(unsigned(cache->page_size));
    const hipStream_t st = as_stream(stream);
    const auto lock = scratch_lock(st);
    void* held = nullptr;
    rc = call_buffer(10, kept * r.heads * (size_t(r.units) * 32 + 16), st, &held);
    if (rc) return rc;
    r.held = static_cast<char*>(held);
    const size_t threads = kept * r.heads * r.units * 2, grid = (threads + 255) / 256;
    LQ_REQUIRE(grid < size_t(1) << 31, LQ_ERR_SHAPE, "kv_cache_compact: %zu rows of %u heads", kept, r.heads);
    const FastDiv per_entry(r.heads * r.units * 2), per_head(r.units * 2);
    kv_rows_kernel<true><<<unsigned(grid), 256, 0, st>>>(r, per_entry, per_head);
    LQ_CHECK_LAUNCH("kv_cache_compact");
    kv_rows_kernel<false><<<unsigned(grid), 256, 0, st>>>(r, per_entry, per_head);
    LQ_CHECK_LAUNCH("kv_cache_compact");
    return LQ_OK;
}

}  // extern "C"
