// Moving what a quantized key / value cache holds: whole pages into other pages, and the rows that a sequence keeps to its beginning.
// Nothing is computed: codes, scales and zero points are moved as they are.
#include <algorithm>

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
    constexpr unsigned EACH = kCopyChunk / 256;
    u4 v[EACH];
    u4* to[EACH];
    // (no branch around the loads: all of a thread's are under way at once)
#pragma unroll
    for (unsigned u = 0; u < EACH; ++u) {
        const unsigned i = chunk + u * 256 + threadIdx.x, in_group = units(i), pair = first + in_group;
        unsigned unit = i - in_group * units.d, length = codes;
        bool there = pair < n && in_group < pages;
        const unsigned from_page = unsigned(src[there ? pair : 0]), to_page = unsigned(dst[there ? pair : 0]);
        there = there && from_page < num_pages && to_page < num_pages;  // (negative ones too)
        unsigned which = 0;
        if (unit >= 2 * codes) unit -= 2 * codes, which = 2, length = numbers;
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (unit >= length) unit -= length, ++which;
        char* const base = b.at[which];
        v[u] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(base + (size_t(there ? from_page : 0) * length + unit) * 16));
        to[u] = there ? reinterpret_cast<u4*>(base + (size_t(to_page) * length + unit) * 16) : nullptr;
    }
#pragma unroll
    for (unsigned u = 0; u < EACH; ++u)
        if (to[u]) __builtin_nontemporal_store(v[u], to[u]);
}

// ---------------------------------------------------------------- rows
// Entry i of a sequence's list moves to place i from place keep[i] >= i, so that what lies at place i is wanted by entries up to i alone: by this
// tile of the list (256 entries of one sequence) or by tiles before it.  A block reads all its rows of a head into registers, says so, waits for
// those tiles before it that read where it will write, and writes: each byte is read once and written once, in place.  Blocks take their
// tiles in the order in which they begin, and a tile says that it has read a head without waiting for any other, so every wait ends.  The word that
// counts them has the launch's number in its upper half; what a tile says is that number, so that nothing needs to be cleared between launches.
//
// Where a tile's rows lie takes six trips to memory to find out (its number, sequence, list, pages, which tiles it waits for), so a block goes on
// to the next of its heads with that, the next head's rows under way while one is written; as many heads as leave 256 blocks, one a CU.  Taking a number
// costs every block 22 ns, one after the other, so tiles are large: of 64, 128 and 256 entries (256, 512 and 1024 threads) 131 072 tokens of 8 heads of
// 128, int8, three quarters kept, take 137, 132 and 105 us, 16 sequences of up to 4096 tokens, 12 heads of 64, half kept, 34, 36 and 31; the waits cost
// nothing that can be measured.  (Gathered into scratch by one launch and put in place by another: 274 and 39 us.)  Bound by memory at 3.9 TB/s,
// half of it writes, where whole pages are copied at 4.8.
constexpr unsigned kTile = 256, kTileThreads = 1024, kMaxUnits = 8;  // entries; 16-byte units of a thread

struct Rows {
    Buffers b;
    const int* table;   // [batch, width]
    const int* keep;    // [n]
    const int* starts;  // [batch + 1]
    unsigned batch, width, n, num_pages, heads, tiles, together;  // together: heads of a block
    FastDiv page_size{1}, units{1}, by_group{1};  // units: 16-byte pieces of a row's codes, keys' and values' together; by_group: groups of heads
    unsigned long long* count;  // launches << 32 | blocks that have begun
    unsigned* read;             // [tiles * heads]: the launch that has read a tile
};

// The row of the cache of a head of a sequence's place, or kNoRow: a place beyond the table, a page that is none.
constexpr unsigned kNoRow = 0xffffffffu;  // (rows of one head are numbered by slots, fewer than 2^31)
__device__ __forceinline__ unsigned slot_of(const Rows& r, unsigned seq, unsigned place) {
    if (place > 0x7fffffffu) return kNoRow;
    const unsigned at = r.page_size(place);
    if (at >= r.width) return kNoRow;
    const unsigned page = unsigned(r.table[size_t(seq) * r.width + at]);
    return page < r.num_pages ? page * r.page_size.d + (place - at * r.page_size.d) : kNoRow;
}
__device__ __forceinline__ size_t row_of(const Rows& r, unsigned slot, unsigned head) {
    const unsigned page = r.page_size(slot);
    return (size_t(page) * r.heads + head) * r.page_size.d + (slot - page * r.page_size.d);
}

// The first tile of sequence b: there are at least as many between it and the next sequence's as its entries take.
__device__ __forceinline__ unsigned first_tile(const Rows& r, unsigned b) {
    const unsigned s = unsigned(r.starts[b]);
    return (s < r.n ? s : r.n) / kTile + b;
}

// How many of 0 .. n - 1 the first are that `is` holds for: a wavefront's lanes ask for 64 at a time.
template <class F>
__device__ __forceinline__ unsigned how_many(unsigned n, unsigned lane, F&& is) {
    unsigned lo = 0, hi = n;
    while (lo < hi) {
        const unsigned step = (hi - lo + 63) / 64, at = lo + lane * step;
        const unsigned many = unsigned(__builtin_popcountll(__builtin_amdgcn_ballot_w64(at < hi && is(at < hi ? at : lo))));
        if (many == 0) break;
        const unsigned last = lo + (many - 1) * step;
        if (last + step < hi) hi = last + step;
        lo = last + 1;
    }
    return lo;
}

template <bool ZERO>
__global__ __launch_bounds__(kTileThreads, kTileThreads / 256) void kv_compact_kernel(Rows r) {
    __shared__ unsigned s_from[kTile], s_to[kTile], s_ticket, s_launch, s_wait[2];
    __shared__ int s_moves;
    const unsigned tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) {
        const unsigned long long c = __hip_atomic_fetch_add(r.count, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_ticket = unsigned(c), s_launch = unsigned(c >> 32) + 1;
        if (unsigned(c) == gridDim.x - 1)  // all have begun: the next launch begins with its own number
            __hip_atomic_store(r.count, (unsigned long long)(s_launch) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_moves = 0;
    }
    __syncthreads();
    const unsigned tile = r.by_group(s_ticket), head0 = (s_ticket - tile * r.by_group.d) * r.together, launch = s_launch;
    const unsigned head_end = head0 + r.together < r.heads ? head0 + r.together : r.heads;
    if (tile >= r.tiles) return;  // (no block of this launch)
    // the sequence whose tiles this one is among
    const unsigned upto = how_many(r.batch, lane, [&](unsigned b) { return first_tile(r, b) <= tile; }), seq = upto ? upto - 1 : 0;
    const unsigned begin0 = unsigned(r.starts[seq]), end0 = unsigned(r.starts[seq + 1]), own_tile = tile - first_tile(r, seq);
    const unsigned begin = begin0 < r.n ? begin0 : r.n, end = end0 < r.n ? end0 : r.n, length = end > begin ? end - begin : 0;
    const unsigned i0 = own_tile < (length + kTile - 1) / kTile ? own_tile * kTile : length, count = length - i0 < kTile ? length - i0 : kTile;
    const int* const keep = r.keep + begin;
    if (tid < kTile) {
        unsigned from = kNoRow, to = kNoRow;
        if (tid < count) {
            const unsigned place = unsigned(keep[i0 + tid]);
            if (place != i0 + tid) {
                from = slot_of(r, seq, place), to = slot_of(r, seq, i0 + tid);
                if (from == kNoRow || to == kNoRow) from = to = kNoRow;
            }
        }
        s_from[tid] = from, s_to[tid] = to;
        if (from != kNoRow) s_moves = 1;
    }
    __syncthreads();
    if (!s_moves) {  // uniform
        for (unsigned h = head0 + tid; h < head_end; h += kTileThreads)
            __hip_atomic_store(&r.read[size_t(tile) * r.heads + h], launch, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return;
    }
    const unsigned all = kTile * r.units.d, half = r.units.d / 2;
    // numbers: a thread has one, of key and value scales (and zero points) of the tile's entries
    const unsigned which_number = tid / kTile, entry = tid % kTile;
    constexpr unsigned NUMBERS = ZERO ? 4 : 2;
    const bool has_number = which_number < NUMBERS && s_from[entry] != kNoRow;
    float* const numbers = reinterpret_cast<float*>(r.b.at[2 + (which_number < NUMBERS ? which_number : 0)]);
    struct Held {
        u4 v[kMaxUnits];
        float number;
    };
    // f(held, codes) of each unit of this thread's with a row that moves, where it lies in that head
    auto over = [&](const unsigned* slots, unsigned head, auto&& f) {
#pragma unroll
        for (unsigned u = 0; u < kMaxUnits; ++u) {
            const unsigned i = u * kTileThreads + tid, e = r.units(i);
            if (i < all && slots[e] != kNoRow) {
                const unsigned unit = i - e * r.units.d, which = unit >= half;
                f(u, reinterpret_cast<u4*>(r.b.at[which]) + row_of(r, slots[e], head) * half + (unit - which * half));
            }
        }
    };
    auto fetch = [&](unsigned head, Held& h) {
        over(s_from, head, [&](unsigned u, u4* at) { h.v[u] = __builtin_nontemporal_load(at); });
        if (has_number) h.number = numbers[row_of(r, s_from[entry], head)];
    };
    auto put = [&](unsigned head, const Held& h) {
        over(s_to, head, [&](unsigned u, u4* at) { __builtin_nontemporal_store(h.v[u], at); });
        if (has_number) numbers[row_of(r, s_to[entry], head)] = h.number;
    };
    auto landed = [&](Held& h) {
#pragma unroll
        for (unsigned u = 0; u < kMaxUnits; ++u) asm volatile("" : "+v"(h.v[u]));
        asm volatile("" : "+v"(h.number));
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    Held held[2];
#pragma unroll
    for (unsigned k = 0; k < 2; ++k) {
        held[k].number = 0.f;
#pragma unroll
        for (unsigned u = 0; u < kMaxUnits; ++u) held[k].v[u] = u4{0u, 0u, 0u, 0u};
    }
    fetch(head0, held[0]);
    if (wave == 0) {
        // the entries before this tile that lie where it writes, `count` at most: the tiles of the first and the last of them
        const unsigned first = how_many(i0, lane, [&](unsigned j) { return unsigned(keep[j]) < i0; });
        unsigned many = 0;
#pragma unroll
        for (unsigned j = 0; j < kTile; j += 64) {
            const unsigned at = first + j + lane;
            many += unsigned(__builtin_popcountll(__builtin_amdgcn_ballot_w64(at < i0 && unsigned(keep[at < i0 ? at : 0]) < i0 + count)));
        }
        if (lane == 0) s_wait[0] = first / kTile, s_wait[1] = many ? (first + many - 1) / kTile + 1 : first / kTile;
    }
    auto turn = [&](unsigned head, Held& now, Held& next) {
        landed(now);
        __syncthreads();  // everybody's rows are in registers
        if (tid == 0) __hip_atomic_store(&r.read[size_t(tile) * r.heads + head], launch, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (head + 1 < head_end) fetch(head + 1, next);
        if (wave == 0) {
            const unsigned t1 = s_wait[1];
            for (unsigned t = s_wait[0] + lane; t < t1; t += 64) {
                const unsigned* const flag = &r.read[size_t(tile - own_tile + t) * r.heads + head];
                while (__hip_atomic_load(flag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != launch) __builtin_amdgcn_s_sleep(2);
            }
        }
        __syncthreads();
        put(head, now);
    };
    for (unsigned head = head0; head < head_end; head += 2) {
        turn(head, held[0], held[1]);
        if (head + 1 < head_end) turn(head + 1, held[1], held[0]);
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
    LQ_REQUIRE(pages < size_t(1) << 31 && grid < size_t(1) << 24, LQ_ERR_SHAPE, "kv_cache_copy: %zu pages of %zu bytes", pages, units * 16);
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
    LQ_REQUIRE(kept < size_t(1) << 31, LQ_ERR_SHAPE, "kv_cache_compact: %zu rows kept", kept);  // (more than the cache has, where pages are shared)
    Rows r;
    r.b = buffers_of(cache), r.table = page_table, r.keep = keep, r.starts = starts, r.batch = unsigned(batch), r.width = unsigned(table_width);
    r.n = unsigned(kept), r.num_pages = unsigned(cache->num_pages), r.heads = unsigned(cache->kv_heads);
    r.units = FastDiv(unsigned(cache->head_dim * cache->bits / 64)), r.page_size = FastDiv(unsigned(cache->page_size));
    r.tiles = unsigned(kept / kTile) + r.batch;
    static_assert(kTile * 32 <= kTileThreads * kMaxUnits && kTile * 4 <= kTileThreads, "rows of 256 codes of 8 bits; their numbers");
    r.together = unsigned(std::min<size_t>(r.heads, std::max<size_t>(1, size_t(r.tiles) * r.heads / 256)));
    const unsigned groups = (r.heads + r.together - 1) / r.together;
    r.by_group = FastDiv(groups);
    const size_t grid = size_t(r.tiles) * groups, words_needed = size_t(r.tiles) * r.heads;
    LQ_REQUIRE(grid < (size_t(1) << 32) / kTileThreads, LQ_ERR_SHAPE, "kv_cache_compact: %zu rows of %u sequences and %u heads", kept, r.batch,
               r.heads);  // (a launch has fewer than 2^32 threads)
    const hipStream_t st = as_stream(stream);
    const auto lock = scratch_lock(st);
    void* words = nullptr;
    size_t fresh = 0;
    rc = kept_buffer(10, 8 + words_needed * 4, size_t(1) << 18, st, &words, &fresh);
    if (!rc) rc = lq_fill_bytes(words, 0, fresh, stream);
    if (rc) return rc;
    r.count = static_cast<unsigned long long*>(words), r.read = reinterpret_cast<unsigned*>(r.count + 1);
    const auto kernel = cache->k_zero ? kv_compact_kernel<true> : kv_compact_kernel<false>;
    kernel<<<unsigned(grid), kTileThreads, 0, st>>>(r);
    LQ_CHECK_LAUNCH("kv_cache_compact");
    return LQ_OK;
}

}  // extern "C"
