// Attention of new tokens over the pages of a quantized key / value cache (lq_paged_attention).
#include <algorithm>
#include <type_traits>

#include "paged_attention.hpp"

using namespace lq;

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
    AttnArgs a{};
    a.k_codes = c->k_codes, a.v_codes = c->v_codes, a.k_scale = c->k_scale, a.v_scale = c->v_scale, a.k_zero = c->k_zero, a.v_zero = c->v_zero;
    a.table = page_table, a.q_starts = q_starts, a.kv_lens = kv_lens, a.ldq = ldq;
    a.page_size = FastDiv(unsigned(c->page_size)), a.group = FastDiv(unsigned(heads / c->kv_heads));
    a.pages = c->num_pages, a.kv_heads = c->kv_heads, a.dim = c->head_dim;
    a.tokens = tokens, a.heads = heads, a.batch = batch, a.width = table_width, a.causal = causal != 0, a.scale = scale;
    const int group = heads / c->kv_heads, sequences = std::max(1, std::min(batch, tokens));  // (of no sequence: the rows' zeros)
    const int64_t all_rows = int64_t(tokens) * group, most = int64_t(table_width) * c->page_size;  // keys of a sequence
    // A place is at least -tokens and below `most`: a window of both together reaches every key, and kernels count places in 32 bits.
    a.window = window < most + tokens ? window : 0;
    const int dim = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
    // The longest chunk, or a guess at it: equally many tokens each, but for what one sequence can have if each of the others has one where that is 8192
    // rows and more (a prompt of 3700 tokens among 255 single ones, four query heads a key head, 765 -> 508 us; of 2000 367 either way).
    const int one = tokens - (sequences - 1);
    const int chunk = max_chunk ? std::min(max_chunk, tokens) : int64_t(one) * group >= 8192 ? one : (tokens + sequences - 1) / sequences;
    // Sequences of more than few_rows rows go to attn_chunk_kernel, the others to attn_rows_kernel, which reads the keys once for every 32
    // rows.  us, rows / chunk kernel, 8 heads of 128, 8 bits: 16 float16 sequences of up to 4096 keys 64 rows 62 / 59, 80 rows 76 / 64, 128 rows
    // 93 / 78; 64 of up to 1024 64 rows 70 / 77, 80 rows 92 / 82; 16 float32 ones of up to 4096 80 rows 87 / 89, 96 rows 90 / 89, 128 rows 104 / 103, 192 rows
    // 152 / 144; one float16 sequence of 16 384 80 rows 39 / 49, 128 rows 41 / 52, 192 rows 57 / 58.  Heads of 64 and 256 cross over at the same rows within
    // some 10 % of the time, but for float32 above 128 (128 rows of 16 sequences 198 / 291: the chunk kernel's registers spill).
    // Where there can be both, both are launched and each takes its own; otherwise either takes all (one prompt of 8192 among 31 single tokens: the chunk
    // kernel alone 1245 us, both 1000).  There are chunks alone where the longest leaves no room for a sequence without tokens, and
    // 512 rows in the mean: an idle launch is lost for little otherwise.
    const int few_rows = batch == 1 ? 128 : dtype == LQ_F32 ? 96 : 64;
    const bool chunks = int64_t(chunk) * group > few_rows, alike = int64_t(sequences) * chunk - tokens < chunk && all_rows >= int64_t(sequences) * 512;
    const bool few = !chunks || (sequences > 1 && !alike);
    hipStream_t st = as_stream(stream);
    auto lock = scratch_lock(st);
    auto room = [&](size_t floats) {
        void* p = nullptr;
        // (in a recording one buffer for all calls on the stream, which run one after another)
        const int rc = kept_buffer(9, floats * sizeof(float), 0, st, &p, nullptr);
        a.partial = static_cast<float*>(p);
        return rc;
    };
    if (chunks) {
        // Tiles of 128 rows, two blocks a CU, one of which has the CU to itself when the other has ended; or of 256, one block a CU, in
        // which a code is turned into float16 for twice as many rows.  The latter where blocks are alike and fill the places: one
        // sequence of 1024 rows or more, in two rounds of blocks or more or behind three times as many keys.  us, 128 / 256 rows, 32 heads of 128 on
        // 8, float16: 8192 tokens of 16 384 2425 / 2347, 8192 of 8192 887 / 826, 1000 of 16 000 420 / 401, 2048 of 8192 403 / 397; but 2048 of 4096
        // 187 / 205, 1000 of 1000 50 / 57, and of four sequences of 1934 to 8192 keys 308 / 351 (of four of 8192 429 / 401: their lengths are
        // on the device).  float32: 3183 / 2855, 1123 / 1011, 544 / 486, 512 / 479, 259 / 248, 64 / 63.
        const int64_t rows = int64_t(chunk) * group;
        const bool wide = dim == 128 && batch == 1 && rows >= 1024 && (rows * c->kv_heads >= 512 * 256 || most >= 4 * int64_t(chunk));
        const int R = wide ? 256 : 128;
        a.min_rows = few ? few_rows + 1 : 1, a.max_rows = 0x7fffffff;
        // (a block at least: of no sequence it clears the rows)
        const int tiles = std::max(1, int(std::min<int64_t>(sequences, all_rows / a.min_rows) + all_rows / R));
        // (parts of 256 / 384 / 512 keys at least: 3 chunks of 333, float32, 53 / 50 / 60 us; 8 of 300 over up to 700 keys 80 / 72 / 72)
        a.each = (dim > 128 || wide ? 1 : 2) * 256, a.least = 384;
        // (four rounds of blocks of one sequence are left whole: joining none of 129 tiles of 8 heads takes 25 us)
        const bool join = most > a.least && !(batch == 1 && rows * c->kv_heads >= int64_t(4) * a.each * R);
        if (!join) a.least = 0x40000000;
        a.blocks = tiles + (join ? (2 * a.each + c->kv_heads - 1) / c->kv_heads : 0);
        LQ_REQUIRE(int64_t(a.blocks) * c->kv_heads <= 0xffffff, LQ_ERR_NOT_IMPLEMENTED, "paged_attention: %d tiles of queries for %d heads", tiles,
                   c->kv_heads);
        if (join) {
            // (parts of tiles of several, see part_keys; its sums' rounding, 2^-24 of them for every 64 sequences, is worth less than 64 parts of all heads)
            a.pieces = std::min(a.blocks, (4 * a.each + 64) / c->kv_heads + 1);
            rc = room(size_t(a.pieces) * c->kv_heads * R * (dim + 2));
            if (rc) return rc;
        }
        auto launch = [&](auto type, auto bits) {
            using T = decltype(type);
            rc = attn::launch_chunk_of<T, decltype(bits)::value>(a, static_cast<const T*>(q), static_cast<T*>(out), wide, tiles, join, st);
        };
        by_type(dtype, c->bits, launch);
        if (rc) return rc;
        LQ_CHECK_LAUNCH("paged_attention");
    }
    if (few) {
        // (the mean of those that the longest one leaves, or of all)
        const int others = !chunks ? chunk : max_chunk ? (tokens - chunk) / (sequences - 1) : tokens / sequences;
        const int qt = int64_t(others) * group <= 16 ? 1 : 2, rows = 16 * qt;
        a.min_rows = 1, a.max_rows = chunks ? few_rows : 0x7fffffff;
        const int tiles = sequences + int((chunks ? std::min<int64_t>(all_rows, int64_t(sequences) * few_rows) : all_rows) / rows);
        LQ_REQUIRE(int64_t(tiles) * c->kv_heads * (most / 128 + 1) < 0x7fffffff, LQ_ERR_NOT_IMPLEMENTED,
                   "paged_attention: %d tiles of queries for %lld keys of %d heads are more than one call takes", tiles, (long long)most, c->kv_heads);
        // Up to 512 keys a block has a whole segment: four steps of each wavefront, where joining pieces takes another launch (one token
        // of 197 keys 10.3 -> 7.6 us; 256 sequences of up to 500 keys, 2048 segments, 56 -> 47), unless segments are so many that each block's way to its
        // own counts (2048 sequences, 16 384 segments, 801 -> 395 as shares).  Beyond, as many shares as blocks are resident.
        const int resident = (dim > 128 ? 1 : 2) * 256;
        const bool join = most > 512 || int64_t(tiles) * c->kv_heads > 8 * resident;
        a.each = join ? resident : 0, a.least = 1;
        a.blocks = join ? resident : tiles * a.kv_heads;
        if (join) {
            rc = room(size_t(2) * a.blocks * rows * (dim + 2));
            if (rc) return rc;
        }
        auto launch = [&](auto type, auto bits) {
            using T = decltype(type);
            attn::launch_rows_of<T, decltype(bits)::value>(a, static_cast<const T*>(q), static_cast<T*>(out), tiles, qt, join, st);
        };
        by_type(dtype, c->bits, launch);
        LQ_CHECK_LAUNCH("paged_attention");
    }
    return LQ_OK;
}
