// Attention of new tokens over the pages of a quantized key / value cache (lq_paged_attention): what its kernels share.
//
// Query rows of one sequence that read the same key / value head are the rows token * group + (head within the group),
// group = heads / kv_heads: whatever the group, one row of the matrix products each.  A row at place p = kv_len - chunk + token
// sees the keys [max(0, p - window + 1), min(kv_len, p + 1)).
//
// The mathematics.  Codes are whole numbers below 2^8, which float16 holds exactly, so that the matrix instruction gets them as they
// are and the scales follow in float32:
//     S_j = (scale log2 e) k_scale_j sum_d q_d (c_jd - z_j)
//     o_d = sum_j w_j (c'_jd - z'_j) / sum_j p_j,   p_j = 2^(S_j - m), w_j = p_j v_scale_j
// A product of a float16 and a code is exact in float32, and so is c - z.  float16 queries enter as they are, float32 ones as two float16
// of 22 bits together (times a power of two for each row, so that neither part is subnormal where it counts).  So do the w_j, for float16
// results too (one float16 alone makes the error 1.4 times that of the result's own rounding).  The sums of the p_j are not rounded.
// What keeps a w_j's 22 bits whatever the scales is that a row's m goes by the keys that the row itself has seen, and by their w_j: it is
// renewed where one may pass 2^15, so that it is 2^7 then, and two float16 hold a number to 2^-25 of 1.  Mostly the scales of the keys of a step
// are within 2^8 of each other; then the exponents' maximum and one `Level` for all of them bound the w_j.  In other steps each key's scale counts
// (scales of all keys 2^-3 to 2^3 times as large, at random: chunks take a quarter longer, few rows up to 6 %).
#pragma once
#include "kv_cache.hpp"
#include "wave_reduce.hpp"

namespace lq {

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
    FastDiv page_size{1}, group{1};
    int pages, kv_heads, dim, tokens, heads, batch, width, causal, window;
    int blocks;
    int each;      // of so many blocks each has a share of the units, at least `least`; 0: a segment
    int least;
    int pieces;    // parts of tiles of several that there is room for
    int min_rows, max_rows;  // sequences of fewer or more rows are another launch's
    float scale;
    float* partial;  // pieces of segments
};

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace attn {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMost = 15.f, kRenewed = 7.f;  // log2 of the largest p v_scale of a row that is let be, and of what it becomes otherwise
constexpr float kValueUnit = 0x1p16f;          // v_scale is kept in this, so that p is no subnormal beside the largest ones

__device__ __forceinline__ h2 as_h2(uint32_t v) { return __builtin_bit_cast(h2, v); }
__device__ __forceinline__ uint32_t as_u32(h2 v) { return __builtin_bit_cast(uint32_t, v); }

// v_mul_legacy_f32: a product in which 0 times anything is 0
__device__ float mul_legacy(float a, float b) __asm("llvm.amdgcn.fmul.legacy");

// The sum over the lanes up to this one, within 16 of them and then across, by the operand's own lane patterns: six of them cost what
// one exchange through shared memory's network does, and this stands in every block's way to its first load.
template <int PATTERN, int ROWS = 0xf, class N>
__device__ __forceinline__ N add_lanes(N v) {
    return v + __builtin_bit_cast(N, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), PATTERN, ROWS, 0xf, false));
}
template <class N>
__device__ __forceinline__ N sum_upto(N v) {
    v = add_lanes<0x111>(v), v = add_lanes<0x112>(v), v = add_lanes<0x114>(v), v = add_lanes<0x118>(v);  // 1, 2, 4, 8 lanes before
    return add_lanes<0x143, 0xc>(add_lanes<0x142, 0xa>(v));  // the last lane of the row of 16, of the half
}
// the last lane's number
template <class N>
__device__ __forceinline__ N of_last(N v) { return __builtin_bit_cast(N, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63)); }

// f over the four lanes of one number in the four rows of 16 lanes; every lane gets it
template <class F>
__device__ __forceinline__ float rows4(float v, F f) {
    auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(x[0]), __uint_as_float(x[1]));
    x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float rows4_max(float v) {
    return rows4(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float rows4_sum(float v) {
    return rows4(v, [](float a, float b) { return a + b; });
}

// |scale| is below 2^level_of(scale) and at least half of it (but for infinity; NaN and what is too small to bound p by count as 2^-84)
__device__ __forceinline__ int level_of(float scale) { return __builtin_amdgcn_frexp_expf(fminf(fmaxf(fabsf(scale), 0x1p-84f), 0x1p112f)); }
// What bounds the values' scales of a step's keys.
struct Level {
    float at = -16.f;    // all of them are at most 2^at = hi
    bool even = true;    // and above lo = 2^(at - 8); if not, each key's own counts
    float hi = 0x1p-16f, lo = 0x1p-24f;
    // a lane has some of them, from `least` to `most`
    __device__ __forceinline__ void follow(float least, float most) {
        even = true;
        if (!__ballot(!(most <= hi && least > lo))) return;
        const int level = __builtin_amdgcn_readfirstlane(level_of(wave_max(fmaxf(most, 0.f)))) + 1;  // (room for what grows a little)
        at = float(level), hi = __builtin_ldexpf(1.f, level), lo = __builtin_ldexpf(1.f, level - 8);
        even = !__ballot(!(most <= hi && least > lo));
    }
};

struct Sequence {
    int q0, chunk, len;  // first row of q, new tokens, keys
};
__device__ __forceinline__ Sequence sequence_of(const AttnArgs& a, int b) {
    Sequence s;
    const int most = a.width * int(a.page_size.d);
    s.q0 = max(0, min(a.q_starts[b], a.tokens));
    s.chunk = max(0, min(a.q_starts[b + 1], a.tokens) - s.q0);
    s.len = max(0, min(a.kv_lens[b], most));
    return s;
}
// keys that some row of tokens first .. last of a sequence sees: [lo, hi), empty as lo = hi
struct Keys {
    int lo, hi;
};
__device__ __forceinline__ Keys keys_of(const AttnArgs& a, const Sequence& s, int first, int last) {
    const int at = s.len - s.chunk;
    Keys k;
    k.hi = a.causal ? max(0, min(s.len, at + last + 1)) : s.len;
    k.lo = a.window > 0 ? min(k.hi, max(0, at + first - a.window + 1)) : 0;
    return k;
}

// What the blocks of a launch do is found by each of them from the lengths, which only the device knows.  A segment is a tile of
// R rows of a sequence with one key head; it is `units` units of UNIT keys long, and all segments of a launch, head by head, make one line of
// units, which the blocks share out evenly: where a sequence ends, a block goes on with the next one.  A segment that several
// blocks have a piece of is joined by another launch.  `each` = 0: a block per segment, for short sequences.
template <int R, int UNIT>
struct Segments {
    const AttnArgs& a;
    const int lane;
    unsigned total;     // units of a head
    // 64 sequences, one a lane: units of their segments, tiles, units of one
    int first;          // the first of them
    unsigned upto, tiles, units;
    Sequence s;

    // units up to the end of a lane's run of `run` sequences
    int run;
    unsigned run_upto;

    __device__ __forceinline__ explicit Segments(const AttnArgs& args) : a(args), lane(threadIdx.x & 63) {
        run = max(1, (a.batch + 63) / 64);
        if (run == 1) {
            first = 0, load(a.batch);
            run_upto = upto;
        } else {
            unsigned sum = 0;
#pragma unroll 4
            for (int i = 0; i < run; ++i) {
                const int b = lane * run + i;
                Sequence x;
                unsigned n, u;
                look(a, min(b, a.batch - 1), x, n, u);
                sum += b < a.batch ? n * u : 0u;
            }
            run_upto = sum_upto(sum);
        }
        total = of_last(run_upto);
    }
    // a sequence of the batch, its tiles, and the units of each
    static __device__ __forceinline__ void look(const AttnArgs& a, int b, Sequence& x, unsigned& n, unsigned& u) {
        x = sequence_of(a, b);
        const int rows = x.chunk * int(a.group.d);
        n = rows < a.min_rows || rows > a.max_rows ? 0u : unsigned(rows + R - 1) / R;
        const Keys k = keys_of(a, x, 0, x.chunk - 1);
        u = a.each ? max(1u, unsigned(k.hi - (k.lo & ~31) + UNIT - 1) / UNIT) : 1u;
    }
    // 64 sequences from `first` on, those before `end`
    __device__ __forceinline__ void load(int end) {
        s = Sequence{0, 0, 0}, tiles = 0, units = 1;
        if (first + lane < end) look(a, first + lane, s, tiles, units);
        upto = sum_upto(tiles * units);
    }
    struct Segment {
        int seq, tile;
        unsigned unit, units;  // the unit asked for, and how many there are
        unsigned tiles;        // of the sequence
        Sequence s;
    };
    // the segment of unit `x` < total of a head; no tiles: there is none (lengths that change meanwhile)
    __device__ __forceinline__ Segment at(unsigned x) {
        if (run > 1) {
            const int l = __builtin_ctzll(__ballot(run_upto > x));
            if (l) x -= unsigned(__builtin_amdgcn_readlane(int(run_upto), l - 1));
            first = l * run, load(a.batch);
        }
        while (true) {
            const unsigned long long past = __ballot(upto > x);
            if (past) {
                const int l = __builtin_ctzll(past);
                auto get = [&](unsigned v) { return unsigned(__builtin_amdgcn_readlane(int(v), l)); };
                Segment g;
                g.seq = first + l, g.units = get(units), g.tiles = get(tiles);
                const unsigned k = x - (get(upto) - g.tiles * g.units);
                g.tile = int(g.units == 1 ? k : k / g.units), g.unit = k - unsigned(g.tile) * g.units;
                g.s = Sequence{int(get(unsigned(s.q0))), int(get(unsigned(s.chunk))), int(get(unsigned(s.len)))};
                return g;
            }
            x -= of_last(upto);
            first += 64;
            if (first >= a.batch) return Segment{0, 0, 0, 1, 0, {0, 0, 0}};
            load(a.batch);
        }
    }
    // units that each of a.each blocks takes
    __device__ __forceinline__ unsigned share() const {
        return max(unsigned(a.least), (total * unsigned(a.kv_heads) + unsigned(a.each) - 1) / unsigned(a.each));
    }
};

// Tiles of R rows of a launch, of each sequence's the last one first (it sees the most keys), their keys in parts, a block each.
struct Tile {
    int seq, tile, part, parts;
    int first;  // number of its first part among those of tiles of several
    Sequence s;
};
// Parts of `extent` keys where none shall have more than `most`, or hardly more: whoever counts them counts alike, and up to `most` it is 1.
__device__ __forceinline__ unsigned parts_of(unsigned extent, unsigned most) {
    return max(1u, unsigned(__builtin_ceilf(float(extent) * __builtin_amdgcn_rcpf(float(most)) * (1.f - 0x1p-20f))));
}
// The most keys of a part: so many that there are about twice as many parts of all tiles as places for blocks (a.each), where lengths differ
// the blocks that end early then take another.  (Tiles of several parts, each longer than one, then have 4 a.each parts at most, for all heads.)  Up to 64 sequences of about the same length (one a lane; 0 tiles: not this launch's)
// have equal parts, which come in whole rounds: a lane each tries the longest in 1, 2, 3, ... parts, and the shortest sum of the rounds'
// lengths counts, in keys, of which a block costs kBlock besides its own and one whose part is joined kPart more (us, parts of the share / in
// rounds: 4 chunks of 512 over 8192 keys 458 / 440, one of 300 115 / 92; but 4 over 1934 to 8192 keys 310 / 321).
constexpr float kBlock = 128.f, kPart = 320.f, kAlike = 0.8f;
__device__ __forceinline__ unsigned part_keys(const AttnArgs& a, float keys, unsigned tiles, unsigned extent, int lane) {
    const float heads = float(a.kv_heads), places = float(a.each);
    const unsigned share = max(unsigned(a.least), unsigned(fminf(keys * heads / (2.f * places), 0x1p30f)) + 1u);
    const unsigned longest = unsigned(wave_max(tiles ? float(extent) : 0.f)), all = of_last(sum_upto(tiles));
    if (a.batch > 64 || keys < kAlike * float(all) * float(longest)) return share;
    const int in = lane < 32 ? lane + 1 : 16 * (lane - 30);
    const unsigned most = max(unsigned(a.least), (longest / unsigned(in) + 64u) & ~63u);
    unsigned n = 0;
    for (int i = 0; i < a.batch; ++i)
        n += unsigned(__builtin_amdgcn_readlane(int(tiles), i)) * parts_of(unsigned(__builtin_amdgcn_readlane(int(extent), i)), most);
    const float rounds = __builtin_ceilf(float(n) * heads / places) * (float(most) + kBlock + (n > all ? kPart : 0.f));
    const float cost = n > unsigned(a.blocks) || (n > all && n > unsigned(a.pieces)) ? __builtin_inff() : rounds;
    const unsigned long long best = __ballot(cost == wave_min(cost));
    return unsigned(__builtin_amdgcn_readlane(int(most), __builtin_ctzll(best)));
}
// Part number `id`, or with `whole` tile number `id`.  False: there is none.
template <int R>
__device__ __forceinline__ bool find_tile(const AttnArgs& a, unsigned id, bool whole, Tile& it) {
    const int lane = threadIdx.x & 63;
    Sequence s{0, 0, 0};
    unsigned tiles = 0, extent = 0;
    auto load = [&](int b) {
        s = Sequence{0, 0, 0};
        if (b < a.batch) s = sequence_of(a, b);
        const int rows = s.chunk * int(a.group.d);
        tiles = rows < a.min_rows || rows > a.max_rows ? 0u : unsigned(rows + R - 1) / R;
        const Keys k = keys_of(a, s, 0, s.chunk - 1);
        extent = unsigned(k.hi - (k.lo & ~63));
    };
    float keys = 0.f;
    for (int first = 0; first < a.batch; first += 64) {
        load(first + lane);
        keys += float(tiles) * float(extent);
    }
    keys = of_last(sum_upto(keys));
    const unsigned most = part_keys(a, keys, tiles, extent, lane);
    unsigned before = 0, tiles_before = 0, split_before = 0;
    for (int first = 0; first < a.batch; first += 64) {
        if (a.batch > 64) load(first + lane);
        const unsigned parts = parts_of(extent, most), split = parts > 1 ? tiles * parts : 0u;
        const unsigned upto = sum_upto(tiles * parts), tiles_to = sum_upto(tiles), split_to = sum_upto(split);
        const unsigned long long past = __ballot((whole ? tiles_before + tiles_to : before + upto) > id);
        if (past) {
            const int l = __builtin_ctzll(past);
            auto get = [&](unsigned v) { return unsigned(__builtin_amdgcn_readlane(int(v), l)); };
            const unsigned n = get(tiles), p = get(parts), begin = before + get(upto) - n * p;
            const unsigned k = whole ? id - (tiles_before + get(tiles_to) - n) : (id - begin) / p;
            it.seq = first + l, it.tile = int(n - 1 - k), it.parts = int(p), it.part = whole ? 0 : int(id - begin - k * p);
            it.first = int(split_before + get(split_to) - get(split) + k * p);
            it.s = Sequence{int(get(unsigned(s.q0))), int(get(unsigned(s.chunk))), int(get(unsigned(s.len)))};
            return true;
        }
        before += of_last(upto);
        tiles_before += of_last(tiles_to);
        split_before += of_last(split_to);
    }
    return false;
}

// A piece of a segment: R rows of DIM sums over its keys, then the rows' maxima and sums of probabilities.  A block has room for two, the
// first for a segment that begins in a block before it, the second for one that goes on in the next.
template <int R, int DIM>
constexpr size_t kPiece = size_t(R) * (DIM + 2);

// Row r of a tile from its pieces: a lane has four columns and, where that leaves lanes, the pieces in turn.  APART: the pieces are dealt to the
// four wavefronts of a block, whose sums meet in LDS; otherwise each wavefront has a row.
template <class T, int DIM, int R, bool APART, class Piece>
__device__ __forceinline__ void join_row(const AttnArgs& a, T* out, const Sequence& s, int tile, int head, int r, int parts, Piece piece) {
    constexpr int QUADS = DIM / 4, EVERY = 64 / QUADS;
    const int lane = threadIdx.x & 63, d = lane % QUADS * 4, mine = lane / QUADS;
    const int group = int(a.group.d);
    if (r >= s.chunk * group - tile * R) return;
    const int wave = APART ? __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6) : 0, step = APART ? 4 : 1;
    const int n = (parts - wave + step - 1) / step;  // of this wavefront's
    // eight pieces of a lane at a time, the first while the maximum is looked for (64 pieces of 16 rows: 6.1 us, four and after it 8.6)
    constexpr int DEEP = 8;
    f32x4 y[DEEP];
    float m[DEEP], l[DEEP];
    auto request = [&](int i0) {
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            if (u == DEEP / 2 && i0 + u * EVERY >= n) break;
            const float* p = piece(min(wave + step * (i0 + u * EVERY + mine), parts - 1));
            y[u] = *reinterpret_cast<const f32x4*>(p + r * DIM + d);
            m[u] = p[R * DIM + r], l[u] = p[R * DIM + R + r];
        }
    };
    request(0);
    float top = -__builtin_inff();
    for (int i = lane; i < parts; i += 64) top = fmaxf(top, piece(i)[R * DIM + r]);
    top = wave_max(top);
    const float mm = top == -__builtin_inff() ? 0.f : top;
    float total = 0.f;
    f32x4 v = {0, 0, 0, 0};
    for (int i0 = 0;;) {
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            if (i0 + u * EVERY + mine >= n) continue;
            const float f = __builtin_amdgcn_exp2f(0.5f * (m[u] - mm));  // (its square may be too small where l is large)
            total += l[u] * f * f, v += y[u] * f * f;
        }
        i0 += DEEP * EVERY;
        if (i0 >= n) break;
        request(i0);
    }
#pragma unroll
    for (int e = QUADS; e < 64; e *= 2) {
        total += __shfl_xor(total, e, 64);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += __shfl_xor(v[k], e, 64);
    }
    if constexpr (APART) {
        __shared__ f32x4 sums[3][QUADS];
        __shared__ float totals[3];
        if (wave && !mine) sums[wave - 1][d / 4] = v;
        if (wave && lane == 0) totals[wave - 1] = total;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 0; w < 3; ++w) total += totals[w], v += sums[w][d / 4];
    }
    if (d >= a.dim || mine) return;
    v *= total == 0.f ? 0.f : 1.f / total;
    const int row = tile * R + r, token = int(a.group(unsigned(row)));
    T* dst = out + (size_t(s.q0 + token) * a.heads + size_t(head * group + row - token * group)) * a.dim + d;
    if constexpr (std::is_same_v<T, float>) *reinterpret_cast<f32x4*>(dst) = v;
    else *reinterpret_cast<uint2*>(dst) = uint2{as_u32(to_h2(v[0], v[1])), as_u32(to_h2(v[2], v[3]))};
}

// Zeros for the rows of q that belong to no sequence, those before row `first` and from row `end`, dealt to the blocks.
template <class T>
__device__ __forceinline__ void clear_other_rows(const AttnArgs& a, T* out, int first, int end, unsigned block, unsigned blocks) {
    const int before = max(0, min(first, a.tokens)), after = max(before, min(end, a.tokens));
    const int rows = before + a.tokens - after;
    const size_t width = size_t(a.heads) * a.dim * sizeof(T) / 16;
    for (unsigned i = block; i < unsigned(rows); i += blocks) {
        uint4* to = reinterpret_cast<uint4*>(out) + size_t(int(i) < before ? int(i) : after + int(i) - before) * width;
        for (size_t e = threadIdx.x; e < width; e += blockDim.x) to[e] = uint4{0, 0, 0, 0};
    }
}

// ---- codes to float16: 1024 + u is the float16 0x6400 | u for u < 1024
// 0x64006400 in a vector register: beside a mask in a scalar one it makes "and, or" one instruction
__device__ __forceinline__ uint32_t magic() {
    uint32_t m = 0x64006400u;
    asm volatile("" : "+v"(m));
    return m;
}

// What turns 1024 + u (and 64 + u) into c - z: c = u + qmin.
template <int BITS>
struct Offsets {
    h2 of1024, of64;
    __device__ __forceinline__ Offsets() : of1024(h2{base, base}), of64(h2{base + 960, base + 960}) {}
    __device__ __forceinline__ Offsets(float za, float zb) {
        of1024 = to_h2(float(base) - za, float(base) - zb), of64 = of1024 + h2{960, 960};
    }
    static constexpr _Float16 base = -1024 - (1 << (BITS - 1));
};
// both halves' low bits: 4-bit codes at bits 0 and 16, or at 4 and 20
__device__ __forceinline__ h2 nibbles0(uint32_t w, uint32_t magic, h2 of1024) { return as_h2((w & 0x000f000fu) | magic) + of1024; }
__device__ __forceinline__ h2 nibbles4(uint32_t w, uint32_t magic, h2 of64) {
    const _Float16 s = _Float16(0.0625f);
    return __builtin_elementwise_fma(as_h2((w & 0x00f000f0u) | magic), h2{s, s}, of64);
}
// bytes 0 and 1, or 2 and 3
__device__ __forceinline__ h2 bytes01(uint32_t w, h2 of1024) {
    return as_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + of1024;
}
__device__ __forceinline__ h2 bytes23(uint32_t w, h2 of1024) {
    return as_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + of1024;
}

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// `bytes` of the cache as a buffer: the address stays in scalar registers, and what lies behind is not read
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00027000);
}

union Frag {
    h2 p[4];
    h8 v;
};

// Keys of a unit of attn_rows_kernel: 16 * NT for each of four wavefronts.  Where a row of codes is short, a wavefront takes 64 keys at a time
// and not 32, with as many registers for them.
constexpr int rows_keys(int bits, int dim, int qt) { return bits * dim <= 512 && qt == 1 ? 64 : 32; }

// One token, or a few, of each sequence: tiles of 16 * qt rows.  `tiles`: a bound for those of all sequences; join: segments may be in pieces.
template <class T, int BITS>
void launch_rows_of(const AttnArgs& a, const T* q, T* out, int tiles, int qt, bool join, hipStream_t st);

// A chunk of a sequence: tiles of 128 rows, or 256 (wide).
template <class T, int BITS>
int launch_chunk_of(const AttnArgs& a, const T* q, T* out, bool wide, int tiles, bool join, hipStream_t st);

}  // namespace attn
}  // namespace lq
