// Attention of new tokens over the pages of a quantized key / value cache (lq_paged_attention): what its kernels share.
//
// Query rows of one sequence that read the same key / value head are the rows token * group + (head within the group),
// group = heads / kv_heads: whatever the group, one row of the matrix products each.  A row at place p = kv_len - chunk + token
// sees the keys [max(0, p - window + 1), min(kv_len, p + 1)).
//
// The mathematics.  Codes are whole numbers below 2^8, which float16 holds exactly, so that the matrix instruction gets them as they
// are and the scales follow in float32:
//     S_j = (scale log2 e) k_scale_j sum_d q_d (c_jd - z_j)
//     o_d = sum_j (2^(S_j - m) v_scale_j) (c'_jd - z'_j) / sum_j 2^(S_j - m)
// A product of a float16 and a code is exact in float32, and so is c - z.  float16 queries enter as they are, float32 ones as two float16
// of 22 bits together (times a power of two for each row, so that neither part is subnormal where it counts).  Probabilities
// times v_scale are rounded to one float16 for a float16 result (half a step, 2^-11, as the result's own rounding), to two for a
// float32 one; their sum is not rounded.  What makes that work whatever the scales is a power of two, `unit`, above the largest v_scale so
// far: 2^7 v_scale / unit times a probability of at most 2^8 fits float16, and outputs are kept in units of unit / 2^7.
#pragma once
#include "kv_cache.hpp"

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
    int items;     // blocks there are for the items of a head
    int target;    // blocks that the keys of a launch are shared out to
    int max_rows;  // sequences of more rows are another launch's
    float scale;
    float* partial;  // results of items that share a tile
};

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace attn {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLazy = 8.f;        // a row's maximum is renewed when it has grown by this (powers of two)
constexpr float kProbability = 0x1p7f;  // probabilities are kept times this
constexpr int kMinKeys = 128;       // of an item's share of keys: a step of 32 for each of four wavefronts

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

// What the blocks of a launch do is found by each of them from the lengths, which only the device knows: tiles of R rows, the
// keys of a sequence's tiles shared out to `chunks` items each, so that all items of a launch are about equally long.
struct Item {
    int seq, tile, part, parts;  // part of its parts
    int first;                   // number of the tile's first item
    Sequence s;
};

// the sums over the lanes before this one and itself
__device__ __forceinline__ unsigned scan(unsigned v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// Item number `id` of a launch with tiles of R rows (tiles instead of items with `whole`: id counts tiles).  False: there is none.
// Every wavefront finds it for itself, 64 sequences at a time.
template <int R>
__device__ __forceinline__ bool find_item(const AttnArgs& a, unsigned id, bool whole, Item& item) {
    const int lane = threadIdx.x & 63;
    auto tiles_of = [&](const Sequence& s) {
        const int rows = s.chunk * int(a.group.d);
        return rows > a.max_rows ? 0u : unsigned(rows + R - 1) / R;
    };
    auto extent_of = [&](const Sequence& s) {
        const Keys k = keys_of(a, s, 0, s.chunk - 1);
        return unsigned(k.hi - (k.lo & ~31));
    };
    unsigned long long sum = 0;
    for (int b = lane; b < a.batch; b += 64) {
        const Sequence s = sequence_of(a, b);
        sum += (unsigned long long)(tiles_of(s)) * extent_of(s);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
    const unsigned long long share = (sum * unsigned(a.kv_heads) + a.target - 1) / unsigned(a.target);
    const unsigned long long keys = (share + kMinKeys - 1) / kMinKeys * kMinKeys;
    const unsigned each = keys < kMinKeys ? kMinKeys : keys > 0x40000000ull ? 0x40000000u : unsigned(keys);
    unsigned items = 0, tiles = 0;  // of the sequences before these
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = b0 + lane;
        Sequence s{0, 0, 0};
        unsigned t = 0, parts = 1;
        if (b < a.batch) {
            s = sequence_of(a, b);
            t = tiles_of(s);
            parts = max(1u, (extent_of(s) + each - 1) / each);
        }
        const unsigned items_to = items + scan(t * parts, lane), tiles_to = tiles + scan(t, lane);
        const unsigned long long past = __ballot((whole ? tiles_to : items_to) > id);
        if (past) {
            const int at = __builtin_ctzll(past);
            auto get = [&](unsigned v) { return __builtin_amdgcn_readlane(int(v), at); };
            item.seq = b0 + at, item.parts = get(parts);
            item.s = Sequence{get(s.q0), get(s.chunk), get(s.len)};
            const int n = get(t), first = get(items_to) - n * item.parts;
            const int k = int(id) - (whole ? get(tiles_to) - n : first);
            item.tile = whole ? k : k / item.parts;
            item.part = whole ? 0 : k - item.tile * item.parts;
            item.first = first + item.tile * item.parts;
            return true;
        }
        items = __builtin_amdgcn_readlane(int(items_to), 63), tiles = __builtin_amdgcn_readlane(int(tiles_to), 63);
    }
    return false;
}

// Partial results of an item and head: R rows of `stride` floats, each the sums over its keys, then the rows' maximum and sum of
// probabilities.
__device__ __forceinline__ size_t partial_at(const AttnArgs& a, int item, int head, int rows, int stride) {
    return (size_t(item) * a.kv_heads + head) * rows * (stride + 2);
}

// Zeros for the rows of q that belong to no sequence, dealt to the blocks.
template <class T>
__device__ __forceinline__ void clear_other_rows(const AttnArgs& a, T* out, unsigned block, unsigned blocks) {
    const int before = max(0, min(a.q_starts[0], a.tokens)), after = max(before, min(a.q_starts[a.batch], a.tokens));
    const int rows = before + a.tokens - after;
    const size_t width = size_t(a.heads) * a.dim * sizeof(T) / 16;
    for (unsigned i = block; i < unsigned(rows); i += blocks) {
        uint4* to = reinterpret_cast<uint4*>(out) + size_t(int(i) < before ? int(i) : after + int(i) - before) * width;
        for (size_t e = threadIdx.x; e < width; e += blockDim.x) to[e] = uint4{0, 0, 0, 0};
    }
}

// ---- codes to float16: 1024 + u is the float16 0x6400 | u for u < 1024
constexpr uint32_t kMagic = 0x64006400u;
__device__ __forceinline__ h2 as_h2(uint32_t v) { return __builtin_bit_cast(h2, v); }
__device__ __forceinline__ uint32_t as_u32(h2 v) { return __builtin_bit_cast(uint32_t, v); }

// What turns 1024 + u (and 64 + u) into c - z: c = u + qmin.
template <int BITS>
struct Offsets {
    h2 of1024, of64;
    __device__ __forceinline__ Offsets() { set(0.f, 0.f); }
    __device__ __forceinline__ void set(float za, float zb) {
        constexpr float half = float(1 << (BITS - 1));
        of1024 = to_h2(-1024.f - half - za, -1024.f - half - zb);
        of64 = to_h2(-64.f - half - za, -64.f - half - zb);
    }
};
// both halves' low bits: 4-bit codes at bits 0 and 16, or at 4 and 20
__device__ __forceinline__ h2 nibbles0(uint32_t w, h2 of1024) { return as_h2((w & 0x000f000fu) | kMagic) + of1024; }
__device__ __forceinline__ h2 nibbles4(uint32_t w, h2 of64) {
    const _Float16 s = _Float16(0.0625f);
    return __builtin_elementwise_fma(as_h2((w & 0x00f000f0u) | kMagic), h2{s, s}, of64);
}
// bytes 0 and 1, or 2 and 3
__device__ __forceinline__ h2 bytes01(uint32_t w, h2 of1024) {
    return as_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + of1024;
}
__device__ __forceinline__ h2 bytes23(uint32_t w, h2 of1024) {
    return as_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + of1024;
}

union Frag {
    h2 p[4];
    h8 v;
};

template <class T, int BITS>
void launch_rows_of(const AttnArgs& a, const T* q, T* out, int tiles, int qt, bool join, hipStream_t st);

}  // namespace attn
}  // namespace lq
