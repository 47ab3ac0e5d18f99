// The residual connection between two blocks, with the norms beside it, in one pass:
//
//   t  = post(x), or x            post, pre: rms    v / sqrt(mean(v^2) + eps) * weight (+ bias)
//   r' = r + gate * scale * t                layer  (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) * weight (+ bias)
//   y  = pre(r')
//
// A row stays in the registers of the TPR threads that have it: x and r are read once, r' and y written once, whatever norms are
// asked for; a layer norm's variance is taken about its mean from the registers.  y comes from r' as it is in float32, before that
// is rounded to its own type.  Bound by memory: what passes once leaves the caches to others (12 608 x 768 float32, both layer norms, a gate of
// 64 rows and a scale 36 -> 29 us, 5.3 TB/s; sums over lane patterns 37 -> 36).  Keeping weights and scales in registers from row to row, with the next
// row under way, gains nothing: 37 to 40 us.
#include <type_traits>

#include "common.hpp"

using namespace lq;

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef f4 f4u __attribute__((aligned(4)));  // (rows need not be aligned)
typedef h4 h4u __attribute__((aligned(2)));

struct Norm {
    const float *weight, *bias;  // NULL: ones, zeros
};

struct Args {
    const void *x, *r, *gate;  // r NULL: no residual; gate NULL: ones
    const float* scale;        // [cols], NULL: ones
    Norm pre, post;
    void *y, *r_out;  // r_out NULL: not wanted
    unsigned rows, cols;
    float eps;
    FastDiv per_gate{1};  // rows of a row of the gate
};

// How rows are cut into fours: kWhole, of a multiple of four; kTail, the four that reaches past the end is the last four of the row, moved up; kTiny,
// of fewer than four, value by value.  (kTail by value: 2325 x 1233 float16 36 us, 8350 x 2125 float32 138; so 14 and 62.)
enum Rows { kWhole, kTail, kTiny };

// Four values of a row from column c on, zeros past its end.  No branch: the compiler waits for a load where two paths that give its register a
// value meet.
template <Rows ROWS, bool STREAM = false, class T>
__device__ __forceinline__ f4 load4(const T* row, unsigned c, unsigned cols) {
    f4 v;
    if constexpr (ROWS != kTiny) {
        const unsigned at = ROWS == kWhole ? (c < cols ? c : 0) : c + 4 <= cols ? c : cols - 4;
        const T* const from = row + at;
        if constexpr (std::is_same_v<T, float>) {
            v = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const f4u*>(from)) : *reinterpret_cast<const f4u*>(from);
        } else {
            const h4 h = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const h4u*>(from)) : *reinterpret_cast<const h4u*>(from);
            v = f4{float(h[0]), float(h[1]), float(h[2]), float(h[3])};
        }
        if constexpr (ROWS == kTail) {
            const unsigned by = c - at;
            v = by & 1 ? f4{v[1], v[2], v[3], 0.f} : v;
            v = by & 2 ? f4{v[2], v[3], 0.f, 0.f} : v;
        }
        return c < cols ? v : f4{0.f, 0.f, 0.f, 0.f};
    } else {
#pragma unroll
        for (unsigned i = 0; i < 4; ++i) {
            const float e = float(row[c + i < cols ? c + i : 0]);
            v[i] = c + i < cols ? e : 0.f;
        }
        return v;
    }
}
template <Rows ROWS, class T>
__device__ __forceinline__ void store4(T* row, unsigned c, unsigned cols, f4 v) {
    if (ROWS == kWhole ? c < cols : ROWS == kTail && c + 4 <= cols) {
        if constexpr (std::is_same_v<T, float>) {
            __builtin_nontemporal_store(f4u(v), reinterpret_cast<f4u*>(row + c));
        } else {
            const h4 h{_Float16(v[0]), _Float16(v[1]), _Float16(v[2]), _Float16(v[3])};
            __builtin_nontemporal_store(h4u(h), reinterpret_cast<h4u*>(row + c));
        }
    } else if constexpr (ROWS != kWhole) {
#pragma unroll
        for (unsigned i = 0; i < 4; ++i)
            if (c + i < cols) row[c + i] = T(v[i]);
    }
}

// A lane's neighbour by the vector unit's own patterns, zeros where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float v) {
    return __uint_as_float(unsigned(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(v)), CTRL, ROWS, 0xf, false)));
}
// The sum over the TPR threads of a row, to all of them.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* s) {
    v += moved<0x111, 0xf>(v);  // over rows of 16 lanes: from 1, 2, 4, 8 lanes before
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);  // lane 15 into rows 1 and 3, lane 31 into rows 2 and 3: lane 63 has the sum
    v += moved<0x143, 0xc>(v);
    v = __uint_as_float(unsigned(__builtin_amdgcn_readlane(int(__float_as_uint(v)), 63)));
    if constexpr (TPR > 64) {
        __syncthreads();  // (the sums before have been read)
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = s[threadIdx.x & (TPR / 64 - 1)];
#pragma unroll
        for (int d = TPR / 128; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    }
    return v;
}

template <bool LAYER, Rows ROWS, int TPR, int NV>
__device__ __forceinline__ void normalize(f4 (&v)[NV], const Norm& n, unsigned at, unsigned cols, float eps, float* s) {
    const float inverse = 1.0f / float(cols);
    float sum = 0.f;
    if constexpr (LAYER) {
#pragma unroll
        for (int i = 0; i < NV; ++i) sum += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
        const float mean = row_sum<TPR>(sum, s) * inverse;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = at + i * TPR * 4 + e < cols ? v[i][e] - mean : 0.f;
        sum = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += (v[i][0] * v[i][0] + v[i][1] * v[i][1]) + (v[i][2] * v[i][2] + v[i][3] * v[i][3]);
    const float f = 1.0f / sqrtf(row_sum<TPR>(sum, s) * inverse + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] *= f;
    if (n.weight) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] *= load4<ROWS>(n.weight, at + i * TPR * 4, cols);
    }
    if (n.bias) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] += load4<ROWS>(n.bias, at + i * TPR * 4, cols);
    }
}

template <class TX, class TR, bool LAYER, bool POST, Rows ROWS, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void residual_norm_kernel(Args a) {
    __shared__ float s[TPR / 64];
    const unsigned row = (blockIdx.y * gridDim.x + blockIdx.x) * (TPR < 256 ? 256 / TPR : 1) + threadIdx.x / TPR, at = threadIdx.x % TPR * 4;
    if (row >= a.rows) return;  // (rows of 64 threads: no barrier follows)
    const size_t base = size_t(row) * a.cols;
    f4 x[NV], r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = load4<ROWS, true>(static_cast<const TX*>(a.x) + base, at + i * TPR * 4, a.cols);
    if (a.r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) r[i] = load4<ROWS, true>(static_cast<const TR*>(a.r) + base, at + i * TPR * 4, a.cols);
    }
    if constexpr (POST) normalize<LAYER, ROWS, TPR, NV>(x, a.post, at, a.cols, a.eps, s);
    if (a.scale) {
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] *= load4<ROWS>(a.scale, at + i * TPR * 4, a.cols);
    }
    if (a.gate) {
        const TX* gate = static_cast<const TX*>(a.gate) + size_t(a.per_gate(row)) * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] *= load4<ROWS>(gate, at + i * TPR * 4, a.cols);
    }
    if (a.r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] += r[i];
    }
    if (a.r_out) {
#pragma unroll
        for (int i = 0; i < NV; ++i) store4<ROWS>(static_cast<TR*>(a.r_out) + base, at + i * TPR * 4, a.cols, x[i]);
    }
    normalize<LAYER, ROWS, TPR, NV>(x, a.pre, at, a.cols, a.eps, s);
#pragma unroll
    for (int i = 0; i < NV; ++i) store4<ROWS>(static_cast<TX*>(a.y) + base, at + i * TPR * 4, a.cols, x[i]);
}

template <int V>
using Int = std::integral_constant<int, V>;

// f with how rows are cut, the threads of a row, and the fours of values that each has: a wavefront or four of them, so that few lanes wait at the
// sums (2^24 float32, both layer norms, rows of 6336: 256 threads 51.2 us, 1024 55.0; of 4556 53.9 and 62.7; of 2912, three fours for four 49.7 and 51.9).
template <class F>
void by_shape(unsigned cols, F&& f) {
    const unsigned fours = (cols + 3) / 4;
    if (cols < 4) return f(Int<kTiny>{}, Int<64>{}, Int<1>{});
    auto of_rows = [&](auto rows) {
        if (fours <= 64) f(rows, Int<64>{}, Int<1>{});
        else if (fours <= 128) f(rows, Int<64>{}, Int<2>{});
        else if (fours <= 192) f(rows, Int<64>{}, Int<3>{});
        else if (fours <= 256) f(rows, Int<64>{}, Int<4>{});
        else if (fours <= 512) f(rows, Int<256>{}, Int<2>{});
        else if (fours <= 768) f(rows, Int<256>{}, Int<3>{});
        else if (fours <= 1024) f(rows, Int<256>{}, Int<4>{});
        else if (fours <= 1536) f(rows, Int<256>{}, Int<6>{});
        else if (fours <= 2048) f(rows, Int<256>{}, Int<8>{});
        else if (fours <= 4096) f(rows, Int<1024>{}, Int<4>{});
        else f(rows, Int<1024>{}, Int<8>{});
    };
    if (cols % 4) of_rows(Int<kTail>{});
    else of_rows(Int<kWhole>{});
}

template <class TX, class TR, bool LAYER>
void launch(const Args& a, bool post, hipStream_t st) {
    by_shape(a.cols, [&](auto rows, auto tpr, auto nv) {
        constexpr Rows ROWS = Rows(decltype(rows)::value);
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, BLOCK = TPR < 256 ? 256 : TPR;
        // (2^32 threads and more are several rows of blocks: a launch has fewer along its first axis)
        const unsigned per = BLOCK / TPR, blocks = (a.rows + per - 1) / per, across = blocks < 1u << 21 ? blocks : 1u << 21;
        const auto kernel = post ? residual_norm_kernel<TX, TR, LAYER, true, ROWS, TPR, NV> : residual_norm_kernel<TX, TR, LAYER, false, ROWS, TPR, NV>;
        kernel<<<dim3(across, (blocks + across - 1) / across), BLOCK, 0, st>>>(a);
    });
}

constexpr int kMaxCols = 32768;  // 1024 threads with 32 values each

}  // namespace

extern "C" int lq_residual_norm(const lq_residual_norm_args* n, lq_stream stream) {
    LQ_REQUIRE(n, LQ_ERR_VALUE, "residual_norm: args is NULL");
    LQ_REQUIRE(n->rows >= 0 && n->cols >= 0, LQ_ERR_SHAPE, "residual_norm: %lld rows of %d", (long long)n->rows, n->cols);
    LQ_REQUIRE(n->layer == 0 || n->layer == 1, LQ_ERR_VALUE, "residual_norm: norm %d; 0 is rms, 1 is layer", n->layer);
    LQ_REQUIRE((n->x_dtype == LQ_F32 || n->x_dtype == LQ_F16) && (n->r_dtype == LQ_F32 || n->r_dtype == n->x_dtype), LQ_ERR_DTYPE,
               "residual_norm: x is float32 or float16, the residual float32 or of its type");
    LQ_REQUIRE(n->gate_rows >= 0 && (n->gate ? n->gate_rows > 0 : n->gate_rows == 0), LQ_ERR_VALUE, "residual_norm: a gate of %lld rows",
               (long long)n->gate_rows);
    if (n->rows == 0 || n->cols == 0) return LQ_OK;
    LQ_REQUIRE(n->x && n->y, LQ_ERR_VALUE, "residual_norm: x or y is NULL");
    LQ_REQUIRE(n->gate_rows == 0 || n->rows % n->gate_rows == 0, LQ_ERR_SHAPE, "residual_norm: a gate of %lld rows for %lld", (long long)n->gate_rows,
               (long long)n->rows);
    LQ_REQUIRE(n->cols <= kMaxCols, LQ_ERR_NOT_IMPLEMENTED, "residual_norm: rows of %d; at most %d are built", n->cols, kMaxCols);
    LQ_REQUIRE(n->rows < int64_t(1) << 31, LQ_ERR_SHAPE, "residual_norm: %lld rows", (long long)n->rows);
    // a row's value is read by the lane that puts a result there, before it does, so a result may lie in such an operand's place, and nowhere else on what is
    // read: every row reads the vectors, and those of the second norm after r' is written
    const size_t values = size_t(n->rows) * n->cols, x_item = n->x_dtype == LQ_F16 ? 2 : 4, r_item = n->r_dtype == LQ_F16 ? 2 : 4;
    const Span x{n->x, values * x_item}, r{n->r, values * r_item}, gate{n->gate, size_t(n->gate_rows) * n->cols * x_item}, y{n->y, values * x_item},
        r_out{n->r_out, values * r_item};
    bool sound = apart(y, r_out);
    for (const Span& to : {y, r_out}) {
        for (const Span& from : {x, r, gate}) sound = sound && (apart(to, from) || (to.at == from.at && to.bytes == from.bytes));
        for (const float* v : {n->scale, n->weight, n->bias, n->post_weight, n->post_bias}) sound = sound && apart(to, Span{v, size_t(n->cols) * sizeof(float)});
    }
    LQ_REQUIRE(sound, LQ_ERR_VALUE, "residual_norm: a result lies on what is read, but not in its place, or on the other result");
    Args a;
    a.x = n->x, a.r = n->r, a.gate = n->gate, a.scale = n->scale;
    a.pre = Norm{n->weight, n->bias}, a.post = Norm{n->post_weight, n->post_bias};
    a.y = n->y, a.r_out = n->r_out, a.rows = unsigned(n->rows), a.cols = unsigned(n->cols), a.eps = n->eps;
    if (n->gate) a.per_gate = FastDiv(unsigned(n->rows / n->gate_rows));
    const hipStream_t st = as_stream(stream);
    const bool post = n->post != 0;
    auto of_norm = [&](auto tx, auto tr) {
        using TX = decltype(tx);
        using TR = decltype(tr);
        if (n->layer) launch<TX, TR, true>(a, post, st);
        else launch<TX, TR, false>(a, post, st);
    };
    if (n->x_dtype == LQ_F32) of_norm(float{}, float{});
    else if (n->r_dtype == LQ_F32) of_norm(_Float16{}, float{});
    else of_norm(_Float16{}, _Float16{});
    LQ_CHECK_LAUNCH("residual_norm");
    return LQ_OK;
}
