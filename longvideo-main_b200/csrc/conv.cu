// conv.cu -- the short causal convolution of each channel with SiLU: sequences, their gradients and single tokens (sm_100a).
//
// With W taps a channel and x_t for t < 0 from the state (or 0),
//   p_t = bias + sum_{w<W} weight[w] x_{t-W+1+w},   y_t = silu(p_t)  (or p_t);
// the state behind a row is its last W - 1 inputs, oldest first.  Gradients: dp = dy silu'(p),
//   dx_t = sum_w weight[w] dp_{t+W-1-w},   dweight[w] = sum_t dp_t x_{t-W+1+w},   dbias = sum_t dp_t,
// and what the final state's gradient adds to the last W - 1 inputs.
//
// Bound by memory both ways: each value is read once (but for the W - 1 tokens in front of a run) and written once.  A
// thread takes VEC channels of a run of tokens; the W inputs that a token sees move through its registers.  Runs are as
// long as leaves every multiprocessor full of threads once, so that the tokens read twice are few and no round of CTAs
// runs half empty.  The backward takes p again from x (the forward saves nothing) and keeps dweight and dbias of its run in
// registers; the runs of a CTA are added in shared memory, and a second kernel adds the CTAs' partial rows in order (no
// atomics: the same inputs give the same bits).
#include <algorithm>

#include "eacs_common.cuh"
#include "eacs_host.h"
#include "row_common.cuh"

namespace eacs {
namespace {

constexpr int kConvMaxWidth = 4;

struct ConvArgs {
    const void* x;
    const void* weight;
    const void* bias;  // or null
    const void* h0;    // (rows, W - 1, D) or null
    const int32_t* lengths;
    void* y;
    void* hN;  // or null; in a step the state itself
    const void* dy;
    const void* dhN;  // or null
    void* dx;
    void* dh0;    // or null
    float* part;  // (CTAs of a column, D W + D) or null
    int64_t sx[2], sdy[2];
    int64_t rows, L;
    int D, w_dtype, silu;
    int64_t run;  // tokens a run
    int runs;     // runs a row
};

__device__ __forceinline__ int64_t conv_length(const ConvArgs& a, int64_t b) {
    if (!a.lengths) return a.L;
    const int64_t n = a.lengths[b];
    return n < 0 ? 0 : (n > a.L ? a.L : n);
}

// sigmoid(v) = 1 / (1 + e^-v)
__device__ __forceinline__ float conv_sigmoid(float v) { return __fdividef(1.0f, 1.0f + ex2_approx(v * -1.44269504f)); }

template <typename T, int VEC>
__device__ __forceinline__ void conv_read(float* v, const T* p) {
    const RowVec<T, VEC> r = *reinterpret_cast<const RowVec<T, VEC>*>(p);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = to_f32(r.e[e]);
}
template <typename T, int VEC>
__device__ __forceinline__ void conv_write(T* p, const float* v) {
    RowVec<T, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.e[e] = from_f32<T>(v[e]);
    *reinterpret_cast<RowVec<T, VEC>*>(p) = r;
}

// One thread's channels: taps, and the inputs in front of token t0.
template <typename T, int VEC, int W>
struct ConvCols {
    float w[W][VEC], bias[VEC];
    __device__ __forceinline__ void taps(const ConvArgs& a, int c) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][e] = read_param(a.weight, a.w_dtype, (c + e) * W + k, 0.f);
            bias[e] = read_param(a.bias, a.w_dtype, c + e, 0.f);
        }
    }
    // input number t of row b (t >= -(W - 1)): the row's, or the state's
    static __device__ __forceinline__ void input(float* v, const ConvArgs& a, const T* x, int64_t b, int64_t t, int c) {
        if (t >= 0) {
            conv_read<T, VEC>(v, x + t * a.sx[1]);
        } else if (a.h0) {
            conv_read<T, VEC>(v, static_cast<const T*>(a.h0) + (b * (W - 1) + t + W - 1) * a.D + c);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = 0.f;
        }
    }
    __device__ __forceinline__ void dot(float* p, const float (&win)[W][VEC]) const {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            p[e] = bias[e];
#pragma unroll
            for (int k = 0; k < W; ++k) p[e] = fmaf(w[k][e], win[k][e], p[e]);
        }
    }
};

// U tokens are read before the first is used, so that many bytes are under way.  Vectors of 4 values: with 16 bytes of a
// 16-bit type a thread's taps and window leave registers for a third of the threads (79 us instead of what stands at
// conv_fwd_launch).
template <typename T, int VEC, int W, int U>
__global__ void __launch_bounds__(128) conv_fwd_k(const ConvArgs a) {
    const int nv = a.D / VEC;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
    const int64_t r = i / nv;
    if (r >= a.rows * a.runs) return;
    const int c = static_cast<int>(i - r * nv) * VEC;
    const int64_t b = r / a.runs, len = conv_length(a, b);
    const int64_t t0 = (r - b * a.runs) * a.run, t1 = min(t0 + a.run, a.L), tl = min(t1, len);
    const T* x = static_cast<const T*>(a.x) + b * a.sx[0] + c;
    T* y = static_cast<T*>(a.y) + b * a.L * a.D + c;
    using Cols = ConvCols<T, VEC, W>;
    Cols cols;
    cols.taps(a, c);
    float win[W][VEC];  // the inputs a token sees, its own last
    if (t0 < tl)
#pragma unroll
        for (int k = 1; k < W; ++k) Cols::input(win[k], a, x, b, t0 - W + k, c);
    const T* px = x + t0 * a.sx[1];
    T* py = y + t0 * a.D;
    auto token = [&](const RowVec<T, VEC>& v) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k) win[k][e] = win[k + 1][e];
            win[W - 1][e] = to_f32(v.e[e]);
        }
        float p[VEC];
        cols.dot(p, win);
        if (a.silu)
#pragma unroll
            for (int e = 0; e < VEC; ++e) p[e] *= conv_sigmoid(p[e]);
        conv_write<T, VEC>(py, p);
        py += a.D;
    };
    int64_t t = t0;
    for (; t + U <= tl; t += U) {
        RowVec<T, VEC> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = *reinterpret_cast<const RowVec<T, VEC>*>(px + u * a.sx[1]);
        px += U * a.sx[1];
#pragma unroll
        for (int u = 0; u < U; ++u) token(raw[u]);
    }
    for (; t < tl; ++t, px += a.sx[1]) token(*reinterpret_cast<const RowVec<T, VEC>*>(px));
    const float nil[VEC] = {};
    for (t = max(t0, tl); t < t1; ++t) conv_write<T, VEC>(y + t * a.D, nil);
    if (a.hN && t0 == 0) {
        float v[VEC];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            Cols::input(v, a, x, b, len - (W - 1) + k, c);
            conv_write<T, VEC>(static_cast<T*>(a.hN) + (b * (W - 1) + k) * a.D + c, v);
        }
    }
}

// CTAs of 32 columns (VEC channels each) times R runs.  A token gives dp; the gradient of the input W - 1 tokens before it
// is then whole.
template <typename T, int VEC, int W, int R, int U>
__global__ void __launch_bounds__(32 * R) conv_bwd_k(const ConvArgs a) {
    __shared__ float comb[R][32];
    const int nv = a.D / VEC, col = blockIdx.x * 32 + threadIdx.x;
    const int64_t r = static_cast<int64_t>(blockIdx.y) * R + threadIdx.y;
    const bool live = col < nv && r < a.rows * a.runs;
    const int c = col * VEC;
    float dw[W][VEC] = {}, db[VEC] = {};
    if (live) {
        const int64_t b = r / a.runs, len = conv_length(a, b);
        const int64_t t0 = (r - b * a.runs) * a.run, t1 = min(t0 + a.run, a.L), tl = min(t1, len);
        const T* x = static_cast<const T*>(a.x) + b * a.sx[0] + c;
        const T* dy = static_cast<const T*>(a.dy) + b * a.sdy[0] + c;
        T* dx = static_cast<T*>(a.dx) + b * a.L * a.D + c;
        const T* dhN = static_cast<const T*>(a.dhN);
        using Cols = ConvCols<T, VEC, W>;
        using V = RowVec<T, VEC>;
        Cols cols;
        cols.taps(a, c);
        float win[W][VEC], dp[W][VEC] = {};  // dp of the token and of the W - 1 before it
        if (t0 < tl)
#pragma unroll
            for (int k = 1; k < W; ++k) Cols::input(win[k], a, x, b, t0 - W + k, c);
        auto shift = [&] {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) dp[k][e] = dp[k + 1][e], win[k][e] = win[k + 1][e];
        };
        auto token = [&](const V& vx, const V& vg, bool mine) {  // mine: one of the run's own
#pragma unroll
            for (int e = 0; e < VEC; ++e) win[W - 1][e] = to_f32(vx.e[e]);
            float p[VEC];
            cols.dot(p, win);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float g = to_f32(vg.e[e]);
                if (a.silu) {
                    const float s = conv_sigmoid(p[e]);
                    g *= s * fmaf(p[e], 1.f - s, 1.f);
                }
                dp[W - 1][e] = g;
            }
            if (mine)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    db[e] += dp[W - 1][e];
#pragma unroll
                    for (int k = 0; k < W; ++k) dw[k][e] = fmaf(dp[W - 1][e], win[k][e], dw[k][e]);
                }
        };
        auto gradient = [&](float* g) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                g[e] = cols.w[0][e] * dp[W - 1][e];
#pragma unroll
                for (int k = 1; k < W; ++k) g[e] = fmaf(cols.w[k][e], dp[W - 1 - k][e], g[e]);
            }
        };
        // the inputs of a row's first run reach back to the state
        const int64_t first = t0 == 0 ? -(W - 1) : t0;
        const int64_t stop = t0 < len || t0 == 0 ? tl + W - 1 : t0;
        auto any = [&](int64_t tt) {  // a token near either end of the run
            const int64_t o = tt - (W - 1);
            shift();
            if (tt < len) {
                token(*reinterpret_cast<const V*>(x + tt * a.sx[1]), *reinterpret_cast<const V*>(dy + tt * a.sdy[1]), tt < tl);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) dp[W - 1][e] = 0.f;
            }
            if (o < first || o >= len) return;
            float g[VEC];
            gradient(g);
            const int64_t f = o - (len - (W - 1));  // its place in the final state
            if (dhN && f >= 0) {
                float v[VEC];
                conv_read<T, VEC>(v, dhN + (b * (W - 1) + f) * a.D + c);
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] += v[e];
            }
            if (o >= 0) conv_write<T, VEC>(dx + o * a.D, g);
            else if (a.dh0) conv_write<T, VEC>(static_cast<T*>(a.dh0) + (b * (W - 1) + o + W - 1) * a.D + c, g);
        };
        int64_t t = t0;
        for (; t < min(t0 + W - 1, stop); ++t) any(t);
        // between them every token is the run's own and completes an input of the run; none of those is in the final state
        const T *px = x + t * a.sx[1], *pg = dy + t * a.sdy[1];
        T* pd = dx + (t - (W - 1)) * a.D;
        for (; t + U <= tl; t += U) {
            V rx[U], rg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = *reinterpret_cast<const V*>(px + u * a.sx[1]);
                rg[u] = *reinterpret_cast<const V*>(pg + u * a.sdy[1]);
            }
            px += U * a.sx[1];
            pg += U * a.sdy[1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                shift();
                token(rx[u], rg[u], true);
                float g[VEC];
                gradient(g);
                conv_write<T, VEC>(pd, g);
                pd += a.D;
            }
        }
        for (; t < stop; ++t) any(t);
        const float nil[VEC] = {};
        for (t = max(t0, tl); t < t1; ++t) conv_write<T, VEC>(dx + t * a.D, nil);
    }
    if (!a.part) return;
    float* part = a.part + static_cast<int64_t>(blockIdx.y) * a.D * (W + 1);
#pragma unroll
    for (int k = 0; k <= W; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            __syncthreads();
            comb[threadIdx.y][threadIdx.x] = k < W ? dw[k < W ? k : 0][e] : db[e];
            __syncthreads();
            if (threadIdx.y == 0 && col < nv) {
                float s = comb[0][threadIdx.x];
#pragma unroll
                for (int j = 1; j < R; ++j) s += comb[j][threadIdx.x];
                part[k < W ? (c + e) * W + k : a.D * W + c + e] = s;
            }
        }
}

template <typename T, int VEC, int W>
__global__ void __launch_bounds__(128) conv_step_k(const ConvArgs a) {
    const int nv = a.D / VEC;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
    const int64_t b = i / nv;
    if (b >= a.rows) return;
    const int c = static_cast<int>(i - b * nv) * VEC;
    T* h = static_cast<T*>(a.hN) + b * (W - 1) * a.D + c;
    RowVec<T, VEC> raw[W];  // the state is moved as it is
#pragma unroll
    for (int k = 0; k < W - 1; ++k) raw[k] = *reinterpret_cast<const RowVec<T, VEC>*>(h + static_cast<int64_t>(k) * a.D);
    raw[W - 1] = *reinterpret_cast<const RowVec<T, VEC>*>(static_cast<const T*>(a.x) + b * a.sx[0] + c);
    ConvCols<T, VEC, W> cols;
    cols.taps(a, c);
    float win[W][VEC], p[VEC];
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) win[k][e] = to_f32(raw[k].e[e]);
    cols.dot(p, win);
    if (a.silu)
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[e] *= conv_sigmoid(p[e]);
    conv_write<T, VEC>(static_cast<T*>(a.y) + b * a.D + c, p);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) *reinterpret_cast<RowVec<T, VEC>*>(h + static_cast<int64_t>(k) * a.D) = raw[k + 1];
}

// ---------------------------------------------------------------------------------------------------------
constexpr int kConvBwdRuns = 4;  // runs a CTA of the backward

// Runs that fill `threads` threads a multiprocessor once with `cols` columns a run; none shorter than 8 tokens.
void conv_runs(ConvArgs& a, int64_t cols, int threads) {
    const int64_t want = std::max<int64_t>(1, int64_t{148} * threads / (cols * std::max<int64_t>(a.rows, 1)));
    a.run = std::max<int64_t>(8, (a.L + want - 1) / want);
    a.runs = static_cast<int>(std::max<int64_t>(1, (a.L + a.run - 1) / a.run));
}
int64_t conv_bwd_cols(int64_t D, int vec) { return ((D + vec - 1) / vec + 31) / 32 * 32; }
int conv_bwd_vec(bool vec) { return vec ? 4 : 1; }
int64_t conv_bwd_rows(const ConvArgs& a) { return (a.rows * a.runs + kConvBwdRuns - 1) / kConvBwdRuns; }

template <typename T, int VEC, int W>
cudaError_t conv_fwd_launch(ConvArgs& a, cudaStream_t s) {
    constexpr int U = VEC > 1 ? 8 : 16;
    static const int per = row_resident(conv_fwd_k<T, VEC, W, U>, 128, 0);
    const int64_t nv = a.D / VEC;
    conv_runs(a, nv, per * 128);
    const int64_t n = a.rows * a.runs * nv;
    conv_fwd_k<T, VEC, W, U><<<static_cast<unsigned>((n + 127) / 128), 128, 0, s>>>(a);
    note_launch();
    return cudaGetLastError();
}
template <typename T, int VEC, int W>
cudaError_t conv_bwd_launch(ConvArgs& a, void* dweight, void* dbias, cudaStream_t s) {
    constexpr int R = kConvBwdRuns;
    const int64_t nv = a.D / VEC, rows = conv_bwd_rows(a);
    conv_bwd_k<T, VEC, W, R, 4><<<dim3(static_cast<unsigned>((nv + 31) / 32), static_cast<unsigned>(rows)), dim3(32, R), 0, s>>>(a);
    note_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || !a.part) return e;
    RowSums r{};
    r.part = a.part, r.rows = static_cast<int>(rows), r.stride = static_cast<int64_t>(a.D) * (W + 1), r.dtype = a.w_dtype;
    r.out[0] = dweight, r.out[1] = dbias, r.n[0] = a.D * W, r.n[1] = a.D, r.at[1] = static_cast<int64_t>(a.D) * W;
    return row_sums(r, 2, s);
}
template <typename T, int VEC, int W>
cudaError_t conv_step_launch(ConvArgs& a, cudaStream_t s) {
    const int64_t n = a.rows * (a.D / VEC);
    conv_step_k<T, VEC, W><<<static_cast<unsigned>((n + 127) / 128), 128, 0, s>>>(a);
    note_launch();
    return cudaGetLastError();
}

#define EACS_CONV_W(T, VEC, F, ...)             \
    (width == 2   ? F<T, VEC, 2>(__VA_ARGS__)   \
     : width == 3 ? F<T, VEC, 3>(__VA_ARGS__)   \
                  : F<T, VEC, 4>(__VA_ARGS__))

template <typename T>
cudaError_t conv_fwd_any(ConvArgs& a, int width, bool vec, cudaStream_t s) {
    return vec ? EACS_CONV_W(T, 4, conv_fwd_launch, a, s) : EACS_CONV_W(T, 1, conv_fwd_launch, a, s);
}
template <typename T>
cudaError_t conv_step_any(ConvArgs& a, int width, bool vec, cudaStream_t s) {
    return vec ? EACS_CONV_W(T, 4, conv_step_launch, a, s) : EACS_CONV_W(T, 1, conv_step_launch, a, s);
}
template <typename T>
cudaError_t conv_bwd_any(ConvArgs& a, int width, bool vec, void* dw, void* db, cudaStream_t s) {
    return vec ? EACS_CONV_W(T, 4, conv_bwd_launch, a, dw, db, s) : EACS_CONV_W(T, 1, conv_bwd_launch, a, dw, db, s);
}

int conv_check(const char* fn, const EacsConv& p, bool single) {
    if (p.rows < 0 || p.L < 0 || p.D < 1) return fail(EACS_ERR_INVALID, "%s: bad sizes", fn);
    for (int dt : {p.dtype, p.w_dtype})
        if (dt != EACS_DTYPE_F32 && dt != EACS_DTYPE_F16 && dt != EACS_DTYPE_BF16)
            return fail(EACS_ERR_INVALID, "%s: unknown dtype %d", fn, dt);
    if (p.width < 2 || p.width > kConvMaxWidth) return fail(EACS_ERR_UNSUPPORTED, "%s: %d taps, not 2 to %d", fn, p.width, kConvMaxWidth);
    if (p.rows > 65535 || p.D > (int64_t{1} << 24) || p.L > (int64_t{1} << 30))
        return fail(EACS_ERR_UNSUPPORTED, "%s: more than 65535 rows, 2^24 channels or 2^30 tokens", fn);
    if (p.rows > 0 && (!p.weight || ((p.L > 0 || single) && !p.x))) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    return EACS_OK;
}
ConvArgs conv_args(const EacsConv& p) {
    ConvArgs a{};
    a.x = p.x, a.weight = p.weight, a.bias = p.bias, a.h0 = p.initial_state, a.lengths = p.lengths;
    a.sx[0] = p.x_stride[0], a.sx[1] = p.x_stride[1];
    a.rows = p.rows, a.L = p.L, a.D = static_cast<int>(p.D), a.w_dtype = p.w_dtype, a.silu = p.silu;
    return a;
}
// Whether vectors of `n` elements may be moved at p and its strides (D of them a row).
bool conv_vec(const EacsConv& p, int n, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
    const uintptr_t bytes = static_cast<uintptr_t>(n) * (p.dtype == EACS_DTYPE_F32 ? 4 : 2);
    if (p.D % n) return false;
    for (const void* q : ptrs)
        if (reinterpret_cast<uintptr_t>(q) % bytes) return false;
    for (int64_t st : strides)
        if (st % n) return false;
    return true;
}

}  // namespace

// The partial rows of a backward, for vectors or single elements, whichever has more.
size_t conv_bwd_workspace_size(const EacsConv& p) {
    if (conv_check("eacs_conv_bwd_workspace_size", p, false) != EACS_OK || p.rows == 0) return 0;
    ConvArgs a = conv_args(p);
    int64_t rows = 0;
    for (int vec : {1, 4}) {
        conv_runs(a, conv_bwd_cols(p.D, vec), 512);
        rows = std::max(rows, conv_bwd_rows(a));
    }
    return static_cast<size_t>(rows) * p.D * (p.width + 1) * sizeof(float);
}

int conv_fwd(const EacsConv& p, void* y, void* final_state, cudaStream_t stream) {
    const char* fn = "eacs_conv_fwd";
    if (const int rc = conv_check(fn, p, false)) return rc;
    if (p.rows == 0) return EACS_OK;
    if (p.L > 0 && !y) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    ConvArgs a = conv_args(p);
    a.y = y;
    a.hN = final_state;
    if (p.L == 0 && !final_state) return EACS_OK;
    const bool vec = conv_vec(p, 4, {p.x, y, p.initial_state, final_state}, {p.x_stride[0], p.x_stride[1]});
    const cudaError_t e = p.dtype == EACS_DTYPE_F32   ? conv_fwd_any<float>(a, p.width, vec, stream)
                          : p.dtype == EACS_DTYPE_F16 ? conv_fwd_any<__half>(a, p.width, vec, stream)
                                                      : conv_fwd_any<__nv_bfloat16>(a, p.width, vec, stream);
    return cuda_check(e, fn);
}

int conv_step(const EacsConv& p, void* y, void* state, cudaStream_t stream) {
    const char* fn = "eacs_conv_step";
    if (const int rc = conv_check(fn, p, true)) return rc;
    if (p.rows == 0) return EACS_OK;
    if (!y || !state) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    ConvArgs a = conv_args(p);
    a.y = y;
    a.hN = state;
    const bool vec = conv_vec(p, 4, {p.x, y, state}, {p.x_stride[0]});
    const cudaError_t e = p.dtype == EACS_DTYPE_F32   ? conv_step_any<float>(a, p.width, vec, stream)
                          : p.dtype == EACS_DTYPE_F16 ? conv_step_any<__half>(a, p.width, vec, stream)
                                                      : conv_step_any<__nv_bfloat16>(a, p.width, vec, stream);
    return cuda_check(e, fn);
}

int conv_bwd(const EacsConv& p, const ConvGrads& g, void* ws, size_t ws_bytes, cudaStream_t stream) {
    const char* fn = "eacs_conv_bwd";
    if (const int rc = conv_check(fn, p, false)) return rc;
    if (p.rows > 0 && p.L > 0 && (!g.dy || !g.dx)) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    const bool want = g.dweight || g.dbias;
    if (p.rows == 0) {  // empty sums
        const size_t e1 = p.w_dtype == EACS_DTYPE_F32 ? 4 : 2;
        cudaError_t e = cudaSuccess;
        if (g.dweight) e = cudaMemsetAsync(g.dweight, 0, e1 * p.D * p.width, stream);
        if (e == cudaSuccess && g.dbias) e = cudaMemsetAsync(g.dbias, 0, e1 * p.D, stream);
        return cuda_check(e, fn);
    }
    if (want && (!ws || ws_bytes < conv_bwd_workspace_size(p)))
        return fail(EACS_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, conv_bwd_workspace_size(p));
    if (reinterpret_cast<uintptr_t>(ws) & 15u) return fail(EACS_ERR_INVALID, "%s: the workspace is not on 16 bytes", fn);
    ConvArgs a = conv_args(p);
    a.dy = g.dy, a.dhN = g.dfinal, a.dx = g.dx, a.dh0 = g.dinitial;
    a.sdy[0] = g.dy_stride[0], a.sdy[1] = g.dy_stride[1];
    a.part = want ? static_cast<float*>(ws) : nullptr;
    const bool vec = conv_vec(p, 4, {p.x, p.initial_state, g.dy, g.dfinal, g.dx, g.dinitial},
                              {p.x_stride[0], p.x_stride[1], g.dy_stride[0], g.dy_stride[1]});
    conv_runs(a, conv_bwd_cols(p.D, conv_bwd_vec(vec)), 512);
    const cudaError_t e = p.dtype == EACS_DTYPE_F32   ? conv_bwd_any<float>(a, p.width, vec, g.dweight, g.dbias, stream)
                          : p.dtype == EACS_DTYPE_F16 ? conv_bwd_any<__half>(a, p.width, vec, g.dweight, g.dbias, stream)
                                                      : conv_bwd_any<__nv_bfloat16>(a, p.width, vec, g.dweight, g.dbias, stream);
    return cuda_check(e, fn);
}

}  // namespace eacs
