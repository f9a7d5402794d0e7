// conv.cu -- the short causal convolution of each channel with SiLU: sequences, their gradients and single tokens (sm_100a).
//
// With W taps a channel and x_t for t < 0 from the state (or 0),
//   p_t = bias + sum_{w<W} weight[w] x_{t-W+1+w},   y_t = silu(p_t)  (or p_t);
// the state behind a row is its last W - 1 inputs, oldest first.  Gradients: dp = dy silu'(p),
//   dx_t = sum_w weight[w] dp_{t+W-1-w},   dweight[w] = sum_t dp_t x_{t-W+1+w},   dbias = sum_t dp_t,
// and what the final state's gradient adds to the last W - 1 inputs.
//
// Each value is read once (but for the W - 1 tokens around a run) and written once.  A warp takes 64 channels, two a
// lane, of a run of tokens; rows of 128 (float32: 256) bytes come through shared memory, asked for three stages of 8
// tokens ahead (cp.async, its own, so without a barrier between warps), and the W inputs that a token sees move
// through the lanes' registers as pairs.  A CTA's four warps lie side by side.  Through registers the same loads left
// too few threads: the forward took 67 us at B=4 L=16384 D=1024 bfloat16 and takes 55 (41 for its bytes), the
// backward at B=8 L=8192 D=768 127 and 75 (46).  What is left is latency and issue: 17 instructions of a warp for 32
// values forward, 28 backward, two of them special functions, at 61 and 57 percent of the issue slots.  Runs are as
// long as gives every multiprocessor its warps once.  Rows of an even number of channels that do not start on 16
// bytes are copied 4 bytes at a time; odd ones take kernels of one channel a thread.
// The backward takes p again from x (the forward saves nothing) and keeps dweight and dbias of its run in registers:
// a run's is one partial row, and a second kernel adds them in order (no atomics: the same inputs give the same
// bits).
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

template <typename T, int VEC>
__device__ __forceinline__ void conv_floats(float* v, const RowVec<T, VEC>& r) {
    if constexpr (VEC > 1 && sizeof(T) == 2) {  // two to a register
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
        for (int e = 0; e < VEC; e += 2) unpack<T>(w[e / 2], v[e], v[e + 1]);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = to_f32(r.e[e]);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void conv_read(float* v, const T* p) {
    conv_floats<T, VEC>(v, *reinterpret_cast<const RowVec<T, VEC>*>(p));
}
template <typename T, int VEC>
__device__ __forceinline__ void conv_write(T* p, const float* v) {
    RowVec<T, VEC> r;
    if constexpr (VEC > 1 && sizeof(T) == 2) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
        for (int e = 0; e < VEC; e += 2) w[e / 2] = pack<T>(v[e], v[e + 1]);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) r.e[e] = from_f32<T>(v[e]);
    }
    *reinterpret_cast<RowVec<T, VEC>*>(p) = r;
}

// A thread's VEC channels as float32, two to a register pair where there are two.
__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ f32x2 vfma(f32x2 a, f32x2 b, f32x2 c) { return fma2(a, b, c); }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ f32x2 vmul(f32x2 a, f32x2 b) { return mul2(a, b); }
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ f32x2 vadd(f32x2 a, f32x2 b) { return add2(a, b); }
template <int VEC>
struct ConvVal {
    using P = f32x2;
    static constexpr int N = VEC / 2;
    P v[N];
    __device__ __forceinline__ void set(const float* f) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = pair(f[2 * i], f[2 * i + 1]);
    }
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int i = 0; i < N; ++i) halves(v[i], f[2 * i], f[2 * i + 1]);
    }
};
template <>
struct ConvVal<1> {
    using P = float;
    static constexpr int N = 1;
    P v[1];
    __device__ __forceinline__ void set(const float* f) { v[0] = f[0]; }
    __device__ __forceinline__ void get(float* f) const { f[0] = v[0]; }
};

// One thread's channels: taps, and the inputs in front of token t0.
template <typename T, int VEC, int W>
struct ConvCols {
    using Val = ConvVal<VEC>;
    Val w[W], bias;
    __device__ __forceinline__ void taps(const ConvArgs& a, int c) {
        float f[VEC];
#pragma unroll
        for (int k = 0; k < W; ++k) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = read_param(a.weight, a.w_dtype, (c + e) * W + k, 0.f);
            w[k].set(f);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = read_param(a.bias, a.w_dtype, c + e, 0.f);
        bias.set(f);
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
    // the window in front of token t0, one place behind (a token moves it on)
    static __device__ __forceinline__ void window(Val* win, const ConvArgs& a, const T* x, int64_t b, int64_t t0, int c) {
        float v[VEC];
#pragma unroll
        for (int k = 1; k < W; ++k) {
            input(v, a, x, b, t0 - W + k, c);
            win[k].set(v);
        }
    }
    __device__ __forceinline__ void dot(float* p, const Val* win) const {
        Val q = bias;
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
            for (int i = 0; i < Val::N; ++i) q.v[i] = vfma(w[k].v[i], win[k].v[i], q.v[i]);
        q.get(p);
    }
};

// One run of one thread's channels, forward: a token's input comes in, its output goes out.
template <typename T, int VEC, int W>
struct ConvFwd {
    using Cols = ConvCols<T, VEC, W>;
    using V = RowVec<T, VEC>;
    Cols cols;
    typename Cols::Val win[W];  // the inputs a token sees, its own last
    __device__ __forceinline__ void token(const V& v, T* y, bool silu) {
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) win[k] = win[k + 1];
        float p[VEC];
        conv_floats<T, VEC>(p, v);
        win[W - 1].set(p);
        cols.dot(p, win);
        if (silu)
#pragma unroll
            for (int e = 0; e < VEC; ++e) p[e] *= sigmoid(p[e]);
        conv_write<T, VEC>(y, p);
    }
};
// The state behind row b, by the threads of its first run.
template <typename T, int VEC, int W>
__device__ __forceinline__ void conv_final(const ConvArgs& a, const T* x, int64_t b, int64_t len, int c) {
    float v[VEC];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        ConvCols<T, VEC, W>::input(v, a, x, b, len - (W - 1) + k, c);
        conv_write<T, VEC>(static_cast<T*>(a.hN) + (b * (W - 1) + k) * a.D + c, v);
    }
}

// ... and backward: a token gives dp; the gradient of the input W - 1 tokens before it is then whole.
template <typename T, int VEC, int W>
struct ConvBwd {
    using Cols = ConvCols<T, VEC, W>;
    using Val = typename Cols::Val;
    using V = RowVec<T, VEC>;
    Cols cols;
    Val win[W], dp[W];  // dp of the token and of the W - 1 before it
    Val dw[W + 1];      // the taps' sums, the bias's last
    __device__ __forceinline__ void clear() {
        const float nil[VEC] = {};
#pragma unroll
        for (int k = 0; k < W; ++k) dp[k].set(nil);
#pragma unroll
        for (int k = 0; k <= W; ++k) dw[k].set(nil);
    }
    __device__ __forceinline__ void shift() {
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) dp[k] = dp[k + 1], win[k] = win[k + 1];
    }
    __device__ __forceinline__ void token(const V& vx, const V& vg, bool mine, bool silu) {  // mine: one of the run's own
        float p[VEC], g[VEC];
        conv_floats<T, VEC>(p, vx);
        conv_floats<T, VEC>(g, vg);
        win[W - 1].set(p);
        if (silu) {
            cols.dot(p, win);
#pragma unroll
            for (int e = 0; e < VEC; ++e) g[e] *= silu_slope(p[e], sigmoid(p[e]));
        }
        dp[W - 1].set(g);
        if (mine)
#pragma unroll
            for (int i = 0; i < Val::N; ++i) {
                dw[W].v[i] = vadd(dw[W].v[i], dp[W - 1].v[i]);
#pragma unroll
                for (int k = 0; k < W; ++k) dw[k].v[i] = vfma(dp[W - 1].v[i], win[k].v[i], dw[k].v[i]);
            }
    }
    __device__ __forceinline__ void gradient(float* f) const {
        Val g;
#pragma unroll
        for (int i = 0; i < Val::N; ++i) {
            g.v[i] = vmul(cols.w[0].v[i], dp[W - 1].v[i]);
#pragma unroll
            for (int k = 1; k < W; ++k) g.v[i] = vfma(cols.w[k].v[i], dp[W - 1 - k].v[i], g.v[i]);
        }
        g.get(f);
    }
    // Token tt of row b near either end of the run t0.., whose own tokens end at tl; dx: the row's first token.
    __device__ __forceinline__ void any(const ConvArgs& a, T* dx, const V& vx, const V& vg, int64_t b, int c, int64_t tt, int64_t t0, int64_t tl,
                                        int64_t len) {
        const int64_t o = tt - (W - 1), first = t0 == 0 ? -(W - 1) : t0;  // a row's first run reaches back to the state
        const float nil[VEC] = {};
        shift();
        if (tt < len) token(vx, vg, tt < tl, a.silu);
        else dp[W - 1].set(nil);
        if (o < first || o >= len) return;
        float g[VEC];
        gradient(g);
        const int64_t f = o - (len - (W - 1));  // its place in the final state
        if (a.dhN && f >= 0) {
            float v[VEC];
            conv_read<T, VEC>(v, static_cast<const T*>(a.dhN) + (b * (W - 1) + f) * a.D + c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) g[e] += v[e];
        }
        if (o >= 0) conv_write<T, VEC>(dx + o * a.D, g);
        else if (a.dh0) conv_write<T, VEC>(static_cast<T*>(a.dh0) + (b * (W - 1) + o + W - 1) * a.D + c, g);
    }
    // The run's sums: one partial row.
    __device__ __forceinline__ void whole(const ConvArgs& a, int c, bool live) const {
        if (!a.part || !live) return;
        float* part = a.part + static_cast<int64_t>(blockIdx.y) * a.D * (W + 1);
#pragma unroll
        for (int k = 0; k <= W; ++k) {
            float v[VEC];
            dw[k].get(v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) part[k < W ? (c + e) * W + k : a.D * W + c + e] = v[e];
        }
    }
    // The sums of the CTA's R runs, added in order: one partial row.
    template <int R>
    __device__ __forceinline__ void sums(const ConvArgs& a, int c, bool live) const {
        __shared__ float comb[R][32];
        if (!a.part) return;
        const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
        float* part = a.part + static_cast<int64_t>(blockIdx.y) * a.D * (W + 1);
#pragma unroll
        for (int k = 0; k <= W; ++k) {
            float v[VEC];
            dw[k].get(v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                __syncthreads();
                comb[run][lane] = v[e];
                __syncthreads();
                if (run == 0 && live) {
                    float s = comb[0][lane];
#pragma unroll
                    for (int j = 1; j < R; ++j) s += comb[j][lane];
                    part[k < W ? (c + e) * W + k : a.D * W + c + e] = s;
                }
            }
        }
    }
};

constexpr int kConvRuns = 4;  // runs a CTA, one a warp

// ---- one channel a thread: any strides --------------------------------------------------------------------
template <typename T, int W, int U>
__global__ void __launch_bounds__(32 * kConvRuns) conv_fwd_any_k(const ConvArgs a) {
    const int c = blockIdx.x * 32 + (threadIdx.x & 31);
    const int64_t r = static_cast<int64_t>(blockIdx.y) * kConvRuns + (threadIdx.x >> 5);
    if (c >= a.D || r >= a.rows * a.runs) return;
    const int64_t b = r / a.runs, len = conv_length(a, b);
    const int64_t t0 = (r - b * a.runs) * a.run, t1 = min(t0 + a.run, a.L), tl = min(t1, len);
    const T* x = static_cast<const T*>(a.x) + b * a.sx[0] + c;
    T* y = static_cast<T*>(a.y) + b * a.L * a.D + c;
    ConvFwd<T, 1, W> f;
    f.cols.taps(a, c);
    if (t0 < tl) ConvCols<T, 1, W>::window(f.win, a, x, b, t0, c);
    for (int64_t t = t0; t < tl; t += U) {
        RowVec<T, 1> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t + u < tl) raw[u].e[0] = x[(t + u) * a.sx[1]];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t + u < tl) f.token(raw[u], y + (t + u) * a.D, a.silu);
    }
    for (int64_t t = max(t0, tl); t < t1; ++t) y[t * a.D] = from_f32<T>(0.f);
    if (a.hN && t0 == 0) conv_final<T, 1, W>(a, x, b, len, c);
}

template <typename T, int W, int U>
__global__ void __launch_bounds__(32 * kConvRuns) conv_bwd_any_k(const ConvArgs a) {
    const int c = blockIdx.x * 32 + (threadIdx.x & 31);
    const int64_t r = static_cast<int64_t>(blockIdx.y) * kConvRuns + (threadIdx.x >> 5);
    ConvBwd<T, 1, W> f;
    f.clear();
    if (c < a.D && r < a.rows * a.runs) {
        const int64_t b = r / a.runs, len = conv_length(a, b);
        const int64_t t0 = (r - b * a.runs) * a.run, t1 = min(t0 + a.run, a.L), tl = min(t1, len);
        const T* x = static_cast<const T*>(a.x) + b * a.sx[0] + c;
        const T* dy = static_cast<const T*>(a.dy) + b * a.sdy[0] + c;
        T* dx = static_cast<T*>(a.dx) + b * a.L * a.D + c;
        f.cols.taps(a, c);
        if (t0 < tl) ConvCols<T, 1, W>::window(f.win, a, x, b, t0, c);
        const int64_t stop = t0 < len || t0 == 0 ? tl + W - 1 : t0;
        for (int64_t t = t0; t < stop; t += U) {
            RowVec<T, 1> rx[U], rg[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (t + u < min(stop, len)) rx[u].e[0] = x[(t + u) * a.sx[1]], rg[u].e[0] = dy[(t + u) * a.sdy[1]];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (t + u < stop) f.any(a, dx, rx[u], rg[u], b, c, t + u, t0, tl, len);
        }
        for (int64_t t = max(t0, tl); t < t1; ++t) dx[t * a.D] = from_f32<T>(0.f);
    }
    f.template sums<kConvRuns>(a, c, c < a.D);
}

// ---- two channels a lane, rows through shared memory -------------------------------------------------------
constexpr int kConvU = 8, kConvStages = 4;  // tokens a stage; stages a warp
constexpr int kConvTiles = 4;               // warps of a CTA, side by side: rows of 512 bytes (float32: 1024) at a time

// A warp's stages of N inputs: rows of 64 channels, copied in pieces of PIECE bytes (16, or 4 where rows are only so
// aligned); tokens from `left` on and channels from `width` on are not read.
template <typename T, int N, int PIECE>
struct ConvStages {
    static constexpr int kRow = 64, kEach = PIECE / sizeof(T), kPieces = kRow / kEach;  // elements a piece, pieces a row
    static constexpr size_t kBytes = static_cast<size_t>(kConvStages) * N * kConvU * kRow * sizeof(T);
    T* mem;
    __device__ __forceinline__ T* row(int stage, int n, int u) const { return mem + ((stage * N + n) * kConvU + u) * kRow; }
    // src[n]: token t, the tile's first channel
    __device__ __forceinline__ void ask(int stage, const T* const (&src)[N], const int64_t (&stride)[N], int64_t left, int width, int lane) const {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < kConvU * kPieces / 32; ++i) {
                const int u = (i * 32 + lane) / kPieces, q = (i * 32 + lane) % kPieces * kEach;
                if (u < left && q < width) {
                    if constexpr (PIECE == 16) cp_async16(row(stage, n, u) + q, src[n] + u * stride[n] + q, true);
                    else cp_async4(row(stage, n, u) + q, src[n] + u * stride[n] + q, true);
                }
            }
        cp_async_commit();
    }
    // the stage asked for longest ago is there (one a turn is asked for, if of nothing)
    __device__ __forceinline__ void wait() const {
        asm volatile("cp.async.wait_group %0;" ::"n"(kConvStages - 2) : "memory");
        __syncwarp();
    }
};

template <typename T, int W, int PIECE>
__global__ void __launch_bounds__(32 * kConvTiles) conv_fwd_k(const ConvArgs a) {
    using V = RowVec<T, 2>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, c0 = (blockIdx.x * kConvTiles + wid) * 64, c = c0 + lane * 2;
    const ConvStages<T, 1, PIECE> st{reinterpret_cast<T*>(smem + wid * ConvStages<T, 1, PIECE>::kBytes)};
    const int64_t r = blockIdx.y;
    if (c0 >= a.D) return;
    const int64_t b = r / a.runs, len = conv_length(a, b);
    const int64_t t0 = (r - b * a.runs) * a.run, t1 = min(t0 + a.run, a.L), tl = min(t1, len);
    const bool live = c < a.D;
    const T* x = static_cast<const T*>(a.x) + b * a.sx[0] + c0;
    T* y = static_cast<T*>(a.y) + b * a.L * a.D + c;
    const T* src[1] = {x + t0 * a.sx[1]};
    const int64_t stride[1] = {a.sx[1]};
    int64_t asked = t0;
    int slot = 0;
    auto ask = [&] {
        st.ask(slot, src, stride, tl - asked, a.D - c0, lane);
        slot = slot + 1 == kConvStages ? 0 : slot + 1;
        src[0] += kConvU * a.sx[1];
        asked += kConvU;
    };
    for (int i = 0; i + 1 < kConvStages; ++i) ask();
    ConvFwd<T, 2, W> f;
    f.cols.taps(a, live ? c : 0);
    if (t0 < tl && live) ConvCols<T, 2, W>::window(f.win, a, x + lane * 2, b, t0, c);
    T* py = y + t0 * a.D;
    int now = 0;
    for (int64_t t = t0; t < tl; t += kConvU, py += kConvU * static_cast<int64_t>(a.D)) {
        st.wait();
        ask();
        const T* p = st.row(now, 0, 0) + lane * 2;
        now = now + 1 == kConvStages ? 0 : now + 1;
        if (!live) continue;
        if (t + kConvU <= tl) {
#pragma unroll
            for (int u = 0; u < kConvU; ++u) f.token(*reinterpret_cast<const V*>(p + u * 64), py + u * static_cast<int64_t>(a.D), a.silu);
        } else {
#pragma unroll 1
            for (int u = 0; t + u < tl; ++u) f.token(*reinterpret_cast<const V*>(p + u * 64), py + u * static_cast<int64_t>(a.D), a.silu);
        }
    }
    cp_async_wait_all();
    if (!live) return;
    const float nil[2] = {};
    for (int64_t t = max(t0, tl); t < t1; ++t) conv_write<T, 2>(y + t * a.D, nil);
    if (a.hN && t0 == 0) conv_final<T, 2, W>(a, x + lane * 2, b, len, c);
}

template <typename T, int W, int PIECE>
__global__ void __launch_bounds__(32 * kConvTiles) conv_bwd_k(const ConvArgs a) {
    using V = RowVec<T, 2>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, c0 = (blockIdx.x * kConvTiles + wid) * 64, c = c0 + lane * 2;
    const ConvStages<T, 2, PIECE> st{reinterpret_cast<T*>(smem + wid * ConvStages<T, 2, PIECE>::kBytes)};
    const int64_t r = blockIdx.y;
    const bool live = c < a.D;
    ConvBwd<T, 2, W> f;
    f.clear();
    if (c0 < a.D) {
        const int64_t b = r / a.runs, len = conv_length(a, b);
        const int64_t t0 = (r - b * a.runs) * a.run, t1 = min(t0 + a.run, a.L), tl = min(t1, len);
        const T* x = static_cast<const T*>(a.x) + b * a.sx[0] + c0;
        const T* dy = static_cast<const T*>(a.dy) + b * a.sdy[0] + c0;
        T* dx = static_cast<T*>(a.dx) + b * a.L * a.D + c;
        const int64_t stop = t0 < len || t0 == 0 ? tl + W - 1 : t0;
        const T* src[2] = {x + t0 * a.sx[1], dy + t0 * a.sdy[1]};
        const int64_t stride[2] = {a.sx[1], a.sdy[1]};
        int64_t asked = t0;
        int slot = 0;
        auto ask = [&] {
            st.ask(slot, src, stride, min(stop, len) - asked, a.D - c0, lane);
            slot = slot + 1 == kConvStages ? 0 : slot + 1;
            src[0] += kConvU * a.sx[1];
            src[1] += kConvU * a.sdy[1];
            asked += kConvU;
        };
        for (int i = 0; i + 1 < kConvStages; ++i) ask();
        f.cols.taps(a, live ? c : 0);
        if (t0 < tl && live) ConvCols<T, 2, W>::window(f.win, a, x + lane * 2, b, t0, c);
        T* pd = dx + (t0 - (W - 1)) * a.D;
        int now = 0;
        for (int64_t t = t0; t < stop; t += kConvU, pd += kConvU * static_cast<int64_t>(a.D)) {
            st.wait();
            ask();
            const T *px = st.row(now, 0, 0) + lane * 2, *pg = st.row(now, 1, 0) + lane * 2;
            now = now + 1 == kConvStages ? 0 : now + 1;
            if (!live) continue;
            // inside the run every token is its own and completes an input of the run, none of which is in the final state
            if (t > t0 && t + kConvU <= tl) {
#pragma unroll
                for (int u = 0; u < kConvU; ++u) {
                    f.shift();
                    f.token(*reinterpret_cast<const V*>(px + u * 64), *reinterpret_cast<const V*>(pg + u * 64), true, a.silu);
                    float g[2];
                    f.gradient(g);
                    conv_write<T, 2>(pd + u * static_cast<int64_t>(a.D), g);
                }
            } else {
#pragma unroll 1
                for (int u = 0; u < kConvU && t + u < stop; ++u)
                    f.any(a, dx, *reinterpret_cast<const V*>(px + u * 64), *reinterpret_cast<const V*>(pg + u * 64), b, c, t + u, t0, tl, len);
            }
        }
        cp_async_wait_all();
        const float nil[2] = {};
        if (live)
            for (int64_t t = max(t0, tl); t < t1; ++t) conv_write<T, 2>(dx + t * a.D, nil);
    }
    f.whole(a, c, live);
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
    ConvVal<VEC> win[W];
    float p[VEC];
#pragma unroll
    for (int k = 0; k < W; ++k) {
        conv_floats<T, VEC>(p, raw[k]);
        win[k].set(p);
    }
    cols.dot(p, win);
    if (a.silu)
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[e] *= sigmoid(p[e]);
    conv_write<T, VEC>(static_cast<T*>(a.y) + b * a.D + c, p);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) *reinterpret_cast<RowVec<T, VEC>*>(h + static_cast<int64_t>(k) * a.D) = raw[k + 1];
}

// ---------------------------------------------------------------------------------------------------------
// Runs that give every multiprocessor its `warps` once, with `tiles` warps side by side a run; whole stages.
void conv_runs(ConvArgs& a, int64_t tiles, int warps) {
    const int64_t want = std::max<int64_t>(1, int64_t{148} * warps / (tiles * std::max<int64_t>(a.rows, 1)));
    a.run = ((a.L + want - 1) / want + kConvU - 1) / kConvU * kConvU;
    a.run = std::max<int64_t>(a.run, kConvU);
    a.runs = static_cast<int>(std::max<int64_t>(1, (a.L + a.run - 1) / a.run));
}
// The backward's: warps that are resident whatever the kernel, as its number of partial rows is part of the workspace.
constexpr int kConvBwdWarps = 16;
int64_t conv_bwd_rows(ConvArgs& a, bool staged) {
    conv_runs(a, (a.D + (staged ? 63 : 31)) / (staged ? 64 : 32), kConvBwdWarps);
    return staged ? a.rows * a.runs : (a.rows * a.runs + kConvRuns - 1) / kConvRuns;
}
dim3 conv_grid(const ConvArgs& a) {
    return dim3((a.D + 64 * kConvTiles - 1) / (64 * kConvTiles), static_cast<unsigned>(a.rows * a.runs));
}
dim3 conv_grid_any(const ConvArgs& a) {
    return dim3((a.D + 31) / 32, static_cast<unsigned>((a.rows * a.runs + kConvRuns - 1) / kConvRuns));
}

template <typename T, int W, int PIECE>
cudaError_t conv_fwd_staged(ConvArgs& a, cudaStream_t s) {
    constexpr size_t smem = kConvTiles * ConvStages<T, 1, PIECE>::kBytes;
    static const int per = row_resident(conv_fwd_k<T, W, PIECE>, 32 * kConvTiles, smem);
    conv_runs(a, (a.D + 63) / 64, per * kConvTiles);
    conv_fwd_k<T, W, PIECE><<<conv_grid(a), 32 * kConvTiles, smem, s>>>(a);
    note_launch();
    return cudaGetLastError();
}
template <typename T, int W, int PIECE>
cudaError_t conv_bwd_staged(const ConvArgs& a, cudaStream_t s) {
    constexpr size_t smem = kConvTiles * ConvStages<T, 2, PIECE>::kBytes;
    const cudaError_t e = cudaFuncSetAttribute(conv_bwd_k<T, W, PIECE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    conv_bwd_k<T, W, PIECE><<<conv_grid(a), 32 * kConvTiles, smem, s>>>(a);
    note_launch();
    return cudaGetLastError();
}
// piece: the bytes that the staged kernels may copy at once, or 0
template <typename T, int W>
cudaError_t conv_fwd_launch(ConvArgs& a, int piece, cudaStream_t s) {
    if (piece == 16) return conv_fwd_staged<T, W, 16>(a, s);
    if (piece == 4) return conv_fwd_staged<T, W, 4>(a, s);
    constexpr int threads = 32 * kConvRuns;
    static const int per = row_resident(conv_fwd_any_k<T, W, 8>, threads, 0);
    conv_runs(a, (a.D + 31) / 32, per * kConvRuns);
    conv_fwd_any_k<T, W, 8><<<conv_grid_any(a), threads, 0, s>>>(a);
    note_launch();
    return cudaGetLastError();
}
template <typename T, int W>
cudaError_t conv_bwd_launch(ConvArgs& a, int piece, void* dweight, void* dbias, cudaStream_t s) {
    const int64_t rows = conv_bwd_rows(a, piece != 0);
    cudaError_t e;
    if (piece) {
        e = piece == 16 ? conv_bwd_staged<T, W, 16>(a, s) : conv_bwd_staged<T, W, 4>(a, s);
    } else {
        conv_bwd_any_k<T, W, 4><<<conv_grid_any(a), 32 * kConvRuns, 0, s>>>(a);
        note_launch();
        e = cudaGetLastError();
    }
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

template <typename T>
cudaError_t conv_fwd_any(ConvArgs& a, int width, int piece, cudaStream_t s) {
    return width == 2 ? conv_fwd_launch<T, 2>(a, piece, s) : width == 3 ? conv_fwd_launch<T, 3>(a, piece, s) : conv_fwd_launch<T, 4>(a, piece, s);
}
template <typename T, int VEC>
cudaError_t conv_step_width(ConvArgs& a, int width, cudaStream_t s) {
    return width == 2 ? conv_step_launch<T, VEC, 2>(a, s) : width == 3 ? conv_step_launch<T, VEC, 3>(a, s) : conv_step_launch<T, VEC, 4>(a, s);
}
template <typename T>
cudaError_t conv_step_any(ConvArgs& a, int width, bool vec, cudaStream_t s) {
    return vec ? conv_step_width<T, 4>(a, width, s) : conv_step_width<T, 1>(a, width, s);
}
template <typename T>
cudaError_t conv_bwd_any(ConvArgs& a, int width, int piece, void* dw, void* db, cudaStream_t s) {
    return width == 2   ? conv_bwd_launch<T, 2>(a, piece, dw, db, s)
           : width == 3 ? conv_bwd_launch<T, 3>(a, piece, dw, db, s)
                        : conv_bwd_launch<T, 4>(a, piece, dw, db, s);
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

// What the staged kernels may copy at once: 16 bytes, or 4 where pairs of channels (which they write) are aligned at least.
int conv_piece(const EacsConv& p, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
    if (conv_vec(p, p.dtype == EACS_DTYPE_F32 ? 4 : 8, ptrs, strides)) return 16;
    return conv_vec(p, 2, ptrs, strides) ? 4 : 0;
}

}  // namespace

// The partial rows of a backward, whichever of its kernels has more.
size_t conv_bwd_workspace_size(const EacsConv& p) {
    if (conv_check("eacs_conv_bwd_workspace_size", p, false) != EACS_OK || p.rows == 0) return 0;
    ConvArgs a = conv_args(p);
    const int64_t rows = std::max(conv_bwd_rows(a, false), conv_bwd_rows(a, true));
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
    const int piece = conv_piece(p, {p.x, y, p.initial_state, final_state}, {p.x_stride[0], p.x_stride[1]});
    const cudaError_t e = p.dtype == EACS_DTYPE_F32   ? conv_fwd_any<float>(a, p.width, piece, stream)
                          : p.dtype == EACS_DTYPE_F16 ? conv_fwd_any<__half>(a, p.width, piece, stream)
                                                      : conv_fwd_any<__nv_bfloat16>(a, p.width, piece, stream);
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
    const int piece = conv_piece(p, {p.x, p.initial_state, g.dy, g.dfinal, g.dx, g.dinitial},
                                 {p.x_stride[0], p.x_stride[1], g.dy_stride[0], g.dy_stride[1]});
    const cudaError_t e = p.dtype == EACS_DTYPE_F32   ? conv_bwd_any<float>(a, p.width, piece, g.dweight, g.dbias, stream)
                          : p.dtype == EACS_DTYPE_F16 ? conv_bwd_any<__half>(a, p.width, piece, g.dweight, g.dbias, stream)
                                                      : conv_bwd_any<__nv_bfloat16>(a, p.width, piece, g.dweight, g.dbias, stream);
    return cuda_check(e, fn);
}

}  // namespace eacs
