// selective.cu -- the selective state space scan: sequences, their gradients and single tokens (sm_100a).
//
// Channel d of a row keeps N states.  With s = softplus(dt + dt_bias) (or dt + dt_bias itself), per token
//   h_t[n] = e^(s_t A[n]) h_{t-1}[n] + s_t x_t B_t[n],   o_t = sum_n C_t[n] h_t[n] + skip x_t,   y_t = o_t silu(z_t).
// Gradients: with do = dy silu(z) and g_t the gradient of h_t, backwards from the final state's gradient,
//   g_t[n] = C_t[n] do_t + e^(s_{t+1} A[n]) g_{t+1}[n]
//   dC_t[n] = sum_d do_t h_t[n]         dB_t[n] = sum_d s_t x_t g_t[n]      (sums over the channels)
//   dv_t    = sum_n B_t[n] g_t[n]       (the gradient of s x)
//   w_t[n]  = g_t[n] e^(s_t A[n]) h_{t-1}[n]
//   ds_t    = sum_n A[n] w_t[n] + x_t dv_t,   dx_t = s_t dv_t + skip do_t
//   dA[n]   = sum_t s_t w_t[n],   dskip = sum_t do_t x_t,   dz = dy o silu'(z),   ddt = ds softplus'.
//
// One exponential per token, channel and state is what it cannot do without: 16 a clock and multiprocessor, which is
// 230 us for the 1.07e9 of B=4 L=16384 D=1024 N=16 (with those of softplus and silu 290) against 82 us of memory traffic.
// A warp takes a slice of 8 tokens of a few channels at a time; the warps of a CTA take consecutive slices of the same
// channels and hand the state around a ring, so that the only thing in sequence is a few multiply-adds a slice.  (One warp
// for all of a row's tokens would leave a scheduler with less than one warp at that size.)  Pairs of states are multiplied
// and added by the two-wide float32 instructions, which take half the issue slots.
//
// Measured, us: forward B=4 L=16384 D=1024 N=16 bfloat16 637; B=1 322; B=8 L=8192 D=768 485 (528 with checkpoints), the
// backward of that 1364 and 28 for the sums of dB and dC.  What holds it off the exponentials' time is latency: 12 warps
// a multiprocessor (backward 8) with the registers that a slice's decays and sums take, at 12 (backward 26) instructions
// for 32 updates; the special function pipe is 45 percent busy, issue slots 59 percent (backward 18 and 47).  The
// backward's kernels for one group a CTA spill registers for N <= 8 (116 to 168 bytes a thread; others at most 72, the
// forward's at most 24).  Tried and slower: slices of 4 tokens with 16 or 20 warps (813 and 894 us where 8 with 12 took
// 745), in the backward slices of 4 with two channels a thread and 12 warps (half the shared memory reads, but half again
// as many instructions: 2477 us a training step where 1971 was), and the tokens' values of all of a CTA's groups worked
// out at once (2180 where 1900 was).
//
// The forward for training writes the state in front of every 8 tokens; the backward starts a slice from it.  Sums over
// channels stay in registers while a warp goes through its CTA's channels, are then folded over its lanes, and a CTA writes
// one partial row of dB and dC that a second kernel adds in order (no atomics: the same inputs give the same bits).
#include <algorithm>

#include "eacs_common.cuh"
#include "eacs_host.h"

namespace eacs {
namespace {

__device__ __forceinline__ float both(f32x2 v) {
    float a, b;
    halves(v, a, b);
    return a + b;
}
__device__ __forceinline__ f32x2 ex2_pair(f32x2 v) {
    float a, b;
    halves(v, a, b);
    return pair(ex2_approx(a), ex2_approx(b));
}
struct alignas(16) Quad { f32x2 lo, hi; };  // four states

// The decays e^(s A) of two states, from s log2(e).  The hardware's 2^v comes out low by 2e-8 to 3e-8 of itself on average
// for v in (-0.25, -0.001) (measured against 64 bits), the same way for every token: a state that decays slowly collects
// it (dA was 3 times further from its value in 64 bits than sums of correctly rounded decays).  kEx2Low, added to v by the
// multiply-add that would be a product otherwise, takes the mean of it back; 2^kEx2Low is 1 exactly, so that a step of 0
// keeps the state.
constexpr float kEx2Low = 2.3e-8f;
__device__ __forceinline__ f32x2 decays(f32x2 s2, f32x2 A) { return ex2_pair(fma2(s2, A, pair(kEx2Low, kEx2Low))); }

// ---- a token's step and gate ----------------------------------------------------------------------------
// softplus(v) = max(v, 0) + log(1 + u) with u = e^-|v| and log(1 + u) = 2 artanh(q), q = u / (2 + u) <= 1/3: relatively
// exact for the small steps that v << 0 gives, where log(1 + u) taken from the rounded 1 + u is not.  2 artanh(q) / q is a
// polynomial of degree 4 in q^2, fitted on [0, 1/9] at Chebyshev's points (8e-9 of the value).  What u's argument lost, the
// product's rounding and that of log2(e), is put back to first order (without the first u is off by |v| 2^-24, without the
// second by |v| 2^-26): 2^-20 of the step in all.  Behind e^-87.3, where float32's normal numbers end, the hardware's 2^v is 0
// (v is held to where the argument's rest is a number), so that -inf or the lowest value in dt masks a token: it takes no step.
// slope is the derivative.
__device__ __forceinline__ float softplus(float v, float& slope) {
    const float t = fmaxf(-fabsf(v), -200.0f), p0 = t * kLog2e;
    float u = ex2_approx(p0);
    u = fmaf(u * fmaf(t, kLog2eLow, fmaf(t, kLog2e, -p0)), kLn2, u);
    const float q = __fdividef(u, 2.0f + u), q2 = q * q;
    float p = fmaf(q2, 0.2817465663f, 0.2796141803f);
    p = fmaf(q2, p, 0.4002485275f);
    p = fmaf(q2, p, 0.6666631699f);
    p = fmaf(q2, p, 2.0f);
    const float inv = __fdividef(1.0f, 1.0f + u);
    slope = v >= 0.0f ? inv : u * inv;
    return fmaf(q, p, v < 0.0f ? 0.0f : v);  // (a NaN stays one)
}

struct SelArgs {
    const void *x, *dt, *z, *B, *C;      // z may be null
    int64_t sx[2], sdt[2], sz[2], sB[2], sC[2];  // strides of batch and token
    const float *A, *skip, *bias;        // skip and bias may be null
    const int32_t* lengths;
    const float* h0;                     // or null
    void* y;
    float* hN;                           // or null
    float* ckpt;                         // or null: states in front of every 8 tokens, (B, ceil(L / 8), D, 4 LN)
    int L, D, N;
    int softplus;
    int vec, vec_bc;                     // rows of x, dt, z (y, dy ...) / of B, C may be read as vectors
    // backward
    const void* dy;
    int64_t sdy[2];
    const float* dhN;                    // or null
    void *dx, *ddt, *dz;
    float *partB, *partC;                // (CTAs of a row, B, L, 4 LN)
    float* partA;                        // (B, D, 4 LN)
    float* partS;                        // (B, 2, D): dskip, ddt_bias
    float* dh0;                          // or null
    int64_t Bn;
    int groups;                          // groups of channels a CTA
};

__device__ __forceinline__ int sel_length(const SelArgs& a, int64_t b) {
    if (!a.lengths) return a.L;
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n > a.L ? a.L : n);
}

// E neighbouring channels of one token as they lie in memory, in whole registers: taken apart only where they are used, so
// that asking for them does not wait for them.
// FULL: all of the channels are there, and vectors may be read.  Else a lane whose channels may not be read as a vector keeps
// each in a register of its own.
template <typename T, int E, bool FULL>
struct Run {
    static constexpr int kBytes = E * sizeof(T), kPacked = (kBytes + 3) / 4, kPer = 4 / sizeof(T), kWords = FULL ? kPacked : E;
    uint32_t w[kWords];
    // the channels d.. of D
    static __device__ __forceinline__ bool packed(int d, int D, bool vec) { return FULL || (vec && d + E <= D); }
    __device__ __forceinline__ void read(const T* p, bool in, int d, int D, bool vec) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
        if (!in) return;
        if (packed(d, D, vec)) {
            if constexpr (kBytes >= 16) {
#pragma unroll
                for (int i = 0; i < kPacked; i += 4) {
                    const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
                    w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
                }
            } else if constexpr (kBytes == 8) {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                w[0] = v.x, w[1] = v.y;
            } else if constexpr (kBytes == 4) {
                w[0] = *reinterpret_cast<const uint32_t*>(p);
            } else {
                w[0] = *reinterpret_cast<const uint16_t*>(p);
            }
        } else if constexpr (!FULL) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (d + e < D) {
                    if constexpr (sizeof(T) == 4) w[e] = reinterpret_cast<const uint32_t*>(p)[e];
                    else w[e] = reinterpret_cast<const uint16_t*>(p)[e];
                }
        }
    }
    __device__ __forceinline__ void floats(float* v, bool is_packed) const {
        float a, b;
        if (FULL || sizeof(T) == 4 || is_packed) {
#pragma unroll
            for (int i = 0; i < kPacked; ++i) {
                unpack<T>(w[i], a, b);
                v[i * kPer] = a;
                if (kPer == 2 && i * kPer + 1 < E) v[i * kPer + 1] = b;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) unpack<T>(w[e < kWords ? e : 0], v[e], b);
        }
    }
};
template <typename T, int E, bool FULL = false>
__device__ __forceinline__ void write_run(const float* v, T* p, int d, int D, bool vec) {
    using R = Run<T, E, true>;
    if ((FULL || (vec && d + E <= D)) && R::kBytes >= 4) {
        uint32_t w[R::kWords];
#pragma unroll
        for (int i = 0; i < R::kWords; ++i) w[i] = pack<T>(v[i * R::kPer], v[(i * R::kPer + 1) % E]);
        if constexpr (R::kBytes >= 16) {
#pragma unroll
            for (int i = 0; i < R::kWords; i += 4) reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else if constexpr (R::kBytes == 8) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else {
            *reinterpret_cast<uint32_t*>(p) = w[0];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (FULL || d + e < D) p[e] = from_f32<T>(v[e]);
    }
}

// E floats to shared memory
template <int E>
__device__ __forceinline__ void put_run(float* p, const float* v) {
    if constexpr (E % 4 == 0) {
#pragma unroll
        for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else if constexpr (E == 2) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else {
        p[0] = v[0];
    }
}

template <int E>
__device__ __forceinline__ void get_run(float* v, const float* p) {
    if constexpr (E % 4 == 0) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 q = *reinterpret_cast<const float4*>(p + e);
            v[e] = q.x, v[e + 1] = q.y, v[e + 2] = q.z, v[e + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = p[e];
    }
}

// Four states of channel d from (.., D, N) float32, zeros outside.
__device__ __forceinline__ float4 read_states(const float* p, int d, int D, int n0, int N) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = d < D && n0 + i < N ? p[static_cast<int64_t>(d) * N + n0 + i] : 0.f;
    return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void write_states(float* p, int d, int D, int n0, int N, Quad h) {
    float v[4];
    halves(h.lo, v[0], v[1]);
    halves(h.hi, v[2], v[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (d < D && n0 + i < N) p[static_cast<int64_t>(d) * N + n0 + i] = v[i];
}
__device__ __forceinline__ Quad quad(float4 v) { return Quad{pair(v.x, v.y), pair(v.z, v.w)}; }

// B and C of a slice of S tokens, by one warp: asked for with cp.async as they lie (where rows allow it), then turned into
// float32 rows of NP = 4 LN states, zeros behind the row's end and behind N.
// FULL: rows of NP states that vectors may be read from.
template <typename T, int LN, int S, bool FULL>
struct SliceBC {
    static constexpr int NP = 4 * LN, V = 16 / sizeof(T);
    static constexpr size_t kRawBytes = 2 * S * NP * sizeof(T), kBytes = 2 * S * NP * sizeof(float);
    const T* B;  // the row's first token
    const T* C;
    T* raw;
    float* out;
    __device__ __forceinline__ void ask(const SelArgs& a, int t0, int len, int lane) const {
        if (!FULL && !a.vec_bc) return;
        constexpr int per = NP / V;  // 16-byte pieces a row, those behind N left out
        const int64_t oB = t0 * a.sB[1], oC = t0 * a.sC[1];
#pragma unroll
        for (int i = 0; i < (S * per + 31) / 32; ++i) {
            const int k = i * 32 + lane, r = k / per, c = k % per * V;
            if (k < S * per && (FULL || c < a.N)) {
                const bool in = t0 + r < len;
                cp_async16(raw + r * NP + c, B + (in ? oB + r * a.sB[1] : 0) + c, in);
                cp_async16(raw + (S + r) * NP + c, C + (in ? oC + r * a.sC[1] : 0) + c, in);
            }
        }
        cp_async_commit();
    }
    __device__ __forceinline__ void take(const SelArgs& a, int t0, int len, int lane) const {
        if (FULL || a.vec_bc) cp_async_wait_all();
        __syncwarp();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const T* g = which ? C : B;
            const int64_t st = which ? a.sC[1] : a.sB[1];
#pragma unroll
            for (int i = 0; i < (S * LN + 31) / 32; ++i) {
                const int k = i * 32 + lane, r = k / LN, n = k % LN * 4;
                if (S * LN < 32 && k >= S * LN) break;
                float v[4] = {};
                if (FULL || a.vec_bc) {
                    if (FULL || n < a.N) {
                        Run<T, 4, true> q;
                        q.read(raw + (which * S + r) * NP + n, true, 0, 4, true);
                        q.floats(v, true);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (t0 + r < len && n + e < a.N) v[e] = to_f32(g[(t0 + r) * st + n + e]);
                }
                *reinterpret_cast<float4*>(out + (which * S + r) * NP + n) = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
    }
    __device__ __forceinline__ Quad b(int t, int ln) const { return *reinterpret_cast<const Quad*>(out + t * NP + ln * 4); }
    __device__ __forceinline__ Quad c(int t, int ln) const { return *reinterpret_cast<const Quad*>(out + (S + t) * NP + ln * 4); }
};

// ---------------------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------------------
// A slice is S tokens of CW channels; a thread holds eight states of a channel.  A token's values are worked out in the
// layout they are read in (lane = token and a quarter of the channels, E of them) and handed to the sweep through shared
// memory.  The sweep starts from a state of zero, so that nothing in it waits for the warp before: it leaves the slice's
// own state, the product P of its decays, its own part of the outputs, and C P of every token.  With the state h handed in,
// the state handed on is own + P h (all that the ring waits for), and the outputs get (C P) . h.
template <int LN>
struct FwdShape {
    static constexpr int S = 8, NP = 4 * LN, L8 = LN / 2, CW = 32 / L8, E = CW / 4;  // L8: threads a channel
    static constexpr int YS = CW + 4;
};
template <typename T, int LN>
constexpr size_t sel_fwd_warp_bytes() {
    using Sh = FwdShape<LN>;
    using BC = SliceBC<T, LN, Sh::S, true>;
    return BC::kRawBytes + BC::kBytes + 2 * Sh::S * Sh::CW * 4 + Sh::S * Sh::YS * 4;
}
// a CTA's own: the states handed on (eight of 32 lanes a warp), dt_bias and skip of its channels
template <int LN>
constexpr size_t sel_fwd_cta_bytes(int W) {
    return W * 1024 + 2 * FwdShape<LN>::CW * 4;
}
constexpr int kSelFwdWarps = 12;  // a multiprocessor's: the registers of one CTA of 12 warps, or of several smaller ones

// FULL: groups of CW channels and rows of NP states, all of them on 16 bytes
template <typename T, int LN, bool CKPT, bool FULL>
__global__ void __launch_bounds__(kSelFwdWarps * 32, 1) sel_fwd_k(const SelArgs a) {
    using Sh = FwdShape<LN>;
    using BC = SliceBC<T, LN, Sh::S, FULL>;
    constexpr int S = Sh::S, NP = Sh::NP, CW = Sh::CW, E = Sh::E;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, W = blockDim.x >> 5;
    Quad* hop = reinterpret_cast<Quad*>(smem);  // [W][2][32]: the state that each warp is handed
    float* pars = reinterpret_cast<float*>(smem + W * 1024);  // [2][CW]: dt_bias, skip
    unsigned char* mine = smem + sel_fwd_cta_bytes<LN>(W) + static_cast<size_t>(w) * sel_fwd_warp_bytes<T, LN>();
    float2* sd = reinterpret_cast<float2*>(mine + BC::kRawBytes + BC::kBytes);  // [S][CW]: s log2 e, s x
    float* yb = reinterpret_cast<float*>(sd + S * CW);                          // [S][YS]: sums over the states

    const int64_t b = blockIdx.y;
    const int d0 = blockIdx.x * CW;
    const int len = sel_length(a, b), slices = (len + S - 1) / S;
    const int ln = lane % Sh::L8, ch = lane / Sh::L8, d = d0 + ch, n0 = ln * 8;  // in the sweep
    const int row = lane / 4, cr = (lane & 3) * E, dr = d0 + cr;             // in memory's layout
    T* y = static_cast<T*>(a.y) + (b * a.L + row) * a.D + dr;
    const BC bc{static_cast<const T*>(a.B) + b * a.sB[0], static_cast<const T*>(a.C) + b * a.sC[0],
                reinterpret_cast<T*>(mine), reinterpret_cast<float*>(mine + BC::kRawBytes)};
    const bool vec = a.vec != 0, gated = a.z != nullptr;

    for (int i = threadIdx.x; i < 2 * CW; i += blockDim.x) {
        const float* p = i < CW ? a.bias : a.skip;
        const int c = d0 + i % CW;
        pars[i] = p && c < a.D ? p[c] : 0.f;
    }
    __syncthreads();
    Quad A[2], h[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        A[c] = quad(read_states(a.A, d, a.D, n0 + 4 * c, a.N));
        h[c] = quad(w == 0 && a.h0 ? read_states(a.h0 + b * a.D * a.N, d, a.D, n0 + 4 * c, a.N) : make_float4(0.f, 0.f, 0.f, 0.f));
    }

    using R = Run<T, E, FULL>;
    R rx, rt, rz;
    const bool packed = R::packed(dr, a.D, vec);
    const int64_t t_first = w * S + row;
    const T* x = static_cast<const T*>(a.x) + b * a.sx[0] + t_first * a.sx[1] + dr;
    const T* dt = static_cast<const T*>(a.dt) + b * a.sdt[0] + t_first * a.sdt[1] + dr;
    const T* z = gated ? static_cast<const T*>(a.z) + b * a.sz[0] + t_first * a.sz[1] + dr : nullptr;
    auto ask = [&](int j) {  // of the warp's next slice
        const bool in = j * S + row < len;
        rx.read(x, in, dr, a.D, vec);
        rt.read(dt, in, dr, a.D, vec);
        if (gated) rz.read(z, in, dr, a.D, vec);
        bc.ask(a, j * S, len, lane);
        x += W * S * a.sx[1];
        dt += W * S * a.sdt[1];
        if (gated) z += W * S * a.sz[1];
    };
    if (w < slices) ask(w);
    for (int j = w; j < slices; j += W) {
        const int t0 = j * S;
        bc.take(a, t0, len, lane);
        const bool in = t0 + row < len;
        const R kx = rx, kz = rz;  // for the outputs
        {
            float xs[E], s[E], bias[E];
            rx.floats(xs, packed);
            rt.floats(s, packed);
            get_run<E>(bias, pars + cr);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float slope;
                s[e] += bias[e];
                if (a.softplus) s[e] = softplus(s[e], slope);
                s[e] = in ? s[e] : 0.f;
                xs[e] *= s[e];
                s[e] *= kLog2e;
            }
            float both_of[2 * E];
#pragma unroll
            for (int e = 0; e < E; ++e) both_of[2 * e] = s[e], both_of[2 * e + 1] = xs[e];
            put_run<2 * E>(reinterpret_cast<float*>(sd + row * CW + cr), both_of);
        }
        __syncwarp();
        if (j + W < slices) ask(j + W);

        Quad own[2], P[2], CP[S][2];
        float v[S];
#pragma unroll
        for (int t = 0; t < S; ++t) {
            const float2 q = sd[t * CW + ch];
            const f32x2 s2 = pair(q.x, q.x), v2 = pair(q.y, q.y);
            f32x2 sum;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Quad Bq = bc.b(t, 2 * ln + c), Cq = bc.c(t, 2 * ln + c);
                const f32x2 a0 = decays(s2, A[c].lo), a1 = decays(s2, A[c].hi);
                const f32x2 b0 = mul2(v2, Bq.lo), b1 = mul2(v2, Bq.hi);
                own[c].lo = t ? fma2(a0, own[c].lo, b0) : b0;
                own[c].hi = t ? fma2(a1, own[c].hi, b1) : b1;
                P[c].lo = t ? mul2(P[c].lo, a0) : a0;
                P[c].hi = t ? mul2(P[c].hi, a1) : a1;
                sum = c ? fma2(Cq.lo, own[c].lo, sum) : mul2(Cq.lo, own[c].lo);
                sum = fma2(Cq.hi, own[c].hi, sum);
                CP[t][c].lo = mul2(Cq.lo, P[c].lo);
                CP[t][c].hi = mul2(Cq.hi, P[c].hi);
            }
            v[t] = both(sum);
        }
        if (j > 0 && W > 1) {
            asm volatile("bar.sync %0, 64;" ::"r"(w) : "memory");
            h[0] = hop[(w * 2) * 32 + lane];
            h[1] = hop[(w * 2 + 1) * 32 + lane];
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            own[c].lo = fma2(P[c].lo, h[c].lo, own[c].lo);
            own[c].hi = fma2(P[c].hi, h[c].hi, own[c].hi);
        }
        if (j + 1 < slices) {
            if (W > 1) {
                const int next = w + 1 == W ? 0 : w + 1;
                hop[(next * 2) * 32 + lane] = own[0];
                hop[(next * 2 + 1) * 32 + lane] = own[1];
                asm volatile("bar.arrive %0, 64;" ::"r"(next) : "memory");
            }
        } else if (a.hN) {
            for (int c = 0; c < 2; ++c) write_states(a.hN + b * a.D * a.N, d, a.D, n0 + 4 * c, a.N, own[c]);
        }
        if constexpr (CKPT) {
            float* k = a.ckpt + ((b * ((a.L + 7) / 8) + j) * a.D + d) * NP + n0;
#pragma unroll
            for (int c = 0; c < 2; ++c)
                if (FULL || d < a.D) *reinterpret_cast<Quad*>(k + 4 * c) = h[c];
        }
#pragma unroll
        for (int t = 0; t < S; ++t) {
            f32x2 sum = mul2(CP[t][0].lo, h[0].lo);
            sum = fma2(CP[t][0].hi, h[0].hi, sum);
            sum = fma2(CP[t][1].lo, h[1].lo, sum);
            v[t] += both(fma2(CP[t][1].hi, h[1].hi, sum));
        }
        if (W == 1) h[0] = own[0], h[1] = own[1];
        Fold<S, Sh::L8 / 2, 1>::run(v, lane);
        const int first = FoldShape<S, Sh::L8 / 2, 1>::held(lane);
#pragma unroll
        for (int i = 0; i < S / Sh::L8; ++i) yb[(first + i) * Sh::YS + ch] = v[i];
        __syncwarp();
        if (t0 + row < a.L) {
            float o[E], xs[E], g[E], skip[E];
            kx.floats(xs, packed);
            get_run<E>(skip, pars + CW + cr);
            get_run<E>(o, yb + row * Sh::YS + cr);
            if (gated) kz.floats(g, packed);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                o[e] = fmaf(skip[e], xs[e], o[e]);
                if (gated) o[e] *= g[e] * sigmoid(g[e]);
                o[e] = in ? o[e] : 0.f;
            }
            write_run<T, E, FULL>(o, y + static_cast<int64_t>(t0) * a.D, dr, a.D, vec);
        }
    }
    // behind the row's end, and a row without a token
    const float nil[E] = {};
    for (int64_t t = static_cast<int64_t>(slices + w) * S; t + row < a.L; t += W * S) write_run<T, E, FULL>(nil, y + t * a.D, dr, a.D, vec);
    if (slices == 0 && w == 0 && a.hN)
        for (int c = 0; c < 2; ++c) write_states(a.hN + b * a.D * a.N, d, a.D, n0 + 4 * c, a.N, h[c]);
}

// ---------------------------------------------------------------------------------------------------------
// single tokens
// ---------------------------------------------------------------------------------------------------------
// LN threads a channel with four states each, R rows a thread (A is read once for them).  64 rows of 2048 channels with N=16:
// 8.9 us where the bytes take 2.8.  A thread moves one vector of states and for it reads A, B, C and the channel's values
// element by element: 17 loads in all, whose issue and latency is the difference.
template <typename T, int LN, int R>
__global__ void __launch_bounds__(256) sel_step_k(const SelArgs a) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int d = i / LN, n0 = i % LN * 4;
    const bool live = d < a.D;
    const float4 A = read_states(a.A, d, a.D, n0, a.N);
    const float bias = live && a.bias ? a.bias[d] : 0.f, skip = live && a.skip ? a.skip[d] : 0.f;
    const int64_t b0 = static_cast<int64_t>(blockIdx.y) * R;
    const bool vec = a.vec != 0;
    float h[R][4], xs[R], raw[R], zs[R], Bv[R][4], Cv[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t b = b0 + r;
        const bool in = live && b < a.Bn;
        const float* p = a.hN + (b * a.D + d) * a.N + n0;
        xs[r] = in ? to_f32(static_cast<const T*>(a.x)[b * a.sx[0] + d]) : 0.f;
        raw[r] = in ? to_f32(static_cast<const T*>(a.dt)[b * a.sdt[0] + d]) + bias : 0.f;
        zs[r] = in && a.z ? to_f32(static_cast<const T*>(a.z)[b * a.sz[0] + d]) : 0.f;
        if (in && vec && n0 < a.N) {
            const float4 q = *reinterpret_cast<const float4*>(p);
            h[r][0] = q.x, h[r][1] = q.y, h[r][2] = q.z, h[r][3] = q.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) h[r][k] = in && n0 + k < a.N ? p[k] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool on = in && n0 + k < a.N;
            Bv[r][k] = on ? to_f32(static_cast<const T*>(a.B)[b * a.sB[0] + n0 + k]) : 0.f;
            Cv[r][k] = on ? to_f32(static_cast<const T*>(a.C)[b * a.sC[0] + n0 + k]) : 0.f;
        }
    }
    const float Av[4] = {A.x, A.y, A.z, A.w};
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t b = b0 + r;
        const bool in = live && b < a.Bn;
        float slope;
        const float s = a.softplus ? softplus(raw[r], slope) : raw[r];
        const float sl = s * kLog2e, v = s * xs[r];
        float o = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[r][k] = fmaf(ex2_approx(fmaf(sl, Av[k], kEx2Low)), h[r][k], v * Bv[r][k]);
            o = fmaf(Cv[r][k], h[r][k], o);
        }
        float* p = a.hN + (b * a.D + d) * a.N + n0;
        if (in && vec && n0 < a.N) {
            *reinterpret_cast<float4*>(p) = make_float4(h[r][0], h[r][1], h[r][2], h[r][3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (in && n0 + k < a.N) p[k] = h[r][k];
        }
#pragma unroll
        for (int m = LN / 2; m > 0; m >>= 1) o += __shfl_xor_sync(0xffffffffu, o, m);
        if (in && i % LN == 0) {
            o = fmaf(skip, xs[r], o);
            if (a.z) o *= zs[r] * sigmoid(zs[r]);
            static_cast<T*>(a.y)[b * a.D + d] = from_f32<T>(o);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------------------
// Slices of 8 tokens from the last to the first, one a warp; a warp takes its slice through the CTA's groups of CW channels
// and hands each group's g on.  Per slice and group: decays and states from the checkpoint, with dC on the way, then
// backwards with dB, dv, w and dA.  A thread holds four states of a channel (LN threads a channel); dB and dC of the slice
// stay in 64 registers a lane over all groups, so that they are folded over the lanes once a slice.
template <int LN>
struct BwdShape {
    static constexpr int S = 8, NP = 4 * LN, CW = 32 / LN;
    static constexpr int E = CW / 4 > 0 ? CW / 4 : 1;  // channels a lane, four lanes a token
    static constexpr int YS = CW + 2;
    static __device__ __forceinline__ int place(int t, int c) { return t * CW + c; }
};
template <typename T, int LN>
constexpr size_t sel_bwd_warp_bytes() {
    using Sh = BwdShape<LN>;
    using BC = SliceBC<T, LN, Sh::S, false>;
    return BC::kRawBytes + BC::kBytes + Sh::S * Sh::CW * 24 + (3 * Sh::S * Sh::YS * 4 + 15) / 16 * 16;
}
// of a group of channels: g handed on, sums of dA, dskip and ddt_bias and a barrier a warp; A, dt_bias and skip
template <int LN>
constexpr size_t sel_bwd_group_bytes(int W) {
    return static_cast<size_t>(W) * (512 + 512 + 2 * BwdShape<LN>::E * 128 + 8) + 512 + 2 * BwdShape<LN>::CW * 4;
}
constexpr int kSelBwdWarps = 8, kSelBwdMaxGroups = 8;

// FULL: groups of CW channels and rows of NP states, all of them on 16 bytes.  AHEAD: what is handed on is worked out
// before the sweep that needs what is handed in (the slice's own end and the product of its decays, as in the forward): with
// one group a CTA nothing else fills the ring's wait (B=1 L=8192 D=768 training step 643 to 546 us); with more the other
// groups do, and the extra products cost (B=8: 1900 us without, 2003 with; two groups, B=2: 741 and 765).  It goes by the
// groups alone: one group is also what the rounds give some sizes with many CTAs (8 rows of 1024 or 1536 channels, N=16).
template <typename T, int LN, bool FULL, bool AHEAD>
__global__ void __launch_bounds__(kSelBwdWarps * 32, 1) sel_bwd_k(const SelArgs a) {
    using Sh = BwdShape<LN>;
    using BC = SliceBC<T, LN, Sh::S, FULL>;
    constexpr int S = Sh::S, NP = Sh::NP, CW = Sh::CW, E = Sh::E, YS = Sh::YS, W = kSelBwdWarps;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, G = a.groups;
    Quad* hop = reinterpret_cast<Quad*>(smem);             // [W][G][32]: the g that each warp is handed
    Quad* dAs = hop + W * G * 32;                          // [W][G][32]
    Quad* As = dAs + W * G * 32;                           // [G][32]
    float* sums = reinterpret_cast<float*>(As + G * 32);   // [W][G][32][2 E]: dskip and ddt_bias of a lane's tokens
    float* pars = sums + W * G * 2 * E * 32;               // [2][G CW]: dt_bias, skip
    uint64_t* bars = reinterpret_cast<uint64_t*>(pars + 2 * G * CW);  // [W][G]
    unsigned char* mine = smem + (sel_bwd_group_bytes<LN>(W) * G + 15) / 16 * 16 + static_cast<size_t>(w) * sel_bwd_warp_bytes<T, LN>();
    Quad* sd = reinterpret_cast<Quad*>(mine + BC::kRawBytes + BC::kBytes);  // [S][CW]: (s log2 e) twice, (s x) twice
    f32x2* gd = reinterpret_cast<f32x2*>(sd + S * CW);                      // [S][CW]: do twice
    float* ob = reinterpret_cast<float*>(gd + S * CW);                      // [3][S][YS]: o, dv, sum_n A w

    const int64_t b = blockIdx.y;
    const int len = sel_length(a, b), slices = (len + S - 1) / S, n8 = (a.L + 7) / 8;
    const int base = blockIdx.x * G * CW;  // the CTA's first channel
    const int ln = lane % LN, ch = lane / LN, n0 = ln * 4;
    const int row = lane / 4, sub = (lane & 3) * E;  // in memory's layout; lanes past CW channels idle (LN = 16)
    const bool reads = sub < CW, gated = a.z != nullptr;
    const BC bc{static_cast<const T*>(a.B) + b * a.sB[0], static_cast<const T*>(a.C) + b * a.sC[0],
                reinterpret_cast<T*>(mine), reinterpret_cast<float*>(mine + BC::kRawBytes)};
    const bool vec = a.vec != 0;

    for (int g = w; g < G; g += W) As[g * 32 + lane] = quad(read_states(a.A, base + g * CW + ch, a.D, n0, a.N));
    for (int i = threadIdx.x; i < 2 * G * CW; i += W * 32) {
        const float* p = i < G * CW ? a.bias : a.skip;
        const int c = base + i % (G * CW);
        pars[i] = p && c < a.D ? p[c] : 0.f;
    }
    for (int g = 0; g < G; ++g) {
        dAs[(w * G + g) * 32 + lane] = quad(make_float4(0.f, 0.f, 0.f, 0.f));
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) sums[((w * G + g) * 32 + lane) * 2 * E + e] = 0.f;
        if (lane == 0) mbar_init(&bars[w * G + g], 1);
    }
    fence_mbar_init();
    __syncthreads();

    using R = Run<T, E, FULL>;
    R rx, rt, rz, rg;
    Quad hn;  // the checkpoint
    const T *px, *pt, *pz = nullptr, *pg;  // the lane's token and channels of the slice and group asked for next
    const float* pc;
    int nj = slices - 1 - w, ng = 0;       // that slice and group
    auto place = [&] {
        const int64_t t = static_cast<int64_t>(nj) * S + row;
        const int d = base + sub;
        px = static_cast<const T*>(a.x) + b * a.sx[0] + t * a.sx[1] + d;
        pt = static_cast<const T*>(a.dt) + b * a.sdt[0] + t * a.sdt[1] + d;
        if (gated) pz = static_cast<const T*>(a.z) + b * a.sz[0] + t * a.sz[1] + d;
        pg = static_cast<const T*>(a.dy) + b * a.sdy[0] + t * a.sdy[1] + d;
        pc = a.ckpt + ((b * n8 + nj) * a.D + base + ch) * NP + n0;
    };
    auto ask = [&] {
        const int o = ng * CW, d = base + o + sub;
        const bool in = nj * S + row < len && reads;
        rx.read(px + o, in, d, a.D, vec);
        rt.read(pt + o, in, d, a.D, vec);
        if (gated) rz.read(pz + o, in, d, a.D, vec);
        rg.read(pg + o, in, d, a.D, vec);
        hn = FULL || base + o + ch < a.D ? *reinterpret_cast<const Quad*>(pc + static_cast<int64_t>(o) * NP) : quad(make_float4(0.f, 0.f, 0.f, 0.f));
        if (++ng == G) {
            ng = 0;
            nj -= W;
            if (nj >= 0) place();
        }
    };
    bool ok = true;
    uint32_t turn = 0;
    if (nj >= 0) {
        bc.ask(a, nj * S, len, lane);
        place();
        ask();
    }
    for (int k = w; k < slices; k += W, ++turn) {  // k: from the row's end
        const int j = slices - 1 - k, t0 = j * S;
        bc.take(a, t0, len, lane);
        __syncwarp();
        if (j >= W) bc.ask(a, (j - W) * S, len, lane);
        Quad accB[S], accC[S];
#pragma unroll
        for (int t = 0; t < S; ++t) accB[t] = accC[t] = quad(make_float4(0.f, 0.f, 0.f, 0.f));
        const bool in = t0 + row < len && reads;
        const int64_t out = (b * a.L + t0 + row) * a.D + base + sub;

        for (int g = 0; g < G; ++g) {
            const int d = base + g * CW + sub, dc = base + g * CW + ch, wg = w * G + g;
            float xs[E], ss[E], slope[E], dof[E], dzf[E];
            const bool packed = R::packed(d, a.D, vec);
            rx.floats(xs, packed);
            rt.floats(ss, packed);
            rg.floats(dof, packed);
            if (gated) rz.floats(dzf, packed);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float raw = ss[e] + pars[g * CW + (reads ? sub : 0) + e];
                slope[e] = 1.f;
                ss[e] = raw;
                if (a.softplus) ss[e] = softplus(raw, slope[e]);
                ss[e] = in && (FULL || d + e < a.D) ? ss[e] : 0.f;
                if (gated) {
                    const float zv = dzf[e], sg = sigmoid(zv), g0 = dof[e];
                    dof[e] = g0 * (zv * sg);
                    dzf[e] = g0 * silu_slope(zv, sg);
                }
                if (reads) {
                    const float sl = ss[e] * kLog2e, v = ss[e] * xs[e];
                    sd[Sh::place(row, sub + e)] = Quad{pair(sl, sl), pair(v, v)};
                    gd[Sh::place(row, sub + e)] = pair(dof[e], dof[e]);
                }
            }
            Quad h = hn;
            __syncwarp();
            if (g + 1 < G || j >= W) ask();

            const Quad A = As[g * 32 + lane];
            Quad dec[S], old[S];  // e^(s A), and e^(s A) h
            float v[S];
#pragma unroll
            for (int t = 0; t < S; ++t) {
                const Quad q = sd[Sh::place(t, ch)];
                const f32x2 do2 = gd[Sh::place(t, ch)];
                const Quad Bq = bc.b(t, ln), Cq = bc.c(t, ln);
                dec[t].lo = decays(q.lo, A.lo);
                dec[t].hi = decays(q.lo, A.hi);
                old[t].lo = mul2(dec[t].lo, h.lo);
                old[t].hi = mul2(dec[t].hi, h.hi);
                h.lo = fma2(q.hi, Bq.lo, old[t].lo);
                h.hi = fma2(q.hi, Bq.hi, old[t].hi);
                accC[t].lo = fma2(h.lo, do2, accC[t].lo);
                accC[t].hi = fma2(h.hi, do2, accC[t].hi);
                v[t] = both(fma2(Cq.hi, h.hi, mul2(Cq.lo, h.lo)));
            }
            const int first = FoldShape<S, LN / 2, 1>::held(lane);
            constexpr int kept = FoldShape<S, LN / 2, 1>::kRem;
            if (gated) {
                Fold<S, LN / 2, 1>::run(v, lane);
#pragma unroll
                for (int i = 0; i < kept; ++i) ob[(first + i) * YS + ch] = v[i];
            }
            Quad gs = quad(make_float4(0.f, 0.f, 0.f, 0.f)), own = gs, P = gs;
            if constexpr (AHEAD) {
#pragma unroll
                for (int t = S - 1; t >= 0; --t) {
                    const f32x2 do2 = gd[Sh::place(t, ch)];
                    const Quad Cq = bc.c(t, ln);
                    own.lo = mul2(dec[t].lo, t == S - 1 ? mul2(Cq.lo, do2) : fma2(Cq.lo, do2, own.lo));
                    own.hi = mul2(dec[t].hi, t == S - 1 ? mul2(Cq.hi, do2) : fma2(Cq.hi, do2, own.hi));
                    P.lo = t == S - 1 ? dec[t].lo : mul2(P.lo, dec[t].lo);
                    P.hi = t == S - 1 ? dec[t].hi : mul2(P.hi, dec[t].hi);
                }
            }
            auto hand_on = [&](const Quad& q) {
                if (j > 0) {
                    const int next = (w + 1 == W ? 0 : w + 1) * G + g;
                    hop[next * 32 + lane] = q;
                    __syncwarp();
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&bars[next])) : "memory");
                } else if (a.dh0) {
                    write_states(a.dh0 + b * a.D * a.N, dc, a.D, n0, a.N, q);
                }
            };
            if (k > 0) {
                const uint32_t phase = (w == 0 ? turn - 1 : turn) & 1;
                if (ok) ok = mbar_wait(&bars[wg], phase);
                gs = hop[wg * 32 + lane];
            } else if (a.dhN) {
                gs = quad(read_states(a.dhN + b * a.D * a.N, dc, a.D, n0, a.N));
            }
            if constexpr (AHEAD) hand_on(Quad{fma2(P.lo, gs.lo, own.lo), fma2(P.hi, gs.hi, own.hi)});
            Quad dA = dAs[wg * 32 + lane];
            float dv[S], aw[S];
#pragma unroll
            for (int t = S - 1; t >= 0; --t) {
                const Quad q = sd[Sh::place(t, ch)];
                const f32x2 do2 = gd[Sh::place(t, ch)];
                const Quad Bq = bc.b(t, ln), Cq = bc.c(t, ln);
                gs.lo = fma2(Cq.lo, do2, gs.lo);
                gs.hi = fma2(Cq.hi, do2, gs.hi);
                accB[t].lo = fma2(gs.lo, q.hi, accB[t].lo);
                accB[t].hi = fma2(gs.hi, q.hi, accB[t].hi);
                dv[t] = both(fma2(gs.hi, Bq.hi, mul2(gs.lo, Bq.lo)));
                const f32x2 w0 = mul2(gs.lo, old[t].lo), w1 = mul2(gs.hi, old[t].hi);
                aw[t] = both(fma2(w1, A.hi, mul2(w0, A.lo)));
                dA.lo = fma2(w0, q.lo, dA.lo);  // (times log2 e, taken out at the end)
                dA.hi = fma2(w1, q.lo, dA.hi);
                gs.lo = mul2(gs.lo, dec[t].lo);
                gs.hi = mul2(gs.hi, dec[t].hi);
            }
            if constexpr (!AHEAD) hand_on(gs);
            dAs[wg * 32 + lane] = dA;
            Fold<S, LN / 2, 1>::run(dv, lane);
            Fold<S, LN / 2, 1>::run(aw, lane);
#pragma unroll
            for (int i = 0; i < kept; ++i) {
                ob[(S + first + i) * YS + ch] = dv[i];
                ob[(2 * S + first + i) * YS + ch] = aw[i];
            }
            __syncwarp();
            if (t0 + row < a.L && reads) {
                float ox[E], ot[E], oz[E], acc[2 * E];
                get_run<2 * E>(acc, sums + (wg * 32 + lane) * 2 * E);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float sk = pars[(G + g) * CW + sub + e];
                    const float dvv = ob[(S + row) * YS + sub + e];
                    ox[e] = in ? fmaf(dvv, ss[e], dof[e] * sk) : 0.f;
                    ot[e] = in ? fmaf(dvv, xs[e], ob[(2 * S + row) * YS + sub + e]) * slope[e] : 0.f;
                    acc[2 * e] = fmaf(dof[e], xs[e], acc[2 * e]);
                    acc[2 * e + 1] += ot[e];
                    if (gated) oz[e] = in ? dzf[e] * fmaf(sk, xs[e], ob[row * YS + sub + e]) : 0.f;
                }
                put_run<2 * E>(sums + (wg * 32 + lane) * 2 * E, acc);
                write_run<T, E, FULL>(ox, static_cast<T*>(a.dx) + out + g * CW, d, a.D, vec);
                write_run<T, E, FULL>(ot, static_cast<T*>(a.ddt) + out + g * CW, d, a.D, vec);
                if (gated) write_run<T, E, FULL>(oz, static_cast<T*>(a.dz) + out + g * CW, d, a.D, vec);
            }
            __syncwarp();  // ob and sd are written again
        }
        // the slice's sums over the CTA's channels, folded over the lanes of a warp that hold the same states
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float v[S * 4];
#pragma unroll
            for (int t = 0; t < S; ++t) {
                const Quad q = which ? accC[t] : accB[t];
                halves(q.lo, v[4 * t], v[4 * t + 1]);
                halves(q.hi, v[4 * t + 2], v[4 * t + 3]);
            }
            Fold<S * 4, 16, LN>::run(v, lane);
            const int first = FoldShape<S * 4, 16, LN>::held(lane);
            constexpr int kept = FoldShape<S * 4, 16, LN>::kRem;  // at least 2
            float* part = (which ? a.partC : a.partB) + ((static_cast<int64_t>(blockIdx.x) * a.Bn + b) * a.L + t0) * NP + n0;
#pragma unroll
            for (int i = 0; i < kept; i += 2) {
                const int t = (first + i) / 4, n = (first + i) % 4;
                if (t0 + t < len) *reinterpret_cast<float2*>(part + t * NP + n) = make_float2(v[i], v[i + 1]);
            }
        }
    }
    // gradients of what lies behind the row's end
    if (reads) {
        const float nil[E] = {};
        for (int64_t t = static_cast<int64_t>(slices + w) * S + row; t < a.L; t += W * S)
            for (int g = 0; g < G; ++g) {
                const int d = base + g * CW + sub;
                const int64_t o = (b * a.L + t) * a.D + d;
                write_run<T, E, FULL>(nil, static_cast<T*>(a.dx) + o, d, a.D, vec);
                write_run<T, E, FULL>(nil, static_cast<T*>(a.ddt) + o, d, a.D, vec);
                if (gated) write_run<T, E, FULL>(nil, static_cast<T*>(a.dz) + o, d, a.D, vec);
            }
    }
    __syncthreads();
    for (int g = w; g < G; g += W) {
        const int dc = base + g * CW + ch;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < W; ++i) {
            const float4 q = reinterpret_cast<const float4*>(dAs)[(i * G + g) * 32 + lane];
            s.x += q.x, s.y += q.y, s.z += q.z, s.w += q.w;
        }
        if (dc < a.D)
            *reinterpret_cast<float4*>(a.partA + (b * a.D + dc) * NP + n0) =
                make_float4(s.x * kLn2, s.y * kLn2, s.z * kLn2, s.w * kLn2);
        if (slices == 0 && a.dh0) {
            const Quad q = a.dhN ? quad(read_states(a.dhN + b * a.D * a.N, dc, a.D, n0, a.N)) : quad(make_float4(0.f, 0.f, 0.f, 0.f));
            write_states(a.dh0 + b * a.D * a.N, dc, a.D, n0, a.N, q);
        }
    }
    for (int i = threadIdx.x; i < G * CW * 2; i += W * 32) {  // dskip and ddt_bias of a channel
        const int g = i / (2 * CW), c = i / 2 % CW, which = i & 1;
        const int d = base + g * CW + c;
        if (d >= a.D) continue;
        float s = 0.f;
        for (int v = 0; v < W; ++v)
            for (int r = 0; r < S; ++r) s += sums[((v * G + g) * 32 + r * 4 + c / E) * 2 * E + 2 * (c % E) + which];
        a.partS[(b * 2 + which) * a.D + d] = s;
    }
}

// dB and dC: the sums of the CTAs' partial rows, in order
template <typename T>
__global__ void __launch_bounds__(256) sel_reduce_bc_k(const float* __restrict__ partB, const float* __restrict__ partC, int parts,
                                                       SelArgs a, int np, T* dB, T* dC) {
    const int64_t n = a.Bn * a.L * a.N;
    const float* p = blockIdx.y ? partC : partB;
    T* out = blockIdx.y ? dC : dB;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t bt = i / a.N, b = bt / a.L;
        float s = 0.f;
        if (bt - b * a.L < sel_length(a, b)) {
            const float* q = p + bt * np + (i - bt * a.N);
            const int64_t step = a.Bn * a.L * np;
#pragma unroll 4
            for (int k = 0; k < parts; ++k) s += q[k * step];
        }
        out[i] = from_f32<T>(s);
    }
}
// dA (D, N), dskip and ddt_bias (D): sums over the rows, in order
__global__ void __launch_bounds__(256) sel_reduce_params_k(SelArgs a, int np, float* dA, float* dskip, float* dbias) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, n = static_cast<int64_t>(a.D) * a.N;
    if (i < n) {
        const int64_t d = i / a.N;
        float s = 0.f;
        for (int64_t b = 0; b < a.Bn; ++b) s += a.partA[(b * a.D + d) * np + (i - d * a.N)];
        dA[i] = s;
    }
    if (i < 2 * static_cast<int64_t>(a.D)) {
        const int which = i >= a.D;
        float* out = which ? dbias : dskip;
        float s = 0.f;
        for (int64_t b = 0; b < a.Bn; ++b) s += a.partS[b * 2 * a.D + i];
        if (out) out[which ? i - a.D : i] = s;
    }
}

// ---------------------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------------------
// threads a channel: four states each, a power of two
int sel_ln(int64_t N) {
    int ln = 2;
    while (ln * 4 < N) ln *= 2;
    return ln;
}
bool sel_aligned(const void* p, const int64_t* st, int64_t esz) {
    return !p || ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(st[0] * esz) | static_cast<uintptr_t>(st[1] * esz)) & 15u) == 0;
}

int sel_check(const char* fn, const EacsSelective& p, bool single) {
    if (p.rows < 0 || p.L < 0 || p.D < 1 || p.N < 1) return fail(EACS_ERR_INVALID, "%s: bad sizes", fn);
    if (p.dtype != EACS_DTYPE_F32 && p.dtype != EACS_DTYPE_F16 && p.dtype != EACS_DTYPE_BF16)
        return fail(EACS_ERR_INVALID, "%s: unknown dtype %d", fn, p.dtype);
    if (p.N > 64) return fail(EACS_ERR_UNSUPPORTED, "%s: N=%lld > 64", fn, (long long)p.N);
    if (p.rows > 65535 || p.D > (int64_t{1} << 24) || p.L > (int64_t{1} << 30))
        return fail(EACS_ERR_UNSUPPORTED, "%s: more than 65535 rows, 2^24 channels or 2^30 tokens", fn);
    if (p.rows > 0 && (p.L > 0 || single) && (!p.x || !p.dt || !p.A || !p.B || !p.C))
        return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    return EACS_OK;
}

SelArgs sel_args(const EacsSelective& p) {
    SelArgs a{};
    a.x = p.x, a.dt = p.dt, a.z = p.z, a.B = p.B, a.C = p.C;
    for (int i = 0; i < 2; ++i)
        a.sx[i] = p.x_stride[i], a.sdt[i] = p.dt_stride[i], a.sz[i] = p.z_stride[i], a.sB[i] = p.B_stride[i], a.sC[i] = p.C_stride[i];
    a.A = p.A, a.skip = p.skip, a.bias = p.dt_bias, a.lengths = p.lengths, a.h0 = p.initial_state;
    a.L = static_cast<int>(p.L), a.D = static_cast<int>(p.D), a.N = static_cast<int>(p.N), a.Bn = p.rows, a.softplus = p.softplus;
    const int64_t esz = p.dtype == EACS_DTYPE_F32 ? 4 : 2;
    const int64_t dense[2] = {p.D, p.D};  // of what is written
    a.vec = sel_aligned(p.x, p.x_stride, esz) && sel_aligned(p.dt, p.dt_stride, esz) && sel_aligned(p.z, p.z_stride, esz) &&
            ((dense[0] * esz) & 15) == 0;
    a.vec_bc = p.N * esz % 16 == 0 && sel_aligned(p.B, p.B_stride, esz) && sel_aligned(p.C, p.C_stride, esz);
    return a;
}

// A CTA of the twelve warps that a multiprocessor has registers for, so that each ring has all of them: two rounds of 148
// such CTAs took 644 us where rings of six warps, two at once, took 699 (B=4 L=16384 D=1024 N=16: 256 groups of channels).
// Rows of few slices take as many warps as they have slices, and a multiprocessor several CTAs.
template <typename T, int LN, bool CKPT, bool FULL>
cudaError_t sel_fwd_launch(const SelArgs& a, cudaStream_t s) {
    constexpr int CW = FwdShape<LN>::CW, S = FwdShape<LN>::S;
    const dim3 grid((a.D + CW - 1) / CW, static_cast<unsigned>(a.Bn));
    const int slices = (a.L + S - 1) / S;
    const int W = slices >= 12 ? kSelFwdWarps : slices >= 6 ? 6 : slices >= 4 ? 4 : slices;
    const size_t smem = sel_fwd_cta_bytes<LN>(W) + W * sel_fwd_warp_bytes<T, LN>();
    const auto k = sel_fwd_k<T, LN, CKPT, FULL>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    k<<<grid, W * 32, smem, s>>>(a);
    note_launch();
    return cudaGetLastError();
}
template <typename T, int LN>
cudaError_t sel_step_launch(const SelArgs& a, cudaStream_t s) {
    // four rows a thread, with A read once for them, while that leaves four CTAs a multiprocessor
    const int64_t x = (static_cast<int64_t>(a.D) * LN + 255) / 256;
    const dim3 one(static_cast<unsigned>(x), static_cast<unsigned>(a.Bn)), four(static_cast<unsigned>(x), static_cast<unsigned>((a.Bn + 3) / 4));
    if (x * ((a.Bn + 3) / 4) >= 148 * 4) sel_step_k<T, LN, 4><<<four, 256, 0, s>>>(a);
    else sel_step_k<T, LN, 1><<<one, 256, 0, s>>>(a);
    note_launch();
    return cudaGetLastError();
}

// Groups of channels that a backward's CTA takes: as many as leave the fewest rounds of CTAs (one a multiprocessor) times
// groups; of equals the most, for fewer partial rows.  Neither the partial rows (8 bytes a padded state, token and CTA of a
// row) nor whether the groups divide D (else every CTA takes the kernel with bounds checks, about 10 percent) is weighed:
// B=8 L=8192 N=16 training steps take 1908 us for D=768 (6 groups, 134 MB of partial rows), 3188 for 1024 (1, 1074 MB),
// 4915 for 1536 (1, 1611 MB) and 4755 for 2048 (7, not dividing, 310 MB).
template <int LN>
int sel_bwd_groups(int64_t rows, int64_t D) {
    constexpr int CW = BwdShape<LN>::CW;
    const int64_t n = (D + CW - 1) / CW;
    int best = 1;
    int64_t cost = INT64_MAX;
    for (int g = 1; g <= kSelBwdMaxGroups && g <= n; ++g) {
        const int64_t ctas = rows * ((n + g - 1) / g), c = (ctas + 147) / 148 * g;
        if (c <= cost) cost = c, best = g;
    }
    return best;
}
int sel_bwd_parts(int64_t rows, int64_t D, int ln, int* groups) {
    const int g = ln == 2 ? sel_bwd_groups<2>(rows, D) : ln == 4 ? sel_bwd_groups<4>(rows, D)
                : ln == 8 ? sel_bwd_groups<8>(rows, D) : sel_bwd_groups<16>(rows, D);
    if (groups) *groups = g;
    const int64_t per = static_cast<int64_t>(g) * (32 / ln);
    return static_cast<int>((D + per - 1) / per);
}
template <typename T, int LN>
cudaError_t sel_bwd_launch(const SelArgs& a, int parts, T* dB, T* dC, float* dA, float* dskip, float* dbias, cudaStream_t s) {
    constexpr int W = kSelBwdWarps;
    const size_t smem = (sel_bwd_group_bytes<LN>(W) * a.groups + 15) / 16 * 16 + W * sel_bwd_warp_bytes<T, LN>();
    // (a group of channels may start past D only where they are not FULL)
    const bool full = a.vec && a.vec_bc && a.N == 4 * LN && a.D % (a.groups * BwdShape<LN>::CW) == 0;
    const bool ahead = a.groups == 1;
    const auto k = full ? (ahead ? sel_bwd_k<T, LN, true, true> : sel_bwd_k<T, LN, true, false>)
                        : (ahead ? sel_bwd_k<T, LN, false, true> : sel_bwd_k<T, LN, false, false>);
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    k<<<dim3(parts, static_cast<unsigned>(a.Bn)), W * 32, smem, s>>>(a);
    note_launch();
    const int64_t n = a.Bn * a.L * a.N;
    sel_reduce_bc_k<T><<<dim3(static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, 148 * 16)), 2), 256, 0, s>>>(
        a.partB, a.partC, parts, a, 4 * LN, dB, dC);
    note_launch();
    const int64_t m = std::max<int64_t>(static_cast<int64_t>(a.D) * a.N, 2 * static_cast<int64_t>(a.D));
    sel_reduce_params_k<<<static_cast<unsigned>((m + 255) / 256), 256, 0, s>>>(a, 4 * LN, dA, dskip, dbias);
    note_launch();
    return cudaGetLastError();
}

// f<T, LN>() for the call's type and threads a channel
#define EACS_SEL_LN(T, F, ...)                       \
    (ln == 2   ? F<T, 2>(__VA_ARGS__)                \
     : ln == 4 ? F<T, 4>(__VA_ARGS__)                \
     : ln == 8 ? F<T, 8>(__VA_ARGS__)                \
               : F<T, 16>(__VA_ARGS__))

template <typename T, int LN>
cudaError_t sel_fwd_any(const SelArgs& a, cudaStream_t s) {
    const bool full = a.vec && a.vec_bc && a.D % FwdShape<LN>::CW == 0 && a.N == 4 * LN;
    if (a.ckpt) return full ? sel_fwd_launch<T, LN, true, true>(a, s) : sel_fwd_launch<T, LN, true, false>(a, s);
    return full ? sel_fwd_launch<T, LN, false, true>(a, s) : sel_fwd_launch<T, LN, false, false>(a, s);
}

size_t sel_up(size_t n) { return (n + 255) / 256 * 256; }
struct SelBwdLayout {
    size_t B, C, A, S, total;
};
SelBwdLayout sel_bwd_layout(const EacsSelective& p, int parts) {
    const size_t np = 4 * static_cast<size_t>(sel_ln(p.N));
    const size_t bc = sel_up(static_cast<size_t>(parts) * p.rows * p.L * np * 4);
    SelBwdLayout l{};
    l.C = bc;
    l.A = 2 * bc;
    l.S = l.A + sel_up(static_cast<size_t>(p.rows) * p.D * np * 4);
    l.total = l.S + sel_up(static_cast<size_t>(p.rows) * 2 * p.D * 4);
    return l;
}

}  // namespace

size_t selective_ckpt_size(const EacsSelective& p) {
    if (sel_check("eacs_selective_ckpt_size", p, false) != EACS_OK) return 0;
    return static_cast<size_t>(p.rows) * ((p.L + 7) / 8) * p.D * 4 * sel_ln(p.N) * 4;
}

size_t selective_bwd_workspace_size(const EacsSelective& p) {
    if (sel_check("eacs_selective_bwd_workspace_size", p, false) != EACS_OK || p.rows == 0) return 0;
    return sel_bwd_layout(p, sel_bwd_parts(p.rows, p.D, sel_ln(p.N), nullptr)).total;
}

int selective_fwd(const EacsSelective& p, void* y, float* final_state, void* ckpt, size_t ckpt_bytes, cudaStream_t stream) {
    const char* fn = "eacs_selective_fwd";
    if (const int rc = sel_check(fn, p, false)) return rc;
    if (p.rows == 0 || p.L == 0) {  // the state stays
        if (!final_state || p.rows == 0) return EACS_OK;
        const size_t n = static_cast<size_t>(p.rows) * p.D * p.N * 4;
        if (!p.initial_state) return cuda_check(cudaMemsetAsync(final_state, 0, n, stream), fn);
        if (p.initial_state == final_state) return EACS_OK;
        return cuda_check(cudaMemcpyAsync(final_state, p.initial_state, n, cudaMemcpyDeviceToDevice, stream), fn);
    }
    if (!y) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    if (ckpt && ckpt_bytes < selective_ckpt_size(p))
        return fail(EACS_ERR_WORKSPACE, "%s: checkpoints of %zu bytes, %zu needed", fn, ckpt_bytes, selective_ckpt_size(p));
    if (reinterpret_cast<uintptr_t>(ckpt) & 15u) return fail(EACS_ERR_INVALID, "%s: checkpoints are not on 16 bytes", fn);
    SelArgs a = sel_args(p);
    a.y = y;
    a.vec = a.vec && (reinterpret_cast<uintptr_t>(y) & 15u) == 0;
    a.hN = final_state;
    a.ckpt = static_cast<float*>(ckpt);
    const int ln = sel_ln(p.N);
    const cudaError_t e = p.dtype == EACS_DTYPE_F32   ? EACS_SEL_LN(float, sel_fwd_any, a, stream)
                          : p.dtype == EACS_DTYPE_F16 ? EACS_SEL_LN(__half, sel_fwd_any, a, stream)
                                                      : EACS_SEL_LN(__nv_bfloat16, sel_fwd_any, a, stream);
    return cuda_check(e, fn);
}

int selective_step(const EacsSelective& p, void* y, float* state, cudaStream_t stream) {
    const char* fn = "eacs_selective_step";
    if (const int rc = sel_check(fn, p, true)) return rc;
    if (p.rows == 0) return EACS_OK;
    if (!y || !state) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    SelArgs a = sel_args(p);
    a.y = y;
    a.hN = state;
    a.vec = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15u) == 0;
    const int ln = sel_ln(p.N);
    const cudaError_t e = p.dtype == EACS_DTYPE_F32   ? EACS_SEL_LN(float, sel_step_launch, a, stream)
                          : p.dtype == EACS_DTYPE_F16 ? EACS_SEL_LN(__half, sel_step_launch, a, stream)
                                                      : EACS_SEL_LN(__nv_bfloat16, sel_step_launch, a, stream);
    return cuda_check(e, fn);
}

int selective_bwd(const EacsSelective& p, const SelectiveGrads& g, const void* ckpt, size_t ckpt_bytes, void* ws, size_t ws_bytes,
                  cudaStream_t stream) {
    const char* fn = "eacs_selective_bwd";
    if (const int rc = sel_check(fn, p, false)) return rc;
    const bool empty = p.rows == 0 || p.L == 0;
    if (!empty && (!g.dy || !g.dx || !g.ddt || (p.z && !g.dz) || !g.dB || !g.dC || !g.dA))
        return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    if (empty) {  // empty sums; the final state is the initial one
        cudaError_t e = cudaSuccess;
        if (g.dA) e = cudaMemsetAsync(g.dA, 0, static_cast<size_t>(p.D) * p.N * 4, stream);
        if (e == cudaSuccess && g.dskip) e = cudaMemsetAsync(g.dskip, 0, static_cast<size_t>(p.D) * 4, stream);
        if (e == cudaSuccess && g.ddt_bias) e = cudaMemsetAsync(g.ddt_bias, 0, static_cast<size_t>(p.D) * 4, stream);
        const size_t n = static_cast<size_t>(p.rows) * p.D * p.N * 4;
        if (e == cudaSuccess && g.dinitial && n)
            e = g.dfinal ? cudaMemcpyAsync(g.dinitial, g.dfinal, n, cudaMemcpyDeviceToDevice, stream)
                         : cudaMemsetAsync(g.dinitial, 0, n, stream);
        return cuda_check(e, fn);
    }
    if (!ckpt || ckpt_bytes < selective_ckpt_size(p))
        return fail(EACS_ERR_WORKSPACE, "%s: checkpoints of %zu bytes, %zu needed", fn, ckpt_bytes, selective_ckpt_size(p));
    if (!ws || ws_bytes < selective_bwd_workspace_size(p))
        return fail(EACS_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, selective_bwd_workspace_size(p));
    if ((reinterpret_cast<uintptr_t>(ckpt) | reinterpret_cast<uintptr_t>(ws)) & 15u)
        return fail(EACS_ERR_INVALID, "%s: checkpoints or workspace are not on 16 bytes", fn);
    SelArgs a = sel_args(p);
    const int64_t esz = p.dtype == EACS_DTYPE_F32 ? 4 : 2;
    a.dy = g.dy;
    a.sdy[0] = g.dy_stride[0], a.sdy[1] = g.dy_stride[1];
    a.vec = a.vec && sel_aligned(g.dy, g.dy_stride, esz) &&
            ((reinterpret_cast<uintptr_t>(g.dx) | reinterpret_cast<uintptr_t>(g.ddt) | reinterpret_cast<uintptr_t>(p.z ? g.dz : nullptr)) & 15u) == 0;
    a.dhN = g.dfinal;
    a.dh0 = g.dinitial;
    a.dx = g.dx, a.ddt = g.ddt, a.dz = g.dz;
    a.ckpt = static_cast<float*>(const_cast<void*>(ckpt));
    const int ln = sel_ln(p.N);
    const int parts = sel_bwd_parts(p.rows, p.D, ln, &a.groups);
    const SelBwdLayout l = sel_bwd_layout(p, parts);
    char* w = static_cast<char*>(ws);
    a.partB = reinterpret_cast<float*>(w + l.B), a.partC = reinterpret_cast<float*>(w + l.C);
    a.partA = reinterpret_cast<float*>(w + l.A), a.partS = reinterpret_cast<float*>(w + l.S);
    cudaError_t e;
    if (p.dtype == EACS_DTYPE_F32) {
        float *dB = static_cast<float*>(g.dB), *dC = static_cast<float*>(g.dC);
        e = EACS_SEL_LN(float, sel_bwd_launch, a, parts, dB, dC, g.dA, g.dskip, g.ddt_bias, stream);
    } else if (p.dtype == EACS_DTYPE_F16) {
        __half *dB = static_cast<__half*>(g.dB), *dC = static_cast<__half*>(g.dC);
        e = EACS_SEL_LN(__half, sel_bwd_launch, a, parts, dB, dC, g.dA, g.dskip, g.ddt_bias, stream);
    } else {
        __nv_bfloat16 *dB = static_cast<__nv_bfloat16*>(g.dB), *dC = static_cast<__nv_bfloat16*>(g.dC);
        e = EACS_SEL_LN(__nv_bfloat16, sel_bwd_launch, a, parts, dB, dC, g.dA, g.dskip, g.ddt_bias, stream);
    }
    return cuda_check(e, fn);
}

cudaError_t selective_read_status(int* out, cudaStream_t stream) { return read_clear_status(out, stream); }

}  // namespace eacs
