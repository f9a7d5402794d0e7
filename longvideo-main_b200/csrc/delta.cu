// delta.cu -- the gated delta rule: chunked forward and backward, single steps (sm_100a).
//
// A head keeps a state S (K x V, float32).  One token with decay e^g, rate
// beta, key k, value v and query q does
//   S' = e^g S,  u = beta (v - S'^T k),  S = S' + k u^T,  o = scale S^T q.
//
// Sequences are taken 64 tokens (one chunk) at a time.  With G the running sum
// of g inside the chunk, gam = e^G, Gam_ij = e^(G_i - G_j), d_j = e^(G_63 - G_j)
// and S0 the state before the chunk, the 64 rank-one updates become products of
// matrices:
//   A_ij = beta_i Gam_ij k_i.k_j (j < i),   T' = (I + A)^-1 diag(beta)
//   U = T' (V - gam K S0),   S1 = gam_63 S0 + K^T diag(d) U
//   O = scale gam Q S0 + M U,   M_ij = scale Gam_ij q_i.k_j (j <= i)
// and for upstream gradients dO and dS1:
//   dU = M^T dO + d K dS1,   dV = T'^T dU
//   dS0 = gam_63 dS1 + Q^T (scale gam dO) - K^T (gam dV)
//   N_ij = scale Gam_ij dO_i.U_j (j <= i),   E_ij = -Gam_ij dV_i.U_j (j < i)
//   dQ = scale gam dO S0^T + N K
//   dK = [-gam dV S0^T + E K] + [d U dS1^T + N^T Q + E^T K] = dK_read + dK_write
//   dbeta_i = (dV_i / beta_i).(U_i / beta_i)
//   dG_i = q_i.dQ_i + k_i.(dK_read - dK_write)_i,
//   dg_i = sum_{j >= i} dG_j + <S1, dS1>
// (a decay reaches every product between a token at or behind it that reads
// and one before it that wrote; for a backward beta is held 2^-64 away from 0 so
// that it can be divided out).  Gam is formed from a sum of g kept in two floats, so that
// a decay of 0 in a chunk takes nothing from the precision behind it.
//
// Only S and dS go from chunk to chunk.  The kernels:
//   delta_prep_k     per chunk: gam, d, T' (and M for a backward)
//   delta_chain_k    the chunks of a head in order: U and S
//   delta_out_k      per chunk: O
//   delta_rchain_k   the chunks in reverse order: dV and dS
//   delta_grad_k     per chunk: dQ, dK, dbeta, dg
//   delta_step_k     a token at a time, for one token or a few
// The two chains are the serial part.  There a warp owns 16 value columns of
// one head's state and keeps S^T (16 x K) as matrix accumulators in registers:
// an accumulator tile of one product is, as it lies, the A operand of the
// next, so U^T = (V^T - gam S^T K^T) T'^T and S^T += U^T K run without a
// shuffle or a barrier between them.
//
// These kernels take float32 inputs, and 16-bit ones that delta_planes.cu does
// not (rows that do not start on 16 bytes, expanded dimensions); delta_grad_k
// takes float16 from there too.  Operands are tf32 split in two (22 bits), three
// products each: errors are 3e-7 to 5e-7 of the norm.  Times at B=4 L=9498 H=10 K=128 V=64, float32: delta_prep_k 248 us,
// delta_chain_k 1650, delta_out_k 662, delta_rchain_k 2980, delta_grad_k 1594.
// The chains are bound by a chunk's dependent products on one warp of each
// scheduler (11 and 20 us a chunk), the others by the products and the
// splitting of every tile as it is read.
#include <algorithm>
#include <initializer_list>

#include "delta_common.cuh"

namespace eacs {
namespace {

// acc += A B with B a tile of inputs / of results
template <class F, int P, bool TR>
__device__ __forceinline__ void mm_in(float* c0, float* c1, const typename F::template Af<P>& a,
                                      const typename F::E* s, int ld, int n0, int k0) {
    F::template mma2<P, TR, true>(c0, c1, a, s, ld, n0, k0);
}
template <class F, int P, bool TR>
__device__ __forceinline__ void mm(float* c0, float* c1, const typename F::template Af<P>& a,
                                   const typename F::E* s, int ld, int n0, int k0) {
    F::template mma2<P, TR>(c0, c1, a, s, ld, n0, k0);
}

// 64 rows of an input (row stride st, `rows` of them in the sequence, `cols`
// columns that exist) into shared memory as [row][colp]; the rest is 0 and is
// not read.  Aligned float32 rows are copied asynchronously (the caller commits
// and waits).
template <class F, typename T>
__device__ __forceinline__ void load_rows(typename F::E* dst, int ld, const T* src, int64_t st, int rows, int cols,
                                          int colp, bool vec, int tid, int nthr) {
    const int groups = colp >> 3;
    for (int i = tid; i < kC * groups; i += nthr) {
        const int r = i / groups, c = (i - r * groups) << 3;
        const bool in = r < rows && c < cols;
        const T* p = src + r * st + c;
        typename F::E* o = dst + r * ld + c;
        if constexpr (sizeof(T) == sizeof(float)) {
            if (vec) {
                cp_async16(o, in ? p : src, in);
                cp_async16(o + 4, in ? p + 4 : src, in);
                continue;
            }
        }
        float v[8];
        if (in && vec) {
            load8<T>(p, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = in && c + e < cols ? to_f32(p[e]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = F::put(v[e]);
    }
}
// `rows` rows of `cols` workspace elements (dense rows of `st`) into shared memory
template <typename E>
__device__ __forceinline__ void load_ws(E* dst, int ld, const E* src, int64_t st, int rows, int cols, int tid, int nthr) {
    constexpr int V = 16 / sizeof(E);
    const int groups = cols / V;
    for (int i = tid; i < rows * groups; i += nthr) {
        const int r = i / groups, c = (i - r * groups) * V;
        cp_async16(dst + r * ld + c, src + r * st + c, true);
    }
}

// ----------------------------------------------------------------------------
// gam, d and T' of a chunk
// ----------------------------------------------------------------------------
template <class F, typename T, int KD>
__global__ void __launch_bounds__(128) delta_prep_k(DArgs a) {
    using E = typename F::E;
    const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int len = row_length(a, b);
    if (c * kC >= len) return;
    const int rows = min(kC, len - c * kC);
    const int hk = h / (a.Hv / a.Hk);
    const int64_t id = (static_cast<int64_t>(b) * a.Hv + h) * a.n + c;
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int LD = KD + 8;
    E* sK = reinterpret_cast<E*>(smem);
    float* sA = reinterpret_cast<float*>(sK + kC * LD);  // [64][64]
    float* sG = sA + kC * kC;                            // G high, low
    float* sB = sG + 2 * kC;
    const int tid = threadIdx.x, warp = tid >> 5;
    const Lane L;
    load_rows<F, T>(sK, LD, static_cast<const T*>(a.k) + b * a.sk.b + static_cast<int64_t>(c) * kC * a.sk.t + hk * a.sk.h,
                    a.sk.t, rows, a.K, KD, a.vec_qk, tid, 128);
    cp_async_commit();
    if (warp == 0) {
        const int64_t t0 = static_cast<int64_t>(c) * kC;
        double s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * L.l + i;
            float gv = 0.f, bv = 0.f;
            if (r < rows) {
                gv = gate_value(a.g, a.gate_dtype, b * a.sg.b + (t0 + r) * a.sg.t + h * a.sg.h);
                bv = gate_value(a.beta, a.gate_dtype, b * a.sb.b + (t0 + r) * a.sb.t + h * a.sb.h);
                if (a.M) bv = hold_beta(bv);  // a backward divides by it
                gv = gv < -200.f ? -200.f : gv;  // e^-200 is 0 in float32
            }
            s[i] = gv;
            sB[r] = bv;
        }
        s[1] += s[0];
        double run = s[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, run, o);
            if (L.l >= o) run += up;
        }
        const double before = run - s[1];
        const double total = __shfl_sync(0xffffffffu, run, 31);
        float* ga = a.gates + id * kGates;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * L.l + i;
            const double G = before + s[i];
            const float hi = static_cast<float>(G), lo = static_cast<float>(G - hi);
            sG[r] = hi;
            sG[kC + r] = lo;
            ga[r] = hi;
            ga[kC + r] = lo;
            ga[2 * kC + r] = expf(static_cast<float>(G));
            ga[3 * kC + r] = expf(static_cast<float>(total - G));
            ga[4 * kC + r] = a.scale * expf(static_cast<float>(G));
        }
    }
    cp_async_wait_all();
    __syncthreads();
    {  // A: a warp 16 rows
        float acc[kC / 8][4] = {};
        const int m0 = warp * 16;
#pragma unroll
        for (int k0 = 0; k0 < KD; k0 += 16) {
            const auto af = F::from_smem(sK, LD, m0, k0);
#pragma unroll
            for (int p = 0; p < kC / 16; ++p)
                if (p <= warp) mm_in<F, 1, false>(acc[2 * p], acc[2 * p + 1], af, sK, LD, 16 * p, k0);
        }
#pragma unroll
        for (int j = 0; j < kC / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = m0 + L.g + (e >> 1) * 8, col = 8 * j + 2 * L.t + (e & 1);
                float v = 0.f;
                if (col < r) v = sB[r] * expf((sG[r] - sG[col]) + (sG[kC + r] - sG[kC + col])) * acc[j][e];
                sA[r * kC + col] = v;
            }
    }
    __syncthreads();
    if (tid < kC) {  // column tid of (I + A)^-1 by forward substitution, in float32
        float x[kC];
#pragma unroll
        for (int i = 0; i < kC; ++i) {
            float s0 = i == tid ? 1.f : 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
            for (int m = 0; m < (i & ~3); m += 4) {
                const float4 r = *reinterpret_cast<const float4*>(sA + i * kC + m);
                s0 = fmaf(-r.x, x[m], s0);
                s1 = fmaf(-r.y, x[m + 1], s1);
                s2 = fmaf(-r.z, x[m + 2], s2);
                s3 = fmaf(-r.w, x[m + 3], s3);
            }
#pragma unroll
            for (int m = i & ~3; m < i; ++m) s0 = fmaf(-sA[i * kC + m], x[m], s0);
            x[i] = (s0 + s1) + (s2 + s3);
        }
        const float bj = sB[tid];
        E* t = static_cast<E*>(a.T) + id * kC * kC;
#pragma unroll
        for (int i = 0; i < kC; ++i) t[i * kC + tid] = x[i] * bj;
    }
}

// ----------------------------------------------------------------------------
// the forward chain
// ----------------------------------------------------------------------------
template <class F, int KD, int W>
struct ChainStage {
    using E = typename F::E;
    static constexpr int LDK = KD + 8, LDV = 16 * W + 8;
    static constexpr int kK = 0;
    static constexpr int kT = kK + kC * LDK;
    static constexpr int kV = kT + kC * kTld;
    static constexpr int kEnd = kV + kC * LDV;
    static constexpr size_t bytes = kEnd * sizeof(E) + 2 * kC * sizeof(float);
};

template <class F, typename T, int KD, int W>
__device__ __forceinline__ void chain_load(const DArgs& a, unsigned char* st, int c, int b, int h, int hk, int len,
                                           int v0, int nthr) {
    using S = ChainStage<F, KD, W>;
    using E = typename F::E;
    E* e = reinterpret_cast<E*>(st);
    float* ga = reinterpret_cast<float*>(e + S::kEnd);
    const int64_t id = (static_cast<int64_t>(b) * a.Hv + h) * a.n + c;
    const int64_t t0 = static_cast<int64_t>(c) * kC;
    const int rows = min(kC, len - c * kC), tid = threadIdx.x;
    load_rows<F, T>(e + S::kK, S::LDK, static_cast<const T*>(a.k) + b * a.sk.b + t0 * a.sk.t + hk * a.sk.h, a.sk.t, rows,
                    a.K, KD, a.vec_qk, tid, nthr);
    load_rows<F, T>(e + S::kV, S::LDV, static_cast<const T*>(a.v) + b * a.sv.b + t0 * a.sv.t + h * a.sv.h + v0, a.sv.t,
                    rows, a.V - v0, 16 * W, a.vec_v, tid, nthr);
    load_ws(e + S::kT, kTld, static_cast<const E*>(a.T) + id * kC * kC, kC, kC, kC, tid,
            nthr);
    load_ws(ga, 2 * kC, a.gates + id * kGates + 2 * kC, 2 * kC, 1, 2 * kC, tid, nthr);
}

// accumulators into a dense [row][ld] workspace tile, rows r0.., as pairs
__device__ __forceinline__ void put2(float* p, float x, float y) { *reinterpret_cast<float2*>(p) = make_float2(x, y); }

template <typename E, int NT>
__device__ __forceinline__ void acc_store(const float (*x)[4], E* p, int ld, const Lane& L) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        put2(p + static_cast<int64_t>(L.g) * ld + 8 * j + 2 * L.t, x[j][0], x[j][1]);
        put2(p + static_cast<int64_t>(L.g + 8) * ld + 8 * j + 2 * L.t, x[j][2], x[j][3]);
    }
}
// the transpose of a (16 x 64) accumulator into a [64][ld] workspace tile at column v0
template <class F>
__device__ __forceinline__ void acc_store_t(const float (*x)[4], typename F::E* p, int ld, int v0, const Lane& L) {
#pragma unroll
    for (int j = 0; j < kC / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            p[static_cast<int64_t>(8 * j + 2 * L.t + (e & 1)) * ld + v0 + L.g + (e >> 1) * 8] = F::put(x[j][e]);
}

// Accumulators that a loop takes two tiles at a time go through shared memory,
// each lane's own: with every tile in registers the loops over the summed index
// would have to be unrolled, and a chunk's instructions (70 KB and more) would
// be fetched anew for every chunk.
template <int NT>
__device__ __forceinline__ void lane_put(float4* s, const float (*x)[4]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) s[j * 32] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
}
__device__ __forceinline__ void lane_get(float* x, const float4* s) {
    const float4 v = *s;
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
}
template <int KD, int W> constexpr size_t kLaneBytes = size_t(W) * 16 * KD * sizeof(float);

// W warps, 16 value columns each.
template <class F, typename T, int KD, int W>
__global__ void __launch_bounds__(W * 32) delta_chain_k(DArgs a) {
    using E = typename F::E;
    using St = ChainStage<F, KD, W>;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / (a.Hv / a.Hk);
    const int len = row_length(a, b), nc = (len + kC - 1) / kC;
    const int warp = threadIdx.x >> 5, vb = blockIdx.x * 16 * W, v0 = vb + warp * 16;
    const Lane L;
    extern __shared__ __align__(16) unsigned char smem[];
    const int64_t head = static_cast<int64_t>(b) * a.Hv + h;
    float S[KD / 8][4];
    state_load<KD>(S, a.initial ? a.initial + head * a.K * a.V : nullptr, a.K, a.V, v0, L);
    const bool on = v0 < a.Vp;
    float4* mine = reinterpret_cast<float4*>(smem + 2 * St::bytes) + warp * 4 * KD + L.l;
    if (nc > 0) chain_load<F, T, KD, W>(a, smem, 0, b, h, hk, len, vb, W * 32);
    cp_async_commit();
    for (int c = 0; c < nc; ++c) {
        unsigned char* st = smem + (c & 1) * St::bytes;
        if (c + 1 < nc) chain_load<F, T, KD, W>(a, smem + ((c + 1) & 1) * St::bytes, c + 1, b, h, hk, len, vb, W * 32);
        cp_async_commit();
        cp_async_wait_group<1>();
        __syncthreads();
        if (on) {
            const E* sK = reinterpret_cast<const E*>(st) + St::kK;
            const E* sT = reinterpret_cast<const E*>(st) + St::kT;
            const E* sV = reinterpret_cast<const E*>(st) + St::kV;
            const float* gam = reinterpret_cast<const float*>(reinterpret_cast<const E*>(st) + St::kEnd);
            const float* dec = gam + kC;
            const int64_t id = head * a.n + c;
            if (a.S) acc_store<E, KD / 8>(S, static_cast<E*>(a.S) + (id * a.Vp + v0) * KD, KD, L);
            // P = (K S0)^T, then X = V^T - gam P in its place
            float X[kC / 8][4] = {};
            lane_put<KD / 8>(mine, S);
#pragma unroll 1
            for (int k0 = 0; k0 < KD; k0 += 16) {
                float x0[4], x1[4];
                lane_get(x0, mine + k0 * 4);
                lane_get(x1, mine + k0 * 4 + 32);
                const auto af = F::template from_acc<2>(x0, x1);
#pragma unroll
                for (int p = 0; p < kC / 16; ++p)
                    mm_in<F, 2, false>(X[2 * p], X[2 * p + 1], af, sK, St::LDK, 16 * p, k0);
            }
#pragma unroll
            for (int p = 0; p < kC / 16; ++p) {
                float x0[4], x1[4];
                F::load_t(x0, x1, sV, St::LDV, warp * 16, 16 * p);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    X[2 * p][e] = x0[e] - gam[16 * p + 2 * L.t + (e & 1)] * X[2 * p][e];
                    X[2 * p + 1][e] = x1[e] - gam[16 * p + 8 + 2 * L.t + (e & 1)] * X[2 * p + 1][e];
                }
            }
            lane_put<kC / 8>(mine, X);
            float U[kC / 8][4] = {};
#pragma unroll 1
            for (int kk = 0; kk < kC / 16; ++kk) {
                float x0[4], x1[4];
                lane_get(x0, mine + kk * 64);
                lane_get(x1, mine + kk * 64 + 32);
                const auto af = F::template from_acc<2>(x0, x1);
#pragma unroll
                for (int p = 0; p < kC / 16; ++p)
                    if (p >= kk) mm<F, 2, false>(U[2 * p], U[2 * p + 1], af, sT, kTld, 16 * p, 16 * kk);
            }
            lane_put<kC / 8>(mine, U);
            acc_store_t<F>(U, static_cast<E*>(a.U) + id * kC * a.Vp, a.Vp, v0, L);
            const float gc = gam[kC - 1];
#pragma unroll
            for (int j = 0; j < KD / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[j][e] *= gc;
#pragma unroll 1
            for (int kk = 0; kk < kC / 16; ++kk) {
                float y0[4], y1[4];
                lane_get(y0, mine + kk * 64);
                lane_get(y1, mine + kk * 64 + 32);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y0[e] *= dec[16 * kk + 2 * L.t + (e & 1)];
                    y1[e] *= dec[16 * kk + 8 + 2 * L.t + (e & 1)];
                }
                const auto af = F::template from_acc<2>(y0, y1);
#pragma unroll
                for (int p = 0; p < KD / 16; ++p)
                    mm_in<F, 2, true>(S[2 * p], S[2 * p + 1], af, sK, St::LDK, 16 * p, 16 * kk);
            }
        }
        __syncthreads();
    }
    if (on && a.final_state) state_store<KD>(S, a.final_state + head * a.K * a.V, a.K, a.V, v0, L);
}

// ----------------------------------------------------------------------------
// O of a chunk
// ----------------------------------------------------------------------------
constexpr int kOutV = 64;  // value columns of one pass

template <class F, int KD>
struct OutSmem {
    using E = typename F::E;
    static constexpr int LDK = KD + 8, LDU = kOutV + 8;
    static constexpr int kQ = 0, kK = kQ + kC * LDK, kS = kK + kC * LDK, kU = kS + kOutV * LDK;
    static constexpr int kEnd = kU + kC * LDU;
    static constexpr size_t bytes = kEnd * sizeof(E) + 3 * kC * sizeof(float);
};

template <typename T> __device__ __forceinline__ void out_store(T* p, float x, float y, bool second, bool pair);
template <> __device__ __forceinline__ void out_store<float>(float* p, float x, float y, bool second, bool pair) {
    if (pair) { *reinterpret_cast<float2*>(p) = make_float2(x, y); return; }
    p[0] = x;
    if (second) p[1] = y;
}
template <> __device__ __forceinline__ void out_store<__half>(__half* p, float x, float y, bool second, bool pair) {
    if (pair) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y); return; }
    p[0] = __float2half_rn(x);
    if (second) p[1] = __float2half_rn(y);
}
template <> __device__ __forceinline__ void out_store<__nv_bfloat16>(__nv_bfloat16* p, float x, float y, bool second,
                                                                     bool pair) {
    if (pair) { *reinterpret_cast<uint32_t*>(p) = pack_bf16(x, y); return; }
    p[0] = __float2bfloat16_rn(x);
    if (second) p[1] = __float2bfloat16_rn(y);
}

// rows [m0, m0+16) x columns of accumulators into a dense output of row stride
// `st` (rows at or behind `rows` get zeros, rows behind `all` do not exist)
template <typename T, int NT>
__device__ __forceinline__ void rows_store(const float (*x)[4], T* p, int64_t st, int m0, int rows, int all, int c0,
                                           int cols, const Lane& L) {
    const bool even = (cols & 1) == 0;  // then every row start and pair is aligned to a pair
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = m0 + L.g + 8 * half, col = c0 + 8 * j + 2 * L.t;
            if (r < all && col < cols) {
                const bool in = r < rows;
                out_store<T>(p + r * st + col, in ? x[j][2 * half] : 0.f, in ? x[j][2 * half + 1] : 0.f, col + 1 < cols,
                             even);
            }
        }
}

template <class F, typename T, int KD>
__global__ void __launch_bounds__(128) delta_out_k(DArgs a) {
    using E = typename F::E;
    using Sm = OutSmem<F, KD>;
    const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / (a.Hv / a.Hk);
    const int len = row_length(a, b);
    const int all = min(kC, a.L - c * kC), rows = min(kC, len - c * kC);
    const int64_t t0 = static_cast<int64_t>(c) * kC, ost = static_cast<int64_t>(a.Hv) * a.V;
    T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.L + t0) * ost + static_cast<int64_t>(h) * a.V;
    const int tid = threadIdx.x, warp = tid >> 5, m0 = warp * 16;
    const Lane L;
    if (rows <= 0) {  // behind the sequence
        for (int i = tid; i < all * a.V; i += 128) out[(i / a.V) * ost + i % a.V] = T(0.f);
        return;
    }
    extern __shared__ __align__(16) unsigned char smem[];
    E* s = reinterpret_cast<E*>(smem);
    float* ga = reinterpret_cast<float*>(s + Sm::kEnd);  // G high, low, gam
    const int64_t id = (static_cast<int64_t>(b) * a.Hv + h) * a.n + c;
    load_rows<F, T>(s + Sm::kQ, Sm::LDK, static_cast<const T*>(a.q) + b * a.sq.b + t0 * a.sq.t + hk * a.sq.h, a.sq.t, rows,
                    a.K, KD, a.vec_qk, tid, 128);
    load_rows<F, T>(s + Sm::kK, Sm::LDK, static_cast<const T*>(a.k) + b * a.sk.b + t0 * a.sk.t + hk * a.sk.h, a.sk.t, rows,
                    a.K, KD, a.vec_qk, tid, 128);
    load_ws(ga, 3 * kC, a.gates + id * kGates, 3 * kC, 1, 3 * kC, tid, 128);
    float Mx[kC / 8][4];
    for (int v0 = 0; v0 < a.Vp; v0 += kOutV) {
        const int vn = min(kOutV, a.Vp - v0);
        load_ws(s + Sm::kS, Sm::LDK, static_cast<const E*>(a.S) + (id * a.Vp + v0) * KD, KD, vn, KD, tid, 128);
        load_ws(s + Sm::kU, Sm::LDU, static_cast<const E*>(a.U) + id * kC * a.Vp + v0, a.Vp, kC, vn, tid, 128);
        cp_async_commit();
        cp_async_wait_all();
        __syncthreads();
        if (v0 == 0) {
#pragma unroll
            for (int j = 0; j < kC / 8; ++j) Mx[j][0] = Mx[j][1] = Mx[j][2] = Mx[j][3] = 0.f;
#pragma unroll
            for (int k0 = 0; k0 < KD; k0 += 16) {
                const auto af = F::from_smem(s + Sm::kQ, Sm::LDK, m0, k0);
#pragma unroll
                for (int p = 0; p < kC / 16; ++p)
                    if (p <= warp) mm_in<F, 1, false>(Mx[2 * p], Mx[2 * p + 1], af, s + Sm::kK, Sm::LDK, 16 * p, k0);
            }
#pragma unroll
            for (int j = 0; j < kC / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = m0 + L.g + (e >> 1) * 8, col = 8 * j + 2 * L.t + (e & 1);
                    Mx[j][e] = col <= r ? a.scale * expf((ga[r] - ga[col]) + (ga[kC + r] - ga[kC + col])) * Mx[j][e] : 0.f;
                }
            if (a.M) acc_store<E, kC / 8>(Mx, static_cast<E*>(a.M) + (id * kC + m0) * kC, kC, L);
        }
        float O[kOutV / 8][4] = {};
#pragma unroll
        for (int k0 = 0; k0 < KD; k0 += 16) {
            const auto af = F::from_smem(s + Sm::kQ, Sm::LDK, m0, k0);
#pragma unroll
            for (int p = 0; p < kOutV / 16; ++p)
                if (16 * p < vn) mm<F, 1, false>(O[2 * p], O[2 * p + 1], af, s + Sm::kS, Sm::LDK, 16 * p, k0);
        }
        const float f0 = a.scale * ga[2 * kC + m0 + L.g], f1 = a.scale * ga[2 * kC + m0 + L.g + 8];
#pragma unroll
        for (int j = 0; j < kOutV / 8; ++j) {
            O[j][0] *= f0;
            O[j][1] *= f0;
            O[j][2] *= f1;
            O[j][3] *= f1;
        }
#pragma unroll
        for (int kk = 0; kk < kC / 16; ++kk)
            if (kk <= warp) {
                const auto af = F::template from_acc<1>(Mx[2 * kk], Mx[2 * kk + 1]);
#pragma unroll
                for (int p = 0; p < kOutV / 16; ++p)
                    if (16 * p < vn) mm<F, 1, true>(O[2 * p], O[2 * p + 1], af, s + Sm::kU, Sm::LDU, 16 * p, 16 * kk);
            }
        rows_store<T, kOutV / 8>(O, out, ost, m0, rows, all, v0, a.V, L);
        __syncthreads();
    }
}

// ----------------------------------------------------------------------------
// the reverse chain
// ----------------------------------------------------------------------------
template <class F, int KD, int W>
struct RStage {
    using E = typename F::E;
    static constexpr int LDK = KD + 8, LDV = 16 * W + 8;
    static constexpr int kQ = 0, kK = kQ + kC * LDK, kT = kK + kC * LDK, kM = kT + kC * kTld, kD = kM + kC * kTld;
    static constexpr int kEnd = kD + kC * LDV;
    static constexpr size_t bytes = kEnd * sizeof(E) + 3 * kC * sizeof(float);
    static constexpr int kStages = 2 * bytes <= 200 * 1024 ? 2 : 1;
};

template <class F, typename T, int KD, int W>
__device__ __forceinline__ void rchain_load(const DArgs& a, unsigned char* st, int c, int b, int h, int hk, int len,
                                            int v0, int nthr) {
    using S = RStage<F, KD, W>;
    using E = typename F::E;
    E* e = reinterpret_cast<E*>(st);
    float* ga = reinterpret_cast<float*>(e + S::kEnd);
    const int64_t id = (static_cast<int64_t>(b) * a.Hv + h) * a.n + c;
    const int64_t t0 = static_cast<int64_t>(c) * kC;
    const int rows = min(kC, len - c * kC), tid = threadIdx.x;
    load_rows<F, T>(e + S::kK, S::LDK, static_cast<const T*>(a.k) + b * a.sk.b + t0 * a.sk.t + hk * a.sk.h, a.sk.t, rows,
                    a.K, KD, a.vec_qk, tid, nthr);
    load_rows<F, T>(e + S::kQ, S::LDK, static_cast<const T*>(a.q) + b * a.sq.b + t0 * a.sq.t + hk * a.sq.h, a.sq.t, rows,
                    a.K, KD, a.vec_qk, tid, nthr);
    load_rows<F, T>(e + S::kD, S::LDV, static_cast<const T*>(a.dout) + b * a.sdo.b + t0 * a.sdo.t + h * a.sdo.h + v0,
                    a.sdo.t, rows, a.V - v0, 16 * W, a.vec_do, tid, nthr);
    load_ws(e + S::kT, kTld, static_cast<const E*>(a.T) + id * kC * kC, kC, kC, kC, tid, nthr);
    load_ws(e + S::kM, kTld, static_cast<const E*>(a.M) + id * kC * kC, kC, kC, kC, tid, nthr);
    load_ws(ga, 3 * kC, a.gates + id * kGates + 2 * kC, 3 * kC, 1, 3 * kC, tid, nthr);
}

template <class F, typename T, int KD, int W>
__global__ void __launch_bounds__(W * 32) delta_rchain_k(DArgs a) {
    using E = typename F::E;
    using St = RStage<F, KD, W>;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / (a.Hv / a.Hk);
    const int len = row_length(a, b), nc = (len + kC - 1) / kC;
    const int warp = threadIdx.x >> 5, vb = blockIdx.x * 16 * W, v0 = vb + warp * 16;
    const Lane L;
    extern __shared__ __align__(16) unsigned char smem[];
    const int64_t head = static_cast<int64_t>(b) * a.Hv + h;
    float S[KD / 8][4];  // dS^T
    state_load<KD>(S, a.dfinal ? a.dfinal + head * a.K * a.V : nullptr, a.K, a.V, v0, L);
    const bool on = v0 < a.Vp;
    constexpr bool two = St::kStages == 2;
    float4* mine = reinterpret_cast<float4*>(smem + St::kStages * St::bytes) + warp * 4 * KD + L.l;
    if (two && nc > 0) {
        rchain_load<F, T, KD, W>(a, smem + ((nc - 1) & 1) * St::bytes, nc - 1, b, h, hk, len, vb, W * 32);
        cp_async_commit();
    }
    for (int c = nc - 1; c >= 0; --c) {
        unsigned char* st = smem + (two ? (c & 1) * St::bytes : 0);
        if (two) {
            if (c > 0) rchain_load<F, T, KD, W>(a, smem + ((c - 1) & 1) * St::bytes, c - 1, b, h, hk, len, vb, W * 32);
            cp_async_commit();
            cp_async_wait_group<1>();
        } else {
            rchain_load<F, T, KD, W>(a, st, c, b, h, hk, len, vb, W * 32);
            cp_async_commit();
            cp_async_wait_group<0>();
        }
        __syncthreads();
        if (on) {
            const E* e = reinterpret_cast<const E*>(st);
            const float* gam = reinterpret_cast<const float*>(e + St::kEnd);
            const float* dec = gam + kC;
            const int64_t id = head * a.n + c;
            acc_store<E, KD / 8>(S, static_cast<E*>(a.dS) + (id * a.Vp + v0) * KD, KD, L);
            float U[kC / 8][4] = {};  // dU^T
            lane_put<KD / 8>(mine, S);
#pragma unroll 1
            for (int k0 = 0; k0 < KD; k0 += 16) {
                float x0[4], x1[4];
                lane_get(x0, mine + k0 * 4);
                lane_get(x1, mine + k0 * 4 + 32);
                const auto af = F::template from_acc<1>(x0, x1);
#pragma unroll
                for (int p = 0; p < kC / 16; ++p)
                    mm_in<F, 1, false>(U[2 * p], U[2 * p + 1], af, e + St::kK, St::LDK, 16 * p, k0);
            }
#pragma unroll
            for (int j = 0; j < kC / 8; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) U[j][x] *= dec[8 * j + 2 * L.t + (x & 1)];
#pragma unroll 1
            for (int kk = 0; kk < kC / 16; ++kk) {
                const auto af = F::from_smem_t(e + St::kD, St::LDV, warp * 16, 16 * kk);
#pragma unroll
                for (int p = 0; p < kC / 16; ++p)
                    if (p <= kk) mm<F, 1, true>(U[2 * p], U[2 * p + 1], af, e + St::kM, kTld, 16 * p, 16 * kk);
            }
            lane_put<kC / 8>(mine, U);
            float X[kC / 8][4] = {};  // dV^T
#pragma unroll 1
            for (int kk = 0; kk < kC / 16; ++kk) {
                float x0[4], x1[4];
                lane_get(x0, mine + kk * 64);
                lane_get(x1, mine + kk * 64 + 32);
                const auto af = F::template from_acc<2>(x0, x1);
#pragma unroll
                for (int p = 0; p < kC / 16; ++p)
                    if (p <= kk) mm<F, 2, true>(X[2 * p], X[2 * p + 1], af, e + St::kT, kTld, 16 * p, 16 * kk);
            }
            lane_put<kC / 8>(mine, X);
            acc_store_t<F>(X, static_cast<E*>(a.dV) + id * kC * a.Vp, a.Vp, v0, L);
            const float gc = gam[kC - 1];
#pragma unroll
            for (int j = 0; j < KD / 8; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) S[j][x] *= gc;
#pragma unroll 1
            for (int kk = 0; kk < kC / 16; ++kk) {
                auto ad = F::from_smem_t(e + St::kD, St::LDV, warp * 16, 16 * kk);
                F::scale_k(ad, gam + 2 * kC, 16 * kk);
                float y0[4], y1[4];
                lane_get(y0, mine + kk * 64);
                lane_get(y1, mine + kk * 64 + 32);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    y0[x] *= -gam[16 * kk + 2 * L.t + (x & 1)];
                    y1[x] *= -gam[16 * kk + 8 + 2 * L.t + (x & 1)];
                }
                const auto av = F::template from_acc<1>(y0, y1);
#pragma unroll
                for (int p = 0; p < KD / 16; ++p) {
                    mm_in<F, 1, true>(S[2 * p], S[2 * p + 1], ad, e + St::kQ, St::LDK, 16 * p, 16 * kk);
                    mm_in<F, 1, true>(S[2 * p], S[2 * p + 1], av, e + St::kK, St::LDK, 16 * p, 16 * kk);
                }
            }
        }
        __syncthreads();
    }
    if (on && a.dinitial) state_store<KD>(S, a.dinitial + head * a.K * a.V, a.K, a.V, v0, L);
}

// ----------------------------------------------------------------------------
// dQ, dK, dV, dbeta and dg of a chunk
// ----------------------------------------------------------------------------
// 8 warps: 4 groups of 16 rows by 2 halves of the key columns.  The value
// columns come in tiles of VT, so that the two states of a chunk pass through
// shared memory in parts.
template <class F, int KD>
struct GradSmem {
    using E = typename F::E;
    static constexpr int VT = 32;
    static constexpr int LDK = KD + 8, LDV = VT + 8;
    static constexpr int kQ = 0, kK = kQ + kC * LDK, kD = kK + kC * LDK, kU = kD + kC * LDV, kX = kU + kC * LDV;
    static constexpr int kS = kX + kC * LDV, kR = kS + VT * LDK, kN = kR + VT * LDK, kM = kN + kC * kTld;
    static constexpr int kEnd = kM + kC * kTld;
    // floats: gates, beta, row sums of both halves, dbeta, partial totals
    static constexpr size_t bytes = kEnd * sizeof(E) + (kGates + 4 * kC + 32) * sizeof(float);
};

template <class F, typename T, int KD>
__global__ void __launch_bounds__(256) delta_grad_k(DArgs a, float* group) {
    using E = typename F::E;
    using Sm = GradSmem<F, KD>;
    constexpr int VT = Sm::VT, NT = KD / 16;  // accumulator tiles of a warp's half of the key columns
    const int c = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, rep = a.Hv / a.Hk;
    const int len = row_length(a, b);
    const int all = min(kC, a.L - c * kC), rows = min(kC, len - c * kC);
    const int64_t t0 = static_cast<int64_t>(c) * kC;
    const int64_t row0 = static_cast<int64_t>(b) * a.L + t0;  // first row of the outputs
    const int tid = threadIdx.x, warp = tid >> 5, rg = warp & 3, half = warp >> 2, m0 = rg * 16;
    const Lane L;
    const int64_t qst = static_cast<int64_t>(a.Hk) * a.K, vst = static_cast<int64_t>(a.Hv) * a.V;
    T* dq = static_cast<T*>(a.dq) + row0 * qst + static_cast<int64_t>(hk) * a.K;
    T* dk = static_cast<T*>(a.dk) + row0 * qst + static_cast<int64_t>(hk) * a.K;
    if (rows <= 0) {  // behind the sequence
        for (int i = tid; i < all * a.K; i += 256) {
            const int64_t o = (i / a.K) * qst + i % a.K;
            dq[o] = T(0.f);
            dk[o] = T(0.f);
        }
        for (int h = hk * rep; h < (hk + 1) * rep; ++h) {
            T* dv = static_cast<T*>(a.dv) + row0 * vst + static_cast<int64_t>(h) * a.V;
            for (int i = tid; i < all * a.V; i += 256) dv[(i / a.V) * vst + i % a.V] = T(0.f);
            for (int i = tid; i < all; i += 256) {
                gate_store(a.dg, a.gate_dtype, (row0 + i) * a.Hv + h, 0.f);
                gate_store(a.dbeta, a.gate_dtype, (row0 + i) * a.Hv + h, 0.f);
            }
        }
        return;
    }
    extern __shared__ __align__(16) unsigned char smem[];
    E* s = reinterpret_cast<E*>(smem);
    float* ga = reinterpret_cast<float*>(s + Sm::kEnd);
    float* sBeta = ga + kGates;
    float* sDot = sBeta + kC;  // [2][64]
    float* sDb = sDot + 2 * kC;
    float* sTot = sDb + kC;    // [8] <S0, dS1>, [8] sums of k.(d U dS1^T)
    load_rows<F, T>(s + Sm::kQ, Sm::LDK, static_cast<const T*>(a.q) + b * a.sq.b + t0 * a.sq.t + hk * a.sq.h, a.sq.t, rows,
                    a.K, KD, a.vec_qk, tid, 256);
    load_rows<F, T>(s + Sm::kK, Sm::LDK, static_cast<const T*>(a.k) + b * a.sk.b + t0 * a.sk.t + hk * a.sk.h, a.sk.t, rows,
                    a.K, KD, a.vec_qk, tid, 256);
    for (int h = hk * rep; h < (hk + 1) * rep; ++h) {
        const int64_t id = (static_cast<int64_t>(b) * a.Hv + h) * a.n + c;
        load_ws(ga, kGates, a.gates + id * kGates, kGates, 1, kGates, tid, 256);
        if (tid < kC)
            sBeta[tid] = tid < rows ? hold_beta(gate_value(a.beta, a.gate_dtype,
                                                           b * a.sb.b + (t0 + tid) * a.sb.t + h * a.sb.h))
                                    : 1.f;
        T* dv = static_cast<T*>(a.dv) + row0 * vst + static_cast<int64_t>(h) * a.V;
        float P[kC / 8][4] = {};  // half 0: dO U^T, half 1: dV U^T
        float aq[NT][4] = {}, ar[NT][4] = {}, aw[NT][4] = {};
        float db = 0.f, sd = 0.f;
        const int n0 = half * (KD / 2);
        for (int v0 = 0; v0 < a.Vp; v0 += VT) {
            const int vn = min(VT, a.Vp - v0);
            load_rows<F, T>(s + Sm::kD, Sm::LDV, static_cast<const T*>(a.dout) + b * a.sdo.b + t0 * a.sdo.t + h * a.sdo.h + v0,
                            a.sdo.t, rows, a.V - v0, vn, a.vec_do, tid, 256);
            load_ws(s + Sm::kU, Sm::LDV, static_cast<const E*>(a.U) + id * kC * a.Vp + v0, a.Vp, kC, vn, tid, 256);
            load_ws(s + Sm::kX, Sm::LDV, static_cast<const E*>(a.dV) + id * kC * a.Vp + v0, a.Vp, kC, vn, tid, 256);
            load_ws(s + Sm::kS, Sm::LDK, static_cast<const E*>(a.S) + (id * a.Vp + v0) * KD, KD, vn, KD, tid, 256);
            load_ws(s + Sm::kR, Sm::LDK, static_cast<const E*>(a.dS) + (id * a.Vp + v0) * KD, KD, vn, KD, tid, 256);
            cp_async_commit();
            cp_async_wait_all();
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < VT / 16; ++kk) {
                if (16 * kk >= vn) break;
                const auto fd = F::from_smem(s + Sm::kD, Sm::LDV, m0, 16 * kk);
                const auto fx = F::from_smem(s + Sm::kX, Sm::LDV, m0, 16 * kk);
                const auto fu = F::from_smem(s + Sm::kU, Sm::LDV, m0, 16 * kk);
#pragma unroll
                for (int p = 0; p < kC / 16; ++p)
                    if (p <= rg) {
                        if (half) mm<F, 1, false>(P[2 * p], P[2 * p + 1], fx, s + Sm::kU, Sm::LDV, 16 * p, 16 * kk);
                        else mm<F, 1, false>(P[2 * p], P[2 * p + 1], fd, s + Sm::kU, Sm::LDV, 16 * p, 16 * kk);
                    }
#pragma unroll
                for (int p = 0; p < NT / 2; ++p) {
                    mm<F, 1, true>(aq[2 * p], aq[2 * p + 1], fd, s + Sm::kS, Sm::LDK, n0 + 16 * p, 16 * kk);
                    mm<F, 1, true>(ar[2 * p], ar[2 * p + 1], fx, s + Sm::kS, Sm::LDK, n0 + 16 * p, 16 * kk);
                    mm<F, 1, true>(aw[2 * p], aw[2 * p + 1], fu, s + Sm::kR, Sm::LDK, n0 + 16 * p, 16 * kk);
                }
            }
            {  // dbeta: four threads a row; dv; <S0, dS1>
                const int r = tid >> 2;
                const float ib = 1.f / sBeta[r];
                for (int v = tid & 3; v < vn; v += 4)
                    db = fmaf(to_f32(s[Sm::kX + r * Sm::LDV + v]) * ib, to_f32(s[Sm::kU + r * Sm::LDV + v]) * ib, db);
                for (int i = tid; i < all * vn; i += 256) {
                    const int rr = i / vn, v = i - rr * vn;
                    if (v0 + v < a.V) dv[rr * vst + v0 + v] = T(rr < rows ? to_f32(s[Sm::kX + rr * Sm::LDV + v]) : 0.f);
                }
                for (int i = tid; i < vn * KD; i += 256) {
                    const int rr = i / KD, k = i - rr * KD;
                    sd = fmaf(to_f32(s[Sm::kS + rr * Sm::LDK + k]), to_f32(s[Sm::kR + rr * Sm::LDK + k]), sd);
                }
            }
            __syncthreads();
        }
        db += __shfl_xor_sync(0xffffffffu, db, 1);
        db += __shfl_xor_sync(0xffffffffu, db, 2);
        if ((tid & 3) == 0) sDb[tid >> 2] = db;
        sd = warp_sum(sd);
        {  // N (half 0) and E (half 1)
            E* o = s + (half ? Sm::kM : Sm::kN);
#pragma unroll
            for (int j = 0; j < kC / 8; ++j) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = m0 + L.g + (e >> 1) * 8, col = 8 * j + 2 * L.t + (e & 1);
                    const bool in = half ? col < r : col <= r;
                    v[e] = in ? (half ? -1.f : a.scale) * expf((ga[r] - ga[col]) + (ga[kC + r] - ga[kC + col])) * P[j][e]
                              : 0.f;
                }
                put2(o + (m0 + L.g) * kTld + 8 * j + 2 * L.t, v[0], v[1]);
                put2(o + (m0 + L.g + 8) * kTld + 8 * j + 2 * L.t, v[2], v[3]);
            }
        }
        __syncthreads();
        const int r0 = m0 + L.g, r1 = r0 + 8;
        const float g0 = ga[2 * kC + r0], g1 = ga[2 * kC + r1], d0 = ga[3 * kC + r0], d1 = ga[3 * kC + r1];
        float tw = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int col = n0 + 8 * j + 2 * L.t;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float gi = e < 2 ? g0 : g1, di = e < 2 ? d0 : d1;
                aq[j][e] *= a.scale * gi;
                ar[j][e] *= -gi;
                aw[j][e] *= di;
                tw = fmaf(to_f32(s[Sm::kK + (e < 2 ? r0 : r1) * Sm::LDK + col + (e & 1)]), aw[j][e], tw);
            }
        }
#pragma unroll
        for (int kk = 0; kk < kC / 16; ++kk) {
            if (kk <= rg) {  // rows of N and E
                const auto fn = F::from_smem(s + Sm::kN, kTld, m0, 16 * kk);
                const auto fe = F::from_smem(s + Sm::kM, kTld, m0, 16 * kk);
#pragma unroll
                for (int p = 0; p < NT / 2; ++p) {
                    mm_in<F, 1, true>(aq[2 * p], aq[2 * p + 1], fn, s + Sm::kK, Sm::LDK, n0 + 16 * p, 16 * kk);
                    mm_in<F, 1, true>(ar[2 * p], ar[2 * p + 1], fe, s + Sm::kK, Sm::LDK, n0 + 16 * p, 16 * kk);
                }
            }
            if (kk >= rg) {  // columns of N and E
                const auto fn = F::from_smem_t(s + Sm::kN, kTld, m0, 16 * kk);
                const auto fe = F::from_smem_t(s + Sm::kM, kTld, m0, 16 * kk);
#pragma unroll
                for (int p = 0; p < NT / 2; ++p) {
                    mm_in<F, 1, true>(aw[2 * p], aw[2 * p + 1], fn, s + Sm::kQ, Sm::LDK, n0 + 16 * p, 16 * kk);
                    mm_in<F, 1, true>(aw[2 * p], aw[2 * p + 1], fe, s + Sm::kK, Sm::LDK, n0 + 16 * p, 16 * kk);
                }
            }
        }
        float dot0 = 0.f, dot1 = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = n0 + 8 * j + 2 * L.t + (e & 1), r = e < 2 ? r0 : r1;
                const float qv = to_f32(s[Sm::kQ + r * Sm::LDK + col]), kv = to_f32(s[Sm::kK + r * Sm::LDK + col]);
                float& dot = e < 2 ? dot0 : dot1;
                dot = fmaf(qv, aq[j][e], dot);
                dot = fmaf(kv, ar[j][e] - aw[j][e], dot);
                ar[j][e] += aw[j][e];  // dK
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            dot0 += __shfl_xor_sync(0xffffffffu, dot0, o);
            dot1 += __shfl_xor_sync(0xffffffffu, dot1, o);
        }
        tw = warp_sum(tw);
        if (L.t == 0) {
            sDot[half * kC + r0] = dot0;
            sDot[half * kC + r1] = dot1;
        }
        if (L.l == 0) {
            sTot[warp] = sd;
            sTot[8 + warp] = tw;
        }
        if (rep > 1) {  // the sum over the value heads of this key head; each thread its own elements
            float* gq = group + ((static_cast<int64_t>(b) * a.Hk + hk) * a.n + c) * 2 * kC * KD;
            float* gk = gq + kC * KD;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int o = (e ? r1 : r0) * KD + n0 + 8 * j + 2 * L.t;
                    float2 x = make_float2(aq[j][2 * e], aq[j][2 * e + 1]), y = make_float2(ar[j][2 * e], ar[j][2 * e + 1]);
                    if (h > hk * rep) {
                        const float2 p = *reinterpret_cast<const float2*>(gq + o), q = *reinterpret_cast<const float2*>(gk + o);
                        x.x += p.x; x.y += p.y; y.x += q.x; y.y += q.y;
                    }
                    *reinterpret_cast<float2*>(gq + o) = x;
                    *reinterpret_cast<float2*>(gk + o) = y;
                    aq[j][2 * e] = x.x; aq[j][2 * e + 1] = x.y;
                    ar[j][2 * e] = y.x; ar[j][2 * e + 1] = y.y;
                }
        }
        if (h == (hk + 1) * rep - 1) {
            rows_store<T, NT>(aq, dq, qst, m0, rows, all, n0, a.K, L);
            rows_store<T, NT>(ar, dk, qst, m0, rows, all, n0, a.K, L);
        }
        __syncthreads();
        if (warp == 0) {
            float tot = 0.f, w = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                tot += sTot[i];
                w += sTot[8 + i];
            }
            tot = fmaf(ga[2 * kC + kC - 1], tot, w);  // <S1, dS1>
            const int i0 = 2 * L.l;
            float y1 = sDot[i0 + 1] + sDot[kC + i0 + 1];
            float y0 = sDot[i0] + sDot[kC + i0] + y1;
            float run = y0;  // sums from here to the end
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float dn = __shfl_down_sync(0xffffffffu, run, o);
                if (L.l + o < 32) run += dn;
            }
            const float behind = run - y0 + tot;
            const int64_t o = (row0 + i0) * a.Hv + h;
            if (i0 < all) {
                // (the first token's decay meets an empty state: no rounding of the terms that cancel)
                const bool none = i0 == 0 && c == 0 && !a.initial;
                gate_store(a.dg, a.gate_dtype, o, i0 < rows && !none ? y0 + behind : 0.f);
                gate_store(a.dbeta, a.gate_dtype, o, i0 < rows ? sDb[i0] : 0.f);
            }
            if (i0 + 1 < all) {
                gate_store(a.dg, a.gate_dtype, o + a.Hv, i0 + 1 < rows ? y1 + behind : 0.f);
                gate_store(a.dbeta, a.gate_dtype, o + a.Hv, i0 + 1 < rows ? sDb[i0 + 1] : 0.f);
            }
        }
        __syncthreads();
    }
}

// ----------------------------------------------------------------------------
// token by token
// ----------------------------------------------------------------------------
// A CTA takes 32 value columns of one head; a thread 4 of them and every 16th
// key row, in registers from the first token to the last.  k^T S' and q^T S'
// are summed together, as o = q^T S' + (q.k) u; one token is one pass over the
// state: read once, written once.
// Bound by the state's bytes, of which a CTA has none under way while it adds up,
// and by the last round of CTAs (64 rows of 16 heads: 4096 on 1184 places): so
// eight CTAs share a multiprocessor (K = 128, 64 rows of 16 heads: 29.0 us, 4.6
// TB/s, against 33.3 with the five that 82 registers a thread allow; 16 rows 6.7
// us against 7.9; six or ten CTAs, 64 or 128 columns a CTA were no faster).
template <typename T, int KD>
__global__ void __launch_bounds__(128, 8) delta_step_k(const __grid_constant__ DArgs a, int vec_s) {
    constexpr int R = KD / 16;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / (a.Hv / a.Hk);
    const int len = row_length(a, b);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kg = tid >> 3;
    const int v = blockIdx.x * 32 + (tid & 7) * 4;
    const int64_t head = static_cast<int64_t>(b) * a.Hv + h, base = head * a.K * a.V;
    __shared__ float sq[2][KD], sk[2][KD];
    __shared__ float4 red[2][2][4][8];
    float S[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int k = kg + 16 * i;
#pragma unroll
        for (int e = 0; e < 4; ++e) S[i][e] = 0.f;
        if (a.initial && k < a.K && v < a.V) {
            const float* p = a.initial + base + (k * a.V + v);
            if (vec_s) {
                const float4 x = *reinterpret_cast<const float4*>(p);
                S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (v + e < a.V) S[i][e] = p[e];
            }
        }
    }
    const T* q = static_cast<const T*>(a.q) + b * a.sq.b + hk * a.sq.h;
    const T* k = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
    const T* vp = static_cast<const T*>(a.v) + b * a.sv.b + h * a.sv.h;
    for (int t = 0; t < len; ++t) {
        const int s = t & 1;
        if (tid < KD) {
            const bool in = tid < a.K;
            sq[s][tid] = in ? to_f32(q[t * a.sq.t + tid]) : 0.f;
            sk[s][tid] = in ? to_f32(k[t * a.sk.t + tid]) : 0.f;
        }
        const float al = expf(gate_value(a.g, a.gate_dtype, b * a.sg.b + t * a.sg.t + h * a.sg.h));
        const float be = gate_value(a.beta, a.gate_dtype, b * a.sb.b + t * a.sb.t + h * a.sb.h);
        __syncthreads();
        float x[4] = {}, y[4] = {}, qk = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float kv = sk[s][kg + 16 * i], qv = sq[s][kg + 16 * i];
            qk = fmaf(qv, kv, qk);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                S[i][e] *= al;
                x[e] = fmaf(kv, S[i][e], x[e]);
                y[e] = fmaf(qv, S[i][e], y[e]);
            }
        }
#pragma unroll
        for (int o = 8; o < 32; o <<= 1) {
            qk += __shfl_xor_sync(0xffffffffu, qk, o);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] += __shfl_xor_sync(0xffffffffu, x[e], o);
                y[e] += __shfl_xor_sync(0xffffffffu, y[e], o);
            }
        }
        __shared__ float sqk[2][4];
        if (lane < 8) {
            red[s][0][warp][lane] = make_float4(x[0], x[1], x[2], x[3]);
            red[s][1][warp][lane] = make_float4(y[0], y[1], y[2], y[3]);
            if (lane == 0) sqk[s][warp] = qk;
        }
        __syncthreads();
        float val[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) val[e] = v + e < a.V ? to_f32(vp[t * a.sv.t + v + e]) : 0.f;
        float4 X = red[s][0][0][lane & 7], Y = red[s][1][0][lane & 7];
        qk = sqk[s][0];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            const float4 p = red[s][0][w][lane & 7], r = red[s][1][w][lane & 7];
            X.x += p.x; X.y += p.y; X.z += p.z; X.w += p.w;
            Y.x += r.x; Y.y += r.y; Y.z += r.z; Y.w += r.w;
            qk += sqk[s][w];
        }
        const float u[4] = {be * (val[0] - X.x), be * (val[1] - X.y), be * (val[2] - X.z), be * (val[3] - X.w)};
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float kv = sk[s][kg + 16 * i];
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] = fmaf(kv, u[e], S[i][e]);
        }
        if (kg == 0) {
            T* o = static_cast<T*>(a.out) + ((static_cast<int64_t>(b) * a.L + t) * a.Hv + h) * a.V + v;
            const float ov[4] = {Y.x + qk * u[0], Y.y + qk * u[1], Y.z + qk * u[2], Y.w + qk * u[3]};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e < a.V) o[e] = T(a.scale * ov[e]);
        }
    }
    if (kg == 0)
        for (int t = len; t < a.L; ++t) {
            T* o = static_cast<T*>(a.out) + ((static_cast<int64_t>(b) * a.L + t) * a.Hv + h) * a.V + v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e < a.V) o[e] = T(0.f);
        }
    if (!a.final_state) return;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int kr = kg + 16 * i;
        if (kr < a.K && v < a.V) {
            float* p = a.final_state + base + (kr * a.V + v);
            if (vec_s) {
                *reinterpret_cast<float4*>(p) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (v + e < a.V) p[e] = S[i][e];
            }
        }
    }
}

// ----------------------------------------------------------------------------
// launches
// ----------------------------------------------------------------------------
template <class F, typename T, int KD, int W>
cudaError_t run_chain(const DArgs& a, bool reverse, cudaStream_t s) {
    const dim3 grid((a.Vp + 16 * W - 1) / (16 * W), a.Hv, a.B);
    if (reverse) {
        using St = RStage<F, KD, W>;
        constexpr size_t bytes = St::kStages * St::bytes + kLaneBytes<KD, W>;
        DELTA_TRY(smem_limit(delta_rchain_k<F, T, KD, W>, bytes));
        delta_rchain_k<F, T, KD, W><<<grid, W * 32, bytes, s>>>(a);
    } else {
        using St = ChainStage<F, KD, W>;
        constexpr size_t bytes = 2 * St::bytes + kLaneBytes<KD, W>;
        DELTA_TRY(smem_limit(delta_chain_k<F, T, KD, W>, bytes));
        delta_chain_k<F, T, KD, W><<<grid, W * 32, bytes, s>>>(a);
    }
    note_launch();
    return cudaGetLastError();
}

// A chain's warps are independent, so they are spread over the SMs: two to a
// CTA while that gives at most two CTAs an SM, else four.
template <class F, typename T, int KD>
cudaError_t run_chain(const DArgs& a, bool reverse, cudaStream_t s) {
    const int64_t pairs = static_cast<int64_t>(a.B) * a.Hv * ((a.Vp + 31) / 32);
    return pairs <= 2 * 148 ? run_chain<F, T, KD, 2>(a, reverse, s) : run_chain<F, T, KD, 4>(a, reverse, s);
}

template <class F, typename T, int KD>
cudaError_t run_fwd(const DArgs& a, cudaStream_t s) {
    const dim3 grid(a.n, a.Hv, a.B);
    const size_t prep = kC * (KD + 8) * sizeof(typename F::E) + (kC * kC + 3 * kC) * sizeof(float);
    DELTA_TRY(smem_limit(delta_prep_k<F, T, KD>, prep));
    delta_prep_k<F, T, KD><<<grid, 128, prep, s>>>(a);
    note_launch();
    DELTA_TRY(cudaGetLastError());
    DELTA_TRY((run_chain<F, T, KD>(a, false, s)));
    DELTA_TRY(smem_limit(delta_out_k<F, T, KD>, OutSmem<F, KD>::bytes));
    delta_out_k<F, T, KD><<<grid, 128, OutSmem<F, KD>::bytes, s>>>(a);
    note_launch();
    return cudaGetLastError();
}

template <class F, typename T, int KD>
cudaError_t run_grad(const DArgs& a, float* group, cudaStream_t s) {
    DELTA_TRY(smem_limit(delta_grad_k<F, T, KD>, GradSmem<F, KD>::bytes));
    delta_grad_k<F, T, KD><<<dim3(a.n, a.Hk, a.B), 256, GradSmem<F, KD>::bytes, s>>>(a, group);
    note_launch();
    return cudaGetLastError();
}

template <class F, typename T, int KD>
cudaError_t run_bwd(const DArgs& a, float* group, cudaStream_t s) {
    DELTA_TRY((run_chain<F, T, KD>(a, true, s)));
    return run_grad<F, T, KD>(a, group, s);
}

template <typename T>
cudaError_t run_step(const DArgs& a, cudaStream_t s) {
    const dim3 grid((a.V + 31) / 32, a.Hv, a.B);
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    const int vec = a.V % 4 == 0 && aligned(a.initial) && aligned(a.final_state);
    if (a.K <= 64) delta_step_k<T, 64><<<grid, 128, 0, s>>>(a, vec);
    else delta_step_k<T, 128><<<grid, 128, 0, s>>>(a, vec);
    note_launch();
    return cudaGetLastError();
}

int64_t chunks(int64_t L) { return (L + kC - 1) / kC; }
int64_t pad16(int64_t v) { return (v + 15) / 16 * 16; }
int64_t key_pad(int64_t K) { return K <= 64 ? 64 : 128; }
size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// EACS_OK, or the error that these sizes and types are refused with
int check_sizes(const EacsDelta& p, const char* fn) {
    if (p.B < 0 || p.L < 0 || p.Hk <= 0 || p.Hv <= 0 || p.K <= 0 || p.V <= 0)
        return fail(EACS_ERR_INVALID, "%s: bad sizes", fn);
    if (p.Hv % p.Hk != 0)
        return fail(EACS_ERR_INVALID, "%s: Hv=%lld is not a multiple of Hk=%lld", fn, (long long)p.Hv, (long long)p.Hk);
    for (int dt : {p.dtype, p.gate_dtype})
        if (dt != EACS_DTYPE_F32 && dt != EACS_DTYPE_F16 && dt != EACS_DTYPE_BF16)
            return fail(EACS_ERR_INVALID, "%s: unknown dtype %d", fn, dt);
    if (p.K > 128) return fail(EACS_ERR_UNSUPPORTED, "%s: K=%lld > 128", fn, (long long)p.K);
    if (p.V > 1024) return fail(EACS_ERR_UNSUPPORTED, "%s: V=%lld > 1024", fn, (long long)p.V);
    if (p.B > 65535 || p.Hv > 65535 || p.L > (int64_t{1} << 30))
        return fail(EACS_ERR_UNSUPPORTED, "%s: B and Hv go to 65535, L to 2^30", fn);
    if (p.B * p.Hv * ((p.L + kC - 1) / kC) > (int64_t{1} << 31) - 1)
        return fail(EACS_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 chunks of 64 tokens in all", fn);
    return EACS_OK;
}

// Whether rows of n elements start on 16 bytes (a dimension of one element has no stride).
bool rows16(const EacsDelta& d, const void* p, const int64_t* st, int64_t H, int64_t n) {
    const int e = d.dtype == EACS_DTYPE_F32 ? 4 : 2;
    const int64_t size[3] = {d.B, d.L, H};
    uintptr_t bits = reinterpret_cast<uintptr_t>(p);
    for (int i = 0; i < 3; ++i)
        if (size[i] > 1) bits |= static_cast<uintptr_t>(st[i]) * e;
    return (bits & 15u) == 0 && n % 8 == 0;
}

DArgs make_args(const EacsDelta& p) {
    DArgs a{};
    auto str = [](const int64_t* s) { return Str{s[0], s[1], s[2]}; };
    a.q = p.q; a.k = p.k; a.v = p.v; a.g = p.g; a.beta = p.beta;
    a.sq = str(p.q_stride); a.sk = str(p.k_stride); a.sv = str(p.v_stride);
    a.sg = str(p.g_stride); a.sb = str(p.beta_stride);
    a.lengths = p.lengths;
    a.initial = p.initial_state;
    a.B = static_cast<int>(p.B); a.L = static_cast<int>(p.L);
    a.Hk = static_cast<int>(p.Hk); a.Hv = static_cast<int>(p.Hv);
    a.K = static_cast<int>(p.K); a.V = static_cast<int>(p.V);
    a.n = static_cast<int>(chunks(p.L)); a.Vp = static_cast<int>(pad16(p.V));
    a.gate_dtype = p.gate_dtype;
    a.half = p.dtype == EACS_DTYPE_F16;
    a.vec_qk = rows16(p, p.q, p.q_stride, p.Hk, p.K) && rows16(p, p.k, p.k_stride, p.Hk, p.K);
    a.vec_v = rows16(p, p.v, p.v_stride, p.Hv, p.V);
    a.scale = p.scale;
    return a;
}
// What a tensor map can describe: rows that start on 16 bytes, and strides above 0
// and below 2^40 bytes (an expanded dimension has stride 0).
bool mapped(int64_t B, int64_t L, int64_t H, const int64_t* st) {
    const int64_t n[3] = {B, L, H};
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (st[i] <= 0 || st[i] >= int64_t{1} << 39)) return false;
    return true;
}
// Whether the 16-bit kernels take these inputs.  The backward goes by the
// forward's path, or by its inputs alone, as it reads what the forward left (an
// upstream gradient in another layout is refused by delta_bwd then).
bool planes_take(const EacsDelta& p, const DArgs& a) {
    return p.dtype != EACS_DTYPE_F32 && a.vec_qk && a.vec_v && mapped(p.B, p.L, p.Hk, p.q_stride) &&
           mapped(p.B, p.L, p.Hk, p.k_stride) && mapped(p.B, p.L, p.Hv, p.v_stride);
}
// The path of a call: the caller's, or the one that its inputs lead to.
bool planes(const EacsDelta& p, const DArgs& a) {
    return p.path == 0 ? planes_take(p, a) : p.path == EACS_DELTA_PATH_16;
}

int check_delta(const EacsDelta& p, const char* fn) {
    if (int rc = check_sizes(p, fn)) return rc;
    if (p.path < 0 || p.path > EACS_DELTA_PATH_16) return fail(EACS_ERR_INVALID, "%s: unknown path %d", fn, p.path);
    if (p.path == EACS_DELTA_PATH_16 && !planes_take(p, make_args(p)))
        return fail(EACS_ERR_INVALID, "%s: the 16-bit kernels do not take these inputs", fn);
    return EACS_OK;
}

struct Sizes { size_t gates, T, M, S, U, total; };
Sizes fwd_sizes(const EacsDelta& p, const DArgs& a, bool training) {
    const size_t ids = static_cast<size_t>(p.B) * p.Hv * chunks(p.L), e = sizeof(float);
    Sizes z{};
    if (planes(p, a)) {
        z.total = planes_saved_size(a, training);
        return z;
    }
    z.gates = align256(ids * kGates * e);
    z.T = align256(ids * kC * kC * e);
    z.M = training ? align256(ids * kC * kC * e) : 0;
    z.S = align256(ids * pad16(p.V) * key_pad(p.K) * e);
    z.U = align256(ids * pad16(p.V) * kC * e);
    z.total = z.gates + z.T + z.M + z.S + z.U;
    return z;
}
struct BSizes { size_t dS, dV, group, total; };
BSizes bwd_sizes(const EacsDelta& p, const DArgs& a) {
    const size_t ids = static_cast<size_t>(p.B) * p.Hv * chunks(p.L), e = sizeof(float);
    BSizes z{};
    if (planes(p, a)) {
        z.dS = align256(planes_bwd_size(a));
    } else {
        z.dS = align256(ids * pad16(p.V) * key_pad(p.K) * e);
        z.dV = align256(ids * pad16(p.V) * kC * e);
    }
    z.group = p.Hv > p.Hk ? align256(static_cast<size_t>(p.B) * p.Hk * chunks(p.L) * 2 * kC * key_pad(p.K) * 4) : 0;
    z.total = z.dS + z.dV + z.group;
    return z;
}

void set_workspace(DArgs& a, const EacsDelta& p, void* ws, bool training) {
    const Sizes z = fwd_sizes(p, a, training);
    char* w = static_cast<char*>(ws);
    a.gates = reinterpret_cast<float*>(w); w += z.gates;
    a.T = w; w += z.T;
    a.M = training ? w : nullptr; w += z.M;
    a.S = w; w += z.S;
    a.U = w;
}
bool inputs_set(const EacsDelta& p) { return p.q && p.k && p.v && p.g && p.beta; }
// Outputs and the gradients of tokens are stored in pairs, or 16 bytes at a time
// where K and V are multiples of 8: every store is aligned if their starts are.
bool on16(std::initializer_list<const void*> ps) {
    uintptr_t bits = 0;
    for (const void* p : ps) bits |= reinterpret_cast<uintptr_t>(p);
    return (bits & 15u) == 0;
}

}  // namespace

int delta_path(const EacsDelta& p) {
    if (check_delta(p, "eacs_delta_path") != EACS_OK) return 0;
    return planes(p, make_args(p)) ? EACS_DELTA_PATH_16 : EACS_DELTA_PATH_GENERAL;
}
size_t delta_workspace_size(const EacsDelta& p, bool training) {
    if (check_delta(p, "eacs_delta_workspace_size") != EACS_OK) return 0;
    return fwd_sizes(p, make_args(p), training).total;
}
size_t delta_bwd_workspace_size(const EacsDelta& p) {
    if (check_delta(p, "eacs_delta_bwd_workspace_size") != EACS_OK) return 0;
    return bwd_sizes(p, make_args(p)).total;
}

int delta_fwd(const EacsDelta& p, void* o, float* final_state, void* ws, size_t ws_bytes, bool training,
              cudaStream_t stream) {
    const char* fn = "eacs_delta_fwd";
    if (int rc = check_delta(p, fn)) return rc;
    const size_t state = static_cast<size_t>(p.B) * p.Hv * p.K * p.V * sizeof(float);
    if (p.B == 0) return EACS_OK;
    if (p.L == 0) {  // no token: the state stays
        if (!final_state || final_state == p.initial_state) return EACS_OK;
        return cuda_check(p.initial_state ? cudaMemcpyAsync(final_state, p.initial_state, state, cudaMemcpyDeviceToDevice,
                                                            stream)
                                          : cudaMemsetAsync(final_state, 0, state, stream),
                          fn);
    }
    if (!inputs_set(p) || !o) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    if (!on16({o})) return fail(EACS_ERR_INVALID, "%s: o must start on 16 bytes", fn);
    DArgs a = make_args(p);
    const size_t need = fwd_sizes(p, a, training).total;
    if (!ws || ws_bytes < need) return fail(EACS_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, need);
    if (reinterpret_cast<uintptr_t>(ws) & 15u) return fail(EACS_ERR_INVALID, "%s: workspace must be 16-byte aligned", fn);
    set_workspace(a, p, ws, training);
    a.out = o;
    a.final_state = final_state;
    cudaError_t e;
    if (planes(p, a))
        e = planes_fwd(a, ws, training, stream);
    else if (p.dtype == EACS_DTYPE_BF16)
        e = p.K <= 64 ? run_fwd<FmtF<true>, __nv_bfloat16, 64>(a, stream) : run_fwd<FmtF<true>, __nv_bfloat16, 128>(a, stream);
    else if (p.dtype == EACS_DTYPE_F16)
        e = p.K <= 64 ? run_fwd<FmtF<true>, __half, 64>(a, stream) : run_fwd<FmtF<true>, __half, 128>(a, stream);
    else
        e = p.K <= 64 ? run_fwd<FmtF<false>, float, 64>(a, stream) : run_fwd<FmtF<false>, float, 128>(a, stream);
    return cuda_check(e, fn);
}

int delta_step(const EacsDelta& p, void* o, float* final_state, cudaStream_t stream) {
    const char* fn = "eacs_delta_step";
    if (int rc = check_sizes(p, fn)) return rc;
    if (p.B == 0) return EACS_OK;
    if ((!inputs_set(p) || !o) && p.L > 0) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    DArgs a = make_args(p);
    a.out = o;
    a.final_state = final_state;
    cudaError_t e;
    if (p.dtype == EACS_DTYPE_BF16) e = run_step<__nv_bfloat16>(a, stream);
    else if (p.dtype == EACS_DTYPE_F16) e = run_step<__half>(a, stream);
    else e = run_step<float>(a, stream);
    return cuda_check(e, fn);
}

int delta_bwd(const EacsDelta& p, const DeltaGrads& d, const void* saved, size_t saved_bytes, void* ws, size_t ws_bytes,
              cudaStream_t stream) {
    const char* fn = "eacs_delta_bwd";
    if (int rc = check_delta(p, fn)) return rc;
    const size_t state = static_cast<size_t>(p.B) * p.Hv * p.K * p.V * sizeof(float);
    if (p.B == 0) return EACS_OK;
    if (p.L == 0) {
        if (!d.dinitial) return EACS_OK;
        return cuda_check(d.dfinal ? cudaMemcpyAsync(d.dinitial, d.dfinal, state, cudaMemcpyDeviceToDevice, stream)
                                   : cudaMemsetAsync(d.dinitial, 0, state, stream),
                          fn);
    }
    if (!inputs_set(p) || !d.dout || !d.dq || !d.dk || !d.dv || !d.dg || !d.dbeta)
        return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    if (!on16({d.dq, d.dk, d.dv})) return fail(EACS_ERR_INVALID, "%s: dq, dk and dv must start on 16 bytes", fn);
    DArgs a = make_args(p);
    const size_t need_saved = fwd_sizes(p, a, true).total, need = bwd_sizes(p, a).total;
    if (!saved || saved_bytes < need_saved)
        return fail(EACS_ERR_WORKSPACE, "%s: the forward's workspace has %zu bytes, %zu needed", fn, saved_bytes, need_saved);
    if (!ws || ws_bytes < need) return fail(EACS_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, need);
    if ((reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(saved)) & 15u)
        return fail(EACS_ERR_INVALID, "%s: workspaces must be 16-byte aligned", fn);
    set_workspace(a, p, const_cast<void*>(saved), true);
    a.dout = d.dout;
    a.sdo = Str{d.dout_stride[0], d.dout_stride[1], d.dout_stride[2]};
    a.vec_do = rows16(p, d.dout, d.dout_stride, p.Hv, p.V);
    a.dq = d.dq; a.dk = d.dk; a.dv = d.dv; a.dg = d.dg; a.dbeta = d.dbeta;
    a.dfinal = d.dfinal;
    a.dinitial = d.dinitial;
    if (planes(p, a) && !(a.vec_do && mapped(p.B, p.L, p.Hv, d.dout_stride)))
        return fail(EACS_ERR_INVALID, "%s: rows of dout must start on 16 bytes, with strides above 0, where those of q, k and v do", fn);
    const BSizes z = bwd_sizes(p, a);
    char* w = static_cast<char*>(ws);
    a.dS = w; w += z.dS;
    a.dV = w; w += z.dV;
    float* group = reinterpret_cast<float*>(w);
    cudaError_t e;
    if (planes(p, a)) {
        e = planes_bwd(a, const_cast<void*>(saved), ws, group, stream);
        if (e == cudaSuccess && a.half)
            e = p.K <= 64 ? run_grad<FmtF<true>, __half, 64>(a, group, stream) : run_grad<FmtF<true>, __half, 128>(a, group, stream);
    } else if (p.dtype == EACS_DTYPE_BF16)
        e = p.K <= 64 ? run_bwd<FmtF<true>, __nv_bfloat16, 64>(a, group, stream) : run_bwd<FmtF<true>, __nv_bfloat16, 128>(a, group, stream);
    else if (p.dtype == EACS_DTYPE_F16)
        e = p.K <= 64 ? run_bwd<FmtF<true>, __half, 64>(a, group, stream) : run_bwd<FmtF<true>, __half, 128>(a, group, stream);
    else
        e = p.K <= 64 ? run_bwd<FmtF<false>, float, 64>(a, group, stream) : run_bwd<FmtF<false>, float, 128>(a, group, stream);
    return cuda_check(e, fn);
}

}  // namespace eacs
