// delta_common.cuh -- what the gated delta rule's kernels share (delta.cu, delta_planes.cu).
#pragma once

#include <cuda_runtime.h>

#include "eacs_common.cuh"
#include "eacs_host.h"

namespace eacs {

constexpr int kC = 64;           // tokens per chunk
constexpr int kGates = 6 * kC;   // floats of a chunk's gates
constexpr int kTld = kC + 8;     // row stride of a 64-column tile in shared memory
constexpr float kBetaMin = 5.421010862427522e-20f;  // 2^-64

// Matrix instructions of a warp; sums are float32 always.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(p));
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(p));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (not volatile: the products of several tiles can be interleaved)
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32_first(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {  // c = a b
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// x = hi + lo in tf32 (11 significant bits each): hi to the nearest, lo cut off,
// of either sign, so x is off by at most 2^-22 of itself.  In integer operations:
// the conversion instruction runs at a fraction of their rate (the chains took
// a fifth longer, delta_out_k half).  A NaN whose bits the addition overflows is
// still one in lo.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

// Lane coordinates: an accumulator tile (16 x 8) holds rows g, g + 8 and
// columns 2t, 2t + 1 as c[0], c[1] and c[2], c[3].
struct Lane {
    int l, g, t;
    __device__ __forceinline__ Lane() : l(threadIdx.x & 31), g(l >> 2), t(l & 3) {}
};

// Operands are tf32 split in two (hi lo' + lo hi' + hi hi': 22 bits).  A tile is
// float32 in shared memory and is split as it is read.  Af<P>: a 16 x 16 A
// operand.  Tiles of B are 16 columns (two accumulators) by 16 of the summed
// index, stored [n][k] or (TR) [k][n].
// X: the inputs (queries, keys, upstream gradients) are exact in tf32, as
// float16 values are: their low part is 0 and is left out.
template <bool X>
struct FmtF {
    using E = float;
    template <int P> struct Af { uint32_t h[2][4], lo[2][4]; };
    static __device__ __forceinline__ E put(float v) { return v; }
    static __device__ __forceinline__ void set(Af<2>& a, int s, int i, float v) { split_tf32(v, a.h[s][i], a.lo[s][i]); }
    // the summed index runs 2t, 2t + 1 inside an accumulator tile; A and B use the same order
    template <int P>
    static __device__ __forceinline__ Af<P> from_acc(const float* c0, const float* c1) {
        Af<P> a;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const float* c = s ? c1 : c0;
            split_tf32(c[0], a.h[s][0], a.lo[s][0]);
            split_tf32(c[2], a.h[s][1], a.lo[s][1]);
            split_tf32(c[1], a.h[s][2], a.lo[s][2]);
            split_tf32(c[3], a.h[s][3], a.lo[s][3]);
        }
        return a;
    }
    static __device__ __forceinline__ Af<1> from_smem(const E* s, int ld, int m0, int k0) {
        const Lane L;
        Af<1> a;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 p = *reinterpret_cast<const float2*>(s + (m0 + L.g) * ld + k0 + 8 * h + 2 * L.t);
            const float2 q = *reinterpret_cast<const float2*>(s + (m0 + L.g + 8) * ld + k0 + 8 * h + 2 * L.t);
            split_tf32(p.x, a.h[h][0], a.lo[h][0]);
            split_tf32(q.x, a.h[h][1], a.lo[h][1]);
            split_tf32(p.y, a.h[h][2], a.lo[h][2]);
            split_tf32(q.y, a.h[h][3], a.lo[h][3]);
        }
        return a;
    }
    static __device__ __forceinline__ Af<1> from_smem_t(const E* s, int ld, int m0, int k0) {
        const Lane L;
        Af<1> a;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                split_tf32(s[(k0 + 8 * h + 2 * L.t + (i >> 1)) * ld + m0 + L.g + (i & 1) * 8], a.h[h][i], a.lo[h][i]);
        return a;
    }
    static __device__ __forceinline__ void scale_k(Af<1>& a, const float* f, int k0) {
        const int t = threadIdx.x & 3;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = __uint_as_float(a.h[h][i]) + __uint_as_float(a.lo[h][i]);
                split_tf32(v * f[k0 + 8 * h + 2 * t + (i >> 1)], a.h[h][i], a.lo[h][i]);
            }
    }
    // IN: B is a tile of inputs.  The products of a step are summed apart, in four
    // chains of three that hide each other's latency, and added in float32: the
    // matrix instruction's own sum is cut off, not rounded, and a state that
    // takes hundreds of steps drifted by it (6e-6 of its norm instead of 3e-7).
    template <int P, bool TR, bool IN = false>
    static __device__ __forceinline__ void mma2(float* c0, float* c1, const Af<P>& a, const E* s, int ld, int n0,
                                                int k0) {
        const Lane L;
        float x[4][4];
        uint32_t hi[4][2], lo[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // i: 8 columns, 8 of the summed index
            const int n = n0 + 8 * (i >> 1) + L.g, k = k0 + 8 * (i & 1) + 2 * L.t;
            float2 v;
            if constexpr (TR) v = make_float2(s[k * ld + n], s[(k + 1) * ld + n]);
            else v = *reinterpret_cast<const float2*>(s + n * ld + k);
            if constexpr (X && IN) {
                hi[i][0] = __float_as_uint(v.x);
                hi[i][1] = __float_as_uint(v.y);
            } else {
                split_tf32(v.x, hi[i][0], lo[i][0]);
                split_tf32(v.y, hi[i][1], lo[i][1]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) mma_tf32_first(x[i], a.lo[i & 1], hi[i][0], hi[i][1]);
        if constexpr (!(X && IN)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) mma_tf32(x[i], a.h[i & 1], lo[i][0], lo[i][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) mma_tf32(x[i], a.h[i & 1], hi[i][0], hi[i][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c0[e] += x[0][e] + x[1][e];
            c1[e] += x[2][e] + x[3][e];
        }
    }
    static __device__ __forceinline__ void load_t(float* x0, float* x1, const E* s, int ld, int r0, int c0) {
        const Lane L;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* x = h ? x1 : x0;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = s[(c0 + 8 * h + 2 * L.t + (i & 1)) * ld + r0 + L.g + (i >> 1) * 8];
        }
    }
};

// ----------------------------------------------------------------------------
// arguments and the workspace
// ----------------------------------------------------------------------------
struct Str { int64_t b, t, h; };  // element strides over batch, token, head

struct DArgs {
    const void *q, *k, *v, *g, *beta, *dout;
    Str sq, sk, sv, sg, sb, sdo;
    const int* lengths;
    const float* initial;  // (B,Hv,K,V) or null
    float* final_state;    // or null
    void* out;             // (B,L,Hv,V)
    void *dq, *dk, *dv, *dg, *dbeta;
    const float* dfinal;   // or null
    float* dinitial;       // or null
    int B, L, Hk, Hv, K, V, n, Vp;  // n chunks, Vp = V rounded up to 16
    int gate_dtype;
    int half;  // q, k, v: float16
    int vec_qk, vec_v, vec_do;  // rows can be read 16 bytes at a time
    float scale;
    // workspace, per chunk id ((b Hv + h) n + c)
    float* gates;  // [id][6][64]: G (high), G (low), gam, d, scale gam, 1 / beta (delta_planes.cu; with float16 beta)
    void* T;       // [id][planes][64][64]
    void* Tr;      // (float16 training, delta_planes.cu) the reverse chain's
    void* M;       // [id][64][64] or null
    void* S;       // [id][Vp][KD]: S0^T or null
    void* U;       // [id][64][Vp]
    void* dS;      // [id][Vp][KD]: dS1^T
    void* dV;      // [id][64][Vp]
};

__device__ __forceinline__ int row_length(const DArgs& a, int b) {
    if (!a.lengths) return a.L;
    return min(max(a.lengths[b], 0), a.L);
}
__device__ __forceinline__ float gate_value(const void* p, int dtype, int64_t i) {
    if (dtype == EACS_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == EACS_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void gate_store(void* p, int dtype, int64_t i, float v) {
    if (dtype == EACS_DTYPE_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == EACS_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float hold_beta(float b) { return fabsf(b) < kBetaMin ? kBetaMin : b; }

template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T> __device__ __forceinline__ void load8(const T* p, float* v);
template <> __device__ __forceinline__ void load8<float>(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float* v) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float* v) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t* h = reinterpret_cast<const uint32_t*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// S^T (16 value rows v0.., K columns) of a (K, V) float32 state, or zeros
template <int KD>
__device__ __forceinline__ void state_load(float (*S)[4], const float* p, int K, int V, int v0, const Lane& L) {
    if (p) {
#pragma unroll
        for (int j = 0; j < KD / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = 8 * j + 2 * L.t + (e & 1), v = v0 + L.g + (e >> 1) * 8;
                S[j][e] = k < K && v < V ? p[static_cast<int64_t>(k) * V + v] : 0.f;
            }
    } else {
#pragma unroll
        for (int j = 0; j < KD / 8; ++j) S[j][0] = S[j][1] = S[j][2] = S[j][3] = 0.f;
    }
}
template <int KD>
__device__ __forceinline__ void state_store(const float (*S)[4], float* p, int K, int V, int v0, const Lane& L) {
#pragma unroll
    for (int j = 0; j < KD / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = 8 * j + 2 * L.t + (e & 1), v = v0 + L.g + (e >> 1) * 8;
            if (k < K && v < V) p[static_cast<int64_t>(k) * V + v] = S[j][e];
        }
}

template <typename K>
cudaError_t smem_limit(K kernel, size_t bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

#define DELTA_TRY(x)                          \
    do {                                      \
        const cudaError_t e_ = (x);           \
        if (e_ != cudaSuccess) return e_;     \
    } while (0)

// delta_planes.cu: 16-bit inputs whose rows start on 16 bytes
size_t planes_saved_size(const DArgs& a, bool training);
size_t planes_bwd_size(const DArgs& a);
cudaError_t planes_fwd(DArgs a, void* ws, bool training, cudaStream_t s);
// float16: up to dS and dV, which are set in `a` with what the forward kept
cudaError_t planes_bwd(DArgs& a, void* saved, void* ws, float* group, cudaStream_t s);
cudaError_t planes_read_status(int* out, cudaStream_t s);

}  // namespace eacs
