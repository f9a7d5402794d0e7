// delta_common.cuh -- what the gated delta rule's kernels share (delta.cu, delta_planes.cu).
#pragma once

#include <cuda_runtime.h>

#include "eacs_common.cuh"
#include "eacs_host.h"

namespace eacs {

constexpr int kC = 64;           // tokens per chunk
constexpr int kGates = 5 * kC;   // floats of a chunk's gates
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
__device__ __forceinline__ void ldsm4(uint32_t* r, const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p)));
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p)));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t to_tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = to_tf32(x);
    lo = to_tf32(x - __uint_as_float(hi));
}

// Lane coordinates: an accumulator tile (16 x 8) holds rows g, g + 8 and
// columns 2t, 2t + 1 as c[0], c[1] and c[2], c[3].
struct Lane {
    int l, g, t;
    __device__ __forceinline__ Lane() : l(threadIdx.x & 31), g(l >> 2), t(l & 3) {}
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
    int vec_qk, vec_v, vec_do;  // rows can be read 16 bytes at a time
    float scale;
    // workspace, per chunk id ((b Hv + h) n + c)
    float* gates;  // [id][5][64]: G (high), G (low), gam, d, scale gam
    void* T;       // [id][planes][64][64]
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

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(valid ? 16 : 0)
                 : "memory");
}
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



}  // namespace eacs
