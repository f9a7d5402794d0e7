// row_common.cuh -- what the kernels over rows of features share (layer_norm.cu, block_norm.cu, conv.cu): vectors of
// elements, parameters as float32, sums over the threads of a row, grids, and the second kernel that adds partial rows.
#pragma once

#include <algorithm>

#include "eacs_common.cuh"
#include "eacs_host.h"

namespace eacs {
namespace {

__device__ __forceinline__ float read_param(const void* p, int dtype, int i, float none) {
    if (!p) return none;
    if (dtype == EACS_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == EACS_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// VEC elements moved as one access (16 bytes, or a single element)
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) RowVec { T e[VEC]; };

// The barrier of the TPR threads that share a row: the CTA's, or one of its own
// for each group (their numbers of rows may differ).
template <int TPR>
__device__ __forceinline__ void row_barrier() {
    if (TPR < static_cast<int>(blockDim.x))
        asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / TPR), "n"(TPR) : "memory");
    else
        __syncthreads();
}
// Sum over those threads; slot alternates so that one barrier a reduction is
// enough.  `red` is the group's own.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red, int& slot) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        float* r = red + slot * W;
        slot ^= 1;
        if ((threadIdx.x & 31) == 0) r[threadIdx.x / 32 % W] = v;
        row_barrier<TPR>();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += r[i];
    }
    return v;
}

// Weight (or bias, or scale) as float32.  In shared memory a thread's values of one vector
// are float4s that lie TPR apart: no two lanes meet in a bank.  With 512 threads
// a row a thread's share (at most 16 values) stays in its registers instead.
template <int VEC, int VPL, int TPR>
struct RowParam {
    static constexpr bool kShared = TPR < 512;
    static constexpr int E = VEC < 4 ? 1 : 4, Q = VEC / E;
    static constexpr int kFloats = kShared ? VPL * TPR * VEC : 4;
    float* s;
    float r[kShared ? 1 : VPL][VEC];
    __device__ __forceinline__ void fill(float* smem, const void* p, int dtype, int d, float none) {
        s = smem;
        if constexpr (kShared) {
            const int t = threadIdx.x % TPR;
            for (int k = threadIdx.x / TPR; k < VPL; k += blockDim.x / TPR)  // dealt to the CTA's groups
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = (k * TPR + t) * VEC + e;
                    s[((k * Q + e / E) * TPR + t) * E + e % E] = i < d ? read_param(p, dtype, i, none) : 0.f;
                }
        } else {
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = (k * TPR + static_cast<int>(threadIdx.x)) * VEC + e;
                    r[k][e] = i < d ? read_param(p, dtype, i, none) : 0.f;
                }
        }
    }
    __device__ __forceinline__ void get(float* v, int k, int t) const {
        if constexpr (!kShared) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = r[k][e];
        } else if constexpr (E == 4) {
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const float4 f = reinterpret_cast<const float4*>(s)[(k * Q + q) * TPR + t];
                v[4 * q] = f.x;
                v[4 * q + 1] = f.y;
                v[4 * q + 2] = f.z;
                v[4 * q + 3] = f.w;
            }
        } else {
            v[0] = s[k * TPR + t];
        }
    }
};

__device__ __forceinline__ void row_cp16(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}

// Columns of `rows` partial rows of `stride` floats: section i has n[i] columns from at[i] on, whose sums go to out[i]
// (or nowhere).
struct RowSums {
    const float* part;
    int64_t stride;
    int rows, dtype;
    void* out[3];
    int64_t at[3];
    int n[3];
};
// 32 columns a CTA (one a lane), the rows dealt to the 32 warps and their sums added in order.
__global__ void __launch_bounds__(1024) row_sums_k(const RowSums a) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + lane, d = a.n[blockIdx.y];
    void* out = a.out[blockIdx.y];
    if (!out || blockIdx.x * 32 >= d) return;
    const float* p = a.part + a.at[blockIdx.y] + i;
    float v = 0.f;
    if (i < d) {
#pragma unroll 8
        for (int r = wid; r < a.rows; r += 32) v += p[r * a.stride];
    }
    s[wid][lane] = v;
    __syncthreads();
    v = warp_sum(s[lane][wid]);  // column wid of this CTA
    const int c = blockIdx.x * 32 + wid;
    if (lane == 0 && c < d) {
        if (a.dtype == EACS_DTYPE_F32) static_cast<float*>(out)[c] = v;
        else if (a.dtype == EACS_DTYPE_F16) static_cast<__half*>(out)[c] = __float2half_rn(v);
        else static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(v);
    }
}
inline cudaError_t row_sums(const RowSums& a, int sections, cudaStream_t stream) {
    const int widest = std::max(a.n[0], std::max(a.n[1], a.n[2]));
    row_sums_k<<<dim3((widest + 31) / 32, sections), 1024, 0, stream>>>(a);
    note_launch();
    return cudaGetLastError();
}

// Grid: every row its group while the rows last, at most the CTAs that are
// resident at once (each then loops over rows, so that the weight is read and the
// sums are kept on the SM, and no second round of CTAs runs half empty).
template <typename K>
int row_resident(K kernel, int threads, size_t smem) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess) n = 1;
    return n < 1 ? 1 : n;
}
int row_grid(int64_t rows, int rpc, int per_sm) {
    return static_cast<int>(std::min<int64_t>((rows + rpc - 1) / rpc, int64_t{148} * per_sm));
}

}  // namespace
}  // namespace eacs
