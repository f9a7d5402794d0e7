// layer_norm.cu -- LayerNorm of x (+ residual) and its backward pass (sm_100a).
//
// For a row s = x (+ residual) of D values with mean m and (biased) variance w:
//   h = (s - m) / sqrt(w + eps),   y = h * weight + bias
// and for an upstream gradient dy, with p = dy * weight:
//   ds = (p - mean(p) - h mean(p h)) / sqrt(w + eps)    (d x = d residual = ds)
//   dweight = sum over rows of dy h,   dbias = sum over rows of dy.
// It is the norm of cst_ssm/modules/eacs.py:334 and of the training epilogue
// out_norm(x + fused) of cst_ssm/modules/multiscale.py:176-179.
//
// Both directions are bound by memory, so each reads its inputs once: a group
// of threads (a warp, or a CTA for wide rows) holds a row in registers, takes
// the mean and then the squared deviations from it (two passes over the
// registers: E[s^2] - m^2 would cancel), and writes its output.  The backward
// takes the row's statistics again from the row it has to read anyway, so the
// forward saves nothing.  Each thread owns the same columns in every row that
// its CTA visits and keeps the sums of dy h and dy there in float32 registers;
// a CTA writes one partial row of each, and a second kernel adds the partial
// rows in a fixed order (no atomics: the same inputs give the same bits).
#include <algorithm>

#include "eacs_common.cuh"
#include "eacs_host.h"

namespace eacs {
namespace {

template <typename T> __device__ __forceinline__ T ln_from_f32(float v);
template <> __device__ __forceinline__ float ln_from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half ln_from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 ln_from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

struct LnArgs {
    const void* x;
    const void* r;  // residual or null
    const void* w;  // or null (ones)
    const void* b;  // or null (zeros)
    void* y;        // forward: y; backward: ds
    const void* dy;
    float* part;    // backward: [CTAs][2][D] partial sums of dy h and dy, or null
    int64_t rows, sx, sr, sdy;  // row strides in elements (y is dense)
    int d, w_dtype;
    float eps;
};

__device__ __forceinline__ float ln_param(const void* p, int dtype, int i, float none) {
    if (!p) return none;
    if (dtype == EACS_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == EACS_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// VEC elements moved as one access (16 bytes, or a single element)
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) LnVec { T e[VEC]; };

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
    v = warp_sum(v);
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

// Three sums at once.  `red` is read a barrier before it is written again: the
// row's other sum lies between.
template <int TPR>
__device__ __forceinline__ void row_sums3(float* v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 3; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < 3; ++i) red[i * W + threadIdx.x / 32 % W] = v[i];
        row_barrier<TPR>();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v[i] += red[i * W + w];
        }
    }
}

// One row of an input as it lies in memory, elements (k TPR + t) VEC + e; kept so
// (16-bit values two to a register) and taken to float32 where they are used.
template <typename T, int VEC, int VPL, int TPR>
struct LnRow {
    LnVec<T, VEC> raw[VPL];
    __device__ __forceinline__ void read(const T* p, int d, int t) {
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int i0 = (k * TPR + t) * VEC;
            if (i0 < d) {
                raw[k] = *reinterpret_cast<const LnVec<T, VEC>*>(p + i0);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) raw[k].e[e] = ln_from_f32<T>(0.f);
            }
        }
    }
    __device__ __forceinline__ float at(int k, int e) const { return to_f32(raw[k].e[e]); }
};
// x, or x + residual (in float32: the sum is not rounded)
template <typename T, int VEC, int VPL, int TPR, bool RES>
struct LnSum {
    LnRow<T, VEC, VPL, TPR> x;
    float v[RES ? VPL : 1][VEC];
    __device__ __forceinline__ void set(const LnRow<T, VEC, VPL, TPR>& a, const LnRow<T, VEC, VPL, TPR>& r) {
        if constexpr (RES) {
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[k][e] = a.at(k, e) + r.at(k, e);
        } else {
            x = a;
        }
    }
    __device__ __forceinline__ float at(int k, int e) const {
        if constexpr (RES) return v[k][e];
        else return x.at(k, e);
    }
};

// Weight (or bias) as float32.  In shared memory a thread's values of one vector
// are float4s that lie TPR apart: no two lanes meet in a bank.  With 512 threads
// a row a thread's share (at most 16 values) stays in its registers instead.
template <int VEC, int VPL, int TPR>
struct LnParam {
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
                    s[((k * Q + e / E) * TPR + t) * E + e % E] = i < d ? ln_param(p, dtype, i, none) : 0.f;
                }
        } else {
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = (k * TPR + static_cast<int>(threadIdx.x)) * VEC + e;
                    r[k][e] = i < d ? ln_param(p, dtype, i, none) : 0.f;
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

// CTAs of RPC groups of TPR threads; a group takes every (grid RPC)th row.  Loads
// are kept in flight by the number of warps, not by reading a row ahead: that
// takes the registers of half the warps (measured on 65536 bf16 rows of 1024: 64
// us ahead, 49 without; the backward at 768: 144 and 72).
template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES, int CTAS>
__global__ void __launch_bounds__(TPR * RPC, CTAS) ln_fwd_k(LnArgs a) {
    using V = LnVec<T, VEC>;
    using Row = LnRow<T, VEC, VPL, TPR>;
    using Par = LnParam<VEC, VPL, TPR>;
    __shared__ float reds[RPC][2 * (TPR / 32)];
    __shared__ __align__(16) float sw[Par::kFloats], sb[Par::kFloats];
    Par w, b;
    int slot = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    float* red = reds[grp];
    const T* x = static_cast<const T*>(a.x);
    const T* r = static_cast<const T*>(a.r);
    const int64_t step = static_cast<int64_t>(gridDim.x) * RPC;
    int64_t row = static_cast<int64_t>(blockIdx.x) * RPC + grp;
    Row nx, nr;
    auto read = [&](int64_t i) {
        nx.read(x + i * a.sx, a.d, t);
        if constexpr (RES) nr.read(r + i * a.sr, a.d, t);
    };
    w.fill(sw, a.w, a.w_dtype, a.d, 1.f);
    b.fill(sb, a.b, a.w_dtype, a.d, 0.f);
    __syncthreads();
    const float inv = 1.0f / static_cast<float>(a.d);
    for (; row < a.rows; row += step) {
        read(row);
        LnSum<T, VEC, VPL, TPR, RES> s;
        s.set(nx, nr);
        float sum = 0.f, sq = 0.f;
#pragma unroll
        for (int k = 0; k < VPL; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += s.at(k, e);
        const float mean = row_sum<TPR>(sum, red, slot) * inv;
#pragma unroll
        for (int k = 0; k < VPL; ++k)
            if ((k * TPR + t) * VEC < a.d)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float c = s.at(k, e) - mean;
                    sq = fmaf(c, c, sq);
                }
        const float rstd = 1.0f / sqrtf(row_sum<TPR>(sq, red, slot) * inv + a.eps);
        T* y = static_cast<T*>(a.y) + row * a.d;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int i0 = (k * TPR + t) * VEC;
            if (i0 < a.d) {
                float wv[VEC], bv[VEC];
                w.get(wv, k, t);
                b.get(bv, k, t);
                V o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) o.e[e] = ln_from_f32<T>(fmaf((s.at(k, e) - mean) * rstd, wv[e], bv[e]));
                *reinterpret_cast<V*>(y + i0) = o;
            }
        }
    }
}

// Two rounds of sums a row: the mean, then with c = s - mean the squares of c,
// p and p c together.  A lane's 64 sums leave no registers to read a row ahead in
// (the forward's warps are many enough without), so rows of 16-byte vectors go
// through shared memory: a thread copies its own vectors of the next row there
// (cp.async, no barrier) while it works on this one.
template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES>
struct LnStage {
    static constexpr bool on = VEC > 1;
    static constexpr int kRow = VPL * TPR * 16, kRows = RES ? 3 : 2;  // bytes of a row, rows of a stage
    static constexpr size_t bytes = on ? static_cast<size_t>(RPC) * 2 * kRows * kRow : 0;
};

__device__ __forceinline__ void ln_cp16(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}

template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES, int CTAS>
__global__ void __launch_bounds__(TPR * RPC, CTAS) ln_bwd_k(LnArgs a) {
    using V = LnVec<T, VEC>;
    using Row = LnRow<T, VEC, VPL, TPR>;
    using Par = LnParam<VEC, VPL, TPR>;
    using St = LnStage<T, VEC, VPL, TPR, RPC, RES>;
    __shared__ float reds[RPC][5 * (TPR / 32)];
    __shared__ __align__(16) float sw[Par::kFloats];
    __shared__ float comb[RPC > 1 ? TPR * VPL * VEC : 1];
    extern __shared__ __align__(16) unsigned char stage[];
    Par w;
    int slot = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    float* red = reds[grp];
    const T* x = static_cast<const T*>(a.x);
    const T* r = static_cast<const T*>(a.r);
    const T* dy = static_cast<const T*>(a.dy);
    const int64_t step = static_cast<int64_t>(gridDim.x) * RPC;
    int64_t row = static_cast<int64_t>(blockIdx.x) * RPC + grp;
    // this thread's vectors of row j (0: x, 1: dy, 2: residual) of stage s
    auto at = [&](int s, int j, int k) {
        return reinterpret_cast<V*>(stage + (static_cast<size_t>(grp * 2 + s) * St::kRows + j) * St::kRow) + k * TPR + t;
    };
    auto fetch = [&](int s, int64_t i) {
        if constexpr (St::on) {
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                const int i0 = (k * TPR + t) * VEC;
                if (i < a.rows && i0 < a.d) {
                    ln_cp16(at(s, 0, k), x + i * a.sx + i0);
                    ln_cp16(at(s, 1, k), dy + i * a.sdy + i0);
                    if constexpr (RES) ln_cp16(at(s, 2, k), r + i * a.sr + i0);
                }
            }
            cp_async_commit();
        }
    };
    fetch(0, row);
    w.fill(sw, a.w, a.w_dtype, a.d, 1.f);
    __syncthreads();
    float dw[VPL][VEC], db[VPL][VEC];
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[k][e] = db[k][e] = 0.f;
    const float inv = 1.0f / static_cast<float>(a.d);
    for (int s = 0; row < a.rows; row += step, s ^= 1) {
        Row rx, rg, rr;  // (without stages)
        if constexpr (St::on) {
            fetch(s ^ 1, row + step);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            rx.read(x + row * a.sx, a.d, t);
            rg.read(dy + row * a.sdy, a.d, t);
            if constexpr (RES) rr.read(r + row * a.sr, a.d, t);
        }
        auto get_s = [&](int k, float* v) {
            V q, u;
            if constexpr (St::on) {
                q = *at(s, 0, k);
                if constexpr (RES) u = *at(s, 2, k);
            } else {
                q = rx.raw[k];
                if constexpr (RES) u = rr.raw[k];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[e] = to_f32(q.e[e]);
                if constexpr (RES) v[e] += to_f32(u.e[e]);
            }
        };
        auto get_g = [&](int k, float* v) {
            V q;
            if constexpr (St::on) q = *at(s, 1, k);
            else q = rg.raw[k];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = to_f32(q.e[e]);
        };
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < VPL; ++k)
            if ((k * TPR + t) * VEC < a.d) {
                float v[VEC];
                get_s(k, v);
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum += v[e];
            }
        const float mean = row_sum<TPR>(sum, red, slot) * inv;
        float q[3] = {};
#pragma unroll
        for (int k = 0; k < VPL; ++k)
            if ((k * TPR + t) * VEC < a.d) {
                float wv[VEC], v[VEC], g[VEC];
                w.get(wv, k, t);
                get_s(k, v);
                get_g(k, g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float c = v[e] - mean, p = g[e] * wv[e];
                    q[0] = fmaf(c, c, q[0]);
                    q[1] += p;
                    q[2] = fmaf(p, c, q[2]);
                }
            }
        row_sums3<TPR>(q, red + 2 * (TPR / 32));
        const float rstd = 1.0f / sqrtf(q[0] * inv + a.eps);
        const float s1 = q[1] * inv, s2 = q[2] * inv * rstd;
        T* dx = static_cast<T*>(a.y) + row * a.d;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int i0 = (k * TPR + t) * VEC;
            if (i0 < a.d) {
                float wv[VEC], v[VEC], g[VEC];
                w.get(wv, k, t);
                get_s(k, v);
                get_g(k, g);
                V o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float h = (v[e] - mean) * rstd;
                    dw[k][e] = fmaf(g[e], h, dw[k][e]);
                    db[k][e] += g[e];
                    o.e[e] = ln_from_f32<T>((fmaf(g[e], wv[e], -s1) - h * s2) * rstd);
                }
                *reinterpret_cast<V*>(dx + i0) = o;
            }
        }
    }
    if (!a.part) return;
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.d;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float(*acc)[VEC] = which ? db : dw;
        if constexpr (RPC > 1) {  // the CTA's groups one after another (a fixed order)
            for (int gi = 0; gi < RPC; ++gi) {
                __syncthreads();
                if (grp == gi)
#pragma unroll
                    for (int k = 0; k < VPL; ++k)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            float* c = comb + (k * VEC + e) * TPR + t;
                            *c = gi ? *c + acc[k][e] : acc[k][e];
                        }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < a.d; i += TPR * RPC) {
                const int k = i / (TPR * VEC), q = i - k * TPR * VEC;
                part[which * a.d + i] = comb[(k * VEC + q % VEC) * TPR + q / VEC];
            }
        } else {
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = (k * TPR + t) * VEC + e;
                    if (i < a.d) part[which * a.d + i] = acc[k][e];
                }
        }
    }
}

// dweight and dbias: sums of `n` partial rows, 32 columns a CTA (one a lane),
// the rows dealt to the 32 warps and their sums added in order.
__global__ void __launch_bounds__(1024) ln_reduce_k(const float* __restrict__ part, int n, int d, void* dw, void* db,
                                                    int w_dtype) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + lane;
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    const float* p = part + blockIdx.y * static_cast<int64_t>(d) + i;
    float v = 0.f;
    if (i < d) {
#pragma unroll 8
        for (int r = wid; r < n; r += 32) v += p[static_cast<int64_t>(r) * 2 * d];
    }
    s[wid][lane] = v;
    __syncthreads();
    v = warp_sum(s[lane][wid]);  // column wid of this CTA
    const int c = blockIdx.x * 32 + wid;
    if (lane == 0 && c < d) {
        if (w_dtype == EACS_DTYPE_F32) static_cast<float*>(out)[c] = v;
        else if (w_dtype == EACS_DTYPE_F16) static_cast<__half*>(out)[c] = __float2half_rn(v);
        else static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(v);
    }
}

constexpr int kLnMaxD = 8192;

// The backward's CTAs an SM at most: its grid is also the number of partial rows
// that the workspace holds and the second kernel adds.
constexpr int kLnBwdCtas = 6;
constexpr int kLnMaxParts = 148 * kLnBwdCtas;

// Grid: every row its group while the rows last, at most the CTAs that are
// resident at once (each then loops over rows, so that the weight is read and the
// sums are kept on the SM, and no second round of CTAs runs half empty).
template <typename K>
int ln_resident(K kernel, int threads, size_t smem) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess) n = 1;
    return n < 1 ? 1 : n;
}
int ln_grid(int64_t rows, int rpc, int per_sm) {
    return static_cast<int>(std::min<int64_t>((rows + rpc - 1) / rpc, int64_t{148} * per_sm));
}

template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES>
cudaError_t ln_fwd_launch(const LnArgs& a, cudaStream_t s) {
    // registers for three CTAs an SM where a lane keeps its sums of two rows in float32
    constexpr int ctas = RPC == 1 || !RES ? 1 : 3;
    static const int per = ln_resident(ln_fwd_k<T, VEC, VPL, TPR, RPC, RES, ctas>, TPR * RPC, 0);
    ln_fwd_k<T, VEC, VPL, TPR, RPC, RES, ctas><<<ln_grid(a.rows, RPC, per), TPR * RPC, 0, s>>>(a);
    note_launch();
    return cudaGetLastError();
}

template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES>
cudaError_t ln_bwd_launch(const LnArgs& a, int* parts, cudaStream_t s) {
    constexpr int ctas = VEC * VPL <= 8 ? 4 : 2;
    constexpr size_t smem = LnStage<T, VEC, VPL, TPR, RPC, RES>::bytes;
    const auto k = ln_bwd_k<T, VEC, VPL, TPR, RPC, RES, ctas>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    static const int per = std::min(ln_resident(k, TPR * RPC, smem), kLnBwdCtas);
    *parts = ln_grid(a.rows, RPC, per);
    k<<<*parts, TPR * RPC, smem, s>>>(a);
    note_launch();
    return cudaGetLastError();
}

// A warp a row while a lane's share fits its registers (forward: the row itself,
// 128 bytes; backward: the sums of 32 columns), then as many threads as that
// share asks for.  Rows whose start or length is not a multiple of 16 bytes are
// read element by element.
template <typename T>
cudaError_t ln_dispatch(const LnArgs& a, bool vec, bool bwd, int* parts, cudaStream_t s) {
    constexpr int E = 16 / sizeof(T);
#define EACS_LN_FWD(VEC, VPL, TPR, RPC)                                \
    return a.r ? ln_fwd_launch<T, VEC, VPL, TPR, RPC, true>(a, s)      \
               : ln_fwd_launch<T, VEC, VPL, TPR, RPC, false>(a, s)
#define EACS_LN_BWD(VEC, VPL, TPR, RPC)                                \
    return a.r ? ln_bwd_launch<T, VEC, VPL, TPR, RPC, true>(a, parts, s) \
               : ln_bwd_launch<T, VEC, VPL, TPR, RPC, false>(a, parts, s)
    const int n = (a.d + E - 1) / E;  // 16-byte vectors a row
    if (vec && !bwd) {
        if (n <= 32) EACS_LN_FWD(E, 1, 32, 8);
        if (n <= 64) EACS_LN_FWD(E, 2, 32, 8);
        if (n <= 96) EACS_LN_FWD(E, 3, 32, 8);
        if (n <= 128) EACS_LN_FWD(E, 4, 32, 8);
        if (n <= 256) EACS_LN_FWD(E, 8, 32, 8);
        if (n <= 512) EACS_LN_FWD(E, 4, 128, 2);
        if (n <= 1024) EACS_LN_FWD(E, 2, 512, 1);
        if constexpr (E == 4) EACS_LN_FWD(E, 4, 512, 1);  // (16-bit rows of 8192 values have 1024 vectors)
    }
    if (vec) {
        if (n <= 32) EACS_LN_BWD(E, 1, 32, 8);
        if (n <= 64) EACS_LN_BWD(E, 2, 32, 8);
        if (n <= 96) EACS_LN_BWD(E, 3, 32, 8);
        if (n <= 128) EACS_LN_BWD(E, 4, 32, 8);
        if (n <= 256) EACS_LN_BWD(E, 4, 64, 4);
        if (n <= 512) EACS_LN_BWD(E, 4, 128, 2);
        if (n <= 1024) EACS_LN_BWD(E, 2, 512, 1);
        if constexpr (E == 4) EACS_LN_BWD(E, 4, 512, 1);
    }
    if (!bwd) {
        if (a.d <= 256) EACS_LN_FWD(1, 8, 32, 8);
        if (a.d <= 512) EACS_LN_FWD(1, 16, 32, 8);
        if (a.d <= 1024) EACS_LN_FWD(1, 16, 64, 4);
        if (a.d <= 4096) EACS_LN_FWD(1, 8, 512, 1);
        EACS_LN_FWD(1, 16, 512, 1);
    }
    if (a.d <= 256) EACS_LN_BWD(1, 8, 32, 8);
    if (a.d <= 512) EACS_LN_BWD(1, 16, 32, 8);
    if (a.d <= 1024) EACS_LN_BWD(1, 16, 64, 4);
    if (a.d <= 4096) EACS_LN_BWD(1, 8, 512, 1);
    EACS_LN_BWD(1, 16, 512, 1);
#undef EACS_LN_FWD
#undef EACS_LN_BWD
}

}  // namespace

size_t layer_norm_bwd_workspace_size(int64_t rows, int64_t d) {
    if (rows <= 0 || d <= 0 || d > kLnMaxD) return 0;
    return static_cast<size_t>(std::min<int64_t>(rows, kLnMaxParts)) * 2 * d * sizeof(float);
}

int layer_norm(const LayerNormCall& c, cudaStream_t stream) {
    const char* fn = c.backward ? "eacs_layer_norm_bwd" : "eacs_layer_norm_fwd";
    if (c.rows < 0 || c.d <= 0) return fail(EACS_ERR_INVALID, "%s: bad sizes", fn);
    if (c.d > kLnMaxD) return fail(EACS_ERR_UNSUPPORTED, "%s: d=%lld > %d", fn, (long long)c.d, kLnMaxD);
    for (int dt : {c.dtype, c.w_dtype})
        if (dt != EACS_DTYPE_F32 && dt != EACS_DTYPE_F16 && dt != EACS_DTYPE_BF16)
            return fail(EACS_ERR_INVALID, "%s: unknown dtype %d", fn, dt);
    if (c.rows > 0 && (!c.x || !c.out || (c.backward && !c.dy))) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    if (c.x_stride < c.d || (c.residual && c.r_stride < c.d) || (c.dy && c.dy_stride < c.d))
        return fail(EACS_ERR_INVALID, "%s: a row stride is below d", fn);
    const bool want = c.backward && (c.dweight || c.dbias);
    const size_t need = want ? layer_norm_bwd_workspace_size(c.rows, c.d) : 0;
    if (want && c.rows > 0 && (!c.workspace || c.workspace_bytes < need))
        return fail(EACS_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, c.workspace_bytes, need);
    const int esz = c.dtype == EACS_DTYPE_F32 ? 4 : 2;
    const size_t wsz = c.w_dtype == EACS_DTYPE_F32 ? 4 : 2;
    if (c.rows == 0) {  // empty sums
        cudaError_t e = cudaSuccess;
        if (c.dweight) e = cudaMemsetAsync(c.dweight, 0, wsz * c.d, stream);
        if (e == cudaSuccess && c.dbias) e = cudaMemsetAsync(c.dbias, 0, wsz * c.d, stream);
        return cuda_check(e, fn);
    }
    LnArgs a{};
    a.x = c.x;
    a.r = c.residual;
    a.w = c.weight;
    a.b = c.bias;
    a.y = c.out;
    a.dy = c.dy;
    a.part = want ? static_cast<float*>(c.workspace) : nullptr;
    a.rows = c.rows;
    a.sx = c.x_stride;
    a.sr = c.r_stride;
    a.sdy = c.dy_stride;
    a.d = static_cast<int>(c.d);
    a.w_dtype = c.w_dtype;
    a.eps = c.eps;
    auto rows16 = [&](const void* p, int64_t stride) {
        return !p || ((reinterpret_cast<uintptr_t>(p) | (static_cast<uintptr_t>(stride) * esz)) & 15u) == 0;
    };
    const bool vec = rows16(c.x, c.x_stride) && rows16(c.residual, c.r_stride) && rows16(c.dy, c.dy_stride) &&
                     rows16(c.out, c.d);
    int parts = 0;
    cudaError_t e;
    if (c.dtype == EACS_DTYPE_F16) e = ln_dispatch<__half>(a, vec, c.backward, &parts, stream);
    else if (c.dtype == EACS_DTYPE_BF16) e = ln_dispatch<__nv_bfloat16>(a, vec, c.backward, &parts, stream);
    else e = ln_dispatch<float>(a, vec, c.backward, &parts, stream);
    if (e == cudaSuccess && want) {
        ln_reduce_k<<<dim3((a.d + 31) / 32, 2), 1024, 0, stream>>>(a.part, parts, a.d, c.dweight, c.dbias, c.w_dtype);
        note_launch();
        e = cudaGetLastError();
    }
    return cuda_check(e, fn);
}

}  // namespace eacs
