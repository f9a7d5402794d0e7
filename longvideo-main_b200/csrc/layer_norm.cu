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

// Sum over the TPR threads that share a row; slot alternates so that one
// barrier a reduction is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red, int& slot) {
    v = warp_sum(v);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        float* r = red + slot * W;
        slot ^= 1;
        if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += r[i];
    }
    return v;
}

// Row s of the group as floats: elements (k TPR + t) VEC + e, zero past d.
template <typename T, int VEC, int VPL, int TPR, bool RES>
__device__ __forceinline__ void ln_load(const LnArgs& a, const T* base, int64_t stride, const T* rbase,
                                        int64_t row, int t, float (*v)[VEC]) {
    using V = LnVec<T, VEC>;
    const T* p = base + row * stride;
    V raw[VPL], rr[VPL];
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        const int i0 = (k * TPR + t) * VEC;
        if (i0 < a.d) raw[k] = *reinterpret_cast<const V*>(p + i0);
    }
    if constexpr (RES) {
        const T* q = rbase + row * a.sr;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int i0 = (k * TPR + t) * VEC;
            if (i0 < a.d) rr[k] = *reinterpret_cast<const V*>(q + i0);
        }
    }
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        const bool in = (k * TPR + t) * VEC < a.d;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            v[k][e] = in ? to_f32(raw[k].e[e]) : 0.f;
            if constexpr (RES) v[k][e] += in ? to_f32(rr[k].e[e]) : 0.f;
        }
    }
}

template <int VEC, int VPL, int TPR>
__device__ __forceinline__ void ln_stats(const LnArgs& a, const float (*v)[VEC], int t, float* red, int& slot,
                                         float& mean, float& rstd) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += v[k][e];
    mean = row_sum<TPR>(s, red, slot) / static_cast<float>(a.d);
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < VPL; ++k)
        if ((k * TPR + t) * VEC < a.d)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float c = v[k][e] - mean;
                q = fmaf(c, c, q);
            }
    rstd = 1.0f / sqrtf(row_sum<TPR>(q, red, slot) / static_cast<float>(a.d) + a.eps);
}

// CTA of RPC groups of TPR threads, each group one row at a time.
template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES>
__global__ void __launch_bounds__(TPR * RPC) ln_fwd_k(LnArgs a) {
    using V = LnVec<T, VEC>;
    __shared__ float red[2 * (TPR / 32)];
    int slot = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    float w[VPL][VEC], b[VPL][VEC];
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int i = (k * TPR + t) * VEC + e;
            w[k][e] = i < a.d ? ln_param(a.w, a.w_dtype, i, 1.f) : 0.f;
            b[k][e] = i < a.d ? ln_param(a.b, a.w_dtype, i, 0.f) : 0.f;
        }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * RPC + grp; row < a.rows;
         row += static_cast<int64_t>(gridDim.x) * RPC) {
        float v[VPL][VEC], mean, rstd;
        ln_load<T, VEC, VPL, TPR, RES>(a, static_cast<const T*>(a.x), a.sx, static_cast<const T*>(a.r), row, t, v);
        ln_stats<VEC, VPL, TPR>(a, v, t, red, slot, mean, rstd);
        T* y = static_cast<T*>(a.y) + row * a.d;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int i0 = (k * TPR + t) * VEC;
            if (i0 < a.d) {
                V o;
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    o.e[e] = ln_from_f32<T>(fmaf((v[k][e] - mean) * rstd, w[k][e], b[k][e]));
                *reinterpret_cast<V*>(y + i0) = o;
            }
        }
    }
}

template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES>
__global__ void __launch_bounds__(TPR * RPC) ln_bwd_k(LnArgs a) {
    using V = LnVec<T, VEC>;
    __shared__ float red[2 * (TPR / 32)];
    __shared__ float comb[RPC > 1 ? TPR * VPL * VEC : 1];
    int slot = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    float w[VPL][VEC], dw[VPL][VEC], db[VPL][VEC];
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int i = (k * TPR + t) * VEC + e;
            w[k][e] = i < a.d ? ln_param(a.w, a.w_dtype, i, 1.f) : 0.f;
            dw[k][e] = db[k][e] = 0.f;
        }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * RPC + grp; row < a.rows;
         row += static_cast<int64_t>(gridDim.x) * RPC) {
        float v[VPL][VEC], gy[VPL][VEC], mean, rstd;
        ln_load<T, VEC, VPL, TPR, RES>(a, static_cast<const T*>(a.x), a.sx, static_cast<const T*>(a.r), row, t, v);
        ln_load<T, VEC, VPL, TPR, false>(a, static_cast<const T*>(a.dy), a.sdy, nullptr, row, t, gy);
        ln_stats<VEC, VPL, TPR>(a, v, t, red, slot, mean, rstd);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < VPL; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float h = (v[k][e] - mean) * rstd;  // past d: gy and w are 0, h does not count
                v[k][e] = h;
                dw[k][e] = fmaf(gy[k][e], h, dw[k][e]);
                db[k][e] += gy[k][e];
                const float p = gy[k][e] * w[k][e];
                gy[k][e] = p;
                s1 += p;
                s2 = fmaf(p, h, s2);
            }
        s1 = row_sum<TPR>(s1, red, slot) / static_cast<float>(a.d);
        s2 = row_sum<TPR>(s2, red, slot) / static_cast<float>(a.d);
        T* dx = static_cast<T*>(a.y) + row * a.d;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int i0 = (k * TPR + t) * VEC;
            if (i0 < a.d) {
                V o;
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    o.e[e] = ln_from_f32<T>((gy[k][e] - s1 - v[k][e] * s2) * rstd);
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
    if (i < d)
        for (int r = wid; r < n; r += 32) v += p[static_cast<int64_t>(r) * 2 * d];
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

// The largest grid of the backward: also the number of partial rows that the
// workspace is sized for.
constexpr int kLnMaxParts = 148 * 4;

template <typename T, int VEC, int VPL, int TPR, int RPC>
cudaError_t ln_launch(const LnArgs& a, bool bwd, int grid, cudaStream_t s) {
    if (bwd) {
        if (a.r) ln_bwd_k<T, VEC, VPL, TPR, RPC, true><<<grid, TPR * RPC, 0, s>>>(a);
        else ln_bwd_k<T, VEC, VPL, TPR, RPC, false><<<grid, TPR * RPC, 0, s>>>(a);
    } else {
        if (a.r) ln_fwd_k<T, VEC, VPL, TPR, RPC, true><<<grid, TPR * RPC, 0, s>>>(a);
        else ln_fwd_k<T, VEC, VPL, TPR, RPC, false><<<grid, TPR * RPC, 0, s>>>(a);
    }
    note_launch();
    return cudaGetLastError();
}

// Grid: every row its group while the rows last, at most `per_sm` CTAs an SM
// (each then loops over rows, so that weight and sums are kept in registers).
int ln_grid(int64_t rows, int rpc, int per_sm) {
    const int64_t want = (rows + rpc - 1) / rpc;
    return static_cast<int>(std::min<int64_t>(want, 148 * per_sm));
}

// A warp a row while a lane's share is at most 32 values, then 128 and 512
// threads a row.  Rows whose start or length is not a multiple of 16 bytes are
// read element by element.
template <typename T>
cudaError_t ln_dispatch(const LnArgs& a, bool vec, bool bwd, int* parts, cudaStream_t s) {
    constexpr int E = 16 / sizeof(T);
    const int per = bwd ? 4 : 8;
#define EACS_LN(VEC, VPL, TPR, RPC)                                    \
    do {                                                               \
        *parts = ln_grid(a.rows, RPC, per);                            \
        return ln_launch<T, VEC, VPL, TPR, RPC>(a, bwd, *parts, s);    \
    } while (0)
    if (vec) {
        const int n = (a.d + E - 1) / E;  // 16-byte vectors a row
        if (n <= 32) EACS_LN(E, 1, 32, 8);
        if (n <= 64) EACS_LN(E, 2, 32, 8);
        if (n <= 96) EACS_LN(E, 3, 32, 8);
        if (n <= 128) EACS_LN(E, 4, 32, 8);
        if (n <= 256) EACS_LN(E, 2, 128, 1);
        if (n <= 512) EACS_LN(E, 4, 128, 1);
        if (n <= 1024) EACS_LN(E, 2, 512, 1);
        EACS_LN(E, 4, 512, 1);
    }
    if (a.d <= 256) EACS_LN(1, 8, 32, 8);
    if (a.d <= 1024) EACS_LN(1, 8, 128, 1);
    if (a.d <= 4096) EACS_LN(1, 8, 512, 1);
    EACS_LN(1, 16, 512, 1);
#undef EACS_LN
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
