// block_norm.cu -- the norms before and after a block, with its gate and its scaled residual, and their gradients (sm_100a).
//
// With r(v) = 1 / sqrt(mean(v^2) + eps) over a row of d values (float32):
//   u = x, or x r(x) post;   u = u silu(gate) where there is a gate;
//   without a residual y = u;  with one  s = residual + scale u,  y = s r(s) weight,  and s is written too.
// Gradients, from dy and ds, with the gradient of v from that of v r(v) = h:  N(q; v) = r (q - v r^2 mean(q v)):
//   dv = ds + N(dy weight; s) (= d residual),  dweight = sum dy s r(s),  dscale = sum dv u,  du = dv scale
//   dgate = du u' silu'(gate),  u' the value before the gate;  du' = du silu(gate)
//   dx = N(du' post; x),  dpost = sum du' x r(x)      (sums over the rows).
//
// Bound by memory: a row is read once into the registers of its threads (a part of a warp, a warp or several) and written
// once; s is never rounded before its norm.  The backward takes everything again from the forward's inputs, so the forward
// saves nothing.  Sums over rows are kept in float32 registers, a thread's own columns; a CTA writes one partial row and a
// second kernel adds them in order (no atomics: the same inputs give the same bits).
// Measured, us (bytes' time in brackets): 65536 x 768 bfloat16 with a scale, forward 62 (62), backward 104 (92) + 8 for the
// sums; heads of 128, 131072 of them, gated 20 (15).  The residual's backward spills registers above 4096 values (96 to 1156
// bytes a thread) and, with gate and post norm together, in 16-bit rows of 129 to 256 (164 to 180); elsewhere at most 28 bytes.
// What there is of gate and post norm is known at compile time for every width of aligned rows: a backward that asks at run
// time holds registers for all of it (with the next row's way through shared memory that took a training step of 65536 x 768
// with a scale from 392 us to 200).
#include <algorithm>

#include "eacs_common.cuh"
#include "eacs_host.h"
#include "row_common.cuh"

namespace eacs {
namespace {

constexpr int kBnMaxD = 8192;

struct BnArgs {
    const void *x, *gate, *res;
    const void *weight, *scale, *post;  // each may be null (ones); post counts only where has_post
    void *y, *s;
    const void *dy, *ds;                // backward; either may be null (zeros)
    void *dx, *dgate, *dres;            // dres null: it is dx
    float* part;                        // [CTAs][3][d] sums for weight, scale and post, or null
    int64_t rows, sx, sg, sr, sdy, sds;
    int d, w_dtype, has_post;
    float eps;
};

// One row of an input: VPL vectors a thread, as they lie in memory (whole registers), taken apart where they are used.
template <typename T, int VEC, int VPL, int TPR>
struct BnRow {
    static constexpr int kPer = VEC > 1 ? 4 / sizeof(T) : 1, kWords = VEC / kPer;  // elements a word; words a vector
    uint32_t raw[VPL][kWords];
    __device__ __forceinline__ void load(int k, const void* p) {
        if constexpr (VEC > 1) {
            const uint4 q = *static_cast<const uint4*>(p);
            raw[k][0] = q.x, raw[k][1] = q.y, raw[k][2] = q.z, raw[k][3] = q.w;
        } else if constexpr (sizeof(T) == 4) {
            raw[k][0] = *static_cast<const uint32_t*>(p);
        } else {
            raw[k][0] = *static_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ void zero(int k) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[k][i] = 0;
    }
    __device__ __forceinline__ void read(const T* p, int d, int t) {
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int i0 = (k * TPR + t) * VEC;
            if (i0 < d) load(k, p + i0);
            else zero(k);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int k = 0; k < VPL; ++k) zero(k);
    }
    __device__ __forceinline__ float at(int k, int e) const {
        float a, b;
        unpack<T>(raw[k][e / kPer], a, b);
        return e % kPer ? b : a;
    }
};
template <typename T, int VEC>
__device__ __forceinline__ void bn_write(T* p, const float* v) {
    if constexpr (VEC > 1) {
        constexpr int per = 4 / sizeof(T);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack<T>(v[i * per], v[i * per + per - 1]);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        p[0] = from_f32<T>(v[0]);
    }
}

// CTAs of RPC groups of TPR threads; a group takes every (grid RPC)th row.  Groups smaller than a warp go through their
// rows together (their sums are the warp's shuffles): a group without a row reads and writes nothing.
// HOW: what there is of gate (1) and post norm (2); 4: the arguments say (rows read element by element).
template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES, int HOW>
__global__ void __launch_bounds__(TPR * RPC) bn_fwd_k(const BnArgs a) {
    const bool gated = HOW == 4 ? a.gate != nullptr : (HOW & 1) != 0, normed = HOW == 4 ? a.has_post != 0 : (HOW & 2) != 0;
    using Row = BnRow<T, VEC, VPL, TPR>;
    using Par = RowParam<VEC, VPL, TPR>;
    __shared__ float reds[RPC][2 * (TPR / 32) + 1];
    __shared__ __align__(16) float sw[Par::kFloats], sp[Par::kFloats], sc[RES ? Par::kFloats : 4];
    Par w, post, scale;
    int slot = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    float* red = reds[grp];
    if constexpr (RES) {
        w.fill(sw, a.weight, a.w_dtype, a.d, 1.f);
        scale.fill(sc, a.scale, a.w_dtype, a.d, 1.f);
    }
    if (normed) post.fill(sp, a.post, a.w_dtype, a.d, 1.f);
    __syncthreads();
    const float inv = 1.0f / static_cast<float>(a.d);
    const int64_t step = static_cast<int64_t>(gridDim.x) * RPC;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * RPC + grp;; row += step) {
        const bool live = row < a.rows;
        if (TPR < 32 ? !__any_sync(0xffffffffu, live) : !live) break;
        const int dl = live ? a.d : 0;
        Row x, g, r;
        x.read(static_cast<const T*>(a.x) + row * a.sx, dl, t);
        if (gated) g.read(static_cast<const T*>(a.gate) + row * a.sg, dl, t);
        if constexpr (RES) r.read(static_cast<const T*>(a.res) + row * a.sr, dl, t);
        float u[VPL][VEC];
#pragma unroll
        for (int k = 0; k < VPL; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[k][e] = x.at(k, e);
        if (normed) {
            float sq = 0.f;
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sq = fmaf(u[k][e], u[k][e], sq);
            const float rs = 1.0f / sqrtf(row_sum<TPR>(sq, red, slot) * inv + a.eps);
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                float p[VEC];
                post.get(p, k, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) u[k][e] = u[k][e] * rs * p[e];
            }
        }
        if (gated)
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float v = g.at(k, e);
                    u[k][e] *= v * sigmoid(v);
                }
        T* y = static_cast<T*>(a.y) + row * a.d;
        if constexpr (!RES) {
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                const int i0 = (k * TPR + t) * VEC;
                if (i0 < dl) bn_write<T, VEC>(y + i0, u[k]);
            }
        } else {
            T* s = static_cast<T*>(a.s) + row * a.d;
            float sq = 0.f;
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                const int i0 = (k * TPR + t) * VEC;
                float c[VEC];
                scale.get(c, k, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    u[k][e] = fmaf(c[e], u[k][e], r.at(k, e));
                    sq = fmaf(u[k][e], u[k][e], sq);
                }
                if (i0 < dl) bn_write<T, VEC>(s + i0, u[k]);
            }
            const float rs = 1.0f / sqrtf(row_sum<TPR>(sq, red, slot) * inv + a.eps);
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                const int i0 = (k * TPR + t) * VEC;
                float p[VEC];
                w.get(p, k, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) p[e] *= u[k][e] * rs;
                if (i0 < dl) bn_write<T, VEC>(y + i0, p);
            }
        }
    }
}

// The backward's inputs of a thread's next row on their way to shared memory (its own 16-byte vectors, so without a
// barrier) while it works on this one: 18 warps that each waited for their row left memory idle (65536 bfloat16 rows of 768
// with a scale: 199 us without, 104 with it and values unpacked from whole registers; the bytes alone take 92).
template <int VEC, int VPL, int TPR, int RPC, bool RES, int HOW>
struct BnStage {
    static constexpr int kInputs = 2 + (HOW & 1) + (RES ? 2 : 0);
    static constexpr size_t kTwo = static_cast<size_t>(2) * kInputs * VPL * TPR * RPC * 16;
    static constexpr bool on = VEC > 1 && kTwo <= 168 * 1024;  // (float32 rows above 4096 values are read as they are needed)
    static constexpr size_t bytes = on ? kTwo : 0;
    unsigned char* mem;
    __device__ __forceinline__ unsigned char* at(int stage, int input, int k) const {
        return mem + (((stage * kInputs + input) * VPL + k) * static_cast<size_t>(TPR * RPC) + threadIdx.x) * 16;
    }
};

// CTAs a multiprocessor that a backward keeps registers for: 18 warps or more without gate and post norm, else 12 to 16.
constexpr int bn_bwd_min(int threads, int how) {
    const int n = (how == 0 ? 640 : 512) / threads;
    return n < 1 ? 1 : n;
}

// Two sums over a row's threads at once.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& p, float& q, float* red, int& slot) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
        p += __shfl_xor_sync(0xffffffffu, p, o);
        q += __shfl_xor_sync(0xffffffffu, q, o);
    }
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        float2* r = reinterpret_cast<float2*>(red) + slot * W;
        slot ^= 1;
        if ((threadIdx.x & 31) == 0) r[threadIdx.x / 32 % W] = make_float2(p, q);
        row_barrier<TPR>();
        p = q = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) p += r[i].x, q += r[i].y;
    }
}

template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES, int HOW>
__global__ void __launch_bounds__(TPR * RPC, bn_bwd_min(TPR * RPC, HOW)) bn_bwd_k(const BnArgs a) {
    const bool gated = HOW == 4 ? a.gate != nullptr : (HOW & 1) != 0, normed = HOW == 4 ? a.has_post != 0 : (HOW & 2) != 0;
    using Row = BnRow<T, VEC, VPL, TPR>;
    using Par = RowParam<VEC, VPL, TPR>;
    __shared__ __align__(8) float reds[RPC][4 * (TPR / 32) + 2];
    __shared__ __align__(16) float sw[Par::kFloats], sp[Par::kFloats], sc[RES ? Par::kFloats : 4];
    __shared__ float comb[RPC > 1 ? TPR * VPL * VEC : 1];
    Par w, post, scale;
    int slot = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    float* red = reds[grp];
    if constexpr (RES) {
        w.fill(sw, a.weight, a.w_dtype, a.d, 1.f);
        scale.fill(sc, a.scale, a.w_dtype, a.d, 1.f);
    }
    if (normed) post.fill(sp, a.post, a.w_dtype, a.d, 1.f);
    __syncthreads();
    float dw[RES ? VPL : 1][VEC] = {}, dc[RES ? VPL : 1][VEC] = {}, dp[VPL][VEC] = {};
    const float inv = 1.0f / static_cast<float>(a.d);
    const int64_t step = static_cast<int64_t>(gridDim.x) * RPC;
    extern __shared__ __align__(16) unsigned char stage_mem[];
    using Stage = BnStage<VEC, VPL, TPR, RPC, RES, HOW>;
    const Stage st{stage_mem};
    // the inputs in order: x, dy, residual, ds, gate
    auto input = [&](int i, int64_t row) -> const T* {
        if (i == 0) return static_cast<const T*>(a.x) + row * a.sx;
        if (i == 1) return a.dy ? static_cast<const T*>(a.dy) + row * a.sdy : nullptr;
        if (RES && i == 2) return static_cast<const T*>(a.res) + row * a.sr;
        if (RES && i == 3) return a.ds ? static_cast<const T*>(a.ds) + row * a.sds : nullptr;
        return static_cast<const T*>(a.gate) + row * a.sg;
    };
    auto fetch = [&](int stage, int64_t row) {
        if constexpr (Stage::on) {
            if (row < a.rows)
#pragma unroll
                for (int i = 0; i < Stage::kInputs; ++i) {
                    const T* p = input(i, row);
#pragma unroll
                    for (int k = 0; k < VPL; ++k) {
                        const int i0 = (k * TPR + t) * VEC;
                        if (p && i0 < a.d) row_cp16(st.at(stage, i, k), p + i0);
                    }
                }
            cp_async_commit();
        }
    };
    int stage = 0;
    int64_t row = static_cast<int64_t>(blockIdx.x) * RPC + grp;
    fetch(0, row);
    for (;; row += step, stage ^= 1) {
        const bool live = row < a.rows;
        if (TPR < 32 ? !__any_sync(0xffffffffu, live) : !live) break;
        const int dl = live ? a.d : 0;
        Row x, g, r, gy, gs;
        if constexpr (Stage::on) {
            fetch(stage ^ 1, row + step);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        }
        auto take = [&](Row& to, int i) {
            const T* p = input(i, row);
            if constexpr (Stage::on) {
#pragma unroll
                for (int k = 0; k < VPL; ++k) {
                    if (p && (k * TPR + t) * VEC < dl) to.load(k, st.at(stage, i, k));
                    else to.zero(k);
                }
            } else if (p) {
                to.read(p, dl, t);
            } else {
                to.zero();
            }
        };
        take(x, 0);
        take(gy, 1);
        if constexpr (RES) take(r, 2), take(gs, 3);
        if (gated) take(g, RES ? 4 : 2);
        float r1 = 1.f;
        if (normed) {
            float sq = 0.f, none = 0.f;
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sq = fmaf(x.at(k, e), x.at(k, e), sq);
            row_sum2<TPR>(sq, none, red, slot);
            r1 = 1.0f / sqrtf(sq * inv + a.eps);
        }
        // v: the gradient of u; before: u before the gate
        auto before = [&](int k, int e, const float* p) { return normed ? x.at(k, e) * r1 * p[e] : x.at(k, e); };
        auto gain = [&](int k, int e) {
            if (!gated) return 1.f;
            const float q = g.at(k, e);
            return q * sigmoid(q);
        };
        float v[VPL][VEC];
        if constexpr (RES) {
            float s[VPL][VEC], sq = 0.f, sg = 0.f;
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                float c[VEC], p[VEC], q[VEC];
                scale.get(c, k, t);
                w.get(q, k, t);
                if (normed) post.get(p, k, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    s[k][e] = fmaf(c[e], before(k, e, p) * gain(k, e), r.at(k, e));
                    sq = fmaf(s[k][e], s[k][e], sq);
                    sg = fmaf(gy.at(k, e) * q[e], s[k][e], sg);
                }
            }
            row_sum2<TPR>(sq, sg, red, slot);
            const float r2 = 1.0f / sqrtf(sq * inv + a.eps), m = sg * inv * r2 * r2;
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                const int i0 = (k * TPR + t) * VEC;
                float c[VEC], p[VEC], q[VEC], o[VEC];
                scale.get(c, k, t);
                w.get(q, k, t);
                if (normed) post.get(p, k, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float dyv = gy.at(k, e);
                    dw[k][e] = fmaf(dyv, s[k][e] * r2, dw[k][e]);
                    o[e] = fmaf(fmaf(dyv, q[e], -s[k][e] * m), r2, gs.at(k, e));
                    dc[k][e] = fmaf(o[e], before(k, e, p) * gain(k, e), dc[k][e]);
                    v[k][e] = o[e] * c[e];
                }
                if (a.dres && i0 < dl) bn_write<T, VEC>(static_cast<T*>(a.dres) + row * a.d + i0, o);
            }
        } else {
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[k][e] = gy.at(k, e);
        }
        if (gated)
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                const int i0 = (k * TPR + t) * VEC;
                float p[VEC], o[VEC];
                if (normed) post.get(p, k, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float q = g.at(k, e), sg = sigmoid(q);
                    o[e] = v[k][e] * before(k, e, p) * silu_slope(q, sg);
                    v[k][e] *= q * sg;
                }
                if (i0 < dl) bn_write<T, VEC>(static_cast<T*>(a.dgate) + row * a.d + i0, o);
            }
        if (normed) {
            float sm = 0.f, none = 0.f;
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                float p[VEC];
                post.get(p, k, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    dp[k][e] = fmaf(v[k][e], x.at(k, e) * r1, dp[k][e]);
                    v[k][e] *= p[e];
                    sm = fmaf(v[k][e], x.at(k, e), sm);
                }
            }
            row_sum2<TPR>(sm, none, red, slot);
            const float m = sm * inv * r1 * r1;
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[k][e] = r1 * fmaf(-x.at(k, e), m, v[k][e]);
        }
        T* dx = static_cast<T*>(a.dx) + row * a.d;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int i0 = (k * TPR + t) * VEC;
            if (i0 < dl) bn_write<T, VEC>(dx + i0, v[k]);
        }
    }
    if (!a.part) return;
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 3 * a.d;
#pragma unroll
    for (int which = RES ? 0 : 2; which < 3; ++which) {
        if (which == 2 && !normed) break;
        float(*acc)[VEC] = which == 0 ? dw : which == 1 ? dc : dp;
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
                part[which * static_cast<int64_t>(a.d) + i] = comb[(k * VEC + q % VEC) * TPR + q / VEC];
            }
        } else {
#pragma unroll
            for (int k = 0; k < VPL; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = (k * TPR + t) * VEC + e;
                    if (i < a.d) part[which * static_cast<int64_t>(a.d) + i] = acc[k][e];
                }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
constexpr int kBnBwdCtas = 4;  // a backward's CTAs an SM at most: also its partial rows
constexpr int kBnMaxParts = 148 * kBnBwdCtas;

template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES, int HOW>
cudaError_t bn_fwd_launch(const BnArgs& a, cudaStream_t s) {
    const auto k = bn_fwd_k<T, VEC, VPL, TPR, RPC, RES, HOW>;
    static const int per = row_resident(k, TPR * RPC, 0);
    k<<<row_grid(a.rows, RPC, per), TPR * RPC, 0, s>>>(a);
    note_launch();
    return cudaGetLastError();
}
template <typename T, int VEC, int VPL, int TPR, int RPC, bool RES, int HOW>
cudaError_t bn_bwd_launch(const BnArgs& a, int* parts, cudaStream_t s) {
    const auto k = bn_bwd_k<T, VEC, VPL, TPR, RPC, RES, HOW>;
    constexpr size_t smem = BnStage<VEC, VPL, TPR, RPC, RES, HOW>::bytes;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    static const int per = std::min(row_resident(k, TPR * RPC, smem), kBnBwdCtas);
    *parts = row_grid(a.rows, RPC, per);
    k<<<*parts, TPR * RPC, smem, s>>>(a);
    note_launch();
    return cudaGetLastError();
}

// As few threads a row as hold it: forward up to four vectors a thread, backward (with three sums a column) up to two.
// Rows whose start or length is not a multiple of 16 bytes are read element by element.
template <typename T, bool RES, int HOW>
cudaError_t bn_fwd_vec(const BnArgs& a, cudaStream_t s) {
    constexpr int E = 16 / sizeof(T);
#define EACS_BN(VPL, TPR, RPC) return bn_fwd_launch<T, E, VPL, TPR, RPC, RES, HOW>(a, s)
    const int n = (a.d + E - 1) / E;
    if (n <= 8) EACS_BN(1, 8, 32);
    if (n <= 16) EACS_BN(1, 16, 16);
    if (n <= 32) EACS_BN(1, 32, 8);
    if (n <= 64) EACS_BN(2, 32, 8);
    if (n <= 96) EACS_BN(3, 32, 8);
    if (n <= 128) EACS_BN(4, 32, 8);
    if (n <= 256) EACS_BN(2, 128, 2);
    if (n <= 512) EACS_BN(1, 512, 1);
    if (n <= 1024) EACS_BN(2, 512, 1);
    if constexpr (E == 4) EACS_BN(4, 512, 1);  // (16-bit rows of 8192 values have 1024 vectors)
    return cudaErrorInvalidValue;
#undef EACS_BN
}
template <typename T, bool RES, int HOW>
cudaError_t bn_bwd_vec(const BnArgs& a, int* parts, cudaStream_t s) {
    constexpr int E = 16 / sizeof(T);
#define EACS_BN(VPL, TPR, RPC) return bn_bwd_launch<T, E, VPL, TPR, RPC, RES, HOW>(a, parts, s)
    const int n = (a.d + E - 1) / E;
    if (n <= 8) EACS_BN(1, 8, 32);
    if (n <= 16) EACS_BN(1, 16, 16);
    if (n <= 32) EACS_BN(1, 32, 8);
    if (n <= 64) EACS_BN(1, 64, 4);
    if (n <= 96) EACS_BN(1, 96, 2);
    if (n <= 128) EACS_BN(1, 128, 2);
    if (n <= 256) EACS_BN(1, 256, 1);
    if (n <= 512) EACS_BN(1, 512, 1);
    if (n <= 1024) EACS_BN(2, 512, 1);
    if constexpr (E == 4) EACS_BN(4, 512, 1);
    return cudaErrorInvalidValue;
#undef EACS_BN
}
template <typename T, bool RES>
cudaError_t bn_fwd_any(const BnArgs& a, bool vec, cudaStream_t s) {
    if constexpr (RES)
        if (vec && !a.has_post) return a.gate ? bn_fwd_vec<T, RES, 1>(a, s) : bn_fwd_vec<T, RES, 0>(a, s);
    if (vec) return a.gate ? bn_fwd_vec<T, RES, 3>(a, s) : bn_fwd_vec<T, RES, 2>(a, s);
    if (a.d <= 64) return bn_fwd_launch<T, 1, 8, 8, 32, RES, 4>(a, s);
    if (a.d <= 128) return bn_fwd_launch<T, 1, 8, 16, 16, RES, 4>(a, s);
    if (a.d <= 256) return bn_fwd_launch<T, 1, 8, 32, 8, RES, 4>(a, s);
    if (a.d <= 512) return bn_fwd_launch<T, 1, 8, 64, 4, RES, 4>(a, s);
    if (a.d <= 1024) return bn_fwd_launch<T, 1, 8, 128, 2, RES, 4>(a, s);
    if (a.d <= 4096) return bn_fwd_launch<T, 1, 8, 512, 1, RES, 4>(a, s);
    return bn_fwd_launch<T, 1, 16, 512, 1, RES, 4>(a, s);
}
template <typename T, bool RES>
cudaError_t bn_bwd_any(const BnArgs& a, bool vec, int* parts, cudaStream_t s) {
    if constexpr (RES)
        if (vec && !a.has_post) return a.gate ? bn_bwd_vec<T, RES, 1>(a, parts, s) : bn_bwd_vec<T, RES, 0>(a, parts, s);
    if (vec) return a.gate ? bn_bwd_vec<T, RES, 3>(a, parts, s) : bn_bwd_vec<T, RES, 2>(a, parts, s);
    if (a.d <= 32) return bn_bwd_launch<T, 1, 4, 8, 32, RES, 4>(a, parts, s);
    if (a.d <= 64) return bn_bwd_launch<T, 1, 4, 16, 16, RES, 4>(a, parts, s);
    if (a.d <= 128) return bn_bwd_launch<T, 1, 4, 32, 8, RES, 4>(a, parts, s);
    if (a.d <= 256) return bn_bwd_launch<T, 1, 4, 64, 4, RES, 4>(a, parts, s);
    if (a.d <= 512) return bn_bwd_launch<T, 1, 4, 128, 2, RES, 4>(a, parts, s);
    if (a.d <= 1024) return bn_bwd_launch<T, 1, 8, 128, 2, RES, 4>(a, parts, s);
    if (a.d <= 4096) return bn_bwd_launch<T, 1, 8, 512, 1, RES, 4>(a, parts, s);
    return bn_bwd_launch<T, 1, 16, 512, 1, RES, 4>(a, parts, s);
}

int bn_check(const char* fn, const EacsNorm& p) {
    if (p.rows < 0 || p.d < 1) return fail(EACS_ERR_INVALID, "%s: bad sizes", fn);
    if (p.d > kBnMaxD) return fail(EACS_ERR_UNSUPPORTED, "%s: d=%lld > %d", fn, (long long)p.d, kBnMaxD);
    for (int dt : {p.dtype, p.w_dtype})
        if (dt != EACS_DTYPE_F32 && dt != EACS_DTYPE_F16 && dt != EACS_DTYPE_BF16)
            return fail(EACS_ERR_INVALID, "%s: unknown dtype %d", fn, dt);
    if (p.rows > 0 && !p.x) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    if (!p.residual && p.scale) return fail(EACS_ERR_INVALID, "%s: a scale without a residual", fn);
    if (p.x_stride < 0 || p.gate_stride < 0 || p.residual_stride < 0) return fail(EACS_ERR_INVALID, "%s: a negative stride", fn);
    return EACS_OK;
}
BnArgs bn_args(const EacsNorm& p) {
    BnArgs a{};
    a.x = p.x, a.gate = p.gate, a.res = p.residual;
    a.sx = p.x_stride, a.sg = p.gate_stride, a.sr = p.residual_stride;
    a.has_post = p.residual ? p.post_norm : 1;
    a.weight = p.weight, a.scale = p.scale, a.post = p.residual ? p.post_weight : p.weight;
    a.rows = p.rows, a.d = static_cast<int>(p.d), a.w_dtype = p.w_dtype, a.eps = p.eps;
    return a;
}
bool bn_rows16(const EacsNorm& p, const void* q, int64_t stride) {
    const int64_t esz = p.dtype == EACS_DTYPE_F32 ? 4 : 2;
    return !q || ((reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(stride * esz)) & 15u) == 0;
}

}  // namespace

size_t norm_bwd_workspace_size(const EacsNorm& p) {
    if (bn_check("eacs_norm_bwd_workspace_size", p) != EACS_OK) return 0;
    return static_cast<size_t>(std::min<int64_t>(p.rows, kBnMaxParts)) * 3 * p.d * sizeof(float);
}

int norm_fwd(const EacsNorm& p, void* y, void* s, cudaStream_t stream) {
    const char* fn = "eacs_norm_fwd";
    if (const int rc = bn_check(fn, p)) return rc;
    if (p.rows == 0) return EACS_OK;
    if (!y || (p.residual && !s)) return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    BnArgs a = bn_args(p);
    a.y = y, a.s = s;
    const bool vec = bn_rows16(p, p.x, p.x_stride) && bn_rows16(p, p.gate, p.gate_stride) &&
                     bn_rows16(p, p.residual, p.residual_stride) && bn_rows16(p, y, p.d) && bn_rows16(p, s, p.d);
    cudaError_t e;
    if (p.dtype == EACS_DTYPE_F32) e = p.residual ? bn_fwd_any<float, true>(a, vec, stream) : bn_fwd_any<float, false>(a, vec, stream);
    else if (p.dtype == EACS_DTYPE_F16) e = p.residual ? bn_fwd_any<__half, true>(a, vec, stream) : bn_fwd_any<__half, false>(a, vec, stream);
    else e = p.residual ? bn_fwd_any<__nv_bfloat16, true>(a, vec, stream) : bn_fwd_any<__nv_bfloat16, false>(a, vec, stream);
    return cuda_check(e, fn);
}

int norm_bwd(const EacsNorm& p, const NormGrads& g, void* ws, size_t ws_bytes, cudaStream_t stream) {
    const char* fn = "eacs_norm_bwd";
    if (const int rc = bn_check(fn, p)) return rc;
    void* const out[3] = {p.residual ? g.dweight : nullptr, p.residual ? g.dscale : nullptr, !p.residual ? g.dweight : p.post_norm ? g.dpost_weight : nullptr};
    const bool want = out[0] || out[1] || out[2];
    if (p.rows == 0) {  // empty sums
        cudaError_t e = cudaSuccess;
        for (void* o : out)
            if (o && e == cudaSuccess) e = cudaMemsetAsync(o, 0, (p.w_dtype == EACS_DTYPE_F32 ? 4 : 2) * p.d, stream);
        return cuda_check(e, fn);
    }
    BnArgs a = bn_args(p);
    const bool apart = p.scale || p.gate || a.has_post;  // d residual is not dx
    if (!g.dx || (p.gate && !g.dgate) || (p.residual && apart && !g.dresidual))
        return fail(EACS_ERR_INVALID, "%s: null pointer argument", fn);
    if (want && (!ws || ws_bytes < norm_bwd_workspace_size(p)))
        return fail(EACS_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, norm_bwd_workspace_size(p));
    a.dy = g.dy, a.ds = p.residual ? g.ds : nullptr;
    a.sdy = g.dy_stride, a.sds = g.ds_stride;
    a.dx = g.dx, a.dgate = g.dgate, a.dres = p.residual ? g.dresidual : nullptr;
    a.part = want ? static_cast<float*>(ws) : nullptr;
    const bool vec = bn_rows16(p, p.x, p.x_stride) && bn_rows16(p, p.gate, p.gate_stride) &&
                     bn_rows16(p, p.residual, p.residual_stride) && bn_rows16(p, g.dy, g.dy_stride) &&
                     bn_rows16(p, a.ds, g.ds_stride) && bn_rows16(p, g.dx, p.d) && bn_rows16(p, g.dgate, p.d) && bn_rows16(p, a.dres, p.d);
    int parts = 0;
    cudaError_t e;
    if (p.dtype == EACS_DTYPE_F32)
        e = p.residual ? bn_bwd_any<float, true>(a, vec, &parts, stream) : bn_bwd_any<float, false>(a, vec, &parts, stream);
    else if (p.dtype == EACS_DTYPE_F16)
        e = p.residual ? bn_bwd_any<__half, true>(a, vec, &parts, stream) : bn_bwd_any<__half, false>(a, vec, &parts, stream);
    else
        e = p.residual ? bn_bwd_any<__nv_bfloat16, true>(a, vec, &parts, stream)
                       : bn_bwd_any<__nv_bfloat16, false>(a, vec, &parts, stream);
    if (e == cudaSuccess && want) {
        RowSums r{};
        r.part = a.part, r.rows = parts, r.stride = 3 * static_cast<int64_t>(a.d), r.dtype = p.w_dtype;
        for (int i = 0; i < 3; ++i) r.out[i] = out[i], r.at[i] = i * static_cast<int64_t>(a.d), r.n[i] = a.d;
        e = row_sums(r, 3, stream);
    }
    return cuda_check(e, fn);
}

}  // namespace eacs
