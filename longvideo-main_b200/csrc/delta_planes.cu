// delta_planes.cu -- the gated delta rule on bfloat16 and float16 inputs (sm_100a).
//
// The formulas are those of delta.cu.  Here every product runs on 16-bit
// operands of the inputs' type: the inputs are exact in it, and a float32
// result that goes back in as an operand is split into two planes of it,
// x = hi + lo (16 significant bits in bfloat16, 22 in float16).  With one plane
// everywhere dg was off by 5e-3 of its norm.  A NaN or an infinity of a token
// spreads over its block of 16 tokens, as what lies above a triangle's diagonal
// there is multiplied by 0.
//
// float16's exponent is too short for this by itself: below 2^-3 the low plane
// runs out.  There T' and M, S, X and U, dS and dU are scaled by powers of two
// (Scaled below), and T' is made without beta: with Ahat_ij = Gam_ij k_i.k_j
// (j < i) and D = diag(beta), e = (I + Ahat D)^-1 X and U = D e, and in reverse
// dV = D (I + D Ahat)^-T dU, so that a small beta meets float32 only (forward at
// B=3 L=1001 H=8 K=64 V=96: 49 us with it, 43 without).  What a backward keeps and
// multiplies (S, U, dS and dV, of all groups in one sum) is stored in float32 and
// goes to delta_grad_k of delta.cu (B=2 L=4096 H=12 K=V=64, forward and backward:
// 52 + 166 + 171 + 263 us; 2400 with everything there).
//
// The kernels, with times at B=4 L=16384 H=8 (forward) and B=8 L=8192 H=6
// (training), K = V = 128, bfloat16:
//   planes_prep_k    per chunk: gam, d, T' and M            141 us; 112 us
//   planes_chain_k   the chunks in order: S, U and the outputs  650 us; 568 us
//   planes_rchain_k  the chunks in reverse order: dV and dS     471 us
//   planes_grad_k    per chunk: dQ, dK, dbeta, dg               873 us
//
// The two chains are bound by the length of one chunk's dependent products (2.4
// to 2.8 us each; 256 chunks of a head follow one another), as only 16-column groups
// of a state run side by side (a warp each, 8 a head of 128): so everything
// that does not depend on the state is taken out of the warp that carries it.
// A CTA holds G such warps, one or more helpers (the forward's outputs; the
// reverse chain's Q^T dO) and a loading warp, which copies each chunk's rows
// and tiles to shared memory, two chunks deep, and stores what a backward
// reads.  Rows of the inputs come by tensor maps (64 tokens by 64 or 16
// columns, swizzled so that ldmatrix meets no bank twice; a bulk copy for each
// row of 256 bytes took 67 cycles a row and bound the chains).  Tiles that
// kernels hand to each other (T', M, S, U, dS, dV) lie in the workspace as
// they lie in shared memory, padding included, so that a tile is one copy.
// Every wait is bounded.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "delta_common.cuh"

namespace eacs {
namespace {

using e16 = uint16_t;  // a bfloat16 or float16 as it lies in memory

// ----------------------------------------------------------------------------
// barriers and bulk copies
// ----------------------------------------------------------------------------
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// global -> shared, 16-byte aligned, counted on `bar`
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// a warp's wait, with one outcome for all its lanes
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
// Two barriers at once, and one that was asked earlier (a wait that is over
// before it begins still takes some 270 cycles of a warp that has no other).
__device__ __forceinline__ bool warp_wait2(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) {
    const bool da = mbar_try_wait(a, pa), db = mbar_try_wait(b, pb);
    if (__all_sync(0xffffffffu, da && db)) return true;
    return warp_wait(a, pa) && warp_wait(b, pb);
}
__device__ __forceinline__ bool warp_wait_asked(bool done, uint64_t* bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, done)) return true;
    return warp_wait(bar, parity);
}
// one arrival for a warp, after what all its lanes did
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// ----------------------------------------------------------------------------
// operands
// ----------------------------------------------------------------------------
// What the products are made of: pairs of a type, and its matrix instruction.
template <typename T> struct Num;
template <> struct Num<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16(lo, hi); }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return unpack_bf16(v); }
    static __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) { mma_bf16(c, a, b0, b1); }
};
template <> struct Num<__half> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 p = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&p);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
    static __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) { mma_f16(c, a, b0, b1); }
};

// float16's exponent is short: two planes hold 22 bits of values from 2^-3 up,
// and a step of 2^-25 below.  So its tiles are kept near 1 by powers of two
// (Scaled): a tile whose largest value is between 2^-3 and 2^13 stays as it is,
// any other is brought to 2^4, and is then off by at most 2^-22 of its largest value.
// bfloat16 has float32's exponent and needs none of it.
template <typename T> constexpr bool Scaled = false;
template <> constexpr bool Scaled<__half> = true;

constexpr int kMaxExp = 100;  // of a scale
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }  // ordered as |v| is
template <int N>
__device__ __forceinline__ uint32_t max_bits(const float (*x)[4]) {  // of a warp's tile
    float m[4] = {};
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = fmaxf(m[e], fabsf(x[j][e]));
    return __reduce_max_sync(0xffffffffu, abs_bits(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))));
}
// The exponent to scale a tile by whose largest absolute value has these bits (0
// for a tile of zeros, and for one that is infinite: nothing helps it)
__device__ __forceinline__ int scale_exp(uint32_t bits) {
    const int e = static_cast<int>(bits >> 23) - 127;
    return bits == 0 || (e >= -3 && e < 13) || e == 128 ? 0 : max(-kMaxExp, min(kMaxExp, 4 - e));
}
template <int N>
__device__ __forceinline__ void scale_tile(float (*x)[4], float f) {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] *= f;
}

template <int P> struct Af { uint32_t r[P][4]; };  // 16 x 16 of A in P planes

template <typename T, int P>
__device__ __forceinline__ Af<P> from_acc(const float* c0, const float* c1) {
    Af<P> a;
    const float v[8] = {c0[0], c0[1], c0[2], c0[3], c1[0], c1[1], c1[2], c1[3]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a.r[0][i] = Num<T>::pack(v[2 * i], v[2 * i + 1]);
        if constexpr (P == 2) {
            const float2 h = Num<T>::unpack(a.r[0][i]);
            a.r[1][i] = Num<T>::pack(v[2 * i] - h.x, v[2 * i + 1] - h.y);
        }
    }
    return a;
}
// Quarter i of that: registers i of both planes.
template <typename T, int P>
__device__ __forceinline__ void from_acc_part(Af<P>& a, int i, float x, float y) {
    a.r[0][i] = Num<T>::pack(x, y);
    if constexpr (P == 2) {
        const float2 h = Num<T>::unpack(a.r[0][i]);
        a.r[1][i] = Num<T>::pack(x - h.x, y - h.y);
    }
}
// A tile in shared memory by its 32-bit address, in elements.  (With generic
// pointers the address arithmetic of unrolled loads was most of the code.)
struct Sh {
    uint32_t a;
    __device__ __forceinline__ Sh operator+(int n) const { return Sh{a + 2u * static_cast<uint32_t>(n)}; }
};
__device__ __forceinline__ Sh sh(const void* p) { return Sh{smem_u32(p)}; }

// A operands of a tile stored [m][k], and stored [k][m]: the lane's part of the
// address, then the tile's (a constant where loops are unrolled).
__device__ __forceinline__ void ld_a(uint32_t* r, Sh s, int ld, int m0, int k0) {
    const int l = threadIdx.x & 31;
    ldsm4(r, (s + ((l & 15) * ld + (l >> 4) * 8) + m0 * ld + k0).a);
}
__device__ __forceinline__ void ld_at(uint32_t* r, Sh s, int ld, int m0, int k0) {
    const int l = threadIdx.x & 31;
    ldsm4t(r, (s + (((l & 7) + ((l >> 4) & 1) * 8) * ld + ((l >> 3) & 1) * 8) + m0 + k0 * ld).a);
}
// 16 columns of B by 16 of the summed index, stored [n][k], and (TR) [k][n]
template <bool TR>
__device__ __forceinline__ void ld_b(uint32_t* b, Sh s, int ld, int n0, int k0) {
    const int l = threadIdx.x & 31;
    if constexpr (TR) ldsm4t(b, (s + (((l & 7) + ((l >> 3) & 1) * 8) * ld + ((l >> 4) & 1) * 8) + n0 + k0 * ld).a);
    else ldsm4(b, (s + (((l & 7) + ((l >> 4) & 1) * 8) * ld + ((l >> 3) & 1) * 8) + n0 * ld + k0).a);
}
// Tiles that tensor maps bring.  Rows of 64 columns in 128-byte swizzle, 64
// rows a box, boxes one after another (queries, keys); rows of 16 columns in
// 32-byte swizzle (values and upstream gradients, a box a group of 16).
__device__ __forceinline__ int at128(int row, int col) {
    return (col >> 6) * (kC * 64) + row * 64 + ((((col >> 3) & 7) ^ (row & 7)) << 3) + (col & 7);
}
// The swizzle is (16-byte column) xor (row mod 8), and a lane's row mod 8 is its
// number mod 8: its own part of the address is made once, a tile's columns are
// xored in (boxes start on 1024 bytes) and its rows added.
template <bool TR>
__device__ __forceinline__ void ld_b128(uint32_t* b, Sh s, int n0, int k0) {
    const int l = threadIdx.x & 31;
    const int row = (l & 7) + ((TR ? l >> 3 : l >> 4) & 1) * 8, bit = (TR ? l >> 4 : l >> 3) & 1;
    const uint32_t mine = s.a + row * 128 + ((bit ^ (l & 7)) << 4);
    const int col = TR ? n0 : k0, r0 = TR ? k0 : n0;
    const uint32_t at = (mine ^ static_cast<uint32_t>(((col >> 3) & 7) << 4)) + (col >> 6) * (kC * 128) + r0 * 128;
    if constexpr (TR) ldsm4t(b, at);
    else ldsm4(b, at);
}
__device__ __forceinline__ void ld_a128(uint32_t* r, Sh s, int m0, int k0) {
    const int l = threadIdx.x & 31;
    const uint32_t mine = s.a + (l & 15) * 128 + (((l >> 4) ^ (l & 7)) << 4);
    ldsm4(r, (mine ^ static_cast<uint32_t>(((k0 >> 3) & 7) << 4)) + (k0 >> 6) * (kC * 128) + m0 * 128);
}
// 16 rows of A: tokens m0.. of a group, and (at) its 16 columns by tokens k0..
__device__ __forceinline__ void ld_a32(uint32_t* r, Sh s, int m0) {
    const int l = threadIdx.x & 31;
    ldsm4(r, (s + ((l & 15) * 16 + (((l >> 4) ^ (l >> 2)) & 1) * 8) + m0 * 16).a);
}
__device__ __forceinline__ void ld_at32(uint32_t* r, Sh s, int k0) {
    const int l = threadIdx.x & 31;
    ldsm4t(r, (s + (((l & 7) + ((l >> 4) & 1) * 8) * 16 + (((l >> 3) ^ (l >> 2)) & 1) * 8) + k0 * 16).a);
}
template <typename T>
__device__ __forceinline__ void mma_pair(float* c0, float* c1, const uint32_t* a, const uint32_t* b) {
    Num<T>::mma(c0, a, b[0], b[1]);
    Num<T>::mma(c1, a, b[2], b[3]);
}
// A in P planes times one plane of B
template <typename T, int P, bool TR>
__device__ __forceinline__ void mm128(float* c0, float* c1, const Af<P>& a, Sh s, int n0, int k0) {
    uint32_t b[4];
    ld_b128<TR>(b, s, n0, k0);
#pragma unroll
    for (int p = P - 1; p >= 0; --p) mma_pair<T>(c0, c1, a.r[p], b);
}
// Steps 0..N-1 of a product: a step's tiles of B (up to four pairs) are read
// while the step before is multiplied.
template <int N, bool AHEAD = true, class Read, class Use>
__device__ __forceinline__ void steps(Read read, Use use) {
    uint32_t b[AHEAD ? 2 : 1][4][4];
    if constexpr (AHEAD) read(0, b[0]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (AHEAD) {
            if (i + 1 < N) read(i + 1, b[(i + 1) & 1]);
            use(i, b[i & 1]);
        } else {
            read(i, b[0]);
            use(i, b[0]);
        }
    }
}
// accumulators j0.. of `n` pairs += A (planes P-1 .. 0) B, plane by plane: eight
// products lie between two that add to the same accumulator
template <typename T, int P>
__device__ __forceinline__ void mma_step(float (*c)[4], const Af<P>& a, const uint32_t (*b)[4], int from = 0, int to = 4) {
#pragma unroll
    for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i >= from && i < to) mma_pair<T>(c[2 * i], c[2 * i + 1], a.r[p], b[i]);
}
// The same with other work of the warp in quarters, side(0..3), between the
// products: a warp alone on its scheduler would otherwise do it while the tensor
// pipe stands still.
template <typename T, int P, class Side>
__device__ __forceinline__ void mma_step_with(float (*c)[4], const Af<P>& a, const uint32_t (*b)[4], Side side, int from = 0,
                                              int to = 4) {
#pragma unroll
    for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= from && i < to) mma_pair<T>(c[2 * i], c[2 * i + 1], a.r[p], b[i]);
            if (p == P - 1) side(i);
        }
}
template <int P> __device__ __forceinline__ Af<1> high(const Af<P>& a) {
    return Af<1>{{{a.r[0][0], a.r[0][1], a.r[0][2], a.r[0][3]}}};
}
// accumulators of 16 rows by 16 columns to a tile [row][col] (as ld_a reads it)
__device__ __forceinline__ void st_tile(Sh s, int ld, int c0, const uint32_t* r) {
    const int l = threadIdx.x & 31;
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(
                     (s + ((l & 15) * ld + (l >> 4) * 8) + c0).a),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}
// and to a tile [col][row]
__device__ __forceinline__ void st_tile_t(Sh s, int ld, int c0, const uint32_t* r) {
    const int l = threadIdx.x & 31;
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(
                     (s + (((l & 7) + (l >> 4) * 8) * ld + ((l >> 3) & 1) * 8) + c0 * ld).a),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}

constexpr int kCC = kC * kTld;  // elements of a 64 x 64 tile

// A tensor map of (B, L, H, D) with a dense last dimension, read as (D, L, H, B).
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int t, int h, int b) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
        "[%2];" ::"r"(smem_u32(dst)),
        "l"(m), "r"(smem_u32(bar)), "r"(x), "r"(t), "r"(h), "r"(b)
        : "memory");
}
struct Maps { CUtensorMap q, k, v, d; };

// Rows `rows`.. of `boxes` boxes of 64 rows x W columns become zeros; the lanes
// of one warp.  (Rows of a padded batch behind a sequence's end: what they hold,
// NaN as it may be, is not to reach a product.  Behind L the copy itself gives 0.)
template <int W>
__device__ __forceinline__ void zero_rows(e16* s, int boxes, int rows) {
    const int per = (kC - rows) * (W / 8);
    for (int i = threadIdx.x & 31; i < boxes * per; i += 32)
        *reinterpret_cast<uint4*>(s + (i / per) * kC * W + rows * W + (i % per) * 8) = make_uint4(0, 0, 0, 0);
}
// The aligned start of dynamic shared memory (swizzled boxes want 1024 bytes).
__device__ __forceinline__ unsigned char* align_smem(unsigned char* p) { return p + ((1024u - (smem_u32(p) & 1023u)) & 1023u); }
constexpr int up1024(int x) { return (x + 1023) / 1024 * 1024; }
// e^(G_i - G_j) from G in units of log 2, high and low parts
__device__ __forceinline__ float ratio(const float* G, int i, int j) {
    return ex2_approx((G[i] - G[j]) + (G[kC + i] - G[kC + j]));
}

// ----------------------------------------------------------------------------
// gates, T' and M of a chunk
// ----------------------------------------------------------------------------
// Two warps make M and two A (float16: Ahat D), of each one block rows 3 and 0 (of
// 16 tokens), the other 2 and 1: five 16 x 16 blocks each.  Blocks above the
// diagonal are neither made nor written, as no product reads them.  The latter two
// then invert I + A by blocks, in float32: the 16 x 16 blocks on the diagonal by forward substitution (a
// thread a column), then twice the step from blocks of s to blocks of 2 s,
// [[P, 0], [R, Q]]^-1 = [[P^-1, 0], [-Q^-1 R P^-1, Q^-1]], whose products run on the
// tensor cores with operands split in two tf32 parts.  (Forward substitution alone
// takes 2016 dependent multiply-adds.)  Bound by the instructions a chunk takes and
// by what it moves, 32 KB in and 39 KB out; A and its inverse lie where K and Q
// were, so that six CTAs share an SM.
constexpr int kAld = kC + 8;  // float32 tiles

__device__ __forceinline__ void sync_inverse() { asm volatile("bar.sync 1, 64;" ::: "memory"); }

// What a scaled tile is to be multiplied by lies behind its first row.
__device__ __forceinline__ float tile_unit(const e16* tile) { return *reinterpret_cast<const float*>(tile + kC); }
__device__ __forceinline__ void set_tile_unit(e16* tile, int e) { *reinterpret_cast<float*>(tile + kC) = pow2(-e); }

template <int KD>
struct Prep {
    static constexpr int kIn = 2 * kC * KD * 2, kTiles = 2 * kC * kAld * 4;
    static constexpr size_t bytes = 1024 + (kIn > kTiles ? kIn : kTiles);
};

template <typename T, int KD>
__global__ void __launch_bounds__(128) planes_prep_k(const __grid_constant__ DArgs a, const __grid_constant__ Maps maps) {
    using F = FmtF<false>;
    const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int len = row_length(a, b);
    if (c * kC >= len) return;
    const int rows = min(kC, len - c * kC);
    const int hk = h / (a.Hv / a.Hk);
    const int64_t id = (static_cast<int64_t>(b) * a.Hv + h) * a.n + c, t0 = static_cast<int64_t>(c) * kC;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    unsigned char* smem = align_smem(smem_raw);
    e16* sK = reinterpret_cast<e16*>(smem);
    e16* sQ = sK + kC * KD;
    float* sA = reinterpret_cast<float*>(smem);  // A below the diagonal blocks, products above (after K and Q)
    float* sT = sA + kC * kAld;                  // its inverse
    __shared__ float sG[2 * kC], sB[kC];
    __shared__ uint32_t sMax[2][4];
    __shared__ uint64_t land;
    const int tid = threadIdx.x, warp = tid >> 5;
    const Lane L;
    float* ga = a.gates + id * kGates;
    if (tid == 0) {
        mbar_init(&land, 1);
        fence_mbar_init();
        mbar_expect_tx(&land, 4 * kC * KD);
#pragma unroll
        for (int x = 0; x < KD; x += 64) {
            tma_load(sK + x * kC, &maps.k, &land, x, c * kC, hk, b);
            tma_load(sQ + x * kC, &maps.q, &land, x, c * kC, hk, b);
        }
    }
    if (warp == 1) {
        double s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * L.l + i;
            float gv = 0.f, bv = 0.f;
            if (r < rows) {
                gv = gate_value(a.g, a.gate_dtype, b * a.sg.b + (t0 + r) * a.sg.t + h * a.sg.h);
                bv = gate_value(a.beta, a.gate_dtype, b * a.sb.b + (t0 + r) * a.sb.t + h * a.sb.h);
                if (a.S) bv = hold_beta(bv);  // a backward divides by it
                gv = gv < -200.f ? -200.f : gv;  // e^-200 is 0 in float32
            }
            s[i] = gv * 1.4426950408889634;  // to powers of two
            sB[r] = bv;
        }
        s[1] += s[0];
        double run = s[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, run, o);
            if (L.l >= o) run += up;
        }
        const double before = run - s[1], total = __shfl_sync(0xffffffffu, run, 31);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * L.l + i;
            const double G = before + s[i];
            const float hi = static_cast<float>(G), lo = static_cast<float>(G - hi);
            const float gam = exp2f(static_cast<float>(G));
            sG[r] = hi;
            sG[kC + r] = lo;
            if constexpr (Scaled<T>) {
                const double Ge = G * 0.6931471805599453;  // as the gradients' kernel takes it
                const float h = static_cast<float>(Ge);
                ga[r] = h;
                ga[kC + r] = static_cast<float>(Ge - h);
                ga[5 * kC + r] = sB[r];
            } else {
                ga[r] = hi;
                ga[kC + r] = lo;
                if (a.S) ga[5 * kC + r] = r < rows ? 1.f / sB[r] : 0.f;
            }
            ga[2 * kC + r] = gam;
            ga[3 * kC + r] = exp2f(static_cast<float>(total - G));
            ga[4 * kC + r] = a.scale * gam;
        }
    }
    __syncthreads();
    mbar_wait(&land, 0);  // (one that runs out is recorded; nobody leaves the barriers below)
    if (rows < min(kC, a.L - c * kC)) {
        if (warp == 0) zero_rows<64>(sK, 2 * (KD / 64), rows);
        __syncthreads();
    }
    // block i of a warp: row block and column block
    const int second = warp & 1, split = 4 - second;
    const int rb0 = 3 - second, rb1 = second;
    const bool left = warp >= 2;  // A
    float x[5][2][4] = {};
    {
        const Sh s = sh(left ? sK : sQ);
#pragma unroll
        for (int k0 = 0; k0 < KD; k0 += 16) {
            uint32_t a0[4], a1[4], bk[4];
            ld_a128(a0, s, 16 * rb0, k0);
            ld_a128(a1, s, 16 * rb1, k0);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                if (p > rb0) break;
                ld_b128<false>(bk, sh(sK), 16 * p, k0);
                mma_pair<T>(x[p][0], x[p][1], a0, bk);
                if (p <= rb1) {
                    if (second) mma_pair<T>(x[3 + p > 4 ? 4 : 3 + p][0], x[3 + p > 4 ? 4 : 3 + p][1], a1, bk);
                    else mma_pair<T>(x[4][0], x[4][1], a1, bk);
                }
            }
        }
    }
    __syncthreads();  // K and Q are done with
    e16* M = static_cast<e16*>(a.M) + id * 2 * kCC;
    auto put_m = [&](const float* v, int r0, int col) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t hi = Num<T>::pack(v[2 * e], v[2 * e + 1]);
            const float2 f = Num<T>::unpack(hi);
            const int o = (r0 + 8 * e) * kTld + col;
            *reinterpret_cast<uint32_t*>(M + o) = hi;
            *reinterpret_cast<uint32_t*>(M + kCC + o) = Num<T>::pack(v[2 * e] - f.x, v[2 * e + 1] - f.y);
        }
    };
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        const int rb = i < split ? rb0 : rb1, cb = i < split ? i : i - split;
        const int r0 = 16 * rb + L.g;
        const float g0 = sG[r0], g1 = sG[r0 + 8], l0 = sG[kC + r0], l1 = sG[kC + r0 + 8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = 16 * cb + 8 * j + 2 * L.t;
            const float2 gc = *reinterpret_cast<const float2*>(sG + col), lc = *reinterpret_cast<const float2*>(sG + kC + col);
            const int last = left ? -1 : 0;  // A without the diagonal
            // A has beta of its row, Ahat D of its column
            float f[4] = {a.scale, a.scale, a.scale, a.scale};
            if (left) {
                f[0] = sB[Scaled<T> ? col : r0];
                f[1] = sB[Scaled<T> ? col + 1 : r0];
                f[2] = sB[Scaled<T> ? col : r0 + 8];
                f[3] = sB[Scaled<T> ? col + 1 : r0 + 8];
            }
            float* v = x[i][j];
            v[0] = col <= r0 + last ? f[0] * ex2_approx((g0 - gc.x) + (l0 - lc.x)) * v[0] : 0.f;
            v[1] = col + 1 <= r0 + last ? f[1] * ex2_approx((g0 - gc.y) + (l0 - lc.y)) * v[1] : 0.f;
            v[2] = col <= r0 + 8 + last ? f[2] * ex2_approx((g1 - gc.x) + (l1 - lc.x)) * v[2] : 0.f;
            v[3] = col + 1 <= r0 + 8 + last ? f[3] * ex2_approx((g1 - gc.y) + (l1 - lc.y)) * v[3] : 0.f;
            if (left) {
                *reinterpret_cast<float2*>(sA + r0 * kAld + col) = make_float2(v[0], v[1]);
                *reinterpret_cast<float2*>(sA + (r0 + 8) * kAld + col) = make_float2(v[2], v[3]);
            } else if (!Scaled<T>) {
                put_m(v, r0, col);
            }
        }
    }
    // From the largest value of the two warps of a tile; `bar`: theirs, `slot`: of the tile
    auto pair_scale = [&](uint32_t bits, int bar, int slot) {
        if (L.l == 0) sMax[slot][warp] = bits;
        asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
        return scale_exp(max(sMax[slot][warp & 2], sMax[slot][warp | 1]));
    };
    if constexpr (Scaled<T>) {
        if (!left) {
            const int e = pair_scale(max_bits<10>(&x[0][0]), 2, 0);
            scale_tile<10>(&x[0][0], pow2(e));
            if (tid == 0) set_tile_unit(M, e);
#pragma unroll
            for (int i = 0; i < 5; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    put_m(x[i][j], 16 * (i < split ? rb0 : rb1) + L.g, 16 * (i < split ? i : i - split) + 8 * j + 2 * L.t);
        }
    }
    if (!left) return;
    sync_inverse();
    const int u = tid - 64;
    {  // column u of its diagonal block
        const int r0 = u & ~15, col = u & 15;
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s[4] = {i == col ? 1.f : 0.f, 0.f, 0.f, 0.f};
            const float* ar = sA + (r0 + i) * kAld + r0;
#pragma unroll
            for (int m = 0; m < i; m += 4) {
                const float4 f = *reinterpret_cast<const float4*>(ar + m);
                s[0] = fmaf(-f.x, y[m], s[0]);
                if (m + 1 < i) s[1] = fmaf(-f.y, y[m + 1], s[1]);
                if (m + 2 < i) s[2] = fmaf(-f.z, y[m + 2], s[2]);
                if (m + 3 < i) s[3] = fmaf(-f.w, y[m + 3], s[3]);
            }
            y[i] = (s[0] + s[1]) + (s[2] + s[3]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) sT[(r0 + i) * kAld + u] = y[i];
    }
    sync_inverse();
    auto put = [&](float* d, int r, int col, const float* x0, const float* x1, float sign) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            float* p = d + (r + L.g + (e >> 1) * 8) * kAld + col + 2 * L.t;
            *reinterpret_cast<float2*>(p) = make_float2(sign * x0[e], sign * x0[e + 1]);
            *reinterpret_cast<float2*>(p + 8) = make_float2(sign * x1[e], sign * x1[e + 1]);
        }
    };
    {  // a pair of 16 x 16 blocks a warp: R P^-1 (kept above the diagonal of A), then -Q^-1 of it
        const int o = 32 * second;
        float* y = sA + o * kAld + o + 16;
        float x0[4] = {}, x1[4] = {}, z0[4] = {}, z1[4] = {};
        F::template mma2<1, true>(x0, x1, F::from_smem(sA, kAld, o + 16, o), sT, kAld, o, o);
        put(y, 0, 0, x0, x1, 1.f);
        __syncwarp();
        F::template mma2<1, true>(z0, z1, F::from_smem(sT, kAld, o + 16, o + 16), y, kAld, 0, 0);
        put(sT, o + 16, o, z0, z1, -1.f);
    }
    sync_inverse();
    {  // the blocks of 32: 16 columns a warp
        const int col = 16 * second;
        float* y = sA + 32;
#pragma unroll
        for (int r = 32; r < 64; r += 16) {
            float x0[4] = {}, x1[4] = {};
#pragma unroll
            for (int k = 0; k < 32; k += 16)
                if (k >= col) F::template mma2<1, true>(x0, x1, F::from_smem(sA, kAld, r, k), sT, kAld, col, k);
            put(y, r - 32, col, x0, x1, 1.f);
        }
        __syncwarp();
#pragma unroll
        for (int r = 32; r < 64; r += 16) {
            float z0[4] = {}, z1[4] = {};
#pragma unroll
            for (int k = 0; k < r - 16; k += 16)
                F::template mma2<1, true>(z0, z1, F::from_smem(sT, kAld, r, 32 + k), y, kAld, col, k);
            put(sT, r, col, z0, z1, -1.f);
        }
    }
    sync_inverse();
    auto at_block = [&](int i, int& r, int& c8) {  // ten blocks of 16 rows by two vectors of 8
        const int at = i * 64 + u, blk = at >> 5, r16 = (at & 31) >> 1;
        const int rb = blk >= 6 ? 3 : blk >= 3 ? 2 : blk >= 1 ? 1 : 0, cb = blk - rb * (rb + 1) / 2;
        r = 16 * rb + r16;
        c8 = 16 * cb + (at & 1) * 8;
    };
    auto put_t = [&](e16* to, auto pair) {  // pair(row, column): of columns column, column + 1
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            int r, c8;
            at_block(i, r, c8);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 v = pair(r, c8 + 2 * e);
                hi[e] = Num<T>::pack(v.x, v.y);
                const float2 f = Num<T>::unpack(hi[e]);
                lo[e] = Num<T>::pack(v.x - f.x, v.y - f.y);
            }
            *reinterpret_cast<uint4*>(to + r * kTld + c8) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(to + kCC + r * kTld + c8) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    };
    e16* to = static_cast<e16*>(a.T) + id * 2 * kCC;
    auto inverse = [&](int r, int c) { return *reinterpret_cast<const float2*>(sT + r * kAld + c); };
    if constexpr (Scaled<T>) {
        auto put_scaled = [&](e16* t, int slot, auto pair) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 5; ++i) {
                int r, c8;
                at_block(i, r, c8);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float2 v = pair(r, c8 + e);
                    m = fmaxf(m, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
            }
            const int e = pair_scale(__reduce_max_sync(0xffffffffu, abs_bits(m)), 1, slot);
            const float f = pow2(e);
            put_t(t, [&](int r, int c) {
                const float2 v = pair(r, c);
                return make_float2(v.x * f, v.y * f);
            });
            if (u == 0) set_tile_unit(t, e);
        };
        put_scaled(to, 0, inverse);
        // (I + D Ahat)^-1 = D (I + Ahat D)^-1 D^-1 for the reverse chain (on the diagonal both have 1)
        if (a.Tr)
            put_scaled(static_cast<e16*>(a.Tr) + id * 2 * kCC, 1, [&](int r, int c) {
                float2 v = inverse(r, c);
                const float2 w = *reinterpret_cast<const float2*>(sB + c);
                v.x = r > c && c < rows ? v.x * (sB[r] / w.x) : r == c ? 1.f : 0.f;
                v.y = r > c + 1 && c + 1 < rows ? v.y * (sB[r] / w.y) : r == c + 1 ? 1.f : 0.f;
                return v;
            });
    } else {
        put_t(to, [&](int r, int c) {
            const float2 v = inverse(r, c), w = *reinterpret_cast<const float2*>(sB + c);
            return make_float2(v.x * w.x, v.y * w.y);
        });
    }
}

// ----------------------------------------------------------------------------
// the forward chain and the outputs
// ----------------------------------------------------------------------------
constexpr int kChainGates = 5 * kC;  // (without 1 / beta)
// What of a chunk's gates a chain loads, and where it then finds them.
template <typename T>
struct Gates {
    static constexpr int first = Scaled<T> ? 2 * kC : 0, n = Scaled<T> ? 4 * kC : kChainGates;
    static constexpr int gam = 2 * kC - first, dec = 3 * kC - first, sgam = 4 * kC - first, beta = 5 * kC - first;
    static constexpr uint32_t less = (kChainGates - n) * 4;  // bytes
};

template <int KD, int G>
struct Fwd {
    static constexpr int LDK = KD + 8, LDO = 24;
    // Warps 0..G-1 carry states, then H helpers, then the loading warp.  (One helper for three
    // groups was the slowest of them: 603 us where two take 510.)
    static constexpr int H = G == 3 ? 2 : G, kWarps = G + H + 1;
    static constexpr int kK = 0, kQ = kK + kC * KD, kV = kQ + kC * KD, kT = kV + kC * 16 * G, kM = kT + 2 * kCC;
    static constexpr int kGa = kM + 2 * kCC;  // (elements) the gates, float32
    static constexpr int kLoad = kGa * 2 + kChainGates * 4, kStage = up1024(kLoad);  // bytes
    // a group's (bytes): S in two planes, U and O in float32 (O's rows too)
    static constexpr int kS = 0, kU = 4 * 16 * LDK, kO = kU + 16 * kC * 4, kGroup = kO + 16 * kC * 4;
    static constexpr int kGroups = kStage + kLoad, kKeep = kGroups + G * kGroup;  // where U's planes are stored from
    static constexpr int kStages = G < 4 ? G : 1;  // of U's planes, to be stored from
    static constexpr int kBars = kKeep + kStages * 4 * 16 * kTld;
    static constexpr int kExp = kBars + 8 * (5 + 4 * G);  // (float16) the exponent of each group's S
    static constexpr size_t bytes = 1024 + kExp + 4 * G;
};

// A group's accumulators (16 x 64) between warps: float32 as the lanes hold them.
__device__ __forceinline__ void frag_put(float4* s, const float (*x)[4], const Lane& L) {
#pragma unroll
    for (int j = 0; j < kC / 8; ++j) s[j * 32 + L.l] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
}
__device__ __forceinline__ void frag_get(float (*x)[4], const float4* s, const Lane& L) {
#pragma unroll
    for (int j = 0; j < kC / 8; ++j) {
        const float4 v = s[j * 32 + L.l];
        x[j][0] = v.x;
        x[j][1] = v.y;
        x[j][2] = v.z;
        x[j][3] = v.w;
    }
}
// What the loading warp does for a backward, between two loads: group by group
// the state's planes (from where its warp put them) and U or dV (split here)
// go to the workspace.  (Done by the warps that carry the states, these stores
// cost them 400 to 1500 cycles a chunk.)
// `n` groups of a CTA, `step` bytes apart in shared memory; lane g stores group g
// and waits for its own copies, so that the groups' copies run side by side.
template <int LDK>
__device__ __forceinline__ bool store_states(e16* to, const unsigned char* tile, int step, int n, int64_t Vp, uint64_t* there,
                                             uint64_t* taken, uint32_t parity) {
    const int l = threadIdx.x & 31;
    bool ok = true;
#pragma unroll 1
    for (int g = 0; g < n; ++g) ok = warp_wait(&there[g], parity) && ok;
    if (l < n) {
        bulk_store(to + l * 16 * LDK, tile + l * step, 32 * LDK);
        bulk_store(to + (Vp + l * 16) * LDK, tile + l * step + 32 * LDK, 32 * LDK);
        bulk_commit();
        bulk_wait_read();  // (and U's or dV's of the chunk before)
        mbar_arrive(&taken[l]);
    }
    __syncwarp();
    return ok;
}
// After store_states, which has seen the stages free.  One stage a group, or
// (stages = 1) one for all, from which a group's copies then have to leave first.
template <typename T>
__device__ __forceinline__ bool store_values(e16* to, const unsigned char* frag, int step, int n, e16* stage, int stages,
                                             int64_t Vp, uint64_t* there, uint64_t* taken, uint32_t parity) {
    const Lane L;
    bool ok = true;
#pragma unroll 1
    for (int g = 0; g < n; ++g) {
        ok = warp_wait(&there[g], parity) && ok;
        float x[kC / 8][4];
        frag_get(x, reinterpret_cast<const float4*>(frag + g * step), L);
        warp_arrive(&taken[g]);
        e16* s = stage + (stages > 1 ? g * 2 * 16 * kTld : 0);
        if (stages == 1 && g > 0) {
            bulk_wait_read();
            __syncwarp();
        }
#pragma unroll
        for (int kk = 0; kk < kC / 16; ++kk) {
            const Af<2> a = from_acc<T, 2>(x[2 * kk], x[2 * kk + 1]);
            st_tile(sh(s), kTld, 16 * kk, a.r[0]);
            st_tile(sh(s) + 16 * kTld, kTld, 16 * kk, a.r[1]);
        }
        fence_async();
        __syncwarp();
        if (L.l == g) {
            bulk_store(to + g * 16 * kTld, s, 32 * kTld);
            bulk_store(to + (Vp + g * 16) * kTld, s + 16 * kTld, 32 * kTld);
            bulk_commit();
        }
    }
    return ok;
}

// What the loading warp does with float16, whose backward reads float32 (laid out
// as delta.cu's kernels have it): the states of `n` groups from their scaled
// planes, [value][key], and U or dV, [token][value].
template <int KD, int LDK>
__device__ __forceinline__ bool store_states_f32(float* to, const unsigned char* tile, int step, int n, const int* exps,
                                                 uint64_t* there, uint64_t* taken, uint32_t parity) {
    using N = Num<__half>;
    const int l = threadIdx.x & 31;
    bool ok = true;
#pragma unroll 1
    for (int g = 0; g < n; ++g) {
        ok = warp_wait(&there[g], parity) && ok;
        const float unit = pow2(-exps[g]);
        const e16* s = reinterpret_cast<const e16*>(tile + g * step);
#pragma unroll 1
        for (int i = l; i < 16 * KD / 8; i += 32) {
            const int r = i / (KD / 8), k = i % (KD / 8) * 8;
            const uint4 hi = *reinterpret_cast<const uint4*>(s + r * LDK + k), lo = *reinterpret_cast<const uint4*>(s + (16 + r) * LDK + k);
            const uint32_t *h = &hi.x, *w = &lo.x;
            float4* o = reinterpret_cast<float4*>(to + (g * 16 + r) * KD + k);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float2 a = N::unpack(h[e]), b = N::unpack(w[e]), c = N::unpack(h[e + 1]), d = N::unpack(w[e + 1]);
                o[e / 2] = make_float4((a.x + b.x) * unit, (a.y + b.y) * unit, (c.x + d.x) * unit, (c.y + d.y) * unit);
            }
        }
        warp_arrive(&taken[g]);
    }
    return ok;
}
__device__ __forceinline__ bool store_values_f32(float* to, int ld, const unsigned char* frag, int step, int n, uint64_t* there,
                                                 uint64_t* taken, uint32_t parity) {
    const Lane L;
    bool ok = true;
#pragma unroll 1
    for (int g = 0; g < n; ++g) {
        ok = warp_wait(&there[g], parity) && ok;
        float x[kC / 8][4];
        frag_get(x, reinterpret_cast<const float4*>(frag + g * step), L);
        warp_arrive(&taken[g]);
#pragma unroll
        for (int j = 0; j < kC / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) to[static_cast<int64_t>(8 * j + 2 * L.t + (e & 1)) * ld + 16 * g + L.g + (e >> 1) * 8] = x[j][e];
    }
    return ok;
}

// KEEP: S and U are written for a backward.
template <typename T, int KD, int G, bool KEEP>
__global__ void __launch_bounds__(Fwd<KD, G>::kWarps * 32, 1) planes_chain_k(const __grid_constant__ DArgs a, const __grid_constant__ Maps maps) {
    using Sm = Fwd<KD, G>;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / (a.Hv / a.Hk);
    const int len = row_length(a, b), nc = (len + kC - 1) / kC;
    const int warp = threadIdx.x >> 5, vb = blockIdx.x * 16 * G;
    const Lane L;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    unsigned char* smem = align_smem(smem_raw);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sm::kBars);
    uint64_t* empty = full + 2;
    uint64_t* land = empty + 2;
    uint64_t *s_full = land + 1, *s_empty = s_full + G, *u_full = s_empty + G, *u_empty = u_full + G;
    int* s_exp = reinterpret_cast<int*>(smem + Sm::kExp);
    const int64_t head = static_cast<int64_t>(b) * a.Hv + h;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], G + Sm::H);
        }
        mbar_init(land, 1);
        for (int i = 0; i < G; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], KEEP ? 2 : 1);
            mbar_init(&u_full[i], 1);
            mbar_init(&u_empty[i], KEEP ? 2 : 1);
        }
        fence_mbar_init();
    }
    __syncthreads();
    bool ok = true;
    if (warp == Sm::kWarps - 1) {
        // ---- loads ----
        auto load = [&](int c) {
            e16* e = reinterpret_cast<e16*>(smem + (c & 1) * Sm::kStage);
            const int t0 = c * kC, rows = min(kC, len - t0);
            const bool tail = rows < min(kC, a.L - t0);
            uint64_t* bar = tail ? land : &full[c & 1];
            ok = warp_wait(&empty[c & 1], ((c >> 1) & 1) ^ 1) && ok;
            if (L.l == 0) {
                const int64_t id = head * a.n + c;
                mbar_expect_tx(bar, Sm::kLoad - Gates<T>::less);
#pragma unroll
                for (int x = 0; x < KD; x += 64) tma_load(e + Sm::kK + x * kC, &maps.k, bar, x, t0, hk, b);
                bulk_load(e + Sm::kT, static_cast<const e16*>(a.T) + id * 2 * kCC, 4 * kCC, bar);
#pragma unroll
                for (int g = 0; g < G; ++g) tma_load(e + Sm::kV + g * kC * 16, &maps.v, bar, vb + 16 * g, t0, h, b);
                bulk_load(e + Sm::kGa, a.gates + id * kGates + Gates<T>::first, Gates<T>::n * 4, bar);
#pragma unroll
                for (int x = 0; x < KD; x += 64) tma_load(e + Sm::kQ + x * kC, &maps.q, bar, x, t0, hk, b);
                bulk_load(e + Sm::kM, static_cast<const e16*>(a.M) + id * 2 * kCC, 4 * kCC, bar);
            }
            __syncwarp();
            if (tail) {
                ok = warp_wait(land, 0) && ok;
                zero_rows<64>(e + Sm::kK, 2 * (KD / 64), rows);  // keys and queries
                zero_rows<16>(e + Sm::kV, G, rows);
                warp_arrive(&full[c & 1]);
            }
        };
#pragma unroll 1
        for (int c = KEEP ? -1 : 0; c < nc && ok; ++c) {
            if constexpr (!KEEP) {
                load(c);
            } else {  // a load ahead of the stores
                if (c + 1 < nc) load(c + 1);
                if (c < 0) continue;
                const int n = min(G, (a.Vp - vb) / 16);
                if constexpr (Scaled<T>) {
                    const int64_t id = head * a.n + c;
                    ok = store_states_f32<KD, Sm::LDK>(static_cast<float*>(a.S) + (id * a.Vp + vb) * KD, smem + Sm::kGroups + Sm::kS,
                                                       Sm::kGroup, n, s_exp, s_full, s_empty, c & 1) && ok;
                    ok = store_values_f32(static_cast<float*>(a.U) + id * kC * a.Vp + vb, a.Vp, smem + Sm::kGroups + Sm::kU, Sm::kGroup, n,
                                          u_full, u_empty, c & 1) && ok;
                } else {
                    const int64_t id = (head * a.n + c) * 2 * a.Vp + vb;
                    ok = store_states<Sm::LDK>(static_cast<e16*>(a.S) + id * Sm::LDK, smem + Sm::kGroups + Sm::kS, Sm::kGroup, n,
                                               a.Vp, s_full, s_empty, c & 1) && ok;
                    ok = store_values<T>(static_cast<e16*>(a.U) + id * kTld, smem + Sm::kGroups + Sm::kU, Sm::kGroup, n,
                                         reinterpret_cast<e16*>(smem + Sm::kKeep), Sm::kStages, a.Vp, u_full, u_empty, c & 1) && ok;
                }
            }
        }
        if constexpr (KEEP) bulk_wait_all();
        return;
    }
    if (warp < G) {
        // ---- a state of 16 value columns ----
        const int v0 = vb + warp * 16;
        const bool on = v0 < a.Vp;
        unsigned char* mine = smem + Sm::kGroups + warp * Sm::kGroup;
        const Sh sS = sh(mine + Sm::kS);
        float4* sU = reinterpret_cast<float4*>(mine + Sm::kU);
        float S[KD / 8][4];
        state_load<KD>(S, a.initial ? a.initial + head * a.K * a.V : nullptr, a.K, a.V, v0, L);
        int se = 0;  // (float16) S holds 2^se times the state
        for (int c = 0; c < nc && ok; ++c) {
            const unsigned char* st = smem + (c & 1) * Sm::kStage;
            const e16* e = reinterpret_cast<const e16*>(st);
            const Sh es = sh(e);
            const float* ga = reinterpret_cast<const float*>(e + Sm::kGa);
            const float *gam = ga + Gates<T>::gam, *dec = ga + Gates<T>::dec;
            const int64_t id = head * a.n + c;
            if (!on) {
                ok = warp_wait(&full[c & 1], (c >> 1) & 1);
            } else {
                ok = warp_wait2(&full[c & 1], (c >> 1) & 1, &s_empty[warp], (c & 1) ^ 1);
                float s_max = 0.f;
                auto scale_state = [&](float largest) {  // by the largest value of S and of what is added to it
                    const int e = max(-kMaxExp, min(kMaxExp, se + scale_exp(__float_as_uint(largest)))) - se;
                    if (e == 0) return 1.f;
                    scale_tile<KD / 8>(S, pow2(e));
                    se += e;
                    return pow2(e);
                };
                if constexpr (Scaled<T>) {
                    s_max = __uint_as_float(max_bits<KD / 8>(S));
                    s_max *= scale_state(s_max);
                    if (L.l == 0) s_exp[warp] = se;
                }
                // (K S0)^T, S in two planes; the next 16 columns of S are split between the products
                float X[kC / 8][4] = {};
                {
                    Af<2> as[2];
                    as[0] = from_acc<T, 2>(S[0], S[1]);
                    steps<KD / 16>(
                        [&](int i, uint32_t(*f)[4]) {
#pragma unroll
                            for (int p = 0; p < 4; ++p) ld_b128<false>(f[p], es + Sm::kK, 16 * p, 16 * i);
                        },
                        [&](int i, const uint32_t(*f)[4]) {
                            Af<2>& af = as[i & 1];
                            st_tile(sS, Sm::LDK, 16 * i, af.r[0]);
                            st_tile(sS + 16 * Sm::LDK, Sm::LDK, 16 * i, af.r[1]);
                            mma_step_with<T>(X, af, f, [&](int q) {
                                if (i + 1 < KD / 16) {
                                    const float* s = S[2 * i + 2 + q / 2];
                                    from_acc_part<T>(as[(i + 1) & 1], q, s[2 * (q & 1)], s[2 * (q & 1) + 1]);
                                }
                            });
                        });
                }
                if constexpr (KEEP) fence_async();
                warp_arrive(&s_full[warp]);
                const bool u_free = mbar_try_wait(&u_empty[warp], (c & 1) ^ 1);
                // X = V^T - gam (K S0)^T
#pragma unroll
                for (int p = 0; p < kC / 16; ++p) {
                    uint32_t r[4];
                    ld_at32(r, es + Sm::kV + warp * kC * 16, 16 * p);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float2 f = *reinterpret_cast<const float2*>(gam + 16 * p + 8 * i + 2 * L.t);
                        if constexpr (Scaled<T>) {
                            f.x *= pow2(-se);
                            f.y *= pow2(-se);
                        }
                        float* x = X[2 * p + i];
                        const float2 lo = Num<T>::unpack(r[2 * i]), hi = Num<T>::unpack(r[2 * i + 1]);
                        x[0] = fmaf(-f.x, x[0], lo.x);
                        x[1] = fmaf(-f.y, x[1], lo.y);
                        x[2] = fmaf(-f.x, x[2], hi.x);
                        x[3] = fmaf(-f.y, x[3], hi.y);
                    }
                }
                // U^T = X T'^T, both in two planes; between the products S is scaled, and the first
                // 16 tokens of U, which are done after theirs, are split for the update (float16: when
                // all of U is known)
                int xe = 0;
                if constexpr (Scaled<T>) {
                    xe = scale_exp(max_bits<kC / 8>(X));
                    if (xe != 0) scale_tile<kC / 8>(X, pow2(xe));
                }
                float U[kC / 8][4] = {};
                const float gc = gam[kC - 1];
                auto decayed = [&](Af<2>& to, int kk, int q) {
                    float2 d = *reinterpret_cast<const float2*>(dec + 16 * kk + 8 * (q / 2) + 2 * L.t);
                    if constexpr (Scaled<T>) {
                        d.x *= pow2(se);
                        d.y *= pow2(se);
                    }
                    const float* u = U[2 * kk + q / 2];
                    from_acc_part<T>(to, q, u[2 * (q & 1)] * d.x, u[2 * (q & 1) + 1] * d.y);
                };
                Af<2> ud[2];
                {
                    Af<2> ax[2];
                    ax[0] = from_acc<T, 2>(X[0], X[1]);
                    steps<8>(  // the low plane of T', then the high one
                        [&](int i, uint32_t(*f)[4]) {
#pragma unroll
                            for (int p = 0; p < 4; ++p)
                                if (p >= i / 2) ld_b<false>(f[p], es + Sm::kT + (i & 1 ? 0 : kCC), kTld, 16 * p, 16 * (i / 2));
                        },
                        [&](int i, const uint32_t(*f)[4]) {
                            const int kk = i / 2;
                            const Af<2>& af = ax[kk & 1];
                            auto side = [&](int q) {
                                if (4 * i + q < KD / 4) {  // half a tile of S in each of 32 places
                                    float* s = S[(4 * i + q) / 2];
                                    s[2 * (q & 1)] *= gc;
                                    s[2 * (q & 1) + 1] *= gc;
                                }
                                if ((i & 1) && kk + 1 < 4) {
                                    const float* x = X[2 * kk + 2 + q / 2];
                                    from_acc_part<T>(ax[(kk + 1) & 1], q, x[2 * (q & 1)], x[2 * (q & 1) + 1]);
                                }
                                if (!Scaled<T> && i == 4) decayed(ud[0], 0, q);
                            };
                            if (i & 1) mma_step_with<T>(U, af, f, side, kk);
                            else mma_step_with<T>(U, high(af), f, side, kk);
                        });
                }
                if constexpr (Scaled<T>) {  // beta, which T' was made without
                    const float unit = tile_unit(e + Sm::kT);
                    float u_max = 0.f;
#pragma unroll
                    for (int j = 0; j < kC / 8; ++j) {
                        const float2 r = *reinterpret_cast<const float2*>(ga + Gates<T>::beta + 8 * j + 2 * L.t);
                        const float2 d = *reinterpret_cast<const float2*>(dec + 8 * j + 2 * L.t);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            U[j][i] = U[j][i] * pow2(-xe) * ((i & 1 ? r.y : r.x) * unit);
                            u_max = fmaxf(u_max, fabsf(U[j][i] * (i & 1 ? d.y : d.x)));
                        }
                    }
                    u_max = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(u_max)));
                    scale_state(fmaxf(s_max * gc, u_max * pow2(se)));
#pragma unroll
                    for (int q = 0; q < 4; ++q) decayed(ud[0], 0, q);
                }
                ok = warp_wait_asked(u_free, &u_empty[warp], (c & 1) ^ 1) && ok;
                frag_put(sU, U, L);
                warp_arrive(&u_full[warp]);
                // S^T = gam_63 S^T + (d U)^T K
                {
                    constexpr int Q = KD / 64;
                    steps<4 * Q>(
                        [&](int i, uint32_t(*f)[4]) {
#pragma unroll
                            for (int p = 0; p < 4; ++p) ld_b128<true>(f[p], es + Sm::kK, 64 * (i % Q) + 16 * p, 16 * (i / Q));
                        },
                        [&](int i, const uint32_t(*f)[4]) {
                            const int kk = i / Q;
                            mma_step_with<T>(S + 8 * (i % Q), ud[kk & 1], f, [&](int q) {
                                if (kk + 1 < 4 && i % Q == 0) decayed(ud[(kk + 1) & 1], kk + 1, q);
                            });
                        });
                }
            }
            warp_arrive(&empty[c & 1]);
        }
        if constexpr (Scaled<T>) scale_tile<KD / 8>(S, pow2(-se));
        if (on && a.final_state && ok) state_store<KD>(S, a.final_state + head * a.K * a.V, a.K, a.V, v0, L);
        return;
    }
    // ---- outputs of the groups g = helper, helper + H, .. ----
    const int helper = warp - G;
    const int64_t ost = static_cast<int64_t>(a.Hv) * a.V;
    e16* out = static_cast<e16*>(a.out) + static_cast<int64_t>(b) * a.L * ost + static_cast<int64_t>(h) * a.V;
    for (int c = 0; c < nc && ok; ++c) {
        const unsigned char* st = smem + (c & 1) * Sm::kStage;
        const e16* e = reinterpret_cast<const e16*>(st);
        const Sh es = sh(e);
        const float* sgam = reinterpret_cast<const float*>(e + Sm::kGa) + Gates<T>::sgam;
        const int rows = min(kC, len - c * kC), all = min(kC, a.L - c * kC);
        ok = warp_wait(&full[c & 1], (c >> 1) & 1);
        // (Loops over the groups are not unrolled: what the warps of a CTA run in a chunk has to fit
        // the instruction cache.  O waits in shared memory between its two products.)
#pragma unroll 1
        for (int g = helper; g < G; g += Sm::H) {
            if (vb + 16 * g >= a.Vp) break;
            unsigned char* theirs = smem + Sm::kGroups + g * Sm::kGroup;
            const Sh sS = sh(theirs + Sm::kS);
            float4* sO = reinterpret_cast<float4*>(theirs + Sm::kO);
            ok = warp_wait(&s_full[g], c & 1) && ok;
            // scale gam Q S0 (with S in one plane y is off by 2.2e-3 in the norm instead of 1.7e-3, and
            // by 2^-9 |q| |S| where the terms cancel)
            float O[kC / 8][4] = {};
            Af<2> as[2];
            steps<KD / 16>(
                [&](int k, uint32_t(*f)[4]) {
                    ld_a(as[k & 1].r[0], sS, Sm::LDK, 0, 16 * k);
                    ld_a(as[k & 1].r[1], sS + 16 * Sm::LDK, Sm::LDK, 0, 16 * k);
#pragma unroll
                    for (int p = 0; p < 4; ++p) ld_b128<false>(f[p], es + Sm::kQ, 16 * p, 16 * k);
                },
                [&](int k, const uint32_t(*f)[4]) { mma_step<T>(O, as[k & 1], f); });
            const float unit = Scaled<T> ? pow2(-s_exp[g]) : 1.f;
            warp_arrive(&s_empty[g]);
#pragma unroll
            for (int j = 0; j < kC / 8; ++j) {
                float2 f = *reinterpret_cast<const float2*>(sgam + 8 * j + 2 * L.t);
                if constexpr (Scaled<T>) {
                    f.x *= unit;
                    f.y *= unit;
                }
                sO[j * 32 + L.l] = make_float4(O[j][0] * f.x, O[j][1] * f.y, O[j][2] * f.x, O[j][3] * f.y);
            }
        }
#pragma unroll 1
        for (int g = helper; g < G; g += Sm::H) {
            const int v0 = vb + 16 * g;
            if (v0 >= a.Vp) break;
            unsigned char* theirs = smem + Sm::kGroups + g * Sm::kGroup;
            e16* sO = reinterpret_cast<e16*>(theirs + Sm::kO);
            float O[kC / 8][4], U[kC / 8][4];
            frag_get(O, reinterpret_cast<const float4*>(sO), L);
            ok = warp_wait(&u_full[g], c & 1) && ok;
            frag_get(U, reinterpret_cast<const float4*>(theirs + Sm::kU), L);
            warp_arrive(&u_empty[g]);
            // float16: M U by itself, as U and M are scaled
            float Y[Scaled<T> ? kC / 8 : 1][4] = {};
            int ue = 0;
            if constexpr (Scaled<T>) {
                ue = scale_exp(max_bits<kC / 8>(U));
                scale_tile<kC / 8>(U, pow2(ue));
            }
            auto& sums = *[&]() { if constexpr (Scaled<T>) return &Y; else return &O; }();
            Af<2> au;
            steps<8>(
                [&](int k, uint32_t(*f)[4]) {
#pragma unroll
                    for (int p = 0; p < 4; ++p)
                        if (p >= k / 2) ld_b<false>(f[p], es + Sm::kM + (k & 1 ? 0 : kCC), kTld, 16 * p, 16 * (k / 2));
                },
                [&](int k, const uint32_t(*f)[4]) {
                    if (k & 1) {
                        mma_step<T>(sums, au, f, k / 2);
                    } else {
                        au = from_acc<T, 2>(U[k], U[k + 1]);
                        mma_step<T>(sums, high(au), f, k / 2);
                    }
                });
            if constexpr (Scaled<T>) {
                const float fm = tile_unit(e + Sm::kM);
#pragma unroll
                for (int j = 0; j < kC / 8; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) O[j][i] = fmaf(Y[j][i] * pow2(-ue), fm, O[j][i]);
            }
            // rows of 16 values through shared memory: 32 bytes a token, two lanes each
            __syncwarp();
#pragma unroll
            for (int p = 0; p < kC / 16; ++p) {
                const Af<1> o = from_acc<T, 1>(O[2 * p], O[2 * p + 1]);
                st_tile_t(sh(sO), Sm::LDO, 16 * p, o.r[0]);
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 16 * j + (L.l >> 1), col = (L.l & 1) * 8;
                if (r < all && v0 + col < a.V) {
                    uint4 x = *reinterpret_cast<const uint4*>(sO + r * Sm::LDO + col);
                    if (r >= rows) x = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(c) * kC + r) * ost + v0 + col) = x;
                }
            }
            __syncwarp();
        }
        warp_arrive(&empty[c & 1]);
    }
    for (int g = helper; g < G; g += Sm::H)  // behind the sequence
        for (int64_t i = static_cast<int64_t>(nc) * kC * 2 + L.l; i < static_cast<int64_t>(a.L) * 2; i += 32) {
            const int v = vb + 16 * g + (i & 1) * 8;
            if (v < a.V) *reinterpret_cast<uint4*>(out + (i >> 1) * ost + v) = make_uint4(0, 0, 0, 0);
        }
}

// ----------------------------------------------------------------------------
// the reverse chain
// ----------------------------------------------------------------------------
// All operands in two planes (with dV in one, float32 gradients of gates were off
// by 1.2e-3 of their norm).
template <int KD, int G>
struct Rev {
    static constexpr int LDK = KD + 8;
    static constexpr int H = G, kWarps = G + H + 1;
    static constexpr int kK = 0, kQ = kK + kC * KD, kD = kQ + kC * KD, kT = kD + kC * 16 * G, kM = kT + 2 * kCC;
    static constexpr int kGa = kM + 2 * kCC;
    static constexpr int kLoad = kGa * 2 + kChainGates * 4, kStage = up1024(kLoad);
    // a group's (bytes): dS in two planes, dV and (scale gam dO)^T Q in float32
    static constexpr int kS = 0, kX = 4 * 16 * LDK, kZ = kX + 16 * kC * 4, kGroup = kZ + 16 * KD * 4;
    static constexpr int kGroups = kStage + kLoad, kKeep = kGroups + G * kGroup;
    static constexpr int kStages = G == 3 && KD == 128 ? 1 : G;
    static constexpr int kBars = kKeep + kStages * 4 * 16 * kTld;
    static constexpr int kExp = kBars + 8 * (5 + 6 * G);  // (float16) the exponent of each group's dS
    static constexpr size_t bytes = 1024 + kExp + 4 * G;
};

template <typename T, int KD, int G>
__global__ void __launch_bounds__(Rev<KD, G>::kWarps * 32, 1) planes_rchain_k(const __grid_constant__ DArgs a, const __grid_constant__ Maps maps) {
    using Sm = Rev<KD, G>;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / (a.Hv / a.Hk);
    const int len = row_length(a, b), nc = (len + kC - 1) / kC;
    const int warp = threadIdx.x >> 5, vb = blockIdx.x * 16 * G;
    const Lane L;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    unsigned char* smem = align_smem(smem_raw);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sm::kBars);
    uint64_t* empty = full + 2;
    uint64_t* land = empty + 2;
    uint64_t *z_full = land + 1, *z_empty = z_full + G;
    uint64_t *s_full = z_empty + G, *s_empty = s_full + G, *x_full = s_empty + G, *x_empty = x_full + G;
    int* s_exp = reinterpret_cast<int*>(smem + Sm::kExp);
    const e16* tiles = static_cast<const e16*>(Scaled<T> ? a.Tr : a.T);
    const int64_t head = static_cast<int64_t>(b) * a.Hv + h;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], G + Sm::H);
        }
        mbar_init(land, 1);
        for (int i = 0; i < 6 * G; ++i) mbar_init(&z_full[i], 1);
        fence_mbar_init();
    }
    __syncthreads();
    bool ok = true;
    if (warp == Sm::kWarps - 1) {
        auto load = [&](int i) {
            const int c = nc - 1 - i;
            e16* e = reinterpret_cast<e16*>(smem + (i & 1) * Sm::kStage);
            const int t0 = c * kC, rows = min(kC, len - t0);
            const bool tail = rows < min(kC, a.L - t0);
            uint64_t* bar = tail ? land : &full[i & 1];
            ok = warp_wait(&empty[i & 1], ((i >> 1) & 1) ^ 1) && ok;
            if (L.l == 0) {
                const int64_t id = head * a.n + c;
                mbar_expect_tx(bar, Sm::kLoad - Gates<T>::less);
#pragma unroll
                for (int x = 0; x < KD; x += 64) tma_load(e + Sm::kK + x * kC, &maps.k, bar, x, t0, hk, b);
#pragma unroll
                for (int g = 0; g < G; ++g) tma_load(e + Sm::kD + g * kC * 16, &maps.d, bar, vb + 16 * g, t0, h, b);
                bulk_load(e + Sm::kM, static_cast<const e16*>(a.M) + id * 2 * kCC, 4 * kCC, bar);
                bulk_load(e + Sm::kGa, a.gates + id * kGates + Gates<T>::first, Gates<T>::n * 4, bar);
                bulk_load(e + Sm::kT, tiles + id * 2 * kCC, 4 * kCC, bar);
#pragma unroll
                for (int x = 0; x < KD; x += 64) tma_load(e + Sm::kQ + x * kC, &maps.q, bar, x, t0, hk, b);
            }
            __syncwarp();
            if (tail) {
                ok = warp_wait(land, 0) && ok;
                zero_rows<64>(e + Sm::kK, 2 * (KD / 64), rows);
                zero_rows<16>(e + Sm::kD, G, rows);
                fence_async();  // later chunks are copied over these rows
                warp_arrive(&full[i & 1]);
            }
        };
#pragma unroll 1
        for (int i = -1; i < nc && ok; ++i) {  // a load ahead of the stores
            if (i + 1 < nc) load(i + 1);
            if (i < 0) continue;
            const int n = min(G, (a.Vp - vb) / 16);
            if constexpr (Scaled<T>) {
                const int64_t id = head * a.n + nc - 1 - i;
                ok = store_states_f32<KD, Sm::LDK>(static_cast<float*>(a.dS) + (id * a.Vp + vb) * KD, smem + Sm::kGroups + Sm::kS,
                                                   Sm::kGroup, n, s_exp, s_full, s_empty, i & 1) && ok;
                ok = store_values_f32(static_cast<float*>(a.dV) + id * kC * a.Vp + vb, a.Vp, smem + Sm::kGroups + Sm::kX, Sm::kGroup, n,
                                      x_full, x_empty, i & 1) && ok;
            } else {
                const int64_t id = (head * a.n + nc - 1 - i) * 2 * a.Vp + vb;
                ok = store_states<Sm::LDK>(static_cast<e16*>(a.dS) + id * Sm::LDK, smem + Sm::kGroups + Sm::kS, Sm::kGroup, n, a.Vp,
                                           s_full, s_empty, i & 1) && ok;
                ok = store_values<T>(static_cast<e16*>(a.dV) + id * kTld, smem + Sm::kGroups + Sm::kX, Sm::kGroup, n,
                                     reinterpret_cast<e16*>(smem + Sm::kKeep), Sm::kStages, a.Vp, x_full, x_empty, i & 1) && ok;
            }
        }
        bulk_wait_all();
        return;
    }
    if (warp < G) {
        const int v0 = vb + warp * 16;
        const bool on = v0 < a.Vp;
        unsigned char* mine = smem + Sm::kGroups + warp * Sm::kGroup;
        const Sh sS = sh(mine + Sm::kS);
        float4* sX = reinterpret_cast<float4*>(mine + Sm::kX);
        const float4* sZ = reinterpret_cast<const float4*>(mine + Sm::kZ);
        float S[KD / 8][4];  // dS^T
        state_load<KD>(S, a.dfinal ? a.dfinal + head * a.K * a.V : nullptr, a.K, a.V, v0, L);
        int se = 0;  // (float16) S holds 2^se times dS
        for (int i = 0; i < nc && ok; ++i) {
            const e16* e = reinterpret_cast<const e16*>(smem + (i & 1) * Sm::kStage);
            const Sh es = sh(e);
            const float* ga = reinterpret_cast<const float*>(e + Sm::kGa);
            const float *gam = ga + Gates<T>::gam, *dec = ga + Gates<T>::dec;
            if (!on) {
                ok = warp_wait(&full[i & 1], (i >> 1) & 1);
            } else {
                ok = warp_wait2(&full[i & 1], (i >> 1) & 1, &s_empty[warp], (i & 1) ^ 1);
                auto scale_state = [&](uint32_t bits) {
                    const int e = max(-kMaxExp, min(kMaxExp, se + scale_exp(bits))) - se;
                    if (e == 0) return;
                    scale_tile<KD / 8>(S, pow2(e));
                    se += e;
                };
                if constexpr (Scaled<T>) {
                    scale_state(max_bits<KD / 8>(S));
                    if (L.l == 0) s_exp[warp] = se;
                }
                float U[kC / 8][4] = {};  // dU^T = d (K dS1)^T + dO^T M
                {
                    Af<2> as[2];
                    as[0] = from_acc<T, 2>(S[0], S[1]);
                    steps<KD / 16>(
                        [&](int k, uint32_t(*f)[4]) {
#pragma unroll
                            for (int p = 0; p < 4; ++p) ld_b128<false>(f[p], es + Sm::kK, 16 * p, 16 * k);
                        },
                        [&](int k, const uint32_t(*f)[4]) {
                            Af<2>& af = as[k & 1];
                            st_tile(sS, Sm::LDK, 16 * k, af.r[0]);
                            st_tile(sS + 16 * Sm::LDK, Sm::LDK, 16 * k, af.r[1]);
                            mma_step_with<T>(U, af, f, [&](int q) {
                                if (k + 1 < KD / 16) {
                                    const float* s = S[2 * k + 2 + q / 2];
                                    from_acc_part<T>(as[(k + 1) & 1], q, s[2 * (q & 1)], s[2 * (q & 1) + 1]);
                                }
                            });
                        });
                }
                fence_async();
                warp_arrive(&s_full[warp]);
                const bool z_there = mbar_try_wait(&z_full[warp], i & 1), x_free = mbar_try_wait(&x_empty[warp], (i & 1) ^ 1);
#pragma unroll
                for (int j = 0; j < kC / 8; ++j) {
                    float2 f = *reinterpret_cast<const float2*>(dec + 8 * j + 2 * L.t);
                    if constexpr (Scaled<T>) {
                        f.x *= pow2(-se);
                        f.y *= pow2(-se);
                    }
                    U[j][0] *= f.x;
                    U[j][1] *= f.y;
                    U[j][2] *= f.x;
                    U[j][3] *= f.y;
                }
                int ue = 0;  // (float16) U holds 2^ue dU
                {
                    float Y[Scaled<T> ? kC / 8 : 1][4] = {};  // float16: dO^T M by itself, as M is scaled
                    auto& sums = *[&]() { if constexpr (Scaled<T>) return &Y; else return &U; }();
                    Af<1> ad[2];
                    steps<8>(
                        [&](int k, uint32_t(*f)[4]) {
                            if (!(k & 1)) ld_at32(ad[(k / 2) & 1].r[0], es + Sm::kD + warp * kC * 16, 8 * k);
#pragma unroll
                            for (int p = 0; p < 4; ++p)
                                if (p <= k / 2) ld_b<true>(f[p], es + Sm::kM + (k & 1 ? 0 : kCC), kTld, 16 * p, 16 * (k / 2));
                        },
                        [&](int k, const uint32_t(*f)[4]) { mma_step<T>(sums, ad[(k / 2) & 1], f, 0, k / 2 + 1); });
                    if constexpr (Scaled<T>) {
                        const float fm = tile_unit(e + Sm::kM);
#pragma unroll
                        for (int j = 0; j < kC / 8; ++j)
#pragma unroll
                            for (int x = 0; x < 4; ++x) U[j][x] = fmaf(Y[j][x], fm, U[j][x]);
                        ue = scale_exp(max_bits<kC / 8>(U));
                        if (ue != 0) scale_tile<kC / 8>(U, pow2(ue));
                    }
                }
                ok = warp_wait_asked(z_there, &z_full[warp], i & 1) && ok;
                // dV^T = dU^T T', the last 16 tokens first; between the products dS is scaled and
                // (scale gam dO)^T Q added, and the last tokens of dV, done first, are split for the update
                // (float16: beta comes after the product, and then the split)
                float X[kC / 8][4] = {};
                const float gc = gam[kC - 1];
                auto decayed = [&](Af<2>& to, int kk, int q) {
                    float2 d = *reinterpret_cast<const float2*>(gam + 16 * kk + 8 * (q / 2) + 2 * L.t);
                    if constexpr (Scaled<T>) {
                        d.x *= pow2(se);
                        d.y *= pow2(se);
                    }
                    const float* u = X[2 * kk + q / 2];
                    from_acc_part<T>(to, q, -u[2 * (q & 1)] * d.x, -u[2 * (q & 1) + 1] * d.y);
                };
                Af<2> xd[2];
                {
                    Af<2> au[2];
                    au[1] = from_acc<T, 2>(U[6], U[7]);
                    steps<8>(
                        [&](int k, uint32_t(*f)[4]) {
                            const int kk = 3 - k / 2;
#pragma unroll
                            for (int p = 0; p < 4; ++p)
                                if (p <= kk) ld_b<true>(f[p], es + Sm::kT + (k & 1 ? 0 : kCC), kTld, 16 * p, 16 * kk);
                        },
                        [&](int k, const uint32_t(*f)[4]) {
                            const int kk = 3 - k / 2;
                            const Af<2>& af = au[kk & 1];
                            auto side = [&](int q) {
                                if (!(q & 1)) {  // dS: KD / 8 tiles in 8 steps of 2
                                    constexpr int N = KD / 8;
                                    const int j = k * 2 + q / 2;
                                    if (j < N) {
                                        float4 z = sZ[j * 32 + L.l];
                                        if constexpr (Scaled<T>) z = make_float4(z.x * pow2(se), z.y * pow2(se), z.z * pow2(se), z.w * pow2(se));
                                        S[j][0] = fmaf(gc, S[j][0], z.x);
                                        S[j][1] = fmaf(gc, S[j][1], z.y);
                                        S[j][2] = fmaf(gc, S[j][2], z.z);
                                        S[j][3] = fmaf(gc, S[j][3], z.w);
                                    }
                                }
                                if ((k & 1) && kk > 0) {
                                    const float* u = U[2 * kk - 2 + q / 2];
                                    from_acc_part<T>(au[(kk - 1) & 1], q, u[2 * (q & 1)], u[2 * (q & 1) + 1]);
                                }
                                if (!Scaled<T> && k == 4) decayed(xd[1], 3, q);
                            };
                            if (k & 1) mma_step_with<T>(X, af, f, side, 0, kk + 1);
                            else mma_step_with<T>(X, high(af), f, side, 0, kk + 1);
                        });
                }
                warp_arrive(&z_empty[warp]);
                if constexpr (Scaled<T>) {
                    const float unit = tile_unit(e + Sm::kT);
                    float x_max = 0.f;
#pragma unroll
                    for (int j = 0; j < kC / 8; ++j) {
                        const float2 r = *reinterpret_cast<const float2*>(ga + Gates<T>::beta + 8 * j + 2 * L.t);
                        const float2 d = *reinterpret_cast<const float2*>(gam + 8 * j + 2 * L.t);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            X[j][x] = X[j][x] * pow2(-ue) * ((x & 1 ? r.y : r.x) * unit);
                            x_max = fmaxf(x_max, fabsf(X[j][x] * (x & 1 ? d.y : d.x)));
                        }
                    }
                    x_max = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x_max))) * pow2(se);
                    scale_state(max(max_bits<KD / 8>(S), __float_as_uint(x_max)));
#pragma unroll
                    for (int q = 0; q < 4; ++q) decayed(xd[1], 3, q);
                }
                ok = warp_wait_asked(x_free, &x_empty[warp], (i & 1) ^ 1) && ok;
                frag_put(sX, X, L);
                warp_arrive(&x_full[warp]);
                // dS^T -= (gam dV)^T K
                {
                    constexpr int Q = KD / 64;
                    steps<4 * Q>(
                        [&](int k, uint32_t(*f)[4]) {
#pragma unroll
                            for (int p = 0; p < 4; ++p)
                                ld_b128<true>(f[p], es + Sm::kK, 64 * (k % Q) + 16 * p, 16 * (3 - k / Q));
                        },
                        [&](int k, const uint32_t(*f)[4]) {
                            const int kk = 3 - k / Q;
                            mma_step_with<T>(S + 8 * (k % Q), xd[kk & 1], f, [&](int q) {
                                if (kk > 0 && k % Q == 0) decayed(xd[(kk - 1) & 1], kk - 1, q);
                            });
                        });
                }
            }
            warp_arrive(&empty[i & 1]);
        }
        if constexpr (Scaled<T>) scale_tile<KD / 8>(S, pow2(-se));
        if (on && a.dinitial && ok) state_store<KD>(S, a.dinitial + head * a.K * a.V, a.K, a.V, v0, L);
        return;
    }
    // ---- (scale gam dO)^T Q of the groups ----
    for (int i = 0; i < nc && ok; ++i) {
        const e16* e = reinterpret_cast<const e16*>(smem + (i & 1) * Sm::kStage);
        const Sh es = sh(e);
        const float* sgam = reinterpret_cast<const float*>(e + Sm::kGa) + Gates<T>::sgam;
        ok = warp_wait(&full[i & 1], (i >> 1) & 1);
        for (int g = warp - G; g < G; g += Sm::H) {
            if (vb + 16 * g >= a.Vp) break;
            float Z[KD / 8][4] = {};
            Af<2> af;
            constexpr int Q = KD / 64;
            int de = 0;  // (float16) of scale gam dO
            if constexpr (Scaled<T>) {
                float m = 0.f;
#pragma unroll 1
                for (int kk = 0; kk < kC / 16; ++kk) {
                    uint32_t r[4];
                    ld_at32(r, es + Sm::kD + g * kC * 16, 16 * kk);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float2 d = *reinterpret_cast<const float2*>(sgam + 16 * kk + 8 * x + 2 * L.t);
                        const float2 lo = Num<T>::unpack(r[2 * x]), hi = Num<T>::unpack(r[2 * x + 1]);
                        m = fmaxf(m, fmaxf(fmaxf(fabsf(lo.x * d.x), fabsf(lo.y * d.y)), fmaxf(fabsf(hi.x * d.x), fabsf(hi.y * d.y))));
                    }
                }
                de = scale_exp(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
            }
            steps<4 * Q>(
                [&](int k, uint32_t(*f)[4]) {
#pragma unroll
                    for (int p = 0; p < 4; ++p) ld_b128<true>(f[p], es + Sm::kQ, 64 * (k % Q) + 16 * p, 16 * (k / Q));
                },
                [&](int k, const uint32_t(*f)[4]) {
                    const int kk = k / Q;
                    if (k % Q == 0) {
                        uint32_t r[4];
                        ld_at32(r, es + Sm::kD + g * kC * 16, 16 * kk);
                        float y[2][4];
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float2 d = *reinterpret_cast<const float2*>(sgam + 16 * kk + 8 * x + 2 * L.t);
                            if constexpr (Scaled<T>) {
                                d.x *= pow2(de);
                                d.y *= pow2(de);
                            }
                            const float2 lo = Num<T>::unpack(r[2 * x]), hi = Num<T>::unpack(r[2 * x + 1]);
                            y[x][0] = lo.x * d.x;
                            y[x][1] = lo.y * d.y;
                            y[x][2] = hi.x * d.x;
                            y[x][3] = hi.y * d.y;
                        }
                        af = from_acc<T, 2>(y[0], y[1]);
                    }
                    mma_step<T>(Z + 8 * (k % Q), af, f);
                });
            float4* sZ = reinterpret_cast<float4*>(smem + Sm::kGroups + g * Sm::kGroup + Sm::kZ);
            ok = warp_wait(&z_empty[g], (i & 1) ^ 1) && ok;
            if constexpr (Scaled<T>) scale_tile<KD / 8>(Z, pow2(-de));
#pragma unroll
            for (int j = 0; j < KD / 8; ++j) sZ[j * 32 + L.l] = make_float4(Z[j][0], Z[j][1], Z[j][2], Z[j][3]);
            warp_arrive(&z_full[g]);
        }
        warp_arrive(&empty[i & 1]);
    }
}

// ----------------------------------------------------------------------------
// dQ, dK, dV, dbeta and dg of a chunk
// ----------------------------------------------------------------------------
// A CTA goes through chunks (of a key head) in a grid-stride loop with sixteen
// warps, of which the first also asks for the loads of the tile after next (a
// seventeenth warp would leave 112 registers a lane).  Eight (the readers) hold dQ and dK_read, eight
// (the writers) dK_write and N or E; of each, 4 groups of 16 rows by 2 halves of
// the key columns.  So a lane has 64 sums and nothing spills: shared memory leaves
// the L1 cache too small for it, and spilled sums went to L2 (1039 us for 393216
// tokens of 128 x 128 with 16 warps of a quarter of all products each).  The value
// columns come in tiles of 32, two deep, so that the two states of a chunk (in two
// planes 139 KB of its 260 KB) never have to be in shared memory whole.
constexpr int kGradWarps = 16;
template <int KD>
struct Grad {
    static constexpr int VT = 32, LDK = KD + 8;
    static constexpr int kD = 0, kU = kD + kC * VT, kX = kU + 2 * VT * kTld, kS = kX + 2 * VT * kTld, kR = kS + 2 * VT * LDK;
    static constexpr int kGa = kR + 2 * VT * LDK;
    static constexpr int kStage = up1024(kGa * 2 + kGates * 4);    // bytes
    static constexpr int kK = 0, kQ = kC * KD, kKQ = 2 * kC * KD * 2;  // (elements, elements, bytes)
    static constexpr int kN = 2 * kStage + 2 * kKQ;                // N and E, two planes each (bytes)
    static constexpr int kF = kN + 4 * kCC * 2;                    // floats: row sums, dbeta, totals
    static constexpr int kBars = kF + (4 * kC + 2 * kC + 2 * kGradWarps) * 4;
    static constexpr size_t bytes = 1024 + kBars + 8 * 9 + 8 * 4;
};

__device__ __forceinline__ void sync_compute() { __syncthreads(); }

template <typename T>
__device__ __forceinline__ void split_store(e16* s, float x, float y) {  // and its low plane kCC further
    const uint32_t hi = Num<T>::pack(x, y);
    const float2 f = Num<T>::unpack(hi);
    *reinterpret_cast<uint32_t*>(s) = hi;
    *reinterpret_cast<uint32_t*>(s + kCC) = Num<T>::pack(x - f.x, y - f.y);
}

// rows m0.. of accumulators to an output of row stride st: zeros from `rows` on, nothing from `all` on
template <typename T, int NT>
__device__ __forceinline__ void rows_out(const float (*x)[4], e16* p, int64_t st, int m0, int rows, int all, int c0,
                                         int cols, const Lane& L) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = m0 + L.g + 8 * half;
        if (r >= all) continue;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int col = c0 + 8 * j + 2 * L.t;
            if (col < cols)
                *reinterpret_cast<uint32_t*>(p + r * st + col) = r < rows ? Num<T>::pack(x[j][2 * half], x[j][2 * half + 1]) : 0u;
        }
    }
}

// The loads of the next tile, by warp 0.  Where they are is kept in shared memory
// (at: chunk, value head, first value column; tiles and chunks so far; waits for
// `land` so far), as a lane has no registers for it.
template <int KD>
__device__ __forceinline__ bool grad_produce(const DArgs& a, const Maps& maps, unsigned char* smem) {
    using Sm = Grad<KD>;
    constexpr int VT = Sm::VT;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sm::kBars);
    uint64_t *empty = full + 2, *qfull = full + 4, *qempty = full + 6, *land = full + 8;
    int* at = reinterpret_cast<int*>(land + 1);
    const int rep = a.Hv / a.Hk, items = a.B * a.Hk * a.n;
    const Lane L;
    bool ok = true;
    int it = at[0], h = at[1], v0 = at[2];
    if (it >= items) return true;
    const int bh = it / a.n, c = it - bh * a.n, b = bh / a.Hk, hk = bh - b * a.Hk, t0 = c * kC;
    const int ptile = at[3], pseen = at[4];
    int landed = at[5];
    const int rows = min(kC, row_length(a, b) - t0);
    const bool tail = rows < min(kC, a.L - t0);
    if (h < 0) {  // a new chunk: its keys and queries
        h = hk * rep;
        e16* e = reinterpret_cast<e16*>(smem + 2 * Sm::kStage + (pseen & 1) * Sm::kKQ);
        uint64_t* bar = tail ? land : &qfull[pseen & 1];
        ok = warp_wait(&qempty[pseen & 1], ((pseen >> 1) & 1) ^ 1) && ok;
        if (L.l == 0) {
            mbar_expect_tx(bar, Sm::kKQ);
#pragma unroll
            for (int x = 0; x < KD; x += 64) {
                tma_load(e + Sm::kK + x * kC, &maps.k, bar, x, t0, hk, b);
                tma_load(e + Sm::kQ + x * kC, &maps.q, bar, x, t0, hk, b);
            }
        }
        __syncwarp();
        if (tail) {
            ok = warp_wait(land, landed++ & 1) && ok;
            zero_rows<64>(e + Sm::kK, 2 * (KD / 64), rows);
            fence_async();
            warp_arrive(&qfull[pseen & 1]);
        }
    }
    const int vn = min(VT, a.Vp - v0);
    e16* e = reinterpret_cast<e16*>(smem + (ptile & 1) * Sm::kStage);
    uint64_t* bar = tail ? land : &full[ptile & 1];
    ok = warp_wait(&empty[ptile & 1], ((ptile >> 1) & 1) ^ 1) && ok;
    if (L.l == 0) {
        const int64_t id = (static_cast<int64_t>(b) * a.Hv + h) * a.n + c;
        mbar_expect_tx(bar, vn * (kC + 4 * kTld + 4 * Sm::LDK) * 2 + kGates * 4);
        for (int v = 0; v < vn; v += 16) tma_load(e + Sm::kD + v * kC, &maps.d, bar, v0 + v, t0, h, b);
        const e16* U = static_cast<const e16*>(a.U) + (id * 2 * a.Vp + v0) * kTld;
        const e16* X = static_cast<const e16*>(a.dV) + (id * 2 * a.Vp + v0) * kTld;
        const e16* S = static_cast<const e16*>(a.S) + (id * 2 * a.Vp + v0) * Sm::LDK;
        const e16* R = static_cast<const e16*>(a.dS) + (id * 2 * a.Vp + v0) * Sm::LDK;
        for (int p = 0; p < 2; ++p) {
            bulk_load(e + Sm::kS + p * VT * Sm::LDK, S + static_cast<int64_t>(p) * a.Vp * Sm::LDK, vn * Sm::LDK * 2, bar);
            bulk_load(e + Sm::kR + p * VT * Sm::LDK, R + static_cast<int64_t>(p) * a.Vp * Sm::LDK, vn * Sm::LDK * 2, bar);
            bulk_load(e + Sm::kU + p * VT * kTld, U + static_cast<int64_t>(p) * a.Vp * kTld, vn * kTld * 2, bar);
            bulk_load(e + Sm::kX + p * VT * kTld, X + static_cast<int64_t>(p) * a.Vp * kTld, vn * kTld * 2, bar);
        }
        bulk_load(e + Sm::kGa, a.gates + id * kGates, kGates * 4, bar);
    }
    __syncwarp();
    if (tail) {
        ok = warp_wait(land, landed++ & 1) && ok;
        zero_rows<16>(e + Sm::kD, vn / 16, rows);
        fence_async();
        warp_arrive(&full[ptile & 1]);
    }
    // the next tile: of this head, of the next, or of the next chunk with a token
    int seen_next = pseen;
    v0 += VT;
    if (v0 >= a.Vp) {
        v0 = 0;
        if (++h == (hk + 1) * rep) {
            h = -1;
            ++seen_next;
            for (it += gridDim.x; it < items; it += gridDim.x) {
                const int nbh = it / a.n;
                if (row_length(a, nbh / a.Hk) > (it - nbh * a.n) * kC) break;
            }
        }
    }
    if (L.l == 0) {
        at[0] = it;
        at[1] = h;
        at[2] = v0;
        at[3] = ptile + 1;
        at[4] = seen_next;
        at[5] = landed;
    }
    __syncwarp();
    return ok;
}

// Zeros for a chunk behind the sequence.
__device__ __forceinline__ void grad_zero(const DArgs& a, int b, int hk, int c) {
    const int rep = a.Hv / a.Hk, all = min(kC, a.L - c * kC), tid = threadIdx.x, n = blockDim.x;
    const int64_t row0 = static_cast<int64_t>(b) * a.L + static_cast<int64_t>(c) * kC;
    const int64_t qst = static_cast<int64_t>(a.Hk) * a.K, vst = static_cast<int64_t>(a.Hv) * a.V;
    const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll 1
    for (int i = tid; i < all * (a.K / 8); i += n) {
        const int64_t o = (row0 + i / (a.K / 8)) * qst + static_cast<int64_t>(hk) * a.K + i % (a.K / 8) * 8;
        *reinterpret_cast<uint4*>(static_cast<e16*>(a.dq) + o) = z;
        *reinterpret_cast<uint4*>(static_cast<e16*>(a.dk) + o) = z;
    }
#pragma unroll 1
    for (int h = hk * rep; h < (hk + 1) * rep; ++h) {
#pragma unroll 1
        for (int i = tid; i < all * (a.V / 8); i += n)
            *reinterpret_cast<uint4*>(static_cast<e16*>(a.dv) + (row0 + i / (a.V / 8)) * vst + static_cast<int64_t>(h) * a.V +
                                      i % (a.V / 8) * 8) = z;
#pragma unroll 1
        for (int i = tid; i < all; i += n) {
            gate_store(a.dg, a.gate_dtype, (row0 + i) * a.Hv + h, 0.f);
            gate_store(a.dbeta, a.gate_dtype, (row0 + i) * a.Hv + h, 0.f);
        }
    }
}

template <typename T, int KD>
__global__ void __launch_bounds__(32 * kGradWarps, 1) planes_grad_k(const __grid_constant__ DArgs a, float* group, const __grid_constant__ Maps maps) {
    using Sm = Grad<KD>;
    constexpr int VT = Sm::VT, NT = KD / 16;  // accumulator tiles of a half of the key columns
    extern __shared__ __align__(128) unsigned char smem_raw[];
    unsigned char* smem = align_smem(smem_raw);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sm::kBars);
    uint64_t *empty = full + 2, *qfull = full + 4, *qempty = full + 6, *land = full + 8;
    const int tid = threadIdx.x, warp = tid >> 5, rep = a.Hv / a.Hk;
    const Lane L;
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kGradWarps);
            mbar_init(&qfull[s], 1);
            mbar_init(&qempty[s], kGradWarps);
        }
        mbar_init(land, 1);
        fence_mbar_init();
    }
    __syncthreads();
    const int items = a.B * a.Hk * a.n;
    bool ok = true;
    int tile = 0, seen = 0;  // tiles and chunks so far
    int* at = reinterpret_cast<int*>(land + 1);
    bool first = true;
    if (warp == 0) {
        int it = blockIdx.x;
        for (; it < items; it += gridDim.x) {
            const int nbh = it / a.n;
            if (row_length(a, nbh / a.Hk) > (it - nbh * a.n) * kC) break;
        }
        if (L.l == 0) {
            at[0] = it;
            at[1] = -1;
            at[2] = at[3] = at[4] = at[5] = 0;
        }
        __syncwarp();
    }
    const int rg = (warp >> 1) & 3, half = warp & 1, m0 = rg * 16, n0 = half * (KD / 2);
    const bool writer = warp >= 8;
    const int r0 = m0 + L.g, r1 = r0 + 8;
    e16* sN = reinterpret_cast<e16*>(smem + Sm::kN);
    e16* sE = sN + 2 * kCC;
    float* sW = reinterpret_cast<float*>(smem + Sm::kN);    // dK_write, once N and E are done with
    float* sDot = reinterpret_cast<float*>(smem + Sm::kF);  // [4][64]
    float* sDb = sDot + 4 * kC;                             // [2][64]
    float* sTot = sDb + 2 * kC;                             // [16], [16]
    for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
        const int bh = it / a.n, c = it - bh * a.n, b = bh / a.Hk, hk = bh - b * a.Hk;
        const int rows = min(kC, row_length(a, b) - c * kC), all = min(kC, a.L - c * kC);
        const int64_t row0 = static_cast<int64_t>(b) * a.L + static_cast<int64_t>(c) * kC;
        const int qst = a.Hk * a.K, vst = a.Hv * a.V;
        e16* dq = static_cast<e16*>(a.dq) + row0 * qst + hk * a.K;
        e16* dk = static_cast<e16*>(a.dk) + row0 * qst + hk * a.K;
        if (rows <= 0) {
            grad_zero(a, b, hk, c);
            continue;
        }
        const e16* kq = reinterpret_cast<const e16*>(smem + 2 * Sm::kStage + (seen & 1) * Sm::kKQ);
        const e16 *sK = kq + Sm::kK, *sQ = kq + Sm::kQ;
        for (int h = hk * rep; h < (hk + 1) * rep; ++h) {
            e16* dv = static_cast<e16*>(a.dv) + row0 * vst + static_cast<int64_t>(h) * a.V;
            // readers: dQ and dK_read; writers: dK_write, and dO U^T (half 0) or dV U^T (half 1)
            float x[NT][4] = {}, y[NT > 8 ? NT : 8][4] = {};
            float db0 = 0.f, db1 = 0.f, sd = 0.f, gc = 0.f;
            float f0[2], f1[2];  // of rows r0, r1: scale gam and gam, or d
            for (int v0 = 0; v0 < a.Vp; v0 += VT, ++tile) {
                const int vn = min(VT, a.Vp - v0);
                const e16* e = reinterpret_cast<const e16*>(smem + (tile & 1) * Sm::kStage);
                const Sh es = sh(e);
                const float* ga = reinterpret_cast<const float*>(e + Sm::kGa);
                if (warp == 0) {
#pragma unroll 1
                    for (int i = first ? 0 : 1; i < 2; ++i) ok = grad_produce<KD>(a, maps, smem) && ok;
                    first = false;
                }
                ok = warp_wait(&full[tile & 1], (tile >> 1) & 1) && ok;
#pragma unroll
                for (int kk = 0; kk < VT / 16; ++kk) {
                    if (16 * kk >= vn) break;
                    if (!writer) {
                        Af<1> fd;
                        Af<2> fx;
                        ld_a32(fd.r[0], es + Sm::kD + kk * kC * 16, m0);
                        ld_at(fx.r[0], es + Sm::kX, kTld, m0, 16 * kk);
                        ld_at(fx.r[1], es + Sm::kX + VT * kTld, kTld, m0, 16 * kk);
#pragma unroll
                        for (int p = 0; p < NT / 2; ++p) {
                            uint32_t sh[4], sl[4];
                            ld_b<true>(sl, es + Sm::kS + VT * Sm::LDK, Sm::LDK, n0 + 16 * p, 16 * kk);
                            ld_b<true>(sh, es + Sm::kS, Sm::LDK, n0 + 16 * p, 16 * kk);
                            mma_pair<T>(x[2 * p], x[2 * p + 1], fd.r[0], sl);
                            mma_pair<T>(y[2 * p], y[2 * p + 1], fx.r[0], sl);
                            mma_pair<T>(x[2 * p], x[2 * p + 1], fd.r[0], sh);
                            mma_pair<T>(y[2 * p], y[2 * p + 1], fx.r[1], sh);
                            mma_pair<T>(y[2 * p], y[2 * p + 1], fx.r[0], sh);
                        }
                        if ((kk & 1) == half) {  // dv
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int r = r0 + (i & 1) * 8, col = v0 + 16 * kk + (i >> 1) * 8 + 2 * L.t;
                                if (r < all && col < a.V)
                                    *reinterpret_cast<uint32_t*>(dv + static_cast<int64_t>(r) * vst + col) =
                                        r < rows ? fx.r[0][i] : 0u;
                            }
                        }
                    } else {
                        Af<2> left, fu;  // (dO has no low plane)
                        ld_at(fu.r[0], es + Sm::kU, kTld, m0, 16 * kk);
                        ld_at(fu.r[1], es + Sm::kU + VT * kTld, kTld, m0, 16 * kk);
                        if (half) {
                            ld_at(left.r[0], es + Sm::kX, kTld, m0, 16 * kk);
                            ld_at(left.r[1], es + Sm::kX + VT * kTld, kTld, m0, 16 * kk);
                        } else {
                            ld_a32(left.r[0], es + Sm::kD + kk * kC * 16, m0);
                        }
                        auto triangle = [&](int p) {
                            uint32_t uh[4], ul[4];
                            ld_b<true>(ul, es + Sm::kU + VT * kTld, kTld, 16 * p, 16 * kk);
                            ld_b<true>(uh, es + Sm::kU, kTld, 16 * p, 16 * kk);
                            mma_pair<T>(y[2 * p], y[2 * p + 1], left.r[0], ul);
                            if (half) mma_pair<T>(y[2 * p], y[2 * p + 1], left.r[1], uh);
                            mma_pair<T>(y[2 * p], y[2 * p + 1], left.r[0], uh);
                        };
#pragma unroll
                        for (int p = 0; p < NT / 2; ++p) {
                            uint32_t rh[4], rl[4];
                            ld_b<true>(rl, es + Sm::kR + VT * Sm::LDK, Sm::LDK, n0 + 16 * p, 16 * kk);
                            ld_b<true>(rh, es + Sm::kR, Sm::LDK, n0 + 16 * p, 16 * kk);
                            mma_pair<T>(x[2 * p], x[2 * p + 1], fu.r[0], rl);
                            if (p <= rg) triangle(p);
                            mma_pair<T>(x[2 * p], x[2 * p + 1], fu.r[1], rh);
                            mma_pair<T>(x[2 * p], x[2 * p + 1], fu.r[0], rh);
                        }
#pragma unroll
                        for (int p = NT / 2; p < kC / 16; ++p)
                            if (p <= rg) triangle(p);
                        if (half) {  // dbeta = (dV / beta).(U / beta)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 p = Num<T>::unpack(left.r[0][i]), q = Num<T>::unpack(left.r[1][i]);
                                const float2 u = Num<T>::unpack(fu.r[0][i]), w = Num<T>::unpack(fu.r[1][i]);
                                const float f = ga[5 * kC + (i & 1 ? r1 : r0)];
                                float& db = i & 1 ? db1 : db0;
                                db = fmaf((p.x + q.x) * f, (u.x + w.x) * f, db);
                                db = fmaf((p.y + q.y) * f, (u.y + w.y) * f, db);
                            }
                        }
                    }
                }
#pragma unroll 1
                for (int i = tid; i < vn * (KD / 8); i += 32 * kGradWarps) {  // <S0, dS1>
                    const int o = i / (KD / 8) * Sm::LDK + i % (KD / 8) * 8;
                    const uint4 sh = *reinterpret_cast<const uint4*>(e + Sm::kS + o);
                    const uint4 sl = *reinterpret_cast<const uint4*>(e + Sm::kS + VT * Sm::LDK + o);
                    const uint4 rh = *reinterpret_cast<const uint4*>(e + Sm::kR + o);
                    const uint4 rl = *reinterpret_cast<const uint4*>(e + Sm::kR + VT * Sm::LDK + o);
                    const uint32_t *s_h = &sh.x, *s_l = &sl.x, *r_h = &rh.x, *r_l = &rl.x;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float2 p = Num<T>::unpack(s_h[w]), q = Num<T>::unpack(s_l[w]), u = Num<T>::unpack(r_h[w]), z = Num<T>::unpack(r_l[w]);
                        sd = fmaf(p.x + q.x, u.x + z.x, sd);
                        sd = fmaf(p.y + q.y, u.y + z.y, sd);
                    }
                }
                if (v0 + VT >= a.Vp) {  // the gates, and N and E, before the tile is given back
                    gc = ga[2 * kC + kC - 1];
                    f0[0] = ga[(writer ? 3 : 4) * kC + r0];
                    f0[1] = ga[(writer ? 3 : 4) * kC + r1];
                    f1[0] = ga[2 * kC + r0];
                    f1[1] = ga[2 * kC + r1];
                    if (writer) {
                        e16* o = half ? sE : sN;
                        const float f = half ? -1.f : a.scale;
#pragma unroll
                        for (int j = 0; j < kC / 8; ++j) {
                            if (j > 2 * rg + 1) break;
                            const int col = 8 * j + 2 * L.t;
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const int r = i ? r1 : r0;
                                const int last = half ? r - 1 : r;  // N with the diagonal, E without
                                split_store<T>(o + r * kTld + col, col <= last ? f * ratio(ga, r, col) * y[j][2 * i] : 0.f,
                                            col + 1 <= last ? f * ratio(ga, r, col + 1) * y[j][2 * i + 1] : 0.f);
                            }
                        }
                    }
                }
                warp_arrive(&empty[tile & 1]);
            }
            ok = warp_wait(&qfull[seen & 1], (seen >> 1) & 1) && ok;
            sd = warp_sum(sd);
            float tw = 0.f;  // writers: k.(d U dS1^T)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int col = n0 + 8 * j + 2 * L.t;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[j][2 * i] *= f0[i];
                    x[j][2 * i + 1] *= f0[i];
                    if (writer) {
                        const float2 kv = Num<T>::unpack(*reinterpret_cast<const uint32_t*>(sK + at128(i ? r1 : r0, col)));
                        tw = fmaf(kv.x, x[j][2 * i], tw);
                        tw = fmaf(kv.y, x[j][2 * i + 1], tw);
                    } else {
                        y[j][2 * i] *= -f1[i];
                        y[j][2 * i + 1] *= -f1[i];
                    }
                }
            }
            tw = warp_sum(tw);
            if (writer && half) {
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    db0 += __shfl_xor_sync(0xffffffffu, db0, o);
                    db1 += __shfl_xor_sync(0xffffffffu, db1, o);
                }
                if (L.t == 0) {
                    sDb[r0] = db0;
                    sDb[r1] = db1;
                }
            }
            if (L.l == 0) {
                sTot[warp] = sd;
                sTot[kGradWarps + warp] = tw;
            }
            sync_compute();  // N, E
            if (!writer) {
#pragma unroll 1
                for (int kk = 0; kk <= rg; ++kk) {  // rows of N and E
                    Af<2> fn, fe;
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        ld_a(fn.r[p], sh(sN) + p * kCC, kTld, m0, 16 * kk);
                        ld_a(fe.r[p], sh(sE) + p * kCC, kTld, m0, 16 * kk);
                    }
#pragma unroll
                    for (int p = 0; p < NT / 2; ++p) {
                        uint32_t bk[4];
                        ld_b128<true>(bk, sh(sK), n0 + 16 * p, 16 * kk);
                        mma_pair<T>(x[2 * p], x[2 * p + 1], fn.r[1], bk);
                        mma_pair<T>(y[2 * p], y[2 * p + 1], fe.r[1], bk);
                        mma_pair<T>(x[2 * p], x[2 * p + 1], fn.r[0], bk);
                        mma_pair<T>(y[2 * p], y[2 * p + 1], fe.r[0], bk);
                    }
                }
            } else {
#pragma unroll 1
                for (int kk = rg; kk < kC / 16; ++kk) {  // columns of N and E
                    Af<2> fn, fe;
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        ld_at(fn.r[p], sh(sN) + p * kCC, kTld, m0, 16 * kk);
                        ld_at(fe.r[p], sh(sE) + p * kCC, kTld, m0, 16 * kk);
                    }
#pragma unroll
                    for (int p = 0; p < NT / 2; ++p) {
                        mm128<T, 2, true>(x[2 * p], x[2 * p + 1], fn, sh(sQ), n0 + 16 * p, 16 * kk);
                        mm128<T, 2, true>(x[2 * p], x[2 * p + 1], fe, sh(sK), n0 + 16 * p, 16 * kk);
                    }
                }
            }
            float dot[2] = {};  // q.dQ + k.dK_read, or -k.dK_write
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int col = n0 + 8 * j + 2 * L.t;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int o = at128(i ? r1 : r0, col);
                    const float2 kv = Num<T>::unpack(*reinterpret_cast<const uint32_t*>(sK + o));
                    if (writer) {
                        dot[i] = fmaf(-kv.x, x[j][2 * i], dot[i]);
                        dot[i] = fmaf(-kv.y, x[j][2 * i + 1], dot[i]);
                    } else {
                        const float2 qv = Num<T>::unpack(*reinterpret_cast<const uint32_t*>(sQ + o));
                        dot[i] = fmaf(qv.x, x[j][2 * i], dot[i]);
                        dot[i] = fmaf(qv.y, x[j][2 * i + 1], dot[i]);
                        dot[i] = fmaf(kv.x, y[j][2 * i], dot[i]);
                        dot[i] = fmaf(kv.y, y[j][2 * i + 1], dot[i]);
                    }
                }
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                dot[0] += __shfl_xor_sync(0xffffffffu, dot[0], o);
                dot[1] += __shfl_xor_sync(0xffffffffu, dot[1], o);
            }
            if (L.t == 0) {
                sDot[(2 * writer + half) * kC + r0] = dot[0];
                sDot[(2 * writer + half) * kC + r1] = dot[1];
            }
            sync_compute();  // N and E are done with
            float4* mine = reinterpret_cast<float4*>(sW) + ((rg * 2 + half) * NT) * 32 + L.l;
            if (writer) {
#pragma unroll
                for (int j = 0; j < NT; ++j) mine[j * 32] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
            }
            sync_compute();
            if (!writer) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float4 w = mine[j * 32];
                    y[j][0] += w.x;
                    y[j][1] += w.y;
                    y[j][2] += w.z;
                    y[j][3] += w.w;
                }
                if (rep > 1) {  // the sum over the value heads of this key head; each thread its own elements
                    float* gq = group + static_cast<int64_t>(it) * 2 * kC * KD;
                    float* gk = gq + kC * KD;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int o = (i ? r1 : r0) * KD + n0 + 8 * j + 2 * L.t;
                            if (h > hk * rep) {
                                const float2 p = *reinterpret_cast<const float2*>(gq + o), q = *reinterpret_cast<const float2*>(gk + o);
                                x[j][2 * i] += p.x;
                                x[j][2 * i + 1] += p.y;
                                y[j][2 * i] += q.x;
                                y[j][2 * i + 1] += q.y;
                            }
                            if (h < (hk + 1) * rep - 1) {
                                *reinterpret_cast<float2*>(gq + o) = make_float2(x[j][2 * i], x[j][2 * i + 1]);
                                *reinterpret_cast<float2*>(gk + o) = make_float2(y[j][2 * i], y[j][2 * i + 1]);
                            }
                        }
                }
                if (h == (hk + 1) * rep - 1) {
                    rows_out<T, NT>(x, dq, qst, m0, rows, all, n0, a.K, L);
                    rows_out<T, NT>(y, dk, qst, m0, rows, all, n0, a.K, L);
                }
            } else if (warp == 8) {
                float tot = L.l < kGradWarps ? gc * sTot[L.l] + sTot[kGradWarps + L.l] : 0.f;
                tot = warp_sum(tot);  // <S1, dS1>
                const int i0 = 2 * L.l;
                const float y1 = (sDot[i0 + 1] + sDot[kC + i0 + 1]) + (sDot[2 * kC + i0 + 1] + sDot[3 * kC + i0 + 1]);
                const float y0 = (sDot[i0] + sDot[kC + i0]) + (sDot[2 * kC + i0] + sDot[3 * kC + i0]) + y1;
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
            // the sums and dK_write have been read; all warps leave together where a wait ran out
            ok = __syncthreads_and(ok);
        }
        warp_arrive(&qempty[seen & 1]);
        ++seen;
    }
}

// ----------------------------------------------------------------------------
// launches
// ----------------------------------------------------------------------------
constexpr int kSms = 148;

// Groups of 16 value columns per CTA of a chain, one CTA on an SM at a time: the
// fewest rounds of CTAs, weighed with what a chunk takes with 2, 3 or 4 groups on
// an SM.  Measured at V = 128, us:
//                                       K = 128            K = 64
//   forward                             2.33 3.35 3.30     1.74 2.71 2.37
//     float16                           2.91 3.59 3.75     2.12 3.01 2.62
//   forward that keeps for a backward   2.72 3.54 4.24     2.31 2.89 3.84
//     float16                           3.44 4.39 5.67     2.47 3.15 4.03
//   reverse                             2.79 3.46          2.34 2.92
//     float16                           3.48 4.50          2.66 3.15
// (four groups do not fit the reverse chain's tiles).
int chain_groups(const DArgs& a, bool reverse) {
    const int64_t heads = static_cast<int64_t>(a.B) * a.Hv, groups = a.Vp / 16;
    auto cost = [&](int64_t g, int64_t per) { return (heads * ((groups + g - 1) / g) + kSms - 1) / kSms * per; };
    const int64_t x2 = cost(2, 27), x3 = cost(3, 34), x4 = cost(4, a.S ? 43 : 36);
    if (reverse) return x2 <= x3 ? 2 : 3;
    if (!a.S) return x2 <= x4 ? 2 : 4;  // (three are no faster than four)
    return x2 <= x3 && x2 <= x4 ? 2 : x3 <= x4 ? 3 : 4;
}

template <typename T, int KD, int G, bool KEEP>
cudaError_t chain_launch(const DArgs& a, const Maps& m, cudaStream_t s) {
    const auto k = planes_chain_k<T, KD, G, KEEP>;
    DELTA_TRY(smem_limit(k, Fwd<KD, G>::bytes));
    k<<<dim3((a.Vp / 16 + G - 1) / G, a.Hv, a.B), Fwd<KD, G>::kWarps * 32, Fwd<KD, G>::bytes, s>>>(a, m);
    note_launch();
    return cudaGetLastError();
}
template <typename T, int KD, int G>
cudaError_t rchain_launch(const DArgs& a, const Maps& m, cudaStream_t s) {
    DELTA_TRY((smem_limit(planes_rchain_k<T, KD, G>, Rev<KD, G>::bytes)));
    planes_rchain_k<T, KD, G><<<dim3((a.Vp / 16 + G - 1) / G, a.Hv, a.B), Rev<KD, G>::kWarps * 32, Rev<KD, G>::bytes, s>>>(a, m);
    note_launch();
    return cudaGetLastError();
}

template <typename T, int KD>
cudaError_t chain(const DArgs& a, const Maps& m, bool reverse, cudaStream_t s) {
    const int g = chain_groups(a, reverse);
    if (reverse) return g == 2 ? rchain_launch<T, KD, 2>(a, m, s) : rchain_launch<T, KD, 3>(a, m, s);
    if (a.S)
        return g == 2   ? chain_launch<T, KD, 2, true>(a, m, s)
               : g == 3 ? chain_launch<T, KD, 3, true>(a, m, s)
                        : chain_launch<T, KD, 4, true>(a, m, s);
    return g == 2 ? chain_launch<T, KD, 2, false>(a, m, s) : chain_launch<T, KD, 4, false>(a, m, s);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

// Boxes of 64 tokens by 64 columns (128-byte swizzle) or by 16 (32-byte).  A
// dimension of one element has no stride of its own: any multiple of 16 does.
bool make_map(CUtensorMap& m, const void* p, const Str& st, int64_t D, int64_t L, int64_t H, int64_t B, int cols, int half) {
    auto enc = encode_fn();
    if (!enc) return false;
    auto bytes = [](int64_t n, int64_t stride) { return static_cast<cuuint64_t>(n > 1 ? stride * 2 : 16); };
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(L), static_cast<cuuint64_t>(H),
                                static_cast<cuuint64_t>(B)};
    const cuuint64_t strides[3] = {bytes(L, st.t), bytes(H, st.h), bytes(B, st.b)};
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(cols), kC, 1, 1}, unit[4] = {1, 1, 1, 1};
    return enc(&m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, unit,
               CU_TENSOR_MAP_INTERLEAVE_NONE, cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_32B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool make_maps(const DArgs& a, Maps& m) {
    return make_map(m.q, a.q, a.sq, a.K, a.L, a.Hk, a.B, 64, a.half) && make_map(m.k, a.k, a.sk, a.K, a.L, a.Hk, a.B, 64, a.half) &&
           make_map(m.v, a.v, a.sv, a.V, a.L, a.Hv, a.B, 16, a.half) &&
           (!a.dout || make_map(m.d, a.dout, a.sdo, a.V, a.L, a.Hv, a.B, 16, a.half));
}

template <typename T, int KD>
cudaError_t fwd(const DArgs& a, cudaStream_t s) {
    // a runtime call first: tensor maps are not made in a thread (autograd's, say) that
    // has not met its device yet
    DELTA_TRY((smem_limit(planes_prep_k<T, KD>, Prep<KD>::bytes)));
    Maps m{};
    if (!make_maps(a, m)) return cudaErrorInvalidValue;
    planes_prep_k<T, KD><<<dim3(a.n, a.Hv, a.B), 128, Prep<KD>::bytes, s>>>(a, m);
    note_launch();
    DELTA_TRY(cudaGetLastError());
    return chain<T, KD>(a, m, false, s);
}

template <typename T, int KD>
cudaError_t bwd(const DArgs& a, float* group, cudaStream_t s) {
    // a runtime call first, as in fwd
    if constexpr (Scaled<T>) DELTA_TRY((smem_limit(planes_rchain_k<T, KD, 2>, Rev<KD, 2>::bytes)));
    else DELTA_TRY((smem_limit(planes_grad_k<T, KD>, Grad<KD>::bytes)));
    Maps m{};
    if (!make_maps(a, m)) return cudaErrorInvalidValue;
    DELTA_TRY((chain<T, KD>(a, m, true, s)));
    if constexpr (!Scaled<T>) {  // (float16's gradients are delta.cu's)
        const int items = a.B * a.Hk * a.n;
        planes_grad_k<T, KD><<<items < kSms ? items : kSms, 32 * kGradWarps, Grad<KD>::bytes, s>>>(a, group, m);
        note_launch();
    }
    return cudaGetLastError();
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }
int key_dim(const DArgs& a) { return a.K <= 64 ? 64 : 128; }
size_t ids(const DArgs& a) { return static_cast<size_t>(a.B) * a.Hv * a.n; }
size_t gates_bytes(const DArgs& a) { return up256(ids(a) * kGates * sizeof(float)); }
size_t square_bytes(const DArgs& a) { return up256(ids(a) * 2 * kCC * sizeof(e16)); }
// float16: float32, without padding
size_t state_bytes(const DArgs& a) {
    return up256(ids(a) * a.Vp * (a.half ? key_dim(a) * sizeof(float) : 2 * (key_dim(a) + 8) * sizeof(e16)));
}
size_t value_bytes(const DArgs& a) { return up256(ids(a) * a.Vp * (a.half ? kC * sizeof(float) : 2 * kTld * sizeof(e16))); }

void set_saved(DArgs& a, void* ws, bool training) {
    char* w = static_cast<char*>(ws);
    a.gates = reinterpret_cast<float*>(w); w += gates_bytes(a);
    a.T = w; w += square_bytes(a);
    a.M = w; w += square_bytes(a);
    a.S = training ? w : nullptr; w += state_bytes(a);
    a.U = training ? w : nullptr; w += value_bytes(a);
    a.Tr = training && a.half ? w : nullptr;
}

}  // namespace

size_t planes_saved_size(const DArgs& a, bool training) {
    return gates_bytes(a) + 2 * square_bytes(a) +
           (training ? state_bytes(a) + value_bytes(a) + (a.half ? square_bytes(a) : 0) : 0);
}
size_t planes_bwd_size(const DArgs& a) { return state_bytes(a) + value_bytes(a); }

cudaError_t planes_fwd(DArgs a, void* ws, bool training, cudaStream_t s) {
    set_saved(a, ws, training);
    if (a.half) return a.K <= 64 ? fwd<__half, 64>(a, s) : fwd<__half, 128>(a, s);
    return a.K <= 64 ? fwd<__nv_bfloat16, 64>(a, s) : fwd<__nv_bfloat16, 128>(a, s);
}

cudaError_t planes_bwd(DArgs& a, void* saved, void* ws, float* group, cudaStream_t s) {
    set_saved(a, saved, true);
    char* w = static_cast<char*>(ws);
    a.dS = w;
    a.dV = w + state_bytes(a);
    if (a.half) return a.K <= 64 ? bwd<__half, 64>(a, group, s) : bwd<__half, 128>(a, group, s);
    return a.K <= 64 ? bwd<__nv_bfloat16, 64>(a, group, s) : bwd<__nv_bfloat16, 128>(a, group, s);
}

cudaError_t planes_read_status(int* out, cudaStream_t s) { return read_clear_status(out, s); }

}  // namespace eacs
