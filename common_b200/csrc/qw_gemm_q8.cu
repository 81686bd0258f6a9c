// qw_gemm_q8.cu -- products of 8-bit codes on the tensor cores (qw_op_linear_q8): s(t, f) = sum_j w(f, j) x(t, j) in 32-bit
// integers (tcgen05.mma kind::i8, accumulators in tensor memory), then y = s w_scale(f) x_scale(t) and the epilogue
// (bias, residual, SwiGLU) on the way out.
//
// W is the M side of the MMAs (128 features per CTA), the tokens are their N side, as in qw_gemm.cu; a k-block is 128 codes,
// one 128-byte row of swizzled shared memory, staged by TMA (no multicast).  The sums are exact, so that every form below
// gives the same bits, however it cuts the work:
//   qw_q8_split_kernel  few tokens or tiles: one tile of 128 or 256 features x 16..256 tokens and one range of its k-blocks per
//                       CTA or pair; the CTAs of a tile form a cluster and add their sums through distributed shared memory;
//   qw_q8_pair_kernel   many tokens: persistent CTA pairs, tiles of 256 features x 256 tokens (cta_group::2).
//
// Both are launched with programmatic dependent launch: barriers, tensor memory and descriptors are set up behind the end of
// the previous kernel; nothing is read or written before it has ended (codes and scales may be its results), and the next
// kernel may start its own set-up only then.  Every mbarrier wait is bounded; on expiry the CTA records TC_DEVERR_TIMEOUT, lets
// its copies and MMAs land, frees its tensor memory and returns.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <mutex>
#include <string>

#include "../../include/qwen3_b200.h"
#include "qw_internal.cuh"
#include "qw_ops.h"
#include "qw_tc.h"
#include "qw_tc_util.cuh"

namespace qw {
namespace {

constexpr int kQ8MaxK = 131071;  // |s| <= 128 * 128 * k < 2^31 for any codes
constexpr int kQ8Threads = 320;  // a warp for the loads, one for the MMAs, eight for the results
// Of 256 tokens over ranges of the k-blocks sixteen: their results leave all at once, behind the last MMA, and what bounds that is
// the loads in flight (512 x 4096 x 12288, RESID: 25.6 us, 29.5 with eight).
__host__ __device__ constexpr int split_threads(int bn) { return bn > 128 ? 576 : kQ8Threads; }
constexpr int kBM = 128, kBK = 128;  // features of a CTA, codes of a k-block
constexpr int kABytes = kBM * kBK;

enum Q8Epi { Q8_F32 = 0, Q8_BF16 = 1, Q8_RESID = 2, Q8_SWIGLU = 3 };

struct Q8GemmArgs {
    const float *w_scale, *x_scale, *bias, *resid;
    void *out;
    int *err;
    long long ld_resid, ld_out;
    int M, K, T;
    int aligned, raligned;  // rows of results and of residuals begin on 16 bytes
    int group;  // pairs that stay: token tiles per group of their order
};

// Instruction descriptor of kind::i8: signed 8-bit A and B, both K-major, 32-bit integer D, M x N.
__host__ __device__ constexpr uint32_t q8_idesc(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int CTAS>
__device__ __forceinline__ void q8_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    if (CTAS == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
            : "memory");
}
// arrive on the mbarrier (of both CTAs of a pair) once the MMAs issued so far complete; rank: this CTA's in its cluster
template <int CTAS>
__device__ __forceinline__ void q8_commit(uint64_t *bar, int rank) {
    if (CTAS == 1)
        tc_commit(bar);
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
            "h"((uint16_t)(3 << (rank & ~1)))
            : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t *base, uint32_t cols) {
    if (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    tc_fence_after();
    if (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
// wait, bounded, for a phase that comes unless a copy or an MMA was never issued
__device__ __forceinline__ void mbar_settle(uint64_t *bar, uint32_t parity) {
    const uint32_t addr = smem_u32(bar);
    const uint64_t c0 = gtime_ns();
    while (!mbar_try(addr, parity) && gtime_ns() - c0 < kTcuWaitCycles) {
    }
}
// N columns of this warp's 32 tensor-memory lanes
template <int N>
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[N]) {
    static_assert(N == 8 || N == 16 || N == 32, "columns");
    if constexpr (N == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(taddr));
    else if constexpr (N == 16)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
    else
        tmem_ld32(taddr, r);
    if constexpr (N < 32) asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ int4 ld_cluster4(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A sum's value.  Each product is rounded, and so is what is added behind it: contracted differently here and there, the forms
// would differ in the last bit.
__device__ __forceinline__ float scaled(int s, float ws, float xs) { return __fmul_rn(__fmul_rn((float)s, ws), xs); }

// up * gate / (1 + e^-gate): the exponential and the division are within (|gate| + 4) 2^-21 of their value, the result is rounded
// to bf16 behind it.  __fdividef gives 0 for divisors above 2^126: both sides are taken 2^-8 times, so that these begin at a gate
// of -92.8, where silu(gate) is below fp32's normal numbers (-87.3 without); what gates below 2^-118 lose by it is 2^-142 of up.  An exponential
// below the normal numbers does not count beside 1.
__device__ __forceinline__ float silu_times(float g, float u) {
    constexpr float LOG2E = 1.44269504f;
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmaf_rn(g, -LOG2E, -8.f)));
    return u * __fdividef(g * 0x1p-8f, 0x1p-8f + e);
}

// What a lane keeps for its feature f across the tokens of a tile.
struct Q8Lane {
    float ws, bias;
    bool on;
};
template <int EPI>
__device__ __forceinline__ Q8Lane q8_lane(const Q8GemmArgs &a, int f) {
    Q8Lane l;
    l.on = f < a.M;
    l.ws = l.on ? a.w_scale[f] : 0.f;
    l.bias = EPI <= Q8_BF16 && a.bias && l.on ? a.bias[f] : 0.f;
    return l;
}

// Results of N consecutive tokens t0 .. t0 + nj - 1 (nj <= N) of feature f (this lane) from their sums; xs: the tokens' scales in
// shared memory, 16-byte aligned.  The lanes of a warp hold 32 consecutive features, so that a token's results are one
// contiguous piece of 128 (fp32), 64 or 32 bytes (bf16): whole sectors where the rows are aligned to them.  FULL: nj = N and
// f < M on every lane; the epilogue's instructions, on one or two warps per scheduler, are what the MMAs of short K wait for.
template <int EPI, int N, bool FULL>
__device__ __forceinline__ void q8_emit_some(const Q8GemmArgs &a, const Q8Lane &l, const uint32_t (&s)[N], const float *xs, int f,
                                             int lane, long long t0, int nj) {
    float y[N];
    if (EPI == Q8_RESID) {  // all loads before the stores: out may be resid
        const float *r = a.resid + t0 * a.ld_resid + f;
#pragma unroll
        for (int j = 0; j < N; j++, r += a.ld_resid) y[j] = FULL || (l.on && j < nj) ? *r : 0.f;
    }
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        const float4 x = *reinterpret_cast<const float4 *>(xs + j);
        const float v[4] = {scaled((int)s[j], l.ws, x.x), scaled((int)s[j + 1], l.ws, x.y), scaled((int)s[j + 2], l.ws, x.z),
                            scaled((int)s[j + 3], l.ws, x.w)};
#pragma unroll
        for (int i = 0; i < 4; i++)
            y[j + i] = EPI == Q8_RESID ? __fadd_rn(y[j + i], v[i]) : EPI <= Q8_BF16 && a.bias ? __fadd_rn(v[i], l.bias) : v[i];
    }
    if (EPI == Q8_SWIGLU) {
        // lanes 0..15 hold gates, 16..31 the ups of the same 16 products: of two tokens the lower lane computes the first and
        // the upper lane the second
        const bool hi = lane & 16;
        __nv_bfloat16 *o = reinterpret_cast<__nv_bfloat16 *>(a.out) + (t0 + hi) * a.ld_out + (f >> 5) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, hi ? y[j] : y[j + 1], 16);
            y[j] = hi ? other : y[j];
            y[j + 1] = hi ? y[j + 1] : other;
        }
#pragma unroll
        for (int j = 0; j < N; j += 2, o += 2 * a.ld_out) {
            const float h = silu_times(y[j], y[j + 1]);
            if (FULL || (l.on && j + hi < nj)) *o = __float2bfloat16_rn(h);
        }
    } else if (EPI == Q8_BF16) {
        __nv_bfloat16 *o = reinterpret_cast<__nv_bfloat16 *>(a.out) + t0 * a.ld_out + f;
#pragma unroll
        for (int j = 0; j < N; j++, o += a.ld_out)
            if (FULL || (l.on && j < nj)) *o = __float2bfloat16_rn(y[j]);
    } else {
        float *o = reinterpret_cast<float *>(a.out) + t0 * a.ld_out + f;
#pragma unroll
        for (int j = 0; j < N; j++, o += a.ld_out)
            if (FULL || (l.on && j < nj)) *o = y[j];
    }
}
template <int EPI, int N>
__device__ __forceinline__ void q8_emit(const Q8GemmArgs &a, const Q8Lane &l, const uint32_t (&s)[N], const float *xs, int f, int lane,
                                        int t0, int nj) {
    if (nj == N && __all_sync(0xffffffffu, l.on)) q8_emit_some<EPI, N, true>(a, l, s, xs, f, lane, t0, nj);
    else q8_emit_some<EPI, N, false>(a, l, s, xs, f, lane, t0, nj);
}

// ---- bf16 results of 32 features x 32 tokens in whole 16-byte pieces ----
// 16 tensor-memory lanes x 32 columns (tcgen05.ld 16x256b): register 4 i + 2 h + e of lane l is feature l / 4 + 8 h of token
// 8 i + 2 (l % 4) + e.  So a lane has a gate and its up in the same place of two loads, two neighbouring tokens of a feature
// make one register of bf16, and stmatrix turns 8 x 8 of them into rows of 8 features of a token.
__device__ __forceinline__ void tmem_get_16x256(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void stmatrix4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float2 scaled2(uint32_t s0, uint32_t s1, float ws, float2 xs) {
    return make_float2(scaled((int)s0, ws, xs.x), scaled((int)s1, ws, xs.y));
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    const __nv_bfloat162 w = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&w);
}
// bytes of a token's results of a warp, and their distance in its part of shared memory: rows of 16 bytes 8 apart meet no bank
// twice
__host__ __device__ constexpr int row_bytes(int epi) { return epi == Q8_SWIGLU ? 32 : 64; }
__host__ __device__ constexpr int row_apart(int epi) { return row_bytes(epi) + 16; }
__host__ __device__ constexpr int turn_bytes(int epi) { return epi == Q8_SWIGLU || epi == Q8_BF16 ? 32 * row_apart(epi) : 0; }

// 32 features from tensor-memory lane taddr on, all there, times tokens t0 .. t0 + nj - 1 (nj <= 32); ws and bias: those of
// features lane / 4 + 0, 8, 16, 24 of them; col: the first result's column.  Rows are 16-byte aligned.
template <int EPI>
__device__ __forceinline__ void q8_emit_rows(const Q8GemmArgs &a, uint32_t taddr, const float (&ws)[4], const float (&bias)[4],
                                             const float *xs, uint8_t *turn, int lane, long long t0, int nj, int col) {
    constexpr int APART = row_apart(EPI), PIECES = row_bytes(EPI) / 16;
    uint32_t g[16], u[16];
    tmem_get_16x256(taddr, g);
    tmem_get_16x256(taddr + (16u << 16), u);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    const uint32_t base = smem_u32(turn) + (uint32_t)(lane & 7) * APART;
    uint32_t w[4][4];  // of 8 tokens: 8 features each
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 x = *reinterpret_cast<const float2 *>(xs + 8 * i + 2 * (lane & 3));
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float2 y = scaled2(g[4 * i + 2 * h], g[4 * i + 2 * h + 1], ws[h], x);
            const float2 z = scaled2(u[4 * i + 2 * h], u[4 * i + 2 * h + 1], ws[2 + h], x);
            if (EPI == Q8_SWIGLU) {
                w[i][h] = bf16x2(silu_times(y.x, z.x), silu_times(y.y, z.y));
            } else {
                w[i][h] = a.bias ? bf16x2(__fadd_rn(y.x, bias[h]), __fadd_rn(y.y, bias[h])) : bf16x2(y.x, y.y);
                w[i][2 + h] = a.bias ? bf16x2(__fadd_rn(z.x, bias[2 + h]), __fadd_rn(z.y, bias[2 + h])) : bf16x2(z.x, z.y);
            }
        }
    }
    __syncwarp();  // the tokens before have left
    if (EPI == Q8_SWIGLU) {
        const uint32_t at = base + (uint32_t)((lane >> 3) & 1) * 16u + (uint32_t)(lane >> 4) * 8u * APART;
#pragma unroll
        for (int i = 0; i < 4; i += 2) stmatrix4_trans(at + (uint32_t)i * 8u * APART, w[i][0], w[i][1], w[i + 1][0], w[i + 1][1]);
    } else {
        const uint32_t at = base + (uint32_t)(lane >> 3) * 16u;
#pragma unroll
        for (int i = 0; i < 4; i++) stmatrix4_trans(at + (uint32_t)i * 8u * APART, w[i][0], w[i][1], w[i][2], w[i][3]);
    }
    __syncwarp();
    uint16_t *o = reinterpret_cast<uint16_t *>(a.out) + t0 * a.ld_out + col + (lane % PIECES) * 8;
#pragma unroll
    for (int k = 0; k < PIECES; k++) {
        const int t = (lane + 32 * k) / PIECES;
        if (t < nj) *reinterpret_cast<uint4 *>(o + t * a.ld_out) = *reinterpret_cast<const uint4 *>(turn + t * APART + (lane % PIECES) * 16);
    }
}

// Results of four consecutive features f .. f + 3 (this lane; 32 lanes, 128 features) of token t from their sums; add: their
// biases or residuals.
template <int EPI>
__device__ __forceinline__ void q8_emit4(const Q8GemmArgs &a, const float (&ws)[4], const float (&add)[4], int4 s, float xs, int f,
                                         int lane, long long t) {
    float y[4] = {scaled(s.x, ws[0], xs), scaled(s.y, ws[1], xs), scaled(s.z, ws[2], xs), scaled(s.w, ws[3], xs)};
    if constexpr (EPI == Q8_SWIGLU) {
        // of 8 lanes the first four hold 16 gates, the others their ups: each computes two of a lane's four products
        const bool hi = lane & 4;
        const float p = __shfl_xor_sync(0xffffffffu, hi ? y[0] : y[2], 4), q = __shfl_xor_sync(0xffffffffu, hi ? y[1] : y[3], 4);
        const float h0 = hi ? silu_times(p, y[2]) : silu_times(y[0], p), h1 = hi ? silu_times(q, y[3]) : silu_times(y[1], q);
        if (f >= a.M) return;
        __nv_bfloat16 *o = reinterpret_cast<__nv_bfloat16 *>(a.out) + t * a.ld_out + (f >> 5) * 16 + (lane & 3) * 4 + (hi ? 2 : 0);
        if (a.aligned) {
            *reinterpret_cast<uint32_t *>(o) = bf16x2(h0, h1);
        } else {
            o[0] = __float2bfloat16_rn(h0);
            o[1] = __float2bfloat16_rn(h1);
        }
    } else {
        if (EPI == Q8_RESID || a.bias) {
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = __fadd_rn(add[i], y[i]);
        }
        const long long at = t * a.ld_out + f;
        if (a.aligned && f + 4 <= a.M) {
            if (EPI == Q8_BF16) *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.out) + at) = make_uint2(bf16x2(y[0], y[1]), bf16x2(y[2], y[3]));
            else *reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (f + i >= a.M) break;
            if (EPI == Q8_BF16) reinterpret_cast<__nv_bfloat16 *>(a.out)[at + i] = __float2bfloat16_rn(y[i]);
            else reinterpret_cast<float *>(a.out)[at + i] = y[i];
        }
    }
}

// ---------------------------------------------------------------------------------------------
// few tokens: a tile's k-blocks cut over the CTAs of a cluster
// ---------------------------------------------------------------------------------------------
// CTAS = 1: a CTA computes 128 features x BN tokens over its range of k-blocks.  CTAS = 2: a pair of CTAs (cta_group::2) does 256
// features, its even CTA issuing the MMAs; each stages its own 128 rows of W and half of the tokens.  The nsplit ranges of a
// tile are the CTAs or pairs of a cluster (up to 8 CTAs).  Their sums meet in distributed shared memory: each CTA leaves its
// own in its ring, which is free by then, and after a cluster barrier adds up its share of the tile's tokens from all of them.
//
// Bound by the weights' bytes and what stands around them.  64 tokens, 4096 x 12288, RESID: 13.9 us in a graph, of which the
// weights' 50 MB take 8.3 (6 TB/s); 1.7 to the first k-block behind the previous kernel's end, 0.3 for the sums, 1.0 for the slowest
// CTA of a cluster, 1.3 to join and store, 1.2 to the end.  One token, 6144 x 4096: 7.5..8.1 us, 4.3 of them the weights'.  Measured and
// rejected: asking for the weights in L2 before the previous kernel has ended (17 us against 14; the requests stand in the way of
// its own loads), eight ranges of 64 tokens (15.8), two tokens' tiles of 32 (14.4).
constexpr int kClusterMax = 8;
__host__ __device__ constexpr int split_stage_bytes(int ctas, int bn) { return (kBM + bn / ctas) * kBK; }
constexpr int kSplitStages = 12;  // at most

template <int CTAS, int BN, int EPI>
__global__ void __launch_bounds__(split_threads(BN), BN > 128 ? 1 : 2)
    qw_q8_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Q8GemmArgs a,
                       int nsplit, int S) {
    constexpr int THREADS = split_threads(BN), ROWS = BN / CTAS, B_BYTES = ROWS * kBK;
    constexpr uint32_t TMEM_COLS = BN < 32 ? 32 : BN, IDESC = q8_idesc(kBM * CTAS, BN);
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kSplitStages], empty_bar[kSplitStages], tfull_bar;
    __shared__ __align__(16) float s_xs[BN];
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_sh;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sA = smem, *sB = smem + S * kABytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int size = nsplit * CTAS, rank = (int)blockIdx.x % size, range = rank / CTAS, side = rank % CTAS;
    const bool leader = side == 0;
    volatile int *abort_flag = &abort_sh;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&tfull_bar, 1);
        abort_sh = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmW) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmX) : "memory");
    }
    if (warp == 1) tmem_alloc<CTAS>(&tmem_base_sh, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync_all();  // both CTAs' barriers exist before any cross-CTA arrival
    tc_fence_after();
    const uint32_t tmem = tmem_base_sh;

    const int nt = (a.T + BN - 1) / BN, nkb = (a.K + kBK - 1) / kBK;
    const int tile = (int)blockIdx.x / size;
    const int t0 = (tile % nt) * BN, f0 = (tile / nt) * (kBM * CTAS) + side * kBM;
    const int kb0 = (int)((long long)nkb * range / nsplit), kb1 = (int)((long long)nkb * (range + 1) / nsplit);
    griddep_wait();
    griddep_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t full0 = CTAS == 2 ? cluster_map(smem_u32(&full_bar[0]), (uint32_t)(rank - side)) : 0u;
            int s = 0;
            uint32_t ph = 0, issued = 0, last_ph = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!mbar_wait(&empty_bar[s], ph ^ 1u, abort_flag, a.err)) { ok = false; break; }
                if (leader) mbar_arrive_expect_tx(&full_bar[s], CTAS * (kABytes + B_BYTES));
                if (CTAS == 2) {
                    tma_load_2d_pair(sA + s * kABytes, &tmW, full0 + 8u * s, kb * kBK, f0);
                    tma_load_2d_pair(sB + s * B_BYTES, &tmX, full0 + 8u * s, kb * kBK, t0 + side * ROWS);
                } else {
                    tma_load_2d(sA + s * kABytes, &tmW, &full_bar[s], kb * kBK, f0);
                    tma_load_2d(sB + s * B_BYTES, &tmX, &full_bar[s], kb * kBK, t0);
                }
                issued |= 1u << s;
                last_ph = (last_ph & ~(1u << s)) | (ph << s);
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            if (!ok && leader) {
                // let every issued copy land before the shared memory goes away
                for (int i = 0; i < S; i++)
                    if (issued >> i & 1u) mbar_settle(&full_bar[i], (last_ph >> i) & 1u);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            int s = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!mbar_wait(&full_bar[s], ph, abort_flag, a.err)) break;
                tc_fence_after();
                const uint64_t ad = sw128_desc(smem_u32(sA + s * kABytes)), bd = sw128_desc(smem_u32(sB + s * B_BYTES));
#pragma unroll
                for (int k = 0; k < kBK / 32; k++)
                    q8_mma<CTAS>(tmem, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), IDESC, (kb > kb0 || k > 0) ? 1u : 0u);
                q8_commit<CTAS>(&empty_bar[s], rank);
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            q8_commit<CTAS>(&tfull_bar, rank);
        }
        // all MMAs that use this CTA's memory complete before it is given up
        if (lane == 0) mbar_settle(&tfull_bar, 0);
    }
    const bool epilogue = warp >= 2;
    const int ncols = min(BN, a.T - t0), c0 = ncols * range / nsplit + warp - 2, c1 = ncols * (range + 1) / nsplit;
    const int f4 = f0 + lane * 4;  // where sums are joined: a warp takes a token, a lane four features
    constexpr int JW = THREADS / 32 - 2, JC = 2;  // warps that join; tokens of a warp at a time
    float ws4[4], add4[JC][4];
    const auto addends = [&](int c) {  // biases, or residuals of tokens c, c + JW, ...
#pragma unroll
        for (int u = 0; u < JC; u++) {
            const float *from = EPI == Q8_RESID ? a.resid + (long long)(t0 + c + u * JW) * a.ld_resid + f4 : a.bias + f4;
            const bool some = EPI == Q8_RESID ? c + u * JW < c1 : EPI <= Q8_BF16 && a.bias;
            if (EPI == Q8_RESID && a.raligned && some && f4 + 4 <= a.M) {
                const float4 v = *reinterpret_cast<const float4 *>(from);
                add4[u][0] = v.x; add4[u][1] = v.y; add4[u][2] = v.z; add4[u][3] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) add4[u][i] = some && f4 + i < a.M ? from[i] : 0.f;
            }
        }
    };
    if (epilogue) {
        // JW / 4 warps per 32 tensor-memory lanes (= features), each for its part of the tokens
        constexpr int PART = BN / (JW / 4), P = PART < 32 ? PART : 32;
        const int q = warp & 3, mine0 = ((warp - 2) >> 2) * PART, f = f0 + q * 32 + lane;
        for (int j = threadIdx.x - 64; j < BN; j += THREADS - 64) s_xs[j] = j < ncols ? a.x_scale[t0 + j] : 0.f;
        Q8Lane l{};
        if (nsplit == 1) {
            l = q8_lane<EPI>(a, f);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) ws4[i] = f4 + i < a.M ? a.w_scale[f4 + i] : 0.f;
            addends(c0);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(THREADS - 64) : "memory");
        mbar_wait(&tfull_bar, 0, abort_flag, a.err);
        tc_fence_after();
        int *part = reinterpret_cast<int *>(smem) + q * 32 + lane;
        for (int c = mine0; c < min(ncols, mine0 + PART); c += P) {
            uint32_t r[P];
            tmem_get<P>(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, r);
            if (nsplit == 1) {
                q8_emit<EPI, P>(a, l, r, s_xs + c, f, lane, t0 + c, min(P, ncols - c));
            } else {
#pragma unroll
                for (int j = 0; j < P; j++)
                    if (c + j < ncols) part[(c + j) * kBM] = (int)r[j];
            }
        }
    }
    if (nsplit > 1) {
        __syncwarp();
        cluster_sync_all();  // every CTA's sums are in its shared memory
        if (epilogue) {
            const uint32_t mine = smem_u32(smem) + (uint32_t)lane * 16u;
            for (int c = c0; c < c1; c += JC * JW) {
                int4 sum[JC] = {};
#pragma unroll
                for (int p0 = 0; p0 < kClusterMax / CTAS; p0 += 4) {
                    int4 v[JC][4];
#pragma unroll
                    for (int p = 0; p < 4; p++)
#pragma unroll
                        for (int u = 0; u < JC; u++)
                            v[u][p] = p0 + p < nsplit && c + u * JW < c1
                                          ? ld_cluster4(cluster_map(mine, (uint32_t)((p0 + p) * CTAS + side)) + (uint32_t)(c + u * JW) * (kBM * 4u))
                                          : make_int4(0, 0, 0, 0);
#pragma unroll
                    for (int p = 0; p < 4; p++)
#pragma unroll
                        for (int u = 0; u < JC; u++) {
                            sum[u].x += v[u][p].x; sum[u].y += v[u][p].y; sum[u].z += v[u][p].z; sum[u].w += v[u][p].w;
                        }
                    if (p0 + 4 >= nsplit) break;
                }
                if (EPI == Q8_RESID && c > c0) addends(c);
                if (c + JC * JW >= c1) cluster_arrive();  // the last sums of others are read
#pragma unroll
                for (int u = 0; u < JC; u++)
                    if (c + u * JW < c1) q8_emit4<EPI>(a, ws4, add4[u], sum[u], s_xs[c + u * JW], f4, lane, t0 + c + u * JW);
            }
            if (c0 >= c1) cluster_arrive();
        } else {
            cluster_arrive();
        }
        __syncwarp();
        cluster_wait();  // no CTA leaves while another reads its sums
    }
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2 && nsplit == 1) cluster_sync_all();  // nor while its peer signals its barriers
    if (warp == 1) tmem_free<CTAS>(tmem, TMEM_COLS);
}

// ---------------------------------------------------------------------------------------------
// many tokens: persistent CTA pairs
// ---------------------------------------------------------------------------------------------
// A cluster of two CTAs computes 256 features x BN tokens with one tcgen05.mma stream issued by the even CTA; each CTA stages its
// own 128 rows of W and half of the tokens, and its tensor memory holds its 128 features' sums, in two accumulators.
//   full[s]   in the even CTA: its producer's expect_tx of both CTAs' bytes; both CTAs' loads count on it;
//   empty[s]  in each CTA, signalled by the MMA commit to both;
//   tfull[i]  in each CTA, signalled by the commit behind the tile's last k-block;
//   tempty[i] in the even CTA: 16 arrivals (the epilogue warps of both CTAs).
//
// 8192 x 24576 x 4096 with SwiGLU: 600..622 us (2.65..2.75 POP/s, at the 1000 W limit), of which 30..50 are the epilogue's:
// without it 570.
// The tensor pipe is bound by the power: SM clocks settle at 1.4 GHz, and a library's plain product of the same codes takes 508..545 us
// with 1.3 GHz.  With four epilogue warps instead of eight the epilogue was longer than the MMAs of K = 4096 (779 us); with results
// stored as they lie in tensor memory, 2 bytes a lane, 655.  RESID (8192 x 4096 x 12288, 336 us) gains nothing from residuals
// fetched ahead (335) and loses where registers spill; rings of four stages take as long as of six.
constexpr int kPairBM = 256;
// Token tiles per group of the tile order: their X tiles, up to 16 MB of them, stay in L2 while W passes by.  8192 x 24576 x 4096
// takes 648 us in groups of 16, 665 of 8, 690 of 4; 8192 x 4096 x 12288 336 us in groups of 8, 349 of 5.
int pair_group(int k) {
    const int g = (16 << 20) / (256 * k);
    return g < 8 ? 8 : g > 16 ? 16 : g;
}

__host__ __device__ constexpr int pair_stage_bytes(int bn) { return kABytes + bn / 2 * kBK; }
__host__ __device__ constexpr int pair_stages(int bn) { return 196 * 1024 / pair_stage_bytes(bn); }
__host__ __device__ constexpr int pair_smem(int bn, int epi) { return pair_stages(bn) * pair_stage_bytes(bn) + 8 * turn_bytes(epi) + 1024; }

struct PairTile {
    int f0, t0;
};
template <int BN>
__device__ __forceinline__ PairTile pair_tile(int tile, int nf, int nt, int group) {
    const int per_group = nf * group;
    const int g = tile / per_group, r = tile % per_group;
    const int t_in = min(group, nt - g * group);
    return {(r / t_in) * kPairBM, (g * group + r % t_in) * BN};
}

template <int BN, int EPI>
__global__ void __launch_bounds__(kQ8Threads, 1)
    qw_q8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Q8GemmArgs a) {
    constexpr int S = pair_stages(BN), HALF = BN / 2, B_BYTES = HALF * kBK;
    constexpr uint32_t TMEM_COLS = 2 * BN, IDESC = q8_idesc(kPairBM, BN);
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S], tfull_bar[2], tempty_bar[2], done_bar;
    __shared__ __align__(16) float s_xs[8][HALF];
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_sh;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sA = smem, *sB = smem + S * kABytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    volatile int *abort_flag = &abort_sh;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&tfull_bar[i], 1);
            mbar_init(&tempty_bar[i], 16);
        }
        mbar_init(&done_bar, 1);
        abort_sh = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmW) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmX) : "memory");
    }
    if (warp == 1) tmem_alloc<2>(&tmem_base_sh, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before any cross-CTA arrival
    tc_fence_after();
    const uint32_t tmem = tmem_base_sh;
    griddep_wait();
    griddep_launch_dependents();

    const int nf = (a.M + kPairBM - 1) / kPairBM, nt = (a.T + BN - 1) / BN, nkb = (a.K + kBK - 1) / kBK;
    const int total = nf * nt, cid = blockIdx.x >> 1, ncl = gridDim.x >> 1;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer (both CTAs) ----------------
            const uint32_t full0 = cluster_map(smem_u32(&full_bar[0]), 0);
            int s = 0;
            uint32_t ph = 0, issued = 0, last_ph = 0;
            bool ok = true;
            for (int tile = cid; tile < total && ok; tile += ncl) {
                const PairTile c = pair_tile<BN>(tile, nf, nt, a.group);
                const int wrow = c.f0 + (int)rank * kBM, trow = c.t0 + (int)rank * HALF;
                for (int kb = 0; kb < nkb; kb++) {
                    if (!mbar_wait(&empty_bar[s], ph ^ 1u, abort_flag, a.err)) { ok = false; break; }
                    if (leader) mbar_arrive_expect_tx(&full_bar[s], 2 * (kABytes + B_BYTES));
                    tma_load_2d_pair(sA + s * kABytes, &tmW, full0 + 8u * s, kb * kBK, wrow);
                    tma_load_2d_pair(sB + s * B_BYTES, &tmX, full0 + 8u * s, kb * kBK, trow);
                    issued |= 1u << s;
                    last_ph = (last_ph & ~(1u << s)) | (ph << s);
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok && leader) {
                for (int i = 0; i < S; i++)
                    if (issued >> i & 1u) mbar_settle(&full_bar[i], (last_ph >> i) & 1u);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            // ---------------- MMA issuer (even CTA) ----------------
            int s = 0, it = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int tile = cid; tile < total && ok; tile += ncl, it++) {
                const int acc = it & 1;
                const uint32_t aph = (uint32_t)(it >> 1) & 1u;
                if (!mbar_wait(&tempty_bar[acc], aph ^ 1u, abort_flag, a.err)) break;
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(acc * BN);
                for (int kb = 0; kb < nkb; kb++) {
                    if (!mbar_wait(&full_bar[s], ph, abort_flag, a.err)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t ad = sw128_desc(smem_u32(sA + s * kABytes)), bd = sw128_desc(smem_u32(sB + s * B_BYTES));
#pragma unroll
                    for (int k = 0; k < kBK / 32; k++)
                        q8_mma<2>(d, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), IDESC, (kb > 0 || k > 0) ? 1u : 0u);
                    q8_commit<2>(&empty_bar[s], 0);
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
                if (ok) q8_commit<2>(&tfull_bar[acc], 0);
            }
            q8_commit<2>(&done_bar, 0);
        }
    } else {
        // ---------------- epilogue (warps 2..9 of both CTAs) ----------------
        // two warps per 32 tensor-memory lanes (= features), one for each half of the tokens
        const uint32_t tempty0 = cluster_map(smem_u32(&tempty_bar[0]), 0);
        const int q = warp & 3, half = (warp - 2) >> 2;
        float *xs = s_xs[warp - 2];
        uint8_t *turn = smem + S * (kABytes + B_BYTES) + (warp - 2) * turn_bytes(EPI);
        int it = 0;
        for (int tile = cid; tile < total; tile += ncl, it++) {
            const PairTile c = pair_tile<BN>(tile, nf, nt, a.group);
            const int acc = it & 1, f = c.f0 + (int)rank * kBM + q * 32 + lane, t0 = c.t0 + half * HALF;
            const int ncols = min(HALF, a.T - t0);
            const int fw = f - lane;  // the warp's first feature
            const bool rows = turn_bytes(EPI) && a.aligned && fw + 32 <= a.M;
            Q8Lane l{};
            float ws[4] = {}, bias[4] = {};
            if (rows) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    ws[i] = a.w_scale[fw + (lane >> 2) + 8 * i];
                    if (EPI == Q8_BF16 && a.bias) bias[i] = a.bias[fw + (lane >> 2) + 8 * i];
                }
            } else {
                l = q8_lane<EPI>(a, f);
            }
#pragma unroll
            for (int j = lane; j < HALF; j += 32) xs[j] = j < ncols ? a.x_scale[t0 + j] : 0.f;
            __syncwarp();
            if (!mbar_wait(&tfull_bar[acc], (uint32_t)(it >> 1) & 1u, abort_flag, a.err)) break;
            tc_fence_after();
            for (int cc = 0; cc < ncols; cc += 32) {
                const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * HALF + cc);
                if (turn_bytes(EPI) && rows) {
                    q8_emit_rows<EPI>(a, at, ws, bias, xs + cc, turn, lane, t0 + cc, min(32, ncols - cc), EPI == Q8_SWIGLU ? fw / 2 : fw);
                } else {
                    uint32_t r[32];
                    tmem_ld32(at, r);
                    q8_emit<EPI, 32>(a, l, r, xs + cc, f, lane, t0 + cc, min(32, ncols - cc));
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * (uint32_t)acc);
        }
    }

    tc_fence_before();
    __syncthreads();
    // every MMA of the pair has completed (they read both CTAs' shared memory and write both TMEMs)
    if (warp == 1 && lane == 0) mbar_settle(&done_bar, 0);
    __syncthreads();
    cluster_sync_all();  // no CTA leaves while its peer may still signal its barriers
    if (warp == 1) tmem_free<2>(tmem, TMEM_COLS);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
cudaError_t launch_cluster(const void *fn, int grid, int threads, int cluster, int smem, cudaStream_t st, void **args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

// A TMA map of (rows, cols) codes, ld apart: boxes of box_rows x 128 codes, 128-byte swizzle, zero fill behind both ends.
cudaError_t codes_map(CUtensorMap *m, const int8_t *base, long long rows, long long cols, long long ld, int box_rows) {
    typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                      const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                      CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const EncodeTiledFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    if (!fn) return cudaErrorNotSupported;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)box_rows}, es[2] = {1, 1};
    CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(base), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// How the work is cut.  ctas: of a tile (1: 128 features, 2: 256); bn: its tokens; nsplit: ranges of its k-blocks; 0: persistent pairs.
struct Q8Plan {
    int ctas, bn, nsplit;
};
// Clusters of 1..8 CTAs that a B200's 148 SMs hold at once, one CTA on an SM (256 tokens) and two (the smaller tiles): what
// cudaOccupancyMaxActiveClusters says of kernels of the same size that hold no tensor memory.  (With it the call counts one
// CTA on an SM; two were seen to run together.)
constexpr int kClusters[2][kClusterMax + 1] = {{0, 148, 74, 45, 33, 26, 22, 15, 15}, {0, 296, 148, 93, 71, 56, 45, 37, 33}};

// Whether a form's CTAs have an SM each: where there is room for all of them so, and of 64 tokens or more.  (Of fewer tokens the ring's bytes are
// mostly weights and half the room keeps HBM busy; the other half lets the next kernel's CTAs start: 1 x 6144 x 4096 7.7 us, 8.0
// with deep rings; 64 x 4096 x 12288 14.0, 14.9 with shallow ones.)
bool q8_alone(const Q8Plan &p, long long tiles) { return p.bn > 128 || (p.bn >= 64 && tiles <= kClusters[0][p.ctas * p.nsplit]); }
// Stages of a form's ring: as deep as its range and its share of the SM allow; the sums of a tile lie there too.
int split_stages(const Q8Plan &p, int kbs, bool alone) {
    const int bytes = split_stage_bytes(p.ctas, p.bn), room = (alone ? 200 : 110) * 1024 / bytes;
    const int sums = p.nsplit > 1 ? (p.bn * kBM * 4 + bytes - 1) / bytes : 1;
    int s = kbs < room ? kbs : room;
    s = s < kSplitStages ? s : kSplitStages;
    return s > sums ? s : sums;
}
template <int EPI>
const void *q8_kernel(const Q8Plan &p) {
    if (p.nsplit == 0) return (const void *)qw_q8_pair_kernel<256, EPI>;
    if (p.ctas == 2) return p.bn == 128 ? (const void *)qw_q8_split_kernel<2, 128, EPI> : (const void *)qw_q8_split_kernel<2, 256, EPI>;
    if (p.bn == 16) return (const void *)qw_q8_split_kernel<1, 16, EPI>;
    return p.bn == 32 ? (const void *)qw_q8_split_kernel<1, 32, EPI> : (const void *)qw_q8_split_kernel<1, 64, EPI>;
}
const void *q8_kernel(int epi, const Q8Plan &p) {
    switch (epi) {
        case Q8_F32: return q8_kernel<Q8_F32>(p);
        case Q8_BF16: return q8_kernel<Q8_BF16>(p);
        case Q8_RESID: return q8_kernel<Q8_RESID>(p);
        default: return q8_kernel<Q8_SWIGLU>(p);
    }
}

// The forms there are: pairs that stay, pairs and single CTAs over ranges of the k-blocks.
constexpr Q8Plan kForms[] = {{2, 256, 0}, {2, 256, 1}, {2, 128, 1}, {1, 64, 1}, {1, 32, 1}, {1, 16, 1}};

// Every kernel opted in to its shared memory, once per device, whose SMs are counted.
cudaError_t q8_device(int dev, int *sms) {
    static std::mutex mu;
    static int count[64] = {};
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    if (!count[dev]) {
        for (int epi = Q8_F32; epi <= Q8_SWIGLU; epi++)
            for (const Q8Plan &p : kForms) {
                const int most = p.nsplit == 0 ? pair_smem(256, epi) : 200 * 1024 + 1024;
                cudaError_t e = cudaFuncSetAttribute(q8_kernel(epi, p), cudaFuncAttributeMaxDynamicSharedMemorySize, most);
                if (e != cudaSuccess) return e;
            }
        cudaError_t e = cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
    }
    *sms = count[dev];
    return cudaSuccess;
}

// Microseconds that a form takes, from what it loads, multiplies and joins.  The constants are fitted to the times of 196 shapes
// (1152..24576 features, 896..12288 codes, 1..4096 tokens, every form and 1..8 ranges), all STORE to bf16 without a bias: the form that
// it picks takes 1.5 % more than the fastest one on average, 36 % at most (384 tokens, 4096 x 12288: 32.1 against 23.6 us; 23 % at
// 1 x 1152 x 896 and 256 x 9728 x 12288).  RESID, which moves 8 bytes a result, and SWIGLU, which stores 1, are not in it:
// 384 x 4096 x 12288 with RESID takes 42 us where 512 tokens take 26.
float q8_cost(const Q8Plan &p, int sms, int M, int T, int nkb) {
    const float tiles = (float)((M + p.ctas * kBM - 1) / (p.ctas * kBM)) * (float)((T + p.bn - 1) / p.bn);
    if (p.nsplit == 0) return 2.5f + ceilf(tiles / (float)(sms / 2)) * (0.411f * nkb + 1.2f);
    const float ctas = tiles * p.ctas * p.nsplit, per = ctas > sms && p.bn <= 128 ? 2.f : 1.f;  // per SM
    const float waves = ceilf(tiles / (float)kClusters[p.bn <= 128][p.ctas * p.nsplit]);
    const int kbs = (nkb + p.nsplit - 1) / p.nsplit;
    const float kb = (kBM + p.bn / p.ctas) * (float)kBK * 1e-3f;  // kilobytes of a k-block
    // a k-block: the ring's bytes in flight over their latency (GB/s of a CTA), the SM's loads, its MMAs
    const float ring = q8_alone(p, (long long)tiles) ? 83.5f : 63.f;
    const float step = fmaxf(fmaxf(kb / ring, per * kb / 93.8f), p.bn > 128 ? 0.34f : per * p.bn * (0.277f / 128.f));
    // and all of them: weights from HBM, operands through L2
    const float load = fmaxf(fmaxf(waves * (kbs * step + 0.34f), (float)M * nkb * (kBK / 6.5e6f)), ctas * kbs * kb * (1.f / 7920.f));
    return load + 1.87f / 64.f * p.bn + (p.nsplit > 1 ? 1.45f + 0.197f * p.nsplit + 0.495f / 64.f * p.bn : 0.f);
}
Q8Plan q8_plan(int M, int T, int K, int sms) {
    const int nkb = (K + kBK - 1) / kBK;
    const long long tiles = (long long)((M + kPairBM - 1) / kPairBM) * ((T + 255) / 256);
    // Pairs stay where there are more tiles than pairs; a tile each is done 5..19 % sooner by those that do not (more warps store).
    Q8Plan best = tiles > sms / 2 ? Q8Plan{2, 256, 0} : Q8Plan{2, 256, 1};
    float least = q8_cost(best, sms, M, T, nkb);
    for (const Q8Plan &form : kForms) {
        if (form.nsplit == 0 || (form.bn < 256 && (long long)form.bn * 8 < T) || (form.bn > 16 && form.bn / 2 >= T)) continue;
        for (int n : {1, 2, 3, 4, 6, 8}) {
            if (n > nkb || n * form.ctas > kClusterMax) break;
            const Q8Plan p{form.ctas, form.bn, n};
            const float c = q8_cost(p, sms, M, T, nkb);
            if (c < least) { least = c; best = p; }
        }
    }
    return best;
}

cudaError_t q8_gemm_launch(const int8_t *w, long long ld_w, const int8_t *x, long long ld_x, const Q8GemmArgs &a, int epi, int dev,
                           cudaStream_t st) {
    int sms;
    cudaError_t e = q8_device(dev, &sms);
    if (e != cudaSuccess) return e;
    const Q8Plan p = q8_plan(a.M, a.T, a.K, sms);
    const void *fn = q8_kernel(epi, p);
    CUtensorMap mw, mx;
    e = codes_map(&mw, w, a.M, a.K, ld_w, kBM);
    if (e == cudaSuccess) e = codes_map(&mx, x, a.T, a.K, ld_x, p.bn / p.ctas);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)((a.M + p.ctas * kBM - 1) / (p.ctas * kBM)) * ((a.T + p.bn - 1) / p.bn);
    if (p.nsplit == 0) {
        void *args[] = {(void *)&mw, (void *)&mx, (void *)&a};
        return launch_cluster(fn, 2 * (int)(tiles < sms / 2 ? tiles : sms / 2), kQ8Threads, 2, pair_smem(256, epi), st, args);
    }
    const int size = p.ctas * p.nsplit, nkb = (a.K + kBK - 1) / kBK;
    int nsplit = p.nsplit, stages = split_stages(p, (nkb + nsplit - 1) / nsplit, q8_alone(p, tiles));
    void *args[] = {(void *)&mw, (void *)&mx, (void *)&a, (void *)&nsplit, (void *)&stages};
    return launch_cluster(fn, (int)tiles * size, split_threads(p.bn), size, stages * split_stage_bytes(p.ctas, p.bn) + 1024, st, args);
}

}  // namespace
}  // namespace qw

using namespace qw;

extern "C" qw_status qw_op_linear_q8(const qw_linear_q8_args *p, void *stream) {
    if (!p) return op_fail(QW_ERR_ARG, "null arguments");
    if (p->epi < QW_LINEAR_STORE || p->epi > QW_LINEAR_SWIGLU) return op_fail(QW_ERR_ARG, "epilogue " + std::to_string(p->epi));
    if (p->out_dtype != QW_DTYPE_F32 && p->out_dtype != QW_DTYPE_BF16) return op_fail(QW_ERR_UNSUPPORTED, "out must be fp32 or bf16");
    if (p->epi == QW_LINEAR_RESID && p->out_dtype != QW_DTYPE_F32) return op_fail(QW_ERR_UNSUPPORTED, "RESID writes fp32");
    if (p->epi == QW_LINEAR_SWIGLU && p->out_dtype != QW_DTYPE_BF16) return op_fail(QW_ERR_UNSUPPORTED, "SWIGLU writes bf16");
    if (p->bias && p->epi != QW_LINEAR_STORE) return op_fail(QW_ERR_ARG, "bias is for STORE");
    if (p->n_out < 1 || p->t < 0 || p->k < 1 || p->k > kQ8MaxK)
        return op_fail(QW_ERR_SHAPE, "n_out >= 1, t >= 0 and k in [1, " + std::to_string(kQ8MaxK) + "]");
    // tiles are numbered in 32 bits, of the smallest form in eight ranges each
    if (((long long)p->n_out / kBM + 1) * ((long long)p->t / 16 + 1) > 0x7FFFFFFFll / kClusterMax || p->n_out > 1 << 30 || p->t > 1 << 30)
        return op_fail(QW_ERR_SHAPE, "n_out x t is too large for one call");
    if (p->epi == QW_LINEAR_SWIGLU && p->n_out % 32) return op_fail(QW_ERR_SHAPE, "SWIGLU needs n_out a multiple of 32");
    const int64_t cols = p->epi == QW_LINEAR_SWIGLU ? p->n_out / 2 : p->n_out;
    Q8GemmArgs a{};
    const int64_t ld_w = p->ld_w ? p->ld_w : p->k, ld_x = p->ld_x ? p->ld_x : p->k;
    a.ld_out = p->ld_out ? p->ld_out : cols; a.ld_resid = p->ld_resid ? p->ld_resid : cols;
    if (ld_w < p->k || ld_x < p->k || ld_w % 16 || ld_x % 16 || ld_w >= 1ll << 31 || ld_x >= 1ll << 31)
        return op_fail(QW_ERR_SHAPE, "ld_w and ld_x must cover k in multiples of 16, below 2^31");
    if (a.ld_out < cols || (p->epi == QW_LINEAR_RESID && a.ld_resid < cols))
        return op_fail(QW_ERR_SHAPE, "ld_out and ld_resid must cover the columns");
    if (p->t == 0) return QW_OK;
    if (!p->w || !p->w_scale || !p->x || !p->x_scale || !p->out) return op_fail(QW_ERR_ARG, "null device pointer");
    if (p->epi == QW_LINEAR_RESID && !p->resid) return op_fail(QW_ERR_ARG, "RESID needs resid");
    if (p->epi == QW_LINEAR_RESID && p->out == (const void *)p->resid && a.ld_out != a.ld_resid)
        return op_fail(QW_ERR_ARG, "out may be resid only with the same stride");
    if (((uintptr_t)p->w | (uintptr_t)p->x) & 15) return op_fail(QW_ERR_ARG, "w and x must be 16-byte aligned");
    if ((((uintptr_t)p->w_scale | (uintptr_t)p->x_scale | (uintptr_t)p->bias | (uintptr_t)p->resid | (uintptr_t)p->err) & 3) ||
        (uintptr_t)p->out % (p->out_dtype == QW_DTYPE_BF16 ? 2 : 4))
        return op_fail(QW_ERR_ARG, "pointers must be aligned to their elements");
    a.w_scale = p->w_scale; a.x_scale = p->x_scale; a.bias = p->bias; a.resid = p->resid;
    a.out = p->out; a.err = p->err; a.M = p->n_out; a.K = p->k; a.T = p->t; a.group = pair_group(p->k);
    a.aligned = !((uintptr_t)p->out & 15) && a.ld_out % (p->out_dtype == QW_DTYPE_BF16 ? 8 : 4) == 0;
    a.raligned = !((uintptr_t)p->resid & 15) && a.ld_resid % 4 == 0;
    const int epi = p->epi == QW_LINEAR_RESID ? Q8_RESID : p->epi == QW_LINEAR_SWIGLU ? Q8_SWIGLU
                  : p->out_dtype == QW_DTYPE_BF16 ? Q8_BF16 : Q8_F32;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return op_fail(QW_ERR_CUDA, "no current device");
    cudaError_t e = q8_gemm_launch(p->w, ld_w, p->x, ld_x, a, epi, dev, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("linear launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
