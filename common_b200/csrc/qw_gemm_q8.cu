// qw_gemm_q8.cu -- products of 8-bit codes on the tensor cores (qw_op_linear_q8): s(t, f) = sum_j w(f, j) x(t, j) in 32-bit
// integers (tcgen05.mma kind::i8, accumulators in tensor memory), then y = s w_scale(f) x_scale(t) and the epilogue
// (bias, residual, SwiGLU) on the way out.
//
// W is the M side of the MMAs (128 features per CTA), the tokens are their N side, as in qw_gemm.cu; a k-block is 128 codes,
// one 128-byte row of swizzled shared memory, staged by TMA (no multicast).  The sums are exact, so that every form below
// gives the same bits, however it cuts the work:
//   qw_q8_split_kernel  few tokens: one tile of 128 features x 16..128 tokens and one range of its k-blocks per CTA; the CTAs
//                       of a tile form a cluster and add their sums through distributed shared memory;
//   qw_q8_pair_kernel   many tokens: persistent CTA pairs, tiles of 256 features x 128 or 256 tokens (cta_group::2).
//
// Both are launched with programmatic dependent launch: barriers, tensor memory and descriptors are set up behind the end of
// the previous kernel; nothing is read or written before it has ended (codes and scales may be its results), and the next
// kernel may start its own set-up only then.  Every mbarrier wait is bounded; on expiry the CTA records TC_DEVERR_TIMEOUT, lets
// its copies and MMAs land, frees its tensor memory and returns.
#include <cuda.h>
#include <cuda_runtime.h>
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
constexpr int kQ8Threads = 192;
constexpr int kBM = 128, kBK = 128;  // features of a CTA, codes of a k-block
constexpr int kABytes = kBM * kBK;

enum Q8Epi { Q8_F32 = 0, Q8_BF16 = 1, Q8_RESID = 2, Q8_SWIGLU = 3 };

struct Q8GemmArgs {
    const float *w_scale, *x_scale, *bias, *resid;
    void *out;
    int *err;
    long long ld_resid, ld_out;
    int M, K, T;
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
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

// Results of N consecutive tokens t0 .. t0 + nj - 1 (nj <= N) of feature f (this lane) from their sums.  The lanes of a warp hold
// 32 consecutive features, so that a token's results are one contiguous piece of 128 (fp32), 64 or 32 bytes (bf16): whole
// sectors where the rows are aligned to them.
template <int EPI, int N>
__device__ __forceinline__ void q8_emit(const Q8GemmArgs &a, const Q8Lane &l, const int (&s)[N], int f, int lane, int t0, int nj) {
    static_assert(N <= 32 && (N == 1 || N % 2 == 0), "tokens of a piece");
    const float xs = lane < nj ? a.x_scale[t0 + lane] : 0.f;
    if (EPI == Q8_SWIGLU) {
        // lanes 0..15 hold gates, 16..31 the ups of the same 16 products: of two tokens the lower lane computes the first and the
        // upper lane the second.  2^(-g log2 e) and its division are within 2^-21 (|g| + 4); the result is rounded to bf16.
        __nv_bfloat16 *o = reinterpret_cast<__nv_bfloat16 *>(a.out);
        const bool hi = lane & 16;
        const int pair = (f >> 5) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float y0 = (float)s[j] * l.ws * __shfl_sync(0xffffffffu, xs, j);
            const float y1 = N == 1 ? 0.f : (float)s[j + (N > 1)] * l.ws * __shfl_sync(0xffffffffu, xs, j + (N > 1));
            const float other = __shfl_xor_sync(0xffffffffu, hi ? y0 : y1, 16);
            const float g = hi ? other : y0, u = hi ? y1 : other;
            const float h = u * __fdividef(g, 1.0f + __expf(-g));
            if (l.on && j + hi < nj) o[(long long)(t0 + j + hi) * a.ld_out + pair] = __float2bfloat16_rn(h);
        }
        return;
    }
    float r[N];
    if (EPI == Q8_RESID) {  // all loads before the stores: out may be resid
#pragma unroll
        for (int j = 0; j < N; j++) r[j] = l.on && j < nj ? a.resid[(long long)(t0 + j) * a.ld_resid + f] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        float y = (float)s[j] * l.ws * __shfl_sync(0xffffffffu, xs, j);
        if (EPI == Q8_RESID) y = r[j] + y;
        else if (a.bias) y += l.bias;
        if (l.on && j < nj) {
            if (EPI == Q8_BF16) reinterpret_cast<__nv_bfloat16 *>(a.out)[(long long)(t0 + j) * a.ld_out + f] = __float2bfloat16_rn(y);
            else reinterpret_cast<float *>(a.out)[(long long)(t0 + j) * a.ld_out + f] = y;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// few tokens: a tile's k-blocks cut over the CTAs of a cluster
// ---------------------------------------------------------------------------------------------
__host__ __device__ constexpr int split_stage_bytes(int bn) { return (kBM + bn) * kBK; }
// two CTAs on an SM: one loads while the other starts or ends
__host__ __device__ constexpr int split_stages(int bn) { return 110 * 1024 / split_stage_bytes(bn); }
__host__ __device__ constexpr int split_smem(int bn) { return split_stages(bn) * split_stage_bytes(bn) + 1024; }

template <int BN, int EPI>
__global__ void __launch_bounds__(kQ8Threads)
    qw_q8_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Q8GemmArgs a,
                       int nsplit) {
    constexpr int S = split_stages(BN), B_BYTES = BN * kBK;
    constexpr uint32_t TMEM_COLS = BN < 32 ? 32 : BN, IDESC = q8_idesc(kBM, BN);
    static_assert(S * (kABytes + B_BYTES) >= BN * kBM * 4, "the sums of a tile lie in the ring's memory");
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S], tfull_bar;
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_sh;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sA = smem, *sB = smem + S * kABytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_sh;
    griddep_wait();
    griddep_launch_dependents();

    const int nt = (a.T + BN - 1) / BN, nkb = (a.K + kBK - 1) / kBK;
    const int tile = (int)blockIdx.x / nsplit, rank = (int)blockIdx.x % nsplit;
    const int t0 = (tile % nt) * BN, f0 = (tile / nt) * kBM;
    const int kb0 = (int)((long long)nkb * rank / nsplit), kb1 = (int)((long long)nkb * (rank + 1) / nsplit);

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0, issued = 0, last_ph = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!mbar_wait(&empty_bar[s], ph ^ 1u, abort_flag, a.err)) { ok = false; break; }
                mbar_arrive_expect_tx(&full_bar[s], kABytes + B_BYTES);
                tma_load_2d(sA + s * kABytes, &tmW, &full_bar[s], kb * kBK, f0);
                tma_load_2d(sB + s * B_BYTES, &tmX, &full_bar[s], kb * kBK, t0);
                issued |= 1u << s;
                last_ph = (last_ph & ~(1u << s)) | (ph << s);
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            if (!ok) {
                // let every issued copy land before the CTA's shared memory goes away
                for (int i = 0; i < S; i++)
                    if (issued >> i & 1u) {
                        const uint32_t addr = smem_u32(&full_bar[i]);
                        const uint64_t c0 = gtime_ns();
                        while (!mbar_try(addr, (last_ph >> i) & 1u) && gtime_ns() - c0 < kTcuWaitCycles) {
                        }
                    }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!mbar_wait(&full_bar[s], ph, abort_flag, a.err)) break;
                tc_fence_after();
                const uint64_t ad = sw128_desc(smem_u32(sA + s * kABytes)), bd = sw128_desc(smem_u32(sB + s * B_BYTES));
#pragma unroll
                for (int k = 0; k < kBK / 32; k++)
                    q8_mma<1>(tmem, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), IDESC, (kb > kb0 || k > 0) ? 1u : 0u);
                tc_commit(&empty_bar[s]);
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            tc_commit(&tfull_bar);
            // all MMAs of this CTA complete before the TMEM is freed
            const uint32_t addr = smem_u32(&tfull_bar);
            const uint64_t c0 = gtime_ns();
            while (!mbar_try(addr, 0) && gtime_ns() - c0 < kTcuWaitCycles) {
            }
        }
    }
    const int q = warp & 3, f = f0 + q * 32 + lane;
    const bool epilogue = warp >= 2;
    Q8Lane l{};
    if (epilogue) {
        l = q8_lane<EPI>(a, f);
        mbar_wait(&tfull_bar, 0, abort_flag, a.err);
        tc_fence_after();
        constexpr int P = BN < 32 ? 16 : 32;
        const int ncols = min(BN, a.T - t0);
        for (int c = 0; c < ncols; c += P) {
            uint32_t r[P];
            if constexpr (P == 16) tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, r);
            else tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, r);
            if (nsplit == 1) {
                int v[P];
#pragma unroll
                for (int j = 0; j < P; j++) v[j] = (int)r[j];
                q8_emit<EPI, P>(a, l, v, f, lane, t0 + c, min(P, ncols - c));
            } else {
                // the ring is free: every MMA that read it has completed
                int *part = reinterpret_cast<int *>(smem) + q * 32 + lane;
#pragma unroll
                for (int j = 0; j < P; j++) part[(c + j) * kBM] = (int)r[j];
            }
        }
    }
    if (nsplit > 1) {
        __syncwarp();
        cluster_sync_all();  // every CTA's sums are in its shared memory
        if (epilogue) {
            // this CTA's share of the tile's tokens, two at a time
            const int ncols = min(BN, a.T - t0);
            const int c0 = ncols * rank / nsplit, c1 = ncols * (rank + 1) / nsplit;
            const uint32_t mine = smem_u32(smem) + (uint32_t)(q * 32 + lane) * 4u;
            for (int c = c0; c < c1; c += 2) {
                int v[2] = {0, 0};
                for (int p = 0; p < nsplit; p++) {
                    const uint32_t at = cluster_map(mine, (uint32_t)p) + (uint32_t)c * (kBM * 4u);
                    v[0] += ld_cluster(at);
                    if (c + 1 < c1) v[1] += ld_cluster(at + kBM * 4u);
                }
                q8_emit<EPI, 2>(a, l, v, f, lane, t0 + c, min(2, c1 - c));
            }
        }
        __syncwarp();
        cluster_sync_all();  // no CTA leaves while another reads its sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------
// many tokens: persistent CTA pairs
// ---------------------------------------------------------------------------------------------
// A cluster of two CTAs computes 256 features x BN tokens with one tcgen05.mma stream issued by the even CTA; each CTA stages its
// own 128 rows of W and half of the tokens, and its tensor memory holds its 128 features' sums, in two accumulators.
//   full[s]   in the even CTA: its producer's expect_tx of both CTAs' bytes; both CTAs' loads count on it;
//   empty[s]  in each CTA, signalled by the MMA commit to both;
//   tfull[i]  in each CTA, signalled by the commit behind the tile's last k-block;
//   tempty[i] in the even CTA: 8 arrivals (the epilogue warps of both CTAs).
constexpr int kPairBM = 256;
constexpr int kPairGroupT = 8;  // token tiles per group of the tile order: their X tiles stay in L2 while W passes by
__host__ __device__ constexpr int pair_stage_bytes(int bn) { return kABytes + bn / 2 * kBK; }
__host__ __device__ constexpr int pair_stages(int bn) { return 224 * 1024 / pair_stage_bytes(bn); }
__host__ __device__ constexpr int pair_smem(int bn) { return pair_stages(bn) * pair_stage_bytes(bn) + 1024; }

struct PairTile {
    int f0, t0;
};
template <int BN>
__device__ __forceinline__ PairTile pair_tile(int tile, int nf, int nt) {
    const int per_group = nf * kPairGroupT;
    const int g = tile / per_group, r = tile % per_group;
    const int t_in = min(kPairGroupT, nt - g * kPairGroupT);
    return {(r / t_in) * kPairBM, (g * kPairGroupT + r % t_in) * BN};
}

template <int BN, int EPI>
__global__ void __launch_bounds__(kQ8Threads, 1)
    qw_q8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Q8GemmArgs a) {
    constexpr int S = pair_stages(BN), HALF = BN / 2, B_BYTES = HALF * kBK;
    constexpr uint32_t TMEM_COLS = 2 * BN, IDESC = q8_idesc(kPairBM, BN);
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S], tfull_bar[2], tempty_bar[2], done_bar;
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
            mbar_init(&tempty_bar[i], 8);
        }
        mbar_init(&done_bar, 1);
        abort_sh = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmW) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmX) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
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
                const PairTile c = pair_tile<BN>(tile, nf, nt);
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
                    if (issued >> i & 1u) {
                        const uint32_t addr = smem_u32(&full_bar[i]);
                        const uint64_t c0 = gtime_ns();
                        while (!mbar_try(addr, (last_ph >> i) & 1u) && gtime_ns() - c0 < kTcuWaitCycles) {
                        }
                    }
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
                    tc_commit_pair(&empty_bar[s]);
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
                if (ok) tc_commit_pair(&tfull_bar[acc]);
            }
            tc_commit_pair(&done_bar);
        }
    } else {
        // ---------------- epilogue (warps 2..5 of both CTAs) ----------------
        const uint32_t tempty0 = cluster_map(smem_u32(&tempty_bar[0]), 0);
        const int q = warp & 3;
        int it = 0;
        for (int tile = cid; tile < total; tile += ncl, it++) {
            const PairTile c = pair_tile<BN>(tile, nf, nt);
            const int acc = it & 1, f = c.f0 + (int)rank * kBM + q * 32 + lane;
            const Q8Lane l = q8_lane<EPI>(a, f);
            if (!mbar_wait(&tfull_bar[acc], (uint32_t)(it >> 1) & 1u, abort_flag, a.err)) break;
            tc_fence_after();
            const int ncols = min(BN, a.T - c.t0);
            for (int cc = 0; cc < ncols; cc += 32) {
                uint32_t r[32];
                tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + cc), r);
                int v[32];
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = (int)r[j];
                q8_emit<EPI, 32>(a, l, v, f, lane, c.t0 + cc, min(32, ncols - cc));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * (uint32_t)acc);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1 && lane == 0) {
        // every MMA of the pair has completed (they read both CTAs' shared memory and write both TMEMs)
        const uint32_t addr = smem_u32(&done_bar);
        const uint64_t c0 = gtime_ns();
        while (!mbar_try(addr, 0) && gtime_ns() - c0 < kTcuWaitCycles) {
        }
    }
    __syncthreads();
    cluster_sync_all();  // no CTA leaves while its peer may still signal its barriers
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
cudaError_t launch_cluster(const void *fn, int grid, int cluster, int smem, cudaStream_t st, void **args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kQ8Threads);
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

struct Q8Kernel {
    const void *fn;
    int smem;
};
template <int EPI>
Q8Kernel split_kernel(int bn) {
    switch (bn) {
        case 16: return {(const void *)qw_q8_split_kernel<16, EPI>, split_smem(16)};
        case 32: return {(const void *)qw_q8_split_kernel<32, EPI>, split_smem(32)};
        case 64: return {(const void *)qw_q8_split_kernel<64, EPI>, split_smem(64)};
        default: return {(const void *)qw_q8_split_kernel<128, EPI>, split_smem(128)};
    }
}
template <int EPI>
Q8Kernel pair_kernel(int bn) {
    return bn == 128 ? Q8Kernel{(const void *)qw_q8_pair_kernel<128, EPI>, pair_smem(128)}
                     : Q8Kernel{(const void *)qw_q8_pair_kernel<256, EPI>, pair_smem(256)};
}
Q8Kernel q8_kernel(int epi, bool pair, int bn) {
    switch (epi) {
        case Q8_F32: return pair ? pair_kernel<Q8_F32>(bn) : split_kernel<Q8_F32>(bn);
        case Q8_BF16: return pair ? pair_kernel<Q8_BF16>(bn) : split_kernel<Q8_BF16>(bn);
        case Q8_RESID: return pair ? pair_kernel<Q8_RESID>(bn) : split_kernel<Q8_RESID>(bn);
        default: return pair ? pair_kernel<Q8_SWIGLU>(bn) : split_kernel<Q8_SWIGLU>(bn);
    }
}

// Every kernel opted in to its shared memory, once per device.
cudaError_t q8_prepare(int dev) {
    static std::mutex mu;
    static bool prepared[64] = {};
    std::lock_guard<std::mutex> lk(mu);
    if (dev < 64 && prepared[dev]) return cudaSuccess;
    for (int epi = Q8_F32; epi <= Q8_SWIGLU; epi++)
        for (int bn = 16; bn <= 256; bn *= 2)
            for (int pair = 0; pair < 2; pair++) {
                if (pair ? bn < 128 : bn > 128) continue;
                const Q8Kernel k = q8_kernel(epi, pair, bn);
                cudaError_t e = cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
                if (e != cudaSuccess) return e;
            }
    if (dev < 64) prepared[dev] = true;
    return cudaSuccess;
}

struct Q8Plan {
    bool pair;
    int bn, nsplit;
};
Q8Plan q8_plan(int M, int T, int K, int sms) {
    const int nkb = (K + kBK - 1) / kBK;
    const long long pairs = (long long)((M + kPairBM - 1) / kPairBM);
    if (T > 128 && pairs * ((T + 127) / 128) >= sms / 4) {
        if (pairs * ((T + 255) / 256) >= sms / 2) return {true, 256, 1};
        return {true, 128, 1};
    }
    const int bn = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
    const long long tiles = (long long)((M + kBM - 1) / kBM) * ((T + bn - 1) / bn);
    int n = (int)(2 * sms / tiles);
    n = n < 1 ? 1 : n > 8 ? 8 : n;
    if (n > (nkb + 1) / 2) n = (nkb + 1) / 2;
    return {false, bn, n};
}

cudaError_t q8_gemm_launch(const int8_t *w, long long ld_w, const int8_t *x, long long ld_x, const Q8GemmArgs &a, int epi, int sms,
                           cudaStream_t st) {
    const Q8Plan p = q8_plan(a.M, a.T, a.K, sms);
    const Q8Kernel k = q8_kernel(epi, p.pair, p.bn);
    CUtensorMap mw, mx;
    cudaError_t e = codes_map(&mw, w, a.M, a.K, ld_w, kBM);
    if (e == cudaSuccess) e = codes_map(&mx, x, a.T, a.K, ld_x, p.pair ? p.bn / 2 : p.bn);
    if (e != cudaSuccess) return e;
    int nsplit = p.nsplit;
    void *args[] = {(void *)&mw, (void *)&mx, (void *)&a, (void *)&nsplit};
    const long long tiles = (long long)((a.M + (p.pair ? kPairBM : kBM) - 1) / (p.pair ? kPairBM : kBM)) * ((a.T + p.bn - 1) / p.bn);
    if (p.pair) {
        const int ncl = (int)(tiles < sms / 2 ? tiles : sms / 2);
        return launch_cluster(k.fn, 2 * ncl, 2, k.smem, st, args);
    }
    if (tiles * nsplit > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    return launch_cluster(k.fn, (int)tiles * nsplit, nsplit, k.smem, st, args);
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
    if (((uintptr_t)p->w | (uintptr_t)p->x) & 15) return op_fail(QW_ERR_ARG, "w and x must be 16-byte aligned");
    if ((((uintptr_t)p->w_scale | (uintptr_t)p->x_scale | (uintptr_t)p->bias | (uintptr_t)p->resid | (uintptr_t)p->err) & 3) ||
        (uintptr_t)p->out % (p->out_dtype == QW_DTYPE_BF16 ? 2 : 4))
        return op_fail(QW_ERR_ARG, "pointers must be aligned to their elements");
    a.w_scale = p->w_scale; a.x_scale = p->x_scale; a.bias = p->bias; a.resid = p->resid;
    a.out = p->out; a.err = p->err; a.M = p->n_out; a.K = p->k; a.T = p->t;
    const int epi = p->epi == QW_LINEAR_RESID ? Q8_RESID : p->epi == QW_LINEAR_SWIGLU ? Q8_SWIGLU
                  : p->out_dtype == QW_DTYPE_BF16 ? Q8_BF16 : Q8_F32;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return op_fail(QW_ERR_CUDA, "no current device");
    cudaError_t e = q8_prepare(dev);
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("linear set-up: ") + cudaGetErrorString(e));
    e = q8_gemm_launch(p->w, ld_w, p->x, ld_x, a, epi, sms, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("linear launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
