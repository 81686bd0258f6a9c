// qw_chunk_attn_tc.cu -- attention of a ragged batch of new tokens over the paged bf16 cache on the 5th-generation
// tensor cores (the semantics are those of qw_chunk_attn.cu).
//
// The G query heads of a KV head share its keys, so the rows of a query tile are (position, head of the group) pairs:
// P = floor(128 / G) positions of all G heads, at most 128 rows, one row per TMEM lane.  An item is two such tiles of
// one sequence and KV head; a K / V block of 128 keys serves both.  The key blocks of all items, in the order
// sequence, KV head, tiles, form one line that is cut into equal shares, one per CTA (one CTA per SM): every SM gets
// the same number of blocks whatever the lengths are.  An item cut once is finished by the CTA in which it begins, from
// the other's partial result (O, maximum, sum) in the workspace; the CTAs that share an item cut more often join its
// rows, each a part of them, once all are there.  Where there are no more items than SMs and none much longer than a
// share would be, a CTA takes each item whole.
//
// An item with one tile only (decoding: G rows; the last rows of a chunk) gives its blocks to the two tile slots in
// turn, so that one slot's softmax still runs while the tensor cores work on the other; the slots' results are joined
// at the item's end.
//
// What bounds it (32 heads over 8 KV heads of 128 where not said otherwise):
//   long chunks: a slot's chain S (690 clocks), softmax (1900, of which the exponentials of two slots on the 16 a clock of
//     an SM take 1024 each), P V (560) and the commits between them, beside the other slot's: a pair of blocks every 3700
//     clocks.  4096 rows over 20096 positions: 1010 us, 1.20 PFLOP/s (0.73 of what cuBLAS reaches); 1140 us once the power
//     limit holds the clock down
//   single tokens: HBM.  64 sequences over 3900..4250 positions: 168 us, 6.4 TB/s (176 under the
//     power limit); one over 120001: 86 us, 5.7 TB/s
//   short ones: the way to the first scores (11000 clocks: lengths, schedule, page table, first keys), a visit of a block
//     after the other (1800 clocks of softmax each), the join of cut items; a token on 300 positions 10 us
// 16 softmax warps with two threads per row against 8 with one: 1187 against 1441 us (4096 rows over 20096 positions).
//
// Warps (five warpgroups):
//   0     K and V: TMA boxes of min(page, 128) rows into rings of tc_stages tiles each, one lane per box
//   1, 2  the MMAs of a slot each: S_t = Q_t K^T, then O_t += P_t V as soon as slot t's softmax has written P_t over S_t;
//         they also clear the rows of a V block that the sequence never sees (0 x NaN is NaN)
//   3     walks the CTA's share of the line, hands its pieces to the other warps through a ring, and loads their queries:
//         one box of (64 columns, G heads, P positions) per 64 columns
//   4..11 softmax and result of slot 0: a warp has 16 rows, two threads per row (64 keys, and half of the columns of O,
//         each), so that one warp's loads, maxima and stores run beside another's exponentials; 12..19 of slot 1
// Every wait is bounded; one that runs out sets the error word and ends the CTA (its copies landed, its TMEM freed).
#include <cuda.h>
#include <cuda_runtime.h>
#include <atomic>

#include "../../include/qwen3_b200.h"
#include "qw_chunk_attn.h"
#include "qw_internal.cuh"
#include "qw_tc.h"
#include "qw_tc_util.cuh"

namespace qw {
namespace {

constexpr int kThreads = 640, kSoftThreads = 512, kRows = 128, kKeys = 128, kMaxStages = 5;
// The running maximum is raised only when it grows by more than 8 (in log2 units): p stays below 2^8, and O is seldom
// rescaled.  4096 rows over 20096 positions 1005 us, 1104 with every maximum; 8 chunks on old sequences 127 and 138.
constexpr float kRescale = 8.f;
constexpr int kPieces = 4;       // ring of pieces
// Rows of an exchange between the slots in shared memory: a token's heads of one KV head.  Through the workspace, as more
// rows go, 64 single tokens took 184 instead of 174 us, 32 of them beside a chunk 96 instead of 84.
constexpr int kFewRows = 8;
// What a tile costs beside its blocks, in blocks: its queries and results.  8 prompts of 1420..1962 tokens take 214 us, 216
// with 1 and 228 with 4 (32 tokens beside a chunk 84, 86, 86; 8 chunks on old sequences 127, 127, 125).
constexpr int kItemUnits = 2;
// Units of a share at least; with fewer it might hold no block of an item that it lies in.  A token on 2000 positions, 8 KV
// heads: 13.2 us; with 3 units 14.1, with 5 15.6, with 10 22.0.
constexpr int kMinShare = 2;
// What a cut costs in units: items are left whole where the longest has at most so many more than a share.  5 tokens on
// 100..1500 positions take 12.7 instead of 18.6 us, 6 chunks under a window 30.8 instead of 35.2.  With 4, 17 tokens on
// 100..1500 positions take 22.3 instead of 19.6; with 8, one on 900 takes 14.8 instead of 12.6.
constexpr int kJoinUnits = 6;
constexpr int kCounterWords = 256;  // arrivals | arrivals at items cut once | departures, one word per CTA each
static_assert(3 * kCounterWords * 4 == kChunkCounterBytes && kNumSMsB200 <= kCounterWords, "counters");

__host__ __device__ constexpr int tc_stages(int d) { return d == 128 ? 2 : 5; }
__host__ __device__ constexpr int tc_tile_bytes(int d) { return kRows * d * 2; }
__host__ __device__ constexpr size_t part_bytes(int d) { return (size_t)kRows * d * 4 + kRows * 8; }

struct Seq {
    int n, kv, r0;  // new rows, cached positions, first row
};

// one piece of an item, as the scheduler hands it out
struct Piece {
    int flags;       // kEnd, kPair, ...
    int blk0, nblk;  // key blocks (absolute number of the first)
    int r0;          // ring index of the first block
    int q0;          // Q ring index of its first tile
    int alt;         // parity of the single-tile blocks before it: which slot takes its first block
    int row0, pos0;  // first row of the item and its position
    int n0, n1;      // positions in its tiles
    int kvh, slot;   // KV head, page-table row
    int lo, hi;      // positions that its rows see
    int clo, chi;    // positions that some row of the sequence sees: the cache holds something there
};
// kHead: the item begins in this share; kTwo: and is cut once; kOnce: no other item has its sequence's keys; kLow: one tile
// of 16 rows at most
enum { kEnd = 1, kPair = 2, kWhole = 4, kHead = 8, kTwo = 16, kOnce = 32, kLow = 64 };

// an item that several CTAs share
struct Shared {
    int on, c0, np, pair, rows0, rows, row, head;
};

struct __align__(16) Smem {
    unsigned pre[kChunkMaxBatch + 1];   // units of the line before each sequence
    unsigned whole[kChunkMaxBatch + 1]; // items of the line before each sequence
    Seq seq[kChunkMaxBatch];
    Piece piece[kPieces];
    Shared shared[2];
    uint64_t k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages], q_full[2], q_empty[2],
        s_full[2], p_full[2], o_full[2], x_full[2], x_empty[2], w_full[kPieces], w_empty[kPieces], turn[2], done[2], zeroed;
    uint32_t tmem;
    float4 xo[2][128 / 4 * kFewRows];  // [slot]: O as float4 columns of kFewRows rows (16-byte aligned by its type)
    float2 xml[2][kFewRows];
    int abort, go;
    int empty;  // some rows stand before their sequence's first position
    int unordered;  // row_start does not ascend
};

// one item's keys
struct Item {
    int nsub, f, pf, pl, klo, j0, nb;  // tiles; first new row; positions of the first and last row; first seen; blocks
    // a visit of a slot is a unit: a block costs as many as the item has tiles, and its queries and results kItemUnits
    // per tile; an item that sees nothing is not on the line
    __device__ __forceinline__ unsigned units() const { return nb ? (nb + kItemUnits) * nsub : 0; }
    // on a line of whole items, each is one unit
    __device__ __forceinline__ unsigned units(bool flat) const { return flat ? nb > 0 : units(); }
    __device__ __forceinline__ int blocks_before(int u, bool flat) const {
        return flat && u ? nb : min(nb, nsub == 2 ? (u + 1) >> 1 : u);
    }
};
__device__ __forceinline__ Item make_item(const Seq &s, int i, int P, int window) {
    Item it;
    it.f = i * 2 * P;
    const int l = min(s.n, it.f + 2 * P) - 1, p0 = s.kv - s.n;
    it.nsub = s.n - it.f > P ? 2 : 1;
    it.pf = p0 + it.f;
    it.pl = p0 + l;
    it.klo = window ? max(0, it.pf - window + 1) : 0;
    it.j0 = it.klo / kKeys;
    it.nb = it.pl < 0 ? 0 : it.pl / kKeys - it.j0 + 1;
    return it;
}

// sum of floor((a i + b) / 128) over i in [0, n), a even and positive, b >= 0: floor(x / 128) = (x - x mod 128) / 128, and the
// remainders repeat every 128 / gcd(a, 128) terms
__device__ __forceinline__ unsigned floor_sum(unsigned n, unsigned a, unsigned b) {
    const unsigned g = min(a & (0u - a), (unsigned)kKeys), p = kKeys / g, r = n & (p - 1);
    unsigned long long rest = (unsigned long long)((n - r) / p) * (p * (b & (g - 1)) + g * p * (p - 1) / 2);
    for (unsigned i = 0, x = b & (kKeys - 1); i < r; i++, x = (x + a) & (kKeys - 1)) rest += x;
    return (unsigned)(((unsigned long long)n * (n - 1) / 2 * a + (unsigned long long)n * b - rest) / kKeys);
}
// units of a sequence of ni > 0 items and one KV head: all items but the last have two whole tiles
__device__ __forceinline__ unsigned seq_units(const Seq &s, int ni, int gone, int P, int window) {
    const int p0 = s.kv - s.n, m = max(0, ni - 1 - gone), step = 2 * P;  // m whole items from item `gone` on see something
    unsigned u = make_item(s, ni - 1, P, window).units();
    if (m > 0) {
        unsigned blocks = floor_sum(m, step, p0 + step * (gone + 1) - 1) + m * (1 + kItemUnits);
        if (window) {
            const int before = window - 1 - p0;  // rows that see from the first position on
            const int i = max(gone, before > 0 ? (before + step - 1) / step : 0);
            if (i < ni - 1) blocks -= floor_sum(ni - 1 - i, step, step * i - before);
        }
        u += 2 * blocks;
    }
    return u;
}

// the line of W units in Ge shares: the first W % Ge of them one unit longer
struct Line {
    unsigned q, rem;
    __device__ __forceinline__ unsigned start(unsigned c) const { return c * q + min(c, rem); }
    __device__ __forceinline__ unsigned owner(unsigned u) const {
        const unsigned head = rem * (q + 1);
        return u < head ? u / (q + 1) : rem + (u - head) / q;
    }
};

// K-major or MN-major 128-byte-swizzled operand descriptor; lbo / sbo in bytes
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
           (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// The MMAs and commits are predicated on the elected lane inside the instruction sequence, not branched around: the
// whole warp computes their operands, which the compiler then keeps in uniform registers.
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc,
                                       uint32_t elect) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc), "r"(elect)
        : "memory");
}
// with the A operand (P) in tensor memory: two bf16 per 32-bit column along K
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc,
                                       uint32_t elect) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc), "r"(elect)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar, uint32_t elect) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "setp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(elect)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d_hint(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], "
        "[%4], %5;" ::"r"(smem_u32(dst)),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(smem_u32(dst)),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
// 16 TMEM lanes in two column groups: threads 0..15 take column taddr + i, threads 16..31 column taddr + SPLIT + i
template <int SPLIT>
__device__ __forceinline__ void ld32(uint32_t taddr, float *v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.16x32bx2.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32], %33;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr), "n"(SPLIT));
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
template <int SPLIT>
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t *o) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x32bx2.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16], %17;"
        : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]), "=r"(o[8]),
          "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
        : "r"(taddr), "n"(SPLIT));
}
template <int SPLIT>
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x32bx2.x16.b32 [%0], %17, "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "n"(SPLIT)
        : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unf2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 32 bytes, a whole sector of a row per lane, where the rows are so aligned (16 bytes are all that is asked of them)
__device__ __forceinline__ void store32(void *p, const uint32_t *v, bool aligned32) {
    if (aligned32) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                     "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4 *>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<uint4 *>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
}
__device__ __forceinline__ void bar_softmax() { asm volatile("bar.sync 1, %0;" ::"n"(kSoftThreads) : "memory"); }
__device__ __forceinline__ unsigned ld_acquire(const unsigned *p) {
    unsigned v;
    asm volatile("ld.acquire.gpu.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void red_release(unsigned *p) {
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory");
}
__device__ __forceinline__ int uni(int x) { return __shfl_sync(0xffffffffu, x, 0); }
// whether a phase is over, without the pause of a wait
__device__ __forceinline__ bool mbar_test(uint64_t *b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// a bounded wait that ends the same way for every lane of the warp
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity, volatile int *abort_flag, int *err) {
    return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, err));
}

// A partial result: O as float4 columns [D / 4][128 rows], then (maximum in log2 units, sum) per row.
template <int D>
struct Part {
    char *p;
    __device__ __forceinline__ float4 *o(int c4, int row) const { return reinterpret_cast<float4 *>(p) + c4 * kRows + row; }
    __device__ __forceinline__ float2 *ml(int row) const { return reinterpret_cast<float2 *>(p + (size_t)kRows * D * 4) + row; }
};
// which: 0 the share's first piece, 1 its last, 2 the exchange between the slots (of more than kFewRows rows; fewer go
// through shared memory); k: tile, or slot in turn
template <int D>
__device__ __forceinline__ Part<D> part_of(const ChunkArgs &a, int cta, int which, int k) {
    return Part<D>{(char *)a.workspace + kChunkCounterBytes + ((size_t)cta * 6 + which * 2 + k) * part_bytes(D)};
}

template <int D>
__device__ __forceinline__ void put_row(const ChunkArgs &a, const Shared &m, int r, int c4, const float4 &o, float M, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t grow = (size_t)(m.row + r / a.G);
    const int head = m.head + r % a.G;
    *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(a.out) + grow * a.ld_out + (size_t)head * D + c4 * 4) =
        make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
    if (c4 == 0 && a.lse) a.lse[grow * a.H + head] = l == 0.f ? -INFINITY : (M + __log2f(l)) * 0.69314718055994531f;
}

// Rows [lo, lo + nr) of a shared item: sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p, m = max m_p, over its parts.  (A part
// of NaN scores has no maximum, but a sum of NaN.)
template <int D>
__device__ __forceinline__ void join_rows(const ChunkArgs &a, const Shared &m, int lo, int nr, int tid, float *red) {
    const int nparts = m.pair ? m.np : 2 * m.np;
    auto part = [&](int p, int tile) {
        const int k = m.pair ? p : p >> 1;
        return part_of<D>(a, m.c0 + k, k == 0 ? 1 : 0, m.pair ? tile : p & 1);
    };
    if (nr >= 16) {
        // lanes take rows (the parts' columns are contiguous over rows), a warp 8 float4 columns of 32 rows at a time
        const int lane = tid & 31, ntask = (nr + 31) / 32 * (D / 32);
        for (int task = tid >> 5; task < ntask; task += kSoftThreads / 32) {
            const int r = lo + task / (D / 32) * 32 + lane, c0 = task % (D / 32) * 8;
            if (r >= lo + nr) continue;
            const int tile = r >= m.rows0, row = r - (tile ? m.rows0 : 0);
            float M = -INFINITY, l = 0.f;
            float4 o[8];
#pragma unroll
            for (int c = 0; c < 8; c++) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int p = 0; p < nparts; p++) {
                const Part<D> px = part(p, tile);
                const float2 ml = __ldcg(px.ml(row));
                float4 x[8];
#pragma unroll
                for (int c = 0; c < 8; c++) x[c] = __ldcg(px.o(c0 + c, row));
                if (ml.y == 0.f) continue;  // nothing seen there (O may not have been written)
                const float mn = fmaxf(M, ml.x), wo = ex2(M - mn), wx = ex2(ml.x - mn);
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    o[c].x = o[c].x * wo + x[c].x * wx; o[c].y = o[c].y * wo + x[c].y * wx;
                    o[c].z = o[c].z * wo + x[c].z * wx; o[c].w = o[c].w * wo + x[c].w * wx;
                }
                l = l * wo + ml.y * wx;
                M = mn;
            }
#pragma unroll
            for (int c = 0; c < 8; c++) put_row<D>(a, m, r, c0 + c, o[c], M, l);
        }
        return;
    }
    // few rows: a thread takes 4 columns of a row, several threads share the parts
    const int E = nr * (D / 4), ng = max(1, kSoftThreads / E);
    for (int e0 = 0; e0 < E; e0 += kSoftThreads) {
        const int g = E < kSoftThreads ? tid / E : 0, e = E < kSoftThreads ? tid % E : e0 + tid;
        const bool on = g < ng && e < E;
        const int r = lo + e % nr, c4 = e / nr;
        const int tile = r >= m.rows0, row = r - (tile ? m.rows0 : 0);
        float M = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on) {
#pragma unroll 4
            for (int p = g; p < nparts; p += ng) {
                const Part<D> px = part(p, tile);
                const float2 ml = __ldcg(px.ml(row));
                const float4 x = __ldcg(px.o(c4, row));
                if (ml.y == 0.f) continue;
                const float mn = fmaxf(M, ml.x), wo = ex2(M - mn), wx = ex2(ml.x - mn);
                o.x = o.x * wo + x.x * wx; o.y = o.y * wo + x.y * wx;
                o.z = o.z * wo + x.z * wx; o.w = o.w * wo + x.w * wx;
                l = l * wo + ml.y * wx;
                M = mn;
            }
        }
        if (ng > 1) {  // one round
            float *mine = red + tid * 8;
            if (on) { mine[0] = M; mine[1] = l; mine[2] = o.x; mine[3] = o.y; mine[4] = o.z; mine[5] = o.w; }
            bar_softmax();
            if (on && g == 0)
                for (int h = 1; h < ng; h++) {
                    const float *x = red + (h * E + e) * 8;
                    if (x[1] == 0.f) continue;
                    const float mn = fmaxf(M, x[0]), wo = ex2(M - mn), wx = ex2(x[0] - mn);
                    o.x = o.x * wo + x[2] * wx; o.y = o.y * wo + x[3] * wx;
                    o.z = o.z * wo + x[4] * wx; o.w = o.w * wo + x[5] * wx;
                    l = l * wo + x[1] * wx;
                    M = mn;
                }
        }
        if (on && g == 0) put_row<D>(a, m, r, c4, o, M, l);
    }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    qw_chunk_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQ1,
                            const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const ChunkArgs a) {
    constexpr int NST = tc_stages(D), TILE = tc_tile_bytes(D), HALF = kRows * 128, NH = D / 64;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Smem sh;
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sQ = sm, *sK = sm + 2 * TILE, *sV = sK + NST * TILE;
    // (values shuffled from lane 0 are known to be the same in the whole warp: what is computed from them stays in
    // uniform registers, where the MMA's operands have to be)
    const int warp = uni(threadIdx.x >> 5), lane = threadIdx.x & 31;
    volatile int *abort_flag = &sh.abort;
    const int G = a.G, P = kRows / G;

    // the scheduler's first lengths are on their way while the rest is set up
    int len0 = 0, len1 = 0, len2 = 0;
    if (warp == 3 && lane < a.batch) {
        len0 = a.row_start[lane];
        len1 = a.row_start[lane + 1];
        len2 = a.kv_len[lane];
    }
    if (warp == 2 && lane == 0) {
        for (int i = 0; i < NST; i++) {
            mbar_init(&sh.k_full[i], 1);
            mbar_init(&sh.k_empty[i], 2);
            mbar_init(&sh.v_full[i], 1);
            mbar_init(&sh.v_empty[i], 2);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.q_empty[i], 2);
            mbar_init(&sh.turn[i], 1);
            mbar_init(&sh.done[i], 1);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 8);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.x_full[i], 8);
            mbar_init(&sh.x_empty[i], 8);
            sh.shared[i].on = 0;
        }
        mbar_init(&sh.zeroed, kSoftThreads / 32);
        for (int i = 0; i < kPieces; i++) {
            mbar_init(&sh.w_full[i], 1);
            mbar_init(&sh.w_empty[i], 19);  // K / V, two MMA warps, sixteen softmax warps
        }
        sh.abort = 0;
        sh.empty = sh.unordered = 0;
        sh.pre[0] = sh.whole[0] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmQ) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmK) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmV) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's: the allocation begins at column 0
    const int cta = blockIdx.x;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 3) {
            // ---------------- the scheduler ----------------
            // units of every sequence and their running sum
            unsigned W = 0;
            unsigned items = 0, most = 0;  // that see something; units of the largest
            for (int b0 = 0; b0 < a.batch; b0 += 32) {
                const int b = b0 + lane;
                Seq s{0, 0, 0};
                if (b < a.batch) {
                    s.r0 = min(max(len0, 0), a.rows);
                    s.n = max(0, min(len1, a.rows) - s.r0);
                    s.kv = min(max(len2, 0), a.max_pages << a.log2_ps);
                    sh.seq[b] = s;
                    if (len1 < len0) sh.unordered = 1;
                }
                if (b + 32 < a.batch) {
                    len0 = a.row_start[b + 32];
                    len1 = a.row_start[b + 33];
                    len2 = a.kv_len[b + 32];
                }
                if (s.n > s.kv) sh.empty = 1;
                const int ni = s.n <= 2 * P ? s.n > 0 : (s.n + 2 * P - 1) / (2 * P);
                const int gone = s.n > s.kv ? (s.n - s.kv) / (2 * P) : 0;  // items before the first position
                const unsigned units = ni ? seq_units(s, ni, gone, P, a.window) : 0;
                unsigned big = ni ? make_item(s, ni - 1, P, a.window).units() : 0;
                if (ni > 1) big = max(big, make_item(s, ni - 2, P, a.window).units());
                most = max(most, __reduce_max_sync(0xffffffffu, big));
                unsigned v = units * a.Hkv, c = s.kv > 0 ? (ni - gone) * a.Hkv : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned w = __shfl_up_sync(0xffffffffu, v, o), x = __shfl_up_sync(0xffffffffu, c, o);
                    if (lane >= o) {
                        v += w;
                        c += x;
                    }
                }
                if (b < a.batch) {
                    sh.pre[b + 1] = W + v;
                    sh.whole[b + 1] = items + c;
                }
                W += __shfl_sync(0xffffffffu, v, 31);
                items += __shfl_sync(0xffffffffu, c, 31);
            }
            __syncwarp();
            if (sh.unordered) {
                // Sequences that overlap may name more units than the host allowed for, and than 32 bits number: then
                // nothing is scheduled.  (Units in 2^16, rounded down for each sequence.)
                unsigned t = 0;
                for (int b = lane; b < a.batch; b += 32) t += (sh.pre[b + 1] - sh.pre[b]) >> 16;
                if (__reduce_add_sync(0xffffffffu, t) >= 0x10000u - kChunkMaxBatch) {
                    W = items = 0;
                    if (lane == 0 && a.err) atomicExch(a.err, TC_DEVERR_LENGTHS);
                }
            }
            // Cut items save time only where the longest one is well above a share; otherwise a CTA takes each item whole.
            const unsigned grid = gridDim.x;
            const bool flat = items <= grid && most <= max((unsigned)kMinShare, W / grid) + kJoinUnits;
            if (flat) W = items;
            const int Ge = flat ? items : min(grid, max(items, W / kMinShare));
            const unsigned *pre = flat ? sh.whole : sh.pre;
            Line line{0, 0};
            unsigned at = 0, end = 0;
            int b = 0, h = 0, i = 0, off = 0;
            if (cta < Ge) {  // W / Ge >= kMinShare where items are cut: an item has three units at least
                line.q = W / Ge;
                line.rem = W - line.q * Ge;
                at = line.start(cta);
                end = line.start(cta + 1);
                unsigned rem = 0, per = 1;
                for (int b0 = 0; b0 < a.batch; b0 += 32) {  // the sequence that holds unit `at`
                    const unsigned p0 = b0 + lane < a.batch ? pre[b0 + lane] : 0xffffffffu;
                    const unsigned p1 = b0 + lane < a.batch ? pre[b0 + lane + 1] : 0xffffffffu;
                    const unsigned m = __ballot_sync(0xffffffffu, p0 <= at && at < p1);
                    if (m) {
                        const int l = __ffs(m) - 1;
                        b = b0 + l;
                        rem = at - __shfl_sync(0xffffffffu, p0, l);
                        per = __shfl_sync(0xffffffffu, p1 - p0, l) / a.Hkv;
                        break;
                    }
                }
                if (rem >= per) {
                    h = (int)(rem / per);
                    rem -= h * per;
                }
                const Seq s = sh.seq[b];
                for (; i * 2 * P < s.n; i += 32) {  // the item that holds unit rem of this head
                    unsigned v = (i + lane) * 2 * P < s.n ? make_item(s, i + lane, P, a.window).units(flat) : 0;
                    if (s.n <= 2 * P) {  // the only one
                        off = (int)rem;
                        break;
                    }
                    const unsigned mine = v;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned w = __shfl_up_sync(0xffffffffu, v, o);
                        if (lane >= o) v += w;
                    }
                    const unsigned m = __ballot_sync(0xffffffffu, v > rem);
                    if (m) {
                        const int k = __ffs(m) - 1;
                        i += k;
                        off = (int)(rem - __shfl_sync(0xffffffffu, v - mine, k));
                        break;
                    }
                    rem -= __shfl_sync(0xffffffffu, v, 31);
                }
            }
            int np = 0, rn = 0, qn = 0, alt = 0, q_sent = 0, clean = 3;  // clean: query tiles whose rows from G on are zero
            bool ok = warp_wait(&sh.zeroed, 0, abort_flag, a.err);
            while (ok) {
                Piece pc;
                pc.flags = kEnd;
                Item it;
                Seq s;
                unsigned u0 = 0;
                int ch = 0, cb = 0;
                while (at < end) {
                    s = sh.seq[b];
                    if (s.n <= 0) { b++; continue; }
                    it = make_item(s, i, P, a.window);
                    const int units = (int)it.units(flat);
                    const int take = min(units - off, (int)(end - at));
                    const int ja = it.blocks_before(off, flat), jb = it.blocks_before(off + take, flat);
                    u0 = at - off;
                    cb = b; ch = h;
                    at += take;
                    off += take;
                    if (off == units) {
                        off = 0;
                        if ((++i) * 2 * P >= s.n) {
                            i = 0;
                            if (++h == a.Hkv) { h = 0; b++; }
                        }
                    }
                    if (ja < jb) {
                        pc.flags = (it.nsub == 2 ? kPair : 0) | (ja == 0 && jb == it.nb ? kWhole : 0) | (ja == 0 ? kHead : 0) |
                                   (s.n <= 2 * P ? kOnce : 0) |
                                   (it.nsub == 1 && (s.n - it.f) * G <= 16 ? kLow : 0);
                        pc.blk0 = it.j0 + ja;
                        pc.nblk = jb - ja;
                        break;
                    }
                }
                ok = warp_wait(&sh.w_empty[np % kPieces], (uint32_t)(np / kPieces + 1) & 1u, abort_flag, a.err);
                if (!ok) break;
                if (!(pc.flags & kEnd)) {
                    pc.r0 = rn; pc.q0 = qn; pc.alt = alt & 1;
                    rn += pc.nblk;
                    qn += it.nsub;
                    if (it.nsub == 1) alt += pc.nblk;
                    pc.row0 = s.r0 + it.f; pc.pos0 = it.pf;
                    pc.n0 = min(P, s.n - it.f); pc.n1 = it.nsub == 2 ? min(P, s.n - it.f - P) : 0;
                    pc.kvh = ch; pc.slot = a.slots ? a.slots[cb] : cb;
                    pc.lo = it.klo; pc.hi = it.pl;
                    pc.clo = a.window ? max(0, s.kv - s.n - a.window + 1) : 0;
                    pc.chi = s.kv;
                    // the CTAs that the item lies in: mostly this one and its neighbour
                    int c0 = cta, ni = 1;
                    if (!(pc.flags & kWhole)) {
                        if (!(pc.flags & kHead)) c0 = u0 >= line.start(cta - 1) ? cta - 1 : (int)line.owner(u0);
                        const unsigned last = u0 + (it.nb - 1) * it.nsub;  // where its last block begins
                        const int c1 = last < line.start(cta + 1) ? cta : last < line.start(cta + 2) ? cta + 1 : (int)line.owner(last);
                        ni = c1 - c0 + 1;
                    }
                    if (ni == 2) pc.flags |= kTwo;
                    if (ni > 2 && lane == 0) {
                        Shared &m = sh.shared[pc.flags & kHead ? 1 : 0];
                        m.on = 1;
                        m.c0 = c0;
                        m.np = ni;
                        m.pair = it.nsub == 2;
                        m.rows0 = pc.n0 * G;
                        m.rows = (pc.n0 + pc.n1) * G;
                        m.row = pc.row0;
                        m.head = ch * G;
                    }
                }
                if (lane == 0) {
                    sh.piece[np % kPieces] = pc;
                    mbar_arrive(&sh.w_full[np % kPieces]);
                }
                __syncwarp();
                np++;
                if (pc.flags & kEnd) break;
                // The piece's queries.  Of a single token only its own rows are fetched, as long as the tile's others are the
                // zeros of the start: rows of other sequences would cost their way here and, multiplied with every key, power
                // (64 tokens over 3900..4250 positions, for seconds, the power limit holding the clock down: 184 us, 194 with them).
                const bool token = pc.n0 == 1 && it.nsub == 1;
                for (int q = pc.q0; q < pc.q0 + it.nsub && ok; q++) {
                    const int e = q & 1;
                    ok = warp_wait(&sh.q_empty[e], ((uint32_t)(q >> 1) & 1u) ^ 1u, abort_flag, a.err);
                    if (!ok) break;
                    const bool own = token && clean >> e & 1;
                    if (!own) clean &= ~(1 << e);
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&sh.q_full[e], (uint32_t)(NH * G * (own ? 1 : P) * 128));
                        for (int c = 0; c < NH; c++)
                            tma_load_3d(sQ + e * TILE + c * HALF, own ? &tmQ1 : &tmQ, &sh.q_full[e], c * 64, ch * G,
                                        pc.row0 + (q - pc.q0) * P);
                        q_sent = q + 1;
                    }
                    __syncwarp();
                }
                if (!ok) break;
            }
            if (*abort_flag && lane == 0) {  // copies in flight land before the shared memory goes away
                const uint64_t t0 = gtime_ns();
                for (int k = max(0, q_sent - 2); k < q_sent; k++)
                    while (!mbar_try(smem_u32(&sh.q_full[k & 1]), (uint32_t)(k >> 1) & 1u) && gtime_ns() - t0 < kTcuWaitCycles / 8) {
                    }
            }
        } else if (warp == 0) {
            // ---------------- K and V ----------------
            const int br = min(a.ps, kKeys), nbox = kKeys / br;
            const int box = lane / NH, half = lane % NH;
            // Keys that no other item of their sequence reads pass through L2 without pushing out what others use: 64 tokens over 3900..4250
            // positions 169 us, 174 without; one over 120001 86 us, 89, and behind an L2 full of written lines 96 and 105.
            // (Sequences whose pages are the same ones lose by it: 64 tokens over the same 4000 positions 129 us, 123 without.)
            uint64_t once;
            asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
            int r = 0;
            bool ok = true;
            for (int np = 0; ok; np++) {
                if (!warp_wait(&sh.w_full[np % kPieces], (uint32_t)(np / kPieces) & 1u, abort_flag, a.err)) break;
                const Piece &pc = sh.piece[np % kPieces];
                const int flags = pc.flags, blk0 = pc.blk0, nblk = pc.nblk, lo = pc.lo, hi = pc.hi, kvh = pc.kvh;
                const int *table = a.page_table + (size_t)pc.slot * a.max_pages;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.w_empty[np % kPieces]);
                if (flags & kEnd) break;
                auto page_row = [&](int j) -> int {  // first cache row of this lane's box; none outside what is seen
                    const int t = (blk0 + j) * kKeys + box * br;
                    if (j >= nblk || box >= nbox || t > hi || t + br <= lo) return -br;
                    const int pg = table[t >> a.log2_ps];
                    return (unsigned)pg < (unsigned)a.num_pages ? (pg * a.Hkv + kvh) * a.ps + (t & (a.ps - 1)) : -br;
                };
                int y = page_row(0);
                for (int j = 0; j < nblk; j++, r++) {
                    const int yn = page_row(j + 1);
                    const int st = r % NST;
                    const uint32_t ph = (uint32_t)(r / NST) & 1u;
#pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        uint64_t *full = kv ? &sh.v_full[st] : &sh.k_full[st];
                        ok = warp_wait(kv ? &sh.v_empty[st] : &sh.k_empty[st], ph ^ 1u, abort_flag, a.err);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(full, TILE);
                        __syncwarp();
                        if (box < nbox) {
                            uint8_t *to = (kv ? sV : sK) + st * TILE + half * HALF + box * br * 128;
                            if (flags & kOnce) tma_load_2d_hint(to, kv ? &tmV : &tmK, full, half * 64, y, once);
                            else tma_load_2d(to, kv ? &tmV : &tmK, full, half * 64, y);
                        }
                    }
                    if (!ok) break;
                    y = yn;
                }
            }
            if (*abort_flag) {  // copies in flight land before the shared memory goes away
                const uint64_t t0 = gtime_ns();
                for (int q = max(0, r - NST); q <= r; q++) {
                    const int k = q % NST;
                    while (!mbar_try(smem_u32(&sh.k_full[k]), (uint32_t)(q / NST) & 1u) && gtime_ns() - t0 < kTcuWaitCycles / 8) {
                    }
                    while (!mbar_try(smem_u32(&sh.v_full[k]), (uint32_t)(q / NST) & 1u) && gtime_ns() - t0 < kTcuWaitCycles / 8) {
                    }
                }
            }
        } else {
            // ---------------- MMAs: a warp per slot, so that one's waits and commits run beside the other's MMAs ----------------
            constexpr uint32_t IDS = tc_idesc_f16(kRows, kKeys, 0), IDP = tc_idesc_f16(kRows, D, 1);
            // Rows 0..15 of a product of 64 rows lie in the same TMEM lanes as of 128.  For a token's heads it takes as long, at
            // less power (64 tokens over 3900..4250 positions, under the power limit: 176 us, 184 with 128 rows).
            constexpr uint32_t IDS64 = tc_idesc_f16(64, kKeys, 0), IDP64 = tc_idesc_f16(64, D, 1);
            const int t = warp - 1;
            const uint32_t elect = lane == 0 ? 1u : 0u;
            const uint64_t dQ = desc_sw128(smem_u32(sQ), 16, 1024), dK = desc_sw128(smem_u32(sK), 16, 1024),
                           dV = desc_sw128(smem_u32(sV), HALF, 1024);
            const uint32_t ts = tmem + (uint32_t)(t * kKeys), to = tmem + 256u + (uint32_t)(t * 128);
            bool ok = true;
            int visits = 0;  // phase of p_full
            // A ring entry's barrier says something about use `phase` only after the use before has been released.
            auto filled = [&](uint64_t *empty, uint64_t *full, int phase) {
                return warp_wait(empty, ((uint32_t)phase & 1u) ^ 1u, abort_flag, a.err) &&
                       warp_wait(full, (uint32_t)phase & 1u, abort_flag, a.err);
            };
            // On the blocks of two tiles the slots take turns, slot 0 first: interleaved, the MMAs of both would take as long
            // together, and each slot's softmax would wait for the end of both (4096 rows over 20096 positions: 1204 us, and
            // 1021 with turns).  (A single tile's blocks are in both slots already, and bound by their loads.)
            int turns = 0;
            auto take_turn = [&]() {
                return warp_wait(&sh.turn[t], (uint32_t)(t == 0 ? turns + 1 : turns) & 1u, abort_flag, a.err);
            };
            auto end_turn = [&]() {
                if (lane == 0) mbar_arrive(&sh.turn[t ^ 1]);
                turns++;
            };
            for (int np = 0; ok; np++) {
                ok = warp_wait(&sh.w_full[np % kPieces], (uint32_t)(np / kPieces) & 1u, abort_flag, a.err);
                if (!ok) break;
                const Piece &pc = sh.piece[np % kPieces];
                const int flags = uni(pc.flags), nblk = uni(pc.nblk);
                const bool one = !(flags & kPair);
                const int j0 = one ? uni(pc.alt) ^ t : 0, step = one ? 2 : 1;  // the slot's first block
                const int q = uni(pc.q0) + (one ? 0 : t), qe = q & 1, clo = uni(pc.clo), chi = uni(pc.chi);
                int r = uni(pc.r0) + j0, k0 = (uni(pc.blk0) + j0) * kKeys;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.w_empty[np % kPieces]);
                if (flags & kEnd) break;
                if (j0 >= nblk) continue;
                // S = Q K^T of block j (ring index rs)
                auto issue_s = [&](int j, int rs) {
                    const int st = rs % NST;
                    const uint64_t da = dQ + (uint64_t)(qe * (TILE >> 4)), db = dK + (uint64_t)(st * (TILE >> 4));
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++) {
                        const uint64_t off = (uint64_t)(((kk >> 2) * HALF + (kk & 3) * 32) >> 4);
                        mma_ss(ts, da + off, db + off, flags & kLow ? IDS64 : IDS, kk > 0 ? 1u : 0u, elect);
                    }
                    commit(&sh.s_full[t], elect);  // also covers the slot's PV before it: O may be rescaled
                    // two arrivals release an entry: of both slots, where both use it
                    commit(&sh.k_empty[st], elect);
                    if (one) commit(&sh.k_empty[st], elect);
                    if (j + step >= nblk) {
                        commit(&sh.q_empty[qe], elect);
                        if (!one || nblk == 1) commit(&sh.q_empty[qe], elect);
                    }
                };
                ok = filled(&sh.q_empty[qe], &sh.q_full[qe], q >> 1) && filled(&sh.k_empty[r % NST], &sh.k_full[r % NST], r / NST);
                if (!ok) break;
                tc_fence_after();
                issue_s(j0, r);
                for (int j = j0; j < nblk; j += step, r += step, k0 += step * kKeys) {
                    const int st = r % NST, ph = r / NST, rn = r + step, sn = rn % NST, pn = rn / NST;
                    const bool last = j + step >= nblk;
                    ok = filled(&sh.v_empty[st], &sh.v_full[st], ph);
                    if (!ok) break;
                    if (chi < k0 + kKeys || clo > k0) {
                        // rows that no row of the sequence sees: P is 0 there, and V must be finite (both slots of a
                        // pair write the same zeros)
                        const int z0 = min(kKeys, max(0, clo - k0)) * 128, z1 = min(kKeys, max(0, chi - k0)) * 128;
#pragma unroll
                        for (int hf = 0; hf < NH; hf++) {
                            uint8_t *v = sV + st * TILE + hf * HALF;
                            for (int x = lane * 16; x < z0; x += 512) *reinterpret_cast<uint4 *>(v + x) = make_uint4(0, 0, 0, 0);
                            for (int x = z1 + lane * 16; x < HALF; x += 512) *reinterpret_cast<uint4 *>(v + x) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                    // the next block's keys, if they are there already: S then follows this PV at once
                    bool next = !last && mbar_test(&sh.k_empty[sn], ((uint32_t)pn & 1u) ^ 1u) && mbar_test(&sh.k_full[sn], (uint32_t)pn & 1u);
                    next = __all_sync(0xffffffffu, next);
                    ok = warp_wait(&sh.p_full[t], (uint32_t)visits++ & 1u, abort_flag, a.err) && (one || take_turn());
                    if (!ok) break;
                    tc_fence_after();
                    // O (+)= P V
                    const uint64_t dv = dV + (uint64_t)(st * (TILE >> 4));
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; kk++)  // P's halves lie over their own halves of S
                        mma_ts(to, ts + (uint32_t)((kk & 3) * 8 + (kk >> 2) * 64), dv + (uint64_t)(kk * 2048 >> 4), flags & kLow ? IDP64 : IDP,
                               kk > 0 ? 1u : (j > j0 ? 1u : 0u), elect);
                    if (next) issue_s(j + step, rn);
                    commit(&sh.v_empty[st], elect);
                    if (one) commit(&sh.v_empty[st], elect);
                    if (last) commit(&sh.o_full[t], elect);
                    if (!one) end_turn();
                    if (!last && !next) {
                        ok = filled(&sh.k_empty[sn], &sh.k_full[sn], pn);
                        if (!ok) break;
                        tc_fence_after();
                        issue_s(j + step, rn);
                    }
                }
            }
            // every MMA of this CTA has completed before the TMEM is freed
            commit(&sh.done[t], elect);
            const uint64_t t0 = gtime_ns();
            while (!mbar_try(smem_u32(&sh.done[t]), 0) && gtime_ns() - t0 < kTcuWaitCycles) {
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        // zeros for the rows that a single token's queries leave (before the first of them are fetched)
        for (int i = threadIdx.x - 128; i < 2 * TILE / 16; i += kSoftThreads) reinterpret_cast<uint4 *>(sQ)[i] = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.zeroed);
        // ---------------- softmax and results ----------------
        const int t = (warp - 4) >> 3, hf = lane >> 4, w0 = (warp & 3) * 32 + ((warp - 4) & 4) * 4, row = w0 + (lane & 15);
        const int rpos = row / G, rhead = row % G;
        const uint32_t trow = tmem + ((uint32_t)w0 << 16);
        const uint32_t ts = trow + (uint32_t)(t * kKeys), to = trow + 256u + (uint32_t)(t * 128);
        const bool wide = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)a.ld_out * 2) & 31) == 0;
        int nv = 0, no = 0, nx[2] = {0, 0};  // visits, pieces with visits, exchanges by writing slot
        bool ok = true;
        for (int np = 0; ok; np++) {
            ok = warp_wait(&sh.w_full[np % kPieces], (uint32_t)(np / kPieces) & 1u, abort_flag, a.err);
            if (!ok) break;
            const Piece &pc = sh.piece[np % kPieces];
            const int flags = pc.flags, nblk = pc.nblk, alt = pc.alt;
            const bool pair = flags & kPair, whole = flags & kWhole;
            const int tp = pair ? t * P : 0;                           // first position of the slot's tile in the item
            const int rows = (pair && t ? pc.n1 : pc.n0) * G;          // valid rows of the tile
            const int pos = pc.pos0 + tp + rpos;
            const int grow = pc.row0 + tp + rpos, head = pc.kvh * G + rhead;
            const int jj = pair ? 0 : alt ^ t, step = pair ? 1 : 2;    // the slot's first block of the piece
            int k0 = (pc.blk0 + jj) * kKeys;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.w_empty[np % kPieces]);
            if (flags & kEnd) break;
            const bool valid = row < rows, warp_on = w0 < rows;
            __nv_bfloat16 *orow = reinterpret_cast<__nv_bfloat16 *>(a.out) + (size_t)grow * a.ld_out + (size_t)head * D + hf * (D / 2);
            const int mine = (nblk - jj + step - 1) / step;
            // An item cut once is finished by the CTA in which it begins, at the end of its share, from the other's part:
            // that came first in the next share and has long been there.
            const bool two = flags & kTwo, closes = whole || (two && (flags & kHead));
            const bool exchange = closes && !pair && nblk > 1;
            const bool finish = closes && (!exchange || ((alt + nblk - 1) & 1) == t);  // the slot of the last block
            const bool few = !pair && rows <= kFewRows;
            const int which = flags & kHead ? 1 : 0, part = pair ? t : jj;
            unsigned *arrived2 = reinterpret_cast<unsigned *>(a.workspace) + kCounterWords + (flags & kHead ? cta : cta - 1);
            if (mine <= 0) {
                if (!closes) {
                    if (valid && hf == 0) __stcg(part_of<D>(a, cta, which, part).ml(row), make_float2(-INFINITY, 0.f));
                    if (two) {
                        __threadfence();
                        __syncwarp();
                        if (lane == 0) red_release(arrived2);
                    }
                }
                continue;
            }
            float m_use = -INFINITY, l = 0.f;  // running maximum (log2 units), sum of this half's probabilities
            for (int v = 0; v < mine; v++, nv++, k0 += step * kKeys) {
                ok = warp_wait(&sh.s_full[t], (uint32_t)nv & 1u, abort_flag, a.err);
                if (!ok) break;
                tc_fence_after();
                if (warp_on) {
                    float x[64];
                    ld32<64>(ts, x);
                    ld32<64>(ts + 32u, x + 32);
                    wait_ld();
                    const int hi = valid ? pos - k0 - hf * 64 : 64;
                    if (hi < 63) {
#pragma unroll
                        for (int e = 0; e < 64; e++)
                            if (e > hi) x[e] = -INFINITY;
                    }
                    if (a.window && valid && hi >= a.window) {
                        const int lo = hi - a.window;
#pragma unroll
                        for (int e = 0; e < 64; e++)
                            if (e <= lo) x[e] = -INFINITY;
                    }
                    // maximum of the raw scores (the scale is positive), with that of the row's other half
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 64; e += 2) m4[(e >> 1) & 3] = fmaxf(m4[(e >> 1) & 3], fmaxf(x[e], x[e + 1]));
                    float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)) * a.sl2;
                    float alpha = 1.f;
                    bool need = false;
                    if (v == 0) {
                        m_use = mx;
                    } else if (mx > m_use + kRescale) {
                        alpha = ex2(m_use - mx);
                        m_use = mx;
                        need = true;
                    }
                    // p = 2^(s scale log2 e - m); P goes to TMEM as packed bf16 pairs over the first half of this half's
                    // columns of S, and its sum is taken before that rounding.  P is rounded because the tensor cores take it in
                    // V's type: each p is off by 2^-8 of itself at most, and a result by as much of sum p |v| / sum p (relative
                    // L2 against 64 bits: 2.3e-3, and 1.7e-3 where only the result is rounded to bf16).  A second product with what
                    // the rounding leaves would double P V.
                    const float off = m_use == -INFINITY ? 0.f : -m_use;
                    const uint64_t off2 = f2(off, off), sl2 = f2(a.sl2, a.sl2);
                    uint64_t s2[2] = {0, 0};
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            float p0, p1;
                            unf2(fma2(f2(x[c * 32 + 2 * e], x[c * 32 + 2 * e + 1]), sl2, off2), p0, p1);
                            p0 = ex2(p0);
                            p1 = ex2(p1);
                            s2[e & 1] = add2(s2[e & 1], f2(p0, p1));
                            pk[e] = pack2(p0, p1);
                        }
                        st16<64>(ts + (uint32_t)(c * 16), pk);
                    }
                    float s0, s1;
                    unf2(add2(s2[0], s2[1]), s0, s1);
                    l = l * alpha + (s0 + s1);
                    // this half of O's columns (the slot's PV before has completed: s_full came after it)
                    if (__any_sync(0xffffffffu, need)) {
#pragma unroll 1
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t o[16];
                            ld16<D / 2>(to + (uint32_t)(c * 16), o);
                            wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            st16<D / 2>(to + (uint32_t)(c * 16), o);
                        }
                    }
                    wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t]);
            }
            if (!ok) break;
            ok = warp_wait(&sh.o_full[t], (uint32_t)no & 1u, abort_flag, a.err);
            if (!ok) break;
            no++;
            tc_fence_after();
            l += __shfl_xor_sync(0xffffffffu, l, 16);  // the row's sum, of both halves
            auto put_few = [&](int slot) {  // this half of O's columns of the valid rows
                float o[D / 2];
#pragma unroll
                for (int c = 0; c < D / 64; c++) ld32<D / 2>(to + (uint32_t)(c * 32), o + c * 32);
                wait_ld();
                if (valid) {
#pragma unroll
                    for (int c = 0; c < D / 8; c++)
                        sh.xo[slot][(hf * (D / 8) + c) * kFewRows + row] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
                }
                __syncwarp();
            };
            if (finish) {
                if (!exchange && whole) {
                    // the item's result
                    if (warp_on) {
                        const float inv = l == 0.f ? 0.f : 1.f / l;
                        float o[D / 2];
#pragma unroll
                        for (int c = 0; c < D / 64; c++) ld32<D / 2>(to + (uint32_t)(c * 32), o + c * 32);
                        wait_ld();
                        if (valid) {
#pragma unroll
                            for (int c = 0; c < D / 2; c += 16) {
                                uint32_t pk[8];
#pragma unroll
                                for (int e = 0; e < 8; e++) pk[e] = pack2(o[c + 2 * e] * inv, o[c + 2 * e + 1] * inv);
                                store32(orow + c, pk, wide);
                            }
                        }
                    }
                } else {
                    // joined with the other slot's (of a single-tile item) and the other CTA's parts
                    const Part<D> p0 = part_of<D>(a, cta, 2, t ^ 1), p1 = part_of<D>(a, cta + 1, 0, pair ? t : 0), p2 = part_of<D>(a, cta + 1, 0, 1);
                    if (few) {  // this slot's own O beside the other's
                        ok = warp_wait(&sh.x_empty[t], ((uint32_t)nx[t] & 1u) ^ 1u, abort_flag, a.err);
                        if (!ok) break;
                        if (warp_on) put_few(t);
                    }
                    if (exchange) {
                        ok = warp_wait(&sh.x_full[t ^ 1], (uint32_t)nx[t ^ 1] & 1u, abort_flag, a.err);
                        if (!ok) break;
                        nx[t ^ 1]++;
                    }
                    if (!whole) {
                        // all sixteen softmax warps of the other CTA
                        if (lane == 0) {
                            const uint64_t t0 = gtime_ns();
                            while (ld_acquire(arrived2) < 16u && !*abort_flag)
                                if (gtime_ns() - t0 > kTcuWaitCycles) {
                                    *abort_flag = 1;
                                    if (a.err) atomicExch(a.err, TC_DEVERR_TIMEOUT);
                                }
                            // the last of the item's finishing warps leaves the counter as it was
                            if (atomicAdd(arrived2, 0x100u) >> 8 == (pair ? 15u : 7u)) *arrived2 = 0u;
                        }
                        __syncwarp();
                    }
                    const float2 none = make_float2(-INFINITY, 0.f);
                    if (few) {
                        if (warp_on) {
                            // few rows: every lane takes one of them and some columns of it
                            const int r = lane & (kFewRows - 1), src = min(r, rows - 1);
                            const float2 own = make_float2(__shfl_sync(0xffffffffu, m_use, src), __shfl_sync(0xffffffffu, l, src));
                            const float2 o0 = exchange ? sh.xml[t ^ 1][src] : none, o1 = whole ? none : __ldcg(p1.ml(src)),
                                         o2 = whole ? none : __ldcg(p2.ml(src));
                            const float M = fmaxf(fmaxf(own.x, o0.x), fmaxf(o1.x, o2.x)), Mu = M == -INFINITY ? 0.f : M;
                            float wo = ex2(own.x - Mu), w0e = ex2(o0.x - Mu), w1 = ex2(o1.x - Mu), w2 = ex2(o2.x - Mu);
                            l = own.y * wo + o0.y * w0e + o1.y * w1 + o2.y * w2;
                            m_use = M;
                            const float inv = l == 0.f ? 0.f : 1.f / l;
                            wo *= inv; w0e *= inv; w1 *= inv; w2 *= inv;
                            const int rg = __shfl_sync(0xffffffffu, grow, src), rh = __shfl_sync(0xffffffffu, head, src);
                            __nv_bfloat16 *to_row = reinterpret_cast<__nv_bfloat16 *>(a.out) + (size_t)rg * a.ld_out + (size_t)rh * D;
#pragma unroll 1
                            for (int g = 0; g < D / 4; g += 16) {
                                float4 q[4][4];
#pragma unroll
                                for (int c = 0; c < 4; c++) {
                                    const int c4 = g + (lane >> 3) + 4 * c;
                                    const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                                    q[0][c] = sh.xo[t][c4 * kFewRows + src];
                                    q[1][c] = exchange ? sh.xo[t ^ 1][c4 * kFewRows + src] : z;
                                    // (a part of weight 0 saw nothing: its O may not have been written)
                                    q[2][c] = w1 != 0.f ? __ldcg(p1.o(c4, src)) : z;
                                    q[3][c] = w2 != 0.f ? __ldcg(p2.o(c4, src)) : z;
                                }
                                if (r < rows) {
#pragma unroll
                                    for (int c = 0; c < 4; c++) {
                                        const float4 o = make_float4(q[0][c].x * wo + q[1][c].x * w0e + q[2][c].x * w1 + q[3][c].x * w2,
                                                                     q[0][c].y * wo + q[1][c].y * w0e + q[2][c].y * w1 + q[3][c].y * w2,
                                                                     q[0][c].z * wo + q[1][c].z * w0e + q[2][c].z * w1 + q[3][c].z * w2,
                                                                     q[0][c].w * wo + q[1][c].w * w0e + q[2][c].w * w1 + q[3][c].w * w2);
                                        *reinterpret_cast<uint2 *>(to_row + (g + (lane >> 3) + 4 * c) * 4) = make_uint2(pack2(o.x, o.y), pack2(o.z, o.w));
                                    }
                                }
                            }
                        }
                    } else if (warp_on) {
                        const float2 o0 = valid && exchange ? __ldcg(p0.ml(row)) : none, o1 = valid && !whole ? __ldcg(p1.ml(row)) : none,
                                     o2 = valid && !whole && !pair ? __ldcg(p2.ml(row)) : none;
                        const float M = fmaxf(fmaxf(m_use, o0.x), fmaxf(o1.x, o2.x)), Mu = M == -INFINITY ? 0.f : M;
                        float wo = ex2(m_use - Mu), w0e = ex2(o0.x - Mu), w1 = ex2(o1.x - Mu), w2 = ex2(o2.x - Mu);
                        l = l * wo + o0.y * w0e + o1.y * w1 + o2.y * w2;
                        m_use = M;
                        const float inv = l == 0.f ? 0.f : 1.f / l;
                        wo *= inv; w0e *= inv; w1 *= inv; w2 *= inv;
#pragma unroll 1
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t u[16];
                            ld16<D / 2>(to + (uint32_t)(c * 16), u);
                            const int c4 = hf * (D / 8) + c * 4;
                            float4 q0[4], q1[4], q2[4];
                            // a part of weight 0 saw nothing (its O may not have been written)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                                q0[e] = w0e != 0.f ? __ldcg(p0.o(c4 + e, row)) : z;
                                q1[e] = w1 != 0.f ? __ldcg(p1.o(c4 + e, row)) : z;
                                q2[e] = w2 != 0.f ? __ldcg(p2.o(c4 + e, row)) : z;
                            }
                            wait_ld();
                            float o[16];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                o[4 * e] = __uint_as_float(u[4 * e]) * wo + q0[e].x * w0e + q1[e].x * w1 + q2[e].x * w2;
                                o[4 * e + 1] = __uint_as_float(u[4 * e + 1]) * wo + q0[e].y * w0e + q1[e].y * w1 + q2[e].y * w2;
                                o[4 * e + 2] = __uint_as_float(u[4 * e + 2]) * wo + q0[e].z * w0e + q1[e].z * w1 + q2[e].z * w2;
                                o[4 * e + 3] = __uint_as_float(u[4 * e + 3]) * wo + q0[e].w * w0e + q1[e].w * w1 + q2[e].w * w2;
                            }
                            if (valid) {
                                uint32_t pk[8];
#pragma unroll
                                for (int e = 0; e < 8; e++) pk[e] = pack2(o[2 * e], o[2 * e + 1]);
                                store32(orow + c * 16, pk, wide);
                            }
                        }
                    }
                }
                if (valid && hf == 0 && a.lse)
                    a.lse[(size_t)grow * a.H + head] = l == 0.f ? -INFINITY : (m_use + __log2f(l)) * 0.69314718055994531f;
                if (exchange) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.x_empty[t ^ 1]);
                }
            } else {
                // a partial result: for the other slot, or for the CTAs that share the item
                const Part<D> pp = part_of<D>(a, cta, closes ? 2 : which, closes ? t : part);
                if (closes) {
                    ok = warp_wait(&sh.x_empty[t], ((uint32_t)nx[t] & 1u) ^ 1u, abort_flag, a.err);
                    if (!ok) break;
                    nx[t]++;
                }
                if (warp_on && closes && few) {
                    put_few(t);
                    if (valid && hf == 0) sh.xml[t][row] = make_float2(m_use, l);
                } else if (warp_on) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t o[16];
                        ld16<D / 2>(to + (uint32_t)(c * 16), o);
                        wait_ld();
                        if (valid) {
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                *reinterpret_cast<uint4 *>(pp.o(hf * (D / 8) + c * 4 + e, row)) =
                                    make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                        }
                    }
                    if (valid && hf == 0) *pp.ml(row) = make_float2(m_use, l);
                }
                if (closes) {
                    __threadfence_block();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.x_full[t]);
                } else if (two) {
                    __threadfence();
                    __syncwarp();
                    if (lane == 0) red_release(arrived2);
                }
            }
        }
        if (sh.empty) {
            // rows of items whose every row stands before the first position
            for (int b = 0; b < a.batch; b++) {
                const Seq s = sh.seq[b];
                const int before = s.n - s.kv;
                if (before <= 0) continue;
                const int rows = s.kv == 0 ? s.n : before / (2 * P) * 2 * P;
                for (unsigned r = blockIdx.x; r < (unsigned)rows; r += gridDim.x) {
                    const size_t grow = (size_t)s.r0 + r;
                    uint4 *to_row = reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(a.out) + grow * a.ld_out);
                    for (int c = threadIdx.x - 128; c < a.H * (D / 8); c += kSoftThreads) to_row[c] = make_uint4(0, 0, 0, 0);
                    for (int h = threadIdx.x - 128; a.lse && h < a.H; h += kSoftThreads) a.lse[grow * a.H + h] = -INFINITY;
                }
            }
        }
        // ---- items in three pieces and more: every CTA joins a part of the rows once all pieces are there ----
        const int tid = threadIdx.x - 128;
        unsigned *arrived = reinterpret_cast<unsigned *>(a.workspace), *left = arrived + 2 * kCounterWords;
        bar_softmax();
        if (tid < 2 && sh.shared[tid].on) {
            __threadfence();
            red_release(arrived + sh.shared[tid].c0);
        }
        for (int k = 0; k < 2; k++) {
            const Shared m = sh.shared[k];
            if (!m.on) continue;
            const int me = cta - m.c0;
            const int lo = (int)((long long)m.rows * me / m.np), nr = (int)((long long)m.rows * (me + 1) / m.np) - lo;
            if (nr > 0) {
                if (tid == 0) {
                    const uint64_t t0 = gtime_ns();
                    bool there = !*abort_flag;
                    while (there && ld_acquire(arrived + m.c0) < (unsigned)m.np)
                        if (gtime_ns() - t0 > kTcuWaitCycles) {
                            there = false;
                            if (a.err) atomicExch(a.err, TC_DEVERR_TIMEOUT);
                        }
                    sh.go = there;
                }
                bar_softmax();
                if (sh.go) join_rows<D>(a, m, lo, nr, tid, reinterpret_cast<float *>(sQ));
                bar_softmax();
            }
            if (tid == 0 && atomicAdd(left + m.c0, 1u) == (unsigned)m.np - 1u) {
                arrived[m.c0] = 0u;  // the last to leave: ready for the next launch
                left[m.c0] = 0u;
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int D>
cudaError_t launch(const ChunkArgs &a, cudaStream_t st) {
    constexpr int smem = (2 + 2 * tc_stages(D)) * tc_tile_bytes(D) + 1024;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    static std::atomic<int> grids[64];  // CTAs of a launch on each device, once its kernel has been prepared
    int grid = grids[dev].load(std::memory_order_acquire);
    if (!grid) {
        e = cudaFuncSetAttribute(qw_chunk_attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        e = cudaDeviceGetAttribute(&grid, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        grid = grid < kNumSMsB200 ? grid : kNumSMsB200;
        grids[dev].store(grid, std::memory_order_release);
    }
    CUtensorMap mq, mq1, mk, mv;
    const int P = kRows / a.G, br = a.ps < kKeys ? a.ps : kKeys;
    const long long crow = (long long)a.num_pages * a.Hkv * a.ps;
    if ((e = tma_map_bf16_sw128_3d(&mq, a.q, a.d, a.H, a.rows, a.d, a.ld_q, a.G, P)) != cudaSuccess) return e;
    if ((e = tma_map_bf16_sw128_3d(&mq1, a.q, a.d, a.H, a.rows, a.d, a.ld_q, a.G, 1)) != cudaSuccess) return e;
    if ((e = tma_map_bf16_sw128(&mk, a.k, crow, a.d, a.d, br)) != cudaSuccess) return e;
    if ((e = tma_map_bf16_sw128(&mv, a.v, crow, a.d, a.d, br)) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeCooperative;  // CTAs that share an item wait for one another
    at[0].val.cooperative = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, qw_chunk_attn_tc_kernel<D>, mq, mq1, mk, mv, a);
}

}  // namespace

cudaError_t chunk_attn_tc_launch(const ChunkArgs &a, cudaStream_t st) {
    return a.d == 128 ? launch<128>(a, st) : launch<64>(a, st);
}

uint64_t chunk_attn_tc_most_units(const ChunkArgs &a) {
    const uint64_t step = 2 * (kRows / a.G), items = a.rows / step + a.batch, cap = (uint64_t)a.max_pages << a.log2_ps;
    const uint64_t seen = a.window && a.window + step < cap ? a.window + step : cap;
    return items * 2 * (seen / kKeys + 2 + kItemUnits) * a.Hkv;
}

size_t chunk_attn_tc_workspace(int head_dim) { return kChunkCounterBytes + (size_t)kNumSMsB200 * 6 * part_bytes(head_dim); }

}  // namespace qw
