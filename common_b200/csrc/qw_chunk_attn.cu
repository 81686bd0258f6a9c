// qw_chunk_attn.cu -- attention of a ragged batch of new tokens over the paged KV cache.
//
// Sequence b brings n_b = row_start[b + 1] - row_start[b] query rows and has kv_len[b] cached positions, those of the
// new rows included; its row i stands at position p = kv_len[b] - n_b + i and sees positions
// max(0, p - window + 1) .. p.  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q . k_j, m = max s_j, and
// lse = m + ln(sum): one pass over the keys with the running maximum and sum.  A row that sees nothing gives zeros and
// -infinity.  Lengths are read on the device, so a captured graph follows them.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <mutex>
#include <string>

#include "../../include/qwen3_b200.h"
#include "qw_chunk_attn.h"
#include "qw_internal.cuh"
#include "qw_ops.h"
#include "qw_tc.h"
#include "qw_tc_util.cuh"

namespace qw {
namespace {

constexpr int kSiRows = 64, kSiKeys = 64, kSiThreads = 256;

// One CTA per (64 rows of a sequence's (position, head of the group) list, KV head): q, K and V tiles in shared memory
// as fp32, a 4 x 4 block of scores and 4 x (D / 16) of the output per thread.
template <typename T, int D>
__global__ void __launch_bounds__(kSiThreads) qw_chunk_attn_simt_kernel(const ChunkArgs a) {
    extern __shared__ float si_smem[];
    constexpr int LD = D + 4;
    float *sq = si_smem, *sk = sq + kSiRows * LD, *sv = sk + kSiKeys * LD, *sp = sv + kSiKeys * LD;
    __shared__ float s_m[kSiRows], s_l[kSiRows], s_alpha[kSiRows];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int G = a.G, kvh = blockIdx.y;
    int b = 0, tile = blockIdx.x, n = 0;
    for (; b < a.batch; b++) {
        n = max(0, min(a.row_start[b + 1], a.rows) - max(a.row_start[b], 0));
        const int t = (n * G + kSiRows - 1) / kSiRows;
        if (tile < t) break;
        tile -= t;
    }
    if (b >= a.batch) return;
    const int r0 = a.row_start[b], kv = min(max(a.kv_len[b], 0), a.max_pages << a.log2_ps);
    const int p0 = kv - n, first = tile * kSiRows, last = min(first + kSiRows, n * G) - 1;
    const int *table = a.page_table + (size_t)(a.slots ? a.slots[b] : b) * a.max_pages;
    const T *q = reinterpret_cast<const T *>(a.q);
    const T *kc = reinterpret_cast<const T *>(a.k), *vc = reinterpret_cast<const T *>(a.v);
    for (int i = tid; i < kSiRows * D; i += kSiThreads) {
        const int r = i / D, c = i % D, pr = first + r;
        sq[r * LD + c] = pr <= last ? Elt<T>::load(q + (size_t)(r0 + pr / G) * a.ld_q + (size_t)(kvh * G + pr % G) * D + c) : 0.f;
    }
    if (tid < kSiRows) { s_m[tid] = -INFINITY; s_l[tid] = 0.f; }
    float o[4][D / 16] = {};
    const int lo = a.window ? max(0, p0 + first / G - a.window + 1) : 0;
    for (int k0 = lo / kSiKeys * kSiKeys; k0 <= p0 + last / G; k0 += kSiKeys) {
        __syncthreads();
        for (int i = tid; i < kSiKeys * D; i += kSiThreads) {
            const int r = i / D, c = i % D, pos = k0 + r;
            float kx = 0.f, vx = 0.f;  // nothing is read where no row of the tile sees anything
            if (pos >= lo && pos < kv) {
                const int pg = table[pos >> a.log2_ps];
                if ((unsigned)pg < (unsigned)a.num_pages) {
                    const size_t at = (((size_t)pg * a.Hkv + kvh) * a.ps + (pos & (a.ps - 1))) * D + c;
                    kx = Elt<T>::load(kc + at);
                    vx = Elt<T>::load(vc + at);
                }
            }
            sk[r * LD + c] = kx;
            sv[r * LD + c] = vx;
        }
        __syncthreads();
        float s[4][4] = {};
        for (int c = 0; c < D; c++) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[i][j] += sq[(ty * 4 + i) * LD + c] * sk[(tx + 16 * j) * LD + c];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int pos = p0 + (first + ty * 4 + i) / G;
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int key = k0 + tx + 16 * j;
                const bool sees = key <= pos && (!a.window || key > pos - a.window);
                s[i][j] = sees ? s[i][j] * a.sl2 : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float mo = s_m[ty * 4 + i], mn = fmaxf(mo, mx), mu = mn == -INFINITY ? 0.f : mn;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float p = exp2f(s[i][j] - mu);
                sum += p;
                sp[(ty * 4 + i) * (kSiKeys + 1) + tx + 16 * j] = p;
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            __syncwarp();
            if (tx == 0) {
                const float al = exp2f(mo - mu);
                s_alpha[ty * 4 + i] = al;
                s_l[ty * 4 + i] = s_l[ty * 4 + i] * al + sum;
                s_m[ty * 4 + i] = mn;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float al = s_alpha[ty * 4 + i];
#pragma unroll
            for (int c = 0; c < D / 16; c++) o[i][c] *= al;
        }
        for (int r = 0; r < kSiKeys; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = sp[(ty * 4 + i) * (kSiKeys + 1) + r];
#pragma unroll
                for (int c = 0; c < D / 16; c++) o[i][c] += p * sv[r * LD + tx + 16 * c];
            }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int pr = first + ty * 4 + i;
        if (pr > last) continue;
        const float l = s_l[ty * 4 + i], inv = l > 0.f ? 1.f / l : 0.f;
        const size_t row = (size_t)(r0 + pr / G), head = (size_t)(kvh * G + pr % G);
        T *out = reinterpret_cast<T *>(a.out) + row * a.ld_out + head * D;
#pragma unroll
        for (int c = 0; c < D / 16; c++) Elt<T>::store(out + tx + 16 * c, l == 0.f ? 0.f : o[i][c] * inv);
        if (a.lse && tx == 0)
            a.lse[row * a.H + head] = l > 0.f ? (s_m[ty * 4 + i] + log2f(l)) * 0.69314718055994531f : l == 0.f ? -INFINITY : l;
    }
}

template <typename T, int D>
cudaError_t simt_launch(const ChunkArgs &a, cudaStream_t st) {
    const int smem = (3 * kSiRows * (D + 4) + kSiRows * (kSiKeys + 1)) * (int)sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(qw_chunk_attn_simt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    // at most one tile more than the whole ones for every sequence
    const long long tiles = (long long)a.rows * a.G / kSiRows + a.batch;
    qw_chunk_attn_simt_kernel<T, D><<<dim3((unsigned)tiles, a.Hkv), kSiThreads, smem, st>>>(a);
    return cudaGetLastError();
}


// ---------------------------------------------------------------------------------------------------------------
// bf16: the tensor cores
// ---------------------------------------------------------------------------------------------------------------
// The G query heads of a KV head share its keys, so the rows of a query tile are (position, head of the group) pairs:
// P = floor(128 / G) positions of all G heads, at most 128 rows, one row per TMEM lane.  An item is two such tiles of
// one sequence and KV head; a K / V block of 128 keys serves both.  The key blocks of all items, in the order
// sequence, KV head, tiles, form one line that is cut into equal shares, one per CTA (one CTA per SM): every SM gets
// the same number of blocks whatever the lengths are.  An item cut by a share's end leaves partial results (O, maximum,
// sum) in the workspace, and the CTAs that share it join them, each a part of its rows, once all are there.
//
// An item with one tile only (decoding: G rows; the last rows of a chunk) gives its blocks to the two tile slots in
// turn, so that one slot's softmax still runs while the tensor cores work on the other; the slots' results are joined
// at the item's end.
//
// Warps (three warpgroups):
//   0     K and V: TMA boxes of min(page, 128) rows into rings of kStages tiles each, one lane per box
//   1     TMEM and the MMAs: S_t = Q_t K^T, then O_t += P_t V as soon as slot t's softmax has written P_t over S_t;
//         it also clears the rows of a V block that no row of the item sees (0 x NaN is NaN)
//   2     Q: one box of (64 columns, G heads, P positions) per 64 columns
//   4..7  softmax and result of slot 0, one row per thread; 8..11 of slot 1
// Every wait is bounded; one that runs out sets the error word and ends the CTA (its copies landed, its TMEM freed).

constexpr int kTcThreads = 384, kTcRows = 128, kTcKeys = 128;
constexpr float kTcRescale = 8.f;  // the running maximum is raised only when it grows by more than 2^8: p stays below 2^8
constexpr int kPartRows = 128;
constexpr int kMinShare = 3;       // a CTA's least share of the line

__host__ __device__ constexpr int tc_stages(int d) { return d == 128 ? 2 : 5; }
__host__ __device__ constexpr int tc_tile_bytes(int d) { return kTcRows * d * 2; }
__host__ __device__ constexpr size_t part_bytes(int d) { return (size_t)kPartRows * d * 4 + kPartRows * 8; }
constexpr size_t kCounterBytes = 2 * 1024;  // arrivals | departures, one word per CTA each
static_assert(kNumSMsB200 * 4 <= 1024, "counter words");

struct Seq {
    int n, kv, r0;  // new rows, cached positions, first row
};

// an item that several CTAs share
struct Shared {
    long long u0;          // its place on the line
    int on, nb, nsub, rows0, rows1, row, head;
};

struct __align__(16) TcShared {
    long long pre[kChunkMaxBatch + 1];  // units of the line before each sequence
    Seq seq[kChunkMaxBatch];
    uint64_t k_full[5], k_empty[5], v_full[5], v_empty[5], q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2],
        x_full[2], x_empty[2], done;
    Shared shared[2];
    uint32_t tmem;
    int abort, go;
    int start_b, start_h, start_i, start_off;  // where this CTA's share begins
};

// one item's rows and keys
struct Item {
    int nsub;        // tiles
    int f;           // first new row of the sequence that the item covers (rows of one head)
    int pf, pl;      // positions of its first and last row
    int klo;         // first position that one of its rows sees
    int j0, nb;      // key blocks j0 .. j0 + nb - 1; none when no row sees anything
};

__device__ __forceinline__ Item make_item(const Seq &s, int i, int P, int window) {
    Item it;
    it.f = i * 2 * P;
    const int l = min(s.n, it.f + 2 * P) - 1, p0 = s.kv - s.n;
    it.nsub = s.n - it.f > P ? 2 : 1;
    it.pf = p0 + it.f;
    it.pl = p0 + l;
    it.klo = window ? max(0, it.pf - window + 1) : 0;
    it.j0 = it.klo / kTcKeys;
    it.nb = it.pl < 0 ? 0 : it.pl / kTcKeys - it.j0 + 1;
    return it;
}

// The pieces of items that make up a CTA's share, in order.  An item costs its blocks and one unit more.
struct Walk {
    int b, h, i, off;
    long long at, end;  // position on the line
    // the current piece
    Item it;
    Seq s;
    int cb, ch;       // its sequence and KV head
    int ja, jb;       // its blocks, relative to it.j0
    long long u0;     // line position of its item

    __device__ __forceinline__ void init(const TcShared &sh, long long a, long long e) {
        b = sh.start_b; h = sh.start_h; i = sh.start_i; off = sh.start_off;
        at = a; end = e;
    }
    __device__ __forceinline__ bool next(const TcShared &sh, const ChunkArgs &a, int P) {
        while (at < end) {
            s = sh.seq[b];
            if (s.n <= 0) { b++; continue; }
            it = make_item(s, i, P, a.window);
            const int units = it.nb + 1;
            const int take = (int)min((long long)(units - off), end - at);
            ja = min(off, it.nb);
            jb = min(off + take, it.nb);
            cb = b; ch = h;
            u0 = at - off;
            at += take;
            off += take;
            if (off == units) {
                off = 0;
                if ((++i) * 2 * P >= s.n) {
                    i = 0;
                    if (++h == a.Hkv) { h = 0; b++; }
                }
            }
            if (ja < jb || it.nb == 0) return true;
        }
        return false;
    }
    __device__ __forceinline__ bool whole() const { return ja == 0 && jb == it.nb; }
};

__device__ __forceinline__ long long share_start(long long c, long long W, int Ge) { return c * W / Ge; }
// the CTA whose share holds line position u
__device__ __forceinline__ int share_owner(long long u, long long W, int Ge) { return (int)(((u + 1) * Ge + W - 1) / W) - 1; }

// K-major or MN-major 128-byte-swizzled operand descriptor; lbo / sbo in bytes
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
           (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// tcgen05.mma with the A operand (P) in tensor memory: two bf16 per 32-bit column along K
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(smem_u32(dst)),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void bar_softmax() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ unsigned ld_acquire(const unsigned *p) {
    unsigned v;
    asm volatile("ld.acquire.gpu.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void red_release(unsigned *p) {
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory");
}

// A partial result: O as float4 columns [D / 4][128 rows], then (maximum in log2 units, sum) per row.
template <int D>
struct Part {
    char *p;
    __device__ __forceinline__ float4 *o(int c4, int row) const { return reinterpret_cast<float4 *>(p) + c4 * kPartRows + row; }
    __device__ __forceinline__ float2 *ml(int row) const {
        return reinterpret_cast<float2 *>(p + (size_t)kPartRows * D * 4) + row;
    }
};
// which: 0 the share's first piece, 1 its last, 2 the exchange between the slots
template <int D>
__device__ __forceinline__ Part<D> part_of(const ChunkArgs &a, int cta, int which, int k) {
    return Part<D>{(char *)a.workspace + kCounterBytes + ((size_t)cta * 6 + which * 2 + k) * part_bytes(D)};
}

// Rows [lo, lo + nr) of an item in np pieces: sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p, m = max m_p, in one pass
// over the pieces.  A thread takes 4 columns of a row; with few rows several threads share the pieces.
template <int D>
__device__ __forceinline__ void join_rows(const ChunkArgs &a, const Shared &m, int c0, int np, int lo, int nr, int tid,
                                          float *red) {
    const int E = nr * (D / 4), ng = max(1, 256 / E), nparts = m.nsub == 2 ? np : 2 * np;
    for (int e0 = 0; e0 < E; e0 += 256) {
        const int g = E < 256 ? tid / E : 0, e = E < 256 ? tid % E : e0 + tid;
        const bool on = g < ng && e < E;
        const int r = lo + e % nr, c4 = e / nr;
        const int tile = r >= m.rows0, row = r - (tile ? m.rows0 : 0);
        float M = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on) {
#pragma unroll 4
            for (int p = g; p < nparts; p += ng) {
                const int k = m.nsub == 2 ? p : p >> 1;
                const Part<D> px = part_of<D>(a, c0 + k, k == 0 ? 1 : 0, m.nsub == 2 ? tile : p & 1);
                const float2 ml = __ldcg(px.ml(row));
                const float4 x = __ldcg(px.o(c4, row));
                if (ml.x == -INFINITY) continue;  // nothing seen there (O may not have been written)
                const float mn = fmaxf(M, ml.x), wo = ex2(M - mn), wx = ex2(ml.x - mn);
                o.x = o.x * wo + x.x * wx; o.y = o.y * wo + x.y * wx;
                o.z = o.z * wo + x.z * wx; o.w = o.w * wo + x.w * wx;
                l = l * wo + ml.y * wx;
                M = mn;
            }
        }
        if (ng > 1) {  // E < 256: one round
            float *mine = red + tid * 8;
            if (on) { mine[0] = M; mine[1] = l; mine[2] = o.x; mine[3] = o.y; mine[4] = o.z; mine[5] = o.w; }
            bar_softmax();
            if (on && g == 0)
                for (int h = 1; h < ng; h++) {
                    const float *x = red + (h * E + e) * 8;
                    if (x[0] == -INFINITY) continue;
                    const float mn = fmaxf(M, x[0]), wo = ex2(M - mn), wx = ex2(x[0] - mn);
                    o.x = o.x * wo + x[2] * wx; o.y = o.y * wo + x[3] * wx;
                    o.z = o.z * wo + x[4] * wx; o.w = o.w * wo + x[5] * wx;
                    l = l * wo + x[1] * wx;
                    M = mn;
                }
        }
        if (on && g == 0) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const size_t grow = (size_t)(m.row + r / a.G);
            const int head = m.head + r % a.G;
            *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(a.out) + grow * a.ld_out + (size_t)head * D + c4 * 4) =
                make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
            if (c4 == 0 && a.lse) a.lse[grow * a.H + head] = l == 0.f ? -INFINITY : (M + __log2f(l)) * 0.69314718055994531f;
        }
    }
}

// a bounded wait that ends the same way for every lane of the warp
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity, volatile int *abort_flag, int *err) {
    return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, err));
}

template <int D>
__global__ void __launch_bounds__(kTcThreads, 1)
    qw_chunk_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmV, const ChunkArgs a) {
    constexpr int NST = tc_stages(D), TILE = tc_tile_bytes(D), HALF = kTcRows * 128, NH = D / 64;
    extern __shared__ uint8_t tc_smem_raw[];
    __shared__ TcShared sh;
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tc_smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sQ = sm, *sK = sm + 2 * TILE, *sV = sK + NST * TILE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort_flag = &sh.abort;
    const int G = a.G, P = kTcRows / G;

    // ---- the line: units of every sequence, their running sum, and where this CTA's share begins ----
    for (int b = warp; b < a.batch; b += kTcThreads / 32) {
        const int r0 = a.row_start[b], r1 = a.row_start[b + 1], kv = a.kv_len[b];
        Seq s;
        s.r0 = min(max(r0, 0), a.rows);
        s.n = max(0, min(r1, a.rows) - s.r0);
        s.kv = min(max(kv, 0), a.max_pages << a.log2_ps);
        const int items = (s.n + 2 * P - 1) / (2 * P);
        long long units = 0;
        for (int i = lane; i < items; i += 32) units += make_item(s, i, P, a.window).nb + 1;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
        if (lane == 0) {
            sh.seq[b] = s;
            sh.pre[b + 1] = units * a.Hkv;
        }
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < NST; i++) {
            mbar_init(&sh.k_full[i], 1);
            mbar_init(&sh.k_empty[i], 2);
            mbar_init(&sh.v_full[i], 1);
            mbar_init(&sh.v_empty[i], 2);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.q_empty[i], 2);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.x_full[i], 4);
            mbar_init(&sh.x_empty[i], 4);
        }
        mbar_init(&sh.done, 1);
        sh.abort = 0;
        sh.shared[0].on = sh.shared[1].on = 0;
        sh.pre[0] = 0;
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
    if (warp == 0) {
        long long run = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 32) {
            const int b = b0 + lane;
            long long v = b < a.batch ? sh.pre[b + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long w = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += w;
            }
            if (b < a.batch) sh.pre[b + 1] = run + v;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
        __syncwarp();
        const long long W = sh.pre[a.batch];
        const int Ge = (int)min((long long)gridDim.x, (W + kMinShare - 1) / kMinShare);
        if ((int)blockIdx.x < Ge) {
            const long long u = share_start(blockIdx.x, W, Ge);
            int lo = 0, hi = a.batch - 1;  // the last sequence that begins at or before u
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (sh.pre[mid] <= u) lo = mid;
                else hi = mid - 1;
            }
            const long long per = (sh.pre[lo + 1] - sh.pre[lo]) / a.Hkv;
            long long rem = u - sh.pre[lo];
            const int h = (int)(rem / per);
            rem -= h * per;
            const Seq s = sh.seq[lo];
            int i0 = 0;
            for (;;) {  // the item that holds unit rem of this head
                long long v = (i0 + lane) * 2 * P < s.n ? make_item(s, i0 + lane, P, a.window).nb + 1 : 0;
                const long long mine = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long w = __shfl_up_sync(0xffffffffu, v, o);
                    if (lane >= o) v += w;
                }
                const unsigned m = __ballot_sync(0xffffffffu, v > rem);
                if (m) {
                    const int k = __ffs(m) - 1;
                    if (lane == k) {
                        sh.start_b = lo; sh.start_h = h; sh.start_i = i0 + k; sh.start_off = (int)(rem - (v - mine));
                    }
                    break;
                }
                rem -= __shfl_sync(0xffffffffu, v, 31);
                i0 += 32;
            }
        }
    }
    __syncthreads();
    const uint32_t tmem = sh.tmem;
    const long long W = sh.pre[a.batch];
    const int Ge = (int)min((long long)gridDim.x, (W + kMinShare - 1) / kMinShare);
    const int cta = blockIdx.x;
    const bool busy = cta < Ge;
    const long long u_begin = busy ? share_start(cta, W, Ge) : 0, u_end = busy ? share_start(cta + 1, W, Ge) : 0;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp == 0) {
            // ---------------- K and V ----------------
            Walk w;
            w.init(sh, u_begin, u_end);
            const int br = min(a.ps, kTcKeys), nbox = kTcKeys / br;
            const int box = lane / NH, half = lane % NH;
            int r = 0;
            bool ok = true;
            while (ok && w.next(sh, a, P)) {
                const int *table = a.page_table + (size_t)(a.slots ? a.slots[w.cb] : w.cb) * a.max_pages;
                auto page_row = [&](int j) -> int {  // first cache row of this lane's box; none outside what is seen
                    const int t = (w.it.j0 + j) * kTcKeys + box * br;
                    if (j >= w.jb || box >= nbox || t > w.it.pl || t + br <= w.it.klo) return -br;
                    const int pg = table[t >> a.log2_ps];
                    return (unsigned)pg < (unsigned)a.num_pages ? (pg * a.Hkv + w.ch) * a.ps + (t & (a.ps - 1)) : -br;
                };
                int y = page_row(w.ja);
                for (int j = w.ja; j < w.jb && ok; j++, r++) {
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
                        if (box < nbox)
                            tma_load_2d((kv ? sV : sK) + st * TILE + half * HALF + box * br * 128, kv ? &tmV : &tmK, full,
                                        half * 64, y);
                    }
                    y = yn;
                }
            }
            // copies in flight land before the shared memory goes away (at a normal end the MMAs have waited for all)
            if (!ok) {
                const uint64_t t0 = gtime_ns();
                for (int k = 0; k < NST; k++)
                    for (int q = max(0, r - NST); q <= r; q++)
                        if (q % NST == k) {
                            while (!mbar_try(smem_u32(&sh.k_full[k]), (uint32_t)(q / NST) & 1u) && gtime_ns() - t0 < kTcuWaitCycles / 8) {
                            }
                            while (!mbar_try(smem_u32(&sh.v_full[k]), (uint32_t)(q / NST) & 1u) && gtime_ns() - t0 < kTcuWaitCycles / 8) {
                            }
                        }
            }
        } else if (warp == 1) {
            // ---------------- MMAs ----------------
            constexpr uint32_t IDS = tc_idesc_f16(kTcRows, kTcKeys, 0), IDP = tc_idesc_f16(kTcRows, D, 1);
            struct Slot {
                Walk w;
                bool live;   // has a current visit
                int r0;      // ring index of the piece's first block
                int q;       // Q entry of its tile
                int qn;      // Q entries of the pieces so far
                int alt;     // blocks of single-tile pieces so far
                int rn;      // blocks so far
                int j, step; // current block and stride
                int done_s, done_p;  // visits whose S / PV have been issued in all (barrier phases)
                int np;      // pieces
            };
            Slot sl[2];
            auto next_piece = [&](Slot &s, int t) {
                s.live = false;
                while (s.w.next(sh, a, P)) {
                    const int nblk = s.w.jb - s.w.ja;
                    if (nblk == 0) continue;
                    s.r0 = s.rn;
                    s.rn += nblk;
                    if (s.w.it.nsub == 2) {
                        s.q = s.qn + t;
                        s.qn += 2;
                        s.j = s.w.ja;
                        s.step = 1;
                    } else {
                        s.q = s.qn++;
                        s.j = s.w.ja + ((s.alt & 1) == t ? 0 : 1);
                        s.alt += nblk;
                        s.step = 2;
                    }
                    if (s.j < s.w.jb) { s.live = true; return; }
                }
            };
            bool ok = true;
            for (int t = 0; t < 2; t++) {
                Slot &s = sl[t];
                s.w.init(sh, u_begin, u_end);
                s.qn = s.alt = s.rn = s.done_s = s.done_p = s.np = 0;
                next_piece(s, t);
            }
            // S_t = Q_t K^T of the slot's current visit into TMEM columns [128 t, 128 t + 128)
            auto issue_s = [&](Slot &s, int t) -> bool {
                const int r = s.r0 + s.j - s.w.ja, st = r % NST;
                if (!warp_wait(&sh.q_full[s.q & 1], (uint32_t)(s.q >> 1) & 1u, abort_flag, a.err)) return false;
                if (!warp_wait(&sh.k_full[st], (uint32_t)(r / NST) & 1u, abort_flag, a.err)) return false;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t qa = smem_u32(sQ + (s.q & 1) * TILE), ka = smem_u32(sK + st * TILE);
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++) {
                        const uint32_t off = (uint32_t)((kk >> 2) * HALF + (kk & 3) * 32);
                        tc_mma(tmem + (uint32_t)(t * kTcKeys), desc_sw128(qa + off, 16, 1024), desc_sw128(ka + off, 16, 1024),
                               IDS, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(&sh.s_full[t]);  // also covers the slot's PV before it: O_t may be rescaled
                    const bool both = s.w.it.nsub == 2 || s.w.jb - s.w.ja > 1;  // the other slot visits this piece too
                    tc_commit(&sh.k_empty[st]);
                    if (s.w.it.nsub == 1) tc_commit(&sh.k_empty[st]);
                    if (s.j + s.step >= s.w.jb) {
                        tc_commit(&sh.q_empty[s.q & 1]);
                        if (s.w.it.nsub == 2 || !both) tc_commit(&sh.q_empty[s.q & 1]);
                    }
                }
                __syncwarp();
                return true;
            };
            // O_t (+)= P_t V of the slot's current visit
            auto issue_pv = [&](Slot &s, int t) -> bool {
                const int r = s.r0 + s.j - s.w.ja, st = r % NST;
                if (!warp_wait(&sh.v_full[st], (uint32_t)(r / NST) & 1u, abort_flag, a.err)) return false;
                const int k0 = (s.w.it.j0 + s.j) * kTcKeys;
                const int lo = max(0, s.w.it.klo - k0), hi = min(kTcKeys, s.w.it.pl + 1 - k0);
                if (lo > 0 || hi < kTcKeys) {
                    // rows that no row of the item sees: whatever the cache holds there, P is 0 and V must be finite
                    // (both slots of a pair write the same zeros; the first has committed nothing that reads them yet
                    // or has already cleared them)
                    for (int e = lane; e < kTcKeys * 8 * NH; e += 32) {
                        const int row = (e >> 3) & (kTcKeys - 1), hf = e >> 10;
                        if (row < lo || row >= hi)
                            *reinterpret_cast<uint4 *>(sV + st * TILE + hf * HALF + row * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (!warp_wait(&sh.p_full[t], (uint32_t)s.done_p & 1u, abort_flag, a.err)) return false;
                s.done_p++;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t va = smem_u32(sV + st * TILE);
                    const int first = (s.w.it.nsub == 2 ? s.w.ja : s.w.ja + ((s.j - s.w.ja) & 1));
#pragma unroll
                    for (int kk = 0; kk < kTcKeys / 16; kk++)
                        mma_ts(tmem + 256u + (uint32_t)(t * 128), tmem + (uint32_t)(t * kTcKeys + kk * 8),
                               desc_sw128(va + (uint32_t)(kk * 2048), HALF, 1024), IDP, (s.j > first || kk > 0) ? 1u : 0u);
                    tc_commit(&sh.v_empty[st]);
                    if (s.w.it.nsub == 1) tc_commit(&sh.v_empty[st]);
                    if (s.j + s.step >= s.w.jb) tc_commit(&sh.o_full[t]);
                }
                __syncwarp();
                return true;
            };
            for (int t = 0; t < 2 && ok; t++)
                if (sl[t].live) ok = issue_s(sl[t], t);
            while (ok && (sl[0].live || sl[1].live)) {
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    Slot &s = sl[t];
                    if (!ok || !s.live) continue;
                    ok = issue_pv(s, t);
                    s.j += s.step;
                    if (s.j >= s.w.jb) next_piece(s, t);
                    if (ok && s.live) ok = issue_s(s, t);
                }
            }
            // every MMA of this CTA has completed before the TMEM is freed
            if (lane == 0) tc_commit(&sh.done);
            const uint64_t t0 = gtime_ns();
            while (!mbar_try(smem_u32(&sh.done), 0) && gtime_ns() - t0 < kTcuWaitCycles) {
            }
        } else if (warp == 2) {
            // ---------------- Q ----------------
            Walk w;
            w.init(sh, u_begin, u_end);
            int q = 0;
            bool ok = true;
            if (lane == 0) {
                while (ok && w.next(sh, a, P)) {
                    if (w.ja == w.jb) continue;
                    for (int t = 0; t < w.it.nsub && ok; t++, q++) {
                        const int e = q & 1;
                        ok = mbar_wait(&sh.q_empty[e], ((uint32_t)(q >> 1) & 1u) ^ 1u, abort_flag, a.err);
                        if (!ok) break;
                        mbar_arrive_expect_tx(&sh.q_full[e], (uint32_t)(NH * G * P * 128));
                        for (int c = 0; c < NH; c++)
                            tma_load_3d(sQ + e * TILE + c * HALF, &tmQ, &sh.q_full[e], c * 64, w.ch * G, w.s.r0 + w.it.f + t * P);
                    }
                }
                if (!ok) {
                    const uint64_t t0 = gtime_ns();
                    for (int k = max(0, q - 2); k < q; k++)
                        while (!mbar_try(smem_u32(&sh.q_full[k & 1]), (uint32_t)(k >> 1) & 1u) && gtime_ns() - t0 < kTcuWaitCycles / 8) {
                        }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---------------- softmax and results ----------------
        const int t = (warp - 4) >> 2, qq = warp & 3, row = qq * 32 + lane;
        const uint32_t trow = tmem + ((uint32_t)(qq * 32) << 16);
        const uint32_t ts = trow + (uint32_t)(t * kTcKeys), to = trow + 256u + (uint32_t)(t * 128);
        Walk w;
        w.init(sh, u_begin, u_end);
        int nv = 0, no = 0, alt = 0, nx[2] = {0, 0};  // visits, pieces with visits, single-tile blocks, exchanges by writer
        bool ok = true;
        while (ok && w.next(sh, a, P)) {
            const bool pair = w.it.nsub == 2;
            const int tile = pair ? t : 0;
            const int nblk = w.jb - w.ja;
            const int rows = min(P, w.s.n - w.it.f - tile * P) * G;  // valid rows of the tile
            const bool valid = row < rows;
            const bool warp_on = qq * 32 < rows;
            const int prow = w.it.f + tile * P + row / G;  // the row within the sequence's new rows
            const int pos = w.s.kv - w.s.n + prow;
            const size_t grow = (size_t)(w.s.r0 + prow);
            const int head = w.ch * G + row % G;
            __nv_bfloat16 *orow = reinterpret_cast<__nv_bfloat16 *>(a.out) + grow * a.ld_out + (size_t)head * D;
            float *lse = a.lse ? a.lse + grow * a.H + head : nullptr;
            if (nblk == 0) {  // the item's rows see nothing
                if (t < w.it.nsub && valid) {
#pragma unroll
                    for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4 *>(orow + c) = make_uint4(0, 0, 0, 0);
                    if (lse) *lse = -INFINITY;
                }
                continue;
            }
            const bool whole = w.whole();
            if (!whole && threadIdx.x == 128) {  // one of the (at most two) items that this CTA shares with others
                Shared &m = sh.shared[w.ja == 0 ? 1 : 0];
                m.on = 1; m.u0 = w.u0; m.nb = w.it.nb; m.nsub = w.it.nsub; m.rows0 = min(P, w.s.n - w.it.f) * G;
                m.rows1 = pair ? min(P, w.s.n - w.it.f - P) * G : 0;
                m.row = w.s.r0 + w.it.f; m.head = w.ch * G;
            }
            int jj = 0, step = 1, slot_of_last = t, mine = nblk;
            if (!pair) {
                jj = (alt & 1) == t ? 0 : 1;
                step = 2;
                slot_of_last = (alt + nblk - 1) & 1;
                alt += nblk;
                mine = (nblk - jj + 1) / 2;
            }
            const bool exchange = whole && !pair && nblk > 1;
            const int part = pair ? t : jj;
            if (mine <= 0) {
                if (!whole && valid) __stcg(part_of<D>(a, cta, w.ja == 0 ? 1 : 0, part).ml(row), make_float2(-INFINITY, 0.f));
                continue;
            }
            float m_use = -INFINITY, l = 0.f;
            for (int v = 0; v < mine && ok; v++, nv++, jj += step) {
                if (!warp_wait(&sh.s_full[t], (uint32_t)nv & 1u, abort_flag, a.err)) { ok = false; break; }
                tc_fence_after();
                if (warp_on) {
                    float x[kTcKeys];
#pragma unroll
                    for (int c = 0; c < 4; c++) tmem_ld32(ts + (uint32_t)(c * 32), x + c * 32);
                    tmem_wait_ld();
                    const int k0 = (w.it.j0 + w.ja + jj) * kTcKeys;
                    const int hi = valid ? pos - k0 : kTcKeys, lo = valid && a.window ? pos - a.window + 1 - k0 : 0;
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (__any_sync(0xffffffffu, hi < kTcKeys - 1 || lo > 0)) {
#pragma unroll
                        for (int e = 0; e < kTcKeys; e++)
                            if (e > hi || e < lo) x[e] = -INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < kTcKeys; e++) m4[e & 3] = fmaxf(m4[e & 3], x[e]);
                    const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.sl2;
                    float alpha = 1.f;
                    bool need = false;
                    if (v == 0) {
                        m_use = mx;
                    } else if (mx > m_use + kTcRescale) {
                        alpha = ex2(m_use - mx);
                        m_use = mx;
                        need = true;
                    }
                    const float off = m_use == -INFINITY ? 0.f : m_use;
                    float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float p0 = ex2(fmaf(x[c * 32 + e], a.sl2, -off)), p1 = ex2(fmaf(x[c * 32 + e + 1], a.sl2, -off));
                            s4[(e >> 1) & 3] += p0 + p1;
                            pk[e / 2] = pack2(p0, p1);
                        }
                        tmem_st16(ts + (uint32_t)(c * 16), pk);
                    }
                    l = l * alpha + ((s4[0] + s4[1]) + (s4[2] + s4[3]));
                    if (v > 0 && __any_sync(0xffffffffu, need)) {
#pragma unroll
                        for (int c = 0; c < D / 16; c++) {
                            uint32_t o[16];
                            asm volatile(
                                "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                                : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]),
                                  "=r"(o[7]), "=r"(o[8]), "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]),
                                  "=r"(o[14]), "=r"(o[15])
                                : "r"(to + (uint32_t)(c * 16)));
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            tmem_st16(to + (uint32_t)(c * 16), o);
                        }
                    }
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t]);
            }
            if (!ok) break;
            if (!warp_wait(&sh.o_full[t], (uint32_t)no & 1u, abort_flag, a.err)) { ok = false; break; }
            no++;
            tc_fence_after();
            if (whole && (!exchange || slot_of_last == t)) {
                // the item's result; of a single-tile item, joined with the other slot's
                float wo = 1.f, wx = 0.f;
                Part<D> px = part_of<D>(a, cta, 2, t ^ 1);
                if (exchange) {
                    if (!warp_wait(&sh.x_full[t ^ 1], (uint32_t)nx[t ^ 1] & 1u, abort_flag, a.err)) { ok = false; break; }
                    nx[t ^ 1]++;
                    if (valid) {
                        const float2 o = __ldcg(px.ml(row));
                        const float M = fmaxf(m_use, o.x);
                        wo = M == -INFINITY ? 0.f : ex2(m_use - M);
                        wx = M == -INFINITY ? 0.f : ex2(o.x - M);
                        l = l * wo + o.y * wx;
                        m_use = M;
                    }
                }
                if (warp_on) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    const float io = wo * inv, ix = wx * inv;
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        float o[32];
                        tmem_ld32(to + (uint32_t)(c * 32), o);
                        tmem_wait_ld();
                        if (valid) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (exchange) z = __ldcg(px.o((c * 32 + e) / 4, row));
                                o[e] = fmaf(z.x, ix, o[e] * io);
                                o[e + 1] = fmaf(z.y, ix, o[e + 1] * io);
                                o[e + 2] = fmaf(z.z, ix, o[e + 2] * io);
                                o[e + 3] = fmaf(z.w, ix, o[e + 3] * io);
                            }
#pragma unroll
                            for (int e = 0; e < 32; e += 8)
                                *reinterpret_cast<uint4 *>(orow + c * 32 + e) =
                                    make_uint4(pack2(o[e], o[e + 1]), pack2(o[e + 2], o[e + 3]), pack2(o[e + 4], o[e + 5]),
                                               pack2(o[e + 6], o[e + 7]));
                        }
                    }
                    if (valid && lse) *lse = l == 0.f ? -INFINITY : (m_use + __log2f(l)) * 0.69314718055994531f;
                }
                if (exchange) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.x_empty[t ^ 1]);
                }
            } else {
                // a partial result: for the other slot, or for the CTAs that share the item
                Part<D> pp = part_of<D>(a, cta, whole ? 2 : w.ja == 0 ? 1 : 0, whole ? t : part);
                if (whole) {
                    if (!warp_wait(&sh.x_empty[t], ((uint32_t)nx[t] & 1u) ^ 1u, abort_flag, a.err)) { ok = false; break; }
                    nx[t]++;
                }
                if (warp_on) {
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        float o[32];
                        tmem_ld32(to + (uint32_t)(c * 32), o);
                        tmem_wait_ld();
                        if (valid) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                __stcg(pp.o((c * 32 + e) / 4, row), make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]));
                        }
                    }
                    if (valid) __stcg(pp.ml(row), make_float2(m_use, l));
                }
                if (whole) {
                    __threadfence_block();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.x_full[t]);
                }
            }
        }
        // ---- items shared with other CTAs: every CTA joins a part of the rows once all pieces are there ----
        const int tid = threadIdx.x - 128;
        unsigned *arrived = reinterpret_cast<unsigned *>(a.workspace), *left = arrived + 256;
        bar_softmax();
        if (tid < 2 && sh.shared[tid].on) {
            __threadfence();
            red_release(arrived + share_owner(sh.shared[tid].u0, W, Ge));
        }
        for (int k = 0; k < 2; k++) {
            const Shared m = sh.shared[k];
            if (!m.on) continue;
            const int c0 = share_owner(m.u0, W, Ge), np = share_owner(m.u0 + m.nb - 1, W, Ge) - c0 + 1, me = cta - c0;
            const int rows = m.rows0 + m.rows1;
            const int lo = rows * me / np, nr = rows * (me + 1) / np - lo;
            if (nr > 0) {
                if (tid == 0) {
                    const uint64_t t0 = gtime_ns();
                    bool there = !*abort_flag;
                    while (there && ld_acquire(arrived + c0) < (unsigned)np)
                        if (gtime_ns() - t0 > kTcuWaitCycles) {
                            there = false;
                            if (a.err) atomicExch(a.err, TC_DEVERR_TIMEOUT);
                        }
                    sh.go = there;
                }
                bar_softmax();
                if (sh.go) join_rows<D>(a, m, c0, np, lo, nr, tid, reinterpret_cast<float *>(sQ));
                bar_softmax();
            }
            if (tid == 0 && atomicAdd(left + c0, 1u) == (unsigned)np - 1u) {
                arrived[c0] = 0u;  // the last to leave: ready for the next launch
                left[c0] = 0u;
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

// 3-D map of the queries: (head_dim, heads, rows), boxes of 64 columns x G heads x P positions, 128-byte swizzle
cudaError_t map_q(CUtensorMap *m, const ChunkArgs &a, int P) {
    return tma_map_bf16_sw128_3d(m, a.q, a.d, a.H, a.rows, a.d, a.ld_q, a.G, P);
}

template <int D>
cudaError_t tc_launch(const ChunkArgs &a, cudaStream_t st) {
    constexpr int smem = (2 + 2 * tc_stages(D)) * tc_tile_bytes(D) + 1024;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    static std::mutex mu;
    static bool prepared[64] = {};
    if (dev >= 0 && dev < 64) {
        std::lock_guard<std::mutex> lk(mu);
        if (!prepared[dev]) {
            e = cudaFuncSetAttribute(qw_chunk_attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e != cudaSuccess) return e;
            prepared[dev] = true;
        }
    }
    CUtensorMap mq, mk, mv;
    const int P = kTcRows / a.G, br = a.ps < kTcKeys ? a.ps : kTcKeys;
    const long long crow = (long long)a.num_pages * a.Hkv * a.ps;
    if ((e = map_q(&mq, a, P)) != cudaSuccess) return e;
    if ((e = tma_map_bf16_sw128(&mk, a.k, crow, a.d, a.d, br)) != cudaSuccess) return e;
    if ((e = tma_map_bf16_sw128(&mv, a.v, crow, a.d, a.d, br)) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms < kNumSMsB200 ? sms : kNumSMsB200);
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeCooperative;  // CTAs that share an item wait for one another
    at[0].val.cooperative = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, qw_chunk_attn_tc_kernel<D>, mq, mk, mv, a);
}

}  // namespace

cudaError_t chunk_attn_launch(const ChunkArgs &a, int dtype, cudaStream_t st) {
    if (dtype == QW_DTYPE_BF16) return a.d == 128 ? tc_launch<128>(a, st) : tc_launch<64>(a, st);
    return a.d == 128 ? simt_launch<float, 128>(a, st) : simt_launch<float, 64>(a, st);
}

size_t chunk_attn_workspace(int head_dim) { return kCounterBytes + (size_t)kNumSMsB200 * 6 * part_bytes(head_dim); }

}  // namespace qw

using namespace qw;

extern "C" uint64_t qw_op_chunk_attn_workspace(int32_t heads, int32_t kv_heads, int32_t head_dim) {
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
    return chunk_attn_workspace(head_dim);
}

extern "C" qw_status qw_op_chunk_attn(const qw_chunk_attn_args *p, void *stream) {
    if (!p) return op_fail(QW_ERR_ARG, "null arguments");
    if (p->dtype != QW_DTYPE_BF16 && p->dtype != QW_DTYPE_F32) return op_fail(QW_ERR_UNSUPPORTED, "dtype must be bf16 or fp32");
    if (p->head_dim != 64 && p->head_dim != 128) return op_fail(QW_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (p->kv_heads < 1 || p->heads < 1 || p->heads % p->kv_heads || p->heads / p->kv_heads > 16)
        return op_fail(QW_ERR_SHAPE, "heads must be 1..16 times kv_heads");
    if (p->batch < 0 || p->rows < 0 || p->batch > kChunkMaxBatch)
        return op_fail(QW_ERR_SHAPE, "batch must be in [0, " + std::to_string(kChunkMaxBatch) + "] and rows >= 0");
    if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
        return op_fail(QW_ERR_SHAPE, "page_size must be a power of two in [16, 256]");
    if (p->num_pages < 1 || p->max_pages < 1 || (long long)p->max_pages * p->page_size > (1ll << 30) ||
        (long long)p->num_pages * p->kv_heads * p->page_size > 0x7FFFFFFFll)
        return op_fail(QW_ERR_SHAPE, "num_pages, max_pages >= 1, below 2^30 positions a slot and 2^31 cached rows");
    if (p->window < 0) return op_fail(QW_ERR_ARG, "window must not be negative");
    if (!(p->scale >= 0.f) || isinf(p->scale)) return op_fail(QW_ERR_ARG, "scale must be positive and finite (0 = 1 / sqrt(head_dim))");
    if (p->rows == 0 || p->batch == 0) return QW_OK;
    if (!p->q || !p->k_cache || !p->v_cache || !p->page_table || !p->row_start || !p->kv_len || !p->out)
        return op_fail(QW_ERR_ARG, "null device pointer");
    const int vec = p->dtype == QW_DTYPE_BF16 ? 8 : 4;
    const int64_t width = (int64_t)p->heads * p->head_dim;
    const int64_t ld_q = p->ld_q ? p->ld_q : width, ld_out = p->ld_out ? p->ld_out : width;
    if (ld_q < width || ld_out < width || ld_q % vec || ld_out % vec || ld_q > (1ll << 31))
        return op_fail(QW_ERR_SHAPE, "ld_q and ld_out must cover heads x head_dim in multiples of 16 bytes");
    if (((uintptr_t)p->q | (uintptr_t)p->k_cache | (uintptr_t)p->v_cache | (uintptr_t)p->out) & 15)
        return op_fail(QW_ERR_ARG, "q, caches and out must be 16-byte aligned");
    if (!p->workspace || ((uintptr_t)p->workspace & 255) ||
        p->workspace_bytes < qw_op_chunk_attn_workspace(p->heads, p->kv_heads, p->head_dim))
        return op_fail(QW_ERR_ARG, "workspace: 256-byte aligned, qw_op_chunk_attn_workspace bytes");
    ChunkArgs a{};
    a.q = p->q; a.k = p->k_cache; a.v = p->v_cache; a.page_table = p->page_table; a.slots = p->slots;
    a.row_start = p->row_start; a.kv_len = p->kv_len; a.out = p->out; a.lse = p->lse; a.err = p->err;
    a.workspace = p->workspace;
    a.ld_q = ld_q; a.ld_out = ld_out;
    a.batch = p->batch; a.rows = p->rows; a.H = p->heads; a.Hkv = p->kv_heads; a.G = p->heads / p->kv_heads;
    a.d = p->head_dim; a.ps = p->page_size; a.num_pages = p->num_pages; a.max_pages = p->max_pages; a.window = p->window;
    a.log2_ps = 0;
    while ((1 << a.log2_ps) < a.ps) a.log2_ps++;
    const float scale = p->scale > 0.f ? p->scale : (float)(1.0 / sqrt((double)p->head_dim));
    a.sl2 = scale * 1.4426950408889634f;
    cudaError_t e = chunk_attn_launch(a, p->dtype, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("chunk attention launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
