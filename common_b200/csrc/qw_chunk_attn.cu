// qw_chunk_attn.cu -- attention of a ragged batch of new tokens over the paged KV cache.
//
// Sequence b brings n_b = row_start[b + 1] - row_start[b] query rows and has kv_len[b] cached positions, those of the
// new rows included; its row i stands at position p = kv_len[b] - n_b + i and sees positions
// max(0, p - window + 1) .. p.  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q . k_j, m = max s_j, and
// lse = m + ln(sum): one pass over the keys with the running maximum and sum.  A row that sees nothing gives zeros and
// -infinity.  Lengths are read on the device, so a captured graph follows them.
#include <cuda_runtime.h>
#include <math.h>
#include <string>

#include "../../include/qwen3_b200.h"
#include "qw_chunk_attn.h"
#include "qw_internal.cuh"
#include "qw_ops.h"

namespace qw {
namespace {

constexpr int kSiRows = 64, kSiKeys = 64, kSiThreads = 256;
constexpr int kSiMaxCtas = 2 * kNumSMsB200;  // of a launch that splits keys: its partial results lie in the workspace

__host__ __device__ constexpr size_t si_part_bytes(int d) { return (size_t)kSiRows * (d + 2) * 4; }

// One CTA per (64 rows of a sequence's (position, head of the group) list, KV head, range of its keys): q, K and V tiles
// in shared memory, a 4 x 4 block of scores and 4 x (D / 16) of the output per thread.  Where the rows alone do not fill
// the GPU the keys are split, and the last CTA of a tile to finish joins the ranges in their order (no sum depends on who
// came when).  fp32 caches have no tensor-core path in this library; the arithmetic of 64 x 64 x D tiles bounds this
// kernel: 13.5 TFLOP/s (512 rows over 4000 positions, 32 heads).
template <int D>
__global__ void __launch_bounds__(kSiThreads) qw_chunk_attn_simt_kernel(const ChunkArgs a, int nsplit) {
    extern __shared__ float si_smem[];
    constexpr int LD = D + 4;
    float *sq = si_smem, *sk = sq + kSiRows * LD, *sv = sk + kSiKeys * LD, *sp = sv + kSiKeys * LD;
    __shared__ float s_m[kSiRows], s_l[kSiRows], s_alpha[kSiRows];
    __shared__ bool s_last;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int G = a.G, kvh = blockIdx.y;
    int b = 0, tile = blockIdx.x, r0 = 0, n = 0;
    for (; b < a.batch; b++) {
        r0 = min(max(a.row_start[b], 0), a.rows);
        n = max(0, min(a.row_start[b + 1], a.rows) - r0);
        const int t = (n * G + kSiRows - 1) / kSiRows;
        if (tile < t) break;
        tile -= t;
    }
    if (b >= a.batch) return;
    const int kv = min(max(a.kv_len[b], 0), a.max_pages << a.log2_ps);
    const int p0 = kv - n, first = tile * kSiRows, last = min(first + kSiRows, n * G) - 1;
    const int *table = a.page_table + (size_t)(a.slots ? a.slots[b] : b) * a.max_pages;
    const float *q = (const float *)a.q, *kc = (const float *)a.k, *vc = (const float *)a.v;
    for (int i = tid; i < kSiRows * D; i += kSiThreads) {
        const int r = i / D, c = i % D, pr = first + r;
        sq[r * LD + c] = pr <= last ? q[(size_t)(r0 + pr / G) * a.ld_q + (size_t)(kvh * G + pr % G) * D + c] : 0.f;
    }
    if (tid < kSiRows) { s_m[tid] = -INFINITY; s_l[tid] = 0.f; }
    float o[4][D / 16] = {};
    const int lo = a.window ? max(0, p0 + first / G - a.window + 1) : 0;
    const int b0 = lo / kSiKeys, nb = p0 + last / G < 0 ? 0 : (p0 + last / G) / kSiKeys + 1 - b0;
    const int kend = (b0 + (int)((long long)nb * (blockIdx.z + 1) / nsplit)) * kSiKeys;
    for (int k0 = (b0 + (int)((long long)nb * blockIdx.z / nsplit)) * kSiKeys; k0 < kend; k0 += kSiKeys) {
        __syncthreads();
        for (int i = tid; i < kSiKeys * D; i += kSiThreads) {
            const int r = i / D, c = i % D, pos = k0 + r;
            float kx = 0.f, vx = 0.f;  // nothing is read where no row of the tile sees anything
            if (pos >= lo && pos < kv) {
                const int pg = table[pos >> a.log2_ps];
                if ((unsigned)pg < (unsigned)a.num_pages) {
                    const size_t at = (((size_t)pg * a.Hkv + kvh) * a.ps + (pos & (a.ps - 1))) * D + c;
                    kx = kc[at];
                    vx = vc[at];
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
    if (nsplit > 1) {
        // partial results: O [row][D], then maximum and sum
        const int tile_id = blockIdx.y * gridDim.x + blockIdx.x;
        unsigned *counter = reinterpret_cast<unsigned *>(a.workspace) + tile_id;
        char *parts = (char *)a.workspace + kChunkCounterBytes + (size_t)tile_id * nsplit * si_part_bytes(D);
        float *mine = reinterpret_cast<float *>(parts + blockIdx.z * si_part_bytes(D));
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < D / 16; c++) mine[(ty * 4 + i) * D + tx + 16 * c] = o[i][c];
        if (tid < kSiRows) {
            mine[kSiRows * D + tid] = s_m[tid];
            mine[kSiRows * (D + 1) + tid] = s_l[tid];
        }
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            s_last = atomicAdd(counter, 1u) == (unsigned)nsplit - 1u;
            if (s_last) *counter = 0u;
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = ty * 4 + i;
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int c = 0; c < D / 16; c++) o[i][c] = 0.f;
            for (int z = 0; z < nsplit; z++) {
                const float *p = reinterpret_cast<const float *>(parts + z * si_part_bytes(D));
                const float pm = __ldcg(p + kSiRows * D + r), pl = __ldcg(p + kSiRows * (D + 1) + r);
                if (pl == 0.f) continue;  // this range showed the row nothing (NaN scores have no maximum, but a sum)
                const float mn = fmaxf(m, pm), wo = exp2f(m - mn), wp = exp2f(pm - mn);
                l = l * wo + pl * wp;
#pragma unroll
                for (int c = 0; c < D / 16; c++) o[i][c] = o[i][c] * wo + __ldcg(p + r * D + tx + 16 * c) * wp;
                m = mn;
            }
            __syncwarp();
            if (tx == 0) { s_m[r] = m; s_l[r] = l; }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int pr = first + ty * 4 + i;
        if (pr > last) continue;
        const float l = s_l[ty * 4 + i], inv = l > 0.f ? 1.f / l : 0.f;
        const size_t row = (size_t)(r0 + pr / G), head = (size_t)(kvh * G + pr % G);
        float *out = (float *)a.out + row * a.ld_out + head * D;
#pragma unroll
        for (int c = 0; c < D / 16; c++) out[tx + 16 * c] = l == 0.f ? 0.f : o[i][c] * inv;
        if (a.lse && tx == 0)
            a.lse[row * a.H + head] = l > 0.f ? (s_m[ty * 4 + i] + log2f(l)) * 0.69314718055994531f : l == 0.f ? -INFINITY : l;
    }
}

// Few rows per sequence (decoding): one CTA per (row, KV head, range of its keys).  A warp takes 4 steps of 32 / (D / 4) keys
// at a time, D / 4 lanes a key (its 16 bytes per lane are one coalesced row of the cache), the dot products of the group's R
// heads are summed across those lanes, and every lane keeps its columns of the R outputs.  Bound by HBM: the lanes' sums
// are about 5 R shuffles a key for 8 D bytes.
template <int D, int R>
__global__ void __launch_bounds__(kSiThreads) qw_chunk_attn_rows_kernel(const ChunkArgs a, int nsplit) {
    constexpr int LK = D / 4, KPS = 32 / LK, W = kSiThreads / 32;
    __shared__ float4 s_o[W][R][32];
    __shared__ float s_m[W][R], s_l[W][R];
    __shared__ bool s_last;
    const int row = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int sub = lane / LK, c = (lane % LK) * 4, G = a.G;
    int b = 0, e = a.batch - 1;  // the sequence that the row belongs to: the last that begins at or before it
    while (b < e) {
        const int mid = (b + e + 1) >> 1;
        if (a.row_start[mid] <= row) b = mid;
        else e = mid - 1;
    }
    if (a.row_start[b] > row || a.row_start[b + 1] <= row) return;
    const int kv = min(max(a.kv_len[b], 0), a.max_pages << a.log2_ps);
    const int pos = kv - (min(a.row_start[b + 1], a.rows) - row);
    const int lo = a.window ? max(0, pos - a.window + 1) : 0, n = pos + 1 - lo;
    const int k_begin = n > 0 ? lo + (int)((long long)n * blockIdx.z / nsplit) : 0;
    const int k_end = n > 0 ? lo + (int)((long long)n * (blockIdx.z + 1) / nsplit) : 0;
    const int *table = a.page_table + (size_t)(a.slots ? a.slots[b] : b) * a.max_pages;
    const float *kc = (const float *)a.k, *vc = (const float *)a.v;
    float4 q[R], o[R];
    float m[R], l[R];
#pragma unroll
    for (int h = 0; h < R; h++) {
        q[h] = o[h] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (h < G) q[h] = *reinterpret_cast<const float4 *>((const float *)a.q + (size_t)row * a.ld_q + (size_t)(kvh * G + h) * D + c);
        m[h] = -INFINITY;
        l[h] = 0.f;
    }
    for (int k0 = k_begin + warp * 4 * KPS; k0 < k_end; k0 += W * 4 * KPS) {
        float4 k[4], v[4];
        bool sees[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int key = k0 + u * KPS + sub;
            sees[u] = key < k_end;
            k[u] = v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            const int pg = sees[u] ? table[key >> a.log2_ps] : -1;
            if ((unsigned)pg < (unsigned)a.num_pages) {
                const size_t at = (((size_t)pg * a.Hkv + kvh) * a.ps + (key & (a.ps - 1))) * D + c;
                k[u] = *reinterpret_cast<const float4 *>(kc + at);
                v[u] = *reinterpret_cast<const float4 *>(vc + at);
            }
        }
#pragma unroll
        for (int h = 0; h < R; h++) {
            float s[4], mx = m[h];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                s[u] = q[h].x * k[u].x + q[h].y * k[u].y + q[h].z * k[u].z + q[h].w * k[u].w;
#pragma unroll
                for (int w = LK / 2; w > 0; w >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], w);
                s[u] = sees[u] ? s[u] * a.sl2 : -INFINITY;
                mx = fmaxf(mx, s[u]);
            }
            const float mu = mx == -INFINITY ? 0.f : mx, al = exp2f(m[h] - mu);
            l[h] *= al;
            o[h].x *= al; o[h].y *= al; o[h].z *= al; o[h].w *= al;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float p = exp2f(s[u] - mu);
                l[h] += p;
                o[h].x += p * v[u].x; o[h].y += p * v[u].y; o[h].z += p * v[u].z; o[h].w += p * v[u].w;
            }
            m[h] = mx;
        }
    }
    // join the lanes that took different keys, then the warps, then (the last CTA of the row) the ranges
    auto join = [](float &m0, float &l0, float4 &o0, float m1, float l1, const float4 &o1) {
        if (l1 == 0.f) return;  // nothing seen (NaN scores have no maximum, but a sum)
        const float mn = fmaxf(m0, m1), w0 = exp2f(m0 - mn), w1 = exp2f(m1 - mn);
        l0 = l0 * w0 + l1 * w1;
        o0 = make_float4(o0.x * w0 + o1.x * w1, o0.y * w0 + o1.y * w1, o0.z * w0 + o1.z * w1, o0.w * w0 + o1.w * w1);
        m0 = mn;
    };
#pragma unroll
    for (int h = 0; h < R; h++) {
#pragma unroll
        for (int w = LK; w < 32; w <<= 1) {
            const float m1 = __shfl_xor_sync(0xffffffffu, m[h], w), l1 = __shfl_xor_sync(0xffffffffu, l[h], w);
            const float4 o1 = make_float4(__shfl_xor_sync(0xffffffffu, o[h].x, w), __shfl_xor_sync(0xffffffffu, o[h].y, w),
                                          __shfl_xor_sync(0xffffffffu, o[h].z, w), __shfl_xor_sync(0xffffffffu, o[h].w, w));
            join(m[h], l[h], o[h], m1, l1, o1);
        }
        s_o[warp][h][lane] = o[h];
        if (lane == 0) { s_m[warp][h] = m[h]; s_l[warp][h] = l[h]; }
    }
    __syncthreads();
    const int id = blockIdx.y * gridDim.x + blockIdx.x;
    unsigned *counter = reinterpret_cast<unsigned *>(a.workspace) + id;
    float *parts = reinterpret_cast<float *>((char *)a.workspace + kChunkCounterBytes) + (size_t)id * nsplit * R * (D + 2);
    auto result = [&](int h, float mm, float ll, const float4 &oo) {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        const size_t head = (size_t)(kvh * G + h);
        if (lane < LK)
            *reinterpret_cast<float4 *>((float *)a.out + (size_t)row * a.ld_out + head * D + c) =
                ll == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(oo.x * inv, oo.y * inv, oo.z * inv, oo.w * inv);
        if (a.lse && lane == 0) a.lse[(size_t)row * a.H + head] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
    };
    for (int h = warp; h < G; h += W) {
        float mm = -INFINITY, ll = 0.f;
        float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < W; w++) join(mm, ll, oo, s_m[w][h], s_l[w][h], s_o[w][h][lane]);
        if (nsplit == 1) {
            result(h, mm, ll, oo);
            continue;
        }
        float *p = parts + ((size_t)blockIdx.z * R + h) * (D + 2);
        if (lane < LK) {
            p[c] = oo.x; p[c + 1] = oo.y; p[c + 2] = oo.z; p[c + 3] = oo.w;
        }
        if (lane == 0) { p[D] = mm; p[D + 1] = ll; }
    }
    if (nsplit == 1) return;
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        s_last = atomicAdd(counter, 1u) == (unsigned)nsplit - 1u;
        if (s_last) *counter = 0u;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    for (int h = warp; h < G; h += W) {
        float mm = -INFINITY, ll = 0.f;
        float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int z = 0; z < nsplit; z++) {
            const float *p = parts + ((size_t)z * R + h) * (D + 2);
            join(mm, ll, oo, __ldcg(p + D), __ldcg(p + D + 1),
                 make_float4(__ldcg(p + c), __ldcg(p + c + 1), __ldcg(p + c + 2), __ldcg(p + c + 3)));
        }
        result(h, mm, ll, oo);
    }
}

template <int D, int R>
cudaError_t rows_launch(const ChunkArgs &a, cudaStream_t st) {
    // ranges of 128 keys at least, and as many CTAs as fill the GPU four times
    const long long ctas = (long long)a.rows * a.Hkv, blocks = ((long long)a.max_pages * a.ps + 127) / 128;
    long long nsplit = 4 * kSiMaxCtas / 2 / ctas;
    if (nsplit > blocks) nsplit = blocks;
    if (nsplit < 1) nsplit = 1;
    qw_chunk_attn_rows_kernel<D, R><<<dim3(a.rows, a.Hkv, (unsigned)nsplit), kSiThreads, 0, st>>>(a, (int)nsplit);
    return cudaGetLastError();
}

template <int D>
cudaError_t simt_launch(const ChunkArgs &a, cudaStream_t st) {
    // Up to two rows a sequence: the rows' kernel reads the cache once per row; above, the tiles' once per 64 / G rows.
    // 8 sequences of one row at 4000 positions, 4 heads per KV head: 987 us by tiles, 87 us (3.0 TB/s)
    // by rows.
    if (a.G <= 8 && a.rows <= 2 * (long long)a.batch) {
        if (a.G == 1) return rows_launch<D, 1>(a, st);
        if (a.G == 2) return rows_launch<D, 2>(a, st);
        if (a.G <= 4) return rows_launch<D, 4>(a, st);
        return rows_launch<D, 8>(a, st);
    }
    const int smem = (3 * kSiRows * (D + 4) + kSiRows * (kSiKeys + 1)) * (int)sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(qw_chunk_attn_simt_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    // at most one tile more than the whole ones for every sequence
    const long long tiles = (long long)a.rows * a.G / kSiRows + a.batch;
    const long long blocks = ((long long)a.max_pages * a.ps + kSiKeys - 1) / kSiKeys;
    long long nsplit = kSiMaxCtas / (tiles * a.Hkv);
    if (nsplit > blocks) nsplit = blocks;
    if (nsplit < 1) nsplit = 1;
    qw_chunk_attn_simt_kernel<D><<<dim3((unsigned)tiles, a.Hkv, (unsigned)nsplit), kSiThreads, smem, st>>>(a, (int)nsplit);
    return cudaGetLastError();
}

}  // namespace

cudaError_t chunk_attn_simt_launch(const ChunkArgs &a, cudaStream_t st) {
    return a.d == 128 ? simt_launch<128>(a, st) : simt_launch<64>(a, st);
}

}  // namespace qw

using namespace qw;

extern "C" uint64_t qw_op_chunk_attn_workspace(int32_t heads, int32_t kv_heads, int32_t head_dim) {
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
    return chunk_attn_tc_workspace(head_dim);
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
    a.d = p->head_dim; a.ps = p->page_size; a.num_pages = p->num_pages; a.max_pages = p->max_pages;
    a.window = p->window < (long long)p->max_pages * p->page_size ? p->window : 0;  // as long as a slot: it cuts nothing off
    a.log2_ps = 0;
    while ((1 << a.log2_ps) < a.ps) a.log2_ps++;
    if (p->dtype == QW_DTYPE_BF16 && chunk_attn_tc_most_units(a) > 0xFFFFFFFFull)
        return op_fail(QW_ERR_SHAPE, "rows over max_pages pages are too many key blocks for one call");
    const float scale = p->scale > 0.f ? p->scale : (float)(1.0 / sqrt((double)p->head_dim));
    a.sl2 = scale * 1.4426950408889634f;
    cudaError_t e = p->dtype == QW_DTYPE_BF16 ? chunk_attn_tc_launch(a, (cudaStream_t)stream)
                                               : chunk_attn_simt_launch(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("chunk attention launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
