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

}  // namespace

cudaError_t chunk_attn_simt_launch(const ChunkArgs &a, cudaStream_t st) {
    return a.d == 128 ? simt_launch<float, 128>(a, st) : simt_launch<float, 64>(a, st);
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
    a.d = p->head_dim; a.ps = p->page_size; a.num_pages = p->num_pages; a.max_pages = p->max_pages; a.window = p->window;
    a.log2_ps = 0;
    while ((1 << a.log2_ps) < a.ps) a.log2_ps++;
    const float scale = p->scale > 0.f ? p->scale : (float)(1.0 / sqrt((double)p->head_dim));
    a.sl2 = scale * 1.4426950408889634f;
    cudaError_t e = p->dtype == QW_DTYPE_BF16 ? chunk_attn_tc_launch(a, (cudaStream_t)stream)
                                               : chunk_attn_simt_launch(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("chunk attention launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
