// qw_kv_append.cu -- new rows of a ragged batch on their way into the paged cache (qw_op_kv_append): norms of queries and
// keys, rotation by the rows' positions, queries to their buffer, keys and values into their pages.
//
//   q' = q r_q w_q, r = 1 / sqrt(mean(q^2) + eps) over the whole vector or per head (k likewise)
//   (x, y) -> (x cos - y sin, y cos + x sin) for the pairs (i, i + head_dim / 2) of every head, angles from the table
//
// Every number is read once and written once: HBM bounds large batches, the launch small ones.
#include <cuda_runtime.h>
#include <string>

#include "../../include/qwen3_b200.h"
#include "qw_chunk_attn.h"
#include "qw_internal.cuh"
#include "qw_ops.h"

namespace qw {
namespace {

constexpr int kAppendMaxItems = 4096;  // pieces of 16 numbers of a row: heads, keys and values

struct AppendArgs {
    const void *q, *k, *v;
    const float *qn, *kn;
    const float2 *rope;
    void *q_out, *k_cache, *v_cache;
    const int *page_table, *slots, *row_start, *kv_len;
    long long ld_q, ld_k, ld_v, ld_q_out;
    int batch, rows, H, Hkv, d, log2_hc, log2_ps, num_pages, max_pages, mode, rope_len;
    double eps;
};

__device__ __forceinline__ void get8(const __nv_bfloat16 *p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    v[0] = bf16lo(u.x); v[1] = bf16hi(u.x); v[2] = bf16lo(u.y); v[3] = bf16hi(u.y);
    v[4] = bf16lo(u.z); v[5] = bf16hi(u.z); v[6] = bf16lo(u.w); v[7] = bf16hi(u.w);
}
__device__ __forceinline__ void get8(const float *p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ uint32_t pair_bf16(float lo, float hi) {
    return (uint32_t)f2bf_bits(lo) | (uint32_t)f2bf_bits(hi) << 16;
}
__device__ __forceinline__ void set8(__nv_bfloat16 *p, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pair_bf16(v[0], v[1]), pair_bf16(v[2], v[3]), pair_bf16(v[4], v[5]), pair_bf16(v[6], v[7]));
}
__device__ __forceinline__ void set8(float *p, const float (&v)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// One CTA per row.  A thread takes pieces of 8 numbers of a head's first half with the matching 8 of its second half.
template <typename IT, typename OT>
__global__ void __launch_bounds__(256) qw_kv_append_kernel(const AppendArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ float s_red[2][8];
    __shared__ int s_pos, s_slot;
    const int r = blockIdx.x, tid = threadIdx.x;
    if (tid == 0) s_pos = -2;
    __syncthreads();
    // the sequence that holds the row, its position and page
    for (int b = tid; b < a.batch; b += 256) {
        const int lo = min(max(a.row_start[b], 0), a.rows), hi = min(a.row_start[b + 1], a.rows);
        if (r >= lo && r < hi) {
            const int kv = min(max(a.kv_len[b], 0), a.max_pages << a.log2_ps);
            s_pos = max(kv - (hi - r), -1);
            s_slot = a.slots ? a.slots[b] : b;
        }
    }
    __syncthreads();
    const int pos = s_pos;
    if (pos == -2) return;  // behind the last sequence
    const bool live = pos >= 0 && !(a.rope && pos >= a.rope_len);
    const int d = a.d, half = d / 2, hc = 1 << a.log2_hc;
    long long cell = -1;
    if (live) {
        const int page = a.page_table[(long long)s_slot * a.max_pages + (pos >> a.log2_ps)];
        if ((unsigned)page < (unsigned)a.num_pages)
            cell = (((long long)page * a.Hkv) << a.log2_ps) * d + (long long)(pos & ((1 << a.log2_ps) - 1)) * d;
    }
    const IT *q = (const IT *)a.q + r * a.ld_q, *k = (const IT *)a.k + r * a.ld_k, *v = (const IT *)a.v + r * a.ld_v;
    const int nq = a.H * hc, nk = a.Hkv * hc, items = nq + 2 * nk;
    float rq = 1.f, rk = 1.f;
    if (a.mode == QW_QKNORM_VECTOR) {
        float sq = 0.f, sk = 0.f;
        for (int i = tid; i < nq + nk; i += 256) {
            float x[8], y[8], s = 0.f;
            const IT *p = i < nq ? q + (i >> a.log2_hc) * d : k + ((i - nq) >> a.log2_hc) * d;
            get8(p + (i & (hc - 1)) * 8, x);
            get8(p + (i & (hc - 1)) * 8 + half, y);
#pragma unroll
            for (int e = 0; e < 8; e++) s += x[e] * x[e] + y[e] * y[e];
            if (i < nq) sq += s;
            else sk += s;
        }
        sq = warp_sum(sq);
        sk = warp_sum(sk);
        if ((tid & 31) == 0) { s_red[0][tid >> 5] = sq; s_red[1][tid >> 5] = sk; }
        __syncthreads();
        sq = sk = 0.f;
        for (int w = 0; w < 8; w++) { sq += s_red[0][w]; sk += s_red[1][w]; }
        rq = 1.0f / sqrtf(sq / (float)(a.H * d) + (float)a.eps);
        rk = 1.0f / sqrtf(sk / (float)(a.Hkv * d) + (float)a.eps);
    }
    OT *q_out = a.q_out ? (OT *)a.q_out + r * a.ld_q_out : nullptr;
    for (int base = 0; base < items; base += 256) {
        const int i = base + tid;
        const bool on = i < items, isq = i < nq, isk = !isq && i < nq + nk;
        const int j = isq ? i : (isk ? i - nq : i - nq - nk);
        const int h = j >> a.log2_hc, f = (j & (hc - 1)) * 8;
        float x[8] = {}, y[8] = {};
        if (on) {
            const IT *p = (isq ? q : isk ? k : v) + (long long)h * d + f;
            get8(p, x);
            get8(p + half, y);
        }
        float n = isq ? rq : rk;
        if (a.mode == QW_QKNORM_HEAD) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) s += x[e] * x[e] + y[e] * y[e];
            for (int o = hc >> 1; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            n = 1.0f / sqrtf(s / (float)d + (float)a.eps);
        }
        if (!on) continue;
        if (isq || isk) {
            if (a.mode != QW_QKNORM_NONE) {
                const float *w = (isq ? a.qn : a.kn) + (a.mode == QW_QKNORM_VECTOR ? h * d : 0) + f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[e] = w[e] * (x[e] * n);
                    y[e] = w[e + half] * (y[e] * n);
                }
            }
            if (a.rope && live) {
                const float2 *cs = a.rope + (long long)pos * half + f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float2 c = cs[e];
                    const float u = x[e] * c.x - y[e] * c.y;
                    y[e] = y[e] * c.x + x[e] * c.y;
                    x[e] = u;
                }
            }
        }
        if (isq) {
            if (q_out) {
                if (!live) {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = y[e] = 0.f;
                }
                set8(q_out + (long long)h * d + f, x);
                set8(q_out + (long long)h * d + f + half, y);
            }
        } else if (cell >= 0) {
            OT *to = (OT *)(isk ? a.k_cache : a.v_cache) + cell + ((long long)h << a.log2_ps) * d + f;
            set8(to, x);
            set8(to + half, y);
        }
    }
}

template <typename IT, typename OT>
cudaError_t append_launch(const AppendArgs &a, cudaStream_t st) {
    return launch_pdl(qw_kv_append_kernel<IT, OT>, dim3(a.rows), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace qw

using namespace qw;

extern "C" qw_status qw_op_kv_append(const qw_kv_append_args *p, void *stream) {
    if (!p) return op_fail(QW_ERR_ARG, "null arguments");
    for (int t : {p->in_dtype, p->dtype})
        if (t != QW_DTYPE_F32 && t != QW_DTYPE_BF16) return op_fail(QW_ERR_UNSUPPORTED, "dtypes must be fp32 or bf16");
    if (p->head_dim < 16 || p->head_dim > 256 || (p->head_dim & (p->head_dim - 1)))
        return op_fail(QW_ERR_UNSUPPORTED, "head_dim must be a power of two in [16, 256]");
    if (p->heads < 1 || p->kv_heads < 1 || ((long long)p->heads + 2ll * p->kv_heads) * p->head_dim > 16ll * kAppendMaxItems)
        return op_fail(QW_ERR_SHAPE, "heads and kv_heads must be positive, (heads + 2 kv_heads) x head_dim up to 65536");
    if (p->batch < 0 || p->rows < 0 || p->batch > kChunkMaxBatch)
        return op_fail(QW_ERR_SHAPE, "batch must be in [0, " + std::to_string(kChunkMaxBatch) + "] and rows >= 0");
    if (p->page_size < 1 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
        return op_fail(QW_ERR_SHAPE, "page_size must be a power of two up to 256");
    if (p->num_pages < 1 || p->max_pages < 1 || (long long)p->max_pages * p->page_size > (1ll << 30))
        return op_fail(QW_ERR_SHAPE, "num_pages, max_pages >= 1 and up to 2^30 positions a slot");
    if (p->qk_norm < QW_QKNORM_NONE || p->qk_norm > QW_QKNORM_HEAD) return op_fail(QW_ERR_ARG, "qk_norm");
    if (p->qk_norm != QW_QKNORM_NONE && (!p->q_norm || !p->k_norm)) return op_fail(QW_ERR_ARG, "qk_norm needs q_norm and k_norm");
    if (!(p->eps >= 0.0)) return op_fail(QW_ERR_ARG, "eps must not be negative");
    if (p->rope && p->rope_len < 1) return op_fail(QW_ERR_SHAPE, "rope_len must be positive");
    AppendArgs a{};
    const long long wq = (long long)p->heads * p->head_dim, wk = (long long)p->kv_heads * p->head_dim;
    a.ld_q = p->ld_q ? p->ld_q : wq; a.ld_k = p->ld_k ? p->ld_k : wk; a.ld_v = p->ld_v ? p->ld_v : wk;
    a.ld_q_out = p->ld_q_out ? p->ld_q_out : wq;
    const int vi = p->in_dtype == QW_DTYPE_BF16 ? 8 : 4, vo = p->dtype == QW_DTYPE_BF16 ? 8 : 4;
    if (a.ld_q < wq || a.ld_k < wk || a.ld_v < wk || a.ld_q_out < wq || a.ld_q % vi || a.ld_k % vi || a.ld_v % vi ||
        a.ld_q_out % vo)
        return op_fail(QW_ERR_SHAPE, "row strides must cover the heads in multiples of 16 bytes");
    if (p->rows == 0 || p->batch == 0) return QW_OK;
    if (!p->q || !p->k || !p->v || !p->k_cache || !p->v_cache || !p->page_table || !p->row_start || !p->kv_len)
        return op_fail(QW_ERR_ARG, "null device pointer");
    if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->q_out | (uintptr_t)p->k_cache |
         (uintptr_t)p->v_cache | (uintptr_t)p->rope | (uintptr_t)p->q_norm | (uintptr_t)p->k_norm) & 15)
        return op_fail(QW_ERR_ARG, "rows, caches, norms and rope must be 16-byte aligned");
    if (p->q_out == p->q && (p->in_dtype != p->dtype || a.ld_q != a.ld_q_out))
        return op_fail(QW_ERR_ARG, "q_out may be q only with the same type and stride");
    a.q = p->q; a.k = p->k; a.v = p->v; a.qn = p->q_norm; a.kn = p->k_norm; a.rope = (const float2 *)p->rope;
    a.q_out = p->q_out; a.k_cache = p->k_cache; a.v_cache = p->v_cache;
    a.page_table = p->page_table; a.slots = p->slots; a.row_start = p->row_start; a.kv_len = p->kv_len;
    a.batch = p->batch; a.rows = p->rows; a.H = p->heads; a.Hkv = p->kv_heads; a.d = p->head_dim;
    a.num_pages = p->num_pages; a.max_pages = p->max_pages; a.mode = p->qk_norm; a.rope_len = p->rope_len; a.eps = p->eps;
    while (16 << a.log2_hc < a.d) a.log2_hc++;
    while (1 << a.log2_ps < p->page_size) a.log2_ps++;
    const bool ib = p->in_dtype == QW_DTYPE_BF16, ob = p->dtype == QW_DTYPE_BF16;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = ib ? (ob ? append_launch<__nv_bfloat16, __nv_bfloat16>(a, st) : append_launch<__nv_bfloat16, float>(a, st))
                       : (ob ? append_launch<float, __nv_bfloat16>(a, st) : append_launch<float, float>(a, st));
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("append launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
