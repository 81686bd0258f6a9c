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

constexpr int kAppendThreads = 128;
constexpr int kAppendFew = 1024;  // rows up to which a CTA takes one each
constexpr int kAppendRows = 4;    // rows of a CTA beyond
constexpr int kAppendMaxItems = 4096;  // pieces of 16 numbers of a row: heads, keys and values

struct AppendArgs {
    const void *q, *k, *v;
    const float *qn, *kn;
    const float2 *rope;
    void *q_out, *k_cache, *v_cache;
    const int *page_table, *slots, *row_start, *kv_len;
    long long ld_q, ld_k, ld_v, ld_q_out;
    int batch, rows, H, Hkv, d, log2_hc, log2_ps, num_pages, max_pages, mode, rope_len;
    float eps, inv_d;
};

// 8 numbers as they lie in memory
template <typename T> struct Raw8 { uint4 v[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw8<T> get8(const T *p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.v[i] = reinterpret_cast<const uint4 *>(p)[i];
    return r;
}
__device__ __forceinline__ void widen8(const Raw8<__nv_bfloat16> &r, float (&v)[8]) {
    const uint4 u = r.v[0];
    v[0] = bf16lo(u.x); v[1] = bf16hi(u.x); v[2] = bf16lo(u.y); v[3] = bf16hi(u.y);
    v[4] = bf16lo(u.z); v[5] = bf16hi(u.z); v[6] = bf16lo(u.w); v[7] = bf16hi(u.w);
}
__device__ __forceinline__ void widen8(const Raw8<float> &r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        v[4 * i] = __uint_as_float(r.v[i].x); v[4 * i + 1] = __uint_as_float(r.v[i].y);
        v[4 * i + 2] = __uint_as_float(r.v[i].z); v[4 * i + 3] = __uint_as_float(r.v[i].w);
    }
}
__device__ __forceinline__ uint32_t pair_bf16(float lo, float hi) {
    const __nv_bfloat162 w = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&w);
}
__device__ __forceinline__ void set8(__nv_bfloat16 *p, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pair_bf16(v[0], v[1]), pair_bf16(v[2], v[3]), pair_bf16(v[4], v[5]), pair_bf16(v[6], v[7]));
}
__device__ __forceinline__ void set8(float *p, const float (&v)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ float squares(const float (&x)[8], const float (&y)[8]) {
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        s += x[e] * x[e];
        t += y[e] * y[e];
    }
    return s + t;
}
// x and y times their weights and n; then turned by the angles of cosines c and sines s
__device__ __forceinline__ void scale8(float (&x)[8], float (&y)[8], const float (&wx)[8], const float (&wy)[8], float n) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = wx[e] * (x[e] * n);
        y[e] = wy[e] * (y[e] * n);
    }
}
__device__ __forceinline__ void turn8(float (&x)[8], float (&y)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float u = x[e] * c[e] - y[e] * s[e];
        y[e] = y[e] * c[e] + x[e] * s[e];
        x[e] = u;
    }
}

// the sum of n numbers' squares in consecutive lanes, n a power of two
__device__ __forceinline__ float lanes_sum(float v, int n) {
    for (int o = n >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One CTA per row, for few rows and for norms over whole vectors.  A thread takes 8 numbers of a head's first half with the
// matching 8 of its second (the rotary pairs), and the same 8 of every further head that it serves, so that a row's angles are
// read once per thread; CH heads are on their way at a time, the first of them while the row's sequence, position and page are
// looked up.  64 sequences of one token, 32 / 8 heads, take 4.1 us from fp32: the launch, and lengths, page and angles one after the
// other; 64 rows of one sequence 3.7, 1024 sequences of one token 17.5, for every CTA reads the lengths of them all.  13,800 rows with
// norms over whole vectors take 79 us (bf16, 4.2 TB/s): every row waits for its sums, and five rows fit an SM's registers.
template <typename IT, typename OT, int CH>
__global__ void __launch_bounds__(kAppendThreads) qw_kv_append_row_kernel(const AppendArgs a) {
    __shared__ float s_red[2][kAppendThreads / 32];
    __shared__ int s_pos;
    __shared__ long long s_cell;
    const int tid = threadIdx.x, hc = 1 << a.log2_hc, d = a.d, half = d >> 1;
    const int f = (tid & (hc - 1)) * 8, step = kAppendThreads >> a.log2_hc, first = tid >> a.log2_hc;
    const int heads = a.H + 2 * a.Hkv;  // queries, keys, values
    const long long r = blockIdx.x;
    if (tid == 0) s_pos = -2;
    griddep_wait();
    griddep_launch_dependents();
    Raw8<IT> lo[CH], hi[CH];
    const auto load = [&](int h0) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int h = h0 + c * step;
            if (h >= heads) break;
            const IT *p = h < a.H ? (const IT *)a.q + r * a.ld_q + h * d
                                  : h < a.H + a.Hkv ? (const IT *)a.k + r * a.ld_k + (h - a.H) * d
                                                    : (const IT *)a.v + r * a.ld_v + (h - a.H - a.Hkv) * d;
            lo[c] = get8(p + f);
            hi[c] = get8(p + f + half);
        }
    };
    load(first);
    __syncthreads();
    for (int b = tid; b < a.batch; b += kAppendThreads) {
        const int begin = min(max(a.row_start[b], 0), a.rows), end = min(max(a.row_start[b + 1], 0), a.rows);
        const int kv = min(max(a.kv_len[b], 0), a.max_pages << a.log2_ps), slot = a.slots ? a.slots[b] : b;
        if (r >= begin && r < end) {
            const int pos = max(kv - (end - (int)r), -1);
            long long cell = -1;
            if (pos >= 0 && !(a.rope && pos >= a.rope_len)) {
                const int page = a.page_table[(long long)slot * a.max_pages + (pos >> a.log2_ps)];
                if ((unsigned)page < (unsigned)a.num_pages)
                    cell = ((((long long)page * a.Hkv) << a.log2_ps) + (pos & ((1 << a.log2_ps) - 1))) * d;
            }
            s_pos = pos;
            s_cell = cell;
        }
    }
    float rq = 1.f, rk = 1.f;
    if (a.mode == QW_QKNORM_VECTOR) {
        float sq = 0.f, sk = 0.f;
        for (int h0 = first; h0 < a.H + a.Hkv; h0 += CH * step) {
            if (h0 != first) load(h0);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const int h = h0 + c * step;
                if (h >= a.H + a.Hkv) break;
                float x[8], y[8];
                widen8(lo[c], x);
                widen8(hi[c], y);
                const float s = squares(x, y);
                if (h < a.H) sq += s;
                else sk += s;
            }
        }
        if (first + CH * step < a.H + a.Hkv) load(first);
        sq = warp_sum(sq);
        sk = warp_sum(sk);
        if ((tid & 31) == 0) { s_red[0][tid >> 5] = sq; s_red[1][tid >> 5] = sk; }
        __syncthreads();
        sq = sk = 0.f;
#pragma unroll
        for (int w = 0; w < kAppendThreads / 32; w++) { sq += s_red[0][w]; sk += s_red[1][w]; }
        rq = rsqrtf(sq / (float)(a.H * d) + a.eps);
        rk = rsqrtf(sk / (float)(a.Hkv * d) + a.eps);
    } else {
        __syncthreads();
    }
    const int pos = s_pos;
    if (pos == -2) return;  // behind the last sequence
    const bool live = pos >= 0 && !(a.rope && pos >= a.rope_len);
    const long long cell = live ? s_cell : -1;
    float cs[8], sn[8];
    if (a.rope && live) {
        const float4 *p = reinterpret_cast<const float4 *>(a.rope + (long long)pos * half + f);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float4 u = p[e >> 1];
            cs[e] = u.x; sn[e] = u.y; cs[e + 1] = u.z; sn[e + 1] = u.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) { cs[e] = 1.f; sn[e] = 0.f; }
    }
    for (int h0 = first; h0 < first + (heads + step - 1) / step * step; h0 += CH * step) {  // the same rounds on every lane
        if (h0 != first) load(h0);
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int h = h0 + c * step;
            if (h - first >= heads) break;
            const bool isq = h < a.H, isv = h >= a.H + a.Hkv;
            float x[8], y[8], n = isq ? rq : rk;
            widen8(lo[c], x);
            widen8(hi[c], y);
            if (a.mode == QW_QKNORM_HEAD) n = rsqrtf(lanes_sum(h < heads ? squares(x, y) : 0.f, hc) * a.inv_d + a.eps);
            if (h >= heads) continue;
            if (!isv) {
                if (a.mode != QW_QKNORM_NONE) {
                    const float *w = (isq ? a.qn : a.kn) + f;
                    if (a.mode == QW_QKNORM_VECTOR) w += (isq ? h : h - a.H) * d;
                    float wx[8], wy[8];
                    widen8(get8(w), wx);
                    widen8(get8(w + half), wy);
                    scale8(x, y, wx, wy, n);
                }
                if (a.rope) turn8(x, y, cs, sn);
            }
            if (isq) {
                if (!live) {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = y[e] = 0.f;
                }
                if (a.q_out) {
                    OT *to = (OT *)a.q_out + r * a.ld_q_out + h * d + f;
                    set8(to, x);
                    set8(to + half, y);
                }
            } else if (cell >= 0) {
                const int kh = isv ? h - a.H - a.Hkv : h - a.H;
                OT *to = (OT *)(isv ? a.v_cache : a.k_cache) + cell + ((long long)kh << a.log2_ps) * d + f;
                set8(to, x);
                set8(to + half, y);
            }
        }
    }
}

// where a row goes
struct AppendRow {
    long long cell;  // of its keys and values in head 0, in elements; -1: nowhere
    int state;       // kNoRow: behind the last sequence; kNowhere: a row before position 0 or behind the angles
};
constexpr int kLive = 1, kNowhere = 0, kNoRow = -1;

// One CTA per R rows, for many of them.  A thread takes 8 numbers of a head's first half with the matching 8 of its second of
// every row, then the same of the next head that it serves: heads outside, rows inside, so that addresses, norm weights and the
// choice between queries, keys and values are made once for R rows; two rows are on their way while two are turned.  The
// rows' sequences, positions, pages and angles are looked up at once, behind the first loads.  13,800 rows of 32 / 8 heads of 128:
// 64 us from bf16 with norms per head (5.2 TB/s; 80 with a CTA per row), 59 without norms, 85 from fp32 (5.9 TB/s); of 14 / 2 heads of
// 64 27 us (49 with a CTA per row, whose threads a row of 1152 numbers does not fill).  Bound by HBM and, at 230 instructions per 32
// pieces, by their issue (half of the slots); 8 rows a CTA take 70 us, 6 CTAs an SM (80 registers) 77;
// fp32 rows need the registers of 4 CTAs (5: 109 us).
template <typename IT, typename OT, int R>
__global__ void __launch_bounds__(kAppendThreads, sizeof(IT) == 2 ? 5 : 4) qw_kv_append_rows_kernel(const AppendArgs a) {
    constexpr int STEP = 2;  // rows on their way at a time
    extern __shared__ __align__(16) float s_angles[];  // [R][cos, sin][d / 2]
    __shared__ AppendRow s_row[R];
    __shared__ int s_pos[R];
    const int tid = threadIdx.x, hc = 1 << a.log2_hc, d = a.d, half = d >> 1;
    const int f = (tid & (hc - 1)) * 8, apart = kAppendThreads >> a.log2_hc, first = tid >> a.log2_hc;
    const int heads = a.H + 2 * a.Hkv;  // queries, keys, values
    const int r0 = blockIdx.x * R, nr = min(R, a.rows - r0);
    if (tid < R) { s_row[tid].state = kNoRow; s_pos[tid] = -1; }
    griddep_wait();
    griddep_launch_dependents();

    // head h of rows r0 + i: where it lies and how far its rows are apart
    struct From { const IT *p; long long ld; };
    const auto from = [&](int h) {
        From s{(const IT *)a.q, a.ld_q};
        if (h >= a.H) {
            h -= a.H;
            s = {(const IT *)a.k, a.ld_k};
            if (h >= a.Hkv) {
                h -= a.Hkv;
                s = {(const IT *)a.v, a.ld_v};
            }
        }
        s.p += (long long)r0 * s.ld + h * d + f;
        return s;
    };
    Raw8<IT> lo[STEP], hi[STEP];
    const auto load = [&](const From &s, int i0) {
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            if (i0 + i >= nr) break;
            const IT *p = s.p + (i0 + i) * s.ld;
            lo[i] = get8(p);
            hi[i] = get8(p + half);
        }
    };
    From src = from(first);
    if (first < heads) load(src, 0);
    __syncthreads();
    for (int b = tid; b < a.batch; b += kAppendThreads) {
        const int begin = min(max(a.row_start[b], 0), a.rows), end = min(max(a.row_start[b + 1], 0), a.rows);
        const int kv = min(max(a.kv_len[b], 0), a.max_pages << a.log2_ps), slot = a.slots ? a.slots[b] : b;
        for (int i = max(begin - r0, 0); i < min(end - r0, nr); i++) {
            const int pos = max(kv - (end - r0 - i), -1);
            AppendRow row{-1, kNowhere};
            if (pos >= 0 && !(a.rope && pos >= a.rope_len)) {
                row.state = kLive;
                const int page = a.page_table[(long long)slot * a.max_pages + (pos >> a.log2_ps)];
                if ((unsigned)page < (unsigned)a.num_pages)
                    row.cell = ((((long long)page * a.Hkv) << a.log2_ps) + (pos & ((1 << a.log2_ps) - 1))) * d;
                s_pos[i] = pos;
            }
            s_row[i] = row;
        }
    }
    __syncthreads();
    if (a.rope)
        for (int i = tid; i < nr * half; i += kAppendThreads) {
            const int row = i / half, at = i - row * half, pos = s_pos[row];
            const float2 c = pos >= 0 ? a.rope[(long long)pos * half + at] : make_float2(0.f, 0.f);
            s_angles[row * d + at] = c.x;
            s_angles[row * d + half + at] = c.y;
        }
    __syncthreads();

    const int rounds = (heads + apart - 1) / apart;  // the same on every lane
    for (int n = 0; n < rounds; n++) {
        const int h = first + n * apart;
        const bool on = h < heads, isq = h < a.H, isv = h >= a.H + a.Hkv;
        const From next = from(h + apart);
        float wx[8], wy[8];
        if (a.mode != QW_QKNORM_NONE && on && !isv) {
            const float *w = (isq ? a.qn : a.kn) + f;
            widen8(get8(w), wx);
            widen8(get8(w + half), wy);
        }
        OT *to = isq ? (OT *)a.q_out + r0 * a.ld_q_out + h * d + f
                     : (OT *)(isv ? a.v_cache : a.k_cache) + ((long long)(h - a.H - (isv ? a.Hkv : 0)) << a.log2_ps) * d + f;
#pragma unroll
        for (int i0 = 0; i0 < R; i0 += STEP) {
            float x[STEP][8], y[STEP][8];
            float m[STEP];
#pragma unroll
            for (int i = 0; i < STEP; i++) {
                widen8(lo[i], x[i]);
                widen8(hi[i], y[i]);
                if (a.mode == QW_QKNORM_HEAD)
                    m[i] = rsqrtf(lanes_sum(on && i0 + i < nr ? squares(x[i], y[i]) : 0.f, hc) * a.inv_d + a.eps);
            }
            if (i0 + STEP < R) {
                if (on) load(src, i0 + STEP);
            } else if (h + apart < heads) {
                load(next, 0);
            }
            if (!on) continue;
#pragma unroll
            for (int i = 0; i < STEP; i++) {
                const int row = i0 + i;
                if (row >= nr) break;
                const AppendRow where = s_row[row];
                if (!isv) {
                    if (a.mode != QW_QKNORM_NONE) scale8(x[i], y[i], wx, wy, m[i]);
                    if (a.rope) {
                        float cs[8], sn[8];
                        widen8(get8(s_angles + row * d + f), cs);
                        widen8(get8(s_angles + row * d + half + f), sn);
                        turn8(x[i], y[i], cs, sn);
                    }
                }
                OT *at = isq ? to + row * a.ld_q_out : to + where.cell;
                if (isq && where.state == kNowhere) {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[i][e] = y[i][e] = 0.f;
                }
                if (isq ? a.q_out && where.state != kNoRow : where.cell >= 0 && where.state == kLive) {
                    set8(at, x[i]);
                    set8(at + half, y[i]);
                }
            }
        }
        src = next;
    }
}

template <typename IT, typename OT>
cudaError_t append_launch(const AppendArgs &a, cudaStream_t st) {
    // A CTA per row below, rows of one sequence: 592 of 32 / 8 heads from bf16 6.7 us (11.0 by fours), 1024 11.3 (11.8), 2048 17.0 (15.3);
    // of 14 / 2 heads of 64 from fp32, without norms, 3.7 (5.4), 6.0 (5.7), 10.2 (6.8).  Norms over whole vectors would read four rows twice: 91 us against 79.
    if (a.rows > kAppendFew && a.mode != QW_QKNORM_VECTOR)
        return launch_pdl(qw_kv_append_rows_kernel<IT, OT, kAppendRows>, dim3(a.rows / kAppendRows + (a.rows % kAppendRows != 0)), dim3(kAppendThreads),
                          kAppendRows * a.d * sizeof(float), st, a);
    return launch_pdl(qw_kv_append_row_kernel<IT, OT, 3>, dim3(a.rows), dim3(kAppendThreads), 0, st, a);
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
    a.num_pages = p->num_pages; a.max_pages = p->max_pages; a.mode = p->qk_norm; a.rope_len = p->rope_len; a.eps = (float)p->eps;
    a.inv_d = 1.0f / (float)a.d;
    while (16 << a.log2_hc < a.d) a.log2_hc++;
    while (1 << a.log2_ps < p->page_size) a.log2_ps++;
    const bool ib = p->in_dtype == QW_DTYPE_BF16, ob = p->dtype == QW_DTYPE_BF16;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = ib ? (ob ? append_launch<__nv_bfloat16, __nv_bfloat16>(a, st) : append_launch<__nv_bfloat16, float>(a, st))
                       : (ob ? append_launch<float, __nv_bfloat16>(a, st) : append_launch<float, float>(a, st));
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("append launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
