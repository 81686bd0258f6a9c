// qw_kv_pages.cu -- moving rows of the paged KV cache of every layer in one launch: page copies (the partly filled
// page of a forked sequence, whole pages of a duplicated one) and compaction (the kept positions of a sequence
// gathered into new pages, their keys turned to the positions they take).
//
// Cache layout: [layer][page][kv_head][page_size][head_dim]; one (layer, page, head) holds page_size contiguous
// rows.  Both operators are bound by HBM: every row is read once and written once.
#include <cuda_runtime.h>
#include <string>

#include "../../include/qwen3_b200.h"
#include "qw_internal.cuh"
#include "qw_ops.h"

namespace qw {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kCompactThreads = 128, kCompactRows = 8;

// One CTA per (page pair, layer, K or V, head): rows [0, n) of the head are contiguous in both pages.  Bound by HBM: 6.7 TB/s
// where whole pages move (453 us for 3.0 GB), the launch where a few do (4.7 us for 4 pages of 28 layers).
__global__ void __launch_bounds__(kCopyThreads)
    qw_kv_copy_kernel(uint4 *kp, uint4 *vp, int layers, int num_pages, int heads, int ps, int row_vec, const int *src,
                      const int *dst, const int *rows) {
    const int pair = blockIdx.x;
    const int s = src[pair], d = dst[pair];
    if ((unsigned)s >= (unsigned)num_pages || (unsigned)d >= (unsigned)num_pages || s == d) return;
    const int n = rows ? min(max(rows[pair], 0), ps) * row_vec : ps * row_vec;
    const int u = blockIdx.y;  // (layer, K or V, head)
    const int head = u % heads, kv = (u / heads) & 1, layer = u / heads / 2;
    uint4 *base = kv ? vp : kp;
    const size_t unit = (size_t)ps * row_vec;
    const uint4 *from = base + (((size_t)layer * num_pages + s) * heads + head) * unit;
    uint4 *to = base + (((size_t)layer * num_pages + d) * heads + head) * unit;
    for (int i = threadIdx.x; i < n; i += kCopyThreads) to[i] = from[i];
}

// turn 8 pairs (x, y) back by the table's angles: (x cos + y sin, y cos - x sin), in fp32, rounded once; `up` holds the sign bit
// alone where they turn forward
__device__ __forceinline__ void turn_back(float (&x)[8], float (&y)[8], const float2 *cs, int up) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float2 c = cs[e];
        const float s = __int_as_float(__float_as_int(c.y) ^ up), a = x[e] * c.x + y[e] * s;
        y[e] = y[e] * c.x - x[e] * s;
        x[e] = a;
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    v[0] = bf16lo(u.x); v[1] = bf16hi(u.x); v[2] = bf16lo(u.y); v[3] = bf16hi(u.y);
    v[4] = bf16lo(u.z); v[5] = bf16hi(u.z); v[6] = bf16lo(u.w); v[7] = bf16hi(u.w);
}
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    return (uint32_t)f2bf_bits(lo) | (uint32_t)f2bf_bits(hi) << 16;
}
__device__ __forceinline__ void put8(__nv_bfloat16 *p, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ void put8(float *p, const float (&v)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

struct CompactArgs {
    void *k, *v;
    int layers, num_pages, heads, ps, log2_ps, d;
    const int *src_table, *dst_table;
    int max_pages;
    const int *keep, *keep_start, *dst_base;
    int batch, rows;
    const float2 *rope;
    int rope_len;
};

// where a kept row lies and where it goes, as element offsets within one layer and head 0
struct RowMove {
    long long from, to;
    const float2 *turn;  // the table's angles of the distance; null: keys stay as they are
    int up;              // the sign bit where it moves up
    int skip;            // nothing to do
};

__device__ __forceinline__ RowMove row_move(const CompactArgs &a, int r) {
    RowMove m{0, 0, nullptr, 0, 1};
    if (r >= a.rows) return m;
    // the sequence that row r belongs to: the last b with keep_start[b] <= r
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.keep_start[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    const int i = r - a.keep_start[lo];
    if (i < 0 || r >= a.keep_start[lo + 1]) return m;
    const int come = a.keep[r], to = (a.dst_base ? a.dst_base[lo] : 0) + i;
    const int cp = come >> a.log2_ps, tp = to >> a.log2_ps;
    if (come < 0 || to < 0 || cp >= a.max_pages || tp >= a.max_pages) return m;
    const int sp = a.src_table[(size_t)lo * a.max_pages + cp], dp = a.dst_table[(size_t)lo * a.max_pages + tp];
    if ((unsigned)sp >= (unsigned)a.num_pages || (unsigned)dp >= (unsigned)a.num_pages) return m;
    const int distance = abs(come - to);
    if (a.rope && distance >= a.rope_len) return m;  // the table has no angle for it
    if (a.rope && distance) m.turn = a.rope + (size_t)distance * (a.d / 2);
    m.skip = 0;
    m.up = (come - to) & (int)0x80000000;
    const long long page = (long long)a.heads * a.ps * a.d;
    m.from = sp * page + (long long)(come & (a.ps - 1)) * a.d;
    m.to = dp * page + (long long)(to & (a.ps - 1)) * a.d;
    return m;
}

// 8 elements as they lie in memory
template <typename T> struct Raw8 { uint4 v[sizeof(T) / 2]; };
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16> &r, float (&v)[8]) {
    const uint4 u = r.v[0];
    v[0] = bf16lo(u.x); v[1] = bf16hi(u.x); v[2] = bf16lo(u.y); v[3] = bf16hi(u.y);
    v[4] = bf16lo(u.z); v[5] = bf16hi(u.z); v[6] = bf16lo(u.w); v[7] = bf16hi(u.w);
}
__device__ __forceinline__ void unpack8(const Raw8<float> &r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        v[4 * i] = __uint_as_float(r.v[i].x); v[4 * i + 1] = __uint_as_float(r.v[i].y);
        v[4 * i + 2] = __uint_as_float(r.v[i].z); v[4 * i + 3] = __uint_as_float(r.v[i].w);
    }
}
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw(const T *p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.v[i] = reinterpret_cast<const uint4 *>(p)[i];
    return r;
}
template <typename T>
__device__ __forceinline__ void store_raw(T *p, const Raw8<T> &r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4 *>(p)[i] = r.v[i];
}

// One CTA per (kCompactRows kept rows, layer).  The rows' places are looked up once; a warp then takes a head at a time: its rows
// are one contiguous piece of a destination page (mostly of a source page too).  A lane takes 8 elements of a row's first
// half and the matching 8 of its second (the rotary pairs), HV lanes a row, and has U rows of keys and values on the way.
// Bound by HBM: 3.74 GB moved at 6.4 TB/s (582 us; 28 layers, 8 heads of 128, bf16), 337 MB at 5.9 TB/s (57 us), where the last
// CTAs and the launch show; 7.5 GB in fp32 at 6.2 TB/s (1200 us); at head size 64 1.87 GB in bf16 at 5.7 TB/s (328 us) and 3.74 GB in
// fp32 at 6.3 TB/s (590 us).  What counts is loads in flight per SM and small CTAs to end on: 2 rows a lane in 4 CTAs of
// 256 threads (64 registers) against 4 rows in 2 CTAs (113 registers) take 604 against 724 us; 128 threads and 8 rows a
// CTA 592 and 57.3, 256 threads and 16 rows 604 and 57.3, 128 and 16 590 and 59.8, 256 and 8 652 and 56.7; the
// turns' arithmetic hides behind the loads.
template <typename T, int HV, int U>
__global__ void __launch_bounds__(kCompactThreads, 8) qw_kv_compact_kernel(const CompactArgs a) {
    constexpr int ROWS = kCompactRows, STEP = 32 / HV, HALF = HV * 8;
    static_assert(ROWS % (U * STEP) == 0, "rows of a warp's round");
    __shared__ RowMove moves[ROWS];
    for (int i = threadIdx.x; i < ROWS; i += blockDim.x) moves[i] = row_move(a, blockIdx.x * ROWS + i);
    __syncthreads();
    const int lane = threadIdx.x & 31, c = (lane % HV) * 8;
    const size_t layer = (size_t)blockIdx.y * a.num_pages * a.heads * a.ps * a.d, head = (size_t)a.ps * a.d;
    for (int h = threadIdx.x >> 5; h < a.heads; h += blockDim.x >> 5) {
        T *k = reinterpret_cast<T *>(a.k) + layer + h * head + c, *v = reinterpret_cast<T *>(a.v) + layer + h * head + c;
        for (int r0 = lane / HV; r0 < ROWS; r0 += U * STEP) {
            Raw8<T> q[U][4];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const RowMove &m = moves[r0 + u * STEP];
                if (m.skip) continue;
                q[u][0] = load_raw(k + m.from);
                q[u][1] = load_raw(k + m.from + HALF);
                q[u][2] = load_raw(v + m.from);
                q[u][3] = load_raw(v + m.from + HALF);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const RowMove &m = moves[r0 + u * STEP];
                if (m.skip) continue;
                store_raw(v + m.to, q[u][2]);
                store_raw(v + m.to + HALF, q[u][3]);
                if (m.turn) {
                    float x[8], y[8];
                    unpack8(q[u][0], x);
                    unpack8(q[u][1], y);
                    turn_back(x, y, m.turn + c, m.up);
                    put8(k + m.to, x);
                    put8(k + m.to + HALF, y);
                } else {
                    store_raw(k + m.to, q[u][0]);
                    store_raw(k + m.to + HALF, q[u][1]);
                }
            }
        }
    }
}

// Head sizes other than 64 and 128: one warp per (kept row, layer).
template <typename T>
__global__ void __launch_bounds__(kCompactThreads) qw_kv_compact_any_kernel(const CompactArgs a) {
    const RowMove m = row_move(a, blockIdx.x * (kCompactThreads / 32) + (threadIdx.x >> 5));
    if (m.skip) return;
    const int lane = threadIdx.x & 31, half = a.d / 2, hv = half / 8;
    const size_t layer = (size_t)blockIdx.y * a.num_pages * a.heads * a.ps * a.d, head = (size_t)a.ps * a.d;
    T *k = reinterpret_cast<T *>(a.k) + layer, *v = reinterpret_cast<T *>(a.v) + layer;
    for (int u = lane; u < a.heads * hv; u += 32) {
        const size_t at = (u / hv) * head + (u % hv) * 8;
        float x[8], y[8], vx[8], vy[8];
        load8(k + m.from + at, x);
        load8(k + m.from + at + half, y);
        load8(v + m.from + at, vx);
        load8(v + m.from + at + half, vy);
        if (m.turn) turn_back(x, y, m.turn + (u % hv) * 8, m.up);
        put8(k + m.to + at, x);
        put8(k + m.to + at + half, y);
        put8(v + m.to + at, vx);
        put8(v + m.to + at + half, vy);
    }
}

template <typename T>
void compact_launch(const CompactArgs &a, cudaStream_t st) {
    const int threads = 32 * (a.heads < kCompactThreads / 32 ? a.heads : kCompactThreads / 32);
    if (a.d == 128)
        qw_kv_compact_kernel<T, 8, sizeof(T) == 2 ? 2 : 1><<<dim3((a.rows + kCompactRows - 1) / kCompactRows, a.layers), threads, 0, st>>>(a);
    else if (a.d == 64)
        qw_kv_compact_kernel<T, 4, 1><<<dim3((a.rows + kCompactRows - 1) / kCompactRows, a.layers), threads, 0, st>>>(a);
    else
        qw_kv_compact_any_kernel<T><<<dim3((a.rows + kCompactThreads / 32 - 1) / (kCompactThreads / 32), a.layers),
                                      kCompactThreads, 0, st>>>(a);
}

int log2_exact(int x) {
    int l = 0;
    while ((1 << l) < x) l++;
    return l;
}

qw_status check_pool(const qw_kv_pool *p) {
    if (!p || !p->k || !p->v) return op_fail(QW_ERR_ARG, "null cache pool");
    if (((uintptr_t)p->k | (uintptr_t)p->v) & 15) return op_fail(QW_ERR_ARG, "cache pools must be 16-byte aligned");
    if (p->dtype != QW_DTYPE_F32 && p->dtype != QW_DTYPE_BF16) return op_fail(QW_ERR_UNSUPPORTED, "cache dtype");
    if (p->layers < 1 || p->num_pages < 1 || p->kv_heads < 1 || p->head_dim < 16 || p->head_dim % 16)
        return op_fail(QW_ERR_SHAPE, "layers, pages, heads >= 1 and head_dim a positive multiple of 16");
    if (p->page_size < 1 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
        return op_fail(QW_ERR_SHAPE, "page_size must be a power of two up to 256");
    if ((long long)p->layers * 2 * p->kv_heads > 65535) return op_fail(QW_ERR_SHAPE, "layers x KV heads beyond 32767");
    return QW_OK;
}

}  // namespace
}  // namespace qw

using namespace qw;

extern "C" qw_status qw_op_kv_copy_pages(const qw_kv_pool *pool, const int32_t *src, const int32_t *dst,
                                         const int32_t *rows, int32_t n, void *stream) {
    qw_status s = check_pool(pool);
    if (s) return s;
    if (n < 0) return op_fail(QW_ERR_SHAPE, "n must not be negative");
    if (n == 0) return QW_OK;
    if (!src || !dst) return op_fail(QW_ERR_ARG, "null device pointer");
    const int row_vec = pool->head_dim * (pool->dtype == QW_DTYPE_F32 ? 4 : 2) / 16;
    qw_kv_copy_kernel<<<dim3(n, pool->layers * 2 * pool->kv_heads), kCopyThreads, 0, (cudaStream_t)stream>>>(
        (uint4 *)pool->k, (uint4 *)pool->v, pool->layers, pool->num_pages, pool->kv_heads, pool->page_size, row_vec, src,
        dst, rows);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("page copy launch: ") + cudaGetErrorString(e));
    return QW_OK;
}

extern "C" qw_status qw_op_kv_compact(const qw_kv_pool *pool, const int32_t *src_table, const int32_t *dst_table,
                                      int32_t max_pages, const int32_t *keep, const int32_t *keep_start,
                                      const int32_t *dst_base, int32_t batch, int32_t rows, const float *rope,
                                      int32_t rope_len, void *stream) {
    qw_status s = check_pool(pool);
    if (s) return s;
    if (batch < 1 || max_pages < 1 || rows < 0) return op_fail(QW_ERR_SHAPE, "batch, max_pages >= 1 and rows >= 0");
    if (rope && rope_len < 1) return op_fail(QW_ERR_SHAPE, "rope_len must be positive");
    if (rows == 0) return QW_OK;
    if (!src_table || !dst_table || !keep || !keep_start) return op_fail(QW_ERR_ARG, "null device pointer");
    if ((uintptr_t)rope & 15) return op_fail(QW_ERR_ARG, "rope must be 16-byte aligned");
    CompactArgs a{};
    a.k = pool->k; a.v = pool->v; a.layers = pool->layers; a.num_pages = pool->num_pages; a.heads = pool->kv_heads;
    a.ps = pool->page_size; a.log2_ps = log2_exact(pool->page_size); a.d = pool->head_dim;
    a.src_table = src_table; a.dst_table = dst_table; a.max_pages = max_pages;
    a.keep = keep; a.keep_start = keep_start; a.dst_base = dst_base; a.batch = batch; a.rows = rows;
    a.rope = (const float2 *)rope; a.rope_len = rope_len;
    if (pool->dtype == QW_DTYPE_F32) compact_launch<float>(a, (cudaStream_t)stream);
    else compact_launch<__nv_bfloat16>(a, (cudaStream_t)stream);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("compaction launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
