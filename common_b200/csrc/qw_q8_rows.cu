// qw_q8_rows.cu -- rows of numbers to rows of 8-bit codes with a scale each, alone (qw_op_quant_q8) or behind the residual's
// addition and the root-mean-square norm (qw_op_norm_q8).
//
// Codes of a row g with t = max|g|: rint(127 g / t), halves to even; scale t / 127.  For the norm y = h r w with
// r = 1 / sqrt(mean(h^2) + eps), the factor r > 0 cancels in the codes: they are those of g = h w, and only the scale,
// t r / 127, waits for the sum of squares.  So one pass over the row yields both reductions at once.
#include <cuda_runtime.h>
#include <string>

#include "../../include/qwen3_b200.h"
#include "qw_internal.cuh"
#include "qw_ops.h"

namespace qw {
namespace {

// rows whose largest magnitude is below this are coded as zeros: 127 times the smallest normal number, so that neither
// the scale nor 127 / t leaves the normal range
constexpr float kQ8Tiny = 127.0f * 1.17549435e-38f;

struct Q8RowsArgs {
    const void *x, *delta;
    const float *w;
    void *sum;
    int8_t *q;
    float *scale;
    long long ld_x, ld_delta, ld_sum, ld_q;
    int rows, dim;
    double eps;
};

// The code of g, given m = 127 / t rounded to fp32.  g m is within 4e-5 of 127 g / t (two roundings of numbers up to
// 127), so that only next to a half of a code the sides have to be told apart: 254 |g| against (2 k + 1) t, both exact
// in 64 bits.
__device__ __forceinline__ int q8_code(float g, float m, float t) {
    const float v = g * m, c = rintf(v);
    if (fabsf(fabsf(v - c) - 0.5f) > 4e-5f) return (int)c;
    const float k = floorf(fabsf(v));
    const double lhs = 254.0 * (double)fabsf(g), rhs = (double)(2.0f * k + 1.0f) * (double)t;
    const int low = (int)k, r = low + (lhs > rhs || (lhs == rhs && (low & 1)));
    return v < 0.f ? -r : r;
}

// One CTA per row of any length and alignment: two passes over the row, the second from the caches.
template <typename XT, typename DT, bool NORM>
__global__ void __launch_bounds__(256) qw_q8_rows_any_kernel(const Q8RowsArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ unsigned s_top[8];
    __shared__ double s_ss[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long r = blockIdx.x;
    const XT *x = (const XT *)a.x + r * a.ld_x;
    const DT *d = NORM && a.delta ? (const DT *)a.delta + r * a.ld_delta : nullptr;
    unsigned top = 0;
    double ss = 0.0;
    for (int i = tid; i < a.dim; i += 256) {
        float h = Elt<XT>::load(x + i);
        if (d) h += Elt<DT>::load(d + i);
        if (NORM) ss += (double)h * (double)h;
        const float g = NORM ? __fmul_rn(h, a.w[i]) : h;
        top = max(top, __float_as_uint(g) & 0x7FFFFFFFu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (NORM)
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) { s_top[warp] = top; s_ss[warp] = ss; }
    __syncthreads();
    top = s_top[0];
    ss = s_ss[0];
    for (int i = 1; i < 8; i++) { top = max(top, s_top[i]); ss += s_ss[i]; }
    const bool finite = top < 0x7F800000u;
    float t = __uint_as_float(top);
    if (t < kQ8Tiny) t = 0.f;
    const bool coded = finite && t > 0.f;
    const float m = coded ? __fdiv_rn(127.f, t) : 0.f;
    XT *sum = NORM && a.sum ? (XT *)a.sum + r * a.ld_sum : nullptr;
    int8_t *q = a.q + r * a.ld_q;
    for (int i = tid; i < a.dim; i += 256) {
        float h = Elt<XT>::load(x + i);
        if (d) h += Elt<DT>::load(d + i);
        const float g = NORM ? __fmul_rn(h, a.w[i]) : h;
        if (sum) Elt<XT>::store(sum + i, h);
        q[i] = coded ? (int8_t)q8_code(g, m, t) : 0;
    }
    if (tid == 0) {
        const float rms = NORM ? (float)(1.0 / sqrt(ss / a.dim + a.eps)) : 1.f;
        a.scale[r] = finite ? t * rms / 127.f : __uint_as_float(0x7FC00000u);
    }
}

template <typename XT, typename DT, bool NORM>
cudaError_t q8_rows_launch(const Q8RowsArgs &a, cudaStream_t st) {
    return launch_pdl(qw_q8_rows_any_kernel<XT, DT, NORM>, dim3(a.rows), dim3(256), 0, st, a);
}

size_t esize(int dtype) { return dtype == QW_DTYPE_BF16 ? 2 : 4; }
bool known(int dtype) { return dtype == QW_DTYPE_F32 || dtype == QW_DTYPE_BF16; }

}  // namespace
}  // namespace qw

using namespace qw;

extern "C" qw_status qw_op_norm_q8(const qw_norm_q8_args *p, void *stream) {
    if (!p) return op_fail(QW_ERR_ARG, "null arguments");
    if (!known(p->x_dtype) || (p->delta && !known(p->delta_dtype)))
        return op_fail(QW_ERR_UNSUPPORTED, "x and delta must be fp32 or bf16");
    if (p->rows < 0 || p->dim < 1) return op_fail(QW_ERR_SHAPE, "rows >= 0 and dim >= 1");
    if (!(p->eps >= 0.0)) return op_fail(QW_ERR_ARG, "eps must not be negative");
    Q8RowsArgs a{};
    a.ld_x = p->ld_x ? p->ld_x : p->dim; a.ld_delta = p->ld_delta ? p->ld_delta : p->dim;
    a.ld_sum = p->ld_sum ? p->ld_sum : p->dim; a.ld_q = p->ld_q ? p->ld_q : p->dim;
    if (a.ld_x < p->dim || a.ld_delta < p->dim || a.ld_sum < p->dim || a.ld_q < p->dim)
        return op_fail(QW_ERR_SHAPE, "row strides must cover dim");
    if (p->rows == 0) return QW_OK;
    if (!p->x || !p->norm_w || !p->q || !p->scale) return op_fail(QW_ERR_ARG, "null device pointer");
    const size_t ex = esize(p->x_dtype), ed = p->delta ? esize(p->delta_dtype) : 1;
    if ((uintptr_t)p->x % ex || (uintptr_t)p->sum % ex || (uintptr_t)p->delta % ed ||
        (((uintptr_t)p->norm_w | (uintptr_t)p->scale) & 3))
        return op_fail(QW_ERR_ARG, "pointers must be aligned to their elements");
    a.x = p->x; a.delta = p->delta; a.w = p->norm_w; a.sum = p->sum; a.q = p->q; a.scale = p->scale;
    a.rows = p->rows; a.dim = p->dim; a.eps = p->eps;
    const bool xb = p->x_dtype == QW_DTYPE_BF16, db = p->delta && p->delta_dtype == QW_DTYPE_BF16;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = xb ? (db ? q8_rows_launch<__nv_bfloat16, __nv_bfloat16, true>(a, st)
                             : q8_rows_launch<__nv_bfloat16, float, true>(a, st))
                       : (db ? q8_rows_launch<float, __nv_bfloat16, true>(a, st)
                             : q8_rows_launch<float, float, true>(a, st));
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("norm launch: ") + cudaGetErrorString(e));
    return QW_OK;
}

extern "C" qw_status qw_op_quant_q8(const void *x, int32_t x_dtype, int32_t rows, int32_t dim, int64_t ld_x, int8_t *q,
                                    int64_t ld_q, float *scale, void *stream) {
    if (!known(x_dtype)) return op_fail(QW_ERR_UNSUPPORTED, "x must be fp32 or bf16");
    if (rows < 0 || dim < 1) return op_fail(QW_ERR_SHAPE, "rows >= 0 and dim >= 1");
    Q8RowsArgs a{};
    a.ld_x = ld_x ? ld_x : dim; a.ld_q = ld_q ? ld_q : dim;
    if (a.ld_x < dim || a.ld_q < dim) return op_fail(QW_ERR_SHAPE, "row strides must cover dim");
    if (rows == 0) return QW_OK;
    if (!x || !q || !scale) return op_fail(QW_ERR_ARG, "null device pointer");
    if ((uintptr_t)x % esize(x_dtype) || ((uintptr_t)scale & 3))
        return op_fail(QW_ERR_ARG, "pointers must be aligned to their elements");
    a.x = x; a.q = q; a.scale = scale; a.rows = rows; a.dim = dim;
    cudaError_t e = x_dtype == QW_DTYPE_BF16 ? q8_rows_launch<__nv_bfloat16, float, false>(a, (cudaStream_t)stream)
                                             : q8_rows_launch<float, float, false>(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("quantisation launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
