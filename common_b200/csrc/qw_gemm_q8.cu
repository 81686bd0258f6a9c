// qw_gemm_q8.cu -- products of 8-bit codes (qw_op_linear_q8): s(t, f) = sum_j w(f, j) x(t, j) in 32-bit integers, then
// y = s w_scale(f) x_scale(t) and the epilogue (bias, residual, SwiGLU).
#include <cuda_runtime.h>
#include <string>

#include "../../include/qwen3_b200.h"
#include "qw_internal.cuh"
#include "qw_ops.h"

namespace qw {
namespace {

constexpr int kQ8MaxK = 131071;  // |s| <= 128 * 128 * k < 2^31 for any codes

struct Q8GemmArgs {
    const int8_t *w, *x;
    const float *w_scale, *x_scale, *bias, *resid;
    void *out;
    int *err;
    long long ld_w, ld_x, ld_resid, ld_out;
    int M, K, T, epi, bf16;
};

// 64 features x 64 tokens per CTA, 4 x 4 sums per thread, dp4a on codes in shared memory.
__global__ void __launch_bounds__(256) qw_q8_gemm_simple_kernel(const Q8GemmArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ int sw[64][9], sx[64][9];
    __shared__ float sy[64][65];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int f0 = blockIdx.x * 64, t0 = blockIdx.y * 64;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 32) {
        for (int i = tid; i < 64 * 8; i += 256) {
            const int r = i >> 3, c = (i & 7) * 4, kk = k0 + c;
            const int left = a.K - kk;
            const unsigned mask = left >= 4 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
            int vw = 0, vx = 0;
            if (mask && f0 + r < a.M) vw = *reinterpret_cast<const int *>(a.w + (long long)(f0 + r) * a.ld_w + kk) & mask;
            if (mask && t0 + r < a.T) vx = *reinterpret_cast<const int *>(a.x + (long long)(t0 + r) * a.ld_x + kk) & mask;
            sw[r][i & 7] = vw;
            sx[r][i & 7] = vx;
        }
        __syncthreads();
        for (int c = 0; c < 8; c++) {
            int wv[4], xv[4];
            for (int i = 0; i < 4; i++) { wv[i] = sw[tx + 16 * i][c]; xv[i] = sx[ty + 16 * i][c]; }
            for (int i = 0; i < 4; i++)
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(wv[j], xv[i], acc[i][j]);
        }
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int f = f0 + tx + 16 * j, t = t0 + ty + 16 * i;
            float y = 0.f;
            if (f < a.M && t < a.T) y = (float)acc[i][j] * a.w_scale[f] * a.x_scale[t];
            sy[ty + 16 * i][tx + 16 * j] = y;
        }
    __syncthreads();
    for (int i = tid; i < 64 * 64; i += 256) {
        const int t = t0 + i / 64, c = i % 64, f = f0 + c;
        if (t >= a.T || f >= a.M) continue;
        float y = sy[i / 64][c];
        if (a.epi == QW_LINEAR_SWIGLU) {
            if (c % 32 >= 16) continue;
            const float u = sy[i / 64][c + 16];
            y = u * (y / (1.0f + expf(-y)));
            reinterpret_cast<__nv_bfloat16 *>(a.out)[t * a.ld_out + f0 / 2 + c / 32 * 16 + c % 16] = __float2bfloat16_rn(y);
        } else {
            if (a.epi == QW_LINEAR_RESID) y = a.resid[t * a.ld_resid + f] + y;
            else if (a.bias) y += a.bias[f];
            if (a.bf16) reinterpret_cast<__nv_bfloat16 *>(a.out)[t * a.ld_out + f] = __float2bfloat16_rn(y);
            else reinterpret_cast<float *>(a.out)[t * a.ld_out + f] = y;
        }
    }
}

cudaError_t q8_gemm_launch(const Q8GemmArgs &a, cudaStream_t st) {
    return launch_pdl(qw_q8_gemm_simple_kernel, dim3((a.M + 63) / 64, (a.T + 63) / 64), dim3(256), 0, st, a);
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
    a.ld_w = p->ld_w ? p->ld_w : p->k; a.ld_x = p->ld_x ? p->ld_x : p->k;
    a.ld_out = p->ld_out ? p->ld_out : cols; a.ld_resid = p->ld_resid ? p->ld_resid : cols;
    if (a.ld_w < p->k || a.ld_x < p->k || a.ld_w % 16 || a.ld_x % 16 || a.ld_w >= 1ll << 31 || a.ld_x >= 1ll << 31)
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
    a.w = p->w; a.x = p->x; a.w_scale = p->w_scale; a.x_scale = p->x_scale; a.bias = p->bias; a.resid = p->resid;
    a.out = p->out; a.err = p->err; a.M = p->n_out; a.K = p->k; a.T = p->t; a.epi = p->epi;
    a.bf16 = p->out_dtype == QW_DTYPE_BF16;
    cudaError_t e = q8_gemm_launch(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_fail(QW_ERR_CUDA, std::string("linear launch: ") + cudaGetErrorString(e));
    return QW_OK;
}
