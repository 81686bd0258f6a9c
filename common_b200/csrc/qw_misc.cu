// qw_misc.cu -- weight placement / conversion, synthetic initialisation, RoPE table, and the
// small reductions used around the tensor-parallel collectives.
#include "qw_internal.cuh"
#include "qw_kernels.h"
#include <float.h>
#include <limits.h>

namespace qw {

// dst[map(r) * ld + c] = convert(src[r * src_ld + c])  or the synthetic value of the full
// tensor's element (src_row0 + r, src_col0 + c).
template <typename DT>
__global__ void qw_place_kernel(const PlaceArgs p) {
    const size_t total = (size_t)p.rows * p.cols;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        int r = (int)(i / p.cols), c = (int)(i % p.cols);
        float v;
        if (p.synth) {
            size_t gidx = (size_t)(p.src_row0 + r) * p.full_cols + (p.src_col0 + c);
            v = p.constant_one ? 1.0f : synth_value(p.seed, p.tensor_id, gidx, p.scale);
        } else {
            size_t s = (size_t)r * p.src_ld + c;
            if (p.src_dtype == 0) v = reinterpret_cast<const float *>(p.src)[s];
            else if (p.src_dtype == 1) v = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(p.src)[s] << 16);
            else v = (float)reinterpret_cast<const double *>(p.src)[s];
        }
        int dr;
        if (p.row_map == 0) dr = p.dst_row0 + r;
        else {
            int blk = r / kGuBlock, w = r % kGuBlock;
            dr = blk * 2 * kGuBlock + (p.row_map == 2 ? kGuBlock : 0) + w;
        }
        Elt<DT>::store(reinterpret_cast<DT *>(p.dst) + (size_t)dr * p.dst_ld + c, v);
    }
}

cudaError_t place_launch(const PlaceArgs &p, cudaStream_t st) {
    size_t total = (size_t)p.rows * p.cols;
    if (!total) return cudaSuccess;
    int grid = (int)((total + 255) / 256);
    if (grid > 148 * 16) grid = 148 * 16;
    if (p.dst_bf16) qw_place_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
    else qw_place_kernel<float><<<grid, 256, 0, st>>>(p);
    return cudaGetLastError();
}

// freq[p][f] = (cos, sin)(p * exp(-2 f ln(theta) / d)), computed in fp64 like the reference's
// default precision (RotationFeatures.java:189-208), stored as fp32.
__global__ void qw_freq_kernel(float2 *freq, int seq_len, int half, double neg2lt_over_d) {
    size_t total = (size_t)seq_len * half;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        int p = (int)(i / half), f = (int)(i % half);
        double inv = exp((double)f * neg2lt_over_d);
        double ang = (double)p * inv;
        freq[i] = make_float2((float)cos(ang), (float)sin(ang));
    }
}

cudaError_t freq_launch(float2 *freq, int seq_len, int head_dim, double theta, cudaStream_t st) {
    int half = head_dim / 2;
    size_t total = (size_t)seq_len * half;
    int grid = (int)((total + 255) / 256);
    if (grid > 148 * 8) grid = 148 * 8;
    qw_freq_kernel<<<grid, 256, 0, st>>>(freq, seq_len, half, -2.0 * log(theta) / head_dim);
    return cudaGetLastError();
}

// Cross-rank greedy pick: (val, idx) gathered from every rank -> winner (ties -> smaller index).
__global__ void qw_argmax_merge_kernel(const float *vals, const int *idxs, int tp, int B, int *argmax_out,
                                    int *next_tokens, int *positions, int advance, int *hist, int hist_ld) {
    int b = threadIdx.x;
    if (b >= B) return;
    float bv = -FLT_MAX;
    int bi = INT_MAX;
    for (int r = 0; r < tp; r++) {
        float v = vals[r * B + b];
        int i = idxs[r * B + b];
        if (v > bv || (v == bv && i < bi)) { bv = v; bi = i; }
    }
    if (argmax_out) argmax_out[b] = bi;
    if (hist) hist[(size_t)b * hist_ld + positions[b] + 1] = bi;
    if (advance) {
        next_tokens[b] = bi;
        positions[b] += 1;
    }
}

cudaError_t argmax_merge_launch(const float *vals, const int *idxs, int tp, int B, int *argmax_out, int *next_tokens,
                                int *positions, int advance, int *hist, int hist_ld, cudaStream_t st) {
    qw_argmax_merge_kernel<<<1, 32 * ((B + 31) / 32), 0, st>>>(vals, idxs, tp, B, argmax_out, next_tokens, positions, advance,
                                                            hist, hist_ld);
    return cudaGetLastError();
}

// Per-rank sums of squares of the local q and k slices (whole-vector QK-norm under tensor
// parallelism; the caller all-reduces them).  out: (B, 2).
__global__ void qw_qk_sumsq_kernel(const float *qkv, int ld, int qw, int kw, float *out) {
    int b = blockIdx.x;
    const float *row = qkv + (size_t)b * ld;
    float sq = 0.f, sk = 0.f;
    for (int i = threadIdx.x; i < qw; i += blockDim.x) sq += row[i] * row[i];
    for (int i = threadIdx.x; i < kw; i += blockDim.x) sk += row[qw + i] * row[qw + i];
    __shared__ float s[2][32];
    sq = warp_sum(sq);
    sk = warp_sum(sk);
    int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (lane == 0) { s[0][w] = sq; s[1][w] = sk; }
    __syncthreads();
    if (threadIdx.x == 0) {
        float a = 0.f, c = 0.f;
        for (int i = 0; i < (int)(blockDim.x / 32); i++) { a += s[0][i]; c += s[1][i]; }
        out[b * 2 + 0] = a;
        out[b * 2 + 1] = c;
    }
}

cudaError_t qk_sumsq_launch(const float *qkv, int ld, int qw, int kw, int B, float *out, cudaStream_t st) {
    qw_qk_sumsq_kernel<<<B, 256, 0, st>>>(qkv, ld, qw, kw, out);
    return cudaGetLastError();
}

// x_out = x_in + part (residual after a tensor-parallel all-reduce), rows x n
__global__ void qw_add_kernel(float *out, const float *a, const float *b, size_t n) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
        out[i] = a[i] + b[i];
}
cudaError_t add_launch(float *out, const float *a, const float *b, size_t n, cudaStream_t st) {
    int grid = (int)((n + 255) / 256);
    if (grid > 148 * 8) grid = 148 * 8;
    if (grid < 1) grid = 1;
    qw_add_kernel<<<grid, 256, 0, st>>>(out, a, b, n);
    return cudaGetLastError();
}

// out[0, n) = 0 inside a chain of programmatically launched kernels (a memset node would end the
// chain): the accumulator of a split-K GEMM that follows.
__global__ void qw_zero_kernel(float4 *out, size_t n4) {
    griddep_launch_dependents();
    griddep_wait();  // the previous kernel may still read the buffer
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n4; i += (size_t)gridDim.x * blockDim.x)
        out[i] = make_float4(0.f, 0.f, 0.f, 0.f);
}
cudaError_t zero_launch(float *out, size_t n, cudaStream_t st) {
    if (n % 4 || (reinterpret_cast<uintptr_t>(out) & 15)) return cudaMemsetAsync(out, 0, n * sizeof(float), st);
    int grid = (int)((n / 4 + 255) / 256);
    if (grid > 148 * 4) grid = 148 * 4;
    if (grid < 1) grid = 1;
    return launch_pdl(qw_zero_kernel, dim3(grid), dim3(256), 0, st, reinterpret_cast<float4 *>(out), n / 4);
}

// h[t][p] = up * silu(gate), then gu = 0, for rows of the (2F) gate/up projection interleaved in blocks of 16 gate then 16 up
// rows, as the GEMM's SwiGLU epilogue computes it (same expression), h bf16 (T, F).
__global__ void qw_swiglu_rows_kernel(float *gu, int F, __nv_bfloat16 *h) {
    griddep_launch_dependents();
    griddep_wait();
    const int t = blockIdx.y;
    float *row = gu + (size_t)t * 2 * F;
    const int p = (blockIdx.x * blockDim.x + threadIdx.x) * 4;  // four pairs of one 16-row block
    if (p >= F) return;
    float4 *pg = reinterpret_cast<float4 *>(row + (p / kGuBlock) * 2 * kGuBlock + p % kGuBlock);
    const float4 g = pg[0], u = pg[kGuBlock / 4];
    pg[0] = make_float4(0.f, 0.f, 0.f, 0.f);  // zeroed again for the next split-K accumulation into this buffer
    pg[kGuBlock / 4] = make_float4(0.f, 0.f, 0.f, 0.f);
    uint2 o;
    o.x = (uint32_t)f2bf_bits(u.x * __fdividef(g.x, 1.0f + __expf(-g.x))) |
          ((uint32_t)f2bf_bits(u.y * __fdividef(g.y, 1.0f + __expf(-g.y))) << 16);
    o.y = (uint32_t)f2bf_bits(u.z * __fdividef(g.z, 1.0f + __expf(-g.z))) |
          ((uint32_t)f2bf_bits(u.w * __fdividef(g.w, 1.0f + __expf(-g.w))) << 16);
    *reinterpret_cast<uint2 *>(h + (size_t)t * F + p) = o;
}
cudaError_t swiglu_rows_launch(float *gu, int T, int F, __nv_bfloat16 *h, cudaStream_t st) {
    if (T < 1 || F < 1 || F % kGuBlock) return cudaErrorInvalidValue;
    const int bx = (F / 4 + 255) / 256;
    return launch_pdl(qw_swiglu_rows_kernel, dim3(bx, T), dim3(256), 0, st, gu, F, h);
}

// Bounded busy-wait of `ns` nanoseconds on the device (globaltimer), used to let the host
// run ahead of the GPU before a profiled sequence of launches.  Ends by itself.
__global__ void qw_hold_kernel(unsigned long long ns) {
    unsigned long long t0, t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    for (int i = 0; i < (1 << 24); i++) {
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
        if (t - t0 >= ns) break;
        __nanosleep(1000);
    }
}
cudaError_t hold_launch(unsigned long long ns, cudaStream_t st) {
    qw_hold_kernel<<<1, 32, 0, st>>>(ns);
    return cudaGetLastError();
}

__global__ void qw_gather_rows_kernel(float *out, const float *x, const float *part, const int *row, int D) {
    const int r = row[blockIdx.x];
    if (r < 0) return;
    for (int i = threadIdx.x * 4; i < D; i += blockDim.x * 4) {
        float4 v = *reinterpret_cast<const float4 *>(x + (size_t)r * D + i);
        if (part) {
            const float4 p = *reinterpret_cast<const float4 *>(part + (size_t)r * D + i);
            v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
        }
        *reinterpret_cast<float4 *>(out + (size_t)blockIdx.x * D + i) = v;
    }
}

cudaError_t gather_rows_launch(float *out, const float *x, const float *part, const int *row, int n, int D, cudaStream_t st) {
    qw_gather_rows_kernel<<<n, 256, 0, st>>>(out, x, part, row, D);
    return cudaGetLastError();
}

}  // namespace qw
