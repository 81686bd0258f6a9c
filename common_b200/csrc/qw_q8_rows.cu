// qw_q8_rows.cu -- rows of numbers to rows of 8-bit codes with a scale each, alone (qw_op_quant_q8) or behind the residual's
// addition and the root-mean-square norm (qw_op_norm_q8).
//
// Codes of a row g with t = max|g|: rint(127 g / t), halves to even; scale t / 127.  For the norm y = h r w with
// r = 1 / sqrt(mean(h^2) + eps), the factor r > 0 cancels in the codes: they are those of g = h w, and only the scale,
// t r / 127, waits for the sum of squares.  So one pass over the row yields both reductions at once.
#include <cuda_runtime.h>
#include <string>
#include <type_traits>

#include "../../include/qwen3_b200.h"
#include "qw_internal.cuh"
#include "qw_ops.h"

namespace qw {
namespace {

// rows whose largest magnitude is below this are coded as zeros: 127 times the smallest normal number, so that neither
// 127 / t nor the scale of a row without a norm leaves the normal range
constexpr float kQ8Tiny = 127.0f * 1.17549435e-38f;

constexpr int kQ8MaxDim = 1 << 30;
constexpr int kFewRows = 296;  // two an SM: as many lanes a row as it has pieces
constexpr int kRowWarps = 16;  // of a row at most

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

// Codes by one multiplication: with m = 127 / t rounded to fp32, g m is within 127 * 2^-24 of 127 g / t, so that only next to a
// half of a code (kNearHalf, which is wider) the sides have to be told apart: 254 |g| against (2 k + 1) t, both exact in 64
// bits.  kMagic: a number whose neighbours are 1 apart, so that adding it rounds to whole numbers, halves to even, and leaves
// the code in the low bits.
constexpr float kNearHalf = 0.5f - 4e-5f, kMagic = 12582912.f;

// the code of g, where 127 |g| / t is that near to k + 1/2, k = floor(|g| m)
__device__ __forceinline__ int q8_code_near(float g, float m, float t) {
    const int k = (int)(fabsf(g) * m);
    const double lhs = 254.0 * (double)fabsf(g), rhs = (double)(2 * k + 1) * (double)t;
    const int r = k + (lhs > rhs || (lhs == rhs && (k & 1)));
    return g < 0.f ? -r : r;
}
__device__ __forceinline__ int q8_code(float g, float m, float t) {
    const float r = __fmaf_rn(g, m, kMagic), c = r - kMagic;
    return fabsf(__fmaf_rn(g, m, -c)) > kNearHalf ? q8_code_near(g, m, t) : (int)(int8_t)__float_as_int(r);
}

// two numbers at a time
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
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
__device__ __forceinline__ uint32_t low_bytes(uint64_t r0, uint64_t r1) {
    const float2 a = unpack2(r0), b = unpack2(r1);
    return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                       __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}
// The codes of four numbers, one to a byte.
__device__ __forceinline__ uint32_t q8_codes4(const float *g, float m, float t) {
    const uint64_t mm = pack2(m, m), magic = pack2(kMagic, kMagic), back = pack2(-kMagic, -kMagic), minus = pack2(-m, -m);
    const uint64_t g0 = pack2(g[0], g[1]), g1 = pack2(g[2], g[3]);
    const uint64_t r0 = fma2(g0, mm, magic), r1 = fma2(g1, mm, magic);
    const float2 d0 = unpack2(fma2(g0, minus, add2(r0, back))), d1 = unpack2(fma2(g1, minus, add2(r1, back)));  // code - value
    const float far = fmaxf(fmaxf(fabsf(d0.x), fabsf(d0.y)), fmaxf(fabsf(d1.x), fabsf(d1.y)));
    uint32_t codes = low_bytes(r0, r1);
    if (far > kNearHalf) {
        const float d[4] = {d0.x, d0.y, d1.x, d1.y};
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (fabsf(d[i]) > kNearHalf)
                codes = (codes & ~(0xFFu << (8 * i))) | (uint32_t)(q8_code_near(g[i], m, t) & 0xFF) << (8 * i);
    }
    return codes;
}
// The same for numbers of a bf16 row.  With 8 significant bits each, |g| = a 2^p and t = b 2^q, halves are common (0.2 % of a
// normal row's numbers: 127 g / t is 63.5 wherever g is t / 2), and nothing else comes near one: 254 a 2^(p - q) / b is odd or
// keeps v / (254 * 255) of v = 127 |g| / t from it.  So v is multiplied by 1 + 2^-20 and by 1 - 2^-20 (the roundings' 2^-23 are less,
// the distance is more): the two whole numbers are the same, or one to each side of a half, and the even one is the code.
__device__ __forceinline__ uint32_t q8_codes4_coarse(const float *g, float m) {
    const float up = m * (1.f + 0x1p-20f), down = m * (1.f - 0x1p-20f);
    const uint64_t uu = pack2(up, up), dd = pack2(down, down), magic = pack2(kMagic, kMagic);
    const uint64_t g0 = pack2(g[0], g[1]), g1 = pack2(g[2], g[3]);
    const uint32_t out = low_bytes(fma2(g0, uu, magic), fma2(g1, uu, magic)), in = low_bytes(fma2(g0, dd, magic), fma2(g1, dd, magic));
    const uint32_t odd = (out & 0x01010101u) * 255u;
    return (out & ~odd) | (in & odd);
}

// t / (127 sqrt(mean)), rounded to fp32 once: 1 / sqrt(mean), or t times it, may be outside fp32 where the scale is not
__device__ __forceinline__ float norm_scale(float t, double mean) { return (float)((double)t * rsqrt(mean) * (1.0 / 127.0)); }

// V consecutive numbers as they lie in memory, and as fp32
template <typename T, int V> struct Piece { uint32_t u[V * sizeof(T) / 4]; };
template <typename T, int V>
__device__ __forceinline__ Piece<T, V> get(const T *p, int n) {
    Piece<T, V> r;
    if (n >= V) {
        if constexpr (V * sizeof(T) == 8) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
            r.u[0] = w.x; r.u[1] = w.y;
        } else {
#pragma unroll
            for (int i = 0; i < (int)(V * sizeof(T) / 16); i++) {
                const uint4 w = reinterpret_cast<const uint4 *>(p)[i];
                r.u[4 * i] = w.x; r.u[4 * i + 1] = w.y; r.u[4 * i + 2] = w.z; r.u[4 * i + 3] = w.w;
            }
        }
    } else {  // behind the row: zeros
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; i++) r.u[i] = i < n ? reinterpret_cast<const uint32_t *>(p)[i] : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2)
                r.u[i / 2] = (i < n ? (uint32_t) reinterpret_cast<const uint16_t *>(p)[i] : 0u) |
                             (i + 1 < n ? (uint32_t) reinterpret_cast<const uint16_t *>(p)[i + 1] << 16 : 0u);
        }
    }
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void widen(const Piece<T, V> &p, float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = __uint_as_float(p.u[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) { v[i] = bf16lo(p.u[i / 2]); v[i + 1] = bf16hi(p.u[i / 2]); }
    }
}
template <typename T, int V>
__device__ __forceinline__ void put(T *p, const float (&v)[V], int n) {
    if (n >= V) {
        uint32_t u[V * sizeof(T) / 4];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; i++) u[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const __nv_bfloat162 w = __floats2bfloat162_rn(v[i], v[i + 1]);
                u[i / 2] = *reinterpret_cast<const uint32_t *>(&w);
            }
        }
        if constexpr (V * sizeof(T) == 8) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(u[0], u[1]);
        } else {
#pragma unroll
            for (int i = 0; i < (int)(V * sizeof(T) / 16); i++)
                reinterpret_cast<uint4 *>(p)[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) Elt<T>::store(p + i, v[i]);
    }
}
// the largest magnitude's bits; those of a NaN or an infinity are above all others
template <int V>
__device__ __forceinline__ unsigned top_of(const Piece<float, V> &p, unsigned top) {
#pragma unroll
    for (int i = 0; i < V; i++) top = max(top, p.u[i] & 0x7FFFFFFFu);
    return top;
}
template <int V>
__device__ __forceinline__ unsigned top_of(const Piece<__nv_bfloat16, V> &p, unsigned top) {
    unsigned t = 0;  // magnitudes of two numbers at a time, as whole numbers of 16 bits
#pragma unroll
    for (int i = 0; i < V / 2; i++) t = __vmaxu2(t, p.u[i] & 0x7FFF7FFFu);
    return max(top, max(t & 0xFFFF0000u, t << 16));
}

// A row per `wpr` warps, held in registers: NC pieces of V numbers a lane, piece j of a lane 32 * wpr pieces behind piece j - 1.
// One pass: the sum of squares and the largest magnitude in one exchange between the warps, codes from the registers.  Bound by
// HBM: the norm of 8192 x 4096 in fp32 with its sum written takes 64 us (6.8 TB/s), rows of 24576 x 4096 in fp32 73 us (6.9 TB/s),
// in bf16 46 us (6.5 TB/s), of 8192 x 12288 in bf16 49 us (6.2 TB/s).  One row takes 2 us, the launch and
// one chain of a load, an exchange and a store.  CTAs that stay and have the next row on its way were slower (68, 76 and 75 us): what
// the loads' latency costs, more small CTAs hide better than more registers.
template <typename XT, typename DT, bool NORM, int V, int NC>
__global__ void __launch_bounds__(32 * kRowWarps) qw_q8_rows_kernel(const Q8RowsArgs a, int wpr) {
    __shared__ unsigned s_top[kRowWarps];
    __shared__ double s_ss[kRowWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * ((blockDim.x >> 5) / wpr) + warp / wpr;
    const int first = ((warp % wpr) * 32 + lane) * V, step = wpr * 32 * V;
    const int left = r < a.rows ? a.dim - first : 0;  // numbers from this lane's first to the row's end
    griddep_wait();
    griddep_launch_dependents();
    Piece<std::conditional_t<NORM, float, XT>, V> g[NC];  // what is coded
    unsigned top = 0;
    double ss = 0.0;
    {
        Piece<XT, V> x[NC];
        const XT *xp = (const XT *)a.x + r * a.ld_x + first;
#pragma unroll
        for (int j = 0; j < NC; j++) x[j] = get<XT, V>(xp + j * step, left - j * step);
        if constexpr (NORM) {
            Piece<DT, V> d[NC];
            Piece<float, V> w[NC];
            const DT *dp = (const DT *)a.delta + r * a.ld_delta + first;
            XT *sp = (XT *)a.sum + r * a.ld_sum + first;
#pragma unroll
            for (int j = 0; j < NC; j++) d[j] = get<DT, V>(dp + j * step, a.delta ? left - j * step : 0);
#pragma unroll
            for (int j = 0; j < NC; j++) w[j] = get<float, V>(a.w + first + j * step, left - j * step);
            double s2 = 0.0;
#pragma unroll
            for (int j = 0; j < NC; j++) {
                float h[V], v[V];
                widen<XT, V>(x[j], h);
                widen<DT, V>(d[j], v);
#pragma unroll
                for (int e = 0; e < V; e++) h[e] = a.delta ? h[e] + v[e] : h[e];
                if (a.sum) put<XT, V>(sp + j * step, h, left - j * step);
                widen<float, V>(w[j], v);
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    ss += (double)h[e] * (double)h[e];
                    s2 += (double)h[e + 1] * (double)h[e + 1];
                    g[j].u[e] = __float_as_uint(__fmul_rn(h[e], v[e]));
                    g[j].u[e + 1] = __float_as_uint(__fmul_rn(h[e + 1], v[e + 1]));
                }
            }
            ss += s2;
        } else {
#pragma unroll
            for (int j = 0; j < NC; j++) g[j] = x[j];
        }
    }
#pragma unroll
    for (int j = 0; j < NC; j++) top = top_of<V>(g[j], top);
    top = __reduce_max_sync(0xffffffffu, top);
    if (NORM)
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (wpr > 1) {
        if (lane == 0) { s_top[warp] = top; s_ss[warp] = ss; }
        __syncthreads();
        const int at = warp / wpr * wpr + (lane & (wpr - 1));
        top = __reduce_max_sync(0xffffffffu, s_top[at]);
        if (NORM) {
            ss = s_ss[at];
            for (int o = wpr >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
    }
    if (left <= 0) return;
    const bool finite = top < 0x7F800000u;
    float t = __uint_as_float(top);
    if (t < kQ8Tiny) t = 0.f;
    const bool coded = finite && t > 0.f;
    const float m = coded ? __fdiv_rn(127.f, t) : 0.f;
    int8_t *q = a.q + r * a.ld_q + first;
#pragma unroll
    for (int j = 0; j < NC; j++) {
        const int n = left - j * step;
        if (n <= 0) break;
        float v[V];
        widen(g[j], v);
        uint32_t c[V / 4];
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            if constexpr (!NORM && sizeof(XT) == 2) c[e / 4] = coded ? q8_codes4_coarse(v + e, m) : 0u;
            else c[e / 4] = coded ? q8_codes4(v + e, m, t) : 0u;
        }
        if (n >= V) {
            if constexpr (V == 8) *reinterpret_cast<uint2 *>(q + j * step) = make_uint2(c[0], c[1]);
            else *reinterpret_cast<uint32_t *>(q + j * step) = c[0];
        } else {
#pragma unroll
            for (int e = 0; e < V; e++)
                if (e < n) q[j * step + e] = (int8_t)(c[e / 4] >> (8 * (e & 3)));
        }
    }
    if (first == 0) {
        a.scale[r] = coded ? (NORM ? norm_scale(t, ss / a.dim + a.eps) : t / 127.f) : finite ? 0.f : __uint_as_float(0x7FC00000u);
    }
}

// One CTA per row of any length and alignment: two passes over the row, the second from the caches, one number a load.  Bound by the
// loads: the norm of 8192 x 4095 takes 97 us in fp32 (64 for rows of 4096), 84 in bf16 (47); codes of 8192 x 12287 in bf16 98 (49).
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
        a.scale[r] = coded ? (NORM ? norm_scale(t, ss / a.dim + a.eps) : t / 127.f) : finite ? 0.f : __uint_as_float(0x7FC00000u);
    }
}

template <typename XT, typename DT, bool NORM, int V, int NC>
cudaError_t q8_rows_regs(const Q8RowsArgs &a, int wpr, cudaStream_t st) {
    const int warps = wpr < 4 ? 4 : wpr, rows = warps / wpr;
    return launch_pdl(qw_q8_rows_kernel<XT, DT, NORM, V, NC>, dim3(a.rows / rows + (a.rows % rows != 0)), dim3(32 * warps), 0, st, a, wpr);
}

template <typename XT, typename DT, bool NORM>
cudaError_t q8_rows_launch(const Q8RowsArgs &a, cudaStream_t st) {
    // pieces of 16 bytes of the widest type, so that every access of a warp is one contiguous piece
    constexpr int V = sizeof(XT) == 2 && (!NORM || sizeof(DT) == 2) ? 8 : 4;
    const auto apart = [](const void *p, long long ld, size_t esz) {
        return p && ((uintptr_t)p % (V * esz) || ld % V);
    };
    const bool vec = !apart(a.x, a.ld_x, sizeof(XT)) && !apart(a.delta, a.ld_delta, sizeof(DT)) && !apart(a.sum, a.ld_sum, sizeof(XT)) &&
                     !apart(a.q, a.ld_q, 1) && (uintptr_t)a.w % 16 == 0;
    // the norm holds its weights too: half the numbers fit its registers
    if (!vec || a.dim > (NORM ? 16384 : 32768)) return launch_pdl(qw_q8_rows_any_kernel<XT, DT, NORM>, dim3(a.rows), dim3(256), 0, st, a);
    // Few rows: as many lanes as there are pieces (64 x 4096: the norm of fp32 and bf16 2.7 us, 2.9 by the rule for many; bf16 rows 1.8 and
    // 2.3; at 256 rows 4.9 and 4.6, 2.5 both).  Many: so many numbers a lane that
    // the exchange between the warps is rare, and so few that several rows fit an SM: 16 beside delta and weights (8192 x 4096 in
    // fp32: 64 us, 69 with 8 or 32), 32 alone (24576 x 4096: 73 us, 81 with 16), 64 of bf16 (8192 x 12288: 49 us; with an exact comparison of halves behind it, 56, and 66 with 32).
    const int pieces = (a.dim + V - 1) / V, most = a.rows <= kFewRows ? 1 : NORM ? 16 / V : 8;
    int wpr = 1;
    while (wpr < kRowWarps && wpr * 32 * most < pieces) wpr *= 2;
    const int nc = (pieces + wpr * 32 - 1) / (wpr * 32);
    if (nc == 1) return q8_rows_regs<XT, DT, NORM, V, 1>(a, wpr, st);
    if (nc == 2) return q8_rows_regs<XT, DT, NORM, V, 2>(a, wpr, st);
    if (nc == 3) return q8_rows_regs<XT, DT, NORM, V, 3>(a, wpr, st);
    if (nc == 4) return q8_rows_regs<XT, DT, NORM, V, 4>(a, wpr, st);
    if constexpr (!NORM || V == 4) {
        if (nc <= 6) return q8_rows_regs<XT, DT, NORM, V, 6>(a, wpr, st);
        if (nc <= 8) return q8_rows_regs<XT, DT, NORM, V, 8>(a, wpr, st);
    }
    if constexpr (!NORM && V == 4) return q8_rows_regs<XT, DT, NORM, V, 16>(a, wpr, st);
    return cudaErrorInvalidValue;
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
    if (p->rows < 0 || p->dim < 1 || p->dim > kQ8MaxDim) return op_fail(QW_ERR_SHAPE, "rows >= 0 and dim in [1, 2^30]");
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
    if (p->sum && ((p->sum == p->x && a.ld_sum != a.ld_x) ||
                   (p->sum == p->delta && (a.ld_sum != a.ld_delta || p->x_dtype != p->delta_dtype))))
        return op_fail(QW_ERR_ARG, "sum may be x or delta only with the same type and stride");
    a.x = p->x; a.delta = p->delta; a.w = p->norm_w; a.sum = p->sum; a.q = p->q; a.scale = p->scale;
    a.rows = p->rows; a.dim = p->dim; a.eps = p->eps;
    // without a delta its type is the stream's, so that pieces are as wide as they can be
    const bool xb = p->x_dtype == QW_DTYPE_BF16, db = p->delta ? p->delta_dtype == QW_DTYPE_BF16 : xb;
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
    if (rows < 0 || dim < 1 || dim > kQ8MaxDim) return op_fail(QW_ERR_SHAPE, "rows >= 0 and dim in [1, 2^30]");
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
