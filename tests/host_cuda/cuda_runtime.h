// What the CUDA sources that the tests run on the host use of CUDA: a launch runs its CTAs one after the other, the threads of
// a CTA as coroutines that hand over at barriers and shuffles.  Loads and stores are the kernel's own, so that a buffer
// which ends at a page without access shows any that pass it.
#pragma once
#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>
#include <utility>
#include <vector>

#define __host__
#define __device__
#define __global__
#define __forceinline__ inline
#define __shared__ static
#define __align__(n) alignas(n)
#define __launch_bounds__(...)

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x = 1, unsigned y = 1, unsigned z = 1) : x(x), y(y), z(z) {}
};
struct alignas(8) float2 { float x, y; };
struct alignas(16) float4 { float x, y, z, w; };
struct alignas(8) uint2 { unsigned x, y; };
struct alignas(16) uint4 { unsigned x, y, z, w; };
inline float2 make_float2(float x, float y) { return {x, y}; }
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }
inline uint4 make_uint4(unsigned x, unsigned y, unsigned z, unsigned w) { return {x, y, z, w}; }
template <typename T> inline T min(T a, T b) { return b < a ? b : a; }
template <typename T> inline T max(T a, T b) { return a < b ? b : a; }
inline float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
inline uint32_t __float_as_uint(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
inline float rsqrtf(float x) { return 1.0f / sqrtf(x); }

inline dim3 threadIdx, blockIdx, blockDim, gridDim;
inline char *host_dynamic_shared;

// ---- the threads of the CTA that runs ----
struct HostThread {
    ucontext_t ctx;
    std::vector<char> stack;
    bool done;
};
inline std::vector<HostThread> host_threads;
inline ucontext_t host_main;
inline unsigned host_now;
struct HostBarrier {
    unsigned arrived = 0, phase = 0;
};
inline HostBarrier host_cta, host_warp[32];
inline float host_lanes[32][32];
inline unsigned host_live(unsigned from, unsigned to) {
    unsigned n = 0;
    for (unsigned t = from; t < to; t++) n += !host_threads[t].done;
    return n;
}
inline void host_hand_over() { swapcontext(&host_threads[host_now].ctx, &host_main); }
inline void host_meet(HostBarrier &b, unsigned from, unsigned to) {
    const unsigned phase = b.phase;
    b.arrived++;
    while (b.phase == phase) {
        if (b.arrived >= host_live(from, to)) {
            b.arrived = 0;
            b.phase++;
            break;
        }
        host_hand_over();
    }
}
inline void __syncthreads() { host_meet(host_cta, 0, blockDim.x); }
inline void __syncwarp() { host_meet(host_warp[host_now / 32], host_now / 32 * 32, host_now / 32 * 32 + 32); }
inline float __shfl_xor_sync(unsigned, float v, int o) {
    float *lanes = host_lanes[host_now / 32];
    lanes[host_now % 32] = v;
    __syncwarp();
    const float r = lanes[(host_now % 32) ^ o];
    __syncwarp();
    return r;
}

typedef int cudaError_t;
typedef void *cudaStream_t;
constexpr cudaError_t cudaSuccess = 0;
inline const char *cudaGetErrorString(cudaError_t) { return "launch"; }
inline cudaError_t cudaGetLastError() { return cudaSuccess; }
constexpr int cudaLaunchAttributeProgrammaticStreamSerialization = 0;
struct cudaLaunchAttribute {
    int id;
    struct { int programmaticStreamSerializationAllowed; } val;
};
struct cudaLaunchConfig_t {
    dim3 gridDim, blockDim;
    size_t dynamicSmemBytes;
    cudaStream_t stream;
    cudaLaunchAttribute *attrs;
    int numAttrs;
};
template <typename F> struct HostCall {
    static inline const F *body;
    static void enter() {
        (*body)();
        host_threads[host_now].done = true;
        host_hand_over();
    }
};
template <typename F> void host_run_cta(const F &body) {
    HostCall<F>::body = &body;
    for (auto &t : host_threads) {
        t.done = false;
        getcontext(&t.ctx);
        t.ctx.uc_stack.ss_sp = t.stack.data();
        t.ctx.uc_stack.ss_size = t.stack.size();
        makecontext(&t.ctx, HostCall<F>::enter, 0);
    }
    while (host_live(0, blockDim.x))
        for (host_now = 0; host_now < blockDim.x; host_now++)
            if (!host_threads[host_now].done) {
                threadIdx = dim3(host_now, 0, 0);
                swapcontext(&host_main, &host_threads[host_now].ctx);
            }
}
template <typename... K, typename... A>
cudaError_t cudaLaunchKernelEx(const cudaLaunchConfig_t *c, void (*kernel)(K...), A &&...args) {
    gridDim = c->gridDim;
    blockDim = c->blockDim;
    std::vector<char> shared(c->dynamicSmemBytes + 16);
    host_dynamic_shared = (char *)(((uintptr_t)shared.data() + 15) & ~(uintptr_t)15);
    host_threads.resize(blockDim.x);
    for (auto &t : host_threads) t.stack.resize(64 << 10);
    for (unsigned b = 0; b < gridDim.x; b++) {
        blockIdx = dim3(b, 0, 0);
        host_run_cta([&] { kernel(args...); });
    }
    return cudaSuccess;
}
