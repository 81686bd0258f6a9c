// bf16 for the CUDA sources that the tests run on the host.
#pragma once
#include <stdint.h>
#include <string.h>

struct __nv_bfloat16 { uint16_t bits; };
struct __nv_bfloat162 { __nv_bfloat16 x, y; };
inline uint16_t host_bf16(float f) {
    uint32_t u;
    memcpy(&u, &f, 4);
    if ((u & 0x7F800000u) == 0x7F800000u && (u & 0x7FFFFFu)) return (uint16_t)(u >> 16 | 0x40);
    return (uint16_t)((u + 0x7FFFu + (u >> 16 & 1u)) >> 16);
}
inline __nv_bfloat162 __floats2bfloat162_rn(float lo, float hi) { return {{host_bf16(lo)}, {host_bf16(hi)}}; }
