// fq_group8.h -- what enters a cache of 8 bits: codes and the scale of 16 tokens.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fq {

constexpr float TINY = 1.1754943508222875e-38f;  // 2^-126: scales below it are as 0

// One over a group's scale; 0 where the scale is as 0.
__device__ __forceinline__ float inverse_of(float s) { return s >= TINY && s < __builtin_inff() ? 1.0f / s : 0.0f; }

// A scale read from a cache: 0 where it is no positive finite number.
__device__ __forceinline__ float held_scale(float s) { return s > 0.0f && s < __builtin_inff() ? s : 0.0f; }

// x / scale to the nearest code (ties to even), held to -127 .. 127; NaN: 0.
__device__ __forceinline__ int code_of(float x, float inverse) {
    const float y = x * inverse;  // (an infinity times 0 is NaN as well)
    return y == y ? (int)rintf(fminf(fmaxf(y, -127.0f), 127.0f)) : 0;
}
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, float inverse) {
    return (uint32_t)(code_of(a, inverse) & 255) | (uint32_t)(code_of(b, inverse) & 255) << 8 |
           (uint32_t)(code_of(c, inverse) & 255) << 16 | (uint32_t)code_of(d, inverse) << 24;
}
__device__ __forceinline__ float code_at(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

// The largest finite magnitude so far.
__device__ __forceinline__ float largest(float m, float x) {
    x = fabsf(x);
    return x < __builtin_inff() ? fmaxf(m, x) : m;
}

// Four codes under another scale: times = old scale * (1 / new scale).
__device__ __forceinline__ uint32_t again(uint32_t w, float times) {
    return four_codes(code_at(w, 0), code_at(w, 1), code_at(w, 2), code_at(w, 3), times);
}

}  // namespace fq
