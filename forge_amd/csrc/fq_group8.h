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

// x / scale to the nearest code (ties to even), held to -127 .. 127; NaN (an infinity times 0
// as well): 0, as the conversion has it, which also holds what is beyond integers to their ends.
__device__ __forceinline__ int code_of(float x, float inverse) {
    int i;
    asm("v_cvt_i32_f32 %0, %1" : "=v"(i) : "v"(rintf(x * inverse)));
    return min(max(i, -127), 127);
}
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, float inverse) {
    const uint32_t ab = __builtin_amdgcn_perm(code_of(b, inverse), code_of(a, inverse), 0x0C0C0400u);
    return __builtin_amdgcn_perm(code_of(d, inverse), code_of(c, inverse), 0x04000C0Cu) | ab;
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
