// fq_rope.h -- one head of a QKV row: bias, norm and rotation, D / 8 lanes (of a group
// of GS) with two runs of four elements each.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "fq_step.h"

namespace fq {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// f over the group's GS lanes, in each of them, by halves of pairs: within rows of 16 by data-parallel moves,
// beyond by swaps of rows.  (Of lanes that hold the same, which of them a move takes is the same.)
template <int GS, class F>
__device__ __forceinline__ float over_group(float x, F f) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const auto moved = [&](auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl.value, 0xF, 0xF, false));
    };
    x = f(x, moved(std::integral_constant<int, 0xB1>()));   // lanes 1 0 3 2 of each four
    x = f(x, moved(std::integral_constant<int, 0x4E>()));   // 2 3 0 1
    x = f(x, moved(std::integral_constant<int, 0x141>()));  // the other four of eight
    if constexpr (GS >= 16) x = f(x, moved(std::integral_constant<int, 0x140>()));  // the other eight of 16
    if constexpr (GS >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const u2 p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
        const uint32_t a = p[0], b = p[1];
        x = f(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    }
    if constexpr (GS >= 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const u2 p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(u, u, false, false));
        const uint32_t a = p[0], b = p[1];
        x = f(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    }
    return x;
}

// A lane's elements d0 .. d0+3 and d1 .. d1+3 of head h of token n (none where not on: lanes past
// D / 8 and those the caller leaves out, which still have their part in the norm's sums).  The
// runs hold whole pairs: (4p, rot/2 + 4p) for the half-split pairs, (8p, 8p + 4) for interleaved
// ones and past the rotated part.
struct HeadRuns {
    f4 x0, x1;
    int d0, d1;
};
template <int GS, bool INTER>
__device__ __forceinline__ HeadRuns head_runs(const RopeArgs& a, int n, int h, int p, bool on) {
    const bool turned = 8 * p < a.rot, isv = h >= a.hq + a.hkv;
    const int d0 = !INTER && turned ? 4 * p : 8 * p;
    const int d1 = !INTER && turned ? a.rot / 2 + 4 * p : 8 * p + 4;
    f4 x0 = 0.0f, x1 = 0.0f;
    if (on) {
        const float* x = a.qkv + n * a.ld + (int64_t)h * a.D;
        x0 = *(const f4u*)(x + d0);
        x1 = *(const f4u*)(x + d1);
        if (a.bias) {
            const float* bi = a.bias + (int64_t)h * a.D;
            x0 += *(const f4u*)(bi + d0);
            x1 += *(const f4u*)(bi + d1);
        }
    }
    const float* wt = isv ? nullptr : h < a.hq ? a.qw : a.kw;
    if (wt) {
        float ss = 0.0f;
        for (int i = 0; i < 4; ++i) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
        ss = over_group<GS>(ss, [](float u, float v) { return u + v; });
        const float r = 1.0f / sqrtf(ss / (float)a.D + a.eps);
        if (on) {
            const f4 w0 = *(const f4u*)(wt + d0), w1 = *(const f4u*)(wt + d1);
            for (int i = 0; i < 4; ++i) {
                x0[i] = x0[i] * r * w0[i];
                x1[i] = x1[i] * r * w1[i];
            }
        }
    }
    if (!isv) {
        const int pos = on ? a.positions[n] : 0;
        const bool known = (unsigned)pos < (unsigned)a.table_rows;
        if (turned) {
            const float* cs = a.table + (int64_t)(known ? pos : 0) * a.rot + 4 * p;
            const f4 c = *(const f4u*)cs, s = *(const f4u*)(cs + a.rot / 2);
            const f4 y0 = x0, y1 = x1;
            for (int i = 0; i < 4; ++i) {
                if (INTER) {  // pairs (0, 1) (2, 3) of y0, then of y1
                    const f4 y = i < 2 ? y0 : y1;
                    const float u = y[2 * (i & 1)], v = y[2 * (i & 1) + 1];
                    const float t0 = fmaf(u, c[i], -(v * s[i])), t1 = fmaf(u, s[i], v * c[i]);
                    if (i < 2) {
                        x0[2 * i] = t0, x0[2 * i + 1] = t1;
                    } else {
                        x1[2 * i - 4] = t0, x1[2 * i - 3] = t1;
                    }
                } else {
                    x0[i] = y0[i] * c[i] - y1[i] * s[i];
                    x1[i] = y1[i] * c[i] + y0[i] * s[i];
                }
            }
        }
        if (!known) x0 = x1 = __builtin_nanf("");
    }
    return {x0, x1, d0, d1};
}

}  // namespace fq
