// fq_rope.hip -- bias, per-head norm and rotation of the QKV rows, keys and
// values to the paged cache.
//
// Bound by bandwidth: each element is read and written once (4095 tokens of 32 + 2 x 8
// heads of 128: 30.7 us, 185 MB at 6.0 TB/s; a large copy runs at 5.2, these inputs
// partly stay in the last-level cache), and by latency for one token (2.4 us).  A head is D / 8 lanes (of
// a group of the next power of two), each with two runs of four elements that hold whole
// pairs: (4p, rot/2 + 4p) for the half-split pairs, (8p, 8p + 4) for
// interleaved ones and past the rotated part, so that a rotation needs no other
// lane and the norm one reduction within the group.
#include <hip/hip_runtime.h>

#include "fq_step.h"

namespace fq {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

template <bool BF16>
__device__ __forceinline__ u16x4 narrow(f4 v) {  // to nearest, ties to even
    u16x4 r;
    for (int i = 0; i < 4; ++i)
        r[i] = BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v[i])
                    : __builtin_bit_cast(uint16_t, (_Float16)v[i]);
    return r;
}

template <int GS, bool BF16, bool INTER>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    const int heads = a.hq + 2 * a.hkv;
    const int64_t item = (int64_t)blockIdx.x * (256 / GS) + threadIdx.x / GS;
    if (item >= (int64_t)a.N * heads) return;
    const int n = (int)(item / heads), h = (int)(item % heads);
    const int p = threadIdx.x % GS;
    const bool on = 8 * p < a.D, turned = 8 * p < a.rot, isv = h >= a.hq + a.hkv;
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
        for (int o = 1; o < GS; o <<= 1) ss += __shfl_xor(ss, o, GS);
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
        const int pos = a.positions[n];
        const bool known = (unsigned)pos < (unsigned)a.table_rows;
        if (turned) {
            const float* cs = a.table + (int64_t)(known ? pos : 0) * a.rot + 4 * p;
            const f4 c = *(const f4u*)cs, s = *(const f4u*)(cs + a.rot / 2);
            const f4 y0 = x0, y1 = x1;
            for (int i = 0; i < 4; ++i) {
                if (INTER) {  // pairs (0, 1) (2, 3) of y0, then of y1
                    const f4 y = i < 2 ? y0 : y1;
                    const float u = y[2 * (i & 1)], v = y[2 * (i & 1) + 1];
                    const float t0 = u * c[i] - v * s[i], t1 = v * c[i] + u * s[i];
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
    if (!on) return;
    if (h < a.hq) {
        float* q = a.q + ((int64_t)n * a.hq + h) * a.D;
        *(f4u*)(q + d0) = x0;
        *(f4u*)(q + d1) = x1;
        return;
    }
    const int slot = a.slots[n];
    if (slot < 0 || (slot >> a.c.bs_log2) >= a.c.num_blocks) return;
    uint16_t* o = (isv ? a.v : a.k) + (slot >> a.c.bs_log2) * a.c.sb +
                  (slot & ((1 << a.c.bs_log2) - 1)) * a.c.st +
                  (h - a.hq - (isv ? a.hkv : 0)) * a.c.sh;
    *(u16x4*)(o + d0) = narrow<BF16>(x0);
    *(u16x4*)(o + d1) = narrow<BF16>(x1);
}

template <int GS>
hipError_t go(const RopeArgs& a, bool bf16, bool inter, hipStream_t st) {
    const int64_t items = (int64_t)a.N * (a.hq + 2 * a.hkv);
    const int64_t grid = (items + 256 / GS - 1) / (256 / GS);
    const dim3 g((unsigned)grid), t(256);
    if (bf16 && inter) hipLaunchKernelGGL((rope_kernel<GS, true, true>), g, t, 0, st, a);
    else if (bf16) hipLaunchKernelGGL((rope_kernel<GS, true, false>), g, t, 0, st, a);
    else if (inter) hipLaunchKernelGGL((rope_kernel<GS, false, true>), g, t, 0, st, a);
    else hipLaunchKernelGGL((rope_kernel<GS, false, false>), g, t, 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, bool bf16, bool interleaved, hipStream_t st) {
    const int lanes = a.D / 8;
    if (lanes <= 8) return go<8>(a, bf16, interleaved, st);
    if (lanes <= 16) return go<16>(a, bf16, interleaved, st);
    if (lanes <= 32) return go<32>(a, bf16, interleaved, st);
    return go<64>(a, bf16, interleaved, st);
}

}  // namespace fq
