// fq_attn8.hip -- attention with a sliding window, or over a cache of 8 bits.
//
// A wave takes one token and one query head and walks the keys it sees, 64 at a time.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fq_group8.h"
#include "fq_step.h"

namespace fq {
namespace {

template <int TYPE>
__device__ __forceinline__ float element(const uint8_t* base, int64_t at) {
    if (TYPE == 2) return (float)((const int8_t*)base)[at];
    const uint16_t b = ((const uint16_t*)base)[at];
    return TYPE == 1 ? __uint_as_float((uint32_t)b << 16) : (float)__builtin_bit_cast(_Float16, b);
}

template <int TYPE>
__global__ __launch_bounds__(64) void window_kernel(AttnArgs a, int D) {
    __shared__ float s_q[256], s_p[64];
    __shared__ int s_slot[64];
    const int n = blockIdx.x / a.hq, h = blockIdx.x % a.hq, lane = threadIdx.x, kvh = h / a.G;
    int b = 0, hi = a.B;
    while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (a.cu[mid] <= n) b = mid;
        else hi = mid;
    }
    const int t0 = min(max(a.cu[b], 0), a.N), t1 = min(max(a.cu[b + 1], t0), a.N);
    float* out = a.out + ((int64_t)n * a.hq + h) * D;
    if (n < t0 || n >= t1) {
        for (int d = lane; d < D; d += 64) out[d] = 0.0f;
        return;
    }
    const int t = n - t0;
    const int64_t most = (int64_t)a.max_blocks << a.c.bs_log2;
    const int keys = (int)min(min((int64_t)max(a.lengths[b], 0) + (t1 - t0), most), (int64_t)INT32_MAX - 4096);
    const int len = min(max(a.lengths[b], 0), keys);
    for (int d = lane; d < D; d += 64) s_q[d] = a.q[n * a.ldq + (int64_t)h * D + d] * a.scale;
    const uint64_t mask = a.masks ? a.masks[n] : 0;
    const int depth = a.masks ? __builtin_popcountll(mask) - 1 : t;
    const TableView table{a.table, a.max_blocks, a.table_stride};
    const int groups = (1 << a.c.bs_log2) / GROUP;
    float m = -3.4e38f, l = 0.0f, acc[4] = {0, 0, 0, 0};
    __syncthreads();
    for (int k0 = 0; k0 < keys; k0 += 64) {
        const int key = k0 + lane;
        bool see = key < keys;
        int place = key;  // its position
        if (see && key >= len) {
            const int j = key - len;
            if (a.masks) {
                see = j < 64 && (mask >> j & 1);
                place = see ? len + __builtin_popcountll(mask & ((1ull << j) - 1)) : 0;
            } else {
                see = j <= t;
            }
        }
        if (a.window && see) see = len + depth - place < a.window || place < a.sinks;
        const int slot = see ? table.slot(b, key, a.c) : -1;
        float s = -__builtin_inff();
        if (slot >= 0) {
            const int page = slot >> a.c.bs_log2, row = slot & ((1 << a.c.bs_log2) - 1);
            const int64_t at = page * a.c.sb + row * a.c.st + (int64_t)kvh * a.c.sh;
            float dot = 0.0f;
            for (int d = 0; d < D; ++d) dot = fmaf(s_q[d], element<TYPE>(a.k, at + d), dot);
            s = TYPE == 2 ? dot * held_scale(a.ks[((int64_t)page * a.hkv + kvh) * groups + row / GROUP]) : dot;
        }
        float mx = s;
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        mx = fmaxf(mx, m);
        const float p = exp2f(s - mx), f = exp2f(m - mx);
        float sum = p;
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
        l = l * f + sum;
        m = mx;
        __syncthreads();
        s_p[lane] = p;
        s_slot[lane] = p != 0.0f ? slot : -1;
        __syncthreads();
        for (int e = 0; e < 4; ++e) acc[e] *= f;
        for (int i = 0; i < 64; ++i) {
            const int sl = s_slot[i];
            if (sl < 0) continue;
            const int page = sl >> a.c.bs_log2, row = sl & ((1 << a.c.bs_log2) - 1);
            const int64_t at = page * a.c.sb + row * a.c.st + (int64_t)kvh * a.c.sh;
            float w = s_p[i];
            if (TYPE == 2) w *= held_scale(a.vs[((int64_t)page * a.hkv + kvh) * groups + row / GROUP]);
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < D) acc[e] = fmaf(w, element<TYPE>(a.v, at + lane + 64 * e), acc[e]);
        }
    }
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < D) out[lane + 64 * e] = l != 0.0f ? acc[e] / l : 0.0f;
}

}  // namespace

hipError_t launch_attn_window(const AttnArgs& a, int type, int D, int, int, uint8_t*, hipStream_t st) {
    const dim3 g((unsigned)((int64_t)a.N * a.hq)), t(64);
    if (type == 0) hipLaunchKernelGGL(window_kernel<0>, g, t, 0, st, a, D);
    else if (type == 1) hipLaunchKernelGGL(window_kernel<1>, g, t, 0, st, a, D);
    else hipLaunchKernelGGL(window_kernel<2>, g, t, 0, st, a, D);
    return hipGetLastError();
}

}  // namespace fq
