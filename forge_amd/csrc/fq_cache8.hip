// fq_cache8.hip -- reads a cache of 8 bits back, and moves an accepted branch's keys and
// values to the slots behind the context (caches of any type).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fq_group8.h"
#include "fq_step.h"

namespace fq {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The last b of 0 .. n-1 with starts[b] <= row (0 if there is none); starts rises.
__device__ __forceinline__ int request_of(const int* starts, int n, int row) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (starts[mid] <= row ? lo : hi) = mid;
    }
    return lo;
}

// 16 codes as 16 values of 4 (TYPE 0) or 2 bytes.
template <int TYPE>
__device__ __forceinline__ void store16(void* out, int64_t at, u4 w, float s) {
    if constexpr (TYPE == 0) {
        f4* o = (f4*)((float*)out + at);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = f4{code_at(w[i], 0) * s, code_at(w[i], 1) * s, code_at(w[i], 2) * s, code_at(w[i], 3) * s};
    } else {
        u4* o = (u4*)((uint16_t*)out + at);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u4 r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = w[2 * i + (e >> 1)] >> (16 * (e & 1));
                const float a = code_at(x, 0) * s, b = code_at(x, 1) * s;
                if (TYPE == 1)
                    r[e] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) |
                           (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
                else
                    r[e] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) |
                           (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16;
            }
            o[i] = r;
        }
    }
}

constexpr int ROWS = 16;  // of a work-group

// Rows of keys and values, a lane 16 codes at a time.  Bound by the bytes: one in, two
// or four out.
template <int TYPE>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
    __shared__ int s_slot[ROWS];
    const int n0 = blockIdx.x * ROWS, tid = threadIdx.x;
    if (tid < ROWS) {
        const int n = n0 + tid;
        int slot = -1;
        if (n < a.N) {
            const int b = request_of(a.starts, a.B, n);
            const int from = a.starts[b];
            if (n >= from && n < a.starts[b + 1])
                slot = a.table.slot(b, (int64_t)(a.first ? a.first[b] : 0) + (n - from), a.c.c);
        }
        s_slot[tid] = slot;
    }
    __syncthreads();
    const int pieces = a.c.D / 16, per_row = a.c.hkv * pieces;
    const int rows = min(ROWS, a.N - n0);
    for (int i = tid; i < 2 * rows * per_row; i += 256) {
        const bool isv = i >= rows * per_row;
        const int j = isv ? i - rows * per_row : i;
        const int row = j / per_row, rest = j % per_row, h = rest / pieces, p = rest % pieces;
        const int slot = s_slot[row];
        u4 w = 0u;
        float s = 0.0f;
        if (slot >= 0) {
            const int page = slot >> a.c.c.bs_log2, at = slot & ((1 << a.c.c.bs_log2) - 1);
            w = *(const u4*)((isv ? a.c.v : a.c.k) + page * a.c.c.sb + at * a.c.c.st + h * a.c.c.sh + 16 * p);
            s = held_scale((isv ? a.c.vs : a.c.ks)[((int64_t)page * a.c.hkv + h) * a.c.groups() + at / GROUP]);
        }
        store16<TYPE>(isv ? a.v : a.k, ((int64_t)(n0 + row) * per_row + rest) * 16, w, s);
    }
}

constexpr int MOST = 64;  // accepted tokens that move

// One request's accepted tokens, one kv head's keys or values: all that move are in LDS
// before any is written.  A handful of tokens: bound by latency (table, path, rows).
template <bool CODES>
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ int s_from[MOST], s_to[MOST], s_any;
    __shared__ float s_scale[MOST], s_need[MOST];
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    const int b = blockIdx.x / (2 * a.hkv), hh = blockIdx.x % (2 * a.hkv), h = hh % a.hkv;
    const bool isv = hh >= a.hkv;
    const int t0 = min(max(a.cu[b], 0), a.N), nt = min(max(a.cu[b + 1], t0), a.N) - t0;
    const int acc = min(min(a.accepted[b], nt), MOST);
    const int64_t len = max(a.lengths[b], 0);
    if (tid < MOST) {
        int from = -1, to = -1;
        if (tid < acc) {
            const int p = a.path[t0 + tid];
            if (p != tid && p >= 0 && p < nt) {
                from = a.table.slot(b, len + p, a.c);
                to = a.table.slot(b, len + tid, a.c);
                if (from < 0 || to < 0) from = to = -1;
            }
        }
        s_from[tid] = from, s_to[tid] = to;
        const uint64_t moves = __ballot(to >= 0);
        if (tid == 0) s_any = moves != 0;
    }
    __syncthreads();
    if (!s_any) return;
    constexpr int SIZE = CODES ? 1 : 2;
    const int bytes = a.D * SIZE, pieces = bytes / 16;
    uint8_t* cache = (uint8_t*)(isv ? a.v : a.k) + h * a.c.sh * SIZE;
    const auto place = [&](int slot) {
        return cache + ((slot >> a.c.bs_log2) * a.c.sb + (slot & ((1 << a.c.bs_log2) - 1)) * a.c.st) * SIZE;
    };
    const int groups = (1 << a.c.bs_log2) / GROUP;
    float* scales = CODES ? (isv ? a.vs : a.ks) + (int64_t)h * groups : nullptr;
    const auto scale_of = [&](int slot) {
        return scales + (int64_t)(slot >> a.c.bs_log2) * a.hkv * groups +
               (slot & ((1 << a.c.bs_log2) - 1)) / GROUP;
    };
    // a wave takes every fourth token
    for (int d = wave; d < acc; d += 4) {
        const int from = s_from[d];
        if (from < 0) continue;
        float most = 0.0f;
        for (int i = lane; i < pieces; i += 64) {
            const u4 w = *(const u4*)(place(from) + 16 * i);
            *(u4*)(lds + d * bytes + 16 * i) = w;
            if (CODES)
#pragma unroll
                for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(code_at(w[e >> 2], e & 3)));
        }
        if (CODES) {
            for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
            if (lane == 0) {
                const float s = held_scale(*scale_of(from));
                s_scale[d] = s;
                s_need[d] = s * (most / 127.0f);
            }
        }
    }
    __syncthreads();
    // Of this wave's tokens; and of those that are their group's first: its new scale, codes held
    // before and what they are rounded again by.
    float inv[MOST / 4], fresh[MOST / 4], times[MOST / 4];
    int held[MOST / 4];
    if constexpr (CODES) {
        // every wave finds its tokens' new scales before any is written
#pragma unroll
        for (int k = 0; k < MOST / 4; ++k) {
            const int d = wave + 4 * k;
            inv[k] = 0.0f, fresh[k] = -1.0f, times[k] = 0.0f, held[k] = 0;
            if (d >= acc || s_to[d] < 0) continue;
            const int to = s_to[d];
            float need = 0.0f;
            int first = GROUP;
            for (int e = max(0, d - GROUP + 1); e < min(acc, d + GROUP); ++e) {
                if (s_to[e] < 0 || s_to[e] / GROUP != to / GROUP) continue;
                need = fmaxf(need, s_need[e]);
                first = min(first, s_to[e] % GROUP);
            }
            const float old = first ? held_scale(*scale_of(to)) : 0.0f;
            const float s = fmaxf(need, old);
            inv[k] = inverse_of(s);
            if (to % GROUP == first) {
                fresh[k] = s;
                if (s > old) held[k] = first, times[k] = old * inv[k];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < MOST / 4; ++k) {
        const int d = wave + 4 * k;
        if (d >= acc || s_to[d] < 0) continue;
        uint8_t* to = place(s_to[d]);
        for (int i = lane; i < pieces; i += 64) {
            u4 w = *(const u4*)(lds + d * bytes + 16 * i);
            if constexpr (CODES) {
                const float s = s_scale[d];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = four_codes(code_at(w[e], 0) * s, code_at(w[e], 1) * s, code_at(w[e], 2) * s,
                                      code_at(w[e], 3) * s, inv[k]);
            }
            *(u4*)(to + 16 * i) = w;
        }
        if constexpr (CODES) {
            if (fresh[k] >= 0.0f && lane == 0) *scale_of(s_to[d]) = fresh[k];
            for (int i = lane; i < held[k] * pieces; i += 64) {
                u4* w = (u4*)(to - (1 + i / pieces) * a.c.st + 16 * (i % pieces));
                u4 v = *w;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = again(v[e], times[k]);
                *w = v;
            }
        }
    }
}

}  // namespace

hipError_t launch_read8(const ReadArgs& a, int type, hipStream_t st) {
    const dim3 g((unsigned)((a.N + ROWS - 1) / ROWS)), t(256);
    if (type == 0) hipLaunchKernelGGL(read_kernel<0>, g, t, 0, st, a);
    else if (type == 1) hipLaunchKernelGGL(read_kernel<1>, g, t, 0, st, a);
    else hipLaunchKernelGGL(read_kernel<2>, g, t, 0, st, a);
    return hipGetLastError();
}

hipError_t launch_keep(const KeepArgs& a, bool codes, hipStream_t st) {
    const dim3 g((unsigned)((int64_t)a.B * 2 * a.hkv)), t(256);
    const size_t lds = (size_t)MOST * a.D * (codes ? 1 : 2);
    if (codes) hipLaunchKernelGGL(keep_kernel<true>, g, t, lds, st, a);
    else hipLaunchKernelGGL(keep_kernel<false>, g, t, lds, st, a);
    return hipGetLastError();
}

}  // namespace fq
