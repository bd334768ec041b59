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

constexpr int ROWS = 16;  // of a work-group at most

// Rows of keys and values, a lane 16 codes at a time.  Bound by the bytes, one in, two or four
// out, and for few rows by three loads one behind the other (requests, table, codes).  3946 tokens, 8 heads
// of 128 to fp16 (25 MB): 8.6 us; four pieces of 16 codes a lane are on their way at a time.  42 tokens 3.9.
template <int TYPE>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a, int most) {
    __shared__ int s_slot[ROWS], s_request[ROWS];
    __shared__ int64_t s_number[ROWS];
    const int n0 = blockIdx.x * most, tid = threadIdx.x;
    if (tid < 64) {
        // 64 requests at a time, a lane each, which enters its rows among these
        if (tid < ROWS) s_request[tid] = -1;
        int lo = 0;
        if (a.B > 64) {
            const int step = (a.B + 63) / 64, at = tid * step;
            const uint64_t in = __ballot(at < a.B && a.starts[min(at, a.B)] <= n0);
            lo = in ? (63 - __builtin_clzll(in)) * step : 0;
        }
        for (bool on = true; on; lo += 64) {
            const int b = lo + tid;
            int from = 0x7FFFFFFF, to = from;
            int64_t first = 0;
            if (b < a.B) {
                from = a.starts[b], to = a.starts[b + 1];
                if (a.first) first = a.first[b];
            }
            for (int n = max(from, n0); n < min(to, n0 + most); ++n)
                s_request[n - n0] = b, s_number[n - n0] = first + (n - from);
            on = lo + 64 < a.B && __builtin_amdgcn_readlane(to, 63) < n0 + most;
        }
    }
    __syncthreads();
    if (tid < ROWS) s_slot[tid] = s_request[tid] < 0 ? -1 : a.table.slot(s_request[tid], s_number[tid], a.c.c);
    __syncthreads();
    const int pieces = a.c.D / 16, per_row = a.c.hkv * pieces;
    const int count = min(most, a.N - n0) * per_row;  // pieces of keys, and of values
    constexpr int AHEAD = 4;
    for (int i0 = tid; i0 < 2 * count; i0 += AHEAD * 256) {
        u4 w[AHEAD];
        float s[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + 256 * k;
            w[k] = 0u, s[k] = 0.0f;
            if (i >= 2 * count) continue;
            const bool isv = i >= count;
            const int j = isv ? i - count : i, rest = j % per_row, h = rest / pieces;
            const int slot = s_slot[j / per_row];
            if (slot < 0) continue;
            const int page = slot >> a.c.c.bs_log2, at = slot & ((1 << a.c.c.bs_log2) - 1);
            w[k] = *(const u4*)((isv ? a.c.v : a.c.k) + page * a.c.c.sb + at * a.c.c.st + h * a.c.c.sh + 16 * (rest % pieces));
            s[k] = (isv ? a.c.vs : a.c.ks)[((int64_t)page * a.c.hkv + h) * a.c.groups() + at / GROUP];
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + 256 * k;
            if (i >= 2 * count) continue;
            const bool isv = i >= count;
            store16<TYPE>(isv ? a.v : a.k, ((int64_t)n0 * per_row + (isv ? i - count : i)) * 16, w[k], held_scale(s[k]));
        }
    }
}

constexpr int MOST = 64;  // accepted tokens that move

// One request's accepted tokens, one kv head's keys or values: all that move are in LDS before
// any is written.  A handful of tokens: bound by latency (path, table, rows).  7 trees of up to 25 tokens, 4 heads of
// 128, 16 bits: 3.4 us; 96 of up to 48, 8 heads, 8 bits: 9.6.
template <bool CODES>
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // of the k-th token that moves: its slots, its scale, its largest code; its new one's inverse
    __shared__ int s_from[MOST], s_to[MOST], s_most[MOST], s_moves;
    __shared__ float s_scale[MOST], s_inv[MOST];
    // and of those that are their group's first: the group's new scale, codes held before, what they are
    // rounded again by
    __shared__ float s_fresh[MOST], s_times[MOST];
    __shared__ int s_held[MOST];
    const int tid = threadIdx.x;
    const int b = blockIdx.x / (2 * a.hkv), hh = blockIdx.x % (2 * a.hkv), h = hh % a.hkv;
    const bool isv = hh >= a.hkv;
    constexpr int SIZE = CODES ? 1 : 2;
    const int groups = (1 << a.c.bs_log2) / GROUP;
    float* scales = CODES ? (isv ? a.vs : a.ks) + (int64_t)h * groups : nullptr;
    const auto scale_of = [&](int slot) {
        return scales + (int64_t)(slot >> a.c.bs_log2) * a.hkv * groups +
               (slot & ((1 << a.c.bs_log2) - 1)) / GROUP;
    };
    if (tid < MOST) {
        const int t0 = min(max(a.cu[b], 0), a.N), nt = min(max(a.cu[b + 1], t0), a.N) - t0;
        const int acc = min(min(a.accepted[b], nt), MOST);
        const int64_t len = max(a.lengths[b], 0);
        int from = -1, to = -1;
        if (tid < acc) {
            const int p = a.path[t0 + tid];
            if (p != tid && p >= 0 && p < nt) {
                from = a.table.slot(b, len + p, a.c);
                to = a.table.slot(b, len + tid, a.c);
            }
        }
        const bool moves = from >= 0 && to >= 0;
        const uint64_t all = __ballot(moves);
        if (tid == 0) s_moves = __builtin_popcountll(all);
        if (moves) {
            const int k = __builtin_popcountll(all & ((1ull << tid) - 1));
            s_from[k] = from, s_to[k] = to, s_most[k] = 0;
            if (CODES) s_scale[k] = held_scale(*scale_of(from));
        }
    }
    __syncthreads();
    const int moves = s_moves;
    if (!moves) return;
    const int bytes = a.D * SIZE, pieces = bytes / 16;
    uint8_t* cache = (uint8_t*)(isv ? a.v : a.k) + h * a.c.sh * SIZE;
    const auto place = [&](int slot) {
        return cache + ((slot >> a.c.bs_log2) * a.c.sb + (slot & ((1 << a.c.bs_log2) - 1)) * a.c.st) * SIZE;
    };
    for (int i = tid; i < moves * pieces; i += 256) {
        const int k = i / pieces;
        const u4 w = *(const u4*)(place(s_from[k]) + 16 * (i % pieces));
        *(u4*)(lds + 16 * i) = w;
        if (CODES) {
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(code_at(w[e >> 2], e & 3)));
            atomicMax(&s_most[k], (int)most);
        }
    }
    __syncthreads();
    if constexpr (CODES) {
        if (tid < moves) {
            const int to = s_to[tid];
            float need = 0.0f;
            int first = GROUP;
            for (int e = 0; e < moves; ++e) {
                const int other = s_to[e];
                if (other / GROUP != to / GROUP) continue;
                need = fmaxf(need, s_scale[e] * ((float)s_most[e] / 127.0f));
                first = min(first, other % GROUP);
            }
            const float old = first ? held_scale(*scale_of(to)) : 0.0f;
            const float s = fmaxf(need, old), inv = inverse_of(s);
            s_inv[tid] = inv;
            s_fresh[tid] = to % GROUP == first ? s : -1.0f;
            s_held[tid] = to % GROUP == first && s > old ? first : 0;
            s_times[tid] = old * inv;
        }
        __syncthreads();
    }
    for (int i = tid; i < moves * pieces; i += 256) {
        const int k = i / pieces, p = i % pieces;
        u4 w = *(const u4*)(lds + 16 * i);
        uint8_t* to = place(s_to[k]);
        if constexpr (CODES) {
            const float s = s_scale[k], inv = s_inv[k];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = four_codes(code_at(w[e], 0) * s, code_at(w[e], 1) * s, code_at(w[e], 2) * s,
                                  code_at(w[e], 3) * s, inv);
            if (p == 0 && s_fresh[k] >= 0.0f) *scale_of(s_to[k]) = s_fresh[k];
        }
        *(u4*)(to + 16 * p) = w;
    }
    if constexpr (CODES) {
        for (int k = 0; k < moves; ++k) {
            uint8_t* to = place(s_to[k]);
            for (int i = tid; i < s_held[k] * pieces; i += 256) {
                u4* w = (u4*)(to - (1 + i / pieces) * a.c.st + 16 * (i % pieces));
                u4 v = *w;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = again(v[e], s_times[k]);
                *w = v;
            }
        }
    }
}

}  // namespace

int read8_rows(const Cache8& c) {
    // (about four pieces a lane)
    int rows = ROWS;
    while (rows > 1 && 2 * rows * (c.hkv * c.D / 16) > 4 * 256) rows /= 2;
    return rows;
}

hipError_t launch_read8(const ReadArgs& a, int type, hipStream_t st) {
    const int rows = read8_rows(a.c);
    const dim3 g((unsigned)(((int64_t)a.N + rows - 1) / rows)), t(256);
    if (type == 0) hipLaunchKernelGGL(read_kernel<0>, g, t, 0, st, a, rows);
    else if (type == 1) hipLaunchKernelGGL(read_kernel<1>, g, t, 0, st, a, rows);
    else hipLaunchKernelGGL(read_kernel<2>, g, t, 0, st, a, rows);
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
