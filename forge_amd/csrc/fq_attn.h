// fq_attn.h -- what the attention kernels share: their items' shares among the work-groups, windows,
// and the kernel that joins the items' parts.  Internal to them.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "fq_dma.h"
#include "fq_step.h"

namespace fq {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;
typedef const __attribute__((address_space(3))) u4 lds_u4;
typedef __attribute__((address_space(3))) float lds_f;

constexpr float LOWEST = -3.402823466e38f;
// A uniform value in a scalar register, read through the scalar cache (memory
// that no kernel writes while this one runs).
__device__ __forceinline__ int sload(const int* p) {
    return *(const __attribute__((address_space(4))) int*)(uintptr_t)p;
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// All waves' LDS accesses are done (their stores to memory may be on their way).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// What a request brings.
struct Request {
    int t0, nt, len;  // its first new token, how many, its cached tokens (of those the table can hold)
    int pos;          // its first new token's position
    int keys, nu;     // keys and units of them that are walked
    int su, skip;     // with a window: units that hold the sinks, units left out behind them
    int rts;          // tiles of RT rows
    int cost;         // an item's units and OV more, or 1 where items are not cut
    int64_t units;    // that of all its items
};
template <int RT, int KU, int OV, bool WIN>
__device__ __forceinline__ Request request(const AttnArgs& a, int c0, int c1, int len) {
    Request r;
    r.t0 = min(max(c0, 0), a.N);
    r.nt = min(max(c1, r.t0), a.N) - r.t0;
    // (no key, cached or new, lies beyond the table's columns)
    const int64_t most = (int64_t)a.max_blocks << a.c.bs_log2;
    r.keys = (int)min((int64_t)max(len, 0) + r.nt, min(most, (int64_t)INT32_MAX - 4096));
    r.len = min(max(len, 0), r.keys);
    r.pos = max(len, 0);
    r.nu = (r.keys + KU - 1) / KU;
    r.su = r.skip = 0;
    if constexpr (WIN) {
        // No new token lies before position pos, so none sees a cached one before this, but for sinks.
        // (Which may be behind all keys there are: a unit stays, masked, so that zeros are written.)
        const int from = a.window ? max(r.pos - a.window + 1, 0) : 0;
        r.su = (min(a.sinks, r.keys) + KU - 1) / KU;
        r.skip = max(min(from / KU - r.su, r.nu - max(r.su, 1)), 0);
        r.nu -= r.skip;
    }
    r.rts = (int)(((int64_t)r.nt * a.G + RT - 1) / RT);
    r.cost = a.whole ? 1 : r.nu + OV;
    r.units = r.nu ? (int64_t)a.hkv * r.rts * r.cost : 0;
    return r;
}

// a / b, in 32 bits where that does (a 64-bit division takes a third of a microsecond).
__device__ __forceinline__ int64_t divided(int64_t a, int64_t b) {
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

__device__ __forceinline__ int64_t uni64(int64_t v) {
    return ((int64_t)uni((int)(v >> 32)) << 32) | (uint32_t)uni((int)v);
}

// The largest of the four lanes (l % 16 + 0, 16, 32, 48).
__device__ __forceinline__ float max4(float x) {
    const uint32_t u = __float_as_uint(x);
    const u2 p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    x = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const uint32_t v = __float_as_uint(x);
    const u2 q = __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(v, v, false, false));
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float sum4(float x) {
    const uint32_t u = __float_as_uint(x);
    const u2 p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    const uint32_t v = __float_as_uint(x);
    const u2 q = __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(v, v, false, false));
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// Ones at the n lowest places (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t low_bits(int n) {
    return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
}
// The places 0 .. 31 of m moved n up (down where n < 0).
__device__ __forceinline__ uint32_t shifted(uint64_t m, int n) {
    return n >= 32 || n <= -64 ? 0u : n >= 0 ? (uint32_t)m << n : (uint32_t)(m >> -n);
}

// What a row of a call with a window sees of the context: the sinks and from `from` on; and a
// draft's bits without those the window has left.  pos: the request's first new token's position, t: the
// row's number among the new tokens.
struct Reach {
    int from;
    uint64_t mask;
};
__device__ __forceinline__ Reach reach(const AttnArgs& a, int pos, int t, uint64_t mask) {
    const int depth = a.masks ? max(__builtin_popcountll(mask) - 1, 0) : t;
    Reach r{a.window ? (int)min(max((int64_t)pos + depth + 1 - a.window, (int64_t)0), (int64_t)INT32_MAX) : 0, mask};
    if (a.masks && a.window && depth >= a.window) {
        // a bit's position is pos and how many are below it
        uint64_t rest = mask;
        r.mask = 0;
        for (int at = 0; rest; rest &= rest - 1, ++at)
            if (depth - at < a.window || (int64_t)pos + at < a.sinks) r.mask |= rest & -rest;
    }
    return r;
}
// A tile's keys that a row sees, as bits: the first one key0, `old` of the context and `all` of the
// request from there on.  mask: of the new tokens, or, for chains, how many it sees.
template <bool WIN>
__device__ __forceinline__ uint32_t seen(const AttnArgs& a, uint64_t mask, int from, int key0, int old, int all) {
    if constexpr (!WIN) {
        const uint32_t s = a.masks ? low_bits(old) | shifted(mask, old) : low_bits(old + (int)(uint32_t)mask);
        return s & low_bits(all);
    } else {
        const uint32_t near = low_bits(a.sinks - key0) | ~low_bits(from - key0);
        const uint32_t s = a.masks ? (low_bits(old) & near) | shifted(mask, old)
                                   : low_bits(old + (int)(uint32_t)mask) & near;
        return s & low_bits(all);
    }
}

// Whether a page is none of the cache's blocks: its keys are seen by nobody.
__device__ __forceinline__ bool no_block(const AttnArgs& a, int page) {
    return (uint32_t)page >= (uint32_t)a.c.num_blocks;
}
constexpr int DESC = 4;          // ints of a work-group's record, beside the number of parts
constexpr int MAX_ITEMS = 1024;  // work-groups at most
constexpr int WIDE = MAX_ITEMS * (DESC + 1);  // behind them: whether an item may have more than NARROW parts
constexpr int MAX_GRID = 4;      // work-groups to a CU at most,
constexpr size_t MAX_PART = 3 * 64 * (128 + 2);  // and floats of a part of all of them


// Joins the parts of the items that are cut: two rows at a time by one wave or, where
// an item has more than NARROW parts, one row by the four waves of a work-group (768
// items of 4 parts: 17 us, 55 the second way; 8 of 96 parts: 11 us, 43 the first way).
constexpr int JOIN_WGS = 8;  // work-groups to a CU
constexpr int NARROW = 16;   // parts of an item that one wave joins

template <int D, int RT, bool NEAR = false>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a) {
    constexpr int PART = RT * (D + 2), E = D == 64 ? 1 : D == 256 ? 4 : 2;
    typedef float fe __attribute__((ext_vector_type(E)));
    struct Item {
        int parts, w, t0, nt, h, rt;
    };
    __shared__ Item s_item[MAX_ITEMS];
    __shared__ int s_count[4], s_most[4];
    __shared__ float s_acc[4][D + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    const auto slot = [&](const Item& x, int p) {
        return a.part + (int64_t)(2 * (x.w + p) + (p == 0)) * PART;
    };
    const auto store = [&](const Item& x, int r, fe acc, float l) {
        const int t = r / a.G;
        fe v = 0.0f;
        if (l != 0.0f) v = acc * (1.0f / l);
        if (E * lane < D)
            *(fe*)(a.out + ((int64_t)(x.t0 + t) * a.hq + x.h * a.G + r % a.G) * D + E * lane) = v;
    };
    // Two rows of an item of few parts, rl the first one's place among its RT.
    constexpr int R = 2;
    const auto two_rows = [&](const Item& x, int rl) {
        const int r0 = x.rt * RT + rl;
        if (r0 >= x.nt * a.G) return;
        float mp[R], lp[R];
        fe o[R][NARROW];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            mp[k] = LOWEST, lp[k] = 0.0f;
            const bool on = r0 + k < x.nt * a.G;
            if (on && lane < x.parts) {
                const float* s = slot(x, lane) + RT * D + rl + k;
                mp[k] = s[0], lp[k] = s[RT];
            }
#pragma unroll
            for (int p = 0; p < NARROW; ++p) {
                o[k][p] = 0.0f;
                if (on && p < x.parts && E * lane < D) o[k][p] = *(const fe*)(slot(x, p) + (rl + k) * D + E * lane);
            }
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            float m = mp[k];
            for (int q = NARROW / 2; q; q >>= 1) m = fmaxf(m, __shfl_xor(m, q));
            m = __shfl(m, 0);
            const float f = __builtin_amdgcn_exp2f(mp[k] - m);
            float l = lp[k] * f;
            for (int q = NARROW / 2; q; q >>= 1) l += __shfl_xor(l, q);
            l = __shfl(l, 0);
            fe acc = 0.0f;
#pragma unroll
            for (int p = 0; p < NARROW; ++p)
                if (p < x.parts) acc += __shfl(f, p) * o[k][p];
            if (r0 + k < x.nt * a.G) store(x, r0 + k, acc, l);
        }
    };
    if (NEAR && !a.desc[WIDE]) {
        // No item has many parts: a work-group takes those of one work-group's, a share of its rows,
        // and looks at no other's.
        const int w = blockIdx.x % a.grid, c = blockIdx.x / a.grid, share = gridDim.x / a.grid;
        if (c >= share) return;
        const int parts = a.desc[w];
        const int4 rec = ((const int4*)(a.desc + MAX_ITEMS))[w];
        if (!parts) return;
        const Item x{parts, w, rec.x, rec.y, rec.z, rec.w};
        for (int job = c * 4 + wave; job < RT / R; job += share * 4) two_rows(x, job * R);
        return;
    }
    // the items, in the order of the work-groups that began them: thread i looks at
    // the K next to each other from K i on
    constexpr int K = MAX_ITEMS / 256;
    int parts[K], most = 0, mine = 0;
    int4 rec[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = tid * K + k;
        parts[k] = i < a.grid ? a.desc[i] : 0;
        rec[k] = i < a.grid ? ((const int4*)(a.desc + MAX_ITEMS))[i] : int4{0, 0, 0, 0};
        most = max(most, parts[k]);
        mine += parts[k] > 0;
    }
    int upto = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
        most = max(most, __shfl_xor(most, o));
    }
    if (lane == 63) s_count[wave] = upto;
    if (lane == 0) s_most[wave] = most;
    __syncthreads();
    int at = upto - mine, items = 0;
    for (int v = 0; v < 4; ++v) {
        at += v < wave ? s_count[v] : 0;
        items += s_count[v];
        most = max(most, s_most[v]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (parts[k]) s_item[at++] = {parts[k], tid * K + k, rec[k].x, rec[k].y, rec[k].z, rec[k].w};
    __syncthreads();
    if (most <= NARROW) {
        for (int job = blockIdx.x * 4 + wave; job < items * (RT / R); job += gridDim.x * 4)
            two_rows(s_item[job / (RT / R)], job % (RT / R) * R);
        return;
    }
    for (int job = blockIdx.x; job < items * RT; job += gridDim.x) {
        const Item x = s_item[job / RT];
        const int rl = job % RT, r = x.rt * RT + rl, parts = x.parts;
        if (r >= x.nt * a.G) continue;
        float m = LOWEST;
        for (int p = lane; p < parts; p += 64) m = fmaxf(m, slot(x, p)[RT * D + rl]);
        for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const int share = (parts + 3) / 4, beg = wave * share, end = min(parts, beg + share);
        fe acc = 0.0f;
        float l = 0.0f;
        for (int p0 = beg; p0 < end; p0 += 64) {
            float f = 0.0f, lp = 0.0f;
            if (p0 + lane < end) {
                const float* s = slot(x, p0 + lane) + RT * D + rl;
                f = __builtin_amdgcn_exp2f(s[0] - m);
                lp = s[RT] * f;
            }
            for (int o = 32; o; o >>= 1) lp += __shfl_xor(lp, o);
            l += lp;
            for (int p = p0; p < min(end, p0 + 64); p += 8) {
                fe o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    o[i] = 0.0f;
                    if (p + i < end && E * lane < D) o[i] = *(const fe*)(slot(x, p + i) + rl * D + E * lane);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float fp = __shfl(f, (p + i - p0) & 63);
                    if (p + i < end) acc += fp * o[i];
                }
            }
        }
        if (E * lane < D)
            for (int e = 0; e < E; ++e) s_acc[wave][E * lane + e] = acc[e];
        if (lane == 0) s_acc[wave][D] = l;
        __syncthreads();
        acc = 0.0f;
        l = 0.0f;
        for (int i = 0; i < 4; ++i) {
            l += s_acc[i][D];
            if (E * lane < D)
                for (int e = 0; e < E; ++e) acc[e] += s_acc[i][E * lane + e];
        }
        __syncthreads();
        if (wave == 0) store(x, r, acc, l);
    }
}

// The most keys that an item walks, by the table's columns and the window.  (A request may have more new
// tokens than it was said: its items only take longer.)
template <class S>
int64_t most_keys(const AttnArgs& a, int max_new) {
    const int64_t keys = (int64_t)a.max_blocks << a.c.bs_log2;
    if (!a.window) return keys;
    return std::min<int64_t>(keys, (int64_t)a.window + max_new + (a.sinks ? S::KU + std::min<int64_t>(a.sinks, keys) : 0));
}

// Whether items are left whole, so that nothing is to be joined: where they have 6 units at most, by
// the table's columns and the window, and up to 12, or any number under a window, where they take no longer one
// after the other on the work-groups than cut into even shares, with the begin of a second part and the
// second launch (about JOIN units).  Without a window the longest item counts against three
// quarters of it on average.  D = 128, 8 x 4 heads, one token, us: 64 requests of 760 keys 21.6, cut 30;
// 64 of 20001 under a window of 1023 37, cut 46 + 8; one of 630 13.1, cut 14.5.
template <class S>
bool uncut(const AttnArgs& a, int max_new) {
    constexpr int JOIN = 2 + 256 / S::KU, MOST_UNITS = 12;
    const int64_t keys = most_keys<S>(a, max_new);
    if (keys <= 6 * std::max(S::KU, 64)) return true;
    if (!a.window && keys > MOST_UNITS * S::KU) return false;
    const int64_t units = keys / S::KU + 2, even = a.window ? units : units * 3 / 4;
    const int64_t items = (int64_t)a.B * a.hkv * (((int64_t)max_new * a.G + S::RT - 1) / S::RT);
    const int64_t turns = (items + a.grid - 1) / a.grid;
    return turns * (units + S::OV) <= items * (even + 2 * S::OV) / a.grid + JOIN;
}

constexpr size_t DESC_BYTES = (size_t)MAX_ITEMS * (DESC + 1) * 4 + 16;

}  // namespace
}  // namespace fq
