// fq_rope8.hip -- bias, per-head norm and rotation of the QKV rows, keys and values
// rounded into a paged cache of 8 bits.
//
// A group of 16 tokens has one scale for each kv head, so that its new tokens have to be
// seen together: s = max|y| / 127 over them (and over the scale before, where the group holds
// tokens already, whose codes are then rounded again).  A work-group takes 16 tokens of the call and one
// kv head's keys or values; it does the runs (new tokens of one group) that begin among its
// tokens, so that each run is done once, by lanes of 16 tokens each for the run's part
// among them and for what lies behind.  What is a run shows in the slots alone: they rise
// by one within a group.
#include <hip/hip_runtime.h>

#include "fq_group8.h"
#include "fq_rope.h"

namespace fq {
namespace {

constexpr int W = 16;  // tokens of a work-group

template <int GS, bool INTER>
__global__ __launch_bounds__(256) void rope8_kernel(RopeArgs a, Cache8 c, int kv_blocks) {
    constexpr int TOK = 256 / GS;  // tokens that the lanes take at a time
    constexpr int R = (2 * W + TOK - 1) / TOK;
    const int p = threadIdx.x % GS, sub = threadIdx.x / GS;
    const bool lane_on = 8 * p < a.D;
    // (keys and values, which take longer, first)
    if ((int)blockIdx.x >= kv_blocks) {  // query heads
        const int64_t item = (int64_t)((int)blockIdx.x - kv_blocks) * TOK + sub;
        if (item >= (int64_t)a.N * a.hq) return;
        const int n = (int)(item / a.hq), h = (int)(item % a.hq);
        const auto [x0, x1, d0, d1] = head_runs<GS, INTER>(a, n, h, p, lane_on);
        if (!lane_on) return;
        float* q = a.q + ((int64_t)n * a.hq + h) * a.D;
        *(f4u*)(q + d0) = x0;
        *(f4u*)(q + d1) = x1;
        return;
    }
    const int hh = blockIdx.x % (2 * c.hkv), n0 = blockIdx.x / (2 * c.hkv) * W;
    const int h = hh % c.hkv;
    const bool isv = hh >= c.hkv;
    __shared__ int s_slot[2 * W + 1];
    __shared__ float s_max[2 * W];
    // (the first tokens' rows are on their way before it shows which of them are this work-group's)
    HeadRuns x[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
        if ((r + 1) * TOK <= W)
            x[r] = head_runs<GS, INTER>(a, n0 + r * TOK + sub, a.hq + hh, p, lane_on && n0 + r * TOK + sub < a.N);
    // slots of tokens n0 - 1 .. n0 + 31
    if (threadIdx.x < 2 * W + 1) {
        const int n = n0 - 1 + (int)threadIdx.x;
        int slot = n >= 0 && n < a.N ? a.slots[n] : -1;
        if (slot < 0 || (slot >> c.c.bs_log2) >= c.c.num_blocks) slot = -1;
        s_slot[threadIdx.x] = slot;
    }
    __syncthreads();
    // bit j: token n0 + j goes on with the run of the one before
    uint32_t goes_on = 0;
    {
        const int j = threadIdx.x & 31, slot = s_slot[j + 1];
        const bool on = slot >= 0 && slot % GROUP && s_slot[j] == slot - 1;
        goes_on = (uint32_t)__ballot(on);
    }
    int slot[R], lead[R];  // lead: where the token's run begins; -1: not this work-group's
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int j = r * TOK + sub;
        slot[r] = j < 2 * W ? s_slot[j + 1] : -1;
        lead[r] = -1;
        if (slot[r] >= 0) {
            const uint32_t begins = ~goes_on & (j < 31 ? (2u << j) - 1 : ~0u);
            lead[r] = begins ? 31 - __builtin_clz(begins) : -1;
            if (lead[r] >= W) lead[r] = -1;
        }
        if ((r + 1) * TOK > W) x[r] = head_runs<GS, INTER>(a, n0 + j, a.hq + hh, p, lane_on && lead[r] >= 0);
        float m = 0.0f;
        if (lane_on && lead[r] >= 0)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = largest(largest(m, x[r].x0[i]), x[r].x1[i]);
        for (int o = 1; o < GS; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, GS));
        if (p == 0 && j < 2 * W) s_max[j] = m;
    }
    __syncthreads();
    int8_t* cache = (isv ? c.v : c.k) + (int64_t)h * c.c.sh;
    float* scales = isv ? c.vs : c.ks;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (lead[r] < 0) continue;
        const int j = r * TOK + sub;
        const int page = slot[r] >> c.c.bs_log2, row = slot[r] & ((1 << c.c.bs_log2) - 1);
        float* sp = scales + ((int64_t)page * c.hkv + h) * c.groups() + row / GROUP;
        // the run's largest: its tokens follow `lead` without a gap
        float m = s_max[lead[r]];
        for (int i = lead[r] + 1; i < 2 * W && (goes_on >> i & 1); ++i) m = fmaxf(m, s_max[i]);
        const int held = row % GROUP - (j - lead[r]);  // tokens before the run
        const float need = m / 127.0f, old = held ? held_scale(*sp) : 0.0f;
        const float s = fmaxf(need, old), inv = inverse_of(s);
        if (!lane_on) continue;
        int8_t* to = cache + page * c.c.sb + row * c.c.st;
        const f4 y0 = x[r].x0, y1 = x[r].x1;
        *(uint32_t*)(to + x[r].d0) = four_codes(y0[0], y0[1], y0[2], y0[3], inv);
        *(uint32_t*)(to + x[r].d1) = four_codes(y1[0], y1[1], y1[2], y1[3], inv);
        if (j == lead[r]) {
            if (s > old) {
                const float times = old * inv;
                for (int i = 1; i <= held; ++i) {
                    uint2* w = (uint2*)(to - i * c.c.st + 8 * p);
                    *w = make_uint2(again(w->x, times), again(w->y, times));
                }
            }
            if (p == 0) *sp = s;
        }
    }
}

template <int GS>
hipError_t go(const RopeArgs& a, const Cache8& c, bool inter, hipStream_t st) {
    constexpr int TOK = 256 / GS;
    const int64_t q_blocks = ((int64_t)a.N * a.hq + TOK - 1) / TOK;
    const int64_t kv_blocks = (int64_t)((a.N + W - 1) / W) * 2 * c.hkv;
    const dim3 g((unsigned)(q_blocks + kv_blocks)), t(256);
    if (inter) hipLaunchKernelGGL((rope8_kernel<GS, true>), g, t, 0, st, a, c, (int)kv_blocks);
    else hipLaunchKernelGGL((rope8_kernel<GS, false>), g, t, 0, st, a, c, (int)kv_blocks);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope8(const RopeArgs& a, const Cache8& c, bool interleaved, hipStream_t st) {
    const int lanes = a.D / 8;
    if (lanes <= 8) return go<8>(a, c, interleaved, st);
    if (lanes <= 16) return go<16>(a, c, interleaved, st);
    if (lanes <= 32) return go<32>(a, c, interleaved, st);
    return go<64>(a, c, interleaved, st);
}

}  // namespace fq
