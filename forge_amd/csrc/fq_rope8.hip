// fq_rope8.hip -- bias, per-head norm and rotation of the QKV rows, keys and values
// rounded into a paged cache of 8 bits.
//
// A group of 16 tokens has one scale for each kv head, so that its new tokens have to be
// seen together: s = max|y| / 127 over them (and over the scale before, where the group holds
// tokens already, whose codes are then rounded again).  A work-group takes 16 tokens of the call and one
// kv head's keys or values; it does the runs (new tokens of one group) that begin among its
// tokens, so that each run is done once, by lanes of 16 tokens each for the run's part
// among them and for what lies behind.  What is a run shows in the slots alone: they rise
// by one within a group.  A work-group's tokens are 16, so that most runs are whole (runs of a prompt
// begin at groups) and no more than 31 tokens are looked at; half its lanes wait where two runs share them.
//
// Bound: the bytes of the rows, read once, and the queries: three prompts of up to 2731 tokens, 32 +
// 2 x 8 heads of 128, norm (the rows' 24 KB, queries' 16 and codes' 2 a token, 170 MB): 35 us, 4.8 TB/s, of which the
// queries alone take 24.  One token: 3.8 us, the launch
// and three loads one behind the other (slots, row, scale).
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
    __shared__ int s_slot[2 * W + 1], s_max[W];
    __shared__ float s_inv[W];
    // slots of tokens n0 - 1 .. n0 + 31
    if (threadIdx.x < 2 * W + 1) {
        const int n = n0 - 1 + (int)threadIdx.x;
        int slot = n >= 0 && n < a.N ? a.slots[n] : -1;
        if (slot < 0 || (slot >> c.c.bs_log2) >= c.c.num_blocks) slot = -1;
        s_slot[threadIdx.x] = slot;
    }
    if (threadIdx.x < W) s_max[threadIdx.x] = 0;
    __syncthreads();
    // bit j: token n0 + j has a slot; goes on with the run of the one before
    uint32_t there, goes_on;
    {
        const int j = threadIdx.x & 31, slot = s_slot[j + 1];
        there = (uint32_t)__ballot(slot >= 0);
        goes_on = (uint32_t)__ballot(slot >= 0 && slot % GROUP && s_slot[j] == slot - 1);
    }
    // the tokens from the first run that begins among the W on to the end of the last one that does
    const uint32_t begins = there & ~goes_on & ((1u << W) - 1);
    if (!begins) return;
    const int from = __builtin_ctz(begins);
    int end = 32 - __builtin_clz(begins);
    end += __builtin_ctzll(~(uint64_t)(goes_on >> end));  // (a run has 16 tokens at most)
    int8_t* cache = (isv ? c.v : c.k) + (int64_t)h * c.c.sh;
    float* scales = isv ? c.vs : c.ks;
    HeadRuns x[R];
    int slot[R], lead[R];  // lead: where the token's run begins; -1: none
#pragma unroll
    for (int r = 0; r < R; ++r) {
        lead[r] = -1;
        if (from + r * TOK >= end) continue;
        const int j = from + r * TOK + sub;
        if (j < end && (there >> j & 1)) {
            slot[r] = s_slot[j + 1];
            lead[r] = 31 - __builtin_clz(there & ~goes_on & ((2u << j) - 1));
        }
        const bool on = lane_on && lead[r] >= 0;
        x[r] = head_runs<GS, INTER>(a, n0 + j, a.hq + hh, p, on);
        const auto most = [](float u, float v) { return fmaxf(u, v); };
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(fmaxf(m, fabsf(x[r].x0[i])), fabsf(x[r].x1[i]));
        if (__any(on && m == __builtin_inff())) {  // of the finite ones
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = largest(largest(m, x[r].x0[i]), x[r].x1[i]);
        }
        m = over_group<GS>(on ? m : 0.0f, most);
        if (p == 0 && lead[r] >= 0) atomicMax(&s_max[lead[r]], __builtin_bit_cast(int, m));
    }
    __syncthreads();
    // A run's scale, by its first token's lanes.
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int j = from + r * TOK + sub;
        if (lead[r] < 0 || lead[r] != j) continue;
        const int page = slot[r] >> c.c.bs_log2, row = slot[r] & ((1 << c.c.bs_log2) - 1), held = row % GROUP;
        float* sp = scales + ((int64_t)page * c.hkv + h) * c.groups() + row / GROUP;
        const float need = __builtin_bit_cast(float, s_max[j]) / 127.0f, old = held ? held_scale(*sp) : 0.0f;
        const float s = fmaxf(need, old), inv = inverse_of(s);
        if (p == 0) s_inv[j] = inv, *sp = s;
        if (s > old && lane_on) {
            const float times = old * inv;
            int8_t* to = cache + page * c.c.sb + row * c.c.st + 8 * p;
            for (int i = 1; i <= held; ++i) {
                uint2* w = (uint2*)(to - i * c.c.st);
                *w = make_uint2(again(w->x, times), again(w->y, times));
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (lead[r] < 0 || !lane_on) continue;
        const float inv = s_inv[lead[r]];
        int8_t* to = cache + (slot[r] >> c.c.bs_log2) * c.c.sb + (slot[r] & ((1 << c.c.bs_log2) - 1)) * c.c.st;
        const f4 y0 = x[r].x0, y1 = x[r].x1;
        *(uint32_t*)(to + x[r].d0) = four_codes(y0[0], y0[1], y0[2], y0[3], inv);
        *(uint32_t*)(to + x[r].d1) = four_codes(y1[0], y1[1], y1[2], y1[3], inv);
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
