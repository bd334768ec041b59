// fq_plan.hip -- the plan of a step: prefix sums, cache blocks, slots, positions
// and tree masks.
//
// Bound by latency: one launch and no exchange between work-groups.  Each sums what
// the requests before its own bring (8 bytes a request, from L2 after the first
// reader), then each of its waves takes one request.  The kernel takes 5.6 us for 7
// trees of 25 tokens and 7.2 us for 1500 requests with 1 to 130 tokens each (an empty
// kernel: 2.4).  Ancestors by doubling: with m_i the set
// of token i and the ancestors within 2^s - 1 steps of it and a_i its ancestor 2^s steps up,
//   m_i <- m_i | m_{a_i},  a_i <- a_{a_i}
// covers all 64 tokens after six exchanges between the wave's lanes.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fq_step.h"

namespace fq {
namespace {

constexpr int WAVES = 16;

// ceil(n / block) as it is, and held to the table's columns.
struct Need {
    int64_t all;
    int held, fresh;
};
__device__ __forceinline__ Need need(const PlanArgs& a, int len, int nw) {
    const int64_t bs1 = (1ll << a.bs_log2) - 1;
    const int64_t have = (len + bs1) >> a.bs_log2, want = (len + (int64_t)nw + bs1) >> a.bs_log2;
    Need n;
    n.all = want - have;
    n.held = (int)min(have, (int64_t)a.max_blocks);
    n.fresh = (int)min(want, (int64_t)a.max_blocks) - n.held;
    return n;
}

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <bool TREE>
__global__ __launch_bounds__(WAVES * 64) void plan_kernel(PlanArgs a) {
    __shared__ int64_t s_sum[3][WAVES];
    __shared__ int64_t s_own[3][WAVES];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int b0 = blockIdx.x * WAVES, b = b0 + w;
    // what the requests before this work-group's bring: tokens, blocks of the
    // table, blocks in all
    int64_t tok = 0, blk = 0, all = 0;
    for (int i = threadIdx.x; i < b0; i += WAVES * 64) {
        const int nw = max(0, a.new_tokens[i]);
        const Need n = need(a, max(0, a.lengths[i]), nw);
        tok += nw;
        blk += n.fresh;
        all += n.all;
    }
    tok = wave_sum(tok), blk = wave_sum(blk), all = wave_sum(all);
    int len = 0, nw = 0;
    if (b < a.B) {
        len = max(0, a.lengths[b]);
        nw = max(0, a.new_tokens[b]);
    }
    const Need own = need(a, len, nw);
    if (lane == 0) {
        s_sum[0][w] = tok, s_sum[1][w] = blk, s_sum[2][w] = all;
        s_own[0][w] = nw, s_own[1][w] = own.fresh, s_own[2][w] = own.all;
    }
    __syncthreads();
    tok = blk = all = 0;
    for (int i = 0; i < WAVES; ++i) {
        tok += s_sum[0][i], blk += s_sum[1][i], all += s_sum[2][i];
        if (i < w) tok += s_own[0][i], blk += s_own[1][i], all += s_own[2][i];
    }
    const bool writer = blockIdx.y == 0;
    if (b < a.B) {
        if (writer) {
            if (lane == 0) {
                if (b == 0) a.cu[0] = 0;
                a.cu[b + 1] = (int)min(tok + nw, (int64_t)INT32_MAX);
            }
            for (int i = lane; i < own.fresh; i += 64)
                a.table[b * a.table_stride + own.held + i] =
                    blk + i < a.n_free ? a.free_blocks[blk + i] : -1;
        }
        const int bs1 = (1 << a.bs_log2) - 1;
        const auto slot = [&](int i) {
            const int64_t at = (int64_t)len + i, c = at >> a.bs_log2;
            if (c >= own.held + own.fresh) return -1;
            int e;
            if (c < own.held) {
                e = a.table[b * a.table_stride + c];
            } else {
                const int64_t f = blk + (c - own.held);
                e = f < a.n_free ? a.free_blocks[f] : -1;
            }
            // (of a block past what an int of slots reaches there is none)
            return e < 0 || e > INT32_MAX >> a.bs_log2 ? -1 : (e << a.bs_log2) + (int)(at & bs1);
        };
        const auto put = [&](int i, int pos, int s) {
            if (tok + i < a.N) {
                a.positions[tok + i] = pos;
                a.slots[tok + i] = s;
            }
        };
        if (TREE) {
            const int n = min(nw, 64);
            int up = lane;
            if (lane < n && tok + lane < a.N) {
                up = a.parents[tok + lane];
                if (up < 0 || up >= lane) up = lane;
            }
            uint64_t m = 1ull << lane;
            for (int s = 0; s < 6; ++s) {
                m |= (uint64_t)__shfl((unsigned long long)m, up);
                up = __shfl(up, up);
            }
            if (lane < n) {
                put(lane, len + __popcll(m) - 1, slot(lane));
                if (tok + lane < a.N) a.masks[tok + lane] = m;
            }
            for (int i = 64 + lane; i < nw && tok + i < a.N; i += 64) {
                put(i, len + 64, -1);
                a.masks[tok + i] = 0;
            }
        } else {
            for (int64_t i = blockIdx.y * 64 + lane; i < nw && tok + i < a.N; i += 64 * gridDim.y)
                put((int)i, len + (int)i, slot((int)i));
        }
    }
    // the last request's wave knows the totals
    if (b == a.B - 1 && writer) {
        if (lane == 0) {
            const int64_t t = min(blk + own.fresh, (int64_t)a.n_free);
            a.info[0] = (int)t;
            a.info[1] = (int)min(all + own.all - t, (int64_t)INT32_MAX);
        }
        for (int64_t i = tok + nw + lane; i < a.N; i += 64) {
            a.positions[i] = 0;
            a.slots[i] = -1;
            if (TREE) a.masks[i] = 0;
        }
    }
}

}  // namespace

hipError_t launch_plan(const PlanArgs& a, hipStream_t st) {
    const int gx = (a.B + WAVES - 1) / WAVES;
    if (a.parents) {
        hipLaunchKernelGGL((plan_kernel<true>), dim3(gx), dim3(WAVES * 64), 0, st, a);
    } else {
        // requests of many tokens (prompts) are shared by several work-groups (one of
        // 8000 tokens: 6.3 us, 30 on one; four of 1500: 6.8, 9.1 on one each)
        const int gy = std::max(1, std::min(64, a.N / (256 * a.B)));
        hipLaunchKernelGGL((plan_kernel<false>), dim3(gx, gy), dim3(WAVES * 64), 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace fq
