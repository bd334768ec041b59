// fq_logp.hip -- log probabilities of given tokens, entropy and the largest
// logits of each row, in one pass over the logits.
//
// With m the running maximum, s = sum e^(x - m) and t = sum e^(x - m) (x - m):
// log p = x - m - log s and the entropy is log s - t / s.  Moving m to m' = m - d
// (d <= 0) takes t' = e^d (t + d s), s' = e^d s.  Every lane keeps its own
// (m, s, t); they are joined at the end.
//
// The largest logits are found through unique 64-bit keys, the value's
// order-preserving bits above the inverted token number, so that ties go to the
// lowest token.  A work-group takes a row, each wave a part of it, 1024 elements at
// a time, and keeps in LDS what may belong to the largest.  Of the first 1024 elements
// of W waves each, the q = ceil(top / W) th largest of a wave's lanes' maxima is reached
// by q elements of it, so the least of these over the waves by top of the row:
// all that is below it is out.  Past KEEP kept keys the top-th largest of a wave's
// becomes its threshold.  At the end the waves' keys are ranked by counting.  Few
// rows are split over several work-groups, whose results a second kernel joins.
//
// Bound: the bytes of the logits once where there are many rows of many tokens (501 x
// 152064 fp32, top 20: 60 to 62 us, 5.0 TB/s; 50 us with top 0; a large copy runs at 5.2
// TB/s), what a row costs for its largest on rows of few chunks (1000 x 32000 bf16: 36 us
// with top 20, 26 with top 1, 14 with top 0, where the bytes take 12), latency for few
// (5 x 32000 fp32: 11 us, one work-group a row).  NaN logits rank above all and have no
// threshold: rows of nothing else keep and prune every key (501 x 152064: 1500 us; 64 x
// 32000 52 us with 1 % of NaN, 21 without).
// No barrier lies between a wave's chunks, and a chunk's elements cost no test
// against the row's end except in its last one: the loop is bound by instructions
// where the logits come fast.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "fq_step.h"

namespace fq {
namespace {

constexpr int E = 16;  // elements of a lane and chunk
constexpr int CHUNK = 64 * E;
constexpr int MAXTOP = 64;
constexpr int KEEP = 128;      // kept keys from which a wave prunes them
constexpr int CAP = 2 * KEEP;  // and at most
constexpr int MAX_SPLITS = 32;
constexpr int MAX_KEYS = 256;  // of a row's splits together
constexpr float LOWEST = -3.402823466e38f;
constexpr float LOG2E = 1.44269504088896341f;

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint64_t k2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u4b __attribute__((ext_vector_type(4), aligned(4)));

// Unsigned integers in the order of the values; -0 and 0 are equal, NaN the largest.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0xFFFFFFFFu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t idx) {
    return ((uint64_t)order_of(x) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float value_of(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}

// The next smaller value (of 0 not -0, which is equal; of -inf NaN).
__device__ __forceinline__ float below_value(uint32_t order) {
    return value_of((uint64_t)(order - (order == 0x80000000u ? 2 : 1)) << 32);
}

struct Stat {
    float m, s, t;
};
constexpr Stat NOTHING = {LOWEST, 0.0f, 0.0f};

// f over all lanes, in every lane: by turns within the rows of 16, then swaps of rows.
template <class T, class F>
__device__ __forceinline__ T over_wave(T x, F f) {
    const auto turned = [&](auto n) {
        return __builtin_bit_cast(
            T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + n.value, 0xF, 0xF, false));
    };
    x = f(x, turned(std::integral_constant<int, 8>()));
    x = f(x, turned(std::integral_constant<int, 4>()));
    x = f(x, turned(std::integral_constant<int, 2>()));
    x = f(x, turned(std::integral_constant<int, 1>()));
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const u2 p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    const uint32_t p0 = p[0], p1 = p[1];  // (a bit cast of an element would take element 0)
    x = f(__builtin_bit_cast(T, p0), __builtin_bit_cast(T, p1));
    const uint32_t v = __builtin_bit_cast(uint32_t, x);
    const u2 q = __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(v, v, false, false));
    const uint32_t q0 = q[0], q1 = q[1];
    return f(__builtin_bit_cast(T, q0), __builtin_bit_cast(T, q1));
}
// The lanes' statistics as one.  (The differences are held finite: a lane that has seen
// nothing has m = LOWEST.)
__device__ __forceinline__ Stat join(Stat a) {
    const auto add = [](float x, float y) { return x + y; };
    Stat r;
    r.m = over_wave(a.m, [](float x, float y) { return fmaxf(x, y); });
    const float d = fmaxf(a.m - r.m, -1e30f), e = exp2f(d * LOG2E);
    r.s = over_wave(e * a.s, add);
    r.t = over_wave(e * (a.t + d * a.s), add);
    return r;
}

template <int TYPE>
__device__ __forceinline__ float load1(const LogpArgs& a, int64_t at) {
    if (TYPE == 0) return ((const float*)a.x)[at];
    if (TYPE == 1) return (float)((const _Float16*)a.x)[at];
    return __uint_as_float((uint32_t)((const uint16_t*)a.x)[at] << 16);
}

template <int WAVES>
struct Lds {
    Stat st[WAVES];
    int n[WAVES];
    uint32_t first[WAVES];         // the waves' thresholds after their first elements
    uint64_t buf[WAVES][CAP];      // the waves' kept keys
    alignas(16) uint64_t key[WAVES * MAXTOP + 4];  // those to rank, one wave's after the other's, then 0
};

// Of one split: its statistics and its largest keys, in falling order, then 0.
struct Part {
    Stat st;
    uint64_t key[MAXTOP];
};

// How many of the n keys (a multiple of 4) are above mine.
__device__ __forceinline__ int above(const uint64_t* key, int n, uint64_t mine) {
    int r = 0;
#pragma unroll 4
    for (int i = 0; i < n; i += 4) {
        const k2 a = *(const k2*)(key + i), b = *(const k2*)(key + i + 2);
        r += (a[0] > mine) + (a[1] > mine) + (b[0] > mine) + (b[1] > mine);
    }
    return r;
}

// A row's results from its statistics: the targets' by thread j < J (target and logit
// read ahead), the entropy, ..
template <int TYPE, int T>
__device__ __forceinline__ void emit(const LogpArgs& a, int m, Stat st, int target, float logit) {
    const int tid = threadIdx.x;
    const float ls = logf(st.s);  // nothing but -inf: s = 0; NaN or +inf among them: s = NaN
    const bool fine = st.s > 0.0f;
    for (int j = tid; j < a.J; j += T) {
        if (j != tid) {
            target = a.targets[(int64_t)m * a.J + j];
            if ((unsigned)target < (unsigned)a.V) logit = load1<TYPE>(a, (int64_t)m * a.ld + target);
        }
        a.logprobs[(int64_t)m * a.J + j] =
            (unsigned)target < (unsigned)a.V && fine ? (logit - st.m) - ls : __builtin_nanf("");
    }
    if (tid == 0 && a.entropy) a.entropy[m] = fine ? ls - st.t / st.s : __builtin_nanf("");
}
// .. and the r-th largest logit.
__device__ __forceinline__ void emit_top(const LogpArgs& a, int m, Stat st, uint64_t key, int r) {
    const int64_t at = (int64_t)m * a.top + r;
    a.top_tokens[at] = (int)(0xFFFFFFFFu - (uint32_t)key);
    a.top_logprobs[at] = st.s > 0.0f ? (value_of(key) - st.m) - logf(st.s) : __builtin_nanf("");
}
template <int TYPE, int T>
__device__ __forceinline__ void read_target(const LogpArgs& a, int m, int& target, float& logit) {
    target = -1;
    logit = 0.0f;
    if ((int)threadIdx.x < a.J) {
        target = a.targets[(int64_t)m * a.J + threadIdx.x];
        if ((unsigned)target < (unsigned)a.V) logit = load1<TYPE>(a, (int64_t)m * a.ld + target);
    }
}

__device__ __forceinline__ uint64_t below(int lane) { return (1ull << lane) - 1; }

// Of the n <= CAP keys at buf (one wave's) the top largest, to buf[0 .. top) in any
// order; returns how many are left.  The top-th largest is found bit by bit.
__device__ __forceinline__ int prune(uint64_t* buf, int n, int top, uint64_t& last) {
    const int lane = threadIdx.x & 63;
    constexpr int J = CAP / 64;
    uint64_t k[J];
    __builtin_amdgcn_wave_barrier();  // (other lanes' keys are read)
#pragma unroll
    for (int j = 0; j < J; ++j) k[j] = 64 * j + lane < n ? buf[64 * j + lane] : 0;
    uint64_t tau = 1;
    if (n > top) {
        tau = 0;
#pragma unroll 1
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t t = tau | (1ull << bit);
            int c = 0;
#pragma unroll
            for (int j = 0; j < J; ++j) c += __popcll(__ballot(k[j] >= t));
            if (c >= top) tau = t;
            if (c == top) break;
        }
    }
    int at = 0;
    last = ~0ull;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const bool keep = k[j] >= tau;
        const uint64_t b = __ballot(keep);
        if (keep) {
            buf[at + __popcll(b & below(lane))] = k[j];
            last = k[j] < last ? k[j] : last;
        }
        at += __popcll(b);
    }
    for (int o = 32; o; o >>= 1) {
        const uint64_t v = __shfl_xor((unsigned long long)last, o);
        last = v < last ? v : last;
    }
    return at;
}
// A lane's E elements of a wave's chunk: runs of 16 bytes, 64 runs apart.
template <int TYPE>
struct Run {
    static constexpr int N = TYPE == 0 ? 4 : 8;
    u4a v[E / N];
};
template <int TYPE>
__device__ __forceinline__ int index_of(int at, int i) {
    constexpr int RN = Run<TYPE>::N;
    return at + ((i / RN) * 64 + (threadIdx.x & 63)) * RN + i % RN;
}

template <int TYPE>
__device__ __forceinline__ void load(const LogpArgs& a, int64_t row, int at, int end, Run<TYPE>& r) {
    constexpr int RN = Run<TYPE>::N;
#pragma unroll
    for (int i = 0; i < E / RN; ++i) {
        const int x = index_of<TYPE>(at, i * RN);
        if (x + RN <= end) {
            if (TYPE == 0) r.v[i] = *(const u4b*)((const float*)a.x + row + x);
            else r.v[i] = *(const u4a*)((const uint16_t*)a.x + row + x);
            continue;
        }
        // the row's last run, and -inf behind it
#pragma unroll
        for (int j = 0; j < RN; ++j) {
            if (TYPE == 0) {
                r.v[i][j % 4] = x + j < end ? ((const uint32_t*)a.x)[row + x + j] : 0xFF800000u;
            } else {
                const uint32_t h = x + j < end ? ((const uint16_t*)a.x)[row + x + j] : TYPE == 1 ? 0xFC00u : 0xFF80u;
                r.v[i][j / 2] = j & 1 ? r.v[i][j / 2] | h << 16 : h;
            }
        }
    }
}
template <int TYPE>
__device__ __forceinline__ float element(const Run<TYPE>& r, int i) {
    if (TYPE == 0) return __uint_as_float(r.v[i / 4][i % 4]);
    const uint32_t h = (r.v[i / 8][i % 8 / 2] >> (16 * (i & 1))) & 0xFFFFu;
    return TYPE == 1 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
}

template <int TYPE, int WAVES, bool TOP>
__global__ __launch_bounds__(64 * WAVES, WAVES == 16 ? 4 : 16 / WAVES) void logp_kernel(LogpArgs a) {
    constexpr int T = 64 * WAVES;
    __shared__ Lds<WAVES> l;
    const int m = blockIdx.x / a.splits, sp = blockIdx.x % a.splits;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = (int64_t)m * a.ld;
    const int from = sp * WAVES * a.seg;  // (the work-group's part)
    const int beg = min(a.V, from + w * a.seg), end = min(a.V, beg + a.seg);
    uint64_t* buf = l.buf[w];
    int target;
    float logit;  // (on their way early)
    if (a.splits == 1) read_target<TYPE, T>(a, m, target, logit);
    int n = 0;
    Stat st = NOTHING;
    float tau = __builtin_nanf("");  // (nothing is <= NaN: all is kept)
    Run<TYPE> next;
    if (beg < end) load<TYPE>(a, row, beg, end, next);
    for (int at = beg; at < end || (TOP && at == beg); at += CHUNK) {
        const Run<TYPE> x = next;
        if (at + CHUNK < end) load<TYPE>(a, row, at + CHUNK, end, next);
        if (TOP && at == beg) {
            // (also by waves without elements: all wait for each other here)
            uint32_t mx = 0;
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (index_of<TYPE>(at, i) < end) mx = max(mx, order_of(element<TYPE>(x, i)));
            const int active = min(WAVES, (a.V - from + a.seg - 1) / a.seg);
            const int q = (a.top + active - 1) / active;
            int r = 0;
            if (q == 1) {
                mx = over_wave(mx, [](uint32_t x, uint32_t y) { return max(x, y); });
                r = lane;
            } else {
#pragma unroll 8
                for (int i = 0; i < 64; ++i) {
                    const uint32_t o = __builtin_amdgcn_readlane(mx, i);
                    r += o > mx || (o == mx && i < lane);
                }
            }
            if (r == q - 1) l.first[w] = w < active ? mx : ~0u;  // (0: too few elements)
            __syncthreads();
            uint32_t least = l.first[0];
#pragma unroll
            for (int v = 1; v < WAVES; ++v) least = min(least, l.first[v]);
            // (what equals the threshold is kept, as its token may be lower)
            if (least > order_of(-__builtin_inff())) tau = below_value(least);
        }
        if (at >= end) break;
        float cm = st.m;
#pragma unroll
        for (int i = 0; i < E; ++i) cm = fmaxf(cm, element<TYPE>(x, i));
        if (cm > st.m) {
            const float d = fmaxf(st.m - cm, -1e30f), e = __builtin_amdgcn_exp2f(d * LOG2E);
            st.t = e * (st.t + d * st.s);
            st.s *= e;
            st.m = cm;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float d = element<TYPE>(x, i) - st.m, e = __builtin_amdgcn_exp2f(d * LOG2E);
            st.s += e;
            st.t = fmaf(e, fmaxf(d, -1e30f), st.t);
        }
        if (TOP) {
            uint64_t in[E];
            int hits = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) in[i] = __ballot(!(element<TYPE>(x, i) <= tau));
            if (at + CHUNK > end) {
#pragma unroll
                for (int i = 0; i < E; ++i) in[i] &= __ballot(index_of<TYPE>(at, i) < end);
            }
#pragma unroll
            for (int i = 0; i < E; ++i) hits += __popcll(in[i]);
            const bool fits = n + hits <= CAP;
            if (fits && hits) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    if (!in[i]) continue;  // (uniform: most have none)
                    if (in[i] >> lane & 1)
                        buf[n + __popcll(in[i] & below(lane))] = key_of(element<TYPE>(x, i), index_of<TYPE>(at, i));
                    n += __popcll(in[i]);
                }
            }
            // Too many kept: the largest of them.  (Too many for the place at once: 64 at a
            // time, read again.  What equals a threshold may come before it in the same
            // chunk, and is behind it from the next on.)
            float after = tau;
#pragma unroll 1
            for (int i = fits ? E - 1 : 0; i < E && (!fits || n > KEEP); ++i) {
                if (!fits) {
                    const int idx = index_of<TYPE>(at, i);
                    const float v = idx < end ? load1<TYPE>(a, row + idx) : 0.0f;
                    const bool add = idx < end && !(v <= tau);
                    const uint64_t b = __ballot(add);
                    if (add) buf[n + __popcll(b & below(lane))] = key_of(v, idx);
                    n += __popcll(b);
                }
                if (n > KEEP) {
                    uint64_t last;
                    n = prune(buf, n, a.top, last);
                    tau = below_value((uint32_t)(last >> 32));
                    after = value_of(last);
                }
            }
            tau = after;
        }
    }
    // --- the waves together ---
    st = join(st);
    if (TOP) {
        uint64_t last;
        if (n > MAXTOP / 2 && n > a.top) n = prune(buf, n, a.top, last);
    }
    if (lane == 0) l.st[w] = st, l.n[w] = n;
    __syncthreads();
    int total = 0;
    if (TOP) {
        int before = 0;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            before += v < w ? l.n[v] : 0;
            total += l.n[v];
        }
        if (lane < n) l.key[before + lane] = buf[lane];
        if (w == 0 && lane < 4) l.key[total + lane] = 0;
        __syncthreads();
    }
    if (w > 0 && 64 * w >= max(total, a.J)) return;  // nothing to write for this wave
    st = join(lane < WAVES ? l.st[lane] : NOTHING);
    Part* p = (Part*)a.ws + (int64_t)m * a.splits + sp;
    if (a.splits == 1) emit<TYPE, T>(a, m, st, target, logit);
    else if (tid == 0) p->st = st;
    if (TOP && tid < total) {
        const uint64_t mine = l.key[tid];
        const int r = above(l.key, (total + 3) & ~3, mine);
        if (r < a.top) {
            if (a.splits == 1) emit_top(a, m, st, mine, r);
            else p->key[r] = mine;
        }
    }
    if (TOP && a.splits > 1 && tid >= total && tid < a.top) p->key[tid] = 0;
}

// The splits' statistics and keys.
template <int TYPE>
__global__ __launch_bounds__(256) void logp_join(LogpArgs a) {
    __shared__ alignas(16) uint64_t s_key[MAX_KEYS + 4];
    const int m = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const Part* p = (const Part*)a.ws + (int64_t)m * a.splits;
    int target;
    float logit;
    read_target<TYPE, 256>(a, m, target, logit);
    Stat st = lane < a.splits ? p[lane].st : NOTHING;
    const int n = a.splits * a.top;
    for (int i = tid; i < n + 3; i += 256) s_key[i] = i < n ? p[i / a.top].key[i % a.top] : 0;
    __syncthreads();
    st = join(st);
    emit<TYPE, 256>(a, m, st, target, logit);
    for (int i = tid; i < n; i += 256) {
        const uint64_t mine = s_key[i];
        if (!mine) continue;
        const int r = above(s_key, (n + 3) & ~3, mine);
        if (r < a.top) emit_top(a, m, st, mine, r);
    }
}

template <int TYPE, int WAVES>
hipError_t go(LogpArgs a, hipStream_t st) {
    const int waves = a.splits * WAVES;
    a.seg = ((a.V + waves - 1) / waves + 511) / 512 * 512;  // whole runs of 64 lanes
    a.splits = (a.V + WAVES * a.seg - 1) / (WAVES * a.seg);
    const dim3 g(a.splits * a.M), t(64 * WAVES);
    if (a.top) hipLaunchKernelGGL((logp_kernel<TYPE, WAVES, true>), g, t, 0, st, a);
    else hipLaunchKernelGGL((logp_kernel<TYPE, WAVES, false>), g, t, 0, st, a);
    if (a.splits > 1) hipLaunchKernelGGL(logp_join<TYPE>, dim3(a.M), dim3(256), 0, st, a);
    return hipGetLastError();
}

// 16 waves to a CU, in as few work-groups as there are rows for (us, 152064 fp32
// logits, top 20, on 4 / 8 / 16 waves a row: 256 rows 66 / 47 / 47, 300 rows 74 / 66 /
// 82, 600 rows 95 / 94 / 129; 1000 rows of 32000 bf16: 42 / 50 / 61).  Few rows take
// several work-groups of 8 waves each where these would have more than six chunks
// each otherwise (1 x 60000: 9.6 us for both kernels, unsplit 17; 64 x 152064: 23.4,
// unsplit 42; 1 x 32000: 8.1 and the second launch, unsplit 10.0), as many as bring one
// key to a thread of the join (1 x 152064, top 20: 15.6 with 256 keys, 19.2 with 512).
template <int TYPE>
hipError_t waves(LogpArgs a, int cus, hipStream_t st) {
    const int chunks = (a.V + 8 * CHUNK - 1) / (8 * CHUNK);  // of one of 8 waves
    a.splits = std::min({cus / a.M, MAX_KEYS / std::max(a.top, 1), chunks, MAX_SPLITS});
    if (chunks > 6 && a.splits > 1) return go<TYPE, 8>(a, st);
    a.splits = 1;
    if (a.M <= cus) return go<TYPE, 16>(a, st);
    if (a.M <= 2 * cus) return go<TYPE, 8>(a, st);
    return go<TYPE, 4>(a, st);
}

}  // namespace

size_t logp_part_bytes(int cus) { return (size_t)cus * sizeof(Part); }

hipError_t launch_logp(const LogpArgs& a, int type, int cus, hipStream_t st) {
    return type == 0 ? waves<0>(a, cus, st) : type == 1 ? waves<1>(a, cus, st) : waves<2>(a, cus, st);
}

}  // namespace fq
