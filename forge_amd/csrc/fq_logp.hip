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
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fq_step.h"

namespace fq {
namespace {

constexpr int E = 16;  // elements of a lane and chunk
constexpr int CHUNK = 64 * E;
constexpr int MAXTOP = 64;
constexpr int KEEP = 128;      // kept keys from which a wave prunes them
constexpr int CAP = 2 * KEEP;  // and at most
constexpr int MAX_SPLITS = 16;
constexpr float LOWEST = -3.402823466e38f;
constexpr float LOG2E = 1.44269504088896341f;

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
// (the differences are held finite: a lane that has seen nothing has m = LOWEST)
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    const float da = fmaxf(a.m - r.m, -1e30f), db = fmaxf(b.m - r.m, -1e30f);
    const float ea = exp2f(da * LOG2E), eb = exp2f(db * LOG2E);
    r.s = ea * a.s + eb * b.s;
    r.t = ea * (a.t + da * a.s) + eb * (b.t + db * b.s);
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
    uint64_t key[WAVES * MAXTOP + 4];  // those to rank, one wave's after the other's, then 0
};

// Of one split: its statistics and its largest keys, in falling order.
struct Part {
    Stat st;
    int n;
    uint64_t key[MAXTOP];
};

// How many of the n keys (a multiple of 4) are above mine.
__device__ __forceinline__ int above(const uint64_t* key, int n, uint64_t mine) {
    int r = 0;
#pragma unroll 4
    for (int i = 0; i < n; i += 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) r += key[i + j] > mine;
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
    if (at + CHUNK <= end) {
#pragma unroll
        for (int i = 0; i < E / Run<TYPE>::N; ++i) {
            const int64_t x = row + index_of<TYPE>(at, i * Run<TYPE>::N);
            if (TYPE == 0) r.v[i] = *(const u4b*)((const float*)a.x + x);
            else r.v[i] = *(const u4a*)((const uint16_t*)a.x + x);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int x = index_of<TYPE>(at, i);
        if (TYPE == 0) {
            r.v[i / 4][i % 4] = x < end ? ((const uint32_t*)a.x)[row + x] : 0xFF800000u;
        } else {
            const uint32_t h = x < end ? ((const uint16_t*)a.x)[row + x] : TYPE == 1 ? 0xFC00u : 0xFF80u;
            r.v[i / 8][i % 8 / 2] = i & 1 ? r.v[i / 8][i % 8 / 2] | h << 16 : h;
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
    Stat st = {LOWEST, 0.0f, 0.0f};
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
#pragma unroll
                for (int o = 32; o; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o));
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
            for (int i = 0; i < E; ++i) {
                in[i] = __ballot(!(element<TYPE>(x, i) <= tau) && index_of<TYPE>(at, i) < end);
                hits += __popcll(in[i]);
            }
            const bool fits = n + hits <= CAP;
            if (fits && hits) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
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
    for (int o = 32; o; o >>= 1) {
        const Stat b = {__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.t, o)};
        st = join(st, b);
    }
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
    st = lane < WAVES ? l.st[lane] : Stat{LOWEST, 0.0f, 0.0f};
#pragma unroll
    for (int o = WAVES / 2; o; o >>= 1) {
        const Stat b = {__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.t, o)};
        st = join(st, b);
    }
    st = {__shfl(st.m, 0), __shfl(st.s, 0), __shfl(st.t, 0)};
    Part* p = (Part*)a.ws + (int64_t)m * a.splits + sp;
    if (a.splits == 1) emit<TYPE, T>(a, m, st, target, logit);
    else if (tid == 0) p->st = st, p->n = min(total, a.top);
    if (TOP && tid < total) {
        const uint64_t mine = l.key[tid];
        const int r = above(l.key, (total + 3) & ~3, mine);
        if (r < a.top) {
            if (a.splits == 1) emit_top(a, m, st, mine, r);
            else p->key[r] = mine;
        }
    }
}

// The splits' statistics and keys.
template <int TYPE>
__global__ __launch_bounds__(256) void logp_join(LogpArgs a) {
    __shared__ Stat s_st[MAX_SPLITS];
    __shared__ uint64_t s_key[MAX_SPLITS * MAXTOP];
    const int m = blockIdx.x, tid = threadIdx.x;
    const Part* p = (const Part*)a.ws + (int64_t)m * a.splits;
    int target;
    float logit;
    read_target<TYPE, 256>(a, m, target, logit);
    if (tid < a.splits) s_st[tid] = p[tid].st;
    const int n = a.splits * a.top;
    for (int i = tid; i < (n + 3) / 4 * 4; i += 256) s_key[i] = i < n && i % a.top < p[i / a.top].n ? p[i / a.top].key[i % a.top] : 0;
    __syncthreads();
    Stat st = s_st[0];
    for (int i = 1; i < a.splits; ++i) st = join(st, s_st[i]);
    emit<TYPE, 256>(a, m, st, target, logit);
    for (int i = tid; i < n; i += 256) {
        const uint64_t mine = s_key[i];
        if (!mine) continue;
        const int r = above(s_key, (n + 3) / 4 * 4, mine);
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

// 16 waves to a CU, in as few work-groups as there are rows for; a row on several CUs
// where its waves would take more than three chunks each.
template <int TYPE>
hipError_t waves(LogpArgs a, int cus, hipStream_t st) {
    const int chunks = (a.V + 16 * CHUNK - 1) / (16 * CHUNK);  // of one of 16 waves
    a.splits = chunks > 3 ? std::max(1, std::min({cus / a.M, chunks, MAX_SPLITS})) : 1;
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
