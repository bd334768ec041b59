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
// lowest token.  Of a group of elements that 256 threads hold, the top-th largest
// of the threads' own maxima is a threshold that at least top elements reach and that only
// top threads' elements can reach: what is left is few and ranked by counting.
// From the first chunk on only elements above the last kept one matter.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fq_step.h"

namespace fq {
namespace {

constexpr int T = 256;           // threads
constexpr int E = 16;            // elements of a thread and chunk
constexpr int CHUNK = T * E;
constexpr int MAXTOP = 64;
constexpr int CAND = MAXTOP * (E + 1);  // candidates at most: top threads' elements
constexpr int MAX_SPLITS = 128;
constexpr float LOWEST = -3.402823466e38f;
constexpr float LOG2E = 1.44269504088896341f;

typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u4b __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ uint64_t key_of(float x, uint32_t idx) {
    uint32_t b = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
    b = x != x ? 0xFFFFFFFFu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return ((uint64_t)b << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float value_of(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
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

struct Lds {
    uint64_t tmax[T];
    uint64_t cand[CAND];
    uint64_t list[MAXTOP];
    uint64_t tau;
    int n, any;
    Stat st[T / 64];
};

// The `top` largest of list and the threads' keys, in falling order, to list.
// Keys are unique, but for 0 (none).  Called by all threads.
template <int NK>
__device__ void select(Lds& l, const uint64_t (&k)[NK], int top, bool has_list) {
    const int tid = threadIdx.x;
    const uint64_t own = has_list && tid < top ? l.list[tid] : 0;
    uint64_t mx = own;
    for (int i = 0; i < NK; ++i) mx = k[i] > mx ? k[i] : mx;
    if (tid == 0) l.n = 0, l.tau = 1;
    l.tmax[tid] = mx;
    __syncthreads();
    if (mx) {
        int rank = 0;
        for (int i = 0; i < T; ++i) rank += l.tmax[i] > mx;
        if (rank == top - 1) l.tau = mx;
    }
    __syncthreads();
    const uint64_t tau = l.tau;
    if (mx >= tau) {
        if (own >= tau) l.cand[atomicAdd(&l.n, 1)] = own;
        for (int i = 0; i < NK; ++i)
            if (k[i] >= tau) l.cand[atomicAdd(&l.n, 1)] = k[i];
    }
    __syncthreads();
    const int n = l.n;
    if (tid < top) l.list[tid] = 0;
    __syncthreads();
    for (int c = tid; c < n; c += T) {
        const uint64_t mine = l.cand[c];
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += l.cand[i] > mine;
        if (rank < top) l.list[rank] = mine;
    }
    __syncthreads();
}

template <int TYPE>
__device__ __forceinline__ float load1(const LogpArgs& a, int64_t at) {
    if (TYPE == 0) return ((const float*)a.x)[at];
    if (TYPE == 1) return (float)((const _Float16*)a.x)[at];
    return __uint_as_float((uint32_t)((const uint16_t*)a.x)[at] << 16);
}

// A thread's E elements of a chunk: runs of 16 bytes, T runs apart.
template <int TYPE>
struct Run {
    static constexpr int N = TYPE == 0 ? 4 : 8;
};

template <int TYPE>
__device__ __forceinline__ void load(const LogpArgs& a, int64_t row, int at, int end,
                                     float (&x)[E], bool whole) {
    constexpr int RN = Run<TYPE>::N;
    if (whole) {
        for (int r = 0; r < E / RN; ++r) {
            const int i = at + (r * T + threadIdx.x) * RN;
            if (TYPE == 0) {
                const u4b v = *(const u4b*)((const float*)a.x + row + i);
                for (int e = 0; e < 4; ++e) x[4 * r + e] = __uint_as_float(v[e]);
            } else {
                const u4a v = *(const u4a*)((const uint16_t*)a.x + row + i);
                for (int e = 0; e < 8; ++e) {
                    const uint32_t h = (v[e / 2] >> (16 * (e & 1))) & 0xFFFFu;
                    x[8 * r + e] = TYPE == 1 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h)
                                             : __uint_as_float(h << 16);
                }
            }
        }
        return;
    }
    for (int r = 0; r < E / RN; ++r)
        for (int e = 0; e < RN; ++e) {
            const int i = at + (r * T + threadIdx.x) * RN + e;
            x[r * RN + e] = i < end ? load1<TYPE>(a, row + i) : -__builtin_inff();
        }
}

// Of one split: its statistics and its largest keys.
struct Part {
    Stat st;
    uint32_t pad;
    uint64_t key[MAXTOP];
};

template <int TYPE>
__device__ void finish(const LogpArgs& a, Lds& l, int m, Stat st) {
    const float ls = logf(st.s);  // nothing but -inf: -inf; NaN or inf: NaN
    for (int j = threadIdx.x; j < a.J; j += T) {
        const int t = a.targets[(int64_t)m * a.J + j];
        const bool in = (unsigned)t < (unsigned)a.V;
        const float x = in ? load1<TYPE>(a, (int64_t)m * a.ld + t) : 0.0f;
        a.logprobs[(int64_t)m * a.J + j] = in && st.s > 0.0f ? (x - st.m) - ls : __builtin_nanf("");
    }
    if (threadIdx.x == 0 && a.entropy)
        a.entropy[m] = st.s > 0.0f ? ls - st.t / st.s : __builtin_nanf("");
    if (threadIdx.x < a.top) {
        const uint64_t k = l.list[threadIdx.x];
        const uint32_t tok = 0xFFFFFFFFu - (uint32_t)k;
        a.top_tokens[(int64_t)m * a.top + threadIdx.x] = (int)tok;
        a.top_logprobs[(int64_t)m * a.top + threadIdx.x] =
            st.s > 0.0f ? (value_of(k) - st.m) - ls : __builtin_nanf("");
    }
}

__device__ __forceinline__ Stat block_join(Lds& l, Stat st) {
    for (int o = 32; o; o >>= 1) {
        const Stat b = {__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.t, o)};
        st = join(st, b);
    }
    if ((threadIdx.x & 63) == 0) l.st[threadIdx.x >> 6] = st;
    __syncthreads();
    st = l.st[0];
    for (int i = 1; i < T / 64; ++i) st = join(st, l.st[i]);
    return st;
}

template <int TYPE>
__global__ __launch_bounds__(T) void logp_kernel(LogpArgs a) {
    __shared__ Lds l;
    const int m = blockIdx.x / a.splits, sp = blockIdx.x % a.splits;
    const int64_t row = (int64_t)m * a.ld;
    const int beg = sp * a.seg, end = min(a.V, beg + a.seg);
    Stat st = {LOWEST, 0.0f, 0.0f};
    float tau = __builtin_nanf("");  // everything is above NaN
    for (int at = beg; at < end; at += CHUNK) {
        float x[E];
        const bool whole = at + CHUNK <= end;
        load<TYPE>(a, row, at, end, x, whole);
        float cm = st.m;
        for (int i = 0; i < E; ++i) cm = fmaxf(cm, x[i]);
        if (cm > st.m) {
            const float d = fmaxf(st.m - cm, -1e30f), e = exp2f(d * LOG2E);
            st.t = e * (st.t + d * st.s);
            st.s *= e;
            st.m = cm;
        }
        for (int i = 0; i < E; ++i) {
            const float d = x[i] - st.m, e = exp2f(d * LOG2E);
            st.s += e;
            st.t = fmaf(e, fmaxf(d, -1e30f), st.t);
        }
        if (a.top) {
            bool more = false;
            for (int i = 0; i < E; ++i) more |= !(x[i] <= tau);
            if (__syncthreads_or(more)) {
                constexpr int RN = Run<TYPE>::N;
                uint64_t k[E];
                for (int i = 0; i < E; ++i) {
                    const int idx = at + ((i / RN) * T + threadIdx.x) * RN + i % RN;
                    k[i] = idx < end && !(x[i] <= tau) ? key_of(x[i], idx) : 0;
                }
                select(l, k, a.top, at > beg);
                const uint64_t last = l.list[a.top - 1];
                tau = last ? value_of(last) : __builtin_nanf("");
            }
        }
    }
    st = block_join(l, st);
    if (a.splits == 1) {
        finish<TYPE>(a, l, m, st);
        return;
    }
    Part* p = (Part*)a.ws + (int64_t)m * a.splits + sp;
    if (threadIdx.x == 0) p->st = st;
    if (threadIdx.x < a.top) p->key[threadIdx.x] = l.list[threadIdx.x];
}

template <int TYPE>
__global__ __launch_bounds__(T) void logp_join(LogpArgs a) {
    __shared__ Lds l;
    const int m = blockIdx.x;
    const Part* p = (const Part*)a.ws + (int64_t)m * a.splits;
    Stat st = {LOWEST, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < a.splits; i += T) st = join(st, p[i].st);
    st = block_join(l, st);
    const int n = a.splits * a.top;
    for (int at = 0; at < n; at += CHUNK) {
        uint64_t k[E];
        for (int i = 0; i < E; ++i) {
            const int c = at + i * T + threadIdx.x;
            k[i] = c < n ? p[c / a.top].key[c % a.top] : 0;
        }
        select(l, k, a.top, at > 0);
    }
    finish<TYPE>(a, l, m, st);
}

constexpr int TARGET_WGS = 1024;

}  // namespace

// Splits only where the rows alone leave work-groups to place: splits * M < 2
// TARGET_WGS.
size_t logp_part_bytes() { return (size_t)2 * TARGET_WGS * sizeof(Part); }

hipError_t launch_logp(LogpArgs a, int type, int, uint8_t* ws, hipStream_t st) {
    const int chunks = (a.V + CHUNK - 1) / CHUNK;
    int splits = std::max(1, std::min({chunks, TARGET_WGS / a.M, MAX_SPLITS}));
    a.seg = (chunks + splits - 1) / splits * CHUNK;
    a.splits = (a.V + a.seg - 1) / a.seg;
    a.ws = ws;
    const dim3 g(a.splits * a.M), t(T);
    const auto two = [&](auto k1, auto k2) {
        hipLaunchKernelGGL(k1, g, t, 0, st, a);
        if (a.splits > 1) hipLaunchKernelGGL(k2, dim3(a.M), t, 0, st, a);
        return hipGetLastError();
    };
    if (type == 0) return two(logp_kernel<0>, logp_join<0>);
    if (type == 1) return two(logp_kernel<1>, logp_join<1>);
    return two(logp_kernel<2>, logp_join<2>);
}

}  // namespace fq
