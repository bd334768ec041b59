// fq_verify.hip -- drafted tokens against the target's probabilities.
//
// Three or four launches.  Statistics: every row's largest logit m and s = sum e^((x - m) / T)
// (at temperatures of 0 or below its first largest), one pass over the logits in 32 bits, rows cut into parts
// where there are few.  Walk: what is accepted.  Whether a token is, were it tried, depends on
// its earlier siblings alone: u (s - sum of their e) < e, e = e^((x - m) / T) of the token's logit, so that all
// tests are made at once, a lane a token, and the walk goes over bits.  s is the statistics', in 32 bits:
// a test on the walk's way whose two sides are nearer to each other than s is exact is made again with
// the row's sum in 64 bits (one in 2^14 or so at 152064 tokens, at random numbers; one wave
// sums them alone).  The same launch sums e of
// each request's last accepted row, without the refused tokens, over chunks in 64 bits (a random number within
// 1e-7 of a border of the cumulated sum would find another token in 32: at 150000
// tokens one number in a hundred).  With draft probabilities, whose subtraction needs the
// whole sum first, another launch sums what is left.  Pick: the chunk in which the sum passes the random number, then
// the token in it.
//
// Bound: the bytes of the logits, read once; a row of each request is read again.  32 trees of up to 25 tokens,
// 152064 fp32 logits (400 rows, 243 MB): 43 us for the statistics, 5.6 TB/s, 14 for the walk, 8 for the pick.  One
// chain of 6 x 32000 with draft probabilities: 3.5, 7.9, 5.0 and 7.4, each a launch's latency and loads that follow
// one another; of given tokens 3.4, 7.8 and 6.7; 64 requests of one token, 152064: 8.4, 18.4 and 7.8.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fq_search.h"
#include "fq_step.h"

namespace fq {
namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(2)));

constexpr float LOWEST = -3.402823466e38f;
constexpr float LOG2E = 1.44269504088896341f;
constexpr int E = 16;             // elements of a lane at a time
constexpr int STEP = 256 * E;     // of a work-group
constexpr int MAX_STATS = 1 << 20;
constexpr int MAX_SUMS = 1 << 18;  // chunks of all requests
constexpr int LANES = 64;          // tokens of a request whose parents count
// Temperatures between which the statistics' exponents, in 32 bits, neither overflow nor lose bits: 2^-100, 2^100.
constexpr float FAR_LOW = 7.8886091e-31f, FAR_HIGH = 1.2676506e30f;

struct Stat {
    float m, s;  // s: NaN for a row with NaN or +inf, 0 for one of -inf alone; > 0 otherwise
    int first;   // the first largest, at temperatures of 0 and below
    int pad;
};
// What the walk leaves of a request.
struct Left {
    int row;      // the last accepted token's row; -1: no next token
    int q;        // the row of draft probabilities to take off; -1: none
    int refused;  // how many tokens are taken out
    int best;     // the next token where it is known already; -1
    float m;      // the row's largest
    int token[LANES];
};
struct Space {
    Stat* stats;
    Left* left;
    double *whole, *rest;  // [B][chunks]
    int chunks, chunk;
    float unsure;  // what part of itself a row's sum of the statistics is off by at most
};

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <int TYPE>
__device__ __forceinline__ float load1(const void* x, int64_t at) {
    if (TYPE == 0) return ((const float*)x)[at];
    if (TYPE == 1) return (float)((const _Float16*)x)[at];
    return __uint_as_float((uint32_t)((const uint16_t*)x)[at] << 16);
}

// 16 elements of a lane: those of a work-group's step lie in runs of 16 bytes a lane.
template <int TYPE>
__device__ __forceinline__ int64_t place16(int i) {  // of element i of this lane in the step
    constexpr int R = TYPE == 0 ? 4 : 8;
    return (int64_t)(i / R) * 256 * R + threadIdx.x * R + i % R;
}
template <int TYPE>
__device__ __forceinline__ void load16(const void* x, int64_t at, int64_t end, float (&v)[E]) {
    if (at + STEP <= end) {
        if constexpr (TYPE == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f4u w = *(const f4u*)((const float*)x + at + place16<TYPE>(4 * k));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * k + e] = w[e];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const u4a w = *(const u4a*)((const uint16_t*)x + at + place16<TYPE>(8 * k));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint16_t b = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                    v[8 * k + e] = TYPE == 1 ? (float)__builtin_bit_cast(_Float16, b) : __uint_as_float((uint32_t)b << 16);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int64_t j = at + place16<TYPE>(i);
            v[i] = j < end ? load1<TYPE>(x, j) : -__builtin_inff();
        }
    }
}

// e^y for y <= 0 in 64 bits: y = n ln 2 + r, |r| <= ln 2 / 2, and e^r by its series up to r^12 / 12!, 2e-16
// of it off (the remainder r^13 / 13! is below 1.7e-16).  Below e^-1000 nothing.
__device__ __forceinline__ double exp_of(double y) {
    y = fmax(y, -1000.0);
    const double n = rint(y * 1.4426950408889634074);
    double r = fma(n, -744261117.0 / 1073741824.0, y);  // (ln 2's first 30 bits, whose products are exact; the rest)
    r = fma(n, -8.893134238886677e-10, r);
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)n);
}

template <int TYPE, bool TEMP>
__global__ __launch_bounds__(256) void stats_kernel(VerifyArgs a, Space w) {
    const int n = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    __shared__ float s_m[4], s_s[4];
    __shared__ int s_i[4];
    float T = 1.0f;
    if (TEMP) T = a.temperature[request_of(a.cu, a.B, n)];
    const int64_t row = (int64_t)n * a.ld, from = (int64_t)part * a.seg, to = std::min<int64_t>(from + a.seg, a.V);
    float m = LOWEST, s = 0.0f;
    int first = 0x7FFFFFFF;
    if (!TEMP || T > 0.0f) {
        const float k = TEMP ? fminf(LOG2E / T, 3e38f) : LOG2E;
        for (int64_t at = from; at < to; at += STEP) {
            float v[E];
            load16<TYPE>(a.x, row + at, row + to, v);
            float mx = v[0];
#pragma unroll
            for (int i = 1; i < E; ++i) mx = fmaxf(mx, v[i]);
            mx = fmaxf(mx, m);
            float sum[2] = {s * exp2f((m - mx) * k), 0.0f};
            m = mx;
#pragma unroll
            for (int i = 0; i < E; ++i) sum[i & 1] += __builtin_amdgcn_exp2f((v[i] - m) * k);
            s = sum[0] + sum[1];
        }
        float mx = m;
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        if (lane == 0) s_m[wave] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
        s = m == mx ? s : s * exp2f((m - mx) * k);  // (an infinity less itself is NaN already)
        for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
        if (lane == 0) s_s[wave] = s;
        __syncthreads();
        if (tid == 0) w.stats[blockIdx.x] = {mx, s_s[0] + s_s[1] + s_s[2] + s_s[3], 0, 0};
        return;
    }
    bool bad = false;
    for (int64_t at = from; at < to; at += STEP) {
        float v[E];
        load16<TYPE>(a.x, row + at, row + to, v);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            bad |= !(v[i] < __builtin_inff());
            const int j = (int)(at + place16<TYPE>(i));
            if (v[i] > m || (v[i] == m && v[i] > -__builtin_inff() && j < first)) m = v[i], first = j;
        }
    }
    for (int o = 1; o < 64; o <<= 1) {
        const float om = __shfl_xor(m, o);
        const int of = __shfl_xor(first, o);
        if (om > m || (om == m && of < first)) m = om, first = of;
    }
    bad = __any(bad);
    if (lane == 0) s_m[wave] = m, s_i[wave] = first, s_s[wave] = bad ? __builtin_nanf("") : 0.0f;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < 4; ++i)
            if (s_m[i] > m || (s_m[i] == m && s_i[i] < first)) m = s_m[i], first = s_i[i];
        s = s_s[0] + s_s[1] + s_s[2] + s_s[3];
        if (first != 0x7FFFFFFF) s += 1.0f;
        w.stats[blockIdx.x] = {m, s, first, 0};
    }
}

// A row's parts as one (four at a time on their way).
__device__ __forceinline__ Stat joined(const VerifyArgs& a, const Space& w, int row, float T) {
    const Stat* p = w.stats + (int64_t)row * a.parts;
    const float k = fminf(LOG2E / T, 3e38f);
    Stat r{LOWEST, 0.0f, 0x7FFFFFFF, 0};
    for (int i0 = 0; i0 < a.parts; i0 += 4) {
        Stat o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = p[min(i0 + i, a.parts - 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i0 + i >= a.parts) continue;
            if (T > 0.0f) {
                const float m = fmaxf(r.m, o[i].m);
                r.s = (r.m == m ? r.s : r.s * exp2f((r.m - m) * k)) + (o[i].m == m ? o[i].s : o[i].s * exp2f((o[i].m - m) * k));
                r.m = m;
            } else {
                r.s += o[i].s;
                if (o[i].m > r.m || (o[i].m == r.m && o[i].first < r.first)) r.m = o[i].m, r.first = o[i].first;
            }
        }
    }
    return r;
}
__device__ __forceinline__ bool usable(const Stat& s) { return s.s > 0.0f && s.s < __builtin_inff(); }

// A row's sum of e^((x - m) / T) in 64 bits, by the wave.
template <int TYPE>
__device__ __forceinline__ double row_sum(const VerifyArgs& a, int row, float m, double inv) {
    constexpr int AHEAD = 8;
    const int lane = threadIdx.x & 63;
    const int64_t begin = (int64_t)row * a.ld;
    double sum = 0.0;
    for (int64_t at = lane; at < a.V; at += 64 * AHEAD) {
        float v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = at + 64 * i < a.V ? load1<TYPE>(a.x, begin + at + 64 * i) : -__builtin_inff();
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) sum += exp_of(((double)v[i] - (double)m) * inv);
    }
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
    return sum;
}

__device__ __forceinline__ double lane_of(double v, int i) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)b, i), hi = __builtin_amdgcn_readlane((uint32_t)(b >> 32), i);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The chunk's tokens that are refused, as bits of s_out.  (All threads of the work-group.)
__device__ __forceinline__ void mark(const Left& l, int64_t at, uint32_t (&s_out)[STEP / 32]) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid < STEP / 32) s_out[tid] = 0;
    __syncthreads();
    if (tid < l.refused) {
        const int64_t i = l.token[tid] - at;
        if (i >= 0 && i < STEP) atomicOr(&s_out[i >> 5], 1u << (i & 31));
    }
    __syncthreads();
}

__device__ __forceinline__ double sum_group(double v, double (&s)[4]) {
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return s[0] + s[1] + s[2] + s[3];
}

// Request b's walk, by one wave; `out`: it writes what is accepted.
template <int TYPE>
__device__ __forceinline__ void walk(const VerifyArgs& a, const Space& w, int b, bool out, Left& to) {
    const int lane = threadIdx.x & 63;
    const int t0 = min(max(a.cu[b], 0), a.N), nt = min(max(a.cu[b + 1], t0), a.N) - t0;
    const float T = a.temperature ? a.temperature[b] : 1.0f;
    const double inv = T > 0.0f ? 1.0 / (double)T : 1.0;
    int row = -1, q_row = -1, best = -1, refused = 0;
    float m = 0.0f;
    int accepted = 0, last = 0;
    if (nt > 0) {
        // What token i of the request has after token `up`: e of the row's sum s, which is off by off * s at most.
        struct Chance {
            double e = 0.0, s = 0.0, off = 0.0;
            float m = 0.0f;
        };
        const double off = T >= FAR_LOW && T <= FAR_HIGH ? w.unsure : __builtin_inf();
        const auto chance = [&](int i, int up) {
            Chance p;
            const int token = a.tokens[t0 + i];
            if (up < 0 || token < 0 || token >= a.V) return p;
            const Stat s = joined(a, w, t0 + up, T);
            if (!usable(s)) return p;
            if (T > 0.0f) {
                const float x = load1<TYPE>(a.x, (int64_t)(t0 + up) * a.ld + token);
                p.e = exp_of(((double)x - (double)s.m) * inv), p.s = s.s, p.off = off, p.m = s.m;
            } else {
                p.e = s.first == token ? 1.0 : 0.0, p.s = 1.0;
            }
            return p;
        };
        // Whether s leaves open if u (s - taken) < e.  (Never where u is 0 or NaN, nor of a sum in 64 bits, off 0.)
        const auto in_doubt = [](const Chance& p, double u, double taken) {
            return fabs(u * (p.s - taken) - p.e) < u * p.s * p.off;
        };
        // The row's sum in 64 bits that lane k's test is about.
        const auto exact = [&](const Chance& p, int up, int k) {
            return row_sum<TYPE>(a, t0 + up, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p.m), k)), inv);
        };
        if (!a.parents) {
            accepted = 1;
            for (int base = 1; base < nt; base += 64) {
                const int i = base + lane;
                Chance p;
                double u = 0.0;
                if (i < nt) {
                    p = chance(i, i - 1);
                    const int token = a.tokens[t0 + i];
                    const bool known = token >= 0 && token < a.V;
                    const double q = a.q && known ? (double)a.q[(int64_t)(t0 + i) * a.ldq + token] : 1.0;
                    u = (double)a.u[t0 + i] * q;
                }
                uint64_t no;
                for (;;) {  // until nothing is in doubt before the first that is refused
                    const bool doubt = in_doubt(p, u, 0.0);
                    no = __ballot(!doubt && !(u * p.s < p.e));
                    const uint64_t open = __ballot(doubt) & (no ? (no & -no) - 1 : ~0ull);
                    if (__builtin_expect(!open, 1)) break;
                    const int k = __builtin_ctzll(open);
                    const double s = exact(p, base + k - 1, k);
                    if (lane == k) p.s = s, p.off = 0.0;
                }
                accepted += no ? __builtin_ctzll(no) : 64;
                if (no) break;
            }
            last = accepted - 1;
            if (out)
                for (int i = lane; i < nt; i += 64) a.path[t0 + i] = i < accepted ? i : -1;
            if (accepted < nt) {
                if (a.q) {
                    q_row = t0 + accepted;
                } else {
                    refused = 1;
                    if (lane == 0) to.token[0] = a.tokens[t0 + accepted];
                }
            }
        } else {
            const int n = min(nt, LANES);
            int par = -9, token = -1;
            Chance p;
            double u = 0.0;
            if (lane < n) {
                par = a.parents[t0 + lane];
                if (par < 0 || par >= lane) par = -9;
                token = a.tokens[t0 + lane];
                u = (double)a.u[t0 + lane];
                p = chance(lane, par);
            }
            // The siblings before a token, as bits; one that was refused before already has nothing.
            uint64_t siblings = 0;
            bool refused_before = false;
            for (int j = 1; j < n; ++j) {
                const bool is = j < lane && __builtin_amdgcn_readlane(par, j) == par;
                siblings |= (uint64_t)is << j;
                refused_before |= is && __builtin_amdgcn_readlane(token, j) == token;
            }
            if (par < 0) siblings = 0;
            if (refused_before) p.e = 0.0;
            double taken = 0.0;
            for (uint64_t rest = siblings; __any(rest != 0); rest &= rest - 1) {
                const double v = __shfl(p.e, rest ? __builtin_ctzll(rest) : 0);
                if (rest) taken += v;
            }
            uint64_t acc;
            for (;;) {  // until nothing is in doubt on the walk's way
                const bool doubt = par >= 0 && in_doubt(p, u, taken);
                const uint64_t good = __ballot(par >= 0 && !doubt && u * (p.s - taken) < p.e);
                const uint64_t pass = __ballot((good >> lane & 1) && !(siblings & good));
                acc = 1;
                for (uint64_t more = 1; more;) {  // a level of the branch at a time
                    more = __ballot((pass >> lane & 1) && (acc >> (par & 63) & 1)) & ~acc;
                    acc |= more;
                }
                // Those behind an accepted token with no sibling before them that is sure to be taken.  The
                // earliest such token's row settles all of its children.
                uint64_t open = __ballot(doubt && (acc >> (par & 63) & 1) && !(siblings & good));
                if (__builtin_expect(!open, 1)) break;
                int up = LANES, k = 0;
                for (; open; open &= open - 1) {
                    const int at = __builtin_ctzll(open), v = __builtin_amdgcn_readlane(par, at);
                    if (v < up) up = v, k = at;
                }
                const double s = exact(p, up, k);
                if (par == up && p.s > 0.0) p.s = s, p.off = 0.0;
            }
            accepted = __builtin_popcountll(acc);
            last = 63 - __builtin_clzll(acc);
            if (out) {
                for (int i = lane; i < nt; i += 64)
                    if (i >= accepted) a.path[t0 + i] = -1;
                if (acc >> lane & 1) a.path[t0 + __builtin_popcountll(acc & ((1ull << lane) - 1))] = lane;
            }
            const uint64_t kids = __ballot(lane < n && par == last);
            refused = __builtin_popcountll(kids);
            if (kids >> lane & 1) to.token[__builtin_popcountll(kids & ((1ull << lane) - 1))] = token;
        }
        const Stat s = joined(a, w, t0 + last, T);
        if (usable(s)) {
            row = t0 + last;
            m = s.m;
            if (!(T > 0.0f)) best = s.first;
        }
    }
    if (lane == 0) {
        to.row = row, to.q = q_row, to.refused = refused, to.best = best, to.m = m;
        if (out) a.accepted[b] = accepted;
    }
}

// Walk, and the sums over the chunks of the last row.
template <int TYPE>
__global__ __launch_bounds__(256) void walk_kernel(VerifyArgs a, Space w) {
    __shared__ Left s_left;
    __shared__ uint32_t s_out[STEP / 32];
    __shared__ double s_sum[4];
    const int b = blockIdx.x / w.chunks, c = blockIdx.x % w.chunks, tid = threadIdx.x;
    if (tid < 64) walk<TYPE>(a, w, b, c == 0, s_left);
    if (b == a.B - 1 && c == 0)  // padding
        for (int64_t i = std::max(a.cu[a.B], 0) + tid; i < a.N; i += 256) a.path[i] = -1;
    if (b == 0 && c == 0)  // (cu begins with 0; what lay before it would be nobody's)
        for (int i = tid; i < std::min(a.cu[0], a.N); i += 256) a.path[i] = -1;
    __syncthreads();
    const Left& l = s_left;
    if (c == 0) {
        if (tid == 0) w.left[b].row = l.row, w.left[b].q = l.q, w.left[b].refused = l.refused,
                      w.left[b].best = l.best, w.left[b].m = l.m;
        if (tid < l.refused) w.left[b].token[tid] = l.token[tid];
    }
    if (l.row < 0 || l.best >= 0) return;
    const double inv = a.temperature ? 1.0 / (double)a.temperature[b] : 1.0, m = l.m;
    const int64_t end = std::min<int64_t>((int64_t)(c + 1) * w.chunk, a.V);
    double whole = 0.0, rest = 0.0;
    for (int64_t at = (int64_t)c * w.chunk; at < end; at += STEP) {
        mark(l, at, s_out);
        float v[E];
        load16<TYPE>(a.x, (int64_t)l.row * a.ld + at, (int64_t)l.row * a.ld + end, v);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const double e = exp_of(((double)v[i] - m) * inv);
            const int j = (int)place16<TYPE>(i);
            whole += e;
            rest += s_out[j >> 5] >> (j & 31) & 1 ? 0.0 : e;
        }
    }
    whole = sum_group(whole, s_sum);
    rest = sum_group(rest, s_sum);
    if (tid == 0) {
        w.whole[blockIdx.x] = whole;
        w.rest[blockIdx.x] = rest;
    }
}

// The sum of a request's n chunks, by the work-group.
__device__ __forceinline__ double total_of(const double* p, int n, double (&s)[4]) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) v += p[i];
    return sum_group(v, s);
}

// With draft probabilities: what is left of each chunk.
template <int TYPE>
__global__ __launch_bounds__(256) void left_kernel(VerifyArgs a, Space w) {
    __shared__ double s_sum[4];
    const int b = blockIdx.x / w.chunks, c = blockIdx.x % w.chunks;
    const int row = w.left[b].row, q = w.left[b].q;
    if (row < 0 || w.left[b].best >= 0 || q < 0) return;
    const double inv = a.temperature ? 1.0 / (double)a.temperature[b] : 1.0, m = w.left[b].m;
    const double all = total_of(w.whole + (int64_t)b * w.chunks, w.chunks, s_sum);
    const int64_t end = std::min<int64_t>((int64_t)(c + 1) * w.chunk, a.V);
    const double share = 1.0 / all;
    double rest = 0.0;
    for (int64_t at = (int64_t)c * w.chunk; at < end; at += STEP) {
        float v[E], d[E];
        load16<TYPE>(a.x, (int64_t)row * a.ld + at, (int64_t)row * a.ld + end, v);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int64_t j = at + place16<TYPE>(i);
            d[i] = j < end ? a.q[(int64_t)q * a.ldq + j] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) rest += fmax(exp_of(((double)v[i] - m) * inv) * share - (double)d[i], 0.0);
    }
    rest = sum_group(rest, s_sum);
    if (threadIdx.x == 0) w.rest[blockIdx.x] = rest;
}

// The lowest token whose cumulated sum is above u times the whole: the chunk by one wave, the
// token by 16, a step of the chunk at a time.
constexpr int PICK = 1024, PE = STEP / PICK;

template <int TYPE>
__global__ __launch_bounds__(PICK) void pick_kernel(VerifyArgs a, Space w) {
    __shared__ uint32_t s_out[STEP / 32];
    __shared__ double s_pre[PICK / 64], s_before, s_target, s_share;
    __shared__ int s_chunk, s_some, s_found, s_last;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    const Left& l = w.left[b];
    const int row = l.row, q = l.q, refused = l.refused;
    if (row < 0 || l.best >= 0) {
        if (tid == 0) a.next[b] = row < 0 ? -1 : l.best;
        return;
    }
    if (wave == 0) {
        const double* whole = w.whole + (int64_t)b * w.chunks;
        const double* rest = w.rest + (int64_t)b * w.chunks;
        const float u = a.u[max(a.cu[b], 0)];
        double all = 0.0, left = 0.0;
        for (int i = lane; i < w.chunks; i += 64) all += whole[i], left += rest[i];
        for (int o = 1; o < 64; o <<= 1) all += __shfl_xor(all, o), left += __shfl_xor(left, o);
        const bool some = left > 0.0;  // else p itself
        const double* sums = some ? rest : whole;
        const double target = (double)u * (some ? left : all);
        // 64 chunks at a time; where none passes the target (by rounding), the last one that has something
        double before = 0.0, at = 0.0;
        int chunk = -1;
        for (int base = 0; base < w.chunks; base += 64) {
            const double v = base + lane < w.chunks ? sums[base + lane] : 0.0;
            double upto = v;
            for (int o = 1; o < 64; o <<= 1) {
                const double x = __shfl_up(upto, o);
                if (lane >= o) upto += x;
            }
            const uint64_t past = __ballot(v > 0.0 && before + upto > target), any = __ballot(v > 0.0);
            const int i = past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : -1;
            if (i >= 0) chunk = base + i, at = before + lane_of(upto, uni(i)) - lane_of(v, uni(i));
            if (past) break;
            before += lane_of(upto, 63);
        }
        if (lane == 0) s_chunk = chunk, s_before = at, s_target = target, s_some = some, s_share = 1.0 / all;
    }
    if (tid == 0) s_found = 0x7FFFFFFF, s_last = -1;
    __syncthreads();
    if (s_chunk < 0) {  // (nothing anywhere: not for a row that is usable)
        if (tid == 0) a.next[b] = -1;
        return;
    }
    const bool some = s_some, drafted = some && q >= 0;
    const double inv = a.temperature ? 1.0 / (double)a.temperature[b] : 1.0, m = l.m, target = s_target, share = s_share;
    const int64_t begin = (int64_t)s_chunk * w.chunk, end = std::min<int64_t>(begin + w.chunk, a.V);
    double before = s_before;
    for (int64_t at = begin; at < end; at += STEP) {
        float x[PE], d[PE];
#pragma unroll
        for (int i = 0; i < PE; ++i) {
            const int64_t j = at + tid * PE + i;
            x[i] = j < end ? load1<TYPE>(a.x, (int64_t)row * a.ld + j) : -__builtin_inff();
            d[i] = drafted && j < end ? a.q[(int64_t)q * a.ldq + j] : 0.0f;
        }
        if (tid < STEP / 32) s_out[tid] = 0;
        __syncthreads();
        if (some && tid < refused) {
            const int64_t i = l.token[tid] - at;
            if (i >= 0 && i < STEP) atomicOr(&s_out[i >> 5], 1u << (i & 31));
        }
        __syncthreads();
        double e[PE], mine = 0.0;
#pragma unroll
        for (int i = 0; i < PE; ++i) {
            const int in = tid * PE + i;
            e[i] = exp_of(((double)x[i] - m) * inv);
            if (drafted) e[i] = fmax(e[i] * share - (double)d[i], 0.0);
            else if (s_out[in >> 5] >> (in & 31) & 1) e[i] = 0.0;
            mine += e[i];
        }
        double upto = mine;
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 63) s_pre[wave] = upto;
        __syncthreads();
        double base = before, step = 0.0;
        for (int i = 0; i < PICK / 64; ++i) {
            if (i < wave) base += s_pre[i];
            step += s_pre[i];
        }
        double sum = base + upto - mine;
        int found = 0x7FFFFFFF, last = -1;
#pragma unroll
        for (int i = 0; i < PE; ++i) {
            sum += e[i];
            if (e[i] > 0.0) {
                last = (int)(at + tid * PE + i);
                if (found == 0x7FFFFFFF && sum > target) found = last;
            }
        }
        // (of a wave the first and the last: a thousand at one place would wait for each other)
        const uint64_t passed = __ballot(found != 0x7FFFFFFF), any = __ballot(last >= 0);
        if (passed && lane == __builtin_ctzll(passed)) atomicMin(&s_found, found);
        if (any && lane == 63 - __builtin_clzll(any)) atomicMax(&s_last, last);
        __syncthreads();
        if (s_found != 0x7FFFFFFF) break;
        before += step;
    }
    // (the last one that counts, where rounding leaves the chunk's end below the target)
    if (tid == 0) a.next[b] = s_found != 0x7FFFFFFF ? s_found : s_last;
}

template <int TYPE>
hipError_t go(const VerifyArgs& a, const Space& w, hipStream_t st) {
    const dim3 t(256), rows((unsigned)(a.N * a.parts)), sums((unsigned)(a.B * w.chunks));
    if (a.N) {
        if (a.temperature) hipLaunchKernelGGL((stats_kernel<TYPE, true>), rows, t, 0, st, a, w);
        else hipLaunchKernelGGL((stats_kernel<TYPE, false>), rows, t, 0, st, a, w);
    }
    hipLaunchKernelGGL(walk_kernel<TYPE>, sums, t, 0, st, a, w);
    if (a.q) hipLaunchKernelGGL(left_kernel<TYPE>, sums, t, 0, st, a, w);
    hipLaunchKernelGGL(pick_kernel<TYPE>, dim3((unsigned)a.B), dim3(PICK), 0, st, a, w);
    return hipGetLastError();
}

constexpr int MAX_B = 8192;

}  // namespace

size_t verify_part_bytes(int) {
    return (size_t)MAX_STATS * sizeof(Stat) + MAX_B * sizeof(Left) + 2 * (size_t)(MAX_SUMS + MAX_B) * sizeof(double);
}

hipError_t launch_verify(const VerifyArgs& a0, int type, int cus, hipStream_t st) {
    VerifyArgs a = a0;
    // Rows are cut until there are two work-groups a CU, into parts of a step at least.
    const int most = (a.V + STEP - 1) / STEP;
    a.parts = a.N ? std::max(1, std::min(most, 2 * cus / a.N)) : 1;
    a.seg = (most + a.parts - 1) / a.parts * STEP;
    a.parts = (a.V + a.seg - 1) / a.seg;
    Space w;
    // In units of 2^-24.  A term's exponent y (to base 2, from the row's largest; the rescalings on its way
    // add up to no more) is a product of rounded numbers, 6 |y| off, the term 6 ln 2 |y|; over the terms
    // that is 4.2 log2 V on average at most, 126 (the average of -y is the entropy less that of the largest
    // term).  Exponentials are 2 off, a lane's step 13 (ten sums, a rescaling), the lanes' and
    // waves' sums 12, the join of a part 4.
    w.unsure = (140.0f + 13.0f * (float)(a.seg / STEP) + 4.0f * (float)a.parts) / 16777216.0f;
    const int per = std::max(1, (int)(((int64_t)a.B * most + MAX_SUMS - 1) / MAX_SUMS));
    w.chunk = per * STEP;
    w.chunks = (a.V + w.chunk - 1) / w.chunk;
    w.stats = (Stat*)a.ws;
    w.left = (Left*)(w.stats + MAX_STATS);
    w.whole = (double*)(w.left + MAX_B);
    w.rest = w.whole + MAX_SUMS + MAX_B;
    return type == 0 ? go<0>(a, w, st) : type == 1 ? go<1>(a, w, st) : go<2>(a, w, st);
}

}  // namespace fq
