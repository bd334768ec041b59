// fq_attn.hip -- attention of drafted tokens over a paged cache and over their
// ancestors in the draft.
//
// An item is one request, one kv head and up to 16 NR rows (a row: one token
// with one of the G query heads that share the kv head).  The keys of all items,
// in units of 32 WK, are shared out evenly over the work-groups, whatever the
// requests' lengths: work-group w takes units [w span, (w + 1) span) and walks
// the items that they belong to.  Every work-group finds its place from the
// lengths alone (no plan, no length on the host).  An item cut by such a border
// leaves partial results (maximum, sum, unnormalised output), which a second
// kernel joins, in the order of the keys, so that results repeat.
//
// A wave takes 32 keys at a time, its own in LDS, copied there straight from
// the cache's pages two tiles ahead; the keys' buffer is refilled while the
// values are used and the other way round.  Scores are S^T = K Q^T: keys along
// the MFMA result's rows (four to a lane and tile of 16), queries along its
// columns (one to a lane), so that a row's statistics are its lanes' own and
// the exponentials are, in place, the second product's B operand: O^T = V^T P^T
// with the contraction's keys in the order in which the lanes hold them.  V^T is read
// from LDS by transposing reads (each 16 lanes take a 4 key x 16 element block).
//
// Queries are fp32 and keep their bits: against fp16 keys a query is hi + lo
// in fp16 (22 bits, its row scaled by a power of two), against bf16 keys three
// bf16 parts (24 bits).  The probabilities take the same two or three parts,
// in fp16 scaled by 2^14 (so that parts down to 2^-38 of the row's largest
// count); statistics and sums are fp32.
//
// Rows and keys outside the lengths cost no branch in the common tile: only
// tiles that reach past the cached tokens mask their scores, and there values that
// are not finite are taken out of the product (a masked key's 0 times NaN
// would reach rows that do not see it) and put back into the rows that see them.
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
constexpr int KT = 32;  // keys of a wave's tile

// A uniform value in a scalar register, read through the scalar cache (memory
// that no kernel writes while this one runs).
__device__ __forceinline__ int sload(const int* p) {
    return *(const __attribute__((address_space(4))) int*)(uintptr_t)p;
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                       __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                      __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// x0, x1 as NL pairs of 16-bit parts that add up to them.
template <bool BF16>
struct Parts {
    static constexpr int N = BF16 ? 3 : 2;
};
template <bool BF16>
__device__ __forceinline__ void split2(float x0, float x1, uint32_t (&p)[Parts<BF16>::N]) {
    if constexpr (BF16) {
        #pragma unroll
        for (int i = 0; i < 3; ++i) {  // truncated: the rest is exact
            const uint32_t a = __float_as_uint(x0), b = __float_as_uint(x1);
            p[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            if (i < 2) {
                x0 -= __uint_as_float(a & 0xFFFF0000u);
                x1 -= __uint_as_float(b & 0xFFFF0000u);
            }
        }
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 hi = {(_Float16)x0, (_Float16)x1};
        const h2 lo = {(_Float16)(x0 - (float)hi[0]), (_Float16)(x1 - (float)hi[1])};
        p[0] = __builtin_bit_cast(uint32_t, hi);
        p[1] = __builtin_bit_cast(uint32_t, lo);
    }
}

// Where a work-group's units begin.
struct Place {
    int b;        // request
    int64_t off;  // units of b before it
};

template <int RT, int KU>
__device__ __forceinline__ void request(const AttnArgs& a, int b, int& t0, int& nt, int& len,
                                        int& keys, int& nu, int& rts) {
    t0 = min(max(sload(a.cu + b), 0), a.N);
    nt = min(max(sload(a.cu + b + 1), t0), a.N) - t0;
    len = max(sload(a.lengths + b), 0);
    // (no key lies beyond the table's columns)
    const int64_t most = (int64_t)a.max_blocks << a.c.bs_log2;
    keys = (int)min((int64_t)len + nt, min(most, (int64_t)INT32_MAX - 64));
    nu = (keys + KU - 1) / KU;
    rts = (int)(((int64_t)nt * a.G + RT - 1) / RT);
}

template <bool BF16, int D, int NR, int WK>
struct Shape {
    static constexpr int DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;  // LDS row, elements
    static constexpr int PITCH = 2 * DP;
    static constexpr int TILE = KT * PITCH;      // bytes
    static constexpr int WAVE = 4 * TILE;        // two of keys, two of values
    static constexpr int RT = 16 * NR;
    static constexpr int KU = KT * WK;
    static constexpr int ROWS = 1024 / PITCH;    // rows of one copy
    static constexpr int J = 16 / ROWS;          // copies of 16 rows
    static constexpr int NI = 2 * J;             // copies of a tile
    static constexpr size_t LDS = (size_t)WK * WAVE;
    static constexpr int PART = RT * (D + 2);    // floats of a partial result
};

constexpr int DESC = 8;  // ints of a work-group's record

template <bool BF16, int D, int NR, int WK>
__global__ __launch_bounds__(64 * WK, 1) void attn_kernel(AttnArgs a) {
    using S = Shape<BF16, D, NR, WK>;
    constexpr int NL = Parts<BF16>::N;
    constexpr int RT = S::RT, KU = S::KU, TILE = S::TILE, PITCH = S::PITCH, J = S::J;
    constexpr int STEPS = D / 32, DT = D / 16, SLOTS = S::DP / 8;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ int64_t s_part[64 * WK];
    __shared__ int s_b;
    __shared__ int64_t s_off;
    __shared__ float s_ml[2][WK][RT];
    const int tid = threadIdx.x, lane = tid & 63, wk = uni(tid >> 6);
    const int n16 = lane & 15, g = lane >> 4;
    const int wg = blockIdx.x;

    // --- the work-group's units ---
    int64_t total, span, u0;
    {
        constexpr int T = 64 * WK;
        const int per = (a.B + T - 1) / T;
        int64_t mine = 0;
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            if (b < a.B) {
                const int c0 = min(max(a.cu[b], 0), a.N);
                const int nt = min(max(a.cu[b + 1], c0), a.N) - c0;
                const int len = max(a.lengths[b], 0);
                const int64_t most = (int64_t)a.max_blocks << a.c.bs_log2;
                const int keys = (int)min((int64_t)len + nt, min(most, (int64_t)INT32_MAX - 64));
                mine += (int64_t)a.hkv * (((int64_t)nt * a.G + RT - 1) / RT) * ((keys + KU - 1) / KU);
            }
        }
        s_part[tid] = mine;
        __syncthreads();
        int64_t before = 0;
        total = 0;
        for (int i = 0; i < T; ++i) {
            const int64_t v = s_part[i];
            total += v;
            if (i < tid) before += v;
        }
        span = (total + gridDim.x - 1) / gridDim.x;
        u0 = wg * span;
        if (u0 >= before && u0 < before + mine) {
            int b = tid * per;
            int64_t off = u0 - before;
            for (;; ++b) {
                const int c0 = min(max(a.cu[b], 0), a.N);
                const int nt = min(max(a.cu[b + 1], c0), a.N) - c0;
                const int len = max(a.lengths[b], 0);
                const int64_t most = (int64_t)a.max_blocks << a.c.bs_log2;
                const int keys = (int)min((int64_t)len + nt, min(most, (int64_t)INT32_MAX - 64));
                const int64_t n =
                    (int64_t)a.hkv * (((int64_t)nt * a.G + RT - 1) / RT) * ((keys + KU - 1) / KU);
                if (off < n) break;
                off -= n;
            }
            s_b = b;
            s_off = off;
        }
        __syncthreads();
    }
    int* desc = a.desc + wg * DESC;
    // padding tokens
    {
        const int end = min(max(sload(a.cu + a.B), 0), a.N);
        const int64_t row = (int64_t)a.hq * D;
        for (int64_t i = end * row + (int64_t)wg * blockDim.x + tid; i < a.N * row;
             i += (int64_t)gridDim.x * blockDim.x)
            a.out[i] = 0.0f;
    }
    if (u0 >= total) {
        if (tid == 0) desc[0] = 0;
        return;
    }
    int64_t left = min(span, total - u0);
    int b = uni(s_b);
    int64_t off = s_off;
    off = ((int64_t)uni((int)(off >> 32)) << 32) | (uint32_t)uni((int)off);
    left = ((int64_t)uni((int)(left >> 32)) << 32) | (uint32_t)uni((int)left);
    int64_t u = u0;
    bool cut = false;  // an item begun here goes on in the next work-group

    // --- constants of a lane ---
    const uint32_t wbase = lds_addr(lds) + wk * S::WAVE;  // K0 K1 V0 V1
    uint32_t koff[J], voff[J];  // a copy's source in its rows: bytes from their first
    #pragma unroll
    for (int j = 0; j < J; ++j) {
        const int row = j * S::ROWS + lane / SLOTS, slot = lane % SLOTS;
        const int fk = D <= 64 ? (row >> 1) & 7 : row & 15;
        const int fv = D <= 64 ? (row >> 1) & 3 : row & 7;
        int ck = slot ^ fk, cv = slot ^ (fv << 1);
        if (8 * ck >= D) ck -= 4;  // (rows of 12 pieces among 16: the rest is not read)
        if (8 * cv >= D) cv -= 4;
        const uint32_t rb = (uint32_t)((lane / SLOTS) * a.c.st * 2);
        koff[j] = rb + ck * 16;
        voff[j] = rb + cv * 16;
    }
    const int fk = D <= 64 ? (n16 >> 1) & 7 : n16;
    const int vrow = 4 * g + (n16 >> 2);
    const int fv = D <= 64 ? (vrow >> 1) & 3 : vrow & 7;
    const uint32_t vlane = vrow * PITCH + (n16 & 3) * 8;

    for (; left > 0; ++b) {
        int t0, nt, len, keys, nu, rts;
        request<RT, KU>(a, b, t0, nt, len, keys, nu, rts);
        const int64_t units = (int64_t)a.hkv * rts * nu;
        while (off < units && left > 0) {
            const int item = (int)(off / nu), first = (int)(off % nu);
            const int h = item / rts, rt = item % rts;
            const int count = (int)min((int64_t)(nu - first), left);

            // --- queries ---
            u4 qf[NR][STEPS][NL];
            float rs[NR];
            uint64_t mask[NR];
            int tq[NR];
            #pragma unroll
            for (int c = 0; c < NR; ++c) {
                const int r = rt * RT + 16 * c + n16;
                const int t = r / a.G, hh = h * a.G + r % a.G;
                const bool on = t < nt;
                tq[c] = on ? t : 0;
                mask[c] = a.masks ? (on ? a.masks[t0 + t] : 0) : 0;
                const float* q = a.q + (int64_t)(t0 + tq[c]) * a.ldq + (int64_t)(on ? hh : 0) * D;
                f4 x[STEPS][2];
                float mx = 0.0f;
                #pragma unroll
                for (int s = 0; s < STEPS; ++s)
                    #pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        x[s][i] = on ? *(const f4u*)(q + 32 * s + 8 * g + 4 * i) : f4{0, 0, 0, 0};
                        #pragma unroll
                        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x[s][i][e]));
                    }
                float up = 1.0f, down = 1.0f;
                if (!BF16) {  // the row's largest to [2^14, 2^15)
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    if (mx > 0.0f && mx < __builtin_inff()) {
                        const int e = min(max(15 - __builtin_amdgcn_frexp_expf(mx), -126), 126);
                        up = ldexpf(1.0f, e);
                        down = ldexpf(1.0f, -e);
                    }
                }
                rs[c] = down * a.scale;
                #pragma unroll
                for (int s = 0; s < STEPS; ++s)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t p[NL];
                        split2<BF16>(x[s][i >> 1][2 * (i & 1)] * up,
                                     x[s][i >> 1][2 * (i & 1) + 1] * up, p);
                        #pragma unroll
                        for (int l = 0; l < NL; ++l) qf[c][s][l][i] = p[l];
                    }
            }

            // --- this wave's tiles: wk, wk + WK, .. of the segment's ---
            const int kbeg = first * KU + wk * KT;
            const int kend = min(keys, (first + count) * KU);
            const int n = kbeg < kend ? (kend - kbeg + KU - 1) / KU : 0;
            const int last16 = (keys - 1) & ~15;
            const uint8_t* kb = a.k + (int64_t)h * a.c.sh * 2;
            const uint8_t* vb = a.v + (int64_t)h * a.c.sh * 2;
            const int* table = a.table + b * a.table_stride;
            const auto copy = [&](int i, const uint8_t* base, const uint32_t (&lo)[J], uint32_t at) {
                #pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int key = min(kbeg + i * KU + 16 * hf, last16);
                    const int page = min(max(sload(table + (key >> a.c.bs_log2)), 0), a.c.num_blocks - 1);
                    const uint8_t* p = base + 2 * (page * a.c.sb + (key & ((1 << a.c.bs_log2) - 1)) * a.c.st);
                    #pragma unroll
                    for (int j = 0; j < J; ++j)
                        dma16s(lo[j], p + 2 * j * S::ROWS * a.c.st, at + (hf * J + j) * 1024);
                }
            };
            const auto copy_k = [&](int i) { copy(i, kb, koff, wbase + (i & 1) * TILE); };
            const auto copy_v = [&](int i) { copy(i, vb, voff, wbase + (2 + (i & 1)) * TILE); };
            f4 o[DT][NR];
            float mrow[NR], lrow[NR];
            bool careful = false;
        again:
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (n > 0) copy_k(0), copy_v(0);
            if (n > 1) copy_k(1), copy_v(1);
            #pragma unroll
            for (int c = 0; c < NR; ++c) {
                mrow[c] = LOWEST;
                lrow[c] = 0.0f;
                #pragma unroll
                for (int d = 0; d < DT; ++d) o[d][c] = f4{0, 0, 0, 0};
            }
            for (int i = 0; i < n; ++i) {
                const int key0 = kbeg + i * KU;
                // scores
                if (i + 1 < n) wait_vm<3 * S::NI>();
                else wait_vm<S::NI>();
                f4 sc[2][NR];
                #pragma unroll
                for (int sub = 0; sub < 2; ++sub) {
                    #pragma unroll
                    for (int c = 0; c < NR; ++c) sc[sub][c] = f4{0, 0, 0, 0};
                    #pragma unroll
                    for (int s = 0; s < STEPS; ++s) {
                        const uint32_t at = wbase + (i & 1) * TILE + (16 * sub + n16) * PITCH +
                                            (((4 * s + g) ^ fk) << 4);
                        const u4 kf = *(lds_u4*)(uintptr_t)at;
                        #pragma unroll
                        for (int c = 0; c < NR; ++c)
                            #pragma unroll
                            for (int l = NL - 1; l >= 0; --l)
                                sc[sub][c] = mfma<BF16>(kf, qf[c][s][l], sc[sub][c]);
                    }
                }
                wait_lds();
                if (i + 2 < n) copy_k(i + 2);

                // softmax
                const bool tail = careful || key0 + KT > len;
                u4 pf[NR][NL];
                float alpha[NR];
                bool moved = false;
                #pragma unroll
                for (int c = 0; c < NR; ++c) {
                    float mx = LOWEST;
                    #pragma unroll
                    for (int sub = 0; sub < 2; ++sub)
                        #pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float s = sc[sub][c][r] * rs[c];
                            if (tail) {
                                const int key = key0 + 16 * sub + 4 * g + r, j = key - len;
                                const bool see =
                                    key < keys && (j < 0 || (a.masks ? j < 64 && ((mask[c] >> (j & 63)) & 1)
                                                                     : j <= tq[c]));
                                s = see ? s : -__builtin_inff();
                            }
                            sc[sub][c][r] = s;
                            mx = fmaxf(mx, s);
                        }
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const float m = fmaxf(mrow[c], mx);
                    moved |= m > mrow[c];
                    alpha[c] = __builtin_amdgcn_exp2f(mrow[c] - m);
                    mrow[c] = m;
                    const float ref = BF16 ? m : m - 14.0f;
                    float p[2][4], sum = 0.0f;
                    #pragma unroll
                    for (int sub = 0; sub < 2; ++sub)
                        #pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            p[sub][r] = __builtin_amdgcn_exp2f(sc[sub][c][r] - ref);
                            sum += p[sub][r];
                        }
                    lrow[c] = lrow[c] * alpha[c] + sum;
                    #pragma unroll
                    for (int sub = 0; sub < 2; ++sub)
                        #pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint32_t q2[NL];
                            split2<BF16>(p[sub][2 * e], p[sub][2 * e + 1], q2);
                            #pragma unroll
                            for (int l = 0; l < NL; ++l) pf[c][l][2 * sub + e] = q2[l];
                        }
                }
                if (__any(moved))
                    #pragma unroll
                    for (int c = 0; c < NR; ++c)
                        #pragma unroll
                        for (int d = 0; d < DT; ++d) o[d][c] *= alpha[c];

                // values
                if (i + 2 < n) wait_vm<3 * S::NI>();
                else if (i + 1 < n) wait_vm<2 * S::NI>();
                else wait_vm<0>();
                #pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const uint32_t at = wbase + (2 + (i & 1)) * TILE + vlane + ((d ^ fv) << 5);
                    const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)at);
                    const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s4*)(uintptr_t)(at + 16 * PITCH));
                    const u2 w0 = __builtin_bit_cast(u2, v0), w1 = __builtin_bit_cast(u2, v1);
                    u4 vf = {w0[0], w0[1], w1[0], w1[1]};
                    if (tail) {
                        constexpr uint32_t EXP = BF16 ? 0x7F80u : 0x7C00u;
                        const u4 raw = vf;
                        bool odd = false;
                        #pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool lo = (raw[e] & EXP) == EXP, hi = (raw[e] >> 16 & EXP) == EXP;
                            odd |= lo | hi;
                            vf[e] = (lo ? 0u : raw[e] & 0xFFFFu) | (hi ? 0u : raw[e] & 0xFFFF0000u);
                        }
                        if (__any(odd)) {
                            // which rows see a NaN, an infinity: counts of ones
                            constexpr uint32_t ONE = BF16 ? 0x3F80u : 0x3C00u;
                            #pragma unroll
                            for (int kind = 0; kind < 3; ++kind) {
                                const float val = kind == 0 ? __builtin_nanf("")
                                                            : kind == 1 ? __builtin_inff() : -__builtin_inff();
                                u4 ind;
                                #pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    uint32_t w = 0;
                                    #pragma unroll
                                    for (int q = 0; q < 2; ++q) {
                                        const uint32_t x = raw[e] >> (16 * q) & 0xFFFFu;
                                        const bool is = kind == 0 ? (x & 0x7FFFu) > EXP
                                                                  : x == (kind == 1 ? EXP : EXP | 0x8000u);
                                        w |= is ? ONE << (16 * q) : 0u;
                                    }
                                    ind[e] = w;
                                }
                                #pragma unroll
                                for (int c = 0; c < NR; ++c) {
                                    u4 seen;
                                    #pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        uint32_t w = 0;
                                        #pragma unroll
                                        for (int q = 0; q < 2; ++q)
                                            w |= sc[e >> 1][c][2 * (e & 1) + q] != -__builtin_inff()
                                                     ? ONE << (16 * q) : 0u;
                                        seen[e] = w;
                                    }
                                    const f4 hits = mfma<BF16>(ind, seen, f4{0, 0, 0, 0});
                                    #pragma unroll
                                    for (int r = 0; r < 4; ++r)
                                        if (hits[r] > 0.0f) o[d][c][r] += val;
                                }
                            }
                        }
                    }
                    #pragma unroll
                    for (int c = 0; c < NR; ++c)
                        #pragma unroll
                        for (int l = NL - 1; l >= 0; --l) o[d][c] = mfma<BF16>(vf, pf[c][l], o[d][c]);
                }
                wait_lds();
                if (i + 2 < n) copy_v(i + 2);
            }

            // an infinite cached value times the two signs (or a zero) of a
            // probability's parts is NaN: once more, with the values looked at
            if (!careful) {
                bool nan = false;
#pragma unroll
                for (int c = 0; c < NR; ++c)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) nan |= o[d][c][r] != o[d][c][r];
                if (__any(nan)) {
                    careful = true;
                    goto again;
                }
            }

            // --- join the waves ---
            #pragma unroll
            for (int c = 0; c < NR; ++c) {
                lrow[c] += __shfl_xor(lrow[c], 16);
                lrow[c] += __shfl_xor(lrow[c], 32);
                if (lane < 16) {
                    s_ml[0][wk][16 * c + n16] = mrow[c];
                    s_ml[1][wk][16 * c + n16] = lrow[c];
                }
            }
            __syncthreads();
            float lsum[NR];
            #pragma unroll
            for (int c = 0; c < NR; ++c) {
                float m = LOWEST;
                #pragma unroll
                for (int w = 0; w < WK; ++w) m = fmaxf(m, s_ml[0][w][16 * c + n16]);
                lsum[c] = 0.0f;
                #pragma unroll
                for (int w = 0; w < WK; ++w)
                    lsum[c] += s_ml[1][w][16 * c + n16] *
                               __builtin_amdgcn_exp2f(s_ml[0][w][16 * c + n16] - m);
                const float f = __builtin_amdgcn_exp2f(mrow[c] - m);
                mrow[c] = m;
                #pragma unroll
                for (int d = 0; d < DT; ++d) o[d][c] *= f;
            }
            float* buf = (float*)lds;  // the tiles are not needed any more
            for (int half = WK / 2; half; half >>= 1) {
                if (wk >= half && wk < 2 * half)
                    #pragma unroll
                    for (int c = 0; c < NR; ++c)
                        #pragma unroll
                        for (int d = 0; d < DT; ++d)
                            #pragma unroll
                            for (int r = 0; r < 4; ++r)
                                buf[(((wk - half) * NR + c) * DT + d) * 256 + r * 64 + lane] = o[d][c][r];
                __syncthreads();
                if (wk < half)
                    #pragma unroll
                    for (int c = 0; c < NR; ++c)
                        #pragma unroll
                        for (int d = 0; d < DT; ++d)
                            #pragma unroll
                            for (int r = 0; r < 4; ++r)
                                o[d][c][r] += buf[((wk * NR + c) * DT + d) * 256 + r * 64 + lane];
                __syncthreads();
            }
            const bool whole = count == nu;
            if (wk == 0) {
                float* part = a.part + (int64_t)(2 * wg + (first == 0)) * S::PART;
                #pragma unroll
                for (int c = 0; c < NR; ++c) {
                    const int rl = 16 * c + n16, r = rt * RT + rl;
                    const int t = r / a.G, hh = h * a.G + r % a.G;
                    const float inv = lsum[c] != 0.0f ? 1.0f / lsum[c] : 0.0f;
                    if (whole) {
                        if (t < nt)
                            #pragma unroll
                            for (int d = 0; d < DT; ++d) {
                                f4 v = o[d][c] * inv;
                                if (lsum[c] == 0.0f) v = f4{0, 0, 0, 0};
                                *(f4*)(a.out + ((int64_t)(t0 + t) * a.hq + hh) * D + 16 * d + 4 * g) = v;
                            }
                    } else {
                        #pragma unroll
                        for (int d = 0; d < DT; ++d)
                            *(f4*)(part + rl * D + 16 * d + 4 * g) = o[d][c];
                        if (g == 0) {
                            part[RT * D + rl] = mrow[c];
                            part[RT * D + RT + rl] = lsum[c];
                        }
                    }
                }
            }
            if (first == 0 && !whole) {
                cut = true;
                if (tid == 0) {
                    const int64_t end = u + nu - 1;  // the item's last unit
                    desc[0] = (int)(end / span) - wg + 1;
                    desc[1] = t0, desc[2] = nt, desc[3] = h, desc[4] = rt;
                }
            }
            u += count;
            off += count;
            left -= count;
        }
        off -= units;
    }
    if (!cut && tid == 0) desc[0] = 0;
}

// The rows of an item whose parts lie in work-groups w .. w + parts - 1: one wave
// to a row.
template <int D, int RT>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a) {
    constexpr int PART = RT * (D + 2);
    const int w = blockIdx.x, lane = threadIdx.x & 63;
    const int* desc = a.desc + w * DESC;
    const int parts = sload(desc);
    if (parts == 0) return;
    const int rl = blockIdx.y * 4 + uni(threadIdx.x >> 6);
    const int t0 = sload(desc + 1), nt = sload(desc + 2), h = sload(desc + 3), rt = sload(desc + 4);
    const int r = rt * RT + rl, t = r / a.G;
    if (t >= nt) return;
    const auto slot = [&](int p) { return a.part + (int64_t)(2 * (w + p) + (p == 0)) * PART; };
    float m = LOWEST;
    for (int p = lane; p < parts; p += 64) m = fmaxf(m, slot(p)[RT * D + rl]);
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    constexpr int V = (D + 63) / 64;
    float acc[V] = {}, l = 0.0f;
    for (int p0 = 0; p0 < parts; p0 += 64) {
        float f = 0.0f, lp = 0.0f;
        if (p0 + lane < parts) {
            const float* s = slot(p0 + lane) + RT * D + rl;
            f = __builtin_amdgcn_exp2f(s[0] - m);
            lp = s[RT];
        }
        const int np = min(64, parts - p0);
        for (int p = 0; p < np; ++p) {
            const float fp = __shfl(f, p);
            l += fp * __shfl(lp, p);
            const float* s = slot(p0 + p) + rl * D;
            #pragma unroll
            for (int v = 0; v < V; ++v)
                if (64 * v + lane < D) acc[v] += fp * s[64 * v + lane];
        }
    }
    float* out = a.out + ((int64_t)(t0 + t) * a.hq + h * a.G + r % a.G) * D;
    #pragma unroll
    for (int v = 0; v < V; ++v)
        if (64 * v + lane < D) out[64 * v + lane] = l != 0.0f ? acc[v] / l : 0.0f;
}

template <bool BF16, int D, int NR, int WK>
hipError_t go(AttnArgs a, int cus, uint8_t* ws, hipStream_t st) {
    using S = Shape<BF16, D, NR, WK>;
    static_assert(S::LDS <= 128 * 1024, "LDS");
    static_assert((size_t)WK / 2 * NR * 16 * D * 4 <= S::LDS, "join");
    a.grid = cus;
    a.desc = (int*)ws;
    a.part = (float*)(ws + (size_t)cus * DESC * 4);
    const auto fn = attn_kernel<BF16, D, NR, WK>;
    hipLaunchKernelGGL(fn, dim3(a.grid), dim3(64 * WK), S::LDS, st, a);
    hipLaunchKernelGGL((attn_join<D, S::RT>), dim3(a.grid, S::RT / 4), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <bool BF16, int D, int WK, int MAXNR>
hipError_t rows(const AttnArgs& a, int max_new, int cus, uint8_t* ws, hipStream_t st) {
    const int64_t r = (int64_t)max_new * a.G;
    if (r <= 16) return go<BF16, D, 1, WK>(a, cus, ws, st);
    if (r <= 32 || MAXNR == 2) return go<BF16, D, 2, WK>(a, cus, ws, st);
    return go<BF16, D, MAXNR, WK>(a, cus, ws, st);
}

template <bool BF16>
hipError_t heads(const AttnArgs& a, int D, int max_new, int cus, uint8_t* ws, hipStream_t st) {
    switch (D) {
        case 64: return rows<BF16, 64, 4, 4>(a, max_new, cus, ws, st);
        case 96: return rows<BF16, 96, 4, 4>(a, max_new, cus, ws, st);
        case 128: return rows<BF16, 128, 4, 4>(a, max_new, cus, ws, st);
        default: return rows<BF16, 256, 2, 2>(a, max_new, cus, ws, st);
    }
}

}  // namespace

size_t attn_part_bytes(int cus) {
    return (size_t)cus * (DESC * 4 + 2 * sizeof(float) * 64 * (128 + 2));
}

hipError_t launch_attn(const AttnArgs& a, bool bf16, int D, int max_new, int cus, uint8_t* ws,
                       hipStream_t st) {
    return bf16 ? heads<true>(a, D, max_new, cus, ws, st) : heads<false>(a, D, max_new, cus, ws, st);
}

}  // namespace fq
