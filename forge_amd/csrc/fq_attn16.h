// fq_attn16.h -- the attention kernel over caches of 16 bits, which fq_attn.hip describes.
#pragma once

#include "fq_attn.h"

namespace fq {
namespace {

constexpr int KT = 32;  // keys of a wave's tile
// By how much (log2) a row's largest score may be above its sums' reference, and what
// fp16 probabilities are raised by: together they stay below fp16's largest.
constexpr float LAG = 4.0f, UP = 11.0f;

template <bool BF16>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                       __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                      __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// x0, x1 as pairs of 16-bit parts that add up to them.  minus1: -1 where the
// compiler does not see it, so that an fp16 rest is one fused multiply-add from the
// packed part (with its rounding to fp16) and not a conversion and a subtraction.
template <bool BF16>
struct Parts {
    static constexpr int N = BF16 ? 3 : 2;
};
template <bool BF16>
__device__ __forceinline__ void split2(float x0, float x1, float minus1,
                                       uint32_t (&p)[Parts<BF16>::N]) {
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
        typedef float f2 __attribute__((ext_vector_type(2)));
        const h2 hi = __builtin_convertvector((f2{x0, x1}), h2);
        p[0] = __builtin_bit_cast(uint32_t, hi);
        asm("" : "+v"(p[0]));  // (one packed conversion, not one more for each rest)
        const h2 back = __builtin_bit_cast(h2, p[0]);
        const h2 lo = {(_Float16)fmaf((float)back[0], minus1, x0),
                       (_Float16)fmaf((float)back[1], minus1, x1)};
        p[1] = __builtin_bit_cast(uint32_t, lo);
    }
}

// Makes split2's parts of a number all of one sign and none zero (where the first is not), so
// that an infinite key's products with them add up to an infinity and not to NaN.  fp16: the
// first part, a rounded one, gives a last place to the second.  bf16: the others, zero
// where the number ends before them, become 2^-126 at least.  Of a first part that is
// infinite (or NaN), all are it.
template <bool BF16>
__device__ __forceinline__ void one_sign(uint32_t (&p)[Parts<BF16>::N]) {
    typedef uint16_t w2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const w2 first = __builtin_bit_cast(w2, p[0]), sign = first & (uint16_t)0x8000, mag = first & (uint16_t)0x7FFF;
    const auto infinite = [&](w2 of) {
        w2 r;
#pragma unroll
        for (int i = 0; i < 2; ++i) r[i] = mag[i] >= (BF16 ? 0x7F80 : 0x7C00) ? first[i] : of[i];
        return __builtin_bit_cast(uint32_t, r);
    };
    if constexpr (BF16) {
#pragma unroll
        for (int l = 1; l < Parts<BF16>::N; ++l) {
            const w2 m = __builtin_bit_cast(w2, p[l]) & (uint16_t)0x7FFF;
            w2 r;
#pragma unroll
            for (int i = 0; i < 2; ++i) r[i] = mag[i] ? max(m[i], (uint16_t)0x0080) | sign[i] : 0;
            p[l] = infinite(r);
        }
    } else {
        w2 less;
#pragma unroll
        for (int i = 0; i < 2; ++i) less[i] = (mag[i] - min(mag[i], (uint16_t)1)) | sign[i];
        const h2 rest = __builtin_bit_cast(h2, p[1]) + (__builtin_bit_cast(h2, first) - __builtin_bit_cast(h2, less));
        p[0] = infinite(less);
        p[1] = infinite(__builtin_bit_cast(w2, rest));
    }
}

// Where a token lies in a cache whose page (block) that is, in bytes (where it is none, in
// the last: copied and masked).  (Strides are below 2^31 elements: 32-bit factors.)
__device__ __forceinline__ uint64_t place_of(const AttnArgs& a, int page, int key) {
    const uint32_t pg = min((uint32_t)page, (uint32_t)a.c.num_blocks - 1);
    const uint32_t in = (uint32_t)key & ((1u << a.c.bs_log2) - 1);
    return 2 * ((uint64_t)pg * (uint32_t)a.c.sb + (uint64_t)in * (uint32_t)a.c.st);
}

// WR x WK waves: each group of WR shares tiles of 32 keys, each of its waves
// with 16 NR rows of its own; the groups take every WK-th tile.  NS tiles of a
// group are in LDS.  PC work-groups to a CU.
template <bool BF16_, bool WIN_, int D_, int NR_, int WR_, int WK_, int NS_, int PC_>
struct Shape {
    static constexpr bool BF16 = BF16_, WIN = WIN_;
    static constexpr int D = D_, NR = NR_, WR = WR_, WK = WK_, NS = NS_, PC = PC_;
    static constexpr int WAVES = WR * WK;
    static constexpr int DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;  // LDS row, elements
    static constexpr int PITCH = 2 * DP;
    static constexpr int RT = 16 * NR * WR;
    static constexpr int KU = KT * WK;
    static constexpr int ROWS = 1024 / PITCH;    // rows of one copy
    static constexpr int J = 16 / ROWS;          // copies of 16 rows
    static constexpr int NI = 2 * J;             // copies of a tile
    static constexpr int CW = 2 * NI / WR;       // copies of a wave for a tile's keys and values
    // Bytes from copy to copy in LDS, and which bits of a row's number change
    // places of its 16-byte pieces (keys: of four, values: of four pairs): chosen so
    // that the 16 lanes of a read find 16 (values: 8) places of the 256
    // bytes that the banks span, with every place an immediate offset from few registers.
    static constexpr int KSTEP = 1024 + (D == 256 ? 32 : 64);
    static constexpr int VSTEP = 1024 + (D == 64 ? 0 : 64);
    static __device__ __forceinline__ int turn(int row) {
        return D == 64 ? (row >> 1) & 3 : D == 256 ? row & 1 : row & 3;
    }
    static constexpr int KTILE = NI * KSTEP, VTILE = NI * VSTEP, STAGE = KTILE + VTILE;
    static constexpr int GROUP = NS * STAGE;
    static constexpr size_t LDS = (size_t)WK * GROUP;
    static constexpr int PART = RT * (D + 2);    // floats of a partial result
    // What an item costs beside its units, in units: finding its blocks, its
    // queries, the first tiles' way, joining the groups and storing.
    static constexpr int OV = 256 / KU;
    static_assert(NI % WR == 0 && (WR <= J || WR == 2 * J) && (WR == 1 ? NS == 2 : NS >= 3), "copies");
    // the waves' outputs are exchanged where the tiles were
    static_assert((size_t)WAVES * NR * 16 * D * 4 <= LDS, "join");
    static_assert(D / 16 % WK == 0, "join");
    static_assert(PC * (LDS + 8 * WK * (RT + 1) + 64) <= 160 * 1024, "LDS");
    static_assert(PC <= MAX_GRID && (size_t)PC * PART <= MAX_PART, "workspace");
};

template <class S>
__global__ __launch_bounds__(64 * S::WAVES, (S::WAVES * S::PC + 3) / 4) void attn_kernel(AttnArgs a) {
    constexpr bool BF16 = S::BF16, WIN = S::WIN;
    constexpr int D = S::D, NR = S::NR, WR = S::WR, WK = S::WK, NS = S::NS;
    constexpr int NL = Parts<BF16>::N;
    constexpr int RT = S::RT, KU = S::KU, PITCH = S::PITCH, J = S::J, NI = S::NI, ROWS = S::ROWS;
    constexpr int OV = S::OV;
    constexpr int STEPS = D / 32, DT = D / 16, SLOTS = S::DP / 8;
    constexpr uint32_t EXP = BF16 ? 0x7F80u : 0x7C00u;  // the exponent of what is not finite
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float s_ml[2][WK][RT];
    __shared__ int s_odd[WK];
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    const int wr = wave % WR, wk = wave / WR;
    const int n16 = lane & 15, g = lane >> 4;
    const int wg = blockIdx.x;

    // --- the work-group's units (every wave finds them for itself) ---
    int64_t total, span, off;
    int b;
    {
        const int per = (a.B + 63) / 64, first = lane * per;
        int64_t mine = 0;
        for (int i = first; i < min(first + per, a.B); ++i)
            mine += request<RT, KU, OV, WIN>(a, a.cu[i], a.cu[i + 1], a.lengths[i]).units;
        int64_t upto = mine;
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t v = __shfl_up(upto, o);
            if (lane >= o) upto += v;
        }
        total = uni64(__shfl(upto, 63));
        span = (total + gridDim.x - 1) / gridDim.x;
        const int64_t u0 = wg * span;
        const uint64_t past = __ballot(upto > u0);
        const int at = past ? __builtin_ctzll(past) : 0;
        b = at * per;
        off = u0 - uni64(__shfl(upto - mine, at));
    }
    int* desc = a.desc + MAX_ITEMS + wg * DESC;
    // padding tokens
    {
        const int end = min(max(sload(a.cu + a.B), 0), a.N);
        const int64_t row = (int64_t)a.hq * D;
        for (int64_t i = end * row + (int64_t)wg * blockDim.x + tid; i < a.N * row;
             i += (int64_t)gridDim.x * blockDim.x)
            a.out[i] = 0.0f;
    }
    int64_t u = wg * span;
    if (u >= total) {
        if (tid == 0) a.desc[wg] = 0;
        return;
    }
    int64_t left = min(span, total - u);
    bool cut = false;  // an item begun here goes on in the next work-group

    if (tid < WK) s_odd[tid] = 0;
    lds_barrier();

    // --- constants of a lane ---
    float minus1 = -1.0f;
    asm("" : "+s"(minus1));
    const uint32_t gbase = lds_addr(lds) + wk * S::GROUP;
    // a copy's source: bytes from its first row
    uint32_t ksrc, vsrc;
    {
        const int row = lane / SLOTS, slot = lane % SLOTS;
        int ck = slot ^ S::turn(row), cv = slot ^ (S::turn(row) << 1);
        if (8 * ck >= D) ck -= 4;  // (rows of 12 pieces among 16: the rest is not read)
        if (8 * cv >= D) cv -= 4;
        ksrc = (uint32_t)(row * a.c.st * 2) + ck * 16;
        vsrc = (uint32_t)(row * a.c.st * 2) + cv * 16;
    }
    const uint32_t klane = gbase + n16 / ROWS * S::KSTEP + n16 % ROWS * PITCH +
                           ((g ^ S::turn(n16)) << 4);
    uint32_t vlane[4];
    {
        const int row = 4 * g + (n16 >> 2);
#pragma unroll
        for (int d = 0; d < 4; ++d)
            vlane[d] = gbase + S::KTILE + row / ROWS * S::VSTEP + row % ROWS * PITCH +
                       ((d ^ S::turn(row)) << 5) + (n16 & 3) * 8;
    }

    for (; left > 0; ++b) {
        const Request rq = request<RT, KU, OV, WIN>(a, sload(a.cu + b), sload(a.cu + b + 1), sload(a.lengths + b));
        const int len = rq.len, keys = rq.keys, nu = rq.nu, t0 = rq.t0, nt = rq.nt;
        if (off >= rq.units) {
            off -= rq.units;
            continue;
        }
        int item = 0, pos = 0;
        if (off) {
            item = (int)(off / rq.cost);
            pos = (int)(off % rq.cost);
        }
        while (off < rq.units && left > 0) {
            const int take = (int)min((int64_t)(rq.cost - pos), left);
            const int first = a.whole ? 0 : max(pos - OV, 0);
            const int count = a.whole ? nu : max(pos + take - OV, 0) - first;
            const int64_t start = u - pos;  // the item's
            u += take;
            off += take;
            left -= take;
            pos = 0;
            if (count == 0) break;  // (the item's work begins in the next work-group)
            const int h = item / rq.rts, rt = item % rq.rts;
            ++item;
            // --- this group's tiles: wk, wk + WK, .. of the segment's.  Waves that
            // share tiles keep step: as many tiles for each group (those past
            // the last key are masked) ---
            // (with a window, units behind the sinks are left out)
            const auto key_at = [&](int i) {
                const int unit = first + i;
                return (WIN && unit >= rq.su ? unit + rq.skip : unit) * KU + wk * KT;
            };
            const int n = WR > 1 || count == 0 || key_at(count - 1) < keys ? count : count - 1;
            const int last16 = (keys - 1) & ~15;
            const uint8_t* kb = a.k + (int64_t)h * a.c.sh * 2;
            const uint8_t* vb = a.v + (int64_t)h * a.c.sh * 2;
            const int* table = a.table + b * a.table_stride;
            // The first key that all of the item's rows see, and all from there on to the context's end.
            const int clear = WIN && a.window ? (int)min((int64_t)rq.pos + (a.masks ? 63 : min(nt - 1, (rt * RT + RT - 1) / a.G)) + 1 - a.window,
                                                         (int64_t)INT32_MAX) : 0;
            // A tile's pages, read ahead; the places of its 16s of keys in a cache;
            // its copies.  (Past the last key: its page again.)
            const auto key_of = [&](int i, int hf) { return min(key_at(i) + 16 * hf, last16); };
            int page[2];
            const auto read_pages = [&](int i) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) page[hf] = sload(table + (key_of(i, hf) >> a.c.bs_log2));
            };
            uint64_t at_k[2], at_v[2];  // of the tiles whose keys, values are copied next
            uint32_t highest = 0;       // of the pages placed so far (unsigned: -1 is above all blocks)
            const auto place = [&](int i) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    at_v[hf] = at_k[hf];
                    at_k[hf] = place_of(a, page[hf], key_of(i, hf));
                    highest = max(highest, (uint32_t)page[hf]);
                }
            };
            // The keys of a tile that lie in a block.
            const auto there = [&](int i) {
                uint32_t m = ~0u;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    if (no_block(a, sload(table + (key_of(i, hf) >> a.c.bs_log2)))) m &= ~(0xFFFFu << (16 * hf));
                return m;
            };
            const int64_t step = 2 * ROWS * a.c.st;  // bytes from copy to copy
            const auto copy_k = [&](int stage) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const uint8_t* from = kb + at_k[hf];
#pragma unroll
                    for (int j = 0; j < J; ++j, from += step)
                        dma16s(ksrc, from, gbase + stage * S::STAGE + (hf * J + j) * S::KSTEP);
                }
            };
            const auto copy_v = [&](int stage) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const uint8_t* from = vb + at_v[hf];
#pragma unroll
                    for (int j = 0; j < J; ++j, from += step)
                        dma16s(vsrc, from, gbase + stage * S::STAGE + S::KTILE + (hf * J + j) * S::VSTEP);
                }
            };
            // This wave's share of a tile's keys and of the one before's values: copies wr,
            // wr + WR, .. of the NI of keys and the NI of values, copy c being number c % J of the
            // 16 keys c / J.  Whatever does not depend on wr is known here.
            const uint8_t *kw = kb + (wr % J) * step, *vw = vb + (wr % J) * step;
            const auto copy_share = [&](bool ks, int kstage, bool vs, int vstage) {
                const uint32_t kto = gbase + kstage * S::STAGE + wr * S::KSTEP;
                const uint32_t vto = gbase + vstage * S::STAGE + S::KTILE + wr * S::VSTEP;
#pragma unroll
                for (int x = 0; x < S::CW; ++x) {
                    constexpr bool LOW = WR <= J;  // (all of a copy's place but wr is known)
                    const int c0 = WR * x % NI;
                    const bool upper = LOW ? c0 >= J : wr >= J;
                    const uint64_t in = LOW ? (uint64_t)((c0 % J) * step) : 0;
                    if (WR * x < NI) {
                        if (ks) dma16s(ksrc, kw + ((upper ? at_k[1] : at_k[0]) + in), kto + c0 * S::KSTEP);
                    } else if (vs) {
                        dma16s(vsrc, vw + ((upper ? at_v[1] : at_v[0]) + in), vto + c0 * S::VSTEP);
                    }
                }
            };

            f4 o[DT][NR];
            float mrow[NR], lrow[NR];
            u4 qf[NR][STEPS][NL];
            float rs[NR];
            uint64_t mask[NR];
            int from[NR];  // (with a window)
            bool careful = false;
        again:
            at_k[0] = at_k[1] = 0;
            if constexpr (WR == 1) {
                // K0 V0 K1 V1; then K2 once K0 is used, V2 once V0 is, ..
                read_pages(0);
                place(0);
                read_pages(1);
                if (n > 0) copy_k(0);
                place(1);
                read_pages(2);
                if (n > 0) copy_v(0);
                if (n > 1) copy_k(1);
                at_v[0] = at_k[0], at_v[1] = at_k[1];
                if (n > 1) copy_v(1);
            } else {
                // K0, K1 V0, K2 V1, ..: each step's batch has the keys of one tile and
                // the values of the one before
                if (careful) lds_barrier();  // (the others may still read)
                read_pages(0);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    place(i);
                    read_pages(i + 1);
                    copy_share(i < n, i, i > 0 && i <= n, i - 1);
                }
            }
            // --- queries (on their way while the first tiles are) ---
#pragma unroll
            for (int c = 0; c < NR; ++c) {
                const int r = rt * RT + wr * 16 * NR + 16 * c + n16;
                const int t = r / a.G, hh = h * a.G + r % a.G;
                const bool on = t < nt;
                // (a chain: how many of the new tokens the row sees)
                mask[c] = !on ? 0 : a.masks ? a.masks[t0 + t] : (uint64_t)t + 1;
                from[c] = 0x7FFFFFFF;  // (a row of nobody's sees none of what the others do not)
                if (WIN && on) {
                    const Reach r = reach(a, rq.pos, t, mask[c]);
                    mask[c] = r.mask, from[c] = r.from;
                }
                const float* q = a.q + (int64_t)(t0 + (on ? t : 0)) * a.ldq + (int64_t)(on ? hh : 0) * D;
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
                    mx = max4(mx);
                    if (mx > 0.0f && mx < __builtin_inff()) {
                        const int e = min(max(15 - __builtin_amdgcn_frexp_expf(mx), -126), 126);
                        up = ldexpf(1.0f, e);
                        down = ldexpf(1.0f, -e);
                    }
                }
                // (the scale's sign goes with the query: the largest score is
                // that of the largest product)
                up = copysignf(up, a.scale);
                rs[c] = down * fabsf(a.scale);
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t p[NL];
                        split2<BF16>(x[s][i >> 1][2 * (i & 1)] * up,
                                     x[s][i >> 1][2 * (i & 1) + 1] * up, minus1, p);
#pragma unroll
                        for (int l = 0; l < NL; ++l) qf[c][s][l][i] = p[l];
                    }
                if (!careful) continue;
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t p[NL];
#pragma unroll
                        for (int l = 0; l < NL; ++l) p[l] = qf[c][s][l][i];
                        one_sign<BF16>(p);
#pragma unroll
                        for (int l = 0; l < NL; ++l) qf[c][s][l][i] = p[l];
                        __builtin_amdgcn_sched_barrier(0);  // (one after the other: few registers)
                    }
            }

#pragma unroll
            for (int c = 0; c < NR; ++c) {
                mrow[c] = LOWEST;
                lrow[c] = 0.0f;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d][c] = f4{0, 0, 0, 0};
            }
            // Products of the keys at `at`, STEPS times 2 NL NR matrix instructions with
            // beside(s) after each.  (The parts of one sum apart, so that no product
            // waits for the one before.)  The waves of a SIMD mostly stand at the same
            // place: in short turns one has the matrix unit while the other has
            // the vector unit.
            const auto products = [&](uint32_t at, f4 (&sc)[2][NR], const auto& beside) {
                const auto keys_of = [&](int s, u4 (&kf)[2]) {
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub)
                        kf[sub] = *(lds_u4*)(uintptr_t)(klane + at + J * sub * S::KSTEP + 64 * s);
                };
                u4 kf[2][2];
                keys_of(0, kf[0]);
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                    for (int c = 0; c < NR; ++c) sc[sub][c] = f4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    if (s + 1 < STEPS) keys_of(s + 1, kf[(s + 1) & 1]);
#pragma unroll
                    for (int l = NL - 1; l >= 0; --l)
#pragma unroll
                        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                            for (int c = 0; c < NR; ++c)
                                sc[sub][c] = mfma<BF16>(kf[s & 1][sub], qf[c][s][l], sc[sub][c]);
                    __builtin_amdgcn_sched_barrier(0);
                    beside(s);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            f4 sc[2][NR];
            if constexpr (WR == 1) {
                if (n > 1) wait_vm<3 * NI>();
                else wait_vm<NI>();
            } else {
                if (n >= NS) wait_vm<(NS - 1) * S::CW>();
                else wait_vm<0>();
                lds_barrier();
            }
            products(0, sc, [](int) {});
            int stage = 0;
            for (int i = 0; i < n; ++i) {
                const int key0 = key_at(i);
                const int stage1 = stage + 1 < NS ? stage + 1 : 0;
                // this tile's values and the next one's keys have landed: this wave's
                // copies of them, then everyone's; and all are done with this one's
                // keys and the last one's values, whose places are filled anew
                if constexpr (WR == 1) {
                    wait_lds();
                    if (i + 2 < n) {
                        place(i + 2);
                        read_pages(i + 3);
                        copy_k(stage);
                        wait_vm<2 * NI>();
                    } else if (i + 1 < n) {
                        wait_vm<NI>();
                    } else {
                        wait_vm<0>();
                    }
                } else {
                    if (i + NS - 1 < n) wait_vm<(NS - 2) * S::CW>();
                    else if (i + 1 < n) wait_vm<S::CW / 2>();
                    else wait_vm<0>();
                    lds_barrier();
                    if (i + NS - 1 < n) {
                        place(i + NS);
                        read_pages(i + NS + 1);
                        copy_share(i + NS < n, stage, true, stage ? stage - 1 : NS - 1);
                    }
                }
                const bool holes = no_block(a, (int)highest);
                const bool tail = careful || holes || key0 + KT > len || (WIN && key0 < clear && key0 + KT > a.sinks);
                float mul[NR];
#pragma unroll
                for (int c = 0; c < NR; ++c) mul[c] = rs[c];
                if (tail) {
                    const int old = len - key0, all = keys - key0;
                    const uint32_t in = holes ? there(i) : ~0u;
#pragma unroll
                    for (int c = 0; c < NR; ++c) {
                        // (with a window a tile seen in part has the bits of one seen whole, whichever it is:
                        // but for factors of 0 and NaN, which would make NaN of the infinity)
                        const bool later = WIN && rs[c] > 0.0f;
                        mul[c] = later ? rs[c] : 1.0f;
                        const uint32_t see = (seen<WIN>(a, mask[c], from[c], key0, old, all) & in) >> (4 * g);
#pragma unroll
                        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                sc[sub][c][r] = see >> (16 * sub + r) & 1 ? (later ? sc[sub][c][r] : sc[sub][c][r] * rs[c])
                                                                          : -__builtin_inff();
                    }
                    // values that are not finite: zeros, and noted where they are the request's.
                    // (Waves that share the tile all do so, to the same effect.)
                    bool odd = false;
#pragma unroll 2
                    for (int x = 0; x < NI; ++x) {
                        auto* at = (__attribute__((address_space(3))) u4*)(uintptr_t)(
                            gbase + stage * S::STAGE + S::KTILE + x * S::VSTEP + lane * 16);
                        u4 v = *at;
                        bool bad = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool lo = (v[e] & EXP) == EXP, hi = (v[e] >> 16 & EXP) == EXP;
                            bad |= lo | hi;
                            v[e] = (lo ? 0u : v[e] & 0xFFFFu) | (hi ? 0u : v[e] & 0xFFFF0000u);
                        }
                        odd |= bad && key0 + x * ROWS + lane / SLOTS < keys;
                        *at = v;
                    }
                    if (odd) s_odd[wk] = 1;
                }

                // the next tile's products (of whatever is there, after the last) beside
                // this one's softmax
                f4 next[2][NR];
                u4 pf[NR][NL];
                float alpha[NR], ref[NR], sum[NR];
                bool moved = false;
                const auto maximum = [&](int c) {
                    float mx = sc[0][c][0];
#pragma unroll
                    for (int r = 1; r < 8; ++r) mx = fmaxf(mx, sc[r >> 2][c][r & 3]);
                    mx = max4(mx) * mul[c];
                    // the sums' reference follows the maximum in steps: exponentials
                    // of up to 2^LAG are as good as those up to 1
                    const float m = mx > mrow[c] + LAG ? mx : mrow[c];
                    moved |= m > mrow[c];
                    alpha[c] = __builtin_amdgcn_exp2f(mrow[c] - m);
                    mrow[c] = m;
                    ref[c] = BF16 ? -m : UP - m;
                    sum[c] = 0.0f;
                };
                const auto exponentials = [&](int c, int sub) {
                    float p[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        p[r] = __builtin_amdgcn_exp2f(fmaf(sc[sub][c][r], mul[c], ref[c]));
                        sum[c] += p[r];
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t q2[NL];
                        split2<BF16>(p[2 * e], p[2 * e + 1], minus1, q2);
#pragma unroll
                        for (int l = 0; l < NL; ++l) pf[c][l][2 * sub + e] = q2[l];
                    }
                    if (sub == 1) lrow[c] = lrow[c] * alpha[c] + sum[c];
                };
                // (with first call on the SIMD's issue, before waves that are at copies and the
                // second product: 103 -> 98 us at 131000 keys, bf16; 220 -> 217 at 32 x 8190)
                __builtin_amdgcn_s_setprio(1);
                products(stage1 * S::STAGE, next, [&](int s) {
                    // the rows' maxima, then their two halves of exponentials, spread over
                    // the steps
                    constexpr int PIECES = 3 * NR;
#pragma unroll
                    for (int x = s * PIECES / STEPS; x < (s + 1) * PIECES / STEPS; ++x) {
                        if (x < NR) maximum(x);
                        else exponentials((x - NR) / 2, (x - NR) % 2);
                    }
                });
                __builtin_amdgcn_s_setprio(0);
                if (__any(moved))
#pragma unroll
                    for (int c = 0; c < NR; ++c)
#pragma unroll
                        for (int d = 0; d < DT; ++d) o[d][c] *= alpha[c];

                const auto value = [&](int d) {
                    const uint32_t at = vlane[d & 3] + stage * S::STAGE + (d >> 2) * 128;
                    const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)at);
                    const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s4*)(uintptr_t)(at + J * S::VSTEP));
                    const u2 w0 = __builtin_bit_cast(u2, v0), w1 = __builtin_bit_cast(u2, v1);
                    return u4{w0[0], w0[1], w1[0], w1[1]};
                };
#pragma unroll
                for (int d = 0; d < DT; d += 2) {
                    const u4 vf[2] = {value(d), value(d + 1)};
#pragma unroll
                    for (int l = NL - 1; l >= 0; --l)
#pragma unroll
                        for (int x = 0; x < 2; ++x)
#pragma unroll
                            for (int c = 0; c < NR; ++c)
                                o[d + x][c] = mfma<BF16>(vf[x], pf[c][l], o[d + x][c]);
                }
                if constexpr (WR == 1) {
                    wait_lds();
                    if (i + 2 < n) {
                        at_v[0] = at_k[0], at_v[1] = at_k[1];
                        copy_v(stage);
                    }
                }
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                    for (int c = 0; c < NR; ++c) sc[sub][c] = next[sub][c];
                stage = stage1;
            }

            // an infinite cached key or value times the two signs (or a zero) of a query's
            // or probability's parts is NaN: once more, with the queries' parts of one sign
            // and all values looked at
            if (!careful) {
                bool nan = false;
#pragma unroll
                for (int c = 0; c < NR; ++c)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) nan |= o[d][c][r] != o[d][c][r];
                nan = WR == 1 ? __any(nan) : __syncthreads_or(nan);
                if (nan) {
                    careful = true;
                    goto again;
                }
            }

            // --- join the groups: each takes D / WK of the columns ---
            int ln = lane;  // (opaque: addresses made from it are not kept through the tiles)
            asm volatile("" : "+v"(ln));
#pragma unroll
            for (int c = 0; c < NR; ++c) {
                lrow[c] = sum4(lrow[c]);
                if (ln < 16) {
                    s_ml[0][wk][16 * (wr * NR + c) + ln % 16] = mrow[c];
                    s_ml[1][wk][16 * (wr * NR + c) + ln % 16] = lrow[c];
                }
            }
            lds_barrier();
            if (s_odd[wk]) {
                // what was taken out, back into the rows that see it
#pragma unroll 1
                for (int x = 0; x < n * KT; ++x) {
                    const int at = x % KT, key0 = key_at(x / KT), key = key0 + at;
                    if (key >= keys) break;
                    const int pg = sload(table + (key >> a.c.bs_log2));
                    if (no_block(a, pg) || !(careful || no_block(a, (int)highest) || key0 + KT > len ||
                                             (WIN && key0 < clear && key0 + KT > a.sinks)))
                        continue;
                    const uint8_t* v = vb + place_of(a, pg, key);
                    bool see[NR];
#pragma unroll
                    for (int c = 0; c < NR; ++c) see[c] = seen<WIN>(a, mask[c], from[c], key0, len - key0, keys - key0) >> at & 1;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const u2 x = *(const u2*)(v + 2 * (16 * d + 4 * (ln / 16)));
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t w = x[r >> 1] >> (16 * (r & 1)) & 0xFFFFu;
                            const float f = (w & EXP) != EXP ? 0.0f
                                            : w & (EXP ^ 0x7FFFu) ? __builtin_nanf("")
                                            : w & 0x8000u ? -__builtin_inff() : __builtin_inff();
#pragma unroll
                            for (int c = 0; c < NR; ++c)
                                if (see[c] && (w & EXP) == EXP) o[d][c][r] += f;
                        }
                    }
                }
            }
            float* buf = (float*)lds;  // the tiles are not needed any more
            float lsum[NR];
#pragma unroll
            for (int c = 0; c < NR; ++c) {
                const int rl = 16 * (wr * NR + c) + ln % 16;
                float m = LOWEST;
#pragma unroll
                for (int w = 0; w < WK; ++w) m = fmaxf(m, s_ml[0][w][rl]);
                lsum[c] = 0.0f;
#pragma unroll
                for (int w = 0; w < WK; ++w)
                    lsum[c] += s_ml[1][w][rl] * __builtin_amdgcn_exp2f(s_ml[0][w][rl] - m);
                const float f = __builtin_amdgcn_exp2f(mrow[c] - m);
                mrow[c] = m;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    o[d][c] *= f;
                    if (WK > 1) *(f4*)(buf + (((wave * NR + c) * DT + d) * 64 + ln) * 4) = o[d][c];
                }
            }
            lds_barrier();
            if (tid < WK) s_odd[tid] = 0;
            const bool whole = count == nu;
            float* part = a.part + (int64_t)(2 * wg + (first == 0)) * S::PART;
#pragma unroll
            for (int c = 0; c < NR; ++c) {
                const int rl = 16 * (wr * NR + c) + ln % 16, r = rt * RT + rl;
                const int t = r / a.G, hh = h * a.G + r % a.G;
                const float inv = lsum[c] != 0.0f ? 1.0f / lsum[c] : 0.0f;
                float* to = whole ? a.out + ((int64_t)(t0 + t) * a.hq + hh) * D : part + rl * D;
#pragma unroll
                for (int d0 = 0; d0 < DT / WK; ++d0) {
                    const int d = wk * (DT / WK) + d0;
                    f4 v;
                    if (WK > 1) {
                        v = f4{0, 0, 0, 0};
#pragma unroll
                        for (int w = 0; w < WK; ++w)
                            v += *(const f4*)(buf + ((((w * WR + wr) * NR + c) * DT + d) * 64 + ln) * 4);
                    } else {
                        v = o[d0][c];
                    }
                    if (whole) v = lsum[c] != 0.0f ? v * inv : f4{0, 0, 0, 0};
                    if (t < nt) *(f4*)(to + 16 * d + 4 * (ln / 16)) = v;
                }
                if (!whole && wk == 0 && ln < 16 && t < nt) {
                    part[RT * D + rl] = mrow[c];
                    part[RT * D + RT + rl] = lsum[c];
                }
            }
            if (first == 0 && !whole) {
                cut = true;
                if (tid == 0) {
                    const int64_t end = start + OV + nu - 1;  // the item's last unit
                    a.desc[wg] = (int)(end / span) - wg + 1;
                    desc[0] = t0, desc[1] = nt, desc[2] = h, desc[3] = rt;
                }
            }
            lds_barrier();  // the exchanged outputs are read
        }
        off -= rq.units;
    }
    if (!cut && tid == 0) a.desc[wg] = 0;
}

template <class S>
hipError_t go(AttnArgs a, int max_new, int cus, uint8_t* ws, hipStream_t st) {
    a.grid = S::PC * cus;
    a.desc = (int*)ws;
    a.part = (float*)(ws + DESC_BYTES);
    // Where a request has few keys at most (by its table's columns), its items are not
    // cut, and there is nothing to join: six units take about as long as a second launch
    // (one of 333 keys, D = 64: 12.4 us, cut 10.0 + 6.1; 64 of 370, one token: 23.1, cut
    // 25.8 + 6.6; 8 of 340, 8 tokens: 21.1, cut 15.3 + 6.2).  In a wider table the same
    // requests are cut: nothing on the host knows the lengths.  A window bounds them also:
    // 64 requests under one of 1000, one token, 48.6, cut 57 (with the launches).
    a.grid = std::min(a.grid, MAX_ITEMS);
    a.whole = S::WIN ? uncut<S>(a, max_new) : (int64_t)a.max_blocks << a.c.bs_log2 <= 6 * std::max(S::KU, 64);
    hipLaunchKernelGGL(attn_kernel<S>, dim3(a.grid), dim3(64 * S::WAVES), S::LDS, st, a);
    if (!a.whole) hipLaunchKernelGGL((attn_join<S::D, S::RT>), dim3(JOIN_WGS * cus), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <bool BF16, bool WIN, int D>
hipError_t rows(const AttnArgs& a, int max_new, int cus, uint8_t* ws, hipStream_t st) {
    // By the rows of an item: few rows take waves with keys of their own, which wait for
    // nobody, more rows waves that share a tile's copies.  Small work-groups, several to a
    // CU, each keeping step by itself, hide each other's waits.  Kernel and join, us,
    // 16 requests of 2045 to 4090 keys, 8 kv heads x 4, fp16:
    //                 16 rows                        32 rows
    //   D = 64    29.0, <1, 4, 1, 3, 3> 36.7    32.4, <1, 4, 1, 3, 3> 37.3
    //   D = 96    38.4, 43.4                    41.0, 43.9
    //   D = 128   44.6, 51.6 (<2, 1, 2, 2, 2>   49.3, 51.8
    //             47.0)
    //   D = 256   90.3, <1, 4, 1, 4, 1> 102     -
    //   D = 128, 36 to 64 rows: 53 to 56, <2, 4, 1, 4, 2> 76.
    // The kernel alone, 32 requests of up to 8190 keys, D = 128: 64 rows 166, <2, 2, 2, 4, 1>
    // 207; 128 rows, fp16 228 to 233, <1, 4, 1, 4, 2> 227, <2, 4, 1, 4, 2> 219 (but 65 against
    // 63 at 16 requests of 4090), <1, 8, 1, 8, 1> 286, <2, 4, 2, 4, 1> 265; bf16 233 to
    // 245, <1, 4, 1, 4, 2> 245 to 278, <2, 4, 1, 4, 2> 283, <1, 8, 1, 8, 1> 345.
    // D = 64, 32 rows, one request of 333 keys: <1, 2, 2, 4, 2> 13.7, <2, 1, 2, 2, 2>
    // 19.5, <2, 1, 4, 2, 1> 15.0.
    const int64_t r = (int64_t)max_new * a.G;
    if constexpr (D == 256) {
        if (r <= 16) return go<Shape<BF16, WIN, D, 1, 1, 2, 2, 1>>(a, max_new, cus, ws, st);
        return go<Shape<BF16, WIN, D, 1, 4, 1, 4, 1>>(a, max_new, cus, ws, st);
    } else {
        if (r <= 16) return go<Shape<BF16, WIN, D, 1, 1, 2, 2, 2>>(a, max_new, cus, ws, st);
        if constexpr (D == 64) {
            if (r <= 32) return go<Shape<BF16, WIN, D, 1, 2, 2, 4, 2>>(a, max_new, cus, ws, st);
        } else {
            if (r <= 32) return go<Shape<BF16, WIN, D, 2, 1, 2, 2, 2>>(a, max_new, cus, ws, st);
        }
        return go<Shape<BF16, WIN, D, 1, 4, 1, 3, 3>>(a, max_new, cus, ws, st);
    }
}

template <bool BF16, bool WIN>
hipError_t heads(const AttnArgs& a, int D, int max_new, int cus, uint8_t* ws, hipStream_t st) {
    switch (D) {
        case 64: return rows<BF16, WIN, 64>(a, max_new, cus, ws, st);
        case 96: return rows<BF16, WIN, 96>(a, max_new, cus, ws, st);
        case 128: return rows<BF16, WIN, 128>(a, max_new, cus, ws, st);
        default: return rows<BF16, WIN, 256>(a, max_new, cus, ws, st);
    }
}


}  // namespace
}  // namespace fq
