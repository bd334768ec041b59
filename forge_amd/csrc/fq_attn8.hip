// fq_attn8.hip -- attention over a cache of 8 bits, with or without a window.
//
// Items, units and their shares among the work-groups, tiles in rings, scores as K Q^T with the
// next tile's products beside this one's softmax, and lagging references are those of fq_attn.hip.  What
// differs: tiles are int8 codes, 32 keys in two groups of 16 that have a scale each.
//
// Scores: the fp32 queries, rounded to 24 bits of their row's largest element, are three signed bytes
// to the power-of-two base 256, so that all products with the codes are int8 matrix instructions
// with exact sums: no key is converted, and three of them take as long as one and a half of fp16's
// (two parts).  A score is its integer times the row's and the group's scale.  With m the row's largest element
// an element is off by 2^-23 m at most and a score by m (2^-23 sum |c| + 2^-14) of the key's scale (the lowest
// bytes' sums lose their fraction of 256): at most 2^-8 m of it for D = 128, where the cache's own rounding, half a
// code an element, is m / 2 of it in that element alone.  Against 64 bits on the same codes (4096 keys, D = 128, L1
// norm of the probabilities) that is 1e-7 for elements alike, 1.4e-6, 5.5e-6 and 3.3e-4 where one is 16, 64 and
// 4096 times the others and the codes there are 0; products in fp32 stay at 6e-8.  A fourth byte, of 16
// registers a lane and as many for its sums, does not fit: waves of 32 rows at D = 128, and all at 256, hold 256.
//
// Values: O = sum p s_v c.  Codes become fp16 (exactly: a byte beside 0x64 is 1024 and itself) and
// p s_v two fp16 parts as in fq_attn.hip.  The references are of the scores plus log2 s_v, so that
// p s_v stays in fp16's range whatever the groups' scales; the sums are of p.  (Where s_v is below
// 2^-80 the parts lose bits: an element is then off by up to 2^-109.)  The transposing read gives a lane
// its column's 8 keys; it is asked for before the softmax.
//
// Bound: for one token a request the bytes of codes, half of those of 16 bits, and what a tile costs to
// begin; with more rows the vector instructions beside the matrix ones: 16 codes become fp16 with 20 (of
// 32 keys x 128 columns for each 32 rows), a score its probability's parts with thirteen.  Kernel + join, us, D = 128:
// 48 requests of up to 5001 keys, one token, 4 kv heads x 7 (184 MB) 45 + 5.4; one of 131000, 13 tokens, 4 x 7
// (135 MB, matrix work 37) 80 + 10; 32 of up to 8190, 1 to 32 tokens, 8 x 4 (410 MB at least,
// 1160 asked of the L2s, 524 of memory; matrix work 79) 173 + 15; 64 of up to 20001 under a window of 1023,
// 8 x 4 (135 MB), items whole, 38; one of 333 keys 9.  There vector instructions are issued in 55 % of the cycles,
// matrix units busy in 28 %, with two waves a SIMD.  Steps (131000 keys / full batch):
// one wave's tiles without copies ahead 73500 / 13964; copies to LDS with the scales among them, eight waves
// a CU 107 / 219; values asked for before the softmax, conversions between the matrix instructions 94 / 186; waves
// of 32 rows on their own, four work-groups a CU 80 / 175; the next scores' conversion held there (the
// compiler moved it behind) 78 / 169; references lowered only where a scale above 2^60 is met, for bits (333 keys
// 5.5e-7 -> 4.9e-7 off), 80 / 173.
//
// A chain's tiles of rows all walk the keys from the first that any of the request's tokens sees to its last
// token's: a prompt of 2731 tokens, 8 x 4, takes 400 + 15 us where products up to each row's own token would take 96,
// and as long under a window of 1023 (58).
#include "fq_attn.h"
#include "fq_group8.h"

namespace fq {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i2 lds_i2;

constexpr int KT = 32;  // keys of a tile
constexpr int SUBS = KT / GROUP;
// By how much (log2) a row's largest score may be above its sums' reference, and what the probabilities'
// parts are raised by: together they stay below fp16's largest.
constexpr float LAG = 4.0f;
constexpr float UP = 2048.0f;
// The references are MOST_BELOW under the scores at most (groups of zeros have their part in the sums).
// From the first scale above LARGE on they are BELOW lower (log2), and p that much larger, so that p does not
// vanish at scales up to 2^121, those of the largest values.  (Not from the start: exponents of small
// magnitude are rounded less; 333 keys 4.9e-7 off, else 5.5e-7.)
constexpr float MOST_BELOW = -80.0f, LARGE = 1.152921504606846976e18f;  // 2^60
constexpr float BELOW = 20.0f, BELOW_TIMES = 1048576.0f;
constexpr float MOST = 8355711.0f;  // 127 (1 + 256 + 65536): the largest that three signed bytes hold
constexpr int LIMBS = 3;

// The largest of three.  (Written out: the compiler makes numbers that may be signalling NaN quiet first.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// x0, x1 as two pairs of fp16 that add up to them.  (The rest is one fused multiply-add from the packed part
// with its own rounding.)
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    hi = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x0, x1}), h2));
    asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(lo) : "v"(hi), "v"(x0));
    asm("v_fma_mixhi_f16 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(lo) : "v"(hi), "v"(x1));
}

// Four codes as fp16: a byte with its sign turned beside 0x64 is 1024 + 128 + code.
__device__ __forceinline__ void four_halves(uint32_t w, uint32_t& a, uint32_t& b) {
    const uint32_t x = w ^ 0x80808080u;
    const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const h2 lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + off;
    const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + off;
    a = __builtin_bit_cast(uint32_t, lo);
    b = __builtin_bit_cast(uint32_t, hi);
}

// WR x WK waves: each group of WR shares tiles of 32 keys, each of its waves with 16 NR rows of its own; the
// groups take every WK-th tile.  NS tiles of a group are in LDS.  PC work-groups to a CU.
template <int D_, int NR_, int WR_, int WK_, int NS_, int PC_>
struct Shape {
    static constexpr int D = D_, NR = NR_, WR = WR_, WK = WK_, NS = NS_, PC = PC_;
    static constexpr int WAVES = WR * WK;
    static constexpr int PITCH = D <= 64 ? 64 : D <= 128 ? 128 : 256;  // LDS row, bytes
    static constexpr int RT = 16 * NR * WR;
    static constexpr int KU = KT * WK;
    static constexpr int ROWS = 1024 / PITCH;  // rows of one copy
    static constexpr int J = 16 / ROWS;        // copies of 16 rows
    static constexpr int NI = SUBS * J;        // copies of a tile's keys, and of its values
    static constexpr int CW = 2 * NI / WR + 1;  // copies of a wave for a tile, its scales' among them
    // Bytes from copy to copy and (values) from group to group in LDS, and which bits of a row's number change
    // places of its 16-byte pieces among four: chosen so that the 16 keys of a read of keys, and the
    // 8 keys that two of the lanes' quarters take of both groups, lie in 16 places of the 256 bytes that
    // the banks span, with every place an immediate offset from few registers.
    static constexpr int KSTEP = 1024 + (D == 64 ? 0 : 64);
    static constexpr int VSTEP = 1024 + (D == 256 ? 64 : 0);
    static constexpr int VGROUP = J * VSTEP + (D == 64 ? 32 : D == 256 ? 128 : 64);
    static __device__ __forceinline__ int turn(int row) {
        return D == 64 ? (row >> 2) & 3 : D == 256 ? row & 3 : (row >> 1) & 3;
    }
    static constexpr int KTILE = NI * KSTEP, VTILE = SUBS * VGROUP;
    static constexpr int SCALES = KTILE + VTILE, STAGE = SCALES + 256;  // (the scales of 16 lanes' four each)
    static constexpr int GROUPS = NS * STAGE;
    // the waves' outputs are exchanged where the tiles were
    static constexpr size_t LDS = std::max((size_t)WK * GROUPS, WK > 1 ? (size_t)WAVES * NR * 16 * D * 4 : 0);
    static constexpr int PART = RT * (D + 2);  // floats of a partial result
    // What an item costs beside its units, in units.
    static constexpr int OV = 256 / KU;
    static_assert(2 * NI % WR == 0 && (WR == 1 ? NS == 2 : NS >= 3), "copies");
    static_assert(NI + (NS - 1) * (2 * NI + 1) < 64, "vmcnt");
    static_assert(PC * (LDS + 8 * WK * RT + 64) <= 160 * 1024, "LDS");
    static_assert(PC <= MAX_GRID && (size_t)PC * PART <= MAX_PART, "workspace");
};

template <class S>
__global__ __launch_bounds__(64 * S::WAVES, (S::WAVES * S::PC + 3) / 4) void attn8_kernel(AttnArgs a) {
    constexpr int D = S::D, NR = S::NR, WR = S::WR, WK = S::WK, NS = S::NS;
    constexpr int RT = S::RT, KU = S::KU, PITCH = S::PITCH, J = S::J, NI = S::NI, ROWS = S::ROWS;
    constexpr int OV = S::OV;
    constexpr int STEPS = (D + 63) / 64, DT = D / 16, SLOTS = PITCH / 16;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float s_ml[2][WK][RT];
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    // (the waves of a second work-group on a CU take their rows in another order: where an item has
    // fewer than RT, those without would be on the same SIMDs)
    const int wr = (wave + (int)(blockIdx.x * S::PC / gridDim.x) * (WR / 2)) % WR, wk = wave / WR;
    const int n16 = lane & 15, g = lane >> 4;
    const int wg = blockIdx.x;

    // --- the work-group's units (every wave finds them for itself) ---
    int64_t total, span, off;
    int b;
    // (up to 64 requests stay in the lanes, so that a request's numbers are not fetched again)
    const int per = (a.B + 63) / 64;
    int cu0 = 0, cu1 = 0, cached = 0;
    {
        const int first = lane * per;
        int64_t mine = 0;
        int longest = 0;
        for (int i = first; i < min(first + per, a.B); ++i) {
            cu0 = a.cu[i], cu1 = a.cu[i + 1], cached = a.lengths[i];
            const Request rq = request<RT, KU, OV, true>(a, cu0, cu1, cached);
            mine += rq.units;
            if (rq.units) longest = max(longest, rq.cost);
        }
        int64_t upto = mine;
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t v = __shfl_up(upto, o);
            if (lane >= o) upto += v;
        }
        total = uni64(__shfl(upto, 63));
        span = divided(total + gridDim.x - 1, gridDim.x);
        // (an item of `longest` units lies on that many work-groups and one at most)
        if (wg == 0) {
            const bool wide = __any(longest > (NARROW - 2) * span);
            if (tid == 0) a.desc[WIDE] = wide;
        }
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

    // --- constants of a lane ---
    const uint32_t gbase = lds_addr(lds) + wk * S::GROUPS;
    // a copy's source: bytes from the first row of its 16; and of this wave's share of the copies
    uint32_t src[J], mine[2 * NI / WR];
    {
        const int row = lane / SLOTS, slot = lane % SLOTS;
        int piece = slot ^ S::turn(row);
        if (16 * piece >= D) piece -= 4;  // (rows of 6 pieces among 8: the rest meets queries of 0)
        const uint32_t at = (uint32_t)(row * a.c.st) + piece * 16;
#pragma unroll
        for (int j = 0; j < J; ++j) src[j] = at + (uint32_t)(j * ROWS * a.c.st);
#pragma unroll
        for (int x = 0; x < 2 * NI / WR; ++x) mine[x] = at + (uint32_t)((WR * x + wr) % J * ROWS * a.c.st);
    }
    const uint32_t klane = gbase + n16 / ROWS * S::KSTEP + n16 % ROWS * PITCH + ((g ^ S::turn(n16)) << 4);
    uint32_t vlane[4];
    {
        const int i = n16 >> 1, row = 4 * g + (i & 3);  // of the lanes' 8 keys: 4 of each group
#pragma unroll
        for (int d = 0; d < 4; ++d)
            vlane[d] = gbase + S::KTILE + (i >> 2) * S::VGROUP + row / ROWS * S::VSTEP + row % ROWS * PITCH +
                       ((d ^ S::turn(row)) << 4) + (n16 & 1) * 8;
    }
    // lane l's of a tile's scales: of the keys' two groups, then the values'
    const uint8_t* scales = (const uint8_t*)(lane & 2 ? a.vs : a.ks);

    for (; left > 0; ++b) {
        const Request rq = per == 1 ? request<RT, KU, OV, true>(a, __builtin_amdgcn_readlane(cu0, b),
                                                                __builtin_amdgcn_readlane(cu1, b),
                                                                __builtin_amdgcn_readlane(cached, b))
                                    : request<RT, KU, OV, true>(a, sload(a.cu + b), sload(a.cu + b + 1),
                                                                sload(a.lengths + b));
        const int len = rq.len, keys = rq.keys, nu = rq.nu, t0 = rq.t0, nt = rq.nt;
        if (off >= rq.units) {
            off -= rq.units;
            continue;
        }
        int item = 0, pos = 0;
        if (off) {
            item = (int)divided(off, rq.cost);
            pos = (int)(off - (int64_t)item * rq.cost);
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
            // --- this group's tiles: wk, wk + WK, .. of the segment's (with a window, units behind the
            // sinks are left out).  Waves that share tiles keep step: as many tiles for each group ---
            const auto key_at = [&](int i) {
                const int unit = first + i;
                return (unit >= rq.su ? unit + rq.skip : unit) * KU + wk * KT;
            };
            const int n = WR > 1 || key_at(count - 1) < keys ? count : count - 1;
            const int last16 = (keys - 1) & ~15, last32 = (keys - 1) & ~31;
            const uint8_t* kb = a.k + (int64_t)h * a.c.sh;
            const uint8_t* vb = a.v + (int64_t)h * a.c.sh;
            const int* table = a.table + b * a.table_stride;
            // The first key that all of the item's rows see, and all from there on to the context's end.
            const int clear = a.window ? (int)min((int64_t)rq.pos + (a.masks ? 63 : min(nt - 1, (rt * RT + RT - 1) / a.G)) + 1 - a.window,
                                                  (int64_t)INT32_MAX) : 0;
            // A tile's pages, read ahead; where its two groups lie in a cache, and their scales; its
            // copies.  (Past the last tile: it again.)  In blocks of 32 tokens and more both are in one.
            const auto key_of = [&](int i) { return min(key_at(i), last32); };
            int page[SUBS];
            const auto read_pages = [&](int i) {
                const int key = key_of(i);
                page[0] = page[1] = sload(table + (key >> a.c.bs_log2));
                if (a.c.bs_log2 < 5) page[1] = sload(table + (min(key + GROUP, last16) >> a.c.bs_log2));
            };
            uint64_t at_k0 = 0, at_k1 = 0, at_v0 = 0, at_v1 = 0;  // of the tiles whose keys, values are copied next
            uint64_t at_s0 = 0, at_s1 = 0;                        // and of the first one's scales
            uint32_t highest = 0;             // of the pages placed so far (unsigned: -1 is above all blocks)
            const auto place = [&](int i) {
                const uint32_t in = (uint32_t)key_of(i) & ((1u << a.c.bs_log2) - 1);
                const uint32_t pg = min((uint32_t)page[0], (uint32_t)a.c.num_blocks - 1);
                at_v0 = at_k0, at_v1 = at_k1;
                at_k0 = (uint64_t)pg * (uint32_t)a.c.sb + (uint64_t)in * (uint32_t)a.c.st;
                at_s0 = (((uint64_t)pg * (uint32_t)a.hkv + (uint32_t)h) << (a.c.bs_log2 - 2)) + in / 4;  // (4 bytes a group)
                at_k1 = at_k0 + (uint64_t)(GROUP * (uint32_t)a.c.st);
                at_s1 = at_s0 + 4;
                highest = max(highest, (uint32_t)page[0]);
                if (a.c.bs_log2 < 5) {
                    const uint32_t other = min((uint32_t)page[1], (uint32_t)a.c.num_blocks - 1);
                    at_k1 = (uint64_t)other * (uint32_t)a.c.sb;
                    at_s1 = ((uint64_t)other * (uint32_t)a.hkv + (uint32_t)h) * 4;
                    highest = max(highest, (uint32_t)page[1]);
                }
            };
            // The keys of a tile that lie in a block.
            const auto there = [&](int i) {
                const int key = key_of(i), more = min(key + GROUP, last16);
                return (no_block(a, sload(table + (key >> a.c.bs_log2))) ? 0u : 0xFFFFu) |
                       (no_block(a, sload(table + (more >> a.c.bs_log2))) ? 0u : 0xFFFF0000u);
            };
            const auto copy_scales = [&](int stage) {
                dma4(scales + (lane & 1 ? at_s1 : at_s0), gbase + stage * S::STAGE + S::SCALES);
            };
            const auto copy_k = [&](int stage) {
                copy_scales(stage);
#pragma unroll
                for (int hf = 0; hf < SUBS; ++hf)
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        dma16s(src[j], kb + (hf ? at_k1 : at_k0), gbase + stage * S::STAGE + (hf * J + j) * S::KSTEP);
            };
            const auto copy_v = [&](int stage) {
#pragma unroll
                for (int hf = 0; hf < SUBS; ++hf)
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        dma16s(src[j], vb + (hf ? at_v1 : at_v0), gbase + stage * S::STAGE + S::KTILE + hf * S::VGROUP + j * S::VSTEP);
            };
            // This wave's share of a tile's keys and of the one before's values: copies wr, wr + WR, .. of the
            // NI of keys and the NI of values, copy c being number c % J of group c / J.
            // (Every wave copies the scales, to the same place.)
            const auto copy_share = [&](bool ks, int kstage, bool vs, int vstage) {
                if (ks) copy_scales(kstage);
#pragma unroll
                for (int x = 0; x < 2 * NI / WR; ++x) {
                    const int c = WR * x + wr;
                    const bool isv = c >= NI;
                    const int i = isv ? c - NI : c, hf = i / J, j = i % J;
                    if (isv) {
                        if (vs) dma16s(mine[x], vb + (hf ? at_v1 : at_v0),
                                       gbase + vstage * S::STAGE + S::KTILE + hf * S::VGROUP + j * S::VSTEP);
                    } else if (ks) {
                        dma16s(mine[x], kb + (hf ? at_k1 : at_k0), gbase + kstage * S::STAGE + i * S::KSTEP);
                    }
                }
            };

            read_pages(0);
            // (Rolled: a launch begins with none of its instructions in the cache.)
            if constexpr (WR == 1) {
                // K0 V0 K1 V1 ..; then the keys of tile i + NS once tile i's are used, and its values once those are
#pragma unroll 1
                for (int i = 0; i < NS; ++i) {
                    place(i);
                    read_pages(i + 1);
                    at_v0 = at_k0, at_v1 = at_k1;
                    if (i < n) {
                        copy_k(i);
                        copy_v(i);
                    }
                }
            } else {
                // K0, K1 V0, K2 V1, ..: each step's batch has the keys of one tile and the values of the one before
#pragma unroll 1
                for (int i = 0; i < NS; ++i) {
                    place(i);
                    read_pages(i + 1);
                    copy_share(i < n, i, i > 0 && i <= n, i - 1);
                }
            }
            // --- queries (on their way while the first tiles are): bytes of their row's largest's 2^-23 ---
            i4 qf[NR][STEPS][LIMBS];
            float rs[NR];
            uint64_t mask[NR];
            int from[NR];
#pragma unroll
            for (int c = 0; c < NR; ++c) {
                const int r = rt * RT + wr * 16 * NR + 16 * c + n16;
                const int t = r / a.G, hh = h * a.G + r % a.G;
                const bool on = t < nt;
                // (a chain: how many of the new tokens the row sees)
                mask[c] = !on ? 0 : a.masks ? a.masks[t0 + t] : (uint64_t)t + 1;
                from[c] = 0x7FFFFFFF;
                if (on) {
                    const Reach reached = reach(a, rq.pos, t, mask[c]);
                    mask[c] = reached.mask, from[c] = reached.from;
                }
                const float* q = a.q + (int64_t)(t0 + (on ? t : 0)) * a.ldq + (int64_t)(on ? hh : 0) * D;
                f4 x[STEPS][4];
                float mx = 0.0f;
                bool finite = true;
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool in = on && (D % 64 == 0 || 64 * s + 16 * g < D);
                        x[s][i] = in ? *(const f4u*)(q + 64 * s + 16 * g + 4 * i) : f4{0, 0, 0, 0};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            finite &= fabsf(x[s][i][e]) < __builtin_inff();
                            mx = fmaxf(mx, fabsf(x[s][i][e]));
                        }
                    }
                mx = max4(finite ? mx : __builtin_inff());
                float up = 0.0f, down = 1.0f;
                if (mx < __builtin_inff()) {
                    int e = min(23 - __builtin_amdgcn_frexp_expf(mx), 126);
                    if (ldexpf(mx, e) > MOST) --e;
                    up = mx > 0.0f ? ldexpf(1.0f, e) : 0.0f;
                    down = ldexpf(1.0f, -e);
                }
                // (the scale's sign goes with the query: the largest score is that of the largest
                // product; a row that is not finite has no score that is a number)
                up = copysignf(up, a.scale);
                rs[c] = mx < __builtin_inff() ? down * 256.0f * fabsf(a.scale) : __builtin_nanf("");
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)  // a byte and 128 in each place
                            v[e] = (uint32_t)((mx < __builtin_inff() ? (int)rintf(x[s][i][e] * up) : 0) + 0x808080);
                        const uint32_t lo = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u);  // bytes 0, 1 of two
                        const uint32_t hi = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u);
                        const uint32_t top = __builtin_amdgcn_perm(v[1], v[0], 0x0C0C0602u) |
                                             __builtin_amdgcn_perm(v[3], v[2], 0x06020C0Cu);
                        qf[c][s][0][i] = (int)(top ^ 0x80808080u);
                        qf[c][s][1][i] = (int)(__builtin_amdgcn_perm(hi, lo, 0x07060302u) ^ 0x80808080u);
                        qf[c][s][2][i] = (int)(__builtin_amdgcn_perm(hi, lo, 0x05040100u) ^ 0x80808080u);
                    }
            }

            // (a wave whose rows are none of the item's copies its share and waits with the others)
            const bool busy = WR == 1 || rt * RT + wr * 16 * NR < nt * a.G;
            f4 o[DT][NR];
            float mrow[NR], lrow[NR];
            float below = 0.0f, up_by = UP;  // (o is in units of up_by, whichever that is)
#pragma unroll
            for (int c = 0; c < NR; ++c) {
                mrow[c] = LOWEST;
                lrow[c] = 0.0f;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d][c] = f4{0, 0, 0, 0};
            }
            // Products of the keys at `at`, LIMBS STEPS runs of SUBS NR matrix instructions with beside(run)
            // after each.  Scores in units of 256: the lowest bytes' sums are shifted down (the
            // fraction, below 2^-15 of a largest element times one code, is the same to within
            // that for all keys) and the middle ones' added to them by the instructions themselves.  (All of
            // it stays below 2^31: 127 128 256 (256 + 2).)
            const auto products = [&](uint32_t at, i4 (&low)[SUBS][NR], i4 (&high)[SUBS][NR], const auto& begun,
                                      const auto& beside) {
                i4 kf[STEPS][SUBS];
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int sub = 0; sub < SUBS; ++sub)
                        kf[s][sub] = __builtin_bit_cast(i4, *(lds_u4*)(uintptr_t)(klane + at + J * sub * S::KSTEP + 64 * s));
                begun();
                const auto run = [&](int l, int s, i4 (&acc)[SUBS][NR], bool begin) {
#pragma unroll
                    for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
                        for (int c = 0; c < NR; ++c)
                            acc[sub][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                                kf[s][sub], qf[c][s][l], begin ? i4{0, 0, 0, 0} : acc[sub][c], 0, 0, 0);
                };
#pragma unroll
                for (int x = 0; x < LIMBS * STEPS; ++x) {
                    const int s = x % STEPS;
                    if (x < STEPS) run(2, s, low, s == 0);
                    else if (x < 2 * STEPS) run(0, s, high, s == 0);
                    else run(1, s, low, false);
                    __builtin_amdgcn_sched_barrier(0);
                    beside(x);
                    if (x == 2 * STEPS - 1)
#pragma unroll
                        for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
                            for (int c = 0; c < NR; ++c) low[sub][c] >>= 8;
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            const auto score = [&](const i4 (&low)[SUBS][NR], const i4 (&high)[SUBS][NR], f4 (&sc)[SUBS][NR], int sub, int c) {
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[sub][c][r] = (float)((high[sub][c][r] << 8) + low[sub][c][r]);
            };
            f4 sc[SUBS][NR];
            if constexpr (WR == 1) {
                if (n >= NS) wait_vm<NI + (NS - 1) * (2 * NI + 1)>();
                else wait_vm<0>();
            } else {
                if (n >= NS) wait_vm<(NS - 1) * S::CW>();
                else wait_vm<0>();
                lds_barrier();
            }
            if (busy) {
                i4 low[SUBS][NR], high[SUBS][NR];
                products(0, low, high, [] {}, [](int) {});
#pragma unroll
                for (int x = 0; x < SUBS * NR; ++x) score(low, high, sc, x / NR, x % NR);
            }
            int stage = 0;
            for (int i = 0; i < n; ++i) {
                const int key0 = key_at(i);
                const int stage1 = stage + 1 < NS ? stage + 1 : 0;
                // (landed with its keys; its place is filled anew from the next wait on)
                const u4 ts = *(lds_u4*)(uintptr_t)(gbase + stage * S::STAGE + S::SCALES);
                // this tile's values and the next one's keys have landed: this wave's copies of them, then
                // everyone's; and all are done with this one's keys and the last one's values, whose places are
                // filled anew
                if constexpr (WR == 1) {
                    wait_lds();
                    if (i + NS < n) {
                        place(i + NS);
                        read_pages(i + NS + 1);
                        copy_k(stage);
                        wait_vm<(NS - 1) * (2 * NI + 1)>();
                    } else if (i + 1 < n) {
                        wait_vm<NI>();
                    } else {
                        wait_vm<0>();
                    }
                } else {
                    if (i + NS - 1 < n) wait_vm<(NS - 2) * S::CW>();
                    else wait_vm<0>();
                    lds_barrier();
                    if (i + NS - 1 < n) {
                        place(i + NS);
                        read_pages(i + NS + 1);
                        copy_share(i + NS < n, stage, true, stage ? stage - 1 : NS - 1);
                    }
                }
                if (!busy) {
                    stage = stage1;
                    continue;
                }
                const bool holes = no_block(a, (int)highest);
                const bool tail = holes || key0 + KT > len || (key0 < clear && key0 + KT > a.sinks);
                float mul[SUBS][NR], sv[SUBS], lift[SUBS];
#pragma unroll
                for (int sub = 0; sub < SUBS; ++sub) {
                    const float sk = held_scale(__uint_as_float(ts[sub]));
                    sv[sub] = held_scale(__uint_as_float(ts[SUBS + sub]));
                    // (any number near log2 sv; a group of zeros still has its part in the sums)
                    lift[sub] = fmaxf(__builtin_amdgcn_logf(sv[sub]), MOST_BELOW);
#pragma unroll
                    for (int c = 0; c < NR; ++c) mul[sub][c] = rs[c] * sk;
                }
                if (__any(fmaxf(sv[0], sv[1]) > LARGE) && below == 0.0f) {
                    below = BELOW;
                    up_by = UP / BELOW_TIMES;
#pragma unroll
                    for (int c = 0; c < NR; ++c) mrow[c] -= BELOW, lrow[c] *= BELOW_TIMES;
                }
#pragma unroll
                for (int sub = 0; sub < SUBS; ++sub) lift[sub] -= below;
                if (tail) {
                    const int old = len - key0, all = keys - key0;
                    const uint32_t in = holes ? there(i) : ~0u;
#pragma unroll
                    for (int c = 0; c < NR; ++c) {
                        const uint32_t see = (seen<true>(a, mask[c], from[c], key0, old, all) & in) >> (4 * g);
#pragma unroll
                        for (int sub = 0; sub < SUBS; ++sub) {
                            // (a factor of 0 or NaN would make NaN of the infinity: put in at once; any
                            // other as in a tile that is seen whole, with the same bits)
                            const bool later = mul[sub][c] > 0.0f;
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                sc[sub][c][r] = see >> (16 * sub + r) & 1 ? (later ? sc[sub][c][r] : sc[sub][c][r] * mul[sub][c])
                                                                          : -__builtin_inff();
                            mul[sub][c] = later ? mul[sub][c] : 1.0f;
                        }
                    }
                }

                // the next tile's products (of whatever is there, after the last) beside this one's softmax
                i4 low[SUBS][NR], high[SUBS][NR];
                i2 raw[DT];  // this tile's values, asked for behind the keys: nothing waits for them
                u4 ph[NR], pl[NR];  // the probabilities' parts
                float alpha[NR], sum[NR];
                bool moved = false;
                const auto maximum = [&](int c) {
                    float most[SUBS];
#pragma unroll
                    for (int sub = 0; sub < SUBS; ++sub) {
                        const f4 v = sc[sub][c];
                        most[sub] = fmaf(max3(v[0], v[1], max3(v[2], v[3], v[3])), mul[sub][c], lift[sub]);
                    }
                    const float mx = max4(max3(most[0], most[1], LOWEST));
                    // the sums' reference follows the maximum in steps: exponentials of up to 2^LAG are as
                    // good as those up to 1
                    const float m = mx > mrow[c] + LAG ? mx : mrow[c];
                    moved |= m > mrow[c];
                    alpha[c] = __builtin_amdgcn_exp2f(mrow[c] - m);
                    mrow[c] = m;
                    sum[c] = 0.0f;
                };
                const auto exponentials = [&](int c, int sub) {
                    float p[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        p[r] = __builtin_amdgcn_exp2f(fmaf(sc[sub][c][r], mul[sub][c], -mrow[c]));
                        sum[c] += p[r];
                        p[r] *= up_by * sv[sub];
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t hi, lo;
                        split2(p[2 * e], p[2 * e + 1], hi, lo);
                        ph[c][2 * sub + e] = hi;
                        pl[c][2 * sub + e] = lo;
                    }
                    if (sub == SUBS - 1) lrow[c] = lrow[c] * alpha[c] + sum[c];
                };
                __builtin_amdgcn_s_setprio(1);
                products(stage1 * S::STAGE, low, high, [&] {
#pragma unroll
                    for (int d = 0; d < DT; ++d)
                        raw[d] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                            (lds_i2*)(uintptr_t)(vlane[d & 3] + stage * S::STAGE + (d >> 2) * 64));
                    // (the rows' maxima while the keys are on their way from LDS)
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 0; c < NR; ++c) maximum(c);
                }, [&](int s) {
                    // the groups' exponentials, spread over the runs
                    constexpr int PIECES = SUBS * NR, RUNS = STEPS * LIMBS;
#pragma unroll
                    for (int x = s * PIECES / RUNS; x < (s + 1) * PIECES / RUNS; ++x) exponentials(x / SUBS, x % SUBS);
                });
                __builtin_amdgcn_s_setprio(0);
                if (__any(moved))
#pragma unroll
                    for (int c = 0; c < NR; ++c)
#pragma unroll
                        for (int d = 0; d < DT; ++d) o[d][c] *= alpha[c];

                // Two of the columns' 16s at a time.  After each of their matrix instructions, while the unit
                // has it: four codes of the next two's, or some of the next scores.
                const auto four = [&](int d, int half, u4& to) {
                    uint32_t x, y;
                    four_halves((uint32_t)raw[d][half], x, y);
                    to[2 * half] = x, to[2 * half + 1] = y;
                };
                u4 vf[2];
#pragma unroll
                for (int x = 0; x < 4; ++x) four(x >> 1, x & 1, vf[x >> 1]);
#pragma unroll
                for (int d = 0; d < DT; d += 2) {
                    constexpr int RUN = 4 * NR, SCORES = SUBS * NR * 4, TWOS = DT / 2;
                    u4 after[2];
#pragma unroll
                    for (int m = 0; m < RUN; ++m) {
                        const int l = m < RUN / 2, x = m / NR % 2, c = m % NR;  // (the lower parts first)
                        o[d + x][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            __builtin_bit_cast(h8, vf[x]), __builtin_bit_cast(h8, l ? pl[c] : ph[c]), o[d + x][c], 0, 0, 0);
                        if (d + 2 < DT && m % NR == 0) four(d + 2 + m / NR / 2, m / NR % 2, after[m / NR / 2]);
                        const int s0 = d / 2 * SCORES / TWOS, s1 = (d / 2 + 1) * SCORES / TWOS;
#pragma unroll
                        for (int e = s0 + m * (s1 - s0) / RUN; e < s0 + (m + 1) * (s1 - s0) / RUN; ++e) {
                            const int sub = e / 4 / NR, k = e / 4 % NR, r = e % 4;
                            float next = (float)((high[sub][k][r] << 8) + low[sub][k][r]);
                            asm volatile("" : "+v"(next));  // (here, and not behind the matrix instructions)
                            sc[sub][k][r] = next;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (d + 2 < DT) vf[0] = after[0], vf[1] = after[1];
                }
                if constexpr (WR == 1) {
                    wait_lds();
                    if (i + NS < n) {
                        at_v0 = at_k0, at_v1 = at_k1;
                        copy_v(stage);
                    }
                }
                stage = stage1;
            }

            // --- join the groups: each takes DW of the columns' 16s ---
            constexpr int DW = (DT + WK - 1) / WK;
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
                const float f = __builtin_amdgcn_exp2f(mrow[c] - m) * (1.0f / up_by);
                mrow[c] = m;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    o[d][c] *= f;
                    if (WK > 1) *(f4*)(buf + ((((wk * WR + wr) * NR + c) * DT + d) * 64 + ln) * 4) = o[d][c];
                }
            }
            lds_barrier();
            const bool whole = count == nu;
            float* part = a.part + (int64_t)(2 * wg + (first == 0)) * S::PART;
#pragma unroll
            for (int c = 0; c < NR; ++c) {
                const int rl = 16 * (wr * NR + c) + ln % 16, r = rt * RT + rl;
                const int t = r / a.G, hh = h * a.G + r % a.G;
                const float inv = lsum[c] != 0.0f ? 1.0f / lsum[c] : 0.0f;
                float* to = whole ? a.out + ((int64_t)(t0 + t) * a.hq + hh) * D : part + rl * D;
#pragma unroll
                for (int d0 = 0; d0 < DW; ++d0) {
                    const int d = wk * DW + d0;
                    if (DT % WK && d >= DT) break;
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
    a.grid = std::min(S::PC * cus, MAX_ITEMS);
    a.desc = (int*)ws;
    a.part = (float*)(ws + DESC_BYTES);
    a.whole = uncut<S>(a, max_new);
    hipLaunchKernelGGL(attn8_kernel<S>, dim3(a.grid), dim3(64 * S::WAVES), S::LDS, st, a);
    if (!a.whole) hipLaunchKernelGGL((attn_join<S::D, S::RT, true>), dim3(std::max(JOIN_WGS * cus, a.grid)), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int D>
hipError_t rows(const AttnArgs& a, int max_new, int cus, uint8_t* ws, hipStream_t st) {
    // By the rows of an item.  Up to 32, and wherever there are too few tiles of rows and keys to fill
    // the work-groups: waves of 16 rows with keys of their own, four groups of keys side by side, which share
    // a short item's units best.  More rows: waves of 32, so that codes are converted half as often, then two
    // that share a tile.  D = 256: 16 rows, whose sums fill the registers.  With the launches, us, the shape taken
    // first:
    //   D = 128, 8 kv heads x 4       <1, 1, 4, 2, 2>  <2, 1, 2, 2, 4>  <2, 2, 2, 3, 2>
    //   32 x 8190 keys, 16 rows             90.0            101              118
    //   16 x 4090, 32 rows                  40.7             46.3             53.0
    //   32 x 8190, 28 rows                 108              106              123
    //   the same, 48 rows                  139              118              128
    //   8 x 8190, 256 rows                 145              105               95.4
    //   32 x 8190, 160 rows                352              219              211
    //   D = 64, 16 x 8000, 32 rows          29.1             34.9             39.7
    //   the same, 96 rows                   42.9             42.2             50.0
    //   8 trees of 25 over 760 keys, 4 x 7 (175 rows, few tiles): 16.5, by rows alone 32
    //   D = 256, 16 x 8000, 2 x 5     <1, 1, 4, 2, 1>  <1, 1, 2, 2, 2>  <1, 2, 1, 3, 2>
    //   5 rows                              34.5             36.0             43.0
    //   30 rows                             44.0             42.4             45.8
    //   80 rows                             72.7             63.6             60.6
    const int64_t r = (int64_t)max_new * a.G;
    using Few = Shape<D, 1, 1, 4, 2, D == 256 ? 1 : 2>;
    const int64_t tiles = (int64_t)a.B * a.hkv * ((r + 15) / 16), units = most_keys<Few>(a, max_new) / Few::KU + 1;
    if (r <= 32 || tiles * units <= 16 * (int64_t)Few::PC * cus) return go<Few>(a, max_new, cus, ws, st);
    if constexpr (D == 256) {
        return go<Shape<D, 1, 2, 1, 3, 2>>(a, max_new, cus, ws, st);
    } else {
        if (r <= 128) return go<Shape<D, 2, 1, 2, 2, 4>>(a, max_new, cus, ws, st);
        return go<Shape<D, 2, 2, 2, 3, 2>>(a, max_new, cus, ws, st);
    }
}

}  // namespace

hipError_t launch_attn8(const AttnArgs& a, int D, int max_new, int cus, uint8_t* ws, hipStream_t st) {
    switch (D) {
        case 64: return rows<64>(a, max_new, cus, ws, st);
        case 96: return rows<96>(a, max_new, cus, ws, st);
        case 128: return rows<128>(a, max_new, cus, ws, st);
        default: return rows<256>(a, max_new, cus, ws, st);
    }
}

}  // namespace fq
