// fq_step_capi.cpp -- the extern "C" entry points of include/forge_step.h:
// argument checks, then one call of the kernels' launchers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "../../include/forge_step.h"
#include "fq_scratch.h"
#include "fq_step.h"

namespace {

using fq::hip_fail;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int log2_of(int n) {
    int l = 0;
    while ((1 << l) < n) ++l;
    return l;
}

bool block_size_ok(int n) { return n >= 16 && n <= 1024 && (n & (n - 1)) == 0; }

// What is wrong with a cache's places (forge_step.h's conventions), or FQ_OK; unit: elements of 16 bytes.
int check_places(const void* k, const void* v, int num_blocks, int block_size, int64_t sb, int64_t st, int64_t sh,
                 int unit) {
    if (num_blocks < 1 || !block_size_ok(block_size) ||
        (int64_t)num_blocks * block_size > INT32_MAX)
        return FQ_ERR_SHAPE;
    // a wave's copy adds up to seven tokens to a 32-bit offset; strides are 32-bit factors
    if (sb < 0 || st < 0 || sh < 0 || sb > INT32_MAX || st > (1 << 26) || sh > INT32_MAX) return FQ_ERR_SHAPE;
    if (!k || !v) return FQ_ERR_NULL;
    if (!aligned16(k) || !aligned16(v) || ((sb | st | sh) & (unit - 1))) return FQ_ERR_ALIGN;
    return FQ_OK;
}

// What is wrong with a cache of 16 bits.
int check_cache(uint32_t type, const void* k, const void* v, int num_blocks, int block_size,
                int64_t sb, int64_t st, int64_t sh) {
    if (type != FQ_TYPE_F16 && type != FQ_TYPE_BF16) return FQ_ERR_DTYPE;
    return check_places(k, v, num_blocks, block_size, sb, st, sh, 8);
}

// What is wrong with one of 8 bits.
int check_cache8(const void* k, const void* v, const void* ks, const void* vs, int num_blocks, int block_size,
                 int64_t sb, int64_t st, int64_t sh) {
    const int rc = check_places(k, v, num_blocks, block_size, sb, st, sh, 16);
    if (rc != FQ_OK) return rc;
    if (!ks || !vs) return FQ_ERR_NULL;
    return ((uintptr_t)ks | (uintptr_t)vs) & 3 ? FQ_ERR_ALIGN : FQ_OK;
}

int device(int* dev) {
    const hipError_t e = hipGetDevice(dev);
    return e == hipSuccess ? FQ_OK : hip_fail(e);
}

int done(hipError_t e) { return e == hipSuccess ? FQ_OK : hip_fail(e); }

// One size for all calls, so that a stream's first call of any of them sizes its workspace for
// the others too, under capture as well (the attention's 51 MB on 256 CUs).
size_t step_bytes(int cus) {
    return std::max({fq::attn_part_bytes(cus), fq::logp_part_bytes(cus), fq::verify_part_bytes(cus)});
}

// RopeArgs of a call whose cache is right, D in units of `unit`.
int rope_args(fq::RopeArgs& a, const float* qkv, int64_t ld, int N, int hq, int hkv, int D, int rot, const float* bias,
              const float* q_weight, const float* k_weight, float eps, const int32_t* positions, const int32_t* slots,
              const float* table, int table_rows, float* q, const fq::CacheView& c, int unit) {
    if (N < 0 || hq < 1 || hkv < 1 || hq % hkv || D < 8 || D > 512 || D % unit || rot < 0 || rot > D || rot % 8 ||
        table_rows < 0)
        return FQ_ERR_SHAPE;
    const int64_t heads = (int64_t)hq + 2 * (int64_t)hkv;
    // (up to 64 lanes to a head: the grid's lanes are 32 bits)
    if (heads * D > INT32_MAX || ld < heads * D || N * heads >= (1 << 26)) return FQ_ERR_SHAPE;
    if (N == 0) return FQ_OK;
    if (!qkv || !positions || !slots || !q || (rot && table_rows && !table)) return FQ_ERR_NULL;
    a.qkv = qkv;
    a.ld = ld;
    a.N = N;
    a.hq = hq;
    a.hkv = hkv;
    a.D = D;
    a.rot = table_rows ? rot : 0;  // (no table: no position is in it)
    a.bias = bias;
    a.qw = q_weight;
    a.kw = k_weight;
    a.eps = eps;
    a.positions = positions;
    a.slots = slots;
    a.table = table;
    a.table_rows = table_rows;
    a.q = q;
    a.c = c;
    return FQ_OK;
}

// Heads of keys that one call reads back or moves.
bool heads_ok(int hkv, int D, int unit) {
    return hkv >= 1 && D >= unit && D <= 512 && D % unit == 0 && (int64_t)hkv * D <= (1 << 24);
}

}  // namespace

extern "C" {

int fq_plan_step(const int32_t* lengths, const int32_t* new_tokens, const int32_t* parents, int B,
                 int N, int block_size, int32_t* block_table, int max_blocks,
                 int64_t table_stride, const int32_t* free_blocks, int n_free, int32_t* cu,
                 int32_t* slots, int32_t* positions, uint64_t* masks, int32_t* info,
                 void* stream) {
    if (B < 1 || B > 8192 || N < 0 || !block_size_ok(block_size) || max_blocks < 1 ||
        table_stride < max_blocks || n_free < 0)
        return FQ_ERR_SHAPE;
    if (!lengths || !new_tokens || !block_table || !cu || !info || (n_free && !free_blocks) ||
        (N && (!slots || !positions || (parents && !masks))))
        return FQ_ERR_NULL;
    fq::PlanArgs a{};
    a.lengths = lengths;
    a.new_tokens = new_tokens;
    a.parents = parents;
    a.B = B;
    a.N = N;
    a.bs_log2 = log2_of(block_size);
    a.table = block_table;
    a.max_blocks = max_blocks;
    a.table_stride = table_stride;
    a.free_blocks = free_blocks;
    a.n_free = n_free;
    a.cu = cu;
    a.slots = slots;
    a.positions = positions;
    a.masks = masks;
    a.info = info;
    return done(fq::launch_plan(a, static_cast<hipStream_t>(stream)));
}

int fq_qk_norm_rope(const float* qkv, int64_t ld, int N, int hq, int hkv, int D, int rot,
                    int interleaved, const float* bias, const float* q_weight,
                    const float* k_weight, float eps, const int32_t* positions,
                    const int32_t* slots, const float* table, int table_rows, float* q,
                    uint32_t cache_type, void* k_cache, void* v_cache, int num_blocks,
                    int block_size, int64_t stride_block, int64_t stride_token,
                    int64_t stride_head, void* stream) {
    const int rc = check_cache(cache_type, k_cache, v_cache, num_blocks, block_size, stride_block,
                               stride_token, stride_head);
    if (rc != FQ_OK) return rc;
    fq::RopeArgs a{};
    const int ra = rope_args(a, qkv, ld, N, hq, hkv, D, rot, bias, q_weight, k_weight, eps, positions, slots, table,
                             table_rows, q, {num_blocks, log2_of(block_size), stride_block, stride_token, stride_head}, 8);
    if (ra != FQ_OK || N == 0) return ra;
    a.k = static_cast<uint16_t*>(k_cache);
    a.v = static_cast<uint16_t*>(v_cache);
    return done(fq::launch_rope(a, cache_type == FQ_TYPE_BF16, interleaved != 0,
                                static_cast<hipStream_t>(stream)));
}

int fq_qk_norm_rope8(const float* qkv, int64_t ld, int N, int hq, int hkv, int D, int rot,
                     int interleaved, const float* bias, const float* q_weight,
                     const float* k_weight, float eps, const int32_t* positions,
                     const int32_t* slots, const float* table, int table_rows, float* q,
                     int8_t* k_cache, int8_t* v_cache, float* k_scales, float* v_scales,
                     int num_blocks, int block_size, int64_t stride_block, int64_t stride_token,
                     int64_t stride_head, void* stream) {
    const int rc = check_cache8(k_cache, v_cache, k_scales, v_scales, num_blocks, block_size, stride_block,
                                stride_token, stride_head);
    if (rc != FQ_OK) return rc;
    fq::RopeArgs a{};
    const int ra = rope_args(a, qkv, ld, N, hq, hkv, D, rot, bias, q_weight, k_weight, eps, positions, slots, table,
                             table_rows, q, {num_blocks, log2_of(block_size), stride_block, stride_token, stride_head}, 16);
    if (ra != FQ_OK || N == 0) return ra;
    return done(fq::launch_rope8(a, {k_cache, v_cache, k_scales, v_scales, a.c, hkv, D}, interleaved != 0,
                                 static_cast<hipStream_t>(stream)));
}

int fq_read_cache8(const int8_t* k_cache, const int8_t* v_cache, const float* k_scales,
                   const float* v_scales, int num_blocks, int block_size, int hkv, int D,
                   int64_t stride_block, int64_t stride_token, int64_t stride_head,
                   const int32_t* block_table, int max_blocks, int64_t table_stride,
                   const int32_t* starts, const int32_t* first, int B, int N, uint32_t type,
                   void* k_out, void* v_out, void* stream) {
    const int rc = check_cache8(k_cache, v_cache, k_scales, v_scales, num_blocks, block_size, stride_block,
                                stride_token, stride_head);
    if (rc != FQ_OK) return rc;
    if (type != FQ_TYPE_F32 && type != FQ_TYPE_F16 && type != FQ_TYPE_BF16) return FQ_ERR_DTYPE;
    if (!heads_ok(hkv, D, 16) || B < 1 || N < 0 || max_blocks < 1 || table_stride < max_blocks) return FQ_ERR_SHAPE;
    fq::ReadArgs a{};
    // (the kernel reads them)
    a.c = {const_cast<int8_t*>(k_cache), const_cast<int8_t*>(v_cache), const_cast<float*>(k_scales),
           const_cast<float*>(v_scales), {num_blocks, log2_of(block_size), stride_block, stride_token, stride_head},
           hkv, D};
    // (the grid's lanes, 256 for some rows, are 32 bits)
    if (((int64_t)N - 1) / fq::read8_rows(a.c) + 1 >= (1 << 24)) return FQ_ERR_SHAPE;
    if (N == 0) return FQ_OK;
    if (!block_table || !starts || !k_out || !v_out) return FQ_ERR_NULL;
    if (!aligned16(k_out) || !aligned16(v_out)) return FQ_ERR_ALIGN;
    a.table = {block_table, max_blocks, table_stride};
    a.starts = starts;
    a.first = first;
    a.B = B;
    a.N = N;
    a.k = k_out;
    a.v = v_out;
    return done(fq::launch_read8(a, type == FQ_TYPE_F32 ? 0 : type == FQ_TYPE_F16 ? 1 : 2,
                                 static_cast<hipStream_t>(stream)));
}

int fq_keep_accepted(uint32_t cache_type, void* k_cache, void* v_cache, float* k_scales,
                     float* v_scales, int num_blocks, int block_size, int hkv, int D,
                     int64_t stride_block, int64_t stride_token, int64_t stride_head,
                     const int32_t* block_table, int max_blocks, int64_t table_stride,
                     const int32_t* lengths, const int32_t* cu, const int32_t* path,
                     const int32_t* accepted, int B, int N, void* stream) {
    const bool codes = cache_type == FQ_TYPE_I8;
    const int rc = codes ? check_cache8(k_cache, v_cache, k_scales, v_scales, num_blocks, block_size, stride_block,
                                        stride_token, stride_head)
                         : check_cache(cache_type, k_cache, v_cache, num_blocks, block_size, stride_block,
                                       stride_token, stride_head);
    if (rc != FQ_OK) return rc;
    if (!heads_ok(hkv, D, codes ? 16 : 8) || B < 1 || N < 0 || max_blocks < 1 || table_stride < max_blocks ||
        (int64_t)B * hkv >= (1 << 23))  // (512 lanes each, the grid's lanes are 32 bits)
        return FQ_ERR_SHAPE;
    if (N == 0) return FQ_OK;
    if (!block_table || !lengths || !cu || !path || !accepted) return FQ_ERR_NULL;
    fq::KeepArgs a{};
    a.k = k_cache;
    a.v = v_cache;
    a.ks = k_scales;
    a.vs = v_scales;
    a.c = {num_blocks, log2_of(block_size), stride_block, stride_token, stride_head};
    a.hkv = hkv;
    a.D = D;
    a.table = {block_table, max_blocks, table_stride};
    a.lengths = lengths;
    a.cu = cu;
    a.path = path;
    a.accepted = accepted;
    a.B = B;
    a.N = N;
    return done(fq::launch_keep(a, codes, static_cast<hipStream_t>(stream)));
}

int fq_verify_draft(const void* logits, uint32_t type, int64_t ld, int V, const int32_t* tokens,
                    const int32_t* cu, int B, int N, const int32_t* parents,
                    const float* uniforms, const float* draft_probs, int64_t ldp,
                    const float* temperature, int32_t* accepted, int32_t* path,
                    int32_t* next_tokens, void* stream) {
    if (type != FQ_TYPE_F32 && type != FQ_TYPE_F16 && type != FQ_TYPE_BF16) return FQ_ERR_DTYPE;
    // (a row's last step ends past V; work-groups of 256 lanes for rows and chunks make up the grids: ints)
    if (B < 1 || B > 8192 || N < 0 || N > (1 << 20) || V < 1 || V > INT32_MAX / 2 || ld < V ||
        (draft_probs && (parents || ldp < V)))
        return FQ_ERR_SHAPE;
    if (!cu || !accepted || !next_tokens || (N && (!logits || !tokens || !uniforms || !path))) return FQ_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(logits) & (type == FQ_TYPE_F32 ? 3 : 1)) return FQ_ERR_ALIGN;
    int dev = 0;
    const int rd = device(&dev);
    if (rd != FQ_OK) return rd;
    const int cus = fq::device_info(dev).cus;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    fq::VerifyArgs a{};
    a.x = logits;
    a.ld = ld;
    a.V = V;
    a.tokens = tokens;
    a.cu = cu;
    a.B = B;
    a.N = N;
    a.parents = parents;
    a.u = uniforms;
    a.q = draft_probs;
    a.ldq = ldp;
    a.temperature = temperature;
    a.accepted = accepted;
    a.path = path;
    a.next = next_tokens;
    fq::StreamScratch::Lease lease(fq::stream_scratch(dev, st, 2));
    const int rs = lease.get(step_bytes(cus), st, &a.ws);
    if (rs != FQ_OK) return rs;
    return done(fq::launch_verify(a, type == FQ_TYPE_F32 ? 0 : type == FQ_TYPE_F16 ? 1 : 2, cus, st));
}

int fq_tree_attention(const float* q, int64_t ldq, const int32_t* lengths, const int32_t* cu,
                      const uint64_t* masks, int B, int N, int max_new, int hq, int hkv, int D,
                      float scale, uint32_t cache_type, const void* k_cache, const void* v_cache,
                      int num_blocks, int block_size, int64_t stride_block,
                      int64_t stride_token, int64_t stride_head, const int32_t* block_table,
                      int max_blocks, int64_t table_stride, float* out, void* stream) {
    if (cache_type == FQ_TYPE_I8) return FQ_ERR_DTYPE;
    return fq_window_attention(q, ldq, lengths, cu, masks, B, N, max_new, hq, hkv, D, scale, 0, 0, cache_type, k_cache,
                               v_cache, nullptr, nullptr, num_blocks, block_size, stride_block, stride_token, stride_head,
                               block_table, max_blocks, table_stride, out, stream);
}

int fq_window_attention(const float* q, int64_t ldq, const int32_t* lengths, const int32_t* cu,
                        const uint64_t* masks, int B, int N, int max_new, int hq, int hkv, int D,
                        float scale, int window, int sinks, uint32_t cache_type,
                        const void* k_cache, const void* v_cache, const float* k_scales,
                        const float* v_scales, int num_blocks, int block_size,
                        int64_t stride_block, int64_t stride_token, int64_t stride_head,
                        const int32_t* block_table, int max_blocks, int64_t table_stride,
                        float* out, void* stream) {
    const bool codes = cache_type == FQ_TYPE_I8;
    const int rc = codes ? check_cache8(k_cache, v_cache, k_scales, v_scales, num_blocks, block_size, stride_block,
                                        stride_token, stride_head)
                         : check_cache(cache_type, k_cache, v_cache, num_blocks, block_size, stride_block,
                                       stride_token, stride_head);
    if (rc != FQ_OK) return rc;
    if (B < 1 || N < 0 || max_new < 0 || hq < 1 || hkv < 1 || hq % hkv || max_blocks < 1 || window < 0 || sinks < 0 ||
        table_stride < max_blocks || (D != 64 && D != 96 && D != 128 && D != 256))
        return FQ_ERR_SHAPE;
    if ((int64_t)hq * D > INT32_MAX / 4 || ldq < (int64_t)hq * D || (int64_t)N * hq > INT32_MAX / 2)
        return FQ_ERR_SHAPE;
    if (N == 0) return FQ_OK;
    if (!q || !lengths || !cu || !block_table || !out) return FQ_ERR_NULL;
    if (!aligned16(out)) return FQ_ERR_ALIGN;
    int dev = 0;
    const int rd = device(&dev);
    if (rd != FQ_OK) return rd;
    const int cus = fq::device_info(dev).cus;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    fq::AttnArgs a{};
    a.q = q;
    a.ldq = ldq;
    a.lengths = lengths;
    a.cu = cu;
    a.masks = masks;
    a.B = B;
    a.N = N;
    a.hq = hq;
    a.hkv = hkv;
    a.G = hq / hkv;
    a.scale = scale * 1.44269504088896341f;
    a.k = static_cast<const uint8_t*>(k_cache);
    a.v = static_cast<const uint8_t*>(v_cache);
    a.c = {num_blocks, log2_of(block_size), stride_block, stride_token, stride_head};
    a.table = block_table;
    a.max_blocks = max_blocks;
    a.table_stride = table_stride;
    a.out = out;
    a.window = window;
    a.sinks = sinks;
    a.ks = k_scales;
    a.vs = v_scales;
    fq::StreamScratch::Lease lease(fq::stream_scratch(dev, st, 2));
    uint8_t* ws = nullptr;
    const int rs = lease.get(step_bytes(cus), st, &ws);
    if (rs != FQ_OK) return rs;
    const bool bf16 = cache_type == FQ_TYPE_BF16;
    max_new = std::min(max_new, N);
    if (codes) return done(fq::launch_attn8(a, D, max_new, cus, ws, st));
    return done(window ? fq::launch_attn_window16(a, bf16, D, max_new, cus, ws, st)
                       : fq::launch_attn(a, bf16, D, max_new, cus, ws, st));
}

int fq_token_logprobs(const void* logits, uint32_t type, int64_t ld, int M, int V,
                      const int32_t* targets, int J, int top, float* logprobs, float* entropy,
                      float* top_logprobs, int32_t* top_tokens, void* stream) {
    if (type != FQ_TYPE_F32 && type != FQ_TYPE_F16 && type != FQ_TYPE_BF16) return FQ_ERR_DTYPE;
    // (a row's last part ends past V, and 256 lanes a row make up the grid: ints)
    if (M < 0 || M > (1 << 22) || V < 1 || V > INT32_MAX / 2 || ld < V || J < 0 || top < 0 || top > 64 ||
        top > V)
        return FQ_ERR_SHAPE;
    if (M == 0) return FQ_OK;
    if (!logits || (J && (!targets || !logprobs)) || (top && (!top_logprobs || !top_tokens)))
        return FQ_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(logits) & (type == FQ_TYPE_F32 ? 3 : 1)) return FQ_ERR_ALIGN;
    int dev = 0;
    const int rd = device(&dev);
    if (rd != FQ_OK) return rd;
    const int cus = fq::device_info(dev).cus;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    fq::LogpArgs a{};
    a.x = logits;
    a.ld = ld;
    a.M = M;
    a.V = V;
    a.targets = targets;
    a.J = J;
    a.top = top;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.top_logprobs = top_logprobs;
    a.top_tokens = top_tokens;
    fq::StreamScratch::Lease lease(fq::stream_scratch(dev, st, 2));
    const int rs = lease.get(step_bytes(cus), st, &a.ws);
    if (rs != FQ_OK) return rs;
    return done(fq::launch_logp(a, type == FQ_TYPE_F32 ? 0 : type == FQ_TYPE_F16 ? 1 : 2, cus, st));
}

int fq_reserve_step(void* stream) {
    int dev = 0;
    const int rd = device(&dev);
    if (rd != FQ_OK) return rd;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    fq::StreamScratch::Lease lease(fq::stream_scratch(dev, st, 2));
    uint8_t* ws = nullptr;
    return lease.get(step_bytes(fq::device_info(dev).cus), st, &ws);
}

}  // extern "C"
