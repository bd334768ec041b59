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

// What is wrong with a cache (forge_step.h's conventions), or FQ_OK.
int check_cache(uint32_t type, const void* k, const void* v, int num_blocks, int block_size,
                int64_t sb, int64_t st, int64_t sh) {
    if (type != FQ_TYPE_F16 && type != FQ_TYPE_BF16) return FQ_ERR_DTYPE;
    if (num_blocks < 1 || !block_size_ok(block_size) ||
        (int64_t)num_blocks * block_size > INT32_MAX)
        return FQ_ERR_SHAPE;
    // a wave's copy adds up to seven tokens to a 32-bit offset; strides are 32-bit factors
    if (sb < 0 || st < 0 || sh < 0 || sb > INT32_MAX || st > (1 << 26) || sh > INT32_MAX) return FQ_ERR_SHAPE;
    if (!k || !v) return FQ_ERR_NULL;
    if (!aligned16(k) || !aligned16(v) || ((sb | st | sh) & 7)) return FQ_ERR_ALIGN;
    return FQ_OK;
}

int device(int* dev) {
    const hipError_t e = hipGetDevice(dev);
    return e == hipSuccess ? FQ_OK : hip_fail(e);
}

int done(hipError_t e) { return e == hipSuccess ? FQ_OK : hip_fail(e); }

// One size for all calls, so that a stream's first call of any of them sizes its workspace for
// the others too, under capture as well (the attention's 51 MB on 256 CUs).
size_t step_bytes(int cus) { return std::max(fq::attn_part_bytes(cus), fq::logp_part_bytes(cus)); }

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
    if (N < 0 || hq < 1 || hkv < 1 || hq % hkv || D < 8 || D > 512 || D % 8 || rot < 0 || rot > D || rot % 8 ||
        table_rows < 0)
        return FQ_ERR_SHAPE;
    const int64_t heads = (int64_t)hq + 2 * (int64_t)hkv;
    // (up to 64 lanes to a head: the grid's lanes are 32 bits)
    if (heads * D > INT32_MAX || ld < heads * D || N * heads >= (1 << 26)) return FQ_ERR_SHAPE;
    if (N == 0) return FQ_OK;
    if (!qkv || !positions || !slots || !q || (rot && table_rows && !table)) return FQ_ERR_NULL;
    fq::RopeArgs a{};
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
    a.k = static_cast<uint16_t*>(k_cache);
    a.v = static_cast<uint16_t*>(v_cache);
    a.c = {num_blocks, log2_of(block_size), stride_block, stride_token, stride_head};
    return done(fq::launch_rope(a, cache_type == FQ_TYPE_BF16, interleaved != 0,
                                static_cast<hipStream_t>(stream)));
}

int fq_tree_attention(const float* q, int64_t ldq, const int32_t* lengths, const int32_t* cu,
                      const uint64_t* masks, int B, int N, int max_new, int hq, int hkv, int D,
                      float scale, uint32_t cache_type, const void* k_cache, const void* v_cache,
                      int num_blocks, int block_size, int64_t stride_block,
                      int64_t stride_token, int64_t stride_head, const int32_t* block_table,
                      int max_blocks, int64_t table_stride, float* out, void* stream) {
    const int rc = check_cache(cache_type, k_cache, v_cache, num_blocks, block_size, stride_block,
                               stride_token, stride_head);
    if (rc != FQ_OK) return rc;
    if (B < 1 || N < 0 || max_new < 0 || hq < 1 || hkv < 1 || hq % hkv || max_blocks < 1 ||
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
    fq::StreamScratch::Lease lease(fq::stream_scratch(dev, st, 2));
    uint8_t* ws = nullptr;
    const int rs = lease.get(step_bytes(cus), st, &ws);
    if (rs != FQ_OK) return rs;
    return done(fq::launch_attn(a, cache_type == FQ_TYPE_BF16, D, std::min(max_new, N), cus, ws, st));
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
