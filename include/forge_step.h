/*
 * forge_step.h -- C ABI of the operators that surround the quantized matmuls
 * of forge_q.h in one decoding or verifying step over a paged key/value cache:
 *
 *   fq_plan_step        cache blocks, slots, positions and tree masks of the
 *                       step's tokens, from the requests' lengths
 *   fq_qk_norm_rope     fq_fused_qkv's rows to queries and cached keys, values
 *   fq_tree_attention   drafted tokens over their context and their ancestors
 *   fq_token_logprobs   log probabilities, entropy and top alternatives of
 *                       the head's rows
 *
 * They take the place of the reference's verification of drafted tokens
 * (src/inference/speculative.cpp:64) and of its paged cache, attention mask,
 * rotation and attention operators, for activations in fp32.
 *
 * Conventions: those of forge_q.h (status codes, stream as void*, asynchronous
 * calls, nothing throws).  Every pointer is a device pointer.
 *
 * A step has B requests.  Request b has lengths[b] cached tokens and brings
 * cu[b+1] - cu[b] new ones, tokens cu[b] .. cu[b+1]-1 of the N in the call; new
 * token i is number lengths[b] + i of the request.  Tokens past cu[B] are
 * padding.
 *
 * Paged cache: keys and values are arrays of num_blocks blocks of block_size
 * tokens (a power of two, 16 .. 1024), element (block, token, kv head, d) at
 * block * stride_block + token * stride_token + head * stride_head + d, in
 * elements of cache_type; strides are multiples of 8 elements below 2^31 (2^26 from
 * token to token) and the bases 16-byte aligned.  The request's token n is in block block_table[b][n / block_size],
 * at n % block_size; a token's slot is its block * block_size plus that.
 * Values read from device memory are held to their ranges by the kernels: no
 * length, table entry, slot or parent leads to an access out of bounds.  A table entry
 * outside 0 .. num_blocks-1 (fq_plan_step enters -1 where blocks ran out) is no block: no
 * token has a slot in it, and fq_tree_attention's tokens see no key of it.  Nor are there
 * slots or keys past the table's max_blocks columns, whatever the length.
 *
 * fq_tree_attention and fq_token_logprobs keep partial results in the
 * library's per-stream workspace; fq_reserve_step sizes it for calls under
 * HIP-graph capture (fq_release_workspace frees it).
 */
#ifndef FORGE_STEP_H
#define FORGE_STEP_H

#include <stdint.h>

#include "forge_q.h"

#ifdef __cplusplus
extern "C" {
#endif

/* DataType values of activations and caches. */
#define FQ_TYPE_F32 0u
#define FQ_TYPE_F16 1u
#define FQ_TYPE_BF16 100u /* no forge::DataType of its own */

/* Plans a step of up to B = 8192 requests and N tokens.
 *   cu [B+1]         prefix sums of new_tokens
 *   block_table      [B][max_blocks], rows table_stride apart: request b's
 *                    missing blocks, up to its ceil((length + new) / block_size),
 *                    are taken from free_blocks [n_free] front to back in request
 *                    order and entered
 *   slots [N]        each token's slot; -1 for padding, where blocks or
 *                    columns of the table ran out and where a block's slots pass
 *                    the largest int
 *   positions [N]    length + depth in the draft (0 for padding)
 *   masks [N]        (with parents only) bit j: the token is, or descends from,
 *                    token j of its request
 *   info [2]         blocks taken; blocks that were missing
 * parents [N]: the number, within the request, of each token's parent, -1 for
 * the context (so is what is no earlier token); NULL: a chain, each token's
 * parent the one before.  With parents, a request's tokens from the 65th on get
 * no slot, mask 0 and the depth 64.  Negative lengths and counts are 0. */
int fq_plan_step(const int32_t* lengths, const int32_t* new_tokens, const int32_t* parents, int B,
                 int N, int block_size, int32_t* block_table, int max_blocks,
                 int64_t table_stride, const int32_t* free_blocks, int n_free, int32_t* cu,
                 int32_t* slots, int32_t* positions, uint64_t* masks, int32_t* info,
                 void* stream);

/* For each token, qkv row [hq query | hkv key | hkv value heads of D] (rows
 * ld floats apart): x + bias (bias NULL: none); query and key heads over their
 * root mean square, x / sqrt(mean(x^2) + eps) * weight[D] (weights NULL: none);
 * their first rot elements rotated by the token's position:
 *   (a, b) -> (a cos - b sin, b cos + a sin),
 * pair i being (i, i + rot/2), interleaved: (2i, 2i + 1), with cos = table[position][i]
 * and sin = table[position][rot/2 + i].  Queries go to q [N][hq][D] in fp32,
 * keys and values to the caches at slots[n] (none where that is no slot), in
 * cache_type.  A position outside the table (table_rows) gives NaN queries and
 * keys.  D and rot: multiples of 8, D <= 512, rot <= D. */
int fq_qk_norm_rope(const float* qkv, int64_t ld, int N, int hq, int hkv, int D, int rot,
                    int interleaved, const float* bias, const float* q_weight,
                    const float* k_weight, float eps, const int32_t* positions,
                    const int32_t* slots, const float* table, int table_rows, float* q,
                    uint32_t cache_type, void* k_cache, void* v_cache, int num_blocks,
                    int block_size, int64_t stride_block, int64_t stride_token,
                    int64_t stride_head, void* stream);

/* out[n][h] = softmax(scale q[n][h] . k) v over the keys that token n sees, query
 * head h reading kv head h / (hq / hkv): all cached tokens of its request, and
 * of its new tokens (in the cache too) those of its mask's bits or, with masks
 * NULL, those up to itself, where the table has a block for them.  Zeros for a token that sees
 * nothing, or whose keys all score -inf, and for padding.  Keys that a token does not see have no part
 * in its result, whatever they hold.  q rows (tokens) are ldq floats apart, out is
 * [N][hq][D]; D is 64, 96, 128 or 256.  max_new: the most new tokens of a
 * request, as far as known (the tiles' size goes by it, results do not). */
int fq_tree_attention(const float* q, int64_t ldq, const int32_t* lengths, const int32_t* cu,
                      const uint64_t* masks, int B, int N, int max_new, int hq, int hkv, int D,
                      float scale, uint32_t cache_type, const void* k_cache, const void* v_cache,
                      int num_blocks, int block_size, int64_t stride_block,
                      int64_t stride_token, int64_t stride_head, const int32_t* block_table,
                      int max_blocks, int64_t table_stride, float* out, void* stream);

/* For each of M rows of V logits (type F32, F16 or BF16, rows ld elements apart),
 * with p = softmax(row):
 *   logprobs [M][J]      log p of targets [M][J] (NaN for one outside 0 .. V-1)
 *   entropy [M]          -sum p log p
 *   top_tokens [M][top], top_logprobs [M][top]   the largest logits, in
 *                        falling order, of equal ones the lowest token first
 * A row with a NaN or +inf logit, or with nothing but -inf, has NaN log
 * probabilities and entropy; NaN logits rank above all others.
 * 0 <= top <= min(64, V); J >= 0. */
int fq_token_logprobs(const void* logits, uint32_t type, int64_t ld, int M, int V,
                      const int32_t* targets, int J, int top, float* logprobs, float* entropy,
                      float* top_logprobs, int32_t* top_tokens, void* stream);

/* Sizes the calling stream's workspace for every call of this header. */
int fq_reserve_step(void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FORGE_STEP_H */
