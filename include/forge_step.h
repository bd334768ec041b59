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
 *   fq_verify_draft     which drafted tokens are accepted, and the next one, from
 *                       the head's rows and given random numbers
 *   fq_keep_accepted    an accepted branch's keys and values to the slots behind
 *                       the context
 *
 * and for caches of 8 bits and windows
 *
 *   fq_qk_norm_rope8    fq_qk_norm_rope into a cache of 8 bits
 *   fq_read_cache8      such a cache's keys and values in 16 or 32 bits
 *   fq_window_attention fq_tree_attention over either kind of cache, with a sliding
 *                       window and first tokens that stay visible
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
 * A cache of 8 bits (FQ_TYPE_I8) has int8 codes in the place of elements (strides multiples of
 * 16) and fp32 scales [num_blocks][kv heads][block_size / 16], contiguous: element =
 * code * scale of the 16 tokens (a group) and kv head.  A scale that is no positive finite number
 * counts as 0.  Codes are -127 .. 127 as written here; any are read.
 *
 * fq_tree_attention, fq_window_attention, fq_token_logprobs and fq_verify_draft keep partial results in the
 * library's per-stream workspace; fq_reserve_step sizes it for calls under
 * HIP-graph capture (fq_release_workspace frees it).  A graph uses the workspace of the stream
 * that it was captured on: such graphs and that stream's calls run one after the other.
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
#define FQ_TYPE_I8 101u   /* nor has this: codes with scales, for caches */

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

/* fq_qk_norm_rope with the keys and values rounded into a cache of 8 bits.  The tokens of a
 * group that come in one call stand next to each other, in rising slots, as fq_plan_step
 * gives them; the group's slots before its first one hold tokens of the request.  With y the
 * largest finite magnitude of the new keys (values) of a group and kv head, the
 * group's scale becomes
 *   s = y / 127            where the first new token is the group's first, else
 *   s = max(old s, y / 127), and where that is more, the codes held become
 *                          rint(code * (old s * (1 / s)))
 * and an element's code is rint(x * (1 / s)), held to -127 .. 127, 0 for NaN and where s is
 * below 2^-126.  Codes behind the group's last new token stay as they are.  Where
 * tokens of a group come otherwise, its codes and scale are unspecified.  The old s counts all that was written
 * since the group's first slot was, drafted tokens that were refused and are overwritten among it: a large
 * one leaves its group a coarser scale until that slot is written again.  D: a multiple of 16. */
int fq_qk_norm_rope8(const float* qkv, int64_t ld, int N, int hq, int hkv, int D, int rot,
                     int interleaved, const float* bias, const float* q_weight,
                     const float* k_weight, float eps, const int32_t* positions,
                     const int32_t* slots, const float* table, int table_rows, float* q,
                     int8_t* k_cache, int8_t* v_cache, float* k_scales, float* v_scales,
                     int num_blocks, int block_size, int64_t stride_block, int64_t stride_token,
                     int64_t stride_head, void* stream);

/* Keys and values of a cache of 8 bits as [N][hkv][D] of type F32, F16 or BF16: rows
 * starts[b] .. starts[b+1]-1 are request b's tokens from number first[b] on (first
 * NULL: from 0), zeros where the table has no block, and for rows past starts[B].  starts
 * [B+1] rises from 0.  D: a multiple of 16, at most 512.  N: at most 2^24 - 1 (2^28 - 16 where hkv * D is
 * 512 or less). */
int fq_read_cache8(const int8_t* k_cache, const int8_t* v_cache, const float* k_scales,
                   const float* v_scales, int num_blocks, int block_size, int hkv, int D,
                   int64_t stride_block, int64_t stride_token, int64_t stride_head,
                   const int32_t* block_table, int max_blocks, int64_t table_stride,
                   const int32_t* starts, const int32_t* first, int B, int N, uint32_t type,
                   void* k_out, void* v_out, void* stream);

/* fq_tree_attention for caches of type F16, BF16 (scales unused) or I8.  With window > 0, a
 * token at position p sees of these keys the ones at positions j with p - j < window or j <
 * sinks; a cached token's position is its number, a new one's lengths[b] + its depth, which
 * is, with masks, the number of its mask's bits less one (each of them a token that is
 * the parent of the next; 0 for a mask of none).  window 0: no window.  That holds for lengths past the
 * table's columns too, whose missing keys are not there.
 * I8: a query's elements are rounded to 24 bits of the largest of its token and head, m, which puts a score
 * off by |scale| m s (2^-23 (sum of |codes|) + 2^-14) at most, s the key's scale, beside fp32's roundings:
 * below a hundredth of what the codes' own rounding may do, but more than products in fp32 where a few
 * elements are far above the others. */
int fq_window_attention(const float* q, int64_t ldq, const int32_t* lengths, const int32_t* cu,
                        const uint64_t* masks, int B, int N, int max_new, int hq, int hkv, int D,
                        float scale, int window, int sinks, uint32_t cache_type,
                        const void* k_cache, const void* v_cache, const float* k_scales,
                        const float* v_scales, int num_blocks, int block_size,
                        int64_t stride_block, int64_t stride_token, int64_t stride_head,
                        const int32_t* block_table, int max_blocks, int64_t table_stride,
                        float* out, void* stream);

/* Verifies drafted tokens.  Request b's tokens are cu[b] .. cu[b+1]-1 of N, each with the
 * logits behind it (type F32, F16 or BF16, rows ld elements apart, V in each).  Token 0 of a request is known; token
 * i is drafted to follow token parents[i] (a number within the request below i, else it is
 * reached by nothing; NULL: i - 1).  With p = softmax(row / temperature[b]) (NULL: 1; at 0 or below: 1
 * for the largest logit, of equal ones the lowest token), from token 0 on, the tokens that follow the
 * last accepted one are tried in their order, token i with the random number uniforms[i]:
 *   draft_probs [N][V] (rows ldp apart; chains only): row i is the distribution that token i was
 *       drawn from; accepted where u q(token) < p(token).  Refused, max(p - q, 0) is left.
 *   NULL: accepted where u m < p(token), m = 1 - the p of those refused before it (a token
 *       that was refused already has p = 0).  Left is p without the tokens refused.
 * Where none is accepted, the next token is drawn from what is left (from p where that is
 * nothing): the lowest whose cumulated sum is above uniforms[cu[b]] times the whole.
 *   accepted [B]     accepted tokens, token 0 included; 0 for a request without tokens
 *   path [N]         path[cu[b] + d]: the number of the d-th accepted token; -1 behind
 *   next_tokens [B]  the next token; -1 for a request without tokens and after a row that
 *                    has a NaN or +inf logit or nothing but -inf: nothing is accepted behind it
 * A drafted token outside 0 .. V-1 is refused.  Uniforms are in [0, 1).  Acceptance and the next token
 * are those of sums in 64 bits.
 * With parents, tokens from the 65th of a request on are reached by nothing.  N at most 2^20. */
int fq_verify_draft(const void* logits, uint32_t type, int64_t ld, int V, const int32_t* tokens,
                    const int32_t* cu, int B, int N, const int32_t* parents,
                    const float* uniforms, const float* draft_probs, int64_t ldp,
                    const float* temperature, int32_t* accepted, int32_t* path,
                    int32_t* next_tokens, void* stream);

/* Moves request b's new tokens path[cu[b] + d] (numbers within the request, as
 * fq_verify_draft gives them), d < accepted[b], to the slots of its tokens lengths[b] + d: keys
 * and values of caches of any type, all read before any is written.  Of the first 64 only; those whose path is d,
 * or no new token, or whose slot is no block's, stay.  Caches of 8 bits: what is moved enters
 * its groups as in fq_qk_norm_rope8, with y / 127 = its scale * (its largest code / 127).  D: a multiple of
 * 8 (8 bits: 16), at most 512.  B * hkv: below 2^23. */
int fq_keep_accepted(uint32_t cache_type, void* k_cache, void* v_cache, float* k_scales,
                     float* v_scales, int num_blocks, int block_size, int hkv, int D,
                     int64_t stride_block, int64_t stride_token, int64_t stride_head,
                     const int32_t* block_table, int max_blocks, int64_t table_stride,
                     const int32_t* lengths, const int32_t* cu, const int32_t* path,
                     const int32_t* accepted, int B, int N, void* stream);

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
