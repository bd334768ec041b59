// fq_attn.hip -- attention of drafted tokens over a paged cache and over their
// ancestors in the draft.
//
// An item is one request, one kv head and up to RT = 16 NR WR rows (a row: one token
// with one of the G query heads that share the kv head).  The keys of all items,
// in units of 32 WK, and a fixed cost of each item are shared out evenly over the
// work-groups, whatever the requests' lengths: work-group w takes units [w span, (w + 1)
// span) and walks the items that they belong to.  Every work-group finds its place from
// the lengths alone (no plan, no length on the host).  An item cut by such a border
// leaves partial results (maximum, sum, unnormalised output), which a second
// kernel joins, in the order of the keys, so that results repeat.
//
// A tile is 32 keys and their values.  WR waves share one, each with 16 NR rows of
// its own; the WK groups of a work-group take every WK-th.  Tiles are copied straight
// from the cache's pages to LDS, one to three ahead, keys and values in rings of their
// own: a tile's keys go while its values are still used.  Scores are S^T = K Q^T: keys
// along the MFMA result's rows (four to a lane and tile of 16), queries along its
// columns (one to a lane), so that a row's statistics are its lanes' own and
// the exponentials are, in place, the second product's B operand: O^T = V^T P^T
// with the contraction's keys in the order in which the lanes hold them.  V^T is read
// from LDS by transposing reads (each 16 lanes take a 4 key x 16 element block).
// The next tile's score products stand between the pieces of this one's softmax,
// and the reference that the exponentials are taken against moves only where a
// row's largest score leaves it by more than 2^LAG: the outputs are seldom rescaled.
//
// Queries are fp32 and keep their bits: against fp16 keys a query is hi + lo
// in fp16 (22 bits, its row scaled by a power of two), against bf16 keys three
// bf16 parts (24 bits).  The probabilities take the same two or three parts,
// in fp16 scaled by 2^11 (so that parts down to 2^-35 of the row's largest
// count); statistics and sums are fp32.  So the matrix work is two or three times
// that of 16-bit queries.
//
// Rows and keys outside the lengths cost no branch in the common tile: only
// tiles that reach past the cached tokens (or past the first table entry that is no
// block) mask their scores, and there values that are not finite are taken out
// of the product (a masked key's 0 times NaN would reach rows that do not see
// it) and put back into the rows that see them.
//
// Bound: the bytes of keys and values, read once for each tile of RT rows: the tiles
// of one kv head are mostly on other dies, and 98 % of what they ask of the L2s is not
// there.  Kernel + join, us, D = 128, a large copy at 5.2 TB/s: 32 requests of 8190
// keys, 8 kv heads x 4, fp16 (1.07 GB, 207 us at that rate): 1 new token 209 + 7,
// 8 215 + 9, 16 235 + 14, 32 (two tiles of rows) 452 + 22, 64 (four) 884 + 31; the same of
// 4095 to 8190 keys and 1 to 32 tokens (0.80 GB, 1.27 asked of the
// L2s: 5.4 TB/s): 236 + 17; 48 of 1001 to 2001 keys, 4 x 7, bf16, one token 34 + 7; one of
// 131000, 13 tokens, 4 x 7, bf16 (two tiles of rows, 0.27 GB, matrix work 60): 100 + 10;
// one of 333 keys 12.4, uncut.  A chain's tiles of rows all walk the keys of its last
// token, with masks from its first new one on: 2048 tokens of a prompt, 8 x 4, fp16,
// take 344 + 18, where half the products would do.
#include "fq_attn16.h"

namespace fq {

size_t attn_part_bytes(int cus) {
    return DESC_BYTES + (size_t)cus * 2 * sizeof(float) * MAX_PART;
}

hipError_t launch_attn(const AttnArgs& a, bool bf16, int D, int max_new, int cus, uint8_t* ws,
                       hipStream_t st) {
    return bf16 ? heads<true, false>(a, D, max_new, cus, ws, st) : heads<false, false>(a, D, max_new, cus, ws, st);
}

}  // namespace fq
