// fq_attnw.hip -- the attention kernel of fq_attn.hip with a sliding window and sinks.
//
// An item's units are those that hold the first `sinks` keys and those from the first key on that any of the
// request's new tokens sees (none lies before position len, so none sees a cached key before len + 1 -
// window); what lies between is neither shared out nor read.  Only tiles at the window's
// edge, where some of the item's rows see more than others, mask their scores.
//
// Bound as without a window, by the bytes of the keys seen and the begin of each item: 16 trees of up to
// 9 tokens behind 30000 keys under a window of 4096 with 5 sinks, 4 kv heads x 7, D = 128, bf16 (128 MB, matrix
// work 11 us): 46 + 9.6 us with the join, of 64 items cut over 768 work-groups, each of whose spans of about 11 units
// carries an item's fixed cost of 8.  64 of up to 20001 keys under one of 1000, one token, 8 x 4, fp16 (262 MB, 50
// us): 53, items whole.  The simple form of the trees, one wave's tiles with masks everywhere: 4939.  A prompt's
// tiles of rows all walk its whole range, as without a window: 2731 tokens, 8 x 4, fp16, under 1023 take 632 us.
#include "fq_attn16.h"

namespace fq {

hipError_t launch_attn_window16(const AttnArgs& a, bool bf16, int D, int max_new, int cus, uint8_t* ws,
                                hipStream_t st) {
    return bf16 ? heads<true, true>(a, D, max_new, cus, ws, st) : heads<false, true>(a, D, max_new, cus, ws, st);
}

}  // namespace fq
