// fq_attnw.hip -- the attention kernel of fq_attn.hip with a sliding window and sinks.
//
// An item's units are those that hold the first `sinks` keys and those from the first key on that any of the
// request's new tokens sees (none lies before position len, so none sees a cached key before len + 1 -
// window); what lies between is neither shared out nor read.  Only tiles at the window's
// edge, where some of the item's rows see more than others, mask their scores.
#include "fq_attn16.h"

namespace fq {

hipError_t launch_attn_window16(const AttnArgs& a, bool bf16, int D, int max_new, int cus, uint8_t* ws,
                                hipStream_t st) {
    return bf16 ? heads<true, true>(a, D, max_new, cus, ws, st) : heads<false, true>(a, D, max_new, cus, ws, st);
}

}  // namespace fq
