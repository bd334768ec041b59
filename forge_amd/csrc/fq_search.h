// fq_search.h -- which request a row belongs to.
#pragma once

#include <hip/hip_runtime.h>

namespace fq {

// The last b of 0 .. n-1 with starts[b] <= row (0 if there is none), starts rising: by the whole
// wave, for one row, 64 of them at a time (three loads one behind the other for 8192, where halving
// takes 13).
__device__ __forceinline__ int request_of(const int* starts, int n, int row) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (n > 1) {  // among lo .. lo + n - 1
        const int step = (n + 63) / 64, at = lane * step;
        const int here = at < n ? starts[lo + at] : 0x7FFFFFFF;
        const uint64_t in = __ballot(at < n && here <= row);
        const int k = in ? 63 - __builtin_clzll(in) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

}  // namespace fq
