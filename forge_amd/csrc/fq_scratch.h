// fq_scratch.h -- device properties and the per-stream scratch memory that the
// entry points share.  Defined in fq_capi.cpp.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <vector>

#include "../../include/forge_q.h"

namespace fq {

// Records e for fq_last_hip_error() and returns FQ_ERR_HIP.
int hip_fail(hipError_t e);

struct DevInfo {
    int cus = 0;
    size_t lds = 0;
};

DevInfo device_info(int dev);

// Device scratch per (device, stream, slot) for the MFMA path (slot 0: token
// operands, group sums, exponents and split-K partial slabs), the GGUF fused
// FFN / QKV (slot 1: the gate/up or per-matrix rows) and the step operators of
// forge_step.h (slot 2: partial results of split rows).
//
// A call holds its slot's lock (StreamScratch::Lease) from taking the pointer
// until its launches are enqueued, so two host threads sharing a stream never
// see a buffer change under them.  The buffer only grows, at least doubling;
// a superseded buffer is not freed inside a compute call (queued work may
// still read it, and waiting for it would block the host mid-stream): it is
// kept until fq_release_workspace(), so the workspace of a stream holds less
// than twice its largest request.  fq_reserve_workspace() sizes it up front;
// during HIP-graph capture a call that would have to grow it fails with
// FQ_ERR_WORKSPACE instead of allocating.
struct StreamScratch {
    std::mutex mu;
    uint8_t* p = nullptr;
    size_t n = 0;
    std::vector<uint8_t*> retired;

    class Lease {
      public:
        explicit Lease(StreamScratch& s) : lk_(s.mu), s_(s) {}
        // the slot's buffer, at least `bytes` long
        int get(size_t bytes, hipStream_t st, uint8_t** out) {
            if (s_.n < bytes) {
                hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
                if (st && hipStreamIsCapturing(st, &cs) == hipSuccess &&
                    cs != hipStreamCaptureStatusNone)
                    return FQ_ERR_WORKSPACE;
                const size_t want = std::max(bytes, 2 * s_.n);
                uint8_t* np = nullptr;
                const hipError_t e = hipMalloc(reinterpret_cast<void**>(&np), want);
                if (e != hipSuccess) return hip_fail(e);
                if (s_.p) s_.retired.push_back(s_.p);
                s_.p = np;
                s_.n = want;
            }
            *out = s_.p;
            return FQ_OK;
        }
        size_t held() const { return s_.n; }

      private:
        std::unique_lock<std::mutex> lk_;
        StreamScratch& s_;
    };
};

constexpr int kScratchSlots = 3;

StreamScratch& stream_scratch(int dev, hipStream_t st, int slot);

}  // namespace fq
