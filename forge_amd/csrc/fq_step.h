// fq_step.h -- launch interface between fq_step_capi.cpp and the kernels of the
// step operators (include/forge_step.h).  Internal to the library.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fq {

struct PlanArgs {
    const int *lengths, *new_tokens, *parents;
    int B, N, bs_log2;
    int* table;
    int max_blocks;
    int64_t table_stride;
    const int* free_blocks;
    int n_free;
    int *cu, *slots, *positions;
    uint64_t* masks;
    int* info;
};
hipError_t launch_plan(const PlanArgs& a, hipStream_t st);

// Element (block, token, head, d) of both caches at block * sb + token * st +
// head * sh + d, in elements of 2 bytes.
struct CacheView {
    int num_blocks, bs_log2;
    int64_t sb, st, sh;
};

struct RopeArgs {
    const float* qkv;
    int64_t ld;
    int N, hq, hkv, D, rot;
    const float *bias, *qw, *kw;
    float eps;
    const int *positions, *slots;
    const float* table;
    int table_rows;
    float* q;
    uint16_t *k, *v;
    CacheView c;
};
hipError_t launch_rope(const RopeArgs& a, bool bf16, bool interleaved, hipStream_t st);

struct AttnArgs {
    const float* q;
    int64_t ldq;
    const int *lengths, *cu;
    const uint64_t* masks;
    int B, N, hq, hkv, G;  // G = hq / hkv
    float scale;           // times log2(e)
    const uint8_t *k, *v;
    CacheView c;
    const int* table;
    int max_blocks;
    int64_t table_stride;
    float* out;
    float* part;  // partial results of split items, attn_part_bytes
    int* desc;    // of each work-group: the parts of an item that it begins and another ends; that item
    int grid;     // work-groups
    bool whole;   // items are not cut
};
size_t attn_part_bytes(int cus);  // of the largest call
hipError_t launch_attn(const AttnArgs& a, bool bf16, int D, int max_new, int cus, uint8_t* ws,
                       hipStream_t st);

struct LogpArgs {
    const void* x;
    int64_t ld;
    int M, V;
    const int* targets;
    int J, top;
    float *logprobs, *entropy, *top_logprobs;
    int* top_tokens;
    int seg, splits;  // elements of a wave; work-groups of a row
    uint8_t* ws;      // results of split rows, logp_part_bytes
};
size_t logp_part_bytes(int cus);  // of the largest call
hipError_t launch_logp(const LogpArgs& a, int type, int cus, hipStream_t st);

}  // namespace fq
