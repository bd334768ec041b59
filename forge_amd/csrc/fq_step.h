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
    int window, sinks;  // window 0: none
    const float *ks, *vs;  // of caches of 8 bits
};
size_t attn_part_bytes(int cus);  // of the largest call
hipError_t launch_attn(const AttnArgs& a, bool bf16, int D, int max_new, int cus, uint8_t* ws,
                       hipStream_t st);
// The same with a window (window 0: none); over a cache of 8 bits, with and without.
hipError_t launch_attn_window16(const AttnArgs& a, bool bf16, int D, int max_new, int cus, uint8_t* ws,
                                hipStream_t st);
hipError_t launch_attn8(const AttnArgs& a, int D, int max_new, int cus, uint8_t* ws, hipStream_t st);

// A cache of 8 bits: codes at a CacheView's places (elements of one byte) and scales
// [block][kv head][16 tokens].
constexpr int GROUP = 16;  // tokens that share a scale

struct Cache8 {
    int8_t *k, *v;
    float *ks, *vs;
    CacheView c;
    int hkv, D;
    __host__ __device__ int groups() const { return (1 << c.bs_log2) / GROUP; }  // of a block
};
// Where a token of a request lies: block * block size + its place there; -1: nowhere.
struct TableView {
    const int* p;
    int cols;
    int64_t stride;
    __device__ __forceinline__ int slot(int b, int64_t number, const CacheView& c) const {
        const int64_t col = number >> c.bs_log2;
        if (number < 0 || col >= cols) return -1;
        const int page = p[b * stride + col];
        if ((uint32_t)page >= (uint32_t)c.num_blocks) return -1;
        return (page << c.bs_log2) + (int)(number & ((1 << c.bs_log2) - 1));
    }
};

hipError_t launch_rope8(const RopeArgs& a, const Cache8& c, bool interleaved, hipStream_t st);

struct ReadArgs {
    Cache8 c;
    TableView table;
    const int *starts, *first;
    int B, N;
    void *k, *v;
};
int read8_rows(const Cache8& c);  // rows of a work-group of 256 lanes
hipError_t launch_read8(const ReadArgs& a, int type, hipStream_t st);

struct KeepArgs {
    void *k, *v;
    float *ks, *vs;
    CacheView c;
    int hkv, D;
    TableView table;
    const int *lengths, *cu, *path, *accepted;
    int B, N;
};
hipError_t launch_keep(const KeepArgs& a, bool codes, hipStream_t st);

struct VerifyArgs {
    const void* x;
    int64_t ld;
    int V;
    const int *tokens, *cu;
    int B, N;
    const int* parents;
    const float* u;
    const float* q;
    int64_t ldq;
    const float* temperature;
    int *accepted, *path, *next;
    int seg, parts;  // elements of a row's part, parts of a row
    uint8_t* ws;
};
size_t verify_part_bytes(int cus);  // of the largest call
hipError_t launch_verify(const VerifyArgs& a, int type, int cus, hipStream_t st);

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
