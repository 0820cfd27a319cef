// What the kernels of attention over the packed cache share.
#pragma once

#include <cuda_fp16.h>
#include <float.h>

#include "packed_cache.cuh"

constexpr float LOG2E = 1.4426950408889634f;

struct PackedAttention {
    const void* q;
    void* out;
    int ldq, ldo, q_aligned, out_aligned;  // rows of q, of out on 16 bytes
    PackedCache cache;
    const int* tables;
    int width;  // blocks of a request's table
    int limit;  // rows that a request may have: those of its table, and no more than the caller says
    const int* q_start;
    const int* start_row;
    int seqs, heads, group, window;
    float scale;  // of the scores, times log2(e)
    float* lse;   // log2 of the softmax's sum of every (token, head), or nullptr
    float* parts;  // unnormalised outputs, maximum and sum (D + 2 floats) of every query row, by [split][token][head] or [part][row]
    int splits, tokens;
    int even;       // the stages of all requests are dealt out evenly (steps whose rows fit one block) ...
    int most_blocks;  // ... to about so many blocks
    int* counters;  // per (request, kv head): blocks that have left their part (even), or nullptr: a kernel joins
    float* scores;  // [request][kv head][stage][32][8 NT], to the base of 2, or nullptr
    int max_stages;
    int few;        // most query rows of a request that the kernel for few rows takes; the other takes those with more
    DivideBy page;  // the page size
    float* weights;
    const int* seq_slot;
    int slots;  // rows of the weights that requests may have
    long long slot_stride;
    int head_stride, max_rows, add;
    int* status;

    __device__ __forceinline__ int block_of(int row) const { return (int)page.quotient((uint32_t)row); }
    // Index of a row of the cache: below 2^32, which the C entry sees to.
    __device__ __forceinline__ uint32_t row_of(int page, int head, int row, int block) const {
        return (uint32_t)(page * cache.kv_heads + head) * cache.page_size + (uint32_t)(row - block * cache.page_size);
    }
};

// The row of the weights that belongs to a request, -1 where it has none.
__device__ __forceinline__ int slot_of(const PackedAttention& p, int seq) {
    const int slot = p.seq_slot ? p.seq_slot[seq] : seq;
    if (slot >= p.slots) {
        ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 104);
        return -1;
    }
    return slot;
}

// The page of a request's row, -1 where it has none.
__device__ __forceinline__ int page_of(const PackedAttention& p, const int* table, int block) {
    const int page = block < p.width ? table[block] : -1;
    if (page >= p.cache.pages) {
        ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 83);
        return -1;
    }
    return page;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// The exponential unit alone: results below the normal range become nought.
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The four pairs of a word of codes less `OFF`, each an operand register: places i and i + 4 (keys), or the two halves' i (values).
template <int OFF>
__device__ __forceinline__ void code_pairs(uint32_t word, uint32_t (&pair)[4]) {
    const uint32_t up = word >> 8;
    pair[0] = (word & 0x000f000fu) | 0x64006400u;  // 1024 + code
    pair[1] = (word & 0x00f000f0u) | 0x64006400u;  // 1024 + 16 code
    pair[2] = (up & 0x000f000fu) | 0x64006400u;
    pair[3] = (up & 0x00f000f0u) | 0x64006400u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 x = *reinterpret_cast<const __half2*>(&pair[i]);
        const __half2 v = i & 1 ? __hfma2(x, __float2half2_rn(0.0625f), __float2half2_rn(-64.0f - OFF)) : __hsub2(x, __float2half2_rn(1024.0f + OFF));
        pair[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}

// The same in bf16, whose eight bits hold 128 + code.
template <int OFF>
__device__ __forceinline__ void code_pairs_bf16(uint32_t word, uint32_t (&pair)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = (word >> (4 * i) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), __float2bfloat162_rn(128.0f + OFF));
        pair[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Steps with more query rows of a request than `few`, for bf16 rows and heads of 64 and 128 (packed_prefill.cu).
struct PrefillPlan {
    int pairs, grid, sms;
    long long bytes, counters;  // scratch; whole numbers that are nought
};
PrefillPlan packed_prefill_plan(int head_dim, int seqs, int kv_heads, int group, int tokens, int max_q, int max_kv);
int packed_prefill(const PackedAttention& p, const PrefillPlan& plan, int max_kv, void* scratch, int* counters, cudaStream_t stream);
