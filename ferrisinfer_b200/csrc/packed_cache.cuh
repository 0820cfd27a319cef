// The paged cache in 4 bits: what its bytes mean, and the small helpers that every kernel on it shares.
//
// Every 32 neighbours of a head (a group) stand as  value = scale * code + least,  codes 0..15, scale and least bf16.
// A head of D elements has W = D / 32 groups and is, for keys and for values alike,
//   codes   D / 2 bytes  at codes  + ((page * kv_heads + head) * page_size + offset) * D / 2
//   scales  4 W bytes    at scales + ((page * kv_heads + head) * page_size + offset) * 4 W, word j: scale | least << 16 of group j
// The codes stand in the order in which the lanes of an mma.sync fragment take them, so that a lane reads its part of a row
// as one run (lane = 4 g + c below):
//   keys    word (4 bytes) c W + j holds elements 32 j + 8 c + 0..7, lowest four bits first: lane c of a row takes its part of all groups
//   values  halfword (2 bytes) g W + j holds elements 32 j + 4 g + 0..3: lanes g = 0..7 share the elements of a row
#pragma once

#include "common.cuh"
#include "sm100.cuh"

// n / d for n below 2^31 by a multiplication: multiplier = ceil(2^(32 + shift) / d) with 2^shift < d <= 2^(shift + 1).
struct DivideBy {
    uint32_t multiplier;
    int shift;

    explicit DivideBy(int d) : multiplier(0), shift(0) {
        if (d <= 1) return;
        while ((2ll << shift) < d) ++shift;
        multiplier = (uint32_t)(((1ull << (32 + shift)) + d - 1) / d);
    }
    DivideBy() = default;
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return multiplier ? __umulhi(n, multiplier) >> shift : n; }
};

struct PackedCache {
    uint8_t* k_codes;
    uint32_t* k_scales;
    uint8_t* v_codes;
    uint32_t* v_scales;
    int pages, kv_heads, page_size, head_dim;

    // Index of the row (page, head, offset); 64 bits: a cache of 180 GB has more bytes than 32 bits count.
    __device__ __forceinline__ size_t row(int page, int head, int off) const {
        return ((size_t)page * kv_heads + head) * page_size + off;
    }
};

// Scale and least of a word of the scales, exactly (bf16 is the upper half of an fp32).
__device__ __forceinline__ float packed_scale(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float packed_least(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// Whether the group stands for no finite numbers (the writer stores NaN in both).
__device__ __forceinline__ bool packed_not_finite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

// Why the C entries refuse a cache (nullptr: they do not).
inline const char* packed_cache_refusal(const PackedCache& c) {
    if (!c.k_codes || !c.k_scales || !c.v_codes || !c.v_scales) return "the packed cache has no memory";
    if (c.pages <= 0 || c.kv_heads <= 0 || c.page_size <= 0) return "the packed cache has no pages, heads or rows";
    if (c.head_dim <= 0 || c.head_dim % 32 || c.head_dim > 256) return "packed heads have a multiple of 32 elements, at most 256";
    if (((uintptr_t)c.k_codes | (uintptr_t)c.v_codes | (uintptr_t)c.k_scales | (uintptr_t)c.v_scales) & 15)
        return "the packed cache must begin on 16 bytes";
    if ((long long)c.pages * c.kv_heads > 0x7fffffff || (long long)c.pages * c.kv_heads * c.page_size > 0xffffffffll)
        return "the packed cache has more rows than 32 bits count";
    return nullptr;
}
