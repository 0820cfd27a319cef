// Writing, reading and evicting rows of the paged cache in 4 bits (its bytes: packed_cache.cuh).
#include "packed_cache.cuh"

namespace {

// ---------------------------------------------------------------------------------------------
// write:  least = the group's minimum rounded down to bf16, scale = bf16((maximum - least) / 15),
//         code = round((x - least) / scale) to even, kept within 0..15; scale 0: code 0.
// Rounding the least DOWN keeps x - least >= 0, so an offset far larger than the group's spread still
// leaves every element within half a step of its value.  A group that holds NaN or infinity, or whose
// spread has no 32-bit number, stands as NaN throughout.
// A lane takes 8 elements of the keys and the same 8 of the values, four neighbouring lanes a group.
// ---------------------------------------------------------------------------------------------
struct Eight {
    float x[8];
};

template <typename T, bool VEC>
__device__ __forceinline__ Eight load8(const T* p) {
    Eight e;
    if constexpr (VEC && sizeof(T) == 2) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e.x[2 * i] = __uint_as_float(w[i] << 16);
            e.x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else if constexpr (VEC) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        e = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) e.x[i] = to_float(p[i]);
    }
    return e;
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const Eight& e) {
    if constexpr (VEC && sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(e.x[0], e.x[1]), pack_bf16(e.x[2], e.x[3]),
                                                  pack_bf16(e.x[4], e.x[5]), pack_bf16(e.x[6], e.x[7]));
    } else if constexpr (VEC) {
        reinterpret_cast<float4*>(p)[0] = make_float4(e.x[0], e.x[1], e.x[2], e.x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(e.x[4], e.x[5], e.x[6], e.x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = from_float<T>(e.x[i]);
    }
}

// The codes of this lane's 8 elements (element i in bits 4 i) and the group's word of scales; all 32 lanes take part.
__device__ __forceinline__ uint32_t quantise8(const Eight& e, uint32_t& scales) {
    float low = e.x[0], high = e.x[0], sum = 0.0f;  // fminf and fmaxf drop NaN: the sum keeps it, and infinities
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        low = fminf(low, e.x[i]);
        high = fmaxf(high, e.x[i]);
        sum += 0.0f * e.x[i];
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const bf16 least_h = __float2bfloat16_rd(low);
    const float least = __bfloat162float(least_h);
    const bf16 scale_h = __float2bfloat16_rn(__fdiv_rn(high - least, 15.0f));
    const float scale = __bfloat162float(scale_h);
    if (!(sum == 0.0f) || !isfinite(least) || !isfinite(scale)) {
        scales = 0x7fc07fc0u;
        return 0;
    }
    scales = (uint32_t)__bfloat16_as_ushort(scale_h) | (uint32_t)__bfloat16_as_ushort(least_h) << 16;
    uint32_t codes = 0;
    if (scale > 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = rintf(__fdiv_rn(e.x[i] - least, scale));
            codes |= (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f) << (4 * i);
        }
    }
    return codes;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) packed_write_kernel(const T* k, const T* v, int ldk, int ldv, const int* __restrict__ slots,
                                                           PackedCache cache, int tokens, int* status) {
    pdl_launch_dependents();
    pdl_wait();
    const int W = cache.head_dim / 32;
    const int per_token = cache.kv_heads * W * 4;
    const long long n = (long long)tokens * per_token, first = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    for (long long i = first; (i & ~31ll) < n; i += (long long)gridDim.x * blockDim.x) {  // whole warps: the shuffles take all lanes
        const bool live = i < n;
        const int t = live ? (int)(i / per_token) : 0, r = live ? (int)(i % per_token) : 0;
        const int c = r & 3, j = (r >> 2) % W, head = (r >> 2) / W;
        const int slot = live ? slots[t] : -1;
        const int page = slot >= 0 ? slot / cache.page_size : -1;
        if (page >= cache.pages) ferris_report(status, FERRIS_STATUS_BAD_INDEX, 80);
        const bool store = page >= 0 && page < cache.pages;
        Eight ek = {}, ev = {};
        if (store) {
            const size_t at = (size_t)head * cache.head_dim + 32 * j + 8 * c;
            ek = load8<T, VEC>(k + (size_t)t * ldk + at);
            ev = load8<T, VEC>(v + (size_t)t * ldv + at);
        }
        uint32_t ks, vs;
        const uint32_t kc = quantise8(ek, ks), vc = quantise8(ev, vs);
        if (store) {
            const size_t row = cache.row(page, head, slot - page * cache.page_size);
            reinterpret_cast<uint32_t*>(cache.k_codes)[row * (4 * W) + c * W + j] = kc;
            uint16_t* vd = reinterpret_cast<uint16_t*>(cache.v_codes) + row * (8 * W);
            vd[(2 * c) * W + j] = (uint16_t)vc;
            vd[(2 * c + 1) * W + j] = (uint16_t)(vc >> 16);
            if (c == 0) {
                cache.k_scales[row * W + j] = ks;
                cache.v_scales[row * W + j] = vs;
            }
        }
    }
}

// read: out[t] = the values that the row at slots[t] stands for, rounded once (zeros for slots below 0)
__device__ __forceinline__ Eight dequantise8(uint32_t codes, uint32_t scales) {
    const float scale = packed_scale(scales), least = packed_least(scales);
    Eight e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e.x[i] = fmaf((float)((codes >> (4 * i)) & 15), scale, least);
    return e;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) packed_read_kernel(PackedCache cache, const int* __restrict__ slots, T* k, T* v, int ldk, int ldv,
                                                          int tokens, int* status) {
    pdl_launch_dependents();
    pdl_wait();
    const int W = cache.head_dim / 32;
    const int per_token = cache.kv_heads * W * 4;
    const long long n = (long long)tokens * per_token;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int t = (int)(i / per_token), r = (int)(i % per_token);
        const int c = r & 3, j = (r >> 2) % W, head = (r >> 2) / W;
        const int slot = slots[t];
        const int page = slot >= 0 ? slot / cache.page_size : -1;
        if (page >= cache.pages) ferris_report(status, FERRIS_STATUS_BAD_INDEX, 81);
        Eight ek = {}, ev = {};
        if (page >= 0 && page < cache.pages) {
            const size_t row = cache.row(page, head, slot - page * cache.page_size);
            const uint32_t kc = reinterpret_cast<const uint32_t*>(cache.k_codes)[row * (4 * W) + c * W + j];
            const uint16_t* vs = reinterpret_cast<const uint16_t*>(cache.v_codes) + row * (8 * W);
            const uint32_t vc = (uint32_t)vs[(2 * c) * W + j] | (uint32_t)vs[(2 * c + 1) * W + j] << 16;
            ek = dequantise8(kc, cache.k_scales[row * W + j]);
            ev = dequantise8(vc, cache.v_scales[row * W + j]);
        }
        const size_t at = (size_t)head * cache.head_dim + 32 * j + 8 * c;
        store8<T, VEC>(k + (size_t)t * ldk + at, ek);
        store8<T, VEC>(v + (size_t)t * ldv + at, ev);
    }
}

// ---------------------------------------------------------------------------------------------
// evict: of the n rows of a request and kv head, `budget` stay: the first `keep_first`, the last
// `keep_last`, and of the others those of the greatest weight, the lower row first among equals.
// The order of floats as unsigned keys; NaN counts as greater than every number, -0 as 0.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t weight_key(float w, int row, int n, int keep_first, int keep_last) {
    if (row < keep_first || row >= n - keep_last) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int EVICT_THREADS = 1024;

// One block per (request, kv head): the budget-th greatest key by its four bytes, most significant first (a histogram
// of 256 bins each), then the kept rows in order, every warp its own run of rows.
__global__ void __launch_bounds__(EVICT_THREADS) packed_evict_select_kernel(const float* weights, long long slot_stride, int head_stride,
                                                                            const int* __restrict__ seq_rows, const int* __restrict__ seq_slot,
                                                                            int* kept_rows, float* kept_weights, long long kept_slot_stride,
                                                                            int kept_head_stride, int budget, int keep_first, int keep_last,
                                                                            int max_rows) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t chosen[2];
    __shared__ int greater[32], equal[32];
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.y, h = blockIdx.x, heads = gridDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = min(max(seq_rows[s], 0), max_rows), slot = seq_slot ? seq_slot[s] : s;
    const float* w = weights + slot * slot_stride + (long long)h * head_stride;
    int* rows = kept_rows + ((size_t)s * heads + h) * budget;
    float* kw = kept_weights ? kept_weights + slot * kept_slot_stride + (long long)h * kept_head_stride : nullptr;
    const int stay = min(n, budget);
    for (int i = stay + tid; i < budget; i += EVICT_THREADS) rows[i] = -1;
    if (n <= budget) {
        for (int i = tid; i < n; i += EVICT_THREADS) {
            rows[i] = i;
            if (kw) kw[i] = w[i];
        }
        return;
    }
    uint32_t prefix = 0;
    int want = budget;  // how many of the rows that share the prefix stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += EVICT_THREADS) hist[i] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
        for (int i = tid; i < n; i += EVICT_THREADS) {
            const uint32_t key = weight_key(w[i], i, n, keep_first, keep_last);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            int left = want, b = 255;
            for (; b > 0 && (int)hist[b] < left; --b) left -= (int)hist[b];
            chosen[0] = (uint32_t)b;
            chosen[1] = (uint32_t)left;
        }
        __syncthreads();
        prefix |= chosen[0] << shift;
        want = (int)chosen[1];
        __syncthreads();
    }
    // rows with key > prefix all stay, of those with key == prefix the first `want`
    const int run = (n + 1023) / 1024 * 32, begin = min(warp * run, n), end = min(begin + run, n);
    int gt = 0, eq = 0;
    for (int i = begin; i < end; i += 32) {
        const int r = i + lane;
        const uint32_t key = r < end ? weight_key(w[r], r, n, keep_first, keep_last) : 0u;
        gt += __popc(__ballot_sync(0xffffffffu, r < end && key > prefix));
        eq += __popc(__ballot_sync(0xffffffffu, r < end && key == prefix));
    }
    if (lane == 0) {
        greater[warp] = gt;
        equal[warp] = eq;
    }
    __syncthreads();
    int before_gt = 0, before_eq = 0;
    for (int i = 0; i < warp; ++i) {
        before_gt += greater[i];
        before_eq += equal[i];
    }
    for (int i = begin; i < end; i += 32) {
        const int r = i + lane;
        const float wr = r < end ? w[r] : 0.0f;
        const uint32_t key = r < end ? weight_key(wr, r, n, keep_first, keep_last) : 0u;
        const uint32_t above = __ballot_sync(0xffffffffu, r < end && key > prefix);
        const uint32_t same = __ballot_sync(0xffffffffu, r < end && key == prefix);
        const uint32_t lower = (1u << lane) - 1;
        const int rank = before_eq + __popc(same & lower);
        const bool stays = r < end && (key > prefix || (key == prefix && rank < want));
        if (stays) {
            const int at = before_gt + __popc(above & lower) + min(rank, want);
            rows[at] = r;
            if (kw) kw[at] = wr;
        }
        before_gt += __popc(above);
        before_eq += __popc(same);
    }
}

// Kept rows from their pages into others: block (rows, head, request), a thread 16 bytes of codes or one word of scales.
__global__ void __launch_bounds__(256) packed_evict_move_kernel(PackedCache from, PackedCache to, const int* __restrict__ from_tables,
                                                                int from_width, const int* __restrict__ to_tables, int to_width,
                                                                const int* kept_rows, int budget, int rows_per_block, int* status) {
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.z, h = blockIdx.y, heads = gridDim.y, W = from.head_dim / 32, ps = from.page_size, qs = to.page_size;
    const int* kept = kept_rows + ((size_t)s * heads + h) * budget;
    const int first = blockIdx.x * rows_per_block, count = min(rows_per_block, budget - first);
    const int per_row = 4 * W;  // W pieces of 16 bytes of codes and W words of scales, of keys and of values
    for (int i = threadIdx.x; i < count * per_row; i += blockDim.x) {
        const int at = first + i / per_row, part = i % per_row;
        const int row = kept[at];
        if (row < 0 || row / ps >= from_width || at / qs >= to_width) continue;
        const int sp = from_tables[(size_t)s * from_width + row / ps], dp = to_tables[(size_t)s * to_width + at / qs];
        if (sp < 0 || dp < 0) continue;
        if (sp >= from.pages || dp >= to.pages) {
            ferris_report(status, FERRIS_STATUS_BAD_INDEX, 82);
            continue;
        }
        const size_t a = from.row(sp, h, row % ps), b = to.row(dp, h, at % qs);
        const int j = part % W;
        if (part < W) {
            reinterpret_cast<uint4*>(to.k_codes)[b * W + j] = reinterpret_cast<const uint4*>(from.k_codes)[a * W + j];
        } else if (part < 2 * W) {
            reinterpret_cast<uint4*>(to.v_codes)[b * W + j] = reinterpret_cast<const uint4*>(from.v_codes)[a * W + j];
        } else if (part < 3 * W) {
            to.k_scales[b * W + j] = from.k_scales[a * W + j];
        } else {
            to.v_scales[b * W + j] = from.v_scales[a * W + j];
        }
    }
}

PackedCache make_cache(void* kc, void* ks, void* vc, void* vs, int pages, int kv_heads, int page_size, int head_dim) {
    return {(uint8_t*)kc, (uint32_t*)ks, (uint8_t*)vc, (uint32_t*)vs, pages, kv_heads, page_size, head_dim};
}

template <typename T>
bool eights_aligned(const void* p, int ld) {
    return ((uintptr_t)p & 15) == 0 && ld % (16 / (int)sizeof(T)) == 0;
}

int blocks_for(long long threads) {
    const long long most = (long long)(ferris_sm_count() > 0 ? ferris_sm_count() : 148) * 8;
    const long long blocks = (threads + 255) / 256;
    return (int)(blocks < most ? blocks : most);
}

template <typename T>
int write_rows(const void* k, const void* v, int ldk, int ldv, const int* slots, const PackedCache& cache, int tokens, cudaStream_t st) {
    const int blocks = blocks_for((long long)tokens * cache.kv_heads * (cache.head_dim / 8));
    auto kernel = eights_aligned<T>(k, ldk) && eights_aligned<T>(v, ldv) ? packed_write_kernel<T, true> : packed_write_kernel<T, false>;
    ferris_launch(kernel, dim3(blocks), dim3(256), 0, st, (const T*)k, (const T*)v, ldk, ldv, slots, cache, tokens, ferris_status_ptr());
    FERRIS_LAUNCH_CHECK();
}

template <typename T>
int read_rows(const PackedCache& cache, const int* slots, void* k, void* v, int ldk, int ldv, int tokens, cudaStream_t st) {
    const int blocks = blocks_for((long long)tokens * cache.kv_heads * (cache.head_dim / 8));
    auto kernel = eights_aligned<T>(k, ldk) && eights_aligned<T>(v, ldv) ? packed_read_kernel<T, true> : packed_read_kernel<T, false>;
    ferris_launch(kernel, dim3(blocks), dim3(256), 0, st, cache, slots, (T*)k, (T*)v, ldk, ldv, tokens, ferris_status_ptr());
    FERRIS_LAUNCH_CHECK();
}

}  // namespace

// The arguments of the two below, as their caller lays them out.
struct FerrisPackedRows {
    void *k, *v;
    const int* slots;
    void *k_codes, *k_scales, *v_codes, *v_scales, *stream;
    int dtype, ldk, ldv, pages, kv_heads, page_size, head_dim, tokens;

    PackedCache cache() const { return make_cache(k_codes, k_scales, v_codes, v_scales, pages, kv_heads, page_size, head_dim); }
};

FERRIS_API int ferris_packed_cache_write(const FerrisPackedRows* a) {
    if (const char* why = packed_cache_refusal(a->cache())) FERRIS_REFUSE("%s", why);
    if (a->tokens <= 0) return FERRIS_OK;
    if (a->dtype == FERRIS_BF16) return write_rows<bf16>(a->k, a->v, a->ldk, a->ldv, a->slots, a->cache(), a->tokens, (cudaStream_t)a->stream);
    if (a->dtype == FERRIS_F32) return write_rows<float>(a->k, a->v, a->ldk, a->ldv, a->slots, a->cache(), a->tokens, (cudaStream_t)a->stream);
    FERRIS_REFUSE("packed cache: dtype %d is not known", a->dtype);
}

FERRIS_API int ferris_packed_cache_read(const FerrisPackedRows* a) {
    if (const char* why = packed_cache_refusal(a->cache())) FERRIS_REFUSE("%s", why);
    if (a->tokens <= 0) return FERRIS_OK;
    if (a->dtype == FERRIS_BF16) return read_rows<bf16>(a->cache(), a->slots, a->k, a->v, a->ldk, a->ldv, a->tokens, (cudaStream_t)a->stream);
    if (a->dtype == FERRIS_F32) return read_rows<float>(a->cache(), a->slots, a->k, a->v, a->ldk, a->ldv, a->tokens, (cudaStream_t)a->stream);
    FERRIS_REFUSE("packed cache: dtype %d is not known", a->dtype);
}

FERRIS_API int ferris_packed_cache_evict(void* from_kc, void* from_ks, void* from_vc, void* from_vs, int from_pages, int from_page_size,
                                         void* to_kc, void* to_ks, void* to_vc, void* to_vs, int to_pages, int to_page_size, int kv_heads,
                                         int head_dim, const int* from_tables, int from_width, const int* to_tables, int to_width,
                                         const int* seq_rows, const int* seq_slot, const float* weights, long long slot_stride,
                                         int head_stride, int max_rows, int* kept_rows, float* kept_weights, long long kept_slot_stride,
                                         int kept_head_stride, int seqs, int budget, int keep_first, int keep_last, void* stream) {
    const PackedCache from = make_cache(from_kc, from_ks, from_vc, from_vs, from_pages, kv_heads, from_page_size, head_dim);
    const PackedCache to = make_cache(to_kc, to_ks, to_vc, to_vs, to_pages, kv_heads, to_page_size, head_dim);
    if (const char* why = packed_cache_refusal(from)) FERRIS_REFUSE("%s", why);
    if (const char* why = packed_cache_refusal(to)) FERRIS_REFUSE("%s", why);
    if (budget <= 0 || keep_first < 0 || keep_last < 0 || keep_first > budget - keep_last)
        FERRIS_REFUSE("eviction: %d first and %d last rows of a budget of %d", keep_first, keep_last, budget);
    if (seqs <= 0) return FERRIS_OK;
    if (seqs > 65535 || kv_heads > 65535) FERRIS_REFUSE("eviction: %d requests of %d kv heads", seqs, kv_heads);
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = ferris_launch(packed_evict_select_kernel, dim3(kv_heads, seqs), dim3(EVICT_THREADS), 0, st, weights, slot_stride, head_stride,
                                  seq_rows, seq_slot, kept_rows, kept_weights, kept_slot_stride, kept_head_stride, budget, keep_first,
                                  keep_last, max_rows);
    if (e == cudaSuccess) {
        const int rows_per_block = 64;
        ferris_launch(packed_evict_move_kernel, dim3((budget + rows_per_block - 1) / rows_per_block, kv_heads, seqs), dim3(256), 0, st, from, to,
                      from_tables, from_width, to_tables, to_width, (const int*)kept_rows, budget, rows_per_block, ferris_status_ptr());
    }
    FERRIS_LAUNCH_CHECK();
}
