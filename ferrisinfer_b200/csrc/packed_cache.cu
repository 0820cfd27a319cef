// Writing, reading and evicting rows of the paged cache in 4 bits (its bytes: packed_cache.cuh).
#include <type_traits>

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

// Minimum and maximum that NaN goes through.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The codes of this lane's 8 elements (element i in bits 4 i) and the group's word of scales; all 32 lanes take part.
//
// code = round(d / scale) to even, d = x - least, without sixteen divisions a thread: q = d (1 / scale) is off by an ulp or two, its
// rounding c (by adding 1.5 x 2^23, whose last bits it then is) at most by one, and that only beside a tie; the rest
// d - c scale, exact in one multiply-add (c scale has 12 bits, the rest no more than d), says which way, and whether it IS a tie.
__device__ __forceinline__ uint32_t quantise8(const Eight& e, uint32_t& scales) {
    float low = e.x[0], high = e.x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        low = min_nan(low, e.x[i]);
        high = max_nan(high, e.x[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    const bf16 least_h = __float2bfloat16_rd(low);
    const float least = __bfloat162float(least_h);
    const bf16 scale_h = __float2bfloat16_rn(__fdiv_rn(high - least, 15.0f));
    const float scale = __bfloat162float(scale_h);
    if (!isfinite(least) || !isfinite(scale)) {  // (NaN and infinities show in one of them)
        scales = 0x7fc07fc0u;
        return 0;
    }
    scales = (uint32_t)__bfloat16_as_ushort(scale_h) | (uint32_t)__bfloat16_as_ushort(least_h) << 16;
    uint32_t codes = 0;
    if (scale >= 0x1p-100f) {
        const float inv = __fdiv_rn(1.0f, scale), half = 0.5f * scale;
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            const float d = e.x[i] - least, t = fmaf(d, inv, 12582912.0f), rest = fmaf(-(t - 12582912.0f), scale, d);
            int code = __float_as_int(t) & 31;
            if (fabsf(rest) > half || (fabsf(rest) == half && (code & 1))) code += rest > 0.0f ? 1 : -1;
            codes = codes << 4 | (uint32_t)min(code, 15);
        }
    } else if (scale > 0.0f) {  // (1 / scale may be no number)
#pragma unroll 1
        for (int i = 7; i >= 0; --i) codes = codes << 4 | (uint32_t)fminf(rintf(__fdiv_rn(e.x[i] - least, scale)), 15.0f);
    }
    return codes;
}

// Where a thread of a call over rows (token, head) stands: elements 8 (4 j + c) .. + 7 of them.
struct RowsCall {
    const int* slots;
    PackedCache cache;
    int tokens, ldk, ldv;
    DivideBy heads, page;
    int* status;

    // The row of the cache that row i of the call names: whether there is one.
    __device__ __forceinline__ bool find(uint32_t i, int& token, int& head, size_t& row, int where) const {
        token = (int)heads.quotient(i);
        head = (int)i - token * cache.kv_heads;
        const int slot = slots[token], page_at = slot >= 0 ? (int)page.quotient((uint32_t)slot) : -1;
        if (page_at >= cache.pages) ferris_report(status, FERRIS_STATUS_BAD_INDEX, where);
        if (page_at < 0 || page_at >= cache.pages) return false;
        row = cache.row(page_at, head, slot - page_at * cache.page_size);
        return true;
    }
};

// Bound by its instructions for many tokens (8,192 tokens of 4 heads of 128: 13.5 us, 1.6 TB/s; 21 us with a division for each
// element), by its launch for a step's (3.1 us): 16-byte loads of a head's elements, lanes side by side; the divisions by
// heads and page size are multiplications (here and in the read, written and read back 28.8 -> 24.8 us against 64-bit divisions).
template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(256) packed_write_kernel(const T* k, const T* v, const RowsCall q) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr uint32_t LANES = 4 * W;  // of a row
    const uint32_t all = (uint32_t)q.tokens * q.cache.kv_heads * LANES;  // (the C entry sees to 32 bits)
    for (uint32_t at = blockIdx.x * 256 + threadIdx.x; (at & ~31u) < all; at += gridDim.x * 256) {  // whole warps: the lanes of a group meet in shuffles
        const uint32_t i = at / LANES, r = at % LANES, c = r & 3, j = r >> 2;
        int token, head;
        size_t row;
        const bool store = at < all && q.find(i, token, head, row, 80);
        Eight ek = {}, ev = {};
        if (store) {
            const size_t col = (size_t)head * (32 * W) + 32 * j + 8 * c;
            ek = load8<T, VEC>(k + (size_t)token * q.ldk + col);
            ev = load8<T, VEC>(v + (size_t)token * q.ldv + col);
        }
        uint32_t ks, vs;
        const uint32_t kc = quantise8(ek, ks), vc = quantise8(ev, vs);
        if (store) {
            reinterpret_cast<uint32_t*>(q.cache.k_codes)[row * (4 * W) + c * W + j] = kc;
            uint16_t* vd = reinterpret_cast<uint16_t*>(q.cache.v_codes) + row * (8 * W);
            vd[(2 * c) * W + j] = (uint16_t)vc;
            vd[(2 * c + 1) * W + j] = (uint16_t)(vc >> 16);
            if (c == 0) {
                q.cache.k_scales[row * W + j] = ks;
                q.cache.v_scales[row * W + j] = vs;
            }
        }
    }
}

// read: out[t] = the values that the row at slots[t] stands for, rounded once (zeros for slots below 0).  Bound by memory for many
// tokens: 65,536 of 4 heads of 128 40 us (4.4 TB/s), 8,192 6.5 us (3.4 TB/s).
__device__ __forceinline__ Eight dequantise8(uint32_t codes, uint32_t scales) {
    const float scale = packed_scale(scales), least = packed_least(scales);
    Eight e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e.x[i] = fmaf((float)((codes >> (4 * i)) & 15), scale, least);
    return e;
}

constexpr int READ_EACH = 4;

template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(256) packed_read_kernel(T* k, T* v, const RowsCall q) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr uint32_t LANES = 4 * W;
    constexpr int EACH = READ_EACH;  // rows of a thread, fetched together
    const uint32_t rows = (uint32_t)q.tokens * q.cache.kv_heads, threads = gridDim.x * 256, first = blockIdx.x * 256 + threadIdx.x;
    {
        uint32_t kc[EACH], vc[EACH], ks[EACH], vs[EACH];
        int token[EACH], head[EACH];
#pragma unroll
        for (int x = 0; x < EACH; ++x) {
            const uint32_t at = first + x * threads, i = at / LANES, r = at % LANES, c = r & 3, j = r >> 2;
            kc[x] = vc[x] = ks[x] = vs[x] = 0;
            token[x] = -1;
            size_t row;
            if (at < rows * LANES && q.find(i, token[x], head[x], row, 81)) {
                const uint16_t* src = reinterpret_cast<const uint16_t*>(q.cache.v_codes) + row * (8 * W);
                kc[x] = reinterpret_cast<const uint32_t*>(q.cache.k_codes)[row * (4 * W) + c * W + j];
                vc[x] = (uint32_t)src[(2 * c) * W + j] | (uint32_t)src[(2 * c + 1) * W + j] << 16;
                ks[x] = q.cache.k_scales[row * W + j];
                vs[x] = q.cache.v_scales[row * W + j];
            }
        }
#pragma unroll
        for (int x = 0; x < EACH; ++x) {
            if (token[x] < 0) continue;
            const uint32_t r = (first + x * threads) % LANES;
            const size_t at = (size_t)head[x] * (32 * W) + 8 * (4 * (r >> 2) + (r & 3));
            store8<T, VEC>(k + (size_t)token[x] * q.ldk + at, dequantise8(kc[x], ks[x]));
            store8<T, VEC>(v + (size_t)token[x] * q.ldv + at, dequantise8(vc[x], vs[x]));
        }
    }
}

// ---------------------------------------------------------------------------------------------
// evict: of the n rows of a request and kv head, `budget` stay: the first `keep_first`, the last
// `keep_last`, and of the others those of the greatest weight, the lower row first among equals.
// A row that has no page is not there and never stays.
// The order of floats as unsigned keys; NaN counts as greater than every number, -0 as 0; no row's key is 0.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t weight_key(float w, int row, int n, int keep_first, int keep_last) {
    if (row < keep_first || row >= n - keep_last) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int EVICT_THREADS = 512, EVICT_WARPS = EVICT_THREADS / 32;
constexpr int EVICT_HELD = 48 * 1024;  // rows whose keys a block's shared memory holds
constexpr int EVICT_COPIES = 4;        // of a histogram: lanes that meet in a bin wait for one another

// A cluster of blocks per (request, kv head), each with a run of its rows, whose keys it holds in shared memory (longer runs are
// read again each time).  The budget-th greatest key by its four bytes, most significant first: a histogram of 256 bins
// each, added up over the cluster; then the kept rows in order, every warp its own run of rows.  What bounds it is the
// chain of short passes and barriers, so a lane takes four rows at a time, each on its own.  16 requests of up to 32,768 rows and
// 4 heads: 29 us (keys formed one after the other, 34; besides one row at a time, lanes that share a bin found by votes, 44 to 47;
// all of the eviction with the read-back was no faster with `match.any`); 5,000 rows of one request 15 us.
__global__ void __launch_bounds__(EVICT_THREADS) packed_evict_select_kernel(const float* weights, long long slot_stride, int head_stride,
                                                                            const int* __restrict__ seq_rows, const int* __restrict__ seq_slot,
                                                                            int* kept_rows, float* kept_weights, long long kept_slot_stride,
                                                                            int kept_head_stride, int budget, int keep_first, int keep_last,
                                                                            int max_rows, int held, int slots, const int* __restrict__ tables,
                                                                            int width, DivideBy page, int page_size, int pages, int* status) {
    extern __shared__ __align__(16) uint32_t keys[];  // [held], read four at a time
    __shared__ uint32_t hist[4][EVICT_COPIES][256], total[256];
    __shared__ int greater[EVICT_WARPS], equal[EVICT_WARPS], has_page[EVICT_WARPS], counts[2];
    const int s = blockIdx.y, h = blockIdx.x, heads = gridDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = gridDim.z, rank = blockIdx.z;
    const int slot = seq_slot ? seq_slot[s] : s;
    if (slot >= slots) ferris_report(status, FERRIS_STATUS_BAD_INDEX, 105);
    if (slot >= 0 && seq_rows[s] > max_rows) ferris_report(status, FERRIS_STATUS_BAD_INDEX, 107);  // (rows that no weight speaks for)
    const int n = slot < 0 || slot >= slots ? 0 : min(max(seq_rows[s], 0), max_rows);  // (without weights: no rows; nothing of w is then read)
    const float* w = weights + slot * slot_stride + (long long)h * head_stride;
    int* rows = kept_rows + ((size_t)s * heads + h) * budget;
    float* kw = kept_weights ? kept_weights + slot * kept_slot_stride + (long long)h * kept_head_stride : nullptr;
    // this block's rows: runs of whole 32 rows for each of its warps
    const int run = (n + 32 * EVICT_WARPS * blocks - 1) / (32 * EVICT_WARPS * blocks) * 32, begin = min(rank * EVICT_WARPS * run, n),
              end = min(begin + EVICT_WARPS * run, n);
    const bool hold = end - begin <= held;
    for (int i = tid; i < 4 * EVICT_COPIES * 256; i += EVICT_THREADS) (&hist[0][0][0])[i] = 0;
    const int* table = tables + (size_t)s * width;
    const int all = n > 0 ? (int)page.quotient(n - 1) + 1 : 0, first_page = tid < min(all, width) ? table[tid] : -1;
    if (hold && n > budget)  // (as if all rows were there: which are is counted meanwhile)
        for (int r0 = begin + tid; r0 < (end + 3) / 4 * 4; r0 += 8 * EVICT_THREADS) {
            float v[8];  // all on their way before the first is used
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = r0 + i * EVICT_THREADS < end ? w[r0 + i * EVICT_THREADS] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = r0 + i * EVICT_THREADS;
                if (r < (end + 3) / 4 * 4) keys[r - begin] = r < end ? weight_key(v[i], r, n, keep_first, keep_last) : 0u;
            }
        }
    // the rows that have a page (every block counts all of them)
    int there = 0;
    for (int b = tid; b < all; b += EVICT_THREADS) {
        const int at = b == tid ? first_page : b < width ? table[b] : -1;
        if (at >= pages) ferris_report(status, FERRIS_STATUS_BAD_INDEX, 106);
        if (at >= 0 && at < pages) there += min(page_size, n - b * page_size);
    }
    there = __reduce_add_sync(0xffffffffu, there);
    if (lane == 0) has_page[warp] = there;
    __syncthreads();
    there = __reduce_add_sync(0xffffffffu, lane < EVICT_WARPS ? has_page[lane] : 0);
    const bool whole = there == n;
    const auto is_there = [&](int r) {
        const int b = (int)page.quotient(r);
        return whole || (b < width && table[b] >= 0 && table[b] < pages);
    };
    const int stay = min(there, budget);
    for (int i = stay + rank * EVICT_THREADS + tid; i < budget; i += blocks * EVICT_THREADS) rows[i] = -1;
    if (whole && n <= budget) {  // (the whole cluster)
        for (int i = rank * EVICT_THREADS + tid; i < n; i += blocks * EVICT_THREADS) {
            rows[i] = i;
            if (kw) kw[i] = w[i];
        }
        return;
    }
    if (hold && !whole) {
        for (int r = begin + tid; r < (end + 3) / 4 * 4; r += EVICT_THREADS)
            keys[r - begin] = r < end && is_there(r) ? weight_key(w[r], r, n, keep_first, keep_last) : 0u;
        __syncthreads();
    }
    // keys of four rows from r (a multiple of four) on; 0 for rows that are not there, and behind the end
    const auto keys_of = [&](int r) {
        if (hold) return *reinterpret_cast<const uint4*>(keys + (r - begin));
        uint32_t k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = r + i < end && is_there(r + i) ? weight_key(w[r + i], r + i, n, keep_first, keep_last) : 0u;
        return make_uint4(k[0], k[1], k[2], k[3]);
    };
    uint32_t prefix = 0;
    int want = there > budget ? budget : 0;  // how many of the rows that share the prefix stay (0: all that have a key do)
#pragma unroll 1
    for (int byte = 0; byte < 4 && there > budget; ++byte) {
        const int shift = 24 - 8 * byte;
        const uint32_t mask = byte == 0 ? 0u : 0xffffffffu << (shift + 8);
        uint32_t* mine_of = hist[byte][lane % EVICT_COPIES];
#pragma unroll 2
        for (int r = begin + 4 * tid; r < end; r += 4 * EVICT_THREADS) {
            const uint4 k = keys_of(r);
            const uint32_t four[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (four[i] && (four[i] & mask) == prefix) atomicAdd(&mine_of[(four[i] >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid < 256) {
            uint32_t sum = 0;
#pragma unroll
            for (int x = 0; x < EVICT_COPIES; ++x) sum += hist[byte][x][tid];
            if (blocks > 1)
                hist[byte][0][tid] = sum;
            else
                total[tid] = sum;
        }
        if (blocks > 1) {
            cluster_sync();
            if (tid < 256) {
                uint32_t sum = 0;
                for (int b = 0; b < blocks; ++b) sum += __float_as_uint(ld_peer_shared_f32(smem_u32(&hist[byte][0][tid]), b));
                total[tid] = sum;
            }
        }
        __syncthreads();
        // every warp finds the bin for itself: eight bins a lane, from the greatest down
        uint32_t mine[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            mine[i] = total[255 - 8 * lane - i];
            sum += mine[i];
        }
        uint32_t upto = sum;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, x);
            if (lane >= x) upto += v;
        }
        const int owner = __ffs(__ballot_sync(0xffffffffu, upto >= (uint32_t)want)) - 1;
        uint32_t before = upto - sum;
        int bin = 0, left = want;
        bool found = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!found && before + mine[i] >= (uint32_t)want) {
                found = true;
                bin = 255 - 8 * lane - i;
                left = want - (int)before;
            }
            before += mine[i];
        }
        prefix |= (uint32_t)__shfl_sync(0xffffffffu, bin, owner) << shift;
        want = __shfl_sync(0xffffffffu, left, owner);
        __syncthreads();  // (`total` is read no more)
    }
    // rows with key > prefix all stay, of those with key == prefix the first `want`
    const int from = min(begin + warp * run, end), to = min(from + run, end);
    int gt = 0, eq = 0;
    for (int r = from + 4 * lane; r < to; r += 128) {
        const uint4 k = keys_of(r);
        gt += (k.x > prefix) + (k.y > prefix) + (k.z > prefix) + (k.w > prefix);
        eq += (k.x == prefix) + (k.y == prefix) + (k.z == prefix) + (k.w == prefix);
    }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        greater[warp] = gt;
        equal[warp] = eq;
    }
    __syncthreads();
    int before_gt = lane < warp ? greater[lane] : 0, before_eq = lane < warp ? equal[lane] : 0;  // (lanes below EVICT_WARPS)
    before_gt = __reduce_add_sync(0xffffffffu, before_gt);
    before_eq = __reduce_add_sync(0xffffffffu, before_eq);
    if (blocks > 1) {
        if (warp == EVICT_WARPS - 1 && lane == 0) {
            counts[0] = before_gt + gt;
            counts[1] = before_eq + eq;
        }
        cluster_sync();
        for (int b = 0; b < rank; ++b) {
            before_gt += (int)__float_as_uint(ld_peer_shared_f32(smem_u32(&counts[0]), b));
            before_eq += (int)__float_as_uint(ld_peer_shared_f32(smem_u32(&counts[1]), b));
        }
        cluster_arrive_release();  // (a block's shared memory stays until all have read it)
    }
    for (int r0 = from; r0 < to; r0 += 128) {
        const int r = r0 + 4 * lane;
        const uint4 k = r < to ? keys_of(r) : make_uint4(0, 0, 0, 0);
        const uint32_t four[4] = {k.x, k.y, k.z, k.w};
        int mine = 0;  // those above in the lower half, the equal ones in the upper
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += (four[i] > prefix) + ((four[i] == prefix) << 16);
        int upto = mine;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, x);
            if (lane >= x) upto += v;
        }
        int above = before_gt + ((upto - mine) & 0xffff), same = before_eq + ((upto - mine) >> 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (four[i] > prefix || (four[i] == prefix && same < want)) {
                const int at = above + min(same, want);
                rows[at] = r + i;
                if (kw) kw[at] = w[r + i];
            }
            above += four[i] > prefix;
            same += four[i] == prefix;
        }
        upto = __shfl_sync(0xffffffffu, upto, 31);
        before_gt += upto & 0xffff;
        before_eq += upto >> 16;
    }
    if (blocks > 1) cluster_wait();
}

// Kept rows from their pages into others: every thread 16 bytes of codes of a row's keys and of its values, W threads a row, and the
// rows' scales by the same threads; four rows of a thread are fetched together.  16 requests of 4,096 kept rows, 4 heads of 128: 25 us
// (84 MB read and written, 3.4 TB/s).
template <int W>
__global__ void __launch_bounds__(256) packed_evict_move_kernel(PackedCache from, PackedCache to, const int* __restrict__ from_tables,
                                                                int from_width, const int* __restrict__ to_tables, int to_width,
                                                                const int* kept_rows, int budget, DivideBy from_page, DivideBy to_page, int* status) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int EACH = 4, ROWS = 256 / W;  // rows that a block takes at once
    const int s = blockIdx.z, h = blockIdx.y, heads = gridDim.y, part = threadIdx.x % W;
    const int* kept = kept_rows + ((size_t)s * heads + h) * budget;
    if (threadIdx.x >= ROWS * W) return;
    uint4 kc[EACH], vc[EACH];
    uint32_t ks[EACH], vs[EACH];
    size_t dst[EACH];
    bool live[EACH];
#pragma unroll
    for (int x = 0; x < EACH; ++x) {
        const int at = (blockIdx.x * EACH + x) * ROWS + threadIdx.x / W, row = at < budget ? kept[at] : -1;
        const int sb = row >= 0 ? (int)from_page.quotient(row) : 0, db = (int)to_page.quotient(at);
        live[x] = row >= 0 && sb < from_width && db < to_width;
        const int sp = live[x] ? from_tables[(size_t)s * from_width + sb] : -1, dp = live[x] ? to_tables[(size_t)s * to_width + db] : -1;
        if (sp >= from.pages || dp >= to.pages) ferris_report(status, FERRIS_STATUS_BAD_INDEX, 82);
        live[x] = sp >= 0 && dp >= 0 && sp < from.pages && dp < to.pages;
        if (!live[x]) continue;
        const size_t a = from.row(sp, h, row - sb * from.page_size) * W + part;
        dst[x] = to.row(dp, h, at - db * to.page_size) * W + part;
        kc[x] = reinterpret_cast<const uint4*>(from.k_codes)[a];
        vc[x] = reinterpret_cast<const uint4*>(from.v_codes)[a];
        ks[x] = from.k_scales[a];
        vs[x] = from.v_scales[a];
    }
#pragma unroll
    for (int x = 0; x < EACH; ++x) {
        if (!live[x]) continue;
        reinterpret_cast<uint4*>(to.k_codes)[dst[x]] = kc[x];
        reinterpret_cast<uint4*>(to.v_codes)[dst[x]] = vc[x];
        to.k_scales[dst[x]] = ks[x];
        to.v_scales[dst[x]] = vs[x];
    }
}

PackedCache make_cache(void* kc, void* ks, void* vc, void* vs, int pages, int kv_heads, int page_size, int head_dim) {
    return {(uint8_t*)kc, (uint32_t*)ks, (uint8_t*)vc, (uint32_t*)vs, pages, kv_heads, page_size, head_dim};
}

template <typename T>
bool eights_aligned(const void* p, int ld) {
    return ((uintptr_t)p & 15) == 0 && ld % (16 / (int)sizeof(T)) == 0;
}

int sms() { return ferris_sm_count() > 0 ? ferris_sm_count() : 148; }

template <typename T, int W>
int write_rows(const void* k, const void* v, const RowsCall& q, cudaStream_t st) {
    const bool vec = eights_aligned<T>(k, q.ldk) && eights_aligned<T>(v, q.ldv);
    const long long need = ((long long)q.tokens * q.cache.kv_heads * 4 * W + 255) / 256, most = sms() * 8;
    const int blocks = (int)(need < most ? need : most);
    if (vec)
        ferris_launch(packed_write_kernel<T, W, true>, dim3(blocks), dim3(256), 0, st, (const T*)k, (const T*)v, q);
    else
        ferris_launch(packed_write_kernel<T, W, false>, dim3(blocks), dim3(256), 0, st, (const T*)k, (const T*)v, q);
    FERRIS_LAUNCH_CHECK();
}

template <typename T, int W>
int read_rows(void* k, void* v, const RowsCall& q, cudaStream_t st) {
    const bool vec = eights_aligned<T>(k, q.ldk) && eights_aligned<T>(v, q.ldv);
    const long long all = (long long)q.tokens * q.cache.kv_heads * 4 * W, few = (long long)sms() * 2;
    // a row a thread where that leaves SMs without work
    const int blocks = (int)((all + 255) / 256 <= few ? (all + 255) / 256 : (all + 256 * READ_EACH - 1) / (256 * READ_EACH) > few ? (all + 256 * READ_EACH - 1) / (256 * READ_EACH) : few);
    if (vec)
        ferris_launch(packed_read_kernel<T, W, true>, dim3(blocks), dim3(256), 0, st, (T*)k, (T*)v, q);
    else
        ferris_launch(packed_read_kernel<T, W, false>, dim3(blocks), dim3(256), 0, st, (T*)k, (T*)v, q);
    FERRIS_LAUNCH_CHECK();
}

// f<W>() for heads of 32 W elements.
template <typename F>
int with_groups(int head_dim, F&& f) {
    switch (head_dim / 32) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        case 4: return f(std::integral_constant<int, 4>());
        case 5: return f(std::integral_constant<int, 5>());
        case 6: return f(std::integral_constant<int, 6>());
        case 7: return f(std::integral_constant<int, 7>());
        default: return f(std::integral_constant<int, 8>());
    }
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

namespace {

template <bool WRITE>
int rows_call(const FerrisPackedRows* a) {
    const PackedCache cache = a->cache();
    if (const char* why = packed_cache_refusal(cache)) FERRIS_REFUSE("%s", why);
    if (a->tokens <= 0) return FERRIS_OK;
    if ((long long)a->tokens * a->kv_heads * (a->head_dim / 8) > 0x3fffffffll) FERRIS_REFUSE("packed cache: %d tokens in one call", a->tokens);
    if (a->dtype != FERRIS_BF16 && a->dtype != FERRIS_F32) FERRIS_REFUSE("packed cache: dtype %d is not known", a->dtype);
    const RowsCall q = {a->slots, cache, a->tokens, a->ldk, a->ldv, DivideBy(a->kv_heads), DivideBy(a->page_size), ferris_status_ptr()};
    cudaStream_t st = (cudaStream_t)a->stream;
    return with_groups(a->head_dim, [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (WRITE) return a->dtype == FERRIS_BF16 ? write_rows<bf16, W>(a->k, a->v, q, st) : write_rows<float, W>(a->k, a->v, q, st);
        return a->dtype == FERRIS_BF16 ? read_rows<bf16, W>(a->k, a->v, q, st) : read_rows<float, W>(a->k, a->v, q, st);
    });
}

}  // namespace

FERRIS_API int ferris_packed_cache_write(const FerrisPackedRows* a) { return rows_call<true>(a); }
FERRIS_API int ferris_packed_cache_read(const FerrisPackedRows* a) { return rows_call<false>(a); }

// The arguments of the one below, as its caller lays them out.
struct FerrisPackedEvict {
    void *from_kc, *from_ks, *from_vc, *from_vs, *to_kc, *to_ks, *to_vc, *to_vs;
    const int *from_tables, *to_tables, *seq_rows, *seq_slot;
    const float* weights;
    int* kept_rows;
    float* kept_weights;
    void* stream;
    long long slot_stride, kept_slot_stride;
    int from_pages, from_page_size, to_pages, to_page_size, kv_heads, head_dim, from_width, to_width, head_stride, max_rows, kept_head_stride,
        seqs, budget, keep_first, keep_last, slots;
};

FERRIS_API int ferris_packed_cache_evict(const FerrisPackedEvict* a) {
    const int kv_heads = a->kv_heads, head_dim = a->head_dim, seqs = a->seqs, budget = a->budget, keep_first = a->keep_first, keep_last = a->keep_last,
              max_rows = a->max_rows;
    const PackedCache from = make_cache(a->from_kc, a->from_ks, a->from_vc, a->from_vs, a->from_pages, kv_heads, a->from_page_size, head_dim);
    const PackedCache to = make_cache(a->to_kc, a->to_ks, a->to_vc, a->to_vs, a->to_pages, kv_heads, a->to_page_size, head_dim);
    if (const char* why = packed_cache_refusal(from)) FERRIS_REFUSE("%s", why);
    if (const char* why = packed_cache_refusal(to)) FERRIS_REFUSE("%s", why);
    if (budget <= 0 || keep_first < 0 || keep_last < 0 || keep_first > budget - keep_last)
        FERRIS_REFUSE("eviction: %d first and %d last rows of a budget of %d", keep_first, keep_last, budget);
    if (seqs <= 0) return FERRIS_OK;
    if (seqs > 65535 || kv_heads > 65535) FERRIS_REFUSE("eviction: %d requests of %d kv heads", seqs, kv_heads);
    cudaStream_t st = (cudaStream_t)a->stream;
    // blocks of a cluster: about 8,192 rows each, at most eight (the most that is portable)
    int blocks = 1;
    while (blocks < 8 && (long long)blocks * 8192 < max_rows) blocks *= 2;
    const int each = ((max_rows + EVICT_THREADS * blocks - 1) / (EVICT_THREADS * blocks)) * EVICT_THREADS, held = each < EVICT_HELD ? each : EVICT_HELD;
    if (const int r = ferris_allow_dynamic_smem((const void*)packed_evict_select_kernel, (size_t)held * 4)) return r;
    // In its turn of the stream, and its dependents not before its blocks end: blocks of this kernel beside those of the one in front, or
    // blocks that move rows beside these, cost more than the launch that they hide (16 requests with the read-back 108 us, not 94).
    cudaError_t e = ferris_launch_cluster<false>(packed_evict_select_kernel, dim3(kv_heads, seqs, blocks), dim3(EVICT_THREADS), (size_t)held * 4, st, blocks,
                                          a->weights, a->slot_stride, a->head_stride, a->seq_rows, a->seq_slot, a->kept_rows, a->kept_weights,
                                          a->kept_slot_stride, a->kept_head_stride, budget, keep_first, keep_last, max_rows, held, a->slots,
                                          a->from_tables, a->from_width, DivideBy(a->from_page_size), a->from_page_size, a->from_pages,
                                          ferris_status_ptr());
    if (e != cudaSuccess) FERRIS_LAUNCH_CHECK();
    return with_groups(head_dim, [&](auto w) {
        constexpr int W = decltype(w)::value, ROWS = 256 / W * 4;
        ferris_launch(packed_evict_move_kernel<W>, dim3((budget + ROWS - 1) / ROWS, kv_heads, seqs), dim3(256), 0, st, from, to,
                      a->from_tables, a->from_width, a->to_tables, a->to_width, (const int*)a->kept_rows, budget, DivideBy(a->from_page_size),
                      DivideBy(a->to_page_size), ferris_status_ptr());
        FERRIS_LAUNCH_CHECK();
    });
}
