// Attention over the paged cache in 4 bits (its bytes: packed_cache.cuh), on mma.sync, for every geometry.
//
// A query row r of a request and kv head is (query i = r / G, head r % G of the G heads that share the kv head); it sees
// the cached rows max(0, p - window + 1) .. p with p = start + i that have a page.  Eight rows are the columns of the
// MMAs, sixteen cached rows their rows:
//   S^T = K Q^T   per group j of 32 elements:  s[key][q] += scale_j[key] (codes_j[key] . q_j) + least_j[key] sum(q_j)
//   O^T = V^T P^T per group j:                 o[elem][q] += codes_j[elem][key] (p[key][q] scale_j[key]) + least_j[key] p[key][q]
// Codes are whole numbers of four bits and least has eight bits, both exact as bf16, so the only roundings before the
// 32-bit sums are those of the other operand: the queries (exact for bf16 rows, three bf16 parts for 32-bit rows) and
// the weights p and p scale (one bf16 part for bf16 rows, three for 32-bit ones).  Neither keys nor values are ever
// formed in fewer than 32 bits.
#include "packed_cache.cuh"

namespace {

constexpr int KEYS = 16;  // cached rows of a tile
constexpr float LOG2E = 1.4426950408889634f;

struct PackedAttention {
    const void* q;
    void* out;
    int ldq, ldo;
    PackedCache cache;
    const int* tables;
    int width;  // blocks of a request's table
    const int* q_start;
    const int* start_row;
    int seqs, heads, group, window;
    float scale;  // of the scores, times log2(e)
    float* lse;   // log2 of the softmax's sum of every (token, head), or nullptr
    float* parts;  // [split][token][head][D + 2]: unnormalised outputs, maximum, sum
    int splits, tokens;
    float* weights;
    const int* seq_slot;
    long long slot_stride;
    int head_stride, max_rows, add;
    int* status;
};

// The page of a request's row, -1 where it has none.
__device__ __forceinline__ int page_of(const PackedAttention& p, const int* table, int row) {
    const int block = row / p.cache.page_size;
    const int page = block < p.width ? table[block] : -1;
    if (page >= p.cache.pages) {
        ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 83);
        return -1;
    }
    return page;
}

// x in NP bf16 parts whose sum is x to 8 NP bits.
template <int NP>
__device__ __forceinline__ void split_parts(float x, float (&part)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        part[i] = i + 1 < NP ? __bfloat162float(__float2bfloat16_rn(x)) : x;
        x -= part[i];
    }
}

// The eight codes of a key word as four pairs (elements i and i + 4), exact bf16 numbers: 128 + code, minus 128.
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int i) {
    const uint32_t v = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __floats2bfloat162_rn(128.0f, 128.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// What a lane (g = lane / 4, c = lane % 4) holds of eight query rows as the B operand: row g of the tile.
template <typename T, int W, int NP>
struct Queries {
    uint32_t b[W][2][2][NP];   // group, half of the group's word, register
    uint32_t sum[(W + 3) / 4][2];  // the group's sum in three parts (group 4 i + c)

    __device__ __forceinline__ void load(const T* row, int c, bool valid) {
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int e = 32 * j + 8 * c + 2 * t + r;  // pairs (e, e + 4): the order of code_pair
                    float lo[NP], hi[NP];
                    split_parts<NP>(valid ? to_float(row[e]) : 0.0f, lo);
                    split_parts<NP>(valid ? to_float(row[e + 4]) : 0.0f, hi);
#pragma unroll
                    for (int i = 0; i < NP; ++i) b[j][t][r][i] = pack_bf16(lo[i], hi[i]);
                }
#pragma unroll
        for (int i = 0; i < (W + 3) / 4; ++i) {
            float s = 0.0f, part[3];
            if (valid && 4 * i + c < W)
                for (int e = 0; e < 32; ++e) s += to_float(row[32 * (4 * i + c) + e]);
            split_parts<3>(s, part);
            sum[i][0] = pack_bf16(part[0], part[1]);
            sum[i][1] = pack_bf16(part[2], 0.0f);
        }
    }
};

// Codes and scales of the keys of a tile: this lane's rows g and g + 8.
template <int W>
struct Keys {
    uint32_t word[2][W], scale[2][W];

    __device__ __forceinline__ void load(const PackedAttention& p, const int* table, int head, int first, int end, int g, int c) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = first + g + 8 * u;
            const int page = row < end ? page_of(p, table, row) : -1;
            const size_t at = page >= 0 ? p.cache.row(page, head, row % p.cache.page_size) : 0;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                word[u][j] = page >= 0 ? reinterpret_cast<const uint32_t*>(p.cache.k_codes)[at * (4 * W) + c * W + j] : 0u;
                scale[u][j] = page >= 0 ? p.cache.k_scales[at * W + j] : 0u;
            }
        }
    }

    // s[0..3]: (key g, rows 2c and 2c + 1), (key g + 8, the same)
    template <typename T, int NP>
    __device__ __forceinline__ void scores(const Queries<T, W, NP>& q, int c, float (&s)[4]) const {
        s[0] = s[1] = s[2] = s[3] = 0.0f;
#pragma unroll
        for (int i = 0; i < (W + 3) / 4; ++i) {  // least times the sums of the queries' groups
            uint32_t l0 = 0, l1 = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (4 * i + k < W && c == k) {
                    l0 = scale[0][4 * i + k];
                    l1 = scale[1][4 * i + k];
                }
            const uint32_t a0 = __byte_perm(l0, l0, 0x3232), a1 = __byte_perm(l1, l1, 0x3232);
            const uint32_t a[4] = {a0, a1, a0, a1};
            mma_bf16_16816(s, a, q.sum[i][0], q.sum[i][1]);
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t a[4] = {code_pair(word[0][j], 2 * t), code_pair(word[1][j], 2 * t), code_pair(word[0][j], 2 * t + 1),
                                       code_pair(word[1][j], 2 * t + 1)};
#pragma unroll
                for (int i = 0; i < NP; ++i) mma_bf16_16816(d, a, q.b[j][t][0][i], q.b[j][t][1][i]);
            }
            const float s0 = packed_scale(scale[0][j]), s1 = packed_scale(scale[1][j]);
            s[0] = fmaf(s0, d[0], s[0]);
            s[1] = fmaf(s0, d[1], s[1]);
            s[2] = fmaf(s1, d[2], s[2]);
            s[3] = fmaf(s1, d[3], s[3]);
        }
    }
};

// What the eight rows of a tile see: for this lane's two columns 2c and 2c + 1 and for all of them.
struct Rows {
    int low[2], high[2];       // first row seen, one past the last
    int least, most;           // over all rows of the tile: the range to go through
    int all_low, all_high;     // rows that every row of the tile sees

    __device__ __forceinline__ void set(const PackedAttention& p, int first, int count, int start, int limit, int lane) {
        least = 0x7fffffff, most = 0, all_low = 0, all_high = 0x7fffffff;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            int lo = 0, hi = 0;
            if (first + r < count) {
                const int at = start + (first + r) / p.group;
                hi = min(at + 1, limit);
                lo = p.window > 0 ? max(0, at - p.window + 1) : 0;
                if (hi > lo) {
                    least = min(least, lo);
                    most = max(most, hi);
                }
                all_low = max(all_low, lo);
                all_high = min(all_high, hi);
            }
            if (r == 2 * (lane & 3)) low[0] = lo, high[0] = hi;
            if (r == 2 * (lane & 3) + 1) low[1] = lo, high[1] = hi;
        }
        if (least > most) least = most;
    }
};

constexpr int WARPS = 8;

// Block (row tile, kv head, request x split): WARPS warps take the tiles of the block's range of cached rows in turn,
// each with its own running maximum and sum, and are joined in shared memory in their order.
template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32) packed_attention_rows_kernel(const PackedAttention p) {
    constexpr int W = D / 32, NP = sizeof(T) == 4 ? 3 : 1;
    extern __shared__ float joined[];  // [WARPS][8][D + 2]
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int head = blockIdx.y, seq = blockIdx.z / p.splits, split = blockIdx.z % p.splits;
    const int t0 = max(p.q_start[seq], 0), count = (min(p.q_start[seq + 1], p.tokens) - t0) * p.group, first = blockIdx.x * 8;
    if (first >= count) return;
    const int* table = p.tables + (size_t)seq * p.width;
    Rows rows;
    rows.set(p, first, count, p.start_row[seq], p.width * p.cache.page_size, lane);
    const int tiles = (rows.most - rows.least / KEYS * KEYS + KEYS - 1) / KEYS, per = (tiles + p.splits - 1) / p.splits;
    const int base = rows.least / KEYS * KEYS + split * per * KEYS, end = min(rows.most, base + per * KEYS);

    Queries<T, W, NP> q;
    {
        const int r = first + g;
        const T* row = (const T*)p.q + (size_t)(t0 + r / p.group) * p.ldq + (size_t)(head * p.group + r % p.group) * D;
        q.load(row, c, r < count);
    }
    float o[W][2][4] = {}, low_o[4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    uint32_t bad = 0;  // groups whose output is not finite: bit j of column 2c, bit j + 8 of column 2c + 1

    for (int at = base + warp * KEYS; at < end; at += WARPS * KEYS) {
        Keys<W> k;
        k.load(p, table, head, at, end, g, c);
        float s[4];
        k.template scores<T, NP>(q, c, s);
        const bool whole = at >= rows.all_low && at + KEYS <= rows.all_high;
        bool seen[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = at + g + 8 * (i >> 1);
            seen[i] = whole || (row >= rows.low[i & 1] && row < rows.high[i & 1]);
            s[i] *= p.scale;
        }
        // rows without a page are seen by nobody
        bool hole = false;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = at + g + 8 * u;
            if (row < end && page_of(p, table, row) < 0) {
                hole = true;
                seen[2 * u] = seen[2 * u + 1] = false;
            }
        }
        const bool masked = __any_sync(0xffffffffu, hole) || !whole;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = seen[i] ? s[i] : -INFINITY;
        float pr[4], rescale[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float top = fmaxf(s[u], s[u + 2]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float now = fmaxf(m[u], top), from = now == -INFINITY ? 0.0f : now;
            rescale[u] = exp2f(m[u] - from);
            m[u] = now;
            pr[u] = seen[u] ? exp2f(s[u] - from) : 0.0f;
            pr[u + 2] = seen[u + 2] ? exp2f(s[u + 2] - from) : 0.0f;
            l[u] = fmaf(l[u], rescale[u], pr[u] + pr[u + 2]);
        }
        // values: this lane's rows (keys) 2c, 2c + 1, 2c + 8, 2c + 9 and, for the scales, g and g + 8
        uint32_t vword[4][(W + 1) / 2], vleast[4], vs[2][W];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int row = at + 2 * c + (u & 1) + 8 * (u >> 1);
            const int page = row < end ? page_of(p, table, row) : -1;
            const size_t r = page >= 0 ? p.cache.row(page, head, row % p.cache.page_size) : 0;
            const uint16_t* src = reinterpret_cast<const uint16_t*>(p.cache.v_codes) + r * (8 * W) + g * W;
#pragma unroll
            for (int j = 0; j < (W + 1) / 2; ++j) {
                uint32_t w = 0;
                if (page >= 0) {
                    w = src[2 * j];
                    if (2 * j + 1 < W) w |= (uint32_t)src[2 * j + 1] << 16;
                }
                vword[u][j] = w;
            }
            vleast[u] = page >= 0 && g < W ? p.cache.v_scales[r * W + g] : 0u;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = at + g + 8 * u;
            const int page = row < end ? page_of(p, table, row) : -1;
            const size_t r = page >= 0 ? p.cache.row(page, head, row % p.cache.page_size) : 0;
#pragma unroll
            for (int j = 0; j < W; ++j) vs[u][j] = page >= 0 ? p.cache.v_scales[r * W + j] : 0u;
        }
        if (masked) {
            // A weight of nought would still carry NaN from a row that the query does not see: groups that are not finite
            // are taken out of the tile, and those outputs that do see them are marked.
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (packed_not_finite(vs[u][j])) {
                        vs[u][j] = 0;
                        bad |= (seen[2 * u] ? 1u << j : 0u) | (seen[2 * u + 1] ? 1u << (j + 8) : 0u);
                    }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (packed_not_finite(vleast[u])) vleast[u] = 0;
        }
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[j][t][i] *= rescale[i & 1];
        low_o[0] *= rescale[0];
        low_o[1] *= rescale[1];
        {  // least times the weights: rows of the product are the groups
            const uint32_t a[4] = {g < W ? __byte_perm(vleast[0], vleast[1], 0x7632) : 0u, 0u, g < W ? __byte_perm(vleast[2], vleast[3], 0x7632) : 0u, 0u};
            float part[4][NP];
#pragma unroll
            for (int i = 0; i < 4; ++i) split_parts<NP>(pr[i], part[i]);
#pragma unroll
            for (int i = 0; i < NP; ++i)
                mma_bf16_16816(low_o, a, movmatrix_trans(pack_bf16(part[0][i], part[1][i])), movmatrix_trans(pack_bf16(part[2][i], part[3][i])));
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const float s0 = packed_scale(vs[0][j]), s1 = packed_scale(vs[1][j]);
            float part[4][NP];
            split_parts<NP>(pr[0] * s0, part[0]);
            split_parts<NP>(pr[1] * s0, part[1]);
            split_parts<NP>(pr[2] * s1, part[2]);
            split_parts<NP>(pr[3] * s1, part[3]);
            const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
            const uint32_t x0 = __byte_perm(vword[0][j / 2], vword[1][j / 2], sel), x1 = __byte_perm(vword[2][j / 2], vword[3][j / 2], sel);
            uint32_t a[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                a[t][0] = code_pair(x0, 2 * t);
                a[t][1] = code_pair(x0, 2 * t + 1);
                a[t][2] = code_pair(x1, 2 * t);
                a[t][3] = code_pair(x1, 2 * t + 1);
            }
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const uint32_t b0 = movmatrix_trans(pack_bf16(part[0][i], part[1][i])), b1 = movmatrix_trans(pack_bf16(part[2][i], part[3][i]));
                mma_bf16_16816(o[j][0], a[0], b0, b1);
                mma_bf16_16816(o[j][1], a[1], b0, b1);
            }
        }
    }

    // over the eight lanes of a column: the sum, the groups that are not finite; then the warp's part in shared memory
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
        l[0] += __shfl_xor_sync(0xffffffffu, l[0], x);
        l[1] += __shfl_xor_sync(0xffffffffu, l[1], x);
        bad |= __shfl_xor_sync(0xffffffffu, bad, x);
    }
    float* mine = joined + (size_t)warp * 8 * (D + 2);
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const float low0 = __shfl_sync(0xffffffffu, low_o[0], 4 * j + c), low1 = __shfl_sync(0xffffffffu, low_o[1], 4 * j + c);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool nan = bad >> (j + 8 * (i & 1)) & 1;
                mine[(2 * c + (i & 1)) * (D + 2) + 32 * j + 4 * g + 2 * t + (i >> 1)] = nan ? NAN : o[j][t][i] + (i & 1 ? low1 : low0);
            }
    }
    if (g == 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            mine[(2 * c + u) * (D + 2) + D] = m[u];
            mine[(2 * c + u) * (D + 2) + D + 1] = l[u];
        }
    }
    __syncthreads();
    const int r = first + warp;  // a warp joins one row
    if (r >= count) return;
    const int token = t0 + r / p.group, qh = head * p.group + r % p.group;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, joined[(w * 8 + warp) * (D + 2) + D]);
    const float from = top == -INFINITY ? 0.0f : top;
    float f[WARPS];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        f[w] = exp2f(joined[(w * 8 + warp) * (D + 2) + D] - from);
        sum += f[w] * joined[(w * 8 + warp) * (D + 2) + D + 1];
    }
    const bool partial = p.splits > 1;
    float* part = partial ? p.parts + (((size_t)split * p.tokens + token) * p.heads + qh) * (D + 2) : nullptr;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int j = 0; j < W; ++j) {
        float acc = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) acc += f[w] * joined[(w * 8 + warp) * (D + 2) + 32 * j + lane];
        if (partial)
            part[32 * j + lane] = acc;
        else
            ((T*)p.out)[(size_t)token * p.ldo + (size_t)qh * D + 32 * j + lane] = from_float<T>(acc * inv);
    }
    if (lane == 0) {
        if (partial) {
            part[D] = top;
            part[D + 1] = sum;
        } else if (p.lse) {
            p.lse[(size_t)token * p.heads + qh] = sum == 0.0f ? INFINITY : from + log2f(sum);
        }
    }
}

// A warp joins the splits of one (token, head) in their order.
template <typename T, int D>
__global__ void __launch_bounds__(256) packed_attention_join_kernel(const PackedAttention p) {
    constexpr int W = D / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= (long long)p.tokens * p.heads || i < (long long)p.q_start[0] * p.heads || i >= (long long)p.q_start[p.seqs] * p.heads) return;
    const float* part = p.parts + (size_t)i * (D + 2);
    const size_t stride = (size_t)p.tokens * p.heads * (D + 2);
    float top = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, part[s * stride + D]);
    top = warp_max(top);
    const float from = top == -INFINITY ? 0.0f : top;
    float acc[W] = {}, sum = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
        const float f = exp2f(part[s * stride + D] - from);
        sum += f * part[s * stride + D + 1];
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] += f * part[s * stride + 32 * j + lane];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int token = (int)(i / p.heads), qh = (int)(i % p.heads);
#pragma unroll
    for (int j = 0; j < W; ++j)
        ((T*)p.out)[(size_t)token * p.ldo + (size_t)qh * D + 32 * j + lane] = from_float<T>(acc[j] * inv);
    if (lane == 0 && p.lse) p.lse[i] = sum == 0.0f ? INFINITY : from + log2f(sum);
}

// Weights of the cached rows:  w[key] (+)= sum over the request's queries and the kv head's query heads of
// exp2(s - lse), a warp sixteen rows of the cache, the query rows in their order.
template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32) packed_attention_weights_kernel(const PackedAttention p) {
    constexpr int W = D / 32, NP = sizeof(T) == 4 ? 3 : 1;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int head = blockIdx.y, seq = blockIdx.z, at = (blockIdx.x * WARPS + warp) * KEYS;
    const int t0 = max(p.q_start[seq], 0), n = min(p.q_start[seq + 1], p.tokens) - t0, count = n * p.group, start = p.start_row[seq];
    const int limit = p.width * p.cache.page_size, end = min(min(start + n, limit), p.max_rows);
    if (at >= end) return;
    const int* table = p.tables + (size_t)seq * p.width;
    Keys<W> k;
    k.load(p, table, head, at, end, g, c);
    bool page[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) page[u] = at + g + 8 * u < end && page_of(p, table, at + g + 8 * u) >= 0;
    float total[2] = {0.0f, 0.0f};
    // the first query row that sees the tile's first cached row
    const int from_row = max(0, at - start) * p.group / 8 * 8;
    for (int first = from_row; first < count; first += 8) {
        Rows rows;
        rows.set(p, first, count, start, limit, lane);
        if (rows.least >= at + KEYS) break;  // with a window: this and all later rows have passed the tile
        if (rows.most <= at) continue;
        Queries<T, W, NP> q;
        const int r = first + g;
        q.load((const T*)p.q + (size_t)(t0 + r / p.group) * p.ldq + (size_t)(head * p.group + r % p.group) * D, c, r < count);
        float s[4];
        k.template scores<T, NP>(q, c, s);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int col = first + 2 * c + u;
            const float lse = col < count ? p.lse[(size_t)(t0 + col / p.group) * p.heads + head * p.group + col % p.group] : INFINITY;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int row = at + g + 8 * x;
                if (page[x] && row >= rows.low[u] && row < rows.high[u]) total[x] += exp2f(s[u + 2 * x] * p.scale - lse);
            }
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        total[x] += __shfl_xor_sync(0xffffffffu, total[x], 1);
        total[x] += __shfl_xor_sync(0xffffffffu, total[x], 2);
    }
    if (c == 0) {
        float* w = p.weights + (long long)(p.seq_slot ? p.seq_slot[seq] : seq) * p.slot_stride + (long long)head * p.head_stride;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int row = at + g + 8 * x;
            if (row < end) w[row] = p.add && row < start ? w[row] + total[x] : total[x];
        }
    }
}

template <typename T, int D>
int attend(const PackedAttention& p, int max_q, int max_kv, cudaStream_t st) {
    const int row_tiles = (max_q * p.group + 7) / 8;
    const size_t smem = (size_t)WARPS * 8 * (D + 2) * sizeof(float);
    if (const int e = ferris_allow_dynamic_smem((const void*)packed_attention_rows_kernel<T, D>, smem)) return e;
    cudaError_t e = ferris_launch(packed_attention_rows_kernel<T, D>, dim3(row_tiles, p.cache.kv_heads, p.seqs * p.splits), dim3(WARPS * 32), smem,
                                  st, p);
    if (e == cudaSuccess && p.splits > 1)
        e = ferris_launch(packed_attention_join_kernel<T, D>, dim3((unsigned)(((long long)p.tokens * p.heads + 7) / 8)), dim3(256), 0, st, p);
    if (e == cudaSuccess && p.weights)
        e = ferris_launch(packed_attention_weights_kernel<T, D>, dim3((max_kv + WARPS * KEYS - 1) / (WARPS * KEYS), p.cache.kv_heads, p.seqs),
                          dim3(WARPS * 32), 0, st, p);
    FERRIS_LAUNCH_CHECK();
}

template <typename T>
int attend_dim(const PackedAttention& p, int max_q, int max_kv, cudaStream_t st) {
    switch (p.cache.head_dim) {
        case 32: return attend<T, 32>(p, max_q, max_kv, st);
        case 64: return attend<T, 64>(p, max_q, max_kv, st);
        case 96: return attend<T, 96>(p, max_q, max_kv, st);
        case 128: return attend<T, 128>(p, max_q, max_kv, st);
        case 160: return attend<T, 160>(p, max_q, max_kv, st);
        case 192: return attend<T, 192>(p, max_q, max_kv, st);
        case 224: return attend<T, 224>(p, max_q, max_kv, st);
        case 256: return attend<T, 256>(p, max_q, max_kv, st);
    }
    FERRIS_REFUSE("packed attention: heads of %d elements", p.cache.head_dim);
}

}  // namespace

// Into how many ranges the cached rows of a step are cut: enough blocks for two to an SM, at least eight tiles of sixteen a warp.
FERRIS_API int ferris_packed_attention_splits(int seqs, int kv_heads, int group, int max_q, int max_kv) {
    const int sms = ferris_sm_count() > 0 ? ferris_sm_count() : 148;
    const long long blocks = (long long)seqs * kv_heads * ((max_q * group + 7) / 8);
    long long want = blocks > 0 ? 2 * sms / blocks : 1, most = max_kv / (WARPS * KEYS * 2);
    if (want > most) want = most;
    if (want > 65535 / (seqs > 0 ? seqs : 1)) want = 65535 / (seqs > 0 ? seqs : 1);
    return want < 1 ? 1 : (int)want;
}

FERRIS_API int ferris_packed_attention(const void* q, int ldq, void* out, int ldo, int dtype, void* k_codes, void* k_scales, void* v_codes,
                                       void* v_scales, int pages, int kv_heads, int page_size, int head_dim, const int* tables, int width,
                                       const int* q_start, const int* start_row, int seqs, int tokens, int heads, int max_q, int max_kv,
                                       int window, float scale, float* lse, float* parts, int splits, float* weights, const int* seq_slot,
                                       long long slot_stride, int head_stride, int max_rows, int add, void* stream) {
    PackedAttention p = {};
    p.cache = {(uint8_t*)k_codes, (uint32_t*)k_scales, (uint8_t*)v_codes, (uint32_t*)v_scales, pages, kv_heads, page_size, head_dim};
    if (const char* why = packed_cache_refusal(p.cache)) FERRIS_REFUSE("%s", why);
    if (heads <= 0 || heads % kv_heads) FERRIS_REFUSE("packed attention: %d heads over %d kv heads", heads, kv_heads);
    if (window < 0 || width <= 0 || splits <= 0) FERRIS_REFUSE("packed attention: window %d, %d blocks, %d splits", window, width, splits);
    if (splits > 1 && !parts) FERRIS_REFUSE("packed attention: %d splits without scratch", splits);
    if (weights && !lse) FERRIS_REFUSE("packed attention: weights without scratch");
    if (seqs <= 0 || tokens <= 0 || max_q <= 0) return FERRIS_OK;
    if ((long long)seqs * splits > 65535 || kv_heads > 65535) FERRIS_REFUSE("packed attention: %d requests, %d splits", seqs, splits);
    if ((long long)width * page_size > 0x7fffffff - 2 * KEYS) FERRIS_REFUSE("packed attention: %d blocks of %d rows", width, page_size);
    p.q = q, p.out = out, p.ldq = ldq, p.ldo = ldo;
    p.tables = tables, p.width = width, p.q_start = q_start, p.start_row = start_row;
    p.seqs = seqs, p.heads = heads, p.group = heads / kv_heads, p.window = window, p.scale = scale * LOG2E;
    p.lse = lse, p.parts = parts, p.splits = splits, p.tokens = tokens;
    p.weights = weights, p.seq_slot = seq_slot, p.slot_stride = slot_stride, p.head_stride = head_stride, p.max_rows = max_rows, p.add = add;
    p.status = ferris_status_ptr();
    if (dtype == FERRIS_BF16) return attend_dim<bf16>(p, max_q, max_kv, (cudaStream_t)stream);
    if (dtype == FERRIS_F32) return attend_dim<float>(p, max_q, max_kv, (cudaStream_t)stream);
    FERRIS_REFUSE("packed attention: dtype %d is not known", dtype);
}
