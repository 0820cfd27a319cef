// Attention for trees of drafted tokens over the paged cache, fp32, on the CUDA cores (who sees what, and how the work is dealt out:
// tree_attention.cuh).
//
// Eight warps share tiles of TILE cached rows, which cp.async brings, one tile ahead.  A warp has eight query rows; GROUPS of warps have the same rows and
// different parts of a tile (few query rows), and are joined at the end.
//   scores   a lane is a cached row (two, of tiles that one group has): a row's four elements meet those of eight query rows, 64 multiply-adds for ten reads of
//            shared memory
//   outputs  a lane is four columns: a cached row's values meet the weights of eight query rows, which are two reads for all lanes
// All in 32 bits.  Whatever a query does not see is never multiplied: what lies there may be NaN.
// What bounds it: six ragged requests of up to 13 nodes after up to 1,533 rows (12 / 2 heads of 128) 34 us.  A tile of 64 cached by 32 query rows takes some 12,000
// cycles, 4,100 if every multiply-add were issued without a pause: with two warps to a scheduler reads of shared memory (nine of 16 bytes a lane for 32
// multiply-adds) and the softmax between the products are waited for.  Blocks of query rows are numbered with the tiles: one block for each of the largest request's
// left those of the others idle (53 us).
#include "tree_attention.cuh"

namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32, WARP_ROWS = 8;

// Heads of up to DP elements, GROUPS groups of warps.
template <int DP, int G>
struct Sizes {
    static constexpr int TILE = DP <= 128 ? 64 : 32, KEYS = TILE / G, EACH = KEYS / 32;  // cached rows of a tile, of a group, of a lane
    static constexpr int ROWS = WARP_ROWS * WARPS / G, LD = DP + 4;                     // query rows of a block; floats of a row: lanes read neighbouring rows
    static constexpr int STAGE = 2 * TILE * LD, WEIGHTS = WARPS * KEYS * WARP_ROWS, QUERIES = ROWS * LD;  // floats
    static constexpr int BYTES = (2 * STAGE + QUERIES + WEIGHTS) * 4;
    static constexpr bool HALVES = DP <= 64;  // half-warps take cached rows in turn, four columns of 64 a lane
    static constexpr int QUADS = DP <= 128 ? 1 : 2;
    static_assert(KEYS % 32 == 0, "a lane a cached row");
    static_assert(WARPS * WARP_ROWS * LD <= 2 * STAGE, "the groups are joined through the tiles' memory");
};

__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

template <int DP, int G>
__global__ void __launch_bounds__(THREADS, 1) tree_attention_f32_kernel(const TreeAttention p) {
    using Z = Sizes<DP, G>;
    constexpr int LD = Z::LD, EACH = Z::EACH;
    extern __shared__ __align__(16) float smem[];
    __shared__ TreeLines tree;
    __shared__ TreeRequests requests;
    __shared__ unsigned long long there[2];  // which of a stage's cached rows have a page
    __shared__ float row_m[WARPS][WARP_ROWS], row_l[WARPS][WARP_ROWS];
    float* qs = smem + 2 * Z::STAGE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.head_dim;
    const int group = warp % G, slab = warp / G;  // which part of a tile; which eight query rows
    float* weights = qs + Z::QUERIES + warp * Z::KEYS * WARP_ROWS;  // [cached row][query row]
    pdl_wait();
    pdl_launch_dependents();
    TreeWalk<Z::TILE, Z::ROWS, true> walk;
    walk.know(p, requests);
    __syncthreads();
    walk.begin(p, requests, blockIdx.x, gridDim.x, 0);
    TreeItem item;
    int4 begun = walk.none();
    while (walk.next(p, requests, item)) {
        const TreeRequest r = item.request;
        const int head = item.head, count = r.nodes * p.group, row0 = item.block * Z::ROWS;
        const int first = item.first, last = item.last, low = item.low;
        const bool whole_item = first == 0 && last == item.tiles;
        walk.note(item, begun);
        const int parent = tree_parent(p, r, threadIdx.x);
        const int* table = p.tables + (size_t)item.seq * p.width;
        // ---- cached rows on their way: a warp takes every eighth of the tile
        auto request = [&](int i) {
            if (i < last) {
                const int s = i & 1, key0 = (low + i) * Z::TILE;
                const uint32_t k_dst = smem_u32(smem + s * Z::STAGE), v_dst = k_dst + Z::TILE * LD * 4;
                constexpr int MINE = Z::TILE / WARPS;
                const int row = key0 + (lane % MINE) * WARPS + warp;  // row lane % MINE of this warp's
                const int page = row < r.rows ? tree_page(p, table, row) : -1;
                const size_t at = page >= 0 ? tree_row_at(p, page, head, row) : 0;
                const uint32_t live = __ballot_sync(0xffffffffu, page >= 0);
#pragma unroll
                for (int j = 0; j < MINE; ++j) {
                    const size_t from = __shfl_sync(0xffffffffu, at, j);
                    const bool ok = live >> j & 1;
                    const uint32_t to = (j * WARPS + warp) * LD * 4;
#pragma unroll
                    for (int c = 0; c < (DP + 127) / 128; ++c) {
                        const int col = c * 128 + lane * 4;
                        if (col < D) {
                            copy_async(k_dst + to + col * 4, (const float*)p.k_cache + from + col, ok);
                            copy_async(v_dst + to + col * 4, (const float*)p.v_cache + from + col, ok);
                        }
                    }
                }
                if (lane == 0) {
                    unsigned long long bits = 0;
#pragma unroll
                    for (int j = 0; j < MINE; ++j) bits |= (unsigned long long)(live >> j & 1) << (j * WARPS + warp);
                    atomicOr(&there[s], bits);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        if (threadIdx.x < 2) there[threadIdx.x] = 0;
        __syncthreads();
        request(first);
        const bool wide = ((uintptr_t)p.q & 15) == 0 && p.ldq % 4 == 0;
#pragma unroll 4
        for (int i = threadIdx.x; i < Z::ROWS * (D / 4); i += THREADS) {
            const int row = i / (D / 4), c = (i - row * (D / 4)) * 4, at = row0 + row;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (at < count) {
                const float* src = (const float*)p.q + (size_t)(r.first + at / p.group) * p.ldq + (head * p.group + at % p.group) * D + c;
                v = wide ? *reinterpret_cast<const float4*>(src) : make_float4(src[0], src[1], src[2], src[3]);
            }
            *reinterpret_cast<float4*>(qs + row * LD + c) = v;
        }
        // (the lines are only looked at where tiles are not seen whole: those of the tree, and with a window)
        if (p.window > 0 || (low + last) * Z::TILE > min(r.start, r.rows)) tree_lines<THREADS>(p, r, tree, parent, [] { __syncthreads(); });
        const int slab0 = row0 + slab * WARP_ROWS;
        const bool live = slab0 < count;
        float m[WARP_ROWS], l[WARP_ROWS];
        float4 o[WARP_ROWS][Z::QUADS];
#pragma unroll
        for (int i = 0; i < WARP_ROWS; ++i) {
            m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < Z::QUADS; ++c) o[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        const int sure_low = p.window > 0 ? max(0, r.start + r.nodes - p.window) : 0, sure_high = min(r.start, r.rows);
        for (int i = first; i < last; ++i) {
            const int s = i & 1;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();
            const unsigned long long pages = there[s];
            if (threadIdx.x == 0) there[s ^ 1] = 0;
            __syncthreads();
            request(i + 1);
            const int key0 = (low + i) * Z::TILE + group * Z::KEYS;
            if (!live || key0 >= r.rows) continue;
            const float* ks = smem + s * Z::STAGE + group * Z::KEYS * LD;
            const float* vs = ks + Z::TILE * LD;
            float x[WARP_ROWS][EACH] = {};
            {
                const float* q = qs + slab * WARP_ROWS * LD;
                const float* k = ks + lane * LD;
#pragma unroll 4
                for (int c = 0; c < D; c += 4) {
                    float4 kv[EACH];
#pragma unroll
                    for (int e = 0; e < EACH; ++e) kv[e] = *reinterpret_cast<const float4*>(k + e * 32 * LD + c);
#pragma unroll
                    for (int j = 0; j < WARP_ROWS; ++j) {
                        const float4 qv = *reinterpret_cast<const float4*>(q + j * LD + c);
#pragma unroll
                        for (int e = 0; e < EACH; ++e)
                            x[j][e] = fmaf(qv.x, kv[e].x, fmaf(qv.y, kv[e].y, fmaf(qv.z, kv[e].z, fmaf(qv.w, kv[e].w, x[j][e]))));
                    }
                }
            }
            const unsigned long long mine = pages >> (group * Z::KEYS);
            const bool whole = key0 >= sure_low && key0 + Z::KEYS <= sure_high && (Z::KEYS == 64 ? mine == ~0ull : (uint32_t)mine == 0xffffffffu);
            uint32_t sees[WARP_ROWS][EACH];
            float top[WARP_ROWS];
#pragma unroll
            for (int j = 0; j < WARP_ROWS; ++j) {
                const int at = slab0 + j, node = at < count ? at / p.group : -1;
                top[j] = m[j];
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    sees[j][e] = whole ? 0xffffffffu : node < 0 ? 0u : tree_sees(p, r, tree, node, key0 + 32 * e) & (uint32_t)(mine >> (32 * e));
                    x[j][e] = sees[j][e] >> lane & 1 ? x[j][e] * p.scale : -INFINITY;
                    top[j] = fmaxf(top[j], x[j][e]);
                }
            }
            // (all rows' maxima step by step together, and no branch where one stays: the chains of eight rows one after the other took longer)
#pragma unroll
            for (int step = 16; step > 0; step >>= 1)
#pragma unroll
                for (int j = 0; j < WARP_ROWS; ++j) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], step));
#pragma unroll
            for (int j = 0; j < WARP_ROWS; ++j) {
                const float base = top[j] == -INFINITY ? 0.0f : top[j], corr = exp2f(m[j] - base);
                l[j] *= corr, m[j] = top[j];
#pragma unroll
                for (int c = 0; c < Z::QUADS; ++c) o[j][c].x *= corr, o[j][c].y *= corr, o[j][c].z *= corr, o[j][c].w *= corr;
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    x[j][e] = sees[j][e] >> lane & 1 ? exp2f(x[j][e] - base) : 0.0f;
                    l[j] += x[j][e];
                }
            }
            __syncwarp();  // (the weights before are done with)
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                float4* to = reinterpret_cast<float4*>(weights + (lane + 32 * e) * WARP_ROWS);
                to[0] = make_float4(x[0][e], x[1][e], x[2][e], x[3][e]);
                to[1] = make_float4(x[4][e], x[5][e], x[6][e], x[7][e]);
            }
            __syncwarp();
            constexpr int STEP = Z::HALVES ? 2 : 1;
            const int half = Z::HALVES ? lane >> 4 : 0, col0 = (Z::HALVES ? lane & 15 : lane) * 4;
            auto add = [&](int key, bool masked) {
                const float4 f0 = *reinterpret_cast<const float4*>(weights + key * WARP_ROWS), f1 = *reinterpret_cast<const float4*>(weights + key * WARP_ROWS + 4);
                const float f[WARP_ROWS] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
#pragma unroll
                for (int c = 0; c < Z::QUADS; ++c) {
                    const int col = c * 128 + col0;
                    if (col >= D) continue;
                    const float4 v = *reinterpret_cast<const float4*>(vs + key * LD + col);
#pragma unroll
                    for (int j = 0; j < WARP_ROWS; ++j)
                        if (!masked || ((key < 32 ? sees[j][0] : sees[j][EACH - 1]) >> (key & 31) & 1)) {
                            o[j][c].x = fmaf(f[j], v.x, o[j][c].x), o[j][c].y = fmaf(f[j], v.y, o[j][c].y);
                            o[j][c].z = fmaf(f[j], v.z, o[j][c].z), o[j][c].w = fmaf(f[j], v.w, o[j][c].w);
                        }
                }
            };
            if (whole) {
#pragma unroll 4
                for (int key = half; key < Z::KEYS; key += STEP) add(key, false);
            } else {
                const int end = min(Z::KEYS, r.rows - key0);
#pragma unroll 1
                for (int key = half; key < end; key += STEP) add(key, true);
            }
        }
        // ---- the groups joined, in their order
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        float* join = smem;  // [warp][query row][LD]
#pragma unroll
        for (int j = 0; j < WARP_ROWS; ++j) {
            const float sum = warp_sum(l[j]);
            if (lane == 0) row_m[warp][j] = m[j], row_l[warp][j] = sum;
#pragma unroll
            for (int c = 0; c < Z::QUADS; ++c) {
                float4 v = o[j][c];
                if (Z::HALVES) {
                    v.x += __shfl_xor_sync(0xffffffffu, v.x, 16), v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
                    v.z += __shfl_xor_sync(0xffffffffu, v.z, 16), v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
                }
                const int col = c * 128 + (Z::HALVES ? lane & 15 : lane) * 4;
                if (col < D && (!Z::HALVES || lane < 16)) *reinterpret_cast<float4*>(join + (warp * WARP_ROWS + j) * LD + col) = v;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < Z::ROWS * (D / 4); i += THREADS) {
            const int row = i % Z::ROWS, c = i / Z::ROWS * 4, at = row0 + row;
            if (at >= count) continue;
            const int w = row / WARP_ROWS * G, in = row % WARP_ROWS;  // the warps w .. w + G - 1 have it
            float most = -INFINITY, sum = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int g = 0; g < G; ++g) most = fmaxf(most, row_m[w + g][in]);
            const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float f = exp2f(row_m[w + g][in] - base);
                const float4 y = *reinterpret_cast<const float4*>(join + ((w + g) * WARP_ROWS + in) * LD + c);
                sum = fmaf(f, row_l[w + g][in], sum);
                v.x = fmaf(f, y.x, v.x), v.y = fmaf(f, y.y, v.y), v.z = fmaf(f, y.z, v.z), v.w = fmaf(f, y.w, v.w);
            }
            if (whole_item) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                float* to = (float*)p.out + (size_t)(r.first + at / p.group) * p.ldo + (head * p.group + at % p.group) * D + c;
                to[0] = v.x * inv, to[1] = v.y * inv, to[2] = v.z * inv, to[3] = v.w * inv;
            } else {
                float* to = tree_part(p, blockIdx.x, first == 0, Z::ROWS) + row;
                to[c * Z::ROWS] = v.x, to[(c + 1) * Z::ROWS] = v.y, to[(c + 2) * Z::ROWS] = v.z, to[(c + 3) * Z::ROWS] = v.w;
                if (c == 0) to[D * Z::ROWS] = most, to[(D + 1) * Z::ROWS] = sum;
            }
        }
        __syncthreads();  // the tiles and the query rows may be written again
    }
    if (threadIdx.x == 0) p.begun[blockIdx.x] = begun;
}

template <int DP, int G>
int launch(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream) {
    const auto kernel = tree_attention_f32_kernel<DP, G>;
    const int rc = ferris_allow_dynamic_smem((const void*)kernel, Sizes<DP, G>::BYTES);
    if (rc != FERRIS_OK) return rc;
    const cudaError_t e = ferris_launch(kernel, dim3(plan.groups), dim3(THREADS), (size_t)Sizes<DP, G>::BYTES, stream, p);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    return FERRIS_OK;
}

// Two groups of warps (blocks of 32 query rows) where 64 would be filled up with more rows that are not there: six requests of 13 nodes (78 query rows) 66 us, in
// blocks of 64 74; of 5 (30 query rows) 37 and 43.
template <typename F>
void with_variant(int D, int rows, F f) {
    const bool two = (rows + 31) / 32 * 32 < (rows + 63) / 64 * 64;
    if (D <= 64) return two ? f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>()) : f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    if (D <= 128) return two ? f(std::integral_constant<int, 128>(), std::integral_constant<int, 2>()) : f(std::integral_constant<int, 128>(), std::integral_constant<int, 1>());
    f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
}

}  // namespace

TreePlan tree_plan_f32(int head_dim, int seqs, int kv_heads, int group, int max_nodes, int max_kv, int window) {
    TreePlan plan = {};
    with_variant(head_dim, max_nodes * group, [&](auto dp, auto g) {
        using Z = Sizes<dp.value, g.value>;
        plan.unit = Z::TILE, plan.rows = Z::ROWS;
    });
    plan.deal(seqs, kv_heads, group, max_nodes, plan.most_rows(max_kv, max_nodes, window, plan.unit), 1, true);
    return plan;
}

int tree_attention_f32(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream) {
    int rc = FERRIS_OK;
    with_variant(p.head_dim, p.max_nodes * p.group, [&](auto dp, auto g) { rc = launch<dp.value, g.value>(p, plan, stream); });
    return rc;
}
