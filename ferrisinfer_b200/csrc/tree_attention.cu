// Attention for trees of drafted tokens over the paged cache (who sees what: tree_attention.cuh).
//
// out = sum_j softmax_j(scale q . k_j) v_j over the rows j that a query's node sees, the softmax by running maximum and sum in
// 32 bits.  The cached rows of a request are cut into `splits` parts that blocks take side by side; a part leaves
// its unnormalised output with its maximum and sum, and a second kernel joins them:
//   m = max m_s, o = sum 2^(m_s - m) o_s, l = sum 2^(m_s - m) l_s, out = o / l  (to the base of 2; nothing seen: zeros).
#include "tree_attention.cuh"

namespace {

// ---------------------------------------------------------------------------------------------
// fp32, on the CUDA cores.  A block takes 32 query rows of a request and kv head, four to a warp, and goes
// over its part in tiles of 32 cached rows, which lie in shared memory in 32 bits:
//   scores   a lane is a cached row: its dot products with the warp's four query rows
//   outputs  a lane is every 32nd group of four columns: a cached row's weights for the four query rows are one read
// Whatever a query does not see is never multiplied: what lies there may be NaN.
// ---------------------------------------------------------------------------------------------
constexpr int ROWS = 32, WARP_ROWS = 4, KEYS = 32, THREADS = 256;

__host__ __device__ constexpr int padded(int d) { return d + 4; }  // rows of 16 bytes more: lanes read neighbouring rows without conflicts

template <int COLUMNS>  // COLUMNS: groups of four columns of a lane
__global__ void __launch_bounds__(THREADS) tree_attention_kernel(const TreeAttention p) {
    extern __shared__ __align__(16) float smem[];
    __shared__ TreeLines tree;
    __shared__ float4 weight[THREADS / 32][KEYS];
    const int D = p.head_dim, LD = padded(D);
    float* qs = smem;
    float* ks = qs + ROWS * LD;
    float* vs = ks + KEYS * LD;
    pdl_wait();
    pdl_launch_dependents();
    const int seq = blockIdx.z, head = blockIdx.y % p.kv_heads, row0 = blockIdx.y / p.kv_heads * ROWS, part = blockIdx.x;
    const TreeRequest r = tree_request(p, seq);
    const int count = r.nodes * p.group;
    if (row0 >= count) return;
    tree_lines<THREADS>(p, r, tree, [] { __syncthreads(); });
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* q = (const float*)p.q;
    for (int i = threadIdx.x; i < ROWS * D; i += THREADS) {
        const int row = i / D, c = i % D, at = row0 + row;
        qs[row * LD + c] = at < count ? q[(size_t)(r.first + at / p.group) * p.ldq + (head * p.group + at % p.group) * D + c] : 0.0f;
    }
    int node[WARP_ROWS];
#pragma unroll
    for (int i = 0; i < WARP_ROWS; ++i) {
        const int at = row0 + warp * WARP_ROWS + i;
        node[i] = at < count ? at / p.group : -1;
    }
    float m[WARP_ROWS], l[WARP_ROWS];
    float4 o[WARP_ROWS][COLUMNS];
#pragma unroll
    for (int i = 0; i < WARP_ROWS; ++i) {
        m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c) o[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    const int* table = p.tables + (size_t)seq * p.width;
    // the part's tiles; with a window those before the first row that the block's first... any of its nodes sees are left out
    const int low = p.window > 0 ? max(0, r.start - p.window + 1) / KEYS : 0;
    const int tiles = max((r.rows + KEYS - 1) / KEYS - low, 0), per = (tiles + p.splits - 1) / p.splits;
    const int begin = low + part * per, end = min(low + tiles, begin + per);
    for (int tile = begin; tile < end; ++tile) {
        const int key0 = tile * KEYS, row = key0 + lane;
        const int page = row < r.rows ? tree_page(p, table, row) : -1;
        const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
        __syncthreads();  // the tile before is done with
        for (int i = warp; i < KEYS; i += THREADS / 32) {
            if (!(there >> i & 1)) continue;
            const size_t at = tree_row_at(p, __shfl_sync(0xffffffffu, page, i), head, key0 + i);
            for (int c = lane * 4; c < D; c += 128) {
                *reinterpret_cast<float4*>(ks + i * LD + c) = *reinterpret_cast<const float4*>((const float*)p.k_cache + at + c);
                *reinterpret_cast<float4*>(vs + i * LD + c) = *reinterpret_cast<const float4*>((const float*)p.v_cache + at + c);
            }
        }
        __syncthreads();
        float s[WARP_ROWS] = {};
        const float* k = ks + lane * LD;
        for (int c = 0; c < D; c += 4) {
            const float4 kv = *reinterpret_cast<const float4*>(k + c);
#pragma unroll
            for (int i = 0; i < WARP_ROWS; ++i) {
                const float4 qv = *reinterpret_cast<const float4*>(qs + (warp * WARP_ROWS + i) * LD + c);
                s[i] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s[i]))));
            }
        }
        uint32_t sees[WARP_ROWS], all = 0xffffffffu, any = 0u;
        float corr[WARP_ROWS], w[WARP_ROWS];
#pragma unroll
        for (int i = 0; i < WARP_ROWS; ++i) {
            sees[i] = node[i] >= 0 ? tree_sees(p, r, tree, node[i], key0) & there : 0u;
            all &= sees[i], any |= sees[i];
            const bool mine = sees[i] >> lane & 1;
            const float x = mine ? s[i] * p.scale : -INFINITY, top = fmaxf(m[i], warp_max(x));
            const float base = top == -INFINITY ? 0.0f : top;
            corr[i] = exp2f(m[i] - base);
            w[i] = mine ? exp2f(x - base) : 0.0f;
            m[i] = top;
            l[i] = l[i] * corr[i] + w[i];
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) o[i][c].x *= corr[i], o[i][c].y *= corr[i], o[i][c].z *= corr[i], o[i][c].w *= corr[i];
        }
        weight[warp][lane] = make_float4(w[0], w[1], w[2], w[3]);
        __syncwarp();
        for (int j = 0; j < KEYS; ++j) {
            if (!(any >> j & 1)) continue;
            const float4 pw = weight[warp][j];
            const float f[WARP_ROWS] = {pw.x, pw.y, pw.z, pw.w};
            const bool whole = all >> j & 1;
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) {
                const int col = (c * 32 + lane) * 4;
                if (col < D) {
                    const float4 v = *reinterpret_cast<const float4*>(vs + j * LD + col);
#pragma unroll
                    for (int i = 0; i < WARP_ROWS; ++i)
                        if (whole || (sees[i] >> j & 1)) {
                            o[i][c].x = fmaf(f[i], v.x, o[i][c].x);
                            o[i][c].y = fmaf(f[i], v.y, o[i][c].y);
                            o[i][c].z = fmaf(f[i], v.z, o[i][c].z);
                            o[i][c].w = fmaf(f[i], v.w, o[i][c].w);
                        }
                }
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < WARP_ROWS; ++i) {
        if (node[i] < 0) continue;
        const float sum = warp_sum(l[i]);
        const int at = row0 + warp * WARP_ROWS + i, token = r.first + node[i], h = head * p.group + at % p.group;
        if (p.parts) {
            float* to = p.parts + (((size_t)part * p.tokens + token) * p.heads + h) * (D + 2);
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) {
                const int col = (c * 32 + lane) * 4;
                if (col < D) {  // (rows of parts begin on 8 bytes)
                    *reinterpret_cast<float2*>(to + col) = make_float2(o[i][c].x, o[i][c].y);
                    *reinterpret_cast<float2*>(to + col + 2) = make_float2(o[i][c].z, o[i][c].w);
                }
            }
            if (lane == 0) to[D] = m[i], to[D + 1] = sum;
        } else {
            float* to = (float*)p.out + (size_t)token * p.ldo + h * D;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) {
                const int col = (c * 32 + lane) * 4;
                if (col < D) {
                    to[col] = o[i][c].x * inv, to[col + 1] = o[i][c].y * inv;
                    to[col + 2] = o[i][c].z * inv, to[col + 3] = o[i][c].w * inv;
                }
            }
        }
    }
}

// The parts of a (token, head) joined, a warp each.  A token that no request brings is left alone.
__global__ void __launch_bounds__(256) tree_join_kernel(const TreeAttention p) {
    pdl_wait();
    pdl_launch_dependents();
    const int D = p.head_dim, lane = threadIdx.x & 31, seq = blockIdx.y;
    const TreeRequest r = tree_request(p, seq);
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= r.nodes * p.heads) return;
    const size_t at = (size_t)(r.first + row / p.heads) * p.heads + row % p.heads, step = (size_t)p.tokens * p.heads * (D + 2);
    const float* from = p.parts + at * (D + 2);
    float m = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, from[s * step + D]);
    m = warp_max(m);
    const float base = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
    for (int s = lane; s < p.splits; s += 32) {
        // (a part that saw nothing has the sum nought and the maximum of minus infinity; one of NaN scores has a NaN sum)
        sum += exp2f(from[s * step + D] - base) * from[s * step + D + 1];
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float* to = (float*)p.out + (size_t)(r.first + row / p.heads) * p.ldo + (row % p.heads) * D;
    for (int c = lane; c < D; c += 32) {
        float o = 0.0f;
        for (int s = 0; s < p.splits; ++s) o = fmaf(exp2f(from[s * step + D] - base), from[s * step + c], o);
        to[c] = o * inv;
    }
}

// The parts that the groups of a bf16 step's blocks left of items that lie in several: a block joins 32 query rows of an item, and as many columns.  A lane
// is a row, as the parts lie; a warp has four columns, and sixteen parts of them on their way at once.  Bound by latency: the item's groups, the parts'
// maxima and sums, the parts.
constexpr int JOIN_PARTS = 64;  // parts that are joined at once

__global__ void __launch_bounds__(256) tree_parts_kernel(const TreeAttention p, int rows, int lanes, int row_blocks) {
    __shared__ float top[8][32], tile[32][33], factor[JOIN_PARTS][32];
    pdl_wait();
    pdl_launch_dependents();
    const int D = p.head_dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y / row_blocks, row0 = (blockIdx.y - head * row_blocks) * min(rows, 32), col = blockIdx.x * 32 + warp * 4, seq = blockIdx.z;
    const int4 span = p.spans[seq * p.kv_heads + head];
    const int count = span.z * p.group, parts = span.y - span.x + 1;
    if (row0 >= count || parts <= 1) return;  // (one part: written by the block that has it)
    const int block = row0 / rows, in = row0 - block * rows + lane;  // (blocks have 16 rows or a multiple of 32)
    const bool live = row0 + lane < count && in < rows;
    auto part = [&](int k) { return tree_part(p, (span.x + k) * lanes + block, k == 0, rows) + in; };
    float m = -INFINITY, l = 0.0f, o[4] = {};  // l: of the warp's own parts
    for (int k0 = 0; k0 < parts; k0 += JOIN_PARTS) {
        const int n = min(parts - k0, JOIN_PARTS);
        float x[JOIN_PARTS / 8], y[JOIN_PARTS / 8], most = m;
#pragma unroll
        for (int u = 0; u < JOIN_PARTS / 8; ++u) {
            const bool there = live && warp + 8 * u < n;
            x[u] = there ? part(k0 + warp + 8 * u)[D * rows] : -INFINITY;
            y[u] = there ? part(k0 + warp + 8 * u)[(D + 1) * rows] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < JOIN_PARTS / 8; ++u) most = fmaxf(most, x[u]);
        if (k0) __syncthreads();  // (the factors before are done with)
        top[warp][lane] = most;
        __syncthreads();
        for (int w = 0; w < 8; ++w) most = fmaxf(most, top[w][lane]);
        const float base = most == -INFINITY ? 0.0f : most, corr = exp2f(m - base);
        m = most, l *= corr;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] *= corr;
#pragma unroll
        for (int u = 0; u < JOIN_PARTS / 8; ++u)
            if (warp + 8 * u < n) {
                const float f = exp2f(x[u] - base);
                factor[warp + 8 * u][lane] = f;
                l = fmaf(f, y[u], l);
            }
        __syncthreads();
        if (live && col < D)  // (heads have a multiple of eight columns)
            for (int k = 0; k < n; k += 16) {
                float v[16][4];
#pragma unroll
                for (int u = 0; u < 16; ++u)
                    if (k + u < n) {
                        const float* from = part(k0 + k + u) + col * rows;
#pragma unroll
                        for (int c = 0; c < 4; ++c) v[u][c] = from[c * rows];
                    }
#pragma unroll
                for (int u = 0; u < 16; ++u)
                    if (k + u < n) {
                        const float f = factor[k + u][lane];
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[c] = fmaf(f, v[u][c], o[c]);
                    }
            }
    }
    __syncthreads();
    top[warp][lane] = l;
    __syncthreads();
    l = 0.0f;
    for (int w = 0; w < 8; ++w) l += top[w][lane];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < 4; ++c) tile[warp * 4 + c][lane] = o[c] * inv;
    __syncthreads();
    // a warp: a row's columns
    const int out_col = blockIdx.x * 32 + lane;
    for (int row = warp; row < 32 && row0 + row < count && in - lane + row < rows; row += 8) {
        const int at = row0 + row;
        if (out_col < D)
            ((bf16*)p.out)[(size_t)(span.w + at / p.group) * p.ldo + (head * p.group + at % p.group) * D + out_col] = from_float<bf16>(tile[lane][row]);
    }
}

int launch(const TreeAttention& p, cudaStream_t stream) {
    const int blocks = (int)(((long long)p.max_nodes * p.group + ROWS - 1) / ROWS) * p.kv_heads;
    const size_t smem = (size_t)(ROWS + 2 * KEYS) * padded(p.head_dim) * sizeof(float);
    const dim3 grid(p.splits, blocks, p.seqs);
    const auto kernel = p.head_dim <= 128 ? tree_attention_kernel<1> : tree_attention_kernel<2>;
    const int rc = ferris_allow_dynamic_smem((const void*)kernel, smem);
    if (rc != FERRIS_OK) return rc;
    cudaError_t e = ferris_launch(kernel, grid, dim3(THREADS), smem, stream, p);
    if (e == cudaSuccess && p.parts)
        e = ferris_launch(tree_join_kernel, dim3((p.max_nodes * p.heads + 7) / 8, p.seqs), dim3(256), 0, stream, p);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    FERRIS_LAUNCH_CHECK();
}

}  // namespace

// How a step is cut: parts of a request's rows (32 bits), floats of scratch, launches.
FERRIS_API int ferris_tree_attention_plan(int dtype, int head_dim, int seqs, int kv_heads, int group, int tokens, int max_nodes, int max_kv, int page_size,
                                          long long cache_rows, float scale, int window, long long* needs) {
    if (dtype == FERRIS_BF16) {
        needs[0] = 1;
        needs[1] = tree_plan(head_dim, seqs, kv_heads, group, max_nodes, max_kv, page_size, cache_rows, scale, window).floats(seqs, kv_heads, head_dim);
        needs[2] = 2;
        return FERRIS_OK;
    }
    const long long blocks = ((long long)max_nodes * group + ROWS - 1) / ROWS * kv_heads * seqs;
    const int sms = ferris_sm_count();
    const long long tiles = (max_kv + KEYS - 1) / KEYS;
    long long splits = 2ll * (sms > 0 ? sms : 148) / (blocks > 0 ? blocks : 1);
    if (splits > tiles / 4) splits = tiles / 4;
    if (splits < 1) splits = 1;
    needs[0] = splits;
    needs[1] = splits > 1 ? splits * tokens * kv_heads * group * (head_dim + 2) : 0;
    needs[2] = splits > 1 ? 2 : 1;
    return FERRIS_OK;
}

// Arguments as ops.tree_attention lays them out.
struct TreeAttentionArgs {
    const void *q, *out, *k_cache, *v_cache, *tables, *q_start, *start_row, *parents, *parts, *stream;
    int ldq, ldo, dtype, pages, kv_heads, page_size, head_dim, width, seqs, tokens, heads, max_nodes, max_kv, window, splits;
    float scale;
};

FERRIS_API int ferris_tree_attention(const TreeAttentionArgs* a) {
    if (a->seqs <= 0 || a->tokens <= 0 || a->max_nodes <= 0) return FERRIS_OK;
    if (a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads) FERRIS_REFUSE("%d heads over %d kv heads", a->heads, a->kv_heads);
    if (a->head_dim <= 0 || a->head_dim % 8 || a->head_dim > 256) FERRIS_REFUSE("heads have a multiple of 8 elements, at most 256, not %d", a->head_dim);
    if (a->max_nodes > TREE_NODES) FERRIS_REFUSE("a request brings at most %d tokens, not %d", TREE_NODES, a->max_nodes);
    if (a->pages <= 0 || a->page_size <= 0 || a->width <= 0) FERRIS_REFUSE("%d pages of %d rows, tables of %d blocks", a->pages, a->page_size, a->width);
    if (((uintptr_t)a->k_cache | (uintptr_t)a->v_cache) & 15) FERRIS_REFUSE("the cache must begin on 16 bytes");
    if (a->seqs > 65535 || (long long)a->max_nodes * a->heads > 65535 * 8ll) FERRIS_REFUSE("%d requests of %d tokens exceed one launch", a->seqs, a->max_nodes);
    if (a->splits > 1 && !a->parts) FERRIS_REFUSE("%d parts need scratch", a->splits);
    TreeAttention p;
    p.q = a->q, p.out = const_cast<void*>(a->out), p.k_cache = a->k_cache, p.v_cache = a->v_cache;
    p.ldq = a->ldq, p.ldo = a->ldo;
    p.tables = (const int*)a->tables, p.width = a->width;
    const long long rows = (long long)a->width * a->page_size;
    p.limit = (int)(rows < a->max_kv ? rows : a->max_kv);
    p.q_start = (const int*)a->q_start, p.start_row = (const int*)a->start_row, p.parents = (const int*)a->parents;
    p.seqs = a->seqs, p.tokens = a->tokens, p.heads = a->heads, p.kv_heads = a->kv_heads, p.group = a->heads / a->kv_heads;
    p.head_dim = a->head_dim, p.pages = a->pages, p.page_size = a->page_size, p.max_nodes = a->max_nodes, p.window = a->window;
    p.scale = a->scale * TREE_LOG2E;
    p.page = DivideBy(a->page_size);
    p.splits = a->splits > 1 ? a->splits : 1;
    p.parts = p.splits > 1 ? (float*)const_cast<void*>(a->parts) : nullptr;
    p.spans = nullptr;
    p.status = ferris_status_ptr();
    if (a->dtype == FERRIS_BF16) {
        if (!a->parts) FERRIS_REFUSE("parts need scratch");
        const TreePlan plan = tree_plan(a->head_dim, a->seqs, a->kv_heads, p.group, a->max_nodes, p.limit, a->page_size,
                                        (long long)a->pages * a->kv_heads * a->page_size, a->scale, a->window);
        if (!plan.fits) FERRIS_REFUSE("%d requests of up to %d rows exceed one launch", a->seqs, p.limit);
        p.parts = (float*)const_cast<void*>(a->parts);
        // (the parts are a multiple of four floats: 2 x rows, which is a multiple of 16)
        p.spans = (int4*)(p.parts + 2ll * plan.groups * plan.lanes * plan.rows * (p.head_dim + 2));
        const int rc = plan.tensor ? tree_attention_tc(p, plan, (cudaStream_t)a->stream) : tree_attention_mma(p, plan, (cudaStream_t)a->stream);
        if (rc != FERRIS_OK) return rc;
        const int at_once = plan.rows < 32 ? plan.rows : 32;  // rows of a block of query rows that a block joins
        const int row_blocks = (p.max_nodes * p.group + at_once - 1) / at_once;
        const dim3 grid((p.head_dim + 31) / 32, row_blocks * p.kv_heads, p.seqs);
        const cudaError_t e = ferris_launch(tree_parts_kernel, grid, dim3(256), 0, (cudaStream_t)a->stream, p, plan.rows, plan.lanes, row_blocks);
        if (e != cudaSuccess) {
            ferris_set_error("%s", cudaGetErrorString(e));
            return (int)e;
        }
        FERRIS_LAUNCH_CHECK();
    }
    return launch(p, (cudaStream_t)a->stream);
}
