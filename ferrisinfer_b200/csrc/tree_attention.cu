// Attention for trees of drafted tokens over the paged cache: the C entry, and the join of what several blocks leave of a row (who sees what, and how the work
// is dealt out: tree_attention.cuh; the kernels: tree_attention_tc.cu, tree_attention_mma.cu, tree_attention_f32.cu).
//
// out = sum_j softmax_j(scale q . k_j) v_j over the rows j that a query's node sees, the softmax by running maximum and sum in
// 32 bits.  A block that has a part of a row's cached rows leaves its unnormalised output with its maximum and sum:
//   m = max m_s, o = sum 2^(m_s - m) o_s, l = sum 2^(m_s - m) l_s, out = o / l  (to the base of 2; nothing seen: zeros).
#include "tree_attention.cuh"

namespace {

// The parts that the groups' blocks left of items that lie in several: a block finds an item in the groups' notes (a block for every group, most of which had nothing
// to join, took 12 us for 8 requests of 16 nodes, so it takes 8.5) and joins 32 query rows of an item, and as many columns.  A lane
// is a row, as the parts lie; a warp has four columns, and sixteen parts of them on their way at once.  Bound by latency: the item's groups, the parts'
// maxima and sums, the parts: 6 us by itself for one request of five nodes.  Where items have few parts a block has 128 columns: 64 requests of 8 nodes
// (two or three parts an item) took 97 us with blocks of 32 columns, 82 so.
constexpr int JOIN_PARTS = 64;  // parts that are joined at once

template <typename T, int COLS>
__global__ void __launch_bounds__(256) tree_parts_kernel(const TreeAttention p, int rows, int groups, int lanes, int slices) {
    constexpr int AHEAD = 64 / COLS;
    __shared__ float top[8][32], tile[8 * COLS][33], factor[JOIN_PARTS][32];
    pdl_wait();
    pdl_launch_dependents();
    const int D = p.head_dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the z-th of the items that go on in other groups than the one that they begin in (others are written by their group); with lanes, the blocks of query rows
    // one after the other
    __shared__ int4 item;
    __shared__ int item_group, counts[8];
    if (threadIdx.x == 0) item_group = -1;
    for (int from = 0, skip = blockIdx.z; from < groups && skip >= 0; from += 256) {
        const int at = from + threadIdx.x;
        const int4 begun = at < groups ? p.begun[at] : make_int4(-1, 0, 0, 0);
        const unsigned have = __ballot_sync(0xffffffffu, begun.x >= 0);
        if (lane == 0) counts[warp] = __popc(have);
        __syncthreads();
        int before = __popc(have & ((1u << lane) - 1)), all = 0;
        for (int w = 0; w < 8; ++w) before += w < warp ? counts[w] : 0, all += counts[w];
        if (begun.x >= 0 && before == skip) item = begun, item_group = at;
        skip -= all;
        __syncthreads();
    }
    if (item_group < 0) return;
    const int group = item_group;
    const int seq = item.x, head = item.y, lane_block = blockIdx.y / slices, block = lanes > 1 ? lane_block : item.z, parts = item.w - group + 1;
    const int from_row = (blockIdx.y - lane_block * slices) * 32, row0 = block * rows + from_row, col = (blockIdx.x * 8 + warp) * COLS;
    const TreeRequest r = tree_request(p, seq);
    const int count = r.nodes * p.group, in = from_row + lane;
    if (row0 >= count) return;
    const bool live = row0 + lane < count && in < rows;
    auto part = [&](int k) { return tree_part(p, (group + k) * lanes + lane_block, k == 0, rows) + in; };
    float m = -INFINITY, l = 0.0f, o[COLS] = {};  // l: of the warp's own parts
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
        for (int c = 0; c < COLS; ++c) o[c] *= corr;
#pragma unroll
        for (int u = 0; u < JOIN_PARTS / 8; ++u)
            if (warp + 8 * u < n) {
                const float f = exp2f(x[u] - base);
                factor[warp + 8 * u][lane] = f;
                l = fmaf(f, y[u], l);
            }
        __syncthreads();
        if (live && col < D)
            for (int k = 0; k < n; k += AHEAD) {
                float v[AHEAD][COLS];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
                    if (k + u < n) {
                        const float* from = part(k0 + k + u) + col * rows;
#pragma unroll
                        for (int c = 0; c < COLS; ++c) v[u][c] = col + c < D ? from[c * rows] : 0.0f;
                    }
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
                    if (k + u < n) {
                        const float f = factor[k + u][lane];
#pragma unroll
                        for (int c = 0; c < COLS; ++c) o[c] = fmaf(f, v[u][c], o[c]);
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
    for (int c = 0; c < COLS; ++c) tile[warp * COLS + c][lane] = o[c] * inv;
    __syncthreads();
    // a warp: a row's columns
    for (int row = warp; row < 32 && row0 + row < count && in - lane + row < rows; row += 8) {
        const int at = row0 + row;
        T* to = (T*)p.out + (size_t)(r.first + at / p.group) * p.ldo + (head * p.group + at % p.group) * D;
#pragma unroll
        for (int c = 0; c < 8 * COLS; c += 32) {
            const int out_col = blockIdx.x * 8 * COLS + c + lane;
            if (out_col < D) to[out_col] = from_float<T>(tile[c + lane][row]);
        }
    }
}

TreePlan plan_of(int dtype, int head_dim, int seqs, int kv_heads, int group, int max_nodes, int max_kv, int page_size, long long cache_rows, float scale, int window) {
    if (dtype != FERRIS_BF16) return tree_plan_f32(head_dim, seqs, kv_heads, group, max_nodes, max_kv, window);
    return tree_plan(head_dim, seqs, kv_heads, group, max_nodes, max_kv, page_size, cache_rows, scale, window);
}

}  // namespace

// Floats of scratch of a step of these sizes.
FERRIS_API long long ferris_tree_attention_scratch(int dtype, int head_dim, int seqs, int kv_heads, int group, int max_nodes, int max_kv, int page_size,
                                                   long long cache_rows, float scale, int window) {
    return plan_of(dtype, head_dim, seqs, kv_heads, group, max_nodes, max_kv, page_size, cache_rows, scale, window).floats(head_dim);
}

// Arguments as ops.tree_attention lays them out.
struct TreeAttentionArgs {
    const void *q, *out, *k_cache, *v_cache, *tables, *q_start, *start_row, *parents, *parts, *stream;
    int ldq, ldo, dtype, pages, kv_heads, page_size, head_dim, width, seqs, tokens, heads, max_nodes, max_kv, window;
    float scale;
};

FERRIS_API int ferris_tree_attention(const TreeAttentionArgs* a) {
    if (a->seqs <= 0 || a->tokens <= 0 || a->max_nodes <= 0) return FERRIS_OK;
    if (a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads) FERRIS_REFUSE("%d heads over %d kv heads", a->heads, a->kv_heads);
    if (a->head_dim <= 0 || a->head_dim % 8 || a->head_dim > 256) FERRIS_REFUSE("heads have a multiple of 8 elements, at most 256, not %d", a->head_dim);
    if (a->max_nodes > TREE_NODES) FERRIS_REFUSE("a request brings at most %d tokens, not %d", TREE_NODES, a->max_nodes);
    if (a->pages <= 0 || a->page_size <= 0 || a->width <= 0 || a->max_kv <= 0)
        FERRIS_REFUSE("%d pages of %d rows, tables of %d blocks, %d rows at most", a->pages, a->page_size, a->width, a->max_kv);
    if (((uintptr_t)a->k_cache | (uintptr_t)a->v_cache) & 15) FERRIS_REFUSE("the cache must begin on 16 bytes");
    if (!a->parts || ((uintptr_t)a->parts & 15)) FERRIS_REFUSE("parts need scratch that begins on 16 bytes");
    TreeAttention p;
    p.q = a->q, p.out = const_cast<void*>(a->out), p.k_cache = a->k_cache, p.v_cache = a->v_cache;
    p.ldq = a->ldq, p.ldo = a->ldo;
    p.tables = (const int*)a->tables, p.width = a->width;
    const long long rows = (long long)a->width * a->page_size;
    p.limit = (int)(rows < a->max_kv ? rows : a->max_kv);
    if (p.limit > 0x7ffffc00) FERRIS_REFUSE("a request has at most %d rows, not %d", 0x7ffffc00, p.limit);
    p.q_start = (const int*)a->q_start, p.start_row = (const int*)a->start_row, p.parents = (const int*)a->parents;
    p.seqs = a->seqs, p.tokens = a->tokens, p.heads = a->heads, p.kv_heads = a->kv_heads, p.group = a->heads / a->kv_heads;
    p.head_dim = a->head_dim, p.pages = a->pages, p.page_size = a->page_size, p.max_nodes = a->max_nodes, p.window = a->window;
    p.scale = a->scale * TREE_LOG2E;
    p.page = DivideBy(a->page_size);
    p.status = ferris_status_ptr();
    const TreePlan plan = plan_of(a->dtype, a->head_dim, a->seqs, a->kv_heads, p.group, a->max_nodes, p.limit, a->page_size,
                                  (long long)a->pages * a->kv_heads * a->page_size, a->scale, a->window);
    if (!plan.fits) FERRIS_REFUSE("%d requests of up to %d tokens and %d rows exceed one launch", a->seqs, a->max_nodes, p.limit);
    // (blocks write their outputs while others still read; columns beside the queries', in rows of one length, are apart from them)
    const long long item = a->dtype == FERRIS_BF16 ? 2 : 4, columns = item * a->heads * a->head_dim, cache = item * a->pages * a->kv_heads * a->page_size * a->head_dim;
    const long long q_bytes = item * (a->tokens - 1) * a->ldq + columns, out_bytes = item * (a->tokens - 1) * a->ldo + columns, line = item * a->ldq;
    if (ferris_share_memory(a->q, q_bytes, a->out, out_bytes)) {
        const long long behind = a->ldq == a->ldo && line > 0 ? (((long long)((uintptr_t)a->out - (uintptr_t)a->q)) % line + line) % line : 0;
        if (behind < columns || behind > line - columns) FERRIS_REFUSE("the output must lie apart from the queries");
    }
    if (ferris_share_memory(a->k_cache, cache, a->out, out_bytes) || ferris_share_memory(a->v_cache, cache, a->out, out_bytes))
        FERRIS_REFUSE("the output must lie apart from the cache");
    p.parts = (float*)const_cast<void*>(a->parts);
    p.begun = (int4*)(p.parts + plan.part_floats(p.head_dim));
    const cudaStream_t stream = (cudaStream_t)a->stream;
    const int rc = a->dtype != FERRIS_BF16 ? tree_attention_f32(p, plan, stream) : plan.tensor ? tree_attention_tc(p, plan, stream) : tree_attention_mma(p, plan, stream);
    if (rc != FERRIS_OK) return rc;
    const int most = p.max_nodes * p.group, slices = ((most < plan.rows ? most : plan.rows) + 31) / 32;
    // sixteen columns a warp where items have few parts, so that there are fewer blocks, all at once
    const long long items = (long long)p.seqs * p.kv_heads * (plan.lanes > 1 ? 1 : (most + plan.rows - 1) / plan.rows);  // (of several groups no more than groups)
    const bool few = 4ll * p.seqs * p.kv_heads >= plan.groups;
    const dim3 grid((p.head_dim + (few ? 127 : 31)) / (few ? 128 : 32), slices * plan.lanes, (unsigned)(items < plan.groups ? items : plan.groups));
    const auto kernel = a->dtype == FERRIS_BF16 ? few ? tree_parts_kernel<bf16, 16> : tree_parts_kernel<bf16, 4> : few ? tree_parts_kernel<float, 16> : tree_parts_kernel<float, 4>;
    const cudaError_t e = ferris_launch(kernel, grid, dim3(256), 0, stream, p, plan.rows, plan.groups, plan.lanes, slices);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    FERRIS_LAUNCH_CHECK();
}
