// What the kernels of attention for trees of drafted tokens share: who sees which row, and where the parts of a row go.
//
// A request brings n tokens, the nodes of a forest (a chain is one): node i has the parent parents[i] < i among them, or none (-1).
// `start` rows of its text are cached; node i's keys and values are row start + i, its position is start + depth(i).  A node
// sees the text, itself and its ancestors; with a window, of these the keys whose position is above its own less the window.
// A query row r of a request and kv head is (node r / G, head r % G of the G heads that share the kv head).
#pragma once

#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "packed_cache.cuh"

constexpr int TREE_NODES = 256;                // most tokens that a request brings
constexpr int TREE_WORDS = TREE_NODES / 32;    // words of a node's line of ancestors
constexpr float TREE_LOG2E = 1.4426950408889634f;

struct TreeAttention {
    const void* q;
    void* out;
    const void* k_cache;
    const void* v_cache;
    int ldq, ldo;
    const int* tables;
    int width;  // blocks of a request's table
    int limit;  // rows that a request may have: those of its table, and no more than the caller says
    const int* q_start;
    const int* start_row;
    const int* parents;
    int seqs, tokens, heads, kv_heads, group, head_dim, pages, page_size, max_nodes, window;
    float scale;  // of the scores, times log2(e)
    DivideBy page;  // the page size
    float* parts;  // of D + 2 numbers a query row: unnormalised output, maximum (to the base of 2) and sum
    int splits;
    int* status;
};

// A request as a block sees it.
struct TreeRequest {
    int first, nodes, start, rows;  // its tokens' first row in q and out, their number; cached rows of text, and with the nodes
};

__device__ __forceinline__ TreeRequest tree_request(const TreeAttention& p, int seq) {
    TreeRequest r;
    r.first = min(max(p.q_start[seq], 0), p.tokens);
    const int len = min(max(p.q_start[seq + 1], r.first), p.tokens) - r.first;
    r.nodes = min(len, p.max_nodes);
    if (len > p.max_nodes) ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 110);
    r.start = max(p.start_row[seq], 0);
    r.rows = (int)min((long long)r.start + r.nodes, (long long)p.limit);
    return r;
}

// The page of a request's row, -1 where it has none.
__device__ __forceinline__ int tree_page(const TreeAttention& p, const int* table, int row) {
    const int block = (int)p.page.quotient((uint32_t)row);
    const int page = block < p.width ? table[block] : -1;
    if (page >= p.pages) {
        ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 111);
        return -1;
    }
    return page;
}

// The first element of a cached row of a kv head; 64 bits: a cache has more elements than 32 bits count.
__device__ __forceinline__ size_t tree_row_at(const TreeAttention& p, int page, int head, int row) {
    const int block = (int)p.page.quotient((uint32_t)row);
    return (((size_t)page * p.kv_heads + head) * p.page_size + (row - block * p.page_size)) * p.head_dim;
}

// Lines of ancestors in shared memory: bit j of node i's line says that i sees node j; and nodes' depths.
struct TreeLines {
    uint32_t line[TREE_NODES][TREE_WORDS];
    short parent[TREE_NODES];
    short depth[TREE_NODES];
};

// By all threads of the block, which are synchronised when it returns.  A parent that is not an earlier node of the request
// counts as none.
__device__ __forceinline__ void tree_lines(const TreeAttention& p, const TreeRequest& r, TreeLines& t) {
    for (int i = threadIdx.x; i < r.nodes; i += blockDim.x) {
        int up = p.parents[r.first + i];
        if (up >= i || up < -1) {
            ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 112);
            up = -1;
        }
        t.parent[i] = (short)up;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < r.nodes; i += blockDim.x) {
#pragma unroll
        for (int w = 0; w < TREE_WORDS; ++w) t.line[i][w] = 0u;
        int depth = 0;
        for (int at = i; at >= 0; at = t.parent[at], ++depth)
            if (p.window <= 0 || depth < p.window) t.line[i][at >> 5] |= 1u << (at & 31);
        t.depth[i] = (short)(depth - 1);
    }
    __syncthreads();
}

// Bits lo .. hi - 1 of 32, for bounds anywhere.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
    lo = max(lo, 0), hi = min(hi, 32);
    return lo >= hi ? 0u : (0xffffffffu >> (32 - (hi - lo))) << lo;
}

// Which of the 32 rows from `key0` on node `i` sees (whether they have a page is another matter).
__device__ __forceinline__ uint32_t tree_sees(const TreeAttention& p, const TreeRequest& r, const TreeLines& t, int i, int key0) {
    const int low = p.window > 0 ? r.start + t.depth[i] - p.window + 1 : 0;
    uint32_t m = bits_between(low - key0, r.start - key0);
    const int at = key0 - r.start;  // the node that the first row would be
    if (at > -32 && at < r.nodes) {
        const int w = at >> 5, s = at & 31;  // (w = -1 below nought)
        const uint32_t a = w >= 0 ? t.line[i][w] : 0u, b = w + 1 < TREE_WORDS ? t.line[i][w + 1] : 0u;
        m |= s ? __funnelshift_r(a, b, s) : a;
    }
    return m & bits_between(0, r.rows - key0);
}

// ---------------------------------------------------------------------------------------------
// The work of a step as units: an item is a block of query rows of a request and kv head, a unit `unit` cached rows of it.  Units are numbered
// through, requests first, then kv heads, then blocks of query rows, then cached rows.
// ---------------------------------------------------------------------------------------------
struct TreeUnits {
    int unit, rows;  // cached rows of a unit, query rows of a block
};

// Units in front of a request's cached rows that none of its nodes sees, units of an item, items.
struct TreeShape {
    int low, tiles, blocks;
};

__device__ __forceinline__ TreeShape tree_shape(const TreeAttention& p, const TreeUnits& u, const TreeRequest& r) {
    TreeShape s;
    s.low = p.window > 0 ? max(0, r.start - p.window + 1) / u.unit : 0;
    s.tiles = max((r.rows + u.unit - 1) / u.unit - s.low, 1);  // (nothing that could be seen: still a unit, which says so)
    s.blocks = (r.nodes * p.group + u.rows - 1) / u.rows;
    return s;
}

__device__ __forceinline__ int tree_scan(int v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += x;
    }
    return v;
}

// Units of the requests 32 i + lane, by a whole warp.
__device__ __forceinline__ int tree_units_of(const TreeAttention& p, const TreeUnits& u, int seq, TreeRequest& r) {
    if (seq >= p.seqs) return 0;
    r = tree_request(p, seq);
    const TreeShape s = tree_shape(p, u, r);
    return s.tiles * s.blocks * p.kv_heads;
}

// All units of the step, and those of the requests before `seq`; by a whole warp.
__device__ __forceinline__ int tree_total_units(const TreeAttention& p, const TreeUnits& u, int seq = -1, int* before = nullptr) {
    int total = 0;
    for (int s0 = 0; s0 < p.seqs; s0 += 32) {
        TreeRequest r;
        const int mine = tree_units_of(p, u, s0 + (threadIdx.x & 31), r), upto = tree_scan(mine);
        if (before && seq >= s0 && seq < s0 + 32) *before = total + __shfl_sync(0xffffffffu, upto - mine, seq - s0);
        total += __shfl_sync(0xffffffffu, upto, 31);
    }
    return total;
}

struct TreeItem {
    TreeRequest request;
    int seq, head, block, tile, tiles, low;
};

// The item that a unit belongs to, and which of its units it is; by a whole warp.
__device__ __forceinline__ TreeItem tree_item(const TreeAttention& p, const TreeUnits& u, int unit) {
    TreeItem item;
    int before = 0;
    for (int s0 = 0;; s0 += 32) {
        TreeRequest r = {};
        const int mine = tree_units_of(p, u, s0 + (threadIdx.x & 31), r), upto = tree_scan(mine);
        const unsigned here = __ballot_sync(0xffffffffu, unit < before + upto);
        if (here) {
            const int at = __ffs(here) - 1;
            item.seq = s0 + at;
            item.request.first = __shfl_sync(0xffffffffu, r.first, at);
            item.request.nodes = __shfl_sync(0xffffffffu, r.nodes, at);
            item.request.start = __shfl_sync(0xffffffffu, r.start, at);
            item.request.rows = __shfl_sync(0xffffffffu, r.rows, at);
            before += __shfl_sync(0xffffffffu, upto - mine, at);
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
        if (s0 >= p.seqs) {  // (no such unit)
            item = TreeItem();
            return item;
        }
    }
    const TreeShape s = tree_shape(p, u, item.request);
    const int in = unit - before, nth = in / s.tiles;
    item.tile = in - nth * s.tiles, item.tiles = s.tiles, item.low = s.low;
    item.head = nth / s.blocks, item.block = nth - item.head * s.blocks;
    return item;
}

// Blocks that get units: every one of them at least one, so that each between the first and the last of an item leaves a part of it.
__device__ __forceinline__ int tree_blocks(int total, int grid) { return min(total, grid); }
// The first unit of a block: the first total % blocks of them have one more than the others.
__device__ __forceinline__ int tree_begin(int block, int total, int blocks) {
    const int per = total / blocks, more = total - per * blocks;
    return block * per + min(block, more);
}
// The block that has a unit.
__device__ __forceinline__ int tree_owner(int unit, int total, int blocks) {
    const int per = total / blocks, more = total - per * blocks, at = more * (per + 1);
    return unit < at ? unit / (per + 1) : more + (unit - at) / per;
}

// bf16, on mma.sync (tree_attention_mma.cu).
struct TreeMmaPlan {
    int unit, rows, blocks;
    bool fits;  // units are counted in 32 bits
};
TreeMmaPlan tree_mma_plan(int head_dim, int seqs, int kv_heads, int group, int max_nodes, int max_kv);
int tree_attention_mma(const TreeAttention& p, const TreeMmaPlan& plan, cudaStream_t stream);
