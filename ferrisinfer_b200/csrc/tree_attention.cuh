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
    float* parts;
    int4* begun;  // of every group: the item that begins in it and goes on in others
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
    r.start = min(max(p.start_row[seq], 0), 0x7ffffe00);  // (positions of the nodes fit 32 bits)
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

// By THREADS of a block, for whom `barrier` is one; they are synchronised when it returns.  A parent that is not an earlier node of the
// request counts as none.
// (`parent`: what tree_parent says of the thread's first node, which may have been on its way for long)
__device__ __forceinline__ int tree_parent(const TreeAttention& p, const TreeRequest& r, int i) { return i < r.nodes ? p.parents[r.first + i] : -1; }
template <int THREADS, typename Barrier>
__device__ __forceinline__ void tree_lines(const TreeAttention& p, const TreeRequest& r, TreeLines& t, int parent, Barrier barrier) {
    for (int i = threadIdx.x % THREADS; i < r.nodes; i += THREADS) {
        int up = i < THREADS ? parent : p.parents[r.first + i];
        if (up >= i || up < -1) {
            ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 112);
            up = -1;
        }
        t.parent[i] = (short)up;
    }
    barrier();
    for (int i = threadIdx.x % THREADS; i < r.nodes; i += THREADS) {
#pragma unroll
        for (int w = 0; w < TREE_WORDS; ++w) t.line[i][w] = 0u;
        int depth = 0;
        for (int at = i; at >= 0; at = t.parent[at], ++depth)
            if (p.window <= 0 || depth < p.window) t.line[i][at >> 5] |= 1u << (at & 31);
        t.depth[i] = (short)(depth - 1);
    }
    barrier();
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
// The work of a step.  An item is a block of query rows of a request and kv head, a tile UNIT cached rows of it; the tiles are numbered through and
// dealt out evenly to the blocks of the grid, whatever the requests' lengths; in short steps, where one more tile costs less than to begin and end a second
// item, in runs of one item each (8 requests of 16 nodes after 4,096 rows 27 -> 22.5 us, 64 nodes after 131,071 rows 95 -> 82).  Two ways:
// FLAT   requests first, then kv heads, blocks of query rows, cached rows: all blocks have the same number of tiles.
// lanes  groups of `lanes` blocks, one for every block of query rows that the largest request has; requests, kv heads, cached rows are dealt out to the groups.
//        The blocks of a group go over the same cached rows side by side, so that those are read from memory once, however long the cache.
// An item that lies in one block is written by it; of others every block leaves its part (at most two of a block), which tree_parts_kernel joins
// in the order of the tiles, so that results do not depend on timing.
// ---------------------------------------------------------------------------------------------
struct TreePlan {
    int unit, rows;          // cached rows of a tile, query rows of a block
    int groups, lanes;       // groups of blocks, blocks of a group
    bool tensor;             // on tcgen05 (tree_attention_tc.cu), otherwise on mma.sync (tree_attention_mma.cu)
    bool fits;               // tiles are counted in 32 bits, and lanes are a launch's second dimension
    long long part_floats(int head_dim) const { return 2ll * groups * lanes * rows * (head_dim + 2); }
    long long floats(int head_dim) const { return part_floats(head_dim) + 4ll * groups; }  // of scratch: parts, and behind them the items that groups have begun
    // The most rows that a request's tiles hold: behind a window those of the window, of the nodes and of the tile in which it begins.
    static int most_rows(int max_kv, int max_nodes, int window, int unit) {
        const long long seen = (long long)window + max_nodes + unit;
        return window > 0 && seen < max_kv ? (int)seen : max_kv;
    }
    // As many blocks as the SMs have room for (`blocks` on each), and there can be tiles for (max_kv: most_rows).
    void deal(int seqs, int kv_heads, int group, int max_nodes, int max_kv, int blocks, bool flat) {
        const int sms = ferris_sm_count();
        const int row_blocks = (max_nodes * group + rows - 1) / rows;
        lanes = flat ? 1 : row_blocks;
        const long long most = (long long)seqs * kv_heads * (flat ? row_blocks : 1) * ((max_kv + unit - 1) / unit + 1);
        const long long room = (long long)(sms > 0 ? sms : 148) * blocks / lanes;
        groups = (int)(room < 1 ? 1 : room < most ? room : most);
        fits = most <= 0x7ff00000 && lanes <= 4096;
    }
};
TreePlan tree_plan(int head_dim, int seqs, int kv_heads, int group, int max_nodes, int max_kv, int page_size, long long cache_rows, float scale, int window);
int tree_attention_mma(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream);
int tree_attention_tc(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream);
TreePlan tree_plan_f32(int head_dim, int seqs, int kv_heads, int group, int max_nodes, int max_kv, int window);
int tree_attention_f32(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream);

__device__ __forceinline__ int tree_scan(int v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += x;
    }
    return v;
}

struct TreeItem {
    TreeRequest request;
    int seq, head, block;
    int first, last, tiles, low;  // its tiles that are this group's, of all its tiles; tiles of the request in front of them, which none of its nodes sees
    int start;                    // number of its first tile
};

// The requests of a step, if they are no more than these, as one block's warps fetch them once for all.
struct TreeRequests {
    static constexpr int MOST = 128;
    int first[MOST], nodes[MOST], start[MOST], rows[MOST];
};

// Goes through a group's share, item by item; by whole warps, each for itself.
template <int UNIT, int ROWS, bool FLAT>
struct TreeWalk {
    int at, end, lane_block;  // where this group is and where it ends; block of query rows of this lane
    int per, more;            // tiles of a group, and groups that have one more
    int round;                // items begin on a multiple of this
    TreeRequest mine;         // of request 32 s0 + lane
    int s0, before, upto;     // tiles before these requests, and up to and with this lane's

    static __device__ __forceinline__ int low(const TreeAttention& p, const TreeRequest& r) { return p.window > 0 ? max(0, r.start - p.window + 1) / UNIT : 0; }
    static __device__ __forceinline__ int tiles(const TreeAttention& p, const TreeRequest& r) {
        return max((r.rows + UNIT - 1) / UNIT - low(p, r), 1);  // (nodes that can see nothing: still a tile, which says so)
    }
    static __device__ __forceinline__ int blocks(const TreeAttention& p, const TreeRequest& r) { return FLAT ? (r.nodes * p.group + ROWS - 1) / ROWS : 1; }

    __device__ __forceinline__ void look_at(const TreeAttention& p, const TreeRequests& known, int chunk) {
        s0 = chunk;
        const int seq = 32 * chunk + (threadIdx.x & 31);
        if (p.seqs <= TreeRequests::MOST) {
            mine.first = known.first[seq], mine.nodes = known.nodes[seq], mine.start = known.start[seq], mine.rows = known.rows[seq];
        } else
            fetch(p, seq);
        upto = tree_scan(mine.nodes > 0 ? span(tiles(p, mine)) * blocks(p, mine) * p.kv_heads : 0);
    }
    __device__ __forceinline__ int span(int tiles) const { return round > 1 ? (tiles + round - 1) / round * round : tiles; }
    __device__ __forceinline__ void fetch(const TreeAttention& p, int seq) {
        mine.first = mine.nodes = mine.start = mine.rows = 0;
        if (seq < p.seqs) mine = tree_request(p, seq);
    }
    // By all threads of a block (at least TreeRequests::MOST), who have to meet before they begin.
    __device__ __forceinline__ void know(const TreeAttention& p, TreeRequests& known) {
        const int seq = threadIdx.x;
        if (p.seqs > TreeRequests::MOST || (seq & ~31) >= p.seqs) return;
        fetch(p, seq);
        known.first[seq] = mine.first, known.nodes[seq] = mine.nodes, known.start[seq] = mine.start, known.rows[seq] = mine.rows;
    }
    // Group `group` of `groups` (one beyond them has nothing).
    __device__ __forceinline__ void begin(const TreeAttention& p, const TreeRequests& known, int group, int groups, int lane) {
        const int chunks = (p.seqs + 31) / 32;
        lane_block = lane, round = 1;
        int total = 0;
        if (p.seqs <= TreeRequests::MOST) {
            constexpr int CHUNKS = TreeRequests::MOST / 32;
            int each[CHUNKS], items[CHUNKS], mine_all = 0;  // tiles of an item of this lane's requests, items
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                items[c] = each[c] = 0;
                if (c < chunks) {
                    const int seq = 32 * c + (threadIdx.x & 31);
                    const TreeRequest r = {known.first[seq], known.nodes[seq], known.start[seq], known.rows[seq]};
                    if (r.nodes > 0) each[c] = tiles(p, r), items[c] = blocks(p, r) * p.kv_heads;
                    mine_all += each[c] * items[c];
                }
            }
            total = __reduce_add_sync(0xffffffffu, mine_all);
            per = total / groups, more = total - per * groups;
            // a group within one item, if it has no more than a tile more for that
            const int even = per + (more > 0);
            for (int u = even; u > 1 && u <= even + 1; ++u) {
                int runs = 0;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
                    if (c < chunks) runs += (each[c] + u - 1) / u * items[c];
                runs = __reduce_add_sync(0xffffffffu, runs);
                if (runs <= groups) {
                    total = runs * u, per = round = u, more = 0;
                    break;
                }
            }
        } else {
            for (int c = 0; c < chunks; ++c) {
                look_at(p, known, c);
                total += __shfl_sync(0xffffffffu, upto, 31);
            }
            per = total / groups, more = total - per * groups;
        }
        at = min(total, group * per + min(group, more)), end = group < groups ? min(total, at + per + (group < more)) : at;  // (groups that have no tiles leave no part either)
        look_at(p, known, 0), before = 0;
    }
    // The group that has a tile.
    __device__ __forceinline__ int owner(int tile) const {
        const int longer = more * (per + 1);
        return tile < longer ? tile / (per + 1) : more + (tile - longer) / per;
    }
    // What is written into TreeAttention::begun when an item goes on in the groups behind this one: request (-1: no such item), kv head, block of query rows, last group.
    static __device__ __forceinline__ int4 none() { return make_int4(-1, 0, 0, 0); }
    __device__ __forceinline__ void note(const TreeItem& i, int4& begun) const {
        if (i.first == 0 && i.last < i.tiles) begun = make_int4(i.seq, i.head, i.block, owner(i.start + i.tiles - 1));
    }

    __device__ __forceinline__ bool next(const TreeAttention& p, const TreeRequests& known, TreeItem& item) {
        while (at < end) {
            unsigned here;
            while (!(here = __ballot_sync(0xffffffffu, at < before + upto))) {
                before += __shfl_sync(0xffffffffu, upto, 31);
                look_at(p, known, s0 + 1);
            }
            const int lane = __ffs(here) - 1;
            item.seq = 32 * s0 + lane;
            item.request.first = __shfl_sync(0xffffffffu, mine.first, lane);
            item.request.nodes = __shfl_sync(0xffffffffu, mine.nodes, lane);
            item.request.start = __shfl_sync(0xffffffffu, mine.start, lane);
            item.request.rows = __shfl_sync(0xffffffffu, mine.rows, lane);
            const TreeRequest& r = item.request;
            item.low = low(p, r), item.tiles = tiles(p, r);
            const int from = before + (lane ? __shfl_sync(0xffffffffu, upto, lane - 1) : 0);
            const int each = span(item.tiles), n = (at - from) / each, blocks_each = blocks(p, r);
            item.head = n / blocks_each;
            item.block = FLAT ? n - item.head * blocks_each : lane_block;
            item.start = from + n * each;
            item.first = at - item.start, item.last = min(item.tiles, end - item.start);
            at = item.start + (item.last == item.tiles ? each : item.last);
            if (FLAT || item.block * ROWS < r.nodes * p.group) return true;
        }
        return false;
    }
};

// Where a block's part lies: of an item that begins in it, or of one that began in front of it.  Column c of row r at [c][r]: D columns of the
// unnormalised output, the maximum (to the base of 2), the sum.
__device__ __forceinline__ float* tree_part(const TreeAttention& p, int block, bool begins, int rows) {
    return p.parts + (size_t)(2 * block + begins) * rows * (p.head_dim + 2);
}
