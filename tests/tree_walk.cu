// How TreeWalk deals the work of a step out: every group's segments and its note, as the attention kernels get them.
#include "tree_attention.cuh"

namespace {

// Of a block: the number of its segments, its group's note (4), and of every segment request, kv head, block of query rows, first tile, last, tiles, tiles in front of
// them, number of the first tile.
constexpr int FIELDS = 8;

template <int UNIT, int ROWS, bool FLAT>
__global__ void __launch_bounds__(TreeRequests::MOST) walk_kernel(const TreeAttention p, int groups, int lanes, int room, int* out) {
    __shared__ TreeRequests requests;
    const int group = blockIdx.x / lanes, lane = blockIdx.x - group * lanes;
    TreeWalk<UNIT, ROWS, FLAT> walk;
    walk.know(p, requests);
    __syncthreads();
    walk.begin(p, requests, group, groups, lane);
    TreeItem item;
    int4 begun = walk.none();
    int n = 0;
    int* mine = out + (size_t)blockIdx.x * (5 + FIELDS * room);
    while (walk.next(p, requests, item)) {
        walk.note(item, begun);
        if (threadIdx.x == 0 && n < room) {
            int* to = mine + 5 + FIELDS * n;
            to[0] = item.seq, to[1] = item.head, to[2] = item.block, to[3] = item.first, to[4] = item.last, to[5] = item.tiles, to[6] = item.low, to[7] = item.start;
        }
        ++n;
    }
    if (threadIdx.x == 0) mine[0] = n, mine[1] = begun.x, mine[2] = begun.y, mine[3] = begun.z, mine[4] = begun.w;
}

template <int UNIT, int ROWS>
int walk(const TreeAttention& p, bool flat, int blocks, int groups, int lanes, int room, int* out) {
    if (flat)
        walk_kernel<UNIT, ROWS, true><<<blocks, TreeRequests::MOST>>>(p, groups, lanes, room, out);
    else
        walk_kernel<UNIT, ROWS, false><<<blocks, TreeRequests::MOST>>>(p, groups, lanes, room, out);
    return (int)cudaDeviceSynchronize();
}

}  // namespace

// `blocks` blocks of `lanes` to a group (groups that there are `groups` of: those behind them have nothing); out: (5 + 8 room) numbers a block.
FERRIS_API int tree_walk(int unit, int rows, int flat, int blocks, int groups, int lanes, int room, int* out, const int* q_start, const int* start_row, int seqs,
                         int tokens, int kv_heads, int group, int max_nodes, int limit, int window) {
    TreeAttention p = {};
    p.q_start = q_start, p.start_row = start_row;
    p.seqs = seqs, p.tokens = tokens, p.kv_heads = kv_heads, p.group = group, p.max_nodes = max_nodes, p.limit = limit, p.window = window;
    if (unit == 64 && rows == 32) return walk<64, 32>(p, flat, blocks, groups, lanes, room, out);
    if (unit == 128 && rows == 16) return walk<128, 16>(p, flat, blocks, groups, lanes, room, out);
    if (unit == 128 && rows == 128) return walk<128, 128>(p, flat, blocks, groups, lanes, room, out);
    if (unit == 128 && rows == 256) return walk<128, 256>(p, flat, blocks, groups, lanes, room, out);
    return -1;
}
