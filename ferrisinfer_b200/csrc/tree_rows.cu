// The cached rows of an accepted path move together behind the text of their request, in all layers at once.
//
// The nodes of a request's tree hold the rows start, start + 1, ...; of these the accepted ones, nodes[1] < nodes[2] < .. (nodes[0] is
// the token that was known), become the rows start + 1, start + 2, ..  A row never moves up, since nodes[j] >= j.  A thread owns 16
// bytes (fewer where the rows are no multiple) of a head of a layer in all of the request's rows: it alone reads and writes them, and
// since nodes[j'] > nodes[j] >= j for j' > j, no row that is still to be read has been written; loads of eight rows go ahead of their stores.
// Bound by latency: tables, then rows, then stores, whatever the sizes up to a few MB: one request in 24 layers 6.8 us, 64 in 28 layers (9 MB read, 9 written) 7.1.
#include "packed_cache.cuh"

namespace {

constexpr int PATH = 256;  // most nodes of a path
constexpr int THREADS = 128;

struct TreeRows {
    const long long* layers;  // [layers][2]: where a layer's keys and values begin
    const int* tables;
    const int* start_row;
    const int* nodes;
    const int* accepted;
    int width, path, seqs, pages, kv_heads, page_size, pieces;  // pieces: of a row of a head
    long long units;  // layers x 2 x kv heads x pieces
    DivideBy page;
    int* status;
};

template <typename V>
__global__ void __launch_bounds__(THREADS) tree_rows_kernel(const TreeRows p) {
    __shared__ long long from[PATH], to[PATH];  // rows of head 0, in rows of the cache; -1: none
    __shared__ int moves;
    pdl_wait();
    pdl_launch_dependents();
    const int seq = blockIdx.y, start = p.start_row[seq];
    const int* nodes = p.nodes + (size_t)seq * p.path;
    const int* table = p.tables + (size_t)seq * p.width;
    const int most = start < 0 ? 0 : min(p.accepted[seq], p.path - 1);
    if (threadIdx.x == 0) moves = max(most, 0);
    __syncthreads();
    auto row_of = [&](long long row) -> long long {
        const int block = row <= 0x7fffffff ? (int)p.page.quotient((uint32_t)row) : p.width;
        const int page = block < p.width ? table[block] : -1;
        if (page < 0 || page >= p.pages) {
            ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 121);
            return -1;
        }
        return (long long)page * p.kv_heads * p.page_size + (row - (long long)block * p.page_size);
    };
    for (int j = 1 + threadIdx.x; j <= most; j += THREADS) {
        const int node = nodes[j];
        // (of nodes that do not go up, neither they nor those behind them move)
        if (node < j || node <= nodes[j - 1] || node >= 0x7fffffff - start) {
            ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 120);
            atomicMin(&moves, j - 1);
            continue;
        }
        from[j] = node == j ? -1 : row_of((long long)start + node);
        to[j] = node == j ? -1 : row_of((long long)start + j);
        if (from[j] < 0 || to[j] < 0) from[j] = to[j] = -1;
    }
    __syncthreads();
    const int n = moves;
    const long long unit = (long long)blockIdx.x * THREADS + threadIdx.x;
    if (unit >= p.units) return;
    const int piece = (int)(unit % p.pieces), head = (int)(unit / p.pieces % p.kv_heads);
    V* base = (V*)p.layers[unit / p.pieces / p.kv_heads] + (long long)head * p.page_size * p.pieces + piece;
    for (int j = 1; j <= n; j += 8) {
        V v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j + i <= n && from[j + i] >= 0) v[i] = base[from[j + i] * p.pieces];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j + i <= n && from[j + i] >= 0) base[to[j + i] * p.pieces] = v[i];
    }
}

}  // namespace

// Arguments as ops.keep_tree_rows lays them out.  row_bytes: of a head's row; align: what the caches' addresses are a multiple of.
struct TreeRowsArgs {
    const void *layers, *tables, *start_row, *nodes, *accepted, *stream;
    int num_layers, pages, kv_heads, page_size, row_bytes, align, width, seqs, path;
};

FERRIS_API int ferris_tree_rows(const TreeRowsArgs* a) {
    if (a->seqs <= 0 || a->num_layers <= 0 || a->path <= 1) return FERRIS_OK;
    if (a->path > PATH) FERRIS_REFUSE("a path has at most %d nodes, not %d", PATH, a->path);
    if (a->pages <= 0 || a->kv_heads <= 0 || a->page_size <= 0 || a->row_bytes <= 0 || a->width <= 0 || a->seqs > 65535)
        FERRIS_REFUSE("%d pages of %d rows of %d heads of %d bytes, %d blocks, %d requests", a->pages, a->page_size, a->kv_heads, a->row_bytes,
                      a->width, a->seqs);
    int piece = 16;
    while (piece > 2 && (a->row_bytes % piece || a->align % piece)) piece /= 2;
    if (a->row_bytes % piece || a->align % piece) FERRIS_REFUSE("rows of %d bytes at a multiple of %d", a->row_bytes, a->align);
    TreeRows p;
    p.layers = (const long long*)a->layers, p.tables = (const int*)a->tables, p.start_row = (const int*)a->start_row;
    p.nodes = (const int*)a->nodes, p.accepted = (const int*)a->accepted;
    p.width = a->width, p.path = a->path, p.seqs = a->seqs, p.pages = a->pages, p.kv_heads = a->kv_heads, p.page_size = a->page_size;
    p.pieces = a->row_bytes / piece;
    p.units = (long long)a->num_layers * 2 * a->kv_heads * p.pieces;
    p.page = DivideBy(a->page_size);
    p.status = ferris_status_ptr();
    const long long blocks = (p.units + THREADS - 1) / THREADS;
    if (blocks > 0x7fffffff) FERRIS_REFUSE("%d layers exceed one launch", a->num_layers);
    const dim3 grid((unsigned)blocks, a->seqs);
    cudaError_t e;
    if (piece == 16)
        e = ferris_launch(tree_rows_kernel<uint4>, grid, dim3(THREADS), 0, (cudaStream_t)a->stream, p);
    else if (piece == 8)
        e = ferris_launch(tree_rows_kernel<uint2>, grid, dim3(THREADS), 0, (cudaStream_t)a->stream, p);
    else if (piece == 4)
        e = ferris_launch(tree_rows_kernel<uint32_t>, grid, dim3(THREADS), 0, (cudaStream_t)a->stream, p);
    else
        e = ferris_launch(tree_rows_kernel<uint16_t>, grid, dim3(THREADS), 0, (cudaStream_t)a->stream, p);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    FERRIS_LAUNCH_CHECK();
}
