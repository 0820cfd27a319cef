// Attention of prompts over the paged cache in 4 bits, on the 5th-generation tensor cores: bf16 rows, heads of 64 and 128.
//
// Query rows (query, head of the group) of a request and kv head go in tiles of 128, two tiles to a block, which take the
// cached rows in blocks of 128 keys.  Four warps form the operands of a block in fp16 once for both tiles:
//   keys    scale (code - 8), which is EXACT in the eleven bits of fp16 (a scale has eight bits, code - 8 at most three or is a power of
//           two), and in sixteen further columns the middle = least + 8 scale of every group in two parts against the sums of
//           the query's groups in two parts:  s = sum_j [scale_j (code_j - 8) . q_j + middle_j sum(q_j)], all but exact in 32 bits
//   values  scale (code - 8) + middle, rounded to fp16
// both times a power of two for the block (of values: for the run of blocks) that keeps them inside the range of fp16.  A
// word of eight codes becomes its sixteen bytes with 13 instructions; in the order in which they come out of the word, which the
// queries' columns and the outputs' follow.
//   S = Q K^T    tcgen05.mma 128 x 128 into tensor memory, fp32
//   P = 2^(S - m + 7) read by a thread a row, written back over S as fp16: the A operand of
//   O += P V     tcgen05.mma 128 x D, accumulated in tensor memory over all blocks.
// The maximum m of a row is left behind by up to 2^8: O is scaled (read and written by its warps) only when a score exceeds
// that, which after the first blocks of a row is rare.  While the softmax warps of one tile work, the tensor cores work for the other.
// Bound by the chain of softmax, product and scores of a tile (the weights stand where the next scores go): 512 tokens after 32,768 rows
// (28 / 4 heads of 128) about 310 us in a sequence of calls, 770 TFLOP/s (345 by itself, caches cold); tensor pipe 35 % busy, issue
// slots 48 %.
#include <algorithm>

#include "packed_attention.cuh"

namespace {

constexpr int ROWS = 128;    // query rows of a tile
constexpr int BLOCK = 128;   // cached rows of a block
constexpr int SOFTMAX = 8, CONVERT = 4, THREADS = (SOFTMAX + CONVERT + 1) * 32;
constexpr int EXTRA = 4096;  // sixteen further columns of an operand: 128 rows x 32 bytes
constexpr int INFOS = 4;
constexpr int TABLE = 1024;  // most pairs of tiles (of one kv head) whose blocks are dealt out evenly
// Weights are formed 2^7 times too great, as are their sums: at most 2^15 then, and eleven bits in fp16 down to 2^-21 of the maximum (2^-14
// without it: thousands of rows of a weight of e^-15 of the greatest came out off by 0.026 of what they add up to).
constexpr float RAISE = 7.0f;
constexpr int LEAST_PIECE = 4, RUN = 16;  // blocks: fewest of a piece; from which on a CTA may go on with the next pair

template <int D>
struct Shape {
    static constexpr int W = D / 32, ATOMS = D / 64, ATOM = 16384;
    static constexpr int OPERAND = ATOMS * ATOM + EXTRA;  // Q tile or K block
    static constexpr int V_BYTES = ATOMS * ATOM;
    static constexpr int SMEM = 4 * OPERAND + 2 * V_BYTES + 1024;
};

// A pair of tiles: request, which one of the request, first block of cached rows and how many; and what a request is.
struct __align__(16) Pair {
    int seq, index, first, count, t0, rows, start, limit;
};

// Scratch of a step: queries as operands, their scales, the pairs, running sums of blocks (or pieces), parts.
struct Layout {
    unsigned char* queries;  // [pair][kv head][2 tiles] operands
    float* scales;           // [pair][kv head][256]: what makes a product one to the base of 2
    float* minus_lse;        // the same: minus the log2 of the row's sum (with weights; minus infinity for rows that are not there)
    int* first_pair;         // [request]
    int room;                // pairs that there is room for
    Pair* pairs;
    int* before;             // [pairs + 1], then the number of pairs, units, blocks of a piece
    float* parts;            // [place][D + 2][256]
    long long bytes;
};

// Places for parts (Deal::place): pieces leave one a CTA, runs two, but those are dealt out to no more CTAs than there are SMs.
int part_places(int grid, int sms) { return std::max(grid, 2 * std::min(grid, sms)); }

template <typename F>
void for_scratch(int D, int pairs, int kv_heads, int seqs, int places, F&& take) {
    const long long operand = (long long)(D / 64) * 16384 + EXTRA;
    take(0, (long long)pairs * kv_heads * 2 * operand);
    take(1, (long long)pairs * kv_heads * 256 * 4);
    take(2, (long long)pairs * sizeof(Pair));
    take(3, (long long)(pairs + 4) * 4);
    take(4, (long long)places * (D + 2) * 256 * 4);
    take(5, (long long)pairs * kv_heads * 256 * 4);
    take(6, (long long)seqs * 4);
}

Layout make_layout(void* base, int D, int pairs, int kv_heads, int seqs, int places) {
    Layout l = {};
    unsigned char* at = (unsigned char*)base;
    long long used = 0;
    for_scratch(D, pairs, kv_heads, seqs, places, [&](int what, long long bytes) {
        unsigned char* p = at + used;
        if (what == 0) l.queries = p;
        if (what == 1) l.scales = (float*)p;
        if (what == 2) l.pairs = (Pair*)p;
        if (what == 3) l.before = (int*)p;
        if (what == 4) l.parts = (float*)p;
        if (what == 5) l.minus_lse = (float*)p;
        if (what == 6) l.first_pair = (int*)p;
        used += (bytes + 1023) / 1024 * 1024;
    });
    l.bytes = used;
    l.room = pairs;
    return l;
}

// How the blocks of all pairs and kv heads are dealt out (packed_attention.cu has the same for few rows): runs that go on
// with the next pair where they are long, pieces of each pair where they are short.
struct Deal {
    int units, blocks, chunk, runs;
    __device__ __forceinline__ Deal(int units, int most, int chunk) : units(units), chunk(chunk) {
        blocks = min(most, max(1, units / LEAST_PIECE));
        runs = chunk >= RUN;
    }
    // Blocks of a piece where every CTA gets the same; pieces may have to be longer (packed_queries_kernel).
    static __device__ __forceinline__ int even_chunk(int units, int most) { return max(LEAST_PIECE, (units + most - 1) / most); }
    __device__ __forceinline__ int pieces(int n) const { return (n + chunk - 1) / chunk; }
    __device__ __forceinline__ int block_of(int u) const { return (int)((((long long)u + 1) * blocks - 1) / units); }
    __device__ __forceinline__ int begin_of(int block) const { return (int)((long long)block * units / blocks); }
    __device__ __forceinline__ int place(int i, int first) const { return runs ? 2 * i + (i == first) : i; }
};

struct Request {
    int t0, rows, start, limit;
    __device__ __forceinline__ explicit Request(const Pair& pair) : t0(pair.t0), rows(pair.rows), start(pair.start), limit(pair.limit) {}
    __device__ __forceinline__ Request(const PackedAttention& p, int seq) {
        t0 = max(p.q_start[seq], 0);
        rows = (min(p.q_start[seq + 1], p.tokens) - t0) * p.group;
        start = p.start_row[seq];
        limit = p.limit;
    }
    __device__ __forceinline__ int pairs(const PackedAttention& p) const { return rows > p.few ? (rows + 2 * ROWS - 1) / (2 * ROWS) : 0; }
    __device__ __forceinline__ void sees(const PackedAttention& p, int r, int& lo, int& hi) const {
        const int at = start + r / p.group;
        hi = max(0, min(at + 1, limit));
        lo = min(p.window > 0 ? max(0, at - p.window + 1) : 0, hi);
    }
    // blocks that the rows first .. last see
    __device__ __forceinline__ void blocks(const PackedAttention& p, int first, int last, int& from, int& to) const {
        int lo, hi, x;
        sees(p, first, lo, x);
        sees(p, last, x, hi);
        lo = min(lo, hi);
        from = lo / BLOCK;
        to = max((hi + BLOCK - 1) / BLOCK, from);
    }
};

__device__ __forceinline__ int warp_inclusive(int v, int lane) {
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, x);
        if (lane >= x) v += u;
    }
    return v;
}

// The first block lists the pairs and how their blocks are dealt out; every other block (of the second row on: of the others) forms the two
// operand tiles of a pair: query rows in fp16, times a power of two that brings a row's greatest element to 2^13, columns in the
// order of the keys' codes (8 elements 0 4 1 5 2 6 3 7), and the rows' group sums over 64 in two parts.
template <int D>
__global__ void __launch_bounds__(256) packed_queries_kernel(const PackedAttention p, const Layout l, int sms) {
    constexpr int W = D / 32;
    __shared__ int sums[9];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x;
    if (blockIdx.x == 0) {
        if (blockIdx.y) return;
        int n_pairs = 0;
        for (int s0 = 0; s0 < p.seqs; s0 += 256) {  // the pairs of 256 requests at a time, a warp's lanes along a request's
            const int n = s0 + tid < p.seqs ? Request(p, s0 + tid).pairs(p) : 0, upto = warp_inclusive(n, lane);
            if (lane == 31) sums[warp] = upto;
            __syncthreads();
            int at = n_pairs + upto - n;
            for (int w = 0; w < warp; ++w) at += sums[w];
            if (s0 + tid < p.seqs) l.first_pair[s0 + tid] = at;
            int all = 0;
            for (int w = 0; w < 8; ++w) all += sums[w];
            for (int i = 0; i < 32; ++i) {
                const int mine = __shfl_sync(0xffffffffu, n, i), first = __shfl_sync(0xffffffffu, at, i), seq = s0 + 32 * warp + i;
                if (mine == 0) continue;
                const Request rq(p, seq);
                for (int k = lane; k < mine && first + k < (int)gridDim.x - 1; k += 32) {  // (as many as there is room for)
                    Pair q = {seq, k, 0, 0, rq.t0, rq.rows, rq.start, rq.limit};
                    int to;
                    rq.blocks(p, k * 2 * ROWS, min((k + 1) * 2 * ROWS, rq.rows) - 1, q.first, to);
                    q.count = max(1, to - q.first);
                    l.pairs[first + k] = q;
                }
            }
            n_pairs += all;
            __syncthreads();
        }
        n_pairs = min(n_pairs, (int)gridDim.x - 1);
        int units = 0;
        for (int i = tid; i < n_pairs; i += 256) units += l.pairs[i].count;
        units = __reduce_add_sync(0xffffffffu, units);
        if (lane == 0) sums[warp] = units;
        __syncthreads();
        units = 0;
        for (int w = 0; w < 8; ++w) units += sums[w];
        __syncthreads();
        units *= p.cache.kv_heads;
        // Pieces that leave a CTA more than there are SMs would make all of them wait for a second round (six prompts of up to 700
        // tokens do not show it: 38.7 us without this, 38.8 with it): where the pairs are few enough, pieces are lengthened until they fit.
        int chunk = Deal::even_chunk(max(units, 1), sms);
        while (chunk < RUN && n_pairs * p.cache.kv_heads <= sms) {
            int pieces = 0;
            for (int i = tid; i < n_pairs; i += 256) pieces += (l.pairs[i].count + chunk - 1) / chunk;
            pieces = __reduce_add_sync(0xffffffffu, pieces);
            __syncthreads();
            if (lane == 0) sums[warp] = pieces;
            __syncthreads();
            pieces = 0;
            for (int w = 0; w < 8; ++w) pieces += sums[w];
            if (pieces * p.cache.kv_heads <= sms) break;
            ++chunk;
        }
        __syncthreads();
        const Deal deal(max(units, 1), sms, chunk);
        int before = 0;
        for (int i0 = 0; i0 < n_pairs; i0 += 256) {
            const int c = i0 + tid < n_pairs ? l.pairs[i0 + tid].count : 0, n = p.cache.kv_heads * (deal.runs ? c : deal.pieces(c));
            const int upto = warp_inclusive(n, lane);
            if (lane == 31) sums[warp] = upto;
            __syncthreads();
            int at = before + upto - n;
            for (int w = 0; w < warp; ++w) at += sums[w];
            for (int w = 0; w < 8; ++w) before += sums[w];
            if (i0 + tid < n_pairs) l.before[i0 + tid] = at;
            __syncthreads();
        }
        if (tid == 0) {
            l.before[n_pairs] = before;
            l.before[gridDim.x] = n_pairs;  // (gridDim.x - 1 pairs at most)
            l.before[gridDim.x + 1] = units;
            l.before[gridDim.x + 2] = chunk;
        }
        return;
    }
    // which request's pair this is: a lane a request
    const int pair = (int)blockIdx.x - 1;
    int seq = -1, k = 0;
    for (int s0 = 0, before = 0; s0 < p.seqs && seq < 0; s0 += 32) {
        const int n = s0 + lane < p.seqs ? Request(p, s0 + lane).pairs(p) : 0, upto = warp_inclusive(n, lane);
        const unsigned here = __ballot_sync(0xffffffffu, pair < before + upto);
        if (here) {
            const int at = __ffs(here) - 1;
            seq = s0 + at;
            k = pair - before - __shfl_sync(0xffffffffu, upto - n, at);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (seq < 0) return;
    const Request rq(p, seq);
    const int head = blockIdx.y, g = lane >> 2, c = lane & 3;
    const size_t index = (size_t)pair * gridDim.y + head;
    for (int rr = 8 * warp + g; rr < 2 * ROWS; rr += 64) {
        const int row = k * 2 * ROWS + rr, r = rr % ROWS;
        const bool valid = row < rq.rows;
        const bf16* src = (const bf16*)p.q + (size_t)(rq.t0 + row / p.group) * p.ldq + (size_t)(head * p.group + row % p.group) * D;
        float x[W][8] = {}, top = 0.0f;
        if (valid && p.q_aligned) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const uint4 v = reinterpret_cast<const uint4*>(src + 32 * j + 8 * c)[0];
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
            }
        } else if (valid) {
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = to_float(src[32 * j + 8 * c + i]);
        }
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[j][i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (int)(__float_as_uint(top) >> 23);
        // (a negative scale goes into the queries, so that what makes a product a score is never below nought)
        const float factor = copysignf(top > 0.0f && e < 255 ? __uint_as_float((uint32_t)min(267 - e, 253) << 23) : 1.0f, p.scale);
        unsigned char* tile = l.queries + (index * 2 + rr / ROWS) * Shape<D>::OPERAND;
        float own = 0.0f;  // the sum of group c
#pragma unroll
        for (int j = 0; j < W; ++j) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[j][i] *= factor;
                sum += x[j][i];
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (j == c) own = sum;
            const int chunk = 4 * j + c;
            *reinterpret_cast<uint4*>(tile + (chunk >> 3) * Shape<D>::ATOM + swizzle128(r, chunk & 7)) =
                make_uint4(pack_f16(x[j][0], x[j][4]), pack_f16(x[j][1], x[j][5]), pack_f16(x[j][2], x[j][6]), pack_f16(x[j][3], x[j][7]));
        }
        // group c: high, high, low, low against the keys' high, low, high, low
        own *= 0.015625f;
        const uint32_t high = pack_f16(own, own);
        const float rest = own - __low2float(*reinterpret_cast<const __half2*>(&high));
        *reinterpret_cast<uint2*>(tile + Shape<D>::ATOMS * Shape<D>::ATOM + (c >> 1) * 2048 + (r >> 3) * 128 + (r & 7) * 16 + (c & 1) * 8) =
            c < W ? make_uint2(high, pack_f16(rest, rest)) : make_uint2(0u, 0u);
        if (c == 0) {
            l.scales[index * 256 + rr] = p.scale / factor;
            l.minus_lse[index * 256 + rr] = -INFINITY;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// tcgen05 with fp16 operands
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t idesc_f16(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

// MMAs and commits for a whole warp that has come here together; the lane with `leads` issues.  (The instructions take their
// operands from the warp's uniform registers; in code that one lane runs by itself the compiler brings them there value
// by value, and an MMA took 120 cycles to issue, however narrow.)  Descriptors by their lower halves: the upper ones are
// the same for all operands of a kind.
__device__ __forceinline__ void mma_from_smem(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, uint32_t accumulate, uint32_t leads) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(accumulate), "r"(leads)
        : "memory");
}

// A from tensor memory: row = lane, a column holds two elements of K.
__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, uint32_t accumulate, uint32_t leads) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(accumulate), "r"(leads)
        : "memory");
}

__device__ __forceinline__ void commit_warp(uint64_t* bar, uint32_t leads) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(leads)
        : "memory");
}

__device__ __forceinline__ void tmem_store_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_store_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// K-major without swizzle, 128 rows x 16 elements: eight rows x 16 bytes lie together, the second eight elements 2 KB further.
__device__ __forceinline__ uint64_t desc_extra(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(2048 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}

template <int N>
__device__ __forceinline__ void named_barrier(int id) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

// All of an SM's tensor memory for this block: the same warp gives it back (tmem_dealloc).
__device__ __forceinline__ void tensor_memory_begin(uint32_t* base) { tmem_alloc(base, 512); }

// A cached row's keys on their way to being an operand.
template <int D>
struct KeyRow {
    static constexpr int W = D / 32;
    uint32_t word[4 * W], scale[W];

    __device__ __forceinline__ void fetch(const PackedCache& cache, uint32_t at, bool there) {
#pragma unroll
        for (int c = 0; c < W; ++c) {
            const uint4 a = there ? reinterpret_cast<const uint4*>(cache.k_codes)[(size_t)at * W + c] : make_uint4(0, 0, 0, 0);
            word[4 * c] = a.x, word[4 * c + 1] = a.y, word[4 * c + 2] = a.z, word[4 * c + 3] = a.w;
            scale[c] = there ? cache.k_scales[(size_t)at * W + c] : 0u;
        }
    }
    __device__ __forceinline__ float top() const {
        float t = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) t = fmaxf(t, fmaxf(8.0f * packed_scale(scale[j]), fabsf(fmaf(8.0f, packed_scale(scale[j]), packed_least(scale[j])))));
        return t;
    }
    // Row t of the operand at `to`, times f.
    __device__ __forceinline__ void store(unsigned char* to, int t, float f) {
        using S = Shape<D>;
        __half2 s2[W];
#pragma unroll
        for (int j = 0; j < W; ++j) s2[j] = __float2half2_rn(packed_scale(scale[j]) * f);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {  // the words of quarter c, which then make room for the next quarter's
#pragma unroll
            for (int j = 0; j < W; ++j) {
                uint32_t x[4];
                code_pairs<8>(word[j], x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&x[e]), s2[j]);
                    x[e] = *reinterpret_cast<const uint32_t*>(&v);
                }
                const int chunk = 4 * j + c;
                *reinterpret_cast<uint4*>(to + (j >> 1) * S::ATOM + swizzle128(t, chunk & 7)) = make_uint4(x[0], x[1], x[2], x[3]);
            }
#pragma unroll
            for (int i = 0; i < 3 * W; ++i) word[i] = word[i + W];
        }
#pragma unroll
        for (int j = 0; j < 4; j += 2) {  // middles over 1 / 64: high, low, high, low of two groups
            uint32_t x[2] = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (j + e < W) {
                    const uint32_t sc = scale[j + e < W ? j + e : 0];
                    const float mid = fmaf(8.0f, packed_scale(sc), packed_least(sc)) * f * 64.0f;
                    const float high = __half2float(__float2half_rn(mid));
                    x[e] = pack_f16(high, mid - high);
                }
            *reinterpret_cast<uint4*>(to + S::ATOMS * S::ATOM + (j >> 1) * 2048 + (t >> 3) * 128 + (t & 7) * 16) = make_uint4(x[0], x[0], x[1], x[1]);
        }
    }
};

// Exponent (biased) of a block's greatest number, within what both of these have: the power of two that brings it between 2^7 and
// 2^8, and the way back.
__device__ __forceinline__ uint32_t top_exponent(float top) { return min(max(__float_as_uint(top) >> 23, 8u), 254u); }
__device__ __forceinline__ float into_range(uint32_t e) { return __uint_as_float((261u - e) << 23); }
__device__ __forceinline__ float out_of_range(uint32_t e) { return __uint_as_float((e - 7u) << 23); }

// The scores of operand a's rows against operand b's from `b_row` (a multiple of 8) on, into tensor memory; for a whole warp.
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t d, uint32_t a, uint32_t b, int b_row, uint32_t idesc, uint32_t leads) {
    using S = Shape<D>;
    const uint64_t da = umma_desc_k_major_sw128(a), db = umma_desc_k_major_sw128(b + 128 * b_row);
    const uint32_t a0 = (uint32_t)da, b0 = (uint32_t)db, high = (uint32_t)(da >> 32);
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
        const uint32_t next = (x >> 2) * (S::ATOM >> 4) + 2 * (x & 3);  // the next 64 columns, 32 bytes along the row
        mma_from_smem(d, a0 + next, b0 + next, high, idesc, x > 0 ? 1u : 0u, leads);
    }
    const uint64_t ea = desc_extra(a + S::ATOMS * S::ATOM), eb = desc_extra(b + S::ATOMS * S::ATOM + 16 * b_row);
    mma_from_smem(d, (uint32_t)ea, (uint32_t)eb, (uint32_t)(ea >> 32), idesc, 1u, leads);
}

// Of 32 rows from `row` on, those in [lo, hi).
__device__ __forceinline__ uint32_t rows_within(int row, int lo, int hi) {
    const int from = max(lo - row, 0), to = min(hi - row, 32);
    return from >= to ? 0u : (0xffffffffu >> (32 - (to - from))) << from;
}

// What the converting warps say of a block.
template <int W>
struct Info {
    float k_unit, v_unit;  // what a product of keys, of values is times
    uint32_t there[4];     // rows that have a page and lie before the end
    uint32_t any_bad, bad[W][4];  // groups of values that are not finite, by row
};

// A pair's blocks first .. first + count - 1 for one kv head.
struct Job {
    int pair, head, first, count, shared, begin_part, last_part, place;
};

// The jobs of a CTA, in order; the same for every thread of it.
struct Jobs {
    int u, stop, pair, direct;
    Deal deal;
    const int* before;
    int n_pairs, kv_heads, grid;
    const Pair* pairs;

    __device__ __forceinline__ bool next(Job& j) {
        if (u >= stop) return false;
        if (direct) {
            j.pair = u / kv_heads, j.head = u % kv_heads, j.shared = 0, j.first = pairs[j.pair].first, j.count = pairs[j.pair].count;
            ++u;
            return true;
        }
        for (int step = TABLE / 2; step; step >>= 1)
            if (pair + step < n_pairs && before[pair + step] <= u) pair += step;
        const Pair q = pairs[pair];
        const int rel = u - before[pair], n = deal.runs ? q.count : deal.pieces(q.count);
        j.pair = pair, j.head = rel / n;
        const int i = rel - j.head * n;
        int from;
        if (deal.runs) {
            from = i, j.count = min(q.count - i, stop - u);
            j.begin_part = deal.block_of(u - i), j.last_part = deal.block_of(u - i + q.count - 1);
            u += j.count;
        } else {
            from = (int)((long long)i * q.count / n), j.count = (int)((long long)(i + 1) * q.count / n) - from;
            j.begin_part = (int)blockIdx.x - i, j.last_part = j.begin_part + n - 1;
            u = stop;
        }
        j.first = q.first + from;
        j.shared = j.count < q.count;
        j.place = deal.place(blockIdx.x, j.begin_part);
        return true;
    }
};

// Which of a job's blocks a tile of its pair works on.
struct Active {
    int from, to;  // counted from the job's first block
    __device__ __forceinline__ Active(const PackedAttention& p, const Request& rq, const Pair& pair, const Job& j, int tile) {
        const int first = pair.index * 2 * ROWS + tile * ROWS, last = min(first + ROWS, rq.rows) - 1;
        from = to = 0;
        if (first > last) return;
        rq.blocks(p, first, last, from, to);
        from = min(max(from - j.first, 0), j.count);
        to = max(min(to - j.first, j.count), from);
    }
};

template <int D>
__global__ void __launch_bounds__(THREADS, 1) packed_prefill_kernel(const PackedAttention p, const Layout l, int* counters, int sms, int pair_room) {
    using S = Shape<D>;
    constexpr int W = S::W;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_ready[2], p_ready[2], pv_done[2];
    __shared__ uint32_t tmem_base;
    __shared__ Info<W> infos[INFOS];
    __shared__ float tops[2][2][CONVERT];
    __shared__ int before[TABLE + 1], last_here;
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* q_smem = smem;                       // two tiles
    unsigned char* k_smem = smem + 2 * S::OPERAND;      // two blocks
    unsigned char* v_smem = smem + 4 * S::OPERAND;      // two blocks
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    const int n_pairs = l.before[pair_room + 1], units = l.before[pair_room + 2];
    Jobs jobs = {0, 0, 0, pair_room > TABLE, Deal(max(units, 1), sms, l.before[pair_room + 3]), before, n_pairs, p.cache.kv_heads, (int)gridDim.x, l.pairs};
    if (jobs.direct) {
        jobs.u = blockIdx.x, jobs.stop = min(jobs.u + 1, n_pairs * p.cache.kv_heads);
    } else {
        const int total = l.before[n_pairs];
        jobs.u = jobs.deal.runs ? jobs.deal.begin_of(min((int)blockIdx.x, jobs.deal.blocks)) : (int)blockIdx.x;
        jobs.stop = jobs.deal.runs ? jobs.deal.begin_of(min((int)blockIdx.x + 1, jobs.deal.blocks)) : min((int)blockIdx.x + 1, total);
    }
    if (jobs.u >= jobs.stop || n_pairs == 0) {
        pdl_launch_dependents();
        return;
    }
    if (!jobs.direct)
        for (int i = threadIdx.x; i <= n_pairs; i += THREADS) before[i] = l.before[i];
    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], CONVERT);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], CONVERT);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_ready[i], 1);
            mbar_init(&p_ready[i], SOFTMAX / 2);
            mbar_init(&pv_done[i], 1);
        }
        mbar_fence_init();
    }
    if (warp == SOFTMAX + CONVERT) tensor_memory_begin(&tmem_base);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    pdl_launch_dependents();  // (only now: a dependent that took tensor memory first would wait for this grid, which would wait for it)
    const uint32_t tmem = tmem_base;  // scores (and weights) of tile t at 128 t, outputs at 256 + D t
    bool ok = true;  // a wait that ran out: everybody carries on without waiting, so that the named barriers are all met
    Job job;

    if (warp < SOFTMAX) {
        // ------------------------------------------------------------------ softmax: a thread a row
        const int t = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, my_s = tmem + 128 * t + lanes, my_o = tmem + 256 + D * t + lanes;
        int n = 0, done = 0;  // blocks of the CTA so far; of this tile
        while (jobs.next(job)) {
            const Pair pair = l.pairs[job.pair];
            const Request rq(pair);
            const Active act(p, rq, pair, job, t);
            const int row = pair.index * 2 * ROWS + t * ROWS + r;
            const bool valid = row < rq.rows;
            int lo = 0, hi = 0;
            if (valid) rq.sees(p, row, lo, hi);
            const size_t place = ((size_t)job.pair * p.cache.kv_heads + job.head) * 256 + t * ROWS + r;
            const float qs = l.scales[place];
            float* my_lse = l.minus_lse + place;
            float m = -FLT_MAX, sum = 0.0f, v_unit = 1.0f;
            uint32_t bad = 0;
            for (int i = act.from; i < act.to; ++i, ++done) {
                const Info<W>& info = infos[(n + i) % INFOS];
                ok = ok && mbar_wait(&s_ready[t], done & 1, p.status, 84);
                __syncwarp();
                tcgen05_fence_after();
                const int key0 = (job.first + i) * BLOCK;
                // Above nought: rows that are not seen stand as minus infinity, which times nought would be NaN.  A product below the
                // normal range (small queries beside keys of nought, a scale of nought) makes scores of nought all the same.
                const float unit = fmaxf(qs * info.k_unit, FLT_MIN);
                const bool whole = key0 >= lo && key0 + BLOCK <= hi && (info.there[0] & info.there[1] & info.there[2] & info.there[3]) == 0xffffffffu;
                if (info.any_bad)  // (rare) which of this row's outputs a value that is not finite reaches
                    for (int k = 0; k < BLOCK; ++k)
                        if (key0 + k >= lo && key0 + k < hi)
#pragma unroll
                            for (int j = 0; j < W; ++j) bad |= (info.bad[j][k >> 5] >> (k & 31) & 1) << j;
                const bool first = i == act.from;
                const float v_now = info.v_unit;
                // The scores are read twice: for their maximum, and for the weights, which go back over them.  Loops that
                // are not unrolled: three kinds of warps share the SM's instruction cache (with the weights of a row held in
                // registers until its maximum is known, every fourth stall was for instructions).
                float top = -INFINITY;
#pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                    uint32_t sc[32];
                    tmem_load_32x32(my_s + 32 * h, sc);
                    tmem_load_wait();
                    if (!whole) {
                        const uint32_t seen = info.there[h] & rows_within(key0 + 32 * h, lo, hi);
#pragma unroll
                        for (int c = 0; c < 32; ++c) sc[c] = seen & 1u << c ? sc[c] : 0xff800000u;
                    }
#pragma unroll
                    for (int c = 0; c < 32; c += 2) top = fmaxf(top, fmaxf(__uint_as_float(sc[c]), __uint_as_float(sc[c + 1])));
                }
                top *= unit;
                const bool moved = !first && v_now != v_unit;  // (the same for all rows)
                if (__any_sync(0xffffffffu, top > m + 8.0f) || moved) {
                    const float now = top > m + 8.0f ? top : m;
                    float f = exp2_fast(m - now);
                    m = now;
                    sum *= f;
                    if (!first) {  // what has been added up so far follows
                        if (moved) f *= v_unit / v_now;
                        ok = ok && mbar_wait(&pv_done[t], (done - 1) & 1, p.status, 85);
                        __syncwarp();
                        tcgen05_fence_after();
#pragma unroll 1
                        for (int h = 0; h < D / 32; ++h) {
                            uint32_t o[32];
                            tmem_load_32x32(my_o + 32 * h, o);
                            tmem_load_wait();
#pragma unroll
                            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
                            tmem_store_32x32(my_o + 32 * h, o);
                        }
                    }
                }
                v_unit = v_now;
                const float minus = RAISE - m;
                float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                    uint32_t sc[32], packed[16];
                    tmem_load_32x32(my_s + 32 * h, sc);
                    tmem_load_wait();
                    if (!whole) {
                        const uint32_t seen = info.there[h] & rows_within(key0 + 32 * h, lo, hi);
#pragma unroll
                        for (int c = 0; c < 32; ++c) sc[c] = seen & 1u << c ? sc[c] : 0xff800000u;
                    }
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const float e0 = exp2_fast(fmaf(__uint_as_float(sc[c]), unit, minus)), e1 = exp2_fast(fmaf(__uint_as_float(sc[c + 1]), unit, minus));
                        part[(c >> 1) & 3] += e0 + e1;
                        packed[c >> 1] = pack_f16(e0, e1);
                    }
                    tmem_store_32x16(my_s + 16 * h, packed);
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
                tmem_store_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[t]);
            }
            n += job.count;
            // the rows' outputs, or the pair's part of them
            const bool any = act.to > act.from;
            if (any) {
                ok = ok && mbar_wait(&pv_done[t], (done - 1) & 1, p.status, 86);
                __syncwarp();
                tcgen05_fence_after();
            }
            float* part = job.shared ? l.parts + (size_t)job.place * (D + 2) * 256 + t * ROWS + r : nullptr;
            const int token = rq.t0 + row / p.group, qh = job.head * p.group + row % p.group;
            bf16* out = (bf16*)p.out + (size_t)token * p.ldo + (size_t)qh * D;
            // Outputs of 32 columns in their order of columns (column 8 (g W / 2 + i) + 2 e + h is element 32 (2 i + h) + 4 g + e) to their places
            const auto store = [&](int h, const float (&v)[32]) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    // eight neighbours: D = 128: of group b, from 8 h on; D = 64: of group b / 2, from 16 h + 8 (b % 2) on
                    const int j = W == 4 ? b : b >> 1, from = W == 4 ? 8 * h : 16 * h + 8 * (b & 1);
                    float x[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int gl = k >> 2, e = k & 3;
                        x[k] = W == 4 ? v[(gl * 2 + (j >> 1)) * 8 + 2 * e + (j & 1)] : v[(2 * (b & 1) + gl) * 8 + 2 * e + j];
                        if (bad >> j & 1) x[k] = NAN;
                    }
                    bf16* to = out + 32 * j + from;
                    if (p.out_aligned)
                        *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
                    else
#pragma unroll
                        for (int k = 0; k < 8; ++k) to[k] = from_float<bf16>(x[k]);
                }
            };
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int h = 0; h < D / 32; ++h) {
                uint32_t o[32] = {};
                if (any) {
                    tmem_load_32x32(my_o + 32 * h, o);
                    tmem_load_wait();
                }
                if (part) {
                    if (any) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            // (a group of values that is not finite goes on as such in the part)
                            const int cc = 32 * h + c, j = 2 * ((cc >> 3) % (W / 2)) + (cc & 1);
                            part[(size_t)cc * 256] = bad >> j & 1 ? NAN : __uint_as_float(o[c]) * v_unit;
                        }
                    }
                } else if (valid) {
                    float v[32];
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(o[c]) * (v_unit * inv);
                    store(h, v);
                }
            }
            tcgen05_fence_before();
            if (!part) {
                if (valid) my_lse[0] = sum == 0.0f ? -INFINITY : -(m - RAISE + log2f(sum));
                continue;
            }
            part[(size_t)D * 256] = m;
            part[(size_t)(D + 1) * 256] = sum;
            __threadfence();
            named_barrier<SOFTMAX * 32>(2);
            if (threadIdx.x == 0) {
                int* counter = counters + (size_t)job.pair * p.cache.kv_heads + job.head;
                last_here = atomicAdd(counter, 1) == job.last_part - job.begin_part;
                if (last_here) *counter = 0;  // for the next launch
                __threadfence();
            }
            named_barrier<SOFTMAX * 32>(2);
            if (!last_here || !valid) continue;
            // the last CTA of the pair joins its parts, in their order
            const auto at = [&](int i) { return l.parts + (size_t)jobs.deal.place(i, job.begin_part) * (D + 2) * 256 + t * ROWS + r; };
            m = -FLT_MAX, sum = 0.0f, bad = 0;
            for (int i = job.begin_part; i <= job.last_part; ++i) m = fmaxf(m, __ldcg(at(i) + D * 256));
            for (int i = job.begin_part; i <= job.last_part; ++i) sum += exp2_fast(__ldcg(at(i) + D * 256) - m) * __ldcg(at(i) + (D + 1) * 256);
            const float share = sum == 0.0f ? 0.0f : 1.0f / sum;
            for (int h = 0; h < D / 32; ++h) {
                float v[32] = {};
                for (int i = job.begin_part; i <= job.last_part; ++i) {
                    const float mi = __ldcg(at(i) + D * 256), f = exp2_fast(mi - m) * share;
                    // nothing that the row sees: a part that was not written (scores of NaN alone leave the maximum there too, not the sum)
                    if (mi == -FLT_MAX && __ldcg(at(i) + (D + 1) * 256) == 0.0f) continue;
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[c] += f * __ldcg(at(i) + (size_t)(32 * h + c) * 256);
                }
                store(h, v);
            }
            my_lse[0] = sum == 0.0f ? -INFINITY : -(m - RAISE + log2f(sum));
        }
    } else if (warp < SOFTMAX + CONVERT) {
        // ------------------------------------------------------------------ operands: a thread a cached row of each block
        const int t = threadIdx.x - SOFTMAX * 32, w = warp - SOFTMAX;
        int n = 0;
        while (jobs.next(job)) {
            const Pair pair = l.pairs[job.pair];
            const Request rq(pair);
            const int* table = p.tables + (size_t)pair.seq * p.width;
            int lo, end;
            rq.sees(p, min((pair.index + 1) * 2 * ROWS, rq.rows) - 1, lo, end);
            KeyRow<D> key;
            uint32_t vw[4 * W], vs[W];
            bool there = false;
            const auto fetch = [&](int i) {  // this thread's row of the job's block i
                const int row = (job.first + i) * BLOCK + t, block = p.block_of(row);
                const int page = row < end ? page_of(p, table, block) : -1;
                there = page >= 0;
                const uint32_t at = there ? p.row_of(page, job.head, row, block) : 0;
                key.fetch(p.cache, at, there);
#pragma unroll
                for (int c = 0; c < W; ++c) {
                    const uint4 b = there ? reinterpret_cast<const uint4*>(p.cache.v_codes)[(size_t)at * W + c] : make_uint4(0, 0, 0, 0);
                    vw[4 * c] = b.x, vw[4 * c + 1] = b.y, vw[4 * c + 2] = b.z, vw[4 * c + 3] = b.w;
                    vs[c] = there ? p.cache.v_scales[(size_t)at * W + c] : 0u;
                }
            };
            float v_top = 0.0f;
            fetch(0);
            for (int i = 0; i < job.count; ++i, ++n) {
                const int stage = n & 1;
                Info<W>& info = infos[n % INFOS];
                float kt = key.top(), vt = 0.0f;
                uint32_t mine_bad = 0;
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    if (packed_not_finite(vs[j])) {
                        mine_bad |= 1u << j;
                        vs[j] = 0;
                    }
                    vt = fmaxf(vt, fmaxf(8.0f * packed_scale(vs[j]), fabsf(fmaf(8.0f, packed_scale(vs[j]), packed_least(vs[j])))));
                }
                kt = warp_max(kt);
                vt = warp_max(vt);
                if (lane == 0) {
                    tops[n & 1][0][w] = kt;
                    tops[n & 1][1][w] = vt;
                }
                // stage and info are free: the block two before has been multiplied, so the one four before has been weighed
                ok = ok && (n < 2 || mbar_wait(&k_empty[stage], ((n >> 1) - 1) & 1, p.status, 87));
                named_barrier<CONVERT * 32>(1);
#pragma unroll
                for (int x = 0; x < CONVERT; ++x) {
                    kt = fmaxf(kt, tops[n & 1][0][x]);
                    vt = fmaxf(vt, tops[n & 1][1][x]);
                }
                v_top = fmaxf(v_top, vt);
                const uint32_t ke = top_exponent(kt), ve = top_exponent(v_top);
                const float vf = into_range(ve);
                const uint32_t here = __ballot_sync(0xffffffffu, there);
                uint32_t bad_rows = 0;
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const uint32_t b = __ballot_sync(0xffffffffu, mine_bad >> j & 1);
                    bad_rows |= b;
                    if (lane == 0) info.bad[j][w] = b;
                }
                if (w == 0 && lane == 0) {
                    info.k_unit = out_of_range(ke);
                    info.v_unit = out_of_range(ve);
                }
                if (lane == 0) info.there[w] = here;
                // (any_bad: every warp sets or clears it for its own rows, so in four places)
                if (lane == 0) reinterpret_cast<volatile unsigned char*>(&info.any_bad)[w] = bad_rows != 0;
                key.store(k_smem + stage * S::OPERAND, t, into_range(ke));
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[stage]);
                ok = ok && (n < 2 || mbar_wait(&v_empty[stage], ((n >> 1) - 1) & 1, p.status, 88));
                unsigned char* vd = v_smem + stage * S::V_BYTES;
                __half2 s2[W / 2], mid[W / 2];
#pragma unroll
                for (int i2 = 0; i2 < W / 2; ++i2) {
                    const float s0 = packed_scale(vs[2 * i2]) * vf, s1 = packed_scale(vs[2 * i2 + 1]) * vf;
                    s2[i2] = __floats2half2_rn(s0, s1);
                    mid[i2] = __floats2half2_rn(fmaf(8.0f, s0, packed_least(vs[2 * i2]) * vf), fmaf(8.0f, s1, packed_least(vs[2 * i2 + 1]) * vf));
                }
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
#pragma unroll
                    for (int j = 0; j < W; ++j) {  // chunk g W / 2 + i2
                        const int chunk = c * W + j;
                        uint32_t x[4];
                        code_pairs<8>(vw[j], x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&x[e]), s2[j % (W / 2)], mid[j % (W / 2)]);
                            x[e] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        *reinterpret_cast<uint4*>(vd + (chunk >> 3) * S::ATOM + swizzle128(t, chunk & 7)) = make_uint4(x[0], x[1], x[2], x[3]);
                    }
#pragma unroll
                    for (int x = 0; x < 3 * W; ++x) vw[x] = vw[x + W];
                }
                if (i + 1 < job.count) fetch(i + 1);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[stage]);
            }
        }
    } else {
        // ------------------------------------------------------------------ the warp that issues
        const uint32_t leads = lane == 0, idesc_s = idesc_f16(ROWS, BLOCK), idesc_o = idesc_f16(ROWS, D) | (1u << 16);  // V is MN-major (rows along K)
        // (What there is one of for each tile stands in two names and is chosen from: an array with an index of the loop would lie in local
        // memory, and this warp's few instructions are the pace of the block.)
        int n = 0, jobs_done = 0;        // blocks, jobs
        int weighed0 = 0, weighed1 = 0;  // blocks of each tile
        const auto weighed = [&](int t) { return t ? weighed1 : weighed0; };
        while (jobs.next(job)) {
            const Pair pair = l.pairs[job.pair];
            const Request rq(pair);
            const Active act0(p, rq, pair, job, 0), act1(p, rq, pair, job, 1);
            const auto has = [&](int t, int i) { return i >= (t ? act1.from : act0.from) && i < (t ? act1.to : act0.to); };
            // the queries of the job before are read no more when its last products are done
            for (int t = 0; t < 2; ++t)
                if (weighed(t)) ok = ok && mbar_wait(&pv_done[t], (weighed(t) - 1) & 1, p.status, 89);
            if (ok && lane == 0) {
                mbar_expect_tx(&q_full, 2 * S::OPERAND);
                bulk_load(smem_u32(q_smem), l.queries + ((size_t)job.pair * p.cache.kv_heads + job.head) * 2 * S::OPERAND, 2 * S::OPERAND, &q_full);
            }
            __syncwarp();
            ok = ok && mbar_wait(&q_full, jobs_done & 1, p.status, 90);
            ++jobs_done;
            const auto scores = [&](int t, int stage) {
                tcgen05_fence_after();
                issue_scores<D>(tmem + 128 * t, smem_u32(q_smem + t * S::OPERAND), smem_u32(k_smem + stage * S::OPERAND), 0, idesc_s, leads);
                commit_warp(&s_ready[t], leads);
            };
            ok = ok && mbar_wait(&k_full[n & 1], (n >> 1) & 1, p.status, 91);
            for (int t = 0; t < 2; ++t)
                if (has(t, 0) && ok) scores(t, n & 1);
            commit_warp(&k_empty[n & 1], leads);
#pragma unroll 1
            for (int i = 0; i < job.count; ++i, ++n) {
                const int stage = n & 1;
                const bool more = i + 1 < job.count;
                ok = ok && mbar_wait(&v_full[stage], (n >> 1) & 1, p.status, 93) && (!more || mbar_wait(&k_full[stage ^ 1], ((n + 1) >> 1) & 1, p.status, 94));
#pragma unroll 1
                for (int t = 0; t < 2; ++t) {
                    if (has(t, i)) {
                        ok = ok && mbar_wait(&p_ready[t], weighed(t) & 1, p.status, 92);
                        if (ok) {
                            tcgen05_fence_after();
                            const uint64_t v = umma_desc_mn_major_sw128(smem_u32(v_smem + stage * S::V_BYTES), S::ATOM);
#pragma unroll
                            for (int x = 0; x < BLOCK / 16; ++x)
                                mma_from_tmem(tmem + 256 + D * t, tmem + 128 * t + 8 * x, (uint32_t)v + x * (2048 >> 4), (uint32_t)(v >> 32), idesc_o,
                                              i > (t ? act1.from : act0.from) || x > 0 ? 1u : 0u, leads);
                            commit_warp(&pv_done[t], leads);
                        }
                        // the next scores come where these weights stand
                        if (has(t, i + 1)) ok = ok && mbar_wait(&pv_done[t], weighed(t) & 1, p.status, 95);
                        weighed0 += t == 0, weighed1 += t == 1;
                    }
                    if (has(t, i + 1) && ok) scores(t, stage ^ 1);
                }
                commit_warp(&v_empty[stage], leads);
                if (more) commit_warp(&k_empty[stage ^ 1], leads);
            }
        }
        for (int t = 0; t < 2; ++t)  // nothing is in flight when the tensor memory goes back
            if (weighed(t)) mbar_wait(&pv_done[t], (weighed(t) - 1) & 1, p.status, 103);
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == SOFTMAX + CONVERT) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Weights of the cached rows:  w[key] (+)= sum over the request's query rows of 2^(s - lse), S^T = K Q^T so that a thread has a key
// and adds up along its row: no sum crosses threads, and the order is that of the queries.  A CTA takes 256 keys of one
// request and kv head (two blocks, each its own operand, formed once) and goes through the query tiles that see any of
// them; every tile meets both blocks.  A thread has the same key of both blocks and one half of a tile's rows, so that what it reads of a row (scale
// and sum, from shared memory, every lane the same) serves two keys (one key a thread: 586 us
// with the attention, two: 562).  512 tokens after 32,768 rows (28 / 4 heads of 128) 233 us; exponential unit 47 % busy, tensor pipe 26 %.
constexpr int W_KEYS = 2, W_STAGES = 3, W_THREADS = (4 * W_KEYS + 1) * 32;

template <int D>
struct WeightShape {
    static constexpr int STAGE = Shape<D>::OPERAND + 1024;  // a query tile, its scales and minus its sums
    static constexpr int SMEM = W_KEYS * Shape<D>::OPERAND + W_STAGES * STAGE + 1024;
};

template <int D>
__global__ void __launch_bounds__(W_THREADS, 1) packed_prefill_weights_kernel(const PackedAttention p, const Layout l) {
    using S = Shape<D>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t q_full[W_STAGES], s_ready[2], s_free[2], k_ready;
    __shared__ uint32_t tmem_base;
    __shared__ float tops[W_KEYS][4], units[W_KEYS], sums[W_KEYS][BLOCK];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* q_smem = smem + W_KEYS * S::OPERAND;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.y, seq = blockIdx.z;
    pdl_wait();
    const Request rq(p, seq);
    const int key0 = blockIdx.x * W_KEYS * BLOCK, end = min(max(0, min(rq.start + rq.rows / p.group, rq.limit)), p.max_rows);
    const int slot = slot_of(p, seq);
    if (rq.rows <= p.few || key0 >= end || slot < 0) {
        pdl_launch_dependents();
        return;
    }
    // the tiles of the query rows that see any of these keys
    const long long first_row = (long long)max(key0 - rq.start, 0) * p.group;
    const long long last_row = p.window > 0 ? ((long long)key0 + W_KEYS * BLOCK - 1 - rq.start + p.window) * p.group : rq.rows;
    const int from = (int)(min(first_row, (long long)rq.rows) / ROWS);
    int to = (int)((max(min(last_row, (long long)rq.rows), 0ll) + ROWS - 1) / ROWS);
    if (threadIdx.x == 0) {
        for (int i = 0; i < W_STAGES; ++i) mbar_init(&q_full[i], 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_ready[i], 1);
            mbar_init(&s_free[i], 4 * W_KEYS);
        }
        mbar_init(&k_ready, 4 * W_KEYS);
        mbar_fence_init();
    }
    if (warp == 4 * W_KEYS) tensor_memory_begin(&tmem_base);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = tmem_base;  // scores of block k, every other tile, at 256 k + 128 (tile % 2)
    const size_t first_pair = l.first_pair[seq];
    to = min(to, max(2 * (l.room - (int)first_pair), from));
    bool ok = true;
    if (warp < 4 * W_KEYS) {
        const int k = warp >> 2, t = (warp & 3) * 32 + lane, row = key0 + k * BLOCK + t, block = p.block_of(row);
        const int page = row < end ? page_of(p, p.tables + (size_t)seq * p.width, block) : -1;
        KeyRow<D> key;
        key.fetch(p.cache, page >= 0 ? p.row_of(page, head, row, block) : 0, page >= 0);
        float top = warp_max(key.top());
        if (lane == 0) tops[k][warp & 3] = top;
        named_barrier<128>(1 + k);
#pragma unroll
        for (int x = 0; x < 4; ++x) top = fmaxf(top, tops[k][x]);
        const uint32_t e = top_exponent(top);
        key.store(smem + k * S::OPERAND, t, into_range(e));
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_ready);
        if (t == 0) units[k] = out_of_range(e);
        named_barrier<256>(3);
        // from here on: key t of both blocks, rows 64 k .. 64 k + 63 of the tiles; the query rows from[x] .. to[x] - 1 see the key of block x
        float unit[W_KEYS], total[W_KEYS][2] = {};
        int seen_from[W_KEYS], seen_to[W_KEYS];
#pragma unroll
        for (int x = 0; x < W_KEYS; ++x) {
            const int row = key0 + x * BLOCK + t;
            const long long reach = p.window > 0 ? ((long long)row - rq.start + p.window) * p.group : rq.rows;
            unit[x] = units[x];
            seen_from[x] = (int)min((long long)max(row - rq.start, 0) * p.group, (long long)rq.rows);
            seen_to[x] = (int)max(min(reach, (long long)rq.rows), 0ll);
            if (row >= end || page_of(p, p.tables + (size_t)seq * p.width, p.block_of(row)) < 0) seen_from[x] = seen_to[x] = 0;
        }
        const uint32_t my_s = tmem + 64 * k + ((uint32_t)((warp & 3) * 32) << 16);
        for (int i = from, n = 0; i < to; ++i, ++n) {
            const float4* scales = reinterpret_cast<const float4*>(q_smem + (n % W_STAGES) * WeightShape<D>::STAGE + S::OPERAND) + 16 * k;
            ok = ok && mbar_wait(&s_ready[n & 1], (n >> 1) & 1, p.status, 96);
            // (the copies have landed before the scores were formed from them: the wait costs nothing, and makes them visible here)
            ok = ok && mbar_wait(&q_full[n % W_STAGES], (n / W_STAGES) & 1, p.status, 97);
            __syncwarp();
            tcgen05_fence_after();
            const int r0 = i * ROWS + 64 * k;
            const bool whole = __all_sync(0xffffffffu, r0 >= max(seen_from[0], seen_from[1]) && r0 + 64 <= min(seen_to[0], seen_to[1]));
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
                uint32_t sc[W_KEYS][16];
                tmem_load_32x16(my_s + 128 * (n & 1) + 16 * h, sc[0]);
                tmem_load_32x16(my_s + 256 + 128 * (n & 1) + 16 * h, sc[1]);
                float4 a[4], b[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) a[c] = scales[4 * h + c], b[c] = scales[32 + 4 * h + c];
                tmem_load_wait();
#pragma unroll
                for (int x = 0; x < W_KEYS; ++x) {
                    float w[16];  // the weights' logarithms
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        w[4 * c] = fmaf(__uint_as_float(sc[x][4 * c]) * unit[x], a[c].x, b[c].x);
                        w[4 * c + 1] = fmaf(__uint_as_float(sc[x][4 * c + 1]) * unit[x], a[c].y, b[c].y);
                        w[4 * c + 2] = fmaf(__uint_as_float(sc[x][4 * c + 2]) * unit[x], a[c].z, b[c].z);
                        w[4 * c + 3] = fmaf(__uint_as_float(sc[x][4 * c + 3]) * unit[x], a[c].w, b[c].w);
                    }
                    if (!whole) {
                        const int first = seen_from[x] - r0 - 16 * h, last = seen_to[x] - r0 - 16 * h;
#pragma unroll
                        for (int c = 0; c < 16; ++c) w[c] = c >= first && c < last ? w[c] : -INFINITY;
                    }
#pragma unroll
                    for (int c = 0; c < 16; ++c) total[x][c & 1] += exp2_fast(w[c]);
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[n & 1]);
        }
        if (k == 1) {
#pragma unroll
            for (int x = 0; x < W_KEYS; ++x) sums[x][t] = total[x][0] + total[x][1];
        }
        named_barrier<256>(3);
        if (k == 0) {
#pragma unroll
            for (int x = 0; x < W_KEYS; ++x) {
                const int row = key0 + x * BLOCK + t;
                if (row < end) {
                    float* w = p.weights + slot * p.slot_stride + (long long)head * p.head_stride + row;
                    const float sum = (total[x][0] + total[x][1]) + sums[x][t];
                    *w = p.add && row < rq.start ? *w + sum : sum;
                }
            }
        }
    } else {
        const uint32_t idesc = idesc_f16(BLOCK, ROWS), leads = lane == 0;
        const int tiles = to - from;
        const auto load = [&](int n) {
            if (lane) return;
            const int i = from + n;
            unsigned char* dst = q_smem + (n % W_STAGES) * WeightShape<D>::STAGE;
            uint64_t* bar = &q_full[n % W_STAGES];
            const size_t index = (first_pair + i / 2) * p.cache.kv_heads + head;
            mbar_expect_tx(bar, S::OPERAND + 2 * ROWS * 4);
            bulk_load(smem_u32(dst), l.queries + (index * 2 + (i & 1)) * S::OPERAND, S::OPERAND, bar);
            bulk_load(smem_u32(dst + S::OPERAND), l.scales + index * 256 + (i & 1) * ROWS, ROWS * 4, bar);
            bulk_load(smem_u32(dst + S::OPERAND + ROWS * 4), l.minus_lse + index * 256 + (i & 1) * ROWS, ROWS * 4, bar);
        };
        for (int n = 0; n < tiles && n < W_STAGES - 1; ++n) load(n);
        if (tiles > 0) ok = ok && mbar_wait(&k_ready, 0, p.status, 98);
        for (int n = 0; n < tiles; ++n) {
            ok = ok && mbar_wait(&q_full[n % W_STAGES], (n / W_STAGES) & 1, p.status, 99);
            if (n >= 2) ok = ok && mbar_wait(&s_free[n & 1], ((n >> 1) - 1) & 1, p.status, 100);
            if (ok) {
                tcgen05_fence_after();
#pragma unroll 1
                for (int k = 0; k < W_KEYS; ++k)
                    issue_scores<D>(tmem + 256 * k + 128 * (n & 1), smem_u32(smem + k * S::OPERAND), smem_u32(q_smem + (n % W_STAGES) * WeightShape<D>::STAGE), 0, idesc, leads);
                commit_warp(&s_ready[n & 1], leads);
            }
            // the place of the tile before this one, once both blocks have been through with it
            const int next = n + W_STAGES - 1;
            if (next < tiles) {
                if (n >= 1) ok = ok && mbar_wait(&s_free[(n - 1) & 1], ((n - 1) >> 1) & 1, p.status, 101);
                if (ok) load(next);
            }
        }
        if (!ok)  // a wait ran out: no copy may land after the block has gone
            for (int i = 0; i < W_STAGES; ++i) mbar_wait(&q_full[i], 0, p.status, 102);
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 4 * W_KEYS) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int D>
int prefill(const PackedAttention& p, const PrefillPlan& plan, int max_kv, void* scratch, int* counters, cudaStream_t st) {
    const Layout l = make_layout(scratch, D, plan.pairs, p.cache.kv_heads, p.seqs, plan.pairs > TABLE ? 0 : part_places(plan.grid, plan.sms));
    cudaError_t e = ferris_launch(packed_queries_kernel<D>, dim3(plan.pairs + 1, p.cache.kv_heads), dim3(256), 0, st, p, l, plan.sms);
    if (e != cudaSuccess) return (int)e;
    auto kernel = packed_prefill_kernel<D>;
    if (const int r = ferris_allow_dynamic_smem((const void*)kernel, Shape<D>::SMEM)) return r;
    e = ferris_launch(kernel, dim3(plan.grid), dim3(THREADS), Shape<D>::SMEM, st, p, l, counters, plan.sms, plan.pairs);
    if (e != cudaSuccess || !p.weights) return (int)e;
    auto weigh = packed_prefill_weights_kernel<D>;
    if (const int r = ferris_allow_dynamic_smem((const void*)weigh, WeightShape<D>::SMEM)) return r;
    const int keys = W_KEYS * BLOCK;
    return (int)ferris_launch(weigh, dim3((max_kv + keys - 1) / keys, p.cache.kv_heads, p.seqs), dim3(W_THREADS), WeightShape<D>::SMEM, st, p, l);
}

}  // namespace

PrefillPlan packed_prefill_plan(int head_dim, int seqs, int kv_heads, int group, int tokens, int max_q, int max_kv) {
    PrefillPlan q = {};
    q.sms = ferris_sm_count() > 0 ? ferris_sm_count() : 148;
    const long long rows = (long long)tokens * group, most = (long long)seqs * (((long long)max_q * group + 2 * ROWS - 1) / (2 * ROWS));
    const long long pairs = rows / (2 * ROWS) + seqs < most ? rows / (2 * ROWS) + seqs : most;  // every request may leave one part-filled
    q.pairs = (int)(pairs > 0 ? pairs : 1);
    // pieces: a pair may leave one that is not full; more pairs than are dealt out evenly: a CTA each
    q.grid = q.pairs > TABLE ? q.pairs * kv_heads : q.sms + q.pairs * kv_heads;
    const long long blocks = (long long)q.pairs * kv_heads * (max_kv / BLOCK + 2);
    if (q.pairs <= TABLE && q.grid > blocks) q.grid = (int)blocks;
    q.bytes = make_layout(nullptr, head_dim, q.pairs, kv_heads, seqs, q.pairs > TABLE ? 0 : part_places(q.grid, q.sms)).bytes;
    q.counters = q.pairs > TABLE ? 0 : (long long)q.pairs * kv_heads;
    return q;
}

int packed_prefill(const PackedAttention& p, const PrefillPlan& plan, int max_kv, void* scratch, int* counters, cudaStream_t stream) {
    return p.cache.head_dim == 64 ? prefill<64>(p, plan, max_kv, scratch, counters, stream) : prefill<128>(p, plan, max_kv, scratch, counters, stream);
}
