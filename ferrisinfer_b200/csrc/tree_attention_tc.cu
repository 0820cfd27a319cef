// Attention for trees of drafted tokens over the paged cache, bf16, on tcgen05: heads of 64 and 128, many query rows (who sees what, and how the work is
// dealt out: tree_attention.cuh).
//
// A block of 128 query rows goes over blocks of 128 cached rows (units):
//   S = Q K^T   128 x 128 x D, operands in shared memory (Q written once, K by TMA), sums in tensor memory
//   P = 2^(S scale - m), rounded to bf16 (eight bits, as the output has; sums take it unrounded), into tensor memory over the scores it came from
//   O = O + P V   P from tensor memory, V as TMA wrote it, sums in tensor memory over all units
// Two groups of four softmax warps, each with scores, maxima, sums and outputs of its own, so that the tensor core works for one while
// the other exponentiates; a thread has a row, so that nothing is exchanged.  Of up to 128 query rows each group goes over a share of its own, with a ring of
// stages, a TMA warp and an MMA warp of its own: one begins or ends an item while the other goes on.  Of more (WIDE) each has 128 rows of one item, and K and V are
// fetched once for both.
// m is the greatest score so far only up to 2^8: outputs are brought to a new m (read, multiplied, written back) where a score exceeds it by
// more than eight, which after the first units is rare; what is divided by in the end has the same m, so that nothing but the range of the weights changes.
// A TMA warp streams K and V through a ring of stages, ahead of the segment that is worked on; an MMA warp issues, in the order of the units,
// P V of a unit and then the scores of the next one (the tensor core keeps the order, so that these do not overwrite weights that are still read).
//
// Units that every node sees whole are worked off as they are.  In others scores that are not seen become nought weights; as nought times NaN is NaN, the softmax
// warps then look through the unit's values, set what is not finite to nought and add it, element by element, to the outputs of those who see it.
//
// A thread that holds a row of scores spills some 420 bytes with heads of 128 (184 and 160 with heads of 64), the wide form as much with 200, 208 or 216 registers; little
// of it is in the loop over units: 64 requests move 1.9 MB out and 3.9 MB back, beside 340 MB of keys and values; 64 nodes after 131,071 rows 1.1 and 1.0.
//
// What bounds it.  64 requests of 8 nodes after up to 4,096 rows (28 / 4 heads of 128): 83 us with the join (floor 53, the cached rows read once); the loop
// runs at the memory's rate (two groups' units, 128 KB, in 4,850 cycles), and a segment takes some 9,000 cycles to begin and to end, which the other group only partly
// fills; both groups on one unit, with one ring and joined in the block, took 108.  64 nodes after 131,071 rows (12 / 2 heads of 128): 80 us (floor 31): a unit
// of both groups takes 3,800 cycles, of which a group waits 1,500 for its products (eight MMAs of 128 x 128 x 16 take 450 to
// 600 cycles) and 1,310 are exponentials, 1,024 at the unit's rate.  Taken back, when it took 94: scores in pieces of 64 cached rows, the next ones ahead of the weights
// (113 us: MMAs half as wide take nearly as long), weights announced in halves (95), three blocks of 128 query rows for two of 256 (98), blocks of query
// rows one after the other (100: K and V come from memory twice).
#include "tree_attention.cuh"

namespace {

constexpr int ROWS = 128, UNIT = 128, PAGE_ROWS = 16;  // (a TMA box: 16 rows of 64 columns)
constexpr int SOFTMAX_WARPS = 8, THREADS = (SOFTMAX_WARPS + 4) * 32;  // + two TMA warps and two MMA warps, of which WIDE has work for one each: whole warpgroups share out registers
// Registers of a thread: the block is launched with LAUNCH_REGISTERS for each (what 384 threads of an SM can have), of which the third warpgroup gives some to
// the softmax's two; what these take must not be more than that, or they would wait for ever.
constexpr int LAUNCH_REGISTERS = 168, SOFTMAX_REGISTERS = 208, OTHER_REGISTERS = 80;
static_assert(2 * SOFTMAX_REGISTERS + OTHER_REGISTERS <= 3 * LAUNCH_REGISTERS, "registers");
constexpr int BOX = PAGE_ROWS * 128, ATOM = UNIT * 128;  // bytes of a box; of 64 columns of a unit
constexpr int SCORES = 0, OUTPUTS = 256, COLUMNS = 512;  // of tensor memory: two groups' scores (128 each), their outputs (D each)

template <int D, bool WIDE>
struct Sizes {
    static constexpr int ATOMS = D / 64, BLOCK = ATOMS * ATOM, STAGES = D == 64 ? 8 : 4;
    static constexpr int RING = WIDE ? STAGES : STAGES / 2;  // stages of a ring: both groups' or each one's
    static constexpr int GROUP_ROWS = WIDE ? 2 * ROWS : ROWS;  // query rows of an item
    static constexpr int SMEM = BLOCK * (2 + STAGES) + 1024;
};

__device__ __forceinline__ float exp2_unit(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ void tensor_memory_take(uint32_t* to, uint32_t columns) { tmem_alloc(to, columns); }

// D[tensor memory] += A[tensor memory] B[shared memory]: A is 128 rows (lanes) of 16 bf16, two to a column.
__device__ __forceinline__ void tcgen05_mma_bf16_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.eq.b32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b_desc), "r"(idesc)
        : "memory");
}
// One lane of a whole warp.  MMAs take their operands from the warp's uniform registers: what they are formed from has to be known to be the same in all
// lanes (a shuffle from one lane says so), or the compiler brings every operand there by itself.
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// 32 lanes x 32 columns: thread i of the warp writes lane (base lane + i).
__device__ __forceinline__ void tmem_store_32x32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_store_32x16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15])
                 : "memory");
}
// 128 columns of a lane.
__device__ __forceinline__ void tmem_load_row(uint32_t taddr, uint32_t (&r)[128]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_load_32x32(taddr + 32 * c, reinterpret_cast<uint32_t(&)[32]>(r[32 * c]));
}
// Two fp32 at once.
__device__ __forceinline__ uint64_t pair(float lo, float hi) { return (uint64_t)__float_as_uint(hi) << 32 | __float_as_uint(lo); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// All softmax warps; those of one group.
__device__ __forceinline__ void softmax_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void group_barrier(int g) { asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory"); }

template <int D, bool WIDE>
__global__ void __launch_bounds__(THREADS, 1)
    tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TreeAttention p, int groups, int lanes, int no_row) {
    using Z = Sizes<D, WIDE>;
    constexpr int ST = Z::RING;
    extern __shared__ uint8_t smem_raw[];
    __shared__ TreeLines trees[WIDE ? 1 : 2];
    __shared__ TreeRequests requests;
    __shared__ uint64_t fulls[Z::STAGES], empties[Z::STAGES], q_ready[2], s_ready[2], p_ready[2], o_done[2], ended[2];
    __shared__ uint32_t tensor_base;
    __shared__ int odd[4];  // threads that have found a value of a unit that is not finite: of units of both groups by turns, of each one's
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_smem = smem;                // of each group [64 columns][128 rows][64] bf16, 128-byte swizzle
    // what this warp works for: softmax warps a group each, TMA and MMA warps with WIDE both
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = warp < SOFTMAX_WARPS ? warp >> 2 : warp & 1, ring = WIDE ? 0 : g * ST;
    uint8_t* kv_smem = smem + (2 + ring) * Z::BLOCK;  // stages of [64 columns][128 cached rows][64]
    uint64_t *full = fulls + ring, *empty = empties + ring;
    if (threadIdx.x == 0) {
        tma_prefetch_descriptor(&map_k);
        tma_prefetch_descriptor(&map_v);
        for (int s = 0; s < Z::STAGES; ++s) mbar_init(&fulls[s], 1), mbar_init(&empties[s], 1);
        for (int k = 0; k < 2; ++k) mbar_init(&q_ready[k], 4), mbar_init(&s_ready[k], 1), mbar_init(&p_ready[k], 4), mbar_init(&o_done[k], 1), mbar_init(&ended[k], 1);
        mbar_fence_init();
    }
    if (warp == SOFTMAX_WARPS + 2) tensor_memory_take(&tensor_base, COLUMNS);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    // (only now: a dependent launch must not take tensor memory that this one waits for)
    pdl_wait();
    pdl_launch_dependents();
    bool dead = false;  // a wait has run out: from then on nobody waits, and the kernel runs on to its end
    auto wait = [&](uint64_t* bar, int parity, int where) {
        if (!dead) dead = !mbar_wait(bar, parity, p.status, where);
    };
    // which group of the step's this one is (of few, one on every SM)
    const int share = WIDE ? blockIdx.x / lanes : blockIdx.x + g * gridDim.x;
    TreeWalk<UNIT, Z::GROUP_ROWS, false> walk;
    walk.know(p, requests);
    __syncthreads();
    walk.begin(p, requests, share, groups, WIDE ? blockIdx.x - share * lanes : 0);
    TreeItem item;
    if (warp >= SOFTMAX_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGISTERS));
        if (WIDE && g) {
            // (nothing to do)
        } else if (warp < SOFTMAX_WARPS + 2) {
            // ---- K and V on their way: eight lanes, a box of 16 rows each
            int place0 = 0, issued = 0;
            int4 begun = walk.none();
            while (walk.next(p, requests, item)) {
                const TreeRequest r = item.request;
                walk.note(item, begun);
                const int* table = p.tables + (size_t)item.seq * p.width;
                const int n = item.last - item.first;
                // the page of a lane's box of unit i, on its way; its row of the cache; outside the cache where there is none: nought
                auto page_of = [&](int i) {
                    const int row = (item.low + item.first + i) * UNIT + lane * PAGE_ROWS, block = (int)p.page.quotient((uint32_t)row);
                    return lane < UNIT / PAGE_ROWS && i < n && row < r.rows && block < p.width ? table[block] : -1;
                };
                auto row_of = [&](int i, int page) {
                    if (page >= p.pages) ferris_report(p.status, FERRIS_STATUS_BAD_INDEX, 111);
                    if (page < 0 || page >= p.pages) return no_row;
                    const int row = (item.low + item.first + i) * UNIT + lane * PAGE_ROWS, block = (int)p.page.quotient((uint32_t)row);
                    return (page * p.kv_heads + item.head) * p.page_size + (row - block * p.page_size);
                };
                auto load = [&](int place, const CUtensorMap* map, int row) {
                    const int at = place0 + place, s = at % ST;
                    if (at >= ST) wait(&empty[s], (at / ST - 1) & 1, 140);
                    dead = __any_sync(0xffffffffu, dead);
                    if (!dead) issued = at + 1;  // (a stage that may be in use is not written)
                    if (!dead && lane == 0) mbar_expect_tx(&full[s], Z::BLOCK);
                    __syncwarp();
                    if (!dead && lane < UNIT / PAGE_ROWS) {
#pragma unroll
                        for (int a = 0; a < Z::ATOMS; ++a) tma_load_2d(kv_smem + (size_t)s * Z::BLOCK + a * ATOM + lane * BOX, map, 64 * a, row, &full[s]);
                    }
                };
                int page = page_of(0), next = page_of(1), after = page_of(2);
                int now = row_of(0, page), then = row_of(1, next);
                load(0, &map_k, now);
                for (int i = 0; i < n; ++i) {
                    const int last = row_of(i + 2, after);
                    after = page_of(i + 3);
                    load(2 * i + 1, &map_v, now);
                    if (i + 1 < n) load(2 * i + 2, &map_k, then);
                    now = then, then = last;
                }
                place0 += 2 * n;
            }
            if (lane == 0 && share < groups && (!WIDE || share * lanes == blockIdx.x)) p.begun[share] = begun;  // (the first lane has query rows of every item)
            // (nothing may still be on its way when the block ends, whosever wait has run out)
            for (int at = max(0, issued - ST); at < issued; ++at) mbar_wait(&full[at % ST], (at / ST) & 1, p.status, 148);
        } else {
            // ---- products
            const uint32_t idesc_qk = umma_idesc_bf16(ROWS, UNIT), idesc_pv = umma_idesc_bf16(ROWS, D) | (1u << 16);  // (V: cached rows x columns)
            const uint32_t base = uniform(tensor_base);
            int place0 = 0, segments = 0, done0 = 0, done1 = 0;  // done: units of each group
            while (walk.next(p, requests, item)) {
                const int n = uniform(item.last - item.first);
                // the groups that share a unit (WIDE: the second, if it has rows)
                const int first = WIDE ? 0 : uniform(g), last = WIDE ? uniform((2 * item.block + 1) * ROWS < item.request.nodes * p.group) : first;
                for (int k = WIDE ? 0 : first; k <= (WIDE ? 1 : first); ++k) wait(&q_ready[k], segments & 1, 141);
                auto scores = [&](int i, int g) {
                    const int at = place0 + 2 * i, s = at % ST;
                    if (g == first) wait(&full[s], (at / ST) & 1, 142);
                    tcgen05_fence_after();
                    if (elected()) {
                        const uint64_t q_desc = umma_desc_k_major_sw128(smem_u32(q_smem + g * Z::BLOCK));
                        const uint64_t k_desc = umma_desc_k_major_sw128(smem_u32(kv_smem + s * Z::BLOCK));
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint64_t next = (k >> 2) * (ATOM >> 4) + 2 * (k & 3);  // the next 64 columns, 32 bytes along the row
                            tcgen05_mma_bf16(base + SCORES + 128 * g, q_desc + next, k_desc + next, idesc_qk, k > 0 ? 1u : 0u);
                        }
                        tcgen05_commit(&s_ready[g]);
                        if (g == last) tcgen05_commit(&empty[s]);
                    }
                    __syncwarp();
                };
                auto outputs = [&](int i, int g, bool end) {
                    const int at = place0 + 2 * i + 1, s = at % ST;
                    if (g == first) wait(&full[s], (at / ST) & 1, 143);
                    wait(&p_ready[g], (g ? done1 : done0) & 1, 144);
                    if (g)
                        ++done1;
                    else
                        ++done0;
                    tcgen05_fence_after();
                    if (elected()) {
                        const uint64_t v_desc = umma_desc_mn_major_sw128(smem_u32(kv_smem + s * Z::BLOCK), ATOM);
#pragma unroll
                        for (int k = 0; k < UNIT / 16; ++k)
                            tcgen05_mma_bf16_ts(base + OUTPUTS + D * g, base + SCORES + 128 * g + 8 * k, v_desc + (uint64_t)(k * (BOX >> 4)), idesc_pv);
                        if (g == last) tcgen05_commit(&empty[s]);
                        if (end) tcgen05_commit(&o_done[g]);
                    }
                    __syncwarp();
                };
                for (int k = first; k <= last; ++k) scores(0, k);
                for (int i = 0; i < n; ++i)
                    for (int k = first; k <= last; ++k) {
                        outputs(i, k, i + 1 == n);
                        if (i + 1 < n) scores(i + 1, k);
                    }
                __syncwarp();
                place0 += 2 * n, ++segments;
            }
            // (nor may a product still read or write when the block gives its memory back)
            if (segments > 0) {
                if (elected()) tcgen05_commit(&ended[g]);
                __syncwarp();
                mbar_wait(&ended[g], 0, p.status, 149);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGISTERS));
        // ---- softmax: group g = warp / 4, a row a thread
        const int t = threadIdx.x & 127;
        TreeLines& tree = trees[WIDE ? 0 : g];
        auto barrier_of_all = [&] {  // of those who work on an item
            if (WIDE)
                softmax_barrier();
            else
                group_barrier(g);
        };
        const uint32_t lanes_at = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t my_scores = tensor_base + SCORES + 128 * g + lanes_at, my_out = tensor_base + OUTPUTS + D * g + lanes_at;
        const float scale = p.scale;
        int place0 = 0, done = 0, segments = 0;
        while (walk.next(p, requests, item)) {
            const TreeRequest r = item.request;
            const int head = item.head, count = r.nodes * p.group, n = item.last - item.first;
            const bool whole_item = item.first == 0 && item.last == item.tiles;
            const int row0 = item.block * Z::GROUP_ROWS;
            const int at = row0 + (WIDE ? g * ROWS : 0) + t, node = at < count ? at / p.group : -1, q_head = head * p.group + at % p.group;
            const bool live = at - lane < count;                                    // any of the warp's rows
            const bool both = WIDE && row0 + ROWS < count, here = !WIDE || both || g == 0;  // both groups have rows; this one has
            const int units = here ? n : 0;
            const int* table = p.tables + (size_t)item.seq * p.width;
            const int sure_low = p.window > 0 ? max(0, r.start + r.nodes - p.window) : 0, sure_high = min(r.start, r.rows);
            const int parent = tree_parent(p, r, WIDE ? threadIdx.x : t);
            {
                // the group's query rows
                const bf16* src = (const bf16*)p.q + (size_t)(r.first + max(node, 0)) * p.ldq + q_head * D;
                const bool wide = ((uintptr_t)p.q & 15) == 0 && p.ldq % 8 == 0;
                constexpr int EACH = D / 8;  // 16 bytes at a time
                uint8_t* to = q_smem + g * Z::BLOCK;
                uint4 v[EACH];  // (all on their way at once)
#pragma unroll
                for (int c = 0; c < EACH; ++c) v[c] = make_uint4(0u, 0u, 0u, 0u);
                if (node >= 0 && wide) {
#pragma unroll
                    for (int c = 0; c < EACH; ++c) v[c] = *reinterpret_cast<const uint4*>(src + 8 * c);
                } else if (node >= 0) {
#pragma unroll
                    for (int c = 0; c < EACH; ++c) {
                        const unsigned short* x = reinterpret_cast<const unsigned short*>(src + 8 * c);
                        v[c] = make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16, x[6] | (uint32_t)x[7] << 16);
                    }
                }
                uint32_t nought[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) nought[c] = 0u;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) tmem_store_32x32(my_out + 32 * c, nought);
                tmem_store_wait();
#pragma unroll
                for (int c = 0; c < EACH; ++c) {
                    *reinterpret_cast<uint4*>(to + (c >> 3) * ATOM + swizzle128(t, c & 7)) = v[c];
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_ready[g]);
            }
            if (p.window > 0 || (item.low + item.last) * UNIT > sure_high) tree_lines<WIDE ? 256 : 128>(p, r, tree, parent, barrier_of_all);
            float m = -INFINITY, l = 0.0f;
            int looked = 0;
            // the page of a lane's box of a unit's eight, on its way while the unit before is worked on; -1: none
            auto page_of = [&](int i) {
                const int row = (item.low + item.first + i) * UNIT + lane * PAGE_ROWS, block = (int)p.page.quotient((uint32_t)row);
                return i < units && lane < UNIT / PAGE_ROWS && row < r.rows && block < p.width ? table[block] : -1;
            };
            int page = page_of(0);
            for (int i = 0; i < units; ++i) {
                const uint32_t boxes = __ballot_sync(0xffffffffu, page >= 0 && page < p.pages);  // (the TMA warp reports pages that are not there)
                page = page_of(i + 1);
                const int key0 = (item.low + item.first + i) * UNIT;
                const bool whole = key0 >= sure_low && key0 + UNIT <= sure_high && boxes == 0xffu;
                wait(&s_ready[g], done & 1, 145);
                ++done;
                tcgen05_fence_after();
                if (live) {  // (rows that are not there have nobody's weights)
                    uint32_t s[UNIT];
                    tmem_load_row(my_scores, s);
                    tmem_load_wait();
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < UNIT / 32; ++c) {
                            uint32_t sees = node >= 0 ? tree_sees(p, r, tree, node, key0 + 32 * c) : 0u;
                            if (!(boxes >> (2 * c) & 1)) sees &= 0xffff0000u;
                            if (!(boxes >> (2 * c + 1) & 1)) sees &= 0xffffu;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(sees >> j & 1)) s[32 * c + j] = 0xff800000u;
                        }
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < UNIT; j += 2) top[j >> 1 & 3] = fmaxf(fmaxf(top[j >> 1 & 3], __uint_as_float(s[j])), __uint_as_float(s[j + 1]));
                    const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;  // (the scale is above nought)
                    const bool up = most > m + 8.0f || (m == -INFINITY && most > m);
                    if (__any_sync(0xffffffffu, up)) {
                        const float now = up ? most : m, corr = now == -INFINITY ? 1.0f : exp2_unit(m - now);
                        l *= corr, m = now;
                        if (i > 0) {
#pragma unroll 1
                            for (int c = 0; c < D / 16; ++c) {
                                uint32_t o[16];
                                tmem_load_32x16(my_out + 16 * c, o);
                                tmem_load_wait();
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                                tmem_store_32x16(my_out + 16 * c, o);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    const uint64_t scale2 = pair(scale, scale), base2 = pair(-base, -base);
                    uint64_t sum[2] = {0, 0};
#pragma unroll
                    for (int c = 0; c < UNIT / 32; ++c) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint64_t x = fma_pair((uint64_t)s[32 * c + 2 * j + 1] << 32 | s[32 * c + 2 * j], scale2, base2);
                            const float a = exp2_unit(__uint_as_float((uint32_t)x)), b = exp2_unit(__uint_as_float((uint32_t)(x >> 32)));
                            sum[j & 1] = add_pair(sum[j & 1], pair(a, b));
                            s[16 * c + j] = pack_bf16(a, b);
                        }
                        tmem_store_32x16(my_scores + 16 * c, s + 16 * c);
                    }
                    {
                        const uint64_t both = add_pair(sum[0], sum[1]);
                        l += __uint_as_float((uint32_t)both) + __uint_as_float((uint32_t)(both >> 32));
                    }
                    tmem_store_wait();
                }
                if (!whole) {
                    // the unit's values: what is not finite becomes nought, and goes to those who see it by itself
                    const int place = place0 + 2 * i + 1, stage = place % ST;
                    wait(&full[stage], (place / ST) & 1, 146);
                    uint8_t* v = kv_smem + (size_t)stage * Z::BLOCK;
                    // (units that both groups work on are looked through and changed by the first, with the second beside it)
                    const bool mine = !both || g == 0;
                    int& found = odd[both ? looked & 1 : 2 + g];  // (while the other group may still read the unit's before)
                    ++looked;
                    auto barrier = [&] {
                        if (both)
                            softmax_barrier();
                        else
                            group_barrier(g);
                    };
                    if (t == 0 && mine) found = 0;
                    barrier();
                    // (a thread: a cached row)
                    uint32_t any = 0;
#pragma unroll 4
                    for (int c = 0; c < D / 8 && mine; ++c) {
                        const uint4 x = *reinterpret_cast<const uint4*>(v + (c >> 3) * ATOM + swizzle128(t, c & 7));
                        const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) any |= __vcmpeq2(word[k] & 0x7f807f80u, 0x7f807f80u);
                    }
                    if (any) atomicAdd(&found, 1);
                    barrier();
                    if (found) {
                        // every thread for its query row: what it sees that is not finite (its weight is above nought, whatever it is)
                        for (int j = 0; j < UNIT; ++j) {
                            const bool sees = node >= 0 && (boxes >> (j >> 4) & 1) && (tree_sees(p, r, tree, node, key0 + (j & ~31)) >> (j & 31) & 1);
                            for (int c = 0; c < D; ++c) {
                                const bf16 x = *reinterpret_cast<const bf16*>(v + (c >> 6) * ATOM + swizzle128(j, (c >> 3) & 7) + 2 * (c & 7));
                                const float f = __bfloat162float(x);
                                if (isfinite(f)) continue;  // (the same for all threads)
                                uint32_t o;
                                asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(o) : "r"(my_out + c) : "memory");
                                tmem_load_wait();
                                if (sees) o = __float_as_uint(__uint_as_float(o) + f);
                                asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(my_out + c), "r"(o) : "memory");
                            }
                        }
                        tmem_store_wait();
                        barrier();
                        for (int c = 0; c < D && mine; ++c) {
                            bf16* x = reinterpret_cast<bf16*>(v + (c >> 6) * ATOM + swizzle128(t, (c >> 3) & 7) + 2 * (c & 7));
                            if (!isfinite(__bfloat162float(*x))) *x = __float2bfloat16_rn(0.0f);
                        }
                        fence_proxy_async();
                        if (both) barrier();
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[g]);
            }
            if (units > 0) wait(&o_done[g], segments & 1, 147);
            tcgen05_fence_after();
            float* part = tree_part(p, WIDE ? blockIdx.x : share, item.first == 0, Z::GROUP_ROWS) + (WIDE ? g * ROWS : 0) + t;
            bf16* out = (bf16*)p.out + (size_t)(r.first + max(node, 0)) * p.ldo + q_head * D;
            const bool wide = ((uintptr_t)p.out & 15) == 0 && p.ldo % 8 == 0;
            // columns of this thread's row, to the output (times `inv`) or to the block's part
            auto leave = [&](auto& o, int col, float inv) {
                if (node < 0) return;
                constexpr int W = sizeof(o) / 4;
                if (!whole_item) {
#pragma unroll
                    for (int j = 0; j < W; ++j) part[(col + j) * Z::GROUP_ROWS] = __uint_as_float(o[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < W; j += 8) {
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(o[j + k]) * inv;
                        if (wide)
                            *reinterpret_cast<uint4*>(out + col + j) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
                        else
#pragma unroll
                            for (int k = 0; k < 8; ++k) out[col + j + k] = from_float<bf16>(v[k]);
                    }
                }
            };
            auto leave_sums = [&](float most, float total) {
                if (!whole_item && node >= 0) part[D * Z::GROUP_ROWS] = most, part[(D + 1) * Z::GROUP_ROWS] = total;
            };
            if (live && here) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_load_32x32(my_out + 32 * c, o);
                    tmem_load_wait();
                    leave(o, 32 * c, inv);
                }
                leave_sums(m, l);
            }
            barrier_of_all();  // (the lines of ancestors may be written again)
            place0 += 2 * n;
            // (a phase of o_done passes in every segment in which the group has units, q_ready's in every segment)
            if (units > 0) ++segments;
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == SOFTMAX_WARPS + 2) {
        tcgen05_fence_after();
        tmem_dealloc(tensor_base, COLUMNS);
    }
}

template <int D, bool WIDE>
int launch(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream) {
    const uint64_t rows = (uint64_t)p.pages * p.kv_heads * p.page_size;
    CUtensorMap map_k, map_v;
    int rc = ferris_make_tensor_map_2d(&map_k, p.k_cache, rows, D, D, PAGE_ROWS, 64);
    if (rc == FERRIS_OK) rc = ferris_make_tensor_map_2d(&map_v, p.v_cache, rows, D, D, PAGE_ROWS, 64);
    if (rc == FERRIS_OK) rc = ferris_allow_dynamic_smem((const void*)tree_attention_tc_kernel<D, WIDE>, Sizes<D, WIDE>::SMEM);
    if (rc != FERRIS_OK) return rc;
    static const int registers = [] {
        cudaFuncAttributes f = {};
        return cudaFuncGetAttributes(&f, tree_attention_tc_kernel<D, WIDE>) == cudaSuccess ? f.numRegs : 0;
    }();
    if (registers < LAUNCH_REGISTERS) FERRIS_REFUSE("a kernel of %d registers a thread, %d are needed", registers, LAUNCH_REGISTERS);
    const int sms = ferris_sm_count(), grid = WIDE ? plan.groups * plan.lanes : plan.groups < sms ? plan.groups : sms;
    const cudaError_t e = ferris_launch(tree_attention_tc_kernel<D, WIDE>, dim3(grid), dim3(THREADS), (size_t)Sizes<D, WIDE>::SMEM, stream, map_k, map_v, p,
                                        plan.groups, plan.lanes, (int)rows);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    return FERRIS_OK;
}

}  // namespace

int tree_attention_tc(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream) {
    if (p.head_dim == 64) return plan.rows > ROWS ? launch<64, true>(p, plan, stream) : launch<64, false>(p, plan, stream);
    return plan.rows > ROWS ? launch<128, true>(p, plan, stream) : launch<128, false>(p, plan, stream);
}
