// Attention for trees of drafted tokens over the paged cache, bf16, on tcgen05: heads of 64 and 128, many query rows (who sees what, and how the work is
// dealt out: tree_attention.cuh).
//
// A block of 128 query rows goes over blocks of 128 cached rows (units):
//   S = Q K^T   128 x 128 x D, operands in shared memory (Q written once, K by TMA), sums in tensor memory
//   P = 2^(S scale - m), rounded to bf16 (eight bits, as the output has; sums take it unrounded), into tensor memory over the scores it came from
//   O = O + P V   P from tensor memory, V as TMA wrote it, sums in tensor memory over all units
// Two groups of four softmax warps, each with scores, maxima, sums and outputs of its own, so that the tensor core works for one while
// the other exponentiates: of up to 128 query rows they take the units in turn and are joined at the end, of more (WIDE) each has 128 rows of its own, and K and V are
// fetched once for both; a thread has a row, so that nothing is exchanged.
// m is the greatest score so far only up to 2^8: outputs are brought to a new m (read, multiplied, written back) where a score exceeds it by
// more than eight, which after the first units is rare; what is divided by in the end has the same m, so that nothing but the range of the weights changes.
// A TMA warp streams K and V through a ring of stages, ahead of the segment that is worked on; an MMA warp issues, in the order of the units,
// P V of a unit and then the scores of the group's next one (the tensor core keeps the order, so that these do not overwrite weights that are still read).
//
// Units that every node sees whole are worked off as they are.  In others scores that are not seen become nought weights; as nought times NaN is NaN, the softmax
// warps then look through the unit's values, set what is not finite to nought and add it, element by element, to the outputs of those who see it.
//
// What bounds it.  64 requests of 8 nodes after up to 4,096 rows (28 / 4 heads of 128): 108 us with the join (floor 53, the cached rows read once); the loop
// runs at the memory's rate, a unit in 2,600 to 2,900 cycles, and every segment costs some 5 us more to begin and to end.  64 nodes after 131,071 rows (12 / 2 heads
// of 128): 94 us (floor 31): a unit of both groups takes 3,800 cycles, of which a group waits 1,500 for its products (eight MMAs of 128 x 128 x 16 take 450 to
// 600 cycles) and 1,310 are exponentials, 1,024 at the unit's rate.  Taken back: scores in pieces of 64 cached rows, the next ones ahead of the weights (113 us: MMAs
// half as wide take nearly as long), weights announced in halves (95), three blocks of 128 query rows for two of 256 (98).
#include "tree_attention.cuh"

namespace {

constexpr int ROWS = 128, UNIT = 128, PAGE_ROWS = 16;  // (a TMA box: 16 rows of 64 columns)
constexpr int SOFTMAX_WARPS = 8, THREADS = (SOFTMAX_WARPS + 4) * 32;  // + a TMA warp, an MMA warp and two without work: whole warpgroups share out registers
// Registers of a thread: the block is launched with LAUNCH_REGISTERS for each (what 384 threads of an SM can have), of which the third warpgroup gives some to
// the softmax's two; what these take must not be more than that, or they would wait for ever.
constexpr int LAUNCH_REGISTERS = 168, SOFTMAX_REGISTERS = 208, OTHER_REGISTERS = 80;
static_assert(2 * SOFTMAX_REGISTERS + OTHER_REGISTERS <= 3 * LAUNCH_REGISTERS, "registers");
constexpr int BOX = PAGE_ROWS * 128, ATOM = UNIT * 128;  // bytes of a box; of 64 columns of a unit
constexpr int SCORES = 0, OUTPUTS = 256, COLUMNS = 512;  // of tensor memory: two groups' scores (128 each), their outputs (D each)

template <int D, bool WIDE>
struct Sizes {
    static constexpr int ATOMS = D / 64, BLOCK = ATOMS * ATOM, TILES = WIDE ? 2 : 1, STAGES = D == 64 ? 8 : WIDE ? 4 : 5;
    static constexpr int SMEM = BLOCK * (TILES + STAGES) + 1024;
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

template <int W>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[W]) {
    if constexpr (W == 32)
        tmem_load_32x32(taddr, r);
    else
        tmem_load_32x16(taddr, r);
}

// All softmax warps; those of one group.
__device__ __forceinline__ void softmax_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void group_barrier(int g) { asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory"); }

// Stages in the order of their use by the tensor core: K 0, K 1, V 0, K 2, V 1, K 3, ..; where both groups use them, K 0, V 0, K 1, ..
template <bool WIDE>
__device__ __forceinline__ int k_place(int i) { return WIDE ? 2 * i : i < 2 ? i : 2 * i - 1; }
template <bool WIDE>
__device__ __forceinline__ int v_place(int i, int n) { return WIDE || i + 1 == n ? 2 * i + 1 : 2 * i + 2; }

template <int D, bool WIDE>
__global__ void __launch_bounds__(THREADS, 1)
    tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TreeAttention p, int lanes, int no_row) {
    using Z = Sizes<D, WIDE>;
    constexpr int ST = Z::STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ TreeLines tree;
    __shared__ uint64_t full[ST], empty[ST], q_ready, s_ready[2], p_ready[2], o_done[2];
    __shared__ uint32_t tensor_base;
    __shared__ float row_m[2][ROWS], row_l[2][ROWS];  // (not WIDE)
    __shared__ int odd[2];  // how many elements of a unit's values are not finite
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_smem = smem;                // [64 columns][128 rows][64] bf16, 128-byte swizzle; at a segment's end, half of a group's outputs
    uint8_t* kv_smem = smem + Z::TILES * Z::BLOCK;  // stages of [64 columns][128 cached rows][64]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        tma_prefetch_descriptor(&map_k);
        tma_prefetch_descriptor(&map_v);
        for (int s = 0; s < ST; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        mbar_init(&q_ready, SOFTMAX_WARPS);
        for (int g = 0; g < 2; ++g) mbar_init(&s_ready[g], 1), mbar_init(&p_ready[g], 4), mbar_init(&o_done[g], 1);
        mbar_fence_init();
    }
    if (warp == SOFTMAX_WARPS + 1) tensor_memory_take(&tensor_base, COLUMNS);
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
    TreeWalk<UNIT, ROWS * Z::TILES, false> walk;
    walk.begin(p, lanes);
    TreeItem item;
    if (warp >= SOFTMAX_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGISTERS));
        if (warp == SOFTMAX_WARPS) {
            // ---- K and V on their way: eight lanes, a box of 16 rows each
            int place0 = 0;
            int4 begun = walk.none();
            while (walk.next(p, item)) {
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
                    if (lane == 0) mbar_expect_tx(&full[s], Z::BLOCK);
                    __syncwarp();
                    if (lane < UNIT / PAGE_ROWS) {
#pragma unroll
                        for (int a = 0; a < Z::ATOMS; ++a) tma_load_2d(kv_smem + (size_t)s * Z::BLOCK + a * ATOM + lane * BOX, map, 64 * a, row, &full[s]);
                    }
                };
                int page = page_of(0), next = page_of(1), after = page_of(2);
                int now = row_of(0, page), then = row_of(1, next);
                load(0, &map_k, now);
                if (!WIDE && n > 1) load(1, &map_k, then);
                for (int i = 0; i < n; ++i) {
                    const int last = row_of(i + 2, after);
                    after = page_of(i + 3);
                    load(v_place<WIDE>(i, n), &map_v, now);
                    if (WIDE && i + 1 < n) load(k_place<WIDE>(i + 1), &map_k, then);
                    if (!WIDE && i + 2 < n) load(k_place<WIDE>(i + 2), &map_k, last);
                    now = then, then = last;
                }
                place0 += 2 * n;
            }
            if (lane == 0 && blockIdx.x % lanes == 0) p.begun[blockIdx.x / lanes] = begun;  // (the first block of a group has query rows of every item)
            // (after a wait that ran out: nothing may still be on its way when the block ends)
            if (dead)
                for (int at = max(0, place0 - ST); at < place0; ++at) mbar_wait(&full[at % ST], (at / ST) & 1, p.status, 148);
        } else if (warp == SOFTMAX_WARPS + 1) {
            // ---- products
            const uint32_t idesc_qk = umma_idesc_bf16(ROWS, UNIT), idesc_pv = umma_idesc_bf16(ROWS, D) | (1u << 16);  // (V: cached rows x columns)
            const uint32_t base = uniform(tensor_base);
            int place0 = 0, segments = 0, done0 = 0, done1 = 0;  // done: units of each group
            while (walk.next(p, item)) {
                const int n = uniform(item.last - item.first);
                const bool two = WIDE && uniform((item.block * Z::TILES + 1) * ROWS < item.request.nodes * p.group);  // (WIDE: the second group has rows)
                wait(&q_ready, segments & 1, 141);
                auto scores = [&](int i, int g) {
                    const int at = place0 + k_place<WIDE>(i), s = at % ST;
                    if (!WIDE || g == 0) wait(&full[s], (at / ST) & 1, 142);
                    tcgen05_fence_after();
                    if (elected()) {
                        const uint64_t q_desc = umma_desc_k_major_sw128(smem_u32(q_smem + (WIDE ? g * Z::BLOCK : 0)));
                        const uint64_t k_desc = umma_desc_k_major_sw128(smem_u32(kv_smem + s * Z::BLOCK));
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint64_t next = (k >> 2) * (ATOM >> 4) + 2 * (k & 3);  // the next 64 columns, 32 bytes along the row
                            tcgen05_mma_bf16(base + SCORES + 128 * g, q_desc + next, k_desc + next, idesc_qk, k > 0 ? 1u : 0u);
                        }
                        tcgen05_commit(&s_ready[g]);
                        if (!two || g) tcgen05_commit(&empty[s]);
                    }
                    __syncwarp();
                };
                auto outputs = [&](int i, int g, bool last) {
                    const int at = place0 + v_place<WIDE>(i, n), s = at % ST;
                    if (!WIDE || g == 0) wait(&full[s], (at / ST) & 1, 143);
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
                        if (!two || g) tcgen05_commit(&empty[s]);
                        if (last) tcgen05_commit(&o_done[g]);
                    }
                    __syncwarp();
                };
                if constexpr (WIDE) {
                    scores(0, 0);
                    if (two) scores(0, 1);
                    for (int i = 0; i < n; ++i)
                        for (int g = 0; g <= two; ++g) {
                            outputs(i, g, i + 1 == n);
                            if (i + 1 < n) scores(i + 1, g);
                        }
                } else {
                    for (int i = 0; i < 2 && i < n; ++i) scores(i, i);
                    for (int i = 0; i < n; ++i) {
                        outputs(i, i & 1, i + 2 >= n);
                        if (i + 2 < n) scores(i + 2, i & 1);
                    }
                }
                __syncwarp();
                place0 += 2 * n, ++segments;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGISTERS));
        // ---- softmax: group g = warp / 4, a row a thread
        const int g = warp >> 2, t = threadIdx.x & 127;
        const uint32_t lanes_at = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t my_scores = tensor_base + SCORES + 128 * g + lanes_at, my_out = tensor_base + OUTPUTS + D * g + lanes_at;
        const float scale = p.scale;
        int place0 = 0, done = 0, segments = 0;
        while (walk.next(p, item)) {
            const TreeRequest r = item.request;
            const int head = item.head, count = r.nodes * p.group, n = item.last - item.first;
            const bool whole_item = item.first == 0 && item.last == item.tiles;
            const int row0 = item.block * ROWS * Z::TILES;
            const int at = row0 + (WIDE ? g * ROWS : 0) + t, node = at < count ? at / p.group : -1, q_head = head * p.group + at % p.group;
            const bool live = at - lane < count;                                    // any of the warp's rows
            const int from = WIDE ? 0 : g, step = WIDE ? 1 : 2;                     // the group's units
            const bool both = !WIDE || row0 + ROWS < count, here = both || g == 0;  // both groups have rows; this one has
            const int units = here ? n : 0;
            const int* table = p.tables + (size_t)item.seq * p.width;
            {
                // the block's query rows, half of the columns by each group
                const bf16* src = (const bf16*)p.q + (size_t)(r.first + max(node, 0)) * p.ldq + q_head * D;
                const bool wide = ((uintptr_t)p.q & 15) == 0 && p.ldq % 8 == 0;
                constexpr int EACH = WIDE ? D / 8 : D / 16;  // 16 bytes at a time: a row, or half of one
                const int first = WIDE ? 0 : g * EACH;
                uint8_t* to = q_smem + (WIDE ? g * Z::BLOCK : 0);
                uint4 v[EACH];  // (all on their way at once)
#pragma unroll
                for (int c = 0; c < EACH; ++c) v[c] = make_uint4(0u, 0u, 0u, 0u);
                if (node >= 0 && wide) {
#pragma unroll
                    for (int c = 0; c < EACH; ++c) v[c] = *reinterpret_cast<const uint4*>(src + 8 * (first + c));
                } else if (node >= 0) {
#pragma unroll
                    for (int c = 0; c < EACH; ++c) {
                        const unsigned short* x = reinterpret_cast<const unsigned short*>(src + 8 * (first + c));
                        v[c] = make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16, x[6] | (uint32_t)x[7] << 16);
                    }
                }
#pragma unroll
                for (int c = 0; c < EACH; ++c) {
                    const int column = first + c;
                    *reinterpret_cast<uint4*>(to + (column >> 3) * ATOM + swizzle128(t, column & 7)) = v[c];
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_ready);
            }
            const int sure_low = p.window > 0 ? max(0, r.start + r.nodes - p.window) : 0, sure_high = min(r.start, r.rows);
            if (p.window > 0 || (item.low + item.last) * UNIT > sure_high) tree_lines<SOFTMAX_WARPS * 32>(p, r, tree, softmax_barrier);
            {
                uint32_t nought[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) nought[c] = 0u;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) tmem_store_32x32(my_out + 32 * c, nought);
                tmem_store_wait();
            }
            float m = -INFINITY, l = 0.0f;
            // the page of a lane's box of a unit's eight, on its way while the unit before is worked on; -1: none
            auto page_of = [&](int i) {
                const int row = (item.low + item.first + i) * UNIT + lane * PAGE_ROWS, block = (int)p.page.quotient((uint32_t)row);
                return i < units && lane < UNIT / PAGE_ROWS && row < r.rows && block < p.width ? table[block] : -1;
            };
            int page = page_of(from);
            for (int i = from; i < units; i += step) {
                const uint32_t boxes = __ballot_sync(0xffffffffu, page >= 0 && page < p.pages);  // (the TMA warp reports pages that are not there)
                page = page_of(i + step);
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
                        if (i > from) {
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
                    const int place = place0 + v_place<WIDE>(i, n), stage = place % ST;
                    wait(&full[stage], (place / ST) & 1, 146);
                    uint8_t* v = kv_smem + (size_t)stage * Z::BLOCK;
                    // (units that both groups work on are looked through and changed by the first, with the second beside it)
                    const bool shared = WIDE && both, mine = !shared || g == 0;
                    int& found = odd[shared ? 0 : g];
                    auto barrier = [&] {
                        if (shared)
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
                        if (shared) barrier();
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[g]);
            }
            if (units > from) wait(&o_done[g], segments & 1, 147);
            tcgen05_fence_after();
            float* part = tree_part(p, blockIdx.x, item.first == 0, ROWS * Z::TILES) + (WIDE ? g * ROWS : 0) + t;
            bf16* out = (bf16*)p.out + (size_t)(r.first + max(node, 0)) * p.ldo + q_head * D;
            const bool wide = ((uintptr_t)p.out & 15) == 0 && p.ldo % 8 == 0;
            // columns of this thread's row, to the output (times `inv`) or to the block's part
            auto leave = [&](auto& o, int col, float inv) {
                if (node < 0) return;
                constexpr int W = sizeof(o) / 4;
                if (!whole_item) {
#pragma unroll
                    for (int j = 0; j < W; ++j) part[(col + j) * (ROWS * Z::TILES)] = __uint_as_float(o[j]);
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
                if (!whole_item && node >= 0) part[D * (ROWS * Z::TILES)] = most, part[(D + 1) * (ROWS * Z::TILES)] = total;
            };
            if constexpr (WIDE) {
                // ---- every group its rows
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
                softmax_barrier();  // (the lines of ancestors may be written again)
            } else {
                // ---- the groups joined through the query rows' memory, each for half of the columns, in two rounds
                row_m[g][t] = m, row_l[g][t] = l;
                softmax_barrier();  // (both groups' products are done: nobody reads the query rows any more)
                const float m1 = row_m[g ^ 1][t], most = fmaxf(m, m1), base = most == -INFINITY ? 0.0f : most;
                const float f0 = exp2_unit(m - base), f1 = exp2_unit(m1 - base), total = l * f0 + row_l[g ^ 1][t] * f1;
                const float inv = total == 0.0f ? 0.0f : 1.0f / total;
                constexpr int W = D / 4;  // columns of a round
                float* mine = reinterpret_cast<float*>(q_smem) + g * W * ROWS + t;  // [column][row]: what the other group needs
                const float* others = reinterpret_cast<const float*>(q_smem) + (g ^ 1) * W * ROWS + t;
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    uint32_t o[W];
                    const int col = g * 2 * W + h * W;
                    if (live) {
                        tmem_load<W>(my_out + (g ^ 1) * 2 * W + h * W, o);
                        tmem_load_wait();
#pragma unroll
                        for (int j = 0; j < W; ++j) mine[j * ROWS] = __uint_as_float(o[j]);
                        tmem_load<W>(my_out + col, o);
                    }
                    softmax_barrier();
                    if (live) {
                        tmem_load_wait();
#pragma unroll
                        for (int j = 0; j < W; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f0 + others[j * ROWS] * f1);
                        leave(o, col, inv);
                    }
                    softmax_barrier();
                }
                if (g == 0) leave_sums(most, total);
            }
            place0 += 2 * n;
            // (a phase of o_done passes in every segment in which the group has units, q_ready's in every segment)
            if (units > from) ++segments;
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == SOFTMAX_WARPS + 1) {
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
    const cudaError_t e = ferris_launch(tree_attention_tc_kernel<D, WIDE>, dim3(plan.groups * plan.lanes), dim3(THREADS), (size_t)Sizes<D, WIDE>::SMEM, stream, map_k, map_v, p,
                                        plan.lanes, (int)rows);
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
