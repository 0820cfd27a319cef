// Attention over the paged cache in 4 bits (its bytes: packed_cache.cuh), on mma.sync, for every geometry.
//
// A query row r of a request and kv head is (query i = r / G, head r % G of the G heads that share the kv head); it sees
// the cached rows max(0, p - window + 1) .. p with p = start + i that have a page.  Query rows are the columns of the
// MMAs (eight to a tile), sixteen cached rows their rows:
//   S^T = K Q^T   per group j of 32 elements:  s[key][q] += scale_j[key] (codes_j[key] . q_j) + least_j[key] sum(q_j)
//   O^T = V^T P^T per group j:                 o[elem][q] += codes_j[elem][key] (p[key][q] scale_j[key]), and least_j[key] p[key][q] in 32 bits
// so that keys and values are never formed.  A word of eight codes becomes four operands of fp16 pairs with an AND / OR (1024 + code
// or, from the upper four bits of a byte, 1024 + 16 code) and a subtraction (or a multiply-add) each; values subtract 8 more and add 8 scale to their
// least, so that what the sums hold is of the size of the result (unsigned codes add up to something that least nearly cancels:
// over 32,768 rows the accumulators' rounding alone came to 0.0015 of the output).  What meets the codes is scaled by powers of two into the
// range of fp16: a query row by its greatest element (bf16 rows then lose nothing that 32 bits would keep; 32-bit rows go in
// two parts, 22 bits), p scale of bf16 rows by the greatest scale of its group that the warp has met, in eleven bits (rows whose
// scale and weight together are below 2^-20 of that scale keep fewer; with one power for all groups, of a group of values 2^-24 the
// size of another was off by 0.007, of 2^-30 by 0.9).  p scale of 32-bit rows goes in three parts of bf16, 24 bits whatever the scales' range, against codes in
// bf16 (two parts of fp16, whose steps end at 2^-24, left a group of values 2^-20 the size of another no more bits than a bf16
// row has; six requests of up to 1,534 rows, 12 / 2 heads of 128, 12.8 us with those, 12.5 with these).
// (In bf16's eight bits the outputs were off by 0.0025 to 0.005 of their norm, 0.0016 of which is their own rounding;
// codes as fp16 numbers below the normal range need no subtraction, but the tensor cores align their products as if they
// were large: 3e-5 of a 32-bit output.)
// Bound by its instructions, about 1,400 for 32 cached rows of a warp at D = 128 with all that is before and behind them, and by their
// latencies: 64 requests of up to 4,097 rows (28 / 4 heads of 128, scores kept) 64 us, 1.7 TB/s, issue slots 42 % used, ALU pipe 34 %,
// tensor pipe 8 %; one of 131,072 rows (12 / 2 heads) 25.5 us and 9.7 for the join of its parts.
#include "packed_attention.cuh"

namespace {

constexpr int KEYS = 16;   // cached rows of an MMA
constexpr int STAGE = 32;  // cached rows that a warp fetches at once
constexpr int WARPS = 8;     // (four to a block, four blocks to an SM: more parts to join, 8 requests of 4,096 rows 13.5 -> 19 us)
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same into nothing: c = A B.
__device__ __forceinline__ void mma_f16_16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ void mma_bf16_16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    c[0] = c[1] = c[2] = c[3] = 0.0f;
    mma_bf16_16816(c, a, b0, b1);
}

// 16 (or 8, or 4) bytes global -> shared without registers; `live` false: zeros, and nothing is read.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool live) {
    const int n = live ? BYTES : 0;
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// W words from shared memory, in the widest loads that their alignment allows.
template <int W>
__device__ __forceinline__ void load_words(uint32_t (&r)[W], const unsigned char* p) {
    if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            r[4 * i] = v.x, r[4 * i + 1] = v.y, r[4 * i + 2] = v.z, r[4 * i + 3] = v.w;
        }
    } else if constexpr (W % 2 == 0) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            const uint2 v = reinterpret_cast<const uint2*>(p)[i];
            r[2 * i] = v.x, r[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) r[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// What a warp fetches at once: STAGE cached rows.  Row strides keep the fragments' loads free of bank conflicts: of keys a
// lane (g, c) takes 4 W bytes of row g at 4 W c, of values 2 W bytes of rows 2c, 2c + 1, 2c + 8, 2c + 9 at 2 W g.
template <int W>
struct Stage {
    static constexpr int K_ROW = W == 8 ? 144 : 16 * W, V_ROW = 16 * W + 16, S_ROW = 4 * W;
    static constexpr int V_AT = STAGE * K_ROW, KS_AT = V_AT + STAGE * V_ROW, VS_AT = KS_AT + STAGE * S_ROW, BYTES = VS_AT + STAGE * S_ROW;
    static_assert(BYTES % 16 == 0 && KS_AT % 16 == 0, "copies of 16 bytes");

    // Requests rows first .. first + 31 (those from `end` on, and those without a page, become zeros); which of them are there.
    static __device__ __forceinline__ uint32_t request(const PackedAttention& p, const int* table, int head, int first, int end, unsigned char* to,
                                                       int lane) {
        const int row = first + lane;
        if (first >= end) {  // (the whole warp) nothing to fetch, but a group to count
            copy_commit();
            return 0;
        }
        const int block = p.block_of(row), page = row < end ? page_of(p, table, block) : -1;
        const uint32_t at = page >= 0 ? p.row_of(page, head, row, block) : 0;
        const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t dst = smem_u32(to);
#pragma unroll
        for (int i = 0; i < W; ++i) {  // W pieces of 16 bytes a row: neighbouring lanes take neighbouring pieces
            const int piece = i * 32 + lane, r = piece / W, part = piece % W;
            const uint32_t a = __shfl_sync(0xffffffffu, at, r);
            const bool live = there >> r & 1;
            // (the piece's offset belongs to the base: a row then costs one wide multiply-add)
            copy_async<16>(dst + r * K_ROW + 16 * part, (p.cache.k_codes + 16 * part) + (size_t)a * (16 * W), live);
            copy_async<16>(dst + V_AT + r * V_ROW + 16 * part, (p.cache.v_codes + 16 * part) + (size_t)a * (16 * W), live);
        }
        constexpr int N = W % 4 == 0 ? 16 : W % 2 == 0 ? 8 : 4;
#pragma unroll
        for (int i = 0; i < S_ROW / N; ++i) {
            copy_async<N>(dst + KS_AT + lane * S_ROW + N * i, (const char*)(p.cache.k_scales + (size_t)at * W) + N * i, page >= 0);
            copy_async<N>(dst + VS_AT + lane * S_ROW + N * i, (const char*)(p.cache.v_scales + (size_t)at * W) + N * i, page >= 0);
        }
        copy_commit();
        return there;
    }
};

// What a lane (g = lane / 4, c = lane % 4) holds of eight query rows as the B operand: row g of the tile, times `factor`, a
// power of two that brings its greatest element to 2^13.
template <typename T, int W, int NP>
struct Queries {
    uint32_t b[W][2][2][NP];       // group, half of the group's word, register
    uint32_t sum[(W + 3) / 4][2];  // the sum of group 4 i + c in three bf16 parts
    float factor;

    __device__ __forceinline__ void load(const T* row, int c, bool valid, bool aligned) {
        float x[W][8] = {}, top = 0.0f;
        if (valid && aligned) {
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int i = 0; i < 8 / N; ++i) {
                    const uint4 v = reinterpret_cast<const uint4*>(row + 32 * j + 8 * c)[i];
                    const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
                    for (int k = 0; k < N; ++k) x[j][N * i + k] = to_float(t[k]);
                }
        } else if (valid) {
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = to_float(row[32 * j + 8 * c + i]);
        }
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[j][i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(13 - e) for 2^e <= top < 2^(e + 1), at most 2^126
        const int e = (int)(__float_as_uint(top) >> 23);
        factor = top > 0.0f && e < 255 ? __uint_as_float((uint32_t)min(267 - e, 253) << 23) : 1.0f;
        float mine[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            mine[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                mine[j] += x[j][i];
                x[j][i] *= factor;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int i = 2 * t + r;  // pairs (i, i + 4): the order of code_pairs
                    float lo = x[j][i], hi = x[j][i + 4];
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const uint32_t v = pack_f16(lo, hi);
                        b[j][t][r][n] = v;
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
                        lo -= f.x, hi -= f.y;
                    }
                }
        }
        float own[(W + 3) / 4] = {};
#pragma unroll
        for (int j = 0; j < W; ++j) {
            mine[j] += __shfl_xor_sync(0xffffffffu, mine[j], 1);
            mine[j] += __shfl_xor_sync(0xffffffffu, mine[j], 2);
            if (j % 4 == c) own[j / 4] = mine[j];
        }
#pragma unroll
        for (int i = 0; i < (W + 3) / 4; ++i) {
            const float s = own[i] * factor;
            const float s1 = __bfloat162float(__float2bfloat16_rn(s)), s2 = __bfloat162float(__float2bfloat16_rn(s - s1));
            sum[i][0] = pack_bf16(s1, s2);
            sum[i][1] = pack_bf16(s - s1 - s2, 0.0f);
        }
    }
};

// Codes and scales of the keys of sixteen rows: this lane's rows g and g + 8.
template <int W>
struct Keys {
    uint32_t word[2][W], scale[2][W], mine[2][(W + 3) / 4];  // mine: the scales' words of groups 4 i + c

    __device__ __forceinline__ void load(const unsigned char* stage, int first, int g, int c) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < (W + 3) / 4; ++i)
                mine[u][i] = 4 * i + c < W ? reinterpret_cast<const uint32_t*>(stage + Stage<W>::KS_AT + (first + g + 8 * u) * Stage<W>::S_ROW)[4 * i + c] : 0u;
            load_words<W>(word[u], stage + (first + g + 8 * u) * Stage<W>::K_ROW + 4 * W * c);
            load_words<W>(scale[u], stage + Stage<W>::KS_AT + (first + g + 8 * u) * Stage<W>::S_ROW);
        }
    }

    // s[n][0..3]: (key g, rows 2c and 2c + 1 of tile n), (key g + 8, the same), times factor
    template <typename T, int NP, int NT>
    __device__ __forceinline__ void scores(const Queries<T, W, NP> (&q)[NT], int c, float (&s)[NT][4]) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < (W + 3) / 4; ++i) {  // least times the sums of the queries' groups
            const uint32_t a0 = __byte_perm(mine[0][i], 0u, 0x3232), a1 = __byte_perm(mine[1][i], 0u, 0x3232);
            const uint32_t a[4] = {a0, a1, a0, a1};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16_16816(s[n], a, q[n].sum[i][0], q[n].sum[i][1]);
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
            uint32_t a0[4], a1[4];
            code_pairs<0>(word[0][j], a0);
            code_pairs<0>(word[1][j], a1);
            const float s0 = packed_scale(scale[0][j]), s1 = packed_scale(scale[1][j]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float d[4];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t a[4] = {a0[2 * t], a1[2 * t], a0[2 * t + 1], a1[2 * t + 1]};
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        if (t == 0 && i == 0)
                            mma_f16_16816_first(d, a, q[n].b[j][t][0][i], q[n].b[j][t][1][i]);
                        else
                            mma_f16_16816(d, a, q[n].b[j][t][0][i], q[n].b[j][t][1][i]);
                    }
                }
                s[n][0] = fmaf(s0, d[0], s[n][0]);
                s[n][1] = fmaf(s0, d[1], s[n][1]);
                s[n][2] = fmaf(s1, d[2], s[n][2]);
                s[n][3] = fmaf(s1, d[3], s[n][3]);
            }
        }
    }
};

// What the rows of NT tiles of eight see: for this lane's columns 2c and 2c + 1 of each and for all of them.
template <int NT>
struct Rows {
    int low[NT][2], high[NT][2];  // first row seen, one past the last
    int least, most;              // over all rows: the range to go through
    int all_low, all_high;        // rows that every row of the tiles sees

    static __device__ __forceinline__ void sees(const PackedAttention& p, int r, int start, int limit, int& lo, int& hi) {
        const int at = start + r / p.group;
        hi = min(at + 1, limit);
        lo = p.window > 0 ? max(0, at - p.window + 1) : 0;
    }

    // (what rows see moves on with their number: the first and the last row of the tiles bound all of them)
    __device__ __forceinline__ void set(const PackedAttention& p, int first, int count, int start, int limit, int c) {
        const int last = min(first + 8 * NT, count) - 1;
        int hi;
        sees(p, first, start, limit, least, all_high);
        sees(p, last, start, limit, all_low, most);
        hi = max(most, 0);
        most = hi;
        least = min(least, most);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = first + 8 * n + 2 * c + u;
                low[n][u] = 0, high[n][u] = 0;
                if (r < count) sees(p, r, start, limit, low[n][u], high[n][u]);
            }
    }
};

template <int D, int NT>
struct RowsPlan {
    static constexpr int W = D / 32, STAGE_BYTES = Stage<W>::BYTES;
    static constexpr int STAGES = D <= 64 ? 3 : 2;
    static constexpr int RING = WARPS * STAGES * STAGE_BYTES;
    static constexpr int ROW = D + 4, JOIN = WARPS * 8 * NT * ROW * 4;  // (a row's output, maximum, sum; lanes store 16 bytes without bank conflicts)
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

// A run of stages of one request, kv head and tiles of query rows.
template <int NT>
struct Segment {
    int seq, head, t0, count, first;
    int base, end;       // cached rows
    float* part;         // where its rows leave their parts: row r at part + offset(r), or nullptr: the whole of it is here
    size_t row_stride;   // between the rows of a part, 0: by token and head
    Rows<NT> rows;
};

// The warps take the stages of the segment in turn, each with a ring of copies, a running maximum and a sum of its own, and
// are joined in shared memory in their order.
template <typename T, int D, int NT>
__device__ __forceinline__ void attend_segment(const PackedAttention& p, const Segment<NT>& seg, unsigned char* smem) {
    using Plan = RowsPlan<D, NT>;
    constexpr int W = D / 32, NP = sizeof(T) == 4 ? 2 : 1, STAGES = Plan::STAGES;  // NP: parts of a query row
    constexpr bool FULL = NP > 1;                                                   // weights times scales in 24 bits
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int head = seg.head, t0 = seg.t0, count = seg.count, first = seg.first, base = seg.base, end = seg.end;
    const int* table = p.tables + (size_t)seg.seq * p.width;
    const Rows<NT>& rows = seg.rows;
    float* scores = p.scores ? p.scores + ((size_t)seg.seq * p.cache.kv_heads + head) * p.max_stages * (STAGE * 8 * NT) + g * (8 * NT) + 2 * c : nullptr;

    unsigned char* ring = smem + warp * STAGES * Plan::STAGE_BYTES;
    uint32_t there[STAGES];
    const int begin = base + warp * STAGE;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        there[i] = Stage<W>::request(p, table, head, begin + i * WARPS * STAGE, end, ring + i * Plan::STAGE_BYTES, lane);

    Queries<T, W, NP> q[NT];
    float qs[NT][2];  // what makes a score of `scores` one to the base of 2
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = first + 8 * n + g;
        q[n].load((const T*)p.q + (size_t)(t0 + r / p.group) * p.ldq + (size_t)(head * p.group + r % p.group) * D, c, r < count, p.q_aligned);
        const float inv = p.scale / q[n].factor;
#pragma unroll
        for (int u = 0; u < 2; ++u) qs[n][u] = __shfl_sync(0xffffffffu, inv, 4 * (2 * c + u));
    }
    float o[NT][W][2][4] = {}, low_o[NT][W][2] = {}, m[NT][2], l[NT][2] = {};
    // of each group: a power of two no scale of values met so far is above, and what brings such scales to 2^6
    float v_top[W], v_fit[W];
#pragma unroll
    for (int j = 0; j < W; ++j) v_top[j] = 0.0f, v_fit[j] = 1.0f;
    uint32_t bad[NT] = {};             // groups whose output is not finite: bit j of column 2c, bit j + 8 of column 2c + 1
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -FLT_MAX;  // (finite: differences of it are numbers)

    int slot = 0;
    for (int at = begin; at < end; at += WARPS * STAGE) {
        {
            const int ahead = slot == 0 ? STAGES - 1 : slot - 1;  // the place that the stage before this one has left
            const uint32_t t = Stage<W>::request(p, table, head, at + (STAGES - 1) * WARPS * STAGE, end, ring + ahead * Plan::STAGE_BYTES, lane);
#pragma unroll
            for (int i = 0; i < STAGES; ++i)
                if (i == ahead) there[i] = t;
        }
        copy_wait<STAGES - 1>();
        __syncwarp();
        const unsigned char* stage = ring + slot * Plan::STAGE_BYTES;
        uint32_t here = 0;
#pragma unroll
        for (int i = 0; i < STAGES; ++i)
            if (i == slot) here = there[i];

        float s[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Keys<W> k;
            k.load(stage, KEYS * h, g, c);
            k.scores(q, c, s[h]);
        }
        const bool whole = at >= rows.all_low && at + STAGE <= rows.all_high && here == 0xffffffffu;
        uint32_t seen = 0xffffffffu;  // bit 4 n + 2 x + u of half h at 16 h
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][n][i] *= qs[n][i & 1];
        if (!whole) {
            seen = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = KEYS * h + g + 8 * (i >> 1);
                        if ((here >> r & 1) && at + r >= rows.low[n][i & 1] && at + r < rows.high[n][i & 1])
                            seen |= 1u << (16 * h + 4 * n + i);
                        else
                            s[h][n][i] = -INFINITY;
                    }
        }
        if (scores) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        *reinterpret_cast<float2*>(scores + (size_t)at * (8 * NT) + (KEYS * h + 8 * x) * (8 * NT) + 8 * n) = make_float2(s[h][n][2 * x], s[h][n][2 * x + 1]);
        }
        // The maximum is left behind by up to 2^8: only a score above that makes the warp find a new one and scale what it has.
        float high[NT][2];
        bool grew = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                high[n][u] = fmaxf(fmaxf(s[0][n][u], s[0][n][u + 2]), fmaxf(s[1][n][u], s[1][n][u + 2]));
                grew |= high[n][u] - 8.0f > m[n][u];
            }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float top = high[n][u];
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float now = fmaxf(m[n][u], top), f = exp2_fast(m[n][u] - now);
                    m[n][u] = now;
                    l[n][u] *= f;
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        low_o[n][j][u] *= f;
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            o[n][j][t][u] *= f;
                            o[n][j][t][u + 2] *= f;
                        }
                    }
                }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = exp2_fast(s[h][n][i] - m[n][i & 1]);
                    s[h][n][i] = e;
                    l[n][i & 1] += e;
                }

        if constexpr (!FULL) {  // a lane a row: whether any of the stage's scales is above what has been met
            uint32_t mine[W];
            load_words<W>(mine, stage + Stage<W>::VS_AT + lane * Stage<W>::S_ROW);
            bool greater = false;
#pragma unroll
            for (int j = 0; j < W; ++j) greater |= packed_scale(mine[j]) > v_top[j];
            if (__any_sync(0xffffffffu, greater)) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float top = warp_max(packed_scale(mine[j]));
                    if (!(top > v_top[j])) continue;  // (NaN is not)
                    // the next power of two, between 2^-120 and 2^127
                    const uint32_t e = min(max((__float_as_uint(top) >> 23) + 1, 7u), 254u);
                    const float now = __uint_as_float(e << 23), f = v_top[j] / now;
                    v_top[j] = now;
                    v_fit[j] = __uint_as_float((260u - e) << 23);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[n][j][t][i] *= f;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t vs[2][W];
#pragma unroll
            for (int u = 0; u < 2; ++u) load_words<W>(vs[u], stage + Stage<W>::VS_AT + (KEYS * h + g + 8 * u) * Stage<W>::S_ROW);
            if (!whole) {
                // A weight of nought would still carry NaN from a row that the query does not see: groups that are not finite
                // are taken out of the stage, and those outputs that do see them are marked.
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (packed_not_finite(vs[u][j])) {
                            vs[u][j] = 0;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint32_t sees = seen >> (16 * h + 4 * n + 2 * u);
                                bad[n] |= (sees & 1) << j | (sees >> 1 & 1) << (j + 8);
                            }
                        }
            }
            uint32_t word[4][(W + 1) / 2];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const unsigned char* src = stage + Stage<W>::V_AT + (KEYS * h + 2 * c + (u & 1) + 8 * (u >> 1)) * Stage<W>::V_ROW + 2 * W * g;
                if constexpr (W % 2 == 0) {
                    load_words<W / 2>(word[u], src);
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        const uint32_t v = reinterpret_cast<const uint16_t*>(src)[j];
                        word[u][j / 2] = j & 1 ? word[u][j / 2] | v << 16 : v;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float s0 = packed_scale(vs[0][j]) * v_fit[j], s1 = packed_scale(vs[1][j]) * v_fit[j];
                const float l0 = fmaf(8.0f, packed_scale(vs[0][j]), packed_least(vs[0][j])), l1 = fmaf(8.0f, packed_scale(vs[1][j]), packed_least(vs[1][j]));
                const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
                uint32_t a0[4], a1[4];
                const uint32_t w0 = __byte_perm(word[0][j / 2], word[1][j / 2], sel), w1 = __byte_perm(word[2][j / 2], word[3][j / 2], sel);
                if constexpr (FULL) {
                    code_pairs_bf16<8>(w0, a0);
                    code_pairs_bf16<8>(w1, a1);
                } else {
                    code_pairs<8>(w0, a0);
                    code_pairs<8>(w1, a1);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float(&pr)[4] = s[h][n];
                    low_o[n][j][0] = fmaf(pr[0], l0, fmaf(pr[2], l1, low_o[n][j][0]));
                    low_o[n][j][1] = fmaf(pr[1], l0, fmaf(pr[3], l1, low_o[n][j][1]));
                    float w[4] = {pr[0] * s0, pr[1] * s0, pr[2] * s1, pr[3] * s1};
                    // 32-bit rows: the tensor cores' sums are of sixteen rows each and are added up in rounded fp32 (theirs are cut off:
                    // over 2,600 rows of a warp 5e-5 of the output)
                    if constexpr (FULL) {
                        float fresh[2][4];
#pragma unroll
                        for (int i = 0; i < 3; ++i) {
                            const uint32_t x0 = pack_bf16(w[0], w[1]), x1 = pack_bf16(w[2], w[3]);
                            w[0] -= __uint_as_float(x0 << 16), w[1] -= __uint_as_float(x0 & 0xffff0000u);
                            w[2] -= __uint_as_float(x1 << 16), w[3] -= __uint_as_float(x1 & 0xffff0000u);
                            const uint32_t b0 = movmatrix_trans(x0), b1 = movmatrix_trans(x1);
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                const uint32_t a[4] = {a0[2 * t], a0[2 * t + 1], a1[2 * t], a1[2 * t + 1]};
                                if (i == 0)
                                    mma_bf16_16816_first(fresh[t], a, b0, b1);
                                else
                                    mma_bf16_16816(fresh[t], a, b0, b1);
                            }
                        }
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[n][j][t][i] += fresh[t][i];
                    } else {
                        const uint32_t b0 = movmatrix_trans(pack_f16(w[0], w[1])), b1 = movmatrix_trans(pack_f16(w[2], w[3]));
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const uint32_t a[4] = {a0[2 * t], a0[2 * t + 1], a1[2 * t], a1[2 * t + 1]};
                            mma_f16_16816(o[n][j][t], a, b0, b1);
                        }
                    }
                }
            }
        }
        __syncwarp();  // the next request overwrites the stage that has just been read
        slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
    copy_wait<0>();
    __syncthreads();  // the rings are read and written no more: the joined rows take their place

    // over the eight lanes of a column: sums, groups that are not finite; then the warp's part in shared memory
    float* joined = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            bad[n] |= __shfl_xor_sync(0xffffffffu, bad[n], x);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                l[n][u] += __shfl_xor_sync(0xffffffffu, l[n][u], x);
#pragma unroll
                for (int j = 0; j < W; ++j) low_o[n][j][u] += __shfl_xor_sync(0xffffffffu, low_o[n][j][u], x);
            }
        }
        float* mine = joined + (size_t)(warp * NT + n) * 8 * Plan::ROW;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float low = low_o[n][j][u], unit = FULL ? 1.0f : 0.015625f * v_top[j];  // the weights of bf16 rows were 2^6 / v_top times the true ones
                float4 v = make_float4(fmaf(o[n][j][0][u], unit, low), fmaf(o[n][j][0][u + 2], unit, low), fmaf(o[n][j][1][u], unit, low),
                                       fmaf(o[n][j][1][u + 2], unit, low));
                if (bad[n] >> (j + 8 * u) & 1) v = make_float4(NAN, NAN, NAN, NAN);
                *reinterpret_cast<float4*>(mine + (2 * c + u) * Plan::ROW + 32 * j + 4 * g) = v;
            }
            if (g == 0) {
                mine[(2 * c + u) * Plan::ROW + D] = m[n][u];
                mine[(2 * c + u) * Plan::ROW + D + 1] = l[n][u];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT * 8 / WARPS; ++i) {  // a warp joins every WARPS-th row
        const int at = i * WARPS + warp, r = first + at;
        if (r >= count) break;
        const int token = t0 + r / p.group, qh = head * p.group + r % p.group;
        const float* row = joined + (size_t)at * Plan::ROW;
        constexpr int NEXT = NT * 8 * Plan::ROW;
        float top = -FLT_MAX, sum = 0.0f, f[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, row[w * NEXT + D]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            f[w] = exp2_fast(row[w * NEXT + D] - top);
            sum += f[w] * row[w * NEXT + D + 1];
        }
        const bool partial = seg.part != nullptr;
        float* part = seg.part + (seg.row_stride ? (size_t)at * seg.row_stride : ((size_t)token * p.heads + qh) * (D + 2));
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            float acc = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) acc += f[w] * row[w * NEXT + 32 * j + lane];
            if (partial)
                part[32 * j + lane] = acc;
            else
                ((T*)p.out)[(size_t)token * p.ldo + (size_t)qh * D + 32 * j + lane] = from_float<T>(acc * inv);
        }
        if (lane == 0) {
            if (partial) {
                part[D] = top;
                part[D + 1] = sum;
            } else if (p.lse) {
                p.lse[(size_t)token * p.heads + qh] = sum == 0.0f ? INFINITY : top + log2f(sum);
            }
        }
    }
}

// Stages of 32 cached rows that a request's queries see together (at least one, so that every request has a block), from which on.
__device__ __forceinline__ int stages_of(const PackedAttention& p, int seq, int& floor) {
    const int t0 = max(p.q_start[seq], 0), n = min(p.q_start[seq + 1], p.tokens) - t0, start = p.start_row[seq];
    const int most = max(0, min(start + n, p.limit));
    const int least = min(p.window > 0 ? max(0, start - p.window + 1) : 0, most);
    floor = least / STAGE * STAGE;
    return n > 0 && n * p.group <= p.few ? max(1, (most - floor + STAGE - 1) / STAGE) : 0;
}

constexpr int EVEN_SEQS = 1024;      // most requests of a step whose stages are dealt out evenly
constexpr int EVEN_STAGES = WARPS;   // fewest stages of a block, so that each warp has one
constexpr int EVEN_RUN = 4 * WARPS;  // stages of a block from which on a block may go on with the next request

// How `units` stages are dealt out to about `most` blocks.  Long runs: block i gets stages i units / blocks up to (i + 1) units /
// blocks, whosever they are, and every block the same.  Shorter ones, where a second request would cost a block its
// start once more (8 requests of 4,096 rows: 20.7 us, in pieces 16.6): every request and kv head is cut into pieces of its own.
struct Deal {
    int units, blocks, chunk, runs;

    __device__ __forceinline__ Deal(int units, int most) : units(units) {
        blocks = min(most, max(1, units / EVEN_STAGES));
        chunk = max(EVEN_STAGES, (units + most - 1) / most);
        runs = chunk >= EVEN_RUN;
    }
    // blocks of a request's kv head (pieces)
    __device__ __forceinline__ int pieces(int stages) const { return (stages + chunk - 1) / chunk; }
    // the block that has unit u (runs)
    __device__ __forceinline__ int block_of(int u) const { return (int)((((long long)u + 1) * blocks - 1) / units); }
    __device__ __forceinline__ int begin_of(int block) const { return (int)((long long)block * units / blocks); }
    // where block i leaves its part of a request whose first part is in block `first`: a run may have two parts, one that
    // another block began and one that it begins itself
    __device__ __forceinline__ int place(int i, int first) const { return runs ? 2 * i + (i == first) : i; }
};

// A warp joins the parts first .. last of one query row in their order.
template <typename T, int D>
__device__ __forceinline__ void join_row(const PackedAttention& p, const Deal& deal, int first, int last, int rows, int r, int token, int qh, int lane) {
    constexpr int W = D / 32;
    const auto at = [&](int i) { return p.parts + ((size_t)deal.place(i, first) * rows + r) * (D + 2); };
    float top = -FLT_MAX;
    for (int i = first + lane; i <= last; i += 32) top = fmaxf(top, __ldcg(at(i) + D));
    top = warp_max(top);
    float acc[W] = {}, sum = 0.0f;
#pragma unroll 4
    for (int i = first; i <= last; ++i) {
        const float* part = at(i);
        const float f = exp2_fast(__ldcg(part + D) - top);
        sum += f * __ldcg(part + D + 1);
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] += f * __ldcg(part + 32 * j + lane);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int j = 0; j < W; ++j) ((T*)p.out)[(size_t)token * p.ldo + (size_t)qh * D + 32 * j + lane] = from_float<T>(acc[j] * inv);
    if (lane == 0 && p.lse) p.lse[(size_t)token * p.heads + qh] = sum == 0.0f ? INFINITY : top + log2f(sum);
}

// Grid (row tiles, kv heads, requests x splits): a block a segment.  Or, where the rows of every request fit one block's tiles
// (single tokens), a grid of as many blocks as the GPU holds: the stages of all requests and kv heads in a row, dealt out evenly
// whatever the requests' lengths; a request that several blocks share is joined by the last of them to finish, or by a kernel.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(WARPS * 32, D * NT <= 128 && sizeof(T) == 2 ? 2 : 1) packed_attention_rows_kernel(const PackedAttention p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int before[EVEN_SEQS + 1];  // stages (or pieces) of the requests before each one
    __shared__ int warp_total[2][WARPS], last_here;
    pdl_launch_dependents();
    pdl_wait();
    const int c = threadIdx.x & 3, limit = p.limit, me = blockIdx.x;
    Segment<NT> seg;
    Deal deal(WARPS, 1);
    int u = 0, stop = 1, s = 0;
    if (p.even) {
        constexpr int EACH = EVEN_SEQS / (WARPS * 32);  // requests of a thread
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        int mine[EACH], sum = 0, floor;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = threadIdx.x * EACH + i;
            mine[i] = at < p.seqs ? stages_of(p, at, floor) : 0;
            sum += mine[i];
        }
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) warp_total[0][warp] = sum;
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) sum += warp_total[0][w];
        deal = Deal(sum * p.cache.kv_heads, p.most_blocks);
        sum = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            mine[i] = p.cache.kv_heads * (deal.runs ? mine[i] : deal.pieces(mine[i]));
            sum += mine[i];
        }
        int upto = sum;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, x);
            if (lane >= x) upto += v;
        }
        if (lane == 31) warp_total[1][warp] = upto;
        __syncthreads();
        upto -= sum;
        for (int w = 0; w < warp; ++w) upto += warp_total[1][w];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            before[threadIdx.x * EACH + i] = upto;
            upto += mine[i];
        }
        if (threadIdx.x == WARPS * 32 - 1) before[EVEN_SEQS] = upto;
        __syncthreads();
        if (me >= (deal.runs ? deal.blocks : before[EVEN_SEQS])) return;
        u = deal.runs ? deal.begin_of(me) : me, stop = deal.runs ? deal.begin_of(me + 1) : me + 1;
    }
    while (u < stop) {
        int stages = 1, take = 1, from = 0, split = 0, first_part = 0, last_part = 0, done = 1;
        if (p.even) {
            for (int step = EVEN_SEQS / 2; step; step >>= 1)  // the last request that begins at or before u (and has any)
                if (s + step < EVEN_SEQS && before[s + step] <= u) s += step;
            int floor;
            stages = stages_of(p, s, floor);
            const int rel = u - before[s], n = deal.runs ? stages : deal.pieces(stages);
            seg.head = rel / n, seg.first = 0;
            const int i = rel - seg.head * n;
            if (deal.runs) {
                from = i, take = done = min(stages - from, stop - u);
                first_part = deal.block_of(u - from), last_part = deal.block_of(u - from + stages - 1);
            } else {
                from = (int)((long long)i * stages / n), take = (int)((long long)(i + 1) * stages / n) - from;
                first_part = me - i, last_part = first_part + n - 1;
            }
        } else {
            s = blockIdx.z / p.splits, split = blockIdx.z % p.splits, seg.head = blockIdx.y, seg.first = blockIdx.x * 8 * NT;
        }
        const int head = seg.head;
        seg.seq = s, seg.t0 = max(p.q_start[s], 0), seg.count = (min(p.q_start[s + 1], p.tokens) - seg.t0) * p.group;
        if (p.even) seg.count = min(seg.count, 8 * NT);  // (what the caller says no request exceeds)
        if (seg.first >= seg.count || (!p.even && seg.count > p.few)) return;  // (more rows than `few`: the other kernel's)
        seg.rows.set(p, seg.first, seg.count, p.start_row[s], limit, c);
        const int floor = seg.rows.least / STAGE * STAGE;
        if (!p.even) {
            stages = (seg.rows.most - floor + STAGE - 1) / STAGE;
            const int per = (stages + p.splits - 1) / p.splits;
            from = split * per, take = per;
        }
        seg.base = floor + from * STAGE, seg.end = min(seg.rows.most, seg.base + take * STAGE);
        const bool shared = p.even && take < stages;
        seg.part = shared ? p.parts + (size_t)deal.place(me, first_part) * (8 * NT) * (D + 2)
                          : !p.even && p.splits > 1 ? p.parts + (size_t)split * p.tokens * p.heads * (D + 2) : nullptr;
        seg.row_stride = p.even ? D + 2 : 0;
        attend_segment<T, D, NT>(p, seg, smem);
        if (shared && p.counters) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                int* counter = p.counters + s * p.cache.kv_heads + head;
                last_here = atomicAdd(counter, 1) == last_part - first_part;
                if (last_here) *counter = 0;  // for the next launch
                __threadfence();
            }
            __syncthreads();
            if (last_here)
                for (int r = threadIdx.x >> 5; r < seg.count; r += WARPS)
                    join_row<T, D>(p, deal, first_part, last_part, 8 * NT, r, seg.t0 + r / p.group, head * p.group + r % p.group, threadIdx.x & 31);
        }
        if (!p.even) return;
        __syncthreads();  // shared memory is free again
        u += done;
    }
    if (!p.counters && me == 0) {  // what the joining kernel needs
        int* to = (int*)(p.parts + (size_t)2 * gridDim.x * (8 * NT) * (D + 2));
        for (int i = threadIdx.x; i <= p.seqs; i += WARPS * 32) to[i] = before[i];
        if (threadIdx.x == 0) to[p.seqs + 1] = deal.units;
    }
}

// Block (row, kv head, request) joins the parts of one query row: the warps take them in turn and are added in their order.
template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32) packed_attention_join_even_kernel(const PackedAttention p, int grid) {
    constexpr int W = D / 32;
    __shared__ float tops[WARPS], sums[WARPS], outs[WARPS][D];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.x, head = blockIdx.y, s = blockIdx.z, rows = gridDim.x;
    const int* before = (const int*)(p.parts + (size_t)2 * grid * rows * (D + 2));
    const int t0 = max(p.q_start[s], 0), count = (min(p.q_start[s + 1], p.tokens) - t0) * p.group;
    if (r >= count || count > p.few) return;
    const Deal deal(before[p.seqs + 1], p.most_blocks);
    const int n = (before[s + 1] - before[s]) / p.cache.kv_heads, begin = before[s] + head * n;
    const int first = deal.runs ? deal.block_of(begin) : begin, last = deal.runs ? deal.block_of(begin + n - 1) : begin + n - 1;
    if (first == last) return;  // one block had all of it
    const auto at = [&](int i) { return p.parts + ((size_t)deal.place(i, first) * rows + r) * (D + 2); };
    float top = -FLT_MAX;
    for (int i = first + threadIdx.x; i <= last; i += WARPS * 32) top = fmaxf(top, at(i)[D]);
    top = warp_max(top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, tops[w]);
    float acc[W] = {}, sum = 0.0f;
#pragma unroll 4
    for (int i = first + warp; i <= last; i += WARPS) {
        const float* part = at(i);
        const float f = exp2_fast(part[D] - top);
        sum += f * part[D + 1];
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] += f * part[32 * j + lane];
    }
    if (lane == 0) sums[warp] = sum;
#pragma unroll
    for (int j = 0; j < W; ++j) outs[warp][32 * j + lane] = acc[j];
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += sums[w];
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int token = t0 + r / p.group, qh = head * p.group + r % p.group;
    for (int d = threadIdx.x; d < D; d += WARPS * 32) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += outs[w][d];
        ((T*)p.out)[(size_t)token * p.ldo + (size_t)qh * D + d] = from_float<T>(v * inv);
    }
    if (threadIdx.x == 0 && p.lse) p.lse[(size_t)token * p.heads + qh] = sum == 0.0f ? INFINITY : top + log2f(sum);
}

// Weights of the cached rows from the scores that the attention kernel has left: a thread a row.
__global__ void __launch_bounds__(256) packed_attention_scored_weights_kernel(const PackedAttention p, int cols) {
    pdl_launch_dependents();
    pdl_wait();
    const int head = blockIdx.y, seq = blockIdx.z, row = blockIdx.x * 256 + threadIdx.x;
    const int t0 = max(p.q_start[seq], 0), n = min(p.q_start[seq + 1], p.tokens) - t0, count = n * p.group, start = p.start_row[seq];
    const int end = min(min(start + n, p.limit), p.max_rows), slot = slot_of(p, seq);
    if (n <= 0 || count > p.few || count > cols || slot < 0) return;  // (the whole block)
    __shared__ float lse[16];  // of the request's query rows
    if (threadIdx.x < count)
        lse[threadIdx.x] = p.lse[(size_t)(t0 + threadIdx.x / p.group) * p.heads + head * p.group + threadIdx.x % p.group];
    __syncthreads();
    if (row >= end) return;
    int floor;
    stages_of(p, seq, floor);
    float total = 0.0f;
    if (row >= floor) {
        const float* s = p.scores + (((size_t)seq * p.cache.kv_heads + head) * p.max_stages * STAGE + row) * cols;
        for (int i = 0; i < cols && 4 * (i / 4) < count; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(s + i);
            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < count && x[k] != -INFINITY)  // (a row that is not seen, beside a sum that is not finite)
                    total += exp2_fast(x[k] - lse[i + k]);
        }
    }
    float* w = p.weights + slot * p.slot_stride + (long long)head * p.head_stride + row;
    *w = p.add && row < start ? *w + total : total;
}

// A warp joins the splits of one (token, head) in their order.
template <typename T, int D>
__global__ void __launch_bounds__(256) packed_attention_join_kernel(const PackedAttention p) {
    constexpr int W = D / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= (long long)p.tokens * p.heads || i < (long long)p.q_start[0] * p.heads || i >= (long long)p.q_start[p.seqs] * p.heads) return;
    const float* part = p.parts + (size_t)i * (D + 2);
    const size_t stride = (size_t)p.tokens * p.heads * (D + 2);
    float top = -FLT_MAX;
    for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, part[s * stride + D]);
    top = warp_max(top);
    float acc[W] = {}, sum = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
        const float f = exp2_fast(part[s * stride + D] - top);
        sum += f * part[s * stride + D + 1];
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] += f * part[s * stride + 32 * j + lane];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int token = (int)(i / p.heads), qh = (int)(i % p.heads);
#pragma unroll
    for (int j = 0; j < W; ++j)
        ((T*)p.out)[(size_t)token * p.ldo + (size_t)qh * D + 32 * j + lane] = from_float<T>(acc[j] * inv);
    if (lane == 0 && p.lse) p.lse[i] = sum == 0.0f ? INFINITY : top + log2f(sum);
}

// Weights of the cached rows:  w[key] (+)= sum over the request's queries and the kv head's query heads of
// exp2(s - lse), a warp 32 rows of the cache, the query rows in their order.
template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32) packed_attention_weights_kernel(const PackedAttention p) {
    constexpr int W = D / 32, NP = sizeof(T) == 4 ? 2 : 1;
    extern __shared__ __align__(16) unsigned char smem[];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int head = blockIdx.y, seq = blockIdx.z, at = (blockIdx.x * WARPS + warp) * STAGE;
    const int t0 = max(p.q_start[seq], 0), n = min(p.q_start[seq + 1], p.tokens) - t0, count = n * p.group, start = p.start_row[seq];
    const int limit = p.limit, end = min(min(start + n, limit), p.max_rows), slot = slot_of(p, seq);
    if (at >= end || n <= 0 || count > p.few || slot < 0) return;
    const int* table = p.tables + (size_t)seq * p.width;
    unsigned char* stage = smem + warp * Stage<W>::BYTES;
    const uint32_t there = Stage<W>::request(p, table, head, at, end, stage, lane);
    copy_wait<0>();
    __syncwarp();
    Keys<W> k[2];
    k[0].load(stage, 0, g, c);
    k[1].load(stage, KEYS, g, c);
    float total[2][2] = {};
    // from the first query row that sees the first of these cached rows
    for (int first = (int)min((long long)max(0, at - start) * p.group, (long long)count) / 8 * 8; first < count; first += 8) {
        Rows<1> rows;
        rows.set(p, first, count, start, limit, c);
        if (rows.least >= at + STAGE) break;  // with a window: this and all later rows have passed these
        if (rows.most <= at) continue;
        Queries<T, W, NP> q[1];
        const int r = first + g;
        q[0].load((const T*)p.q + (size_t)(t0 + r / p.group) * p.ldq + (size_t)(head * p.group + r % p.group) * D, c, r < count, p.q_aligned);
        const float inv = p.scale / q[0].factor;
        float qs[2], lse[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int col = first + 2 * c + u;
            qs[u] = __shfl_sync(0xffffffffu, inv, 4 * (2 * c + u));
            lse[u] = col < count ? p.lse[(size_t)(t0 + col / p.group) * p.heads + head * p.group + col % p.group] : INFINITY;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float s[1][4];
            k[h].scores(q, c, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int off = KEYS * h + g + 8 * (i >> 1), row = at + off;
                if ((there >> off & 1) && row >= rows.low[0][i & 1] && row < rows.high[0][i & 1])
                    total[h][i >> 1] += exp2_fast(s[0][i] * qs[i & 1] - lse[i & 1]);
            }
        }
    }
    float* w = p.weights + slot * p.slot_stride + (long long)head * p.head_stride;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float t = total[h][x];
            t += __shfl_xor_sync(0xffffffffu, t, 1);
            t += __shfl_xor_sync(0xffffffffu, t, 2);
            const int row = at + KEYS * h + g + 8 * x;
            if (c == 0 && row < end) w[row] = p.add && row < start ? w[row] + t : t;
        }
}

// How a step is cut.  bf16 portions of prompts with heads of 64 or 128 go to the 5th-generation tensor cores (packed_prefill.cu), the
// requests beside them that bring at most `few` query rows stay here; elsewhere all do.
// Tiles of eight query rows that a block takes: two where there are more rows than eight and the registers hold them.
struct Plan {
    int tiles, even, most, blocks, splits, join_kernel, few, here, prefill;
    PrefillPlan prompts;
    long long lse_floats, part_floats, score_floats, prompt_floats, counters;

    long long scratch() const { return lse_floats + part_floats + score_floats + prompt_floats; }
    long long all_counters() const { return counters + (prefill ? prompts.counters : 0); }
};

Plan make_plan(int dtype, int head_dim, int seqs, int kv_heads, int group, int tokens, int max_q, int max_kv, int weights) {
    const int sms = ferris_sm_count() > 0 ? ferris_sm_count() : 148;
    Plan q = {};
    const auto fours = [](long long floats) { return (floats + 3) / 4 * 4; };  // (what follows begins on 16 bytes)
    long long rows = (long long)max_q * group;
    q.few = 0x7fffffff, q.here = 1;
    if (dtype == FERRIS_BF16 && (head_dim == 64 || head_dim == 128) && rows > 16 && kv_heads <= 65535) {
        q.prefill = 1;
        q.few = group <= 8 ? 8 : group <= 16 ? 16 : 0;
        q.here = seqs > 1 && q.few > 0;
        if (!q.here) q.few = 0;  // (the tensor cores' kernel takes every request: max_q only bounds what they bring)
        q.prompts = packed_prefill_plan(head_dim, seqs, kv_heads, group, tokens, max_q, max_kv);
        q.prompt_floats = fours((q.prompts.bytes + 3) / 4);
        rows = q.few;
    }
    q.tiles = rows > 8 && (dtype == FERRIS_BF16 || head_dim <= 128) ? 2 : 1;
    const int per_sm = head_dim * q.tiles <= 128 && dtype == FERRIS_BF16 ? 2 : 1;
    const long long stages = max_kv / STAGE + 2, pairs = (long long)seqs * kv_heads;
    q.splits = 1;
    q.lse_floats = weights ? fours((long long)tokens * kv_heads * group) : 0;
    if (!q.here) return q;
    q.even = rows <= 8 * q.tiles && seqs <= EVEN_SEQS && pairs * stages < 0x7fffffff;
    if (q.even) {
        const long long most = pairs * stages / EVEN_STAGES;
        q.most = (int)(most < 1 ? 1 : most < sms * per_sm ? most : sms * per_sm);
        q.blocks = q.most + (int)pairs;  // (pieces: each request and kv head may have one that is not full)
        q.join_kernel = q.most > 32 * pairs;  // so many parts of a request that one block would be long at joining them
        q.part_floats = fours(2ll * q.blocks * 8 * q.tiles * (head_dim + 2) + (q.join_kernel ? seqs + 2 : 0));
        q.counters = q.join_kernel ? 0 : pairs;
        q.score_floats = weights ? pairs * stages * STAGE * 8 * q.tiles : 0;
        if (q.score_floats > (1ll << 27)) q.score_floats = 0;  // (above 512 MB the scores are formed again)
    } else {
        const long long blocks = pairs * ((rows + 8 * q.tiles - 1) / (8 * q.tiles));
        long long want = blocks > 0 ? (long long)sms * per_sm / blocks : 1;
        if (want > max_kv / (WARPS * STAGE)) want = max_kv / (WARPS * STAGE);
        if (want > 65535 / (seqs > 0 ? seqs : 1)) want = 65535 / (seqs > 0 ? seqs : 1);
        q.splits = want < 1 ? 1 : (int)want;
        q.part_floats = q.splits > 1 ? fours((long long)q.splits * tokens * kv_heads * group * (head_dim + 2)) : 0;
    }
    return q;
}

template <typename T, int D, int NT>
int attend_rows(const PackedAttention& p, const Plan& q, int max_q, cudaStream_t st) {
    auto kernel = packed_attention_rows_kernel<T, D, NT>;
    constexpr size_t smem = RowsPlan<D, NT>::SMEM;
    if (const int e = ferris_allow_dynamic_smem((const void*)kernel, smem)) return e;
    const long long rows = (long long)max_q * p.group < p.few ? (long long)max_q * p.group : p.few;  // of a request that this kernel takes
    const dim3 grid = q.even ? dim3(q.blocks) : dim3((unsigned)((rows + 8 * NT - 1) / (8 * NT)), p.cache.kv_heads, p.seqs * p.splits);
    return (int)ferris_launch(kernel, grid, dim3(WARPS * 32), smem, st, p);
}

template <typename T, int D>
int attend(const PackedAttention& p, const Plan& q, int max_q, int max_kv, void* prompt_scratch, int* prompt_counters, cudaStream_t st) {
    constexpr int MOST = sizeof(T) == 2 || D <= 128 ? 2 : 1;
    int e = 0;
    if (q.here) {
        e = q.tiles == 2 ? attend_rows<T, D, MOST>(p, q, max_q, st) : attend_rows<T, D, 1>(p, q, max_q, st);
        if (e == 0 && q.join_kernel)
            e = (int)ferris_launch(packed_attention_join_even_kernel<T, D>, dim3(8 * q.tiles, p.cache.kv_heads, p.seqs), dim3(WARPS * 32), 0, st, p, q.blocks);
        if (e == 0 && p.splits > 1)
            e = (int)ferris_launch(packed_attention_join_kernel<T, D>, dim3((unsigned)(((long long)p.tokens * p.heads + 7) / 8)), dim3(256), 0, st, p);
    }
    if (e == 0 && q.prefill) e = packed_prefill(p, q.prompts, max_kv, prompt_scratch, prompt_counters, st);
    if (e == 0 && p.weights && p.scores)
        e = (int)ferris_launch(packed_attention_scored_weights_kernel, dim3((max_kv + 255) / 256, p.cache.kv_heads, p.seqs), dim3(256), 0, st, p, 8 * q.tiles);
    if (e == 0 && p.weights && q.here && !p.scores) {
        auto kernel = packed_attention_weights_kernel<T, D>;
        constexpr size_t smem = (size_t)WARPS * Stage<D / 32>::BYTES;
        e = ferris_allow_dynamic_smem((const void*)kernel, smem);
        if (e == 0)
            e = (int)ferris_launch(kernel, dim3((max_kv + WARPS * STAGE - 1) / (WARPS * STAGE), p.cache.kv_heads, p.seqs), dim3(WARPS * 32), smem, st, p);
    }
    FERRIS_LAUNCH_CHECK();
}

template <typename T>
int attend_dim(const PackedAttention& p, const Plan& q, int max_q, int max_kv, void* ps, int* pc, cudaStream_t st) {
    switch (p.cache.head_dim) {
        case 32: return attend<T, 32>(p, q, max_q, max_kv, ps, pc, st);
        case 64: return attend<T, 64>(p, q, max_q, max_kv, ps, pc, st);
        case 96: return attend<T, 96>(p, q, max_q, max_kv, ps, pc, st);
        case 128: return attend<T, 128>(p, q, max_q, max_kv, ps, pc, st);
        case 160: return attend<T, 160>(p, q, max_q, max_kv, ps, pc, st);
        case 192: return attend<T, 192>(p, q, max_q, max_kv, ps, pc, st);
        case 224: return attend<T, 224>(p, q, max_q, max_kv, ps, pc, st);
        case 256: return attend<T, 256>(p, q, max_q, max_kv, ps, pc, st);
    }
    FERRIS_REFUSE("packed attention: heads of %d elements", p.cache.head_dim);
}

}  // namespace

// What a step needs: floats of scratch, counters (whole numbers that are nought, and are left so), launches.
FERRIS_API int ferris_packed_attention_plan(int dtype, int head_dim, int seqs, int kv_heads, int group, int tokens, int max_q, int max_kv,
                                            int weights, long long* needs) {
    const Plan q = make_plan(dtype, head_dim, seqs, kv_heads, group, tokens, max_q, max_kv, weights);
    needs[0] = q.scratch();
    needs[1] = q.all_counters();
    needs[2] = q.here + (q.join_kernel || q.splits > 1) + 2 * q.prefill + (weights ? q.here + q.prefill : 0);
    return FERRIS_OK;
}

// The arguments of ferris_packed_attention, as its caller lays them out: a call of this many arguments would cost its host
// more than the launch.
struct FerrisPackedAttention {
    const void* q;
    void *out, *k_codes, *k_scales, *v_codes, *v_scales;
    const int *tables, *q_start, *start_row;
    float* scratch;  // sums of the softmax (with weights), parts, scores, in this order
    int* counters;
    float* weights;
    const int* seq_slot;
    void* stream;
    long long slot_stride;
    int ldq, ldo, dtype, pages, kv_heads, page_size, head_dim, width, seqs, tokens, heads, max_q, max_kv, window, head_stride, max_rows, add,
        slots;
    float scale;
};

FERRIS_API int ferris_packed_attention(const FerrisPackedAttention* a) {
    PackedAttention p = {};
    p.cache = {(uint8_t*)a->k_codes, (uint32_t*)a->k_scales, (uint8_t*)a->v_codes, (uint32_t*)a->v_scales, a->pages, a->kv_heads, a->page_size,
               a->head_dim};
    if (const char* why = packed_cache_refusal(p.cache)) FERRIS_REFUSE("%s", why);
    if (a->heads <= 0 || a->heads % a->kv_heads) FERRIS_REFUSE("packed attention: %d heads over %d kv heads", a->heads, a->kv_heads);
    if (a->window < 0 || a->width <= 0 || a->max_kv <= 0)
        FERRIS_REFUSE("packed attention: window %d, %d blocks, at most %d rows", a->window, a->width, a->max_kv);
    if (a->seqs <= 0 || a->tokens <= 0 || a->max_q <= 0) return FERRIS_OK;
    if ((long long)a->width * a->page_size > 0x7fffffff - 16 * WARPS * STAGE) FERRIS_REFUSE("packed attention: %d blocks of %d rows", a->width, a->page_size);
    const Plan plan = make_plan(a->dtype, a->head_dim, a->seqs, a->kv_heads, a->heads / a->kv_heads, a->tokens, a->max_q, a->max_kv, a->weights != nullptr);
    if (plan.scratch() && !a->scratch) FERRIS_REFUSE("packed attention: no scratch");
    if (plan.all_counters() && !a->counters) FERRIS_REFUSE("packed attention: no counters");
    if (a->kv_heads > 65535 || (plan.here && !plan.even && (long long)a->seqs * plan.splits > 65535) || a->seqs > 65535)
        FERRIS_REFUSE("packed attention: %d requests of %d kv heads", a->seqs, a->kv_heads);
    p.q = a->q, p.out = a->out, p.ldq = a->ldq, p.ldo = a->ldo;
    p.q_aligned = ((uintptr_t)a->q & 15) == 0 && (long long)a->ldq * (a->dtype == FERRIS_BF16 ? 2 : 4) % 16 == 0;
    p.out_aligned = ((uintptr_t)a->out & 15) == 0 && (long long)a->ldo * (a->dtype == FERRIS_BF16 ? 2 : 4) % 16 == 0;
    p.scale = a->scale * LOG2E;
    if (!isfinite(p.scale)) FERRIS_REFUSE("packed attention: scale %g", (double)a->scale);
    p.few = plan.few;
    p.tables = a->tables, p.width = a->width, p.q_start = a->q_start, p.start_row = a->start_row;
    p.seqs = a->seqs, p.heads = a->heads, p.group = a->heads / a->kv_heads, p.window = a->window;
    p.lse = plan.lse_floats ? a->scratch : nullptr, p.parts = a->scratch + plan.lse_floats;
    p.scores = plan.score_floats ? a->scratch + plan.lse_floats + plan.part_floats : nullptr;
    p.splits = plan.splits, p.tokens = a->tokens;
    p.even = plan.even, p.most_blocks = plan.most, p.counters = plan.counters ? a->counters : nullptr;
    p.max_stages = a->max_kv / STAGE + 2;
    p.page = DivideBy(a->page_size);
    p.limit = a->width * a->page_size < a->max_kv ? a->width * a->page_size : a->max_kv;
    p.weights = a->weights, p.seq_slot = a->seq_slot, p.slots = a->slots, p.slot_stride = a->slot_stride, p.head_stride = a->head_stride, p.max_rows = a->max_rows, p.add = a->add;
    p.status = ferris_status_ptr();
    void* ps = a->scratch + (plan.scratch() - plan.prompt_floats);
    int* pc = a->counters + plan.counters;
    if (a->dtype == FERRIS_BF16) return attend_dim<bf16>(p, plan, a->max_q, a->max_kv, ps, pc, (cudaStream_t)a->stream);
    if (a->dtype == FERRIS_F32) return attend_dim<float>(p, plan, a->max_q, a->max_kv, ps, pc, (cudaStream_t)a->stream);
    FERRIS_REFUSE("packed attention: dtype %d is not known", a->dtype);
}
