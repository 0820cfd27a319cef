// Attention for trees of drafted tokens over the paged cache, bf16, on mma.sync (who sees what: tree_attention.cuh).
//
// Query rows are the rows of the MMAs, cached rows their columns, scores and outputs in registers:
//   S = Q K^T (K read as it lies, columns of the operand), P = 2^(S scale - m) rounded to bf16 (eight bits, as the output has; the sums
//   take them unrounded), O = O 2^(m_before - m) + P V (V transposed on its way out of shared memory).
// How the work is dealt out: tree_attention.cuh.
// In a block, WR warps share a tile of 16 WR cached rows, each with 16 MS query rows; NW / WR such groups take the tiles of a unit and have
// a ring of cp.async copies each.  Few query rows: every warp has its own tiles (WR = 1) and no barrier but at the end; many: the
// warps share tiles, so that shared memory is read less often.
// A tile that every query row sees whole is multiplied as it is.  In others scores that are not seen become nought weights; as nought times
// NaN is NaN, a tile of values that holds something not finite is multiplied element by element, by those who see it.
// What bounds it: few query rows, and what there is to read is little beside the chain of tables, pages, tiles and the join: a chain of five tokens after 999 rows (14 / 2
// heads of 64) 12.3 us, of which this kernel takes 9.5; 8 requests of one node after 4,096 rows 14.5, floor 1.3.  Longer steps approach the memory's rate: 32 requests
// of two nodes (28 / 4 heads of 128) 54 to 58 us for 268 MB, 4.6 to 5 TB/s.
#include "tree_attention.cuh"

namespace {

__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ float exp2_unit(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Sizes of a variant: heads padded to DP elements, MS slabs of 16 query rows to a warp, WR warps to a tile, NW warps.
template <int DP, int MS, int WR, int NW, int ST>
struct Plan {
    static constexpr int FETCH = NW == 4 ? 16 : 128 / NW;  // cached rows of a stage that a warp fetches
    static constexpr int GROUPS = NW / WR, TILE = FETCH * WR, UNIT = TILE * GROUPS, ROWS = 16 * MS * WR;
    static_assert(TILE % 16 == 0, "tiles of whole MMAs");
    static constexpr int ROW = DP * 2 + (DP % 64 ? 16 : 0);  // bytes of a row: eight rows of one 16-byte column lie on different banks
    static constexpr int RING = UNIT * 2 * ROW * ST;
    static constexpr int JOIN = NW * 16 * MS * (DP + 4) * 4;
    static constexpr int Q_AT = RING > JOIN ? RING : JOIN;
    static constexpr int SMEM = Q_AT + ROWS * ROW;
    static constexpr bool Q_HELD = MS * DP <= (NW == 16 ? 64 : 128);  // fragments of the query rows stay in registers
    static constexpr int BLOCKS = DP <= 64 && NW == 8 ? 2 : 1;
};

// Byte offset of a 16-byte column of a row.
template <int DP>
__device__ __forceinline__ uint32_t place(int row, int column) {
    if constexpr (DP % 64 == 0)
        return row * (DP * 2) + ((column ^ (row & 7)) << 4);
    else
        return row * (DP * 2 + 16) + (column << 4);
}

template <int DP, int MS, int WR, int NW, int ST>
__global__ void __launch_bounds__(NW * 32, Plan<DP, MS, WR, NW, ST>::BLOCKS) tree_attention_mma_kernel(const TreeAttention p) {
    using P = Plan<DP, MS, WR, NW, ST>;
    constexpr int KS = DP / 16, SUB = P::TILE < 32 ? P::TILE : 32, NT = SUB / 8, FETCH = P::FETCH;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ TreeLines tree;
    __shared__ TreeRequests requests;
    __shared__ uint32_t there[ST][NW];  // which of the cached rows that a warp fetched have a page
    __shared__ float row_m[NW][16 * MS], row_l[NW][16 * MS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = warp / WR, wr = warp % WR, D = p.head_dim;
    unsigned char* ring = smem + (size_t)group * P::TILE * 2 * P::ROW * ST;
    unsigned char* q_smem = smem + P::Q_AT;
    pdl_wait();
    pdl_launch_dependents();
    TreeWalk<P::UNIT, P::ROWS, true> walk;
    walk.know(p, requests);
    __syncthreads();
    walk.begin(p, requests, blockIdx.x, gridDim.x, 0);
    TreeItem item;
    int4 begun = walk.none();
    while (walk.next(p, requests, item)) {
        const TreeRequest r = item.request;
        const int head = item.head, count = r.nodes * p.group, row0 = item.block * P::ROWS;
        const int first = item.first, last = item.last, low = item.low;
        const bool whole_item = first == 0 && last == item.tiles;
        walk.note(item, begun);
        const int parent = tree_parent(p, r, threadIdx.x);
        const int* table = p.tables + (size_t)item.seq * p.width;
        // ---- cached rows on their way
        auto request = [&](int i) {
            const int s = i % ST;
            if (i < last) {
                const int row = (low + i) * P::UNIT + group * P::TILE + wr * FETCH + (lane & (FETCH - 1));
                const int page = row < r.rows ? tree_page(p, table, row) : -1;
                const size_t at = page >= 0 ? tree_row_at(p, page, head, row) : 0;
                const uint32_t live = __ballot_sync(0xffffffffu, page >= 0) & ((1u << FETCH) - 1);
                if (lane == 0) there[s][warp] = live;
                const uint32_t k_dst = smem_u32(ring + (size_t)(2 * s) * P::TILE * P::ROW), v_dst = k_dst + P::TILE * P::ROW;
                constexpr int CH = DP / 8;
#pragma unroll
                for (int c = 0; c < (FETCH * CH + 31) / 32; ++c) {
                    const int piece = c * 32 + lane, rr = piece / CH, column = piece % CH;
                    const size_t from = __shfl_sync(0xffffffffu, at, rr & (FETCH - 1)) + column * 8;
                    const bool ok = (live >> rr & 1) && column * 8 < D;
                    if (FETCH * CH % 32 == 0 || rr < FETCH) {
                        const uint32_t to = place<DP>(wr * FETCH + rr, column);
                        copy_async(k_dst + to, (const bf16*)p.k_cache + (ok ? from : 0), ok);
                        copy_async(v_dst + to, (const bf16*)p.v_cache + (ok ? from : 0), ok);
                    }
                }
            }
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) request(first + i);
        // ---- the block's query rows
        {
            const bf16* q = (const bf16*)p.q;
            const bool wide = ((uintptr_t)q & 15) == 0 && p.ldq % 8 == 0;
            constexpr int CH = DP / 8, EACH = (P::ROWS * CH + NW * 32 - 1) / (NW * 32);
            uint4 v[EACH];  // (all on their way at once)
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const int i = threadIdx.x + k * NW * 32, row = i / CH, column = i % CH, at = row0 + row;
                v[k] = make_uint4(0u, 0u, 0u, 0u);
                if (at < count && column * 8 < D && i < P::ROWS * CH) {
                    const unsigned short* src = (const unsigned short*)(q + (size_t)(r.first + at / p.group) * p.ldq + (head * p.group + at % p.group) * D + column * 8);
                    if (wide)
                        v[k] = *reinterpret_cast<const uint4*>(src);
                    else
                        v[k] = make_uint4(src[0] | (uint32_t)src[1] << 16, src[2] | (uint32_t)src[3] << 16, src[4] | (uint32_t)src[5] << 16, src[6] | (uint32_t)src[7] << 16);
                }
            }
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const int i = threadIdx.x + k * NW * 32;
                if (i < P::ROWS * CH) *reinterpret_cast<uint4*>(q_smem + place<DP>(i / CH, i % CH)) = v[k];
            }
        }
        // (the lines are only looked at where tiles are not seen whole: those of the tree, and with a window)
        if (p.window > 0 || (low + last) * P::UNIT > min(r.start, r.rows))
            tree_lines<NW * 32>(p, r, tree, parent, [] { __syncthreads(); });  // (ends with a barrier)
        else
            __syncthreads();
        int node[MS][2];
#pragma unroll
        for (int m = 0; m < MS; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = row0 + (wr * MS + m) * 16 + g + 8 * h;
                node[m][h] = at < count ? at / p.group : -1;
            }
        const bool live = row0 + wr * MS * 16 < count;  // any of the warp's rows
        uint32_t q_held[P::Q_HELD ? MS : 1][P::Q_HELD ? KS : 1][4];
        const uint32_t q_base = smem_u32(q_smem);
        auto load_q = [&](int m, int ks, uint32_t(&f)[4]) {
            ldmatrix_x4(f, q_base + place<DP>((wr * MS + m) * 16 + (lane & 7) + (lane >> 3 & 1) * 8, 2 * ks + (lane >> 4)));
        };
        if constexpr (P::Q_HELD) {
#pragma unroll
            for (int m = 0; m < MS; ++m)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) load_q(m, ks, q_held[m][ks]);
        }
        float o[MS][DP / 8][4], top[MS][2], sum[MS][2];
#pragma unroll
        for (int m = 0; m < MS; ++m) {
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.0f;
            top[m][0] = top[m][1] = -INFINITY, sum[m][0] = sum[m][1] = 0.0f;
        }
        // rows that all nodes see: from the first that the deepest node's window holds (not known: none) up to the text's end
        const int sure_low = p.window > 0 ? max(0, r.start + r.nodes - p.window) : 0, sure_high = min(r.start, r.rows);
        for (int i = first; i < last; ++i) {
            copy_wait<ST - 2>();
            if constexpr (WR == 1)
                __syncwarp();
            else
                asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(WR * 32) : "memory");
            request(i + ST - 1);
            if (!live) continue;
            const int s = i % ST;
            const uint32_t k_base = smem_u32(ring + (size_t)(2 * s) * P::TILE * P::ROW), v_base = k_base + P::TILE * P::ROW;
            const int tile0 = (low + i) * P::UNIT + group * P::TILE;
            if (tile0 >= r.rows) continue;
#pragma unroll 1
            for (int sub = 0; sub < P::TILE / SUB; ++sub) {
                const int key0 = tile0 + sub * SUB, at0 = sub * SUB;
                float x[MS][NT][4];
#pragma unroll
                for (int m = 0; m < MS; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) x[m][n][0] = x[m][n][1] = x[m][n][2] = x[m][n][3] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t a[MS][4];
#pragma unroll
                    for (int m = 0; m < MS; ++m) {
                        if constexpr (P::Q_HELD) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) a[m][e] = q_held[m][ks][e];
                        } else
                            load_q(m, ks, a[m]);
                    }
#pragma unroll
                    for (int n = 0; n < NT; n += 2) {
                        uint32_t b[4];
                        ldmatrix_x4(b, k_base + place<DP>(at0 + n * 8 + (lane >> 4) * 8 + (lane & 7), 2 * ks + (lane >> 3 & 1)));
#pragma unroll
                        for (int m = 0; m < MS; ++m) {
                            mma_bf16_16816(x[m][n], a[m], b[0], b[1]);
                            mma_bf16_16816(x[m][n + 1], a[m], b[2], b[3]);
                        }
                    }
                }
                uint32_t pages = 0;
#pragma unroll
                for (int k = 0; k < SUB / FETCH; ++k) pages |= there[s][group * WR + sub * (SUB / FETCH) + k] << (k * FETCH);
                const bool whole = key0 >= sure_low && key0 + SUB <= sure_high && pages == (SUB == 32 ? 0xffffffffu : 0xffffu);
                uint32_t sees[MS][2];
                if (!whole) {
#pragma unroll
                    for (int m = 0; m < MS; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) sees[m][h] = node[m][h] >= 0 ? tree_sees(p, r, tree, node[m][h], key0) & pages : 0u;
                }
                bool moved = false;
                float base[MS][2], corr[MS][2];
#pragma unroll
                for (int m = 0; m < MS; ++m) {
                    float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = x[m][n][e] * p.scale;
                            if (!whole && !(sees[m][e >> 1] >> (8 * n + 2 * t + (e & 1)) & 1)) v = -INFINITY;
                            x[m][n][e] = v;
                            most[e >> 1] = fmaxf(most[e >> 1], v);
                        }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
                        most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 2));
                        const float now = fmaxf(top[m][h], most[h]);
                        base[m][h] = now == -INFINITY ? 0.0f : now;
                        corr[m][h] = exp2_unit(top[m][h] - base[m][h]);
                        moved |= !(now == top[m][h]);
                        top[m][h] = now;
                    }
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int m = 0; m < MS; ++m) {
                        sum[m][0] *= corr[m][0], sum[m][1] *= corr[m][1];
#pragma unroll
                        for (int n = 0; n < DP / 8; ++n) {
                            o[m][n][0] *= corr[m][0], o[m][n][1] *= corr[m][0];
                            o[m][n][2] *= corr[m][1], o[m][n][3] *= corr[m][1];
                        }
                    }
                }
                uint32_t w[MS][NT][2];  // weights of (row g, two columns), (row g + 8, two columns)
#pragma unroll
                for (int m = 0; m < MS; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[m][n][e] = exp2_unit(x[m][n][e] - base[m][e >> 1]);
                        sum[m][0] += x[m][n][0] + x[m][n][1];
                        sum[m][1] += x[m][n][2] + x[m][n][3];
                        w[m][n][0] = pack_bf16(x[m][n][0], x[m][n][1]);
                        w[m][n][1] = pack_bf16(x[m][n][2], x[m][n][3]);
                    }
                bool careful = false;
                if (!whole) {
                    // whether the tile's values are all finite
                    uint32_t odd = 0;
                    for (int c = lane; c < SUB * (DP / 8); c += 32) {
                        uint4 v;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(v_base + place<DP>(at0 + c / (DP / 8), c % (DP / 8))));
                        const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) odd |= __vcmpeq2(word[k] & 0x7f807f80u, 0x7f807f80u);
                    }
                    careful = __any_sync(0xffffffffu, odd != 0);
                }
                if (!careful) {
#pragma unroll
                    for (int kk = 0; kk < SUB / 16; ++kk)
#pragma unroll
                        for (int n = 0; n < DP / 8; n += 2) {
                            uint32_t b[4];
                            ldmatrix_x4_trans(b, v_base + place<DP>(at0 + kk * 16 + (lane & 7) + (lane >> 3 & 1) * 8, n + (lane >> 4)));
#pragma unroll
                            for (int m = 0; m < MS; ++m) {
                                const uint32_t a[4] = {w[m][2 * kk][0], w[m][2 * kk][1], w[m][2 * kk + 1][0], w[m][2 * kk + 1][1]};
                                mma_bf16_16816(o[m][n], a, b[0], b[1]);
                                mma_bf16_16816(o[m][n + 1], a, b[2], b[3]);
                            }
                        }
                } else {
#pragma unroll
                    for (int q = 0; q < NT; ++q)  // (by registers' names: a place chosen at run time would put the weights into memory)
#pragma unroll 1
                        for (int j = 8 * q; j < 8 * q + 8; j += 2)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float f[MS][2];
#pragma unroll
                                for (int m = 0; m < MS; ++m)
#pragma unroll
                                    for (int h = 0; h < 2; ++h) f[m][h] = __shfl_sync(0xffffffffu, x[m][q][2 * h + e], (lane & ~3) | (j & 7) >> 1);
#pragma unroll
                                for (int n = 0; n < DP / 8; ++n) {
                                    uint32_t v;
                                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(v_base + place<DP>(at0 + j + e, n) + 4 * t));
                                    const float v0 = __uint_as_float(v << 16), v1 = __uint_as_float(v & 0xffff0000u);
#pragma unroll
                                    for (int m = 0; m < MS; ++m)
#pragma unroll
                                        for (int h = 0; h < 2; ++h)
                                            if (sees[m][h] >> (j + e) & 1) {
                                                o[m][n][2 * h] = fmaf(f[m][h], v0, o[m][n][2 * h]);
                                                o[m][n][2 * h + 1] = fmaf(f[m][h], v1, o[m][n][2 * h + 1]);
                                            }
                                }
                            }
                }
            }
        }
        // ---- the groups joined, in their order
        copy_wait<0>();
        __syncthreads();  // nobody reads the rings any more
        float* join = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int m = 0; m < MS; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float l = sum[m][h];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                if (t == 0) row_m[warp][m * 16 + g + 8 * h] = top[m][h], row_l[warp][m * 16 + g + 8 * h] = l;
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
                    *reinterpret_cast<float2*>(join + ((size_t)warp * 16 * MS + m * 16 + g + 8 * h) * (DP + 4) + n * 8 + 2 * t) =
                        make_float2(o[m][n][2 * h], o[m][n][2 * h + 1]);
            }
        __syncthreads();
        constexpr int QUADS = DP / 4;
        const bool pairs = ((uintptr_t)p.out & 3) == 0 && p.ldo % 2 == 0;
        for (int i = threadIdx.x; i < P::ROWS * QUADS; i += NW * 32) {
            const int row = i % P::ROWS, c = i / P::ROWS * 4, at = row0 + row;
            if (at >= count || c >= D) continue;
            const int w = row / (16 * MS), in = row % (16 * MS);  // the warps group * WR + w have it
            float m = -INFINITY, l = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int k = 0; k < P::GROUPS; ++k) m = fmaxf(m, row_m[k * WR + w][in]);
            const float b = m == -INFINITY ? 0.0f : m;
            for (int k = 0; k < P::GROUPS; ++k) {
                const float f = exp2_unit(row_m[k * WR + w][in] - b);
                const float4 x = *reinterpret_cast<const float4*>(join + ((size_t)(k * WR + w) * 16 * MS + in) * (DP + 4) + c);
                l = fmaf(f, row_l[k * WR + w][in], l);
                v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
            }
            if (whole_item) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                bf16* to = (bf16*)p.out + (size_t)(r.first + at / p.group) * p.ldo + (head * p.group + at % p.group) * D + c;
                if (pairs) {
                    reinterpret_cast<uint32_t*>(to)[0] = pack_bf16(v.x * inv, v.y * inv);
                    reinterpret_cast<uint32_t*>(to)[1] = pack_bf16(v.z * inv, v.w * inv);
                } else
                    to[0] = from_float<bf16>(v.x * inv), to[1] = from_float<bf16>(v.y * inv), to[2] = from_float<bf16>(v.z * inv), to[3] = from_float<bf16>(v.w * inv);
            } else {
                float* to = tree_part(p, blockIdx.x, first == 0, P::ROWS) + row;
                to[c * P::ROWS] = v.x, to[(c + 1) * P::ROWS] = v.y, to[(c + 2) * P::ROWS] = v.z, to[(c + 3) * P::ROWS] = v.w;
                if (c == 0) to[D * P::ROWS] = m, to[(D + 1) * P::ROWS] = l;
            }
        }
        __syncthreads();  // the rings and the query rows may be written again
    }
    if (threadIdx.x == 0) p.begun[blockIdx.x] = begun;
}

template <int DP, int MS, int WR, int NW, int ST>
int launch(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream) {
    using P = Plan<DP, MS, WR, NW, ST>;
    const auto kernel = tree_attention_mma_kernel<DP, MS, WR, NW, ST>;
    const int rc = ferris_allow_dynamic_smem((const void*)kernel, P::SMEM);
    if (rc != FERRIS_OK) return rc;
    const cudaError_t e = ferris_launch(kernel, dim3(plan.groups), dim3(NW * 32), (size_t)P::SMEM, stream, p);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    return FERRIS_OK;
}

// What goes with heads of D elements and a request's most query rows: f(variant's sizes as integral constants).
template <typename F>
void with_variant(int D, int rows, F f) {
#define TREE_VARIANT(DP, MS, WR, NW, ST) return f(std::integral_constant<int, DP>(), std::integral_constant<int, MS>(), std::integral_constant<int, WR>(), \
                                                  std::integral_constant<int, NW>(), std::integral_constant<int, ST>())
#define TREE_ROWS_OF(DP, ST)              \
    do {                                  \
        if (rows <= 16) TREE_VARIANT(DP, 1, 1, 8, ST); \
        if (rows <= 32) TREE_VARIANT(DP, 1, 2, 16, ST); \
        if (rows <= 64) TREE_VARIANT(DP, 1, 4, 16, ST); \
        TREE_VARIANT(DP, 1, 8, 16, 2);     \
    } while (0)
    if (D <= 32) TREE_ROWS_OF(32, 3);
    if (D <= 64) TREE_ROWS_OF(64, 3);
    if (D <= 96) TREE_ROWS_OF(96, 3);
    if (D <= 128) TREE_ROWS_OF(128, 3);
    if (D <= 192) {
        if (rows <= 16) TREE_VARIANT(192, 1, 1, 4, 3);
        TREE_VARIANT(192, 1, 4, 4, 3);
    }
    if (rows <= 16) TREE_VARIANT(256, 1, 1, 4, 3);
    TREE_VARIANT(256, 1, 4, 4, 2);
#undef TREE_ROWS_OF
#undef TREE_VARIANT
}

}  // namespace

TreePlan tree_plan(int head_dim, int seqs, int kv_heads, int group, int max_nodes, int max_kv, int page_size, long long cache_rows, float scale, int window) {
    TreePlan plan = {};
    int blocks = 1;  // of an SM
    with_variant(head_dim, max_nodes * group, [&](auto dp, auto ms, auto wr, auto nw, auto st) {
        using P = Plan<dp.value, ms.value, wr.value, nw.value, st.value>;
        plan.unit = P::UNIT, plan.rows = P::ROWS, blocks = P::BLOCKS;
    });
    // tcgen05 where its products outweigh what it takes to begin with: from 65 query rows on, from 17 where there are more than four units for an SM.  Microseconds,
    // mma.sync (with pages of 24 rows) and tcgen05: 8 requests after 4,096 rows, 14 / 2 heads of 64, 14 query rows 14.5 and 19.1, 56 rows 18.5 and 19.6, 70 rows 23.5 and
    // 20.2; 32 requests, 28 / 4 heads of 128, 14 rows 54 and 67, 28 rows 73 and 67, 56 rows 95 and 69, 112 rows 165 and 78.  With a window it is the units in it that count:
    // 32 requests after 16,384 rows, 14 / 2 heads of 64, 56 rows, window 128 12.5 and 18.2; 28 / 4 heads of 128, window 1,024 35.9 and 33.8; 64 requests, 300, 47 and 28.
    // (the row of a box that lies nowhere is a number too; a scale below nought would turn maxima into minima)
    const int rows = max_nodes * group, sms = ferris_sm_count();
    const bool many = rows > 64 || (rows > 16 && (long long)seqs * kv_heads * ((TreePlan::most_rows(max_kv, max_nodes, window, 128) + 127) / 128) > 4ll * (sms > 0 ? sms : 148));
    plan.tensor = many && (head_dim == 64 || head_dim == 128) && page_size % 16 == 0 && cache_rows < 0x7fffffff && scale > 0.0f && scale < 1e30f;
    if (plan.tensor) plan.unit = 128, plan.rows = rows > 128 ? 256 : 128, blocks = rows > 128 ? 1 : 2;  // (two groups to a block)
    plan.deal(seqs, kv_heads, group, max_nodes, plan.most_rows(max_kv, max_nodes, window, plan.unit), blocks, !plan.tensor);
    return plan;
}

int tree_attention_mma(const TreeAttention& p, const TreePlan& plan, cudaStream_t stream) {
    int rc = FERRIS_OK;
    with_variant(p.head_dim, p.max_nodes * p.group, [&](auto dp, auto ms, auto wr, auto nw, auto st) {
        rc = launch<dp.value, ms.value, wr.value, nw.value, st.value>(p, plan, stream);
    });
    return rc;
}
