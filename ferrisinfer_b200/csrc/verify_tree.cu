// Verification of trees of drafted tokens against the target's probabilities, from given random numbers.
//
// At a node x the target's distribution is r / R, at first r = p_x (its row of probabilities) and R = 1.  Its children are tried in
// their order; child c, drawn from the draft's distribution q_x, is accepted if u_c q_x(t_c) R < r(t_c), that is with the
// probability min(1, (r(t_c) / R) / q_x(t_c)), and the walk goes on from it.  Refused, it leaves the residual: r <- max(r - R q_x, 0), R <- sum r (where
// nothing is left, r and R stay).  A draft without probabilities has chosen its tokens for certain: q_x(t_c) = 1, r(t_c) <- 0, R <- R - r(t_c).
// Where no child is accepted the next token is drawn from r: the first i with sum_{j <= i} r_j > u_root sum_j r_j.  Chosen tokens may have been all that p_x had, and
// then, as R is a little more than what is left (32-bit probabilities do not quite add up to 1), even the last of them can be refused: it is the one that follows.  So tokens
// follow the target's distribution whatever was drafted.  All of it in 64 bits: at a border a rounding would be another token.
//
// A cluster of eight blocks takes a request, each an eighth of the vocabulary.  The tree, the random numbers and every node's p and q
// are fetched at once; each block then walks by itself, all of them the same way, and the blocks meet only where a row has to be gone through: after
// the refusal of a token that has a q, and for the last draw, whose passes leave the sums of every warp's run of elements, so that the draw goes
// through one run again.  Sums are added up in one order whatever the timing.
//
// What bounds it (151,936 tokens): one request 9.6 us, a chain of tables, one pass and the draw; 64 requests of 8 nodes with drafts' probabilities 45 to 56 us, as the random
// numbers have it (floor 12, every request's rows once): four to five passes a request with instructions in 64 bits and barriers of the cluster between, by 512 blocks of
// which 296 run at once.  A pass goes through all refusals of its node so far, so that the work grows with their square: it is small trees that are meant.  Taken back: the
// rows kept in shared memory between passes by clusters of sixteen (57 us where it took 47), blocks of 256 threads (54).
#include <math.h>

#include "common.cuh"
#include "sm100.cuh"

namespace {

constexpr int CLUSTER = 8, THREADS = 512, WARPS = THREADS / 32, NODES = 256;

struct VerifyTree {
    const float* probs;
    const float* draft;  // or nullptr
    long long ldp, ldd;
    const int* tokens;
    const int* parents;
    const int* q_start;
    const float* uniforms;
    int* out_nodes;
    int* out_accepted;
    int* out_token;
    int seqs, rows, vocab, width;
    int* status;
};

__device__ __forceinline__ void st_peer_shared_f64(uint32_t addr, uint32_t rank, double v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(v) : "memory");
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Whatever is no probability counts as none.
__device__ __forceinline__ float probability(float v) { return v > 0.0f ? v : 0.0f; }

struct Shared {
    float p[NODES], q[NODES], u[NODES];  // of each node's token in its parent's rows
    int token[NODES];
    short parent[NODES];
    double refused[NODES];   // R of each refusal that left a residual
    int gone[NODES];         // tokens that were refused without probabilities
    double part[2][WARPS];   // sums of the warps' runs of the last pass, by the parity of its number
    double block[2][CLUSTER];  // those of the row's blocks
};

struct Pass {
    const float* p;
    const float* q;
    int lo, hi;  // the warp's run
    bool aligned;
};

// What is left of elements after the refusals so far.
template <int N>
__device__ __forceinline__ void residuals(const Shared& s, int refusals, const float (&p)[N], const float (&q)[N], double (&r)[N]) {
    double qq[N];
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] = (double)probability(p[j]), qq[j] = (double)probability(q[j]);
    for (int k = 0; k < refusals; ++k) {
        const double left = s.refused[k];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const double x = __dsub_rn(r[j], __dmul_rn(left, qq[j]));  // (two roundings, as written)
            r[j] = x > 0.0 ? x : 0.0;
        }
    }
}

// Four neighbours from i on, of both rows; nought behind the run's end.
template <bool DRAFT>
__device__ __forceinline__ void fetch(const Pass& w, int i, float4& p, float4& q) {
    p = q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (w.aligned && i + 4 <= w.hi) {
        p = *reinterpret_cast<const float4*>(w.p + i);
        if (DRAFT) q = *reinterpret_cast<const float4*>(w.q + i);
    } else {
        if (i < w.hi) p.x = w.p[i], q.x = DRAFT ? w.q[i] : 0.0f;
        if (i + 1 < w.hi) p.y = w.p[i + 1], q.y = DRAFT ? w.q[i + 1] : 0.0f;
        if (i + 2 < w.hi) p.z = w.p[i + 2], q.z = DRAFT ? w.q[i + 2] : 0.0f;
        if (i + 3 < w.hi) p.w = w.p[i + 3], q.w = DRAFT ? w.q[i + 3] : 0.0f;
    }
}

// What is left of them.
template <bool DRAFT>
__device__ __forceinline__ void left_of(const Shared& s, int i, float4 p, float4 q, int refusals, int gone, double (&r)[4]) {
    if (!DRAFT)
        for (int g = 0; g < gone; ++g) {
            const unsigned at = (unsigned)(s.gone[g] - i);
            if (at == 0) p.x = 0.0f;
            if (at == 1) p.y = 0.0f;
            if (at == 2) p.z = 0.0f;
            if (at == 3) p.w = 0.0f;
        }
    const float ps[4] = {p.x, p.y, p.z, p.w}, qs[4] = {q.x, q.y, q.z, q.w};
    residuals(s, DRAFT ? refusals : 0, ps, qs, r);
}

// The sum of what is left of a warp's run, AHEAD groups of 128 elements on their way at once: two (five are more than registers have room for beside the doubles
// of two blocks an SM: 64 requests took 66 us, with three 51, with two 48).
template <bool DRAFT>
__device__ __forceinline__ double run_sum(const Shared& s, const Pass& w, int refusals, int gone) {
    constexpr int AHEAD = 2;
    double sum = 0.0, r[4];
    for (int i0 = w.lo + 4 * (threadIdx.x & 31); i0 < w.hi; i0 += 128 * AHEAD) {
        float4 p[AHEAD], q[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) fetch<DRAFT>(w, i0 + 128 * k, p[k], q[k]);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            left_of<DRAFT>(s, i0 + 128 * k, p[k], q[k], refusals, gone, r);
            sum += (r[0] + r[1]) + (r[2] + r[3]);
        }
    }
    return warp_sum64(sum);
}

__global__ void __launch_bounds__(THREADS, 2) verify_tree_kernel(const VerifyTree a) {
    __shared__ Shared s;
    cluster_arrive_relaxed();
    pdl_wait();
    pdl_launch_dependents();
    const int seq = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int first = min(max(a.q_start[seq], 0), a.rows);
    int n = min(max(a.q_start[seq + 1], first), a.rows) - first;
    if (n > NODES) {
        if (threadIdx.x == 0) ferris_report(a.status, FERRIS_STATUS_BAD_INDEX, 130);
        n = NODES;
    }
    const bool drafted = a.draft != nullptr;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        int up = a.parents[first + i];
        const int t = a.tokens[first + i];
        float p = 0.0f, q = 1.0f;
        if (i && (up >= i || up < -1)) {
            ferris_report(a.status, FERRIS_STATUS_BAD_INDEX, 131);
            up = -1;
        }
        if (i && up >= 0) {
            if (t < 0 || t >= a.vocab) {
                ferris_report(a.status, FERRIS_STATUS_BAD_INDEX, 132);
                up = -1;  // nobody's child
            } else {
                p = probability(a.probs[(first + up) * a.ldp + t]);
                if (drafted) q = probability(a.draft[(first + up) * a.ldd + t]);
            }
        }
        s.parent[i] = (short)(i ? up : -1), s.token[i] = t, s.p[i] = p, s.q[i] = q, s.u[i] = a.uniforms[first + i];
    }
    __syncthreads();
    cluster_wait();  // (all blocks have begun: their memory may be written)
    // this warp's run of elements: runs begin on four elements, and follow one another over the blocks of the cluster
    const int per = (((a.vocab + CLUSTER * WARPS - 1) / (CLUSTER * WARPS)) + 3) & ~3;
    Pass w;
    w.lo = min(a.vocab, (int)(rank * WARPS + warp) * per), w.hi = min(a.vocab, w.lo + per);
    int passes = 0;
    // the sum over the row of what is left, the same in all blocks; the runs' sums stay in s.part, the blocks' in s.block
    auto sum_up = [&](int refusals, int gone) {
        const int b = passes++ & 1;
        const double mine = refusals ? run_sum<true>(s, w, refusals, gone) : run_sum<false>(s, w, refusals, gone);
        if (lane == 0) s.part[b][warp] = mine;
        __syncthreads();
        if (threadIdx.x < CLUSTER) {
            // (every block's sum into every block's memory; nobody writes a half again before all have read it: there is a barrier of the cluster more between)
            double t = 0.0;
            for (int i = 0; i < WARPS; ++i) t += s.part[b][i];
            st_peer_shared_f64(smem_u32(&s.block[b][rank]), threadIdx.x, t);
        }
        cluster_sync();
        double t = 0.0;
        for (int i = 0; i < CLUSTER; ++i) t += s.block[b][i];
        return t;
    };
    int node = 0, path = 1, refusals = 0, gone = 0;
    int token = -1;  // the last of the refused ones that had a probability (drafts without probabilities)
    double left = 1.0, total = -1.0;  // total: of the last pass over what is left as it is now, below 0: none
    if (rank == 0 && threadIdx.x == 0 && n) a.out_nodes[(size_t)seq * a.width] = 0;
    auto look_at = [&](int x) {
        w.p = a.probs + (first + x) * a.ldp;
        w.q = drafted ? a.draft + (first + x) * a.ldd : w.p;
        w.aligned = (((uintptr_t)w.p | (uintptr_t)w.q) & 15) == 0;
    };
    if (n) look_at(0);
    for (int c = 1; c < n; ++c) {
        if (s.parent[c] != node || path == a.width) continue;
        double r;
        if (drafted) {
            const float ps[1] = {s.p[c]}, qs[1] = {s.q[c]};
            double rs[1];
            residuals(s, refusals, ps, qs, rs);
            r = rs[0];
        } else {
            r = s.p[c];
            for (int g = 0; g < gone; ++g)
                if (s.gone[g] == s.token[c]) r = 0.0;
        }
        if ((double)s.u[c] * (drafted ? (double)s.q[c] : 1.0) * left < r) {
            if (rank == 0 && threadIdx.x == 0) a.out_nodes[(size_t)seq * a.width + path] = c;
            node = c, ++path, refusals = 0, gone = 0, token = -1, left = 1.0, total = -1.0;
            look_at(c);
            continue;
        }
        // (the barrier keeps those who still read the list from those who add to it)
        __syncthreads();
        if (drafted) {
            if (threadIdx.x == 0) s.refused[refusals] = left;
            __syncthreads();
            const double t = sum_up(refusals + 1, 0);
            if (t > 0.0) ++refusals, left = t, total = t;
            else total = -1.0;  // (the sums of the runs are no longer those of what is left)
        } else {
            if (threadIdx.x == 0) s.gone[gone] = s.token[c];
            ++gone, left -= r;
            if (r > 0.0) token = s.token[c];
            __syncthreads();
        }
    }
    if (n && total < 0.0) total = sum_up(refusals, gone);
    if (n && total > 0.0) {
        const int b = (passes - 1) & 1;
        const double u = (double)s.u[0], aim = u > 0.0 ? u * total : 0.0;
        // the last block whose elements begin at or below the aim and hold anything; in it the last such run; in it the first element beyond the aim
        double before = 0.0, at = 0.0;
        int owner = -1;
        for (int i = 0; i < CLUSTER; ++i) {
            if (s.block[b][i] > 0.0 && at <= aim) owner = i, before = at;
            at += s.block[b][i];
        }
        if (owner == (int)rank && warp == 0) {
            at = before;
            int run = -1;
            for (int i = 0; i < WARPS; ++i) {
                if (s.part[b][i] > 0.0 && at <= aim) run = i, before = at;
                at += s.part[b][i];
            }
            w.lo = min(a.vocab, (int)(rank * WARPS + run) * per), w.hi = min(a.vocab, w.lo + per);
            int found = -1, last = -1;
            for (int i0 = w.lo; i0 < w.hi && found < 0; i0 += 128) {
                const int i = i0 + 4 * lane;
                double r[4] = {};
                if (i < w.hi) {
                    float4 p, q;
                    if (refusals) {
                        fetch<true>(w, i, p, q);
                        left_of<true>(s, i, p, q, refusals, gone, r);
                    } else {
                        fetch<false>(w, i, p, q);
                        left_of<false>(s, i, p, q, refusals, gone, r);
                    }
                }
                const double mine = (r[0] + r[1]) + (r[2] + r[3]);
                double upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double x = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += x;
                }
                double run_at = before + (upto - mine);
                int hit = -1, any = -1;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    run_at += r[k];
                    if (r[k] > 0.0) {
                        any = i + k;
                        if (hit < 0 && run_at > aim) hit = i + k;
                    }
                }
                const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, any >= 0);
                if (some) last = __shfl_sync(0xffffffffu, any, 31 - __clz(some));
                if (hits) found = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (lane == 0) a.out_token[seq] = found >= 0 ? found : last;
        }
    } else if (rank == 0 && threadIdx.x == 0)
        a.out_token[seq] = token;
    if (rank == 0) {
        if (threadIdx.x == 0) a.out_accepted[seq] = n ? path - 1 : 0;
        for (int i = (n ? path : 0) + threadIdx.x; i < a.width; i += THREADS) a.out_nodes[(size_t)seq * a.width + i] = -1;
    }
}

}  // namespace

// Arguments as ops.verify_tree lays them out.
struct VerifyTreeArgs {
    const void *probs, *draft, *tokens, *parents, *q_start, *uniforms, *out_nodes, *out_accepted, *out_token, *stream;
    long long ldp, ldd;
    int seqs, rows, vocab, width;
};

FERRIS_API int ferris_verify_tree(const VerifyTreeArgs* x) {
    if (x->seqs <= 0) return FERRIS_OK;
    if (x->rows < 0 || x->vocab <= 0 || x->width <= 0 || x->ldp < x->vocab || (x->draft && x->ldd < x->vocab))
        FERRIS_REFUSE("%d rows of %d probabilities, paths of %d nodes", x->rows, x->vocab, x->width);
    // (a request's blocks write while another's may not have begun to read)
    const long long ints = 4, paths = ints * x->seqs * x->width, each = ints * x->seqs, nodes = ints * x->rows;
    const struct { const void* at; long long bytes; } out[3] = {{x->out_nodes, paths}, {x->out_accepted, each}, {x->out_token, each}},
        in[6] = {{x->probs, x->rows ? 4 * ((x->rows - 1) * x->ldp + x->vocab) : 0}, {x->draft, x->draft && x->rows ? 4 * ((x->rows - 1) * x->ldd + x->vocab) : 0},
                 {x->tokens, nodes}, {x->parents, nodes}, {x->uniforms, nodes}, {x->q_start, each + 4}};
    for (int i = 0; i < 3; ++i) {
        for (int j = 0; j < i; ++j)
            if (ferris_share_memory(out[i].at, out[i].bytes, out[j].at, out[j].bytes)) FERRIS_REFUSE("the outputs must lie apart from one another");
        for (const auto& read : in)
            if (ferris_share_memory(out[i].at, out[i].bytes, read.at, read.bytes)) FERRIS_REFUSE("the outputs must lie apart from what is read");
    }
    VerifyTree a;
    a.probs = (const float*)x->probs, a.draft = (const float*)x->draft, a.ldp = x->ldp, a.ldd = x->ldd;
    a.tokens = (const int*)x->tokens, a.parents = (const int*)x->parents, a.q_start = (const int*)x->q_start;
    a.uniforms = (const float*)x->uniforms;
    a.out_nodes = (int*)const_cast<void*>(x->out_nodes), a.out_accepted = (int*)const_cast<void*>(x->out_accepted);
    a.out_token = (int*)const_cast<void*>(x->out_token);
    a.seqs = x->seqs, a.rows = x->rows, a.vocab = x->vocab, a.width = x->width;
    a.status = ferris_status_ptr();
    const cudaError_t e = ferris_launch_cluster(verify_tree_kernel, dim3(x->seqs, 1, CLUSTER), dim3(THREADS), 0, (cudaStream_t)x->stream, CLUSTER, a);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    FERRIS_LAUNCH_CHECK();
}
