// The probabilities that the sampler draws from: rows of logits under a temperature, top-k and top-p (the rules: sampling.cu).
//
// w_i = exp((l_i - max) / T); of the tokens, in descending order of their logits (the lower index first among equals), the first
// top_k stay, and of these the shortest prefix whose mass reaches top_p times the mass of all of them; p_i = w_i / mass of those that stay, 0 for
// the others.  Greedy rows (T <= 0, top_k == 1 or top_p <= 0): 1 at the greatest logit.  A logit that is NaN counts as minus infinity; where the greatest
// is infinite, those that equal it share the mass.
//
// Which tokens stay is decided on masses in 64 bits: w is computed in 64 bits and held as a whole number of 2^-45, so that sums are exact
// and do not depend on the order of additions, and borders fall as they do in exact arithmetic up to 2^-45 of the greatest weight.
//
// A cluster of eight blocks takes a row; each keeps its eighth in shared memory where it fits.  Rows without top-k and top-p are a softmax: the maximum, the sum, the quotients.  Otherwise
// a histogram of 1,024 bins, linear in the logit, finds the bin in which the top_k-th token, or the mass, falls (each block adds up an
// eighth of the bins of all blocks); the elements of that bin (with top_k <= 512 all from it upward) are gathered, at most 512, and ordered by counting for
// each what lies before it.  A bin of more elements is cut up by the digits of its elements' keys until one has no more than that.
#include <float.h>
#include <math.h>

#include "common.cuh"
#include "sm100.cuh"

namespace {

typedef unsigned long long u64;
typedef unsigned int u32;

constexpr int CLUSTER = 8, THREADS = 512, WARPS = THREADS / 32;
constexpr int BINS = 1024, OWN_BINS = BINS / CLUSTER;
constexpr int LIST = 512;    // elements that are ordered by counting
constexpr int DIGIT = 10;    // bits of a digit of the keys: a histogram's bins
constexpr double UNIT = 35184372088832.0;  // 2^45

__device__ __forceinline__ u64 ld_peer_shared_u64(const void* at, u32 rank) {
    u32 remote;
    u64 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(at)), "r"(rank));
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote) : "memory");
    return v;
}
__device__ __forceinline__ u32 ld_peer_shared_u32(const void* at, u32 rank) {
    u32 remote, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(at)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
    return v;
}

struct SamplingProbs {
    const float* logits;
    float* out;
    long long ldl, ldo;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    int vocab, per;  // elements of a block
};

struct Found {
    int bin;
    u32 count;             // of the bin
    u64 before_count, before_mass;  // of the bins above it
};

struct Entry {
    u64 key, mass;
};

struct Shared {
    u32 count[BINS];   // this block's histogram
    u64 mass[BINS];
    u32 own_count[OWN_BINS];  // the row's, of this block's eighth of the bins
    u64 own_mass[OWN_BINS];
    u64 total_count, total_mass;  // of these
    Found found;
    u64 best;          // the block's greatest key
    float least, sum;  // its least finite logit, its part of the softmax's sum
    u64 kept_mass;
    u32 listed;
    Entry list[LIST];  // this block's
    Entry all[LIST];   // the row's
    u64 threshold, retained;
    u64 red[WARPS];
    float fred[33];
};

// Ordered as the logits are, the lower index first among equals.
__device__ __forceinline__ u64 key_of(float l, int i) {
    const u32 u = __float_as_uint(l == 0.0f ? 0.0f : l);  // (both noughts are one)
    return (u64)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (u32)~(u32)i;
}
__device__ __forceinline__ float number(float l) { return l != l ? -INFINITY : l; }

struct Row {
    const float* at;  // this block's elements: shared memory, or the row itself
    int lo, n;        // the first one's index, their number
    float top, T, bins_per;

    __device__ __forceinline__ float logit(int i) const { return number(at[i]); }
    __device__ __forceinline__ double weight(float l) const {
        return l == top ? 1.0 : exp(((double)l - (double)top) / (double)T);
    }
    __device__ __forceinline__ u64 mass(float l) const { return (u64)__double2ull_rn(weight(l) * UNIT); }
    // The greatest logits in the highest bin; what lies below the histogram's range in bin 0.
    __device__ __forceinline__ int bin(float l) const {
        const float x = l == top ? 0.0f : (top - l) * bins_per;
        return BINS - 1 - (int)fminf(x, (float)(BINS - 1));
    }
};

__device__ __forceinline__ u64 block_sum_u64(Shared& s, u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 t = 0;
    for (int w = 0; w < WARPS; ++w) t += s.red[w];
    __syncthreads();
    return t;
}

// Which elements a search goes through: those of a bin of the linear histogram whose keys begin with some digits.
struct Subset {
    int bin = -1;  // -1: all
    u64 prefix = 0;
    int digits = 0;  // of the prefix
    static __device__ __forceinline__ int shift(int digit) { return 64 - DIGIT * (digit + 1); }  // (the last digit has four bits: below nought)
    static __device__ __forceinline__ int value(u64 key, int digit) {
        const int s = shift(digit);
        return (int)((s >= 0 ? key >> s : key << -s) & (BINS - 1));
    }
    __device__ __forceinline__ bool holds(const Row& r, float l, u64 key) const {
        if (bin >= 0 && r.bin(l) != bin) return false;
        return digits == 0 || (key >> shift(digits - 1)) == (prefix >> shift(digits - 1));
    }
};

// The histogram of a subset (linear for all elements, by the next digit of their keys for others) over the whole row: every block is
// left with its eighth of the bins, and with its sums.  Ends behind a barrier of the cluster.
template <bool MASS>
__device__ void histogram(Shared& s, const Row& r, const Subset& in) {
    for (int b = threadIdx.x; b < BINS; b += THREADS) {
        s.count[b] = 0;
        if (MASS) s.mass[b] = 0;
    }
    __syncthreads();
    u32 low = 0;  // what falls into bin 0 of the linear histogram, mostly far below all others: added up first
    u64 low_mass = 0;
    for (int i = threadIdx.x; i < r.n; i += THREADS) {
        const float l = r.logit(i);
        int b;
        if (in.bin < 0)
            b = r.bin(l);
        else {
            const u64 key = key_of(l, r.lo + i);
            if (!in.holds(r, l, key)) continue;
            b = Subset::value(key, in.digits);
        }
        const u64 m = MASS ? r.mass(l) : 0;
        if (in.bin < 0 && b == 0)
            ++low, low_mass += m;
        else {
            atomicAdd(&s.count[b], 1u);
            if (MASS) atomicAdd(&s.mass[b], m);
        }
    }
    if (low) {
        atomicAdd(&s.count[0], low);
        if (MASS) atomicAdd(&s.mass[0], low_mass);
    }
    cluster_sync();
    const u32 rank = cluster_ctarank();
    u64 c = 0, m = 0;
    if (threadIdx.x < OWN_BINS) {
        const int b = rank * OWN_BINS + threadIdx.x;
        for (int k = 0; k < CLUSTER; ++k) {
            c += ld_peer_shared_u32(&s.count[b], k);
            if (MASS) m += ld_peer_shared_u64(&s.mass[b], k);
        }
        s.own_count[threadIdx.x] = (u32)c;
        s.own_mass[threadIdx.x] = m;
    }
    c = block_sum_u64(s, c);
    if (MASS) m = block_sum_u64(s, m);
    if (threadIdx.x == 0) s.total_count = c, s.total_mass = m;
    cluster_sync();  // the sums are there; nobody reads the blocks' histograms any more
}

// The bin in which the running total of a histogram, from the highest bin down, first reaches `aim` (of counts, or of
// masses); the lowest that holds anything where it does not.  All blocks get the same.  Ends behind a barrier of the cluster.
__device__ Found find_bin(Shared& s, bool by_count, u64 aim) {
    u64 count[CLUSTER], mass[CLUSTER];
#pragma unroll
    for (int k = 0; k < CLUSTER; ++k) count[k] = ld_peer_shared_u64(&s.total_count, k), mass[k] = ld_peer_shared_u64(&s.total_mass, k);
    u64 c = 0, m = 0, before_c = 0, before_m = 0;
    int owner = -1;
#pragma unroll
    for (int k = CLUSTER - 1; k >= 0; --k) {
        // (the last block with anything in it that begins below the aim)
        if (count[k] && (owner < 0 || (by_count ? c : m) < aim)) owner = k, before_c = c, before_m = m;
        c += count[k], m += mass[k];
    }
    if (owner == (int)cluster_ctarank() && threadIdx.x < 32) {
        // four bins a lane, the highest first
        const int lane = threadIdx.x, top = OWN_BINS - 1 - 4 * lane;
        u64 pc = 0, pm = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) pc += s.own_count[top - k], pm += s.own_mass[top - k];
        u64 uc = pc, um = pm;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 tc = __shfl_up_sync(0xffffffffu, uc, o), tm = __shfl_up_sync(0xffffffffu, um, o);
            if (lane >= o) uc += tc, um += tm;
        }
        u64 ac = before_c + (uc - pc), am = before_m + (um - pm);
        int bin = -1;
        u64 bc = 0, bm = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const u32 n = s.own_count[top - k];
            if (n && (by_count ? ac : am) < aim) bin = top - k, bc = ac, bm = am;
            ac += n, am += s.own_mass[top - k];
        }
        const unsigned some = __ballot_sync(0xffffffffu, bin >= 0);
        const int last = 31 - __clz(some);
        if (lane == last) {
            s.found.bin = cluster_ctarank() * OWN_BINS + bin;
            s.found.count = s.own_count[bin];
            s.found.before_count = bc, s.found.before_mass = bm;
        }
    }
    cluster_sync();
    Found f;
    f.bin = (int)ld_peer_shared_u32(&s.found.bin, owner);
    f.count = ld_peer_shared_u32(&s.found.count, owner);
    f.before_count = ld_peer_shared_u64(&s.found.before_count, owner);
    f.before_mass = ld_peer_shared_u64(&s.found.before_mass, owner);
    return f;
}

// The elements that `in` holds (with `upward` those of higher bins too), `n` <= LIST of them in the row, into s.all of every block.
__device__ void gather(Shared& s, const Row& r, const Subset& in, bool upward, bool mass) {
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < r.n; i += THREADS) {
        const float l = r.logit(i);
        const u64 key = key_of(l, r.lo + i);
        if (upward ? r.bin(l) < in.bin : !in.holds(r, l, key)) continue;
        const u32 at = atomicAdd(&s.listed, 1u);
        if (at < LIST) s.list[at].key = key, s.list[at].mass = mass ? r.mass(l) : 0;
    }
    cluster_sync();
    u32 offset = 0;
    for (int k = 0; k < CLUSTER; ++k) {
        const u32 n = min(ld_peer_shared_u32(&s.listed, k), (u32)LIST);
        for (u32 i = threadIdx.x; i < n && offset + i < LIST; i += THREADS) {
            s.all[offset + i].key = ld_peer_shared_u64(&s.list[i].key, k);
            s.all[offset + i].mass = ld_peer_shared_u64(&s.list[i].mass, k);
        }
        offset += n;
    }
    cluster_sync();  // the lists are complete, and nobody's own is read any more
}

// ceil(p m), exactly, for 0 < p < 1: what a mass has to reach.
__device__ __forceinline__ u64 share_of(u64 m, float p) {
    const u32 bits = __float_as_uint(p);
    int e = (int)(bits >> 23);
    const u64 f = e ? (bits & 0x7fffffu) | 0x800000u : bits & 0x7fffffu;
    const int shift = 150 - (e ? e : 1);  // p = f 2^-shift, shift > 23
    const u64 lo = f * m, hi = __umul64hi(f, m);
    if (shift >= 128) return (lo | hi) != 0;
    u64 whole, rest;
    if (shift >= 64) {
        whole = shift == 64 ? hi : hi >> (shift - 64);
        rest = lo | (shift == 64 ? 0 : hi & ((1ull << (shift - 64)) - 1));
    } else {
        whole = lo >> shift | hi << (64 - shift);
        rest = lo & ((1ull << shift) - 1);
    }
    return whole + (rest != 0);
}

// The key of the element at which the running total reaches `aim`, and the mass up to and with it.
struct Quantile {
    u64 key, mass;
};

// From the row's linear histogram, which stands in the blocks' eighths (masses too where they are wanted).
__device__ Quantile quantile(Shared& s, const Row& r, bool by_count, u64 aim) {
    Found f = find_bin(s, by_count, aim);
    Subset in;
    in.bin = f.bin;
    u64 before_mass = f.before_mass;
    aim -= min(aim, by_count ? f.before_count : f.before_mass);
    while (f.count > LIST) {
        histogram<true>(s, r, in);
        f = find_bin(s, by_count, aim);
        const int shift = Subset::shift(in.digits);
        in.prefix |= shift >= 0 ? (u64)f.bin << shift : (u64)f.bin >> -shift;
        ++in.digits;
        before_mass += f.before_mass;
        aim -= min(aim, by_count ? f.before_count : f.before_mass);
    }
    gather(s, r, in, false, true);
    const int n = (int)f.count;
    if (threadIdx.x == 0) s.threshold = 0, s.retained = 0;
    __syncthreads();
    if ((int)threadIdx.x < n) {
        const Entry mine = s.all[threadIdx.x];
        u64 count = 0, mass = 0;
        for (int i = 0; i < n; ++i)
            if (s.all[i].key > mine.key) ++count, mass += s.all[i].mass;
        // the last one that begins below the aim: its predecessor's end lies below, and its own does not or nothing follows
        const u64 begins = by_count ? count : mass, ends = by_count ? count + 1 : mass + mine.mass;
        if ((begins < aim && ends >= aim) || (count == (u64)n - 1 && ends < aim)) s.threshold = mine.key, s.retained = mass + mine.mass;
    }
    __syncthreads();
    Quantile q = {s.threshold, before_mass + s.retained};
    __syncthreads();
    return q;
}

template <bool KEEP>  // the block's elements fit shared memory
__global__ void __launch_bounds__(THREADS) sampling_probs_kernel(const SamplingProbs a) {
    __shared__ Shared s;
    extern __shared__ __align__(16) float kept[];
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x;
    const u32 rank = cluster_ctarank();
    const float* logits = a.logits + (long long)row * a.ldl;
    float* out = a.out + (long long)row * a.ldo;
    const float T = a.temperature ? a.temperature[row] : 0.0f, p = a.top_p ? a.top_p[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const bool greedy = !(T > 0.0f) || k == 1 || !(p > 0.0f);
    Row r;
    r.lo = min(a.vocab, (int)rank * a.per), r.n = min(a.vocab, r.lo + a.per) - r.lo;
    r.at = KEEP ? kept : logits + r.lo;
    r.T = fmaxf(T, FLT_EPSILON);
    // fetch, greatest key, least finite logit
    u64 best = 0;
    float least = INFINITY;
    auto take = [&](float l, int i) {
        if (KEEP) kept[i] = l;
        l = number(l);
        const u64 key = key_of(l, r.lo + i);
        best = key > best ? key : best;
        if (l > -INFINITY) least = fminf(least, l);
    };
    if ((((uintptr_t)(logits + r.lo)) & 15) == 0) {
        const int whole = r.n & ~3;
        for (int i = 4 * threadIdx.x; i < whole; i += 4 * THREADS) {
            const float4 v = *reinterpret_cast<const float4*>(logits + r.lo + i);
            take(v.x, i), take(v.y, i + 1), take(v.z, i + 2), take(v.w, i + 3);
        }
        for (int i = whole + threadIdx.x; i < r.n; i += THREADS) take(logits[r.lo + i], i);
    } else
        for (int i = threadIdx.x; i < r.n; i += THREADS) take(logits[r.lo + i], i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 x = __shfl_xor_sync(0xffffffffu, best, o);
        best = x > best ? x : best;
    }
    least = -warp_max(-least);
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = best, s.fred[threadIdx.x >> 5] = least;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < WARPS; ++w) {
            best = s.red[w] > best ? s.red[w] : best;
            least = fminf(least, s.fred[w]);
        }
        s.best = best, s.least = least;
    }
    cluster_sync();
    best = 0, least = INFINITY;
#pragma unroll
    for (int c = 0; c < CLUSTER; ++c) {
        const u64 x = ld_peer_shared_u64(&s.best, c);
        best = x > best ? x : best;
        least = fminf(least, __uint_as_float(ld_peer_shared_u32(&s.least, c)));
    }
    const u32 ordered = (u32)(best >> 32);
    r.top = __uint_as_float(ordered & 0x80000000u ? ordered & 0x7fffffffu : ~ordered);
    u64 threshold = 0;    // the least key that stays
    float inv = 1.0f;     // of the softmax's sum (rows without top-k and top-p)
    double retained = 1.0;
    const bool by_k = !greedy && k > 0 && k < a.vocab, by_p = !greedy && p < 1.0f;
    if (greedy)
        threshold = best;
    else if (!by_k && !by_p) {
        float sum = 0.0f;
        for (int i = threadIdx.x; i < r.n; i += THREADS) {
            const float l = r.logit(i);
            sum += l == r.top ? 1.0f : expf((l - r.top) / r.T);
        }
        sum = block_sum(sum, s.fred);
        if (threadIdx.x == 0) s.sum = sum;
        cluster_sync();
        float total = 0.0f;
#pragma unroll
        for (int c = 0; c < CLUSTER; ++c) total += __uint_as_float(ld_peer_shared_u32(&s.sum, c));
        inv = 1.0f / total;
    } else {
        float range = r.top - least;
        if (!(range > 0.0f) || range == INFINITY) range = range == INFINITY ? FLT_MAX : 1.0f;
        // what weighs less than 2^-46 of the greatest has no mass: where only masses count, bin 0 takes all of it
        if (!by_k) range = fminf(range, 32.0f * r.T);
        r.bins_per = (float)(BINS - 1) / range;
        u64 mass = 0;
        const Subset all;
        bool listed = false;
        if (by_k) {
            if (k > LIST)
                histogram<true>(s, r, all);
            else {
                histogram<false>(s, r, all);
                const Found f = find_bin(s, true, (u64)k);
                if (f.before_count + f.count <= LIST) {  // they and all above them, ordered at once
                    Subset in;
                    in.bin = f.bin;
                    gather(s, r, in, true, true);
                    const int n = (int)(f.before_count + f.count);
                    if (threadIdx.x == 0) s.threshold = ~0ull, s.retained = 0, s.kept_mass = 0;
                    __syncthreads();
                    Entry mine = {0, 0};
                    u64 count = 0, before = 0;
                    const bool here = (int)threadIdx.x < n;
                    if (here) {
                        mine = s.all[threadIdx.x];
                        for (int i = 0; i < n; ++i)
                            if (s.all[i].key > mine.key) ++count, before += s.all[i].mass;
                        if (count == (u64)k - 1) s.kept_mass = before + mine.mass;
                    }
                    __syncthreads();
                    const u64 aim = by_p ? share_of(s.kept_mass, p) : ~0ull;
                    if (here && count < (u64)k && (count == 0 || before < aim)) {
                        atomicMin(&s.threshold, mine.key);
                        atomicMax(&s.retained, before + mine.mass);
                    }
                    __syncthreads();
                    threshold = s.threshold, mass = s.retained;
                    listed = true;
                }
            }
            if (!listed) {
                if (k <= LIST) histogram<true>(s, r, all);
                const Quantile q = quantile(s, r, true, (u64)k);
                threshold = q.key, mass = q.mass;
                if (by_p) histogram<true>(s, r, all);  // (the search may have cut a bin up in its place)
            }
        } else
            histogram<true>(s, r, all);
        if (by_p && !listed) {
            if (!by_k) {
                mass = 0;
#pragma unroll
                for (int c = 0; c < CLUSTER; ++c) mass += ld_peer_shared_u64(&s.total_mass, c);
            }
            u64 aim = share_of(mass, p);
            const Quantile q = quantile(s, r, false, aim ? aim : 1);
            threshold = q.key, mass = q.mass;
        }
        retained = (double)mass / UNIT;
    }
    // the probabilities
    auto of = [&](int i) -> float {
        const float l = r.logit(i);
        if (greedy) return key_of(l, r.lo + i) == threshold ? 1.0f : 0.0f;
        if (!by_k && !by_p) return l == r.top ? inv : expf((l - r.top) / r.T) * inv;
        return key_of(l, r.lo + i) >= threshold ? (float)(r.weight(l) / retained) : 0.0f;
    };
    out += r.lo;
    if (((uintptr_t)out & 15) == 0) {
        const int whole = r.n & ~3;
        for (int i = 4 * threadIdx.x; i < whole; i += 4 * THREADS)
            *reinterpret_cast<float4*>(out + i) = make_float4(of(i), of(i + 1), of(i + 2), of(i + 3));
        for (int i = whole + threadIdx.x; i < r.n; i += THREADS) out[i] = of(i);
    } else
        for (int i = threadIdx.x; i < r.n; i += THREADS) out[i] = of(i);
    cluster_sync();  // nobody leaves while others may read its shared memory
}

}  // namespace

// logits, out fp32 [rows, vocab] with row strides ldl, ldo: the same memory, or apart.  temperature, top_k, top_p: per row, or null for greedy rows.
FERRIS_API int ferris_sampling_probs(const float* logits, long long ldl, float* out, long long ldo, int rows, int vocab, const float* temperature,
                                     const int* top_k, const float* top_p, void* stream) {
    if (rows <= 0) return FERRIS_OK;
    if (vocab <= 0 || ldl < vocab || ldo < vocab || vocab > 0x7fffffff - 64) FERRIS_REFUSE("vocabulary %d, row strides %lld and %lld", vocab, ldl, ldo);
    SamplingProbs a = {logits, out, ldl, ldo, temperature, top_k, top_p, vocab, ((vocab + 4 * CLUSTER - 1) / (4 * CLUSTER)) * 4};
    const size_t bytes = (size_t)a.per * 4, most = 227 * 1024 - sizeof(Shared) - 1024;
    cudaError_t e;
    if (bytes <= most) {
        const int rc = ferris_allow_dynamic_smem((const void*)sampling_probs_kernel<true>, bytes);
        if (rc != FERRIS_OK) return rc;
        e = ferris_launch_cluster(sampling_probs_kernel<true>, dim3(rows, 1, CLUSTER), dim3(THREADS), bytes, (cudaStream_t)stream, CLUSTER, a);
    } else
        e = ferris_launch_cluster(sampling_probs_kernel<false>, dim3(rows, 1, CLUSTER), dim3(THREADS), 0, (cudaStream_t)stream, CLUSTER, a);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    FERRIS_LAUNCH_CHECK();
}
