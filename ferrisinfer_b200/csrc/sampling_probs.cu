// The probabilities that the sampler draws from: rows of logits under a temperature, top-k and top-p (the rules: sampling.cu).
//
// w_i = exp((l_i - max) / T); of the tokens, in descending order of their logits (the lower index first among equals), the first
// top_k stay, and of these the shortest prefix whose mass reaches top_p times the mass of all of them; p_i = w_i / mass of those that stay, 0 for
// the others.  Greedy rows (T <= 0, top_k == 1 or top_p <= 0): 1 at the greatest logit.  A logit that is NaN counts as minus infinity; where the greatest
// is infinite, those that equal it share the mass.
//
// Which tokens stay is decided on masses in 64 bits: w is computed in 64 bits and held as a whole number of 2^-45 (of 2^-44 from 2^19 tokens on, whose masses would
// add up to 2^64 otherwise), so that sums are exact and do not depend on the order of additions.  A weight is off by half of that and by 2^-46 of itself (what is below
// 2^-46 counts as nothing), and a border lies where it does for a mass that is off by as much for every token: 2^-28.8 of the greatest weight for 151,936.
//
// A cluster of up to eight blocks takes a row; each keeps its share in shared memory where it fits (two blocks to an SM), so that a row is read once and written once.
//   neither top-k nor top-p   a softmax in 32 bits: the maximum, the exponentials and their sum, the quotients
//   top_k <= 512              the top_k-th of the threads' own maxima bounds the top_k-th logit from below, and few logits lie above it: a histogram of the maxima
//                             (one a thread), the logits from the bin of the top_k-th on gathered, ordered by counting for each what lies before it
//   top-p alone               masses above seven bounds (each thread's in registers) say between which two the border lies; a histogram of what lies there,
//                             linear in the logit, in which bin; the bin's elements are gathered and ordered in the same way
//   otherwise                 a histogram of the whole row
// A bin of more than 512 elements is cut up by the digits of its elements' keys until one has no more.
//
// What bounds it (151,936 tokens): 512 plain rows 120 us, 5.2 TB/s (floor 95); 40 rows by mass 57 us (floor 7.4), where the pass of masses in 64 bits takes 55
// instructions an element and most of the time, and some ten barriers of the cluster are waited for; five rows with top-k and top-p 15.5 us, those barriers and a launch.
// 512 rows in waves of clusters: top-k 20 and top-p 313 us, by mass 662, top-k 3,001 and top-p 1,006.
#include <float.h>
#include <math.h>

#include "common.cuh"
#include "sm100.cuh"

namespace {

typedef unsigned long long u64;
typedef unsigned int u32;

constexpr int MOST_BLOCKS = 8, THREADS = 512, WARPS = THREADS / 32;
constexpr int BINS = 512, OWN_BINS = 128;  // a block adds up BINS / blocks of the row's bins: at most a quarter
constexpr int LEAST_BLOCKS = BINS / OWN_BINS;
constexpr int LIST = THREADS;  // elements that are ordered by counting, one a thread
constexpr int DIGIT = 9;    // bits of a digit of the keys: a histogram's bins
constexpr int BOUNDS = 7;
constexpr int MOST_ELEMENTS = 65536;  // of a block
constexpr int MASS_BITS = 45;  // a row's masses are below 2^64 with them up to 2^19 - 1 tokens
constexpr u64 MASS_OFFSET = 0x4330000000000000ull;  // the bits of 2^52
constexpr double LOG2E = 1.4426950408889634;

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
__device__ __forceinline__ void st_peer_shared_u32(const void* at, u32 rank, u32 v) {
    u32 remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(at)), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
__device__ __forceinline__ void st_peer_shared_u64(const void* at, u32 rank, u64 v) {
    u32 remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(at)), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(v) : "memory");
}
__device__ __forceinline__ u32 cluster_blocks() {
    u32 n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}

struct SamplingProbs {
    const float* logits;
    float* out;
    long long ldl, ldo;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    int vocab, per;  // elements of a block
    int rows, skip;  // skip: rows without top-k and top-p are another kernel's
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
    union {
        struct {
            u32 count[BINS];  // this block's histogram; masses by their lower, middle and upper sixteen bits (additions of 32 bits are native, of 64 are not)
            u32 mass[3][BINS];
        };
        Entry list[LIST];  // this block's elements of a bin, when the histograms have been added up
        Entry all[LIST];   // and then the row's, when nobody reads the others' any more
    };
    u32 own_count[OWN_BINS];  // the row's, of this block's bins
    u64 own_mass[OWN_BINS];
    // what blocks tell each other, by the teller's rank (stores into the others' memory; reading it from there takes thousands of cycles)
    u64 total_count[MOST_BLOCKS], total_mass[MOST_BLOCKS];  // of its bins
    Found found;
    float value[4][MOST_BLOCKS];
    float above[MOST_BLOCKS][BOUNDS + 1];  // masses above the bounds, and of all
    u64 over[MOST_BLOCKS], sum[MOST_BLOCKS];
    u32 index[MOST_BLOCKS], listed[MOST_BLOCKS];
    float parts[WARPS][BOUNDS + 1];
    u32 count_listed;
    double powers[32];  // the weight of the greatest logit, times 2^(j / 32)
    u64 threshold, retained, kept_mass;
    u64 red[2][WARPS];
    float fred[4][WARPS], scratch[33];
};

// Ordered as the logits are, the lower index first among equals.
__device__ __forceinline__ u32 order_of(float l) {
    const u32 u = __float_as_uint(l + 0.0f);  // (both noughts are one)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(u32 order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }
__device__ __forceinline__ u64 key_of(float l, int i) { return (u64)order_of(l) << 32 | (u32)~(u32)i; }

__device__ __forceinline__ float exp2_unit(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ const double powers_of_two[32] = {  // 2^(j / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};

// unit 2^(z / 32) + 2^52 for -6000 <= z <= 0, up to 2^-46 of the power: the nearest whole number apart, of which five bits choose one of unit 2^(0/32) .. unit 2^(31/32)
// (`powers`) and the others are the exponent, and the Taylor polynomial of 2^(f / 32) for |f| <= 1/2, whose sixth term is 2e-15.
__device__ __forceinline__ double exp2_64_whole(double z, const double* powers) {
    const double magic = 6755399441055744.0;  // 1.5 x 2^52: adding it rounds to a whole number
    const double t = z + magic, f = z - (t - magic);
    double r = 3.9737099845494154e-11;  // (ln(2) / 32)^k / k! for k = 5 .. 0
    r = fma(r, f, 9.172562701824643e-09);
    r = fma(r, f, 1.6938509724371819e-06);
    r = fma(r, f, 0.00023459619820224677);
    r = fma(r, f, 0.02166084939249829);
    r = fma(r, f, 1.0);
    const int n = __double2loint(t);
    const double power = powers[n & 31];
    return fma(r, __hiloint2double(__double2hiint(power) + (n >> 5) * (1 << 20), __double2loint(power)), 4503599627370496.0);
}

struct Row {
    const float* at;  // this block's elements: shared memory, or the row itself
    int lo, n;        // the first one's index, their number
    bool odd;         // a NaN counts as minus infinity; where the greatest logit is infinite or near that, the others stand as their distance from it (at 0)
    float given_top;  // the greatest logit as it is,
    float top;        // and as it stands
    float high, bins_per;  // where the linear histogram begins, bins per unit of logit
    float least;      // what lies below has no mass: 2^-86 of the greatest weight
    double rate;      // 32 log2(e) / T
    const double* powers;

    __device__ __forceinline__ float number(float l) const {
        if (!odd) return l;
        l = fmaxf(l, -INFINITY);
        return fabsf(given_top) < 1e37f ? l : l == given_top ? 0.0f : l - given_top;
    }
    __device__ __forceinline__ float logit(int i) const { return number(at[i]); }
    // (with 2^52 it is rounded to a whole number, which the lower bits are; MASS_OFFSET are the others)
    __device__ __forceinline__ u64 mass_and_offset(float l) const {
        return (u64)__double_as_longlong(exp2_64_whole(((double)fmaxf(l, least) - (double)top) * rate, powers));
    }
    __device__ __forceinline__ u64 mass(float l) const { return mass_and_offset(l) - MASS_OFFSET; }
    // The greatest logits in the highest bin; what lies below the histogram's range in bin 0.
    __device__ __forceinline__ float depth(float l) const { return l >= high ? 0.0f : (high - l) * bins_per; }
    __device__ __forceinline__ int bin(float l) const { return BINS - 1 - (int)fminf(depth(l), (float)(BINS - 1)); }
    // Logits between which all of a bin's lie, a bin more to each side: most elements are told apart by them alone.
    __device__ __forceinline__ float below_bin(int b) const { return b == 0 ? -INFINITY : high - (float)(BINS + 1 - b) / bins_per; }
    __device__ __forceinline__ float above_bin(int b) const { return b >= BINS - 2 ? INFINITY : high - (float)(BINS - 3 - b) / bins_per; }
    // (the same comparisons without a bin's number)
    __device__ __forceinline__ bool from_bin_on(float l, int b) const { return b == 0 || depth(l) < (float)(BINS - b); }
    __device__ __forceinline__ bool in_bin(float l, int b) const { return from_bin_on(l, b) && (b == BINS - 1 || depth(l) >= (float)(BINS - 1 - b)); }
};

// f(logit, index) for all elements of the block.  (One by one: what a row goes through once is fetched once, and four elements at a time, four times the
// instructions, took longer: 40 rows by mass 97 us for 85.)
template <typename F>
__device__ __forceinline__ void each(const Row& r, F f) {
#pragma unroll 1
    for (int i = threadIdx.x; i < r.n; i += THREADS) f(r.logit(i), r.lo + i);
}

// Sums over the block and over the row's blocks, for all threads; the one ends behind a barrier of the block, the others are of what the blocks have told (a
// barrier of the cluster in between).
__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// (of two numbers at once)
__device__ __forceinline__ void block_sum_u64(Shared& s, u64& v, u64& w) {
    const int lane = threadIdx.x & 31;
    v = warp_sum_u64(v), w = warp_sum_u64(w);
    if (lane == 0) s.red[0][threadIdx.x >> 5] = v, s.red[1][threadIdx.x >> 5] = w;
    __syncthreads();
    v = warp_sum_u64(lane < WARPS ? s.red[0][lane] : 0), w = warp_sum_u64(lane < WARPS ? s.red[1][lane] : 0);
    __syncthreads();
}
__device__ __forceinline__ u64 row_sum_u64(const u64* at) {
    const u32 lane = threadIdx.x & 31;
    return warp_sum_u64(lane < cluster_blocks() ? at[lane] : 0);
}
__device__ __forceinline__ float row_value(const float* at, float none) {
    const u32 lane = threadIdx.x & 31;
    return lane < cluster_blocks() ? at[lane] : none;
}
// By all threads of the first warp: a number of this block's to all of the row's.
__device__ __forceinline__ void tell(float* at, float v) {
    const u32 lane = threadIdx.x & 31;
    if (lane < cluster_blocks()) st_peer_shared_u32(at + cluster_ctarank(), lane, __float_as_uint(v));
}
__device__ __forceinline__ void tell(u32* at, u32 v) {
    const u32 lane = threadIdx.x & 31;
    if (lane < cluster_blocks()) st_peer_shared_u32(at + cluster_ctarank(), lane, v);
}
__device__ __forceinline__ void tell(u64* at, u64 v) {
    const u32 lane = threadIdx.x & 31;
    if (lane < cluster_blocks()) st_peer_shared_u64(at + cluster_ctarank(), lane, v);
}
// (`place`: every call its own)
__device__ __forceinline__ float block_max(Shared& s, int place, float v) {
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) s.fred[place][threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_max(s.fred[place][threadIdx.x & (WARPS - 1)]);
}

// Which elements a search goes through: those between two logits, of a bin of the linear histogram, whose keys begin with some digits.
struct Subset {
    float low = -INFINITY, high = INFINITY;  // low < l <= high (or all that is at least minus infinity)
    int bin = -1;  // -1: all
    u64 prefix = 0;
    int digits = 0;  // of the prefix
    static __device__ __forceinline__ int shift(int digit) { return 64 - DIGIT * (digit + 1); }  // (the last digit has one bit: below nought)
    static __device__ __forceinline__ int value(u64 key, int digit) {
        const int s = shift(digit);
        return (int)((s >= 0 ? key >> s : key << -s) & (BINS - 1));
    }
    __device__ __forceinline__ bool between(float l) const { return l <= high && (l > low || low == -INFINITY); }
    __device__ __forceinline__ bool holds(const Row& r, float l, int i) const {
        if (!between(l) || (bin >= 0 && !r.in_bin(l, bin))) return false;
        return digits == 0 || (key_of(l, i) >> shift(digits - 1)) == (prefix >> shift(digits - 1));
    }
};

// The histogram of a block adds up to the row's: every block is left with its share of the bins, and with its sums.  Ends behind a barrier of the cluster.
template <bool MASS>
__device__ void add_up(Shared& s) {
    cluster_sync();
    const u32 rank = cluster_ctarank(), blocks = cluster_blocks();
    const int first = rank * BINS / blocks, own = (rank + 1) * BINS / blocks - first;
    u64 c = 0, m = 0;
    if ((int)threadIdx.x < own) {
        const int b = first + threadIdx.x;
        u32 cc[MOST_BLOCKS];
        u64 mm[MOST_BLOCKS];
#pragma unroll
        for (int k = 0; k < MOST_BLOCKS; ++k) {
            cc[k] = k < (int)blocks ? ld_peer_shared_u32(&s.count[b], k) : 0;
            mm[k] = 0;
            if (MASS && k < (int)blocks)
                mm[k] = ld_peer_shared_u32(&s.mass[0][b], k) + ((u64)ld_peer_shared_u32(&s.mass[1][b], k) << 16) + ((u64)ld_peer_shared_u32(&s.mass[2][b], k) << 32);
        }
#pragma unroll
        for (int k = 0; k < MOST_BLOCKS; ++k) c += cc[k], m += mm[k];
    }
    if (threadIdx.x < OWN_BINS) s.own_count[threadIdx.x] = (u32)c, s.own_mass[threadIdx.x] = m;  // (nought behind its bins)
    block_sum_u64(s, c, m);
    if (threadIdx.x < 32) tell(s.total_count, c), tell(s.total_mass, m);
    cluster_sync();  // the sums are there; nobody reads the blocks' histograms any more
}

__device__ __forceinline__ void clear(Shared& s) {
    for (int b = threadIdx.x; b < BINS; b += THREADS) s.count[b] = 0, s.mass[0][b] = 0, s.mass[1][b] = 0, s.mass[2][b] = 0;
    __syncthreads();
}

// An element into its bin: sums of sixteen bits of no more than MOST_ELEMENTS of them fit 32.
__device__ __forceinline__ void put(Shared& s, int b, u64 mass) {
    atomicAdd(&s.count[b], 1u);
    atomicAdd(&s.mass[0][b], (u32)mass & 0xffffu);
    atomicAdd(&s.mass[1][b], (u32)(mass >> 16) & 0xffffu);
    atomicAdd(&s.mass[2][b], (u32)(mass >> 32));
}

// A thread's elements of bin 0, which nobody else puts there.
__device__ __forceinline__ void put_low(Shared& s, u32 count, u64 mass) {
    count = __reduce_add_sync(0xffffffffu, count), mass = warp_sum_u64(mass);
    if ((threadIdx.x & 31) == 0 && count) {
        atomicAdd(&s.count[0], count);
        // (what lies above 2^48 stays in the upper part: a block's masses together are at most 2^61)
        atomicAdd(&s.mass[0][0], (u32)mass & 0xffffu);
        atomicAdd(&s.mass[1][0], (u32)(mass >> 16) & 0xffffu);
        atomicAdd(&s.mass[2][0], (u32)(mass >> 32));
    }
}

// The histogram of a subset over the whole row: linear, or of elements of one bin by the next digit of their keys.
__device__ void histogram(Shared& s, const Row& r, const Subset& in) {
    clear(s);
    u32 low = 0;  // what falls into bin 0 of the linear histogram, mostly far below all others, is counted first
    u64 low_mass = 0;
    each(r, [&](float l, int i) {
        if (!in.holds(r, l, i)) return;
        const int b = in.bin < 0 ? r.bin(l) : Subset::value(key_of(l, i), in.digits);
        const u64 m = r.mass(l);
        if (in.bin < 0 && b == 0)
            ++low, low_mass += m;
        else
            put(s, b, m);
    });
    put_low(s, low, low_mass);
    add_up<true>(s);
}

// The bin in which the running total of a histogram, from the highest bin down, first reaches `aim` (of counts, or of
// masses); the lowest that holds anything where it does not.  All blocks get the same.  Ends behind a barrier of the cluster.
__device__ Found find_bin(Shared& s, bool by_count, u64 aim) {
    const int lane = threadIdx.x & 31, blocks = cluster_blocks();
    // the blocks' sums, the last block (which has the highest bins) first
    const u64 count = lane < blocks ? s.total_count[blocks - 1 - lane] : 0, mass = lane < blocks ? s.total_mass[blocks - 1 - lane] : 0;
    u64 upto_c = count, upto_m = mass;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 tc = __shfl_up_sync(0xffffffffu, upto_c, o), tm = __shfl_up_sync(0xffffffffu, upto_m, o);
        if (lane >= o) upto_c += tc, upto_m += tm;
    }
    // the last block with anything in it that begins below the aim
    const unsigned some = __ballot_sync(0xffffffffu, count != 0 && (by_count ? upto_c - count : upto_m - mass) < aim);
    const int at = some ? 31 - __clz(some) : 0, owner = blocks - 1 - at;
    const u64 before_c = __shfl_sync(0xffffffffu, upto_c - count, at), before_m = __shfl_sync(0xffffffffu, upto_m - mass, at);
    if (owner == (int)cluster_ctarank() && threadIdx.x < 32) {
        // eight bins a lane, the highest first
        constexpr int EACH = OWN_BINS / 32;
        const int top = OWN_BINS - 1 - EACH * lane;
        u64 pc = 0, pm = 0;
#pragma unroll
        for (int k = 0; k < EACH; ++k) pc += s.own_count[top - k], pm += s.own_mass[top - k];
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
        for (int k = 0; k < EACH; ++k) {
            const u32 n = s.own_count[top - k];
            if (n && (by_count ? ac : am) < aim) bin = top - k, bc = ac, bm = am;
            ac += n, am += s.own_mass[top - k];
        }
        const unsigned any = __ballot_sync(0xffffffffu, bin >= 0);
        const int from = any ? 31 - __clz(any) : 0;
        bin = max(__shfl_sync(0xffffffffu, bin, from), 0), bc = __shfl_sync(0xffffffffu, bc, from), bm = __shfl_sync(0xffffffffu, bm, from);
        if (lane < blocks) {
            st_peer_shared_u32(&s.found.bin, lane, owner * BINS / blocks + bin);
            st_peer_shared_u32(&s.found.count, lane, s.own_count[bin]);
            st_peer_shared_u64(&s.found.before_count, lane, bc);
            st_peer_shared_u64(&s.found.before_mass, lane, bm);
        }
    }
    cluster_sync();
    return s.found;
}

// The elements for which take(l, i) holds, none of which lies outside low .. high, into s.all of every block: how many of them there are in the row (if more than LIST, some are missing).
template <typename Take>
__device__ u32 gather(Shared& s, const Row& r, float low, float high, Take take) {
    if (threadIdx.x == 0) s.count_listed = 0;
    __syncthreads();
    each(r, [&](float l, int i) {
        if (!(l >= low && l <= high) || !take(l, i)) return;
        const u32 at = atomicAdd(&s.count_listed, 1u);
        if (at < LIST) s.list[at].key = key_of(l, i);
    });
    __syncthreads();
    if (threadIdx.x < s.count_listed && threadIdx.x < LIST) s.list[threadIdx.x].mass = r.mass(logit_of((u32)(s.list[threadIdx.x].key >> 32)));
    __syncthreads();
    if (threadIdx.x < 32) tell(s.listed, s.count_listed);
    cluster_sync();
    // thread t takes the row's element t, wherever it lies
    const u32 lane = threadIdx.x & 31, blocks = cluster_blocks();
    u32 upto = lane < blocks ? s.listed[lane] : 0;
#pragma unroll
    for (int o = 1; o < MOST_BLOCKS; o <<= 1) {
        const u32 x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= (u32)o) upto += x;
    }
    const u32 total = __shfl_sync(0xffffffffu, upto, MOST_BLOCKS - 1);
    u32 from = 0, before = 0;
#pragma unroll
    for (int k = 0; k < MOST_BLOCKS - 1; ++k) {
        const u32 x = __shfl_sync(0xffffffffu, upto, k);
        if (threadIdx.x >= x) from = k + 1, before = x;
    }
    const bool in = threadIdx.x < total && threadIdx.x - before < LIST;
    Entry mine;
    if (in) mine.key = ld_peer_shared_u64(&s.list[threadIdx.x - before].key, from), mine.mass = ld_peer_shared_u64(&s.list[threadIdx.x - before].mass, from);
    cluster_sync();  // (nobody's own is read any more)
    if (in) s.all[threadIdx.x] = mine;
    __syncthreads();
    return total;
}

// Of this thread's element of the n in s.all: how many lie before it, and their mass.
__device__ __forceinline__ void ranks(const Shared& s, int n, const Entry& mine, u64& count, u64& mass) {
    count = 0, mass = 0;
    if ((int)threadIdx.x < n)
        for (int i = 0; i < n; ++i)
            if (s.all[i].key > mine.key) ++count, mass += s.all[i].mass;
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

// From the linear histogram of `in`, which stands in the blocks' shares.
__device__ Quantile quantile(Shared& s, const Row& r, Subset in, bool by_count, u64 aim) {
    Found f = find_bin(s, by_count, aim);
    in.bin = f.bin;
    u64 before_mass = f.before_mass;
    aim -= min(aim, by_count ? f.before_count : f.before_mass);
    while (f.count > LIST) {
        histogram(s, r, in);
        f = find_bin(s, by_count, aim);
        const int shift = Subset::shift(in.digits);
        in.prefix |= shift >= 0 ? (u64)f.bin << shift : (u64)f.bin >> -shift;
        ++in.digits;
        before_mass += f.before_mass;
        aim -= min(aim, by_count ? f.before_count : f.before_mass);
    }
    const int n = (int)gather(s, r, r.below_bin(in.bin), r.above_bin(in.bin), [&](float l, int i) { return in.holds(r, l, i); });
    if (threadIdx.x == 0) s.threshold = 0, s.retained = 0;
    __syncthreads();
    const Entry mine = s.all[threadIdx.x];
    u64 count, mass;
    ranks(s, n, mine, count, mass);
    if ((int)threadIdx.x < n) {
        // the last one that begins below the aim: its own end does not lie below, or nothing follows
        const u64 begins = by_count ? count : mass, ends = by_count ? count + 1 : mass + mine.mass;
        if ((begins < aim && ends >= aim) || (count == (u64)n - 1 && ends < aim)) s.threshold = mine.key, s.retained = mass + mine.mass;
    }
    __syncthreads();
    Quantile q = {s.threshold, before_mass + s.retained};
    __syncthreads();
    return q;
}

// f(i, four neighbours from i on) over this block's elements, and one by one(i) over those at the end; with loads and stores of 16 bytes where `wide`.
template <typename Four, typename One>
__device__ __forceinline__ void for_elements(int n, bool wide, Four four, One one) {
    const int whole = wide ? n & ~3 : 0;
#pragma unroll 2
    for (int i = 4 * threadIdx.x; i < whole; i += 4 * THREADS) four(i);
    for (int i = whole + threadIdx.x; i < n; i += THREADS) one(i);
}

// Whether a row is sampled from as it is, without top-k and top-p.
__device__ __forceinline__ bool plain_row(const SamplingProbs& a, int row) {
    const int k = a.top_k ? a.top_k[row] : 0;  // (all three on their way together)
    const float T = a.temperature ? a.temperature[row] : 0.0f, p = a.top_p ? a.top_p[row] : 1.0f;
    return (T > 0.0f) & (k <= 0 || (k >= a.vocab && k != 1)) & (p >= 1.0f);
}

template <bool KEEP>  // the block's elements fit shared memory: `kept`
__device__ __forceinline__ void probabilities(const SamplingProbs& a, int row, Shared& s, float* kept) {
    const u32 rank = cluster_ctarank();
    const float* logits = a.logits + (long long)row * a.ldl;
    float* out = a.out + (long long)row * a.ldo;
    const float given = a.temperature ? a.temperature[row] : 0.0f, p = a.top_p ? a.top_p[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const bool greedy = !(given > 0.0f) || k == 1 || !(p > 0.0f);
    const float T = fminf(fmaxf(given, FLT_EPSILON), 1e30f);
    Row r;
    r.lo = min(a.vocab, (int)rank * a.per), r.n = min(a.vocab, r.lo + a.per) - r.lo;
    r.at = KEEP ? kept : logits + r.lo;
    r.powers = s.powers;
    const float rate = (float)(LOG2E / (double)T);
    const bool wide_in = (((uintptr_t)(logits + r.lo)) & 15) == 0, wide_out = (((uintptr_t)(out + r.lo)) & 15) == 0;
    const bool by_k = !greedy && k > 0 && k < a.vocab, by_p = !greedy && p < 1.0f;
    // the row's share on its way, all of it at once
    if (KEEP) {
        const uint32_t to = smem_u32(kept);
        const int whole = wide_in ? r.n & ~3 : 0;
        for (int i = 4 * threadIdx.x; i < whole; i += 4 * THREADS)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 4 * i), "l"(logits + r.lo + i) : "memory");
        for (int i = whole + threadIdx.x; i < r.n; i += THREADS)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4 * i), "l"(logits + r.lo + i) : "memory");
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    // the greatest logit: the thread's (of those that it has fetched itself), the block's, the row's
    float mine = -INFINITY;
    bool nan = false;
    for_elements(
        r.n, wide_in,
        [&](int i) {
            const float4 v = *reinterpret_cast<const float4*>(r.at + i);
            mine = fmaxf(fmaxf(mine, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
            nan |= isnan(v.x) | isnan(v.y) | isnan(v.z) | isnan(v.w);
        },
        [&](int i) {
            mine = fmaxf(mine, r.at[i]);
            nan |= isnan(r.at[i]);
        });
    nan = __any_sync(0xffffffffu, nan);
    if ((threadIdx.x & 31) == 0) s.fred[3][threadIdx.x >> 5] = nan ? 1.0f : 0.0f;
    const float block_top = block_max(s, 0, mine);
    nan = __any_sync(0xffffffffu, s.fred[3][threadIdx.x & (WARPS - 1)] != 0.0f);
    // (for top-k) the least finite maximum of a thread
    const int quads = wide_in ? r.n & ~3 : 0;
    const bool has = 4 * (int)threadIdx.x < quads || quads + (int)threadIdx.x < r.n;
    const float block_least = by_k ? -block_max(s, 1, mine > -INFINITY ? -mine : -INFINITY) : 0.0f;
    if (threadIdx.x < 32) tell(s.value[0], block_top), tell(s.value[1], block_least);
    cluster_sync();
    r.given_top = warp_max(row_value(s.value[0], -INFINITY));
    r.odd = nan || !(fabsf(r.given_top) < 1e37f);
    r.top = r.high = fabsf(r.given_top) < 1e37f ? r.given_top : 0.0f;
    r.least = r.top - 60.0f * T, r.rate = 32.0 * LOG2E / (double)T;
    if (!(r.least < r.top)) {  // a temperature that is nothing beside the logits: the next logit below has none of the mass, as it would have by far
        r.least = nextafterf(r.top, -INFINITY);
        r.rate = 32.0 * LOG2E * 60.0 / ((double)r.top - (double)r.least);
    }
    out += r.lo;
    if (greedy) {
        // the first index among those of the greatest logit
        u32 first = 0xffffffffu;
        for (int i = threadIdx.x; i < r.n; i += THREADS)
            if (r.logit(i) == r.top) first = min(first, (u32)(r.lo + i));
        first = __reduce_min_sync(0xffffffffu, first);
        if (threadIdx.x == 0) s.count_listed = 0xffffffffu;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) atomicMin(&s.count_listed, first);
        __syncthreads();
        if (threadIdx.x < 32) tell(s.index, s.count_listed);
        cluster_sync();
        const u32 lane = threadIdx.x & 31;
        first = __reduce_min_sync(0xffffffffu, lane < cluster_blocks() ? s.index[lane] : 0xffffffffu) - (u32)r.lo;
        auto of = [&](int i) { return (u32)i == first ? 1.0f : 0.0f; };
        for_elements(
            r.n, wide_out, [&](int i) { *reinterpret_cast<float4*>(out + i) = make_float4(of(i), of(i + 1), of(i + 2), of(i + 3)); },
            [&](int i) { out[i] = of(i); });
    } else if (!by_k && !by_p) {
        // (the difference is rounded once, its product with log2(e) / T twice: an exponent is off by 2^-23 of itself, as if it were divided by T)
        auto weight = [&](float l) { return exp2_unit((r.number(l) - r.top) * rate); };
        float sum = 0.0f;
        for_elements(
            r.n, KEEP,
            [&](int i) {
                float4 v = *reinterpret_cast<const float4*>(r.at + i);
                v = make_float4(weight(v.x), weight(v.y), weight(v.z), weight(v.w));
                if (KEEP) *reinterpret_cast<float4*>(kept + i) = v;
                sum += (v.x + v.y) + (v.z + v.w);
            },
            [&](int i) {
                const float w = weight(r.at[i]);
                if (KEEP) kept[i] = w;
                sum += w;
            });
        sum = block_sum(sum, s.scratch);  // (ends with a barrier: the weights are there for all)
        if (threadIdx.x < 32) tell(s.value[2], sum);
        cluster_sync();
        const float inv = 1.0f / warp_sum(row_value(s.value[2], 0.0f));
        auto of = [&](int i) { return (KEEP ? kept[i] : weight(r.at[i])) * inv; };
        for_elements(
            r.n, wide_out,
            [&](int i) {
                if (KEEP) {
                    const float4 v = *reinterpret_cast<const float4*>(kept + i);
                    *reinterpret_cast<float4*>(out + i) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                } else
                    *reinterpret_cast<float4*>(out + i) = make_float4(of(i), of(i + 1), of(i + 2), of(i + 3));
            },
            [&](int i) { out[i] = of(i); });
    } else {
        u64 threshold = 0, mass = 0;  // the least key that stays; the mass of those that do
        bool done = false;
        auto set_range = [&](float range) {
            if (!(range > 0.0f)) range = 1.0f;
            r.bins_per = (float)(BINS - 1) / fminf(range, FLT_MAX);
        };
        Subset all;
        if (by_k && k <= LIST) {
            // the k-th of the threads' maxima: no fewer than k logits lie in its bin and above
            set_range(r.top - -warp_max(-row_value(s.value[1], INFINITY)));
            clear(s);
            if (has) atomicAdd(&s.count[r.bin(r.number(mine))], 1u);
            add_up<false>(s);
            const u64 threads = row_sum_u64(s.total_count);
            if (threads >= (u64)k) {
                const Found f = find_bin(s, true, (u64)k);
                const int n = (int)gather(s, r, r.below_bin(f.bin), INFINITY, [&](float l, int) { return r.from_bin_on(l, f.bin); });
                if (n <= LIST) {
                    if (threadIdx.x == 0) s.threshold = ~0ull, s.retained = 0, s.kept_mass = 0;
                    __syncthreads();
                    const Entry here = s.all[threadIdx.x];
                    u64 count, before;
                    ranks(s, n, here, count, before);
                    const bool in = (int)threadIdx.x < n;
                    if (in && count == (u64)k - 1) s.kept_mass = before + here.mass;
                    __syncthreads();
                    const u64 aim = by_p ? share_of(s.kept_mass, p) : ~0ull;
                    if (in && count < (u64)k && (count == 0 || before < aim)) {
                        atomicMin(&s.threshold, here.key);
                        atomicMax(&s.retained, before + here.mass);
                    }
                    __syncthreads();
                    threshold = s.threshold, mass = s.retained;
                    done = true;
                }
            }
        }
        if (!done && by_k) {
            // the whole row's histogram, from the greatest logit to the least finite one
            float low = INFINITY;
            each(r, [&](float l, int) {
                if (l > -INFINITY) low = fminf(low, l);
            });
            low = -block_max(s, 2, -low);
            if (threadIdx.x < 32) tell(s.value[3], low);
            cluster_sync();
            set_range(r.top - -warp_max(-row_value(s.value[3], INFINITY)));
            histogram(s, r, all);
            const Quantile q = quantile(s, r, all, true, (u64)k);
            threshold = q.key, mass = q.mass;
            if (by_p) {
                histogram(s, r, all);  // (the search may have cut a bin up in its place)
                const u64 aim = share_of(mass, p);
                const Quantile qp = quantile(s, r, all, false, aim ? aim : 1);
                threshold = qp.key, mass = qp.mass;
            }
        } else if (!done) {
            // Masses above bounds that lie so many units of temperature below the greatest logit, in 32 bits: between which two the border lies, with 2^-10
            // for what they are off by.
            const float depth[BOUNDS] = {1.0f, 2.0f, 4.0f, 6.0f, 8.0f, 11.0f, 16.0f};
            float bound[BOUNDS], above[BOUNDS] = {}, all_mass = 0.0f;
#pragma unroll
            for (int b = 0; b < BOUNDS; ++b) bound[b] = r.top - depth[b] * T;
            each(r, [&](float l, int) {
                const float w = exp2_unit((l - r.top) * rate);
                all_mass += w;
#pragma unroll
                for (int b = 0; b < BOUNDS; ++b)
                    if (l > bound[b]) above[b] += w;
            });
#pragma unroll
            for (int b = 0; b <= BOUNDS; ++b) {
                const float t = warp_sum(b < BOUNDS ? above[b] : all_mass);
                if ((threadIdx.x & 31) == 0) s.parts[threadIdx.x >> 5][b] = t;
            }
            __syncthreads();
            if (threadIdx.x < MOST_BLOCKS * (BOUNDS + 1)) {
                const u32 b = threadIdx.x % (BOUNDS + 1), to = threadIdx.x / (BOUNDS + 1);
                float t = 0.0f;
                for (int w = 0; w < WARPS; ++w) t += s.parts[w][b];
                if (to < cluster_blocks()) st_peer_shared_u32(&s.above[cluster_ctarank()][b], to, __float_as_uint(t));
            }
            cluster_sync();
            {
                const int b = threadIdx.x % (BOUNDS + 1);
                float t = 0.0f;
                for (u32 k = 0; k < cluster_blocks(); ++k) t += s.above[k][b];
#pragma unroll
                for (int c = 0; c < BOUNDS; ++c) above[c] = __shfl_sync(0xffffffffu, t, c);
                all_mass = __shfl_sync(0xffffffffu, t, BOUNDS);
            }
            Subset in;
            in.high = r.top;
#pragma unroll
            for (int b = BOUNDS - 1; b >= 0; --b)
                if (above[b] > p * all_mass * (1.0f + 1.0f / 1024)) in.low = bound[b];
#pragma unroll
            for (int b = 0; b < BOUNDS; ++b)
                if (above[b] < p * all_mass * (1.0f - 1.0f / 1024)) in.high = bound[b];
            // the histogram of what lies between them, and the masses of what lies above and of all
            r.high = in.high;
            set_range(in.low > -INFINITY ? in.high - in.low : 32.0f * T);  // (what weighs less than 2^-46 of the greatest has no mass)
            clear(s);
            u64 over = 0, sum = 0, low_mass = 0;
            u32 low = 0;
            u32 overs = 0;
            auto take = [&](float l, u64 m) {  // (sums with what the masses are offset by, which is taken away behind the loop)
                sum += m;
                if (l > in.high) over += m, ++overs;
                if (!in.between(l)) return;
                const int b = r.bin(l);
                if (b == 0)
                    ++low, low_mass += m;
                else
                    put(s, b, m - MASS_OFFSET);
            };
            // (two masses at once; 40 rows 59 us for 60)
            int i = threadIdx.x;
#pragma unroll 1
            for (; i + THREADS < r.n; i += 2 * THREADS) {
                const float l = r.logit(i), next = r.logit(i + THREADS);
                const u64 m = r.mass_and_offset(l), next_m = r.mass_and_offset(next);
                take(l, m), take(next, next_m);
            }
            if (i < r.n) take(r.logit(i), r.mass_and_offset(r.logit(i)));
            sum -= MASS_OFFSET * (u64)((r.n - (int)threadIdx.x + THREADS - 1) / THREADS), over -= MASS_OFFSET * overs, low_mass -= MASS_OFFSET * low;
            put_low(s, low, low_mass);
            block_sum_u64(s, over, sum);
            if (threadIdx.x < 32) tell(s.over, over), tell(s.sum, sum);
            add_up<true>(s);
            over = row_sum_u64(s.over), sum = row_sum_u64(s.sum);
            const u64 aim = share_of(sum, p);
            const Quantile q = quantile(s, r, in, false, (aim ? aim : 1) - over);
            threshold = q.key, mass = over + q.mass;
        }
        // (which tokens stay is decided; their probabilities in 32 bits, as without top-k and top-p)
        const float inv = (float)(s.powers[0] / (double)mass), border = logit_of((u32)(threshold >> 32));
        auto of = [&](float l, int i) -> float {
            l = r.number(l);
            if (!(l >= border) || (l == border && key_of(l, r.lo + i) < threshold)) return 0.0f;
            return exp2_unit((l - r.top) * rate) * inv;
        };
        for_elements(
            r.n, wide_out && KEEP,
            [&](int i) {
                const float4 v = *reinterpret_cast<const float4*>(r.at + i);
                *reinterpret_cast<float4*>(out + i) = make_float4(of(v.x, i), of(v.y, i + 1), of(v.z, i + 2), of(v.w, i + 3));
            },
            [&](int i) { out[i] = of(r.at[i], i); });
    }
    cluster_sync();  // nobody goes on, or leaves, while others may read its shared memory
}

// A cluster a row, or (`skip`) clusters that go over the rows which are left.
template <bool KEEP>
__global__ void __launch_bounds__(THREADS, 2) sampling_probs_kernel(const SamplingProbs a) {
    __shared__ Shared s;
    extern __shared__ __align__(16) float kept[];
    if (threadIdx.x < 32) s.powers[threadIdx.x] = powers_of_two[threadIdx.x] * (double)(1ull << (a.vocab < 1 << 19 ? MASS_BITS : MASS_BITS - 1));
    cluster_sync();  // (all blocks have begun: their memory may be written)
    pdl_wait();
    pdl_launch_dependents();
    for (int first = blockIdx.x; first < a.rows; first += 32 * gridDim.x) {
        const int mine = first + (threadIdx.x & 31) * gridDim.x;
        unsigned here = __ballot_sync(0xffffffffu, mine < a.rows && !(a.skip && plain_row(a, mine)));
        for (; here; here &= here - 1) probabilities<KEEP>(a, first + (__ffs(here) - 1) * gridDim.x, s, kept);
    }
}

// ---------------------------------------------------------------------------------------------
// Many rows without top-k and top-p: a cluster of up to sixteen blocks a row, of which four share an SM, so that some wait for their shares while others
// exponentiate and write.  A thread holds its forty elements in registers and exponentiates against the greatest of them; warps, blocks and the cluster bring their
// sums to a common maximum, once each.  Blocks hand each other maximum and sum by stores (reading them from the others took 5,000 cycles of 26,000).
// Sixteen blocks hold 163,840 elements (512 rows of them 120 us); longer rows are the other kernel's (163,844 elements 197 us, 200,000 204).
// ---------------------------------------------------------------------------------------------
constexpr int PLAIN_THREADS = 256, PLAIN_WARPS = PLAIN_THREADS / 32, PLAIN_QUADS = 10, PLAIN_SHARE = 4 * PLAIN_QUADS * PLAIN_THREADS, PLAIN_BLOCKS = 16;

__global__ void __launch_bounds__(PLAIN_THREADS, 4) sampling_softmax_kernel(const SamplingProbs a) {
    __shared__ float part[2][PLAIN_WARPS], row_part[2][PLAIN_BLOCKS];
    cluster_arrive_relaxed();
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = cluster_blocks();
    const int lo = min(a.vocab, (int)cluster_ctarank() * a.per), n = min(a.vocab, lo + a.per) - lo;
    const float* logits = a.logits + row * a.ldl + lo;
    if (!plain_row(a, row)) {
        cluster_wait();
        return;
    }
    const bool wide = ((uintptr_t)logits & 15) == 0;
    float4 v[PLAIN_QUADS];
#pragma unroll
    for (int q = 0; q < PLAIN_QUADS; ++q) {
        const int i = 4 * (threadIdx.x + q * PLAIN_THREADS);
        if (wide && i + 4 <= n)
            v[q] = *reinterpret_cast<const float4*>(logits + i);
        else
            v[q] = make_float4(i < n ? logits[i] : -INFINITY, i + 1 < n ? logits[i + 1] : -INFINITY, i + 2 < n ? logits[i + 2] : -INFINITY, i + 3 < n ? logits[i + 3] : -INFINITY);
    }
    const float rate = (float)LOG2E / fminf(fmaxf(a.temperature[row], FLT_EPSILON), 1e30f);
    float top = -INFINITY;
#pragma unroll
    for (int q = 0; q < PLAIN_QUADS; ++q) top = fmaxf(fmaxf(top, fmaxf(v[q].x, v[q].y)), fmaxf(v[q].z, v[q].w));
    // (of an infinite maximum: those that equal it, all alike; a NaN counts as minus infinity)
    const bool infinite = isinf(top);
    auto weight = [&](float l, int i) { return infinite ? (fmaxf(l, -INFINITY) == top && i < n ? 1.0f : 0.0f) : exp2_unit((fmaxf(l, -INFINITY) - top) * rate); };
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < PLAIN_QUADS; ++q) {
        const int i = 4 * (threadIdx.x + q * PLAIN_THREADS);
        v[q] = make_float4(weight(v[q].x, i), weight(v[q].y, i + 1), weight(v[q].z, i + 2), weight(v[q].w, i + 3));
        sum += (v[q].x + v[q].y) + (v[q].z + v[q].w);
    }
    // what a sum against `t` is against `most`
    auto factor = [&](float t, float most) { return t == most ? 1.0f : exp2_unit((t - most) * rate); };
    float most = warp_max(top), total = warp_sum(sum * factor(top, most));
    if (lane == 0) part[0][warp] = most, part[1][warp] = total;
    __syncthreads();
    cluster_wait();  // (all blocks have begun)
    if (warp == 0) {
        const float t = lane < PLAIN_WARPS ? part[0][lane] : -INFINITY, x = lane < PLAIN_WARPS ? part[1][lane] : 0.0f;
        most = warp_max(t), total = warp_sum(x * factor(t, most));
        if (lane < blocks) {
            st_peer_shared_f32(smem_u32(&row_part[0][cluster_ctarank()]), lane, most);
            st_peer_shared_f32(smem_u32(&row_part[1][cluster_ctarank()]), lane, total);
        }
    }
    cluster_sync();
    {
        const float t = lane < blocks ? row_part[0][lane] : -INFINITY, x = lane < blocks ? row_part[1][lane] : 0.0f;
        most = warp_max(t), total = warp_sum(x * factor(t, most));
    }
    const float scale = factor(top, most) / total;
    float* out = a.out + row * a.ldo + lo;
    const bool wide_out = ((uintptr_t)out & 15) == 0;
#pragma unroll
    for (int q = 0; q < PLAIN_QUADS; ++q) {
        const int i = 4 * (threadIdx.x + q * PLAIN_THREADS);
        const float4 w = make_float4(v[q].x * scale, v[q].y * scale, v[q].z * scale, v[q].w * scale);
        if (wide_out && i + 4 <= n)
            *reinterpret_cast<float4*>(out + i) = w;
        else {
            if (i < n) out[i] = w.x;
            if (i + 1 < n) out[i + 1] = w.y;
            if (i + 2 < n) out[i + 2] = w.z;
            if (i + 3 < n) out[i + 3] = w.w;
        }
    }
}

}  // namespace

// logits, out fp32 [rows, vocab] with row strides ldl, ldo: the same memory, or apart.  temperature, top_k, top_p: per row, or null for greedy rows.
// How many clusters of `blocks` run at once: clusters lie in parts of the GPU that have different numbers of SMs, so that these are fewer than the SMs have room
// for (of seven blocks, two on an SM, 37 for 42).
static int clusters_at_once(int blocks, bool keep, size_t bytes) {
    static thread_local struct { size_t bytes; int clusters; } asked[MOST_BLOCKS + 1] = {};
    auto& known = asked[blocks];
    if (known.clusters && known.bytes == bytes) return known.clusters;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, 1, blocks), cfg.blockDim = dim3(THREADS), cfg.dynamicSmemBytes = bytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = blocks;
    cfg.attrs = attr, cfg.numAttrs = 1;
    int n = 0;
    if (keep && ferris_allow_dynamic_smem((const void*)sampling_probs_kernel<true>, (int)bytes) != FERRIS_OK) return 1;
    const cudaError_t e = keep ? cudaOccupancyMaxActiveClusters(&n, sampling_probs_kernel<true>, &cfg) : cudaOccupancyMaxActiveClusters(&n, sampling_probs_kernel<false>, &cfg);
    if (e != cudaSuccess || n <= 0) {
        cudaGetLastError();
        return 1;
    }
    known.bytes = bytes, known.clusters = n;
    return n;
}

FERRIS_API int ferris_sampling_probs(const float* logits, long long ldl, float* out, long long ldo, int rows, int vocab, const float* temperature,
                                     const int* top_k, const float* top_p, void* stream) {
    if (rows <= 0) return FERRIS_OK;
    if (vocab <= 0 || ldl < vocab || ldo < vocab) FERRIS_REFUSE("vocabulary %d, row strides %lld and %lld", vocab, ldl, ldo);
    if (vocab > MOST_BLOCKS * MOST_ELEMENTS) FERRIS_REFUSE("a vocabulary of %d, at most %d", vocab, MOST_BLOCKS * MOST_ELEMENTS);
    // Blocks of a row: of as many as give the least time if clusters run in waves, each as long as a block's share of the row (40 rows of 151,936: six, all at once,
    // 60 us; seven, of which 37 run at once, 84).
    const int sms = ferris_sm_count();
    int blocks = MOST_BLOCKS, at_once = 1;
    double least = 0.0;
    auto per_block = [&](int b) { return (int)(((long long)vocab + 4 * b - 1) / (4 * b)) * 4; };
    const size_t fixed = sizeof(Shared) + 1024, most = 227 * 1024;  // (an SM keeps a KB of every block's for itself)
    for (int b = MOST_BLOCKS; b >= LEAST_BLOCKS; --b) {
        const size_t bytes = (size_t)per_block(b) * 4;
        const bool keep = bytes + fixed <= most;
        const int clusters = clusters_at_once(b, keep, keep ? bytes : 0);
        const double time = (double)((rows + clusters - 1) / clusters) / b;
        if (b == MOST_BLOCKS || (time < least && per_block(b) <= MOST_ELEMENTS)) least = time, blocks = b, at_once = clusters;
    }
    SamplingProbs a = {logits, out, ldl, ldo, temperature, top_k, top_p, vocab, per_block(blocks), rows, 0};
    cudaError_t e;
    // More rows than run at once: those without top-k and top-p by the kernel of smaller blocks (37 rows without it 14.7 us, 38 with it 13.0, 512 rows 190 without and
    // 120 with; of fewer rows the launch would cost more than it saves: 16 rows 10.8).
    int parts = (vocab + PLAIN_SHARE - 1) / PLAIN_SHARE;
    if ((long long)rows * MOST_BLOCKS > 2ll * sms && per_block(PLAIN_BLOCKS) <= PLAIN_SHARE && temperature) {
        while (per_block(parts) > PLAIN_SHARE) ++parts;
        if (parts > 8) {
            e = cudaFuncSetAttribute(sampling_softmax_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) {
                ferris_set_error("%s", cudaGetErrorString(e));
                return (int)e;
            }
        }
        SamplingProbs b = a;
        b.per = per_block(parts);
        e = ferris_launch_cluster(sampling_softmax_kernel, dim3(rows, 1, parts), dim3(PLAIN_THREADS), 0, (cudaStream_t)stream, parts, b);
        if (e != cudaSuccess) {
            ferris_set_error("%s", cudaGetErrorString(e));
            return (int)e;
        }
        a.skip = 1;
    }
    const size_t bytes = (size_t)a.per * 4;
    const int clusters = a.skip && at_once < rows ? at_once : rows;
    if (bytes + fixed <= most) {
        const int rc = ferris_allow_dynamic_smem((const void*)sampling_probs_kernel<true>, bytes);
        if (rc != FERRIS_OK) return rc;
        e = ferris_launch_cluster(sampling_probs_kernel<true>, dim3(clusters, 1, blocks), dim3(THREADS), bytes, (cudaStream_t)stream, blocks, a);
    } else
        e = ferris_launch_cluster(sampling_probs_kernel<false>, dim3(clusters, 1, blocks), dim3(THREADS), 0, (cudaStream_t)stream, blocks, a);
    if (e != cudaSuccess) {
        ferris_set_error("%s", cudaGetErrorString(e));
        return (int)e;
    }
    FERRIS_LAUNCH_CHECK();
}
