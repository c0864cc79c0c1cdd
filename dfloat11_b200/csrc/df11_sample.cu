// One token per row of logits, drawn with temperature, top-k, top-p and min-p from given random
// numbers.
//
// With z the logits, c the largest and T the temperature, a token's weight is exp((z - c) / T), in
// (0, 1].  A sum over 10^5 tokens decides at which token a border (u * mass, top_p * mass) is
// crossed; summed in fp32 it is off by some 1e-7 of the mass, and with 10^5 borders about one row in
// a hundred would be decided wrongly, and differently in another order.  So weights are computed in fp64
// and held as 64-bit integers, weight * 2^S with S such that V of them fit: sums of integers are
// exact, the same in every order, and S >= 45 for V < 2^18 leaves each weight off by 2^-46 at most.
//
// A filter keeps all tokens above some logit and, of those equal to it, the ones up to some index.
// That border is found without sorting the row:
//   * top-k of a few: the k-th largest of the threads' own largest logits is a lower bound of the k-th
//     largest of all.  The tokens above it are few; they are listed, and all filters and the draw are
//     done on the list.
//   * otherwise the tokens are counted in 4096 intervals of equal width between the largest logit
//     and the one whose weight no longer matters (or the smallest).  Counts give the interval of the top-k border
//     exactly, and, times the weight in the interval's middle, that of the top-p border almost.
//     One pass over the row then adds up the exact mass above those intervals and lists what lies in them;
//     the list gives the border, and exact sums prove that it lies there.
//   * where a list would overflow (thousands of equal logits at the border) or the guess was
//     wrong, one CTA finds the border digit by digit of the logits' bits.
// The draw needs masses in index order: sums of blocks of 256 or more tokens are kept by the same
// pass, and only the block that holds the border is looked at again.
//
// A row is divided among a cluster of 1 to 8 CTAs, as many as leave every SM with work.  The row is
// read two or three times, the first time from memory, then from the L2 cache.  Bound: for few rows the chain of
// barriers, for many the instructions (27 per token where weights are added up, 11 where tokens are counted).
// Measured in a graph of such calls, rows of 151936 (one) and 128256 (256) BF16 logits: arg-max 6.3 and 30.5 us,
// top-k of 20 with top-p 14.9 and 38.5, no filter 13.8 and 73, top-p 0.9 alone 38 and 157.
#include <math.h>

#include <type_traits>

#include "df11_launch.h"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 4096;
constexpr int kList = 2048;
constexpr int kFew = 128;                     // numbers that are compared with one another
constexpr int kBlocks = kThreads;             // block sums per CTA, at most
// Top-k up to here goes by the threads' largest (one row of 151936, k = 20: 14.5 us); beyond, the bound lets through
// more and more, and with k above the number of threads there is none: by counts (k = 500: 20.5 us).
constexpr int kFewTokens = 256;
constexpr uint32_t kLowestKey = 0x00800000u;  // key of the lowest finite float
constexpr uint32_t kAny = 0xFFFFFFFFu;

using u64 = unsigned long long;

// A number that orders like the logit (-0 like 0).
__device__ __forceinline__ uint32_t key_of(float z)
{
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// Weights exp((z - c) / T) 2^S, in fp64 to 2^-44 of themselves and rounded to integers.
// With t = 64 (z - c) / (T ln 2), n an integer next to it and f = t - n:  2^(t/64) = 2^(n/64) 2^(f/64);
// the first factor is one of 64 numbers times a power of two, the second the Taylor sum of exp(f ln2 / 64)
// up to the fourth power (|f ln2 / 64| < 0.0055, remainder below 5e-14).  n is found in fp32, which leaves nine
// fp64 operations.
constexpr int kRoots = 64;
constexpr double kOne52 = 4503599627370496.0;  // 2^52: added to a number below it, the sum's low bits are the nearest integer
struct Weigher {
    float cap, cut;                           // the largest logit that counts, and one below which a weight is less than 2^-60
    float half, slope32;                      // -cap / 2; twice the slope
    bool plain;                               // fast() may be asked for any logit, -inf included
    double peak, slope, unit;
    int shift;                                // S
    const double *roots;                      // 2^(j/64), in shared memory

    __device__ __forceinline__ Weigher(float best, double t, int s, const double *r) : shift(s), roots(r)
    {
        constexpr float kMost = 3.402823466e38f;
        cap = fminf(best, kMost);
        const float low = (float)fmax(cap - 60.0 * 0.69314718055994530942 * t, -(double)kMost);
        cut = low > -kMost ? logit_of(key_of(low) - 1) : low;     // rounded down
        peak = (double)cap;
        slope = fmin(kRoots * 1.4426950408889634074 / t, 1e300);
        slope32 = (float)fmin(2.0 * slope, 1e38);
        half = -0.5f * cap;
        plain = best <= kMost && low > -kMost && (peak - (double)cut) * slope < 70.0 * kRoots;
        unit = ldexp(1.0, s);
    }
    // For logits from `cut` to `cap`; exactly 2^S for the largest.
    __device__ __forceinline__ double inner(float z) const
    {
        constexpr double a = 0.69314718055994530942 / kRoots;
        // halves: the whole difference may not fit a float.  The sum with 1.5 * 2^23 has the integer in its low bits
        const int n = __float_as_int(fmaf(fmaf(z, 0.5f, half), slope32, 12582912.0f)) - 0x4B400000;
        const double k = __hiloint2double(0x43300000, n ^ 0x80000000) - (kOne52 + 2147483648.0);
        const double f = fma((double)z - peak, slope, -k);
        double p = fma(a * a * a * a / 24, f, a * a * a / 6);
        p = fma(p, f, a * a / 2);
        p = fma(p, f, a);
        const double root = roots[n & (kRoots - 1)];
        const double scaled = __hiloint2double(__double2hiint(root) + (n & -kRoots) * ((1 << 20) / kRoots) + (shift << 20),
                                               __double2loint(root));
        return fma(scaled, p * f, scaled);
    }
    // Where `plain`: less than 1/2 for what is below `cut`, -inf included.
    __device__ __forceinline__ double fast(float z) const { return inner(fmaxf(z, cut)); }
    // 0 below `cut`; whatever lies above `cap` counts as it.
    __device__ __forceinline__ double real(float z) const
    {
        const double w = inner(z >= cut ? fminf(z, cap) : cap);
        return z >= cut && (z == cap || (peak - (double)fminf(z, cap)) * slope < 70.0 * kRoots) ? w : 0.0;
    }
    // The nearest integer to w < 2^51, plus kBias; sums of such numbers are put right by as many kBias.
    static constexpr u64 kBias = 0x4330000000000000ull;
    __device__ __forceinline__ static u64 biased(double w) { return (u64)__double_as_longlong(w + kOne52); }
    __device__ __forceinline__ u64 operator()(float z) const { return biased(real(z)) - kBias; }
};

struct Yes {
    static constexpr bool value = true;
};
struct No {
    static constexpr bool value = false;
};

struct Row {             // settings of a row
    double t, p, low, u;
    long long k;
};

struct Exchange {        // what the CTAs of a cluster tell one another
    float best, least, bound;
    u64 mass, above, blocks;
};

struct Verdict {         // what the first CTA finds on its list
    float logit;                              // kept: logits above, or equal with an index up to this one
    uint32_t index;
    int fallback;
};

struct Shared {
    alignas(16) uint32_t count[kBins];        // this CTA's counts
    uint32_t merged[kBins];                   // the row's
    u64 list[kList], weight[kList];
    u64 blocks[kBlocks];
    u64 partial[kWarps];
    double roots[kRoots];
    float partial_real[kWarps];
    uint32_t partial_count[kWarps];
    float partial_top[kWarps], partial_bottom[kWarps];
    Exchange mine;
    Verdict verdict;
    u64 few[kFew], few_measure[kFew], partial_most[kWarps], border;         // find_border's
    uint32_t parts_low[kThreads], parts_high[kThreads];
    uint32_t few_n, part;
    uint32_t list_n, found;
    int bin_k, bin_p, bin_low, bin_high;      // interval of the top-k border; of the top-p border, and those around it
    uint32_t above_k, above_low, upto_high;   // tokens above bin_k; above bin_low; and down to bin_high
    u64 base;
};

// The block's shared memory.  Functions that are not inlined name it themselves: through a reference handed to
// them every access would have to find out first which memory it goes to.
extern __shared__ __align__(16) unsigned char raw_shared[];
#define DF11_SHARED Shared &s = *reinterpret_cast<Shared *>(raw_shared)

__device__ __forceinline__ void cluster_sync(uint32_t size)
{
    if (size > 1) asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
    else __syncthreads();
}

template <typename T> __device__ __forceinline__ T *remote(T *local, uint32_t rank)
{
    T *there;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(there) : "l"(local), "r"(rank));
    return there;
}

template <typename V> __device__ V block_sum(V x, V *partial)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) partial[threadIdx.x >> 5] = x;
    __syncthreads();
    V all = 0;
    for (int w = 0; w < kWarps; ++w) all += partial[w];
    return all;
}

// Sum of the x of all threads before this one, and of all.
template <typename V> __device__ V block_scan(V x, V *partial, V *total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V sum = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += y;
    }
    __syncthreads();
    if (lane == 31) partial[warp] = sum;
    __syncthreads();
    V before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += partial[w];
        all += partial[w];
    }
    *total = all;
    return before + sum - x;
}

__device__ __forceinline__ u64 listed(float z, uint32_t index) { return (u64)key_of(z) << 32 | (0xFFFFFFFFu - index); }
__device__ __forceinline__ float listed_logit(u64 x) { return logit_of((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint32_t listed_index(u64 x) { return 0xFFFFFFFFu - (uint32_t)x; }

// The least of the different numbers key(0) .. key(n - 1) up to which the measures sum to `want` or more
// (1 <= want <= the sum of all).  The numbers' range is divided among the threads, the measures are added up there,
// and the part in which the border lies is divided again, until so few are left that every number can be
// compared with every other.
template <typename K, typename M> __device__ __noinline__ u64 find_border(int n, K key, M measure, u64 want)
{
    DF11_SHARED;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 low = 0, high = ~0ull;
    for (bool first = true;; first = false) {
        // what is left, and its range
        u64 least = ~0ull, most = 0;
        __syncthreads();
        if (tid == 0) s.few_n = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const u64 x = key(i);
            if (x < low || x > high) continue;
            least = min(least, x), most = max(most, x);
            if (first && n > kFew) continue;
            const uint32_t at = atomicAdd(&s.few_n, 1u);
            if (at < (uint32_t)kFew) s.few[at] = x, s.few_measure[at] = measure(i);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            least = min(least, __shfl_xor_sync(0xffffffffu, least, d));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
        }
        if (lane == 0) s.partial[warp] = least, s.partial_most[warp] = most;
        __syncthreads();
        const int few = (int)s.few_n;
        if (few > 0 && few <= kFew) {
            // kThreads / kFew threads per number, each compares it with as large a part of the others
            constexpr int kWays = kThreads / kFew;
            const int mine = tid / kWays;
            const u64 x = mine < few ? s.few[mine] : 0, m = mine < few ? s.few_measure[mine] : 0;
            u64 ahead = 0;
#pragma unroll 4
            for (int j = tid % kWays; j < few; j += kWays) {
                const u64 y = s.few[j], z = s.few_measure[j];
                ahead += y < x ? z : 0;
            }
#pragma unroll
            for (int d = kWays / 2; d; d >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, d);
            if (mine < few && ahead < want && want <= ahead + m) s.border = x;
            __syncthreads();
            return s.border;
        }
        low = ~0ull, high = 0;
        for (int w = 0; w < kWarps; ++w) low = min(low, s.partial[w]), high = max(high, s.partial_most[w]);
        const int shift = max(64 - __clzll(high - low) - 9, 0);             // 512 parts
        s.parts_low[tid] = s.parts_high[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const u64 x = key(i);
            if (x < low || x > high) continue;
            // two additions of 32 bits: one of 64 in shared memory is a loop that many equal parts would stall
            const u64 m = measure(i);
            const uint32_t at = (uint32_t)((x - low) >> shift), m0 = (uint32_t)m;
            const uint32_t was = atomicAdd(&s.parts_low[at], m0), carry = (uint32_t)(was + m0) < was;
            if ((uint32_t)(m >> 32) + carry) atomicAdd(&s.parts_high[at], (uint32_t)(m >> 32) + carry);
        }
        __syncthreads();
        u64 all;
        const u64 mine = (u64)s.parts_high[tid] << 32 | s.parts_low[tid], before = block_scan(mine, s.partial, &all);
        if (before < want && want <= before + mine) s.part = tid, s.base = before;
        __syncthreads();
        want -= s.base;
        low += (u64)s.part << shift;
        if (shift == 0) return low;
        high = min(high, low + ((u64)1 << shift) - 1);
    }
}

// Orders and measures of the tokens on the list.
struct ByRank {
    __device__ __forceinline__ u64 operator()(int i) const { DF11_SHARED; return ~s.list[i]; }
};
struct ByIndex {
    __device__ __forceinline__ u64 operator()(int i) const { DF11_SHARED; return listed_index(s.list[i]); }
};
struct ByCount {
    __device__ __forceinline__ u64 operator()(int) const { return 1; }
};
struct ByMass {
    __device__ __forceinline__ u64 operator()(int i) const { DF11_SHARED; return s.weight[i]; }
};

// Weights of the logits on the list.
__device__ __forceinline__ void weigh_list(int n, const Weigher &weigh)
{
    DF11_SHARED;
    for (int i = threadIdx.x; i < n; i += kThreads) s.weight[i] = weigh(listed_logit(s.list[i]));
    __syncthreads();
}

__device__ __forceinline__ u64 list_mass(int n)
{
    DF11_SHARED;
    u64 mass = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) mass += s.weight[i];
    return block_sum(mass, s.partial);
}

__device__ __forceinline__ u64 share_of(double p, u64 total) { return max((u64)ceil(fmax(p, 0.0) * (double)total), 1ull); }

// The running mass at which the draw falls: the token whose mass takes the sum above it.
__device__ __forceinline__ u64 draw_of(double u, u64 total)
{
    const double border = u > 0.0 ? u * (double)total : 0.0;
    return border >= (double)total ? total - 1 : min((u64)border, total - 1);
}

// ---------------------------------------------------------------------------------------------
// The row's tokens in groups of 8 that start on a 16-byte (or, of floats, a 32-byte) boundary.
template <typename T> struct Tokens {
    static constexpr uint32_t kInfPair = std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
    const T *row;
    uint32_t vocab;
    int lead;                                 // tokens that the first group lacks
    uint32_t groups;
    __device__ __forceinline__ Tokens(const T *r, uint32_t v) : row(r), vocab(v)
    {
        lead = (int)(reinterpret_cast<uintptr_t>(r) / sizeof(T) % 8);
        groups = (v + lead + 7) / 8;
    }
    struct Raw {
        uint4 words[sizeof(T) / 2];
    };
    // Group g as it lies in memory; -inf where there is no token.  Token j of it has the index 8 g - lead + j.
    __device__ __forceinline__ Raw load(uint32_t g) const
    {
        Raw raw;
        const int64_t first = (int64_t)g * 8 - lead;
        if (first >= 0 && first + 8 <= vocab) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw.words[i] = __ldg(reinterpret_cast<const uint4 *>(row + first) + i);
        } else {
            constexpr uint32_t kNone = sizeof(T) == 4 ? 0xFF800000u : kInfPair;
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw.words[i] = make_uint4(kNone, kNone, kNone, kNone);
            T *const x = reinterpret_cast<T *>(raw.words);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (first + j >= 0 && first + j < vocab) x[j] = row[first + j];
        }
        return raw;
    }
    // Its logits; -inf for a NaN.
    __device__ __forceinline__ static void unpack(const Raw &raw, float (&z)[8])
    {
        const T *const x = reinterpret_cast<const T *>(raw.words);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = fmaxf(df11_to_float(x[j]), -INFINITY);
    }
    // Calls f(g, logits) for g = first, first + step, ... below `end`, with four groups on their way at once.
    template <typename F> __device__ __forceinline__ void each4(uint32_t first, uint32_t end, uint32_t step, F f) const
    {
        for (uint32_t g = first; g < end; g += 4 * step) {
            Raw raw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (g + i * step < end) raw[i] = load(g + i * step);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (g + i * step >= end) break;
                float z[8];
                unpack(raw[i], z);
                f(g + i * step, z);
            }
        }
    }
    // Calls f(g, logits) for g = first, first + step, ... below `end`; the next group is on its way meanwhile.
    template <typename F> __device__ __forceinline__ void each(uint32_t first, uint32_t end, uint32_t step, F f) const
    {
        if (first >= end) return;
        Raw next = load(first);
        for (uint32_t g = first; g < end; g += step) {
            const Raw now = next;
            if (g + step < end) next = load(g + step);
            float z[8];
            unpack(now, z);
            f(g, z);
        }
    }
    __device__ __forceinline__ float at(int64_t i) const { return fmaxf(df11_to_float(row[i]), -INFINITY); }
};

// ---------------------------------------------------------------------------------------------
// The slow way, one CTA for the whole row.
//
// The key in which the running measure (from the largest key down) reaches `want`, and the measure
// above it.
template <typename T, typename M>
__device__ void descend(const Tokens<T> &tokens, float lowest, u64 want, M measure, float *found, u64 *above)
{
    DF11_SHARED;
    u64 *digits = s.list;
    uint32_t prefix = 0;
    u64 over = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += kThreads) digits[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < tokens.vocab; i += kThreads) {
            const float z = tokens.at(i);
            const uint32_t key = key_of(z);
            if (z >= lowest && (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)))
                atomicAdd(&digits[(key >> shift) & 255u], measure(z));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 run = over;
            int d = 255;
            while (d > 0 && run + digits[d] < want) run += digits[d--];
            s.found = prefix | (uint32_t)d << shift;
            s.base = run;
        }
        __syncthreads();
        prefix = s.found;
        over = s.base;
    }
    __syncthreads();
    *found = logit_of(prefix);
    *above = over;
}

template <typename T> __device__ __noinline__ void sample_slowly(const Tokens<T> &tokens, const Row &row, float lowest, const Weigher &weigh, int64_t *out)
{
    DF11_SHARED;
    const int tid = threadIdx.x;
    const uint32_t vocab = tokens.vocab;
    float kept = lowest;
    u64 ties_kept = ~0ull, above, total;
    if (row.k > 0 && row.k < vocab) {
        u64 alive = 0;
        for (uint32_t i = tid; i < vocab; i += kThreads) alive += tokens.at(i) >= lowest;
        alive = block_sum(alive, s.partial);
        if ((u64)row.k < alive) {
            descend(tokens, lowest, (u64)row.k, [](float) { return (u64)1; }, &kept, &above);
            ties_kept = (u64)row.k - above;
        }
    }
    if (row.p < 1.0) {
        u64 mass = 0, equal = 0;
        for (uint32_t i = tid; i < vocab; i += kThreads) {
            const float z = tokens.at(i);
            if (z > kept) mass += weigh(z);
            equal += z == kept;
        }
        mass = block_sum(mass, s.partial);
        equal = block_sum(equal, s.partial);
        const u64 each = weigh(kept);
        total = mass + min(equal, ties_kept) * each;
        const u64 want = share_of(row.p, total);
        if (want <= mass) {                       // the border lies above the ties of top-k
            float z;
            const float before = kept;
            descend(tokens, lowest, want, [&](float x) { return x > before ? weigh(x) : (u64)0; }, &z, &above);
            const u64 w = weigh(z);
            kept = z;
            ties_kept = (want - above + w - 1) / w;
        } else if (each > 0) {
            ties_kept = min(ties_kept, (want - mass + each - 1) / each);
        }
    }
    // the draw: every thread has a stretch of the vocabulary, in order
    const double floor = row.low * weigh.unit;
    const uint32_t per = (vocab + kThreads - 1) / kThreads, begin = min(per * tid, vocab), end = min(begin + per, vocab);
    u64 equal = 0;
    for (uint32_t i = begin; i < end; ++i) equal += tokens.at(i) == kept;
    u64 ignored;
    const u64 seen = block_scan(equal, s.partial, &ignored);
    auto weight_at = [&](uint32_t i, u64 &ties) -> u64 {
        const float z = tokens.at(i);
        if (!(z >= kept)) return 0;
        if (z == kept && ties++ >= ties_kept) return 0;
        const double w = weigh.real(z);
        return w < floor ? 0 : weigh.biased(w) - weigh.kBias;
    };
    u64 mine = 0, ties = seen;
    for (uint32_t i = begin; i < end; ++i) mine += weight_at(i, ties);
    u64 run = block_scan(mine, s.partial, &total);
    const u64 want = draw_of(row.u, total);
    if (run <= want && want < run + mine) {
        ties = seen;
        for (uint32_t i = begin; i < end; ++i) {
            run += weight_at(i, ties);
            if (run > want) {
                *out = i;
                break;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// A short list, in any order: every token's rank, the mass before it in that order, and the kept mass
// before it by index come from comparing it with all others, by WAYS threads per token.
template <int WAYS> __device__ __forceinline__ void draw_from_few(int n, const Row &row, const Weigher &weigh, int64_t *out)
{
    DF11_SHARED;
    const int tid = threadIdx.x, mine = tid / WAYS, way = tid % WAYS;
    const bool some = mine < n;
    const u64 me = some ? s.list[mine] : 0;
    const double real = some ? weigh.real(listed_logit(me)) : 0.0;
    const u64 w = weigh.biased(real) - weigh.kBias;
    if (some && way == 0) s.weight[mine] = w;
    __syncthreads();
    int rank = 0;
    u64 before = 0;
#pragma unroll 4
    for (int i = way; i < n; i += WAYS) {
        const u64 x = s.list[i], y = s.weight[i];
        rank += x > me;
        before += x > me ? y : 0;
    }
#pragma unroll
    for (int d = WAYS / 2; d; d >>= 1) {
        rank += __shfl_xor_sync(0xffffffffu, rank, d);
        before += __shfl_xor_sync(0xffffffffu, before, d);
    }
    bool kept = some && (row.k <= 0 || rank < row.k);
    if (row.p < 1.0) {
        const u64 total = block_sum(kept && way == 0 ? w : 0, s.partial);
        kept = kept && (rank == 0 || before < share_of(row.p, total));
    }
    kept = kept && real >= row.low * weigh.unit;
    __syncthreads();
    if (some && way == 0) s.weight[mine] = kept ? w : 0;
    const u64 total = block_sum(kept && way == 0 ? w : 0, s.partial), want = draw_of(row.u, total);
    u64 upto = 0;
    const uint32_t index = (uint32_t)me;                         // larger for a lower index
#pragma unroll 4
    for (int i = way; i < n; i += WAYS) {
        const uint32_t x = (uint32_t)s.list[i];
        const u64 y = s.weight[i];
        upto += x > index ? y : 0;
    }
#pragma unroll
    for (int d = WAYS / 2; d; d >>= 1) upto += __shfl_xor_sync(0xffffffffu, upto, d);
    if (kept && upto <= want && want < upto + w) *out = listed_index(me);
}

// The list holds the highest-ranked n tokens of the row, at least those that top-k keeps: all filters and the draw.
__device__ __noinline__ void draw_from_list(int n, const Row &row, const Weigher &weigh, int64_t *out)
{
    DF11_SHARED;
    if (n > kFew && row.k > 0 && row.k <= kFew) {
        // only what top-k keeps stays on the list
        const u64 border = find_border(n, ByRank(), ByCount(), (u64)row.k);
        u64 mine[kList / kThreads];
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j) mine[j] = threadIdx.x + j * kThreads < n ? s.list[threadIdx.x + j * kThreads] : 0;
        __syncthreads();
        if (threadIdx.x == 0) s.few_n = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j)
            if (mine[j] && ~mine[j] <= border) s.list[atomicAdd(&s.few_n, 1u)] = mine[j];
        __syncthreads();
        n = (int)s.few_n;
    }
    if (n <= kThreads / 16) return draw_from_few<16>(n, row, weigh, out);
    if (n <= kFew) return draw_from_few<kThreads / kFew>(n, row, weigh, out);
    weigh_list(n, weigh);
    const ByRank by_rank;
    const ByMass mass;
    auto drop_behind = [&](u64 border) {
        for (int i = threadIdx.x; i < n; i += kThreads)
            if (by_rank(i) > border) s.weight[i] = 0;
        __syncthreads();
    };
    if (row.k > 0 && row.k < n) drop_behind(find_border(n, by_rank, ByCount(), (u64)row.k));
    if (row.p < 1.0) drop_behind(find_border(n, by_rank, mass, share_of(row.p, list_mass(n))));
    if (row.low > 0.0) {                      // min-p
        const double floor = row.low * weigh.unit;
        for (int i = threadIdx.x; i < n; i += kThreads)
            if (weigh.real(listed_logit(s.list[i])) < floor) s.weight[i] = 0;
        __syncthreads();
    }
    const u64 want = draw_of(row.u, list_mass(n)) + 1;
    const u64 index = find_border(n, ByIndex(), mass, want);
    if (threadIdx.x == 0) *out = (int64_t)index;
}

struct SampleArgs {
    const void *logits;
    int64_t stride;
    uint32_t vocab, cluster;
    const float *uniform, *temperature, *top_p, *min_p;
    const int *top_k;
    double temperature_value, top_p_value, min_p_value;
    int top_k_value;
    int64_t *out;
    int *status;
};

template <typename T> __global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs a)
{
    DF11_SHARED;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t size = a.cluster, at = blockIdx.x / size, rank = blockIdx.x % size;
    Row row;
    row.t = a.temperature ? (double)a.temperature[at] : a.temperature_value;
    row.k = a.top_k ? a.top_k[at] : a.top_k_value;
    row.p = a.top_p ? (double)a.top_p[at] : a.top_p_value;
    row.low = a.min_p ? (double)a.min_p[at] : a.min_p_value;
    row.low = row.low > 0.0 ? fmin(row.low, 1.0) : 0.0;
    row.u = (double)a.uniform[at];
    if (row.k >= a.vocab) row.k = 0;
    const Tokens<T> tokens((const T *)a.logits + (int64_t)at * a.stride, a.vocab);

    // this CTA's groups, in blocks of 32 << wide of them
    int wide = 0;
    while (((tokens.groups + size - 1) / size + (32u << wide) - 1) >> (5 + wide) > (uint32_t)kBlocks) ++wide;
    const uint32_t block_groups = 32u << wide, all_blocks = (tokens.groups + block_groups - 1) / block_groups;
    const uint32_t my_blocks = (all_blocks + size - 1) / size, block0 = min(rank * my_blocks, all_blocks);
    const uint32_t blocks = min(my_blocks, all_blocks - block0);
    const uint32_t g0 = block0 * block_groups, g1 = min(g0 + blocks * block_groups, tokens.groups);

    // the largest and the smallest logit
    const bool greedy = !(row.t > 0.0), few = !greedy && row.k > 0 && row.k <= kFewTokens;
    float top = -INFINITY, bottom = INFINITY;
    tokens.each4(g0 + tid, g1, kThreads, [&](uint32_t, const float (&z)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            top = fmaxf(top, z[j]);
            bottom = fminf(bottom, z[j] > -INFINITY ? z[j] : INFINITY);
        }
    });
    if (tid < kRoots) s.roots[tid] = exp2((double)tid / kRoots);
    if (tid == 0) s.mine.bound = -INFINITY, s.list_n = 0, s.found = kAny;
    {
        float x = top, y = bottom;
#pragma unroll
        for (int d = 16; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d)), y = fminf(y, __shfl_xor_sync(0xffffffffu, y, d));
        if (lane == 0) s.partial_top[warp] = x, s.partial_bottom[warp] = y;
    }
    if (few) {
        // a bound that k of the threads' largest logits reach: at least k tokens reach it, too.  Any such
        // bound will do; the search ends when half as many again reach it
        const uint32_t key = key_of(top);
        uint32_t low = 0, high = kAny;
        for (int i = 0; i < 32 && low < high; ++i) {
            const uint32_t middle = low + (high - low) / 2 + 1;
            const int n = __syncthreads_count(key >= middle);
            if (n >= row.k) low = middle;
            else high = middle - 1;
            if (n >= row.k && n <= row.k + row.k / 2) break;
        }
        if (tid == 0) s.mine.bound = low < kLowestKey ? -INFINITY : logit_of(low);
    }
    __syncthreads();
    if (tid == 0) {
        float x = -INFINITY, y = INFINITY;
        for (int w = 0; w < kWarps; ++w) x = fmaxf(x, s.partial_top[w]), y = fminf(y, s.partial_bottom[w]);
        s.mine.best = x, s.mine.least = y;
    }
    cluster_sync(size);
    float best = -INFINITY, least = INFINITY, bound = -INFINITY;
    if (lane < (int)size) {
        const Exchange *x = size > 1 ? remote(&s.mine, lane) : &s.mine;
        best = x->best, least = x->least, bound = x->bound;
    }
#pragma unroll
    for (int d = 4; d; d >>= 1) {
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d));
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, d));
        bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, d));
    }
    best = __shfl_sync(0xffffffffu, best, 0), least = __shfl_sync(0xffffffffu, least, 0), bound = __shfl_sync(0xffffffffu, bound, 0);
    if (best == -INFINITY) {                                 // nothing to draw from
        if (rank == 0 && tid == 0) {
            a.out[at] = 0;
            if (a.status) atomicOr(a.status, DF11_STATUS_EMPTY_ROW);
        }
        cluster_sync(size);
        return;
    }
    Shared &head = *(size > 1 ? remote(&s, 0) : &s);
    if (greedy) {
        uint32_t index = kAny;
        tokens.each4(g0 + tid, g1, kThreads, [&](uint32_t g, const float (&z)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (z[j] == best) index = min(index, g * 8 - tokens.lead + j);
        });
        index = __reduce_min_sync(0xffffffffu, index);
        if (lane == 0 && index != kAny) atomicMin(&head.found, index);
        cluster_sync(size);
        if (rank == 0 && tid == 0) a.out[at] = s.found;
        return;
    }
    const float lowest = best == INFINITY ? best : -3.402823466e38f;    // beside a +inf nothing else is drawn
    const int shift = min(31 + __clz(a.vocab), 50);                     // vocab * 2^shift < 2^63
    const Weigher weigh(best, row.t, shift, s.roots);
    const double floor = row.low * weigh.unit;                          // weights below it are min-p's

    auto list_token = [&](float z, uint32_t index) {
        const uint32_t n = atomicAdd(&s.list_n, 1u);
        if (n < (uint32_t)kList) s.list[n] = listed(z, index);
    };
    // The first CTA, after a barrier: everyone's list behind its own; more than kList if they do not fit.
    auto collect = [&]() {
        if (size == 1) return s.list_n;
        // every lane below the cluster's size learns one CTA's count; a warp copies one CTA's list
        uint32_t n = lane < (int)size ? remote(&s, lane)->list_n : 0, behind = n;
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, behind, d);
            if (lane >= d) behind += x;
        }
        const uint32_t all = __shfl_sync(0xffffffffu, behind, size - 1);
        const uint32_t r = warp % size, more = __shfl_sync(0xffffffffu, n, r), at_list = __shfl_sync(0xffffffffu, behind, r) - more;
        if (r > 0 && all <= (uint32_t)kList) {
            const Shared &there = *remote(&s, r);
            for (uint32_t i = warp / size * 32 + lane; i < more; i += kWarps / size * 32) s.list[at_list + i] = there.list[i];
        }
        __syncthreads();
        return all;
    };
    if (few) {
        bound = fmaxf(bound, lowest);
        tokens.each4(g0 + tid, g1, kThreads, [&](uint32_t g, const float (&z)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (z[j] >= bound) list_token(z[j], g * 8 - tokens.lead + j);
        });
        cluster_sync(size);
        const uint32_t n = rank == 0 ? collect() : 0;
        if (size > 1) cluster_sync(size);
        if (rank != 0) return;
        if (n <= (uint32_t)kList) draw_from_list((int)n, row, weigh, a.out + at);
        else sample_slowly(tokens, row, lowest, weigh, a.out + at);
        return;
    }

    // Calls f(g, logits, part) for all groups, a block per warp; what f adds to `part` becomes the block's sum.
    auto each_block = [&](auto f) {
        if ((uint32_t)warp >= blocks) return;
        const uint32_t last_of = (1u << wide) - 1, steps = (blocks - warp + kWarps - 1) / kWarps << wide;
        auto group_of = [&](uint32_t q) { return g0 + (warp + (q >> wide) * kWarps) * block_groups + (q & last_of) * 32 + lane; };
        u64 part = 0;
        for (uint32_t q = 0; q < steps; ++q) {
            const uint32_t g = group_of(q);
            if (g < g1) {
                float z[8];
                tokens.unpack(tokens.load(g), z);
                f(g, z, part);
            }
            if ((q & last_of) == last_of) {
#pragma unroll
                for (int d = 16; d; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
                if (lane == 0) s.blocks[warp + (q >> wide) * kWarps] = part;
                part = 0;
            }
        }
    };

    float kept_logit = lowest;                                          // the filters' border so far
    uint32_t kept_index = kAny;
    auto is_kept = [&](float z, uint32_t index) { return z > kept_logit || (z == kept_logit && index <= kept_index); };
    const bool by_rank = row.k > 0, by_mass = row.p < 1.0;
    if (by_rank || by_mass) {
        // tokens per interval
        const float range = fminf(best - fmaxf(least, lowest), 31.2f * (float)fmin(row.t, 1e37));
        const float scale = range > 0.0f ? fminf((float)kBins / range, 1e30f) : 0.0f;
        // An interval's number, as the low bits of a float.  Beside a +inf all that counts is equal.
        constexpr float kMagic = 8388608.0f;
        const float from = fminf(best, 3.402823466e38f);
        auto place_of = [&](float z) { return fminf(fmaf(from - z, scale, kMagic), kMagic + (kBins - 1)); };
        auto bin_of = [&](float z) { return (int)(__float_as_uint(place_of(fminf(z, from))) & (kBins - 1)); };
        for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0;
        __syncthreads();
        tokens.each(g0 + tid, g1, kThreads, [&](uint32_t, const float (&z)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (z[j] >= lowest) atomicAdd(&s.count[bin_of(z[j])], 1u);
        });
        cluster_sync(size);
        if (size > 1) {
            for (int i = (int)rank * (kBins / (int)size) + tid; i < ((int)rank + 1) * (kBins / (int)size); i += kThreads) {
                uint32_t n = 0;
                for (uint32_t r = 0; r < size; ++r) n += *remote(&s.count[i], r);
                for (uint32_t r = 0; r < size; ++r) *remote(&s.merged[i], r) = n;
            }
            cluster_sync(size);
        }
        const uint32_t *const count = size > 1 ? s.merged : s.count;

        // the intervals of the borders; every CTA finds the same ones
        constexpr int kEach = kBins / kThreads;
        if (tid == 0) {
            s.bin_k = s.bin_p = s.bin_high = kBins - 1, s.above_k = s.bin_low = s.above_low = 0;
            s.verdict.fallback = 0;
        }
        uint32_t c[kEach], mine = 0, whole;
#pragma unroll
        for (int j = 0; j < kEach; j += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(count + tid * kEach + j);
            c[j] = x.x, c[j + 1] = x.y, c[j + 2] = x.z, c[j + 3] = x.w;
            mine += x.x + x.y + x.z + x.w;
        }
        const uint32_t ahead = block_scan(mine, s.partial_count, &whole);
        if (tid == 0) s.upto_high = whole;
        const uint32_t limit = by_rank ? (uint32_t)min(row.k, (long long)whole) : whole;
        // an interval's width in octaves; its tokens weigh what its middle weighs, to half of that
        const float width = scale > 0.0f ? (float)fmin(1.4426950408889634074 / row.t / scale, 1e30) : 0.0f;
        float mass[kEach], sum = 0.0f, squares = 0.0f;
        {
            uint32_t n = ahead;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int bin = tid * kEach + j;
                if (n < limit && n + c[j] >= limit) s.bin_k = bin, s.above_k = n;
                mass[j] = by_mass && c[j] && n < limit ? (float)min(c[j], limit - n) * exp2f(-width * (bin + 0.5f)) : 0.0f;
                sum += mass[j];
                squares += mass[j] * mass[j];
                n += c[j];
            }
        }
        if (by_mass) {
            float all, run = block_scan(sum, s.partial_real, &all);
            // The border's place is off by what the masses before it and their sum are.  No interval is off by
            // more than half its width, which bounds it; if they are off independently of one another,
            // by a tenth of that or less, for which five standard deviations are allowed here.
            const float spread = sqrtf(block_sum(squares, s.partial_real)) * (0.2f * width) * 10.0f + 1e-5f * all;
            const float want = (float)fmax(row.p, 0.0) * all, margin = fminf(2.1f * (exp2f(0.5f * width) - 1.0f) * all + 1e-5f * all, spread);
            uint32_t n = ahead;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int bin = tid * kEach + j;
                const float next = run + mass[j];
                if (mass[j] > 0.0f) {
                    if (run < want && next >= want) s.bin_p = bin;
                    if (run < want - margin && next >= want - margin) s.bin_low = bin, s.above_low = n;
                    if (run < want + margin && next >= want + margin) s.bin_high = bin, s.upto_high = n + c[j];
                }
                run = next;
                n += c[j];
            }
        }
        __syncthreads();
        if (by_rank) {
            const int bin = s.bin_k;
            // what top-k keeps, as a whole or the interval of its border
            const bool all = s.above_k + count[bin] <= (uint32_t)kList;
            tokens.each(g0 + tid, g1, kThreads, [&](uint32_t g, const float (&z)[8]) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (z[j] >= lowest) {
                        const int b = bin_of(z[j]);
                        if (b == bin || (all && b < bin)) list_token(z[j], g * 8 - tokens.lead + j);
                    }
            });
            cluster_sync(size);
            if (rank == 0) {
                const uint32_t n = collect();
                if (n > (uint32_t)kList) {
                    if (tid == 0) s.verdict.fallback = 1;
                } else if (all) {
                    draw_from_list((int)n, row, weigh, a.out + at);
                    if (tid == 0) s.verdict.fallback = 2;
                } else {
                    const u64 last = ~find_border((int)n, ByRank(), ByCount(), (u64)(limit - s.above_k));
                    if (tid == 0) s.verdict.logit = listed_logit(last), s.verdict.index = listed_index(last);
                }
            }
            cluster_sync(size);
            if (tid == 0) s.list_n = 0;
            const Verdict v = head.verdict;
            if (v.fallback) {
                cluster_sync(size);
                if (v.fallback == 1 && rank == 0) sample_slowly(tokens, row, lowest, weigh, a.out + at);
                return;
            }
            kept_logit = v.logit, kept_index = v.index;
        }
        if (by_mass) {
            // all intervals in which the border can lie, or as many around the likely one as the list takes
            if (tid == 0 && s.upto_high - s.above_low > (uint32_t)kList) {
                int low = s.bin_p, high = low;
                uint32_t n = count[low];
                for (int i = 0; i < 8; ++i) {
                    if (low > 0 && n + count[low - 1] <= (uint32_t)kList) n += count[--low];
                    if (high < kBins - 1 && n + count[high + 1] <= (uint32_t)kList) n += count[++high];
                }
                s.bin_low = low, s.bin_high = high;
            }
            __syncthreads();
            // one pass: mass of what top-k keeps, mass above the intervals, sums of blocks of the latter
            const float low = kMagic + s.bin_low, high = kMagic + s.bin_high;
            u64 mass_all = 0, mass_above = 0;
            auto add_up = [&](auto filtered, auto plain) {
                each_block([&](uint32_t g, const float (&z)[8], u64 &part) {
                    const uint32_t index = g * 8 - tokens.lead;
                    uint32_t on_list = 0;
                    u64 above = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool kept = !filtered.value || is_kept(z[j], index + j);
                        const float place = place_of(plain.value ? z[j] : fminf(z[j], from));
                        const double w = plain.value ? weigh.fast(z[j]) : weigh.real(z[j]);
                        const u64 all = weigh.biased(kept ? w : 0.0);
                        mass_all += all;
                        above += place < low ? all : weigh.kBias;
                        if (filtered.value) part += place < low && w >= floor ? all : weigh.kBias;
                        if (place >= low && place <= high && kept && z[j] >= lowest) on_list |= 1u << j;
                    }
                    mass_all -= 8 * weigh.kBias, above -= 8 * weigh.kBias;
                    mass_above += above;
                    part += filtered.value ? 0 - 8 * weigh.kBias : above;
                    if (on_list) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (on_list >> j & 1) list_token(z[j], index + j);
                    }
                });
            };
            if (!weigh.plain) add_up(Yes{}, No{});
            else if (by_rank || floor > 0.0) add_up(Yes{}, Yes{});
            else add_up(No{}, Yes{});
            mass_all = block_sum(mass_all, s.partial);
            mass_above = block_sum(mass_above, s.partial);
            if (tid == 0) s.mine.mass = mass_all, s.mine.above = mass_above;
            cluster_sync(size);
            if (rank == 0) {
                mass_all = mass_above = 0;
                for (uint32_t r = 0; r < size; ++r) {
                    const Exchange *x = size > 1 ? remote(&s.mine, r) : &s.mine;
                    mass_all += x->mass, mass_above += x->above;
                }
                const u64 want = share_of(row.p, mass_all);
                const uint32_t in_all = collect();
                const int n = (int)min(in_all, (uint32_t)kList);
                weigh_list(n, weigh);
                const u64 on_list = list_mass(n);
                if (in_all > (uint32_t)kList || mass_above >= want || mass_above + on_list < want) {
                    if (tid == 0) s.verdict.fallback = 1;
                } else {
                    const u64 last = find_border(n, ByRank(), ByMass(),
                                                 want - mass_above);
                    if (tid == 0) s.verdict.logit = listed_logit(~last), s.verdict.index = listed_index(~last);
                    for (int i = tid; i < n; i += kThreads) {
                        if (~s.list[i] > last || (floor > 0.0 && weigh.real(listed_logit(s.list[i])) < floor)) continue;
                        const uint32_t index = listed_index(s.list[i]);
                        const uint32_t block = (index + tokens.lead) / 8 / block_groups, owner = block / my_blocks;
                        atomicAdd(&(size > 1 ? remote(&s, owner) : &s)->blocks[block - owner * my_blocks], s.weight[i]);
                    }
                }
            }
            cluster_sync(size);
            const Verdict v = head.verdict;
            if (v.fallback) {
                cluster_sync(size);
                if (rank == 0) sample_slowly(tokens, row, lowest, weigh, a.out + at);
                return;
            }
            kept_logit = v.logit, kept_index = v.index;
        }
    }
    if (!by_mass) {
        auto add_up = [&](auto filtered, auto plain) {
            each_block([&](uint32_t g, const float (&z)[8], u64 &part) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double w = plain.value ? weigh.fast(z[j]) : weigh.real(z[j]);
                    part += weigh.biased(!filtered.value || (is_kept(z[j], g * 8 - tokens.lead + j) && w >= floor) ? w : 0.0);
                }
                part -= 8 * weigh.kBias;
            });
        };
        if (!weigh.plain) add_up(Yes{}, No{});
        else if (by_rank || floor > 0.0) add_up(Yes{}, Yes{});
        else add_up(No{}, Yes{});
    }
    // the draw: the CTA, the block, the token
    __syncthreads();
    u64 sum = (uint32_t)tid < blocks ? s.blocks[tid] : 0, mine;
    u64 run = block_scan(sum, s.partial, &mine);
    if (tid == 0) s.mine.blocks = mine;
    cluster_sync(size);
    u64 before = 0, total = 0;
    for (uint32_t r = 0; r < size; ++r) {
        const u64 x = size > 1 ? remote(&s.mine, r)->blocks : s.mine.blocks;
        if (r < rank) before += x;
        total += x;
    }
    const u64 want = draw_of(row.u, total);
    run += before;
    if (before <= want && want < before + mine) {
        if (run <= want && want < run + sum) s.found = (uint32_t)tid, s.base = run;
        __syncthreads();
        if (warp == 0) {
            run = s.base;
            for (int x = 0; x < 1 << wide; ++x) {
                const uint32_t g = g0 + s.found * block_groups + x * 32 + lane;
                float z[8];
                if (g < g1) tokens.unpack(tokens.load(g), z);
                u64 w[8];
                sum = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = 0;
                    if (g < g1 && is_kept(z[j], g * 8 - tokens.lead + j)) {
                        const double real = weigh.real(z[j]);
                        if (real >= floor) w[j] = weigh.biased(real) - weigh.kBias;
                    }
                    sum += w[j];
                }
                u64 upto = sum;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const u64 y = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += y;
                }
                u64 here = run + upto - sum;
                if (here <= want && want < here + sum) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (here <= want && want < here + w[j]) a.out[at] = (int64_t)g * 8 - tokens.lead + j;
                        here += w[j];
                    }
                }
                run += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
    }
    cluster_sync(size);                       // nobody leaves while its memory is read
}

}  // namespace

extern "C" int df11_sample(const void *logits, int64_t row_stride, int32_t element_type, int64_t rows, int64_t vocab,
                           const void *uniform, const void *temperature, double temperature_value, const void *top_k,
                           int32_t top_k_value, const void *top_p, double top_p_value, const void *min_p, double min_p_value,
                           void *out, void *status, int32_t device, void *stream)
{
    if (!logits || !uniform || !out) return df11_fail(DF11_ERR_BADARG, "null pointer");
    if (element_type < DF11_TYPE_BF16 || element_type > DF11_TYPE_FP32)
        return df11_fail(DF11_ERR_BADARG, "unknown element type %d", element_type);
    if (rows < 0 || rows > 0x7FFFFFFF || vocab < 1 || vocab > 0x7FFFFFF0)
        return df11_fail(DF11_ERR_BADARG, "rows or vocab out of range");
    if (row_stride < 0) return df11_fail(DF11_ERR_BADARG, "negative row stride");
    const uintptr_t unit = element_type == DF11_TYPE_FP32 ? 3 : 1;
    if (((uintptr_t)logits & unit) || ((uintptr_t)out & 7) ||
        (((uintptr_t)uniform | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)status) & 3))
        return df11_fail(DF11_ERR_BADARG, "misaligned pointer");
    if (rows == 0) return DF11_OK;
    // CTAs per row: two fit on an SM; a row of a few thousand tokens is not worth dividing
    uint32_t cluster = rows <= 37 ? 8 : rows <= 74 ? 4 : rows <= 148 ? 2 : 1;
    while (cluster > 1 && vocab < (int64_t)cluster * 8 * kThreads) cluster >>= 1;
    if (rows * cluster > 0x7FFFFFFF) cluster = 1;
    Df11DeviceScope scope(device);
    if (!scope.ok) return df11_fail(DF11_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    SampleArgs a = {};
    a.logits = logits, a.stride = row_stride, a.vocab = (uint32_t)vocab, a.cluster = cluster;
    a.uniform = (const float *)uniform, a.temperature = (const float *)temperature, a.top_p = (const float *)top_p;
    a.min_p = (const float *)min_p, a.top_k = (const int *)top_k;
    a.temperature_value = temperature_value, a.top_p_value = top_p_value, a.min_p_value = min_p_value, a.top_k_value = top_k_value;
    a.out = (int64_t *)out, a.status = (int *)status;
    auto go = [&](auto kernel) {
        const cudaError_t set = df11_allow_shared((const void *)kernel, sizeof(Shared), device);
        if (set != cudaSuccess) return set;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)(rows * cluster));
        config.blockDim = dim3(kThreads);
        config.dynamicSmemBytes = sizeof(Shared);
        config.stream = (cudaStream_t)stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        config.attrs = attr;
        config.numAttrs = cluster > 1;
        return cudaLaunchKernelEx(&config, kernel, a);
    };
    const cudaError_t e = element_type == DF11_TYPE_BF16 ? go(sample_kernel<__nv_bfloat16>)
                        : element_type == DF11_TYPE_FP16 ? go(sample_kernel<__half>) : go(sample_kernel<float>);
    if (e != cudaSuccess) return df11_fail(DF11_ERR_CUDA, "kernel launch failed: %s", cudaGetErrorString(e));
    return DF11_OK;
}
