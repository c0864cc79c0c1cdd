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
//     largest of all.  The tokens above it are few; they are listed, sorted, and all filters and the
//     draw are done on the list.
//   * otherwise the tokens are counted in 4096 intervals of equal width between the largest logit
//     and the one whose weight no longer matters (or the smallest).  Counts give the interval of the top-k border
//     exactly, and, times the weight in the interval's middle, that of the top-p border almost.
//     One pass over the row then adds up the exact mass above those intervals and lists what lies in them;
//     the sorted list gives the border, and exact sums prove that it lies there.
//   * where a list would overflow (thousands of equal logits at the border) or the guess was
//     wrong, one CTA finds the border digit by digit of the logits' bits.
// The draw needs masses in index order: sums of blocks of 256 or more tokens are kept by the same
// pass, and only the block that holds the border is looked at again.
//
// A row is divided among a cluster of 1 to 8 CTAs, as many as leave every SM with work.  The row is
// read two or three times, the first time from memory, then from the L2 cache.  Bound: for few rows the chain of
// cluster barriers, for many the fp64 units (about 11 operations per token at half a warp per clock).
#include <math.h>

#include "df11_launch.h"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 4096;
constexpr int kList = 2048;
constexpr int kBlocks = kThreads;             // block sums per CTA, at most
constexpr int kFewTokens = 256;               // top-k up to here goes by the threads' largest
constexpr uint32_t kLowestKey = 0x00800000u;  // key of the lowest finite float; NaN and -inf lie below
constexpr uint32_t kInfKey = 0xFF800000u;
constexpr uint32_t kAny = 0xFFFFFFFFu;

using u64 = unsigned long long;

// A number that orders like the logit (-0 like 0); 0 for a NaN.
__device__ __forceinline__ uint32_t key_of(float z)
{
    const uint32_t b = __float_as_uint(z + 0.0f);
    return z != z ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
}

__device__ __forceinline__ float logit_of(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

struct Weigher {
    double peak, inverse, unit;
    __device__ __forceinline__ double real(uint32_t key) const
    {
        const double z = (double)logit_of(key);
        const double d = z == peak ? 0.0 : z - peak;
        return d == -INFINITY ? 0.0 : exp(d * inverse);   // beside a +inf; an infinite temperature must not bring it back
    }
    __device__ __forceinline__ u64 operator()(uint32_t key) const { return __double2ull_rn(real(key) * unit); }
};

struct Row {             // settings of a row
    double t, p, low, u;
    long long k;
};

struct Exchange {        // what the CTAs of a cluster tell one another
    uint32_t best, least, bound;
    u64 mass, above, blocks;
};

struct Verdict {         // what the first CTA finds on its list
    uint32_t key, index;                      // kept: keys above, or equal with an index up to this one
    int fallback;
};

struct Shared {
    uint32_t count[kBins];                    // this CTA's counts
    uint32_t merged[kBins];                   // the row's
    u64 list[kList], weight[kList];
    u64 blocks[kBlocks];
    u64 partial[kWarps];
    double partial_real[kWarps];
    Exchange mine;
    Verdict verdict;
    uint32_t list_n, found;
    int bin_k, bin_low, bin_high;             // interval of the top-k border; intervals of the top-p border
    uint32_t above_k;                         // tokens above bin_k
    u64 base;
};

__device__ __forceinline__ void cluster_sync(uint32_t size)
{
    if (size > 1) asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
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

// Sorts list[0 .. n) in descending order (n <= kList); what is behind it, up to a power of two, is lost.
__device__ void sort_list(u64 *list, int n)
{
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = 0;
    __syncthreads();
    for (int span = 2; span <= size; span <<= 1)
        for (int step = span >> 1; step; step >>= 1) {
            for (int i = threadIdx.x; i < size / 2; i += kThreads) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const u64 x = list[a], y = list[b];
                if ((x < y) == ((a & span) == 0)) list[a] = y, list[b] = x;
            }
            __syncthreads();
        }
}

__device__ __forceinline__ u64 listed(uint32_t key, uint32_t index) { return (u64)key << 32 | (0xFFFFFFFFu - index); }
__device__ __forceinline__ uint32_t listed_key(u64 x) { return (uint32_t)(x >> 32); }
__device__ __forceinline__ uint32_t listed_index(u64 x) { return 0xFFFFFFFFu - (uint32_t)x; }

// Running sums of weigh(key) over list[0 .. n), in `sums`; the whole sum is returned.
template <typename K> __device__ u64 scan_list(const u64 *list, int n, u64 *sums, u64 *partial, K key, const Weigher &weigh)
{
    constexpr int kEach = kList / kThreads;
    u64 w[kEach], mine = 0, total;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = threadIdx.x * kEach + j;
        w[j] = i < n ? weigh(key(list[i])) : 0;
        mine += w[j];
    }
    u64 run = block_scan(mine, partial, &total);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = threadIdx.x * kEach + j;
        run += w[j];
        if (i < n) sums[i] = run;
    }
    __syncthreads();
    return total;
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
    const T *row;
    uint32_t vocab;
    int lead;                                 // tokens that the first group lacks
    uint32_t groups;
    __device__ __forceinline__ Tokens(const T *r, uint32_t v) : row(r), vocab(v)
    {
        lead = (int)(reinterpret_cast<uintptr_t>(r) / sizeof(T) % 8);
        groups = (v + lead + 7) / 8;
    }
    // keys of group g; 0 where there is no token.  Token j of it has the index 8 g - lead + j.
    __device__ __forceinline__ void keys(uint32_t g, uint32_t (&key)[8]) const
    {
        const int64_t first = (int64_t)g * 8 - lead;
        if (first >= 0 && first + 8 <= vocab) {
            uint4 raw[sizeof(T) / 2];
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4 *>(row + first) + i);
            const T *z = reinterpret_cast<const T *>(raw);
#pragma unroll
            for (int j = 0; j < 8; ++j) key[j] = key_of(df11_to_float(z[j]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) key[j] = first + j >= 0 && first + j < vocab ? key_of(df11_to_float(row[first + j])) : 0u;
        }
    }
    __device__ __forceinline__ uint32_t key_at(int64_t i) const { return key_of(df11_to_float(row[i])); }
};

// ---------------------------------------------------------------------------------------------
// The slow way, one CTA for the whole row.
//
// The key in which the running measure (from the largest key down) reaches `want`, and the measure
// above it.
template <typename T, typename M>
__device__ void descend(const Tokens<T> &tokens, uint32_t lowest, u64 want, M measure, Shared &s, uint32_t *found, u64 *above)
{
    u64 *digits = s.list;
    uint32_t prefix = 0;
    u64 over = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += kThreads) digits[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < tokens.vocab; i += kThreads) {
            const uint32_t key = tokens.key_at(i);
            if (key >= lowest && (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)))
                atomicAdd(&digits[(key >> shift) & 255u], measure(key));
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
    *found = prefix;
    *above = over;
}

template <typename T> __device__ void sample_slowly(const Tokens<T> &tokens, const Row &row, uint32_t best, uint32_t lowest, const Weigher &weigh,
                                                    Shared &s, int64_t *out)
{
    const int tid = threadIdx.x;
    const uint32_t vocab = tokens.vocab;
    uint32_t kept = lowest;
    u64 ties_kept = ~0ull, above, total;
    if (row.k > 0 && row.k < vocab) {
        descend(tokens, lowest, (u64)row.k, [](uint32_t) { return (u64)1; }, s, &kept, &above);
        ties_kept = (u64)row.k - min(above, (u64)row.k);
        if (kept < lowest) kept = lowest, ties_kept = ~0ull;
    }
    if (row.p < 1.0) {
        u64 mass = 0, equal = 0;
        for (uint32_t i = tid; i < vocab; i += kThreads) {
            const uint32_t key = tokens.key_at(i);
            if (key > kept) mass += weigh(key);
            equal += key == kept;
        }
        mass = block_sum(mass, s.partial);
        equal = block_sum(equal, s.partial);
        const u64 each = weigh(kept);
        total = mass + min(equal, ties_kept) * each;
        const u64 want = share_of(row.p, total);
        if (want <= mass) {                       // the border lies above the ties of top-k
            uint32_t key;
            const uint32_t before = kept;
            descend(tokens, lowest, want, [&](uint32_t x) { return x > before ? weigh(x) : (u64)0; }, s, &key, &above);
            const u64 w = weigh(key);
            kept = key;
            ties_kept = (want - above + w - 1) / w;
        } else if (each > 0) {
            ties_kept = min(ties_kept, (want - mass + each - 1) / each);
        }
    }
    // the draw: every thread has a stretch of the vocabulary, in order
    const uint32_t per = (vocab + kThreads - 1) / kThreads, begin = min(per * tid, vocab), end = min(begin + per, vocab);
    u64 equal = 0;
    for (uint32_t i = begin; i < end; ++i) equal += tokens.key_at(i) == kept;
    u64 ignored;
    const u64 seen = block_scan(equal, s.partial, &ignored);
    auto weight_at = [&](uint32_t i, u64 &ties) -> u64 {
        const uint32_t key = tokens.key_at(i);
        if (key < kept || key < lowest) return 0;
        if (key == kept && ties++ >= ties_kept) return 0;
        if (row.low > 0.0 && key != best && weigh.real(key) < row.low) return 0;
        return weigh(key);
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
// The list holds the highest-ranked n tokens of the row, at least those that top-k (or top-p with the mass
// `total`) keeps: all filters and the draw.  total 0: the mass of what top-k keeps.
__device__ void draw_from_list(int n, const Row &row, u64 total, uint32_t best, const Weigher &weigh, Shared &s, int64_t *out)
{
    sort_list(s.list, n);
    if (row.k > 0 && row.k < n) n = (int)row.k;
    const u64 sum = scan_list(s.list, n, s.weight, s.partial, listed_key, weigh);
    if (row.p < 1.0) {
        const u64 want = share_of(row.p, total ? total : sum);
        int fit = 0;
        for (int i = threadIdx.x; i < n; i += kThreads) fit += i == 0 || s.weight[i - 1] < want;
        n = (int)block_sum((u64)fit, s.partial);
    }
    if (row.low > 0.0) {
        int fit = 0;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t key = listed_key(s.list[i]);
            fit += key == best || weigh.real(key) >= row.low;
        }
        n = (int)block_sum((u64)fit, s.partial);
    }
    for (int i = threadIdx.x; i < n; i += kThreads) s.list[i] = s.list[i] << 32 | s.list[i] >> 32;   // now by index
    __syncthreads();
    sort_list(s.list, n);
    const u64 kept = scan_list(s.list, n, s.weight, s.partial, [](u64 x) { return (uint32_t)x; }, weigh);
    const u64 want = draw_of(row.u, kept);
    for (int i = threadIdx.x; i < n; i += kThreads)
        if (s.weight[i] > want && (i == 0 || s.weight[i - 1] <= want)) *out = 0xFFFFFFFFu - (uint32_t)(s.list[i] >> 32);
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
    extern __shared__ __align__(16) unsigned char raw_shared[];
    Shared &s = *reinterpret_cast<Shared *>(raw_shared);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t size = a.cluster, at = blockIdx.x / size, rank = blockIdx.x % size;
    Row row;
    row.t = a.temperature ? (double)a.temperature[at] : a.temperature_value;
    row.k = a.top_k ? a.top_k[at] : a.top_k_value;
    row.p = a.top_p ? (double)a.top_p[at] : a.top_p_value;
    row.low = fmin(a.min_p ? (double)a.min_p[at] : a.min_p_value, 1.0);
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
    uint32_t top = 0, bottom = kAny;
    for (uint32_t g = g0 + tid; g < g1; g += kThreads) {
        uint32_t key[8];
        tokens.keys(g, key);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            top = max(top, key[j]);
            if (key[j] >= kLowestKey) bottom = min(bottom, key[j]);
        }
    }
    if (tid == 0) s.mine.best = 0, s.mine.least = kAny, s.mine.bound = 0, s.list_n = 0;
    __syncthreads();
    {
        const uint32_t t = __reduce_max_sync(0xffffffffu, top), b = __reduce_min_sync(0xffffffffu, bottom);
        if (lane == 0) atomicMax(&s.mine.best, t), atomicMin(&s.mine.least, b);
    }
    const bool greedy = !(row.t > 0.0), few = !greedy && row.k > 0 && row.k <= kFewTokens;
    if (few) {
        // the largest bound that k of the threads' largest logits reach: at least k tokens reach it, too
        uint32_t low = 0, high = kAny;
        for (int i = 0; i < 32 && low < high; ++i) {
            const uint32_t middle = low + (high - low) / 2 + 1;
            if (__syncthreads_count(top >= middle) >= row.k) low = middle;
            else high = middle - 1;
        }
        if (tid == 0) s.mine.bound = low;
    }
    cluster_sync(size);
    uint32_t best = 0, least = kAny, bound = 0;
    for (uint32_t r = 0; r < size; ++r) {
        const Exchange *x = size > 1 ? remote(&s.mine, r) : &s.mine;
        best = max(best, x->best), least = min(least, x->least), bound = max(bound, x->bound);
    }
    if (best < kLowestKey) {                                 // nothing to draw from
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
        for (uint32_t g = g0 + tid; g < g1 && index == kAny; g += kThreads) {
            uint32_t key[8];
            tokens.keys(g, key);
#pragma unroll
            for (int j = 7; j >= 0; --j)
                if (key[j] == best) index = g * 8 - tokens.lead + j;
        }
        if (rank == 0 && tid == 0) s.found = kAny;
        cluster_sync(size);
        index = __reduce_min_sync(0xffffffffu, index);
        if (lane == 0 && index != kAny) atomicMin(&head.found, index);
        cluster_sync(size);
        if (rank == 0 && tid == 0) a.out[at] = s.found;
        return;
    }
    const uint32_t lowest = best == kInfKey ? best : kLowestKey;        // beside a +inf nothing else is drawn
    const int bits = 32 - __clz(a.vocab);                               // vocab < 2^bits
    const Weigher weigh = {(double)logit_of(best), fmin(1.0 / row.t, 1e300), ldexp(1.0, min(63 - bits, 50))};

    auto list_token = [&](uint32_t key, uint32_t index) {
        const uint32_t n = atomicAdd(&head.list_n, 1u);
        if (n < (uint32_t)kList) head.list[n] = listed(key, index);
    };
    if (few) {
        bound = max(bound, lowest);
        for (uint32_t g = g0 + tid; g < g1; g += kThreads) {
            uint32_t key[8];
            tokens.keys(g, key);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (key[j] >= bound) list_token(key[j], g * 8 - tokens.lead + j);
        }
        cluster_sync(size);
        if (rank != 0) return;
        if (s.list_n <= (uint32_t)kList) draw_from_list((int)s.list_n, row, 0, best, weigh, s, a.out + at);
        else sample_slowly(tokens, row, best, lowest, weigh, s, a.out + at);
        return;
    }

    uint32_t kept_key = lowest, kept_index = kAny;                      // the filters' border so far
    const bool by_rank = row.k > 0, by_mass = row.p < 1.0;
    if (by_rank || by_mass) {
        // tokens per interval
        const float peak = logit_of(best), range = fminf(peak - logit_of(max(least, lowest)), 31.2f * (float)fmin(row.t, 1e37));
        const float scale = range > 0.0f ? fminf((float)kBins / range, 1e30f) : 0.0f;
        auto bin_of = [&](uint32_t key) {
            return key == best ? 0 : (int)fminf((peak - logit_of(key)) * scale, (float)(kBins - 1));
        };
        for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0;
        __syncthreads();
        for (uint32_t g = g0 + tid; g < g1; g += kThreads) {
            uint32_t key[8];
            tokens.keys(g, key);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (key[j] >= lowest) atomicAdd(&s.count[bin_of(key[j])], 1u);
        }
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
        if (tid == 0) s.bin_k = kBins - 1, s.above_k = 0, s.found = kBins - 1;
        u64 mine = 0, whole;
        for (int j = 0; j < kEach; ++j) mine += count[tid * kEach + j];
        u64 ahead = block_scan(mine, s.partial, &whole);
        const u64 limit = by_rank ? min((u64)row.k, whole) : whole;
        double mass = 0.0, step = scale > 0.0f ? -1.0 / scale * weigh.inverse : 0.0;
        {
            u64 n = ahead;
            for (int j = 0; j < kEach; ++j) {
                const int bin = tid * kEach + j;
                const u64 c = count[bin];
                if (n < limit && n + c >= limit) s.bin_k = bin, s.above_k = (uint32_t)n;
                if (by_mass && c && n < limit) mass += (double)min(c, limit - n) * exp(step * (bin + 0.5));
                n += c;
            }
        }
        if (by_mass) {
            double all, run = block_scan(mass, s.partial_real, &all);
            const double want = fmax(row.p, 0.0) * all;
            u64 n = ahead;
            for (int j = 0; j < kEach; ++j) {
                const int bin = tid * kEach + j;
                const u64 c = count[bin];
                if (c && n < limit) {
                    const double m = (double)min(c, limit - n) * exp(step * (bin + 0.5));
                    if (run < want && run + m >= want) s.found = (uint32_t)bin;
                    run += m;
                }
                n += c;
            }
        }
        if (tid == 0) s.verdict.fallback = 0;
        __syncthreads();
        if (by_rank) {
            const int bin = s.bin_k;
            // what top-k keeps, as a whole or the interval of its border
            const bool all = s.above_k + count[bin] <= (uint32_t)kList;
            for (uint32_t g = g0 + tid; g < g1; g += kThreads) {
                uint32_t key[8];
                tokens.keys(g, key);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (key[j] >= lowest) {
                        const int b = bin_of(key[j]);
                        if (b == bin || (all && b < bin)) list_token(key[j], g * 8 - tokens.lead + j);
                    }
            }
            cluster_sync(size);
            if (rank == 0) {
                if (s.list_n > (uint32_t)kList) {
                    if (tid == 0) s.verdict.fallback = 1;
                } else if (all) {
                    draw_from_list((int)s.list_n, row, 0, best, weigh, s, a.out + at);
                    if (tid == 0) s.verdict.fallback = 2;
                } else {
                    sort_list(s.list, (int)s.list_n);
                    if (tid == 0) {
                        const u64 last = s.list[min(limit, whole) - s.above_k - 1];
                        s.verdict.key = listed_key(last), s.verdict.index = listed_index(last);
                    }
                }
                __syncthreads();
                if (tid == 0) s.list_n = 0;
            }
            cluster_sync(size);
            const Verdict v = head.verdict;
            if (v.fallback) {
                cluster_sync(size);
                if (v.fallback == 1 && rank == 0) sample_slowly(tokens, row, best, lowest, weigh, s, a.out + at);
                return;
            }
            kept_key = v.key, kept_index = v.index;
        }
        if (by_mass) {
            // as many intervals around the likely border as the list has room for, up to four on either side
            if (tid == 0) {
                int low = (int)s.found, high = low;
                uint32_t n = count[low];
                for (int i = 0; i < 4; ++i) {
                    if (low > 0 && n + count[low - 1] <= (uint32_t)kList) n += count[--low];
                    if (high < kBins - 1 && n + count[high + 1] <= (uint32_t)kList) n += count[++high];
                }
                s.bin_low = low, s.bin_high = high;
            }
            __syncthreads();
        }
        // one pass: mass of what top-k keeps, mass above the intervals, sums of blocks of the latter
        if (by_mass) {
            const int low = s.bin_low, high = s.bin_high;
            u64 mass_all = 0, mass_above = 0;
            for (uint32_t block = warp; block < blocks; block += kWarps) {
                u64 sum = 0;
                for (int x = 0; x < 1 << wide; ++x) {
                    const uint32_t g = g0 + block * block_groups + x * 32 + lane;
                    if (g >= g1) continue;
                    uint32_t key[8];
                    tokens.keys(g, key);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t index = g * 8 - tokens.lead + j;
                        if (key[j] < kept_key || (key[j] == kept_key && index > kept_index)) continue;
                        const int b = bin_of(key[j]);
                        const double real = weigh.real(key[j]);
                        const u64 w = __double2ull_rn(real * weigh.unit);
                        mass_all += w;
                        if (b < low) {
                            mass_above += w;
                            if (!(row.low > 0.0 && key[j] != best && real < row.low)) sum += w;
                        } else if (b <= high) {
                            list_token(key[j], index);
                        }
                    }
                }
#pragma unroll
                for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                if (lane == 0) s.blocks[block] = sum;
            }
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
                const int n = (int)min(s.list_n, (uint32_t)kList);
                sort_list(s.list, n);
                const u64 sum = scan_list(s.list, n, s.weight, s.partial, listed_key, weigh);
                if (s.list_n > (uint32_t)kList || mass_above >= want || mass_above + sum < want) {
                    if (tid == 0) s.verdict.fallback = 1;
                } else {
                    for (int i = tid; i < n; i += kThreads) {
                        const u64 before = mass_above + (i ? s.weight[i - 1] : 0), after = mass_above + s.weight[i];
                        if (before >= want) continue;
                        const uint32_t key = listed_key(s.list[i]), index = listed_index(s.list[i]);
                        if (after >= want) s.verdict.key = key, s.verdict.index = index;
                        if (row.low > 0.0 && key != best && weigh.real(key) < row.low) continue;
                        const uint32_t block = (index + tokens.lead) / 8 / block_groups, owner = block / my_blocks;
                        atomicAdd(&(size > 1 ? remote(&s, owner) : &s)->blocks[block - owner * my_blocks], after - before);
                    }
                }
            }
            cluster_sync(size);
            const Verdict v = head.verdict;
            if (v.fallback) {
                cluster_sync(size);
                if (rank == 0) sample_slowly(tokens, row, best, lowest, weigh, s, a.out + at);
                return;
            }
            kept_key = v.key, kept_index = v.index;
        }
    }
    if (!by_mass) {
        for (uint32_t block = warp; block < blocks; block += kWarps) {
            u64 sum = 0;
            for (int x = 0; x < 1 << wide; ++x) {
                const uint32_t g = g0 + block * block_groups + x * 32 + lane;
                if (g >= g1) continue;
                uint32_t key[8];
                tokens.keys(g, key);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (key[j] < kept_key || (key[j] == kept_key && g * 8 - tokens.lead + j > kept_index)) continue;
                    const double real = weigh.real(key[j]);
                    if (row.low > 0.0 && key[j] != best && real < row.low) continue;
                    sum += __double2ull_rn(real * weigh.unit);
                }
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane == 0) s.blocks[block] = sum;
        }
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
                uint32_t key[8] = {};
                if (g < g1) tokens.keys(g, key);
                u64 w[8];
                sum = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = 0;
                    if (key[j] >= kept_key && !(key[j] == kept_key && g * 8 - tokens.lead + j > kept_index)) {
                        const double real = weigh.real(key[j]);
                        if (!(row.low > 0.0 && key[j] != best && real < row.low)) w[j] = __double2ull_rn(real * weigh.unit);
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
        const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared));
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
