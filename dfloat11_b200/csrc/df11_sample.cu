// One token per row of logits, drawn with temperature, top-k, top-p and min-p from given random
// numbers.
//
// With z the logits, c the largest and T the temperature, a token's weight is exp((z - c) / T), in
// (0, 1].  A sum over 10^5 tokens decides at which token a border (u * mass, top_p * mass) is
// crossed; summed in fp32 it is off by some 1e-7 of the mass, and with 10^5 borders about one row in
// a hundred would be decided wrongly, and differently in another order.  So weights are computed in fp64
// and held as 64-bit integers, weight * 2^S with S such that V of them fit: sums of integers are
// exact, the same in every order, and S >= 44 for V < 2^18 leaves each border off by 2^-45 at most.
//
// A filter keeps all tokens above some logit and the first few, by index, of those equal to it.
// Both filters that need an order find that logit digit by digit: the tokens (top-k) or the masses
// (top-p) of the 256 values of a digit are added up, the digit in which the border lies is fixed,
// and the next digit is looked at among the tokens that share it.
#include <math.h>

#include "df11_launch.h"

namespace {

constexpr int kThreads = 1024;
constexpr uint32_t kLowestKey = 0x00800000u;  // key of the lowest finite float; NaN and -inf lie below

// A number that orders like the logit (-0 like 0); 0 for a NaN.
__device__ __forceinline__ uint32_t key_of(float z)
{
    if (isnan(z)) return 0u;
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

struct Weigher {
    double peak, inverse, unit;
    __device__ __forceinline__ unsigned long long operator()(uint32_t key) const
    {
        const double z = (double)logit_of(key);
        const double d = z == peak ? 0.0 : z - peak;
        if (d == -INFINITY) return 0;           // beside a +inf; an infinite temperature must not bring it back
        return __double2ull_rn(exp(d * inverse) * unit);
    }
};

struct Filter {          // keeps keys above `key`, and of those equal to it the first `ties` by index
    uint32_t key;
    uint32_t ties;
};

template <typename V> struct Shared {
    V digits[256];
    V partial[kThreads / 32];
    V total;
    uint32_t key;
    V above;
};

template <typename V> __device__ V block_sum(V x, V *partial)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) partial[threadIdx.x >> 5] = x;
    __syncthreads();
    V all = 0;
    for (int w = 0; w < kThreads / 32; ++w) all += partial[w];
    return all;
}

template <typename T> __device__ __forceinline__ uint32_t key_at(const T *row, int64_t i) { return key_of(df11_to_float(row[i])); }

// How many tokens with this key lie before `end`.
template <typename T> __device__ uint32_t ties_before(const T *row, int64_t end, uint32_t key, unsigned long long *partial)
{
    unsigned long long n = 0;
    for (int64_t i = threadIdx.x; i < end; i += kThreads) n += key_at(row, i) == key;
    return (uint32_t)block_sum(n, partial);
}

// The key in which the running measure (from the largest key down) reaches `want`, and the measure
// above it.  measure(key) is 1 or a weight; keys outside `within` measure nothing.
template <typename T, typename M>
__device__ void descend(const T *row, int64_t vocab, unsigned long long want, M measure, unsigned long long *digits,
                        uint32_t *found, unsigned long long *above)
{
    __shared__ uint32_t s_key;
    __shared__ unsigned long long s_above;
    uint32_t prefix = 0;
    unsigned long long over = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kThreads) digits[i] = 0;
        __syncthreads();
        for (int64_t i = threadIdx.x; i < vocab; i += kThreads) {
            const uint32_t key = key_at(row, i);
            if (key >= kLowestKey && (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)))
                atomicAdd(&digits[(key >> shift) & 255u], measure(key));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned long long run = over;
            int d = 255;
            while (d > 0 && run + digits[d] < want) run += digits[d--];
            s_key = prefix | (uint32_t)d << shift;
            s_above = run;
        }
        __syncthreads();
        prefix = s_key;
        over = s_above;
        __syncthreads();
    }
    *found = prefix;
    *above = over;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const T *logits, int64_t stride, int64_t vocab, const float *uniform,
                                                          const float *temperature, double temperature_value, const int *top_k,
                                                          int top_k_value, const float *top_p, double top_p_value,
                                                          const float *min_p, double min_p_value, int64_t *out, int *status)
{
    __shared__ unsigned long long digits[256], partial[kThreads / 32], sums[kThreads];
    __shared__ uint32_t s_best;
    __shared__ unsigned long long s_first;
    const int tid = threadIdx.x;
    const T *row = logits + (int64_t)blockIdx.x * stride;
    const double t = temperature ? (double)temperature[blockIdx.x] : temperature_value;
    const long long k = top_k ? top_k[blockIdx.x] : top_k_value;
    const double p = top_p ? (double)top_p[blockIdx.x] : top_p_value;
    const double low = min_p ? (double)min_p[blockIdx.x] : min_p_value;
    const double u = (double)uniform[blockIdx.x];

    // the largest logit
    if (tid == 0) s_best = 0, s_first = ~0ull;
    __syncthreads();
    uint32_t best = 0;
    for (int64_t i = tid; i < vocab; i += kThreads) best = max(best, key_at(row, i));
    atomicMax(&s_best, best);
    __syncthreads();
    best = s_best;
    if (best < kLowestKey) {
        if (tid == 0) {
            out[blockIdx.x] = 0;
            if (status) atomicOr(status, DF11_STATUS_EMPTY_ROW);
        }
        return;
    }
    if (!(t > 0.0)) {
        for (int64_t i = tid; i < vocab; i += kThreads)
            if (key_at(row, i) == best) {
                atomicMin(&s_first, (unsigned long long)i);
                break;
            }
        __syncthreads();
        if (tid == 0) out[blockIdx.x] = (int64_t)s_first;
        return;
    }
    const int bits = 64 - __clzll(vocab);          // vocab < 2^bits
    const Weigher weigh = {(double)logit_of(best), fmin(1.0 / t, 1e300), ldexp(1.0, min(63 - bits, 50))};

    // the filters: a token is kept if all three keep it
    Filter kept = {kLowestKey, 0xFFFFFFFFu};
    unsigned long long above, total;
    if (k > 0 && k < vocab) {
        descend(row, vocab, (unsigned long long)k, [](uint32_t) { return 1ull; }, digits, &kept.key, &above);
        kept.ties = (uint32_t)min((unsigned long long)k - min(above, (unsigned long long)k), 0xFFFFFFFFull);
        if (kept.key < kLowestKey) kept.key = kLowestKey;
    }
    if (p < 1.0) {
        unsigned long long mass = 0, equal = 0;
        for (int64_t i = tid; i < vocab; i += kThreads) {
            const uint32_t key = key_at(row, i);
            if (key > kept.key) mass += weigh(key);
            equal += key == kept.key;
        }
        mass = block_sum(mass, partial);
        equal = block_sum(equal, partial);
        const unsigned long long each = weigh(kept.key);
        total = mass + min(equal, (unsigned long long)kept.ties) * each;
        const unsigned long long want = max((unsigned long long)ceil(fmax(p, 0.0) * (double)total), 1ull);
        if (want <= mass) {                       // the border lies above the ties of top-k
            uint32_t key;
            const Filter before = kept;
            descend(row, vocab, want, [&](uint32_t x) { return x > before.key ? weigh(x) : 0ull; }, digits, &key, &above);
            const unsigned long long w = weigh(key);
            kept.key = key;
            kept.ties = (uint32_t)((want - above + w - 1) / w);
        } else if (each > 0) {
            kept.ties = (uint32_t)min((unsigned long long)kept.ties, (want - mass + each - 1) / each);
        }
    }
    const double floor_weight = fmin(low, 1.0);

    // the draw: every thread has a stretch of the vocabulary, in order
    const int64_t per = (vocab + kThreads - 1) / kThreads, begin = min(per * tid, vocab), end = min(begin + per, vocab);
    unsigned long long equal = 0;
    for (int64_t i = begin; i < end; ++i) equal += key_at(row, i) == kept.key;
    sums[tid] = equal;
    __syncthreads();
    unsigned long long seen = 0;
    for (int j = 0; j < tid; ++j) seen += sums[j];
    auto weight_at = [&](int64_t i, unsigned long long &ties) -> unsigned long long {
        const uint32_t key = key_at(row, i);
        if (key < kept.key || key < kLowestKey) return 0;
        if (key == kept.key && ties++ >= kept.ties) return 0;
        const double d = (double)logit_of(key) - weigh.peak;
        if (low > 0.0 && key != best && exp(d * weigh.inverse) < floor_weight) return 0;
        return weigh(key);
    };
    unsigned long long mine = 0, ties = seen;
    for (int64_t i = begin; i < end; ++i) mine += weight_at(i, ties);
    total = block_sum(mine, partial);
    sums[tid] = mine;
    __syncthreads();
    unsigned long long run = 0;
    for (int j = 0; j < tid; ++j) run += sums[j];
    const double border = u > 0.0 ? u * (double)total : 0.0;
    const unsigned long long want = border >= (double)total ? total - 1 : min((unsigned long long)border, total - 1);
    if (run <= want && want < run + mine) {
        ties = seen;
        for (int64_t i = begin; i < end; ++i) {
            run += weight_at(i, ties);
            if (run > want) {
                out[blockIdx.x] = i;
                break;
            }
        }
    }
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
    if (rows < 0 || rows > 0x7FFFFFFF || vocab < 1 || vocab > 0x7FFFFFFF)
        return df11_fail(DF11_ERR_BADARG, "rows or vocab out of range");
    if (row_stride < 0) return df11_fail(DF11_ERR_BADARG, "negative row stride");
    const uintptr_t unit = element_type == DF11_TYPE_FP32 ? 3 : 1;
    if (((uintptr_t)logits & unit) || ((uintptr_t)out & 7) ||
        (((uintptr_t)uniform | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)status) & 3))
        return df11_fail(DF11_ERR_BADARG, "misaligned pointer");
    if (rows == 0) return DF11_OK;
    Df11DeviceScope scope(device);
    if (!scope.ok) return df11_fail(DF11_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    auto go = [&](auto *typed) {
        sample_kernel<<<(unsigned)rows, kThreads, 0, (cudaStream_t)stream>>>(
            typed, row_stride, vocab, (const float *)uniform, (const float *)temperature, temperature_value, (const int *)top_k,
            top_k_value, (const float *)top_p, top_p_value, (const float *)min_p, min_p_value, (int64_t *)out, (int *)status);
    };
    if (element_type == DF11_TYPE_BF16) go((const __nv_bfloat16 *)logits);
    else if (element_type == DF11_TYPE_FP16) go((const __half *)logits);
    else go((const float *)logits);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return df11_fail(DF11_ERR_CUDA, "kernel launch failed: %s", cudaGetErrorString(e));
    return DF11_OK;
}
