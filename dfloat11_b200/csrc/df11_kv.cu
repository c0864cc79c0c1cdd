// The 8-bit key/value cache of a generation step: rows quantised as they are written, read back,
// and attended to in their 8-bit form.
//
// A row x (one token of one head, d numbers) of largest magnitude a is stored as a scale and d
// codes: int8, scale = a / 127 and code = rint(x * 127 / a); e4m3, scale = a / 448 and
// code = e4m3(x * 448 / a); ties to even.  x * 127 and x * 448 are exact in fp32 (x has 8 or 11
// significant bits), and the correctly rounded fp32 quotient lies on a border between two codes only
// if the exact quotient does: numerator and denominator are integers of at most 18 and 11 bits times
// powers of two, so a quotient that is not on a border is at least 2^-16 of itself away from it, far
// more than half a step of fp32.  So the code is the one of the exact quotient, and a plain 64-bit
// computation gives the same.
#include <cuda_fp8.h>

#include "df11_launch.h"

namespace {

__device__ __forceinline__ float top_of(int format) { return format == DF11_KV_INT8 ? 127.0f : 448.0f; }

__device__ __forceinline__ float code_value(uint8_t code, int format)
{
    if (format == DF11_KV_INT8) return (float)(int8_t)code;
    const __half_raw h = __nv_cvt_fp8_to_halfraw(code, __NV_E4M3);
    return __half2float(__half(h));
}

__device__ __forceinline__ float warp_max(float x)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

__device__ __forceinline__ float warp_sum(float x)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

// A length as the user's program may have it; what is beyond any cache must not overflow below.
__device__ __forceinline__ int64_t clamped_length(int64_t n) { return n < 0 ? 0 : n > (1ll << 40) ? 1ll << 40 : n; }

struct Strides {
    int64_t b, h, t;
};

// One warp per row of k or v.
template <typename T>
__global__ void __launch_bounds__(128) kv_append_kernel(const T *k, const T *v, Strides ks, Strides vs, uint8_t *k_codes,
                                                        float *k_scales, uint8_t *v_codes, float *v_scales,
                                                        const int64_t *positions, int per_sequence, int64_t rows,
                                                        int heads, int64_t tokens, int dim, int64_t max_slots, int format,
                                                        int *status)
{
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= 2 * rows) return;
    const bool value = row >= rows;
    const int64_t r = value ? row - rows : row;
    const int64_t t = r % tokens, h = r / tokens % heads, b = r / tokens / heads;
    const Strides s = value ? vs : ks;
    const T *x = (value ? v : k) + b * s.b + h * s.h + t * s.t;
    const int64_t position = positions[per_sequence ? b : 0];
    if (position < -t || position >= max_slots - t) {
        if (lane == 0 && status) atomicOr(status, DF11_STATUS_BAD_POSITIONS);
        return;
    }
    const int64_t slot = position + t;
    float a = 0.0f;
    bool finite = true;
    for (int i = lane; i < dim; i += 32) {
        const float m = fabsf(df11_to_float(x[i]));
        finite &= m <= 3.402823466e38f;
        a = fmaxf(a, m);
    }
    a = warp_max(a);
    finite = __all_sync(0xffffffffu, finite);
    const float top = top_of(format);
    const int64_t cell = (b * heads + h) * max_slots + slot;
    uint8_t *codes = (value ? v_codes : k_codes) + cell * dim;
    // a power of two that keeps x * top away from overflow and x away from the subnormals
    const float shift = a > 1e30f ? 0x1p-40f : a < 1e-30f ? 0x1p40f : 1.0f;
    for (int i = lane; i < dim; i += 32) {
        float q = 0.0f;
        if (finite && a > 0.0f) q = __fdiv_rn(df11_to_float(x[i]) * shift * top, a * shift);
        codes[i] = format == DF11_KV_INT8 ? (uint8_t)(int8_t)__float2int_rn(q)
                                          : (uint8_t)__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
    }
    if (lane == 0) (value ? v_scales : k_scales)[cell] = finite ? __fdiv_rn(a, top) : __int_as_float(0x7fc00000);
}

// One warp per row of the result.
template <typename T>
__global__ void __launch_bounds__(128) kv_read_kernel(const uint8_t *k_codes, const float *k_scales, const uint8_t *v_codes,
                                                      const float *v_scales, T *k_out, T *v_out, int64_t rows,
                                                      int64_t max_slots, int dim, int64_t first, int64_t n, int format)
{
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= 2 * rows) return;
    const bool value = row >= rows;
    const int64_t r = value ? row - rows : row;
    const int64_t cell = r / n * max_slots + first + r % n;
    const uint8_t *codes = (value ? v_codes : k_codes) + cell * dim;
    const float scale = (value ? v_scales : k_scales)[cell];
    T *out = (value ? v_out : k_out) + r * dim;
    for (int i = lane; i < dim; i += 32) out[i] = df11_from_float<T>(code_value(codes[i], format) * scale);
}

// One CTA of four warps per query row; a warp takes every fourth slot, one pass with a running
// maximum and sum, and the warps' results are joined at the end.
template <typename T>
__global__ void __launch_bounds__(128) kv_attention_kernel(const T *q, Strides qs, const uint8_t *k_codes,
                                                           const float *k_scales, const uint8_t *v_codes,
                                                           const float *v_scales, const int64_t *lengths, int length_per,
                                                           const int64_t *first, int first_per, T *out, int heads,
                                                           int kv_heads, int64_t queries, int dim, int64_t max_slots,
                                                           int window, float scale, int format)
{
    __shared__ float part_o[4][DF11_KV_MAX_HEAD_DIM], part_m[4], part_l[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = blockIdx.x % queries, h = blockIdx.x / queries % heads, b = blockIdx.x / queries / heads;
    const int64_t cell0 = (b * kv_heads + h / (heads / kv_heads)) * max_slots;
    const int64_t place = clamped_length(lengths[length_per ? b : 0]) - queries + i;
    int64_t low = first ? first[first_per ? b : 0] : 0;
    if (window > 0 && place - window + 1 > low) low = place - window + 1;
    if (low < 0) low = 0;
    const int64_t high = place < max_slots ? place : max_slots - 1;
    constexpr int kPer = DF11_KV_MAX_HEAD_DIM / 32;
    float x[kPer], o[kPer] = {};
    for (int j = 0; j < kPer; ++j)
        x[j] = lane + 32 * j < dim ? df11_to_float(q[b * qs.b + h * qs.h + i * qs.t + lane + 32 * j]) * scale : 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int64_t t = low + warp; t <= high; t += 4) {
        const uint8_t *kc = k_codes + (cell0 + t) * dim, *vc = v_codes + (cell0 + t) * dim;
        float s = 0.0f;
        for (int j = 0; j < kPer; ++j)
            if (lane + 32 * j < dim) s += x[j] * code_value(kc[lane + 32 * j], format);
        s = warp_sum(s) * k_scales[cell0 + t];
        const float peak = fmaxf(m, s), base = peak == -INFINITY ? 0.0f : peak;
        const float old = expf(m - base), p = expf(s - base);
        l = l * old + p;
        const float w = p * v_scales[cell0 + t];
        for (int j = 0; j < kPer; ++j) {
            o[j] *= old;
            if (lane + 32 * j < dim) o[j] += w * code_value(vc[lane + 32 * j], format);
        }
        m = peak;
    }
    for (int j = 0; j < kPer; ++j) part_o[warp][lane + 32 * j] = o[j];
    if (lane == 0) part_m[warp] = m, part_l[warp] = l;
    __syncthreads();
    float peak = fmaxf(fmaxf(part_m[0], part_m[1]), fmaxf(part_m[2], part_m[3]));
    if (peak == -INFINITY) peak = 0.0f;
    float total = 0.0f, w[4];
    for (int k = 0; k < 4; ++k) {
        w[k] = expf(part_m[k] - peak);
        total += w[k] * part_l[k];
    }
    T *row = out + ((b * queries + i) * heads + h) * dim;
    for (int c = threadIdx.x; c < dim; c += 128) {
        float sum = 0.0f;
        for (int k = 0; k < 4; ++k) sum += w[k] * part_o[k][c];
        row[c] = df11_from_float<T>(total == 0.0f ? 0.0f : sum / total);
    }
}

int check_cache(const void *kc, const void *ks, const void *vc, const void *vs, int64_t batch, int32_t kv_heads,
                int64_t max_slots, int32_t head_dim, int32_t element_type, int32_t format)
{
    if (!kc || !ks || !vc || !vs) return df11_fail(DF11_ERR_BADARG, "null cache pointer");
    if (((uintptr_t)kc | (uintptr_t)vc) & 15) return df11_fail(DF11_ERR_BADARG, "the codes must be 16-byte aligned");
    if (((uintptr_t)ks | (uintptr_t)vs) & 3) return df11_fail(DF11_ERR_BADARG, "the scales must be 4-byte aligned");
    if (element_type != DF11_TYPE_BF16 && element_type != DF11_TYPE_FP16)
        return df11_fail(DF11_ERR_BADARG, "element type %d: bf16 and fp16 are supported", element_type);
    if (format != DF11_KV_INT8 && format != DF11_KV_E4M3) return df11_fail(DF11_ERR_BADARG, "unknown cache format %d", format);
    if (batch < 0 || batch > 0x7FFFFFFF || kv_heads < 1 || max_slots < 1 || max_slots > 0x7FFFFFFF)
        return df11_fail(DF11_ERR_BADARG, "batch, kv_heads or max_slots out of range");
    if (head_dim < 16 || head_dim > DF11_KV_MAX_HEAD_DIM || head_dim % 16)
        return df11_fail(DF11_ERR_BADARG, "head_dim %d: multiples of 16 up to %d are supported", head_dim, DF11_KV_MAX_HEAD_DIM);
    if ((double)batch * kv_heads * (double)max_slots * head_dim > 4e18)
        return df11_fail(DF11_ERR_BADARG, "the cache is larger than any memory");
    return DF11_OK;
}

int launched()
{
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return df11_fail(DF11_ERR_CUDA, "kernel launch failed: %s", cudaGetErrorString(e));
    return DF11_OK;
}

}  // namespace

extern "C" int df11_kv_append(const void *k, const void *v, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t,
                              int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_t, void *k_codes, void *k_scales,
                              void *v_codes, void *v_scales, const void *positions, int64_t n_positions, int64_t batch,
                              int32_t kv_heads, int64_t tokens, int32_t head_dim, int64_t max_slots,
                              int32_t element_type, int32_t format, void *status, int32_t device, void *stream)
{
    const int rc = check_cache(k_codes, k_scales, v_codes, v_scales, batch, kv_heads, max_slots, head_dim, element_type, format);
    if (rc != DF11_OK) return rc;
    if (!k || !v || !positions) return df11_fail(DF11_ERR_BADARG, "null pointer");
    if (((uintptr_t)k | (uintptr_t)v) & 1 || ((uintptr_t)positions & 7)) return df11_fail(DF11_ERR_BADARG, "misaligned pointer");
    if (n_positions != 1 && n_positions != batch) return df11_fail(DF11_ERR_BADARG, "positions must have 1 or batch entries");
    if (tokens < 0 || tokens > 0x7FFFFFFF) return df11_fail(DF11_ERR_BADARG, "bad token count");
    const double all = 2.0 * (double)batch * kv_heads * (double)tokens;
    if (all > 8e9) return df11_fail(DF11_ERR_BADARG, "too many rows for one call");
    if (all == 0) return DF11_OK;
    const int64_t rows = batch * kv_heads * tokens;
    Df11DeviceScope scope(device);
    if (!scope.ok) return df11_fail(DF11_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const Strides ks = {k_stride_b, k_stride_h, k_stride_t}, vs = {v_stride_b, v_stride_h, v_stride_t};
    const unsigned grid = (unsigned)((2 * rows + 3) / 4);
    if (element_type == DF11_TYPE_BF16)
        kv_append_kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(
            (const __nv_bfloat16 *)k, (const __nv_bfloat16 *)v, ks, vs, (uint8_t *)k_codes, (float *)k_scales, (uint8_t *)v_codes,
            (float *)v_scales, (const int64_t *)positions, n_positions > 1, rows, kv_heads, tokens, head_dim, max_slots, format,
            (int *)status);
    else
        kv_append_kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(
            (const __half *)k, (const __half *)v, ks, vs, (uint8_t *)k_codes, (float *)k_scales, (uint8_t *)v_codes,
            (float *)v_scales, (const int64_t *)positions, n_positions > 1, rows, kv_heads, tokens, head_dim, max_slots, format,
            (int *)status);
    return launched();
}

extern "C" int df11_kv_read(const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales, void *k_out,
                            void *v_out, int64_t batch, int32_t kv_heads, int64_t max_slots, int32_t head_dim,
                            int64_t first_slot, int64_t n_slots, int32_t element_type, int32_t format, int32_t device,
                            void *stream)
{
    const int rc = check_cache(k_codes, k_scales, v_codes, v_scales, batch, kv_heads, max_slots, head_dim, element_type, format);
    if (rc != DF11_OK) return rc;
    if (!k_out || !v_out) return df11_fail(DF11_ERR_BADARG, "null pointer");
    if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return df11_fail(DF11_ERR_BADARG, "the results must be 16-byte aligned");
    if (first_slot < 0 || n_slots < 0 || first_slot > max_slots || n_slots > max_slots - first_slot)
        return df11_fail(DF11_ERR_BADARG, "slots %lld + %lld of %lld", (long long)first_slot, (long long)n_slots, (long long)max_slots);
    const double all = 2.0 * (double)batch * kv_heads * (double)n_slots;
    if (all > 8e9) return df11_fail(DF11_ERR_BADARG, "too many rows for one call");
    if (all == 0) return DF11_OK;
    const int64_t rows = batch * kv_heads * n_slots;
    Df11DeviceScope scope(device);
    if (!scope.ok) return df11_fail(DF11_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const unsigned grid = (unsigned)((2 * rows + 3) / 4);
    if (element_type == DF11_TYPE_BF16)
        kv_read_kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(
            (const uint8_t *)k_codes, (const float *)k_scales, (const uint8_t *)v_codes, (const float *)v_scales,
            (__nv_bfloat16 *)k_out, (__nv_bfloat16 *)v_out, rows, max_slots, head_dim, first_slot, n_slots, format);
    else
        kv_read_kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(
            (const uint8_t *)k_codes, (const float *)k_scales, (const uint8_t *)v_codes, (const float *)v_scales,
            (__half *)k_out, (__half *)v_out, rows, max_slots, head_dim, first_slot, n_slots, format);
    return launched();
}

extern "C" int64_t df11_kv_attention_workspace_bytes(int64_t batch, int32_t heads, int32_t kv_heads, int64_t queries,
                                                     int32_t head_dim, int64_t max_slots, int32_t window)
{
    (void)batch, (void)heads, (void)kv_heads, (void)queries, (void)head_dim, (void)max_slots, (void)window;
    return 0;
}

extern "C" int df11_kv_attention(const void *q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
                                 const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales,
                                 const void *lengths, int64_t n_lengths, const void *first, int64_t n_first, void *out,
                                 void *workspace, int64_t workspace_bytes, int64_t batch, int32_t heads, int32_t kv_heads,
                                 int64_t queries, int32_t head_dim, int64_t max_slots, int32_t window, float scale,
                                 int32_t element_type, int32_t format, int32_t device, void *stream)
{
    const int rc = check_cache(k_codes, k_scales, v_codes, v_scales, batch, kv_heads, max_slots, head_dim, element_type, format);
    if (rc != DF11_OK) return rc;
    if (!q || !lengths || !out) return df11_fail(DF11_ERR_BADARG, "null pointer");
    if (((uintptr_t)q & 1) || ((uintptr_t)out & 15) || (((uintptr_t)lengths | (uintptr_t)first) & 7))
        return df11_fail(DF11_ERR_BADARG, "misaligned pointer");
    if (heads < 1 || heads % kv_heads) return df11_fail(DF11_ERR_BADARG, "%d heads on %d key/value heads", heads, kv_heads);
    if (n_lengths != 1 && n_lengths != batch) return df11_fail(DF11_ERR_BADARG, "lengths must have 1 or batch entries");
    if (first && n_first != 1 && n_first != batch) return df11_fail(DF11_ERR_BADARG, "first must have 1 or batch entries");
    if (queries < 0 || queries > 0x7FFFFFFF || window < 0) return df11_fail(DF11_ERR_BADARG, "negative query count or window");
    const double rows = (double)batch * heads * (double)queries;
    if (rows > 2e9) return df11_fail(DF11_ERR_BADARG, "too many query rows for one call");
    const int64_t need = df11_kv_attention_workspace_bytes(batch, heads, kv_heads, queries, head_dim, max_slots, window);
    if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return df11_fail(DF11_ERR_NOSPACE, "the workspace must have %lld bytes, 16-byte aligned", (long long)need);
    if (rows == 0) return DF11_OK;
    Df11DeviceScope scope(device);
    if (!scope.ok) return df11_fail(DF11_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const Strides qs = {q_stride_b, q_stride_h, q_stride_t};
    if (element_type == DF11_TYPE_BF16)
        kv_attention_kernel<<<(unsigned)rows, 128, 0, (cudaStream_t)stream>>>(
            (const __nv_bfloat16 *)q, qs, (const uint8_t *)k_codes, (const float *)k_scales, (const uint8_t *)v_codes,
            (const float *)v_scales, (const int64_t *)lengths, n_lengths > 1, (const int64_t *)first, n_first > 1,
            (__nv_bfloat16 *)out, heads, kv_heads, queries, head_dim, max_slots, window, scale, format);
    else
        kv_attention_kernel<<<(unsigned)rows, 128, 0, (cudaStream_t)stream>>>(
            (const __half *)q, qs, (const uint8_t *)k_codes, (const float *)k_scales, (const uint8_t *)v_codes,
            (const float *)v_scales, (const int64_t *)lengths, n_lengths > 1, (const int64_t *)first, n_first > 1,
            (__half *)out, heads, kv_heads, queries, head_dim, max_slots, window, scale, format);
    return launched();
}
