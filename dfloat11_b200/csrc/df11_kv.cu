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

// A length or a first slot as the user's program may have it; what is beyond any cache must not
// overflow in what is computed from it.
__device__ __forceinline__ int64_t clamped_length(int64_t n) { return n < 0 ? 0 : n > (1ll << 40) ? 1ll << 40 : n; }

struct Strides {
    int64_t b, h, t;
};

// Writing and reading move bytes and compute little: 3 bytes per number either way.  65536 rows of 128 keys and
// values each (403 MB): written in 79 us (5.1 TB/s; some 9 instructions per number keep it from the copy rate), read
// in 63 us (6.4 TB/s, the copy rate).  A group of LANES
// threads (a power of two) holds a row in registers, 16 numbers per thread, so that a row's maximum is a few
// shuffles and its codes leave as one 16-byte store per thread.
// 16 numbers from an address that may have any alignment of the type.
template <typename T> __device__ __forceinline__ void load16(const T *p, bool aligned, uint4 (&raw)[2])
{
    if (aligned) {
        raw[0] = __ldg(reinterpret_cast<const uint4 *>(p)), raw[1] = __ldg(reinterpret_cast<const uint4 *>(p) + 1);
    } else {
        const uint16_t *y = reinterpret_cast<const uint16_t *>(p);
        uint32_t *w = reinterpret_cast<uint32_t *>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (uint32_t)y[2 * i] | (uint32_t)y[2 * i + 1] << 16;
    }
}

struct AppendArgs {
    const void *k, *v;
    Strides ks, vs;
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    const int64_t *positions;
    int *status;
    int64_t max_slots;
    uint32_t batch, heads, tokens;
    int per_sequence, dim, aligned;
};

template <typename T> constexpr uint32_t kInfBits = 0;
template <> constexpr uint32_t kInfBits<__nv_bfloat16> = 0x7F80;
template <> constexpr uint32_t kInfBits<__half> = 0x7C00;

// The codes of x * up / over.  A product with the reciprocal is off by 2^-21 of itself at most; only where
// that could decide (one number in some thousands), or where `extreme` says that the factor does not fit a
// float, is the quotient itself computed.
template <int FMT> __device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float up, float over, float factor, bool extreme)
{
    constexpr float kMagic = 12582912.0f;       // 1.5 * 2^23: the sum's low bits are the nearest integer
    uint32_t y;
    bool close;
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = x[i] * factor;
    if (FMT == DF11_KV_INT8) {
        uint32_t n[4];
        float far = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float m = q[i] + kMagic;
            n[i] = __float_as_uint(m);
            far = fmaxf(far, fabsf(q[i] - (m - kMagic)));
        }
        y = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
        close = far > 0.4999f;                  // 127 * 2^-21 < 0.0001
    } else {
        auto pack = [&](float scale) {
            return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q[0] * scale, q[1] * scale), __NV_SATFINITE, __NV_E4M3) |
                   (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q[2] * scale, q[3] * scale), __NV_SATFINITE, __NV_E4M3) << 16;
        };
        y = pack(1.0f - 0x1p-20f);
        close = y != pack(1.0f + 0x1p-20f);
    }
    if (close || extreme) {
        y = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float exact = __fdiv_rn(x[i] * up, over);
            y |= (FMT == DF11_KV_INT8 ? (uint32_t)(__float2int_rn(exact) & 255)
                                      : (uint32_t)__nv_cvt_float_to_fp8(exact, __NV_SATFINITE, __NV_E4M3)) << (8 * i);
        }
    }
    return y;
}

// The codes and the scale of one row, of which this thread has 16 numbers.
template <int LANES, int FMT, typename T>
__device__ __forceinline__ void quantise_row(const uint4 (&raw)[2], bool store, bool lead, uint8_t *to, float *scale)
{
    // magnitudes order like their bits, a NaN above an infinity
    uint32_t bits = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) bits = __vmaxu2(bits, reinterpret_cast<const uint32_t *>(raw)[w] & 0x7FFF7FFFu);
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) bits = __vmaxu2(bits, __shfl_xor_sync(0xffffffffu, bits, d));
    if (!store) return;
    bits = max(bits & 0xFFFFu, bits >> 16);
    const bool finite = bits < kInfBits<T>, zero = bits == 0 || !finite;
    const uint16_t top_bits = (uint16_t)bits;
    const float most = FMT == DF11_KV_INT8 ? 127.0f : 448.0f, top = df11_to_float(*reinterpret_cast<const T *>(&top_bits));
    // a power of two that keeps x * most away from overflow and x away from the subnormals
    const float shift = top > 1e30f ? 0x1p-40f : top < 1e-30f ? 0x1p40f : 1.0f;
    const float over = zero ? 1.0f : top * shift, up = shift * most, factor = up * __frcp_rn(over);
    uint32_t codes[4];
    const T *const x = reinterpret_cast<const T *>(raw);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float four[4] = {df11_to_float(x[4 * w]), df11_to_float(x[4 * w + 1]), df11_to_float(x[4 * w + 2]), df11_to_float(x[4 * w + 3])};
        codes[w] = zero ? 0 : codes_of<FMT>(four, up, over, factor, shift != 1.0f);
    }
    *reinterpret_cast<uint4 *>(to) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
    if (lead) *scale = finite ? __fdiv_rn(top, most) : __int_as_float(0x7fc00000);
}

// One block: rows of one sequence (blockIdx.y, and every gridDim.y-th after it), keys and values; what
// is loaded does not wait for the position.
template <int LANES, int FMT, typename T> __global__ void __launch_bounds__(256) kv_append_kernel(AppendArgs a)
{
    constexpr int kRows = 256 / LANES;
    const uint32_t per = a.heads * a.tokens, r = blockIdx.x * kRows + threadIdx.x / LANES;
    const int part = threadIdx.x % LANES * 16;
    const bool mine = r < per && part < a.dim;
    const uint32_t within = mine ? r : 0, t = within / a.heads, h = within - t * a.heads;
    for (uint32_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
        uint4 key[2] = {}, value[2] = {};
        if (mine) {
            load16((const T *)a.k + b * a.ks.b + h * a.ks.h + t * a.ks.t + part, a.aligned, key);
            load16((const T *)a.v + b * a.vs.b + h * a.vs.h + t * a.vs.t + part, a.aligned, value);
        }
        const int64_t position = a.positions[a.per_sequence ? b : 0];
        const bool there = position >= -(int64_t)t && position < a.max_slots - (int64_t)t, store = mine && there;
        const int64_t cell = there ? ((int64_t)b * a.heads + h) * a.max_slots + position + t : 0;
        if (mine && !there && part == 0 && a.status) atomicOr(a.status, DF11_STATUS_BAD_POSITIONS);
        quantise_row<LANES, FMT, T>(key, store, part == 0, a.k_codes + cell * a.dim + part, a.k_scales + cell);
        quantise_row<LANES, FMT, T>(value, store, part == 0, a.v_codes + cell * a.dim + part, a.v_scales + cell);
    }
}

struct ReadArgs {
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    void *k_out, *v_out;
    int64_t max_slots, first;
    uint32_t units, n, chunks;          // heads of all sequences, slots read, 8-byte chunks per row
};

// A thread takes 8 codes at a time, so that a warp's stores cover consecutive bytes, kEach times for loads
// in flight; blockIdx.y is the head of a sequence, blockIdx.z keys or values.
template <int FMT, typename T> __global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a)
{
    constexpr int kEach = 4;
    const uint64_t all = (uint64_t)a.n * a.chunks, i0 = (uint64_t)blockIdx.x * (256 * kEach) + threadIdx.x;
    for (int64_t unit = blockIdx.y; unit < a.units; unit += gridDim.y) {
        const uint8_t *const codes = (blockIdx.z ? a.v_codes : a.k_codes) + (unit * a.max_slots + a.first) * a.chunks * 8;
        const float *const scales = (blockIdx.z ? a.v_scales : a.k_scales) + unit * a.max_slots + a.first;
        T *const out = (T *)(blockIdx.z ? a.v_out : a.k_out) + unit * a.n * a.chunks * 8;
        uint2 raw[kEach];
        float scale[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const uint64_t i = i0 + e * 256;
            if (i >= all) continue;
            raw[e] = __ldg(reinterpret_cast<const uint2 *>(codes) + i);
            scale[e] = __ldg(scales + (a.chunks == 16 ? i >> 4 : i / a.chunks));
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const uint64_t i = i0 + e * 256;
            if (i >= all) continue;
            const uint32_t words[2] = {raw[e].x, raw[e].y};
            __align__(16) T y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t code = words[k / 4] >> (8 * (k % 4));
                float x;
                if (FMT == DF11_KV_INT8) x = (float)(int8_t)code;
                else x = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
                y[k] = df11_from_float<T>(x * scale[e]);
            }
            reinterpret_cast<uint4 *>(out)[i] = *reinterpret_cast<const uint4 *>(y);
        }
    }
}

template <int LANES, typename T> void launch_append(const AppendArgs &a, int format, cudaStream_t stream)
{
    const dim3 grid((unsigned)(((uint64_t)a.heads * a.tokens + 256 / LANES - 1) / (256 / LANES)), a.batch < 65535 ? a.batch : 65535);
    if (format == DF11_KV_INT8) kv_append_kernel<LANES, DF11_KV_INT8, T><<<grid, 256, 0, stream>>>(a);
    else kv_append_kernel<LANES, DF11_KV_E4M3, T><<<grid, 256, 0, stream>>>(a);
}

template <typename T> void launch_append(const AppendArgs &a, int format, cudaStream_t stream)
{
    if (a.dim <= 64) launch_append<4, T>(a, format, stream);
    else if (a.dim <= 128) launch_append<8, T>(a, format, stream);
    else launch_append<16, T>(a, format, stream);
}

// ---------------------------------------------------------------------------------------------
// Attention.  For a few query rows per key head the work is reading the cache once: 2 (d + 4) bytes
// per slot against 4 d multiply-adds per row, so one pass, in which a code is copied to shared memory
// ahead of time, goes to one register, is widened to fp16 there (exactly: int8 and e4m3 are subsets of
// fp16) and meets the matrix unit in that register:
//
//   scores   S^T[16 slots x 8 rows] += K[16 x 16] Q^T[16 x 8]     (m16n8k16, fp32 sums)
//   values   O^T[16 dims x 8 rows]  += V^T[16 x 16] P^T[16 x 8]
//
// The query rows are the narrow side, so a group of up to 8 rows wastes nothing.  A product may
// number its inner dimension as it likes as long as both operands agree: a thread loads 16
// consecutive bytes of a key row and calls them the elements that the fragment layout gives it (the
// query fragments are loaded in the same order), and of a value row 16 consecutive bytes whose
// dimensions become the rows of eight fragments.  The scores come out with the slots across lanes
// and the rows across registers; an 8x8 transposition between registers (movmatrix) turns the
// weights into the second product's operand.
//
// Scales.  A key's scale multiplies its score.  A value's scale multiplies its weight before that is
// rounded to fp16; so that neither over- nor underflows, weights are held relative to a running
// bound of weight * scale, per row, in powers of two (2^6 below which 2^-30 of the largest is still
// distinguished).  The running maximum is renewed only when a weight outgrows 2^14: a vote per tile
// instead of a reduction over lanes.  Query rows are scaled by a power of two to just below 2, which
// fp16 holds exactly from there down to 2^-24; smaller entries are rounded to multiples of 2^-24 of that.
// Sums, maxima and denominators are fp32.
//
// Small calls: the slots of a sequence are divided among a cluster of CTAs that join their results
// through distributed shared memory, in one launch.  Long ones: the tiles of all sequences and heads are
// cut into equal lengths, one per resident CTA, so that sequences of any lengths keep every SM busy
// to the end; a second kernel joins, in a fixed order, what was cut.
//
// Why mma.sync: with 4 to 16 query rows the tensor pipe is 15 % busy; a tcgen05 tile would be filled to an
// eighth and would want the widened operands written back to shared memory.  What bounds it: memory, with
// the instructions that widen and weigh (about 300 per tile of 16 slots) close behind, and 3 us per stretch for
// its start and end.  Measured in a graph of such calls: 131071 slots x 8 heads of 128 (277 MB) 55 us = 5.0 TB/s, of
// which the loads alone take 50; 32 left-padded sequences of 2048-4096 slots (174 MB) 39 us = 4.4 TB/s.  Copies of
// 512 consecutive bytes instead of the fragments' own 64-byte pieces: 78 -> 59 us for the former.
constexpr int kAttWarps = 4;
// Tiles of 16 slots under way per warp, one in use.  Heads of 128: four with three CTAs per SM against three with
// four CTAs, 32 ragged sequences 39.4 and 40.2 us, 131071 slots 54.8 and 56.9 us.
template <int D> constexpr int kAttStages = D == 256 ? 3 : 4;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Four codes to two pairs of fp16.
// int8: the code plus 128 becomes the bits of a subnormal, so a number stands for (code + 128) 2^-24,
// exactly; the products' sums are put right by 128 times the sum of the other operand.
// e4m3, keys: the conversion instruction, which gives the values themselves at a quarter of the rate of
// other instructions.  Values: the same with integer instructions -- sign to bit 15, exponent and
// mantissa to bits 13..7, which stands for the value times 2^-8 --, so that both units share the work.
constexpr float kInt8Unit = 0x1p24f, kE4m3ValueUnit = 0x1p8f;
template <int FMT, bool VALUE> __device__ __forceinline__ void widen(uint32_t codes, uint32_t &lo, uint32_t &hi)
{
    if (FMT == DF11_KV_INT8) {
        const uint32_t u = codes ^ 0x80808080u;
        lo = __byte_perm(u, 0, 0x4140);
        hi = __byte_perm(u, 0, 0x4342);
    } else if (!VALUE) {
        asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }"
            : "=r"(lo), "=r"(hi)
            : "r"(codes));
    } else {
        const uint32_t high = (codes & 0x80808080u) | ((codes & 0x7E7E7E7Eu) >> 1), low = (codes << 7) & 0x80808080u;
        lo = __byte_perm(low, high, 0x5140);
        hi = __byte_perm(low, high, 0x7362);
    }
}

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }

// A warp's tile in shared memory: 16 rows of D bytes in 16-byte chunks.  The chunks of a row are
// exchanged by its number so that neither way of reading meets a bank twice: keys, 8 lanes taking 4 even
// (or odd) chunks of two rows; values, 8 lanes taking two chunks of four rows.
template <int D> __device__ __forceinline__ int chunk_place(int row, int chunk)
{
    if (D == 64) {                                          // two rows to a line of 128 bytes
        const int line = row >> 1;
        return line * 128 + ((((row & 1) * 4 + chunk) ^ ((line & 3) * 2)) * 16);
    }
    return row * D + ((chunk ^ (row & 7)) * 16);
}

__device__ __forceinline__ void copy_chunk(uint32_t to, const uint8_t *from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

template <int BYTES> struct Bytes {
    uint32_t w[BYTES / 4];
    __device__ __forceinline__ void load(const uint8_t *from)
    {
        if (BYTES == 16) {
            const uint4 x = *reinterpret_cast<const uint4 *>(from);
            w[0] = x.x, w[1] = x.y, w[BYTES / 4 - 2] = x.z, w[BYTES / 4 - 1] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(from);
            w[0] = x.x, w[BYTES / 4 - 1] = x.y;
        }
    }
};

struct AttentionArgs {
    const void *q;
    Strides qs;
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int64_t *lengths, *first;
    int length_per, first_per;
    void *out;
    uint32_t *cuts;                     // shared out: per unit, the first result and the last CTA
    float *workspace;                   // and two results of rows * (D + 2) numbers per CTA
    uint32_t batch, kv_heads, group, queries, row_groups, cluster, ctas;
    int dim, window, q_aligned;
    int64_t max_slots;
    float scale;
};

// Where a query stands and the slots that it sees.
struct Sight {
    int64_t low, high;
};
__device__ __forceinline__ Sight sight_of(const AttentionArgs &a, int64_t length, int64_t first, uint32_t query)
{
    const int64_t place = length - (int64_t)a.queries + query;
    int64_t low = first;
    if (a.window > 0 && place - a.window + 1 > low) low = place - a.window + 1;
    return {low, place < a.max_slots ? place : a.max_slots - 1};
}

// Shared out: the slots of all sequences in tiles of 16, one row of tiles per key head and row group, cut
// into equal lengths.  Everything here follows from the sequences' lengths, so every CTA finds its own
// share, and the joining kernel every share, without asking anyone.
struct Sequence {
    uint32_t index, tiles, before;      // before: tiles per head of the sequences ahead of it
};

__device__ __forceinline__ int64_t length_of(const AttentionArgs &a, uint32_t b) { return clamped_length(a.lengths[a.length_per ? b : 0]); }
__device__ __forceinline__ int64_t start_of(const AttentionArgs &a, uint32_t b)
{
    return a.first ? clamped_length(a.first[a.first_per ? b : 0]) : 0;
}

__device__ __forceinline__ uint32_t tiles_of(const AttentionArgs &a, uint32_t b)
{
    if (b >= a.batch) return 0;
    const int64_t length = length_of(a, b), start = start_of(a, b);
    const int64_t n = sight_of(a, length, start, a.queries - 1).high - sight_of(a, length, start, 0).low + 1;
    return n > 0 ? (uint32_t)((n + 15) / 16) : 0;
}

// The whole warp: tiles per head of all sequences.
__device__ __forceinline__ uint32_t all_tiles(const AttentionArgs &a)
{
    uint32_t sum = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 32) sum += __reduce_add_sync(0xffffffffu, tiles_of(a, b0 + (threadIdx.x & 31)));
    return sum;
}

// The whole warp: the sequence that holds tile `want` of all heads' tiles.
__device__ __forceinline__ Sequence find_sequence(const AttentionArgs &a, uint32_t want)
{
    const uint32_t lane = threadIdx.x & 31, heads = a.kv_heads * a.row_groups;
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 32) {
        const uint32_t mine = tiles_of(a, b0 + lane);
        uint32_t sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= (uint32_t)d) sum += x;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, (before + sum) * heads > want);
        if (hit) {
            const int at = __ffs(hit) - 1;
            return {b0 + at, __shfl_sync(0xffffffffu, mine, at), before + __shfl_sync(0xffffffffu, sum - mine, at)};
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return {a.batch, 0, before};
}

// Tiles per CTA: equal parts, but no fewer than a tile per warp where the sequences have as many.
__device__ __forceinline__ uint32_t share_of(uint32_t total, uint32_t units, uint32_t ctas)
{
    return max((total + ctas - 1) / ctas, min(max(total / units, 1u), (uint32_t)kAttWarps));
}

constexpr uint32_t kNotCut = 0xFFFFFFFFu;

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
}

__device__ __forceinline__ uint32_t remote_address(const float *local, uint32_t rank)
{
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    return there;
}

__device__ __forceinline__ float remote_load(const float *local, uint32_t rank)
{
    float x;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(remote_address(local, rank)));
    return x;
}

__device__ __forceinline__ float4 remote_load4(const float *local, uint32_t rank)
{
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                 : "r"(remote_address(local, rank)));
    return x;
}

template <typename T> __device__ __forceinline__ void store4(T *p, float4 x)
{
    T y[4] = {df11_from_float<T>(x.x), df11_from_float<T>(x.y), df11_from_float<T>(x.z), df11_from_float<T>(x.w)};
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(y);
}

// One CTA: up to NT * 8 query rows of one key head, and its share of the slots they see.
// EXACT: head_dim is D; otherwise it is smaller, and what is loaded beyond it is some other chunk of the
// same row that meets a zero of the query or ends in a result that nobody reads.
// SHARED: tiles [first_tile, last_tile) of the sequence, the result to `ws` if they are not all of them;
// otherwise the CTAs of a cluster take equal parts.
template <int D, int NT, int FMT, bool EXACT, bool SHARED, typename T>
__device__ __forceinline__ void attend(const AttentionArgs &a, uint32_t unit, int64_t length, int64_t start, uint32_t first_tile,
                                       uint32_t last_tile, float *ws)
{
    constexpr int kRows = NT * 8;
    constexpr int kKeyChunks = D / 64;                      // 16-byte chunks of a key row per thread
    constexpr int kValBytes = D >= 128 ? 16 : D / 8;        // consecutive bytes of a value row per thread
    constexpr int kValChunks = D / 8 / kValBytes;
    constexpr int kBlocks = D / 16;                         // fragments of 16 dimensions
    constexpr int kStages = kAttStages<D>, kStageBytes = 32 * D + 128;
    extern __shared__ __align__(16) float shared[];
    float *part_o = shared;                                 // [warps][rows][D]
    float *part_m = part_o + kAttWarps * kRows * D;         // [warps][rows]
    float *part_l = part_m + kAttWarps * kRows;
    float *all_m = part_l + kAttWarps * kRows;              // [rows]
    float *all_l = all_m + kRows;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
    auto key_chunk = [&](int j) { return D == 64 ? c : (j >> 1) * 8 + 2 * c + (j & 1); };    // the j-th of this thread
    const uint32_t head = unit / a.row_groups, b = head / a.kv_heads, h = head % a.kv_heads;
    const uint32_t row0 = unit % a.row_groups * kRows, rows = a.group * a.queries, last_row = min(row0 + kRows, rows) - 1;

    // the slots that any of the rows sees, and those that all of them see
    const Sight top = sight_of(a, length, start, row0 / a.group), bottom = sight_of(a, length, start, last_row / a.group);
    const int64_t low = SHARED ? sight_of(a, length, start, 0).low : top.low;
    const int64_t n = max((SHARED ? sight_of(a, length, start, a.queries - 1).high : bottom.high) - low + 1, (int64_t)0);
    const int inner_low = (int)min(bottom.low - low, n), inner_high = (int)max(top.high - low, (int64_t)-1);
    const int count = (int)n;
    int col_low[NT][2], col_high[NT][2];                    // relative to `low`
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Sight s = sight_of(a, length, start, min(row0 + nt * 8 + 2 * c + i, last_row) / a.group);
            col_low[nt][i] = (int)min(s.low - low, n);
            col_high[nt][i] = (int)max(s.high - low, (int64_t)-1);
        }

    const uint32_t rank = !SHARED && a.cluster > 1 ? cluster_rank() : 0;
    if (!SHARED) {
        const uint32_t tiles = (uint32_t)((n + 15) / 16), share = tiles / a.cluster, extra = tiles - share * a.cluster;
        first_tile = share * rank + min(rank, extra), last_tile = first_tile + share + (rank < extra);
    }
    const int begin = (int)first_tile, end = min((int)last_tile, (int)((n + 15) / 16));
    const int64_t cell0 = (int64_t)head * a.max_slots + low;

    float o[kBlocks][NT][4] = {}, o128[NT][4] = {};         // o128: 128 times the sum of the weights, in the codes' unit
    // running maximum, sum, factor on weight * scale, and the largest weight * scale when it was set;
    // the factor starts so large that the first weight * scale that is not zero sets it
    float m[NT][2], l[NT][2] = {}, f[NT][2], big[NT][2] = {};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY, f[nt][0] = f[nt][1] = 0x1p126f;

    const int dim = EXACT ? D : a.dim;
    // A warp's tiles come through a ring in shared memory, each operand of a tile in D / 32 copies of 512
    // consecutive bytes.  Past the last slot the last one is copied again, and past the last chunk of a
    // row that one: whatever lies in the cache there (a NaN, say) does not reach a product.
    constexpr int kRowChunks = D / 16, kRowsPerCopy = 32 / kRowChunks, kCopies = 16 / kRowsPerCopy;
    const int copy_row = lane / kRowChunks, copy_chunk_at = EXACT ? lane % kRowChunks * 16 : min(lane % kRowChunks * 16, dim - 16);
    const uint8_t *const key_base = a.k_codes + cell0 * dim + copy_chunk_at, *const value_base = a.v_codes + cell0 * dim + copy_chunk_at;
    uint8_t *const ring = reinterpret_cast<uint8_t *>(shared) + warp * (kStages * kStageBytes);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const float *const scale_base = (c < 2 ? a.k_scales : a.v_scales) + cell0;      // scales of rows r and r + 8, for all lanes of r
    auto fetch = [&](int tile, uint32_t stage) {
        const int s0 = tile * 16, left = count - 1 - s0;
        const uint8_t *const kp = key_base + (int64_t)s0 * dim, *const vp = value_base + (int64_t)s0 * dim;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(stage + 32 * D + lane * 4),
                     "l"(scale_base + s0 + min(r + 8 * (c & 1), left))
                     : "memory");
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int row = i * kRowsPerCopy + copy_row, from = (left >= 15 ? row : min(row, left)) * dim;
            const uint32_t to = stage + chunk_place<D>(row, lane % kRowChunks);
            copy_chunk(to, kp + from);
            copy_chunk(to + 16 * D, vp + from);
        }
    };
    // which warp takes the first tile differs from CTA to CTA, so that no scheduler gets all the odd ones
    const int turn_of = (warp + (int)blockIdx.x) & (kAttWarps - 1);
    int ahead = begin + turn_of;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (ahead < end) fetch(ahead, ring_at + i * kStageBytes);
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead += kAttWarps;
    }
    // The query fragments, in the order in which the key bytes lie, while the first tiles are on their way.
    uint32_t qf[NT][D / 16][2];
    float mult[NT][2];                                      // score = sum * mult * key scale, in powers of two
    float offset[NT][2] = {};                               // what the sum starts from: - 128 sum(q) in the codes' unit
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const uint32_t row = min(row0 + nt * 8 + r, last_row), query = row / a.group;
        const T *x = (const T *)a.q + b * a.qs.b + (h * a.group + (row - query * a.group)) * a.qs.h + query * a.qs.t;
        float peak = 0.0f;
        uint32_t raw[D / 16][2];
#pragma unroll
        for (int j = 0; j < kKeyChunks; ++j) {
            const int d0 = key_chunk(j) * 16;
            if (d0 >= a.dim) {
#pragma unroll
                for (int w = 0; w < 4; ++w) raw[j * 4 + w][0] = raw[j * 4 + w][1] = 0;
            } else if (a.q_aligned) {
                const uint4 lo = *reinterpret_cast<const uint4 *>(x + d0), hi = *reinterpret_cast<const uint4 *>(x + d0 + 8);
                raw[j * 4][0] = lo.x, raw[j * 4][1] = lo.y, raw[j * 4 + 1][0] = lo.z, raw[j * 4 + 1][1] = lo.w;
                raw[j * 4 + 2][0] = hi.x, raw[j * 4 + 2][1] = hi.y, raw[j * 4 + 3][0] = hi.z, raw[j * 4 + 3][1] = hi.w;
            } else {
                const uint16_t *y = reinterpret_cast<const uint16_t *>(x) + d0;
#pragma unroll
                for (int w = 0; w < 8; ++w) raw[j * 4 + w / 2][w & 1] = (uint32_t)y[2 * w] | (uint32_t)y[2 * w + 1] << 16;
            }
        }
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const T *pair = reinterpret_cast<const T *>(&raw[s][i]);
                peak = fmaxf(peak, fmaxf(fabsf(df11_to_float(pair[0])), fabsf(df11_to_float(pair[1]))));
            }
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
        // 2^e <= peak < 2^(e+1); an infinity stays one
        const int e = peak > 0.0f && peak <= 3.402823466e38f ? max((int)(__float_as_uint(peak) >> 23) - 127, -126) : 0;
        const float down = power_of_two(-e);
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const T *pair = reinterpret_cast<const T *>(&raw[s][i]);
                qf[nt][s][i] = pack_half(df11_to_float(pair[0]) * down, df11_to_float(pair[1]) * down);
            }
        if (FMT == DF11_KV_INT8) {
            float sum = 0.0f;
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 pair = __half22float2(*reinterpret_cast<const __half2 *>(&qf[nt][s][i]));
                    sum += pair.x + pair.y;
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= -128.0f / kInt8Unit;
            offset[nt][0] = __shfl_sync(0xffffffffu, sum, 8 * c);
            offset[nt][1] = __shfl_sync(0xffffffffu, sum, 8 * c + 4);
        }
        const float up = power_of_two(e) * (a.scale * kLog2e) * (FMT == DF11_KV_INT8 ? kInt8Unit : 1.0f);
        mult[nt][0] = __shfl_sync(0xffffffffu, up, 8 * c);          // the row of this thread's first column
        mult[nt][1] = __shfl_sync(0xffffffffu, up, 8 * c + 4);
    }

    int at_stage = 0;
    for (int tile = begin + turn_of; tile < end; tile += kAttWarps) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        const uint8_t *const stage = ring + at_stage * kStageBytes;
        {
            const int to = at_stage == 0 ? kStages - 1 : at_stage - 1;      // read in the step before
            if (ahead < end) fetch(ahead, ring_at + to * kStageBytes);
            asm volatile("cp.async.commit_group;" ::: "memory");
            ahead += kAttWarps;
            at_stage = at_stage == kStages - 1 ? 0 : at_stage + 1;
        }
        const float4 scales = *reinterpret_cast<const float4 *>(stage + 32 * D + r * 16);
        const float key_scale[2] = {scales.x, scales.y}, value_scale[2] = {scales.z, scales.w};
        Bytes<16> kx[2][kKeyChunks];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < kKeyChunks; ++j) kx[i][j].load(stage + chunk_place<D>(r + 8 * i, key_chunk(j)));
        float s[NT][4], s2[NT][4] = {};                     // two chains of sums: a product waits for the last of its chain
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][2] = offset[nt][0], s[nt][1] = s[nt][3] = offset[nt][1];
#pragma unroll
        for (int j = 0; j < kKeyChunks; ++j)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t a0, a1, a2, a3;
                widen<FMT, false>(kx[0][j].w[w], a0, a2);
                widen<FMT, false>(kx[1][j].w[w], a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16x8x16(w & 1 ? s2[nt] : s[nt], a0, a1, a2, a3, qf[nt][j * 4 + w][0], qf[nt][j * 4 + w][1]);
            }
        Bytes<kValBytes> vx[4][kValChunks];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < kValChunks; ++j) {
                const int row = 2 * c + (i & 1) + 8 * (i >> 1);
                vx[i][j].load(stage + 16 * D + (kValBytes == 16 ? chunk_place<D>(row, j * 8 + r) : chunk_place<D>(row, r >> 1) + (r & 1) * 8));
            }

        const int s0 = tile * 16;
        const bool whole = s0 >= inner_low && s0 + 15 <= inner_high;    // every row sees every slot
        float p[NT][4], w[NT][4];
        auto weigh = [&]() {                                            // true if a weight has outgrown its bound
            float most = 0.0f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int col = i & 1, slot = s0 + r + 8 * (i >> 1);
                    p[nt][i] = exp2_approx(s[nt][i] - m[nt][col]);
                    w[nt][i] = p[nt][i] * value_scale[i >> 1] * f[nt][col];
                    if (!whole && (slot < col_low[nt][col] || slot > col_high[nt][col])) p[nt][i] = w[nt][i] = 0.0f;
                    most = fmaxf(most, fmaxf(p[nt][i], w[nt][i]));
                }
            return most > 16384.0f;
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][i] = (s[nt][i] + s2[nt][i]) * (key_scale[i >> 1] * mult[nt][i & 1]);
        if (__any_sync(0xffffffffu, weigh())) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int col = 0; col < 2; ++col) {
                    float peak = m[nt][col];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int slot = s0 + r + 8 * i;
                        if (whole || (slot >= col_low[nt][col] && slot <= col_high[nt][col])) peak = fmaxf(peak, s[nt][col + 2 * i]);
                    }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, x));
                    const float was = m[nt][col];
                    const float back = was == -INFINITY ? 0.0f : exp2_approx(was - peak);
                    float heavy = 0.0f;                                  // the largest weight * scale, relative to `peak`
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int slot = s0 + r + 8 * i;
                        if (whole || (slot >= col_low[nt][col] && slot <= col_high[nt][col]))
                            heavy = fmaxf(heavy, exp2_approx(s[nt][col + 2 * i] - peak) * value_scale[i]);
                    }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) heavy = fmaxf(heavy, __shfl_xor_sync(0xffffffffu, heavy, x));
                    heavy = fmaxf(heavy, big[nt][col] * back);
                    // f brings it to [2^6, 2^7)
                    const float now = heavy > 0.0f && heavy <= 3.402823466e38f
                        ? power_of_two(133 - (int)(__float_as_uint(heavy) >> 23)) : f[nt][col];
                    const float turn = back * (now / f[nt][col]);
                    l[nt][col] *= back;
#pragma unroll
                    for (int k = 0; k < kBlocks; ++k) o[k][nt][col] *= turn, o[k][nt][col + 2] *= turn;
                    o128[nt][col] *= turn;
                    m[nt][col] = peak, big[nt][col] = heavy, f[nt][col] = now;
                }
            weigh();
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            l[nt][0] += p[nt][0] + p[nt][2];
            l[nt][1] += p[nt][1] + p[nt][3];
            pb[nt][0] = transpose_8x8(pack_half(w[nt][0], w[nt][1]));
            pb[nt][1] = transpose_8x8(pack_half(w[nt][2], w[nt][3]));
            if (FMT == DF11_KV_INT8) mma_16x8x16(o128[nt], 0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u, pb[nt][0], pb[nt][1]);
        }
#pragma unroll
        for (int j = 0; j < kValChunks; ++j)
#pragma unroll
            for (int x = 0; x < kValBytes / 4; ++x)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t pick = half ? 0x7362 : 0x5140;       // two dimensions of two slots
                    uint32_t a0, a1, a2, a3;
                    widen<FMT, true>(__byte_perm(vx[0][j].w[x], vx[1][j].w[x], pick), a0, a1);
                    widen<FMT, true>(__byte_perm(vx[2][j].w[x], vx[3][j].w[x], pick), a2, a3);
                    const int k = (j * (kValBytes / 4) + x) * 2 + half;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16x8x16(o[k][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                        // the ring's memory is used for the results

    // the warps' results are joined
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int col = 0; col < 2; ++col) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[nt][col] += __shfl_xor_sync(0xffffffffu, l[nt][col], x);
            if (r == 0) {
                part_m[warp * kRows + nt * 8 + 2 * c + col] = m[nt][col];
                part_l[warp * kRows + nt * 8 + 2 * c + col] = l[nt][col];
            }
        }
    __syncthreads();
    if (threadIdx.x < kRows) {
        float peak = -INFINITY, total = 0.0f;
        for (int k = 0; k < kAttWarps; ++k) peak = fmaxf(peak, part_m[k * kRows + threadIdx.x]);
        for (int k = 0; k < kAttWarps; ++k) {
            const float x = part_m[k * kRows + threadIdx.x];
            if (x != -INFINITY) total += exp2_approx(x - peak) * part_l[k * kRows + threadIdx.x];
            else total += part_l[k * kRows + threadIdx.x];      // nothing, or a NaN
        }
        all_m[threadIdx.x] = peak;
        all_l[threadIdx.x] = total;
    }
    __syncthreads();
    const int live = (int)(last_row - row0 + 1);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int col = 0; col < 2; ++col) {
            const int row = nt * 8 + 2 * c + col;
            if (row >= live) continue;
            const float turn = (m[nt][col] == -INFINITY ? 1.0f : exp2_approx(m[nt][col] - all_m[row]) / f[nt][col]) *
                               (FMT == DF11_KV_INT8 ? kInt8Unit : kE4m3ValueUnit);
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) {
                // fragment k: this thread's bytes 2k and 2k + 1 of its chunk
                const int byte = 2 * k % kValBytes, d0 = ((2 * k / kValBytes) * 8 + r) * kValBytes + byte;
                *reinterpret_cast<float2 *>(part_o + (warp * kRows + row) * D + d0) =
                    make_float2((o[k][nt][col] - o128[nt][col]) * turn, (o[k][nt][col + 2] - o128[nt][col]) * turn);
            }
        }
    __syncthreads();
    for (int i = threadIdx.x * 4; i < live * D; i += kAttWarps * 128) {
        float4 sum = *reinterpret_cast<const float4 *>(part_o + i);
#pragma unroll
        for (int k = 1; k < kAttWarps; ++k) {
            const float4 x = *reinterpret_cast<const float4 *>(part_o + k * kRows * D + i);
            sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
        }
        *reinterpret_cast<float4 *>(part_o + i) = sum;
    }

    // the results of a cluster's CTAs are joined, a share of the numbers by each
    if (!SHARED && a.cluster > 1) cluster_barrier();
    else __syncthreads();
    for (int i = ((int)rank * kAttWarps * 32 + threadIdx.x) * 4; i < live * D; i += (SHARED ? 1 : a.cluster) * kAttWarps * 128) {
        const int row = i / D, d = i % D;
        if (d >= dim) continue;
        float peak = -INFINITY, total = 0.0f;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (SHARED || a.cluster == 1) {
            peak = all_m[row], total = all_l[row], sum = *reinterpret_cast<const float4 *>(part_o + i);
        } else {
            for (uint32_t k = 0; k < a.cluster; ++k) peak = fmaxf(peak, remote_load(all_m + row, k));
            for (uint32_t k = 0; k < a.cluster; ++k) {
                const float x = remote_load(all_m + row, k), turn = x == -INFINITY ? 1.0f : exp2_approx(x - peak);
                const float4 y = remote_load4(part_o + i, k);
                total += turn * remote_load(all_l + row, k);
                sum.x += turn * y.x, sum.y += turn * y.y, sum.z += turn * y.z, sum.w += turn * y.w;
            }
        }
        if (SHARED && ws) {
            *reinterpret_cast<float4 *>(ws + i) = sum;
            if (d == 0) ws[kRows * D + row] = peak, ws[kRows * D + kRows + row] = total;
        } else {
            const uint32_t at = row0 + row, query = at / a.group, hq = h * a.group + (at - query * a.group);
            const float turn = total == 0.0f ? 0.0f : 1.0f / total;
            sum.x *= turn, sum.y *= turn, sum.z *= turn, sum.w *= turn;
            store4((T *)a.out + (((int64_t)b * a.queries + query) * (a.kv_heads * a.group) + hq) * dim + d, sum);
        }
    }
    if (!SHARED && a.cluster > 1) cluster_barrier();    // nobody leaves while its memory is read
    if (SHARED) __syncthreads();                        // the next stretch fills the same memory
}

template <int D, int NT> constexpr int kAttCtas = D == 256 ? 2 : D == 128 ? 4 - NT : 5 - NT;     // per SM, by registers and memory

template <int D, int NT, int FMT, bool EXACT, typename T>
__global__ void __launch_bounds__(kAttWarps * 32, (kAttCtas<D, NT>)) kv_attention_kernel(AttentionArgs a)
{
    const uint32_t unit = blockIdx.x / a.cluster, b = unit / a.row_groups / a.kv_heads;
    attend<D, NT, FMT, EXACT, false, T>(a, unit, length_of(a, b), start_of(a, b), 0, 0, nullptr);
}

template <int D, int NT, int FMT, bool EXACT, typename T>
__global__ void __launch_bounds__(kAttWarps * 32, (kAttCtas<D, NT>)) kv_attention_shared_kernel(AttentionArgs a)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // the joining kernel may take its places
    const uint32_t heads = a.kv_heads * a.row_groups, total = all_tiles(a) * heads, share = share_of(total, a.batch * heads, gridDim.x);
    if ((uint64_t)share * blockIdx.x >= total) return;
    uint32_t at = share * blockIdx.x;
    const uint32_t end = min(at + share, total);
    Sequence s = find_sequence(a, at);
    int64_t length = length_of(a, s.index), start = start_of(a, s.index);
    bool front = true;
    while (at < end && s.tiles) {
        const uint32_t inside = at - s.before * heads, unit = inside / s.tiles, first = inside - unit * s.tiles;
        const uint32_t last = min(s.tiles, first + (end - at)), slot = blockIdx.x * 2 + !front;
        const bool whole = first == 0 && last == s.tiles;
        if (threadIdx.x == 0) {
            // where the results are: nowhere but in `out`, or in the workspace from `slot` up to some CTA's
            uint32_t *const cut = a.cuts + 2 * (s.index * heads + unit);
            if (first == 0) cut[0] = whole ? kNotCut : slot;
            if (last == s.tiles) cut[1] = blockIdx.x;
        }
        attend<D, NT, FMT, EXACT, true, T>(a, s.index * heads + unit, length, start, first, last,
                                           whole ? nullptr : a.workspace + (int64_t)slot * (NT * 8 * (D + 2)));
        at += last - first;
        front = false;
        if (at < end && unit + 1 == heads && last == s.tiles) {
            s.before += s.tiles;
            do s.tiles = tiles_of(a, ++s.index); while (s.tiles == 0 && s.index < a.batch);
            if (s.tiles) length = length_of(a, s.index), start = start_of(a, s.index);
        }
    }
}

// Joins the shares of a sequence that was cut, and writes the zeros of one that has no slots: one CTA
// per query row, its threads in WAYS ways that take every WAYS-th share.
template <int D, int NT, int WAYS, typename T> __global__ void __launch_bounds__(D * WAYS) kv_attention_join_kernel(AttentionArgs a)
{
    constexpr int kRows = NT * 8, kSlot = kRows * (D + 2);
    __shared__ float sums[WAYS][D], totals[WAYS], peaks[WAYS];
    const uint32_t rows = a.group * a.queries, at = blockIdx.x % rows, head = blockIdx.x / rows, b = head / a.kv_heads;
    const uint32_t tiles = tiles_of(a, b);
    asm volatile("griddepcontrol.wait;" ::: "memory");                  // the shares are written
    const uint32_t *const cut = a.cuts + 2 * (head * a.row_groups + at / kRows);
    const uint32_t from = cut[0], last = cut[1];
    if (tiles && (from == kNotCut || from / 2 > last || last >= a.ctas)) return;    // whole: written where it was computed
    const int row = (int)(at % kRows), d = threadIdx.x % D, way = threadIdx.x / D;
    float peak = -INFINITY, sum = 0.0f, l = 0.0f;
    if (tiles) {
        // the first share may be the second of its CTA, all others are their CTA's first
        const uint32_t j0 = from / 2;
#pragma unroll 4
        for (uint32_t j = j0 + way; j <= last; j += WAYS) {
            const float *const x = a.workspace + (int64_t)(j == j0 ? from : j * 2) * kSlot;
            const float m = x[kRows * D + row], y = x[row * D + d], z = x[kRows * D + kRows + row];
            const float now = fmaxf(peak, m), old = peak == -INFINITY ? 0.0f : exp2_approx(peak - now);
            const float turn = m == -INFINITY ? 1.0f : exp2_approx(m - now);
            l = l * old + turn * z;
            sum = sum * old + turn * y;
            peak = now;
        }
    }
    if (WAYS > 1) {
        sums[way][d] = sum;
        if (d == 0) totals[way] = l, peaks[way] = peak;
        __syncthreads();
        if (way) return;
#pragma unroll
        for (int k = 1; k < WAYS; ++k) peak = fmaxf(peak, peaks[k]);
        sum = l = 0.0f;
#pragma unroll
        for (int k = 0; k < WAYS; ++k) {
            const float turn = peaks[k] == -INFINITY ? 1.0f : exp2_approx(peaks[k] - peak);
            l += turn * totals[k];
            sum += turn * sums[k][d];
        }
    }
    if (d >= a.dim) return;
    const uint32_t query = at / a.group, hq = head % a.kv_heads * a.group + (at - query * a.group);
    ((T *)a.out)[(((int64_t)b * a.queries + query) * (a.kv_heads * a.group) + hq) * a.dim + d] =
        df11_from_float<T>(l == 0.0f ? 0.0f : sum / l);
}

// How a call is divided, from its sizes alone.
struct Division {
    int width, tiles_n;         // padded head_dim, row tiles of 8
    int cluster;                // CTAs per unit; 0: the work is shared out
    int64_t row_groups, units, ctas, cuts, workspace;
};

constexpr int kSms = 148;
// Codes that a warp of a cluster may have to read at most.  Above it, sharing out pays for its second launch and the
// joining: 8 key heads of 128, 8192 slots (64 KB per warp): cluster 12.7 us, shared out 15.7; 16384 slots: 19.2
// and 17.5; 2 heads, 32768 slots: 32 and 24; 32 sequences of 1024 slots (32 KB): 16.2 and 21.9.
constexpr int64_t kLongStretch = 96 << 10;

Division divide(int64_t batch, int32_t heads, int32_t kv_heads, int64_t queries, int32_t head_dim, int64_t max_slots, int32_t window)
{
    Division d;
    const int64_t rows = (int64_t)(heads / kv_heads) * queries;
    d.width = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    d.tiles_n = rows > 8 && d.width < 256 ? 2 : 1;
    d.row_groups = (rows + d.tiles_n * 8 - 1) / (d.tiles_n * 8);
    d.units = batch * kv_heads * d.row_groups;
    d.cuts = d.workspace = 0;
    const int64_t span = window > 0 && (int64_t)window + queries < max_slots ? window + queries : max_slots;
    const int64_t tiles = (span + 15) / 16;
    const int per_sm = d.width == 256 ? kAttCtas<256, 1> : d.width == 128 ? (d.tiles_n == 1 ? kAttCtas<128, 1> : kAttCtas<128, 2>)
                                                         : (d.tiles_n == 1 ? kAttCtas<64, 1> : kAttCtas<64, 2>);
    const int64_t most = (tiles + 2 * kAttWarps - 1) / (2 * kAttWarps);                         // two tiles per warp
    int64_t want = d.units > 0 ? kSms * per_sm / d.units : 1;
    if (want > most) want = most;
    d.cluster = want >= 8 ? 8 : want >= 4 ? 4 : want >= 2 ? 2 : 1;
    d.ctas = d.units * d.cluster;
    const int64_t bytes_per_warp = (tiles + d.cluster * kAttWarps - 1) / (d.cluster * kAttWarps) * 32 * d.width;
    if (bytes_per_warp > kLongStretch && (double)d.units * (double)tiles < 2e9) {
        d.cluster = 0;
        d.ctas = kSms * per_sm;
        d.cuts = (d.units * 2 * (int64_t)sizeof(uint32_t) + 15) / 16 * 16;
        d.workspace = d.cuts + d.ctas * 2 * d.tiles_n * 8 * (d.width + 2) * (int64_t)sizeof(float);
    }
    return d;
}

template <typename K> cudaError_t launch_wide(K kernel, unsigned grid, unsigned block, size_t shared, unsigned cluster,
                                              int device, cudaStream_t stream, const AttentionArgs &a)
{
    if (shared > 48 * 1024) {
        const cudaError_t e = df11_allow_shared((const void *)kernel, shared, device);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = cluster > 1;
    return cudaLaunchKernelEx(&config, kernel, a);
}

template <int D, int NT, int FMT, bool EXACT, typename T>
cudaError_t launch_attention(const AttentionArgs &a, const Division &d, int device, cudaStream_t stream)
{
    constexpr int kRows = NT * 8;
    constexpr size_t kJoin = (size_t)(kAttWarps * kRows * D + 2 * kAttWarps * kRows + 2 * kRows) * sizeof(float);
    constexpr size_t kRing = (size_t)kAttWarps * kAttStages<D> * (32 * D + 128), kShared = kRing > kJoin ? kRing : kJoin;
    if (d.cluster)
        return launch_wide(kv_attention_kernel<D, NT, FMT, EXACT, T>, (unsigned)d.ctas, kAttWarps * 32, kShared, (unsigned)d.cluster,
                           device, stream, a);
    const cudaError_t e = launch_wide(kv_attention_shared_kernel<D, NT, FMT, EXACT, T>, (unsigned)d.ctas, kAttWarps * 32, kShared, 1,
                                      device, stream, a);
    if (e != cudaSuccess) return e;
    // The joining kernel is launched while the first still runs and waits for its end on the device.  Where many
    // CTAs meet in a sequence, several threads share its results; otherwise small CTAs all fit at once.
    constexpr int kWays = 1024 / D;
    const bool many = d.ctas > 8 * d.units;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(d.units / d.row_groups * ((int64_t)a.group * a.queries)));
    config.blockDim = dim3(many ? D * kWays : D);
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    return many ? cudaLaunchKernelEx(&config, kv_attention_join_kernel<D, NT, kWays, T>, a)
                : cudaLaunchKernelEx(&config, kv_attention_join_kernel<D, NT, 1, T>, a);
}

template <typename T> cudaError_t launch_attention(const AttentionArgs &a, const Division &d, int format, int device, cudaStream_t stream)
{
#define DF11_ATTENTION(D, NT)                                                                             \
    if (d.width == D && d.tiles_n == NT) {                                                                \
        if (format == DF11_KV_INT8)                                                                       \
            return a.dim == D ? launch_attention<D, NT, DF11_KV_INT8, true, T>(a, d, device, stream)              \
                              : launch_attention<D, NT, DF11_KV_INT8, false, T>(a, d, device, stream);            \
        return a.dim == D ? launch_attention<D, NT, DF11_KV_E4M3, true, T>(a, d, device, stream)                  \
                          : launch_attention<D, NT, DF11_KV_E4M3, false, T>(a, d, device, stream);                \
    }
    DF11_ATTENTION(64, 1)
    DF11_ATTENTION(64, 2)
    DF11_ATTENTION(128, 1)
    DF11_ATTENTION(128, 2)
    DF11_ATTENTION(256, 1)
#undef DF11_ATTENTION
    return cudaErrorInvalidValue;
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
    if (2.0 * kv_heads * (double)tokens > 2e9) return df11_fail(DF11_ERR_BADARG, "too many rows for one call");
    if (batch == 0 || tokens == 0) return DF11_OK;
    Df11DeviceScope scope(device);
    if (!scope.ok) return df11_fail(DF11_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    AppendArgs a = {};
    a.k = k, a.v = v, a.ks = {k_stride_b, k_stride_h, k_stride_t}, a.vs = {v_stride_b, v_stride_h, v_stride_t};
    a.k_codes = (uint8_t *)k_codes, a.v_codes = (uint8_t *)v_codes, a.k_scales = (float *)k_scales, a.v_scales = (float *)v_scales;
    a.positions = (const int64_t *)positions, a.per_sequence = n_positions > 1, a.status = (int *)status;
    a.max_slots = max_slots, a.batch = (uint32_t)batch, a.heads = (uint32_t)kv_heads, a.tokens = (uint32_t)tokens, a.dim = head_dim;
    a.aligned = !((((uintptr_t)k | (uintptr_t)v) & 15) ||
                  ((k_stride_b | k_stride_h | k_stride_t | v_stride_b | v_stride_h | v_stride_t) & 7));
    if (element_type == DF11_TYPE_BF16) launch_append<__nv_bfloat16>(a, format, (cudaStream_t)stream);
    else launch_append<__half>(a, format, (cudaStream_t)stream);
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
    const int64_t units = batch * kv_heads, chunks = head_dim / 8, blocks = (n_slots * chunks + 1023) / 1024;
    if (blocks > 0x7FFFFFFF || units > 0x7FFFFFFF) return df11_fail(DF11_ERR_BADARG, "too many slots for one call");
    if (units == 0 || n_slots == 0) return DF11_OK;
    Df11DeviceScope scope(device);
    if (!scope.ok) return df11_fail(DF11_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    ReadArgs a = {};
    a.k_codes = (const uint8_t *)k_codes, a.v_codes = (const uint8_t *)v_codes, a.k_scales = (const float *)k_scales;
    a.v_scales = (const float *)v_scales, a.k_out = k_out, a.v_out = v_out, a.max_slots = max_slots, a.first = first_slot;
    a.units = (uint32_t)units, a.n = (uint32_t)n_slots, a.chunks = (uint32_t)chunks;
    const dim3 grid((unsigned)blocks, (unsigned)(units < 65535 ? units : 65535), 2);
    auto go = [&](auto kernel) { kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(a); };
    if (element_type == DF11_TYPE_BF16) format == DF11_KV_INT8 ? go(kv_read_kernel<DF11_KV_INT8, __nv_bfloat16>) : go(kv_read_kernel<DF11_KV_E4M3, __nv_bfloat16>);
    else format == DF11_KV_INT8 ? go(kv_read_kernel<DF11_KV_INT8, __half>) : go(kv_read_kernel<DF11_KV_E4M3, __half>);
    return launched();
}

extern "C" int64_t df11_kv_attention_workspace_bytes(int64_t batch, int32_t heads, int32_t kv_heads, int64_t queries,
                                                     int32_t head_dim, int64_t max_slots, int32_t window)
{
    if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || queries < 0 || max_slots < 1 || window < 0)
        return df11_fail(DF11_ERR_BADARG, "batch, heads, queries, max_slots or window out of range");
    if (head_dim < 16 || head_dim > DF11_KV_MAX_HEAD_DIM || head_dim % 16)
        return df11_fail(DF11_ERR_BADARG, "head_dim %d: multiples of 16 up to %d are supported", head_dim, DF11_KV_MAX_HEAD_DIM);
    if ((double)batch * heads * (double)queries > 2e9) return df11_fail(DF11_ERR_BADARG, "too many query rows for one call");
    const Division d = divide(batch, heads, kv_heads, queries, head_dim, max_slots, window);
    return d.workspace;
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
    const Division d = divide(batch, heads, kv_heads, queries, head_dim, max_slots, window);
    if ((double)d.ctas > 2e9) return df11_fail(DF11_ERR_BADARG, "too many query rows for one call");
    AttentionArgs a = {};
    a.q = q, a.qs = {q_stride_b, q_stride_h, q_stride_t};
    a.q_aligned = !(((uintptr_t)q & 15) || (q_stride_b | q_stride_h | q_stride_t) & 7);
    a.k_codes = (const uint8_t *)k_codes, a.v_codes = (const uint8_t *)v_codes;
    a.k_scales = (const float *)k_scales, a.v_scales = (const float *)v_scales;
    a.lengths = (const int64_t *)lengths, a.length_per = n_lengths > 1;
    a.first = (const int64_t *)first, a.first_per = n_first > 1;
    a.out = out, a.cuts = (uint32_t *)workspace, a.workspace = (float *)((uint8_t *)workspace + d.cuts);
    a.kv_heads = (uint32_t)kv_heads, a.group = (uint32_t)(heads / kv_heads), a.dim = head_dim, a.window = window;
    a.batch = (uint32_t)batch, a.row_groups = (uint32_t)d.row_groups, a.cluster = (uint32_t)d.cluster, a.ctas = (uint32_t)d.ctas;
    a.queries = (uint32_t)queries, a.max_slots = max_slots, a.scale = scale;
    const cudaError_t e = element_type == DF11_TYPE_BF16 ? launch_attention<__nv_bfloat16>(a, d, format, device, (cudaStream_t)stream)
                                                         : launch_attention<__half>(a, d, format, device, (cudaStream_t)stream);
    if (e != cudaSuccess) return df11_fail(DF11_ERR_CUDA, "kernel launch failed: %s", cudaGetErrorString(e));
    return DF11_OK;
}
