// attn.cuh -- device helpers of the attention sublayer: activation types, batch
// and page lookups with their checks, and the norm and rotation of a query head.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>

#include <type_traits>

#include "../../include/jeromoe.h"
#include "attn.h"
#include "ptx.cuh"

namespace jmoe {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// one rounding to the row's type, to nearest even
__device__ __forceinline__ void from_f32(float &d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__half &d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(__nv_bfloat16 &d, float v) { d = __float2bfloat16_rn(v); }

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x)
{
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// An untiled copy to shared memory, counted by a barrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}

// Four signed bytes to f16 pairs: byte + 128 under the exponent of 1024, minus 1152.
__device__ __forceinline__ void bytes_f16(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), bias), y = __hsub2(*reinterpret_cast<__half2 *>(&b), bias);
    lo = *reinterpret_cast<const uint32_t *>(&x);
    hi = *reinterpret_cast<const uint32_t *>(&y);
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Attention's weights carry the scale of their block's values, 2^(logit + log2 sv - m)
// with m the row's largest such exponent, and the denominator takes it out again.
// Scales range over 2^-74 .. 2^121, further than the exponents of f32 reach, and a
// block far below the largest one adds nothing to the sums but counts in the
// denominator like any other: there its weights are formed from an exponent of
// their own, kFar above the block's largest (so that they are zero as f16), and
// rescaled with what that exponent is below m.
constexpr float kFar = 60.0f;
// Values of a block without a scale (all zeros): far below any real scale (>= 2^-74),
// so their weights stay small and the sums in range.
constexpr float kNoScaleLog2 = -80.0f;

// The exponent that a block's weights are formed from. top: the block's largest, -inf for none seen.
__device__ __forceinline__ float block_ref(float ms, float top) { return top > -INFINITY ? fminf(ms, top + kFar) : ms; }

// l 2^x for a denominator l, where 2^x alone may underflow (x down to -250).
__device__ __forceinline__ float scale_den(float l, float a, float x)       // a = ex2(x)
{
    if (x > -100.0f) return l * a;
    const float h = ex2(0.5f * x);
    return l * h * h;
}

// Queries take two halves of 11 bits with F32 rows, and with F16 rows that are normed
// and turned as they are read: cut to one, they add as much to an output's error as
// its rounding to f16 (1.7 times that in all; so 1.0 to 1.3 times). BF16 rows' own
// rounding hides it, and rows that come as they are fit one half.
template <typename T>
inline bool keep_queries(const AttnParams &p)
{
    return sizeof(T) == 4 || (std::is_same<T, __half>::value && p.use_rope);
}

// Loads of memory that a kernel before this one may have written: this kernel
// may have been launched while that one ran, so none goes through the read-only path.
template <typename T>
__device__ __forceinline__ T ld_plain(const T *p) { return *p; }

// N consecutive values (N * size a multiple of 4 bytes, so aligned) to and from f32.
template <int N, typename T>
__device__ __forceinline__ void load_vals(const T *p, float (&v)[N])
{
    constexpr int kBytes = N * (int)sizeof(T), kWord = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : 4;
    static_assert(kBytes % kWord == 0, "vector");
    alignas(16) T t[N];
#pragma unroll
    for (int i = 0; i < kBytes / kWord; i++) {
        if (kWord == 16) reinterpret_cast<uint4 *>(t)[i] = ld_plain(reinterpret_cast<const uint4 *>(p) + i);
        else if (kWord == 8) reinterpret_cast<uint2 *>(t)[i] = ld_plain(reinterpret_cast<const uint2 *>(p) + i);
        else reinterpret_cast<uint32_t *>(t)[i] = ld_plain(reinterpret_cast<const uint32_t *>(p) + i);
    }
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_f32(t[i]);
}

template <int N, typename T>
__device__ __forceinline__ void store_vals(T *p, const float (&v)[N])
{
    constexpr int kBytes = N * (int)sizeof(T), kWord = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : 4;
    static_assert(kBytes % kWord == 0, "vector");
    alignas(16) T t[N];
#pragma unroll
    for (int i = 0; i < N; i++) from_f32(t[i], v[i]);
#pragma unroll
    for (int i = 0; i < kBytes / kWord; i++) {
        if (kWord == 16) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(t)[i];
        else if (kWord == 8) reinterpret_cast<uint2 *>(p)[i] = reinterpret_cast<const uint2 *>(t)[i];
        else reinterpret_cast<uint32_t *>(p)[i] = reinterpret_cast<const uint32_t *>(t)[i];
    }
}

// A wait that ran out is left in the word: after one no output of the call is good.
__device__ __forceinline__ void kv_error(int *err) { atomicCAS(err, 0, kErrKvBounds); }

__device__ __forceinline__ int row_of(const KvBatchDev &b, int s) { return b.row_start ? ld_plain(b.row_start + s) : s; }

struct SeqInfo {
    int past, row0, n;
};

// Sequence s of the batch; false where its entries are out of range.
__device__ __forceinline__ bool seq_info(const KvBatchDev &b, int s, SeqInfo &q)
{
    q.past = ld_plain(b.past + s);
    q.row0 = row_of(b, s);
    const int end = row_of(b, s + 1);
    q.n = end - q.row0;
    return q.row0 >= 0 && end >= q.row0 && end <= b.T && q.n <= b.max_new && q.past >= 0 &&
           q.past <= INT_MAX - 4096 - q.n;
}

// The same against a cache: the slot exists and its table holds the sequence's tokens.
__device__ __forceinline__ bool seq_in_cache(const KvCacheDev &c, const KvBatchDev &b, int s, const SeqInfo &q, int &slot)
{
    slot = b.slot ? ld_plain(b.slot + s) : s;
    return slot >= 0 && slot < c.n_slots &&
           ((int64_t)q.past + q.n + kKvBlock - 1) / kKvBlock <= ((int64_t)c.table_stride << c.page_shift);
}

// Block `blk` of a slot's sequence: index of (page, block in page) for head 0
// in units of blocks, with the head stride page_blocks; -1 for a bad page id.
__device__ __forceinline__ int64_t block_index(const KvCacheDev &c, int slot, int blk, int head)
{
    const int page = ld_plain(c.table + (int64_t)slot * c.table_stride + (blk >> c.page_shift));
    if (page < 0 || page >= c.n_pages) return -1;
    return (((int64_t)page * c.heads + head) << c.page_shift) + (blk & ((1 << c.page_shift) - 1));
}

// An angle less its whole quarter turns, in f64 (far positions lose nothing):
// the rest, in [-pi/4, pi/4], and the number of turns mod 4, which the low bits
// of angle * 2/pi + 1.5 * 2^52 hold: for angles up to 2^47 (MOE_ROPE_MAX_FREQ
// times a position), where the rounding of 2/pi (2^-53) moves the rest by 2 % at most.
__device__ __forceinline__ int quarter_turns(double &angle)
{
    const double t = fma(angle, 0.6366197723675814, 6755399441055744.0), n = t - 6755399441055744.0;
    angle = fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, angle));   // pi / 2 in two parts
    return __double2loint(t) & 3;
}

// cos and sin of an angle, in f32 from the rest on: the Taylor series up to x^10
// and x^9 (the next terms are below 2e-9).
__device__ __forceinline__ void turn_f32(double angle, float &c, float &s)
{
    const int k = quarter_turns(angle);
    const float x = (float)angle, z = x * x;
    float a = 1.0f / 362880.0f, b = -1.0f / 3628800.0f;
    b = fmaf(b, z, 1.0f / 40320.0f);
    a = fmaf(a, z, -1.0f / 5040.0f);
    b = fmaf(b, z, -1.0f / 720.0f);
    a = fmaf(a, z, 1.0f / 120.0f);
    b = fmaf(b, z, 1.0f / 24.0f);
    a = fmaf(a, z, -1.0f / 6.0f);
    b = fmaf(b, z, -0.5f);
    a = fmaf(a * z, x, x);
    b = fmaf(b, z, 1.0f);
    c = k & 1 ? a : b;
    s = k & 1 ? b : a;
    if (k == 1 || k == 2) c = -c;
    if (k >= 2) s = -s;
}

// Indices of pair i of a head's first R values.
__device__ __forceinline__ int2 rope_pair(const RopeDev &r, int i)
{
    return r.interleaved ? make_int2(2 * i, 2 * i + 1) : make_int2(i, i + r.R / 2);
}

// A warp: the sequence whose rows hold `row` (row_start ascending), -1 for none.
__device__ __forceinline__ int seq_of_row_warp(const KvBatchDev &b, int row, int lane)
{
    if (!b.row_start) return row < b.B ? row : -1;
    int n = 0;
    for (int s = lane; s < b.B; s += 32) n += ld_plain(b.row_start + s) <= row;
    return __reduce_add_sync(0xffffffffu, n) - 1;
}

// A norm's factor 1 / sqrt(mean square + eps), in f32, is good where the mean lies
// well inside f32's range: squares that underflow are then far below it, and
// none has overflowed.
__device__ __forceinline__ bool plain_root(float inv) { return inv > 0.0f && inv < 1e10f; }

// Where it does not (values above some 1e18 or below 1e-10, which only F32 and
// BF16 rows have): a head in LANES lanes, N values in each, is scaled by the power
// of two d that takes its largest value to [1, 2), and its factor formed anew, with
// eps d^2. Where that would be above 2^100 the squares are nothing beside it, and a
// d of 2^60 keeps it in range. The whole warp comes here; heads with !mine are left alone.
template <int N, int LANES>
__device__ __forceinline__ void scale_head(float (&v)[N], float &inv, double eps, bool mine)
{
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const int e = min(126, max(-126, (int)(__float_as_uint(amax) >> 23) - 127));
    float d = mine ? __int_as_float((127 - e) << 23) : 1.0f, add = (float)(eps * (double)d * (double)d);
    if (mine && add > 0x1p100f) {
        d = 0x1p60f;
        add = (float)(eps * 0x1p120);
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] *= d;
        ss = fmaf(v[i], v[i], ss);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (mine) inv = rsqrtf(ss * (1.0f / (N * LANES)) + add);
}

// A token's heads by one warp, 16 bytes of a head to a lane: the lane's values
// lie at the same place of every head, so its angles and norm weights are
// fetched once for the token and stay in registers.
template <int D, typename T>
struct HeadLanes {
    static constexpr int kVals = 16 / (int)sizeof(T);      // values of a lane
    static constexpr int kLanes = D / kVals;               // lanes of a head
    static constexpr int kHeads = 32 / kLanes;             // heads a warp takes at once
    static constexpr int kScratch = D;                     // floats of shared memory of a warp's own (see begin and turn)
    int lane, d0;               // first value of the lane
    int half, shift;            // R / 2; lanes to the partner's (0: not a whole number of lanes)
    bool inter, first, turns;   // interleaved pairs; the lane's values are first of their pairs; they turn
    float c[kVals], s[kVals];

    // Angles of a position: formed by the warp in y, each lane's kept.
    __device__ __forceinline__ void begin(const RopeDev &r, int pos, float *y, int lane_)
    {
        lane = lane_;
        d0 = lane % kLanes * kVals;
        half = r.R / 2;
        inter = r.interleaved || r.R == 2;
        shift = half % kVals ? 0 : half / kVals;
        first = d0 < half;
        turns = r.R > 0;
        if (!turns) return;
        float2 *turn = reinterpret_cast<float2 *>(y);
        for (int i = lane; i < half; i += 32) {
            float cs, sn;
            turn_f32((double)pos * r.inv[i], cs, sn);
            turn[i] = make_float2(cs * (float)r.mscale, sn * (float)r.mscale);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kVals; i++) {
            const int d = d0 + i;
            const float2 t = d < 2 * half ? turn[inter ? d / 2 : d < half ? d : d - half] : make_float2(1.0f, 0.0f);
            // a cos - b sin for the first of a pair, b cos + a sin for the second
            c[i] = t.x;
            s[i] = (inter ? d & 1 : d >= half) ? t.y : -t.y;
        }
        __syncwarp();
    }
    // The lane's values of a norm's weights.
    __device__ __forceinline__ void weights(const float *w, float (&v)[kVals]) const
    {
#pragma unroll
        for (int i = 0; i < kVals; i++) v[i] = w ? ld_plain(w + d0 + i) : 1.0f;
    }
    __device__ __forceinline__ float head_max(float v) const
    {
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
    // M heads at a time normed, in f32; the whole warp, each kLanes a head.
    template <int M>
    __device__ __forceinline__ void norms(float (&v)[M][kVals], const float (&w)[kVals], double eps) const
    {
        float inv[M];
        bool plain = true;
#pragma unroll
        for (int h = 0; h < M; h++) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < kVals; i++) ss = fmaf(v[h][i], v[h][i], ss);
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv[h] = rsqrtf(ss * (1.0f / D) + (float)eps);
            if (!std::is_same<T, __half>::value) plain &= plain_root(inv[h]);
        }
        // (one vote for all of them: with one for each they wait for one another)
        if (!__all_sync(0xffffffffu, plain))
#pragma unroll
            for (int h = 0; h < M; h++) scale_head<kVals, kLanes>(v[h], inv[h], eps, !plain_root(inv[h]));
#pragma unroll
        for (int h = 0; h < M; h++)
#pragma unroll
            for (int i = 0; i < kVals; i++) v[h][i] = v[h][i] * inv[h] * w[i];
    }
    // v turned, in f32; the whole warp.
    __device__ __forceinline__ void turn(float (&v)[kVals], float *y) const
    {
        if (!turns) return;
        float other[kVals];
        if (inter) {
#pragma unroll
            for (int i = 0; i < kVals; i++) other[i] = v[i ^ 1];
        } else if (shift) {
            const int from = first ? lane + shift : lane - shift;
#pragma unroll
            for (int i = 0; i < kVals; i++) other[i] = __shfl_sync(0xffffffffu, v[i], from & 31);
        } else {        // pairs that do not lie lane by lane: through shared memory, a head at a time
#pragma unroll
            for (int i = 0; i < kVals; i++) other[i] = 0.0f;
            for (int h = 0; h < kHeads; h++) {
                __syncwarp();
                if (lane / kLanes == h)
#pragma unroll
                    for (int i = 0; i < kVals; i++) y[d0 + i] = v[i];
                __syncwarp();
                if (lane / kLanes == h)
#pragma unroll
                    for (int i = 0; i < kVals; i++) {
                        const int d = d0 + i;
                        if (d < 2 * half) other[i] = y[d < half ? d + half : d - half];
                    }
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < kVals; i++)
            if (d0 + i < 2 * half) v[i] = v[i] * c[i] + other[i] * s[i];
    }
};

// One warp: a head row of D values, D / 32 consecutive ones in each lane's v,
// normed (w != nullptr) and rotated at position pos into y[D] (shared memory),
// all in f32 but the angles.
template <int D>
__device__ __forceinline__ void norm_rope_vals(float (&v)[D / 32], const float *w, const RopeDev &r, int pos, float *y, int lane)
{
    constexpr int N = D / 32;
    if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) ss = fmaf(v[i], v[i], ss);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        float inv = 1.0f / sqrtf(ss * (1.0f / D) + (float)r.eps);
        if (!plain_root(inv)) scale_head<N, 32>(v, inv, r.eps, true);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = v[i] * inv * ld_plain(w + lane * N + i);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; i++) y[lane * N + i] = v[i];
    __syncwarp();
    for (int i = lane; i < r.R / 2; i += 32) {
        float c, s;
        turn_f32((double)pos * r.inv[i], c, s);
        c *= (float)r.mscale;
        s *= (float)r.mscale;
        const int2 ab = rope_pair(r, i);
        const float a = y[ab.x], b = y[ab.y];
        y[ab.x] = a * c - b * s;
        y[ab.y] = b * c + a * s;
    }
    __syncwarp();
}

}  // namespace jmoe
