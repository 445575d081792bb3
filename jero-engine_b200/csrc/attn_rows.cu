// attn_rows.cu -- the row operators of the attention sublayer: norms of query
// and key heads with the rotation in the same pass, appending keys and values
// to the paged 8-bit cache, and reading cached rows back.
//
// All three touch each value once and are bound by memory (or, for a decode
// step's few rows, by the launch): bytes per call = rows in + rows out, and for
// the append the 8-bit blocks, their scales and the open blocks in f32.
#include "attn.cuh"
#include "kernels.h"

namespace jmoe {
namespace {

constexpr int kRowWarps = 4;

// Norms and rotation: a warp takes a group of a token's heads, kAhead loads of
// 16 bytes a lane under way before the first is worked on.
constexpr int kAhead = 4;

template <int D, typename T>
__global__ void __launch_bounds__(kRowWarps * 32) qk_norm_rope_kernel(KvBatchDev b, const __grid_constant__ RopeDev rope,
                                                                      AttnRows in, AttnRows out, int group, int groups, int *err)
{
    using L = HeadLanes<D, T>;
    __shared__ __align__(16) float s_y[kRowWarps][L::kScratch];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0)
        for (int s = threadIdx.x; s < b.B; s += blockDim.x) {
            SeqInfo q;
            if (!seq_info(b, s, q)) kv_error(err);
        }
    const int64_t item = (int64_t)blockIdx.x * kRowWarps + warp;
    const int row = (int)(item / groups);
    if (row >= b.T) return;
    const int q_heads = in.q ? in.q_heads : 0, heads = q_heads + (in.k ? in.kv_heads : 0);
    int h = (int)(item - (int64_t)row * groups) * group + lane / L::kLanes;
    const int head1 = min(heads, h - lane / L::kLanes + group), d0 = lane % L::kLanes * L::kVals;
    const T *in_q = static_cast<const T *>(in.q) + row * in.q_stride + d0, *in_k = static_cast<const T *>(in.k) + row * in.k_stride + d0;
    T *out_q = static_cast<T *>(const_cast<void *>(out.q)) + row * out.q_stride + d0,
      *out_k = static_cast<T *>(const_cast<void *>(out.k)) + row * out.k_stride + d0;
    float v[kAhead][L::kVals];
    auto load = [&](int h) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int x = h + i * L::kHeads;
            if (x < head1) load_vals<L::kVals>(x < q_heads ? in_q + x * D : in_k + (x - q_heads) * D, v[i]);
            else
#pragma unroll
                for (int k = 0; k < L::kVals; k++) v[i][k] = 0.0f;
        }
    };
    load(h);
    const int s = seq_of_row_warp(b, row, lane);
    SeqInfo q;
    if (s < 0 || !seq_info(b, s, q) || row < q.row0 || row >= q.row0 + q.n) return;
    L l;
    l.begin(rope, q.past + row - q.row0, s_y[warp], lane);
    float wq[L::kVals], wk[L::kVals];
    l.weights(rope.q_norm, wq);
    l.weights(rope.k_norm, wk);
    for (;;) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int x = h + i * L::kHeads;
            if (x - lane / L::kLanes >= head1) break;
            const bool is_q = x < q_heads;
            float w[L::kVals];
#pragma unroll
            for (int k = 0; k < L::kVals; k++) w[k] = is_q ? wq[k] : wk[k];
            l.turn(v[i], __any_sync(0xffffffffu, (is_q ? rope.q_norm : rope.k_norm) != nullptr), w, (float)rope.eps, s_y[warp]);
            if (x < head1) store_vals<L::kVals>(is_q ? out_q + x * D : out_k + (x - q_heads) * D, v[i]);
        }
        h += kAhead * L::kHeads;
        if (h - lane / L::kLanes >= head1) break;
        load(h);
    }
}

// ------------------------------------------------------------------ append

// q = x / s rounded to nearest even, exactly: the quotient by the reciprocal
// may be one off, and the remainder x - q s, exact in f32 (x and q s are
// multiples of ulp(s), the remainder is below 2 s), says which way.
__device__ __forceinline__ int quantise(float x, float s, float inv)
{
    if (!(fabsf(x) <= 3.402823466e38f)) return isnan(x) ? 0 : (x > 0.0f ? 127 : -127);
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), h = 0.5f * s;
    if (fabsf(r) > h || (fabsf(r) == h && ((int)q & 1))) q += copysignf(1.0f, r);
    return (int)q;
}

// One CTA per (touched block, head). Flat block index u: sequence s owns the
// indices from row_start[s] / 16 + 2 s on, at least as many as the blocks its
// rows can touch (ceil((15 + n) / 16)), so no prefix sum is needed.
template <int D, typename T>
__global__ void __launch_bounds__(128) kv_append_kernel(KvCacheDev c, KvBatchDev b, const __grid_constant__ RopeDev rope,
                                                        int use_rope, AttnRows rows, int *err)
{
    __shared__ float s_x[2][kKvBlock][D];      // keys, values
    __shared__ double s_inv[kKvBlock];
    __shared__ float s_amax[2];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, head = blockIdx.y;
    const int u = blockIdx.x;
    int lo = 0, hi = b.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (row_of(b, mid) / kKvBlock + 2 * mid <= u) lo = mid;
        else hi = mid - 1;
    }
    const int s = lo;
    SeqInfo q;
    int slot = -1;
    const bool ok = seq_info(b, s, q) && seq_in_cache(c, b, s, q, slot);
    if (blockIdx.x == 0 && head == 0)
        for (int i = tid; i < b.B; i += blockDim.x) {
            SeqInfo qi;
            int sl;
            if (!seq_info(b, i, qi) || !seq_in_cache(c, b, i, qi, sl)) kv_error(err);
        }
    if (!ok || q.n == 0) return;
    const int total = q.past + q.n, blk0 = q.past / kKvBlock, blk_end = (total + kKvBlock - 1) / kKvBlock;
    const int blk1 = blk0 + (u - (q.row0 / kKvBlock + 2 * s));
    if (blk1 >= blk_end) return;
    // The first block reads the open rows and the last writes them: where both
    // do, one CTA takes the two in turn.
    const bool both = blk_end - 1 > blk0 && q.past % kKvBlock && total % kKvBlock;
    if (both && blk1 == blk_end - 1) return;
    // a slot that an earlier sequence of the batch appends to: refused
    if (b.slot) {
        bool twice = false;
        for (int i = tid; i < s; i += blockDim.x)
            twice |= ld_plain(b.slot + i) == slot && row_of(b, i + 1) > row_of(b, i);
        if (__syncthreads_or(twice)) {
            if (tid == 0) kv_error(err);
            return;
        }
    }
    constexpr int N = D / 32;
    const int64_t open = ((int64_t)slot * c.heads + head) * kKvBlock * D;
    for (int blk = blk1;; blk = blk_end - 1) {
        const int first = blk * kKvBlock;                       // position of the block's first token
        const int64_t at = block_index(c, slot, blk, head);
        if (at < 0 && tid == 0) kv_error(err);
        const int count = min(kKvBlock, total - first);
        for (int t = warp; t < kKvBlock; t += 4) {
            float kv[N], vv[N];
#pragma unroll
            for (int i = 0; i < N; i++) kv[i] = vv[i] = 0.0f;
            const int pos = first + t;
            double inv = 0.0;
            if (pos < q.past) {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    kv[i] = c.open_k[open + t * D + lane * N + i];
                    vv[i] = c.open_v[open + t * D + lane * N + i];
                }
            } else if (t < count) {
                const int64_t row = q.row0 + pos - q.past;
                load_vals<N>(static_cast<const T *>(rows.k) + row * rows.k_stride + head * D + lane * N, kv);
                load_vals<N>(static_cast<const T *>(rows.v) + row * rows.v_stride + head * D + lane * N, vv);
                if (use_rope && rope.k_norm) {
                    double ss = 0.0;
#pragma unroll
                    for (int i = 0; i < N; i++) ss = fma((double)kv[i], (double)kv[i], ss);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    inv = 1.0 / sqrt(ss / D + rope.eps);
                }
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                s_x[0][t][lane * N + i] = kv[i];
                s_x[1][t][lane * N + i] = vv[i];
            }
            if (lane == 0) s_inv[t] = inv;
        }
        if (tid < 2) s_amax[tid] = 0.0f;
        __syncthreads();
        if (use_rope) {
            // the new tokens' keys, in f64: pairs first, then the values that do not turn
            const int t0 = max(0, q.past - first), pairs = rope.R / 2, units = pairs + (D - rope.R);
            for (int e = tid; e < (count - t0) * units; e += blockDim.x) {
                const int t = t0 + e / units, i = e % units;
                float *x = s_x[0][t];
                const double inv = rope.k_norm ? s_inv[t] : 1.0;
                if (i < pairs) {
                    const int2 ab = rope_pair(rope, i);
                    double cs, sn;
                    sincos((double)(first + t) * rope.inv[i], &sn, &cs);
                    double va = x[ab.x] * inv, vb = x[ab.y] * inv;
                    if (rope.k_norm) {
                        va *= ld_plain(rope.k_norm + ab.x);
                        vb *= ld_plain(rope.k_norm + ab.y);
                    }
                    x[ab.x] = (float)((va * cs - vb * sn) * rope.mscale);
                    x[ab.y] = (float)((vb * cs + va * sn) * rope.mscale);
                } else if (rope.k_norm) {
                    const int d = rope.R + i - pairs;
                    x[d] = (float)(x[d] * inv * ld_plain(rope.k_norm + d));
                }
            }
            __syncthreads();
        }
        // scales
#pragma unroll
        for (int m = 0; m < 2; m++) {
            float a = 0.0f;
            for (int e = tid; e < kKvBlock * D; e += blockDim.x) {
                const float x = fabsf((&s_x[m][0][0])[e]);
                if (x <= 3.402823466e38f) a = fmaxf(a, x);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            if (lane == 0) atomicMax(reinterpret_cast<int *>(&s_amax[m]), __float_as_int(a));   // a >= 0: ordered as integers
        }
        __syncthreads();
        if (at >= 0) {
            float sc[2], inv[2];
#pragma unroll
            for (int m = 0; m < 2; m++) {
                sc[m] = s_amax[m] >= kKvTiny ? __fdiv_rn(s_amax[m], 127.0f) : 0.0f;
                inv[m] = sc[m] > 0.0f ? 1.0f / sc[m] : 0.0f;
            }
            if (tid < 2) (tid ? c.v_scale : c.k_scale)[at] = sc[tid];
            // four bytes at a time: keys [D/64][16][64], values [D][16]
            uint32_t *ko = reinterpret_cast<uint32_t *>(c.k + at * kKvBlock * D);
            uint32_t *vo = reinterpret_cast<uint32_t *>(c.v + at * kKvBlock * D);
            for (int e = tid; e < kKvBlock * D / 4; e += blockDim.x) {
                const int slab = e / (kKvBlock * 16), t = e / 16 % kKvBlock, d = slab * 64 + e % 16 * 4;
                uint32_t w = 0, z = 0;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    w |= (uint32_t)(uint8_t)(sc[0] > 0.0f ? quantise(s_x[0][t][d + i], sc[0], inv[0]) : 0) << (8 * i);
                const int vd = e / 4, vt = e % 4 * 4;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    z |= (uint32_t)(uint8_t)(sc[1] > 0.0f ? quantise(s_x[1][vt + i][vd], sc[1], inv[1]) : 0) << (8 * i);
                ko[e] = w;
                vo[e] = z;
            }
        }
        // the rows of the block left open
        if (count < kKvBlock)
            for (int t = warp; t < count; t += 4)
                if (first + t >= q.past)
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        c.open_k[open + t * D + lane * N + i] = s_x[0][t][lane * N + i];
                        c.open_v[open + t * D + lane * N + i] = s_x[1][t][lane * N + i];
                    }
        if (!both || blk != blk0) break;
        __syncthreads();
    }
}

// -------------------------------------------------------------------- read

// One CTA per row: a warp a head, keys and values at a time. A value's 16 tokens
// lie together, so a row's bytes are D sectors of which it needs one byte each:
// rows that follow one another find them in the caches.
template <int D, typename T>
__global__ void __launch_bounds__(kRowWarps * 32) kv_read_kernel(KvCacheDev c, KvBatchDev b, AttnRows out, int *err)
{
    constexpr int N = D / 32;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = blockIdx.x;
    pdl_wait();
    pdl_trigger();
    if (row == 0)
        for (int s = threadIdx.x; s < b.B; s += blockDim.x) {
            SeqInfo q;
            int slot;
            if (!seq_info(b, s, q) || !seq_in_cache(c, b, s, q, slot)) kv_error(err);
        }
    const int s = seq_of_row_warp(b, row, lane);
    if (s < 0) return;
    SeqInfo q;
    int slot;
    if (!seq_info(b, s, q) || row < q.row0 || row >= q.row0 + q.n || !seq_in_cache(c, b, s, q, slot)) return;
    const int pos = q.past + row - q.row0, t = pos % kKvBlock;
    for (int head = warp; head < c.heads; head += kRowWarps) {
        const int64_t at = block_index(c, slot, pos / kKvBlock, head);
        if (at < 0 && lane == 0) kv_error(err);
        float kv[N], vv[N];
#pragma unroll
        for (int i = 0; i < N; i++) kv[i] = vv[i] = 0.0f;
        if (at >= 0) {
            const float ks = ld_plain(c.k_scale + at), vs = ld_plain(c.v_scale + at);
            const int8_t *k = c.k + at * kKvBlock * D + lane * N / 64 * 1024 + t * 64 + lane * N % 64;
            const int8_t *v = c.v + at * kKvBlock * D + lane * N * kKvBlock + t;
#pragma unroll
            for (int i = 0; i < N; i++) {
                kv[i] = ks * (float)k[i];
                vv[i] = vs * (float)v[i * kKvBlock];
            }
        }
        if (out.k) store_vals<N>(static_cast<T *>(const_cast<void *>(out.k)) + row * out.k_stride + head * D + lane * N, kv);
        if (out.v) store_vals<N>(static_cast<T *>(const_cast<void *>(out.v)) + row * out.v_stride + head * D + lane * N, vv);
    }
}

template <typename F>
cudaError_t by_type(int act, int D, F &&f)
{
    switch (act) {
    case MOE_ACT_F32: return D == 64 ? f(std::integral_constant<int, 64>{}, 0.0f) : f(std::integral_constant<int, 128>{}, 0.0f);
    case MOE_ACT_F16:
        return D == 64 ? f(std::integral_constant<int, 64>{}, __half{}) : f(std::integral_constant<int, 128>{}, __half{});
    default:
        return D == 64 ? f(std::integral_constant<int, 64>{}, __nv_bfloat16{})
                       : f(std::integral_constant<int, 128>{}, __nv_bfloat16{});
    }
}

}  // namespace

cudaError_t launch_qk_norm_rope(const KvBatchDev &b, const RopeDev &rope, const AttnRows &in, const AttnRows &out, int D,
                                int *err, cudaStream_t st)
{
    // few tokens: one load a warp, for the shortest time; many: a token's heads up to four loads' worth a turn
    const int heads = (in.q ? in.q_heads : 0) + (in.k ? in.kv_heads : 0);
    return by_type(in.act, D, [&](auto d, auto t) {
        using L = HeadLanes<decltype(d)::value, decltype(t)>;
        const int group = b.T <= 512 ? L::kHeads : kAhead * L::kHeads * 2, groups = (heads + group - 1) / group;
        return launch_dependent(qk_norm_rope_kernel<decltype(d)::value, decltype(t)>,
                                dim3((unsigned)(((int64_t)b.T * groups + kRowWarps - 1) / kRowWarps)), dim3(kRowWarps * 32), 0, st, b,
                                rope, in, out, group, groups, err);
    });
}

cudaError_t launch_kv_append(const KvCacheDev &c, const KvBatchDev &b, const RopeDev *rope, const AttnRows &rows, int *err,
                             cudaStream_t st)
{
    const dim3 grid((unsigned)(b.T / kKvBlock + 2 * b.B), (unsigned)c.heads);
    const RopeDev none{};
    return by_type(rows.act, c.D, [&](auto d, auto t) {
        kv_append_kernel<decltype(d)::value, decltype(t)><<<grid, 128, 0, st>>>(c, b, rope ? *rope : none, rope != nullptr,
                                                                               rows, err);
        return cudaGetLastError();
    });
}

cudaError_t launch_kv_read(const KvCacheDev &c, const KvBatchDev &b, const AttnRows &out, int *err, cudaStream_t st)
{
    return by_type(out.act, c.D, [&](auto d, auto t) {
        return launch_dependent(kv_read_kernel<decltype(d)::value, decltype(t)>, dim3(b.T), dim3(kRowWarps * 32), 0, st, c, b, out,
                                err);
    });
}

}  // namespace jmoe
