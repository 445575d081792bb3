// attn_rows.cu -- the row operators of the attention sublayer: norms of query
// and key heads with the rotation in the same pass, appending keys and values
// to the paged 8-bit cache, and reading cached rows back.
//
// All three touch each value once: bytes per call = rows in + rows out, and for
// the append the 8-bit blocks, their scales and the open blocks in f32. At a
// decode step's few rows they are bound by the launch and a chain of dependent
// loads (batch entry, page, rows). At prompts the norms and the append are bound
// by their instructions and the latencies between them, not yet by memory:
//   norms and rotation  11093 tokens of 14 + 2 heads of 64, bf16   23 us, 2.0 TB/s
//                       8 tokens of 32 + 4 heads of 128, f32       4 us
//   append              8483 tokens of 4 heads of 128, bf16        41 us
//                       64 tokens of 64 sequences, f32             7 us
#include <algorithm>

#include "attn.cuh"
#include "kernels.h"

namespace jmoe {
namespace {

constexpr int kRowWarps = 4;

// Norms and rotation: y = x / sqrt(mean x^2 + eps) w, then pairs turned by
// position * frequency. A warp takes a group of a token's heads, or all of them,
// kAhead loads of 16 bytes a lane under way before the first is worked on (four:
// 25.6 us where two take 23.5, the registers; five CTAs an SM 22.9, four 27.5).
constexpr int kAhead = 2;

template <int D, typename T>
__global__ void __launch_bounds__(kRowWarps * 32, sizeof(T) == 4 ? 8 : 5) qk_norm_rope_kernel(KvBatchDev b, const __grid_constant__ RopeDev rope,
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
    // groups of query heads, then of key heads; or, with one group, both in turn
    const int q_heads = in.q ? in.q_heads : 0, k_heads = in.k ? in.kv_heads : 0, gi = (int)(item - (int64_t)row * groups);
    const int q_groups = groups == 1 ? 0 : (q_heads + group - 1) / group;
    const int sub = lane / L::kLanes, d0 = lane % L::kLanes * L::kVals;
    bool is_q = groups == 1 ? q_heads > 0 : gi < q_groups;
    int h, head1;
    const T *src;
    T *dst;
    float v[kAhead][L::kVals];
    auto load = [&] {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int x = h + i * L::kHeads;
            if (x < head1) load_vals<L::kVals>(src + x * D, v[i]);
            else
#pragma unroll
                for (int k = 0; k < L::kVals; k++) v[i][k] = 0.0f;
        }
    };
    auto begin = [&] {
        const int heads = is_q ? q_heads : k_heads;
        h = groups == 1 ? sub : (is_q ? gi : gi - q_groups) * group + sub;
        head1 = groups == 1 ? heads : min(heads, h - sub + group);
        src = static_cast<const T *>(is_q ? in.q : in.k) + row * (is_q ? in.q_stride : in.k_stride) + d0;
        dst = static_cast<T *>(const_cast<void *>(is_q ? out.q : out.k)) + row * (is_q ? out.q_stride : out.k_stride) + d0;
        load();
    };
    begin();
    const int s = seq_of_row_warp(b, row, lane);
    SeqInfo q;
    if (s < 0 || !seq_info(b, s, q) || row < q.row0 || row >= q.row0 + q.n) return;
    L l;
    l.begin(rope, q.past + row - q.row0, s_y[warp], lane);
    for (;;) {
        const float *norm = is_q ? rope.q_norm : rope.k_norm;
        float w[L::kVals];
        l.weights(norm, w);
        for (;;) {
            if (norm) l.norms(v, w, rope.eps);
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                const int x = h + i * L::kHeads;
                if (x - sub >= head1) break;
                l.turn(v[i], s_y[warp]);
                if (x < head1) store_vals<L::kVals>(dst + x * D, v[i]);
            }
            h += kAhead * L::kHeads;
            if (h - sub >= head1) break;
            load();
        }
        if (groups > 1 || !is_q || !k_heads) break;
        is_q = false;
        begin();
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

// The same for the values of a lane at once: x inv + 1.5 2^23 holds the rounded
// quotient in its low bits, and the remainder shows whether it is the nearest
// (all but always); where one is not, or lies half way, or is not finite, the
// lane takes them one by one. by[i]: the byte in the low eight bits.
template <int M>
__device__ __forceinline__ void quantise_all(const float (&x)[M], float s, float inv, uint32_t (&by)[M])
{
    const float h = 0.5f * s;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < M; i++) {
        const float t = fmaf(x[i], inv, 12582912.0f), r = fmaf(-(t - 12582912.0f), s, x[i]);
        odd |= !(fabsf(r) < h);
        by[i] = __float_as_uint(t);
    }
    if (odd) {
#pragma unroll 1
        for (int i = 0; i < M; i++) {
            float v = x[0];
#pragma unroll
            for (int k = 1; k < M; k++) v = i == k ? x[k] : v;
            const uint32_t q = s > 0.0f ? (uint32_t)quantise(v, s, inv) : 0u;
#pragma unroll
            for (int k = 0; k < M; k++) by[k] = i == k ? q : by[k];
        }
    }
}

__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// cos and sin in f64, of the angle's rest the Taylor series up to x^14 and x^13
// (the next terms are below 2e-14; the keys are rounded to f32 afterwards). A
// third of the library function's work.
__device__ __forceinline__ void turn_f64(double angle, double &c, double &s)
{
    double x = angle;
    const int k = quarter_turns(x);
    const double z = x * x;
    double a = 1.0 / 6227020800.0, b = -1.0 / 87178291200.0;
    a = fma(a, z, -1.0 / 39916800.0);
    b = fma(b, z, 1.0 / 479001600.0);
    a = fma(a, z, 1.0 / 362880.0);
    b = fma(b, z, -1.0 / 3628800.0);
    a = fma(a, z, -1.0 / 5040.0);
    b = fma(b, z, 1.0 / 40320.0);
    a = fma(a, z, 1.0 / 120.0);
    b = fma(b, z, -1.0 / 720.0);
    a = fma(a, z, -1.0 / 6.0);
    b = fma(b, z, 1.0 / 24.0);
    a = fma(a * z, x, x);
    b = fma(b, z, -0.5);
    b = fma(b, z, 1.0);
    c = k & 1 ? a : b;
    s = k & 1 ? b : a;
    if (k == 1 || k == 2) c = -c;
    if (k >= 2) s = -s;
}

// 1 / sqrt in f64 by one Newton step from f32's, which has 22 bits: 2^-43.
__device__ __forceinline__ double root_f64(double x)
{
    if (!(x > 1e-30 && x < 1e30)) return 1.0 / sqrt(x);
    const double y = (double)rsqrtf((float)x);
    return y * fma(-0.5 * x * y, y, 1.5);
}

constexpr int kAppendWarps = 8, kPer = kKvBlock / kAppendWarps;      // tokens of a warp

// A number as the unevaluated sum of two f32, good to 2^-45 or so: the keys'
// arithmetic, at f32's rate (64 tokens of 64 sequences: 8.1 us in f64, 6.9 so).
struct Two {
    float h, l;
};
__device__ __forceinline__ Two two(double x)
{
    const float h = (float)x;
    return {h, (float)(x - (double)h)};
}
// a b + c d
__device__ __forceinline__ Two dot2(Two a, Two b, Two c, Two d)
{
    const float p = a.h * b.h, q = c.h * d.h;
    const float e = fmaf(a.l, b.h, fmaf(a.h, b.l, fmaf(a.h, b.h, -p)));
    const float f = fmaf(c.l, d.h, fmaf(c.h, d.l, fmaf(c.h, d.h, -q)));
    const float s = p + q, t = s - p;
    const float l = ((p - (s - t)) + (q - t)) + (e + f);
    const float h = s + l;
    return fabsf(s) < INFINITY ? Two{h, (s - h) + l} : Two{s, 0.0f};   // an infinite key stays one
}

// One CTA per (touched block, group of heads): warp w has the block's tokens
// 2 w and 2 w + 1, a lane D / 32 of their values (four CTAs an SM: 8483 tokens of
// 4 heads 41 us, three 44, two 50). The angles are formed once for
// the group, in f64 for every fourth token and from there by turns of the
// frequency.
//
// Flat block index u: `per` indices a sequence, where that many blocks hold
// max_new rows wherever they begin; with per = 0 sequence s owns the indices from
// row_start[s] / 16 + 2 s on, at least as many as the blocks its rows can touch
// (ceil((15 + n) / 16)), so no prefix sum is needed.
template <int D, typename T>
__global__ void __launch_bounds__(kAppendWarps * 32, 4)
    kv_append_kernel(KvCacheDev c, KvBatchDev b, const __grid_constant__ RopeDev rope, int use_rope, AttnRows rows, int group, int per, int *err)
{
    constexpr int N = D / 32;
    __shared__ __align__(16) float4 s_turn[kKvBlock][64];      // [token][place of a pair]: cos and sin, two f32 each
    __shared__ __align__(16) uint16_t s_v[2][kAppendWarps][D]; // a head's value bytes, a warp's two tokens together
    __shared__ float2 s_row[kAppendWarps][D];                  // a row of pairs that do not lie lane by lane
    __shared__ unsigned s_amax[2][2];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int head0 = blockIdx.y * group, head1 = min(c.heads, head0 + group), half = rope.R / 2;
    const int u = blockIdx.x;
    // pair p's place: a lane's pairs of a head lie apart, the lanes' side by side
    auto place = [](int p) { return (p & (N - 1)) * (64 / N) + p / N; };
    if (tid < 4) s_amax[tid / 2][tid % 2] = 0u;
    pdl_wait();
    pdl_trigger();
    int s = 0;
    if (per) {
        s = u / per;
    } else {      // the last whose indices start at or before u
#pragma unroll 4
        for (int i = lane; i < b.B; i += 32) s += row_of(b, i) / kKvBlock + 2 * i <= u;
        s = __reduce_add_sync(0xffffffffu, s) - 1;
    }
    if (u == 0 && head0 == 0)
        for (int i = tid; i < b.B; i += blockDim.x) {
            SeqInfo qi;
            int sl;
            if (!seq_info(b, i, qi) || !seq_in_cache(c, b, i, qi, sl)) kv_error(err);
        }
    SeqInfo q;
    int slot = -1;
    if (s < 0 || !seq_info(b, s, q) || !seq_in_cache(c, b, s, q, slot) || q.n == 0) return;
    const int total = q.past + q.n, blk0 = q.past / kKvBlock, blk_end = (total + kKvBlock - 1) / kKvBlock;
    const int blk1 = blk0 + (per ? u - s * per : u - (q.row0 / kKvBlock + 2 * s));
    if (blk1 < blk0 || blk1 >= blk_end) return;     // below: row_start out of order
    // The first block reads the open rows and the last writes them: where both
    // do, one CTA takes the two in turn.
    const bool both = blk_end - 1 > blk0 && q.past % kKvBlock && total % kKvBlock;
    if (both && blk1 == blk_end - 1) return;
    // a slot that an earlier sequence of the batch appends to: refused
    bool twice = false;
    if (b.slot)
        for (int i = tid; i < s; i += blockDim.x) twice |= ld_plain(b.slot + i) == slot && row_of(b, i + 1) > row_of(b, i);
    if (__syncthreads_or(twice)) {
        if (tid == 0) kv_error(err);
        return;
    }
    const bool inter = rope.interleaved || rope.R == 2;
    const int shift = half % N ? 0 : half / N, d0 = lane * N;
    float w[N];
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = use_rope && rope.k_norm ? ld_plain(rope.k_norm + d0 + i) : 1.0f;

    for (int blk = blk1;; blk = blk_end - 1) {
        const int first = blk * kKvBlock + kPer * warp;         // position of this warp's first token
        const int count = min(kKvBlock, total - blk * kKvBlock);
        const int new0 = max(0, q.past - first), new1 = min(kPer, total - first);   // this warp's new tokens: new0 .. new1 - 1
        float kx[kPer][N], vx[kPer][N];
        auto load = [&](int head) {
            const int64_t open = (((int64_t)slot * c.heads + head) * kKvBlock + kPer * warp) * D + d0;
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                if (j < new0 && j < new1) {
                    load_vals<N>(c.open_k + open + j * D, kx[j]);
                    load_vals<N>(c.open_v + open + j * D, vx[j]);
                } else if (j < new1) {
                    const int64_t row = q.row0 + first + j - q.past;
                    load_vals<N>(static_cast<const T *>(rows.k) + row * rows.k_stride + head * D + d0, kx[j]);
                    load_vals<N>(static_cast<const T *>(rows.v) + row * rows.v_stride + head * D + d0, vx[j]);
                } else {
#pragma unroll
                    for (int i = 0; i < N; i++) kx[j][i] = vx[j][i] = 0.0f;
                }
            }
        };
        load(head0);
        if (use_rope && half) {
            // thread (pair, four tokens): the first in f64, the others from it, new or not: a
            // token's angles have the same bits however its block was filled
            const int p = tid % 64, t0 = tid / 64 * 4, t1 = min(t0 + 4, count);
            if (p < half && t0 < t1 && blk * kKvBlock + t1 > q.past) {
                double cs, sn, cf, sf;
                turn_f64((double)(blk * kKvBlock + t0) * rope.inv[p], cs, sn);
                turn_f64(rope.inv[p], cf, sf);
                Two x = two(cs * rope.mscale), y = two(sn * rope.mscale);
                const Two c1 = two(cf), s1 = two(sf), minus{-s1.h, -s1.l};
                for (int t = t0;;) {
                    s_turn[t][place(p)] = make_float4(x.h, x.l, y.h, y.l);
                    if (++t >= t1) break;
                    const Two z = dot2(x, c1, y, minus);
                    y = dot2(y, c1, x, s1);
                    x = z;
                }
            }
            __syncthreads();
        }
        for (int head = head0; head < head1; head++) {
            const int par = (head - head0) & 1;
            const int64_t at = block_index(c, slot, blk, head);
            if (at < 0 && tid == 0) kv_error(err);
            if (use_rope) {
                // ---- the new keys. Each token's values are taken to [1, 2) by a power of
                // two; the two sums of squares are halved together: after one exchange a
                // lane carries one token, after four more its sum, and one root serves both.
                static_assert(kPer == 2, "two tokens a warp");
                Two inv[kPer];
                float down[kPer];
                if (rope.k_norm && new0 < new1) {
                    double ss[kPer];
                    int ex[kPer];
#pragma unroll
                    for (int j = 0; j < kPer; j++) {
                        float amax = 0.0f;
#pragma unroll
                        for (int i = 0; i < N; i++) amax = fmaxf(amax, fabsf(kx[j][i]));
                        ex[j] = min(126, max(-126, (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)) >> 23) - 127));
                        down[j] = __int_as_float((127 - ex[j]) << 23);
                        float h = 0.0f, l = 0.0f;
#pragma unroll
                        for (int i = 0; i < N; i++) {
                            const float x = kx[j][i] * down[j], p = x * x, t = h + p, b = t - h;
                            l += ((h - (t - b)) + (p - b)) + fmaf(x, x, -p);
                            h = t;
                        }
                        ss[j] = (double)h + (double)l;
                    }
                    const bool up = lane & 16;
                    double x = (up ? ss[1] : ss[0]) + __shfl_xor_sync(0xffffffffu, up ? ss[0] : ss[1], 16);
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                    const Two r = two(root_f64(x * (1.0 / D) + rope.eps * __hiloint2double((1023 - 2 * (up ? ex[1] : ex[0])) << 20, 0)));
#pragma unroll
                    for (int j = 0; j < kPer; j++) {
                        inv[j].h = __shfl_sync(0xffffffffu, r.h, j * 16);
                        inv[j].l = __shfl_sync(0xffffffffu, r.l, j * 16);
                    }
                }
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    if (j < new0 || j >= new1) continue;
                    Two x[N];
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        if (rope.k_norm) {
                            const float v = kx[j][i] * down[j], m = inv[j].h * w[i], ml = fmaf(inv[j].l, w[i], fmaf(inv[j].h, w[i], -m));
                            x[i].h = v * m;
                            x[i].l = fmaf(v, ml, fmaf(v, m, -x[i].h));
                        } else {
                            x[i] = {kx[j][i], 0.0f};
                        }
                    }
                    if (half) {
                        Two other[N];
                        if (inter) {
#pragma unroll
                            for (int i = 0; i < N; i++) other[i] = x[i ^ 1];
                        } else if (shift) {
                            const int from = (d0 < half ? lane + shift : lane - shift) & 31;
#pragma unroll
                            for (int i = 0; i < N; i++)
                                other[i] = {__shfl_sync(0xffffffffu, x[i].h, from), __shfl_sync(0xffffffffu, x[i].l, from)};
                        } else {
                            __syncwarp();
#pragma unroll
                            for (int i = 0; i < N; i++) s_row[warp][d0 + i] = make_float2(x[i].h, x[i].l);
                            __syncwarp();
#pragma unroll
                            for (int i = 0; i < N; i++) {
                                const int d = d0 + i;
                                const float2 o = d < 2 * half ? s_row[warp][d < half ? d + half : d - half] : make_float2(0.0f, 0.0f);
                                other[i] = {o.x, o.y};
                            }
                        }
#pragma unroll
                        for (int i = 0; i < N; i++) {
                            const int d = d0 + i;
                            if (d >= 2 * half) continue;
                            const float4 t = s_turn[kPer * warp + j][place(inter ? d / 2 : d < half ? d : d - half)];
                            // a cos - b sin for the first of a pair, b cos + a sin for the second
                            const bool second = inter ? d & 1 : d >= half;
                            x[i] = dot2(x[i], Two{t.x, t.y}, other[i], second ? Two{t.z, t.w} : Two{-t.z, -t.w});
                        }
                    }
#pragma unroll
                    for (int i = 0; i < N; i++) kx[j][i] = x[i].h + x[i].l;
                }
            }
            // ---- the block's scales
            float ka = 0.0f, va = 0.0f;
#pragma unroll
            for (int j = 0; j < kPer; j++)
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float x = fabsf(kx[j][i]), y = fabsf(vx[j][i]);
                    ka = x <= 3.402823466e38f ? fmaxf(ka, x) : ka;
                    va = y <= 3.402823466e38f ? fmaxf(va, y) : va;
                }
            const unsigned kb = __reduce_max_sync(0xffffffffu, __float_as_uint(ka)), vb = __reduce_max_sync(0xffffffffu, __float_as_uint(va));
            if (lane == 0) {
                atomicMax(&s_amax[par][0], kb);      // not negative: ordered as integers
                atomicMax(&s_amax[par][1], vb);
            }
            __syncthreads();
            float sc[2], inv[2];
#pragma unroll
            for (int m = 0; m < 2; m++) {
                const float amax = __uint_as_float(s_amax[par][m]);
                sc[m] = amax >= kKvTiny ? __fdiv_rn(amax, 127.0f) : 0.0f;
                inv[m] = sc[m] > 0.0f ? 1.0f / sc[m] : 0.0f;
            }
            if (tid < 2) s_amax[par ^ 1][tid] = 0u;  // for the next head: read last before this barrier's head
            // ---- bytes: keys [D/64][16][64] from the lanes, values [D][16] by way of shared memory
            {
                uint32_t by[kPer][N];
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    quantise_all<N>(kx[j], sc[0], inv[0], by[j]);
                    if (at >= 0) {
                        int8_t *k = c.k + at * kKvBlock * D + d0 / 64 * 1024 + (kPer * warp + j) * 64 + d0 % 64;
                        if constexpr (N == 4) *reinterpret_cast<uint32_t *>(k) = pack_bytes(by[j][0], by[j][1], by[j][2], by[j][3]);
                        else *reinterpret_cast<uint16_t *>(k) = (uint16_t)__byte_perm(by[j][0], by[j][1], 0x0040);
                    }
                }
#pragma unroll
                for (int j = 0; j < kPer; j++) quantise_all<N>(vx[j], sc[1], inv[1], by[j]);
                uint32_t vw[N / 2];
#pragma unroll
                for (int i = 0; i < N / 2; i++) vw[i] = pack_bytes(by[0][2 * i], by[1][2 * i], by[0][2 * i + 1], by[1][2 * i + 1]);
                if constexpr (N == 4) *reinterpret_cast<uint2 *>(&s_v[par][warp][d0]) = make_uint2(vw[0], vw[1]);
                else *reinterpret_cast<uint32_t *>(&s_v[par][warp][d0]) = vw[0];
            }
            // ---- the rows of the block left open
            if (count < kKvBlock) {
                const int64_t open = (((int64_t)slot * c.heads + head) * kKvBlock + kPer * warp) * D + d0;
#pragma unroll
                for (int j = 0; j < kPer; j++)
                    if (j >= new0 && j < new1) {
                        store_vals<N>(c.open_k + open + j * D, kx[j]);
                        store_vals<N>(c.open_v + open + j * D, vx[j]);
                    }
            }
            if (head + 1 < head1) load(head + 1);
            __syncthreads();
            if (at >= 0) {
                if (tid < 2) (tid ? c.v_scale : c.k_scale)[at] = tid ? sc[1] : sc[0];
                if (tid < D) {
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i] = s_v[par][2 * i][tid] | (uint32_t)s_v[par][2 * i + 1][tid] << 16;
                    reinterpret_cast<uint4 *>(c.v + at * kKvBlock * D)[tid] = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
        }
        if (!both || blk != blk0) break;
        __syncthreads();       // the open rows have been read, and the next block's maxima start at zero
        if (tid < 4) s_amax[tid / 2][tid % 2] = 0u;
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
    // Few warps: one load each, for the shortest time; where that would be many, a
    // warp a token, which forms its angles once. 32 + 4 heads of 128, bf16, us for
    // one load a warp and for a warp a token: 64 tokens 4.1 and 9.9, 256 tokens
    // (4608 warps) 8.9 and 10.1, 512 tokens 13.8 and 10.1, 4096 tokens 87 and 31.
    return by_type(in.act, D, [&](auto d, auto t) {
        using L = HeadLanes<decltype(d)::value, decltype(t)>;
        const int group = L::kHeads;
        int groups = (in.q ? (in.q_heads + group - 1) / group : 0) + (in.k ? (in.kv_heads + group - 1) / group : 0);
        if ((int64_t)b.T * groups > 6144) groups = 1;
        return launch_dependent(qk_norm_rope_kernel<decltype(d)::value, decltype(t)>,
                                dim3((unsigned)(((int64_t)b.T * groups + kRowWarps - 1) / kRowWarps)), dim3(kRowWarps * 32), 0, st, b,
                                rope, in, out, group, groups, err);
    });
}

cudaError_t launch_kv_append(const KvCacheDev &c, const KvBatchDev &b, const RopeDev *rope, const AttnRows &rows, int *err,
                             cudaStream_t st)
{
    // Few blocks: a head a CTA, for the shortest time. Many: two heads share the
    // angles. 4 heads of 128, bf16, a head a CTA and two: 1000 tokens 12.0 and
    // 15.7 us, 4000 tokens 20.4 and 20.4, 8483 tokens 44.6 and 43.2.
    // a sequence's rows touch at most so many blocks (1024 single tokens 37 us, searched for among 55)
    const int most = (kKvBlock - 1 + b.max_new + kKvBlock - 1) / kKvBlock, per = most <= 2 ? most : 0;
    const unsigned blocks = (unsigned)(per ? per * b.B : b.T / kKvBlock + 2 * b.B);
    const int group = blocks >= 512 ? std::min(c.heads, 2) : 1;
    const RopeDev none{};
    return by_type(rows.act, c.D, [&](auto d, auto t) {
        return launch_dependent(kv_append_kernel<decltype(d)::value, decltype(t)>, dim3(blocks, (c.heads + group - 1) / group),
                                dim3(kAppendWarps * 32), 0, st, c, b, rope ? *rope : none, (int)(rope != nullptr), rows, group, per,
                                err);
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
