// attn_tiles.cu -- attention of prompts over the paged 8-bit cache on tcgen05:
// the mathematics of attn.cu for row chunks of 256 (tokens of a sequence times
// the query heads of one key head), two tiles of 128 rows a CTA.
//
// Per 128 cached tokens: four conversion warps turn the cache's bytes into f16
// operands in shared memory (exact; K-major, 128-byte swizzle: a value block
// lies as [D][16 tokens] in the cache, so neither keys nor values are
// transposed), one thread issues S = Q K^T (tcgen05.mma, M 128, N 128) and
// O += P V (N = D, the weights P read from TMEM), and a warpgroup for each row
// tile does its softmax: a thread holds a row. TMEM: S0, S1 (128 columns each,
// P over S once S has been read) and O0, O1 (D columns each).
//
// The sums O are scaled down only when a row's maximum has grown by more than
// 2^8 since they were last: the weights then reach 2^8 instead of 1, which f16
// holds as exactly. With F32 rows queries and weights are split in two f16
// halves, each half a product of its own: 22 bits for twice the products.
//
// Bound by the tensor cores and, as much, by the exponentials: 128 x 128
// weights take 1024 cycles of the 16 a cycle that the SM gives, the two
// products of a row tile 2 x 512.
#include <algorithm>
#include <type_traits>

#include "attn.cuh"
#include "kernels.h"
#include "tc_common.cuh"

namespace jmoe {
namespace {

constexpr int kRowsTile = 128, kRowsItem = 256, kKv = 128;
constexpr int kSoftWarps = 8, kConvWarps = 4, kMmaWarp = kSoftWarps + kConvWarps;
constexpr int kThreads = 16 * 32;    // whole warpgroups: three warps beside the product warp only lend registers
// Registers a thread after the split: 2 x 152 + 2 x 104 = 4 x the launch's 128.
constexpr int kSoftRegs = 152, kOtherRegs = 104;
constexpr float kNoScaleLog2 = -80.0f;
constexpr int kCubic = 4;            // one pair of weights in this many takes the cubic
constexpr float kLazy = 8.0f;        // growth of a row's maximum (log2) that its sums are left unscaled for

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

// Two f32 at a time.
using f32x2 = uint64_t;
__device__ __forceinline__ f32x2 pair(float a, float b)
{
    f32x2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 unpair(f32x2 a)
{
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(a));
    return v;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 2^x of a pair on the multiply-add pipes, which have room where the
// exponential's own is full: x = n + f with n its nearest integer (the low bits
// of x + 1.5 * 2^23), and a cubic for 2^f on [-1/2, 1/2] with the smallest
// largest relative error, 7.5e-5 (2^-13.7), below the 2^-12 that the weights'
// rounding to f16 brings.
__device__ __forceinline__ float2 ex2_cubic(f32x2 x)
{
    float2 v = unpair(x);
    v.x = fmaxf(v.x, -126.0f);
    v.y = fmaxf(v.y, -126.0f);
    x = pair(v.x, v.y);
    const f32x2 t = add2(x, pair(12582912.0f, 12582912.0f));
    const f32x2 f = fma2(add2(t, pair(-12582912.0f, -12582912.0f)), pair(-1.0f, -1.0f), x);
    f32x2 y = fma2(f, pair(0.0551716685f, 0.0551716685f), pair(0.2426111251f, 0.2426111251f));
    y = fma2(y, f, pair(0.6932609677f, 0.6932609677f));
    y = fma2(y, f, pair(0.9999280572f, 0.9999280572f));
    const float2 n = unpair(t), z = unpair(y);
    return make_float2(__int_as_float(__float_as_int(z.x) + (__float_as_int(n.x) << 23)),
                       __int_as_float(__float_as_int(z.y) + (__float_as_int(n.y) << 23)));
}

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// A bounded wait of a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *err)
{
    return __all_sync(0xffffffffu, tc_spin_wait(bar, parity, abort_flag, err));
}

// ------------------------------------------------------------ the item list

// Chunk c of sequence b is entry row_start[b] * g / 256 + b + c of the list: at
// least as many entries per sequence as it has chunks, without a prefix sum.
__device__ __forceinline__ int first_entry(const KvBatchDev &b, int s, int g) { return row_of(b, s) * g / kRowsItem + s; }

struct Item {
    SeqInfo q;
    int slot, tok, rem, rows, pos_first, pos_last, tile0, tiles;
};

// Entry `e` of the list, by a whole warp; false where it holds no chunk (or one
// of a sequence with at most few_rows rows, which attn.cu takes).
__device__ __forceinline__ bool find_item(const AttnParams &p, int e, int g, int few_rows, int lane, Item &it)
{
    int n = 0;
    for (int s = lane; s < p.b.B; s += 32) n += first_entry(p.b, s, g) <= e;
    const int s = __reduce_add_sync(0xffffffffu, n) - 1;
    if (s < 0) return false;
    const bool ok = seq_info(p.b, s, it.q) && seq_in_cache(p.c, p.b, s, it.q, it.slot);
    if (!ok) return false;
    const int first = (e - first_entry(p.b, s, g)) * kRowsItem, rows = it.q.n * g;
    if (first >= rows || rows <= few_rows) return false;
    it.tok = first / g;
    it.rem = first - it.tok * g;
    it.rows = min(kRowsItem, rows - first);
    it.pos_first = it.q.past + it.tok;
    it.pos_last = it.pos_first + (it.rem + it.rows - 1) / g;
    it.tile0 = p.window ? max(0, it.pos_first - p.window + 1) / kKv : 0;
    it.tiles = it.pos_last / kKv + 1 - it.tile0;
    return true;
}

template <int D, bool SPLIT>
struct TileShape {
    static constexpr int kSlabs = D / 64;
    static constexpr int kQTile = (SPLIT ? 2 : 1) * kSlabs * kRowsTile * 128;   // bytes of a row tile's queries
    static constexpr int kBufs = SPLIT ? 1 : 2;
    static constexpr int kOperand = kKv * D * 2;                                // bytes of a key or value operand
    static constexpr int kStage = kKv * D;                                      // ... and of the cache's bytes behind it
    static constexpr int kSmem = 2 * kQTile + 2 * kBufs * kOperand + 2 * kStage;
    static constexpr size_t kImage = 2 * kQTile;                                // an item's queries in the workspace
};

// ------------------------------------------------------------ queries

// Queries as the item's shared-memory image: f16 rows scaled by a power of two
// that takes the largest value to [2^14, 2^15), and the factor that a row's
// logits then need. One CTA per token, heads over its warps.
template <int D, typename T, bool SPLIT>
__global__ void __launch_bounds__(128) query_tiles_kernel(const __grid_constant__ AttnParams p, int entry0, int entry1,
                                                          int few_rows, uint8_t *images, float *factors)
{
    using Sh = TileShape<D, SPLIT>;
    constexpr int N = D / 32;
    __shared__ float2 s_turn[D / 2];
    __shared__ float s_y[4][D];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, row = blockIdx.x;
    pdl_wait();
    pdl_trigger();
    const int g = p.rows.q_heads / p.c.heads;
    const int s = seq_of_row_warp(p.b, row, lane);
    SeqInfo q;
    if (s < 0 || !seq_info(p.b, s, q) || row < q.row0 || row >= q.row0 + q.n || q.n * g <= few_rows) return;
    const int tok = row - q.row0, entry = first_entry(p.b, s, g);
    if (entry + (tok * g + g - 1) / kRowsItem < entry0 || entry + tok * g / kRowsItem >= entry1) return;
    if (p.use_rope) {
        rope_table(p.rope, q.past + tok, s_turn, tid, 128);
        __syncthreads();
    }
    for (int h = blockIdx.y * 4 + warp; h < p.rows.q_heads; h += gridDim.y * 4) {
        const int kvh = h / g, flat = tok * g + h - kvh * g, e = entry + flat / kRowsItem, r = flat % kRowsItem;
        if (e < entry0 || e >= entry1) continue;
        float v[N];
        load_vals<N>(static_cast<const T *>(p.rows.q) + (int64_t)row * p.rows.q_stride + h * D + lane * N, v);
        if (p.use_rope) turn_head<D>(v, p.rope.q_norm, p.rope, s_turn, s_y[warp], lane);
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) amax = fmaxf(amax, fabsf(v[i]));
        const int x = max(-112, (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)) >> 23) - 127);
        float up = __int_as_float((14 - x + 127) << 23);
        const int64_t image = (int64_t)(e - entry0) * p.c.heads + kvh;
        if (lane == 0) factors[image * kRowsItem + r] = __int_as_float((x - 14 + 127) << 23) * fabsf(p.scale) * 1.4426950408889634f;
        if (p.scale < 0.0f) up = -up;      // the factors are not negative: maxima stay maxima
        uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const float a = v[2 * i] * up, b = v[2 * i + 1] * up;
            hi[i] = pack_f16(a, b);
            if constexpr (SPLIT) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[i]));
                lo[i] = pack_f16(a - f.x, b - f.y);
            }
        }
        const int d = lane * N, rt = r % kRowsTile;
        uint8_t *dst = images + image * Sh::kImage + r / kRowsTile * Sh::kQTile + d / 64 * (kRowsTile * 128) + rt * 128 +
                       (((d % 64) / 8) ^ (rt & 7)) * 16 + d % 8 * 2;
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            reinterpret_cast<uint32_t *>(dst)[i] = hi[i];
            if constexpr (SPLIT) reinterpret_cast<uint32_t *>(dst + Sh::kQTile / 2)[i] = lo[i];
        }
    }
}

// ------------------------------------------------------------ attention

template <int D, typename T, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    attend_tiles_kernel(const __grid_constant__ AttnParams p, int entry0, int entry1, int few_rows, const uint8_t *images,
                        const float *factors)
{
    using Sh = TileShape<D, SPLIT>;
    constexpr int NB = Sh::kBufs, SL = Sh::kSlabs;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t q_full, q_free, k_full[NB], k_empty[NB], v_full[NB], v_empty[NB], st_full[2], s_full[2],
        p_full[2], o_done[2], drained;
    __shared__ __align__(16) float s_sk[4][8], s_lsv[4][8], s_isv[4][8];
    __shared__ uint32_t s_ok[4];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    uint8_t *sm_q = smem, *sm_k = sm_q + 2 * Sh::kQTile, *sm_v = sm_k + NB * Sh::kOperand, *sm_st = sm_v + NB * Sh::kOperand;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int g = p.rows.q_heads / p.c.heads;

    if (tid == 0) {
        mbar_init(&q_full, 1);
        mbar_init(&q_free, 1);
        mbar_init(&drained, 1);
        for (int i = 0; i < NB; i++) {
            mbar_init(&k_full[i], kConvWarps);
            mbar_init(&v_full[i], kConvWarps);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&st_full[i], 1);
            mbar_init(&s_full[i], 2);      // the products' end, and what the product thread has seen
            mbar_init(&p_full[i], 4);
            mbar_init(&o_done[i], 1);
        }
        s_abort = 0;
        fence_barrier_init();
    }
    if (warp == kMmaWarp) tmem_alloc(&s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_wait();
    pdl_trigger();
    volatile int *abort_flag = &s_abort;

    // Items go to the CTAs there and back, longest first: neighbours' lengths differ little.
    const int G = gridDim.x, entries = entry1 - entry0, total = entries * p.c.heads;
    Item it;
    int head = 0, image = 0;
    auto item = [&](int j) -> int {       // 1: an item, 0: none here, -1: the end
        if ((int64_t)j * G >= total) return -1;
        const int64_t u = (j & 1) ? (int64_t)(j + 1) * G - 1 - (int)blockIdx.x : (int64_t)j * G + (int)blockIdx.x;
        if (u >= total) return 0;
        const int e = (int)(u / p.c.heads);
        head = (int)(u - (int64_t)e * p.c.heads);
        image = (entries - 1 - e) * p.c.heads + head;
        return find_item(p, entry1 - 1 - e, g, few_rows, lane, it) ? 1 : 0;
    };

    if (warp >= kSoftWarps && warp < kMmaWarp) {
        // ============ conversion: cache bytes -> f16 operands. (After a wait that ran out
        // the warps go on through their barriers: every wait then gives up at once.)
        regs_down<kOtherRegs>();
        const int ct = tid - kSoftWarps * 32, cw = warp - kSoftWarps;
        fence_proxy_async_global();       // the cache as an append before this left it, to the bulk copies
        uint32_t done = 0, staged = 0;
        bool ok = true;
        for (int j = 0, have; (have = item(j)) >= 0; j++) {
            if (!have) continue;
            int64_t at = -1;
            float sk = 0.0f, sv = 0.0f;
            // Warp 0: asks for tile t's keys (0) or values (1); lanes 0 .. 7 look after a block each.
            auto stage = [&](int which, int t) {
                if (which == 0) {
                    at = -1;
                    const int blk = (it.tile0 + t) * (kKv / kKvBlock) + lane, first = blk * kKvBlock;
                    if (lane < 8 && first <= it.pos_last && (!p.window || first + kKvBlock - 1 > it.pos_first - p.window)) {
                        at = block_index(p.c, it.slot, blk, head);
                        if (at < 0) kv_error(p.err);
                    }
                }
                const unsigned n = __popc(__ballot_sync(0xffffffffu, at >= 0));
                if (lane == 0) mbar_arrive_expect_tx(&st_full[which], n * (kKvBlock * D));
                __syncwarp();
                if (at >= 0)
                    bulk_load(smem_addr(sm_st + which * Sh::kStage + lane * kKvBlock * D),
                              (which ? p.c.v : p.c.k) + at * (kKvBlock * D), kKvBlock * D, &st_full[which]);
                if (which == 0) {
                    sk = sv = 0.0f;
                    if (at >= 0) {
                        sk = __ldg(p.c.k_scale + at);
                        sv = __ldg(p.c.v_scale + at);
                    }
                }
            };
            if (cw == 0) {
                stage(0, 0);
                stage(1, 0);
            }
            staged = done + 1;
            for (int t = 0; t < it.tiles; t++, done++) {
                const int buf = done % NB;
                const uint32_t ph = (done / NB) & 1;
                // ---- keys: rows are tokens, 64 values a slab
                ok &= warp_wait(&st_full[0], done & 1, abort_flag, p.err);
                ok &= warp_wait(&k_empty[buf], ph ^ 1, abort_flag, p.err);
                if (cw == 0) {
                    const int r = done & 3;
                    const unsigned live = __ballot_sync(0xffffffffu, at >= 0);
                    if (lane < 8) {
                        const float ls = sv > 0.0f ? lg2(sv) : kNoScaleLog2;
                        s_sk[r][lane] = sk;
                        s_lsv[r][lane] = ls;
                        s_isv[r][lane] = ex2(-ls);
                    }
                    if (lane == 0) s_ok[r] = live & 0xFFu;
                }
                {
                    const int tb = ct % D, sub = ct / D, slab = tb / 64, tok = tb % 64 / 4, c = tb % 4 * 2;
                    uint8_t *dst = sm_k + buf * Sh::kOperand + slab * (kKv * 128) + tok * 128;
                    const uint32_t src = smem_addr(sm_st) + ct * 16, x = smem_addr(dst) + ((c ^ (tok & 7)) * 16),
                                   y = smem_addr(dst) + (((c + 1) ^ (tok & 7)) * 16);
                    uint4 in[8 * D / 128];
#pragma unroll
                    for (int i = 0; i < 8 * D / 128; i++) in[i] = lds128(src + i * 2048);
#pragma unroll
                    for (int i = 0; i < 8 * D / 128; i++) {
                        const uint4 w = in[i];
                        uint4 a, b;
                        bytes_f16(w.x, a.x, a.y);
                        bytes_f16(w.y, a.z, a.w);
                        bytes_f16(w.z, b.x, b.y);
                        bytes_f16(w.w, b.z, b.w);
                        const uint32_t o = (i * (128 / D) + sub) * (kKvBlock * 128);
                        sts128(x + o, a);
                        sts128(y + o, b);
                    }
                }
                fence_async_smem();
                named_bar(1, kConvWarps * 32);       // every warp has read the staged bytes and written its part
                if (lane == 0) mbar_arrive(&k_full[buf]);
                if (cw == 0 && t + 1 < it.tiles) stage(0, t + 1);
                // ---- values: rows are the head's values, 64 tokens a slab
                ok &= warp_wait(&st_full[1], done & 1, abort_flag, p.err);
                ok &= warp_wait(&v_empty[buf], ph ^ 1, abort_flag, p.err);
                {
                    const int d = ct % D, sub = ct / D;
                    uint8_t *dst = sm_v + buf * Sh::kOperand + d * 128;
                    const uint32_t src = smem_addr(sm_st + Sh::kStage) + ct * 16, base = smem_addr(dst);
                    uint4 in[8 * D / 128];
#pragma unroll
                    for (int i = 0; i < 8 * D / 128; i++) in[i] = lds128(src + i * 2048);
#pragma unroll
                    for (int i = 0; i < 8 * D / 128; i++) {
                        const uint4 w = in[i];
                        uint4 a, b;
                        bytes_f16(w.x, a.x, a.y);
                        bytes_f16(w.y, a.z, a.w);
                        bytes_f16(w.z, b.x, b.y);
                        bytes_f16(w.w, b.z, b.w);
                        const int blk = i * (128 / D) + sub, c = blk % 4 * 2;
                        const uint32_t o = base + blk / 4 * (D * 128);
                        sts128(o + ((c ^ (d & 7)) * 16), a);
                        sts128(o + (((c + 1) ^ (d & 7)) * 16), b);
                    }
                }
                fence_async_smem();
                named_bar(1, kConvWarps * 32);
                if (lane == 0) mbar_arrive(&v_full[buf]);
                if (cw == 0 && t + 1 < it.tiles) {
                    stage(1, t + 1);
                    staged = done + 2;
                }
            }
        }
        if (!ok && cw == 0)        // copies may still be in flight
            for (int w = 0; w < 2; w++)
                if (staged) drain_wait(&st_full[w], (staged - 1) & 1);
    } else if (warp >= kMmaWarp) {
        regs_down<kOtherRegs>();
        if (warp == kMmaWarp) {
            // ============ products
            fence_proxy_async_global();       // the queries as the kernel before left them
            const uint32_t id_s = (1u << 4) | ((uint32_t)(kKv >> 3) << 17) | ((uint32_t)(kRowsTile >> 4) << 24);
            const uint32_t id_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRowsTile >> 4) << 24);
            const uint64_t dq = umma_desc_sw128(smem_addr(sm_q)), dk = umma_desc_sw128(smem_addr(sm_k)), dv = umma_desc_sw128(smem_addr(sm_v));
            uint32_t done = 0, items = 0, turns[2] = {0, 0};     // tiles and items of the CTA, tiles of each row tile
            bool ok = true, loading = false;
            for (int j = 0, have; ok && (have = item(j)) >= 0; j++) {
                if (!have) continue;
                if (lane == 0) {
                    const int mt = it.rows > kRowsTile ? 2 : 1;
                    auto scores = [&](int i, int buf) {
                        uint32_t acc = 0;
                        mbar_arrive(&s_full[i]);      // with the scales that the keys came with
#pragma unroll
                        for (int half = 0; half < (SPLIT ? 2 : 1); half++)
#pragma unroll
                            for (int s = 0; s < SL; s++)
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    tc_mma_f16(tmem + i * kKv, dq + ((i * Sh::kQTile + (half * SL + s) * kRowsTile * 128) >> 4) + 2 * k,
                                               dk + ((buf * Sh::kOperand + s * kKv * 128) >> 4) + 2 * k, id_s, acc);
                                    acc = 1;
                                }
                        tc_commit(&s_full[i]);
                    };
                    auto sums = [&](int i, int buf, uint32_t acc) {
#pragma unroll
                        for (int k = 0; k < 8; k++)
#pragma unroll
                            for (int half = 0; half < (SPLIT ? 2 : 1); half++) {
                                tc_mma_f16_ts(tmem + 2 * kKv + i * D, tmem + i * kKv + k / 2 * 32 + k % 2 * 8 + half * 16,
                                              dv + ((buf * Sh::kOperand + k / 4 * D * 128) >> 4) + 2 * (k % 4), id_o, acc);
                                acc = 1;
                            }
                    };
                    do {
                        if (items && !(ok = tc_spin_wait(&q_free, (items - 1) & 1, abort_flag, p.err))) break;
                        mbar_arrive_expect_tx(&q_full, mt * Sh::kQTile);
                        bulk_load(smem_addr(sm_q), images + (int64_t)image * Sh::kImage, mt * Sh::kQTile, &q_full);
                        loading = true;
                        if (!(ok = tc_spin_wait(&q_full, items & 1, abort_flag, p.err))) break;
                        loading = false;
                        if (!(ok = tc_spin_wait(&k_full[done % NB], (done / NB) & 1, abort_flag, p.err))) break;
                        tc_fence_after();
                        for (int i = 0; i < mt; i++) scores(i, done % NB);
                        tc_commit(&k_empty[done % NB]);
                        if (it.tiles == 1) tc_commit(&q_free);
                        for (int t = 0; t < it.tiles; t++, done++) {
                            const bool last = t + 1 == it.tiles;
                            const int buf = done % NB, nbuf = (done + 1) % NB;
                            if (!(ok = tc_spin_wait(&v_full[buf], (done / NB) & 1, abort_flag, p.err))) break;
                            for (int i = 0; i < mt; i++) {
                                const uint32_t turn = i ? turns[1]++ : turns[0]++;
                                if (!(ok = tc_spin_wait(&p_full[i], turn & 1, abort_flag, p.err))) break;
                                tc_fence_after();
                                sums(i, buf, t > 0);
                                if (i == mt - 1) tc_commit(&v_empty[buf]);
                                if (last) {
                                    tc_commit(&o_done[i]);
                                    continue;
                                }
                                if (i == 0) {
                                    if (!(ok = tc_spin_wait(&k_full[nbuf], ((done + 1) / NB) & 1, abort_flag, p.err))) break;
                                    tc_fence_after();
                                }
                                // (issued behind the product that reads the weights it overwrites: one
                                // thread's tcgen05.mma run in the order of their issue)
                                scores(i, nbuf);
                                if (i == mt - 1) {
                                    tc_commit(&k_empty[nbuf]);
                                    if (t + 2 == it.tiles) tc_commit(&q_free);
                                }
                            }
                            if (!ok) break;
                        }
                        items++;
                    } while (0);
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0);
                done = __shfl_sync(0xffffffffu, done, 0);
                items = __shfl_sync(0xffffffffu, items, 0);
            }
            if (lane == 0 && !ok) {
                if (loading) drain_wait(&q_full, items & 1);
                tc_commit(&drained);
                drain_wait(&drained, 0);
            }
            __syncwarp();
        }
    } else {
        // ============ softmax: warpgroup w has row tile w, a thread a row
        regs_up<kSoftRegs>();
        const int w = warp / 4, r = tid % kRowsTile + w * kRowsTile;
        const uint32_t ts = tmem + w * kKv + ((uint32_t)(warp % 4 * 32) << 16), to = tmem + 2 * kKv + w * D + ((uint32_t)(warp % 4 * 32) << 16);
        uint32_t done = 0, turns = 0, items = 0;       // tiles of the CTA, tiles and items of this row tile
        bool ok = true;
        for (int j = 0, have; ok && (have = item(j)) >= 0; j++) {
            if (!have) continue;
            if (w == 1 && it.rows <= kRowsTile) {
                done += it.tiles;
                continue;
            }
            const bool live = r < it.rows;
            const int tok = it.tok + (it.rem + r) / g;
            const int pos = live ? it.q.past + tok : INT_MAX;
            const float rf = live ? __ldg(factors + (int64_t)image * kRowsItem + r) : 0.0f;
            float m = -INFINITY, l = 0.0f;
            for (int t = 0; t < it.tiles; t++, done++, turns++) {
                if (!(ok = warp_wait(&s_full[w], turns & 1, abort_flag, p.err))) break;
                tc_fence_after();
                const int rr = done & 3, tok0 = (it.tile0 + t) * kKv;
                const int hi = pos - tok0, lo = p.window ? max(-1, pos - p.window - tok0) : -1;   // seen: lo < column <= hi
                const uint32_t okm = s_ok[rr];
                const bool whole = __all_sync(0xffffffffu, hi >= kKv - 1 && (!live || lo < 0)) && okm == 0xFFu;
                // bit i: column 32 c + i is seen
                auto seen = [&](int c) -> uint32_t {
                    const int up = hi - 32 * c, down = lo - 32 * c;
                    uint32_t mask = up < 0 ? 0u : up >= 31 ? ~0u : (2u << up) - 1;
                    if (down >= 0) mask &= down >= 31 ? 0u : ~((2u << down) - 1);
                    const uint32_t ok2 = okm >> (2 * c);
                    return mask & ((ok2 & 1 ? 0xFFFFu : 0u) | (ok2 & 2 ? 0xFFFF0000u : 0u));
                };
                // The tile's logits by halves, in two quarters. (Rolled: unrolled, the two
                // passes outgrow the instruction caches.)
                auto quarters = [&](auto &&take) {
#pragma unroll 1
                    for (int c = 0; c < 4; c += 2) {
                        uint32_t x[32], y[32];
                        tmem_ld32(ts + c * 32, x);
                        tmem_ld32(ts + c * 32 + 32, y);
                        tmem_ld_wait();
                        take(c, x);
                        take(c + 1, y);
                    }
                };
                // ---- the row's maximum
                float top = -INFINITY;
                auto maxima = [&](auto kind) {
                    quarters([&](int c, uint32_t (&s)[32]) {
                        constexpr bool masked = decltype(kind)::value;
                        const uint32_t mask = masked ? seen(c) : ~0u;
                        const float2 sk = *reinterpret_cast<const float2 *>(&s_sk[rr][c * 2]);
                        const float2 ls = *reinterpret_cast<const float2 *>(&s_lsv[rr][c * 2]);
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            float x[4];
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                float v = __uint_as_float(s[b * 16 + i]);
                                if (masked) v = mask >> (b * 16 + i) & 1 ? v : -INFINITY;
                                x[i % 4] = i < 4 ? v : fmaxf(x[i % 4], v);
                            }
                            const float y = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                            const float u = fmaf(y, rf * (b ? sk.y : sk.x), b ? ls.y : ls.x);
                            // (a block unseen stays at -inf whatever its factor)
                            top = fmaxf(top, masked && y == -INFINITY ? -INFINITY : u);
                        }
                    });
                };
                if (whole) maxima(std::false_type{});
                else maxima(std::true_type{});
                const bool grow = top > m + kLazy || (m == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, grow)) {
                    const float a = grow ? ex2(m - top) : 1.0f;
                    if (grow) m = top;
                    l *= a;
                    if (t > 0) {
#pragma unroll 1
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t o[32];
                            tmem_ld32(to + c * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
                            tmem_st32(to + c * 32, o);
                        }
                        tmem_st_wait();
                    }
                }
                // ---- the weights, over the logits they come from
                const float ms = m == -INFINITY ? 0.0f : m;
                auto weights = [&](auto kind) {
                    quarters([&](int c, uint32_t (&s)[32]) {
                        constexpr bool masked = decltype(kind)::value;
                        uint32_t hi16[16];
                        [[maybe_unused]] uint32_t lo16[16];
                        const uint32_t mask = masked ? seen(c) : ~0u;
                        const float2 sk = *reinterpret_cast<const float2 *>(&s_sk[rr][c * 2]);
                        const float2 ls = *reinterpret_cast<const float2 *>(&s_lsv[rr][c * 2]);
                        const float2 is = *reinterpret_cast<const float2 *>(&s_isv[rr][c * 2]);
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const float f = rf * (b ? sk.y : sk.x), z = (b ? ls.y : ls.x) - ms;
                            const f32x2 f2 = pair(f, f), z2 = pair(z, z);
                            f32x2 add = pair(0.0f, 0.0f);
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                const f32x2 u = fma2(pair(__uint_as_float(s[b * 16 + i]), __uint_as_float(s[b * 16 + i + 1])), f2, z2);
                                float2 e;
                                if (!SPLIT && i / 2 % kCubic == kCubic - 1) e = ex2_cubic(u);
                                else e = make_float2(ex2(unpair(u).x), ex2(unpair(u).y));
                                if (masked) {
                                    e.x = mask >> (b * 16 + i) & 1 ? e.x : 0.0f;
                                    e.y = mask >> (b * 16 + i + 1) & 1 ? e.y : 0.0f;
                                }
                                add = add2(add, pair(e.x, e.y));
                                hi16[b * 8 + i / 2] = pack_f16(e.x, e.y);
                                if constexpr (SPLIT) {
                                    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi16[b * 8 + i / 2]));
                                    lo16[b * 8 + i / 2] = pack_f16(e.x - h.x, e.y - h.y);
                                }
                            }
                            l = fmaf(unpair(add).x + unpair(add).y, b ? is.y : is.x, l);
                        }
                        tmem_st16(ts + c * 32, hi16);
                        if constexpr (SPLIT) tmem_st16(ts + c * 32 + 16, lo16);
                    });
                };
                if (whole) weights(std::false_type{});
                else weights(std::true_type{});
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[w]);
            }
            if (!ok || !(ok = warp_wait(&o_done[w], items & 1, abort_flag, p.err))) break;
            items++;
            tc_fence_after();
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            const int t = (it.rem + r) / g;
            T *out = static_cast<T *>(p.out) + (int64_t)(it.q.row0 + it.tok + t) * p.out_stride + (head * g + it.rem + r - t * g) * D;
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                tmem_ld32(to + c * 32, o);
                tmem_ld_wait();
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = __uint_as_float(o[i]) * inv;
                if (live) store_vals<32>(out + c * 32, v);
            }
            tc_fence_before();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <int D, typename T>
cudaError_t launch_tiles_d(const AttnParams &p, int few_rows, uint8_t *ws, size_t ws_bytes, cudaStream_t st)
{
    constexpr bool kSplit = sizeof(T) == 4;
    using Sh = TileShape<D, kSplit>;
    auto kern = attend_tiles_kernel<D, T, kSplit>;
    static bool set[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !set[dev]) {
        if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem)) != cudaSuccess) return e;
        if (dev < 64) set[dev] = true;
    }
    // the list goes in slices whose queries fit the workspace
    const int g = p.rows.q_heads / p.c.heads;
    const int64_t entries = (int64_t)p.b.T * g / kRowsItem + p.b.B;
    const size_t per = (size_t)p.c.heads * (Sh::kImage + kRowsItem * 4);
    const int64_t slice = (int64_t)(ws_bytes / per);
    if (slice < 1) return cudaErrorInvalidValue;
    for (int64_t e0 = 0; e0 < entries; e0 += slice) {
        const int e1 = (int)std::min(entries, e0 + slice);
        float *factors = reinterpret_cast<float *>(ws + (size_t)(e1 - e0) * p.c.heads * Sh::kImage);
        const unsigned gy = p.b.T >= 512 ? 1 : (unsigned)((p.rows.q_heads + 3) / 4);
        if ((e = launch_dependent(query_tiles_kernel<D, T, kSplit>, dim3(p.b.T, gy), dim3(128), 0, st, p, (int)e0, e1, few_rows, ws,
                                  factors)) != cudaSuccess)
            return e;
        const int grid = (int)std::min<int64_t>(p.num_sms, (e1 - e0) * p.c.heads);
        if ((e = launch_dependent(kern, dim3(grid), dim3(kThreads), Sh::kSmem, st, p, (int)e0, e1, few_rows, (const uint8_t *)ws,
                                  (const float *)factors)) != cudaSuccess)
            return e;
    }
    return cudaSuccess;
}

}  // namespace

template <typename T>
static cudaError_t launch_tiles_t(const AttnParams &p, int few_rows, uint8_t *ws, size_t ws_bytes, cudaStream_t st)
{
    return p.c.D == 64 ? launch_tiles_d<64, T>(p, few_rows, ws, ws_bytes, st) : launch_tiles_d<128, T>(p, few_rows, ws, ws_bytes, st);
}

cudaError_t launch_attention_tiles(const AttnParams &p, int few_rows, void *ws, size_t ws_bytes, cudaStream_t st)
{
    uint8_t *w = static_cast<uint8_t *>(ws);
    switch (p.rows.act) {
    case MOE_ACT_F32: return launch_tiles_t<float>(p, few_rows, w, ws_bytes, st);
    case MOE_ACT_F16: return launch_tiles_t<__half>(p, few_rows, w, ws_bytes, st);
    default: return launch_tiles_t<__nv_bfloat16>(p, few_rows, w, ws_bytes, st);
    }
}

}  // namespace jmoe
