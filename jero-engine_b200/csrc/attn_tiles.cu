// attn_tiles.cu -- attention of prompts over the paged 8-bit cache on tcgen05:
// the mathematics of attn.cu for row chunks of 256 (tokens of a sequence times
// the query heads of one key head), two tiles of 128 rows a CTA.
//
// Per 128 cached tokens: a warp looks up the pages and stages the cache's bytes
// a tile ahead, four conversion warps turn the cache's bytes into f16
// operands in shared memory (exact; K-major, 128-byte swizzle: a value block
// lies as [D][16 tokens] in the cache, so neither keys nor values are
// transposed), one thread issues S = Q K^T (tcgen05.mma, M 128, N 64) and
// O += P V (N = D, the weights P read from TMEM), and a warpgroup for each row
// tile does its softmax: a thread holds a row. TMEM: for each row tile S in two
// halves of 64 tokens (P over S once S has been read) and O (D columns). While
// a warpgroup weighs one half, the tensor cores add the other half's weights
// and refill it: with one S of 128 columns a row tile the two waited for one
// another, and the same work took 561 us where it took 504 then (4096 rows of 32 heads
// over 4096 + 4096 tokens, bf16).
//
// The sums O are scaled down only when a row's maximum has grown by more than
// 2^8 since they were last: the weights then reach 2^8 instead of 1, which f16
// holds as exactly. With F32 rows queries and weights are split in two f16
// halves, each half a product of its own: 22 bits for twice the products. The
// tensor cores cut a sum off where f32 would round it, some 2^-26 of it lost,
// one way, with each step of 16; so there TMEM holds the sums of two tiles only
// and the softmax threads keep their rows' in registers (rounded sums: 7.8e-7
// off in all over 2500 tokens, 5e-6 with all the tiles in TMEM), which costs
// room: 201 us where it took 176 then (1500 + 1025 tokens of 3 sequences, 32 heads).
// F16 rows that are normed and turned on the way here have their queries split
// too, for errors of 2.7e-4 where one half gives 3.5e-4 and rounding alone 2.1e-4:
// 658 us, 543 with one half (4096 rows over 4096 + 4096 tokens, the append with them).
//
// Bound by the chain from one half's logits to the next one's: a softmax warp
// takes some 2450 cycles for 64 columns (loads 360, maxima 410, a look at their
// growth 210, weights 920, stores 90), the products and their operands' reads
// from shared memory about as long for the four halves that are under way, and
// neither covers the other wholly. 4096 rows of 32 heads over 4096 + 4096
// tokens, bf16: 507 us, 0.81 PFLOP/s; 2064 tokens in 3 prompts, F32 rows: 160 us.
// (Not better: two threads a row and twice the warps, 578 us: the halves then
// hand the maxima to one another; a third or half of the weights by the cubic
// instead of a quarter, 494 and 505.)
#include <algorithm>
#include <type_traits>

#include "attn.cuh"
#include "kernels.h"
#include "tc_common.cuh"

namespace jmoe {
namespace {

constexpr int kRowsTile = 128, kRowsItem = 256, kKv = 128, kHalf = 64;
constexpr int kSoftWarps = 8;
constexpr int kConvWarps = 4, kMmaWarp = kSoftWarps + kConvWarps;
constexpr int kThreads = 16 * 32;    // whole warpgroups: one warp beside the product warps and the loading one only lends registers
// Registers a thread after the split: 2 x (kSoft + kOther) = 4 x the launch's 128.
// With F32 rows the softmax threads keep their rows' sums.
template <bool SPLIT>
struct Regs {
    static constexpr int kSoft = SPLIT ? 200 : 152, kOther = SPLIT ? 56 : 104;
};
// Chunks of a launch that are put in order, at most (a launch of more has several for each SM)
constexpr int kMaxSorted = 1024;
// F32 rows: tiles whose products are summed in TMEM before they join the row's
// sums (one: 210 us where two take 202; four: 198, and over 1e-6 off).
constexpr int kFold = 2;
constexpr int kCubic = 4;            // one pair of weights in this many takes the cubic
// A tile with a block whose scale is below 2^-kWide of the largest so far takes the halves' general form
// (blocks of zeros where values reach 8 or so). Closer ones lose weights of 2^-50 of the largest at most.
constexpr float kWide = 76.0f;
constexpr float kLazy = 8.0f;        // growth of a row's maximum (log2) that its sums are left unscaled for

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
// largest relative error, 7.5e-5 (2^-13.7), below the 2^-12 to 2^-11 that the
// weights' rounding to f16 brings.
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

// tcgen05.mma and commit by one lane of a converged warp: with everything
// around them uniform the descriptors stay in uniform registers (issued under
// "if (lane == 0)" each product took 70 to 100 cycles to issue).
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0)
        : "memory");
}
__device__ __forceinline__ void commit_one(uint64_t *bar)
{
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
        : "memory");
}

// TMEM to registers, load and wait in one: between the two the registers do not
// hold the values yet, and the compiler, which does not know, may move or spill them.
__device__ __forceinline__ void tmem_get32(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_get16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
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

// Chunk `e` of the list as one of sequence s; false where it holds none (or one
// of a sequence with at most few_rows rows, which attn.cu takes).
__device__ __forceinline__ bool item_of(const AttnParams &p, int s, int e, int g, int few_rows, Item &it)
{
    const bool ok = seq_info(p.b, s, it.q) && seq_in_cache(p.c, p.b, s, it.q, it.slot);
    if (!ok) return false;
    const int first = (e - first_entry(p.b, s, g)) * kRowsItem, rows = it.q.n * g;
    if (first < 0 || first >= rows || rows <= few_rows) return false;   // below 0: row_start out of order
    it.tok = first / g;
    it.rem = first - it.tok * g;
    it.rows = min(kRowsItem, rows - first);
    it.pos_first = it.q.past + it.tok;
    it.pos_last = it.pos_first + (it.rem + it.rows - 1) / g;
    it.tile0 = p.window ? max(0, it.pos_first - p.window + 1) / kKv : 0;
    it.tiles = it.pos_last / kKv + 1 - it.tile0;
    return true;
}

// The same for a whole warp, which finds the sequence.
__device__ __forceinline__ bool find_item(const AttnParams &p, int e, int g, int few_rows, int lane, Item &it)
{
    int n = 0;
    for (int s = lane; s < p.b.B; s += 32) n += first_entry(p.b, s, g) <= e;
    const int s = __reduce_add_sync(0xffffffffu, n) - 1;
    return s >= 0 && item_of(p, s, e, g, few_rows, it);
}

// The list's chunks by length, longest first: their places in `order`, by the
// whole CTA, in time for its last barrier. `length`: room for an int each.
__device__ __forceinline__ void sort_items(const AttnParams &p, int entry0, int entries, int g, int few_rows, int *length, uint16_t *order)
{
    for (int e = threadIdx.x; e < entries; e += kThreads) {
        int lo = 0, hi = p.b.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (first_entry(p.b, mid, g) <= entry0 + e ? lo : hi) = mid;
        }
        Item it;
        length[e] = item_of(p, lo, entry0 + e, g, few_rows, it) ? it.tiles : 0;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < entries; e += kThreads) {
        const int mine = length[e];
        int place = 0;
#pragma unroll 4
        for (int i = 0; i < entries; i++) place += length[i] > mine || (length[i] == mine && i < e);
        order[place] = (uint16_t)e;
    }
    fence_async_smem();        // copies are to land where the lengths lay
    __syncthreads();
}

// QS: queries in two halves of 11 bits.
template <int D, bool QS>
struct TileShape {
    static constexpr int kSlabs = D / 64;
    static constexpr int kQTile = (QS ? 2 : 1) * kSlabs * kRowsTile * 128;      // bytes of a row tile's queries
    static constexpr int kBufs = QS ? 1 : 2;
    static constexpr int kOperand = kKv * D * 2;                                // bytes of a key or value operand
    static constexpr int kStage = kKv * D;                                      // ... and of the cache's bytes behind it
    static constexpr int kSmem = 2 * kQTile + 2 * kBufs * kOperand + 2 * kStage;
    static constexpr size_t kImage = 2 * kQTile;                                // an item's queries in the workspace
};

// ------------------------------------------------------------ queries

// Queries as the item's shared-memory image: f16 rows scaled by a power of two
// that takes the largest value to [2^14, 2^15), and the factor that a row's
// logits then need. A warp takes a group of a token's heads; with 16-bit rows five
// CTAs an SM (a layer's 4 prompts 143.5 us, four 148.4).
constexpr int kQueryWarps = 4, kAhead = 4;

template <int D, typename T, bool QS>
__global__ void __launch_bounds__(kQueryWarps * 32, sizeof(T) == 4 ? 0 : 5)
    query_tiles_kernel(const __grid_constant__ AttnParams p, int entry0, int entry1, int head0, int heads, int few_rows, int group,
                       int groups, uint8_t *images, float *factors)
{
    using Sh = TileShape<D, QS>;
    using L = HeadLanes<D, T>;
    __shared__ __align__(16) float s_y[kQueryWarps][L::kScratch];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    pdl_wait();
    pdl_trigger();
    const int64_t item = (int64_t)blockIdx.x * kQueryWarps + warp;
    const int row = (int)(item / groups);
    if (row >= p.b.T) return;
    const int g = p.rows.q_heads / p.c.heads, sub = lane / L::kLanes;
    int h = (int)(item - (int64_t)row * groups) * group + sub;
    const int head1 = min(p.rows.q_heads, h - sub + group), d0 = lane % L::kLanes * L::kVals;
    const T *src = static_cast<const T *>(p.rows.q) + row * p.rows.q_stride + d0;
    float v[kAhead][L::kVals];
    auto load = [&](int h) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int x = h + i * L::kHeads;
            if (x < head1) load_vals<L::kVals>(src + x * D, v[i]);
            else
#pragma unroll
                for (int k = 0; k < L::kVals; k++) v[i][k] = 0.0f;
        }
    };
    load(h);
    const int s = seq_of_row_warp(p.b, row, lane);
    SeqInfo q;
    if (s < 0 || !seq_info(p.b, s, q) || row < q.row0 || row >= q.row0 + q.n || q.n * g <= few_rows) return;
    const int tok = row - q.row0, entry = first_entry(p.b, s, g);
    if (entry + (tok * g + g - 1) / kRowsItem < entry0 || entry + tok * g / kRowsItem >= entry1) return;
    L l;
    float w[L::kVals];
    if (p.use_rope) {
        l.begin(p.rope, q.past + tok, s_y[warp], lane);
        l.weights(p.rope.q_norm, w);
    } else {
        l.lane = lane;
    }
    for (;;) {
        if (p.use_rope && p.rope.q_norm) l.norms(v, w, p.rope.eps);
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int x = h + i * L::kHeads;
            if (x - sub >= head1) break;
            float (&a)[L::kVals] = v[i];
            if (p.use_rope) l.turn(a, s_y[warp]);
            float amax = 0.0f;
#pragma unroll
            for (int k = 0; k < L::kVals; k++) amax = fmaxf(amax, fabsf(a[k]));
            amax = l.head_max(amax);
            const int kvh = x / g, flat = tok * g + x - kvh * g, e = entry + flat / kRowsItem, r = flat % kRowsItem;
            if (x >= head1 || e < entry0 || e >= entry1 || kvh < head0 || kvh >= head0 + heads) continue;
            const int ex = max(-112, (int)(__float_as_uint(amax) >> 23) - 127);
            float up = __int_as_float((14 - ex + 127) << 23);
            const int64_t image = (int64_t)(e - entry0) * heads + kvh - head0;
            if (d0 == 0) factors[image * kRowsItem + r] = __int_as_float((ex - 14 + 127) << 23) * fabsf(p.scale) * 1.4426950408889634f;
            if (p.scale < 0.0f) up = -up;      // the factors are not negative: maxima stay maxima
            uint32_t hi[L::kVals / 2], lo[L::kVals / 2];
#pragma unroll
            for (int k = 0; k < L::kVals / 2; k++) {
                const float y = a[2 * k] * up, z = a[2 * k + 1] * up;
                hi[k] = pack_f16(y, z);
                if constexpr (QS) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[k]));
                    lo[k] = pack_f16(y - f.x, z - f.y);
                }
            }
            const int rt = r % kRowsTile;
            uint8_t *dst = images + image * Sh::kImage + r / kRowsTile * Sh::kQTile + d0 / 64 * (kRowsTile * 128) + rt * 128 +
                           (((d0 % 64) / 8) ^ (rt & 7)) * 16 + d0 % 8 * 2;
            if constexpr (L::kVals == 8) {
                *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (QS) *reinterpret_cast<uint4 *>(dst + Sh::kQTile / 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            } else {
                *reinterpret_cast<uint2 *>(dst) = make_uint2(hi[0], hi[1]);
                if constexpr (QS) *reinterpret_cast<uint2 *>(dst + Sh::kQTile / 2) = make_uint2(lo[0], lo[1]);
            }
        }
        h += kAhead * L::kHeads;
        if (h - sub >= head1) break;
        load(h);
    }
}

// ------------------------------------------------------------ attention

template <int D, typename T, bool SPLIT, bool QS>
__global__ void __launch_bounds__(kThreads, 1)
    attend_tiles_kernel(const __grid_constant__ AttnParams p, int entry0, int entry1, int head0, int heads, int few_rows,
                        const uint8_t *images, const float *factors)
{
    using Sh = TileShape<D, QS>;
    constexpr int NB = Sh::kBufs, SL = Sh::kSlabs;
    // a conversion thread's unit of 16 bytes in every kStep-th block; SPLIT: half of them at a time, for the registers
    constexpr int kStep = kConvWarps * 32 / D, kTurns = SPLIT ? 2 : 1, kIn = 8 / kStep / kTurns;
    static_assert(kStep >= 1 && kIn >= 1, "threads");
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t q_full[2], q_free[2], k_full[NB], k_empty[NB], v_full[NB], v_empty[NB], st_full[2], st_empty[2], s_full[2][2],
        p_full[2][2], o_sum[2], o_done[2], drained[2];
    __shared__ __align__(16) float s_sk[4][8], s_lsv[4][8], s_isv[4][8];
    __shared__ uint32_t s_ok[4];
    __shared__ uint16_t s_order[kMaxSorted];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    uint8_t *sm_q = smem, *sm_k = sm_q + 2 * Sh::kQTile, *sm_v = sm_k + NB * Sh::kOperand, *sm_st = sm_v + NB * Sh::kOperand;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int g = p.rows.q_heads / p.c.heads;

    if (tid == 0) {
        for (int i = 0; i < NB; i++) {
            mbar_init(&k_full[i], kConvWarps);
            mbar_init(&v_full[i], kConvWarps);
            mbar_init(&k_empty[i], 2);
            mbar_init(&v_empty[i], 2);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&st_full[i], 1);
            mbar_init(&st_empty[i], kConvWarps);
            for (int h = 0; h < 2; h++) {
                mbar_init(&s_full[i][h], 2);      // the products' end, and what the product thread has seen
                mbar_init(&p_full[i][h], 4);
            }
            mbar_init(&o_sum[i], 1);
            mbar_init(&o_done[i], 1);
            mbar_init(&q_full[i], 1);
            mbar_init(&q_free[i], 1);
            mbar_init(&drained[i], 1);
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

    // Items go to the CTAs there and back, longest first. (In the list's own order, which
    // is by length within a sequence only: 3 prompts with F32 rows 194 us instead of 158.)
    const int G = gridDim.x, entries = entry1 - entry0, total = entries * heads;
    const bool sorted = entries <= kMaxSorted;
    if (sorted) sort_items(p, entry0, entries, g, few_rows, reinterpret_cast<int *>(smem), s_order);
    Item it;
    int head = 0, image = 0;
    auto item = [&](int j) -> int {       // 1: an item, 0: none here, -1: the end
        if ((int64_t)j * G >= total) return -1;
        const int64_t u = (j & 1) ? (int64_t)(j + 1) * G - 1 - (int)blockIdx.x : (int64_t)j * G + (int)blockIdx.x;
        if (u >= total) return 0;
        const int i = (int)(u / heads), e = sorted ? s_order[i] : entries - 1 - i, h = (int)(u - (int64_t)i * heads);
        head = head0 + h;
        image = e * heads + h;
        return find_item(p, entry0 + e, g, few_rows, lane, it) ? 1 : 0;
    };

    if (warp >= kSoftWarps && warp < kMmaWarp) {
        // ============ conversion: cache bytes -> f16 operands. (After a wait that ran out
        // the warps go on through their barriers: every wait then gives up at once.)
        regs_down<Regs<SPLIT>::kOther>();
        const int ct = tid - kSoftWarps * 32;
        uint32_t done = 0;
        bool ok = true;
        for (int j = 0, have; (have = item(j)) >= 0; j++) {
            if (!have) continue;
            for (int t = 0; t < it.tiles; t++, done++) {
                const int buf = done % NB;
                const uint32_t ph = (done / NB) & 1;
                // ---- keys: rows are tokens, 64 values a slab
                ok &= warp_wait(&st_full[0], done & 1, abort_flag, p.err);
                ok &= warp_wait(&k_empty[buf], ph ^ 1, abort_flag, p.err);
#pragma unroll
                for (int u = 0; u < kTurns; u++) {
                    const int tb = ct % D, sub = ct / D + u * kIn * kStep, slab = tb / 64, tok = tb % 64 / 4, c = tb % 4 * 2;
                    uint8_t *dst = sm_k + buf * Sh::kOperand + slab * (kKv * 128) + tok * 128;
                    const uint32_t src = smem_addr(sm_st) + (sub * D + tb) * 16, x = smem_addr(dst) + ((c ^ (tok & 7)) * 16),
                                   y = smem_addr(dst) + (((c + 1) ^ (tok & 7)) * 16);
                    uint4 in[kIn];
#pragma unroll
                    for (int i = 0; i < kIn; i++) in[i] = lds128(src + i * (kStep * D * 16));
#pragma unroll
                    for (int i = 0; i < kIn; i++) {
                        const uint4 w = in[i];
                        uint4 a, b;
                        bytes_f16(w.x, a.x, a.y);
                        bytes_f16(w.y, a.z, a.w);
                        bytes_f16(w.z, b.x, b.y);
                        bytes_f16(w.w, b.z, b.w);
                        const uint32_t o = (i * kStep + sub) * (kKvBlock * 128);
                        sts128(x + o, a);
                        sts128(y + o, b);
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&st_empty[0]);      // only now: what was loaded has been used
                    mbar_arrive(&k_full[buf]);
                }
                // ---- values: rows are the head's values, 64 tokens a slab
                ok &= warp_wait(&st_full[1], done & 1, abort_flag, p.err);
                ok &= warp_wait(&v_empty[buf], ph ^ 1, abort_flag, p.err);
#pragma unroll
                for (int u = 0; u < kTurns; u++) {
                    const int d = ct % D, sub = ct / D + u * kIn * kStep;
                    uint8_t *dst = sm_v + buf * Sh::kOperand + d * 128;
                    const uint32_t src = smem_addr(sm_st + Sh::kStage) + (sub * D + d) * 16, base = smem_addr(dst);
                    uint4 in[kIn];
#pragma unroll
                    for (int i = 0; i < kIn; i++) in[i] = lds128(src + i * (kStep * D * 16));
#pragma unroll
                    for (int i = 0; i < kIn; i++) {
                        const uint4 w = in[i];
                        uint4 a, b;
                        bytes_f16(w.x, a.x, a.y);
                        bytes_f16(w.y, a.z, a.w);
                        bytes_f16(w.z, b.x, b.y);
                        bytes_f16(w.w, b.z, b.w);
                        const int blk = i * kStep + sub, c = blk % 4 * 2;
                        const uint32_t o = base + blk / 4 * (D * 128);
                        sts128(o + ((c ^ (d & 7)) * 16), a);
                        sts128(o + (((c + 1) ^ (d & 7)) * 16), b);
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&st_empty[1]);      // only now: what was loaded has been used
                    mbar_arrive(&v_full[buf]);
                }
            }
        }
    } else if (warp >= kMmaWarp) {
        regs_down<Regs<SPLIT>::kOther>();
        if (warp < kMmaWarp + 2) {
            // ============ products: a warp for each row tile
            fence_proxy_async_global();       // the queries as the kernel before left them
            const int i = warp - kMmaWarp;
            const uint32_t id_s = (1u << 4) | ((uint32_t)(kHalf >> 3) << 17) | ((uint32_t)(kRowsTile >> 4) << 24);
            const uint32_t id_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRowsTile >> 4) << 24);
            const uint64_t dq = umma_desc_sw128(smem_addr(sm_q + i * Sh::kQTile)), dk = umma_desc_sw128(smem_addr(sm_k)),
                           dv = umma_desc_sw128(smem_addr(sm_v));
            const uint32_t ts = tmem + i * kKv, to = tmem + 2 * kKv + i * D;
            // S of half h from the keys in buffer buf
            auto scores = [&](int h, int buf) {
                if (lane == 0) mbar_arrive(&s_full[i][h]);      // with the scales that the keys came with
                const uint64_t b = dk + ((buf * Sh::kOperand + h * kHalf * 128) >> 4);
#pragma unroll
                for (int half = QS ? 1 : 0; half >= 0; half--)      // the lower halves first: what they lose is small
#pragma unroll
                    for (int s = 0; s < SL; s++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            mma_ss(ts + h * kHalf, dq + ((half * SL + s) * kRowsTile * 128 >> 4) + 2 * k, b + (s * kKv * 128 >> 4) + 2 * k,
                                   id_s, (QS && half == 0) || s + k != 0);
                commit_one(&s_full[i][h]);
            };
            // O: the weights of half h times the values in buffer buf
            auto sums = [&](int h, int buf, uint32_t acc) {
                const uint64_t b = dv + ((buf * Sh::kOperand + h * D * 128) >> 4);
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int half = 0; half < (SPLIT ? 2 : 1); half++)
                        mma_ts(to, ts + h * kHalf + (SPLIT ? k * 16 + half * 8 : k / 2 * 32 + k % 2 * 8), b + 2 * k, id_o, half + k != 0 ? 1u : acc);
                commit_one(&o_sum[i]);
            };
            uint32_t done = 0, items = 0, turns = 0;     // tiles of the CTA, items and tiles of this row tile
            bool ok = true, loading = false;
            auto wait = [&](uint64_t *bar, uint32_t phase) -> bool { return ok = warp_wait(bar, phase & 1, abort_flag, p.err); };
            for (int j = 0, have; ok && (have = item(j)) >= 0; j++) {
                if (!have) continue;
                if (it.rows <= i * kRowsTile) {       // nothing here: the buffers pass by
                    for (int t = 0; t < it.tiles; t++, done++) {
                        if (!wait(&k_full[done % NB], done / NB)) break;
                        if (lane == 0) mbar_arrive(&k_empty[done % NB]);
                        if (!wait(&v_full[done % NB], done / NB)) break;
                        if (lane == 0) mbar_arrive(&v_empty[done % NB]);
                    }
                    continue;
                }
                if (items && !wait(&q_free[i], items - 1)) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&q_full[i], Sh::kQTile);
                    bulk_load(smem_addr(sm_q + i * Sh::kQTile), images + (int64_t)image * Sh::kImage + i * Sh::kQTile, Sh::kQTile, &q_full[i]);
                }
                loading = true;
                if (!wait(&q_full[i], items)) break;
                loading = false;
                if (!wait(&k_full[done % NB], done / NB)) break;
                tc_fence_after();
                scores(0, done % NB);
                scores(1, done % NB);
                commit_one(&k_empty[done % NB]);
                if (it.tiles == 1) commit_one(&q_free[i]);
                for (int t = 0; t < it.tiles; t++, done++, turns++) {
                    const bool last = t + 1 == it.tiles;
                    const int buf = done % NB, nbuf = (done + 1) % NB;
                    if (!wait(&v_full[buf], done / NB)) break;
#pragma unroll 1
                    for (int h = 0; h < 2; h++) {
                        if (!wait(&p_full[i][h], turns)) break;
                        tc_fence_after();
                        sums(h, buf, (SPLIT ? t % kFold : t) > 0 || h > 0);
                        if (h) commit_one(&v_empty[buf]);
                        if (last) continue;
                        if (h == 0) {
                            if (!wait(&k_full[nbuf], (done + 1) / NB)) break;
                            tc_fence_after();
                        }
                        // (issued behind the product that reads the weights it overwrites: one
                        // thread's tcgen05.mma run in the order of their issue)
                        scores(h, nbuf);
                        if (h) {
                            commit_one(&k_empty[nbuf]);
                            if (t + 2 == it.tiles) commit_one(&q_free[i]);
                        }
                    }
                    if (!ok) break;
                    if (last) commit_one(&o_done[i]);
                }
                items++;
            }
            if (!ok) {
                if (loading) drain_wait(&q_full[i], items & 1);
                commit_one(&drained[i]);
                drain_wait(&drained[i], 0);
            }
            __syncwarp();
        } else if (warp == kMmaWarp + 2) {
            // ============ loads: lanes 0 .. 7 look after a block of the tile each, a tile ahead
            fence_proxy_async_global();       // the cache as an append before this left it, to the bulk copies
            uint32_t done = 0, staged[2] = {0, 0};
            bool ok = true;
            for (int j = 0, have; ok && (have = item(j)) >= 0; j++) {
                if (!have) continue;
                float largest = -INFINITY;        // log2 of the item's scales so far
                auto lookup = [&](int t) -> int64_t {
                    const int blk = (it.tile0 + t) * (kKv / kKvBlock) + lane, first = blk * kKvBlock;
                    if (t >= it.tiles || lane >= 8 || first > it.pos_last || (p.window && first + kKvBlock - 1 <= it.pos_first - p.window))
                        return -1;
                    const int64_t i = block_index(p.c, it.slot, blk, head);
                    if (i < 0) kv_error(p.err);
                    return i;
                };
                auto scales = [&](int64_t i, float &k, float &v) {
                    k = i >= 0 ? ld_plain(p.c.k_scale + i) : 0.0f;
                    v = i >= 0 ? ld_plain(p.c.v_scale + i) : 0.0f;
                };
                int64_t at = lookup(0);
                float sk, sv;
                scales(at, sk, sv);
                for (int t = 0; t < it.tiles; t++, done++) {
                    const unsigned live = __ballot_sync(0xffffffffu, at >= 0);
                    for (int which = 0; which < 2; which++) {
                        // read by every conversion warp
                        if (done && !(ok = warp_wait(&st_empty[which], (done - 1) & 1, abort_flag, p.err))) break;
                        if (which == 0) {
                            // (this slot's last tile, four before, has its weights: the keys of the
                            // one before are converted, so those of three before have been used)
                            const int r = done & 3;
                            const float ls = sv > 0.0f ? lg2(sv) : kNoScaleLog2;
                            float big = at >= 0 ? ls : -INFINITY;
#pragma unroll
                            for (int o = 4; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                            largest = fmaxf(largest, big);      // (lanes 0 .. 7)
                            const bool wide = __any_sync(0xffffffffu, at >= 0 && ls < largest - kWide);
                            if (lane < 8) {
                                s_sk[r][lane] = sk;
                                s_lsv[r][lane] = ls;
                                s_isv[r][lane] = ex2(-ls);
                            }
                            if (lane == 0) s_ok[r] = (live & 0xFFu) | (wide ? 0x100u : 0u);
                            __syncwarp();
                        }
                        if (lane == 0) mbar_arrive_expect_tx(&st_full[which], __popc(live) * (kKvBlock * D));
                        __syncwarp();
                        if (at >= 0)
                            bulk_load(smem_addr(sm_st + which * Sh::kStage + lane * kKvBlock * D),
                                      (which ? p.c.v : p.c.k) + at * (kKvBlock * D), kKvBlock * D, &st_full[which]);
                        staged[which] = done + 1;
                    }
                    if (!ok) break;
                    at = lookup(t + 1);
                    scales(at, sk, sv);
                }
            }
            if (!ok)        // copies may still be in flight
                for (int which = 0; which < 2; which++)
                    if (staged[which]) drain_wait(&st_full[which], (staged[which] - 1) & 1);
            __syncwarp();
        }
    } else {
        // ============ softmax: warpgroup w has row tile w, a thread a row
        regs_up<Regs<SPLIT>::kSoft>();
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
            const float rf = live ? ld_plain(factors + (int64_t)image * kRowsItem + r) : 0.0f;
            float m = -INFINITY, l = 0.0f;
            [[maybe_unused]] float tot[SPLIT ? D : 1];     // the row's sums of the tiles before, F32 rows
            if constexpr (SPLIT)
#pragma unroll
                for (int i = 0; i < D; i++) tot[i] = 0.0f;
            for (int u = 0; u < 2 * it.tiles; u++) {
                // ---- half u & 1 of tile u / 2
                const int h = u & 1, rr = done & 3, tok0 = (it.tile0 + u / 2) * kKv + h * kHalf;
                if (!(ok = warp_wait(&s_full[w][h], turns & 1, abort_flag, p.err))) break;
                tc_fence_after();
                uint32_t s[SPLIT ? 32 : kHalf];
                // factors and offsets of the half's four blocks
                const float4 sk = *reinterpret_cast<const float4 *>(&s_sk[rr][4 * h]), ls = *reinterpret_cast<const float4 *>(&s_lsv[rr][4 * h]),
                             is = *reinterpret_cast<const float4 *>(&s_isv[rr][4 * h]);
                const float f[4] = {rf * sk.x, rf * sk.y, rf * sk.z, rf * sk.w}, off[4] = {ls.x, ls.y, ls.z, ls.w},
                            isv[4] = {is.x, is.y, is.z, is.w};
                const int hi = pos - tok0, lo = p.window ? max(-1, pos - p.window - tok0) : -1;   // seen: lo < column <= hi
                const uint32_t flags = s_ok[rr], okm = flags >> (4 * h) & 0xFu;
                const bool whole = __all_sync(0xffffffffu, hi >= kHalf - 1 && (!live || lo < 0)) && okm == 0xFu && !(flags & 0x100u);
                // (a copy of its own for halves that every row sees whole: F32 rows 201 -> 194 us)
                auto weigh = [&](auto whole_half) {
                    constexpr bool WHOLE = decltype(whole_half)::value;
                    if constexpr (!SPLIT) {
                        tmem_get32(ts + h * kHalf, reinterpret_cast<uint32_t (&)[32]>(s[0]));
                        tmem_get32(ts + h * kHalf + 32, reinterpret_cast<uint32_t (&)[32]>(s[32]));
                    }
                    // columns of 32 that this row sees
                    auto seen = [&](int c) -> uint32_t {
                        const int up = hi - 32 * c, down = lo - 32 * c;
                        uint32_t mask = up < 0 ? 0u : up >= 31 ? ~0u : (2u << up) - 1;
                        if (down >= 0) mask &= down >= 31 ? 0u : ~((2u << down) - 1);
                        return mask & ((okm >> (2 * c) & 1 ? 0xFFFFu : 0u) | (okm >> (2 * c) & 2 ? 0xFFFF0000u : 0u));
                    };
                    // ---- the row's maximum; unseen columns to -inf (the other values are finite:
                    // cache bytes times f16)
                    float top = -INFINITY;
                    [[maybe_unused]] float ref[4];      // the blocks' largest
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t (&x32)[32] = reinterpret_cast<uint32_t (&)[32]>(s[SPLIT ? 0 : 32 * c]);
                        if constexpr (SPLIT) {
                            tmem_get32(ts + h * kHalf + 32 * c, x32);
                        }
                        if constexpr (!WHOLE) {
                            const uint32_t mask = seen(c);
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (!(mask >> i & 1)) x32[i] = 0xFF800000u;
                        }
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            float x[4];
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const float v = __uint_as_float(x32[b * 16 + i]);
                                x[i % 4] = i < 4 ? v : fmaxf(x[i % 4], v);
                            }
                            const float y = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                            const float z = y == -INFINITY ? -INFINITY : fmaf(y, f[2 * c + b], off[2 * c + b]);       // (0 * -inf)
                            if constexpr (!WHOLE) ref[2 * c + b] = z;
                            top = fmaxf(top, z);
                        }
                    }
                    const bool grow = top > m + kLazy || (m == -INFINITY && top > -INFINITY);
                    [[maybe_unused]] float down = 1.0f;
                    const bool fold = SPLIT && u > 0 && u % (2 * kFold) == 0;      // what TMEM holds joins the row's sums below
                    if (__any_sync(0xffffffffu, grow)) {
                        const float a = grow ? ex2(m - top) : 1.0f;
                        if (grow) {
                            l = scale_den(l, a, m - top);
                            m = top;
                        }
                        down = a;
                        if (u > 0 && !fold) {
                            // the sums so far, the other half's product among them (the one before
                            // that is done: these logits came after it)
                            if (!(ok = warp_wait(&o_sum[w], (2 * turns + h - 1) & 1, abort_flag, p.err))) return;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D / 32; c++) {
                                uint32_t o[32];
                                tmem_get32(to + c * 32, o);
#pragma unroll
                                for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
                                tmem_st32(to + c * 32, o);
                            }
                            tmem_st_wait();
                            if constexpr (SPLIT)
#pragma unroll
                                for (int i = 0; i < D; i++) tot[i] *= a;
                        }
                    }
                    // ---- the weights, over the logits they come from
                    const float ms = m == -INFINITY ? 0.0f : m;
                    // a block's exponent, and what takes its scale out of the denominator (nothing counts where the
                    // row sees none of it: the cubic is 2^-126 at least)
                    auto take_out = [&](float top_b, float off_b, float isv_b, float &r) -> float {
                        r = block_ref(ms, top_b);
                        return top_b == -INFINITY ? 0.0f : r == ms ? isv_b : ex2(r - ms - off_b);
                    };
                    if constexpr (SPLIT) {
#pragma unroll 1
                        for (int b = 0; b < 4; b++) {
                            uint32_t x16[16], hi8[8], lo8[8];
                            const float fb = rf * s_sk[rr][4 * h + b], ob = s_lsv[rr][4 * h + b];
                            float ib = s_isv[rr][4 * h + b], rb = ms;
                            tmem_get16(ts + h * kHalf + b * 16, x16);
                            if constexpr (!WHOLE) {
                                const uint32_t mask = seen(b / 2) >> (b % 2 * 16);
#pragma unroll
                                for (int i = 0; i < 16; i++)
                                    if (!(mask >> i & 1)) x16[i] = 0xFF800000u;
                                float y = __uint_as_float(x16[0]);
#pragma unroll
                                for (int i = 1; i < 16; i++) y = fmaxf(y, __uint_as_float(x16[i]));
                                ib = take_out(y == -INFINITY ? y : fmaf(y, fb, ob), ob, ib, rb);
                            }
                            const float zb = ob - rb;
                            const float ff = WHOLE ? fb : fmaxf(fb, 1e-30f);    // (0 * -inf)
                            const f32x2 f2 = pair(ff, ff), z2 = pair(zb, zb);
                            f32x2 add = pair(0.0f, 0.0f);
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                const f32x2 x = fma2(pair(__uint_as_float(x16[i]), __uint_as_float(x16[i + 1])), f2, z2);
                                const float2 e = make_float2(ex2(unpair(x).x), ex2(unpair(x).y));
                                add = add2(add, pair(e.x, e.y));
                                hi8[i / 2] = pack_f16(e.x, e.y);
                                const float2 q = __half22float2(*reinterpret_cast<const __half2 *>(&hi8[i / 2]));
                                lo8[i / 2] = pack_f16(e.x - q.x, e.y - q.y);
                            }
                            l = fmaf(unpair(add).x + unpair(add).y, ib, l);
                            tmem_st8(ts + h * kHalf + b * 16, hi8);
                            tmem_st8(ts + h * kHalf + b * 16 + 8, lo8);
                        }
                        if (fold) {
                            // (the product before the last is done: these logits came after it)
                            if (!(ok = warp_wait(&o_sum[w], (2 * turns - 1) & 1, abort_flag, p.err))) return;
                            tc_fence_after();
#pragma unroll
                            for (int c = 0; c < D / 32; c++) {
                                tmem_get32(to + c * 32, s);
#pragma unroll
                                for (int i = 0; i < 32; i++) tot[c * 32 + i] = (tot[c * 32 + i] + __uint_as_float(s[i])) * down;
                            }
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            uint32_t hi16[16];
#pragma unroll
                            for (int b = 0; b < 2; b++) {
                                float ib = isv[2 * c + b], rb = ms;
                                if constexpr (!WHOLE) ib = take_out(ref[2 * c + b], off[2 * c + b], ib, rb);
                                const float ff = WHOLE ? f[2 * c + b] : fmaxf(f[2 * c + b], 1e-30f), z = off[2 * c + b] - rb;    // (0 * -inf)
                                const f32x2 f2 = pair(ff, ff), z2 = pair(z, z);
                                f32x2 add = pair(0.0f, 0.0f);
#pragma unroll
                                for (int i = 0; i < 16; i += 2) {
                                    const int k = c * 32 + b * 16 + i;
                                    const f32x2 x = fma2(pair(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), f2, z2);
                                    float2 e;
                                    if (i / 2 % kCubic == kCubic - 1) e = ex2_cubic(x);
                                    else e = make_float2(ex2(unpair(x).x), ex2(unpair(x).y));
                                    add = add2(add, pair(e.x, e.y));
                                    hi16[b * 8 + i / 2] = pack_f16(e.x, e.y);
                                }
                                l = fmaf(unpair(add).x + unpair(add).y, ib, l);
                            }
                            tmem_st16(ts + h * kHalf + c * 32, hi16);
                        }
                    }
                };
                if (whole) weigh(std::true_type{});
                else weigh(std::false_type{});
                if (!ok) break;
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[w][h]);
                if (h) {
                    done++;
                    turns++;
                }
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
                tmem_get32(to + c * 32, o);
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = (SPLIT ? tot[SPLIT ? c * 32 + i : 0] + __uint_as_float(o[i]) : __uint_as_float(o[i])) * inv;
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

template <int D, typename T, bool QS>
cudaError_t launch_tiles_d(const AttnParams &p, int few_rows, uint8_t *ws, size_t ws_bytes, cudaStream_t st)
{
    constexpr bool kSplit = sizeof(T) == 4;
    using Sh = TileShape<D, QS>;
    auto kern = attend_tiles_kernel<D, T, kSplit, QS>;
    static bool set[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !set[dev]) {
        if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem)) != cudaSuccess) return e;
        // the split of the registers must not ask for more than the launch brings: it would wait for good
        cudaFuncAttributes at;
        if ((e = cudaFuncGetAttributes(&at, kern)) != cudaSuccess) return e;
        if (2 * at.numRegs < Regs<kSplit>::kSoft + Regs<kSplit>::kOther) return cudaErrorInvalidConfiguration;
        if (dev < 64) set[dev] = true;
    }
    // the list goes in slices whose queries fit the workspace: of its chunks, and where not even one chunk's
    // fit (more than 635 key heads of F32 rows of 128) of the key heads too
    const int g = p.rows.q_heads / p.c.heads;
    const int64_t entries = (int64_t)p.b.T * g / kRowsItem + p.b.B;
    constexpr size_t kPerHead = Sh::kImage + kRowsItem * 4;
    const int fit = (int)std::min<size_t>(p.c.heads, ws_bytes / kPerHead);
    if (fit < 1) return cudaErrorInvalidValue;
    const int64_t slice = (int64_t)(ws_bytes / (fit * kPerHead));
    using L = HeadLanes<D, T>;
    // few tokens: one load a warp (the whole call with 128 tokens 53 us, grouped 57); many: a group of
    // heads, which share a token's angles (1024 tokens 76 us, one load a warp 80)
    const int group = p.b.T <= 512 ? L::kHeads : kAhead * L::kHeads * 2, groups = (p.rows.q_heads + group - 1) / group;
    for (int h0 = 0; h0 < p.c.heads; h0 += fit) {
        const int heads = std::min(fit, p.c.heads - h0);
        for (int64_t e0 = 0; e0 < entries; e0 += slice) {
            const int e1 = (int)std::min(entries, e0 + slice);
            float *factors = reinterpret_cast<float *>(ws + (size_t)(e1 - e0) * heads * Sh::kImage);
            if ((e = launch_dependent(query_tiles_kernel<D, T, QS>,
                                      dim3((unsigned)(((int64_t)p.b.T * groups + kQueryWarps - 1) / kQueryWarps)), dim3(kQueryWarps * 32),
                                      0, st, p, (int)e0, e1, h0, heads, few_rows, group, groups, ws, factors)) != cudaSuccess)
                return e;
            const int grid = (int)std::min<int64_t>(p.num_sms, (e1 - e0) * heads);
            if ((e = launch_dependent(kern, dim3(grid), dim3(kThreads), Sh::kSmem, st, p, (int)e0, e1, h0, heads, few_rows,
                                      (const uint8_t *)ws, (const float *)factors)) != cudaSuccess)
                return e;
        }
    }
    return cudaSuccess;
}

}  // namespace

template <typename T>
static cudaError_t launch_tiles_t(const AttnParams &p, int few_rows, uint8_t *ws, size_t ws_bytes, cudaStream_t st)
{
    if constexpr (!std::is_same<T, __nv_bfloat16>::value)
        if (keep_queries<T>(p))
            return p.c.D == 64 ? launch_tiles_d<64, T, true>(p, few_rows, ws, ws_bytes, st)
                               : launch_tiles_d<128, T, true>(p, few_rows, ws, ws_bytes, st);
    if constexpr (sizeof(T) == 2)
        return p.c.D == 64 ? launch_tiles_d<64, T, false>(p, few_rows, ws, ws_bytes, st)
                           : launch_tiles_d<128, T, false>(p, few_rows, ws, ws_bytes, st);
    return cudaErrorInvalidValue;
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
