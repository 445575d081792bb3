// attn.cu -- grouped-query attention over the paged 8-bit cache:
//   o = sum_j p_j (sv_j V_j) / sum_j p_j,  p_j = exp(scale q . (sk_j K_j) - m),
// over the tokens j <= position of the row (and inside its window), with the
// running maximum m and the sums in f32, in one pass over the cache.
//
// attend_stream_kernel: the whole batch's (sequence, row chunk, key head, tile
// of 64 tokens) list is cut into runs, one per CTA, found on the device from the
// batch arrays. A run's tiles go to the CTA's warps in turn, each with a slot of
// shared memory that bulk copies refill; each warp keeps the softmax of the row
// tile in registers, and the warps' (and, where a segment is cut, the CTAs')
// parts are joined by their maxima. Warps that shared a tile among several row
// tiles took longer at every size but one (32 rows over 2000 tokens, 1 sequence:
// 25 us, a row tile a CTA 14).
//
// Bound by the cache's bytes and, as much, by what hides their latency: shared
// memory holds 192 KB a SM in flight, and a warp's slot waits while its tile is
// worked on. Without the products the copies alone run at 5.4 TB/s.
//   64 single tokens over 398752 cached, 4 heads of 128, bf16  96 us, 4.3 TB/s
//   one token over 131001 cached, F32 rows                     41 us, 3.3 TB/s
//   one token over 701 cached, F32 rows                        12 us (latency)
//   66 drafted tokens, 17 sequences, window 1024, f16          16.5 us
//
// The products run on mma.m16n8k16 with f16 operands: a decode row tile has 8
// rows, which the 128-row tcgen05 form would leave 15/16 empty, and the kernel
// is bound by the cache's bytes. Cache bytes are exact in f16. Queries are
// scaled per row by a power of two; with F32 rows they and the weights are
// split in two f16 halves that take the upper and lower 8 rows of the same
// instruction, so 22 bits cost no more than 11 there. With 16-bit rows one f16
// each: the weights' rounding adds 2.1e-4 in the root mean square, as much as an
// F16 output's own. (F16 rows that are normed and turned here take the split
// form: see keep_queries.)
//
// The value scale sv of a block enters as a term of the exponent: the weights
// w = exp2(s + log2 sv - m) stay in (0, 1] whatever the scales, and p = w / sv
// is summed for the denominator (attn.cuh: where scales are far apart).
#include <algorithm>
#include <type_traits>

#include "attn.cuh"
#include "kernels.h"
#include "tc_common.cuh"

namespace jmoe {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
// CTAs of an SM: one joins its parts while the others stream. Three where a CTA
// holds eight rows of queries (a decoder layer's 32 histories 44 us, with two
// 54), else two (registers).
constexpr int kMaxCtasPerSm = 3;
constexpr int kTile = 64;                    // tokens of a tile: 4 blocks
constexpr int kMaxRows = 16;                 // rows of a chunk, at most
// A run has at least this many tiles, one for each warp: fewer CTAs share a short
// sequence (one of 200 tokens 8.2 us, with 2 tiles 11.0; of 3000 13.6 and 15.5;
// 8 of 700 13.6 and 12.8).
constexpr int kMinTiles = kWarps;
// What beginning and joining one more segment costs a CTA, in tiles: runs that
// end with their segment may be longer by this (with 0 and 40 instead of 8: one
// sequence of 3000 tokens 22.0 and 15.5 us for 15.5, 40 of 3000 44.5 and 47.8
// for 44.4, 64 of 500 26.2 and 18.8 for 18.7).
constexpr int kSegmentTiles = 8;

// A segment's parts are joined in groups of this many CTAs, all of a group's
// loads under way at once, then the groups.
constexpr int kJoin = 16;
// Workspace: status word | arrival counters [2][ctas][2] | partials [ctas][2].
constexpr size_t kCounterOff = 256;
constexpr size_t partial_off(int ctas) { return kCounterOff + ((size_t)ctas * 16 + 255) / 256 * 256; }
constexpr size_t kPartialBytes = (size_t)kMaxRows * (kMaxHeadDim + 2) * 4;

// Behind them the queries of attn_tiles.cu, a slice of the rows at a time.
constexpr size_t kTilesBytes = (size_t)80 << 20;
constexpr size_t tiles_off(int num_sms)
{
    return partial_off(num_sms * kMaxCtasPerSm) + (size_t)num_sms * kMaxCtasPerSm * 2 * kPartialBytes;
}
static_assert(tiles_off(148) + kTilesBytes <= MOE_ATTENTION_WORKSPACE_BYTES, "what callers set aside");

// Adds with acquire and release at GPU scope: what the CTA wrote before its
// last barrier is seen by whoever counts after it.
__device__ __forceinline__ int atom_add_acq_rel(int *p, int v)
{
    int old;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
    return old;
}

__device__ __forceinline__ float warp_max_f(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float warp_sum_f(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// c += a b, and c = a b. (volatile: they stay before the refill of the slot that b came from)
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// a and b as f16 pairs hi + lo (22 bits).
__device__ __forceinline__ void split_f16(float a, float b, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = pack_f16(a - f.x, b - f.y);
}

// x / d for 0 <= x < 2^24, inv about 1 / d.
__device__ __forceinline__ int quot(int x, int d, float inv)
{
    int q = (int)((float)x * inv);
    q -= q * d > x;
    return q + ((q + 1) * d <= x);
}

// `total` tiles over `ctas` runs, the first `more` of them one tile longer.
struct Runs {
    int each, more, edge;    // edge: first tile of the shorter runs
    __device__ void set(int total, int ctas)
    {
        each = total / ctas;
        more = total - each * ctas;
        edge = more * (each + 1);
    }
    __device__ int first(int cta) const { return cta < more ? cta * (each + 1) : edge + (cta - more) * each; }
    __device__ int of(int tile) const { return tile < edge ? tile / (each + 1) : more + (tile - edge) / each; }
};

// A sequence of the batch as work: `segs` segments (row chunk x key head) of
// `tiles` tiles each.
struct SeqWork {
    SeqInfo q;
    int slot, tile0, tiles, segs;
};

__device__ __forceinline__ void seq_work(const AttnParams &p, int s, int g, int few_rows, int chunk_rows, SeqWork &w, bool &bad)
{
    const bool listed = seq_info(p.b, s, w.q), cached = seq_in_cache(p.c, p.b, s, w.q, w.slot);
    bad = !listed || !cached;
    w.tile0 = w.tiles = w.segs = 0;
    if (bad || w.q.n == 0 || w.q.n * g > few_rows) return;
    w.tile0 = p.window ? max(0, w.q.past - p.window + 1) / kTile : 0;
    w.tiles = (w.q.past + w.q.n - 1) / kTile + 1 - w.tile0;
    w.segs = p.c.heads;
    if (w.q.n * g > chunk_rows) w.segs *= (w.q.n * g + chunk_rows - 1) / chunk_rows;
}

// A part of a CTA's run: tiles t0 .. t1 - 1 of one segment.
struct Segment {
    SeqInfo q;
    int slot, tile0, tiles, head, t0, t1;
    int tok, rem;              // token and query head of the group of the chunk's first row
    int rows;                  // rows of the chunk
    int pos_first, pos_last;   // positions of its first and last row
    int cta0, cta1;            // CTAs that share the segment
};

template <int D, bool SPLIT>
struct Shape {
    static constexpr int kRows = SPLIT ? 8 : 16;                 // rows of a row tile
    static constexpr int kBlk = kKvBlock * D;                    // bytes of a block
    static constexpr int kVBlk = kBlk + 32;                      // value blocks in shared memory: off the banks of each other
    static constexpr int kQRow = D * 2 + 16;                     // bytes of a query row in f16
    static constexpr int kKBytes = kWarps * 4 * kBlk, kVBytes = kWarps * 4 * kVBlk;
    static constexpr int kRowOff = kKBytes + kVBytes;            // a head row of each warp while it is rotated
    static constexpr int kQOff = kRowOff + kWarps * D * 4;       // queries, upper halves, then the lower ones
    static constexpr int kSmem = kQOff + kRows * kQRow * (SPLIT ? 2 : 1);
    static_assert(kWarps * kRows * D * 4 <= kKBytes + kVBytes, "the warps' sums lie where their tiles were");
};

template <int D, typename T, bool SPLIT>
__global__ void __launch_bounds__(kThreads, SPLIT ? 3 : 2)
    attend_stream_kernel(const __grid_constant__ AttnParams p, int seq0, int seq1, int few_rows, uint32_t g_mul, int *counters,
                         float *partials)
{
    using Sh = Shape<D, SPLIT>;
    constexpr int RR = Sh::kRows, U = SPLIT ? 1 : 2, NT = D / 8, KS = D / 16, N = D / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_full[2][kWarps];       // keys, values
    __shared__ float s_m[kWarps][RR], s_l[kWarps][RR], s_rf[kMaxRows];
    __shared__ int s_last, s_abort;
    uint8_t *s_q = smem + Sh::kQOff;                          // queries: f16 rows, with SPLIT the lower halves behind them
    float *s_sum = reinterpret_cast<float *>(smem);           // the warps' sums of a finished segment
    const uint32_t kbase = smem_addr(smem), vbase = kbase + Sh::kKBytes;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, ln = lane / 4, lj = lane % 4;
    const int g = p.rows.q_heads / p.c.heads, me = blockIdx.x;
    constexpr int q_lower = RR * Sh::kQRow;
    // n / g for numbers below 2^32 / g
    auto over_g = [&](int n) -> int { return g == 1 ? n : (int)__umulhi((uint32_t)n, g_mul); };

    if (tid == 0) {
        for (int i = 0; i < kWarps; i++) {
            mbar_init(&s_full[0][i], 1);
            mbar_init(&s_full[1][i], 1);
        }
        s_abort = 0;
        fence_barrier_init();
    }
    pdl_wait();
    pdl_trigger();
    fence_proxy_async_global();   // the cache as an append before this left it, to the bulk copies

    // ---- this CTA's run of the batch's tiles; each warp finds it on its own, a
    // sequence per lane
    SeqWork w;
    bool bad = false;
    w.tiles = w.segs = 0;
    if (seq0 + lane < seq1) seq_work(p, seq0 + lane, g, few_rows, RR, w, bad);
    const SeqWork w0 = w;
    int total = w.tiles * w.segs, segs = w.segs, longest = w.tiles;
#pragma unroll 4
    for (int s = seq0 + 32 + lane; s < seq1; s += 32) {
        bool worse;
        seq_work(p, s, g, few_rows, RR, w, worse);
        total += w.tiles * w.segs;
        segs += w.segs;
        longest = max(longest, w.tiles);
        bad |= worse;
    }
    if (bad && me == 0) kv_error(p.err);
    total = __reduce_add_sync(0xffffffffu, total);
    segs = __reduce_add_sync(0xffffffffu, segs);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (total == 0) return;
    // Runs of `cut` tiles that end with their segment, where the CTAs suffice for
    // that without much longer runs; else equal runs across segments.
    const int ctas = min((int)gridDim.x, (total + kMinTiles - 1) / kMinTiles);
    int cut = 0;
    if (segs < (int)gridDim.x) {
        cut = max(kMinTiles, (int)__fdividef((float)total, (float)((int)gridDim.x - segs)) + 1);
        if (cut > (int)__fdividef((float)total, (float)ctas) + kSegmentTiles) cut = 0;
    }
    // ... or, where all of those are short, across whole segments: each belongs to the run that
    // its first tile lies in, and none is cut and joined (4 heads, 150 sequences of 500
    // tokens 36.5 us, cut 43.1; 1024 of 100 102 and 108; 128 of 500 34.0 and 34.4).
    const bool uncut = !cut && total <= segs * kSegmentTiles && longest <= total / ctas + kSegmentTiles;
    const float inv_cut = cut ? __fdividef(1.0f, (float)cut) : 1.0f;
    if (!cut && me >= ctas) return;
    Runs runs;
    int at = me, end = me + 1;
    if (!cut) {
        runs.set(total, ctas);
        at = runs.first(me);
        end = runs.first(me + 1);
    }
    int b = -1, base = 0;      // the sequence, and the list's units before it
    for (int s0 = seq0; s0 < seq1 && b < 0; s0 += 128) {
        int n[4];              // units of this lane's sequences, all loads under way at once
#pragma unroll
        for (int k = 0; k < 4; k++) {
            w = w0;
            if (k || s0 != seq0) {
                w.tiles = w.segs = 0;
                if (s0 + 32 * k + lane < seq1) seq_work(p, s0 + 32 * k + lane, g, few_rows, RR, w, bad);
            }
            n[k] = w.segs * (cut ? quot(w.tiles + cut - 1, cut, inv_cut) : w.tiles);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (b >= 0 || s0 + 32 * k >= seq1) break;
            int last = n[k];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, last, o);
                if (lane >= o) last += v;
            }
            last += base;
            const unsigned hit = __ballot_sync(0xffffffffu, n[k] && last - n[k] <= at && at < last);
            b = hit ? s0 + 32 * k + __ffs(hit) - 1 : -1;
            base = __shfl_sync(0xffffffffu, hit ? last - n[k] : last, hit ? __ffs(hit) - 1 : 31);
        }
    }
    if (b < 0) return;         // fewer runs than CTAs

    // The next segment of the run; false at its end.
    auto next_segment = [&](Segment &sg) -> bool {
        if (at >= end) return false;
        int per, idx, off;                         // units of a segment; which one, and where in it
        for (;;) {
            const int i = b - seq0;
            if (i < 32) {
                w.q.past = __shfl_sync(0xffffffffu, w0.q.past, i);
                w.q.row0 = __shfl_sync(0xffffffffu, w0.q.row0, i);
                w.q.n = __shfl_sync(0xffffffffu, w0.q.n, i);
                w.slot = __shfl_sync(0xffffffffu, w0.slot, i);
                w.tile0 = __shfl_sync(0xffffffffu, w0.tile0, i);
                w.tiles = __shfl_sync(0xffffffffu, w0.tiles, i);
                w.segs = __shfl_sync(0xffffffffu, w0.segs, i);
            } else {
                seq_work(p, b, g, few_rows, RR, w, bad);
            }
            per = cut ? quot(w.tiles + cut - 1, cut, inv_cut) : w.tiles;
            if (at < base + w.segs * per) {
                idx = at - base < per ? 0 : (at - base) / per;
                off = at - base - idx * per;
                if (!uncut || !off) break;
                at += per - off;                   // the run before has the segment
                if (at >= end) return false;
            } else {
                base += w.segs * per;
                if (++b >= seq1) return false;
            }
        }
        sg.q = w.q;
        sg.slot = w.slot;
        sg.tile0 = w.tile0;
        sg.tiles = w.tiles;
        if (cut) {
            sg.t0 = off * cut;
            sg.t1 = min(w.tiles, sg.t0 + cut);
            sg.cta0 = me - off;
            sg.cta1 = sg.cta0 + per - 1;
            at++;
        } else {
            sg.t0 = off;
            sg.t1 = uncut ? w.tiles : min(w.tiles, off + end - at);
            sg.cta0 = off == 0 ? me : runs.of(at - off);
            sg.cta1 = sg.t1 == w.tiles ? me : runs.of(at - off + w.tiles - 1);       // (uncut: me)
            at += sg.t1 - off;
        }
        const int chunk = idx < p.c.heads ? 0 : idx / p.c.heads;
        sg.head = idx - chunk * p.c.heads;
        sg.rows = min(RR, w.q.n * g - chunk * RR);
        sg.tok = chunk ? chunk * RR / g : 0;
        sg.rem = chunk * RR - sg.tok * g;
        sg.pos_first = w.q.past + sg.tok;
        sg.pos_last = sg.pos_first + over_g(sg.rem + sg.rows - 1);
        return true;
    };
    // Block of tile t that this lane (mod 4) looks after; -1: none of its tokens is seen, or a bad page.
    auto lookup = [&](const Segment &sg, int t) -> int64_t {
        if (t >= sg.t1) return -1;
        const int blk = (sg.tile0 + t) * (kTile / kKvBlock) + lj, first = blk * kKvBlock;
        if (first > sg.pos_last || (p.window && first + kKvBlock - 1 <= sg.pos_first - p.window)) return -1;
        const int64_t i = block_index(p.c, sg.slot, blk, sg.head);
        if (i < 0) kv_error(p.err);
        return i;
    };
    // The warp loads a tile's keys (0) or values (1) into its slot. `refill`: a tile of the
    // segment was there, the n-th that the warp was given is to follow. Nothing is loaded
    // once a wait of the CTA has run out: the slot's barrier may then still count the copies
    // before. (Lane 31 brings the flag to the ballot; segments end with the first such one:
    // in all 96 us instead of 95 for the 64 single tokens.)
    uint32_t held = 0;                // 0: none did; else 1 + 2 n + which of the first load held back
    auto issue = [&](auto refill, int which, int64_t blk, uint32_t n) {
        constexpr bool REFILL = decltype(refill)::value;
        uint64_t *full = &s_full[which][warp];
        const unsigned all = __ballot_sync(0xffffffffu, REFILL && lane == 31 ? *(volatile int *)&s_abort != 0 : blk >= 0), have = all & 0xFu;
        if (REFILL && all >> 31) {
            if (!held) held = 1 + 2 * n + which;
            return;
        }
        if (lane == 0) mbar_arrive_expect_tx(full, __popc(have) * Sh::kBlk);
        __syncwarp();
        if (lane < 4 && blk >= 0) {
            const uint32_t dst = which ? vbase + (warp * 4 + lj) * Sh::kVBlk : kbase + (warp * 4 + lj) * Sh::kBlk;
            bulk_load(dst, (which ? p.c.v : p.c.k) + blk * Sh::kBlk, Sh::kBlk, full);
        }
    };
    // A slot is its warp's own and is refilled once its bytes have been used: every lane
    // puts its reads of the tile before the bulk copies that are issued after this. (The
    // copies go through another proxy, which neither the products' order nor a barrier
    // of the warp holds back alone.)
    auto given_back = [&] {
        fence_async_smem();
        __syncwarp();
    };
    auto scales = [&](int64_t i, float &k, float &v) {
        k = v = 0.0f;
        if (i >= 0) {
            k = ld_plain(p.c.k_scale + i);
            v = ld_plain(p.c.v_scale + i);
        }
    };
    auto row_ptr = [&](const Segment &sg, int r, int &tok) -> const T * {
        const int t = over_g(sg.rem + r);
        tok = sg.tok + t;
        return static_cast<const T *>(p.rows.q) + (int64_t)(sg.q.row0 + tok) * p.rows.q_stride +
               (sg.head * g + sg.rem + r - t * g) * D + lane * N;
    };

    Segment cur, sg;
    bool joining = false;      // cur's tiles are done, its parts not yet joined
    uint32_t done = 0;         // tiles this warp has taken
    float m[U], l[U], o[NT][SPLIT ? 2 : 4];
    __syncthreads();
    for (;;) {
        // ---- the warps' parts of the segment before, and the CTAs'
        if (joining) {
            const int taken = cur.t1 - cur.t0, used = min(kWarps, taken);
            float *part = s_sum + warp * RR * D;
            __syncthreads();          // every warp is done with its tiles
#pragma unroll
            for (int u = 0; u < U; u++) {
                l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
                l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
                if (lj == 0) {
                    s_m[warp][ln + 8 * u] = m[u];
                    s_l[warp][ln + 8 * u] = l[u];
                }
#pragma unroll
                for (int i = 0; i < NT; i++)
                    *reinterpret_cast<float2 *>(part + (ln + 8 * u) * D + i * 8 + lj * 2) = make_float2(o[i][2 * u], o[i][2 * u + 1]);
            }
            __syncthreads();
            const bool whole_seg = taken == cur.tiles;
            auto part_of = [&](int c) { return partials + (size_t)(c * 2 + (c == cur.cta0)) * (kPartialBytes / 4); };
            float *mine = part_of(me);
            auto write_out = [&](int r, int d, auto &acc, float den) {
                constexpr int V = sizeof(acc) / 4;
                const int t = over_g(cur.rem + r);
                const float inv = den > 0.0f ? 1.0f / den : 0.0f;
                float v[V];
#pragma unroll
                for (int i = 0; i < V; i++) v[i] = acc[i] * inv;
                store_vals<V>(static_cast<T *>(p.out) + (int64_t)(cur.q.row0 + cur.tok + t) * p.out_stride +
                                  (cur.head * g + cur.rem + r - t * g) * D + d,
                              v);
            };
            // Counts the CTA in; whether it is the last of n. (Thread 0's release covers what
            // the CTA wrote before the barrier.)
            auto arrive = [&](int *counter, int n) -> bool {
                __syncthreads();
                if (tid == 0) {
                    s_last = atom_add_acq_rel(counter, 1) == n - 1;
                    if (s_last) *counter = 0;
                }
                __syncthreads();
                return s_last;
            };
            // Joins the parts of n CTAs, c, c + step, ...: into the output, or into the
            // first one's part. A warp takes a row at a time, a lane D / 32 values and a
            // part's maximum and sum; all loads are under way before the first is used.
            auto join = [&](int c, int step, int n, bool finish) {
                for (int r = warp; r < cur.rows; r += kWarps) {
                    float M = -INFINITY, den = 0.0f, acc[N];
#pragma unroll
                    for (int i = 0; i < N; i++) acc[i] = 0.0f;
                    for (int i0 = 0; i0 < n; i0 += kJoin) {
                        const int cn = min(kJoin, n - i0);
                        float v[kJoin][N];
                        const float2 ml = lane < cn ? __ldcg(reinterpret_cast<const float2 *>(part_of(c + (i0 + lane) * step) + 2 * r))
                                                    : make_float2(-INFINITY, 0.0f);
#pragma unroll
                        for (int i = 0; i < kJoin; i++) {
                            if (i < cn) {
                                const float *src = part_of(c + (i0 + i) * step) + 2 * kMaxRows + r * D + lane * N;
                                if constexpr (N == 4) {
                                    const float4 x = __ldcg(reinterpret_cast<const float4 *>(src));
                                    v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
                                } else {
                                    const float2 x = __ldcg(reinterpret_cast<const float2 *>(src));
                                    v[i][0] = x.x; v[i][1] = x.y;
                                }
                            } else {
#pragma unroll
                                for (int j = 0; j < N; j++) v[i][j] = 0.0f;
                            }
                        }
                        const float top = fmaxf(M, warp_max_f(ml.x)), ms = top == -INFINITY ? 0.0f : top;
                        const float before = ex2(M - ms), a = ex2(ml.x - ms);
                        den = scale_den(den, before, M - ms) + warp_sum_f(scale_den(ml.y, a, ml.x - ms));
                        M = top;
#pragma unroll
                        for (int j = 0; j < N; j++) acc[j] *= before;
#pragma unroll
                        for (int i = 0; i < kJoin; i++) {
                            const float ai = __shfl_sync(0xffffffffu, a, i);
#pragma unroll
                            for (int j = 0; j < N; j++) acc[j] = fmaf(v[i][j], ai, acc[j]);
                        }
                    }
                    if (finish) {
                        write_out(r, lane * N, acc, den);
                    } else {
                        float *dst = part_of(c);
                        __syncwarp();          // its maximum and sum have been read
#pragma unroll
                        for (int j = 0; j < N; j++) dst[2 * kMaxRows + r * D + lane * N + j] = acc[j];
                        if (lane == 0) *reinterpret_cast<float2 *>(dst + 2 * r) = make_float2(M, den);
                    }
                }
            };
            constexpr int Q4 = D / 4;
            for (int e = tid; e < cur.rows * Q4; e += kThreads) {
                const int r = e / Q4, d = e % Q4 * 4;
                float M = -INFINITY;
                for (int w = 0; w < used; w++) M = fmaxf(M, s_m[w][r]);
                const float Ms = M == -INFINITY ? 0.0f : M;
                float acc[4] = {}, den = 0.0f;
                for (int w = 0; w < used; w++) {
                    const float a = ex2(s_m[w][r] - Ms);
                    const float4 v = *reinterpret_cast<const float4 *>(s_sum + (w * RR + r) * D + d);
                    den += scale_den(s_l[w][r], a, s_m[w][r] - Ms);
                    acc[0] = fmaf(v.x, a, acc[0]);
                    acc[1] = fmaf(v.y, a, acc[1]);
                    acc[2] = fmaf(v.z, a, acc[2]);
                    acc[3] = fmaf(v.w, a, acc[3]);
                }
                if (whole_seg) {
                    write_out(r, d, acc, den);
                } else {
                    *reinterpret_cast<float4 *>(mine + 2 * kMaxRows + r * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                    if (d == 0) *reinterpret_cast<float2 *>(mine + 2 * r) = make_float2(M, den);
                }
            }
            fence_async_smem();
            __syncthreads();   // the sums are read before the next tiles are copied there
            if (!whole_seg) {
                // Whichever CTA brings a group's last part joins the group, in order;
                // whichever brings the last group joins the groups.
                const int first = cur.cta0 + (me - cur.cta0) / kJoin * kJoin, parts = cur.cta1 - cur.cta0 + 1;
                bool last = arrive(counters + first * 2 + (first == cur.cta0), min(kJoin, cur.cta1 - first + 1));
                const int groups = (parts + kJoin - 1) / kJoin;
                if (last) join(first, 1, min(kJoin, cur.cta1 - first + 1), groups == 1);
                if (last && groups > 1) {
                    last = arrive(counters + 2 * gridDim.x + cur.cta0 * 2, groups);
                    if (last) join(cur.cta0, kJoin, groups, true);
                }
            }
        }
        // ---- a segment's beginning: its first loads
        // (all waits lie between two barriers: every thread reads the same flag here)
        if (*(volatile int *)&s_abort || !next_segment(sg)) break;
        constexpr int kAhead = 2;             // query rows a warp asks for at once
        float qv[kAhead][N], sk = 0.0f, sv = 0.0f;
        int64_t blk = -1;
        {
            int tok;
#pragma unroll
            for (int i = 0; i < kAhead; i++)
                if (warp + i * kWarps < sg.rows) load_vals<N>(row_ptr(sg, warp + i * kWarps, tok), qv[i]);
            const int t = sg.t0 + warp;
            blk = lookup(sg, t);
            if (t < sg.t1)
#pragma unroll 1
                for (int which = 0; which < 2; which++) issue(std::false_type{}, which, blk, done);
            scales(blk, sk, sv);
        }

        // ---- queries of the chunk to shared memory as f16, scaled per row by a power
        // of two that takes the largest value to [2^14, 2^15): what is 2^-28 of it is still held in full
#pragma unroll 1
        for (int r0 = warp; r0 < sg.rows; r0 += kAhead * kWarps) {
            float amax[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int r = min(r0 + k * kWarps, sg.rows - 1);     // (a last odd row goes twice)
                int tok;
                const T *x = row_ptr(sg, r, tok);
                float (&v)[N] = qv[k];
                if (r0 != warp || r != r0 + k * kWarps) load_vals<N>(x, v);
                if (p.use_rope) {
                    float *y = reinterpret_cast<float *>(smem + Sh::kRowOff) + warp * D;
                    norm_rope_vals<D>(v, p.rope.q_norm, p.rope, sg.q.past + tok, y, lane);
#pragma unroll
                    for (int i = 0; i < N; i++) v[i] = y[lane * N + i];
                    __syncwarp();
                }
                amax[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < N; i++) amax[k] = fmaxf(amax[k], fabsf(v[i]));
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++) amax[k] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax[k])));
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int r = min(r0 + k * kWarps, sg.rows - 1);
                const float (&v)[N] = qv[k];
                const int e = max(-112, (int)(__float_as_uint(amax[k]) >> 23) - 127);
                const float up = __int_as_float((14 - e + 127) << 23);
                if (lane == 0) s_rf[r] = __int_as_float((e - 14 + 127) << 23) * p.scale * 1.4426950408889634f;
                uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
                for (int i = 0; i < N / 2; i++) {
                    if constexpr (SPLIT) split_f16(v[2 * i] * up, v[2 * i + 1] * up, hi[i], lo[i]);
                    else hi[i] = pack_f16(v[2 * i] * up, v[2 * i + 1] * up);
                }
                uint32_t *y = reinterpret_cast<uint32_t *>(s_q + r * Sh::kQRow) + lane * (N / 2);
#pragma unroll
                for (int i = 0; i < N / 2; i++) {
                    y[i] = hi[i];
                    if (SPLIT) y[i + q_lower / 4] = lo[i];
                }
            }
        }
        __syncthreads();

        // ---- this warp's row tile as A fragments. Lane (ln, lj) holds the values
        // 16 lj .. 16 lj + 15 of every 64 of its row, in the order in which a key's
        // 16 bytes come out of one load.
        uint32_t qa[KS][4];
        float rf[U];
        int pos[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = ln + 8 * u;
            const bool live = r < sg.rows;
            pos[u] = live ? sg.pos_first + over_g(sg.rem + r) : -1;
            rf[u] = live ? s_rf[r] : 0.0f;
            const uint4 *y = reinterpret_cast<const uint4 *>(s_q + (live ? r : 0) * Sh::kQRow + lj * 32);
#pragma unroll
            for (int h = 0; h < D / 64; h++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint4 a = y[h * 8 + i];
                    uint32_t (&x)[4] = qa[h * 4 + 2 * i], (&z)[4] = qa[h * 4 + 2 * i + 1];
                    x[u] = a.x;
                    x[2 + u] = a.y;
                    z[u] = a.z;
                    z[2 + u] = a.w;
                    if constexpr (SPLIT) {
                        const uint4 c = y[q_lower / 16 + h * 8 + i];
                        x[1] = c.x;
                        x[3] = c.y;
                        z[1] = c.z;
                        z[3] = c.w;
                    }
                }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            m[u] = -INFINITY;
            l[u] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int x = 0; x < (SPLIT ? 2 : 4); x++) o[i][x] = 0.0f;

        // ---- the warp's tiles
        for (int t = sg.t0 + warp; t < sg.t1; t += kWarps, done++) {
            const uint32_t ph = done & 1;
            const int64_t next = lookup(sg, t + kWarps);
            float s[8][4];
            tc_spin_wait(&s_full[0][warp], ph, &s_abort, p.err);
            // column c of the 8-token group i: token 16 (c / 2) + 2 i + (c & 1) of the
            // tile, so that this lane's columns all lie in block lj (four groups at a
            // time: their accumulators do not wait for one another)
            const uint32_t ka = kbase + (warp * 4 + ln / 2) * Sh::kBlk + (ln & 1) * 64 + lj * 16;
#pragma unroll
            for (int i0 = 0; i0 < 8; i0 += 4)
#pragma unroll
                for (int h = 0; h < D / 64; h++) {
                    uint4 kw[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) kw[i] = lds128(ka + h * 1024 + (i0 + i) * 128);
#pragma unroll
                    for (int q = 0; q < 4; q++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            uint32_t b0, b1;
                            bytes_f16(word(kw[i], q), b0, b1);
                            if (h == 0 && q == 0) mma16816_first(s[i0 + i], qa[0], b0, b1);
                            else mma16816(s[i0 + i], qa[h * 4 + q], b0, b1);
                        }
                }
            const bool reload = t + kWarps < sg.t1;
            if (reload) {
                given_back();
                issue(std::true_type{}, 0, next, done + 1);
            }
            float sk_next, sv_next;
            scales(next, sk_next, sv_next);

            // ---- weights
            const float lsv = sv > 0.0f ? lg2(sv) : kNoScaleLog2, isv = ex2(-lsv);
            const int tok0 = (sg.tile0 + t) * kTile;
            const bool clear = tok0 + kTile - 1 <= sg.pos_first && (!p.window || tok0 > sg.pos_last - p.window);
            const bool whole = __all_sync(0xffffffffu, clear && blk >= 0);
            float alpha[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float f = rf[u] * sk;
                float mx[4];
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        float v = SPLIT ? s[i][x] + s[i][2 + x] : s[i][2 * u + x];
                        v = fmaf(v, f, lsv);
                        if (!whole) {
                            const int j = tok0 + lj * 16 + 2 * i + x;
                            if (blk < 0 || j > pos[u] || (p.window && j <= pos[u] - p.window)) v = -INFINITY;
                        }
                        s[i][2 * u + x] = v;
                        mx[i % 4] = i < 4 && x == 0 ? v : fmaxf(mx[i % 4], v);
                    }
                const float mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));      // of this lane's block
                float top = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m[u], top), ms = mn == -INFINITY ? 0.0f : mn;
                const float step = m[u] - ms, ref = block_ref(ms, mine);
                alpha[u] = ex2(step);
                m[u] = mn;
                float sum[4];
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const float e = ex2(s[i][2 * u + x] - ref);
                        s[i][2 * u + x] = e;
                        sum[i % 4] = i < 4 && x == 0 ? e : sum[i % 4] + e;
                    }
                l[u] = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), ref == ms ? isv : ex2(ref - ms - lsv), scale_den(l[u], alpha[u], step));
            }
            // A fragments of the weights: k step q takes tokens 4 q .. 4 q + 3 of each lane's block
            uint32_t pa[4][4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if constexpr (SPLIT) {
                    split_f16(s[2 * q][0], s[2 * q][1], pa[q][0], pa[q][1]);
                    split_f16(s[2 * q + 1][0], s[2 * q + 1][1], pa[q][2], pa[q][3]);
                } else {
                    pa[q][0] = pack_f16(s[2 * q][0], s[2 * q][1]);
                    pa[q][1] = pack_f16(s[2 * q][2], s[2 * q][3]);
                    pa[q][2] = pack_f16(s[2 * q + 1][0], s[2 * q + 1][1]);
                    pa[q][3] = pack_f16(s[2 * q + 1][2], s[2 * q + 1][3]);
                }
            }
            tc_spin_wait(&s_full[1][warp], ph, &s_abort, p.err);
            const uint32_t va = vbase + (warp * 4 + lj) * Sh::kVBlk + ln * 16;
            // a tile's sums start at zero and join the running ones in f32, rounded to
            // nearest: the tensor cores' additions round towards zero
            constexpr int PV = 4;
#pragma unroll
            for (int i0 = 0; i0 < NT; i0 += PV) {
                uint4 vw[PV];
                float c[PV][4];
#pragma unroll
                for (int i = 0; i < PV; i++) vw[i] = lds128(va + (i0 + i) * 128);
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int i = 0; i < PV; i++) {
                        uint32_t b0, b1;
                        bytes_f16(word(vw[i], q), b0, b1);
                        if (q == 0) mma16816_first(c[i], pa[0], b0, b1);
                        else mma16816(c[i], pa[q], b0, b1);
                    }
#pragma unroll
                for (int i = 0; i < PV; i++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        if constexpr (SPLIT) {
                            o[i0 + i][x] = fmaf(o[i0 + i][x], alpha[0], c[i][x] + c[i][2 + x]);
                        } else {
                            o[i0 + i][x] = fmaf(o[i0 + i][x], alpha[0], c[i][x]);
                            o[i0 + i][2 + x] = fmaf(o[i0 + i][2 + x], alpha[U - 1], c[i][2 + x]);
                        }
                    }
            }
            if (reload) {
                given_back();
                issue(std::true_type{}, 1, next, done + 1);
            }
            blk = next;
            sk = sk_next;
            sv = sv_next;
        }
        cur = sg;
        joining = true;
    }
    // after a wait that ran out, copies may still be in flight
    if (*(volatile int *)&s_abort) {
        // loads of each kind: all that were asked for, or those before the first one held back
        const uint32_t values = held ? (held - 1) / 2 : done, keys = values + (held ? (held - 1) & 1 : 0);
        if (keys) drain_wait(&s_full[0][warp], (keys - 1) & 1);
        if (values) drain_wait(&s_full[1][warp], (values - 1) & 1);
    }
}

// Sequences with more rows (new tokens times query heads of a key head) than
// this go to attn_tiles.cu, which takes 256 rows and a key head a CTA over their
// whole history: better where such items fill the SMs, while the runs here split
// a history, but read it anew for each 8 or 16 rows. With 2000 cached tokens, 4
// key heads of 128, bf16 / f32, us here and there:
//   1 sequence,  512 rows  36 / 41 and 52 / 76    16 sequences, 32 rows  35 / 42 and 42 / 63
//   4 sequences, 256 rows  49 / 65 and 51 / 74    16 sequences, 64 rows  51 / 67 and 42 / 64
//   64 sequences, 16 rows  53 / 70 and 81 / 124   64 sequences, 32 rows  96 / 130 and 83 / 127
// (1 sequence of 20000, 128 rows: 51 / 74 and 287 / 476.)
int few_rows(const AttnParams &p)
{
    const int fill = (p.rows.act == MOE_ACT_F32 ? 32 : 24) * p.num_sms / std::max(1, p.b.B * p.c.heads);
    return std::max(16, std::min(512, fill));
}

template <int D, typename T, bool SPLIT>
cudaError_t launch_stream(const AttnParams &p, cudaStream_t st)
{
    using Sh = Shape<D, SPLIT>;
    auto kern = attend_stream_kernel<D, T, SPLIT>;
    static bool set[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !set[dev]) {
        if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem)) != cudaSuccess) return e;
        if (dev < 64) set[dev] = true;
    }
    const int g = p.rows.q_heads / p.c.heads;
    const int64_t rows = (int64_t)p.b.max_new * g;
    // tiles are counted in 32 bits: a sequence's, ...
    const int64_t chunk = (((int64_t)p.c.table_stride * kKvBlock << p.c.page_shift) / kTile + 2) * p.c.heads;
    const int few = (int)std::min<int64_t>(few_rows(p), INT_MAX / chunk * Sh::kRows);
    uint8_t *ws = static_cast<uint8_t *>(p.ws);
    const int ctas = p.num_sms * (SPLIT ? 3 : 2);
    // ... and a launch's: sequences that could have more go in several
    const int64_t most = chunk * ((std::min<int64_t>(rows, few) + Sh::kRows - 1) / Sh::kRows);
    const int step = (int)std::max<int64_t>(1, std::min<int64_t>(p.b.B, (int64_t)INT_MAX / most));
    for (int s = 0; s < p.b.B; s += step) {
        e = launch_dependent(kern, dim3(ctas), dim3(kThreads), Sh::kSmem, st, p, s, std::min(p.b.B, s + step), few,
                             g > 1 ? (uint32_t)((1ull << 32) / g + 1) : 0u, reinterpret_cast<int *>(ws + kCounterOff),
                             reinterpret_cast<float *>(ws + partial_off(p.num_sms * kMaxCtasPerSm)));
        if (e != cudaSuccess) return e;
    }
    if (rows > few) return launch_attention_tiles(p, few, ws + tiles_off(p.num_sms), kTilesBytes, st);
    return cudaSuccess;
}

template <typename T>
cudaError_t launch_t(const AttnParams &p, cudaStream_t st)
{
    // Eight rows at a time where no sequence has more, or for queries of 22 bits: half the registers, three CTAs
    // an SM (8 rows of bf16, 64 sequences of 4000 tokens: 72 us, 16 at a time 83; one of 100000: 38 and 40)
    if (keep_queries<T>(p) || (int64_t)p.b.max_new * (p.rows.q_heads / p.c.heads) <= 8)
        return p.c.D == 64 ? launch_stream<64, T, true>(p, st) : launch_stream<128, T, true>(p, st);
    if constexpr (sizeof(T) == 2)
        return p.c.D == 64 ? launch_stream<64, T, false>(p, st) : launch_stream<128, T, false>(p, st);
    return cudaErrorInvalidValue;
}

}  // namespace

size_t attn_counter_bytes(int num_sms) { return partial_off(num_sms * kMaxCtasPerSm); }
size_t attn_workspace_bytes(int num_sms) { return tiles_off(num_sms) + kTilesBytes; }

cudaError_t launch_attention(const AttnParams &p, cudaStream_t st)
{
    switch (p.rows.act) {
    case MOE_ACT_F32: return launch_t<float>(p, st);
    case MOE_ACT_F16: return launch_t<__half>(p, st);
    default: return launch_t<__nv_bfloat16>(p, st);
    }
}

}  // namespace jmoe
