// attn.cu -- grouped-query attention over the paged 8-bit cache:
//   o = sum_j p_j (sv_j V_j) / sum_j p_j,  p_j = exp(scale q . (sk_j K_j) - m),
// over the tokens j <= position of the row (and inside its window), with the
// running maximum m and the sums in f32, in one pass over the cache.
//
// attend_stream_kernel: the whole batch's (sequence, row chunk, key head, tile
// of 64 tokens) list is cut into equal runs, one per CTA, found on the device
// from the batch arrays. A run's tiles go to the CTA's warps in turn; each warp
// keeps the softmax of its row tile in registers, and the warps' (and, where a
// run ends inside a sequence, the CTAs') parts are joined by their maxima.
//
// The products run on mma.m16n8k16 with f16 operands: a decode row tile has 8
// rows, which the 128-row tcgen05 form would leave 15/16 empty, and the kernel
// is bound by the cache's bytes. Cache bytes are exact in f16. Queries are
// scaled per row by a power of two; with F32 rows they and the weights are
// split in two f16 halves that take the upper and lower 8 rows of the same
// instruction, so 22 bits cost no more than 11.
//
// The value scale sv of a block enters as a term of the exponent: the weights
// w = exp2(s + log2 sv - m) stay in (0, 1] whatever the scales, and p = w / sv
// is summed for the denominator.
#include "attn.cuh"
#include "kernels.h"
#include "tc_common.cuh"

namespace jmoe {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kTile = 64;                    // tokens of a tile: 4 blocks
constexpr int kMaxRows = 128;                // rows of a chunk (8 warps x 16)
// A run has at least this many tiles: fewer CTAs share a short sequence.
constexpr int kMinTiles = 2;

// Workspace: status word | arrival counters [ctas] | partials [ctas][2].
constexpr size_t kCounterOff = 256;
size_t partial_off(int ctas) { return kCounterOff + ((size_t)ctas * 4 + 255) / 256 * 256; }
constexpr size_t kPartialBytes = (size_t)kMaxRows * (kMaxHeadDim + 2) * 4;

// Values of a sequence without a scale (an all-zero block): far below any real
// scale (>= 2^-74), so its weights stay small and its sums in range.
constexpr float kNoScaleLog2 = -80.0f;

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}

// c += a b, and c = a b.
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

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

// a and b as f16 pairs hi + lo (22 bits).
__device__ __forceinline__ void split_f16(float a, float b, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = pack_f16(a - f.x, b - f.y);
}

// Quotients of numbers that nearly always fit in 32 bits.
__device__ __forceinline__ int64_t div64(int64_t a, int64_t b)
{
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// The batch's `total` tiles over `ctas` runs, the first `more` of them one tile longer.
struct Runs {
    int64_t each, more, edge;    // edge: first tile of the shorter runs
    __device__ Runs(int64_t total, int ctas) : each(div64(total, ctas)), more(total - each * ctas), edge(more * (each + 1)) {}
    __device__ int64_t first(int cta) const { return cta < more ? cta * (each + 1) : edge + (cta - more) * each; }
    __device__ int of(int64_t tile) const
    {
        return (int)(tile < edge ? div64(tile, each + 1) : more + div64(tile - edge, each));
    }
};

// A sequence of the batch as work: `chunks` row chunks x key heads x `tiles`.
struct SeqWork {
    SeqInfo q;
    int slot, tile0, tiles, chunks;
};

__device__ __forceinline__ int64_t seq_work(const AttnParams &p, int s, int g, int chunk_rows, SeqWork &w, bool &bad)
{
    const bool listed = seq_info(p.b, s, w.q), cached = seq_in_cache(p.c, p.b, s, w.q, w.slot);
    bad = !listed || !cached;
    if (bad || w.q.n == 0) return 0;
    w.tile0 = p.window ? max(0, w.q.past - p.window + 1) / kTile : 0;
    w.tiles = (w.q.past + w.q.n - 1) / kTile + 1 - w.tile0;
    w.chunks = w.q.n * g <= chunk_rows ? 1 : (w.q.n * g + chunk_rows - 1) / chunk_rows;
    return (int64_t)w.tiles * w.chunks * p.c.heads;
}

// A part of a CTA's run: tiles t0 .. t1 - 1 of one (sequence, chunk, key head).
struct Segment {
    SeqWork w;
    int chunk, head, t0, t1;
    int rows, row_first;       // rows of the chunk, its first flat row
    int tok, rem;              // that row's token and its query head of the group
    int pos_first, pos_last;   // positions of its first and last row
    int64_t unit;              // index of the segment's tile 0 in the batch's list
};

template <int D, typename T, bool SPLIT>
struct Shape {
    static constexpr int kRows = SPLIT ? 8 : 16;                 // rows of a row tile
    static constexpr int kBlk = kKvBlock * D;                    // bytes of a block
    static constexpr int kVBlk = kBlk + 32;                      // value blocks in shared memory: off the banks of each other
    static constexpr int kQStride = D + 4;
    static constexpr int kQBytes = kWarps * kRows * kQStride * 4;   // queries, then the warps' sums
    static constexpr int kKBytes = kWarps * 4 * kBlk, kVBytes = kWarps * 4 * kVBlk;
    static constexpr int kSmem = kKBytes + kVBytes + kQBytes;
};

template <int D, typename T, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) attend_stream_kernel(const __grid_constant__ AttnParams p, int group,
                                                                    uint32_t g_mul, int *counters, float *partials)
{
    using Sh = Shape<D, T, SPLIT>;
    constexpr int RR = Sh::kRows, NT = D / 8, KS = D / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_full[2][kWarps], s_empty[2][kWarps];   // keys, values
    __shared__ float s_m[kWarps][RR], s_l[kWarps][RR];
    __shared__ int s_last, s_abort;
    float *s_q = reinterpret_cast<float *>(smem + Sh::kKBytes + Sh::kVBytes);
    const uint32_t kbase = smem_addr(smem), vbase = kbase + Sh::kKBytes;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, ln = lane / 4, lj = lane % 4;
    const int streams = kWarps / group, stream = warp / group, rt = warp % group, depth = group;
    const int g = p.rows.q_heads / p.c.heads, chunk_rows = group * RR, G = gridDim.x;
    const bool leader = rt == 0;

    if (tid == 0) {
        for (int i = 0; i < kWarps; i++) {
            mbar_init(&s_full[0][i], 1);
            mbar_init(&s_full[1][i], 1);
            mbar_init(&s_empty[0][i], group);
            mbar_init(&s_empty[1][i], group);
        }
        s_abort = 0;
        fence_barrier_init();
    }
    pdl_wait();
    fence_proxy_async_global();   // the cache as an append before this left it, to the bulk copies

    // (flat row of a chunk's first token on) / g, for numbers below 2^32 / g
    auto over_g = [&](int n) -> int { return g == 1 ? n : (int)__umulhi((uint32_t)n, g_mul); };

    // ---- this CTA's run of the batch's tiles; each warp finds it on its own
    SeqWork w0;
    bool bad0 = false;
    const int64_t n0 = lane < p.b.B ? seq_work(p, lane, g, chunk_rows, w0, bad0) : 0;
    int64_t total = n0;
    bool any_bad = bad0;
    for (int s = 32 + lane; s < p.b.B; s += 32) {
        SeqWork w;
        total += seq_work(p, s, g, chunk_rows, w, bad0);
        any_bad |= bad0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (any_bad && blockIdx.x == 0) kv_error(p.err);
    if (total == 0) return;
    const int ctas = (int)min((int64_t)G, (total + kMinTiles - 1) / kMinTiles), me = blockIdx.x;
    if (me >= ctas) return;
    const Runs runs(total, ctas);
    const int64_t run0 = runs.first(me), run1 = runs.first(me + 1);
    int b = -1;
    int64_t base = 0, at = run0;
    for (int s0 = 0; s0 < p.b.B && b < 0; s0 += 32) {
        SeqWork w;
        const int64_t n = s0 == 0 ? n0 : s0 + lane < p.b.B ? seq_work(p, s0 + lane, g, chunk_rows, w, bad0) : 0;
        int64_t end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += v;
        }
        end += base;
        const unsigned hit = __ballot_sync(0xffffffffu, n && end - n <= run0 && run0 < end);
        if (hit) {
            b = s0 + __ffs(hit) - 1;
            base = __shfl_sync(0xffffffffu, end - n, __ffs(hit) - 1);
        } else {
            base = __shfl_sync(0xffffffffu, end, 31);
        }
    }
    if (b < 0) return;

    // The next segment of the run; false at its end.
    auto next_segment = [&](Segment &sg) -> bool {
        if (at >= run1) return false;
        bool bad;
        int64_t n = seq_work(p, b, g, chunk_rows, sg.w, bad);
        while (at >= base + n) {
            base += n;
            if (b + 1 >= p.b.B) return false;
            n = seq_work(p, ++b, g, chunk_rows, sg.w, bad);
        }
        const int64_t off = at - base;
        const int idx = (int)div64(off, sg.w.tiles);
        sg.t0 = (int)(off - (int64_t)idx * sg.w.tiles);
        sg.t1 = (int)min((int64_t)sg.w.tiles, sg.t0 + (run1 - at));
        sg.unit = at - sg.t0;
        sg.chunk = idx < p.c.heads ? 0 : idx / p.c.heads;
        sg.head = idx - sg.chunk * p.c.heads;
        sg.row_first = sg.chunk * chunk_rows;
        sg.rows = min(chunk_rows, sg.w.q.n * g - sg.row_first);
        sg.tok = sg.chunk ? sg.row_first / g : 0;
        sg.rem = sg.row_first - sg.tok * g;
        sg.pos_first = sg.w.q.past + sg.tok;
        sg.pos_last = sg.pos_first + over_g(sg.rem + sg.rows - 1);
        at += sg.t1 - sg.t0;
        return true;
    };
    // Block of tile t that this lane (mod 4) looks after; -1: none of its tokens is seen, or a bad page.
    auto lookup = [&](const Segment &sg, int t) -> int64_t {
        if (t >= sg.t1) return -1;
        const int blk = (sg.w.tile0 + t) * (kTile / kKvBlock) + lj, first = blk * kKvBlock;
        if (first > sg.pos_last || (p.window && first + kKvBlock - 1 <= sg.pos_first - p.window)) return -1;
        const int64_t i = block_index(p.c, sg.w.slot, blk, sg.head);
        if (i < 0) kv_error(p.err);
        return i;
    };
    // The leader warp loads tile t's keys or values into the stream's slot.
    uint32_t issued[2] = {0, 0};
    auto issue = [&](int which, int64_t blk) {
        const uint32_t n = issued[which]++;
        const int slot = stream * depth + (int)(n % depth);
        uint64_t *full = &s_full[which][slot];
        const unsigned have = __ballot_sync(0xffffffffu, blk >= 0) & 0xFu;
        // the slot's last tile has been read by every warp of the group
        if (n >= (uint32_t)depth) tc_spin_wait(&s_empty[which][slot], (n / depth - 1) & 1, &s_abort, p.err);
        if (lane == 0) mbar_arrive_expect_tx(full, __popc(have) * Sh::kBlk);
        __syncwarp();
        if (lane < 4 && blk >= 0) {
            const uint32_t dst = which ? vbase + (slot * 4 + lj) * Sh::kVBlk : kbase + (slot * 4 + lj) * Sh::kBlk;
            bulk_load(dst, (which ? p.c.v : p.c.k) + blk * Sh::kBlk, Sh::kBlk, full);
        }
    };
    // A segment's beginning: this warp's first query row and block scales are
    // asked for, then the stream's first tiles.
    constexpr int N = D / 32;
    float qv[N], sk = 0.0f, sv = 0.0f;
    int64_t blk = -1;
    auto row_ptr = [&](const Segment &sg, int r, int &tok) -> const T * {
        const int t = over_g(sg.rem + r);
        tok = sg.tok + t;
        return static_cast<const T *>(p.rows.q) + (int64_t)(sg.w.q.row0 + tok) * p.rows.q_stride +
               (sg.head * g + sg.rem + r - t * g) * D;
    };
    auto scales = [&](int64_t i, float &k, float &v) {
        k = v = 0.0f;
        if (i >= 0) {
            k = __ldg(p.c.k_scale + i);
            v = __ldg(p.c.v_scale + i);
        }
    };
    auto begin = [&](const Segment &sg) {
        int tok;
        if (warp < sg.rows) load_vals<N>(row_ptr(sg, warp, tok) + lane * N, qv);
        blk = lookup(sg, sg.t0 + stream);
        if (leader)
            for (int i = 0; i < depth; i++) {
                const int t = sg.t0 + stream + i * streams;
                if (t >= sg.t1) break;
                const int64_t first = i ? lookup(sg, t) : blk;
                issue(0, first);
                issue(1, first);
            }
        scales(blk, sk, sv);
    };

    Segment sg;
    if (!next_segment(sg)) return;
    __syncthreads();
    begin(sg);
    uint32_t done = 0;   // tiles this stream has taken
    const float log2e = 1.4426950408889634f;

    for (;;) {
        // ---- queries of the chunk to shared memory, in f32
        for (int r = warp; r < sg.rows; r += kWarps) {
            int tok;
            const T *x = row_ptr(sg, r, tok);
            if (r != warp) load_vals<N>(x + lane * N, qv);
            float *y = s_q + r * Sh::kQStride;
            if (p.use_rope) {
                norm_rope_vals<D>(qv, p.rope.q_norm, p.rope, sg.w.q.past + tok, y, lane);
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) y[lane * N + i] = qv[i];
            }
        }
        __syncthreads();

        // ---- this warp's row tile as A fragments. Lane (ln, lj) holds the
        // values 16 lj .. 16 lj + 15 of every 64 of its row, in the order in
        // which a key's 16 bytes come out of one load.
        uint32_t qa[KS][4];
        float rf[SPLIT ? 1 : 2];        // per row: logit factor
        int pos[SPLIT ? 1 : 2];
        const int row_base = rt * RR;
#pragma unroll
        for (int u = 0; u < (SPLIT ? 1 : 2); u++) {
            const int r = row_base + ln + 8 * u;
            const bool live = r < sg.rows;
            pos[u] = live ? sg.pos_first + over_g(sg.rem + r) : -1;
            const float *y = s_q + (live ? r : 0) * Sh::kQStride;
            float amax = 0.0f;
#pragma unroll
            for (int h = 0; h < D / 64; h++)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(y + h * 64 + lj * 16 + i);
                    amax = fmaxf(fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
                }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // largest value to [2^14, 2^15): f16 then holds values 2^-28 of it in full
            const int e = max(-112, (__float_as_int(amax) >> 23) - 127);
            const float up = __int_as_float((14 - e + 127) << 23);
            rf[u] = __int_as_float((e - 14 + 127) << 23) * p.scale * log2e;
#pragma unroll
            for (int h = 0; h < D / 64; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float4 v = *reinterpret_cast<const float4 *>(y + h * 64 + lj * 16 + 4 * i);
                    if (!live) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    uint32_t (&a)[4] = qa[h * 4 + i];
                    if constexpr (SPLIT) {
                        split_f16(v.x * up, v.y * up, a[0], a[1]);
                        split_f16(v.z * up, v.w * up, a[2], a[3]);
                    } else {
                        a[u] = pack_f16(v.x * up, v.y * up);
                        a[2 + u] = pack_f16(v.z * up, v.w * up);
                    }
                }
        }
        const int tile_pos0 = sg.pos_first + over_g(sg.rem + min(row_base, sg.rows - 1));   // of the first row
        const int tile_pos1 = sg.pos_first + over_g(sg.rem + min(row_base + RR, sg.rows) - 1);

        float m[SPLIT ? 1 : 2], l[SPLIT ? 1 : 2], o[NT][SPLIT ? 2 : 4];
#pragma unroll
        for (int u = 0; u < (SPLIT ? 1 : 2); u++) {
            m[u] = -INFINITY;
            l[u] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int x = 0; x < (SPLIT ? 2 : 4); x++) o[i][x] = 0.0f;

        // ---- the stream's tiles
        for (int t = sg.t0 + stream; t < sg.t1; t += streams, done++) {
            const int slot = stream * depth + (int)(done % depth);
            const uint32_t ph = (done / depth) & 1;
            const int64_t next = lookup(sg, t + streams);
            const int64_t ahead = depth == 1 ? next : leader ? lookup(sg, t + depth * streams) : -1;
            float s[8][4];
            tc_spin_wait(&s_full[0][slot], ph, &s_abort, p.err);
            // column c of the 8-token group i: token 16 (c / 2) + 2 i + (c & 1) of the
            // tile, so that this lane's columns all lie in block lj
            const uint32_t ka = kbase + (slot * 4 + ln / 2) * Sh::kBlk + (ln & 1) * 64 + lj * 16;
            // (four groups at a time: their accumulators do not wait for one another)
#pragma unroll
            for (int i0 = 0; i0 < 8; i0 += 4)
#pragma unroll
                for (int h = 0; h < D / 64; h++) {
                    uint4 w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = lds128(ka + h * 1024 + (i0 + i) * 128);
#pragma unroll
                    for (int q = 0; q < 4; q++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            uint32_t b0, b1;
                            bytes_f16(word(w[i], q), b0, b1);
                            if (h == 0 && q == 0) mma16816_first(s[i0 + i], qa[0], b0, b1);
                            else mma16816(s[i0 + i], qa[h * 4 + q], b0, b1);
                        }
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_empty[0][slot]);
            if (leader && t + depth * streams < sg.t1) issue(0, ahead);
            float sk_next, sv_next;
            scales(next, sk_next, sv_next);

            // ---- weights
            const float lsv = sv > 0.0f ? log2f(sv) : kNoScaleLog2, isv = sv > 0.0f ? 1.0f / sv : ex2(-kNoScaleLog2);
            const int tok0 = (sg.w.tile0 + t) * kTile;
            const bool clear = tok0 + kTile - 1 <= tile_pos0 && (!p.window || tok0 > tile_pos1 - p.window);
            const bool whole = __all_sync(0xffffffffu, clear && blk >= 0);
            float alpha[SPLIT ? 1 : 2];
#pragma unroll
            for (int u = 0; u < (SPLIT ? 1 : 2); u++) {
                const float f = rf[u] * sk;
                float mx = -INFINITY;
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
                        mx = fmaxf(mx, v);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[u], mx), ms = mn == -INFINITY ? 0.0f : mn;
                alpha[u] = ex2(m[u] - ms);
                m[u] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const float w = ex2(s[i][2 * u + x] - ms);
                        s[i][2 * u + x] = w;
                        sum += w;
                    }
                l[u] = fmaf(l[u], alpha[u], sum * isv);
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
            tc_spin_wait(&s_full[1][slot], ph, &s_abort, p.err);
            const uint32_t va = vbase + (slot * 4 + lj) * Sh::kVBlk + ln * 16;
            // a tile's sums start at zero and join the running ones in f32, rounded to
            // nearest: the tensor cores' additions round towards zero
#pragma unroll
            for (int i0 = 0; i0 < NT; i0 += 4) {
                uint4 w[4];
                float c[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = lds128(va + (i0 + i) * 128);
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t b0, b1;
                        bytes_f16(word(w[i], q), b0, b1);
                        if (q == 0) mma16816_first(c[i], pa[0], b0, b1);
                        else mma16816(c[i], pa[q], b0, b1);
                    }
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        if constexpr (SPLIT) {
                            o[i0 + i][x] = fmaf(o[i0 + i][x], alpha[0], c[i][x] + c[i][2 + x]);
                        } else {
                            o[i0 + i][x] = fmaf(o[i0 + i][x], alpha[0], c[i][x]);
                            o[i0 + i][2 + x] = fmaf(o[i0 + i][2 + x], alpha[1], c[i][2 + x]);
                        }
                    }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_empty[1][slot]);
            if (leader && t + depth * streams < sg.t1) issue(1, ahead);
            blk = next;
            sk = sk_next;
            sv = sv_next;
        }

        // ---- the next segment's first tiles are on their way while this one is joined
        const Segment cur = sg;
        const bool more = next_segment(sg);
        if (more) begin(sg);

        const int taken = cur.t1 - cur.t0, used = min(streams, taken);
        float *part = s_q + warp * RR * D;      // the queries are in registers by now
        __syncthreads();
#pragma unroll
        for (int u = 0; u < (SPLIT ? 1 : 2); u++) {
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
            if (lj == 0) {
                s_m[warp][ln + 8 * u] = m[u];
                s_l[warp][ln + 8 * u] = l[u];
            }
#pragma unroll
            for (int i = 0; i < NT; i++) {
                *reinterpret_cast<float2 *>(part + (ln + 8 * u) * D + i * 8 + lj * 2) = make_float2(o[i][2 * u], o[i][2 * u + 1]);
            }
        }
        __syncthreads();
        const bool whole_seq = taken == cur.w.tiles;
        const int64_t last_unit = cur.unit + cur.w.tiles - 1;
        const int c0 = cur.t0 == 0 ? me : runs.of(cur.unit), c1 = cur.t1 == cur.w.tiles ? me : runs.of(last_unit);
        float *mine = partials + (size_t)(me * 2 + (me == c0 ? 1 : 0)) * (kPartialBytes / 4);
        auto write_out = [&](int r, int d, auto &acc, float den) {
            constexpr int V = sizeof(acc) / 4;
            const int t = over_g(cur.rem + r);
            const float inv = den > 0.0f ? 1.0f / den : 0.0f;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = acc[i] * inv;
            store_vals<V>(static_cast<T *>(p.out) + (int64_t)(cur.w.q.row0 + cur.tok + t) * p.out_stride +
                              (cur.head * g + cur.rem + r - t * g) * D + d,
                          v);
        };
        constexpr int Q4 = D / 4;
        for (int e = tid; e < cur.rows * Q4; e += kThreads) {
            const int r = e / Q4, d = e % Q4 * 4, w0 = r / RR, rr = r % RR;
            float M = -INFINITY;
            for (int i = 0; i < used; i++) M = fmaxf(M, s_m[i * group + w0][rr]);
            const float Ms = M == -INFINITY ? 0.0f : M;
            float acc[4] = {}, den = 0.0f;
            for (int i = 0; i < used; i++) {
                const int w = i * group + w0;
                const float a = ex2(s_m[w][rr] - Ms);
                const float4 v = *reinterpret_cast<const float4 *>(s_q + (w * RR + rr) * D + d);
                den = fmaf(s_l[w][rr], a, den);
                acc[0] = fmaf(v.x, a, acc[0]);
                acc[1] = fmaf(v.y, a, acc[1]);
                acc[2] = fmaf(v.z, a, acc[2]);
                acc[3] = fmaf(v.w, a, acc[3]);
            }
            if (whole_seq) {
                write_out(r, d, acc, den);
            } else {
                *reinterpret_cast<float4 *>(mine + 2 * kMaxRows + r * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                if (d == 0) *reinterpret_cast<float2 *>(mine + 2 * r) = make_float2(M, den);
            }
        }
        if (!whole_seq) {
            // the CTA that brings the last part joins them all, in their order: a
            // warp per row, lanes over the parts for the maximum, then over the values
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                const int n = atomicAdd(counters + c0, 1);
                s_last = n == c1 - c0;
                if (s_last) counters[c0] = 0;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                auto part_of = [&](int c) { return partials + (size_t)(c * 2 + (c == c0)) * (kPartialBytes / 4); };
                for (int r = warp; r < cur.rows; r += kWarps) {
                    float M = -INFINITY;
                    for (int c = c0 + lane; c <= c1; c += 32) M = fmaxf(M, __ldcg(part_of(c) + 2 * r));
                    M = warp_max_f(M);
                    const float Ms = M == -INFINITY ? 0.0f : M;
                    constexpr int V = D / 32;
                    float acc[V], den = 0.0f;
#pragma unroll
                    for (int i = 0; i < V; i++) acc[i] = 0.0f;
                    for (int cb = c0; cb <= c1; cb += 32) {
                        float a = 0.0f;
                        if (cb + lane <= c1) {
                            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part_of(cb + lane) + 2 * r));
                            a = ex2(ml.x - Ms);
                            den = fmaf(ml.y, a, den);
                        }
                        const int n = min(32, c1 - cb + 1);
#pragma unroll 8
                        for (int i = 0; i < n; i++) {
                            const float *src = part_of(cb + i) + 2 * kMaxRows + r * D + lane * V;
                            float v[V];
                            if constexpr (V == 4) {
                                const float4 x = __ldcg(reinterpret_cast<const float4 *>(src));
                                v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                            } else {
                                const float2 x = __ldcg(reinterpret_cast<const float2 *>(src));
                                v[0] = x.x; v[1] = x.y;
                            }
                            const float ai = __shfl_sync(0xffffffffu, a, i);
#pragma unroll
                            for (int k = 0; k < V; k++) acc[k] = fmaf(v[k], ai, acc[k]);
                        }
                    }
                    den = warp_sum_f(den);
                    write_out(r, lane * V, acc, den);
                }
            }
        }
        if (!more) break;
        __syncthreads();   // the sums are read before the next queries go there
    }
    // after a wait that ran out, copies may still be in flight
    if (*(volatile int *)&s_abort && leader)
        for (int which = 0; which < 2; which++)
            for (uint32_t n = issued[which] > (uint32_t)depth ? issued[which] - depth : 0; n < issued[which]; n++)
                drain_wait(&s_full[which][stream * depth + n % depth], (n / depth) & 1);
}

template <int D, typename T, bool SPLIT>
cudaError_t launch_stream(const AttnParams &p, cudaStream_t st)
{
    using Sh = Shape<D, T, SPLIT>;
    auto kern = attend_stream_kernel<D, T, SPLIT>;
    static bool set[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !set[dev]) {
        if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem)) != cudaSuccess) return e;
        if (dev < 64) set[dev] = true;
    }
    // warps that share a tile: one for each row tile, up to all eight
    const int g = p.rows.q_heads / p.c.heads;
    const int64_t rows = (int64_t)p.b.max_new * g;
    int group = 1;
    while (group < kWarps && (int64_t)group * Sh::kRows < rows) group *= 2;
    uint8_t *ws = static_cast<uint8_t *>(p.ws);
    return launch_dependent(kern, dim3(p.num_sms), dim3(kThreads), Sh::kSmem, st, p, group, g > 1 ? (uint32_t)((1ull << 32) / g + 1) : 0u,
                            reinterpret_cast<int *>(ws + kCounterOff), reinterpret_cast<float *>(ws + partial_off(p.num_sms)));
}

template <typename T>
cudaError_t launch_t(const AttnParams &p, cudaStream_t st)
{
    // eight rows at a time where no sequence has more (half the registers), or for 22 bits
    if (sizeof(T) == 4 || (int64_t)p.b.max_new * (p.rows.q_heads / p.c.heads) <= 8)
        return p.c.D == 64 ? launch_stream<64, T, true>(p, st) : launch_stream<128, T, true>(p, st);
    if constexpr (sizeof(T) == 2)
        return p.c.D == 64 ? launch_stream<64, T, false>(p, st) : launch_stream<128, T, false>(p, st);
    return cudaErrorInvalidValue;
}

}  // namespace

size_t attn_workspace_bytes(int num_sms) { return partial_off(num_sms) + (size_t)num_sms * 2 * kPartialBytes; }

cudaError_t launch_attention(const AttnParams &p, cudaStream_t st)
{
    switch (p.rows.act) {
    case MOE_ACT_F32: return launch_t<float>(p, st);
    case MOE_ACT_F16: return launch_t<__half>(p, st);
    default: return launch_t<__nv_bfloat16>(p, st);
    }
}

}  // namespace jmoe
