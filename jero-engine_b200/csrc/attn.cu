// attn.cu -- grouped-query attention over the paged 8-bit cache:
//   o = sum_j p_j (sv_j V_j) / sum_j p_j,  p_j = exp(scale q . (sk_j K_j) - m),
// over the tokens j <= position of the row (and inside its window), with the
// running maximum m and the sums in f32, in one pass over the cache.
#include "attn.cuh"
#include "kernels.h"

namespace jmoe {
namespace {

constexpr int kSimpleWarps = 4;

// One warp per (row, query head): lanes split the head's values, tokens go by
// one after another.
template <int D, typename T>
__global__ void __launch_bounds__(kSimpleWarps * 32) attention_simple_kernel(const __grid_constant__ AttnParams p)
{
    __shared__ float s_q[kSimpleWarps][D];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const KvCacheDev &c = p.c;
    if (blockIdx.x == 0)
        for (int s = threadIdx.x; s < p.b.B; s += blockDim.x) {
            SeqInfo q;
            int slot;
            if (!seq_info(p.b, s, q) || !seq_in_cache(c, p.b, s, q, slot)) kv_error(p.err);
        }
    const int64_t item = (int64_t)blockIdx.x * kSimpleWarps + warp;
    const int row = (int)(item / p.rows.q_heads), head = (int)(item - (int64_t)row * p.rows.q_heads);
    if (row >= p.b.T) return;
    int lo = 0, hi = p.b.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (row_of(p.b, mid) <= row) lo = mid;
        else hi = mid - 1;
    }
    SeqInfo q;
    int slot;
    if (!seq_info(p.b, lo, q) || row < q.row0 || row >= q.row0 + q.n || !seq_in_cache(c, p.b, lo, q, slot)) return;
    constexpr int N = D / 32;
    const int pos = q.past + row - q.row0, kvh = head / (p.rows.q_heads / c.heads);
    const T *x = static_cast<const T *>(p.rows.q) + row * p.rows.q_stride + head * D;
    float qv[N], o[N], m = -INFINITY, l = 0.0f;
    if (p.use_rope) {
        norm_rope_head<D>(x, p.rope.q_norm, p.rope, pos, s_q[warp], lane);
#pragma unroll
        for (int i = 0; i < N; i++) qv[i] = s_q[warp][lane * N + i];
    } else {
        load_vals<N>(x + lane * N, qv);
    }
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = 0.0f;
    const int first = p.window ? max(0, pos - p.window + 1) : 0;
    for (int blk = first / kKvBlock; blk <= pos / kKvBlock; blk++) {
        const int64_t at = block_index(c, slot, blk, kvh);
        if (at < 0) {
            if (lane == 0) kv_error(p.err);
            continue;
        }
        const float ks = __ldg(c.k_scale + at) * p.scale, vs = __ldg(c.v_scale + at);
        const int8_t *kb = c.k + at * kKvBlock * D, *vb = c.v + at * kKvBlock * D;
        for (int t = max(0, first - blk * kKvBlock); t <= min(kKvBlock - 1, pos - blk * kKvBlock); t++) {
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int d = lane * N + i;
                dot = fmaf(qv[i], (float)kb[d / 64 * 1024 + t * 64 + d % 64], dot);
            }
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
            dot *= ks;
            const float mn = fmaxf(m, dot), a = __expf(m - mn), w = __expf(dot - mn);
            m = mn;
            l = l * a + w;
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = o[i] * a + w * vs * (float)vb[(lane * N + i) * kKvBlock + t];
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = l > 0.0f ? o[i] / l : 0.0f;
    store_vals<N>(static_cast<T *>(p.out) + row * p.out_stride + head * D + lane * N, o);
}

template <typename T>
cudaError_t launch_t(const AttnParams &p, cudaStream_t st)
{
    const int64_t items = (int64_t)p.b.T * p.rows.q_heads;
    const unsigned grid = (unsigned)((items + kSimpleWarps - 1) / kSimpleWarps);
    if (p.c.D == 64) attention_simple_kernel<64, T><<<grid, kSimpleWarps * 32, 0, st>>>(p);
    else attention_simple_kernel<128, T><<<grid, kSimpleWarps * 32, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

size_t attn_workspace_bytes(int) { return 256; }

cudaError_t launch_attention(const AttnParams &p, cudaStream_t st)
{
    switch (p.rows.act) {
    case MOE_ACT_F32: return launch_t<float>(p, st);
    case MOE_ACT_F16: return launch_t<__half>(p, st);
    default: return launch_t<__nv_bfloat16>(p, st);
    }
}

}  // namespace jmoe
