// attn.h -- the attention sublayer (internal): the paged 8-bit KV cache, its
// batches, and the launchers of the kernels in attn_rows.cu (norms, rotation,
// append, read) and attn.cu (attention).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace jmoe {

constexpr int kKvBlock = 16;        // tokens of a cache block (one scale per head)
constexpr int kMaxHeadDim = 128;
constexpr int kErrKvBounds = 5;     // device status: a bad batch entry or page id
// Blocks whose largest magnitude is below this are held as zeros: the scale of
// any other block is then at least 2^-74, far from the f32 denormals.
constexpr float kKvTiny = 1e-20f;

struct KvCacheDev {
    int D, heads, n_pages, n_slots, table_stride;
    int page_shift;                 // log2(blocks of a page)
    const int32_t *table;
    int8_t *k, *v;
    float *k_scale, *v_scale, *open_k, *open_v;
};

struct KvBatchDev {
    int B, T, max_new;
    const int32_t *past, *row_start, *slot;
};

struct RopeDev {
    int R, interleaved;
    double eps, mscale;
    const float *q_norm, *k_norm;
    double inv[kMaxHeadDim / 2];
};

struct AttnRows {
    int act, q_heads, kv_heads;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
};

struct AttnParams {
    KvCacheDev c;
    KvBatchDev b;
    RopeDev rope;                   // queries normed and rotated as they are read when use_rope
    int use_rope;
    AttnRows rows;
    float scale;
    int window;
    void *out;
    int64_t out_stride;
    int *err;
    void *ws;                       // the context's workspace; the status word at its start
    int num_sms;
};

// Bytes of a context's attention workspace.
size_t attn_workspace_bytes(int num_sms);
// Of them, from the start: the status word and the arrival counters, zero between calls.
size_t attn_counter_bytes(int num_sms);

// Attention of the sequences with more than few_rows rows (tokens times query
// heads of a key head) on tcgen05; the others' rows are left alone.
cudaError_t launch_attention_tiles(const AttnParams &p, int few_rows, void *ws, size_t ws_bytes, cudaStream_t st);

cudaError_t launch_qk_norm_rope(const KvBatchDev &b, const RopeDev &rope, const AttnRows &in, const AttnRows &out, int D,
                                int *err, cudaStream_t st);
cudaError_t launch_kv_append(const KvCacheDev &c, const KvBatchDev &b, const RopeDev *rope, const AttnRows &rows, int *err,
                             cudaStream_t st);
cudaError_t launch_kv_read(const KvCacheDev &c, const KvBatchDev &b, const AttnRows &out, int *err, cudaStream_t st);
cudaError_t launch_attention(const AttnParams &p, cudaStream_t st);

}  // namespace jmoe
