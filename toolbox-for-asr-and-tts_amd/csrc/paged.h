// Paged cache of keys and values, the attention over it and the choice of a token: kernel parameter blocks and launchers.
#pragma once

#include "common.h"

namespace asrfe {

// the cache and the batch's place in it, as every kernel here takes them (see asrfe_kv_cache)
struct PagedView {
    char* k;
    char* v;
    uint8_t* k_exp;
    uint8_t* v_exp;
    int n_pages, page_shift, n_heads;
    const int32_t* cu_q;
    const int32_t* kv_lens;
    const int32_t* block_table;
    int table_stride, batch;
};

struct KvAppendParams {
    PagedView c;
    const uint16_t* k;
    const uint16_t* v;
    int64_t k_ts, k_hs, v_ts, v_hs;  // element strides
    int n_tokens;
};

struct KvReadParams {
    PagedView c;
    int t_max;
    uint16_t* k;
    uint16_t* v;
};

struct PagedAttnParams {
    PagedView c;
    const uint16_t* q;
    int64_t q_ts, q_hs, o_ts, o_hs;  // element strides
    uint16_t* out;
    int n_tokens, n_q_heads, group;  // group = n_q_heads / n_heads
    int max_kv, window, sinks, causal;
    float scale_log2;                // scale * log2(e)
};

struct SampleParams {
    const void* logits;
    int64_t ld;
    int rows, vocab;
    const float* u;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const int32_t* token_num;
    int rows_per;
    int32_t* ids;
    float* logprobs;
};

int32_t launch_kv_append(asrfe_ctx* ctx, const KvAppendParams& p, int head_dim, int dtype, bool e4m3, hipStream_t s);
int32_t launch_kv_read(asrfe_ctx* ctx, const KvReadParams& p, int head_dim, int dtype, bool e4m3, hipStream_t s);
int64_t paged_attention_workspace(const asrfe_ctx* ctx, int head_dim, bool e4m3, int n_heads, int n_tokens, int n_q_heads, int batch, int max_kv);
// max_kv: the caller's number, which shapes the launch and the workspace (p.max_kv is cut to the table's width)
int32_t launch_paged_attention(asrfe_ctx* ctx, const PagedAttnParams& p, int head_dim, int dtype, bool e4m3, void* ws, int max_kv,
                               hipStream_t s);
int32_t launch_sample(asrfe_ctx* ctx, const SampleParams& p, int dtype, hipStream_t s);

}  // namespace asrfe
