// Entry points of the paged key / value cache, the attention over it and the choice of a token: argument checks only.
// Nothing here allocates or waits; what lies in device memory (lengths, page numbers) is checked by the kernels, which
// skip what does not exist.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "paged.h"

using namespace asrfe;

namespace {
int32_t bad(asrfe_ctx* ctx, int32_t code, const char* who, const char* what) {
    return set_err(ctx, code, std::string(who) + ": " + what);
}

// (asked last: what is wrong with the arguments alone is then told without a device, too)
int32_t on_device(asrfe_ctx* ctx, const char* who) {
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess || dev != ctx->device)
        return bad(ctx, ASRFE_ERR_BAD_ARG, who, "the context belongs to another device than the current one");
    return ASRFE_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Checks what the entry points share and fills the kernels' view of the cache.
int32_t view_of(asrfe_ctx* ctx, const char* who, const asrfe_kv_cache* c, int32_t dtype, const int32_t* cu_q, const int32_t* kv_lens,
                const int32_t* block_table, int32_t table_stride, int32_t batch, PagedView* out) {
    if (!c) return bad(ctx, ASRFE_ERR_BAD_ARG, who, "null cache");
    if (c->dtype != ASRFE_DT_F16 && c->dtype != ASRFE_DT_BF16 && c->dtype != ASRFE_DT_E4M3)
        return bad(ctx, ASRFE_ERR_BAD_ARG, who, "the cache's dtype must be F16, BF16 or E4M3");
    if (dtype != ASRFE_DT_F16 && dtype != ASRFE_DT_BF16) return bad(ctx, ASRFE_ERR_BAD_ARG, who, "dtype must be F16 or BF16");
    if (c->dtype != ASRFE_DT_E4M3 && dtype != c->dtype) return bad(ctx, ASRFE_ERR_BAD_ARG, who, "a 16-bit cache takes and gives its own dtype only");
    if (c->head_dim != 64 && c->head_dim != 128) return bad(ctx, ASRFE_ERR_SHAPE, who, "head_dim must be 64 or 128");
    int shift = 4;
    while (shift < 8 && (1 << shift) != c->page_size) ++shift;
    if ((1 << shift) != c->page_size) return bad(ctx, ASRFE_ERR_SHAPE, who, "page_size must be 16, 32, 64, 128 or 256");
    if (c->n_heads < 1 || c->n_heads > 256) return bad(ctx, ASRFE_ERR_SHAPE, who, "1 to 256 key / value heads");
    if (c->n_pages < 1) return bad(ctx, ASRFE_ERR_SHAPE, who, "the cache has no pages");
    if ((static_cast<int64_t>(c->n_pages) * c->n_heads << shift) > UINT32_MAX) return bad(ctx, ASRFE_ERR_SHAPE, who, "the cache has 2^32 rows or more");
    if (batch < 0 || batch > 65535 || table_stride < 0 || table_stride > ((1 << 30) >> shift))
        return bad(ctx, ASRFE_ERR_SHAPE, who, "batch in 0..65535, table_stride >= 0 with at most 2^30 positions in a row of the table");
    if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v)) return bad(ctx, ASRFE_ERR_BAD_ARG, who, "the cache's k and v must be 16-byte aligned");
    if ((c->dtype == ASRFE_DT_E4M3) != (c->k_exp != nullptr) || (c->dtype == ASRFE_DT_E4M3) != (c->v_exp != nullptr))
        return bad(ctx, ASRFE_ERR_BAD_ARG, who, "k_exp and v_exp belong to an E4M3 cache and to no other");
    if (!aligned16(c->k_exp) || !aligned16(c->v_exp)) return bad(ctx, ASRFE_ERR_BAD_ARG, who, "k_exp and v_exp must be 16-byte aligned");
    if (batch > 0 && (!kv_lens || !cu_q || (table_stride > 0 && !block_table))) return bad(ctx, ASRFE_ERR_BAD_ARG, who, "null argument");
    out->k = static_cast<char*>(c->k);
    out->v = static_cast<char*>(c->v);
    out->k_exp = c->k_exp;
    out->v_exp = c->v_exp;
    out->n_pages = c->n_pages;
    out->page_shift = shift;
    out->n_heads = c->n_heads;
    out->cu_q = cu_q;
    out->kv_lens = kv_lens;
    out->block_table = block_table;
    out->table_stride = table_stride;
    out->batch = batch;
    return ASRFE_OK;
}

bool stride_ok(int64_t s) { return s >= 0 && s % 8 == 0; }

// Whether no two of the n x heads rows of `dim` elements at t * ts + h * hs share an element.  Mostly one stride spans all rows
// of the other; else every distance of heads is held against the distances of tokens next to it.
bool rows_apart(int64_t n, int64_t heads, int64_t dim, int64_t ts, int64_t hs) {
    if ((n > 1 && ts < dim) || (heads > 1 && hs < dim)) return false;
    if (n <= 1 || heads <= 1) return true;
    if (ts >> 38 || hs >> 38) return false;  // (no memory is that large, and the products below stay inside 64 bits)
    if (ts >= (heads - 1) * hs + dim || hs >= (n - 1) * ts + dim) return true;
    for (int64_t h = 1; h < heads; ++h) {
        const int64_t t = std::min(h * hs / ts, n - 1);
        if (std::abs(h * hs - t * ts) < dim || (t + 1 < n && std::abs((t + 1) * ts - h * hs) < dim)) return false;
    }
    return true;
}
}  // namespace

extern "C" int32_t asrfe_kv_append(asrfe_ctx* ctx, const asrfe_kv_cache* cache, const void* k, const void* v, int32_t dtype,
                                   int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                   int32_t n_tokens, const int32_t* cu_q, const int32_t* kv_lens, const int32_t* block_table,
                                   int32_t table_stride, int32_t batch, void* stream) {
    constexpr const char* kWho = "asrfe_kv_append";
    if (!ctx) return ASRFE_ERR_BAD_ARG;
    KvAppendParams p{};
    if (int32_t rc = view_of(ctx, kWho, cache, dtype, cu_q, kv_lens, block_table, table_stride, batch, &p.c)) return rc;
    if (n_tokens < 0 || n_tokens > (1 << 24)) return bad(ctx, ASRFE_ERR_SHAPE, kWho, "n_tokens in 0..2^24");
    if (n_tokens == 0 || batch == 0 || table_stride == 0) return ASRFE_OK;
    if (!k || !v || !aligned16(k) || !aligned16(v)) return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "k and v must be 16-byte aligned");
    if (!stride_ok(k_token_stride) || !stride_ok(k_head_stride) || !stride_ok(v_token_stride) || !stride_ok(v_head_stride))
        return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "strides must be non-negative multiples of 8 elements");
    if (int32_t rc = on_device(ctx, kWho)) return rc;
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.k_ts = k_token_stride; p.k_hs = k_head_stride; p.v_ts = v_token_stride; p.v_hs = v_head_stride;
    p.n_tokens = n_tokens;
    return launch_kv_append(ctx, p, cache->head_dim, dtype, cache->dtype == ASRFE_DT_E4M3, static_cast<hipStream_t>(stream));
}

extern "C" int32_t asrfe_kv_read(asrfe_ctx* ctx, const asrfe_kv_cache* cache, const int32_t* kv_lens, const int32_t* block_table,
                                 int32_t table_stride, int32_t batch, int32_t t_max, void* k, void* v, int32_t dtype, void* stream) {
    constexpr const char* kWho = "asrfe_kv_read";
    if (!ctx) return ASRFE_ERR_BAD_ARG;
    KvReadParams p{};
    if (t_max < 0 || static_cast<int64_t>(batch) * t_max >= (int64_t{1} << 26))  // (a wave each: a launch holds fewer than 2^32 threads)
        return bad(ctx, ASRFE_ERR_SHAPE, kWho, "t_max >= 0, batch * t_max below 2^26");
    if (int32_t rc = view_of(ctx, kWho, cache, dtype, kv_lens, kv_lens, block_table, table_stride, batch, &p.c)) return rc;
    if (batch == 0 || t_max == 0) return ASRFE_OK;
    if (!k || !v || !aligned16(k) || !aligned16(v)) return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "k and v must be 16-byte aligned");
    if (int32_t rc = on_device(ctx, kWho)) return rc;
    p.t_max = t_max;
    p.k = static_cast<uint16_t*>(k);
    p.v = static_cast<uint16_t*>(v);
    return launch_kv_read(ctx, p, cache->head_dim, dtype, cache->dtype == ASRFE_DT_E4M3, static_cast<hipStream_t>(stream));
}

extern "C" int64_t asrfe_paged_attention_workspace_bytes(const asrfe_ctx* ctx, const asrfe_kv_cache* cache, int32_t n_tokens,
                                                         int32_t n_q_heads, int32_t batch, int32_t max_kv) {
    if (!ctx || !cache || n_tokens < 0 || n_tokens > (1 << 24) || batch < 0 || batch > 65535 || max_kv < 0) return -1;
    if (cache->n_heads < 1 || cache->n_heads > 256 || n_q_heads < 1 || n_q_heads % cache->n_heads != 0 || n_q_heads / cache->n_heads > 256) return -1;
    return paged_attention_workspace(ctx, cache->head_dim, cache->dtype == ASRFE_DT_E4M3, cache->n_heads, n_tokens, n_q_heads, batch, max_kv);
}

extern "C" int32_t asrfe_paged_attention(asrfe_ctx* ctx, const asrfe_kv_cache* cache, const void* q, int32_t dtype, int64_t q_token_stride,
                                         int64_t q_head_stride, int32_t n_tokens, int32_t n_q_heads, const int32_t* cu_q,
                                         const int32_t* kv_lens, const int32_t* block_table, int32_t table_stride, int32_t batch,
                                         int32_t max_kv, int32_t window, int32_t sinks, int32_t causal, float scale, void* out,
                                         int64_t out_token_stride, int64_t out_head_stride, void* workspace, int64_t workspace_bytes,
                                         void* stream) {
    constexpr const char* kWho = "asrfe_paged_attention";
    if (!ctx) return ASRFE_ERR_BAD_ARG;
    PagedAttnParams p{};
    if (int32_t rc = view_of(ctx, kWho, cache, dtype, cu_q, kv_lens, block_table, table_stride, batch, &p.c)) return rc;
    if (n_q_heads < 1 || n_q_heads % cache->n_heads != 0 || n_q_heads / cache->n_heads > 256)
        return bad(ctx, ASRFE_ERR_SHAPE, kWho, "n_q_heads must be a multiple of the cache's heads, up to 256 times as many");
    if (n_tokens < 0 || n_tokens > (1 << 24) || static_cast<int64_t>(n_tokens) * n_q_heads > (int64_t{1} << 30))
        return bad(ctx, ASRFE_ERR_SHAPE, kWho, "n_tokens in 0..2^24, n_tokens * n_q_heads up to 2^30");
    if (max_kv < 0 || window < 0 || sinks < 0) return bad(ctx, ASRFE_ERR_SHAPE, kWho, "max_kv, window and sinks must not be negative");
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!std::isfinite(scale_log2)) return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "scale must be finite, and below 2.3e38");
    if (n_tokens == 0 || batch == 0) return ASRFE_OK;
    if (!q || !out || !aligned16(q) || !aligned16(out)) return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "q and out must be 16-byte aligned");
    if (!stride_ok(q_token_stride) || !stride_ok(q_head_stride) || !stride_ok(out_token_stride) || !stride_ok(out_head_stride))
        return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "strides must be non-negative multiples of 8 elements");
    if (!rows_apart(n_tokens, n_q_heads, cache->head_dim, out_token_stride, out_head_stride))
        return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "the rows of out must not overlap");
    const int64_t need = paged_attention_workspace(ctx, cache->head_dim, cache->dtype == ASRFE_DT_E4M3, cache->n_heads, n_tokens, n_q_heads, batch, max_kv);
    if (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
        return bad(ctx, ASRFE_ERR_WORKSPACE, kWho, "workspace must be 256-byte aligned");
    if (workspace_bytes < need) return bad(ctx, ASRFE_ERR_WORKSPACE, kWho, "workspace too small");
    if (int32_t rc = on_device(ctx, kWho)) return rc;
    p.q = static_cast<const uint16_t*>(q);
    p.out = static_cast<uint16_t*>(out);
    p.q_ts = q_token_stride; p.q_hs = q_head_stride; p.o_ts = out_token_stride; p.o_hs = out_head_stride;
    p.n_tokens = n_tokens;
    p.n_q_heads = n_q_heads;
    p.group = n_q_heads / cache->n_heads;
    p.max_kv = std::min(max_kv, table_stride << p.c.page_shift);  // (at most 2^30: checked above)
    p.window = std::min(window, 1 << 30);
    p.sinks = std::min(sinks, 1 << 30);
    p.causal = causal != 0;
    p.scale_log2 = scale_log2;
    return launch_paged_attention(ctx, p, cache->head_dim, dtype, cache->dtype == ASRFE_DT_E4M3, workspace, max_kv, static_cast<hipStream_t>(stream));
}

extern "C" int32_t asrfe_sample_tokens(asrfe_ctx* ctx, const void* logits, int32_t dtype, int64_t ld, int32_t rows, int32_t vocab,
                                       const float* u, const float* temperature, const int32_t* top_k, const float* top_p,
                                       const float* min_p, const int32_t* token_num, int32_t rows_per, int32_t* ids, float* logprobs,
                                       void* stream) {
    constexpr const char* kWho = "asrfe_sample_tokens";
    if (!ctx) return ASRFE_ERR_BAD_ARG;
    if (dtype != ASRFE_DT_F32 && dtype != ASRFE_DT_F16 && dtype != ASRFE_DT_BF16) return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "dtype must be F32, F16 or BF16");
    if (rows < 0 || rows > (1 << 23) || vocab < 1 || vocab > (1 << 18) || ld < vocab)
        return bad(ctx, ASRFE_ERR_SHAPE, kWho, "rows in 0..2^23, vocab in 1..2^18, ld >= vocab");
    if (token_num && rows_per < 1) return bad(ctx, ASRFE_ERR_SHAPE, kWho, "rows_per must be positive where token_num is given");
    if (rows == 0) return ASRFE_OK;
    if (!logits || !u || !ids) return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "null argument");
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == ASRFE_DT_F32 ? 4 : 2) != 0) return bad(ctx, ASRFE_ERR_BAD_ARG, kWho, "logits must be aligned to their type");
    if (int32_t rc = on_device(ctx, kWho)) return rc;
    SampleParams p{};
    p.logits = logits; p.ld = ld; p.rows = rows; p.vocab = vocab; p.u = u; p.temperature = temperature; p.top_k = top_k;
    p.top_p = top_p; p.min_p = min_p; p.token_num = token_num; p.rows_per = rows_per; p.ids = ids; p.logprobs = logprobs;
    return launch_sample(ctx, p, dtype, static_cast<hipStream_t>(stream));
}
