// serve_capi.cpp -- extern "C" entry points of the operators around the packed linears: the
// 8-bit paged cache, its attention and token log probabilities (declared in
// include/ojasx_e8t.h).  Checks arguments, then enqueues on the caller's stream; allocates
// nothing.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/ojasx_e8t.h"
#include "serve.h"

#define OJX_API __attribute__((visibility("default")))

namespace {

using ojx::api_failf;

bool valid_dtype(int dt) { return dt == OJX_F32 || dt == OJX_F16 || dt == OJX_BF16; }

// Sizes that the kernels' 32-bit arithmetic relies on.
constexpr int64_t kMaxCount = (int64_t)1 << 30;

bool misaligned(const void* p, uintptr_t unit) { return ((uintptr_t)p & (unit - 1)) != 0; }

int check_cache(const void* k, const void* v, const void* scales, int64_t num_blocks,
                int64_t kv_heads, int64_t block_size, int64_t head_dim) {
    if (num_blocks < 0 || num_blocks > kMaxCount)
        return api_failf(OJX_EINVAL, "num_blocks %lld is outside 0..2^30", (long long)num_blocks);
    if (kv_heads < 1 || kv_heads > ojx::kKvMaxHeads)
        return api_failf(OJX_EINVAL, "kv_heads %lld is outside 1..%d", (long long)kv_heads,
                        (int)ojx::kKvMaxHeads);
    if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128 &&
        block_size != 256)
        return api_failf(OJX_ELAYOUT, "block_size must be 16, 32, 64, 128 or 256 (got %lld)",
                        (long long)block_size);
    if (head_dim < 1 || head_dim > 256)
        return api_failf(OJX_ELAYOUT, "head_dim %lld is outside 1..256", (long long)head_dim);
    if (num_blocks > 0 && (!k || !v || !scales))
        return api_failf(OJX_EINVAL, "null cache pointer");
    if (misaligned(k, 16) || misaligned(v, 16) || misaligned(scales, 8))
        return api_failf(OJX_ELAYOUT, "codes must be 16-byte aligned, scales 8-byte");
    return OJX_OK;
}

ojx::KvCache cache_of(const int8_t* k, const int8_t* v, const float* scales, int64_t num_blocks,
                      int64_t kv_heads, int64_t block_size, int64_t head_dim) {
    ojx::KvCache c;
    c.k = const_cast<int8_t*>(k);
    c.v = const_cast<int8_t*>(v);
    c.scales = const_cast<float*>(scales);
    c.blocks = (int)num_blocks;
    c.heads = (int)kv_heads;
    c.log_block = __builtin_ctzll((unsigned long long)block_size);
    c.d = (int)head_dim;
    c.dp = (int)((head_dim + 63) / 64 * 64);
    return c;
}

int check_attention(int64_t tokens, int64_t requests, int64_t heads, int64_t kv_heads,
                    int64_t head_dim, int64_t window, int64_t max_query_len, int64_t max_seq_len,
                    int dtype) {
    if (!valid_dtype(dtype)) return api_failf(OJX_EDTYPE, "unknown dtype code %d", dtype);
    if (tokens < 0 || tokens > kMaxCount || requests < 0 || requests > kMaxCount)
        return api_failf(OJX_EINVAL, "%lld tokens of %lld requests", (long long)tokens,
                        (long long)requests);
    if (kv_heads < 1 || kv_heads > ojx::kKvMaxHeads || heads < 1 || heads > ojx::kKvMaxHeads ||
        heads % kv_heads != 0)
        return api_failf(OJX_EINVAL, "%lld heads over %lld key heads", (long long)heads,
                        (long long)kv_heads);
    if (head_dim < 1 || head_dim > 256)
        return api_failf(OJX_ELAYOUT, "head_dim %lld is outside 1..256", (long long)head_dim);
    if (window < 0) return api_failf(OJX_EINVAL, "negative window %lld", (long long)window);
    if (max_query_len < 0 || max_query_len > kMaxCount || max_seq_len < 0 ||
        max_seq_len > kMaxCount)
        return api_failf(OJX_EINVAL, "max_query_len %lld, max_seq_len %lld",
                        (long long)max_query_len, (long long)max_seq_len);
    return OJX_OK;
}

// Of windows that no key seen is outside of, the kernels have none.  One longer than max_seq_len is
// not one: a request may have more tokens than its table's blocks hold.
int window_of(int64_t window) { return window > kMaxCount ? 0 : (int)window; }

int check_logits(int64_t ld, int64_t rows, int64_t vocab, int64_t top_k, int dtype) {
    if (!valid_dtype(dtype)) return api_failf(OJX_EDTYPE, "unknown dtype code %d", dtype);
    if (rows < 0 || rows > kMaxCount || vocab < 1 || vocab > kMaxCount)
        return api_failf(OJX_EINVAL, "%lld rows of %lld logits", (long long)rows, (long long)vocab);
    if (ld < vocab && rows > 1)
        return api_failf(OJX_EINVAL, "row stride %lld is under the row's %lld logits", (long long)ld,
                        (long long)vocab);
    if (top_k < 0 || top_k > ojx::kTopMax || top_k > vocab)
        return api_failf(OJX_EINVAL, "top_k %lld is outside 0..%lld", (long long)top_k,
                        (long long)(vocab < ojx::kTopMax ? vocab : ojx::kTopMax));
    return OJX_OK;
}

int check_workspace(const void* ws, size_t bytes) {
    if (bytes > 0 && !ws)
        return api_failf(OJX_EINVAL, "workspace_bytes %zu with a null workspace", bytes);
    if (misaligned(ws, 16)) return api_failf(OJX_ELAYOUT, "workspace must be 16-byte aligned");
    return OJX_OK;
}

}  // namespace

extern "C" {

OJX_API int ojx_kv8_plan(const int32_t* seq_lens, const int32_t* new_lens, int64_t requests,
                         int32_t* block_tables, int64_t table_ld, int64_t table_width,
                         const int32_t* free_blocks, int64_t free_capacity,
                         const int32_t* num_free, int64_t block_size, int64_t tokens,
                         int64_t* slots, int32_t* positions, int32_t* request_ids,
                         int32_t* query_starts, int32_t* seq_lens_out, int32_t* num_free_out,
                         void* stream) {
    if (requests < 0 || requests > kMaxCount || tokens < 0 || tokens > kMaxCount ||
        table_width < 0 || table_width > kMaxCount || free_capacity < 0 ||
        free_capacity > kMaxCount)
        return api_failf(OJX_EINVAL, "%lld requests, %lld tokens, %lld table columns, %lld blocks",
                        (long long)requests, (long long)tokens, (long long)table_width,
                        (long long)free_capacity);
    if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128 &&
        block_size != 256)
        return api_failf(OJX_ELAYOUT, "block_size must be 16, 32, 64, 128 or 256 (got %lld)",
                        (long long)block_size);
    if (table_ld < table_width && requests > 1)
        return api_failf(OJX_EINVAL, "table stride %lld is under its width %lld",
                        (long long)table_ld, (long long)table_width);
    if (!num_free || !num_free_out || !query_starts || (free_capacity > 0 && !free_blocks) ||
        (requests > 0 && (!seq_lens || !new_lens || !seq_lens_out)) ||
        (requests > 0 && table_width > 0 && !block_tables) ||
        (tokens > 0 && (!slots || !positions || !request_ids)))
        return api_failf(OJX_EINVAL, "null pointer");
    if (int r = ojx::api_check_device()) return r;
    ojx::PlanArgs a;
    a.seq_lens = seq_lens;
    a.new_lens = new_lens;
    a.tables = block_tables;
    a.free_blocks = free_blocks;
    a.num_free = num_free;
    a.slots = slots;
    a.positions = positions;
    a.request_ids = request_ids;
    a.query_starts = query_starts;
    a.seq_lens_out = seq_lens_out;
    a.num_free_out = num_free_out;
    a.table_ld = table_ld;
    a.requests = (int)requests;
    a.width = (int)table_width;
    a.capacity = (int)free_capacity;
    a.log_block = __builtin_ctzll((unsigned long long)block_size);
    a.tokens = (int)tokens;
    return ojx::api_done(ojx::launch_kv8_plan(a, (hipStream_t)stream), "kv8 plan launch");
}

OJX_API int ojx_kv8_append(int8_t* k_codes, int8_t* v_codes, float* scales, int64_t num_blocks,
                           int64_t kv_heads, int64_t block_size, int64_t head_dim, const void* k,
                           int64_t k_token_stride, int64_t k_head_stride, const void* v,
                           int64_t v_token_stride, int64_t v_head_stride, int dtype,
                           const int64_t* slots, int64_t tokens, void* stream) {
    if (!valid_dtype(dtype)) return api_failf(OJX_EDTYPE, "unknown dtype code %d", dtype);
    if (int r = check_cache(k_codes, v_codes, scales, num_blocks, kv_heads, block_size, head_dim))
        return r;
    if (tokens < 0 || tokens > kMaxCount)
        return api_failf(OJX_EINVAL, "%lld tokens", (long long)tokens);
    if (tokens == 0) return OJX_OK;
    if (!k || !v || !slots) return api_failf(OJX_EINVAL, "null pointer");
    if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0)
        return api_failf(OJX_EINVAL, "negative stride");
    if (int r = ojx::api_check_device()) return r;
    const ojx::KvCache c = cache_of(k_codes, v_codes, scales, num_blocks, kv_heads, block_size,
                                    head_dim);
    const ojx::KvRows kr{k, k_token_stride, k_head_stride}, vr{v, v_token_stride, v_head_stride};
    return ojx::api_done(
        ojx::launch_kv8_append(c, kr, vr, dtype, slots, (int)tokens, (hipStream_t)stream),
        "kv8 append launch");
}

OJX_API int ojx_kv8_read(const int8_t* k_codes, const int8_t* v_codes, const float* scales,
                         int64_t num_blocks, int64_t kv_heads, int64_t block_size,
                         int64_t head_dim, const int32_t* blocks, int64_t n, int dtype,
                         void* k_out, void* v_out, float* scales_out, void* stream) {
    if (!valid_dtype(dtype)) return api_failf(OJX_EDTYPE, "unknown dtype code %d", dtype);
    if (int r = check_cache(k_codes, v_codes, scales, num_blocks, kv_heads, block_size, head_dim))
        return r;
    if (n < 0 || n > kMaxCount) return api_failf(OJX_EINVAL, "%lld blocks", (long long)n);
    if (n == 0) return OJX_OK;
    if (!blocks || !k_out || !v_out || !scales_out) return api_failf(OJX_EINVAL, "null pointer");
    if (misaligned(k_out, 16) || misaligned(v_out, 16))
        return api_failf(OJX_ELAYOUT, "outputs must be 16-byte aligned");
    if (int r = ojx::api_check_device()) return r;
    const ojx::KvCache c = cache_of(k_codes, v_codes, scales, num_blocks, kv_heads, block_size,
                                    head_dim);
    return ojx::api_done(
        ojx::launch_kv8_read(c, blocks, (int)n, dtype, k_out, v_out, scales_out,
                             (hipStream_t)stream),
        "kv8 read launch");
}

OJX_API int ojx_kv8_attention_workspace_bytes(int64_t tokens, int64_t requests, int64_t heads,
                                              int64_t kv_heads, int64_t head_dim, int64_t window,
                                              int64_t max_query_len, int64_t max_seq_len,
                                              int dtype, size_t* bytes) {
    if (!bytes) return api_failf(OJX_EINVAL, "null pointer");
    *bytes = 0;
    if (int r = check_attention(tokens, requests, heads, kv_heads, head_dim, window, max_query_len,
                                max_seq_len, dtype))
        return r;
    ojx::AttnShape s;
    s.tokens = (int)tokens;
    s.requests = (int)requests;
    s.heads = (int)heads;
    s.kv_heads = (int)kv_heads;
    s.d = (int)head_dim;
    s.window = window_of(window);
    s.max_query = (int)max_query_len;
    s.max_seq = (int)max_seq_len;
    s.dtype = dtype;
    *bytes = ojx::kv8_attention_bytes(s);
    return OJX_OK;
}

OJX_API int ojx_kv8_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                              int64_t tokens, int64_t heads, int dtype, const int8_t* k_codes,
                              const int8_t* v_codes, const float* scales, int64_t num_blocks,
                              int64_t kv_heads, int64_t block_size, int64_t head_dim,
                              const int32_t* block_tables, int64_t table_ld, int64_t table_width,
                              const int32_t* seq_lens, const int32_t* query_starts,
                              int64_t requests, int64_t max_query_len, int64_t max_seq_len,
                              float softmax_scale, int64_t window, void* out, float* lse,
                              void* workspace, size_t workspace_bytes, void* stream) {
    if (int r = check_cache(k_codes, v_codes, scales, num_blocks, kv_heads, block_size, head_dim))
        return r;
    if (int r = check_attention(tokens, requests, heads, kv_heads, head_dim, window, max_query_len,
                                max_seq_len, dtype))
        return r;
    if (int r = check_workspace(workspace, workspace_bytes)) return r;
    if (!std::isfinite(softmax_scale)) return api_failf(OJX_EINVAL, "softmax_scale is not finite");
    if (!query_starts && tokens != requests)
        return api_failf(OJX_EINVAL, "%lld tokens of %lld requests without query_starts",
                        (long long)tokens, (long long)requests);
    if (table_width < 0 || table_width > kMaxCount || (table_ld < table_width && requests > 1))
        return api_failf(OJX_EINVAL, "block table of %lld columns at stride %lld",
                        (long long)table_width, (long long)table_ld);
    if (q_token_stride < 0 || q_head_stride < 0) return api_failf(OJX_EINVAL, "negative stride");
    if (tokens == 0) return OJX_OK;
    if (requests == 0) return api_failf(OJX_EINVAL, "tokens without a request");
    if (!q || !out || !seq_lens || (table_width > 0 && !block_tables))
        return api_failf(OJX_EINVAL, "null pointer");
    if (int r = ojx::api_check_device()) return r;
    ojx::AttnArgs a;
    a.cache = cache_of(k_codes, v_codes, scales, num_blocks, kv_heads, block_size, head_dim);
    a.q = ojx::KvRows{q, q_token_stride, q_head_stride};
    a.tables = block_tables;
    a.table_ld = table_ld;
    a.seq_lens = seq_lens;
    a.query_starts = query_starts;
    a.out = out;
    a.lse = lse;
    a.scale = softmax_scale;
    // tokens past the table have no block
    const int64_t held = table_width * block_size;
    a.width = (int)table_width;
    a.shape.tokens = (int)tokens;
    a.shape.requests = (int)requests;
    a.shape.heads = (int)heads;
    a.shape.kv_heads = (int)kv_heads;
    a.shape.d = (int)head_dim;
    a.shape.window = window_of(window);
    a.shape.max_query = query_starts ? (int)max_query_len : 1;
    a.shape.max_seq = (int)(max_seq_len < held ? max_seq_len : held);
    a.shape.dtype = dtype;
    return ojx::api_done(
        ojx::launch_kv8_attention(a, workspace, workspace_bytes, (hipStream_t)stream),
        "kv8 attention launch");
}

OJX_API int ojx_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top_k,
                                               int dtype, size_t* bytes) {
    if (!bytes) return api_failf(OJX_EINVAL, "null pointer");
    *bytes = 0;
    if (int r = check_logits(vocab, rows, vocab, top_k, dtype)) return r;
    *bytes = ojx::token_logprobs_bytes((int)rows, (int)vocab, (int)top_k, dtype);
    return OJX_OK;
}

OJX_API int ojx_token_logprobs(const void* logits, int64_t ld, int64_t rows, int64_t vocab,
                               int dtype, const int64_t* ids, int64_t top_k, float* logprob,
                               float* entropy, float* lse, float* stats, float* top_logprobs,
                               int64_t* top_ids, void* workspace, size_t workspace_bytes,
                               void* stream) {
    if (int r = check_logits(ld, rows, vocab, top_k, dtype)) return r;
    if (int r = check_workspace(workspace, workspace_bytes)) return r;
    if (rows == 0) return OJX_OK;
    if (!logits || !ids || !logprob || !entropy || !lse || !stats ||
        (top_k > 0 && (!top_logprobs || !top_ids)))
        return api_failf(OJX_EINVAL, "null pointer");
    if (int r = ojx::api_check_device()) return r;
    ojx::LogprobArgs a;
    a.x = logits;
    a.ld = ld;
    a.rows = (int)rows;
    a.vocab = (int)vocab;
    a.dtype = dtype;
    a.top = (int)top_k;
    a.ids = ids;
    a.logprob = logprob;
    a.entropy = entropy;
    a.lse = lse;
    a.stats = stats;
    a.top_lp = top_logprobs;
    a.top_ids = top_ids;
    return ojx::api_done(
        ojx::launch_token_logprobs(a, workspace, workspace_bytes, (hipStream_t)stream),
        "token_logprobs launch");
}

OJX_API int ojx_token_logprobs_bwd(const void* logits, int64_t ld, int64_t rows, int64_t vocab,
                                   int dtype, const int64_t* ids, const float* entropy,
                                   const float* stats, int64_t top_k, const int64_t* top_ids,
                                   const float* grad_logprob, const float* grad_entropy,
                                   const float* grad_lse, const float* grad_top,
                                   void* grad_logits, void* stream) {
    if (int r = check_logits(ld, rows, vocab, top_k, dtype)) return r;
    if (rows == 0) return OJX_OK;
    if (!logits || !ids || !entropy || !stats || !grad_logits || (top_k > 0 && grad_top && !top_ids))
        return api_failf(OJX_EINVAL, "null pointer");
    if (int r = ojx::api_check_device()) return r;
    ojx::LogprobGradArgs a;
    a.x = logits;
    a.ld = ld;
    a.rows = (int)rows;
    a.vocab = (int)vocab;
    a.dtype = dtype;
    a.top = grad_top ? (int)top_k : 0;
    a.ids = ids;
    a.entropy = entropy;
    a.stats = stats;
    a.top_ids = top_ids;
    a.g_lp = grad_logprob;
    a.g_h = grad_entropy;
    a.g_lse = grad_lse;
    a.g_top = grad_top;
    a.gx = grad_logits;
    return ojx::api_done(ojx::launch_token_logprobs_bwd(a, (hipStream_t)stream),
                         "token_logprobs_bwd launch");
}

}  // extern "C"
