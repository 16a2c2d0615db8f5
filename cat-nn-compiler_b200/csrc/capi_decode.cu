// extern "C" entry points of the decoding operators (declared in
// include/catnn_b200.h): argument validation, then the launchers of
// qk_norm.cu, paged_attention.cu and moe_few.cu. Device memory that a call
// needs comes from its caller, so nothing here touches the context's arenas.
#include <climits>

#include "ops.cuh"

using namespace catnn;

namespace {

void need(bool ok, const char* what) { CATNN_CHECK(ok, CATNN_ERR_INVALID, std::string("null argument: ") + what); }
void shape(bool ok, const std::string& what) { CATNN_CHECK(ok, CATNN_ERR_SHAPE, what); }

constexpr int SLOT_APPEND = 14, SLOT_PAGED = 15;

// n values of a size that a kernel indexes with 32 bits
bool in32(i64 v) { return v >= 0 && v <= INT_MAX; }

void workspace_ok(const void* p, size_t have, size_t want, const char* what) {
    if (want == 0) return;
    CATNN_CHECK(p && have >= want, CATNN_ERR_INVALID,
                std::string(what) + ": workspace of " + std::to_string(have) + " bytes, " + std::to_string(want) + " needed");
    CATNN_CHECK(aligned_to(p, 256), CATNN_ERR_INVALID, std::string(what) + ": workspace must be 256-byte aligned");
}

void heads_ok(i64 b, i64 s, i64 h, i64 hkv, i64 hd, const char* what) {
    shape(in32(b) && in32(s) && in32(b * s) && h >= 1 && h <= 16384 && hkv >= 1 && hkv <= 16384 && hd >= 1 && hd <= 16384,
          std::string(what) + ": sizes");
}

void stride_ok(i64 stride, i64 tokens, i64 width, const char* what) {
    shape(stride >= width || tokens <= 1, std::string(what) + ": token stride below the row");
}

// Clears a status word before a checked launch; an unchecked launch gets none.
int* flag(Context* c, int check, int slot) {
    if (!check) return nullptr;
    CUDA_OK(cudaMemsetAsync(c->status + slot, 0, 4, c->stream));
    return c->status + slot;
}

// Positions of a table, with the tile that follows the last one, stay below 2^31.
void cache_ok(i64 pages, i64 page, i64 max_pages, const char* what) {
    shape(in32(pages) && page >= 1 && in32(page) && in32(max_pages) && (max_pages == 0 || page <= (INT_MAX - 1024) / max_pages),
          std::string(what) + ": a table must address fewer than 2^31 positions of pages of at least one slot");
}

// Whether [p, p + n) and [q, q + m) share a byte.
bool overlap(const void* p, i64 n, const void* q, i64 m) { return (const char*)p < (const char*)q + m && (const char*)q < (const char*)p + n; }

}  // namespace

extern "C" {

int catnn_qk_norm_rope_fwd(catnn_ctx* h, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const float* wq,
                           const float* wk, const int32_t* positions, void* q_out, void* k_out, int64_t b, int64_t s,
                           int64_t n_heads, int64_t n_kv, int64_t hd, double theta, float eps, int dtype) {
    ABI_BEGIN
    Context* c = unwrap(h);
    check_dtype(dtype);
    heads_ok(b, s, n_heads, n_kv, hd, "qk_norm_rope");
    shape(theta > 0.0, "qk_norm_rope: theta must be positive");
    if (b * s == 0) return CATNN_OK;
    need(q && k && wq && wk && q_out && k_out, "q/k/wq/wk/q_out/k_out");
    stride_ok(q_stride, b * s, n_heads * hd, "qk_norm_rope q");
    stride_ok(k_stride, b * s, n_kv * hd, "qk_norm_rope k");
    qk_norm_rope_fwd(c, q, q_stride, k, k_stride, wq, wk, positions, q_out, k_out, b, s, n_heads, n_kv, hd, theta, eps, dtype);
    ABI_END
}

int catnn_qk_norm_rope_bwd_workspace(catnn_ctx* h, int64_t b, int64_t s, int64_t n_heads, int64_t n_kv, int64_t hd,
                                     size_t* bytes) {
    ABI_BEGIN
    Context* c = unwrap(h);
    need(bytes, "bytes");
    heads_ok(b, s, n_heads, n_kv, hd, "qk_norm_rope backward");
    *bytes = qk_norm_rope_bwd_workspace(c, b, s, n_heads, n_kv, hd);
    ABI_END
}

int catnn_qk_norm_rope_bwd(catnn_ctx* h, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const float* wq,
                           const float* wk, const int32_t* positions, const void* dq_out, int64_t dq_out_stride,
                           const void* dk_out, int64_t dk_out_stride, void* dq, void* dk, float* dwq, float* dwk, int64_t b,
                           int64_t s, int64_t n_heads, int64_t n_kv, int64_t hd, double theta, float eps, int dtype,
                           void* workspace, size_t workspace_bytes) {
    ABI_BEGIN
    Context* c = unwrap(h);
    check_dtype(dtype);
    heads_ok(b, s, n_heads, n_kv, hd, "qk_norm_rope backward");
    shape(theta > 0.0, "qk_norm_rope backward: theta must be positive");
    need(dwq && dwk, "dwq/dwk");
    need(b * s == 0 || (q && k && wq && wk && dq_out && dk_out && dq && dk), "qk_norm_rope_bwd arguments");
    stride_ok(q_stride, b * s, n_heads * hd, "qk_norm_rope backward q");
    stride_ok(k_stride, b * s, n_kv * hd, "qk_norm_rope backward k");
    stride_ok(dq_out_stride, b * s, n_heads * hd, "qk_norm_rope backward dq_out");
    stride_ok(dk_out_stride, b * s, n_kv * hd, "qk_norm_rope backward dk_out");
    workspace_ok(workspace, workspace_bytes, qk_norm_rope_bwd_workspace(c, b, s, n_heads, n_kv, hd), "qk_norm_rope backward");
    qk_norm_rope_bwd(c, q, q_stride, k, k_stride, wq, wk, positions, dq_out, dq_out_stride, dk_out, dk_out_stride, dq, dk, dwq,
                     dwk, b, s, n_heads, n_kv, hd, theta, eps, dtype, (float*)workspace);
    ABI_END
}

int catnn_kv_append(catnn_ctx* h, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                    int64_t v_stride, const float* wq, const float* wk, void* q_out, void* k_cache, void* v_cache,
                    const int32_t* page_table, const int32_t* seq_lens, const int32_t* cu_tokens, int64_t tokens, int64_t seqs,
                    int64_t n_heads, int64_t n_kv, int64_t hd, int64_t n_pages, int64_t page_size, int64_t max_pages,
                    double theta, float eps, int dtype, int check) {
    ABI_BEGIN
    Context* c = unwrap(h);
    check_dtype(dtype);
    heads_ok(tokens, 1, n_heads == 0 ? 1 : n_heads, n_kv, hd, "kv_append");
    shape(in32(seqs), "kv_append: sizes");
    shape(theta > 0.0, "kv_append: theta must be positive");
    cache_ok(n_pages, page_size, max_pages, "kv_append");
    shape(cu_tokens || tokens == seqs, "kv_append: without cu_tokens every sequence has one new token");
    if (tokens == 0) return CATNN_OK;
    need(k && v && (n_pages == 0 || (k_cache && v_cache)), "k/v/k_cache/v_cache");
    need((q != nullptr) == (n_heads > 0) && (q != nullptr) == (q_out != nullptr), "q, q_out and n_heads go together");
    need(seqs == 0 || (seq_lens && (max_pages == 0 || page_table)), "page_table/seq_lens");
    CATNN_CHECK((wq != nullptr) == (wk != nullptr), CATNN_ERR_INVALID, "kv_append: both norm weights or neither");
    if (q) stride_ok(q_stride, tokens, n_heads * hd, "kv_append q");
    stride_ok(k_stride, tokens, n_kv * hd, "kv_append k");
    stride_ok(v_stride, tokens, n_kv * hd, "kv_append v");
    kv_append(c, q, q_stride, k, k_stride, v, v_stride, wq, wk, q_out, k_cache, v_cache, page_table, seq_lens, cu_tokens,
              tokens, seqs, n_heads, n_kv, hd, n_pages, page_size, max_pages, theta, eps, dtype, flag(c, check, SLOT_APPEND));
    if (check && take_status(c, SLOT_APPEND))
        throw Error(CATNN_ERR_SHAPE, "kv_append: a position has no page in the table or the pool");
    ABI_END
}

int catnn_paged_attention_workspace(catnn_ctx* h, int64_t seqs, int64_t n_heads, int64_t n_kv, int64_t hd, int dtype,
                                    size_t* bytes) {
    ABI_BEGIN
    Context* c = unwrap(h);
    check_dtype(dtype);
    need(bytes, "bytes");
    heads_ok(seqs, 1, n_heads, n_kv, hd, "paged_attention");
    shape(n_heads % n_kv == 0, "paged_attention: n_heads must be a multiple of n_kv");
    *bytes = paged_attention_workspace(c, seqs, n_heads, n_kv, hd, dtype);
    ABI_END
}

int catnn_paged_attention_fwd(catnn_ctx* h, const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                              const int32_t* page_table, const int32_t* seq_lens, void* o, float* lse, int64_t seqs,
                              int64_t n_heads, int64_t n_kv, int64_t hd, int64_t n_pages, int64_t page_size, int64_t max_pages,
                              int64_t window, int dtype, void* workspace, size_t workspace_bytes, int check) {
    ABI_BEGIN
    Context* c = unwrap(h);
    check_dtype(dtype);
    heads_ok(seqs, 1, n_heads, n_kv, hd, "paged_attention");
    shape(n_heads % n_kv == 0, "paged_attention: n_heads must be a multiple of n_kv");
    CATNN_CHECK(hd <= 128, CATNN_ERR_UNSUPPORTED, "paged_attention: head_dim must be in [1, 128]");
    shape(in32(seqs * n_heads), "paged_attention: too many heads for one call");
    cache_ok(n_pages, page_size, max_pages, "paged_attention");
    if (seqs == 0) return CATNN_OK;
    need(q && o && lse && seq_lens, "q/o/lse/seq_lens");
    need(max_pages == 0 || n_pages == 0 || (k_cache && v_cache && page_table), "k_cache/v_cache/page_table");
    stride_ok(q_stride, seqs, n_heads * hd, "paged_attention q");
    if (window <= 0 || window > INT_MAX) window = 0;  // none, or longer than any table's positions
    workspace_ok(workspace, workspace_bytes, paged_attention_workspace(c, seqs, n_heads, n_kv, hd, dtype), "paged_attention");
    paged_attention(c, q, q_stride, k_cache, v_cache, page_table, seq_lens, o, lse, seqs, n_heads, n_kv, hd, n_pages, page_size,
                    n_pages == 0 ? 0 : max_pages, window, dtype, workspace, flag(c, check, SLOT_PAGED));
    if (check && take_status(c, SLOT_PAGED))
        throw Error(CATNN_ERR_SHAPE, "paged_attention: a position has no page in the table or the pool");
    ABI_END
}

int catnn_moe_few_workspace(catnn_ctx* h, int64_t T, int64_t hidden, int64_t mid, int64_t E, int64_t k, int dtype,
                            size_t* bytes) {
    ABI_BEGIN
    Context* c = unwrap(h);
    check_dtype(dtype);
    need(bytes, "bytes");
    shape(T >= 0 && T <= CATNN_MOE_FEW_MAX_TOKENS && E >= 1 && E <= 32 && k >= 1 && k <= E && hidden >= 1 && in32(hidden) &&
              mid >= 1 && in32(mid),
          "moe_few: need at most 64 tokens and 1 <= k <= E <= 32");
    *bytes = moe_few_workspace(c, T, hidden, mid, E, k, dtype);
    ABI_END
}

int catnn_moe_few_fwd(catnn_ctx* h, const void* x, const void* gate, const void* w1s, const void* w3s, const void* w2s,
                      void* y, int64_t T, int64_t hidden, int64_t mid, int64_t E, int64_t k, int dtype, void* workspace,
                      size_t workspace_bytes) {
    ABI_BEGIN
    Context* c = unwrap(h);
    check_dtype(dtype);
    shape(T >= 0 && T <= CATNN_MOE_FEW_MAX_TOKENS && E >= 1 && E <= 32 && k >= 1 && k <= E && hidden >= 1 && in32(hidden) &&
              mid >= 1 && in32(mid),
          "moe_few: need at most 64 tokens and 1 <= k <= E <= 32");
    if (T == 0) return CATNN_OK;
    need(x && gate && w1s && w3s && w2s && y, "moe_few arguments");
    const i64 rows = T * hidden * (i64)dsize(dtype);
    CATNN_CHECK(!overlap(x, rows, y, rows), CATNN_ERR_INVALID, "moe_few: y overlaps x, which both kernels read");
    workspace_ok(workspace, workspace_bytes, moe_few_workspace(c, T, hidden, mid, E, k, dtype), "moe_few");
    moe_few(c, x, gate, w1s, w3s, w2s, y, T, hidden, mid, E, k, dtype, workspace);
    ABI_END
}

int catnn_moe_few_set_timeout_ms(catnn_ctx* h, int64_t ms) {
    ABI_BEGIN
    Context* c = unwrap(h);
    CATNN_CHECK(ms >= 0 && ms <= 3600000, CATNN_ERR_INVALID, "moe_few: timeout must be in [0, 3600000] ms");
    c->few_patience = ms * 2000000ll;  // cycles at 2 GHz
    ABI_END
}

int catnn_moe_few_check(catnn_ctx* h) {
    ABI_BEGIN
    if (take_status(unwrap(h), FEW_STATUS_SLOT)) throw Error(CATNN_ERR_TIMEOUT, "moe_few: a bounded device wait ran out");
    ABI_END
}

}  // extern "C"
