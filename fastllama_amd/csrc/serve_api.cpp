// serve_api.cpp -- C entry points of the serving operators (include/fastllama_hip.h): every argument that the host can see is checked here, the
// rest (row starts, lengths, page numbers: device data) is cut to the buffers by the kernels.
#include <hip/hip_runtime.h>
#include <cmath>

#include "../../include/fastllama_hip.h"
#include "runtime.h"
#include "serve_kernels.h"

using namespace fl;

#define FL_TRY(call)                                        \
    do {                                                    \
        const int rc_ = (call);                             \
        if (rc_ != FL_OK) return rc_;                       \
    } while (0)

static int size_of(int type) { return type == FL_TYPE_F32 ? 4 : type == FL_TYPE_F16 || type == FL_TYPE_BF16 ? 2 : 0; }
static hipStream_t S(void *s) { return reinterpret_cast<hipStream_t>(s); }
static bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

static int check_dim(const char *fn, int type, int head_dim, int n_head_kv) {
    if (!size_of(type)) return set_error(FL_EINVAL, "%s: type %d is not f32 (0), f16 (1) or bf16 (%d)", fn, type, FL_TYPE_BF16);
    if (head_dim < 8 || head_dim > 128 || head_dim % 8) return set_error(FL_EINVAL, "%s: head_dim %d is not a multiple of 8 in 8..128", fn, head_dim);
    if (n_head_kv < 1 || n_head_kv > 65535) return set_error(FL_EINVAL, "%s: %d key heads", fn, n_head_kv);
    return FL_OK;
}

// Rows are read and written in 16-byte pieces, and 64 of them are within 32 bits of an address.
constexpr int64_t MAX_ROW = 1 << 22;
// Kernels count rows and keys in 32 bits, up to the end of a block (256 rows) or tile (64 keys) that the last one is in.
constexpr int MAX_COUNT = INT32_MAX - 511;
static int check_heads(const char *fn, const char *what, const fl_heads *h, int type, int rows) {
    if (!h || rows < 0) return set_error(FL_EINVAL, "%s: %s: null view or %d rows", fn, what, rows);
    if (rows == 0) return FL_OK;
    if (!h->data_dev) return set_error(FL_EINVAL, "%s: %s: null data", fn, what);
    const int unit = 16 / size_of(type);
    if (!aligned(h->data_dev, 16) || h->token_stride < 0 || h->head_stride < 0 || h->token_stride > MAX_ROW || h->token_stride % unit || h->head_stride % unit)
        return set_error(FL_EINVAL, "%s: %s: data or strides (%lld, %lld) not multiples of 16 bytes, or past 2^22 elements", fn, what, (long long)h->token_stride, (long long)h->head_stride);
    return FL_OK;
}

// ... and where they are written, no two of them share a place.
static int check_out(const char *fn, const char *what, const fl_heads *h, int type, int rows, int n_head) {
    FL_TRY(check_heads(fn, what, h, type, rows));
    if ((rows > 1 && !h->token_stride) || (rows && n_head > 1 && !h->head_stride)) return set_error(FL_EINVAL, "%s: %s: a stride of 0", fn, what);
    return FL_OK;
}

static int check_pages(const char *fn, const fl_kv_pages *c) {
    if (!c) return set_error(FL_EINVAL, "%s: null cache", fn);
    FL_TRY(check_dim(fn, c->type, c->head_dim, c->n_head_kv));
    if (c->page_size < 16 || c->page_size > 65536 || c->page_size & (c->page_size - 1))
        return set_error(FL_EINVAL, "%s: page_size %d is not a power of two in 16..65536", fn, c->page_size);
    if (c->n_pages < 1 || !c->k_dev || !c->v_dev) return set_error(FL_EINVAL, "%s: a cache of %d pages, or null pages", fn, c->n_pages);
    const int unit = 16 / size_of(c->type);
    if (!aligned(c->k_dev, 16) || !aligned(c->v_dev, 16) || c->page_stride < 0 || c->head_stride < 0 || c->slot_stride < 0 || c->slot_stride > MAX_ROW || c->page_stride % unit ||
        c->head_stride % unit || c->slot_stride % unit)
        return set_error(FL_EINVAL, "%s: pages or their strides are not multiples of 16 bytes, or slot_stride past 2^22", fn);
    return FL_OK;
}

static int check_table(const char *fn, const fl_kv_pages *c, const int32_t *table, int table_ld, int n_table, int n_seq) {
    if (n_seq < 1 || n_table < 1 || table_ld < 0 || (n_seq > 1 && table_ld < n_table) || !table)
        return set_error(FL_EINVAL, "%s: page table of %d rows, %d pages each, row stride %d", fn, n_seq, n_table, table_ld);
    if ((int64_t)n_table * c->page_size > 1 << 30) return set_error(FL_EINVAL, "%s: %d pages of %d: more than 2^30 positions", fn, n_table, c->page_size);
    return FL_OK;
}

static int page_shift(const fl_kv_pages *c) { return __builtin_ctz((unsigned)c->page_size); }

extern "C" {

int fl_kv_append(const fl_kv_pages *c, int src_type, const fl_heads *k, const fl_heads *v, int n_tokens, const int32_t *cu_dev, const int32_t *n_past_dev,
                 const int32_t *table_dev, int table_ld, int n_table, int n_seq, void *stream) {
    const char *fn = "fl_kv_append";
    FL_TRY(check_pages(fn, c));
    if (src_type != c->type && src_type != FL_TYPE_F32) return set_error(FL_EINVAL, "%s: rows of type %d into a cache of type %d (want f32 or the cache's)", fn, src_type, c->type);
    FL_TRY(check_heads(fn, "k", k, src_type, n_tokens));
    FL_TRY(check_heads(fn, "v", v, src_type, n_tokens));
    if ((c->n_pages > 1 && !c->page_stride) || (c->n_head_kv > 1 && !c->head_stride) || !c->slot_stride) return set_error(FL_EINVAL, "%s: a stride of 0 in the cache", fn);
    if (n_tokens == 0) return FL_OK;
    FL_TRY(check_table(fn, c, table_dev, table_ld, n_table, n_seq));
    if ((int64_t)n_tokens * c->n_head_kv * (c->head_dim / 8) > UINT32_MAX - 255)         // (a launch has fewer than 2^32 threads)
        return set_error(FL_EINVAL, "%s: %d rows of %d heads of %d: more than 2^35 elements", fn, n_tokens, c->n_head_kv, c->head_dim);
    if (!n_past_dev || (!cu_dev && n_seq != n_tokens)) return set_error(FL_EINVAL, "%s: no n_past, or no row starts for %d rows of %d sequences", fn, n_tokens, n_seq);
    FL_TRY(ensure_device());
    AppendArgs a{};
    a.kc = c->k_dev, a.vc = c->v_dev, a.page_stride = c->page_stride, a.head_stride = c->head_stride, a.slot_stride = c->slot_stride;
    a.k = k->data_dev, a.v = v->data_dev, a.k_ld = k->token_stride, a.k_hs = k->head_stride, a.v_ld = v->token_stride, a.v_hs = v->head_stride;
    a.cu = cu_dev, a.n_past = n_past_dev, a.table = table_dev, a.table_ld = table_ld, a.n_table = n_table, a.page_shift = page_shift(c), a.n_pages = c->n_pages;
    a.n_tok = n_tokens, a.n_seq = n_seq, a.n_head_kv = c->n_head_kv, a.head_dim = c->head_dim;
    const hipError_t e = kv_append(a, src_type, c->type, S(stream));
    return e == hipSuccess ? FL_OK : hip_fail(e, fn);
}

static int fill(AttnArgs &a, const char *fn, int type, int head_dim, int n_head, int n_head_kv, float scale, const fl_heads *q, const fl_heads *out, int n_q, int n_seq) {
    FL_TRY(check_dim(fn, type, head_dim, n_head_kv));
    if (n_head < 1 || n_head > 65535 || n_head % n_head_kv) return set_error(FL_EINVAL, "%s: %d query heads over %d key heads", fn, n_head, n_head_kv);
    if (!(scale > 0) || !std::isfinite(scale * 1.44269504088896341f)) return set_error(FL_EINVAL, "%s: scale %g is not a positive number", fn, (double)scale);
    if (n_seq < 0) return set_error(FL_EINVAL, "%s: %d sequences", fn, n_seq);
    if ((int64_t)n_q * n_head > MAX_COUNT) return set_error(FL_EINVAL, "%s: %d rows of %d heads: more than 2^31 - 512", fn, n_q, n_head);
    FL_TRY(check_heads(fn, "q", q, type, n_q));
    FL_TRY(check_out(fn, "out", out, type, n_q, n_head));
    a.q = q->data_dev, a.q_ld = q->token_stride, a.q_hs = q->head_stride;
    a.out = out->data_dev, a.o_ld = out->token_stride, a.o_hs = out->head_stride;
    a.n_q = n_q, a.n_seq = n_seq, a.n_head = n_head, a.group = n_head / n_head_kv, a.head_dim = head_dim;
    a.scale_log2 = scale * 1.44269504088896341f;
    return FL_OK;
}

static int check_workspace(const char *fn, const char *query, size_t need, const void *ws, size_t bytes) {
    if (need && (!ws || bytes < need || !aligned(ws, 16)))
        return set_error(FL_EINVAL, "%s: a workspace of %zu bytes, aligned to 16 (want %zu: %s)", fn, ws ? bytes : 0, need, query);
    return FL_OK;
}

size_t fl_attn_prompt_workspace(int type, int head_dim, int n_head, int n_head_kv, int n_q, int n_kv, int n_seq) {
    if (!size_of(type) || head_dim < 1 || n_head_kv < 1 || n_head < n_head_kv || n_q < 1 || n_kv < 1 || n_seq < 1) return 0;
    return attn_prompt_workspace(type, n_q, n_seq, n_head, n_head_kv, head_dim, n_kv);
}

int fl_attn_prompt(int type, int head_dim, int n_head, int n_head_kv, float scale, const fl_heads *q, int n_q, const fl_heads *k, const fl_heads *v, int n_kv,
                   const int32_t *cu_q_dev, const int32_t *cu_kv_dev, int n_seq, const fl_heads *out, void *workspace_dev, size_t workspace_bytes, void *stream) {
    const char *fn = "fl_attn_prompt";
    AttnArgs a{};
    FL_TRY(fill(a, fn, type, head_dim, n_head, n_head_kv, scale, q, out, n_q, n_seq));
    FL_TRY(check_heads(fn, "k", k, type, n_kv));
    FL_TRY(check_heads(fn, "v", v, type, n_kv));
    if (n_kv > MAX_COUNT) return set_error(FL_EINVAL, "%s: %d keys: more than 2^31 - 512", fn, n_kv);
    if (n_q == 0 || n_seq == 0) return FL_OK;
    if (!cu_q_dev || !cu_kv_dev) return set_error(FL_EINVAL, "%s: null row starts", fn);
    FL_TRY(check_workspace(fn, "fl_attn_prompt_workspace", fl_attn_prompt_workspace(type, head_dim, n_head, n_head_kv, n_q, n_kv, n_seq), workspace_dev, workspace_bytes));
    a.ws = workspace_dev;
    FL_TRY(ensure_device());
    a.k = k->data_dev, a.v = v->data_dev, a.k_ld = k->token_stride, a.k_hs = k->head_stride, a.v_ld = v->token_stride, a.v_hs = v->head_stride;
    a.cu_q = cu_q_dev, a.cu_kv = cu_kv_dev, a.n_kv = n_kv;
    const hipError_t e = attn_prompt(a, type, false, S(stream));
    return e == hipSuccess ? FL_OK : hip_fail(e, fn);
}

size_t fl_attn_pages_workspace(const fl_kv_pages *c, int n_head, int n_q, int n_table, int n_seq, int one_row) {
    if (!c || !size_of(c->type) || c->head_dim < 1 || c->n_head_kv < 1 || n_head < c->n_head_kv || n_q < 1 || n_table < 1 || n_seq < 1 || c->page_size < 1) return 0;
    if (!one_row) return attn_prompt_workspace(c->type, n_q, n_seq, n_head, c->n_head_kv, c->head_dim, (int64_t)n_table * c->page_size);
    return attn_decode_workspace(c->type, n_seq, n_head, c->n_head_kv, c->head_dim, (int64_t)n_table * c->page_size);
}

int fl_attn_pages(const fl_kv_pages *c, int n_head, float scale, const fl_heads *q, int n_q, const int32_t *cu_q_dev, const int32_t *kv_len_dev,
                  const int32_t *table_dev, int table_ld, int n_table, int n_seq, const fl_heads *out, void *workspace_dev, size_t workspace_bytes, void *stream) {
    const char *fn = "fl_attn_pages";
    FL_TRY(check_pages(fn, c));
    AttnArgs a{};
    FL_TRY(fill(a, fn, c->type, c->head_dim, n_head, c->n_head_kv, scale, q, out, n_q, n_seq));
    if (n_q == 0 || n_seq == 0) return FL_OK;
    FL_TRY(check_table(fn, c, table_dev, table_ld, n_table, n_seq));
    if (!kv_len_dev || (!cu_q_dev && n_seq != n_q)) return set_error(FL_EINVAL, "%s: no lengths, or no row starts for %d rows of %d sequences", fn, n_q, n_seq);
    a.k = c->k_dev, a.v = c->v_dev, a.k_ld = a.v_ld = c->slot_stride, a.k_hs = a.v_hs = c->head_stride, a.page_stride = c->page_stride;
    a.cu_q = cu_q_dev, a.kv_len = kv_len_dev, a.table = table_dev, a.table_ld = table_ld, a.n_table = n_table, a.page_shift = page_shift(c), a.n_pages = c->n_pages;
    FL_TRY(check_workspace(fn, "fl_attn_pages_workspace", fl_attn_pages_workspace(c, n_head, n_q, n_table, n_seq, !cu_q_dev), workspace_dev, workspace_bytes));
    a.ws = workspace_dev;
    FL_TRY(ensure_device());
    const hipError_t e = cu_q_dev ? attn_prompt(a, c->type, true, S(stream)) : attn_decode(a, c->type, S(stream));
    return e == hipSuccess ? FL_OK : hip_fail(e, fn);
}

size_t fl_sample_workspace(int rows, int n_vocab) { return rows < 1 || n_vocab < 1 || n_vocab > FL_SAMPLE_MAX_VOCAB ? 0 : sample_workspace(rows, n_vocab); }

int fl_sample(int type, const void *logits_dev, int64_t ld, int rows, int n_vocab, const float *u_dev, const fl_sample_params *p, int32_t *tokens_dev,
              void *workspace_dev, size_t workspace_bytes, void *stream) {
    const char *fn = "fl_sample";
    if (!size_of(type)) return set_error(FL_EINVAL, "%s: type %d is not f32 (0), f16 (1) or bf16 (%d)", fn, type, FL_TYPE_BF16);
    if (rows < 0 || n_vocab < 1 || n_vocab > FL_SAMPLE_MAX_VOCAB || ld < 0 || (rows > 1 && ld < n_vocab))
        return set_error(FL_EINVAL, "%s: %d rows of %d logits (1..%d), row stride %lld", fn, rows, n_vocab, FL_SAMPLE_MAX_VOCAB, (long long)ld);
    if (rows == 0) return FL_OK;
    if (!logits_dev || !u_dev || !p || !tokens_dev) return set_error(FL_EINVAL, "%s: null argument", fn);
    if (!aligned(logits_dev, (size_t)size_of(type))) return set_error(FL_EINVAL, "%s: logits not aligned to their type", fn);
    FL_TRY(check_workspace(fn, "fl_sample_workspace", sample_workspace(rows, n_vocab), workspace_dev, workspace_bytes));
    FL_TRY(ensure_device());
    SampleArgs a{};
    a.logits = logits_dev, a.ld = ld, a.rows = rows, a.n_vocab = n_vocab, a.u = u_dev, a.tokens = tokens_dev, a.ws = workspace_dev;
    a.temperature_p = p->temperature_dev, a.top_k_p = p->top_k_dev, a.top_p_p = p->top_p_dev, a.min_p_p = p->min_p_dev;
    a.temperature = p->temperature, a.top_k = p->top_k, a.top_p = p->top_p, a.min_p = p->min_p;
    const hipError_t e = sample(a, type, S(stream));
    return e == hipSuccess ? FL_OK : hip_fail(e, fn);
}

}  // extern "C"
