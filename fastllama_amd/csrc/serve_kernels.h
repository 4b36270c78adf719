// serve_kernels.h -- operators over several sequences: a paged K/V cache, the attention that reads it, attention over packed prompts and
// sampling.  Argument blocks and launchers; the entry points that check and fill them are in serve_api.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace fl {

// Keys and values of the attention operators: either packed rows (element (row, head, d) at row * ld + head * hs + d, sequence b owns rows
// cu[b] .. cu[b+1] - 1) or pages (position p of sequence b in slot p % page_size of page table[b][p / page_size]).  All strides in elements.
struct AttnArgs {
    const void *q;
    int64_t q_ld, q_hs;
    void *out;
    int64_t o_ld, o_hs;
    const void *k, *v;
    int64_t k_ld, k_hs, v_ld, v_hs;      // packed: row and head strides; pages: slot and head strides (K and V alike)
    int64_t page_stride;
    const int32_t *cu_q, *cu_kv, *kv_len, *table;
    int table_ld, n_table, page_shift, n_pages;
    int n_q, n_kv, n_seq, n_head, group, head_dim;   // group: query heads per key head
    float scale_log2;                    // scale * log2(e): the softmax runs on powers of two
    void *ws;
};

struct AppendArgs {
    void *kc, *vc;
    int64_t page_stride, head_stride, slot_stride;
    const void *k, *v;
    int64_t k_ld, k_hs, v_ld, v_hs;
    const int32_t *cu, *n_past, *table;
    int table_ld, n_table, page_shift, n_pages, n_tok, n_seq, n_head_kv, head_dim;
};

struct SampleArgs {
    const void *logits;
    int64_t ld;
    int rows, n_vocab;
    const float *u, *temperature_p, *top_p_p, *min_p_p;   // *_p: one value for each row, or NULL: the scalar for all
    const int32_t *top_k_p;
    float temperature, top_p, min_p;
    int top_k;
    int32_t *tokens;
    void *ws;
};

hipError_t attn_prompt(const AttnArgs &a, int type, bool paged, hipStream_t st);
size_t attn_prompt_workspace(int type, int n_q, int n_seq, int n_head, int n_head_kv, int head_dim, int64_t max_keys);
hipError_t attn_decode(const AttnArgs &a, int type, hipStream_t st);
size_t attn_decode_workspace(int type, int n_seq, int n_head, int n_head_kv, int head_dim, int64_t max_len);
hipError_t kv_append(const AppendArgs &a, int src_type, int type, hipStream_t st);
hipError_t sample(const SampleArgs &a, int type, hipStream_t st);
size_t sample_workspace(int rows, int n_vocab);

}  // namespace fl
