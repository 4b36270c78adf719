// kv_append.hip -- rows of new keys and values into the pages of a cache.
//
// Row j of sequence b goes to position n_past[b] + j: slot position % page_size of page table[b][position / page_size].  A copy with at most one
// rounding (f32 -> f16 / bf16, to nearest even): bound by HBM, and for single tokens by the launch.
#include "serve_kernels.h"
#include "serve_device.h"
#include "../../include/fastllama_hip.h"

namespace fl {

// A thread moves 8 elements (one 16-byte store of a 16-bit cache); the 256 threads of a workgroup take consecutive (row, head, chunk).
template <typename S, typename T>
__global__ __launch_bounds__(256) void kv_append_k(AppendArgs a) {
    typedef S vs __attribute__((ext_vector_type(8)));
    typedef T vt __attribute__((ext_vector_type(8)));
    const int chunks = a.head_dim >> 3, per_row = chunks * a.n_head_kv;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(i / per_row), rest = (int)(i - (int64_t)row * per_row);
    if (row >= a.n_tok) return;
    int b = row, first = row;
    if (a.cu) {                          // the last sequence that starts at or before the row, by halving
        int lo = 0, hi = a.n_seq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu[mid] <= row) lo = mid;
            else hi = mid;
        }
        int end;
        b = lo;
        seq_rows(a.cu, b, a.n_tok, &first, &end);
        if (row < first || row >= end) return;
    }
    const int64_t pos = (int64_t)a.n_past[b] + (row - first);
    if (pos < 0 || (pos >> a.page_shift) >= a.n_table) return;
    const int page = a.table[(int64_t)b * a.table_ld + (pos >> a.page_shift)];
    if (page < 0 || page >= a.n_pages) return;
    const int h = rest / chunks, d = (rest - h * chunks) * 8;
    const int64_t to = page * a.page_stride + h * a.head_stride + (pos & ((1 << a.page_shift) - 1)) * a.slot_stride + d;
    const vs k = *(const vs *)((const S *)a.k + row * a.k_ld + h * a.k_hs + d), v = *(const vs *)((const S *)a.v + row * a.v_ld + h * a.v_hs + d);
    *(vt *)((T *)a.kc + to) = __builtin_convertvector(k, vt);
    *(vt *)((T *)a.vc + to) = __builtin_convertvector(v, vt);
}

hipError_t kv_append(const AppendArgs &a, int src_type, int type, hipStream_t st) {
    const int64_t n = (int64_t)a.n_tok * a.n_head_kv * (a.head_dim >> 3);
    const dim3 g((unsigned)((n + 255) / 256));
    if (type == FL_TYPE_F32) kv_append_k<float, float><<<g, 256, 0, st>>>(a);
    else if (type == FL_TYPE_F16 && src_type == FL_TYPE_F32) kv_append_k<float, h16><<<g, 256, 0, st>>>(a);
    else if (type == FL_TYPE_F16) kv_append_k<h16, h16><<<g, 256, 0, st>>>(a);
    else if (src_type == FL_TYPE_F32) kv_append_k<float, b16><<<g, 256, 0, st>>>(a);
    else kv_append_k<b16, b16><<<g, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace fl
