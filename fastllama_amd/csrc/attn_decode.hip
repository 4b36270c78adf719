// attn_decode.hip -- attention of one new token for each sequence over a paged cache.
//
//   out[i][h] = sum_j exp(s_ij - max) v_j / sum_j exp(s_ij - max),  s_ij = scale q_i . k_j,  keys j <= lk - lq + i of i's own sequence
//
// First form: one wave for a row and head, a lane for a key; the maximum and sum run along (one pass over K and V).
#include "serve_kernels.h"
#include "serve_device.h"
#include "../../include/fastllama_hip.h"

namespace fl {

template <typename T, bool PAGED>
__global__ __launch_bounds__(256) void attn_rows_k(AttnArgs a, bool decode) {
    const int lane = threadIdx.x & 63, head = blockIdx.y, row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.n_q) return;
    int b = -1, q0 = 0, q1 = 0;
    if (decode) b = row, q0 = row, q1 = row + 1;
    else
        for (int s = 0; s < a.n_seq; ++s) {
            seq_rows(a.cu_q, s, a.n_q, &q0, &q1);
            if (row >= q0 && row < q1) { b = s; break; }
        }
    if (b < 0) return;
    int k0 = 0, lk;
    if (PAGED) lk = (int)min((int64_t)max(a.kv_len[b], 0), (int64_t)a.n_table << a.page_shift);
    else {
        int k1;
        seq_rows(a.cu_kv, b, a.n_kv, &k0, &k1);
        lk = k1 - k0;
    }
    const int seen = min(lk, lk - (q1 - q0) + (row - q0) + 1);
    const int D = a.head_dim, hk = head / a.group;
    const T *q = (const T *)a.q + row * a.q_ld + head * a.q_hs;
    float m = -INFINITY, l = 0, o0 = 0, o1 = 0;
    for (int j0 = 0; j0 < seen; j0 += 64) {
        const int j = j0 + lane;
        int64_t ko = 0, vo = 0;
        bool in = j < seen;
        if (PAGED) {
            const int pg = in ? a.table[(int64_t)b * a.table_ld + (j >> a.page_shift)] : -1;
            in = in && pg >= 0 && pg < a.n_pages;
            ko = vo = (in ? pg : 0) * a.page_stride + (j & ((1 << a.page_shift) - 1)) * a.k_ld;
        } else ko = (in ? k0 + j : 0) * a.k_ld, vo = (in ? k0 + j : 0) * a.v_ld;
        float s = -INFINITY;
        if (in) {
            const T *k = (const T *)a.k + ko + hk * a.k_hs;
            s = 0;
            for (int d = 0; d < D; ++d) s = fmaf((float)q[d], (float)k[d], s);
            s *= a.scale_log2;
        }
        float mx = s;
        for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        const float c = exp2f(m - ref), p = exp2f(s - ref);
        float ps = p;
        for (int o = 32; o; o >>= 1) ps += __shfl_xor(ps, o);
        l = l * c + ps, o0 *= c, o1 *= c, m = mn;
        const unsigned long long live = __ballot(in);
        for (int t = 0; t < 64; ++t) {
            if (!(live >> t & 1)) continue;
            const float pt = __shfl(p, t);
            const T *v = (const T *)a.v + __shfl(vo, t) + hk * a.v_hs;
            if (lane < D) o0 = fmaf(pt, (float)v[lane], o0);
            if (lane + 64 < D) o1 = fmaf(pt, (float)v[lane + 64], o1);
        }
    }
    T *o = (T *)a.out + row * a.o_ld + head * a.o_hs;
    const float r = l > 0 || l != l ? 1 / l : 0.f;
    if (lane < D) o[lane] = (T)(o0 * r);
    if (lane + 64 < D) o[lane + 64] = (T)(o1 * r);
}

hipError_t attn_decode(const AttnArgs &a, int type, hipStream_t st) {
    const dim3 g((a.n_q + 3) / 4, a.n_head);
    switch (type) {
        case FL_TYPE_F32: attn_rows_k<float, true><<<g, 256, 0, st>>>(a, true); break;
        case FL_TYPE_F16: attn_rows_k<h16, true><<<g, 256, 0, st>>>(a, true); break;
        default: attn_rows_k<b16, true><<<g, 256, 0, st>>>(a, true); break;
    }
    return hipGetLastError();
}
size_t attn_decode_workspace(int, int, int, int, int64_t) { return 0; }

}  // namespace fl
