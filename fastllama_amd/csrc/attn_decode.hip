// attn_decode.hip -- attention of one new token for each sequence over a paged cache.
//
//   out[b][h] = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max),  s_j = scale q . k_j,  j < kv_len[b]
//
// Bound by reading K and V once.  The query heads of a key head (16 at most at a time) are the columns of one small problem on the matrix units;
// with one query head 15 of 16 columns are idle, which costs nothing that is missed: the reads still take longer.  Both products are taken
// transposed (attn_prompt.hip): S^T = K Q^T, O^T = V^T P^T, so K goes from memory straight into its operand's registers, P stays where S was
// made, and V alone passes through LDS, each wave by itself: there is no barrier before the end.  A wave has the next tile's K and V in flight
// while it works on this one.
//
// A sequence's keys are cut into chunks; a workgroup's four waves take every fourth tile of a chunk and join their maxima, sums and outputs in LDS.
// A sequence of one chunk is done then; the chunks of a longer one leave theirs in the workspace for a second launch to join.  Chunks are
// of one length, so the work of a ragged batch is even, and workgroups behind a sequence's end leave at once.
#include "serve_kernels.h"
#include "serve_device.h"
#include "../../include/fastllama_hip.h"

namespace fl {

// Keys of a chunk.  The host knows the page table's width, not the lengths.  512 keep a workgroup's life short (a wave has four tiles of f16) beside
// what starting and joining it costs: 16 sequences of 2048, 32 heads of 128 in f16 take 117 us at 128, 106 at 256, 105 at 512, 103 at 1024; 64 of 1 to
// 4096, 8 key heads, 48, 39, 35, 38.  Few sequences are cut finer until each CU could have two workgroups, down to a tile a wave: one of 300, 32 heads
// in f32, takes 14.3 us at 512 and 9.7 at 64.  Many long ones are cut coarser to bound the workspace.
constexpr int DEC_WAVES = 4;
static int decode_chunk(int64_t blocks, int64_t max_len, int least) {
    int64_t chunk = 512;
    if (max_len <= 2 * least) return 512;              // (two tiles a wave: 7.3 us for 256 keys in f16, 8.9 cut in two and joined)
    while (chunk > least && blocks * ((max_len + chunk - 1) / chunk) < 512) chunk /= 2;
    while (blocks * ((max_len + chunk - 1) / chunk) > 16384 && chunk < max_len) chunk *= 2;
    return (int)chunk;
}
static int least_chunk(int type) { return type == FL_TYPE_F32 ? 16 * DEC_WAVES : 32 * DEC_WAVES; }
static int64_t decode_blocks(int n_seq, int n_head, int n_head_kv) { return (int64_t)n_seq * n_head_kv * ((n_head / n_head_kv + 15) / 16); }

// The workspace: for each (sequence, head, chunk) its output's D sums, then its maximum and sum.
size_t attn_decode_workspace(int type, int n_seq, int n_head, int n_head_kv, int head_dim, int64_t max_len) {
    const int chunk = decode_chunk(decode_blocks(n_seq, n_head, n_head_kv), max_len, least_chunk(type));
    const int64_t splits = (max_len + chunk - 1) / chunk;
    return splits > 1 ? (size_t)n_seq * n_head * splits * (head_dim + 2) * 4 : 0;
}

__device__ inline int decode_len(const AttnArgs &a, int b) { return min(max(a.kv_len[b], 0), a.n_table << a.page_shift); }

template <typename T, int DP>
__global__ __launch_bounds__(64 * DEC_WAVES, 2) void attn_decode_k(AttnArgs a, int chunk, int splits, int q_blocks) {
    constexpr int KB = sizeof(T) == 2 ? 2 : 1, KT = 16 * KB, UNIT = 16 / sizeof(T), DS = DP / 32, DB = DP / 16;   // KB blocks of 16 keys make a tile
    constexpr int CPR = DP / UNIT, RPP = 64 / CPR, PASSES = KT / RPP, VLD = DP + (sizeof(T) == 2 ? 16 : 4);
    typedef typename Vec<T>::x8 x8;
    typedef T xp __attribute__((ext_vector_type(4 * KB)));             // a lane's part of P and V^T
    __shared__ __attribute__((aligned(16))) T vs[DEC_WAVES][KT * VLD];
    __shared__ float ms[DEC_WAVES][16], ls[DEC_WAVES][16];
    static_assert(RPP <= 16 && 16 % RPP == 0, "a pass of V stays inside a block of 16 keys");
    static_assert(KT * VLD * sizeof(T) >= 16 * DP * 4, "a wave's outputs fit where its V was");

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int n_head_kv = a.n_head / a.group;
    int x = blockIdx.x;
    const int qb = x % q_blocks;
    x /= q_blocks;
    const int hk = x % n_head_kv;
    x /= n_head_kv;
    const int b = x % a.n_seq, split = x / a.n_seq;
    const int len = decode_len(a, b), c0 = split * chunk, c1 = min(c0 + chunk, len);
    if (c0 >= len && split) return;
    const int D = a.head_dim, heads = min(16, a.group - 16 * qb), head0 = hk * a.group + 16 * qb;

    x8 qf[DS];
    {
        const T *q = (const T *)a.q + b * a.q_ld + (head0 + (n < heads ? n : 0)) * a.q_hs;
#pragma unroll
        for (int s = 0; s < DS; ++s) {
            const int d = 32 * s + 8 * g;
            qf[s] = n < heads && d < D ? *(const x8 *)(q + d) : (x8)(T)0;
        }
    }
    const int tiles = (c1 - c0 + KT - 1) / KT;                         // this wave: tiles wave, wave + 4, ...
    const int32_t *table = a.table + (int64_t)b * a.table_ld;
    const int smask = (1 << a.page_shift) - 1;
    const int vc = (lane % CPR) * UNIT, vrow = lane / CPR;
    const T *kbase = (const T *)a.k + hk * a.k_hs, *vbase = (const T *)a.v + hk * a.v_hs + vc;

    // Page numbers of the wave's next 64 blocks of 16 keys, one a lane; -1: no page there.
    int pages = 0, batch = -1;
    auto page_of = [&](int i, int kb) {                                // block kb of the wave's i-th tile
        const int at = i * KB + kb;
        if (at >> 6 != batch) {
            batch = at >> 6;
            const int e = batch * 64 + lane, j = c0 + ((e / KB) * DEC_WAVES + wave) * KT + (e % KB) * 16;
            const int p = j < c1 ? table[j >> a.page_shift] : -1;
            pages = p >= 0 && p < a.n_pages ? p : -1;
        }
        return __builtin_amdgcn_readlane(pages, at & 63);
    };
    x8 kr[KB][DS];
    u32x4 vr[PASSES];
    uint32_t there = 0, there_next = 0;
    auto load_k = [&](int i) {
        const int kv = c0 + (i * DEC_WAVES + wave) * KT;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int p = page_of(i, kb), j = kv + 16 * kb + n;
            const T *k = kbase + p * a.page_stride + (j & smask) * a.k_ld;
            const bool in = p >= 0 && j < c1;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                const int d = 32 * s + 8 * g;
                kr[kb][s] = (x8)(T)0;
                if (in && d < D) kr[kb][s] = *(const x8 *)(k + d);
            }
        }
    };
    auto load_v = [&](int i) {
        const int kv = c0 + (i * DEC_WAVES + wave) * KT;
        int p[KB];
        there_next = 0;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) p[kb] = page_of(i, kb), there_next |= (p[kb] >= 0) << kb;
#pragma unroll
        for (int s = 0; s < PASSES; ++s) {
            const int r = vrow + RPP * s, j = kv + r;
            const int pg = p[(RPP * s) >> 4];                          // (a pass stays inside a block of 16)
            vr[s] = (u32x4)0u;
            if (pg >= 0 && j < c1 && vc < D) vr[s] = *(const u32x4 *)(vbase + pg * a.page_stride + (j & smask) * a.v_ld);
        }
    };

    f32x4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = (f32x4)0.f;
    float m = -INFINITY, l = 0;                                        // of column n; l: this lane's keys
    T *v = vs[wave];
    if (wave < tiles) load_k(0), load_v(0);
    for (int i = 0; i * DEC_WAVES + wave < tiles; ++i) {
        const int kv = c0 + (i * DEC_WAVES + wave) * KT;
        const bool more = (i + 1) * DEC_WAVES + wave < tiles;
        there = there_next;
        f32x4 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            s[kb] = (f32x4)0.f;
#pragma unroll
            for (int st = 0; st < DS; ++st) s[kb] = mfma16(kr[kb][st], qf[st], s[kb]);
        }
        if (more) load_k(i + 1);
#pragma unroll
        for (int p = 0; p < PASSES; ++p) *(u32x4 *)(v + (vrow + RPP * p) * VLD + vc) = vr[p];
        if (more) load_v(i + 1);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (kv + KT > c1 || there != (1u << KB) - 1)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[kb][r] = kv + 16 * kb + 4 * g + r < c1 && (there >> kb & 1) ? s[kb][r] : -INFINITY;
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[kb][r]);
        mx *= a.scale_log2;
        if (__any(mx > m + 8.f)) {                                     // (the reference may lag the maximum by 2^8: attn_prompt.hip)
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn, l *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= f;
        }
        const float ref = (m == -INFINITY ? 0.f : m) - P_SHIFT<T>;
        xp p;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[kb][r], a.scale_log2, -ref));
                l += e;
                p[4 * kb + r] = (T)e;                                  // (rounded for the second product, as in attn_prompt.hip)
            }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            xp vt;                                                     // keys 4 g + 0..3 of each block at component 16 d + n
            if constexpr (sizeof(T) == 2) {
                const T *at = v + (4 * g + (n >> 2)) * VLD + 16 * d + 4 * (n & 3);
                typedef short s16x8 __attribute__((ext_vector_type(8)));
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 16 * VLD));
                vt = __builtin_bit_cast(xp, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) vt[r] = v[(4 * g + r) * VLD + 16 * d + n];
            }
            o[d] = mfma16(vt, p, o[d]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // the four waves' parts
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) ms[wave][n] = m, ls[wave][n] = l;
    __syncthreads();
    float M = ms[0][n];
    for (int w = 1; w < DEC_WAVES; ++w) M = fmaxf(M, ms[w][n]);
    const float f = factor(m, M);
    float *mine = (float *)vs[wave];
#pragma unroll
    for (int d = 0; d < DB; ++d)
        if (n < heads) *(f32x4 *)(mine + n * DP + 16 * d + 4 * g) = o[d] * f;
    __syncthreads();
    for (int e = threadIdx.x; e < heads * DP; e += 64 * DEC_WAVES) {
        const int q = e / DP, d = e % DP;
        if (d >= D) continue;
        float mq = ms[0][q], lq = 0, sum = 0;
        for (int w = 1; w < DEC_WAVES; ++w) mq = fmaxf(mq, ms[w][q]);
        for (int w = 0; w < DEC_WAVES; ++w) {
            lq += ls[w][q] * factor(ms[w][q], mq);
            sum += ((const float *)vs[w])[e];
        }
        const int head = head0 + q;
        if (len <= chunk) {
            ((T *)a.out)[b * a.o_ld + head * a.o_hs + d] = (T)(lq == 0 ? 0.f : sum / lq);
        } else {
            float *to = (float *)a.ws + (((int64_t)b * a.n_head + head) * splits + split) * (D + 2);
            to[d] = sum;
            if (d == 0) to[D] = mq, to[D + 1] = lq;
        }
    }
}

// The chunks of the sequences that have several: a workgroup for each (sequence, head), GROUPS groups of 128 threads (one for each component) that
// take every GROUPS-th chunk.
template <typename T, int GROUPS>
__global__ __launch_bounds__(128 * GROUPS) void attn_join_k(AttnArgs a, int chunk, int splits) {
    const int head = blockIdx.x % a.n_head, b = blockIdx.x / a.n_head, D = a.head_dim, d = threadIdx.x & 127, g = threadIdx.x >> 7;
    const int len = decode_len(a, b);
    if (len <= chunk) return;
    const int n = (len + chunk - 1) / chunk;
    const float *part = (const float *)a.ws + ((int64_t)b * a.n_head + head) * splits * (D + 2);
    __shared__ float red[2 * GROUPS], acc[GROUPS][128], den[GROUPS];
    float M = -INFINITY;
    for (int s = threadIdx.x; s < n; s += 128 * GROUPS) M = fmaxf(M, part[(int64_t)s * (D + 2) + D]);
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = M;
    __syncthreads();
    for (int w = 0; w < 2 * GROUPS; ++w) M = fmaxf(M, red[w]);
    float sum = 0, l = 0;
    const int dd = min(d, D - 1);
#pragma unroll 4
    for (int s = g; s < n; s += GROUPS) {
        const float *p = part + (int64_t)s * (D + 2);
        const float x = p[dd], m = p[D], ls = p[D + 1];
        const float f = factor(m, M);
        l += ls * f, sum += x * f;
    }
    acc[g][d] = sum;
    if (d == 0) den[g] = l;
    __syncthreads();
    if (g == 0 && d < D) {
        for (int i = 1; i < GROUPS; ++i) l += den[i], sum += acc[i][d];
        ((T *)a.out)[b * a.o_ld + head * a.o_hs + d] = (T)(l == 0 ? 0.f : sum / l);
    }
}

template <typename T>
static hipError_t decode_launch(const AttnArgs &a, hipStream_t st) {
    const int n_head_kv = a.n_head / a.group, q_blocks = (a.group + 15) / 16;
    const int64_t max_len = (int64_t)a.n_table << a.page_shift, blocks = decode_blocks(a.n_seq, a.n_head, n_head_kv);
    const int chunk = decode_chunk(blocks, max_len, sizeof(T) == 4 ? 16 * DEC_WAVES : 32 * DEC_WAVES), splits = (int)((max_len + chunk - 1) / chunk);
    if (blocks * splits * 64 * DEC_WAVES > UINT32_MAX) return hipErrorInvalidValue;
    const dim3 g((unsigned)(blocks * splits));
    if (a.head_dim <= 32) attn_decode_k<T, 32><<<g, 64 * DEC_WAVES, 0, st>>>(a, chunk, splits, q_blocks);
    else if (a.head_dim <= 64) attn_decode_k<T, 64><<<g, 64 * DEC_WAVES, 0, st>>>(a, chunk, splits, q_blocks);
    else attn_decode_k<T, 128><<<g, 64 * DEC_WAVES, 0, st>>>(a, chunk, splits, q_blocks);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && splits > 1) {
        const dim3 j((unsigned)(a.n_seq * a.n_head));
        if (splits <= 8) attn_join_k<T, 2><<<j, 256, 0, st>>>(a, chunk, splits);
        else attn_join_k<T, 8><<<j, 1024, 0, st>>>(a, chunk, splits);
        e = hipGetLastError();
    }
    return e;
}

hipError_t attn_decode(const AttnArgs &a, int type, hipStream_t st) {
    switch (type) {
        case FL_TYPE_F32: return decode_launch<float>(a, st);
        case FL_TYPE_F16: return decode_launch<h16>(a, st);
        default: return decode_launch<b16>(a, st);
    }
}

}  // namespace fl
