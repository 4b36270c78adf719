// attn_prompt.hip -- causal attention with grouped heads over packed prompts or a paged cache.
//
//   out[i][h] = sum_j exp(s_ij - max) v_j / sum_j exp(s_ij - max),  s_ij = scale q_i . k_j,  keys j <= lk - lq + i of i's own sequence
//
// The query heads that share a key head are rows of one problem: row r of (sequence, key head) is token r / group, head r % group, so a
// workgroup's rows read each key and value once for the whole group, and few tokens still fill a tile.  A wave has 32 rows; K and V pass
// through LDS in tiles of KT keys, the next tile's loads in flight (registers) while this one is computed, two LDS tiles in turn: one barrier a tile.
//
// Both products are taken transposed: S^T = K Q^T leaves each lane a column, one query row with half of the tile's keys (lane and lane + 32
// share the row), so maximum and sum run inside a lane; and its registers are, in their order, the operand P^T of O^T = V^T P^T, whose
// columns are query rows again: the rescaling factor is a lane's own.  V^T comes out of LDS by transposing reads.
//
// The softmax's reference is not the running maximum but a value at most 2^8 below it: the accumulators are rescaled only when the maximum
// has moved by more.  p is rounded to the inputs' type for the second product, which the 16-bit matrix units ask for (the error of a weighted mean of
// values that are themselves of that type: against 64 bits 0.0017 of the outputs' size in place of the 0.0016 of the last rounding alone in bf16, 0.00018
// in place of 0.00017 in f16); scores, sums and outputs are f32 until the one rounding at the end.  f16 has p only down to 2^-24, so there it is
// taken 2^P_SHIFT times as large, which cancels against the sum: p <= 2^15 still fits, and what is lost of a key is at most 2^-32 of the largest weight.
#include "serve_kernels.h"
#include "serve_device.h"
#include "../../include/fastllama_hip.h"

namespace fl {

template <typename T>
struct Tile {                            // LDS tiles of a type
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32, KPAD = 16 / sizeof(T), VPAD = sizeof(T) == 2 ? 32 : 4;
};

// Four keys 4 * (lane / 32) + 0..3 and four more 8 behind them, of the 16 that start at `row`, at component d0 + lane % 32: the transposed operand.
template <typename T, int LD>
__device__ inline typename Vec<T>::x8 read_vt(const T *v, int row, int d0, int lane) {
    typename Vec<T>::x8 r;
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        // each group of 16 lanes reads 4 keys x 16 components, 4 components a lane, and gets them transposed
        const int L = lane & 15;
        const T *p = v + (row + 4 * h + (L >> 2)) * LD + d0 + ((lane >> 4) & 1) * 16 + 4 * (L & 3);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 8 * LD));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        r = __builtin_bit_cast(typename Vec<T>::x8, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        const T *p = v + (row + 4 * h) * LD + d0 + (lane & 31);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = p[(i < 4 ? i : i + 4) * LD];
    }
    return r;
}

// A workgroup's block of rows: sequence b has rows q0 .. q0 + lq - 1 and lk keys (packed ones from k0 on); the block is its number blk.  All values are
// the same in all threads.  b = -1: there is none.
struct Block {
    int b, q0, lq, k0, lk, blk;
};
template <bool PAGED, int ROWS>
__device__ Block find_block(const AttnArgs &a, int blk, int blocks) {
    const int lane = threadIdx.x & 63;
    int b = -1, q0 = 0, lq = 0;
    auto blocks_of = [&](int s, int *f, int *e) {                      // sequence s's first row and end; returns its blocks
        *f = *e = 0;
        if (s < a.n_seq) seq_rows(a.cu_q, s, a.n_q, f, e);
        return (int)(((int64_t)(*e - *f) * a.group + ROWS - 1) / ROWS);
    };
    if (a.n_seq <= 64) {
        // The longest ways first, or the last to start ends long behind the others: a block's number in its sequence is (but for keys of the past) its
        // number of tiles, so the blocks go by that number, falling, through all sequences that have one of it.
        int f, e;
        const int n = blocks_of(lane, &f, &e);
        auto most = [](int x) {
            for (int o = 32; o; o >>= 1) x = max(x, __shfl_xor(x, o));
            return __builtin_amdgcn_readfirstlane(x);
        };
        const int max1 = most(n), first = max1 ? __builtin_ctzll(__ballot(n == max1)) : 0, max2 = most(lane == first ? 0 : n);
        int level = max1 - 1 - blk;                                    // (alone above the second longest)
        if (level >= max2) blk = 0;
        else {
            blk -= max1 - max2, level = max2 - 1;
            for (; level >= 0; --level) {
                const int c = __popcll(__ballot(n > level));
                if (blk < c) break;
                blk -= c;
            }
        }
        if (level < 0) return Block{-1, 0, 0, 0, 0, 0};
        const unsigned long long has = __ballot(n > level);
        const int w = __builtin_ctzll(__ballot(n > level && __popcll(has & ((1ull << lane) - 1)) == blk));
        b = w, q0 = __builtin_amdgcn_readlane(f, w), lq = __builtin_amdgcn_readlane(e, w) - q0, blk = level;
    } else {
        blk = blocks - 1 - blk;
        for (int s0 = 0; s0 < a.n_seq; s0 += 64) {                     // 64 sequences at a time
            int f, e;
            const int n = blocks_of(s0 + lane, &f, &e);
            int incl = n;
            for (int o = 1; o < 64; o <<= 1) {
                const int up = __shfl_up(incl, o);
                if (lane >= o) incl += up;
            }
            const int total = __builtin_amdgcn_readlane(incl, 63);
            if (blk < total) {
                const int w = __builtin_ctzll(__ballot(incl > blk));
                b = s0 + w, q0 = __builtin_amdgcn_readlane(f, w), lq = __builtin_amdgcn_readlane(e, w) - q0, blk -= __builtin_amdgcn_readlane(incl - n, w);
                break;
            }
            blk -= total;
        }
    }
    if (b < 0) return Block{-1, 0, 0, 0, 0, 0};
    int k0 = 0, lk;
    if (PAGED) lk = (int)min(max(a.kv_len[b], 0), a.n_table << a.page_shift);
    else {
        int k1;
        seq_rows(a.cu_kv, b, a.n_kv, &k0, &k1);
        lk = k1 - k0;
    }
    return Block{b, q0, lq, k0, lk, blk};
}

// The tiles of a block of rows whose last row sees `end` keys, cut into parts of at least four: part `part` has tiles *t0 .. *t1 - 1.  Returns the number
// of parts that have any (0 keys: 1).
template <int KT>
__device__ inline int cut_tiles(int end, int parts, int part, int *t0, int *t1) {
    const int tiles = end > 0 ? (end + KT - 1) / KT : 0, n = max(1, min(parts, tiles / 4)), per = (tiles + n - 1) / n;
    *t0 = min(part * per, tiles), *t1 = min(*t0 + per, tiles);
    return tiles ? (tiles + per - 1) / per : 1;
}

// W waves; KS of them share 32 rows, each with its part of every tile's keys, and join at the end.
template <typename T, int DP, bool PAGED, int KS, int W>
__global__ __launch_bounds__(64 * W, 2) void attn_prompt_k(AttnArgs a, int parts) {
    typedef typename Vec<T>::x8 x8;
    constexpr int KT = Tile<T>::KT, KLD = DP + Tile<T>::KPAD, VLD = DP + Tile<T>::VPAD;
    constexpr int UNIT = 16 / sizeof(T), CPR = DP / UNIT, RPP = 64 * W / CPR, PASSES = KT / RPP;   // 16-byte chunks of a row, rows of a pass over the tile
    constexpr int KB = KT / 32 / KS, DB = DP / 32, DS = DP / 16, RW = W / KS, PR_ROWS = 32 * RW;   // KB blocks of 32 keys a wave, RW waves of rows
    static_assert(KT % RPP == 0 && PASSES >= 1, "a tile is whole passes of the workgroup");
    __shared__ __attribute__((aligned(16))) T ks[2][KT * KLD], vs[2][KT * VLD];

    __shared__ int odd;
    if (threadIdx.x == 0) odd = 0;
    __syncthreads();

    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, kb0 = wave / RW * KB, n_head_kv = a.n_head / a.group;
    // Workgroups go round the 8 XCDs by their number: with 8 key heads (or a multiple) all that read a head's keys share an L2.
    const int hk = blockIdx.x % n_head_kv;
    const Block at = find_block<PAGED, PR_ROWS>(a, blockIdx.x / n_head_kv, gridDim.x / n_head_kv);
    if (at.b < 0) return;
    const int b = at.b, q0 = at.q0, lq = at.lq, k0 = at.k0, lk = at.lk, blk = at.blk;
    const int D = a.head_dim, rows = lq * a.group, r0 = blk * PR_ROWS, rw = r0 + wave % RW * 32, row = rw + (lane & 31);
    const bool valid = row < rows;
    const int tok = (valid ? row : rows - 1) / a.group, head = hk * a.group + (valid ? row : rows - 1) % a.group;
    const int past = lk - lq, lim = past + tok;                    // the last key that this lane's row sees
    const int lim_first = past + min(rw, rows - 1) / a.group, lim_last = past + min(rw + 31, rows - 1) / a.group;   // of the wave's rows
    const int end = min(past + min(r0 + PR_ROWS - 1, rows - 1) / a.group + 1, lk);
    int t0, tiles;                                                     // of this part; `tiles` ends it
    const int used = cut_tiles<KT>(end, parts, blockIdx.y, &t0, &tiles);
    if ((int)blockIdx.y >= used) return;

    x8 qf[DS];
    {
        const T *q = (const T *)a.q + (int64_t)(q0 + tok) * a.q_ld + head * a.q_hs;
#pragma unroll
        for (int s = 0; s < DS; ++s) {
            const int d = 16 * s + 8 * h;
            qf[s] = valid && d < D ? *(const x8 *)(q + d) : (x8)(T)0;
        }
    }

    // This thread's part of a tile: chunk c of rows pr + RPP * p.  Addresses are a base of the pass that the scalar unit keeps and an offset of the
    // thread that never changes.
    const int c = (t % CPR) * UNIT, pr = t / CPR;
    const char *kbase = (const char *)a.k + hk * a.k_hs * (int64_t)sizeof(T), *vbase = (const char *)a.v + hk * a.v_hs * (int64_t)sizeof(T);
    const uint32_t koff = (uint32_t)((PAGED && RPP > 16 ? pr & 15 : pr) * a.k_ld + c) * (uint32_t)sizeof(T);
    const uint32_t voff = (uint32_t)((PAGED && RPP > 16 ? pr & 15 : pr) * a.v_ld + c) * (uint32_t)sizeof(T);
    const int32_t *table = PAGED ? a.table + (int64_t)b * a.table_ld : nullptr;
    const int smask = (1 << a.page_shift) - 1;
    // A tile on its way to LDS; pages: a bit for each 16 keys that have a page.
    struct Stage {
        u32x4 k[PASSES], v[PASSES];
        uint32_t there;
    } stage;
    int pages = -1;                               // page numbers of 64 blocks of 16 keys, one a lane; -1: none there
    constexpr int BLOCKS = KT / 16, BATCH = 64 / BLOCKS;
    constexpr uint32_t ALL = (1u << BLOCKS) - 1;
    auto load = [&](int tile, Stage &to) {
        to.there = ALL;
        if constexpr (PAGED) {
            if (tile == t0 || tile % BATCH == 0) {
                const int j = (tile / BATCH * 64 + lane) * 16, p = j < end ? table[j >> a.page_shift] : -1;
                pages = p >= 0 && p < a.n_pages ? p : -1;
            }
            to.there = (uint32_t)(__ballot(pages >= 0) >> (tile % BATCH * BLOCKS)) & ALL;
        }
        const char *kp[PASSES], *vp[PASSES];
        bool page[PASSES];                                            // (of the pass's keys that this thread loads)
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int j0 = tile * KT + RPP * p;                       // the pass's first key
            page[p] = true;
            if constexpr (!PAGED) {
                kp[p] = p ? kp[p - 1] + RPP * a.k_ld * (int64_t)sizeof(T) : kbase + (k0 + j0) * a.k_ld * (int64_t)sizeof(T);
                vp[p] = p ? vp[p - 1] + RPP * a.v_ld * (int64_t)sizeof(T) : vbase + (k0 + j0) * a.v_ld * (int64_t)sizeof(T);
            } else {
                constexpr bool one = RPP <= 16;                       // a pass inside one block of 16 keys
                const int j = one ? j0 : j0 + (pr & ~15), at = tile % BATCH * BLOCKS + (one ? RPP * p : RPP * p + pr) / 16;
                const int pg = one ? __builtin_amdgcn_readlane(pages, at) : __shfl(pages, at);
                const int64_t off = (pg * a.page_stride + (j & smask) * a.k_ld) * (int64_t)sizeof(T);
                kp[p] = kbase + off, vp[p] = vbase + off;
                page[p] = pg >= 0;
            }
            if constexpr (!PAGED || RPP <= 16) asm("" : "+s"(kp[p]), "+s"(vp[p]));   // (kept scalar: a load adds the thread's offset by itself)
        }
        if (D == DP && (tile + 1) * KT <= end && to.there == ALL) {
#pragma unroll
            for (int p = 0; p < PASSES; ++p) to.k[p] = *(const u32x4 *)(kp[p] + koff), to.v[p] = *(const u32x4 *)(vp[p] + voff);
        } else {
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                to.k[p] = to.v[p] = (u32x4)0u;
                if (tile * KT + RPP * p + pr < end && c < D && page[p]) to.k[p] = *(const u32x4 *)(kp[p] + koff), to.v[p] = *(const u32x4 *)(vp[p] + voff);
            }
        }
    };
    // A value that is not finite may not reach a row that does not see it, and 0 times it is not 0: in the tiles that some row of the workgroup sees
    // in part it is stored as 0, and put back at the end for the rows that do see it.
    const int whole = past + min(r0, rows - 1) / a.group + 1;      // every row sees the keys before this one
    auto store = [&](int buf, int tile, Stage &from) {
        if ((tile + 1) * KT > whole) {
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                typedef T xu __attribute__((ext_vector_type(UNIT)));
                xu v = __builtin_bit_cast(xu, from.v[p]);
                bool any = false;
#pragma unroll
                for (int e = 0; e < UNIT; ++e) {
                    any |= !finite(v[e]);
                    v[e] = finite(v[e]) ? v[e] : (T)0.f;
                }
                if (any) odd = 1;
                from.v[p] = __builtin_bit_cast(u32x4, v);
            }
        }
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            *(u32x4 *)(ks[buf] + (pr + RPP * p) * KLD + c) = from.k[p];
            *(u32x4 *)(vs[buf] + (pr + RPP * p) * VLD + c) = from.v[p];
        }
    };

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = (f32x16)0.f;
    float m = -INFINITY, ls[4] = {0, 0, 0, 0};                        // the sum in four chains
    uint32_t there = ALL;
    if (tiles > t0) {
        load(t0, stage);
        store(t0 & 1, t0, stage);
        there = stage.there;
        if (tiles > t0 + 1) load(t0 + 1, stage);
    }
    // Tile `tile` is in LDS, the next one in registers or on its way there.  Behind the first product, while the matrix units still work on it, that one is
    // stored and the one behind it sets out: in front, its eight loads held back the product's LDS reads; at the end, the stores were waited for.
    for (int tile = t0; tile < tiles; ++tile) {
        const int buf = tile & 1, kv = tile * KT;
        __syncthreads();
        const bool live = kv <= lim_last;
        f32x16 s[KB];
        if (live) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) s[kb] = (f32x16)0.f;
#pragma unroll
            for (int st = 0; st < DS; ++st)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) s[kb] = mfma32(*(const x8 *)(ks[buf] + (32 * (kb0 + kb) + (lane & 31)) * KLD + 16 * st + 8 * h), qf[st], s[kb]);
        }
        const uint32_t there_next = stage.there;
        if (tile + 1 < tiles) store(buf ^ 1, tile + 1, stage);
        if (tile + 2 < tiles) load(tile + 2, stage);
        if (live) {
            const bool masked = kv + KT - 1 > lim_first || (PAGED && there != ALL);
            auto seen = [&](int kb, int r) {              // register r of block kb: key 32 kb + 8 (r / 4) + 4 h + r % 4
                return kv + 32 * (kb0 + kb) + 8 * (r >> 2) + 4 * h + (r & 3) <= lim && (!PAGED || (there >> (2 * (kb0 + kb) + (r >> 3)) & 1));
            };
            if (masked)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] = seen(kb, r) ? s[kb][r] : -INFINITY;
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
            mx = max_halves(mx) * a.scale_log2;
            if (__any(mx > m + 8.f)) {
                const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
#pragma unroll
                for (int i = 0; i < 4; ++i) ls[i] *= f;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] *= f;
            }
            const float ref = (m == -INFINITY ? 0.f : m) - P_SHIFT<T>;
            x8 p[KB][2];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[kb][r], a.scale_log2, -ref));
                    ls[r & 3] += e;
                    p[kb][r >> 3][r & 7] = (T)e;
                }
#pragma unroll
            for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = mfma32(read_vt<T, VLD>(vs[buf], 32 * kb0 + 16 * i, 32 * d, lane), p[i >> 1][i & 1], o[d]);
        }
        there = there_next;
    }
    float l = (ls[0] + ls[1]) + (ls[2] + ls[3]);
    if constexpr (KS == 2) {             // the two waves' parts of 32 rows: the second leaves its own in LDS
        static_assert(sizeof(ks) >= RW * 64 * (16 * DB + 2) * 4, "the parts fit where K was");
        float *part = (float *)ks + wave % RW * 64 * (16 * DB + 2) + lane;
        __syncthreads();
        if (kb0) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) part[(16 * d + r) * 64] = o[d][r];
            part[16 * DB * 64] = m, part[(16 * DB + 1) * 64] = l;
        }
        __syncthreads();
        if (kb0) return;
        const float m2 = part[16 * DB * 64], l2 = part[(16 * DB + 1) * 64], M = fmaxf(m, m2);
        const float f = factor(m, M), f2 = factor(m2, M);
        l = l * f + l2 * f2, m = M;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * f + part[(16 * d + r) * 64] * f2;
    }
    l = sum_halves(l);
    if (!valid) return;
    if (tiles > t0 && odd)
        for (int j = max(max(whole, 0) / KT, t0) * KT; j <= min(lim, min(end, tiles * KT) - 1); ++j) {
            int64_t vo = (int64_t)(k0 + j) * a.v_ld;
            if (PAGED) {
                const int p = table[j >> a.page_shift];
                if (p < 0 || p >= a.n_pages) continue;
                vo = p * a.page_stride + (j & smask) * a.v_ld;
            }
            const T *v = (const T *)a.v + vo + hk * a.v_hs;
            // (By selection, and adding -0 changes nothing.  With a branch for each value the compiler spilled 15 thousand registers at head_dim 33..64, 3.5 KB
            // of scratch a lane; without, 3 waves a SIMD in place of 2: 4096 rows, 32/8 heads of 64 in f16 take 109 us in place of 129.)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = 32 * d + 8 * (r >> 2) + 4 * h + (r & 3);
                    const float x = (float)v[min(at, D - 1)];
                    o[d][r] += at < D && !finite(x) ? x : -0.f;
                }
        }
    if (used > 1) {                      // this part's sums of the row, for attn_prompt_join_k
        float *to = (float *)a.ws + (((int64_t)(q0 + tok) * a.n_head + head) * parts + blockIdx.y) * (DP + 4);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) *(f32x4 *)(to + 32 * d + 2 * r + 4 * h) = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        if (h == 0) to[DP] = m, to[DP + 1] = l;
        return;
    }
    const float inv = l == 0 ? 0.f : 1 / l;
    T *out = (T *)a.out + (int64_t)(q0 + tok) * a.o_ld + head * a.o_hs;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            typedef T x4 __attribute__((ext_vector_type(4)));
            const int at = 32 * d + 2 * r + 4 * h;
            const f32x4 y = {o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv};
            if (at < D) *(x4 *)(out + at) = __builtin_convertvector(y, x4);
        }
}

// The rows whose keys were cut into parts: the same blocks, a thread for four features of a row.
template <typename T, int DP, bool PAGED, int ROWS>
__global__ __launch_bounds__(256) void attn_prompt_join_k(AttnArgs a, int parts) {
    constexpr int LANES = DP / 4, SIDE = 256 / LANES;
    const int n_head_kv = a.n_head / a.group, hk = blockIdx.x % n_head_kv, c = threadIdx.x % LANES * 4;
    const Block at = find_block<PAGED, ROWS>(a, blockIdx.x / n_head_kv, gridDim.x / n_head_kv);
    if (at.b < 0) return;
    const int rows = at.lq * a.group, r0 = at.blk * ROWS, past = at.lk - at.lq;
    const int end = min(past + min(r0 + ROWS - 1, rows - 1) / a.group + 1, at.lk);
    int t0, t1;
    const int used = cut_tiles<Tile<T>::KT>(end, parts, 0, &t0, &t1);
    if (used == 1) return;
    for (int row = r0 + blockIdx.y * SIDE + threadIdx.x / LANES; row < min(r0 + ROWS, rows); row += SIDE * gridDim.y) {
        const int tok = row / a.group, head = hk * a.group + row % a.group;
        const float *part = (const float *)a.ws + ((int64_t)(at.q0 + tok) * a.n_head + head) * parts * (DP + 4);
        float M = -INFINITY, l = 0;
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll 4
        for (int s = 0; s < used; ++s) M = fmaxf(M, part[s * (DP + 4) + DP]);
#pragma unroll 4
        for (int s = 0; s < used; ++s) {
            const float *p = part + s * (DP + 4);
            const f32x4 x = *(const f32x4 *)(p + c);
            const float ls = p[DP + 1], f = factor(p[DP], M);
            l += ls * f, sum += x * f;
        }
        typedef T x4 __attribute__((ext_vector_type(4)));
        if (c < a.head_dim) *(x4 *)((T *)a.out + (int64_t)(at.q0 + tok) * a.o_ld + head * a.o_hs + c) = __builtin_convertvector(sum * (l == 0 ? 0.f : 1 / l), x4);
    }
}

template <typename T, int DP, bool PAGED, int KS, int W>
static hipError_t prompt_launch(const AttnArgs &a, int parts, hipStream_t st) {
    constexpr int ROWS = 32 * W / KS;
    const int64_t rows = (int64_t)a.n_q * a.group, blocks = (rows / ROWS + a.n_seq) * (a.n_head / a.group);   // every sequence may end inside a block
    if (blocks * 64 * W > UINT32_MAX) return hipErrorInvalidValue;
    attn_prompt_k<T, DP, PAGED, KS, W><<<dim3((unsigned)blocks, parts), 64 * W, 0, st>>>(a, parts);
    if (parts > 1) attn_prompt_join_k<T, DP, PAGED, ROWS><<<dim3((unsigned)blocks, ROWS * DP / 1024), 256, 0, st>>>(a, parts);
    return hipGetLastError();
}

// Few workgroups (16-bit types): two waves for 32 rows.  A tile then takes a wave 1.3 us instead of 1.6, and there are twice as many workgroups: 512
// rows behind 1536, 32 heads of 128 in f16 (128 blocks of 128 rows) 51 -> 42 us; 1000 rows, 32/8 heads in bf16 (256) 30 -> 27; but 2048, 32/32 (544)
// 60 -> 64 and 4096, 32/8 (1032) 170 -> 202: each wave's share of a tile's loads and waits is as large as before.
// Many rows of long sequences: eight waves, which load a tile once for 256 rows.  8192 rows, 32/8 heads of 128 in bf16: 596 -> 555 us, 4096 in f16 178 -> 160,
// two of 4096 316 -> 298; 2048, 32/32 in f16, as before (60).  With fewer than 2048 keys a sequence the last block's empty rows and the longest block's
// way outweigh that: 16 of 512, 32/32 87 -> 95, 48 of 100 40 -> 58, 200 of 40 101 -> 160; four of 1024, 32/8 59 -> 57, eight packed ones of 1 to 1500
// 61 either way.
// Very few, behind many keys: the keys too are cut into parts of four tiles or more, until each CU has two workgroups, and joined by a second launch.  64
// rows behind 30000, 32/8 heads of 128 in bf16: 575 -> 79 us (105 at one workgroup a CU); 16 behind 2000 in f16: 47 -> 20 (25 with parts of eight
// tiles); 200 behind 1600, 8 heads in f32: 249 -> 44.  Where nearly each CU has one anyway, from 32 tiles on: 512 rows against 8192 keys, 32/32 in f16 (256
// blocks), 168 -> 119, 4096 88 -> 71, 2048 49 -> 45; 1536 39 -> 40, 512 of a longer table 18 -> 24.  Three or four parts there, against 8192: 145, 122.
static bool few_blocks(int type, int64_t rows, int64_t n_head_kv, int n_seq) { return type != FL_TYPE_F32 && (rows / 128 + n_seq) * n_head_kv < 512; }
static int prompt_parts(int type, int64_t rows, int64_t n_head_kv, int n_seq, int64_t max_keys) {
    const int tile = type == FL_TYPE_F32 ? 32 : 64, block = few_blocks(type, rows, n_head_kv, n_seq) ? 64 : 128;
    const int64_t blocks = max((rows + block - 1) / block, (int64_t)n_seq) * n_head_kv;
    if (blocks > 192 && max_keys < 32 * tile) return 1;
    return (int)max((int64_t)1, min(min((int64_t)16, 512 / max(blocks, (int64_t)1)), max_keys / (4 * tile)));
}
size_t attn_prompt_workspace(int type, int n_q, int n_seq, int n_head, int n_head_kv, int head_dim, int64_t max_keys) {
    const int parts = prompt_parts(type, (int64_t)n_q * (n_head / n_head_kv), n_head_kv, n_seq, max_keys);
    return parts > 1 ? (size_t)n_q * n_head * parts * ((head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : 128) + 4) * 4 : 0;
}

template <typename T, int DP, bool PAGED>
static hipError_t prompt_rows(const AttnArgs &a, hipStream_t st) {
    const int64_t rows = (int64_t)a.n_q * a.group, n_head_kv = a.n_head / a.group;
    const int type = sizeof(T) == 4 ? FL_TYPE_F32 : FL_TYPE_F16, parts = prompt_parts(type, rows, n_head_kv, a.n_seq, PAGED ? (int64_t)a.n_table << a.page_shift : a.n_kv);
    if constexpr (sizeof(T) == 2) {
        if (few_blocks(type, rows, n_head_kv, a.n_seq)) return prompt_launch<T, DP, PAGED, 2, 4>(a, parts, st);
        if constexpr (DP == 128 && !PAGED)
            if (rows / 256 * n_head_kv >= 512 && a.n_kv / 2048 >= a.n_seq) return prompt_launch<T, DP, PAGED, 1, 8>(a, 1, st);
    }
    return prompt_launch<T, DP, PAGED, 1, 4>(a, parts, st);
}

template <typename T>
static hipError_t prompt_dim(const AttnArgs &a, bool paged, hipStream_t st) {
    if (a.head_dim <= 32) return paged ? prompt_rows<T, 32, true>(a, st) : prompt_rows<T, 32, false>(a, st);
    if (a.head_dim <= 64) return paged ? prompt_rows<T, 64, true>(a, st) : prompt_rows<T, 64, false>(a, st);
    return paged ? prompt_rows<T, 128, true>(a, st) : prompt_rows<T, 128, false>(a, st);
}

hipError_t attn_prompt(const AttnArgs &a, int type, bool paged, hipStream_t st) {
    return type == FL_TYPE_F32 ? prompt_dim<float>(a, paged, st) : type == FL_TYPE_F16 ? prompt_dim<h16>(a, paged, st) : prompt_dim<b16>(a, paged, st);
}

}  // namespace fl
