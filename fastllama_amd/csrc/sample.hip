// sample.hip -- a token for each row of logits: temperature, top-k, top-p and min-p from a given uniform number.
//
//   w_i = exp((l_i - max l) / T), the tokens in the order of (l falling, index rising):
//   kept = the shortest of: the first top_k;  the shortest prefix of those whose sum is >= top_p * theirs;  those with w_i >= min_p;  at least one
//   token = the first kept i, in the order of the indexes, whose running sum of w exceeds u * (the sum of all kept w)
//
// Weights are whole numbers, w_i * 2^44 rounded once from a 64-bit exponential: their sums are exact and do not depend on the order of
// additions or atomics, and 2^18 of them fit 63 bits.  A kept set is a threshold: all keys above `tkey` and the first `ties` that equal it.
#include "serve_kernels.h"
#include "serve_device.h"
#include "../../include/fastllama_hip.h"

namespace fl {

typedef unsigned long long u64;
constexpr int S_THREADS = 1024, S_BITS = 44;

// Keys in the order of the values: NaN counts as -infinity, -0 as 0.
__device__ inline uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ inline float value_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

// 2^44 exp((value - max) / T) as a whole number; c = log2(e) / T.  2^f, |f| <= 1/2, by its series to f^12 (the rest is below 2^-50).
__device__ inline u64 weight_of(uint32_t key, uint32_t kmax, double max, double c) {
    if (key == kmax) return 1ull << S_BITS;
    if (key == 0) return 0;
    const double y = ((double)value_of(key) - max) * c;
    if (!(y > -(S_BITS + 2))) return 0;
    const double n = rint(y), f = y - n;
    double p = 2.5678435993488206e-11;                 // ln(2)^k / k!
    p = fma(p, f, 4.4455382718708116e-10);
    p = fma(p, f, 7.0549116208011234e-09);
    p = fma(p, f, 1.0178086009239700e-07);
    p = fma(p, f, 1.3215486790144310e-06);
    p = fma(p, f, 1.5252733804059841e-05);
    p = fma(p, f, 1.5403530393381609e-04);
    p = fma(p, f, 1.3333558146428443e-03);
    p = fma(p, f, 9.6181291076284769e-03);
    p = fma(p, f, 5.5504108664821583e-02);
    p = fma(p, f, 2.4022650695910072e-01);
    p = fma(p, f, 6.9314718055994529e-01);
    p = fma(p, f, 1.0);
    const double w = ldexp(p, (int)n + S_BITS) + 4503599627370496.0;     // + 2^52: the fraction's bits are the rounded whole number
    return (u64)__double_as_longlong(w) & ((1ull << 52) - 1);
}

template <typename V>
__device__ inline V wave_sum(V x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
template <typename V>
__device__ inline V wave_scan(V x) {     // over the lanes up to and with this one
    for (int o = 1; o < 64; o <<= 1) {
        const V up = __shfl_up(x, o);
        if ((int)(threadIdx.x & 63) >= o) x += up;
    }
    return x;
}

constexpr int BINS = 2048, LIST = 256, WAVES = S_THREADS / 64;

struct Shared {
    u64 whist[BINS];
    uint32_t chist[BINS];
    u64 wsum[WAVES];
    uint32_t wcount[WAVES];
    u64 lw[LIST];                        // a short list of candidates: weight, key, index
    uint32_t lkey[LIST], lidx[LIST];
    u64 before, need;
    uint32_t kmax, prefix, n;
    int bin, first;
};

// One row, seen by all passes in the same way: wave w has the stretch [w * seg, (w + 1) * seg) and takes 256 consecutive logits at a time, four a lane.
template <typename T>
struct Row {
    typedef T x4 __attribute__((ext_vector_type(4)));
    const T *x;
    int n, i0, i1;
    bool wide;                           // aligned to four logits
    __device__ void four(int i, uint32_t k[4]) const {
        if (wide && i + 4 <= i1) {
            const x4 v = *(const x4 *)(x + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = key_of((float)v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = i + e < i1 ? key_of((float)x[i + e]) : 0;
        }
    }
    template <typename F>
    __device__ void each(F f) const {    // f(key, index) of the logits that are not -infinity
#pragma unroll 4
        for (int i = i0 + 4 * (threadIdx.x & 63); i < i1; i += 256) {
            uint32_t k[4];
            four(i, k);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (k[e]) f(k[e], i + e);
        }
    }
};

// Distance below the largest logit in steps of T / 64, never falling as the logit falls; from BINS on the weight is 0 (2^-46 = e^-31.9).
__device__ inline int bin_of(uint32_t key, uint32_t kmax, float max, float per) {
    if (key == kmax) return 0;
    const float d = (0.5f * max - 0.5f * value_of(key)) * per;         // (halves: their difference does not overflow)
    return d < (float)BINS ? (int)d : BINS;
}

// The bin in which the sums over the bins (weights or counts) reach `need`: s.bin, and s.before, the sum in front of it.  All threads call;
// returns the sum of all bins.
template <bool WEIGHTS>
__device__ u64 scan_bins(Shared &s, u64 need) {
    const int t = threadIdx.x;
    static_assert(BINS == 2 * S_THREADS, "two bins a thread");
    const u64 a = WEIGHTS ? s.whist[2 * t] : s.chist[2 * t], b = WEIGHTS ? s.whist[2 * t + 1] : s.chist[2 * t + 1];
    const u64 incl = wave_scan(a + b);
    if ((t & 63) == 63) s.wsum[t >> 6] = incl;
    __syncthreads();
    u64 base = 0, total = 0;
    for (int w = 0; w < WAVES; ++w) {
        if (w < t >> 6) base += s.wsum[w];
        total += s.wsum[w];
    }
    u64 at = base + incl - a - b;
    if (at < need && at + a >= need) s.bin = 2 * t, s.before = at;
    at += a;
    if (at < need && at + b >= need) s.bin = 2 * t + 1, s.before = at;
    __syncthreads();
    return total;
}

// The candidates for which in(key, index) holds, in any order: s.lkey, s.lidx, s.lw and s.n of them (LIST at most are kept).
template <typename T, typename In>
__device__ void gather(Shared &s, const Row<T> &r, uint32_t kmax, double max, double c, In in) {
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    r.each([&](uint32_t k, int i) {
        if (in(k, i)) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < LIST) s.lkey[at] = k, s.lidx[at] = i;
        }
    });
    __syncthreads();
    const int n = min(s.n, (uint32_t)LIST);
    if ((int)threadIdx.x < n) s.lw[threadIdx.x] = weight_of(s.lkey[threadIdx.x], kmax, max, c);
    __syncthreads();
}

// The key at which the sum over the keys with in(), in falling order (of 1 each, or of the weights), reaches `need`: *tkey, and in *ties how many
// equal keys that takes.  0 < need <= the sum over all.  A short list is ranked by comparing all with all; a long one (many logits within T / 64 of each
// other) goes by the key's four bytes from the top.
template <bool WEIGHTS, typename T, typename In>
__device__ void cut(Shared &s, const Row<T> &r, uint32_t kmax, double max, double c, u64 need, In in, uint32_t *tkey, u64 *ties) {
    const int t = threadIdx.x;
    gather(s, r, kmax, max, c, in);
    const int n = s.n;
    if (n <= LIST) {
        if (t < n) {
            const uint32_t key = s.lkey[t], idx = s.lidx[t];
            const u64 own = WEIGHTS ? s.lw[t] : 1;
            u64 sum = 0;
            uint32_t same = 1;
            for (int j = 0; j < n; ++j) {
                const uint32_t kj = s.lkey[j];
                const bool before = kj > key || (kj == key && s.lidx[j] < idx);
                sum += before ? (WEIGHTS ? s.lw[j] : 1) : 0;
                same += before && kj == key;
            }
            if (sum < need && sum + own >= need) s.prefix = key, s.need = same;
        }
        __syncthreads();
        *tkey = s.prefix, *ties = s.need;
        __syncthreads();
        return;
    }
    uint32_t prefix = 0, mask = 0;
    u64 left = need;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) s.whist[t] = 0;
        __syncthreads();
        r.each([&](uint32_t k, int i) {
            if (((k ^ prefix) & mask) == 0 && in(k, i)) {
                const u64 w = WEIGHTS ? weight_of(k, kmax, max, c) : 1;
                if (w) atomicAdd(&s.whist[k >> shift & 255], w);
            }
        });
        __syncthreads();
        if (t < 64) {                    // lane L: bytes 255 - 4 L .. 252 - 4 L, in falling order
            u64 own = 0;
            for (int e = 0; e < 4; ++e) own += s.whist[255 - 4 * t - e];
            u64 at = wave_scan(own) - own;
            for (int e = 0; e < 4; ++e) {
                const int byte = 255 - 4 * t - e;
                const u64 h = s.whist[byte];
                if (at < left && at + h >= left) s.prefix = prefix | (uint32_t)byte << shift, s.need = left - at;
                at += h;
            }
        }
        __syncthreads();
        prefix = s.prefix, left = s.need, mask |= 255u << shift;
        __syncthreads();
    }
    const u64 w = WEIGHTS ? weight_of(prefix, kmax, max, c) : 1;
    *tkey = prefix, *ties = (left + w - 1) / w;
}

__device__ inline u64 share(float p, u64 sum) {      // the least whole number that is p of the sum, at least 1
    return min(max(p > 0 ? (u64)ceil((double)p * (double)sum) : (u64)1, (u64)1), sum);
}
__device__ inline u64 target_of(float u, u64 total) {
    const double x = u > 0 ? (u < 1 ? (double)u : 1.0) : 0.0;
    return min((u64)floor(x * (double)total), total - 1);
}

template <typename T>
__global__ __launch_bounds__(S_THREADS) void sample_k(SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
    Row<T> r;
    r.x = (const T *)a.logits + row * a.ld, r.n = a.n_vocab;
    r.wide = (uintptr_t)r.x % sizeof(typename Row<T>::x4) == 0;
    const int seg = ((r.n + WAVES - 1) / WAVES + 3) & ~3;
    r.i0 = min(wave * seg, r.n), r.i1 = min(r.i0 + seg, r.n);
    const float temp = a.temperature_p ? a.temperature_p[row] : a.temperature, top_p = a.top_p_p ? a.top_p_p[row] : a.top_p;
    const float min_p = a.min_p_p ? a.min_p_p[row] : a.min_p, u = a.u[row];
    const int top_k = a.top_k_p ? a.top_k_p[row] : a.top_k;

    if (t == 0) s.kmax = 0, s.first = INT32_MAX;
    s.chist[2 * t] = s.chist[2 * t + 1] = 0;
    s.whist[2 * t] = s.whist[2 * t + 1] = 0;
    __syncthreads();
    uint32_t kmax = 0;
    r.each([&](uint32_t k, int) { kmax = max(kmax, k); });
    for (int o = 32; o; o >>= 1) kmax = max(kmax, (uint32_t)__shfl_xor((int)kmax, o));
    if (lane == 0 && kmax) atomicMax(&s.kmax, kmax);
    __syncthreads();
    kmax = s.kmax;
    if (kmax == 0) {                     // no token is allowed
        if (t == 0) a.tokens[row] = -1;
        return;
    }
    if (!(temp > 0)) {                   // greedy
        r.each([&](uint32_t k, int i) {
            if (k == kmax) atomicMin(&s.first, i);
        });
        __syncthreads();
        if (t == 0) a.tokens[row] = s.first;
        return;
    }
    const float mf = value_of(kmax), per = fminf(128.f / temp, 3e38f);
    const double mx = mf, c = 1.4426950408889634074 / (double)temp;
    const u64 wmin = min_p > 0 ? (u64)ceil(fmin((double)min_p, 1.0) * (double)(1ull << S_BITS)) : 0;

    uint32_t tkey = 0;                   // kept so far: keys above tkey, and the first `ties` equal to it; 0: all
    u64 ties = 0;
    if (top_k > 0 && top_k < r.n) {
        r.each([&](uint32_t k, int) {
            const int b = bin_of(k, kmax, mf, per);
            if (b < BINS) atomicAdd(&s.chist[b], 1u);
        });
        __syncthreads();
        const u64 total = scan_bins<false>(s, top_k);
        if ((u64)top_k <= total) {       // (otherwise what top_k drops has no weight)
            const int bin = s.bin;
            const u64 before = s.before;
            const uint32_t upto = (uint32_t)before + s.chist[bin];
            __syncthreads();
            if (upto <= LIST) {
                // few candidates: every question is answered by comparing all with all
                gather(s, r, kmax, mx, c, [&](uint32_t k, int) { return bin_of(k, kmax, mf, per) <= bin; });
                const int n = s.n;
                uint32_t key = 0, idx = 0;
                u64 w = 0, sum = 0;
                int rank = 0;
                if (t < n) {
                    key = s.lkey[t], idx = s.lidx[t], w = s.lw[t];
                    for (int j = 0; j < n; ++j) {
                        const bool before = s.lkey[j] > key || (s.lkey[j] == key && s.lidx[j] < idx);
                        rank += before, sum += before ? s.lw[j] : 0;
                    }
                    if (rank == top_k - 1) s.need = sum + w;           // the sum over the first top_k
                }
                __syncthreads();
                const u64 need = top_p < 1 ? share(top_p, s.need) : s.need;
                const bool keep = t < n && rank < top_k && sum < need && w >= wmin;
                __syncthreads();
                if (t < n) s.lw[t] = keep ? w : 0;
                __syncthreads();
                if (keep) {
                    u64 run = 0, all = 0;
                    for (int j = 0; j < n; ++j) {
                        const u64 x = s.lw[j];
                        all += x, run += s.lidx[j] < idx ? x : 0;
                    }
                    const u64 target = target_of(u, all);
                    if (run <= target && target < run + w) a.tokens[row] = (int32_t)idx;
                }
                return;
            }
            cut<false>(s, r, kmax, mx, c, top_k - before, [&](uint32_t k, int) { return bin_of(k, kmax, mf, per) == bin; }, &tkey, &ties);
        }
    }
    if (top_p < 1) {
        if (top_k > 0 && top_k < r.n) {                               // (the radix steps of a cut use whist too)
            s.whist[2 * t] = s.whist[2 * t + 1] = 0;
            __syncthreads();
        }
        r.each([&](uint32_t k, int) {
            if (k > tkey) {
                const u64 w = weight_of(k, kmax, mx, c);
                const int b = bin_of(k, kmax, mf, per);
                if (w && b < BINS) atomicAdd(&s.whist[b], w);
            }
        });
        if (t == 0 && tkey) {
            const u64 w = ties * weight_of(tkey, kmax, mx, c);
            const int b = bin_of(tkey, kmax, mf, per);
            if (w && b < BINS) atomicAdd(&s.whist[b], w);
        }
        __syncthreads();
        const u64 sum = scan_bins<true>(s, ~0ull), need = share(top_p, sum);
        scan_bins<true>(s, need);
        const int bin = s.bin;
        const u64 before = s.before;
        const uint32_t low = tkey;
        __syncthreads();
        cut<true>(s, r, kmax, mx, c, need - before, [&](uint32_t k, int) { return k >= low && bin_of(k, kmax, mf, per) == bin; }, &tkey, &ties);
    }

    // The kept weights in the order of the indexes: each wave's sum over its stretch, then the wave whose stretch holds the target looks for it.
    const u64 wt = tkey ? weight_of(tkey, kmax, mx, c) : 0;
    const bool tied = tkey && wt >= wmin;
    u64 above = 0;
    uint32_t equal = 0;
    r.each([&](uint32_t k, int) {
        if (k > tkey) {
            const u64 w = weight_of(k, kmax, mx, c);
            above += w >= wmin ? w : 0;
        } else if (k == tkey && tied) ++equal;
    });
    above = wave_sum(above), equal = wave_sum(equal);
    if (lane == 0) s.wsum[wave] = above, s.wcount[wave] = equal;
    __syncthreads();
    u64 run = 0, total = 0, seen = 0, count = 0;
    for (int w = 0; w < WAVES; ++w) {
        if (w == wave) run = total, seen = count;
        total += s.wsum[w], count += s.wcount[w];
    }
    run += min(seen, ties) * wt;
    total += min(count, ties) * wt;
    const u64 target = target_of(u, total);
    if (run > target || target >= run + above + (min(seen + equal, ties) - min(seen, ties)) * wt) return;
    for (int i = r.i0 + 4 * lane; i - 4 * lane < r.i1; i += 256) {
        uint32_t k[4];
        r.four(min(i, r.i1), k);
        u64 w[4], own = 0;
        uint32_t eq = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = k[e] > tkey ? weight_of(k[e], kmax, mx, c) : 0;
            w[e] = w[e] >= wmin ? w[e] : 0;
            own += w[e], eq += tied && k[e] == tkey;
        }
        const uint32_t eq_incl = wave_scan(eq);
        u64 at = seen + eq_incl - eq;                                  // equal keys in front of this lane's
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (tied && k[e] == tkey) {
                w[e] = at++ < ties ? wt : 0;
                own += w[e];
            }
        const u64 incl = wave_scan(own);
        u64 pos = run + incl - own;
        if (pos <= target && target < pos + own)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (pos <= target && target < pos + w[e]) a.tokens[row] = i + e;
                pos += w[e];
            }
        run += __shfl(incl, 63), seen += __shfl(eq_incl, 63);
        if (target < run) return;
    }
}

hipError_t sample(const SampleArgs &a, int type, hipStream_t st) {
    if (type == FL_TYPE_F32) sample_k<float><<<a.rows, S_THREADS, 0, st>>>(a);
    else if (type == FL_TYPE_F16) sample_k<h16><<<a.rows, S_THREADS, 0, st>>>(a);
    else sample_k<b16><<<a.rows, S_THREADS, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace fl
