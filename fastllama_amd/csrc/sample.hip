// sample.hip -- a token for each row of logits: temperature, top-k, top-p and min-p from a given uniform number.
//
//   w_i = exp((l_i - max l) / T), the tokens in the order of (l falling, index rising):
//   kept = the shortest of: the first top_k;  the shortest prefix of those whose sum is >= top_p * theirs;  those with w_i >= min_p;  at least one
//   token = the first kept i, in the order of the indexes, whose running sum of w exceeds u * (the sum of all kept w)
//
// One CU streams a row of logits far more slowly than the card does, so a row is cut into parts of 4096 logits or a few times that, a workgroup of 256
// threads each:
//   scan    each part's largest logit; where top_k is small also what can be among the row's first top_k: what is not below the top_k-th largest of
//           the threads' own largest, part by part
//   hist    otherwise, for the rows that have a top_k or a top_p: how the row's counts or weights spread over the distance from its largest logit, by
//           whole-number atomics; for the others each part's sum
//   gather  what the exact cut is found among: for a top_p alone the part's logits at the distance that holds the cut, and the sum of those above; for
//           a top_k all up to that distance
//   draw    a workgroup for each row: the exact cuts, and the token
// Where one top_k of at most 128 is given for all rows, scan and draw are all.  The lists hold 512 candidates a part and 8192 a row.  A row with more -- very
// many logits alike, or a top_k that is larger -- is done by draw alone, over all of it: 128 rows of 32000 (8 parts) take 43 us at a top_k of 500, 47 at
// 2000 and 124 at 5000; 256 of 128256 (16 parts of two rounds) 116 at 2000 and 505 at 5000; one of 32000 28, 33 and 95.
//
// Weights are whole numbers, w_i * 2^44 rounded once from a 64-bit exponential: their sums are exact and do not depend on the order of
// additions or atomics, and 2^18 of them fit 63 bits.  A kept set is a threshold: all keys above `tkey` and the first `ties` that equal it.
#include <cfloat>
#include <cmath>
#include "serve_kernels.h"
#include "serve_device.h"
#include "../../include/fastllama_hip.h"

namespace fl {

typedef unsigned long long u64;
constexpr int S_THREADS = 1024, S_BITS = 44, P_THREADS = 256;

// Keys in the order of the values: NaN counts as -infinity, -0 as 0.
__device__ inline uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ inline float value_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

// 2^(j/32) for j = 0..31, times 2^44: the whole numbers' unit.
struct PowerTable {
    double t[32];
};

// Weights of one row, 2^44 exp((value - max) / T) as whole numbers: 2^y, y = (value - max) log2(e) / T, with y = n + j/32 + f, |f| <= 1/64, is
// 2^n 2^(j/32) e^(f ln 2), the last by its series to f^5 (the rest is below 2^-48).
struct Weigher {
    float top;                           // the largest
    double max, c;
    const double *table;
    __device__ u64 of(float x) const {
        const double d = ((double)x - max) * c;
        const bool some = d > -(S_BITS + 2);                          // (otherwise 0; no number where both are infinite)
        const double y = some ? d : 0.0;
        constexpr double shift = 6755399441055744.0 / 32;             // 1.5 * 2^52 / 32: the sum's last bits are 32 y rounded
        const double r = y + shift, f = y - (r - shift);
        const int k = (int)(uint32_t)__double_as_longlong(r);
        double p = 1.3333558146428443e-03;                            // ln(2)^i / i!
        p = fma(p, f, 9.6181291076284769e-03);
        p = fma(p, f, 5.5504108664821583e-02);
        p = fma(p, f, 2.4022650695910072e-01);
        p = fma(p, f, 6.9314718055994529e-01);
        p = fma(p, f, 1.0);
        const double t = __longlong_as_double(__double_as_longlong(table[k & 31]) + ((long long)(k >> 5) << 52));
        const double w = fma(t, p, 4503599627370496.0);               // + 2^52: the fraction's bits are the rounded whole number
        const u64 v = some ? (u64)__double_as_longlong(w) & ((1ull << 52) - 1) : 0;
        return x == top ? 1ull << S_BITS : v;                         // (also +infinity, which is no distance from itself)
    }
    __device__ u64 of_key(uint32_t key) const { return key ? of(value_of(key)) : 0; }
};

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

__device__ inline u64 share(float p, u64 sum) {      // the least whole number that is p of the sum, at least 1
    return min(max(p > 0 ? (u64)ceil((double)p * (double)sum) : (u64)1, (u64)1), sum);
}
__device__ inline u64 target_of(float u, u64 total) {
    const double x = u > 0 ? (u < 1 ? (double)u : 1.0) : 0.0;
    return min((u64)floor(x * (double)total), total - 1);
}

constexpr int BINS = 2048, SHORT = 256, WAVES = S_THREADS / 64, CAP = 8192;
constexpr int ROUND = 4096, P_CAP = 512;     // logits that a part's workgroup has in registers at a time; candidates of a part
constexpr int FEW = 128;                     // "small" top_k: half of a part's threads
constexpr int COARSE = P_THREADS;            // bins, one a thread, for a part's own cut

struct Part {
    uint32_t kmax, first, held, pad;         // the largest key, its first index, candidates (may be more than P_CAP)
    u64 sum, pad2;                           // weights: all (no cut), or those of the bins above the cut's (top_p alone)
};
// The workspace: for each row its parts, the bins, and each part's candidates (key, index).
struct Work {
    Part *part;
    u64 *hist;
    uint2 *list;
    __host__ __device__ static size_t row_bytes(int parts) { return (size_t)parts * (sizeof(Part) + P_CAP * sizeof(uint2)) + BINS * sizeof(u64); }
    __device__ Work(void *ws, int row, int parts) {
        char *p = (char *)ws + row * row_bytes(parts);
        hist = (u64 *)p, part = (Part *)(p + BINS * sizeof(u64)), list = (uint2 *)(part + parts);
    }
};

// A row's settings and what they ask for.
struct Settings {
    float temp, top_p;
    int top_k;                               // 0: none
    u64 wmin;
    bool greedy, few;
    __device__ Settings(const SampleArgs &a, int row) {
        temp = a.temperature_p ? a.temperature_p[row] : a.temperature, top_p = a.top_p_p ? a.top_p_p[row] : a.top_p;
        const float min_p = a.min_p_p ? a.min_p_p[row] : a.min_p;
        const int k = a.top_k_p ? a.top_k_p[row] : a.top_k;
        top_k = k > 0 && k < a.n_vocab ? k : 0;
        wmin = min_p > 0 ? (u64)ceil(fmin((double)min_p, 1.0) * (double)(1ull << S_BITS)) : 0;
        greedy = !(temp > 0), few = top_k > 0 && top_k <= FEW;
    }
};

// Distance below the largest logit in steps of T / 64, never falling as the logit falls; from BINS on, and for -infinity, the weight is 0
// (2^-46 = e^-31.9).  Taken from the halves, whose difference does not overflow.  +infinity below itself is no number: med3 makes it bin 0.
struct Bins {
    float half_max, per;                 // per > 0
    __device__ uint32_t operator()(float x) const { return (uint32_t)__builtin_amdgcn_fmed3f(fmaf(x, -0.5f, half_max) * per, 0.f, 2.f * BINS); }
    __device__ Bins(float max, float temp) : half_max(0.5f * max), per(fmaxf(fminf(128.f / temp, 3e38f), FLT_MIN)) {}   // (f32's whole range is 8 FLT_MIN steps)
    __device__ uint32_t of_key(uint32_t key) const { return (*this)(value_of(key)); }
};

__device__ inline Weigher weigher(float max, float temp, const double *table) { return Weigher{max, (double)max, 1.4426950408889634074 / (double)temp, table}; }

// A row's logits: NaN reads as -infinity.
template <typename T>
struct Row {
    typedef T x4 __attribute__((ext_vector_type(4)));
    const T *x;
    int n;
    bool wide;                               // aligned to four logits
    __device__ Row(const SampleArgs &a, int row) : x((const T *)a.logits + row * a.ld), n(a.n_vocab), wide((uintptr_t)x % sizeof(x4) == 0) {}
    __device__ f32x4 four(int i) const {
        f32x4 y;
        if (wide && i + 4 <= n) y = __builtin_convertvector(*(const x4 *)(x + i), f32x4);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = i + e < n ? (float)x[i + e] : -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaxf(y[e], -INFINITY);
        return y;
    }
    // The round's four fours of this thread: wave w has 1024 consecutive logits, a lane four of every 256.
    __device__ int at(int p0, int d) const { return p0 + (threadIdx.x >> 6) * 1024 + 256 * d + 4 * (threadIdx.x & 63); }
    __device__ void round(int p0, f32x4 y[4]) const {
        if (wide && p0 + ROUND <= n) {       // (uniform: all loads at once)
#pragma unroll
            for (int d = 0; d < 4; ++d) y[d] = __builtin_convertvector(*(const x4 *)(x + at(p0, d)), f32x4);
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[d][e] = fmaxf(y[d][e], -INFINITY);
        } else {
#pragma unroll
            for (int d = 0; d < 4; ++d) y[d] = four(min(at(p0, d), n));
        }
    }
};

// The bin in which the sums over the bins (in order, v[] of them: thread t holds the bins from t * PER on) reach need_of(sum of all): *bin and *before, the sum in
// front of it, for all threads; returns the sum.  `sums`: a place for each wave, `found`: two.
template <int PER, int N, typename Need>
__device__ u64 scan_bins(const u64 v[PER], u64 *sums, u64 *found, Need need_of, uint32_t *bin, u64 *before) {
    const int t = threadIdx.x;
    u64 own = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) own += v[i];
    const u64 incl = wave_scan(own);
    if ((t & 63) == 63) sums[t >> 6] = incl;
    if (t == 0) found[0] = BINS - 1, found[1] = 0;
    __syncthreads();
    u64 base = 0, total = 0;
#pragma unroll 4
    for (int w = 0; w < N / 64; ++w) {
        if (w < t >> 6) base += sums[w];
        total += sums[w];
    }
    const u64 need = need_of(total);
    u64 at = base + incl - own;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (at < need && at + v[i] >= need) found[0] = t * PER + i, found[1] = at;
        at += v[i];
    }
    __syncthreads();
    *bin = (uint32_t)found[0], *before = found[1];
    __syncthreads();
    return total;
}

// A part's logits of bins low..high, in the order of the indexes, into its list; returns how many there are.  below(logit): called for those of bins
// under `low`.
template <typename T, typename Below>
__device__ int compact(const Row<T> &r, int p0, int p1, Bins bins, uint32_t low, uint32_t high, uint2 *list, int *counts, Below below) {
    const int wave = threadIdx.x >> 6;
    int held = 0;
    for (int p = p0; p < p1; p += ROUND) {
        f32x4 y[4];
        r.round(p, y);
        uint32_t in = 0;                     // a bit for each of the sixteen
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float z = d == 0 ? y[0][e] : d == 1 ? y[1][e] : d == 2 ? y[2][e] : y[3][e];
                const uint32_t b = bins(z);
                in |= (uint32_t)(b >= low && b <= high) << (4 * d + e);
                if (b < low) below(z);
            }
        const int n = wave_sum(__popc(in));
        if ((threadIdx.x & 63) == 0) counts[wave] = n;
        __syncthreads();
        int at = held;
        for (int w = 0; w < P_THREADS / 64; ++w) {
            if (w < wave) at += counts[w];
            held += counts[w];
        }
        if (n)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int m = __popc(in >> (4 * d) & 15), incl = wave_scan(m);
                int to = at + incl - m;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (in >> (4 * d + e) & 1) {
                        if (to < P_CAP) list[to] = make_uint2(key_of(y[d][e]), r.at(p, d) + e);
                        ++to;
                    }
                at += __builtin_amdgcn_readlane(incl, 63);
            }
        __syncthreads();
    }
    return held;
}

// The largest key of a row's parts (LDS or registers of all threads agree).
__device__ inline uint32_t row_max(const Work &w, int parts) {
    uint32_t k = 0;
    for (int p = threadIdx.x & 63; p < parts; p += 64) k = max(k, w.part[p].kmax);
    for (int o = 32; o; o >>= 1) k = max(k, (uint32_t)__shfl_xor((int)k, o));
    return k;
}

template <typename T>
__global__ __launch_bounds__(P_THREADS) void sample_scan_k(SampleArgs a, int part_len, int parts) {
    __shared__ uint32_t hist[COARSE];
    __shared__ u64 sums[P_THREADS / 64], found[2];
    __shared__ int counts[P_THREADS / 64];
    __shared__ u64 best[P_THREADS / 64];
    const int p = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    const Row<T> r(a, row);
    const Settings set(a, row);
    const Work w(a.ws, row, parts);
    const int p0 = p * part_len, p1 = min(p0 + part_len, r.n);
    const bool few = set.few && !set.greedy;
    if (few)
        hist[t] = 0;
    else
        for (int i = p * P_THREADS + t; i < BINS; i += parts * P_THREADS) w.hist[i] = 0;
    float mine = -INFINITY;                  // this thread's largest, and where it stands first
    int first = 0;
    for (int q = p0; q < p1; q += ROUND) {
        f32x4 y[4];
        r.round(q, y);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (y[d][e] > mine) mine = y[d][e], first = r.at(q, d) + e;
    }
    u64 b = (u64)key_of(mine) << 32 | (uint32_t)~first;                // (of equal keys the lower index)
    for (int o = 32; o; o >>= 1) b = max(b, (u64)__shfl_xor(b, o));
    if ((t & 63) == 0) best[t >> 6] = b;
    __syncthreads();
    for (int i = 0; i < P_THREADS / 64; ++i) b = max(b, best[i]);
    const uint32_t kmax = (uint32_t)(b >> 32);
    int held = 0;
    if (few && kmax) {
        const Bins bins(value_of(kmax), set.temp);
        const uint32_t own = bins(mine);
        if (own < BINS) atomicAdd(&hist[own / (BINS / COARSE)], 1u);
        __syncthreads();
        u64 before;
        uint32_t bin;
        const u64 v[1] = {hist[t]};
        // where fewer threads than top_k are in range, the last bin: all that can have a weight
        scan_bins<1, P_THREADS>(v, sums, found, [&](u64) { return (u64)set.top_k; }, &bin, &before);
        held = compact(r, p0, p1, bins, 0, min(bin * (BINS / COARSE) + BINS / COARSE - 1, (uint32_t)BINS - 1), w.list + (size_t)p * P_CAP, counts, [](float) {});
    }
    if (t == 0) w.part[p].kmax = kmax, w.part[p].first = ~(uint32_t)b, w.part[p].held = held;
}

template <typename T>
__global__ __launch_bounds__(P_THREADS) void sample_hist_k(SampleArgs a, PowerTable powers, int part_len, int parts) {
    __shared__ u64 hist[BINS], sums[P_THREADS / 64];
    __shared__ double table[32];
    const int p = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    const Settings set(a, row);
    if (set.greedy || set.few) return;
    const Row<T> r(a, row);
    const Work w(a.ws, row, parts);
    const uint32_t kmax = row_max(w, parts);
    if (kmax == 0) return;
    if (t < 32) table[t] = powers.t[t];
    for (int i = t; i < BINS; i += P_THREADS) hist[i] = 0;
    __syncthreads();
    const Bins bins(value_of(kmax), set.temp);
    const Weigher weigh = weigher(value_of(kmax), set.temp, table);
    const bool cuts = set.top_k || set.top_p < 1;
    u64 sum = 0;
    for (int q = p * part_len; q < min((p + 1) * part_len, r.n); q += ROUND) {
        f32x4 y[4];
        r.round(q, y);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll 1
            for (int e = 0; e < 4; ++e) {
                const float z = e == 0 ? y[d][0] : e == 1 ? y[d][1] : e == 2 ? y[d][2] : y[d][3];
                const uint32_t b = bins(z);
                if (b >= BINS) continue;
                const u64 x = set.top_k ? 1 : weigh.of(z);
                if (cuts) atomicAdd(&hist[b], x);
                else sum += x >= set.wmin ? x : 0;
            }
    }
    if (cuts) {
        __syncthreads();
        for (int i = t; i < BINS; i += P_THREADS)
            if (const u64 x = hist[i]) atomicAdd(&w.hist[i], x);
    } else {
        sum = wave_sum(sum);
        if ((t & 63) == 0) sums[t >> 6] = sum;
        __syncthreads();
        if (t == 0) w.part[p].sum = sums[0] + sums[1] + sums[2] + sums[3];
    }
}

template <typename T>
__global__ __launch_bounds__(P_THREADS) void sample_gather_k(SampleArgs a, PowerTable powers, int part_len, int parts) {
    __shared__ double table[32];
    __shared__ u64 sums[P_THREADS / 64], found[2];
    __shared__ int counts[P_THREADS / 64];
    const int p = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    const Settings set(a, row);
    if (set.greedy || set.few || !(set.top_k || set.top_p < 1)) return;
    const Row<T> r(a, row);
    const Work w(a.ws, row, parts);
    const uint32_t kmax = row_max(w, parts);
    if (kmax == 0) return;
    if (t < 32) table[t] = powers.t[t];
    constexpr int PER = BINS / P_THREADS;
    u64 v[PER], before;
    uint32_t bin;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = w.hist[t * PER + i];
    scan_bins<PER, P_THREADS>(v, sums, found, [&](u64 sum) { return set.top_k ? (u64)set.top_k : share(set.top_p, sum); }, &bin, &before);
    const int p0 = p * part_len, p1 = min(p0 + part_len, r.n);
    const float mf = value_of(kmax);
    const Bins bins(mf, set.temp);
    const Weigher weigh = weigher(mf, set.temp, table);
    uint2 *list = w.list + (size_t)p * P_CAP;
    u64 sum = 0;
    const int held = compact(r, p0, p1, bins, set.top_k ? 0 : bin, bin, list, counts, [&](float z) {
        const u64 x = weigh.of(z);
        sum += x >= set.wmin ? x : 0;
    });
    sum = wave_sum(sum);
    if ((t & 63) == 0) sums[t >> 6] = sum;
    __syncthreads();
    if (t == 0) w.part[p].held = held, w.part[p].sum = sums[0] + sums[1] + sums[2] + sums[3];
}

struct Shared {
    u64 whist[BINS];
    uint32_t key[CAP], idx[CAP];             // the candidates, in the order of the indexes
    u64 weight[CAP];
    u64 wsum[WAVES], found[2];
    uint32_t wcount[WAVES];
    u64 lw[SHORT];                           // a short list in any order: weight, key, index
    uint32_t lkey[SHORT], lidx[SHORT];
    u64 before, need;
    uint32_t prefix, n;
    double table[32];
};

// What the cuts of one row are made from: the candidates in LDS, or all of a row.  Wave w has the stretch [i0, i1), in turns of 64.  (One code for both,
// and the kernel below has each step once, in a loop: a launch fetches its instructions anew.  Against a form that had all steps twice, of 71 KB against
// 22, 128 rows of 128256 took 28 us in place of 31, the call 87 in place of 91; rows whose logits are nearly all alike, which go to all of a row, took
// 730 us in place of 630.)
template <typename T>
struct Source {
    Shared &s;
    const Row<T> &r;
    const Weigher &weigh;
    bool list;
    int i0, i1;
    __device__ Source(Shared &s, const Row<T> &r, const Weigher &weigh, bool list, int n) : s(s), r(r), weigh(weigh), list(list) {
        const int seg = ((n + WAVES - 1) / WAVES + 63) & ~63, wave = threadIdx.x >> 6;
        i0 = min(wave * seg, n), i1 = min(i0 + seg, n);
    }
    __device__ uint32_t key(int i) const { return list ? s.key[i] : key_of((float)r.x[i]); }
    __device__ u64 weight(int i, uint32_t key) const { return list ? s.weight[i] : weigh.of_key(key); }
    __device__ int index(int i) const { return list ? (int)s.idx[i] : i; }
    template <typename F>
    __device__ void each(F f) const {        // f(key, index, weight()) of those that are not -infinity
#pragma unroll 1
        for (int i = i0 + (threadIdx.x & 63); i < i1; i += 64) {
            const uint32_t k = key(i);
            if (k) f(k, index(i), [&] { return weight(i, k); });
        }
    }
};

// The key at which the sum over the keys with in(), in falling order (of 1 each, or of the weights), reaches `need`: *tkey, and in *ties how many
// equal keys that takes.  0 < need <= the sum over all.  A short list is ranked by comparing all with all; a long one (many logits within T / 64 of each
// other) goes by the key's four bytes from the top.
template <typename Src, typename In>
__device__ void cut(Shared &s, const Src &src, bool weights, u64 need, In in, uint32_t *tkey, u64 *ties) {
    const int t = threadIdx.x;
    if (t == 0) s.n = 0;
    __syncthreads();
    src.each([&](uint32_t k, int i, auto weight) {
        if (in(k)) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < SHORT) s.lkey[at] = k, s.lidx[at] = i, s.lw[at] = weights ? weight() : 1;
        }
    });
    __syncthreads();
    const int n = s.n;
    if (n <= SHORT) {
        if (t < n) {
            const uint32_t key = s.lkey[t], idx = s.lidx[t];
            const u64 own = s.lw[t];
            u64 sum = 0;
            uint32_t same = 1;
#pragma unroll 8
            for (int j = 0; j < n; ++j) {
                const uint32_t kj = s.lkey[j], ij = s.lidx[j];
                const u64 wj = s.lw[j];
                const bool tie = (kj == key) & (ij < idx);
                sum += ((kj > key) | tie) ? wj : 0;
                same += tie;
            }
            if (sum < need && sum + own >= need) s.prefix = key, s.need = same;
        }
        __syncthreads();
        *tkey = s.prefix, *ties = s.need;
        __syncthreads();
        return;
    }
    uint32_t prefix = 0, mask = 0;
    u64 left = need, unit = 1;
#pragma unroll 1                             // (seldom run: small code, here and below; a launch fetches its instructions anew)
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) s.whist[t] = 0;
        if (t == 0) s.before = 1;
        __syncthreads();
        src.each([&](uint32_t k, int, auto weight) {
            if (((k ^ prefix) & mask) == 0 && in(k)) {
                const u64 w = weights ? weight() : 1;
                if (w) atomicAdd(&s.whist[k >> shift & 255], w);
            }
        });
        __syncthreads();
        if (t < 64) {                    // lane L: bytes 255 - 4 L .. 252 - 4 L, in falling order
            u64 own = 0;
#pragma unroll 1
            for (int e = 0; e < 4; ++e) own += s.whist[255 - 4 * t - e];
            u64 at = wave_scan(own) - own;
#pragma unroll 1
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
    if (weights) {                       // one of the equal keys knows their weight
        src.each([&](uint32_t k, int, auto weight) {
            if (k == prefix && in(k)) s.before = weight();
        });
        __syncthreads();
        unit = s.before;
        __syncthreads();
    }
    *tkey = prefix, *ties = (left + unit - 1) / unit;
}

struct Kept {                            // keys above tkey, and the first `ties` equal to it; 0: all.  Weights of wmin and more.
    uint32_t tkey;
    u64 ties, wt, wmin;
};

// The kept weights in the order of the indexes: each wave's sum over its stretch, then the wave whose stretch holds the target looks for it.
template <typename Src>
__device__ void pick(Shared &s, const Src &src, const Kept &k, float u, int32_t *token) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const bool tied = k.tkey && k.wt >= k.wmin;
    u64 above = 0, run = 0, seen = 0, total = 0, count = 0;
    uint32_t equal = 0;
    src.each([&](uint32_t x, int, auto weight) {
        if (x > k.tkey) {
            const u64 w = weight();
            above += w >= k.wmin ? w : 0;
        } else if (x == k.tkey && tied) ++equal;
    });
    above = wave_sum(above), equal = wave_sum(equal);
    if (lane == 0) s.wsum[wave] = above, s.wcount[wave] = equal;
    __syncthreads();
#pragma unroll 4
    for (int w = 0; w < WAVES; ++w) {
        if (w == wave) run = total, seen = count;
        total += s.wsum[w], count += s.wcount[w];
    }
    run += min(seen, k.ties) * k.wt;
    total += min(count, k.ties) * k.wt;
    const u64 target = target_of(u, total);
    if (run > target || target >= run + above + (min(seen + equal, k.ties) - min(seen, k.ties)) * k.wt) return;
    uint32_t next = src.i0 + lane < src.i1 ? src.key(src.i0 + lane) : 0;
#pragma unroll 1
    for (int i = src.i0; i < src.i1; i += 64) {
        const uint32_t x = next;
        next = i + 64 + lane < src.i1 ? src.key(i + 64 + lane) : 0;
        const bool eq = tied && x == k.tkey;
        u64 w = x > k.tkey ? src.weight(i + lane, x) : 0;
        w = w >= k.wmin ? w : 0;
        const unsigned long long eqs = __ballot(eq);
        if (eq) w = seen + __popcll(eqs & ((1ull << lane) - 1)) < k.ties ? k.wt : 0;
        const u64 incl = wave_scan(w), pos = run + incl - w;
        if (pos <= target && target < pos + w) *token = src.index(i + lane);
        run += __shfl(incl, 63), seen += __popcll(eqs);
        if (target < run) return;
    }
}

// The same in a part of a row that is known to hold the target: `run` is what is kept above the threshold in front of it, `seen` the keys equal to it.  Each
// thread has four, eight or sixteen consecutive logits; the one that finds the target among its own walks them.
template <typename T>
__device__ void pick_part(Shared &s, const Row<T> &r, const Weigher &weigh, int i0, int len, const Kept &k, u64 run, u64 seen, u64 target, int32_t *token) {
    const int t = threadIdx.x, wave = t >> 6, per = len / S_THREADS, first = i0 + t * per, end = min(i0 + len, r.n);
    const bool tied = k.tkey && k.wt >= k.wmin;
    u64 above = 0;
    uint32_t equal = 0;
    auto weight = [&](float y) {
        const u64 w = weigh.of(y);
        return key_of(y) > k.tkey && w >= k.wmin ? w : 0;
    };
#pragma unroll 1
    for (int i = first; i < first + per; i += 4) {
        const f32x4 y = r.four(min(i, end));
#pragma unroll
        for (int e = 0; e < 4; ++e) above += weight(y[e]), equal += tied && key_of(y[e]) == k.tkey;
    }
    const u64 sums = wave_scan(above);
    const uint32_t eqs = wave_scan(equal);
    if ((t & 63) == 63) s.wsum[wave] = sums, s.wcount[wave] = eqs;
    __syncthreads();
    for (int w = 0; w < wave; ++w) run += s.wsum[w], seen += s.wcount[w];
    run += sums - above, seen += eqs - equal;
    u64 at = run + min(seen, k.ties) * k.wt;
    if (at > target || target >= run + above + min(seen + equal, k.ties) * k.wt) return;
#pragma unroll 1
    for (int i = first; i < first + per; i += 4) {
        const f32x4 y = r.four(min(i, end));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            u64 w = weight(y[e]);
            if (tied && key_of(y[e]) == k.tkey) w = seen++ < k.ties ? k.wt : 0;
            if (at <= target && target < at + w) *token = i + e;
            at += w;
        }
    }
}

// All of it for a short list (in any order: s.lkey, s.lidx, s.lw), by comparing all with all.
__device__ inline void draw_short(Shared &s, int n, int top_k, float top_p, u64 wmin, float u, int32_t *token) {
    const int t = threadIdx.x;
    uint32_t idx = 0;
    u64 w = 0, sum = 0;
    int rank = 0;
    if (t < n) {
        const uint32_t key = s.lkey[t];
        idx = s.lidx[t], w = s.lw[t];
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
            const uint32_t kj = s.lkey[j], ij = s.lidx[j];
            const u64 wj = s.lw[j];
            const bool before = (kj > key) | ((kj == key) & (ij < idx));
            rank += before, sum += before ? wj : 0;
        }
        if (rank == top_k - 1) s.need = sum + w;                       // the sum of the first top_k
    }
    __syncthreads();
    const u64 need = top_p < 1 ? share(top_p, s.need) : s.need;
    const u64 kept = t < n && rank < top_k && sum < need && w >= wmin ? w : 0;
    if (t < n) s.lw[t] = kept;
    __syncthreads();
    if (!kept) return;
    u64 run = 0, total = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
        const u64 x = s.lw[j];
        const uint32_t ij = s.lidx[j];
        total += x, run += ij < idx ? x : 0;
    }
    const u64 target = target_of(u, total);
    if (run <= target && target < run + kept) *token = (int32_t)idx;
}

template <typename T>
__global__ __launch_bounds__(S_THREADS) void sample_draw_k(SampleArgs a, PowerTable powers, int part_len, int parts) {
    __shared__ Shared s;
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const Settings set(a, row);
    const Work w(a.ws, row, parts);
    const float u = a.u[row];
    int32_t *token = a.tokens + row;
    const uint32_t kmax = row_max(w, parts);
    if (kmax == 0) {                         // no token is allowed
        if (t == 0) *token = -1;
        return;
    }
    if (set.greedy) {                        // the first part that has the largest
        if (t == 0)
            for (int p = 0; p < parts; ++p)
                if (w.part[p].kmax == kmax) {
                    *token = (int32_t)w.part[p].first;
                    break;
                }
        return;
    }
    if (t < 32) s.table[t] = powers.t[t];
    const float mf = value_of(kmax);
    const Bins bins(mf, set.temp);
    const Weigher weigh = weigher(mf, set.temp, s.table);
    const Row<T> r(a, row);
    Kept k{0, 0, 0, set.wmin};
    __syncthreads();

    // all parts' candidates, if they fit; lane p of each wave knows part p (there are 64 at most)
    const bool cuts = set.top_k || set.top_p < 1;
    const int held = cuts && lane < parts ? (int)w.part[lane].held : 0, past = wave_scan(held), n = __shfl(past, 63);
    const bool fits = !__any(held > P_CAP) && n <= CAP;
    if (fits)
        for (int q = t >> 6; q < parts; q += WAVES) {
            const int to = __shfl(past - held, q), m = __shfl(held, q);
            for (int i = lane; i < m; i += 64) {
                const uint2 c = w.list[(size_t)q * P_CAP + i];
                s.key[to + i] = c.x, s.idx[to + i] = c.y;
                s.weight[to + i] = weigh.of_key(c.x);
            }
        }
    __syncthreads();

    // The bin that holds the cut.
    const Source<T> src(s, r, weigh, fits, fits ? n : r.n);
    u64 before = 0, need = 0, total = 0;
    uint32_t bin = 0, low = 0;
    bool weights = !set.top_k, counted = !set.few && fits;             // (few: of the candidates that there are)
#pragma unroll 1
    for (bool more = cuts; more;) {
        if (!counted) {
            s.whist[2 * t] = s.whist[2 * t + 1] = 0;
            __syncthreads();
            src.each([&](uint32_t x, int, auto weight) {
                const uint32_t at = bins.of_key(x);
                if (x <= k.tkey || at >= BINS) return;
                const u64 y = weights ? weight() : 1;
                if (y) atomicAdd(&s.whist[at], y);
            });
            if (t == 0 && k.tkey) {
                const u64 y = k.ties * k.wt;
                const uint32_t at = bins.of_key(k.tkey);
                if (y && at < BINS) atomicAdd(&s.whist[at], y);
            }
            __syncthreads();
        }
        const u64 v[2] = {counted ? w.hist[2 * t] : s.whist[2 * t], counted ? w.hist[2 * t + 1] : s.whist[2 * t + 1]};
        total = scan_bins<2, S_THREADS>(v, s.wsum, s.found, [&](u64 sum) { return need = weights ? share(set.top_p, sum) : (u64)set.top_k; }, &bin, &before);
        if (set.few && fits && !weights) {
            if (t == 0) s.n = 0;
            __syncthreads();
            for (int i = t; i < n; i += S_THREADS)
                if (bins.of_key(s.key[i]) <= bin) {
                    const uint32_t at = atomicAdd(&s.n, 1u);
                    if (at < SHORT) s.lkey[at] = s.key[i], s.lidx[at] = s.idx[i], s.lw[at] = s.weight[i];
                }
            __syncthreads();
            const int m = s.n;
            if (m <= SHORT) return draw_short(s, m, min(set.top_k, m), set.top_p, set.wmin, u, token);
            __syncthreads();
        }
        if (weights || need <= total) {      // (a top_k beyond all that has a weight cuts nothing)
            cut(s, src, weights, need - before, [&](uint32_t x) { return x >= low && bins.of_key(x) == bin; }, &k.tkey, &k.ties);
            k.wt = weigh.of_key(k.tkey);
        }
        more = !weights && set.top_p < 1;    // then top_p among what top_k left
        weights = true, counted = false, low = k.tkey;
    }
    if (set.top_k || !fits) return pick(s, src, k, u, token);

    // The parts' sums are known but for what of the lists is kept: the part that holds the target, then the token in it.
    const bool tied = k.tkey && k.wt >= k.wmin;
    if (t < 64) s.lw[t] = t < parts ? w.part[t].sum : 0, s.lidx[t] = 0;
    __syncthreads();
    for (int i = t; cuts && i < n; i += S_THREADS) {
        const uint32_t key = s.key[i], at = s.idx[i] / (uint32_t)part_len;
        const u64 x = s.weight[i];
        if (key > k.tkey && x >= k.wmin) atomicAdd(&s.lw[at], x);
        if (tied && key == k.tkey) atomicAdd(&s.lidx[at], 1u);
    }
    __syncthreads();
    const u64 sum = s.lw[lane], sums = wave_scan(sum), front = sums - sum;
    const uint32_t eq = s.lidx[lane], eqs = wave_scan(eq);
    const u64 run = front + min((u64)(eqs - eq), k.ties) * k.wt, end = sums + min((u64)eqs, k.ties) * k.wt;
    const u64 target = target_of(u, __shfl(end, 63));
    const int part = __builtin_ctzll(__ballot(run <= target && target < end));
    pick_part(s, r, weigh, part * part_len, part_len, k, __shfl(front, part), (u64)__shfl(eqs - eq, part), target, token);
}

constexpr int MAX_ROWS = 2048;               // of a launch

// Parts of one round while that makes at most 2048 workgroups, of up to four rounds beyond: fewer of them join their bins.
static int part_rounds(int rows, int n_vocab) {
    const int64_t blocks = (int64_t)rows * ((n_vocab + ROUND - 1) / ROUND);
    return blocks <= 2048 ? 1 : blocks <= 4096 ? 2 : 4;
}
static int part_count(int rows, int n_vocab) {
    const int len = ROUND * part_rounds(rows, n_vocab);
    return (n_vocab + len - 1) / len;
}

size_t sample_workspace(int rows, int n_vocab) { return min(rows, MAX_ROWS) * Work::row_bytes(part_count(rows, n_vocab)); }

template <typename T>
static hipError_t sample_launch(const SampleArgs &a, hipStream_t st) {
    static const PowerTable powers = [] {
        PowerTable p;
        for (int j = 0; j < 32; ++j) p.t[j] = ldexp(exp2(j / 32.0), S_BITS);
        return p;
    }();
    const int parts = part_count(a.rows, a.n_vocab), len = ROUND * part_rounds(a.rows, a.n_vocab);
    // what the host knows of all rows
    const bool greedy = !a.temperature_p && !(a.temperature > 0), few = !a.top_k_p && a.top_k > 0 && a.top_k < a.n_vocab && a.top_k <= FEW;
    const bool cuts = a.top_k_p || a.top_p_p || (a.top_k > 0 && a.top_k < a.n_vocab) || a.top_p < 1;
    for (int row = 0; row < a.rows; row += MAX_ROWS) {                 // (one after the other on the stream, in the same workspace)
        SampleArgs b = a;
        const int rows = b.rows = min(a.rows - row, MAX_ROWS);
        b.logits = (const T *)a.logits + row * a.ld, b.u += row, b.tokens += row;
        if (b.temperature_p) b.temperature_p += row;
        if (b.top_k_p) b.top_k_p += row;
        if (b.top_p_p) b.top_p_p += row;
        if (b.min_p_p) b.min_p_p += row;
        const dim3 g(parts, rows);
        sample_scan_k<T><<<g, P_THREADS, 0, st>>>(b, len, parts);
        if (!greedy && !few) {
            sample_hist_k<T><<<g, P_THREADS, 0, st>>>(b, powers, len, parts);
            if (cuts) sample_gather_k<T><<<g, P_THREADS, 0, st>>>(b, powers, len, parts);
        }
        sample_draw_k<T><<<rows, S_THREADS, 0, st>>>(b, powers, len, parts);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t sample(const SampleArgs &a, int type, hipStream_t st) {
    return type == FL_TYPE_F32 ? sample_launch<float>(a, st) : type == FL_TYPE_F16 ? sample_launch<h16>(a, st) : sample_launch<b16>(a, st);
}

}  // namespace fl
