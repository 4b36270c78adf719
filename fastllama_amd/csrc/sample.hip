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

template <typename T>
struct Row {
    const T *x;
    int n;
    __device__ uint32_t key(int i) const { return key_of((float)x[i]); }
};

struct Shared {
    u64 hist[256];
    u64 wave[S_THREADS / 64], wave2[S_THREADS / 64];
    uint32_t kmax, prefix;
    u64 need;
    int found;
};

// The key at which the sum over the keys in falling order (of 1 each, or of the weights) reaches `need`, by the key's four bytes from the top:
// *tkey, and in *need what is left to take from the keys equal to it.  0 < need <= the sum over all.
template <bool WEIGHTS, typename T>
__device__ void select(Shared &s, const Row<T> &r, uint32_t kmax, double max, double c, uint32_t *tkey, u64 *need) {
    uint32_t prefix = 0, mask = 0;
    u64 left = *need;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) s.hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < r.n; i += S_THREADS) {
            const uint32_t k = r.key(i);
            if (k && ((k ^ prefix) & mask) == 0) {
                const u64 w = WEIGHTS ? weight_of(k, kmax, max, c) : 1;
                if (w) atomicAdd(&s.hist[k >> shift & 255], w);
            }
        }
        __syncthreads();
        if (threadIdx.x < 64) {          // lane L: bins 255 - 4 L .. 252 - 4 L, in falling order
            u64 own = 0;
            for (int t = 0; t < 4; ++t) own += s.hist[255 - 4 * threadIdx.x - t];
            u64 incl = own;
            for (int o = 1; o < 64; o <<= 1) {
                const u64 up = __shfl_up(incl, o);
                if ((int)threadIdx.x >= o) incl += up;
            }
            u64 before = incl - own;
            if (before < left && incl >= left)
                for (int t = 0; t < 4; ++t) {
                    const int bin = 255 - 4 * threadIdx.x - t;
                    const u64 h = s.hist[bin];
                    if (before < left && before + h >= left) s.prefix = prefix | (uint32_t)bin << shift, s.need = left - before;
                    before += h;
                }
        }
        __syncthreads();
        prefix = s.prefix, left = s.need, mask |= 255u << shift;
        __syncthreads();
    }
    *tkey = prefix, *need = left;
}

template <typename T>
__global__ __launch_bounds__(S_THREADS) void sample_k(SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const Row<T> r{(const T *)a.logits + row * a.ld, a.n_vocab};
    const float temp = a.temperature_p ? a.temperature_p[row] : a.temperature, top_p = a.top_p_p ? a.top_p_p[row] : a.top_p;
    const float min_p = a.min_p_p ? a.min_p_p[row] : a.min_p, u = a.u[row];
    const int top_k = a.top_k_p ? a.top_k_p[row] : a.top_k;

    if (t == 0) s.kmax = 0;
    __syncthreads();
    uint32_t kmax = 0;
    for (int i = t; i < r.n; i += S_THREADS) kmax = max(kmax, r.key(i));
    for (int o = 32; o; o >>= 1) kmax = max(kmax, (uint32_t)__shfl_xor((int)kmax, o));
    if (lane == 0) atomicMax(&s.kmax, kmax);
    __syncthreads();
    kmax = s.kmax;
    if (kmax == 0) {                     // no token is allowed
        if (t == 0) a.tokens[row] = -1;
        return;
    }
    const bool greedy = !(temp > 0);
    const double mx = value_of(kmax), c = greedy ? 0 : 1.4426950408889634074 / (double)temp;

    uint32_t tkey = 1;                   // keep all
    u64 ties = ~0ull;
    if (greedy) tkey = kmax, ties = 1;
    else {
        int allowed = 0;                 // tokens that are not at -infinity
        if (top_k > 0) {
            for (int i = t; i < r.n; i += S_THREADS) allowed += r.key(i) != 0;
            allowed = wave_sum(allowed);
            if (lane == 0) s.wave[wave] = allowed;
            __syncthreads();
            allowed = 0;
            for (int w = 0; w < S_THREADS / 64; ++w) allowed += (int)s.wave[w];
            __syncthreads();
            if (top_k < allowed) {
                ties = top_k;
                select<false>(s, r, kmax, mx, c, &tkey, &ties);
            }
        }
        if (top_p < 1) {
            u64 sum = 0;
            for (int i = t; i < r.n; i += S_THREADS) {
                const uint32_t k = r.key(i);
                if (k > tkey || (k == tkey && ties == ~0ull)) sum += weight_of(k, kmax, mx, c);
            }
            sum = wave_sum(sum);
            if (lane == 0) s.wave[wave] = sum;
            __syncthreads();
            sum = 0;
            for (int w = 0; w < S_THREADS / 64; ++w) sum += s.wave[w];
            __syncthreads();
            if (ties != ~0ull) sum += ties * weight_of(tkey, kmax, mx, c);
            u64 need = top_p > 0 ? (u64)ceil((double)top_p * (double)sum) : 1;
            need = min(max(need, (u64)1), sum);
            select<true>(s, r, kmax, mx, c, &tkey, &need);
            const u64 w = weight_of(tkey, kmax, mx, c);
            ties = (need + w - 1) / w;
        }
    }
    const u64 wmin = min_p > 0 && !greedy ? (u64)ceil(fmin((double)min_p, 1.0) * (double)(1ull << S_BITS)) : 0;
    const u64 wt = weight_of(tkey, kmax, mx, c);

    // each thread sums a stretch of consecutive tokens: the weights above the threshold, and how many equal it
    const int per = (r.n + S_THREADS - 1) / S_THREADS, i0 = min(t * per, r.n), i1 = min(i0 + per, r.n);
    u64 above = 0, equal = 0;
    for (int i = i0; i < i1; ++i) {
        const uint32_t k = r.key(i);
        if (k == 0) continue;
        if (k > tkey) {
            const u64 w = weight_of(k, kmax, mx, c);
            above += w >= wmin ? w : 0;
        } else if (k == tkey && wt >= wmin) ++equal;
    }
    u64 ia = above, ie = equal;          // running sums over the threads
    for (int o = 1; o < 64; o <<= 1) {
        const u64 pa = __shfl_up(ia, o), pe = __shfl_up(ie, o);
        if (lane >= o) ia += pa, ie += pe;
    }
    if (lane == 63) s.wave[wave] = ia, s.wave2[wave] = ie;
    if (t == 0) s.found = 0;
    __syncthreads();
    u64 sa = 0, se = 0, ba = 0, be = 0;
    for (int w = 0; w < S_THREADS / 64; ++w) {
        if (w == wave) ba = sa, be = se;
        sa += s.wave[w], se += s.wave2[w];
    }
    const u64 total = sa + min(se, ties) * wt;
    ba += ia - above, be += ie - equal;
    const double uc = u > 0 ? (u < 1 ? (double)u : 1.0) : 0.0;
    const u64 target = min((u64)floor(uc * (double)total), total - 1);
    u64 run = ba + min(be, ties) * wt;
    const u64 end = ba + above + min(be + equal, ties) * wt;
    if (run <= target && target < end) {
        for (int i = i0; i < i1; ++i) {
            const uint32_t k = r.key(i);
            if (k == 0) continue;
            u64 w = 0;
            if (k > tkey) {
                w = weight_of(k, kmax, mx, c);
                w = w >= wmin ? w : 0;
            } else if (k == tkey && wt >= wmin) w = be++ < ties ? wt : 0;
            if (target < run + w) {
                a.tokens[row] = i;
                break;
            }
            run += w;
        }
    }
}

hipError_t sample(const SampleArgs &a, int type, hipStream_t st) {
    if (type == FL_TYPE_F32) sample_k<float><<<a.rows, S_THREADS, 0, st>>>(a);
    else if (type == FL_TYPE_F16) sample_k<h16><<<a.rows, S_THREADS, 0, st>>>(a);
    else sample_k<b16><<<a.rows, S_THREADS, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace fl
