// serve_device.h -- device helpers of the serving operators (serve_kernels.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fl {

typedef _Float16 h16;
typedef __bf16 b16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Sequence b's rows [*first, *end) of `total` packed rows.  What the caller wrote into cu is cut to the rows that exist: no start makes a
// kernel leave the buffers.
__device__ inline void seq_rows(const int32_t *cu, int b, int total, int *first, int *end) {
    const int f = min(max(cu[b], 0), total);
    *first = f;
    *end = min(max(cu[b + 1], f), total);
}

// Eight consecutive elements: what a lane gives to one matrix step.
template <typename T>
struct Vec {
    typedef T x8 __attribute__((ext_vector_type(8)));
};

// A step of 16 (32 x 32 outputs) or 32 (16 x 16) along the summed axis: lane l holds the eight elements 8 (l / 32) + i, or 8 (l / 16) + i, of row
// l % 32, or l % 16, of either operand.  The f32 units take one element of each lane at a time; which element of the sum that is does not matter
// as long as both operands agree, so a lane's eight elements go through eight instructions and every type has the same operand layout.
__device__ inline f32x16 mfma32(Vec<h16>::x8 a, Vec<h16>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mfma32(Vec<b16>::x8 a, Vec<b16>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mfma32(Vec<float>::x8 a, Vec<float>::x8 b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

__device__ inline f32x4 mfma16(Vec<h16>::x8 a, Vec<h16>::x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x4 mfma16(Vec<b16>::x8 a, Vec<b16>::x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
template <int N>
__device__ inline f32x4 mfma16(float __attribute__((ext_vector_type(N))) a, float __attribute__((ext_vector_type(N))) b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < N; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

// The larger of a lane's value and that of the lane 32 away.
__device__ inline float max_halves(float x) {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
__device__ inline float sum_halves(float x) {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}

// What a part of a row's keys with the maximum m counts for beside the whole's, M.  A part without keys has m = -infinity and sums of 0, one whose scores
// are all no numbers has the sum NaN with it: that stays NaN whatever it is multiplied by.
__device__ inline float factor(float m, float M) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M); }

// Numerators of the softmax are 2^P_SHIFT as large in f16, whose smallest is 2^-24 (attn_prompt.hip).
template <typename T>
constexpr float P_SHIFT = 0.f;
template <>
inline constexpr float P_SHIFT<h16> = 7.f;

typedef __attribute__((address_space(3))) s16x4 *lds_s16x4;

template <typename T>
__device__ inline bool finite(T x) { return fabsf((float)x) < INFINITY; }

}  // namespace fl
