// What the attention kernels have in common: what a query sees, the matrix operands' types, and reductions over the lanes that hold a
// column of scores.
#pragma once
#include "common.h"

#define NEG_INF (-__builtin_inff())

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// What a query at position p sees, and how scores become weights.
struct Sight {
  int window;  // > 0: keys p - window + 1 .. p; 0: every key up to p
  int keep;    // with a window: the sequence's first `keep` keys stay visible behind it
  int chunk;   // > 0: keys of the query's own chunk only, chunks of this many positions counted from 0 (without a window)
  float cap;   // > 0: a score s counts as cap tanh(s / cap)
  int sink;    // 1: the denominator has one more score, which has no value
  const float* sinks;  // [H]: that score per query head (not scaled); null: 0 for all
  int wide;    // 1: the kernels of bfloat16 heads write their results in fp32 (for a consumer that takes differences of them)
};
// The result of a head's coordinate i, in the type of the heads or in fp32 (`Sight::wide`).
template <typename T>
__device__ __forceinline__ void put(T* out, size_t i, float v, int wide) {
  if (wide) reinterpret_cast<float*>(out)[i] = v;
  else out[i] = from_f32<T>(v);
}
__device__ __forceinline__ int first_in_window(const Sight& sight, int ctx) {
  if (sight.chunk > 0) return (ctx - 1) / sight.chunk * sight.chunk;
  return sight.window > 0 ? max(0, ctx - sight.window) : 0;
}
__device__ __forceinline__ float sink_score(int sink, const float* sinks, int head) { return sink && sinks ? sinks[head] : 0.f; }
static inline bool sight_ok(const Sight& s) {
  return s.window >= 0 && s.keep >= 0 && (s.keep == 0 || s.window > 0) && s.cap >= 0.f && (s.sink == 0 || s.sink == 1) &&
         (s.wide == 0 || s.wide == 1) && s.chunk >= 0 && (s.chunk == 0 || s.window == 0);
}
// tanh through the hardware's exponential and reciprocal: an absolute error of 1e-7, which is what a capped score
// (times the cap) of the bf16 kernels may carry.
__device__ __forceinline__ float quick_tanh(float x) {
  return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.8853900817779268f * x));
}

// Sums and maxima over the four lanes that share `lane % 16` (lane ^ 16, lane ^ 32) without a
// trip through LDS: v_permlane16_swap / v_permlane32_swap exchange rows of 16 lanes between
// two registers.  With both operands equal to x, the results hold (rows 0 0 2 2, rows 1 1 3 3)
// and (rows 0 1 0 1, rows 2 3 2 3) of x.
__device__ __forceinline__ float quad_rows_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_rows_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// max(a, b, c) as the one instruction it is; NaN operands lose, as with fmaxf.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// s_waitcnt that only constrains the vector-memory counter (vmcnt: bits 3:0 and 15:14)
#define PF_WAIT_VM(N) __builtin_amdgcn_s_waitcnt(((N) & 15) | (((N) >> 4) << 14) | (7 << 4) | (15 << 8))
