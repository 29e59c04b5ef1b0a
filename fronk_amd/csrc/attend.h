// attend.h - what attention over many rows is built from (prompt.hip, tree.hip).
//
// Matrix-core fragments of 32 x 32 (v_mfma_f32_32x32x16, v_mfma_f32_32x32x2; i =
// lane % 32, h = lane / 32): A holds row i, B column i; the result holds column i, in
// register r its row 8 (r / 4) + 4 h + r % 4.
#pragma once
#include <math.h>

#include "dense.h"

namespace {

// Four wavefronts of 32 rows.
constexpr uint32_t kWaves = 4, R = 32 * kWaves;

typedef float float16v __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));

template <typename T> struct Kind;
template <> struct Kind<__bf16> {
  typedef bf16x8 frag;
};
template <> struct Kind<_Float16> {
  typedef half8v frag;
};
template <> struct Kind<float> {
  typedef float4v frag;
};

__device__ __forceinline__ float16v mma32(bf16x8 a, bf16x8 b, float16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float16v mma32(half8v a, half8v b, float16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float16v mma32(float4v a, float4v b, float16v c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

typedef __attribute__((address_space(3))) char lds_char;

// 64 lanes' 16 bytes to consecutive places of LDS from `at` on. Of the counter of
// loads in flight that this raises the compiler knows nothing: whoever reads the
// places waits for it, and then for the other wavefronts.
__device__ __forceinline__ void to_lds(const char* base, uint32_t offset, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// N operands of READS reads each, one matrix instruction each: a few ahead.
template <int N, int READS> __device__ __forceinline__ void schedule() {
  constexpr int kAhead = 4;
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead * READS, 0);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (n + kAhead < N) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// Four of a row's sums, by its sum of weights; a row that sees nothing has zeros.
template <typename T> __device__ __forceinline__ void put4(T* p, float4v x, float sum, bool wide) {
  typedef T vec __attribute__((ext_vector_type(4)));
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  vec y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(x[e] * f);
  if (wide) {
    *reinterpret_cast<vec*>(p) = y;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = y[e];
  }
}

// Four dims of a row from its stretches, in their order: `part` its place in the first.
template <int D>
__device__ __forceinline__ float4v join(const float* part_o, const float* part_ml, size_t part, uint32_t splits, uint32_t d, float* sum) {
  float top = -INFINITY, total = 0;
  for (uint32_t s = 0; s < splits; ++s) top = fmaxf(top, part_ml[(part + (size_t)s * R) * 2]);
  float4v x = {0, 0, 0, 0};
  for (uint32_t s = 0; s < splits; ++s, part += R) {
    const float shift = part_ml[part * 2];
    if (shift == -INFINITY) continue;   // nothing seen there, and no sums written
    const float w = __builtin_amdgcn_exp2f(shift - top);
    total += w * part_ml[part * 2 + 1];
    x += w * *reinterpret_cast<const float4v*>(part_o + part * D + d);
  }
  *sum = total;
  return x;
}

}  // namespace
