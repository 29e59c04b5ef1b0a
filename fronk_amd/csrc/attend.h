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

// What all lanes have alike, so that the compiler keeps it, and addresses made of it, once.
__device__ __forceinline__ int32_t same(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }

typedef __attribute__((address_space(3))) char lds_char;

// 64 lanes' 16 bytes to consecutive places of LDS from `at` on. Of the counter of
// loads in flight that this raises the compiler knows nothing: whoever reads the
// places waits for it, and then for the other wavefronts.
__device__ __forceinline__ void to_lds(const char* base, uint32_t offset, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(base) : "memory", "m0");
}
// The largest of a lane's scores (NaN is none), in four chains.
template <int N> __device__ __forceinline__ float largest(const float16v (&st)[N]) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) m[r % 4] = fmaxf(m[r % 4], st[t][r]);
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// Waits for this wavefront's loads but the last N, and then for all wavefronts'.
template <int N> __device__ __forceinline__ void loads_done() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// N operands of READS reads each, for EACH matrix instructions: kAhead ahead.
template <int N, int READS, int kAhead, int EACH = 1> __device__ __forceinline__ void schedule() {
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead * READS, 0);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
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

// A stretch's sums, for another kernel: not kept in this die's L2, which would have to be
// written out when the kernel ends.
__device__ __forceinline__ void part_store(float* to, float4v x) { __builtin_nontemporal_store(x, reinterpret_cast<float4v*>(to)); }
// Four dims of a row from its stretches, joined in their order; `part` is the row's
// place in the first, of `block_rows`. Many rows: D / 4 lanes each.
template <int D>
__device__ __forceinline__ float4v join_few(const float* part_o, const float* part_ml, size_t part, uint32_t splits, uint32_t block_rows, float* sum) {
  constexpr uint32_t kFirst = 4;
  const uint32_t d = threadIdx.x % (D / 4) * 4;
  auto value = [&](uint32_t s) { return *reinterpret_cast<const float4v*>(part_o + (part + (size_t)s * block_rows) * D + d); };
  auto of = [&](uint32_t s) { return *reinterpret_cast<const float2v*>(part_ml + (part + (size_t)s * block_rows) * 2); };
  // The first ones are under way at once.
  float4v y[kFirst];
  float2v ml[kFirst];
#pragma unroll
  for (uint32_t s = 0; s < kFirst; ++s) y[s] = value(min(s, splits - 1)), ml[s] = of(min(s, splits - 1));
  float top = -INFINITY, total = 0;
#pragma unroll
  for (uint32_t s = 0; s < kFirst; ++s) top = fmaxf(top, ml[s][0]);
#pragma unroll 8
  for (uint32_t s = kFirst; s < splits; ++s) top = fmaxf(top, of(s)[0]);
  float4v x = {0, 0, 0, 0};
  auto add = [&](float2v ml, float4v y) {
    const float w = __builtin_amdgcn_exp2f(ml[0] - top);
    if (ml[0] != -INFINITY) total += w * ml[1], x += w * y;   // (else nothing is seen there, and y was not written)
  };
#pragma unroll
  for (uint32_t s = 0; s < kFirst; ++s)
    if (s < splits) add(ml[s], y[s]);
#pragma unroll 8
  for (uint32_t s = kFirst; s < splits; ++s) add(of(s), value(s));
  *sum = total;
  return x;
}
// Up to 256 stretches of few rows: a workgroup of 256 a row; the first D / 4 threads have the result.
template <int D>
__device__ __forceinline__ float4v join_many(const float* part_o, const float* part_ml, size_t part, uint32_t splits, uint32_t block_rows, float* sum) {
  constexpr uint32_t L = D / 4, G = 256 / L, kFirst = 16;
  __shared__ float weight[256], red[2][4];
  __shared__ float4v parts[G][L];
  const uint32_t s = threadIdx.x, c = s % L, g = s / L;
  const float m = s < splits ? part_ml[(part + (size_t)s * block_rows) * 2] : -INFINITY;
  const float l = s < splits ? part_ml[(part + (size_t)s * block_rows) * 2 + 1] : 0.f;
  // The first values are under way while their weights are found.
  float4v y[kFirst];
#pragma unroll
  for (uint32_t j = 0; j < kFirst; ++j)
    y[j] = *reinterpret_cast<const float4v*>(part_o + (part + (size_t)min(g + j * G, splits - 1) * block_rows) * D + c * 4);
  float top = m;
  for (int o = 1; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
  if ((s & 63) == 0) red[0][s >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const bool seen = m != -INFINITY;
  const float w = seen ? __builtin_amdgcn_exp2f(m - top) : -1.f;
  weight[s] = w;
  float total = seen ? w * l : 0.f;
  for (int o = 1; o < 64; o *= 2) total += __shfl_xor(total, o);
  if ((s & 63) == 0) red[1][s >> 6] = total;
  __syncthreads();
  *sum = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  float4v x = {0, 0, 0, 0};
  auto add = [&](uint32_t k, float4v y) {
    const float f = weight[k];
    if (!(f < 0.f)) x += f * y;   // (else nothing is seen there, or it is none, and y was not written)
  };
#pragma unroll
  for (uint32_t j = 0; j < kFirst; ++j)
    if (g + j * G < splits) add(g + j * G, y[j]);
#pragma unroll 8
  for (uint32_t k = g + kFirst * G; k < splits; k += G)
    add(k, *reinterpret_cast<const float4v*>(part_o + (part + (size_t)k * block_rows) * D + c * 4));
  parts[g][c] = x;
  __syncthreads();
  for (uint32_t k = 1; k < G; ++k) x += parts[k][c];   // (by all, for the first group)
  return x;
}
// Rows below which each has a workgroup (join_many). Whole calls of trees (bf16, dim 128), us, by a
// workgroup each and by D / 4 lanes each: 512 rows of 64 stretches 36 and 42, 1024 of 32 48 and
// 53, 2048 of 16 49 and 48, 4096 of eight 54 and 47, 8192 of four 99 and 79.
constexpr uint64_t kJoinRows = 2048;

}  // namespace
