// kv.h - what the sources around the paged 8-bit cache share: where it lies, its
// codes as operands, and the checks of its sizes.
#pragma once
#include <limits.h>

#include "bounds.h"
#include "dense.h"

namespace {

struct Cache {
  uint8_t *k_codes, *v_codes, *k_exp, *v_exp;
  uint32_t pages, heads, page, dim;
};

__device__ __forceinline__ size_t exp_at(const Cache& C, uint32_t page, uint32_t head, uint32_t at) {
  return fronk::exp_at(C.heads, C.page, page, head, at);
}
__device__ __forceinline__ size_t v_at(const Cache& C, uint32_t page, uint32_t head, uint32_t at) {
  return fronk::v_at(C.heads, C.page, C.dim, page, head, at);
}

// 2^(e - 127) of an exponent byte; 255 (a vector with a non-finite value) is
// infinity, which makes NaN of its zero codes.
__device__ __forceinline__ float power(uint32_t e) { return __builtin_bit_cast(float, e << 23); }

// Eight e4m3 codes as an operand, exactly.
__device__ __forceinline__ bf16x8 codes8(uint32_t lo, uint32_t hi, bf16x8) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ half8v codes8(uint32_t lo, uint32_t hi, half8v) {
  const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ... and times a power of two.
__device__ __forceinline__ bf16x8 codes8(uint32_t lo, uint32_t hi, float power, bf16x8) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, true);
  return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x as `N` bf16 parts whose sum it is (up to 2^-8N of it).
template <int N> __device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&out)[N]) {
  float rest[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
  for (int p = 0; p < N; ++p)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const bf16x2 h = to_bf16(rest[e], rest[e + 1]);
      out[p][e] = h[0], out[p][e + 1] = h[1];
      if (p + 1 < N) rest[e] -= (float)h[0], rest[e + 1] -= (float)h[1];
    }
}

int check_cache(const fr_hip_kv_cache* c, unsigned type) {
  if (type > FR_HIP_BF16 || !c->pages || !c->heads || !c->page || !c->dim) return FR_HIP_INVALID;
  if (!c->k_codes || !c->v_codes || !c->k_exp || !c->v_exp) return FR_HIP_INVALID;
  if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes | (uintptr_t)c->k_exp | (uintptr_t)c->v_exp) % 16) return FR_HIP_INVALID;
  if ((c->dim != 64 && c->dim != 128 && c->dim != 256) || c->page % 16 || c->page > 4096) return FR_HIP_UNSUPPORTED;
  if ((uint64_t)c->pages * c->page > INT_MAX || c->heads > 1024) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

Cache cache_of(const fr_hip_kv_cache& c) {
  return Cache{c.k_codes, c.v_codes, c.k_exp, c.v_exp, c.pages, c.heads, c.page, c.dim};
}

bool rows_wide(unsigned type, const void* k, const void* v, int64_t a, int64_t b, int64_t c, int64_t d) {
  const int64_t n = 16 / (int64_t)elem_size(type);
  return ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && a % n == 0 && b % n == 0 && c % n == 0 && d % n == 0;
}

}  // namespace
