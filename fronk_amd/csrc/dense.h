// dense.h - what the dense operators' sources share: the engine's side of a
// call, element types, and the matrix-core fragments they are built from.
//
// Matrix-core fragments (v_mfma_f32_16x16x32, 64 lanes; i = lane % 16,
// j = lane / 16): A holds row i, B column i, at eight values of the summed
// index each (which eight is free, as long as A and B agree); the result holds
// column i at rows 4j .. 4j+3.
#pragma once
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "devices.h"
#include "fronk_hip.h"

namespace fronk {

// Makes the open engine's device current and resolves `stream`; FR_HIP_STATE
// without an open engine.
__attribute__((visibility("hidden"))) int enter(void* stream, hipStream_t* out);

}  // namespace fronk

namespace {

constexpr uint32_t kUnits = 256;   // an MI355X's compute units, of four SIMDs each

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

inline size_t elem_size(unsigned type) { return type == FR_HIP_F32 ? 4 : 2; }

// N consecutive elements as floats; `wide`: the address is aligned to the
// smaller of 16 bytes and the N elements.
template <int N, typename T>
__device__ __forceinline__ void load_row(const T* p, bool wide, float (&out)[N]) {
  if (wide) {
    constexpr int kBytes = N * (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kBytes > 16 ? 16 / sizeof(T) : N)));
    constexpr int kEach = kBytes > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += kEach) {
      const vec v = *reinterpret_cast<const vec*>(p + i);
#pragma unroll
      for (int e = 0; e < kEach; ++e) out[i + e] = (float)v[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)p[i];
  }
}

// Sums over lanes: x + the value of the lane whose index differs in bit 4
// (resp. 5), by the gfx950 row swaps.
__device__ __forceinline__ float add_xor16(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float add_xor32(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float max_xor16(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float max_xor32(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
// Within each row of 16 lanes: the lane N places on (cyclic).
template <int N> __device__ __forceinline__ float row_rotate(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, false));
}

__device__ __forceinline__ float4v mma(bf16x8 a, bf16x8 b, float4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float4v mma(half8v a, half8v b, float4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bf16x2 to_bf16(float a, float b) {
  const float2v v = {a, b};
  return __builtin_convertvector(v, bf16x2);
}

// Lets a kernel have `bytes` of dynamic LDS on the engine's device. `done` is the
// kernel's own.
template <typename Kernel> int allow_lds(Kernel kernel, size_t bytes, fronk::Devices* done) {
  return fronk::once_a_device(done, fr_hip_device(), [&] {
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  });
}

#define FRONK_CK(x) do { if ((x) != hipSuccess) return FR_HIP_IO; } while (0)

}  // namespace
