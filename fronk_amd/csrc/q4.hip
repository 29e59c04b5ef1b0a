// q4.hip - products with 4-bit weights and group scales (fr_hip_q4_product):
//     y[t][n] = sum_g scale[n][g] sum_{k in g} x[t][k] (code[n][k] - zero[n][g]) .
#include <limits.h>

#include <type_traits>

#include "dense.h"

namespace {

struct Q4Args {
  const void* x;
  const uint8_t* codes;
  const uint16_t* scales;
  const uint8_t* zeros;
  void* y;
  int64_t x_token, y_token;
  uint32_t tokens, rows, cols, groups;
  bool bf16_scales, wide;   // wide: x rows are of whole 16 bytes
};

// The matrix cores' operand type: fp16 activations meet fp16 codes, all others
// bf16 ones (codes 0..15 and zero points are exact in both). fp32 activations
// are the sum of three bf16 parts (8 + 8 + 8 bits), each a row of its own.
template <typename T> struct Operand {
  typedef bf16x8 frag;
  typedef bf16x2 pair;
  typedef __bf16 one;
  static constexpr int kParts = std::is_same<T, float>::value ? 3 : 1;
};
template <> struct Operand<_Float16> {
  typedef half8v frag;
  typedef half2v pair;
  typedef _Float16 one;
  static constexpr int kParts = 1;
};

// Two bytes of w (the low or the high half) as numbers: a byte below 16 read
// as e4m3 is its value * 2^-9 exactly.
template <bool HIGH> __device__ __forceinline__ bf16x2 two(uint32_t w, bf16x2) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.f, HIGH);
}
template <bool HIGH> __device__ __forceinline__ half2v two(uint32_t w, half2v) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 512.f, HIGH);
}

// Eight codes in their order.
template <typename O> __device__ __forceinline__ typename O::frag decode(uint32_t w) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  const uint32_t lo = __builtin_amdgcn_perm(odd, even, 0x05010400u), hi = __builtin_amdgcn_perm(odd, even, 0x07030602u);
  const typename O::pair z = {};
  const auto a = two<false>(lo, z), b = two<true>(lo, z), c = two<false>(hi, z), d = two<true>(hi, z);
  return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Lanes 16s + i exchange four words so that word s of lane 16j + i becomes
// word j of lane 16s + i: a transpose over the four rows of 16 lanes.
__device__ __forceinline__ void transpose4(uint32_t (&d)[4]) {
  auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
  auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  auto e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  d[0] = c[0], d[1] = c[1], d[2] = e[0], d[3] = e[1];
}

// Eight activations of one lane as an operand; part: which bf16 part of them.
__device__ __forceinline__ bf16x8 operand(const float (&x)[8], int part, bf16x8) {
  bf16x8 out;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const bf16x2 p0 = to_bf16(x[e], x[e + 1]);
    const float a = x[e] - (float)p0[0], b = x[e + 1] - (float)p0[1];
    const bf16x2 p1 = to_bf16(a, b);
    const bf16x2 p2 = to_bf16(a - (float)p1[0], b - (float)p1[1]);
    const bf16x2 p = part == 0 ? p0 : part == 1 ? p1 : p2;
    out[e] = p[0], out[e + 1] = p[1];
  }
  return out;
}

__device__ __forceinline__ float scale_of(uint16_t bits, bool bf16) {
  if (bf16) return __builtin_bit_cast(float, (uint32_t)bits << 16);
  return (float)__builtin_bit_cast(_Float16, bits);
}

// One workgroup: 16 NT rows of W by MT * 16 / parts tokens; its wavefronts take
// every (waves)th block of 128 columns and add up through LDS at the end.
//
// x is the A operand (tokens as rows), 16 rows of W the B operand, so that a
// lane's four results belong to its own weight row: one scale a lane and group.
// A lane reads 16 bytes of its row (32 codes). With groups of 128 a block is
// one group and step s takes columns 32 j + 8 s ..; smaller groups must not mix
// in one instruction, so the words are transposed over the lane rows and step s
// takes columns 32 s + 8 j .. . The zero point is an operand too, the constant
// row -zero, which keeps code - zero exact.
template <typename T, int MT, int NT, int G>
__global__ __launch_bounds__(512) void q4_rows(Q4Args A) {
  typedef Operand<T> O;
  typedef typename O::frag frag;
  constexpr int P = O::kParts, SPG = G / 32, GPB = 128 / G, TB = MT * 16 / P;
  extern __shared__ float sums[];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const uint32_t i = lane & 15, j = lane >> 4;
  const uint32_t n0 = blockIdx.x * 16 * NT, t0 = blockIdx.y * TB;
  const uint32_t tb = A.tokens - t0 < (uint32_t)TB ? A.tokens - t0 : (uint32_t)TB;

  const uint8_t* code[NT];
  size_t group0[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const uint32_t row = n0 + n * 16 + i < A.rows ? n0 + n * 16 + i : A.rows - 1;
    code[n] = A.codes + (size_t)row * (A.cols / 2) + j * 16;
    group0[n] = (size_t)row * A.groups;
  }
  const T* x[MT];
  int part[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint32_t r = m * 16 + i;
    part[m] = r < P * tb ? (int)(r / tb) : -1;
    x[m] = static_cast<const T*>(A.x) + (int64_t)(t0 + (r < P * tb ? r % tb : 0)) * A.x_token;
  }

  struct Block {
    uint4v w[NT];
    uint16_t scale[NT][GPB];
    uint8_t zero[NT][GPB];
    frag a[MT][4];
  };
  auto fetch = [&](uint32_t kb, Block& b) {
    const bool in = kb + j * 32 < A.cols;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      b.w[n] = uint4v{0, 0, 0, 0};
      if (in) b.w[n] = *reinterpret_cast<const uint4v*>(code[n] + kb / 2);
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        const uint32_t at = kb / G + g < A.groups ? kb / G + g : A.groups - 1;
        b.scale[n][g] = A.scales[group0[n] + at];
        b.zero[n][g] = A.zeros ? A.zeros[group0[n] + at] : 8;
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t k = kb + (G == 128 ? 32 * j + 8 * s : 32 * s + 8 * j);
        b.a[m][s] = frag{};
        if (part[m] >= 0 && k < A.cols) {
          if constexpr (P == 1) {
            if (A.wide) {
              b.a[m][s] = *reinterpret_cast<const frag*>(x[m] + k);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) b.a[m][s][e] = x[m][k + e];
            }
          } else {
            float v[8];
            load_row<8>(x[m] + k, A.wide, v);
            b.a[m][s] = operand(v, part[m], frag{});
          }
        }
      }
  };

  float4v acc[MT][NT] = {};
  auto compute = [&](const Block& b) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t d[4] = {b.w[n][0], b.w[n][1], b.w[n][2], b.w[n][3]};
      if constexpr (G < 128) transpose4(d);
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        const typename O::one z = (typename O::one)(-(float)b.zero[n][g]);
        const frag zero = {z, z, z, z, z, z, z, z};
        const float scale = scale_of(b.scale[n][g], A.bf16_scales);
        float4v c[MT] = {};
#pragma unroll
        for (int s = 0; s < SPG; ++s) {
          const frag w = decode<O>(d[g * SPG + s]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            c[m] = mma(b.a[m][g * SPG + s], w, c[m]);
            c[m] = mma(b.a[m][g * SPG + s], zero, c[m]);
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[m][n][r] = fmaf(scale, c[m][r], acc[m][n][r]);
      }
    }
  };

  const uint32_t step = waves * 128;
  Block b[2];
  uint32_t kb = wave * 128;
  if (kb < A.cols) fetch(kb, b[0]);
  while (kb < A.cols) {
    if (kb + step < A.cols) fetch(kb + step, b[1]);
    compute(b[0]);
    kb += step;
    if (kb >= A.cols) break;
    if (kb + step < A.cols) fetch(kb + step, b[0]);
    compute(b[1]);
    kb += step;
  }

  // sums[wave][row][16 NT]
  constexpr uint32_t kWidth = 16 * NT, kTile = MT * 16 * kWidth;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sums[wave * kTile + (m * 16 + 4 * j + r) * kWidth + n * 16 + i] = acc[m][n][r];
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < tb * kWidth; e += blockDim.x) {
    const uint32_t t = e / kWidth, n = e % kWidth;
    float y = 0;
    for (uint32_t w = 0; w < waves; ++w)
#pragma unroll
      for (int p = P - 1; p >= 0; --p) y += sums[w * kTile + (p * tb + t) * kWidth + n];
    if (n0 + n < A.rows) static_cast<T*>(A.y)[(int64_t)(t0 + t) * A.y_token + n0 + n] = (T)y;
  }
}

// ---------------------------------------------------------------------- host

int check(const fr_hip_q4* r) {
  if (!r || r->type > FR_HIP_BF16 || (r->scale_type != FR_HIP_F16 && r->scale_type != FR_HIP_BF16)) return FR_HIP_INVALID;
  if (r->group != 32 && r->group != 64 && r->group != 128) return FR_HIP_INVALID;
  if (!r->cols || r->cols % r->group) return FR_HIP_INVALID;
  if (r->tokens && r->rows && (!r->x || !r->codes || !r->scales || !r->y)) return FR_HIP_INVALID;
  if ((uintptr_t)r->codes % 16 || (uintptr_t)r->scales % 2) return FR_HIP_INVALID;
  if (((uintptr_t)r->x | (uintptr_t)r->y) % elem_size(r->type)) return FR_HIP_INVALID;
  if (r->tokens > 4096 || r->cols > 65536 || r->rows > (1u << 28)) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

template <typename T, int MT, int G>
void launch_rows(const Q4Args& A, hipStream_t s) {
  constexpr int TB = MT * 16 / Operand<T>::kParts;
  const uint32_t tiles = (A.rows + 15) / 16, blocks = (A.cols + 127) / 128;
  const dim3 grid(tiles, (A.tokens + TB - 1) / TB);
  // The columns are split until there are about eight wavefronts for each of
  // the card's compute units.
  uint32_t waves = 1;
  while (waves < 8 && (uint64_t)grid.x * grid.y * waves < 2048 && waves * 2 <= blocks) waves *= 2;
  hipLaunchKernelGGL((q4_rows<T, MT, 1, G>), grid, dim3(64 * waves), waves * MT * 16 * 16 * sizeof(float), s, A);
}

template <typename T, int MT>
void launch_group(const Q4Args& A, unsigned group, hipStream_t s) {
  switch (group) {
    case 32: launch_rows<T, MT, 32>(A, s); break;
    case 64: launch_rows<T, MT, 64>(A, s); break;
    default: launch_rows<T, MT, 128>(A, s); break;
  }
}

template <typename T>
void launch_tokens(const Q4Args& A, unsigned group, hipStream_t s) {
  const uint32_t rows = A.tokens * Operand<T>::kParts;
  if (rows <= 16) launch_group<T, 1>(A, group, s);
  else if (rows <= 32) launch_group<T, 2>(A, group, s);
  else launch_group<T, 4>(A, group, s);
}

}  // namespace

extern "C" {

size_t fr_hip_q4_workspace(const fr_hip_q4* req) {
  (void)req;
  return 0;
}

int fr_hip_q4_product(const fr_hip_q4* req, void* workspace, size_t bytes, void* stream) {
  (void)workspace, (void)bytes;
  int rc = check(req);
  if (rc) return rc;
  hipStream_t s;
  unsigned cus;
  rc = fronk::enter(stream, &s, &cus);
  if (rc || !req->tokens || !req->rows) return rc;
  const int64_t n = 16 / (int64_t)elem_size(req->type);
  Q4Args A;
  A.x = req->x, A.codes = req->codes, A.scales = static_cast<const uint16_t*>(req->scales), A.zeros = req->zeros;
  A.y = req->y, A.x_token = req->x_token, A.y_token = req->y_token;
  A.tokens = req->tokens, A.rows = req->rows, A.cols = req->cols, A.groups = req->cols / req->group;
  A.bf16_scales = req->scale_type == FR_HIP_BF16;
  A.wide = (uintptr_t)req->x % 16 == 0 && req->x_token % n == 0;
  switch (req->type) {
    case FR_HIP_F32: launch_tokens<float>(A, req->group, s); break;
    case FR_HIP_F16: launch_tokens<_Float16>(A, req->group, s); break;
    default: launch_tokens<__bf16>(A, req->group, s); break;
  }
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}

}  // extern "C"
