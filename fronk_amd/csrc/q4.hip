// q4.hip - products with 4-bit weights and group scales (fr_hip_q4_product):
//     y[t][n] = sum_g scale[n][g] sum_{k in g} x[t][k] (code[n][k] - zero[n][g]) .
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "dense.h"
#include "q4_order.h"

namespace {

struct Q4Args {
  const void* x;
  const uint8_t* codes;
  const uint16_t* scales;
  const uint8_t* zeros;
  void* y;
  int64_t x_token, y_token;
  uint32_t tokens, rows, cols, groups;
  bool bf16_scales, wide, wide_y;   // wide: rows of x (of y) are of whole 16 bytes
};

// The matrix cores' operand type: fp16 activations meet fp16 codes, all others
// bf16 ones (codes 0..15 are exact in both). fp32 activations are the sum of
// three bf16 parts (8 + 8 + 8 bits).
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

// Eight activations as loaded (any alignment of the type's own), and as
// operands: their three bf16 parts, or themselves.
template <typename T> struct Eight {
  typedef T vec __attribute__((ext_vector_type(8)));
  typedef vec loose __attribute__((aligned(sizeof(T))));
};
__device__ __forceinline__ void operands(Eight<float>::vec x, bf16x8 (&out)[3]) {
#pragma unroll
  for (int p = 0; p < 3; ++p)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const bf16x2 h = to_bf16(x[e], x[e + 1]);
      out[p][e] = h[0], out[p][e + 1] = h[1];
      if (p < 2) x[e] -= (float)h[0], x[e + 1] -= (float)h[1];
    }
}
__device__ __forceinline__ void operands(bf16x8 x, bf16x8 (&out)[1]) { out[0] = x; }
__device__ __forceinline__ void operands(half8v x, half8v (&out)[1]) { out[0] = x; }

__device__ __forceinline__ float scale_of(uint16_t bits, bool bf16) {
  if (bf16) return __builtin_bit_cast(float, (uint32_t)bits << 16);
  return (float)__builtin_bit_cast(_Float16, bits);
}

// One workgroup: 16 rows of W for each `splits` of its wavefronts, by 16 MT
// tokens. Those of the same rows take every (splits)th block of 128 columns and
// add up through LDS at the end. The codes are read once, so that reading them is
// the time there is: each wavefront has DEPTH blocks of them in flight, and asks
// for a block's successor as soon as it is multiplied. x is laid out as operands
// in LDS, `segment` blocks at a time, once for the workgroup (from memory, four
// of a block's five reads would be x's). 4096 x 65536 of one token: 35 us, 3.9 TB/s
// (52 with x from memory); 7 fp32 tokens of 2592 x 4099: 13.3; 2560 x 2560: 5.2.
//
// x is the A operand (tokens as rows; beyond the last it is repeated), 16 rows of
// W the B operand, so that a lane's four results belong to its own weight row: one
// scale a lane and group. A lane reads 16 bytes of its row (32 codes). With groups
// of 128 a block is one group and step s takes columns 32 j + 8 s ..; smaller
// groups must not mix in one instruction, so the words are transposed over the
// lane rows and step s takes columns 32 s + 8 j .. . The zero point meets the sum
// of x over its group, formed like a row of W whose codes are all 1.
template <typename T, int MT> constexpr uint32_t kDepth = Operand<T>::kParts * MT == 1 ? 4 : 2;
struct RowsArgs {
  Q4Args a;
  uint32_t splits, segment;
};

template <typename T, int MT, int G, bool ZEROS, bool WHOLE>
__global__ __launch_bounds__(512) void q4_rows(RowsArgs R) {
  typedef Operand<T> O;
  typedef typename O::frag frag;
  const Q4Args& A = R.a;
  constexpr int P = O::kParts, SPG = G / 32, GPB = 128 / G, TB = MT * 16;
  constexpr uint32_t DEPTH = kDepth<T, MT>;
  extern __shared__ uint4v lds[];
  const uint32_t lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t i = lane & 15, j = lane >> 4;
  const uint32_t split = wave % R.splits, tile = blockIdx.x * (waves / R.splits) + wave / R.splits;
  const uint32_t t0 = blockIdx.y * TB, blocks = (A.cols + 127) / 128;
  const uint32_t tb = A.tokens - t0 < (uint32_t)TB ? A.tokens - t0 : (uint32_t)TB;

  const uint32_t row = tile * 16 + i < A.rows ? tile * 16 + i : A.rows - 1;
  const uint8_t* code = A.codes + (size_t)row * (A.cols / 2) + j * 16;
  const uint16_t* scales = A.scales + (size_t)row * A.groups;
  const uint8_t* zeros = ZEROS ? A.zeros + (size_t)row * A.groups : nullptr;

  struct Block {
    uint4v w;
    uint16_t scale[GPB];
    uint8_t zero[GPB];
  };
  // Behind the last block that one is read again: a load that may be left out
  // would make every wait one for all loads.
  auto fetch = [&](uint32_t k, Block& b) {
    const uint32_t kb = k < blocks ? k : blocks - 1, back = kb * 128 + j * 32 < A.cols ? 0 : j * 16;
    b.w = *reinterpret_cast<const uint4v*>(code + kb * 64 - back);
    if constexpr (GPB > 1 && WHOLE) {
      typedef uint16_t words __attribute__((ext_vector_type(GPB)));
      typedef uint8_t bytes __attribute__((ext_vector_type(GPB)));
      const words s = *reinterpret_cast<const words*>(scales + kb * GPB);
      bytes z;
      if constexpr (ZEROS) z = *reinterpret_cast<const bytes*>(zeros + kb * GPB);
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        b.scale[g] = s[g];
        if constexpr (ZEROS) b.zero[g] = z[g];
      }
    } else {
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        const uint32_t at = kb * GPB + g < A.groups ? kb * GPB + g : A.groups - 1;
        b.scale[g] = scales[at];
        if constexpr (ZEROS) b.zero[g] = zeros[at];
      }
    }
  };

  // Operands of x: [block][step][part][token][lane row].
  auto stage = [&](uint32_t first, uint32_t last) {
    const uint32_t units = (last - first) * 16 * tb;
    for (uint32_t u = threadIdx.x; u < units; u += blockDim.x) {
      const uint32_t uj = u % 4, t = u / 4 % tb, s = u / 4 / tb % 4, kb = u / 16 / tb;
      const uint32_t c = (first + kb) * 128 + (G == 128 ? 32 * uj + 8 * s : 32 * s + 8 * uj);
      typename Eight<T>::vec v = {};
      if (c < A.cols)
        v = *reinterpret_cast<const typename Eight<T>::loose*>(static_cast<const T*>(A.x) + (int64_t)(t0 + t) * A.x_token + c);
      frag f[P];
      operands(v, f);
#pragma unroll
      for (int p = 0; p < P; ++p) lds[((kb * 4 + s) * P + p) * tb * 4 + t * 4 + uj] = __builtin_bit_cast(uint4v, f[p]);
    }
  };

  const typename O::one one = (typename O::one)1.f;
  const frag ones = {one, one, one, one, one, one, one, one};
  uint32_t unit[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) unit[m] = min(m * 16 + i, tb - 1) * 4 + j;
  float4v acc[MT] = {};
  auto compute = [&](uint32_t kb, const Block& b) {   // kb: from the segment's first
    const uint4v* x = lds + kb * 4 * P * tb * 4;
    uint32_t d[4] = {b.w[0], b.w[1], b.w[2], b.w[3]};
    if constexpr (G < 128) transpose4(d);
#pragma unroll
    for (int g = 0; g < GPB; ++g) {
      float4v c[MT] = {}, all[MT] = {};
#pragma unroll
      for (int s = g * SPG; s < (g + 1) * SPG; ++s) {
        const frag w = decode<O>(d[s]);
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const frag a = __builtin_bit_cast(frag, x[(s * P + p) * tb * 4 + unit[m]]);
            c[m] = mma(a, w, c[m]);
            all[m] = mma(a, ones, all[m]);
          }
      }
      const float scale = scale_of(b.scale[g], A.bf16_scales), zero = ZEROS ? (float)b.zero[g] : 8.f;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(scale, fmaf(-zero, all[m][r], c[m][r]), acc[m][r]);
    }
  };

  Block b[DEPTH];
#pragma unroll
  for (uint32_t d = 0; d < DEPTH; ++d) fetch(split + d * R.splits, b[d]);
  const uint32_t round = DEPTH * R.splits;
  uint32_t first = 0, last = 0;   // of the segment in LDS, of whole rows of splits
  auto step = [&](uint32_t k, Block& now, bool more) {
    if (k == last) {
      first = k, last = k + R.segment < blocks ? k + R.segment : blocks;
      if (k) __syncthreads();
      stage(first, last);
      __syncthreads();
    }
    if (k + split < blocks) compute(k + split - first, now);
    if (more) fetch(k + round + split, now);
    __builtin_amdgcn_sched_barrier(0);   // no operands of later blocks held meanwhile
  };
  uint32_t k = 0;
  for (; k + round < blocks; k += round)
#pragma unroll
    for (uint32_t d = 0; d < DEPTH; ++d) step(k + d * R.splits, b[d], true);
#pragma unroll
  for (uint32_t d = 0; d < DEPTH; ++d)
    if (k + d * R.splits < blocks) step(k + d * R.splits, b[d], false);

  // [wave][token][row]
  float* sums = reinterpret_cast<float*>(lds);
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[(wave * TB + m * 16 + 4 * j + r) * 16 + i] = acc[m][r];
  __syncthreads();
  const uint32_t width = waves / R.splits * 16, n0 = blockIdx.x * width;
  for (uint32_t e = threadIdx.x; e < tb * width; e += blockDim.x) {
    const uint32_t t = e / width, n = e % width;
    float y = 0;
    for (uint32_t w = 0; w < R.splits; ++w) y += sums[((n / 16 * R.splits + w) * TB + t) * 16 + n % 16];
    if (n0 + n < A.rows) static_cast<T*>(A.y)[(int64_t)(t0 + t) * A.y_token + n0 + n] = (T)y;
  }
}

// ------------------------------------------------------------ many tokens
//
// From a block of tokens on, W is decoded for 64 tokens at a time straight into
// the wavefronts that multiply it, and x is laid out beforehand (q4_pack) as the
// operands that all of them share through LDS.
//
// Both operands are fp16 here, where two codes are numbers after two packed
// instructions (published by Kim et al., Who Says Elephants Can't Run, 2022): 0x6400 | c is 1024 + c, and with c four bits higher 1024 + 16 c,
// so that one packed add or fma gives c - zero exactly. fp16 activations go as
// they are; a bf16 token is scaled by the power of two that brings its largest
// to 2^14 .. 2^15, which keeps every value down to 2^-32 of the largest exact
// and the others to 2^-40 of it, below fp32's rounding of their sum; an fp32
// token takes two such parts: 2^-23 of each value down to 2^-16 of the token's
// largest, and 2^-39 of the largest below.
constexpr int kTokens = 64;

template <typename T> struct Packed { static constexpr int kParts = std::is_same<T, float>::value ? 2 : 1; };

// Blocks of 128 columns of x, as many for either half of a workgroup.
__host__ __device__ __forceinline__ uint32_t padded_blocks(uint32_t cols) { return (cols + 255) / 256 * 2; }

struct TileArgs {
  Q4Args a;
  uint4v* packed;      // [block of 128 columns][tile of 16 tokens][part][step][lane]
  int32_t* exponent;   // of each token
  uint32_t tiles;      // of tokens, a multiple of 4
  bool whole;          // whole_groups
};

// One workgroup: 16 tokens, and every gridDim.y-th sixteenth of their operands.
// Two passes over x, the first for the largest values: 9 us for 512 x 4096.
template <typename T, int G>
__global__ __launch_bounds__(1024) void q4_pack(TileArgs C) {
  const Q4Args& A = C.a;
  constexpr int P = Packed<T>::kParts;
  constexpr bool kScaled = !std::is_same<T, _Float16>::value;
  __shared__ uint32_t largest[16];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, j = lane >> 4, tile = blockIdx.x;
  if constexpr (kScaled) {
    uint32_t top = 0;
    if (tile * 16 + wave < A.tokens) {
      const T* x = static_cast<const T*>(A.x) + (int64_t)(tile * 16 + wave) * A.x_token;
#pragma unroll 4
      for (uint32_t c = lane * 8; c < A.cols; c += 512) {
        float v[8];
        load_row<8>(x + c, A.wide, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
      }
    }
    for (int d = 1; d < 64; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if (lane == 0) largest[wave] = top;
    __syncthreads();
  }
  const uint32_t top = kScaled ? largest[i] : 0;
  const bool finite = top < 0x7f800000u;
  const int shift = kScaled ? 141 - (int)max(top >> 23, 1u) : 0;
  if (blockIdx.y == 0 && wave == 0 && j == 0) C.exponent[tile * 16 + i] = finite ? -shift : 0;
  const uint32_t pieces = padded_blocks(A.cols) * 4;
  const T* x = static_cast<const T*>(A.x) + (int64_t)(tile * 16 + i) * A.x_token;
  for (uint32_t f = blockIdx.y * 16 + wave; f < pieces; f += gridDim.y * 16) {
    const uint32_t kb = f / 4, s = f % 4, c = kb * 128 + (G == 128 ? 32 * j + 8 * s : 32 * s + 8 * j);
    float v[8] = {};
    if (tile * 16 + i < A.tokens && c < A.cols) load_row<8>(x + c, A.wide, v);
    half8v out[P];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // The order in which a word of codes is decoded: 0 4 1 5 2 6 3 7.
      const float y = v[e / 2 + e % 2 * 4];
      const float z = kScaled ? (finite ? ldexpf(y, shift) : NAN) : y;
      out[0][e] = (_Float16)z;
      if constexpr (P == 2) out[1][e] = (_Float16)(z - (float)out[0][e]);
    }
#pragma unroll
    for (int p = 0; p < P; ++p)
      C.packed[(((size_t)kb * C.tiles + tile) * P + p) * 256 + s * 64 + lane] = __builtin_bit_cast(uint4v, out[p]);
  }
}

// What decoding needs in registers, where the compiler would otherwise put it
// into each instruction and split the bit select into an and and an or.
struct Magic {
  uint32_t low = 0x000f000fu, high = 0x00f000f0u, base = 0x64006400u;
  __device__ __forceinline__ Magic() { asm("" : "+s"(low), "+s"(high), "+v"(base)); }
};
__device__ __forceinline__ half8v minus_zero(uint32_t w, half2v z1024, half2v z64, const Magic& c) {
  const half2v sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  auto pick = [&](uint32_t x, uint32_t mask) { return __builtin_bit_cast(half2v, (x & mask) | c.base); };
  const uint32_t v = w >> 8;
  const half2v a = pick(w, c.low) + z1024, b = pick(w, c.high) * sixteenth + z64;
  const half2v d = pick(v, c.low) + z1024, e = pick(v, c.high) * sixteenth + z64;
  return {a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// One workgroup: 64 tokens by 64 NT rows of W. Its two halves of four wavefronts
// take half of the blocks of 128 columns each and join through LDS; a wavefront
// has 16 NT rows of its own, which nothing else decodes, and all of the tokens.
//
// The matrix instructions of 16 rows and one group start from zero, and their
// sums enter the result times the group's scale. What else there is to do goes
// on beside them: the sums before are scaled and added, the next 16 rows are
// decoded, their codes of the next block are asked for, and with a block's last
// rows x of the next one comes from LDS, each operand into the registers that
// it was the last to use. Loads are never left out, not even behind the last
// block (they then read another one): only so a wait tells those that it is for
// from those behind them. Two parts of x, or sums of 32 columns each, leave no
// registers for x ahead of its block (kAhead).
//
// 512 x 4096 x 8192 in groups of 128: 47 us (and 9 for q4_pack), of which the matrix
// cores work for 14; the others' LDS reads, decoding and scaled sums go on beside
// them only in part. Without what goes beside: 65 us. Groups of 64: 62, of 32: 66.
template <typename T, int G, int NT, bool ZEROS, bool WHOLE>
__global__ __launch_bounds__(512) void q4_tiles(TileArgs C, uint32_t token_blocks) {
  const Q4Args& A = C.a;
  constexpr int P = Packed<T>::kParts, GPB = 128 / G, SPG = G / 32;
  constexpr int kPitch = 64 * NT + 4;
  constexpr bool kAhead = P == 1 && G > 32;
  extern __shared__ uint4v lds[];   // [half][2][P * 1024], then the sums [64][kPitch]
  const int lane = threadIdx.x & 63, i = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave >> 2, w = wave & 3;
  // Workgroups go to the dies in turn: all blocks of tokens of the same rows to one.
  const uint32_t tn = blockIdx.x % 8 + blockIdx.x / (8 * token_blocks) * 8, tm = blockIdx.x / 8 % token_blocks;
  const uint32_t n0 = (tn * 4 + w) * 16 * NT;
  if (tn * 64 * NT >= A.rows) return;

  const uint32_t blocks = (A.cols + 127) / 128, count = (blocks + 1) / 2, from = half * count;
  // The wavefront's first row, and the lane's from there (below 2^21 bytes).
  const uint32_t row0 = n0 < A.rows ? n0 : A.rows - 1;
  const uint8_t* codes = A.codes + (size_t)row0 * (A.cols / 2);
  const uint16_t* scales = A.scales + (size_t)row0 * A.groups;
  const uint8_t* zeros = ZEROS ? A.zeros + (size_t)row0 * A.groups : nullptr;
  uint32_t code[NT], group0[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const uint32_t row = (n0 + n * 16 + i < A.rows ? n0 + n * 16 + i : A.rows - 1) - row0;
    code[n] = row * (A.cols / 2) + j * 16;
    group0[n] = row * A.groups;
  }
  // Block k of this half; past the last column any codes do, x is zero there.
  uint4v w4[NT];
  uint16_t scale16[NT][GPB];
  uint8_t zero8[NT][GPB];
  auto load_w = [&](uint32_t k, int n) {
    const uint32_t kb = min(from + (k < count ? k : 0), blocks - 1);
    const uint32_t back = kb * 128 + j * 32 < A.cols ? 0 : j * 16;
    w4[n] = *reinterpret_cast<const uint4v*>(codes + (size_t)kb * 64 + (code[n] - back));
    if constexpr (GPB > 1 && WHOLE) {
      typedef uint16_t words __attribute__((ext_vector_type(GPB)));
      typedef uint8_t bytes __attribute__((ext_vector_type(GPB)));
      const words s = *reinterpret_cast<const words*>(scales + kb * GPB + group0[n]);
      bytes z;
      if constexpr (ZEROS) z = *reinterpret_cast<const bytes*>(zeros + kb * GPB + group0[n]);
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        scale16[n][g] = s[g];
        if constexpr (ZEROS) zero8[n][g] = z[g];
      }
    } else {
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        const uint32_t at = (kb * GPB + g < A.groups ? kb * GPB + g : A.groups - 1) + group0[n];
        scale16[n][g] = scales[at];
        if constexpr (ZEROS) zero8[n][g] = zeros[at];
      }
    }
  };
  uint4v stage[4 * P];
  const int thread = threadIdx.x & 255;
  auto load_x = [&](uint32_t k) {
    const uint4v* p = C.packed + ((size_t)(from + (k < count ? k : 0)) * C.tiles + tm * 4) * P * 256 + thread;
#pragma unroll
    for (int n = 0; n < 4 * P; ++n) stage[n] = p[n * 256];
  };
  auto store_x = [&](uint32_t k) {
#pragma unroll
    for (int n = 0; n < 4 * P; ++n) lds[(half * 2 + k % 2) * P * 1024 + n * 256 + thread] = stage[n];
  };
  half8v a[4][P][4], b[2][4];
  auto read_x = [&](uint32_t k, int s) {
    const uint4v* x = lds + (half * 2 + k % 2) * P * 1024 + lane;
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int p = 0; p < P; ++p) a[m][p][s] = __builtin_bit_cast(half8v, x[((m * P + p) * 4 + s) * 64]);
  };
  const Magic magic;
  float scale[2][GPB];
  auto decode = [&](int n, int to) {
    uint32_t d[4] = {w4[n][0], w4[n][1], w4[n][2], w4[n][3]};
    if constexpr (G < 128) transpose4(d);
#pragma unroll
    for (int g = 0; g < GPB; ++g) {
      // -(1024 + zero) by its bits, and 960 more than it.
      const uint32_t z = ZEROS ? zero8[n][g] : 8u;
      const half2v z1 = __builtin_bit_cast(half2v, (z | z << 16) | 0xe400e400u);
      const half2v z2 = z1 + half2v{(_Float16)960.f, (_Float16)960.f};
#pragma unroll
      for (int s = g * SPG; s < (g + 1) * SPG; ++s) b[to][s] = minus_zero(d[s], z1, z2, magic);
      scale[to][g] = scale_of(scale16[n][g], A.bf16_scales);
    }
  };

  float4v acc[4][NT] = {}, sum[4] = {};
  float sum_scale = 0;
  auto add = [&](int n) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[m][n][r] = fmaf(sum_scale, sum[m][r], acc[m][n][r]);
  };
#pragma unroll
  for (int n = 0; n < NT; ++n) load_w(0, n);
  auto barrier = [] { __syncthreads(); };
  auto read_block = [&](uint32_t k) {
#pragma unroll
    for (int s = 0; s < 4; ++s) read_x(k, s);
  };
  fronk::tiles_first<kAhead>(load_x, store_x, barrier, read_block);
  decode(0, 0);
  load_w(1, 0);
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): the loop's own waits are then for its own loads
  for (uint32_t k = 0; k < count; ++k) {
    fronk::tiles_before<kAhead>(k, load_x, barrier, read_block);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      constexpr bool kBeside = NT > 1;   // else the rows just multiplied make way first
      const int then = (n + 1) % NT, now = n % 2, to = kBeside ? 1 - now : 0;
      if constexpr (kBeside) decode(then, to), load_w(n + 1 < NT ? k + 1 : k + 2, then);
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        float4v c[4] = {};
#pragma unroll
        for (int s = g * SPG; s < (g + 1) * SPG; ++s)
#pragma unroll
          for (int p = P - 1; p >= 0; --p)
#pragma unroll
            for (int m = 0; m < 4; ++m) c[m] = mma(a[m][p][s], b[now][s], c[m]);
        add(g ? n : (n + NT - 1) % NT);
#pragma unroll
        for (int m = 0; m < 4; ++m) sum[m] = c[m];
        sum_scale = scale[now][g];
        if (kAhead && n == NT - 1) {
#pragma unroll
          for (int s = g * SPG; s < (g + 1) * SPG; ++s) read_x(k + 1, s);
        }
      }
      if constexpr (!kBeside) decode(then, to), load_w(k + 2, then);
      if constexpr (kAhead) {
#pragma unroll
        for (int m = 0; m < 16; ++m) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // a matrix instruction,
          __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);   // and what fits beside it
          if (n == NT - 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
      }
    }
    fronk::tiles_after<kAhead>(k, store_x, barrier);
  }
  add(NT - 1);

  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);
  auto each = [&](auto f) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) f(sums[(m * 16 + 4 * j + r) * kPitch + (w * NT + n) * 16 + i], acc[m][n][r]);
  };
  if (half) each([](float& at, float x) { at = x; });
  __syncthreads();
  if (!half) each([](float& at, float x) { at += x; });
  __syncthreads();
  const uint32_t t0 = tm * kTokens, left = A.rows - tn * 64 * NT;
  for (uint32_t e = threadIdx.x; e < kTokens * 8 * NT; e += 512) {
    const uint32_t t = e / (8 * NT), n = e % (8 * NT) * 8;
    if (t0 + t >= A.tokens) break;
    const int ex = C.exponent[t0 + t];
    T* y = static_cast<T*>(A.y) + (int64_t)(t0 + t) * A.y_token + tn * 64 * NT + n;
    typedef T vec __attribute__((ext_vector_type(8)));
    vec out;
#pragma unroll
    for (int r = 0; r < 8; ++r) out[r] = (T)ldexpf(sums[t * kPitch + n + r], ex);
    if (A.wide_y && n + 8 <= left) {
      *reinterpret_cast<vec*>(y) = out;
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (n + r < left) y[r] = out[r];
    }
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
  // Grids of less than 2^32 threads: 512 for 64 tokens and 128 rows.
  if ((uint64_t)(r->rows / 128 + 8) * (r->tokens / 64 + 1) > UINT32_MAX / 512) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

// The scales (and zero points) of a block of columns are aligned words.
template <int G> bool whole_groups(const Q4Args& A) {
  constexpr unsigned GPB = 128 / G;
  return A.groups % GPB == 0 && (uintptr_t)A.scales % (2 * GPB) == 0 && (uintptr_t)A.zeros % GPB == 0;
}

constexpr size_t kRowsLds = 64 << 10;   // two workgroups a compute unit

template <typename T, int MT, int G, bool ZEROS, bool WHOLE>
int launch_rows(const RowsArgs& C, dim3 grid, uint32_t waves, hipStream_t s) {
  const size_t x = (size_t)C.segment * 256 * Operand<T>::kParts * (C.a.tokens < MT * 16 ? C.a.tokens : MT * 16);
  const size_t sums = (size_t)waves * MT * 16 * 16 * sizeof(float);
  static fronk::Devices allowed;
  if (allow_lds(&q4_rows<T, MT, G, ZEROS, WHOLE>, kRowsLds, &allowed)) return FR_HIP_IO;
  hipLaunchKernelGGL((q4_rows<T, MT, G, ZEROS, WHOLE>), grid, dim3(64 * waves), x > sums ? x : sums, s, C);
  return FR_HIP_OK;
}

template <typename T, int MT, int G>
int launch_rows(const Q4Args& A, bool whole, hipStream_t s) {
  const uint32_t tiles = (A.rows + 15) / 16, blocks = (A.cols + 127) / 128;
  const uint32_t y = (A.tokens + MT * 16 - 1) / (MT * 16);
  const uint32_t tb = A.tokens < MT * 16 ? A.tokens : MT * 16;
  const size_t block = (size_t)256 * Operand<T>::kParts * tb;   // of x in LDS
  // The columns are split until there are about eight wavefronts for each of
  // the card's compute units, but not below one block for each, nor beyond what
  // LDS holds of x for all of them (at least one split's: 12 KB a block).
  RowsArgs C = {A, 1, 0};
  while (C.splits < 8 && (uint64_t)tiles * y * C.splits < 8 * kUnits && C.splits * 2 <= blocks && 2 * C.splits * block <= kRowsLds)
    C.splits *= 2;
  const uint32_t waves = 8, each = waves / C.splits;
  C.segment = (uint32_t)(kRowsLds / block) / C.splits * C.splits;
  if (C.segment > blocks) C.segment = (blocks + C.splits - 1) / C.splits * C.splits;
  const dim3 grid((tiles + each - 1) / each, y);
  if constexpr (G < 128)
    if (!whole) return A.zeros ? launch_rows<T, MT, G, true, false>(C, grid, waves, s) : launch_rows<T, MT, G, false, false>(C, grid, waves, s);
  return A.zeros ? launch_rows<T, MT, G, true, true>(C, grid, waves, s) : launch_rows<T, MT, G, false, true>(C, grid, waves, s);
}

// Tiles of 64 tokens, or rows for 32 (fp32: 16) at a time? Tiles cost 6 to 10 us
// more to begin with (q4_pack, and x through one more launch), rows decode W once
// for each of their blocks of tokens. Measured, rows against tiles in us, bf16 64
// tokens: 15.0, 17.7 (2560 x 2560, 6400 cells), 18.1, 22.3 (4096 x 4096, 16384),
// 26.4, 23.8 (4096 x 8192, 32768); 256 tokens of 2560 x 2560 (25600) 23.6, 19.5;
// fp32 32 tokens of 4096 x 8192 (32768) 27.4, 37.6.
bool in_tiles(const fr_hip_q4* r) {
  const uint32_t tokens = r->type == FR_HIP_F32 ? 16 : 32;
  const uint64_t cells = (uint64_t)((r->rows + 15) / 16) * ((r->cols + 127) / 128) * ((r->tokens + tokens - 1) / tokens);
  return r->tokens > tokens && cells > (r->type == FR_HIP_F32 ? 48 << 10 : 24 << 10);
}
uint32_t token_blocks(const fr_hip_q4* r) { return (r->tokens + kTokens - 1) / kTokens; }
size_t packed_units(const fr_hip_q4* r) {   // of 16 bytes
  return (size_t)padded_blocks(r->cols) * token_blocks(r) * 4 * 256 * (r->type == FR_HIP_F32 ? 2 : 1);
}
size_t workspace_bytes(const fr_hip_q4* r) {
  if (!in_tiles(r) || !r->rows) return 0;
  return packed_units(r) * 16 + (size_t)token_blocks(r) * kTokens * sizeof(int32_t);
}

template <typename T, int G, int NT, bool ZEROS, bool WHOLE>
int launch_tiles(const TileArgs& C, uint32_t blocks, hipStream_t s) {
  constexpr size_t x = (size_t)4 * Packed<T>::kParts * 1024 * 16, sums = (size_t)kTokens * (64 * NT + 4) * sizeof(float);
  constexpr size_t lds = x > sums ? x : sums;
  static fronk::Devices allowed;
  if (allow_lds(&q4_tiles<T, G, NT, ZEROS, WHOLE>, lds, &allowed)) return FR_HIP_IO;
  const uint32_t tiles = (C.a.rows + 64 * NT - 1) / (64 * NT);
  hipLaunchKernelGGL((q4_tiles<T, G, NT, ZEROS, WHOLE>), dim3((tiles + 7) / 8 * 8 * blocks), dim3(512), lds, s, C, blocks);
  return FR_HIP_OK;
}
template <typename T, int G, int NT, bool ZEROS>
int launch_tiles(const TileArgs& C, uint32_t blocks, hipStream_t s) {
  if constexpr (G < 128)
    if (!C.whole) return launch_tiles<T, G, NT, ZEROS, false>(C, blocks, s);
  return launch_tiles<T, G, NT, ZEROS, true>(C, blocks, s);
}
// The widest tiles that still give every compute unit one, up to those that are the
// fastest of their kind: 256 rows leave no registers for a second part of x, zero
// points or several groups a block. 512 x 4096 x 8192 in us with 64, 128 and 256 rows:
// 16 bits in groups of 128 75, 68, 51, of 64 95, 70, of 32 75, 73, 92; with zero points
// 85, 84 (128), 93, 83 (64), 84, 101 (32); fp32 141, 97 (128), 136, 100 (64), 161, 135
// (32), with zero points 149, 101, 146, 111, 164, 157, though some of its wide tiles in
// groups of 32 keep registers in memory.
template <typename T, int G, bool ZEROS>
int launch_widest(const TileArgs& C, uint32_t blocks, hipStream_t s) {
  constexpr int kMost = Packed<T>::kParts > 1 ? 2 : G == 128 && !ZEROS ? 4 : G == 32 && ZEROS ? 1 : 2;
  const uint64_t tiles = (uint64_t)((C.a.rows + 63) / 64) * blocks;
  if constexpr (kMost >= 4)
    if (tiles >= 4 * kUnits) return launch_tiles<T, G, 4, ZEROS>(C, blocks, s);
  if constexpr (kMost >= 2)
    if (tiles >= 2 * kUnits) return launch_tiles<T, G, 2, ZEROS>(C, blocks, s);
  return launch_tiles<T, G, 1, ZEROS>(C, blocks, s);
}

template <typename T, int G>
int launch_blocks(const fr_hip_q4* r, const Q4Args& A, void* workspace, hipStream_t s) {
  const uint32_t blocks = token_blocks(r);
  TileArgs C;
  C.a = A;
  C.packed = static_cast<uint4v*>(workspace);
  C.exponent = reinterpret_cast<int32_t*>(C.packed + packed_units(r));
  C.tiles = blocks * 4;
  C.whole = whole_groups<G>(A);
  const uint32_t pieces = padded_blocks(A.cols) * 4;
  hipLaunchKernelGGL((q4_pack<T, G>), dim3(C.tiles, pieces >= 64 ? 4 : 1), dim3(1024), 0, s, C);
  return A.zeros ? launch_widest<T, G, true>(C, blocks, s) : launch_widest<T, G, false>(C, blocks, s);
}

template <typename T, int MT>
int launch_group(const Q4Args& A, unsigned group, hipStream_t s) {
  switch (group) {
    case 32: return launch_rows<T, MT, 32>(A, whole_groups<32>(A), s);
    case 64: return launch_rows<T, MT, 64>(A, whole_groups<64>(A), s);
    default: return launch_rows<T, MT, 128>(A, true, s);
  }
}

template <typename T>
int launch(const fr_hip_q4* r, const Q4Args& A, void* workspace, hipStream_t s) {
  const unsigned group = r->group;
  if (in_tiles(r)) {
    switch (group) {
      case 32: return launch_blocks<T, 32>(r, A, workspace, s);
      case 64: return launch_blocks<T, 64>(r, A, workspace, s);
      default: return launch_blocks<T, 128>(r, A, workspace, s);
    }
  }
  if constexpr (Operand<T>::kParts == 1)
    if (A.tokens > 16) return launch_group<T, 2>(A, group, s);
  return launch_group<T, 1>(A, group, s);
}

}  // namespace

extern "C" {

size_t fr_hip_q4_workspace(const fr_hip_q4* req) { return check(req) ? 0 : workspace_bytes(req); }

int fr_hip_q4_product(const fr_hip_q4* req, void* workspace, size_t bytes, void* stream) {
  int rc = check(req);
  if (rc) return rc;
  const size_t need = workspace_bytes(req);
  if (need && (!workspace || bytes < need || (uintptr_t)workspace % 16)) return FR_HIP_INVALID;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !req->tokens || !req->rows) return rc;
  const int64_t n = 16 / (int64_t)elem_size(req->type);
  Q4Args A;
  A.x = req->x, A.codes = req->codes, A.scales = static_cast<const uint16_t*>(req->scales), A.zeros = req->zeros;
  A.y = req->y, A.x_token = req->x_token, A.y_token = req->y_token;
  A.tokens = req->tokens, A.rows = req->rows, A.cols = req->cols, A.groups = req->cols / req->group;
  A.bf16_scales = req->scale_type == FR_HIP_BF16;
  A.wide = (uintptr_t)req->x % 16 == 0 && req->x_token % n == 0;
  A.wide_y = (uintptr_t)req->y % 16 == 0 && req->y_token % n == 0;
  switch (req->type) {
    case FR_HIP_F32: rc = launch<float>(req, A, workspace, s); break;
    case FR_HIP_F16: rc = launch<_Float16>(req, A, workspace, s); break;
    default: rc = launch<__bf16>(req, A, workspace, s); break;
  }
  if (rc) return rc;
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}

}  // extern "C"
