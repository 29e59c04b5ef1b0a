// prompt.hip - causal attention of packed prompts (fr_hip_prompt_attend).
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "attend.h"
#include "bounds.h"
#include "dense.h"

namespace {

struct PromptArgs {
  const void *q, *k, *v;
  void* o;
  float *part_o, *part_ml;   // [item][split][R][D], [item][split][R][2]
  const int32_t *offsets, *k_offsets;
  uint32_t* status;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  uint32_t sequences, tokens, k_tokens, max_tokens, max_context, kv_heads, per, blocks, splits, chunk;
  float scale;
};

// A sequence: its first query and key, and how many. By a whole workgroup.
struct Prompt {
  int32_t q0, k0;
  uint32_t n, m;
  bool bad;
};
__device__ __forceinline__ Prompt prompt_of(const PromptArgs& A, uint32_t seq) {
  int32_t q0 = seq * A.max_tokens, q1 = q0 + A.max_tokens, k0 = seq * A.max_context, k1 = k0 + A.max_context;
  // Whether an offset before a sequence's is above it.
  auto falls = [&](const int32_t* offsets, int32_t own) {
    int32_t most = 0;
    for (uint32_t s = threadIdx.x; s < seq; s += blockDim.x) most = max(most, offsets[s]);
    return most > own;
  };
  bool bad = false;
  if (A.offsets) {
    q0 = same(A.offsets[seq]), q1 = same(A.offsets[seq + 1]);
    bad = falls(A.offsets, q0);
    if (!A.k_offsets) k0 = q0, k1 = q1;
  }
  if (A.k_offsets) {
    k0 = same(A.k_offsets[seq]), k1 = same(A.k_offsets[seq + 1]);
    bad |= falls(A.k_offsets, k0);
  }
  bad |= (fronk::bad_sequence(0, 1, q0, q1, A.tokens, A.max_tokens) | fronk::bad_sequence(0, 1, k0, k1, A.k_tokens, A.max_context)) != 0;
  return Prompt{q0, k0, (uint32_t)(q1 - q0), (uint32_t)(k1 - k0), __syncthreads_or(bad) != 0};
}
template <typename T> __device__ __forceinline__ T* output_row(const PromptArgs& A, const Prompt& P, uint32_t head, uint32_t row) {
  return static_cast<T*>(A.o) + (int64_t)(P.q0 + row / A.per) * A.o_token + (int64_t)(head * A.per + row % A.per) * A.o_head;
}
// One workgroup: one sequence, one key head and R of its rows, a row being a query
// head of that key head and a token (token-major, so that the heads of a token share
// every key), over one stretch of the keys. Tiles of KT keys and their values go to
// LDS, the next one while this one is used; each of four wavefronts has 32 rows with
// a running maximum and sum.
//
// Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a
// lane's column is one row throughout (its maximum, sum and rescaling are the lane's
// own, joined over two halves), and P goes from the first product's result into the
// second's operand where it stands: register r of a lane in half h is key
// 8 (r / 4) + 4 h + r % 4 of 32, and V^T's operand is read in that order.
//
// 16-bit types: v_mfma_f32_32x32x16, eight values a lane, with P in two parts (Weights);
// fp32: v_mfma_f32_32x32x2, exact products.
//
// Bound by the matrix cores and by the vector work beside them (per 32 x 32 scores a
// maximum, 16 exponentials a lane, their sum and P's parts), which overlap in part: 4096
// tokens of 16 heads of 256 over two key heads, bf16, take 211 to 245 us from run to run, at
// 213 640 TFLOP/s of what is seen and 960 of what is multiplied, and have the matrix cores
// busy for 60 % of the cycles and the vector units for 35; at dim 128 it is 43 to 53 % and 52
// to 56. Eight prompts of 1 to 1531 tokens (20 heads of 128 over four) 112 us in fp16 and 105 in
// bf16; in fp32 2048 tokens of 16 heads 141 us at dim 64, 264 at 128 (four key heads), 550 at
// 256 (two). 128 rows share what a tile of keys takes to load. The running maximum is let
// stay while no weight would pass 2^8, which saves rescaling the sums at nearly every tile.
// Steps of both products are interleaved with the LDS reads of the one after next
// (schedule), and matrix work goes before other wavefronts' vector work. One to three
// registers of the 16-bit forms at dims 128 and 256 are in scratch.
//
// Keys of a tile, and workgroups a compute unit that the registers are for.
template <typename T, int D> constexpr int kKeys = sizeof(T) == 4 || D > 64 ? 32 : 64;
template <typename T, int D> constexpr int kResident = D * sizeof(T) > 512 ? 1 : sizeof(T) == 2 && D == 128 ? 3 : 2;

// How weights are held. Parts: with P rounded to 16 bits once, outputs are off by about as
// much again as their own rounding makes, and by far more where values nearly cancel. A
// second part leaves 2^-16 of a weight in bf16, 2^-22 in fp16, and outputs off by their
// rounding alone: against 64 bits (relative, 512 tokens over 8192 keys of 128) 0.00165 in
// bf16 for 0.00223 with one part, 0.00021 in fp16 for 0.00028. It is half as many products
// again: those 512 tokens take 116 us for 87, 4096 of 16 heads of 256 213 for 165.
//
// Range: a half has no bits for what is far below a row's largest weight, though
// thousands of such keys may be all that a row gets (the largest one's value being zero). So
// in fp16 a row's largest weight of each tile is kept within 1 and 2^15, and set to 2^kBias
// when it leaves that: what weights are taken from goes down again where a tile's scores
// are all lower. A weight is then off by 2^-25 of its tile's largest beside its
// rounding. Down by 2^60 at most from the row's largest, which leaves the sums in fp32
// (2^75 of a weight, 2^16 of a value and 2^31 keys are 2^122); keys yet lower add nothing
// that a half holds. It takes 1 to 2 % of a call.
template <typename T> struct Weights {
  static constexpr int kParts = 2;
  static constexpr bool kDown = false;
  static constexpr float kBias = 0.f;
};
template <> struct Weights<_Float16> {
  static constexpr int kParts = 2;
  static constexpr bool kDown = true;
  static constexpr float kBias = 7.f;
};
template <> struct Weights<float> {
  static constexpr int kParts = 1;
  static constexpr bool kDown = false;
  static constexpr float kBias = 0.f;
};

// WIDE: rows begin at multiples of 16 bytes.
template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(64 * kWaves, (kResident<T, D>)) void prompt_attend(PromptArgs A) {
  typedef typename Kind<T>::frag frag;
  constexpr int kEach = 16 / sizeof(T), KT = kKeys<T, D>;      // elements of 16 bytes; keys of a tile
  constexpr uint32_t kRow = D * sizeof(T), kChunks = kRow / 16;
  constexpr uint32_t kTile = KT * kRow;               // bytes of a tile of K, or of V
  constexpr int KS = D / (2 * kEach), ST = KT / 32, PS = 16 / kEach;   // steps of QK, subtiles, steps of PV a subtile
  constexpr int DT = D / 32;
  constexpr uint32_t kLoads = kTile / 1024 / kWaves;  // a wavefront's, of 64 chunks each
  static_assert(kTile % (1024 * kWaves) == 0, "whole loads");
  extern __shared__ __attribute__((aligned(16))) char lds[];   // [2][K, V][kTile]
  __shared__ int32_t first_bad[D];

  const uint32_t lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Key heads vary fastest, which leaves each die few of them; then sequences, stretches
  // and last row blocks, from the last (with the most keys) to the first.
  uint32_t at = blockIdx.x;
  const uint32_t head = at % A.kv_heads;
  at /= A.kv_heads;
  const uint32_t seq = at % A.sequences;
  at /= A.sequences;
  const uint32_t split = at % A.splits, block = A.blocks - 1 - at / A.splits;
  const Prompt P = prompt_of(A, seq);
  if (P.bad) {
    if (A.status && threadIdx.x == 0) atomicOr(A.status, FR_HIP_BAD_OFFSET);
    return;
  }
  const uint32_t n = P.n, m = P.m, rows = n * A.per, row0 = block * R;   // n * per < 2^31
  if (row0 >= rows) return;
  // Row r sees keys below base_seen + r / per (a signed number).
  const int32_t base_seen = (int32_t)(m - n) + 1;
  const int32_t seen_most = base_seen + (int32_t)((min(row0 + R, rows) - 1) / A.per);
  const uint32_t begin = split * A.chunk;
  const uint32_t end = seen_most <= (int32_t)begin ? begin : min((uint32_t)seen_most, begin + A.chunk);
  const uint32_t wave_row = row0 + wave * 32, row = wave_row + i;
  const int32_t limit = row < rows ? base_seen + (int32_t)(row / A.per) : 0;
  // Keys that all rows of the wavefront see, and that any sees.
  const int32_t all_see = wave_row + 32 <= rows ? base_seen + (int32_t)(wave_row / A.per) : 0;
  const int32_t any_see = wave_row < rows ? base_seen + (int32_t)((min(wave_row + 32, rows) - 1) / A.per) : 0;

  // Q: lane (i, h) of step s holds row i's 16 bytes 2 s + h. A negative scale is
  // taken to Q, so that the largest product is the largest score.
  const float scale = fmaxf(fabsf(A.scale) * kLog2e, 1e-37f);   // 0 would make NaN of a masked score
  frag qf[KS];
  {
    const uint32_t r = min(row, rows - 1);
    const T* p = static_cast<const T*>(A.q) + (int64_t)(P.q0 + r / A.per) * A.q_token +
                 (int64_t)(head * A.per + r % A.per) * A.q_head + h * kEach;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (WIDE) {
        qf[s] = *reinterpret_cast<const frag*>(p + s * 2 * kEach);
      } else {
#pragma unroll
        for (int e = 0; e < kEach; ++e) qf[s][e] = p[s * 2 * kEach + e];
      }
      if (A.scale < 0.f) qf[s] = -qf[s];
    }
  }

  // Loads of a tile: 16 bytes of a lane to 64 consecutive places, so the order in a
  // row is turned by the address read: chunk c of row r stands at c ^ (r & 7) (K,
  // whose lanes read one chunk of 32 rows) or c ^ 2 (r & 3) (V, whose lanes read 32
  // bytes of four rows), which spreads those over the banks.
  const char* const kp = reinterpret_cast<const char*>(static_cast<const T*>(A.k) + (int64_t)P.k0 * A.k_token + (int64_t)head * A.k_head);
  const char* const vp = reinterpret_cast<const char*>(static_cast<const T*>(A.v) + (int64_t)P.k0 * A.v_token + (int64_t)head * A.v_head);
  const int64_t k_row = A.k_token * (int64_t)sizeof(T), v_row = A.v_token * (int64_t)sizeof(T);
  // Load l of a wavefront begins kRows l rows behind its first; of kTurns of them the order differs.
  constexpr uint32_t kRows = 64 * kWaves / kChunks, kTurns = kRows % 8 ? 8 / kRows : 1;
  const uint32_t place0 = wave * 64 + lane, lane_row = place0 / kChunks, lane_chunk = place0 % kChunks;
  uint32_t k_off[kTurns], v_off[kTurns];
#pragma unroll
  for (uint32_t l = 0; l < kTurns; ++l) {
    const uint32_t r = lane_row + l * kRows;
    k_off[l] = lane_row * (uint32_t)k_row + (lane_chunk ^ (r & 7)) * 16;
    v_off[l] = lane_row * (uint32_t)v_row + (lane_chunk ^ 2 * (r & 3)) * 16;
  }
  auto load = [&](uint32_t base, uint32_t buffer) __attribute__((always_inline)) {
    char* const to = lds + buffer * 2 * kTile;
    if constexpr (WIDE) {
      const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char*)to + wave * 1024);
      const char *ks = kp + base * k_row, *vs = vp + base * v_row;
      if (base + KT <= m) {
#pragma unroll
        for (uint32_t l = 0; l < kLoads; ++l) {
          to_lds(ks + l * kRows * k_row, k_off[l % kTurns], at + l * kWaves * 1024);
          to_lds(vs + l * kRows * v_row, v_off[l % kTurns], at + kTile + l * kWaves * 1024);
        }
      } else {   // rows behind the last key are that key's, and count for nothing
#pragma unroll
        for (uint32_t l = 0; l < kLoads; ++l) {
          const uint32_t r = lane_row + l * kRows, there = min(r, m - 1 - base);
          to_lds(ks, there * (uint32_t)k_row + (lane_chunk ^ (r & 7)) * 16, at + l * kWaves * 1024);
          to_lds(vs, there * (uint32_t)v_row + (lane_chunk ^ 2 * (r & 3)) * 16, at + kTile + l * kWaves * 1024);
        }
      }
    } else {
#pragma unroll 1
      for (uint32_t place = threadIdx.x; place < kTile / 16; place += 64 * kWaves) {
        const uint32_t r = place / kChunks, c = place % kChunks;
        const int64_t token = min(base + r, m - 1);
        const T* ks = reinterpret_cast<const T*>(kp + token * k_row + (c ^ (r & 7)) * 16);
        const T* vs = reinterpret_cast<const T*>(vp + token * v_row + (c ^ 2 * (r & 3)) * 16);
        typedef T vec __attribute__((ext_vector_type(kEach)));
        vec x, y;
#pragma unroll
        for (int e = 0; e < kEach; ++e) x[e] = ks[e], y[e] = vs[e];
        *reinterpret_cast<vec*>(to + place * 16) = x;
        *reinterpret_cast<vec*>(to + kTile + place * 16) = y;
      }
    }
  };

  // Where the lane's operands begin in a tile. K: the chunks of step s are those of
  // s % 4, 8 on for every four. V: lane l of 16 reads row l / 4, columns 4 (l % 4) ..
  // and receives column l of the four rows; dims 32 d ..: as d % 2, 8 chunks on for
  // every two (fp32: single values, of four rows).
  uint32_t k_at[4], v_at[sizeof(T) == 2 ? 2 : 4];
#pragma unroll
  for (uint32_t s = 0; s < 4; ++s) k_at[s] = i * kRow + ((2 * s + h) ^ (i & 7)) * 16;
  if constexpr (sizeof(T) == 2) {
    const uint32_t r = lane / 4 % 4, c = lane / 16 % 2 * 2 + lane % 4 / 2;
#pragma unroll
    for (uint32_t d = 0; d < 2; ++d) v_at[d] = kTile + (4 * h + r) * kRow + ((4 * d + c) ^ 2 * r) * 16 + lane % 2 * 8;
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) v_at[e] = kTile + (4 * h + e) * kRow + ((i / 4) ^ 2 * e) * 16 + i % 4 * 4;
  }

  typedef Weights<T> W;
  float top, peak, shift, sum;
  float16v acc[DT];
  // A tile: scores, weights, outputs. `masked`: rows see different parts of it. (One
  // body with a branch over the mask alone: as two, the accumulators took twice the
  // registers.)
  auto compute = [&](uint32_t base, uint32_t buffer, bool masked) __attribute__((always_inline)) {
    const char* const tile = lds + buffer * 2 * kTile;
    // (The matrix cores' work goes before another wavefront's vector work.)
    __builtin_amdgcn_s_setprio(1);
    float16v st[ST];
#pragma unroll
    for (int t = 0; t < ST; ++t) {
      st[t] = float16v{};
#pragma unroll
      for (int s = 0; s < KS; ++s)
        st[t] = mma32(*reinterpret_cast<const frag*>(tile + k_at[s % 4] + t * 32 * kRow + s / 4 * 128), qf[s], st[t]);
    }
    schedule<ST * KS, 1, 2>();
    if (masked) {
#pragma unroll
      for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((int32_t)(base + t * 32 + 8 * (r / 4) + 4 * h + r % 4) >= limit) st[t][r] = -INFINITY;
    }
    // What weights are taken from moves only where one would pass 2^8 (in fp16 2^15, or
    // all would be small): sums and outputs are scaled seldom.
    const float most = max_xor32(largest(st)) * scale;
    bool moves = most > top + 8.f;
    float now = fmaxf(top, most);
    if constexpr (W::kDown) {
      peak = fmaxf(peak, most);
      const float low = fmaxf(most, peak - 60.f);
      moves |= most != -INFINITY && low < top - W::kBias;
      now = moves ? low : top;
    }
    if (__any(moves)) {
      const float to = now == -INFINITY ? 0.f : now;
      const float f = __builtin_amdgcn_exp2f(top - to);
      top = now, shift = to - W::kBias, sum *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f;
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    frag pf[ST][PS][W::kParts];
    float total[4] = {};
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][r], scale, -shift));
        total[r % 4] += p;
        float rest = p;
#pragma unroll
        for (int n = 0; n < W::kParts; ++n) {
          const T part = (T)rest;
          pf[t][r / kEach][n][r % kEach] = part, rest -= (float)part;
        }
      }
    sum += (total[0] + total[1]) + (total[2] + total[3]);
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int s = 0; s < PS; ++s)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          frag a;
          if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) short4v lds4;
            const char* p = tile + v_at[d % 2] + (t * 32 + s * 16) * kRow + d / 2 * 128;
            const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
            const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 8 * kRow));
            a = __builtin_bit_cast(frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              a[e] = *reinterpret_cast<const float*>(tile + v_at[e] + (t * 32 + s * 8) * kRow + d * 128);
          }
#pragma unroll
          for (int n = W::kParts - 1; n >= 0; --n) acc[d] = mma32(a, pf[t][s][n], acc[d]);
        }
    schedule<ST * PS * DT, sizeof(T) == 2 ? 2 : 4, 3, W::kParts>();
  };

  // A value that is not finite times a weight of zero is NaN, also in rows that do
  // not see its key. So where outputs are not finite, all is done again with such values
  // as zeros, the first key that has one noted for each dim, and NaN for those
  // outputs whose row sees it.
  // (as code of its own: in one loop, what the second time needs was spilled)
  auto pass = [&](auto second) __attribute__((always_inline)) {
    constexpr bool kSecond = decltype(second)::value;
    top = peak = -INFINITY, shift = 0, sum = 0;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = float16v{};
    if constexpr (kSecond)
      for (uint32_t d = threadIdx.x; d < D; d += 64 * kWaves) first_bad[d] = INT_MAX;
    if (begin < end) load(begin, 0);
    uint32_t buffer = 0;
#pragma unroll 1
    for (uint32_t base = begin; base < end; base += KT) {
      if constexpr (WIDE) loads_done<0>();
      else __syncthreads();
      if (base + KT < end) load(base + KT, buffer ^ 1);
      if constexpr (kSecond) {
        char* const v = lds + buffer * 2 * kTile + kTile;
#pragma unroll 1
        for (uint32_t e = threadIdx.x; e < KT * D; e += 64 * kWaves) {
          const uint32_t r = e / D, d = e % D;
          T* x = reinterpret_cast<T*>(v + r * kRow + ((d / kEach) ^ 2 * (r & 3)) * 16) + d % kEach;
          const float value = (float)*x;
          if (value - value != 0.f) {
            *x = (T)0.f;
            atomicMin(&first_bad[d], (int32_t)(base + r));
          }
        }
        __syncthreads();
      }
      if ((int32_t)base < any_see) compute(base, buffer, (int32_t)base + KT > all_see);
      buffer ^= 1;
    }
  };
  pass(std::false_type{});
  float finite = 0;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) finite = __builtin_fmaf(acc[d][r], 0.f, finite);
  if (__syncthreads_or(finite != 0.f)) {
    pass(std::true_type{});
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (first_bad[d * 32 + r / 4 * 8 + 4 * h + r % 4] < limit) acc[d][r] = NAN;
  }

  __builtin_amdgcn_s_setprio(0);
  sum = add_xor32(sum);
  if (row >= rows) return;
  if (A.splits > 1) {
    const uint32_t item = (block * A.sequences + seq) * A.kv_heads + head;
    const size_t to = ((size_t)item * A.splits + split) * R + (row - row0);
    if (h == 0) A.part_ml[to * 2] = sum == 0.f ? -INFINITY : shift, A.part_ml[to * 2 + 1] = sum;
    if (begin == end) return;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        part_store(A.part_o + to * D + d * 32 + g * 8 + 4 * h,
                   float4v{acc[d][g * 4], acc[d][g * 4 + 1], acc[d][g * 4 + 2], acc[d][g * 4 + 3]});
    return;
  }
  T* const p = output_row<T>(A, P, head, row) + 4 * h;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      put4<T>(p + d * 32 + g * 8, float4v{acc[d][g * 4], acc[d][g * 4 + 1], acc[d][g * 4 + 2], acc[d][g * 4 + 3]}, sum, WIDE);
}

// The stretches of rows joined: one row a workgroup, or as many as have D / 4 lanes.
template <typename T, int D, bool WIDE, bool MANY>
__global__ __launch_bounds__(256) void prompt_merge(PromptArgs A) {
  constexpr uint32_t L = D / 4, kAtOnce = MANY ? 1 : 256 / L;
  const uint32_t item = blockIdx.x / (R / kAtOnce), r = blockIdx.x % (R / kAtOnce) * kAtOnce + (MANY ? 0 : threadIdx.x / L);
  const uint32_t head = item % A.kv_heads, seq = item / A.kv_heads % A.sequences, block = item / A.kv_heads / A.sequences;
  const Prompt P = prompt_of(A, seq);
  const uint32_t row = block * R + r;
  if (P.bad || row >= P.n * A.per) return;
  float sum;
  const size_t part = (size_t)item * A.splits * R + r;
  const float4v x = MANY ? join_many<D>(A.part_o, A.part_ml, part, A.splits, R, &sum) : join_few<D>(A.part_o, A.part_ml, part, A.splits, R, &sum);
  if (!MANY || threadIdx.x < L) put4<T>(output_row<T>(A, P, head, row) + threadIdx.x % L * 4, x, sum, WIDE);
}

// ---------------------------------------------------------------------- host

int check_prompt(const fr_hip_prompt* r) {
  if (!r || r->type > FR_HIP_BF16 || !r->heads || !r->kv_heads || r->heads % r->kv_heads || !r->dim || !isfinite(r->scale))
    return FR_HIP_INVALID;
  if (r->tokens > INT_MAX || r->k_tokens > INT_MAX - (1 << 16)) return FR_HIP_INVALID;
  if (r->tokens && (!r->q || !r->o)) return FR_HIP_INVALID;
  if (r->tokens && r->k_tokens && (!r->k || !r->v)) return FR_HIP_INVALID;
  if (((uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->o) % elem_size(r->type)) return FR_HIP_INVALID;
  if (!r->offsets && (uint64_t)r->sequences * r->max_tokens > r->tokens) return FR_HIP_INVALID;
  if (!r->offsets && !r->k_offsets && (uint64_t)r->sequences * r->max_context > r->k_tokens) return FR_HIP_INVALID;
  if (r->dim != 64 && r->dim != 128 && r->dim != 256) return FR_HIP_UNSUPPORTED;
  if (r->kv_heads > 1024 || r->heads / r->kv_heads > 64) return FR_HIP_UNSUPPORTED;
  if ((uint64_t)r->tokens * r->heads > INT_MAX) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

// How a call is cut: blocks of rows of a sequence, stretches of its keys.
struct PromptCut {
  uint32_t blocks, splits, chunk;
  uint64_t items;
  size_t bytes;
};
PromptCut prompt_cut(const fr_hip_prompt* r) {
  PromptCut c;
  const uint32_t tokens = r->max_tokens < r->tokens ? r->max_tokens : r->tokens;
  const uint32_t context = r->max_context < r->k_tokens ? r->max_context : r->k_tokens;
  c.blocks = (uint32_t)(((uint64_t)tokens * (r->heads / r->kv_heads) + R - 1) / R);
  c.items = (uint64_t)c.blocks * r->sequences * r->kv_heads;
  // Two workgroups for each of 256 compute units, at dim 256 one (two fit a unit there too, but their
  // parts are twice the size); none with less than 256 keys. 512 tokens over 8192 keys, 32 heads of 128
  // over four, bf16: 118 us with the join of four stretches, 227 in one, 140 in two, 119 in six; 128
  // tokens over them of 16 heads of 256 over two: 50 with one workgroup a unit, 62 with two, 60 with a half.
  const uint64_t want = c.items ? (r->dim == 256 ? 1 : 2) * kUnits / c.items : 1, most = (context + 255) / 256;
  uint64_t n = want < most ? want : most;
  n = n < 1 ? 1 : n > 64 ? 64 : n;
  c.chunk = (uint32_t)((context + n * 64 - 1) / (n * 64)) * 64;
  if (!c.chunk) c.chunk = 64;
  c.splits = (context + c.chunk - 1) / c.chunk;
  if (!c.splits) c.splits = 1;
  c.bytes = c.splits > 1 ? (size_t)c.items * c.splits * R * (r->dim + 2) * sizeof(float) : 0;
  return c;
}
// Grids of less than 2^32 threads.
bool prompt_fits(const fr_hip_prompt* r, const PromptCut& c) {
  return c.items * c.splits * 64 * kWaves <= UINT32_MAX && (c.splits == 1 || c.items * R * 256 <= UINT32_MAX);
}

bool prompt_wide(const fr_hip_prompt* r) {
  const int64_t size = (int64_t)elem_size(r->type), each = 16 / size;
  if (((uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->o) % 16) return false;
  for (const int64_t s : {r->q_token, r->q_head, r->k_token, r->k_head, r->v_token, r->v_head, r->o_token, r->o_head})
    if (s % each) return false;
  // A tile's rows are addressed by 32 bits.
  for (const int64_t s : {r->k_token, r->v_token})
    if (s < 0 || s * size > 1 << 24) return false;
  return true;
}

template <typename T, int D, bool WIDE>
int launch_prompt(const PromptArgs& A, const PromptCut& c, hipStream_t s) {
  constexpr size_t kLds = 4ull * kKeys<T, D> * D * sizeof(T);
  static fronk::Devices done;
  if (allow_lds(prompt_attend<T, D, WIDE>, kLds, &done)) return FR_HIP_IO;
  hipLaunchKernelGGL((prompt_attend<T, D, WIDE>), dim3((uint32_t)(c.items * c.splits)), dim3(64 * kWaves), kLds, s, A);
  if (c.splits > 1 && c.items * R < kJoinRows)
    hipLaunchKernelGGL((prompt_merge<T, D, WIDE, true>), dim3((uint32_t)(c.items * R)), dim3(256), 0, s, A);
  else if (c.splits > 1)
    hipLaunchKernelGGL((prompt_merge<T, D, WIDE, false>), dim3((uint32_t)(c.items * R / (1024 / D))), dim3(256), 0, s, A);
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}
template <typename T, bool WIDE>
int launch_dims(unsigned dim, const PromptArgs& A, const PromptCut& c, hipStream_t s) {
  switch (dim) {
    case 64: return launch_prompt<T, 64, WIDE>(A, c, s);
    case 128: return launch_prompt<T, 128, WIDE>(A, c, s);
    default: return launch_prompt<T, 256, WIDE>(A, c, s);
  }
}
template <typename T>
int launch_type(unsigned dim, bool wide, const PromptArgs& A, const PromptCut& c, hipStream_t s) {
  return wide ? launch_dims<T, true>(dim, A, c, s) : launch_dims<T, false>(dim, A, c, s);
}

}  // namespace

extern "C" {

size_t fr_hip_prompt_workspace(const fr_hip_prompt* r) {
  if (check_prompt(r)) return 0;
  const PromptCut c = prompt_cut(r);
  return prompt_fits(r, c) ? c.bytes : 0;
}

int fr_hip_prompt_attend(const fr_hip_prompt* r, void* workspace, size_t bytes, void* stream) {
  int rc = check_prompt(r);
  if (rc) return rc;
  const PromptCut c = prompt_cut(r);
  if (!prompt_fits(r, c)) return FR_HIP_UNSUPPORTED;
  if (c.bytes && (!workspace || bytes < c.bytes || (uintptr_t)workspace % 16)) return FR_HIP_INVALID;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !c.items) return rc;
  PromptArgs A;
  A.q = r->q, A.k = r->k, A.v = r->v, A.o = r->o;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + (c.splits > 1 ? (size_t)c.items * c.splits * R * r->dim : 0);
  A.offsets = r->offsets, A.k_offsets = r->k_offsets, A.status = r->status;
  A.q_token = r->q_token, A.q_head = r->q_head, A.k_token = r->k_token, A.k_head = r->k_head;
  A.v_token = r->v_token, A.v_head = r->v_head, A.o_token = r->o_token, A.o_head = r->o_head;
  A.sequences = r->sequences, A.tokens = r->tokens, A.k_tokens = r->k_tokens;
  A.max_tokens = r->max_tokens, A.max_context = r->max_context, A.kv_heads = r->kv_heads, A.per = r->heads / r->kv_heads;
  A.blocks = c.blocks, A.splits = c.splits, A.chunk = c.chunk, A.scale = r->scale;
  const bool wide = prompt_wide(r);
  switch (r->type) {
    case FR_HIP_F32: return launch_type<float>(r->dim, wide, A, c, s);
    case FR_HIP_F16: return launch_type<_Float16>(r->dim, wide, A, c, s);
    default: return launch_type<__bf16>(r->dim, wide, A, c, s);
  }
}

}  // extern "C"
