// kv.hip - the paged 8-bit key/value cache: written (fr_hip_kv_append), read
// back (fr_hip_kv_read) and attended to (fr_hip_kv_attend).
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "bounds.h"
#include "dense.h"
#include "kv.h"

namespace {

__device__ __forceinline__ uint32_t umax_rotate(uint32_t x) {
  uint32_t y = max(x, __builtin_bit_cast(uint32_t, row_rotate<1>(__builtin_bit_cast(float, x))));
  y = max(y, __builtin_bit_cast(uint32_t, row_rotate<2>(__builtin_bit_cast(float, y))));
  y = max(y, __builtin_bit_cast(uint32_t, row_rotate<4>(__builtin_bit_cast(float, y))));
  return max(y, __builtin_bit_cast(uint32_t, row_rotate<8>(__builtin_bit_cast(float, y))));
}

struct KvArgs {
  Cache cache;
  void *k, *v;
  const int32_t* slot;
  uint32_t* status;
  int64_t k_token, k_head, v_token, v_head;
  uint32_t tokens;
  bool wide;
};

// Four of a vector's values as codes, the vector being in L lanes; its exponent.
template <uint32_t L> __device__ __forceinline__ uint32_t quantize(const float (&x)[4], uint32_t* exponent) {
  // The largest magnitude as bits, which order like it and put infinity and NaN
  // on top.
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
  top = umax_rotate(top);
  if constexpr (L > 16) top = max(top, (uint32_t)__shfl_xor((int)top, 16));
  if constexpr (L > 32) top = max(top, (uint32_t)__shfl_xor((int)top, 32));
  const int raw = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);
  const bool finite = top < 0x7f800000u;
  *exponent = finite ? (uint32_t)max(raw, 1) : 255u;
  const float m = __builtin_bit_cast(float, (254u - (uint32_t)max(raw, 1)) << 23);
  const int codes = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * m, x[1] * m, 0, false);
  return finite ? (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * m, x[3] * m, codes, true) : 0u;
}
// ... and as values, at a row of the output.
template <typename T>
__device__ __forceinline__ void put_values(T* out, uint32_t codes, uint32_t exponent, bool wide) {
  const float m = power(exponent);
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const vec4 y = {(T)(a[0] * m), (T)(a[1] * m), (T)(b[0] * m), (T)(b[1] * m)};
  if (wide) {
    *reinterpret_cast<vec4*>(out) = y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = y[i];
  }
}

// One vector (token, head, k or v) to D / 4 lanes: all reads, and writes of few
// tokens.
template <typename T, int D, bool READ>
__global__ __launch_bounds__(256) void kv_single(KvArgs A) {
  constexpr uint32_t L = D / 4;
  const Cache& C = A.cache;
  const uint64_t item = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / L, t = item / 2 / C.heads;
  const uint32_t lane = threadIdx.x % L, h = (uint32_t)(item / 2 % C.heads);
  const bool is_v = item & 1;
  if (t >= A.tokens || !(is_v ? A.v : A.k)) return;   // whole rows of 16 lanes: their reductions stay whole
  uint32_t page = 0, at = 0;
  const int there = fronk::locate(A.slot[t], C.page, C.pages, &page, &at);
  if (there == 2 && A.status && lane == 0) atomicOr(A.status, FR_HIP_BAD_SLOT);
  if (!READ && there != 1) return;
  T* row = (is_v ? static_cast<T*>(A.v) + (int64_t)t * A.v_token + h * A.v_head
                 : static_cast<T*>(A.k) + (int64_t)t * A.k_token + h * A.k_head) + lane * 4;
  uint8_t* v = C.v_codes + v_at(C, page, h, at) + lane * 64;
  uint32_t* k = reinterpret_cast<uint32_t*>(C.k_codes + exp_at(C, page, h, at) * D + lane * 4);
  uint8_t* exponent = (is_v ? C.v_exp : C.k_exp) + exp_at(C, page, h, at);
  if constexpr (READ) {
    uint32_t codes = 0, e = 1;
    if (there == 1) {
      e = *exponent;
      if (is_v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) codes |= (uint32_t)v[16 * i] << (8 * i);
      } else {
        codes = *k;
      }
    }
    put_values(row, codes, e, A.wide);
  } else {
    float x[4];
    load_row<4>(row, A.wide, x);
    uint32_t e;
    const uint32_t codes = quantize<L>(x, &e);
    if (is_v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[16 * i] = (uint8_t)(codes >> (8 * i));
    } else {
      *k = codes;
    }
    if (lane == 0) *exponent = (uint8_t)e;
  }
}

// A prompt: one workgroup writes 16 tokens of one head. The V codes of one dim
// of 16 neighbouring tokens lie together, and those of a token 16 bytes apart, so
// they go through LDS: where the 16 slots are one block of the cache, a lane
// writes a dim's 16 bytes at once; where they are not, four bytes where four
// slots follow each other from a multiple of four, and single bytes otherwise.
// (Reads gather V by single bytes, which share their lines in the caches.) 4096
// tokens of 2 heads of 256: 8.5 us in a row of writes (11.6 in turn with reads), 15.1 by
// single vectors.
constexpr int kWindow = 16;

struct Window {
  uint32_t page[kWindow], at[kWindow];
  int there[kWindow];     // as of fronk::locate
  int run[kWindow];       // 4: first of four that lie together, 1: by itself, 0: one of four, or not there
  bool block;             // all 16 are one block
};
// By the workgroup's first wavefront; to be followed by a barrier.
__device__ __forceinline__ void look_up(const KvArgs& A, uint32_t t0, Window& w) {
  if (threadIdx.x >= 64) return;
  const uint32_t t = threadIdx.x;
  uint32_t page = 0, at = 0;
  const int32_t slot = t < kWindow && t0 + t < A.tokens ? A.slot[t0 + t] : -1;
  const int there = fronk::locate(slot, A.cache.page, A.cache.pages, &page, &at);
  if (there == 2 && A.status) atomicOr(A.status, FR_HIP_BAD_SLOT);
  // Slots that follow each other from a multiple of 4 (16) are of one page.
  const int32_t first = __shfl(slot, (int)(t & ~15u));
  const bool block = __all(t >= kWindow || (there == 1 && slot == first + (int32_t)t && first % kWindow == 0));
  bool four = t + 3 < kWindow && there == 1 && slot % 4 == 0;
  bool of_four = false;
#pragma unroll
  for (int e = 1; e < 4; ++e) four &= __shfl_down(there, e) == 1 && __shfl_down(slot, e) == slot + e;
#pragma unroll
  for (int e = 1; e < 4; ++e) {
    const bool before = __shfl_up((int)four, e);
    of_four |= t >= (uint32_t)e && before;
  }
  if (t < kWindow) {
    w.page[t] = page, w.at[t] = at, w.there[t] = there;
    w.run[t] = there != 1 || of_four ? 0 : four ? 4 : 1;
    if (t == 0) w.block = block;
  }
}

// A vector (token, k or v) to D / 4 lanes, four values each.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_append(KvArgs A) {
  constexpr uint32_t L = D / 4, kAtOnce = 256 / L, kPasses = 2 * kWindow / kAtOnce;
  __shared__ Window w;
  __shared__ __attribute__((aligned(16))) uint8_t v_tile[D][kWindow];
  const Cache& C = A.cache;
  const uint32_t h = blockIdx.x % C.heads, t0 = blockIdx.x / C.heads * kWindow, lane = threadIdx.x % L;
  float x[kPasses][4];
#pragma unroll
  for (uint32_t p = 0; p < kPasses; ++p) {
    const uint32_t vec = p * kAtOnce + threadIdx.x / L, t = vec % kWindow;
    const int64_t token = t0 + t < A.tokens ? t0 + t : A.tokens - 1;
    const T* src = vec / kWindow ? static_cast<const T*>(A.v) + token * A.v_token + h * A.v_head
                                 : static_cast<const T*>(A.k) + token * A.k_token + h * A.k_head;
    load_row<4>(src + lane * 4, A.wide, x[p]);
  }
  look_up(A, t0, w);
  __syncthreads();
#pragma unroll
  for (uint32_t p = 0; p < kPasses; ++p) {
    const uint32_t vec = p * kAtOnce + threadIdx.x / L, t = vec % kWindow;
    const bool is_v = vec / kWindow;
    uint32_t e;
    const uint32_t codes = quantize<L>(x[p], &e);
    if (is_v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v_tile[lane * 4 + i][t] = (uint8_t)(codes >> (8 * i));
    }
    if (w.there[t] != 1) continue;
    const size_t at = exp_at(C, w.page[t], h, w.at[t]);
    if (!is_v) *reinterpret_cast<uint32_t*>(C.k_codes + at * D + lane * 4) = codes;
    if (lane == 0) (is_v ? C.v_exp : C.k_exp)[at] = (uint8_t)e;
  }
  __syncthreads();
  if (w.block) {
    if (threadIdx.x < D)
      *reinterpret_cast<uint4v*>(C.v_codes + v_at(C, w.page[0], h, w.at[0]) + threadIdx.x * 16) =
          *reinterpret_cast<const uint4v*>(v_tile[threadIdx.x]);
    return;
  }
  for (uint32_t u = threadIdx.x; u < D * kWindow; u += 256) {
    const uint32_t d = u % D, t = u / D;
    if (!w.run[t]) continue;
    uint8_t* out = C.v_codes + v_at(C, w.page[t], h, w.at[t]) + d * 16;
    if (w.run[t] == 4) {
      const uint8_t* in = &v_tile[d][t];
      *reinterpret_cast<uint32_t*>(out) = in[0] | in[1] << 8 | in[2] << 16 | (uint32_t)in[3] << 24;
    } else {
      *out = v_tile[d][t];
    }
  }
}

// ------------------------------------------------------------------- attend
//
// One workgroup: one sequence, one cache head, 16 RT rows (query heads of that
// cache head by tokens of the burst) and one stretch of the context; each of
// its four wavefronts takes every fourth tile of 64 tokens with a running
// maximum and sum of its own, joined through LDS at the end. Stretches are
// joined by kv_merge.
//
// Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a
// lane's column is one query row throughout: the row's maximum, sum and
// rescaling are the lane's own scalars (joined over the four lane rows), and P
// goes from the first product's result into the second's B operand without
// leaving the registers. That fixes which tokens a lane holds: row m of K tile
// t is token 16 (m / 4) + 4 t + m % 4, so that lane row j ends up with tokens
// 16 j .. 16 j + 15, the sixteen bytes that the cache's V blocks keep together.
//
// Codes times one are exact in bf16 and fp16. Q is an exact operand too (fp32:
// three bf16 parts); P 2^e is fp32 in two bf16 parts (error 2^-17 of it, below
// a 16-bit output's own rounding), three for fp32 outputs.
//
// 131072 tokens of 2 heads of 256 (134 MB): 26 us, 5.1 TB/s, and 5 to join 128
// stretches. 32 streams of 4 to 8192 tokens, 32 rows of dim 128: 26 us, bound by the
// vector work on the scores.
struct AttendArgs {
  Cache cache;
  const void* q;
  void* o;
  float *part_o, *part_ml;       // [item][split][16 RT][D], [item][split][16 RT][2]
  const int32_t *table, *length;
  uint32_t* status;
  int64_t q_token, q_head, o_token, o_head;
  uint32_t sequences, burst, heads, per, max_context, table_stride, splits, chunk, row_blocks;
  uint32_t page16, reciprocal;   // blocks of 16 tokens a page, and 2^32 by it, rounded down
  float scale;
  bool wide;
};

template <typename T> struct Query {
  typedef bf16x8 frag;
  static constexpr int kParts = 1, kP = 2;
};
template <> struct Query<_Float16> {
  typedef half8v frag;
  static constexpr int kParts = 1, kP = 2;
};
template <> struct Query<float> {
  typedef bf16x8 frag;
  static constexpr int kParts = 3, kP = 3;
};

// Workgroups a compute unit that the registers are for: at dim 256, and with
// fp32's parts at 32 rows, one that prefetches beats two that spill (131072
// tokens at dim 256: 28 us against 33).
template <typename T, int D, int RT>
constexpr int kResident = D == 256 || D * RT * (int)sizeof(T) > 512 ? 1 : 2;
template <typename T, int D, int RT>
__global__ __launch_bounds__(256, (kResident<T, D, RT>)) void kv_attend(AttendArgs A) {
  typedef Query<T> Q;
  typedef typename Q::frag frag;
  constexpr int QP = Q::kParts, PP = Q::kP, KS = D / 32, SEG = D / 64, DT = D / 16, R = 16 * RT;
  constexpr int kPad = D + 4;
  __shared__ union {
    uint4v q[RT][QP][KS][64];
    float o[R][kPad];
  } sh;
  __shared__ float stat[4][R][2];
  const uint32_t lane = threadIdx.x & 63, i = lane & 15, j = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Stretches vary slowest: neighbouring workgroups, which go to different dies,
  // are the same stretch of different items, and contexts that end early leave
  // work for all dies.
  const uint32_t items = A.sequences * A.cache.heads * A.row_blocks;
  const uint32_t split = blockIdx.x / items, item = blockIdx.x % items;
  const uint32_t rb = item % A.row_blocks, head = item / A.row_blocks % A.cache.heads;
  const uint32_t seq = item / A.row_blocks / A.cache.heads;
  const uint32_t rows = A.burst * A.per, row0 = rb * R;

  int32_t len = A.length[seq];
  if (len < 0 || (uint32_t)len > A.max_context) {
    if (A.status && threadIdx.x == 0) atomicOr(A.status, FR_HIP_BAD_LENGTH);
    len = 0;
  }
  const uint32_t begin = split * A.chunk;
  const uint32_t end = min((uint32_t)len, begin + A.chunk);   // chunk * splits < 2^31
  const Cache& C = A.cache;
  const int32_t* table = A.table + (size_t)seq * A.table_stride;

  // The lane's blocks of 16 tokens of a tile, for K by its row, for V by j: what
  // the table says, and where they begin (as exponents are counted). Blocks past
  // the end are taken to be the last one.
  struct Pages {
    int32_t k, v;
  };
  struct Tile {
    size_t k, v;
    bool there;   // v's page
  };
  auto block_of = [&](uint32_t token, uint32_t* page, uint32_t* in) {
    const uint32_t n = (token < end ? token : end - 1) >> 4;
    uint32_t q = __umulhi(n, A.reciprocal), r = n - q * A.page16;   // q or one below
    if (r >= A.page16) ++q, r -= A.page16;
    *page = q, *in = r * 16;
  };
  auto look_up = [&](uint32_t base) {
    uint32_t page, in;
    Pages p;
    block_of(base + (i >> 2) * 16, &page, &in);
    p.k = table[page];
    block_of(base + j * 16, &page, &in);
    p.v = table[page];
    return p;
  };
  bool bad = false;
  auto locate = [&](uint32_t base, Pages p) {
    uint32_t page, in;
    Tile t;
    const bool k = fronk::page_there(p.k, C.pages), v = fronk::page_there(p.v, C.pages);
    block_of(base + (i >> 2) * 16, &page, &in);
    t.k = exp_at(C, k ? (uint32_t)p.k : 0, head, in);
    block_of(base + j * 16, &page, &in);
    t.v = exp_at(C, v ? (uint32_t)p.v : 0, head, in);
    t.there = v;
    bad |= !v;   // (past the end it is the last block's page)
    return t;
  };
  uint4v kc[4][SEG], vc[DT], ke, ve;
  // What is not there is read from somewhere that is, and counts for nothing.
  auto load_k = [&](const Tile& t) {
    const uint8_t* p = C.k_codes + (t.k + (i & 3)) * D + j * 16;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int s = 0; s < SEG; ++s) kc[r][s] = *reinterpret_cast<const uint4v*>(p + r * 4 * D + s * 64);
    ke = *reinterpret_cast<const uint4v*>(C.k_exp + t.v);
  };
  auto load_v = [&](const Tile& t) {
    ve = *reinterpret_cast<const uint4v*>(C.v_exp + t.v);
    const uint8_t* p = C.v_codes + t.v * D + i * 16;
#pragma unroll
    for (int d = 0; d < DT; ++d) vc[d] = *reinterpret_cast<const uint4v*>(p + d * 256);
  };
  uint32_t base = begin + wave * 64;
  Tile now;
  Pages pages;   // of the tile after this one
  if (base < end) {
    const Pages first = look_up(base);
    pages = look_up(base + 256);
    now = locate(base, first);
    load_k(now);
    load_v(now);
  }

  // Q, by operand: step ks of lane (i, j) holds dims 64 (ks / 2) + 16 j + 8 (ks % 2) ..
  if (begin < end) {
    for (uint32_t f = wave; f < RT * KS; f += 4) {
      const uint32_t rt = f / KS, ks = f % KS, row = row0 + rt * 16 + i;
      const uint32_t d = ks / 2 * 64 + j * 16 + ks % 2 * 8;
      float v[8] = {};
      if (row < rows) {
        const T* p = static_cast<const T*>(A.q) + (int64_t)(seq * A.burst + row / A.per) * A.q_token +
                     (int64_t)(head * A.per + row % A.per) * A.q_head + d;
        load_row<8>(p, A.wide, v);
      }
      if constexpr (QP == 3) {
        bf16x8 parts[3];
        split8<3>(v, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) sh.q[rt][p][ks][lane] = __builtin_bit_cast(uint4v, parts[p]);
      } else {
        frag one;
#pragma unroll
        for (int e = 0; e < 8; ++e) one[e] = (decltype(one[0] + one[0]))v[e];
        sh.q[rt][0][ks][lane] = __builtin_bit_cast(uint4v, one);
      }
    }
  }
  __syncthreads();

  uint32_t limit[RT];   // the tokens that this lane's row sees
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const uint32_t row = row0 + rt * 16 + i;
    const int32_t n = len - (int32_t)A.burst + (int32_t)(row / A.per) + 1;
    // (what rows beyond the last would see is not of account)
    limit[rt] = n <= 0 ? 0 : n < len ? (uint32_t)n : (uint32_t)len;
  }
  const uint32_t all_see = (uint32_t)max(len - (int32_t)A.burst + 1, 0);
  float top[RT], sum[RT];
  float4v acc[RT][DT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = -INFINITY, sum[rt] = 0;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[rt][d] = float4v{0, 0, 0, 0};
  }
  const float scale = A.scale * kLog2e;

  // One tile. Its K's registers take the next tile's as soon as the scores are
  // there (with 32 rows of dim 256, where they would be too many, with V's), V's as
  // soon as the outputs are; the tile after that is looked up.
  constexpr bool kEarly = D * RT < 512;
  auto tile = [&](auto more) {
    constexpr bool kMore = decltype(more)::value;
    Tile next = now;
    if constexpr (kMore) {
      next = locate(base + 256, pages);
      pages = look_up(base + 512);
    }
    float4v st[RT][4] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      frag qf[RT][QP];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int p = 0; p < QP; ++p) qf[rt][p] = __builtin_bit_cast(frag, sh.q[rt][p][ks][lane]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const frag a = codes8(kc[t][ks / 2][ks % 2 * 2], kc[t][ks / 2][ks % 2 * 2 + 1], frag{});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int p = QP - 1; p >= 0; --p) st[rt][t] = mma(a, qf[rt][p], st[rt][t]);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = power(ke[t] >> (8 * r) & 255) * scale;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) st[rt][t][r] *= x;
      }
    if constexpr (kMore && kEarly) load_k(next);

    // The tile's end, pages that are not there and tokens that a row does not
    // see: weights of zero, and codes of zero, as they may be NaN.
    const uint32_t tv = base + j * 16;
    const bool masked = !__all(now.there) || base + 64 > all_see;
    if (masked) {
      const bool ok = now.there;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t mask = ok ? fronk::first_bytes((int)end - (int)(tv + 4 * w)) : 0;
#pragma unroll
        for (int d = 0; d < DT; ++d) vc[d][w] &= mask;
        ve[w] &= mask;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!ok || tv + 4 * w + r >= limit[rt]) st[rt][w][r] = -INFINITY;
      }
    }
    bf16x8 pf[RT][2][PP];
#pragma unroll
    for (int rt = RT - 1; rt >= 0; --rt) {
      // A token with infinities is nothing to a row that does not see it. Rows see
      // more the later they are, so the last ones go first.
      if (masked) {
#pragma unroll
        for (int t = 0; t < 4; ++t) ve[t] &= fronk::first_bytes((int)(limit[rt] - (tv + 4 * t)));
      }
      float most = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, st[rt][t][r]);
      most = fmaxf(top[rt], max_xor32(max_xor16(most)));
      const float base_m = most == -INFINITY ? 0.f : most;
      const float alpha = __builtin_amdgcn_exp2f(top[rt] - base_m);
      top[rt] = most;
      float total = 0, w[2][8];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(st[rt][t][r] - base_m);
          total += p;
          w[t / 2][t % 2 * 4 + r] = p * power(ve[t] >> (8 * r) & 255);
        }
      sum[rt] = sum[rt] * alpha + total;
      split8<PP>(w[0], pf[rt][0]);
      split8<PP>(w[1], pf[rt][1]);
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[rt][d] *= alpha;
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bf16x8 a = codes8(vc[d][s * 2], vc[d][s * 2 + 1], bf16x8{});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int p = PP - 1; p >= 0; --p) acc[rt][d] = mma(a, pf[rt][s][p], acc[rt][d]);
      }
    if constexpr (kMore && !kEarly) load_k(next);
    if constexpr (kMore) load_v(next);
    now = next;
    base += 256;
  };
  if (base < end) {
    while (base + 256 < end) tile(std::true_type{});
    tile(std::false_type{});
    if (bad && A.status) atomicOr(A.status, FR_HIP_BAD_PAGE);
  }

  // Join the four wavefronts.
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    sum[rt] = add_xor32(add_xor16(sum[rt]));
    if (j == 0) stat[wave][rt * 16 + i][0] = top[rt], stat[wave][rt * 16 + i][1] = sum[rt];
  }
  __syncthreads();   // also: Q is read no more
  float all[RT], denom[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const uint32_t row = rt * 16 + i;
    all[rt] = fmaxf(fmaxf(stat[0][row][0], stat[1][row][0]), fmaxf(stat[2][row][0], stat[3][row][0]));
    const float m = all[rt] == -INFINITY ? 0.f : all[rt];
    denom[rt] = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) denom[rt] += stat[w][row][1] * __builtin_amdgcn_exp2f(stat[w][row][0] - m);
    const float f = __builtin_amdgcn_exp2f(top[rt] - m);
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[rt][d] *= f;
  }
  for (uint32_t w = 0; w < 4; ++w) {
    if (w == wave) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          float4v* p = reinterpret_cast<float4v*>(&sh.o[rt * 16 + i][d * 16 + 4 * j]);
          *p = w ? *p + acc[rt][d] : acc[rt][d];
        }
    }
    __syncthreads();
  }
  if (A.splits > 1) {
    const size_t at = ((size_t)item * A.splits + split) * R;
    if (wave == 0 && j == 0) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        A.part_ml[(at + rt * 16 + i) * 2] = all[rt];
        A.part_ml[(at + rt * 16 + i) * 2 + 1] = denom[rt];
      }
    }
    if (begin < end)   // kv_merge reads no sums of an empty stretch
      for (uint32_t e = threadIdx.x; e < R * D / 4; e += 256) {
        const uint32_t row = e / (D / 4), d = e % (D / 4) * 4;
        *reinterpret_cast<float4v*>(A.part_o + (at + row) * D + d) = *reinterpret_cast<float4v*>(&sh.o[row][d]);
      }
    return;
  }
  if (wave == 0 && j == 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) stat[0][rt * 16 + i][0] = denom[rt];
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < R * D; e += 256) {
    const uint32_t r = e / D, d = e % D, row = row0 + r;
    if (row >= rows) break;
    const float l = stat[0][r][0];
    T* out = static_cast<T*>(A.o) + (int64_t)(seq * A.burst + row / A.per) * A.o_token +
             (int64_t)(head * A.per + row % A.per) * A.o_head;
    out[d] = (T)(l == 0.f ? 0.f : sh.o[r][d] / l);
  }
}

// The stretches of one row joined, in their order; one workgroup takes L * 4 of
// its dims.
template <typename T, int D, int L>
__global__ __launch_bounds__(256) void kv_merge(AttendArgs A, uint32_t R) {
  constexpr uint32_t G = 256 / L, kSlices = D / 4 / L;
  __shared__ float weight[256], red[4];
  __shared__ float4v part[G][L];
  const uint32_t rows = A.burst * A.per, at_row = blockIdx.x / kSlices;
  const uint32_t row = at_row % rows, head = at_row / rows % A.cache.heads, seq = at_row / rows / A.cache.heads;
  const uint32_t item = (seq * A.cache.heads + head) * A.row_blocks + row / R, at = row % R;
  const uint32_t s = threadIdx.x, wave = s >> 6;
  const uint32_t c = s % L, g = s / L, d = (blockIdx.x % kSlices * L + c) * 4;
  float m = -INFINITY, l = 0;
  if (s < A.splits) {
    const float* p = A.part_ml + (((size_t)item * A.splits + s) * R + at) * 2;
    m = p[0], l = p[1];
  }
  float top = m;
  for (int o = 1; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
  if ((s & 63) == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (top == -INFINITY) top = 0.f;
  const float f = __builtin_amdgcn_exp2f(m - top);   // 0 for an empty stretch
  weight[s] = f;
  l *= f;
  for (int o = 1; o < 64; o *= 2) l += __shfl_xor(l, o);
  __syncthreads();
  if ((s & 63) == 0) red[wave] = l;
  __syncthreads();
  l = (red[0] + red[1]) + (red[2] + red[3]);
  float4v x = {0, 0, 0, 0};
#pragma unroll 4
  for (uint32_t k = g; k < A.splits; k += G) {
    const float w = weight[k];
    if (w != 0.f) x += w * *reinterpret_cast<const float4v*>(A.part_o + (((size_t)item * A.splits + k) * R + at) * D + d);
  }
  part[g][c] = x;
  __syncthreads();
  if (g) return;
  for (uint32_t k = 1; k < G; ++k) x += part[k][c];
  T* out = static_cast<T*>(A.o) + (int64_t)(seq * A.burst + row / A.per) * A.o_token +
           (int64_t)(head * A.per + row % A.per) * A.o_head + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(l == 0.f ? 0.f : x[e] / l);
}

// ---------------------------------------------------------------------- host

int check_tokens(const fr_hip_kv_cache* c, unsigned tokens, unsigned type, const void* k, const void* v, bool both,
                 const int32_t* slot) {
  const int rc = check_cache(c, type);
  if (rc == FR_HIP_INVALID) return rc;
  if (tokens > INT_MAX || (tokens && (!slot || (both ? !k || !v : !k && !v)))) return FR_HIP_INVALID;
  if (((uintptr_t)k | (uintptr_t)v) % elem_size(type)) return FR_HIP_INVALID;
  if (rc) return rc;
  // Grids of less than 2^32 threads.
  return (uint64_t)tokens * c->heads * 2 * (c->dim / 4) > UINT32_MAX - 256 ? FR_HIP_UNSUPPORTED : FR_HIP_OK;
}

// From this many values of K on, 16 tokens are written together. Measured, single
// against together in us: 3.3, 6.9 (256 tokens, 2 heads of 256), 5.8, 4.7 (512, 8
// of 128: 2^19 values), 10.2, 4.5 (4096, 4 of 64), 15.1, 8.5 (4096, 2 of 256).
constexpr uint64_t kTogether = 1 << 19;

template <typename T, int D, bool READ>
void launch_dim(const KvArgs& A, hipStream_t s) {
  const uint64_t vectors = (uint64_t)A.tokens * A.cache.heads;
  const dim3 block(256);
  if constexpr (!READ)
    if (vectors * D >= kTogether) {
      hipLaunchKernelGGL((kv_append<T, D>), dim3((A.tokens + kWindow - 1) / kWindow * A.cache.heads), block, 0, s, A);
      return;
    }
  hipLaunchKernelGGL((kv_single<T, D, READ>), dim3((uint32_t)((vectors * 2 * (D / 4) + 255) / 256)), block, 0, s, A);
}
template <typename T, bool READ>
void launch_tokens(const KvArgs& A, hipStream_t s) {
  switch (A.cache.dim) {
    case 64: launch_dim<T, 64, READ>(A, s); break;
    case 128: launch_dim<T, 128, READ>(A, s); break;
    default: launch_dim<T, 256, READ>(A, s); break;
  }
}

template <bool READ>
int tokens_call(const KvArgs& A, unsigned type, void* stream) {
  hipStream_t s;
  const int rc = fronk::enter(stream, &s);
  if (rc || !A.tokens) return rc;
  switch (type) {
    case FR_HIP_F32: launch_tokens<float, READ>(A, s); break;
    case FR_HIP_F16: launch_tokens<_Float16, READ>(A, s); break;
    default: launch_tokens<__bf16, READ>(A, s); break;
  }
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}

int check_query(const fr_hip_kv_query* r) {
  if (!r) return FR_HIP_INVALID;
  const int rc = check_cache(&r->cache, r->type);
  if (rc == FR_HIP_INVALID) return rc;
  if (!r->burst || !r->heads || r->heads % r->cache.heads || !isfinite(r->scale)) return FR_HIP_INVALID;
  if (r->sequences && (!r->q || !r->o || !r->length || (r->max_context && !r->table))) return FR_HIP_INVALID;
  if (((uintptr_t)r->q | (uintptr_t)r->o) % elem_size(r->type)) return FR_HIP_INVALID;
  if (r->max_context > INT_MAX - (1u << 20)) return FR_HIP_INVALID;
  if (r->table_stride < (r->max_context + r->cache.page - 1) / r->cache.page) return FR_HIP_INVALID;
  if (rc) return rc;
  if (r->burst > 8 || r->heads / r->cache.heads > 64) return FR_HIP_UNSUPPORTED;
  if ((uint64_t)r->sequences * r->burst * r->heads > INT_MAX / 256) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

// How a call is cut: row tiles of a workgroup, blocks of rows, stretches.
struct Cut {
  uint32_t rt, row_blocks, splits, chunk;
  uint64_t items;
  size_t bytes;
};
Cut cut_of(const fr_hip_kv_query* r) {
  Cut c;
  const uint32_t rows = r->burst * (r->heads / r->cache.heads);
  // fp32's parts of 32 rows of dim 256 would not fit the registers.
  c.rt = rows > 16 && !(r->type == FR_HIP_F32 && r->cache.dim == 256) ? 2 : 1;
  c.row_blocks = (rows + 16 * c.rt - 1) / (16 * c.rt);
  c.items = (uint64_t)r->sequences * r->cache.heads * c.row_blocks;
  // About one workgroup for each of 256 compute units (two: 131072 tokens of one
  // stream 34 + 6 us against 28 + 5, a ragged batch of 32 the same), none with less
  // than a tile for each of its wavefronts.
  const uint64_t want = c.items ? (kUnits + c.items - 1) / c.items : 1, most = (r->max_context + 255) / 256;
  uint64_t n = want < most ? want : most;
  n = n < 1 ? 1 : n > 256 ? 256 : n;
  c.chunk = (uint32_t)((r->max_context + n * 256 - 1) / (n * 256)) * 256;
  if (!c.chunk) c.chunk = 256;
  c.splits = (r->max_context + c.chunk - 1) / c.chunk;
  if (!c.splits) c.splits = 1;
  c.bytes = c.splits > 1 ? (size_t)c.items * c.splits * 16 * c.rt * (r->cache.dim + 2) * sizeof(float) : 0;
  return c;
}

template <typename T, int D>
void launch_attend(const AttendArgs& A, const Cut& c, hipStream_t s) {
  const dim3 grid((uint32_t)(c.items * c.splits)), block(256);
  if constexpr (!(std::is_same<T, float>::value && D == 256)) {
    if (c.rt == 1) hipLaunchKernelGGL((kv_attend<T, D, 1>), grid, block, 0, s, A);
    else hipLaunchKernelGGL((kv_attend<T, D, 2>), grid, block, 0, s, A);
  } else {
    hipLaunchKernelGGL((kv_attend<T, D, 1>), grid, block, 0, s, A);
  }
  if (c.splits <= 1) return;
  // Many stretches of few rows: several workgroups a row.
  const uint32_t merges = A.sequences * A.burst * A.heads;
  if (c.splits > 32) hipLaunchKernelGGL((kv_merge<T, D, 4>), dim3(merges * (D / 16)), block, 0, s, A, 16 * c.rt);
  else hipLaunchKernelGGL((kv_merge<T, D, D / 4>), dim3(merges), block, 0, s, A, 16 * c.rt);
}

template <typename T>
void launch_dims(const AttendArgs& A, const Cut& c, hipStream_t s) {
  switch (A.cache.dim) {
    case 64: launch_attend<T, 64>(A, c, s); break;
    case 128: launch_attend<T, 128>(A, c, s); break;
    default: launch_attend<T, 256>(A, c, s); break;
  }
}

}  // namespace

extern "C" {

int fr_hip_kv_append(const fr_hip_kv_write* r, void* stream) {
  if (!r) return FR_HIP_INVALID;
  const int rc = check_tokens(&r->cache, r->tokens, r->type, r->k, r->v, true, r->slot);
  if (rc) return rc;
  const KvArgs A = {cache_of(r->cache), const_cast<void*>(r->k), const_cast<void*>(r->v), r->slot, r->status,
                    r->k_token, r->k_head, r->v_token, r->v_head, r->tokens,
                    rows_wide(r->type, r->k, r->v, r->k_token, r->k_head, r->v_token, r->v_head)};
  return tokens_call<false>(A, r->type, stream);
}

int fr_hip_kv_read(const fr_hip_kv_values* r, void* stream) {
  if (!r) return FR_HIP_INVALID;
  const int rc = check_tokens(&r->cache, r->tokens, r->type, r->k, r->v, false, r->slot);
  if (rc) return rc;
  const KvArgs A = {cache_of(r->cache), r->k, r->v, r->slot, r->status, r->k_token, r->k_head, r->v_token, r->v_head,
                    r->tokens, rows_wide(r->type, r->k, r->v, r->k_token, r->k_head, r->v_token, r->v_head)};
  return tokens_call<true>(A, r->type, stream);
}

size_t fr_hip_kv_workspace(const fr_hip_kv_query* r) { return check_query(r) ? 0 : cut_of(r).bytes; }

int fr_hip_kv_attend(const fr_hip_kv_query* r, void* workspace, size_t bytes, void* stream) {
  int rc = check_query(r);
  if (rc) return rc;
  const Cut c = cut_of(r);
  if (c.bytes && (!workspace || bytes < c.bytes || (uintptr_t)workspace % 16)) return FR_HIP_INVALID;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !r->sequences) return rc;
  AttendArgs A;
  A.cache = cache_of(r->cache);
  A.q = r->q, A.o = r->o, A.table = r->table, A.length = r->length, A.status = r->status;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + (c.splits > 1 ? (size_t)c.items * c.splits * 16 * c.rt * r->cache.dim : 0);
  A.q_token = r->q_token, A.q_head = r->q_head, A.o_token = r->o_token, A.o_head = r->o_head;
  A.sequences = r->sequences, A.burst = r->burst, A.heads = r->heads, A.per = r->heads / r->cache.heads;
  A.max_context = r->max_context, A.table_stride = r->table_stride;
  A.page16 = r->cache.page / 16, A.reciprocal = 0xffffffffu / A.page16;
  A.splits = c.splits, A.chunk = c.chunk, A.row_blocks = c.row_blocks, A.scale = r->scale;
  A.wide = rows_wide(r->type, r->q, r->q, r->q_token, r->q_head, 0, 0);
  switch (r->type) {
    case FR_HIP_F32: launch_dims<float>(A, c, s); break;
    case FR_HIP_F16: launch_dims<_Float16>(A, c, s); break;
    default: launch_dims<__bf16>(A, c, s); break;
  }
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}

}  // extern "C"
