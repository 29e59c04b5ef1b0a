// tree.hip - attention of trees of drafted tokens over the paged 8-bit cache
// (fr_hip_kv_attend_tree).
#include <limits.h>
#include <math.h>

#include "attend.h"
#include "kv.h"

namespace {

struct TreeArgs {
  Cache cache;
  const void* q;
  void* o;
  float *part_o, *part_ml;       // [item][split][R][D], [item][split][R][2]
  const int64_t* tree;
  const int32_t *offsets, *table, *length;
  uint32_t* status;
  int64_t q_token, q_head, o_token, o_head;
  uint32_t sequences, tokens, max_tokens, per, max_context, table_stride, splits, chunk, blocks;
  uint32_t page16, reciprocal;   // blocks of 16 tokens a page, and 2^32 by it, rounded down
  float scale;
  bool wide;
};

// A sequence's drafts: the first one's row of q, how many, and the tokens with them (none:
// a bad length, whose outputs are zeros). By a whole workgroup.
struct Drafts {
  int32_t q0;
  uint32_t n, length, bad;
};
__device__ __forceinline__ Drafts drafts_of(const TreeArgs& A, uint32_t seq) {
  int32_t q0 = seq * A.max_tokens, q1 = q0 + A.max_tokens, before = 0;
  if (A.offsets) {
    q0 = A.offsets[seq], q1 = A.offsets[seq + 1];
    for (uint32_t s = threadIdx.x; s < seq; s += blockDim.x) before = max(before, A.offsets[s]);
  }
  Drafts d = {q0, (uint32_t)(q1 - q0), (uint32_t)A.length[seq], 0};
  if (__syncthreads_or(before > q0) || fronk::bad_sequence(0, 1, q0, q1, A.tokens, A.max_tokens)) d.bad = FR_HIP_BAD_OFFSET;
  else if ((int32_t)d.length < (int32_t)d.n || d.length > A.max_context) d.bad = FR_HIP_BAD_LENGTH, d.length = 0;
  return d;
}
template <typename T> __device__ __forceinline__ T* draft_row(const TreeArgs& A, const Drafts& S, uint32_t head, uint32_t row) {
  return static_cast<T*>(A.o) + (int64_t)(S.q0 + row / A.per) * A.o_token + (int64_t)(head * A.per + row % A.per) * A.o_head;
}

// One workgroup: one sequence, one cache head, R of its rows (query heads of that
// cache head by drafts, draft-major) and one stretch of the context. Products and
// fragments are those of prompt_attend (attend.h); codes become 16-bit operands on
// their way to LDS, once for the four wavefronts' 128 rows. Codes times one are exact
// in bf16 and fp16, a token's powers of two go to its scores and weights.
//
// K in LDS: [token][dim], chunk c of 16 bytes at c ^ (token & 7). V: [block of 16
// tokens][dim][16 tokens], in the order 0-3, 8-11, 4-7, 12-15 in which a half's lanes
// hold weights.
//
// Q is an exact operand (fp32: three bf16 parts); P 2^e is in bf16 parts, of which there
// are as many as keep it well below the output's own rounding but for bf16, where
// half a step of independent weights is no more than that.
template <typename T> struct Row;
template <> struct Row<__bf16> {
  typedef bf16x8 frag;
  static constexpr int kQ = 1, kP = 1;
};
template <> struct Row<_Float16> {
  typedef half8v frag;
  static constexpr int kQ = 1, kP = 2;
};
template <> struct Row<float> {
  typedef bf16x8 frag;
  static constexpr int kQ = 3, kP = 3;
};

// Four codes, those that are no number (which nothing writes) as zeros.
__device__ __forceinline__ uint32_t numbers(uint32_t codes) {
  const uint32_t nan = (((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return codes & ~(nan * 255u);
}

template <int D> constexpr int kTreeKeys = D == 64 ? 64 : 32;
template <typename T, int D> constexpr int kTreeResident = D * sizeof(T) > 512 ? 1 : 2;

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, (kTreeResident<T, D>)) void kv_attend_tree(TreeArgs A) {
  typedef Row<T> Q;
  typedef typename Q::frag frag;
  constexpr int QP = Q::kQ, PP = Q::kP, KT = kTreeKeys<D>, KS = D / 16, ST = KT / 32, DT = D / 32;
  constexpr uint32_t kRow = D * 2, kTile = KT * kRow, kUnits16 = KT * D / 16 / 256;   // 16 codes each, a thread
  extern __shared__ __attribute__((aligned(16))) char lds[];   // [2][K, V][kTile]
  // Per token: the factor of its scores, what is added to them (-infinity: there is no such
  // token), and the power of two of its values.
  __shared__ __attribute__((aligned(16))) float per_token[2][3][KT];
  __shared__ uint32_t bad_drafts[2];   // drafts whose values are not finite

  const uint32_t lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Cache& C = A.cache;
  // Stretches vary slowest, so that contexts that end early leave work for all dies.
  uint32_t at = blockIdx.x;
  const uint32_t head = at % C.heads;
  at /= C.heads;
  const uint32_t block = at % A.blocks;
  at /= A.blocks;
  const uint32_t seq = at % A.sequences, split = at / A.sequences;
  if (threadIdx.x < 2) bad_drafts[threadIdx.x] = 0;
  const Drafts S = drafts_of(A, seq);
  if (S.bad) {
    if (A.status && threadIdx.x == 0) atomicOr(A.status, S.bad);
    if (S.bad == FR_HIP_BAD_OFFSET) return;
  }
  const uint32_t rows = S.n * A.per, row0 = block * R;
  if (row0 >= rows) return;
  const uint32_t begin = split * A.chunk, end = max(begin, min(S.length, begin + A.chunk));
  const uint32_t prefix = S.length - S.n;
  const uint32_t wave_row = row0 + wave * 32, row = wave_row + i;
  const uint64_t seen = row < rows ? (uint64_t)A.tree[S.q0 + row / A.per] & (~0ull >> (64 - S.n)) : 0;
  const int32_t* const table = A.table + (size_t)seq * A.table_stride;

  // Q: lane (i, h) of step s holds row i's dims 16 s + 8 h ..
  frag qf[QP][KS];
  {
    const uint32_t r = min(row, rows - 1);
    const T* p = static_cast<const T*>(A.q) + (int64_t)(S.q0 + r / A.per) * A.q_token +
                 (int64_t)(head * A.per + r % A.per) * A.q_head + h * 8;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
      load_row<8>(p + s * 16, A.wide, x);
      if constexpr (QP == 3) {
        bf16x8 parts[3];
        split8<3>(x, parts);
#pragma unroll
        for (int q = 0; q < 3; ++q) qf[q][s] = parts[q];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[0][s][e] = (T)x[e];
      }
    }
  }

  // A thread's units of a tile: 16 codes of a K token, 16 tokens of a V dim; each
  // wavefront's are of one block of 16 tokens. Blocks past the end are taken to be the
  // last one.
  struct Pages {
    int32_t k[kUnits16], v[kUnits16], e;
  };
  auto place_of = [&](uint32_t n, uint32_t* page, uint32_t* in) {   // of the n-th block
    n = min(n, (end - 1) >> 4);
    uint32_t q = __umulhi(n, A.reciprocal), r = n - q * A.page16;   // q or one below
    if (r >= A.page16) ++q, r -= A.page16;
    *page = q, *in = r * 16;
  };
  const uint32_t e_token = threadIdx.x % KT;
  auto k_block = [&](uint32_t base, uint32_t u) { return (base >> 4) + (wave * 64 + u * 256) / D; };   // (D / 16 units a token)
  auto v_block = [&](uint32_t base, uint32_t u) { return (base >> 4) + (wave * 64 + u * 256) / D; };
  auto look_up = [&](uint32_t base) {
    Pages p;
    uint32_t page, in;
#pragma unroll
    for (uint32_t u = 0; u < kUnits16; ++u) {
      place_of(k_block(base, u), &page, &in);
      p.k[u] = table[page];
      place_of(v_block(base, u), &page, &in);
      p.v[u] = table[page];
    }
    place_of((base + e_token) >> 4, &page, &in);
    p.e = table[page];
    return p;
  };
  uint4v kc[kUnits16], vc[kUnits16];
  uint32_t ke, ve;
  bool k_there[kUnits16], v_there[kUnits16], e_there, missing = false;
  auto load = [&](uint32_t base, const Pages& p) {
    uint32_t page, in;
#pragma unroll
    for (uint32_t u = 0; u < kUnits16; ++u) {
      place_of(k_block(base, u), &page, &in);
      k_there[u] = fronk::page_there(p.k[u], C.pages);
      const uint32_t unit = threadIdx.x + u * 256;
      kc[u] = *reinterpret_cast<const uint4v*>(C.k_codes + exp_at(C, k_there[u] ? p.k[u] : 0, head, in) * D + (unit / (D / 16) % 16) * D + unit % (D / 16) * 16);
      place_of(v_block(base, u), &page, &in);
      v_there[u] = fronk::page_there(p.v[u], C.pages);
      vc[u] = *reinterpret_cast<const uint4v*>(C.v_codes + exp_at(C, v_there[u] ? p.v[u] : 0, head, in) * D + unit % D * 16);
    }
    place_of((base + e_token) >> 4, &page, &in);
    e_there = fronk::page_there(p.e, C.pages);
    const size_t e = exp_at(C, e_there ? p.e : 0, head, in) + e_token % 16;
    ke = C.k_exp[e], ve = C.v_exp[e];
    missing |= !e_there;
  };
  // ... to LDS, as operands. What is not there, or past the end, is zeros.
  const float scale = A.scale * kLog2e;
  auto store = [&](uint32_t base, uint32_t buffer) {
    char* const to = lds + buffer * 2 * kTile;
    const bool drafts = base + KT > prefix;
#pragma unroll
    for (uint32_t u = 0; u < kUnits16; ++u) {
      const uint32_t unit = threadIdx.x + u * 256, token = unit / (D / 16), c = unit % (D / 16) * 2;
      if (!k_there[u] || base + token >= end) kc[u] = uint4v{0, 0, 0, 0};
      const uint32_t first = unit / D * 16;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        vc[u][w] &= v_there[u] ? fronk::first_bytes((int)end - (int)(base + first + 4 * w)) : 0;
        if (drafts) kc[u][w] = numbers(kc[u][w]), vc[u][w] = numbers(vc[u][w]);
      }
      *reinterpret_cast<frag*>(to + token * kRow + (c ^ (token & 7)) * 16) = codes8(kc[u][0], kc[u][1], frag{});
      *reinterpret_cast<frag*>(to + token * kRow + ((c + 1) ^ (token & 7)) * 16) = codes8(kc[u][2], kc[u][3], frag{});
      char* const v = to + kTile + unit * 32;
      *reinterpret_cast<bf16x8*>(v) = codes8(vc[u][0], vc[u][2], bf16x8{});
      *reinterpret_cast<bf16x8*>(v + 16) = codes8(vc[u][1], vc[u][3], bf16x8{});
    }
    if (threadIdx.x < KT) {
      const uint32_t token = base + threadIdx.x;
      const bool there = e_there && token < end;
      // A draft whose values are not finite (zero codes) makes the rows that see it NaN at the end.
      const bool bad = there && token >= prefix && ve == 255;
      if (bad) atomicOr(&bad_drafts[(token - prefix) / 32], 1u << (token - prefix) % 32);
      per_token[buffer][0][threadIdx.x] = there ? power(ke) * scale : 0.f;
      per_token[buffer][1][threadIdx.x] = there ? 0.f : -INFINITY;
      per_token[buffer][2][threadIdx.x] = there && !bad ? power(ve) : 0.f;
    }
  };

  uint32_t k_at[4];   // as in prompt_attend
#pragma unroll
  for (uint32_t s = 0; s < 4; ++s) k_at[s] = i * kRow + ((2 * s + h) ^ (i & 7)) * 16;
  const uint32_t v_at = kTile + i * 32 + h * 16;
  float top = -INFINITY, shift = 0, sum = 0;
  float16v acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = float16v{};

  auto compute = [&](uint32_t base, uint32_t buffer) {
    const char* const tile = lds + buffer * 2 * kTile;
    float16v st[ST];
#pragma unroll
    for (int t = 0; t < ST; ++t) {
      st[t] = float16v{};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const frag a = *reinterpret_cast<const frag*>(tile + k_at[s % 4] + t * 32 * kRow + s / 4 * 128);
#pragma unroll
        for (int q = QP - 1; q >= 0; --q) st[t] = mma32(a, qf[q][s], st[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4v f = *reinterpret_cast<const float4v*>(&per_token[buffer][0][t * 32 + 8 * g + 4 * h]);
        const float4v b = *reinterpret_cast<const float4v*>(&per_token[buffer][1][t * 32 + 8 * g + 4 * h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) st[t][g * 4 + e] = __builtin_fmaf(st[t][g * 4 + e], f[e], b[e]);
      }
    if (base + KT > prefix) {
#pragma unroll
      for (int t = 0; t < ST; ++t) {
        // Which of 32 tokens the row sees: all before the drafts, and its own of those.
        const int32_t first = (int32_t)(base + t * 32 - prefix);
        const uint32_t bits = first <= -32 ? ~0u : first >= 64 ? 0u : first < 0 ? (uint32_t)(seen << -first) | ~(~0u << -first) : (uint32_t)(seen >> first);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!(bits >> (4 * h) & 1u << (8 * (r / 4) + r % 4))) st[t][r] = -INFINITY;
      }
    }
    float most = -INFINITY;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, st[t][r]);
    most = max_xor32(most);
    if (__any(most > top + 8.f)) {   // (as in prompt_attend)
      const float now = fmaxf(top, most), to = now == -INFINITY ? 0.f : now;
      const float f = __builtin_amdgcn_exp2f(top - to);
      top = now, shift = to, sum *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f;
    }
    bf16x8 pf[ST][2][PP];
    float total = 0;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float w[8];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const float4v f = *reinterpret_cast<const float4v*>(&per_token[buffer][2][t * 32 + s * 16 + 8 * g + 4 * h]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(st[t][s * 8 + g * 4 + e] - shift);
            total += p;
            w[g * 4 + e] = p * f[e];
          }
        }
        split8<PP>(w, pf[t][s]);
      }
    sum += total;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const bf16x8 a = *reinterpret_cast<const bf16x8*>(tile + v_at + ((t * 2 + s) * D + d * 32) * 32);
#pragma unroll
          for (int p = PP - 1; p >= 0; --p) acc[d] = mma32(a, pf[t][s][p], acc[d]);
        }
  };

  if (begin < end) {
    Pages pages = look_up(begin);
    load(begin, pages);
    pages = look_up(begin + KT);
    store(begin, 0);
    uint32_t buffer = 0;
    for (uint32_t base = begin; base < end; base += KT) {
      __syncthreads();
      load(base + KT, pages);   // (past the end the last block once more: a load under a condition is waited for)
      pages = look_up(base + 2 * KT);
      if (wave_row < rows) compute(base, buffer);
      if (base + KT < end) store(base + KT, buffer ^ 1);
      buffer ^= 1;
    }
    if (missing && A.status) atomicOr(A.status, FR_HIP_BAD_PAGE);
  }
  __syncthreads();   // bad_drafts

  sum = add_xor32(sum);
  if (row >= rows) return;
  if (seen & (bad_drafts[0] | (uint64_t)bad_drafts[1] << 32)) sum = NAN;
  if (A.splits > 1) {
    const uint32_t item = (seq * A.blocks + block) * C.heads + head;
    const size_t to = ((size_t)item * A.splits + split) * R + (row - row0);
    if (h == 0) A.part_ml[to * 2] = sum == 0.f ? -INFINITY : shift, A.part_ml[to * 2 + 1] = sum;
    if (begin == end) return;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4v*>(A.part_o + to * D + d * 32 + g * 8 + 4 * h) =
            float4v{acc[d][g * 4], acc[d][g * 4 + 1], acc[d][g * 4 + 2], acc[d][g * 4 + 3]};
    return;
  }
  T* const p = draft_row<T>(A, S, head, row) + 4 * h;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      put4<T>(p + d * 32 + g * 8, float4v{acc[d][g * 4], acc[d][g * 4 + 1], acc[d][g * 4 + 2], acc[d][g * 4 + 3]}, sum, A.wide);
}

// The stretches of a row joined, in their order: D / 4 lanes a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void tree_merge(TreeArgs A) {
  constexpr uint32_t L = D / 4, kAtOnce = 256 / L;
  const uint32_t item = blockIdx.x / (R / kAtOnce), r = blockIdx.x % (R / kAtOnce) * kAtOnce + threadIdx.x / L;
  const uint32_t head = item % A.cache.heads, block = item / A.cache.heads % A.blocks, seq = item / A.cache.heads / A.blocks;
  const Drafts S = drafts_of(A, seq);
  const uint32_t row = block * R + r, d = threadIdx.x % L * 4;
  if (S.bad == FR_HIP_BAD_OFFSET || row >= S.n * A.per) return;
  float sum;
  const float4v x = join<D>(A.part_o, A.part_ml, (size_t)item * A.splits * R + r, A.splits, d, &sum);
  put4<T>(draft_row<T>(A, S, head, row) + d, x, sum, A.wide);
}

// ---------------------------------------------------------------------- host

int check_tree(const fr_hip_kv_tree* r) {
  if (!r) return FR_HIP_INVALID;
  const int rc = check_cache(&r->cache, r->type);
  if (rc == FR_HIP_INVALID) return rc;
  if (!r->heads || r->heads % r->cache.heads || !isfinite(r->scale)) return FR_HIP_INVALID;
  if (r->tokens > INT_MAX) return FR_HIP_INVALID;
  if (r->tokens && r->sequences && (!r->q || !r->o || !r->tree || !r->length || (r->max_context && !r->table))) return FR_HIP_INVALID;
  if (!r->offsets && (uint64_t)r->sequences * r->max_tokens > r->tokens) return FR_HIP_INVALID;
  if (((uintptr_t)r->q | (uintptr_t)r->o) % elem_size(r->type) || (uintptr_t)r->tree % 8) return FR_HIP_INVALID;
  if (r->max_context > INT_MAX - (1u << 20)) return FR_HIP_INVALID;
  if (r->table_stride < (r->max_context + r->cache.page - 1) / r->cache.page) return FR_HIP_INVALID;
  if (rc) return rc;
  if (r->max_tokens > 64 || r->heads / r->cache.heads > 64) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

// How a call is cut: blocks of rows of a sequence, stretches of the context.
struct TreeCut {
  uint32_t blocks, splits, chunk;
  uint64_t items;
  size_t bytes;
};
TreeCut tree_cut(const fr_hip_kv_tree* r) {
  TreeCut c;
  const uint32_t drafts = r->max_tokens < r->tokens ? r->max_tokens : r->tokens;
  c.blocks = (drafts * (r->heads / r->cache.heads) + R - 1) / R;
  c.items = (uint64_t)c.blocks * r->sequences * r->cache.heads;
  const uint64_t want = c.items ? (kUnits + c.items - 1) / c.items : 1, most = (r->max_context + 255) / 256;
  uint64_t n = want < most ? want : most;
  n = n < 1 ? 1 : n > 256 ? 256 : n;
  c.chunk = (uint32_t)((r->max_context + n * 64 - 1) / (n * 64)) * 64;
  if (!c.chunk) c.chunk = 64;
  c.splits = (r->max_context + c.chunk - 1) / c.chunk;
  if (!c.splits) c.splits = 1;
  c.bytes = c.splits > 1 ? (size_t)c.items * c.splits * R * (r->cache.dim + 2) * sizeof(float) : 0;
  return c;
}
// Grids of less than 2^32 threads.
bool tree_fits(const fr_hip_kv_tree* r, const TreeCut& c) {
  return c.items * c.splits * 64 * kWaves <= UINT32_MAX && (c.splits == 1 || c.items * R * (r->cache.dim / 4) <= UINT32_MAX);
}

template <typename T, int D>
int launch_tree(const TreeArgs& A, const TreeCut& c, hipStream_t s) {
  constexpr size_t kLds = 8ull * kTreeKeys<D> * D;
  static fronk::Devices done;
  if (allow_lds(kv_attend_tree<T, D>, kLds, &done)) return FR_HIP_IO;
  hipLaunchKernelGGL((kv_attend_tree<T, D>), dim3((uint32_t)(c.items * c.splits)), dim3(64 * kWaves), kLds, s, A);
  if (c.splits > 1) hipLaunchKernelGGL((tree_merge<T, D>), dim3((uint32_t)(c.items * R / (1024 / D))), dim3(256), 0, s, A);
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}
template <typename T>
int launch_dims(const TreeArgs& A, const TreeCut& c, hipStream_t s) {
  switch (A.cache.dim) {
    case 64: return launch_tree<T, 64>(A, c, s);
    case 128: return launch_tree<T, 128>(A, c, s);
    default: return launch_tree<T, 256>(A, c, s);
  }
}

}  // namespace

extern "C" {

size_t fr_hip_tree_workspace(const fr_hip_kv_tree* r) {
  if (check_tree(r)) return 0;
  const TreeCut c = tree_cut(r);
  return tree_fits(r, c) ? c.bytes : 0;
}

int fr_hip_kv_attend_tree(const fr_hip_kv_tree* r, void* workspace, size_t bytes, void* stream) {
  int rc = check_tree(r);
  if (rc) return rc;
  const TreeCut c = tree_cut(r);
  if (!tree_fits(r, c)) return FR_HIP_UNSUPPORTED;
  if (c.bytes && (!workspace || bytes < c.bytes || (uintptr_t)workspace % 16)) return FR_HIP_INVALID;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !c.items) return rc;
  TreeArgs A;
  A.cache = cache_of(r->cache);
  A.q = r->q, A.o = r->o, A.tree = r->tree, A.offsets = r->offsets, A.table = r->table, A.length = r->length;
  A.status = r->status;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + (c.splits > 1 ? (size_t)c.items * c.splits * R * r->cache.dim : 0);
  A.q_token = r->q_token, A.q_head = r->q_head, A.o_token = r->o_token, A.o_head = r->o_head;
  A.sequences = r->sequences, A.tokens = r->tokens, A.max_tokens = r->max_tokens, A.per = r->heads / r->cache.heads;
  A.max_context = r->max_context, A.table_stride = r->table_stride, A.splits = c.splits, A.chunk = c.chunk, A.blocks = c.blocks;
  A.page16 = r->cache.page / 16, A.reciprocal = 0xffffffffu / A.page16;
  A.scale = r->scale;
  A.wide = rows_wide(r->type, r->q, r->o, r->q_token, r->q_head, r->o_token, r->o_head);
  switch (r->type) {
    case FR_HIP_F32: return launch_dims<float>(A, c, s);
    case FR_HIP_F16: return launch_dims<_Float16>(A, c, s);
    default: return launch_dims<__bf16>(A, c, s);
  }
}

}  // extern "C"
