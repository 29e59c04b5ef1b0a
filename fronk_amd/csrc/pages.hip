// pages.hip - what is held in the paged 8-bit cache moved within it: single tokens
// (fr_hip_kv_move) and whole pages (fr_hip_kv_copy).
#include <limits.h>

#include "kv.h"

namespace {

constexpr uint32_t kMoves = 64;   // of a group, at most

struct MoveArgs {
  Cache cache;
  const int32_t *source, *target;
  uint32_t* status;
  uint32_t groups, moves;
};

// One workgroup: the K or the V of one head of one group of up to M moves, all of which it
// reads before it writes any. A move's codes are D / 4 dwords of K, or D single bytes of
// V, 16 apart; a thread's are in registers, all loaded before the first is waited for.
//
// One path of 6 tokens takes 3.4 us (4.8 with its launch), three latencies: the slots, the
// codes and their exponents, the writes. 128 groups of up to 24 tokens, 8 heads of 128: 11.2
// us, bound by V's lines: a token's 128 codes of a head lie in 2 KB, which are fetched
// and written back for them.
constexpr size_t kNowhere = ~(size_t)0;
template <typename T, int U, int APART, int M>
__device__ __forceinline__ void move_codes(T* codes, const size_t* from, const size_t* to) {
  constexpr uint32_t N = (M * U + 255) / 256;
  T held[N];
  size_t source[N], target[N];
#pragma unroll
  for (uint32_t n = 0; n < N; ++n) {
    const uint32_t u = threadIdx.x + n * 256, move = min(u / U, M - 1u);
    source[n] = from[move], target[n] = u < M * U ? to[move] : kNowhere;
  }
#pragma unroll
  for (uint32_t n = 0; n < N; ++n)
    if (target[n] != kNowhere) held[n] = codes[source[n] / sizeof(T) + (threadIdx.x + n * 256) % U * APART];
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): all is read
  __syncthreads();
#pragma unroll
  for (uint32_t n = 0; n < N; ++n)
    if (target[n] != kNowhere) codes[target[n] / sizeof(T) + (threadIdx.x + n * 256) % U * APART] = held[n];
}
template <int D, int M>
__global__ __launch_bounds__(256) void kv_move(MoveArgs A) {
  __shared__ size_t from[M], to[M];   // of the codes
  const Cache& C = A.cache;
  const bool is_v = blockIdx.x & 1;
  const uint32_t head = blockIdx.x / 2 % C.heads, group = blockIdx.x / 2 / C.heads;
  uint8_t* const exponents = is_v ? C.v_exp : C.k_exp;
  size_t to_exp = 0;
  uint32_t exponent = 0;
  bool there = false;
  if (threadIdx.x < M) {
    uint32_t p0 = 0, a0 = 0, p1 = 0, a1 = 0;
    if (threadIdx.x < A.moves) {
      const size_t at = (size_t)group * A.moves + threadIdx.x;
      const int32_t source = A.source[at], target = A.target[at];
      const int s = fronk::locate(source, C.page, C.pages, &p0, &a0), t = fronk::locate(target, C.page, C.pages, &p1, &a1);
      if ((s == 2 || t == 2) && A.status) atomicOr(A.status, FR_HIP_BAD_SLOT);
      there = s == 1 && t == 1;
    }
    const size_t from_exp = there ? exp_at(C, p0, head, a0) : 0;
    to_exp = there ? exp_at(C, p1, head, a1) : 0;
    from[threadIdx.x] = !there ? 0 : is_v ? v_at(C, p0, head, a0) : from_exp * D;
    to[threadIdx.x] = !there ? kNowhere : is_v ? v_at(C, p1, head, a1) : to_exp * D;
    exponent = exponents[from_exp];
  }
  __syncthreads();
  // (Its barrier is also the exponents': they are read by then and not yet written.)
  if (is_v) move_codes<uint8_t, D, 16, M>(C.v_codes, from, to);
  else move_codes<uint32_t, D / 4, 1, M>(reinterpret_cast<uint32_t*>(C.k_codes), from, to);
  if (there) exponents[to_exp] = (uint8_t)exponent;
}

struct CopyArgs {
  Cache cache;
  const int32_t *source, *target;
  uint32_t* status;
  uint32_t count, parts;   // workgroups a page
};
constexpr uint32_t kVectors = 8;   // of 16 bytes, a thread

// One workgroup: up to 32 KB of a page, which lies together in each of the cache's four
// tensors, all loads before the first store. 1024 pages of 64 tokens, two heads of 256 (135 MB
// read and written): 21.3 us by itself, as part of it stays in the card's 256 MB cache, 30.8 in
// a row with others, where a copy at its largest rate takes 26.
__global__ __launch_bounds__(256) void kv_copy(CopyArgs A) {
  const Cache& C = A.cache;
  const uint32_t entry = blockIdx.x / A.parts, part = blockIdx.x % A.parts;
  const int32_t source = A.source[entry], target = A.target[entry];
  const bool from = fronk::page_there(source, C.pages), to = fronk::page_there(target, C.pages);
  if (!from || !to) {   // (-1: skipped)
    if (((!from && source != -1) || (!to && target != -1)) && A.status && threadIdx.x == 0) atomicOr(A.status, FR_HIP_BAD_PAGE);
    return;
  }
  const uint32_t exps = C.heads * C.page / 16, codes = exps * C.dim;   // of 16 bytes
  const uint32_t all = 2 * (codes + exps);
  uint4v held[kVectors];
  auto place = [&](uint32_t u, int32_t page) -> uint4v* {
    uint8_t* const base = u < codes ? C.k_codes : u < 2 * codes ? C.v_codes : u < 2 * codes + exps ? C.k_exp : C.v_exp;
    const uint32_t in = u < codes ? u : u < 2 * codes ? u - codes : u < 2 * codes + exps ? u - 2 * codes : u - 2 * codes - exps;
    return reinterpret_cast<uint4v*>(base) + (size_t)page * (u < 2 * codes ? codes : exps) + in;
  };
  const uint32_t first = part * kVectors * 256 + threadIdx.x;
#pragma unroll
  for (uint32_t n = 0; n < kVectors; ++n) held[n] = *place(min(first + n * 256, all - 1), source);
#pragma unroll
  for (uint32_t n = 0; n < kVectors; ++n)
    if (first + n * 256 < all) *place(first + n * 256, target) = held[n];
}

// ---------------------------------------------------------------------- host

int check_moves(const fr_hip_kv_cache* c, uint64_t n, const int32_t* source, const int32_t* target) {
  const int rc = check_cache(c, FR_HIP_F32);
  if (rc == FR_HIP_INVALID || n > INT_MAX || (n && (!source || !target))) return FR_HIP_INVALID;
  return rc;
}

template <int D>
void launch_move(const MoveArgs& A, uint32_t grid, hipStream_t s) {
  // (4 moves of one group take 3.0 us, of 128 groups 5.0, in the kernel for 64 4.0 and 11.1;
  // 16 moves in that for 32 3.7 and 11.2, in that for 64 4.2 and 13.3)
  if (A.moves <= 8) hipLaunchKernelGGL((kv_move<D, 8>), dim3(grid), dim3(256), 0, s, A);
  else if (A.moves <= 32) hipLaunchKernelGGL((kv_move<D, 32>), dim3(grid), dim3(256), 0, s, A);
  else hipLaunchKernelGGL((kv_move<D, kMoves>), dim3(grid), dim3(256), 0, s, A);
}

}  // namespace

extern "C" {

int fr_hip_kv_move(const fr_hip_kv_moves* r, void* stream) {
  if (!r) return FR_HIP_INVALID;
  int rc = check_moves(&r->cache, (uint64_t)r->groups * r->moves, r->source, r->target);
  if (rc) return rc;
  const uint64_t grid = (uint64_t)r->groups * r->cache.heads * 2;
  if (r->moves > kMoves || grid * 256 > UINT32_MAX) return FR_HIP_UNSUPPORTED;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !grid || !r->moves) return rc;
  const MoveArgs A = {cache_of(r->cache), r->source, r->target, r->status, r->groups, r->moves};
  switch (A.cache.dim) {
    case 64: launch_move<64>(A, (uint32_t)grid, s); break;
    case 128: launch_move<128>(A, (uint32_t)grid, s); break;
    default: launch_move<256>(A, (uint32_t)grid, s); break;
  }
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}

int fr_hip_kv_copy(const fr_hip_kv_copies* r, void* stream) {
  if (!r) return FR_HIP_INVALID;
  int rc = check_moves(&r->cache, r->count, r->source, r->target);
  if (rc) return rc;
  const uint64_t vectors = 2 * (uint64_t)r->cache.heads * (r->cache.page / 16) * (r->cache.dim + 1);
  const uint64_t parts = (vectors + kVectors * 256 - 1) / (kVectors * 256);
  if (r->count * parts * 256 > UINT32_MAX) return FR_HIP_UNSUPPORTED;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !r->count) return rc;
  const CopyArgs A = {cache_of(r->cache), r->source, r->target, r->status, r->count, (uint32_t)parts};
  hipLaunchKernelGGL(kv_copy, dim3((uint32_t)(r->count * parts)), dim3(256), 0, s, A);
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}

}  // extern "C"
