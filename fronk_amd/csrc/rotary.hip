// rotary.hip - rotary positions of q and k (fr_hip_rotate).
#include <limits.h>
#include <math.h>

#include "dense.h"

namespace {

struct RotaryArgs {
  const void *q, *k;
  void *q_out, *k_out;
  const int32_t* positions;
  const double* frequencies;
  int64_t q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head;
  uint32_t tokens, heads, all_heads, dim, pairs;
  uint32_t each, at_once;   // tokens a workgroup; of each, the heads that one has
  float magnitude;
  bool in_place;
};

// One workgroup: `each` tokens and `at_once` of their heads (q's, then k's). First the
// tokens' cosines and sines, once for all heads: the angle in turns is formed in 64
// bits and brought to half a turn to either side of zero, which costs a cosine no more
// than fp32's rounding for angles up to 2^27 radians (2^-51 of them beyond). Then one pass
// over the heads, V elements (16 bytes) a step, or single ones where addresses or sizes
// are not of whole 16 bytes. What is rotated is read and written by one lane: in place is safe.
// Results are rounded once, from fp32.
//
// Bound by memory: 4096 tokens of 24 interleaved heads of 128 in fp16 (50 MB) take 9.9 us,
// 5.1 TB/s, as a large copy does, in fp32 17.2; 4096 of 24 heads of 126 in single elements
// 53 (two divisions a step). One token of 18 heads of 256 takes two workgroups 3.9 us: position and
// frequency, the cosine, a head (5.5 with its launch).
template <typename T, bool INTERLEAVED, int V>
__global__ __launch_bounds__(256) void rotary(RotaryArgs A) {
  extern __shared__ __attribute__((aligned(16))) float2v turn[];   // [each][pairs]
  typedef T vec __attribute__((ext_vector_type(V)));
  const uint32_t parts = (A.all_heads + A.at_once - 1) / A.at_once;
  const uint32_t t0 = blockIdx.x / parts * A.each, h0 = blockIdx.x % parts * A.at_once;
  const uint32_t tokens = min(A.each, A.tokens - t0), heads = min(A.at_once, A.all_heads - h0);
  for (uint32_t e = threadIdx.x; e < tokens * A.pairs; e += 256) {
    const double turns = A.positions[t0 + e / A.pairs] * (A.frequencies[e % A.pairs] * 0.15915494309189535);
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    turn[e] = float2v{c * A.magnitude, s * A.magnitude};
  }
  __syncthreads();
  // Steps of a head: of its pairs, then of what is left as it was.
  const uint32_t rotated = INTERLEAVED ? (V == 1 ? A.pairs : 2 * A.pairs / V) : A.pairs / V;
  const uint32_t steps = rotated + (A.in_place ? 0 : (A.dim - 2 * A.pairs) / V);
  for (uint32_t e = threadIdx.x; e < tokens * heads * steps; e += 256) {
    const uint32_t step = e % steps, th = e / steps, t = th / heads, head = h0 + th % heads;
    const bool is_k = head >= A.heads;
    const int64_t token = t0 + t;
    const T* in = is_k ? static_cast<const T*>(A.k) + token * A.k_token + (head - A.heads) * A.k_head
                       : static_cast<const T*>(A.q) + token * A.q_token + head * A.q_head;
    T* out = is_k ? static_cast<T*>(A.k_out) + token * A.ko_token + (head - A.heads) * A.ko_head
                  : static_cast<T*>(A.q_out) + token * A.qo_token + head * A.qo_head;
    const float2v* cs = turn + t * A.pairs;
    if (step >= rotated) {
      const uint32_t d = 2 * A.pairs + (step - rotated) * V;
      *reinterpret_cast<vec*>(out + d) = *reinterpret_cast<const vec*>(in + d);
    } else if (INTERLEAVED && V > 1) {
      const vec x = *reinterpret_cast<const vec*>(in + step * V);
      vec y;
#pragma unroll
      for (int p = 0; p < V / 2; ++p) {
        const float2v r = cs[step * (V / 2) + p];
        const float a = (float)x[2 * p], b = (float)x[2 * p + 1];
        y[2 * p] = (T)(a * r[0] - b * r[1]), y[2 * p + 1] = (T)(a * r[1] + b * r[0]);
      }
      *reinterpret_cast<vec*>(out + step * V) = y;
    } else {
      const uint32_t at = INTERLEAVED ? 2 * step : step * V, on = INTERLEAVED ? 1 : A.pairs;
      const vec x = *reinterpret_cast<const vec*>(in + at), z = *reinterpret_cast<const vec*>(in + at + on);
      vec u, w;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        const float2v r = cs[step * V + p];
        const float a = (float)x[p], b = (float)z[p];
        u[p] = (T)(a * r[0] - b * r[1]), w[p] = (T)(a * r[1] + b * r[0]);
      }
      *reinterpret_cast<vec*>(out + at) = u, *reinterpret_cast<vec*>(out + at + on) = w;
    }
  }
}

// ---------------------------------------------------------------------- host

int check_rotary(const fr_hip_rotary* r) {
  if (!r || r->type > FR_HIP_BF16 || r->flags > FR_HIP_ROTARY_INTERLEAVED || !r->dim || !isfinite(r->magnitude)) return FR_HIP_INVALID;
  if (!r->pairs || r->pairs > r->dim / 2 || r->tokens > INT_MAX) return FR_HIP_INVALID;
  if (r->tokens && (!r->positions || !r->frequencies)) return FR_HIP_INVALID;
  if (r->tokens && ((r->heads && (!r->q || !r->q_out)) || (r->kv_heads && (!r->k || !r->k_out)))) return FR_HIP_INVALID;
  if (((uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->q_out | (uintptr_t)r->k_out) % elem_size(r->type)) return FR_HIP_INVALID;
  if ((uintptr_t)r->frequencies % 8 || (uintptr_t)r->positions % 4) return FR_HIP_INVALID;
  // In place, or apart.
  if (r->heads && r->q == r->q_out && (r->q_token != r->qo_token || r->q_head != r->qo_head)) return FR_HIP_INVALID;
  if (r->kv_heads && r->k == r->k_out && (r->k_token != r->ko_token || r->k_head != r->ko_head)) return FR_HIP_INVALID;
  if (r->dim > 1024 || r->heads > 65535 || r->kv_heads > 65535) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

bool rotary_wide(const fr_hip_rotary* r) {
  const int64_t n = 16 / (int64_t)elem_size(r->type);
  if (((r->flags ? 2 * r->pairs : r->pairs) | r->dim) % n || (r->dim - 2 * r->pairs) % n) return false;
  if (r->heads && (((uintptr_t)r->q | (uintptr_t)r->q_out) % 16 || r->q_token % n || r->q_head % n || r->qo_token % n || r->qo_head % n))
    return false;
  return !r->kv_heads || !(((uintptr_t)r->k | (uintptr_t)r->k_out) % 16 || r->k_token % n || r->k_head % n || r->ko_token % n || r->ko_head % n);
}

template <typename T, bool INTERLEAVED>
void launch_rotary(const RotaryArgs& A, bool wide, uint32_t grid, hipStream_t s) {
  const size_t lds = (size_t)A.each * A.pairs * sizeof(float2v);
  if (wide) hipLaunchKernelGGL((rotary<T, INTERLEAVED, 16 / sizeof(T)>), dim3(grid), dim3(256), lds, s, A);
  else hipLaunchKernelGGL((rotary<T, INTERLEAVED, 1>), dim3(grid), dim3(256), lds, s, A);
}
template <typename T>
void launch_rotary_of(const RotaryArgs& A, bool interleaved, bool wide, uint32_t grid, hipStream_t s) {
  if (interleaved) launch_rotary<T, true>(A, wide, grid, s);
  else launch_rotary<T, false>(A, wide, grid, s);
}

}  // namespace

extern "C" int fr_hip_rotate(const fr_hip_rotary* r, void* stream) {
  int rc = check_rotary(r);
  if (rc) return rc;
  RotaryArgs A;
  A.q = r->q, A.k = r->k, A.q_out = r->q_out, A.k_out = r->k_out;
  A.positions = r->positions, A.frequencies = r->frequencies;
  A.q_token = r->q_token, A.q_head = r->q_head, A.k_token = r->k_token, A.k_head = r->k_head;
  A.qo_token = r->qo_token, A.qo_head = r->qo_head, A.ko_token = r->ko_token, A.ko_head = r->ko_head;
  A.tokens = r->tokens, A.heads = r->heads, A.all_heads = r->heads + r->kv_heads, A.dim = r->dim, A.pairs = r->pairs;
  A.magnitude = r->magnitude;
  A.in_place = (!r->heads || r->q == r->q_out) && (!r->kv_heads || r->k == r->k_out);
  // A cosine and sine for each thread, and what several tokens of few heads have together.
  A.each = r->pairs < 256 ? 256 / r->pairs : 1;
  if (A.each > 16) A.each = 16;
  if (A.each > A.tokens && A.tokens) A.each = A.tokens;
  // Few tokens: their heads over more workgroups, of 256 steps of 16 bytes or more each (16
  // tokens of 136 heads of 64: 10 us in two workgroups, 2.9 in ten).
  const uint32_t groups = (A.tokens + A.each - 1) / A.each, bytes = A.each * A.dim * (uint32_t)elem_size(r->type);
  const uint32_t most = groups && kUnits > groups ? kUnits / groups : 1, least = (8192 + bytes - 1) / bytes;
  A.at_once = (A.all_heads + most - 1) / most;
  if (A.at_once < least) A.at_once = least;
  if (A.at_once > A.all_heads) A.at_once = A.all_heads;
  const uint64_t grid = A.all_heads ? (uint64_t)((A.tokens + A.each - 1) / A.each) * ((A.all_heads + A.at_once - 1) / A.at_once) : 0;
  if (grid * 256 > UINT32_MAX) return FR_HIP_UNSUPPORTED;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !grid) return rc;
  const bool wide = rotary_wide(r), interleaved = r->flags & FR_HIP_ROTARY_INTERLEAVED;
  switch (r->type) {
    case FR_HIP_F32: launch_rotary_of<float>(A, interleaved, wide, (uint32_t)grid, s); break;
    case FR_HIP_F16: launch_rotary_of<_Float16>(A, interleaved, wide, (uint32_t)grid, s); break;
    default: launch_rotary_of<__bf16>(A, interleaved, wide, (uint32_t)grid, s); break;
  }
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}
