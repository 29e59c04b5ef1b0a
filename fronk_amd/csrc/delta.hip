// delta.hip - the gated delta rule (fr_hip_delta_rule).
//
// Per sequence and value head, with a = exp(g) and the state S [dk][dv]:
//     u = beta (v - a S^T k);   S <- a S + k u^T;   o = scale S^T q .
// Columns of S never meet, so the work splits over (sequence, head, columns).
#include <limits.h>
#include <math.h>

#include "bounds.h"
#include "dense.h"

namespace {

struct DeltaArgs {
  const void *q, *k, *v;
  const float *g, *beta;
  void* o;
  const int32_t *offsets, *slot;
  const float* state_in;
  float* state_out;
  uint32_t* status;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head, g_token, beta_token;
  uint32_t sequences, tokens, max_tokens, key_heads, heads, dv, slots;
  float scale;
  bool normalize, wide;   // wide: q, k and v rows and strides are of whole 16 bytes
};

// Sequence i's tokens and state row; false when it is to be skipped (slot -1,
// or an entry out of range, which sets its status bit).
__device__ __forceinline__ bool sequence(const DeltaArgs& A, uint32_t i, uint32_t* first, uint32_t* count, size_t* row) {
  const int32_t s = A.slot ? A.slot[i] : (int32_t)i;
  const int32_t a = A.offsets ? A.offsets[i] : (int32_t)(i * A.max_tokens);
  const int32_t b = A.offsets ? A.offsets[i + 1] : (int32_t)((i + 1) * A.max_tokens);
  const uint32_t bad = fronk::bad_sequence(s, A.slots, a, b, A.tokens, A.max_tokens);
  *first = (uint32_t)a;
  *count = (uint32_t)(b - a);
  *row = (size_t)(s < 0 ? 0 : s);
  if (bad && A.status && threadIdx.x == 0) atomicOr(A.status, bad);
  return !bad && s >= 0;
}

// ------------------------------------------------------------ token by token
//
// One wavefront holds 16 columns of one head's state in registers: lane 4r + c
// keeps rows r * R .. r * R + R - 1 (R = dk / 16) of columns 4c .. 4c + 3. Both
// products over dk are taken of the state before the token,
//     p = S^T k,  w = S^T q,  o = scale (a w + (q . k) u),
// so that a token needs one reduction over the 16 row lanes: two row rotations
// and the two row swaps, no LDS and no barrier.
template <typename T, int DK>
__global__ __launch_bounds__(256) void delta_step(DeltaArgs A) {
  constexpr int R = DK / 16;
  const uint32_t lane = threadIdx.x & 63, waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
  const uint32_t tiles = A.dv / 16, groups = (tiles + waves - 1) / waves;
  const uint32_t tile = blockIdx.x % groups * waves + wave;
  const uint32_t head = blockIdx.x / groups % A.heads, seq = blockIdx.x / groups / A.heads;
  uint32_t first, count;
  size_t row;
  if (!sequence(A, seq, &first, &count, &row) || tile >= tiles) return;
  const uint32_t r = lane >> 2, col = tile * 16 + (lane & 3) * 4, kh = head / (A.heads / A.key_heads);

  const size_t at = ((row * A.heads + head) * DK + r * R) * A.dv + col;
  float s[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float4v x = {0, 0, 0, 0};
    if (A.state_in) x = *reinterpret_cast<const float4v*>(A.state_in + at + (size_t)i * A.dv);
#pragma unroll
    for (int c = 0; c < 4; ++c) s[i][c] = x[c];
  }

  const T* q = static_cast<const T*>(A.q) + (int64_t)first * A.q_token + kh * A.q_head + r * R;
  const T* k = static_cast<const T*>(A.k) + (int64_t)first * A.k_token + kh * A.k_head + r * R;
  const T* v = static_cast<const T*>(A.v) + (int64_t)first * A.v_token + head * A.v_head + col;
  T* o = static_cast<T*>(A.o) + (int64_t)first * A.o_token + head * A.o_head + col;
  const float* g = A.g + (int64_t)first * A.g_token + head;
  const float* beta = A.beta + (int64_t)first * A.beta_token + head;

  // The next token's rows are asked for before this one's reduction.
  float nq[R], nk[R], nv[4], ng = 0, nb = 0;
  auto fetch = [&](uint32_t t) {
    load_row<R>(q + (int64_t)t * A.q_token, A.wide, nq);
    load_row<R>(k + (int64_t)t * A.k_token, A.wide, nk);
    load_row<4>(v + (int64_t)t * A.v_token, A.wide, nv);
    ng = g[(int64_t)t * A.g_token];
    nb = beta[(int64_t)t * A.beta_token];
  };
  if (count) fetch(0);
  for (uint32_t t = 0; t < count; ++t) {
    float kk[R], qq[R], vv[4];
    const float decay = expf(ng), b = nb;
#pragma unroll
    for (int i = 0; i < R; ++i) kk[i] = nk[i], qq[i] = nq[i];
#pragma unroll
    for (int c = 0; c < 4; ++c) vv[c] = nv[c];
    if (t + 1 < count) fetch(t + 1);
    // p[0..3], w[0..3], q.k, |k|^2, |q|^2
    float z[11] = {};
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        z[c] = fmaf(kk[i], s[i][c], z[c]);
        z[4 + c] = fmaf(qq[i], s[i][c], z[4 + c]);
      }
      z[8] = fmaf(qq[i], kk[i], z[8]);
      z[9] = fmaf(kk[i], kk[i], z[9]);
      z[10] = fmaf(qq[i], qq[i], z[10]);
    }
#pragma unroll
    for (int e = 0; e < 11; ++e) z[e] += row_rotate<4>(z[e]);
#pragma unroll
    for (int e = 0; e < 11; ++e) z[e] += row_rotate<8>(z[e]);
#pragma unroll
    for (int e = 0; e < 11; ++e) z[e] = add_xor16(z[e]);
#pragma unroll
    for (int e = 0; e < 11; ++e) z[e] = add_xor32(z[e]);
    const float kn = A.normalize ? 1.f / sqrtf(z[9] + 1e-6f) : 1.f;
    const float qn = (A.normalize ? 1.f / sqrtf(z[10] + 1e-6f) : 1.f) * A.scale;
    float u[4], out[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = b * (vv[c] - decay * (kn * z[c]));
      out[c] = qn * (decay * z[4 + c] + z[8] * kn * u[c]);
      u[c] *= kn;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[i][c] = fmaf(kk[i], u[c], decay * s[i][c]);
    if (r == 0) {
#pragma unroll
      for (int c = 0; c < 4; ++c) o[(int64_t)t * A.o_token + c] = (T)out[c];
    }
  }
  if (A.state_out) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float4v x = {s[i][0], s[i][1], s[i][2], s[i][3]};
      *reinterpret_cast<float4v*>(A.state_out + at + (size_t)i * A.dv) = x;
    }
  }
}

// ---------------------------------------------------------------------- host

int check(const fr_hip_delta* r) {
  if (!r || r->type > FR_HIP_BF16 || (r->flags & ~(unsigned)FR_HIP_DELTA_NORMALIZE)) return FR_HIP_INVALID;
  if (!r->key_heads || !r->heads || r->heads % r->key_heads || !r->key_dim || !r->value_dim) return FR_HIP_INVALID;
  if (!isfinite(r->scale)) return FR_HIP_INVALID;
  if (r->tokens > INT_MAX || r->sequences > INT_MAX || r->slots > INT_MAX) return FR_HIP_INVALID;
  if (!r->offsets && r->tokens != (uint64_t)r->sequences * r->max_tokens) return FR_HIP_INVALID;
  if (!r->slot && r->slots < r->sequences && (r->state_in || r->state_out)) return FR_HIP_INVALID;
  if (r->tokens && r->sequences && (!r->q || !r->k || !r->v || !r->g || !r->beta || !r->o)) return FR_HIP_INVALID;
  if (((uintptr_t)r->state_in | (uintptr_t)r->state_out) % 16) return FR_HIP_INVALID;
  if (((uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->o) % elem_size(r->type)) return FR_HIP_INVALID;
  if (r->key_dim != 64 && r->key_dim != 128 && r->key_dim != 256) return FR_HIP_UNSUPPORTED;
  if (r->value_dim % 16 || r->value_dim > 1024 || r->heads > 65535) return FR_HIP_UNSUPPORTED;
  // One-dimensional grids of (sequence, head, 16 columns).
  if ((uint64_t)r->sequences * r->heads * (r->value_dim / 16) > INT_MAX) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

bool all16(const fr_hip_delta* r) {
  const int64_t n = 16 / (int64_t)elem_size(r->type);
  const int64_t strides[] = {r->q_token, r->q_head, r->k_token, r->k_head, r->v_token, r->v_head};
  for (int64_t s : strides)
    if (s % n) return false;
  return ((uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->v) % 16 == 0;
}

DeltaArgs arguments(const fr_hip_delta* r) {
  DeltaArgs A;
  A.q = r->q, A.k = r->k, A.v = r->v, A.g = r->g, A.beta = r->beta, A.o = r->o;
  A.offsets = r->offsets, A.slot = r->slot, A.state_in = r->state_in, A.state_out = r->state_out, A.status = r->status;
  A.q_token = r->q_token, A.q_head = r->q_head, A.k_token = r->k_token, A.k_head = r->k_head;
  A.v_token = r->v_token, A.v_head = r->v_head, A.o_token = r->o_token, A.o_head = r->o_head;
  A.g_token = r->g_token, A.beta_token = r->beta_token;
  A.sequences = r->sequences, A.tokens = r->tokens, A.max_tokens = r->max_tokens;
  A.key_heads = r->key_heads, A.heads = r->heads, A.dv = r->value_dim;
  // Without state pools a slot only says whether the sequence is skipped.
  A.slots = r->state_in || r->state_out || r->slot ? r->slots : (uint32_t)INT_MAX;
  A.scale = r->scale;
  A.normalize = r->flags & FR_HIP_DELTA_NORMALIZE;
  A.wide = all16(r);
  return A;
}

template <typename T>
void launch_step(const fr_hip_delta* r, const DeltaArgs& A, hipStream_t s) {
  const uint32_t tiles = r->value_dim / 16;
  const uint64_t total = (uint64_t)r->sequences * r->heads * tiles;
  // Single wavefronts while they fit the card's SIMDs once over, so that they
  // spread over all of them; then four neighbouring tiles a workgroup, whose
  // 64-byte rows make whole lines.
  const uint32_t waves = total <= 1024 ? 1 : tiles < 4 ? tiles : 4;
  const dim3 grid((uint32_t)((uint64_t)r->sequences * r->heads * ((tiles + waves - 1) / waves))), block(64 * waves);
  switch (r->key_dim) {
    case 64: hipLaunchKernelGGL((delta_step<T, 64>), grid, block, 0, s, A); break;
    case 128: hipLaunchKernelGGL((delta_step<T, 128>), grid, block, 0, s, A); break;
    default: hipLaunchKernelGGL((delta_step<T, 256>), grid, block, 0, s, A); break;
  }
}

}  // namespace

extern "C" {

size_t fr_hip_delta_workspace(const fr_hip_delta* req) {
  (void)req;
  return 0;
}

int fr_hip_delta_rule(const fr_hip_delta* req, void* workspace, size_t bytes, void* stream) {
  (void)workspace, (void)bytes;
  int rc = check(req);
  if (rc) return rc;
  hipStream_t s;
  unsigned cus;
  rc = fronk::enter(stream, &s, &cus);
  if (rc || !req->sequences) return rc;
  const DeltaArgs A = arguments(req);
  switch (req->type) {
    case FR_HIP_F32: launch_step<float>(req, A, s); break;
    case FR_HIP_F16: launch_step<_Float16>(req, A, s); break;
    default: launch_step<__bf16>(req, A, s); break;
  }
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}

}  // extern "C"
