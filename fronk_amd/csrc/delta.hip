// delta.hip - the gated delta rule (fr_hip_delta_rule).
//
// Per sequence and value head, with a = exp(g) and the state S [dk][dv]:
//     u = beta (v - a S^T k);   S <- a S + k u^T;   o = scale S^T q .
// Columns of S never meet, so the work splits over (sequence, head, columns).
#include <limits.h>
#include <math.h>

#include <type_traits>

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
  const int32_t* before;   // [sequences]: the largest of the offsets before (delta_order); or NULL
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
  uint32_t bad = fronk::bad_sequence(s, A.slots, a, b, A.tokens, A.max_tokens);
  // Behind offsets that go down, a sequence could share tokens with one before.
  bool below = false;
  if (A.before)
    below = A.before[i] > a;
  else if (A.offsets)
    for (uint32_t e = threadIdx.x & 63; e < i; e += 64) below |= A.offsets[e] > a;
  if (__any(below)) bad |= FR_HIP_BAD_OFFSET;
  *first = (uint32_t)a;
  *count = (uint32_t)(b - a);
  *row = (size_t)(s < 0 ? 0 : s);
  if (bad && A.status && threadIdx.x == 0) atomicOr(A.status, bad);
  return !bad && s >= 0;
}

// The running maximum of the offsets before each sequence's own, where there are too
// many for every wavefront to look through: one workgroup, a stretch of 4096 at a time.
__global__ __launch_bounds__(1024) void delta_order(const int32_t* offsets, uint32_t sequences, int32_t* before) {
  __shared__ int32_t top[16];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t carry = INT_MIN;
  for (uint32_t base = 0; base < sequences; base += 4096) {
    const uint32_t first = base + threadIdx.x * 4;
    int32_t x[4], most = INT_MIN;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = most;   // of this thread's, those before
      most = max(most, first + e < sequences ? offsets[first + e] : INT_MIN);
    }
    for (int d = 1; d < 64; d *= 2) {
      const int32_t y = __shfl_up(most, d);
      if (lane >= (uint32_t)d) most = max(most, y);
    }
    if (lane == 63) top[wave] = most;
    int32_t mine = __shfl_up(most, 1);
    if (lane == 0) mine = INT_MIN;
    __syncthreads();
    mine = max(mine, carry);
    for (uint32_t w = 0; w < 16; ++w) {
      if (w < wave) mine = max(mine, top[w]);
      carry = max(carry, top[w]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (first + e < sequences) before[first + e] = max(mine, x[e]);
    __syncthreads();   // top is read
  }
}

// ------------------------------------------------------------ token by token
//
// One wavefront holds 16 columns of one head's state in registers: lane 4r + c
// keeps rows r * R .. r * R + R - 1 (R = dk / 16) of columns 4c .. 4c + 3. Both
// products over dk are taken of the state before the token,
//     p = S^T k,  w = S^T q,  o = scale (a w + (q . k) u),
// so that a token needs one reduction over the 16 row lanes: two row rotations
// and the two row swaps, no LDS and no barrier. Bound by reading and writing the
// states: 64 streams of 32 heads of 128 x 128 (268 MB) in 57.7 us, 4.7 TB/s; one
// stream's in 4.5 us, a launch and a memory latency.

// `count` tokens from `first` on of 16 columns (`tile`) of a head, s being its state.
template <typename T, int DK>
__device__ __forceinline__ void walk(const DeltaArgs& A, uint32_t first, uint32_t count, uint32_t head, uint32_t tile,
                                     float (&s)[DK / 16][4]) {
  constexpr int R = DK / 16;
  const uint32_t lane = threadIdx.x & 63, r = lane >> 2, col = tile * 16 + (lane & 3) * 4, kh = head / (A.heads / A.key_heads);
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
}

// All `count` tokens of a sequence, from its state to its state.
template <typename T, int DK>
__device__ __forceinline__ void walk_all(const DeltaArgs& A, uint32_t first, uint32_t count, size_t row, uint32_t head,
                                         uint32_t tile) {
  constexpr int R = DK / 16;
  const uint32_t lane = threadIdx.x & 63, r = lane >> 2, col = tile * 16 + (lane & 3) * 4;
  const size_t at = ((row * A.heads + head) * DK + r * R) * A.dv + col;
  float s[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float4v x = {0, 0, 0, 0};
    if (A.state_in) x = *reinterpret_cast<const float4v*>(A.state_in + at + (size_t)i * A.dv);
#pragma unroll
    for (int c = 0; c < 4; ++c) s[i][c] = x[c];
  }
  walk<T, DK>(A, first, count, head, tile, s);
  if (A.state_out) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float4v x = {s[i][0], s[i][1], s[i][2], s[i][3]};
      *reinterpret_cast<float4v*>(A.state_out + at + (size_t)i * A.dv) = x;
    }
  }
}

template <typename T, int DK>
__global__ __launch_bounds__(256) void delta_step(DeltaArgs A) {
  const uint32_t waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
  const uint32_t tiles = A.dv / 16, groups = (tiles + waves - 1) / waves;
  const uint32_t tile = blockIdx.x % groups * waves + wave;
  const uint32_t head = blockIdx.x / groups % A.heads, seq = blockIdx.x / groups / A.heads;
  uint32_t first, count;
  size_t row;
  if (!sequence(A, seq, &first, &count, &row) || tile >= tiles) return;
  walk_all<T, DK>(A, first, count, row, head, tile);
}

// ------------------------------------------------------------ chunk by chunk
//
// The published chunk form of the delta rule (Yang et al., Parallelizing Linear
// Transformers with the Delta Rule over Sequence Length, 2024), with its decays:
// within a chunk of 64 tokens, with G the running sum of g and D_ij =
// e^(G_i - G_j), the rule's updates u solve a lower triangular system
//     A_ij = beta_i (k_i . k_j) D_ij  (j < i),   T = (I + A)^-1 diag(beta)
//     U = T (V - e^G K S)
//     O = scale (e^G Q S + (Q K^T . D) U),   S <- e^(G_last) S + (e^(G_last - G) K)^T U
// delta_prepare forms what does not depend on S, for all chunks at once: T, P =
// scale Q K^T . D, and K and Q as operands. delta_scan then goes through the
// chunks of one sequence, head and 16 columns of S.
//
// All products run on the bf16 matrix cores. A number that is not one bf16 is
// the sum of parts: fp32 (T, S, U and fp32 activations) of three (8 + 8 + 8
// bits), fp16 activations of two; products of parts down to 2^-16 of the
// largest are taken, so that the state keeps fp32's accuracy. Outputs of 16
// bits take two parts of S, P and U (2^-17, against their own rounding of 2^-8
// or 2^-11). fp32 matrix instructions would do without parts at a sixteenth of
// the rate.
//
// The order of the summed index in an operand is free. Over dims it is theirs,
// so that rows of K and Q are read as they lie; over tokens it is taken so that
// a result's registers are the next product's operand: a lane (i, j) of a result
// holds rows 4j .. 4j+3 of a tile of 16, so operand element e of lane row j
// stands for token 32 s + 16 (e / 4) + 4 j + e % 4 of step s.
//
// Sums over a chunk's tokens meet zeros where a token is not seen, and zero times
// infinity is NaN; and e^G may pass fp32 where the recurrence, whose decays meet
// smaller values one by one, does not. Both leave the final state non-finite: what an
// infinity or NaN in S, U, T or the scalars gets into is every row of its columns, for
// good (P, and the scalars of Q, are looked at by themselves). So where a final state
// has a number of 2^127 or more, or NaN, the sequence is gone through again token by
// token, and tokens before a non-finite one keep their values.
constexpr int kChunk = 64;
__device__ __forceinline__ bool huge(float x) { return !(fabsf(x) < 0x1p127f); }
__device__ __forceinline__ bool huge(float4v x, float4v y) {   // one of them, or their sum
  return huge((fabsf(x[0]) + fabsf(x[1])) + (fabsf(x[2]) + fabsf(x[3])) + ((fabsf(y[0]) + fabsf(y[1])) + (fabsf(y[2]) + fabsf(y[3]))));
}

template <typename T> struct Parts;
template <> struct Parts<__bf16> { static constexpr int kIn = 1, kOut = 2; };
template <> struct Parts<_Float16> { static constexpr int kIn = 2, kOut = 2; };
template <> struct Parts<float> { static constexpr int kIn = 3, kOut = 3; };

// The workspace, in operands of 64 lanes x 16 bytes, for each chunk slot.
// A sequence's chunks begin at slot first / 64 + its index, which leaves room
// for every sequence's last, partial chunk.
template <typename T, int DK> struct Room {
  static constexpr int kN = Parts<T>::kIn, kSteps = DK / 32;
  static constexpr size_t kRows = (size_t)4 * kSteps * kN;     // K (and Q) with tokens as rows
  static constexpr size_t kKey = 3 * kRows;                    // ... K, Q, and K with dims as rows
  static constexpr size_t kMatrix = (size_t)kChunk * (kChunk + 4) * sizeof(float);   // in LDS
  static constexpr size_t kShared = kRows * 1024 > kMatrix ? kRows * 1024 : kMatrix;
  static constexpr size_t kT = 6 * 3, kP = 6 * Parts<T>::kOut; // lower triangles: 1, 1, 2, 2 steps
  static constexpr size_t kHead = kT + kP + 1;                 // ... and 256 floats
  static size_t bytes(const fr_hip_delta* r) {
    const size_t slots = (size_t)r->tokens / kChunk + r->sequences;
    return slots * (kKey * r->key_heads + kHead * r->heads) * 1024;
  }
};
// Triangle operands: tile w's first.
__device__ __forceinline__ int triangle(int w) { return w < 2 ? w : 2 * w - 2; }

struct ChunkArgs {
  DeltaArgs d;
  uint4v *key, *head;   // [slot][key head][Room::kKey][64], [slot][head][Room::kHead][64]
  uint32_t each;        // value heads of a workgroup of delta_prepare
};
// Floats of a head's last kilobyte. kLast NaN makes the state NaN, and so sends the
// sequence through `walk`.
enum { kRowK = 0, kRowQ = 64, kColU = 128, kLast = 192 };

template <int N> __device__ __forceinline__ void split4(float4v x, bf16x4 (&out)[N]) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const bf16x2 a = to_bf16(x[0], x[1]), b = to_bf16(x[2], x[3]);
    out[p] = bf16x4{a[0], a[1], b[0], b[1]};
    if (p + 1 < N) x -= float4v{(float)a[0], (float)a[1], (float)b[0], (float)b[1]};
  }
}
template <int N> __device__ __forceinline__ void split8(float4v x, float4v y, bf16x8 (&out)[N]) {
  bf16x4 a[N], b[N];
  split4<N>(x, a);
  split4<N>(y, b);
#pragma unroll
  for (int p = 0; p < N; ++p) out[p] = bf16x8{a[p][0], a[p][1], a[p][2], a[p][3], b[p][0], b[p][1], b[p][2], b[p][3]};
}
// What this wavefront's lanes wrote to LDS is there for all of them.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// All of the workgroup's LDS writes are there for all of it; loads and stores of
// memory go on.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
__device__ __forceinline__ bf16x8 frag(uint4v x) { return __builtin_bit_cast(bf16x8, x); }

// One workgroup: one chunk and key head, and `each` of the value heads that share
// it; wavefront w holds tokens 16 w .. 16 w + 15 as rows. A head takes about 6 us:
// decays and P 2.5, the inverse 2, the barriers between them the rest. 4096 tokens
// of 32 heads: 43 us, 113 MB written; 5 sequences with 33 chunks of 9 heads: 17 us.
template <typename T, int DK>
__global__ __launch_bounds__(256) void delta_prepare(ChunkArgs C) {
  typedef Room<T, DK> W;
  constexpr int N = W::kN, KS = W::kSteps, PO = Parts<T>::kOut, kPitch = kChunk + 4;
  const DeltaArgs& A = C.d;
  extern __shared__ uint4v lds[];
  uint4v* kf = lds;                                            // [4][KS][N][64]
  float(*m1)[kPitch] = reinterpret_cast<float(*)[kPitch]>(lds);   // in kf's place, once that is read
  float(*m2)[kPitch] = reinterpret_cast<float(*)[kPitch]>(lds + W::kShared / 16);
  __shared__ double total[kChunk];
  __shared__ int odd;   // a huge number in this head's P or scalars
  __shared__ __attribute__((aligned(16))) float kn[kChunk], qn[kChunk], bt[kChunk];

  const uint32_t chunks = (A.max_tokens + kChunk - 1) / kChunk;
  const uint32_t group = A.heads / A.key_heads, first_head = blockIdx.y * C.each;
  const uint32_t kh = blockIdx.x % A.key_heads, chunk = blockIdx.x / A.key_heads % chunks;
  const uint32_t seq = blockIdx.x / A.key_heads / chunks;
  uint32_t first, count;
  size_t row;
  if (!sequence(A, seq, &first, &count, &row) || chunk * kChunk >= count) return;
  const uint32_t slot = first / kChunk + seq + chunk;
  first += chunk * kChunk;
  const int n = (int)min(count - chunk * kChunk, (uint32_t)kChunk);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = lane & 15, j = lane >> 4;
  uint4v* key = C.key + ((size_t)slot * A.key_heads + kh) * W::kKey * 64;

  // K and Q of this wavefront's tokens as operands, and their norms.
  bf16x8 ka[KS][N], qa[KS][N];
  auto rows = [&](const void* base, int64_t token, int64_t head, bf16x8(&out)[KS][N], float* norm) {
    const T* p = static_cast<const T*>(base) + (int64_t)(first + (16 * w + i < n ? 16 * w + i : 0)) * token + kh * head;
    float sum = 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float f[8];
      load_row<8>(p + 32 * s + 8 * j, A.wide, f);
      float4v x = {f[0], f[1], f[2], f[3]}, y = {f[4], f[5], f[6], f[7]};
      if (16 * w + i >= n) x = float4v{0, 0, 0, 0}, y = x;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fmaf(x[e], x[e], fmaf(y[e], y[e], sum));
      split8<N>(x, y, out[s]);
    }
    sum = add_xor32(add_xor16(sum));
    if (j == 0) norm[16 * w + i] = A.normalize ? 1.f / sqrtf(sum + 1e-6f) : 1.f;
  };
  rows(A.k, A.k_token, A.k_head, ka, kn);
  rows(A.q, A.q_token, A.q_head, qa, qn);
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int p = 0; p < N; ++p) {
      const int at = ((w * KS + s) * N + p) * 64 + lane;
      kf[at] = __builtin_bit_cast(uint4v, ka[s][p]);
      if (first_head) continue;   // the first heads' workgroup writes for all
      key[at] = kf[at];
      key[W::kRows * 64 + at] = __builtin_bit_cast(uint4v, qa[s][p]);
    }
  lds_barrier();

  // K with dims as rows: dim 16 t + i, tokens 32 s + 16 (e / 4) + 4 j + e % 4.
  const __bf16* k16 = reinterpret_cast<const __bf16*>(kf);
  for (int f = w; f < DK / 16 * 2 * N && !first_head; f += 4) {
    const int p = f % N, s = f / N % 2, t = f / N / 2;
    bf16x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = k16[((((2 * s + e / 4) * KS + t / 2) * N + p) * 64 + 16 * (2 * (t % 2) + (i >> 3)) + 4 * j + e % 4) * 8 + (i & 7)];
    key[2 * W::kRows * 64 + f * 64 + lane] = __builtin_bit_cast(uint4v, x);
  }

  // K K^T and Q K^T, tiles at and below the diagonal.
  float4v kk[4], qk[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    kk[u] = qk[u] = float4v{0, 0, 0, 0};
    if (u > w) continue;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int b = N - 1; b >= 0; --b) {
        const bf16x8 x = frag(kf[((u * KS + s) * N + b) * 64 + lane]);
#pragma unroll
        for (int a = N - 1; a >= 0; --a)
          if (a + b <= 2) {
            kk[u] = mma(ka[s][a], x, kk[u]);
            qk[u] = mma(qa[s][a], x, qk[u]);
          }
      }
  }

  for (uint32_t r = first_head; r < first_head + C.each && r < group; ++r) {
    const uint32_t head = kh * group + r;
    uint4v* out = C.head + ((size_t)slot * A.heads + head) * W::kHead * 64;
    float* scalars = reinterpret_cast<float*>(out + (W::kT + W::kP) * 64);
    if (w == 0) {
      // In 64 bits: a sum of far decays would take the near ones' differences
      // with it. One of -1e5 empties the state as -infinity does. In powers of
      // two: exp2 of a difference d is off by |d| 2^-24 of itself, at most 2^-24.
      double x = lane < n ? (double)A.g[(int64_t)(first + lane) * A.g_token + head] : 0.0;
      x = (x < -1e5 ? -1e5 : x) * 1.4426950408889634;
      for (int d = 1; d < 64; d *= 2) {
        const double y = __shfl_up(x, d);
        if (lane >= d) x += y;
      }
      total[lane] = x;
      bt[lane] = lane < n ? A.beta[(int64_t)(first + lane) * A.beta_token + head] : 0.f;
      const double last = __shfl(x, 63);
      const float gamma = __builtin_amdgcn_exp2f((float)x);
      const float row_k = gamma * kn[lane], row_q = gamma * qn[lane] * A.scale;
      const float col_u = __builtin_amdgcn_exp2f((float)(last - x)) * kn[lane], all = __builtin_amdgcn_exp2f((float)last);
      scalars[kRowK + lane] = row_k;
      scalars[kRowQ + lane] = row_q;
      scalars[kColU + lane] = col_u;
      const bool any = __any(huge(row_k) | huge(row_q) | huge(col_u) | huge(all));
      if (lane == 0) scalars[kLast] = all, odd = any;
    }
    lds_barrier();
    // P row by row, then A, through m1.
    float decay[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int a = 16 * w + 4 * j + e, b = 16 * u + i;
        const float d = __builtin_amdgcn_exp2f((float)(total[a] - total[b])) * kn[b];
        decay[u][e] = a >= b ? d : 0.f;
        m1[a][b] = a >= b ? qk[u][e] * decay[u][e] * (qn[a] * A.scale) : 0.f;
      }
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s > w / 2) continue;
      bf16x8 x[PO];
      const float4v y = *reinterpret_cast<const float4v*>(&m1[16 * w + i][32 * s + 4 * j]);
      const float4v z = *reinterpret_cast<const float4v*>(&m1[16 * w + i][32 * s + 16 + 4 * j]);
      if (huge(y, z)) odd = 1;
      split8<PO>(y, z, x);
#pragma unroll
      for (int p = 0; p < PO; ++p)
        out[(W::kT + (triangle(w) + s) * PO + p) * 64 + lane] = __builtin_bit_cast(uint4v, x[p]);
    }
    lds_barrier();
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int a = 16 * w + 4 * j + e, b = 16 * u + i;
        m1[a][b] = a > b ? kk[u][e] * decay[u][e] * (bt[a] * kn[a]) : 0.f;
        m2[a][b] = 0.f;
      }
    lds_barrier();
    // (I + A)^-1 in m2 by blocks of 16: the diagonal ones by substitution
    // (lane i column i; products of powers of A would lose digits where keys
    // are alike), then those below by the distance from it, each from blocks
    // that are there: X_wu = -X_ww sum_{u <= v < w} A_wv X_vu.
    {
      float x[16];
#pragma unroll
      for (int a = 0; a < 16; ++a) {
        float y = a == i ? 1.f : 0.f;
#pragma unroll
        for (int b = 0; b < a; ++b) y = fmaf(-m1[16 * w + a][16 * w + b], x[b], y);
        x[a] = y;
      }
      if (j == 0) {
#pragma unroll
        for (int a = 0; a < 16; ++a) m2[16 * w + a][16 * w + i] = x[a];
      }
    }
    for (int dist = 1; dist < 4; ++dist) {
      lds_barrier();
      if (w >= dist) {
        const int u = w - dist;
        float4v c = {0, 0, 0, 0};
        for (int v = u; v < w; ++v)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(m1[16 * w + i][16 * v + 4 * s + j], m2[16 * v + 4 * s + j][16 * u + i], c, 0, 0, 0);
        // The sum's place until it is an operand: the block that it becomes.
#pragma unroll
        for (int e = 0; e < 4; ++e) m2[16 * w + 4 * j + e][16 * u + i] = c[e];
        wave_lds_sync();
        float4v y = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 4; ++s)
          y = __builtin_amdgcn_mfma_f32_16x16x4f32(m2[16 * w + i][16 * w + 4 * s + j], m2[16 * w + 4 * s + j][16 * u + i], y, 0, 0, 0);
        wave_lds_sync();
#pragma unroll
        for (int e = 0; e < 4; ++e) m2[16 * w + 4 * j + e][16 * u + i] = -y[e];
      }
    }
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s > w / 2) continue;
      const int c = 32 * s + 4 * j;
      bf16x8 x[3];
      const float4v y = *reinterpret_cast<const float4v*>(&m2[16 * w + i][c]) * *reinterpret_cast<const float4v*>(&bt[c]);
      const float4v z = *reinterpret_cast<const float4v*>(&m2[16 * w + i][c + 16]) * *reinterpret_cast<const float4v*>(&bt[c + 16]);
      split8<3>(y, z, x);
#pragma unroll
      for (int p = 0; p < 3; ++p) out[((triangle(w) + s) * 3 + p) * 64 + lane] = __builtin_bit_cast(uint4v, x[p]);
    }
    lds_barrier();
    if (threadIdx.x == 0 && odd) scalars[kLast] = NAN;   // behind its own store of the same place
  }
}

// One workgroup: one sequence, head and 16 columns of S, chunk after chunk.
// Wavefronts 0..3 carry the state: wavefront w has tokens 16 w .. of the chunk
// and dims w * dk / 4 .. of S (in registers, fp32), and three times a chunk they
// exchange operands through LDS: S, then V - e^G K S, then U. Wavefronts 4..7
// form the outputs of the same tokens beside them. 64 chunks of 32 heads of 128 x
// 128 in 100 us, 1.6 us a chunk, of which the chain's products, splits and LDS
// exchanges by themselves are 1.3 and memory hardly any.
//
// A chunk costs three barriers and the products between them, so nothing may
// wait for memory there: each operand's registers are filled anew in the phase
// after the product that read them, two phases before the next (kAhead; with
// fp32's 54 operands at dk 256, which do not fit, K's rows and dims take turns). The two kinds of wavefronts have loops of their own, so that
// neither's loads are waited for on account of the other's.
template <typename T, int DK>
__global__ __launch_bounds__(512) void delta_scan(ChunkArgs C) {
  typedef Room<T, DK> W;
  constexpr int N = W::kN, KS = W::kSteps, PO = Parts<T>::kOut, TPW = DK / 64;
  constexpr bool kAhead = KS * N + TPW * 2 * N <= 32;
  const DeltaArgs& A = C.d;
  __shared__ uint4v sf[3][KS][64], rf[3][2][64], uf[PO][2][64], wf[3][2][64];
  __shared__ int odd;   // a huge number in the final state
  const int lane = threadIdx.x & 63, i = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const bool chain = wave < 4;
  // The heads of a key head and their tiles follow each other at a distance of
  // key_heads, which for a multiple of 8 puts them on one die and its L2.
  const uint32_t group = A.heads / A.key_heads, tiles = A.dv / 16;
  const uint32_t kh = blockIdx.x % A.key_heads, head = kh * group + blockIdx.x / A.key_heads % group;
  const uint32_t tile = blockIdx.x / A.heads % tiles, seq = blockIdx.x / A.heads / tiles;
  uint32_t first, count;
  size_t row;
  if (!sequence(A, seq, &first, &count, &row)) return;
  const uint32_t slot = first / kChunk + seq, chunks = (count + kChunk - 1) / kChunk;
  const uint32_t col = tile * 16 + i;
  if (threadIdx.x == 0) odd = 0;
  const int steps = w < 2 ? 1 : 2;   // of T's and P's row tile w

  // Four values of lane row r into half h of an operand's parts.
  auto put = [&](uint4v* base, int stride, int r, int half, float4v x, auto parts) {
    constexpr int P = decltype(parts)::value;
    bf16x4 y[P];
    split4<P>(x, y);
#pragma unroll
    for (int p = 0; p < P; ++p) reinterpret_cast<bf16x4*>(base + p * stride)[(i + 16 * r) * 2 + half] = y[p];
  };
  constexpr std::integral_constant<int, 3> three{};
  constexpr std::integral_constant<int, PO> few{};

  const uint4v* key = C.key + ((size_t)slot * A.key_heads + kh) * W::kKey * 64 + (chain ? 0 : W::kRows * 64) + lane;
  const uint4v* per = C.head + ((size_t)slot * A.heads + head) * W::kHead * 64 + lane;
  const size_t key_next = (size_t)A.key_heads * W::kKey * 64, per_next = (size_t)A.heads * W::kHead * 64;
  // Chunk c's rows of K (or Q), rows of T (or P), and scalars from `at` on.
  uint4v a1[KS][N], a2[2][3];
  auto load1 = [&](uint32_t c) {
    const uint4v* p = key + c * key_next + w * KS * N * 64;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int a = 0; a < N; ++a) a1[s][a] = p[(s * N + a) * 64];
  };
  auto load2 = [&](uint32_t c, auto parts) {
    constexpr int P = decltype(parts)::value;
    const uint4v* p = per + c * per_next + triangle(w) * P * 64;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int a = 0; a < P; ++a)
        if (s < steps) a2[s][a] = p[(s * P + a) * 64];
  };
  auto scalars = [&](uint32_t c, int at) {
    return *reinterpret_cast<const float4v*>(reinterpret_cast<const float*>(per - lane + c * per_next + (W::kT + W::kP) * 64) +
                                             at + 16 * w + 4 * j);
  };

  if (chain) {
    uint4v a3[TPW][2][N];
    float4v row_scale, col_scale;
    float last;
    T v[4];
    auto load3 = [&](uint32_t c) {
      const uint4v* p = key + c * key_next + (2 * W::kRows + w * TPW * 2 * N) * 64;
#pragma unroll
      for (int t = 0; t < TPW; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int a = 0; a < N; ++a) a3[t][s][a] = p[((t * 2 + s) * N + a) * 64];
      last = reinterpret_cast<const float*>(per - lane + c * per_next + (W::kT + W::kP) * 64)[kLast];
    };
    const T* values = static_cast<const T*>(A.v) + (int64_t)first * A.v_token + head * A.v_head + col;
    const T* mine[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) mine[e] = values + (int64_t)(16 * w + 4 * j + e) * A.v_token;
    auto load_v = [&](uint32_t c) {
      if ((c + 1) * kChunk <= count) {
        const int64_t on = (int64_t)(c * kChunk) * A.v_token;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = mine[e][on];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = values[(int64_t)min(c * kChunk + 16 * w + 4 * j + e, count - 1) * A.v_token];
      }
      row_scale = scalars(c, kRowK);
    };
    // S's operands go by dims in their order, as rows of K and Q lie in memory.
    auto put_state = [&](int t, float4v x) {
      const int at = w * TPW + t;
      put(&sf[0][at / 2][0], KS * 64, 2 * (at % 2) + j / 2, j % 2, x, three);
    };
    if (chunks) {
      load1(0), load_v(0), load2(0, three);
      col_scale = scalars(0, kColU);
    }
    float4v state[TPW];
    const size_t at = ((row * A.heads + head) * DK + 16 * w * TPW + 4 * j) * A.dv + col;
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) state[t][e] = A.state_in ? A.state_in[at + (size_t)(16 * t + e) * A.dv] : 0.f;
      put_state(t, state[t]);
    }
    // The chain is what the chunk's time is: its instructions go first.
    __builtin_amdgcn_s_setprio(3);
    for (uint32_t c = 0; c < chunks; ++c) {
      const uint32_t next = c + 1 < chunks ? c + 1 : c;
      lds_barrier();   // S is there
      float4v x[3] = {};
      bf16x8 y[3][2];
      if constexpr (kAhead) load3(c);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int b = 2; b >= 0; --b) {
          const bf16x8 z = frag(sf[b][s][lane]);
#pragma unroll
          for (int a = 0; a < N && a + b <= 2; ++a) x[a + b] = mma(frag(a1[s][a]), z, x[a + b]);
        }
      const uint32_t token = c * kChunk + 16 * w + 4 * j;
      float4v r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = token + e < count ? (float)v[e] : 0.f;
      r -= row_scale * (x[0] + (x[1] + x[2]));
      put(&rf[0][w / 2][0], 2 * 64, j, w % 2, r, three);
      lds_barrier();   // V - e^G K S is there
#pragma unroll
      for (int b = 2; b >= 0; --b)
#pragma unroll
        for (int s = 0; s < 2; ++s) y[b][s] = frag(rf[b][s][lane]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kAhead) load1(next);
      else load3(c);
      load_v(next);
      __builtin_amdgcn_sched_barrier(0);
      float4v u[3] = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (s >= steps) continue;
#pragma unroll
        for (int b = 2; b >= 0; --b)
#pragma unroll
          for (int a = 0; a + b <= 2; ++a) u[a + b] = mma(frag(a2[s][a]), y[b][s], u[a + b]);
      }
      u[0] += u[1] + u[2];
      put(&wf[0][w / 2][0], 2 * 64, j, w % 2, u[0] * col_scale, three);
      put(&uf[0][w / 2][0], 2 * 64, j, w % 2, u[0], few);
      lds_barrier();   // U is there
#pragma unroll
      for (int b = 2; b >= 0; --b)
#pragma unroll
        for (int s = 0; s < 2; ++s) y[b][s] = frag(wf[b][s][lane]);
      __builtin_amdgcn_sched_barrier(0);
      load2(next, three);
      col_scale = scalars(next, kColU);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < TPW; ++t) {
        float4v z[3] = {};
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int b = 2; b >= 0; --b)
#pragma unroll
            for (int a = 0; a < N && a + b <= 2; ++a) z[a + b] = mma(frag(a3[t][s][a]), y[b][s], z[a + b]);
        state[t] = last * state[t] + (z[0] + (z[1] + z[2]));
        put_state(t, state[t]);
      }
      if constexpr (!kAhead) load1(next);
    }
    __builtin_amdgcn_s_setprio(0);
    bool any = false;
#pragma unroll
    for (int t = 0; t < TPW; ++t) any |= huge(state[t], float4v{0, 0, 0, 0});
    if (chunks && any) odd = 1;
    __syncthreads();   // the outputs are written, too
    if (odd) {
      if (w == 0) walk_all<T, DK>(A, first, count, row, head, tile);
      return;
    }
    if (A.state_out) {
#pragma unroll
      for (int t = 0; t < TPW; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) A.state_out[at + (size_t)(16 * t + e) * A.dv] = state[t][e];
    }
  } else {
    per += W::kT * 64;   // P
    float4v row_scale;
    auto rows_of = [&](uint32_t c) {
      load1(c);
      row_scale = *reinterpret_cast<const float4v*>(
          reinterpret_cast<const float*>(per - lane + c * per_next + W::kP * 64) + kRowQ + 16 * w + 4 * j);
    };
    if (chunks) rows_of(0), load2(0, few);
    for (uint32_t c = 0; c < chunks; ++c) {
      const uint32_t next = c + 1 < chunks ? c + 1 : c;
      lds_barrier();   // S is there
      lds_barrier();   // ... and read by the chain, which now leaves LDS to these
      float4v acc[3] = {};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int b = PO - 1; b >= 0; --b) {
          const bf16x8 y = frag(sf[b][s][lane]);
#pragma unroll
          for (int a = 0; a < N && a + b < PO; ++a) acc[a + b] = mma(frag(a1[s][a]), y, acc[a + b]);
        }
      acc[0] = row_scale * (acc[0] + (acc[1] + acc[2]));
      acc[1] = acc[2] = float4v{0, 0, 0, 0};
      rows_of(next);
      lds_barrier();   // U is there, and S is read
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (s >= steps) continue;
#pragma unroll
        for (int b = PO - 1; b >= 0; --b) {
          const bf16x8 y = frag(uf[b][s][lane]);
#pragma unroll
          for (int a = 0; a + b < PO; ++a) acc[a + b] = mma(frag(a2[s][a]), y, acc[a + b]);
        }
      }
      load2(next, few);
      acc[0] += acc[1] + acc[2];
      const uint32_t token = c * kChunk + 16 * w + 4 * j;
      T* out = static_cast<T*>(A.o) + (int64_t)first * A.o_token + head * A.o_head + col;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (token + e < count) out[(int64_t)(token + e) * A.o_token] = (T)acc[0][e];
    }
    __syncthreads();   // the chain's last one
  }
}

// ---------------------------------------------------------------------- host

// Calls go token by token; where a sequence may have this many, in chunks. Measured,
// token by token against chunks in us: one stream of 32 heads of 128 x 128 in bf16 21,
// 19 (16 tokens), 36, 19 (32), 67, 20 (64), in fp32 20, 23 (16), 34, 23 (32); 64 such
// streams 235, 316 (24), 309, 323 (32), 457, 335 (48), in fp32 305, 487 (32), 452, 493
// (48), 595, 500 (64). Between the borders of few streams (about 16) and of many (about
// 33 and, fp32, 50).
constexpr unsigned kChunkFrom = 33;
bool in_chunks(const fr_hip_delta* r) { return r->max_tokens >= kChunkFrom && r->tokens >= kChunkFrom; }

int check(const fr_hip_delta* r) {
  if (!r || r->type > FR_HIP_BF16 || (r->flags & ~(unsigned)FR_HIP_DELTA_NORMALIZE)) return FR_HIP_INVALID;
  if (!r->key_heads || !r->heads || r->heads % r->key_heads || !r->key_dim || !r->value_dim) return FR_HIP_INVALID;
  if (!isfinite(r->scale)) return FR_HIP_INVALID;
  if (r->tokens > INT_MAX || r->sequences > INT_MAX || r->slots > INT_MAX) return FR_HIP_INVALID;
  if (!r->offsets && r->tokens != (uint64_t)r->sequences * r->max_tokens) return FR_HIP_INVALID;
  if (!r->slot && r->slots < r->sequences && (r->state_in || r->state_out)) return FR_HIP_INVALID;
  if (r->tokens && r->sequences && (!r->q || !r->k || !r->v || !r->g || !r->beta || !r->o)) return FR_HIP_INVALID;
  if (((uintptr_t)r->state_in | (uintptr_t)r->state_out) % 16) return FR_HIP_INVALID;
  if (r->state_in && r->state_out && r->state_in != r->state_out) {   // pools that share some rows, not all
    const uintptr_t a = (uintptr_t)r->state_in, b = (uintptr_t)r->state_out, apart = a < b ? b - a : a - b;
    if (apart / ((uint64_t)r->heads * r->key_dim * r->value_dim * sizeof(float)) < r->slots) return FR_HIP_INVALID;
  }
  if (((uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->o) % elem_size(r->type)) return FR_HIP_INVALID;
  if (r->key_dim != 64 && r->key_dim != 128 && r->key_dim != 256) return FR_HIP_UNSUPPORTED;
  if (r->value_dim % 16 || r->value_dim > 1024 || r->heads > 65535) return FR_HIP_UNSUPPORTED;
  // One-dimensional grids of (sequence, head, 16 columns) and (sequence, chunk, key
  // head), of less than 2^32 threads.
  const uint64_t columns = (uint64_t)r->sequences * r->heads * (r->value_dim / 16), longest = r->max_tokens < r->tokens ? r->max_tokens : r->tokens;
  if (columns > UINT32_MAX / (in_chunks(r) ? 512 : 128)) return FR_HIP_UNSUPPORTED;
  if (r->sequences * (longest / kChunk + 1) > UINT32_MAX / 256 / r->key_heads) return FR_HIP_UNSUPPORTED;
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
  A.before = nullptr;
  A.offsets = r->offsets, A.slot = r->slot, A.state_in = r->state_in, A.state_out = r->state_out, A.status = r->status;
  A.q_token = r->q_token, A.q_head = r->q_head, A.k_token = r->k_token, A.k_head = r->k_head;
  A.v_token = r->v_token, A.v_head = r->v_head, A.o_token = r->o_token, A.o_head = r->o_head;
  A.g_token = r->g_token, A.beta_token = r->beta_token;
  A.sequences = r->sequences, A.tokens = r->tokens, A.max_tokens = r->max_tokens < r->tokens ? r->max_tokens : r->tokens;
  A.key_heads = r->key_heads, A.heads = r->heads, A.dv = r->value_dim;
  // Without state pools a slot only says whether the sequence is skipped.
  A.slots = r->state_in || r->state_out ? r->slots : (uint32_t)INT_MAX;
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
  const uint32_t waves = total <= 4 * kUnits ? 1 : tiles < 4 ? tiles : 4;
  const dim3 grid((uint32_t)((uint64_t)r->sequences * r->heads * ((tiles + waves - 1) / waves))), block(64 * waves);
  switch (r->key_dim) {
    case 64: hipLaunchKernelGGL((delta_step<T, 64>), grid, block, 0, s, A); break;
    case 128: hipLaunchKernelGGL((delta_step<T, 128>), grid, block, 0, s, A); break;
    default: hipLaunchKernelGGL((delta_step<T, 256>), grid, block, 0, s, A); break;
  }
}

template <typename T, int DK>
int launch_chunks(const fr_hip_delta* r, const DeltaArgs& A, void* workspace, hipStream_t s) {
  typedef Room<T, DK> W;
  constexpr size_t kLds = W::kShared + W::kMatrix;
  const size_t slots = (size_t)r->tokens / kChunk + r->sequences;
  ChunkArgs C = {A, static_cast<uint4v*>(workspace), static_cast<uint4v*>(workspace) + slots * W::kKey * r->key_heads * 64, 1};
  static fronk::Devices allowed;
  if (allow_lds(&delta_prepare<T, DK>, kLds, &allowed)) return FR_HIP_IO;
  const uint32_t chunks = (A.max_tokens + kChunk - 1) / kChunk;
  // The heads of a key head share its products where there are enough chunks to
  // fill the card without: six workgroups a unit, were there one a head. Measured, one
  // a head against one for all of a call in us, bf16, by workgroups of the first kind:
  // 16 key heads and 32 heads of 128 44, 48 (512), 75, 72 (1024), 90, 91 (1280), 103,
  // 102 (1536), 134, 127 (2048); 4 and 16 heads 61, 76 (512), 88, 95 (768), 109, 114
  // (1024), 158, 156 (1536), 208, 196 (2048); 16 and 48 heads of 64 44, 47 (768), 72, 66
  // (1536). (Chunks as far as they are known here: no more than the tokens have.)
  const uint32_t prepares = r->sequences * chunks * r->key_heads, group = r->heads / r->key_heads;
  const uint64_t there = (uint64_t)r->tokens / kChunk + r->sequences;
  if ((there < (uint64_t)r->sequences * chunks ? there * r->key_heads : prepares) * group >= 6 * kUnits) C.each = group;
  hipLaunchKernelGGL((delta_prepare<T, DK>), dim3(prepares, (group + C.each - 1) / C.each), dim3(256), kLds, s, C);
  hipLaunchKernelGGL((delta_scan<T, DK>), dim3(r->sequences * r->heads * (r->value_dim / 16)), dim3(512), 0, s, C);
  return FR_HIP_OK;
}

template <typename T>
size_t room(const fr_hip_delta* r) {
  return r->key_dim == 64 ? Room<T, 64>::bytes(r) : r->key_dim == 128 ? Room<T, 128>::bytes(r) : Room<T, 256>::bytes(r);
}
size_t chunk_bytes(const fr_hip_delta* r) {   // a multiple of 1024
  if (!in_chunks(r)) return 0;
  return r->type == FR_HIP_F32 ? room<float>(r) : r->type == FR_HIP_F16 ? room<_Float16>(r) : room<__bf16>(r);
}
// With more sequences than this, their order is looked at beforehand. Measured, in
// place against beforehand in us, one token each: 10.9, 14.4 (2048 sequences of one
// head of 64 x 16), 16.7, 14.7 (4096), 36, 21 (8192), 828, 140 (65536); 214, 224
// (2048 of four heads of 128 x 128), 450, 446 (4096).
constexpr unsigned kScanned = 2048;
bool ordered(const fr_hip_delta* r) { return r->offsets && r->sequences > kScanned; }
size_t workspace_bytes(const fr_hip_delta* r) {
  return chunk_bytes(r) + (ordered(r) ? (size_t)r->sequences * sizeof(int32_t) : 0);
}

template <typename T>
int launch(const fr_hip_delta* r, const DeltaArgs& A, void* workspace, hipStream_t s) {
  if (!in_chunks(r)) {
    launch_step<T>(r, A, s);
    return FR_HIP_OK;
  }
  switch (r->key_dim) {
    case 64: return launch_chunks<T, 64>(r, A, workspace, s);
    case 128: return launch_chunks<T, 128>(r, A, workspace, s);
    default: return launch_chunks<T, 256>(r, A, workspace, s);
  }
}

}  // namespace

extern "C" {

size_t fr_hip_delta_workspace(const fr_hip_delta* req) { return check(req) ? 0 : workspace_bytes(req); }

int fr_hip_delta_rule(const fr_hip_delta* req, void* workspace, size_t bytes, void* stream) {
  int rc = check(req);
  if (rc) return rc;
  const size_t need = workspace_bytes(req);
  if (need && (!workspace || bytes < need || (uintptr_t)workspace % 16)) return FR_HIP_INVALID;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !req->sequences) return rc;
  DeltaArgs A = arguments(req);
  if (ordered(req)) {
    int32_t* before = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + chunk_bytes(req));
    hipLaunchKernelGGL(delta_order, dim3(1), dim3(1024), 0, s, req->offsets, req->sequences, before);
    A.before = before;
  }
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
