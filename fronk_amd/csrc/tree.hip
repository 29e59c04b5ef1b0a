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
  float *part_o, *part_ml;       // [workgroup][row][D], [workgroup][row][2]
  uint2v* plan;                  // of each sequence: its first workgroup, stretches
  const int64_t* tree;
  const int32_t *offsets, *table, *length;
  uint32_t* status;
  int64_t q_token, q_head, o_token, o_head;
  uint32_t sequences, tokens, max_tokens, per, max_context, table_stride, blocks;
  uint32_t slots, at_once;       // workgroups that may have a part (0: nothing is split); that run at once
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
    q0 = same(A.offsets[seq]), q1 = same(A.offsets[seq + 1]);
    for (uint32_t s = threadIdx.x; s < seq; s += blockDim.x) before = max(before, A.offsets[s]);
  }
  Drafts d = {q0, (uint32_t)(q1 - q0), (uint32_t)same(A.length[seq]), 0};
  if (__syncthreads_or(before > q0) || fronk::bad_sequence(0, 1, q0, q1, A.tokens, A.max_tokens)) d.bad = FR_HIP_BAD_OFFSET;
  else if ((int32_t)d.length < (int32_t)d.n || d.length > A.max_context) d.bad = FR_HIP_BAD_LENGTH, d.length = 0;
  return d;
}
// Where a workgroup works: `block` of the rows of one sequence and cache head, and one of
// `splits` stretches of `chunk` tokens.
struct Place {
  Drafts d;
  uint32_t seq, head, block, split, splits, chunk, part;   // (part ~0: no work)
};

constexpr uint32_t kPlanned = 512;   // sequences, at most, of a call that is split
constexpr uint32_t kPlanBytes = (kPlanned * 6 + 8 * 64 + 4) * 4;

// How the call is cut, which each workgroup finds out by itself from the sequences' lengths
// (the host does not know them): stretches of all sequences are no longer than one bound,
// for which 64 values are tried, a lane each, and that is taken with which the workgroups,
// in rounds of as many as run at once, end first; a workgroup's beginning and end take as
// long as about 300 tokens, and more where two share a unit (one stream of 32768 tokens and 16
// drafts, bf16, dim 128: 26.1 us in 256 workgroups, 27.7 in 512; of 131072 53.6 and 51.6). Work
// then varies by less than two between workgroups however ragged the batch is: 24 sequences
// of 1 to 61 drafts and up to 8192 tokens (16 heads of 128, four of the cache, fp16) take 63
// us, with one stretch length from the host 117. For 32 equal ones, for which nothing is to be
// found, it is 3 us more. 96 of 1 to 61 drafts in bf16 take 216 us.
// Workgroups of one stretch (its row blocks) follow each other, and each die, to which
// every eighth goes, has an eighth of the list: its L2 has the stretch for all of them.
template <int W, int ROWS, int D>
__device__ __forceinline__ Place plan(const TreeArgs& A, uint32_t* lds) {
  Place p;
  const uint32_t heads = A.cache.heads, die = blockIdx.x % 8, nth = blockIdx.x / 8, tid = threadIdx.x;
  // A list of `total`: this workgroup's place in it, ~0 for none.
  auto in_list = [&](uint32_t total) {
    const uint32_t eighth = (total + 7) / 8, mine = die * eighth + nth;
    return nth < eighth && mine < total ? mine : ~0u;
  };
  auto at = [&](uint32_t local, uint32_t blocks) {
    p.block = local % blocks, p.head = local / blocks % heads, p.split = local / blocks / heads;
    p.chunk = ((p.d.length + p.splits - 1) / p.splits + 63) & ~63u;
  };
  // What `total` workgroups of `chunk` tokens take, in 64 tokens of one that has a unit to
  // itself. Two on a unit take 1.5 times as long, and begin and end for longer.
  auto cost = [&](uint32_t total, uint32_t chunk) {
    const uint32_t rounds = (total + A.at_once - 1) / A.at_once, c = chunk / 64;
    if (D == 256) return rounds * (c + 5);
    return 2 * total <= A.at_once ? c + 5 : rounds * (c + c / 2 + 5) + (D == 64 ? 2 : 5);
  };
  if (A.sequences > kPlanned) {   // nothing is split
    p.part = in_list(A.sequences * heads * A.blocks);
    if (p.part == ~0u) return p;
    p.seq = p.part / A.blocks / heads, p.splits = 1;
    p.d = drafts_of(A, p.seq);
    at(p.part % (A.blocks * heads), A.blocks);
    if (p.d.bad && A.status && tid == 0) atomicOr(A.status, p.d.bad);
    if (p.d.bad == FR_HIP_BAD_OFFSET || p.block * ROWS >= p.d.n * A.per) p.part = ~0u;
    return p;
  }
  if (A.sequences == 1) {         // as many stretches as there may be workgroups, or as units
    p.seq = 0, p.d = drafts_of(A, 0);
    if (p.d.bad && A.status && blockIdx.x == 0 && tid == 0) atomicOr(A.status, p.d.bad);
    const uint32_t blocks = p.d.bad == FR_HIP_BAD_OFFSET ? 0 : (p.d.n * A.per + ROWS - 1) / ROWS, work = blocks * heads;
    p.splits = 1;
    if (work && 2 * work <= A.slots) {
      auto stretches = [&](uint32_t n, uint32_t* chunk) {
        *chunk = max((p.d.length / n + 64) & ~63u, 256u);
        return max((p.d.length + *chunk - 1) / *chunk, 1u);
      };
      uint32_t chunk, other;
      p.splits = stretches(min(A.slots / work, 256u), &chunk);
      if (D < 256 && 2 * work <= A.at_once) {
        const uint32_t fewer = stretches(min(A.at_once / 2 / work, 256u), &other);
        if (cost(work * fewer, other) <= cost(work * p.splits, chunk)) p.splits = fewer;
      }
    }
    if (blockIdx.x == 0 && tid == 0 && A.slots) A.plan[0] = uint2v{0, p.splits};
    p.part = in_list(work * p.splits);
    if (p.part != ~0u) at(p.part, blocks);
    return p;
  }
  uint32_t* const length = lds;                    // [sequences]
  uint32_t* const blocks = length + kPlanned;      // row blocks (none: a sequence without work)
  uint32_t* const first = blocks + kPlanned;       // its workgroups' place in the list
  uint32_t* const stretches = first + kPlanned;
  uint32_t* const start = stretches + kPlanned;    // its first row of q
  uint32_t* const drafts = start + kPlanned;
  uint32_t* const sums = drafts + kPlanned;        // [W][64]
  uint32_t* const found = sums + 8 * 64;
  const uint32_t lane = tid & 63, wave = tid >> 6;
  if (wave == 0) {
    uint32_t bad = 0, longest = 0;
    int32_t before = 0;   // the largest offset so far
    for (uint32_t s0 = 0; s0 < A.sequences; s0 += 64) {
      const uint32_t s = min(s0 + lane, A.sequences - 1);
      int32_t q0 = s * A.max_tokens, q1 = q0 + A.max_tokens;
      if (A.offsets) q0 = A.offsets[s], q1 = A.offsets[s + 1];
      int32_t most = max(q0, before);
      if (__any(q1 < q0 || before > q0)) {   // (else they are in order)
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
          const int32_t other = __shfl_up(most, o);
          if (lane >= (uint32_t)o) most = max(most, other);
        }
      }
      before = __shfl(most, 63);
      uint32_t n = 0, len = (uint32_t)A.length[s];
      if (most > q0 || fronk::bad_sequence(0, 1, q0, q1, A.tokens, A.max_tokens)) bad |= FR_HIP_BAD_OFFSET, len = 0;
      else if (n = q1 - q0, (int32_t)len < (int32_t)n || len > A.max_context) bad |= FR_HIP_BAD_LENGTH, len = 0;
      longest = max(longest, len);
      if (s0 + lane < A.sequences) length[s] = len, blocks[s] = (n * A.per + ROWS - 1) / ROWS, start[s] = q0, drafts[s] = n;
    }
    if (blockIdx.x == 0 && A.status && bad) atomicOr(A.status, bad);
#pragma unroll
    for (int o = 1; o < 64; o *= 2) longest = max(longest, (uint32_t)__shfl_xor((int)longest, o));
    if (lane == 0) found[0] = ~0u, found[1] = longest;
  }
  __syncthreads();
  uint32_t chunk = ((max(found[1], 1u) + 63) & ~63u);
  auto count = [&](uint32_t s, uint32_t chunk, uint32_t reciprocal) { return fronk::stretches(length[s], chunk, reciprocal); };
  if (A.slots) {
    // (2^(7/8) and so on; 64 of these: 2^7.9 stretches of the longest)
    const uint32_t mine = fronk::stretch_bound(chunk, lane ? __builtin_amdgcn_exp2f(lane * -.125f) : 1.f);
    const uint32_t reciprocal = 0xffffffffu / mine;
    uint32_t total = 0;
    for (uint32_t s = wave; s < A.sequences; s += W)
      if (blocks[s]) total += blocks[s] * count(s, mine, reciprocal);
    sums[wave * 64 + lane] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) total += sums[w * 64 + lane];
    total *= heads;
    // (in 64 tokens; what has too many workgroups, or stretches beyond all use, comes last)
    const uint32_t most = (1u << 26) - 1;
    uint32_t best = (total <= A.slots ? min(cost(total, mine), most) : most) << 6 | lane;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) best = min(best, (uint32_t)__shfl_xor((int)best, o));
    chunk = __shfl((int)mine, (int)(best & 63));
  }
  if (wave == 0) {
    const uint32_t reciprocal = 0xffffffffu / chunk;
    uint32_t total = 0;
    for (uint32_t s0 = 0; s0 < A.sequences; s0 += 64) {
      const uint32_t s = s0 + lane;
      const uint32_t n = s < A.sequences && blocks[s] ? count(s, chunk, reciprocal) : 0, work = n ? n * blocks[s] * heads : 0;
      uint32_t sum = work;
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const uint32_t other = __shfl_up((int)sum, o);
        if (lane >= (uint32_t)o) sum += other;
      }
      if (s < A.sequences) {
        first[s] = total + sum - work, stretches[s] = n;
        if (blockIdx.x == 0 && A.slots) A.plan[s] = uint2v{total + sum - work, n};
      }
      total += __shfl((int)sum, 63);
    }
    const uint32_t mine = in_list(total);
    if (mine != ~0u)
      for (uint32_t s = lane; s < A.sequences; s += 64)
        if (mine - first[s] < stretches[s] * blocks[s] * heads) found[0] = s;
    found[2] = mine;
  }
  __syncthreads();
  p.seq = same(found[0]), p.part = same(found[2]);
  if (p.part == ~0u) return p;
  p.d = Drafts{same(start[p.seq]), (uint32_t)same(drafts[p.seq]), (uint32_t)same(length[p.seq]), 0};
  p.splits = same(stretches[p.seq]);
  at(p.part - same(first[p.seq]), same(blocks[p.seq]));
  __syncthreads();   // (LDS is written anew)
  return p;
}
template <typename T> __device__ __forceinline__ T* draft_row(const TreeArgs& A, const Drafts& S, uint32_t head, uint32_t row) {
  return static_cast<T*>(A.o) + (int64_t)(S.q0 + row / A.per) * A.o_token + (int64_t)(head * A.per + row % A.per) * A.o_head;
}

// One workgroup: one sequence, one cache head, 32 RG of its rows (query heads of that
// cache head by drafts, draft-major) and one stretch of the context. Its W wavefronts
// are RG groups of 32 rows by KG groups of keys; each takes every KG-th tile of KT keys,
// and the key groups are joined in LDS at the end. Products and fragments are those of
// prompt_attend (attend.h), but that codes become operands as they are read from LDS:
// there they are as the cache has them, which halves the bytes of its tiles and reads.
// Codes times one are exact in bf16 and fp16; a token's powers of two go to its K
// operand, or its scores (fp16, whose range they may leave), and to its weights.
//
// Bound by the vector work of making operands of the codes, masks, exponentials and
// parts of P, by waits between it and the matrix work, and for few tiles by beginning and
// end; memory is read at a quarter to a half of its rate. 24 sequences of up to 8192 tokens
// with 1 to 61 drafts (16 heads of 128, four of the cache): in fp16 60 us and 6.0 for the join,
// the vector units busy for 44 % of the cycles and the matrix cores for 26; in bf16 60 and 6.0,
// in fp32 81 and 6.5. 32 equal ones with 64 drafts in bf16: 240 us. One of 32768 tokens with 15 drafts
// (16 heads of 256, two of the cache, bf16): 33.4 us and 5.7 (32 % and 19), of which 8 pass until the
// first tile is there, 4 with each of four tiles, 4 with the join in LDS and 2 with writing 17
// MB of parts; in fp32 86 and 5.7, as two of a unit's four SIMDs have work. One to eight registers of
// the 16-bit forms at dim 256, and three of fp32's at dim 128 and 64 rows, are in scratch.
//
// K in LDS: [token][dim], chunk c of 16 codes at another place for each of eight
// tokens, so that a read of one chunk of 32 of them goes to all banks; a lane's 16
// codes are operands of two steps (Q is laid out alike). V: [block of 16 tokens][dim]
// [16 tokens]; rows of K's operand are tokens in an order that leaves a lane of half h with
// the weights of tokens 16 s + 8 h .. 16 s + 8 h + 7, eight bytes of V.
//
// Q is an exact operand (fp32: three bf16 parts); P 2^e is in bf16 parts, of which there
// are as many as keep it well below the output's own rounding: two for 16-bit types,
// as in kv_attend, three for fp32. (In bf16 one made outputs off by 2^-8 of the weighted
// values' size; the ragged batch above took 53.6 us so and takes 62, one stream of 32768
// tokens and 15 drafts 34.9 and 39.6.)
template <typename T> struct Row;
template <> struct Row<__bf16> {   // (kFold: K's powers of two go into its operand)
  static constexpr bool kFold = true;
  typedef bf16x8 frag;
  static constexpr int kQ = 1, kP = 2;
};
template <> struct Row<_Float16> {
  static constexpr bool kFold = false;
  typedef half8v frag;
  static constexpr int kQ = 1, kP = 2;
};
template <> struct Row<float> {
  static constexpr bool kFold = true;
  typedef bf16x8 frag;
  static constexpr int kQ = 3, kP = 3;
};

// Wavefronts, keys of a tile, stages, wavefronts a SIMD that the registers are for.
// Where Q's three parts do not fit them beside the sums, Q is kept in LDS, and split
// where it is used. Two stages: with three, one workgroup less fits a unit (32 sequences of
// 8192 tokens and 64 drafts, bf16, dim 128: 240 us with two, 298 with three); tiles of 32 keys
// instead of 64 there: 255. Eight wavefronts at dim 256, as four of 512 registers each are
// slower (one stream of 32768 tokens 43 us for 39.5).
template <typename T, int D> constexpr bool kTreeQInLds = D * sizeof(T) > 512;
template <typename T, int D, int RG> constexpr int kTreeWaves = kTreeQInLds<T, D> ? 2 : D == 256 && RG > 1 ? 8 : 4;
template <int D, int RG> constexpr int kTreeKeys = D == 256 || (D == 128 && RG == 1) ? 32 : 64;
constexpr int kTreeStages = 2;
template <typename T, int D> constexpr int kTreeResident = sizeof(T) == 2 && D == 64 ? 3 : 2;
// LDS: the stages, and Q; at the end the key groups are joined in it.
template <typename T, int D, int RG> constexpr size_t kTreeTiles =
    (size_t)kTreeStages * (kTreeWaves<T, D, RG> / RG) * 2 * kTreeKeys<D, RG> * D;
template <typename T, int D, int RG> constexpr size_t kTreeUsed = kTreeTiles<T, D, RG> + (kTreeQInLds<T, D> ? 128 * RG * D : 0);
template <typename T, int D, int RG> constexpr size_t kTreeJoin = RG == kTreeWaves<T, D, RG> ? 0 : 64 * kTreeWaves<T, D, RG> * (D + 4);
template <typename T, int D, int RG> constexpr size_t kTreeLds = kTreeUsed<T, D, RG> > kTreeJoin<T, D, RG> ? kTreeUsed<T, D, RG> : kTreeJoin<T, D, RG>;

// The turn of a token's chunks of K in LDS: another one for each of eight lanes that
// follow each other, whose tokens differ in bits 0, 1 and 3.
template <int D> __device__ __forceinline__ uint32_t turn_of(uint32_t token) {
  return D == 64 ? (token >> 1 & 1) | (token >> 2 & 2) : (token & 3) | (token >> 1 & 4);
}

// A lane's four bytes to consecutive places, as to_lds.
__device__ __forceinline__ void four_to_lds(const void* from, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(at), "v"(from) : "memory", "m0");
}

template <typename T, int D, int RG>
__global__ __launch_bounds__((64 * kTreeWaves<T, D, RG>), (kTreeResident<T, D>)) void kv_attend_tree(TreeArgs A) {
  typedef Row<T> Q;
  typedef typename Q::frag frag;
  constexpr int W = kTreeWaves<T, D, RG>, QP = Q::kQ, PP = Q::kP, KG = W / RG, KT = kTreeKeys<D, RG>, S = kTreeStages;
  constexpr int KS = D / 32, ST = KT / 32, DT = D / 32, kRows = 32 * RG;
  constexpr uint32_t kHalf = KT * D, kStage = KG * 2 * kHalf;      // a tile's K, or V; a stage
  constexpr uint32_t kLoads = kHalf / 1024 / RG;                   // of a wavefront: a tile's K, or V, 64 units of 16 codes each
  constexpr int kPerStage = 2 * kLoads + 1;
  constexpr uint32_t kUnits = D / 16;                              // a token's units of K
  extern __shared__ __attribute__((aligned(16))) char lds[];       // [S][KG][K, V][kHalf]
  __shared__ __attribute__((aligned(16))) uint8_t exps[S][W][2][KT];
  __shared__ __attribute__((aligned(16))) float powers[W][Q::kFold ? 1 : 2][KT];   // of a tile's values, and keys
  __shared__ float stat[W][32][2];
  __shared__ uint64_t seen_words[W][32];   // the drafts that a row sees (by its own wavefront)

  const uint32_t lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % RG, kg = wave / RG;
  const Cache& C = A.cache;
  static_assert(kTreeLds<T, D, RG> >= kPlanBytes, "the plan is made in the tiles' place");
  const Place place = plan<W, kRows, D>(A, reinterpret_cast<uint32_t*>(lds));
  if (place.part == ~0u) return;
  const Drafts P = place.d;
  const uint32_t seq = place.seq, head = place.head, block = place.block;
  const uint32_t rows = P.n * A.per, row0 = block * kRows;
  const uint32_t begin = place.split * place.chunk, end = max(begin, min(P.length, begin + place.chunk));
  const uint32_t prefix = P.length - P.n;
  const uint32_t wave_row = row0 + rg * 32, row = wave_row + i;
  const int32_t* const table = A.table + (size_t)seq * A.table_stride;
  // Where 64 blocks of 16 tokens are (in blocks of the cache; kGone: their page is not
  // there), a lane each, and the 64 behind them. Blocks past the end are taken to be the
  // last one.
  constexpr uint32_t kGone = ~0u;
  uint32_t first_place = begin >> 4;   // the block of `places`' first lane; a stage is of whole ones of 64
  auto look_up = [&](uint32_t block) {
    const uint32_t n = min(block + lane, (end - 1) >> 4);
    uint32_t q = __umulhi(n, A.reciprocal), r = n - q * A.page16;   // q or one below
    if (r >= A.page16) ++q, r -= A.page16;
    const int32_t page = table[q];
    return fronk::page_there(page, C.pages) ? ((uint32_t)page * C.heads + head) * A.page16 + r : kGone;
  };
  uint32_t places = 0, places_next = 0;
  bool missing = false;
  uint32_t gone = 0;       // four bits a stage: blocks of the tile that are not there
  // A stage's loads: this wavefront's part of its key group's tile, 64 units of 16 codes
  // each, and all of the tile's exponents. (Past the end they are the last block's once
  // more, so that there are always as many in flight.)
  const uint32_t lane_token = lane / kUnits, lane_unit = lane % kUnits;
  const uint32_t k_lane = (lane_token * kUnits + (lane_unit ^ turn_of<D>(lane_token))) * 16;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)lds + kg * 2 * kHalf;
  const uint32_t exps0 = (uint32_t)(uintptr_t)(lds_char*)reinterpret_cast<char*>(&exps[0][wave][0][0]);
  const uint8_t* const e_lane = (lane < KT / 4 ? C.k_exp : C.v_exp) + lane % 4 * 4;
  auto load = [&](uint32_t base, uint32_t stage) __attribute__((always_inline)) {
    if ((base >> 4) - first_place >= 64) first_place += 64, places = places_next, places_next = look_up(first_place + 64);
    const uint32_t first = (base >> 4) - first_place + kg * (KT / 16);
    uint32_t bits = 0;
#pragma unroll
    for (uint32_t b = 0; b < KT / 16; ++b) bits |= (uint32_t)(__builtin_amdgcn_readlane(places, first + b) == kGone) << b;
    gone = (gone & ~(15u << 4 * stage)) | bits << 4 * stage, missing |= bits;
    const uint32_t to_k = lds0 + stage * kStage;
#pragma unroll
    for (uint32_t l = 0; l < kLoads; ++l) {
      const uint32_t u = rg * 64 + l * RG * 64, token = u / kUnits % 16;
      const uint32_t place = __builtin_amdgcn_readlane(places, first + u / D);
      const size_t from = (size_t)(place == kGone ? 0 : place) * (16 * D);
      to_lds(reinterpret_cast<const char*>(C.k_codes) + from + token * D, k_lane ^ turn_of<D>(token) * 16, to_k + u * 16);
      to_lds(reinterpret_cast<const char*>(C.v_codes) + from + u % D * 16, lane * 16, to_k + kHalf + u * 16);
    }
    const uint32_t place = __shfl(places, (int)(first + lane % (KT / 4) / 4));
    if (lane < KT / 2) four_to_lds(e_lane + (size_t)(place == kGone ? 0 : place) * 16, exps0 + stage * (W * 2 * KT));
  };

  if (begin < end) {
    places = look_up(first_place), places_next = look_up(first_place + 64);
#pragma unroll 1
    for (uint32_t k = 0; k < S - 1; ++k) load(begin + k * KG * KT, k);
  }

  if (h == 0) seen_words[wave][i] = row < rows ? (uint64_t)A.tree[P.q0 + row / A.per] & (~0ull >> (64 - P.n)) : 0;
  // Drafts that any sees: what is held of others may be anything.
  uint64_t any_seen = lane < P.n ? (uint64_t)A.tree[P.q0 + lane] : 0;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) any_seen |= __shfl_xor((unsigned long long)any_seen, o);
  any_seen = (uint32_t)same((int32_t)any_seen) | (uint64_t)(uint32_t)same((int32_t)(any_seen >> 32)) << 32;
  // Q: lane (i, h) of step 2 s + j holds row i's dims 32 s + 16 h + 8 j ..
  constexpr bool kQInLds = kTreeQInLds<T, D>;
  frag qf[kQInLds ? 1 : QP][kQInLds ? 1 : 2 * KS];
  float4v* const q_lds = reinterpret_cast<float4v*>(lds + kTreeTiles<T, D, RG>) + (rg * 2 * KS * 64 + lane) * 2;   // 128 on for each step
  {
    const uint32_t r = min(row, rows - 1);
    const T* p = static_cast<const T*>(A.q) + (int64_t)(P.q0 + r / A.per) * A.q_token +
                 (int64_t)(head * A.per + r % A.per) * A.q_head + h * 16;
    auto take = [&](bool wide) __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < 2 * KS; ++s) {
        float x[8];
        load_row<8>(p + s / 2 * 32 + s % 2 * 8, wide, x);
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
    };
    if constexpr (kQInLds) {
      if (kg == 0) {
#pragma unroll 2
        for (int s = 0; s < 2 * KS; ++s) {
          float x[8];
          load_row<8>(p + s / 2 * 32 + s % 2 * 8, A.wide, x);
          const float one = A.scale < 0.f ? -1.f : 1.f;
          q_lds[s * 128] = float4v{x[0], x[1], x[2], x[3]} * one, q_lds[s * 128 + 1] = float4v{x[4], x[5], x[6], x[7]} * one;
        }
      }
    } else if constexpr (QP == 1) {
      if (A.wide) {
#pragma unroll
        for (int s = 0; s < 2 * KS; ++s) qf[0][s] = *reinterpret_cast<const frag*>(p + s / 2 * 32 + s % 2 * 8);
      } else {
        take(false);
      }
    } else {
      if (A.wide) take(true);
      else take(false);
    }
    // A negative scale is taken to Q, as in prompt_attend.
    const uint32_t sign = A.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int q = 0; q < (kQInLds ? 0 : QP); ++q)
#pragma unroll
      for (int s = 0; s < 2 * KS; ++s) qf[q][s] = __builtin_bit_cast(frag, __builtin_bit_cast(uint4v, qf[q][s]) ^ sign);
  }

  const float scale = fmaxf(fabsf(A.scale) * kLog2e, 1e-37f);
  float top = -INFINITY, shift = 0, sum = 0;
  float16v acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = float16v{};
  bool poisoned = false;
  // Row i of a K operand is the token with bits 2 and 3 of i changed over, which leaves a
  // lane in half h, in registers 8 s .. 8 s + 7, with tokens 16 s + 8 h ..: eight bytes of V.
  const uint32_t k_token = (i & ~12u) | (i & 4) << 1 | (i & 8) >> 1;

  auto compute = [&](uint32_t base, uint32_t stage) __attribute__((always_inline)) {
    base += kg * KT;
    if (base >= end) return;
    char* const kt = lds + stage * kStage + kg * 2 * kHalf;
    char* const vt = kt + kHalf;
    const uint32_t none = gone >> 4 * stage & 15;
    // A tile of which rows see different parts, or not all is there; and tokens held with
    // infinities or NaN (as zeros).
    const uint32_t ke = exps[stage][wave][0][lane % KT], ve = exps[stage][wave][1][lane % KT];
    const bool masked = base + KT > prefix || base + KT > end || none || __any(ke == 255 || ve == 255);
    powers[wave][0][lane % KT] = ve == 255 ? 0.f : power(ve);
    float k_power[ST];
    if constexpr (Q::kFold) {
#pragma unroll
      for (int t = 0; t < ST; ++t) {
        const uint32_t e = exps[stage][wave][0][t * 32 + k_token];
        k_power[t] = e == 255 ? 1.f : power(e);   // (zero codes)
      }
    } else {
      powers[wave][1][lane % KT] = ke == 255 ? 0.f : power(ke);
    }
    uint32_t seen_bits[ST] = {}, bad_bits[ST] = {};
    if (masked) {
      const uint64_t bad_k = __ballot(ke == 255), bad_v = __ballot(ve == 255), seen = seen_words[wave][i];
#pragma unroll
      for (int t = 0; t < ST; ++t) {
        const int32_t left = (int32_t)(end - base) - t * 32, first = (int32_t)(base + t * 32 - prefix);
        uint32_t there = left >= 32 ? ~0u : left <= 0 ? 0u : ~(~0u << left);
        if (none >> 2 * t & 1) there &= 0xffff0000u;
        if (none >> 2 * t & 2) there &= 0x0000ffffu;
        // Which of 32 tokens are seen: all before the drafts, and of those the words' bits.
        auto of = [&](uint64_t word) {
          const uint32_t bits = first <= -32 ? ~0u : first >= 64 ? 0u : first < 0 ? (uint32_t)(word << -first) | ~(~0u << -first) : (uint32_t)(word >> first);
          return bits & there;
        };
        seen_bits[t] = of(seen);
        bad_bits[t] = seen_bits[t] & (uint32_t)(bad_k >> 32 * t);
        poisoned |= (seen_bits[t] & (uint32_t)(bad_v >> 32 * t)) || bad_bits[t];
        // Codes of V that count for nothing may be no numbers: zeros (which all
        // wavefronts of the tile write alike).
        const uint32_t any = of(any_seen);
        if (any != ~0u)
          for (uint32_t u = lane; u < 2 * D; u += 64) {
            uint4v* const c = reinterpret_cast<uint4v*>(vt + t * 32 * D) + u;
            uint4v x = *c;
#pragma unroll
            for (int w = 0; w < 4; ++w) x[w] &= ((any >> (u / D * 16 + 4 * w) & 15) * 0x00204081u & 0x01010101u) * 255u;
            *c = x;
          }
      }
    }
    // Each step's operands are read while the one before it is worked on.
    __builtin_amdgcn_s_setprio(1);   // (matrix work before other wavefronts': 7 % less at 64 rows)
    float16v st[ST];
    // Reads at once, as many as registers are left for.
    constexpr int kK = KS == 4 ? 2 : 1, kV = D == 256 ? 2 : DT < 4 ? DT : 4;
    uint4v kc[2][kK];
    auto read_k = [&](int n) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const int s = n % (KS / kK) * kK + k;
        kc[n % 2][k] = *reinterpret_cast<const uint4v*>(kt + (n / (KS / kK) * 32 + k_token) * D + ((2 * s + h) ^ turn_of<D>(k_token)) * 16);
      }
    };
    read_k(0);
#pragma unroll
    for (int n = 0; n < ST * KS / kK; ++n) {
      __builtin_amdgcn_sched_barrier(0);
      if (n + 1 < ST * KS / kK) read_k(n + 1);
      __builtin_amdgcn_sched_barrier(0);
      const int t = n / (KS / kK);
      if (n % (KS / kK) == 0) st[t] = float16v{};
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const uint4v c = kc[n % 2][k];
        const int step = 2 * (n % (KS / kK) * kK + k);
        frag a, b;
        if constexpr (Q::kFold) a = codes8(c[0], c[1], k_power[t], frag{}), b = codes8(c[2], c[3], k_power[t], frag{});
        else a = codes8(c[0], c[1], frag{}), b = codes8(c[2], c[3], frag{});
        if constexpr (kQInLds) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float4v x = q_lds[(step + j) * 128], y = q_lds[(step + j) * 128 + 1];
            const float row[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            bf16x8 parts[QP];
            split8<QP>(row, parts);
#pragma unroll
            for (int q = QP - 1; q >= 0; --q) st[t] = mma32(j ? b : a, __builtin_bit_cast(frag, parts[q]), st[t]);
          }
        } else {
#pragma unroll
          for (int q = QP - 1; q >= 0; --q) st[t] = mma32(a, qf[q][step], st[t]);
#pragma unroll
          for (int q = QP - 1; q >= 0; --q) st[t] = mma32(b, qf[q][step + 1], st[t]);
        }
      }
    }
    uint2v vc[2][kV];
    auto read_v = [&](int n) __attribute__((always_inline)) {   // of 16 tokens
#pragma unroll
      for (int d = 0; d < kV; ++d)
        vc[n % 2][d] = *reinterpret_cast<const uint2v*>(vt + (n / (DT / kV) * D + (n % (DT / kV) * kV + d) * 32 + i) * 16 + h * 8);
    };
    if constexpr (!Q::kFold) {
#pragma unroll
      for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4v f = *reinterpret_cast<const float4v*>(&powers[wave][1][t * 32 + g / 2 * 16 + 8 * h + g % 2 * 4]);
#pragma unroll
          for (int e = 0; e < 4; ++e) st[t][g * 4 + e] *= f[e];
        }
    }
    if (masked) {
#pragma unroll
      for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!(seen_bits[t] >> (8 * h) & 1u << (16 * (r / 8) + r % 8))) st[t][r] = -INFINITY;
    }
    __builtin_amdgcn_s_setprio(0);
    const float most = max_xor32(largest(st));
    if (__any(most * scale > top * scale + 8.f)) {   // (as in prompt_attend)
      const float now = fmaxf(top, most), to = now == -INFINITY ? 0.f : now * scale;
      const float f = __builtin_amdgcn_exp2f(top * scale - to);
      top = now, shift = to, sum *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f;
    }
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 pf[ST][2][PP];
    float total[4] = {};
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float w[8];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const float4v f = *reinterpret_cast<const float4v*>(&powers[wave][0][t * 32 + s * 16 + 8 * h + 4 * g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][s * 8 + g * 4 + e], scale, -shift));
            total[e] += p;
            w[g * 4 + e] = p * f[e];
          }
        }
        split8<PP>(w, pf[t][s]);
      }
    sum += (total[0] + total[1]) + (total[2] + total[3]);
    read_v(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int n = 0; n < 2 * ST * (DT / kV); ++n) {
      __builtin_amdgcn_sched_barrier(0);
      if (n + 1 < 2 * ST * (DT / kV)) read_v(n + 1);
      __builtin_amdgcn_sched_barrier(0);
      const int s = n / (DT / kV);
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        const int d = n % (DT / kV) * kV + k;
        const bf16x8 a = codes8(vc[n % 2][k][0], vc[n % 2][k][1], bf16x8{});
#pragma unroll
        for (int p = PP - 1; p >= 0; --p) acc[d] = mma32(a, pf[s / 2][s % 2][p], acc[d]);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };

  if (begin < end) {
    uint32_t stage = 0;
#pragma unroll 1
    for (uint32_t base = begin; base < end; base += KG * KT) {
      loads_done<(S - 2) * kPerStage>();   // and all wavefronts'
      load(base + (S - 1) * KG * KT, (stage + S - 1) % S);
      if (wave_row < rows) compute(base, stage);
      stage = (stage + 1) % S;
    }
    if (missing && A.status) atomicOr(A.status, FR_HIP_BAD_PAGE);
    loads_done<0>();
  }

  sum = add_xor32(sum);
  if (poisoned) sum = NAN;
  const bool many = place.splits > 1;
  if constexpr (KG > 1) {
    // Join the key groups by halves, in LDS; from there all write the rows.
    if (h == 0) stat[wave][i][0] = sum == 0.f ? -INFINITY : shift, stat[wave][i][1] = sum;
    __syncthreads();
    float all = -INFINITY;
#pragma unroll
    for (int g = 0; g < KG; ++g) all = fmaxf(all, stat[g * RG + rg][i][0]);
    const float to = all == -INFINITY ? 0.f : all, mine = stat[wave][i][0];
    const float f = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - to);
    float joined = 0;
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const float m = stat[g * RG + rg][i][0];
      if (m != -INFINITY) joined += stat[g * RG + rg][i][1] * __builtin_amdgcn_exp2f(m - to);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] *= f;
    constexpr uint32_t kPitch = D + 4;
    float* const o = reinterpret_cast<float*>(lds);
    auto lds_row = [&](uint32_t group, int d, int q) __attribute__((always_inline)) {
      return reinterpret_cast<float4v*>(o + (group * kRows + rg * 32 + i) * kPitch + d * 32 + q * 8 + 4 * h);
    };
#pragma unroll
    for (int half = KG / 2; half >= 0; half /= 2) {
      if (kg >= (uint32_t)half && kg < (uint32_t)(half ? 2 * half : 1)) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *lds_row(kg - half, d, q) = float4v{acc[d][q * 4], acc[d][q * 4 + 1], acc[d][q * 4 + 2], acc[d][q * 4 + 3]};
        if (!half && h == 0) stat[wave][i][0] = joined == 0.f ? -INFINITY : to, stat[wave][i][1] = joined;
      }
      __syncthreads();
      if (!half) break;
      if (kg < (uint32_t)half) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4v x = *lds_row(kg, d, q);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[d][q * 4 + e] += x[e];
          }
      }
      __syncthreads();
    }
    const size_t part = (size_t)place.part * kRows;
    for (uint32_t e = threadIdx.x; e < kRows * (D / 4); e += 64 * W) {
      const uint32_t r = e / (D / 4), d = e % (D / 4) * 4;
      if (row0 + r >= rows) break;
      const float total = stat[r / 32][r % 32][1];
      const float4v x = *reinterpret_cast<const float4v*>(o + r * kPitch + d);
      if (many) {
        if (d == 0) A.part_ml[(part + r) * 2] = stat[r / 32][r % 32][0], A.part_ml[(part + r) * 2 + 1] = total;
        if (begin < end) part_store(A.part_o + (part + r) * D + d, x);
      } else {
        put4<T>(draft_row<T>(A, P, head, row0 + r) + d, x, total, A.wide);
      }
    }
    return;
  }
  if (row >= rows) return;
  if (many) {
    const size_t to = (size_t)place.part * kRows + (row - row0);
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
  T* const p = draft_row<T>(A, P, head, row) + 4 * h;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      put4<T>(p + d * 32 + g * 8, float4v{acc[d][g * 4], acc[d][g * 4 + 1], acc[d][g * 4 + 2], acc[d][g * 4 + 3]}, sum, A.wide);
}

// The stretches of rows joined: one row a workgroup, or as many as have D / 4 lanes.
template <typename T, int D, bool MANY>
__global__ __launch_bounds__(256) void tree_merge(TreeArgs A, uint32_t block_rows) {
  constexpr uint32_t L = D / 4, kAtOnce = MANY ? 1 : 256 / L;
  const uint32_t parts = block_rows / kAtOnce;
  const uint32_t item = blockIdx.x / parts, r = blockIdx.x % parts * kAtOnce + (MANY ? 0 : threadIdx.x / L);
  const uint32_t head = item % A.cache.heads, block = item / A.cache.heads % A.blocks, seq = item / A.cache.heads / A.blocks;
  const uint2v plan = A.plan[seq];
  Drafts W = {(int32_t)(seq * A.max_tokens), A.max_tokens, 0, 0};
  if (A.offsets) W.q0 = A.offsets[seq], W.n = A.offsets[seq + 1] - W.q0;
  if (plan[1] < 2) return;   // (written as it is)
  const uint32_t row = block * block_rows + r, rows = W.n * A.per;
  if (row >= rows) return;
  float sum;
  const uint32_t blocks = (rows + block_rows - 1) / block_rows, apart = A.cache.heads * blocks * block_rows;
  const size_t part = (size_t)(plan[0] + head * blocks + block) * block_rows + r;
  const float4v x = MANY ? join_many<D>(A.part_o, A.part_ml, part, plan[1], apart, &sum)
                         : join_few<D>(A.part_o, A.part_ml, part, plan[1], apart, &sum);
  if (!MANY || threadIdx.x < L) put4<T>(draft_row<T>(A, W, head, row) + threadIdx.x % L * 4, x, sum, A.wide);
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
  if ((uint64_t)r->cache.pages * r->cache.heads * (r->cache.page / 16) >= UINT32_MAX) return FR_HIP_UNSUPPORTED;
  if (r->max_tokens > 64 || r->heads / r->cache.heads > 64) return FR_HIP_UNSUPPORTED;
  return FR_HIP_OK;
}

// How a call is cut: blocks of 32 `groups` rows of a sequence, and into how many
// workgroups at most (plan).
struct TreeCut {
  uint32_t groups, blocks, at_once, slots;
  uint64_t items, grid;
  size_t bytes;
};
TreeCut tree_cut(const fr_hip_kv_tree* r) {
  TreeCut c;
  const uint32_t drafts = r->max_tokens < r->tokens ? r->max_tokens : r->tokens;
  const uint32_t rows = drafts * (r->heads / r->cache.heads);
  // 64 rows, or 32 where there are no more: 16 sequences of 8192 tokens with 8 drafts of four
  // heads (bf16, dim 128) take 40.2 us in groups of 32 and 40.8 of 64, with 16 drafts 52.0 and 49.8, 32
  // of them with 64 drafts 286 and 238 (128 rows: the same to 20 % slower at 16 to 64 drafts).
  c.groups = rows <= 32 ? 1 : 2;
  c.blocks = (rows + 32 * c.groups - 1) / (32 * c.groups);
  c.items = (uint64_t)c.blocks * r->sequences * r->cache.heads;
  // Two workgroups a unit at once, one at dim 256 (16 drafts over 131072 tokens, 16 heads, bf16: two
  // key heads of 256 84 us with one a unit and 104 with two, four of 128 50 and 47); up to
  // three such rounds are split, and no call of more sequences than are planned: beyond, each of
  // a sequence's blocks is one workgroup's, however long it is.
  c.at_once = kUnits * (r->cache.dim == 256 ? 1 : 2);
  const uint64_t rounds = (c.items + c.at_once - 1) / c.at_once;
  c.slots = rounds > 3 || r->sequences > kPlanned || r->max_context <= 256 ? 0 : (uint32_t)rounds * c.at_once;
  c.grid = ((c.items > c.slots ? c.items : c.slots) + 7) / 8 * 8;
  c.bytes = c.slots ? (size_t)c.slots * 32 * c.groups * (r->cache.dim + 2) * sizeof(float) + r->sequences * sizeof(uint2v) : 0;
  return c;
}
// Grids of less than 2^32 threads.
bool tree_fits(const TreeCut& c) {
  return c.grid * 512 <= UINT32_MAX && c.items * 32 * c.groups * 256 <= (c.slots ? UINT32_MAX : UINT64_MAX);
}

template <typename T, int D, int RG>
int launch_tree(const TreeArgs& A, const TreeCut& c, hipStream_t s) {
  static fronk::Devices done;
  if (allow_lds(kv_attend_tree<T, D, RG>, kTreeLds<T, D, RG>, &done)) return FR_HIP_IO;
  hipLaunchKernelGGL((kv_attend_tree<T, D, RG>), dim3((uint32_t)c.grid), dim3(64 * kTreeWaves<T, D, RG>), (kTreeLds<T, D, RG>), s, A);
  return FR_HIP_OK;
}
template <typename T, int D>
int launch_dim(const TreeArgs& A, const TreeCut& c, hipStream_t s) {
  const int rc = c.groups == 1 ? launch_tree<T, D, 1>(A, c, s) : launch_tree<T, D, 2>(A, c, s);
  if (rc) return rc;
  const uint32_t rows = 32 * c.groups;
  if (c.slots && c.items * rows < kJoinRows) hipLaunchKernelGGL((tree_merge<T, D, true>), dim3((uint32_t)(c.items * rows)), dim3(256), 0, s, A, rows);
  else if (c.slots) hipLaunchKernelGGL((tree_merge<T, D, false>), dim3((uint32_t)(c.items * rows / (1024 / D))), dim3(256), 0, s, A, rows);
  FRONK_CK(hipGetLastError());
  return FR_HIP_OK;
}
template <typename T>
int launch_dims(const TreeArgs& A, const TreeCut& c, hipStream_t s) {
  switch (A.cache.dim) {
    case 64: return launch_dim<T, 64>(A, c, s);
    case 128: return launch_dim<T, 128>(A, c, s);
    default: return launch_dim<T, 256>(A, c, s);
  }
}

}  // namespace

extern "C" {

size_t fr_hip_tree_workspace(const fr_hip_kv_tree* r) {
  if (check_tree(r)) return 0;
  const TreeCut c = tree_cut(r);
  return tree_fits(c) ? c.bytes : 0;
}

int fr_hip_kv_attend_tree(const fr_hip_kv_tree* r, void* workspace, size_t bytes, void* stream) {
  int rc = check_tree(r);
  if (rc) return rc;
  const TreeCut c = tree_cut(r);
  if (!tree_fits(c)) return FR_HIP_UNSUPPORTED;
  if (c.bytes && (!workspace || bytes < c.bytes || (uintptr_t)workspace % 16)) return FR_HIP_INVALID;
  hipStream_t s;
  rc = fronk::enter(stream, &s);
  if (rc || !c.items) return rc;
  TreeArgs A;
  A.cache = cache_of(r->cache);
  A.q = r->q, A.o = r->o, A.tree = r->tree, A.offsets = r->offsets, A.table = r->table, A.length = r->length;
  A.status = r->status;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + (size_t)c.slots * 32 * c.groups * r->cache.dim;
  A.plan = reinterpret_cast<uint2v*>(A.part_ml + (size_t)c.slots * 32 * c.groups * 2);
  A.q_token = r->q_token, A.q_head = r->q_head, A.o_token = r->o_token, A.o_head = r->o_head;
  A.sequences = r->sequences, A.tokens = r->tokens, A.max_tokens = r->max_tokens, A.per = r->heads / r->cache.heads;
  A.max_context = r->max_context, A.table_stride = r->table_stride, A.blocks = c.blocks;
  A.slots = c.slots, A.at_once = c.at_once;
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
