// bounds.h - the bounds checks and addresses of what only the device can see
// (slots, pages, offsets), in plain C++ so that they are tested on the host.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define FRONK_BOTH __host__ __device__ __forceinline__
#else
#define FRONK_BOTH inline
#endif

namespace fronk {

// A cache slot's page and place in it; 0: skipped (-1), 1: there, 2: out of
// range.
FRONK_BOTH int locate(int32_t slot, uint32_t page_tokens, uint32_t pages, uint32_t* page, uint32_t* at) {
  if (slot == -1) return 0;
  *page = (uint32_t)slot / page_tokens;
  *at = (uint32_t)slot % page_tokens;
  return slot >= 0 && *page < pages ? 1 : 2;
}

FRONK_BOTH bool page_there(int32_t page, uint32_t pages) { return page >= 0 && (uint32_t)page < pages; }

// The exponent byte of a token of a page and head; times dim, byte 0 of its K
// codes.
FRONK_BOTH size_t exp_at(uint32_t heads, uint32_t page_tokens, uint32_t page, uint32_t head, uint32_t at) {
  return ((size_t)page * heads + head) * page_tokens + at;
}
// Its V code of dim 0; 16 bytes on for each dim.
FRONK_BOTH size_t v_at(uint32_t heads, uint32_t page_tokens, uint32_t dim, uint32_t page, uint32_t head, uint32_t at) {
  return (exp_at(heads, page_tokens, page, head, 0) + (at & ~15u)) * dim + (at & 15);
}

// Of four bytes, the first n.
FRONK_BOTH uint32_t first_bytes(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1; }

// What is wrong with a sequence's slot and offsets (FR_HIP_BAD_OFFSET 1,
// FR_HIP_BAD_SLOT 2), 0: nothing.
FRONK_BOTH uint32_t bad_sequence(int32_t slot, uint32_t slots, int32_t first, int32_t last, uint32_t tokens,
                                 uint32_t max_tokens) {
  uint32_t bad = 0;
  if (slot < -1 || (slot >= 0 && (uint32_t)slot >= slots)) bad |= 2;
  if (first < 0 || last < first || (uint32_t)last > tokens || (uint32_t)(last - first) > max_tokens) bad |= 1;
  return bad;
}

// A bound on the tokens of a stretch: `part` of the longest sequence's (a multiple of 64), 256 or
// more. A part of 1 is all of it, which leaves every sequence whole: not by way of a float, which from
// 2^30 on may be less.
FRONK_BOTH uint32_t stretch_bound(uint32_t longest, float part) {
  const uint32_t n = part < 1.f ? ((uint32_t)((float)longest * part) + 63) & ~63u : longest;
  return n > 256 ? n : 256;
}
// Stretches of at most `bound` tokens, at least one; reciprocal: 2^32 - 1 by it, rounded down.
FRONK_BOTH uint32_t stretches(uint32_t length, uint32_t bound, uint32_t reciprocal) {
  uint32_t n = (uint32_t)(((uint64_t)length * reciprocal) >> 32);   // this, one or two more
  while (n * bound < length) ++n;
  return n ? n : 1;
}

}  // namespace fronk
