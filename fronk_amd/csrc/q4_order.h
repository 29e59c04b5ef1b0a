// q4_order.h - the order in which q4_tiles' wavefronts use the two LDS buffers
// of x, apart from what they do between, so that it is tested on the host.
//
// Block k lies in buffer k % 2. All wavefronts of a half store a part of it, and
// all of them read all of it, so that there is a barrier between a store and the
// reads of what it stored, and between a buffer's last read and its next store.
//
// AHEAD: block k + 1 is read between the products of block k, and fetched two
// blocks before its product; otherwise block k is read before its products.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define FRONK_TILES __host__ __device__ __forceinline__
#else
#define FRONK_TILES inline
#endif

namespace fronk {

template <bool AHEAD> constexpr uint32_t kTilesLead = AHEAD ? 2 : 1;

// Before the first block. fetch(k): block k from memory into registers, store(k):
// from there into its buffer, read(k): its operands.
template <bool AHEAD, typename Fetch, typename Store, typename Barrier, typename Read>
FRONK_TILES void tiles_first(Fetch fetch, Store store, Barrier barrier, Read read) {
  fetch(0);
  store(0);
  if constexpr (AHEAD) {
    fetch(1);
    store(1);
    barrier();
    read(0);
    barrier();   // block 0's end stores to the buffer just read
  }
}
// Before block k's products ...
template <bool AHEAD, typename Fetch, typename Barrier, typename Read>
FRONK_TILES void tiles_before(uint32_t k, Fetch fetch, Barrier barrier, Read read) {
  if constexpr (!AHEAD) {
    barrier();   // this block's x is there, and the last one's is read
    read(k);
  }
  fetch(k + kTilesLead<AHEAD>);
}
// ... and behind them.
template <bool AHEAD, typename Store, typename Barrier>
FRONK_TILES void tiles_after(uint32_t k, Store store, Barrier barrier) {
  store(k + kTilesLead<AHEAD>);
  if constexpr (AHEAD) barrier();   // x of the block after the next is there, that of the next in registers
}

}  // namespace fronk
