// Who may use a warp's slot of shared memory, when blocks leave it by bulk stores
// that read it later.  Plain C++ with the bulk operations as a parameter, so that
// the order can be run on the host as well.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define WAVE_SLOT_FN __host__ __device__ __forceinline__
#else
#define WAVE_SLOT_FN inline
#endif

namespace wave {
namespace linear_detail {

// With halves the two of them are taken in turn, and a use waits until at most one
// bulk group is pending.  Groups complete in the order of their commits as far as
// that wait can tell, so the one that may be left is the newest -- which is the use
// before this one, of the other half, because EVERY use commits exactly one group:
// an empty one where it wrote its block without a bulk store.  (Were nothing
// committed there, the group left pending could be the store that still reads the
// half being taken.)  Without halves a use waits for all.
// Bulk: wait_read<N>() (at most N groups still read their source) and commit(), by
// the one thread that issues the stores.
template <bool kHalves, typename Bulk>
WAVE_SLOT_FN void slot_take(uint8_t *&slot, int &other_half, const Bulk &bulk) {
  if constexpr (kHalves) {
    slot += other_half;
    other_half = -other_half;
    bulk.template wait_read<1>();
  } else {
    bulk.template wait_read<0>();
  }
}
// Ends a use, whether its block left by a bulk store or not.
template <typename Bulk> WAVE_SLOT_FN void slot_leave(const Bulk &bulk) { bulk.commit(); }

} // namespace linear_detail
} // namespace wave
