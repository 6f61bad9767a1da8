// What the two softmax groups of a pair (attention.cu) tell each other about a tile: each has half of its keys, and both
// have to come to the same maximum, the same reference and the same decision to rescale, because the rescaling has a
// barrier of its own and a group that takes it alone waits there for good.
//
// So the decision hangs on nothing but what lies in the trade, read behind a barrier that both have passed. That has to
// hold for every order of the two groups that the barriers alone allow: once a bounded wait has run out all others
// return at once and order nothing any more. The reference of the tile before, which the other pair publishes, is
// therefore read by the first group alone and handed on; and a tile's trade is not the one of the group's tile before,
// so that a group which has gone on meets a barrier before it writes where the other may still read.
//
// Plain C++ beside the CUDA qualifiers: tests run it on the host.
#ifndef HALO_B200_SOFTMAX_PAIR_CUH_
#define HALO_B200_SOFTMAX_PAIR_CUH_

#include <cmath>
#include <cstdint>

#ifdef __CUDACC__
#define HALO_PAIR_FN __host__ __device__ __forceinline__
#else
#define HALO_PAIR_FN inline
#endif

namespace halo_b200 {

template <uint32_t Rows>
struct PairTrade {
  float mx[2][Rows];  // maxima over the groups' halves of the keys
  float ref[Rows];    // the reference of the tile before
};
constexpr uint32_t kPairTrades = 2;

// The trade of tile g of a CTA's tiles; a pair has every other one.
HALO_PAIR_FN uint32_t trade_of(uint32_t g) { return (g >> 1) % kPairTrades; }

// In: the maximum over this group's half of a row, and the reference of the tile before (from half 0). Out: the same for both.
template <uint32_t Rows, typename Sync>
HALO_PAIR_FN void trade_maxima(PairTrade<Rows>& t, uint32_t half, uint32_t row, float& mx, float& ref, Sync&& sync) {
  t.mx[half][row] = mx;
  if (half == 0) t.ref[row] = ref;
  sync();
  mx = fmaxf(t.mx[0][row], t.mx[1][row]);
  if (half == 1) ref = t.ref[row];
}

}  // namespace halo_b200

#endif  // HALO_B200_SOFTMAX_PAIR_CUH_
