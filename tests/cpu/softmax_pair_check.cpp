// The exchange between the two softmax groups of a pair, in the worst orders that its barrier alone allows (no other wait
// orders anything once one has run out): both groups must come to the same maximum and the same reference, since the
// decision to rescale, and with it the number of barriers that each passes, follows from these.
//
// Prints the number of tiles and of disagreements.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <limits>

#include "softmax_pair.cuh"

using namespace halo_b200;

namespace {
constexpr uint32_t kR = 4;
struct Stop {};
uint32_t Bits(float v) {
  uint32_t u;
  std::memcpy(&u, &v, 4);
  return u;
}
float Pick() {
  const int k = std::rand() % 8;
  return k == 0 ? -std::numeric_limits<float>::infinity() : k == 1 ? std::numeric_limits<float>::quiet_NaN() : static_cast<float>(std::rand() % 2000 - 1000);
}
}  // namespace

int main() {
  std::srand(7);
  PairTrade<kR> trades[kPairTrades];
  for (auto& t : trades)
    for (uint32_t r = 0; r < kR; ++r) t.mx[0][r] = t.mx[1][r] = t.ref[r] = Pick();
  unsigned tiles = 0, bad = 0;
  for (uint32_t pair = 0; pair < 2; ++pair)
    for (uint32_t i = 0; i < 20000; ++i) {
      // Tile g of this pair. What either group finds where the other pair publishes its references is anything.
      const uint32_t g = 2 * i + pair, row = static_cast<uint32_t>(std::rand()) % kR, first = static_cast<uint32_t>(std::rand()) % 2;
      float mx[2] = {Pick(), Pick()}, ref[2] = {Pick(), Pick()};
      // Group `first` arrives at the barrier first; the other one passes it at once, finishes the tile, goes on to the
      // pair's next tile and writes there whatever it finds before the next barrier stops it. Only then `first` goes on.
      trade_maxima(trades[trade_of(g)], first, row, mx[first], ref[first], [&] {
        const uint32_t o = 1 - first;
        trade_maxima(trades[trade_of(g)], o, row, mx[o], ref[o], [] {});
        float m = Pick(), r = Pick();
        try {
          trade_maxima(trades[trade_of(g + 2)], o, row, m, r, [] { throw Stop{}; });
        } catch (const Stop&) {
        }
      });
      ++tiles;
      bad += Bits(mx[0]) != Bits(mx[1]) || Bits(ref[0]) != Bits(ref[1]);
    }
  std::printf("%u %u\n", tiles, bad);
  return 0;
}
