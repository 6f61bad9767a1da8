// csrc/overlap.h against sets of bytes: random small views, and views of the layouts that calls have.
// Prints the number of pairs, of disagreements on pairs, of disagreements on single views, and of pairs that overlap.
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#include "overlap.h"

using halo_b200::View;

namespace {
struct Plain {
  uint64_t base, run, n[3], s[3];
};
View Make(const Plain& p, uint64_t size) {
  View v(reinterpret_cast<const void*>(p.base), p.run * size);
  for (int i = 0; i < 3; ++i) v.Along(p.n[i], p.s[i], size);
  return v;
}
// How often each byte is written.
std::vector<int> Bytes(const Plain& p, uint64_t size) {
  std::vector<int> c(20000, 0);
  for (uint64_t x = 0; x < p.n[0]; ++x)
    for (uint64_t y = 0; y < p.n[1]; ++y)
      for (uint64_t z = 0; z < p.n[2]; ++z)
        for (uint64_t e = 0; e < p.run * size; ++e) ++c[p.base + (x * p.s[0] + y * p.s[1] + z * p.s[2]) * size + e];
  return c;
}
}  // namespace

int main() {
  std::mt19937 rng(11);
  auto pick = [&](uint64_t lo, uint64_t hi) { return lo + rng() % (hi - lo + 1); };
  unsigned pairs = 0, bad = 0, bad_self = 0, meet = 0;
  for (int round = 0; round < 30000; ++round) {
    const uint64_t size = pick(0, 1) ? 2 : 4;
    Plain p[2];
    const bool same = pick(0, 1);  // the same strides: two views of one buffer
    for (int k = 0; k < 2; ++k) {
      p[k].base = size * pick(0, 150), p[k].run = pick(0, 9) ? pick(1, 8) : 0;
      for (int i = 0; i < 3; ++i) {
        p[k].n[i] = pick(0, 20) ? pick(1, 5) : 0;
        p[k].s[i] = k && same ? p[0].s[i] : pick(0, 3) ? pick(1, i == 0 ? 150 : i == 1 ? 40 : 12) : pick(0, 1) * 8;
      }
    }
    const std::vector<int> a = Bytes(p[0], size), b = Bytes(p[1], size);
    bool both = false, twice = false;
    for (size_t i = 0; i < a.size(); ++i) both |= a[i] && b[i], twice |= a[i] > 1;
    const View v = Make(p[0], size), w = Make(p[1], size);
    ++pairs;
    meet += both;
    bad += halo_b200::Overlap(v, w) != both || halo_b200::Overlap(w, v) != both;
    bad_self += halo_b200::OverlapsItself(v) != twice;
  }
  std::printf("%u %u %u %u\n", pairs, bad, bad_self, meet);
  return 0;
}
