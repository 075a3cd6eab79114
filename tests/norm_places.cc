// The places of the layer norm gradient's ring (kernels/norm_ring.h), for every
// thread: each is one thread's alone, and together they are the ring.
#include <cstdint>
#include <cstdio>
#include <vector>

#include "kernels/norm_ring.h"

template <uint32_t PER, uint32_t THREADS, bool SINGLES>
int shared_or_missing(uint32_t packs) {
  std::vector<int> owner(packs * THREADS * PER, -1);
  int bad = 0;
  for (uint32_t t = 0; t < THREADS; ++t)
    for (uint32_t p = 0; p < packs; ++p)
      for (uint32_t e = 0; e < PER; ++e) {
        const uint32_t at = hexir::NormRing<PER, THREADS, SINGLES>::at(p, e, t);
        if (at >= owner.size() || owner[at] != -1)
          ++bad;
        else
          owner[at] = static_cast<int>(t);
        // A pack's elements follow each other and start on 16 bytes.
        if (!SINGLES && at != hexir::NormRing<PER, THREADS, SINGLES>::at(p, 0, t) + e)
          ++bad;
        if (!SINGLES && e == 0 && at % PER)
          ++bad;
      }
  for (int o : owner)
    bad += o == -1;
  return bad;
}

// Elements whose thread differs between the two kinds: what one kind's pack
// writes is mostly other threads' in the other's.
template <uint32_t PER, uint32_t THREADS>
int mixed(uint32_t packs) {
  std::vector<uint32_t> owner(packs * THREADS * PER);
  for (uint32_t t = 0; t < THREADS; ++t)
    for (uint32_t p = 0; p < packs; ++p)
      for (uint32_t e = 0; e < PER; ++e)
        owner[hexir::NormRing<PER, THREADS, true>::at(p, e, t)] = t;
  int other = 0;
  for (uint32_t t = 0; t < THREADS; ++t)
    for (uint32_t p = 0; p < packs; ++p)
      for (uint32_t e = 0; e < PER; ++e)
        other += owner[hexir::NormRing<PER, THREADS, false>::at(p, e, t)] != t;
  return other;
}

int main() {
  int bad = 0;
  for (uint32_t packs : {1u, 2u, 4u, 12u, 24u}) {
    bad += shared_or_missing<4, 256, true>(packs) + shared_or_missing<4, 320, true>(packs) +
           shared_or_missing<4, 512, true>(packs) + shared_or_missing<2, 192, true>(packs) +
           shared_or_missing<2, 512, true>(packs) + shared_or_missing<4, 512, false>(packs) +
           shared_or_missing<8, 256, false>(packs) + shared_or_missing<8, 1024, false>(packs);
  }
  std::printf("%d %d %d\n", bad, mixed<4, 512>(2), mixed<2, 192>(4));
  return 0;
}
