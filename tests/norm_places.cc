// The rules of kernels/norm_ring.h: every place of the gradient's ring is one
// thread's alone, and together they are the ring; a row whose 16-byte blocks
// reach outside its tensor is an edge.
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

// Rows with a block outside the tensor's memory that no edge guards, and, of rows
// of a pack or more, edges beside the first and the last row.
template <uint32_t PER>
int outside(int *needless) {
  int bad = 0;
  for (uint64_t offset = 0; offset < PER; ++offset)
    for (uint64_t cols = 1; cols < 3 * PER; ++cols)
      for (uint64_t ld = cols; ld < cols + PER + 2; ++ld)
        for (uint64_t rows = 1; rows < 3 * PER; ++rows) {
          const uint64_t first = 8 * PER + offset, last = first + (rows - 1) * ld + cols;
          for (uint64_t row = 0; row < rows; ++row) {
            const uint64_t begin = first + row * ld, end = begin + cols;
            const uint64_t low = begin / PER * PER, high = (end + PER - 1) / PER * PER;
            const bool edge = hexir::norm_row_at_edge<PER>(row, rows, cols);
            bad += !edge && (low < first || high > last);
            *needless += cols >= PER && edge && row != 0 && row != rows - 1;
          }
        }
  return bad;
}

int main() {
  int bad = 0;
  for (uint32_t packs : {1u, 2u, 4u, 12u, 24u}) {
    bad += shared_or_missing<4, 256, true>(packs) + shared_or_missing<4, 320, true>(packs) +
           shared_or_missing<4, 512, true>(packs) + shared_or_missing<2, 192, true>(packs) +
           shared_or_missing<2, 512, true>(packs) + shared_or_missing<4, 512, false>(packs) +
           shared_or_missing<8, 256, false>(packs) + shared_or_missing<8, 1024, false>(packs);
  }
  int needless = 0;
  const int reach = outside<8>(&needless) + outside<4>(&needless);
  std::printf("%d %d %d %d %d\n", bad, mixed<4, 512>(2), mixed<2, 192>(4), reach,
              needless);
  return 0;
}
