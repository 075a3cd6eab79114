/*
 * norm_ring.h -- where the layer norm gradient's ring of rows (layer_norm.cu)
 * keeps each thread's elements in shared memory, and which rows' packs may reach
 * outside their tensor; also compiled for the host by the tests.
 */
#ifndef HEXIR_B200_NORM_RING_H
#define HEXIR_B200_NORM_RING_H

#include <stdint.h>

#ifdef __CUDACC__
#define HEXIR_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define HEXIR_HOST_DEVICE inline
#endif

namespace hexir {

// A pack is 16 bytes: PER of a thread's elements.  `pack` counts a thread's
// packs over the ring (rows, tensors and a row's packs).
//
// Packs lie one per thread, PER elements each; with SINGLES (rows that are
// copied an element at a time) a warp's elements lie next to each other, so that
// its accesses fall into different banks.  In either, every place belongs to one
// thread alone, and that thread zeroes, fills and reads it: this is why the ring
// needs no barrier.  A place of one kind taken as the other's is another
// thread's.
template <uint32_t PER, uint32_t THREADS, bool SINGLES>
struct NormRing {
  // The element's place, in elements.
  static HEXIR_HOST_DEVICE uint32_t at(uint32_t pack, uint32_t element,
                                       uint32_t thread) {
    return SINGLES ? (pack * PER + element) * THREADS + thread
                   : (pack * THREADS + thread) * PER + element;
  }
};

// Whether a pack of row `row` of `rows` may hold elements outside the tensor's
// memory, for rows of `cols` elements that start anywhere and are at least that
// far apart.  A pack reaches PER - 1 elements beyond its row at most.  Of rows as
// long as that, the next one holds them; of shorter ones it takes up to PER
// rows.
template <uint32_t PER>
HEXIR_HOST_DEVICE bool norm_row_at_edge(uint64_t row, uint64_t rows, uint32_t cols) {
  const uint32_t near = cols >= PER ? 1u : PER;
  return row < near || row + near >= rows;
}

}  // namespace hexir

#endif /* HEXIR_B200_NORM_RING_H */
