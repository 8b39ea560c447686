// si_kv4_split.hpp -- where the partial sums of an attention whose keys are split
// lie in the scratch.  Plain C++, for the kernels and the host alike.
//
// A slot is one (token, head, split): its output of D floats and its (maximum, sum).
// All outputs come first: D is a multiple of 64, so each begins on a multiple of
// 256 bytes, as its loads and stores of 16 bytes need, and the pairs behind them on
// one of 8.  (Behind the pairs an odd number of slots would put them off by 8.)
#pragma once
#include <stddef.h>

#ifdef __CUDACC__
#define SI_KV4_HD __host__ __device__
#else
#define SI_KV4_HD
#endif

namespace si {

// In floats from the scratch's begin.
SI_KV4_HD constexpr size_t kv4_part_out(size_t slot, int D) { return slot * (size_t)D; }
SI_KV4_HD constexpr size_t kv4_part_ml(size_t slots, size_t slot, int D) {
  return slots * (size_t)D + 2 * slot;
}
SI_KV4_HD constexpr size_t kv4_part_size(size_t slots, int D) { return slots * (size_t)(D + 2); }

}  // namespace si
