// What the launches of the norms' kernels share: the variant of a row's width and the
// partial rows of a backward.
#pragma once

#include <algorithm>
#include <type_traits>

#include "capi_common.h"

namespace mtf {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Calls f with the kernels' template arguments for a row of H elements: the
// fewest threads and registers that hold it (vec: rows of whole aligned 16-byte
// vectors).
template <class T, class F>
int norm_pick(int64_t H, bool vec, F f) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vec) {
    if (H <= 64 * 2 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 2>(),
                                  std::integral_constant<int, 64>());
    if (H <= 256 * 1 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 1>(),
                                   std::integral_constant<int, 256>());
    if (H <= 256 * 2 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 2>(),
                                   std::integral_constant<int, 256>());
    if (H <= 256 * 4 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 4>(),
                                   std::integral_constant<int, 256>());
    if (H <= 1024 * 4 * V) return f(std::integral_constant<int, V>(), std::integral_constant<int, 4>(),
                                    std::integral_constant<int, 1024>());
  }
  if (H <= 256 * 8) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 8>(),
                             std::integral_constant<int, 256>());
  if (H <= 1024 * 8) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 8>(),
                              std::integral_constant<int, 1024>());
  return f(std::integral_constant<int, 1>(), std::integral_constant<int, 32>(),
           std::integral_constant<int, 1024>());
}

constexpr int64_t kNormMaxH = 1024 * 32;
// Workgroups of the backward, each walking its rows and summing their weight
// gradients: two per CU.  Its 198 to 232 registers (norm before the block and
// gate) let no more reside: 147 us for 16384 x 3584, with 768 182, with 1024 157;
// the plain form, 65536 x 4096: 382, 387, 453 us.
constexpr int64_t kNormGroups = 512;

// Rows at a time of the backward, and so partial rows of the weight gradients, at
// most: kNormGroups workgroups, of four rows up to the width that a wave holds
// (norm_pick, bf16) and of one above it.
inline int64_t norm_parts(int64_t T, int64_t H) {
  return H <= 64 * 2 * 8 ? std::max<int64_t>(4, std::min<int64_t>(cdiv(T, 4), kNormGroups) * 4)
                         : std::min<int64_t>(T, kNormGroups);
}

}  // namespace mtf
