// Which of 32 keys a row of attention sees, a bit each (paged_tile.h). Plain C++; sizes and positions are from 0 to 2^31 - 1, and nothing here wraps:
// the assertions below would not compile.
#pragma once
#include <cstdint>

namespace hexmi {

// the first n bits of 32, none for n < 0
__attribute__((always_inline)) constexpr uint32_t first_bits(int n) {
  const int m = n < 0 ? 0 : n < 32 ? n : 32;
  return (uint32_t)(0xffffffffull >> (32 - m));
}
// Of the keys first .. first + 31 those below `keys` and, where a window hides any, from keys - window on; and whatever hides the others, `sinks`
// of the 32 that begin with the first. window: from 1, 2^31 - 1 for none.
__attribute__((always_inline)) constexpr uint32_t seen_of_32(int keys, int first, int window, int sinks) {
  const int from = keys - window;                                  // from 0 on: a row with few keys may be far below `first`
  return first_bits(keys - first) & (~first_bits((from > 0 ? from : 0) - first) | first_bits(sinks));
}
static_assert(seen_of_32(0, 64, 0x7fffffff, -64) == 0 && seen_of_32(0, 0x7fffffff, 0x7fffffff, -0x7fffffff) == 0);
static_assert(seen_of_32(0x7fffffff, 0, 0x7fffffff, 0) == ~0u && seen_of_32(40, 32, 5, -32) == 0xf8 && seen_of_32(40, 0, 5, 3) == 7);

}  // namespace hexmi
