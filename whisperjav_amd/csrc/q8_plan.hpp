// q8_plan.hpp -- plain arithmetic of the 8-bit operators, the same on the host and in the kernels: which rows a sequence owns.
#pragma once

#include <stdint.h>

namespace wj {

// What a sequence of a call owns.  first .. first + n - 1: its rows of the row arrays; pos0: position of the first of them
struct Span { int slot, first, n, len, pos0; };

// Whatever the arrays hold, the rows lie inside 0 .. rows - 1 and no position passes 32 bits: a sequence that starts before row 0 or ends before
// it starts owns no rows, a negative length is none (its rows lie before position 0).
constexpr Span span_from(int slot, int first, int last, int len, int slots, int rows) {
  const bool there = first >= 0 && first < rows && last > first;
  const int n = there ? (last < rows ? last : rows) - first : 0, positions = len > 0 ? len : 0;
  return Span{slot >= 0 && slot < slots ? slot : -1, there ? first : rows, n, positions, positions - n};
}

}  // namespace wj
