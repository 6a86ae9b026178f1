// px_recur.h -- which units of a level a lane of the recurrence's kernels has,
// what it reads of a row and which words of other tiles it waits for.
#pragma once

#include <hip/hip_runtime.h>

namespace px {

constexpr int kSlab = 128;  // units of a workgroup: two a lane

// Rows are read without a branch: lanes past the row's end read something of
// it. FORM kEven: a level's units are even in number; kOdd: the last lane reads
// the pair before its single unit, and takes the second; kOne: a level of one
// unit, read alone.
enum { kEven, kOdd, kOne };
struct Lane {
  unsigned col, at;     // the first unit; where its pair is read
  unsigned word, next;  // whose words are waited for
  int n;                // of the two, how many are there
};
// Words are of the lane's own slab, for units that are not there as well: a
// slab's tiles are taken in order, but nothing says that another slab's have
// been taken at all, and a wait for one of them need not end.
template <int FORM>
__host__ __device__ __forceinline__ Lane lane_of(unsigned first, int lane, int units) {
  Lane l;
  l.col = first + lane * 2;
  l.n = units - static_cast<int>(l.col);
  l.word = l.n > 0 ? l.col : first, l.next = l.n > 1 ? l.col + 1 : l.word;
  l.at = FORM == kOdd && l.n == 1 ? l.col - 1 : l.n > 0 ? l.col : 0;
  return l;
}

}  // namespace px
