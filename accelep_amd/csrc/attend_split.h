// The division of a key range over workgroups: the parts' memory and how many parts there are.
#pragma once

#include <mutex>

#include "common.h"

namespace accel_hip {

// Partial results of key ranges: of each (row, range) the reference m and the sum l, and the weighted sum o
// of PartialDims(dim) floats, 16-byte aligned (attend_common.h says how l and o are held).
constexpr int32_t PartialDims(int32_t dim) { return (dim + 3) & ~3; }
struct AttendPartial {
  float* ml;  // [rows][splits][2]
  float* o;   // [rows][splits][PartialDims]
};

// Into how many key ranges the rows of `units` workgroups are cut: up to one workgroup per CU, at most
// `most` ranges. Where the partial sums have no room (no memory is left, or a capture runs and the
// buffer is too small) the range stays whole. Their buffer serves these calls alone, and is held until both
// launches are queued: calls from several threads, and replays of graphs, take turns.
struct AttendSplit {
  int32_t count = 1;
  AttendPartial partial{nullptr, nullptr};
  std::unique_lock<std::mutex> held;
};
AttendSplit SplitRange(const AttendArgs& a, int64_t units, int64_t most);

}  // namespace accel_hip
