#include "attend_split.h"

#include <algorithm>

namespace accel_hip {

AttendSplit SplitRange(const AttendArgs& a, int64_t units, int64_t most) {
  const int64_t cus = Ctx().cu_count > 0 ? Ctx().cu_count : 256;
  const int64_t count = std::max<int64_t>(1, std::min<int64_t>(cus / units, most));
  const int64_t parts = int64_t(a.seq) * a.heads * count;
  const size_t ml_bytes = (static_cast<size_t>(parts) * 2 * sizeof(float) + 15) & ~size_t(15);
  const size_t bytes = ml_bytes + static_cast<size_t>(parts * PartialDims(a.dim)) * sizeof(float);
  AttendSplit split;
  if (count == 1) return split;
  split.held = std::unique_lock<std::mutex>(AttendPartsMutex());
  if (!ScratchReady(0, kTempAttend, bytes)) return split;
  try {
    split.partial.ml = static_cast<float*>(Temp(kTempAttend, bytes));
  } catch (const Error& e) {
    if (e.code != ACCEL_HIP_BAD_ALLOC) throw;
    return split;
  }
  split.partial.o = split.partial.ml + ml_bytes / sizeof(float);
  split.count = static_cast<int32_t>(count);
  return split;
}

}  // namespace accel_hip
