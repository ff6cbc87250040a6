// New keys and values into the pages of a cache, each row into its slot, as fp32 or f16. Every value is read and written
// once. 8191 rows of 8 heads of 128 to f16: 100 MB, 16.4 us where they lie in the caches, 19.1 where they do not, a large
// copy's rate; 16 rows of 3 of 64 to fp32: 4.1 - 4.6 us, the launch.
#include <algorithm>

#include "device_common.h"

namespace accel_hip {
namespace {

constexpr int kThreads = 256;

typedef _Float16 h4 __attribute__((ext_vector_type(4)));

// kDims values of a row of one plane a thread and round.
template <bool kF16, int kDims>
__global__ __launch_bounds__(kThreads) void AppendPagedKernel(AppendPagedArgs a, uint32_t per_row, int64_t items) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  const float* src = a.src[blockIdx.y];
  void* dst = a.dst[blockIdx.y];
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; item < items; item += step) {
    const int64_t row = item / per_row;
    const uint32_t d = static_cast<uint32_t>(item - row * per_row) * kDims;
    const int32_t slot = a.slots[row];
    if (slot < 0 || slot >= a.slot_count) continue;
    const float* p = src + row * a.row_stride + d;
    const int64_t to = static_cast<int64_t>(slot) * a.width + d;
    if constexpr (kDims == 4) {
      const float4 x = *reinterpret_cast<const float4*>(p);
      if constexpr (kF16)
        *reinterpret_cast<h4*>(static_cast<_Float16*>(dst) + to) = h4{static_cast<_Float16>(x.x), static_cast<_Float16>(x.y),
                                                                      static_cast<_Float16>(x.z), static_cast<_Float16>(x.w)};
      else
        *reinterpret_cast<float4*>(static_cast<float*>(dst) + to) = x;
    } else {
      if constexpr (kF16) static_cast<_Float16*>(dst)[to] = static_cast<_Float16>(*p);
      else static_cast<float*>(dst)[to] = *p;
    }
  }
}

bool AlignedTo(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

template <bool kF16, int kDims>
void Launch(const AppendPagedArgs& a, hipStream_t stream) {
  const int64_t per_row = a.width / kDims;
  const int64_t items = per_row * a.rows;
  const int64_t groups = std::min<int64_t>((items + kThreads - 1) / kThreads, 1 << 20);
  hipLaunchKernelGGL((AppendPagedKernel<kF16, kDims>), dim3(static_cast<uint32_t>(groups), 2), dim3(kThreads), 0, stream, a,
                     static_cast<uint32_t>(per_row), items);
  Check(hipGetLastError(), "AppendPagedKernel launch");
}

}  // namespace

void LaunchAppendPaged(const AppendPagedArgs& a, hipStream_t stream) {
  const size_t to = a.f16 ? 8 : 16;
  const bool vec = a.width % 4 == 0 && a.row_stride % 4 == 0 && AlignedTo(a.src[0], 16) && AlignedTo(a.src[1], 16) &&
                   AlignedTo(a.dst[0], to) && AlignedTo(a.dst[1], to);
  if (a.f16) {
    if (vec) Launch<true, 4>(a, stream);
    else Launch<true, 1>(a, stream);
  } else {
    if (vec) Launch<false, 4>(a, stream);
    else Launch<false, 1>(a, stream);
  }
}

}  // namespace accel_hip
