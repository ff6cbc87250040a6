// Batches whose requests all have few new rows.
#include "attend_batch_step.h"

namespace accel_hip {
namespace {

template <int DP, bool kHalf, int kLoad, bool kPaged>
__global__ __launch_bounds__(kBatchThreads, DP <= 128 && kHalf && kLoad == 16 ? 2 : 1) void BatchStepKernel(BatchLaunch args) {
  __shared__ BatchParts<DP> parts;
  __shared__ BatchScan<kBatchThreads> scan;
  StepGroup<DP, kHalf, kLoad, kPaged>(args.a, args.step, static_cast<int32_t>(blockIdx.x), parts, scan);
}

template <int DP>
void LaunchOf(const BatchLaunch& args, bool vec, hipStream_t stream) {
#define ACCEL_STEP(H, L, P) \
  hipLaunchKernelGGL((BatchStepKernel<DP, H, L, P>), dim3(args.step_groups), dim3(kBatchThreads), 0, stream, args)
  if (args.a.f16) {
    if (vec) ACCEL_STEP(true, 16, true);
    else ACCEL_STEP(true, 2, true);
  } else if (args.a.paged) {
    if (vec) ACCEL_STEP(false, 16, true);
    else ACCEL_STEP(false, 4, true);
  } else {
    if (vec) ACCEL_STEP(false, 16, false);
    else ACCEL_STEP(false, 4, false);
  }
#undef ACCEL_STEP
  Check(hipGetLastError(), "BatchStepKernel launch");
}

}  // namespace

void LaunchBatchStep(const BatchLaunch& args, bool vec, hipStream_t stream) {
  if (args.a.dim <= 64) LaunchOf<64>(args, vec, stream);
  else if (args.a.dim <= 128) LaunchOf<128>(args, vec, stream);
  else LaunchOf<256>(args, vec, stream);
}

}  // namespace accel_hip
