// Batches over pages with requests of few new rows and of many. Both kinds of tiles are workgroups of one launch: those
// of many rows come first and keep the matrix cores busy, those of few fill the CUs' memory time and the end. Both
// run two workgroups a CU. 30 single tokens beside chunks of 1071 and 1196 over 1000 .. 9000 tokens in f16 (32 heads on 8
// of 128): 328 - 347 us, with the join; in two launches one behind the other 477, when one took 374. Bound: the chunks' products (195 us at a large product's
// rate) and their softmax.
#include "attend_batch_prompt.h"

namespace accel_hip {
namespace {

template <int DP, bool kHalf>
union MixedLds {
  PromptTiles<DP, kHalf> prompt;
  BatchParts<DP == 96 ? 128 : DP> step;
};

template <int DP, bool kHalf, int kLoad>
__global__ __launch_bounds__(kBatchThreads, DP > 128 || kLoad < 16 ? 1 : 2) void BatchMixedKernel(BatchLaunch args) {
  __shared__ MixedLds<DP, kHalf> lds;
  __shared__ BatchScan<kBatchThreads> scan;
  if (blockIdx.x < args.prompt_groups)
    PromptGroup<DP, kHalf, kLoad, true>(args.a, args.prompt, static_cast<int32_t>(blockIdx.x), lds.prompt, scan);
  else
    StepGroup<DP == 96 ? 128 : DP, kHalf, kLoad, true>(args.a, args.step, static_cast<int32_t>(blockIdx.x - args.prompt_groups),
                                                       lds.step, scan);
}

template <int DP>
void LaunchOf(const BatchLaunch& args, bool vec, hipStream_t stream) {
  const dim3 grid(args.prompt_groups + args.step_groups), block(kBatchThreads);
#define ACCEL_MIXED(H, L) hipLaunchKernelGGL((BatchMixedKernel<DP, H, L>), grid, block, 0, stream, args)
  if (args.a.f16) {
    if (vec) ACCEL_MIXED(true, 16);
    else ACCEL_MIXED(true, 2);
  } else {
    if (vec) ACCEL_MIXED(false, 16);
    else ACCEL_MIXED(false, 4);
  }
#undef ACCEL_MIXED
  Check(hipGetLastError(), "BatchMixedKernel launch");
}

}  // namespace

void LaunchBatchMixed(const BatchLaunch& args, bool vec, hipStream_t stream) {
  if (args.a.dim <= 64) LaunchOf<64>(args, vec, stream);
  else if (args.a.dim <= 96) LaunchOf<96>(args, vec, stream);
  else if (args.a.dim <= 128) LaunchOf<128>(args, vec, stream);
  else LaunchOf<256>(args, vec, stream);
}

}  // namespace accel_hip
