// Packed prompts: fp32 keys and values in rows, no cache.
#include "attend_batch_prompt.h"

namespace accel_hip {
namespace {

template <int DP, int kLoad>
__global__ __launch_bounds__(kBatchThreads, DP > 128 || kLoad < 16 ? 1 : 2) void BatchPromptKernel(BatchLaunch args) {
  __shared__ PromptTiles<DP, false> tiles;
  __shared__ BatchScan<kBatchThreads> scan;
  PromptGroup<DP, false, kLoad, false>(args.a, args.prompt, static_cast<int32_t>(blockIdx.x), tiles, scan);
}

template <int DP>
void LaunchOf(const BatchLaunch& args, bool vec, hipStream_t stream) {
  const dim3 grid(args.prompt_groups), block(kBatchThreads);
  if (vec) hipLaunchKernelGGL((BatchPromptKernel<DP, 16>), grid, block, 0, stream, args);
  else hipLaunchKernelGGL((BatchPromptKernel<DP, 4>), grid, block, 0, stream, args);
  Check(hipGetLastError(), "BatchPromptKernel launch");
}

}  // namespace

void LaunchBatchPrompt(const BatchLaunch& args, bool vec, hipStream_t stream) {
  if (args.a.dim <= 64) LaunchOf<64>(args, vec, stream);
  else if (args.a.dim <= 96) LaunchOf<96>(args, vec, stream);
  else if (args.a.dim <= 128) LaunchOf<128>(args, vec, stream);
  else LaunchOf<256>(args, vec, stream);
}

}  // namespace accel_hip
