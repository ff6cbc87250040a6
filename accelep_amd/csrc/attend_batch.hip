// Attention of a batch of requests, over the pages of a cache or over packed prompts: which kernels a call takes,
// into how many key ranges, and the join of the ranges.
#include "attend_batch.h"

namespace accel_hip {
namespace {

constexpr int kJoinRows = 4;  // of a workgroup and round
constexpr int kJoinEach = 4;  // ranges in flight at once

// A workgroup's threads are (row, key range, 16-byte piece). Its items are 4 rows of a divided tile and key head each,
// taken in turn: how many tiles are divided is known on the device alone, mostly few of those that there is room for.
__global__ __launch_bounds__(kBatchThreads) void BatchJoinKernel(BatchLaunch args, bool vec) {
  __shared__ __align__(16) f4 part_o[kBatchThreads];
  __shared__ float part_m[kBatchThreads];
  __shared__ float part_l[kBatchThreads];
  const BatchAttendArgs& a = args.a;
  const int32_t prompt_blocks = args.prompt.ranges > 0 ? args.prompt.tiles[0] * a.kv_heads : 0;
  const int32_t step_blocks = args.step.ranges > 0 ? args.step.tiles[0] * a.kv_heads : 0;
  const int32_t prompt_items = prompt_blocks * (kPromptTileRows / kJoinRows);
  const int32_t step_items = step_blocks * (kStepTileRows / kJoinRows);
  const int32_t group = a.heads / a.kv_heads;
  const int dims = PartialDims(a.dim);
  const int pieces = dims / 4;
  for (int32_t item = static_cast<int32_t>(blockIdx.x); item < prompt_items + step_items;
       item += static_cast<int32_t>(gridDim.x)) {
    const bool prompt = item < prompt_items;
    const BatchSplit& b = prompt ? args.prompt : args.step;
    const int32_t tile_rows = prompt ? kPromptTileRows : kStepTileRows;
    const int32_t local_item = prompt ? item : item - prompt_items;
    const int32_t blocks = prompt ? prompt_blocks : step_blocks;
    const int32_t row_group = local_item / blocks;  // all tiles' first rows first: many tiles have no others
    const int32_t block = local_item - row_group * blocks;
    const int32_t which = Quotient(block, a.by_kv_heads);
    const int32_t kv = block - which * a.kv_heads;
    const int32_t* tile = b.tiles + static_cast<int64_t>(kTileInts) * (1 + which);
    const int32_t first = tile[0], splits = tile[1], start = tile[2], r0 = tile[3], rows = tile[4];
    const int32_t base_row = kJoinRows * row_group;
    if (splits == 1 || base_row >= rows) continue;  // uniform
    const int lanes = min(splits, kBatchThreads / (kJoinRows * pieces));
    const int per_row = pieces * lanes;
    const int local = static_cast<int>(threadIdx.x) / per_row;
    const int rest = static_cast<int>(threadIdx.x) - local * per_row;
    const int of = rest / pieces;
    const int piece = rest - of * pieces;
    const int32_t rl = base_row + local;
    const bool active = local < kJoinRows && rl < rows;
    const int64_t at0 = (static_cast<int64_t>(kv) * b.items + first) * tile_rows + rl;  // the next range's: tile_rows on
    const auto ml_of = [&](int c) {
      return *reinterpret_cast<const float2*>(b.partial.ml + 2 * (at0 + static_cast<int64_t>(c) * tile_rows));
    };
    const auto o_of = [&](int c) {
      return *reinterpret_cast<const f4*>(b.partial.o + (at0 + static_cast<int64_t>(c) * tile_rows) * dims + 4 * piece);
    };
    float m = -INFINITY, l = 0.f, low = 0.f;
    f4 sum = f4{0.f, 0.f, 0.f, 0.f};
    if (active) {
      for (int c0 = of; c0 < splits; c0 += lanes * kJoinEach) {
        float2 y[kJoinEach];
        f4 x[kJoinEach];
#pragma unroll
        for (int i = 0; i < kJoinEach; ++i) {
          const int c = min(c0 + i * lanes, splits - 1);
          y[i] = ml_of(c);
          x[i] = o_of(c);
        }
        float big = m;
#pragma unroll
        for (int i = 0; i < kJoinEach; ++i)
          if (c0 + i * lanes < splits) big = fmaxf(big, y[i].x);
        const float base = big == -INFINITY ? 0.f : big;
        const float corr = __builtin_amdgcn_exp2f(m - base);
        l *= corr;
        sum *= corr;
#pragma unroll
        for (int i = 0; i < kJoinEach; ++i) {
          if (c0 + i * lanes >= splits) break;
          const float wt = __builtin_amdgcn_exp2f(y[i].x - base);
          low = fminf(low, y[i].y);
          l += wt * y[i].y;
          sum += wt * x[i];
        }
        m = big;
      }
      part_m[threadIdx.x] = m;
      part_l[threadIdx.x] = low < 0.f ? -1.f : l;
      part_o[threadIdx.x] = sum;
    }
    __syncthreads();
    if (active && of == 0) {
      const int at = threadIdx.x;
      float big = -INFINITY;
      for (int i = 0; i < lanes; ++i) big = fmaxf(big, part_m[at + i * pieces]);
      const float base = big == -INFINITY ? 0.f : big;
      float total = 0.f;
      low = 0.f;
      sum = f4{0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < lanes; ++i) {
        const float wt = __builtin_amdgcn_exp2f(part_m[at + i * pieces] - base);
        low = fminf(low, part_l[at + i * pieces]);
        total += wt * part_l[at + i * pieces];
        sum += wt * part_o[at + i * pieces];
      }
      f4 far = f4{0.f, 0.f, 0.f, 0.f};
      if (low < 0.f) {  // some parts are held times 2^-64: their sum is one of its own
        total = 0.f;
        sum = far;
        for (int c = 0; c < splits; ++c) {
          const float2 y = ml_of(c);
          const float wt = __builtin_amdgcn_exp2f(y.x - base);
          const f4 x = wt * o_of(c);
          total += wt * fabsf(y.y);
          if (y.y < 0.f) far += x;
          else sum += x;
        }
      }
      float* dst = a.out + BatchOutRow(a, start, r0 + rl, group, kv) * a.dim + 4 * piece;
      f4 y = f4{__fdiv_rn(sum[0], total), __fdiv_rn(sum[1], total), __fdiv_rn(sum[2], total), __fdiv_rn(sum[3], total)};
      if (low < 0.f)
        y += f4{__fdiv_rn(far[0], total), __fdiv_rn(far[1], total), __fdiv_rn(far[2], total), __fdiv_rn(far[3], total)} * kFarUp;
      if (vec) {
        *reinterpret_cast<f4*>(dst) = y;
      } else {
        for (int e = 0; e < 4; ++e)
          if (4 * piece + e < a.dim) dst[e] = y[e];
      }
    }
    __syncthreads();
  }
}

// Workgroups of the join: enough to fill the CUs' threads. 24 short prompts with 2, 4, 8 and 16 a CU: 23.3, 21.0, 19.7 and
// 20.0 us, chunks in a window 87.0, 84.8, 84.8 and 84.7; with one for each tile that there is room for 20.2 and 87.5.
constexpr int64_t kJoinGroupsPerCu = 8;

// One share of a call: the tiles of requests with few rows, or of those with many.
struct Share {
  int32_t tile_rows;
  int64_t tiles;      // of a key head, at most
  int64_t ranges;     // a key head's key ranges, about; 0: no range is divided
  int64_t min_steps;  // of a range
  int64_t items;      // a key head's partial items, at most
  int64_t divided;    // a key head's divided tiles, at most
  size_t ml_bytes, o_bytes, tile_bytes;
  size_t Bytes() const { return ml_bytes + o_bytes + tile_bytes; }
};

size_t Round16(size_t bytes) { return (bytes + 15) & ~size_t(15); }

Share ShareOf(const BatchAttendArgs& a, int32_t tile_rows, int32_t keys, int64_t tiles, int64_t groups, int64_t min_steps) {
  Share s{tile_rows, tiles, 0, min_steps, 0, 0, 0, 0, 0};
  const int64_t most_keys = std::min<int64_t>(a.paged ? (int64_t(a.width) << a.page_shift) + a.rows : a.rows,
                                              int64_t(a.window) + tile_rows + 2 * keys);
  const int64_t most_steps = (most_keys + keys - 1) / keys;
  if (most_steps <= min_steps || groups < 2 * a.kv_heads) return s;  // one range would be all there is
  s.ranges = groups / a.kv_heads;
  s.items = std::min<int64_t>(4 * s.ranges, tiles * ((most_steps + min_steps - 1) / min_steps));
  s.divided = std::min<int64_t>(2 * s.ranges, tiles);
  const size_t parts = static_cast<size_t>(s.items) * a.kv_heads * tile_rows;
  s.ml_bytes = Round16(parts * 2 * sizeof(float));
  s.o_bytes = Round16(parts * PartialDims(a.dim) * sizeof(float));
  s.tile_bytes = Round16(static_cast<size_t>(s.divided + 1) * kTileInts * sizeof(int32_t));
  return s;
}

BatchSplit SplitOf(const Share& s, int32_t few, char* scratch) {
  BatchSplit b{};
  b.few = few;
  b.min_steps = static_cast<int32_t>(s.min_steps);
  if (s.ranges == 0 || scratch == nullptr) return b;
  b.ranges = static_cast<int32_t>(s.ranges);
  b.items = static_cast<int32_t>(s.items);
  b.partial.ml = reinterpret_cast<float*>(scratch);
  b.partial.o = reinterpret_cast<float*>(scratch + s.ml_bytes);
  b.tiles = reinterpret_cast<int32_t*>(scratch + s.ml_bytes + s.o_bytes);
  return b;
}

constexpr const char* kTooLarge = "Attention is too large";

void LaunchJoin(const BatchLaunch& args, const Share& step, const Share& prompt, int64_t cus, hipStream_t stream) {
  const BatchAttendArgs& a = args.a;
  const int64_t items = (args.step.ranges > 0 ? step.divided * kStepTileRows : 0) +
                        (args.prompt.ranges > 0 ? prompt.divided * kPromptTileRows : 0);
  if (items == 0) return;
  const bool vec = a.dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  const dim3 grid(static_cast<uint32_t>(std::min(items / kJoinRows * a.kv_heads, kJoinGroupsPerCu * cus)));
  hipLaunchKernelGGL(BatchJoinKernel, grid, dim3(kBatchThreads), 0, stream, args, vec);
  Check(hipGetLastError(), "BatchJoinKernel launch");
}

}  // namespace

void LaunchAttendBatch(const BatchAttendArgs& a, hipStream_t stream) {
  const int64_t cus = Ctx().cu_count > 0 ? Ctx().cu_count : 256;
  const int64_t group = a.heads / a.kv_heads;
  const int64_t all_rows = int64_t(a.rows) * group;
  const int32_t align = a.f16 ? 8 : 4;
  const bool vec = a.dim % align == 0 && a.kv_stride % align == 0 && reinterpret_cast<uintptr_t>(a.k) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.v) % 16 == 0;
  // Requests of up to 16 rows of a key head are the step tiles', larger ones the prompt tiles'. Where no request
  // has more, the first have all (also one that is longer than `longest` says); packed prompts, whose short ones
  // have few keys too, are the second's. 32 requests over 4000 tokens of 8 heads of 128, in step tiles and in prompt
  // tiles: 4 or 16 rows 107 - 111 and 178 us in f16, 191 and 291 in fp32; 32 rows 143 and 150, 258 and 265; 64 rows
  // 222 and 159, 454 and 283. At 32 rows the first gain 3 to 5 %, which is not worth a third rule. 24 packed prompts of 5
  // .. 300 tokens: 28 and 21. Single tokens whose `longest` is 0 have the prompt tiles' workgroups in front, which find no
  // tile, and the mixed kernel's registers: 4 requests take 11.9 us for 12.2 with 1, 32 133.2 for 130.9, 125 107.7 for 104.3.
  constexpr int32_t kAll = 0x7fffffff;
  const bool steps_only = a.longest * group <= kStepTileRows;
  const bool steps = steps_only || (a.paged && group <= kStepTileRows);
  const int32_t few = steps_only ? kAll : steps ? kStepTileRows : 0;
  Share step{}, prompt{};
  if (steps) {
    const int64_t tiles = std::min<int64_t>(a.requests, a.rows) + (steps_only ? all_rows / kStepTileRows : 0);
    // A step tile's range costs little to begin and join. With 2, 3 and 4 ranges a CU: 32 requests of up to 16384 tokens
    // 142, 130 and 135 us, 125 of up to 2048 102, 97 and 97. At least 8 steps each, two a wave: 4 requests of a small
    // model 12.1 us, with 4 11.8 and with 16 14.0.
    step = ShareOf(a, kStepTileRows, StepKeys(a.f16), tiles, 3 * cus, 8);
  }
  if (!steps_only) {
    const int64_t tiles = all_rows / kPromptTileRows + std::min<int64_t>(a.requests, all_rows / (few + 1));
    // A prompt tile's part is 64 KB to write and to read again, so it is cut less: as if a CU had one. With 1, 1.5, 2 and
    // 3 ranges a CU: chunks in a window 88, 110, 98 and 115 us; a mixed batch 339, 343, 365 and 411; heads of 80 126, 133,
    // 145 and 140; long prompts 717, 718, 719 and 727. At least 4 steps each: 24 short prompts 20.2 us, with 8 22.8.
    prompt = ShareOf(a, kPromptTileRows, PromptKeys(a.f16), tiles, cus, 4);
  }
  // Where there is no memory for the parts the ranges stay whole.
  std::unique_lock<std::mutex> held;
  char* scratch = nullptr;
  const size_t bytes = step.Bytes() + prompt.Bytes();
  if (bytes > 0) {
    held = std::unique_lock<std::mutex>(AttendPartsMutex());
    if (ScratchReady(0, kTempAttend, bytes)) {
      try {
        scratch = static_cast<char*>(Temp(kTempAttend, bytes));
      } catch (const Error& e) {
        if (e.code != ACCEL_HIP_BAD_ALLOC) throw;
      }
    }
  }
  BatchLaunch args{a, SplitOf(step, few, scratch), SplitOf(prompt, few, scratch == nullptr ? nullptr : scratch + step.Bytes()), 0, 0};
  // A key head's items are 2 * ranges and the tiles at most.
  args.step_groups = steps ? GridOf((step.tiles + 2 * args.step.ranges) * a.kv_heads, kBatchThreads, kTooLarge) : 0;
  args.prompt_groups = steps_only ? 0 : GridOf((prompt.tiles + 2 * args.prompt.ranges) * a.kv_heads, kBatchThreads, kTooLarge);
  GridOf(int64_t(args.step_groups) + args.prompt_groups, kBatchThreads, kTooLarge);
  if (steps_only) LaunchBatchStep(args, vec, stream);
  else if (a.paged) LaunchBatchMixed(args, vec, stream);
  else LaunchBatchPrompt(args, vec, stream);
  LaunchJoin(args, step, prompt, cus, stream);
}

}  // namespace accel_hip
