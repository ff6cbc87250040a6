// What the attention kernels over a batch of requests share: which part of the batch a workgroup has.
//
// How long the requests are is known on the device alone, so every workgroup reads the lengths, counts the steps
// of all requests and finds its own part: no table of work is made ahead, and a captured launch follows
// the lengths. A tile is kTileRows rows of a request and key head, row = query * group + head of the group; a step
// is kStep keys. Ranges of keys have about (all steps) / target steps, so that a batch fills the CUs whatever
// its lengths, and each part of a tile's range is an item.
#pragma once

#include "attend_common.h"

namespace accel_hip {

// How the work is divided. ranges 0: no key range is.
struct BatchSplit {
  int32_t few;        // the step kernel has the requests of up to `few` rows, the prompt kernel those of more
  int32_t ranges;     // key ranges a key head that the tiles are cut to, about
  int32_t min_steps;  // of a range
  int32_t items;      // room for a key head's partial items: 4 * ranges at most (see FindWork)
  AttendPartial partial;  // [kv_heads][items][tile rows]
  int32_t* tiles;     // [tile][kTileInts]: the tiles whose ranges are divided, their count before them
};
constexpr int kTileInts = 8;  // first item, items, first row of the request in the batch, first row of the tile, its rows

__device__ __forceinline__ int32_t Quotient(int32_t x, const QuickDivisor& d) {
  return static_cast<int32_t>(static_cast<uint64_t>(static_cast<uint32_t>(x)) * d.mul >> d.shift);
}

// Sums over the lanes up to this one: shifts inside rows of 16, then the ends of the rows before.
__device__ __forceinline__ int32_t WaveSums(int32_t x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

struct BatchItem {
  int32_t request, start, seen, rows;  // rows: of the request and a key head
  int32_t r0;                          // the tile's first
  int32_t p_first, p_last;             // positions of the tile's rows
  int32_t low, high;                   // its keys; low is a multiple of a step
  int32_t begin, end;                  // steps of this item, the first at low
  int32_t split, splits, partial;      // of the tile's range; where splits > 1, the item's place
};

// The requests' part of FindWork: shape of request r as this kernel sees it.
template <int kTileRows, int kStep, bool kFew>
struct BatchShape {
  int32_t start = 0, seen = 0, rows = 0, tiles = 0, steps = 0;  // steps: of one tile's range, at most
  int64_t work = 0;  // of all tiles' ranges, half of tiles * steps at least
  bool descends = false;  // the next request begins before this one
  __device__ __forceinline__ BatchShape() {}
  __device__ __forceinline__ BatchShape(const BatchAttendArgs& a, const BatchSplit& b, int32_t group, int32_t r) {
    start = a.starts[r];
    const int32_t stop = a.starts[r + 1];
    descends = stop < start;
    seen = a.paged ? min(max(a.seen[r], 0), a.width << a.page_shift) : 0;
    start = min(max(start, 0), a.rows);
    const int32_t n = min(max(stop, start), a.rows) - start;
    rows = n * group;
    if (kFew ? rows > b.few : rows <= b.few) rows = 0;
    tiles = (rows + kTileRows - 1) / kTileRows;
    const int32_t end = seen + n;
    steps = (end + kStep - 1) / kStep;
    if (a.window < min(end, 1 << 30)) steps = min(steps, (a.window + Quotient(kTileRows + group - 2, a.group) + 2 * kStep - 2) / kStep);
    if (rows == 0) steps = 0;
    // The first tile's range ends at its own rows, and without a window those between grow evenly.
    const int32_t first = min(steps, (seen + min(n, Quotient(kTileRows + group - 1, a.group)) + kStep - 1) / kStep);
    work = (static_cast<int64_t>(tiles) * (a.window < end ? 2 * steps : first + steps) + 1) / 2;
  }
  // The first tiles, whose rows all end within `most` steps.
  __device__ __forceinline__ int32_t ShortTiles(int32_t group, int32_t most) const {
    const int64_t rows_below = min(max(int64_t(0), static_cast<int64_t>(most) * kStep - seen), int64_t(rows)) * group;
    return static_cast<int32_t>(min(rows_below / kTileRows, int64_t(tiles)));
  }
};

// What a wave passes on to the others.
template <int kThreads>
struct BatchScan {
  int64_t steps[kThreads / 64];
  int32_t sums[kThreads / 64][4];
  int32_t found[8];
};

// The item-th item of a key head's work; false: there are fewer, or it is empty. Uniform over the workgroup. lead: of
// the first key head, whose workgroups note the divided tiles.
// Items: a request's long tiles, those of more than size / 2 steps, are cut into `per` = ceil(steps / size) ranges each,
// size >= all work / ranges; they come first, all requests' short tiles behind them, each one item, so that what is begun
// last is short. A request's tiles * steps is at most twice its work, so all items are at most 2 * ranges + all tiles, and
// those of divided tiles, whose steps / size is above 1, at most twice their steps / size: 4 * ranges. Divided tiles:
// 2 * ranges. That holds while no row is of two requests, so starts that descend leave no item.
template <int kThreads, int kTileRows, int kStep, bool kFew>
__device__ __forceinline__ bool FindWork(const BatchAttendArgs& a, const BatchSplit& b, int32_t item, bool lead,
                                         BatchScan<kThreads>& shared, BatchItem* w) {
  using Shape = BatchShape<kTileRows, kStep, kFew>;
  constexpr int kWaves = kThreads / 64;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int32_t group = a.heads / a.kv_heads;
  const bool first_group = lead && item == 0;
  int64_t all = 0;
  Shape own;  // of the first kThreads requests, which are looked at once
  if (tid < a.requests) own = Shape(a, b, group, tid);
  constexpr int32_t kMostSteps = 0x3fffffff;
  int32_t size = kMostSteps;
  if (b.ranges > 0) {  // uniform
    all = own.work;
    bool descends = own.descends;
    for (int32_t r = tid + kThreads; r < a.requests; r += kThreads) {
      const Shape x(a, b, group, r);
      all += x.work;
      descends = descends || x.descends;
    }
    all = WaveButterfly(all, [](int64_t x, int64_t y) { return x + y; });
    descends = __any(descends);
    if (lane == 0) shared.steps[wave] = descends ? -1 : all;
    __syncthreads();
    all = 0;
    descends = false;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const int64_t x = shared.steps[i];
      descends = descends || x < 0;
      all += x;
    }
    if (descends) {  // uniform
      if (first_group && tid == 0) b.tiles[0] = 0;
      return false;
    }
    int64_t least = static_cast<int64_t>(static_cast<double>(all) / b.ranges);  // all < 2^53: within 1
    while (least * b.ranges < all) ++least;
    size = static_cast<int32_t>(min(int64_t(kMostSteps), max(int64_t(b.min_steps), least)));
  }
  int32_t before = 0, parts_before = 0, divided_before = 0;  // items, items of divided tiles, divided tiles
  bool here = false;
  // Long tiles, then short ones: in one look where the requests are few enough for one, otherwise in a second.
  const bool at_once = a.requests <= kThreads;
  for (int pass = 0; pass < 2 && !here; ++pass) {
    for (int32_t r0 = 0; r0 < a.requests; r0 += kThreads) {
      if (!at_once) own = r0 + tid < a.requests ? Shape(a, b, group, r0 + tid) : Shape();
      const int32_t per = own.steps <= size ? 1 : (own.steps + size - 1) / size;
      const int32_t short_tiles = kFew ? 0 : own.ShortTiles(group, size / 2);
      const int32_t long_tiles = own.tiles - short_tiles;
      const int32_t mine = pass == 0 ? long_tiles * per : 0, mine_short = at_once || pass == 1 ? short_tiles : 0;
      const int32_t items = WaveSums(mine), parts = WaveSums(per > 1 ? mine : 0), divided = WaveSums(per > 1 ? long_tiles : 0);
      const int32_t shorts = kFew ? 0 : WaveSums(mine_short);
      if (lane == 63) {
        shared.sums[wave][0] = items;
        shared.sums[wave][1] = parts;
        shared.sums[wave][2] = divided;
        shared.sums[wave][3] = shorts;
      }
      __syncthreads();
      int32_t from = before + items - mine, part = parts_before + parts, tile = divided_before + divided;
      int32_t from_short = shorts - mine_short, short_sum = 0;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        const int32_t x = shared.sums[v][0], y = shared.sums[v][1], z = shared.sums[v][2], t = shared.sums[v][3];
        if (v < wave) {
          from += x;
          part += y;
          tile += z;
          from_short += t;
        }
        before += x;
        parts_before += y;
        divided_before += z;
        short_sum += t;
      }
      from_short += before;  // behind all long ones
      before += short_sum;
      const bool in_long = item >= from && item - from < mine, in_short = item >= from_short && item - from_short < mine_short;
      if (in_long || in_short) {
        const int32_t found[8] = {r0 + tid, item - (in_long ? from : from_short), part - mine, tile - long_tiles, own.start,
                                  own.seen, own.rows, in_long ? per : -short_tiles};
#pragma unroll
        for (int i = 0; i < 8; ++i) shared.found[i] = found[i];
      }
      __syncthreads();
      here = item < before;
      if (here && !(first_group && pass == 0 && b.ranges > 0)) break;  // the first workgroup counts on
    }
    if (first_group && pass == 0 && b.ranges > 0 && tid == 0) b.tiles[0] = divided_before;
    if (kFew || at_once) break;
  }
  if (!here) return false;
  const auto uniform = [](int32_t x) { return __builtin_amdgcn_readfirstlane(x); };  // and in scalar registers
  const int32_t local = uniform(shared.found[1]), first_part = uniform(shared.found[2]), first_tile = uniform(shared.found[3]);
  const int32_t kind = uniform(shared.found[7]);  // long tiles: ranges of each; short ones: minus their count
  w->request = uniform(shared.found[0]);
  w->start = uniform(shared.found[4]);
  w->seen = uniform(shared.found[5]);
  w->rows = uniform(shared.found[6]);
  const int32_t per = max(kind, 1);
  const int32_t at = per == 1 ? local : uniform(local / per);
  const int32_t tiles = kind > 0 ? (w->rows + kTileRows - 1) / kTileRows : -kind;
  const int32_t tile = tiles - 1 - at;  // the rows with the most keys first
  w->r0 = tile * kTileRows;
  w->p_first = w->seen + Quotient(w->r0, a.group);
  w->p_last = w->seen + Quotient(min(w->r0 + kTileRows, w->rows) - 1, a.group);
  w->low = a.window > w->p_first ? 0 : (w->p_first - a.window + 1) / kStep * kStep;
  w->high = w->p_last + 1;
  const int32_t steps = (w->high - w->low + kStep - 1) / kStep;
  w->split = local - at * per;
  w->splits = per == 1 ? 1 : uniform(min((steps + size - 1) / size, per));
  if (w->split >= w->splits) return false;
  const int32_t each = w->splits == 1 ? steps : uniform((steps + w->splits - 1) / w->splits);
  w->begin = min(steps, w->split * each);
  w->end = min(steps, w->begin + each);
  const int32_t first = first_part + at * per;
  w->partial = first + w->split;
  if (per > 1 && w->split == 0 && lead && tid == 0) {
    int32_t* p = b.tiles + static_cast<int64_t>(kTileInts) * (1 + first_tile + at);
    p[0] = first;
    p[1] = w->splits;
    p[2] = w->start;
    p[3] = w->r0;
    p[4] = min(kTileRows, w->rows - w->r0);
  }
  return true;
}

__device__ __forceinline__ bool SeesKey(const BatchAttendArgs& a, int32_t p, int32_t t) { return t <= p && t > p - a.window; }

// Where row rl of the item's tile (rl < rows - r0) lies in the output, in rows of a head.
__device__ __forceinline__ int64_t BatchOutRow(const BatchAttendArgs& a, int32_t start, int32_t r, int32_t group, int32_t kv) {
  const int32_t s = Quotient(r, a.group);
  return static_cast<int64_t>(start + s) * a.heads + kv * group + (r - s * group);
}

// x * s = hi + lo for two values, both parts rounded to nearest: 22 bits where lo is a normal number, and within 2^-25
// where it is not. Four instructions: fp32 in, products and differences exact, each half of a pair on its own.
__device__ __forceinline__ void SplitScaled(float x, float y, float s, h2& hi, h2& lo) {
  uint32_t h, l;
  asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(x), "v"(s));
  asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(y), "v"(s));
  asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(x), "v"(s), "v"(h));
  asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(y), "v"(s), "v"(h));
  hi = __builtin_bit_cast(h2, h);
  lo = __builtin_bit_cast(h2, l);
}
// x = hi + lo for two weights, hi cut towards zero and lo to nearest: three instructions.
__device__ __forceinline__ void SplitWeights(float x, float y, h2& hi, h2& lo) {
  hi = PackRtz(x, y);
  const uint32_t h = __builtin_bit_cast(uint32_t, hi);
  uint32_t l;
  asm("v_fma_mixlo_f16 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(x), "v"(h));
  asm("v_fma_mixhi_f16 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(y), "v"(h));
  lo = __builtin_bit_cast(h2, l);
}
// The larger of |x| and what was largest so far, half by half; a NaN stays one.
__device__ __forceinline__ h2 LargestHalves(h2 x, h2 so_far) {
  asm("v_pk_maximum3_f16 %0, %1, %1, %0 neg_lo:[0,1,0] neg_hi:[0,1,0]" : "+v"(so_far) : "v"(x));
  return so_far;
}

// The page of the 16 tokens from t on, and whether there is one.
struct BatchPages {
  const int32_t* entries;
  int32_t width, pages, shift;
  __device__ __forceinline__ BatchPages(const BatchAttendArgs& a, int32_t request)
      : entries(a.table + static_cast<int64_t>(request) * a.width), width(a.width), pages(a.pages), shift(a.page_shift) {}
  __device__ __forceinline__ int32_t Entry(int32_t t) const {
    const int32_t q = t >> shift;
    return q < width ? entries[q] : -1;
  }
  __device__ __forceinline__ bool Is(int32_t entry) const { return entry >= 0 && entry < pages; }
  // The slot of token t, on page `entry`, or on page 0 where that is none.
  __device__ __forceinline__ int64_t Slot(int32_t entry, int32_t t) const {
    return (static_cast<int64_t>(Is(entry) ? entry : 0) << shift) + (t & ((1 << shift) - 1));
  }
};

// kN floats of a query row from dim d on; past the row its last ones, for MaskQuery: no branch between the loads.
template <int kN>
__device__ __forceinline__ void LoadBatchQuery(const float* q, int32_t dim, int d, bool vec, float (&x)[kN]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      const f4 y = *reinterpret_cast<const f4*>(q + min(d + 4 * i, dim - 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < kN; ++e) x[e] = q[min(d + e, dim - 1)];
  }
}
template <int kN>
__device__ __forceinline__ void MaskQuery(int32_t dim, int d, float (&x)[kN]) {
#pragma unroll
  for (int e = 0; e < kN; ++e) x[e] = d + e < dim ? x[e] : 0.f;
}
__device__ __forceinline__ bool BatchQueryVec(const BatchAttendArgs& a) {  // uniform
  return a.dim % 4 == 0 && a.q_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
}

// Whether row i of the batch was put into the cache. A row that was not is answered as one whose query is not finite: its
// request may have been refused a page, and what lies where its key would be may be of another.
__device__ __forceinline__ bool BatchRowStored(const BatchAttendArgs& a, int32_t i) {
  return a.slots == nullptr || static_cast<uint32_t>(a.slots[i]) < static_cast<uint32_t>(a.pages) << a.page_shift;
}

constexpr int kBatchThreads = 256;
constexpr int kStepTileRows = 16, kPromptTileRows = 128;
constexpr int StepKeys(bool f16) { return f16 ? 32 : 16; }
constexpr int PromptKeys(bool f16) { return f16 ? 64 : 32; }

// A call's two shares: the tiles of requests with few rows and of those with many. groups: workgroups of each.
struct BatchLaunch {
  BatchAttendArgs a;
  BatchSplit step, prompt;
  uint32_t step_groups, prompt_groups;
};
// One of them alone (attend_batch_step.hip, attend_batch_prompt.hip), or both in one launch (attend_batch_mixed.hip).
void LaunchBatchStep(const BatchLaunch& args, bool vec, hipStream_t stream);
void LaunchBatchPrompt(const BatchLaunch& args, bool vec, hipStream_t stream);
void LaunchBatchMixed(const BatchLaunch& args, bool vec, hipStream_t stream);

}  // namespace accel_hip
