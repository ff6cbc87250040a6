// Attention over the 8-bit cache. Codes are integers up to 127 and exact in f16; a query row, brought
// to [2^13, 2^14) by a power of two, and the softmax weights enter as two f16 parts of 11 bits each, so
// both products run on the f16 matrix cores with fp32 sums at two instructions a tile, and the scales
// of the blocks multiply scores and weights.
//
// Few rows (a decode step, drafted tokens): AttendQ8StepKernel below.
#include "attend_common.h"

namespace accel_hip {
namespace {

constexpr int kStepRows = 16;
constexpr int kStepKeys = 32;

// One workgroup per (16 rows of up to 4 key heads, key range): wave w serves head w % hw of them, and the
// waves of a head take its steps of 32 keys in turn, so that a workgroup reads a key row's heads together
// (131072 keys of 8 heads of 128, loads alone: a workgroup a head read them at 4.7 TB/s, 4 heads at 5.7).
// Bound: the cache's bytes over a long range (131072 keys, 32 heads on 8 key heads of 128: 52.3 us, 5.1
// TB/s, and 5.4 of the join); over a short one the chain of load, products, softmax and products of a
// wave's few steps (2048 keys, 9 heads on 3 of 64: 5.7 us and 3.7 of the join). Medians, as in all these
// comments. Keys and values go from memory to registers, and there to f16: no LDS and no barrier in the
// loop. Lane (j, g) = (lane % 16, lane / 16). Per step
//  * S^T = K Q^T on v_mfma_f32_16x16x32_f16: the A operand of instruction (c, half) are the codes
//    64c + 16g + 8 half .. + 7 of key row j, so a lane loads 16 bytes of a key at a time;
//  * O^T += V^T P^T: S^T leaves lane (j, g) the scores of keys 4g .. 4g + 3 and 16 + 4g .. of row j,
//    which are its 8 k-slots of P^T; the A operand of dim tile c is byte c of the DP / 16 bytes that
//    the lane loads at V[key][DP / 16 * j], transposed in registers.
// The next step's keys are requested after the scores, its values after the sums.
template <int DP, int kLoad, int kScales>
__global__ __launch_bounds__(64 * StepWaves(DP)) void AttendQ8StepKernel(
    AttendArgs a, Q8Cache c, int32_t hw, int32_t splits, AttendPartial partial) {
  constexpr int kC = DP / 64;       // 16-byte pieces of a key row per lane
  constexpr int kTiles = DP / 16;   // dim tiles
  constexpr int kVWords = DP / 64;  // 4-byte words of a value row per lane
  constexpr int kGroups = kScales == 1 ? 1 : 2;  // scale loads a step: one, one per 4 keys, one per key
  constexpr int kEach = kScales == 8 ? 4 : 1;
  __shared__ __align__(16) WaveParts<DP, StepWaves(DP), kStepRows> parts;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15;
  const int g = lane >> 4;
  const int32_t unit = static_cast<int32_t>(blockIdx.x);
  const int32_t head_groups = a.kv_heads / hw;
  const int32_t kv0 = unit % head_groups * hw;
  const int32_t kv = kv0 + wave % hw;
  const int32_t rest = unit / head_groups;
  const int32_t split = rest % splits;
  const int32_t tile = rest / splits;
  const int32_t sw = static_cast<int32_t>(blockDim.x) / 64 / hw;  // waves of a head
  const int32_t group = a.heads / a.kv_heads;
  const int32_t rows = a.seq * group;
  const int32_t r0 = tile * kStepRows;
  const KeyRange<kStepKeys> range(a, r0, min(r0 + kStepRows, rows), group);
  const int32_t per = (range.steps + splits - 1) / splits;
  const int32_t end = min(range.steps, (split + 1) * per);
  const int32_t row = min(r0 + j, rows - 1);
  const int32_t s = row / group;
  const int32_t head = kv * group + (row - s * group);
  const int32_t p_row = r0 + j < rows ? a.position + s : -1;  // a row past the last sees nothing
  const int32_t kv_row = a.kv_heads * a.dim;
  const int8_t* kbase = c.k.code + static_cast<int64_t>(kv) * a.dim;
  const int8_t* vbase = c.v.code + static_cast<int64_t>(kv) * a.dim;

  uint32_t kx[2][kC][4];    // [16-key half][piece][word]
  uint32_t vx[8][kVWords];  // [key slot][word]
  float ks[kGroups][kEach], vs[kGroups][kEach];
  const uint32_t koff = static_cast<uint32_t>(j * kv_row + 16 * g);
  const uint32_t voff = static_cast<uint32_t>(4 * g * kv_row + DP / 16 * j);
  const auto load_k = [&](int32_t t0) {
    const CodeRows rows = RowsFrom(kbase, kv_row, a.dim, t0, range.high);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kC; ++i) LoadCodes<4, kLoad>(rows, koff + 16 * h * kv_row + 64 * i, kx[h][i]);
  };
  const auto load_v = [&](int32_t t0) {
    const CodeRows rows = RowsFrom(vbase, kv_row, a.dim, t0, range.high);
#pragma unroll
    for (int e = 0; e < 8; ++e) LoadCodes<kVWords, kLoad>(rows, voff + ((e & 4) * 4 + (e & 3)) * kv_row, vx[e]);
  };
  const auto load_scales = [&](const float* scale, int32_t t0, float (&x)[kGroups][kEach]) {
#pragma unroll
    for (int h = 0; h < kGroups; ++h)
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int32_t t = kScales == 1 ? t0 : t0 + 16 * h + 4 * g + e;
        x[h][e] = scale[static_cast<int64_t>(min(t, range.high - 1) >> c.block_shift) * a.kv_heads + kv];
      }
  };

  int32_t u = split * per + wave / hw;
  if (u < end) {
    const int32_t t0 = range.Key(u);
    load_k(t0);
    load_scales(c.k.scale, t0, ks);
    load_v(t0);
    load_scales(c.v.scale, t0, vs);
  }
  // The row's queries: piece (c, half) of dims 64c + 16g + 8 half .. + 7.
  h8 qh[kC][2], ql[kC][2];
  float row_back;  // a power of two: takes the row's scale out of its scores again
  {
    float x[kC][16];
    const float* q = a.q + s * a.q_stride + static_cast<int64_t>(head) * a.dim;
    const bool vec = QueryVec(a);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kC; ++i) LoadQuery(a, q, 64 * i + 16 * g, vec, x[i]);
#pragma unroll
    for (int i = 0; i < kC; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
    top = max(top, XorLane<16>(top));
    top = max(top, XorLane<32>(top));
    const bool bad = top >= 0x7f800000u;  // no finite row: all of it NaN
    const float scale = RowScale(top);
    row_back = 1.f / scale;
#pragma unroll
    for (int i = 0; i < kC; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        h2 hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y0 = x[i][8 * half + 2 * e] * scale, y1 = x[i][8 * half + 2 * e + 1] * scale;
          SplitF16Nearest(bad ? NAN : y0, bad ? NAN : y1, hi[e], lo[e]);
        }
        qh[i][half] = Join(hi[0], hi[1], hi[2], hi[3]);
        ql[i][half] = Join(lo[0], lo[1], lo[2], lo[3]);
      }
  }

  float m = -INFINITY, l = 0.f, top = 0.f;  // l: this lane's share of the row's sum
  int32_t power = kPowerMax;
  f4 acc[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
  for (; u < end; u += sw) {  // uniform over the wave
    const int32_t t0 = range.Key(u);
    const int32_t next = u + sw < end ? range.Key(u + sw) : -1;
    // The second parts' products first: they are rounded among themselves, before the sums are large.
    f4 st[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      h8 k8[kC][2];
      st[h] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kC; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t w0 = kx[h][i][2 * half] ^ 0x80808080u, w1 = kx[h][i][2 * half + 1] ^ 0x80808080u;
          k8[i][half] = Join(CodesLow(w0), CodesHigh(w0), CodesLow(w1), CodesHigh(w1));
          st[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[i][half], ql[i][half], st[h], 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < kC; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          st[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[i][half], qh[i][half], st[h], 0, 0, 0);
    }
    float factor[kGroups][kEach], value[kGroups][kEach];
#pragma unroll
    for (int h = 0; h < kGroups; ++h)
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        // A value scale that is not finite makes the scores NaN, and a weight of 0 stays one.
        const bool finite = fabsf(vs[h][e]) < INFINITY;
        factor[h][e] = finite ? row_back * ks[h][e] * a.factor : NAN;
        value[h][e] = finite ? vs[h][e] : 0.f;
      }
    float largest = 0.f;
#pragma unroll
    for (int h = 0; h < kGroups; ++h)
#pragma unroll
      for (int e = 0; e < kEach; ++e) largest = fmaxf(largest, value[h][e]);
    const float slack = Slack(__any(largest >= kLargeScale));
    if (next >= 0) {
      load_k(next);
      load_scales(c.k.scale, next, ks);
    }
    __builtin_amdgcn_sched_barrier(0);
    // Scores, and the row's largest. The reference m moves only when a score passes it by 8, so the sums
    // are seldom scaled.
    const bool whole = range.Whole(a, t0);  // a row past the last may see what it likes
    float p[8];
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = st[e >> 2][e & 3] * factor[(e >> 2) % kGroups][(e & 3) % kEach];
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        p[e] = Sees(a, p_row, t0 + (e & 4) * 4 + 4 * g + (e & 3)) ? p[e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, p[e]);
    mx = fmaxf(mx, XorLane<16>(mx));
    mx = fmaxf(mx, XorLane<32>(mx));
    const float m_old = m;
    if (mx > m + slack) m = mx;
    const float base = m == -INFINITY ? 0.f : m;
    const float corr = __builtin_amdgcn_exp2f(m_old - base);
    float sum = 0.f;
    const bool far_scores = __any(fabsf(base) >= kFarScore);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // The product once more, unrounded: near the reference little is left of it.
      const float f = factor[(e >> 2) % kGroups][(e & 3) % kEach];
      const float x = far_scores ? p[e] - base : __builtin_fmaf(st[e >> 2][e & 3], f, -base);
      p[e] = __builtin_amdgcn_exp2f(whole || p[e] != -INFINITY ? x : -INFINITY);
      sum += p[e];
    }
    l = l * corr + sum;
    // The weights times the values' scales, and their largest.
    float step_top = 0.f;
    if (kScales == 1) {
      step_top = __builtin_amdgcn_exp2f(mx - base) * value[0][0];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] *= value[(e >> 2) % kGroups][(e & 3) % kEach];
        step_top = fmaxf(step_top, fabsf(p[e]));
      }
      step_top = fmaxf(step_top, XorLane<16>(step_top));
      step_top = fmaxf(step_top, XorLane<32>(step_top));
    }
    top = fmaxf(top * corr, step_top);
    const int32_t power_old = power;
    power = WeightPower(top, power);
    const float again = ldexpf(corr, power - power_old);
    if (__any(again != 1.f)) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) acc[t] *= again;
    }
    if (kScales == 1) {
      const float f = ldexpf(value[0][0], power);
      if (__any(!(f < 0x1p100f))) {  // a block that is far larger than the sum so far: in two steps
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = ldexpf(p[e] * value[0][0], power);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] *= f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = ldexpf(p[e], power);
    }
    h2 ph[4], pl[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) SplitF16(p[2 * e], p[2 * e + 1], ph[e], pl[e]);
    const h8 p_hi = Join(ph[0], ph[1], ph[2], ph[3]), p_lo = Join(pl[0], pl[1], pl[2], pl[3]);
#pragma unroll
    for (int w = 0; w < kVWords; ++w) {
      uint32_t lo2[4], hi2[4];  // keys 2i, 2i + 1: bytes 0, 0, 1, 1 and 2, 2, 3, 3
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w0 = vx[2 * i][w] ^ 0x80808080u, w1 = vx[2 * i + 1][w] ^ 0x80808080u;
        lo2[i] = __builtin_amdgcn_perm(w1, w0, 0x05010400u);
        hi2[i] = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        h2 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t pair = b < 2 ? lo2[i] : hi2[i];
          x[i] = b & 1 ? CodesHigh(pair) : CodesLow(pair);
        }
        const h8 v8 = Join(x[0], x[1], x[2], x[3]);
        acc[4 * w + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, p_hi, acc[4 * w + b], 0, 0, 0);
        acc[4 * w + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, p_lo, acc[4 * w + b], 0, 0, 0);
      }
    }
    if (next >= 0) {
      load_v(next);
      load_scales(c.v.scale, next, vs);
    }
  }
  // acc[t][r] is O^T[dim DP / 16 (4g + r) + t][row j]; the waves' parts meet in LDS.
  l = l + XorLane<16>(l);
  l = l + XorLane<32>(l);
  const bool far = power < kFarPower;
  if (g == 0) {
    parts.m[wave][j] = m;
    parts.l[wave][j] = far ? -l : l;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int t = 0; t < kTiles; t += 4) {
      const int32_t down = far ? -power - kFarShift : -power;
      *reinterpret_cast<f4*>(&parts.o[wave][j][kTiles * (4 * g + r) + t]) =
          f4{ldexpf(acc[t][r], down), ldexpf(acc[t + 1][r], down), ldexpf(acc[t + 2][r], down), ldexpf(acc[t + 3][r], down)};
    }
  __syncthreads();
  parts.Join(a, kv0, hw, group, r0, rows, split, splits, partial);
}

// A workgroup's threads are (row, key range, 16-byte piece), `lanes` ranges of a row at a time, up to 8
// of a thread in flight at once: a round trip to what other workgroups left is all this costs (3.7-5.7 us; the
// last workgroup of a row to arrive joining them in the step kernel instead took 1-5 us more than this
// launch, for its stores and loads past the XCDs' caches).
constexpr int kJoinThreads = 512;
constexpr int kJoinEach = 8;
__global__ __launch_bounds__(kJoinThreads) void AttendJoinKernel(const float* ml, const float* o, float* out, int32_t rows,
                                                                 int32_t splits, int32_t dim, int32_t lanes, bool vec) {
  __shared__ __align__(16) f4 part_o[kJoinThreads];
  __shared__ float part_m[kJoinThreads];
  __shared__ float part_l[kJoinThreads];
  const int dims = PartialDims(dim);
  const int pieces = dims / 4;
  const int per_row = pieces * lanes;
  const int local = threadIdx.x / per_row;
  const int rest = threadIdx.x - local * per_row;
  const int of = rest / pieces;
  const int piece = rest - of * pieces;
  const int row = static_cast<int>(blockIdx.x) * (kJoinThreads / per_row) + local;
  const bool active = local < kJoinThreads / per_row && row < rows;
  ml += static_cast<int64_t>(row) * splits * 2;
  o += static_cast<int64_t>(row) * splits * dims + 4 * piece;
  float m = -INFINITY, l = 0.f, low = 0.f;
  f4 sum = f4{0.f, 0.f, 0.f, 0.f};
  if (active) {
    for (int c0 = of; c0 < splits; c0 += lanes * kJoinEach) {
      float2 y[kJoinEach];
      f4 x[kJoinEach];
#pragma unroll
      for (int i = 0; i < kJoinEach; ++i) {
        const int c = min(c0 + i * lanes, splits - 1);
        y[i] = *reinterpret_cast<const float2*>(ml + 2 * c);
        x[i] = *reinterpret_cast<const f4*>(o + static_cast<int64_t>(c) * dims);
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
        const float w = __builtin_amdgcn_exp2f(y[i].x - base);
        low = fminf(low, y[i].y);
        l += w * y[i].y;
        sum += w * x[i];
      }
      m = big;
    }
    part_m[threadIdx.x] = m;
    part_l[threadIdx.x] = low < 0.f ? -1.f : l;
    part_o[threadIdx.x] = sum;
  }
  __syncthreads();
  if (!active || of != 0) return;
  const int first = threadIdx.x;
  float big = -INFINITY;
  for (int i = 0; i < lanes; ++i) big = fmaxf(big, part_m[first + i * pieces]);
  const float base = big == -INFINITY ? 0.f : big;
  float total = 0.f;
  low = 0.f;
  sum = f4{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < lanes; ++i) {
    const float w = __builtin_amdgcn_exp2f(part_m[first + i * pieces] - base);
    low = fminf(low, part_l[first + i * pieces]);
    total += w * part_l[first + i * pieces];
    sum += w * part_o[first + i * pieces];
  }
  f4 far = f4{0.f, 0.f, 0.f, 0.f};
  if (low < 0.f) {  // some parts are held times 2^-64: their sum is one of its own
    total = 0.f;
    sum = far;
    for (int c = 0; c < splits; ++c) {
      const float w = __builtin_amdgcn_exp2f(ml[2 * c] - base);
      const f4 x = w * *reinterpret_cast<const f4*>(o + static_cast<int64_t>(c) * dims);
      total += w * fabsf(ml[2 * c + 1]);
      if (ml[2 * c + 1] < 0.f) far += x;
      else sum += x;
    }
  }
  float* dst = out + static_cast<int64_t>(row) * dim + 4 * piece;
  f4 y = f4{__fdiv_rn(sum[0], total), __fdiv_rn(sum[1], total), __fdiv_rn(sum[2], total), __fdiv_rn(sum[3], total)};
  if (low < 0.f)
    y += f4{__fdiv_rn(far[0], total), __fdiv_rn(far[1], total), __fdiv_rn(far[2], total), __fdiv_rn(far[3], total)} * kFarUp;
  if (vec) {
    *reinterpret_cast<f4*>(dst) = y;
  } else {
    for (int e = 0; e < 4; ++e)
      if (4 * piece + e < dim) dst[e] = y[e];
  }
}

}  // namespace

void LaunchAttendJoin(const AttendArgs& a, const AttendPartial& partial, int32_t splits, hipStream_t stream) {
  const bool vec = a.dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  const int32_t rows = a.seq * a.heads;
  const int32_t pieces = PartialDims(a.dim) / 4;
  const int32_t lanes = std::min(splits, kJoinThreads / pieces);
  const int32_t per_group = kJoinThreads / (pieces * lanes);
  const dim3 grid(GridOf((int64_t(rows) + per_group - 1) / per_group, kJoinThreads, "Attention is too large"));
  hipLaunchKernelGGL(AttendJoinKernel, grid, dim3(kJoinThreads), 0, stream, partial.ml, partial.o, a.out, rows, splits,
                     a.dim, lanes, vec);
  Check(hipGetLastError(), "AttendJoinKernel launch");
}

namespace {

template <int DP, int kLoad, int kScales>
void LaunchStep(const AttendArgs& a, const Q8Cache& c, hipStream_t stream) {
  constexpr int kWaves = StepWaves(DP);
  const int64_t cus = Ctx().cu_count > 0 ? Ctx().cu_count : 256;
  const int64_t group = a.heads / a.kv_heads;
  const int64_t tiles = (int64_t(a.seq) * group + kStepRows - 1) / kStepRows;
  const int64_t steps = AttendRangeSteps(a, kStepRows, kStepKeys);
  // Heads together where each wave has several steps; a short range is latency, and fewer parts to join.
  int32_t hw = steps * a.kv_heads * tiles >= 4 * cus * kWaves ? 4 : 1;
  while (a.kv_heads % hw != 0) --hw;
  const int64_t units = tiles * (a.kv_heads / hw);
  if (units > 0x7fffffff) Fail(ACCEL_HIP_INVALID_ARGUMENT, "Attention is too large");
  // Steps that do not fill the CUs are spread one wave a SIMD (2048 keys, 9 heads of 64: 7.6 us in
  // workgroups of four waves, 9.0 of eight, 14.2 in one of sixteen a key head).
  const int32_t sw = hw == 1 && units * steps < cus * kWaves ? 4 : kWaves / hw;
  const AttendSplit split = SplitRange(a, units, steps <= 2 * sw ? 1 : steps / sw);
  const dim3 grid(GridOf(units * split.count, 64 * hw * sw, "Attention is too large")), block(64 * hw * sw);
  hipLaunchKernelGGL((AttendQ8StepKernel<DP, kLoad, kScales>), grid, block, 0, stream, a, c, hw, split.count, split.partial);
  Check(hipGetLastError(), "AttendQ8StepKernel launch");
  if (split.count > 1) LaunchAttendJoin(a, split.partial, split.count, stream);
}

template <int DP>
void LaunchStepOf(const AttendArgs& a, const Q8Cache& c, int load, hipStream_t stream) {
  if (load == 1) LaunchStep<DP, 1, 8>(a, c, stream);
  else if (load == 4) LaunchStep<DP, 4, 8>(a, c, stream);
  else if (c.block_shift >= 5) LaunchStep<DP, 16, 1>(a, c, stream);
  else if (c.block_shift >= 2) LaunchStep<DP, 16, 2>(a, c, stream);
  else LaunchStep<DP, 16, 8>(a, c, stream);
}

}  // namespace

void LaunchAttentionQ8(const AttendArgs& a, const Q8Cache& c, hipStream_t stream) {
  const auto aligned = [&](size_t to) {
    return a.dim % to == 0 && reinterpret_cast<uintptr_t>(c.k.code) % to == 0 &&
           reinterpret_cast<uintptr_t>(c.v.code) % to == 0;
  };
  const int load = aligned(16) ? 16 : aligned(4) ? 4 : 1;
  if (AttendManyRows(a, kPromptPairsQ8)) LaunchAttendPromptQ8(a, c, load, stream);
  else if (a.dim <= 64) LaunchStepOf<64>(a, c, load, stream);
  else if (a.dim <= 128) LaunchStepOf<128>(a, c, load, stream);
  else LaunchStepOf<256>(a, c, load, stream);
}

}  // namespace accel_hip
