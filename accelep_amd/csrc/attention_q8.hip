// Attention over the 8-bit cache. Codes are integers up to 127 and exact in f16; a query row, brought
// to [2^13, 2^14) by a power of two, and the softmax weights enter as two f16 parts of 11 bits each, so
// both products run on the f16 matrix cores with fp32 sums at two instructions a tile, and the scales
// of the blocks multiply scores and weights.
//
// Few rows (a decode step, drafted tokens): AttendQ8StepKernel below.
#include "attend_common.h"

namespace accel_hip {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kStepRows = 16;
constexpr int kStepKeys = 32;

// One workgroup per (16 rows of a key head, key range); its waves take every fourth step of 32 keys.
// Bound: the cache's bytes. Keys and values go from memory to registers, and there to f16: no LDS and
// no barrier in the loop. Lane (j, g) = (lane % 16, lane / 16). Per step
//  * S^T = K Q^T on v_mfma_f32_16x16x32_f16: the A operand of instruction (c, half) are the codes
//    64c + 16g + 8 half .. + 7 of key row j, so a lane loads 16 bytes of a key at a time;
//  * O^T += V^T P^T: S^T leaves lane (j, g) the scores of keys 4g .. 4g + 3 and 16 + 4g .. of row j,
//    which are its 8 k-slots of P^T; the A operand of dim tile c is byte c of the DP / 16 bytes that
//    the lane loads at V[key][DP / 16 * j], transposed in registers.
// The next step's keys are requested after the scores, its values after the sums.
template <int DP, int kLoad, int kScales>
__global__ __launch_bounds__(kThreads) void AttendQ8StepKernel(AttendArgs a, Q8Cache c, int32_t splits,
                                                               AttendPartial partial) {
  constexpr int kC = DP / 64;       // 16-byte pieces of a key row per lane
  constexpr int kTiles = DP / 16;   // dim tiles
  constexpr int kVWords = DP / 64;  // 4-byte words of a value row per lane
  constexpr int kGroups = kScales == 1 ? 1 : 2;  // scale loads a step: one, one per 4 keys, one per key
  constexpr int kEach = kScales == 8 ? 4 : 1;
  __shared__ __align__(16) WaveParts<DP, kWaves, kStepRows> parts;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15;
  const int g = lane >> 4;
  const int32_t unit = static_cast<int32_t>(blockIdx.x);
  const int32_t kv = unit % a.kv_heads;
  const int32_t rest = unit / a.kv_heads;
  const int32_t split = rest % splits;
  const int32_t tile = rest / splits;
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
  const int64_t kv_row = static_cast<int64_t>(a.kv_heads) * a.dim;
  const int8_t* kbase = c.k.code + static_cast<int64_t>(kv) * a.dim;
  const int8_t* vbase = c.v.code + static_cast<int64_t>(kv) * a.dim;

  uint32_t kx[2][kC][4];    // [16-key half][piece][word]
  uint32_t vx[8][kVWords];  // [key slot][word]
  float ks[kGroups][kEach], vs[kGroups][kEach];
  const auto load_k = [&](int32_t t0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int8_t* p = kbase + min(t0 + 16 * h + j, range.high - 1) * kv_row;
#pragma unroll
      for (int i = 0; i < kC; ++i) {
        const int d = 64 * i + 16 * g;
        if (kLoad == 16) {
          const uint4 w = d < a.dim ? *reinterpret_cast<const uint4*>(p + d) : make_uint4(0, 0, 0, 0);
          kx[h][i][0] = w.x, kx[h][i][1] = w.y, kx[h][i][2] = w.z, kx[h][i][3] = w.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) kx[h][i][e] = LoadCodes4<kLoad>(p + d + 4 * e, d + 4 * e, a.dim);
        }
      }
    }
  };
  const auto load_v = [&](int32_t t0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = DP / 16 * j;
      const int8_t* p = vbase + min(t0 + (e & 4) * 4 + 4 * g + (e & 3), range.high - 1) * kv_row + d;
      if (kLoad == 16 && kVWords == 2) {
        const uint2 w = d < a.dim ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
        vx[e][0] = w.x, vx[e][1 % kVWords] = w.y;
      } else if (kLoad == 16 && kVWords == 4) {
        const uint4 w = d < a.dim ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
        vx[e][0] = w.x, vx[e][1 % kVWords] = w.y, vx[e][2 % kVWords] = w.z, vx[e][3 % kVWords] = w.w;
      } else {
#pragma unroll
        for (int w = 0; w < kVWords; ++w) vx[e][w] = LoadCodes4<kLoad>(p + 4 * w, d + 4 * w, a.dim);
      }
    }
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

  int32_t u = split * per + wave;
  if (u < end) {
    const int32_t t0 = range.Key(u);
    load_k(t0);
    load_scales(c.k.scale, t0, ks);
    load_v(t0);
    load_scales(c.v.scale, t0, vs);
  }
  // The row's queries: piece (c, half) of dims 64c + 16g + 8 half .. + 7.
  h8 qh[kC][2], ql[kC][2];
  float row_factor;
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
    row_factor = kLog2e / scale * __fdiv_rn(1.f, __fsqrt_rn(static_cast<float>(a.dim)));
#pragma unroll
    for (int i = 0; i < kC; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        h2 hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y0 = x[i][8 * half + 2 * e] * scale, y1 = x[i][8 * half + 2 * e + 1] * scale;
          SplitF16(bad ? NAN : y0, bad ? NAN : y1, hi[e], lo[e]);
        }
        qh[i][half] = Join(hi[0], hi[1], hi[2], hi[3]);
        ql[i][half] = Join(lo[0], lo[1], lo[2], lo[3]);
      }
  }

  RowState row_state;
  float& m = row_state.m;
  float& l = row_state.l;  // this lane's share of the row's sum
  f4 acc[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
  for (; u < end; u += kWaves) {  // uniform over the wave
    const int32_t t0 = range.Key(u);
    const int32_t next = u + kWaves < end ? range.Key(u + kWaves) : -1;
    f4 st[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      st[h] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kC; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t w0 = kx[h][i][2 * half] ^ 0x80808080u, w1 = kx[h][i][2 * half + 1] ^ 0x80808080u;
          const h8 k8 = Join(CodesLow(w0), CodesHigh(w0), CodesLow(w1), CodesHigh(w1));
          st[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[i][half], st[h], 0, 0, 0);
          st[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[i][half], st[h], 0, 0, 0);
        }
    }
    float factor[kGroups][kEach], value[kGroups][kEach];
#pragma unroll
    for (int h = 0; h < kGroups; ++h)
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        factor[h][e] = row_factor * ks[h][e];
        value[h][e] = vs[h][e];
      }
    if (next >= 0) {
      load_k(next);
      load_scales(c.k.scale, next, ks);
    }
    __builtin_amdgcn_sched_barrier(0);
    // Scores, and the row's largest.
    const bool whole = range.Whole(a, t0) && r0 + kStepRows <= rows;
    uint32_t seen = 255;
    if (!whole) {
      seen = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        seen |= Sees(a, p_row, t0 + (e & 4) * 4 + 4 * g + (e & 3)) ? 1u << e : 0u;
    }
    float p[8];
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = seen >> e & 1 ? st[e >> 2][e & 3] * factor[(e >> 2) % kGroups][(e & 3) % kEach] : -INFINITY;
      mx = fmaxf(mx, p[e]);
    }
    mx = fmaxf(mx, XorLane<16>(mx));
    mx = fmaxf(mx, XorLane<32>(mx));
    const float m_new = fmaxf(m, mx);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = __builtin_amdgcn_exp2f(m - base);
    float sum = 0.f, top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = __builtin_amdgcn_exp2f(p[e] - base);
      sum += p[e];
      p[e] = seen >> e & 1 ? p[e] * value[(e >> 2) % kGroups][(e & 3) % kEach] : 0.f;
      top = fmaxf(top, fabsf(p[e]));
    }
    l = l * corr + sum;
    m = m_new;
    top = fmaxf(top, XorLane<16>(top));
    top = fmaxf(top, XorLane<32>(top));
    row_state.top = fmaxf(row_state.top * corr, top);
    const int32_t power = RowState::PowerOf(row_state.top);
    const float again = ldexpf(corr, power - row_state.power);
    row_state.power = power;
    if (__any(again != 1.f)) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) acc[t] *= again;
    }
    h2 ph[4], pl[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) SplitF16(ldexpf(p[2 * e], power), ldexpf(p[2 * e + 1], power), ph[e], pl[e]);
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
  if (g == 0) {
    parts.m[wave][j] = m;
    parts.l[wave][j] = l;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int t = 0; t < kTiles; t += 4) {
      const int32_t down = -row_state.power;
      *reinterpret_cast<f4*>(&parts.o[wave][j][kTiles * (4 * g + r) + t]) =
          f4{ldexpf(acc[t][r], down), ldexpf(acc[t + 1][r], down), ldexpf(acc[t + 2][r], down), ldexpf(acc[t + 3][r], down)};
    }
  __syncthreads();
  parts.Join(a, kv, group, r0, rows, split, splits, partial);
}

// One workgroup per row: its threads are the row's 16-byte pieces times the key ranges, 8 ranges of a
// thread in flight at once, since a round trip to what other workgroups left is all this costs.
constexpr int kJoinEach = 8;
__global__ __launch_bounds__(kThreads) void AttendJoinKernel(const float* ml, const float* o, float* out, int32_t splits,
                                                             int32_t dim, bool vec) {
  __shared__ __align__(16) f4 part_o[kThreads];
  __shared__ float part_m[kThreads];
  __shared__ float part_l[kThreads];
  const int dims = PartialDims(dim);
  const int pieces = dims / 4;
  const int lanes = kThreads / pieces;  // key ranges at a time
  const int piece = threadIdx.x % pieces;
  const int of = threadIdx.x / pieces;
  const int64_t row = blockIdx.x;
  ml += row * splits * 2;
  o += row * splits * dims + 4 * piece;
  float m = -INFINITY, l = 0.f;
  f4 sum = f4{0.f, 0.f, 0.f, 0.f};
  if (of < lanes) {
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
        l += w * y[i].y;
        sum += w * x[i];
      }
      m = big;
    }
    part_m[threadIdx.x] = m;
    part_l[threadIdx.x] = l;
    part_o[threadIdx.x] = sum;
  }
  __syncthreads();
  if (of != 0) return;
  float big = part_m[piece];
  for (int i = 1; i < lanes; ++i) big = fmaxf(big, part_m[piece + i * pieces]);
  const float base = big == -INFINITY ? 0.f : big;
  float total = 0.f;
  sum = f4{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < lanes; ++i) {
    const float w = __builtin_amdgcn_exp2f(part_m[piece + i * pieces] - base);
    total += w * part_l[piece + i * pieces];
    sum += w * part_o[piece + i * pieces];
  }
  float* dst = out + row * dim + 4 * piece;
  const f4 y = f4{__fdiv_rn(sum[0], total), __fdiv_rn(sum[1], total), __fdiv_rn(sum[2], total), __fdiv_rn(sum[3], total)};
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
  hipLaunchKernelGGL(AttendJoinKernel, dim3(static_cast<uint32_t>(a.seq) * static_cast<uint32_t>(a.heads)), dim3(kThreads), 0,
                     stream, partial.ml, partial.o, a.out, splits, a.dim, vec);
  Check(hipGetLastError(), "AttendJoinKernel launch");
}

AttendSplit SplitRange(const AttendArgs& a, int64_t units, int64_t most) {
  const int64_t cus = Ctx().cu_count > 0 ? Ctx().cu_count : 256;
  const int64_t count = std::max<int64_t>(1, std::min<int64_t>(2 * cus / units, most));
  const int64_t parts = int64_t(a.seq) * a.heads * count;
  const size_t ml_bytes = (static_cast<size_t>(parts) * 2 * sizeof(float) + 15) & ~size_t(15);
  const size_t bytes = ml_bytes + static_cast<size_t>(parts * PartialDims(a.dim)) * sizeof(float);
  AttendSplit split;
  if (count == 1 || !ScratchReady(bytes, kTempFlags, 0)) return split;
  split.count = static_cast<int32_t>(count);
  split.partial.ml = static_cast<float*>(Workspace(bytes));
  split.partial.o = split.partial.ml + ml_bytes / sizeof(float);
  return split;
}

namespace {

template <int DP>
void LaunchStep(const AttendArgs& a, const Q8Cache& c, int load, const AttendSplit& split, int64_t units,
                hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(units * split.count)), block(kThreads);
#define ACCEL_STEP(L, S) \
  hipLaunchKernelGGL((AttendQ8StepKernel<DP, L, S>), grid, block, 0, stream, a, c, split.count, split.partial)
  if (load == 16) {
    if (c.block_shift >= 5) ACCEL_STEP(16, 1);
    else if (c.block_shift >= 2) ACCEL_STEP(16, 2);
    else ACCEL_STEP(16, 8);
  } else if (load == 4) {
    ACCEL_STEP(4, 8);
  } else {
    ACCEL_STEP(1, 8);
  }
#undef ACCEL_STEP
  Check(hipGetLastError(), "AttendQ8StepKernel launch");
}

}  // namespace

void LaunchAttentionQ8(const AttendArgs& a, const Q8Cache& c, hipStream_t stream) {
  const auto aligned = [&](size_t to) {
    return a.dim % to == 0 && reinterpret_cast<uintptr_t>(c.k.code) % to == 0 && reinterpret_cast<uintptr_t>(c.v.code) % to == 0;
  };
  const int load = aligned(16) ? 16 : aligned(4) ? 4 : 1;
  const int64_t group = a.heads / a.kv_heads;
  if (int64_t(a.seq) * group > kAttendPromptRows) {
    LaunchAttendPromptQ8(a, c, load, stream);
    return;
  }
  const int64_t tiles = (int64_t(a.seq) * group + kStepRows - 1) / kStepRows;
  const int64_t units = tiles * a.kv_heads;
  if (units > 0x7fffffff) Fail(ACCEL_HIP_INVALID_ARGUMENT, "Attention is too large");
  const AttendSplit split = SplitRange(a, units, AttendRangeSteps(a, kStepRows, kStepKeys) / kWaves);
  if (a.dim <= 64) LaunchStep<64>(a, c, load, split, units, stream);
  else if (a.dim <= 128) LaunchStep<128>(a, c, load, split, units, stream);
  else LaunchStep<256>(a, c, load, split, units, stream);
  if (split.count > 1) LaunchAttendJoin(a, split.partial, split.count, stream);
}

}  // namespace accel_hip
