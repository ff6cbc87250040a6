// Attention with a sliding window over an fp32 cache: the row at p sees the keys t <= p with
// t > p - window or t < sinks, and reads no others.
//
// Few rows (a decode step, drafted tokens): AttendF32StepKernel below. Many: attend_prompt.hip.
#include "attend_common.h"

namespace accel_hip {
namespace {

constexpr int kRows = 16;
constexpr int kKeys = 16;  // of a wave's step
constexpr uint32_t kLargeBits = (127 + 96) << 23;  // 2^96

// One argument, not five: less of the host's work for a launch (a step over a window of 4096: 16.5 -> 16.1 us).
struct StepArgs {
  AttendArgs a;
  const float* k;
  const float* v;
  int32_t splits;
  AttendPartial partial;
};

// One workgroup per (16 rows of a key head, key range); its waves take its steps of 16 keys in turn.
// Bound: the bytes of the keys that are seen, and over a window the chain of a wave's one or two steps (4100
// keys, 32 heads on 8 key heads of 128: 33.6 MB in 13.1 us, 2.6 TB/s). Both products run on
// v_mfma_f32_16x16x4f32, which takes fp32 as it is, with every operand straight from memory. Lane (j, g) =
// (lane % 16, lane / 16):
//  * S^T = K Q^T: k slot g of instruction (i, e) is dim 16i + 4g + e, so a lane loads 16 bytes of key
//    row j at a time and a key row's pieces lie side by side;
//  * O^T += V^T P^T: S^T leaves the lane the scores of keys 4g .. 4g + 3 of row j; k slot g of
//    instruction s is key 4g + s, the A operand of dim tile (c, t) float t of the 16 bytes at
//    V[key][64c + 4j].
// A key or value row that is not finite would reach rows that do not see it, as 0 * NaN: a step that
// holds one (a test of the bits, uniform) has its values taken as zeros and its weights as NaN. The same test
// finds values from 2^96 on, whose sum over the keys may pass the largest float: a row that gives one of them a
// weight holds its sum times 2^-64 until that weight is next to nothing beside later ones.
template <int DP, int kLoad>
__global__ __launch_bounds__(64 * StepWaves(DP)) void AttendF32StepKernel(
    StepArgs args) {
  const AttendArgs& a = args.a;
  const float* k = args.k;
  const float* v = args.v;
  const int32_t splits = args.splits;
  const int32_t waves = static_cast<int32_t>(blockDim.x) / 64;
  constexpr int kI = DP / 16;  // 16-byte pieces of a key row per lane
  constexpr int kC = DP / 64;  // of a value row
  __shared__ __align__(16) WaveParts<DP, StepWaves(DP), kRows> parts;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15;
  const int g = lane >> 4;
  const int32_t kv = static_cast<int32_t>(blockIdx.x) % a.kv_heads;
  const int32_t rest = static_cast<int32_t>(blockIdx.x) / a.kv_heads;
  const int32_t split = rest % splits;
  const int32_t group = a.heads / a.kv_heads;
  const int32_t rows = a.seq * group;
  const int32_t r0 = rest / splits * kRows;
  const KeyRange<kKeys> range(a, r0, min(r0 + kRows, rows), group);
  const int32_t per = (range.steps + splits - 1) / splits;
  const int32_t begin = min(range.steps, split * per);
  const int32_t end = min(range.steps, begin + per);
  const int32_t row = min(r0 + j, rows - 1);
  const int32_t s = row / group;
  const int32_t head = kv * group + (row - s * group);
  const int32_t p_row = r0 + j < rows ? a.position + s : -1;  // a row past the last sees nothing
  const int64_t kv_row = static_cast<int64_t>(a.kv_heads) * a.dim;
  const float* kbase = k + static_cast<int64_t>(kv) * a.dim;
  const float* vbase = v + static_cast<int64_t>(kv) * a.dim;

  f4 kx[kI], vx[4][kC];
  // A piece past a head's dims reads its last (it meets a query of 0, or makes a dim that is not stored), a
  // row past the range the last one.
  const auto piece = [&](const float* p, int d) {
    if (kLoad == 16) return *reinterpret_cast<const f4*>(p + min(d, a.dim - 4));
    f4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = p[min(d + e, a.dim - 1)];
    return x;
  };
  const auto load_k = [&](int32_t t0) {
    const float* p = kbase + min(t0 + j, range.high - 1) * kv_row;
#pragma unroll
    for (int i = 0; i < kI; ++i) kx[i] = piece(p, 16 * i + 4 * g);
  };
  const auto load_v = [&](int32_t t0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* p = vbase + min(t0 + 4 * g + e, range.high - 1) * kv_row;
#pragma unroll
      for (int c = 0; c < kC; ++c) vx[e][c] = piece(p, 64 * c + 4 * j);
    }
  };
  // The queries are requested first: the first products wait for them and the keys, not for the values
  // (a step over a window of 4096: 16.9 -> 16.5 us).
  f4 q[kI];
  {
    const float* p = a.q + s * a.q_stride + static_cast<int64_t>(head) * a.dim;
    const bool vec = QueryVec(a);
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      float x[4];
      LoadQuery(a, p, 16 * i + 4 * g, vec, x);
      q[i] = f4{x[0], x[1], x[2], x[3]};
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  int32_t u = begin + wave;
  if (u < end) {
    const int32_t t0 = range.Key(u);
    load_k(t0);
    load_v(t0);
  }

  float m = -INFINITY, l = 0.f;  // l: this lane's share of the row's sum
  float shift = 1.f, share = 0.f;  // the weighted sum's power of two, and the largest weight now of a large value
  f4 acc[kC][4];
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[c][t] = f4{0.f, 0.f, 0.f, 0.f};
  for (; u < end; u += waves) {  // uniform over the wave
    const int32_t t0 = range.Key(u);
    const int32_t next = u + waves < end ? range.Key(u + waves) : -1;
    f4 st0 = f4{0.f, 0.f, 0.f, 0.f}, st1 = st0;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        st0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[i][e], q[i][e], st0, 0, 0, 0);
        st1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[i][e + 1], q[i][e + 1], st1, 0, 0, 0);
        top = max(top, max(FloatBits(kx[i][e]) & 0x7fffffffu, FloatBits(kx[i][e + 1]) & 0x7fffffffu));
      }
    const uint64_t bad_keys = __ballot(top >= 0x7f800000u);
    if (next >= 0) load_k(next);
    __builtin_amdgcn_sched_barrier(0);
    uint32_t vtop[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      vtop[e] = 0;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) vtop[e] = max(vtop[e], FloatBits(vx[e][c][t]) & 0x7fffffffu);
    }
    uint32_t bad = 0, large = 0;  // of the lane's keys 4g + e
    if (__any(max(max(vtop[0], vtop[1]), max(vtop[2], vtop[3])) >= kLargeBits) || bad_keys != 0) {
      const uint32_t keys16 = static_cast<uint32_t>(bad_keys | bad_keys >> 16 | bad_keys >> 32 | bad_keys >> 48) & 0xffffu;
      bad = keys16 >> (4 * g) & 15u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t lanes = __ballot(vtop[e] >= 0x7f800000u);
        if ((__ballot(vtop[e] >= kLargeBits) >> (16 * g) & 0xffffu) != 0) large |= 1u << e;
        if ((lanes >> (16 * g) & 0xffffu) != 0) {
          bad |= 1u << e;
#pragma unroll
          for (int c = 0; c < kC; ++c) vx[e][c] = f4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
    float p[4];
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = Sees(a, p_row, t0 + 4 * g + e);
      st0[e] = in ? (bad >> e & 1 ? NAN : st0[e] + st1[e]) : -INFINITY;
      mx = fmaxf(mx, st0[e]);
    }
    mx = fmaxf(mx, XorLane<16>(mx));
    mx = fmaxf(mx, XorLane<32>(mx)) * a.factor;
    const float m_new = fmaxf(m, mx);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = __builtin_amdgcn_exp2f(m - base);
    float sum = 0.f;
    const bool far_scores = __any(fabsf(base) >= kFarScore);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[e] = __builtin_amdgcn_exp2f(far_scores ? st0[e] * a.factor - base : __builtin_fmaf(st0[e], a.factor, -base));
      sum += p[e];
    }
    l = l * corr + sum;
    m = m_new;
    float again = corr;
    share *= corr;
    if (shift != 1.f && share < 0x1p-40f) {  // little is left of the large values
      again *= kFarUp;
      shift = 1.f;
    }
    if (__any(large != 0)) {
      bool weighs = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) weighs = weighs || ((large >> e & 1) != 0 && p[e] > 0.f);
      const uint64_t lanes = __ballot(weighs);
      if (((lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) >> j & 1) != 0) {
        share = 1.f;
        again *= shift == 1.f ? kFarDown : 1.f;
        shift = kFarDown;
      }
    }
    if (__any(again != 1.f)) {
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[c][t] *= again;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] *= shift;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          acc[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[e][c][t], p[e], acc[c][t], 0, 0, 0);
    if (next >= 0) load_v(next);
  }
  // acc[c][t][r] is O^T[dim 64c + 16g + 4r + t][row j]; the waves' parts meet in LDS.
  l = l + XorLane<16>(l);
  l = l + XorLane<32>(l);
  if (g == 0) {
    parts.m[wave][j] = m;
    parts.l[wave][j] = shift == 1.f ? l : -l;
  }
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f4*>(&parts.o[wave][j][64 * c + 16 * g + 4 * r]) =
          f4{acc[c][0][r], acc[c][1][r], acc[c][2][r], acc[c][3][r]};
  __syncthreads();
  parts.Join(a, kv, 1, group, r0, rows, split, splits, args.partial);
}

template <int DP>
void LaunchStep(const AttendArgs& a, const float* k, const float* v, bool vec, hipStream_t stream) {
  constexpr int kWaves = StepWaves(DP);
  const int64_t group = a.heads / a.kv_heads;
  const int64_t units = (int64_t(a.seq) * group + kRows - 1) / kRows * a.kv_heads;
  if (units > 0x7fffffff) Fail(ACCEL_HIP_INVALID_ARGUMENT, "Attention is too large");
  const int64_t steps = AttendRangeSteps(a, kRows, kKeys);
  // Steps that do not fill the CUs are spread one wave a SIMD.
  const int64_t cus = Ctx().cu_count > 0 ? Ctx().cu_count : 256;
  const int32_t waves = units * steps < cus * kWaves ? 4 : kWaves;
  const AttendSplit split = SplitRange(a, units, steps <= 2 * waves ? 1 : steps / waves);
  const dim3 grid(GridOf(units * split.count, 64 * waves, "Attention is too large")), block(64 * waves);
  const StepArgs args{a, k, v, split.count, split.partial};
  if (vec) hipLaunchKernelGGL((AttendF32StepKernel<DP, 16>), grid, block, 0, stream, args);
  else hipLaunchKernelGGL((AttendF32StepKernel<DP, 4>), grid, block, 0, stream, args);
  Check(hipGetLastError(), "AttendF32StepKernel launch");
  if (split.count > 1) LaunchAttendJoin(a, split.partial, split.count, stream);
}

}  // namespace

void LaunchAttentionWindow(const AttendArgs& a, const float* k, const float* v, hipStream_t stream) {
  const bool vec = a.dim % 4 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0;
  if (AttendManyRows(a, kPromptPairsF32)) LaunchAttendPromptF32(a, k, v, vec ? 16 : 4, stream);
  else if (a.dim <= 64) LaunchStep<64>(a, k, v, vec, stream);
  else if (a.dim <= 128) LaunchStep<128>(a, k, v, vec, stream);
  else LaunchStep<256>(a, k, v, vec, stream);
}

}  // namespace accel_hip
