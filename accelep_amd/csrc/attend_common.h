// What the attention kernels over the 8-bit cache and in a window share: which keys a block of query
// rows reads and a row sees, queries and softmax weights as two f16 parts, codes as f16, and the join
// of key ranges.
#pragma once

#include <algorithm>

#include "attend_split.h"
#include "device_common.h"

namespace accel_hip {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

// Rows are pairs (query s, head g of a key head's group), row = s * group + g: a key head's rows share
// its keys. The keys that rows [r0, r1) read, in steps of kStep keys: first those before `low` that
// stay visible, then [low, high). Both parts begin at a multiple of kStep, so a step lies in one part,
// and scale blocks of kStep tokens and more hold whole steps.
template <int kStep>
struct KeyRange {
  int32_t low, high;          // high: one past the last row's own key
  int32_t first_steps, steps;
  int32_t p_first, p_last;    // the rows' positions
  __device__ __forceinline__ KeyRange(const AttendArgs& a, int32_t r0, int32_t r1, int32_t group) {
    p_first = a.position + r0 / group;
    p_last = a.position + (r1 - 1) / group;
    low = a.window == kNoWindow ? 0 : max(0, p_first - a.window + 1) / kStep * kStep;
    high = p_last + 1;
    first_steps = (min(a.sinks, low) + kStep - 1) / kStep;
    steps = first_steps + (high - low + kStep - 1) / kStep;
  }
  __device__ __forceinline__ int32_t Key(int32_t step) const {
    return step < first_steps ? step * kStep : low + (step - first_steps) * kStep;
  }
  // Every row sees every key of the step.
  __device__ __forceinline__ bool Whole(const AttendArgs& a, int32_t t0) const {
    const int32_t last = t0 + kStep - 1;
    return last <= p_first && (t0 > p_last - a.window || last < a.sinks);
  }
};
__device__ __forceinline__ bool Sees(const AttendArgs& a, int32_t p, int32_t t) {
  return t <= p && (t > p - a.window || t < a.sinks);
}

__device__ __forceinline__ h2 PackRtz(float x, float y) {
  return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(x, y));
}
// x = hi + lo to 22 bits, each part 11 cut towards zero: for |x| between 2^-3 and 2^15 what is left, the last
// two of x's 24 bits at most, is within 1.5 * 2^-22 |x|, under that below 2^-24 (the spacing of f16's
// subnormal numbers). Both products with exact f16 operands are exact in the matrix core's fp32 sums.
__device__ __forceinline__ void SplitF16(float x, float y, h2& hi, h2& lo) {
  hi = PackRtz(x, y);
  float rx, ry;  // x - hi[0], y - hi[1]: one instruction each, which the compiler makes two of
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rx) : "v"(hi), "v"(x));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(ry) : "v"(hi), "v"(y));
  lo = PackRtz(rx, ry);
}

// The same with both parts rounded to nearest, for what is split once: the second part's sign is then no
// longer the first's, so the product of two second parts, which the fp32 kernels leave out, has no bias.
__device__ __forceinline__ void SplitF16Nearest(float x, float y, h2& hi, h2& lo) {
  hi = h2{static_cast<_Float16>(x), static_cast<_Float16>(y)};
  lo = h2{static_cast<_Float16>(x - static_cast<float>(hi[0])), static_cast<_Float16>(y - static_cast<float>(hi[1]))};
}

// 2^(13 - e) for a row whose largest magnitude has the exponent e: the row then fills [2^13, 2^14).
__device__ __forceinline__ float RowScale(uint32_t top_bits) {
  const int32_t e = static_cast<int32_t>(top_bits >> 23) - 127;
  return top_bits == 0 ? 1.f : __uint_as_float(static_cast<uint32_t>(min(13 - e, 127) + 127) << 23);
}

// Four codes, already biased by 128 (w ^ 0x80808080), as two pairs of f16: 0x64uu is 1024 + uu.
__device__ __forceinline__ h2 CodesLow(uint32_t w) {
  return __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - h2{1152, 1152};
}
__device__ __forceinline__ h2 CodesHigh(uint32_t w) {
  return __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - h2{1152, 1152};
}
__device__ __forceinline__ h8 Join(h2 a, h2 b, h2 c, h2 d) { return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]}; }

// A row's softmax while its keys pass holds m, a reference for its scores in log2 units, l, the sum of
// p = 2^(s - m), and `top`, the largest p * value scale so far. The weighted sum holds p * value scale *
// 2^power, with top * 2^power kept in [2^3, 2^15): a weight then has 22 bits down to 2^-6 of the largest
// and is off by 2^-27 of that below, whatever the scales, and a key that a row does not see has no say.
constexpr int32_t kPowerMax = 127;
// From this power on the sum of up to 2^31 keys is less than 2^100 when the power is taken out.
constexpr int32_t kFarPower = -40;
__device__ __forceinline__ int32_t WeightPower(float top, int32_t power) {
  const float at = ldexpf(top, power);
  if (at < 0x1p15f && (at >= 8.f || !(top > 0.f))) return power;
  const int32_t e = static_cast<int32_t>(__float_as_uint(top) >> 23) - 127;
  return min(6 - e, kPowerMax);
}

// By how much a score may pass the reference before it moves, in log2 units: p then stays within 2^8. Where a
// value scale is near the largest float (they reach 2^121) p times it has to stay in range.
constexpr float kLargeScale = 0x1p112f;
__device__ __forceinline__ float Slack(bool large_scale) { return large_scale ? 0.f : 8.f; }

// The exponent s - m is one fma of the unrounded product s, and the reference m a rounded one: their distance,
// up to 2^-24 |m|, counts for nothing until it is as large as the exponents that matter. From here on s is
// rounded as m was, so that the largest key's exponent is 0.
constexpr float kFarScore = 0x1p20f;

// Codes are read through buffer descriptors whose bounds are the range's last key row: rows past it read
// as 0, with no address to clamp. Dims past a head's read whatever lies there, a code of the next head or
// 0, which meets a query of 0, or as a value makes a dim that is not stored.
typedef __amdgpu_buffer_rsrc_t CodeRows;
__device__ __forceinline__ CodeRows RowsFrom(const int8_t* head, int32_t kv_row, int32_t dim, int32_t t0, int32_t high) {
  // The bytes from this head's part of row t0 to its end in the last row; a step's offsets stay below 2^30.
  const int64_t bytes = static_cast<int64_t>(high - 1 - t0) * kv_row + dim;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(head + static_cast<int64_t>(t0) * kv_row), 0,
                                           static_cast<int32_t>(min(bytes, int64_t(1) << 30)), 0x00027000);
}
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// kWords * 4 codes at the offset; kLoad: the bytes that lie at a multiple of themselves (4 or more: words).
template <int kWords, int kLoad>
__device__ __forceinline__ void LoadCodes(CodeRows rows, uint32_t offset, uint32_t (&w)[kWords]) {
  if constexpr (kLoad == 16 && kWords == 4) {
    const u4 x = __builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = x[e];
  } else if constexpr (kLoad == 16 && kWords == 2) {
    const u2 x = __builtin_amdgcn_raw_buffer_load_b64(rows, offset, 0, 0);
    w[0] = x[0];
    w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if (kLoad >= 4) {
        w[i] = __builtin_amdgcn_raw_buffer_load_b32(rows, offset + 4 * i, 0, 0);
      } else {
        w[i] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[i] |= static_cast<uint32_t>(__builtin_amdgcn_raw_buffer_load_b8(rows, offset + 4 * i + e, 0, 0)) << (8 * e);
      }
    }
  }
}

// The most steps of a block of `rows` rows' key range.
inline int64_t AttendRangeSteps(const AttendArgs& a, int64_t rows, int64_t step) {
  const int64_t group = a.heads / a.kv_heads;
  const int64_t queries = std::min<int64_t>(a.seq, (rows + group - 2) / group + 1);
  const int64_t end = int64_t(a.position) + a.seq;
  if (a.window == kNoWindow) return (end + step - 1) / step;
  const int64_t keys = std::min<int64_t>(end, int64_t(a.window) + queries + step);
  return (keys + step - 1) / step + (std::min<int64_t>(a.sinks, end) + step - 1) / step;
}

// Waves of a step workgroup at most: two a SIMD, one of head dim 256, whose sums and operands take more than
// half of a SIMD's registers.
constexpr int StepWaves(int dp) { return dp > 128 ? 4 : 8; }

// Whether the rows are many enough for the tiles of keys to go through LDS: more than 16 of a key head,
// and `pairs` of rows (in 16s) and keys. Below, the step kernels' spread over the CUs wins. 16 heads, 4 key
// heads of 128, us (step kernel, prompt kernel): 8-bit, 24 rows of 1000 keys 11.3, 18.2; 24 of 16000 25.9,
// 26.3 (6.1 M pairs); 32 of 16000 30.0, 27.7; fp32, 16 rows of 1000 12.6, 19.1; 8 of 16000 26.2, 30.3; 16
// of 16000 38.6, 31.2 (4.1 M pairs).
constexpr int64_t kPromptPairsQ8 = 6 << 20;
constexpr int64_t kPromptPairsF32 = 3 << 20;
inline bool AttendManyRows(const AttendArgs& a, int64_t pairs) {
  const int64_t rows = int64_t(a.seq) * (a.heads / a.kv_heads);
  if (rows <= 16) return false;
  const int64_t each = AttendRangeSteps(a, 16, 32) * 32 * a.kv_heads;
  return (rows + 15) / 16 * 16 >= (pairs + each - 1) / each;
}
// Many rows (attend_prompt.hip). load: the bytes that a thread may load at once from keys and values.
void LaunchAttendPromptQ8(const AttendArgs& a, const Q8Cache& c, int load, hipStream_t stream);
void LaunchAttendPromptF32(const AttendArgs& a, const float* k, const float* v, int load, hipStream_t stream);

// kN floats of a query row from dim d on, 0 past the row. vec: whole 16-byte pieces (a.dim % 4 == 0).
template <int kN>
__device__ __forceinline__ void LoadQuery(const AttendArgs& a, const float* q, int d, bool vec, float (&x)[kN]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      const f4 y = d + 4 * i < a.dim ? *reinterpret_cast<const f4*>(q + d + 4 * i) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < kN; ++e) x[e] = d + e < a.dim ? q[d + e] : 0.f;
  }
}
__device__ __forceinline__ bool QueryVec(const AttendArgs& a) {  // uniform
  return a.dim % 4 == 0 && a.q_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
}

// A part of a row's keys leaves (m, l, o): its reference, the sum of its weights, and the sum o of weight *
// value. Where that sum may pass the largest float (its quotient does not) it is held times 2^-64, and l is
// negative as a sign of it.
constexpr int32_t kFarShift = 64;
constexpr float kFarDown = 0x1p-64f, kFarUp = 0x1p64f;

// The results of a workgroup's waves for kRows rows meet in LDS. Wave w serves head w % heads of the
// workgroup's `heads` key heads and has every (waves / heads)-th step of the key range: each row's joined
// (m, l, sum) goes to `partial`, or with one key range the quotient to the output.
template <int DP, int kWaves, int kRows>
struct WaveParts {
  float o[kWaves][kRows][DP + 4];
  float m[kWaves][kRows];
  float l[kWaves][kRows];
  __device__ __forceinline__ void Join(const AttendArgs& a, int32_t kv0, int32_t heads, int32_t group, int32_t r0,
                                       int32_t rows, int32_t split, int32_t splits, const AttendPartial& partial) const {
    const bool vec = a.dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
    const int32_t n = min(kRows, rows - r0);
    const int32_t waves = static_cast<int32_t>(blockDim.x) / 64;
    for (int32_t item = threadIdx.x; item < heads * n * (DP / 4); item += blockDim.x) {
      const int32_t hr = item / (DP / 4);
      const int32_t d = item % (DP / 4) * 4;
      const int32_t h = hr / n;
      const int32_t rl = hr - h * n;
      if (d >= a.dim) continue;
      float big = -INFINITY;
      for (int32_t w = h; w < waves; w += heads) big = fmaxf(big, m[w][rl]);
      const float base = big == -INFINITY ? 0.f : big;
      float total = 0.f, low = 0.f;
      f4 x = f4{0.f, 0.f, 0.f, 0.f};
      for (int32_t w = h; w < waves; w += heads) {
        const float wt = __builtin_amdgcn_exp2f(m[w][rl] - base);
        low = fminf(low, l[w][rl]);
        total += wt * l[w][rl];
        x += wt * *reinterpret_cast<const f4*>(&o[w][rl][d]);
      }
      float up = 1.f;
      if (low < 0.f) {  // some parts are held times 2^-64: the sum is then too, unless they count for little
        float most = 0.f;
        for (int32_t w = h; w < waves; w += heads)
          if (l[w][rl] < 0.f) most = fmaxf(most, __builtin_amdgcn_exp2f(m[w][rl] - base));
        const bool far = most >= 0x1p-60f;
        total = 0.f;
        x = f4{0.f, 0.f, 0.f, 0.f};
        for (int32_t w = h; w < waves; w += heads) {
          const float wt = __builtin_amdgcn_exp2f(m[w][rl] - base);
          const bool held = l[w][rl] < 0.f;
          total += wt * fabsf(l[w][rl]);
          x += wt * (held == far ? 1.f : far ? kFarDown : kFarUp) * *reinterpret_cast<const f4*>(&o[w][rl][d]);
        }
        if (far) up = kFarUp;
      }
      const int32_t s = (r0 + rl) / group;
      const int64_t out_row = static_cast<int64_t>(s) * a.heads + (kv0 + h) * group + (r0 + rl - s * group);
      if (splits > 1) {
        const int64_t at = out_row * splits + split;
        if (d == 0) {
          partial.ml[2 * at] = big;
          partial.ml[2 * at + 1] = up == 1.f ? total : -total;
        }
        *reinterpret_cast<f4*>(partial.o + at * PartialDims(a.dim) + d) = x;
      } else {
        float* dst = a.out + out_row * a.dim + d;
        const f4 y = f4{__fdiv_rn(x[0], total), __fdiv_rn(x[1], total), __fdiv_rn(x[2], total), __fdiv_rn(x[3], total)} * up;
        if (vec) {
          *reinterpret_cast<f4*>(dst) = y;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < a.dim) dst[e] = y[e];
        }
      }
    }
  }
};

// Joins the key ranges of each row into the output (attention_q8.hip).
void LaunchAttendJoin(const AttendArgs& a, const AttendPartial& partial, int32_t splits, hipStream_t stream);

}  // namespace accel_hip
