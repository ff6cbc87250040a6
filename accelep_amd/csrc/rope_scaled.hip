// Rotary positions with given frequencies: y0 = m (x0 cos a - x1 sin a), y1 = m (x1 cos a + x0 sin a)
// for pair i of a head at position p, a = p * f_i, m the magnitude; pairs are dims (i, i + r/2) or
// (2i, 2i + 1), dims from r on come out unchanged.
//
// The angle is formed in fp64, in half turns reduced to [-1, 1]. The product of position and frequency and the
// change to half turns each round by 2^-53 of it: within 2^-24 radians together up to 2^27 radians, within 2^-20
// at 2^31. What the reduced angle's rounding to fp32 leaves over goes back in to first order
// (sin(a + d) = sin a + d cos a); cos and sin themselves are fp32. One workgroup per row (and part of its
// heads): its pairs' cos and sin are computed once into LDS, then the heads stream through (their first loads
// are on the way while the angles are formed).
//
// Bound: the bytes of the values, 8 each in a pass (4096 rows of 40 heads of 128, half of each turned:
// 168 MB in 35 us, 4.8 TB/s, nearly a copy's rate); a single row is a launch and one dependent load (2.3 us).
#include <algorithm>

#include "device_common.h"

namespace accel_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;  // 16-byte items of a thread in flight
constexpr int kMaxPairs = 128;

struct Turn {
  float c, s;
};

__device__ __forceinline__ Turn TurnOf(double radians, float magnitude) {
  double x = radians * 0.31830988618379067154;  // half turns
  x = x - 2.0 * rint(x * 0.5);
  const float hi = static_cast<float>(x);
  const float d = static_cast<float>((x - static_cast<double>(hi)) * 3.14159265358979323846);
  float s, c;
  sincospif(hi, &s, &c);
  Turn t;
  t.c = (c - d * s) * magnitude;
  t.s = (s + d * c) * magnitude;
  return t;
}

// A head's items: its pairs (kVec: 4 of them in the half layout, 2 in the interleaved one), then, where
// the output is not the input, its other dims (kVec: 4).
template <bool kHalf, bool kVec>
__global__ __launch_bounds__(kThreads) void RopeScaledKernel(RopeScaledArgs a, int32_t heads_per, uint32_t pair_items,
                                                             uint32_t items) {
  __shared__ Turn turns[kMaxPairs];
  const int32_t h0 = static_cast<int32_t>(blockIdx.y) * heads_per;
  const uint32_t count = static_cast<uint32_t>(min(heads_per, a.heads - h0)) * items;
  const int pairs = a.rotary / 2;
  for (int64_t s = blockIdx.x; s < a.seq; s += gridDim.x) {
    const float* src = a.states + s * a.row_stride + static_cast<int64_t>(h0) * a.dim;
    float* dst = a.out + s * a.row_stride + static_cast<int64_t>(h0) * a.dim;
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
      const double p = static_cast<double>(a.position + (a.positions != nullptr ? static_cast<int64_t>(a.positions[s]) : s));
      turns[i] = TurnOf(p * a.frequencies[i], a.magnitude);
    }
    const auto place = [&](uint32_t item, int32_t* i) {  // the item's head, and in it the first dim or pair
      const uint32_t h = item / items;
      *i = static_cast<int32_t>(item - h * items);
      return static_cast<int32_t>(h) * a.dim;
    };
    for (uint32_t begin = 0; begin < count; begin += blockDim.x * kItems) {  // uniform
      const uint32_t base = begin + threadIdx.x;
      float4 x[kItems], y[kItems];
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const uint32_t item = base + u * blockDim.x;
        if (item >= count) break;
        int32_t i;
        const float* row = src + place(item, &i);
        const bool turn = i < static_cast<int32_t>(pair_items);
        const int32_t pass = a.rotary + (i - static_cast<int32_t>(pair_items)) * (kVec ? 4 : 1);
        if (kVec) {
          x[u] = *reinterpret_cast<const float4*>(row + (turn ? 4 * i : pass));
          if (kHalf && turn) y[u] = *reinterpret_cast<const float4*>(row + pairs + 4 * i);
        } else {
          x[u].x = row[turn ? (kHalf ? i : 2 * i) : pass];
          if (turn) y[u].x = row[kHalf ? i + pairs : 2 * i + 1];
        }
      }
      if (begin == 0) __syncthreads();  // the turns are there; the first items are on their way
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const uint32_t item = base + u * blockDim.x;
        if (item >= count) break;
        int32_t i;
        float* row = dst + place(item, &i);
        if (i >= static_cast<int32_t>(pair_items)) {
          const int32_t pass = a.rotary + (i - static_cast<int32_t>(pair_items)) * (kVec ? 4 : 1);
          if (kVec) *reinterpret_cast<float4*>(row + pass) = x[u];
          else row[pass] = x[u].x;
        } else if (kVec && kHalf) {
          const float* x0 = &x[u].x;
          const float* x1 = &y[u].x;
          float4 o0, o1;
          float* q0 = &o0.x;
          float* q1 = &o1.x;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const Turn t = turns[4 * i + e];
            q0[e] = x0[e] * t.c - x1[e] * t.s;
            q1[e] = x1[e] * t.c + x0[e] * t.s;
          }
          *reinterpret_cast<float4*>(row + 4 * i) = o0;
          *reinterpret_cast<float4*>(row + pairs + 4 * i) = o1;
        } else if (kVec) {
          const Turn t0 = turns[2 * i], t1 = turns[2 * i + 1];
          *reinterpret_cast<float4*>(row + 4 * i) =
              make_float4(x[u].x * t0.c - x[u].y * t0.s, x[u].y * t0.c + x[u].x * t0.s, x[u].z * t1.c - x[u].w * t1.s,
                          x[u].w * t1.c + x[u].z * t1.s);
        } else {
          const Turn t = turns[i];
          row[kHalf ? i : 2 * i] = x[u].x * t.c - y[u].x * t.s;
          row[kHalf ? i + pairs : 2 * i + 1] = y[u].x * t.c + x[u].x * t.s;
        }
      }
    }
    __syncthreads();  // the turns are read
  }
}

}  // namespace

void LaunchRopeScaled(const RopeScaledArgs& a, hipStream_t stream) {
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool half = a.layout == ACCEL_HIP_ROPE_HALF;
  const bool vec = aligned(a.states) && aligned(a.out) && a.row_stride % 4 == 0 && a.dim % 4 == 0 &&
                   a.rotary % (half ? 8 : 4) == 0;
  const int32_t pass = a.states == a.out ? 0 : a.dim - a.rotary;
  const int32_t pair_items = vec ? (half ? a.rotary / 8 : a.rotary / 4) : a.rotary / 2;
  const int32_t items = pair_items + (vec ? pass / 4 : pass);
  if (items == 0) return;
  // At most kItems items a thread, over equal parts of the heads.
  const int64_t per = std::max<int64_t>(1, kThreads * kItems / items);
  const int64_t parts = (a.heads + per - 1) / per;
  const int32_t heads_per = static_cast<int32_t>((a.heads + parts - 1) / parts);
  const int64_t grid_y = (a.heads + heads_per - 1) / heads_per;
  if (grid_y > 65535) Fail(ACCEL_HIP_INVALID_ARGUMENT, "Rope is too large");
  const int threads = static_cast<int64_t>(heads_per) * items <= 128 ? 64 : kThreads;
  // More rows than this take turns in a workgroup (a grid holds fewer than 2^32 threads).
  const int64_t rows = std::min<int64_t>(a.seq, (int64_t(1) << 23) / grid_y);
  const dim3 grid(static_cast<uint32_t>(rows), static_cast<uint32_t>(grid_y)), block(threads);
#define ACCEL_ROPE(H, V)                                                                                     \
  hipLaunchKernelGGL((RopeScaledKernel<H, V>), grid, block, 0, stream, a, heads_per, \
                     static_cast<uint32_t>(pair_items), static_cast<uint32_t>(items))
  if (half) {
    if (vec) ACCEL_ROPE(true, true);
    else ACCEL_ROPE(true, false);
  } else {
    if (vec) ACCEL_ROPE(false, true);
    else ACCEL_ROPE(false, false);
  }
#undef ACCEL_ROPE
  Check(hipGetLastError(), "RopeScaledKernel launch");
}

}  // namespace accel_hip
