// The 8-bit KV cache, written and read back: codes int8 with one fp32 scale for each block of tokens
// and head, value = code * scale.
//
// Append: each touched (block, head, plane) is one unit of one wave, or of one workgroup where it is
// large. A unit holds its new rows in registers, takes their largest magnitude, forms the scale
// (amax / 127, or the stored one where that is larger and the block has older rows), and writes the codes:
// one pass over the rows. Older rows of the block are only touched when the scale grows.
//
// Bound: the bytes, 5 a value each way. 4095 rows of 8 heads of 128: append 11.0 us, 42 MB at 3.8 TB/s
// (the loads of a unit, then its largest, then its stores: a unit's phases follow one another, and a
// reduction stands between); 32768 rows read back 59 us, 336 MB at 5.7 TB/s. One row: 3.7 and 2.2 us,
// launch and two dependent round trips.
#include <algorithm>

#include "device_common.h"

namespace accel_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kHeld = 8;  // items of a unit a thread holds in registers

// The integer nearest to the true quotient x / s (ties to even), |x| <= 127.5 s. x times the rounded
// reciprocal is off by 2^-17 at most, so its nearest integer is the quotient's unless it lies within
// 2^-16 of the middle between two (one wave in 64 has such a value). There the remainder x - r s tells,
// since the fma forms it with one rounding and near s / 2, where it matters, without any (x and r s are
// multiples of half an ulp of s there). A scale below 2^-126 is itself rounded to few bits, so that its
// codes may pass 127: they stay there.
struct Coder {
  float s, half, inv, pre;
  __device__ __forceinline__ explicit Coder(float scale) {
    pre = scale < 0x1p-100f ? 0x1p100f : 1.f;  // keeps the reciprocal of a small scale finite
    s = scale * pre;
    half = 0.5f * s;
    inv = scale > 0.f ? __fdiv_rn(1.f, s) : 0.f;  // no scale, or NaN: every code is 0
  }
  __device__ __forceinline__ int32_t Exact(float x0) const {
    const float x = x0 * pre;
    const float r = rintf(x * inv);
    const float e = fmaf(-r, s, x);
    const float ae = fabsf(e);
    const int32_t n = static_cast<int32_t>(r);
    const bool off = ae > half || (ae == half && (n & 1) != 0);
    return min(max(n + (off && inv != 0.f ? (e < 0.f ? -1 : 1) : 0), -127), 127);
  }
  // The codes of x[0 .. kN) in the bytes of a word. 3 * 2^22 + r holds r in its low bits.
  template <int kN>
  __device__ __forceinline__ uint32_t Word(const float (&x0)[4]) const {
    constexpr float kMagic = 12582912.f;
    uint32_t bits[4] = {0, 0, 0, 0};
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float x = x0[e] * pre;
      const float m = fmaf(x, inv, kMagic);
      bits[e] = __float_as_uint(m);
      off = fmaxf(off, fabsf(fmaf(x, inv, kMagic - m)));
    }
    if (__any(!(off < 0.5f - 0x1p-16f)) || !(inv > 0.f) || pre != 1.f) {
#pragma unroll
      for (int e = 0; e < kN; ++e) bits[e] = static_cast<uint32_t>(Exact(x0[e]));
    }
    const uint32_t low = __builtin_amdgcn_perm(bits[1], bits[0], 0x0c0c0400u);
    const uint32_t high = __builtin_amdgcn_perm(bits[3], bits[2], 0x04000c0cu);
    return low | high;
  }
};

struct AppendArgs {
  const float* src[2];
  Q8Plane plane[2];
  int64_t row_stride;
  int32_t kv_heads, dim, block_shift;
  int32_t seq, position;
  uint32_t units;
};

__device__ __forceinline__ uint32_t MagnitudeBits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// kVec: items of 4 dims, otherwise of one. kWaves: the waves of a unit.
template <bool kVec, int kWaves>
__global__ __launch_bounds__(kThreads) void AppendQ8Kernel(AppendArgs a) {
  constexpr int kLanes = 64 * kWaves;
  constexpr int kUnits = kThreads / kLanes;  // of a workgroup
  constexpr int kDims = kVec ? 4 : 1;
  __shared__ uint32_t red[4];
  __shared__ float shared_old;
  const int lane = threadIdx.x % kLanes;
  const uint32_t unit = blockIdx.x * kUnits + threadIdx.x / kLanes;
  if (unit >= a.units) return;  // whole units: uniform over a unit's waves
  const int pl = static_cast<int>(unit & 1);
  const uint32_t bh = unit >> 1;
  const int32_t block = static_cast<int32_t>(bh / static_cast<uint32_t>(a.kv_heads));
  const int32_t head = static_cast<int32_t>(bh) - block * a.kv_heads;
  const int32_t begin = ((a.position >> a.block_shift) + block) << a.block_shift;  // the block's first row
  const int32_t lo = max(a.position, begin);
  const int64_t block_end = static_cast<int64_t>(begin) + (1 << a.block_shift);
  const int32_t hi = static_cast<int32_t>(min(static_cast<int64_t>(a.position) + a.seq, block_end));
  const int32_t per_row = a.dim / kDims;
  const int32_t items = (hi - lo) * per_row;
  const float* src = a.src[pl] + static_cast<int64_t>(lo - a.position) * a.row_stride + static_cast<int64_t>(head) * a.dim;
  const int64_t code_row = static_cast<int64_t>(a.kv_heads) * a.dim;
  int8_t* codes = a.plane[pl].code + static_cast<int64_t>(head) * a.dim;
  float* scale = a.plane[pl].scale + static_cast<int64_t>(begin >> a.block_shift) * a.kv_heads + head;

  const auto load = [&](int32_t item) {
    const int32_t r = static_cast<int32_t>(static_cast<uint32_t>(item) / static_cast<uint32_t>(per_row));
    const float* p = src + r * a.row_stride + (item - r * per_row) * kDims;
    if (kVec) return *reinterpret_cast<const float4*>(p);
    return make_float4(*p, 0.f, 0.f, 0.f);
  };
  const auto magnitude = [&](const float4& x) {
    return max(max(MagnitudeBits(x.x), MagnitudeBits(x.y)), max(MagnitudeBits(x.z), MagnitudeBits(x.w)));
  };
  const bool held = items <= kLanes * kHeld;  // uniform over the unit
  float4 x[kHeld];
  uint32_t top = 0;
  if (held) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      x[i] = lane + i * kLanes < items ? load(lane + i * kLanes) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float old = 0.f;
  if (lo > begin && (kWaves == 1 || lane == 0)) old = *scale;
  if (held) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top = max(top, magnitude(x[i]));
  } else {
    for (int32_t item = lane; item < items; item += kLanes) top = max(top, magnitude(load(item)));
  }
  top = WaveButterfly(top, [](uint32_t p, uint32_t q) { return max(p, q); });
  if (kWaves > 1) {
    if ((lane & 63) == 0) red[lane >> 6] = top;
    if (lane == 0) shared_old = old;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = max(top, red[w]);
    old = shared_old;
  }
  const float need = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(top), 127.f);
  // A NaN on either side stays one.
  const float now = old != old ? old : (need != need || need > old ? need : old);
  const Coder code(now);

  if (lo > begin && now > old) {  // uniform over the unit
    const int32_t kept = (lo - begin) * per_row;
    const double grown_from = static_cast<double>(old), to = static_cast<double>(now);
    for (int32_t item = lane; item < kept; item += kLanes) {
      const int32_t r = static_cast<int32_t>(static_cast<uint32_t>(item) / static_cast<uint32_t>(per_row));
      int8_t* p = codes + (begin + r) * code_row + (item - r * per_row) * kDims;
      const auto again = [&](int32_t c) { return static_cast<int32_t>(rint(c * grown_from / to)); };
      if (kVec) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
        uint32_t o = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o |= (static_cast<uint32_t>(again(static_cast<int8_t>(w >> (8 * e)))) & 255u) << (8 * e);
        *reinterpret_cast<uint32_t*>(p) = o;
      } else {
        *p = static_cast<int8_t>(again(*p));
      }
    }
  }
  if (lane == 0) *scale = now;
  const auto store = [&](int32_t item, const float4& v) {
    const int32_t r = static_cast<int32_t>(static_cast<uint32_t>(item) / static_cast<uint32_t>(per_row));
    int8_t* p = codes + (lo + r) * code_row + (item - r * per_row) * kDims;
    const float y[4] = {v.x, v.y, v.z, v.w};
    if (kVec) *reinterpret_cast<uint32_t*>(p) = code.Word<4>(y);
    else *p = static_cast<int8_t>(code.Word<1>(y));
  };
  if (held) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (lane + i * kLanes < items) store(lane + i * kLanes, x[i]);
  } else {
    for (int32_t item = lane; item < items; item += kLanes) store(item, load(item));
  }
}

struct ReadArgs {
  Q8Plane plane[2];
  float* out[2];
  int64_t first, items;  // items of one plane
  int32_t kv_heads, per_head, block_shift;
};

constexpr int kReadItems = 4;

// One item (4 dims, or one) a thread and round: a wave stores 1 KB in a row.
template <bool kVec>
__global__ __launch_bounds__(kThreads) void ReadQ8Kernel(ReadArgs a) {
  constexpr int kDims = kVec ? 4 : 1;
  const int pl = static_cast<int>(blockIdx.y);
  const uint32_t per_row = static_cast<uint32_t>(a.kv_heads * a.per_head);
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kThreads * kReadItems);
  const int64_t row0 = base / per_row;
  const uint32_t rem = static_cast<uint32_t>(base - row0 * per_row) + threadIdx.x;
  const int8_t* codes = a.plane[pl].code + a.first * per_row * kDims;
  float* out = a.out[pl];
  uint32_t w[kReadItems];
  float s[kReadItems];
#pragma unroll
  for (int u = 0; u < kReadItems; ++u) {
    const int64_t item = base + threadIdx.x + u * kThreads;
    if (item >= a.items) break;
    const uint32_t r = (rem + u * kThreads) / per_row;
    const uint32_t head = (rem + u * kThreads - r * per_row) / static_cast<uint32_t>(a.per_head);
    w[u] = kVec ? reinterpret_cast<const uint32_t*>(codes)[item] : static_cast<uint32_t>(static_cast<uint8_t>(codes[item]));
    s[u] = a.plane[pl].scale[((a.first + row0 + r) >> a.block_shift) * a.kv_heads + head];
  }
#pragma unroll
  for (int u = 0; u < kReadItems; ++u) {
    const int64_t item = base + threadIdx.x + u * kThreads;
    if (item >= a.items) break;
    if (kVec)
      reinterpret_cast<float4*>(out)[item] =
          make_float4(__fmul_rn(ByteToFloat(w[u], 0), s[u]), __fmul_rn(ByteToFloat(w[u], 1), s[u]),
                      __fmul_rn(ByteToFloat(w[u], 2), s[u]), __fmul_rn(ByteToFloat(w[u], 3), s[u]));
    else
      out[item] = __fmul_rn(ByteToFloat(w[u], 0), s[u]);
  }
}

bool AlignedTo(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

void LaunchAppendCacheQ8(const float* k, const float* v, const Q8Cache& cache, int64_t seq, int64_t position,
                         int64_t row_stride, hipStream_t stream) {
  AppendArgs a;
  a.src[0] = k;
  a.src[1] = v;
  a.plane[0] = cache.k;
  a.plane[1] = cache.v;
  a.row_stride = row_stride;
  a.kv_heads = cache.kv_heads;
  a.dim = cache.dim;
  a.block_shift = cache.block_shift;
  a.seq = static_cast<int32_t>(seq);
  a.position = static_cast<int32_t>(position);
  const int64_t blocks = ((position + seq - 1) >> cache.block_shift) - (position >> cache.block_shift) + 1;
  const int64_t units = blocks * cache.kv_heads * 2;
  constexpr int64_t kMostUnits = int64_t(1) << 23;  // a grid holds fewer than 2^32 threads
  if (units > kMostUnits && blocks > 1) {  // whole blocks at a time
    const int64_t first = std::max<int64_t>(1, kMostUnits / (cache.kv_heads * 2)) << cache.block_shift;
    const int64_t rows = first - (position & ((int64_t(1) << cache.block_shift) - 1));
    LaunchAppendCacheQ8(k, v, cache, rows, position, row_stride, stream);
    LaunchAppendCacheQ8(k + rows * row_stride, v + rows * row_stride, cache, seq - rows, position + rows, row_stride, stream);
    return;
  }
  a.units = static_cast<uint32_t>(units);
  const bool vec = AlignedTo(k, 16) && AlignedTo(v, 16) && row_stride % 4 == 0 && cache.dim % 4 == 0 &&
                   AlignedTo(cache.k.code, 4) && AlignedTo(cache.v.code, 4);
  // A unit that one wave holds in registers is one wave's; larger ones are a workgroup's, and so are all
  // where they are few (a block's older rows may have to be coded again).
  const int64_t rows = std::min<int64_t>(int64_t(1) << cache.block_shift, seq);
  const bool wide = rows * cache.dim > 64 * kHeld * (vec ? 4 : 1) ||
                    (units <= 256 && (int64_t(cache.dim) << cache.block_shift) > 2048);
  const dim3 grid(GridOf(wide ? units : (units + 3) / 4, kThreads, "AppendCache is too large")), block(kThreads);
  if (vec && wide) hipLaunchKernelGGL((AppendQ8Kernel<true, 4>), grid, block, 0, stream, a);
  else if (vec) hipLaunchKernelGGL((AppendQ8Kernel<true, 1>), grid, block, 0, stream, a);
  else if (wide) hipLaunchKernelGGL((AppendQ8Kernel<false, 4>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((AppendQ8Kernel<false, 1>), grid, block, 0, stream, a);
  Check(hipGetLastError(), "AppendQ8Kernel launch");
}

void LaunchReadCacheQ8(const Q8Cache& cache, int64_t first, int64_t count, float* k_out, float* v_out,
                       hipStream_t stream) {
  ReadArgs a;
  int planes = 0;
  bool vec = cache.dim % 4 == 0;
  const auto add = [&](const Q8Plane& plane, float* out) {
    if (out == nullptr) return;
    a.plane[planes] = plane;
    a.out[planes++] = out;
    vec = vec && AlignedTo(out, 16) && AlignedTo(plane.code, 4);
  };
  add(cache.k, k_out);
  add(cache.v, v_out);
  if (planes == 0 || count == 0) return;
  a.first = first;
  a.kv_heads = cache.kv_heads;
  a.per_head = vec ? cache.dim / 4 : cache.dim;
  a.block_shift = cache.block_shift;
  a.items = count * a.kv_heads * a.per_head;
  const int64_t grid_x = (a.items + kThreads * kReadItems - 1) / (kThreads * kReadItems);
  const dim3 grid(GridOf(grid_x, kThreads * planes, "the range is too large"), static_cast<uint32_t>(planes)), block(kThreads);
  if (vec) hipLaunchKernelGGL(ReadQ8Kernel<true>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(ReadQ8Kernel<false>, grid, block, 0, stream, a);
  Check(hipGetLastError(), "ReadQ8Kernel launch");
}

}  // namespace accel_hip
