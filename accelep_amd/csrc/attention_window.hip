// Attention with a sliding window over an fp32 cache: for the row at p,
// out = sum_t e^(s_t - max s) v_t / sum_t e^(s_t - max s) over the keys it sees, t <= p with
// t > p - window or t < sinks, s_t = (q . k_t) / sqrt(dim), in one pass with a running maximum.
//
// The simplest form: one wave per (row, head), 64 keys at a time, a key a lane for the scores, then
// dims over the lanes for the weighted sum.
#include "attend_common.h"

namespace accel_hip {
namespace {

constexpr int kMaxDim = 256;

struct F32Rows {
  const float* k;
  const float* v;
  __device__ __forceinline__ float KScale(int64_t, int32_t, int32_t) const { return 1.f; }
  __device__ __forceinline__ float VScale(int64_t, int32_t, int32_t) const { return 1.f; }
  __device__ __forceinline__ float K(int64_t at) const { return k[at]; }
  __device__ __forceinline__ float V(int64_t at) const { return v[at]; }
};

template <typename Rows>
__global__ __launch_bounds__(64) void AttendSimpleKernel(AttendArgs a, Rows rows) {
  __shared__ float qs[kMaxDim];
  __shared__ float es[64];
  const int lane = threadIdx.x;
  const int32_t s = static_cast<int32_t>(blockIdx.x / static_cast<uint32_t>(a.heads));
  const int32_t h = static_cast<int32_t>(blockIdx.x) - s * a.heads;
  const int32_t kv = h / (a.heads / a.kv_heads);
  const int32_t p = a.position + s;
  const float* q = a.q + s * a.q_stride + static_cast<int64_t>(h) * a.dim;
  for (int d = lane; d < a.dim; d += 64) qs[d] = q[d];
  const float scale = __fdiv_rn(1.f, __fsqrt_rn(static_cast<float>(a.dim)));
  const int64_t stride = static_cast<int64_t>(a.kv_heads) * a.dim;
  const int32_t low = a.window == kNoWindow ? 0 : max(0, p - a.window + 1);
  const int32_t first = min(low, a.sinks);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[kMaxDim / 64] = {0.f, 0.f, 0.f, 0.f};
  for (int part = 0; part < 2; ++part) {
    const int32_t begin = part == 0 ? 0 : low, end = part == 0 ? first : p + 1;
    for (int32_t t0 = begin; t0 < end; t0 += 64) {
      const int32_t n = min(64, end - t0);
      const int64_t t = t0 + lane;
      float x = -INFINITY;
      if (lane < n) {
        float dot = 0.f;
        for (int d = 0; d < a.dim; ++d) dot += qs[d] * rows.K(t * stride + kv * a.dim + d);
        x = dot * (scale * rows.KScale(t, a.kv_heads, kv));
      }
      const float m_new = fmaxf(m, WaveButterfly(x, [](float u, float w) { return fmaxf(u, w); }));
      const float corr = m == m_new ? 1.f : expf(m - m_new);
      const float e = lane < n ? expf(x - m_new) : 0.f;
      l = l * corr + WaveButterfly(e, [](float u, float w) { return u + w; });
      m = m_new;
      es[lane] = lane < n ? e * rows.VScale(t, a.kv_heads, kv) : 0.f;
      __syncthreads();
      for (int i = 0; i < kMaxDim / 64; ++i) {
        const int d = lane + 64 * i;
        acc[i] *= corr;
        if (d < a.dim)
          for (int j = 0; j < n; ++j) acc[i] += es[j] * rows.V((t0 + j) * stride + kv * a.dim + d);
      }
      __syncthreads();
    }
  }
  for (int i = 0; i < kMaxDim / 64; ++i)
    if (lane + 64 * i < a.dim)
      a.out[(static_cast<int64_t>(s) * a.heads + h) * a.dim + lane + 64 * i] = __fdiv_rn(acc[i], l);
}

}  // namespace

void LaunchAttentionWindow(const AttendArgs& a, const float* k, const float* v, hipStream_t stream) {
  if (int64_t(a.seq) * (a.heads / a.kv_heads) > 64) {
    const bool vec = a.dim % 4 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0;
    LaunchAttendPromptF32(a, k, v, vec ? 16 : 4, stream);
    return;
  }
  hipLaunchKernelGGL(AttendSimpleKernel<F32Rows>, dim3(static_cast<uint32_t>(a.seq) * a.heads), dim3(64), 0, stream, a,
                     F32Rows{k, v});
  Check(hipGetLastError(), "AttendSimpleKernel launch");
}

}  // namespace accel_hip
