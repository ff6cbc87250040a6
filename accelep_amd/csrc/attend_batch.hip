// Attention of a batch of requests, over the pages of a cache or over packed prompts.
#include "attend_common.h"

namespace accel_hip {
namespace {

// A wave a row and head: 64 keys at a time, a key a lane for the scores and some dims a lane for the sums.
__global__ __launch_bounds__(64) void AttendBatchKernel(BatchAttendArgs a) {
  __shared__ float query[256];
  const int lane = threadIdx.x;
  const int32_t row = static_cast<int32_t>(blockIdx.x / static_cast<uint32_t>(a.heads));
  const int32_t head = static_cast<int32_t>(blockIdx.x - static_cast<uint32_t>(row) * a.heads);
  const int32_t kv = head / (a.heads / a.kv_heads);
  int32_t low = -1, high = a.requests;  // the last request whose rows begin at or before this one
  while (high - low > 1) {
    const int32_t mid = low + (high - low) / 2;
    if (a.starts[mid] <= row) low = mid;
    else high = mid;
  }
  if (low < 0 || row >= a.starts[low + 1]) return;
  const int32_t r = low, start = max(a.starts[r], 0);
  const int32_t p = (a.paged ? min(max(a.seen[r], 0), a.width << a.page_shift) : 0) + row - start;
  const float* q = a.q + row * a.q_stride + static_cast<int64_t>(head) * a.dim;
  bool bad = false;
  for (int d = lane; d < a.dim; d += 64) {
    query[d] = q[d];
    bad = bad || !(fabsf(q[d]) < INFINITY);
  }
  __syncthreads();
  const int32_t first = a.window == kNoWindow ? 0 : max(0, p - a.window + 1);
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  const auto value = [&](const void* x, int64_t at) {
    return a.f16 ? static_cast<float>(static_cast<const _Float16*>(x)[at]) : static_cast<const float*>(x)[at];
  };
  for (int32_t t0 = first; t0 <= p; t0 += 64) {
    const int32_t t = min(t0 + lane, p);
    int64_t at = start + t;
    if (a.paged) {
      const int32_t q = t >> a.page_shift;
      const int32_t page = q < a.width ? a.table[static_cast<int64_t>(r) * a.width + q] : -1;
      const bool is = page >= 0 && page < a.pages;
      bad = bad || !is;
      at = is ? (static_cast<int64_t>(page) << a.page_shift) + (t & ((1 << a.page_shift) - 1)) : 0;
    }
    at = at * a.kv_stride + static_cast<int64_t>(kv) * a.dim;
    float s = 0.f;
    for (int d = 0; d < a.dim; ++d) {
      const float k = value(a.k, at + d), v = value(a.v, at + d);
      bad = bad || !(fabsf(k) < INFINITY) || !(fabsf(v) < INFINITY);
      s = fmaf(query[d], k, s);
    }
    s = t0 + lane <= p ? s * a.factor : -INFINITY;
    bad = bad || s == INFINITY;
    const float m_new = fmaxf(m, WaveButterfly(s, [](float x, float y) { return fmaxf(x, y); }));
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = exp2f(m - base), w = exp2f(s - base - 40.f);  // times 2^-40: sums of large values stay in range
    l = l * corr + WaveButterfly(w, [](float x, float y) { return x + y; });
    m = m_new;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= corr;
    for (int e = 0; e < 64; ++e) {
      const float we = __shfl(w, e);
      const int64_t ae = __shfl(at, e);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.dim) acc[i] = fmaf(we, value(a.v, ae + lane + 64 * i), acc[i]);
    }
  }
  bad = __any(bad);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.dim)
      a.out[(static_cast<int64_t>(row) * a.heads + head) * a.dim + lane + 64 * i] = bad ? NAN : __fdiv_rn(acc[i], l);
}

}  // namespace

void LaunchAttendBatch(const BatchAttendArgs& a, hipStream_t stream) {
  const int64_t units = int64_t(a.rows) * a.heads;
  hipLaunchKernelGGL(AttendBatchKernel, dim3(GridOf(units, 64, "Attention is too large")), dim3(64), 0, stream, a);
  Check(hipGetLastError(), "AttendBatchKernel launch");
}

}  // namespace accel_hip
