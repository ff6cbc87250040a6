// The tables of a batch's step, from the lengths of its requests: first rows, pages for new tokens from a stack,
// positions and slots; and pages taken back. Whole numbers throughout.
//
// The first row of a request is the sum of the new tokens before it, and the pages that it takes are those
// behind the new pages before it: one scan of both over the requests, by one workgroup. A new page is
// begun by exactly one new row, the one at a multiple of the page, so each row finds its own page without the
// others: an old entry of the table, or an entry of the stack, which it also writes into the table.
//
// Bound: latency. 64 single tokens 5.1 us, of which a launch and a chain of lengths, two scans and a row's search, page
// and stores; 1000 requests with 21000 rows 9.3 us in two launches, of which 5.6 are the scan. Their bytes would
// take 0.1 us.
#include <algorithm>

#include "attend_split.h"
#include "device_common.h"

namespace accel_hip {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kHeldRequests = 2048;      // whose descriptions one workgroup keeps in LDS (32 KB)
constexpr int kSearchedRequests = 8191;  // whose starts a workgroup of the rows' launch does
constexpr int32_t kRefused = INT32_MIN;

// Page q (>= have) of a request is stack[top - q]; top is kRefused where it gets none.
struct RequestInfo {
  int32_t start, length, have, top;
};

// Sums over the workgroup's threads before this one, and over all.
struct Sums {
  int64_t rows, pages;
};
__device__ __forceinline__ Sums ScanThreads(Sums x, Sums* total, Sums* of_wave) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  Sums sum = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t rows = __shfl_up(sum.rows, off), pages = __shfl_up(sum.pages, off);
    if (lane >= off) {
      sum.rows += rows;
      sum.pages += pages;
    }
  }
  if (lane == 63) of_wave[wave] = sum;
  __syncthreads();
  Sums before{0, 0};
  *total = Sums{0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const Sums s = of_wave[w];
    if (w < wave) before = Sums{before.rows + s.rows, before.pages + s.pages};
    *total = Sums{total->rows + s.rows, total->pages + s.pages};
  }
  __syncthreads();
  return Sums{before.rows + sum.rows - x.rows, before.pages + sum.pages - x.pages};
}

__device__ __forceinline__ int64_t PagesOf(int64_t tokens, int32_t page_shift) {
  return (tokens + (int64_t(1) << page_shift) - 1) >> page_shift;
}

// The scan over the requests: everything but slots, positions and table entries. Returns the rows of all.
__device__ __forceinline__ int32_t ScanRequests(const BatchTablesArgs& a, RequestInfo* info) {
  __shared__ Sums of_wave[kWaves];
  __shared__ int32_t used_shared, refused_shared;
  if (threadIdx.x == 0) used_shared = refused_shared = 0;
  const int64_t left = min(max(a.state[0], 0), a.pages);
  Sums carry{0, 0};
  int64_t used = 0;
  int32_t refused = 0;
  for (int32_t r0 = 0; r0 < a.requests; r0 += kThreads) {
    const int32_t r = r0 + threadIdx.x;
    const bool in = r < a.requests;
    const int64_t count = in ? min(max(a.counts[r], 0), a.rows) : 0;
    const int64_t length = in ? max(a.lengths[r], 0) : 0;
    Sums total;
    // Rows first: they say how many of the last request's tokens there is room for.
    const int64_t start = min(carry.rows + ScanThreads(Sums{count, 0}, &total, of_wave).rows, int64_t(a.rows));
    carry.rows += total.rows;
    const int64_t n = min(count, a.rows - start);
    const int64_t have = PagesOf(length, a.page_shift), need = PagesOf(length + n, a.page_shift);
    const bool fits = n == 0 || need <= a.width;
    const int64_t fresh = fits && n > 0 ? need - have : 0;
    const int64_t before = carry.pages + ScanThreads(Sums{0, fresh}, &total, of_wave).pages;
    carry.pages += total.pages;
    const bool served = fits && (fresh == 0 || before + fresh <= left);
    if (in) {
      a.starts[r] = static_cast<int32_t>(start);
      a.seen[r] = static_cast<int32_t>(length);
      a.lengths_after[r] = static_cast<int32_t>(served ? length + n : length);
      info[r] = RequestInfo{static_cast<int32_t>(start), static_cast<int32_t>(length), static_cast<int32_t>(have),
                            served ? static_cast<int32_t>(left - 1 - before + have) : kRefused};
      if (served && fresh > 0) used = max(used, before + fresh);
      if (!served) ++refused;
    }
  }
  if (used > 0) atomicMax(&used_shared, static_cast<int32_t>(used));
  if (refused > 0) atomicAdd(&refused_shared, refused);
  const int32_t rows = static_cast<int32_t>(min(carry.rows, int64_t(a.rows)));
  __syncthreads();
  if (threadIdx.x == 0) {
    a.starts[a.requests] = rows;
    a.state_after[0] = static_cast<int32_t>(left - used_shared);
    a.state_after[1] = refused_shared;
  }
  return rows;
}

// The last request whose rows begin at or before row i: of those with the same start the one that has rows.
template <typename At>
__device__ __forceinline__ int32_t RequestOf(int32_t i, int32_t requests, At at) {
  int32_t low = 0, high = requests;  // start(low) <= i < start(high)
  while (high - low > 1) {
    const int32_t mid = low + (high - low) / 2;
    if (at(mid) <= i) low = mid;
    else high = mid;
  }
  return low;
}

__device__ __forceinline__ void PlaceRow(const BatchTablesArgs& a, int32_t i, int32_t r, const RequestInfo& x) {
  const int64_t position = static_cast<int64_t>(x.length) + (i - x.start);
  const int32_t mask = (1 << a.page_shift) - 1;
  const int64_t q = position >> a.page_shift;
  int32_t* entry = a.table + static_cast<int64_t>(r) * a.width + q;
  int64_t slot = -1;
  if (x.top != kRefused) {
    const int32_t page = q < x.have ? *entry : a.stack[x.top - q];
    if (page >= 0 && page < a.pages) slot = (static_cast<int64_t>(page) << a.page_shift) + (position & mask);
    if (q >= x.have && (position & mask) == 0) *entry = page;
  } else if (q >= x.have && q < a.width && (position & mask) == 0) {
    *entry = -1;
  }
  a.slots[i] = static_cast<int32_t>(slot);
  a.positions[i] = static_cast<int32_t>(min(position, int64_t(INT32_MAX)));
}
__device__ __forceinline__ void PlacePadding(const BatchTablesArgs& a, int32_t i) {
  a.slots[i] = -1;
  a.positions[i] = 0;
}

// One workgroup for all of it.
__global__ __launch_bounds__(kThreads) void BatchTablesKernel(BatchTablesArgs a) {
  __shared__ RequestInfo info[kHeldRequests];
  const int32_t rows = ScanRequests(a, info);
  for (int32_t i = threadIdx.x; i < a.rows; i += kThreads) {
    if (i >= rows) {
      PlacePadding(a, i);
    } else {
      const int32_t r = RequestOf(i, a.requests, [&](int32_t s) { return info[s].start; });
      PlaceRow(a, i, r, info[r]);
    }
  }
}

__global__ __launch_bounds__(kThreads) void BatchScanKernel(BatchTablesArgs a, RequestInfo* info) { ScanRequests(a, info); }

__global__ __launch_bounds__(kThreads) void BatchRowsKernel(BatchTablesArgs a, const RequestInfo* info) {
  __shared__ int32_t starts[kSearchedRequests];
  const bool held = a.requests <= kSearchedRequests;
  if (held)
    for (int32_t r = threadIdx.x; r < a.requests; r += kThreads) starts[r] = a.starts[r];
  __syncthreads();
  const int32_t rows = a.starts[a.requests];
  for (int64_t i64 = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i64 < a.rows;
       i64 += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int32_t i = static_cast<int32_t>(i64);
    if (i >= rows) {
      PlacePadding(a, i);
      continue;
    }
    const int32_t r = held ? RequestOf(i, a.requests, [&](int32_t s) { return starts[s]; })
                           : RequestOf(i, a.requests, [&](int32_t s) { return a.starts[s]; });
    PlaceRow(a, i, r, info[r]);
  }
}

// A wave a request, twice: its pages are counted, the counts summed over the requests, and the pages put where the
// sums say. Between, the chunk's counts are in LDS.
// Bound: latency. Each of the 16 waves goes from request to request, and waits for its lengths and for 64 entries at a
// time. Requests of 500 .. 4000 tokens, pages of 64: 1000 of which none is cut 29 us, ten of them 30, all by up to
// 4 tokens 38, all of them ended 102 (pages of 16: 187); 64 requests over pages of 16 4.7, by up to 4 tokens 6.5, all
// ended 16. The bytes of the largest would take 0.1 us.
__global__ __launch_bounds__(kThreads) void ReleasePagesKernel(ReleasePagesArgs a) {
  __shared__ Sums of_wave[kWaves];
  __shared__ int32_t count[kThreads];
  __shared__ int64_t before[kThreads];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int64_t left = min(max(a.state[0], 0), a.pages);
  int64_t carry = 0;
  // The entries [first, last) of request r that are given back; empty where it is not cut.
  const auto range = [&](int32_t r, int32_t* first, int32_t* last) {
    const int64_t keep = max(a.keep[r], 0), length = max(a.lengths[r], 0);
    *last = static_cast<int32_t>(min(PagesOf(length, a.page_shift), int64_t(a.width)));
    *first = static_cast<int32_t>(min(PagesOf(min(keep, length), a.page_shift), int64_t(*last)));
  };
  for (int32_t r0 = 0; r0 < a.requests; r0 += kThreads) {
    const int32_t n = min(kThreads, a.requests - r0);
    for (int32_t i = wave; i < n; i += kWaves) {
      int32_t first, last, sum = 0;
      range(r0 + i, &first, &last);
      const int32_t* row = a.table + static_cast<int64_t>(r0 + i) * a.width;
      for (int32_t q = first; q < last; q += 64) {
        const int32_t page = q + lane < last ? row[q + lane] : -1;
        sum += __popcll(__ballot(page >= 0 && page < a.pages));
      }
      if (lane == 0) count[i] = sum;
    }
    __syncthreads();
    Sums total;
    before[threadIdx.x] =
        carry + ScanThreads(Sums{0, static_cast<int>(threadIdx.x) < n ? count[threadIdx.x] : 0}, &total, of_wave).pages;
    carry += total.pages;
    __syncthreads();
    for (int32_t i = wave; i < n; i += kWaves) {
      int32_t first, last;
      range(r0 + i, &first, &last);
      int32_t* row = a.table + static_cast<int64_t>(r0 + i) * a.width;
      int64_t to = left + before[i];
      for (int32_t q = first; q < last; q += 64) {
        const int32_t page = q + lane < last ? row[q + lane] : -1;
        const bool valid = page >= 0 && page < a.pages;
        const uint64_t all = __ballot(valid);
        const int64_t at = to + __popcll(all & ((uint64_t(1) << lane) - 1));
        if (valid && at < a.pages) a.stack[at] = page;
        if (q + lane < last) row[q + lane] = -1;
        to += __popcll(all);
      }
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < n) {
      const int32_t r = r0 + threadIdx.x, keep = max(a.keep[r], 0);
      if (keep < a.lengths[r]) a.lengths[r] = keep;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) a.state[0] = static_cast<int32_t>(min(left + carry, int64_t(a.pages)));
}

// Rows from which on a second launch with many workgroups is worth its start: 64 requests with 2048 rows take 8.0 us in
// one and 9.7 in two launches, with 4096 9.6 and 9.9, with 8192 12.8 and 10.3.
constexpr int32_t kOneGroupRows = 4096;

}  // namespace

void LaunchBatchTables(const BatchTablesArgs& a, hipStream_t stream) {
  if (a.requests <= kHeldRequests && a.rows <= kOneGroupRows) {
    hipLaunchKernelGGL(BatchTablesKernel, dim3(1), dim3(kThreads), 0, stream, a);
    Check(hipGetLastError(), "BatchTablesKernel launch");
    return;
  }
  // Between the two launches the requests' descriptions lie in the attention's scratch, whose lock keeps other
  // threads' calls and replays from coming between.
  std::lock_guard<std::mutex> held(AttendPartsMutex());
  RequestInfo* info = static_cast<RequestInfo*>(Temp(kTempAttend, sizeof(RequestInfo) * std::max(a.requests, 1)));
  hipLaunchKernelGGL(BatchScanKernel, dim3(1), dim3(kThreads), 0, stream, a, info);
  Check(hipGetLastError(), "BatchScanKernel launch");
  if (a.rows == 0) return;
  const int32_t groups = std::min((a.rows + kThreads - 1) / kThreads, 2048);
  hipLaunchKernelGGL(BatchRowsKernel, dim3(groups), dim3(kThreads), 0, stream, a, info);
  Check(hipGetLastError(), "BatchRowsKernel launch");
}

void LaunchReleasePages(const ReleasePagesArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(ReleasePagesKernel, dim3(1), dim3(kThreads), 0, stream, a);
  Check(hipGetLastError(), "ReleasePagesKernel launch");
}

}  // namespace accel_hip
