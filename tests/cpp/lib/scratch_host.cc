// The library's process state (accelep_amd/csrc/context.cc) and the division of key ranges (attend_split.cc) over a HIP runtime of host memory, for the CPU
// tests of what happens when an allocation fails. TEST INFRASTRUCTURE ONLY: the functions below stand in for
// the HIP runtime's and the kernel files'. A failed call leaves its error for hipGetLastError, as HIP does.
#include <hip/hip_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>

#include "attend_split.h"
#include "common.h"
#include "host_util.h"

#define HOST_API extern "C" __attribute__((visibility("default")))

namespace {
std::mutex g_mu;
std::map<void*, size_t> g_blocks;
size_t g_refused_from = SIZE_MAX;  // allocations of this many bytes and more fail
bool g_capturing = false;
thread_local hipError_t g_last = hipSuccess;

hipError_t Done(hipError_t e) {
  if (e != hipSuccess) g_last = e;
  return e;
}
}  // namespace

extern "C" {
hipError_t hipGetLastError() {
  const hipError_t e = g_last;
  g_last = hipSuccess;
  return e;
}
const char* hipGetErrorString(hipError_t) { return "an error"; }
hipError_t hipGetDeviceCount(int* count) {
  *count = 1;
  return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
  std::memset(p, 0, sizeof(*p));
  std::strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipMalloc(void** ptr, size_t bytes) {
  std::lock_guard<std::mutex> lock(g_mu);
  if (bytes >= g_refused_from) {
    *ptr = nullptr;
    return Done(hipErrorOutOfMemory);
  }
  *ptr = std::malloc(bytes);
  g_blocks[*ptr] = bytes;
  return hipSuccess;
}
hipError_t hipFree(void* ptr) {
  std::lock_guard<std::mutex> lock(g_mu);
  if (g_blocks.erase(ptr) == 0) return Done(hipErrorInvalidValue);
  std::free(ptr);
  return hipSuccess;
}
hipError_t hipMemsetAsync(void* ptr, int value, size_t bytes, hipStream_t) {
  std::memset(ptr, value, bytes);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void* to, const void* from, size_t bytes, hipMemcpyKind, hipStream_t) {
  std::memcpy(to, from, bytes);
  return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
  *s = nullptr;
  return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* status) {
  *status = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipStreamBeginCapture(hipStream_t, hipStreamCaptureMode) {
  g_capturing = true;
  return hipSuccess;
}
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* graph) {
  g_capturing = false;
  *graph = nullptr;
  return hipSuccess;
}
hipError_t hipGraphInstantiate(hipGraphExec_t* exec, hipGraph_t, hipGraphNode_t*, char*, size_t) {
  *exec = nullptr;
  return hipSuccess;
}
hipError_t hipGraphDestroy(hipGraph_t) { return hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t) { return hipSuccess; }
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) {
  *e = nullptr;
  return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventRecordWithFlags(hipEvent_t, hipStream_t, unsigned) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) {
  *ms = 0;
  return hipSuccess;
}
}

namespace accel_hip {
void LaunchFill(float* dst, float value, int64_t count, hipStream_t) {
  for (int64_t i = 0; i < count; ++i) dst[i] = value;
}
void InitNoAllocScratch(const Context&) {}
void BeginStagedUses() {}
StagedUses EndStagedUses() { return {}; }
bool StagedUsesLive(const StagedUses&) { return true; }
void NoteDeviceWrite(const void*, size_t) {}
void DropStagedForAllocation(uint64_t) {}
}  // namespace accel_hip

using namespace accel_hip;

HOST_API void scratch_host_refuse_from(size_t bytes) { g_refused_from = bytes; }
HOST_API int scratch_host_last_error() { return static_cast<int>(hipGetLastError()); }
HOST_API uint64_t scratch_host_generation() { return Generation(); }
// The bytes of the block that `ptr` begins, 0 where none does.
HOST_API size_t scratch_host_block(void* ptr) {
  std::lock_guard<std::mutex> lock(g_mu);
  const auto it = g_blocks.find(ptr);
  return it == g_blocks.end() ? 0 : it->second;
}
HOST_API int scratch_host_temp(int slot, size_t bytes, void** out) {
  return Guard([&] { *out = Temp(static_cast<TempSlot>(slot), bytes); });
}
HOST_API int scratch_host_workspace(size_t bytes, void** out) {
  return Guard([&] { *out = Workspace(bytes); });
}
// The parts of key ranges, held by this thread until the release.
namespace {
AttendSplit g_held;
}
HOST_API int scratch_host_hold_parts() {
  return Guard([&] {
    AttendArgs a{};
    a.seq = a.heads = a.kv_heads = 1;
    a.dim = 64;
    g_held = SplitRange(a, 1, 8);
    if (g_held.count != 8) Fail(ACCEL_HIP_LOGIC_ERROR, "the range is whole");
  });
}
HOST_API void scratch_host_release_parts() { g_held = AttendSplit{}; }
// Into how many ranges an attention call of one row of `heads` heads of `dim` is cut.
HOST_API int scratch_host_split(int heads, int dim, int64_t most, int* count) {
  return Guard([&] {
    AttendArgs a{};
    a.seq = 1;
    a.heads = heads;
    a.kv_heads = 1;
    a.dim = dim;
    const AttendSplit split = SplitRange(a, 1, most);
    *count = split.count;
    const size_t bytes = static_cast<size_t>(split.count) * heads * (2 + PartialDims(dim)) * sizeof(float);
    if (split.count > 1 && scratch_host_block(split.partial.ml) < bytes) Fail(ACCEL_HIP_LOGIC_ERROR, "the parts have no room");
  });
}
