// C-ABI entry points for long contexts: scaled rotary positions, the 8-bit KV cache, attention over
// it and sliding-window attention. The checks of arguments and the frequencies; the kernels are in
// rope_scaled.hip, cache_q8.hip, attention_q8.hip and attention_window.hip. None of these calls has a
// reference counterpart; their checks and statuses follow Rope, AppendCache and Attention in capi.cc.
#include <algorithm>
#include <cmath>
#include <vector>

#include "common.h"
#include "host_util.h"

namespace accel_hip {
namespace {

constexpr int64_t kMaxHeadDim = 256;
constexpr int64_t kMaxBlock = 256;
constexpr int64_t kMaxRows = 0x7fffffff - 256;  // positions and row counts are 32-bit in the kernels
constexpr int64_t kMaxKvRow = 1 << 24;           // and a step's offsets from its first key row
constexpr double kTwoPi = 6.283185307179586476925286766559;
constexpr double kLog2e = 1.4426950408889634073599246810019;

void Invalid(const char* what) { Fail(ACCEL_HIP_INVALID_ARGUMENT, what); }

// Floats of `rows` rows of `width`, row_stride apart (0: dense).
int64_t Stride(int64_t row_stride, int64_t width, const char* what) {
  if (row_stride != 0 && row_stride < width) Invalid(what);
  return row_stride == 0 ? width : row_stride;
}
size_t StridedBytes(int64_t rows, int64_t stride, int64_t width) {
  if (rows == 0 || width == 0) return 0;
  const size_t before = CheckedBytes(rows - 1, stride);
  const size_t last = CheckedBytes(width, 1);
  if (before > SIZE_MAX - last) Fail(ACCEL_HIP_OVERFLOW, "matrix is too large");
  return before + last;
}

bool Overlap(const AccelHipBuffer& a, size_t a_bytes, const AccelHipBuffer& b, size_t b_bytes) {
  const char* x = static_cast<const char*>(a.data);
  const char* y = static_cast<const char*>(b.data);
  return a_bytes > 0 && b_bytes > 0 && x < y + b_bytes && y < x + a_bytes;
}

// b against `rows` rows of `width` bytes, `stride` bytes apart: what lies between the rows is not theirs.
bool OverlapsStrided(const AccelHipBuffer& b, size_t bytes, const AccelHipBuffer& to, int64_t rows, size_t stride,
                     size_t width) {
  if (rows == 0 || !Overlap(b, bytes, to, static_cast<size_t>(rows - 1) * stride + width)) return false;
  if (b.data <= to.data) return true;
  const size_t in_row = static_cast<size_t>(static_cast<const char*>(b.data) - static_cast<const char*>(to.data)) % stride;
  return in_row < width || bytes > stride - in_row;
}

void RequireAligned(const AccelHipBuffer& b, size_t to, const char* what) {
  if (reinterpret_cast<uintptr_t>(b.data) % to != 0) Invalid(what);
}

int64_t HeadRow(int64_t heads, int64_t dim) {
  CheckedBytes(heads, dim);
  if (heads > kMaxRows || dim > kMaxRows || heads * dim > kMaxRows) Fail(ACCEL_HIP_OVERFLOW, "matrix is too large");
  return heads * dim;
}

// The cache's shape and room.
Q8Cache CheckedCache(const AccelHipCacheQ8* c) {
  if (c == nullptr) Invalid("the 8-bit cache is missing");
  if (c->capacity < 0 || c->kv_heads <= 0 || c->head_dim <= 0) Invalid("8-bit cache shape is out of range");
  if (c->head_dim > kMaxHeadDim) Invalid("8-bit cache head_dim must be in 1..256");
  if (c->block < 1 || c->block > kMaxBlock || (c->block & (c->block - 1)) != 0)
    Invalid("8-bit cache block must be a power of two up to 256");
  const int64_t row = HeadRow(c->kv_heads, c->head_dim);
  const size_t codes = CheckedBytes(c->capacity, row) / sizeof(float);
  const size_t scales = CheckedBytes(c->capacity / c->block + (c->capacity % c->block != 0), c->kv_heads);
  RequireBytes(c->k, codes, "8-bit cache keys are out of range");
  RequireBytes(c->v, codes, "8-bit cache values are out of range");
  RequireBytes(c->k_scale, scales, "8-bit cache key scales are out of range");
  RequireBytes(c->v_scale, scales, "8-bit cache value scales are out of range");
  RequireAligned(c->k_scale, sizeof(float), "8-bit cache key scales are not aligned");
  RequireAligned(c->v_scale, sizeof(float), "8-bit cache value scales are not aligned");
  Q8Cache out;
  out.k = {static_cast<int8_t*>(c->k.data), static_cast<float*>(c->k_scale.data)};
  out.v = {static_cast<int8_t*>(c->v.data), static_cast<float*>(c->v_scale.data)};
  out.kv_heads = static_cast<int32_t>(c->kv_heads);
  out.dim = static_cast<int32_t>(c->head_dim);
  out.block_shift = 0;
  while ((int64_t(1) << out.block_shift) < c->block) ++out.block_shift;
  return out;
}

// Whether b covers codes or scales of rows [first, end) of one plane of a checked cache; first < end.
bool OverlapsRows(const AccelHipBuffer& b, size_t bytes, const AccelHipCacheQ8* c, const AccelHipBuffer& codes,
                  const AccelHipBuffer& scales, int64_t first, int64_t end) {
  const auto overlap = [&](const AccelHipBuffer& plane, int64_t from, int64_t to, size_t each) {
    const AccelHipBuffer part{static_cast<char*>(plane.data) + static_cast<size_t>(from) * each, plane.bytes, 0};
    return Overlap(b, bytes, part, static_cast<size_t>(to - from) * each);
  };
  return overlap(codes, first, end, static_cast<size_t>(c->kv_heads * c->head_dim)) ||
         overlap(scales, first / c->block, (end - 1) / c->block + 1, static_cast<size_t>(c->kv_heads) * sizeof(float));
}

// Everything of the two attention calls but the cache. False: nothing to do.
bool CheckedAttend(const AccelHipBuffer& q, const AccelHipBuffer& out, int64_t seq, int64_t position, int64_t heads,
                   int64_t kv_heads, int64_t dim, int64_t row_stride, int64_t window, int64_t sinks, AttendArgs* a) {
  if (kv_heads <= 0 || kv_heads > kMaxRows || (heads > 0 && heads % kv_heads != 0)) Invalid("Attention kv heads are out of range");
  if (window < 0 || sinks < 0) Invalid("Attention window is out of range");
  if (heads < 0 || dim < 0) Invalid("negative matrix dimension");
  if (dim > kMaxHeadDim) Invalid("Attention head_dim must be in 1..256");
  const int64_t seen = CheckedSpan(position, seq);
  const int64_t row = HeadRow(heads, dim);
  const int64_t stride = Stride(row_stride, row, "Attention query rows overlap");
  const size_t q_bytes = StridedBytes(seq, stride, row);
  const size_t out_bytes = CheckedBytes(seq, row);
  RequireBytes(q, q_bytes, "Attention query is out of range");
  RequireBytes(out, out_bytes, "Attention output is out of range");
  RequireAligned(q, sizeof(float), "Attention query is not aligned");
  RequireAligned(out, sizeof(float), "Attention output is not aligned");
  if (Overlap(q, q_bytes, out, out_bytes)) Invalid("Attention output overlaps the query");
  if (kv_heads * dim > kMaxKvRow) Invalid("Attention is too large");
  if (seen > kMaxRows || (heads > 0 && seq > kMaxRows / heads)) Invalid("Attention is too large");
  a->q = static_cast<const float*>(q.data);
  a->out = static_cast<float*>(out.data);
  a->q_stride = stride;
  a->seq = static_cast<int32_t>(seq);
  a->position = static_cast<int32_t>(position);
  a->heads = static_cast<int32_t>(heads);
  a->kv_heads = static_cast<int32_t>(kv_heads);
  a->dim = static_cast<int32_t>(dim);
  a->window = window == 0 || window >= seen ? kNoWindow : static_cast<int32_t>(window);
  a->sinks = static_cast<int32_t>(std::min(sinks, seen));
  a->factor = dim > 0 ? static_cast<float>(kLog2e / std::sqrt(static_cast<double>(dim))) : 0.f;
  return out_bytes > 0;
}

std::vector<double> Frequencies(const AccelHipRopeScaling& s, int64_t rotary) {
  if (s.kind < ACCEL_HIP_ROPE_SCALE_NONE || s.kind > ACCEL_HIP_ROPE_SCALE_WAVELENGTH) Invalid("unknown rope scaling");
  if (!(s.theta > 0) || !std::isfinite(s.theta)) Invalid("rope theta is out of range");
  if (s.kind != ACCEL_HIP_ROPE_SCALE_NONE && (!(s.factor > 0) || !std::isfinite(s.factor)))
    Invalid("rope scaling factor is out of range");
  const bool ramps = s.kind == ACCEL_HIP_ROPE_SCALE_YARN || s.kind == ACCEL_HIP_ROPE_SCALE_WAVELENGTH;
  if (ramps && (!(s.original_context > 0) || !(s.slow > 0) || !(s.fast > s.slow) || !std::isfinite(s.fast) ||
                !std::isfinite(s.original_context)))
    Invalid("rope scaling borders are out of range");
  if (s.kind == ACCEL_HIP_ROPE_SCALE_YARN && !(s.theta > 1)) Invalid("rope theta is out of range");
  if (s.kind == ACCEL_HIP_ROPE_SCALE_NTK && rotary < 4) Invalid("rope scaling needs a rotary_dim of 4 at least");
  const double r = static_cast<double>(rotary);
  const double theta =
      s.kind == ACCEL_HIP_ROPE_SCALE_NTK ? s.theta * std::pow(s.factor, r / (r - 2)) : s.theta;
  double low = 0, high = 0;
  if (s.kind == ACCEL_HIP_ROPE_SCALE_YARN) {
    // The (fractional) pair that makes n turns over the original context: theta^(-2i/r) L / 2 pi = n.
    const auto at = [&](double turns) {
      return r * std::log(s.original_context / (turns * kTwoPi)) / (2 * std::log(s.theta));
    };
    low = std::max(std::floor(at(s.fast)), 0.0);
    high = std::min(std::ceil(at(s.slow)), r - 1);
  }
  std::vector<double> f(static_cast<size_t>(rotary / 2));
  for (size_t i = 0; i < f.size(); ++i) {
    const double plain = std::pow(theta, -2.0 * static_cast<double>(i) / r);
    double part = 0;  // how much of the frequency is divided by the factor
    if (s.kind == ACCEL_HIP_ROPE_SCALE_LINEAR) part = 1;
    if (s.kind == ACCEL_HIP_ROPE_SCALE_YARN) part = (static_cast<double>(i) - low) / std::max(high - low, 0.001);
    if (s.kind == ACCEL_HIP_ROPE_SCALE_WAVELENGTH)
      part = 1 - (s.original_context * plain / kTwoPi - s.slow) / (s.fast - s.slow);
    part = std::min(std::max(part, 0.0), 1.0);
    f[i] = part == 0 ? plain : plain / s.factor * part + plain * (1 - part);
  }
  return f;
}

}  // namespace
}  // namespace accel_hip

using namespace accel_hip;

extern "C" {

ACCEL_HIP_API int accel_hip_rope_frequencies(const AccelHipRopeScaling* scaling, int64_t rotary_dim,
                                             AccelHipBuffer frequencies, float* magnitude) {
  return Guard([&] {
    if (scaling == nullptr) Invalid("rope scaling is missing");
    if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > kMaxHeadDim) Invalid("rotary_dim must be even, in 0..256");
    RequireBytes(frequencies, static_cast<size_t>(rotary_dim / 2) * sizeof(double), "Rope frequencies are out of range");
    RequireAligned(frequencies, sizeof(double), "Rope frequencies are not aligned");
    const std::vector<double> f = Frequencies(*scaling, rotary_dim);
    if (!f.empty()) {
      Context& ctx = Ctx();
      RefuseInCapture("writing the rope frequencies");
      const size_t bytes = f.size() * sizeof(double);
      NoteDeviceWrite(frequencies.data, bytes);
      Check(hipMemcpyAsync(frequencies.data, f.data(), bytes, hipMemcpyHostToDevice, ctx.stream), "hipMemcpyAsync");
      Check(hipStreamSynchronize(ctx.stream), "hipStreamSynchronize");
    }
    if (magnitude != nullptr)
      *magnitude = scaling->kind == ACCEL_HIP_ROPE_SCALE_YARN && scaling->factor > 1
                       ? static_cast<float>(0.1 * std::log(scaling->factor) + 1.0)
                       : 1.f;
  });
}

ACCEL_HIP_API int accel_hip_rope_scaled(AccelHipBuffer states, AccelHipBuffer out, AccelHipBuffer frequencies,
                                        AccelHipBuffer positions, int64_t seq, int64_t n_heads, int64_t head_dim,
                                        int64_t row_stride, int64_t rotary_dim, int32_t layout, int64_t position,
                                        float magnitude) {
  return Guard([&] {
    if (seq < 0 || n_heads < 0 || head_dim < 0) Invalid("negative matrix dimension");
    if (head_dim > kMaxHeadDim) Invalid("Rope head_dim must be in 1..256");
    if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim) Invalid("rotary_dim must be even, in 0..head_dim");
    if (layout != ACCEL_HIP_ROPE_HALF && layout != ACCEL_HIP_ROPE_INTERLEAVED) Invalid("unknown rope layout");
    if (CheckedSpan(position, seq) > kMaxRows) Invalid("Rope position is out of range");
    const int64_t row = HeadRow(n_heads, head_dim);
    const int64_t stride = Stride(row_stride, row, "Rope rows overlap");
    const size_t bytes = StridedBytes(seq, stride, row);
    RequireBytes(states, bytes, "Rope states are out of range");
    RequireBytes(out, bytes, "Rope output is out of range");
    RequireAligned(states, sizeof(float), "Rope states are not aligned");
    RequireAligned(out, sizeof(float), "Rope output is not aligned");
    if (out.data != states.data && Overlap(states, bytes, out, bytes)) Invalid("Rope output overlaps the states");
    if (bytes == 0) return;
    RequireBytes(frequencies, static_cast<size_t>(rotary_dim / 2) * sizeof(double), "Rope frequencies are out of range");
    RequireAligned(frequencies, sizeof(double), "Rope frequencies are not aligned");
    if (positions.data != nullptr) {
      RequireBytes(positions, CheckedIntBytes(seq), "Rope positions are out of range");
      RequireAligned(positions, sizeof(int32_t), "Rope positions are not aligned");
    }
    // Other workgroups may still read them.
    const size_t stride_bytes = static_cast<size_t>(stride) * sizeof(float);
    const size_t row_bytes = static_cast<size_t>(row) * sizeof(float);
    const size_t frequency_bytes = static_cast<size_t>(rotary_dim / 2) * sizeof(double);
    if (OverlapsStrided(frequencies, frequency_bytes, out, seq, stride_bytes, row_bytes))
      Invalid("Rope output overlaps the frequencies");
    if (rotary_dim > 0 && OverlapsStrided(positions, CheckedIntBytes(seq), out, seq, stride_bytes, row_bytes))
      Invalid("Rope output overlaps the positions");
    NoteDeviceWrite(out.data, bytes);
    RopeScaledArgs a;
    a.states = static_cast<const float*>(states.data);
    a.out = static_cast<float*>(out.data);
    a.frequencies = static_cast<const double*>(frequencies.data);
    a.positions = static_cast<const int32_t*>(positions.data);
    a.seq = seq;
    a.row_stride = stride;
    a.position = position;
    a.heads = static_cast<int32_t>(n_heads);
    a.dim = static_cast<int32_t>(head_dim);
    a.rotary = static_cast<int32_t>(rotary_dim);
    a.layout = layout;
    a.magnitude = magnitude;
    LaunchRopeScaled(a, Ctx().stream);
  });
}

ACCEL_HIP_API int accel_hip_append_cache_q8(AccelHipBuffer k, AccelHipBuffer v, const AccelHipCacheQ8* cache,
                                            int64_t seq, int64_t position, int64_t row_stride) {
  return Guard([&] {
    const Q8Cache c = CheckedCache(cache);
    const int64_t end = CheckedSpan(position, seq);
    if (end > cache->capacity) Invalid("8-bit cache rows are out of range");
    if (end > kMaxRows) Invalid("8-bit cache position is out of range");
    const int64_t row = cache->kv_heads * cache->head_dim;
    const int64_t stride = Stride(row_stride, row, "AppendCache rows overlap");
    const size_t bytes = StridedBytes(seq, stride, row);
    RequireBytes(k, bytes, "AppendCache keys are out of range");
    RequireBytes(v, bytes, "AppendCache values are out of range");
    RequireAligned(k, sizeof(float), "AppendCache keys are not aligned");
    RequireAligned(v, sizeof(float), "AppendCache values are not aligned");
    if (seq == 0) return;
    const size_t code_bytes = CheckedBytes(cache->capacity, row) / sizeof(float);
    const size_t scale_bytes = CheckedBytes((cache->capacity - 1) / cache->block + 1, cache->kv_heads);
    const struct { const AccelHipBuffer& buffer; size_t bytes; } parts[] = {
        {cache->k, code_bytes}, {cache->v, code_bytes}, {cache->k_scale, scale_bytes}, {cache->v_scale, scale_bytes},
        {k, bytes}, {v, bytes}};
    for (int i = 0; i < 4; ++i)  // k and v may share rows
      for (int j = i + 1; j < 6; ++j)
        if (Overlap(parts[i].buffer, parts[i].bytes, parts[j].buffer, parts[j].bytes)) Invalid("AppendCache planes overlap");
    const int64_t b0 = position / cache->block;
    const size_t first = static_cast<size_t>(b0 * cache->block * row);
    const size_t codes = static_cast<size_t>(end * row) - first;
    NoteDeviceWrite(c.k.code + first, codes);
    NoteDeviceWrite(c.v.code + first, codes);
    NoteDeviceWrite(c.k.scale, sizeof(float));
    NoteDeviceWrite(c.v.scale, sizeof(float));
    LaunchAppendCacheQ8(static_cast<const float*>(k.data), static_cast<const float*>(v.data), c, seq, position, stride,
                        Ctx().stream);
  });
}

ACCEL_HIP_API int accel_hip_read_cache_q8(const AccelHipCacheQ8* cache, int64_t first, int64_t count,
                                          AccelHipBuffer k_out, AccelHipBuffer v_out) {
  return Guard([&] {
    const Q8Cache c = CheckedCache(cache);
    const int64_t end = CheckedSpan(first, count);
    if (end > cache->capacity) Invalid("8-bit cache rows are out of range");
    if (end > kMaxRows) Invalid("8-bit cache position is out of range");
    const size_t bytes = CheckedBytes(count, cache->kv_heads * cache->head_dim);
    const auto checked = [&](const AccelHipBuffer& out, const char* what) {
      if (out.data == nullptr || bytes == 0) return static_cast<float*>(nullptr);
      RequireBytes(out, bytes, what);
      RequireAligned(out, sizeof(float), what);
      return static_cast<float*>(out.data);
    };
    float* k = checked(k_out, "cache key output is out of range");
    float* v = checked(v_out, "cache value output is out of range");
    if (k == nullptr && v == nullptr) return;
    if (k != nullptr && v != nullptr && Overlap(k_out, bytes, v_out, bytes)) Invalid("cache outputs overlap");
    for (const AccelHipBuffer& out : {k_out, v_out}) {
      if (out.data == nullptr) continue;
      if ((k != nullptr && OverlapsRows(out, bytes, cache, cache->k, cache->k_scale, first, end)) ||
          (v != nullptr && OverlapsRows(out, bytes, cache, cache->v, cache->v_scale, first, end)))
        Invalid("cache outputs overlap the cache");
    }
    if (k != nullptr) NoteDeviceWrite(k, bytes);
    if (v != nullptr) NoteDeviceWrite(v, bytes);
    LaunchReadCacheQ8(c, first, count, k, v, Ctx().stream);
  });
}

ACCEL_HIP_API int accel_hip_attention_q8(AccelHipBuffer q, const AccelHipCacheQ8* cache, AccelHipBuffer out,
                                         int64_t seq, int64_t position, int64_t heads, int64_t row_stride,
                                         int64_t window, int64_t sinks) {
  return Guard([&] {
    const Q8Cache c = CheckedCache(cache);
    AttendArgs a;
    const bool any = CheckedAttend(q, out, seq, position, heads, c.kv_heads, c.dim, row_stride, window, sinks, &a);
    if (position + seq > cache->capacity) Invalid("8-bit cache rows are out of range");
    if (!any) return;
    const size_t out_bytes = CheckedBytes(seq, heads * c.dim);
    if (OverlapsRows(out, out_bytes, cache, cache->k, cache->k_scale, 0, position + seq) ||
        OverlapsRows(out, out_bytes, cache, cache->v, cache->v_scale, 0, position + seq))
      Invalid("Attention output overlaps the cache");
    NoteDeviceWrite(out.data, sizeof(float));
    LaunchAttentionQ8(a, c, Ctx().stream);
  });
}

ACCEL_HIP_API int accel_hip_attention_window(AccelHipBuffer q, AccelHipBuffer k, AccelHipBuffer v, AccelHipBuffer out,
                                             int64_t seq, int64_t position, int64_t heads, int64_t kv_heads,
                                             int64_t head_dim, int64_t row_stride, int64_t window, int64_t sinks) {
  return Guard([&] {
    AttendArgs a;
    const bool any =
        CheckedAttend(q, out, seq, position, heads, kv_heads, head_dim, row_stride, window, sinks, &a);
    const size_t bytes = CheckedBytes(position + seq, HeadRow(kv_heads, head_dim));
    RequireBytes(k, bytes, "Attention key is out of range");
    RequireBytes(v, bytes, "Attention value is out of range");
    RequireAligned(k, sizeof(float), "Attention key is not aligned");
    RequireAligned(v, sizeof(float), "Attention value is not aligned");
    if (!any) return;
    const size_t out_bytes = CheckedBytes(seq, heads * head_dim);
    if (Overlap(out, out_bytes, k, bytes) || Overlap(out, out_bytes, v, bytes))
      Invalid("Attention output overlaps the cache");
    NoteDeviceWrite(out.data, sizeof(float));
    LaunchAttentionWindow(a, static_cast<const float*>(k.data), static_cast<const float*>(v.data), Ctx().stream);
  });
}

}  // extern "C"
