// C-ABI entry points for many requests served from one cache in pages: the tables of a step, pages taken
// back, rows into pages, attention over pages and over packed prompts. The checks of arguments; the
// kernels are in batch_tables.hip, cache_paged.hip and attend_batch*.{h,hip}. What lies in device memory (lengths,
// tables, slots) is checked by the kernels that read it. No reference counterpart; checks and statuses follow
// AppendCache and Attention in capi.cc.
#include <algorithm>

#include "common.h"
#include "host_util.h"

namespace accel_hip {
namespace {

constexpr int64_t kMinPage = 16;
constexpr int64_t kMaxPage = 256;

struct Part {
  const AccelHipBuffer* buffer;
  size_t bytes;
};

void RequireInts(const AccelHipBuffer& b, size_t bytes, const char* what) {
  RequireBytes(b, bytes, what);
  if (bytes > 0) RequireAligned(b, sizeof(int32_t), what);
}

int32_t PageShift(int64_t page) {
  if (page < kMinPage || page > kMaxPage || (page & (page - 1)) != 0) Invalid("a page must be a power of two in 16..256");
  int32_t shift = 0;
  while ((int64_t(1) << shift) < page) ++shift;
  return shift;
}

// The sizes of a batch. table_bytes: of its table, where it has one.
void CheckBatch(const AccelHipBatch* b, int32_t page_shift, bool table, size_t* table_bytes) {
  if (b == nullptr) Invalid("the batch is missing");
  if (b->requests < 0 || b->rows < 0 || b->longest < 0) Invalid("batch sizes are out of range");
  if (b->requests > kMaxRows - 1 || b->rows > kMaxRows) Invalid("the batch is too large");
  if (!table) return;
  if (b->width < 0) Invalid("batch sizes are out of range");
  if (b->width > (kMaxRows - b->rows) >> page_shift) Invalid("the batch's table is too wide");
  *table_bytes = CheckedBytes(b->requests, b->width);
}

size_t StartsBytes(const AccelHipBatch* b) { return CheckedIntBytes(b->requests + 1); }

// Every output apart from all that follow it, and from all inputs.
void RequireApart(const Part* outputs, int output_count, const Part* inputs, int input_count, const char* what) {
  for (int i = 0; i < output_count; ++i) {
    for (int j = i + 1; j < output_count; ++j)
      if (Overlap(*outputs[i].buffer, outputs[i].bytes, *outputs[j].buffer, outputs[j].bytes)) Invalid(what);
    for (int j = 0; j < input_count; ++j)
      if (Overlap(*outputs[i].buffer, outputs[i].bytes, *inputs[j].buffer, inputs[j].bytes)) Invalid(what);
  }
}

void CheckPool(const AccelHipPagePool* p, int32_t* page_shift, size_t* stack_bytes) {
  if (p == nullptr) Invalid("the page pool is missing");
  *page_shift = PageShift(p->page);
  if (p->pages < 0 || p->pages > kMaxRows >> *page_shift) Invalid("the page pool's size is out of range");
  *stack_bytes = CheckedIntBytes(p->pages);
  RequireInts(p->stack, *stack_bytes, "the page pool's stack is out of range");
  RequireInts(p->state, 2 * sizeof(int32_t), "the page pool's state is out of range");
}

// The bytes of one plane.
size_t CheckCache(const AccelHipCachePaged* c, int32_t* page_shift) {
  if (c == nullptr) Invalid("the paged cache is missing");
  if (c->type != ACCEL_HIP_CACHE_F32 && c->type != ACCEL_HIP_CACHE_F16) Invalid("unknown cache type");
  if (c->pages <= 0 || c->kv_heads <= 0 || c->head_dim <= 0) Invalid("paged cache shape is out of range");
  if (c->head_dim > kMaxHeadDim) Invalid("paged cache head_dim must be in 1..256");
  *page_shift = PageShift(c->page);
  if (c->pages > kMaxRows >> *page_shift) Invalid("the paged cache is too large");
  const int64_t row = HeadRow(c->kv_heads, c->head_dim);
  if (row > kMaxKvRow) Invalid("the paged cache is too large");
  const size_t each = c->type == ACCEL_HIP_CACHE_F16 ? 2 : 4;
  const size_t bytes = CheckedBytes(c->pages << *page_shift, row) / sizeof(float) * each;
  RequireBytes(c->k, bytes, "paged cache keys are out of range");
  RequireBytes(c->v, bytes, "paged cache values are out of range");
  RequireAligned(c->k, each, "paged cache keys are not aligned");
  RequireAligned(c->v, each, "paged cache values are not aligned");
  return bytes;
}

// What both attention calls share. False: nothing to do.
bool CheckAttend(const AccelHipBuffer& q, const AccelHipBatch* batch, const AccelHipBuffer& out, int64_t heads,
                 int64_t kv_heads, int64_t dim, int64_t row_stride, int64_t window, size_t* q_bytes, size_t* out_bytes,
                 BatchAttendArgs* a) {
  if (kv_heads <= 0 || kv_heads > kMaxRows || heads < 0 || heads % kv_heads != 0) Invalid("Attention kv heads are out of range");
  if (window < 0) Invalid("Attention window is out of range");
  if (dim <= 0 || dim > kMaxHeadDim) Invalid("Attention head_dim must be in 1..256");
  const int64_t row = HeadRow(heads, dim);
  const int64_t stride = Stride(row_stride, row, "Attention query rows overlap");
  *q_bytes = StridedBytes(batch->rows, stride, row);
  *out_bytes = CheckedBytes(batch->rows, row);
  RequireInts(batch->starts, StartsBytes(batch), "the batch's starts are out of range");
  RequireBytes(q, *q_bytes, "Attention query is out of range");
  RequireBytes(out, *out_bytes, "Attention output is out of range");
  RequireAligned(q, sizeof(float), "Attention query is not aligned");
  RequireAligned(out, sizeof(float), "Attention output is not aligned");
  if (heads > 0 && batch->rows > kMaxRows / heads) Invalid("Attention is too large");
  a->q = static_cast<const float*>(q.data);
  a->out = static_cast<float*>(out.data);
  a->starts = static_cast<const int32_t*>(batch->starts.data);
  a->q_stride = stride;
  a->requests = static_cast<int32_t>(batch->requests);
  a->rows = static_cast<int32_t>(batch->rows);
  a->heads = static_cast<int32_t>(heads);
  a->kv_heads = static_cast<int32_t>(kv_heads);
  a->dim = static_cast<int32_t>(dim);
  a->window = window == 0 || window > kMaxRows ? kNoWindow : static_cast<int32_t>(window);
  a->longest = static_cast<int32_t>(batch->longest == 0 ? batch->rows : std::min(batch->longest, batch->rows));
  a->factor = AttendFactor(dim);
  a->group = DivisorOf(std::max<int64_t>(heads / kv_heads, 1));
  a->by_kv_heads = DivisorOf(kv_heads);
  return batch->requests > 0 && *out_bytes > 0;
}

}  // namespace
}  // namespace accel_hip

using namespace accel_hip;

extern "C" {

ACCEL_HIP_API int accel_hip_batch_tables(AccelHipBuffer counts, AccelHipBuffer lengths, const AccelHipPagePool* pool,
                                         const AccelHipBatch* batch, AccelHipBuffer slots, AccelHipBuffer positions,
                                         AccelHipBuffer lengths_after, AccelHipBuffer state_after) {
  return Guard([&] {
    BatchTablesArgs a;
    size_t stack_bytes = 0, table_bytes = 0;
    CheckPool(pool, &a.page_shift, &stack_bytes);
    CheckBatch(batch, a.page_shift, true, &table_bytes);
    const size_t each = CheckedIntBytes(batch->requests), rows = CheckedIntBytes(batch->rows);
    constexpr size_t kState = 2 * sizeof(int32_t);
    RequireInts(counts, each, "the new tokens' counts are out of range");
    RequireInts(lengths, each, "the requests' lengths are out of range");
    RequireInts(batch->starts, StartsBytes(batch), "the batch's starts are out of range");
    RequireInts(batch->seen, each, "the batch's seen tokens are out of range");
    RequireInts(batch->table, table_bytes, "the batch's table is out of range");
    RequireInts(slots, rows, "the slots are out of range");
    RequireInts(positions, rows, "the positions are out of range");
    RequireInts(lengths_after, each, "the requests' later lengths are out of range");
    RequireInts(state_after, kState, "the page pool's later state is out of range");
    const bool same_lengths = lengths_after.data == lengths.data, same_state = state_after.data == pool->state.data;
    const Part outputs[] = {{&batch->starts, StartsBytes(batch)}, {&batch->seen, each}, {&batch->table, table_bytes},
                            {&slots, rows}, {&positions, rows}, {&lengths_after, each}, {&state_after, kState}};
    const Part inputs[] = {{&counts, each}, {&pool->stack, stack_bytes}, {&lengths, same_lengths ? 0 : each},
                           {&pool->state, same_state ? 0 : kState}};
    RequireApart(outputs, 7, inputs, 4, "the batch's tables overlap");
    for (const Part& p : outputs)
      if (p.bytes > 0) NoteDeviceWrite(p.buffer->data, p.bytes);
    a.counts = static_cast<const int32_t*>(counts.data);
    a.lengths = static_cast<const int32_t*>(lengths.data);
    a.stack = static_cast<const int32_t*>(pool->stack.data);
    a.state = static_cast<const int32_t*>(pool->state.data);
    a.starts = static_cast<int32_t*>(batch->starts.data);
    a.seen = static_cast<int32_t*>(batch->seen.data);
    a.table = static_cast<int32_t*>(batch->table.data);
    a.slots = static_cast<int32_t*>(slots.data);
    a.positions = static_cast<int32_t*>(positions.data);
    a.lengths_after = static_cast<int32_t*>(lengths_after.data);
    a.state_after = static_cast<int32_t*>(state_after.data);
    a.requests = static_cast<int32_t>(batch->requests);
    a.rows = static_cast<int32_t>(batch->rows);
    a.width = static_cast<int32_t>(batch->width);
    a.pages = static_cast<int32_t>(pool->pages);
    LaunchBatchTables(a, Ctx().stream);
  });
}

ACCEL_HIP_API int accel_hip_release_pages(AccelHipBuffer keep, AccelHipBuffer lengths, const AccelHipPagePool* pool,
                                          const AccelHipBatch* batch) {
  return Guard([&] {
    ReleasePagesArgs a;
    size_t stack_bytes = 0, table_bytes = 0;
    CheckPool(pool, &a.page_shift, &stack_bytes);
    CheckBatch(batch, a.page_shift, true, &table_bytes);
    const size_t each = CheckedIntBytes(batch->requests);
    constexpr size_t kState = 2 * sizeof(int32_t);
    RequireInts(keep, each, "the tokens to keep are out of range");
    RequireInts(lengths, each, "the requests' lengths are out of range");
    RequireInts(batch->table, table_bytes, "the batch's table is out of range");
    const Part outputs[] = {{&lengths, each}, {&batch->table, table_bytes}, {&pool->stack, stack_bytes}, {&pool->state, kState}};
    const Part inputs[] = {{&keep, each}};
    RequireApart(outputs, 4, inputs, 1, "the batch's tables overlap");
    if (batch->requests == 0) return;
    for (const Part& p : outputs)
      if (p.bytes > 0) NoteDeviceWrite(p.buffer->data, p.bytes);
    a.keep = static_cast<const int32_t*>(keep.data);
    a.lengths = static_cast<int32_t*>(lengths.data);
    a.table = static_cast<int32_t*>(batch->table.data);
    a.stack = static_cast<int32_t*>(pool->stack.data);
    a.state = static_cast<int32_t*>(pool->state.data);
    a.requests = static_cast<int32_t>(batch->requests);
    a.width = static_cast<int32_t>(batch->width);
    a.pages = static_cast<int32_t>(pool->pages);
    LaunchReleasePages(a, Ctx().stream);
  });
}

ACCEL_HIP_API int accel_hip_append_paged(AccelHipBuffer k, AccelHipBuffer v, const AccelHipCachePaged* cache,
                                         AccelHipBuffer slots, int64_t rows, int64_t row_stride) {
  return Guard([&] {
    int32_t shift = 0;
    const size_t plane = CheckCache(cache, &shift);
    if (rows < 0) Invalid("negative matrix dimension");
    if (rows > kMaxRows) Invalid("AppendCache is too large");
    const int64_t row = cache->kv_heads * cache->head_dim;
    const int64_t stride = Stride(row_stride, row, "AppendCache rows overlap");
    const size_t bytes = StridedBytes(rows, stride, row), slot_bytes = CheckedIntBytes(rows);
    RequireBytes(k, bytes, "AppendCache keys are out of range");
    RequireBytes(v, bytes, "AppendCache values are out of range");
    RequireAligned(k, sizeof(float), "AppendCache keys are not aligned");
    RequireAligned(v, sizeof(float), "AppendCache values are not aligned");
    RequireInts(slots, slot_bytes, "AppendCache slots are out of range");
    const Part outputs[] = {{&cache->k, plane}, {&cache->v, plane}};
    const Part inputs[] = {{&k, bytes}, {&v, bytes}, {&slots, slot_bytes}};
    RequireApart(outputs, 2, inputs, 3, "AppendCache planes overlap");
    if (rows == 0) return;
    NoteDeviceWrite(cache->k.data, plane);
    NoteDeviceWrite(cache->v.data, plane);
    AppendPagedArgs a;
    a.src[0] = static_cast<const float*>(k.data);
    a.src[1] = static_cast<const float*>(v.data);
    a.dst[0] = cache->k.data;
    a.dst[1] = cache->v.data;
    a.slots = static_cast<const int32_t*>(slots.data);
    a.row_stride = stride;
    a.rows = static_cast<int32_t>(rows);
    a.width = static_cast<int32_t>(row);
    a.slot_count = static_cast<int32_t>(cache->pages << shift);
    a.f16 = cache->type == ACCEL_HIP_CACHE_F16;
    LaunchAppendPaged(a, Ctx().stream);
  });
}

ACCEL_HIP_API int accel_hip_attention_paged(AccelHipBuffer q, const AccelHipCachePaged* cache, const AccelHipBatch* batch,
                                            AccelHipBuffer out, int64_t heads, int64_t row_stride, int64_t window) {
  return Guard([&] {
    BatchAttendArgs a;
    const size_t plane = CheckCache(cache, &a.page_shift);
    size_t table_bytes = 0, q_bytes = 0, out_bytes = 0;
    CheckBatch(batch, a.page_shift, true, &table_bytes);
    const size_t seen_bytes = CheckedIntBytes(batch->requests);
    const size_t slot_bytes = batch->slots.data == nullptr ? 0 : CheckedIntBytes(batch->rows);
    RequireInts(batch->seen, seen_bytes, "the batch's seen tokens are out of range");
    RequireInts(batch->table, table_bytes, "the batch's table is out of range");
    RequireInts(batch->slots, slot_bytes, "the batch's slots are out of range");
    const bool any = CheckAttend(q, batch, out, heads, cache->kv_heads, cache->head_dim, row_stride, window, &q_bytes,
                                 &out_bytes, &a);
    const Part outputs[] = {{&out, out_bytes}};
    const Part inputs[] = {{&q, q_bytes}, {&cache->k, plane}, {&cache->v, plane}, {&batch->starts, StartsBytes(batch)},
                           {&batch->seen, seen_bytes}, {&batch->table, table_bytes}, {&batch->slots, slot_bytes}};
    RequireApart(outputs, 1, inputs, 7, "Attention output overlaps what is read");
    if (!any) return;
    NoteDeviceWrite(out.data, out_bytes);
    a.k = cache->k.data;
    a.v = cache->v.data;
    a.kv_stride = cache->kv_heads * cache->head_dim;
    a.seen = static_cast<const int32_t*>(batch->seen.data);
    a.table = static_cast<const int32_t*>(batch->table.data);
    a.width = static_cast<int32_t>(batch->width);
    a.pages = static_cast<int32_t>(cache->pages);
    a.f16 = cache->type == ACCEL_HIP_CACHE_F16;
    a.paged = true;
    a.slots = slot_bytes == 0 ? nullptr : static_cast<const int32_t*>(batch->slots.data);
    LaunchAttendBatch(a, Ctx().stream);
  });
}

ACCEL_HIP_API int accel_hip_attention_packed(AccelHipBuffer q, AccelHipBuffer k, AccelHipBuffer v,
                                             const AccelHipBatch* batch, AccelHipBuffer out, int64_t heads,
                                             int64_t kv_heads, int64_t head_dim, int64_t row_stride, int64_t kv_stride,
                                             int64_t window) {
  return Guard([&] {
    BatchAttendArgs a{};
    size_t q_bytes = 0, out_bytes = 0;
    CheckBatch(batch, 0, false, nullptr);
    const bool any = CheckAttend(q, batch, out, heads, kv_heads, head_dim, row_stride, window, &q_bytes, &out_bytes, &a);
    const int64_t row = HeadRow(kv_heads, head_dim);
    if (row > kMaxKvRow) Invalid("Attention is too large");
    const int64_t stride = Stride(kv_stride, row, "Attention key rows overlap");
    const size_t bytes = StridedBytes(batch->rows, stride, row);
    RequireBytes(k, bytes, "Attention key is out of range");
    RequireBytes(v, bytes, "Attention value is out of range");
    RequireAligned(k, sizeof(float), "Attention key is not aligned");
    RequireAligned(v, sizeof(float), "Attention value is not aligned");
    const Part outputs[] = {{&out, out_bytes}};
    const Part inputs[] = {{&q, q_bytes}, {&k, bytes}, {&v, bytes}, {&batch->starts, StartsBytes(batch)}};
    RequireApart(outputs, 1, inputs, 4, "Attention output overlaps what is read");
    if (!any) return;
    NoteDeviceWrite(out.data, out_bytes);
    a.k = k.data;
    a.v = v.data;
    a.kv_stride = stride;
    LaunchAttendBatch(a, Ctx().stream);
  });
}

}  // extern "C"
