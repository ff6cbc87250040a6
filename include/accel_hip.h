/*
 * accel_hip: the C-ABI device layer behind AccelEP's accel::Device seam, on one
 * MI355X (gfx950). Plain pointers and sizes only; every compute call is a HIP
 * kernel launched on the library's single stream.
 *
 * Each entry point replaces one call of the reference's device contract
 * (AccelEP include/accel/device.h, include/accel/runtime.h) and keeps its
 * argument meaning and error behaviour: where the reference throws, the call
 * returns the status code named for that exception type and leaves a message in
 * accel_hip_last_error(). The C++ shim (include/accel/device.h,
 * accel::CreateHipDevice) rethrows the same exception types.
 *
 * Memory: every pointer argument named as a device pointer must come from
 * accel_hip_allocate (or be an offset into such an allocation). Calls are
 * stream-ordered; accel_hip_copy_d2h and accel_hip_peek return after the data
 * is on the host.
 */
#ifndef ACCEL_HIP_H_
#define ACCEL_HIP_H_

#include <stddef.h>
#include <stdint.h>

#define ACCEL_HIP_API __attribute__((visibility("default")))

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes: the exception the reference throws for the same condition. */
enum {
  ACCEL_HIP_OK = 0,
  ACCEL_HIP_INVALID_ARGUMENT = 1, /* std::invalid_argument */
  ACCEL_HIP_OVERFLOW = 2,         /* std::overflow_error */
  ACCEL_HIP_LOGIC_ERROR = 3,      /* std::logic_error */
  ACCEL_HIP_BAD_ALLOC = 4,        /* std::bad_alloc */
  ACCEL_HIP_RUNTIME_ERROR = 5     /* a HIP runtime failure (no reference counterpart) */
};

enum { ACCEL_HIP_ACT_NONE = 0, ACCEL_HIP_ACT_RELU = 1, ACCEL_HIP_ACT_GELU = 2 }; /* accel::Activation */

/* accel::DeviceBuffer (include/accel/device.h:28-32). id 0 marks a slice. */
typedef struct AccelHipBuffer {
  void* data;
  size_t bytes;
  uint64_t id;
} AccelHipBuffer;

/* accel::QuantPlane (include/accel/runtime.h:71-78) with the shape inline.
 * q/scale/zero are device pointers; zero is NULL when the op has none. */
typedef struct AccelHipQuantPlane {
  const int8_t* q;
  const float* scale;
  const int8_t* zero;
  int32_t rank; /* 1..8 */
  int64_t shape[8];
  int64_t axis; /* < 0: one scale (and zero) for the whole tensor */
  int64_t offset;
} AccelHipQuantPlane;

/* accel::AcceleratorStats (include/accel/runtime.h:11-21). */
typedef struct AccelHipStats {
  int64_t matmul_ops, gemm_ops, kernel_matmuls, relu_epilogues, gelu_epilogues, add_epilogues, device_transposes,
      bytes_to_device, bytes_to_host;
} AccelHipStats;

/* Fused register epilogue applied to C before it is stored (no reference
 * counterpart as one call: it is the reference's call sequence
 * MatMul/MatMulQuantized -> GemmEpilogue(alpha, bias, beta, act) ->
 * GemmEpilogue(residual) (src/runtime.cc:332-344,709-719) -> RmsNorm
 * (src/ep.cc:1602-1626), with the same rounding steps:
 *   v = alpha*acc; if bias: v = v + beta*bias[bcast(i, j)]; act(v);
 *   if residual: v = v + residual[i*n + j]; store v;
 *   if rms_weight: rms_out[i, :] = RmsNorm(v[i, :]) with eps = rms_eps. */
typedef struct AccelHipEpilogue {
  float alpha;
  float beta;
  const float* bias; /* device pointer or NULL */
  int32_t bias_rank; /* 0..2, right-aligned against [m, n] */
  int64_t bias_shape[2];
  int32_t activation;    /* ACCEL_HIP_ACT_* */
  const float* residual; /* device pointer [m, n] or NULL */
  const float* rms_weight; /* device pointer [n] or NULL */
  float rms_eps;
  float* rms_out; /* device pointer [m, n]; required when rms_weight is set */
} AccelHipEpilogue;

/* ---- runtime ----------------------------------------------------------------------------- */
/* Message of this thread's last failed call; "" after a call that worked. */
ACCEL_HIP_API const char* accel_hip_last_error(void);
/* Binds GPU 0 and creates the stream. Every other entry point calls it on first use. */
ACCEL_HIP_API int accel_hip_init(void);
/* Waits for all work on the library's stream. */
ACCEL_HIP_API int accel_hip_synchronize(void);
/* gcnArchName of the bound GPU, e.g. "gfx950:sramecc+:xnack-". */
ACCEL_HIP_API const char* accel_hip_device_arch(void);

/* ---- heap and copies: Device::Allocate/Free/CopyHostToDevice/CopyDeviceToHost ----------
 * (include/accel/device.h:75-79; semantics src/sim_device.cc:133-183). Allocate zero-fills,
 * returns a non-null pointer for 0 bytes, and mints a process-wide id from 1. Free of a null
 * pointer is a no-op; an unknown (data, bytes, id) triple is ACCEL_HIP_LOGIC_ERROR. Copies of
 * 0 bytes do nothing; a null pointer or bytes > buffer.bytes is ACCEL_HIP_INVALID_ARGUMENT;
 * each copy adds to bytes_to_device / bytes_to_host. */
ACCEL_HIP_API int accel_hip_allocate(size_t bytes, AccelHipBuffer* out);
ACCEL_HIP_API int accel_hip_free(AccelHipBuffer buffer);
ACCEL_HIP_API int accel_hip_copy_h2d(AccelHipBuffer dst, const void* src, size_t bytes);
ACCEL_HIP_API int accel_hip_copy_d2h(void* dst, AccelHipBuffer src, size_t bytes);
/* Uncounted reads/writes: the reference's host code reads device memory through raw
 * pointers without a counted copy (src/llama_model.cc:118,146,172,204). */
ACCEL_HIP_API int accel_hip_peek(void* dst, const void* device_src, size_t bytes);
ACCEL_HIP_API int accel_hip_poke(void* device_dst, const void* src, size_t bytes);
/* LiveDeviceAllocs (include/accel/device.h:133-135). */
ACCEL_HIP_API int64_t accel_hip_live_allocs(void);
/* Releases cached device blocks back to HIP (does not change live counts). */
ACCEL_HIP_API int accel_hip_trim(void);

/* ---- stats (src/runtime.cc:420-458) and packed-GEMM probes (src/sim_device.cc:379-385) --- */
ACCEL_HIP_API void accel_hip_get_stats(AccelHipStats* out);
ACCEL_HIP_API void accel_hip_reset_stats(void);
ACCEL_HIP_API int64_t accel_hip_packed_matmul_calls(void);
ACCEL_HIP_API int64_t accel_hip_packed_k_trips(void);
ACCEL_HIP_API void accel_hip_reset_packed_probes(void);

/* ---- compute ---------------------------------------------------------------------------- */
/* Device::MatMul (include/accel/device.h:81-82; src/sim_device.cc:185-196): row-major
 * C[m, n] = A[m, k] @ B[k, n], overwrites C (zeros when k == 0). m <= 16 and k < 32: fp32 MFMA;
 * otherwise six products of exact bf16 parts with fp32 results, summed again on the fp32 MFMA where the
 * parts cannot hold the operands (except on small grids of whole 64 x 64 tiles, where operands below
 * 2^-110 keep their bits down to 2^-134 and an infinity gives NaN). */
ACCEL_HIP_API int accel_hip_matmul(AccelHipBuffer a, AccelHipBuffer b, AccelHipBuffer c, int64_t m, int64_t k,
                                   int64_t n);
/* accel::MatMulQuantized (include/accel/runtime.h:124-125; src/sim_device.cc:541-602).
 * Device pointers; a NULL plane reads the float pointer. Either side may be quantized.
 * w = (float(q) - float(zero)) * scale at the plane's coordinate. m <= 16: the int8 GEMV
 * (VALU for m <= 2 and small matrices at m <= 4, else exact bf16-split products on the matrix
 * cores, from the group-interleaved copy where a large matrix has one, else in place). Above
 * that, an int8 weight with k >= 32 and n >= 8 runs on the bf16 matrix cores with the activation
 * split exactly into three bf16 parts (with a per-column or whole-tensor scale, no zero points,
 * k % 32 == 0 and n % 8 == 0 the weight is staged once as bf16); smaller ones on the fp32 MFMA
 * GEMM with the int8 panel dequantized in LDS. Infinite and NaN activations come out as fp32 products
 * of them do. Activations below 2^-110 keep their bits down to 2^-134 on the group-interleaved copy
 * and, above 16 rows, with the planes that are staged as bf16; elsewhere, where their lower bits show in
 * the result, they keep all of them. */
ACCEL_HIP_API int accel_hip_matmul_quantized(const float* a, const AccelHipQuantPlane* a_quant, const float* b,
                                             const AccelHipQuantPlane* b_quant, float* c, int64_t m, int64_t k,
                                             int64_t n);
/* Weight preparation. No counterpart in the reference, whose MatMulQuantized dequantizes each
 * panel on the fly (src/sim_device.cc:541-602); it belongs where the reference uploads and
 * binds the weight (UploadDequantized and BindConstant, src/ep.cc:843-900,1430-1463). Builds
 * now, on the library stream, the staged copies of the int8 weight b_quant ([k, n] at its
 * offset) that the matmuls otherwise build at the weight's first use: layouts is a mask of
 * ACCEL_HIP_STAGE_*, 0 for every layout this plane's form allows, also one that no kernel reads
 * at its size (the group-interleaved copy, k * n bytes, below 28 Mi weights: a mask leaves it out).
 * A copy lasts until the weight's allocation is freed or written. Refused
 * (ACCEL_HIP_RUNTIME_ERROR) during a graph capture; ACCEL_HIP_INVALID_ARGUMENT for a layout the
 * plane cannot take or a weight outside this library's heap. *staged (if not NULL) receives the
 * layouts built. */
#define ACCEL_HIP_STAGE_GEMV_TILES 1u  /* 8-column tiles: the int8 GEMV at m <= 2, and at m <= 4 for small matrices */
#define ACCEL_HIP_STAGE_GEMV_GROUPS 2u /* group-interleaved tiles: the bf16-split GEMV, 3 <= m <= 16, from 28 Mi weights */
#define ACCEL_HIP_STAGE_GEMM_BF16 4u   /* bf16 in MFMA operand order: the int8-weight GEMM, m > 16 */
#define ACCEL_HIP_STAGE_GEMM_SMALL 8u  /* bf16 in the small GEMM's operand order: m > 16, k <= 768 */
#define ACCEL_HIP_STAGE_ALL 15u
ACCEL_HIP_API int accel_hip_prepare_quantized(const AccelHipQuantPlane* b_quant, int64_t k, int64_t n,
                                              uint32_t layouts, uint32_t* staged);
/* Exact products (no reference counterpart as a switch; it selects the reference's own
 * arithmetic). When on, every matmul entry point sums each output in k order from zero with
 * each product rounded before its add, and dequantizes an int8 operand per element as
 * (float(q) - float(zero)) * scale: the bits of ReferenceMatMul / MatMulQuantized
 * (src/sim_device.cc:387-402,541-602). When off (the default) the GEMMs and GEMVs add in
 * their own order: within 2*gamma_K*(|A|@|B|) of the exact product. Process-wide;
 * accel_hip_exact_products() reads the setting (1 on, 0 off). */
ACCEL_HIP_API int accel_hip_set_exact_products(int32_t on);
ACCEL_HIP_API int32_t accel_hip_exact_products(void);
/* Fused forms of the two calls above (see AccelHipEpilogue). Count as one kernel matmul
 * each, like the unfused call; the caller notes its epilogue counters as the runtime does. */
ACCEL_HIP_API int accel_hip_matmul_fused(const float* a, const float* b, float* c, int64_t m, int64_t k, int64_t n,
                                         const AccelHipEpilogue* epilogue);
ACCEL_HIP_API int accel_hip_matmul_quantized_fused(const float* a, const AccelHipQuantPlane* a_quant, const float* b,
                                                   const AccelHipQuantPlane* b_quant, float* c, int64_t m, int64_t k,
                                                   int64_t n, const AccelHipEpilogue* epilogue);
/* No counterpart in the reference. accel_hip_matmul_quantized_fused for callers that cannot
 * allocate device memory: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc. Same arguments, checks, results and counters. It calls no hipMalloc,
 * hipFree or other allocating routine: the scratch its kernels need (split-K partial sums,
 * arrival counters, a dequantized operand for plane layouts the kernels do not index) comes
 * from one fixed 64 MiB device array per GPU, held until the process ends, and a call whose
 * scratch would exceed it returns ACCEL_HIP_INVALID_ARGUMENT. A staged GEMV copy of W is read
 * only if an earlier call built one (otherwise W is read in place). Every call on a GPU
 * shares that GPU's array: calls that overlap on one GPU race. */
ACCEL_HIP_API int accel_hip_matmul_quantized_fused_noalloc(const float* a, const AccelHipQuantPlane* a_quant,
                                                           const float* b, const AccelHipQuantPlane* b_quant, float* c,
                                                           int64_t m, int64_t k, int64_t n,
                                                           const AccelHipEpilogue* epilogue);
/* Device::Transpose (device.h:84-85; src/sim_device.cc:198-209): dst[j, i] = src[i, j]. */
ACCEL_HIP_API int accel_hip_transpose(AccelHipBuffer src, AccelHipBuffer dst, int64_t rows, int64_t cols);
/* Device::GemmEpilogue (device.h:87-92; src/sim_device.cc:211-245). bias may be NULL. */
ACCEL_HIP_API int accel_hip_gemm_epilogue(AccelHipBuffer c, int64_t m, int64_t n, float alpha,
                                          const AccelHipBuffer* bias, int32_t bias_rank, const int64_t* bias_shape,
                                          float beta, int32_t activation);
/* Device::Embedding (device.h:94-96; src/sim_embed.cc:9-20). An id outside [0, vocab) is
 * ACCEL_HIP_INVALID_ARGUMENT ("token id is outside the vocabulary"), detected on the device. */
ACCEL_HIP_API int accel_hip_embedding(AccelHipBuffer ids, int64_t id_offset, AccelHipBuffer table, AccelHipBuffer out,
                                      int64_t seq, int64_t hidden, int64_t vocab);
/* Embedding from an int8 table with one scale per row: out = float(q) * scale[id], the
 * same fl(q*s) value a float table quantized that way holds. No reference counterpart as
 * one call; used by the int8 Llama. */
ACCEL_HIP_API int accel_hip_embedding_q8(AccelHipBuffer ids, int64_t id_offset, const int8_t* table,
                                         const float* row_scale, AccelHipBuffer out, int64_t seq, int64_t hidden,
                                         int64_t vocab);
/* Device::RmsNorm (device.h:98-100; src/sim_rmsnorm.cc:7-20). */
ACCEL_HIP_API int accel_hip_rms_norm(AccelHipBuffer x, AccelHipBuffer weight, AccelHipBuffer y, int64_t rows,
                                     int64_t dim, float eps, int64_t row_offset);
/* Device::Rope (device.h:102-104; src/sim_rope.cc:5-21). */
ACCEL_HIP_API int accel_hip_rope(AccelHipBuffer states, AccelHipBuffer cos_table, AccelHipBuffer sin_table,
                                 int64_t seq, int64_t n_heads, int64_t head_dim, int64_t position);
/* Device::AppendCache (device.h:106-108; src/sim_cache.cc:8-13). */
ACCEL_HIP_API int accel_hip_append_cache(AccelHipBuffer src, AccelHipBuffer cache, int64_t seq, int64_t position,
                                         int64_t n_heads, int64_t head_dim);
/* Device::Attention (device.h:110-112; src/sim_attend.cc:9-46). scores is not used as
 * scratch by the HIP kernel but must still be large enough, as in the reference. Several rows
 * (seq > 1) with head_dim 64 or 128 form their scores and sums on the fp32 matrix cores in another
 * order than the reference's (rounding only) unless exact products are on. */
ACCEL_HIP_API int accel_hip_attention(AccelHipBuffer q, AccelHipBuffer k, AccelHipBuffer v, AccelHipBuffer scores,
                                      AccelHipBuffer out, int64_t seq, int64_t position, int64_t heads,
                                      int64_t kv_heads, int64_t head_dim);
/* Device::SiluMul (device.h:114-115; src/sim_silu.cc:8-13). */
ACCEL_HIP_API int accel_hip_silu_mul(AccelHipBuffer gate, AccelHipBuffer up, int64_t count);
/* Device::ResidualAdd (device.h:117-118; src/sim_add.cc:5-9). */
ACCEL_HIP_API int accel_hip_residual_add(AccelHipBuffer dest, AccelHipBuffer extra, int64_t count);
/* Device::SampleToken (device.h:120-124; src/sim_sample.cc:25-115). *rng_state is read
 * before and written after the draw, as the reference's xorshift32 state. */
ACCEL_HIP_API int accel_hip_sample_token(AccelHipBuffer logits, AccelHipBuffer chosen_ids, int64_t chosen_index,
                                         int64_t vocab, float temperature, uint32_t* rng_state, int32_t top_k);

/* ---- long contexts -----------------------------------------------------------------------
 * No reference counterpart: beside Rope, AppendCache and Attention above, what a long context needs.
 * These calls also take device memory of this GPU that another allocator made (a buffer with id 0); they
 * run on the library's stream like every other call, so data written elsewhere has to be there first.
 * Rows lie `row_stride` floats apart (0: dense). Exact products do not apply to them. */
enum { ACCEL_HIP_ROPE_HALF = 0, ACCEL_HIP_ROPE_INTERLEAVED = 1 }; /* pair i: dims (i, i + r/2), or (2i, 2i + 1) */
enum {
  ACCEL_HIP_ROPE_SCALE_NONE = 0,
  ACCEL_HIP_ROPE_SCALE_LINEAR = 1,    /* every frequency / factor */
  ACCEL_HIP_ROPE_SCALE_NTK = 2,       /* theta * factor^(r / (r - 2)) in theta's place */
  ACCEL_HIP_ROPE_SCALE_YARN = 3,      /* / factor below `slow` turns, as it is above `fast`, a ramp over the pairs between */
  ACCEL_HIP_ROPE_SCALE_WAVELENGTH = 4 /* the same borders, a ramp over the turns between */
};
/* How a model's rotary frequencies theta^(-2i/r) are scaled. A pair's turns are those it makes over
 * original_context positions; original_context, fast and slow are read by the last two kinds only
 * (usual borders: fast 32 and slow 1, and fast 4 and slow 1), factor by all but the first. */
typedef struct AccelHipRopeScaling {
  int32_t kind; /* ACCEL_HIP_ROPE_SCALE_* */
  double theta, factor, original_context, fast, slow;
} AccelHipRopeScaling;
/* Writes the rotary_dim / 2 frequencies (double, radians per position) of `scaling` into the device
 * buffer, once per model: it synchronizes and is refused in a capture. *magnitude (may be NULL)
 * receives what the rotated values are multiplied with: 0.1 ln(factor) + 1 for YaRN with a factor
 * above 1, otherwise 1. */
ACCEL_HIP_API int accel_hip_rope_frequencies(const AccelHipRopeScaling* scaling, int64_t rotary_dim,
                                             AccelHipBuffer frequencies, float* magnitude);
/* Rotates the first rotary_dim (even) dims of every head by the angle position_s * frequency_i and
 * multiplies them with magnitude; the other dims come out as they are. states and out are rows of
 * n_heads * head_dim floats (and row_stride apart both; what lies behind a row's heads is left alone):
 * the query and key heads of a fused projection's rows turn in one call. out may be states itself, and
 * may not overlap it otherwise, nor the frequencies and positions. position_s is position + s, or position +
 * positions[s] where positions (int32 [seq]) has data; it counts up to 2^32. Angles are formed in 64 bits
 * (within 2^-24 radians up to 2^27 of them, within 2^-20 at 2^31), their cos and sin in fp32. */
ACCEL_HIP_API int accel_hip_rope_scaled(AccelHipBuffer states, AccelHipBuffer out, AccelHipBuffer frequencies,
                                        AccelHipBuffer positions, int64_t seq, int64_t n_heads, int64_t head_dim,
                                        int64_t row_stride, int64_t rotary_dim, int32_t layout, int64_t position,
                                        float magnitude);
/* A layer's KV cache in 8 bits: codes int8 [capacity, kv_heads, head_dim] and one fp32 scale for each
 * block of `block` tokens and head, [ceil(capacity / block), kv_heads], for keys and values. A value is
 * code * scale, and scales are not negative. block is a power of two up to 256, head_dim at most 256. */
typedef struct AccelHipCacheQ8 {
  AccelHipBuffer k, v, k_scale, v_scale;
  int64_t capacity, kv_heads, head_dim, block;
} AccelHipCacheQ8;
/* AppendCache into the 8-bit cache: rows [position, position + seq) of k and v (fp32, kv_heads *
 * head_dim a row). Each touched block and head gets the scale max|x| / 127 of its new rows. A block that
 * has rows before `position` keeps the scale it has where that is larger, also where only rows that are
 * written over now (a rejected draft) needed it; when it grows, the codes of the rows before become the
 * nearest code of code * old / new. A block written from its start is new. A code is the nearest integer to
 * x / scale (the true quotient; ties to even), within -127 .. 127, where only a scale below 2^-126 leaves
 * it. Rows of the block from position + seq on do not count any more. A NaN or an infinity makes its block's
 * scale of that head NaN, and all that is read of it, until the block is written from its start. The planes
 * may not overlap one another or k and v. */
ACCEL_HIP_API int accel_hip_append_cache_q8(AccelHipBuffer k, AccelHipBuffer v, const AccelHipCacheQ8* cache,
                                            int64_t seq, int64_t position, int64_t row_stride);
/* Rows [first, first + count) of the 8-bit cache as fp32 [count, kv_heads, head_dim], code * scale
 * rounded once. k_out or v_out without data leaves that plane out; they may overlap neither one another
 * nor the codes and scales that are read. */
ACCEL_HIP_API int accel_hip_read_cache_q8(const AccelHipCacheQ8* cache, int64_t first, int64_t count,
                                          AccelHipBuffer k_out, AccelHipBuffer v_out);
/* Attention (as accel_hip_attention: causal, grouped heads, 1 / sqrt(head_dim)) over the 8-bit cache,
 * whose rows up to position + seq are written. With window > 0 the row at p sees the keys t <= p with
 * t > p - window or t < sinks; with window 0 every t <= p. q's rows are row_stride apart, out is dense
 * and may not overlap q or the cache. head_dim is at most 256, kv_heads * head_dim at most 2^24.
 * Rounding: queries and softmax weights enter the products with 22 bits (a query relative to its row's
 * largest value, a weight to the largest), sums are fp32. A row whose query is not finite, or that sees a
 * scale that is not finite or a score past the largest float, is NaN. Inside a capture whose workspace was
 * not grown before (by the same call, once), the key range is not divided over workgroups. */
ACCEL_HIP_API int accel_hip_attention_q8(AccelHipBuffer q, const AccelHipCacheQ8* cache, AccelHipBuffer out,
                                         int64_t seq, int64_t position, int64_t heads, int64_t row_stride,
                                         int64_t window, int64_t sinks);
/* Attention over an fp32 cache k, v [>= position + seq, kv_heads, head_dim] with a sliding window: the
 * row at p sees the keys t <= p with t > p - window or t < sinks (window 0: every t <= p). Keys that no
 * row sees count for nothing, NaN included. q's rows are row_stride apart, out is dense and may not
 * overlap q, k or v. Sizes, captures and queries as above. Rounding: with many rows (more than 16 of a
 * key head, over a long range) queries, keys and values enter the products with 22 bits of their row's
 * largest value and weights with 22 bits of the largest; otherwise in fp32, where a weight below 2^-126 of the
 * largest may count as 0, and the sums of a row that gives a value from 2^96 on a weight are held times 2^-64. A key
 * or value that is not finite makes the rows that see it NaN, and so does a score past the largest float. */
ACCEL_HIP_API int accel_hip_attention_window(AccelHipBuffer q, AccelHipBuffer k, AccelHipBuffer v, AccelHipBuffer out,
                                             int64_t seq, int64_t position, int64_t heads, int64_t kv_heads,
                                             int64_t head_dim, int64_t row_stride, int64_t window, int64_t sinks);

/* ---- many requests from one cache --------------------------------------------------------
 * No reference counterpart: what serves a batch of requests of different lengths. Keys and values lie in
 * pages that any request may own; how long each request is stays in device memory, so that a captured step
 * can be replayed while requests grow. Memory and stream as for long contexts above; exact products do not
 * apply. int32 buffers are aligned to 4 bytes. */
enum { ACCEL_HIP_CACHE_F32 = 0, ACCEL_HIP_CACHE_F16 = 1 };
/* The pages of a layer: k and v are [pages, page, kv_heads, head_dim] of `type`. page is a power of two in
 * 16 .. 256, head_dim at most 256. Slot s is row s % page of page s / page. */
typedef struct AccelHipCachePaged {
  AccelHipBuffer k, v;
  int32_t type; /* ACCEL_HIP_CACHE_* */
  int64_t pages, page, kv_heads, head_dim;
} AccelHipCachePaged;
/* One step of a batch. The new tokens of all requests are rows that lie one behind the other: those of
 * request r are starts[r] .. starts[r + 1] - 1, its first token is its token seen[r]. table[r] are the pages
 * of its tokens in order. rows is what there is room for; rows past starts[requests] are padding. Where starts
 * descend, the output's rows (no others) hold anything. longest is the most new rows of one request where the
 * host knows it, otherwise 0: it chooses kernels, not results. slots, where it has data, are the rows' slots as
 * accel_hip_batch_tables wrote them and accel_hip_append_paged took them: a row without one is not in the cache,
 * and accel_hip_attention_paged gives it NaN. The other calls do not read it. */
typedef struct AccelHipBatch {
  AccelHipBuffer seen;   /* int32 [requests] */
  AccelHipBuffer starts; /* int32 [requests + 1] */
  AccelHipBuffer table;  /* int32 [requests, width] */
  int64_t requests, rows, width, longest;
  AccelHipBuffer slots;  /* int32 [rows], or none */
} AccelHipBatch;
/* The pages that no request owns: the first state[0] entries of `stack`, the last of them taken first. */
typedef struct AccelHipPagePool {
  AccelHipBuffer stack; /* int32 [pages] */
  AccelHipBuffer state; /* int32 [2]: pages on the stack; requests that the last step had no page for */
  int64_t pages, page;
} AccelHipPagePool;
/* The tables of one step. Request r has lengths[r] tokens in the cache and counts[r] new ones (below 0: 0; what
 * is past `rows` does not count). Writes starts and seen (the lengths) of the batch; for the pages that the new
 * tokens begin, in the order of the requests, the pages from the stack's end into the table; for each row its
 * position and its slot (padding: 0 and -1); lengths_after (lengths + counts) and state_after, which may be
 * `lengths` and the pool's state themselves. A request whose new pages are not all there, nor those of the requests
 * before it, or do not fit its table row, takes none: its rows have slot -1, its missing entries become -1,
 * its length stays, and it is counted in state_after[1]. Its first new tokens may belong on a page that it has: they
 * are not written there, so what the page held before, another request's tokens perhaps, is still there, and only the
 * batch's slots keep attention from it; without them all its rows of the output mean nothing. Who needs no new page
 * is always served. Other
 * outputs may overlap neither one another nor the inputs. More than 2048 requests or 4096 rows take a workspace,
 * which a call before a capture has to have grown. */
ACCEL_HIP_API int accel_hip_batch_tables(AccelHipBuffer counts, AccelHipBuffer lengths, const AccelHipPagePool* pool,
                                         const AccelHipBatch* batch, AccelHipBuffer slots, AccelHipBuffer positions,
                                         AccelHipBuffer lengths_after, AccelHipBuffer state_after);
/* Cuts requests short: a request with keep[r] (below 0: 0) less than lengths[r] keeps that many tokens (0: it has
 * ended; drafts that were rejected go the same way). The pages past them, in the order of the requests and
 * of their tokens, go onto the pool's stack, their table entries become -1 and lengths[r] becomes keep[r].
 * Entries that are no page are left out; a page that two requests share goes on once for each, so it is taken
 * out of one's table first. batch gives requests, width and the table; pool's state[1] stays. */
ACCEL_HIP_API int accel_hip_release_pages(AccelHipBuffer keep, AccelHipBuffer lengths, const AccelHipPagePool* pool,
                                          const AccelHipBatch* batch);
/* Rows of k and v (fp32, kv_heads * head_dim a row, row_stride apart) into their slots (int32 [rows]),
 * rounded to nearest even; past the largest f16 that is an infinity. Rows whose slot is outside the cache are
 * left out. Two rows may not have the same slot. The planes may overlap neither one another nor k, v and slots. */
ACCEL_HIP_API int accel_hip_append_paged(AccelHipBuffer k, AccelHipBuffer v, const AccelHipCachePaged* cache,
                                         AccelHipBuffer slots, int64_t rows, int64_t row_stride);
/* Causal grouped-query attention (1 / sqrt(head_dim)) of every request's new rows over its own tokens, whose
 * keys and values, the new rows' too, are in the cache: the row at p sees the keys t <= p, with window > 0 those
 * with t > p - window. q's rows are row_stride floats apart, out is dense and may not overlap q, the cache
 * or the batch; padding rows of it stay as they were. Rounding: with an f16 cache, and with many rows
 * (over fp32), queries, softmax weights and fp32 keys and values enter the products with 22 bits (of their row's
 * largest value, the weights of the largest), otherwise with all, where a weight below 2^-126 of the largest may count
 * as 0; sums are fp32 (of a row that gives a value from 2^96 on a weight, times 2^-64). A row whose query is not finite,
 * that sees a key or value that is not, a score past the largest float, or a token without a page (an entry of
 * the table that is none, a token past the table's width), or whose slot (where the batch has slots) is outside the
 * cache, is NaN; a value that no row sees has no say.
 * Inside a capture whose workspace was not grown before (by the same call, once), key ranges are not divided
 * over workgroups. */
ACCEL_HIP_API int accel_hip_attention_paged(AccelHipBuffer q, const AccelHipCachePaged* cache, const AccelHipBatch* batch,
                                            AccelHipBuffer out, int64_t heads, int64_t row_stride, int64_t window);
/* The same over whole prompts that are not in a cache: the keys and values of request r are rows starts[r] ..
 * starts[r + 1] - 1 of k and v (fp32, kv_heads * head_dim a row, kv_stride floats apart; 0: dense), and its
 * positions begin at 0. seen, table and width of the batch are not read. q, k and v may be parts of the same rows. */
ACCEL_HIP_API int accel_hip_attention_packed(AccelHipBuffer q, AccelHipBuffer k, AccelHipBuffer v,
                                             const AccelHipBatch* batch, AccelHipBuffer out, int64_t heads,
                                             int64_t kv_heads, int64_t head_dim, int64_t row_stride, int64_t kv_stride,
                                             int64_t window);

/* ---- timing ----------------------------------------------------------------------------- */
/* Milliseconds between two HIP events recorded on the library's stream around `iters`
 * back-to-back calls of fn(user); returns < 0 on failure. Used by bench.py. */
typedef int (*AccelHipWorkFn)(void* user);
ACCEL_HIP_API double accel_hip_time_ms(AccelHipWorkFn fn, void* user, int32_t iters);
/* Records/reads events on the library's stream (for timing regions driven from Python), in
 * slots 0 .. 15. Recorded during a capture (accel_hip_capture_begin), the event becomes a node
 * of the graph, recorded each time the graph is replayed, and stays timeable. */
ACCEL_HIP_API int accel_hip_event_record(int32_t slot);
ACCEL_HIP_API double accel_hip_event_elapsed_ms(int32_t start_slot, int32_t end_slot);

/* ---- HIP graphs --------------------------------------------------------------------------
 * Captures the kernels that the calls between begin and end enqueue on the library stream
 * into an executable graph, replayed by accel_hip_graph_launch. Calls made during a capture
 * must not synchronize (no counted copies, allocations or first-use workspace growth):
 * warm them up once before capturing. No reference counterpart (the reference runs on the
 * host); used to replay a fixed launch sequence without host launch overhead. */
ACCEL_HIP_API int accel_hip_capture_begin(void);
ACCEL_HIP_API int accel_hip_capture_end(void** graph_exec);
ACCEL_HIP_API int accel_hip_graph_launch(void* graph_exec, int32_t times);
ACCEL_HIP_API int accel_hip_graph_destroy(void* graph_exec);

#ifdef __cplusplus
}
#endif

#endif /* ACCEL_HIP_H_ */
