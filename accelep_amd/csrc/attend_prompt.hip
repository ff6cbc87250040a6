// Attention of many rows (a prompt) over the 8-bit cache and in a window over an fp32 one, on the f16
// matrix cores: queries, softmax weights and fp32 keys and values as two f16 parts (22 bits), codes as
// one, scales and powers of two beside them in fp32.
//
// One workgroup per (128 rows of a key head, key range): four waves of 32 rows share each tile of keys,
// which is brought to f16 once, through LDS, while the tile before is worked on (two buffers, one
// barrier a tile). Lane (j, g) = (lane % 32, lane / 32) serves row j. Per 32 keys
//  * S^T = K Q^T on v_mfma_f32_32x32x16_f16, keys as rows: the lane's 16 results are the scores of keys
//    8a + 4g + b (a, b < 4) of row j, so a row's softmax needs one exchange between two lanes;
//  * O^T += V^T P^T: those scores are the lane's own k-slots of P^T if slot e of 16 keys is key
//    (e % 4) + 8 (e / 4) + 4g, and the value operand is read transposed from the row-major tile
//    (ds_read_b64_tr_b16 gives a lane four keys of one dim).
// An fp32 row enters as its parts times a power of two, whose inverse takes the place of a block's scale:
// 2^9 for rows whose largest magnitude lies in [2^-6, 2^6) (or keys that are zero), which keeps 22 bits of all
// of them, and a tile of such rows has one scale; otherwise one from the row's own largest magnitude (of values
// that are zero 2^127, so that they take no bits from others). A row that is not finite has a NaN for a scale
// and zeros for values.
//
// Bound: the matrix cores at the clock that they leave themselves (1.7-1.9 GHz under this load), with the
// softmax and the split of its weights between their phases. 2048 rows from position 4097 on, 32 heads on
// 8 of 128: 316 us, 172 GFLOP in two products, 1.09 PFLOP/s of f16; the matrix cores are busy 64 % of the
// cycles. fp32, 4096 rows in a window of 1024: 234 us, 60 GFLOP in three products, 0.77 PFLOP/s; busy
// 41 %, since each tile of keys is also split there, by every workgroup that reads it.
// Dims are padded to 64, 128 or 256: the 8-bit case takes 306 us with heads of 80, 310 of 96, 713 of 192 and
// 711 of 256 (198 of 64), where the registers of a wave no longer hold queries, sums and staging.
// Pieces of 8 codes, whose LDS writes have no bank conflicts (those of 16 have, 8 % of the cycles), took
// 311 us; fp32 in workgroups of eight waves 225, which a variant of its own was not worth.
#include "attend_common.h"

namespace accel_hip {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kWaveRows = 32;
constexpr float kCommonScale = 0x1p9f;
constexpr float kFarKey = 0x1p90f;  // scores are below 2^37 before the scales
constexpr float kBackFirst = 0x1p60f;
constexpr uint32_t kCommonLow = 121u << 23, kCommonHigh = 133u << 23;  // bits of 2^-6 and 2^6
constexpr int kRows = kWaves * kWaveRows;
typedef short s4 __attribute__((ext_vector_type(4)));

struct PromptArgs {
  const void* k;  // codes or floats
  const void* v;
  const float* k_scale;  // 8-bit only
  const float* v_scale;
  int32_t block_shift, splits, tiles;
  AttendPartial partial;
};

// What the registers are shared out for. Head dim 64 fits three waves at 16-byte loads, and needs to be held to
// it with a scale per key (blocks of 16, 1024 rows: 42.3 us, with 173 registers and two waves 42.6).
constexpr int WavesPerSimd(int dp, int load) { return dp > 128 ? 1 : dp > 64 || load < 16 ? 2 : 3; }

// kF32: an fp32 cache. kLoad: bytes that may be loaded at once (16, 4 or 1; 16 or 4 for fp32).
// kUniform: a block holds whole tiles, one scale each.
template <int DP, bool kF32, int kLoad, bool kUniform>
__global__ __launch_bounds__(kThreads, WavesPerSimd(DP, kLoad)) void AttendPromptKernel(AttendArgs a, PromptArgs b) {
  constexpr int kParts = kF32 ? 2 : 1;
  constexpr int kKeys = kF32 ? 32 : 64;
  constexpr int kSub = kKeys / 32;
  constexpr int kSteps = DP / 16;
  constexpr int kDims = DP / 32;
  constexpr int kKStride = DP + 8;   // halves: 8 key rows' 16-byte pieces fall into different banks
  constexpr int kVStride = DP + 32;  // and so do 4 key rows' 64-byte pieces (two tile reads)
  constexpr int kChunks = kF32 ? DP / 32 : kKeys * DP / 16 / kThreads;  // 16-byte pieces of a plane a thread stages
  __shared__ __align__(16) _Float16 kt[2][kParts][kKeys][kKStride];
  __shared__ __align__(16) _Float16 vt[2][kParts][kKeys][kVStride];
  __shared__ __align__(16) float sk[2][kKeys];
  __shared__ __align__(16) float sv[2][kKeys];
  __shared__ int odd[3];  // fp32: the tile has rows of scales of their own
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 31;
  const int g = lane >> 5;
  const int32_t kv = static_cast<int32_t>(blockIdx.x) % a.kv_heads;
  const int32_t rest = static_cast<int32_t>(blockIdx.x) / a.kv_heads;
  const int32_t split = rest % b.splits;
  const int32_t tile = b.tiles - 1 - rest / b.splits;  // the rows with the most keys first
  const int32_t group = a.heads / a.kv_heads;
  const int32_t rows = a.seq * group;
  const int32_t r0 = tile * kRows;
  const KeyRange<kKeys> range(a, r0, min(r0 + kRows, rows), group);
  const int32_t per = (range.steps + b.splits - 1) / b.splits;
  const int32_t begin = min(range.steps, split * per);
  const int32_t end = min(range.steps, begin + per);
  const int32_t w0 = r0 + wave * kWaveRows;  // the wave's rows
  const int32_t row = min(w0 + j, rows - 1);
  const int32_t s = row / group;
  const int32_t head = kv * group + (row - s * group);
  const int32_t p_row = w0 + j < rows ? a.position + s : -1;
  const int32_t pw_first = a.position + min(w0, rows - 1) / group;
  const int32_t pw_last = w0 < rows ? a.position + (min(w0 + kWaveRows, rows) - 1) / group : -1;
  const bool full_rows = w0 + kWaveRows <= rows;
  const int64_t kv_row = static_cast<int64_t>(a.kv_heads) * a.dim;

  // ---- staging: a thread's pieces of the next tile, from memory to registers and on to LDS ----
  uint4 kreg[kChunks], vreg[kChunks];
  float ks_next = 0.f, vs_next = 0.f;  // each wave has the scales of all the tile's keys
  bool marked_next = false;            // and a large one among them
  const auto fetch_plane = [&](const void* base, int32_t t0, uint4 (&x)[kChunks]) {
    if constexpr (kF32) {
      // A row past the range reads its last one, a piece past a head's dims its last: both are not used.
      const float* p = static_cast<const float*>(base) + min(t0 + tid / 8, range.high - 1) * kv_row +
                       static_cast<int64_t>(kv) * a.dim;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int d = 8 * (tid % 8 + 8 * (i / 2)) + 4 * (i % 2);
        if (kLoad == 16) {
          x[i] = *reinterpret_cast<const uint4*>(p + min(d, a.dim - 4));
        } else {
          const auto at = [&](int e) { return __float_as_uint(p[min(d + e, a.dim - 1)]); };
          x[i] = make_uint4(at(0), at(1), at(2), at(3));
        }
      }
    } else {
      const CodeRows rows = RowsFrom(static_cast<const int8_t*>(base) + static_cast<int64_t>(kv) * a.dim,
                                     static_cast<int32_t>(kv_row), a.dim, t0, range.high);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int key = (tid + i * kThreads) / (DP / 16);
        const int d = 16 * ((tid + i * kThreads) % (DP / 16));
        uint32_t w[4];
        LoadCodes<4, kLoad>(rows, static_cast<uint32_t>(key * static_cast<int32_t>(kv_row) + d), w);
        x[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  };
  const auto scale_at = [&](const float* scale, int32_t t) {
    return scale[static_cast<int64_t>(min(t, range.high - 1) >> b.block_shift) * a.kv_heads + kv];
  };
  const auto fetch = [&](int32_t t0) {
    fetch_plane(b.k, t0, kreg);
    fetch_plane(b.v, t0, vreg);
    if (!kF32) {
      const int32_t t = kUniform ? t0 : t0 + (tid & (kKeys - 1));
      ks_next = scale_at(b.k_scale, t);
      vs_next = scale_at(b.v_scale, t);
    }
  };
  // Writes a thread's pieces of one plane; tile row `key` begins at dst + key * stride, its second part
  // `part` halves later. least: 0, or 1 for values, the bits of what a row of zeros counts as.
  const auto put_plane = [&](const uint4 (&x)[kChunks], _Float16* dst, int stride, int part, float& row_back, int slot,
                             uint32_t least) {
    if (kF32) {
      // The row's largest magnitude: of the bits as signed numbers for its positive values, as unsigned
      // ones for its negative.
      int32_t pos = 0;
      uint32_t neg = 0;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        pos = max(max(pos, max(static_cast<int32_t>(x[i].x), static_cast<int32_t>(x[i].y))),
                  max(static_cast<int32_t>(x[i].z), static_cast<int32_t>(x[i].w)));
        neg = max(max(neg, max(x[i].x, x[i].y)), max(x[i].z, x[i].w));
      }
      uint32_t top = max(static_cast<uint32_t>(pos), neg & 0x7fffffffu);
      top = max(top, XorLane<1>(top));
      top = max(top, XorLane<2>(top));
      top = max(max(top, XorLane<4>(top)), least);
      float scale = kCommonScale, back = 1.f / kCommonScale;
      const bool common = top == 0 || (top >= kCommonLow && top < kCommonHigh);
      if (!__all(common)) {
        odd[slot] = 1;
        scale = RowScale(top);
        back = top >= 0x7f800000u ? NAN : 1.f / scale;
      }
      row_back = back;
      h8* p = reinterpret_cast<h8*>(dst + (tid / 8) * stride + 8 * (tid % 8));
#pragma unroll
      for (int i = 0; i < kChunks; i += 2) {
        const uint4 a0 = x[i], a1 = x[i + 1];
        h2 hi[4], lo[4];
        SplitF16(__uint_as_float(a0.x) * scale, __uint_as_float(a0.y) * scale, hi[0], lo[0]);
        SplitF16(__uint_as_float(a0.z) * scale, __uint_as_float(a0.w) * scale, hi[1], lo[1]);
        SplitF16(__uint_as_float(a1.x) * scale, __uint_as_float(a1.y) * scale, hi[2], lo[2]);
        SplitF16(__uint_as_float(a1.z) * scale, __uint_as_float(a1.w) * scale, hi[3], lo[3]);
        p[4 * i] = Join(hi[0], hi[1], hi[2], hi[3]);
        p[4 * i + part / 8] = Join(lo[0], lo[1], lo[2], lo[3]);
      }
      if (top >= 0x7f800000u) {  // written again: zeros
        const _Float16 z = 0;
#pragma unroll
        for (int i = 0; i < kChunks; i += 2) p[4 * i] = p[4 * i + part / 8] = h8{z, z, z, z, z, z, z, z};
      }
    } else {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int key = (tid + i * kThreads) / (DP / 16);
        const int d = 16 * ((tid + i * kThreads) % (DP / 16));
        const uint32_t x0 = x[i].x ^ 0x80808080u, x1 = x[i].y ^ 0x80808080u;
        const uint32_t x2 = x[i].z ^ 0x80808080u, x3 = x[i].w ^ 0x80808080u;
        h8* p = reinterpret_cast<h8*>(dst + key * stride + d);
        p[0] = Join(CodesLow(x0), CodesHigh(x0), CodesLow(x1), CodesHigh(x1));
        p[1] = Join(CodesLow(x2), CodesHigh(x2), CodesLow(x3), CodesHigh(x3));
      }
    }
  };
  // A value scale that is not finite moves to its keys, as NaN: the scores of the rows that see them are
  // NaN then, and a weight of 0 stays one.
  const auto move_nan = [](float& key, float& value) {
    if (!(fabsf(value) < INFINITY)) {
      key = NAN;
      value = 0.f;
    }
  };
  const auto put = [&](int buf, int slot) {
    float k_back = 1.f, v_back = 1.f;
    put_plane(kreg, &kt[buf][0][0][0], kKStride, kKeys * kKStride, k_back, slot, 0);
    put_plane(vreg, &vt[buf][0][0][0], kVStride, kKeys * kVStride, v_back, slot, 1);
    if (kF32) {
      move_nan(k_back, v_back);
      if (tid % 8 == 0) {
        sk[buf][tid / 8] = k_back;
        sv[buf][tid / 8] = v_back;
      }
    } else {
      move_nan(ks_next, vs_next);
      marked_next = __any(ks_next >= kFarKey || vs_next >= kLargeScale);
      if (!kUniform && tid < kKeys) {
        sk[buf][tid] = ks_next;
        sv[buf][tid] = vs_next;
      }
    }
  };
  if (begin < end) fetch(range.Key(begin));

  // ---- the rows' queries ----
  h8 qh[kSteps], ql[kSteps];
  float row_back;  // a power of two: takes the row's scale out of its scores again
  {
    const float* q = a.q + s * a.q_stride + static_cast<int64_t>(head) * a.dim;
    const bool vec = QueryVec(a);
    float x[kSteps][8];
    uint32_t top = 0;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) LoadQuery(a, q, 16 * st + 8 * g, vec, x[st]);
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[st][e]) & 0x7fffffffu);
    top = max(top, XorLane<32>(top));
    const bool bad = top >= 0x7f800000u;
    const float scale = RowScale(top);
    row_back = 1.f / scale;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      h2 hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        SplitF16Nearest(bad ? NAN : x[st][2 * e] * scale, bad ? NAN : x[st][2 * e + 1] * scale, hi[e], lo[e]);
      qh[st] = Join(hi[0], hi[1], hi[2], hi[3]);
      ql[st] = Join(lo[0], lo[1], lo[2], lo[3]);
    }
  }

  float m = -INFINITY, l = 0.f, top = 0.f;
  int32_t power = kPowerMax;
  f16v acc[kDims];
#pragma unroll
  for (int t = 0; t < kDims; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

  if (tid < 3) odd[tid] = 0;
  __syncthreads();
  if (begin < end) put(0, 0);
  float ks = ks_next, vs = vs_next;
  bool marked = marked_next;
  for (int32_t u = begin; u < end; ++u) {
    const int buf = (u - begin) & 1;
    const int32_t t0 = range.Key(u);
    __syncthreads();
    if (kF32 && tid == 0) odd[(u + 2 - begin) % 3] = 0;  // next written behind the next barrier
    if (u + 1 < end) fetch(range.Key(u + 1));
    __builtin_amdgcn_sched_barrier(0);
    const int32_t last = t0 + kKeys - 1;
    const bool none = t0 > pw_last || (last <= pw_first - a.window && t0 >= a.sinks);
    if (!none) {  // uniform over the wave
      const bool whole = full_rows && last <= pw_first && (t0 > pw_last - a.window || last < a.sinks);
      f16v st[kSub];
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[h][r] = 0.f;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        // Neighbouring instructions add to different sums.
        h8 k8[kSub];
#pragma unroll
        for (int h = 0; h < kSub; ++h) {
          k8[h] = *reinterpret_cast<const h8*>(&kt[buf][0][32 * h + j][16 * step + 8 * g]);
          st[h] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[h], qh[step], st[h], 0, 0, 0);
        }
#pragma unroll
        for (int h = 0; h < kSub; ++h) st[h] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[h], ql[step], st[h], 0, 0, 0);
        if (kF32) {
          const h8 k8l = *reinterpret_cast<const h8*>(&kt[buf][kParts - 1][j][16 * step + 8 * g]);
          st[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8l, qh[step], st[0], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      const bool one_scale = kUniform || (kF32 && odd[(u - begin) % 3] == 0);  // uniform
      float c = a.factor;
      if (one_scale) {
        c *= row_back * (kF32 ? 1.f / kCommonScale : ks);
      } else {
        if (kF32 || marked) {
          // A key's scale could carry the product past the range: the row's scale out first, as far as that
          // itself cannot.
          c *= row_back > kBackFirst ? row_back / kBackFirst : 1.f;
#pragma unroll
          for (int h = 0; h < kSub; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[h][r] *= fminf(row_back, kBackFirst);
        } else {
          c *= row_back;
        }
#pragma unroll
        for (int h = 0; h < kSub; ++h)
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const f4 f = *reinterpret_cast<const f4*>(&sk[buf][32 * h + 8 * r4 + 4 * g]);
#pragma unroll
            for (int e = 0; e < 4; ++e) st[h][4 * r4 + e] *= f[e];
          }
      }
      if (!whole) {
#pragma unroll
        for (int h = 0; h < kSub; ++h)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            st[h][r] = Sees(a, p_row, t0 + 32 * h + (r & 3) + 8 * (r >> 2) + 4 * g) ? st[h][r] * c : -INFINITY;
        c = 1.f;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[h][r]);
      mx = fmaxf(mx, XorLane<32>(mx)) * c;
      // The reference moves only when a score passes it by 8, so the sums are seldom scaled. (fp32 rows'
      // powers of two stay below 2^115, and a weight of 2^8 times that in range.)
      const float slack = Slack(!kF32 && marked);
      const float m_old = m;
      if (mx > m + slack) m = mx;
      const float base = m == -INFINITY ? 0.f : m;
      const float corr = __builtin_amdgcn_exp2f(m_old - base);
      float sum = 0.f, below = base;
      if (__any(fabsf(base) >= kFarScore)) {
#pragma unroll
        for (int h = 0; h < kSub; ++h)
#pragma unroll
          for (int r = 0; r < 16; ++r) st[h][r] = st[h][r] * c - base;
        c = 1.f;
        below = 0.f;
      }
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          st[h][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[h][r], c, -below));
          sum += st[h][r];
        }
      l = l * corr + sum;
      // The weights times the values' scales, and their largest.
      const float v_scale = kF32 ? 1.f / kCommonScale : vs;
      float tile_top = 0.f;
      if (one_scale) {
        tile_top = __builtin_amdgcn_exp2f(mx - base) * v_scale;
      } else {
#pragma unroll
        for (int h = 0; h < kSub; ++h)
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const f4 f = *reinterpret_cast<const f4*>(&sv[buf][32 * h + 8 * r4 + 4 * g]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              st[h][4 * r4 + e] *= f[e];
              tile_top = fmaxf(tile_top, fabsf(st[h][4 * r4 + e]));
            }
          }
        tile_top = fmaxf(tile_top, XorLane<32>(tile_top));
      }
      top = fmaxf(top * corr, tile_top);
      const int32_t power_old = power;
      power = WeightPower(top, power);
      const float again = ldexpf(corr, power - power_old);
      if (__any(again != 1.f)) {
#pragma unroll
        for (int t = 0; t < kDims; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[t][r] *= again;
      }
      if (one_scale) {
        const float f = ldexpf(v_scale, power);
        if (!kF32 && __any(!(f < 0x1p100f))) {  // a block that is far larger than the sum so far: in two steps
#pragma unroll
          for (int h = 0; h < kSub; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[h][r] = ldexpf(st[h][r] * v_scale, power);
        } else {
#pragma unroll
          for (int h = 0; h < kSub; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[h][r] *= f;
        }
      } else {
#pragma unroll
        for (int h = 0; h < kSub; ++h)
#pragma unroll
          for (int r = 0; r < 16; ++r) st[h][r] = ldexpf(st[h][r], power);
      }
      // O^T += V^T P^T, 16 keys at a time.
      __builtin_amdgcn_s_setprio(1);
      const _Float16* vrow = &vt[buf][0][4 * g + ((lane & 15) >> 2)][16 * ((lane >> 4) & 1) + 4 * (lane & 3)];
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int k16 = 0; k16 < 2; ++k16) {
          h2 hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) SplitF16(st[h][8 * k16 + 2 * e], st[h][8 * k16 + 2 * e + 1], hi[e], lo[e]);
          const h8 ph = Join(hi[0], hi[1], hi[2], hi[3]), pl = Join(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
          for (int t0 = 0; t0 < kDims; t0 += 2) {
            const auto read = [&](int t, int part) {
              const _Float16* p = vrow + part * kKeys * kVStride + (32 * h + 16 * k16) * kVStride + 32 * t;
              const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
              const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 8 * kVStride));
              return __builtin_bit_cast(h8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            const h8 v0 = read(t0, 0), v1 = read(t0 + 1, 0);
            acc[t0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, ph, acc[t0], 0, 0, 0);
            acc[t0 + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, ph, acc[t0 + 1], 0, 0, 0);
            acc[t0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, pl, acc[t0], 0, 0, 0);
            acc[t0 + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, pl, acc[t0 + 1], 0, 0, 0);
            if (kF32) {
              acc[t0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(read(t0, kParts - 1), ph, acc[t0], 0, 0, 0);
              acc[t0 + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(read(t0 + 1, kParts - 1), ph, acc[t0 + 1], 0, 0, 0);
            }
          }
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (u + 1 < end) {
      put(buf ^ 1, (u + 1 - begin) % 3);
      ks = ks_next;
      vs = vs_next;
      marked = marked_next;
    }
  }

  // acc[t][r] is O^T[dim 32t + 8 (r / 4) + 4g + r % 4][row j].
  l = l + XorLane<32>(l);
  if (w0 + j >= rows) return;
  const bool far = power < kFarPower;
  const int32_t down = far ? -power - kFarShift : -power;
  const float up = far ? kFarUp : 1.f;
  const int64_t out_row = static_cast<int64_t>(s) * a.heads + head;
  float* dst = a.out + out_row * a.dim;
  bool vec = a.dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  if (b.splits > 1) {
    const int64_t at = out_row * b.splits + split;
    dst = b.partial.o + at * PartialDims(a.dim);
    vec = true;
    if (g == 0) {
      b.partial.ml[2 * at] = m;
      b.partial.ml[2 * at + 1] = far ? -l : l;
    }
  }
#pragma unroll
  for (int t = 0; t < kDims; ++t)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int d = 32 * t + 8 * r4 + 4 * g;
      f4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = ldexpf(acc[t][4 * r4 + e], down);
        if (b.splits == 1) o[e] = __fdiv_rn(o[e], l) * up;
      }
      if (vec) {
        if (d < a.dim) *reinterpret_cast<f4*>(dst + d) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < a.dim) dst[d + e] = o[e];
      }
    }
}

template <int DP, bool kF32>
void LaunchPrompt(const AttendArgs& a, const PromptArgs& b, int load, hipStream_t stream) {
  const dim3 grid(GridOf(int64_t(a.kv_heads) * b.splits * b.tiles, kThreads, "Attention is too large")), block(kThreads);
#define ACCEL_PROMPT(L, U) hipLaunchKernelGGL((AttendPromptKernel<DP, kF32, L, U>), grid, block, 0, stream, a, b)
  if constexpr (kF32) {
    if (load == 16) ACCEL_PROMPT(16, false);
    else ACCEL_PROMPT(4, false);
  } else if (load == 16 && b.block_shift >= 6) {
    ACCEL_PROMPT(16, true);
  } else if (load == 16) {
    ACCEL_PROMPT(16, false);
  } else if (load == 4) {
    ACCEL_PROMPT(4, false);
  } else {
    ACCEL_PROMPT(1, false);
  }
#undef ACCEL_PROMPT
  Check(hipGetLastError(), "AttendPromptKernel launch");
}

template <bool kF32>
void LaunchPromptOf(const AttendArgs& a, PromptArgs b, int load, hipStream_t stream) {
  const int64_t group = a.heads / a.kv_heads;
  const int64_t tiles = (int64_t(a.seq) * group + kRows - 1) / kRows;
  const int64_t units = tiles * a.kv_heads;
  if (units > 0x7fffffff) Fail(ACCEL_HIP_INVALID_ARGUMENT, "Attention is too large");
  const AttendSplit split = SplitRange(a, units, AttendRangeSteps(a, kRows, kF32 ? 32 : 64) / 4);
  b.splits = split.count;
  b.tiles = static_cast<int32_t>(tiles);
  b.partial = split.partial;
  if (a.dim <= 64) LaunchPrompt<64, kF32>(a, b, load, stream);
  else if (a.dim <= 128) LaunchPrompt<128, kF32>(a, b, load, stream);
  else LaunchPrompt<256, kF32>(a, b, load, stream);
  if (b.splits > 1) LaunchAttendJoin(a, b.partial, b.splits, stream);
}

}  // namespace

void LaunchAttendPromptQ8(const AttendArgs& a, const Q8Cache& c, int load, hipStream_t stream) {
  PromptArgs b{};
  b.k = c.k.code;
  b.v = c.v.code;
  b.k_scale = c.k.scale;
  b.v_scale = c.v.scale;
  b.block_shift = c.block_shift;
  LaunchPromptOf<false>(a, b, load, stream);
}

void LaunchAttendPromptF32(const AttendArgs& a, const float* k, const float* v, int load, hipStream_t stream) {
  PromptArgs b{};
  b.k = k;
  b.v = v;
  LaunchPromptOf<true>(a, b, load, stream);
}

}  // namespace accel_hip
