// Attention of a batch's requests with many new rows (chunks of prompts over pages, whole prompts), as device
// functions.
//
// One workgroup per (128 rows of a request and key head, key range): four waves of 32 rows share each tile of keys
// through LDS, which the next one is brought to while it is worked on (two buffers, one barrier a tile). Everything
// runs on the f16 matrix cores: queries and softmax weights as two f16 parts (22 bits), an f16 cache as it is (tiles
// of 64 keys), fp32 keys and values as two parts (tiles of 32). Lane (j, g) = (lane % 32, lane / 32) serves
// row j. Per 32 keys
//  * S^T = K Q^T on v_mfma_f32_32x32x16_f16, keys as rows: the lane's 16 results are the scores of keys
//    8a + 4g + b (a, b < 4) of row j, so a row's softmax needs one exchange between two lanes;
//  * O^T += V^T P^T: those scores are the lane's own k-slots of P^T if slot e of 16 keys is key
//    (e % 4) + 8 (e / 4) + 4g, and the value operand is read transposed from the row-major tile
//    (ds_read_b64_tr_b16 gives a lane four keys of one dim).
// An fp32 row enters as its parts times a power of two: 2^9 for rows whose largest magnitude lies in [2^-6, 2^6),
// which keeps 22 bits of all of them, otherwise one from the row's own largest magnitude (of a row of zeros 2^127), whose
// inverse meets its scores or weights. A row that is not finite, or has no page, has NaN there and zeros for values.
//
// Bound: the matrix cores, at the clock that they leave. Prompts of 474 .. 3410 tokens, 32 heads on 8 of 128, take
// 693 - 753 us, 274 - 297 TFLOP/s counted once and three f16 products each; these products alone, from registers and over
// random values, 372, at a large library product's rate 468. The cores
// are busy 41 % of the cycles, at 1.9 GHz. A workgroup by itself took 4100 cycles a tile of 32 keys: 1536 of products,
// 510 of softmax, 700 to send the loads in a burst, 800 to split rows and weights; a second one on the CU fills part
// of that. So
//  * two workgroups a CU (at head dim 128 245 registers for packed prompts, 251 over fp32 pages and 255 over f16 ones),
//    rather than tiles of 256 rows, which spill;
//  * loads go out between the score products, and what only tiles of odd scales or moving references need is behind
//    uniform branches (144 -> 126 us for 3 prompts of 16 heads of 80). Splitting rows between the value products
//    as well would spill 72 registers at 128;
//  * no other part is the bound by itself: of 735 us before these steps, without softmax 592, without the split and
//    its stores 649, without the loads 692; with 15 % fewer vector instructions in all 735.
// Head dims of 129 .. 256 are worked on as 256, in one workgroup a CU, and do not fit its 512 registers: 38 are spilled for
// packed prompts, 45 over fp32 pages, 62 over f16 ones. 5 prompts of 426 .. 1819 tokens, 16 heads on 4: 524 us at 256 and 519
// at 192 (165 at 128); chunks of 200 .. 500 over up to 4000 tokens 169 and 164 in fp32 (62), 120 and 116 in f16 (48).
// Rows off the 16-byte grid are loaded an element at a time, from head dim 65 on in one workgroup a CU too, at 256 with 94 to
// 338 registers spilled: the same chunks over f16 with heads of 100 take 88 us, of 96 43.
#pragma once

#include "attend_batch_step.h"

namespace accel_hip {

constexpr int kPromptWaves = kBatchThreads / 64;
constexpr int kWaveRows = 32;
static_assert(kPromptTileRows == kPromptWaves * kWaveRows, "a wave has 32 rows");
constexpr float kCommonScale = 0x1p9f;
constexpr int32_t kCommonPower = 9;
constexpr float kBackFirst = 0x1p60f;
constexpr uint32_t kCommonLow = 0x4800, kCommonHigh = 0x7800;  // f16's bits of 2^-6 and 2^6 times that
// What a barrier of the scheduler's lets pass: vector and scalar arithmetic, LDS; no product and no load.
constexpr int kNotLoads = 0x2 | 0x4 | 0x80;
// Weights of up to 2^14 meet values' scales, 2^-127 .. 2^114, times 2^-1: all of these products are floats, and the
// largest of a row, whose weight is 2^6 at least, is 2^-122 or more, so that what it loses below 2^-126 is within 2^-27.
constexpr int32_t kUnits = 1;
typedef short s4 __attribute__((ext_vector_type(4)));

template <int DP, bool kHalf>
struct alignas(16) PromptTiles {
  static constexpr int kParts = kHalf ? 1 : 2;
  static constexpr int kKeys = PromptKeys(kHalf);
  // Halves: 8 key rows' 16-byte pieces fall into different banks, and so do 4 value rows' 64-byte pieces (two tile reads).
  static constexpr int kKStride = DP + 8;
  static constexpr int kVStride = DP == 96 ? 96 : DP + 32;
  alignas(16) _Float16 kt[2][kParts][kKeys][kKStride];
  alignas(16) _Float16 vt[2][kParts][kKeys][kVStride];
  alignas(16) float sk[2][kKeys];  // f16: 1 or NaN, read where the tile has marks
  alignas(16) float sv[2][kHalf ? 4 : kKeys];
  int odd[3];  // the tile has rows of scales of their own, or marks
};

// kHalf: an f16 cache. kLoad: bytes that may be loaded at once (16, or an element's).
template <int DP, bool kHalf, int kLoad, bool kPaged>
__device__ __forceinline__ void PromptGroup(const BatchAttendArgs& a, const BatchSplit& b, int32_t block,
                                            PromptTiles<DP, kHalf>& lds, BatchScan<kBatchThreads>& scan) {
  static_assert(kPaged || !kHalf, "prompts without a cache are fp32");
  using Tiles = PromptTiles<DP, kHalf>;
  constexpr int kParts = Tiles::kParts, kKeys = Tiles::kKeys, kKStride = Tiles::kKStride, kVStride = Tiles::kVStride;
  constexpr int kSub = kKeys / 32;
  constexpr int kSteps = DP / 16;
  constexpr int kDims = DP / 32;
  constexpr int kStaged = DP == 96 && kHalf ? 128 : DP;  // dims that the threads of a key row are dealt
  constexpr int kRowLanes = kHalf ? kStaged / 8 : 8;  // threads that stage a key row, neighbours
  constexpr int kStagedRows = kBatchThreads / kRowLanes;  // rows staged at once
  constexpr int kChunks = kHalf ? kKeys / kStagedRows : kStaged / 32;  // 16-byte pieces of a plane a thread stages
  constexpr int kPages = kHalf ? kChunks : 1;  // page entries a thread needs, uniform over its wave
  auto& kt = lds.kt;
  auto& vt = lds.vt;
  auto& sk = lds.sk;
  auto& sv = lds.sv;
  auto& odd = lds.odd;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 31;
  const int g = lane >> 5;
  const int32_t kv = block - Quotient(block, a.by_kv_heads) * a.kv_heads;
  const int32_t group = a.heads / a.kv_heads;
  BatchItem w;
  if (!FindWork<kBatchThreads, kPromptTileRows, kKeys, false>(a, b, Quotient(block, a.by_kv_heads), kv == 0, scan, &w)) return;
  const int32_t w0 = w.r0 + wave * kWaveRows;  // the wave's rows
  const int32_t row = min(w0 + j, w.rows - 1);
  const int32_t s = Quotient(row, a.group);
  const int32_t head = kv * group + (row - s * group);
  const int32_t p_row = w0 + j < w.rows ? w.seen + s : -1;
  const int32_t pw_first = w.seen + Quotient(min(w0, w.rows - 1), a.group);
  const int32_t pw_last = w0 < w.rows ? w.seen + Quotient(min(w0 + kWaveRows, w.rows) - 1, a.group) : -1;
  const bool full_rows = w0 + kWaveRows <= w.rows;
  const BatchPages pages(a, kPaged ? w.request : 0);
  const auto key_of = [&](int32_t step) { return w.low + step * kKeys; };
  // Where a tile's row holds which dims: 4 from a place that is a multiple of 4 on. Eight threads load 128 bytes of an
  // fp32 row at a time, and each writes what it has of two such loads as 16 bytes: places 8l .. 8l + 7 of 64 are dims
  // 4l .. 4l + 3 and 32 + 4l .. Of 96, the last 32 are in order.
  const auto dim_of = [](int place) {
    if (kHalf || (DP == 96 && place >= 64)) return place;
    return (place & ~63) + (place >> 2 & 1) * 32 + (place >> 3 & 7) * 4;
  };

  // ---- staging: a thread's pieces of the next tile, from memory to registers and on to LDS ----
  uint4 kreg[kChunks], vreg[kChunks];
  int32_t entry[kPages], entry_next[kPages];
  const auto find_pages = [&](int32_t t0) {  // piece i of an f16 tile is of key row tid / kRowLanes + i * kStagedRows
    if constexpr (kPaged) {
#pragma unroll
      for (int i = 0; i < kPages; ++i)
        entry_next[i] = pages.Entry(t0 + (wave * 64 / kRowLanes + i * kStagedRows) / 16 * 16);
    }
  };
  // The tile at t0: its pages, then its pieces, one by one.
  const float* fetched[2];
  int32_t t_fetch = 0;
  const auto fetch_at = [&](int32_t t0) {
    if constexpr (kPaged) {
#pragma unroll
      for (int i = 0; i < kPages; ++i) entry[i] = __builtin_amdgcn_readfirstlane(entry_next[i]);
    }
    t_fetch = t0;
    if constexpr (!kHalf) {
      // A row past a prompt's last reads its last one, a piece past a head's dims its last: both are not used.
      const int32_t t = t0 + tid / kRowLanes;
      const int64_t row_at = kPaged ? pages.Slot(entry[0], t) : static_cast<int64_t>(w.start) + min(t, w.high - 1);
      const int64_t at = row_at * a.kv_stride + static_cast<int64_t>(kv) * a.dim;
      fetched[0] = static_cast<const float*>(a.k) + at;
      fetched[1] = static_cast<const float*>(a.v) + at;
    }
  };
  const auto fetch_piece = [&](int i) {
    if constexpr (kHalf) {
      const int d = 8 * (tid % kRowLanes);
      const int64_t at = pages.Slot(entry[i], t_fetch + tid / kRowLanes + i * kStagedRows) * a.kv_stride + static_cast<int64_t>(kv) * a.dim;
      const auto piece = [&](const void* plane) {
        const _Float16* p = static_cast<const _Float16*>(plane) + at;
        if (kLoad == 16) return *reinterpret_cast<const uint4*>(p + min(d, a.dim - 8));
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
        const auto two = [&](int e) {
          return h[min(d + e, a.dim - 1)] | static_cast<uint32_t>(h[min(d + e + 1, a.dim - 1)]) << 16;
        };
        return make_uint4(two(0), two(2), two(4), two(6));
      };
      kreg[i] = piece(a.k);
      vreg[i] = piece(a.v);
    } else {
      const int d = 32 * i + 4 * (tid % 8);
      const auto piece = [&](const float* p) {
        if (kLoad == 16) return *reinterpret_cast<const uint4*>(p + min(d, a.dim - 4));
        const auto one = [&](int e) { return __float_as_uint(p[min(d + e, a.dim - 1)]); };
        return make_uint4(one(0), one(1), one(2), one(3));
      };
      kreg[i] = piece(fetched[0]);
      vreg[i] = piece(fetched[1]);
    }
  };
  const auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) fetch_piece(i);
  };
  // fp32: writes a thread's pieces of one plane; tile row `key` begins at dst + key * stride, its second part
  // `part` halves later. All rows are written at the common scale, and again where a row of the wave's is not common.
  const auto put_plane = [&](const uint4 (&x)[kChunks], _Float16* dst, int stride, int part, float& row_back, int slot) {
    _Float16* p = dst + (tid / 8) * stride;
    const auto write = [&](float scale, bool zero) {
      h2 most = h2{0, 0};
#pragma unroll
      for (int i = 0; i < kChunks; i += 2) {
        h2 hi[4], lo[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if (i + n == kChunks) break;
          const uint32_t v[4] = {x[i + n].x, x[i + n].y, x[i + n].z, x[i + n].w};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            SplitScaled(zero ? 0.f : __uint_as_float(v[2 * e]), zero ? 0.f : __uint_as_float(v[2 * e + 1]), scale, hi[2 * n + e],
                        lo[2 * n + e]);
            most = LargestHalves(hi[2 * n + e], most);
          }
        }
        if (i + 1 < kChunks) {
          *reinterpret_cast<h8*>(p + 32 * i + 8 * (tid % 8)) = Join(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<h8*>(p + 32 * i + 8 * (tid % 8) + part) = Join(lo[0], lo[1], lo[2], lo[3]);
        } else {
          *reinterpret_cast<h4*>(p + 32 * i + 4 * (tid % 8)) = __builtin_shufflevector(hi[0], hi[1], 0, 1, 2, 3);
          *reinterpret_cast<h4*>(p + 32 * i + 4 * (tid % 8) + part) = __builtin_shufflevector(lo[0], lo[1], 0, 1, 2, 3);
        }
      }
      return __builtin_bit_cast(uint32_t, most);
    };
    uint32_t most = write(kCommonScale, false);
    most = max(most & 0xffffu, most >> 16);
    most = max(most, XorLane<1>(most));
    most = max(most, XorLane<2>(most));
    most = max(most, XorLane<4>(most));
    row_back = 1.f / kCommonScale;
    const bool common = most - kCommonLow < kCommonHigh - kCommonLow && (!kPaged || pages.Is(entry[0]));
    if (!__all(common)) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
        top = max(max(top, max(x[i].x & 0x7fffffffu, x[i].y & 0x7fffffffu)), max(x[i].z & 0x7fffffffu, x[i].w & 0x7fffffffu));
      top = max(top, XorLane<1>(top));
      top = max(top, XorLane<2>(top));
      top = max(top, XorLane<4>(top));
      if (kPaged && !pages.Is(entry[0])) top = 0x7f800000u;  // uniform
      const bool finite = top < 0x7f800000u;
      const float scale = RowScale(finite ? max(top, 1u) : 0);  // zeros: as of the smallest values, so that they weigh nothing
      odd[slot] = 1;
      row_back = finite ? 1.f / scale : NAN;
      write(scale, !finite);
    }
  };
  const auto put = [&](int buf, int slot) {
    if constexpr (kHalf) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const auto zero = [](uint32_t x, float z) { return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), h2{0, 0}, z, false); };
        float z = pages.Is(entry[i]) ? 0.f : NAN;  // NaN where a value is not finite
        z = zero(kreg[i].w, zero(kreg[i].z, zero(kreg[i].y, zero(kreg[i].x, z))));
        z = zero(vreg[i].w, zero(vreg[i].z, zero(vreg[i].y, zero(vreg[i].x, z))));
        const int key = tid / kRowLanes + i * kStagedRows;
        const int d = 8 * (tid % kRowLanes);
        const uint64_t bad = __ballot(!(z == 0.f));
        float mark = 1.f;
        uint4 v = vreg[i], k = kreg[i];
        if (bad != 0) {  // uniform over the wave
          odd[slot] = 1;
          const uint64_t row_lanes = (kRowLanes == 64 ? ~uint64_t(0) : ((uint64_t(1) << (kRowLanes & 63)) - 1))
                                     << (lane / kRowLanes * kRowLanes);
          if ((bad & row_lanes) != 0) {
            mark = NAN;
            v = k = make_uint4(0, 0, 0, 0);
          }
        }
        if (DP == kStaged || d < DP) {
          *reinterpret_cast<uint4*>(&kt[buf][0][key][d]) = k;
          *reinterpret_cast<uint4*>(&vt[buf][0][key][d]) = v;
        }
        if (tid % kRowLanes == 0) sk[buf][key] = mark;
      }
    } else {
      float k_back = 1.f, v_back = 1.f;
      put_plane(kreg, &kt[buf][0][0][0], kKStride, kKeys * kKStride, k_back, slot);
      put_plane(vreg, &vt[buf][0][0][0], kVStride, kKeys * kVStride, v_back, slot);
      if (!(fabsf(v_back) < INFINITY)) {  // a value row that is not finite marks its key: a weight of 0 stays one
        k_back = NAN;
        v_back = 0.f;
      }
      if (tid % 8 == 0) {
        sk[buf][tid / 8] = k_back;
        sv[buf][tid / 8] = v_back;
      }
    }
  };
  if (w.begin < w.end) {
    find_pages(key_of(w.begin));
    fetch_at(key_of(w.begin));
    fetch();
    find_pages(key_of(min(w.begin + 1, w.end - 1)));
  }

  // ---- the rows' queries ----
  h8 qh[kSteps], ql[kSteps];
  float row_back;  // a power of two: takes the row's scale out of its scores again
  {
    const float* q = a.q + (w.start + s) * a.q_stride + static_cast<int64_t>(head) * a.dim;
    const bool vec = BatchQueryVec(a);
    const bool stored = !kPaged || BatchRowStored(a, w.start + s);
    float x[kSteps][2][4];
    uint32_t top = 0;
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int n = 0; n < 2; ++n) LoadBatchQuery(q, a.dim, dim_of(16 * st + 8 * g + 4 * n), vec, x[st][n]);
    if (a.dim < DP) {
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
#pragma unroll
        for (int n = 0; n < 2; ++n) MaskQuery(a.dim, dim_of(16 * st + 8 * g + 4 * n), x[st][n]);
    }
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[st][e >> 2][e & 3]) & 0x7fffffffu);
    top = max(top, XorLane<32>(top));
    const float scale = top >= 0x7f800000u || !stored ? NAN : RowScale(top);  // no finite row: all of it NaN
    row_back = 1.f / scale;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      h2 hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        SplitF16Nearest(x[st][e >> 1][2 * (e & 1)] * scale, x[st][e >> 1][2 * (e & 1) + 1] * scale, hi[e], lo[e]);
      qh[st] = Join(hi[0], hi[1], hi[2], hi[3]);
      ql[st] = Join(lo[0], lo[1], lo[2], lo[3]);
    }
  }

  float m = -INFINITY, base = 0.f, l = 0.f, hi = -INFINITY, top = 0.f;  // base: m, or 0 where there is none
  bool far = false, mixed = false;  // one of the wave's rows has far scores; a tile was not of common scale
  int32_t power = kCommonPower;  // fp32: the sums hold weight * value * 2^power
  f16v acc[kDims];
#pragma unroll
  for (int t = 0; t < kDims; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

  if (tid < 3) odd[tid] = 0;
  __syncthreads();
  if (w.begin < w.end) put(0, 0);
  for (int32_t u = w.begin; u < w.end; ++u) {
    const int buf = (u - w.begin) & 1;
    const int32_t t0 = key_of(u);
    __syncthreads();
    if (tid == 0) odd[(u + 2 - w.begin) % 3] = 0;  // next written behind the next barrier
    // Behind the last tile it is fetched again, so that nothing here branches.
    fetch_at(key_of(min(u + 1, w.end - 1)));
    find_pages(key_of(min(u + 2, w.end - 1)));
    const int32_t last = t0 + kKeys - 1;
    const bool none = t0 > pw_last || last <= pw_first - a.window;
    const bool whole = full_rows && last <= pw_first && t0 > pw_last - a.window;
    // A wave whose rows see none of the tile makes these products too: its loads go out among them.
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
      if constexpr (!kHalf) {
        const h8 k8l = *reinterpret_cast<const h8*>(&kt[buf][kParts - 1][j][16 * step + 8 * g]);
        st[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8l, qh[step], st[0], 0, 0, 0);
      }
      // The next tile's loads go out between the products, none of which waits for the memory pipe then.
      constexpr int kEach = (kChunks + kSteps - 1) / kSteps;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (step * kEach + i < kChunks) fetch_piece(step * kEach + i);
      __builtin_amdgcn_sched_barrier(kNotLoads);
    }
    __builtin_amdgcn_s_setprio(0);
    if (!none) {  // uniform over the wave
      const bool plain = odd[(u - w.begin) % 3] == 0;  // uniform
      float c = a.factor;
      if (kHalf || plain) {
        c *= row_back * (kHalf ? 1.f : 1.f / kCommonScale);
      } else {
        // A key's scale could carry the product past the range: the row's scale out first, as far as that
        // itself cannot.
        c *= row_back > kBackFirst ? row_back / kBackFirst : 1.f;
#pragma unroll
        for (int h = 0; h < kSub; ++h)
#pragma unroll
          for (int r = 0; r < 16; ++r) st[h][r] *= fminf(row_back, kBackFirst);
      }
      if (!plain) {
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
            st[h][r] = SeesKey(a, p_row, t0 + 32 * h + (r & 3) + 8 * (r >> 2) + 4 * g) ? st[h][r] * c : -INFINITY;
        c = 1.f;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[h][r]);
      mx = fmaxf(mx, XorLane<32>(mx)) * c;
      // The reference moves only when a score passes it far enough, so the sums are seldom scaled.
      const bool moves = mx > m + (kHeadroom + kSlack);
      bool scale = __any(moves);  // uniform, as are far and mixed
      float again = 1.f;
      if (scale) {
        if (moves) {
          again = __builtin_amdgcn_exp2f(m - (mx - kHeadroom));
          base = m = mx - kHeadroom;
          l *= again;
        }
        far = __any(fabsf(base) >= kFarScore);
      }
      float sum = 0.f, below = base;
      if (far) {
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
      l += sum;
      const float before = hi;  // the largest score of the tiles before, while all are of common scale
      if constexpr (!kHalf) hi = fmaxf(hi, mx);
      if (!kHalf && (mixed || !plain)) {
        // Values of common scale meet the weights as they are; others, and weights that are held otherwise since, times
        // the values' scales and a power of two that follows the largest of them.
        constexpr float kDown = 1.f / (1 << kUnits);
        top = mixed ? top * again : __builtin_amdgcn_exp2f(before - base) * (kDown / kCommonScale);
        mixed = true;
        if (plain) {
          top = fmaxf(top, __builtin_amdgcn_exp2f(mx - base) * (kDown / kCommonScale));
        } else {
          float tile_top = 0.f;
#pragma unroll
          for (int h = 0; h < kSub; ++h)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
              const f4 f = *reinterpret_cast<const f4*>(&sv[buf][32 * h + 8 * r4 + 4 * g]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                st[h][4 * r4 + e] = st[h][4 * r4 + e] * kDown * f[e];
                tile_top = fmaxf(tile_top, fabsf(st[h][4 * r4 + e]));
              }
            }
          top = fmaxf(top, fmaxf(tile_top, XorLane<32>(tile_top)));
        }
        const int32_t power_old = power;
        power = WeightPower(top, power + kUnits) - kUnits;
        again = ldexpf(again, power - power_old);
        scale = true;
        if (!plain || __any(power != kCommonPower)) {
          const int32_t by = plain ? power - kCommonPower : power + kUnits;
#pragma unroll
          for (int h = 0; h < kSub; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[h][r] = ldexpf(st[h][r], by);
        }
      }
      if (scale) {
#pragma unroll
        for (int t = 0; t < kDims; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[t][r] *= again;
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
          for (int e = 0; e < 4; ++e) SplitWeights(st[h][8 * k16 + 2 * e], st[h][8 * k16 + 2 * e + 1], hi[e], lo[e]);
          const h8 ph = Join(hi[0], hi[1], hi[2], hi[3]), pl = Join(lo[0], lo[1], lo[2], lo[3]);
          const auto read = [&](int t, int part) {
            const _Float16* p = vrow + part * kKeys * kVStride + (32 * h + 16 * k16) * kVStride + 32 * t;
            const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
            const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 8 * kVStride));
            return __builtin_bit_cast(h8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
          };
#pragma unroll
          for (int t0 = 0; t0 < kDims; t0 += 2) {
            // Neighbouring instructions add to different sums.
            constexpr auto kOf = [](int t) { return t + 1 < kDims ? 2 : 1; };
            h8 v[2];
#pragma unroll
            for (int t = 0; t < kOf(t0); ++t) v[t] = read(t0 + t, 0);
#pragma unroll
            for (int t = 0; t < kOf(t0); ++t) acc[t0 + t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[t], ph, acc[t0 + t], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < kOf(t0); ++t) acc[t0 + t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[t], pl, acc[t0 + t], 0, 0, 0);
            if constexpr (!kHalf) {
#pragma unroll
              for (int t = 0; t < kOf(t0); ++t)
                acc[t0 + t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(read(t0 + t, kParts - 1), ph, acc[t0 + t], 0, 0, 0);
            }
          }
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (u + 1 < w.end) put(buf ^ 1, (u + 1 - w.begin) % 3);
  }

  // acc[t][r] is O^T[place 32t + 8 (r / 4) + 4g + r % 4][row j].
  l = l + XorLane<32>(l);
  if (w0 + j >= w.rows) return;
  // fp32: the sums hold 2^power times what they are, and where they may pass the largest float 2^-64 of that is left.
  const bool held = !kHalf && power < kFarPower;
  const int32_t down = kHalf ? 0 : held ? -power - kFarShift : -power;
  const float inverse = w.splits > 1 ? 1.f : __fdiv_rn(1.f, l);
  float* dst = a.out + (static_cast<int64_t>(w.start + s) * a.heads + head) * a.dim;
  bool vec = a.dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  if (w.splits > 1) {
    const int64_t at = (static_cast<int64_t>(kv) * b.items + w.partial) * kPromptTileRows + wave * kWaveRows + j;
    dst = b.partial.o + at * PartialDims(a.dim);
    vec = true;
    if (g == 0) {
      b.partial.ml[2 * at] = m;
      b.partial.ml[2 * at + 1] = held ? -l : l;
    }
  }
#pragma unroll
  for (int t = 0; t < kDims; ++t)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int d = dim_of(32 * t + 8 * r4 + 4 * g);
      f4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (kHalf ? acc[t][4 * r4 + e] : ldexpf(acc[t][4 * r4 + e], down)) * inverse;
      if (!kHalf && held && w.splits == 1) o *= kFarUp;
      if (vec) {
        if (d < a.dim) *reinterpret_cast<f4*>(dst + d) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < a.dim) dst[d + e] = o[e];
      }
    }
}

}  // namespace accel_hip
