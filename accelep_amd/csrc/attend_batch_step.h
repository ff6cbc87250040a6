// Attention of a batch's requests with few new rows (single tokens, drafts), as device functions.
//
// One workgroup per (16 rows of a request and key head, key range); its four waves take the range's steps in turn
// and meet in LDS. Keys and values go from memory to registers and from there to the matrix cores, without LDS and
// barriers in the loop; a step's keys lie in one or two pages, whose table entries are read a step ahead.
// Lane (j, g) = (lane % 16, lane / 16). Bound: the bytes of the keys and values. 32 requests of 512 .. 16384 tokens in f16
// (32 heads on 8 of 128): 130 us, 4.7 TB/s, with the join; a large copy reaches 5.16. 125 requests of 16 .. 2048 in fp32:
// 97 - 105 us, 4.1 - 4.4 TB/s. 4 requests of a small model: 12 us, of which 8.3 this kernel (lengths, query, one page entry,
// keys, softmax and values wait for one another) and 3.6 the join. Rows off the 16-byte grid (f16 head dims that are no
// multiple of 8, memory that is not aligned) are loaded an element at a time, from head dim 65 on in one workgroup a CU: the
// 32 requests with heads of 100 take 522 us, of 96 111; in fp32, where 100 is on the grid, 205 and 195. Head dim 256, 16 heads
// on 4, the same bytes as 32 on 8 of 128: 146 us in f16, 258 in fp32, where 128 takes 130 and 222.
#pragma once

#include "attend_batch.h"

namespace accel_hip {

constexpr int kStepWaves = kBatchThreads / 64;
constexpr uint32_t kLargeBits = (127 + 96) << 23;  // 2^96
constexpr float kHeldWeight = 0x1p-40f;

// The results of a workgroup's waves meet in LDS; l and o are held as in AttendPartial.
template <int DP>
struct alignas(16) BatchParts {
  float o[kStepWaves][kStepTileRows][DP + 4];
  float m[kStepWaves][kStepTileRows];
  float l[kStepWaves][kStepTileRows];
  __device__ __forceinline__ void Join(const BatchAttendArgs& a, const BatchSplit& b, const BatchItem& w, int32_t group,
                                       int32_t kv) const {
    const bool vec = a.dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
    const int32_t n = min(kStepTileRows, w.rows - w.r0);
    for (int32_t item = threadIdx.x; item < n * (DP / 4); item += kBatchThreads) {
      const int32_t rl = item / (DP / 4);
      const int32_t d = item % (DP / 4) * 4;
      if (d >= a.dim) continue;
      float big = -INFINITY;
#pragma unroll
      for (int v = 0; v < kStepWaves; ++v) big = fmaxf(big, m[v][rl]);
      const float base = big == -INFINITY ? 0.f : big;
      float weight[kStepWaves], most = 0.f;  // most: of the parts that are held times 2^-64
#pragma unroll
      for (int v = 0; v < kStepWaves; ++v) {
        weight[v] = __builtin_amdgcn_exp2f(m[v][rl] - base);
        if (l[v][rl] < 0.f) most = fmaxf(most, weight[v]);
      }
      const bool far = most >= 0x1p-60f;  // the sum is held so too, unless they count for little
      float total = 0.f;
      f4 x = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < kStepWaves; ++v) {
        const bool held = l[v][rl] < 0.f;
        total += weight[v] * fabsf(l[v][rl]);
        x += weight[v] * (held == far ? 1.f : far ? kFarDown : kFarUp) * *reinterpret_cast<const f4*>(&o[v][rl][d]);
      }
      if (w.splits > 1) {
        const int64_t at = (static_cast<int64_t>(kv) * b.items + w.partial) * kStepTileRows + rl;
        if (d == 0) {
          b.partial.ml[2 * at] = big;
          b.partial.ml[2 * at + 1] = far ? -total : total;
        }
        *reinterpret_cast<f4*>(b.partial.o + at * PartialDims(a.dim) + d) = x;
      } else {
        float* dst = a.out + BatchOutRow(a, w.start, w.r0 + rl, group, kv) * a.dim + d;
        const f4 y = f4{__fdiv_rn(x[0], total), __fdiv_rn(x[1], total), __fdiv_rn(x[2], total), __fdiv_rn(x[3], total)} *
                     (far ? kFarUp : 1.f);
        if (vec) {
          *reinterpret_cast<f4*>(dst) = y;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < a.dim) dst[e] = y[e];
        }
      }
    }
  }
};

// fp32 keys and values, 16 a step. Both products run on v_mfma_f32_16x16x4f32, which takes fp32 as it is:
//  * S^T = K Q^T: k slot g of instruction (i, e) is dim 16i + 4g + e, so a lane loads 16 bytes of key
//    row j at a time and a key row's pieces lie side by side;
//  * O^T += V^T P^T: S^T leaves the lane the scores of keys 4g .. 4g + 3 of row j; k slot g of
//    instruction s is key 4g + s, the A operand of dim tile (c, t) float t of the 16 bytes at
//    V[key][64c + 4j].
// A key or value row that is not finite would reach rows that do not see it, as 0 * NaN: a step that
// holds one (a test of the bits, uniform) has its values taken as zeros and its weights as NaN, and so has a step
// without a page. The same test finds values from 2^96 on, whose sum over the keys may pass the largest float: a row
// that gives one of them a weight from 2^-40 on holds its sum times 2^-64 until that weight is next to nothing beside
// later ones. Such a value is itself taken times 2^-64, and its weight, times 2^64 where the row's sum is not held, keeps
// its bits however small it is: 2^-80 of 2^126 outweighs all ordinary values.
template <int DP, int kLoad, bool kPaged>
__device__ __forceinline__ void StepF32Group(const BatchAttendArgs& a, const BatchSplit& b, int32_t block,
                                             BatchParts<DP>& parts, BatchScan<kBatchThreads>& scan) {
  constexpr int kKeys = 16;
  constexpr int kI = DP / 16;  // 16-byte pieces of a key row per lane
  constexpr int kC = DP / 64;  // of a value row
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15;
  const int g = lane >> 4;
  const int32_t kv = block - Quotient(block, a.by_kv_heads) * a.kv_heads;
  const int32_t group = a.heads / a.kv_heads;
  BatchItem w;
  if (!FindWork<kBatchThreads, kStepTileRows, kKeys, true>(a, b, Quotient(block, a.by_kv_heads), kv == 0, scan, &w)) return;
  const int32_t row = min(w.r0 + j, w.rows - 1);
  const int32_t s = Quotient(row, a.group);
  const int32_t p_row = w.r0 + j < w.rows ? w.seen + s : -1;  // a row past the last sees nothing
  const float* kbase = static_cast<const float*>(a.k) + static_cast<int64_t>(kv) * a.dim;
  const float* vbase = static_cast<const float*>(a.v) + static_cast<int64_t>(kv) * a.dim;
  const BatchPages pages(a, kPaged ? w.request : 0);

  f4 kx[kI], vx[4][kC];
  // A piece past a head's dims reads its last (it meets a query of 0, or makes a dim that is not stored), a
  // row past a prompt's last the last one. A page's rows are all there.
  const auto piece = [&](const float* p, int d) {
    if (kLoad == 16) return *reinterpret_cast<const f4*>(p + min(d, a.dim - 4));
    f4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = p[min(d + e, a.dim - 1)];
    return x;
  };
  const auto row_at = [&](int32_t t0, int32_t entry, int32_t key) {
    return kPaged ? pages.Slot(entry, t0) + key : static_cast<int64_t>(w.start) + min(t0 + key, w.high - 1);
  };
  const auto load_k = [&](int32_t t0, int32_t entry) {
    const float* p = kbase + row_at(t0, entry, j) * a.kv_stride;
#pragma unroll
    for (int i = 0; i < kI; ++i) kx[i] = piece(p, 16 * i + 4 * g);
  };
  const auto load_v = [&](int32_t t0, int32_t entry) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* p = vbase + row_at(t0, entry, 4 * g + e) * a.kv_stride;
#pragma unroll
      for (int c = 0; c < kC; ++c) vx[e][c] = piece(p, 64 * c + 4 * j);
    }
  };
  int32_t u = w.begin + wave;
  const auto key_of = [&](int32_t step) { return w.low + step * kKeys; };
  int32_t entry = -1, entry_next = -1;
  if (kPaged && u < w.end) {
    entry = pages.Entry(key_of(u));
    if (u + kStepWaves < w.end) entry_next = pages.Entry(key_of(u + kStepWaves));
  }
  f4 q[kI];
  {
    const float* p = a.q + (w.start + s) * a.q_stride + static_cast<int64_t>(kv * group + (row - s * group)) * a.dim;
    const bool vec = BatchQueryVec(a);
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      float x[4];
      LoadBatchQuery(p, a.dim, 16 * i + 4 * g, vec, x);
      q[i] = f4{x[0], x[1], x[2], x[3]};
    }
  }
  const bool stored = !kPaged || BatchRowStored(a, w.start + s);
  if (u < w.end) {
    entry = __builtin_amdgcn_readfirstlane(entry);
    load_k(key_of(u), entry);
    load_v(key_of(u), entry);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < kI; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) q[i][e] = 16 * i + 4 * g + e < a.dim ? q[i][e] : 0.f;
  if (!stored) q[0][0] = NAN;

  float m = -INFINITY, l = 0.f;  // l: this lane's share of the row's sum
  float shift = 1.f, share = 0.f;  // the weighted sum's power of two, and the largest weight now of a large value
  f4 acc[kC][4];
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[c][t] = f4{0.f, 0.f, 0.f, 0.f};
  for (; u < w.end; u += kStepWaves) {  // uniform over the wave
    const int32_t t0 = key_of(u);
    const bool more = u + kStepWaves < w.end;
    const int32_t next = key_of(u + kStepWaves);
    f4 st0 = f4{0.f, 0.f, 0.f, 0.f}, st1 = st0;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        st0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[i][e], q[i][e], st0, 0, 0, 0);
        st1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[i][e + 1], q[i][e + 1], st1, 0, 0, 0);
        top = max(top, max(FloatBits(kx[i][e]) & 0x7fffffffu, FloatBits(kx[i][e + 1]) & 0x7fffffffu));
      }
    if (kPaged && !pages.Is(entry)) top = 0x7f800000u;
    const uint64_t bad_keys = __ballot(top >= 0x7f800000u);
    const int32_t entry_v = __builtin_amdgcn_readfirstlane(entry_next);
    if (more) {
      load_k(next, entry_v);
      if (kPaged && u + 2 * kStepWaves < w.end) entry_next = pages.Entry(key_of(u + 2 * kStepWaves));
    }
    __builtin_amdgcn_sched_barrier(0);
    uint32_t vtop[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      vtop[e] = 0;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) vtop[e] = max(vtop[e], FloatBits(vx[e][c][t]) & 0x7fffffffu);
    }
    uint32_t bad = 0, large = 0;  // of the lane's keys 4g + e
    if (__any(max(max(vtop[0], vtop[1]), max(vtop[2], vtop[3])) >= kLargeBits) || bad_keys != 0) {
      const uint32_t keys16 = static_cast<uint32_t>(bad_keys | bad_keys >> 16 | bad_keys >> 32 | bad_keys >> 48) & 0xffffu;
      bad = keys16 >> (4 * g) & 15u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t lanes = __ballot(vtop[e] >= 0x7f800000u);
        if ((__ballot(vtop[e] >= kLargeBits) >> (16 * g) & 0xffffu) != 0) large |= 1u << e;
        if ((lanes >> (16 * g) & 0xffffu) != 0) {
          bad |= 1u << e;
#pragma unroll
          for (int c = 0; c < kC; ++c) vx[e][c] = f4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
    float p[4];
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = SeesKey(a, p_row, t0 + 4 * g + e);
      st0[e] = in ? (bad >> e & 1 ? NAN : st0[e] + st1[e]) : -INFINITY;
      mx = fmaxf(mx, st0[e]);
    }
    mx = fmaxf(mx, XorLane<16>(mx));
    mx = fmaxf(mx, XorLane<32>(mx)) * a.factor;
    const float m_new = fmaxf(m, mx);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = __builtin_amdgcn_exp2f(m - base);
    float sum = 0.f;
    const bool far_scores = __any(fabsf(base) >= kFarScore);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[e] = __builtin_amdgcn_exp2f(far_scores ? st0[e] * a.factor - base : __builtin_fmaf(st0[e], a.factor, -base));
      sum += p[e];
    }
    l = l * corr + sum;
    m = m_new;
    float again = corr;
    share *= corr;
    if (shift != 1.f && share < kHeldWeight) {  // little is left of the large values
      again *= kFarUp;
      shift = 1.f;
    }
    if (__any(large != 0)) {
      bool weighs = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) weighs = weighs || ((large >> e & 1) != 0 && p[e] >= kHeldWeight);
      const uint64_t lanes = __ballot(weighs);
      if (((lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) >> j & 1) != 0) {
        share = 1.f;
        again *= shift == 1.f ? kFarDown : 1.f;
        shift = kFarDown;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if ((large >> e & 1) == 0) continue;
        p[e] *= kFarUp;
#pragma unroll
        for (int c = 0; c < kC; ++c) vx[e][c] *= kFarDown;
      }
    }
    if (__any(again != 1.f)) {
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[c][t] *= again;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] *= shift;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          acc[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[e][c][t], p[e], acc[c][t], 0, 0, 0);
    if (more) load_v(next, entry_v);
    entry = entry_v;
  }
  // acc[c][t][r] is O^T[dim 64c + 16g + 4r + t][row j].
  l = l + XorLane<16>(l);
  l = l + XorLane<32>(l);
  if (g == 0) {
    parts.m[wave][j] = m;
    parts.l[wave][j] = shift == 1.f ? l : -l;
  }
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f4*>(&parts.o[wave][j][64 * c + 16 * g + 4 * r]) =
          f4{acc[c][0][r], acc[c][1][r], acc[c][2][r], acc[c][3][r]};
  __syncthreads();
  parts.Join(a, b, w, group, kv);
}

// By how much the reference of a row's scores lies below their largest, at most and at least, in log2 units: the
// weights are then at most 2^14 and the largest 2^6, so that of two f16 parts the second is a normal number down
// to 2^-9 of it and what is lost is within 2^-30 of the largest.
constexpr float kHeadroom = 6.f, kSlack = 8.f;

// kN words of f16 pairs from dim d of a row on; dims past the head read its last.
template <int kN, int kLoad>
__device__ __forceinline__ void LoadHalves(const _Float16* p, int32_t dim, int d, uint32_t (&x)[kN]) {
  if constexpr (kLoad == 16 && kN == 4) {
    const u4 y = *reinterpret_cast<const u4*>(p + min(d, dim - 8));
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = y[e];
  } else if constexpr (kLoad == 16 && kN == 2) {
    const u2 y = *reinterpret_cast<const u2*>(p + min(d, dim - 4));
    x[0] = y[0];
    x[1] = y[1];
  } else {
    const uint16_t* b = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int e = 0; e < kN; ++e)
      x[e] = b[min(d + 2 * e, dim - 1)] | static_cast<uint32_t>(b[min(d + 2 * e + 1, dim - 1)]) << 16;
  }
}
// z + 0 * (both halves): NaN where one is not finite.
__device__ __forceinline__ float Finite(uint32_t x, float z) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), h2{0, 0}, z, false);
}

// f16 keys and values, 32 a step, of two pages at most. A query row, brought to [2^13, 2^14) by a power of two,
// and the weights enter as two f16 parts each.
//  * S^T = K Q^T on v_mfma_f32_16x16x32_f16: the A operand of instruction (c, half) is the 8 dims from
//    64c + 16g + 8 half on of key row j;
//  * O^T += V^T P^T: S^T leaves lane (j, g) the scores of keys 4g .. 4g + 3 and 16 + 4g .. of row j, which
//    are its 8 k-slots of P^T; the A operand of dim tile t is dim t of the DP / 16 that the lane loads at
//    V[key][DP / 16 * j], transposed in registers.
template <int DP, int kLoad>
__device__ __forceinline__ void StepF16Group(const BatchAttendArgs& a, const BatchSplit& b, int32_t block,
                                             BatchParts<DP>& parts, BatchScan<kBatchThreads>& scan) {
  constexpr int kKeys = 32;
  constexpr int kC = DP / 64;
  constexpr int kTiles = DP / 16;
  constexpr int kVWords = DP / 32;                     // words of a value row a lane loads
  constexpr int kVPiece = kVWords < 4 ? kVWords : 4;   // at once
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15;
  const int g = lane >> 4;
  const int32_t kv = block - Quotient(block, a.by_kv_heads) * a.kv_heads;
  const int32_t group = a.heads / a.kv_heads;
  BatchItem w;
  if (!FindWork<kBatchThreads, kStepTileRows, kKeys, true>(a, b, Quotient(block, a.by_kv_heads), kv == 0, scan, &w)) return;
  const int32_t row = min(w.r0 + j, w.rows - 1);
  const int32_t s = Quotient(row, a.group);
  const int32_t p_row = w.r0 + j < w.rows ? w.seen + s : -1;  // a row past the last sees nothing
  const _Float16* kbase = static_cast<const _Float16*>(a.k) + static_cast<int64_t>(kv) * a.dim;
  const _Float16* vbase = static_cast<const _Float16*>(a.v) + static_cast<int64_t>(kv) * a.dim;
  const BatchPages pages(a, w.request);

  uint32_t kx[2][kC][2][4];  // [16-key half][c][half][word]
  uint32_t vx[8][kVWords];   // [key slot][word]
  const auto load_k = [&](int32_t t0, const int32_t (&entry)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const _Float16* p = kbase + (pages.Slot(entry[h], t0 + 16 * h) + j) * a.kv_stride;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half) LoadHalves<4, kLoad>(p, a.dim, 64 * c + 16 * g + 8 * half, kx[h][c][half]);
    }
  };
  const auto load_v = [&](int32_t t0, const int32_t (&entry)[2]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const _Float16* p = vbase + (pages.Slot(entry[e >> 2], t0 + 16 * (e >> 2)) + 4 * g + (e & 3)) * a.kv_stride;
#pragma unroll
      for (int i = 0; i < kVWords; i += kVPiece) {
        uint32_t x[kVPiece];
        LoadHalves<kVPiece, kLoad>(p, a.dim, DP / 16 * j + 2 * i, x);
#pragma unroll
        for (int n = 0; n < kVPiece; ++n) vx[e][i + n] = x[n];
      }
    }
  };
  int32_t u = w.begin + wave;
  const auto key_of = [&](int32_t step) { return w.low + step * kKeys; };
  // A 16-key half that no row sees needs no page.
  const auto entries = [&](int32_t t0, int32_t (&entry)[2]) {
    entry[0] = pages.Entry(t0);
    entry[1] = pages.Entry(t0 + 16);
  };
  const auto uniform = [](const int32_t (&from)[2], int32_t (&to)[2]) {
    to[0] = __builtin_amdgcn_readfirstlane(from[0]);
    to[1] = __builtin_amdgcn_readfirstlane(from[1]);
  };
  int32_t entry[2] = {-1, -1}, entry_next[2] = {-1, -1};
  if (u < w.end) {
    entries(key_of(u), entry);
    if (u + kStepWaves < w.end) entries(key_of(u + kStepWaves), entry_next);
  }
  // The row's queries: piece (c, half) of dims 64c + 16g + 8 half .. + 7.
  float x[kC][16];
  {
    const float* q = a.q + (w.start + s) * a.q_stride + static_cast<int64_t>(kv * group + (row - s * group)) * a.dim;
    const bool vec = BatchQueryVec(a);
#pragma unroll
    for (int i = 0; i < kC; ++i) LoadBatchQuery(q, a.dim, 64 * i + 16 * g, vec, x[i]);
  }
  const bool stored = BatchRowStored(a, w.start + s);
  if (u < w.end) {
    uniform(entry, entry);
    load_k(key_of(u), entry);
    load_v(key_of(u), entry);
  }
  __builtin_amdgcn_sched_barrier(0);
  h8 qh[kC][2], ql[kC][2];
  float factor;  // takes the row's scale out of its scores again
  {
    uint32_t top = 0;
    if (a.dim < DP) {
#pragma unroll
      for (int i = 0; i < kC; ++i) MaskQuery(a.dim, 64 * i + 16 * g, x[i]);
    }
#pragma unroll
    for (int i = 0; i < kC; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
    top = max(top, XorLane<16>(top));
    top = max(top, XorLane<32>(top));
    const float scale = top >= 0x7f800000u || !stored ? NAN : RowScale(top);  // no finite row: all of it NaN
    factor = 1.f / scale * a.factor;
#pragma unroll
    for (int i = 0; i < kC; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        h2 hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y0 = x[i][8 * half + 2 * e] * scale, y1 = x[i][8 * half + 2 * e + 1] * scale;
          SplitF16Nearest(y0, y1, hi[e], lo[e]);
        }
        qh[i][half] = Join(hi[0], hi[1], hi[2], hi[3]);
        ql[i][half] = Join(lo[0], lo[1], lo[2], lo[3]);
      }
  }

  float m = -INFINITY, l = 0.f;  // l: this lane's share of the row's sum
  f4 acc[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
  for (; u < w.end; u += kStepWaves) {  // uniform over the wave
    const int32_t t0 = key_of(u);
    const bool more = u + kStepWaves < w.end;
    const int32_t next = key_of(u + kStepWaves);
    // The second parts' products first: they are rounded among themselves, before the sums are large.
    f4 st[2];
    float zk[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      st[h] = f4{0.f, 0.f, 0.f, 0.f};
      zk[h] = pages.Is(entry[h]) ? 0.f : NAN;
      h8 k8[kC][2];
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          k8[c][half] = __builtin_bit_cast(h8, u4{kx[h][c][half][0], kx[h][c][half][1], kx[h][c][half][2], kx[h][c][half][3]});
          st[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[c][half], ql[c][half], st[h], 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) zk[h] = Finite(kx[h][c][half][e], zk[h]);
        }
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          st[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[c][half], qh[c][half], st[h], 0, 0, 0);
    }
    int32_t entry_v[2];
    uniform(entry_next, entry_v);
    if (more) {
      load_k(next, entry_v);
      if (u + 2 * kStepWaves < w.end) entries(key_of(u + 2 * kStepWaves), entry_next);
    }
    __builtin_amdgcn_sched_barrier(0);
    float zv[8], z = zk[0] + zk[1];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      zv[e] = 0.f;
#pragma unroll
      for (int i = 0; i < kVWords; ++i) zv[e] = Finite(vx[e][i], zv[e]);
      z += zv[e];
    }
    uint32_t bad = 0;  // of the lane's keys
    if (__any(!(z == 0.f))) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t lanes = __ballot(!(zk[h] == 0.f));
        const uint32_t keys = static_cast<uint32_t>(lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) & 0xffffu;
        bad |= (keys >> (4 * g) & 15u) << (4 * h);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((__ballot(!(zv[e] == 0.f)) >> (16 * g) & 0xffffu) != 0) {
          bad |= 1u << e;
#pragma unroll
          for (int i = 0; i < kVWords; ++i) vx[e][i] = 0;
        }
    }
    const int32_t last = t0 + kKeys - 1;
    const bool whole = last <= w.p_first && t0 > w.p_last - a.window;  // a row past the last may see what it likes
    float p[8];
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = st[e >> 2][e & 3] * factor;
    if (!whole || __any(bad != 0)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = whole || SeesKey(a, p_row, t0 + 16 * (e >> 2) + 4 * g + (e & 3));
        p[e] = in ? (bad >> e & 1 ? NAN : p[e]) : -INFINITY;
        st[e >> 2][e & 3] = bad >> e & 1 ? NAN : st[e >> 2][e & 3];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, p[e]);
    mx = fmaxf(mx, XorLane<16>(mx));
    mx = fmaxf(mx, XorLane<32>(mx));
    const float m_old = m;
    if (mx > m + (kHeadroom + kSlack)) m = mx - kHeadroom;
    const float base = m == -INFINITY ? 0.f : m;
    const float corr = __builtin_amdgcn_exp2f(m_old - base);
    float sum = 0.f;
    const bool far_scores = __any(fabsf(base) >= kFarScore);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // The product once more, unrounded: near the reference little is left of it.
      const float y = far_scores ? p[e] - base : __builtin_fmaf(st[e >> 2][e & 3], factor, -base);
      p[e] = __builtin_amdgcn_exp2f(whole || p[e] != -INFINITY ? y : -INFINITY);
      sum += p[e];
    }
    l = l * corr + sum;
    if (__any(corr != 1.f)) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) acc[t] *= corr;
    }
    h2 ph[4], pl[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) SplitWeights(p[2 * e], p[2 * e + 1], ph[e], pl[e]);
    const h8 p_hi = Join(ph[0], ph[1], ph[2], ph[3]), p_lo = Join(pl[0], pl[1], pl[2], pl[3]);
#pragma unroll
    for (int i = 0; i < kVWords; ++i) {
      u4 lo4, hi4;  // dims 2i and 2i + 1 of the keys in pairs
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo4[e] = __builtin_amdgcn_perm(vx[2 * e + 1][i], vx[2 * e][i], 0x05040100u);
        hi4[e] = __builtin_amdgcn_perm(vx[2 * e + 1][i], vx[2 * e][i], 0x07060302u);
      }
      const h8 v0 = __builtin_bit_cast(h8, lo4), v1 = __builtin_bit_cast(h8, hi4);
      acc[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p_hi, acc[2 * i], 0, 0, 0);
      acc[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p_hi, acc[2 * i + 1], 0, 0, 0);
      acc[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p_lo, acc[2 * i], 0, 0, 0);
      acc[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p_lo, acc[2 * i + 1], 0, 0, 0);
    }
    if (more) load_v(next, entry_v);
    entry[0] = entry_v[0];
    entry[1] = entry_v[1];
  }
  // acc[t][r] is O^T[dim DP / 16 (4g + r) + t][row j].
  l = l + XorLane<16>(l);
  l = l + XorLane<32>(l);
  if (g == 0) {
    parts.m[wave][j] = m;
    parts.l[wave][j] = l;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int t = 0; t < kTiles; t += 4)
      *reinterpret_cast<f4*>(&parts.o[wave][j][kTiles * (4 * g + r) + t]) =
          f4{acc[t][r], acc[t + 1][r], acc[t + 2][r], acc[t + 3][r]};
  __syncthreads();
  parts.Join(a, b, w, group, kv);
}


// A workgroup's tile of few rows, of any type.
template <int DP, bool kHalf, int kLoad, bool kPaged>
__device__ __forceinline__ void StepGroup(const BatchAttendArgs& a, const BatchSplit& b, int32_t block, BatchParts<DP>& parts,
                                          BatchScan<kBatchThreads>& scan) {
  if constexpr (kHalf) StepF16Group<DP, kLoad>(a, b, block, parts, scan);
  else StepF32Group<DP, kLoad, kPaged>(a, b, block, parts, scan);
}

}  // namespace accel_hip
