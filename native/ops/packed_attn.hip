// Attention over packed sequences (one token axis, sequences one after the
// other), grouped heads, causal or not, forward and gradient, for 16-bit
// inputs with fp32 accumulation; head dimension 64 or 128.
//
//   o_i = sum_j p_ij v_j,  p_ij = softmax_j(s q_i k_j) over the keys j of row
//   i's own sequence (j <= i when causal), after an optional prefix whose keys
//   and values every sequence sees.  A row that sees nothing (padding) is 0.
//   dV_j = sum_i p_ij dO_i          dP_ij = dO_i v_j      D_i = dO_i o_i
//   dS = p (dP - D)   dQ_i = s sum_j dS_ij k_j   dK_j = s sum_i dS_ij q_i
//
// P is rounded to 16 bits once in the forward, P and dS once each in the
// gradient: the matrix instructions take 16-bit operands, and a second one for
// what the rounding dropped would be half as many products again.  It shows as
// an error of up to 2.2e-3 (o) and 2.4e-3 (o and gradients) of the norm in bf16,
// where the rounding of the result alone is 1.7e-3.  Sums, row statistics and
// states are fp32.
//
// D comes from the unrounded o: the forward also stores what its rounding
// dropped (one more 16-bit value per element of o, 134 MB at 16,384 rows of 32
// heads x 128), since D is subtracted from every dP of the row and an error of
// o's rounding would move them all one way: 2.6e-3 in bf16 with centred values,
// far more where keys and values have a common mean.
//
// One workgroup = 4 waves = 128 rows of one sequence and head (a job of the
// batch's plan, longest sweep first); q, k, v are read through their strides,
// so slices of a fused projection need no copy.  Tiles of 64 keys go HBM ->
// LDS by DMA, double buffered, one barrier per tile; a tile that straddles the
// sequence's end is loaded with zeros past it, so what the next sequence (or
// nothing) holds there never enters.
//
// Bounds, measured in bf16 with 32 / 8 heads: one sequence of 16,384 rows,
// causal, D 128, runs at 1.09 to 1.15 PF/s forward (1.92 to 2.02 ms, by the
// card), 1.18 to 1.24 in dQ (2.65 to 2.79 ms) and 1.08 to 1.13 in dK / dV (3.89
// to 4.06 ms), a plain matrix product of 8,192^3 at 1.37; the matrix cores are
// busy 63, 67 and 57 % of the time and the clock is down to 1.77 GHz at the
// card's power limit (operands of zeros run 25 % faster), so fewer operations
// would help, a better schedule does not.  At D 64 the softmax weighs twice as
// much: 32 exponentials and as many multiply-adds per 16 matrix instructions,
// 0.94 PF/s at 8,000 rows.  Ragged batches (24 documents of 64 to 4,096 rows:
// 0.23 + 0.35 + 0.41 ms, 580 TF/s over all three) keep the matrix cores busy 36,
// 36 and 41 %: the SIMDs hold 2.3, 1.7 and 1.3 waves of 3, 2 and 2 on average
// (2.7, 1.9 and 1.7 at 16,384 rows), which wait for loads and barriers 25 to 32
// % of their time (19 to 27).  Masked and empty keys are 8 % of the products.
//
// Tried and slower: 8 waves and 256 rows per tile (documents 210 -> 235 us),
// two workgroup halves on alternate tiles where there are workgroups enough (32
// prompts of 16 to 1,024 rows, D 64: 39.8 -> 46.8 us), the next tile's S product
// under this tile's exponentials (40.7 -> 43.3 us: registers),
// row sums as dot products of the packed pairs (1.98 -> 2.01 ms), 64 rows per
// wave for half the LDS reads (1.91 -> 2.37 ms), tiles of 32 keys (D 64: 33.9 ->
// 39 us for 16 short prompts behind 1,000 shared keys), an L2 prefetch two
// steps ahead in dK / dV (8.57 -> 8.82 ms, all three kernels).
#include <algorithm>
#include <type_traits>

#include "attn_tile.h"

using namespace kgwe;

namespace {

typedef unsigned short u16;
// On a lambda that the compiler might call instead (a call keeps its captured
// tiles in memory: 9 times the time).
#define KGWE_INLINE __attribute__((always_inline))

constexpr int kRows = 128;    // rows of a job (packed_plan.hip)
constexpr int kTile = 64;     // keys per tile
constexpr float kLog2e = 1.4426950408889634f;

// Sequences of up to this many rows.  A row of two or three keys has nothing
// for the roundings to average out over: with dS as one 16-bit value and D from
// an o whose P was rounded, dQ and dK were up to 1.8 times the rounding of the
// result off there (1.45 times in longer sequences).  These few take D as the
// sum of P dP, and dS as two 16-bit values; o is not read again, nor its low part
// written.
constexpr int kShort = kTile;

struct View {
  const u16* p;
  int64_t row, head;  // strides in elements
};

struct Batch {
  const int4* jobs;
  int T, Hq, Hkv, G;
  Div by_hq, by_hkv, by_g;
};

// A workgroup's block of a sequence: `rows` rows from `row0` on, of which it
// takes 128 from 128 * blk on; `keys` of them are keys too (padding: none).
struct Job {
  int row0, rows, blk, keys;
};

// Job and head of this workgroup: all heads of a job are neighbours, and on
// Hq % 8 == 0 each of the 8 XCDs (workgroups go round them) takes a contiguous
// run of heads, so the heads that share keys share an L2.
__device__ __forceinline__ bool pick(const Batch& b, int heads, Div by_heads, Job* job, int* head) {
  const int j = by_heads(blockIdx.x), p = blockIdx.x - j * heads;
  *head = heads % 8 == 0 ? (p % 8) * (heads / 8) + p / 8 : p;
  const int4 v = b.jobs[j];
  job->row0 = __builtin_amdgcn_readfirstlane(v.x);
  job->rows = __builtin_amdgcn_readfirstlane(v.y);
  job->blk = __builtin_amdgcn_readfirstlane(v.z);
  job->keys = __builtin_amdgcn_readfirstlane(v.w);
  return job->rows > 0;
}

// A block of few rows (a short sequence, or the end of one) would keep one or
// two of the workgroup's four waves busy, and always the same ones.  Where the
// group has the heads for it, 4 heads share a workgroup at 32 rows or less and
// 2 at 64 or less; the workgroups of the other heads leave.  Moves *head to
// this wave's head; returns the wave's first row in the sequence, -1: leave.
__device__ __forceinline__ int wave_rows(const Batch& b, const Job& job, int wave, int* head) {
  const int here = job.rows - job.blk * kRows;
  const int share = here <= 32 && b.G % 4 == 0 ? 2 : here <= 64 && b.G % 2 == 0 ? 1 : 0;  // log2
  if (*head & ((1 << share) - 1)) return -1;
  const int per = 2 - share;  // log2 of the waves per head
  *head += wave >> per;
  return job.blk * kRows + 32 * (wave & ((1 << per) - 1));
}

// The gradient's 16-bit operands, P and dS, in fp16.  At their natural size P =
// 1 / n and dS = P (dP - D) of long rows fall among fp16's steps of 2^-24 (dQ for
// incoming gradients of 1e-3 was off by 1.1e-2 of its norm at 12,000 keys, by
// 3.7e-2 at 40,000; it is 1.2e-3 and 2.1e-3, of which the result's own rounding
// 1.1e-3 and 2.1e-3), and dS of large incoming gradients passes its largest
// value, 65,504, where dQ and dK do not.  bf16 has fp32's range.
//   P is at most 1: it is lifted by 2^14, by way of the stored row sums.
//   dS has no bound that is worth having, so every accumulated row (of dQ or
//   dK) has a factor of its own, a power of two from 2^60 down: where a tile's
//   dS would pass 2^15 the factor and the sums so far are scaled down together,
//   the largest to 2^13 .. 2^14.  What is 2^27 below a row's largest dS still
//   counts in full.
// Factors are powers of two and leave the accumulators through the result's own
// multiplier, so they round nothing.  The maxima cost 3 to 8 % of a training
// call (16,384 rows, 32 / 8 heads x 128: 8.91 -> 9.19 ms, 300 sequences of 10 to
// 60 rows 269 -> 285 us).
template <class T>
constexpr bool kScaled = std::is_same<T, Fp16>::value;
template <class T>
constexpr int kLiftP = kScaled<T> ? 14 : 0;  // log2; stored row sums are lse - kLiftP
constexpr int kFirst = 60;  // log2 of the first factor: times any dS of fp16 inputs far below fp32's largest
constexpr float kTop = 32768.f;

// Largest magnitude in the accumulator row that this lane and its partner hold.
__device__ __forceinline__ float row_top(const f32x16& p) {
  float top = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(p[r]));
  return half_max(top);
}

// log2 of what brings a row's largest dS back to 2^13 .. 2^14, 0 where it has
// room (and for infinity, which nothing brings back).
__device__ __forceinline__ int fit(float top) {
  return top > kTop && top < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
}

struct FwdArgs {
  Batch b;
  View q, k, v, pk, pv;
  u16* o;      // [T, Hq, D]
  u16* o_low;  // what the rounding of o dropped, rounded in turn; null: not wanted
  float* lse;  // [Hq, T], log2 units, less kLiftP; null: not wanted
  int P, causal;
  float c;     // scale * log2 e
};

// TWO_V: V tiles are double-buffered as K tiles are.  At D = 128 one V buffer
// (V(t) is fetched during the tile's own scores, one more barrier) leaves room
// for a third workgroup on the CU, which is worth more where there are
// workgroups enough (see fwd()).
// HALVES = 2: 8 waves, of which the second four walk every other tile of the
// same rows; the halves' states meet in LDS at the end.
template <class T, int D, bool PREFIX, bool TWO_V, int HALVES>
__global__ __launch_bounds__(256 * HALVES, HALVES == 2 ? 1 : TWO_V ? 2 : 3) void packed_fwd_kernel(FwdArgs a) {
  constexpr int NB = D / 32, NT = D / 16;
  constexpr int kImg = kTile * D * 2;
  // One array per stage: the compiler orders an LDS read after every DMA in
  // flight that it cannot prove to go to another object.
  constexpr int kStage = HALVES * kImg;
  __shared__ __attribute__((aligned(1024))) char K0[kStage], V0[kStage], K1[kStage], V2[TWO_V ? kStage : 16];
  char* const V1 = TWO_V ? V2 : V0;
  Job job;
  int h;
  if (!pick(a.b, a.b.Hq, a.b.by_hq, &job, &h)) return;
  const int w8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = w8 & 3, half = HALVES == 1 ? 0 : w8 >> 2;  // row group, key half
  const int hkv = a.b.by_g(h), q0 = wave_rows(a.b, job, w, &h);
  if (q0 < 0) return;
  const int row0 = job.row0, len = job.rows, blk = job.blk;
  const int klen = job.keys;  // padding rows see nothing
  const int plen = PREFIX && klen > 0 ? a.P : 0;
  const int lane = threadIdx.x & 63;
  const int lq = lane & 31, hh = lane >> 5;
  const int qrow = q0 + lq;
  const bool mine = q0 < len;  // wave-uniform: this wave has rows

  bf16x8 qf[NT];
  {
    const u16* qp = a.q.p + (static_cast<int64_t>(row0) + qrow) * a.q.row + h * a.q.head;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      qf[t] = qrow < len ? *reinterpret_cast<const bf16x8*>(qp + 16 * t + 8 * hh) : bf16x8{};
  }
  f32x16 oacc[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) oacc[i] = f32x16{};
  float m = -INFINITY, l = 0.f;

  const int ntp = (plen + kTile - 1) / kTile;
  const int kv_end = a.causal ? min(klen, blk * kRows + kRows) : klen;
  const int nt = ntp + (kv_end + kTile - 1) / kTile;
  const TileDma<D, kTile> dma(w, lane);
  const TileAddr<D> ad(lane);
  const u16* kb = a.k.p + static_cast<int64_t>(row0) * a.k.row + hkv * a.k.head;
  const u16* vb = a.v.p + static_cast<int64_t>(row0) * a.v.row + hkv * a.v.head;
  const u16* pkb = PREFIX ? a.pk.p + hkv * a.pk.head : nullptr;
  const u16* pvb = PREFIX ? a.pv.p + hkv * a.pv.head : nullptr;

  auto load = [&](bool keys, char* dst, int t) {
    const bool pre = PREFIX && t < ntp;
    const int k0 = (pre ? t : t - ntp) * kTile;
    const int rows = min(kTile, (pre ? plen : klen) - k0);
    const int64_t row = keys ? (pre ? a.pk.row : a.k.row) : (pre ? a.pv.row : a.v.row);
    const u16* from = keys ? (pre ? pkb : kb) : (pre ? pvb : vb);
    const int bytes = static_cast<int>(2 * row);
    dma.load(row_buffer(from + k0 * row, rows, bytes), bytes, dst);
  };

  const int mine_at = half * kImg;  // this half's tile of a stage
  auto tile = [&](const char* Ks, const char* Vs, char* Kn, char* Vn, int t) {
    const char *Kc = Ks + mine_at, *Vc = Vs + mine_at;
    if constexpr (!TWO_V) load(false, Vn, t);
    if (t + HALVES < nt) {  // lands during this tile's work
      load(true, Kn + mine_at, t + HALVES);
      if constexpr (TWO_V) load(false, Vn + mine_at, t + HALVES);
    }
    const bool pre = PREFIX && t < ntp;
    const int k0 = (pre ? t : t - ntp) * kTile;
    const bool causal = a.causal && !pre;
    // else: the tile is past this wave's diagonal, or the other half had the last one
    const bool sees = mine && (HALVES == 1 || t < nt) && (!causal || k0 <= q0 + 31);
    u32x4 pb[4];
    if (sees) {
      // S^T = K Q^T: key on the accumulator's rows, query on the lane
      f32x16 s[2];
      s[0] = s[1] = f32x16{};
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int u = 0; u < NT; ++u) s[st] = mfma32<T>(ad.rows(Kc, 32 * st, u), qf[u], s[st]);
      const int kend = pre ? plen : klen;
      const bool edge = (causal && k0 + kTile - 1 > q0) || k0 + kTile > kend;  // wave-uniform
      if (edge) {
        // Last key this row sees, counted as tile_row counts without its lane part.
        const int last = (causal ? min(kend - 1, qrow) : kend - 1) - k0 - 4 * hh;
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * st + tile_row(r, 0) > last) s[st][r] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[st][r]);
      const float m_new = next_max<T>(half_max(mx), a.c, m);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      if (__any(m_new > m && m > -INFINITY)) {  // before a row's first max there is nothing to rescale
        const float alpha = exp2_fast(m - m_use);
        l *= alpha;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[i][r] *= alpha;
      }
      m = m_new;
      // P = 2^(S c - m) in pairs; the accumulator tile is the next product's operand as it is
      float r0 = 0.f, r1 = 0.f;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float p0 = exp2_fast(fmaf(s[st][r], a.c, -m_use));
          const float p1 = exp2_fast(fmaf(s[st][r + 1], a.c, -m_use));
          r0 += p0;
          r1 += p1;
          pb[2 * st + (r >> 3)][(r & 7) >> 1] = pack2<T>(p0, p1);
        }
      l += r0 + r1;  // this lane half's keys; the halves meet in the epilogue
    }
    if constexpr (!TWO_V) {  // V(t) has landed, K(t + 1) may be on its way
      if (t + 1 < nt) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(TileDma<D, kTile>::kN) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    if (sees) {  // O^T += V^T P
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int db = 0; db < NB; ++db) oacc[db] = mfma32<T>(ad.cols(Vc, 16 * u, db), as_op(pb[u]), oacc[db]);
    }
    dma_join();
  };

  if (nt > 0) {
    if (half < nt) {
      load(true, K0 + mine_at, half);
      if constexpr (TWO_V) load(false, V0 + mine_at, half);
    }
    // The Q loads end before the loop: sunk into it, they would make the
    // first products of every tile wait for the next tile's DMA.
#pragma unroll
    for (int t = 0; t < NT; ++t) asm volatile("" ::"v"(qf[t]));
    dma_join();
    for (int t = 0; t < nt; t += 2 * HALVES) {
      tile(K0, V0, K1, V1, t + half);
      if (t + HALVES < nt) tile(K1, V1, K0, V0, t + HALVES + half);
    }
  }
  if constexpr (HALVES == 2) {
    // The second half's state of each lane, lane after lane (every tile buffer
    // is free: the last step ended with a barrier).
    __shared__ float2 ml[4][64];
    char* at = (w == 0 ? K0 : w == 1 ? V0 : w == 2 ? K1 : V1) + 16 * lane;
    static_assert(NB * 4 * 1024 <= kStage, "a wave's state fits a stage buffer");
    if (half == 1) {
      ml[w][lane] = {m, l};
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(at + 1024 * (4 * i + g)) =
              f32x4{oacc[i][4 * g], oacc[i][4 * g + 1], oacc[i][4 * g + 2], oacc[i][4 * g + 3]};
    }
    __syncthreads();
    if (half == 1) return;
    const float2 o = ml[w][lane];
    const float M = fmaxf(m, o.x), M_use = M == -INFINITY ? 0.f : M;
    const float f0 = exp2_fast(m - M_use), f1 = exp2_fast(o.x - M_use);
    m = M;
    l = l * f0 + o.y * f1;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(at + 1024 * (4 * i + g));
#pragma unroll
        for (int j = 0; j < 4; ++j) oacc[i][4 * g + j] = oacc[i][4 * g + j] * f0 + v[j] * f1;
      }
  }
  const float lt = half_add(l);
  const bool ok = qrow < len;
  const int64_t orow = static_cast<int64_t>(row0) + qrow;
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  const int64_t off = (orow * a.b.Hq + h) * D;
  store_row<T, NB>(a.o + off, oacc, inv, hh, ok);
  if (a.o_low != nullptr && klen > kShort) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[i][r] = oacc[i][r] * inv - T::up(T::down(oacc[i][r] * inv));
    store_row<T, NB>(a.o_low + off, oacc, 1.f, hh, ok);
  }
  if (a.lse != nullptr && ok && hh == 0) {
    float z = lt == 0.f ? -INFINITY : m + log2f(lt) - kLiftP<T>;
    // Where a step of it is 1 and more it is rounded up, or P might pass its 2^14 by more than fp16 holds.
    if constexpr (kScaled<T>) z += fabsf(z) > 0x1p23f && lt != 0.f ? fabsf(z) * 0x1p-22f : 0.f;
    a.lse[static_cast<int64_t>(h) * a.b.T + orow] = z;
  }
}

struct BwdArgs {
  Batch b;
  View q, k, v;
  const u16* o;       // [T, Hq, D]
  const u16* o_low;
  const u16* dout;    // [T, Hq, D]
  const float* lse;   // [Hq, T]
  float* delta;       // [Hq, T], -D: written by the dQ kernel, read by the dK / dV kernel
  u16* dq;            // [T, Hq, D]
  u16* dk;            // [T, Hkv, D]
  u16* dv;
  float* part;        // [2, parts, T, Hkv, D], dK's then dV's; parts > 1 only
  int causal, parts, per;  // workgroups per key head, query heads of each
  Div by_parts, by_hkv_parts;
  float c, scale;
};

// What the rounding of two values to the pair `w` dropped, rounded in turn.
template <class T>
__device__ __forceinline__ unsigned pack2_low(float lo, float hi, unsigned w) {
  return pack2<T>(lo - T::up(static_cast<u16>(w)), hi - T::up(static_cast<u16>(w >> 16)));
}

// dQ: the forward's geometry (query on the lane).  Recomputes S^T and dP^T and
// accumulates dQ^T += K^T dS^T, K^T read transposed from the K image.  dQ and
// dK / dV are two kernels, 7 products where one kernel would need 5: that one
// would have to add dQ up by atomics, in an order that changes from run to run.
template <class T, int D>
__global__ __launch_bounds__(256, 2) void packed_dq_kernel(BwdArgs a) {
  constexpr int NB = D / 32, NT = D / 16;
  constexpr int kImg = kTile * D * 2;
  __shared__ __attribute__((aligned(1024))) char K0[kImg], V0[kImg], K1[kImg], V1[kImg];
  Job job;
  int h;
  if (!pick(a.b, a.b.Hq, a.b.by_hq, &job, &h)) return;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hkv = a.b.by_g(h), q0 = wave_rows(a.b, job, w, &h);
  if (q0 < 0) return;
  const int row0 = job.row0, len = job.rows, blk = job.blk, klen = job.keys;
  const int lane = threadIdx.x & 63;
  const int lq = lane & 31, hh = lane >> 5;
  const int qrow = q0 + lq;
  const bool mine = q0 < len;
  const bool ok = qrow < len;
  const int64_t row = static_cast<int64_t>(row0) + qrow;

  bf16x8 qf[NT], df[NT];
  float dsum = 0.f;
  {
    const u16* qp = a.q.p + row * a.q.row + h * a.q.head;
    const int64_t off = (row * a.b.Hq + h) * D;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      qf[t] = ok ? *reinterpret_cast<const bf16x8*>(qp + 16 * t + 8 * hh) : bf16x8{};
      df[t] = ok ? *reinterpret_cast<const bf16x8*>(a.dout + off + 16 * t + 8 * hh) : bf16x8{};
    }
    if (klen > kShort) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const bf16x8 ov = ok ? *reinterpret_cast<const bf16x8*>(a.o + off + 16 * t + 8 * hh) : bf16x8{};
        const bf16x8 lv = ok ? *reinterpret_cast<const bf16x8*>(a.o_low + off + 16 * t + 8 * hh) : bf16x8{};
#pragma unroll
        for (int e = 0; e < 8; ++e) dsum = fmaf(T::up(df[t][e]), T::up(ov[e]) + T::up(lv[e]), dsum);
      }
    }
  }
  const int64_t li = static_cast<int64_t>(h) * a.b.T + row;
  float lse = ok ? a.lse[li] : 0.f;
  if constexpr (kScaled<T>) lse += kLiftP<T>;
  float delta = half_add(dsum);
  int factor = kFirst;   // log2 of this row's
  float shift = -lse;    // of the exponents
  if constexpr (kScaled<T>) shift = factor - lse;
  f32x16 acc[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] = f32x16{};

  const int kv_end = a.causal ? min(klen, blk * kRows + kRows) : klen;
  const int nt = (kv_end + kTile - 1) / kTile;
  const TileDma<D, kTile> dma(w, lane);
  const TileAddr<D> ad(lane);
  const u16* kb = a.k.p + static_cast<int64_t>(row0) * a.k.row + hkv * a.k.head;
  const u16* vb = a.v.p + static_cast<int64_t>(row0) * a.v.row + hkv * a.v.head;
  const int kbytes = static_cast<int>(2 * a.k.row), vbytes = static_cast<int>(2 * a.v.row);
  auto load = [&](char* Kd, char* Vd, int t) KGWE_INLINE {
    const int k0 = t * kTile, rows = min(kTile, klen - k0);
    dma.load(row_buffer(kb + k0 * a.k.row, rows, kbytes), kbytes, Kd);
    dma.load(row_buffer(vb + k0 * a.v.row, rows, vbytes), vbytes, Vd);
  };
  // S^T and dP^T + d of 32 keys.
  auto scores = [&](const char* Kc, const char* Vc, int st, float d, f32x16& s, f32x16& p) KGWE_INLINE {
    s = f32x16{};
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = d;  // dP - D without a subtraction
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      s = mfma32<T>(ad.rows(Kc, 32 * st, u), qf[u], s);
      p = mfma32<T>(ad.rows(Vc, 32 * st, u), df[u], p);
    }
  };
  auto tile = [&](auto brief_c, const char* Kc, const char* Vc, char* Kn, char* Vn, int t) KGWE_INLINE {
    if (t + 1 < nt) load(Kn, Vn, t + 1);
    const int k0 = t * kTile;
    if (mine && (!a.causal || k0 <= q0 + 31)) {
      const bool edge = (a.causal && k0 + kTile - 1 > q0) || k0 + kTile > klen;
      const int last = (a.causal ? min(klen - 1, qrow) : klen - 1) - k0 - 4 * hh;  // as in the forward
      // Two 32-key halves in turn: one S^T / dP^T pair live at a time.
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        f32x16 s, p;
        scores(Kc, Vc, st, -delta, s, p);
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] *= exp2_fast(fmaf(s[r], a.c, shift));
        if (edge) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * st + tile_row(r, 0) > last) p[r] = 0.f;
        }
        if constexpr (kScaled<T>) {
          const float top = row_top(p);
          if (__any(top > kTop)) {
            const int n = fit(top);
            const float f = ldexpf(1.f, n);
            factor += n;
            shift = factor - lse;
            p *= f;
#pragma unroll
            for (int db = 0; db < NB; ++db) acc[db] *= f;
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          u32x4 sw;
#pragma unroll
          for (int j = 0; j < 4; ++j) sw[j] = pack2<T>(p[8 * u + 2 * j], p[8 * u + 2 * j + 1]);
#pragma unroll
          for (int db = 0; db < NB; ++db)
            acc[db] = mfma32<T>(ad.cols(Kc, 32 * st + 16 * u, db), as_op(sw), acc[db]);
          if constexpr (brief_c.value) {
#pragma unroll
            for (int j = 0; j < 4; ++j) sw[j] = pack2_low<T>(p[8 * u + 2 * j], p[8 * u + 2 * j + 1], sw[j]);
#pragma unroll
            for (int db = 0; db < NB; ++db)
              acc[db] = mfma32<T>(ad.cols(Kc, 32 * st + 16 * u, db), as_op(sw), acc[db]);
          }
        }
      }
    }
    dma_join();
  };
  if (nt > 0) {
    load(K0, V0, 0);
#pragma unroll
    for (int t = 0; t < NT; ++t) asm volatile("" ::"v"(qf[t]), "v"(df[t]));
    asm volatile("" ::"v"(lse), "v"(delta));
    dma_join();
    if (klen <= kShort) {  // one tile
      if (mine) {
        const int last = a.causal ? min(klen - 1, qrow) : klen - 1;
        float d = 0.f;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          f32x16 s, p;
          scores(K0, V0, st, 0.f, s, p);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * st + tile_row(r, hh) <= last) d = fmaf(exp2_fast(fmaf(s[r], a.c, -lse)), p[r], d);
        }
        delta = half_add(d);
      }
      tile(std::true_type{}, K0, V0, K1, V1, 0);
    } else {
      for (int t = 0; t < nt; t += 2) {
        tile(std::false_type{}, K0, V0, K1, V1, t);
        if (t + 1 < nt) tile(std::false_type{}, K1, V1, K0, V0, t + 1);
      }
    }
  }
  if (hh == 0 && ok) a.delta[li] = -delta;
  float mul = a.scale;
  if constexpr (kScaled<T>) mul = ldexpf(mul, -factor);
  store_row<T, NB>(a.dq + (row * a.b.Hq + h) * D, acc, mul, hh, ok);
}

constexpr int kQt = 32;  // query rows per step of the dK / dV sweep

// dK, dV: 128 keys of one sequence and key head, 32 per wave (key on the
// lane), swept by every query head of the group and every query tile that sees
// them, last tile first.  P and dS feed the next products as they are; Q and
// dO are read by rows for S and dP and by columns for dV and dK.  Where that
// would leave the chip short of workgroups, `parts` of them share a group's
// query heads and their sums are joined by packed_join_kernel (see bwd()).
template <class T, int D>
__global__ __launch_bounds__(256, 2) void packed_dkv_kernel(BwdArgs a) {
  constexpr int NB = D / 32, NT = D / 16;
  constexpr int kImg = kQt * D * 2;
  __shared__ __attribute__((aligned(1024))) char Q0[kImg], O0[kImg], Q1[kImg], O1[kImg];
  __shared__ __attribute__((aligned(1024))) char Vw[kRows * D * 2];
  __shared__ __attribute__((aligned(256))) float L0[64], L1[64];  // lse and -D of a tile's 32 rows
  Job job;
  int hkv;
  if (!pick(a.b, a.b.Hkv * a.parts, a.by_hkv_parts, &job, &hkv)) return;
  const int unit = hkv;
  hkv = a.by_parts(unit);
  const int part = unit - hkv * a.parts;
  const int G = a.b.G, g_begin = part * a.per, g_end = min(G, g_begin + a.per);
  const int row0 = job.row0, len = job.rows;
  const int qlen = job.keys;  // nothing looks at padding
  const int nblk = (len + kRows - 1) / kRows;
  const int kb = nblk - 1 - job.blk;  // the job table's order, mirrored: the first keys sweep longest
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lk = lane & 31, hh = lane >> 5;
  const int key0 = kb * kRows + w * 32, key = key0 + lk;
  const bool ok = key < len;
  const int64_t krow = static_cast<int64_t>(row0) + key;

  const TileDma<D, kQt> dma(w, lane);
  const TileAddr<D> ad(lane);
  const int vbytes = static_cast<int>(2 * a.v.row), qbytes = static_cast<int>(2 * a.q.row);
  const int obytes = 2 * a.b.Hq * D;
  {
    const TileDma<D, kRows> vdma(w, lane);
    const int v0 = kb * kRows;
    vdma.load(row_buffer(a.v.p + (static_cast<int64_t>(row0) + v0) * a.v.row + hkv * a.v.head, min(kRows, len - v0),
                         vbytes), vbytes, Vw);
  }
  bf16x8 kf[NT];
  {
    const u16* kp = a.k.p + krow * a.k.row + hkv * a.k.head;
#pragma unroll
    for (int t = 0; t < NT; ++t) kf[t] = ok ? *reinterpret_cast<const bf16x8*>(kp + 16 * t + 8 * hh) : bf16x8{};
  }
  f32x16 dka[NB], dva[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) dka[i] = dva[i] = f32x16{};
  float factor = ldexpf(1.f, kFirst - kLiftP<T>);  // this key's, besides P's

  const int nq = (qlen + kQt - 1) / kQt;
  const int first = a.causal ? kb * (kRows / kQt) : 0;
  const int total = max(0, nq - first) * (g_end - g_begin);
  auto load = [&](char* Qd, char* Od, float* Ld, int qt, int g) KGWE_INLINE {
    const int h = hkv * G + g, s0 = qt * kQt, rows = min(kQt, qlen - s0);
    const int64_t r = static_cast<int64_t>(row0) + s0;
    dma.load(row_buffer(a.q.p + r * a.q.row + h * a.q.head, rows, qbytes), qbytes, Qd);
    dma.load(row_buffer(a.dout + (r * a.b.Hq + h) * D, rows, obytes), obytes, Od);
    if (w < 2 && lane < 32) {  // wave 0: lse, wave 1: -D
      const float* src = (w == 0 ? a.lse : a.delta) + static_cast<int64_t>(h) * a.b.T + r;
      dma_lane<4>(row_buffer(src, rows, 4), 4 * lane, Ld + 32 * w);
    }
  };
  int qt = nq - 1, g = g_begin;
  auto step = [&](auto brief_c, const char* Qc, const char* Oc, const float* Lc, char* Qn, char* On, float* Ln,
                  bool more) KGWE_INLINE {
    const bool wrap = g + 1 == g_end;
    const int g2 = wrap ? g_begin : g + 1, qt2 = wrap ? qt - 1 : qt;
    if (more) load(Qn, On, Ln, qt2, g2);
    const int qb = qt * kQt;
    if (key0 < len && (!a.causal || qb + kQt - 1 >= key0)) {  // else every query here precedes our keys
      f32x16 s = f32x16{}, p;  // p starts from -D: dP - D without a subtraction
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const f32x4 de = *reinterpret_cast<const f32x4*>(Lc + 32 + 8 * g4 + 4 * hh);
#pragma unroll
        for (int j = 0; j < 4; ++j) p[4 * g4 + j] = de[j];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        s = mfma32<T>(ad.rows(Qc, 0, t), kf[t], s);
        p = mfma32<T>(ad.rows(Oc, 0, t), ad.rows(Vw, 32 * w, t), p);
      }
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(Lc + 8 * g4 + 4 * hh);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * g4 + j;
          s[r] = exp2_fast(fmaf(s[r], a.c, -ls[j]));
          p[r] *= s[r];
        }
      }
      // A branch around the masking: selected element by element in the line
      // above it cost 80 of the step's 185 vector instructions.
      if (a.causal && key0 + 31 > qb) {
        const int before = key - qb - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (tile_row(r, 0) < before) s[r] = p[r] = 0.f;
      }
      if constexpr (kScaled<T>) {
        const float top = row_top(p) * factor;
        if (__any(top > kTop)) {
          const float f = ldexpf(1.f, fit(top));
          factor *= f;
#pragma unroll
          for (int db = 0; db < NB; ++db) dka[db] *= f;
        }
        p *= factor;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4 pw, sw;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pw[j] = pack2<T>(s[8 * u + 2 * j], s[8 * u + 2 * j + 1]);
          sw[j] = pack2<T>(p[8 * u + 2 * j], p[8 * u + 2 * j + 1]);
        }
#pragma unroll
        for (int db = 0; db < NB; ++db) {
          dva[db] = mfma32<T>(ad.cols(Oc, 16 * u, db), as_op(pw), dva[db]);
          dka[db] = mfma32<T>(ad.cols(Qc, 16 * u, db), as_op(sw), dka[db]);
        }
        if constexpr (brief_c.value) {
#pragma unroll
          for (int j = 0; j < 4; ++j) sw[j] = pack2_low<T>(p[8 * u + 2 * j], p[8 * u + 2 * j + 1], sw[j]);
#pragma unroll
          for (int db = 0; db < NB; ++db) dka[db] = mfma32<T>(ad.cols(Qc, 16 * u, db), as_op(sw), dka[db]);
        }
      }
    }
    dma_join();
    g = g2;
    qt = qt2;
  };
  if (total > 0) {
    load(Q0, O0, L0, qt, g);
#pragma unroll
    for (int t = 0; t < NT; ++t) asm volatile("" ::"v"(kf[t]));
    dma_join();
    auto sweep = [&](auto brief_c) KGWE_INLINE {
      for (int it = 0; it < total; it += 2) {
        step(brief_c, Q0, O0, L0, Q1, O1, L1, it + 1 < total);
        if (it + 1 < total) step(brief_c, Q1, O1, L1, Q0, O0, L0, it + 2 < total);
      }
    };
    if (qlen <= kShort) sweep(std::true_type{});
    else sweep(std::false_type{});
  } else {
    dma_join();  // the V image's DMA ends before the workgroup does
  }
  const int64_t off = (krow * a.b.Hkv + hkv) * D;
  float mul_k = 1.f, mul_v = 1.f;
  if constexpr (kScaled<T>) {
    mul_v = ldexpf(1.f, -kLiftP<T>);
    mul_k = mul_v / factor;
  }
  if (a.parts == 1) {
    store_row<T, NB>(a.dk + off, dka, a.scale * mul_k, hh, ok);
    store_row<T, NB>(a.dv + off, dva, mul_v, hh, ok);
  } else if (ok) {
    const int64_t all = static_cast<int64_t>(a.b.T) * a.b.Hkv * D;
    float* pk = a.part + part * all + off + 4 * hh;
    float* pv = pk + a.parts * all;
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        f32x4 x, y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = dka[db][4 * g4 + j] * mul_k;
          y[j] = dva[db][4 * g4 + j] * mul_v;
        }
        *reinterpret_cast<f32x4*>(pk + 32 * db + 8 * g4) = x;
        *reinterpret_cast<f32x4*>(pv + 32 * db + 8 * g4) = y;
      }
  }
}

// dK (y = 0) and dV (y = 1) of the parts' sums, in the parts' order; `all`
// elements of each.
template <class T>
__global__ __launch_bounds__(256) void packed_join_kernel(const float* __restrict__ part, int parts, int64_t all,
                                                          u16* dk, u16* dv, float scale) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i >= all) return;
  const float* p = part + blockIdx.y * parts * all + i;
  f32x4 lo = {}, hi = {};
  for (int j = 0; j < parts; ++j, p += all) {
    lo += *reinterpret_cast<const f32x4*>(p);
    hi += *reinterpret_cast<const f32x4*>(p + 4);
  }
  const float mul = blockIdx.y == 0 ? scale : 1.f;
  u32x4 v;
  v[0] = pack2<T>(lo[0] * mul, lo[1] * mul);
  v[1] = pack2<T>(lo[2] * mul, lo[3] * mul);
  v[2] = pack2<T>(hi[0] * mul, hi[1] * mul);
  v[3] = pack2<T>(hi[2] * mul, hi[3] * mul);
  *reinterpret_cast<u32x4*>((blockIdx.y == 0 ? dk : dv) + i) = v;
}

// Strides fit the kernels' 32-bit offsets inside a tile of 128 rows, and rows
// do not overlap: a descriptor's extent is counted in row strides.
inline bool view_ok(const void* p, int64_t row, int64_t head, int D) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row % 8 == 0 && head % 8 == 0 && row >= D && head >= 0 &&
         row <= (1 << 22);
}

inline bool shape_ok(int T, int J, int Hq, int Hkv, int D, int dtype) {
  return T > 0 && J > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && (D == 64 || D == 128) &&
         (dtype == kTypeBf16 || dtype == kTypeFp16) && static_cast<int64_t>(J) * Hq < (1LL << 31) &&
         static_cast<int64_t>(J) * Hq * Hq < (1LL << 32) &&
         static_cast<int64_t>(Hq) * D < (1 << 22);
}

template <class T, int D, bool TWO_V, int HALVES>
int fwd_as(const FwdArgs& a, int J, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(J) * a.b.Hq), threads(256 * HALVES);
  if (a.P > 0) hipLaunchKernelGGL((packed_fwd_kernel<T, D, true, TWO_V, HALVES>), grid, threads, 0, s, a);
  else hipLaunchKernelGGL((packed_fwd_kernel<T, D, false, TWO_V, HALVES>), grid, threads, 0, s, a);
  return KGWE_CHECK_LAUNCH();
}

// The form by the number of workgroups, 2.5 a CU being the border.
//
// Fewer: a workgroup's sweep is the call's time, so two halves share it where
// it is long, by the sequences' mean length (32 heads, one against two halves:
// 4 prompts of 20 to 200 rows behind 2,000 keys, D 64: 31.8 / 24.9 us, D 128:
// 43.5 / 34.2; one prompt of 1,000 rows 15.9 / 13.7 and 23.1 / 20.7, of 2,000
// 31.7 / 30.2 and 47.7 / 45.0; but 4 prompts of 200 to 800 rows 11.2 / 11.7 and
// 16.7 / 19.1, 4 of 1 to 61 rows 4.1 / 4.8).
//
// More: at D = 64 four workgroups fit a CU with two V buffers.  At D = 128 two
// do, three with one V buffer (two against one: 16,384 rows 1.96 / 1.89 ms,
// 4,000 rows 140 / 132 us, 16 short prompts behind 3,000 shared keys 146 / 119
// us; below the border 2,000 rows 47.4 / 49.7 us, 500 rows 13.4 / 14.6 us).
template <class T, int D>
int fwd(const FwdArgs& a, int J, hipStream_t s) {
  if (static_cast<int64_t>(J) * a.b.Hq < 640) {
    const int seqs = std::max(1, J - a.b.T / kRows - 1);  // how packed_plan.hip counts J
    if (a.P + a.b.T / seqs >= 640) return fwd_as<T, D, true, 2>(a, J, s);
  } else if (D == 128) {
    return fwd_as<T, D, D != 128, 1>(a, J, s);
  }
  return fwd_as<T, D, true, 1>(a, J, s);
}

template <class T, int D>
int bwd(const BwdArgs& a, int J, hipStream_t s) {
  hipLaunchKernelGGL((packed_dq_kernel<T, D>), dim3(static_cast<unsigned>(J) * a.b.Hq), dim3(256), 0, s, a);
  if (int rc = KGWE_CHECK_LAUNCH()) return rc;
  hipLaunchKernelGGL((packed_dkv_kernel<T, D>), dim3(static_cast<unsigned>(J) * a.b.Hkv * a.parts), dim3(256), 0, s, a);
  int rc = KGWE_CHECK_LAUNCH();
  if (rc || a.parts == 1) return rc;
  const int64_t all = static_cast<int64_t>(a.b.T) * a.b.Hkv * D;
  hipLaunchKernelGGL((packed_join_kernel<T>), dim3(static_cast<unsigned>((all / 8 + 255) / 256), 2), dim3(256), 0, s,
                     a.part, a.parts, all, a.dk, a.dv, a.scale);
  return KGWE_CHECK_LAUNCH();
}

// Workgroups per key head of the dK / dV kernel: the query heads of a group are
// shared out until there are 4 workgroups a CU (two run at a time, and their
// sweeps differ in length).  What the parts cost is fp32 sums, written and read
// once.  Forward + gradient, 32 / 8 heads x 128, without and with: 500 rows 105
// / 70 us, 2,000 rows 371 / 220 us, 4,096 rows 856 / 643 us, 8,192 rows 2.51 /
// 2.27 ms; 4,000 rows of 14 / 2 heads 1,057 / 363 us.  Up to 8 workgroups a CU:
// 16,384 rows 8.69 / 8.44 ms, but 8 documents of 500 to 2,000 rows 632 / 693 us.
constexpr int kFill = 1024;
inline int dkv_parts(int J, int Hkv, int G) {
  const int64_t have = static_cast<int64_t>(J) * Hkv;
  const int want = static_cast<int>(std::min<int64_t>(G, (kFill + have - 1) / have));
  const int per = (G + want - 1) / want;
  return (G + per - 1) / per;
}

}  // namespace

namespace {
inline Batch batch_of(const int* jobs, int T, int Hq, int Hkv) {
  return {reinterpret_cast<const int4*>(jobs), T, Hq, Hkv, Hq / Hkv, Div(Hq), Div(Hkv), Div(Hq / Hkv)};
}
}  // namespace

// One record per call in place of 27 and 25 arguments: converting them one by
// one cost the Python caller 3.6 us of a 11 us call, packing a record 0.8 us.
// Strides in elements; jobs [J, 4] from kgwe_packed_plan for the same T.
struct PackedFwdCall {
  const void *q, *k, *v, *pk, *pv;  // prefix keys / values [Hkv, P, D] by strides; P = 0: none
  void *o, *o_low;                  // contiguous [T, Hq, D]; o_low (or null) and
  float* lse;                       // [Hq, T] (or null) are what the gradient needs
  const int* jobs;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, pk_row, pk_head, pv_row, pv_head;
  int P, J, T, Hq, Hkv, D, causal, dtype;
  float scale;
};

struct PackedBwdCall {
  const void *q, *k, *v, *o, *o_low;  // o, o_low, lse: the forward's
  const float* lse;
  const void* dout;        // contiguous [T, Hq, D]
  float* delta;            // [Hq, T] workspace
  void *dq, *dk, *dv;      // [T, Hq, D], [T, Hkv, D]: contiguous, every row written
  float* work;             // kgwe_packed_attn_bwd_workspace words
  const int* jobs;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int J, T, Hq, Hkv, D, causal, dtype;
  float scale;
};

KGWE_API int kgwe_packed_attn_fwd_bytes() { return sizeof(PackedFwdCall); }
KGWE_API int kgwe_packed_attn_bwd_bytes() { return sizeof(PackedBwdCall); }

// fp32 words of workspace that a gradient needs besides delta; 0: none.
KGWE_API int64_t kgwe_packed_attn_bwd_workspace(int J, int T, int Hq, int Hkv, int D) {
  if (!shape_ok(T, J, Hq, Hkv, D, kTypeBf16)) return 0;  // refused by the call itself
  const int parts = dkv_parts(J, Hkv, Hq / Hkv);
  return parts == 1 ? 0 : 2 * static_cast<int64_t>(parts) * T * Hkv * D;
}

KGWE_API int kgwe_packed_attn_fwd(const PackedFwdCall* c, hipStream_t s) {
  if (!shape_ok(c->T, c->J, c->Hq, c->Hkv, c->D, c->dtype) || c->P < 0 || !c->o || !c->jobs) return -1;
  if (!view_ok(c->q, c->q_row, c->q_head, c->D) || !view_ok(c->k, c->k_row, c->k_head, c->D) ||
      !view_ok(c->v, c->v_row, c->v_head, c->D))
    return -1;
  if (c->P > 0 && (!c->pk || !c->pv || !view_ok(c->pk, c->pk_row, c->pk_head, c->D) ||
                   !view_ok(c->pv, c->pv_row, c->pv_head, c->D)))
    return -1;
  if ((reinterpret_cast<uintptr_t>(c->o) | reinterpret_cast<uintptr_t>(c->o_low) |
       reinterpret_cast<uintptr_t>(c->jobs)) & 15)
    return -1;
  auto in = [](const void* p) { return static_cast<const u16*>(p); };
  const FwdArgs a{batch_of(c->jobs, c->T, c->Hq, c->Hkv),
                  {in(c->q), c->q_row, c->q_head}, {in(c->k), c->k_row, c->k_head}, {in(c->v), c->v_row, c->v_head},
                  {in(c->pk), c->pk_row, c->pk_head}, {in(c->pv), c->pv_row, c->pv_head},
                  static_cast<u16*>(c->o), static_cast<u16*>(c->o_low), c->lse, c->P, c->causal, c->scale * kLog2e};
  if (c->dtype == kTypeBf16) return c->D == 64 ? fwd<Bf16, 64>(a, c->J, s) : fwd<Bf16, 128>(a, c->J, s);
  return c->D == 64 ? fwd<Fp16, 64>(a, c->J, s) : fwd<Fp16, 128>(a, c->J, s);
}

KGWE_API int kgwe_packed_attn_bwd(const PackedBwdCall* c, hipStream_t s) {
  if (!shape_ok(c->T, c->J, c->Hq, c->Hkv, c->D, c->dtype) || !c->lse || !c->delta || !c->jobs) return -1;
  if (!view_ok(c->q, c->q_row, c->q_head, c->D) || !view_ok(c->k, c->k_row, c->k_head, c->D) ||
      !view_ok(c->v, c->v_row, c->v_head, c->D))
    return -1;
  for (const void* p : {c->o, c->o_low, c->dout, static_cast<const void*>(c->dq), static_cast<const void*>(c->dk),
                        static_cast<const void*>(c->dv), static_cast<const void*>(c->jobs)})
    if (!p || (reinterpret_cast<uintptr_t>(p) & 15)) return -1;
  const int G = c->Hq / c->Hkv, parts = dkv_parts(c->J, c->Hkv, G);
  if (parts > 1 && (!c->work || (reinterpret_cast<uintptr_t>(c->work) & 15))) return -2;
  auto in = [](const void* p) { return static_cast<const u16*>(p); };
  const BwdArgs a{batch_of(c->jobs, c->T, c->Hq, c->Hkv),
                  {in(c->q), c->q_row, c->q_head}, {in(c->k), c->k_row, c->k_head}, {in(c->v), c->v_row, c->v_head},
                  in(c->o), in(c->o_low), in(c->dout), c->lse, c->delta, static_cast<u16*>(c->dq),
                  static_cast<u16*>(c->dk), static_cast<u16*>(c->dv), c->work, c->causal, parts,
                  (G + parts - 1) / parts, Div(parts), Div(c->Hkv * parts), c->scale * kLog2e, c->scale};
  if (c->dtype == kTypeBf16) return c->D == 64 ? bwd<Bf16, 64>(a, c->J, s) : bwd<Bf16, 128>(a, c->J, s);
  return c->D == 64 ? bwd<Fp16, 64>(a, c->J, s) : bwd<Fp16, 128>(a, c->J, s);
}
