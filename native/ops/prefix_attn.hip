// Attention of one query token per sequence where all sequences of the batch
// share a prefix: keys = the prefix's [Hkv, P, D], held once, then the
// sequence's own cache [B, Hkv, Smax, D] up to lens[b].
//
//   out[b, h] = sum_j softmax_j(s q[b, h] k_j) v_j,  j over prefix + own keys
//
// The bound is HBM: the prefix's keys and values have to be read once per
// step, not once per sequence.  The rows of one key head, B x G of them (G =
// Hq / Hkv), are therefore one matrix: a workgroup takes a chunk of the
// prefix's keys for 128 rows (or for all of them, where there are at most 32)
// on the matrix cores, another one chunks of single sequences' own keys for
// their G rows; a second small launch joins the chunks' (max, sum, output)
// states.  Where prefix and cache are short, one workgroup per (sequence, key
// head) walks both and nothing is joined.
//
// The grid depends on capacities only (P, Smax, B), never on lens, so a step
// can be captured in a graph and replayed at any length: the workgroups of the
// own keys count the chunks that hold keys from lens and take every o_wgs-th.
//
// Measured (32 / 8 heads, bf16, GPU time of a call): 64 rows, 32,768 shared
// keys and up to 1,500 own ones, D 128: 54 + 7.6 us, the second for the join
// (52.5 in all where the call repeats on the same inputs, which the last-level
// cache can hold); the 184 MB alone take 37 us at the card's copy rate, 3.4 TB/s
// is reached while every prefix key is also multiplied with 256 rows, by 1.2
// waves per SIMD.  32 rows, 2,048 + up to 1,000 keys, D 64: 8.2 + 3.9 us for 14
// MB, two launches whose waves wait 63 and 71 % of their time.  4 rows, 200 +
// up to 60 keys: 4.8 us, one launch.  1,024 rows, 500 + up to 1,000 keys,
// D 64: 123 us.
#include <algorithm>

#include "attn_tile.h"

using namespace kgwe;

namespace {

typedef unsigned short u16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWide = 64;      // keys per tile of the 128-row form, shared by 4 waves
constexpr int kSlim = 32;      // keys per tile of the 32-row form, one wave's own

struct Args {
  const u16* q;   // [B, Hq, D]
  const u16 *pk, *pv;
  int64_t p_row, p_head;
  const u16 *kc, *vc;  // [B, Hkv, Smax, D]
  const int* lens;
  u16* out;            // [B, Hq, D]
  float *part_o, *part_ml;  // [B * Hq, slots, D], [B * Hq, slots, 2]
  int B, Hq, Hkv, G, P, Smax;
  Div by_g, by_hkv;
  int p_chunk, p_splits, o_chunk, o_splits;  // splits 0: no workgroups of that kind
  int o_wgs;           // workgroups that share the own chunks
  int direct;          // one workgroup walks prefix and own keys and writes out
  float c;
};

// State of 32 query rows (row on the lane) over the keys seen so far.
template <class T, int D>
struct State {
  static constexpr int NB = D / 32, NT = D / 16;
  f32x16 o[NB];
  float m, l;
  __device__ __forceinline__ State() : m(-INFINITY), l(0.f) {
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x16{};
  }
  // Scores of NS x 32 keys (key on the accumulator's rows), of which the first
  // `valid` count -> P as the next product's operand.
  template <int NS>
  __device__ __forceinline__ void soften(f32x16 (&s)[NS], int valid, float c, int hh, u32x4 (&pb)[2 * NS]) {
    if (valid < 32 * NS) {
#pragma unroll
      for (int st = 0; st < NS; ++st)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * st + tile_row(r, 0) >= valid - 4 * hh) s[st][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[st][r]);
    const float m_new = next_max<T>(half_max(mx), c, m);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    if (__any(m_new > m && m > -INFINITY)) {  // before a row's first max there is nothing to rescale
      const float alpha = exp2_fast(m - m_use);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
    }
    m = m_new;
    float r0 = 0.f, r1 = 0.f;
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = exp2_fast(fmaf(s[st][r], c, -m_use)), p1 = exp2_fast(fmaf(s[st][r + 1], c, -m_use));
        r0 += p0;
        r1 += p1;
        pb[2 * st + (r >> 3)][(r & 7) >> 1] = pack2<T>(p0, p1);
      }
    l += r0 + r1;
  }
};

template <class T, int D>
__device__ __forceinline__ void load_q(const u16* qrow, bool ok, int hh, bf16x8 (&qf)[D / 16]) {
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
    qf[t] = ok ? *reinterpret_cast<const bf16x8*>(qrow + 16 * t + 8 * hh) : bf16x8{};
}

// Keys of a walk: n0 rows at k0 / v0, then n1 rows at k1 / v1 (row strides in bytes).
struct Walk {
  const u16 *k0, *v0, *k1, *v1;
  int n0, n1, row0, row1;
};

// WIDE: more than 32 rows a key head.  Two kernels, as with both forms of the
// prefix walk in one the short cases take 15 % longer.
template <class T, int D, bool WIDE>
__global__ __launch_bounds__(256, 2) void prefix_attn_kernel(Args a) {
  constexpr int NB = D / 32, NT = D / 16;
  constexpr int kImg = kWide * D * 2;  // = two waves' slim tiles
  // The shared tiles of the wide form; of the slim form wave w's K and V halves of piece w.
  __shared__ __attribute__((aligned(1024))) char K0[kImg], V0[kImg], K1[kImg], V1[kImg];
  __shared__ float ml[4][32][2], joined[32][2];  // (max, sum) of each wave's rows; of all four
  __shared__ int4 job;  // found, sequence, its keys, chunk
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lq = lane & 31, hh = lane >> 5;
  const int G = a.G, rows_all = a.B * G, slots = a.p_splits + a.o_splits;
  const bool direct = !WIDE && a.direct;
  const int tiles = WIDE ? (rows_all + 127) / 128 : 1;
  const TileAddr<D> ad(lane);

  const bool final = direct || slots == 1;
  // ---- which work: chunk of the prefix (all row tiles of one chunk on one XCD), or of a sequence's own keys
  const int units = a.p_splits * a.Hkv;
  const int prefix_wgs = (units + 7) / 8 * 8 * tiles;
  int i = blockIdx.x;
  const bool prefix_job = !direct && i < prefix_wgs;
  int slot = 0, kvh = 0, nrows = G, first_row = 0;  // first_row: of the rows b * G + g
  Walk wk{};
  wk.row0 = static_cast<int>(2 * a.p_row);
  wk.row1 = 2 * D;
  if (prefix_job) {
    const int base = tiles == 1 ? i / 8 : i / (8 * tiles), rem = i - base * 8 * tiles;
    const int unit = base * 8 + rem % 8;
    if (unit >= units) return;
    slot = a.by_hkv(unit);
    kvh = unit - slot * a.Hkv;
    first_row = rem / 8 * 128;
    nrows = min(rows_all - first_row, WIDE ? 128 : 32);
    const int64_t at = kvh * a.p_head + static_cast<int64_t>(slot) * a.p_chunk * a.p_row;
    wk.k0 = a.pk + at;
    wk.v0 = a.pv + at;
    wk.n0 = min(a.p_chunk, a.P - slot * a.p_chunk);
  } else if (!direct) {
    i -= prefix_wgs;
  }

  bf16x8 qf[NT];
  if (WIDE && prefix_job) {
    State<T, D> st;
    // 128 rows, 32 per wave, on tiles of 64 keys that the waves share.
    const int r = first_row + 32 * w + lq, rb = a.by_g(r);
    const bool ok = 32 * w + lq < nrows;
    const int64_t qi = static_cast<int64_t>(rb) * a.Hq + kvh * G + (r - rb * G);
    load_q<T, D>(a.q + qi * D, ok, hh, qf);
    const bool mine = 32 * w < nrows;
    const TileDma<D, kWide> dma(w, lane);
    const int nt = (wk.n0 + kWide - 1) / kWide;
    auto load = [&](char* Kd, char* Vd, int t) {
      const int rows = min(kWide, wk.n0 - t * kWide);
      const int64_t at = static_cast<int64_t>(t) * kWide * a.p_row;
      dma.load(row_buffer(wk.k0 + at, rows, wk.row0), wk.row0, Kd);
      dma.load(row_buffer(wk.v0 + at, rows, wk.row0), wk.row0, Vd);
    };
    auto tile = [&](const char* Kc, const char* Vc, char* Kn, char* Vn, int t) {
      if (t + 1 < nt) load(Kn, Vn, t + 1);
      if (mine) {
        f32x16 s[2];
        s[0] = s[1] = f32x16{};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int u = 0; u < NT; ++u) s[h] = mfma32<T>(ad.rows(Kc, 32 * h, u), qf[u], s[h]);
        u32x4 pb[4];
        st.template soften<2>(s, wk.n0 - t * kWide, a.c, hh, pb);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int db = 0; db < NB; ++db) st.o[db] = mfma32<T>(ad.cols(Vc, 16 * u, db), as_op(pb[u]), st.o[db]);
      }
      dma_join();
    };
    load(K0, V0, 0);
#pragma unroll
    for (int t = 0; t < NT; ++t) asm volatile("" ::"v"(qf[t]));
    dma_join();
    for (int t = 0; t < nt; t += 2) {
      tile(K0, V0, K1, V1, t);
      if (t + 1 < nt) tile(K1, V1, K0, V0, t + 1);
    }
    const float lt = half_add(st.l);
    if (final) {
      store_row<T, NB>(a.out + qi * D, st.o, lt == 0.f ? 0.f : 1.f / lt, hh, ok);
    } else if (ok) {
      float* po = a.part_o + (qi * slots + slot) * D;
#pragma unroll
      for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = st.o[db][4 * g + j];
          *reinterpret_cast<f32x4*>(po + 32 * db + 8 * g + 4 * hh) = v;
        }
      if (hh == 0) {
        a.part_ml[(qi * slots + slot) * 2] = st.m;
        a.part_ml[(qi * slots + slot) * 2 + 1] = lt;
      }
    }
    return;
  }

  // (Own chunks outside the one-workgroup form are always joined with something:
  // the entry sees to it, so a sequence without keys needs no workgroup here.)
  //
  // At most 32 rows: every wave walks tiles of its own (tile index = wave mod
  // 4) with its own K and V buffer and no barrier: the next K tile is on its
  // way from the S product on, the next V tile from the O product on.
  const TileDma<D, kSlim, 1> dma(0, lane);
  int scan_b = 0, scan_chunks = 0;  // (wave 0) sequences counted so far, chunks that they hold
  for (;; i += a.o_wgs) {
    State<T, D> st;
    if (WIDE || !prefix_job) {
      // The i-th (chunk of a sequence's own keys, key head): the chunks that hold
      // keys, counted from lens, 64 sequences at a time.
      int b, len, start = 0;
      if (direct) {
        b = a.by_hkv(i);
        kvh = i - b * a.Hkv;
        len = min(max(a.lens[b], 0), a.Smax);
      } else {
        const int unit = a.by_hkv(i);
        kvh = i - unit * a.Hkv;
        if (w == 0) {  // one wave decides for all four, whatever happens to lens meanwhile
          int left = unit - scan_chunks, b0 = scan_b, found = 0;
          for (; b0 < a.B; b0 += 64) {
            const int n = b0 + lane < a.B ? min(max(a.lens[b0 + lane], 0), a.Smax) : 0;
            const int chunks = (n + a.o_chunk - 1) / a.o_chunk;
            int upto = chunks;
#pragma unroll
            for (int off = 1; off < kWave; off <<= 1) {
              const int y = __shfl_up(upto, off, kWave);
              if (lane >= off) upto += y;
            }
            const unsigned long long past = __ballot(upto > left);
            if (past != 0) {
              const int f = __builtin_ctzll(past);
              const int first = left - __shfl(upto - chunks, f, kWave), own = __shfl(n, f, kWave);
              if (lane == 0) job = make_int4(1, b0 + f, own, first);
              scan_b = b0;  // the next chunk of this workgroup lies behind this one
              scan_chunks = unit - left;
              found = 1;
              break;
            }
            left -= __shfl(upto, 63, kWave);
          }
          if (!found && lane == 0) job = make_int4(0, 0, 0, 0);
        }
        __syncthreads();
        const int4 j = job;
        if (j.x == 0) return;  // every chunk is taken
        b = j.y;
        len = j.z;
        slot = __builtin_amdgcn_readfirstlane(a.p_splits + j.w);
        start = j.w * a.o_chunk;
      }
      b = __builtin_amdgcn_readfirstlane(b);
      start = __builtin_amdgcn_readfirstlane(start);
      first_row = b * G;
      wk.n1 = __builtin_amdgcn_readfirstlane(direct ? len : min(a.o_chunk, len - start));
      const int64_t at = ((static_cast<int64_t>(b) * a.Hkv + kvh) * a.Smax + start) * D;
      wk.k1 = a.kc + at;
      wk.v1 = a.vc + at;
      if (direct) {
        wk.k0 = a.pk + kvh * a.p_head;
        wk.v0 = a.pv + kvh * a.p_head;
        wk.n0 = a.P;
      }
    }
    {
      const int r = first_row + lq, rb = a.by_g(r);
      const int64_t qi = static_cast<int64_t>(rb) * a.Hq + kvh * G + (r - rb * G);
      load_q<T, D>(a.q + qi * D, lq < nrows, hh, qf);
    }
    const int t0 = WIDE ? 0 : (wk.n0 + kSlim - 1) / kSlim, nt = t0 + (wk.n1 + kSlim - 1) / kSlim;
    auto load = [&](bool keys, char* dst, int t) {
      const bool own = WIDE || t >= t0;
      const int at = (own ? t - t0 : t) * kSlim, rows = min(kSlim, (own ? wk.n1 : wk.n0) - at);
      const int row = own ? wk.row1 : wk.row0;
      const u16* base = own ? (keys ? wk.k1 : wk.v1) : (keys ? wk.k0 : wk.v0);
      dma.load(row_buffer(base + static_cast<int64_t>(at) * (row / 2), rows, row), row, dst);
    };
    constexpr int kDma = TileDma<D, kSlim, 1>::kN;
    char* const piece_w = w == 0 ? K0 : w == 1 ? V0 : w == 2 ? K1 : V1;
    char* const Kb = piece_w;
    char* const Vb = Kb + kImg / 2;
    if (w < nt) {
      load(true, Kb, w);
      load(false, Vb, w);
#pragma unroll
      for (int t = 0; t < NT; ++t) asm volatile("" ::"v"(qf[t]));  // Q has landed before the loop (see packed_attn.hip)
      for (int t = w; t < nt; t += 4) {
        const bool more = t + 4 < nt;
        f32x16 s[1];
        s[0] = f32x16{};
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kDma) : "memory");  // K has landed, V may be on its way
#pragma unroll
        for (int u = 0; u < NT; ++u) s[0] = mfma32<T>(ad.rows(Kb, 0, u), qf[u], s[0]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read: its buffer is free
        if (more) load(true, Kb, t + 4);
        u32x4 pb[2];
        st.template soften<1>(s, WIDE || t >= t0 ? wk.n1 - (t - t0) * kSlim : wk.n0 - t * kSlim, a.c, hh, pb);
        // V has landed, the next K may be on its way
        if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kDma) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int db = 0; db < NB; ++db) st.o[db] = mfma32<T>(ad.cols(Vb, 16 * u, db), as_op(pb[u]), st.o[db]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) load(false, Vb, t + 4);
      }
    }

    // Join the four waves through LDS: a common max, then the scaled outputs.
    const float lw = half_add(st.l);
    if (hh == 0) {
      ml[w][lq][0] = st.m;
      ml[w][lq][1] = lw;
    }
    __syncthreads();  // also: every wave is done with the tile buffers
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) M = fmaxf(M, ml[v][lq][0]);
    const float M_use = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int v = 0; v < 4; ++v) L += ml[v][lq][1] * exp2_fast(ml[v][lq][0] - M_use);
    {
      // Row lq of this wave's [32][D] fp32 region, its 16-byte pieces XOR-swizzled
      // by the row (rows are a multiple of all banks apart).
      constexpr int kPieces = D / 4;
      char* reg = piece_w;
      const float mul = exp2_fast(st.m - M_use);
      if (lq < nrows) {
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = st.o[db][4 * g + j] * mul;
            const int piece = 8 * db + 2 * g + hh;
            *reinterpret_cast<f32x4*>(reg + lq * D * 4 + 16 * (piece ^ (lq & (kPieces - 1)))) = v;
          }
        if (w == 0 && hh == 0) {
          joined[lq][0] = M;
          joined[lq][1] = L;
        }
      }
      __syncthreads();
      for (int e = threadIdx.x; e < nrows * kPieces; e += 256) {
        const int row = e / kPieces, piece = e - row * kPieces;
        const int off = row * D * 4 + 16 * (piece ^ (row & (kPieces - 1)));
        const f32x4 v = (*reinterpret_cast<const f32x4*>(K0 + off) + *reinterpret_cast<const f32x4*>(V0 + off)) +
                        (*reinterpret_cast<const f32x4*>(K1 + off) + *reinterpret_cast<const f32x4*>(V1 + off));
        const int rr = first_row + row, rb = a.by_g(rr);
        const int64_t qi = static_cast<int64_t>(rb) * a.Hq + kvh * G + (rr - rb * G);
        const float Lr = joined[row][1];
        if (final) {
          const float inv = Lr == 0.f ? 0.f : 1.f / Lr;
          u16x4 y;
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = T::down(v[j] * inv);
          *reinterpret_cast<u16x4*>(a.out + qi * D + 4 * piece) = y;
        } else {
          *reinterpret_cast<f32x4*>(a.part_o + (qi * slots + slot) * D + 4 * piece) = v;
          if (piece == 0) {
            a.part_ml[(qi * slots + slot) * 2] = joined[row][0];
            a.part_ml[(qi * slots + slot) * 2 + 1] = Lr;
          }
        }
      }
    }
    if (!WIDE && (prefix_job || direct)) return;
    __syncthreads();  // the tile buffers are read before the next chunk fills them
  }
}

// Join the slots of one (b, h): the prefix's, then those of the own chunks that
// hold keys.  W waves share a row; wave w of them takes every W-th slot, lane i
// of it the (max, sum) of the i-th of those.  Few rows have many slots and want
// 4 waves each (1 row x 32 heads, 66 slots: 21.2 -> 16.5 us with the launch
// before it), many rows one (32 x 32 heads, 12 slots: 12.2 -> 10.7 us), unless
// 32 slots give each of 4 waves its 8 loads at once (60 x 8 heads, 34 slots:
// 25.9 -> 24.3 us).  The first loads of a wave are issued before anything is known of n: what lies
// past it is the workspace's own memory, and is dropped by selection.
template <class T, int D, int W>
__global__ __launch_bounds__(256) void prefix_join_kernel(Args a) {
  constexpr int E = D / 64;  // outputs per lane
  const int lane = threadIdx.x & 63, w = (threadIdx.x >> 6) % W;
  const int row = blockIdx.x * (4 / W) + (threadIdx.x >> 6) / W;
  if (row >= a.B * a.Hq) return;  // W = 4: never
  const int slots = a.p_splits + a.o_splits;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + static_cast<int64_t>(row) * slots;
  const float* po = a.part_o + static_cast<int64_t>(row) * slots * D + E * lane;
  const int len = min(max(a.lens[row / a.Hq], 0), a.Smax);
  const int n = a.p_splits + (a.o_splits > 0 ? (len + a.o_chunk - 1) / a.o_chunk : 0);
  float M = -INFINITY, L = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s0 = w; s0 < slots; s0 += 64 * W) {  // up to 64 slots of this wave
    const int mine = s0 + W * lane;
    const float2 x = mine < slots ? ml[mine] : float2{-INFINITY, 0.f};
    const bool used = mine < n;
    const float M2 = fmaxf(M, wave_max(used ? x.x : -INFINITY));
    const float M_use = M2 == -INFINITY ? 0.f : M2;
    const float f = used ? exp2_fast(x.x - M_use) : 0.f, keep = exp2_fast(M - M_use);
    L = L * keep + wave_sum(used ? f * x.y : 0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= keep;
    M = M2;
    const int some = min(64, (slots - s0 + W - 1) / W);
    for (int j0 = 0; j0 < some; j0 += 8) {
      float v[8][E];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) v[j][e] = po[static_cast<int64_t>(s0 + W * min(j0 + j, some - 1)) * D + e];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float fj = __shfl(f, min(j0 + j, 63), kWave);
        const bool use = j0 + j < some && s0 + W * (j0 + j) < n;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += use ? fj * v[j][e] : 0.f;
      }
    }
  }
  if constexpr (W == 1) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < E; ++e) a.out[static_cast<int64_t>(row) * D + E * lane + e] = T::down(o[e] * inv);
    return;
  }
  __shared__ float wave_ml[4][2], wave_o[4][D];
  if (lane == 0) {
    wave_ml[w][0] = M;
    wave_ml[w][1] = L;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) wave_o[w][E * lane + e] = o[e];
  __syncthreads();
  if (threadIdx.x >= D) return;
  float M4 = -INFINITY, L4 = 0.f, y = 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) M4 = fmaxf(M4, wave_ml[v][0]);
  if (M4 == -INFINITY) M4 = 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float f = exp2_fast(wave_ml[v][0] - M4);
    L4 += f * wave_ml[v][1];
    y += f * wave_o[v][threadIdx.x];
  }
  a.out[static_cast<int64_t>(row) * D + threadIdx.x] = T::down(L4 == 0.f ? 0.f : y / L4);
}

// Chunks, for 256 CUs that hold two workgroups each.
//
// Prefix: 256 workgroups in all where its length allows (one per CU; the other
// half of each CU walks own keys meanwhile).  Every chunk leaves a state of
// (D + 2) floats per row to write and to join: 512 chunks-times-tiles instead
// of 256 read 53.9 -> 61.1 us at 64 rows x 32,768 keys (32 / 8 heads x 128) and
// 25.8 -> 33.9 us at 60 x 20,000 (8 / 8 heads); 128 leave half the chip idle
// (83 us).  A chunk has at least 256 keys (128: 10.5 -> 11.2 us at 32 x 2,048,
// 32 / 8 heads x 64), 384 for a wave's own tiles (1 x 8,192, 32 / 8 heads x
// 128: 11.4 us against 12.7 with 256 and 15.8 with 128).
//
// Own keys: chunks of 256 that 512 workgroups share out among them by counting
// (a workgroup for every possible chunk, most of them empty, cost 8 us more at
// 64 rows of 2,048).  A workgroup counts on from its last chunk; from the first
// sequence each time, 1,024 rows took 194 us instead of 123.
//
// One workgroup per (sequence, key head), no join: while prefix and cache hold
// at most 1,024 keys and the workgroups fit the chip at once (48 rows, 16 / 2
// heads x 128, 500 + 300 keys: 9.9 against 13.2 us; at 4 rows of 1,000 + 500
// the split form is the faster, 8.9 against 10.6), else 512 keys.
struct Plan {
  int direct, p_chunk, p_splits, o_chunk, o_splits, o_wgs;
};

Plan make_plan(int B, int Hq, int Hkv, int P, int Smax) {
  Plan p{};
  const int rows = B * (Hq / Hkv), tiles = rows > 32 ? (rows + 127) / 128 : 1;
  p.direct = P + Smax <= (B * Hkv <= 512 ? 1024 : 512);
  if (p.direct) return p;
  if (P > 0) {
    const int64_t want = std::max(1, 256 / (Hkv * tiles));
    p.p_chunk = static_cast<int>(std::max<int64_t>(rows > 32 ? 256 : 384, ((P + want - 1) / want + 63) / 64 * 64));
    p.p_splits = (P + p.p_chunk - 1) / p.p_chunk;
  }
  p.o_chunk = 256;
  p.o_splits = (Smax + p.o_chunk - 1) / p.o_chunk;
  p.o_wgs = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(B) * Hkv * p.o_splits, 512));
  return p;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class T, int D>
int launch(Args a, hipStream_t s) {
  const int G = a.Hq / a.Hkv, rows = a.B * G, tiles = !a.direct && rows > 32 ? (rows + 127) / 128 : 1;
  const int64_t grid = a.direct ? static_cast<int64_t>(a.B) * a.Hkv
                                : static_cast<int64_t>((a.p_splits * a.Hkv + 7) / 8 * 8) * tiles + a.o_wgs;
  if (grid <= 0 || grid > 0x7fffffff) return -1;
  if (!a.direct && rows > 32)
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, true>), dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, false>), dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, a);
  int rc = KGWE_CHECK_LAUNCH();
  if (rc || a.direct || a.p_splits + a.o_splits == 1) return rc;
  const int n = a.B * a.Hq;
  if (n <= 256 || (n <= 1024 && a.p_splits + a.o_splits >= 32))
    hipLaunchKernelGGL((prefix_join_kernel<T, D, 4>), dim3(n), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((prefix_join_kernel<T, D, 1>), dim3((n + 3) / 4), dim3(256), 0, s, a);
  return KGWE_CHECK_LAUNCH();
}

// (The last term: numbers that the kernel divides by the head count, see Div.)
inline bool shape_ok(int B, int Hq, int Hkv, int D, int P, int Smax) {
  return B > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 32 && (D == 64 || D == 128) && P >= 0 &&
         Smax >= 0 && P + static_cast<int64_t>(Smax) > 0 && P < (1 << 30) && Smax < (1 << 30) &&
         static_cast<int64_t>(B) * Hq < (1 << 24) && Hkv <= 1024 &&
         (static_cast<int64_t>(B) * (Smax / 256 + 1) * Hkv + 512) * Hkv < (1LL << 32);
}

}  // namespace

// fp32 words of workspace that a call needs (0: none), -1: unsupported shape.
KGWE_API int64_t kgwe_prefix_attn_workspace(int B, int Hq, int Hkv, int D, int P, int Smax) {
  if (!shape_ok(B, Hq, Hkv, D, P, Smax)) return -1;
  const Plan p = make_plan(B, Hq, Hkv, P, Smax);
  const int slots = p.p_splits + p.o_splits;
  return p.direct || slots == 1 ? 0 : static_cast<int64_t>(B) * Hq * slots * (D + 2);
}

// One record per call (see packed_attn.hip).  q, out contiguous [B, Hq, D];
// prefix [Hkv, P, D] by strides (elements, both tensors alike); caches
// contiguous [B, Hkv, Smax, D]; lens int32 [B], cut to [0, Smax].  The
// workspace needs no clearing and is the call's own.
struct PrefixCall {
  const void *q, *pk, *pv, *kc, *vc;
  const int* lens;
  float* work;
  void* out;
  int64_t p_row, p_head;
  int B, Hq, Hkv, D, P, Smax, dtype;
  float scale;
};

KGWE_API int kgwe_prefix_attn_bytes() { return sizeof(PrefixCall); }

KGWE_API int kgwe_prefix_attn(const PrefixCall* c, hipStream_t s) {
  const int B = c->B, Hq = c->Hq, Hkv = c->Hkv, D = c->D, P = c->P, Smax = c->Smax;
  if (!shape_ok(B, Hq, Hkv, D, P, Smax) || (c->dtype != kTypeBf16 && c->dtype != kTypeFp16)) return -1;
  if (P > 0 && (!c->pk || !c->pv || !aligned16(c->pk) || !aligned16(c->pv) || c->p_row % 8 || c->p_head % 8 ||
                c->p_row < D || c->p_row > (1 << 22) || c->p_head < 0))
    return -1;
  if (!aligned16(c->q) || !aligned16(c->out) || !aligned16(c->kc) || !aligned16(c->vc) || !aligned16(c->work))
    return -1;
  const Plan p = make_plan(B, Hq, Hkv, P, Smax);
  const int slots = p.p_splits + p.o_splits;
  if (!p.direct && p.o_splits > 0 && slots < 2) return -1;  // a sequence without keys would stay unwritten
  if (!p.direct && slots > 1 && !c->work) return -2;
  float* ml = c->work + static_cast<int64_t>(B) * Hq * slots * D;
  const Args a{static_cast<const u16*>(c->q), static_cast<const u16*>(c->pk), static_cast<const u16*>(c->pv),
               c->p_row, c->p_head, static_cast<const u16*>(c->kc), static_cast<const u16*>(c->vc), c->lens,
               static_cast<u16*>(c->out), c->work, ml, B, Hq, Hkv, Hq / Hkv, P, Smax, Div(Hq / Hkv), Div(Hkv),
               p.p_chunk, p.p_splits, p.o_chunk,
               p.o_splits, p.o_wgs, p.direct, c->scale * kLog2e};
  if (c->dtype == kTypeBf16) return D == 64 ? launch<Bf16, 64>(a, s) : launch<Bf16, 128>(a, s);
  return D == 64 ? launch<Fp16, 64>(a, s) : launch<Fp16, 128>(a, s);
}
