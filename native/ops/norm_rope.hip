// Norm of every query and key head + position rotation in one pass over the
// fused projection's output, with its gradient, for rows at given positions.
//
// qkv [T, (Hq + 2 Hkv) D] (row stride given) -> q [T, Hq, D], k, v [T, Hkv, D]:
//   n = x * rsqrt(mean(x^2) + eps) * w        per head, w [D] (absent: n = x)
//   y[i]       = n[i] cos[p, i] - n[i + D/2] sin[p, i]         i < D/2
//   y[i + D/2] = n[i + D/2] cos[p, i] + n[i] sin[p, i]
// with p = pos[t] + offset and fp32 tables (no pos: row t is at t % period, a
// rectangular batch).  v is copied.  A row whose p is
// outside the tables (a packed batch marks its padding rows with position -1)
// gives zeros and takes no gradient.  Everything between the load and the
// store is fp32: ONE rounding per output, where norm and rotation as two
// passes round twice.
//
// Optionally the same launch appends k and v to a head-major cache
// [rows, Hkv, Smax, D] at (cache_row[t], pos[t]).
//
// Gradient, with g = the rotation's transpose applied to dy and r = 1 / rms:
//   dx = r (w g - x r^2 mean(w g x)),   dw = sum over rows and heads of g x r.
//
// Both passes are bound by HBM: a thread holds one 8-wide chunk of a head's
// first half and the matching chunk of its second half (the pair that the
// rotation mixes), D / 16 neighbouring lanes hold a head, and the mean is a
// shuffle tree over them.  10,339 rows of 32 / 8 heads x 128 in bf16: forward
// 50 us (254 MB, 5.1 TB/s), gradient 65 us (360 MB, v's x is not needed; 5.5
// TB/s) and 4 us for the sums of dw; a large copy reaches 5.0 TB/s.  Few rows
// are one launch's latency, 3 us.
#include <algorithm>

#include "half_types.h"

using namespace kgwe;

namespace {

constexpr int kThreads = 256;
constexpr int kDwBlocks = 1024;  // partial sums of dw: one [2, D] row per workgroup

// Sum over the L lanes that hold one head.
template <int L>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

__device__ __forceinline__ void load_table(const float* __restrict__ p, float (&out)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    out[j] = a[j];
    out[4 + j] = b[j];
  }
}

template <class T>
__device__ __forceinline__ void up8(bf16x8 v, float (&out)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) out[j] = T::up(v[j]);
}

template <class T>
__device__ __forceinline__ bf16x8 down8(const float (&in)[8]) {
  bf16x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = T::down(in[j]);
  return v;
}

__device__ __forceinline__ bf16x8 ld8(const unsigned short* p) { return *reinterpret_cast<const bf16x8*>(p); }
__device__ __forceinline__ void st8(unsigned short* p, bf16x8 v) { *reinterpret_cast<bf16x8*>(p) = v; }

struct FwdArgs {
  const unsigned short* qkv;
  int64_t row_stride;
  const int* pos;
  const float* cosT;
  const float* sinT;
  const unsigned short* wq;  // null: no norm
  const unsigned short* wk;
  unsigned short* q;
  unsigned short* k;         // null: k and v go to the cache only
  unsigned short* v;
  unsigned short* kc;        // null: no cache
  unsigned short* vc;
  const int* cache_row;      // null: row t
  int T, period, offset, table_rows, Hq, Hkv, Smax, cache_rows;
  float eps;
};

// L = D / 16 lanes per head.
template <class T, int L>
__global__ __launch_bounds__(kThreads) void norm_rope_fwd_kernel(FwdArgs a) {
  constexpr int D = 16 * L, half = D / 2;
  const int Ht = a.Hq + 2 * a.Hkv;
  const int64_t n = static_cast<int64_t>(a.T) * Ht * L;
  // Every lane of a wave runs the same number of rounds (the shuffles need all
  // lanes of a head, and a wave holds whole heads: 64 % L == 0).
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t th = i / L;
    const int c = static_cast<int>(i % L) * 8;
    const int64_t t = th / Ht;
    const int head = static_cast<int>(th - t * Ht);
    const int cp = a.pos != nullptr ? a.pos[t] : static_cast<int>(t % a.period);
    const int64_t p = static_cast<int64_t>(cp) + a.offset;
    const bool live = cp >= 0 && p < a.table_rows;
    const unsigned short* in = a.qkv + t * a.row_stride + static_cast<int64_t>(head) * D + c;
    const bf16x8 lo = live ? ld8(in) : bf16x8{}, hi = live ? ld8(in + half) : bf16x8{};
    const bool is_q = head < a.Hq, is_v = head >= a.Hq + a.Hkv;
    bf16x8 ylo = lo, yhi = hi;
    float x0[8], x1[8];
    up8<T>(lo, x0);
    up8<T>(hi, x1);
    if (a.wq != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += x0[j] * x0[j] + x1[j] * x1[j];
      ss = head_sum<L>(ss);
      const float r = 1.f / sqrtf(ss * (1.f / D) + a.eps);
      const unsigned short* w = is_q ? a.wq : a.wk;
      float w0[8], w1[8];
      up8<T>(ld8(w + c), w0);
      up8<T>(ld8(w + half + c), w1);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x0[j] *= r * w0[j];
        x1[j] *= r * w1[j];
      }
    }
    if (live && !is_v) {
      float cs[8], sn[8], y0[8], y1[8];
      load_table(a.cosT + p * half + c, cs);
      load_table(a.sinT + p * half + c, sn);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y0[j] = x0[j] * cs[j] - x1[j] * sn[j];
        y1[j] = x1[j] * cs[j] + x0[j] * sn[j];
      }
      ylo = down8<T>(y0);
      yhi = down8<T>(y1);
    }
    unsigned short* out = nullptr;
    if (is_q) out = a.q + (t * a.Hq + head) * D;
    else if (a.k != nullptr) out = (is_v ? a.v : a.k) + (t * a.Hkv + (head - a.Hq - (is_v ? a.Hkv : 0))) * D;
    if (out != nullptr) {
      st8(out + c, ylo);
      st8(out + half + c, yhi);
    }
    if (a.kc != nullptr && !is_q && live && cp < a.Smax) {
      const int row = a.cache_row != nullptr ? a.cache_row[t] : static_cast<int>(t);
      if (row >= 0 && row < a.cache_rows) {  // never write outside the cache
        unsigned short* dst = (is_v ? a.vc : a.kc) +
            ((static_cast<int64_t>(row) * a.Hkv + (head - a.Hq - (is_v ? a.Hkv : 0))) * a.Smax + cp) * D;
        st8(dst + c, ylo);
        st8(dst + half + c, yhi);
      }
    }
  }
}

struct BwdArgs {
  const unsigned short* qkv;  // the forward's input (norm only)
  int64_t row_stride;
  const int* pos;
  const float* cosT;
  const float* sinT;
  const unsigned short* wq;
  const unsigned short* wk;
  const unsigned short* dq;
  const unsigned short* dk;
  const unsigned short* dv;
  unsigned short* dqkv;
  float* part;                // [grid, 2, D] sums of dw (norm only)
  int T, period, offset, table_rows, Hq, Hkv;
  float eps;
};

// Sums of a thread's share of dw over the lanes that hold the same chunk, then
// over the four waves, in a fixed order; out [D].
template <int L>
__device__ __forceinline__ void reduce_dw(float (&acc)[16], int c, float (&red)[kThreads / kWave][16 * L], float* out) {
  constexpr int D = 16 * L, half = D / 2;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int off = kWave / 2; off >= L; off >>= 1) acc[j] += __shfl_xor(acc[j], off, kWave);
  if (lane < L) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      red[wave][c + j] = acc[j];
      red[wave][half + c + j] = acc[8 + j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) s += red[w][i];
    out[i] = s;
  }
  __syncthreads();
}

// The query heads of all rows, then the key heads, then the value heads: one
// weight and one set of dw sums live at a time (one sweep over all heads held
// two of each: 136 registers, 3 workgroups per CU, 88 us at 10,339 rows of
// 32 / 8 heads x 128 against 66 us).
template <class T, int L, bool NORM>
__global__ __launch_bounds__(kThreads) void norm_rope_bwd_kernel(BwdArgs a) {
  constexpr int D = 16 * L, half = D / 2;
  __shared__ float red[kThreads / kWave][D];
  const int Ht = a.Hq + 2 * a.Hkv;
  // The strides are multiples of L, so a thread always holds the same chunk of
  // a head and sums its share of dw in registers.
  const int c = static_cast<int>(threadIdx.x % L) * 8;
  const int64_t start = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  auto sweep = [&](const unsigned short* dy, const unsigned short* w, int heads, int first, float (&acc)[16]) {
    float w0[8], w1[8];
    if (NORM) {
      up8<T>(ld8(w + c), w0);
      up8<T>(ld8(w + half + c), w1);
    }
    const int64_t n = static_cast<int64_t>(a.T) * heads * L;
    for (int64_t i = start; i < n; i += step) {
      const int64_t th = i / L, t = th / heads;
      const int head = static_cast<int>(th - t * heads);
      const int cp = a.pos != nullptr ? a.pos[t] : static_cast<int>(t % a.period);
      const int64_t p = static_cast<int64_t>(cp) + a.offset;
      const bool live = cp >= 0 && p < a.table_rows;
      unsigned short* out = a.dqkv + (t * Ht + first + head) * static_cast<int64_t>(D) + c;
      float g0[8] = {}, g1[8] = {};
      if (live) {  // the same for all lanes of a head
        const unsigned short* y = dy + th * D + c;
        float y0[8], y1[8], cs[8], sn[8];
        up8<T>(ld8(y), y0);
        up8<T>(ld8(y + half), y1);
        load_table(a.cosT + p * half + c, cs);
        load_table(a.sinT + p * half + c, sn);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g0[j] = y0[j] * cs[j] + y1[j] * sn[j];
          g1[j] = y1[j] * cs[j] - y0[j] * sn[j];
        }
        if (NORM) {
          const unsigned short* x = a.qkv + t * a.row_stride + static_cast<int64_t>(first + head) * D + c;
          float x0[8], x1[8];
          up8<T>(ld8(x), x0);
          up8<T>(ld8(x + half), x1);
          float ss = 0.f, gx = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            ss += x0[j] * x0[j] + x1[j] * x1[j];
            gx += g0[j] * w0[j] * x0[j] + g1[j] * w1[j] * x1[j];
          }
          ss = head_sum<L>(ss);
          gx = head_sum<L>(gx);
          const float r = 1.f / sqrtf(ss * (1.f / D) + a.eps);
          const float m = gx * (1.f / D) * r * r;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            acc[j] += g0[j] * x0[j] * r;
            acc[8 + j] += g1[j] * x1[j] * r;
            g0[j] = r * (g0[j] * w0[j] - x0[j] * m);
            g1[j] = r * (g1[j] * w1[j] - x1[j] * m);
          }
        }
      }
      st8(out, down8<T>(g0));
      st8(out + half, down8<T>(g1));
    }
  };
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * D;
  {
    float acc[16] = {};
    sweep(a.dq, a.wq, a.Hq, 0, acc);
    if (NORM) reduce_dw<L>(acc, c, red, part);
  }
  {
    float acc[16] = {};
    sweep(a.dk, a.wk, a.Hkv, a.Hq, acc);
    if (NORM) reduce_dw<L>(acc, c, red, part + D);
  }
  const int64_t n = static_cast<int64_t>(a.T) * a.Hkv * L;
  for (int64_t i = start; i < n; i += step) {  // values: a copy
    const int64_t th = i / L, t = th / a.Hkv;
    const int head = static_cast<int>(th - t * a.Hkv);
    const int cp = a.pos != nullptr ? a.pos[t] : static_cast<int>(t % a.period);
    const bool live = cp >= 0 && static_cast<int64_t>(cp) + a.offset < a.table_rows;
    const unsigned short* y = a.dv + th * D + c;
    unsigned short* out = a.dqkv + (t * Ht + a.Hq + a.Hkv + head) * static_cast<int64_t>(D) + c;
    st8(out, live ? ld8(y) : bf16x8{});
    st8(out + half, live ? ld8(y + half) : bf16x8{});
  }
}

// dw[2, D] = sum of the workgroups' partials: 16 columns x 64 row groups per
// workgroup (16 rows each at most, four loads in flight), the groups joined
// through LDS in a fixed order.  With 16 row groups: 20 us.
constexpr int kDwThreads = 1024, kDwGroups = kDwThreads / 16;
template <class T>
__global__ __launch_bounds__(kDwThreads) void norm_rope_dw_kernel(const float* __restrict__ part, int blocks,
                                                                int D, unsigned short* __restrict__ dwq,
                                                                unsigned short* __restrict__ dwk) {
  __shared__ float red[kDwGroups][17];
  const int col = threadIdx.x % 16, grp = threadIdx.x / 16;
  const int i = blockIdx.x * 16 + col;  // 2 * D is a multiple of 16
  float s = 0.f;
#pragma unroll 4
  for (int b = grp; b < blocks; b += kDwGroups) s += part[static_cast<int64_t>(b) * 2 * D + i];
  red[grp][col] = s;
  __syncthreads();
  if (grp == 0) {
    float t = 0.f;
#pragma unroll
    for (int g = 0; g < kDwGroups; ++g) t += red[g][col];
    (i < D ? dwq[i] : dwk[i - D]) = T::down(t);
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline bool shape_ok(int T, int Hq, int Hkv, int D, int dtype, int64_t row_stride) {
  return T > 0 && Hq > 0 && Hkv > 0 && Hq <= 4096 && Hkv <= 4096 && (D == 32 || D == 64 || D == 128 || D == 256) &&
         (dtype == kTypeBf16 || dtype == kTypeFp16) && row_stride % 8 == 0;
}

inline int grid_for(int64_t items, int most) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((items + kThreads - 1) / kThreads, most)));
}

template <class T>
int fwd(const FwdArgs& a, int D, hipStream_t s) {
  const int grid = grid_for(static_cast<int64_t>(a.T) * (a.Hq + 2 * a.Hkv) * (D / 16), 1 << 20);
  switch (D) {
    case 32: hipLaunchKernelGGL((norm_rope_fwd_kernel<T, 2>), dim3(grid), dim3(kThreads), 0, s, a); break;
    case 64: hipLaunchKernelGGL((norm_rope_fwd_kernel<T, 4>), dim3(grid), dim3(kThreads), 0, s, a); break;
    case 128: hipLaunchKernelGGL((norm_rope_fwd_kernel<T, 8>), dim3(grid), dim3(kThreads), 0, s, a); break;
    case 256: hipLaunchKernelGGL((norm_rope_fwd_kernel<T, 16>), dim3(grid), dim3(kThreads), 0, s, a); break;
    default: return -1;
  }
  return KGWE_CHECK_LAUNCH();
}

template <class T, int L>
int bwd_launch(const BwdArgs& a, int grid, hipStream_t s) {
  if (a.wq != nullptr)
    hipLaunchKernelGGL((norm_rope_bwd_kernel<T, L, true>), dim3(grid), dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((norm_rope_bwd_kernel<T, L, false>), dim3(grid), dim3(kThreads), 0, s, a);
  return KGWE_CHECK_LAUNCH();
}

template <class T>
int bwd(const BwdArgs& a, int D, int grid, unsigned short* dwq, unsigned short* dwk, hipStream_t s) {
  int rc = -1;
  switch (D) {
    case 32: rc = bwd_launch<T, 2>(a, grid, s); break;
    case 64: rc = bwd_launch<T, 4>(a, grid, s); break;
    case 128: rc = bwd_launch<T, 8>(a, grid, s); break;
    case 256: rc = bwd_launch<T, 16>(a, grid, s); break;
  }
  if (rc || a.wq == nullptr) return rc;
  hipLaunchKernelGGL((norm_rope_dw_kernel<T>), dim3(2 * D / 16), dim3(kDwThreads), 0, s, a.part, grid, D, dwq, dwk);
  return KGWE_CHECK_LAUNCH();
}

}  // namespace

// One record per call (see packed_attn.hip).  pos null: row t is at t % period.
// wq / wk null: rotation alone.  k / v null: the rotated keys and the values go
// to the cache only (kc, vc then required).  cache_row null: row t of the cache.
struct NormRopeFwdCall {
  const void* qkv;
  const int* pos;
  const float *cos_t, *sin_t;
  const void *wq, *wk;
  void *q, *k, *v, *kc, *vc;
  const int* cache_row;
  int64_t row_stride;
  int T, period, offset, table_rows, Hq, Hkv, D, Smax, cache_rows, dtype;
  float eps;
};

// dq, dk, dv contiguous; dqkv contiguous [T, (Hq + 2 Hkv) D].  With norms also
// qkv, part [blocks, 2, D] fp32 and dwq, dwk [D] (always both).
struct NormRopeBwdCall {
  const void* qkv;
  const int* pos;
  const float *cos_t, *sin_t;
  const void *wq, *wk, *dq, *dk, *dv;
  void* dqkv;
  float* part;
  void *dwq, *dwk;
  int64_t row_stride;
  int T, period, offset, table_rows, Hq, Hkv, D, dtype;
  float eps;
};

KGWE_API int kgwe_norm_rope_fwd_bytes() { return sizeof(NormRopeFwdCall); }
KGWE_API int kgwe_norm_rope_bwd_bytes() { return sizeof(NormRopeBwdCall); }

KGWE_API int kgwe_norm_rope_fwd(const NormRopeFwdCall* c, hipStream_t s) {
  if (!shape_ok(c->T, c->Hq, c->Hkv, c->D, c->dtype, c->row_stride) || c->offset < 0 || c->table_rows <= 0 ||
      (!c->pos && c->period <= 0))
    return -1;
  if (!c->wq != !c->wk || !c->k != !c->v || !c->kc != !c->vc || (!c->k && !c->kc) || !c->q ||
      (c->kc && (c->Smax <= 0 || c->cache_rows <= 0)))
    return -1;
  if (!aligned16(c->qkv) || !aligned16(c->wq) || !aligned16(c->wk) || !aligned16(c->q) || !aligned16(c->k) ||
      !aligned16(c->v) || !aligned16(c->kc) || !aligned16(c->vc) || !aligned16(c->cos_t) || !aligned16(c->sin_t))
    return -1;
  using u16 = unsigned short;
  const FwdArgs a{static_cast<const u16*>(c->qkv), c->row_stride, c->pos, c->cos_t, c->sin_t,
                  static_cast<const u16*>(c->wq), static_cast<const u16*>(c->wk), static_cast<u16*>(c->q),
                  static_cast<u16*>(c->k), static_cast<u16*>(c->v), static_cast<u16*>(c->kc),
                  static_cast<u16*>(c->vc), c->cache_row, c->T, c->period, c->offset, c->table_rows, c->Hq, c->Hkv,
                  c->Smax, c->cache_rows, c->eps};
  return c->dtype == kTypeBf16 ? fwd<Bf16>(a, c->D, s) : fwd<Fp16>(a, c->D, s);
}

// Workgroups of the gradient's launch = rows [2, D] of its fp32 workspace.
KGWE_API int kgwe_norm_rope_bwd_blocks(int T, int Hq, int Hkv, int D) {
  if (T <= 0 || Hq <= 0 || Hkv <= 0 || D < 16) return 0;
  return grid_for(static_cast<int64_t>(T) * (Hq + 2 * Hkv) * (D / 16), kDwBlocks);
}

KGWE_API int kgwe_norm_rope_bwd(const NormRopeBwdCall* c, hipStream_t s) {
  if (!shape_ok(c->T, c->Hq, c->Hkv, c->D, c->dtype, c->row_stride) || c->offset < 0 || c->table_rows <= 0 ||
      (!c->pos && c->period <= 0))
    return -1;
  if (!c->wq != !c->wk || (c->wq && (!c->part || !c->dwq || !c->dwk || !c->qkv))) return -1;
  if (!aligned16(c->qkv) || !aligned16(c->wq) || !aligned16(c->wk) || !aligned16(c->dq) || !aligned16(c->dk) ||
      !aligned16(c->dv) || !aligned16(c->dqkv) || !aligned16(c->cos_t) || !aligned16(c->sin_t))
    return -1;
  using u16 = unsigned short;
  const BwdArgs a{static_cast<const u16*>(c->qkv), c->row_stride, c->pos, c->cos_t, c->sin_t,
                  static_cast<const u16*>(c->wq), static_cast<const u16*>(c->wk), static_cast<const u16*>(c->dq),
                  static_cast<const u16*>(c->dk), static_cast<const u16*>(c->dv), static_cast<u16*>(c->dqkv), c->part,
                  c->T, c->period, c->offset, c->table_rows, c->Hq, c->Hkv, c->eps};
  const int grid = kgwe_norm_rope_bwd_blocks(c->T, c->Hq, c->Hkv, c->D);
  u16 *dwq = static_cast<u16*>(c->dwq), *dwk = static_cast<u16*>(c->dwk);
  return c->dtype == kTypeBf16 ? bwd<Bf16>(a, c->D, grid, dwq, dwk, s) : bwd<Fp16>(a, c->D, grid, dwq, dwk, s);
}
