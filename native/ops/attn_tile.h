// Building blocks of the attention kernels on packed and prefix-sharing
// batches: 32x32x16 matrix instructions on both 16-bit types, the LDS image
// that tiles of 16-bit rows are staged in, and the LDS-DMA that fills it.
//
// Image of a tile of rows of D elements: subtiles of 8 rows x 32 columns, 512
// bytes each, the four 16-byte chunks of a subtile row XOR-swizzled by the
// row.  Row reads (ds_read_b128) and hardware-transposed reads
// (ds_read_b64_tr_b16) of one matrix operand then touch every bank once, and
// all of an operand's reads differ from two base addresses by immediates.
//
// A wave's LDS-DMA instruction writes 1024 consecutive bytes of the image
// (two subtiles), so the swizzle is applied to the source address.  The loads
// go through a buffer descriptor whose extent ends with the tile's last valid
// row: rows past it arrive as zeros, whatever memory holds there.
#pragma once
#include <type_traits>

#include "half_types.h"

namespace kgwe {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) unsigned short u16x4;

template <class T>
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mfma32<Bf16>(bf16x8 a, bf16x8 b, f32x16 c) {
  typedef __attribute__((ext_vector_type(8))) __bf16 op;
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(op, a), __builtin_bit_cast(op, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mfma32<Fp16>(bf16x8 a, bf16x8 b, f32x16 c) {
  typedef __attribute__((ext_vector_type(8))) _Float16 op;
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(op, a), __builtin_bit_cast(op, b), c, 0, 0, 0);
}

// Two floats to a packed pair, to nearest even.
template <class T>
__device__ __forceinline__ unsigned pack2(float lo, float hi);
template <>
__device__ __forceinline__ unsigned pack2<Bf16>(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) float f2;
  typedef __attribute__((ext_vector_type(2))) __bf16 b2;
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){lo, hi}, b2));
}
template <>
__device__ __forceinline__ unsigned pack2<Fp16>(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) float f2;
  typedef __attribute__((ext_vector_type(2))) _Float16 h2;
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){lo, hi}, h2));
}

__device__ __forceinline__ bf16x8 as_op(const u32x4& w) { return __builtin_bit_cast(bf16x8, w); }

// 2^x as one v_exp_f32: arguments here are far below 128, and a result below
// 2^-126 is zero to any 16-bit output.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Running maximum (log2 units) kept until a tile's largest score passes it by
// this much, so outputs are rescaled on few tiles.
constexpr float kDefer = 4.f;

// The reference that exponents are taken against, after a tile whose largest
// score is `top`: the running maximum, in fp16 less 11, which multiplies all
// probabilities and their sum by 2^11 before they are rounded to T.  fp16 has
// steps of 2^-24 below 2^-14, and what many keys far from the maximum add up to
// would be lost (65,536 keys at 2^-26 of it: all).  With kDefer that is 2^15 at
// most, and fp16 ends at 65,504.  Scores past 2^20 are not lifted: the rounding
// of top * c, which the exponents do not share, needs the room there.
template <class T>
__device__ __forceinline__ float next_max(float top, float c, float m) {
  const float x = top * c;
  float lift = 0.f;
  if constexpr (std::is_same<T, Fp16>::value) lift = fabsf(x) < 0x1p20f ? 11.f : 0.f;
  return x > m + (kDefer + lift) ? x - lift : m;
}

// Row of a 32x32 accumulator tile that register r of this lane half holds.
__device__ __forceinline__ int tile_row(int r, int half) { return (r & 3) + 8 * (r >> 2) + 4 * half; }

// Combine lane l with lane l ^ 32 (a VALU half exchange).
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_add(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Lane-dependent parts of an image's read addresses (bytes).
template <int D>
struct TileAddr {
  static constexpr int kGroup = 16 * D;  // bytes of 8 rows
  int row[2], tr[2];
  __device__ __forceinline__ explicit TileAddr(int lane) {
    const int lk = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int p = 0; p < 2; ++p) row[p] = kGroup * (lk >> 3) + 64 * (lk & 7) + 16 * ((2 * p + hh) ^ ((lk >> 2) & 3));
    const int g = lane >> 4, q = (lane >> 2) & 3, pp = lane & 3;
    const int r = 4 * (g >> 1) + q, ch = 2 * (g & 1) + (pp >> 1), byte = 8 * (pp & 1);
    tr[0] = 64 * r + 16 * (ch ^ ((r >> 2) & 3)) + byte;
    tr[1] = kGroup + 64 * r + 16 * (ch ^ (((8 + r) >> 2) & 3)) + byte;
  }
  // Lane (lk, hh): elements 16 t + 8 hh .. + 7 of row r0 + lk; r0 % 8 == 0.
  __device__ __forceinline__ bf16x8 rows(const char* img, int r0, int t) const {
    return *reinterpret_cast<const bf16x8*>(img + row[t & 1] + 512 * (t >> 1) + (kGroup / 8) * r0);
  }
  // Lane (c, hh): column 32 db + c of rows base + {0..3, 8..11} + 4 hh, the
  // order in which an accumulator tile holds its rows; base % 16 == 0.
  __device__ __forceinline__ bf16x8 cols(const char* img, int base, int db) const {
    typedef __attribute__((ext_vector_type(4))) short s4;
    const int o = (kGroup / 8) * base + 512 * db;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(img + tr[0] + o));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(img + tr[1] + o));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// Descriptor of `rows` rows of a strided view (row stride in bytes), for loads
// that return zeros past the last row.
// (The host pass has neither the type nor the builtins, and drops the launch
// stubs of templates that name them, so it sees empty stand-ins.)
#ifdef __HIP_DEVICE_COMPILE__
typedef __amdgpu_buffer_rsrc_t buf_t;
#else
struct buf_t {};
#endif
__device__ __forceinline__ buf_t row_buffer(const void* p, int rows, int row_bytes) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, rows * row_bytes, 0x00020000);
#else
  return buf_t{};
#endif
}

// BYTES (4 or 16) per lane from src + offset to consecutive LDS from dst on
// (wave-uniform); zeros where the offset is past the descriptor's extent.  (The
// instruction's immediate offset would move the LDS address along.)
template <int BYTES>
__device__ __forceinline__ void dma_lane(buf_t src, int offset, void* dst) {
#ifdef __HIP_DEVICE_COMPILE__
  auto d = (__attribute__((address_space(3))) void*)dst;
  static_assert(BYTES == 4 || BYTES == 16, "4 or 16 bytes per lane");
  if constexpr (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(src, d, 16, offset, 0, 0, 0);
  else __builtin_amdgcn_raw_ptr_buffer_load_lds(src, d, 4, offset, 0, 0, 0);
#endif
}

// One wave's share (of W) of a tile of ROWS rows: kN instructions, each of 1024
// bytes of the image = 8 rows x 64 columns, 8 rows further on every one (D =
// 64) or two (D = 128).  The swizzle of a chunk depends on the parity of its
// row group alone, so two lane offsets serve all of them.
template <int D, int ROWS, int W = 4>
struct TileDma {
  static constexpr int kBytes = ROWS * D * 2;
  static constexpr int kN = kBytes / 1024 / W;
  static constexpr int kPer = D / 64;  // instructions per row group
  static_assert(kN >= kPer && kN % kPer == 0 && kBytes % (1024 * W) == 0, "whole row groups per wave");
  int row, chunk[2];
  int first;  // wave-uniform byte offset of the wave's share
  __device__ __forceinline__ TileDma(int wave, int lane) : first(wave * kN * 1024) {
    const int group = wave * (kN / kPer), r7 = (lane >> 2) & 7;
    row = 8 * group + r7;
#pragma unroll
    for (int p = 0; p < 2; ++p)
      chunk[p] = 64 * (lane >> 5) + 16 * ((lane & 3) ^ ((2 * (group + p) + (r7 >> 2)) & 3));
  }
  __device__ __forceinline__ void load(buf_t src, int row_bytes, char* img) const {
    const int at = row * row_bytes;
#pragma unroll
    for (int g = 0; g < kN / kPer; ++g) {
      const int off = at + 8 * g * row_bytes + chunk[g & 1];
      dma_lane<16>(src, off, img + first + 1024 * kPer * g);
      if constexpr (kPer == 2) dma_lane<16>(src, off + 128, img + first + 1024 * kPer * g + 1024);
    }
  }
};

// Every LDS-DMA of this wave has landed; then everyone's.
__device__ __forceinline__ void dma_join() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Division by a host-known divisor: n / d for n * d < 2^32 by one multiply
// (an integer division is some 20 instructions, which count in short kernels).
struct Div {
  unsigned mul;  // ceil(2^32 / d); 0 for d = 1
  __host__ explicit Div(int d = 1) : mul(d == 1 ? 0u : static_cast<unsigned>(0xffffffffu / d + 1)) {}
  __device__ __forceinline__ int operator()(int n) const {
    return mul == 0 ? n : static_cast<int>(__umulhi(static_cast<unsigned>(n), mul));
  }
};

// Store one row of transposed accumulators (acc[db] register r holds column
// 32 db + tile_row(r, hh) of this lane's row) times `mul` with 16-byte stores:
// a lane holds 4 consecutive columns per register group, its partner lane the
// next 4, and a half exchange per dword pairs them.  All lanes take part; `ok`
// guards the stores.
template <class T, int NB>
__device__ __forceinline__ void store_row(unsigned short* row, const f32x16 (&acc)[NB], float mul, int hh, bool ok) {
#pragma unroll
  for (int db = 0; db < NB; ++db)
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
      const f32x16& a = acc[db];
      const int g0 = 8 * pr, g1 = 8 * pr + 4;
      const auto r0 = __builtin_amdgcn_permlane32_swap(pack2<T>(a[g0] * mul, a[g0 + 1] * mul),
                                                       pack2<T>(a[g1] * mul, a[g1 + 1] * mul), false, false);
      const auto r1 = __builtin_amdgcn_permlane32_swap(pack2<T>(a[g0 + 2] * mul, a[g0 + 3] * mul),
                                                       pack2<T>(a[g1 + 2] * mul, a[g1 + 3] * mul), false, false);
      const u32x4 v = {r0[0], r1[0], r0[1], r1[1]};
      if (ok) *reinterpret_cast<u32x4*>(row + db * 32 + 16 * pr + 8 * hh) = v;
    }
}

}  // namespace kgwe
