// The 4-bit microscaled operand (OCP MXFP4: e2m1 elements, one e8m0 scale per 32 of them along
// the contracted axis) as the kernels keep it: in the order in which the block-scaled MFMA
// (v_mfma_scale_f32_16x16x128_f8f6f4) takes it.
//
// A unit is 16 rows x 256 of the contracted axis:
//   codes   2048 B: [2 steps of 128][64 lanes][16 B]; lane l of a step holds row l & 15 and the
//           32 elements number l >> 4 of the step's four blocks, two elements a byte, the first
//           in the low half;
//   scales  128 B: [64 lanes][2 steps], the biased exponent of that block (255 = NaN).
// Units lie [contracted / 256][rows / 16].  A wave's operand of one MFMA is 1 KiB in a row - a
// load instruction of 16 B per lane, from memory or from LDS, with no address arithmetic and no
// bank conflict - and the slab of a matrix tile is one contiguous piece, which spreads evenly over
// the cache and memory channels whatever the sizes (with the units of a row side by side instead,
// the pieces of a slab lie a power of two apart for most models' widths).
// Rows and columns are padded to whole units; padding holds code 0 with scale 0.
#pragma once

#include "smr_internal.hpp"

namespace smr {

constexpr int kMxRows = 16;         // rows of a unit
constexpr int kMxSlab = 256;        // extent of a unit along the contracted axis
constexpr int kMxCodeBytes = 2048;  // codes of a unit
constexpr int kMxScaleBytes = 128;  // scales of a unit
constexpr int64_t kMxMaxExtent = (int64_t)1 << 31;
constexpr int64_t kMxMaxGrid = ((int64_t)1 << 24) - 1;  // workgroups of 256 threads in one launch

__host__ __device__ inline int64_t mx_row_units(int64_t rows) { return (rows + kMxRows - 1) / kMxRows; }
__host__ __device__ inline int64_t mx_slabs(int64_t cols) { return (cols + kMxSlab - 1) / kMxSlab; }

// Number of the unit of row unit `row_unit` and slab `slab`.
__host__ __device__ inline int64_t mx_unit(int64_t row_unit, int64_t slab, int64_t row_units) {
  return slab * row_units + row_unit;
}

// Byte offsets inside a unit of block b (0..7) of row r (0..15).
__host__ __device__ inline int mx_code_offset(int b, int r) { return ((b >> 2) * 64 + (b & 3) * 16 + r) * 16; }
__host__ __device__ inline int mx_scale_offset(int b, int r) { return ((b & 3) * 16 + r) * 2 + (b >> 2); }

// ---------------------------------------------------------------- conversion
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// Rows need not start on 16-byte boundaries (odd widths, slices): the same 128-bit instructions,
// at the alignment of an element.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(2)));

// The scale code of a block whose largest |value| has these bits, and the scale as a float.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t top_bits) {
  const uint32_t field = top_bits >> 23;
  return field == 255u ? 255u : (field > 2u ? field - 2u : 0u);
}
__device__ __forceinline__ float mx_scale_value(uint32_t code) {
  return __uint_as_float(code == 0u ? 0x00400000u : (code == 255u ? 0x7FC00000u : code << 23));
}

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Eight consecutive elements of a row as they come: 4 words of bf16 pairs or 8 of fp32.
template <bool BF16>
struct Mx8 {
  static constexpr int kSize = BF16 ? 2 : 4;
  uint32_t w[BF16 ? 4 : 8];

  template <bool STREAM>
  static __device__ __forceinline__ u32x4 get(const uint8_t* p) {
    const u32x4_any* q = reinterpret_cast<const u32x4_any*>(p);
    if constexpr (STREAM) return __builtin_nontemporal_load(q);
    else return *q;
  }
  // (STREAM: past the caches, for what is read once)
  template <bool STREAM = false>
  __device__ __forceinline__ void load(const uint8_t* p) {
    const u32x4 v = get<STREAM>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = v[k];
    if constexpr (!BF16) {
      const u32x4 u = get<STREAM>(p + 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[4 + k] = u[k];
    }
  }
  // the first `valid` of them (may be negative), zeros behind
  __device__ __forceinline__ void load(const uint8_t* p, int64_t valid) {
#pragma unroll
    for (int k = 0; k < (BF16 ? 4 : 8); ++k) w[k] = 0;
    if (valid >= 8) {
      load(p);
    } else if (valid > 0) {
#pragma unroll
      for (int k = 0; k < 7; ++k)
        if (k < valid) {
          if constexpr (BF16) w[k >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[k] << (16 * (k & 1));
          else w[k] = reinterpret_cast<const uint32_t*>(p)[k];
        }
    }
  }
};
// The largest magnitude of N of them, as the bits of an fp32 value: magnitudes order like the
// integers their bits are, infinities and NaN on top.
template <bool BF16, int N>
__device__ __forceinline__ uint32_t mx_top(const Mx8<BF16> (&v)[N]) {
  if constexpr (BF16) {
    u16x2 top = {0, 0};
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[n].w[k] & 0x7FFF7FFFu));
    return (uint32_t)(top.x > top.y ? top.x : top.y) << 16;
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max_u32(top, v[n].w[k] & 0x7FFFFFFFu);
    return top;
  }
}
// Their codes.
template <bool BF16>
__device__ __forceinline__ uint32_t mx_pack8(const Mx8<BF16>& v, float scale) {
  uint32_t w = 0;
  if constexpr (BF16) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, v.w[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, v.w[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, v.w[2]), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, v.w[3]), scale, 3);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __uint_as_float(v.w[0]), __uint_as_float(v.w[1]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __uint_as_float(v.w[2]), __uint_as_float(v.w[3]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __uint_as_float(v.w[4]), __uint_as_float(v.w[5]), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __uint_as_float(v.w[6]), __uint_as_float(v.w[7]), scale, 3);
  }
  return w;
}

}  // namespace smr
