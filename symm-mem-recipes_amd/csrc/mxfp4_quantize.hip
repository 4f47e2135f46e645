// Quantisation to 4-bit microscaled floats (OCP MXFP4) and back.
//
// A block of 32 values v along the contracted axis becomes a scale 2^e and 32 e2m1 codes:
//   e    = floor(log2(max |v|)) - 2, at least -127 (2 is the exponent of e2m1's largest value, 6),
//   code = v * 2^-e rounded to nearest even on {0, .5, 1, 1.5, 2, 3, 4, 6}, saturated at 6.
// floor(log2) is the exponent field of the largest magnitude, taken as an integer, so infinities
// and NaN come out on top: a block that holds one gets the scale code 255 (NaN) and element codes
// 0, and is NaN as a whole.  A block of zeros gets scale code 0.  The rounding is the hardware's
// (v_cvt_scalef32_pk_fp4_f32: the scale is a power of two, so the division is exact and there is
// one rounding).
#include "mxfp4_layout.hpp"

namespace smr {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// Rows need not start on 16-byte boundaries (odd widths, slices): the same 128-bit instructions,
// at the alignment of an element.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(2)));

constexpr int kQuantThreads = 256;

// The scale code of a block whose largest |value| has these bits, and the scale as a float.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t top_bits) {
  const uint32_t field = top_bits >> 23;
  return field == 255u ? 255u : (field > 2u ? field - 2u : 0u);
}
__device__ __forceinline__ float mx_scale_value(uint32_t code) {
  return __uint_as_float(code == 0u ? 0x00400000u : (code == 255u ? 0x7FC00000u : code << 23));
}
// Eight values to eight codes.
__device__ __forceinline__ uint32_t mx_pack8(const float* v, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// Eight consecutive elements of a row, zeros from `valid` on.
template <bool BF16>
__device__ __forceinline__ void load8(const uint8_t* p, int valid, float (&v)[8]) {
  if constexpr (BF16) {
    if (valid >= 8) {
      const u32x4 w = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = bf16_lo(w[k]);
        v[2 * k + 1] = bf16_hi(w[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = k < valid ? __uint_as_float((uint32_t) reinterpret_cast<const uint16_t*>(p)[k] << 16) : 0.0f;
    }
  } else {
    if (valid >= 8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 w = reinterpret_cast<const u32x4_any*>(p)[h];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * h + k] = __uint_as_float(w[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k < valid ? reinterpret_cast<const float*>(p)[k] : 0.0f;
    }
  }
}

// Along the rows of x.  A wave takes one unit: two rows of 512 B (bf16) at a time, 8 values per
// lane, 4 lanes per block.
template <bool BF16>
__global__ __launch_bounds__(kQuantThreads) void mxfp4_quantize_kernel(const uint8_t* __restrict__ x, int64_t row_bytes,
                                                                      uint8_t* __restrict__ codes,
                                                                      uint8_t* __restrict__ scales, int64_t rows,
                                                                      int64_t cols, int64_t slabs, int64_t units) {
  constexpr int kSize = BF16 ? 2 : 4;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kQuantThreads / 64) + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t row0 = unit / slabs * kMxRows, col0 = unit % slabs * kMxSlab;
  const int col = (lane & 31) * 8, b = (lane & 31) >> 2, q = lane & 3;
  const int64_t left = cols - col0 - col;
  const int valid = left < 0 ? 0 : (left > 8 ? 8 : (int)left);
  uint8_t* unit_codes = codes + unit * kMxCodeBytes;
  uint8_t* unit_scales = scales + unit * kMxScaleBytes;
#pragma unroll
  for (int i = 0; i < kMxRows / 2; ++i) {
    const int r = i * 2 + (lane >> 5);
    const int64_t row = row0 + r;
    float v[8];
    load8<BF16>(x + row * row_bytes + (col0 + col) * kSize, row < rows ? valid : 0, v);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max_u32(top, abs_bits(v[k]));
    top = max_u32(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max_u32(top, (uint32_t)__shfl_xor((int)top, 2));
    const uint32_t code = mx_scale_code(top);
    const uint32_t w = code == 255u ? 0u : mx_pack8(v, mx_scale_value(code));
    *reinterpret_cast<uint32_t*>(unit_codes + mx_code_offset(b, r) + q * 4) = w;
    if (q == 0) unit_scales[mx_scale_offset(b, r)] = (uint8_t)code;
  }
}

// Along the columns of x [depth, width]: the result's rows are x's columns, its contracted axis
// x's rows.  A workgroup takes 64 columns x 256 rows; a thread takes two columns of one block,
// so a wave reads whole 128-byte lines and a block is one thread's alone.
template <bool BF16>
__global__ __launch_bounds__(kQuantThreads) void mxfp4_quantize_columns_kernel(
    const uint8_t* __restrict__ x, int64_t row_bytes, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
    int64_t depth, int64_t width, int64_t slabs, int64_t row_units) {
  constexpr int kSize = BF16 ? 2 : 4;
  const int64_t slab = blockIdx.x % slabs;
  const int64_t col = blockIdx.x / slabs * 64 + (threadIdx.x & 31) * 2;
  const int b = threadIdx.x >> 5;
  const int64_t k0 = slab * kMxSlab + b * 32;
  const int64_t unit_row = col / kMxRows;
  if (unit_row >= row_units) return;
  const uint8_t* p = x + k0 * row_bytes + col * kSize;
  float v[2][32];
  if (col + 1 < width && k0 + 32 <= depth) {
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      if constexpr (BF16) {
        const uint32_t w = *reinterpret_cast<const u32_any*>(p + k * row_bytes);
        v[0][k] = bf16_lo(w);
        v[1][k] = bf16_hi(w);
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2_any*>(p + k * row_bytes);
        v[0][k] = __uint_as_float(w.x);
        v[1][k] = __uint_as_float(w.y);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        v[c][k] = 0.0f;
        if (col + c < width && k0 + k < depth) {
          if constexpr (BF16)
            v[c][k] = __uint_as_float((uint32_t) reinterpret_cast<const uint16_t*>(p + k * row_bytes)[c] << 16);
          else
            v[c][k] = reinterpret_cast<const float*>(p + k * row_bytes)[c];
        }
      }
  }
  const int64_t unit = unit_row * slabs + slab;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) top = max_u32(top, abs_bits(v[c][k]));
    const uint32_t code = mx_scale_code(top);
    const float scale = mx_scale_value(code);
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = code == 255u ? 0u : mx_pack8(&v[c][8 * j], scale);
    const int r = (int)(col % kMxRows) + c;
    *reinterpret_cast<u32x4*>(codes + unit * kMxCodeBytes + mx_code_offset(b, r)) = w;
    scales[unit * kMxScaleBytes + mx_scale_offset(b, r)] = (uint8_t)code;
  }
}

// Back to rows of bf16 or fp32 (both hold every value exactly: two significant bits, exponents
// from -128 to 127).  The mapping of the quantiser: a wave takes a unit, 8 values per lane.
template <bool BF16>
__global__ __launch_bounds__(kQuantThreads) void mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                        const uint8_t* __restrict__ scales,
                                                                        uint8_t* __restrict__ out, int64_t rows,
                                                                        int64_t cols, int64_t slabs, int64_t units) {
  constexpr int kSize = BF16 ? 2 : 4;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kQuantThreads / 64) + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t row0 = unit / slabs * kMxRows, col0 = unit % slabs * kMxSlab;
  const int col = (lane & 31) * 8, b = (lane & 31) >> 2, q = lane & 3;
  const int64_t left = cols - col0 - col;
  if (left <= 0) return;
  const uint8_t* unit_codes = codes + unit * kMxCodeBytes;
  const uint8_t* unit_scales = scales + unit * kMxScaleBytes;
#pragma unroll
  for (int i = 0; i < kMxRows / 2; ++i) {
    const int r = i * 2 + (lane >> 5);
    const int64_t row = row0 + r;
    if (row >= rows) break;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(unit_codes + mx_code_offset(b, r) + q * 4);
    const float scale = mx_scale_value(unit_scales[mx_scale_offset(b, r)]);
    f32x2_t v[4];
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    uint8_t* p = out + (row * cols + col0 + col) * kSize;
    if constexpr (BF16) {
      u32x4 o;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = pack_bf16x2(v[k].x, v[k].y);
      if (left >= 8) {
        *reinterpret_cast<u32x4_any*>(p) = o;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < left) reinterpret_cast<uint16_t*>(p)[k] = (uint16_t)(o[k >> 1] >> (16 * (k & 1)));
      }
    } else {
      if (left >= 8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 o = {__float_as_uint(v[2 * h].x), __float_as_uint(v[2 * h].y), __float_as_uint(v[2 * h + 1].x),
                           __float_as_uint(v[2 * h + 1].y)};
          reinterpret_cast<u32x4_any*>(p)[h] = o;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < left) reinterpret_cast<float*>(p)[k] = (k & 1) ? v[k >> 1].y : v[k >> 1].x;
      }
    }
  }
}

}  // namespace smr

extern "C" {

int64_t smr_mxfp4_code_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || rows >= smr::kMxMaxExtent || cols >= smr::kMxMaxExtent) return SMR_E_INVALID;
  return smr::mx_row_units(rows) * smr::mx_slabs(cols) * smr::kMxCodeBytes;
}

int64_t smr_mxfp4_scale_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || rows >= smr::kMxMaxExtent || cols >= smr::kMxMaxExtent) return SMR_E_INVALID;
  return smr::mx_row_units(rows) * smr::mx_slabs(cols) * smr::kMxScaleBytes;
}

int smr_mxfp4_quantize(const void* x_dev, int64_t row_stride, void* codes_dev, void* scales_dev, int64_t rows,
                       int64_t cols, int dtype, int transpose, void* stream) {
  using namespace smr;
  if (dtype != SMR_DTYPE_BF16 && dtype != SMR_DTYPE_FP32)
    return fail(SMR_E_INVALID, "smr_mxfp4_quantize: dtype must be bf16 (0) or fp32 (1)");
  if (rows < 0 || cols < 0 || rows >= kMxMaxExtent || cols >= kMxMaxExtent)
    return fail(SMR_E_INVALID, "smr_mxfp4_quantize: rows and cols must be in 0..2^31-1");
  if (rows > 1 && row_stride < cols)
    return fail(SMR_E_INVALID, "smr_mxfp4_quantize: rows must not overlap (row_stride < cols)");
  if (rows == 0 || cols == 0) return 0;
  if (x_dev == nullptr || codes_dev == nullptr || scales_dev == nullptr)
    return fail(SMR_E_INVALID, "smr_mxfp4_quantize: NULL argument");
  const bool bf16 = dtype == SMR_DTYPE_BF16;
  const int64_t size = bf16 ? 2 : 4;
  if ((reinterpret_cast<uintptr_t>(x_dev) & (size - 1)) || (reinterpret_cast<uintptr_t>(codes_dev) & 15u))
    return fail(SMR_E_INVALID, "smr_mxfp4_quantize: misaligned argument (codes: 16 bytes, x: one element)");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const uint8_t* x = static_cast<const uint8_t*>(x_dev);
  uint8_t* codes = static_cast<uint8_t*>(codes_dev);
  uint8_t* scales = static_cast<uint8_t*>(scales_dev);
  if (transpose) {
    const int64_t slabs = mx_slabs(rows), row_units = mx_row_units(cols);
    const int64_t grid = (cols + 63) / 64 * slabs;
    if (grid > kMxMaxGrid) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_quantize: too large for one launch");
    if (bf16)
      hipLaunchKernelGGL((mxfp4_quantize_columns_kernel<true>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, x,
                         row_stride * size, codes, scales, rows, cols, slabs, row_units);
    else
      hipLaunchKernelGGL((mxfp4_quantize_columns_kernel<false>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, x,
                         row_stride * size, codes, scales, rows, cols, slabs, row_units);
  } else {
    const int64_t slabs = mx_slabs(cols), units = mx_row_units(rows) * slabs;
    const int64_t grid = (units + kQuantThreads / 64 - 1) / (kQuantThreads / 64);
    if (grid > kMxMaxGrid) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_quantize: too large for one launch");
    if (bf16)
      hipLaunchKernelGGL((mxfp4_quantize_kernel<true>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, x,
                         row_stride * size, codes, scales, rows, cols, slabs, units);
    else
      hipLaunchKernelGGL((mxfp4_quantize_kernel<false>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, x,
                         row_stride * size, codes, scales, rows, cols, slabs, units);
  }
  return check_hip(hipGetLastError(), "smr_mxfp4_quantize launch");
}

int smr_mxfp4_dequantize(const void* codes_dev, const void* scales_dev, void* out_dev, int64_t rows, int64_t cols,
                         int dtype, void* stream) {
  using namespace smr;
  if (dtype != SMR_DTYPE_BF16 && dtype != SMR_DTYPE_FP32)
    return fail(SMR_E_INVALID, "smr_mxfp4_dequantize: dtype must be bf16 (0) or fp32 (1)");
  if (rows < 0 || cols < 0 || rows >= kMxMaxExtent || cols >= kMxMaxExtent)
    return fail(SMR_E_INVALID, "smr_mxfp4_dequantize: rows and cols must be in 0..2^31-1");
  if (rows == 0 || cols == 0) return 0;
  if (codes_dev == nullptr || scales_dev == nullptr || out_dev == nullptr)
    return fail(SMR_E_INVALID, "smr_mxfp4_dequantize: NULL argument");
  const bool bf16 = dtype == SMR_DTYPE_BF16;
  if ((reinterpret_cast<uintptr_t>(out_dev) & (bf16 ? 1u : 3u)) || (reinterpret_cast<uintptr_t>(codes_dev) & 15u))
    return fail(SMR_E_INVALID, "smr_mxfp4_dequantize: misaligned argument (codes: 16 bytes, out: one element)");
  const int64_t slabs = mx_slabs(cols), units = mx_row_units(rows) * slabs;
  const int64_t grid = (units + kQuantThreads / 64 - 1) / (kQuantThreads / 64);
  if (grid > kMxMaxGrid) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_dequantize: too large for one launch");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const uint8_t* codes = static_cast<const uint8_t*>(codes_dev);
  const uint8_t* scales = static_cast<const uint8_t*>(scales_dev);
  uint8_t* out = static_cast<uint8_t*>(out_dev);
  if (bf16)
    hipLaunchKernelGGL((mxfp4_dequantize_kernel<true>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, codes, scales,
                       out, rows, cols, slabs, units);
  else
    hipLaunchKernelGGL((mxfp4_dequantize_kernel<false>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, codes, scales,
                       out, rows, cols, slabs, units);
  return check_hip(hipGetLastError(), "smr_mxfp4_dequantize launch");
}

}  // extern "C"
