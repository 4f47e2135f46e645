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
//
// All of it is bound by memory: 16384 x 8192 bf16 55 us (340 MB, 6.2 TB/s) and back 50 us, 8191 x 3584 fp32 along
// the columns 26.6 us (5.0 TB/s); a single row takes a launch and two trips to memory, 3.3 us.
#include "mxfp4_layout.hpp"

namespace smr {

constexpr int kQuantThreads = 256;

// Along the rows of x.  A wave takes one unit, 8 elements of a block per lane and load; four lanes that share
// a block find its scale, and between them hold the scales of their rows' eight blocks.  A load takes one
// block of all 16 rows, and their codes are 256 contiguous bytes - or, from memory (STREAM), two blocks of 8
// rows, whole lines of bf16 (16384 x 8192 55 us, block by block 60; 16384 x 8200 63 and 74; out of the caches
// 1001 x 4000 4.5 and 4.3, fp32 6.6 and 6.1).
template <bool BF16, bool STREAM>
__global__ __launch_bounds__(kQuantThreads) void mxfp4_quantize_kernel(const uint8_t* __restrict__ x, int64_t row_bytes,
                                                                      uint8_t* __restrict__ codes,
                                                                      uint8_t* __restrict__ scales, int64_t rows,
                                                                      int64_t cols, uint32_t slabs, uint32_t units) {
  constexpr int kSize = BF16 ? 2 : 4;
  constexpr int kWide = STREAM ? 2 : 1;                       // blocks per load
  constexpr int kRows = kMxRows / kWide, kSteps = 8 / kWide;  // rows per load, loads per row
  const int lane = threadIdx.x & 63;
  const uint32_t at = blockIdx.x * (kQuantThreads / 64) + (threadIdx.x >> 6);
  if (at >= units) return;
  const uint32_t row_unit = at / slabs, slab = at - row_unit * slabs;
  const int64_t row0 = (int64_t)row_unit * kMxRows, col0 = (int64_t)slab * kMxSlab;
  const int64_t unit = mx_unit(row_unit, slab, units / slabs);
  const int r = lane / (4 * kWide), side = (lane >> 2) % kWide, q = lane & 3;
  const int64_t col = col0 + side * 32 + q * 8;
  Mx8<BF16> v[kWide][kSteps][1];
#pragma unroll
  for (int i = 0; i < kWide; ++i) {
    // (rows past the last repeat it and are cleared: loads under a branch would wait for one another)
    const int64_t row = row0 + i * kRows + r;
    const uint8_t* p = x + (row < rows ? row : rows - 1) * row_bytes + col * kSize;
    if (col0 + kMxSlab <= cols) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j) v[i][j][0].template load<STREAM>(p + j * (kWide * 32 * kSize));
    } else {
#pragma unroll
      for (int j = 0; j < kSteps; ++j) v[i][j][0].load(p + j * (kWide * 32 * kSize), cols - col - j * (kWide * 32));
    }
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (uint32_t& w : v[i][j][0].w) w = row < rows ? w : 0u;
  }
  uint32_t* out = reinterpret_cast<uint32_t*>(codes + unit * kMxCodeBytes) + q;
  uint32_t mine = 0;              // scales of a block and the fourth after it, of one of the lane's rows
#pragma unroll
  for (int i = 0; i < kWide; ++i)
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      uint32_t top = mx_top<BF16>(v[i][j]);
      top = max_u32(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));   // quad_perm [1,0,3,2]
      top = max_u32(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));   // quad_perm [2,3,0,1]
      const uint32_t code = mx_scale_code(top);
      out[mx_code_offset(j * kWide + side, i * kRows + r) / 4] =
          code == 255u ? 0u : mx_pack8<BF16>(v[i][j][0], mx_scale_value(code));
      if (q == i * (kSteps / 2) + j % (kSteps / 2)) mine |= code << (8 * (j / (kSteps / 2)));
    }
  const int of_row = q / (kSteps / 2) * kRows + r, of_block = q % (kSteps / 2) * kWide + side;
  reinterpret_cast<uint16_t*>(scales + unit * kMxScaleBytes)[of_block * 16 + of_row] = (uint16_t)mine;
}

// Along the columns of x [depth, width]: the result's rows are x's columns, its contracted axis
// x's rows.  A workgroup takes 64 columns x 256 rows; a thread takes two columns of one block,
// so a wave reads whole 128-byte lines and a block is one thread's alone.
template <bool BF16, bool STREAM>
__global__ __launch_bounds__(kQuantThreads) void mxfp4_quantize_columns_kernel(
    const uint8_t* __restrict__ x, int64_t row_bytes, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
    int64_t depth, int64_t width, uint32_t slabs, int64_t row_units, bool across) {
  constexpr int kSize = BF16 ? 2 : 4;
  // neighbours take the slabs of the same columns, or (across) the same rows' next columns
  const uint32_t groups = (uint32_t)((width + 63) / 64), inner = across ? groups : slabs;
  const uint32_t outer_at = blockIdx.x / inner, inner_at = blockIdx.x - outer_at * inner;
  const uint32_t slab = across ? outer_at : inner_at, group = across ? inner_at : outer_at;
  const int64_t col = (int64_t)group * 64 + (threadIdx.x & 31) * 2;
  const int b = threadIdx.x >> 5;
  const int64_t k0 = (int64_t)slab * kMxSlab + b * 32;
  const int64_t unit_row = col / kMxRows;
  if (unit_row >= row_units) return;
  float v[2][32];
  auto load = [&](const uint8_t* p, int k) __attribute__((always_inline)) {
    if constexpr (BF16) {
      const u32_any* at = reinterpret_cast<const u32_any*>(p);
      const uint32_t w = STREAM ? __builtin_nontemporal_load(at) : *at;
      v[0][k] = bf16_lo(w);
      v[1][k] = bf16_hi(w);
    } else {
      const u32x2_any* at = reinterpret_cast<const u32x2_any*>(p);
      const u32x2 w = STREAM ? __builtin_nontemporal_load(at) : *at;
      v[0][k] = __uint_as_float(w.x);
      v[1][k] = __uint_as_float(w.y);
    }
  };
  if (col + 1 < width && k0 + 32 <= depth) {
    const uint8_t* p = x + k0 * row_bytes + col * kSize;
#pragma unroll
    for (int k = 0; k < 32; ++k) load(p + k * row_bytes, k);
  } else if (width > 1) {
    // The last row and the last pair of columns again for what lies behind them, cleared afterwards: loads under
    // branches would wait for one another (1001 x 4000 bf16: 8.0 us, so 5.3).
    const int64_t first = col < width - 2 ? col : width - 2, past = col - first;
    int64_t at = (k0 < depth ? k0 : depth - 1) * row_bytes + first * kSize;
    const int rows = k0 < depth ? (depth - k0 < 32 ? (int)(depth - k0) : 32) : 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      load(x + at, k);
      at += k + 1 < rows ? row_bytes : 0;
      asm volatile("" : "+v"(at));                 // (one running address, not 32)
    }
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const bool there = k < rows;
      v[0][k] = there && past < 2 ? (past == 1 ? v[1][k] : v[0][k]) : 0.0f;
      v[1][k] = there && past == 0 ? v[1][k] : 0.0f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      v[0][k] = v[1][k] = 0.0f;
      if (col == 0 && k0 + k < depth) {
        if constexpr (BF16) v[0][k] = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(x + (k0 + k) * row_bytes) << 16);
        else v[0][k] = *reinterpret_cast<const float*>(x + (k0 + k) * row_bytes);
      }
    }
  }
  const int64_t unit = mx_unit(unit_row, slab, row_units);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) top = max_u32(top, abs_bits(v[c][k]));
    const uint32_t code = mx_scale_code(top);
    const float scale = mx_scale_value(code);
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Mx8<false> part;
#pragma unroll
      for (int k = 0; k < 8; ++k) part.w[k] = __float_as_uint(v[c][8 * j + k]);
      w[j] = code == 255u ? 0u : mx_pack8<false>(part, scale);
    }
    const int r = (int)(col % kMxRows) + c;
    *reinterpret_cast<u32x4*>(codes + unit * kMxCodeBytes + mx_code_offset(b, r)) = w;
    scales[unit * kMxScaleBytes + mx_scale_offset(b, r)] = (uint8_t)code;
  }
}

template <bool STREAM>
__device__ __forceinline__ void put_vec(uint8_t* p, const u32x4& v) {
  if constexpr (STREAM) __builtin_nontemporal_store((u32x4_any)v, reinterpret_cast<u32x4_any*>(p));
  else *reinterpret_cast<u32x4_any*>(p) = v;
}

// Back to rows of bf16 or fp32 (both hold every value exactly: two significant bits, exponents
// from -128 to 127).  A wave takes a unit, 8 values per lane, two rows at a time.
template <bool BF16, bool STREAM>
__global__ __launch_bounds__(kQuantThreads) void mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                        const uint8_t* __restrict__ scales,
                                                                        uint8_t* __restrict__ out, int64_t rows,
                                                                        int64_t cols, uint32_t slabs, uint32_t units) {
  constexpr int kSize = BF16 ? 2 : 4;
  const int lane = threadIdx.x & 63;
  const uint32_t at = blockIdx.x * (kQuantThreads / 64) + (threadIdx.x >> 6);
  if (at >= units) return;
  const uint32_t row_unit = at / slabs, slab = at - row_unit * slabs;
  const int64_t row0 = (int64_t)row_unit * kMxRows, col0 = (int64_t)slab * kMxSlab;
  const int64_t unit = mx_unit(row_unit, slab, units / slabs);
  const int col = (lane & 31) * 8, b = (lane & 31) >> 2, q = lane & 3;
  const int64_t left = cols - col0 - col;
  if (left <= 0) return;
  const uint8_t* unit_codes = codes + unit * kMxCodeBytes;
  const uint8_t* unit_scales = scales + unit * kMxScaleBytes;
  // (all rows of a unit are stored, also those behind the matrix: the loads need no branch)
  uint32_t words[kMxRows / 2], scale_codes[kMxRows / 2];
#pragma unroll
  for (int i = 0; i < kMxRows / 2; ++i) {
    const int r = i * 2 + (lane >> 5);
    words[i] = *reinterpret_cast<const uint32_t*>(unit_codes + mx_code_offset(b, r) + q * 4);
    scale_codes[i] = unit_scales[mx_scale_offset(b, r)];
  }
#pragma unroll
  for (int i = 0; i < kMxRows / 2; ++i) {
    const int64_t row = row0 + i * 2 + (lane >> 5);
    if (row >= rows) break;
    const uint32_t w = words[i];
    const float scale = mx_scale_value(scale_codes[i]);
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
        put_vec<STREAM>(p, o);
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
          put_vec<STREAM>(p + h * 16, o);
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
                       int64_t cols, int dtype, int transpose, void* stream_ptr) {
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
  if ((reinterpret_cast<uintptr_t>(x_dev) & (size - 1)) ||
      ((reinterpret_cast<uintptr_t>(codes_dev) | reinterpret_cast<uintptr_t>(scales_dev)) & 15u))
    return fail(SMR_E_INVALID, "smr_mxfp4_quantize: misaligned argument (codes and scales: 16 bytes, x: one element)");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream_ptr);
  const uint8_t* x = static_cast<const uint8_t*>(x_dev);
  uint8_t* codes = static_cast<uint8_t*>(codes_dev);
  uint8_t* scales = static_cast<uint8_t*>(scales_dev);
  // Past the caches from 64 MiB on: what the caches can hold may be there (4096 x 4096 bf16 9.3 us, streamed
  // 10.0), what they cannot only drives the codes out of them (16384 x 8192 64 us, streamed 55; along
  // the columns bf16 75 and 65; with the codes read back behind it 164 and 133).
  const bool stream = rows * cols * size >= ((int64_t)64 << 20);
  if (transpose) {
    const int64_t slabs = mx_slabs(rows), row_units = mx_row_units(cols);
    const int64_t grid = (cols + 63) / 64 * slabs;
    if (grid > kMxMaxGrid) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_quantize: too large for one launch");
    // Large fp32 inputs across the rows (16384 x 8192 106 us, down the columns 122; 8191 x 3584 26.6 and 27.9; 4096 x
    // 4096 15.6 and 13.9; 16384 x 8192 bf16 69 and 65).
    const bool across = !bf16 && rows * cols * size > ((int64_t)96 << 20);
#define SMR_QUANT(B, S)                                                                                                \
  hipLaunchKernelGGL((mxfp4_quantize_columns_kernel<B, S>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, x,        \
                     row_stride * size, codes, scales, rows, cols, (uint32_t)slabs, row_units, across)
    if (bf16 && stream) SMR_QUANT(true, true);
    else if (bf16) SMR_QUANT(true, false);
    else if (stream) SMR_QUANT(false, true);
    else SMR_QUANT(false, false);
#undef SMR_QUANT
  } else {
    const int64_t slabs = mx_slabs(cols), units = mx_row_units(rows) * slabs;
    const int64_t grid = (units + kQuantThreads / 64 - 1) / (kQuantThreads / 64);
    if (grid > kMxMaxGrid) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_quantize: too large for one launch");
#define SMR_QUANT(B, S)                                                                                             \
  hipLaunchKernelGGL((mxfp4_quantize_kernel<B, S>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, x,             \
                     row_stride * size, codes, scales, rows, cols, (uint32_t)slabs, (uint32_t)units)
    if (bf16 && stream) SMR_QUANT(true, true);
    else if (bf16) SMR_QUANT(true, false);
    else if (stream) SMR_QUANT(false, true);
    else SMR_QUANT(false, false);
#undef SMR_QUANT
  }
  return check_hip(hipGetLastError(), "smr_mxfp4_quantize launch");
}

int smr_mxfp4_dequantize(const void* codes_dev, const void* scales_dev, void* out_dev, int64_t rows, int64_t cols,
                         int dtype, void* stream_ptr) {
  using namespace smr;
  if (dtype != SMR_DTYPE_BF16 && dtype != SMR_DTYPE_FP32)
    return fail(SMR_E_INVALID, "smr_mxfp4_dequantize: dtype must be bf16 (0) or fp32 (1)");
  if (rows < 0 || cols < 0 || rows >= kMxMaxExtent || cols >= kMxMaxExtent)
    return fail(SMR_E_INVALID, "smr_mxfp4_dequantize: rows and cols must be in 0..2^31-1");
  if (rows == 0 || cols == 0) return 0;
  if (codes_dev == nullptr || scales_dev == nullptr || out_dev == nullptr)
    return fail(SMR_E_INVALID, "smr_mxfp4_dequantize: NULL argument");
  const bool bf16 = dtype == SMR_DTYPE_BF16;
  if ((reinterpret_cast<uintptr_t>(out_dev) & (bf16 ? 1u : 3u)) ||
      ((reinterpret_cast<uintptr_t>(codes_dev) | reinterpret_cast<uintptr_t>(scales_dev)) & 15u))
    return fail(SMR_E_INVALID, "smr_mxfp4_dequantize: misaligned argument (codes and scales: 16 bytes, out: one element)");
  const int64_t slabs = mx_slabs(cols), units = mx_row_units(rows) * slabs;
  const int64_t grid = (units + kQuantThreads / 64 - 1) / (kQuantThreads / 64);
  if (grid > kMxMaxGrid) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_dequantize: too large for one launch");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream_ptr);
  const uint8_t* codes = static_cast<const uint8_t*>(codes_dev);
  const uint8_t* scales = static_cast<const uint8_t*>(scales_dev);
  uint8_t* out = static_cast<uint8_t*>(out_dev);
  // Past the caches where rows are whole 16-byte pieces (16384 x 8192 bf16 50 us, through them 80; 4096 x 4096 7.8
  // and 9.2), else only from 128 MiB on: pieces of a line that come apart are written apart (3584 x 8191 19.1 and
  // 14.4 us, 16383 x 8191 87 and 105).
  const int64_t size = bf16 ? 2 : 4;
  const bool stream = (cols * size % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0) ||
                      rows * cols * size >= ((int64_t)128 << 20);
#define SMR_DEQUANT(B, S)                                                                                            \
  hipLaunchKernelGGL((mxfp4_dequantize_kernel<B, S>), dim3((unsigned)grid), dim3(kQuantThreads), 0, s, codes, scales, \
                     out, rows, cols, (uint32_t)slabs, (uint32_t)units)
  if (bf16 && stream) SMR_DEQUANT(true, true);
  else if (bf16) SMR_DEQUANT(true, false);
  else if (stream) SMR_DEQUANT(false, true);
  else SMR_DEQUANT(false, false);
#undef SMR_DEQUANT
  return check_hip(hipGetLastError(), "smr_mxfp4_dequantize launch");
}

}  // extern "C"
