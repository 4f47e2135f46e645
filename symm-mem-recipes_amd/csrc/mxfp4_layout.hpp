// The 4-bit microscaled operand (OCP MXFP4: e2m1 elements, one e8m0 scale per 32 of them along
// the contracted axis) as the kernels keep it: in the order in which the block-scaled MFMA
// (v_mfma_scale_f32_16x16x128_f8f6f4) takes it.
//
// A unit is 16 rows x 256 of the contracted axis:
//   codes   2048 B: [2 steps of 128][64 lanes][16 B]; lane l of a step holds row l & 15 and the
//           32 elements number l >> 4 of the step's four blocks, two elements a byte, the first
//           in the low half;
//   scales  128 B: [64 lanes][2 steps], the biased exponent of that block (255 = NaN).
// Units lie [rows / 16][contracted / 256], so a wave's operand of one MFMA is 1 KiB in a row -
// a load instruction of 16 B per lane, from memory or from LDS, with no address arithmetic and
// no bank conflict - and a run along the contracted axis is one contiguous stream.
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

// Byte offsets inside a unit of block b (0..7) of row r (0..15).
__host__ __device__ inline int mx_code_offset(int b, int r) { return ((b >> 2) * 64 + (b & 3) * 16 + r) * 16; }
__host__ __device__ inline int mx_scale_offset(int b, int r) { return ((b & 3) * 16 + r) * 2 + (b >> 2); }

}  // namespace smr
