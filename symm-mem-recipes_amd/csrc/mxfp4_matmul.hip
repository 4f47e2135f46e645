// Product of two 4-bit microscaled operands:  C[M,N] = A[M,K] * B[N,K]^T, fp32 accumulation in
// v_mfma_scale_f32_16x16x128_f8f6f4 (e2m1 operands; the instruction applies the scales of both
// operands' blocks), one rounding to bf16 (or none: fp32).
//
// Operands come in MFMA order (mxfp4_layout.hpp).  B's fragment is the instruction's first
// operand, so a lane ends up with 4 consecutive columns of one row of C.
#include "mxfp4_layout.hpp"

namespace smr {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// D += A x B over 128 of K; `step` picks the byte of the scale words that belongs to it.
template <int STEP>
__device__ __forceinline__ f32x4 mfma_mx(const i32x4& first, const i32x4& second, const f32x4& acc, uint32_t first_scale,
                                         uint32_t second_scale) {
  const i32x8 a = {first.x, first.y, first.z, first.w, 0, 0, 0, 0};
  const i32x8 b = {second.x, second.y, second.z, second.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, STEP, (int)first_scale, STEP,
                                                          (int)second_scale);
}

// Four consecutive columns n .. n+3 of row m.
template <bool BF16>
__device__ __forceinline__ void store4(uint8_t* c, int64_t m, int64_t n, int64_t N, const f32x4& d) {
  const int64_t at = m * N + n;
  if constexpr (BF16) {
    const u32x2 v = {pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3])};
    uint16_t* p = reinterpret_cast<uint16_t*>(c) + at;
    if (n + 4 <= N) {
      *reinterpret_cast<u32x2_any*>(p) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) p[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
  } else {
    float* p = reinterpret_cast<float*>(c) + at;
    if (n + 4 <= N) {
      const u32x4_any v = {__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3])};
      *reinterpret_cast<u32x4_any*>(p) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) p[e] = d[e];
    }
  }
}

// A workgroup computes NG * 16 columns of C for TG * 16 of its rows.  Its WAVES waves share K:
// wave w takes slabs w, w + WAVES, ... straight from memory into registers, and the partial sums
// are added in wave order through LDS.
template <bool BF16, int TG, int NG, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void mxfp4_matmul_few_kernel(
    const uint8_t* __restrict__ a_codes, const uint8_t* __restrict__ a_scales, const uint8_t* __restrict__ b_codes,
    const uint8_t* __restrict__ b_scales, uint8_t* __restrict__ c, int64_t M, int64_t N, int64_t slabs,
    int64_t m_units, int64_t n_units) {
  __shared__ f32x4 part[WAVES][NG * TG][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n_unit0 = (int64_t)blockIdx.x * NG, m_unit0 = (int64_t)blockIdx.y * TG;
  const uint8_t *ac[TG], *as[TG], *bc[NG], *bs[NG];
#pragma unroll
  for (int t = 0; t < TG; ++t) {
    // (units past the last repeat it; their products are not stored)
    const int64_t u = (m_unit0 + t < m_units ? m_unit0 + t : m_units - 1) * slabs;
    ac[t] = a_codes + u * kMxCodeBytes + lane * 16;
    as[t] = a_scales + u * kMxScaleBytes + lane * 2;
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int64_t u = (n_unit0 + g < n_units ? n_unit0 + g : n_units - 1) * slabs;
    bc[g] = b_codes + u * kMxCodeBytes + lane * 16;
    bs[g] = b_scales + u * kMxScaleBytes + lane * 2;
  }
  f32x4 acc[NG][TG];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int t = 0; t < TG; ++t) acc[g][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll 2
  for (int64_t s = wave; s < slabs; s += WAVES) {
    i32x4 bf[NG][2], af[TG][2];
    uint32_t bsc[NG], asc[TG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      bf[g][0] = *reinterpret_cast<const i32x4*>(bc[g] + s * kMxCodeBytes);
      bf[g][1] = *reinterpret_cast<const i32x4*>(bc[g] + s * kMxCodeBytes + 1024);
      bsc[g] = *reinterpret_cast<const uint16_t*>(bs[g] + s * kMxScaleBytes);
    }
#pragma unroll
    for (int t = 0; t < TG; ++t) {
      af[t][0] = *reinterpret_cast<const i32x4*>(ac[t] + s * kMxCodeBytes);
      af[t][1] = *reinterpret_cast<const i32x4*>(ac[t] + s * kMxCodeBytes + 1024);
      asc[t] = *reinterpret_cast<const uint16_t*>(as[t] + s * kMxScaleBytes);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int t = 0; t < TG; ++t) {
        acc[g][t] = mfma_mx<0>(bf[g][0], af[t][0], acc[g][t], bsc[g], asc[t]);
        acc[g][t] = mfma_mx<1>(bf[g][1], af[t][1], acc[g][t], bsc[g], asc[t]);
      }
  }
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int t = 0; t < TG; ++t) part[wave][g * TG + t][lane] = acc[g][t];
  __syncthreads();
  for (int f = wave; f < NG * TG; f += WAVES) {
    f32x4 d = part[0][f][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const f32x4 p = part[w][f][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] += p[e];
    }
    const int g = f / TG, t = f % TG;
    const int64_t m = (m_unit0 + t) * kMxRows + (lane & 15);
    const int64_t n = (n_unit0 + g) * kMxRows + (lane >> 4) * 4;
    if (m < M && n < N) store4<BF16>(c, m, n, N, d);
  }
}

struct MxOperands {
  const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
  uint8_t* c;
  int64_t M, N, K;
};

template <bool BF16, int TG, int NG, int WAVES>
static int launch_few(const MxOperands& o, hipStream_t s) {
  const int64_t m_units = mx_row_units(o.M), n_units = mx_row_units(o.N);
  const int64_t gx = (n_units + NG - 1) / NG, gy = (m_units + TG - 1) / TG;
  if (gx > kMxMaxGrid / 4 || gy > 65535) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_matmul: too large for one launch");
  hipLaunchKernelGGL((mxfp4_matmul_few_kernel<BF16, TG, NG, WAVES>), dim3((unsigned)gx, (unsigned)gy), dim3(WAVES * 64),
                     0, s, o.a_codes, o.a_scales, o.b_codes, o.b_scales, o.c, o.M, o.N, mx_slabs(o.K), m_units, n_units);
  return check_hip(hipGetLastError(), "smr_mxfp4_matmul launch");
}

template <bool BF16>
static int launch_matmul(const MxOperands& o, hipStream_t s) {
  if (o.M <= 16) return launch_few<BF16, 1, 1, 8>(o, s);
  return launch_few<BF16, 4, 2, 4>(o, s);
}

}  // namespace smr

extern "C" {

int smr_mxfp4_matmul(const void* a_codes_dev, const void* a_scales_dev, const void* b_codes_dev,
                     const void* b_scales_dev, void* c_dev, int64_t M, int64_t N, int64_t K, int out_dtype,
                     void* stream) {
  using namespace smr;
  if (out_dtype != SMR_DTYPE_BF16 && out_dtype != SMR_DTYPE_FP32)
    return fail(SMR_E_INVALID, "smr_mxfp4_matmul: out_dtype must be bf16 (0) or fp32 (1)");
  if (M < 0 || N < 0 || K < 1 || M >= kMxMaxExtent || N >= kMxMaxExtent || K >= kMxMaxExtent)
    return fail(SMR_E_INVALID, "smr_mxfp4_matmul: M and N must be in 0..2^31-1, K in 1..2^31-1");
  if (M == 0 || N == 0) return 0;
  if (a_codes_dev == nullptr || a_scales_dev == nullptr || b_codes_dev == nullptr || b_scales_dev == nullptr ||
      c_dev == nullptr)
    return fail(SMR_E_INVALID, "smr_mxfp4_matmul: NULL argument");
  const uintptr_t unaligned = reinterpret_cast<uintptr_t>(a_codes_dev) | reinterpret_cast<uintptr_t>(a_scales_dev) |
                              reinterpret_cast<uintptr_t>(b_codes_dev) | reinterpret_cast<uintptr_t>(b_scales_dev);
  if ((unaligned & 15u) || (reinterpret_cast<uintptr_t>(c_dev) & (out_dtype == SMR_DTYPE_BF16 ? 1u : 3u)))
    return fail(SMR_E_INVALID, "smr_mxfp4_matmul: misaligned argument (operands: 16 bytes, c: one element)");
  const MxOperands o = {static_cast<const uint8_t*>(a_codes_dev), static_cast<const uint8_t*>(a_scales_dev),
                        static_cast<const uint8_t*>(b_codes_dev), static_cast<const uint8_t*>(b_scales_dev),
                        static_cast<uint8_t*>(c_dev), M, N, K};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return out_dtype == SMR_DTYPE_BF16 ? launch_matmul<true>(o, s) : launch_matmul<false>(o, s);
}

}  // extern "C"
