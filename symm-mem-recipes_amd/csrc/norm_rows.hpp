// What the kernels that reduce rows share (all_reduce_norm*.hip, norm_backward.hip): vectors of a row
// of any width and alignment, and sums over a row.
#pragma once

#include <type_traits>

#include "smr_internal.hpp"

namespace smr {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 128-bit accesses at an element's alignment: rows of an odd width start anywhere
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __attribute__((address_space(1))) const u32x4_any GlobalVecAny;

enum GateKind : int { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateElement = 3 };

constexpr int kNormMaxCols = 16384;

template <bool BF16>
struct Row {
  static constexpr int kVec = BF16 ? 8 : 4;       // elements of a 128-bit access
  static constexpr int kSize = BF16 ? 2 : 4;

  // A row's vector at element `col`, or the row's last whole vector where that would reach past the end:
  // no branch around the load.  `Tail` puts the elements in place.  STREAM: past the caches, for what is
  // read once.
  template <bool STREAM = false>
  static __device__ __forceinline__ u32x4 load(const void* row, int col, int cols) {
    const int at = col < cols - kVec ? col : cols - kVec;
    GlobalVecAny* p = (GlobalVecAny*)(uintptr_t)(static_cast<const uint8_t*>(row) + (uint32_t)at * (uint32_t)kSize);
    return STREAM ? __builtin_nontemporal_load(p) : *p;
  }
  static __device__ __forceinline__ float get(const u32x4& v, int e) {
    if constexpr (BF16) return (e & 1) ? bf16_hi(v[e >> 1]) : bf16_lo(v[e >> 1]);
    else return __uint_as_float(v[e]);
  }
  template <bool STREAM = false>
  static __device__ __forceinline__ void store(void* row, int col, int cols, const float (&f)[kVec]) {
    uint8_t* p = static_cast<uint8_t*>(row) + (uint32_t)col * (uint32_t)kSize;
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (BF16) v[k] = pack_bf16x2(f[2 * k], f[2 * k + 1]);
      else v[k] = __float_as_uint(f[k]);
    }
    if (col + kVec <= cols) {
      if constexpr (STREAM) __builtin_nontemporal_store((u32x4_any)v, reinterpret_cast<u32x4_any*>(p));
      else *reinterpret_cast<u32x4_any*>(p) = v;
    } else if (col < cols) {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (col + e < cols) {
          if constexpr (BF16) reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
          else reinterpret_cast<uint32_t*>(p)[e] = v[e];
        }
    }
  }
  static __device__ __forceinline__ float one(const void* p, int64_t i) {
    if constexpr (BF16) return __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
    else return static_cast<const float*>(p)[i];
  }
  static __device__ __forceinline__ void put_one(void* p, int64_t i, float f) {
    if constexpr (BF16) static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16_bits(f);
    else static_cast<float*>(p)[i] = f;
  }
};

// How a vector at element `col` lies in a row of `cols` elements: `shift` of the elements that Row::load
// brought belong to vectors before it (all of them where it lies behind the row).
template <int V>
struct Tail {
  int shift;
  __device__ __forceinline__ Tail(int col, int cols) {
    const int over = col - (cols - V);
    shift = over < 0 ? 0 : (over > V ? V : over);
    // (made anew where it is used: the comparisons with it, kept for every element of every chunk, would
    // take more scalar registers than there are)
    asm volatile("" : "+v"(shift));
  }
  // elements to their places, zeros behind the row
  __device__ __forceinline__ void place(float (&f)[V]) const {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (shift & V) ? 0.0f : f[e];
#pragma unroll
    for (int d = V / 2; d > 0; d /= 2)
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = (shift & d) ? (e + d < V ? f[e + d] : 0.0f) : f[e];
  }
};

// Sum over a wave in every lane's row of 16 (and `wave_sum` over all four), the order the same in all.
__device__ __forceinline__ float row16_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});      // quad_perm [1,0,3,2]
  v += dpp(v, std::integral_constant<int, 0x4E>{});      // quad_perm [2,3,0,1]
  v += dpp(v, std::integral_constant<int, 0x141>{});     // row_half_mirror
  v += dpp(v, std::integral_constant<int, 0x140>{});     // row_mirror
  return v;
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = row16_sum(v);
  return ((lane_value(v, 0) + lane_value(v, 16)) + lane_value(v, 32)) + lane_value(v, 48);
}

// Sums of N values over the workgroup's `waves` waves, the same bits in every thread.  `slots` is not
// read or written by the call before the last one, so one barrier per call is enough with two sets
// taken in turn.
template <int N>
__device__ __forceinline__ void workgroup_sums(float (&v)[N], float (*slots)[N], int waves) {
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = wave_sum(v[n]);
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) slots[threadIdx.x >> 6][n] = v[n];
  }
  __syncthreads();
  // at most 16 waves: one of their sums per lane of a row of 16
  const int w = threadIdx.x & 15;
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = row16_sum(w < waves ? slots[w][n] : 0.0f);
}

// Squares leave fp32's range long before values do: past 2^64 they are infinite, below 2^-63 they lose bits.  A row
// whose mean square (eps added) comes out outside [kLeastMean, infinity) is scaled by a power of two and its
// squares are summed again; the factor drops out of v * (mean)^-1/2.  With up to 2^14 columns the scaled squares'
// sum is in [2^-46, 2^110] one way and below 2^114 the other.
constexpr float kLeastMean = 0x1p-100f;
__device__ __forceinline__ bool mean_out_of_range(float mean) { return !(mean >= kLeastMean && mean < __builtin_inff()); }
__device__ __forceinline__ float mean_rescale(float mean) { return mean < kLeastMean ? 0x1p100f : 0x1p-80f; }

// Threads and 128-bit chunks per thread for a row; the smallest number of chunks that fits.
inline bool norm_shape(int cols, int vec, int max_threads, int& threads, int& chunks) {
  for (chunks = 1; chunks <= 8; chunks *= 2) {
    const int need = (cols + vec * chunks - 1) / (vec * chunks);
    if (need <= max_threads) {
      threads = (need + 63) / 64 * 64;
      return true;
    }
  }
  return false;
}

// What both passes refuse; nullptr if nothing.
inline const char* check_norm_sizes(int64_t rows, int64_t cols, int dtype, int gate_kind, const void* gate) {
  if (dtype != SMR_DTYPE_BF16 && dtype != SMR_DTYPE_FP32) return "dtype must be bf16 (0) or fp32 (1)";
  if (rows < 0 || rows >= ((int64_t)1 << 40)) return "rows out of range";
  if (cols < 1) return "cols must be at least 1";
  if (gate_kind < kGateNone || gate_kind > kGateElement) return "unknown gate kind";
  if ((gate_kind == kGateNone) != (gate == nullptr)) return "gate and gate_kind must both be set or neither";
  return nullptr;
}
int fail_norm(int code, const char* who, const char* what);

}  // namespace smr
