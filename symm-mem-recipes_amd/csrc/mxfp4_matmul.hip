// Product of two 4-bit microscaled operands:  C[M,N] = A[M,K] * B[N,K]^T, fp32 accumulation in
// v_mfma_scale_f32_16x16x128_f8f6f4 (e2m1 operands; the instruction applies the scales of both
// operands' blocks), one rounding to bf16 (or none: fp32).
//
// Operands come in MFMA order (mxfp4_layout.hpp).  B's fragment is the instruction's first
// operand, so a lane ends up with 4 consecutive columns of one row of C.
//
// Three families.  A few rows are bound by reading B: K is split over the waves of a workgroup, and
// B streams into registers (1 x 8192 x 8192: 8.0 us, 4.5 TB/s) or, wide, through LDS (64 x 28672 x 8192:
// 23.7 us, 5.4 TB/s).  Results with too few large tiles are bound by the latency of a slab (ring, small
// tiles); large ones by the matrix cores (tiles).
#include "mxfp4_layout.hpp"

namespace smr {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// D += A x B over 128 of K; `step` picks the byte of the scale words that belongs to it.
template <int STEP>
__device__ __forceinline__ f32x4 mfma_mx(const i32x4& first, const i32x4& second, const f32x4& acc, uint32_t first_scale,
                                         uint32_t second_scale) {
  const i32x8 a = {first.x, first.y, first.z, first.w, 0, 0, 0, 0};
  const i32x8 b = {second.x, second.y, second.z, second.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, STEP, (int)first_scale, STEP,
                                                          (int)second_scale);
}

// Four consecutive columns of a row, all of them there.
template <bool BF16>
__device__ __forceinline__ void put4(uint8_t* p, const f32x4& d) {
  if constexpr (BF16) {
    const u32x2 v = {pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3])};
    *reinterpret_cast<u32x2_any*>(p) = v;
  } else {
    const u32x4 v = {__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3])};
    *reinterpret_cast<u32x4_any*>(p) = v;
  }
}
// Two fragments of 16 columns side by side: lane group g (16 lanes) holds columns 4g .. 4g+3 of each.  Swapping
// the odd groups of the first for the even ones of the second gives group g columns 8 (g >> 1) .. +7 of
// fragment g & 1.  (Lanes 16 apart hold the same row: both are there or neither.)  Stores of 32 bytes a row
// instead of 64: 16384 x 3584 x 8192 224 us, so 214.
__device__ __forceinline__ void put8_of_two(uint8_t* p, const f32x4& d0, const f32x4& d1) {
  const auto lo = __builtin_amdgcn_permlane16_swap(pack_bf16x2(d0[0], d0[1]), pack_bf16x2(d1[0], d1[1]), false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(pack_bf16x2(d0[2], d0[3]), pack_bf16x2(d1[2], d1[3]), false, false);
  const u32x4 v = {lo[0], hi[0], lo[1], hi[1]};
  *reinterpret_cast<u32x4_any*>(p) = v;
}
// Columns n .. n+3 of row m, as far as they exist.
template <bool BF16>
__device__ __forceinline__ void store4(uint8_t* c, int64_t m, int64_t n, int64_t N, const f32x4& d) {
  const int64_t at = m * N + n;
  if (n + 4 <= N) {
    put4<BF16>(c + at * (BF16 ? 2 : 4), d);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) {
        if constexpr (BF16) reinterpret_cast<uint16_t*>(c)[at + e] = (uint16_t)f32_to_bf16_bits(d[e]);
        else reinterpret_cast<float*>(c)[at + e] = d[e];
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
  const int lane = threadIdx.x & 63;
  // in a scalar register: branches on it are scalar ones (a matrix instruction does not look at the
  // lanes' mask, so it must not stand under one)
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t n_unit0 = (int64_t)blockIdx.x * NG, m_unit0 = (int64_t)blockIdx.y * TG;
  // Uniform addresses (units past the last repeat it; their products are not stored) and a lane's
  // offset: the loads then need no address arithmetic per lane.
  const uint32_t code_at = lane * 16, scale_at = lane * 2;
  int64_t au[TG], bu[NG];
#pragma unroll
  for (int t = 0; t < TG; ++t) au[t] = m_unit0 + t < m_units ? m_unit0 + t : m_units - 1;
#pragma unroll
  for (int g = 0; g < NG; ++g) bu[g] = n_unit0 + g < n_units ? n_unit0 + g : n_units - 1;
  f32x4 acc[NG][TG];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int t = 0; t < TG; ++t) acc[g][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  struct Slab {
    i32x4 b[NG][2], a[TG][2];
    uint32_t bs[NG], as[TG];
  };
  auto load = [&](Slab& v, int64_t s) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint8_t* p = b_codes + (s * n_units + bu[g]) * kMxCodeBytes;
      v.b[g][0] = *reinterpret_cast<const i32x4*>(p + code_at);
      v.b[g][1] = *reinterpret_cast<const i32x4*>(p + 1024 + code_at);
      v.bs[g] = *reinterpret_cast<const uint16_t*>(b_scales + (s * n_units + bu[g]) * kMxScaleBytes + scale_at);
    }
#pragma unroll
    for (int t = 0; t < TG; ++t) {
      const uint8_t* p = a_codes + (s * m_units + au[t]) * kMxCodeBytes;
      v.a[t][0] = *reinterpret_cast<const i32x4*>(p + code_at);
      v.a[t][1] = *reinterpret_cast<const i32x4*>(p + 1024 + code_at);
      v.as[t] = *reinterpret_cast<const uint16_t*>(a_scales + (s * m_units + au[t]) * kMxScaleBytes + scale_at);
    }
  };
  auto multiply = [&](const Slab& v) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int t = 0; t < TG; ++t) acc[g][t] = mfma_mx<0>(v.b[g][0], v.a[t][0], acc[g][t], v.bs[g], v.as[t]);
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int t = 0; t < TG; ++t) acc[g][t] = mfma_mx<1>(v.b[g][1], v.a[t][1], acc[g][t], v.bs[g], v.as[t]);
  };
  // (a second and third slab in flight per wave gained nothing: with eight waves the loads of one fill
  // the path to the compute unit)
  for (int64_t s = wave; s < slabs; s += WAVES) {
    Slab v;
    load(v, s);
    multiply(v);
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

// The same for the product of a few rows that are still bf16 or fp32 (generation: one launch instead
// of two, and no operand written and read back).  Every workgroup quantises all of them into LDS, a
// block of 32 per thread - its share of B is on the way meanwhile - and goes on as above; the lanes of
// rows that do not exist repeat the last one.
template <bool BF16, bool XBF16, int NG, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void mxfp4_matmul_rows_kernel(
    const uint8_t* __restrict__ x, int64_t row_bytes, const uint8_t* __restrict__ b_codes,
    const uint8_t* __restrict__ b_scales, uint8_t* __restrict__ c, int M, int64_t N, int64_t K, int slabs,
    int64_t n_units) {
  extern __shared__ __attribute__((aligned(16))) uint8_t rows_lds[];
  __shared__ f32x4 part[WAVES][NG][64];
  // codes [slabs * 8 blocks][M][16 B], then scales [slabs][4][M][2 steps]
  i32x4* codes = reinterpret_cast<i32x4*>(rows_lds);
  uint8_t* scales = rows_lds + (size_t)slabs * 8 * M * 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t n_unit0 = (int64_t)blockIdx.x * NG;
  const uint32_t code_at = lane * 16, scale_at = lane * 2;
  int64_t bu[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) bu[g] = n_unit0 + g < n_units ? n_unit0 + g : n_units - 1;
  struct Slab {
    i32x4 b[NG][2];
    uint32_t bs[NG];
  };
  auto load = [&](Slab& v, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint8_t* p = b_codes + (s * n_units + bu[g]) * kMxCodeBytes;
      v.b[g][0] = *reinterpret_cast<const i32x4*>(p + code_at);
      v.b[g][1] = *reinterpret_cast<const i32x4*>(p + 1024 + code_at);
      v.bs[g] = *reinterpret_cast<const uint16_t*>(b_scales + (s * n_units + bu[g]) * kMxScaleBytes + scale_at);
    }
  };
  Slab next;
  load(next, wave < slabs ? wave : slabs - 1);

  const int blocks = slabs * 8;
  for (int i = threadIdx.x; i < blocks * M; i += WAVES * 64) {
    const int r = i / blocks, b = i - r * blocks;
    const uint8_t* p = x + r * row_bytes + (int64_t)b * 32 * Mx8<XBF16>::kSize;
    const int64_t left = K - (int64_t)b * 32;
    Mx8<XBF16> v[4];
    if (left >= 32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j].load(p + j * 8 * Mx8<XBF16>::kSize);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j].load(p + j * 8 * Mx8<XBF16>::kSize, left - j * 8);
    }
    const uint32_t code = mx_scale_code(mx_top<XBF16>(v));
    const float scale = mx_scale_value(code);
    i32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = code == 255u ? 0 : (int)mx_pack8<XBF16>(v[j], scale);
    codes[b * M + r] = w;
    scales[((((b >> 3) * 4 + (b & 3)) * M) + r) * 2 + ((b >> 2) & 1)] = (uint8_t)code;
  }
  __syncthreads();

  f32x4 acc[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) acc[g] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int row = (lane & 15) < M ? (lane & 15) : M - 1;
  for (int s = wave; s < slabs; s += WAVES) {
    const Slab v = next;
    load(next, s + WAVES < slabs ? s + WAVES : s);
    const i32x4 a0 = codes[(s * 8 + (lane >> 4)) * M + row], a1 = codes[(s * 8 + 4 + (lane >> 4)) * M + row];
    const uint32_t as = *reinterpret_cast<const uint16_t*>(scales + ((s * 4 + (lane >> 4)) * M + row) * 2);
#pragma unroll
    for (int g = 0; g < NG; ++g) acc[g] = mfma_mx<0>(v.b[g][0], a0, acc[g], v.bs[g], as);
#pragma unroll
    for (int g = 0; g < NG; ++g) acc[g] = mfma_mx<1>(v.b[g][1], a1, acc[g], v.bs[g], as);
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) part[wave][g][lane] = acc[g];
  __syncthreads();
  for (int g = wave; g < NG; g += WAVES) {
    f32x4 d = part[0][g][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const f32x4 p = part[w][g][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] += p[e];
    }
    const int64_t n = (n_unit0 + g) * kMxRows + (lane >> 4) * 4;
    if ((lane & 15) < M && n < N) store4<BF16>(c, lane & 15, n, N, d);
  }
}

// ---------------------------------------------------------------------------
// The tiled kernel, for products with enough rows to fill matrix tiles: a persistent grid of
// 256-thread workgroups, one per compute unit, each computing BM x BN tiles with 4 waves in a
// 2 x 2 arrangement.  A slab (rows x 256 of K, 128 bytes a row) comes from memory straight into
// LDS with 128-bit direct-to-LDS loads; operands being in MFMA order, loads and fragment reads
// are both linear.  LDS holds three slabs of A (of a 256 x 256 tile two), two of B and two sets of
// scales: while one pair of slabs is multiplied, the next is complete or landing and the A slab
// after that is on its way.  With the bf16 MFMA replaced by one that does four times the work on the same bytes in
// the same time, the bytes per cycle are those of the bf16 GEMM of ag_matmul.hip, and so is the
// order of work inside a slab pair (two steps of 128 of K):
//   first step    MFMAs of step 0; the fragments of step 1 are read; A slab kt+2 is requested
//   barrier       pair kt is read by everyone, pair kt+1 has landed
//   second step   MFMAs of step 1; fragments of step 0 and the scales of pair kt+1 are read;
//                 B slab and scales of pair kt+2 (and its A slab where LDS holds two) are requested
// 16384 x 3584 x 8192: 201-205 us, 4.7-4.8 PFLOP/s.  Nothing but its MFMAs on such data takes 149 us (6.5 PFLOP/s: the
// clock is power-limited; zeros reach 8.9).  With 32 bytes a row per store it took 224: 187 without the stores, 190
// without the loads from memory, 178 without those and the fragment reads.  Stores that stay in flight under the next
// tile's first slabs, and 128 bytes a row per store, were no faster than 64.
typedef __attribute__((address_space(3))) void LdsVoid;

constexpr int kTileThreads = 256;

__device__ __forceinline__ i32x4 lds_frag(uint32_t addr) {
  return *reinterpret_cast<__attribute__((address_space(3))) const i32x4*>((uintptr_t)addr);
}
// (32 bits wide from the load on: the compiler would widen a 16-bit value in front of the MFMA that takes it, and an
// MFMA in assembly has to be two wait states behind a vector instruction that writes one of its operands)
__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
  return *reinterpret_cast<__attribute__((address_space(3))) const uint16_t*>((uintptr_t)addr);
}
// A pointer that is the same in every lane, kept in scalar registers.
__device__ __forceinline__ const uint8_t* uniform_ptr(const uint8_t* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}
// 1 KiB from memory to LDS: lane l's 16 bytes at base + voff land at lds_dst + 16 l.  In assembly so that the
// compiler does not count it: it would make every fragment read wait for it.  All waits for these
// loads are the explicit vmcnt below (loads return in order).
__device__ __forceinline__ void load_kib(const uint8_t* base, uint32_t voff, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds_dst), "v"(voff), "s"(base)
               : "memory", "m0");
}
// D += A x B with the accumulator named as an accumulation register, so that the compiler does not
// move the accumulators between the register files inside the loop.  STEP picks the byte of the
// scale registers.
template <int STEP>
__device__ __forceinline__ void mfma_mx_acc(f32x4& acc, const i32x4& first, const i32x4& second, uint32_t first_scale,
                                            uint32_t second_scale) {
  if constexpr (STEP == 0)
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                 : "+a"(acc)
                 : "v"(first), "v"(second), "v"(first_scale), "v"(second_scale));
  else
    asm volatile(
        "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
        : "+a"(acc)
        : "v"(first), "v"(second), "v"(first_scale), "v"(second_scale));
}
// The same with a load_kib behind it.  With one wave per SIMD an instruction between two MFMAs costs
// an issue slot, and an MFMA lasts four of them: the write of M0 stands ahead of the MFMA, which is
// the distance the load needs from it.
template <int STEP, int OFFSET>
__device__ __forceinline__ void mfma_mx_load(f32x4& acc, const i32x4& first, const i32x4& second, uint32_t first_scale,
                                             uint32_t second_scale, const uint8_t* base, uint32_t voff,
                                             uint32_t lds_dst) {
  if constexpr (STEP == 0)
    asm volatile(
        "s_add_i32 m0, %5, %6\n\t"
        "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t"
        "global_load_lds_dwordx4 %7, %8"
        : "+a"(acc)
        : "v"(first), "v"(second), "v"(first_scale), "v"(second_scale), "s"(lds_dst), "i"(OFFSET), "v"(voff), "s"(base)
        : "memory", "m0", "scc");
  else
    asm volatile(
        "s_add_i32 m0, %5, %6\n\t"
        "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t"
        "global_load_lds_dwordx4 %7, %8"
        : "+a"(acc)
        : "v"(first), "v"(second), "v"(first_scale), "v"(second_scale), "s"(lds_dst), "i"(OFFSET), "v"(voff), "s"(base)
        : "memory", "m0", "scc");
}

// Where the other instructions of a step go: every LOAD_GAP-th of the first MFMAs carries a load, and
// `reads` LDS reads are spread over the MFMAs in between among the first SPAN, one each.
// The read behind MFMA `at` (the MFMA-th slot), or -1.
template <int LOADS, int LOAD_GAP, int READS, int SPAN>
struct StepPlan {
  static constexpr bool is_load(int at) { return at % LOAD_GAP == 0 && at / LOAD_GAP < LOADS; }
  static constexpr int free_before(int at) {
    int n = 0;
    for (int i = 0; i < at; ++i) n += !is_load(i);
    return n;
  }
  static constexpr int kFree = free_before(SPAN);
  // reads first .. last - 1 go behind MFMA `at`
  static constexpr int first(int at) {
    if constexpr (kFree == 0) return at == 0 ? 0 : READS;         // (tiles of a few MFMAs)
    else return at >= SPAN ? READS : (free_before(at) * READS + kFree - 1) / kFree;
  }
};
template <int I>
struct Index {
  static constexpr int value = I;
};
// f(Index<0>), ..., f(Index<N - 1>): a loop whose counter is a constant in every turn
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(Index<I>{});
    unrolled<N, I + 1>(f);
  }
}

struct MxTiles {
  const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
  uint8_t* c;
  int64_t M, N;
  int slabs, m_units, n_units;
  int tiles_m, tiles_n, group_m;
};

// Tile number `lin` of the order: groups of group_m row tiles, column by column inside a group.
__device__ __forceinline__ void mx_tile_at(const MxTiles& t, int lin, int& tile_m, int& tile_n) {
  const int per_group = t.group_m * t.tiles_n;
  const int first = lin / per_group * t.group_m;
  const int rows = t.tiles_m - first < t.group_m ? t.tiles_m - first : t.group_m;
  const int in_group = lin % per_group;
  tile_m = first + in_group % rows;
  tile_n = in_group / rows;
}

// The tile of workgroup `wg` in pass `pass` over the grid, -1 if it has none: within a pass XCD x
// (workgroups with wg % 8 == x) takes a contiguous run of the tile order, a patch about as wide
// as it is high, so that the workgroups that share an L2 share rows of A and B.
__device__ __forceinline__ int mx_tile_number(int total, int grid, int wg, int pass) {
  const int64_t start = (int64_t)pass * grid;
  if (start >= total) return -1;
  const int count = total - start < grid ? (int)(total - start) : grid;
  const int per_xcd = (count + 7) >> 3;
  const int at = (wg & 7) * per_xcd + (wg >> 3);
  return (wg >> 3) < per_xcd && at < count ? (int)start + at : -1;
}

// A fragment's value where it is used.  IN_ACC: it lies in accumulation registers; left to itself the compiler
// copies all of a tile to vector registers ahead of the stores (16384 x 8192 x 8192 495 us, so 483; 4096 x 4096 x
// 4096 52.5 and 50), and a 256 x 256 tile to scratch memory.
template <bool IN_ACC>
__device__ __forceinline__ f32x4 fetched(const f32x4& acc) {
  if constexpr (!IN_ACC) return acc;
  f32x4 d;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float f;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(f) : "a"(acc[e]));
    d[e] = f;
  }
  return d;
}

// A wave's FM x FN fragments to rows m0.., columns n0.. of C.
template <bool BF16, int FM, int FN, bool IN_ACC>
__device__ __forceinline__ void store_tile(const MxTiles& p, int64_t m0, int64_t n0, int lane, const f32x4 (&acc)[FN][FM]) {
  constexpr int kSize = BF16 ? 2 : 4;
  const int64_t m_lane = m0 + (lane & 15), n_lane = n0 + (lane >> 4) * 4;
  if (n0 + FN * 16 <= p.N) {
    // all columns exist: one address per row of fragments, the columns are immediate offsets
    uint8_t* out = p.c + (m_lane * p.N + n_lane) * kSize;
    const int g = lane >> 4, shift = ((g & 1) * 16 + (g >> 1) * 8 - g * 4) * kSize;
#pragma unroll
    for (int mi = 0; mi < FM; ++mi) {
      if (m_lane + mi * 16 < p.M) {
        if constexpr (BF16) {
#pragma unroll
          for (int ni = 0; ni + 1 < FN; ni += 2) put8_of_two(out + shift + ni * 16 * kSize, fetched<IN_ACC>(acc[ni][mi]), fetched<IN_ACC>(acc[ni + 1][mi]));
          if constexpr (FN & 1) put4<BF16>(out + (FN - 1) * 16 * kSize, fetched<IN_ACC>(acc[FN - 1][mi]));
        } else {
#pragma unroll
          for (int ni = 0; ni < FN; ++ni) put4<BF16>(out + ni * 16 * kSize, fetched<IN_ACC>(acc[ni][mi]));
        }
      }
      out += p.N * (16 * kSize);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
#pragma unroll
    for (int mi = 0; mi < FM; ++mi) {
#pragma unroll
      for (int ni = 0; ni < FN; ++ni)
        if (m_lane + mi * 16 < p.M && n_lane + ni * 16 < p.N)
          store4<BF16>(p.c, m_lane + mi * 16, n_lane + ni * 16, p.N, fetched<IN_ACC>(acc[ni][mi]));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <bool BF16, int BM, int BN>
__global__ __launch_bounds__(kTileThreads, 1) void mxfp4_matmul_tile_kernel(MxTiles p) {
  constexpr int FM = BM / 32, FN = BN / 32;             // 16 x 16 fragments per wave, either way
  constexpr int GA = BM / 32, GB = BN / 32;             // 1 KiB loads per wave and slab
  constexpr int kA = BM * 128, kB = BN * 128;           // bytes of a slab
  constexpr int SA = (BM / 16 + 7) / 8, SB = (BN / 16 + 7) / 8;        // 1 KiB loads of scales (8 units each)
  constexpr int kS = (SA + SB) * 1024;
  // a third slab of A where LDS has room for it
  constexpr bool kDeep = 3 * kA + 2 * kB + 2 * kS <= 160 * 1024;
  constexpr int kOffB = (kDeep ? 3 : 2) * kA, kOffS = kOffB + 2 * kB;
  static_assert(SA + SB <= 4, "one load of scales per wave");
  static_assert(kOffS + 2 * kS <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kOffS + 2 * kS];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LdsVoid*)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = wave >> 1, wn = wave & 1;
  const int nk = p.slabs;
  // from one slab of an operand to the next
  const int64_t a_step = (int64_t)p.m_units * kMxCodeBytes, b_step = (int64_t)p.n_units * kMxCodeBytes;
  const int total = p.tiles_m * p.tiles_n;

  const uint8_t *a_base, *b_base, *s_base;
  uint32_t a_off[GA], b_off[GB], s_off;
  // Addresses of a tile's loads.  Units past the last repeat it: they feed results nobody stores.
  auto aim = [&](int tile_m, int tile_n) {
    const int mu = tile_m * (BM / 16), nu = tile_n * (BN / 16);
    a_base = uniform_ptr(p.a_codes + (int64_t)mu * kMxCodeBytes);
    b_base = uniform_ptr(p.b_codes + (int64_t)nu * kMxCodeBytes);
    const int a_last = p.m_units - 1 - mu, b_last = p.n_units - 1 - nu;
    int ln = lane;
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int j = 0; j < GA; ++j) {
      const int q = wave * GA + j, u = (q >> 1) < a_last ? (q >> 1) : a_last;
      a_off[j] = (uint32_t)u * kMxCodeBytes + (uint32_t)((q & 1) * 1024 + ln * 16);
    }
#pragma unroll
    for (int j = 0; j < GB; ++j) {
      const int q = wave * GB + j, u = (q >> 1) < b_last ? (q >> 1) : b_last;
      b_off[j] = (uint32_t)u * kMxCodeBytes + (uint32_t)((q & 1) * 1024 + ln * 16);
    }
    const int g = wave % (SA + SB);
    if (g < SA) {
      s_base = uniform_ptr(p.a_scales + (int64_t)mu * kMxScaleBytes);
      const int u = g * 8 + (ln >> 3);
      s_off = (uint32_t)(u < a_last ? u : a_last) * kMxScaleBytes + (uint32_t)(ln & 7) * 16;
    } else {
      s_base = uniform_ptr(p.b_scales + (int64_t)nu * kMxScaleBytes);
      const int u = (g - SA) * 8 + (ln >> 3);
      s_off = (uint32_t)(u < b_last ? u : b_last) * kMxScaleBytes + (uint32_t)(ln & 7) * 16;
    }
  };
  const int64_t s_step = (int64_t)(wave % (SA + SB) < SA ? p.m_units : p.n_units) * kMxScaleBytes;
  const uint32_t s_dst = lds0 + kOffS + (uint32_t)(wave % (SA + SB)) * 1024;
  auto prologue = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = i < nk ? i : nk - 1;
#pragma unroll
      for (int j = 0; j < GA; ++j)
        load_kib(a_base + k * a_step, a_off[j], lds0 + i * kA + (wave * GA + j) * 1024);
#pragma unroll
      for (int j = 0; j < GB; ++j)
        load_kib(b_base + k * b_step, b_off[j], lds0 + kOffB + i * kB + (wave * GB + j) * 1024);
      load_kib(s_base + k * s_step, s_off, s_dst + i * kS);
    }
  };

  int pass = 0, number = mx_tile_number(total, gridDim.x, blockIdx.x, 0);
  if (number < 0) return;
  int tile_m, tile_n;
  mx_tile_at(p, number, tile_m, tile_n);
  aim(tile_m, tile_n);
  prologue();
  for (;;) {
    f32x4 acc[FN][FM];
#pragma unroll
    for (int ni = 0; ni < FN; ++ni)
#pragma unroll
      for (int mi = 0; mi < FM; ++mi) acc[ni][mi] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // (loads and the previous tile's stores do not retire in one order: wait for everything)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();

    int ln = lane;
    asm volatile("" : "+v"(ln));
    uint32_t a_fr = lds0 + (uint32_t)(wm * FM * 2048 + ln * 16);
    uint32_t b_fr = lds0 + kOffB + (uint32_t)(wn * FN * 2048 + ln * 16);
    uint32_t sa_fr = lds0 + kOffS + (uint32_t)(wm * FM * 128 + ln * 2);
    uint32_t sb_fr = lds0 + kOffS + SA * 1024 + (uint32_t)(wn * FN * 128 + ln * 2);
    i32x4 af0[FM], bf0[FN], af1[FM], bf1[FN];
    uint32_t sa[2][FM], sb[2][FN];               // by parity of the slab pair
#pragma unroll
    for (int f = 0; f < FM; ++f) af0[f] = lds_frag(a_fr + f * 2048);
#pragma unroll
    for (int f = 0; f < FN; ++f) bf0[f] = lds_frag(b_fr + f * 2048);
#pragma unroll
    for (int f = 0; f < FM; ++f) sa[0][f] = lds_u16(sa_fr + f * 128);
#pragma unroll
    for (int f = 0; f < FN; ++f) sb[0][f] = lds_u16(sb_fr + f * 128);

    // What the trip requests: slab kt + 2, the last one again past the end (into places nobody reads
    // any more; one code path keeps the accumulators in place).
    const uint8_t* ap = a_base + (2 < nk ? 2 : nk - 1) * a_step;
    const uint8_t* bp = b_base + (2 < nk ? 2 : nk - 1) * b_step;
    const uint8_t* sp = s_base + (2 < nk ? 2 : nk - 1) * s_step;
    uint32_t a_at = 0;                           // offset of A slab kt in its ring of three
    uint32_t a_to = lds0 + (kDeep ? 2 * kA : 0) + wave * (GA * 1024);        // where A slab kt + 2 goes

    constexpr int kMfma = FM * FN, kFrags = FM + FN;
    using Plan0 = StepPlan<kDeep ? GA : 0, kMfma / GA, kFrags, kMfma * 13 / 16>;
    constexpr int kLoads1 = GB + 1 + (kDeep ? 0 : GA), kGap1 = kDeep ? (kMfma / 2) / GB : (kMfma * 3 / 4) / kLoads1;
    using Plan1 = StepPlan<kLoads1, kGap1, 2 * kFrags, kMfma * 15 / 16>;
    // (the last load of the first step stands at (GA - 1) * (kMfma / GA))
    constexpr bool kRoom = kMfma - 6 >= kMfma * 13 / 16 && kMfma - 6 > (GA - 1) * (kMfma / GA);
    constexpr int kBook = kRoom ? kMfma - 6 : kMfma - 1, kBookGap = kRoom ? 1 : 0;
    auto trip = [&](auto parity, int kt) __attribute__((always_inline)) {
      constexpr int P = decltype(parity)::value;
      unrolled<kMfma>([&](auto slot) __attribute__((always_inline)) {
        constexpr int at = decltype(slot)::value, ni = at / FM, mi = at % FM, g = at / (kMfma / GA);
        if constexpr (Plan0::is_load(at))
          mfma_mx_load<0, g * 1024>(acc[ni][mi], bf0[ni], af0[mi], sb[P][ni], sa[P][mi], ap, a_off[g], a_to);
        else
          mfma_mx_acc<0>(acc[ni][mi], bf0[ni], af0[mi], sb[P][ni], sa[P][mi]);
        constexpr int r0 = Plan0::first(at), r1 = Plan0::first(at + 1);
        unrolled<r1 - r0>([&](auto read) __attribute__((always_inline)) {
          constexpr int r = r0 + decltype(read)::value;
          if constexpr (r == 0) bf1[0] = lds_frag(b_fr + 1024);
          else if constexpr (r <= FM) af1[r - 1] = lds_frag(a_fr + 1024 + (r - 1) * 2048);
          else bf1[r - FM] = lds_frag(b_fr + 1024 + (r - FM) * 2048);
        });
        // the uniform bookkeeping goes between the last MFMAs, behind the step's loads and reads
        if constexpr (at == kBook && kDeep) {
          const uint32_t next = a_at == 2 * kA ? 0 : a_at + kA;
          a_fr += next - a_at;
          a_at = next;
        }
        if constexpr (at == kBook && !kDeep) a_fr += P == 0 ? (uint32_t)kA : (uint32_t)-kA;
        if constexpr (at == kBook + kBookGap && kDeep) a_to = lds0 + wave * (GA * 1024) + (a_at >= kA ? a_at - kA : 2 * kA);
        if constexpr (at == kBook + 2 * kBookGap) b_fr += P == 0 ? (uint32_t)kB : (uint32_t)-kB;
        if constexpr (at == kBook + 3 * kBookGap) {
          sa_fr += P == 0 ? (uint32_t)kS : (uint32_t)-kS;
          sb_fr += P == 0 ? (uint32_t)kS : (uint32_t)-kS;
        }
        if constexpr (at == kBook + 4 * kBookGap && kDeep) ap += kt + 3 < nk ? a_step : 0;
        __builtin_amdgcn_sched_barrier(0);
      });
      // this wave's loads of pair kt+1 are complete; those of A slab kt+2, if any yet, may be in flight
      static_assert(GA == 8 || GA == 4 || GA == 2, "explicit vmcnt below");
      if constexpr (!kDeep) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else if constexpr (GA == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      else if constexpr (GA == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
      __syncthreads();
      unrolled<kMfma>([&](auto slot) __attribute__((always_inline)) {
        constexpr int at = decltype(slot)::value, ni = at / FM, mi = at % FM, g = at / kGap1;
        if constexpr (Plan1::is_load(at) && g < GB)
          mfma_mx_load<1, g * 1024>(acc[ni][mi], bf1[ni], af1[mi], sb[P][ni], sa[P][mi], bp, b_off[g < GB ? g : 0],
                                    lds0 + kOffB + P * kB + wave * (GB * 1024));
        else if constexpr (Plan1::is_load(at) && g < kLoads1 - 1)
          mfma_mx_load<1, P * kA + (g - GB) * 1024>(acc[ni][mi], bf1[ni], af1[mi], sb[P][ni], sa[P][mi], ap,
                                                    a_off[g - GB < GA && g >= GB ? g - GB : 0], a_to);
        else if constexpr (Plan1::is_load(at))
          mfma_mx_load<1, P * kS>(acc[ni][mi], bf1[ni], af1[mi], sb[P][ni], sa[P][mi], sp, s_off, s_dst);
        else
          mfma_mx_acc<1>(acc[ni][mi], bf1[ni], af1[mi], sb[P][ni], sa[P][mi]);
        // pair kt+1: fragment and scale of B row 0, those of A, the other B rows
        constexpr int r0 = Plan1::first(at), r1 = Plan1::first(at + 1);
        unrolled<r1 - r0>([&](auto read) __attribute__((always_inline)) {
          constexpr int r = r0 + decltype(read)::value, f = r >> 1;
          if constexpr ((r & 1) == 0) {
            if constexpr (f == 0) bf0[0] = lds_frag(b_fr);
            else if constexpr (f <= FM) af0[f - 1] = lds_frag(a_fr + (f - 1) * 2048);
            else bf0[f - FM] = lds_frag(b_fr + (f - FM) * 2048);
          } else {
            if constexpr (f == 0) sb[1 - P][0] = lds_u16(sb_fr);
            else if constexpr (f <= FM) sa[1 - P][f - 1] = lds_u16(sa_fr + (f - 1) * 128);
            else sb[1 - P][f - FM] = lds_u16(sb_fr + (f - FM) * 128);
          }
        });
        if constexpr (at == kMfma - 4 && !kDeep) ap += kt + 3 < nk ? a_step : 0;
        if constexpr (at == kMfma - 3) bp += kt + 3 < nk ? b_step : 0;
        if constexpr (at == kMfma - 2) sp += kt + 3 < nk ? s_step : 0;
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    // two trips per turn of the loop, one for each set of scales; an odd last trip stands behind it
    int kt = 0;
    for (; kt + 1 < nk; kt += 2) {
      trip(Index<0>{}, kt);
      trip(Index<1>{}, kt + 1);
    }
    if (kt < nk) trip(Index<0>{}, kt);
    // The repeated loads of the last steps must not land on top of the next tile's slabs, and the
    // last MFMAs (assembly the compiler does not time) must be through before their results are read.
    asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");
    __syncthreads();
    const int64_t m0 = (int64_t)tile_m * BM + wm * (BM / 2), n0 = (int64_t)tile_n * BN + wn * (BN / 2);
    number = mx_tile_number(total, gridDim.x, blockIdx.x, ++pass);
    if (number >= 0) {
      mx_tile_at(p, number, tile_m, tile_n);
      aim(tile_m, tile_n);
      prologue();
    }
    int le = lane;
    asm volatile("" : "+v"(le));
    store_tile<BF16, FM, FN, true>(p, m0, n0, le, acc);
    if (number < 0) return;
  }
}

// ---------------------------------------------------------------------------
// The same product in smaller tiles, for results that have too few of the large ones to fill the
// chip.  What bounds those is the arrival of the slabs - first the latency, then the 62 bytes/ns that a compute
// unit takes in, four fifths of them L2 hits (64 x 128: 26 KB per slab pair in 0.42 us) - so LDS holds BUFFERS whole
// slab pairs and all but the two being multiplied and read are on their way; the order inside a pair is the compiler's.
// Three: two workgroups
// fit a compute unit (1500 x 3500 x 1100: 11.9 us, with four 14.6), and alone four to six are no faster (1001 x
// 1777 x 4000: 11.8, 12.0, 12.3, 12.4), nor is a second group of waves that takes every other slab (12.2).
// One tile per workgroup.
template <bool BF16, int BM, int BN, int BUFFERS>
__global__ __launch_bounds__(kTileThreads) void mxfp4_matmul_ring_kernel(MxTiles p) {
  constexpr int FM = BM / 32, FN = BN / 32;
  constexpr int GA = BM / 32, GB = BN / 32;
  constexpr int SA = (BM / 16 + 7) / 8, SB = (BN / 16 + 7) / 8;
  constexpr int kA = BM * 128, kB = BN * 128, kPair = kA + kB + (SA + SB) * 1024;
  constexpr int kInFlight = (BUFFERS - 2) * (GA + GB + 1);
  static_assert(SA + SB <= 4 && BUFFERS * kPair <= 160 * 1024 && (BUFFERS - 1) * (GA + GB + 1) < 64, "LDS, loads in flight");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[BUFFERS * kPair];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LdsVoid*)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = wave >> 1, wn = wave & 1;
  const int nk = p.slabs;
  const int number = mx_tile_number(p.tiles_m * p.tiles_n, gridDim.x, blockIdx.x, 0);
  if (number < 0) return;
  int tile_m, tile_n;
  mx_tile_at(p, number, tile_m, tile_n);
  const int mu = tile_m * (BM / 16), nu = tile_n * (BN / 16);
  const int a_last = p.m_units - 1 - mu, b_last = p.n_units - 1 - nu;

  const int64_t a_step = (int64_t)p.m_units * kMxCodeBytes, b_step = (int64_t)p.n_units * kMxCodeBytes;
  const uint8_t* ap = uniform_ptr(p.a_codes + (int64_t)mu * kMxCodeBytes);
  const uint8_t* bp = uniform_ptr(p.b_codes + (int64_t)nu * kMxCodeBytes);
  uint32_t a_off[GA], b_off[GB], s_off;
#pragma unroll
  for (int j = 0; j < GA; ++j) {
    const int q = wave * GA + j, u = (q >> 1) < a_last ? (q >> 1) : a_last;
    a_off[j] = (uint32_t)u * kMxCodeBytes + (uint32_t)((q & 1) * 1024 + lane * 16);
  }
#pragma unroll
  for (int j = 0; j < GB; ++j) {
    const int q = wave * GB + j, u = (q >> 1) < b_last ? (q >> 1) : b_last;
    b_off[j] = (uint32_t)u * kMxCodeBytes + (uint32_t)((q & 1) * 1024 + lane * 16);
  }
  const int g = wave % (SA + SB);                    // (waves past the last piece of scales repeat one)
  const bool of_a = g < SA;
  const uint8_t* sp = uniform_ptr(of_a ? p.a_scales + (int64_t)mu * kMxScaleBytes : p.b_scales + (int64_t)nu * kMxScaleBytes);
  const int64_t s_step = (int64_t)(of_a ? p.m_units : p.n_units) * kMxScaleBytes;
  {
    const int u = (of_a ? g : g - SA) * 8 + (lane >> 3), last = of_a ? a_last : b_last;
    s_off = (uint32_t)(u < last ? u : last) * kMxScaleBytes + (uint32_t)(lane & 7) * 16;
  }
  int loaded = 0;                                    // next pair to request; past the end the last one again
  auto request = [&](uint32_t at) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < GA; ++j) load_kib(ap, a_off[j], at + (wave * GA + j) * 1024);
#pragma unroll
    for (int j = 0; j < GB; ++j) load_kib(bp, b_off[j], at + kA + (wave * GB + j) * 1024);
    load_kib(sp, s_off, at + kA + kB + g * 1024);
    if (++loaded < nk) {
      ap += a_step;
      bp += b_step;
      sp += s_step;
    }
  };
#pragma unroll
  for (int b = 0; b < BUFFERS; ++b) request(lds0 + b * kPair);

  f32x4 acc[FN][FM];
#pragma unroll
  for (int ni = 0; ni < FN; ++ni)
#pragma unroll
    for (int mi = 0; mi < FM; ++mi) acc[ni][mi] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // Fragments are read a pair ahead, into the other of two register sets.
  struct Frags {
    i32x4 a[2][FM], b[2][FN];
    uint16_t sa[FM], sb[FN];
  };
  auto read = [&](Frags& v, uint32_t at) __attribute__((always_inline)) {
    const uint32_t a_fr = at + (uint32_t)(wm * FM * 2048 + lane * 16);
    const uint32_t b_fr = at + kA + (uint32_t)(wn * FN * 2048 + lane * 16);
    const uint32_t sa_fr = at + kA + kB + (uint32_t)(wm * FM * 128 + lane * 2);
    const uint32_t sb_fr = at + kA + kB + SA * 1024 + (uint32_t)(wn * FN * 128 + lane * 2);
#pragma unroll
    for (int f = 0; f < FM; ++f) v.sa[f] = lds_u16(sa_fr + f * 128);
#pragma unroll
    for (int f = 0; f < FN; ++f) v.sb[f] = lds_u16(sb_fr + f * 128);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
#pragma unroll
      for (int f = 0; f < FM; ++f) v.a[step][f] = lds_frag(a_fr + step * 1024 + f * 2048);
#pragma unroll
      for (int f = 0; f < FN; ++f) v.b[step][f] = lds_frag(b_fr + step * 1024 + f * 2048);
    }
  };
  uint32_t here = lds0;                              // buffer of pair kt
  // One pair: its fragments are in `now`; pair kt + 1 goes to `then`, pair kt + BUFFERS into its place.
  auto turn = [&](const Frags& now, Frags& then) __attribute__((always_inline)) {
    // this wave's share of pair kt + 1 is there; behind the barrier everyone's is, and everyone has pair kt
    asm volatile("s_waitcnt vmcnt(%0)" : : "i"(kInFlight) : "memory");
    __syncthreads();
    request(here);
    here = here + kPair < lds0 + BUFFERS * kPair ? here + kPair : lds0;
    read(then, here);
#pragma unroll
    for (int ni = 0; ni < FN; ++ni)
#pragma unroll
      for (int mi = 0; mi < FM; ++mi)
        acc[ni][mi] = mfma_mx<0>(now.b[0][ni], now.a[0][mi], acc[ni][mi], now.sb[ni], now.sa[mi]);
#pragma unroll
    for (int ni = 0; ni < FN; ++ni)
#pragma unroll
      for (int mi = 0; mi < FM; ++mi)
        acc[ni][mi] = mfma_mx<1>(now.b[1][ni], now.a[1][mi], acc[ni][mi], now.sb[ni], now.sa[mi]);
  };
  Frags even, odd;
  asm volatile("s_waitcnt vmcnt(%0)" : : "i"((BUFFERS - 1) * (GA + GB + 1)) : "memory");
  __syncthreads();
  read(even, lds0);
  int kt = 0;
  for (; kt + 1 < nk; kt += 2) {
    turn(even, odd);
    turn(odd, even);
  }
  if (kt < nk) turn(even, odd);
  // (LDS is given back when the workgroup ends: nothing may still be landing in it)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  store_tile<BF16, FM, FN, false>(p, (int64_t)tile_m * BM + wm * (BM / 2), (int64_t)tile_n * BN + wn * (BN / 2), lane, acc);
}

struct MxOperands {
  const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
  uint8_t* c;
  int64_t M, N, K;
};

// The few-rows kernel's grid: groups of rows in y, groups of columns in x.
static bool few_fits(int64_t m_groups, int64_t n_groups) { return m_groups <= 65535 && n_groups <= kMxMaxGrid / 4; }

template <bool BF16, int TG, int NG, int WAVES>
static int launch_few(const MxOperands& o, hipStream_t s) {
  const int64_t m_units = mx_row_units(o.M), n_units = mx_row_units(o.N);
  const int64_t gx = (n_units + NG - 1) / NG, gy = (m_units + TG - 1) / TG;
  if (!few_fits(gy, gx)) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_matmul: too large for one launch");
  hipLaunchKernelGGL((mxfp4_matmul_few_kernel<BF16, TG, NG, WAVES>), dim3((unsigned)gx, (unsigned)gy),
                     dim3(WAVES * 64), 0, s, o.a_codes, o.a_scales, o.b_codes, o.b_scales, o.c, o.M, o.N,
                     mx_slabs(o.K), m_units, n_units);
  return check_hip(hipGetLastError(), "smr_mxfp4_matmul launch");
}

struct MxRows {
  const uint8_t* x;
  int64_t row_bytes;
  const uint8_t *b_codes, *b_scales;
  uint8_t* c;
  int64_t M, N, K;
};
// Rows times slabs of one launch: their codes and scales (136 B each) and 32 KiB of partial sums are half of a compute
// unit's LDS, so that two workgroups fit.  Quantising takes a workgroup longer the more there are, and with one
// workgroup per compute unit wide results wait for it; K = 8192, us of one launch / quantiser and product:
//   rows (units)   8 (256)        11 (352)       12 (384)       16 (512)
//   N =  3584     8.3 /  8.0     9.3 /  8.1     9.7 /  8.2    11.1 /  8.1
//   N =  8192    10.4 / 10.8    11.1 / 10.8    11.5 / 10.8    12.6 / 10.9
//   N = 28672    28.4 / 26.3    29.1 / 26.1    33.0 / 24.9    35.8 / 25.3
// Up to there the second launch would cost a caller on the host (4 us) more than one launch costs the GPU.
constexpr int kRowsLdsUnits = 352;
// Columns that one launch of four units of columns per workgroup takes.
constexpr int64_t kRowsMaxN = kMxMaxGrid / 4 * 4 * kMxRows;

template <bool BF16, bool XBF16, int NG, int WAVES>
static int launch_rows_as(const MxRows& o, hipStream_t s) {
  const int64_t n_units = mx_row_units(o.N), slabs = mx_slabs(o.K), grid = (n_units + NG - 1) / NG;
  hipLaunchKernelGGL((mxfp4_matmul_rows_kernel<BF16, XBF16, NG, WAVES>), dim3((unsigned)grid), dim3(WAVES * 64),
                     (size_t)(slabs * o.M * 136), s, o.x, o.row_bytes, o.b_codes, o.b_scales, o.c, (int)o.M, o.N, o.K,
                     (int)slabs, n_units);
  return check_hip(hipGetLastError(), "smr_mxfp4_matmul_rows launch");
}
template <bool BF16, bool XBF16>
static int launch_rows(const MxRows& o, hipStream_t s) {
  // Column units and waves per workgroup, K = 8192, us at M = 1 (M = 8):    1 x 8        2 x 16       4 x 8
  //   N =  3584                                                              5.7  (8.2)   6.3  (8.3)   7.2  (9.6)
  //   N =  8192                                                              8.3 (11.1)   8.4 (10.5)   8.8 (11.2)
  //   N = 28672                                                             25.4 (38.4)  26.1 (33.3)  24.4 (27.2)
  if (o.N <= 4096) return launch_rows_as<BF16, XBF16, 1, 8>(o, s);
  if (o.N <= 16384) return launch_rows_as<BF16, XBF16, 2, 16>(o, s);
  return launch_rows_as<BF16, XBF16, 4, 8>(o, s);
}

template <int BM, int BN>
static MxTiles tiles_of(const MxOperands& o) {
  MxTiles t = {o.a_codes, o.a_scales, o.b_codes, o.b_scales, o.c, o.M, o.N};
  t.slabs = (int)mx_slabs(o.K);
  t.m_units = (int)mx_row_units(o.M);
  t.n_units = (int)mx_row_units(o.N);
  t.tiles_m = (int)((o.M + BM - 1) / BM);
  t.tiles_n = (int)((o.N + BN - 1) / BN);
  t.group_m = 8;
  return t;
}

// Grids are multiples of 8, so that a workgroup's number says which XCD it is on.
constexpr int64_t kMxMaxTiles = kMxMaxGrid - 8;
template <bool BF16, int BM, int BN>
static int launch_tiles(const MxOperands& o, hipStream_t s) {
  const MxTiles t = tiles_of<BM, BN>(o);
  const int64_t total = (int64_t)t.tiles_m * t.tiles_n, cus = compute_units() / 8 * 8;
  if (total > kMxMaxTiles) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_matmul: too large for one launch");
  const int64_t grid = total < cus ? (total + 7) / 8 * 8 : cus;
  hipLaunchKernelGGL((mxfp4_matmul_tile_kernel<BF16, BM, BN>), dim3((unsigned)grid), dim3(kTileThreads), 0, s, t);
  return check_hip(hipGetLastError(), "smr_mxfp4_matmul launch");
}

template <bool BF16, int BM, int BN, int BUFFERS>
static int launch_ring(const MxOperands& o, hipStream_t s) {
  const MxTiles t = tiles_of<BM, BN>(o);
  const int64_t total = (int64_t)t.tiles_m * t.tiles_n;
  if (total > kMxMaxTiles) return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_matmul: too large for one launch");
  hipLaunchKernelGGL((mxfp4_matmul_ring_kernel<BF16, BM, BN, BUFFERS>), dim3((unsigned)((total + 7) / 8 * 8)),
                     dim3(kTileThreads), 0, s, t);
  return check_hip(hipGetLastError(), "smr_mxfp4_matmul launch");
}

// Which kernel: the one with the lowest estimate of its time in microseconds, fitted to launches on 256 compute
// units.  A launch costs a few microseconds to start and drain; a pass of the chip over one tile per compute unit
// costs its first loads and stores and so much per slab, a last one that is not full 0.6 of that and up, less the
// more passes went before it (the workgroups drift apart); the two kernels without a persistent grid are bound by
// latency while they fill the chip once.
//                     n slabs           M x 3584: us of few / 64x128 / 128x128 / 256x128 / 256x224 / 256x256
//   few    64 x 32    0.75 + 0.117 n     512, K = 8192:  20.5 / 17.9 / 20.0 / 25 / 37 / 45    K = 768:  6.6 /  5.1 /  6.0 /  7.9 / 11.3 / 12.0
//   ring   64 x 128   1.3  + 0.35  n    1024            33.5 / 25.9 / 21.8 / 26 / 38 / 46             10.9 /  7.2 /  6.7 /  8.7 / 12.0 / 12.6
//   tiles 128 x 128   2.7  + 0.53  n    2048            66   / 50   / 41   / 33 / 42 / 48             19.0 / 12.2 / 11.7 / 10.4 / 13.7 / 14.2
//   tiles 256 x 128   5.2  + 0.87  n    4096           130   / 91   / 80   / 63 / 54 / 57             34   / 19.7 / 19.5 / 16.8 / 15.2 / 15.7
//   tiles 256 x 224   8.8  + 1.34  n    8192                                                          66   / 35   / 31   / 29.7 / 28.0 / 27.0
//   tiles 256 x 256   9.7  + 1.54  n    (4096 x 4096 x 4096: 58 / 48 / 42 / 50 / 36.6 from 64x128 on; 8192 x 8192 x 8192: 405 / 350 / 278 / 250 / 242)
// A kernel whose grid cannot be launched is no candidate: narrow results are best off with the first at any height, but
// its groups of rows end at 65535.
enum MxKernel { kMxFew, kMxRing64x128, kMxTile128x128, kMxTile256x128, kMxTile256x224, kMxTile256x256 };

static MxKernel pick_kernel(int64_t M, int64_t N, int64_t slabs, int cus) {
  auto tiles = [&](int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  const bool fits[6] = {few_fits((M + 63) / 64, (N + 31) / 32), tiles(64, 128) <= kMxMaxTiles, tiles(128, 128) <= kMxMaxTiles,
                        tiles(256, 128) <= kMxMaxTiles, tiles(256, 224) <= kMxMaxTiles, tiles(256, 256) <= kMxMaxTiles};
  auto larger = [](double a, double b) { return a > b ? a : b; };
  auto passes = [&](int64_t bm, int64_t bn) {
    const double full = (double)(tiles(bm, bn) / cus), rest = (double)(tiles(bm, bn) % cus) / cus;
    return full + (rest > 0 ? larger(rest, 0.6 + 0.4 * rest - 0.06 * full) : 0.0);
  };
  const double n = (double)slabs;
  const double time[6] = {larger(3.3 + 0.157 * n, 3 + (double)tiles(64, 32) / cus * (0.75 + 0.117 * n)),
                          larger(3.8 + 0.42 * n, 2.5 + passes(64, 128) * (1.3 + 0.35 * n)),
                          2.4 + passes(128, 128) * (2.7 + 0.53 * n), 2.5 + passes(256, 128) * (5.2 + 0.87 * n),
                          2.3 + passes(256, 224) * (8.8 + 1.34 * n), 2.5 + passes(256, 256) * (9.7 + 1.54 * n)};
  int best = kMxTile256x256;                         // the fewest workgroups
  for (int k = kMxTile256x224; k >= kMxFew; --k)
    if (fits[k] && time[k] <= time[best]) best = k;
  return (MxKernel)best;
}

template <bool BF16>
static int launch_matmul(const MxOperands& o, hipStream_t s) {
  // Up to 64 rows B is read once and little else counts.  Times in us, K = 8192, units of columns per workgroup
  // of the few-rows kernel:
  //            N = 3584: one / two      8192: one / two      16384: one / two / ring     28672: two / four / ring
  //   M = 16   5.2 /                     8.0 /                12.6 /      /                    / 24.0 / 22.1
  //   M = 37   7.0 / 7.3                 9.8 / 8.4
  //   M = 64   7.3 / 8.3                11.1 / 9.1            18.3 / 14.7 / 16.1          36.9 / 33   / 23.7
  // Wide products do best with B through LDS, a single unit of rows from K = 2048 on (16 x 131072 x 2048: 28.3 us,
  // four units 31.7; 16 x 28672 x 1024: 6.1 and 5.4).
  const int64_t slabs = mx_slabs(o.K);
  const bool wide = o.N > 16384;
  if (o.M <= 16 && !wide) return launch_few<BF16, 1, 1, 8>(o, s);
  if (o.M <= 16 && slabs < 8 && o.N <= kRowsMaxN) return launch_few<BF16, 1, 4, 8>(o, s);
  if (o.M <= 64 && wide) return launch_ring<BF16, 64, 128, 3>(o, s);
  if (o.M <= 32) return o.N <= 4096 ? launch_few<BF16, 2, 1, 8>(o, s) : launch_few<BF16, 2, 2, 8>(o, s);
  if (o.M <= 48) return o.N <= 4096 ? launch_few<BF16, 3, 1, 8>(o, s) : launch_few<BF16, 3, 2, 8>(o, s);
  if (o.M <= 64) return o.N <= 4096 ? launch_few<BF16, 4, 1, 8>(o, s) : launch_few<BF16, 4, 2, 8>(o, s);
  switch (pick_kernel(o.M, o.N, slabs, compute_units())) {
    case kMxFew: return launch_few<BF16, 4, 2, 8>(o, s);
    case kMxRing64x128: return launch_ring<BF16, 64, 128, 3>(o, s);
    case kMxTile128x128: return launch_tiles<BF16, 128, 128>(o, s);
    case kMxTile256x128: return launch_tiles<BF16, 256, 128>(o, s);
    case kMxTile256x224: return launch_tiles<BF16, 256, 224>(o, s);
    default: return launch_tiles<BF16, 256, 256>(o, s);
  }
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

int64_t smr_mxfp4_matmul_rows_limit(int64_t K) {
  if (K < 1 || K >= smr::kMxMaxExtent) return SMR_E_INVALID;
  const int64_t rows = smr::kRowsLdsUnits / smr::mx_slabs(K);
  return rows < smr::kMxRows ? rows : smr::kMxRows;
}

int smr_mxfp4_matmul_rows(const void* x_dev, int64_t row_stride, int dtype, const void* b_codes_dev,
                          const void* b_scales_dev, void* c_dev, int64_t M, int64_t N, int64_t K, int out_dtype,
                          void* stream) {
  using namespace smr;
  if ((dtype != SMR_DTYPE_BF16 && dtype != SMR_DTYPE_FP32) || (out_dtype != SMR_DTYPE_BF16 && out_dtype != SMR_DTYPE_FP32))
    return fail(SMR_E_INVALID, "smr_mxfp4_matmul_rows: dtype and out_dtype must be bf16 (0) or fp32 (1)");
  if (M < 0 || N < 0 || K < 1 || N >= kMxMaxExtent || K >= kMxMaxExtent)
    return fail(SMR_E_INVALID, "smr_mxfp4_matmul_rows: N must be in 0..2^31-1, K in 1..2^31-1");
  if (M > smr_mxfp4_matmul_rows_limit(K))
    return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_matmul_rows: more rows than smr_mxfp4_matmul_rows_limit (quantise them first)");
  if (N > kRowsMaxN)
    return fail(SMR_E_UNSUPPORTED, "smr_mxfp4_matmul_rows: more than 2^28 - 64 columns (quantise the rows first)");
  if (M > 1 && row_stride < K) return fail(SMR_E_INVALID, "smr_mxfp4_matmul_rows: rows must not overlap (row_stride < K)");
  if (M == 0 || N == 0) return 0;
  if (x_dev == nullptr || b_codes_dev == nullptr || b_scales_dev == nullptr || c_dev == nullptr)
    return fail(SMR_E_INVALID, "smr_mxfp4_matmul_rows: NULL argument");
  const bool bf16 = dtype == SMR_DTYPE_BF16, out_bf16 = out_dtype == SMR_DTYPE_BF16;
  if (((reinterpret_cast<uintptr_t>(b_codes_dev) | reinterpret_cast<uintptr_t>(b_scales_dev)) & 15u) ||
      (reinterpret_cast<uintptr_t>(x_dev) & (bf16 ? 1u : 3u)) || (reinterpret_cast<uintptr_t>(c_dev) & (out_bf16 ? 1u : 3u)))
    return fail(SMR_E_INVALID, "smr_mxfp4_matmul_rows: misaligned argument (operand: 16 bytes, x and c: one element)");
  const MxRows o = {static_cast<const uint8_t*>(x_dev), row_stride * (bf16 ? 2 : 4), static_cast<const uint8_t*>(b_codes_dev),
                    static_cast<const uint8_t*>(b_scales_dev), static_cast<uint8_t*>(c_dev), M, N, K};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (bf16) return out_bf16 ? launch_rows<true, true>(o, s) : launch_rows<false, true>(o, s);
  return out_bf16 ? launch_rows<true, false>(o, s) : launch_rows<false, false>(o, s);
}

}  // extern "C"
