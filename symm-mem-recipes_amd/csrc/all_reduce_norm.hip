// The end of a tensor-parallel block in one pass over its partial sums: one-shot all-reduce, the
// norm behind the block, its gate, the scaled residual and the norm in front of the next block.
//
//   s = sum over the ranks of their partial sums            fp32, rank order, as one_shot_all_reduce
//   n = s * (mean(s^2) + eps)^-1/2 * post_weight            (n = s without a post_weight)
//   h = residual_scale * residual + gate * n                -> residual_out
//   y = h * (mean(h^2) + eps)^-1/2 * weight                 -> normed
//
// A row stays in its workgroup's registers from the sum to the stores, in fp32; each output is
// rounded once.  The bound is HBM: (world_size + 3) * cols elements per row.
//
// The backward pass, with D the whole gradient of h, r1 and r2 the two reciprocal roots:
//   D  = grad_residual_out + r2 * (dy*weight - h * r2^2 * mean(dy*weight*h)),  dy = grad_normed
//   residual: residual_scale * D          weight: sum over rows of dy * h * r2
//   gate: D * n, summed over what the gate was broadcast over
//   with dn = gate * D:  post_weight: sum over rows of dn * s * r1
//   partial: r1 * (dn*post_weight - s * r1^2 * mean(dn*post_weight*s)), the same for every rank
// One pass over the rows; a workgroup keeps its rows' contributions to the column sums in
// registers and a second kernel adds the workgroups' sums in a fixed order.
#include <cstdio>

#include "stand_ins.hpp"

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

  // Elements col .. col + kVec - 1 of a row of `cols`, zeros past its end.
  static __device__ __forceinline__ u32x4 load(const void* row, int col, int cols) {
    const uint8_t* p = static_cast<const uint8_t*>(row) + (int64_t)col * kSize;
    u32x4 v = {0, 0, 0, 0};
    if (col + kVec <= cols) {
      v = *(GlobalVecAny*)(uintptr_t)p;
    } else if (col < cols) {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (col + e < cols) {
          if constexpr (BF16) v[e >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
          else v[e] = reinterpret_cast<const uint32_t*>(p)[e];
        }
    }
    return v;
  }
  static __device__ __forceinline__ float get(const u32x4& v, int e) {
    if constexpr (BF16) return (e & 1) ? bf16_hi(v[e >> 1]) : bf16_lo(v[e >> 1]);
    else return __uint_as_float(v[e]);
  }
  static __device__ __forceinline__ void store(void* row, int col, int cols, const float (&f)[kVec]) {
    uint8_t* p = static_cast<uint8_t*>(row) + (int64_t)col * kSize;
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (BF16) v[k] = pack_bf16x2(f[2 * k], f[2 * k + 1]);
      else v[k] = __float_as_uint(f[k]);
    }
    if (col + kVec <= cols) {
      *reinterpret_cast<u32x4_any*>(p) = v;
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

// Sums of N values over the workgroup, the same bits in every thread.  `slots` is not read or
// written by the call before the last one, so one barrier per call is enough with two sets
// taken in turn.
template <int N>
__device__ __forceinline__ void workgroup_sums(float (&v)[N], float (*slots)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v[n] += __shfl_xor(v[n], d);
  const int waves = blockDim.x >> 6;
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) slots[threadIdx.x >> 6][n] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = slots[0][n];
  for (int w = 1; w < waves; ++w)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += slots[w][n];
}

struct NormForward {
  PeerPtrs peers;
  const void *residual, *weight, *post_weight, *gate;
  void *normed, *residual_out, *summed;
  int64_t rows;
  int cols, gate_kind, world_size;
  float residual_scale, eps;
};

template <bool BF16, int CHUNKS>
__global__ __launch_bounds__(1024) void all_reduce_norm_kernel(NormForward f, SignalPads pads, int rank, int do_barrier,
                                                               uint64_t limit_ticks, uint32_t* status) {
  using R = Row<BF16>;
  constexpr int V = R::kVec;
  __shared__ float slots[2][16][1];
  // (as in one_shot_all_reduce_kernel: nothing of this kernel to publish, and no cache holds
  // lines of the peers' data from before the handshake)
  if (do_barrier) {
    switch (f.world_size) {
#define SMR_NORM_WS(W) case W: barrier_with_stand_ins<W>(pads, blockIdx.x, rank, limit_ticks, status, false, false); break;
      SMR_NORM_WS(1) SMR_NORM_WS(2) SMR_NORM_WS(3) SMR_NORM_WS(4)
      SMR_NORM_WS(5) SMR_NORM_WS(6) SMR_NORM_WS(7) SMR_NORM_WS(8)
#undef SMR_NORM_WS
    }
  }
  const int cols = f.cols;
  const float inv_cols = 1.0f / (float)cols;
  for (int64_t row = blockIdx.x; row < f.rows; row += gridDim.x) {
    const int64_t base = row * cols * R::kSize;
    float s[CHUNKS][V];
    u32x4 x[CHUNKS], g[CHUNKS];
    float sq[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * V;
      u32x4 v[SMR_MAX_WORLD_SIZE];
#pragma unroll
      for (int r = 0; r < SMR_MAX_WORLD_SIZE; ++r)
        if (r < f.world_size) v[r] = R::load((const uint8_t*)(uintptr_t)f.peers.p[r] + base, col, cols);
      x[c] = R::load((const uint8_t*)f.residual + base, col, cols);
      if (f.gate_kind == kGateElement) g[c] = R::load((const uint8_t*)f.gate + base, col, cols);
      if (f.gate_kind == kGateChannel) g[c] = R::load(f.gate, col, cols);
#pragma unroll
      for (int e = 0; e < V; ++e) s[c][e] = 0.0f;
#pragma unroll
      for (int r = 0; r < SMR_MAX_WORLD_SIZE; ++r)
        if (r < f.world_size) {
#pragma unroll
          for (int e = 0; e < V; ++e) s[c][e] += R::get(v[r], e);
        }
#pragma unroll
      for (int e = 0; e < V; ++e) sq[0] += s[c][e] * s[c][e];
      if (f.summed != nullptr) R::store((uint8_t*)f.summed + base, col, cols, s[c]);
    }
    const float token_gate = f.gate_kind == kGateToken ? R::one(f.gate, row) : 1.0f;
    float r1 = 1.0f;
    if (f.post_weight != nullptr) {
      workgroup_sums<1>(sq, slots[0]);
      r1 = 1.0f / sqrtf(sq[0] * inv_cols + f.eps);
    }
    sq[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * V;
      u32x4 w = {0, 0, 0, 0};
      if (f.post_weight != nullptr) w = R::load(f.post_weight, col, cols);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float n = s[c][e];
        if (f.post_weight != nullptr) n = n * r1 * R::get(w, e);
        if (f.gate_kind == kGateElement || f.gate_kind == kGateChannel) n *= R::get(g[c], e);
        else n *= token_gate;
        s[c][e] = f.residual_scale * R::get(x[c], e) + n;
        sq[0] += s[c][e] * s[c][e];
      }
      R::store((uint8_t*)f.residual_out + base, col, cols, s[c]);
    }
    workgroup_sums<1>(sq, slots[1]);
    const float r2 = 1.0f / sqrtf(sq[0] * inv_cols + f.eps);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * V;
      const u32x4 w = R::load(f.weight, col, cols);
#pragma unroll
      for (int e = 0; e < V; ++e) s[c][e] = s[c][e] * r2 * R::get(w, e);
      R::store((uint8_t*)f.normed + base, col, cols, s[c]);
    }
    // without a post norm there is one reduction per row: its slots must not be overtaken
    if (f.post_weight == nullptr) __syncthreads();
  }
}

struct NormBackward {
  const void *grad_normed, *grad_residual_out, *summed, *residual_out, *weight, *post_weight, *gate;
  void *grad_partial, *grad_residual, *grad_gate;     // grad_gate: kinds token and element only
  float* sums;                                        // [kinds][gridDim.x][cols]: weight, post_weight, gate (channel)
  int64_t rows;
  int cols, gate_kind;
  float residual_scale, eps;
};

template <bool BF16, int CHUNKS>
__global__ __launch_bounds__(512) void norm_backward_kernel(NormBackward f) {
  using R = Row<BF16>;
  constexpr int V = R::kVec;
  __shared__ float slots3[8][3], slots2[8][2];
  const int cols = f.cols;
  const float inv_cols = 1.0f / (float)cols;
  const bool post = f.post_weight != nullptr;
  float sum_w[CHUNKS][V], sum_p[CHUNKS][V], sum_g[CHUNKS][V];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) sum_w[c][e] = sum_p[c][e] = sum_g[c][e] = 0.0f;

  for (int64_t row = blockIdx.x; row < f.rows; row += gridDim.x) {
    const int64_t base = row * cols * R::kSize;
    u32x4 s[CHUNKS], h[CHUNKS], dy[CHUNKS], dh[CHUNKS], g[CHUNKS];
    float t[3] = {0.0f, 0.0f, 0.0f};          // sums of h^2, dy*weight*h, s^2
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * V;
      h[c] = R::load((const uint8_t*)f.residual_out + base, col, cols);
      dy[c] = R::load((const uint8_t*)f.grad_normed + base, col, cols);
      s[c] = R::load((const uint8_t*)f.summed + base, col, cols);
      dh[c] = u32x4{0, 0, 0, 0};
      if (f.grad_residual_out != nullptr) dh[c] = R::load((const uint8_t*)f.grad_residual_out + base, col, cols);
      if (f.gate_kind == kGateElement) g[c] = R::load((const uint8_t*)f.gate + base, col, cols);
      if (f.gate_kind == kGateChannel) g[c] = R::load(f.gate, col, cols);
      const u32x4 w = R::load(f.weight, col, cols);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float he = R::get(h[c], e), se = R::get(s[c], e);
        t[0] += he * he;
        t[1] += R::get(dy[c], e) * R::get(w, e) * he;
        t[2] += se * se;
      }
    }
    const float token_gate = f.gate_kind == kGateToken ? R::one(f.gate, row) : 1.0f;
    workgroup_sums<3>(t, slots3);
    const float r2 = 1.0f / sqrtf(t[0] * inv_cols + f.eps);
    const float along = t[1] * inv_cols * r2 * r2;
    const float r1 = post ? 1.0f / sqrtf(t[2] * inv_cols + f.eps) : 1.0f;
    float d[CHUNKS][V];
    float u[2] = {0.0f, 0.0f};                // sums of dn*post_weight*s and D*n
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * V;
      const u32x4 w = R::load(f.weight, col, cols);
      u32x4 p = {0, 0, 0, 0};
      if (post) p = R::load(f.post_weight, col, cols);
      float out[V], dg[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float he = R::get(h[c], e), se = R::get(s[c], e), dye = R::get(dy[c], e);
        const float D = R::get(dh[c], e) + r2 * (dye * R::get(w, e) - he * along);
        sum_w[c][e] += dye * he * r2;
        out[e] = f.residual_scale * D;
        const float n = post ? se * r1 * R::get(p, e) : se;
        dg[e] = D * n;
        u[1] += dg[e];
        const float ge = f.gate_kind == kGateElement || f.gate_kind == kGateChannel ? R::get(g[c], e) : token_gate;
        float dn = D * ge;
        if (f.gate_kind == kGateChannel) sum_g[c][e] += dg[e];
        if (post) {
          sum_p[c][e] += dn * se * r1;
          dn *= R::get(p, e);
          u[0] += dn * se;
        }
        d[c][e] = dn;
      }
      R::store((uint8_t*)f.grad_residual + base, col, cols, out);
      if (f.gate_kind == kGateElement) R::store((uint8_t*)f.grad_gate + base, col, cols, dg);
    }
    workgroup_sums<2>(u, slots2);
    if (f.gate_kind == kGateToken && threadIdx.x == 0) R::put_one(f.grad_gate, row, u[1]);
    const float back = post ? u[0] * inv_cols * r1 * r1 : 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = (c * blockDim.x + threadIdx.x) * V;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (post) d[c][e] = r1 * (d[c][e] - R::get(s[c], e) * back);
      R::store((uint8_t*)f.grad_partial + base, col, cols, d[c]);
    }
  }
  auto put_sums = [&](const float (&v)[CHUNKS][V], int kind) {
    float* out = f.sums + ((int64_t)kind * gridDim.x + blockIdx.x) * cols;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int col = (c * blockDim.x + threadIdx.x) * V + e;
        if (col < cols) out[col] = v[c][e];
      }
  };
  put_sums(sum_w, 0);
  if (post) put_sums(sum_p, 1);
  if (f.gate_kind == kGateChannel) put_sums(sum_g, post ? 2 : 1);
}

// Column sums of the workgroups' contributions: out[kind][col] = sum over parts in order.  64
// columns per workgroup, 16 threads per column.
constexpr int kSumThreads = 1024;
template <bool BF16>
__global__ __launch_bounds__(kSumThreads) void norm_sums_kernel(const float* __restrict__ sums, int parts, int cols,
                                                                void* out0, void* out1, void* out2) {
  using R = Row<BF16>;
  __shared__ float share[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), who = threadIdx.x >> 6;
  void* out = blockIdx.y == 0 ? out0 : (blockIdx.y == 1 ? out1 : out2);
  const float* in = sums + (int64_t)blockIdx.y * parts * cols;
  float t = 0.0f;
  if (col < cols)
    for (int p = who; p < parts; p += 16) t += in[(int64_t)p * cols + col];
  share[who][threadIdx.x & 63] = t;
  __syncthreads();
  if (who == 0 && col < cols) {
#pragma unroll
    for (int w = 1; w < 16; ++w) t += share[w][threadIdx.x];
    R::put_one(out, col, t);
  }
}

// Threads and 128-bit chunks per thread for a row; the smallest number of chunks that fits.
static bool norm_shape(int cols, int vec, int max_threads, int& threads, int& chunks) {
  for (chunks = 1; chunks <= 8; chunks *= 2) {
    const int need = (cols + vec * chunks - 1) / (vec * chunks);
    if (need <= max_threads) {
      threads = (need + 63) / 64 * 64;
      return true;
    }
  }
  return false;
}

// Workgroups of a backward launch (each leaves cols fp32 sums per kind).
static int backward_blocks(int64_t rows) {
  const int64_t cap = 256;
  return (int)(rows < cap ? rows : cap);
}

static const char* check_norm_sizes(int64_t rows, int64_t cols, int dtype, int gate_kind, const void* gate) {
  if (dtype != SMR_DTYPE_BF16 && dtype != SMR_DTYPE_FP32) return "dtype must be bf16 (0) or fp32 (1)";
  if (rows < 0 || rows >= ((int64_t)1 << 40)) return "rows out of range";
  if (cols < 1) return "cols must be at least 1";
  if (gate_kind < kGateNone || gate_kind > kGateElement) return "unknown gate kind";
  if ((gate_kind == kGateNone) != (gate == nullptr)) return "gate and gate_kind must both be set or neither";
  return nullptr;
}

static int fail_norm(int code, const char* who, const char* what) {
  char buf[200];
  snprintf(buf, sizeof(buf), "%s: %s", who, what);
  return fail(code, buf);
}

template <bool BF16>
static int launch_forward(const NormForward& f, const SignalPads& pads, int rank, int do_barrier, uint32_t* status,
                          hipStream_t s) {
  int threads = 0, chunks = 0;
  if (!norm_shape(f.cols, Row<BF16>::kVec, 1024, threads, chunks))
    return fail(SMR_E_UNSUPPORTED, "smr_all_reduce_norm: more than 16384 columns");
  int64_t grid = (int64_t)compute_units() * (2048 / threads > 8 ? 8 : 2048 / threads);
  if (grid > f.rows) grid = f.rows;
  if (grid > 4096) grid = 4096;
  const uint64_t lim = spin_limit_ticks();
#define SMR_NORM_CASE(C)                                                                                              \
  case C:                                                                                                             \
    hipLaunchKernelGGL((all_reduce_norm_kernel<BF16, C>), dim3((unsigned)grid), dim3(threads), 0, s, f, pads, rank,   \
                       do_barrier, lim, status);                                                                      \
    break;
  switch (chunks) {
    SMR_NORM_CASE(1) SMR_NORM_CASE(2) SMR_NORM_CASE(4)
    default: return fail(SMR_E_UNSUPPORTED, "smr_all_reduce_norm: more than 16384 columns");
  }
#undef SMR_NORM_CASE
  return check_hip(hipGetLastError(), "smr_all_reduce_norm launch");
}

template <bool BF16>
static int launch_backward(const NormBackward& f, void* grad_weight, void* grad_post_weight, void* grad_gate_channel,
                           hipStream_t s) {
  int threads = 0, chunks = 0;
  if (!norm_shape(f.cols, Row<BF16>::kVec, 512, threads, chunks))
    return fail(SMR_E_UNSUPPORTED, "smr_norm_backward: more than 16384 columns");
  const int grid = backward_blocks(f.rows);
#define SMR_NORM_CASE(C)                                                                                 \
  case C:                                                                                                \
    hipLaunchKernelGGL((norm_backward_kernel<BF16, C>), dim3((unsigned)grid), dim3(threads), 0, s, f);   \
    break;
  switch (chunks) {
    SMR_NORM_CASE(1) SMR_NORM_CASE(2) SMR_NORM_CASE(4) SMR_NORM_CASE(8)
    default: return fail(SMR_E_UNSUPPORTED, "smr_norm_backward: more than 16384 columns");
  }
#undef SMR_NORM_CASE
  int rc = check_hip(hipGetLastError(), "smr_norm_backward launch");
  if (rc != 0) return rc;
  void* out[3] = {grad_weight, nullptr, nullptr};
  int kinds = 1;
  if (f.post_weight != nullptr) out[kinds++] = grad_post_weight;
  if (f.gate_kind == kGateChannel) out[kinds++] = grad_gate_channel;
  hipLaunchKernelGGL((norm_sums_kernel<BF16>), dim3((unsigned)((f.cols + 63) / 64), (unsigned)kinds), dim3(kSumThreads), 0,
                     s, f.sums, grid, f.cols, out[0], out[1], out[2]);
  return check_hip(hipGetLastError(), "smr_norm_backward launch");
}

}  // namespace smr

extern "C" {

int smr_all_reduce_norm(const uint64_t* buffer_ptrs_host, const uint64_t* signal_pad_ptrs_host, const void* residual,
                        const void* weight, const void* post_weight, const void* gate, int gate_kind, void* normed,
                        void* residual_out, void* summed, int64_t rows, int64_t cols, int dtype, double residual_scale,
                        double eps, int rank, int world_size, int barrier_mode, uint32_t* status, void* stream) {
  using namespace smr;
  static const char* who = "smr_all_reduce_norm";
  if (const char* what = check_norm_sizes(rows, cols, dtype, gate_kind, gate)) return fail_norm(SMR_E_INVALID, who, what);
  if (cols > kNormMaxCols) return fail_norm(SMR_E_UNSUPPORTED, who, "more than 16384 columns");
  if (world_size < 1 || world_size > SMR_MAX_WORLD_SIZE) return fail_norm(SMR_E_INVALID, who, "world_size must be 1..8");
  if (rank < 0 || rank >= world_size) return fail_norm(SMR_E_INVALID, who, "rank out of range");
  if (barrier_mode != SMR_BARRIER_NONE && barrier_mode != SMR_BARRIER_PROXY)
    return fail_norm(SMR_E_INVALID, who, "barrier_mode must be SMR_BARRIER_NONE or SMR_BARRIER_PROXY");
  if (buffer_ptrs_host == nullptr || (barrier_mode != SMR_BARRIER_NONE && signal_pad_ptrs_host == nullptr))
    return fail_norm(SMR_E_INVALID, who, "address table is NULL");
  const uintptr_t elem = dtype == SMR_DTYPE_BF16 ? 1u : 3u;
  NormForward f = {};
  SignalPads pads = {};
  for (int r = 0; r < world_size; ++r) {
    if (buffer_ptrs_host[r] == 0 || (buffer_ptrs_host[r] & elem))
      return fail_norm(SMR_E_INVALID, who, "buffer addresses must be non-zero and aligned to an element");
    f.peers.p[r] = buffer_ptrs_host[r];
    if (barrier_mode != SMR_BARRIER_NONE) {
      if (signal_pad_ptrs_host[r] == 0 || (signal_pad_ptrs_host[r] & 3u))
        return fail_norm(SMR_E_INVALID, who, "signal pad addresses must be non-zero and 4-byte aligned");
      pads.p[r] = signal_pad_ptrs_host[r];
    }
  }
  if (rows == 0) return 0;
  if (residual == nullptr || weight == nullptr || normed == nullptr || residual_out == nullptr)
    return fail_norm(SMR_E_INVALID, who, "NULL argument");
  uintptr_t all = 0;
  for (const void* p : {residual, weight, post_weight, gate, (const void*)normed, (const void*)residual_out, (const void*)summed})
    all |= reinterpret_cast<uintptr_t>(p);
  if (all & elem) return fail_norm(SMR_E_INVALID, who, "arguments must be aligned to an element");
  f.residual = residual;
  f.weight = weight;
  f.post_weight = post_weight;
  f.gate = gate;
  f.normed = normed;
  f.residual_out = residual_out;
  f.summed = summed;
  f.rows = rows;
  f.cols = (int)cols;
  f.gate_kind = gate_kind;
  f.world_size = world_size;
  f.residual_scale = (float)residual_scale;
  f.eps = (float)eps;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int do_barrier = barrier_mode != SMR_BARRIER_NONE;
  return dtype == SMR_DTYPE_BF16 ? launch_forward<true>(f, pads, rank, do_barrier, status, s)
                                 : launch_forward<false>(f, pads, rank, do_barrier, status, s);
}

int64_t smr_norm_backward_scratch_bytes(int64_t rows, int64_t cols, int has_post_weight, int gate_kind) {
  using namespace smr;
  if (rows < 0 || cols < 1 || cols > kNormMaxCols) return SMR_E_INVALID;
  const int kinds = 1 + (has_post_weight ? 1 : 0) + (gate_kind == kGateChannel ? 1 : 0);
  return (int64_t)kinds * backward_blocks(rows) * cols * 4;
}

int smr_norm_backward(const void* grad_normed, const void* grad_residual_out, const void* summed,
                      const void* residual_out, const void* weight, const void* post_weight, const void* gate,
                      int gate_kind, void* grad_partial, void* grad_residual, void* grad_weight,
                      void* grad_post_weight, void* grad_gate, float* scratch, int64_t scratch_bytes, int64_t rows,
                      int64_t cols, int dtype, double residual_scale, double eps, void* stream) {
  using namespace smr;
  static const char* who = "smr_norm_backward";
  if (const char* what = check_norm_sizes(rows, cols, dtype, gate_kind, gate)) return fail_norm(SMR_E_INVALID, who, what);
  if (cols > kNormMaxCols) return fail_norm(SMR_E_UNSUPPORTED, who, "more than 16384 columns");
  if (rows < 1) return fail_norm(SMR_E_INVALID, who, "rows must be at least 1");
  if (grad_normed == nullptr || summed == nullptr || residual_out == nullptr || weight == nullptr ||
      grad_partial == nullptr || grad_residual == nullptr || grad_weight == nullptr || scratch == nullptr)
    return fail_norm(SMR_E_INVALID, who, "NULL argument");
  if ((post_weight == nullptr) != (grad_post_weight == nullptr) || (gate == nullptr) != (grad_gate == nullptr))
    return fail_norm(SMR_E_INVALID, who, "a weight or gate and its gradient must both be given or neither");
  if (scratch_bytes < smr_norm_backward_scratch_bytes(rows, cols, post_weight != nullptr, gate_kind))
    return fail_norm(SMR_E_INVALID, who, "the scratch array is too small");
  const uintptr_t elem = dtype == SMR_DTYPE_BF16 ? 1u : 3u;
  uintptr_t all = 0;
  for (const void* p : {grad_normed, grad_residual_out, summed, residual_out, weight, post_weight, gate,
                        (const void*)grad_partial, (const void*)grad_residual, (const void*)grad_weight,
                        (const void*)grad_post_weight, (const void*)grad_gate})
    all |= reinterpret_cast<uintptr_t>(p);
  if ((all & elem) || (reinterpret_cast<uintptr_t>(scratch) & 3u))
    return fail_norm(SMR_E_INVALID, who, "arguments must be aligned to an element");
  NormBackward f = {grad_normed, grad_residual_out, summed, residual_out, weight, post_weight, gate,
                    grad_partial, grad_residual,
                    gate_kind == kGateToken || gate_kind == kGateElement ? grad_gate : nullptr,
                    scratch, rows, (int)cols, gate_kind, (float)residual_scale, (float)eps};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  void* channel = gate_kind == kGateChannel ? grad_gate : nullptr;
  return dtype == SMR_DTYPE_BF16 ? launch_backward<true>(f, grad_weight, grad_post_weight, channel, s)
                                 : launch_backward<false>(f, grad_weight, grad_post_weight, channel, s);
}

}  // extern "C"
