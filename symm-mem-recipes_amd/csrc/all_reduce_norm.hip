// The end of a tensor-parallel block in one pass over its partial sums: one-shot all-reduce, the
// norm behind the block, its gate, the scaled residual and the norm in front of the next block.
//
//   s = sum over the ranks of their partial sums            fp32, rank order, as one_shot_all_reduce
//   n = s * (mean(s^2) + eps)^-1/2 * post_weight            (n = s without a post_weight)
//   h = residual_scale * residual + gate * n                -> residual_out
//   y = h * (mean(h^2) + eps)^-1/2 * weight                 -> normed
//
// A row stays in its workgroup's registers from the sum to the stores, in fp32; each output is
// rounded once.  The bound is HBM, (world_size + 3) * cols elements per row (and the sum where it is
// wanted): 4096 x 8192 bf16 over 8 ranks with the sum 134-139 us, 5.8-6.0 TB/s.  One row takes 7.3 us:
// launch, handshake (1.7-2 us), a trip to memory, two reductions, stores.
#include <cstdio>

#include "all_reduce_norm.hpp"

#define SMR_ELSEWHERE(WS) extern SMR_INSTANTIATE_FORWARD(true, WS) extern SMR_INSTANTIATE_FORWARD(false, WS)
SMR_ELSEWHERE(1) SMR_ELSEWHERE(2) SMR_ELSEWHERE(3) SMR_ELSEWHERE(4)
SMR_ELSEWHERE(5) SMR_ELSEWHERE(6) SMR_ELSEWHERE(7) SMR_ELSEWHERE(8)

namespace smr {

int fail_norm(int code, const char* who, const char* what) {
  char buf[200];
  snprintf(buf, sizeof(buf), "%s: %s", who, what);
  return fail(code, buf);
}

// Rows narrower than a vector: a thread per row.
template <bool BF16>
__global__ __launch_bounds__(256) void all_reduce_norm_narrow_kernel(NormForward f, SignalPads pads, int rank, int do_barrier,
                                                                     uint64_t limit_ticks, uint32_t* status) {
  using R = Row<BF16>;
  constexpr int N = R::kVec - 1;
  if (do_barrier) {
    switch (f.world_size) {
#define SMR_NORM_WS(W) case W: barrier_with_stand_ins<W>(pads, blockIdx.x, rank, limit_ticks, status, false, false); break;
      SMR_NORM_WS(1) SMR_NORM_WS(2) SMR_NORM_WS(3) SMR_NORM_WS(4)
      SMR_NORM_WS(5) SMR_NORM_WS(6) SMR_NORM_WS(7) SMR_NORM_WS(8)
#undef SMR_NORM_WS
    }
  }
  for (int64_t row = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; row < f.rows; row += (int64_t)gridDim.x * blockDim.x) {
    const int64_t at = row * f.cols;
    float v[N], sq = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      v[c] = 0.0f;
      if (c < f.cols)
        for (int r = 0; r < f.world_size; ++r) v[c] += R::one((const void*)(uintptr_t)f.peers.p[r], at + c);
      sq += v[c] * v[c];
      if (f.summed != nullptr && c < f.cols) R::put_one(f.summed, at + c, v[c]);
    }
    // (mean square + eps)^-1/2; v is scaled where its squares do not fit
    auto reciprocal_root = [&]() {
      float mean = sq / (float)f.cols + f.eps;
      if (mean_out_of_range(mean)) {
        const float by = mean_rescale(mean);
        sq = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) {
          v[c] *= c < f.cols ? by : 0.0f;
          sq += v[c] * v[c];
        }
        mean = sq / (float)f.cols + f.eps * by * by;
      }
      return 1.0f / sqrtf(mean);
    };
    const float r1 = f.post_weight != nullptr ? reciprocal_root() : 1.0f;
    sq = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < f.cols) {
        float n = v[c];
        if (f.post_weight != nullptr) n *= r1 * R::one(f.post_weight, c);
        if (f.gate_kind == kGateChannel) n *= R::one(f.gate, c);
        if (f.gate_kind == kGateToken) n *= R::one(f.gate, row);
        if (f.gate_kind == kGateElement) n *= R::one(f.gate, at + c);
        v[c] = f.residual_scale * R::one(f.residual, at + c) + n;
        sq += v[c] * v[c];
        R::put_one(f.residual_out, at + c, v[c]);
      }
    const float r2 = reciprocal_root();
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < f.cols) R::put_one(f.normed, at + c, v[c] * r2 * R::one(f.weight, c));
  }
}

template <bool BF16>
static int launch_forward(const NormForward& f, const SignalPads& pads, int rank, int do_barrier, uint32_t* status,
                          hipStream_t s) {
  if (f.cols < Row<BF16>::kVec) {
    const int64_t blocks = (f.rows + 255) / 256, cus = compute_units();
    hipLaunchKernelGGL((all_reduce_norm_narrow_kernel<BF16>), dim3((unsigned)(blocks < cus ? blocks : cus)), dim3(256), 0, s,
                       f, pads, rank, do_barrier, spin_limit_ticks(), status);
    return check_hip(hipGetLastError(), "smr_all_reduce_norm launch");
  }
#define SMR_NORM_CASE(W) \
  case W: return launch_forward_ws<BF16, W>(f, pads, rank, do_barrier, status, s);
  switch (f.world_size) {
    SMR_NORM_CASE(1) SMR_NORM_CASE(2) SMR_NORM_CASE(3) SMR_NORM_CASE(4)
    SMR_NORM_CASE(5) SMR_NORM_CASE(6) SMR_NORM_CASE(7) SMR_NORM_CASE(8)
  }
#undef SMR_NORM_CASE
  return fail(SMR_E_INVALID, "smr_all_reduce_norm: world_size must be 1..8");
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

}  // extern "C"
