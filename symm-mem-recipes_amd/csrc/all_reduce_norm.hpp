// Forward kernel of the reduce fused with norms, gate and residual: see all_reduce_norm.hip.  The kernels
// are instantiated for every world size in files of their own, so that they are compiled side by side.
#pragma once

#include "norm_rows.hpp"
#include "stand_ins.hpp"

namespace smr {

struct NormForward {
  PeerPtrs peers;
  const void *residual, *weight, *post_weight, *gate;
  void *normed, *residual_out, *summed;
  int64_t rows;
  int cols, gate_kind, world_size;
  float residual_scale, eps;
};

// A workgroup takes rows blockIdx.x, + gridDim.x, ...  AHEAD: the next row's loads are issued before the
// two reductions of the present one, so memory is busy while they run (4096 x 8192 over 8 ranks: 138 us,
// without 164).  STREAM: results past the caches (138, through them 148).  WHOLE: every vector of every
// thread is known to lie inside the row (136, found out at run time 143: stores under a branch).
template <bool BF16, int WS, int CHUNKS, bool AHEAD, bool STREAM, bool WHOLE, int THREADS>
__global__ __launch_bounds__(THREADS) void all_reduce_norm_kernel(NormForward f, SignalPads pads, int rank, int do_barrier,
                                                                  uint64_t limit_ticks, uint32_t* status) {
  using R = Row<BF16>;
  constexpr int V = R::kVec;
  constexpr bool kKeepWeights = CHUNKS <= 2;
  __shared__ float slots[3][THREADS / 64][1];
  const int waves = blockDim.x >> 6;
  const int cols = f.cols;
  const bool whole = WHOLE || cols == (int)blockDim.x * CHUNKS * V;
  const float inv_cols = 1.0f / (float)cols;
  const bool post = f.post_weight != nullptr;
  const bool gated = f.gate_kind == kGateElement || f.gate_kind == kGateChannel;
  const int64_t row_bytes = (int64_t)cols * R::kSize;
  // (without a gate to load, the weight stands in for it: one code path, and its values are not used)
  const uint8_t* gate = static_cast<const uint8_t*>(gated ? f.gate : f.weight);
  const int64_t gate_step = f.gate_kind == kGateElement ? row_bytes : 0;
  const void* token = f.gate_kind == kGateToken ? f.gate : f.weight;
  const int64_t token_step = f.gate_kind == kGateToken ? 1 : 0;
  const void* post_weight = post ? f.post_weight : f.weight;

  struct Peers {
    u32x4 v[AHEAD ? CHUNKS : 1][WS];
  };
  struct Own {
    u32x4 x[CHUNKS], g[CHUNKS];
    float token;
  };
  auto column = [&](int c) { return (int)(c * blockDim.x + threadIdx.x) * V; };
  Peers in;
  auto load_chunk = [&](int64_t row, int c, int to) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < WS; ++r)
      in.v[to][r] = R::template load<true>((const uint8_t*)(uintptr_t)f.peers.p[r] + row * row_bytes, column(c), cols);
  };
  auto load_peers = [&](int64_t row) __attribute__((always_inline)) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) load_chunk(row, c, c);
    }
  };
  auto load_own = [&](Own& o, int64_t row) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      o.x[c] = R::template load<true>((const uint8_t*)f.residual + row * row_bytes, column(c), cols);
      o.g[c] = R::load(gate + row * gate_step, column(c), cols);
    }
    o.token = R::one(token, row * token_step);
  };
  // What does not come from the peers is on its way before the handshake.
  Own own;
  load_own(own, blockIdx.x);
  u32x4 w[CHUNKS], pw[CHUNKS];
  if constexpr (kKeepWeights) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      w[c] = R::load(f.weight, column(c), cols);
      pw[c] = R::load(post_weight, column(c), cols);
    }
  }
  // (as in one_shot_all_reduce_kernel: nothing of this kernel to publish, and no cache holds
  // lines of the peers' data from before the handshake)
  if (do_barrier) barrier_with_stand_ins<WS>(pads, blockIdx.x, rank, limit_ticks, status, false, false);

  // The arithmetic runs on the vectors as they were loaded, the same shift in all of them; what is
  // summed over the row counts no element twice, and the results are put in place before they are stored.
  float s[CHUNKS][V];                         // the sum, then h, then the normed row
  float sq[1];
  auto count = [&](int c) __attribute__((always_inline)) {
    // (the elements of a vector that lies over the row's end belong to the vector before it)
    const Tail<V> tail(column(c), cols);
#pragma unroll
    for (int e = 0; e < V; ++e) sq[0] += whole || e >= tail.shift ? s[c][e] * s[c][e] : 0.0f;
  };
  auto put = [&](void* out, int64_t row, int c) __attribute__((always_inline)) {
    uint8_t* p = static_cast<uint8_t*>(out) + row * row_bytes;
    if (whole) {
      R::template store<STREAM>(p, column(c), cols, s[c]);
    } else {
      float t[V];
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = s[c][e];
      Tail<V>(column(c), cols).place(t);
      R::template store<STREAM>(p, column(c), cols, t);
    }
  };
  auto add = [&](int64_t row) __attribute__((always_inline)) {
    sq[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if constexpr (!AHEAD) load_chunk(row, c, 0);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        s[c][e] = 0.0f;
#pragma unroll
        for (int r = 0; r < WS; ++r) s[c][e] += R::get(in.v[AHEAD ? c : 0][r], e);
      }
      count(c);
      // (all chunks' loads at once would not fit the registers)
      if constexpr (!AHEAD && CHUNKS > 1) __builtin_amdgcn_sched_barrier(0);
    }
  };
  // (mean square + eps)^-1/2 of the row in s, whose sum of squares is sq; the row is scaled where its squares do not fit
  auto reciprocal_root = [&]() __attribute__((always_inline)) {
    float mean = sq[0] * inv_cols + f.eps;
    // (the same bits in every thread: a scalar branch)
    if (__builtin_expect(mean_out_of_range(__int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(mean)))), 0)) {
      const float by = mean_rescale(mean);
      sq[0] = 0.0f;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
        for (int e = 0; e < V; ++e) s[c][e] *= by;
        count(c);
      }
      workgroup_sums<1>(sq, slots[2], waves);
      mean = sq[0] * inv_cols + f.eps * by * by;
    }
    return 1.0f / sqrtf(mean);
  };
  auto finish = [&](int64_t row) __attribute__((always_inline)) {
    const float token_gate = f.gate_kind == kGateToken ? own.token : 1.0f;
    if (f.summed != nullptr) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) put(f.summed, row, c);
    }
    float r1 = 1.0f;
    if (post) {
      workgroup_sums<1>(sq, slots[0], waves);
      r1 = reciprocal_root();
    }
    sq[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if constexpr (!kKeepWeights) pw[c] = R::load(post_weight, column(c), cols);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float n = post ? s[c][e] * r1 * R::get(pw[c], e) : s[c][e];
        s[c][e] = f.residual_scale * R::get(own.x[c], e) + (gated ? R::get(own.g[c], e) : token_gate) * n;
      }
      count(c);
      put(f.residual_out, row, c);
    }
    workgroup_sums<1>(sq, slots[1], waves);
    const float r2 = reciprocal_root();
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if constexpr (!kKeepWeights) w[c] = R::load(f.weight, column(c), cols);
#pragma unroll
      for (int e = 0; e < V; ++e) s[c][e] = s[c][e] * r2 * R::get(w[c], e);
      put(f.normed, row, c);
    }
    // without a post norm there is one reduction per row: its slots must not be overtaken
    if (!post) __syncthreads();
  };
  int64_t row = blockIdx.x;                                      // the grid has no more workgroups than rows
  load_peers(row);
  for (;;) {
    add(row);
    const int64_t next = row + gridDim.x;
    if (next >= f.rows) break;
    if constexpr (AHEAD) {
      Own own_next;
      load_own(own_next, next);
      load_peers(next);
      finish(row);
      own = own_next;
    } else {
      finish(row);
      load_own(own, next);
    }
    row = next;
  }
  finish(row);
}

template <bool BF16, int WS>
int launch_forward_ws(const NormForward& f, const SignalPads& pads, int rank, int do_barrier, uint32_t* status,
                      hipStream_t s) {
  constexpr int V = Row<BF16>::kVec;
  const int64_t cus = compute_units();
  const uint64_t lim = spin_limit_ticks();
  int threads = 0, chunks = 0;
  int64_t grid = 0;
#define SMR_NORM_LAUNCH(C, AHEAD, STREAM, WHOLE, T)                                                                    \
  hipLaunchKernelGGL((all_reduce_norm_kernel<BF16, WS, C, AHEAD, STREAM, WHOLE, T>), dim3((unsigned)grid), dim3(threads), \
                     0, s, f, pads, rank, do_barrier, lim, status)
  // Several rows per compute unit and rows that occupy one: a workgroup per compute unit that loads ahead.  Rows
  // of up to 128 threads do better as many workgroups (16384 x 1024: 72 us, loading ahead 87), rows of 129 to 256
  // unless there are many (16384 x 2048: 136 and 129; 777 x 1001 fp32: 12.9 and 14.6).
  if (f.rows > cus && norm_shape(f.cols, V, 512, threads, chunks) && chunks <= 2 &&
      (threads > 256 || (threads > 128 && f.rows >= 16 * cus))) {
    grid = cus;
    const bool whole = f.cols == threads * chunks * V;
    if (chunks == 1 && whole) SMR_NORM_LAUNCH(1, true, true, true, 512);
    else if (chunks == 1) SMR_NORM_LAUNCH(1, true, true, false, 512);
    else if (whole) SMR_NORM_LAUNCH(2, true, true, true, 512);
    else SMR_NORM_LAUNCH(2, true, true, false, 512);
    return check_hip(hipGetLastError(), "smr_all_reduce_norm launch");
  }
  // One or two rows per workgroup, as many threads on a row as it has vectors for.
  if (!norm_shape(f.cols, V, 1024, threads, chunks))
    return fail(SMR_E_UNSUPPORTED, "smr_all_reduce_norm: more than 16384 columns");
  grid = cus * (threads <= 256 ? 8 : 2048 / threads);
  if (grid > f.rows) grid = f.rows;
  if (grid > 4096) grid = 4096;                 // blocks that a signal pad has slots for
  // (the wide rows' results past the caches: 2048 x 16384 135 us, through them 144; 16384 x 1024 72 and 69)
  if (chunks == 1) SMR_NORM_LAUNCH(1, false, false, false, 1024);
  else if (chunks == 2) SMR_NORM_LAUNCH(2, false, true, false, 1024);
  else if constexpr (!BF16) SMR_NORM_LAUNCH(4, false, true, false, 1024);        // (16384 bf16 fit two chunks)
#undef SMR_NORM_LAUNCH
  return check_hip(hipGetLastError(), "smr_all_reduce_norm launch");
}

}  // namespace smr

// (`extern` in front: in another file)
#define SMR_INSTANTIATE_FORWARD(BF16, WS)                                                                     \
  template int smr::launch_forward_ws<BF16, WS>(const smr::NormForward&, const smr::SignalPads&, int, int,    \
                                                uint32_t*, hipStream_t);
