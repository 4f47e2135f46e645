// Backward pass of all_reduce_norm.hip.  With s, h, y and the weights as there, r1 and r2 the two
// reciprocal roots and D the whole gradient of h:
//   D  = grad_residual_out + r2 * (dy*weight - h * r2^2 * mean(dy*weight*h)),  dy = grad_normed
//   residual: residual_scale * D          weight: sum over rows of dy * h * r2
//   gate: D * n, summed over what the gate was broadcast over
//   with dn = gate * D:  post_weight: sum over rows of dn * s * r1
//   partial: r1 * (dn*post_weight - s * r1^2 * mean(dn*post_weight*s)), the same for every rank
// One pass over the rows, bound by HBM: four reads and two writes of an element (and the gate's).  A
// workgroup keeps its rows' contributions to the column sums in registers and a second kernel adds
// the workgroups' sums in a fixed order; a single workgroup writes them itself.
#include "norm_rows.hpp"

namespace smr {

struct NormBackward {
  const void *grad_normed, *grad_residual_out, *summed, *residual_out, *weight, *post_weight, *gate;
  void *grad_partial, *grad_residual, *grad_gate;     // grad_gate: kinds token and element only
  float* sums;                                        // [kinds][gridDim.x][cols]
  void* out[3];                                       // by kind: weight, post_weight, gate (channel)
  int64_t rows;
  int cols, gate_kind;
  float residual_scale, eps;
};

// AHEAD: the next row's loads are issued before the reductions of the present one.  WHOLE: every vector
// of every thread is known to lie inside the row.
template <bool BF16, int CHUNKS, bool AHEAD, bool WHOLE, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_backward_kernel(NormBackward f) {
  using R = Row<BF16>;
  constexpr int V = R::kVec;
  constexpr bool kKeepWeights = CHUNKS <= 2;
  __shared__ float slots3[THREADS / 64][3], slots2[THREADS / 64][2];
  const int waves = blockDim.x >> 6;
  const int cols = f.cols;
  const bool whole = WHOLE || cols == (int)blockDim.x * CHUNKS * V;
  const float inv_cols = 1.0f / (float)cols;
  const bool post = f.post_weight != nullptr, has_dh = f.grad_residual_out != nullptr;
  const bool gated = f.gate_kind == kGateElement || f.gate_kind == kGateChannel;
  const int64_t row_bytes = (int64_t)cols * R::kSize;
  // (where there is nothing to load something else is, and not used: one code path)
  const uint8_t* dh_rows = static_cast<const uint8_t*>(has_dh ? f.grad_residual_out : f.residual_out);
  const uint8_t* gate = static_cast<const uint8_t*>(gated ? f.gate : f.weight);
  const int64_t gate_step = f.gate_kind == kGateElement ? row_bytes : 0;
  const void* token = f.gate_kind == kGateToken ? f.gate : f.weight;
  const int64_t token_step = f.gate_kind == kGateToken ? 1 : 0;
  const void* post_weight = post ? f.post_weight : f.weight;

  struct In {
    u32x4 h[CHUNKS], dy[CHUNKS], s[CHUNKS], dh[CHUNKS], g[CHUNKS];
    float token;
  };
  auto column = [&](int c) { return (int)(c * blockDim.x + threadIdx.x) * V; };
  auto load = [&](In& v, int64_t row) __attribute__((always_inline)) {
    const int64_t base = row * row_bytes;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      v.h[c] = R::template load<true>((const uint8_t*)f.residual_out + base, column(c), cols);
      v.dy[c] = R::template load<true>((const uint8_t*)f.grad_normed + base, column(c), cols);
      v.s[c] = R::template load<true>((const uint8_t*)f.summed + base, column(c), cols);
      v.dh[c] = R::template load<true>(dh_rows + base, column(c), cols);
      v.g[c] = R::load(gate + row * gate_step, column(c), cols);
    }
    v.token = R::one(token, row * token_step);
  };
  // (the elements of a vector that lies over the row's end belong to the vector before it: its threads
  // compute them too, but count and store only their own)
  auto own = [&](int c, int e) { return whole || e >= Tail<V>(column(c), cols).shift; };
  auto put = [&](void* out, int64_t row, int c, float (&v)[V]) __attribute__((always_inline)) {
    if (!whole) Tail<V>(column(c), cols).place(v);
    R::template store<AHEAD>(static_cast<uint8_t*>(out) + row * row_bytes, column(c), cols, v);
  };

  u32x4 w[CHUNKS], p[CHUNKS];
  if constexpr (kKeepWeights) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      w[c] = R::load(f.weight, column(c), cols);
      p[c] = R::load(post_weight, column(c), cols);
    }
  }
  float sum_w[CHUNKS][V], sum_p[CHUNKS][V], sum_g[CHUNKS][V];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) sum_w[c][e] = sum_p[c][e] = sum_g[c][e] = 0.0f;

  In in;
  float t[3];                                 // sums of h^2, dy*weight*h, s^2
  auto begin = [&]() __attribute__((always_inline)) {
    t[0] = t[1] = t[2] = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if constexpr (!kKeepWeights) w[c] = R::load(f.weight, column(c), cols);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float he = own(c, e) ? R::get(in.h[c], e) : 0.0f, se = own(c, e) ? R::get(in.s[c], e) : 0.0f;
        t[0] += he * he;
        t[1] += R::get(in.dy[c], e) * R::get(w[c], e) * he;
        t[2] += se * se;
      }
    }
  };
  auto finish = [&](int64_t row) __attribute__((always_inline)) {
    const float token_gate = f.gate_kind == kGateToken ? in.token : 1.0f;
    workgroup_sums<3>(t, slots3, waves);
    const float r2 = 1.0f / sqrtf(t[0] * inv_cols + f.eps);
    const float along = t[1] * inv_cols * r2 * r2;
    const float r1 = post ? 1.0f / sqrtf(t[2] * inv_cols + f.eps) : 1.0f;
    float d[CHUNKS][V];
    float u[2] = {0.0f, 0.0f};                // sums of dn*post_weight*s and D*n
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if constexpr (!kKeepWeights) p[c] = R::load(post_weight, column(c), cols);
      float out[V], dg[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float he = R::get(in.h[c], e), se = R::get(in.s[c], e), dye = R::get(in.dy[c], e);
        const float D = (has_dh ? R::get(in.dh[c], e) : 0.0f) + r2 * (dye * R::get(w[c], e) - he * along);
        sum_w[c][e] += dye * he * r2;
        out[e] = f.residual_scale * D;
        const float pe = post ? R::get(p[c], e) : 1.0f, n = se * r1 * pe;
        dg[e] = D * n;
        const float dn = D * (gated ? R::get(in.g[c], e) : token_gate);
        sum_g[c][e] += dg[e];
        sum_p[c][e] += dn * se * r1;
        d[c][e] = dn * pe;
        if (own(c, e)) {
          u[0] += d[c][e] * se;
          u[1] += dg[e];
        }
      }
      put(f.grad_residual, row, c, out);
      if (f.gate_kind == kGateElement) put(f.grad_gate, row, c, dg);
    }
    workgroup_sums<2>(u, slots2, waves);
    if (f.gate_kind == kGateToken && threadIdx.x == 0) R::put_one(f.grad_gate, row, u[1]);
    const float back = u[0] * inv_cols * r1 * r1;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (post) d[c][e] = r1 * (d[c][e] - R::get(in.s[c], e) * back);
      put(f.grad_partial, row, c, d[c]);
    }
  };
  int64_t row = blockIdx.x;                   // the grid has no more workgroups than rows
  load(in, row);
  for (;;) {
    begin();
    const int64_t next = row + gridDim.x;
    if (next >= f.rows) break;
    if constexpr (AHEAD) {
      In in_next;
      load(in_next, next);
      finish(row);
      in = in_next;
    } else {
      finish(row);
      load(in, next);
    }
    row = next;
  }
  finish(row);

  auto put_sums = [&](const float (&v)[CHUNKS][V], int kind) {
    float* out = f.sums + ((int64_t)kind * gridDim.x + blockIdx.x) * cols;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int col = (column(c) < cols - V ? column(c) : cols - V) + e;
        if (own(c, e)) {
          if (gridDim.x == 1) R::put_one(f.out[kind], col, v[c][e]);
          else out[col] = v[c][e];
        }
      }
  };
  put_sums(sum_w, 0);
  if (post) put_sums(sum_p, 1);
  if (f.gate_kind == kGateChannel) put_sums(sum_g, post ? 2 : 1);
}

// Rows narrower than a vector: one workgroup, a thread per row.
template <bool BF16>
__global__ __launch_bounds__(256) void norm_backward_narrow_kernel(NormBackward f) {
  using R = Row<BF16>;
  constexpr int N = R::kVec - 1;
  __shared__ float share[3][N][256];
  float sums[3][N];
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int c = 0; c < N; ++c) sums[k][c] = 0.0f;
  const bool post = f.post_weight != nullptr;
  const float inv_cols = 1.0f / (float)f.cols;
  for (int64_t row = threadIdx.x; row < f.rows; row += 256) {
    const int64_t at = row * f.cols;
    float h2 = 0.0f, dyh = 0.0f, s2 = 0.0f;
    for (int c = 0; c < f.cols; ++c) {
      const float h = R::one(f.residual_out, at + c), s = R::one(f.summed, at + c);
      h2 += h * h;
      dyh += R::one(f.grad_normed, at + c) * R::one(f.weight, c) * h;
      s2 += s * s;
    }
    const float r2 = 1.0f / sqrtf(h2 * inv_cols + f.eps), along = dyh * inv_cols * r2 * r2;
    const float r1 = post ? 1.0f / sqrtf(s2 * inv_cols + f.eps) : 1.0f;
    float d[N], dns = 0.0f, token = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < f.cols) {
        const float h = R::one(f.residual_out, at + c), s = R::one(f.summed, at + c), dy = R::one(f.grad_normed, at + c);
        const float D = (f.grad_residual_out != nullptr ? R::one(f.grad_residual_out, at + c) : 0.0f) +
                        r2 * (dy * R::one(f.weight, c) - h * along);
        const float p = post ? R::one(f.post_weight, c) : 1.0f, dg = D * s * r1 * p;
        float g = 1.0f;
        if (f.gate_kind == kGateChannel) g = R::one(f.gate, c);
        if (f.gate_kind == kGateToken) g = R::one(f.gate, row);
        if (f.gate_kind == kGateElement) g = R::one(f.gate, at + c);
        if (f.gate_kind == kGateElement) R::put_one(f.grad_gate, at + c, dg);
        R::put_one(f.grad_residual, at + c, f.residual_scale * D);
        sums[0][c] += dy * h * r2;
        sums[1][c] += D * g * s * r1;
        sums[2][c] += dg;
        token += dg;
        d[c] = D * g * p;
        dns += d[c] * s;
      }
    if (f.gate_kind == kGateToken) R::put_one(f.grad_gate, row, token);
    const float back = dns * inv_cols * r1 * r1;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < f.cols) R::put_one(f.grad_partial, at + c, post ? r1 * (d[c] - R::one(f.summed, at + c) * back) : d[c]);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int c = 0; c < N; ++c) share[k][c][threadIdx.x] = sums[k][c];
  __syncthreads();
  if (threadIdx.x < 3 * N) {
    const int k = threadIdx.x / N, c = threadIdx.x % N;
    float t = 0.0f;
    for (int i = 0; i < 256; ++i) t += share[k][c][i];
    // (sums are kept by what they are of; `out` lists those that are wanted)
    void* out = k == 0 ? f.out[0] : (k == 1 ? (post ? f.out[1] : nullptr) : (f.gate_kind == kGateChannel ? f.out[post ? 2 : 1] : nullptr));
    if (c < f.cols && out != nullptr) R::put_one(out, c, t);
  }
}

// Column sums of the workgroups' contributions: out[kind][col] = sum over parts in an order that depends
// on their number only.  64 columns per workgroup, 16 threads per column.
constexpr int kSumThreads = 1024;
template <bool BF16>
__global__ __launch_bounds__(kSumThreads) void norm_sums_kernel(const float* __restrict__ sums, int parts, int cols,
                                                                void* out0, void* out1, void* out2) {
  using R = Row<BF16>;
  __shared__ float share[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), who = threadIdx.x >> 6;
  void* out = blockIdx.y == 0 ? out0 : (blockIdx.y == 1 ? out1 : out2);
  const float* in = sums + (int64_t)blockIdx.y * parts * cols + (col < cols ? col : cols - 1);
  float t = 0.0f;
  int p = who;
  for (; p + 7 * 16 < parts; p += 8 * 16) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = in[(int64_t)(p + k * 16) * cols];
#pragma unroll
    for (int k = 0; k < 8; ++k) t += v[k];
  }
  for (; p < parts; p += 16) t += in[(int64_t)p * cols];
  share[who][threadIdx.x & 63] = t;
  __syncthreads();
  if (who == 0 && col < cols) {
#pragma unroll
    for (int w = 1; w < 16; ++w) t += share[w][threadIdx.x];
    R::put_one(out, col, t);
  }
}

#ifndef DIRECT
#define DIRECT 5
#endif
// How a backward pass is launched; `blocks` > 1 leave cols fp32 sums per kind each.
struct BackwardShape {
  int threads, chunks, blocks;
  bool ahead;
};
static BackwardShape backward_shape(int64_t rows, int cols, bool bf16) {
  BackwardShape s = {0, 0, 1, true};
  const int vec = bf16 ? 8 : 4;
  if (!norm_shape(cols, vec, 512, s.threads, s.chunks) || s.chunks > 2) {
    s.ahead = false;                          // wide rows: more threads rather than more registers
    norm_shape(cols, vec, 1024, s.threads, s.chunks);
  }
  if (rows > DIRECT) {
    const int64_t most = 256 * (int64_t)(s.threads <= 256 ? 512 / s.threads : 1);
    s.blocks = (int)(rows < most ? rows : most);
  }
  return s;
}

template <bool BF16>
static int launch_backward(NormBackward f, hipStream_t s) {
  constexpr int V = Row<BF16>::kVec;
  if (f.cols < V) {
    hipLaunchKernelGGL((norm_backward_narrow_kernel<BF16>), dim3(1), dim3(256), 0, s, f);
    return check_hip(hipGetLastError(), "smr_norm_backward launch");
  }
  const BackwardShape b = backward_shape(f.rows, f.cols, BF16);
  const bool whole = f.cols == b.threads * b.chunks * V;
#define SMR_NORM_LAUNCH(C, AHEAD, WHOLE, T)                                                                            \
  hipLaunchKernelGGL((norm_backward_kernel<BF16, C, AHEAD, WHOLE, T>), dim3((unsigned)b.blocks), dim3(b.threads), 0, s, f)
  if (b.ahead && b.chunks == 1 && whole) SMR_NORM_LAUNCH(1, true, true, 512);
  else if (b.ahead && b.chunks == 1) SMR_NORM_LAUNCH(1, true, false, 512);
  else if (b.ahead && whole) SMR_NORM_LAUNCH(2, true, true, 512);
  else if (b.ahead) SMR_NORM_LAUNCH(2, true, false, 512);
  else if (b.chunks <= 2) SMR_NORM_LAUNCH(2, false, false, 1024);
  else if constexpr (!BF16) SMR_NORM_LAUNCH(4, false, false, 1024);
#undef SMR_NORM_LAUNCH
  const int rc = check_hip(hipGetLastError(), "smr_norm_backward launch");
  if (rc != 0 || b.blocks == 1) return rc;
  const int kinds = 1 + (f.out[1] != nullptr) + (f.out[2] != nullptr);
  hipLaunchKernelGGL((norm_sums_kernel<BF16>), dim3((unsigned)((f.cols + 63) / 64), (unsigned)kinds), dim3(kSumThreads), 0,
                     s, f.sums, b.blocks, f.cols, f.out[0], f.out[1], f.out[2]);
  return check_hip(hipGetLastError(), "smr_norm_backward launch");
}

}  // namespace smr

extern "C" {

int64_t smr_norm_backward_scratch_bytes(int64_t rows, int64_t cols, int dtype, int has_post_weight, int gate_kind) {
  using namespace smr;
  if (rows < 0 || cols < 1 || cols > kNormMaxCols || (dtype != SMR_DTYPE_BF16 && dtype != SMR_DTYPE_FP32))
    return fail_norm(SMR_E_INVALID, "smr_norm_backward_scratch_bytes", "bad size or dtype");
  const bool bf16 = dtype == SMR_DTYPE_BF16;
  if (cols < (bf16 ? 8 : 4)) return 0;
  const int blocks = backward_shape(rows, (int)cols, bf16).blocks;
  const int kinds = 1 + (has_post_weight ? 1 : 0) + (gate_kind == kGateChannel ? 1 : 0);
  return blocks == 1 ? 0 : (int64_t)kinds * blocks * cols * 4;
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
      grad_partial == nullptr || grad_residual == nullptr || grad_weight == nullptr)
    return fail_norm(SMR_E_INVALID, who, "NULL argument");
  if ((post_weight == nullptr) != (grad_post_weight == nullptr) || (gate == nullptr) != (grad_gate == nullptr))
    return fail_norm(SMR_E_INVALID, who, "a weight or gate and its gradient must both be given or neither");
  const int64_t need = smr_norm_backward_scratch_bytes(rows, cols, dtype, post_weight != nullptr, gate_kind);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need))
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
                    scratch, {grad_weight, nullptr, nullptr}, rows, (int)cols, gate_kind, (float)residual_scale, (float)eps};
  int kinds = 1;
  if (post_weight != nullptr) f.out[kinds++] = grad_post_weight;
  if (gate_kind == kGateChannel) f.out[kinds++] = grad_gate;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == SMR_DTYPE_BF16 ? launch_backward<true>(f, s) : launch_backward<false>(f, s);
}

}  // extern "C"
