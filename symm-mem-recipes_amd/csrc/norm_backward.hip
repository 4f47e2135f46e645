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
// 4096 x 8192 bf16, a gate per element: 94-101 us (5.3-5.7 TB/s) and 5 us for the sums; fp32 200 us (5.4 TB/s).  Rows
// beyond 8192 columns are read three times and once more for their column sums: 2048 x 16384 bf16 230 us (2.3 TB/s).
#include "norm_rows.hpp"

namespace smr {

struct NormBackward {
  const void *grad_normed, *grad_residual_out, *summed, *residual_out, *weight, *post_weight, *gate;
  void *grad_partial, *grad_residual, *grad_gate;     // grad_gate: kinds token and element only
  float* sums;                                        // [kinds][parts][cols]
  float* row_values;                                  // wide rows: r2, r2^2 * mean(dy*weight*h), r1 of each
  void* out[3];                                       // by kind: weight, post_weight, gate (channel)
  int64_t rows;
  int cols, gate_kind;
  float residual_scale, eps;
};

// A row's vectors are loaded AHEAD, before the reductions of the row in front of it, or only KEPT in
// registers, where two rows would not fit; of rows wider than that they are read again, from the caches,
// for each phase, and the column sums are another kernel's (norm_columns_kernel).  WHOLE: every vector of
// every thread is known to lie inside the row.  No variant may spill: builds that kept column sums in
// scratch memory gave one of them wrong (the ISA test looks for scratch memory).
enum RowUse { kReread, kKept, kAhead };
template <bool BF16, int CHUNKS, RowUse USE, bool WHOLE, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_backward_kernel(NormBackward f) {
  using R = Row<BF16>;
  constexpr int V = R::kVec;
  constexpr bool kKeep = USE != kReread;
  constexpr int kHeld = kKeep ? CHUNKS : 1;
  __shared__ u32x4 weights[2][kKeep ? CHUNKS * THREADS : 1];      // a thread's own vectors of weight and post_weight
  __shared__ float slots3[2][THREADS / 64][3], slots2[THREADS / 64][2];
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
    u32x4 h[kHeld], dy[kHeld], s[kHeld], dh[kHeld], g[kHeld];
    float token;
  };
  int tid = threadIdx.x;
  auto column = [&](int c) { return (int)(c * blockDim.x + tid) * V; };
  auto load_chunk = [&](In& v, int64_t row, int c, int to) __attribute__((always_inline)) {
    const int64_t base = row * row_bytes;
    v.h[to] = R::template load<kKeep>((const uint8_t*)f.residual_out + base, column(c), cols);
    v.dy[to] = R::template load<kKeep>((const uint8_t*)f.grad_normed + base, column(c), cols);
    v.s[to] = R::template load<kKeep>((const uint8_t*)f.summed + base, column(c), cols);
    v.dh[to] = R::template load<kKeep>(dh_rows + base, column(c), cols);
    v.g[to] = R::load(gate + row * gate_step, column(c), cols);
  };
  auto load = [&](In& v, int64_t row) __attribute__((always_inline)) {
    if constexpr (kKeep) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) load_chunk(v, row, c, c);
    }
    v.token = R::one(token, row * token_step);
  };
  // (the elements of a vector that lies over the row's end belong to the vector before it: its threads
  // compute them too, but count and store only their own)
  auto first_own = [&](int c) __attribute__((always_inline)) { return whole ? 0 : Tail<V>(column(c), cols).shift; };
  auto put = [&](void* out, int64_t row, int c, float (&v)[V]) __attribute__((always_inline)) {
    if (!whole) Tail<V>(column(c), cols).place(v);
    R::template store<kKeep>(static_cast<uint8_t*>(out) + row * row_bytes, column(c), cols, v);
  };

  if constexpr (kKeep) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      weights[0][c * THREADS + threadIdx.x] = R::load(f.weight, column(c), cols);
      weights[1][c * THREADS + threadIdx.x] = R::load(post_weight, column(c), cols);
    }
  }
  // (from LDS: a load from memory would queue up behind the next row's)
  auto weight_of = [&](int which, int c) __attribute__((always_inline)) {
    if constexpr (kKeep) return weights[which][c * THREADS + threadIdx.x];
    else return R::load(which == 0 ? f.weight : post_weight, column(c), cols);
  };
  // Column sums of the workgroup's rows: the weight's, and D * s * r1 times the gate.  With a gate per channel the gate
  // stays out: the sum is the post weight's but for the gate and the gate's but for the post weight.
  const bool channel = f.gate_kind == kGateChannel;
  float sum_w[kHeld][V], sum_n[kHeld][V];
#pragma unroll
  for (int c = 0; c < kHeld; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) sum_w[c][e] = sum_n[c][e] = 0.0f;

  In in;
  float t[3];                                 // sums of h^2, dy*weight*h, s^2
  // (SCALED: of h and s times a factor each, for rows whose squares do not fit fp32)
  auto row_sums = [&](auto scaled, int64_t row, float by_h, float by_s) __attribute__((always_inline)) {
    constexpr bool SCALED = decltype(scaled)::value;
    // (recomputed for every row: kept, the addresses of all chunks would take the sums' registers)
    if constexpr (USE != kAhead) asm volatile("" : "+v"(tid));
    t[0] = t[1] = t[2] = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int k = kKeep ? c : 0;
      if constexpr (!kKeep) load_chunk(in, row, c, 0);
      const u32x4 w = weight_of(0, c);
      const int first = first_own(c);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // (the products are masked, not their factors: another vector's infinity must not become a NaN here)
        const float he = R::get(in.h[k], e) * (SCALED ? by_h : 1.0f), se = R::get(in.s[k], e) * (SCALED ? by_s : 1.0f);
        const bool own = e >= first;
        t[0] += own ? he * he : 0.0f;
        t[1] += own ? R::get(in.dy[k], e) * R::get(w, e) * he : 0.0f;
        t[2] += own ? se * se : 0.0f;
        if constexpr (USE != kAhead)
          if (e & 1) __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (!kKeep) __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto begin = [&](int64_t row) __attribute__((always_inline)) { row_sums(std::false_type{}, row, 1.0f, 1.0f); };
  auto finish = [&](int64_t row) __attribute__((always_inline)) {
    if constexpr (USE != kAhead) asm volatile("" : "+v"(tid));
    const float token_gate = f.gate_kind == kGateToken ? in.token : 1.0f;
    workgroup_sums<3>(t, slots3[0], waves);
    float mean_h = t[0] * inv_cols + f.eps, mean_s = t[2] * inv_cols + f.eps, by_h = 1.0f, by_s = 1.0f;
    const bool odd_h = mean_out_of_range(mean_h), odd_s = post && mean_out_of_range(mean_s);
    // (the same in every thread: a scalar branch)
    if (__builtin_expect(__any(odd_h || odd_s), 0)) {
      by_h = odd_h ? mean_rescale(mean_h) : 1.0f;
      by_s = odd_s ? mean_rescale(mean_s) : 1.0f;
      row_sums(std::true_type{}, row, by_h, by_s);
      workgroup_sums<3>(t, slots3[1], waves);
      mean_h = t[0] * inv_cols + f.eps * by_h * by_h;
      mean_s = t[2] * inv_cols + f.eps * by_s * by_s;
    }
    const float root_h = 1.0f / sqrtf(mean_h);
    const float r2 = root_h * by_h;
    const float along = t[1] * inv_cols * root_h * r2;
    const float r1 = post ? 1.0f / sqrtf(mean_s) * by_s : 1.0f;
    float d[kKeep ? CHUNKS : 1][V];           // dn*post_weight
    float u[2] = {0.0f, 0.0f};                // sums of dn*post_weight*s*r1 and D*n
    // D of an element
    auto whole_gradient = [&](int k, int e, const u32x4& w) __attribute__((always_inline)) {
      const float he = R::get(in.h[k], e), dye = R::get(in.dy[k], e);
      return (has_dh ? R::get(in.dh[k], e) : 0.0f) + r2 * (dye * R::get(w, e) - he * along);
    };
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int k = kKeep ? c : 0;
      if constexpr (!kKeep) load_chunk(in, row, c, 0);
      const u32x4 w = weight_of(0, c), p = weight_of(1, c);
      const int first = first_own(c);
      float out[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // (h and s meet their reciprocal root first: a product of theirs with a gradient may be out of range)
        const float D = whole_gradient(k, e, w), se = R::get(in.s[k], e) * r1;
        out[e] = f.residual_scale * D;
        const float pe = post ? R::get(p, e) : 1.0f, dg = D * (se * pe);
        const float dn = D * (gated ? R::get(in.g[k], e) : token_gate);
        if constexpr (kKeep) {
          sum_w[c][e] += R::get(in.dy[k], e) * (R::get(in.h[k], e) * r2);
          sum_n[c][e] += (channel ? D : dn) * se;
        }
        const float dnp = dn * pe;
        if constexpr (kKeep) d[c][e] = dnp;
        u[0] += e >= first ? dnp * se : 0.0f;
        u[1] += e >= first ? dg : 0.0f;
        // (a few elements at a time: all of a vector's terms at once would not fit beside the sums)
        if constexpr (USE != kAhead)
          if (e & 1) __builtin_amdgcn_sched_barrier(0);
      }
      put(f.grad_residual, row, c, out);
      if (f.gate_kind == kGateElement) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          out[e] = whole_gradient(k, e, w) * (R::get(in.s[k], e) * r1 * (post ? R::get(p, e) : 1.0f));
          if constexpr (!kKeep)
            if (e & 1) __builtin_amdgcn_sched_barrier(0);
        }
        put(f.grad_gate, row, c, out);
      }
      if constexpr (!kKeep) __builtin_amdgcn_sched_barrier(0);
    }
    workgroup_sums<2>(u, slots2, waves);
    if (f.gate_kind == kGateToken && threadIdx.x == 0) R::put_one(f.grad_gate, row, u[1]);
    const float back = u[0] * inv_cols * r1;
    if constexpr (!kKeep)
      if (threadIdx.x == 0) {
        f.row_values[row * 3] = r2;
        f.row_values[row * 3 + 1] = along;
        f.row_values[row * 3 + 2] = r1;
      }
    if constexpr (USE != kAhead) asm volatile("" : "+v"(tid));
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int k = kKeep ? c : 0;
      if constexpr (!kKeep) {
        load_chunk(in, row, c, 0);
        const u32x4 w = weight_of(0, c), p = weight_of(1, c);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          d[0][e] = whole_gradient(0, e, w) * (gated ? R::get(in.g[0], e) : token_gate) * (post ? R::get(p, e) : 1.0f);
          if (e & 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (post) d[k][e] = r1 * (d[k][e] - R::get(in.s[k], e) * back);
      put(f.grad_partial, row, c, d[k]);
      if constexpr (!kKeep) __builtin_amdgcn_sched_barrier(0);
    }
  };
  int64_t row = blockIdx.x;                   // the grid has no more workgroups than rows
  if constexpr (USE == kAhead) {
    load(in, row);
    for (;;) {
      begin(row);
      const int64_t next = row + gridDim.x;
      if (next >= f.rows) break;
      In in_next;
      load(in_next, next);
      finish(row);
      in = in_next;
      row = next;
    }
    finish(row);
  } else {
    for (; row < f.rows; row += gridDim.x) {
      load(in, row);
      begin(row);
      finish(row);
    }
  }

  if constexpr (kKeep) {
    auto put_sum = [&](float v, int c, int e, int kind) __attribute__((always_inline)) {
      const int col = (column(c) < cols - V ? column(c) : cols - V) + e;
      if (e >= first_own(c)) {
        if (gridDim.x == 1) R::put_one(f.out[kind], col, v);
        else f.sums[((int64_t)kind * gridDim.x + blockIdx.x) * cols + col] = v;
      }
    };
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e) put_sum(sum_w[c][e], c, e, 0);
      if (channel) {
        const u32x4 p = weight_of(1, c), g = R::load(gate, column(c), cols);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          put_sum(post ? sum_n[c][e] * R::get(p, e) : sum_n[c][e], c, e, post ? 2 : 1);
          if (post) put_sum(sum_n[c][e] * R::get(g, e), c, e, 1);
        }
      } else if (post) {
#pragma unroll
        for (int e = 0; e < V; ++e) put_sum(sum_n[c][e], c, e, 1);
      }
    }
  }
}

// Column sums for rows whose values norm_backward_kernel left in row_values: a wave takes 64 vectors of
// columns and every parts-th row; sums as there, [kinds][parts][cols].
template <bool BF16>
__global__ __launch_bounds__(64) void norm_columns_kernel(NormBackward f) {
  using R = Row<BF16>;
  constexpr int V = R::kVec;
  const int cols = f.cols, parts = gridDim.y, col = (int)(blockIdx.x * 64 + threadIdx.x) * V;
  const bool post = f.post_weight != nullptr, has_dh = f.grad_residual_out != nullptr;
  const bool gated = f.gate_kind == kGateElement || f.gate_kind == kGateChannel;
  const int64_t row_bytes = (int64_t)cols * R::kSize;
  const uint8_t* dh_rows = static_cast<const uint8_t*>(has_dh ? f.grad_residual_out : f.residual_out);
  const uint8_t* gate = static_cast<const uint8_t*>(gated ? f.gate : f.weight);
  const int64_t gate_step = f.gate_kind == kGateElement ? row_bytes : 0;
  const void* token = f.gate_kind == kGateToken ? f.gate : f.weight;
  const int64_t token_step = f.gate_kind == kGateToken ? 1 : 0;
  const u32x4 w = R::load(f.weight, col, cols), p = R::load(post ? f.post_weight : f.weight, col, cols);
  float sums[3][V];
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) sums[k][e] = 0.0f;
#pragma unroll 2
  for (int64_t row = blockIdx.y; row < f.rows; row += parts) {
    const int64_t base = row * row_bytes;
    const u32x4 h = R::load((const uint8_t*)f.residual_out + base, col, cols);
    const u32x4 dy = R::load((const uint8_t*)f.grad_normed + base, col, cols);
    const u32x4 s = R::load((const uint8_t*)f.summed + base, col, cols);
    const u32x4 dh = R::load(dh_rows + base, col, cols);
    const u32x4 g = R::load(gate + row * gate_step, col, cols);
    const float t = R::one(token, row * token_step), token_gate = f.gate_kind == kGateToken ? t : 1.0f;
    const float r2 = f.row_values[row * 3], along = f.row_values[row * 3 + 1], r1 = f.row_values[row * 3 + 2];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float he = R::get(h, e), dye = R::get(dy, e), se = R::get(s, e);
      const float D = (has_dh ? R::get(dh, e) : 0.0f) + r2 * (dye * R::get(w, e) - he * along);
      sums[0][e] += dye * (he * r2);
      sums[1][e] += D * (gated ? R::get(g, e) : token_gate) * (se * r1);
      sums[2][e] += D * (se * r1 * (post ? R::get(p, e) : 1.0f));
    }
  }
  const int first = Tail<V>(col, cols).shift, at = col < cols - V ? col : cols - V;
  const int kinds = 1 + post + (f.gate_kind == kGateChannel);
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (e >= first) {
      float* out = f.sums + (int64_t)blockIdx.y * cols + at + e;
      const int64_t step = (int64_t)parts * cols;
      out[0] = sums[0][e];
      if (post) out[step] = sums[1][e];
      if (f.gate_kind == kGateChannel) out[(kinds - 1) * step] = sums[2][e];
    }
}

// Rows narrower than a vector: one workgroup, a thread per row, however many there are (65536 x 7 bf16: 1.43 ms; no
// model has such rows).
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
    float mean_h = h2 * inv_cols + f.eps, mean_s = s2 * inv_cols + f.eps, by_h = 1.0f, by_s = 1.0f;
    if (mean_out_of_range(mean_h) || (post && mean_out_of_range(mean_s))) {
      by_h = mean_out_of_range(mean_h) ? mean_rescale(mean_h) : 1.0f;
      by_s = mean_out_of_range(mean_s) ? mean_rescale(mean_s) : 1.0f;
      h2 = dyh = s2 = 0.0f;
      for (int c = 0; c < f.cols; ++c) {
        const float h = R::one(f.residual_out, at + c) * by_h, s = R::one(f.summed, at + c) * by_s;
        h2 += h * h;
        dyh += R::one(f.grad_normed, at + c) * R::one(f.weight, c) * h;
        s2 += s * s;
      }
      mean_h = h2 * inv_cols + f.eps * by_h * by_h;
      mean_s = s2 * inv_cols + f.eps * by_s * by_s;
    }
    const float root_h = 1.0f / sqrtf(mean_h), r2 = root_h * by_h, along = dyh * inv_cols * root_h * r2;
    const float r1 = post ? 1.0f / sqrtf(mean_s) * by_s : 1.0f;
    float d[N], dns = 0.0f, token = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < f.cols) {
        const float h = R::one(f.residual_out, at + c), s = R::one(f.summed, at + c) * r1, dy = R::one(f.grad_normed, at + c);
        const float D = (f.grad_residual_out != nullptr ? R::one(f.grad_residual_out, at + c) : 0.0f) +
                        r2 * (dy * R::one(f.weight, c) - h * along);
        const float p = post ? R::one(f.post_weight, c) : 1.0f, dg = D * (s * p);
        float g = 1.0f;
        if (f.gate_kind == kGateChannel) g = R::one(f.gate, c);
        if (f.gate_kind == kGateToken) g = R::one(f.gate, row);
        if (f.gate_kind == kGateElement) g = R::one(f.gate, at + c);
        if (f.gate_kind == kGateElement) R::put_one(f.grad_gate, at + c, dg);
        R::put_one(f.grad_residual, at + c, f.residual_scale * D);
        sums[0][c] += dy * (h * r2);
        sums[1][c] += D * g * s;
        sums[2][c] += dg;
        token += dg;
        d[c] = D * g * p;
        dns += d[c] * s;
      }
    if (f.gate_kind == kGateToken) R::put_one(f.grad_gate, row, token);
    const float back = dns * inv_cols * r1;
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
// on their number only.  32 columns (a 128-byte line) per workgroup, 32 threads per column.
constexpr int kSumThreads = 1024;
template <bool BF16>
__global__ __launch_bounds__(kSumThreads) void norm_sums_kernel(const float* __restrict__ sums, int parts, int cols,
                                                                void* out0, void* out1, void* out2) {
  using R = Row<BF16>;
  __shared__ float share[32][32];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), who = threadIdx.x >> 5;
  void* out = blockIdx.y == 0 ? out0 : (blockIdx.y == 1 ? out1 : out2);
  const float* in = sums + (int64_t)blockIdx.y * parts * cols + (col < cols ? col : cols - 1);
  float t = 0.0f;
  int p = who;
  for (; p + 7 * 32 < parts; p += 8 * 32) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = in[(int64_t)(p + k * 32) * cols];
#pragma unroll
    for (int k = 0; k < 8; ++k) t += v[k];
  }
  for (; p < parts; p += 32) t += in[(int64_t)p * cols];
  share[who][threadIdx.x & 31] = t;
  __syncthreads();
  if (who == 0 && col < cols) {
#pragma unroll
    for (int w = 1; w < 32; ++w) t += share[w][threadIdx.x];
    R::put_one(out, col, t);
  }
}

// Rows that one workgroup takes, one after the other, instead of one workgroup each and a second launch for their sums.
// The second launch and its scratch array cost the host 4 us (12.4 us a call, 16.4 with them), so one workgroup is
// taken while it is slower on the GPU by no more than that.  A row's time grows with its width: times on the GPU, one
// workgroup / two launches, in us:
//     rows          2            3            4            5            8
//    512 bf16    5.3 /  6.1   6.4 /  6.0   7.5 /  6.1   8.7 /  6.1  12.0 /  6.1    one vector a thread
//   2048 fp32    5.9 /  6.7   7.3 /  6.7   8.7 /  6.8  10.2 /  6.8                 one
//   4096 bf16    7.7 /  9.8   9.5 /  9.9  11.3 /  9.8  13.2 /  9.9  18.7 /  9.9    one
//   8192 bf16   11.2 / 14.6  13.9 / 14.7  16.6 / 14.7  19.3 / 14.7                 two
//   8192 fp32   12.9 / 11.8  16.6 / 11.9               23.9 / 11.9                 two, 1024 threads
// Where the host has no part in it, in a replayed graph, two launches would do better from three or four rows on; a
// single call that is waited for breaks even at four (4 x 4096 29.5 us and 29.7, 5 x 4096 31.7 and 30.1).
// (As many rows at a time as 1024 threads have room for, their sums joined in LDS: 16 x 512 10.4 us against 6.4 in two
// launches, 40 x 1000 30 against 8.2.)
static int one_workgroup_rows(int threads, int chunks) { return threads > 512 ? 2 : (chunks == 1 ? 5 : 4); }

// How a backward pass is launched; `parts` > 1 leave cols fp32 sums per kind each.
struct BackwardShape {
  int threads, chunks, parts;
  bool wide;                                  // for norm_columns_kernel
};
static BackwardShape backward_shape(int64_t rows, int cols, bool bf16) {
  BackwardShape s = {0, 0, 1, false};
  const int vec = bf16 ? 8 : 4;
  norm_shape(cols, vec, 512, s.threads, s.chunks);
  if (s.chunks > 2) {
    norm_shape(cols, vec, 1024, s.threads, s.chunks);
    // (two chunks of fp32 beside their sums fit 1024 threads' registers, of bf16, twice as many columns, do not)
    s.wide = bf16 || s.chunks > 2;
  }
  if (s.wide) {
    s.parts = (int)(rows < 128 ? rows : 128);
  } else if (rows > one_workgroup_rows(s.threads, s.chunks)) {
    const int64_t most = 256 * (int64_t)(s.threads <= 256 ? 512 / s.threads : 1);
    s.parts = (int)(rows < most ? rows : most);
  }
  return s;
}
static int64_t backward_sums(const BackwardShape& s, int64_t cols, int kinds) {
  return s.parts == 1 && !s.wide ? 0 : (int64_t)kinds * s.parts * cols;
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
  const int kinds = 1 + (f.out[1] != nullptr) + (f.out[2] != nullptr);
#define SMR_NORM_LAUNCH(C, USE, WHOLE, T, GRID)                                                                       \
  hipLaunchKernelGGL((norm_backward_kernel<BF16, C, USE, WHOLE, T>), dim3((unsigned)(GRID)), dim3(b.threads), 0, s, f)
  if (b.wide) {
    f.row_values = f.sums + backward_sums(b, f.cols, kinds);
    const int64_t cus = compute_units(), grid = f.rows < 2 * cus ? f.rows : 2 * cus;
    if constexpr (BF16) SMR_NORM_LAUNCH(2, kReread, false, 1024, grid);
    else SMR_NORM_LAUNCH(4, kReread, false, 1024, grid);
    const int rc = check_hip(hipGetLastError(), "smr_norm_backward launch");
    if (rc != 0) return rc;
    hipLaunchKernelGGL((norm_columns_kernel<BF16>), dim3((unsigned)((f.cols + 64 * V - 1) / (64 * V)), (unsigned)b.parts),
                       dim3(64), 0, s, f);
  } else if (b.threads > 512) {
    if constexpr (!BF16) SMR_NORM_LAUNCH(2, kKept, false, 1024, b.parts);
  } else if (b.chunks == 1 && whole) SMR_NORM_LAUNCH(1, kAhead, true, 512, b.parts);
  else if (b.chunks == 1) SMR_NORM_LAUNCH(1, kAhead, false, 512, b.parts);
  else if (whole) SMR_NORM_LAUNCH(2, kAhead, true, 512, b.parts);
  else SMR_NORM_LAUNCH(2, kAhead, false, 512, b.parts);
#undef SMR_NORM_LAUNCH
  const int rc = check_hip(hipGetLastError(), "smr_norm_backward launch");
  if (rc != 0 || (b.parts == 1 && !b.wide)) return rc;
  hipLaunchKernelGGL((norm_sums_kernel<BF16>), dim3((unsigned)((f.cols + 31) / 32), (unsigned)kinds), dim3(kSumThreads), 0,
                     s, f.sums, b.parts, f.cols, f.out[0], f.out[1], f.out[2]);
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
  const int kinds = 1 + (has_post_weight ? 1 : 0) + (gate_kind == kGateChannel ? 1 : 0);
  const BackwardShape b = backward_shape(rows, (int)cols, bf16);
  return (backward_sums(b, cols, kinds) + (b.wide ? rows * 3 : 0)) * 4;
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
                    scratch, nullptr, {grad_weight, nullptr, nullptr}, rows, (int)cols, gate_kind, (float)residual_scale, (float)eps};
  int kinds = 1;
  if (post_weight != nullptr) f.out[kinds++] = grad_post_weight;
  if (gate_kind == kGateChannel) f.out[kinds++] = grad_gate;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == SMR_DTYPE_BF16 ? launch_backward<true>(f, s) : launch_backward<false>(f, s);
}

}  // extern "C"
