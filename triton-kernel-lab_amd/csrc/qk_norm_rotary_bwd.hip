// Gradients of the norms of queries and keys with rotary positions (qk_norm_rotary.hip). Per row,
// with r = 1 / sqrt(mean(x^2) + eps) and dz = R^T dy (the rotation by the negative angle):
//   dw += dz x r (over the side's rows),  g = dz w,  dx = r (g - x r^2 mean(g x)).
// x and dy are read and dx written once; r is formed again from x rather than kept from the forward
// (the row is there in any case), and both of a row's sums are reduced together.
//
// dw: every workgroup walks its side's runs in a fixed order, sums in registers (a lane's features
// are the same in every row), folds its rows' lanes in LDS and writes one float32 row of partial
// sums; a second kernel adds those rows in a fixed order. Results do not depend on timing.
//
// Bound by HBM: 2 x 8192 tokens of 32 query and 8 KV heads, D128, bf16 (503 MB) 100 us with the second
// kernel's 4, 5 TB/s (104 in neighbouring pairs); 3 x 1000 tokens of 16 and 4 heads of 96 features, fp16
// (35 MB) 20 + 4 us. Measured and not kept: four workgroups per CU in 128 registers, which spill (135 us),
// runs twice as long (28 % more, the last round half empty) or half as long (6 % more, the angles' phases).
#include "qk_norm_rotary.hpp"

namespace tk_qk_norm {

template <typename T, int VEC, int NU, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void qk_norm_rotary_bwd_kernel(Args a) {
  using R = Row<T, VEC, NU, kInterleaved>;
  constexpr int PER = NU * R::N;    // sums per lane
  extern __shared__ float shared[];  // cos, sin of a run; then the lanes' sums
  const int w = blockIdx.x >= a.side[0].groups;
  const uint32_t group = blockIdx.x - (w ? a.side[0].groups : 0);
  const Side& s = a.side[w];
  float* cosv = shared;
  float* sinv = shared + s.block_tokens * a.half;

  const int lanes = 1 << a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const uint32_t step = kThreads >> a.lanes_log2;  // rows at a time
  const typename R::Layout layout(a, lane);
  typename R::Raw weight;
  weight.load(static_cast<const T*>(s.weight), layout);
  float sum[NU][R::N];
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int k = 0; k < R::N; ++k) sum[i][k] = 0.f;

  for (uint32_t j = group; j < s.runs; j += s.groups) {
    const Run run(a, s, j);
    uint32_t p = threadIdx.x >> a.lanes_log2;
    Run::At here;
    bool live = run.at(a, s, p, here);
    typename R::Raw x, dy;
    if (live) {
      x.load(static_cast<const T*>(s.x) + offset(s.xs, here), layout);
      dy.load(static_cast<const T*>(s.dy) + offset(s.ys, here), layout);
    }
    __syncthreads();  // the last run's angles have been read
    fill_angles(a, s, run.t0, cosv, sinv);
    __syncthreads();
    while (p < run.count) {
      float f[NU][R::N], d[NU][R::N], g[NU][R::N];
      x.expand(layout, f);
      dy.expand(layout, d);
      // The next row's loads take the registers that this one's have left.
      __builtin_amdgcn_sched_barrier(0);
      Run::At next;
      const bool next_live = run.at(a, s, p + step, next);
      if (next_live) {
        x.load(static_cast<const T*>(s.x) + offset(s.xs, next), layout);
        dy.load(static_cast<const T*>(s.dy) + offset(s.ys, next), layout);
      }
      weight.expand(layout, g);
      float square = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        if (layout.angle[i] >= 0 && live) {
          const int at = here.token * a.half + layout.angle[i];
#pragma unroll
          for (int k = 0; k < R::PAIRS; ++k) {
            const float c = cosv[at + k], sn = sinv[at + k];
            const float d1 = d[i][R::first(k)], d2 = d[i][R::second(k)];
            d[i][R::first(k)] = d1 * c + d2 * sn;
            d[i][R::second(k)] = d2 * c - d1 * sn;
          }
        }
#pragma unroll
        for (int k = 0; k < R::N; ++k) {
          square = fmaf(f[i][k], f[i][k], square);
          dot = fmaf(d[i][k] * g[i][k], f[i][k], dot);
        }
      }
      square = row_sum(square, a.lanes_log2);
      dot = row_sum(dot, a.lanes_log2);
      const float inverse = 1.0f / sqrtf(fmaf(square, a.inv_dim, a.eps));
      const float share = dot * inverse * inverse * a.inv_dim;
      if (live) {
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
          for (int k = 0; k < R::N; ++k) {
            sum[i][k] = fmaf(d[i][k], f[i][k] * inverse, sum[i][k]);
            f[i][k] = inverse * (d[i][k] * g[i][k] - f[i][k] * share);
          }
        R::store(static_cast<T*>(s.out) + offset(s.os, here), layout, f);
      }
      live = next_live;
      here = next;
      p += step;
    }
  }

  __syncthreads();
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int k = 0; k < R::N; ++k) shared[threadIdx.x * PER + i * R::N + k] = sum[i][k];
  __syncthreads();
  float* out = a.partials + int64_t(blockIdx.x) * a.head_dim;
  for (int e = threadIdx.x; e < lanes * PER; e += kThreads) {
    const int owner = e / PER, i = e % PER / R::N, k = e % R::N;
    const typename R::Layout at(a, owner);
    int col = -1;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      if (n != i || at.col[n] < 0) continue;
      if (!R::TWO || k < VEC)
        col = at.col[n] + k;
      else if (at.angle[n] >= 0)
        col = at.col[n] + at.gap + k - VEC;
    }
    if (col < 0) continue;
    float v = 0.f;
    for (uint32_t row = 0; row < step; ++row) v += shared[row * lanes * PER + e];
    out[col] = v;
  }
}

// Sums of the partial rows: 8 features by 128 slices of the rows a workgroup, so that a thread adds a
// handful of rows (32 features by 32 slices: 9.9 us, the loads one behind the other, where the partial rows
// were 1023; now they are kGroups at most).
constexpr int kCols = 8, kSlices = 128;
template <typename T>
__global__ __launch_bounds__(kCols* kSlices) void qk_norm_weight_kernel(Args a) {
  __shared__ float part[kSlices][kCols];
  const int w = blockIdx.y;
  const Side& s = a.side[w];
  const int c = threadIdx.x % kCols, col = blockIdx.x * kCols + c, slice = threadIdx.x / kCols;
  const float* rows = a.partials + (w ? int64_t(a.side[0].groups) * a.head_dim : 0);
  float v = 0.f;
  if (col < a.head_dim)
#pragma unroll 8
    for (uint32_t r = slice; r < s.groups; r += kSlices) v += rows[int64_t(r) * a.head_dim + col];
  part[slice][c] = v;
#pragma unroll
  for (int half = kSlices / 2; half > 0; half /= 2) {
    __syncthreads();
    if (slice < half) part[slice][c] += part[slice + half][c];
  }
  if (slice == 0 && col < a.head_dim) static_cast<T*>(s.dweight)[col] = tk::from_f32<T>(part[0][c]);
}

template <typename T, int VEC, int NU>
static void launch(const Args& a, bool interleaved, hipStream_t s) {
  const int block_tokens = a.side[0].block_tokens > a.side[1].block_tokens ? a.side[0].block_tokens
                                                                           : a.side[1].block_tokens;
  size_t lds = static_cast<size_t>(block_tokens) * a.half * 2 * sizeof(float);
  const size_t sums = sizeof(float) * kThreads * NU * Row<T, VEC, NU, false>::N;
  if (lds < sums) lds = sums;
  const dim3 grid(a.side[0].groups + a.side[1].groups);
  if (interleaved)
    hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<T, VEC, NU, true>), grid, dim3(kThreads), lds, s, a);
  else if constexpr (VEC * NU < 16)  // (two units of 8 are of the interleaved layout)
    hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<T, VEC, NU, false>), grid, dim3(kThreads), lds, s, a);
}

template <typename T>
static void launch_all(int vec, int nu, const Args& a, bool interleaved, hipStream_t s) {
#define TK_LAUNCH(T, V, N) launch<T, V, N>(a, interleaved, s)
  TK_QK_NORM_VARIANTS(T, vec, nu, TK_LAUNCH)
#undef TK_LAUNCH
  hipLaunchKernelGGL((qk_norm_weight_kernel<T>),
                     dim3(static_cast<uint32_t>(tk::cdiv(a.head_dim, kCols)), a.side[1].groups ? 2 : 1),
                     dim3(kCols * kSlices), 0, s, a);
}

// Workgroups of each side, kGroups in all at most: as few rounds of runs as that allows, where a run
// costs its rows and, a quarter of a row for each, its angles per thread. (A run of 8 heads has four
// times the angles of one of 32: B2 N8192 Hq32 Hkv8 106.6 us with workgroups by runs alone, 99.8 so.)
static void share_groups(Args& a) {
  int64_t cost[2], all = 0;
  for (int w = 0; w < 2; ++w) {
    const Side& s = a.side[w];
    const int64_t step = kThreads >> a.lanes_log2;
    cost[w] = 16 * tk::cdiv(int64_t(s.block_tokens) * s.block_heads.d, step) +
              4 * int64_t(s.block_tokens) * a.half / kThreads;
    all += cost[w] * s.runs;
  }
  int64_t most = all / kGroups;  // a workgroup's share, if it came out even
  for (;;) {
    int64_t groups = 0, next = INT64_MAX;
    for (int w = 0; w < 2; ++w) {
      Side& s = a.side[w];
      const int64_t rounds = most / cost[w] > 1 ? most / cost[w] : 1;
      s.groups = static_cast<uint32_t>(tk::cdiv(s.runs, rounds));
      groups += s.groups;
      if (next > (rounds + 1) * cost[w]) next = (rounds + 1) * cost[w];
    }
    if (groups <= kGroups) return;
    most = next;
  }
}

}  // namespace tk_qk_norm

extern "C" int tk_qk_norm_rotary_bwd(
    int dtype, const void* q, const void* dq_out, void* dq, const void* k, const void* dk_out,
    void* dk, const void* q_weight, const void* k_weight, void* dq_weight, void* dk_weight,
    float* partials, const void* positions, const double* frequencies, int64_t batch,
    int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
    const int64_t* q_strides, const int64_t* dq_out_strides, const int64_t* dq_strides,
    const int64_t* k_strides, const int64_t* dk_out_strides, const int64_t* dk_strides,
    const int64_t* position_strides, float eps, float magnitude, int interleaved,
    int wide_positions, void* stream) {
  using namespace tk_qk_norm;
  const void* pointers[2][4] = {{q, dq_out, dq, q_weight}, {k, dk_out, dk, k_weight}};
  const Tables tables[2] = {{q_strides, dq_out_strides, dq_strides},
                            {k_strides, dk_out_strides, dk_strides}};
  if (tk::valid_dtype(dtype) && (dq_out_strides == nullptr || partials == nullptr ||
                                 dq_weight == nullptr || (k != nullptr && dk_weight == nullptr)))
    return tk::fail("qk norm: null pointer");
  Args a;
  int vec, nu;
  if (plan(dtype, pointers, tables, positions, frequencies, batch, tokens, q_heads, kv_heads,
           head_dim, rotary_dim, position_strides, eps, magnitude, interleaved, wide_positions, a,
           vec, nu))
    return 1;
  if (reinterpret_cast<uintptr_t>(partials) % 4 != 0)
    return tk::fail("qk norm: tensors must be aligned to their dtype");
  for (const void* p : {dq_weight, k != nullptr ? dk_weight : dq_weight})
    if (reinterpret_cast<uintptr_t>(p) % tk::elem_size(dtype) != 0)
      return tk::fail("qk norm: tensors must be aligned to their dtype");
  a.partials = partials;
  a.side[0].dweight = dq_weight;
  a.side[1].dweight = k != nullptr ? dk_weight : dq_weight;
  share_groups(a);
  hipStream_t s = tk::as_stream(stream);
  switch (dtype) {
    case TK_DTYPE_F32: launch_all<float>(vec, nu, a, interleaved != 0, s); break;
    case TK_DTYPE_F16: launch_all<_Float16>(vec, nu, a, interleaved != 0, s); break;
    default: launch_all<__bf16>(vec, nu, a, interleaved != 0, s); break;
  }
  return tk::check_launch("qk norm backward");
}
