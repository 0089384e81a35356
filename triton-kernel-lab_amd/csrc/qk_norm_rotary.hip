// Norms of queries and keys for each head with rotary positions in the same pass:
//   z = x w / sqrt(mean(x^2) + eps),  y = R z,
// R the rotation of rotary.hip over the first rotary_dim features. x is read and y written once;
// everything between is float32 in registers. Rows and lanes: qk_norm_rotary.hpp.
//
// Bound by HBM: 2 x 8192 tokens of 32 query and 8 KV heads, D128, bf16 (336 MB) 61 us, 5.5 TB/s (65 in
// neighbouring pairs), of which the angles' arithmetic costs 3; 3 x 1000 tokens of 16 and 4 heads of 96
// features, 48 of them turned, fp16 (23 MB) 10 us; one token 3.3 us.
#include "qk_norm_rotary.hpp"

namespace tk_qk_norm {

template <typename T, int VEC, int NU, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void qk_norm_rotary_kernel(Args a) {
  using R = Row<T, VEC, NU, kInterleaved>;
  extern __shared__ float table[];  // cos[block_tokens * half], then sin
  uint32_t j = blockIdx.z * gridDim.x + blockIdx.x;
  if (j >= a.side[0].runs + a.side[1].runs) return;
  const int w = j >= a.side[0].runs;
  if (w) j -= a.side[0].runs;
  const Side& s = a.side[w];
  const Run run(a, s, j);
  float* cosv = table;
  float* sinv = table + s.block_tokens * a.half;

  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1);
  const uint32_t step = kThreads >> a.lanes_log2;  // rows at a time
  const typename R::Layout layout(a, lane);
  uint32_t p = threadIdx.x >> a.lanes_log2;
  Run::At here;
  bool live = run.at(a, s, p, here);
  typename R::Raw raw, weight;
  weight.load(static_cast<const T*>(s.weight), layout);
  if (live) raw.load(static_cast<const T*>(s.x) + offset(s.xs, here), layout);
  fill_angles(a, s, run.t0, cosv, sinv);
  __syncthreads();
  float g[NU][R::N];
  weight.expand(layout, g);

  while (p < run.count) {
    Run::At next;
    typename R::Raw ahead;
    const bool next_live = run.at(a, s, p + step, next);
    if (next_live) ahead.load(static_cast<const T*>(s.x) + offset(s.xs, next), layout);
    float f[NU][R::N];
    raw.expand(layout, f);
    float square = 0.f;
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int k = 0; k < R::N; ++k) square = fmaf(f[i][k], f[i][k], square);
    square = row_sum(square, a.lanes_log2);
    const float inverse = 1.0f / sqrtf(fmaf(square, a.inv_dim, a.eps));
#pragma unroll
    for (int i = 0; i < NU; ++i) {
#pragma unroll
      for (int k = 0; k < R::N; ++k) f[i][k] = f[i][k] * inverse * g[i][k];
      if (layout.angle[i] >= 0 && live) {
        const int at = here.token * a.half + layout.angle[i];
#pragma unroll
        for (int k = 0; k < R::PAIRS; ++k) {
          const float c = cosv[at + k], sn = sinv[at + k];
          const float x1 = f[i][R::first(k)], x2 = f[i][R::second(k)];
          f[i][R::first(k)] = x1 * c - x2 * sn;
          f[i][R::second(k)] = x2 * c + x1 * sn;
        }
      }
    }
    if (live) R::store(static_cast<T*>(s.out) + offset(s.os, here), layout, f);
    raw = ahead;
    live = next_live;
    here = next;
    p += step;
  }
}

// Largest power of two up to `most` that divides every value.
static int common_vector(int most, std::initializer_list<int64_t> values) {
  int v = most;
  for (int64_t x : values)
    while (v > 1 && x % v != 0) v >>= 1;
  return v;
}

int plan(int dtype, const void* const pointers[2][4], const Tables tables[2], const void* positions,
         const double* frequencies, int64_t batch, int64_t tokens, int64_t q_heads,
         int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, const int64_t* position_strides,
         float eps, float magnitude, int interleaved, int wide_positions, Args& a, int& vec,
         int& units_per_lane) {
  if (!tk::valid_dtype(dtype)) return tk::fail("unsupported dtype code %d", dtype);
  if (positions == nullptr || frequencies == nullptr || position_strides == nullptr)
    return tk::fail("qk norm: null pointer");
  const bool with_k = pointers[1][0] != nullptr;
  for (int w = 0; w < (with_k ? 2 : 1); ++w) {
    const Tables& t = tables[w];
    const bool backward = tables[0].dy != nullptr;
    if (pointers[w][0] == nullptr || pointers[w][2] == nullptr || pointers[w][3] == nullptr ||
        t.x == nullptr || t.out == nullptr ||
        (backward && (pointers[w][1] == nullptr || t.dy == nullptr)))
      return tk::fail("qk norm: null pointer");
  }
  if (batch <= 0 || tokens <= 0 || q_heads <= 0 || (with_k && kv_heads <= 0))
    return tk::fail("qk norm: empty problem");
  if (head_dim <= 0 || head_dim > kMaxHeadDim)
    return tk::fail("qk norm: head_dim must be 1 to %d", kMaxHeadDim);
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return tk::fail("qk norm: rotary_dim must be even, positive and at most head_dim");
  int64_t total;
  if (__builtin_mul_overflow(batch, tokens, &total) || total > INT32_MAX - 65536 ||
      q_heads > 65535 || (with_k && kv_heads > 65535))
    return tk::fail("qk norm: problem too large");
  const int size = tk::elem_size(dtype);
  vec = 16 / size;
  for (int w = 0; w < 2; ++w) {
    Side& s = a.side[w];
    const int from = w && !with_k ? 0 : w;
    s.heads = static_cast<int>(w ? kv_heads : q_heads);
    s.x = pointers[from][0];
    s.dy = pointers[from][1];
    s.out = const_cast<void*>(pointers[from][2]);
    s.weight = pointers[from][3];
    for (int d = 0; d < 3; ++d) s.xs[d] = s.ys[d] = s.os[d] = 0;
    if (from != w) continue;
    const int64_t* rows[3] = {tables[w].x, tables[w].dy, tables[w].out};
    int64_t* into[3] = {s.xs, s.ys, s.os};
    for (int i = 0; i < 3; ++i) {
      if (rows[i] == nullptr) continue;
      __int128 last = head_dim;
      const int64_t counts[3] = {batch, s.heads, tokens};
      for (int d = 0; d < 3; ++d) {
        if (rows[i][d] < 0) return tk::fail("qk norm: strides must be non-negative");
        last += static_cast<__int128>(counts[d] - 1) * rows[i][d];
        into[i][d] = rows[i][d];
        if (counts[d] > 1) vec = common_vector(vec, {rows[i][d]});
      }
      if (last >= (static_cast<__int128>(1) << 52))
        return tk::fail("qk norm: strides must keep rows in range");
    }
    for (int i = 0; i < 4; ++i) {
      const uintptr_t base = reinterpret_cast<uintptr_t>(pointers[w][i]);
      if (base % size != 0) return tk::fail("qk norm: tensors must be aligned to their dtype");
      vec = common_vector(vec, {static_cast<int64_t>(base / size)});
    }
  }
  for (int d = 0; d < 2; ++d)
    if (position_strides[d] < 0) return tk::fail("qk norm: strides must be non-negative");
  if (static_cast<__int128>(batch - 1) * position_strides[0] +
          static_cast<__int128>(tokens - 1) * position_strides[1] >=
      (static_cast<__int128>(1) << 52))
    return tk::fail("qk norm: strides must keep rows in range");
  if (!(eps >= 0.f)) return tk::fail("qk norm: eps must be non-negative");

  const int half = static_cast<int>(rotary_dim / 2);
  // Vectors may not cross the end of a half, of the rotated part or of the head.
  vec = common_vector(vec, {interleaved ? rotary_dim : half, head_dim - rotary_dim});
  a.rotated_units = interleaved && vec > 1 ? int(rotary_dim) / vec : half / (interleaved ? 1 : vec);
  a.units = a.rotated_units + int(head_dim - rotary_dim) / vec;
  a.lanes_log2 = 0;
  // Full vectors of the interleaved layout, which hold half the features of a unit of two, go two to a
  // lane (D128 with one: forward 71 us, backward 120; with two 65 and 104).
  const int per_lane = interleaved && vec * size == 16 ? 2 : 1;
  while ((per_lane << a.lanes_log2) < a.units && a.lanes_log2 < 6) ++a.lanes_log2;
  units_per_lane = (a.units + (1 << a.lanes_log2) - 1) >> a.lanes_log2;
  a.positions = positions;
  a.frequencies = frequencies;
  a.partials = nullptr;
  a.pos_b = position_strides[0];
  a.pos_n = position_strides[1];
  a.tokens = tk::FastDiv(static_cast<uint32_t>(tokens));
  a.total_tokens = static_cast<int>(total);
  a.head_dim = static_cast<int>(head_dim);
  a.half = half;
  a.eps = eps;
  a.magnitude = magnitude;
  a.inv_dim = 1.0f / static_cast<float>(head_dim);
  a.pos64 = wide_positions;

  // A lane takes about four rows where the side has enough of them for 1024 workgroups of that
  // size, otherwise one.
  for (int w = 0; w < 2; ++w) {
    Side& s = a.side[w];
    if (w && !with_k) {
      s.runs = 0;
      s.heads = 0;
      s.block_tokens = 1;
      s.block_heads = s.head_runs = tk::FastDiv(1);
      continue;
    }
    const int64_t step = kThreads >> a.lanes_log2;
    const int64_t rows = total * s.heads >= 1024 * 4 * step ? 4 * step : step;
    int64_t block_tokens = 1, block_heads = s.heads;
    if (s.heads <= rows) {
      block_tokens = rows / s.heads;
      const int64_t most = kMaxAngles / half > 1 ? kMaxAngles / half : 1;
      if (block_tokens > most) block_tokens = most;
      if (block_tokens > total) block_tokens = total;
    } else {
      block_heads = rows;
    }
    const int64_t head_runs = tk::cdiv(s.heads, block_heads);
    const int64_t runs = tk::cdiv(total, block_tokens) * head_runs;
    if (runs > INT32_MAX / 2) return tk::fail("qk norm: problem too large");
    s.block_tokens = static_cast<int>(block_tokens);
    s.block_heads = tk::FastDiv(static_cast<uint32_t>(block_heads));
    s.head_runs = tk::FastDiv(static_cast<uint32_t>(head_runs));
    s.runs = static_cast<uint32_t>(runs);
  }
  return 0;
}

template <typename T, int VEC, int NU>
static void launch(const Args& a, bool interleaved, dim3 grid, size_t lds, hipStream_t s) {
  if (interleaved)
    hipLaunchKernelGGL((qk_norm_rotary_kernel<T, VEC, NU, true>), grid, dim3(kThreads), lds, s, a);
  else if constexpr (VEC * NU < 16)  // (two units of 8 are of the interleaved layout)
    hipLaunchKernelGGL((qk_norm_rotary_kernel<T, VEC, NU, false>), grid, dim3(kThreads), lds, s, a);
}

template <typename T>
static void launch_vec(int vec, int nu, const Args& a, bool interleaved, dim3 grid, size_t lds,
                       hipStream_t s) {
#define TK_LAUNCH(T, V, N) launch<T, V, N>(a, interleaved, grid, lds, s)
  TK_QK_NORM_VARIANTS(T, vec, nu, TK_LAUNCH)
#undef TK_LAUNCH
}

}  // namespace tk_qk_norm

extern "C" int tk_qk_norm_rotary(int dtype, const void* q, void* q_out, const void* k, void* k_out,
                                 const void* q_weight, const void* k_weight, const void* positions,
                                 const double* frequencies, int64_t batch, int64_t tokens,
                                 int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                 int64_t rotary_dim, const int64_t* q_strides,
                                 const int64_t* q_out_strides, const int64_t* k_strides,
                                 const int64_t* k_out_strides, const int64_t* position_strides,
                                 float eps, float magnitude, int interleaved, int wide_positions,
                                 void* stream) {
  using namespace tk_qk_norm;
  const void* pointers[2][4] = {{q, nullptr, q_out, q_weight}, {k, nullptr, k_out, k_weight}};
  const Tables tables[2] = {{q_strides, nullptr, q_out_strides}, {k_strides, nullptr, k_out_strides}};
  Args a;
  int vec, nu;
  if (plan(dtype, pointers, tables, positions, frequencies, batch, tokens, q_heads, kv_heads,
           head_dim, rotary_dim, position_strides, eps, magnitude, interleaved, wide_positions, a,
           vec, nu))
    return 1;
  // A launch holds fewer than 2^32 threads in each dimension, so the runs spread over two.
  const int64_t runs = int64_t(a.side[0].runs) + a.side[1].runs;
  const int64_t layers = tk::cdiv(runs, (int64_t(1) << 24) - 1);
  const dim3 grid(static_cast<uint32_t>(tk::cdiv(runs, layers)), 1, static_cast<uint32_t>(layers));
  const int block_tokens = a.side[0].block_tokens > a.side[1].block_tokens ? a.side[0].block_tokens
                                                                           : a.side[1].block_tokens;
  const size_t lds = static_cast<size_t>(block_tokens) * a.half * 2 * sizeof(float);
  hipStream_t s = tk::as_stream(stream);
  switch (dtype) {
    case TK_DTYPE_F32: launch_vec<float>(vec, nu, a, interleaved != 0, grid, lds, s); break;
    case TK_DTYPE_F16: launch_vec<_Float16>(vec, nu, a, interleaved != 0, grid, lds, s); break;
    default: launch_vec<__bf16>(vec, nu, a, interleaved != 0, grid, lds, s); break;
  }
  return tk::check_launch("qk norm");
}
