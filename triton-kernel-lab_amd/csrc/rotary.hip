// Rotary positions for the queries and keys of one call: every pair of the first rotary_dim
// features is turned by position * frequency[pair] radians and multiplied by `magnitude`, the
// features behind them are copied:
//   y1 = m (x1 cos a - x2 sin a),  y2 = m (x2 cos a + x1 sin a),
// with the pair (i, i + rotary_dim / 2) (halves) or (2i, 2i + 1) (interleaved). The rotation is
// orthogonal up to m, so the gradient is the same kernel with -a (`inverse`).
//
// Angles: position * frequency is formed in float64 and reduced modulo pi/2 there (at position
// 10^6 a float32 angle is off by up to 0.03 rad); sine and cosine of the reduced angle are the
// Taylor series in float64, cut where the next term is below 2e-10, and rounded to float32.
// One (token, pair) angle serves every head, so a workgroup takes whole tokens (or, when few
// tokens would leave CUs idle, a run of one token's heads), evaluates their angles once into
// LDS, one per thread, and then streams the rows. The first rows are requested before the
// angles are formed, so the two latencies overlap.
//
// Bound by HBM: q and k are read and written once. B2 N8192 Hq32 Hkv8 D128 bf16 (336 MB a pass):
// 60 us, 5.6 TB/s, with about four units a thread and non-temporal accesses; two units 65 us, eight
// 66, plain loads 64. One token of the same heads: 2.9 us.
#include "tk_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 1024;
constexpr int kMaxAngles = 2048;  // per workgroup: 16 KiB of LDS, so LDS never limits residency

struct RotaryArgs {
  const void* src[2];   // q, k
  void* dst[2];
  const void* positions;
  const double* frequencies;
  int64_t ss[2][3], ds[2][3];  // source and destination strides {batch, head, token}
  int64_t pos_b, pos_n;
  tk::FastDiv tokens;       // tokens per batch entry
  tk::FastDiv units;        // vector units per head row
  tk::FastDiv block_heads;  // heads per workgroup
  int total_tokens, heads[2], half, rotated_units;
  int block_tokens;
  float magnitude;
  int pos64, inverse;
};

// sin and cos of r in [-pi/4, pi/4] by their Taylor series (coefficients 1/n!).
__device__ __forceinline__ void sincos_reduced(double r, double& s, double& c) {
  const double z = r * r;
  double p = -1.0 / 39916800.0;
  p = fma(p, z, 1.0 / 362880.0);
  p = fma(p, z, -1.0 / 5040.0);
  p = fma(p, z, 1.0 / 120.0);
  p = fma(p, z, -1.0 / 6.0);
  s = fma(p * z, r, r);
  double q = 1.0 / 479001600.0;
  q = fma(q, z, -1.0 / 3628800.0);
  q = fma(q, z, 1.0 / 40320.0);
  q = fma(q, z, -1.0 / 720.0);
  q = fma(q, z, 1.0 / 24.0);
  q = fma(q, z, -0.5);
  c = fma(q, z, 1.0);
}

// Features of one unit: a rotated unit of the halves layout is VEC pairs (two vectors), one of
// the interleaved layout a vector of VEC / 2 pairs (a single pair for VEC 1); a unit past the
// rotated ones is VEC copied features.
template <typename T, int VEC, bool kInterleaved>
struct Unit {
  static constexpr int PAIRS = kInterleaved ? (VEC + 1) / 2 : VEC;
  static constexpr int N = 2 * PAIRS;  // values held
  const T* src;
  T* dst;
  int angle;  // LDS index of the unit's first angle, -1: copied
  float v[N];

  __device__ __forceinline__ void locate(const RotaryArgs& a, int t0, int h0, uint32_t idx,
                                         bool& live) {
    const uint32_t p = a.units.div(idx);
    const int u = int(idx - p * a.units.d);
    const uint32_t tl = a.block_heads.div(p);
    int h = h0 + int(p - tl * a.block_heads.d);
    const int t = t0 + int(tl);
    live = int(tl) < a.block_tokens && t < a.total_tokens && h < a.heads[0] + a.heads[1];
    if (!live) return;
    const int w = h >= a.heads[0];
    if (w) h -= a.heads[0];
    const uint32_t b = a.tokens.div(t);
    const int64_t n = t - int64_t(b) * a.tokens.d;
    const bool turned = u < a.rotated_units;
    int col;
    if (turned) {
      col = (kInterleaved ? N : VEC) * u;
      angle = int(tl) * a.half + PAIRS * u;
    } else {
      col = 2 * a.half + VEC * (u - a.rotated_units);
      angle = -1;
    }
    src = static_cast<const T*>(a.src[w]) + b * a.ss[w][0] + h * a.ss[w][1] + n * a.ss[w][2] + col;
    dst = static_cast<T*>(a.dst[w]) + b * a.ds[w][0] + h * a.ds[w][1] + n * a.ds[w][2] + col;
  }

  __device__ __forceinline__ void load(const RotaryArgs& a) {
    if constexpr (kInterleaved && VEC > 1) {
      tk::load_vec_stream<T, VEC>(src, v);
    } else if constexpr (kInterleaved) {
      v[0] = tk::to_f32(src[0]);
      if (angle >= 0) v[1] = tk::to_f32(src[1]);
    } else {
      tk::load_vec_stream<T, VEC>(src, v);
      if (angle >= 0) tk::load_vec_stream<T, VEC>(src + a.half, v + VEC);
    }
  }

  __device__ __forceinline__ void finish(const RotaryArgs& a, const float* cosv,
                                         const float* sinv) {
    if (angle >= 0) {
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const float c = cosv[angle + j], s = sinv[angle + j];
        const int i1 = kInterleaved ? 2 * j : j, i2 = kInterleaved ? 2 * j + 1 : j + VEC;
        const float x1 = v[i1], x2 = v[i2];
        v[i1] = x1 * c - x2 * s;
        v[i2] = x2 * c + x1 * s;
      }
    }
    if constexpr (kInterleaved && VEC > 1) {
      tk::store_vec_stream<T, VEC>(dst, v);
    } else if constexpr (kInterleaved) {
      dst[0] = tk::from_f32<T>(v[0]);
      if (angle >= 0) dst[1] = tk::from_f32<T>(v[1]);
    } else {
      tk::store_vec_stream<T, VEC>(dst, v);
      if (angle >= 0) tk::store_vec_stream<T, VEC>(dst + a.half, v + VEC);
    }
  }
};

template <typename T, int VEC, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float table[];  // cos[block_tokens * half], then sin
  const int t0 = int(blockIdx.z * gridDim.x + blockIdx.x) * a.block_tokens;
  const int h0 = blockIdx.y * int(a.block_heads.d);
  const int angles = a.block_tokens * a.half;
  const uint32_t count = a.units.d * a.block_heads.d * uint32_t(a.block_tokens);
  float* cosv = table;
  float* sinv = table + angles;

  using U = Unit<T, VEC, kInterleaved>;
  U unit;
  bool live = false;
  uint32_t idx = threadIdx.x;
  if (idx < count) {
    unit.locate(a, t0, h0, idx, live);
    if (live) unit.load(a);
  }

  for (int i = threadIdx.x; i < angles; i += kThreads) {
    const int tl = i / a.half;
    const int pair = i - tl * a.half;
    const int t = t0 + tl;
    if (t >= a.total_tokens) break;
    const uint32_t b = a.tokens.div(t);
    const int64_t at = b * a.pos_b + (t - int64_t(b) * a.tokens.d) * a.pos_n;
    const double pos = a.pos64 ? double(static_cast<const int64_t*>(a.positions)[at])
                               : double(static_cast<const int32_t*>(a.positions)[at]);
    const double x = pos * a.frequencies[pair];
    // x = k pi/2 + r; pi/2 in two parts, the first with all 53 bits. Past 2^51 the rounding of
    // x * 2/pi is off by whole quarter turns: the second pass takes off those that are left.
    const double k = rint(x * 0.63661977236758134308);
    double r = fma(k, -1.5707963267948965580, x);
    r = fma(k, -6.1232339957367658e-17, r);
    const double more = rint(r * 0.63661977236758134308);
    r = fma(more, -1.5707963267948965580, r);
    r = fma(more, -6.1232339957367658e-17, r);
    double s, c;
    sincos_reduced(r, s, c);
    // k modulo 4 is exact for every finite k.
    const int quarter = int(k - 4.0 * floor(0.25 * k)) + int(more);
    if (quarter & 1) {
      const double swap = s;
      s = c;
      c = -swap;
    }
    if (quarter & 2) {
      s = -s;
      c = -c;
    }
    const double m = a.magnitude;
    cosv[i] = float(c * m);
    sinv[i] = float(a.inverse ? -s * m : s * m);
  }
  __syncthreads();

  while (idx < count) {
    const uint32_t next = idx + kThreads;
    U ahead;
    bool ahead_live = false;
    if (next < count) {
      ahead.locate(a, t0, h0, next, ahead_live);
      if (ahead_live) ahead.load(a);
    }
    if (live) unit.finish(a, cosv, sinv);
    unit = ahead;
    live = ahead_live;
    idx = next;
  }
}

// Largest power of two up to `most` that divides every value.
int common_vector(int most, std::initializer_list<int64_t> values) {
  int v = most;
  for (int64_t x : values)
    while (v > 1 && x % v != 0) v >>= 1;
  return v;
}

template <typename T, int VEC>
void launch(const RotaryArgs& a, bool interleaved, dim3 grid, size_t lds, hipStream_t s) {
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<T, VEC, true>), grid, dim3(kThreads), lds, s, a);
  else
    hipLaunchKernelGGL((rotary_kernel<T, VEC, false>), grid, dim3(kThreads), lds, s, a);
}

template <typename T>
void launch_vec(int vec, const RotaryArgs& a, bool interleaved, dim3 grid, size_t lds,
                hipStream_t s) {
  switch (vec) {
    case 8:
      if constexpr (sizeof(T) == 2) launch<T, 8>(a, interleaved, grid, lds, s);
      break;
    case 4: launch<T, 4>(a, interleaved, grid, lds, s); break;
    case 2: launch<T, 2>(a, interleaved, grid, lds, s); break;
    default: launch<T, 1>(a, interleaved, grid, lds, s); break;
  }
}

}  // namespace

extern "C" int tk_rotary(int dtype, const void* q, void* q_out, const void* k, void* k_out,
                         const void* positions, const double* frequencies, int64_t batch,
                         int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                         int64_t rotary_dim, const int64_t* q_strides,
                         const int64_t* q_out_strides, const int64_t* k_strides,
                         const int64_t* k_out_strides, const int64_t* position_strides,
                         float magnitude, int interleaved, int wide_positions, int inverse,
                         void* stream) {
  if (!tk::valid_dtype(dtype)) return tk::fail("unsupported dtype code %d", dtype);
  if (q == nullptr || q_out == nullptr || positions == nullptr || frequencies == nullptr ||
      q_strides == nullptr || q_out_strides == nullptr || position_strides == nullptr)
    return tk::fail("rotary: null pointer");
  const bool with_k = k != nullptr;
  if (with_k && (k_out == nullptr || k_strides == nullptr || k_out_strides == nullptr))
    return tk::fail("rotary: null pointer");
  if (batch <= 0 || tokens <= 0 || q_heads <= 0 || (with_k && kv_heads <= 0))
    return tk::fail("rotary: empty problem");
  if (head_dim <= 0 || head_dim > kMaxHeadDim)
    return tk::fail("rotary: head_dim must be 1 to %d", kMaxHeadDim);
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return tk::fail("rotary: rotary_dim must be even, positive and at most head_dim");
  const int64_t heads = q_heads + (with_k ? kv_heads : 0);
  int64_t total;
  if (__builtin_mul_overflow(batch, tokens, &total) || total > INT32_MAX - 65536 ||
      heads > 65535)
    return tk::fail("rotary: problem too large");

  RotaryArgs a;
  a.src[0] = q;
  a.dst[0] = q_out;
  a.src[1] = with_k ? k : q;
  a.dst[1] = with_k ? k_out : q_out;
  const int64_t* tables[2][2] = {{q_strides, q_out_strides},
                                 {with_k ? k_strides : q_strides,
                                  with_k ? k_out_strides : q_out_strides}};
  const int size = tk::elem_size(dtype);
  int vec = 16 / size;
  for (int w = 0; w < (with_k ? 2 : 1); ++w) {
    for (int io = 0; io < 2; ++io) {
      const int64_t* st = tables[w][io];
      int64_t* out = io ? a.ds[w] : a.ss[w];
      __int128 last = head_dim;
      const int64_t counts[3] = {batch, w ? kv_heads : q_heads, tokens};
      for (int d = 0; d < 3; ++d) {
        if (st[d] < 0) return tk::fail("rotary: strides must be non-negative");
        last += static_cast<__int128>(counts[d] - 1) * st[d];
        out[d] = st[d];
        if (counts[d] > 1) vec = common_vector(vec, {st[d]});
      }
      if (last >= (static_cast<__int128>(1) << 52))
        return tk::fail("rotary: strides must keep rows in range");
      const uintptr_t base = reinterpret_cast<uintptr_t>(io ? a.dst[w] : a.src[w]);
      if (base % size != 0) return tk::fail("rotary: tensors must be aligned to their dtype");
      vec = common_vector(vec, {static_cast<int64_t>(base / size)});
    }
  }
  for (int d = 0; d < 2; ++d)
    if (position_strides[d] < 0) return tk::fail("rotary: strides must be non-negative");
  if (static_cast<__int128>(batch - 1) * position_strides[0] +
          static_cast<__int128>(tokens - 1) * position_strides[1] >=
      (static_cast<__int128>(1) << 52))
    return tk::fail("rotary: strides must keep rows in range");
  if (!with_k)
    for (int d = 0; d < 3; ++d) a.ss[1][d] = a.ds[1][d] = 0;

  const int half = static_cast<int>(rotary_dim / 2);
  // Vectors may not cross the end of a half, of the rotated part or of the head.
  vec = common_vector(vec, {interleaved ? rotary_dim : half, head_dim - rotary_dim});
  const int rotated = interleaved && vec > 1 ? int(rotary_dim) / vec : half / (interleaved ? 1 : vec);
  const int copied = int(head_dim - rotary_dim) / vec;
  const int units = rotated + copied;

  // A thread takes about four units where the call has enough of them for 1024 workgroups of
  // that size, otherwise one.
  const int64_t all = total * heads * units;
  const int64_t target = all >= int64_t(1024) * 4 * kThreads ? 4 * kThreads : kThreads;
  int64_t block_tokens = 1, block_heads = heads;
  if (heads * units <= target) {
    block_tokens = target / (heads * units);
    const int64_t most = kMaxAngles / half > 1 ? kMaxAngles / half : 1;
    if (block_tokens > most) block_tokens = most;
    if (block_tokens > total) block_tokens = total;
  } else {
    block_heads = target / units > 1 ? target / units : 1;
    if (block_heads > heads) block_heads = heads;
  }
  a.positions = positions;
  a.frequencies = frequencies;
  a.pos_b = position_strides[0];
  a.pos_n = position_strides[1];
  a.tokens = tk::FastDiv(static_cast<uint32_t>(tokens));
  a.units = tk::FastDiv(static_cast<uint32_t>(units));
  a.block_heads = tk::FastDiv(static_cast<uint32_t>(block_heads));
  a.total_tokens = static_cast<int>(total);
  a.heads[0] = static_cast<int>(q_heads);
  a.heads[1] = with_k ? static_cast<int>(kv_heads) : 0;
  a.half = half;
  a.rotated_units = rotated;
  a.block_tokens = static_cast<int>(block_tokens);
  a.magnitude = magnitude;
  a.pos64 = wide_positions;
  a.inverse = inverse;
  // A launch holds fewer than 2^32 threads in each dimension, so the runs of tokens spread over
  // two. The last layer's last runs may lie past the tokens: fewer of them than layers, and two
  // layers have runs of at most 2^7 tokens, so less than 2^10 tokens in all, within 32 bits.
  const int64_t token_runs = tk::cdiv(total, block_tokens);
  const int64_t layers = tk::cdiv(token_runs, (int64_t(1) << 24) - 1);
  const dim3 grid(static_cast<uint32_t>(tk::cdiv(token_runs, layers)),
                  static_cast<uint32_t>(tk::cdiv(heads, block_heads)),
                  static_cast<uint32_t>(layers));
  const size_t lds = static_cast<size_t>(block_tokens) * half * 2 * sizeof(float);
  hipStream_t s = tk::as_stream(stream);
  switch (dtype) {
    case TK_DTYPE_F32: launch_vec<float>(vec, a, interleaved != 0, grid, lds, s); break;
    case TK_DTYPE_F16: launch_vec<_Float16>(vec, a, interleaved != 0, grid, lds, s); break;
    default: launch_vec<__bf16>(vec, a, interleaved != 0, grid, lds, s); break;
  }
  return tk::check_launch("rotary");
}
