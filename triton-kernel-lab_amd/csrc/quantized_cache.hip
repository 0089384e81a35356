// Keys and values quantised into a cache as they are written, and read back. A row (one token's key
// or value of one head) is held as 8-bit codes and a float32 scale:
//   a = max(max |x|, 2^-100),  scale = a / M,  code = round(x (M (1 / a))),  M = 448 (e4m3) or 127 (int8),
// every step rounded to float32, the code then to nearest even: the same codes wherever arithmetic is
// IEEE's. The bound 2^-100 keeps 1 / a finite, so a row of zeros gets codes of zero and needs no case
// of its own. A row with an infinity or a NaN gets a scale of NaN and
// codes of zero, so that every value read back of it is NaN.
//
// A lane holds 16 bytes of tokens (8 features of 16 bits, 4 of 32), so that every wave reads and writes
// whole lines of the wider tensors: with 16 features a lane, its two 16-byte accesses 32 bytes apart
// from the next lane's, reading back ran at 2.4 TB/s. The same lanes take a token's key and its value,
// so both rows' loads are in flight together and the pair of scales is one store.
//
// Bound by HBM: the tokens are read and the codes written once. 8 x 4096 tokens of 8 KV heads, D128, from
// bf16: 38.6 us, 5.3 TB/s; padded to that from 0 to 4096 (120 MB) 25.7 us, 4.7 TB/s. With one token a
// lane, heads apart and default stores of codes 42 to 45 and 32 us; four or eight tokens a lane 41 and 45.
// Reading back 8 x 8192 positions 66.5 us, 6.1 TB/s.
#include "eight_bit.hpp"
#include "tk_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 1024;
constexpr int kSteps = 2;  // tokens that a lane takes where this many workgroups are left
constexpr int kManyWorkgroups = 1024;

// PER codes as one access.
template <int kPer>
struct alignas(kPer) Codes {
  int c[kPer / 4];
};

struct AppendArgs {
  uint8_t* cache[2];
  const void* x[2];
  float* scales;
  const int32_t* seqlens;
  const int32_t* counts;  // null: every token
  int32_t* new_seqlens;
  int64_t cs[2][3], xs[2][3], ss[3];
  tk::FastDiv head_blocks, token_blocks;
  int tokens, heads, max_len;
  int units, lanes_log2;       // 16-byte parts of a row of tokens; lanes a row
  int tokens_log2, heads_log2; // rows side by side in a workgroup
};

__device__ __forceinline__ uint32_t row_max(uint32_t v, int lanes_log2) {
  for (int i = 0; i < lanes_log2; ++i) v = max(v, uint32_t(__shfl_xor(int(v), 1 << i)));
  return v;
}

// 2^lanes_log2 lanes a row (a power of two), lane l its parts l, l + lanes, ..: up to NU. A workgroup
// takes 2^tokens_log2 * STEPS tokens of 2^heads_log2 heads; neighbouring workgroups take the heads of
// the same tokens, which lie side by side in a projection's output.
template <typename T, int kType, int NU, int STEPS>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  constexpr int PER = 16 / sizeof(T);
  typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
  const uint32_t tokens_of = a.head_blocks.div(blockIdx.x);
  const int64_t b = a.token_blocks.div(tokens_of);
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1);
  const int row = threadIdx.x >> a.lanes_log2;
  const int t0 = (int(tokens_of - b * a.token_blocks.d) * STEPS << a.tokens_log2) +
                 (row & ((1 << a.tokens_log2) - 1));
  const int64_t h = ((blockIdx.x - tokens_of * a.head_blocks.d) << a.heads_log2) + (row >> a.tokens_log2);
  const int start = min(max(a.seqlens[b], 0), a.max_len);
  const int given = a.counts != nullptr ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
  const int count = min(given, a.max_len - start);
  if (h == 0 && t0 == 0 && lane == 0) a.new_seqlens[b] = start + count;
  if (t0 >= count || h >= a.heads) return;
  u32x4v raw[STEPS][2][NU];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int t = t0 + (i << a.tokens_log2);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const T* p = static_cast<const T*>(a.x[w]) + b * a.xs[w][0] + h * a.xs[w][1] + t * a.xs[w][2];
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const int u = lane + (n << a.lanes_log2);
        raw[i][w][n] = t < count && u < a.units
                           ? __builtin_nontemporal_load(reinterpret_cast<const u32x4v*>(p + u * PER))
                           : u32x4v{0u, 0u, 0u, 0u};
      }
    }
  }
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int t = t0 + (i << a.tokens_log2);
    const int64_t at = int64_t(start) + t;
    float scale[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float x[NU][PER];
      // Magnitudes compare as their bits, NaN above infinity above every number.
      uint32_t most = 0;
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const auto v = __builtin_bit_cast(tk::Vec<T, PER>, raw[i][w][n]);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          x[n][j] = tk::to_f32(v.v[j]);
          most = max(most, __float_as_uint(x[n][j]) & 0x7FFFFFFFu);
        }
      }
      most = row_max(most, a.lanes_log2);
      const bool sound = most < 0x7F800000u;
      const float top = fmaxf(__uint_as_float(most), 0x1p-100f);
      const float inverse = tk8::kMost<kType> * (1.0f / top);
      scale[w] = sound ? top / tk8::kMost<kType> : __uint_as_float(0x7FC00000u);
      uint8_t* out = a.cache[w] + b * a.cs[w][0] + h * a.cs[w][1] + at * a.cs[w][2];
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        Codes<PER> codes;
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = x[n][j + k] * inverse;
          codes.c[j / 4] = sound ? tk8::encode4<kType>(v) : 0;
        }
        const int u = lane + (n << a.lanes_log2);
        if (t >= count || u >= a.units) continue;
        // Many tokens' codes pass through the caches; a few tokens' are read next.
        if constexpr (STEPS > 1 && PER == 8)
          __builtin_nontemporal_store(__builtin_bit_cast(uint64_t, codes),
                                      reinterpret_cast<uint64_t*>(out + u * PER));
        else
          *reinterpret_cast<Codes<PER>*>(out + u * PER) = codes;
      }
    }
    if (t < count && lane == 0)
      *reinterpret_cast<float2*>(a.scales + b * a.ss[0] + h * a.ss[1] + at * a.ss[2]) =
          make_float2(scale[0], scale[1]);
  }
}

struct ReadArgs {
  const uint8_t* cache[2];
  const float* scales;
  const int32_t* seqlens;
  void* out[2];  // [batch][heads][max_len][head_dim]
  int64_t cs[2][3], ss[3];
  tk::FastDiv units;  // 16-byte parts of a row of the output
  int max_len;
};

template <typename T, int kType>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
  constexpr int PER = 16 / sizeof(T);
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  const int64_t h = blockIdx.y, b = blockIdx.z;
  const uint32_t row = a.units.div(i);
  const int u = int(i - row * a.units.d);
  if (row >= uint32_t(a.max_len)) return;
  const int length = a.seqlens != nullptr ? a.seqlens[b] : a.max_len;
  const int64_t to = (((b * gridDim.y + h) * a.max_len + row) * a.units.d + u) * PER;
  Codes<PER> codes[2] = {};
  float2 scale = {};
  if (int(row) < length) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
      codes[w] = *reinterpret_cast<const Codes<PER>*>(a.cache[w] + b * a.cs[w][0] + h * a.cs[w][1] +
                                                      row * a.cs[w][2] + u * PER);
    scale = *reinterpret_cast<const float2*>(a.scales + b * a.ss[0] + h * a.ss[1] + row * a.ss[2]);
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float x[PER];
#pragma unroll
    for (int j = 0; j < PER; j += 4) tk8::decode4<kType>(codes[w].c[j / 4], x + j);
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] *= w ? scale.y : scale.x;
    tk::store_vec_stream<T, PER>(static_cast<T*>(a.out[w]) + to, x);
  }
}

// Strides {batch, head, position} that keep rows on a `unit`-element boundary and in range; a null
// table is the caller's to refuse.
const char* bad_strides(const int64_t* s, int64_t unit, int64_t batch, int64_t heads, int64_t rows,
                        int64_t row) {
  __int128 last = row;
  const int64_t counts[3] = {batch, heads, rows};
  for (int d = 0; d < 3; ++d) {
    if (s[d] < 0) return "strides must be non-negative";
    if (s[d] % unit != 0 && counts[d] > 1) return "strides must keep rows 16-byte aligned";
    last += static_cast<__int128>(counts[d] - 1) * s[d];
  }
  return last >= (static_cast<__int128>(1) << 52) ? "strides must keep rows in range" : nullptr;
}

template <typename T, int kType>
void launch_append(const AppendArgs& a, int steps, uint32_t workgroups, hipStream_t s) {
  const dim3 grid(workgroups), block(kThreads);
  if (a.units <= 64 && steps > 1)
    hipLaunchKernelGGL((append_kernel<T, kType, 1, kSteps>), grid, block, 0, s, a);
  else if (a.units <= 64)
    hipLaunchKernelGGL((append_kernel<T, kType, 1, 1>), grid, block, 0, s, a);
  else if (sizeof(T) == 2 || a.units <= 128)
    hipLaunchKernelGGL((append_kernel<T, kType, 2, 1>), grid, block, 0, s, a);
  else if constexpr (sizeof(T) == 4)
    hipLaunchKernelGGL((append_kernel<T, kType, 4, 1>), grid, block, 0, s, a);
}

template <typename T>
void launch_append(const AppendArgs& a, int type, int steps, uint32_t workgroups, hipStream_t s) {
  if (type == tk8::kE4M3)
    launch_append<T, tk8::kE4M3>(a, steps, workgroups, s);
  else
    launch_append<T, tk8::kInt8>(a, steps, workgroups, s);
}

template <typename T>
void launch_read(const ReadArgs& a, int type, dim3 grid, hipStream_t s) {
  if (type == tk8::kE4M3)
    hipLaunchKernelGGL((read_kernel<T, tk8::kE4M3>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((read_kernel<T, tk8::kInt8>), grid, dim3(kThreads), 0, s, a);
}

}  // namespace

extern "C" int tk_append_quantized(int dtype, void* k_cache, void* v_cache, float* scales,
                                   const int32_t* seqlens, const void* k, const void* v,
                                   const int32_t* counts, int32_t* new_seqlens, int64_t batch,
                                   int64_t kv_heads, int64_t max_len, int64_t tokens,
                                   int64_t head_dim, const int64_t* k_cache_strides,
                                   const int64_t* v_cache_strides, const int64_t* scale_strides,
                                   const int64_t* k_strides, const int64_t* v_strides,
                                   int cache_type, void* stream) {
  if (!tk::valid_dtype(dtype)) return tk::fail("append: unsupported dtype code %d", dtype);
  if (k_cache == nullptr || v_cache == nullptr || scales == nullptr || seqlens == nullptr ||
      k == nullptr || v == nullptr || new_seqlens == nullptr || k_cache_strides == nullptr ||
      v_cache_strides == nullptr || scale_strides == nullptr || k_strides == nullptr ||
      v_strides == nullptr)
    return tk::fail("append: null pointer");
  if (cache_type != tk8::kE4M3 && cache_type != tk8::kInt8)
    return tk::fail("append: unsupported cache type %d", cache_type);
  if (batch <= 0 || kv_heads <= 0 || max_len <= 0 || tokens <= 0 || head_dim <= 0)
    return tk::fail("append: empty problem");
  if (head_dim % 16 != 0 || head_dim > kMaxHeadDim)
    return tk::fail("append: head_dim must be a multiple of 16, at most %d", kMaxHeadDim);
  if (batch > 65535 || kv_heads > 65535 || max_len > (1 << 30) || tokens > (1 << 30))
    return tk::fail("append: problem too large");
  AppendArgs a;
  a.units = static_cast<int>(head_dim * tk::elem_size(dtype) / 16);
  a.lanes_log2 = 0;
  while ((1 << a.lanes_log2) < a.units && a.lanes_log2 < 6) ++a.lanes_log2;
  // Rows side by side: as many tokens as there are, then heads. Lanes take several tokens where enough
  // workgroups are left.
  const int rows_log2 = 8 - a.lanes_log2;
  a.tokens_log2 = 0;
  while (a.tokens_log2 < rows_log2 && (int64_t(1) << a.tokens_log2) < tokens) ++a.tokens_log2;
  a.heads_log2 = rows_log2 - a.tokens_log2;
  const int64_t head_blocks = tk::cdiv(kv_heads, int64_t(1) << a.heads_log2);
  int64_t token_blocks = tk::cdiv(tokens, int64_t(1) << a.tokens_log2);
  int steps = 1;
  if (a.units <= 64 && batch * head_blocks * token_blocks >= kSteps * kManyWorkgroups) {
    steps = kSteps;
    token_blocks = tk::cdiv(tokens, int64_t(kSteps) << a.tokens_log2);
  }
  // A launch holds fewer than 2^32 threads, and workgroups are divided as numbers below 2^31.
  const __int128 workgroups = static_cast<__int128>(batch) * head_blocks * token_blocks;
  if (workgroups >= (static_cast<__int128>(1) << 24)) return tk::fail("append: problem too large");
  const int64_t* cache_strides[2] = {k_cache_strides, v_cache_strides};
  const int64_t* x_strides[2] = {k_strides, v_strides};
  for (int w = 0; w < 2; ++w) {
    if (const char* why = bad_strides(cache_strides[w], 16, batch, kv_heads, max_len, head_dim))
      return tk::fail("append: cache %s", why);
    if (const char* why = bad_strides(x_strides[w], 16 / tk::elem_size(dtype), batch, kv_heads,
                                      tokens, head_dim))
      return tk::fail("append: %s", why);
    for (int d = 0; d < 3; ++d) {
      a.cs[w][d] = cache_strides[w][d];
      a.xs[w][d] = x_strides[w][d];
    }
  }
  if (const char* why = bad_strides(scale_strides, 2, batch, kv_heads, max_len, 2))
    return tk::fail("append: scale %s", why);
  for (const void* p : {static_cast<const void*>(k_cache), static_cast<const void*>(v_cache), k, v})
    if (!tk::aligned16(p)) return tk::fail("append: tensors must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(scales) % 8 != 0)
    return tk::fail("append: scales must be 8-byte aligned");
  for (int d = 0; d < 3; ++d) a.ss[d] = scale_strides[d];
  a.cache[0] = static_cast<uint8_t*>(k_cache);
  a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.x[0] = k;
  a.x[1] = v;
  a.scales = scales;
  a.seqlens = seqlens;
  a.counts = counts;
  a.new_seqlens = new_seqlens;
  a.head_blocks = tk::FastDiv(static_cast<uint32_t>(head_blocks));
  a.token_blocks = tk::FastDiv(static_cast<uint32_t>(token_blocks));
  a.tokens = static_cast<int>(tokens);
  a.heads = static_cast<int>(kv_heads);
  a.max_len = static_cast<int>(max_len);
  const uint32_t grid = static_cast<uint32_t>(workgroups);
  hipStream_t s = tk::as_stream(stream);
  switch (dtype) {
    case TK_DTYPE_F32: launch_append<float>(a, cache_type, steps, grid, s); break;
    case TK_DTYPE_F16: launch_append<_Float16>(a, cache_type, steps, grid, s); break;
    default: launch_append<__bf16>(a, cache_type, steps, grid, s); break;
  }
  return tk::check_launch("append");
}

extern "C" int tk_read_quantized(int dtype, const void* k_cache, const void* v_cache,
                                 const float* scales, const int32_t* seqlens, void* k, void* v,
                                 int64_t batch, int64_t kv_heads, int64_t max_len,
                                 int64_t head_dim, const int64_t* k_cache_strides,
                                 const int64_t* v_cache_strides, const int64_t* scale_strides,
                                 int cache_type, void* stream) {
  if (!tk::valid_dtype(dtype)) return tk::fail("read: unsupported dtype code %d", dtype);
  if (k_cache == nullptr || v_cache == nullptr || scales == nullptr || k == nullptr ||
      v == nullptr || k_cache_strides == nullptr || v_cache_strides == nullptr ||
      scale_strides == nullptr)
    return tk::fail("read: null pointer");
  if (cache_type != tk8::kE4M3 && cache_type != tk8::kInt8)
    return tk::fail("read: unsupported cache type %d", cache_type);
  if (batch <= 0 || kv_heads <= 0 || max_len <= 0 || head_dim <= 0)
    return tk::fail("read: empty problem");
  if (head_dim % 16 != 0 || head_dim > kMaxHeadDim)
    return tk::fail("read: head_dim must be a multiple of 16, at most %d", kMaxHeadDim);
  const int64_t units = head_dim * tk::elem_size(dtype) / 16;
  if (batch > 65535 || kv_heads > 65535 || max_len > (1 << 30) ||
      max_len * units > INT32_MAX - kThreads)
    return tk::fail("read: problem too large");
  ReadArgs a;
  const int64_t* cache_strides[2] = {k_cache_strides, v_cache_strides};
  for (int w = 0; w < 2; ++w) {
    if (const char* why = bad_strides(cache_strides[w], 16, batch, kv_heads, max_len, head_dim))
      return tk::fail("read: cache %s", why);
    for (int d = 0; d < 3; ++d) a.cs[w][d] = cache_strides[w][d];
  }
  if (const char* why = bad_strides(scale_strides, 2, batch, kv_heads, max_len, 2))
    return tk::fail("read: scale %s", why);
  for (const void* p : {k_cache, v_cache, static_cast<const void*>(k), static_cast<const void*>(v)})
    if (!tk::aligned16(p)) return tk::fail("read: tensors must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(scales) % 8 != 0)
    return tk::fail("read: scales must be 8-byte aligned");
  for (int d = 0; d < 3; ++d) a.ss[d] = scale_strides[d];
  a.cache[0] = static_cast<const uint8_t*>(k_cache);
  a.cache[1] = static_cast<const uint8_t*>(v_cache);
  a.scales = scales;
  a.seqlens = seqlens;
  a.out[0] = k;
  a.out[1] = v;
  a.units = tk::FastDiv(static_cast<uint32_t>(units));
  a.max_len = static_cast<int>(max_len);
  const dim3 grid(static_cast<uint32_t>(tk::cdiv(max_len * units, kThreads)),
                  static_cast<uint32_t>(kv_heads), static_cast<uint32_t>(batch));
  hipStream_t s = tk::as_stream(stream);
  switch (dtype) {
    case TK_DTYPE_F32: launch_read<float>(a, cache_type, grid, s); break;
    case TK_DTYPE_F16: launch_read<_Float16>(a, cache_type, grid, s); break;
    default: launch_read<__bf16>(a, cache_type, grid, s); break;
  }
  return tk::check_launch("read");
}
