// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Nodes 0 .. nodes-1 of a sequence are a tree in which parents precede children
// (node 0 the last accepted token, a chain when no parents are given); target row i is the
// target's distribution behind node i. Walk from the root: the children of the current node are
// tried in order, child i with token x and random number u_i is kept (and becomes the current
// node) if
//   u_i q(x) < p(x)   where the children were drawn from q (draft rows; chains only), else
//   u_i m < p(x)      where m = 1 - the rejected siblings' p (drafts taken without drawing;
//                     a token rejected once is not tried again).
// The next token is then drawn from the current node's w = max(p - q, 0) after a rejection, p
// without the rejected tokens, or p: the first v with w_0 + .. + w_v > u_0 sum(w). If w has no
// mass, p stands in for it; if p has none either, the token is -1. All of it is float64, where a
// product of two float32 is exact and a difference is rounded once, by at most 2^-53 of it. The
// sums' order depends on the splits: with c entries a split a sum passes through at most
// c / 128 + 64 additions, so a border within (c / 128 + 64) 2^-52 sum(w) of u_0 sum(w) may fall to
// either side (2^-45 of the sum where c is 8192).
//
// The children test a probability each, known from parents and tokens alone, so one wave
// gathers all nodes' at once and walks in registers: the path costs two trips to memory. Then
// only one row (two where the draft's is taken off) of `vocabulary` entries is read: by
// `splits` workgroups per sequence, each of which repeats the walk (cheaper than a launch to
// share it), and a second launch finds the split of the drawn token from the partial sums and
// reads that split alone again.
//
// 64 chains of 7 drafts over 131072 float32 entries (about 50 MB of rows): 14 us + 5.5 us, the
// walk's two trips to memory in front of the rows' stream; one chain over 32001 entries: 4.6 + 4 us,
// all latency. Two passes' loads of a thread issued together: 18 us instead of 16 (at 2048 entries a
// workgroup), not kept.
#include "tk_common.hpp"

namespace {

constexpr int kMaxNodes = 256;
constexpr int kWeighThreads = 256;
constexpr int kDrawThreads = 1024;
constexpr int kMaxSplits = 64;  // one wave scans the partial sums
constexpr int kStateHead = 4;   // node, against, rejected tokens' number, padding

struct VerifyArgs {
  const void* target;
  const void* draft;
  const void* tokens;
  const int32_t* parents;
  const float* uniforms;
  int32_t* path;
  int32_t* count;
  int64_t* next;
  double* sums;    // [batch][2][splits]: of w, of p
  int32_t* state;  // [batch][kStateHead + nodes]: the walk's end, rejected tokens
  int64_t tb, tn, db, dn, token_b, parent_b, uniform_b;
  int nodes, vocabulary, splits, chunk, tokens64;
};

// Eight entries of a row from any element boundary.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* f) {
  constexpr int N = 16 / int(sizeof(T));
#pragma unroll
  for (int i = 0; i < 8; i += N) {
    const tk::Vec<T, N> r = __builtin_bit_cast(
        tk::Vec<T, N>, *reinterpret_cast<const u32x4_any*>(p + i));
#pragma unroll
    for (int j = 0; j < N; ++j) f[i + j] = tk::to_f32(r.v[j]);
  }
}

// Entries that are no positive finite number carry no weight.
__device__ __forceinline__ double mass(float p) {
  return p > 0.f && p < INFINITY ? double(p) : 0.0;
}

// Eight entries' weights from column e of [.., end): p's own in `plain`, those drawn from in `w`.
template <typename T>
__device__ __forceinline__ void weights8(const T* p, const T* q, int e, int end,
                                         const int32_t* rejected, int n_rejected, double* plain,
                                         double* w) {
  float pf[8], qf[8];
  if (e + 8 <= end) {
    load8<T>(p + e, pf);
    if (q != nullptr) load8<T>(q + e, qf);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      pf[j] = e + j < end ? tk::to_f32(p[e + j]) : 0.f;
      if (q != nullptr) qf[j] = e + j < end ? tk::to_f32(q[e + j]) : 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    plain[j] = mass(pf[j]);
    w[j] = q != nullptr ? fmax(plain[j] - mass(qf[j]), 0.0) : plain[j];
  }
  for (int r = 0; r < n_rejected; ++r) {
    const int at = rejected[r] - e;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at == j) w[j] = 0.0;
  }
}

__device__ __forceinline__ double lane_value(double v, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(uint32_t(bits), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(uint32_t(bits >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t(hi) << 32) | lo);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// Inclusive prefix sums over the wave's lanes.
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double up = __shfl_up(v, d);
    if (lane >= d) v += up;
  }
  return v;
}

// The walk, by one wave; `kept` and `rejected` are bit masks over the nodes.
struct Walk {
  int node = 0, against = -1;
  uint64_t kept[kMaxNodes / 64] = {1, 0, 0, 0}, rejected[kMaxNodes / 64] = {};
  int token[kMaxNodes / 64];  // this lane's nodes' tokens, -1: none
};

template <typename T>
__device__ __forceinline__ void walk(const VerifyArgs& a, int b, int lane, Walk& w) {
  constexpr int C = kMaxNodes / 64;
  int parent[C];
  double p[C], q[C];
  float u[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * 64 + lane;
    parent[c] = -2;
    w.token[c] = -1;
    u[c] = 0.f;
    if (i >= 1 && i < a.nodes) {
      const int64_t t = a.tokens64
                            ? static_cast<const int64_t*>(a.tokens)[b * a.token_b + i]
                            : int64_t(static_cast<const int32_t*>(a.tokens)[b * a.token_b + i]);
      const int up = a.parents != nullptr ? a.parents[b * a.parent_b + i] : i - 1;
      u[c] = a.uniforms[b * a.uniform_b + i];
      if (up >= 0 && up < i && t >= 0 && t < a.vocabulary) {
        parent[c] = up;
        w.token[c] = int(t);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * 64 + lane;
    p[c] = q[c] = 0.0;
    if (parent[c] >= 0) {
      p[c] = mass(tk::to_f32(
          (static_cast<const T*>(a.target) + b * a.tb + parent[c] * a.tn)[w.token[c]]));
      if (a.draft != nullptr)
        q[c] = mass(tk::to_f32(
            (static_cast<const T*>(a.draft) + b * a.db + (i - 1) * a.dn)[w.token[c]]));
    }
  }
  double left = 1.0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c * 64 >= a.nodes) break;
    uint64_t after = ~0ull;
    for (;;) {
      const uint64_t asked = __ballot(parent[c] == w.node) & after;
      if (asked == 0) break;
      const int i = __builtin_ctzll(asked);
      after = ~((2ull << i) - 1);
      const double pi = lane_value(p[c], i);
      const double ui = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(u[c]), i));
      bool good;
      if (a.draft != nullptr) {
        good = ui * lane_value(q[c], i) < pi;
        if (!good) w.against = c * 64 + i;
      } else {
        const int t = __builtin_amdgcn_readlane(w.token[c], i);
        bool again = false;
#pragma unroll
        for (int d = 0; d < C; ++d) again |= (__ballot(w.token[d] == t) & w.rejected[d]) != 0;
        good = !again && ui * left < pi;
        if (!again && !good) {
          left = fmax(left - pi, 0.0);
          w.rejected[c] |= 1ull << i;
        }
      }
      if (good) {
        w.node = c * 64 + i;
        w.kept[c] |= 1ull << i;
        left = 1.0;
#pragma unroll
        for (int d = 0; d < C; ++d) w.rejected[d] = 0;
      }
    }
  }
}

// Grid (splits, batch): sums of one split's weights; split 0 also writes the path, its length and
// the walk's end.
template <typename T>
__global__ __launch_bounds__(kWeighThreads) void verify_weigh_kernel(VerifyArgs a) {
  __shared__ int32_t end[2];
  __shared__ int32_t rejected[kMaxNodes];
  __shared__ int n_rejected;
  __shared__ double part[2][kWeighThreads / 64];
  const int split = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c0 = split * a.chunk;
  const int c1 = c0 + min(a.chunk, a.vocabulary - c0);  // c0 + chunk may pass 32 bits
  constexpr int C = kMaxNodes / 64;
  if (wave == 0) {
    Walk w;
    walk<T>(a, b, lane, w);
    const uint64_t below = (1ull << lane) - 1;
    int kept = 0, here = 0, all = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (c * 64 >= a.nodes) break;
      const bool mine = (w.rejected[c] >> lane) & 1;
      const bool inside = mine && w.token[c] >= c0 && w.token[c] < c1;
      const uint64_t local = __ballot(inside);
      if (inside) rejected[here + __popcll(local & below)] = w.token[c];
      here += __popcll(local);
      if (split == 0) {
        int32_t* state = a.state + int64_t(b) * (kStateHead + a.nodes);
        int32_t* path = a.path + int64_t(b) * a.nodes;
        if (mine) state[kStateHead + all + __popcll(w.rejected[c] & below)] = w.token[c];
        if ((w.kept[c] >> lane) & 1) path[kept + __popcll(w.kept[c] & below)] = c * 64 + lane;
      }
      all += __popcll(w.rejected[c]);
      kept += __popcll(w.kept[c]);
    }
    if (split == 0) {
      for (int i = kept + lane; i < a.nodes; i += 64) a.path[int64_t(b) * a.nodes + i] = -1;
      if (lane == 0) {
        int32_t* state = a.state + int64_t(b) * (kStateHead + a.nodes);
        state[0] = w.node;
        state[1] = w.against;
        state[2] = all;
        a.count[b] = kept;
      }
    }
    if (lane == 0) {
      end[0] = w.node;
      end[1] = w.against;
      n_rejected = here;
    }
  }
  __syncthreads();
  const T* p = static_cast<const T*>(a.target) + b * a.tb + end[0] * a.tn;
  const T* q = end[1] > 0 ? static_cast<const T*>(a.draft) + b * a.db + (end[1] - 1) * a.dn
                          : nullptr;
  const int n = n_rejected;
  double sum = 0.0, plain_sum = 0.0;
  for (int e = c0 + int(threadIdx.x) * 8; e < c1; e += kWeighThreads * 8) {
    double plain[8], w[8];
    weights8<T>(p, q, e, c1, rejected, n, plain, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sum += w[j];
      plain_sum += plain[j];
    }
  }
  sum = wave_sum(sum);
  plain_sum = wave_sum(plain_sum);
  if (lane == 0) {
    part[0][wave] = sum;
    part[1][wave] = plain_sum;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    double s = part[threadIdx.x][0];
#pragma unroll
    for (int i = 1; i < kWeighThreads / 64; ++i) s += part[threadIdx.x][i];
    a.sums[(int64_t(b) * 2 + threadIdx.x) * a.splits + split] = s;
  }
}

// Grid (batch): the drawn token.
template <typename T>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs a) {
  constexpr int W = kDrawThreads / 64;
  __shared__ int32_t rejected[kMaxNodes];
  __shared__ double wave_total[2][W];
  __shared__ int winner[2];
  const int b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t* state = a.state + int64_t(b) * (kStateHead + a.nodes);
  const int node = state[0], against = state[1];
  int n = state[2];
  for (int i = tid; i < n; i += kDrawThreads) rejected[i] = state[kStateHead + i];
  // Every wave scans the splits' sums: those of w, or of p where w has no mass.
  double own = lane < a.splits ? a.sums[int64_t(b) * 2 * a.splits + lane] : 0.0;
  const double other = lane < a.splits ? a.sums[(int64_t(b) * 2 + 1) * a.splits + lane] : 0.0;
  const T* p = static_cast<const T*>(a.target) + b * a.tb + node * a.tn;
  const T* q = against > 0 ? static_cast<const T*>(a.draft) + b * a.db + (against - 1) * a.dn
                           : nullptr;
  if (__ballot(own > 0.0) == 0) {
    own = other;
    q = nullptr;
    n = 0;
  }
  const uint64_t some = __ballot(own > 0.0);
  if (some == 0) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  const double upto = wave_scan(own, lane);
  // The random number is taken into [0, 1): below 0 (or not a number) is 0.
  const double u = fmin(fmax(double(a.uniforms[b * a.uniform_b]), 0.0), 1.0 - 0x1p-53);
  const double goal = u * lane_value(upto, 63);
  const uint64_t past = __ballot(own > 0.0 && upto > goal);
  const int split = past != 0 ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  double base = split > 0 ? lane_value(upto, split - 1) : 0.0;
  const int c0 = split * a.chunk;
  const int c1 = c0 + min(a.chunk, a.vocabulary - c0);  // c0 + chunk may pass 32 bits
  if (tid < 2) winner[tid] = kDrawThreads;
  __syncthreads();

  int turn = 0;
  for (int t0 = c0; t0 < c1; t0 += kDrawThreads * 8, turn ^= 1) {
    const int e = t0 + tid * 8;
    double plain[8], w[8], mine = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 0.0;
    if (e < c1) weights8<T>(p, q, e, c1, rejected, n, plain, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) mine += w[j];
    const double in_wave = wave_scan(mine, lane);
    if (lane == 63) wave_total[turn][wave] = in_wave;
    __syncthreads();
    double before = base, total = base;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i == wave) before = total;
      total += wave_total[turn][i];
    }
    const uint64_t hit = __ballot(mine > 0.0 && before + in_wave > goal);
    if (hit != 0 && lane == __builtin_ctzll(hit)) atomicMin(&winner[turn], tid);
    double run = __shfl_up(in_wave, 1);
    run = before + (lane > 0 ? run : 0.0);
    __syncthreads();
    const int first = winner[turn];
    if (first < kDrawThreads) {
      if (tid == first) {
        int at = -1, last = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          run += w[j];
          if (w[j] > 0.0) {
            last = j;
            if (at < 0 && run > goal) at = j;
          }
        }
        a.next[b] = e + (at >= 0 ? at : last);
      }
      return;
    }
    base = total;
  }
  // The split's sum passed the goal but, added in this order, its entries did not: the two
  // agree up to the last bits, so the token is the split's last one that has weight.
  if (wave == 0) {
    int last = -1;
    for (int e = c0 + lane * 8; e < c1; e += 64 * 8) {
      double plain[8], w[8];
      weights8<T>(p, q, e, c1, rejected, n, plain, w);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (w[j] > 0.0) last = e + j;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) last = max(last, __shfl_xor(last, d));
    if (lane == 0) a.next[b] = last;
  }
}

}  // namespace

extern "C" int tk_verify_draft(int dtype, const void* target, const void* draft,
                               const void* tokens, const int32_t* parents, const float* uniforms,
                               int32_t* path, int32_t* count, int64_t* next_token,
                               void* workspace, int64_t batch, int64_t nodes, int64_t vocabulary,
                               int64_t chunk, const int64_t* target_strides,
                               const int64_t* draft_strides, const int64_t* node_strides,
                               int wide_tokens, void* stream) {
  if (!tk::valid_dtype(dtype)) return tk::fail("unsupported dtype code %d", dtype);
  if (target == nullptr || tokens == nullptr || uniforms == nullptr || path == nullptr ||
      count == nullptr || next_token == nullptr || workspace == nullptr ||
      target_strides == nullptr || node_strides == nullptr ||
      (draft != nullptr && draft_strides == nullptr))
    return tk::fail("verify draft: null pointer");
  if (batch <= 0 || nodes <= 0 || vocabulary <= 0) return tk::fail("verify draft: empty problem");
  if (nodes > kMaxNodes) return tk::fail("verify draft: at most %d nodes", kMaxNodes);
  if (batch > 65535 || vocabulary > INT32_MAX - 65536)
    return tk::fail("verify draft: problem too large");
  if (chunk <= 0 || chunk % 8 != 0 || chunk > INT32_MAX - 65536 ||
      tk::cdiv(vocabulary, chunk) > kMaxSplits)
    return tk::fail("verify draft: chunk must be a multiple of 8 that makes at most %d splits",
                    kMaxSplits);
  if (reinterpret_cast<uintptr_t>(workspace) % 8 != 0)
    return tk::fail("verify draft: workspace must be 8-byte aligned");
  VerifyArgs a;
  a.tb = target_strides[0];
  a.tn = target_strides[1];
  a.db = draft != nullptr ? draft_strides[0] : 0;
  a.dn = draft != nullptr ? draft_strides[1] : 0;
  a.token_b = node_strides[0];
  a.parent_b = node_strides[1];
  a.uniform_b = node_strides[2];
  if (!tk::row_strides_ok(batch, nodes, {a.token_b, a.parent_b, a.uniform_b}) || a.tb < 0 ||
      a.tn < 0 || a.db < 0 || a.dn < 0 ||
      tk::extent(batch, a.tb, nodes, a.tn) >= (static_cast<__int128>(1) << 52) ||
      tk::extent(batch, a.db, nodes, a.dn) >= (static_cast<__int128>(1) << 52))
    return tk::fail("verify draft: strides must be non-negative and keep rows in range");
  if (draft != nullptr && parents != nullptr)
    return tk::fail("verify draft: draft probabilities belong to a chain, without parents");
  const int64_t splits = tk::cdiv(vocabulary, chunk);
  a.target = target;
  a.draft = draft;
  a.tokens = tokens;
  a.parents = parents;
  a.uniforms = uniforms;
  a.path = path;
  a.count = count;
  a.next = next_token;
  a.sums = static_cast<double*>(workspace);
  a.state = reinterpret_cast<int32_t*>(a.sums + batch * 2 * splits);
  a.nodes = static_cast<int>(nodes);
  a.vocabulary = static_cast<int>(vocabulary);
  a.splits = static_cast<int>(splits);
  a.chunk = static_cast<int>(chunk);
  a.tokens64 = wide_tokens;
  hipStream_t s = tk::as_stream(stream);
  const dim3 grid(static_cast<uint32_t>(splits), static_cast<uint32_t>(batch));
  TK_DISPATCH_DTYPE(dtype, T,
    hipLaunchKernelGGL((verify_weigh_kernel<T>), grid, dim3(kWeighThreads), 0, s, a);
    hipLaunchKernelGGL((verify_draw_kernel<T>), dim3(static_cast<uint32_t>(batch)),
                       dim3(kDrawThreads), 0, s, a));
  return tk::check_launch("verify draft");
}
