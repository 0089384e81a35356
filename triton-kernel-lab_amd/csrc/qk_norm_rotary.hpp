// Rows of the query and key norms with rotary positions (qk_norm_rotary.hip, forward, and
// qk_norm_rotary_bwd.hip): how a call's rows are dealt to workgroups and a row's features to lanes.
//
// A row is one head of one token. It is cut into units: a rotated unit of the halves layout is VEC
// pairs (two vectors, half a rotated part apart), one of the interleaved layout a vector of VEC / 2
// pairs (one pair for VEC 1), and a unit past the rotated ones a vector of copied features. `lanes`
// lanes (a power of two) hold a row, lane l its units l, l + lanes, ..: NU of them, so a row's
// statistics are one reduction over those lanes and every feature stays in registers from its load
// to its store. A lane's units are the same in every row, so its weights are loaded once.
//
// A workgroup takes rows of queries or of keys, never both: a run of whole tokens, or a run of one
// token's heads where a token has many. It evaluates its tokens' angles once into LDS.
#pragma once
#include "rotary_angles.hpp"
#include "tk_common.hpp"

namespace tk_qk_norm {

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 512;
constexpr int kMaxAngles = 2048;  // per workgroup: 16 KiB of LDS, so LDS never limits residency

struct Side {  // queries or keys
  const void* x;
  const void* dy;  // backward
  void* out;       // y, or dx
  const void* weight;
  void* dweight;
  int64_t xs[3], ys[3], os[3];  // strides {batch, head, token} of x, dy, out
  int heads;
  int block_tokens;
  tk::FastDiv block_heads;  // heads per run
  tk::FastDiv head_runs;    // runs that a token's heads make
  uint32_t runs;            // of the side
  uint32_t groups;          // backward: workgroups of the side
};

struct Args {
  Side side[2];
  const void* positions;
  const double* frequencies;
  float* partials;  // backward: [workgroup][head_dim]
  int64_t pos_b, pos_n;
  tk::FastDiv tokens;  // tokens per batch entry
  int total_tokens, head_dim, half, rotated_units, units;
  int lanes_log2;
  float eps, magnitude, inv_dim;
  int pos64;
};

template <typename T, int VEC, int NU, bool kInterleaved>
struct Row {
  static constexpr bool TWO = !kInterleaved || VEC == 1;  // a rotated unit is two vectors
  static constexpr int PAIRS = TWO ? VEC : VEC / 2;
  static constexpr int N = 2 * PAIRS;  // values per unit
  static __device__ __forceinline__ int first(int j) { return TWO ? j : 2 * j; }
  static __device__ __forceinline__ int second(int j) { return TWO ? j + VEC : 2 * j + 1; }

  // Where this lane's units lie in any row: first feature (-1: no such unit) and the index of the
  // first angle among a token's (-1: copied).
  struct Layout {
    int col[NU], angle[NU];
    int gap;  // features from a rotated unit's first vector to its second
    __device__ __forceinline__ Layout(const Args& a, int lane) {
      gap = kInterleaved ? 1 : a.half;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int u = lane + (i << a.lanes_log2);
        const bool turned = u < a.rotated_units;
        angle[i] = turned ? PAIRS * u : -1;
        col[i] = turned ? (kInterleaved ? N : VEC) * u
                        : u < a.units ? 2 * a.half + VEC * (u - a.rotated_units) : -1;
      }
    }
  };

  // A row's features as they are stored, so that a load stays in flight until they are needed.
  typedef tk::Vec<T, VEC> V;
  struct Raw {
    V v[NU][TWO ? 2 : 1];
    static __device__ __forceinline__ V get(const T* p) {
      if constexpr (sizeof(V) == 16) {
        typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(V, __builtin_nontemporal_load(reinterpret_cast<const u32x4v*>(p)));
      } else {
        return *reinterpret_cast<const V*>(p);
      }
    }
    __device__ __forceinline__ void load(const T* row, const Layout& at) {
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        if (at.col[i] < 0) continue;
        v[i][0] = get(row + at.col[i]);
        if constexpr (TWO)
          if (at.angle[i] >= 0) v[i][1] = get(row + at.col[i] + at.gap);
      }
    }
    // In float32; zeros where there is no feature.
    __device__ __forceinline__ void expand(const Layout& at, float (&f)[NU][N]) const {
#pragma unroll
      for (int i = 0; i < NU; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          f[i][j] = at.col[i] >= 0 ? tk::to_f32(v[i][0].v[j]) : 0.f;
          if constexpr (TWO) f[i][VEC + j] = at.angle[i] >= 0 ? tk::to_f32(v[i][1].v[j]) : 0.f;
        }
      }
    }
  };

  // Non-temporal stores: they leave the caches to the tensors that are read again (B2 N8192 Hq32 Hkv8 D128:
  // a forward followed by its backward 162 us, 173 with ordinary stores; each among its like 61 and 100, 59
  // and 96 with ordinary ones).
  static __device__ __forceinline__ void store(T* row, const Layout& at, const float (&f)[NU][N]) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (at.col[i] < 0) continue;
      tk::store_vec_stream<T, VEC>(row + at.col[i], f[i]);
      if constexpr (TWO)
        if (at.angle[i] >= 0) tk::store_vec_stream<T, VEC>(row + at.col[i] + at.gap, f[i] + VEC);
    }
  }
};

// Rows of run j of a side: token t0 + p / heads, head h0 + p % heads for p below `count`.
struct Run {
  int t0, h0;
  uint32_t count;
  __device__ __forceinline__ Run(const Args& a, const Side& s, uint32_t j) {
    const uint32_t run = s.head_runs.div(j);
    t0 = int(run) * s.block_tokens;
    h0 = int(j - run * s.head_runs.d) * int(s.block_heads.d);
    count = s.block_heads.d * uint32_t(s.block_tokens);
  }
  // Batch entry, token and head of row p, false where there is none.
  struct At {
    int b, n, h, token;  // token: within the run
  };
  __device__ __forceinline__ bool at(const Args& a, const Side& s, uint32_t p, At& r) const {
    r.token = int(s.block_heads.div(p));
    r.h = h0 + int(p - uint32_t(r.token) * s.block_heads.d);
    const int t = t0 + r.token;
    if (p >= count || t >= a.total_tokens || r.h >= s.heads) return false;
    r.b = int(a.tokens.div(t));
    r.n = t - r.b * int(a.tokens.d);
    return true;
  }
};

__device__ __forceinline__ int64_t offset(const int64_t (&strides)[3], const Run::At& r) {
  return r.b * strides[0] + r.h * strides[1] + r.n * strides[2];
}

// m cos and m sin of the angles of a run's tokens, [token][pair].
__device__ __forceinline__ void fill_angles(const Args& a, const Side& s, int t0, float* cosv,
                                            float* sinv) {
  for (int i = threadIdx.x; i < s.block_tokens * a.half; i += kThreads) {
    const int token = i / a.half;
    const int t = t0 + token;
    if (t >= a.total_tokens) break;
    const uint32_t b = a.tokens.div(t);
    const int64_t at = b * a.pos_b + (t - int64_t(b) * a.tokens.d) * a.pos_n;
    const double pos = a.pos64 ? double(static_cast<const int64_t*>(a.positions)[at])
                               : double(static_cast<const int32_t*>(a.positions)[at]);
    double sn, cs;
    tk_rotary_angles::sincos_any(pos * a.frequencies[i - token * a.half], sn, cs);
    cosv[i] = float(cs * a.magnitude);
    sinv[i] = float(sn * a.magnitude);
  }
}

// Sum over the 2^lanes_log2 neighbouring lanes that hold a row.
__device__ __forceinline__ float row_sum(float v, int lanes_log2) {
  if (lanes_log2 > 0) v += tk::dpp_f32<tk::kDppQuadXor1>(v);
  if (lanes_log2 > 1) v += tk::dpp_f32<tk::kDppQuadXor2>(v);
  if (lanes_log2 > 2) v += tk::dpp_f32<tk::kDppRowHalfMirror>(v);
  if (lanes_log2 > 3) v += tk::dpp_f32<tk::kDppRowMirror>(v);
  if (lanes_log2 > 4) v += __shfl_xor(v, 16);
  if (lanes_log2 > 5) v += __shfl_xor(v, 32);
  return v;
}

// ---------------------------------------------------------------- host side

// What both directions check and plan. Returns 0, or fails; `vec` and `units_per_lane` name the
// kernel. dy strides are null in the forward.
struct Tables {
  const int64_t *x, *dy, *out;
};
int plan(int dtype, const void* const pointers[2][4], const Tables tables[2], const void* positions,
         const double* frequencies, int64_t batch, int64_t tokens, int64_t q_heads,
         int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, const int64_t* position_strides,
         float eps, float magnitude, int interleaved, int wide_positions, Args& a, int& vec,
         int& units_per_lane);

// Workgroups (float32 partial rows) of the backward: three per CU, as many as its registers let run at
// once for rows of 128 features (1024 had a second round: 122 us against 108).
constexpr int kGroups = 768;

// f(kernel's vector and units) for the variants that plan() picks.
#define TK_QK_NORM_VARIANTS(T, vec, nu, F)                                \
  if constexpr (sizeof(T) == 2) {                                         \
    if (vec == 8) {                                                       \
      if (nu == 1) { F(T, 8, 1); } else { F(T, 8, 2); }                   \
    }                                                                     \
  }                                                                       \
  if (vec == 4) {                                                         \
    if (nu == 1) { F(T, 4, 1); } else { F(T, 4, 2); }                     \
  } else if (vec == 2) {                                                  \
    if (nu == 1) { F(T, 2, 1); } else { F(T, 2, 4); }                     \
  } else if (vec == 1) {                                                  \
    if (nu <= 2) { F(T, 1, 2); } else { F(T, 1, 8); }                     \
  }

}  // namespace tk_qk_norm
