// Runs of key tiles for the decode kernels over caches whose lengths only the device knows: the
// tiles of all sequences are dealt in equal runs, found by every workgroup from the lengths, so a
// ragged batch fills the chip; and the joining of the runs' partial results.
#pragma once
#include "attention_dma.hpp"
#include "tk_common.hpp"

namespace tk_runs {

constexpr int kTileKeys = 32;
constexpr float kLog2e = 1.4426950408889634f;
// The running maximum before any key: finite, so that a masked score (-inf) minus it stays
// -inf, and below every score that carries weight.
constexpr float kNoMax = -3.0e38f;

struct Schedule {
  const int32_t* seqlens;  // null: every sequence has max_len keys
  int batch, max_len;
  int runs;   // the tiles of all sequences over this many runs give the run length
  int fewer;  // and over this many where that makes runs of less than kLongRun tiles
  int whole;  // a sequence of at most this many tiles is one run
};
constexpr int kMinRun = 2, kLongRun = 8;  // tiles

__device__ __forceinline__ int context_length(const Schedule& s, int b) {
  const int n = s.seqlens != nullptr ? s.seqlens[b] : s.max_len;
  return min(max(n, 0), s.max_len);
}

// At least one tile (an empty one writes the result of no keys).
__device__ __forceinline__ int tiles_of(int length) {
  return max((length + kTileKeys - 1) / kTileKeys, 1);
}

// Inclusive prefix sums over the wave's lanes: within rows of 16 lanes by shifts, then the rows'
// and the halves' last sums broadcast to the next ones.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_part(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ int wave_prefix(int v) {
  v += dpp_part<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v += dpp_part<0x112, 0xF>(v);
  v += dpp_part<0x114, 0xF>(v);
  v += dpp_part<0x118, 0xF>(v);
  v += dpp_part<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp_part<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}

struct Lengths {
  int first;  // this lane's sequence's length (sequence = lane)
  int chunk;  // tiles per run
};

__device__ __forceinline__ Lengths read_lengths(const Schedule& s, int lane) {
  Lengths r;
  r.first = lane < s.batch ? context_length(s, lane) : 0;
  int sum = lane < s.batch ? tiles_of(r.first) : 0;
  for (int b = lane + 64; b < s.batch; b += 64) sum += tiles_of(context_length(s, b));
  const int total = __builtin_amdgcn_readlane(wave_prefix(sum), 63);
  // One round of workgroups, unless that makes short runs: then half as many, as a workgroup's start and
  // its partial results cost as much as some tiles (D128 e4m3, both kernels: B8 Hkv1 G32 L16384 25.3 ->
  // 21.8 us, G8 16.7 -> 15.4; B1 Hkv8 G4 L2000 with 4 tiles 10.7, 2 tiles 9.6).
  r.chunk = max((total + s.runs - 1) / s.runs, kMinRun);
  if (r.chunk < kLongRun) r.chunk = max(r.chunk, min((total + s.fewer - 1) / s.fewer, kLongRun));
  // Long runs are of an odd number of tiles: a power of two's start in step on the memory's channels
  // (B32 of 8192 equal keys: runs of 64 tiles 102 us, of 65 97).
  if (r.chunk >= 2 * kLongRun) r.chunk |= 1;
  return r;
}

__device__ __forceinline__ int runs_of(const Schedule& s, int chunk, int tiles) {
  return tiles <= s.whole ? 1 : (tiles + chunk - 1) / chunk;
}

struct Run {
  int b, length, split, splits, flat0;  // flat0: the sequence's first flat run
};

// Sequence and split of flat run f (all wave-uniform); false past the last.
__device__ __forceinline__ bool find_run(const Schedule& s, const Lengths& n, int f, int lane,
                                         Run& out) {
  int before = 0;
  for (int b0 = 0; b0 < s.batch; b0 += 64) {
    const int b = b0 + lane;
    const int len = b0 == 0 ? n.first : (b < s.batch ? context_length(s, b) : 0);
    const int mine = b < s.batch ? runs_of(s, n.chunk, tiles_of(len)) : 0;
    const int upto = before + wave_prefix(mine);
    const uint64_t hit = __ballot(upto > f);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      out.b = b0 + at;
      out.length = __builtin_amdgcn_readlane(len, at);
      out.splits = __builtin_amdgcn_readlane(mine, at);
      out.flat0 = __builtin_amdgcn_readlane(upto, at) - out.splits;
      out.split = f - out.flat0;
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// Splits and first flat run of sequence b (wave-uniform).
__device__ __forceinline__ void sequence_runs(const Schedule& s, const Lengths& n, int b, int lane,
                                              Run& out) {
  int before = 0;
  for (int b0 = 0; b0 <= b; b0 += 64) {
    const int i = b0 + lane;
    const int len = b0 == 0 ? n.first : (i < s.batch ? context_length(s, i) : 0);
    const int mine = i < s.batch ? runs_of(s, n.chunk, tiles_of(len)) : 0;
    const int upto = before + wave_prefix(mine);
    if (b < b0 + 64) {
      out.splits = __builtin_amdgcn_readlane(mine, b - b0);
      out.flat0 = __builtin_amdgcn_readlane(upto, b - b0) - out.splits;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
}

// LDS ring of 16-bit tiles: rows stored whole, chunks swizzled, as the DMA writes contiguous LDS.
template <int D>
struct Ring {
  static constexpr int RB = D * 2;             // bytes per row
  static constexpr int TILE = kTileKeys * RB;  // bytes per tensor tile
  static constexpr int STAGE = 2 * TILE;
  static constexpr int IPT = TILE / 1024;      // DMA instructions per tensor tile
  static constexpr int RPI = 1024 / RB;        // rows per DMA instruction
  static constexpr int CPR = RB / 16;          // 16-byte chunks per row
  // K: chunk c of row r at slot c ^ kswz(r): a ds_read_b128 phase (16 lanes, one chunk of 16
  // rows) touches 16 distinct bank groups. V: 32-byte granule g of row r at g ^ vswz(r): a
  // transposing read's phase takes one granule of 8 rows, on distinct positions.
  static __device__ __forceinline__ int kswz(int r) { return D == 128 ? (r & 15) : ((r >> 1) & 7); }
  static __device__ __forceinline__ int vswz(int r) { return D == 128 ? (r & 7) : ((r >> 1) & 3); }
};

// A wave-uniform address, asserted to the compiler, so that buffer descriptors built from it stay
// in scalar registers.
__device__ __forceinline__ void* uniform_ptr(const void* p) {
  const uint64_t x = reinterpret_cast<uintptr_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(x >> 32));
  return reinterpret_cast<void*>((uint64_t(hi) << 32) | lo);
}

// A buffer of `rows` rows of `row` bytes, `stride` bytes apart: what lies past the last row's end
// reads as zero without an access.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const void* p, int rows,
                                                              uint32_t stride, int row) {
  const uint32_t range = rows > 0 ? uint32_t(rows - 1) * stride + row : 0;
  return __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(p), (short)0,
                                           __builtin_amdgcn_readfirstlane(range), 0x00020000);
}

// ---- Joining partial results. One wave a row, or, for rows that leave CUs idle (at most kFewRows), a
// workgroup of four: the parts are shared out among them (8 rows of 128 parts 21.3 -> 16.4 us for both
// kernels, 1024 rows of few parts 92.5 -> 98.8). L = D / 4 lanes hold a partial row of O as float4, 64 / L
// of them at a time in a wave, each slice of the lanes with a running maximum of its own; slices are
// joined by exchanges, waves through LDS. The order is fixed.
constexpr int kJoinWaves = 4;
constexpr int64_t kFewRows = 256;

template <int D>
struct JoinScratch {
  tk_attn::f32x4 acc[kJoinWaves][D / 4];
  float top[kJoinWaves], sum[kJoinWaves];
};

// slot(i): index of part i of `parts`, i of which part_ml holds (reference of the exponentials, their sum)
// and part_o D unnormalized floats. Writes the row of the output and, where `lse` is not null, its base-2
// LSE; no weight at all gives 0 and -inf. References lie kLift below maxima: without it the sum's logarithm
// is the smaller and the LSE's rounding with it (7.7e-8 of it for 4.5e-8). WAVES of the workgroup's waves,
// `wave` among them, join the row.
template <typename T, int D, int WAVES, int kLift = 0, typename Slot>
__device__ __forceinline__ void join_parts(const float* part_o, const float2* part_ml, int parts, Slot slot, T* out,
                                           float* lse, int wave, JoinScratch<D>& shared) {
  using tk_attn::f32x4;
  constexpr int L = D / 4, S = 64 / L;
  const int lane = threadIdx.x & 63;
  const int d = lane % L;
  float top = kNoMax, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = (WAVES == 1 ? 0 : wave * S) + lane / L; i < parts; i += WAVES * S) {
    const int64_t at = slot(i);
    const float2 ml = part_ml[at];
    const f32x4 v = *reinterpret_cast<const f32x4*>(part_o + at * D + 4 * d);
    const float next = fmaxf(top, ml.x);
    const float old = __builtin_amdgcn_exp2f(top - next), fresh = __builtin_amdgcn_exp2f(ml.x - next);
    top = next;
    sum = sum * old + ml.y * fresh;
    acc = acc * old + v * fresh;
  }
#pragma unroll
  for (int x = L; x < 64; x <<= 1) {
    const float other = __shfl_xor(top, x);
    const float next = fmaxf(top, other);
    const float mine = __builtin_amdgcn_exp2f(top - next), theirs = __builtin_amdgcn_exp2f(other - next);
    top = next;
    sum = sum * mine + __shfl_xor(sum, x) * theirs;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = acc[i] * mine + __shfl_xor(acc[i], x) * theirs;
  }
  if constexpr (WAVES > 1) {
    if (lane < L) shared.acc[wave][d] = acc;
    if (lane == 0) {
      shared.top[wave] = top;
      shared.sum[wave] = sum;
    }
    __syncthreads();
    if (wave != 0) return;
    float high = kNoMax;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) high = fmaxf(high, shared.top[i]);
    sum = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      const float w = __builtin_amdgcn_exp2f(shared.top[i] - high);
      sum += shared.sum[i] * w;
      acc += shared.acc[i][d] * w;
    }
    top = high;
  }
  if (lane >= L) return;
  float row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) row[i] = sum == 0.f ? 0.f : acc[i] / sum;
  tk::store_vec<T, 4>(out + 4 * d, row);
  if (lane == 0 && lse != nullptr) *lse = sum == 0.f ? -INFINITY : top + kLift + log2f(sum * (1.f / (1 << kLift)));
}

}  // namespace tk_runs
