// Attention of drafted tokens over a KV cache and over each other: sequence b has `nodes` query
// tokens, each of which sees the first clamp(seqlens[b], 0, max_len) cache keys and the drafted
// keys that its row of the mask names. Query head h reads KV head h / (q_heads / kv_heads).
//
// The nodes x group query rows of one KV head form one matrix (row r = node r / group, head
// r % group), so each key is read once for all of them. Split kernel: a workgroup of W waves
// takes 16 W MT rows (MT row tiles per wave) over a run of 32-key tiles; the drafted keys are
// the tiles behind the context's. Both products run on v_mfma_f32_16x16x32 with the keys as the
// first operand's rows, as in the one-token decode:
//   S^T (16 keys x 16 rows) = K . Q^T, Q^T in registers; a row's maximum and sum are over a
//     lane's values and lanes ^ 16, ^ 32.
//   O^T (16 dims x 16 rows) += V^T . P^T, P^T from the score registers, V^T by transposing LDS
//     reads.
// K and V tiles reach LDS by non-temporal buffer->LDS DMA into one ring per workgroup (each wave
// fetches its share; one barrier per tile), so LDS holds a key once for all waves. Rows outside
// the context or the tree lie outside the tile's buffer range and arrive as zeros.
//
// Softmax statistics and sums are float32, P is rounded to the storage dtype for the second
// product (as in every attention of this library; bfloat16 results are 2.3e-3 from float64's instead
// of 1.7e-3), O once at the end.
//
// Masked keys must not reach a row by way of 0 * inf or 0 * NaN in the second product. Past the
// context's end V is zero; a drafted tile's V is checked, and if it holds an infinity or a NaN
// the tile is added key by key, and only to the rows that see the key.
//
// Splits: the tiles of all sequences are shared out in equal runs of `chunk` tiles, found by
// every workgroup from the lengths (which only the device knows), so a ragged batch fills the
// chip evenly whatever max_len is. A sequence that is one run is normalized and written by its
// workgroup; longer ones are joined by the combine kernel in a fixed order.
//
// What bounds it (D128 bf16, Hkv8, split + combine kernel): up to 128 rows per KV head HBM, and for
// short contexts the chain of latencies (2.5 us to find the run, 1.5 to the first tile, about 0.75
// per tile, 1.5 and more for the partial results). B1 T8 G4 L2000 (32 rows): 9 + 4 us. B16 T16 G4
// of lengths up to 8192 (64 rows, 304 MB): 57 + 6.4 us, 5.3 TB/s in the split kernel; equal lengths
// of 8192 with 16 or 32 rows 6.3 to 6.5 TB/s. B1 T64 G4 L131072 (256 rows, 538 MB, 137.5 GFLOP):
// 135 to 146 + 7.6 us, about 0.97 PFLOP/s; of it 10 us before the key loop (4 with fewer rows; what
// the others consist of is not known) and 6 to 10 behind it (33.5 MB of partial results). No unit is
// full there: of a wave's 269 k cycles the SIMD's matrix unit is busy 132 k, other vector
// instructions issue for 95 k, and the wave stands ready but not issued for 91 k and waits for reads
// or barriers for 74 k. Half the LDS reads, or the same tile read again and again, takes as long;
// without the exponentials it is 8 % shorter. 129 to 192 rows take this shape too, idle waves
// multiplying zeros: 132 rows of the same cache 131 to 138 + 6 us, 160 rows 134 to 137 + 6.3, 192
// rows 136 to 138 + 6.9.
// D64, same heads: B1 T64 L131072 (269 MB, 68.7 GFLOP) 88 to 91 + 8.2 us; B16 T16 L8192 (64 rows,
// 270 MB) 52 + 6, ragged up to 8192 (152 MB) 34.6 + 5.5.
// Measured and not kept: four waves of 64 rows, one per SIMD, with the exponentials of one tile
// between the products of another (175 to 193 us: a wave issues in order, and its issue slots are
// the bound); the DMA spread over the matrix phase (150 us against 147); default-policy loads
// (B16: 66.8 us against 57.8); non-temporal stores of partial results (B16 L1024 24.8 -> 21.3 us,
// ragged 57 -> 61); all V reads of a tile up front (B1 L2000 9.1 -> 9.7 us).
#include <type_traits>

#include "attention_dma.hpp"
#include "tk_common.hpp"

namespace {

using tk_attn::f32x4;
using tk_attn::i32x2;
using tk_attn::i32x4;

constexpr int kTileKeys = 32;
constexpr int kMaxNodes = 256;
constexpr int kMaskWords = kMaxNodes / 32;
constexpr int kNonTemporal = 2;
constexpr float kLog2e = 1.4426950408889634f;
// The running maximum before any key: finite, so that a masked score (-inf) minus it stays
// -inf, and below every score that carries weight.
constexpr float kNoMax = -3.0e38f;

struct TreeArgs {
  const void *q, *k, *v, *k_tree, *v_tree;
  const uint8_t* mask;
  const int32_t* seqlens;
  void* o;
  float* lse;
  float* part_o;   // [slot][row][D], slot = (flat split, KV head)
  float2* part_ml; // [slot][row]
  int64_t qb, qh, qt, ob, oh, ot;
  int64_t kb, kh, kl, vb, vh, vl;
  int64_t ktb, kth, ktl, vtb, vth, vtl;
  int64_t mb, mt;
  int batch, q_heads, kv_heads, group, nodes, rows, max_len;
  tk::FastDiv by_group, by_kv_heads, by_row_blocks;
  int tree_tiles, runs, row_blocks, flat;  // flat: upper bound on the flat splits
  int whole;         // a sequence of at most this many tiles is one run
  int heads_blocks;  // kv_heads * row_blocks
  int many;          // tiles of all sequences that make 128 * 16 with heads_blocks
  float scale_log2;  // positive
  int flip;          // Q's sign bits to turn (a negative scale)
};

// ---- Runs of tiles

// 32-key tiles of sequence b: the context's and the tree's.
__device__ __forceinline__ int context_length(const TreeArgs& a, int b) {
  const int n = a.seqlens != nullptr ? a.seqlens[b] : a.max_len;
  return min(max(n, 0), a.max_len);
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

// Tiles of the shortest run of a sequence that is split.
constexpr int kMinChunk = 4;

struct Lengths {
  int first;  // this lane's sequence's length (sequence = lane)
  int chunk;  // tiles per run
};

__device__ __forceinline__ int tiles_of(const TreeArgs& a, int length) {
  return (length + kTileKeys - 1) / kTileKeys + a.tree_tiles;
}

__device__ __forceinline__ Lengths read_lengths(const TreeArgs& a, int lane) {
  Lengths r;
  r.first = lane < a.batch ? context_length(a, lane) : 0;
  int sum = lane < a.batch ? tiles_of(a, r.first) : 0;
  for (int b = lane + 64; b < a.batch; b += 64) sum += tiles_of(a, context_length(a, b));
  const int total = __builtin_amdgcn_readlane(wave_prefix(sum), 63);
  // One round of workgroups, unless that makes runs of less than 8 tiles: then about 128
  // workgroups with runs of 4 to 16, as fewer partial results are worth more than idle CUs (D128
  // Hkv8, split + combine: B4 64 rows L1024 20.4 -> 17.1 us, B8 128 rows L1024 33.9 -> 29.8; with
  // longer runs for all that make less than 16, B4 128 rows L4096 37.2 -> 39.7).
  r.chunk = (total + a.runs - 1) / a.runs;
  if (r.chunk < 8) {
    const int few = total >= a.many ? 16 : int(uint32_t(total * a.heads_blocks) / 128);
    r.chunk = max(max(few, r.chunk), kMinChunk);
  }
  return r;
}

// Runs of a sequence of `tiles` tiles.
__device__ __forceinline__ int runs_of(const TreeArgs& a, const Lengths& n, int tiles) {
  return tiles <= a.whole ? 1 : (tiles + n.chunk - 1) / n.chunk;
}

struct Run {
  int b, length, split, splits, flat0;  // flat0: the sequence's first flat split
};

// Sequence and split of flat split f (all wave-uniform); false past the last.
__device__ __forceinline__ bool find_run(const TreeArgs& a, const Lengths& n, int f, int lane,
                                         Run& out) {
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane;
    const int len = b0 == 0 ? n.first : (b < a.batch ? context_length(a, b) : 0);
    const int mine = b < a.batch ? runs_of(a, n, tiles_of(a, len)) : 0;
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

// Splits and first flat split of sequence b (wave-uniform).
__device__ __forceinline__ void sequence_runs(const TreeArgs& a, const Lengths& n, int b, int lane,
                                              Run& out) {
  int before = 0;
  for (int b0 = 0; b0 <= b; b0 += 64) {
    const int i = b0 + lane;
    const int len = b0 == 0 ? n.first : (i < a.batch ? context_length(a, i) : 0);
    const int mine = i < a.batch ? runs_of(a, n, tiles_of(a, len)) : 0;
    const int upto = before + wave_prefix(mine);
    if (b < b0 + 64) {
      out.splits = __builtin_amdgcn_readlane(mine, b - b0);
      out.flat0 = __builtin_amdgcn_readlane(upto, b - b0) - out.splits;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
}

// ---- LDS ring (rows stored whole, chunks swizzled, as the DMA writes contiguous LDS)

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

__device__ __forceinline__ void* uniform_ptr(const void* p) {
  const uint64_t x = reinterpret_cast<uintptr_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(x >> 32));
  return reinterpret_cast<void*>((uint64_t(hi) << 32) | lo);
}

// The stream of a run's tiles into the ring: context rows, then the tree's. All fields but the
// lane offsets are wave-uniform.
template <typename T, int D, int W>
struct Fetcher {
  using R = Ring<D>;
  static constexpr int PER = R::IPT / W;  // this wave's instructions per tensor tile
  const char *k, *v;        // first row of the next tile
  const T *k_tree, *v_tree;
  uint32_t k2, v2;          // bytes per row
  uint32_t kt2, vt2;
  int left;                 // rows from there to the end of the run's part of the segment
  int tiles;                // of this segment (padded with empty ones), not yet issued
  int tree_rows;            // rows of the tree in the run, 0 once it is the current segment
  char* dst;                // this wave's share of the ring's first stage
  uint32_t koff[PER], voff[PER];

  __device__ __forceinline__ void offsets(int wave, int lane) {
    // Instruction i covers rows RPI (wave PER + i) .. +RPI-1; the lane fetches the chunk that
    // belongs at its LDS slot.
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = (wave * PER + i) * R::RPI + lane / R::CPR;
      const int slot = lane % R::CPR;
      koff[i] = r * k2 + (slot ^ R::kswz(r)) * 16;
      voff[i] = r * v2 + ((((slot >> 1) ^ R::vswz(r)) << 1) | (slot & 1)) * 16;
    }
  }

  // The next tile into `stage`. Tiles past a segment's rows (issued to fill a step and to keep
  // the wait counts static) have an empty range: nothing is read, LDS gets zeros.
  __device__ __forceinline__ void next(int stage, int wave, int lane) {
    if (tiles <= 0 && tree_rows > 0) {
      k = reinterpret_cast<const char*>(k_tree);
      v = reinterpret_cast<const char*>(v_tree);
      k2 = kt2;
      v2 = vt2;
      left = tree_rows;
      tree_rows = 0;
      offsets(wave, lane);
    }
    const int rows = min(left, kTileKeys);
    // The last row ends D elements in: bytes past it are outside the range.
    const uint32_t krange = rows > 0 ? uint32_t(rows - 1) * k2 + D * 2 : 0;
    const uint32_t vrange = rows > 0 ? uint32_t(rows - 1) * v2 + D * 2 : 0;
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
        uniform_ptr(k), (short)0, __builtin_amdgcn_readfirstlane(krange), 0x00020000);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
        uniform_ptr(v), (short)0, __builtin_amdgcn_readfirstlane(vrange), 0x00020000);
    char* to = dst + stage * R::STAGE;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (tk_attn::lds_void*)(to + i * 1024), 16, koff[i],
                                               0, 0, kNonTemporal);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (tk_attn::lds_void*)(to + R::TILE + i * 1024),
                                               16, voff[i], 0, 0, kNonTemporal);
    k += kTileKeys * int64_t(k2);
    v += kTileKeys * int64_t(v2);
    left -= kTileKeys;
    --tiles;
  }
};

// Largest |x| bit pattern of packed 16-bit values, kept per half.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 max_magnitude(u16x2 m, int x) {
  return __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x & 0x7FFF7FFF));
}

// The elements of a fragment that belong to key j of the tile (element e of this lane is key
// 16 (e / 4) + 4 quad + e % 4), the others zero.
__device__ __forceinline__ i32x4 only_key(i32x4 f, int j, int quad) {
  i32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int key = 16 * (i / 2) + 4 * quad + 2 * (i % 2);
    r[i] = key == j ? (f[i] & 0xFFFF) : key + 1 == j ? int(uint32_t(f[i]) & 0xFFFF0000u) : 0;
  }
  return r;
}

// KT tiles per step (one barrier each), NS ring stages.
template <typename T, int D, int W, int MT, int KT, int NS>
__global__ __launch_bounds__(64 * W, W >= 4 ? 2 : 1) void tree_split_kernel(TreeArgs a) {
  using R = Ring<D>;
  // Ping-pong (eight waves, two per SIMD): see the context loop.
  constexpr bool PP = W == 8;
  constexpr int RS = NS / KT;          // steps the ring holds
  constexpr int LA = PP ? 2 : RS - 1;  // steps fetched ahead
  static_assert(NS % KT == 0 && RS >= 2 && (!PP || RS >= 4), "a stage is refilled while it is read");
  constexpr int DC = D / 32, OC = D / 16, RB = R::RB, PER = R::IPT / W;
  // vmcnt is 6 bits: at most 63 DMA instructions may be outstanding.
  constexpr int STEP = KT * 2 * PER;   // this wave's DMA instructions per step
  static_assert(LA * STEP < 64, "ring deeper than the vmcnt counter");
  constexpr int ROWS = 16 * W * MT;
  constexpr int HB = 4;  // output chunks per batch of V reads
  constexpr int NONFINITE = __is_same(T, __bf16) ? 0x7F80 : 0x7C00;
  __shared__ __attribute__((aligned(1024))) char ring[NS * R::STAGE];
  // Drafted keys by the block's nodes; behind them the waves' SIMDs.
  __shared__ uint32_t seen[ROWS * kMaskWords + W];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroup -> (flat split, KV head, row block): the row blocks of a run are dealt to one XCD
  // (workgroup index modulo 8), one after the other, so that they share its L2.
  const int eighth = a.by_row_blocks.div(blockIdx.x / 8);
  const int pair = eighth * 8 + blockIdx.x % 8;
  const int rb = blockIdx.x / 8 - eighth * a.row_blocks;
  const int f = a.by_kv_heads.div(pair);
  const int kvh = pair - f * a.kv_heads;
  const Lengths lengths = read_lengths(a, lane);
  Run run;
  if (f >= a.flat || !find_run(a, lengths, f, lane, run)) return;

  const int b = run.b;
  const int context_tiles = (run.length + kTileKeys - 1) / kTileKeys;
  const int t0 = run.split * lengths.chunk;
  const int tiles = context_tiles + a.tree_tiles;
  const int t1 = run.splits == 1 ? tiles : min(t0 + lengths.chunk, tiles);
  const int c1 = min(t1, context_tiles);  // context tiles t0 .. c1-1, then drafted ones
  const int limit = min(run.length, c1 * kTileKeys);

  const int row16 = lane & 15;
  const int quad = lane >> 4;
  const int r0 = rb * ROWS;
  const int w0 = r0 + wave * 16 * MT;   // this wave's first row
  const bool busy = w0 < a.rows;        // waves past the last row only fetch
  const int node0 = a.by_group.div(r0);

  Fetcher<T, D, W> fetch;
  {
    const bool drafted = t0 >= context_tiles;
    const int first = (drafted ? t0 - context_tiles : t0) * kTileKeys;
    const T* kc = static_cast<const T*>(a.k) + b * a.kb + kvh * a.kh;
    const T* vc = static_cast<const T*>(a.v) + b * a.vb + kvh * a.vh;
    fetch.k_tree = static_cast<const T*>(a.k_tree) + b * a.ktb + kvh * a.kth;
    fetch.v_tree = static_cast<const T*>(a.v_tree) + b * a.vtb + kvh * a.vth;
    fetch.k = reinterpret_cast<const char*>(drafted ? fetch.k_tree + first * a.ktl
                                                    : kc + first * a.kl);
    fetch.v = reinterpret_cast<const char*>(drafted ? fetch.v_tree + first * a.vtl
                                                    : vc + first * a.vl);
    fetch.kt2 = uint32_t(a.ktl * 2);
    fetch.vt2 = uint32_t(a.vtl * 2);
    fetch.k2 = drafted ? fetch.kt2 : uint32_t(a.kl * 2);
    fetch.v2 = drafted ? fetch.vt2 : uint32_t(a.vl * 2);
    const int tree_rows = min(a.nodes, (t1 - context_tiles) * kTileKeys);
    fetch.left = (drafted ? tree_rows : limit) - first;
    fetch.tiles = ((max(c1 - t0, 0) + KT - 1) / KT) * KT;
    fetch.tree_rows = drafted ? 0 : tree_rows;
    fetch.dst = ring + wave * PER * 1024;
    fetch.offsets(wave, lane);
  }
#pragma unroll
  for (int i = 0; i < LA * KT; ++i) fetch.next(i, wave, lane);

  // Q^T fragments: row w0 + 16 mt + row16 (zero past the last), dims 32 c + 8 quad .. +7. A
  // negative scale is taken into Q's signs (exact), so that the largest score is the largest
  // product.
  i32x4 qf[MT][DC];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = w0 + 16 * m + row16;
    const int node = a.by_group.div(r);
    const int h = kvh * a.group + (r - node * a.group);
    const T* p = static_cast<const T*>(a.q) + b * a.qb + h * a.qh + node * a.qt + 8 * quad;
#pragma unroll
    for (int c = 0; c < DC; ++c)
      qf[m][c] = r < a.rows ? *reinterpret_cast<const i32x4*>(p + 32 * c) : i32x4{0, 0, 0, 0};
  }
  // The block's nodes' mask rows as bits, if the run holds drafted tiles; eight rows of a wave
  // are requested at a time.
  if (t1 > context_tiles) {
    const int last = a.by_group.div(min(r0 + ROWS, a.rows) - 1);
    const uint8_t* mask = a.mask + b * a.mb;
    for (int j0 = 0; j0 < a.nodes; j0 += 64) {
      const int j = j0 + lane;
      for (int n0 = node0 + wave; n0 <= last; n0 += 8 * W) {
        uint8_t byte[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int n = n0 + i * W;
          byte[i] = j < a.nodes && n <= last ? mask[n * a.mt + j] : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int n = n0 + i * W;
          const uint64_t bits = __ballot(byte[i] != 0);
          if (lane < 2 && n <= last)
            seen[(n - node0) * kMaskWords + j0 / 32 + lane] = uint32_t(bits >> (32 * lane));
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      qf[m][c] ^= a.flip;
      tk_attn::pin(qf[m][c]);
    }

  const uint32_t ring_base = (uint32_t)(uintptr_t)(tk_attn::lds_void*)ring;
  uint32_t ka[DC], va[OC];
#pragma unroll
  for (int c = 0; c < DC; ++c) ka[c] = row16 * RB + (((4 * c + quad) ^ R::kswz(row16)) * 16);
  const int trow = 4 * quad + (row16 >> 2);
#pragma unroll
  for (int c = 0; c < OC; ++c)
    va[c] = R::TILE + trow * RB + ((c ^ R::vswz(trow)) * 32) + 8 * (row16 & 3);

  f32x4 o[MT][OC];
  float top[MT], sum[MT];  // reference maximum of row row16, this lane's share of its sum
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    top[m] = kNoMax;
    sum[m] = 0.f;
#pragma unroll
    for (int c = 0; c < OC; ++c) o[m][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float scale = a.scale_log2;

  int step = 0;  // modulo RS, the ring's next step to read
  auto fetch_step = [&](int slot) {
#pragma unroll
    for (int i = 0; i < KT; ++i) fetch.next(slot * KT + i, wave, lane);
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step has landed (this wave's share) once only the LA - 1 younger steps' loads are
  // outstanding; behind the barrier every wave's share has, and every wave has read the step
  // before it, whose slot (or a free one) the step fetched now takes. Returns the step's stage.
  auto arrive = [&]() {
    tk_attn::wait_vmcnt<(LA - 1) * STEP>();
    if constexpr (W > 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    fetch_step(step + LA < RS ? step + LA : step + LA - RS);
    const uint32_t sb = ring_base + step * KT * R::STAGE;
    step = step == RS - 1 ? 0 : step + 1;
    return sb;
  };
  // s[n][m][i][r]: product of row row16 of row tile m and key 16 i + 4 quad + r of the n-th of N
  // tiles. The fragments of DEPTH 32-feature steps are in flight at a time, so that the first
  // products start while the later reads are still on their way.
  constexpr int DEPTH = 4 < DC ? 4 : DC;
  auto request_k = [&](uint32_t sb, auto& kc, int u) {
    kc[u][0] = tk_attn::lds_read_b128<0>(sb + (u / DC) * R::STAGE + ka[u % DC]);
    kc[u][1] = tk_attn::lds_read_b128<16 * RB>(sb + (u / DC) * R::STAGE + ka[u % DC]);
  };
  auto request_first_k = [&](uint32_t sb, auto& kc) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) request_k(sb, kc, u);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto products = [&](uint32_t sb, auto& kc, auto& s) {
    constexpr int U = sizeof(kc) / sizeof(kc[0]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int younger = (u + DEPTH < U ? u + DEPTH : U) - (u + 1);
      if (younger >= 3)
        tk_attn::wait_lgkm<6>();
      else if (younger == 2)
        tk_attn::wait_lgkm<4>();
      else if (younger == 1)
        tk_attn::wait_lgkm<2>();
      else
        tk_attn::wait_lgkm<0>();
      tk_attn::pin(kc[u][0]);
      tk_attn::pin(kc[u][1]);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          s[u / DC][m][i] = tk_attn::Mma16<T>::run(
              kc[u][i], qf[m][u % DC],
              u % DC == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[u / DC][m][i]);
      if (u + DEPTH < U) request_k(sb, kc, u + DEPTH);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // P = exp2(scale s - top) of N tiles into pf. The reference maximum moves only when the
  // tiles' exceeds it by more than 8 (base 2), so p <= 2^8 and o and sum are rescaled in few
  // steps: a lane whose exponentials sum to at most 2^8 has none above it, and then no maximum
  // is formed.
  auto softmax = [&](auto& s, auto& pf) {
    constexpr int N = sizeof(s) / sizeof(f32x4[MT][2]);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      f32x4 p[N][2];
      float part = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[n][i][r] = __builtin_amdgcn_exp2f(fmaf(s[n][m][i][r], scale, -top[m]));
            part += p[n][i][r];
          }
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(part <= 256.f)) != 0, 0)) {
        float high = s[0][m][0][0];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) high = fmaxf(high, s[n][m][i][r]);
        high = tk_attn::max_over_column(high) * scale;
        const float next = high > top[m] + 8.f ? high : top[m];
        const float alpha = __builtin_amdgcn_exp2f(top[m] - next);
        top[m] = next;
        sum[m] *= alpha;
#pragma unroll
        for (int c = 0; c < OC; ++c) o[m][c] *= alpha;
        part = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              p[n][i][r] = __builtin_amdgcn_exp2f(fmaf(s[n][m][i][r], scale, -next));
              part += p[n][i][r];
            }
      }
      sum[m] += part;
#pragma unroll
      for (int n = 0; n < N; ++n) pf[n][m] = tk_attn::acc_frag2<T>(p[n][0], p[n][1]);
    }
  };
  // o += V^T P^T of a tile; the first batch of its V fragments is already on its way, and what
  // comes next is sent for before the last batch's products.
  i32x2 lo[OC], hi[OC];
  auto request_v = [&](uint32_t sb, int c0) {
#pragma unroll
    for (int c = c0; c < c0 + HB; ++c) {
      lo[c] = tk_attn::lds_read_tr16<0>(sb + va[c]);
      hi[c] = tk_attn::lds_read_tr16<16 * RB>(sb + va[c]);
    }
  };
  auto accumulate = [&](uint32_t sb, const i32x4(&pf)[MT], auto&& request_next) {
#pragma unroll
    for (int c0 = 0; c0 < OC; c0 += HB) {
      tk_attn::wait_lgkm<0>();
      i32x4 vf[HB];
#pragma unroll
      for (int c = 0; c < HB; ++c) {
        asm volatile("" : "+v"(lo[c0 + c]), "+v"(hi[c0 + c]));
        vf[c] = i32x4{lo[c0 + c][0], lo[c0 + c][1], hi[c0 + c][0], hi[c0 + c][1]};
      }
      if (c0 + HB < OC)
        request_v(sb, c0 + HB);
      else
        request_next();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < HB; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          o[m][c0 + c] = tk_attn::Mma16<T>::run(vf[c], pf[m], o[m][c0 + c]);
    }
  };
  auto accumulate_step = [&](uint32_t sb, const i32x4(&pf)[KT][MT], auto&& request_next) {
    if constexpr (KT == 2) {
      accumulate(sb, pf[0], [&]() { request_v(sb + R::STAGE, 0); });
      accumulate(sb + R::STAGE, pf[1], request_next);
    } else {
      accumulate(sb, pf[0], request_next);
    }
  };
  auto nothing = []() {};
  // The keys past the run's context in the step from tile t on are no keys.
  auto cut = [&](int t, f32x4(&s)[KT][MT][2]) {
    const int live = limit - t * kTileKeys;
    if (__builtin_expect(live < KT * kTileKeys, 0)) {
#pragma unroll
      for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (32 * n + 16 * i + 4 * quad + r >= live) s[n][m][i][r] = -INFINITY;
    }
  };

  if constexpr (!PP) {
    for (int t = t0; t < c1; t += KT) {
      const uint32_t sb = arrive();
      if (!busy) continue;
      f32x4 s[KT][MT][2];
      i32x4 pf[KT][MT], kc[KT * DC][2];
      request_first_k(sb, kc);
      products(sb, kc, s);
      request_v(sb, 0);
      cut(t, s);
      softmax(s, pf);
      accumulate_step(sb, pf, nothing);
    }
  } else if (c1 > t0) {
    // Eight waves, two per SIMD, in phases ended by barriers: a wave alternates a matrix phase
    // (step j - 1's output products, then step j's scores) with a softmax phase, the second wave
    // of each SIMD (by the hardware's SIMD id) one phase behind the first, so that one wave's
    // exponentials run beside the other's products (B1 T64 G4 L131072 148 -> 143 us). Step j's
    // slot is read in phases 2j .. 2j + 3; step j + 2, fetched from phase 2j on, takes the slot of
    // step j - 2. Waves without rows run along on zeros.
    const int steps = (c1 - t0 + KT - 1) / KT;
    int second = 0;
    {
      int* simd = reinterpret_cast<int*>(&seen[ROWS * kMaskWords]);
      if (lane == 0) simd[wave] = tk_attn::simd_id();
      tk_attn::wait_vmcnt<STEP>();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int w = 0; w < W; ++w) second += w < wave && simd[w] == simd[wave] ? 1 : 0;
      second = __builtin_amdgcn_readfirstlane(second) & 1;
    }
    f32x4 s[KT][MT][2];
    i32x4 pf[KT][MT];
    auto stage_of = [&](int j) { return ring_base + (j % RS) * KT * R::STAGE; };
    // Step j + 2 is fetched from phase 2j on, and step j + 1 has landed by the end of phase 2j + 1.
    auto matrix_end = [&](int j) {
#pragma unroll
      for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          tk_attn::pin(s[n][m][0]);
          tk_attn::pin(s[n][m][1]);
        }
      if (second) tk_attn::wait_vmcnt<STEP>();
      tk_attn::barrier_no_fence();
      if (second && j + 1 < steps) fetch_step((j + 3) % RS);
    };
    auto softmax_phase = [&](int j) {
      cut(t0 + j * KT, s);
      softmax(s, pf);
#pragma unroll
      for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) tk_attn::pin(pf[n][m]);
      if (!second) tk_attn::wait_vmcnt<STEP>();
      tk_attn::barrier_no_fence();
      if (!second && j + 1 < steps) fetch_step((j + 3) % RS);
    };
    // A matrix phase as a pipeline of read units, four of them in flight: output units (a tile's
    // pair of output chunks: four transposing reads) of the step before, then score units (a
    // tile's 32-feature step: two reads).
    auto matrix_phase = [&](auto with_output, auto with_scores, uint32_t last, uint32_t now) {
      constexpr int NV = decltype(with_output)::value ? KT * OC / 2 : 0;
      constexpr int NU = NV + (decltype(with_scores)::value ? KT * DC : 0);
      constexpr int IN_FLIGHT = 4;
      i32x2 vlo[KT * OC / 2][2], vhi[KT * OC / 2][2];
      i32x4 kc[KT * DC][2];
      auto issue = [&](int u) {
        if (u < NV) {
          const uint32_t at = last + (u / (OC / 2)) * R::STAGE;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t v = at + va[2 * (u % (OC / 2)) + x];
            vlo[u][x] = tk_attn::lds_read_tr16<0>(v);
            vhi[u][x] = tk_attn::lds_read_tr16<16 * RB>(v);
          }
        } else {
          request_k(now, kc, u - NV);
        }
      };
#pragma unroll
      for (int u = 0; u < IN_FLIGHT && u < NU; ++u) issue(u);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        int younger = 0;  // reads that may still be in flight
        for (int x = u + 1; x < u + IN_FLIGHT && x < NU; ++x) younger += x < NV ? 4 : 2;
        if (younger == 12)
          tk_attn::wait_lgkm<12>();
        else if (younger == 10)
          tk_attn::wait_lgkm<10>();
        else if (younger == 8)
          tk_attn::wait_lgkm<8>();
        else if (younger == 6)
          tk_attn::wait_lgkm<6>();
        else if (younger == 4)
          tk_attn::wait_lgkm<4>();
        else if (younger == 2)
          tk_attn::wait_lgkm<2>();
        else
          tk_attn::wait_lgkm<0>();
        if (u < NV) {
          const int n = u / (OC / 2), c = 2 * (u % (OC / 2));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            asm volatile("" : "+v"(vlo[u][x]), "+v"(vhi[u][x]));
            const i32x4 vf = {vlo[u][x][0], vlo[u][x][1], vhi[u][x][0], vhi[u][x][1]};
#pragma unroll
            for (int m = 0; m < MT; ++m)
              o[m][c + x] = tk_attn::Mma16<T>::run(vf, pf[n][m], o[m][c + x]);
          }
        } else {
          const int k = u - NV;
          tk_attn::pin(kc[k][0]);
          tk_attn::pin(kc[k][1]);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              s[k / DC][m][i] = tk_attn::Mma16<T>::run(
                  kc[k][i], qf[m][k % DC],
                  k % DC == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[k / DC][m][i]);
        }
        if (u + IN_FLIGHT < NU) issue(u + IN_FLIGHT);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const std::true_type yes;
    const std::false_type no;
    fetch_step(2 % RS);
    if (second) tk_attn::barrier_no_fence();
    matrix_phase(no, yes, 0u, stage_of(0));
    matrix_end(0);
    softmax_phase(0);
    for (int j = 1; j < steps; ++j) {
      matrix_phase(yes, yes, stage_of(j + RS - 1), stage_of(j));
      matrix_end(j);
      softmax_phase(j);
    }
    matrix_phase(yes, no, stage_of(steps - 1), 0u);
    // Both waves of a SIMD have passed 2 steps + 2 barriers, so the ring is read by none.
    tk_attn::barrier_no_fence();
    if (!second) tk_attn::barrier_no_fence();
    step = steps % RS;
  }

  for (int t = max(t0, context_tiles); t < t1; t += KT) {
    uint32_t sb = arrive();
    if (!busy) continue;
    for (int tile = t; tile < min(t + KT, t1); ++tile, sb += R::STAGE) {
      const int word = tile - context_tiles;
      uint32_t bits[MT];  // the tile's keys that row row16 sees
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = w0 + 16 * m + row16;
        bits[m] = r < a.rows ? seen[(a.by_group.div(r) - node0) * kMaskWords + word] : 0;
      }
      f32x4 s[1][MT][2];
      i32x4 pf[1][MT], kc[DC][2];
      request_first_k(sb, kc);
      products(sb, kc, s);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!((bits[m] >> (16 * i + 4 * quad + r)) & 1)) s[0][m][i][r] = -INFINITY;
      softmax(s, pf);
      u16x2 most = {0, 0};
#pragma unroll
      for (int c0 = 0; c0 < OC; c0 += HB) {
        request_v(sb, c0);
        tk_attn::wait_lgkm<0>();
#pragma unroll
        for (int c = c0; c < c0 + HB; ++c) {
          asm volatile("" : "+v"(lo[c]), "+v"(hi[c]));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            most = max_magnitude(most, lo[c][i]);
            most = max_magnitude(most, hi[c][i]);
          }
        }
      }
      if (__builtin_expect(__ballot(most[0] >= NONFINITE || most[1] >= NONFINITE) == 0, 1)) {
        request_v(sb, 0);
        accumulate(sb, pf[0], nothing);
        continue;
      }
      for (int j = 0; j < kTileKeys; ++j) {
        i32x4 pj[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) pj[m] = only_key(pf[0][m], j, quad);
#pragma unroll
        for (int c = 0; c < OC; ++c) {
          const i32x4 vj = only_key(i32x4{lo[c][0], lo[c][1], hi[c][0], hi[c][1]}, j, quad);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const f32x4 one = tk_attn::Mma16<T>::run(vj, pj[m], f32x4{0.f, 0.f, 0.f, 0.f});
            if ((bits[m] >> j) & 1) o[m][c] += one;
          }
        }
      }
    }
  }
  // The tiles issued past the end still write (zeros) into the ring.
  tk_attn::wait_vmcnt<0>();
  if (!busy) return;

  const int slot = f * a.kv_heads + kvh;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const float l = tk_attn::sum_over_column(sum[m]);
    const int r = w0 + 16 * m + row16;
    if (r >= a.rows) continue;
    if (run.splits == 1) {
      const int node = a.by_group.div(r);
      const int h = kvh * a.group + (r - node * a.group);
      const float share = l == 0.f ? 0.f : 1.f / l;
      T* dst = static_cast<T*>(a.o) + b * a.ob + h * a.oh + node * a.ot + 4 * quad;
#pragma unroll
      for (int c = 0; c < OC; ++c) {
        float out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = o[m][c][i] * share;
        tk::store_vec<T, 4>(dst + 16 * c, out);
      }
      if (quad == 0 && a.lse != nullptr)
        a.lse[(int64_t(b) * a.q_heads + h) * a.nodes + node] =
            l == 0.f ? -INFINITY : top[m] + log2f(l);
    } else {
      const int64_t at = int64_t(slot) * a.rows + r;
#pragma unroll
      for (int c = 0; c < OC; ++c)
        *reinterpret_cast<f32x4*>(a.part_o + at * D + 16 * c + 4 * quad) = o[m][c];
      if (quad == 0) a.part_ml[at] = float2{top[m], l};
    }
  }
}

// One wave per (sequence, KV head, row): L = D / 4 lanes hold a row of O as float4, 64 / L splits
// at a time, folded in a fixed order.
constexpr int kCombineWaves = 4;
template <typename T, int D>
__global__ __launch_bounds__(64 * kCombineWaves) void tree_combine_kernel(TreeArgs a) {
  constexpr int L = D / 4, S = 64 / L;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = blockIdx.x * kCombineWaves + wave;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const Lengths lengths = read_lengths(a, lane);
  Run run;
  sequence_runs(a, lengths, b, lane, run);
  if (run.splits == 1 || r >= a.rows) return;
  const int64_t step = int64_t(a.kv_heads) * a.rows;  // rows between a row's splits
  const int64_t at0 = (int64_t(run.flat0) * a.kv_heads + kvh) * a.rows + r;
  float high = kNoMax;
  for (int i = lane; i < run.splits; i += 64) high = fmaxf(high, a.part_ml[at0 + i * step].x);
  high = tk::wave_allreduce(high, tk::MaxOp{});
  float total = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int part = lane / L, d = (lane % L) * 4;
#pragma unroll 4
  for (int i = part; i < run.splits; i += S) {
    const float2 ml = a.part_ml[at0 + i * step];
    const f32x4 v = *reinterpret_cast<const f32x4*>(a.part_o + (at0 + i * step) * D + d);
    const float w = __builtin_amdgcn_exp2f(ml.x - high);
    total += ml.y * w;
    acc += v * w;
  }
#pragma unroll
  for (int x = L; x < 64; x <<= 1) {
    total += __shfl_xor(total, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], x);
  }
  if (part != 0) return;
  const int node = a.by_group.div(r);
  const int h = kvh * a.group + (r - node * a.group);
  float out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = total == 0.f ? 0.f : acc[i] / total;
  tk::store_vec<T, 4>(static_cast<T*>(a.o) + b * a.ob + h * a.oh + node * a.ot + d, out);
  if (lane == 0 && a.lse != nullptr)
    a.lse[(int64_t(b) * a.q_heads + h) * a.nodes + node] =
        total == 0.f ? -INFINITY : high + log2f(total);
}

// Workgroup shapes by the rows a KV head has: 16 rows a wave up to four waves, then more rows a
// wave, 256 rows at most. `resident`: workgroups that run at once, two per CU with a 64 KiB ring,
// one with 128 KiB (256 rows at head_dim 128, eight waves of 256 registers). Half the waves with
// twice the rows each: 32 rows 12.1 us against 10.1 (B1 L2000) and 89.5 against 87 (B16 L8192), 64
// rows level, 128 rows 67 against 57 (B8 L8192).
struct Shape {
  int rows, resident;
};
Shape shape_for(int64_t rows, int64_t head_dim) {
  for (int n : {16, 32, 64, 128})
    if (rows <= n) return {n, 512};
  return {256, head_dim == 128 ? 256 : 512};
}

// Instantiated here by name: left to the launches below, the host compiler leaves some of these
// kernels' launch stubs undefined.
#define TK_TREE_SPLIT(T, D, W, MT, KT, NS) \
  template __global__ void tree_split_kernel<T, D, W, MT, KT, NS>(TreeArgs)
#define TK_TREE_SPLITS(T)                                                           \
  TK_TREE_SPLIT(T, 128, 1, 1, 1, 4); TK_TREE_SPLIT(T, 128, 2, 1, 1, 4);             \
  TK_TREE_SPLIT(T, 128, 4, 1, 1, 4); TK_TREE_SPLIT(T, 128, 4, 2, 1, 4);             \
  TK_TREE_SPLIT(T, 128, 8, 2, 2, 8); TK_TREE_SPLIT(T, 64, 1, 1, 1, 8);              \
  TK_TREE_SPLIT(T, 64, 2, 1, 1, 8); TK_TREE_SPLIT(T, 64, 4, 1, 1, 8);               \
  TK_TREE_SPLIT(T, 64, 4, 2, 1, 8); TK_TREE_SPLIT(T, 64, 4, 4, 2, 8)
TK_TREE_SPLITS(__bf16);
TK_TREE_SPLITS(_Float16);

template <typename T, int D, int W, int MT, int KT, int NS>
void launch_split(const TreeArgs& a, dim3 grid, hipStream_t s) {
  hipLaunchKernelGGL((tree_split_kernel<T, D, W, MT, KT, NS>), grid, dim3(64 * W), 0, s, a);
}

template <typename T, int D>
void launch(const TreeArgs& a, bool combine, hipStream_t s) {
  constexpr int NS = D == 128 ? 4 : 8;
  const int64_t pairs = tk::cdiv(int64_t(a.flat) * a.kv_heads, 8) * 8;
  const dim3 grid(static_cast<uint32_t>(pairs * a.row_blocks));
  switch (shape_for(a.rows, D).rows) {
    case 16: launch_split<T, D, 1, 1, 1, NS>(a, grid, s); break;
    case 32: launch_split<T, D, 2, 1, 1, NS>(a, grid, s); break;
    case 64: launch_split<T, D, 4, 1, 1, NS>(a, grid, s); break;
    case 128: launch_split<T, D, 4, 2, 1, NS>(a, grid, s); break;
    default:
      if constexpr (D == 128)
        launch_split<T, D, 8, 2, 2, 8>(a, grid, s);
      else
        launch_split<T, D, 4, 4, 2, 8>(a, grid, s);
  }
  if (combine)
    hipLaunchKernelGGL((tree_combine_kernel<T, D>),
                       dim3(static_cast<uint32_t>(tk::cdiv(a.rows, kCombineWaves)), a.kv_heads,
                            a.batch),
                       dim3(64 * kCombineWaves), 0, s, a);
}

// A call whose caches hold at most this many tiles per sequence is not split, by its pairs of a
// sequence's KV head and a row block (with 128 pairs and more no sequence of so few tiles is, however
// long the cache): writing and joining partial results costs more than the tiles that runs of their
// own would save. D128 Hkv8, whole against split + combine: B16 (128 pairs) L1024 64 rows 24 against
// 30 us, 128 rows 32 against 40, 256 rows 45 against 55; L2048 39 against 39, 52 against 49, 70
// against 67. B4 and B8 L512 16 against 15 to 18, 21 against 21 to 24, 29 against 29 to 35; L1024
// 24 against 20, 31 against 28, 42 against 38. B1 L256 11 to 15 against as much; L512 14 against 11.
// D64 B4 lengths 300 to 500, caches of 512 (whole) against 8192: 64 rows 11.8 against 8.2 + 4.0, 256
// rows 24.3 against 19.8 + 5.8 (D128 13.8 against 10 + 4.4, 28 against 22.9 + 6.1). B16 is whole in
// both: 12.6 against 12.7 + 3.4, the joining launch that finds nothing to join.
int64_t whole_tiles(int64_t pairs) { return pairs >= 128 ? 40 : pairs >= 32 ? 18 : 10; }

// How the call is cut: runs (the tiles of all sequences over `runs` give the run length), the
// bound on their number, row blocks. The sequences' last runs are shorter, so `runs` leaves room
// for one more per sequence where that keeps the launch to one round of workgroups.
struct Plan {
  int64_t row_blocks, runs, flat, whole;
  bool combine;
};
Plan make_plan(int64_t batch, int64_t kv_heads, int64_t rows, int64_t max_len, int64_t nodes,
               int64_t head_dim) {
  Plan p;
  const Shape shape = shape_for(rows, head_dim);
  p.row_blocks = tk::cdiv(rows, shape.rows);
  const int64_t most = tk::cdiv(max_len, kTileKeys) + tk::cdiv(nodes, kTileKeys);
  const int64_t base = shape.resident / (kv_heads * p.row_blocks);
  p.runs = base > 2 * batch ? base - batch + 1 : base > 1 ? base : 1;
  const int64_t pairs = batch * kv_heads * p.row_blocks;
  p.whole = whole_tiles(pairs);
  p.combine = most > p.whole;
  // Where the lengths may ask for the combine kernel it runs in any case, and a short sequence is
  // worth splitting unless there are workgroups enough without.
  if (p.combine && pairs < 128) p.whole = 0;
  p.flat = p.runs + batch;
  const int64_t bound = p.combine ? batch * tk::cdiv(most, kMinChunk) : batch;
  if (p.flat > bound) p.flat = bound;
  return p;
}

// Why a problem of these (positive) sizes is not taken, or null. The grid holds at most 2^22
// workgroups, and tiles and partial results are counted in 32 bits.
const char* unsupported(int64_t batch, int64_t kv_heads, int64_t group, int64_t max_len,
                        int64_t nodes, int64_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
  if (nodes > kMaxNodes) return "at most 256 nodes";
  if (batch > 65535 || kv_heads > 65535 || group > 65535 || kv_heads * group > 65535 ||
      max_len > INT32_MAX - 65536)
    return "problem too large";
  const Plan p = make_plan(batch, kv_heads, nodes * group, max_len, nodes, head_dim);
  const int64_t most = tk::cdiv(max_len, kTileKeys) + tk::cdiv(nodes, kTileKeys);
  if (batch * most > INT32_MAX / 2 || p.flat * kv_heads * p.row_blocks > (1 << 22))
    return "problem too large";
  return nullptr;
}

}  // namespace

extern "C" int tk_tree_decode_slots(int64_t batch, int64_t kv_heads, int64_t group,
                                    int64_t max_len, int64_t nodes, int64_t head_dim) {
  if (batch <= 0 || kv_heads <= 0 || group <= 0 || max_len <= 0 || nodes <= 0) return -1;
  if (unsupported(batch, kv_heads, group, max_len, nodes, head_dim) != nullptr) return -1;
  const Plan p = make_plan(batch, kv_heads, nodes * group, max_len, nodes, head_dim);
  return p.combine ? static_cast<int>(p.flat * kv_heads) : 0;
}

extern "C" int tk_tree_decode(int dtype, const void* q, const void* k_cache, const void* v_cache,
                              const void* k_tree, const void* v_tree, const void* mask,
                              const int32_t* seqlens, void* o, float* lse, float* workspace,
                              int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t max_len,
                              int64_t nodes, int64_t head_dim, const int64_t* q_strides,
                              const int64_t* k_strides, const int64_t* v_strides,
                              const int64_t* k_tree_strides, const int64_t* v_tree_strides,
                              const int64_t* mask_strides, const int64_t* o_strides, float scale,
                              void* stream) {
  if (dtype != TK_DTYPE_F16 && dtype != TK_DTYPE_BF16)
    return tk::fail("tree decode: dtype must be float16 or bfloat16");
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || k_tree == nullptr ||
      v_tree == nullptr || mask == nullptr || o == nullptr ||
      q_strides == nullptr || k_strides == nullptr || v_strides == nullptr ||
      k_tree_strides == nullptr || v_tree_strides == nullptr || mask_strides == nullptr ||
      o_strides == nullptr)
    return tk::fail("tree decode: null pointer");
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || max_len <= 0 || nodes <= 0)
    return tk::fail("tree decode: empty problem");
  if (q_heads % kv_heads != 0) return tk::fail("tree decode: q_heads must be a multiple of kv_heads");
  const int64_t group = q_heads / kv_heads, rows = nodes * group;
  if (const char* why = unsupported(batch, kv_heads, group, max_len, nodes, head_dim))
    return tk::fail("tree decode: %s", why);
  const Plan plan = make_plan(batch, kv_heads, rows, max_len, nodes, head_dim);
  if (plan.combine && workspace == nullptr) return tk::fail("tree decode: null pointer");
  for (const void* p : {q, k_cache, v_cache, k_tree, v_tree, static_cast<const void*>(o),
                        static_cast<const void*>(workspace)})
    if (!tk::aligned16(p)) return tk::fail("tree decode: tensors must be 16-byte aligned");
  for (const int64_t* st : {q_strides, k_strides, v_strides, k_tree_strides, v_tree_strides,
                            o_strides})
    for (int d = 0; d < 3; ++d)
      if (st[d] < 0 || st[d] % 8 != 0 || st[d] >= (int64_t(1) << 40))
        return tk::fail("tree decode: strides must be non-negative multiples of 8 elements");
  if (mask_strides[0] < 0 || mask_strides[1] < 0 || mask_strides[0] >= (int64_t(1) << 40) ||
      mask_strides[1] >= (int64_t(1) << 30))
    return tk::fail("tree decode: mask strides must be non-negative and keep rows in range");
  // The DMA addresses a tile's 32 rows through 32-bit buffer offsets.
  for (const int64_t* st : {k_strides, v_strides, k_tree_strides, v_tree_strides})
    if (st[2] >= (int64_t(1) << 24))
      return tk::fail("tree decode: key strides must be below 2^24 elements");
  TreeArgs a;
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.k_tree = k_tree;
  a.v_tree = v_tree;
  a.mask = static_cast<const uint8_t*>(mask);
  a.seqlens = seqlens;
  a.o = o;
  a.lse = lse;
  a.part_o = workspace;
  a.part_ml = reinterpret_cast<float2*>(workspace + plan.flat * kv_heads * rows * head_dim);
  a.qb = q_strides[0], a.qh = q_strides[1], a.qt = q_strides[2];
  a.ob = o_strides[0], a.oh = o_strides[1], a.ot = o_strides[2];
  a.kb = k_strides[0], a.kh = k_strides[1], a.kl = k_strides[2];
  a.vb = v_strides[0], a.vh = v_strides[1], a.vl = v_strides[2];
  a.ktb = k_tree_strides[0], a.kth = k_tree_strides[1], a.ktl = k_tree_strides[2];
  a.vtb = v_tree_strides[0], a.vth = v_tree_strides[1], a.vtl = v_tree_strides[2];
  a.mb = mask_strides[0], a.mt = mask_strides[1];
  a.batch = static_cast<int>(batch);
  a.q_heads = static_cast<int>(q_heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(group);
  a.nodes = static_cast<int>(nodes);
  a.rows = static_cast<int>(rows);
  a.max_len = static_cast<int>(max_len);
  a.tree_tiles = static_cast<int>(tk::cdiv(nodes, kTileKeys));
  a.whole = static_cast<int>(plan.whole);
  a.heads_blocks = static_cast<int>(kv_heads * plan.row_blocks);
  a.many = static_cast<int>(tk::cdiv(16 * 128, kv_heads * plan.row_blocks));
  a.runs = static_cast<int>(plan.runs);
  a.row_blocks = static_cast<int>(plan.row_blocks);
  a.by_group = tk::FastDiv(static_cast<uint32_t>(group));
  a.by_kv_heads = tk::FastDiv(static_cast<uint32_t>(kv_heads));
  a.by_row_blocks = tk::FastDiv(static_cast<uint32_t>(plan.row_blocks));
  a.flat = static_cast<int>(plan.flat);
  // Not 0, which would turn a masked score (-inf) into NaN: the least subnormal float (which the
  // kernel's multiplications keep) leaves no score at or above 2^-149 * 2^128 = 2^-21, as good as 0
  // to the hardware exponential. Scales this small are off by 2^-150, scores then by 2^-22.
  a.scale_log2 = fmaxf(fabsf(scale) * kLog2e, 0x1p-149f);
  a.flip = scale < 0.f ? int(0x80008000u) : 0;
  hipStream_t s = tk::as_stream(stream);
  if (dtype == TK_DTYPE_BF16) {
    if (head_dim == 128)
      launch<__bf16, 128>(a, plan.combine, s);
    else
      launch<__bf16, 64>(a, plan.combine, s);
  } else {
    if (head_dim == 128)
      launch<_Float16, 128>(a, plan.combine, s);
    else
      launch<_Float16, 64>(a, plan.combine, s);
  }
  return tk::check_launch("tree decode");
}
