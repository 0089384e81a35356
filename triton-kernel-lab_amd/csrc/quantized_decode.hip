// Grouped-query attention decode over a cache held in 8 bits (quantized_cache.hip): one query token
// per sequence, G = q_heads / kv_heads query heads to a KV head, lengths per sequence.
//   s_j = (q . kc_j) ks_j scale log2(e),  p_j = exp2(s_j - m),  o = sum_j p_j vs_j vc_j / sum_j p_j.
// A key's scale multiplies its score and a value's its weight, so codes are only widened (exact in
// both 16-bit types) and no row is ever multiplied out.
//
// Split kernel: one wave per (run of 32-key tiles, KV head, block of 16 MT heads; groups above 32 heads read
// the cache once for every 32), both products on v_mfma_f32_16x16x32 as in the 16-bit decode:
//   S^T (16 keys x 16 heads) = K . Q^T in q's type. A lane's 16 bytes of a key are features 64 c + 16 quad .. +15:
//     two operands, with Q^T's features in the same order.
//   O^T (16 dims x 16 heads) += V^T . P^T in bfloat16. P^T comes from the score registers, V^T from
//     ds_read_b64_tr_b8 (in each 16-lane group, lanes 2 j and 2 j + 1 read 16 bytes of row j, lane i
//     receives column i of rows 0 .. 7): rows 4 quad .. +3 and 16 + 4 quad .. +3, the keys whose
//     scores the lane holds.
// K, V and the scales reach LDS by non-temporal buffer->LDS DMA into a ring of tiles.
//
// Weights. The running maximum m moves only when a tile's exceeds it by more than 8, so p <= 2^8.
// p vs, divided by a running power of two above every |vs| met so far so that no scale overflows, is
// rounded to bfloat16 for the second product, and what that left to bfloat16 once more as a product of
// its own: together off by at most 2^-16 of the weight, however small the weight is and whatever the other
// keys' scales are. float16 cannot hold them: what falls below 2^-24 of the unit is nothing there (runs of
// 1000 keys, one of them without a value and 14 nats above the rest, one with a value 32 times the others'
// and no weight: results off by 20 to 44 %, now by 2.3e-4). HBM leaves the matrix units the time for the
// second product: 89.1 -> 89.7 us at B32 L16384 ragged, and bfloat16 results are off by 1.65e-3 of their
// size, as float32 arithmetic's are, instead of 2.4e-3; float16's by 2.1e-4, as those. Widening int8 codes
// to bfloat16 costs float16 queries at D64 4 % (B32 L16384 110 -> 114 us), the others nothing. Sums are
// float32.
//
// What bounds it (D128 Hkv8, both kernels): HBM. B32 Hq32 e4m3, ragged up to 16384 (508 MB) 90 us, 5.6 TB/s,
// the last runs to end among it; of 8192 equal keys (554 MB) 95 us, 5.8; B2 Hq64 L131072 int8 (554 MB)
// 90 us, 6.2. B1 L2000: 5.8 + 3.7 us, latencies one after the other.
// Measured and not kept: ordinary loads in place of non-temporal ones (15 % more), a ring of 3 or 6 stages,
// two rounds of workgroups, runs that may span sequences (ragged 95.5 -> 92.4 us, but equal 95 -> 101 and
// B8 Hkv1 15.9 -> 20.2), a search of the least run length that fits (ragged 96 -> 93, equal 95.6 -> 102).
#include "attention_dma.hpp"
#include "decode_runs.hpp"
#include "eight_bit.hpp"
#include "tk_common.hpp"

namespace {

using namespace tk_runs;
using tk_attn::f32x4;
using tk_attn::i32x2;
using tk_attn::i32x4;

constexpr int kNonTemporal = 2;

struct DecodeArgs {
  Schedule schedule;
  const void* q;
  const uint8_t *k, *v;
  const float* scales;
  void* o;
  float* lse;
  float* part_o;   // [slot][head of the group][D], slot = (flat run, KV head)
  float2* part_ml; // [slot][head of the group]: reference maximum, sum
  int64_t qb, qh, ob, oh, kb, kh, kl, vb, vh, vl, sb, sh, sl;
  tk::FastDiv by_group, by_kv_heads, by_row_blocks;
  int q_heads, kv_heads, group, row_blocks, flat;
  float scale_log2;
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two codes (bytes 2 kHalf and 2 kHalf + 1 of c) as T: exact.
template <typename T, int kType, bool kHalf>
__device__ __forceinline__ int widen2(int c) {
  if constexpr (kType == tk8::kE4M3) {
    if constexpr (__is_same(T, __bf16))
      return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, kHalf));
    else
      return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, kHalf));
  } else if constexpr (__is_same(T, __bf16)) {
    // float32 of at most 8 significant bits: its upper half is the bfloat16.
    const float a = float(int8_t(uint32_t(c) >> (kHalf ? 16 : 0)));
    const float b = float(int8_t(uint32_t(c) >> (kHalf ? 24 : 8)));
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  } else {
    // 0x6400 + u is 1024 + u in float16, u = c + 128.
    const uint32_t u = uint32_t(c) ^ 0x80808080u;
    const uint32_t h = __builtin_amdgcn_perm(0x64646464u, u, kHalf ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(int, __builtin_bit_cast(f16x2, h) - f16x2{1152, 1152});
  }
}

// Eight codes as an MFMA operand.
template <typename T, int kType>
__device__ __forceinline__ i32x4 widen8(int lo, int hi) {
  return i32x4{widen2<T, kType, false>(lo), widen2<T, kType, true>(lo),
               widen2<T, kType, false>(hi), widen2<T, kType, true>(hi)};
}

// The low or high bfloat16 of a register as float32.
__device__ __forceinline__ float half_of(int x, int high) {
  return __uint_as_float(high ? uint32_t(x) & 0xFFFF0000u : uint32_t(x) << 16);
}

template <int OFF>
__device__ __forceinline__ i32x2 lds_read_tr8(uint32_t addr) {
  i32x2 r;
  asm volatile("ds_read_b64_tr_b8 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(OFF));
  return r;
}

// LDS ring: NS stages of a 32-key tile of K, the same keys of V, and their scales. Rows are stored
// whole with their 16-byte chunks swizzled (the DMA writes contiguous LDS).
template <int D>
struct Ring8 {
  static constexpr int RB = D;                 // bytes per row
  static constexpr int TILE = kTileKeys * RB;  // bytes per tensor tile
  static constexpr int SCALES = 2 * TILE;      // offset of the scales
  static constexpr int STAGE = 2 * TILE + kTileKeys * 8;
  static constexpr int NS = D == 128 ? 4 : 8;  // about 34 KiB: four waves share a CU
  static constexpr int IPT = TILE / 1024;      // DMA instructions per tensor tile
  static constexpr int PER = 2 * IPT + 1;      // and per stage
  static constexpr int RPI = 1024 / RB;        // rows per DMA instruction
  static constexpr int CPR = RB / 16;          // chunks per row
  static_assert((NS - 1) * PER < 64, "ring deeper than the vmcnt counter");
  // K: chunk c of row r at c ^ kswz(r); a ds_read_b128 phase (16 lanes, one chunk of 16 rows) touches
  // 16 distinct bank groups. V: at c ^ vswz(r); a transposing read's phase (32 lanes) takes one chunk
  // of rows 8 x .. 8 x + 7 and 16 more, on distinct positions.
  static __device__ __forceinline__ int kswz(int r) { return D == 128 ? (r >> 1) & 7 : (r >> 2) & 3; }
  static __device__ __forceinline__ int vswz(int r) {
    return D == 128 ? ((r >> 1) & 3) | ((r >> 4) & 1) << 2 : ((r >> 2) & 1) | ((r >> 4) & 1) << 1;
  }
};

// The stream of a run's tiles into the ring. All fields but the lane offsets are wave-uniform.
template <int D>
struct Fetcher {
  using R = Ring8<D>;
  const uint8_t *k, *v;  // first row of the next tile
  const char* scales;
  uint32_t k_row, v_row, s_row;  // bytes per row
  int left;                      // rows from there to the end of the run
  char* ring;
  uint32_t koff[R::IPT], voff[R::IPT], soff;

  // Instruction i covers rows RPI i .. +RPI-1; the lane fetches the chunk that belongs at its LDS
  // slot, and one float of the 32 pairs of scales.
  __device__ __forceinline__ void offsets(int lane) {
#pragma unroll
    for (int i = 0; i < R::IPT; ++i) {
      const int r = i * R::RPI + lane / R::CPR;
      const int slot = lane % R::CPR;
      koff[i] = r * k_row + (slot ^ R::kswz(r)) * 16;
      voff[i] = r * v_row + (slot ^ R::vswz(r)) * 16;
    }
    soff = (lane >> 1) * s_row + (lane & 1) * 4;
  }

  // The next tile into `stage`. Tiles past the run's end (issued to keep the wait counts static)
  // read nothing and give zeros.
  __device__ __forceinline__ void next(int stage) {
    const int rows = min(max(left, 0), kTileKeys);
    const __amdgpu_buffer_rsrc_t rk = rows_buffer(k, rows, k_row, D);
    const __amdgpu_buffer_rsrc_t rv = rows_buffer(v, rows, v_row, D);
    const __amdgpu_buffer_rsrc_t rs = rows_buffer(scales, rows, s_row, 8);
    char* to = ring + stage * R::STAGE;
#pragma unroll
    for (int i = 0; i < R::IPT; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (tk_attn::lds_void*)(to + i * 1024), 16, koff[i],
                                               0, 0, kNonTemporal);
#pragma unroll
    for (int i = 0; i < R::IPT; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (tk_attn::lds_void*)(to + R::TILE + i * 1024),
                                               16, voff[i], 0, 0, kNonTemporal);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (tk_attn::lds_void*)(to + R::SCALES), 4, soff, 0,
                                             0, kNonTemporal);
    k += int64_t(kTileKeys) * k_row;
    v += int64_t(kTileKeys) * v_row;
    scales += int64_t(kTileKeys) * s_row;
    left -= kTileKeys;
  }
};

template <typename T, int kType, int D, int MT>
__global__ __launch_bounds__(64, 1) void quantized_split_kernel(DecodeArgs a) {
  using R = Ring8<D>;
  constexpr int DC = D / 64;  // 16-byte chunks of a key per lane, two products each
  constexpr int OC = D / 16;  // 16-dim output chunks
  constexpr int NS = R::NS, RB = R::RB;
  __shared__ __attribute__((aligned(1024))) char ring[NS * R::STAGE];

  const int lane = threadIdx.x;
  const int pair = a.by_row_blocks.div(blockIdx.x);
  const int rb = blockIdx.x - pair * a.row_blocks;
  const int f = a.by_kv_heads.div(pair);
  const int kvh = pair - f * a.kv_heads;
  const Lengths lengths = read_lengths(a.schedule, lane);
  Run run;
  if (!find_run(a.schedule, lengths, f, lane, run)) return;
  const int b = run.b;
  const int t0 = run.split * lengths.chunk;
  const int t1 = run.splits == 1 ? tiles_of(run.length)
                                 : min(t0 + lengths.chunk, tiles_of(run.length));
  const int limit = min(run.length, t1 * kTileKeys);  // keys from t0 * 32 up to it

  const int row16 = lane & 15;
  const int quad = lane >> 4;
  const int r0 = rb * 16 * MT;

  Fetcher<D> fetch;
  {
    const int64_t first = int64_t(t0) * kTileKeys;
    fetch.k = a.k + b * a.kb + kvh * a.kh + first * a.kl;
    fetch.v = a.v + b * a.vb + kvh * a.vh + first * a.vl;
    fetch.scales = reinterpret_cast<const char*>(a.scales + b * a.sb + kvh * a.sh + first * a.sl);
    fetch.k_row = uint32_t(a.kl);
    fetch.v_row = uint32_t(a.vl);
    fetch.s_row = uint32_t(a.sl * 4);
    fetch.left = limit - t0 * kTileKeys;
    fetch.ring = ring;
    fetch.offsets(lane);
  }

  // Q^T operands: head r0 + 16 m + row16 (zero past the group), dims 64 c + 16 quad + 8 e .. +7.
  i32x4 qf[MT][DC][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = r0 + 16 * m + row16;
    const T* p = static_cast<const T*>(a.q) + b * a.qb + (kvh * a.group + r) * a.qh + 16 * quad;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        qf[m][c][e] = r < a.group ? *reinterpret_cast<const i32x4*>(p + 64 * c + 8 * e)
                                  : i32x4{0, 0, 0, 0};
  }
  // (The loads of Q are the oldest, so waiting for them leaves the tiles in flight.)
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) fetch.next(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      tk_attn::pin(qf[m][c][0]);
      tk_attn::pin(qf[m][c][1]);
    }

  const uint32_t ring_base = (uint32_t)(uintptr_t)(tk_attn::lds_void*)ring;
  uint32_t ka[DC], va[OC];
#pragma unroll
  for (int c = 0; c < DC; ++c) ka[c] = row16 * RB + (((4 * c + quad) ^ R::kswz(row16)) * 16);
  const int trow = 4 * quad + ((row16 >> 1) & 3) + 16 * (row16 >> 3);
#pragma unroll
  for (int c = 0; c < OC; ++c)
    va[c] = R::TILE + trow * RB + ((c ^ R::vswz(trow)) * 16) + 8 * (row16 & 1);
  const uint32_t sa = R::SCALES + quad * 32;

  f32x4 o[MT][OC];
  float top[MT], sum[MT];  // reference maximum of head row16, this lane's share of its sum
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    top[m] = kNoMax;
    sum[m] = 0.f;
#pragma unroll
    for (int c = 0; c < OC; ++c) o[m][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // o holds sums in units of 2^unit, above every |vs| so far.
  int unit = -125;
  float above = 0x1p-125f, inverse = 0x1p125f;

  int stage = 0;
  for (int t = t0; t < t1; ++t) {
    // The tile has landed once only the NS - 2 younger ones' loads are outstanding; the stage read
    // in the last iteration (its reads have returned) takes the next.
    tk_attn::wait_vmcnt<(NS - 2) * R::PER>();
    fetch.next(stage == 0 ? NS - 1 : stage - 1);
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t sb = ring_base + stage * R::STAGE;
    stage = stage == NS - 1 ? 0 : stage + 1;

    i32x4 kc[DC][2], sc[2][2];
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      kc[c][0] = tk_attn::lds_read_b128<0>(sb + ka[c]);
      kc[c][1] = tk_attn::lds_read_b128<16 * RB>(sb + ka[c]);
    }
    sc[0][0] = tk_attn::lds_read_b128<0>(sb + sa);
    sc[0][1] = tk_attn::lds_read_b128<16>(sb + sa);
    sc[1][0] = tk_attn::lds_read_b128<128>(sb + sa);
    sc[1][1] = tk_attn::lds_read_b128<144>(sb + sa);
    tk_attn::wait_lgkm<0>();
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      tk_attn::pin(kc[c][0]);
      tk_attn::pin(kc[c][1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      tk_attn::pin(sc[i][0]);
      tk_attn::pin(sc[i][1]);
    }
    // s[m][i][r]: product of head row16 and key 16 i + 4 quad + r.
    f32x4 s[MT][2];
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const i32x4 first = widen8<T, kType>(kc[c][i][0], kc[c][i][1]);
        const i32x4 second = widen8<T, kType>(kc[c][i][2], kc[c][i][3]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          s[m][i] = tk_attn::Mma16<T>::run(first, qf[m][c][0],
                                           c == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[m][i]);
          s[m][i] = tk_attn::Mma16<T>::run(second, qf[m][c][1], s[m][i]);
        }
      }
    // V^T, read while the softmax runs.
    i32x2 vc[OC];
#pragma unroll
    for (int c = 0; c < OC; ++c) vc[c] = lds_read_tr8<0>(sb + va[c]);
    // Key and value scales of keys 16 i + 4 quad + r.
    float ks[2][4], vs[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ks[i][r] = __int_as_float(sc[i][r / 2][2 * (r % 2)]) * a.scale_log2;
        vs[i][r] = __int_as_float(sc[i][r / 2][2 * (r % 2) + 1]);
      }
    const int live = limit - t * kTileKeys;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][i][r] *= ks[i][r];
    if (__builtin_expect(live < kTileKeys, 0)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * i + 4 * quad + r >= live) s[m][i][r] = -INFINITY;
    }
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(vs[i][r]));
    if (__ballot(most >= above) != 0) {
      const float all = fmaxf(tk_attn::max_over_column(most), 0x1p-126f);
      const int next = max(__builtin_amdgcn_frexp_expf(all), unit);
      const float down = __builtin_ldexpf(1.f, unit - next);
      unit = next;
      above = __builtin_ldexpf(1.f, unit);
      inverse = __builtin_ldexpf(1.f, -unit);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < OC; ++c) o[m][c] *= down;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) vs[i][r] *= inverse;
    // P = exp2(s - top): a lane whose exponentials sum to at most 2^8 has none above it, and then no
    // maximum is formed.
    i32x4 pf[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      f32x4 p[2];
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[i][r] = __builtin_amdgcn_exp2f(s[m][i][r] - top[m]);
          part += p[i][r];
        }
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(part <= 256.f)) != 0, 0)) {
        float high = s[m][0][0];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) high = fmaxf(high, s[m][i][r]);
        high = tk_attn::max_over_column(high);
        const float next = high > top[m] + 8.f ? high : top[m];
        const float alpha = __builtin_amdgcn_exp2f(top[m] - next);
        top[m] = next;
        sum[m] *= alpha;
#pragma unroll
        for (int c = 0; c < OC; ++c) o[m][c] *= alpha;
        part = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[i][r] = __builtin_amdgcn_exp2f(s[m][i][r] - next);
            part += p[i][r];
          }
      }
      sum[m] += part;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[i][r] *= vs[i][r];
      pf[m][0] = tk_attn::acc_frag2<__bf16>(p[0], p[1]);
      f32x4 rest[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) rest[i][r] = p[i][r] - half_of(pf[m][0][2 * i + r / 2], r % 2);
      pf[m][1] = tk_attn::acc_frag2<__bf16>(rest[0], rest[1]);
    }
    tk_attn::wait_lgkm<0>();
#pragma unroll
    for (int c = 0; c < OC; ++c) asm volatile("" : "+v"(vc[c]));
#pragma unroll
    for (int c = 0; c < OC; ++c) {
      const i32x4 vf = widen8<__bf16, kType>(vc[c][0], vc[c][1]);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[m][c] = tk_attn::Mma16<__bf16>::run(vf, pf[m][e], o[m][c]);
    }
  }
  // The tiles issued past the end still write (zeros) into the ring.
  tk_attn::wait_vmcnt<0>();

  const int slot = f * a.kv_heads + kvh;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const float l = tk_attn::sum_over_column(sum[m]);
    const int r = r0 + 16 * m + row16;
    if (r >= a.group) continue;
#pragma unroll
    for (int c = 0; c < OC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[m][c][i] = __builtin_ldexpf(o[m][c][i], unit);
    if (run.splits == 1) {
      const int h = kvh * a.group + r;
      T* dst = static_cast<T*>(a.o) + b * a.ob + h * a.oh + 4 * quad;
#pragma unroll
      for (int c = 0; c < OC; ++c) {
        float out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = l == 0.f ? 0.f : o[m][c][i] / l;
        tk::store_vec<T, 4>(dst + 16 * c, out);
      }
      if (quad == 0 && a.lse != nullptr)
        a.lse[int64_t(b) * a.q_heads + h] = l == 0.f ? -INFINITY : top[m] + log2f(l);
    } else {
      const int64_t at = int64_t(slot) * a.group + r;
#pragma unroll
      for (int c = 0; c < OC; ++c)
        *reinterpret_cast<f32x4*>(a.part_o + at * D + 16 * c + 4 * quad) = o[m][c];
      if (quad == 0) a.part_ml[at] = float2{top[m], l};
    }
  }
}

template <typename T, int D, int WAVES>
__global__ __launch_bounds__(64 * kJoinWaves) void quantized_combine_kernel(DecodeArgs a) {
  __shared__ JoinScratch<D> shared;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = WAVES == 1 ? blockIdx.x * kJoinWaves + wave : blockIdx.x;
  const int b = blockIdx.y;
  const Lengths lengths = read_lengths(a.schedule, lane);
  Run run;
  sequence_runs(a.schedule, lengths, b, lane, run);
  if (run.splits == 1 || h >= a.q_heads) return;  // (one run: written by the split kernel)
  const int kvh = a.by_group.div(h);
  const int64_t step = int64_t(a.kv_heads) * a.group;  // between a head's splits
  const int64_t at0 = (int64_t(run.flat0) * a.kv_heads + kvh) * a.group + (h - kvh * a.group);
  join_parts<T, D, WAVES>(a.part_o, a.part_ml, run.splits, [&](int i) { return at0 + i * step; },
                          static_cast<T*>(a.o) + b * a.ob + h * a.oh,
                          a.lse == nullptr ? nullptr : a.lse + int64_t(b) * a.q_heads + h, wave, shared);
}

constexpr int kResident = 1024;  // workgroups that run at once: four per CU
constexpr int kWhole = 4;         // tiles of a sequence that is not split

// Instantiated here by name: left to the launches below, the host compiler leaves some of these
// kernels' launch stubs undefined.
#define TK_SPLIT(T, K, D, MT) template __global__ void quantized_split_kernel<T, K, D, MT>(DecodeArgs)
#define TK_SPLITS(T, K) \
  TK_SPLIT(T, K, 128, 1); TK_SPLIT(T, K, 128, 2); TK_SPLIT(T, K, 64, 1); TK_SPLIT(T, K, 64, 2)
TK_SPLITS(__bf16, tk8::kE4M3);
TK_SPLITS(__bf16, tk8::kInt8);
TK_SPLITS(_Float16, tk8::kE4M3);
TK_SPLITS(_Float16, tk8::kInt8);

template <typename T, int kType, int D>
void launch(const DecodeArgs& a, bool combine, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(int64_t(a.flat) * a.kv_heads * a.row_blocks));
  if (a.group <= 16)
    hipLaunchKernelGGL((quantized_split_kernel<T, kType, D, 1>), grid, dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL((quantized_split_kernel<T, kType, D, 2>), grid, dim3(64), 0, s, a);
  if (!combine) return;
  if (int64_t(a.q_heads) * a.schedule.batch <= kFewRows)
    hipLaunchKernelGGL((quantized_combine_kernel<T, D, kJoinWaves>), dim3(a.q_heads, a.schedule.batch),
                       dim3(64 * kJoinWaves), 0, s, a);
  else
    hipLaunchKernelGGL((quantized_combine_kernel<T, D, 1>),
                       dim3(static_cast<uint32_t>(tk::cdiv(a.q_heads, kJoinWaves)), a.schedule.batch),
                       dim3(64 * kJoinWaves), 0, s, a);
}

// How the call is cut: runs (the tiles of all sequences over `runs` give the run length), the bound
// on their number, blocks of heads. The sequences' last runs are shorter, so `runs` leaves room for
// one more per sequence where that keeps the launch to one round of workgroups.
struct Plan {
  int64_t row_blocks, runs, fewer, flat, whole;
  bool combine;
};
Plan make_plan(int64_t batch, int64_t kv_heads, int64_t group, int64_t max_len) {
  Plan p;
  p.row_blocks = group <= 16 ? 1 : tk::cdiv(group, 32);
  const int64_t most = tk::cdiv(max_len, kTileKeys);
  const int64_t base = kResident / (kv_heads * p.row_blocks);
  p.runs = base > 2 * batch ? base - batch + 1 : base > 1 ? base : 1;
  p.fewer = base > 1 ? tk::cdiv(base, 2) : 1;
  p.whole = kWhole;
  p.combine = most > p.whole;
  p.flat = p.runs + batch;
  const int64_t bound = p.combine ? batch * tk::cdiv(most, kMinRun) : batch;
  if (p.flat > bound) p.flat = bound;
  return p;
}

// Why a problem of these (positive) sizes is not taken, or null. The grid holds at most 2^22
// workgroups, and tiles and partial results are counted in 32 bits.
const char* unsupported(int64_t batch, int64_t kv_heads, int64_t group, int64_t max_len,
                        int64_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
  if (batch > 65535 || kv_heads > 65535 || group > 65535 || kv_heads * group > 65535 ||
      max_len > (1 << 30))
    return "problem too large";
  const Plan p = make_plan(batch, kv_heads, group, max_len);
  if (batch * tk::cdiv(max_len, kTileKeys) > INT32_MAX / 2 ||
      p.flat * kv_heads * p.row_blocks > (1 << 22))
    return "problem too large";
  return nullptr;
}

}  // namespace

extern "C" int tk_quantized_decode_slots(int64_t batch, int64_t kv_heads, int64_t group,
                                         int64_t max_len, int64_t head_dim) {
  if (batch <= 0 || kv_heads <= 0 || group <= 0 || max_len <= 0) return -1;
  if (unsupported(batch, kv_heads, group, max_len, head_dim) != nullptr) return -1;
  const Plan p = make_plan(batch, kv_heads, group, max_len);
  return p.combine ? static_cast<int>(p.flat * kv_heads) : 0;
}

extern "C" int tk_quantized_decode(int dtype, const void* q, const void* k_cache,
                                   const void* v_cache, const float* scales,
                                   const int32_t* seqlens, void* o, float* lse, float* workspace,
                                   int64_t batch, int64_t q_heads, int64_t kv_heads,
                                   int64_t max_len, int64_t head_dim, const int64_t* q_strides,
                                   const int64_t* k_strides, const int64_t* v_strides,
                                   const int64_t* scale_strides, const int64_t* o_strides,
                                   float scale, int cache_type, void* stream) {
  if (dtype != TK_DTYPE_F16 && dtype != TK_DTYPE_BF16)
    return tk::fail("quantized decode: dtype must be float16 or bfloat16");
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || scales == nullptr ||
      o == nullptr || q_strides == nullptr || k_strides == nullptr || v_strides == nullptr ||
      scale_strides == nullptr || o_strides == nullptr)
    return tk::fail("quantized decode: null pointer");
  if (cache_type != tk8::kE4M3 && cache_type != tk8::kInt8)
    return tk::fail("quantized decode: unsupported cache type %d", cache_type);
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || max_len <= 0)
    return tk::fail("quantized decode: empty problem");
  if (q_heads % kv_heads != 0)
    return tk::fail("quantized decode: q_heads must be a multiple of kv_heads");
  const int64_t group = q_heads / kv_heads;
  if (const char* why = unsupported(batch, kv_heads, group, max_len, head_dim))
    return tk::fail("quantized decode: %s", why);
  const Plan plan = make_plan(batch, kv_heads, group, max_len);
  if (plan.combine && workspace == nullptr) return tk::fail("quantized decode: null pointer");
  for (const void* p : {q, k_cache, v_cache, static_cast<const void*>(o),
                        static_cast<const void*>(workspace)})
    if (!tk::aligned16(p)) return tk::fail("quantized decode: tensors must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(scales) % 4 != 0)
    return tk::fail("quantized decode: scales must be 4-byte aligned");
  for (const int64_t* st : {q_strides, o_strides})
    for (int d = 0; d < 2; ++d)
      if (st[d] < 0 || st[d] % 8 != 0 || st[d] >= (int64_t(1) << 40))
        return tk::fail("quantized decode: strides must be non-negative multiples of 8 elements");
  for (const int64_t* st : {k_strides, v_strides})
    for (int d = 0; d < 3; ++d)
      if (st[d] < 0 || st[d] % 16 != 0 || st[d] >= (int64_t(1) << 40))
        return tk::fail("quantized decode: cache strides must be non-negative multiples of 16");
  for (int d = 0; d < 3; ++d)
    if (scale_strides[d] < 0 || scale_strides[d] >= (int64_t(1) << 40))
      return tk::fail("quantized decode: scale strides must be non-negative and in range");
  // The DMA addresses a tile's 32 rows through 32-bit buffer offsets.
  for (const int64_t* st : {k_strides, v_strides, scale_strides})
    if (st[2] >= (int64_t(1) << 24))
      return tk::fail("quantized decode: key strides must be below 2^24 elements");
  DecodeArgs a;
  a.schedule.seqlens = seqlens;
  a.schedule.batch = static_cast<int>(batch);
  a.schedule.max_len = static_cast<int>(max_len);
  a.schedule.runs = static_cast<int>(plan.runs);
  a.schedule.fewer = static_cast<int>(plan.fewer);
  a.schedule.whole = static_cast<int>(plan.whole);
  a.q = q;
  a.k = static_cast<const uint8_t*>(k_cache);
  a.v = static_cast<const uint8_t*>(v_cache);
  a.scales = scales;
  a.o = o;
  a.lse = lse;
  a.part_o = workspace;
  a.part_ml = reinterpret_cast<float2*>(workspace + plan.flat * kv_heads * group * head_dim);
  a.qb = q_strides[0], a.qh = q_strides[1];
  a.ob = o_strides[0], a.oh = o_strides[1];
  a.kb = k_strides[0], a.kh = k_strides[1], a.kl = k_strides[2];
  a.vb = v_strides[0], a.vh = v_strides[1], a.vl = v_strides[2];
  a.sb = scale_strides[0], a.sh = scale_strides[1], a.sl = scale_strides[2];
  a.by_group = tk::FastDiv(static_cast<uint32_t>(group));
  a.by_kv_heads = tk::FastDiv(static_cast<uint32_t>(kv_heads));
  a.by_row_blocks = tk::FastDiv(static_cast<uint32_t>(plan.row_blocks));
  a.q_heads = static_cast<int>(q_heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(group);
  a.row_blocks = static_cast<int>(plan.row_blocks);
  a.flat = static_cast<int>(plan.flat);
  a.scale_log2 = scale * kLog2e;
  hipStream_t s = tk::as_stream(stream);
  const bool e4m3 = cache_type == tk8::kE4M3;
#define TK_LAUNCH(T, D)                                                         \
  do {                                                                          \
    if (e4m3)                                                                   \
      launch<T, tk8::kE4M3, D>(a, plan.combine, s);                             \
    else                                                                        \
      launch<T, tk8::kInt8, D>(a, plan.combine, s);                             \
  } while (0)
  if (dtype == TK_DTYPE_BF16) {
    if (head_dim == 128)
      TK_LAUNCH(__bf16, 128);
    else
      TK_LAUNCH(__bf16, 64);
  } else {
    if (head_dim == 128)
      TK_LAUNCH(_Float16, 128);
    else
      TK_LAUNCH(_Float16, 64);
  }
#undef TK_LAUNCH
  return tk::check_launch("quantized decode");
}
