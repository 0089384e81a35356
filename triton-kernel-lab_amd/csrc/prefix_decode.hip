// Grouped-query attention decode for a batch behind a shared prefix: sequence b's one query token sees
// the prefix_len keys that the whole batch shares and the first clamp(seqlens[b], 0, max_len) keys of
// its own cache; G = q_heads / kv_heads query heads read a KV head.
//
// The prefix is attended once for all: the batch * G query rows of a KV head (row r = sequence r / G,
// head r % G) form one matrix against its keys, so a key is read once for up to 64 or 128 rows instead
// of once per sequence. Both parts are cut into runs of 32-key tiles, whose partial results (float32
// sums, reference maximum and sum of the weights) a second kernel joins per row in a fixed order.
//
// Both products run on v_mfma_f32_16x16x32 with the keys as the first operand's rows, as in the other
// decode kernels:
//   S^T (16 keys x 16 rows) = K . Q^T, Q^T in registers; a row's maximum and sum are over a lane's
//     values and lanes ^ 16, ^ 32.
//   O^T (16 dims x 16 rows) += V^T . P^T, P^T from the score registers, V^T by transposing LDS reads.
// K and V reach LDS by non-temporal buffer->LDS DMA. Rows past a run's end lie outside the buffer range
// and arrive as zeros.
//
// One launch does both parts. A workgroup of W waves is either of the prefix (the waves share a ring of
// tiles, each has 16 MT rows of its own) or of the sequences' own caches (each of up to two waves has a
// run and a part of the ring to itself, and the G rows of its sequence): the first kind is bound by
// issuing its instructions once there are many rows, the second by HBM, and side by side they share a CU.
// The work is dealt on the device from the lengths: a share is the work of all tiles over the workgroups
// that run at once, with a prefix tile priced against an own one; the prefix's runs are a share long and
// come first, own ones half a share, so that none that starts late ends late.
//
// Softmax statistics and sums are float32, P is rounded to the storage dtype for the second product, as
// in every attention of this library: bfloat16 results are 2.3e-3 from float64's instead of 1.7e-3, float16
// ones 2.9e-4 instead of 2.1e-4. (What the rounding leaves as a second product would have to be in both
// parts and in every shape, or a sequence's accuracy would depend on its batch: 11.0 -> 11.5 us for a few
// sequences, 41.7 -> 43.3 at 16, and 16 matrix instructions more beside a tile's 32 in the prefix part of
// many rows, which issue bounds.) O is rounded once at the end.
//
// Rows past a workgroup's 128 make further row blocks, which read the same keys at about the same time:
// they run on one XCD, and the prefix's loads are then ordinary ones, so that its L2 keeps a tile for all
// of them (with non-temporal loads 845 MB came from HBM where 668 do: 149 -> 133 us; where one row block
// reads the prefix, non-temporal ones are faster: 24.3 us against 26.0).
//
// What bounds it (bf16 D128 Hq32 Hkv8, both kernels): B128, prefix 32768, own lengths up to 2048 (668 MB,
// 71 GFLOP) 133 us: every CU has one workgroup of each kind, a prefix tile takes 0.92 us beside own runs
// (0.78 with the CU to itself: about 200 instructions of one wave a SIMD, 32 of them matrix ones) and HBM
// delivers 5.3 TB/s. The same with own lengths of 2048 195 us, 6.2 TB/s; own caches alone (1.07 GB) 177 us,
// 6.1 TB/s; the prefix alone 85 us, 0.8 PFLOP/s. B4 behind 2048 keys: 6.5 + 4.3 us, latencies.
// Measured and not kept (against the 149 us): tile after tile without overlap 172 us (the prefix alone
// 101); four own waves of one stage each instead of two of two: 163 us, and own caches alone 187; a fifth
// ring stage, scheduling groups that alternate matrix and vector instructions (149 to 152 us both); the
// exponentials of both row tiles behind one test of the maximum, which leaves no registers (180 us).
// Against the 133 us: 32 rows of a wave on 32x32x16 products, half the matrix instructions at a lower clock
// (133.7; equal lengths 191 for 195, but the prefix alone 90 for 86 and 256 sequences behind 16384 keys
// 145 for 138); DMA and reads of keys issued among the output products, a higher priority for the prefix's
// waves (no difference) or for the others (152).
#include "attention_dma.hpp"
#include "decode_runs.hpp"
#include "tk_common.hpp"

namespace {

using namespace tk_runs;
using tk_attn::f32x4;
using tk_attn::i32x2;
using tk_attn::i32x4;

constexpr int kNonTemporal = 2;
constexpr int kLeastRun = 4;  // tiles of the shortest run of a part that is cut

struct PrefixArgs {
  const void *q, *kp, *vp, *k, *v;
  const int32_t* seqlens;
  void* o;
  float* lse;
  float* part_o;   // [slot][D]: prefix [run][KV head][row], then own [flat run][KV head][head of G]
  float2* part_ml; // [slot]
  int64_t qb, qh, ob, oh, kph, kpl, vph, vpl, kb, kh, kl, vb, vh, vl;
  tk::FastDiv by_group, by_kv_heads, by_row_blocks;
  int batch, q_heads, kv_heads, group, rows, max_len, prefix_len, prefix_tiles, row_blocks;
  int workgroups;           // that run at once
  int price;                // of a prefix tile for a workgroup, in 1/16 of an own tile for a wave
  int most_runs, most_own;  // bounds on the prefix's runs and the own flat runs
  float scale_log2;         // positive
  int flip;                 // Q's sign bits to turn (a negative scale)
};

__device__ __forceinline__ int own_length(const PrefixArgs& a, int b) {
  const int n = a.seqlens != nullptr ? a.seqlens[b] : a.max_len;
  return min(max(n, 0), a.max_len);
}
__device__ __forceinline__ int tiles_in(int length) { return (length + kTileKeys - 1) / kTileKeys; }

// How the work is cut, the same for every workgroup of the call.
struct Deal {
  int first;         // this lane's sequence's length (sequence = lane)
  int own_chunk;     // tiles of an own run
  int prefix_chunk;  // and of a prefix run
  int prefix_runs;
};

// Waves of a workgroup of W that take own runs. With four, each with a stage of the ring, so many loads
// are in flight that the prefix's waves wait for theirs: two stages each for two waves.
__host__ __device__ constexpr int own_waves(int waves) { return waves < 2 ? waves : 2; }

template <int W>
__device__ __forceinline__ Deal make_deal(const PrefixArgs& a, int lane) {
#pragma clang fp contract(off)  // both kernels have to come to the same numbers
  Deal d;
  d.first = lane < a.batch ? own_length(a, lane) : 0;
  int sum = tiles_in(d.first);
  for (int b = lane + 64; b < a.batch; b += 64) sum += tiles_in(own_length(a, b));
  const int own = __builtin_amdgcn_readlane(wave_prefix(sum), 63);
  const float prefix_work =
      float(a.prefix_tiles) * float(a.kv_heads * a.row_blocks) * float(a.price) * (1.f / 16);
  const float own_work = float(own) * float(a.kv_heads) * (1.f / own_waves(W));
  const float share = (prefix_work + own_work) / float(a.workgroups);
  // The bounds hold whatever the rounding above did.
  const int spare = max(a.most_own - a.batch, 1);
  const int own_share = __builtin_amdgcn_readfirstlane(int(share));
  const int prefix_share = __builtin_amdgcn_readfirstlane(int(share * 16 / float(a.price)));
  // Own runs are half a share, so that the last ones to start are not long ones.
  d.own_chunk = max(max(own_share / 2 + 1, kLeastRun), (own + spare - 1) / spare);
  const int chunk = max(prefix_share + 1, kLeastRun);
  const int runs = min((a.prefix_tiles + chunk - 1) / chunk, a.most_runs);
  d.prefix_chunk = (a.prefix_tiles + runs - 1) / runs;
  d.prefix_runs = (a.prefix_tiles + d.prefix_chunk - 1) / d.prefix_chunk;
  return d;
}

// Own flat run f: sequence, split and number of splits (wave-uniform); false past the last.
struct OwnRun {
  int b, length, split, splits, flat0;
};
__device__ __forceinline__ bool find_own(const PrefixArgs& a, const Deal& d, int f, int lane, OwnRun& out) {
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane;
    const int len = b0 == 0 ? d.first : (b < a.batch ? own_length(a, b) : 0);
    const int mine = (tiles_in(len) + d.own_chunk - 1) / d.own_chunk;
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

// A tensor's rows as a stream of 32-row tiles into LDS; PER DMA instructions of this wave per tile,
// from instruction `wave` * PER on. All fields but the lane offsets are wave-uniform. POLICY 0 is for rows
// that other workgroups read at about the same time.
template <int D, int PER, int POLICY = kNonTemporal>
struct Stream {
  using R = Ring<D>;
  const char* p;  // first row of the next tile
  uint32_t row;   // bytes per row
  int left;       // rows from there to the end of the run
  uint32_t off[PER];

  // Instruction i covers rows RPI (wave PER + i) .. +RPI-1; the lane fetches the chunk that belongs at
  // its LDS slot.
  template <bool kValues>
  __device__ __forceinline__ void start(const void* base, int64_t stride, int rows, int wave, int lane) {
    p = static_cast<const char*>(base);
    row = uint32_t(stride * 2);
    left = rows;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = (wave * PER + i) * R::RPI + lane / R::CPR;
      const int slot = lane % R::CPR;
      const int chunk = kValues ? ((((slot >> 1) ^ R::vswz(r)) << 1) | (slot & 1)) : slot ^ R::kswz(r);
      off[i] = r * row + chunk * 16;
    }
  }
  // The next tile to `to`, this wave's share of the tile in LDS. Past the end (issued to keep the wait
  // counts static) nothing is read and LDS gets zeros.
  __device__ __forceinline__ void next(char* to) {
    const __amdgpu_buffer_rsrc_t r = rows_buffer(p, min(max(left, 0), kTileKeys), row, D * 2);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (tk_attn::lds_void*)(to + i * 1024), 16, off[i], 0, 0,
                                               POLICY);
    p += int64_t(kTileKeys) * row;
    left -= kTileKeys;
  }
};

// 16 MT query rows against tiles of keys.
template <typename T, int D, int MT>
struct Rows {
  using R = Ring<D>;
  static constexpr int DC = D / 32, OC = D / 16, RB = R::RB;
  static constexpr int HB = 4;  // output chunks per batch of V reads
  i32x4 qf[MT][DC];
  f32x4 o[MT][OC];
  float top[MT], sum[MT];  // reference of row row16's exponentials, this lane's share of their sum
  uint32_t ka[DC], va[OC];

  __device__ __forceinline__ void start(int row16, int quad) {
#pragma unroll
    for (int c = 0; c < DC; ++c) ka[c] = row16 * RB + (((4 * c + quad) ^ R::kswz(row16)) * 16);
    const int trow = 4 * quad + (row16 >> 2);
#pragma unroll
    for (int c = 0; c < OC; ++c) va[c] = R::TILE + trow * RB + ((c ^ R::vswz(trow)) * 32) + 8 * (row16 & 3);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      top[m] = kNoMax;
      sum[m] = 0.f;
#pragma unroll
      for (int c = 0; c < OC; ++c) o[m][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // s[m][i][r]: product of row row16 of row tile m and key 16 i + 4 quad + r of the tile at LDS address
  // `at`. The reads of four 32-feature steps are in flight at a time; `read` runs behind the last one.
  template <typename F>
  __device__ __forceinline__ void scores(uint32_t at, f32x4 (&s)[MT][2], F&& read) {
    i32x4 kc[DC][2];
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      kc[c][0] = tk_attn::lds_read_b128<0>(at + ka[c]);
      kc[c][1] = tk_attn::lds_read_b128<16 * RB>(at + ka[c]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      const int younger = DC - 1 - c;
      if (younger >= 3)
        tk_attn::wait_lgkm<6>();
      else if (younger == 2)
        tk_attn::wait_lgkm<4>();
      else if (younger == 1)
        tk_attn::wait_lgkm<2>();
      else
        tk_attn::wait_lgkm<0>();
      tk_attn::pin(kc[c][0]);
      tk_attn::pin(kc[c][1]);
      if (c == DC - 1) read();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          s[m][i] = tk_attn::Mma16<T>::run(kc[c][i], qf[m][c], c == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[m][i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // The keys from `live` on are no keys.
  __device__ __forceinline__ void cut(int live, int quad, f32x4 (&s)[MT][2]) {
    if (__builtin_expect(live < kTileKeys, 0)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * i + 4 * quad + r >= live) s[m][i][r] = -INFINITY;
    }
  }

  // P = exp2(scale s - top) into pf. The reference moves only when the tile's maximum exceeds it by
  // more than kMost (base 2), and then to kLift below that, so p <= 2^kMost and o and sum are rescaled in
  // few tiles: a lane whose exponentials sum to at most 2^kMost has none above it, and then no maximum is
  // formed. In float16 P is kept near that type's upper end: below 2^-14 it is off by up to 2^-25, with the
  // lift 2^-32 of the run's largest (where valueless keys are 17 or 20 nats above the others, results were
  // off by 3.8 % and 88 % without it and are by 1.7e-4 and 6e-4, at no cost). bfloat16 has float32's range.
  static constexpr int kLift = __is_same(T, __bf16) ? 0 : 7, kMost = kLift + 8;
  __device__ __forceinline__ void weigh(const f32x4 (&s)[2], float scale, int m, f32x4 (&p)[2], float& part) const {
    part = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], scale, -top[m]));
        part += p[i][r];
      }
  }
  __device__ __forceinline__ void settle(const f32x4 (&s)[2], float scale, int m, f32x4 (&p)[2], float part,
                                         i32x4& pf) {
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(part <= float(1 << kMost))) != 0, 0)) {
      float high = s[0][0];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) high = fmaxf(high, s[i][r]);
      high = tk_attn::max_over_column(high) * scale;
      const float next = high > top[m] + kMost ? high - kLift : top[m];
      const float alpha = __builtin_amdgcn_exp2f(top[m] - next);
      top[m] = next;
      sum[m] *= alpha;
#pragma unroll
      for (int c = 0; c < OC; ++c) o[m][c] *= alpha;
      weigh(s, scale, m, p, part);
    }
    sum[m] += part;
    pf = tk_attn::acc_frag2<T>(p[0], p[1]);
  }
  __device__ __forceinline__ void softmax(const f32x4 (&s)[MT][2], float scale, i32x4 (&pf)[MT]) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      f32x4 p[2];
      float part;
      weigh(s[m], scale, m, p, part);
      settle(s[m], scale, m, p, part, pf[m]);
    }
  }

  // o += V^T P^T of the tile at `at`, whose first batch of V fragments has been requested; `read` runs
  // behind the last read.
  i32x2 lo[OC], hi[OC];
  __device__ __forceinline__ void request_v(uint32_t at, int c0) {
#pragma unroll
    for (int c = c0; c < c0 + HB && c < OC; ++c) {
      lo[c] = tk_attn::lds_read_tr16<0>(at + va[c]);
      hi[c] = tk_attn::lds_read_tr16<16 * RB>(at + va[c]);
    }
  }
  template <typename F>
  __device__ __forceinline__ void accumulate(uint32_t at, const i32x4 (&pf)[MT], F&& read) {
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
        request_v(at, c0 + HB);
      else
        read();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < HB; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m) o[m][c0 + c] = tk_attn::Mma16<T>::run(vf[c], pf[m], o[m][c0 + c]);
    }
  }

  // The tiles t0 .. t1-1 of a run with the matrix units kept busy: while a tile's exponentials are
  // formed, the next one's scores are; its output products follow with the reads of the keys after that.
  // Keys are read two tiles ahead of values, so each have a ring of their own, NS tiles at `ring` and
  // behind them; tile t is in stage (t - t0) % NS. One barrier in every step ends all waves' reads of
  // keys t + 1 and values t, whose stages then take keys t + 1 + NS and values t + NS, and shows keys t + 2
  // and values t + 1 to all of them, which were sent for NS - 1 steps before. Keys and values 0 .. NS-1
  // have been sent for, PER instructions each, in turns.
  template <int NS, int PER, typename FK, typename FV>
  __device__ __forceinline__ void pipeline(uint32_t ring, int t0, int t1, int limit, int quad, float scale,
                                           bool busy, FK&& fetch_k, FV&& fetch_v) {
    static_assert(NS >= 4, "a stage is refilled while it is read");
    auto arrive = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    auto after = [](int stage) { return stage == NS - 1 ? 0 : stage + 1; };
    i32x4 kc[DC][2];
    auto request_k = [&](int stage) {
      const uint32_t at = ring + stage * R::TILE;
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        kc[c][0] = tk_attn::lds_read_b128<0>(at + ka[c]);
        kc[c][1] = tk_attn::lds_read_b128<16 * RB>(at + ka[c]);
      }
    };
    auto pin_k = [&]() {
      tk_attn::wait_lgkm<0>();
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        tk_attn::pin(kc[c][0]);
        tk_attn::pin(kc[c][1]);
      }
    };
    auto multiply = [&](int c0, int c1, f32x4(&s)[MT][2]) {
#pragma unroll
      for (int c = c0; c < c1; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            s[m][i] = tk_attn::Mma16<T>::run(kc[c][i], qf[m][c], c == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[m][i]);
    };
    f32x4 even[MT][2], odd[MT][2];
    tk_attn::wait_vmcnt<(2 * NS - 1) * PER>();
    arrive();
    if (busy) {
      request_k(0);
      pin_k();
      multiply(0, DC, even);
    }
    tk_attn::wait_vmcnt<(2 * NS - 3) * PER>();
    arrive();
    fetch_k(0);
    int t = t0, stage = 0;
    auto turn = [&]() {  // a step's barrier, and what it lets be sent for
      tk_attn::wait_vmcnt<(2 * NS - 4) * PER>();
      arrive();
      fetch_k(after(stage));
      fetch_v(stage);
    };
    if (!busy) {
      for (; t < t1; ++t) {
        turn();
        stage = after(stage);
      }
      return;
    }
    request_k(1);
    auto step = [&](f32x4(&s)[MT][2], f32x4(&next)[MT][2]) {
      const uint32_t at = ring + (NS - 1 + stage) * R::TILE;  // va counts from a stage of both
      cut(limit - t * kTileKeys, quad, s);
      pin_k();
      f32x4 p[MT][2];
      float part[MT];
      i32x4 pf[MT];
      // Half of the next scores beside each row tile's exponentials, and half of the value reads.
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        __builtin_amdgcn_sched_barrier(0);
        if (m > 0) tk_attn::wait_lgkm<4>();  // lgkmcnt counts at most 15 outstanding reads
#pragma unroll
        for (int c = m * OC / MT; c < (m + 1) * OC / MT; ++c) {
          lo[c] = tk_attn::lds_read_tr16<0>(at + va[c]);
          hi[c] = tk_attn::lds_read_tr16<16 * RB>(at + va[c]);
        }
        multiply(m * DC / MT, (m + 1) * DC / MT, next);
        weigh(s[m], scale, m, p[m], part[m]);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < MT; ++m) settle(s[m], scale, m, p[m], part[m], pf[m]);
      turn();
#pragma unroll
      for (int c = 0; c < OC; ++c) asm volatile("" : "+v"(lo[c]), "+v"(hi[c]));
      stage = after(stage);
      request_k(after(stage));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < OC; ++c) {
        const i32x4 vf = {lo[c][0], lo[c][1], hi[c][0], hi[c][1]};
#pragma unroll
        for (int m = 0; m < MT; ++m) o[m][c] = tk_attn::Mma16<T>::run(vf, pf[m], o[m][c]);
      }
      return ++t == t1;
    };
    for (;;) {
      if (step(even, odd)) break;
      if (step(odd, even)) break;
    }
    pin_k();  // the keys past the end
  }

  // Row row16 of row tile m into slot `slot`.
  __device__ __forceinline__ void write(const PrefixArgs& a, int m, int64_t slot, bool mine, int quad) const {
    const float l = tk_attn::sum_over_column(sum[m]);
    if (!mine) return;
#pragma unroll
    for (int c = 0; c < OC; ++c)
      *reinterpret_cast<f32x4*>(a.part_o + slot * D + 16 * c + 4 * quad) = o[m][c];
    if (quad == 0) a.part_ml[slot] = float2{top[m], l};
  }
};

// NS ring stages of a workgroup; an own run's wave has up to NS / own_waves(W) of them. kShared: there are
// several row blocks, which share the prefix's tiles in L2.
template <typename T, int D, int W, int MT, int NS, bool kShared>
__global__ __launch_bounds__(64 * W, W >= 4 ? 2 : 1) void prefix_split_kernel(PrefixArgs a) {
  using R = Ring<D>;
  constexpr int DC = D / 32;
  __shared__ __attribute__((aligned(1024))) char ring[NS * R::STAGE];
  const uint32_t ring_base = (uint32_t)(uintptr_t)(tk_attn::lds_void*)ring;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row16 = lane & 15;
  const int quad = lane >> 4;
  const Deal deal = make_deal<W>(a, lane);
  const float scale = a.scale_log2;
  auto nothing = []() {};
  // The prefix's workgroups come first: the row blocks of a (run, KV head) are dealt to one XCD
  // (workgroup index modulo 8), one after the other, so that they share its L2.
  const int pairs = deal.prefix_runs * a.kv_heads;
  const int prefix_groups = (pairs + 7) / 8 * 8 * a.row_blocks;

  if (int(blockIdx.x) < prefix_groups) {
    constexpr int PER = R::IPT / W;     // this wave's instructions per tensor tile
    constexpr int STEP = 2 * PER, LA = NS - 1;
    static_assert((MT == 1 ? LA : NS) * STEP + MT * DC < 64, "ring deeper than the vmcnt counter");
    const int eighth = a.by_row_blocks.div(blockIdx.x / 8);
    const int pair = eighth * 8 + blockIdx.x % 8;
    const int rb = blockIdx.x / 8 - eighth * a.row_blocks;
    if (pair >= pairs) return;
    const int run = a.by_kv_heads.div(pair);
    const int kvh = pair - run * a.kv_heads;
    const int t0 = run * deal.prefix_chunk;
    const int t1 = min(t0 + deal.prefix_chunk, a.prefix_tiles);
    const int limit = min(a.prefix_len, t1 * kTileKeys);
    const int w0 = rb * 16 * W * MT + wave * 16 * MT;  // this wave's first row
    const bool busy = w0 < a.rows;                      // waves past the last row only fetch

    Rows<T, D, MT> x;
    // Q^T fragments: row w0 + 16 m + row16 (zero past the last), dims 32 c + 8 quad .. +7. A negative
    // scale is taken into Q's signs (exact), so that the largest score is the largest product.
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = w0 + 16 * m + row16;
      const int64_t b = a.by_group.div(r);
      const int64_t h = kvh * a.group + (r - b * a.group);
      const T* p = static_cast<const T*>(a.q) + b * a.qb + h * a.qh + 8 * quad;
#pragma unroll
      for (int c = 0; c < DC; ++c)
        x.qf[m][c] = r < a.rows ? *reinterpret_cast<const i32x4*>(p + 32 * c) : i32x4{0, 0, 0, 0};
    }
    __builtin_amdgcn_sched_barrier(0);
    Stream<D, PER, kShared ? 0 : kNonTemporal> ks, vs;
    const int first = t0 * kTileKeys;
    ks.template start<false>(static_cast<const T*>(a.kp) + kvh * a.kph + first * a.kpl, a.kpl, limit - first,
                             wave, lane);
    vs.template start<true>(static_cast<const T*>(a.vp) + kvh * a.vph + first * a.vpl, a.vpl, limit - first,
                            wave, lane);
    char* mine = ring + wave * PER * 1024;
    auto fetch = [&](int stage) {
      ks.next(mine + stage * R::STAGE);
      vs.next(mine + stage * R::STAGE + R::TILE);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto fetch_k = [&](int stage) {
      ks.next(mine + stage * R::TILE);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto fetch_v = [&](int stage) {
      vs.next(mine + (NS + stage) * R::TILE);
      __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (MT == 1) {
#pragma unroll
      for (int i = 0; i < LA; ++i) fetch(i);
    } else {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        fetch_k(i);
        fetch_v(i);
      }
    }
    x.start(row16, quad);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        x.qf[m][c] ^= a.flip;
        tk_attn::pin(x.qf[m][c]);
      }
    if constexpr (MT == 1) {
      int stage = 0;
      for (int t = t0; t < t1; ++t) {
        // A tile has landed (this wave's share) once only the LA - 1 younger tiles' loads are
        // outstanding; behind the barrier every wave's share has, and every wave has read the tile
        // before it, whose stage the tile fetched now takes.
        tk_attn::wait_vmcnt<(LA - 1) * STEP>();
        if constexpr (W > 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        fetch(stage == 0 ? NS - 1 : stage - 1);
        const uint32_t at = ring_base + stage * R::STAGE;
        stage = stage == NS - 1 ? 0 : stage + 1;
        if (!busy) continue;
        f32x4 s[MT][2];
        i32x4 pf[MT];
        x.scores(at, s, nothing);
        x.request_v(at, 0);
        x.cut(limit - t * kTileKeys, quad, s);
        x.softmax(s, scale, pf);
        x.accumulate(at, pf, nothing);
      }
    } else {
      x.template pipeline<NS, PER>(ring_base, t0, t1, limit, quad, scale, busy, fetch_k, fetch_v);
    }
    // The tiles issued past the end still write (zeros) into the ring.
    tk_attn::wait_vmcnt<0>();
    if (!busy) return;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = w0 + 16 * m + row16;
      x.write(a, m, (int64_t(run) * a.kv_heads + kvh) * a.rows + r, r < a.rows, quad);
    }
    return;
  }

  // A run of a sequence's own cache for each wave. K and V of a stage are refilled apart, each as soon
  // as it has been read, so that even a single stage keeps loads in flight.
  // Stages of the slice: at most 63 loads may be outstanding, Q's among them.
  constexpr int OW = own_waves(W), PER = R::IPT;
  constexpr int SS = NS / OW * 2 * PER + DC < 64 ? NS / OW : NS / OW - 1;
  static_assert(SS >= 1 && SS * 2 * PER + DC < 64, "slice deeper than the vmcnt counter");
  if (wave >= OW) return;
  const int unit = (blockIdx.x - prefix_groups) * OW + wave;
  const int f = a.by_kv_heads.div(unit);
  const int kvh = unit - f * a.kv_heads;
  OwnRun run;
  if (!find_own(a, deal, f, lane, run)) return;
  const int64_t b = run.b;
  // A sequence's runs are of one length, but for the last.
  const int tiles = tiles_in(run.length);
  const int per = (tiles + run.splits - 1) / run.splits;
  const int t0 = min(run.split * per, tiles);
  const int t1 = min(t0 + per, tiles);
  const int limit = min(run.length, t1 * kTileKeys);
  // Every run's rows are the G heads of its sequence, 16 at a time: a larger group reads the run again for
  // every 16 (16 sequences of 2 KV heads and 16384 own keys, 271 MB: G16 62 us, G32 115, G64 220), which
  // make_deal's price of an own tile leaves out.
  for (int r0 = 0; r0 < a.group; r0 += 16) {
    Rows<T, D, 1> x;
    const int r = r0 + row16;
    const T* p = static_cast<const T*>(a.q) + b * a.qb + (kvh * a.group + r) * a.qh + 8 * quad;
#pragma unroll
    for (int c = 0; c < DC; ++c)
      x.qf[0][c] = r < a.group ? *reinterpret_cast<const i32x4*>(p + 32 * c) : i32x4{0, 0, 0, 0};
    __builtin_amdgcn_sched_barrier(0);
    Stream<D, PER> ks, vs;
    const int first = t0 * kTileKeys;
    ks.template start<false>(static_cast<const T*>(a.k) + b * a.kb + kvh * a.kh + first * a.kl, a.kl,
                             limit - first, 0, lane);
    vs.template start<true>(static_cast<const T*>(a.v) + b * a.vb + kvh * a.vh + first * a.vl, a.vl,
                            limit - first, 0, lane);
    char* slice = ring + wave * (NS / OW) * R::STAGE;
#pragma unroll
    for (int i = 0; i < SS; ++i) {
      ks.next(slice + i * R::STAGE);
      vs.next(slice + i * R::STAGE + R::TILE);
    }
    __builtin_amdgcn_sched_barrier(0);
    x.start(row16, quad);
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      x.qf[0][c] ^= a.flip;
      tk_attn::pin(x.qf[0][c]);
    }
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
      char* here = slice + stage * R::STAGE;
      const uint32_t at = ring_base + uint32_t(here - ring);
      stage = stage == SS - 1 ? 0 : stage + 1;
      f32x4 s[1][2];
      i32x4 pf[1];
      // The tile's keys are followed by its values and SS - 1 tiles.
      tk_attn::wait_vmcnt<(SS - 1) * 2 * PER + PER>();
      x.scores(at, s, [&]() { ks.next(here); });
      // And its values by SS - 1 tiles and the keys just sent for.
      tk_attn::wait_vmcnt<(SS - 1) * 2 * PER + PER>();
      x.request_v(at, 0);
      x.cut(limit - t * kTileKeys, quad, s);
      x.softmax(s, scale, pf);
      x.accumulate(at, pf, [&]() { vs.next(here + R::TILE); });
    }
    // The tiles issued past the end still write (zeros) into the slice.
    tk_attn::wait_vmcnt<0>();
    const int64_t slot = int64_t(a.most_runs) * a.kv_heads * a.rows + (int64_t(f) * a.kv_heads + kvh) * a.group + r;
    x.write(a, 0, slot, r < a.group, quad);
  }
}

// A row's partial results, the prefix's first.
template <typename T, int D, int W, int WAVES>
__global__ __launch_bounds__(64 * kJoinWaves) void prefix_combine_kernel(PrefixArgs a) {
  __shared__ JoinScratch<D> shared;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = WAVES == 1 ? blockIdx.x * kJoinWaves + wave : blockIdx.x;
  const int b = blockIdx.y;
  const Deal deal = make_deal<W>(a, lane);
  // Runs and first flat run of sequence b.
  int before = 0, splits = 0, flat0 = 0;
  for (int b0 = 0; b0 <= b; b0 += 64) {
    const int i = b0 + lane;
    const int len = b0 == 0 ? deal.first : (i < a.batch ? own_length(a, i) : 0);
    const int mine = (tiles_in(len) + deal.own_chunk - 1) / deal.own_chunk;
    const int upto = before + wave_prefix(mine);
    if (b < b0 + 64) {
      splits = __builtin_amdgcn_readlane(mine, b - b0);
      flat0 = __builtin_amdgcn_readlane(upto, b - b0) - splits;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  if (h >= a.q_heads) return;
  const int kvh = a.by_group.div(h);
  const int g = h - kvh * a.group;
  const int64_t prefix_step = int64_t(a.kv_heads) * a.rows, own_step = int64_t(a.kv_heads) * a.group;
  const int64_t prefix0 = int64_t(kvh) * a.rows + int64_t(b) * a.group + g;
  const int64_t own0 = int64_t(a.most_runs) * prefix_step + (int64_t(flat0) * a.kv_heads + kvh) * a.group + g;
  join_parts<T, D, WAVES, Rows<T, D, 1>::kLift>(a.part_o, a.part_ml, deal.prefix_runs + splits,
                          [&](int i) {
                            return i < deal.prefix_runs ? prefix0 + i * prefix_step
                                                        : own0 + (i - deal.prefix_runs) * own_step;
                          },
                          static_cast<T*>(a.o) + b * a.ob + h * a.oh,
                          a.lse == nullptr ? nullptr : a.lse + int64_t(b) * a.q_heads + h, wave, shared);
}

// Workgroup shapes by the rows a KV head has: 16 rows a wave up to four waves, then 32 rows a wave.
// `price` of a prefix tile for a workgroup, in 1/16 of an own tile for a wave.
struct Shape {
  int waves, row_tiles, price;
};
Shape shape_for(int64_t rows) {
  if (rows <= 16) return {1, 1, 16};
  if (rows <= 32) return {2, 1, 10};
  if (rows <= 64) return {4, 1, 6};
  return {4, 2, 7};
}
constexpr int kWorkgroups = 512;  // two per CU, each with a 64 KiB ring

// Instantiated here by name: left to the launches below, the host compiler leaves some of these
// kernels' launch stubs undefined.
#define TK_SPLIT(T, D, W, MT, NS, SHARED) \
  template __global__ void prefix_split_kernel<T, D, W, MT, NS, SHARED>(PrefixArgs)
#define TK_SPLITS(T)                                                                                  \
  TK_SPLIT(T, 128, 1, 1, 4, false); TK_SPLIT(T, 128, 2, 1, 4, false); TK_SPLIT(T, 128, 4, 1, 4, false); \
  TK_SPLIT(T, 128, 4, 2, 4, false); TK_SPLIT(T, 128, 4, 2, 4, true);                                  \
  TK_SPLIT(T, 64, 1, 1, 8, false); TK_SPLIT(T, 64, 2, 1, 8, false); TK_SPLIT(T, 64, 4, 1, 8, false);  \
  TK_SPLIT(T, 64, 4, 2, 8, false); TK_SPLIT(T, 64, 4, 2, 8, true)
TK_SPLITS(__bf16);
TK_SPLITS(_Float16);

template <typename T, int D, int W, int MT>
void launch_shape(const PrefixArgs& a, uint32_t workgroups, hipStream_t s) {
  constexpr int NS = D == 128 ? 4 : 8;
  if (MT == 2 && a.row_blocks > 1)
    hipLaunchKernelGGL((prefix_split_kernel<T, D, W, MT, NS, MT == 2>), dim3(workgroups), dim3(64 * W), 0, s, a);
  else
    hipLaunchKernelGGL((prefix_split_kernel<T, D, W, MT, NS, false>), dim3(workgroups), dim3(64 * W), 0, s, a);
  if (int64_t(a.q_heads) * a.batch <= kFewRows)
    hipLaunchKernelGGL((prefix_combine_kernel<T, D, W, kJoinWaves>), dim3(a.q_heads, a.batch),
                       dim3(64 * kJoinWaves), 0, s, a);
  else
    hipLaunchKernelGGL((prefix_combine_kernel<T, D, W, 1>),
                       dim3(static_cast<uint32_t>(tk::cdiv(a.q_heads, kJoinWaves)), a.batch),
                       dim3(64 * kJoinWaves), 0, s, a);
}

template <typename T, int D>
void launch(const PrefixArgs& a, uint32_t workgroups, hipStream_t s) {
  const Shape shape = shape_for(a.rows);
  if (shape.waves == 1)
    launch_shape<T, D, 1, 1>(a, workgroups, s);
  else if (shape.waves == 2)
    launch_shape<T, D, 2, 1>(a, workgroups, s);
  else if (shape.row_tiles == 1)
    launch_shape<T, D, 4, 1>(a, workgroups, s);
  else
    launch_shape<T, D, 4, 2>(a, workgroups, s);
}

// Bounds on how the device cuts a call: prefix runs, own flat runs, workgroups.
struct Plan {
  int64_t row_blocks, most_runs, most_own, workgroups;
};
Plan make_plan(int64_t batch, int64_t kv_heads, int64_t group, int64_t prefix_len, int64_t max_len) {
  Plan p;
  const Shape shape = shape_for(batch * group);
  p.row_blocks = tk::cdiv(batch * group, 16 * shape.waves * shape.row_tiles);
  const int64_t prefix_tiles = tk::cdiv(prefix_len, kTileKeys), own_tiles = tk::cdiv(max_len, kTileKeys);
  // The prefix's runs if it were alone, and at most one for every kLeastRun tiles.
  p.most_runs = tk::cdiv(kWorkgroups, kv_heads * p.row_blocks);
  if (p.most_runs > tk::cdiv(prefix_tiles, kLeastRun)) p.most_runs = tk::cdiv(prefix_tiles, kLeastRun);
  // The own runs if they were alone, and one more per sequence, which ends in a shorter one.
  p.most_own = tk::cdiv(2 * kWorkgroups * own_waves(shape.waves), kv_heads) + batch;
  if (p.most_own > batch * tk::cdiv(own_tiles, kLeastRun)) p.most_own = batch * tk::cdiv(own_tiles, kLeastRun);
  p.workgroups = tk::cdiv(p.most_runs * kv_heads, 8) * 8 * p.row_blocks + tk::cdiv(p.most_own * kv_heads, own_waves(shape.waves));
  return p;
}

// Why a problem of these (positive) sizes is not taken, or null. The grid holds at most 2^22
// workgroups, and tiles, partial results and a share's tiles (make_deal) are counted in 32 bits.
const char* unsupported(int64_t batch, int64_t kv_heads, int64_t group, int64_t prefix_len, int64_t max_len,
                        int64_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
  if (batch > 65535 || kv_heads > 65535 || group > 65535 || kv_heads * group > 65535 ||
      prefix_len > (1 << 30) || max_len > (1 << 30) || batch * group > (1 << 22))
    return "problem too large";
  const Plan p = make_plan(batch, kv_heads, group, prefix_len, max_len);
  if (batch * tk::cdiv(max_len, kTileKeys) > INT32_MAX / 2 || p.workgroups > (1 << 22) ||
      p.most_runs * kv_heads * batch * group + p.most_own * kv_heads * group > INT32_MAX)
    return "problem too large";
  const Shape shape = shape_for(batch * group);
  const double prefix_work = double(tk::cdiv(prefix_len, kTileKeys)) * double(kv_heads * p.row_blocks);
  const double own_work = double(batch * tk::cdiv(max_len, kTileKeys)) * double(kv_heads) / own_waves(shape.waves);
  if (prefix_work + own_work * 16 / shape.price > double(kWorkgroups) * (1 << 30)) return "problem too large";
  return nullptr;
}

}  // namespace

extern "C" int tk_prefix_decode_slots(int64_t batch, int64_t kv_heads, int64_t group, int64_t prefix_len,
                                      int64_t max_len, int64_t head_dim) {
  if (batch <= 0 || kv_heads <= 0 || group <= 0 || prefix_len <= 0 || max_len <= 0) return -1;
  if (unsupported(batch, kv_heads, group, prefix_len, max_len, head_dim) != nullptr) return -1;
  const Plan p = make_plan(batch, kv_heads, group, prefix_len, max_len);
  return static_cast<int>(p.most_runs * kv_heads * batch * group + p.most_own * kv_heads * group);
}

extern "C" int tk_prefix_decode(int dtype, const void* q, const void* k_prefix, const void* v_prefix,
                                const void* k_cache, const void* v_cache, const int32_t* seqlens, void* o,
                                float* lse, float* workspace, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                int64_t prefix_len, int64_t max_len, int64_t head_dim, const int64_t* q_strides,
                                const int64_t* k_prefix_strides, const int64_t* v_prefix_strides,
                                const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                                float scale, void* stream) {
  if (dtype != TK_DTYPE_F16 && dtype != TK_DTYPE_BF16)
    return tk::fail("prefix decode: dtype must be float16 or bfloat16");
  if (q == nullptr || k_prefix == nullptr || v_prefix == nullptr || k_cache == nullptr || v_cache == nullptr ||
      o == nullptr || workspace == nullptr || q_strides == nullptr || k_prefix_strides == nullptr ||
      v_prefix_strides == nullptr || k_strides == nullptr || v_strides == nullptr || o_strides == nullptr)
    return tk::fail("prefix decode: null pointer");
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || prefix_len <= 0 || max_len <= 0)
    return tk::fail("prefix decode: empty problem");
  if (q_heads % kv_heads != 0) return tk::fail("prefix decode: q_heads must be a multiple of kv_heads");
  const int64_t group = q_heads / kv_heads;
  if (const char* why = unsupported(batch, kv_heads, group, prefix_len, max_len, head_dim))
    return tk::fail("prefix decode: %s", why);
  const Plan plan = make_plan(batch, kv_heads, group, prefix_len, max_len);
  for (const void* p : {q, k_prefix, v_prefix, k_cache, v_cache, static_cast<const void*>(o),
                        static_cast<const void*>(workspace)})
    if (!tk::aligned16(p)) return tk::fail("prefix decode: tensors must be 16-byte aligned");
  struct {
    const int64_t* strides;
    int count;
  } tables[] = {{q_strides, 2}, {o_strides, 2}, {k_prefix_strides, 2}, {v_prefix_strides, 2}, {k_strides, 3}, {v_strides, 3}};
  for (const auto& t : tables)
    for (int d = 0; d < t.count; ++d)
      if (t.strides[d] < 0 || t.strides[d] % 8 != 0 || t.strides[d] >= (int64_t(1) << 40))
        return tk::fail("prefix decode: strides must be non-negative multiples of 8 elements");
  // The DMA addresses a tile's 32 rows through 32-bit buffer offsets.
  for (int64_t stride : {k_prefix_strides[1], v_prefix_strides[1], k_strides[2], v_strides[2]})
    if (stride >= (int64_t(1) << 24))
      return tk::fail("prefix decode: key strides must be below 2^24 elements");
  const Shape shape = shape_for(batch * group);
  PrefixArgs a;
  a.q = q, a.kp = k_prefix, a.vp = v_prefix, a.k = k_cache, a.v = v_cache;
  a.seqlens = seqlens;
  a.o = o;
  a.lse = lse;
  a.part_o = workspace;
  const int64_t slots = plan.most_runs * kv_heads * batch * group + plan.most_own * kv_heads * group;
  a.part_ml = reinterpret_cast<float2*>(workspace + slots * head_dim);
  a.qb = q_strides[0], a.qh = q_strides[1];
  a.ob = o_strides[0], a.oh = o_strides[1];
  a.kph = k_prefix_strides[0], a.kpl = k_prefix_strides[1];
  a.vph = v_prefix_strides[0], a.vpl = v_prefix_strides[1];
  a.kb = k_strides[0], a.kh = k_strides[1], a.kl = k_strides[2];
  a.vb = v_strides[0], a.vh = v_strides[1], a.vl = v_strides[2];
  a.by_group = tk::FastDiv(static_cast<uint32_t>(group));
  a.by_kv_heads = tk::FastDiv(static_cast<uint32_t>(kv_heads));
  a.by_row_blocks = tk::FastDiv(static_cast<uint32_t>(plan.row_blocks));
  a.batch = static_cast<int>(batch);
  a.q_heads = static_cast<int>(q_heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(group);
  a.rows = static_cast<int>(batch * group);
  a.max_len = static_cast<int>(max_len);
  a.prefix_len = static_cast<int>(prefix_len);
  a.prefix_tiles = static_cast<int>(tk::cdiv(prefix_len, kTileKeys));
  a.row_blocks = static_cast<int>(plan.row_blocks);
  a.workgroups = kWorkgroups;
  a.price = shape.price;
  a.most_runs = static_cast<int>(plan.most_runs);
  a.most_own = static_cast<int>(plan.most_own);
  // Not 0, which would turn a masked score (-inf) into NaN: the least subnormal float (which the
  // kernel's multiplications keep) leaves no score at or above 2^-149 * 2^128 = 2^-21, as good as 0
  // to the hardware exponential.
  a.scale_log2 = fmaxf(fabsf(scale) * kLog2e, 0x1p-149f);
  a.flip = scale < 0.f ? int(0x80008000u) : 0;
  hipStream_t s = tk::as_stream(stream);
  const uint32_t workgroups = static_cast<uint32_t>(plan.workgroups);
  if (dtype == TK_DTYPE_BF16) {
    if (head_dim == 128)
      launch<__bf16, 128>(a, workgroups, s);
    else
      launch<__bf16, 64>(a, workgroups, s);
  } else {
    if (head_dim == 128)
      launch<_Float16, 128>(a, workgroups, s);
    else
      launch<_Float16, 64>(a, workgroups, s);
  }
  return tk::check_launch("prefix decode");
}
