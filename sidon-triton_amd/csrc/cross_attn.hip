// cross_attn.hip -- attention over states of another length (MI355X / gfx950):
//
//   o_i = sum_{j < lens} softmax_j(scale q_i . k_j) v_j
//   lse_i = log(sum_{j < lens} exp(scale q_i . k_j))
//
// for queries i < q_lens, head dim D 64 or 128.  Grouped heads share keys and
// values: the G heads of a group and their L queries are G L rows over one key
// head, a query's heads side by side.
//
// A wavefront owns 32 rows: S^T = K . Q^T by v_mfma_f32_32x32x16, an online softmax
// with the running maximum raised only when a step's probabilities would leave the
// fp16 range, O^T += V^T . P^T.  Key rows enter the A operand with bits 2 and 3 of
// their index swapped, which makes the accumulator, rounded to 16 bits, the B operand
// of the second product; the sums of the rounded probabilities, which the result is
// divided by, come from the matrix core too.  In a round a wavefront takes the
// softmax of one step and the values of the step before, whose vector and matrix
// instructions do not wait for each other.
//
// Keys go by steps of 32: a step's keys and values are copied global -> LDS by
// global_load_lds_dwordx4, as tiles of 32 rows x 128 bytes with swizzled 16-byte
// chunks; keys are read with ds_read_b128, values transposed with
// ds_read_b64_tr_b16.  RB row blocks share a ring of two key and three value slots;
// KS such groups take every KS-th step and are merged through LDS; over the grid a
// row block's steps can be split again, each part leaving (max, sums, O) in fp32 for
// a joining launch.
//
// What bounds it, and what it reached.  Long prompts: of a step's 20 matrix and 180
// vector instructions (64 rows) neither hides all of the other; 16 heads x 4800 x 4800 take
// 122 us at D 64 (0.77 PFLOP/s) and 209 at D 128 (0.90).  Short ones: a workgroup's first
// copies, merge and stores, 6 to 8 us, beside few rounds (4 x 16 heads x 224 x 1500 14 us).  Single
// tokens: memory; 32 streams of up to 4800 keys, 4 key heads (81 MB) 23 us, 3.5 TB/s; one
// of 1500 keys, two launches of a few memory latencies, 9 us.
#include <hip/hip_runtime.h>

#include <float.h>
#include <math.h>
#include <stdint.h>

#include "attn_device.h"
#include "sidon_host.h"
#include "sidon_operators.h"
#include "sidon_wave.h"

#define SIDON_API extern "C" __attribute__((visibility("default")))
#define SIDON_INLINE __attribute__((always_inline))

namespace {

using namespace sidon_attn;

constexpr int kBlock = 32;          // rows per wavefront
constexpr int kMaxGridSplits = 64;
constexpr float kLn2 = 0.6931471805599453f;

struct CrossParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;            // [B, H, L] or null
  const int32_t* lens;
  const int32_t* q_lens;
  float4* part_ml;       // [B Hk, splits, rest] (maximum, sum, sum before the rounding, -)
  float* part_o;         // [B Hk, splits, rest, D]
  int64_t qb, qh, ql, kb, kh, vb, vh, ob, oh, ol;   // strides (elements): batch, head, row
  int kl, vl;            // row strides (< 2^25)
  int B, H, Hk, G, L, S, R;
  int whole, cut, splits;   // row blocks of a key head that a workgroup takes whole, those that `splits` share
  int first, rest;          // the rows of the latter: from `first` on, `rest` of them
  Deal deal;                // a key head's units: blocks, then (split, block)
  float scale;           // log2(e) times the caller's
};

// A workgroup: RB wavefronts of NB row blocks each x KS key groups.  The wavefronts of a
// key group share a ring of two key slots and three value slots, a step of 32 keys each.
template <int D, int NB, int RB, int KS>
struct Shape {
  static constexpr int kWaves = RB * KS;
  static constexpr int kP = D / 64;                   // 128-byte panels
  static constexpr int kSlot = kP * kTile;            // bytes of a step's keys, or of its values
  static constexpr int kV = 2 * kSlot;                // value slots behind the key slots
  static constexpr int kRing = 5 * kSlot;
  static constexpr int kDb = D / 32;                  // 32-wide blocks of the values
  static constexpr int kPart = NB * (kDb * 16 + 4) * 64 * 4;   // bytes of a wavefront's partial result
  static constexpr int kMerge = KS > 1 ? KS / 2 * RB * kPart : 0;
  static constexpr int kLds = KS * kRing > kMerge ? KS * kRing : kMerge;
  static constexpr int kCopies = kSlot / 1024 / RB;   // 1 KB copies per wavefront and slot
  static_assert(kLds <= 160 * 1024, "LDS");
  static_assert(kSlot / 1024 % RB == 0, "an even split of the copies");
};

// kFine: probabilities as two summands of the type, the rounded value and what the
// rounding left, so that only the output is rounded.  For few rows, where memory and
// latency leave the matrix cores idle.
// kLse: the sums of probabilities before their rounding are wanted, and the rounded ones'
// do not stand for them (kFine's do).
template <typename E, int D, int NB, int RB, int KS, bool kFine, bool kLse, int kMinWaves>
__global__ void __launch_bounds__(64 * RB * KS, kMinWaves) cross_attn_kernel(const CrossParams p) {
  using C = Shape<D, NB, RB, KS>;
  static_assert(!(kFine && kLse), "the sums of two summands are as good");
  typedef typename Half<E>::v2 v2;
  typedef typename Half<E>::v4 v4;
  constexpr int kDb = C::kDb;
  constexpr int kQ = D / 16;          // Q operands
  __shared__ __attribute__((aligned(16))) char smem[C::kLds];

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = w % RB, ks = w / RB;
  const int n = lane & 31, g = lane >> 5;

  int bh;
  const int unit = dealt(p.deal, blockIdx.x, bh);
  if (unit >= p.deal.units) return;
  const bool alone = unit < p.whole;
  const int split = alone ? 0 : (unit - p.whole) / p.cut;
  const int blk = alone ? unit : unit - split * p.cut;
  const uint32_t splits = alone ? 1 : p.splits;
  const int b = bh / p.Hk, hk = bh - b * p.Hk;
  const int row0 = (blk * RB + rb) * (NB * kBlock);   // of this wavefront
  // Lane n holds the rows row0 + 32 j + n, j < NB: query row / G, head row % G of the group.

  int lk = p.S, rows = p.R;                    // valid keys, rows of valid queries
  if (p.lens != nullptr) lk = __builtin_amdgcn_readfirstlane(min(max(p.lens[b], 0), p.S));
  if (p.q_lens != nullptr) rows = p.G * __builtin_amdgcn_readfirstlane(min(max(p.q_lens[b], 0), p.L));

  const int steps = blk * RB * NB * kBlock < rows ? (lk + kStep - 1) / kStep : 0;   // of the workgroup
  const int t0 = (int)((uint32_t)steps * (uint32_t)split / splits);   // (steps <= 2^25, splits <= 2^6)
  const int t1 = (int)((uint32_t)steps * (uint32_t)(split + 1) / splits);
  const auto mine = [&](int u) SIDON_INLINE { return t0 + u * KS + ks; };   // step u of this group
  const int all = (t1 - t0 + KS - 1) / KS;         // most steps of a group: the workgroup's rounds
  const int count = row0 < rows ? max(t1 - t0 - ks + KS - 1, 0) / KS : 0;    // of this wavefront

  // ---- copies into the ring, split over its wavefronts: 1 KB copy i is rows
  // 8 (i % 4) + [0, 8) of panel i / 4 (dims 64 (i / 4)) ----
  const uint32_t ring = (uint32_t)(uintptr_t)SIDON_LDS_PTR(char, smem) + ks * C::kRing + rb * C::kCopies * 1024;
  const int pid0 = rb * C::kCopies / 4, crow = rb * C::kCopies % 4 * 8 + (lane >> 3);
  const char* const kbase = static_cast<const char*>(p.k) + 2 * (b * p.kb + hk * p.kh) + pid0 * 128 - kBack;
  const char* const vbase = static_cast<const char*>(p.v) + 2 * (b * p.vb + hk * p.vh) + pid0 * 128 - kBack;
  const int whole = min(t1, lk / kStep);   // steps below it have all their rows
  // Copy j of a set adds 1024 j to the LDS and to the global address; copies of
  // the next panel (j >= 4) lie 128 bytes on.
  constexpr int kOffs = C::kCopies;
  const auto offset = [&](int j, int r, int stride) SIDON_INLINE {
    return (uint32_t)r * (uint32_t)(2 * stride) + 16u * ((lane & 7) ^ tile_swz(crow + 8 * (j % 4))) + j / 4 * 128u +
           1024u * (3 - j % 4);
  };
  uint32_t koff[kOffs], voff[kOffs];
#pragma unroll
  for (int j = 0; j < kOffs; ++j) {
    koff[j] = offset(j, crow + 8 * (j % 4), p.kl);
    voff[j] = offset(j, crow + 8 * (j % 4), p.vl);
  }
  const auto issue = [&](uint32_t at, const char* src, const uint32_t (&off)[kOffs]) SIDON_INLINE {
    static_assert(kOffs == 1 || kOffs == 2 || kOffs % 4 == 0, "copies go by one, two or four");
    if constexpr (kOffs >= 4) {
#pragma unroll
      for (int j = 0; j < kOffs; j += 4) dma_tile(at + j * 1024, src, off[j], off[j + 1], off[j + 2], off[j + 3]);
    } else if constexpr (kOffs == 2) {
      dma_2k(at, src, off[0], off[1]);
    } else {
      dma_1k(at, src, off[0]);
    }
  };
  // Step t's copies; `src` is where its rows begin, less the 3 KB that the offsets hold.
  const auto copy = [&](int t, uint32_t at, const char* src, int stride, const uint32_t (&off)[kOffs]) SIDON_INLINE {
    if (t < whole) {
      issue(at, src, off);
    } else if (t < t1) {
      // Rows past the valid keys read the last valid one again: their
      // probabilities are 0, and what lies there may be anything.
      uint32_t part[kOffs];
#pragma unroll
      for (int j = 0; j < kOffs; ++j) part[j] = offset(j, min(crow + 8 * (j % 4), lk - t * kStep - 1), stride);
      issue(at, src, part);
    }
  };
  int tk = mine(0), tv = mine(0);   // the steps that are copied next
  uint32_t kat = ring, vat = ring + C::kV;
  const int64_t kgo = (int64_t)p.kl * (2 * kStep * KS), vgo = (int64_t)p.vl * (2 * kStep * KS);
  const char* ksrc = kbase + (int64_t)p.kl * (2 * kStep) * tk;
  const char* vsrc = vbase + (int64_t)p.vl * (2 * kStep) * tv;
  const auto copy_k = [&]() SIDON_INLINE {
    copy(tk, kat, uniform(ksrc), p.kl, koff);
    tk += KS;
    ksrc += kgo;
    kat = 2 * ring + C::kSlot - kat;
  };
  const auto copy_v = [&]() SIDON_INLINE {
    copy(tv, vat, uniform(vsrc), p.vl, voff);
    tv += KS;
    vsrc += vgo;
    vat = vat == ring + C::kV + 2 * C::kSlot ? ring + C::kV : vat + C::kSlot;
  };
  copy_k();
  copy_k();
  copy_v();

  // ---- Q^T operands: lane (n, g) holds query n, dims 16 s + 8 g + [0, 8); rows past
  // the valid ones hold the last valid one (or the first row, where none is) ----
  i4 qop[NB][kQ];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int rr = max(min(row0 + 32 * j + n, rows - 1), 0);
    const E* qp = static_cast<const E*>(p.q) + b * p.qb + (hk * p.G + rr % p.G) * p.qh + (rr / p.G) * p.ql + 8 * g;
#pragma unroll
    for (int s = 0; s < kQ; ++s) qop[j][s] = *reinterpret_cast<const i4*>(qp + 16 * s);
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) arrived(qop[j]);

  // ---- operand offsets from the first key and value slot ----
  int kaddr[4], vaddr[2][2];
  {
    const int krow = mfma_row_perm(n);
#pragma unroll
    for (int i = 0; i < 4; ++i) kaddr[i] = ks * C::kRing + krow * 128 + (((2 * i + g) ^ tile_swz(krow)) << 4);
    const int G4 = lane >> 4, a = (lane >> 2) & 3, bq = lane & 3;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        const int r = 8 * (G4 >> 1) + 4 * hf + a;
        const int chunk = 4 * db + 2 * (G4 & 1) + (bq >> 1);
        vaddr[hf][db] = ks * C::kRing + C::kV + r * 128 + ((chunk ^ tile_swz(r)) << 4) + 8 * (bq & 1);
      }
  }

  i4 sel;
  {
    const E one = (((lane >> 4) ^ (lane >> 2)) & 1) == 0 ? (E)1.f : (E)0.f;
    const int pair = __builtin_bit_cast(int, v2{one, one});
    sel = i4{pair, pair, pair, pair};
  }

  f32x16 o[NB][kDb];
  // Of a row: maximum of the scaled scores, less kLift; sum of the rounded probabilities;
  // this lane's share of their sum before the rounding.
  float mx[NB], sum[NB], raw[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    mx[j] = kFloorMax, sum[j] = 0.f, raw[j] = 0.f;
#pragma unroll
    for (int d = 0; d < kDb; ++d) o[j][d] = f32x16{};
  }
  f32x16 s[NB];                      // scores of a step: element i is key 16 (i / 8) + 8 g + i % 8
  constexpr int kTerms = kFine ? 2 : 1;
  i4 pk[NB][kTerms][2];              // its probabilities

  // The three parts of a step.  In round u a wavefront takes the softmax of step
  // u and the product with the values of step u - 1, whose vector and matrix
  // instructions are independent, then the scores of step u + 1.
  i4 kop[kQ];
  uint32_t kread = 0, vread = 0;   // slots that are read next
  const auto load_keys = [&]() SIDON_INLINE {
#pragma unroll
    for (int i = 0; i < kQ; ++i)
      kop[i] = *reinterpret_cast<const i4*>(smem + (kaddr[i % 4] + kread) + i / 4 * kTile);
    kread ^= C::kSlot;
  };
  const auto scores = [&]() SIDON_INLINE {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      f32x16 acc = {};
#pragma unroll
      for (int i = 0; i < kQ; ++i) acc = Half<E>::mfma(kop[i], qop[j][i], acc);
      s[j] = acc;
    }
  };
  int k0 = mine(0) * kStep;   // first key of the step in s
  const auto hide = [&]() SIDON_INLINE {
    if (k0 + kStep > lk) {
      const int left = lk - k0 - 8 * g;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (16 * (i >> 3) + (i & 7) >= left) s[j][i] = -INFINITY;
    }
    k0 += KS * kStep;
  };
  const auto exps = [&](int j, float (&e)[16]) SIDON_INLINE {
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = fast_exp2(fmaf(s[j][i], p.scale, -mx[j]));
  };
  const auto total_of = [&](const float (&e)[16]) SIDON_INLINE {
    float t[4] = {};
    if constexpr (kLse) {
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i % 4] += e[i];
    }
    return (t[0] + t[1]) + (t[2] + t[3]);
  };
  // The step's probabilities, rounded.
  const auto round_to = [&](int j, const float (&e)[16]) SIDON_INLINE {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const v2 hi = __builtin_convertvector(f2{e[i], e[i + 1]}, v2);
      pk[j][0][i >> 3][(i & 7) >> 1] = __builtin_bit_cast(int, hi);
      if constexpr (kFine) {
        const f2 left = {e[i] - (float)hi[0], e[i + 1] - (float)hi[1]};
        pk[j][kTerms - 1][i >> 3][(i & 7) >> 1] = __builtin_bit_cast(int, __builtin_convertvector(left, v2));
      }
    }
  };
  // Their sum, on the matrix core, where the vector unit is the busier one.  Read
  // as a 16x16x32 B operand, a lane's half of them holds row c + 16 (l % 2) of
  // lane c + 16 l, keys 8 (l / 2) + [0, 8); the A operand is 1 where bit 4 of the
  // lane equals bit 2, so that the four numbers a lane receives are its own row's
  // sum.  The other row of the column enters times 0: where its probabilities are
  // infinite or NaN, so is this sum, and `settle` takes the row's own.
  const auto matrix_sum = [&](int j) SIDON_INLINE {
    f4 total = {};
#pragma unroll
    for (int k = 0; k < kTerms; ++k) {
      total = Half<E>::small(sel, pk[j][k][0], total);
      total = Half<E>::small(sel, pk[j][k][1], total);
    }
    return total[0];
  };
  // The same from the lane pair that holds the row, nothing else.
  const auto own_sum = [&](int j) SIDON_INLINE {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < kTerms; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = pk[j][k][i >> 2][i & 3];   // (a bit cast of the element itself takes the vector's first)
        const v2 x = __builtin_bit_cast(v2, pair);
        total += (float)x[0] + (float)x[1];
      }
    return pair_sum(total);
  };
  const auto values = [&]() SIDON_INLINE {
    typedef int i2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int d = 0; d < kDb; ++d) {
        const char* tile = smem + vread + (d / 2) * kTile + 2048 * hh;
        const i2 lo = __builtin_bit_cast(i2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(SIDON_LDS_PTR(s4, tile + vaddr[0][d & 1])));
        const i2 hi = __builtin_bit_cast(i2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(SIDON_LDS_PTR(s4, tile + vaddr[1][d & 1])));
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int k = 0; k < kTerms; ++k) o[j][d] = Half<E>::mfma(i4{lo[0], lo[1], hi[0], hi[1]}, pk[j][k][hh], o[j][d]);
      }
    vread = vread == 2 * C::kSlot ? 0 : vread + C::kSlot;
  };
  // Raises the running maximum of the rows whose probabilities do not all fit, with
  // what they have so far.  (The condition is a lane's, not the wavefront's: behind a
  // branch of the wavefront the compiler keeps the accumulators in two places.)
  const auto settle = [&](int j, float total, float exact) SIDON_INLINE {
    // One that left fp16 is an infinity in the sum.
    if (!(total < kSumLimit)) {
      total = own_sum(j);
      if (!(total < kSumLimit)) {
        float top = s[j][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[j][i]);
        top = fmaxf(mx[j], pair_max(top) * p.scale - Half<E>::kLift);
        const float alpha = fast_exp2(mx[j] - top);   // 0 from kFloorMax
#pragma unroll
        for (int d = 0; d < kDb; ++d) o[j][d] *= alpha;
        sum[j] *= alpha;
        raw[j] *= alpha;
        mx[j] = top;
        float e[16];
        exps(j, e);
        exact = total_of(e);
        round_to(j, e);
        total = own_sum(j);
      }
    }
    sum[j] += total;
    raw[j] += exact;
  };
  // Behind it the values of step u - 1 are there and, where wavefronts share the ring,
  // for all of them, with the keys of step u + 1; nobody reads the keys of step u or the
  // values of step u - 2 any more: their slots are filled with the keys of step u + 2
  // and the values of step u + 1.  Copies arrive in the order in which they were issued
  // (keys, then values, round by round), so a wait names how many of the newest it
  // leaves under way; past the last step's none are issued, and it leaves none.
  constexpr int kSet = C::kCopies;
  const int mine_all = max(t1 - t0 - ks + KS - 1, 0) / KS;   // steps that this group copies
  const auto round = [&](int u) SIDON_INLINE {
    if constexpr (RB == 1) {
      if (u + 1 < mine_all) wait_vmcnt<2 * kSet>(); else wait_vmcnt<0>();
      wait_lgkm0();
    } else {
      if (u < mine_all) wait_vmcnt<kSet>(); else wait_vmcnt<0>();
      lds_barrier();
    }
    copy_k();
    copy_v();
  };
  // The keys of step u + 1 are there too (a ring of one wavefront waits for them late).
  const auto keys_there = [&](int u) SIDON_INLINE {
    if constexpr (RB == 1) {
      if (u + 2 < mine_all) wait_vmcnt<3 * kSet>(); else wait_vmcnt<0>();
    }
  };

  // ---- rounds -1 to `all` (the first needs the first keys alone) ----
  int u = 0;
  if (all > 0) {
    wait_vmcnt<0>();
    lds_barrier();
    if (count > 0) {
      load_keys();
      scores();
    }
    round(0);
    if (count > 0) {
      hide();
      float exact[NB], total[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float e[16];
        exps(j, e);
        exact[j] = total_of(e);
        round_to(j, e);
        total[j] = matrix_sum(j);
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) settle(j, total[j], exact[j]);
      if (count > 1) {
        keys_there(0);
        load_keys();
        scores();
      }
    }
    for (u = 1; u < count; ++u) {
      round(u);
      hide();
      float e[NB][16], exact[NB], total[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) exps(j, e[j]);
      values();
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        exact[j] = total_of(e[j]);
        round_to(j, e[j]);
        total[j] = matrix_sum(j);
      }
      keys_there(u);
      load_keys();   // (of the last round: what an earlier step left in the slot, for nothing)
#pragma unroll
      for (int j = 0; j < NB; ++j) settle(j, total[j], exact[j]);
      scores();
    }
    for (; u <= all; ++u) {
      round(u);
      if (u == count && count > 0) values();
    }
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) raw[j] = kLse ? pair_sum(raw[j]) : sum[j];

  // ---- merge the key groups, half of them into the other half at a time: a wavefront's
  // partial result in LDS, lane by lane, its values, then (maximum, sums) ----
  if constexpr (KS > 1) {
    float* const mem = reinterpret_cast<float*>(smem) + lane * 4;
#pragma unroll
    for (int half = KS / 2; half >= 1; half >>= 1) {
      wait_vmcnt<0>();
      lds_barrier();   // the rings, or the last round's values, are done with
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float* at = mem + (((ks % half) * RB + rb) * NB + j) * (C::kPart / NB / 4);
        if (ks >= half) {
#pragma unroll
          for (int d = 0; d < kDb; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<f4*>(at + (d * 4 + i) * 256) =
                  f4{o[j][d][4 * i], o[j][d][4 * i + 1], o[j][d][4 * i + 2], o[j][d][4 * i + 3]};
          *reinterpret_cast<f4*>(at + kDb * 4 * 256) = f4{mx[j], sum[j], raw[j], 0.f};
        }
      }
      lds_barrier();
      if (ks >= half) return;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const float* at = mem + (((ks % half) * RB + rb) * NB + j) * (C::kPart / NB / 4);
        const f4 other = *reinterpret_cast<const f4*>(at + kDb * 4 * 256);
        const float top = fmaxf(mx[j], other[0]);
        const float fa = fast_exp2(mx[j] - top), fb = fast_exp2(other[0] - top);
        mx[j] = top;
        sum[j] = fmaf(sum[j], fa, other[1] * fb);
        raw[j] = fmaf(raw[j], fa, other[2] * fb);
#pragma unroll
        for (int d = 0; d < kDb; ++d) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f4 v = *reinterpret_cast<const f4*>(at + (d * 4 + i) * 256);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][d][4 * i + e] = fmaf(o[j][d][4 * i + e], fa, v[e] * fb);
          }
          if (d % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  // Lane (n, g) holds of row n the values 32 d + 8 i + 4 g + [0, 4).
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int row = row0 + 32 * j + n;
    if (row >= p.R) return;
    if (splits > 1) {
      const int64_t at = ((int64_t)bh * p.splits + split) * p.rest + (row - p.first);
      float* dst = p.part_o + at * D + 4 * g;
      if (g == 0) p.part_ml[at] = make_float4(mx[j], sum[j], raw[j], 0.f);
#pragma unroll
      for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f4*>(dst + 32 * d + 8 * i) =
              f4{o[j][d][4 * i], o[j][d][4 * i + 1], o[j][d][4 * i + 2], o[j][d][4 * i + 3]};
      continue;
    }
    const bool there = row < rows && lk > 0;
    const float f = there ? 1.f / sum[j] : 0.f;
    const int head = hk * p.G + row % p.G, query = row / p.G;
    if (p.lse != nullptr && g == 0)
      p.lse[((int64_t)b * p.H + head) * p.L + query] = there ? (mx[j] + __log2f(raw[j])) * kLn2 : -INFINITY;
    E* dst = static_cast<E*>(p.out) + b * p.ob + head * p.oh + query * p.ol + 4 * g;
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = there ? (E)(o[j][d][4 * i + e] * f) : (E)0.f;
        *reinterpret_cast<v4*>(dst + 32 * d + 8 * i) = r;
      }
  }
}

// Join the grid splits of a row: a workgroup per row that has them, whose wavefronts take every
// fourth part; a lane has D / 64 of the values.
constexpr int kJoinWaves = 4;
template <typename E, int D>
__global__ void __launch_bounds__(64 * kJoinWaves) cross_attn_join_kernel(const CrossParams p) {
  constexpr int N = D / 64;
  typedef float fn __attribute__((ext_vector_type(N)));
  __shared__ fn part[kJoinWaves][64];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = blockIdx.x / p.rest;
  const int at = blockIdx.x - bh * p.rest, row = p.first + at;
  const int b = bh / p.Hk, hk = bh - b * p.Hk;
  const int head = hk * p.G + row % p.G, query = row / p.G;
  bool there = p.lens == nullptr || p.lens[b] > 0;
  if (p.q_lens != nullptr) there = there && query < p.q_lens[b];

  // Lane s < splits holds the statistics of part s (kMaxGridSplits <= 64).
  float4 ml = make_float4(kFloorMax, 0.f, 0.f, 0.f);
  if (lane < p.splits) ml = p.part_ml[((int64_t)bh * p.splits + lane) * p.rest + at];
  const float* src = p.part_o + ((int64_t)bh * p.splits * p.rest + at) * D + N * lane;
  float top = ml.x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float f = fast_exp2(ml.x - top);
  const float sum = sidon::wave_sum(ml.y * f), raw = sidon::wave_sum(ml.z * f);
  const float weight = there ? f / sum : 0.f;
  // Four parts of a wavefront at a time, their loads together.  (A part without keys
  // holds zeros and weighs nothing.)
  constexpr int kAtOnce = 4;
  fn x = {};
  for (int s0 = w; s0 < p.splits; s0 += kAtOnce * kJoinWaves) {
    fn u[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      u[i] = *reinterpret_cast<const fn*>(src + (int64_t)min(s0 + i * kJoinWaves, p.splits - 1) * p.rest * D);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int s = s0 + i * kJoinWaves;
      if (s < p.splits) x += u[i] * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), s));
    }
  }
  part[w][lane] = x;
  __syncthreads();
  if (w != 0) return;
#pragma unroll
  for (int i = 1; i < kJoinWaves; ++i) x += part[i][lane];
  if (p.lse != nullptr && lane == 0)
    p.lse[((int64_t)b * p.H + head) * p.L + query] = there ? (top + __log2f(raw)) * kLn2 : -INFINITY;
  E* dst = static_cast<E*>(p.out) + b * p.ob + head * p.oh + query * p.ol + N * lane;
  typedef E en __attribute__((ext_vector_type(N)));
  en r;
#pragma unroll
  for (int e = 0; e < N; ++e) r[e] = there ? (E)x[e] : (E)0.f;
  *reinterpret_cast<en*>(dst) = r;
}

// ---- host -------------------------------------------------------------------------

// The kernels.
struct Kind {
  int dim, rows, groups;   // rows and key groups of a workgroup
  bool fine;
  int fit;                 // workgroups that a CU runs at once
  double base, ends, alone, more, join, part, traffic;
  double cut, cut_round;   // of cut row blocks (0: none of this kernel's)
};
// Which, and how many grid splits: the least estimate (us) of
//
//   base + turns (ends + rounds (alone + more running)) + what splits cost
//
// where a CU's share of the workgroups takes full turns of `fit` at once and one with
// the rest, `running` is what a turn holds, and a workgroup's rounds are its steps over
// its key groups.  Splits add a joining launch, its walk over the parts, and the partial
// results, written and read (per MB).  Fitted to 165000 timings of 31600 shapes (1 to 32
// items, 1 to 1400 queries, 30 to 6000 keys, in every kernel and with every number of splits):
// the choice is on average within 1% of the best one's time, in 99 of 100 within 17%.  (32
// rows at D 64 are for short launches: 4 x 16 heads x 224 x 1500 15.6 us, with 64 rows
// 16.8; 1 x 16 x 4800 x 4800 151 and 123.  Rows shared by more wavefronts, 128 and 256 a
// workgroup, took 131 and 144 there: fewer copies, but waits for one another.)
//
// Where one or two workgroups a CU leave a few row blocks over, whose turn would hold few CUs,
// those alone are split, and run beside the others. Their estimate is the others' and
//   cut + cut_round rounds workgroups a CU
// for heads that divide evenly over the XCDs, 40 steps and more and a quarter of a turn at
// most; fitted to 45000 shapes, of which it takes 622, to 0.86 of their time on average and 1.06 at
// worst (2 x 8 heads (2 key heads) x 1037 x 4800, D 128, 260 row blocks on 256 CUs: 78 -> 58 us).
constexpr Kind kKinds[] = {{64, 32, 4, true, 2, 1.53, 4.24, 0, .677, 2.5, .018, .744, 0, 0},
                           {64, 32, 4, false, 2, 2.39, 3.98, .111, .343, 2.62, 0, .601, 0, 0},
                           {64, 64, 4, false, 2, 2.58, 5.72, .05, .637, 2.29, 0, .502, 9, .5},
                           {128, 32, 2, true, 2, 1.24, 5.02, .329, .484, 2.43, .022, .351, 0, 0},
                           {128, 64, 2, false, 2, 1.5, 6, .4, .3, 3.2, 0, .4, 6, .3}};
constexpr int kNumKinds = sizeof(kKinds) / sizeof(kKinds[0]);

struct Plan {
  int kind;   // -1: none yet
  int whole, cut, splits;   // row blocks of a workgroup each, and of `splits` workgroups each
};

Plan search(int B, int Hk, int R, int S, int D, int cus) {
  const int64_t heads = (int64_t)B * Hk;
  const int steps = (S + kStep - 1) / kStep;
  Plan best{-1, 0, 0, 1};
  double best_us = 0;
  for (int i = 0; i < kNumKinds; ++i) {
    const Kind& k = kKinds[i];
    // up to 32 rows keep two summands (the header says so)
    if (k.dim != D || (R <= kBlock && !k.fine) || (R > kBlock && k.fine && D == 64)) continue;
    const int blocks = (R + k.rows - 1) / k.rows;
    const auto turns = [&](int64_t load, int rounds) {
      const int64_t full = load / k.fit, rest = load % k.fit;
      double us = (double)full * (k.ends + rounds * (k.alone + k.more * k.fit));
      if (rest > 0) us += k.ends + rounds * (k.alone + k.more * (double)rest);
      return us;
    };
    for (const int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, kMaxGridSplits}) {
      const int64_t load = (heads * blocks * s + cus - 1) / cus;   // workgroups of the busiest CU
      if (s > 1 && (s * k.groups > steps + 1 || load > 6)) break;
      const int rounds = (steps + k.groups * s - 1) / (k.groups * s);
      double us = k.base + turns(load, rounds);
      if (s > 1) us += k.join + k.part * s + (double)heads * R * s * D * 8e-6 * k.traffic;
      if (best.kind < 0 || us < best_us) best = s > 1 ? Plan{i, 0, blocks, s} : Plan{i, blocks, 0, 1}, best_us = us;
    }
    if (k.cut == 0 || steps < 40 || (heads % 8 != 0 && 8 % heads != 0)) continue;
    for (int load = 1; load <= k.fit; ++load) {
      const int whole = (int)(load * (int64_t)cus / heads), cut = blocks - whole;
      if (whole < 1 || cut < 1 || 4 * heads * cut > cus) continue;
      for (const int s : {4, 8, 16}) {
        const int64_t more = (heads * cut * s + cus - 1) / cus;
        if (more > k.fit) break;
        const int rounds = (steps + k.groups * s - 1) / (k.groups * s);
        const double us = k.base + turns(load, (steps + k.groups - 1) / k.groups) + k.cut + k.cut_round * rounds * (double)more;
        if (us < best_us) best = Plan{i, whole, cut, s}, best_us = us;
      }
    }
  }
  return best;
}

// The search once per shape: one table per thread, the newest shape kept.
Plan plan(int B, int Hk, int R, int S, int D, int cus) {
  struct Entry {
    int B, Hk, R, S, D, cus;
    Plan plan;
  };
  constexpr unsigned kEntries = 16;
  static thread_local Entry table[kEntries] = {};
  const unsigned hash = ((unsigned)S * 2654435761u ^ (unsigned)R * 40503u ^ (unsigned)B * 97u) >> 9;
  Entry& e = table[hash % kEntries];
  if (e.B != B || e.Hk != Hk || e.R != R || e.S != S || e.D != D || e.cus != cus)
    e = Entry{B, Hk, R, S, D, cus, search(B, Hk, R, S, D, cus)};
  return e.plan;
}

bool shape_ok(int B, int H, int Hk, int L, int S, int D) {
  return B >= 1 && H >= 1 && Hk >= 1 && H % Hk == 0 && L >= 1 && S >= 1 && (D == 64 || D == 128) &&
         S <= (1 << 30) && (int64_t)(H / Hk) * L <= (1 << 24) && (int64_t)B * Hk <= (1 << 24);
}

size_t part_bytes(int B, int Hk, int R, int D, const Plan& c) {
  if (c.splits == 1) return 0;
  return (size_t)B * Hk * (R - c.whole * kKinds[c.kind].rows) * c.splits * (16 + (size_t)D * 4);
}

template <typename E, int D, int NB, int RB, int KS, bool kFine, int kMinWaves>
void launch_kind(const CrossParams& p, hipStream_t stream) {
  const dim3 grid(p.deal.groups()), block(64 * RB * KS);
  if constexpr (kFine) {
    hipLaunchKernelGGL((cross_attn_kernel<E, D, NB, RB, KS, true, false, kMinWaves>), grid, block, 0, stream, p);
  } else if (p.lse != nullptr) {
    hipLaunchKernelGGL((cross_attn_kernel<E, D, NB, RB, KS, false, true, kMinWaves>), grid, block, 0, stream, p);
  } else {
    hipLaunchKernelGGL((cross_attn_kernel<E, D, NB, RB, KS, false, false, kMinWaves>), grid, block, 0, stream, p);
  }
}

template <typename E>
void launch(const CrossParams& p, int kind, int D, hipStream_t stream) {
  switch (kind) {   // kKinds
    case 0: launch_kind<E, 64, 1, 1, 4, true, 2>(p, stream); break;
    case 1: launch_kind<E, 64, 1, 1, 4, false, 2>(p, stream); break;
    case 2: launch_kind<E, 64, 2, 1, 4, false, 2>(p, stream); break;
    case 3: launch_kind<E, 128, 1, 1, 2, true, 1>(p, stream); break;
    default: launch_kind<E, 128, 1, 2, 2, false, 2>(p, stream); break;
  }
  if (p.splits > 1) {
    const dim3 join((unsigned)((int64_t)p.B * p.Hk * p.rest));
    if (D == 64) {
      hipLaunchKernelGGL((cross_attn_join_kernel<E, 64>), join, dim3(64 * kJoinWaves), 0, stream, p);
    } else {
      hipLaunchKernelGGL((cross_attn_join_kernel<E, 128>), join, dim3(64 * kJoinWaves), 0, stream, p);
    }
  }
}

}  // namespace

SIDON_API size_t sidon_cross_attention_workspace_bytes(int B, int H, int Hk, int L, int S, int D) {
  if (!shape_ok(B, H, Hk, L, S, D)) return 0;
  const int R = H / Hk * L;
  return part_bytes(B, Hk, R, D, plan(B, Hk, R, S, D, sidon::compute_units()));
}

SIDON_API int sidon_cross_attention(const void* q, const void* k, const void* v, const int32_t* lens,
                                    const int32_t* q_lens, float scale, void* out, float* lse, void* ws,
                                    size_t ws_bytes, int B, int H, int Hk, int L, int S, int D, int dtype,
                                    const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                    const int64_t* o_strides, sidon_stream_t stream) {
  using sidon::fail;
  using sidon::Rows;
  sidon::clear_error();
  if (!q || !k || !v || !out || !q_strides || !k_strides || !v_strides || !o_strides)
    return fail(SIDON_E_NULL, "q, k, v, out and the strides must be non-NULL");
  if (dtype != SIDON_FP16 && dtype != SIDON_BF16) return fail(SIDON_E_SHAPE, "dtype=%d is neither SIDON_FP16 nor SIDON_BF16", dtype);
  if (!shape_ok(B, H, Hk, L, S, D))
    return fail(SIDON_E_SHAPE, "B=%d H=%d Hk=%d L=%d S=%d D=%d: need sizes >= 1, H a multiple of Hk, D 64 or 128, H / Hk * L and B * Hk <= 2^24, S <= 2^30",
                B, H, Hk, L, S, D);
  if (!(scale >= FLT_MIN && scale <= 0x1p100f)) return fail(SIDON_E_SHAPE, "scale=%g must be positive and at most 2^100", scale);
  const struct {
    const char* name;
    const void* at;
    const int64_t* s;
    int heads, len;
    int64_t row_most;
  } all[] = {{"q", q, q_strides, H, L, int64_t(1) << 40}, {"k", k, k_strides, Hk, S, (int64_t(1) << 25) - 1},
             {"v", v, v_strides, Hk, S, (int64_t(1) << 25) - 1}, {"out", out, o_strides, H, L, int64_t(1) << 40}};
  Rows rows[4];
  const __int128 most = (__int128)1 << 61;
  for (int t = 0; t < 4; ++t) {
    for (int i = 0; i < 3; ++i)
      if (all[t].s[i] < 0 || all[t].s[i] % 8 != 0 || all[t].s[i] > (i == 2 ? all[t].row_most : int64_t(1) << 40))
        return fail(SIDON_E_STRIDE, "%s stride %lld (number %d) must be a multiple of 8 in [0, %s]", all[t].name,
                    (long long)all[t].s[i], i, i == 2 && all[t].row_most < (int64_t(1) << 40) ? "2^25)" : "2^40]");
    if (!sidon::aligned16(all[t].at)) return fail(SIDON_E_ALIGN, "%s must be 16-byte aligned", all[t].name);
    rows[t] = Rows{all[t].at, {B, all[t].heads, all[t].len}, {all[t].s[0], all[t].s[1], all[t].s[2]}, D, 2};
    if (rows[t].bytes() > most) return fail(SIDON_E_STRIDE, "%s spans more than the address space", all[t].name);
  }
  if (((reinterpret_cast<uintptr_t>(lens) | reinterpret_cast<uintptr_t>(q_lens) | reinterpret_cast<uintptr_t>(lse)) & 3u) != 0 ||
      !sidon::aligned16(ws))
    return fail(SIDON_E_ALIGN, "lens, q_lens and lse must be 4-byte aligned, ws 16-byte aligned");
  if (!sidon::apart(rows[3].n, rows[3].st, 3, D)) return fail(SIDON_E_STRIDE, "rows of out overlap one another");
  const int R = H / Hk * L;
  const Plan c = plan(B, Hk, R, S, D, sidon::compute_units());
  const size_t need = part_bytes(B, Hk, R, D, c);
  if (ws_bytes < need || (need > 0 && ws == nullptr))
    return fail(SIDON_E_SHAPE, "ws holds %zu bytes, the call needs %zu", ws_bytes, need);
  // Workgroups read the inputs while others already write out, lse, or ws.
  {
    for (int t = 0; t < 3; ++t)
      if (sidon::tensors_meet(rows[t], rows[3])) return fail(SIDON_E_SHAPE, "out must lie apart from %s", all[t].name);
    const struct {
      const char* name;
      const void* at;
      int64_t bytes;
      bool written;
    } flat[] = {{"lens", lens, lens ? (int64_t)4 * B : 0, false},
                {"q_lens", q_lens, q_lens ? (int64_t)4 * B : 0, false},
                {"lse", lse, lse ? (int64_t)4 * B * H * L : 0, true},
                {"ws", ws, (int64_t)need, true}};
    for (int i = 0; i < 4; ++i) {
      if (flat[i].bytes == 0) continue;
      for (int t = flat[i].written ? 0 : 3; t < 4; ++t)
        if (sidon::ranges_meet(flat[i].at, flat[i].bytes, rows[t].at, (int64_t)rows[t].bytes()))
          return fail(SIDON_E_SHAPE, "%s must lie apart from %s", flat[i].name, all[t].name);
      for (int j = 0; j < i; ++j)
        if (flat[j].bytes > 0 && (flat[i].written || flat[j].written) &&
            sidon::ranges_meet(flat[i].at, flat[i].bytes, flat[j].at, flat[j].bytes))
          return fail(SIDON_E_SHAPE, "%s must lie apart from %s", flat[i].name, flat[j].name);
    }
  }
  const int64_t heads = (int64_t)B * Hk, units = c.whole + (int64_t)c.cut * c.splits;
  if (!deal_fits(heads, units) || (c.splits > 1 && heads * R > INT32_MAX / 256))
    return fail(SIDON_E_SHAPE, "too many rows for one launch");
  const int rc = sidon::check_device();
  if (rc) return rc;
  CrossParams p{};
  p.q = q, p.k = k, p.v = v, p.out = out, p.lse = lse, p.lens = lens, p.q_lens = q_lens;
  p.part_ml = static_cast<float4*>(ws);
  p.whole = c.whole, p.cut = c.cut, p.splits = c.splits;
  p.first = c.whole * kKinds[c.kind].rows, p.rest = c.cut > 0 ? R - p.first : 0;
  p.part_o = static_cast<float*>(ws) + (size_t)B * Hk * p.rest * c.splits * 4;
  p.qb = q_strides[0], p.qh = q_strides[1], p.ql = q_strides[2];
  p.kb = k_strides[0], p.kh = k_strides[1], p.kl = (int)k_strides[2];
  p.vb = v_strides[0], p.vh = v_strides[1], p.vl = (int)v_strides[2];
  p.ob = o_strides[0], p.oh = o_strides[1], p.ol = o_strides[2];
  p.B = B, p.H = H, p.Hk = Hk, p.G = H / Hk, p.L = L, p.S = S, p.R = R;
  p.deal = deal(heads, units, (int64_t)S * D * 4);
  p.scale = (float)(1.4426950408889634 * scale);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SIDON_FP16) {
    launch<_Float16>(p, c.kind, D, s);
  } else {
    launch<__bf16>(p, c.kind, D, s);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(SIDON_E_LAUNCH, "cross attention launch failed: %s", hipGetErrorString(err));
  return SIDON_OK;
}
