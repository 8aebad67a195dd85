// diff_attn.hip -- differential attention (MI355X / gfx950): the difference of
// two softmax maps over one set of values, with a learned weight,
//
//   o_i = sum_j softmax_j(q1_i . k1_j / sqrt D) v_j - lambda sum_j softmax_j(q2_i . k2_j / sqrt D) v_j
//   lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init
//   out_i = o_i,  or  (1 - lambda_init) norm_w o_i / sqrt(mean(o_i^2) + eps)
//
// with head dim D (64 or 128) per map and 2 D values, keys j < lens[b], and
// optionally j <= lens[b] - L + i.  Grouped heads share keys and values: the
// G heads of a group and their L queries are G L rows over one key head, a
// query's heads side by side.
//
// A wavefront owns 32 rows of one map (the accumulators of both would not fit its
// registers beside the operands): S^T = K . Q^T by v_mfma_f32_32x32x16, an online
// softmax with the running maximum raised only when a step's probabilities would
// leave the fp16 range, O^T += V^T . P^T.  Key rows enter the A operand with bits 2
// and 3 of their index swapped, which makes the accumulator, rounded to 16 bits,
// the B operand of the second product; the sums of the rounded probabilities, which
// the result is divided by, come from the matrix core too.  In a round a wavefront
// takes the softmax of one step and the values of the step before, whose vector
// and matrix instructions do not wait for each other.
//
// Keys go by steps of 32: a step's keys of both maps and its values (8 D x 32
// bytes) are copied global -> LDS by global_load_lds_dwordx4, as tiles of 32 rows
// x 128 bytes with swizzled 16-byte chunks; keys are read with ds_read_b128,
// values transposed with ds_read_b64_tr_b16.  The two maps of RB row blocks share a
// ring of two key and three value slots, so the values are read once for both maps;
// KS such groups take every KS-th step and are merged through LDS; over the grid a
// row block's steps can be split again, each part leaving (max, sum, O) of both maps
// in fp32 for a joining launch.
//
// Two forms: 64 rows on one ring, and 32 rows for few (D 64: on two rings of every
// other step, which one workgroup's latency hides; D 128: on one, two workgroups a CU).
// Measured (D 64, fp16 or bf16, whole calls in a graph, on the same operands again and
// again | on others each time, past the 256 MB of the Infinity Cache):
//   1 x 8 heads x 4800 x 4800        170 | 172 us, 834 TFLOP/s (a large matrix product: 1330)
//   3 x 8 heads (2 key heads) x 1037, D 128, ragged, causal   42 | 43 us
//   32 x 16 heads (4 key heads) x 1 x 6000, ragged   42 | 56 us: 3.6 TB/s from memory (a large copy: 5.0)
//   1 x 8 heads x 1 x 4800           10.2 | 14.3 us, two launches
// Prompts are bound by the vector unit's exponentials and roundings beside the
// matrix core (16 exponentials per two 32x32x16 score products and four value
// products), and by whole workgroups: 600 on 256 CUs are three on the busiest.
// The 64-row form at D 128 has more values than its 256 registers hold (88 bytes of
// scratch a lane) and one wavefront on most SIMDs: its rounds wait for one another.
// Single tokens against a large cache wait for memory, whose copies drain at every
// round; against a small one for launches and the first copies' latency.
#include <hip/hip_runtime.h>

#include <float.h>
#include <stdint.h>

#include "attn_device.h"
#include "flexrel_device.h"
#include "sidon_host.h"
#include "sidon_operators.h"
#include "sidon_wave.h"

#define SIDON_API extern "C" __attribute__((visibility("default")))
#define SIDON_INLINE __attribute__((always_inline))

namespace {

using namespace sidon_attn;

constexpr int kBlock = 32;          // rows per wavefront
constexpr int kMaxGridSplits = 64;

struct DiffParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const float* lam;      // [4, D] per head (or shared: lam_h == 0)
  const float* norm_w;   // [2 D] or null
  const int32_t* lens;
  float2* part_ml;       // [B Hk, splits, R, 2] (maximum, sum)
  float* part_o;         // [B Hk, splits, R, 2, 2 D]
  int64_t qb, qh, qm, kb, kh, km, vb, vh, ob, oh;   // strides (elements): batch, head, map
  int64_t ql, ol;        // row strides
  int kl, vl;            // row strides (< 2^25)
  int lam_h;
  int B, H, Hk, G, L, S, R;
  int blocks, splits;
  int parts, parts_per_xcd;   // of a key head, of all of them on an XCD
  int causal;
  float scale;           // log2(e) / sqrt(D)
  float lam_init, eps;
};

// The learned weight of head h, in every lane of a wavefront.
template <int D>
__device__ __forceinline__ float head_lambda(const DiffParams& p, int h, int lane) {
  const float* l = p.lam + (int64_t)h * p.lam_h;
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int d = 0; d < D; d += 64) {
    a = fmaf(l[d + lane], l[D + d + lane], a);
    b = fmaf(l[2 * D + d + lane], l[3 * D + d + lane], b);
  }
  return expf(sidon::wave_sum(a)) - expf(sidon::wave_sum(b)) + p.lam_init;
}

// The same for a wavefront whose rows may be of several heads of its group.
template <int D>
__device__ __forceinline__ float wave_lambda(const DiffParams& p, int hk, int row, int lane) {
  if (p.lam_h == 0) return head_lambda<D>(p, 0, lane);
  float lambda = 0.f;
  for (int j = 0; j < p.G; ++j) {
    const float l = head_lambda<D>(p, hk * p.G + j, lane);
    if (row % p.G == j) lambda = l;
  }
  return lambda;
}

// A workgroup: RB row blocks x 2 maps x KS key groups, a wavefront each.  The
// wavefronts of a key group share a ring of two key slots and three value
// slots, a step of 32 keys each.
template <int D, int RB, int KS>
struct Shape {
  static constexpr int kRingWaves = 2 * RB;
  static constexpr int kWaves = kRingWaves * KS;
  static constexpr int kP = D / 64;                   // 128-byte panels per key map (twice as many for V)
  static constexpr int kSlot = 2 * kP * kTile;        // bytes of a step's keys (both maps), or of its values
  static constexpr int kV = 2 * kSlot;                // value slots behind the key slots
  static constexpr int kRing = 5 * kSlot;
  static constexpr int kDb = 2 * D / 32;              // 32-wide blocks of the values
  static constexpr int kPart = (kDb * 16 + 4) * 64 * 4;   // bytes of a wavefront's partial result
  static constexpr int kMerge = KS > 1 ? KS / 2 * kRingWaves * kPart : 0;
  static constexpr int kCross = RB * kPart;
  static constexpr int kNorm = kCross;                // the norm's weights behind it
  static constexpr int kNeed = kMerge > kCross + 8 * D ? kMerge : kCross + 8 * D;
  static constexpr int kLds = KS * kRing > kNeed ? KS * kRing : kNeed;
  static constexpr int kCopies = kSlot / 1024 / kRingWaves;   // 1 KB copies per wavefront and slot
  static_assert(kLds <= 160 * 1024, "LDS");
  static_assert(kSlot / 1024 % kRingWaves == 0, "an even split of the copies");
};

// kFine: probabilities as two summands of the type, the rounded value and what the
// rounding left, so that only the output is rounded.  For few rows, where memory and
// latency leave the matrix cores idle (32 x 1 against 6000 41.9 us, with single
// probabilities 40.3; 1 x 1 against 4800 11.0 and 10.4).  Prompts round once, as
// flexrel's do: each probability off by half a step of itself, in sum about what
// rounding the output costs; a second summand would be two thirds more matrix work.
template <typename E, int D, int RB, int KS, bool kFine, int kMinWaves>
__global__ void __launch_bounds__(128 * RB * KS, kMinWaves) diff_attn_kernel(const DiffParams p) {
  using C = Shape<D, RB, KS>;
  typedef typename Half<E>::v2 v2;
  typedef typename Half<E>::v4 v4;
  constexpr int P = C::kP, kDb = C::kDb;
  constexpr int kQ = D / 16;          // Q operands
  __shared__ __attribute__((aligned(16))) char smem[C::kLds];

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = w % C::kRingWaves, ks = w / C::kRingWaves;
  const int rb = wr >> 1, map = wr & 1;
  const int n = lane & 31, g = lane >> 5;

  // Workgroups go round-robin over the 8 XCDs.  A key head's (row block, split)
  // units are dealt into `parts` parts and the parts to the XCDs, so that each
  // L2 holds the keys and values of few heads and every XCD gets long and short
  // items, and causal blocks of every length; the longest come first.
  const int xcd = blockIdx.x & 7, at_xcd = blockIdx.x >> 3;
  const int part = at_xcd % p.parts_per_xcd * 8 + xcd;
  const int bh = part / p.parts;
  const int unit = at_xcd / p.parts_per_xcd * p.parts + part % p.parts;
  if (unit >= p.blocks * p.splits) return;
  const int split = unit / p.blocks;
  const int blk = p.blocks - 1 - (unit - split * p.blocks);
  const int b = bh / p.Hk, hk = bh - b * p.Hk;
  const int row0 = (blk * RB + rb) * kBlock;   // of this wavefront
  const int row = row0 + n;                    // of this lane: query row / G, head row % G of the group

  int lk = p.S;
  if (p.lens != nullptr) lk = __builtin_amdgcn_readfirstlane(min(max(p.lens[b], 0), p.S));

  // Keys that this lane's row sees, the fewest that a row of the wavefront
  // does, and the steps that some row of the wavefront, of the workgroup needs.
  int lim, wave_least, wave_steps, steps;
  {
    // (grows with the row; rows past R, never stored, see what the last one does)
    const auto limit = [&](int r) SIDON_INLINE {
      return p.causal ? min(max(lk - p.L + 1 + min(r, p.R - 1) / p.G, 0), lk) : lk;
    };
    lim = limit(row);
    wave_least = limit(row0);
    wave_steps = row0 < p.R ? (limit(row0 + kBlock - 1) + kStep - 1) / kStep : 0;
    steps = (limit((blk + 1) * RB * kBlock - 1) + kStep - 1) / kStep;
  }
  const int t0 = (int)((uint32_t)steps * (uint32_t)split / (uint32_t)p.splits);   // (steps <= 2^25, splits <= 2^6)
  const int t1 = (int)((uint32_t)steps * (uint32_t)(split + 1) / (uint32_t)p.splits);
  const auto mine = [&](int u) SIDON_INLINE { return t0 + u * KS + ks; };   // step u of this group
  const auto until = [&](int t) SIDON_INLINE { return max(t - t0 - ks + KS - 1, 0) / KS; };   // steps u with mine(u) < t
  const int all = (t1 - t0 + KS - 1) / KS;         // most steps of a group: the workgroup's rounds
  const int count = until(min(t1, wave_steps));    // of this wavefront

  // ---- copies into the ring, split over its wavefronts: 1 KB copy i is rows
  // 8 (i % 4) + [0, 8) of panel i / 4 (of the keys: dims 64 (pid % P) of map pid / P;
  // of the values: columns 64 pid) ----
  const uint32_t ring = (uint32_t)(uintptr_t)SIDON_LDS_PTR(char, smem) + ks * C::kRing + wr * C::kCopies * 1024;
  const int pid0 = wr * C::kCopies / 4, crow = wr * C::kCopies % 4 * 8 + (lane >> 3);
  const char* const kbase = static_cast<const char*>(p.k) + 2 * (b * p.kb + hk * p.kh + pid0 / P * p.km) +
                            pid0 % P * 128 - kBack;
  const char* const vbase = static_cast<const char*>(p.v) + 2 * (b * p.vb + hk * p.vh) + pid0 * 128 - kBack;
  const int whole = min(t1, lk / kStep);   // steps below it have all their rows
  // Copy j of a set adds 1024 j to the LDS and to the global address; copies of
  // the next panel (j >= 4) lie 128 bytes on.
  constexpr int kOffs = C::kCopies;
  static_assert(C::kCopies <= 4 || P == 2, "a set is within a panel, or two panels side by side");
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
#pragma unroll
    for (int j = 0; j < C::kCopies; j += 4) {
      if constexpr (C::kCopies >= 4) {
        dma_tile(at + j * 1024, src, off[j], off[j + 1], off[j + 2], off[j + 3]);
      } else {
        static_assert(C::kCopies == 2 || C::kCopies % 4 == 0, "copies go by two or four");
        dma_2k(at, src, off[0], off[1]);
      }
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

  // ---- Q^T operands: lane (n, g) holds query n, dims 16 s + 8 g + [0, 8) ----
  const int rr = min(row, p.R - 1);
  i4 qop[kQ];
  {
    const E* qp = static_cast<const E*>(p.q) + b * p.qb + (hk * p.G + rr % p.G) * p.qh + (rr / p.G) * p.ql + 8 * g +
                  map * p.qm;
#pragma unroll
    for (int s = 0; s < kQ; ++s) qop[s] = *reinterpret_cast<const i4*>(qp + 16 * s);
  }

  // ---- operand offsets from the first key and value slot ----
  int kaddr[4], vaddr[2][2];
  {
    const int krow = mfma_row_perm(n);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      kaddr[i] = ks * C::kRing + map * P * kTile + krow * 128 + (((2 * i + g) ^ tile_swz(krow)) << 4);
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

  // (here, so that its loads overlap the first copies)
  float lambda = 1.f;
  if (p.splits == 1 && map == 1) lambda = wave_lambda<D>(p, hk, rr, lane);

  f32x16 o[kDb];
#pragma unroll
  for (int d = 0; d < kDb; ++d) o[d] = f32x16{};
  float mx = kFloorMax, sum = 0.f;   // maximum of the scaled scores, less kLift, and sum of the probabilities of query n
  f32x16 s;                          // scores of a step: element i is key 16 (i / 8) + 8 g + i % 8
  constexpr int kTerms = kFine ? 2 : 1;
  i4 pk[kTerms][2];                  // its probabilities

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
    f32x16 acc = {};
#pragma unroll
    for (int i = 0; i < kQ; ++i) acc = Half<E>::mfma(kop[i], qop[i], acc);
    s = acc;
  };
  int k0 = mine(0) * kStep;   // first key of the step in s
  const auto hide = [&]() SIDON_INLINE {
    if (k0 + kStep > wave_least) {
      const int left = lim - k0 - 8 * g;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i >> 3) + (i & 7) >= left) s[i] = -INFINITY;
    }
    k0 += KS * kStep;
  };
  const auto exps = [&](float (&e)[16]) SIDON_INLINE {
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = fast_exp2(fmaf(s[i], p.scale, -mx));
  };
  // The step's probabilities, rounded.
  const auto round_to = [&](const float (&e)[16]) SIDON_INLINE {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const v2 hi = __builtin_convertvector(f2{e[i], e[i + 1]}, v2);
      pk[0][i >> 3][(i & 7) >> 1] = __builtin_bit_cast(int, hi);
      if constexpr (kFine) {
        const f2 left = {e[i] - (float)hi[0], e[i + 1] - (float)hi[1]};
        pk[kTerms - 1][i >> 3][(i & 7) >> 1] = __builtin_bit_cast(int, __builtin_convertvector(left, v2));
      }
    }
  };
  // Their sum, on the matrix core, where the vector unit is the busier one.  Read
  // as a 16x16x32 B operand, a lane's half of them holds query c + 16 (j % 2) of
  // lane c + 16 j, keys 8 (j / 2) + [0, 8); the A operand is 1 where bit 4 of the
  // lane equals bit 2, so that the four rows a lane receives are its own query's
  // sum.  The other query of the column enters times 0: where its probabilities are
  // infinite or NaN, so is this sum, and `settle` takes the query's own.
  const auto matrix_sum = [&]() SIDON_INLINE {
    f4 total = {};
#pragma unroll
    for (int k = 0; k < kTerms; ++k) {
      total = Half<E>::small(sel, pk[k][0], total);
      total = Half<E>::small(sel, pk[k][1], total);
    }
    return total[0];
  };
  // The same from the lane pair that holds the query, nothing else.
  const auto own_sum = [&]() SIDON_INLINE {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < kTerms; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = pk[k][i >> 2][i & 3];   // (a bit cast of the element itself takes the vector's first)
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
        for (int k = 0; k < kTerms; ++k) o[d] = Half<E>::mfma(i4{lo[0], lo[1], hi[0], hi[1]}, pk[k][hh], o[d]);
      }
    vread = vread == 2 * C::kSlot ? 0 : vread + C::kSlot;
  };
  // Raises the running maximum of the queries whose probabilities do not all
  // fit, with what they have so far, and takes their sums apart from the other
  // queries'.  (The condition is a lane's, not the
  // wavefront's: behind a branch of the wavefront the compiler keeps the
  // accumulators in two places.)
  const auto settle = [&](float total) SIDON_INLINE {
    // One that left fp16 is an infinity in the sum.
    if (!(total < kSumLimit)) {
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
      top = fmaxf(mx, pair_max(top) * p.scale - Half<E>::kLift);
      const float alpha = fast_exp2(mx - top);   // 0 from kFloorMax
#pragma unroll
      for (int d = 0; d < kDb; ++d) o[d] *= alpha;
      sum *= alpha;
      mx = top;
      float e[16];
      exps(e);
      round_to(e);
      total = own_sum();
    }
    sum += total;
  };
  // Behind it, what the last round copied (the keys of step u + 1, the values
  // of step u) is there for every wavefront of the ring, and nobody reads the
  // keys of step u or the values of step u - 2 any more: their slots are filled
  // with the keys of step u + 2 and the values of step u + 1.
  const auto round = [&]() SIDON_INLINE {
    wait_vmcnt<0>();
    lds_barrier();
    copy_k();
    copy_v();
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
    round();
    if (count > 0) {
      hide();
      float e[16];
      exps(e);
      round_to(e);
      settle(matrix_sum());
      if (count > 1) {
        load_keys();
        scores();
      }
    }
    for (u = 1; u < count; ++u) {
      round();
      hide();
      float e[16];
      exps(e);
      values();
      round_to(e);
      const float total = matrix_sum();
      load_keys();   // (of the last round: what an earlier step left in the slot, for nothing)
      settle(total);
      scores();
    }
    for (; u <= all; ++u) {
      round();
      if (u == count && count > 0) values();
    }
  }

  // A wavefront's partial result in LDS, lane by lane: its values, then (maximum, sum).
  float* const mem = reinterpret_cast<float*>(smem) + lane * 4;
  const auto put = [&](float* at, int d, int i, float by) SIDON_INLINE {
    *reinterpret_cast<f4*>(at + (d * 4 + i) * 256) =
        f4{o[d][4 * i] * by, o[d][4 * i + 1] * by, o[d][4 * i + 2] * by, o[d][4 * i + 3] * by};
  };
  const auto get = [&](const float* at, int d, int i) SIDON_INLINE {
    return *reinterpret_cast<const f4*>(at + (d * 4 + i) * 256);
  };

  // ---- merge the key groups, half of them into the other half at a time ----
  if constexpr (KS > 1) {
#pragma unroll
    for (int half = KS / 2; half >= 1; half >>= 1) {
      wait_vmcnt<0>();
      lds_barrier();   // the rings, or the last round's values, are done with
      float* at = mem + ((ks % half) * C::kRingWaves + wr) * (C::kPart / 4);
      float* ml = at + kDb * 4 * 256;
      if (ks >= half) {
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) put(at, d, i, 1.f);
        ml[0] = mx;
        ml[1] = sum;
      }
      lds_barrier();
      if (ks >= half) return;
      const float top = fmaxf(mx, ml[0]);
      const float fa = fast_exp2(mx - top), fb = fast_exp2(ml[0] - top);
      mx = top;
      sum = sum * fa + ml[1] * fb;
#pragma unroll
      for (int d = 0; d < kDb; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f4 v = get(at, d, i);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][4 * i + e] = o[d][4 * i + e] * fa + v[e] * fb;
        }
        if (d % 2 == 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // Lane (n, g) holds of row n the values 32 d + 8 i + 4 g + [0, 4).
  if (p.splits > 1) {
    if (row >= p.R) return;
    const int64_t at = ((int64_t)bh * p.splits + split) * p.R + row;
    float* dst = p.part_o + at * (4 * D) + map * 2 * D + 4 * g;
    if (g == 0) p.part_ml[at * 2 + map] = make_float2(mx, sum);
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f4*>(dst + 32 * d + 8 * i) = f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    return;
  }

  // What this map's accumulators weigh in the difference (0 where no key was seen).
  float f = sum == 0.f ? 0.f : 1.f / sum;
  float* const at = mem + rb * (C::kPart / 4);
  // The norm's weights through LDS: a lane needs 2 D / 2 of them, whose loads from
  // memory would wait for each other (the registers are full).
  float* const nw = reinterpret_cast<float*>(smem + C::kNorm);
  constexpr int kThreads = 64 * C::kRingWaves, kNw = (2 * D + kThreads - 1) / kThreads;
  float mine_w[kNw];
  const int tid = wr * 64 + lane;
#pragma unroll
  for (int i = 0; i < kNw; ++i) {
    const int c = tid + i * kThreads;
    mine_w[i] = p.norm_w != nullptr && c < 2 * D ? p.norm_w[c] : 1.f;
  }
  lds_barrier();   // the ring, or the merge, is done with
#pragma unroll
  for (int i = 0; i < kNw; ++i)
    if (tid + i * kThreads < 2 * D) nw[tid + i * kThreads] = mine_w[i];
  if (map == 1) {
    f *= lambda;
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) put(at, d, i, f);
  }
  lds_barrier();
  if (map == 1) return;
  float sq = 0.f;
#pragma unroll
  for (int d = 0; d < kDb; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f4 v = get(at, d, i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = o[d][4 * i + e] * f - v[e];
        o[d][4 * i + e] = x;
        sq = fmaf(x, x, sq);
      }
      if (i == 3) __builtin_amdgcn_sched_barrier(0);   // (few loads at a time: the registers are full)
    }
  float gain = 1.f;
  if (p.norm_w != nullptr) gain = (1.f - p.lam_init) * rsqrtf(pair_sum(sq) * (1.f / (2 * D)) + p.eps);
  if (row >= p.R) return;
  E* dst = static_cast<E*>(p.out) + b * p.ob + (hk * p.G + row % p.G) * p.oh + (row / p.G) * p.ol + 4 * g;
#pragma unroll
  for (int d = 0; d < kDb; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f4 wv = *reinterpret_cast<const f4*>(nw + 32 * d + 8 * i + 4 * g);
      v4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = (E)(o[d][4 * i + e] * gain * wv[e]);
      *reinterpret_cast<v4*>(dst + 32 * d + 8 * i) = r;
      if (i == 3) __builtin_amdgcn_sched_barrier(0);
    }
}

// Join the grid splits of a row: a workgroup per row, whose wavefronts take every
// fourth part; a lane has 2 D / 64 of the values.
constexpr int kJoinWaves = 4;
template <typename E, int D>
__global__ void __launch_bounds__(64 * kJoinWaves) diff_attn_join_kernel(const DiffParams p) {
  constexpr int N = 2 * D / 64;
  typedef float fn __attribute__((ext_vector_type(N)));
  __shared__ fn part[kJoinWaves][64];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = blockIdx.x / p.R;
  const int row = blockIdx.x - bh * p.R;
  const int b = bh / p.Hk, hk = bh - b * p.Hk;
  const int head = hk * p.G + row % p.G;

  // Lane s < splits holds the statistics of part s (kMaxGridSplits <= 64).
  float4 ml = make_float4(kFloorMax, 0.f, kFloorMax, 0.f);
  if (lane < p.splits)
    ml = *reinterpret_cast<const float4*>(p.part_ml + (((int64_t)bh * p.splits + lane) * p.R + row) * 2);
  const float* src = p.part_o + ((int64_t)bh * p.splits * p.R + row) * (4 * D) + N * lane;
  const float lambda = head_lambda<D>(p, head, lane);
  float m1 = ml.x, m2 = ml.z;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    m1 = fmaxf(m1, __shfl_xor(m1, d));
    m2 = fmaxf(m2, __shfl_xor(m2, d));
  }
  const float f1 = fast_exp2(ml.x - m1), f2 = fast_exp2(ml.z - m2);
  const float s1 = sidon::wave_sum(ml.y * f1), s2 = sidon::wave_sum(ml.w * f2);
  // What each part weighs in the difference.
  const float w1 = s1 == 0.f ? 0.f : f1 / s1, w2 = s2 == 0.f ? 0.f : f2 / s2 * lambda;
  // Four parts of a wavefront at a time, their loads together.  (A part without keys
  // holds zeros and weighs nothing.)
  constexpr int kAtOnce = 4;
  fn x = {};
  for (int s0 = w; s0 < p.splits; s0 += kAtOnce * kJoinWaves) {
    fn u[kAtOnce], v[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float* at = src + (int64_t)min(s0 + i * kJoinWaves, p.splits - 1) * p.R * (4 * D);
      u[i] = *reinterpret_cast<const fn*>(at);
      v[i] = *reinterpret_cast<const fn*>(at + 2 * D);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int s = s0 + i * kJoinWaves;
      if (s < p.splits) {
        const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w1), s));
        const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w2), s));
        x += u[i] * a - v[i] * c;
      }
    }
  }
  part[w][lane] = x;
  __syncthreads();
  if (w != 0) return;
#pragma unroll
  for (int i = 1; i < kJoinWaves; ++i) x += part[i][lane];
  fn nw;
#pragma unroll
  for (int e = 0; e < N; ++e) nw[e] = p.norm_w != nullptr ? p.norm_w[N * lane + e] : 1.f;
  float gain = 1.f;
  if (p.norm_w != nullptr) {
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) sq = fmaf(x[e], x[e], sq);
    gain = (1.f - p.lam_init) * rsqrtf(sidon::wave_sum(sq) * (1.f / (2 * D)) + p.eps);
  }
  E* dst = static_cast<E*>(p.out) + b * p.ob + head * p.oh + (row / p.G) * p.ol + N * lane;
  typedef E en __attribute__((ext_vector_type(N)));
  en r;
#pragma unroll
  for (int e = 0; e < N; ++e) r[e] = (E)(x[e] * gain * nw[e]);
  *reinterpret_cast<en*>(dst) = r;
}

// ---- host -------------------------------------------------------------------------

struct Plan {
  int rows;     // per workgroup
  int blocks, splits;
};

// Rows per workgroup and grid splits: the least estimate (us) of
//
//   turns (ends + rounds (alone + more running)) + what a split costs
//
// where a CU runs up to `fit` workgroups at once, so that its share of them takes
// full turns and one with the rest, `running` is what a turn holds, and a workgroup's
// rounds are its steps over its key groups.  A split adds the joining launch, its walk
// over the parts, and the partial results, written and read.  (A launch's own
// share is the same for every choice.)  Constants fitted to 7700 shapes of 1 to
// 32 items, 1 to 5000 queries and 32 to 8000 keys, each timed in every choice, causal
// ones too, whose blocks differ: on average within 1% of the best choice, 24% at
// most.  (Counting every turn as full, and splits at half their cost, it was 7%,
// twice the best at worst.)  A single block of rows takes the 32-row form, whose
// probabilities keep two summands: 2 to 4% over the other's time at its best.
Plan search(int B, int Hk, int R, int S, int D, int cus) {
  static const struct {
    int dim, rows, groups, fit;
    double ends, alone, more, join, part, bytes;   // bytes: per us of the partial results' traffic
  } kinds[] = {{64, 32, 2, 2, 2.7, 0.2, 0.47, 2.0, 0.05, 2.64e6},
               {64, 64, 1, 3, 2.4, 0.275, 0.15, 2.0, 0.05, 2.64e6},
               {128, 32, 1, 2, 4.05, 0.32, 0.83, 1.75, 0.04, 4.6e6},
               {128, 64, 1, 2, 6.5, 0.57, 0.24, 1.75, 0.04, 4.6e6}};
  const int64_t heads = (int64_t)B * Hk;
  const int steps = (S + kStep - 1) / kStep;
  Plan best{};
  double best_us = 0;
  for (const auto& k : kinds) {
    if (k.dim != D || (R <= kBlock && k.rows != kBlock)) continue;
    const int blocks = (R + k.rows - 1) / k.rows;
    for (const int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, kMaxGridSplits}) {
      const int64_t load = (heads * blocks * s + cus - 1) / cus;   // workgroups of the busiest CU
      if (s > 1 && (s * k.groups > steps || load > 6)) break;
      const int rounds = (steps + k.groups * s - 1) / (k.groups * s);
      const int64_t full = load / k.fit, rest = load % k.fit;
      double us = (double)full * (k.ends + rounds * (k.alone + k.more * k.fit));
      if (rest > 0) us += k.ends + rounds * (k.alone + k.more * (double)rest);
      if (s > 1) us += k.join + k.part * s + (double)heads * R * s * (4 * D) * 8 / k.bytes;
      if (best.rows == 0 || us < best_us) best = Plan{k.rows, blocks, s}, best_us = us;
    }
  }
  return best;
}

// The search (a few microseconds) once per shape: one table per thread, the
// newest shape kept.
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

size_t part_bytes(int B, int Hk, int R, int D, int splits) {
  return splits > 1 ? (size_t)B * Hk * R * splits * (16 + (size_t)D * 16) : 0;
}

template <typename E>
void launch(const DiffParams& p, int D, int rows, hipStream_t stream) {
  const dim3 grid((unsigned)(8 * p.parts_per_xcd * ((p.blocks * p.splits + p.parts - 1) / p.parts)));
  if (D == 64) {
    if (rows == kBlock) {
      hipLaunchKernelGGL((diff_attn_kernel<E, 64, 1, 2, true, 2>), grid, dim3(256), 0, stream, p);
    } else {
      hipLaunchKernelGGL((diff_attn_kernel<E, 64, 2, 1, false, 3>), grid, dim3(256), 0, stream, p);
    }
  } else {
    if (rows == kBlock) {
      hipLaunchKernelGGL((diff_attn_kernel<E, 128, 1, 1, true, 1>), grid, dim3(128), 0, stream, p);
    } else {
      hipLaunchKernelGGL((diff_attn_kernel<E, 128, 2, 1, false, 2>), grid, dim3(256), 0, stream, p);
    }
  }
  if (p.splits > 1) {
    const dim3 join((unsigned)((int64_t)p.B * p.Hk * p.R));
    if (D == 64) {
      hipLaunchKernelGGL((diff_attn_join_kernel<E, 64>), join, dim3(64 * kJoinWaves), 0, stream, p);
    } else {
      hipLaunchKernelGGL((diff_attn_join_kernel<E, 128>), join, dim3(64 * kJoinWaves), 0, stream, p);
    }
  }
}

}  // namespace

SIDON_API size_t sidon_diff_attention_workspace_bytes(int B, int H, int Hk, int L, int S, int D) {
  if (!shape_ok(B, H, Hk, L, S, D)) return 0;
  const int R = H / Hk * L;
  return part_bytes(B, Hk, R, D, plan(B, Hk, R, S, D, sidon::compute_units()).splits);
}

SIDON_API int sidon_diff_attention(const void* q, const void* k, const void* v, const float* lam, int lam_heads,
                                   float lam_init, const int32_t* lens, const float* norm_w, float eps, void* out,
                                   void* ws, size_t ws_bytes, int B, int H, int Hk, int L, int S, int D, int causal,
                                   int dtype, const int64_t* q_strides, const int64_t* k_strides,
                                   const int64_t* v_strides, const int64_t* o_strides, sidon_stream_t stream) {
  using sidon::fail;
  sidon::clear_error();
  if (!q || !k || !v || !lam || !out || !q_strides || !k_strides || !v_strides || !o_strides)
    return fail(SIDON_E_NULL, "q, k, v, lam, out and the strides must be non-NULL");
  if (dtype != SIDON_FP16 && dtype != SIDON_BF16) return fail(SIDON_E_SHAPE, "dtype=%d is neither SIDON_FP16 nor SIDON_BF16", dtype);
  if (!shape_ok(B, H, Hk, L, S, D))
    return fail(SIDON_E_SHAPE, "B=%d H=%d Hk=%d L=%d S=%d D=%d: need sizes >= 1, H a multiple of Hk, D 64 or 128, H / Hk * L and B * Hk <= 2^24, S <= 2^30",
                B, H, Hk, L, S, D);
  if (lam_heads != 1 && lam_heads != H) return fail(SIDON_E_SHAPE, "lam_heads=%d must be 1 or H=%d", lam_heads, H);
  // Strides in the order (batch, head, map, row) for q and k, (batch, head, row) for v and out.
  const struct {
    const char* name;
    const int64_t* s;
    int n;
    int64_t row_most;
  } all[] = {{"q", q_strides, 4, int64_t(1) << 40}, {"k", k_strides, 4, (int64_t(1) << 25) - 1},
             {"v", v_strides, 3, (int64_t(1) << 25) - 1}, {"out", o_strides, 3, int64_t(1) << 40}};
  for (const auto& t : all) {
    for (int i = 0; i < t.n; ++i)
      if (t.s[i] < 0 || t.s[i] % 8 != 0 || t.s[i] > (i == t.n - 1 ? t.row_most : int64_t(1) << 40))
        return fail(SIDON_E_STRIDE, "%s stride %lld (number %d) must be a multiple of 8 in [0, %s]", t.name,
                    (long long)t.s[i], i, i == t.n - 1 && t.row_most < (int64_t(1) << 40) ? "2^25)" : "2^40]");
  }
  if (!sidon::aligned16(q) || !sidon::aligned16(k) || !sidon::aligned16(v) || !sidon::aligned16(out) ||
      (norm_w && !sidon::aligned16(norm_w)) || (reinterpret_cast<uintptr_t>(lam) & 3u) != 0 ||
      (reinterpret_cast<uintptr_t>(lens) & 3u) != 0 || !sidon::aligned16(ws))
    return fail(SIDON_E_ALIGN, "q, k, v, out, norm_w and ws must be 16-byte aligned, lam and lens 4-byte aligned");
  if (norm_w && !(eps >= FLT_MIN)) return fail(SIDON_E_SHAPE, "eps=%g must be positive (a query without keys has no mean square)", eps);
  // Workgroups read the inputs while others already write out, or ws.
  struct Range {
    const void* at;
    __int128 bytes;
    const char* name;
  };
  Range in[7];
  {
    const int qn[] = {B, H, 2, L}, kn[] = {B, Hk, 2, S}, vn[] = {B, Hk, S}, on[] = {B, H, L};
    if (!sidon::apart(on, o_strides, 3, 2 * D)) return fail(SIDON_E_STRIDE, "rows of out overlap one another");
    const __int128 most = (__int128)1 << 61, o_span = sidon::span(on, o_strides, 3, 2 * D) * 2;
    in[0] = Range{q, sidon::span(qn, q_strides, 4, D) * 2, "q"};
    in[1] = Range{k, sidon::span(kn, k_strides, 4, D) * 2, "k"};
    in[2] = Range{v, sidon::span(vn, v_strides, 3, 2 * D) * 2, "v"};
    in[3] = Range{lam, (__int128)lam_heads * D * 16, "lam"};
    in[4] = Range{norm_w, norm_w ? D * 8 : 0, "norm_w"};
    in[5] = Range{lens, lens ? (__int128)B * 4 : 0, "lens"};
    in[6] = Range{out, o_span, "out"};
    for (const Range& t : in)
      if (t.bytes > most) return fail(SIDON_E_STRIDE, "a tensor spans more than the address space");
    for (const Range& t : in) {
      if (&t != &in[6] && t.bytes > 0 && sidon::ranges_meet(out, (int64_t)o_span, t.at, (int64_t)t.bytes))
        return fail(SIDON_E_SHAPE, "out must lie apart from %s", t.name);
    }
  }
  int rc;
  if ((rc = sidon::check_device())) return rc;
  const int R = H / Hk * L;
  const Plan c = plan(B, Hk, R, S, D, sidon::compute_units());
  if (ws_bytes < part_bytes(B, Hk, R, D, c.splits) || (c.splits > 1 && ws == nullptr))
    return fail(SIDON_E_SHAPE, "ws holds %zu bytes, the call needs %zu", ws_bytes, part_bytes(B, Hk, R, D, c.splits));
  if (c.splits > 1) {
    for (const Range& t : in)
      if (t.bytes > 0 && sidon::ranges_meet(ws, (int64_t)part_bytes(B, Hk, R, D, c.splits), t.at, (int64_t)t.bytes))
        return fail(SIDON_E_SHAPE, "ws must lie apart from %s", t.name);
  }
  // Parts per key head (DiffParams): enough for whole heads on an XCD where
  // possible, and all 8 where every head's keys and values fit one L2 together.
  const int64_t heads = (int64_t)B * Hk;
  int parts = 8;
  while (parts > 1 && heads * (parts / 2) % 8 == 0 &&
         (heads * S * D * 8 > (int64_t)3 << 20 || parts > c.blocks * c.splits))
    parts /= 2;
  if (heads * parts * (((int64_t)c.blocks * c.splits + parts - 1) / parts) > INT32_MAX / 256 ||
      (c.splits > 1 && heads * R > INT32_MAX / 256))
    return fail(SIDON_E_SHAPE, "too many rows for one launch");
  DiffParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.lam = lam;
  p.norm_w = norm_w;
  p.lens = lens;
  p.part_ml = static_cast<float2*>(ws);
  p.part_o = static_cast<float*>(ws) + (size_t)B * Hk * R * c.splits * 4;
  p.qb = q_strides[0], p.qh = q_strides[1], p.qm = q_strides[2], p.ql = q_strides[3];
  p.kb = k_strides[0], p.kh = k_strides[1], p.km = k_strides[2], p.kl = (int)k_strides[3];
  p.vb = v_strides[0], p.vh = v_strides[1], p.vl = (int)v_strides[2];
  p.ob = o_strides[0], p.oh = o_strides[1], p.ol = o_strides[2];
  p.lam_h = lam_heads == 1 ? 0 : 4 * D;
  p.B = B, p.H = H, p.Hk = Hk, p.G = H / Hk, p.L = L, p.S = S, p.R = R;
  p.blocks = c.blocks, p.splits = c.splits;
  p.parts = parts, p.parts_per_xcd = (int)(heads * parts / 8);
  p.causal = causal != 0;
  p.scale = 1.4426950408889634f / (D == 64 ? 8.f : 11.313708498984761f);
  p.lam_init = lam_init;
  p.eps = eps;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SIDON_FP16) {
    launch<_Float16>(p, D, c.rows, s);
  } else {
    launch<__bf16>(p, D, c.rows, s);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(SIDON_E_LAUNCH, "differential attention launch failed: %s", hipGetErrorString(err));
  return SIDON_OK;
}
