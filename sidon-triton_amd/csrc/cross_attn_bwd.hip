// cross_attn_bwd.hip -- gradients of the attention over states of another length
// (MI355X / gfx950).  With P_ij = exp(scale q_i . k_j - lse_i) from the forward
// call's lse, and delta_i = sum_j P_ij dP_ij (= dout_i . out_i, but for out's rounding):
//
//   dv_j = sum_i P_ij dout_i          dP_ij = dout_i . v_j
//   dS_ij = P_ij (dP_ij - delta_i)    dq_i = scale sum_j dS_ij k_j    dk_j = scale sum_i dS_ij q_i
//
// Two launches.  In the first, wavefronts that own 32 queries each go over the keys for delta: S and dP,
// and the sum of P (dP - dout . out).  In the second some wavefronts own 32 keys each, whose k
// and v stay in their registers as B operands, and go over the queries of the heads that share them:
// S = Q . K^T and dP = dO . V^T by v_mfma_f32_32x32x16, whose accumulators, rounded, are the B
// operands of dV^T += dO^T . P and dK^T += Q^T . dS; others own 32 queries and go over the keys:
// S^T = K . Q^T, dP^T = V . dO^T, dQ^T += K^T . dS^T.  (Nine products, where one pass would do with five
// if delta came from the rounded output and dq were added up across workgroups: here no atomics, so
// the same bits every time.)  The tiles of 32 rows that the wavefronts of a workgroup share are
// copied global -> LDS by global_load_lds_dwordx4 one step ahead, and read as they are and
// transposed.  (Where the second launch spills `4 * lane`, at D 128 but for one block of either
// kind, at D 64 in two blocks of keys by four of queries and, queries first, in four by two of
// bf16, its reload stands between the copies and waits for the ones just issued.)
//
// fp16 holds P times 2^15, and dS times a power of two that keeps it below 2^15: the
// bound |dS_ij| <= 2 |dout_i| |v_j| needs the longest v, and for dk the longest dout,
// of a key head, which the first launch leaves.  bf16 has fp32's exponents.
//
// What bounds it, and what it reached.  16 heads x 4800 x 4800 take 444 us at D 64 (112 of them the first
// launch; the five products at 0.53 PFLOP/s) and 835 at D 128 (212; 0.57).  First launch: a tile's 16 exponentials and 32 other
// vector instructions beside 8 products (16 at D 128).  Second: matrix cores and vector units are each
// busy a third of the time and overlap little, LDS a fifth.  2 x 16 heads x 300 x 1463 takes 44 us: a
// wavefront's longest chains of steps, and some 14 us of launches, first copies and merges.
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

constexpr int kBlock = 32;          // rows of a tile, rows or keys of a wavefront
constexpr float kLog2e = 1.4426950408889634f;

struct BwdParams {
  const void* q;
  const void* k;
  const void* v;
  const void* out;
  const void* dout;
  const float* lse;      // [B, H, L]
  void* dq;
  void* dk;
  void* dv;
  const int32_t* lens;
  const int32_t* q_lens;
  float* stat;           // [B, H, tiles, 2, 32]: kLift less lse in powers of two (-infinite: no such row), -delta
  float* length;         // [B, H, tiles, 32]: |dout_i|
  float* longest;        // [B, H, tiles]: of a tile
  float* longest_v;      // [B, Hk, key tiles]: |v_j|
  int64_t qb, qh, kb, kh, vb, vh, ob, oh, gb, gh;           // strides (elements): batch, head
  int64_t dqb, dqh, dql, dkb, dkh, dkl, dvb, dvh, dvl, ol;
  int ql, kl, vl, gl;    // row strides (< 2^25)
  int B, H, Hk, G, L, S;
  int tiles, key_tiles;  // of 32 queries, of 32 keys
  Deal keys, queries;    // blocks of keys, of queries of a group's heads
  Deal rows;             // of the first launch
  float scale;
};

template <typename E>
struct Range;   // P and dS are held times 2^kLift and a power of two
template <>
struct Range<_Float16> {
  static constexpr bool kScaled = true;
  static constexpr float kLift = 15.f;
};
template <>
struct Range<__bf16> {
  static constexpr bool kScaled = false;
  static constexpr float kLift = 0.f;
};

// The power of two that keeps numbers up to 2 a b below 1 (1 where there is none).
__device__ __forceinline__ float below_one(float a, float b) {
  const float bound = 2.f * a * b;
  if (!(bound > 0.f && bound < FLT_MAX)) return 1.f;
  return __uint_as_float((253u - (__float_as_uint(bound) >> 23)) << 23);   // 2^-(exponent + 1)
}

__device__ __forceinline__ int valid(const int32_t* lens, int b, int most) {
  return lens == nullptr ? most : __builtin_amdgcn_readfirstlane(min(max(lens[b], 0), most));
}

// Sum over a team of N lanes (8 or 16), in each of them.
template <int N>
__device__ __forceinline__ float team_sum(float v) {
  v += sidon::dpp_mov<0xb1>(v);                          // quad_perm [1, 0, 3, 2]
  v += sidon::dpp_mov<0x4e>(v);                          // quad_perm [2, 3, 0, 1]
  v += sidon::dpp_mov<0x141>(v);                         // row_half_mirror
  if constexpr (N > 8) v += sidon::dpp_mov<0x140>(v);    // row_mirror
  return v;
}

// The largest of `count` numbers, by a wavefront.
__device__ __forceinline__ float largest(const float* at, int count, int lane) {
  float top = 0.f;
  for (int i = lane; i < count; i += 64) top = fmaxf(top, at[i]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  return top;
}

// Copies of tiles of 32 rows x D into LDS, 1 KB copies split over W wavefronts: copy i
// is rows 8 (i % 4) + [0, 8) of panel i / 4 (dims 64 (i / 4)).
template <int D, int W>
struct Copies {
  static constexpr int kBytes = D / 64 * kTile;      // of a tile
  static constexpr int kCount = kBytes / 1024 / W;   // per wavefront
  static_assert(kBytes / 1024 % W == 0 && (kCount <= 2 || kCount % 4 == 0), "an even split of the copies");
  uint32_t off[kCount];
  int crow, lane, stride;
  uint32_t at;   // this wavefront's share of a tile in LDS
  int panel;

  __device__ __forceinline__ uint32_t offset(int j, int r) const {
    return (uint32_t)r * (uint32_t)(2 * stride) + 16u * ((lane & 7) ^ tile_swz(crow + 8 * (j % 4))) + j / 4 * 128u +
           1024u * (3 - j % 4);
  }
  __device__ __forceinline__ void init(int w, int lane_, int stride_) {
    lane = lane_, stride = stride_;
    panel = w * kCount / 4;
    crow = w * kCount % 4 * 8 + (lane >> 3);
    at = w * kCount * 1024;
#pragma unroll
    for (int j = 0; j < kCount; ++j) off[j] = offset(j, crow + 8 * (j % 4));
  }
  // Rows of `src` (the tile's first row) into the tile at LDS address lds; rows from
  // `rows` on read the last one again.
  __device__ __forceinline__ void copy(uint32_t lds, const char* src, int rows) const {
    const char* const base = uniform(src + panel * 128 - kBack);
    uint32_t o[kCount];
#pragma unroll
    for (int j = 0; j < kCount; ++j) o[j] = rows >= kBlock ? off[j] : offset(j, min(crow + 8 * (j % 4), rows - 1));
    if constexpr (kCount % 4 == 0) {
#pragma unroll
      for (int j = 0; j < kCount; j += 4) dma_tile(lds + at + j * 1024, base, o[j], o[j + 1], o[j + 2], o[j + 3]);
    } else if constexpr (kCount == 2) {
      dma_2k(lds + at, base, o[0], o[1]);
    } else {
      dma_1k(lds + at, base, o[0]);
    }
  }
};

// Where a lane reads a tile: rows with bits 2 and 3 swapped as an A operand, and
// transposed (rows 16 hh + 8 (lane / 32) + [0, 8) of dims 32 d + ...) as one.
struct Reads {
  int row[4], turned[2][2];
  __device__ __forceinline__ void init(int lane) {
    const int krow = mfma_row_perm(lane & 31), g = lane >> 5;
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = krow * 128 + (((2 * i + g) ^ tile_swz(krow)) << 4);
    const int G4 = lane >> 4, a = (lane >> 2) & 3, bq = lane & 3;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        const int r = 8 * (G4 >> 1) + 4 * hf + a;
        const int chunk = 4 * db + 2 * (G4 & 1) + (bq >> 1);
        turned[hf][db] = r * 128 + ((chunk ^ tile_swz(r)) << 4) + 8 * (bq & 1);
      }
  }
  __device__ __forceinline__ i4 rows(const char* tile, int i) const {
    return *reinterpret_cast<const i4*>(tile + row[i % 4] + i / 4 * kTile);
  }
  __device__ __forceinline__ i4 columns(const char* tile, int hh, int d) const {
    typedef int i2 __attribute__((ext_vector_type(2)));
    const char* at = tile + (d / 2) * kTile + 2048 * hh;
    const i2 lo = __builtin_bit_cast(i2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(SIDON_LDS_PTR(s4, at + turned[0][d & 1])));
    const i2 hi = __builtin_bit_cast(i2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(SIDON_LDS_PTR(s4, at + turned[1][d & 1])));
    return i4{lo[0], lo[1], hi[0], hi[1]};
  }
};

// An accumulator, rounded: the B operands of two products.
template <typename E>
__device__ __forceinline__ void round_to(const f32x16& x, i4 (&r)[2]) {
  typedef typename Half<E>::v2 v2;
#pragma unroll
  for (int i = 0; i < 16; i += 2)
    r[i >> 3][(i & 7) >> 1] = __builtin_bit_cast(int, __builtin_convertvector(f2{x[i], x[i + 1]}, v2));
}

// Stores of an accumulator set: lane (n, g) holds of its row the values 32 d + 8 i + 4 g + [0, 4).
template <typename E, int N>
__device__ __forceinline__ void store(E* dst, const f32x16 (&x)[N], float by, bool there) {
  typedef typename Half<E>::v4 v4;
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = there ? (E)(x[d][4 * i + e] * by) : (E)0.f;
      *reinterpret_cast<v4*>(dst + 32 * d + 8 * i) = r;
    }
}

// Groups of a workgroup of so many blocks: four wavefronts, two for a block alone at D 128.
constexpr int groups_of(int dim, int blocks) { return dim == 128 && blocks == 1 ? 2 : 4 / blocks; }

// LDS of a workgroup: KS rings of two slots, which hold a step's q, dout and statistics or
// its k and v; then the partial results of half of the groups.
template <int D, int RB, int KS>
struct Lds {
  static constexpr int kStat = 2 * kBlock * 4;
  static constexpr int kTiles = 2 * Copies<D, RB>::kBytes, kKeysSlot = kTiles + kStat;
  static constexpr int kMerge = KS / 2 * RB * 2 * (D / 32) * 16 * 64 * 4;
  static constexpr int kBytes = KS * 2 * kKeysSlot > kMerge ? KS * 2 * kKeysSlot : kMerge;
};

// ---- the first launch: delta and lse of every query, and (fp16) the longest rows ----

// A workgroup of RB wavefronts of 32 queries each x KS key groups.  delta is the sum of P dP, taken
// as dout . out plus the sum of P (dP - dout . out): from the rounded output alone it is off by half a
// step of |dout| |out|, which is all of dS where a query's softmax is nearly one key (dP - delta is
// what the other keys leave).  The difference that is summed up is small, so that what lse's
// and the products' roundings do to P does not matter beside it.
template <typename E, int D, int RB, int KS>
__device__ __forceinline__ void rows_body(const BwdParams& p, char* smem, int block) {
  typedef typename Half<E>::v8 v8;
  using C = Copies<D, RB>;
  constexpr int kQ = D / 16, kRows = RB * kBlock, kSlot = Lds<D, RB, KS>::kTiles;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = w % RB, ks = w / RB;
  const int n = lane & 31, g = lane >> 5;
  int bh;   // of a key head
  const int unit = dealt(p.rows, block, bh);
  if (unit >= p.rows.units) return;
  const int b = bh / p.Hk, hk = bh - b * p.Hk;
  const int head = hk * p.G + unit % p.G, block0 = unit / p.G * kRows;
  const int row = block0 + rb * kBlock + n;   // of this lane
  const int lk = valid(p.lens, b, p.S), lq = valid(p.q_lens, b, p.L);
  const int steps = block0 < lq ? (lk + kBlock - 1) / kBlock : 0;
  const int rounds = (steps + KS - 1) / KS;

  C ck, cv;
  ck.init(rb, lane, p.kl);
  cv.init(rb, lane, p.vl);
  const uint32_t lds = (uint32_t)(uintptr_t)SIDON_LDS_PTR(char, smem) + ks * 2 * kSlot;
  const char* const k0 = static_cast<const char*>(p.k) + 2 * (b * p.kb + hk * p.kh);
  const char* const v0 = static_cast<const char*>(p.v) + 2 * (b * p.vb + hk * p.vh);
  const auto copy = [&](int u) SIDON_INLINE {
    const int t = u * KS + ks;
    if (t < steps) {
      const uint32_t at = lds + (u & 1) * kSlot;
      ck.copy(at, k0 + (int64_t)t * kBlock * p.kl * 2, lk - t * kBlock);
      cv.copy(at + C::kBytes, v0 + (int64_t)t * kBlock * p.vl * 2, lk - t * kBlock);
    }
  };
  copy(0);

  Reads at;
  at.init(lane);
  i4 qop[kQ], gop[kQ];
  float dot = 0.f, sq = 0.f, lse = INFINITY;   // lse of no such row, or of one that sees no key: P = 0
  const int rr = max(min(row, lq - 1), 0);
  {
    const E* const qp = static_cast<const E*>(p.q) + b * p.qb + head * p.qh + (int64_t)rr * p.ql + 8 * g;
    const E* const gp = static_cast<const E*>(p.dout) + b * p.gb + head * p.gh + (int64_t)rr * p.gl + 8 * g;
    const E* const op = static_cast<const E*>(p.out) + b * p.ob + head * p.oh + rr * p.ol + 8 * g;
    i4 oop[kQ];
#pragma unroll
    for (int s = 0; s < kQ; ++s) {
      qop[s] = *reinterpret_cast<const i4*>(qp + 16 * s);
      gop[s] = *reinterpret_cast<const i4*>(gp + 16 * s);
      oop[s] = *reinterpret_cast<const i4*>(op + 16 * s);
    }
    if (row < lq) {
      lse = p.lse[((int64_t)b * p.H + head) * p.L + row];
      lse = lse == -INFINITY ? INFINITY : lse * kLog2e;
#pragma unroll
      for (int s = 0; s < kQ; ++s) {
        const v8 x = __builtin_bit_cast(v8, gop[s]), y = __builtin_bit_cast(v8, oop[s]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          dot = fmaf((float)x[k], (float)y[k], dot);
          sq = fmaf((float)x[k], (float)x[k], sq);
        }
      }
    }
  }
  dot = pair_sum(dot);
  sq = pair_sum(sq);
  arrived(qop);
  arrived(gop);
  asm volatile("" : "+v"(lse), "+v"(dot), "+v"(sq));
  const float scale2 = p.scale * kLog2e;

  float more[4] = {};   // sum of P (dP - dout . out), of this lane's keys
  for (int u = 0; u < rounds; ++u) {
    wait_vmcnt<0>();
    lds_barrier();   // round u is there, and round u - 1 is read
    copy(u + 1);
    const int t = u * KS + ks;
    if (t >= steps) continue;
    const char* const tk = smem + (ks * 2 + (u & 1)) * kSlot;
    const char* const tv = tk + C::kBytes;
    f32x16 s = {}, dp;
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] = -dot;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      s = Half<E>::mfma(at.rows(tk, i), qop[i], s);
      dp = Half<E>::mfma(at.rows(tv, i), gop[i], dp);
    }
    if ((t + 1) * kBlock > lk) {
      const int left = lk - t * kBlock - 8 * g;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i >> 3) + (i & 7) >= left) s[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) more[i % 4] = fmaf(fast_exp2(fmaf(s[i], scale2, -lse)), dp[i], more[i % 4]);
  }
  float sum = pair_sum((more[0] + more[1]) + (more[2] + more[3]));
  if constexpr (KS > 1) {
    float* const part = reinterpret_cast<float*>(smem);
    lds_barrier();   // the rings are done with
    if (g == 0) part[w * kBlock + n] = sum;
    lds_barrier();
    if (ks > 0) return;
    sum = part[rb * kBlock + n];
#pragma unroll
    for (int k = 1; k < KS; ++k) sum += part[(k * RB + rb) * kBlock + n];
  }
  const int tile = block0 / kBlock + rb;
  if (tile >= p.tiles) return;
  const int64_t to = ((int64_t)b * p.H + head) * p.tiles + tile;
  const float length = sqrtf(sq);
  if (g == 0) {
    p.stat[to * (2 * kBlock) + n] = Range<E>::kLift - lse;
    p.stat[to * (2 * kBlock) + kBlock + n] = row < lq ? -(dot + sum) : 0.f;
    if (Range<E>::kScaled) p.length[to * kBlock + n] = length;
  }
  if constexpr (Range<E>::kScaled) {
    float top = length;
#pragma unroll
    for (int d = 1; d < kBlock; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (lane == 0) p.longest[to] = top;
  }
}

// The longest v of a tile of 32 keys, by a wavefront.
template <typename E, int D>
__device__ __forceinline__ void longest_key(const BwdParams& p, int64_t at) {
  typedef typename Half<E>::v8 v8;
  constexpr int kTeam = D / 8, kAtOnce = 64 / kTeam;   // lanes of a row, rows
  const int lane = threadIdx.x & 63, i = lane % kTeam;
  const int tile = (int)(at % p.key_tiles), bh = (int)(at / p.key_tiles), b = bh / p.Hk, h = bh - b * p.Hk;
  const int rows = valid(p.lens, b, p.S);
  const E* const vp = static_cast<const E*>(p.v) + b * p.vb + h * p.vh + 8 * i;
  float top = 0.f;
#pragma unroll
  for (int r0 = 0; r0 < kBlock; r0 += kAtOnce) {
    const int row = tile * kBlock + r0 + lane / kTeam;
    float sq = 0.f;
    if (row < rows) {
      const v8 x = *reinterpret_cast<const v8*>(vp + (int64_t)row * p.vl);
#pragma unroll
      for (int k = 0; k < 8; ++k) sq = fmaf((float)x[k], (float)x[k], sq);
    }
    top = fmaxf(top, team_sum<kTeam>(sq));
  }
  for (int d = kTeam; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) p.longest_v[at] = sqrtf(top);
}

template <typename E, int D, int RB>
__global__ void __launch_bounds__(256, 2) cross_bwd_rows_kernel(const BwdParams p) {
  constexpr int KS = 4 / RB;
  __shared__ __attribute__((aligned(16))) char smem[KS * 2 * Lds<D, RB, KS>::kTiles];
  const int first = (int)p.rows.groups();
  if ((int)blockIdx.x < first) {
    rows_body<E, D, RB, KS>(p, smem, blockIdx.x);
  } else if constexpr (Range<E>::kScaled) {
    const int64_t at = (int64_t)(blockIdx.x - first) * 4 + (threadIdx.x >> 6);
    if (at < (int64_t)p.B * p.Hk * p.key_tiles) longest_key<E, D>(p, at);
  }
}

// ---- dk and dv: a workgroup of RB wavefronts of 32 keys each x KS row groups, which take
// every KS-th step of 32 queries (of the heads in turn) from a ring of their own ----
template <typename E, int D, int RB, int KS>
__device__ __forceinline__ void keys_body(const BwdParams& p, char* smem, int block) {
  using C = Copies<D, RB>;
  constexpr int kQ = D / 16, kDb = D / 32, kSlot = Lds<D, RB, KS>::kKeysSlot;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = w % RB, ks = w / RB;
  const int n = lane & 31, g = lane >> 5;
  int bh;
  const int unit = dealt(p.keys, block, bh);
  if (unit >= p.keys.units) return;
  const int b = bh / p.Hk, hk = bh - b * p.Hk;
  const int key = (unit * RB + rb) * kBlock + n;
  const int lk = valid(p.lens, b, p.S), lq = valid(p.q_lens, b, p.L);
  const int tiles = unit * RB * kBlock < lk ? (lq + kBlock - 1) / kBlock : 0;   // of a head
  const int steps = tiles * p.G, rounds = (steps + KS - 1) / KS;

  C cq, cg;
  cq.init(rb, lane, p.ql);
  cg.init(rb, lane, p.gl);
  const uint32_t lds = (uint32_t)(uintptr_t)SIDON_LDS_PTR(char, smem) + ks * 2 * kSlot;
  const char* const q0 = static_cast<const char*>(p.q) + 2 * (b * p.qb + (int64_t)hk * p.G * p.qh);
  const char* const g0 = static_cast<const char*>(p.dout) + 2 * (b * p.gb + (int64_t)hk * p.G * p.gh);
  const char* const s0 = reinterpret_cast<const char*>(p.stat + ((int64_t)b * p.H + hk * p.G) * p.tiles * (2 * kBlock));
  int ch = 0, ct = ks;   // head of the group and tile that are copied next
  const auto copy = [&](int slot) SIDON_INLINE {
    while (ct >= tiles && ch < p.G) ct -= tiles, ++ch;
    if (ch < p.G) {
      const int rows = lq - ct * kBlock;
      const uint32_t at = lds + slot * kSlot;
      cq.copy(at, q0 + 2 * (ch * p.qh + (int64_t)ct * kBlock * p.ql), rows);
      cg.copy(at + C::kBytes, g0 + 2 * (ch * p.gh + (int64_t)ct * kBlock * p.gl), rows);
      if (rb == 0) dma_256(at + 2 * C::kBytes, uniform(s0 + ((int64_t)ch * p.tiles + ct) * (2 * kBlock * 4)), 4 * lane);
      ct += KS;
    }
  };
  if (steps > 0) copy(0);

  Reads at;
  at.init(lane);
  i4 kop[kQ], vop[kQ];
  {
    const int kk = max(min(key, lk - 1), 0);
    const E* kp = static_cast<const E*>(p.k) + b * p.kb + hk * p.kh + (int64_t)kk * p.kl + 8 * g;
    const E* vp = static_cast<const E*>(p.v) + b * p.vb + hk * p.vh + (int64_t)kk * p.vl + 8 * g;
#pragma unroll
    for (int s = 0; s < kQ; ++s) {
      kop[s] = *reinterpret_cast<const i4*>(kp + 16 * s);
      vop[s] = *reinterpret_cast<const i4*>(vp + 16 * s);
    }
  }
  constexpr float kLift = Range<E>::kLift;
  float c = 1.f;
  if constexpr (Range<E>::kScaled)
    c = below_one(largest(p.longest + ((int64_t)b * p.H + hk * p.G) * p.tiles, p.G * p.tiles, lane),
                  largest(p.longest_v + (int64_t)bh * p.key_tiles, p.key_tiles, lane));
  asm volatile("" : "+v"(c));
  const float scale2 = p.scale * kLog2e;

  arrived(kop);
  arrived(vop);
  f32x16 dk[kDb], dv[kDb];
#pragma unroll
  for (int d = 0; d < kDb; ++d) dk[d] = f32x16{}, dv[d] = f32x16{};
  for (int u = 0; u < rounds; ++u) {
    wait_vmcnt<0>();
    lds_barrier();   // round u is there, and round u - 1 is read
    copy((u + 1) & 1);
    if (u * KS + ks >= steps) continue;
    const char* const tq = smem + (ks * 2 + (u & 1)) * kSlot;
    const char* const tg = tq + C::kBytes;
    // element i of an accumulator is row 16 (i / 8) + 8 g + i % 8
    const float* const st = reinterpret_cast<const float*>(tq + 2 * C::kBytes) + 8 * g;
    f32x16 s = {}, dp, lse;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const f4 x = *reinterpret_cast<const f4*>(st + kBlock + 16 * (i >> 3) + (i & 7));
      const f4 y = *reinterpret_cast<const f4*>(st + 16 * (i >> 3) + (i & 7));
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[i + e] = x[e], lse[i + e] = y[e];   // -delta, kLift - lse
    }
    i4 qa[kQ], ga[kQ];
#pragma unroll
    for (int i = 0; i < kQ; ++i) qa[i] = at.rows(tq, i), ga[i] = at.rows(tg, i);
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      s = Half<E>::mfma(qa[i], kop[i], s);
      dp = Half<E>::mfma(ga[i], vop[i], dp);
    }
    i4 pk[2], dk16[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], scale2, lse[i]));
    round_to<E>(s, pk);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= Range<E>::kScaled ? dp[i] * c : dp[i];
    round_to<E>(s, dk16);
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int d = 0; d < kDb; ++d) {
        dv[d] = Half<E>::mfma(at.columns(tg, hh, d), pk[hh], dv[d]);
        dk[d] = Half<E>::mfma(at.columns(tq, hh, d), dk16[hh], dk[d]);
      }
  }

  // ---- sum the row groups, half of them into the other half at a time ----
  if constexpr (KS > 1) {
    float* const mem = reinterpret_cast<float*>(smem) + lane * 4;
#pragma unroll
    for (int half = KS / 2; half >= 1; half >>= 1) {
      lds_barrier();
      float* const part = mem + ((ks % half) * RB + rb) * (2 * kDb * 16 * 64);
      const auto each = [&](auto&& f) SIDON_INLINE {
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f(dk[d], i, reinterpret_cast<f4*>(part + (d * 8 + i) * 256));
            f(dv[d], i, reinterpret_cast<f4*>(part + (d * 8 + 4 + i) * 256));
          }
      };
      if (ks >= half)
        each([](const f32x16& x, int i, f4* to) SIDON_INLINE { *to = f4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]}; });
      lds_barrier();
      if (ks >= half) return;
      each([](f32x16& x, int i, const f4* from) SIDON_INLINE {
        const f4 v = *from;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] += v[e];
      });
    }
  }
  if (key >= p.S) return;
  const bool there = key < lk;
  const float down = fast_exp2(-kLift);
  store<E>(static_cast<E*>(p.dk) + b * p.dkb + hk * p.dkh + key * p.dkl + 4 * g, dk, p.scale * down / c, there);
  store<E>(static_cast<E*>(p.dv) + b * p.dvb + hk * p.dvh + key * p.dvl + 4 * g, dv, down, there);
}

// ---- dq: a workgroup of RB wavefronts of 32 queries each x KS key groups, which take
// every KS-th step of 32 keys from a ring of their own ----
template <typename E, int D, int RB, int KS>
__device__ __forceinline__ void queries_body(const BwdParams& p, char* smem, int block) {
  using C = Copies<D, RB>;
  constexpr int kQ = D / 16, kDb = D / 32, kRows = RB * kBlock, kSlot = Lds<D, RB, KS>::kTiles;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = w % RB, ks = w / RB;
  const int n = lane & 31, g = lane >> 5;
  int bh;   // of a key head
  const int unit = dealt(p.queries, block, bh);
  if (unit >= p.queries.units) return;
  const int b = bh / p.Hk, hk = bh - b * p.Hk;
  const int head = hk * p.G + unit % p.G, block0 = unit / p.G * kRows;
  const int row = block0 + rb * kBlock + n;   // of this lane
  const int lk = valid(p.lens, b, p.S), lq = valid(p.q_lens, b, p.L);
  const int steps = block0 < lq ? (lk + kBlock - 1) / kBlock : 0;
  const int rounds = (steps + KS - 1) / KS;

  C ck, cv;
  ck.init(rb, lane, p.kl);
  cv.init(rb, lane, p.vl);
  const uint32_t lds = (uint32_t)(uintptr_t)SIDON_LDS_PTR(char, smem) + ks * 2 * kSlot;
  const char* const k0 = static_cast<const char*>(p.k) + 2 * (b * p.kb + hk * p.kh);
  const char* const v0 = static_cast<const char*>(p.v) + 2 * (b * p.vb + hk * p.vh);
  const auto copy = [&](int u) SIDON_INLINE {
    const int t = u * KS + ks;
    if (t < steps) {
      const uint32_t at = lds + (u & 1) * kSlot;
      ck.copy(at, k0 + (int64_t)t * kBlock * p.kl * 2, lk - t * kBlock);
      cv.copy(at + C::kBytes, v0 + (int64_t)t * kBlock * p.vl * 2, lk - t * kBlock);
    }
  };
  copy(0);

  Reads at;
  at.init(lane);
  constexpr float kLift = Range<E>::kLift;
  i4 qop[kQ], gop[kQ];
  const int rr = max(min(row, lq - 1), 0);
  const E* const qp = static_cast<const E*>(p.q) + b * p.qb + head * p.qh + (int64_t)rr * p.ql + 8 * g;
  const E* const gp = static_cast<const E*>(p.dout) + b * p.gb + head * p.gh + (int64_t)rr * p.gl + 8 * g;
#pragma unroll
  for (int s = 0; s < kQ; ++s) {
    qop[s] = *reinterpret_cast<const i4*>(qp + 16 * s);
    gop[s] = *reinterpret_cast<const i4*>(gp + 16 * s);
  }
  const int64_t tile = ((int64_t)b * p.H + head) * p.tiles + rr / kBlock;
  float lse = p.stat[tile * (2 * kBlock) + rr % kBlock];              // kLift - lse
  float delta = p.stat[tile * (2 * kBlock) + kBlock + rr % kBlock];   // -delta
  float c = 1.f;
  if constexpr (Range<E>::kScaled)
    c = below_one(p.length[tile * kBlock + rr % kBlock], largest(p.longest_v + (int64_t)bh * p.key_tiles, p.key_tiles, lane));
  if constexpr (Range<E>::kScaled) lse += __log2f(c);   // (P itself is not wanted here: its exponent takes the power of two)
  arrived(qop);
  arrived(gop);
  asm volatile("" : "+v"(lse), "+v"(delta));
  const float scale2 = p.scale * kLog2e;

  f32x16 dq[kDb];
#pragma unroll
  for (int d = 0; d < kDb; ++d) dq[d] = f32x16{};
  for (int u = 0; u < rounds; ++u) {
    wait_vmcnt<0>();
    lds_barrier();
    copy(u + 1);
    const int t = u * KS + ks;
    if (t >= steps) continue;
    const char* const tk = smem + (ks * 2 + (u & 1)) * kSlot;
    const char* const tv = tk + C::kBytes;
    f32x16 s = {}, dp;
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] = delta;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      s = Half<E>::mfma(at.rows(tk, i), qop[i], s);
      dp = Half<E>::mfma(at.rows(tv, i), gop[i], dp);
    }
    if ((t + 1) * kBlock > lk) {
      const int left = lk - t * kBlock - 8 * g;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i >> 3) + (i & 7) >= left) s[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], scale2, lse)) * dp[i];
    i4 pk[2];
    round_to<E>(s, pk);
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int d = 0; d < kDb; ++d) dq[d] = Half<E>::mfma(at.columns(tk, hh, d), pk[hh], dq[d]);
  }

  // ---- sum the key groups, half of them into the other half at a time ----
  if constexpr (KS > 1) {
    float* const mem = reinterpret_cast<float*>(smem) + lane * 4;
#pragma unroll
    for (int half = KS / 2; half >= 1; half >>= 1) {
      lds_barrier();   // the rings, or the last round's values, are done with
      float* const part = mem + ((ks % half) * RB + rb) * (kDb * 16 * 64);
      if (ks >= half) {
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f4*>(part + (d * 4 + i) * 256) = f4{dq[d][4 * i], dq[d][4 * i + 1], dq[d][4 * i + 2], dq[d][4 * i + 3]};
      }
      lds_barrier();
      if (ks >= half) return;
#pragma unroll
      for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f4 v = *reinterpret_cast<const f4*>(part + (d * 4 + i) * 256);
#pragma unroll
          for (int e = 0; e < 4; ++e) dq[d][4 * i + e] += v[e];
        }
    }
  }
  if (row >= p.L) return;
  store<E>(static_cast<E*>(p.dq) + b * p.dqb + head * p.dqh + row * p.dql + 4 * g, dq, p.scale * fast_exp2(-kLift) / c,
           row < lq && lk > 0);
}

// Both in one launch: neither needs the other's results, and the workgroups of the second
// fill what the last ones of the first leave idle (1 x 16 heads x 4800 x 4800, D 128: 620 us,
// one after the other 751).
template <typename E, int D, int KB, int QB, int kWaves, bool kQueriesFirst>
__global__ void __launch_bounds__(64 * KB * groups_of(D, KB)) __attribute__((amdgpu_waves_per_eu(kWaves, kWaves)))
cross_bwd_kernel(const BwdParams p) {
  constexpr int KS = groups_of(D, KB), QS = groups_of(D, QB);
  static_assert(KB * KS == QB * QS, "as many wavefronts");
  constexpr int kKeys = Lds<D, KB, KS>::kBytes, kQueries = Lds<D, QB, QS>::kBytes;
  __shared__ __attribute__((aligned(16))) char smem[kKeys > kQueries ? kKeys : kQueries];
  const int first = (int)(kQueriesFirst ? p.queries.groups() : p.keys.groups());   // (a multiple of 8: the XCDs go on in turn)
  if (((int)blockIdx.x < first) != kQueriesFirst) {
    keys_body<E, D, KB, KS>(p, smem, blockIdx.x - (kQueriesFirst ? first : 0));
  } else {
    queries_body<E, D, QB, QS>(p, smem, blockIdx.x - (kQueriesFirst ? 0 : first));
  }
}

// ---- host -------------------------------------------------------------------------

bool shape_ok(int B, int H, int Hk, int L, int S, int D) {
  return B >= 1 && H >= 1 && Hk >= 1 && H % Hk == 0 && L >= 1 && S >= 1 && (D == 64 || D == 128) &&
         S <= (1 << 24) && (int64_t)(H / Hk) * L <= (1 << 24) && (int64_t)B * H <= (1 << 20);
}

int tiles_of(int rows) { return (rows + kBlock - 1) / kBlock; }

// In floats: statistics, lengths, the longest of a tile and of a key tile.
struct Workspace {
  size_t stat, length, longest, longest_v;
  size_t bytes() const { return 4 * (stat + length + longest + longest_v); }
};
Workspace workspace(int B, int H, int Hk, int L, int S, int dtype) {
  const size_t tiles = (size_t)B * H * tiles_of(L);
  if (dtype == SIDON_BF16) return Workspace{tiles * 2 * kBlock, 0, 0, 0};
  return Workspace{tiles * 2 * kBlock, tiles * kBlock, tiles, (size_t)B * Hk * tiles_of(S)};
}

// Which form: blocks of 32 keys and of 32 rows of a workgroup, and whose are launched first, by
// the least estimate (us)
//
//   base + keys n_k + queries n_q + keys_round n_k r_k + queries_round n_q r_q
//        + keys_turn r_k ceil(n_k / fit) + queries_turn r_q ceil(n_q / fit) + longest max(r_k, r_q) + last r
//
// with n workgroups a CU of either kind, of r rounds each (its steps over its groups), the
// last ones' r (with a first launch of 5 us, the same for all of them): what all of them take together, and what the busiest CU's, the longest one and
// the last take.  (More groups make a workgroup shorter, more blocks share copies, and where the
// longer kind waits for the other it ends late.)  20000 shapes of 1 to 24 items, 8 to 2400
// queries and 30 to 5000 keys were timed in 18 forms at D 64 and 10 at 128; these are the ones
// that the others rarely beat, and their numbers chosen for the choice: it takes 1.02 times the
// best one's time on average, 1.2 in 99 of 100 (one form for both kinds, in the better order: 1.06 at
// best, at D 64; 4 x 16 heads (4 key heads) x 1200 x 4800 306 us, with one form 324; 1 x 16 x 300 x 4800 42 and 55; the first launch
// is 15 to 115 now, whichever form).
struct Form {
  int dim, key_blocks, query_blocks;
  bool queries_first;
  int fit;
  double base, keys, queries, keys_round, queries_round, keys_turn, queries_turn, longest, last;
};
constexpr Form kForms[] = {{64, 4, 2, false, 1, 9.55, 1.59, 1.15, .00519, .00611, .233, 0, .825, 0},
                           {64, 4, 2, true, 1, 9.02, 1.42, 2.19, 0, 0, .00427, .253, .109, 1.06},
                           {64, 4, 1, false, 1, 3.58, 6.06, .777, 0, .00899, .736, .665, 1.13, 0},
                           {64, 4, 1, true, 1, 7.5, .0957, 6.87, .00644, .477, .538, .0867, .011, .215},
                           {64, 2, 4, false, 2, 9.01, 3.63, .0469, .0182, .328, .471, 0, .722, 0},
                           {64, 2, 4, true, 1, 8.19, 1.53, 4.57, .0645, 0, .566, .173, .0621, .77},
                           {64, 2, 1, false, 1, 4.99, 7.03, 2.32, 0, .00386, .449, .11, .754, 0},
                           {64, 2, 1, true, 1, 5.46, 1.62, 7.92, 0, .0103, .625, .0126, .543, .191},
                           {64, 1, 4, false, 1, 6.43, 5.11, 1.18, .362, 0, .468, .229, .0192, .297},
                           {64, 1, 4, true, 1, 7.73, 1.87, 3.37, .38, .681, .0298, .161, .126, .448},
                           {64, 1, 2, false, 1, 5.42, 4.87, 2.18, .211, .404, .307, .00446, .284, .449},
                           {64, 1, 2, true, 1, 5.86, 2.6, 5.61, .457, .0501, .635, .161, .364, 0},
                           {128, 4, 2, false, 1, 8.66, 3.39, 3.88, .00365, .00429, .661, 0, 1.18, .383},
                           {128, 4, 2, true, 1, 9.01, .391, 7.66, .00418, 0, .527, .0384, .932, .946},
                           {128, 2, 4, false, 2, 10.6, 5.42, .081, .705, .607, 1.35, 0, .447, 0},
                           {128, 1, 1, false, 1, 7.85, 3.8, 1.31, .241, .845, .0651, .178, .466, .761},
                           {128, 1, 1, true, 1, 8.52, 1.72, 5.33, 1.52, 0, .0846, .379, .0187, .332}};

int choose(const BwdParams& p, int D, int cus) {
  int best = -1;
  double best_us = 0;
  for (int i = 0; i < (int)(sizeof(kForms) / sizeof(kForms[0])); ++i) {
    const Form& f = kForms[i];
    if (f.dim != D) continue;
    const int keys = f.key_blocks * kBlock, rows = f.query_blocks * kBlock;
    const int ks = groups_of(D, f.key_blocks), qs = groups_of(D, f.query_blocks);
    const double nk = (double)((int64_t)p.B * p.Hk * ((p.S + keys - 1) / keys)) / cus;
    const double nq = (double)((int64_t)p.B * p.H * ((p.L + rows - 1) / rows)) / cus;
    const double rk = (double)(((int64_t)p.G * p.tiles + ks - 1) / ks), rq = (double)((p.key_tiles + qs - 1) / qs);
    const double us = f.base + f.keys * nk + f.queries * nq + f.keys_round * nk * rk + f.queries_round * nq * rq +
                      f.keys_turn * rk * ceil(nk / f.fit) + f.queries_turn * rq * ceil(nq / f.fit) +
                      f.longest * (rk > rq ? rk : rq) + f.last * (f.queries_first ? rk : rq);
    if (best < 0 || us < best_us) best = i, best_us = us;
  }
  return best;
}

template <typename E, int D, int KB, int QB>
void launch_form(BwdParams& p, bool queries_first, hipStream_t stream) {
  constexpr int kKeys = KB * kBlock, kRows = QB * kBlock;
  // (wavefronts a SIMD: three of 168 registers at D 64 and two of 256 at 128, for which most of these
  // kernels spill 1 to 13 of them, or as the LDS of a block alone allows, whose four groups have rings
  // of their own)
  constexpr int kWaves = (D == 64 ? 3 : 2) - (KB == 1 || QB == 1 ? 1 : 0);
  const int64_t heads = (int64_t)p.B * p.Hk;
  p.keys = deal(heads, (p.S + kKeys - 1) / kKeys, (int64_t)p.G * p.L * D * 4);
  p.queries = deal(heads, (int64_t)p.G * ((p.L + kRows - 1) / kRows), (int64_t)p.S * D * 4);
  const dim3 grid(p.keys.groups() + p.queries.groups()), block(64 * KB * groups_of(D, KB));
  if constexpr (D == 64 || KB != 2) {   // (not of kForms)
    if (queries_first) {
      hipLaunchKernelGGL((cross_bwd_kernel<E, D, KB, QB, kWaves, true>), grid, block, 0, stream, p);
      return;
    }
  }
  hipLaunchKernelGGL((cross_bwd_kernel<E, D, KB, QB, kWaves, false>), grid, block, 0, stream, p);
}

template <typename E, int D, int RB>
void launch_row_blocks(BwdParams& p, hipStream_t stream) {
  constexpr int kRows = RB * kBlock;
  const int64_t heads = (int64_t)p.B * p.Hk;
  p.rows = deal(heads, (int64_t)p.G * ((p.L + kRows - 1) / kRows), (int64_t)p.S * D * 4);
  unsigned groups = p.rows.groups();
  if (Range<E>::kScaled) groups += (unsigned)((heads * p.key_tiles + 3) / 4);
  hipLaunchKernelGGL((cross_bwd_rows_kernel<E, D, RB>), dim3(groups), dim3(256), 0, stream, p);
}

// A block of 32 queries of four key groups while all of them run at once (the LDS of their rings lets
// a CU hold two at D 64, one at 128), else two blocks of two groups: us of both launches, 1 x 16 heads x 300 x 4800
// 70 and 79, 2 x 16 x 300 x 1463 43.6 and 44.4, but 8 x 16 x 448 x 1500 174 and 151, 4 x 16 (4 key heads) x 1200 x 4800
// 439 and 408; at D 128 2 x 16 (4) x 128 x 3000 82 and 92, 2 x 16 x 300 x 1463 85 and 75.
template <typename E, int D>
void launch_rows(BwdParams& p, hipStream_t stream) {
  if ((int64_t)p.B * p.H * p.tiles <= (int64_t)(D == 64 ? 2 : 1) * sidon::compute_units())
    launch_row_blocks<E, D, 1>(p, stream);
  else
    launch_row_blocks<E, D, 2>(p, stream);
}

template <typename E, int D>
void launch(BwdParams& p, hipStream_t stream) {
  launch_rows<E, D>(p, stream);
  const Form& f = kForms[choose(p, D, sidon::compute_units())];
  switch (f.key_blocks * 10 + f.query_blocks) {   // (those of kForms)
    case 42: return launch_form<E, D, 4, 2>(p, f.queries_first, stream);
    case 24: return launch_form<E, D, 2, 4>(p, f.queries_first, stream);
    default: break;
  }
  if constexpr (D == 64) {
    switch (f.key_blocks * 10 + f.query_blocks) {
      case 41: return launch_form<E, D, 4, 1>(p, f.queries_first, stream);
      case 21: return launch_form<E, D, 2, 1>(p, f.queries_first, stream);
      case 14: return launch_form<E, D, 1, 4>(p, f.queries_first, stream);
      default: return launch_form<E, D, 1, 2>(p, f.queries_first, stream);
    }
  } else {
    launch_form<E, D, 1, 1>(p, f.queries_first, stream);
  }
}

}  // namespace

SIDON_API size_t sidon_cross_attention_bwd_workspace_bytes(int B, int H, int Hk, int L, int S, int D, int dtype) {
  if (!shape_ok(B, H, Hk, L, S, D) || (dtype != SIDON_FP16 && dtype != SIDON_BF16)) return 0;
  return workspace(B, H, Hk, L, S, dtype).bytes();
}

SIDON_API int sidon_cross_attention_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                        const float* lse, const int32_t* lens, const int32_t* q_lens, float scale,
                                        void* dq, void* dk, void* dv, void* ws, size_t ws_bytes, int B, int H, int Hk,
                                        int L, int S, int D, int dtype, const int64_t* g_strides,
                                        const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                        const int64_t* o_strides, const int64_t* dq_strides, const int64_t* dk_strides,
                                        const int64_t* dv_strides, sidon_stream_t stream) {
  using sidon::fail;
  using sidon::Rows;
  sidon::clear_error();
  if (!dout || !q || !k || !v || !out || !lse || !dq || !dk || !dv || !ws || !g_strides || !q_strides || !k_strides ||
      !v_strides || !o_strides || !dq_strides || !dk_strides || !dv_strides)
    return fail(SIDON_E_NULL, "dout, q, k, v, out, lse, dq, dk, dv, ws and the strides must be non-NULL");
  if (dtype != SIDON_FP16 && dtype != SIDON_BF16) return fail(SIDON_E_SHAPE, "dtype=%d is neither SIDON_FP16 nor SIDON_BF16", dtype);
  if (!shape_ok(B, H, Hk, L, S, D))
    return fail(SIDON_E_SHAPE, "B=%d H=%d Hk=%d L=%d S=%d D=%d: need sizes >= 1, H a multiple of Hk, D 64 or 128, H / Hk * L and S <= 2^24, B * H <= 2^20",
                B, H, Hk, L, S, D);
  if (!(scale >= FLT_MIN && scale <= 0x1p100f)) return fail(SIDON_E_SHAPE, "scale=%g must be positive and at most 2^100", scale);
  const int64_t far = int64_t(1) << 40, near = (int64_t(1) << 25) - 1;
  const struct {
    const char* name;
    const void* at;
    const int64_t* s;
    int heads, len;
    int64_t row_most;
  } all[] = {{"dout", dout, g_strides, H, L, near}, {"q", q, q_strides, H, L, near}, {"k", k, k_strides, Hk, S, near},
             {"v", v, v_strides, Hk, S, near},      {"out", out, o_strides, H, L, far}, {"dq", dq, dq_strides, H, L, far},
             {"dk", dk, dk_strides, Hk, S, far},    {"dv", dv, dv_strides, Hk, S, far}};
  constexpr int kTensors = 8, kRead = 5;
  Rows rows[kTensors];
  const __int128 most = (__int128)1 << 61;
  for (int t = 0; t < kTensors; ++t) {
    for (int i = 0; i < 3; ++i)
      if (all[t].s[i] < 0 || all[t].s[i] % 8 != 0 || all[t].s[i] > (i == 2 ? all[t].row_most : far))
        return fail(SIDON_E_STRIDE, "%s stride %lld (number %d) must be a multiple of 8 in [0, %s]", all[t].name,
                    (long long)all[t].s[i], i, i == 2 && all[t].row_most < far ? "2^25)" : "2^40]");
    if (!sidon::aligned16(all[t].at)) return fail(SIDON_E_ALIGN, "%s must be 16-byte aligned", all[t].name);
    rows[t] = Rows{all[t].at, {B, all[t].heads, all[t].len}, {all[t].s[0], all[t].s[1], all[t].s[2]}, D, 2};
    if (rows[t].bytes() > most) return fail(SIDON_E_STRIDE, "%s spans more than the address space", all[t].name);
    if (t >= kRead && !sidon::apart(rows[t].n, rows[t].st, 3, D)) return fail(SIDON_E_STRIDE, "rows of %s overlap one another", all[t].name);
  }
  if (((reinterpret_cast<uintptr_t>(lens) | reinterpret_cast<uintptr_t>(q_lens) | reinterpret_cast<uintptr_t>(lse)) & 3u) != 0 ||
      !sidon::aligned16(ws))
    return fail(SIDON_E_ALIGN, "lens, q_lens and lse must be 4-byte aligned, ws 16-byte aligned");
  const Workspace need = workspace(B, H, Hk, L, S, dtype);
  if (ws_bytes < need.bytes()) return fail(SIDON_E_SHAPE, "ws holds %zu bytes, the call needs %zu", ws_bytes, need.bytes());
  for (int t = kRead; t < kTensors; ++t)
    for (int o = 0; o < t; ++o)
      if (sidon::tensors_meet(rows[o], rows[t])) return fail(SIDON_E_SHAPE, "%s must lie apart from %s", all[t].name, all[o].name);
  const struct {
    const char* name;
    const void* at;
    int64_t bytes;
  } flat[] = {{"ws", ws, (int64_t)need.bytes()},
              {"lse", lse, (int64_t)4 * B * H * L},
              {"lens", lens, lens ? (int64_t)4 * B : 0},
              {"q_lens", q_lens, q_lens ? (int64_t)4 * B : 0}};
  for (int i = 0; i < 4; ++i) {
    if (flat[i].bytes == 0) continue;
    for (int t = i == 0 ? 0 : kRead; t < kTensors; ++t)
      if (sidon::ranges_meet(flat[i].at, flat[i].bytes, rows[t].at, (int64_t)rows[t].bytes()))
        return fail(SIDON_E_SHAPE, "%s must lie apart from %s", flat[i].name, all[t].name);
    if (i > 0 && sidon::ranges_meet(ws, flat[0].bytes, flat[i].at, flat[i].bytes))
      return fail(SIDON_E_SHAPE, "ws must lie apart from %s", flat[i].name);
  }
  const int64_t heads = (int64_t)B * Hk;
  if ((int64_t)B * H * tiles_of(L) + heads * tiles_of(S) > INT32_MAX / 512 ||
      !deal_fits(heads, tiles_of(S) + (int64_t)(H / Hk) * tiles_of(L) + 8))
    return fail(SIDON_E_SHAPE, "too many rows for one launch");
  const int rc = sidon::check_device();
  if (rc) return rc;
  BwdParams p{};
  p.q = q, p.k = k, p.v = v, p.out = out, p.dout = dout, p.lse = lse, p.dq = dq, p.dk = dk, p.dv = dv;
  p.lens = lens, p.q_lens = q_lens;
  p.stat = static_cast<float*>(ws);
  p.length = p.stat + need.stat;
  p.longest = p.length + need.length;
  p.longest_v = p.longest + need.longest;
  p.gb = g_strides[0], p.gh = g_strides[1], p.gl = (int)g_strides[2];
  p.qb = q_strides[0], p.qh = q_strides[1], p.ql = (int)q_strides[2];
  p.kb = k_strides[0], p.kh = k_strides[1], p.kl = (int)k_strides[2];
  p.vb = v_strides[0], p.vh = v_strides[1], p.vl = (int)v_strides[2];
  p.ob = o_strides[0], p.oh = o_strides[1], p.ol = o_strides[2];
  p.dqb = dq_strides[0], p.dqh = dq_strides[1], p.dql = dq_strides[2];
  p.dkb = dk_strides[0], p.dkh = dk_strides[1], p.dkl = dk_strides[2];
  p.dvb = dv_strides[0], p.dvh = dv_strides[1], p.dvl = dv_strides[2];
  p.B = B, p.H = H, p.Hk = Hk, p.G = H / Hk, p.L = L, p.S = S;
  p.tiles = tiles_of(L), p.key_tiles = tiles_of(S);
  p.scale = scale;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SIDON_FP16) {
    if (D == 64) launch<_Float16, 64>(p, s);
    else launch<_Float16, 128>(p, s);
  } else {
    if (D == 64) launch<__bf16, 64>(p, s);
    else launch<__bf16, 128>(p, s);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(SIDON_E_LAUNCH, "cross attention gradient launch failed: %s", hipGetErrorString(err));
  return SIDON_OK;
}
