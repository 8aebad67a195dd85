// head_norm.hip -- the norm of queries and keys for each head with the position
// rotation in the same pass, and its gradients (MI355X / gfx950).  A row is a
// head's D values of one token at place p:
//
//   y = R_p (w n),   n = x r,   r = 1 / sqrt(mean(x^2) + eps)
//
// R_p turns pairs of the first `rot` values, (j, j + rot / 2) or (2 j, 2 j + 1), by
// the angle whose cosine and sine are row p, column j of the tables.  With g = R_p^T dy:
//
//   dw = sum over rows of g n,   dx = r (w g - n mean(w g n))
//
// Memory is the bound: x in, y out (and x, dy in, dx out).  A team of lanes holds a
// row, 8 values (16 or 32 bytes) a lane, so that a row is loaded once, in full
// lines, and reduced by DPP moves within the team; the rotation's other half comes
// from a lane of the team.  A team takes several heads of its token, which share
// its place, the tables' values (64 bytes a lane against 16 of x) and the weights.
// Queries and keys go in one launch.  The weights' gradients are summed in registers
// by a workgroup over its tokens, and over the workgroups in a fixed order by a
// second launch.
//
// Reached: 8 x 4800 tokens, 16 and 16 heads of 64, bf16, forward 57 us (4.2 TB/s), gradients 90 and
// the sum 5 (3.9); a token 3.2 us, most of them a launch's.
#include <hip/hip_runtime.h>

#include <float.h>
#include <math.h>
#include <stdint.h>

#include "sidon_host.h"
#include "sidon_operators.h"
#include "sidon_wave.h"

#define SIDON_API extern "C" __attribute__((visibility("default")))

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kVec = 8;           // values of a lane
constexpr int kMaxBlocks = 1024;  // workgroups of a side in the backward pass: rows of partial sums
constexpr int kSumThreads = 1024, kSumCols = 16;
constexpr uint32_t kMostBlocks = (1u << 24) - 1;   // (a launch holds less than 2^32 threads)

struct Side {
  const void* x;
  const void* dy;
  void* y;              // forward: y, backward: dx
  const float* w;
  const int32_t* pos;   // [B, len], or null: 0, 1, ...
  float* part;          // [blocks, D] partial sums of dw
  float* dw;
  int64_t xb, xh, xl, gb, gh, gl, yb, yh, yl;
  uint32_t heads, len, tokens;
  uint32_t chunks;      // of NH heads of a token
  uint32_t blocks;
};

struct NormParams {
  Side side[2];
  const float* cos;
  const float* sin;
  int D, half, places;   // half: rot / 2
  int pairs;
  float eps;
};

// 8 values as they lie in memory.
template <typename E>
struct Raw {
  static constexpr int kDw = 2 * sizeof(E);
  int v[kDw];
  __device__ __forceinline__ void load(const E* at) {
#pragma unroll
    for (int i = 0; i < kDw; i += 4) {
      const i4 q = *reinterpret_cast<const i4*>(reinterpret_cast<const int*>(at) + i);
      v[i] = q[0], v[i + 1] = q[1], v[i + 2] = q[2], v[i + 3] = q[3];
    }
  }
  __device__ __forceinline__ void store(E* at) const {
#pragma unroll
    for (int i = 0; i < kDw; i += 4)
      *reinterpret_cast<i4*>(reinterpret_cast<int*>(at) + i) = i4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  }
  __device__ __forceinline__ void to(float (&f)[kVec]) const {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[i] = __builtin_bit_cast(float, v[i]);
    } else {
      typedef E e2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const e2 p = __builtin_bit_cast(e2, v[i]);
        f[2 * i] = (float)p[0], f[2 * i + 1] = (float)p[1];
      }
    }
  }
  __device__ __forceinline__ void from(const float (&f)[kVec]) {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = __builtin_bit_cast(int, f[i]);
    } else {
      typedef E e2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(int, e2{(E)f[2 * i], (E)f[2 * i + 1]});
    }
  }
  // The values of lane `from`.
  __device__ __forceinline__ Raw of(int from) const {
    Raw r;
#pragma unroll
    for (int i = 0; i < kDw; ++i) r.v[i] = __builtin_amdgcn_ds_bpermute(4 * from, v[i]);
    return r;
  }
};

// Sum over a team of LP lanes (a power of two from 2 to 32), in each of them.
template <int LP>
__device__ __forceinline__ float team_sum(float v) {
  v += sidon::dpp_mov<0xb1>(v);                          // quad_perm [1, 0, 3, 2]
  if constexpr (LP > 2) v += sidon::dpp_mov<0x4e>(v);    // quad_perm [2, 3, 0, 1]
  if constexpr (LP > 4) v += sidon::dpp_mov<0x141>(v);   // row_half_mirror
  if constexpr (LP > 8) v += sidon::dpp_mov<0x140>(v);   // row_mirror
  if constexpr (LP > 16) v += __shfl_xor(v, 16);
  return v;
}

// What a lane needs of its place in a row and of the token's place.
template <typename E>
struct Turn {
  float c[kVec], s[kVec];   // pairs: cosine and sine of value i's pair; halves: the sine with the sign of the partner's term
  int from;                 // the lane that holds the other half

  // lane: within the wavefront, i: within the team, place in [0, places).
  __device__ __forceinline__ void load(const NormParams& p, int lane, int i, int place) {
    const int at = kVec * i;
    from = lane;
    if (at >= 2 * p.half) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) c[k] = 1.f, s[k] = 0.f;
      return;
    }
    const int64_t row = (int64_t)place * p.half;
    if (p.pairs) {
      const f4 cs = *reinterpret_cast<const f4*>(p.cos + row + at / 2);
      const f4 sn = *reinterpret_cast<const f4*>(p.sin + row + at / 2);
#pragma unroll
      for (int k = 0; k < kVec; ++k) c[k] = cs[k / 2], s[k] = k % 2 == 0 ? -sn[k / 2] : sn[k / 2];
    } else {
      const bool second = at >= p.half;
      const int64_t on = row + (second ? at - p.half : at);
      from = second ? lane - p.half / kVec : lane + p.half / kVec;
      const float sign = second ? 1.f : -1.f;
#pragma unroll
      for (int k = 0; k < kVec; k += 4) {
        const f4 cs = *reinterpret_cast<const f4*>(p.cos + on + k);
        const f4 sn = *reinterpret_cast<const f4*>(p.sin + on + k);
#pragma unroll
        for (int e = 0; e < 4; ++e) c[k + e] = cs[e], s[k + e] = sign * sn[e];
      }
    }
  }
  __device__ __forceinline__ void poison() {
#pragma unroll
    for (int k = 0; k < kVec; ++k) c[k] = s[k] = __builtin_nanf("");
  }
};

// Where a team works.
struct Spot {
  bool there;        // the token has a place (a negative one: padding)
  bool known;        // and the tables have it
  int place;
  uint32_t b, l;
};

__device__ __forceinline__ Spot spot(const NormParams& p, const Side& s, uint32_t token) {
  Spot t;
  t.b = token / s.len;
  t.l = token - t.b * s.len;
  t.place = s.pos != nullptr ? s.pos[token] : (int)t.l;
  t.there = t.place >= 0;
  t.known = p.half == 0 || t.place < p.places;
  return t;
}

// 1 / sqrt(mean + eps) of squares that sum up to `sum` over the row, as f * r: f is 1,
// but for rows whose squares leave fp32, whose values are multiplied by f first.
template <int LP>
__device__ __forceinline__ void inverse_rms(const NormParams& p, float (&x)[kVec], float& f, float& r) {
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kVec; ++k) sum = fmaf(x[k], x[k], sum);
  sum = team_sum<LP>(sum);
  f = 1.f;
  const float mean = 1.f / (float)p.D;
  r = rsqrtf(sum * mean + p.eps);
  if (!(sum < FLT_MAX)) {
    // (the whole team comes here; 2^-72 of fp32's largest, squared and summed, is 2^121,
    // and eps beside values of at least 2^59 is nothing)
    f = 0x1p-72f;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      x[k] *= f;
      sum = fmaf(x[k], x[k], sum);
    }
    r = rsqrtf(team_sum<LP>(sum) * mean);
  }
}

template <typename E, int LP, int NH>
__global__ void __launch_bounds__(kThreads) head_norm_kernel(const NormParams p) {
  const bool second = blockIdx.x >= p.side[0].blocks;
  const Side& s = p.side[second ? 1 : 0];
  const uint32_t block = blockIdx.x - (second ? p.side[0].blocks : 0);
  const int lane = threadIdx.x & 63, i = threadIdx.x & (LP - 1);
  const uint32_t unit = block * (kThreads / LP) + threadIdx.x / LP;
  const uint32_t token = unit / s.chunks;
  if (token >= s.tokens) return;
  const uint32_t h0 = (unit - token * s.chunks) * NH;
  const Spot t = spot(p, s, token);
  const bool mine = kVec * i < p.D;
  const E* const xp = static_cast<const E*>(s.x) + (int64_t)t.b * s.xb + (int64_t)t.l * s.xl + kVec * i;
  E* const yp = static_cast<E*>(s.y) + (int64_t)t.b * s.yb + (int64_t)t.l * s.yl + kVec * i;

  Raw<E> raw[NH] = {};
  if (mine && t.there) {
#pragma unroll
    for (int n = 0; n < NH; ++n)
      if (h0 + n < s.heads) raw[n].load(xp + (int64_t)(h0 + n) * s.xh);
  }
  Turn<E> turn = {};
  float w[kVec] = {};
  float wo[kVec];   // of the other half
  turn.from = lane;
  if (mine && t.there) {
    turn.load(p, lane, i, t.known ? t.place : 0);
    if (!t.known && kVec * i < 2 * p.half) turn.poison();
#pragma unroll
    for (int k = 0; k < kVec; k += 4) *reinterpret_cast<f4*>(w + k) = *reinterpret_cast<const f4*>(s.w + kVec * i + k);
  }
#pragma unroll
  for (int k = 0; k < kVec; ++k)
    wo[k] = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * turn.from, __builtin_bit_cast(int, w[k])));

#pragma unroll
  for (int n = 0; n < NH; ++n) {
    if (h0 + n >= s.heads) break;   // (the whole team)
    float x[kVec], f, r, y[kVec];
    raw[n].to(x);
    inverse_rms<LP>(p, x, f, r);
    if (p.pairs) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) y[k] = x[k] * r * w[k];
#pragma unroll
      for (int k = 0; k < kVec; k += 2) {
        const float a = y[k], b = y[k + 1];
        y[k] = a * turn.c[k] + b * turn.s[k];
        y[k + 1] = b * turn.c[k + 1] + a * turn.s[k + 1];
      }
    } else {
      float o[kVec];
      raw[n].of(turn.from).to(o);
#pragma unroll
      for (int k = 0; k < kVec; ++k) y[k] = x[k] * r * w[k] * turn.c[k] + o[k] * f * r * wo[k] * turn.s[k];
    }
    if (mine) {
      if (!t.there) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) y[k] = 0.f;
      }
      Raw<E> out;
      out.from(y);
      out.store(yp + (int64_t)(h0 + n) * s.yh);
    }
  }
}

// A workgroup keeps to one chunk of heads and takes its tokens in turn.
template <typename E, int LP, int NH>
__global__ void __launch_bounds__(kThreads) head_norm_bwd_kernel(const NormParams p) {
  constexpr int kTeams = kThreads / LP;
  __shared__ float sums[kTeams][LP * kVec];
  const bool second = blockIdx.x >= p.side[0].blocks;
  const Side& s = p.side[second ? 1 : 0];
  const uint32_t block = blockIdx.x - (second ? p.side[0].blocks : 0);
  const int lane = threadIdx.x & 63, i = threadIdx.x & (LP - 1);
  const uint32_t team = threadIdx.x / LP;
  const uint32_t h0 = block % s.chunks * NH, turns = s.blocks / s.chunks;
  const bool mine = kVec * i < p.D;

  float w[kVec] = {}, dw[kVec] = {};
  if (mine) {
#pragma unroll
    for (int k = 0; k < kVec; k += 4) *reinterpret_cast<f4*>(w + k) = *reinterpret_cast<const f4*>(s.w + kVec * i + k);
  }
  for (uint32_t token = block / s.chunks * kTeams + team; token < s.tokens; token += turns * kTeams) {
    const Spot t = spot(p, s, token);
    const int64_t xo = (int64_t)t.b * s.xb + (int64_t)t.l * s.xl + kVec * i;
    const int64_t go = (int64_t)t.b * s.gb + (int64_t)t.l * s.gl + kVec * i;
    const int64_t yo = (int64_t)t.b * s.yb + (int64_t)t.l * s.yl + kVec * i;
    Raw<E> raw[NH] = {}, grad[NH] = {};
    Turn<E> turn = {};
    turn.from = lane;
    if (mine && t.there) {
#pragma unroll
      for (int n = 0; n < NH; ++n)
        if (h0 + n < s.heads) {
          raw[n].load(static_cast<const E*>(s.x) + xo + (int64_t)(h0 + n) * s.xh);
          grad[n].load(static_cast<const E*>(s.dy) + go + (int64_t)(h0 + n) * s.gh);
        }
      turn.load(p, lane, i, t.known ? t.place : 0);
      if (!t.known && kVec * i < 2 * p.half) turn.poison();
    }
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      if (h0 + n >= s.heads) break;   // (the whole team)
      float x[kVec], g[kVec], f, r;
      raw[n].to(x);
      grad[n].to(g);
      inverse_rms<LP>(p, x, f, r);
      // g = R^T dy: the sines change sign
      if (p.pairs) {
#pragma unroll
        for (int k = 0; k < kVec; k += 2) {
          const float a = g[k], b = g[k + 1];
          g[k] = a * turn.c[k] - b * turn.s[k];
          g[k + 1] = b * turn.c[k + 1] - a * turn.s[k + 1];
        }
      } else {
        float o[kVec];
        grad[n].of(turn.from).to(o);
#pragma unroll
        for (int k = 0; k < kVec; ++k) g[k] = g[k] * turn.c[k] - o[k] * turn.s[k];
      }
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        x[k] *= r;   // n
        dw[k] = fmaf(g[k], x[k], dw[k]);
        g[k] *= w[k];
        dot = fmaf(g[k], x[k], dot);
      }
      dot = team_sum<LP>(dot) / (float)p.D;
      if (mine) {
        const float rf = r * f;
#pragma unroll
        for (int k = 0; k < kVec; ++k) g[k] = t.there ? rf * (g[k] - x[k] * dot) : 0.f;
        Raw<E> out;
        out.from(g);
        out.store(static_cast<E*>(s.y) + yo + (int64_t)(h0 + n) * s.yh);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kVec; ++k) sums[team][kVec * i + k] = dw[k];
  __syncthreads();
  if ((int)threadIdx.x < p.D) {
    float sum = 0.f;
    for (int j = 0; j < kTeams; ++j) sum += sums[j][threadIdx.x];
    s.part[(int64_t)block * p.D + threadIdx.x] = sum;
  }
}

// dw of a side from its workgroups' sums: a workgroup per 16 values.
__global__ void __launch_bounds__(kSumThreads) head_norm_sum_kernel(const NormParams p) {
  constexpr int kCols = kSumCols, kRows = kSumThreads / kCols;
  __shared__ float sums[kRows][kCols];
  const Side& s = p.side[blockIdx.y];
  const int c = threadIdx.x % kCols, row = threadIdx.x / kCols;
  const int at = blockIdx.x * kCols + c;
  float sum = 0.f;
  constexpr int kAtOnce = 8;   // loads together, or each would wait for the one before
  for (uint32_t b0 = row; b0 < s.blocks; b0 += kAtOnce * kRows) {
    float v[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t b = b0 + i * kRows;
      v[i] = b < s.blocks ? s.part[(int64_t)b * p.D + at] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) sum += v[i];
  }
  sums[row][c] = sum;
  __syncthreads();
  if (row == 0) {
    sum = 0.f;
#pragma unroll 16
    for (int j = 0; j < kRows; ++j) sum += sums[j][c];
    s.dw[at] = sum;
  }
}

// ---- host -------------------------------------------------------------------------

// Lanes of a team: the power of two that holds D.
int team_lanes(int D) {
  int n = 2;
  while (n * kVec < D) n *= 2;
  return n;
}

// Heads that a team takes: several where that still leaves the chip enough wavefronts.
int team_heads(int64_t rows, int D) { return rows * team_lanes(D) / 64 >= 4 * 2048 ? 4 : 1; }

struct Blocks {
  uint32_t chunks, blocks;
};
// Workgroups of a side's backward pass.
Blocks backward_blocks(int64_t tokens, int heads, int nh, int D) {
  const int64_t teams = kThreads / team_lanes(D);
  const int64_t chunks = (heads + nh - 1) / nh;
  int64_t turns = (tokens + teams - 1) / teams;
  const int64_t most = chunks >= kMaxBlocks ? 1 : kMaxBlocks / chunks;
  const int64_t each = (turns + most - 1) / most;   // tokens of a team, the same for nearly all of them
  turns = (turns + each - 1) / each;
  return Blocks{(uint32_t)chunks, (uint32_t)(chunks * turns)};
}

bool sizes_ok(int B, int heads, int len) {
  return heads >= 1 && heads <= 4096 && len >= 1 && (int64_t)B * heads * len <= INT32_MAX / 2;
}

template <typename E, int LP>
void launch_nh(const NormParams& p, int nh, bool backward, uint32_t blocks, hipStream_t stream) {
  if (backward) {
    if (nh == 4)
      hipLaunchKernelGGL((head_norm_bwd_kernel<E, LP, 4>), dim3(blocks), dim3(kThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((head_norm_bwd_kernel<E, LP, 1>), dim3(blocks), dim3(kThreads), 0, stream, p);
  } else {
    if (nh == 4)
      hipLaunchKernelGGL((head_norm_kernel<E, LP, 4>), dim3(blocks), dim3(kThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((head_norm_kernel<E, LP, 1>), dim3(blocks), dim3(kThreads), 0, stream, p);
  }
}

template <typename E>
void launch(const NormParams& p, int nh, bool backward, uint32_t blocks, hipStream_t stream) {
  switch (team_lanes(p.D)) {
    case 2: return launch_nh<E, 2>(p, nh, backward, blocks, stream);
    case 4: return launch_nh<E, 4>(p, nh, backward, blocks, stream);
    case 8: return launch_nh<E, 8>(p, nh, backward, blocks, stream);
    case 16: return launch_nh<E, 16>(p, nh, backward, blocks, stream);
    default: return launch_nh<E, 32>(p, nh, backward, blocks, stream);
  }
}

// What both directions check and set alike.  x, y (and dy) per side; a side with
// heads == 0 is not there.
struct SideArgs {
  const void* x;
  const void* dy;
  void* y;
  const float* w;
  float* dw;
  const int32_t* pos;
  const int64_t* xs;
  const int64_t* gs;
  const int64_t* ys;
  int heads, len;
};

int prepare(NormParams& p, const SideArgs (&a)[2], bool backward, const float* cos, const float* sin, int places,
            int rot, int pairs, float eps, int B, int D, int dtype, void* ws, size_t need) {
  using sidon::fail;
  using sidon::Rows;
  if (dtype != SIDON_FP32 && dtype != SIDON_FP16 && dtype != SIDON_BF16)
    return fail(SIDON_E_SHAPE, "dtype=%d is none of SIDON_FP32, SIDON_FP16, SIDON_BF16", dtype);
  if (B < 1 || D < 16 || D > 256 || D % 16 != 0 || rot < 0 || rot > D || rot % 16 != 0)
    return fail(SIDON_E_SHAPE, "B=%d D=%d rot=%d: need B >= 1, D a multiple of 16 in [16, 256], rot one in [0, D]", B, D, rot);
  if (!(eps >= FLT_MIN) || !(eps <= FLT_MAX)) return fail(SIDON_E_SHAPE, "eps=%g must be positive and finite", eps);
  if (rot > 0 && (cos == nullptr || sin == nullptr)) return fail(SIDON_E_NULL, "cos and sin must be non-NULL with rot=%d", rot);
  if (rot > 0 && places < 1) return fail(SIDON_E_SHAPE, "places=%d must be positive", places);
  if (!sidon::aligned16(cos) || !sidon::aligned16(sin)) return fail(SIDON_E_ALIGN, "cos and sin must be 16-byte aligned");
  const int size = dtype == SIDON_FP32 ? 4 : 2, unit = 16 / size;
  struct Piece {
    const char* name;
    Rows rows;
    bool written;
  };
  Piece piece[6];
  struct Flat {
    const char* name;
    const void* at;
    int64_t bytes;
    bool written;
  };
  Flat flat[9];
  int pieces = 0, flats = 0;
  const __int128 most = (__int128)1 << 61;
  static const char* const names[2][7] = {{"q", "the gradient of q's output", "q's output", "q_w", "dq_w", "q_pos", "q"},
                                          {"k", "the gradient of k's output", "k's output", "k_w", "dk_w", "k_pos", "k"}};
  for (int i = 0; i < 2; ++i) {
    const SideArgs& t = a[i];
    if (t.heads == 0 && i == 1) continue;
    if (t.x == nullptr || t.y == nullptr || t.w == nullptr || t.xs == nullptr || t.ys == nullptr ||
        (backward && (t.dy == nullptr || t.gs == nullptr || t.dw == nullptr)))
      return fail(SIDON_E_NULL, "%s, its output, weights and strides must be non-NULL", names[i][0]);
    if (!sizes_ok(B, t.heads, t.len))
      return fail(SIDON_E_SHAPE, "%s: heads=%d len=%d: need 1 <= heads <= 4096, len >= 1, B * heads * len < 2^30", names[i][0], t.heads, t.len);
    if (rot > 0 && t.pos == nullptr && t.len > places)
      return fail(SIDON_E_SHAPE, "%s has %d tokens, the tables have %d places", names[i][0], t.len, places);
    const int64_t* const st[3] = {t.xs, t.gs, t.ys};
    const void* const at[3] = {t.x, t.dy, t.y};
    for (int k = 0; k < 3; ++k) {
      if (k == 1 && !backward) continue;
      for (int d = 0; d < 3; ++d)
        if (st[k][d] < 0 || st[k][d] % unit != 0 || st[k][d] > (int64_t)1 << 40)
          return fail(SIDON_E_STRIDE, "%s stride %lld (number %d) must be a multiple of %d in [0, 2^40]", names[i][k],
                      (long long)st[k][d], d, unit);
      if (!sidon::aligned16(at[k])) return fail(SIDON_E_ALIGN, "%s must be 16-byte aligned", names[i][k]);
      const Rows rows{at[k], {B, t.heads, t.len}, {st[k][0], st[k][1], st[k][2]}, D, size};
      if (rows.bytes() > most) return fail(SIDON_E_STRIDE, "%s spans more than the address space", names[i][k]);
      if (k == 2 && !sidon::apart(rows.n, rows.st, 3, D)) return fail(SIDON_E_STRIDE, "rows of %s overlap one another", names[i][k]);
      piece[pieces++] = Piece{names[i][k], rows, k == 2};
    }
    if (!sidon::aligned16(t.w)) return fail(SIDON_E_ALIGN, "%s must be 16-byte aligned", names[i][3]);
    if (((reinterpret_cast<uintptr_t>(t.pos) | reinterpret_cast<uintptr_t>(t.dw)) & 3u) != 0)
      return fail(SIDON_E_ALIGN, "%s and %s must be 4-byte aligned", names[i][5], names[i][4]);
    flat[flats++] = Flat{names[i][3], t.w, (int64_t)4 * D, false};
    if (t.pos != nullptr) flat[flats++] = Flat{names[i][5], t.pos, (int64_t)4 * B * t.len, false};
    if (backward) flat[flats++] = Flat{names[i][4], t.dw, (int64_t)4 * D, true};
  }
  if (rot > 0) {
    flat[flats++] = Flat{"cos", cos, (int64_t)2 * rot * places, false};
    flat[flats++] = Flat{"sin", sin, (int64_t)2 * rot * places, false};
  }
  if (need > 0) flat[flats++] = Flat{"ws", ws, (int64_t)need, true};
  // A team reads a row before it writes it, so an output may be the very tensor that
  // its own side reads; any other shared memory is refused.
  for (int i = 0; i < pieces; ++i) {
    for (int j = i + 1; j < pieces; ++j) {
      const Piece &x = piece[i], &y = piece[j];
      if (!x.written && !y.written) continue;
      const int per = backward ? 3 : 2;
      bool same = i / per == j / per && x.rows.at == y.rows.at;
      for (int d = 0; d < 3; ++d) same = same && (x.rows.st[d] == y.rows.st[d] || x.rows.n[d] == 1);
      if (!same && sidon::tensors_meet(x.rows, y.rows)) return fail(SIDON_E_SHAPE, "%s must lie apart from %s", y.name, x.name);
    }
    for (int j = 0; j < flats; ++j) {
      const Flat& f = flat[j];
      if (!piece[i].written && !f.written) continue;
      const Rows whole{f.at, {1, 1, 1}, {0, 0, 0}, (int)(f.bytes < INT32_MAX ? f.bytes : INT32_MAX), 1};
      if (f.bytes < INT32_MAX ? sidon::tensors_meet(piece[i].rows, whole)
                              : sidon::ranges_meet(piece[i].rows.at, (int64_t)piece[i].rows.bytes(), f.at, f.bytes))
        return fail(SIDON_E_SHAPE, "%s must lie apart from %s", piece[i].written ? piece[i].name : f.name,
                    piece[i].written ? f.name : piece[i].name);
    }
  }
  for (int i = 0; i < flats; ++i)
    for (int j = i + 1; j < flats; ++j)
      if ((flat[i].written || flat[j].written) && sidon::ranges_meet(flat[i].at, flat[i].bytes, flat[j].at, flat[j].bytes))
        return fail(SIDON_E_SHAPE, "%s must lie apart from %s", flat[j].name, flat[i].name);
  p = NormParams{};
  p.cos = cos, p.sin = sin;
  p.D = D, p.half = rot / 2, p.places = places, p.pairs = pairs != 0, p.eps = eps;
  for (int i = 0; i < 2; ++i) {
    const SideArgs& t = a[i];
    if (t.heads == 0) continue;
    Side& s = p.side[i];
    s.x = t.x, s.dy = t.dy, s.y = t.y, s.w = t.w, s.dw = t.dw, s.pos = t.pos;
    s.xb = t.xs[0], s.xh = t.xs[1], s.xl = t.xs[2], s.yb = t.ys[0], s.yh = t.ys[1], s.yl = t.ys[2];
    if (backward) s.gb = t.gs[0], s.gh = t.gs[1], s.gl = t.gs[2];
    s.heads = (uint32_t)t.heads, s.len = (uint32_t)t.len, s.tokens = (uint32_t)B * (uint32_t)t.len;
  }
  return SIDON_OK;
}

int heads_of_teams(int B, int H, int Hk, int L, int S, int D) {
  return team_heads((int64_t)B * ((int64_t)H * L + (int64_t)Hk * S), D);
}

void launch_any(const NormParams& p, int nh, bool backward, uint32_t blocks, int dtype, hipStream_t s) {
  if (dtype == SIDON_FP32) return launch<float>(p, nh, backward, blocks, s);
  if (dtype == SIDON_FP16) return launch<_Float16>(p, nh, backward, blocks, s);
  return launch<__bf16>(p, nh, backward, blocks, s);
}

}  // namespace

SIDON_API int sidon_qk_norm_rotary(const void* q, const void* k, void* q_out, void* k_out, const float* q_w,
                                   const float* k_w, const float* cos, const float* sin, int places, int rot,
                                   int interleaved, const int32_t* q_pos, const int32_t* k_pos, float eps, int B, int H,
                                   int Hk, int L, int S, int D, int dtype, const int64_t* q_strides,
                                   const int64_t* k_strides, const int64_t* q_out_strides,
                                   const int64_t* k_out_strides, sidon_stream_t stream) {
  sidon::clear_error();
  const SideArgs a[2] = {{q, nullptr, q_out, q_w, nullptr, q_pos, q_strides, nullptr, q_out_strides, H, L},
                         {k, nullptr, k_out, k_w, nullptr, k_pos, k_strides, nullptr, k_out_strides, Hk, S}};
  NormParams p;
  int rc = prepare(p, a, false, cos, sin, places, rot, interleaved, eps, B, D, dtype, nullptr, 0);
  if (rc != SIDON_OK || (rc = sidon::check_device())) return rc;
  const int nh = heads_of_teams(B, H, Hk, L, Hk == 0 ? 0 : S, D);
  const int64_t teams = kThreads / team_lanes(D);
  uint32_t blocks = 0;
  for (Side& s : p.side) {
    s.chunks = (s.heads + nh - 1) / nh;
    s.blocks = (uint32_t)(((int64_t)s.tokens * s.chunks + teams - 1) / teams);
    blocks += s.blocks;
  }
  if (blocks > kMostBlocks) return sidon::fail(SIDON_E_SHAPE, "too many rows for one launch");
  launch_any(p, nh, false, blocks, dtype, reinterpret_cast<hipStream_t>(stream));
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return sidon::fail(SIDON_E_LAUNCH, "norm and rotation launch failed: %s", hipGetErrorString(err));
  return SIDON_OK;
}

SIDON_API size_t sidon_qk_norm_rotary_workspace_bytes(int B, int H, int Hk, int L, int S, int D) {
  if (B < 1 || D < 16 || D > 256 || D % 16 != 0 || !sizes_ok(B, H, L) || (Hk != 0 && !sizes_ok(B, Hk, S))) return 0;
  if (Hk == 0) S = 0;
  const int nh = heads_of_teams(B, H, Hk, L, S, D);
  size_t rows = backward_blocks((int64_t)B * L, H, nh, D).blocks;
  if (Hk != 0) rows += backward_blocks((int64_t)B * S, Hk, nh, D).blocks;
  return rows * D * 4;
}

SIDON_API int sidon_qk_norm_rotary_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k, void* dq,
                                       void* dk, float* dq_w, float* dk_w, const float* q_w, const float* k_w,
                                       const float* cos, const float* sin, int places, int rot, int interleaved,
                                       const int32_t* q_pos, const int32_t* k_pos, float eps, void* ws, size_t ws_bytes,
                                       int B, int H, int Hk, int L, int S, int D, int dtype,
                                       const int64_t* dq_out_strides, const int64_t* dk_out_strides,
                                       const int64_t* q_strides, const int64_t* k_strides, const int64_t* dq_strides,
                                       const int64_t* dk_strides, sidon_stream_t stream) {
  using sidon::fail;
  sidon::clear_error();
  const SideArgs a[2] = {{q, dq_out, dq, q_w, dq_w, q_pos, q_strides, dq_out_strides, dq_strides, H, L},
                         {k, dk_out, dk, k_w, dk_w, k_pos, k_strides, dk_out_strides, dk_strides, Hk, S}};
  const size_t need = sidon_qk_norm_rotary_workspace_bytes(B, H, Hk, L, S, D);
  if (need > 0 && ws == nullptr) return fail(SIDON_E_NULL, "ws must be non-NULL");
  if (!sidon::aligned16(ws)) return fail(SIDON_E_ALIGN, "ws must be 16-byte aligned");
  NormParams p;
  int rc = prepare(p, a, true, cos, sin, places, rot, interleaved, eps, B, D, dtype, ws, need);
  if (rc != SIDON_OK) return rc;
  if (ws_bytes < need) return fail(SIDON_E_SHAPE, "ws holds %zu bytes, the call needs %zu", ws_bytes, need);
  if ((rc = sidon::check_device())) return rc;
  const int nh = heads_of_teams(B, H, Hk, L, Hk == 0 ? 0 : S, D);
  float* part = static_cast<float*>(ws);
  uint32_t blocks = 0;
  for (Side& s : p.side) {
    if (s.heads == 0) continue;
    const Blocks c = backward_blocks(s.tokens, (int)s.heads, nh, D);
    s.chunks = c.chunks, s.blocks = c.blocks;
    s.part = part;
    part += (size_t)s.blocks * D;
    blocks += s.blocks;
  }
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  launch_any(p, nh, true, blocks, dtype, st);
  hipLaunchKernelGGL(head_norm_sum_kernel, dim3(D / kSumCols, Hk == 0 ? 1 : 2), dim3(kSumThreads), 0, st, p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(SIDON_E_LAUNCH, "norm and rotation gradient launch failed: %s", hipGetErrorString(err));
  return SIDON_OK;
}
