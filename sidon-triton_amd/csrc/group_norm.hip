// group_norm.hip -- group norm with an activation, channels last, over the
// valid rows of B items (MI355X / gfx950):
//
//   y = act((x - mean_bg) * rsqrt(var_bg + eps) * w_c + bias_c)
//
// with mean and variance over an item's rows t < lens[b] and the C / G
// channels of a group.  Memory bound: the floor is x once and y once.
//
// Two ways through it:
//
//   slab     one workgroup owns a whole (item, group), keeps its values in
//            registers between the statistics and the store: one launch, x
//            read once.  For groups whose rows fit a workgroup's registers.
//   passes   workgroups over row chunks leave (mean, M2) per group, a second
//            launch joins them and writes y: x read twice.
//
// Measured, whole calls in a graph: 1 x 150 x 1024 fp16 in 32 groups 4.4 us (slab: one
// launch, a few memory latencies), 3 x 1463 x 1024 bf16 in 16 groups with GELU 14 us
// (passes: two launches, the second's arithmetic), 8 x 4800 x 1024 fp32 in 32 groups
// 83-87 us on the same x again and again, which the Infinity Cache holds half of, 106-108
// on another x each time (passes: x twice and y once at 4.4 TB/s; a copy of x takes 63).
//
// Statistics never form a difference of large sums: every thread takes the
// mean of what it holds and the squares around that mean, and partial results
// (n, mean, M2) are joined by  M2 = sum M2_i + n_i (mean_i - mean)^2, in fp32, the
// count multiplied in before the square: one of 0 leaves 0 also where the square
// of a mean past 2^63 would be infinite.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "sidon_host.h"
#include "sidon_operators.h"
#include "sidon_wave.h"

#define SIDON_API extern "C" __attribute__((visibility("default")))
#define SIDON_INLINE __attribute__((always_inline))

namespace {

constexpr int kMaxC = 8192;
constexpr int kThreads = 256;      // of the two-pass kernels
constexpr int kMaxChunks = 64;     // row chunks per item that the second pass joins
constexpr int kBlockVecs = 32;     // vectors per row of a column block, or one group
constexpr int kStatWgs = 1024;     // workgroups a statistics launch aims for
constexpr int kApplyWgs = 2048;
constexpr int kSlabThreads = 1024;
constexpr int kSlabVecs = 16;      // 16-byte vectors per thread that a slab may take

struct Params {
  const void* x;
  const int32_t* lens;
  const float* w;
  const float* bias;
  void* y;
  float2* part;   // [B, chunks, G] (mean, M2)
  int64_t ldx, ldy;
  float eps;
  int B, T, C, G, act;
  int block_groups;                 // groups per column block of the two passes
  int chunks, rows_per_chunk;       // statistics
  int apply_rows;                   // rows per workgroup of the second pass
};

template <typename T, int V>
struct Vec {
  typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct Vec<T, 1> {
  typedef T type;
};

// V elements at p (aligned to their size) as fp32, and back with one rounding.
template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  const typename Vec<T, V>::type r = *reinterpret_cast<const typename Vec<T, V>::type*>(p);
  if constexpr (V == 1) {
    v[0] = (float)r;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)r[e];
  }
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  typename Vec<T, V>::type r;
  if constexpr (V == 1) {
    r = (T)v[0];
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) r[e] = (T)v[e];
  }
  *reinterpret_cast<typename Vec<T, V>::type*>(p) = r;
}

// erfc(z) for z >= 0: e^(-z^2) times a polynomial in t = 1 / (1 + 0.4 z), fitted
// to erfc(z) e^(z^2) over [0, 40] for the least relative error (1.3e-7, 3e-7
// with fp32 arithmetic).  erfcf costs a memory-bound kernel three times as much
// arithmetic (1463 x 64 values of bf16 on a CU: 27 us against 15 with SiLU).
__device__ __forceinline__ float erfc_positive(float z) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.4f, z, 1.f));
  float c = 0.0500626639f;
  c = fmaf(c, t, -0.182005256f);
  c = fmaf(c, t, 0.167402819f);
  c = fmaf(c, t, -0.00389658613f);
  c = fmaf(c, t, 0.140410721f);
  c = fmaf(c, t, 0.168903336f);
  c = fmaf(c, t, 0.207769737f);
  c = fmaf(c, t, 0.225677118f);
  c = fmaf(c, t, 0.225675568f);
  return c * t * __expf(-z * z);
}

// kExact: results kept in fp32, where the hardware exponential's and
// reciprocal's error (about |v| 2^-24) would show; 16-bit results hide it.
template <bool kExact, int V>
__device__ __forceinline__ void activate(float (&v)[V], int act) {
  if (act == SIDON_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      v[e] = kExact ? v[e] / (1.f + expf(-v[e])) : v[e] * __builtin_amdgcn_rcpf(1.f + __expf(-v[e]));
  } else if (act == SIDON_ACT_GELU) {
    // v / 2 erfc(-v / sqrt 2): erfc keeps the far negative side's digits, where 1 + erf loses them
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (kExact) {
        v[e] *= 0.5f * erfcf(-0.70710678118654752f * v[e]);
      } else {
        const float half = 0.5f * erfc_positive(0.70710678118654752f * fabsf(v[e]));
        v[e] *= v[e] < 0.f ? half : 1.f - half;
      }
    }
  } else if (act == SIDON_ACT_RELU) {
    // (a comparison, so that NaN stays NaN)
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
  }
}

// Keeps what is computed from r on either side of this apart: without it the
// compiler keeps a slab's fp32 values live between its passes, twice the
// registers (181 of them spilled at 16 vectors of fp16 a thread).
template <typename R>
__device__ __forceinline__ void opaque(R& r) {
  typedef int int4_t __attribute__((ext_vector_type(4)));
  static_assert(sizeof(R) == sizeof(int4_t), "16-byte vectors");
  int4_t v = __builtin_bit_cast(int4_t, r);
  asm volatile("" : "+v"(v));
  r = __builtin_bit_cast(R, v);
}

__device__ __forceinline__ int valid_rows(const Params& p, int b) {
  return p.lens == nullptr ? p.T : min(max(p.lens[b], 0), p.T);
}

// ---- slab -------------------------------------------------------------------------

// TH threads hold TH x NV vectors of 16 bytes: all T rows of one group.
// Neighbouring groups share cache lines where a group's row is under 128
// bytes, so each XCD (workgroups go round-robin over the 8) takes a contiguous
// range of groups.
template <typename T, int NV, int TH>
__global__ void __launch_bounds__(TH) gn_slab_kernel(const Params p) {
  constexpr int V = 16 / sizeof(T);
  constexpr int kWaves = TH / 64;
  __shared__ float red[2][kWaves];
  const int xcd = blockIdx.x & 7, per = gridDim.x >> 3, rem = gridDim.x & 7;
  const int lin = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + ((int)blockIdx.x >> 3);
  const int b = lin / p.G;
  const int g = lin - b * p.G;
  const int cg = p.C / p.G;
  const int vpr = cg / V;
  const int n = valid_rows(p, b);
  const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.T * p.ldx + g * cg;
  T* y = static_cast<T*>(p.y) + (int64_t)b * p.T * p.ldy + g * cg;

  // Vector j of a thread: number threadIdx.x + TH j of the slab.
  const int row0 = (int)threadIdx.x / vpr, col0 = (int)threadIdx.x - row0 * vpr;
  const int drow = TH / vpr, dcol = TH - drow * vpr;
  typedef typename Vec<T, V>::type vec_t;
  vec_t raw[NV];
  {
    int row = row0, col = col0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      raw[j] = vec_t{};
      if (row < n) raw[j] = *reinterpret_cast<const vec_t*>(x + row * p.ldx + col * V);
      row += drow;
      col += dcol;
      if (col >= vpr) {
        col -= vpr;
        ++row;
      }
    }
  }
  auto block_sum = [&](float v, int which) SIDON_INLINE {
    v = sidon::wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[which][threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += red[which][i];
    return s;
  };
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) sum += (float)raw[j][e];
  const float inv = n > 0 ? 1.f / ((float)n * (float)cg) : 0.f;
  const float mean = block_sum(sum, 0) * inv;
  float sq = 0.f;
  {
    int row = row0, col = col0;
    asm volatile("" : "+v"(row), "+v"(col));   // (the same for the indices)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      opaque(raw[j]);
      if (row < n) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = (float)raw[j][e] - mean;
          sq = fmaf(d, d, sq);
        }
      }
      row += drow;
      col += dcol;
      if (col >= vpr) {
        col -= vpr;
        ++row;
      }
    }
  }
  const float rstd = rsqrtf(block_sum(sq, 1) * inv + p.eps);
  int row = row0, col = col0;
  asm volatile("" : "+v"(row), "+v"(col));
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (row < p.T) {
      float v[V] = {};
      if (row < n) {
        opaque(raw[j]);
        float w[V], bias[V];
        load<float, V>(p.w + g * cg + col * V, w);
        load<float, V>(p.bias + g * cg + col * V, bias);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = fmaf(((float)raw[j][e] - mean) * rstd, w[e], bias[e]);
        activate<sizeof(T) == 4, V>(v, p.act);
      }
      store<T, V>(y + row * p.ldy + col * V, v);
    }
    row += drow;
    col += dcol;
    if (col >= vpr) {
      col -= vpr;
      ++row;
    }
  }
}

// ---- two passes -------------------------------------------------------------------

// Lanes of a power-of-two team (of consecutive lanes of a wavefront).
__device__ __forceinline__ float team_sum(float v, int team) {
  for (int o = team >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The threads of a workgroup over C channels: a thread owns one vector of V
// columns and every `lanes`-th row (or, past kThreads vectors, a vector per
// pass and every row).
struct Layout {
  int nv, lanes, passes;
};
template <int V>
__device__ __forceinline__ Layout layout(int C) {
  Layout l;
  l.nv = C / V;
  l.lanes = l.nv < kThreads ? kThreads / l.nv : 1;
  l.passes = (l.nv + kThreads - 1) / kThreads;
  return l;
}

// Team size for G groups on the workgroup's threads: all of them busy.
__device__ __forceinline__ int team_size(int G) {
  int t = 64;
  while (t > 1 && t * G > kThreads) t >>= 1;
  return t;
}

// The columns of block blockIdx.z: whole groups, whole vectors.
struct Block {
  int g0, groups, c0, cols;
};
__device__ __forceinline__ Block column_block(const Params& p) {
  Block k;
  const int cg = p.C / p.G;
  k.g0 = (int)blockIdx.z * p.block_groups;
  k.groups = min(p.block_groups, p.G - k.g0);
  k.c0 = k.g0 * cg;
  k.cols = k.groups * cg;
  return k;
}

// (mean, M2) of each group over the rows of chunk blockIdx.x of item
// blockIdx.y.  A unit is what a thread keeps one (mean, M2) for: its whole
// vector where the vector lies in one group (kWide), else a channel.
template <typename T, int V, bool kWide>
__global__ void __launch_bounds__(kThreads) gn_stat_kernel(const Params p) {
  constexpr int U = kWide ? 1 : V;
  constexpr int kPer = kWide ? V : 1;        // values per row of a unit
  constexpr int NB = V == 1 ? 16 : 8;        // rows held at once
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float2* unit = reinterpret_cast<float2*>(smem);
  const int b = blockIdx.y;
  const int r0 = blockIdx.x * p.rows_per_chunk;
  const int r1 = min(r0 + p.rows_per_chunk, valid_rows(p, b));
  if (r0 >= r1) return;   // the second pass counts the rows itself
  const Block k = column_block(p);
  const Layout l = layout<V>(k.cols);
  const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.T * p.ldx + k.c0;
  const int lr = l.passes == 1 ? (int)threadIdx.x / l.nv : 0;
  for (int pass = 0; pass < l.passes; ++pass) {
    const int vec = l.passes == 1 ? (int)threadIdx.x - lr * l.nv : pass * kThreads + (int)threadIdx.x;
    if (lr >= l.lanes || vec >= l.nv) continue;
    const T* xc = x + vec * V;
    float mean[U] = {}, m2[U] = {};
    float have = 0.f;   // values per unit so far
    for (int r = r0 + lr; r < r1; r += NB * l.lanes) {
      typedef typename Vec<T, V>::type vec_t;
      float v[NB][V];
      int rows = 0;
      vec_t raw[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int row = r + i * l.lanes;
        raw[i] = vec_t{};
        if (row < r1) {
          raw[i] = *reinterpret_cast<const vec_t*>(xc + row * p.ldx);
          ++rows;
        }
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        if constexpr (V == 1) {
          v[i][0] = (float)raw[i];
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) v[i][e] = (float)raw[i][e];
        }
      }
      const float more = (float)(rows * kPer);
      const float inv = 1.f / more;
      const float frac = more / (have + more);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < kPer; ++e) s += v[i][u * kPer + e];
        const float m = s * inv;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          if (i < rows) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
              const float d = v[i][u * kPer + e] - m;
              q = fmaf(d, d, q);
            }
          }
        }
        const float delta = m - mean[u];
        mean[u] = fmaf(delta, frac, mean[u]);
        m2[u] += q + delta * (delta * (have * frac));
      }
      have += more;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) unit[(lr * l.nv + vec) * U + u] = make_float2(mean[u], m2[u]);
  }
  __syncthreads();
  // Join a group's units: per row lane, `cols` of them side by side.
  const int cols = l.nv * U / k.groups;
  const int stride = l.nv * U;
  const int cnt_rows = r1 - r0;
  const int team = team_size(k.groups);
  const int tl = (int)threadIdx.x & (team - 1);
  const float inv_n = 1.f / ((float)cnt_rows * (float)(p.C / p.G));
  float2* out = p.part + ((int64_t)b * p.chunks + blockIdx.x) * p.G + k.g0;
  for (int g = (int)threadIdx.x / team; g < k.groups; g += kThreads / team) {
    // Unit u of the group: row lane u / cols, column u % cols.  A lane beyond the
    // chunk's rows kept nothing: its count is 0.
    const auto count = [&](int lane) { return (float)((cnt_rows - lane + l.lanes - 1) / l.lanes * kPer); };
    float s = 0.f;
    for (int u = tl; u < l.lanes * cols; u += team) {
      const int i = u / cols;
      s = fmaf(unit[i * stride + g * cols + u - i * cols].x, count(i), s);
    }
    const float mean = team_sum(s, team) * inv_n;
    float q = 0.f;
    for (int u = tl; u < l.lanes * cols; u += team) {
      const int i = u / cols;
      const float2 v = unit[i * stride + g * cols + u - i * cols];
      const float d = v.x - mean;
      q += fmaf(d, d * count(i), v.y);
    }
    const float m2 = team_sum(q, team);
    if (tl == 0) out[g] = make_float2(mean, m2);
  }
}

// Join the chunks' statistics of item blockIdx.y, then y for apply_rows rows.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) gn_apply_kernel(const Params p) {
  constexpr int NB = V == 1 ? 8 : 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float2* stat = reinterpret_cast<float2*>(smem);   // of the block's groups: (mean, rstd)
  const int b = blockIdx.y;
  const int r0 = blockIdx.x * p.apply_rows;
  const int r1 = min(r0 + p.apply_rows, p.T);
  const int n = valid_rows(p, b);
  const int cg = p.C / p.G;
  const Block k = column_block(p);
  if (r0 < n) {
    const int used = (n + p.rows_per_chunk - 1) / p.rows_per_chunk;
    const int team = team_size(k.groups);
    const int tl = (int)threadIdx.x & (team - 1);
    const float2* part = p.part + (int64_t)b * p.chunks * p.G + k.g0;
    const float inv_n = 1.f / ((float)n * (float)cg);
    for (int g = (int)threadIdx.x / team; g < k.groups; g += kThreads / team) {
      float s = 0.f;
#pragma unroll 4
      for (int c = tl; c < used; c += team) {
        const float cnt = (float)(min(p.rows_per_chunk, n - c * p.rows_per_chunk)) * (float)cg;
        s = fmaf(part[(int64_t)c * p.G + g].x, cnt, s);
      }
      const float mean = team_sum(s, team) * inv_n;
      float q = 0.f;
#pragma unroll 4
      for (int c = tl; c < used; c += team) {
        const float cnt = (float)(min(p.rows_per_chunk, n - c * p.rows_per_chunk)) * (float)cg;
        const float2 v = part[(int64_t)c * p.G + g];
        const float d = v.x - mean;
        q += fmaf(d, d * cnt, v.y);
      }
      const float var = team_sum(q, team) * inv_n;
      if (tl == 0) stat[g] = make_float2(mean, rsqrtf(var + p.eps));
    }
  }
  __syncthreads();
  const Layout l = layout<V>(k.cols);
  const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.T * p.ldx + k.c0;
  T* y = static_cast<T*>(p.y) + (int64_t)b * p.T * p.ldy + k.c0;
  const int lr = l.passes == 1 ? (int)threadIdx.x / l.nv : 0;
  for (int pass = 0; pass < l.passes; ++pass) {
    const int vec = l.passes == 1 ? (int)threadIdx.x - lr * l.nv : pass * kThreads + (int)threadIdx.x;
    if (lr >= l.lanes || vec >= l.nv) continue;
    float mean[V], w[V], bias[V];   // w: times rstd
    if (r0 < n) {
      load<float, V>(p.w + k.c0 + vec * V, w);
      load<float, V>(p.bias + k.c0 + vec * V, bias);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 s = stat[(vec * V + e) / cg];
        mean[e] = s.x;
        w[e] *= s.y;
      }
    }
    for (int r = r0 + lr; r < r1; r += NB * l.lanes) {
      float v[NB][V];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int row = r + i * l.lanes;
        if (row < r1 && row < n) load<T, V>(x + row * p.ldx + vec * V, v[i]);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int row = r + i * l.lanes;
        if (row >= r1) break;
        if (row < n) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[i][e] = fmaf(v[i][e] - mean[e], w[e], bias[e]);
          activate<sizeof(T) == 4, V>(v[i], p.act);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) v[i][e] = 0.f;
        }
        store<T, V>(y + row * p.ldy + vec * V, v[i]);
      }
    }
  }
}

// ---- host -------------------------------------------------------------------------

int element_size(int dtype) { return dtype == SIDON_FP32 ? 4 : 2; }

// Column blocks of whole groups and about kBlockVecs vectors: whole cache
// lines per row, and only these groups' partial results to join.  Row chunks:
// enough workgroups to fill the chip, a few rows per thread at least, at most
// kMaxChunks for the second pass to join.  (With all columns in a block and 128
// chunks, joining 128 x 32 groups in every workgroup of the second pass took
// as long as its rows: 1 x 4800 x 1024 fp16 21 us against 16.)
void plan_passes(Params& p, int vec) {
  const int cg = p.C / p.G;
  int step = 1;   // groups whose channels are whole vectors
  while (step * cg % vec != 0) ++step;
  int groups = (kBlockVecs * vec + cg * step - 1) / (cg * step) * step;
  if (groups > p.G) groups = p.G;
  p.block_groups = groups;
  const int blocks = (p.G + groups - 1) / groups;
  const int nv = groups * cg / vec;
  const int lanes = nv < kThreads ? kThreads / nv : 1;
  const auto split = [&](int wgs, int rows, int most) {
    int64_t n = wgs / ((int64_t)p.B * blocks);
    const int64_t cap = (p.T + rows * lanes - 1) / (rows * lanes);
    if (n > cap) n = cap;
    if (n > most) n = most;
    if (n < 1) n = 1;
    return (int)((p.T + n - 1) / n);
  };
  p.rows_per_chunk = split(kStatWgs, 8, kMaxChunks);
  p.chunks = (p.T + p.rows_per_chunk - 1) / p.rows_per_chunk;
  p.apply_rows = split(kApplyWgs, 4, 65535);
}

// LDS of the statistics launch: the units of every thread that has a vector, in
// the full column blocks or in a last, narrower one, which leaves the threads more
// row lanes (33 vectors: 7 lanes, 231 threads; 3 vectors: 85 lanes, 255).
size_t unit_bytes(const Params& p, int vec) {
  const int cg = p.C / p.G;
  const auto vectors = [&](int groups) {
    const int nv = groups * cg / vec;
    return nv < kThreads ? kThreads / nv * nv : nv;
  };
  const int full = vectors(p.block_groups), last = vectors(p.G - (p.G - 1) / p.block_groups * p.block_groups);
  return (size_t)(full > last ? full : last) * (cg % vec == 0 ? 1 : vec) * sizeof(float2);
}

template <typename T, int NV, int TH>
void slab_launch(const Params& p, hipStream_t stream) {
  hipLaunchKernelGGL((gn_slab_kernel<T, NV, TH>), dim3((unsigned)(p.B * p.G)), dim3(TH), 0, stream, p);
}

template <typename T>
void slab(const Params& p, int64_t vecs, hipStream_t stream) {
  if (vecs <= 256 * 4) {
    slab_launch<T, 4, 256>(p, stream);
  } else if (vecs <= 1024 * 4) {
    slab_launch<T, 4, 1024>(p, stream);
  } else if (vecs <= 1024 * 8) {
    slab_launch<T, 8, 1024>(p, stream);
  } else {
    slab_launch<T, kSlabVecs, kSlabThreads>(p, stream);
  }
}

template <typename T, int V>
void passes(const Params& p, hipStream_t stream) {
  const bool wide = (p.C / p.G) % V == 0;
  const size_t units = unit_bytes(p, V);
  const unsigned blocks = (unsigned)((p.G + p.block_groups - 1) / p.block_groups);
  const dim3 grid((unsigned)p.chunks, (unsigned)p.B, blocks);
  if (wide) {
    hipLaunchKernelGGL((gn_stat_kernel<T, V, true>), grid, dim3(kThreads), units, stream, p);
  } else {
    hipLaunchKernelGGL((gn_stat_kernel<T, V, false>), grid, dim3(kThreads), units, stream, p);
  }
  hipLaunchKernelGGL((gn_apply_kernel<T, V>), 
                     dim3((unsigned)((p.T + p.apply_rows - 1) / p.apply_rows), (unsigned)p.B, blocks), dim3(kThreads),
                     (size_t)p.block_groups * sizeof(float2), stream, p);
}

// Whether the slab way is taken, for elements of `size` bytes; `vector`: the tensors
// lie on 16 bytes.
bool slab_way(const Params& p, int size, bool vector) {
  const int v = 16 / size, cg = p.C / p.G;
  const int64_t vecs = (int64_t)p.T * (cg / v);
  // A workgroup takes about 3.5 us + 0.085 us/KB for its slab (fp16, SiLU: the CU's
  // own arithmetic; less without an activation, more with GELU and where a group's
  // row is one vector of a cache line), the two passes 10.5 us + 0.6 us/MB for the whole
  // tensor, so a large slab pays only where many of them run at once.  us, slab |
  // passes: 1 x 500 x 32 channels a group 6.0 | 11.5, 1 x 1463 x 32 10.7 | 11.7, 1 x 1463 x
  // 64 18.5 | 12.0, 8 x 1500 x 64 21.5 | 25.8, fp32 1 x 1463 x 32 18.0 | 12.5, 4 x
  // 1463 x 32 21.0 | 22.7, 8 x 1500 x 32 25.6 | 34.5; fp32 4 x 13 x 2048 without
  // activation 7.4 | 11.9, fp16 GELU 8 x 7985 x 8 23.5 | 14.5.  Fitted to 13000
  // shapes in both ways: 0.1% over the better one on average (without the
  // weights 0.6%).
  const double slab_kb = vecs * 16.0 / 1024, all_mb = slab_kb * p.B * p.G / 1024;
  const bool plain = p.act == SIDON_ACT_NONE || p.act == SIDON_ACT_RELU;
  const double weight = (plain ? (size == 4 ? 0.65 : 0.8) : p.act == SIDON_ACT_GELU ? 1.33 : 1.0) * (cg == v ? 1.25 : 1.0);
  return vector && cg % v == 0 && vecs <= kSlabVecs * kSlabThreads && slab_kb * weight <= 85 + 4.2 * all_mb &&
         (int64_t)p.B * p.G <= INT32_MAX / kSlabThreads;   // (a launch holds less than 2^32 threads)
}

template <typename T>
void run(Params& p, bool vector, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if (slab_way(p, sizeof(T), vector)) {
    slab<T>(p, (int64_t)p.T * (p.C / p.G / V), stream);
  } else if (vector) {
    plan_passes(p, V);
    passes<T, V>(p, stream);
  } else {
    plan_passes(p, 1);
    passes<T, 1>(p, stream);
  }
}

bool shape_ok(int B, int T, int C, int G, int dtype) {
  return B >= 1 && T >= 1 && C >= 1 && C <= kMaxC && G >= 1 && C % G == 0 && dtype >= SIDON_FP32 && dtype <= SIDON_BF16 &&
         B <= 65535 && T <= (1 << 30);
}

}  // namespace

SIDON_API size_t sidon_group_norm_workspace_bytes(int B, int T, int C, int G, int dtype) {
  if (!shape_ok(B, T, C, G, dtype)) return 0;
  const int64_t chunks = T < kMaxChunks ? T : kMaxChunks;
  return (size_t)B * (size_t)chunks * (size_t)G * sizeof(float2);
}

SIDON_API int sidon_group_norm_passes(int B, int T, int C, int G, int dtype, int vec, int* block_groups, int* chunks,
                                      int* lds_bytes) {
  sidon::clear_error();
  if (!block_groups || !chunks || !lds_bytes) return sidon::fail(SIDON_E_NULL, "the results must be non-NULL");
  if (!shape_ok(B, T, C, G, dtype) || (vec != 1 && (vec != 16 / element_size(dtype) || C % vec != 0)))
    return sidon::fail(SIDON_E_SHAPE, "B=%d T=%d C=%d G=%d dtype=%d vec=%d is no shape of sidon_group_norm_act", B, T, C,
                       G, dtype, vec);
  Params p{};
  p.B = B, p.T = T, p.C = C, p.G = G;
  plan_passes(p, vec);
  *block_groups = p.block_groups;
  *chunks = p.chunks;
  *lds_bytes = (int)unit_bytes(p, vec);
  return SIDON_OK;
}

SIDON_API int sidon_group_norm_act(const void* x, int64_t ldx, const int32_t* lens, const float* w, const float* bias,
                                   float eps, void* y, int64_t ldy, void* ws, size_t ws_bytes, int B, int T, int C,
                                   int G, int dtype, int act, sidon_stream_t stream) {
  using sidon::fail;
  sidon::clear_error();
  if (!x || !w || !bias || !y || !ws) return fail(SIDON_E_NULL, "x, w, bias, y and ws must be non-NULL");
  if (dtype < SIDON_FP32 || dtype > SIDON_BF16) return fail(SIDON_E_SHAPE, "dtype=%d is no SIDON_FP32 / FP16 / BF16", dtype);
  if (act < SIDON_ACT_NONE || act > SIDON_ACT_RELU) return fail(SIDON_E_SHAPE, "act=%d is no SIDON_ACT_*", act);
  if (!shape_ok(B, T, C, G, dtype))
    return fail(SIDON_E_SHAPE, "B=%d T=%d C=%d G=%d: need B in [1, 65535], T in [1, 2^30], C in [1, %d], C a multiple of G", B,
                T, C, G, kMaxC);
  const int size = element_size(dtype);
  const int64_t rows = (int64_t)B * T;
  if (ldx < C || ldy < C || ldx > (int64_t(1) << 31) || ldy > (int64_t(1) << 31))
    return fail(SIDON_E_STRIDE, "row strides ldx=%lld ldy=%lld must be >= C and at most 2^31", (long long)ldx,
                (long long)ldy);
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % (uintptr_t)size != 0 ||
      ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(bias)) & 3u) != 0 ||
      (reinterpret_cast<uintptr_t>(lens) & 3u) != 0 || (reinterpret_cast<uintptr_t>(ws) & 7u) != 0)
    return fail(SIDON_E_ALIGN, "x and y must be aligned to their elements, w, bias and lens to 4 bytes, ws to 8");
  if (ws_bytes < sidon_group_norm_workspace_bytes(B, T, C, G, dtype))
    return fail(SIDON_E_SHAPE, "ws holds %zu bytes, the call needs %zu", ws_bytes,
                sidon_group_norm_workspace_bytes(B, T, C, G, dtype));
  if (!(x == y && ldx == ldy) && sidon::rows_meet(x, ldx * size, C * size, y, ldy * size, C * size, rows))
    return fail(SIDON_E_SHAPE, "y may be x itself but must not overlap it otherwise");
  Params p{};
  p.x = x;
  p.lens = lens;
  p.w = w;
  p.bias = bias;
  p.y = y;
  p.part = static_cast<float2*>(ws);
  p.ldx = ldx;
  p.ldy = ldy;
  p.eps = eps;
  p.B = B;
  p.T = T;
  p.C = C;
  p.G = G;
  p.act = act;
  const int v = 16 / size;
  const bool vector = C % v == 0 && ldx % v == 0 && ldy % v == 0 && sidon::aligned16(x) && sidon::aligned16(y) &&
                      sidon::aligned16(w) && sidon::aligned16(bias);
  // Workgroups read w, bias and lens while others already write y; ws is written beside
  // all of them, where the call takes two launches.
  const struct {
    const void* at;
    int64_t bytes;
  } in[] = {{w, (int64_t)C * 4}, {bias, (int64_t)C * 4}, {lens, lens ? (int64_t)B * 4 : 0}};
  const bool ws_used = !slab_way(p, size, vector);
  const int64_t ws_need = (int64_t)sidon_group_norm_workspace_bytes(B, T, C, G, dtype);
  for (const auto& t : in) {
    if (t.bytes == 0) continue;
    if (sidon::row_meets(y, ldy * size, (int64_t)C * size, rows, t.at, t.bytes))
      return fail(SIDON_E_SHAPE, "y must not overlap w, bias or lens");
    if (ws_used && sidon::ranges_meet(ws, ws_need, t.at, t.bytes))
      return fail(SIDON_E_SHAPE, "ws must not overlap w, bias or lens");
  }
  if (ws_used && (sidon::row_meets(x, ldx * size, (int64_t)C * size, rows, ws, ws_need) ||
                  sidon::row_meets(y, ldy * size, (int64_t)C * size, rows, ws, ws_need)))
    return fail(SIDON_E_SHAPE, "ws must not overlap x or y");
  int rc;
  if ((rc = sidon::check_device())) return rc;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SIDON_FP32) {
    run<float>(p, vector, s);
  } else if (dtype == SIDON_FP16) {
    run<_Float16>(p, vector, s);
  } else {
    run<__bf16>(p, vector, s);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(SIDON_E_LAUNCH, "group norm launch failed: %s", hipGetErrorString(err));
  return SIDON_OK;
}
