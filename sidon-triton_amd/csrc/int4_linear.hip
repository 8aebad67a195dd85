// int4_linear.hip -- projections with 4-bit weights and group scales for few rows
// (MI355X / gfx950):
//
//   y[m, n] = act(bias[n] + sum_g s[n, g] sum_{k in g} x[m, k] (w[n, k] - z[n, g]))
//
// Few rows read every weight once, so the weights' bytes bound it.  They are laid out
// when they are loaded (include/sidon_operators.h), 16 outputs x 128 inputs as the 1 KB
// that a wavefront loads with 16 bytes a lane, in the order in which its lanes hold
// the B operands of four v_mfma_f32_16x16x32.  A nibble becomes an operand by its bits
// alone: q | 0x6400 is the fp16 1024 + q (less 1032, exactly, q - 8), q | 0x4300 the
// bf16 128 + q.  What that adds, and the zero point, times the sum of the group's
// inputs, which a product with ones gives in the accumulator's own layout, is taken
// off in fp32 with the group's scale.
//
// A wavefront has 16 NT outputs of 16 MT rows and every WK-th block of 128 inputs, and
// sends for the next one's weights and inputs before it takes a block's products; the WK
// wavefronts of a workgroup are summed through LDS.  Inputs come through LDS too, copied as
// whole rows: the operand's own lanes are of 16 rows, whose loads the cache takes one at a time
// (32 x 4096 x 14336 33 us; so 16).
//
// Reached: 1 x 32768 x 4096 (71 MB) 16 us, 4.4 TB/s; 32 rows of it 18 to 23, where 40 matrix and 200
// vector instructions a block stand beside the weights' 4 KB; 1 x 4096 x 1024 2.8, latency.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "attn_device.h"
#include "sidon_host.h"
#include "sidon_operators.h"

#define SIDON_API extern "C" __attribute__((visibility("default")))

namespace {

using namespace sidon_attn;

constexpr int kTileN = 16, kTileK = 128;

struct Int4Params {
  const void* x;
  const void* words;        // [N / 16, K / 128, 64 lanes] of 16 bytes
  const uint32_t* scales;   // [N / 16, K / 128, 128 / group, 16]: scale, and in the high half what goes off the weights
  const void* bias;
  void* y;
  int64_t ldx, ldy;
  int M, N, K;
  int tiles, blocks;        // of N by 16, of K by 128
  int act;
};

// Eight nibbles of a word (in the order 0 2 4 6 1 3 5 7 from the lowest) as an operand.
// `mask` and `lead` in vector registers, so that an insertion is one instruction.
template <typename E>
__device__ __forceinline__ i4 operand(uint32_t word, uint32_t mask, uint32_t lead) {
  const auto insert = [&](uint32_t x) { return (mask & x) | (~mask & lead); };
  i4 r;
  if constexpr (__is_same(E, _Float16)) {
    // The upper nibble of a byte stands 4 bits higher in the mantissa: 1024 + 16 q.
    const uint32_t high = word >> 8;
    const auto insert16 = [&](uint32_t x) { return ((mask << 4) & x) | (~(mask << 4) & lead); };
    const h2 less = {(_Float16)-1032.f, (_Float16)-1032.f}, down = {(_Float16)0.0625f, (_Float16)0.0625f},
             less16 = {(_Float16)-72.f, (_Float16)-72.f};
    r[0] = __builtin_bit_cast(int, __builtin_bit_cast(h2, insert(word)) + less);
    r[1] = __builtin_bit_cast(int, __builtin_elementwise_fma(__builtin_bit_cast(h2, insert16(word)), down, less16));
    r[2] = __builtin_bit_cast(int, __builtin_bit_cast(h2, insert(high)) + less);
    r[3] = __builtin_bit_cast(int, __builtin_elementwise_fma(__builtin_bit_cast(h2, insert16(high)), down, less16));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (int)insert(word >> (4 * i));
  }
  return r;
}

// SPG: steps of 32 inputs per group within a block.  kOff: something goes off the weights.
template <typename E, int MT, int NT, int WK, int SPG, bool kOff>
__global__ void __launch_bounds__(64 * WK, 2) int4_linear_kernel(const Int4Params p) {
  constexpr int kGroups = 4 / SPG;
  constexpr int kX = MT * 16 * kTileK * 2;   // bytes of a block's inputs
  static_assert(sizeof(E) == 2, "16-bit inputs");
  __shared__ __attribute__((aligned(16))) char smem[WK * (kX > MT * NT * 1024 ? kX : MT * NT * 1024)];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int tile0 = blockIdx.x * NT, row0 = blockIdx.y * (16 * MT);

  const i4* wp[NT];
  const uint32_t* sp[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t tile = min(tile0 + j, p.tiles - 1);   // (tiles past the last are not stored)
    wp[j] = static_cast<const i4*>(p.words) + tile * p.blocks * 64 + lane;
    sp[j] = p.scales + tile * p.blocks * (kGroups * 16) + c;
  }
  // A block's inputs go through LDS, 4 rows x 256 bytes a copy: lanes that lie side by side read
  // one row, where the operand's are of 16 rows, whose loads would go through the cache one by
  // one.  Chunk q of 16 bytes of row r lies at q ^ (r % 16).  (Rows past the last are not copied
  // and not stored; inputs past the last, whose scales are 0, are the last 32.)
  const char* const xs = smem + w * kX;
  const uint32_t xat = (uint32_t)(uintptr_t)SIDON_LDS_PTR(char, smem) + w * kX;
  const int xr = lane >> 4, left = p.M - row0 - xr;
  const E* const xl = static_cast<const E*>(p.x) + (int64_t)(row0 + xr) * p.ldx + 8 * ((lane & 3) ^ xr);
  const auto copy_x = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (16 * m + 4 * j < left) {
          const int k = min(b * kTileK + 32 * (((lane >> 2) & 3) ^ j), p.K - 32);
          dma_lanes(xat + (4 * m + j) * 1024, xl + (16 * m + 4 * j) * p.ldx + k);
        }
  };
  const auto load_w = [&](int b, i4 (&words)[NT], uint32_t (&scale)[NT][kGroups]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      words[j] = wp[j][(int64_t)b * 64];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) scale[j][k] = sp[j][(int64_t)b * (kGroups * 16) + k * 16];
    }
  };
  uint32_t mask = 0x000f000fu, lead = __is_same(E, _Float16) ? 0x64006400u : 0x43004300u;
  asm("" : "+v"(mask), "+v"(lead));

  f4 total[MT][NT] = {};
  const int one2 = __is_same(E, _Float16) ? 0x3c003c00 : 0x3f803f80;
  const i4 ones = {one2, one2, one2, one2};
  i4 words[NT];
  uint32_t scale[NT][kGroups];
  if (w < p.blocks) {
    load_w(w, words, scale);
    copy_x(w);
  }
#pragma unroll 1
  for (int b = w; b < p.blocks; b += WK) {
    wait_vmcnt<0>();
    arrived(words);   // (or the compiler would wait for them again, and for what is sent for below)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < kGroups; ++k) asm volatile("" : "+v"(scale[j][k]));
    i4 xop[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        xop[m][i] = *reinterpret_cast<const i4*>(xs + m * 4096 + c * 256 + (((4 * i + g) ^ c) << 4));
    wait_lgkm0();
    i4 next[NT] = {};
    uint32_t next_scale[NT][kGroups] = {};
    if (b + WK < p.blocks) {   // a block ahead
      load_w(b + WK, next, next_scale);
      copy_x(b + WK);
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      f4 sums[MT] = {};
      if constexpr (kOff) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = k * SPG; i < (k + 1) * SPG; ++i) sums[m] = Half<E>::small(xop[m][i], ones, sums[m]);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        f4 acc[MT] = {};
#pragma unroll
        for (int i = k * SPG; i < (k + 1) * SPG; ++i) {
          const i4 op = operand<E>((uint32_t)words[j][i], mask, lead);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m] = Half<E>::small(xop[m][i], op, acc[m]);
        }
        typedef E e2 __attribute__((ext_vector_type(2)));
        const e2 so = __builtin_bit_cast(e2, scale[j][k]);
        const float s = (float)so[0], off = -(float)so[1];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a = acc[m][e];
            if constexpr (kOff) a = fmaf(off, sums[m][e], a);
            total[m][j][e] = fmaf(s, a, total[m][j][e]);
          }
      }
    }
    __builtin_amdgcn_sched_barrier(0);   // (or these would wait for the next block among the products)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      words[j] = next[j];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) scale[j][k] = next_scale[j][k];
    }
  }

  __syncthreads();   // (the inputs are done with)
  f4(*const part)[MT * NT][64] = reinterpret_cast<f4(*)[MT * NT][64]>(smem);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[w][m * NT + j][lane] = total[m][j];
  __syncthreads();
  for (int t = w; t < MT * NT; t += WK) {
    f4 sum = part[0][t][lane];
#pragma unroll
    for (int k = 1; k < WK; ++k) sum += part[k][t][lane];
    const int n = (tile0 + t % NT) * kTileN + c, row = row0 + t / NT * 16 + 4 * g;
    if (n >= p.N) continue;
    const float bias = p.bias != nullptr ? (float)static_cast<const E*>(p.bias)[n] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (row + e >= p.M) break;
      float v = sum[e] + bias;
      if (p.act == SIDON_ACT_SILU) v = v / (1.f + __expf(-v));
      static_cast<E*>(p.y)[(int64_t)(row + e) * p.ldy + n] = (E)v;
    }
  }
}

// ---- host -------------------------------------------------------------------------

struct Shape {
  int mt, nt, wk;
};

// Rows of a workgroup by what M needs.  A wavefront takes one tile of outputs where that gives no
// CU more than one workgroup, two where two do, else four (each tile more is x loaded once less,
// and a CU with two workgroups takes longer: 64 x 8192 x 4096 in one, two, four tiles 17.9, 13.0
// and 15.2 us; 64 x 16384 x 2048 22.3, 15.1 and 12.0; 32 x 4096 x 14336 15.6, 16.7 and 22.5), and K is
// split over eight wavefronts, or four where four tiles give CUs several workgroups (32 x 32768 x
// 4096 21.8 us, with eight 23.9; 64 x 16384 x 2048 12.8 and 12.0).
Shape shape(int M, int N, int cus) {
  const int mt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  const int64_t units = (int64_t)((N + kTileN - 1) / kTileN) * ((M + 16 * mt - 1) / (16 * mt));
  return Shape{mt, units <= cus ? 1 : units <= 2 * (int64_t)cus ? 2 : 4, units <= 4 * (int64_t)cus ? 8 : 4};
}

template <typename E, int MT, int NT, int WK>
void launch_groups(const Int4Params& p, int group, bool off, dim3 grid, hipStream_t s) {
#define SIDON_INT4(SPG)                                                                                      \
  if (off)                                                                                                   \
    hipLaunchKernelGGL((int4_linear_kernel<E, MT, NT, WK, SPG, true>), grid, dim3(64 * WK), 0, s, p);        \
  else if constexpr (__is_same(E, _Float16))                                                                 \
    hipLaunchKernelGGL((int4_linear_kernel<E, MT, NT, WK, SPG, false>), grid, dim3(64 * WK), 0, s, p);
  if (group == 32) {
    SIDON_INT4(1)
  } else if (group == 64) {
    SIDON_INT4(2)
  } else {
    SIDON_INT4(4)
  }
#undef SIDON_INT4
}

template <typename E, int MT>
void launch_shape(const Int4Params& p, const Shape& c, int group, bool off, hipStream_t s) {
  const dim3 grid((p.tiles + c.nt - 1) / c.nt, (p.M + 16 * MT - 1) / (16 * MT));
  if (c.nt == 1)
    launch_groups<E, MT, 1, 8>(p, group, off, grid, s);
  else if (c.nt == 2)
    launch_groups<E, MT, 2, 8>(p, group, off, grid, s);
  else if (c.wk == 8)
    launch_groups<E, MT, 4, 8>(p, group, off, grid, s);
  else
    launch_groups<E, MT, 4, 4>(p, group, off, grid, s);
}

template <typename E>
void launch(const Int4Params& p, const Shape& c, int group, bool off, hipStream_t s) {
  if (c.mt == 1)
    launch_shape<E, 1>(p, c, group, off, s);
  else if (c.mt == 2)
    launch_shape<E, 2>(p, c, group, off, s);
  else
    launch_shape<E, 4>(p, c, group, off, s);
}

}  // namespace

SIDON_API int sidon_int4_linear_tiles(int M, int N, int* rows, int* outputs, int* splits) {
  sidon::clear_error();
  if (!rows || !outputs || !splits) return sidon::fail(SIDON_E_NULL, "rows, outputs and splits must be non-NULL");
  if (M < 1 || N < 1 || M > (1 << 21) || N > (1 << 24))
    return sidon::fail(SIDON_E_SHAPE, "M=%d N=%d: need 1 <= M <= 2^21, N <= 2^24", M, N);
  const Shape c = shape(M, N, sidon::compute_units());
  *rows = c.mt, *outputs = c.nt, *splits = c.wk;
  return SIDON_OK;
}

SIDON_API int sidon_int4_linear(const void* x, int64_t ldx, const void* words, const void* scales, const void* bias,
                                void* y, int64_t ldy, int M, int N, int K, int group, int zeros, int act, int dtype,
                                sidon_stream_t stream) {
  using sidon::fail;
  using sidon::Rows;
  sidon::clear_error();
  if (!x || !words || !scales || !y) return fail(SIDON_E_NULL, "x, words, scales and y must be non-NULL");
  if (dtype != SIDON_FP16 && dtype != SIDON_BF16) return fail(SIDON_E_SHAPE, "dtype=%d is neither SIDON_FP16 nor SIDON_BF16", dtype);
  if (act != SIDON_ACT_NONE && act != SIDON_ACT_SILU) return fail(SIDON_E_SHAPE, "act=%d is neither SIDON_ACT_NONE nor SIDON_ACT_SILU", act);
  if (M < 1 || N < 1 || K < 1 || M > (1 << 21) || N > (1 << 24) || K > (1 << 20))
    return fail(SIDON_E_SHAPE, "M=%d N=%d K=%d: need 1 <= M <= 2^21, N <= 2^24, K <= 2^20", M, N, K);
  if ((group != 32 && group != 64 && group != 128) || K % group != 0)
    return fail(SIDON_E_SHAPE, "group=%d K=%d: need group 32, 64 or 128 and K a multiple of it", group, K);
  if (ldx < K || ldx % 8 != 0 || ldx > (int64_t)1 << 40 || ldy < N || ldy > (int64_t)1 << 40)
    return fail(SIDON_E_STRIDE, "ldx=%lld must be a multiple of 8 from K=%d, ldy=%lld at least N=%d, both at most 2^40",
                (long long)ldx, K, (long long)ldy, N);
  if (!sidon::aligned16(x) || !sidon::aligned16(words) || !sidon::aligned16(scales) ||
      ((reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(y)) & 1u) != 0)
    return fail(SIDON_E_ALIGN, "x, words and scales must be 16-byte aligned, bias and y 2-byte aligned");
  Int4Params p{};
  p.tiles = (N + kTileN - 1) / kTileN, p.blocks = (K + kTileK - 1) / kTileK;
  {
    const Rows out{y, {1, 1, M}, {0, 0, ldy}, N, 2};
    if (sidon::tensors_meet(out, Rows{x, {1, 1, M}, {0, 0, ldx}, K, 2})) return fail(SIDON_E_SHAPE, "y must lie apart from x");
    const struct {
      const char* name;
      const void* at;
      int64_t bytes;
    } flat[] = {{"words", words, (int64_t)p.tiles * p.blocks * 1024},
                {"scales", scales, (int64_t)p.tiles * p.blocks * (kTileK / group) * 64},
                {"bias", bias, bias ? (int64_t)2 * N : 0}};
    for (const auto& f : flat)
      if (f.bytes > 0 && sidon::ranges_meet(y, (int64_t)out.bytes(), f.at, f.bytes))
        return fail(SIDON_E_SHAPE, "y must lie apart from %s", f.name);
  }
  const int rc = sidon::check_device();
  if (rc) return rc;
  p.x = x, p.words = words, p.scales = static_cast<const uint32_t*>(scales), p.bias = bias, p.y = y;
  p.ldx = ldx, p.ldy = ldy;
  p.M = M, p.N = N, p.K = K, p.act = act;
  const Shape c = shape(M, N, sidon::compute_units());
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // (fp16's operands are off by 8 already, bf16's by -128)
  if (dtype == SIDON_FP16)
    launch<_Float16>(p, c, group, zeros != 0, s);
  else
    launch<__bf16>(p, c, group, true, s);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(SIDON_E_LAUNCH, "4-bit projection launch failed: %s", hipGetErrorString(err));
  return SIDON_OK;
}
