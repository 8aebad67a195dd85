// adapters.hip -- a shared projection with a low-rank adapter per request
// (MI355X / gfx950):
//
//   y[m] = act(x[m] . w^T + bias + scale_e (x[m] . a_e^T) . b_e^T),   e = ids[m / rows_per_id]
//
// and the same into an fp32 stream.  Two launches:
//
//   shrink   low[m] = scale_e x[m] . a_e^T   [M, R]
//   expand   the tiled GEMM of gemm_tile.h over x . w^T, whose accumulators take
//            low[m] . b_e^T in front of the epilogue, so y is written once
//
// Rows of different adapters share tiles: the shared product does not see
// them, and the low-rank terms cost a product per adapter among a block's rows.
// Few rows are bound by the two launches' latencies, many by the shared product
// (4800 x 4096 x 1024 0.74 PFLOP/s with the low-rank term, rank 64), many items of a
// few rows by the lanes' own reads of b (300 x 1 x 4096 x 1024: rank 8 17 us, 64 73, 128 142).
#include "gemm_tile.h"

#include "sidon_host.h"
#include "sidon_operators.h"

#define SIDON_API extern "C" __attribute__((visibility("default")))

namespace {

using namespace sidon_gemm;
using sidon::fail;
using sidon::ranges_meet;

constexpr int kMaxRank = 128;
constexpr int kShrinkRows = 16;     // rows of a matrix product

struct ShrinkParams {
  const void* x;
  const void* a;             // [adapters, R, K]
  const float* scale;
  const int32_t* ids;
  void* low;                 // [planes, M, R]
  int64_t plane;
  int ldx, M, K, R, adapters, rows_per_id, planes;
  int rows;                  // per workgroup, <= 16
};

// RB blocks of 16 ranks, W wavefronts.  A workgroup owns `rows` rows; its
// wavefronts take 64 columns of K in turn, copied global -> LDS as 128-byte rows
// into two slots of their own (16-byte chunk c of row r at c ^ ((r >> 1) & 7)), and
// are summed through LDS in order.  Products are 16 ranks x 16 rows: a lane's
// accumulators are 4 ranks of one row, so of several adapters among the rows each
// costs a pass over K whose other rows' results are dropped.
// 16-bit outputs get the products rounded once: u of each, beside the output's own
// u of the sum, a few per cent of the error of a projection with an adapter of the usual
// size; a second summand would double the second launch's low-rank products and
// the bytes between the launches.  fp16 keeps them relative to their row (LowRow).
// (Operands read from memory by the lanes that multiply them cost a cache access
// per lane, its neighbours holding other rows: 17.2 us instead of 8.3 at 4800 rows, K 1024,
// rank 64.)
template <typename E, int RB, int W>
__global__ void __launch_bounds__(64 * W) shrink_kernel(const ShrinkParams p) {
  typedef typename Elem<E>::e8 e8;
  constexpr int kSlot = (1 + RB) * 2048;
  constexpr int kPer = 2 * (1 + RB);            // copies per slice
  static_assert(2 * W * kSlot <= 160 * 1024 && W * RB * 1024 + W * 64 <= 2 * W * kSlot, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[2 * W * kSlot];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lg = lane >> 4;
  const int row0 = blockIdx.x * p.rows;
  const auto row_of = [&](int i) SIDON_INLINE { return min(row0 + min(i, p.rows - 1), p.M - 1); };
  int id = p.ids[row_of(ln) / p.rows_per_id];
  if (id < 0 || id >= p.adapters) id = -1;

  // Copy i of a slice: rows 8 i + lane / 8 of x's 16, then of the adapter's 16 RB.
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + w * 2 * kSlot;
  const auto chunk = [&](int r) SIDON_INLINE { return 16u * ((lane & 7) ^ ((r >> 1) & 7)); };
  uint32_t xoff[2], aoff[2 * RB];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 8 * i + (lane >> 3);
    xoff[i] = (uint32_t)(row_of(r) - row0) * (uint32_t)(2 * p.ldx) + chunk(r);
  }
#pragma unroll
  for (int i = 0; i < 2 * RB; ++i) {
    const int r = 8 * i + (lane >> 3);
    aoff[i] = (uint32_t)min(r, p.R - 1) * (uint32_t)(2 * p.K) + chunk(r);
  }
  const char* const xbase = static_cast<const char*>(p.x) + 2 * ((int64_t)row0 * p.ldx);
  const int slices = p.K / 64, mine = slices > w ? (slices - w + W - 1) / W : 0;
  const char* const ops = smem + w * 2 * kSlot + ln * 128;
  const int swz = (ln >> 1) & 7;

  // (the same for every wavefront: they hold the same rows)
  uint64_t todo = __builtin_amdgcn_ballot_w64(id >= 0);
  while (todo != 0) {
    const int e = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    todo &= ~__builtin_amdgcn_ballot_w64(id == e);
    const float scale = p.scale[e];
    const char* const abase = static_cast<const char*>(p.a) + 2 * ((int64_t)e * p.R * p.K);
    const auto copy = [&](int t) SIDON_INLINE {
      const uint32_t at = lds + (t & 1) * kSlot;
      const int64_t col = 128 * (int64_t)(w + t * W);
#pragma unroll
      for (int i = 0; i < 2; ++i) copy_1k(at + i * 1024, xbase + col, xoff[i]);
#pragma unroll
      for (int i = 0; i < 2 * RB; ++i) copy_1k(at + (2 + i) * 1024, abase + col, aoff[i]);
    };
    f4 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[b] = f4{};
    if (mine > 0) copy(0);
    for (int t = 0; t < mine; ++t) {
      if (t + 1 < mine) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot's reads have retired
        copy(t + 1);
        wait_vmcnt<kPer>();
      } else {
        wait_vmcnt<0>();
      }
      const char* at = ops + (t & 1) * kSlot;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int c = ((4 * s + lg) ^ swz) << 4;
        const e8 xv = *reinterpret_cast<const e8*>(at + c);
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = mma(*reinterpret_cast<const e8*>(at + (1 + b) * 2048 + c), xv, acc[b]);
      }
    }
    lds_barrier();   // everyone is done with the slots, which the sums reuse
    f4* const part = reinterpret_cast<f4*>(smem);
#pragma unroll
    for (int b = 0; b < RB; ++b) part[(w * RB + b) * 64 + lane] = acc[b];
    lds_barrier();
    // A lane's sums are of the row it holds.
    constexpr int NB = (RB + W - 1) / W;
    using Row = LowRow<E>;
    f4 sum[NB];
    uint32_t largest = 0;   // magnitude's bits, in whose order infinity and NaN come last
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int b = w + k * W;
      if (b >= RB) break;
      sum[k] = part[b * 64 + lane];
#pragma unroll
      for (int i = 1; i < W; ++i) sum[k] += part[(i * RB + b) * 64 + lane];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        sum[k][c] *= scale;
        const float v = sum[k][c];
        largest = max(largest, __builtin_bit_cast(uint32_t, v) & 0x7fffffffu);
      }
    }
    uint32_t power = 0;
    if constexpr (Row::kDivided) {
      // The row's: of the four lanes that hold it, and of all wavefronts.
      const auto p16 = __builtin_amdgcn_permlane16_swap(largest, largest, false, false);
      largest = max(p16[0], p16[1]);
      const auto p32 = __builtin_amdgcn_permlane32_swap(largest, largest, false, false);
      largest = max(p32[0], p32[1]);
      if constexpr (RB > 1) {
        uint32_t* const all = reinterpret_cast<uint32_t*>(smem + W * RB * 1024);   // (behind the sums)
        if (lg == 0) all[w * 16 + ln] = largest;
        lds_barrier();
#pragma unroll
        for (int i = 0; i < (RB < W ? RB : W); ++i) largest = max(largest, all[i * 16 + ln]);
      }
      power = Row::power(largest);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int b = w + k * W;
      if (b >= RB) break;
      const int r = 16 * b + 4 * lg, m = row0 + ln;
      if (ln < p.rows && m < p.M && r < p.R && id == e) {
        f4 s = sum[k];
        if constexpr (Row::kDivided) {
#pragma unroll
          for (int c = 0; c < 4; ++c) s[c] = Row::divided(s[c], power);
        }
        E* dst = static_cast<E*>(p.low) + (int64_t)m * p.R + r;
        for (int plane = 0; plane < p.planes; ++plane) {
          typename Elem<E>::e4 v;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            v[c] = to_elem<E>(s[c]);
            s[c] -= (float)v[c];   // exact: what the rounding left
          }
          if constexpr (Row::kDivided)
            v = __builtin_bit_cast(typename Elem<E>::e4, Row::packed(__builtin_bit_cast(typename Row::i2, v), power, r / 4));
          *reinterpret_cast<typename Elem<E>::e4*>(dst + plane * p.plane) = v;
        }
      }
    }
    if (todo != 0) lds_barrier();
  }
}

// ---- expand -----------------------------------------------------------------------

typedef void (*ExpandFn)(LowParams);
struct ExpandKernel {
  int bm, bn, threads;
  bool direct;         // takes rows of any adapters (kDirectTile)
  ExpandFn fn[2][2];   // [fp16, bf16][half out, fp32 add]
};

#define SIDON_LOW(BM, BN, WM, WN, MF, ST, MODE, E) gemm_tile_kernel<BM, BN, WM, WN, MF, ST, MODE, E, LowParams>
#define SIDON_BOTH(BM, BN, WM, WN, MF, ST)                                              \
  {BM, BN, 64 * WM * WN, kDirectTile<BM, BN>,                                           \
   {{SIDON_LOW(BM, BN, WM, WN, MF, ST, kHalf, _Float16), SIDON_LOW(BM, BN, WM, WN, MF, ST, kAdd, _Float16)}, \
    {SIDON_LOW(BM, BN, WM, WN, MF, ST, kHalf, __bf16), SIDON_LOW(BM, BN, WM, WN, MF, ST, kAdd, __bf16)}}}
#define SIDON_HALF(BM, BN, WM, WN, MF, ST)                                              \
  {BM, BN, 64 * WM * WN, kDirectTile<BM, BN>,                                           \
   {{SIDON_LOW(BM, BN, WM, WN, MF, ST, kHalf, _Float16), nullptr},                      \
    {SIDON_LOW(BM, BN, WM, WN, MF, ST, kHalf, __bf16), nullptr}}}

// gemm.hip's shapes, half of them: what the rest would gain is small next to the
// low-rank term.  us, of it the shrink launch, and the shared projection alone
// (conformer.linear_silu_lt, residual_gemm): 1 x 1024 x 1024 rank 16 9.0 (2.6) | 5.8,
// 48 rows of 43 adapters x 4096 x 1024 rank 16 12.2 (3.3) | 6.0, 4 x 400 x 2048 x 1024
// rank 32 20.3 (5.0; bf16 19.0) | 12.3, 8 x 600 x 4096 x 1024 rank 64 59 (9.0; fp16 64) |
// 51-57, rank 16 56 | 51, residual 3 x 1463 x 1024 x 4096 rank 16 57.5 (11.3) | 40.  The shared projection's
// cost picks the tile: on 5000 calls, each timed with every tile, 1% over the best on average.
const ExpandKernel kExpand[] = {
    SIDON_BOTH(32, 64, 2, 2, 16, 6),   SIDON_BOTH(64, 64, 2, 2, 16, 4),   SIDON_BOTH(64, 128, 2, 4, 16, 4),
    SIDON_BOTH(128, 128, 2, 4, 16, 4), SIDON_BOTH(192, 128, 2, 4, 16, 3), SIDON_HALF(128, 256, 2, 4, 16, 3),
    SIDON_HALF(160, 256, 1, 4, 32, 3), SIDON_HALF(192, 256, 2, 4, 16, 2),
    SIDON_HALF(320, 256, 2, 4, 32, 2),
};

struct Call {
  LowParams p;
  const void* a;
  const float* scale;
  void* ws;
  size_t ws_bytes;
  int items, dtype;
  bool residual;
};

int planes_of(bool residual, int dtype) { return !residual ? 1 : dtype == SIDON_FP16 ? 2 : 3; }

int check_and_launch(Call& c, sidon_stream_t stream) {
  LowParams& p = c.p;
  if (!p.x || !p.w || !c.a || !p.up || !c.scale || !p.ids || !p.y || !c.ws || (c.residual && !p.add))
    return fail(SIDON_E_NULL, "only bias may be NULL");
  if (c.dtype != SIDON_FP16 && c.dtype != SIDON_BF16)
    return fail(SIDON_E_SHAPE, "dtype=%d is neither SIDON_FP16 nor SIDON_BF16", c.dtype);
  if (p.M < 1 || p.N < 64 || p.N % 64 != 0 || p.K < 64 || p.K % 64 != 0 || p.rank < 8 || p.rank > kMaxRank ||
      p.rank % 8 != 0 || p.adapters < 1 || c.items < 1 || p.M % c.items != 0)
    return fail(SIDON_E_SHAPE,
                "M=%d N=%d K=%d R=%d adapters=%d items=%d: need M >= 1 and a multiple of items, N and K multiples of 64, "
                "R a multiple of 8 up to %d, adapters >= 1",
                p.M, p.N, p.K, p.rank, p.adapters, c.items, kMaxRank);
  if (p.act != SIDON_ACT_NONE && p.act != SIDON_ACT_SILU) return fail(SIDON_E_SHAPE, "act=%d: 0 (none) or 1 (SiLU)", p.act);
  const int step = c.residual ? 4 : 8;
  if (p.ldx < p.K || p.ldw < p.K || p.ldy < p.N || (p.ldx | p.ldw) % 8 != 0 || p.ldy % step != 0 ||
      (c.residual && (p.ldadd < p.N || p.ldadd % step != 0)))
    return fail(SIDON_E_STRIDE, "row strides ldx=%d ldw=%d (multiples of 8, >= K) ldy=%d ldadd=%d (multiples of %d, >= N)",
                p.ldx, p.ldw, p.ldy, p.ldadd, step);
  if ((int64_t)p.M * p.ldx * 2 >= (int64_t(1) << 32) || (int64_t)p.N * p.ldw * 2 >= (int64_t(1) << 32) ||
      (int64_t)p.rank * p.K * 2 >= (int64_t(1) << 32))
    return fail(SIDON_E_SHAPE, "x, w and an adapter's a must each span less than 4 GiB");
  if (!sidon::aligned16(p.x) || !sidon::aligned16(p.w) || !sidon::aligned16(c.a) || !sidon::aligned16(p.up) ||
      !sidon::aligned16(p.y) || !sidon::aligned16(c.ws) || (c.residual && !sidon::aligned16(p.add)) ||
      (reinterpret_cast<uintptr_t>(p.bias) & 7u) != 0 || (reinterpret_cast<uintptr_t>(p.ids) & 3u) != 0 ||
      (reinterpret_cast<uintptr_t>(c.scale) & 3u) != 0)
    return fail(SIDON_E_ALIGN, "x, w, a, b, y, add and ws must be 16-byte aligned, bias 8, ids and scale 4");
  const size_t need = sidon_adapter_workspace_bytes(p.M, p.rank, c.residual, c.dtype);
  if (c.ws_bytes < need) return fail(SIDON_E_SHAPE, "ws holds %zu bytes, the call needs %zu", c.ws_bytes, need);
  // Workgroups read the inputs while others already write y, or ws.
  const int64_t ysize = c.residual ? 4 : 2;
  const int64_t ybytes = ((int64_t)(p.M - 1) * p.ldy + p.N) * ysize;
  const int64_t up_bytes = (int64_t)p.adapters * p.N * p.rank * 2, a_bytes = (int64_t)p.adapters * p.rank * p.K * 2;
  if (sidon::rows_meet(p.y, p.ldy * ysize, p.N * ysize, p.x, (int64_t)p.ldx * 2, (int64_t)p.K * 2, p.M) ||
      ranges_meet(p.y, ybytes, p.w, ((int64_t)(p.N - 1) * p.ldw + p.K) * 2) || ranges_meet(p.y, ybytes, p.up, up_bytes) ||
      ranges_meet(p.y, ybytes, c.a, a_bytes) || ranges_meet(p.y, ybytes, c.ws, (int64_t)need) ||
      (p.bias != nullptr && ranges_meet(p.y, ybytes, p.bias, (int64_t)p.N * 2)))
    return fail(SIDON_E_SHAPE, "y must not overlap an input or ws");
  const struct {
    const void* at;
    int64_t bytes;
  } in[] = {{p.ids, (int64_t)c.items * 4}, {c.scale, (int64_t)p.adapters * 4}, {c.a, a_bytes}, {p.up, up_bytes},
            {p.bias, p.bias != nullptr ? (int64_t)p.N * 2 : 0}};
  for (int i = 0; i < 5; ++i) {
    if (i < 2 && sidon::row_meets(p.y, p.ldy * ysize, p.N * ysize, p.M, in[i].at, in[i].bytes))
      return fail(SIDON_E_SHAPE, "y must not overlap an input or ws");
    if (in[i].bytes > 0 && ranges_meet(c.ws, (int64_t)need, in[i].at, in[i].bytes))
      return fail(SIDON_E_SHAPE, "ws must not overlap an input");
  }
  if (sidon::row_meets(p.x, (int64_t)p.ldx * 2, (int64_t)p.K * 2, p.M, c.ws, (int64_t)need) ||
      sidon::row_meets(p.w, (int64_t)p.ldw * 2, (int64_t)p.K * 2, p.N, c.ws, (int64_t)need) ||
      (c.residual && sidon::row_meets(p.add, (int64_t)p.ldadd * 4, (int64_t)p.N * 4, p.M, c.ws, (int64_t)need)))
    return fail(SIDON_E_SHAPE, "ws must not overlap an input");
  if (c.residual && !(p.add == p.y && p.ldadd == p.ldy) &&
      sidon::rows_meet(p.y, p.ldy * ysize, p.N * ysize, p.add, (int64_t)p.ldadd * 4, (int64_t)p.N * 4, p.M))
    return fail(SIDON_E_SHAPE, "y may be add itself but must not overlap it otherwise");
  int rc;
  if ((rc = sidon::check_device())) return rc;
  const int cus = sidon::compute_units();

  p.rows_per_id = p.M / c.items;
  p.planes = planes_of(c.residual, c.dtype);
  p.plane = (int64_t)p.M * p.rank;
  p.low = c.ws;
  ShrinkParams s{};
  s.x = p.x;
  s.a = c.a;
  s.scale = c.scale;
  s.ids = p.ids;
  s.low = c.ws;
  s.plane = p.plane;
  s.ldx = p.ldx, s.M = p.M, s.K = p.K, s.R = p.rank, s.adapters = p.adapters, s.rows_per_id = p.rows_per_id;
  s.planes = p.planes;
  // Few rows: one per workgroup, so that rows of different adapters run side by side.
  s.rows = (p.M + cus - 1) / cus;
  if (s.rows > kShrinkRows) s.rows = kShrinkRows;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((p.M + s.rows - 1) / s.rows));
  const auto shrink = [&](auto zero) {
    typedef decltype(zero) E;
    if (s.R <= 16) {
      hipLaunchKernelGGL((shrink_kernel<E, 1, 8>), grid, dim3(512), 0, st, s);
    } else if (s.R <= 32) {
      hipLaunchKernelGGL((shrink_kernel<E, 2, 8>), grid, dim3(512), 0, st, s);
    } else if (s.R <= 64) {
      hipLaunchKernelGGL((shrink_kernel<E, 4, 4>), grid, dim3(256), 0, st, s);
    } else {
      hipLaunchKernelGGL((shrink_kernel<E, 8, 4>), grid, dim3(256), 0, st, s);
    }
  };
  if (c.dtype == SIDON_FP16) {
    shrink(_Float16(0));
  } else {
    shrink(__bf16(0));
  }

  const ExpandKernel* best = nullptr;
  double best_us = 0;
  for (const ExpandKernel& t : kExpand) {
    if (t.fn[0][c.residual] == nullptr || p.N % t.bn != 0) continue;
    if (!t.direct && !low_staged(t.bm, t.bn, p.rows_per_id, p.rank)) continue;
    const double us = tile_us(t.bm, t.bn, p.M, p.N, p.K, 1, !c.residual, cus);
    if (best == nullptr || us < best_us) best = &t, best_us = us;
  }
  p.tiles_m = (p.M + best->bm - 1) / best->bm;
  p.tiles_n = p.N / best->bn;
  p.splits = 1;
  p.group = p.tiles_m < 8 ? p.tiles_m : 8;
  const int64_t wgs = (int64_t)p.tiles_m * p.tiles_n;
  if (wgs >= (int64_t(1) << 31)) return fail(SIDON_E_SHAPE, "too many tiles");
  hipLaunchKernelGGL(best->fn[c.dtype == SIDON_BF16][c.residual], dim3((unsigned)wgs), dim3(best->threads), 0, st, p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(SIDON_E_LAUNCH, "adapter projection launch failed: %s", hipGetErrorString(err));
  return SIDON_OK;
}

}  // namespace

SIDON_API size_t sidon_adapter_workspace_bytes(int M, int R, int residual, int dtype) {
  if (M < 1 || R < 8 || R > kMaxRank || R % 8 != 0 || (dtype != SIDON_FP16 && dtype != SIDON_BF16)) return 0;
  return (size_t)M * R * 2 * planes_of(residual != 0, dtype);
}

SIDON_API int sidon_adapter_linear(const void* x, int ldx, const void* w, int ldw, const void* bias, const void* a,
                                   const void* b, const float* scale, const int32_t* ids, void* y, int ldy, void* ws,
                                   size_t ws_bytes, int M, int N, int K, int R, int adapters, int items, int act,
                                   int dtype, sidon_stream_t stream) {
  sidon::clear_error();
  Call c{};
  LowParams& p = c.p;
  p.x = x, p.w = w, p.bias = bias, p.y = y, p.up = b, p.ids = ids;
  p.ldx = ldx, p.ldw = ldw, p.ldy = ldy, p.M = M, p.N = N, p.K = K, p.rank = R, p.adapters = adapters, p.act = act;
  c.a = a, c.scale = scale, c.ws = ws, c.ws_bytes = ws_bytes, c.items = items, c.dtype = dtype;
  static_assert(kNone == SIDON_ACT_NONE && kSilu == SIDON_ACT_SILU, "the tile kernel's activation codes");
  return check_and_launch(c, stream);
}

SIDON_API int sidon_adapter_residual(const void* x, int ldx, const void* w, int ldw, const void* a, const void* b,
                                     const float* scale, const int32_t* ids, const float* add, int ldadd, float* y,
                                     int ldy, void* ws, size_t ws_bytes, int M, int N, int K, int R, int adapters,
                                     int items, int dtype, sidon_stream_t stream) {
  sidon::clear_error();
  Call c{};
  LowParams& p = c.p;
  p.x = x, p.w = w, p.y = y, p.up = b, p.ids = ids, p.add = add;
  p.ldx = ldx, p.ldw = ldw, p.ldy = ldy, p.ldadd = ldadd;
  p.M = M, p.N = N, p.K = K, p.rank = R, p.adapters = adapters;
  c.a = a, c.scale = scale, c.ws = ws, c.ws_bytes = ws_bytes, c.items = items, c.dtype = dtype, c.residual = true;
  return check_and_launch(c, stream);
}
