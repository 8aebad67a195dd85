// attn_device.h -- device helpers of the attention kernels that take fp16 and
// bf16 (diff_attn.hip, cross_attn.hip, cross_attn_bwd.hip).  Internal to the
// library.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "flexrel_device.h"

namespace sidon_attn {

using namespace sidon_flexrel;
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));

constexpr float kFloorMax = -1e30f; // a running maximum that no key has raised yet (finite: -inf - -inf is NaN)
constexpr int kBack = 3 * 1024;     // bytes that the copies' offsets hold beyond their rows (dma_tile's last copy adds none)

template <typename E>
struct Half;
template <>
struct Half<_Float16> {
  typedef h8 v8;
  typedef h2 v2;
  typedef h4 v4;
  // The running maximum stands for a probability of 2^kLift, not of 1, so that
  // probabilities keep their 11 bits down to 2^-23 of the largest and vanish below
  // 2^-34 (with 1: 2^-14 and 2^-25, which the keys of a long cache add up to).  A
  // step's 32 sum to 2^14 at most, under what raises the maximum.
  static constexpr float kLift = 9.f;
  static __device__ __forceinline__ f32x16 mfma(i4 a, i4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f4 small(i4 a, i4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
};
template <>
struct Half<__bf16> {
  typedef b8 v8;
  typedef b2 v2;
  typedef b4 v4;
  static constexpr float kLift = 0.f;   // (as many exponents as fp32)
  static __device__ __forceinline__ f32x16 mfma(i4 a, i4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f4 small(i4 a, i4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
};

// A pointer that is the same in every lane, in scalar registers (the copies
// take it there, and under pressure the compiler forms it in vector ones).
__device__ __forceinline__ const char* uniform(const char* x) {
  const uint64_t u = reinterpret_cast<uint64_t>(x);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
  return reinterpret_cast<const char*>((uint64_t)hi << 32 | lo);
}

// x of lane l plus x of lane l ^ 32.
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// Two copies as dma_1k's, the second 1024 beyond both addresses.
__device__ __forceinline__ void dma_2k(uint32_t lds_addr, const char* gbase, uint32_t v0, uint32_t v1) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %3\n\t"
      "global_load_lds_dwordx4 %2, %3 offset:1024"
      :: "s"(lds_addr), "v"(v0), "v"(v1), "s"(gbase) : "memory", "m0");
}
#pragma clang diagnostic pop

// One copy of 256 bytes, 4 a lane: lane l's at gbase[v0 .. +4) to LDS lds_addr + 4 l.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma_256(uint32_t lds_addr, const char* gbase, uint32_t v0) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :: "s"(lds_addr), "v"(v0), "s"(gbase) : "memory", "m0");
}
#pragma clang diagnostic pop

// One copy of 1 KB, 16 bytes a lane from an address of its own, to LDS lds_addr + 16 l of lane l
// (of those that take part).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma_lanes(uint32_t lds_addr, const void* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds_addr), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop

// Waits for the loads of x here.  Left to its first use, within a loop, the compiler's
// wait would come round with every turn and take the loop's own copies with it.
template <int N>
__device__ __forceinline__ void arrived(i4 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// How a launch's workgroups go over the heads.  They are dispatched round-robin over
// the 8 XCDs; a head's `units` of work are dealt into `parts` parts and the parts to
// the XCDs, so that each L2 holds the keys and values of few heads and every XCD gets
// long and short items.
struct Deal {
  int units, parts, per_xcd;   // of a head, of a head, parts of all heads on an XCD
  __host__ __device__ unsigned groups() const { return (unsigned)(8 * per_xcd) * (unsigned)((units + parts - 1) / parts); }
};
// Parts: whole heads on an XCD where possible, and all 8 where what `heads` heads of
// `bytes` read fits one L2 together.
inline Deal deal(int64_t heads, int64_t units, int64_t bytes) {
  int parts = 8;
  while (parts > 1 && heads * (parts / 2) % 8 == 0 && (heads * bytes > (int64_t)3 << 20 || parts > units)) parts /= 2;
  return Deal{(int)units, parts, (int)(heads * parts / 8)};
}
// Whether its grid holds less than 2^31 workgroups of less than 2^32 threads.
inline bool deal_fits(int64_t heads, int64_t units) { return heads * 8 * ((units + 7) / 8 + 1) <= INT32_MAX / 256; }
// -> the unit of this workgroup, of head `head`; at least `units`: none.
__device__ __forceinline__ int dealt(const Deal& d, int block, int& head) {
  const int at_xcd = block >> 3;
  const int part = at_xcd % d.per_xcd * 8 + (block & 7);
  head = part / d.parts;
  return at_xcd / d.per_xcd * d.parts + part % d.parts;
}

}  // namespace sidon_attn
