// sidon_host.h -- host-side helpers shared by the library's translation units
// (error text, device check).  Not part of the C ABI: every symbol here has
// hidden visibility.
#pragma once

#include <stdint.h>

#include "sidon_flexrel.h"

namespace sidon {

// Record a printf-style message as the thread's last error; returns `code`.
int fail(int code, const char* fmt, ...);
// Clear the thread's last error (start of every entry point).
void clear_error();
// SIDON_OK when the current HIP device is a gfx950, else SIDON_E_DEVICE.
int check_device();
// Compute units of the current device (after a successful check_device).
int compute_units();

// The tiled GEMM kernel's fp16-output form (gemm.hip): y = act(x . w^T + bias)
// with one rounding, act 1 = SiLU of the fp32 sum.  gemm_half_takes: the
// operands fit it and it is expected to beat the library; gemm_half launches
// it on operands that fit.
bool gemm_half_preferred(int M, int N, int K);
bool gemm_half_takes(const void* x, int ldx, const void* w, int ldw, const void* bias, const void* y, int ldy, int M,
                     int N, int K);
int gemm_half(const void* x, int ldx, const void* w, int ldw, const void* bias, void* y, int ldy, int M, int N, int K,
              int act, void* stream);

inline bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

// Whether two ranges of bytes share memory.
inline bool ranges_meet(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t ab = reinterpret_cast<uintptr_t>(a), bb = reinterpret_cast<uintptr_t>(b);
  return ab < bb + (uintptr_t)b_bytes && bb < ab + (uintptr_t)a_bytes;
}
// Whether `rows` rows of `width` bytes, `pitch` apart, share memory with a range: one
// between two rows does not.
inline bool row_meets(const void* a, int64_t pitch, int64_t width, int64_t rows, const void* b, int64_t bytes) {
  if (!ranges_meet(a, (rows - 1) * pitch + width, b, bytes)) return false;
  const int64_t on = (int64_t)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a));
  return on < 0 || on % pitch < width || on % pitch + bytes > pitch;
}
// Whether `rows` rows of a_width and b_width bytes, a_pitch and b_pitch apart, share
// memory.  Column blocks of one wider tensor do not, though their ranges meet.
inline bool rows_meet(const void* a, int64_t a_pitch, int64_t a_width, const void* b, int64_t b_pitch, int64_t b_width,
                      int64_t rows) {
  if (!ranges_meet(a, (rows - 1) * a_pitch + a_width, b, (rows - 1) * b_pitch + b_width)) return false;
  if (a_pitch != b_pitch) return true;
  const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a)) % a_pitch;
  const int64_t on = d < 0 ? d + a_pitch : d;   // from a's column to b's
  return on < a_width || a_pitch - on < b_width;
}

// Elements from the first to past the last of sizes n and strides st, with `last` contiguous ones.
inline __int128 span(const int* n, const int64_t* st, int dims, int last) {
  __int128 e = last;
  for (int i = 0; i < dims; ++i) e += (__int128)(n[i] - 1) * st[i];
  return e;
}

// Whether rows of `last` elements lie apart: in the order of their strides, every
// dimension steps past all that the ones before it cover.
inline bool apart(const int* n, const int64_t* st, int dims, int last) {
  __int128 covered = last;
  bool used[3] = {};
  for (int k = 0; k < dims; ++k) {
    int at = -1;
    for (int i = 0; i < dims; ++i)
      if (!used[i] && (at < 0 || st[i] < st[at])) at = i;
    used[at] = true;
    if (n[at] == 1) continue;
    if (st[at] < covered) return false;
    covered += (__int128)(n[at] - 1) * st[at];
  }
  return true;
}

// Rows of `last` elements of `size` bytes over (batch, head, row), with element strides.
struct Rows {
  const void* at;
  int n[3];
  int64_t st[3];
  int last, size;
  __int128 bytes() const { return span(n, st, 3, last) * size; }
};
// Whether two such tensors may share memory.  Those whose ranges meet do not where some step
// of theirs divides them: dimensions of steps that are multiples of it shift either tensor
// by whole pitches, the others stay within one, and there in columns apart (column blocks of one
// wider tensor, items of two tensors in turn).
inline bool tensors_meet(const Rows& a, const Rows& b) {
  if (!ranges_meet(a.at, (int64_t)a.bytes(), b.at, (int64_t)b.bytes())) return false;
  for (const Rows* by : {&a, &b})
    for (int i = 0; i < 3; ++i) {
      if (by->n[i] == 1 || by->st[i] <= 0) continue;
      const int64_t pitch = by->st[i] * by->size;
      __int128 width[2];
      int k = 0;
      for (const Rows* t : {&a, &b}) {
        __int128 w = t->last;
        for (int d = 0; d < 3; ++d)
          if (t->st[d] * t->size % pitch != 0) w += (__int128)(t->n[d] - 1) * t->st[d];
        width[k++] = w * t->size;
      }
      const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(b.at) - reinterpret_cast<uintptr_t>(a.at)) % pitch;
      const int64_t on = d < 0 ? d + pitch : d;   // from a's column to b's
      if (on >= width[0] && pitch - on >= width[1]) return false;
    }
  return true;
}

}  // namespace sidon
