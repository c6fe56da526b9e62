// Shared parts of the 8-bit key/value cache kernels (kv8_append.cu, kv8_attention.cu).
#pragma once

#include <math.h>

#include "common.cuh"
#include "gemm.cuh"

namespace glt {

// Host checks shared by every call on a cache.
int kv8_check(const GltKv8Cache* c, const GltKv8Batch* b);

// The most new rows a sequence can bring: max_new is the caller's bound, and may say less than the others.
inline int kv8_most_new(const GltKv8Cache& c, const GltKv8Batch& b) {
  const int64_t room = static_cast<int64_t>(b.max_blocks) * c.block_tokens;
  const int most = b.max_new < b.rows ? b.max_new : b.rows;
  return most < room ? most : static_cast<int>(room);
}

// Where sequence b stands in this step: `past` tokens held before it, new rows
// [row0, row0 + n).  n = 0 for a sequence without new rows and for one that
// does not fit the batch's bounds (which also sets the device error word when
// err is given).
struct Kv8Span {
  int past, n, row0;
};
__device__ __forceinline__ Kv8Span kv8_span(const GltKv8Batch& b, int seq, int block_tokens, unsigned int* err) {
  Kv8Span s;
  s.past = b.lengths[seq];
  if (b.row_start) {
    s.row0 = b.row_start[seq];
    const int end = b.row_start[seq + 1];
    s.n = s.row0 < 0 || end < s.row0 || end > b.rows ? -1 : end - s.row0;
  } else {
    s.n = b.rows / b.num_seqs;
    s.row0 = seq * s.n;
  }
  const int64_t room = static_cast<int64_t>(b.max_blocks) * block_tokens;
  if (s.n < 0 || s.n > b.max_new || s.past < 0 || static_cast<int64_t>(s.past) + s.n > room) {
    if (err) atomicOr(err, GLT_DEVERR_BAD_SHAPE);
    s.n = 0;
    s.past = 0;
  }
  return s;
}

// Block id of a sequence's block, -1 (and the error word) when outside the pool.
__device__ __forceinline__ int64_t kv8_block(const GltKv8Cache& c, const GltKv8Batch& b, int seq, int index,
                                             unsigned int* err) {
  const int id = b.block_table[static_cast<int64_t>(seq) * b.max_blocks + index];
  if (id >= 0 && id < c.num_blocks) return id;
  if (err) atomicOr(err, GLT_DEVERR_BAD_SHAPE);
  return -1;
}

// Two e4m3 codes (the low 16 bits) as two f16 numbers: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
  return r;
}
__device__ __forceinline__ float kv8_decode(uint32_t code, int format) {
  if (format == GLT_KV8_INT8) return static_cast<float>(code) - 128.f;
  const uint32_t h = e4m3x2_to_f16x2(code & 0xFFu);
  float f;
  asm("{.reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.f32.f16 %0, lo;}" : "=f"(f) : "r"(h));
  return f;
}
// The four codes of a word.
template <int FMT>
__device__ __forceinline__ void kv8_decode4(uint32_t w, float (&f)[4]) {
  if constexpr (FMT == GLT_KV8_INT8) {
    // a code in the low mantissa bits of 2^23
#pragma unroll
    for (int q = 0; q < 4; ++q) f[q] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 + q)) - 8388736.f;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t two = e4m3x2_to_f16x2(h ? w >> 16 : w & 0xFFFFu);
      asm("{.reg .b16 lo, hi; mov.b32 {lo, hi}, %2; cvt.f32.f16 %0, lo; cvt.f32.f16 %1, hi;}"
          : "=f"(f[2 * h]), "=f"(f[2 * h + 1])
          : "r"(two));
    }
  }
}
// Largest code magnitude of a format.
__device__ __forceinline__ float kv8_top(int format) { return format == GLT_KV8_INT8 ? 127.f : 448.f; }
// Nearest code of a value already divided by its scale (ties to even), saturating.
__device__ __forceinline__ uint32_t kv8_encode(float y, int format) {
  if (format == GLT_KV8_INT8)
    return static_cast<uint32_t>(static_cast<int>(rintf(fminf(fmaxf(y, -127.f), 127.f))) + 128);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(y));
  return r & 0xFFu;
}

}  // namespace glt
