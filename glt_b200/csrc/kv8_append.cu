// Writing and reading the 8-bit key/value cache (glt_kv8_append, glt_kv8_read).
#include <float.h>

#include "kv8.cuh"

namespace glt {

int kv8_check(const GltKv8Cache* c, const GltKv8Batch* b) {
  if (!c || !b) return fail(GLT_EINVAL, "null argument");
  if (c->format != GLT_KV8_INT8 && c->format != GLT_KV8_E4M3) return fail(GLT_EINVAL, "kv8: format %d", c->format);
  const int bt = c->block_tokens;
  if (bt != 16 && bt != 32 && bt != 64 && bt != 128)
    return fail(GLT_EINVAL, "kv8: block_tokens %d (16, 32, 64 or 128)", bt);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(GLT_EINVAL, "kv8: head_dim %d (64 or 128)", c->head_dim);
  if (c->num_kv_heads < 1 || c->num_kv_heads > 4096) return fail(GLT_EINVAL, "kv8: num_kv_heads %d", c->num_kv_heads);
  if (c->num_blocks < 1 || c->num_blocks > INT_MAX) return fail(GLT_EINVAL, "kv8: num_blocks %lld", (long long)c->num_blocks);
  if (c->num_blocks * c->num_kv_heads * bt > INT_MAX)
    return fail(GLT_EINVAL, "kv8: a pool of %lld rows (at most 2^31 - 1)", (long long)(c->num_blocks * c->num_kv_heads * bt));
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(GLT_EINVAL, "kv8: null cache buffer");
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(GLT_EINVAL, "kv8: cache pools must be 16-byte aligned");
  if (b->num_seqs < 0 || b->num_seqs > 65535 || b->rows < 0 || b->max_new < 0)
    return fail(GLT_EINVAL, "kv8: num_seqs %d (0..65535), rows %d, max_new %d", b->num_seqs, b->rows, b->max_new);
  if (b->num_seqs == 0 && b->rows > 0) return fail(GLT_EINVAL, "kv8: rows without sequences");
  if (b->num_seqs > 0) {
    if (b->max_blocks < 1 || static_cast<int64_t>(b->max_blocks) * bt > INT_MAX - 4096)
      return fail(GLT_EINVAL, "kv8: max_blocks %d", b->max_blocks);
    if (!b->block_table || !b->lengths) return fail(GLT_EINVAL, "kv8: null block table or lengths");
    if (!b->row_start && b->rows % b->num_seqs)
      return fail(GLT_EINVAL, "kv8: %d rows for %d sequences need row_start", b->rows, b->num_seqs);
    if (!b->row_start && b->rows / b->num_seqs > b->max_new)
      return fail(GLT_EINVAL, "kv8: %d new rows a sequence, max_new %d", b->rows / b->num_seqs, b->max_new);
  }
  return GLT_OK;
}

namespace {

constexpr int kThreads = 256;

// Eight codes of x / s, exactly: s, or 1 / s, may be out of the fast way's range, x not finite.
__device__ __forceinline__ uint2 codes_exact(const float (&x)[8], float s, int format) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float y = s > 0.f && x[q] == x[q] ? x[q] / s : 0.f;
    w[q >> 2] |= kv8_encode(y, format) << (8 * (q & 3));
  }
  return make_uint2(w[0], w[1]);
}

// The same without a division, for s >= 2^-60 and finite x, r being 1 / s rounded to nearest.  A quotient within a unit
// in the last place becomes the one rounded to nearest by q + r (x - q s), both sums fused (Markstein's theorem, IBM
// Journal of Research and Development 34, 1990); x r may be off by a little more, so there is one step before.  Nothing
// underflows that matters: below 2^-11 the code is 0.
// 24 prompts of 2048 tokens x 8 heads x 128: 105 us with divisions, 77 us so.  (Products with two neighbours of r and
// a division where their codes differ took 88: values that meet a boundary, as half the maximum does, are one in 200.)
template <int FMT>
__device__ __forceinline__ uint2 codes_fast(const float (&x)[8], float s, float r) {
  float y[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    y[q] = x[q] * r;
    y[q] = fmaf(fmaf(-y[q], s, x[q]), r, y[q]);
    y[q] = fmaf(fmaf(-y[q], s, x[q]), r, y[q]);
  }
  uint32_t w[2];
  if constexpr (FMT == GLT_KV8_INT8) {
    // y + 1.5 2^23 is rounded to an integer, whose low byte is the code less its offset
    uint32_t a[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) a[q] = __float_as_uint(y[q] + 12582912.f);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = __byte_perm(__byte_perm(a[4 * h], a[4 * h + 1], 0x0040), __byte_perm(a[4 * h + 2], a[4 * h + 3], 0x0040), 0x5410) ^ 0x80808080u;
  } else {
    uint16_t a[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a[q]) : "f"(y[2 * q + 1]), "f"(y[2 * q]));
    w[0] = a[0] | static_cast<uint32_t>(a[1]) << 16;
    w[1] = a[2] | static_cast<uint32_t>(a[3]) << 16;
  }
  return make_uint2(w[0], w[1]);
}

// One CTA: the part of one sequence's new tokens that falls into one block, for
// one KV head, keys (z = 0) or values (z = 1).  The rows are read once and kept
// in registers between the scale and the codes.  HBM bounds prompts, the chain length ->
// table -> scale bounds single tokens, so all that can be is loaded before the maximum.
// VECS: vectors of eight values a thread holds of a whole block.
template <int FMT, int VECS>
__global__ void __launch_bounds__(kThreads, VECS <= 4 ? 4 : 3) kv8_append_kernel(GltKv8Cache c, GltKv8Batch b,
                                                              const uint16_t* __restrict__ k, int64_t ld_k,
                                                              const uint16_t* __restrict__ v, int64_t ld_v,
                                                              unsigned int* err) {
  __shared__ float red[kThreads / 32];
  const int seq = blockIdx.y, head = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  const Kv8Span sp = kv8_span(b, seq, c.block_tokens, blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0 ? err : nullptr);
  const int index = sp.past / c.block_tokens + blockIdx.x;
  const int base = index * c.block_tokens;
  const int lo = max(sp.past, base) - base, hi = min(sp.past + sp.n, base + c.block_tokens) - base;
  if (lo >= hi) return;
  const int vec_log = c.head_dim == 128 ? 4 : 3;   // vectors of eight values in a row
  const int64_t ld = is_v ? ld_v : ld_k;
  const uint16_t* src = (is_v ? v : k) + (sp.row0 + static_cast<int64_t>(base + lo - sp.past)) * ld + head * c.head_dim;
  const int n = (hi - lo) << vec_log, held = lo << vec_log;
  uint4 x[VECS];   // on its way beside the block's id
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    const int i = threadIdx.x + j * kThreads;
    if (i < n) x[j] = *reinterpret_cast<const uint4*>(src + (i >> vec_log) * ld + (i & ((1 << vec_log) - 1)) * 8);
  }
  const int64_t id = kv8_block(c, b, seq, index, blockIdx.z == 0 && threadIdx.x == 0 ? err : nullptr);
  if (id < 0) return;
  const int64_t slab = (id * c.num_kv_heads + head) * c.block_tokens * c.head_dim;
  uint2* codes = reinterpret_cast<uint2*>((is_v ? c.v : c.k) + slab);
  float* scale = (is_v ? c.v_scale : c.k_scale) + id * c.num_kv_heads + head;
  // the block's own tokens of earlier steps keep its scale from falling
  const float before = lo > 0 ? *scale : 0.f;
  uint2 old[VECS];
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    const int i = threadIdx.x + j * kThreads;
    if (i < held) old[j] = codes[i];
  }
  // magnitudes of bf16 order like their bits, two at a time
  uint32_t two = 0;
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    if (threadIdx.x + j * kThreads >= n) break;
    const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
    for (int q = 0; q < 4; ++q) asm("max.u16x2 %0, %0, %1;" : "+r"(two) : "r"(w[q] & 0x7FFF7FFFu));
  }
  float peak = __uint_as_float(max(two >> 16, two & 0xFFFFu) << 16);
  const bool odd = !(peak <= FLT_MAX);   // something not finite among this thread's values
  if (odd) {
    peak = 0.f;
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      if (threadIdx.x + j * kThreads >= n) break;
      float f[8];
      unpack8(x[j], f);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (fabsf(f[q]) <= FLT_MAX) peak = fmaxf(peak, fabsf(f[q]));
    }
  }
  peak = warp_max(peak);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = peak;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) peak = fmaxf(peak, red[w]);
  const float after = fmaxf(before, peak / kv8_top(FMT));
  const float r = 1.f / after;
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    const int i = threadIdx.x + j * kThreads;
    if (i >= n) break;
    float f[8];
    unpack8(x[j], f);
    codes[held + i] = !odd && after >= 0x1p-60f ? codes_fast<FMT>(f, after, r) : codes_exact(f, after, FMT);
  }
  if (after > before) {
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      const int i = threadIdx.x + j * kThreads;
      if (i >= held) break;
      const uint32_t o[2] = {old[j].x, old[j].y};
      float f[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float d[4];
        kv8_decode4<FMT>(o[h], d);
#pragma unroll
        for (int q = 0; q < 4; ++q) f[4 * h + q] = fmaxf(d[q], -kv8_top(FMT)) * before;   // -128 is no code of ours
      }
      codes[i] = after >= 0x1p-60f ? codes_fast<FMT>(f, after, r) : codes_exact(f, after, FMT);
    }
  }
  // every thread has read the old scale (before the barrier above)
  if (threadIdx.x == 0 && (lo == 0 || after > before)) *scale = after;
}

// One CTA: the positions of one sequence that lie in one block, for one KV head, keys (z = 0) or values.
constexpr int kReadBatch = 8;
template <int FMT>
__global__ void __launch_bounds__(kThreads) kv8_read_kernel(GltKv8Cache c, GltKv8Batch b,
                                                            const int32_t* __restrict__ start, int count,
                                                            float* __restrict__ k, float* __restrict__ v,
                                                            unsigned int* err) {
  const int seq = blockIdx.y, bt = c.block_tokens;
  const Kv8Span sp = kv8_span(b, seq, bt, blockIdx.x == 0 && threadIdx.x == 0 ? err : nullptr);
  const int64_t from = start ? start[seq] : 0;
  const int64_t end = sp.past + sp.n;
  // cut at multiples of a block's tokens, below zero too
  const int64_t cut = (from >= 0 ? from / bt : -((-from + bt - 1) / bt)) + blockIdx.x;
  const int64_t p0 = max(from, cut * bt), p1 = min(from + count, (cut + 1) * bt);
  if (p0 >= p1) return;
  int64_t id = -1;
  if (p0 >= 0 && p0 < end) id = kv8_block(c, b, seq, static_cast<int>(cut), threadIdx.x == 0 ? err : nullptr);
  const int vec_log = c.head_dim == 128 ? 5 : 4, vecs = 1 << vec_log;   // of four values
  const int head = blockIdx.z >> 1, total = static_cast<int>(p1 - p0) << vec_log;
  const bool is_v = blockIdx.z & 1;
  const int64_t hb = id * c.num_kv_heads + head;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>((is_v ? c.v : c.k) + (hb * bt + (p0 - cut * bt)) * c.head_dim);
  const int held = id >= 0 ? static_cast<int>(min(static_cast<int64_t>(total), (end - p0) << vec_log)) : 0;   // vectors the sequence holds
  const float s = held > 0 ? (is_v ? c.v_scale : c.k_scale)[hb] : 0.f;
  float* dst = (is_v ? v : k) + ((static_cast<int64_t>(seq) * count + (p0 - from)) * c.num_kv_heads + head) * c.head_dim;
  const int64_t row = static_cast<int64_t>(c.num_kv_heads) * c.head_dim;
  for (int u = threadIdx.x; u < total; u += kReadBatch * kThreads) {
    uint32_t w[kReadBatch];
#pragma unroll
    for (int j = 0; j < kReadBatch; ++j) {
      const int i = u + j * kThreads;
      w[j] = FMT == GLT_KV8_INT8 ? 0x80808080u : 0u;   // codes of 0
      if (i < held) w[j] = codes[i];
    }
#pragma unroll
    for (int j = 0; j < kReadBatch; ++j) {
      const int i = u + j * kThreads;
      if (i >= total) break;
      float f[4];
      kv8_decode4<FMT>(w[j], f);
      *reinterpret_cast<float4*>(dst + (i >> vec_log) * row + (i & (vecs - 1)) * 4) = make_float4(f[0] * s, f[1] * s, f[2] * s, f[3] * s);
    }
  }
}

template <int FMT>
int launch_append(const GltKv8Cache& c, const GltKv8Batch& b, const uint16_t* k, int64_t ld_k, const uint16_t* v,
                  int64_t ld_v, cudaStream_t st) {
  // blocks a sequence's new tokens can reach into, the first one partly filled
  const dim3 grid((kv8_most_new(c, b) + c.block_tokens - 2) / c.block_tokens + 1, b.num_seqs, 2 * c.num_kv_heads);
  const int vecs = c.block_tokens * c.head_dim / 8;
  const auto kernel = vecs <= kThreads ? kv8_append_kernel<FMT, 1> : vecs <= 2 * kThreads ? kv8_append_kernel<FMT, 2>
                      : vecs <= 4 * kThreads ? kv8_append_kernel<FMT, 4> : kv8_append_kernel<FMT, 8>;
  kernel<<<grid, kThreads, 0, st>>>(c, b, k, ld_k, v, ld_v, device_error_word());
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

}  // namespace
}  // namespace glt

extern "C" int glt_kv8_append(const GltKv8Cache* cache, const GltKv8Batch* batch, const uint16_t* k,
                              int64_t ld_k, const uint16_t* v, int64_t ld_v, void* stream) {
  GLT_TRY(glt::kv8_check(cache, batch));
  if (batch->rows == 0) return GLT_OK;
  if (!k || !v) return glt::fail(GLT_EINVAL, "null argument");
  const int64_t width = static_cast<int64_t>(cache->num_kv_heads) * cache->head_dim;
  if (ld_k < width || ld_v < width || ld_k % 8 || ld_v % 8 || !glt::aligned16(k) || !glt::aligned16(v))
    return glt::fail(GLT_EINVAL, "kv8: new rows must be 16-byte aligned (strides multiples of 8, at least %lld)", (long long)width);
  if (batch->max_new == 0) return GLT_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->format == GLT_KV8_INT8 ? glt::launch_append<GLT_KV8_INT8>(*cache, *batch, k, ld_k, v, ld_v, st)
                                       : glt::launch_append<GLT_KV8_E4M3>(*cache, *batch, k, ld_k, v, ld_v, st);
}

extern "C" int glt_kv8_read(const GltKv8Cache* cache, const GltKv8Batch* batch, const int32_t* start,
                            int count, float* k, float* v, void* stream) {
  GLT_TRY(glt::kv8_check(cache, batch));
  if (count < 0) return glt::fail(GLT_EINVAL, "kv8: negative count");
  if (count == 0 || batch->num_seqs == 0) return GLT_OK;
  if (!k || !v) return glt::fail(GLT_EINVAL, "null argument");
  if (!glt::aligned16(k) || !glt::aligned16(v)) return glt::fail(GLT_EINVAL, "kv8: outputs must be 16-byte aligned");
  // blocks a range can touch
  const dim3 grid((count + cache->block_tokens - 2) / cache->block_tokens + 1, batch->num_seqs, 2 * cache->num_kv_heads);
  const auto kernel = cache->format == GLT_KV8_INT8 ? glt::kv8_read_kernel<GLT_KV8_INT8> : glt::kv8_read_kernel<GLT_KV8_E4M3>;
  kernel<<<grid, glt::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(*cache, *batch, start, count, k, v,
                                                                       glt::device_error_word());
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}
