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
constexpr int kMaxVec = 128 * 128 / 8 / kThreads;  // 8-value vectors a thread holds of one block

// One CTA: the part of one sequence's new tokens that falls into one block, for
// one KV head, keys (z = 0) or values (z = 1).  The rows are read once and kept
// in registers between the scale and the codes.
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(GltKv8Cache c, GltKv8Batch b,
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
  const int64_t id = kv8_block(c, b, seq, index, blockIdx.z == 0 && threadIdx.x == 0 ? err : nullptr);
  if (id < 0) return;
  const int vecs = c.head_dim >> 3;
  const int64_t slab = (id * c.num_kv_heads + head) * c.block_tokens * c.head_dim;
  uint8_t* codes = (is_v ? c.v : c.k) + slab;
  float* scale = (is_v ? c.v_scale : c.k_scale) + id * c.num_kv_heads + head;
  const int64_t ld = is_v ? ld_v : ld_k;
  const uint16_t* src = (is_v ? v : k) + (sp.row0 + static_cast<int64_t>(base + lo - sp.past)) * ld + head * c.head_dim;
  const int n = (hi - lo) * vecs;
  uint4 x[kMaxVec];
  float peak = 0.f;
#pragma unroll
  for (int j = 0; j < kMaxVec; ++j) {
    const int i = threadIdx.x + j * kThreads;
    if (i >= n) break;
    x[j] = *reinterpret_cast<const uint4*>(src + (i / vecs) * ld + (i % vecs) * 8);
    float f[8];
    unpack8(x[j], f);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float a = fabsf(f[q]);
      if (a <= FLT_MAX) peak = fmaxf(peak, a);
    }
  }
  peak = warp_max(peak);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = peak;
  // the block's own tokens of earlier steps keep its scale from falling
  const float before = lo > 0 ? *scale : 0.f;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) peak = fmaxf(peak, red[w]);
  const float after = fmaxf(before, peak / kv8_top(c.format));
#pragma unroll
  for (int j = 0; j < kMaxVec; ++j) {
    const int i = threadIdx.x + j * kThreads;
    if (i >= n) break;
    float f[8];
    unpack8(x[j], f);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float y = after > 0.f && f[q] == f[q] ? f[q] / after : 0.f;
      w[q >> 2] |= kv8_encode(y, c.format) << (8 * (q & 3));
    }
    *reinterpret_cast<uint2*>(codes + (lo * vecs + i) * 8) = make_uint2(w[0], w[1]);
  }
  if (after > before) {
    for (int i = threadIdx.x; i < lo * vecs; i += kThreads) {
      const uint2 old = *reinterpret_cast<const uint2*>(codes + i * 8);
      const uint32_t o[2] = {old.x, old.y};
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float val = kv8_decode((o[q >> 2] >> (8 * (q & 3))) & 0xFFu, c.format) * before;
        w[q >> 2] |= kv8_encode(val / after, c.format) << (8 * (q & 3));
      }
      *reinterpret_cast<uint2*>(codes + i * 8) = make_uint2(w[0], w[1]);
    }
  }
  // every thread has read the old scale (it is behind the barrier above)
  if (threadIdx.x == 0) *scale = after;
}

// One CTA a position: 8 values a thread of all heads, keys then values.
__global__ void __launch_bounds__(kThreads) kv8_read_kernel(GltKv8Cache c, GltKv8Batch b,
                                                            const int32_t* __restrict__ start, int count,
                                                            float* __restrict__ k, float* __restrict__ v,
                                                            unsigned int* err) {
  const int seq = blockIdx.y;
  const Kv8Span sp = kv8_span(b, seq, c.block_tokens, blockIdx.x == 0 && threadIdx.x == 0 ? err : nullptr);
  const int vecs = c.head_dim >> 3, per = c.num_kv_heads * vecs;
  for (int i = blockIdx.x; i < count; i += gridDim.x) {
    const int64_t pos = (start ? start[seq] : 0) + static_cast<int64_t>(i);
    int64_t id = -1;
    if (pos >= 0 && pos < sp.past + sp.n)
      id = kv8_block(c, b, seq, static_cast<int>(pos / c.block_tokens), threadIdx.x == 0 ? err : nullptr);
    const int64_t out = (static_cast<int64_t>(seq) * count + i) * per * 8;
    for (int u = threadIdx.x; u < 2 * per; u += kThreads) {
      const bool is_v = u >= per;
      const int w = is_v ? u - per : u, head = w / vecs;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (id >= 0) {
        const int64_t hb = id * c.num_kv_heads + head;
        const float s = (is_v ? c.v_scale : c.k_scale)[hb];
        const uint2 old = *reinterpret_cast<const uint2*>((is_v ? c.v : c.k) +
                                                          (hb * c.block_tokens + pos % c.block_tokens) * c.head_dim +
                                                          (w % vecs) * 8);
        const uint32_t o[2] = {old.x, old.y};
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = kv8_decode((o[q >> 2] >> (8 * (q & 3))) & 0xFFu, c.format) * s;
      }
      float* dst = (is_v ? v : k) + out + w * 8;
      reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
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
  const int bt = cache->block_tokens;
  // blocks a sequence's new tokens can reach into, the first one partly filled
  const dim3 grid((batch->max_new + bt - 2) / bt + 1, batch->num_seqs, 2 * cache->num_kv_heads);
  glt::kv8_append_kernel<<<grid, glt::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      *cache, *batch, k, ld_k, v, ld_v, glt::device_error_word());
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

extern "C" int glt_kv8_read(const GltKv8Cache* cache, const GltKv8Batch* batch, const int32_t* start,
                            int count, float* k, float* v, void* stream) {
  GLT_TRY(glt::kv8_check(cache, batch));
  if (count < 0) return glt::fail(GLT_EINVAL, "kv8: negative count");
  if (count == 0 || batch->num_seqs == 0) return GLT_OK;
  if (!k || !v) return glt::fail(GLT_EINVAL, "null argument");
  if (!glt::aligned16(k) || !glt::aligned16(v)) return glt::fail(GLT_EINVAL, "kv8: outputs must be 16-byte aligned");
  const dim3 grid(count < 65535 ? count : 65535, batch->num_seqs);
  glt::kv8_read_kernel<<<grid, glt::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      *cache, *batch, start, count, k, v, glt::device_error_word());
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}
