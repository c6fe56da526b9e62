// Attention of a step's queries over the 8-bit key/value cache (glt_kv8_attention).
#include <float.h>

#include "kv8.cuh"

namespace glt {
namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ float block_max(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
__device__ __forceinline__ float block_add(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// One CTA a (query, head): 128 tokens at a time with a running maximum and sum.
__global__ void __launch_bounds__(kThreads) kv8_attention_kernel(GltKv8Cache c, GltKv8Batch b,
                                                                 const uint16_t* __restrict__ q, int64_t ld_q,
                                                                 uint16_t* __restrict__ o, int64_t ld_o,
                                                                 float* __restrict__ lse, int nh, float scale,
                                                                 int window, const uint8_t* __restrict__ mask,
                                                                 int64_t ld_mask, unsigned int* err) {
  __shared__ float sq[128], sp[kThreads], red[4];
  const int seq = blockIdx.y, head = blockIdx.z, kvh = head / (nh / c.num_kv_heads);
  const bool first = blockIdx.x == 0 && head == 0 && threadIdx.x == 0;
  const Kv8Span span = kv8_span(b, seq, c.block_tokens, first ? err : nullptr);
  for (int i = blockIdx.x; i < span.n; i += gridDim.x) {
    const int64_t row = span.row0 + i;
    const int pos = span.past + i;
    __syncthreads();
    if (threadIdx.x < c.head_dim) sq[threadIdx.x] = bf16_bits_to_f32(q[row * ld_q + head * c.head_dim + threadIdx.x]);
    __syncthreads();
    const int t0 = window > 0 ? max(0, pos - window + 1) : 0;
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int base = t0; base <= pos; base += kThreads) {
      const int t = base + threadIdx.x;
      float s = -INFINITY;
      if (t <= pos && (!mask || mask[seq * ld_mask + t])) {
        const int64_t id = kv8_block(c, b, seq, t / c.block_tokens, err);
        if (id >= 0) {
          const int64_t hb = id * c.num_kv_heads + kvh;
          const uint8_t* kr = c.k + (hb * c.block_tokens + t % c.block_tokens) * c.head_dim;
          s = 0.f;
          for (int d = 0; d < c.head_dim; ++d) s += sq[d] * kv8_decode(kr[d], c.format);
          s *= c.k_scale[hb] * scale;
        }
      }
      const float mx = fmaxf(m, block_max(s, red));
      if (mx == -INFINITY) continue;
      const float corr = expf(m - mx), p = expf(s - mx);
      m = mx;
      l = l * corr + block_add(p, red);
      acc *= corr;
      __syncthreads();
      sp[threadIdx.x] = p;
      __syncthreads();
      const int n = min(kThreads, pos + 1 - base);
      if (threadIdx.x < c.head_dim)
        for (int j = 0; j < n; ++j) {
          if (sp[j] == 0.f) continue;
          const int tj = base + j;
          const int64_t id = kv8_block(c, b, seq, tj / c.block_tokens, nullptr);
          const int64_t hb = id * c.num_kv_heads + kvh;
          acc += sp[j] * (c.v_scale[hb] *
                          kv8_decode(c.v[(hb * c.block_tokens + tj % c.block_tokens) * c.head_dim + threadIdx.x], c.format));
        }
    }
    if (threadIdx.x < c.head_dim)
      o[row * ld_o + head * c.head_dim + threadIdx.x] = bf16_bits_rn(m == -INFINITY ? 0.f : acc / l);
    if (lse && threadIdx.x == 0) lse[row * nh + head] = m == -INFINITY ? -INFINITY : m + logf(l);
  }
}

int check_heads(const GltKv8Cache* c, const GltKv8Batch* b, int nh) {
  GLT_TRY(kv8_check(c, b));
  if (nh < 1 || nh % c->num_kv_heads || nh > 65535)
    return fail(GLT_EINVAL, "kv8: num_heads %d must be a multiple of num_kv_heads %d", nh, c->num_kv_heads);
  return GLT_OK;
}

}  // namespace
}  // namespace glt

extern "C" int glt_kv8_attention_workspace(const GltKv8Cache* cache, const GltKv8Batch* batch,
                                           int num_heads, int64_t* bytes) {
  if (!bytes) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_heads(cache, batch, num_heads));
  *bytes = 0;
  return GLT_OK;
}

extern "C" int glt_kv8_attention(const GltKv8Cache* cache, const GltKv8Batch* batch, const uint16_t* q,
                                 int64_t ld_q, uint16_t* o, int64_t ld_o, float* lse, int num_heads,
                                 float scale, int window, const uint8_t* token_mask, int64_t ld_mask,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  GLT_TRY(glt::check_heads(cache, batch, num_heads));
  if (batch->rows == 0 || batch->max_new == 0) return GLT_OK;
  if (!q || !o) return glt::fail(GLT_EINVAL, "null argument");
  const int64_t width = static_cast<int64_t>(num_heads) * cache->head_dim;
  if (ld_q < width || ld_o < width || ld_q % 8 || ld_o % 8 || !glt::aligned16(q) || !glt::aligned16(o))
    return glt::fail(GLT_EINVAL, "kv8: q and o rows must be 16-byte aligned (strides multiples of 8, at least %lld)", (long long)width);
  if (!(scale >= 0.f) || scale > FLT_MAX) return glt::fail(GLT_EINVAL, "kv8: scale must be finite and not negative");
  if (window < 0) return glt::fail(GLT_EINVAL, "kv8: negative window");
  if (token_mask && ld_mask < static_cast<int64_t>(batch->max_blocks) * cache->block_tokens)
    return glt::fail(GLT_EINVAL, "kv8: mask row stride below max_blocks * block_tokens");
  int64_t need = 0;
  GLT_TRY(glt_kv8_attention_workspace(cache, batch, num_heads, &need));
  if (workspace_bytes < need || (need > 0 && (!workspace || !glt::aligned16(workspace))))
    return glt::fail(GLT_EINVAL, "kv8: workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
  const dim3 grid(batch->max_new < 65535 ? batch->max_new : 65535, batch->num_seqs, num_heads);
  glt::kv8_attention_kernel<<<grid, glt::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      *cache, *batch, q, ld_q, o, ld_o, lse, num_heads, scale > 0.f ? scale : 1.f / sqrtf(static_cast<float>(cache->head_dim)),
      window, token_mask, ld_mask, glt::device_error_word());
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}
