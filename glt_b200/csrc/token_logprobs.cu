// Log probabilities of given tokens, entropy and the most likely tokens of rows
// of logits, and their gradient (glt_token_logprobs, glt_token_logprobs_bwd).
#include <float.h>
#include <math.h>

#include "common.cuh"
#include "gemm.cuh"

namespace glt {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;

template <typename T>
__device__ __forceinline__ float load_logit(const T* p);
template <>
__device__ __forceinline__ float load_logit<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load_logit<uint16_t>(const uint16_t* p) { return bf16_bits_to_f32(*p); }
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(uint16_t* p, float v) { *p = bf16_bits_rn(v); }

// Rank of a logit as a 64-bit key: larger logits first, then lower indices.
// NaN ranks below every number; -0 equals +0.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = (u >> 31) ? ~u : (u | 0x80000000u);
  if (x != x) u = 0;
  return (static_cast<uint64_t>(u) << 32) | (0xFFFFFFFFu - index);
}

template <typename Op, typename V>
__device__ __forceinline__ V block_reduce(V v, V* red, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kThreads / 32; ++w) v = op(v, red[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(
    const T* __restrict__ logits, int64_t ld, int V, const int32_t* __restrict__ targets, float scale,
    int top, float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ lse_out,
    int32_t* __restrict__ top_ids, float* __restrict__ top_logp, unsigned int* err) {
  __shared__ float redf[kThreads / 32];
  __shared__ unsigned long long redk[kThreads / 32];
  const int64_t r = blockIdx.x;
  const T* x = logits + r * ld;
  auto fmx = [](float a, float b) { return fmaxf(a, b); };
  auto add = [](float a, float b) { return a + b; };
  float m = -INFINITY, bad = 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float z = load_logit(x + i) * scale;
    if (!(z < INFINITY)) bad = 1.f;
    m = fmaxf(m, z);
  }
  m = block_reduce(m, redf, fmx);
  bad = block_reduce(bad, redf, fmx);
  float s = 0.f, t = 0.f;
  if (m > -INFINITY)
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float d = load_logit(x + i) * scale - m;
      const float e = expf(d);
      s += e;
      if (e > 0.f) t += e * d;
    }
  s = block_reduce(s, redf, add);
  t = block_reduce(t, redf, add);
  const float lse = bad > 0.f ? NAN : m + logf(s);
  const bool empty = m == -INFINITY;
  if (threadIdx.x == 0) {
    lse_out[r] = empty && bad == 0.f ? -INFINITY : lse;
    if (entropy) entropy[r] = bad > 0.f ? NAN : empty ? 0.f : logf(s) - t / s;
    if (targets) {
      int g = targets[r];
      if (g >= V) {
        if (err) atomicOr(err, GLT_DEVERR_BAD_SHAPE);
        g = -1;
      }
      logp[r] = g < 0 ? 0.f : bad > 0.f ? NAN : empty ? -INFINITY : load_logit(x + g) * scale - lse;
    }
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < top; ++j) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const unsigned long long k = rank_key(load_logit(x + i), i);
      if (k < last && k > best) best = k;
    }
    best = block_reduce(best, redk, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
    last = best;
    if (threadIdx.x == 0) {
      const int id = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best));
      top_ids[r * top + j] = id;
      top_logp[r * top + j] = bad > 0.f ? NAN : empty ? -INFINITY : load_logit(x + id) * scale - lse;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(
    const T* logits, int64_t ld, int V, const int32_t* __restrict__ targets, float scale,
    const float* __restrict__ lse, const float* __restrict__ entropy, const float* __restrict__ d_logp,
    const float* __restrict__ d_entropy, T* dlogits, int64_t ld_d) {
  const int64_t r = blockIdx.x;
  const int g = targets ? targets[r] : -1;
  const float dl = (d_logp && g >= 0 && g < V) ? d_logp[r] : 0.f;
  const float de = d_entropy ? d_entropy[r] : 0.f;
  const float l = lse[r], h = d_entropy ? entropy[r] : 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float z = load_logit(logits + r * ld + i) * scale;
    float d = 0.f;
    if (l != -INFINITY) {
      const float lp = z - l, p = expf(lp);
      d = p == 0.f ? 0.f : -p * (dl + de * (lp + h));
      if (i == g) d += dl;
    }
    store_logit(dlogits + r * ld_d + i, d * scale);
  }
}

}  // namespace
}  // namespace glt

extern "C" int glt_token_logprobs(const void* logits, int dtype, int64_t ld, int rows, int V,
                                  const int32_t* targets, float scale, int top, float* logp,
                                  float* entropy, float* lse, int32_t* top_ids, float* top_logp,
                                  void* stream) {
  if (rows > 0 && (!logits || !lse)) return glt::fail(GLT_EINVAL, "null argument");
  if (dtype != 0 && dtype != 1) return glt::fail(GLT_EINVAL, "token_logprobs: dtype %d (0 fp32, 1 bf16)", dtype);
  if (rows < 0 || V < 1 || ld < V) return glt::fail(GLT_EINVAL, "token_logprobs: rows %d, V %d, ld %lld", rows, V, (long long)ld);
  if (!(scale > 0.f) || !(scale <= FLT_MAX)) return glt::fail(GLT_EINVAL, "token_logprobs: scale must be positive and finite");
  if (top < 0 || top > glt::kMaxTop || top > V)
    return glt::fail(GLT_EINVAL, "token_logprobs: top %d (0..%d, at most V)", top, glt::kMaxTop);
  if (rows > 0 && top > 0 && (!top_ids || !top_logp)) return glt::fail(GLT_EINVAL, "token_logprobs: top without outputs");
  if (rows > 0 && (targets != nullptr) != (logp != nullptr))
    return glt::fail(GLT_EINVAL, "token_logprobs: targets and logp go together");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype ? 2 : 4))
    return glt::fail(GLT_EINVAL, "token_logprobs: logits not aligned to their type");
  if (rows == 0) return GLT_OK;
  unsigned int* err = glt::device_error_word();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype)
    glt::token_logprobs_kernel<<<rows, glt::kThreads, 0, st>>>(
        static_cast<const uint16_t*>(logits), ld, V, targets, scale, top, logp, entropy, lse, top_ids, top_logp, err);
  else
    glt::token_logprobs_kernel<<<rows, glt::kThreads, 0, st>>>(
        static_cast<const float*>(logits), ld, V, targets, scale, top, logp, entropy, lse, top_ids, top_logp, err);
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

extern "C" int glt_token_logprobs_bwd(const void* logits, int dtype, int64_t ld, int rows, int V,
                                      const int32_t* targets, float scale, const float* lse,
                                      const float* entropy, const float* d_logp,
                                      const float* d_entropy, void* dlogits, int64_t ld_d,
                                      void* stream) {
  if (rows > 0 && (!logits || !lse || !dlogits)) return glt::fail(GLT_EINVAL, "null argument");
  if (dtype != 0 && dtype != 1) return glt::fail(GLT_EINVAL, "token_logprobs: dtype %d (0 fp32, 1 bf16)", dtype);
  if (rows < 0 || V < 1 || ld < V || ld_d < V)
    return glt::fail(GLT_EINVAL, "token_logprobs: rows %d, V %d, ld %lld, ld_d %lld", rows, V, (long long)ld, (long long)ld_d);
  if (!(scale > 0.f) || !(scale <= FLT_MAX)) return glt::fail(GLT_EINVAL, "token_logprobs: scale must be positive and finite");
  if (d_logp && !targets) return glt::fail(GLT_EINVAL, "token_logprobs: d_logp without targets");
  if (d_entropy && !entropy) return glt::fail(GLT_EINVAL, "token_logprobs: d_entropy without the forward's entropy");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype ? 2 : 4) || reinterpret_cast<uintptr_t>(dlogits) % (dtype ? 2 : 4))
    return glt::fail(GLT_EINVAL, "token_logprobs: buffers not aligned to their type");
  if (logits == dlogits && ld != ld_d) return glt::fail(GLT_EINVAL, "token_logprobs: in place needs ld = ld_d");
  if (rows == 0) return GLT_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype)
    glt::token_logprobs_bwd_kernel<<<rows, glt::kThreads, 0, st>>>(
        static_cast<const uint16_t*>(logits), ld, V, targets, scale, lse, entropy, d_logp, d_entropy,
        static_cast<uint16_t*>(dlogits), ld_d);
  else
    glt::token_logprobs_bwd_kernel<<<rows, glt::kThreads, 0, st>>>(
        static_cast<const float*>(logits), ld, V, targets, scale, lse, entropy, d_logp, d_entropy,
        static_cast<float*>(dlogits), ld_d);
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}
