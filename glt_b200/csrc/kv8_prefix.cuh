// What kv8_prefix_kernel leaves of a prefix that all sequences of a batch share, and how it joins the attention to a
// sequence's own tokens.
//
// Query rows (token x head of the group) of one KV head are cut into tiles of 128.  A unit is one KV head with
// `lanes` neighbouring tiles; its steps of 128 tokens, laid end to end with those of all units, are dealt to
// the CTAs in equal runs.  A CTA leaves, for each unit it has steps of, unnormalised sums of values, maxima (base 2)
// and sums of weights in a slot of its own.
#pragma once

#include "kv8.cuh"

namespace glt {

constexpr int kPrefixStep = 128;   // tokens of a step
constexpr int kPrefixRows = 128;   // query rows of a tile

struct PrefixParts {
  const int32_t* length;   // dev [1]
  int capacity;            // tokens the prefix's blocks hold
  int kv_heads, tiles;     // tiles of query rows a KV head
  int lanes;               // tiles of a unit: 2, or 1, and then the unit's two results are of every second step
  int grid;                // CTAs of the kernel
  float* slots;

  __host__ __device__ int units() const { return kv_heads * ((tiles + lanes - 1) / lanes); }
  static __host__ __device__ int slot_floats(int hd) { return 2 * kPrefixRows * (hd + 2); }
  // A unit's parts lie with consecutive CTAs, and no CTA but a unit's last is also another's, so unit + CTA
  // names a slot.
  __host__ __device__ int64_t bytes(int hd) const { return (static_cast<int64_t>(units()) + grid) * slot_floats(hd) * 4; }
  // Tokens of the prefix; a length that its blocks do not hold counts as none (and sets the error word).
  __device__ __forceinline__ int tokens(unsigned int* err) const {
    const int n = *length;
    if (n >= 0 && n <= capacity) return n;
    if (err) atomicOr(err, GLT_DEVERR_BAD_SHAPE);
    return 0;
  }
};

// The steps of all units in equal runs, the first `more` of them one longer.
struct PrefixShares {
  int64_t each;
  int steps, ctas, more;
  __device__ __forceinline__ PrefixShares(const PrefixParts& p, int tokens) {
    steps = (tokens + kPrefixStep - 1) / kPrefixStep;
    const int64_t total = static_cast<int64_t>(steps) * p.units();
    ctas = total < p.grid ? static_cast<int>(total) : p.grid;
    each = ctas > 0 ? total / ctas : 0;
    more = static_cast<int>(total - each * ctas);
  }
  __device__ __forceinline__ int64_t begin(int i) const { return each * i + min(i, more); }
  __device__ __forceinline__ int owner(int64_t x) const {
    const int64_t head = (each + 1) * more;
    return static_cast<int>(x < head ? x / (each + 1) : more + (x - head) / each);
  }
};

// 2^(m - top) for partial results: weights that saw nothing are 0 (or NaN) already.
__device__ __forceinline__ float join_factor(float m, float top) { return top == -INFINITY ? 1.f : ex2_approx(m - top); }

// Adds the prefix's parts to four channels (from d on) of a query row: its sum z of values, maximum and sum of weights.
__device__ __forceinline__ void join_prefix(const PrefixParts& p, int row, int kvh, int hd, int d, float4& z, float& top,
                                            float& sum) {
  const int tokens = p.tokens(nullptr);
  if (tokens == 0) return;
  const PrefixShares sh(p, tokens);
  const int tile = row / kPrefixRows, r = row % kPrefixRows;
  const int unit = tile / p.lanes * p.kv_heads + kvh;
  const int first = sh.owner(static_cast<int64_t>(unit) * sh.steps);
  const int last = sh.owner(static_cast<int64_t>(unit + 1) * sh.steps - 1);
  // the row's results: one a CTA, or two
  const int lane0 = p.lanes == 2 ? tile & 1 : 0, per = p.lanes == 2 ? 1 : 2;
  const int parts = (last - first + 1) * per, slot = PrefixParts::slot_floats(hd);
  const float* base = p.slots + static_cast<int64_t>(unit + first) * slot;
  constexpr int kBatch = 4;   // parts whose loads are in flight at once
  for (int k0 = 0; k0 < parts; k0 += kBatch) {
    float m[kBatch], l[kBatch];
    float4 x[kBatch];
    float peak = top;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = min(k0 + k, parts - 1);
      const int cta = per == 2 ? i >> 1 : i, lane = per == 2 ? i & 1 : lane0;
      const float* s = base + static_cast<int64_t>(cta) * slot;
      const int at = lane * kPrefixRows + r;
      x[k] = *reinterpret_cast<const float4*>(s + static_cast<int64_t>(at) * hd + d);
      m[k] = s[2 * kPrefixRows * hd + at];
      l[k] = s[2 * kPrefixRows * (hd + 1) + at];
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (k0 + k < parts) peak = fmaxf(peak, m[k]);
    const float old = join_factor(top, peak);
    sum *= old;
    z = make_float4(z.x * old, z.y * old, z.z * old, z.w * old);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (k0 + k >= parts) continue;
      const float f = join_factor(m[k], peak);
      sum = fmaf(l[k], f, sum);
      z.x = fmaf(x[k].x, f, z.x);
      z.y = fmaf(x[k].y, f, z.y);
      z.z = fmaf(x[k].z, f, z.z);
      z.w = fmaf(x[k].w, f, z.w);
    }
    top = peak;
  }
}

}  // namespace glt
