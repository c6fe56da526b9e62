// What kv8_prefix_kernel leaves of a prefix that all sequences of a batch share, and how it joins the attention to a
// sequence's own tokens.
//
// Query rows (token x head of the group) of one KV head are cut into tiles of 128.  A unit is one KV head with
// `lanes` neighbouring tiles; its steps of 64 tokens and what it costs to begin and to end it, laid end to end with
// those of all units, are dealt to the CTAs in equal runs.  A CTA leaves, for each unit it has steps of,
// unnormalised sums of values, maxima (base 2) and sums of weights in a slot of its own.
#pragma once

#include "kv8.cuh"

namespace glt {

constexpr int kPrefixStep = 64;    // tokens of a step
constexpr int kPrefixRows = 128;   // query rows of a tile
constexpr int kPrefixUnitCost = 4;   // what laying out a unit's queries and writing its result cost, in steps

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

// The costs of all units (kPrefixUnitCost and the steps) in equal runs, the first `more` of them one longer.
struct PrefixShares {
  int64_t each;
  int steps, ctas, more;
  __device__ __forceinline__ PrefixShares(const PrefixParts& p, int tokens) {
    steps = (tokens + kPrefixStep - 1) / kPrefixStep;
    const int64_t total = steps > 0 ? static_cast<int64_t>(steps + kPrefixUnitCost) * p.units() : 0;
    ctas = total < p.grid ? static_cast<int>(total) : p.grid;
    each = ctas > 0 ? quotient(total, ctas) : 0;
    more = static_cast<int>(total - each * ctas);
  }
  // by the much shorter 32-bit division where that is enough
  static __device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
  }
  __device__ __forceinline__ int64_t begin(int i) const { return each * i + min(i, more); }
  __device__ __forceinline__ int owner(int64_t x) const {
    const int64_t head = (each + 1) * more;
    return static_cast<int>(x < head ? quotient(x, each + 1) : more + quotient(x - head, each));
  }
};

}  // namespace glt
