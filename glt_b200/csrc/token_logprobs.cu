// Log probabilities of given tokens, entropy and the most likely tokens of rows of
// logits, and their gradient (glt_token_logprobs, glt_token_logprobs_bwd).
//
// With z = scale x, the running maximum m and the sums s = sum 2^d, t = sum 2^d d of
// d = (z - m) / ln 2:  lse = m + ln s,  entropy = ln s - ln 2 t / s.  One pass over the
// logits finds all three, and the maximum that each thread meets on the way decides
// where the most likely tokens can be: the `top`-th largest of the threads' maxima has
// `top` logits at or above it, so only the shares of the threads whose maximum reaches
// it (about `top` of 256) are read again, from L2.
//
// HBM bounds both kernels: the forward reads the logits once, the backward reads and
// writes them once.  An element costs the forward about five instructions, one of them
// on the special-function unit (16 a clock and SM, against the 12 bf16 logits that HBM
// brings): sums run two at a time (f32x2), maxima and clamps in packed bf16.
//
// Measured: 4096 x 128256 bf16 170 us without the most likely tokens (6.2 TB/s), 188 with 5 of them; the gradient of
// 2047 x 128257 176 us (6.0 TB/s read and written).
//
// A row belongs to one CTA; with fewer rows than would fill the SMs, to a cluster of up
// to eight, joined over distributed shared memory.
#include <cooperative_groups.h>
#include <float.h>
#include <math.h>

#include "common.cuh"
#include "gemm.cuh"

namespace cg = cooperative_groups;

namespace glt {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCtasPerSm = 4;
constexpr int kMaxTop = 32;
constexpr int kBatch = 4;            // 16-byte vectors a thread has in flight
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// The fast path takes exponents as a x - a m in one fused sum, for |a m| up to kNear: beyond it a logit's
// own spacing is 1/8 or more, and further up a m overflows while the logits are finite.  What the rounding
// of a m adds to every exponent (carried() below) is known exactly and taken off the sums whenever they are
// compared with others: at a maximum of 1000 it was 1.6e-5 of a log probability.
// Logits below kFloor count as probability 0 there, which is exact: with a scale of 1e-6 or more, m is above -1e12.
constexpr float kFloor = -1e30f, kNear = 1048576.f;
// Exponents a x - fl(a m) are (x - m) a plus this; `near_to` is kNear, or below 0 with a scale that the fast path leaves out.
__device__ __forceinline__ float carried(float m, float a, float near_to) {
  return fabsf(m * a) <= near_to ? fmaf(m, a, -(m * a)) : 0.f;
}

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const uint16_t* p) { return bf16_bits_to_f32(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = bf16_bits_rn(v); }

// A row as 16-byte vectors, with `head` and `tail` elements outside of them.
template <typename T>
struct RowView {
  static constexpr int kVec = 16 / sizeof(T);
  const T* x;
  int V, head, nv, tail;
  __device__ __forceinline__ RowView(const T* x_, int V_) : x(x_), V(V_) {
    head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
    if (head > V) head = V;
    nv = (V - head) / kVec;
    tail = V - head - nv * kVec;
  }
  __device__ __forceinline__ const uint4* vec(int v) const { return reinterpret_cast<const uint4*>(x + head) + v; }
  // index of the e-th element outside of the vectors
  __device__ __forceinline__ int edge(int e) const { return e < head ? e : V - tail + (e - head); }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 2) {
    unpack8(u, f);
  } else {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  }
}

// Largest element, NaN if any is.
template <typename T>
__device__ __forceinline__ float vector_max(const uint4 (&b)[kBatch]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = b[0].x;
    auto take = [&](uint32_t w) { asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w)); };
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (j) take(b[j].x);
      take(b[j].y), take(b[j].z), take(b[j].w);
    }
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(bf16_lo(m)), "f"(bf16_hi(m)));
    return r;
  } else {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      for (uint32_t w : {b[j].x, b[j].y, b[j].z, b[j].w}) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(w)));
    return m;
  }
}

// Two floats in one 64-bit register, and sums on them.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Rank of a logit as a 64-bit key: larger logits first, then lower indices.
// NaN ranks below every number; -0 equals +0.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = (u >> 31) ? ~u : (u | 0x80000000u);
  if (x != x) u = 0;
  return (static_cast<uint64_t>(u) << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xFFFFFFFFu - static_cast<uint32_t>(k); }

// Running statistics of some logits: maximum m (a logit), sums to base 2^(a (x - m)).
struct Stats {
  float m, s, t;
  __device__ __forceinline__ void join(float m2, float s2, float t2, float a) {
    const float top = fmaxf(m, m2);
    if (top == -INFINITY) return;
    // the difference before the product: m and m2 may be large and close
    const float d1 = m == -INFINITY ? 0.f : (m - top) * a, d2 = m2 == -INFINITY ? 0.f : (m2 - top) * a;
    const float f1 = exp2f(d1), f2 = exp2f(d2);
    const float u1 = s > 0.f && f1 > 0.f ? f1 * fmaf(s, d1, t) : 0.f, u2 = s2 > 0.f && f2 > 0.f ? f2 * fmaf(s2, d2, t2) : 0.f;
    s = s * f1 + s2 * f2;
    t = u1 + u2;
    m = top;
  }
};

// The larger (or smaller) of a lane's key and its partner's.
__device__ __forceinline__ void exchange(uint64_t& key, int partner, bool larger) {
  const uint64_t o = __shfl_xor_sync(0xffffffffu, key, partner);
  if ((o > key) == larger) key = o;
}

// A warp's 32 keys in falling order.
__device__ __forceinline__ uint64_t falling(uint64_t key, int lane) {
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int d = n >> 1; d > 0; d >>= 1) exchange(key, d, ((lane & d) == 0) == ((lane & n) == 0 || n == 32));
  return key;
}

// The largest keys a warp has seen, one a lane in falling order (0: none).
struct TopList {
  uint64_t key = 0;
  // Takes another falling list (`other`: this lane's entry).
  __device__ __forceinline__ void merge(uint64_t other, int lane) {
    const uint64_t o = __shfl_sync(0xffffffffu, other, 31 - lane);
    if (o > key) key = o;   // the 32 largest of both, rising then falling
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) exchange(key, d, (lane & d) == 0);
  }
  // Takes 32 keys in any order.
  __device__ __forceinline__ void merge_unsorted(uint64_t other, int lane) { merge(falling(other, lane), lane); }
  // Takes every lane's candidate (0: none) that ranks above the top-th.
  __device__ __forceinline__ void take(uint64_t cand, int top, int lane) {
    uint32_t who = __ballot_sync(0xffffffffu, cand > __shfl_sync(0xffffffffu, key, top - 1));
    while (who) {
      const int from = __ffs(who) - 1;
      who &= who - 1;
      const uint64_t k = __shfl_sync(0xffffffffu, cand, from);
      const int at = __popc(__ballot_sync(0xffffffffu, key > k));
      const uint64_t up = __shfl_up_sync(0xffffffffu, key, 1);
      if (lane == at) key = k;
      if (lane > at) key = up;
    }
  }
};

constexpr int kPick = (kMaxTop + kWarps - 1) / kWarps + 2;   // maxima a warp puts forward
constexpr int kCand = 256;                                   // logits that reach `least`, before the slow way
struct RowSmem {
  Stats stats[kWarps];
  uint64_t least;                  // a key that `top` logits of this CTA reach (0: there may be fewer)
  union {
    uint64_t maxima[kWarps * kPick];
    uint64_t cand[kCand];
    uint64_t lists[kWarps][32];
  };
  unsigned char slots[kThreads];   // threads whose share is read again
  int nslots, ncand, bad;
  // joined over the cluster by its first CTA
  Stats cta;
  int cta_bad;
  uint64_t cta_keys[kMaxTop];
};

template <typename T, int CLUSTER>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) token_logprobs_kernel(
    const T* __restrict__ logits, int64_t ld, int V, const int32_t* __restrict__ targets, float scale,
    int top, float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ lse_out,
    int32_t* __restrict__ top_ids, float* __restrict__ top_logp, int ahead, unsigned int* err) {
  using Row = RowView<T>;
  constexpr int kVec = Row::kVec;
  __shared__ RowSmem sm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = blockIdx.x / CLUSTER;
  const int rank = blockIdx.x % CLUSTER;
  const Row row(logits + r * ld, V);
  // this CTA's vectors [v0, v1)
  const int v0 = static_cast<int>(static_cast<int64_t>(row.nv) * rank / CLUSTER);
  const int v1 = static_cast<int>(static_cast<int64_t>(row.nv) * (rank + 1) / CLUSTER);
  const float a = scale * kLog2e;
  if (threadIdx.x == 0) {
    sm.nslots = sm.ncand = sm.bad = 0;
    sm.least = 0;
  }

  // ---- one pass
  Stats st{-INFINITY, 0.f, 0.f};
  bool bad = false;
  // first vector of the batch where st.m was met first; -1: no vectors
  int best = v0 + static_cast<int>(threadIdx.x) < v1 ? v0 + static_cast<int>(threadIdx.x) : -1;
  uint64_t s2 = 0, t2 = 0;
  const uint64_t aa = pair(a, a);
  auto load = [&](uint4 (&b)[kBatch], int v) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int at = v + j * kThreads;
      if (at < v1)
        b[j] = *row.vec(at);
      else if constexpr (sizeof(T) == 2)
        b[j] = make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u);
      else
        b[j] = make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
    }
  };
  uint4 cur[kBatch], nxt[kBatch];
  const float near_to = scale >= 1e-6f && scale <= 1e6f ? kNear : -1.f;
  load(nxt, v0 + threadIdx.x);
  for (int v = v0 + threadIdx.x; v < v1; v += kBatch * kThreads) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) cur[j] = nxt[j];
    load(nxt, v + kBatch * kThreads);
    const float cm = vector_max<T>(cur);
    if (!(cm < INFINITY)) bad = true;
    if (cm > st.m) {
      if (st.m > -INFINITY) {
        // from one rounded product to the other, or as far as one of them is out of the fast path's range
        const float from = __fmul_rn(st.m, a), to = __fmul_rn(cm, a);
        float d = from - to;
        if (!(fmaxf(fabsf(from), fabsf(to)) <= near_to))
          d = (st.m - cm) * a + (carried(cm, a, near_to) - carried(st.m, a, near_to));
        const float f = exp2f(d);
        float s0, s1, t0, t1;
        unpair(s2, s0, s1);
        unpair(t2, t0, t1);
        s2 = pair(s0 * f, s1 * f);
        t2 = f > 0.f ? pair(f * fmaf(s0, d, t0), f * fmaf(s1, d, t1)) : 0;
      }
      st.m = cm;
      best = v;
    }
    const float ma = st.m * a;
    if (fabsf(ma) <= near_to) {
      const uint64_t mm = pair(-ma, -ma);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const uint32_t w[4] = {cur[j].x, cur[j].y, cur[j].z, cur[j].w};
#pragma unroll
        for (int q = 0; q < (sizeof(T) == 2 ? 4 : 2); ++q) {
          uint64_t x;
          if constexpr (sizeof(T) == 2) {
            uint32_t c;
            asm("max.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(w[q]), "r"(0xF149F149u));   // -1e30 in bf16
            x = pair(bf16_lo(c), bf16_hi(c));
          } else {
            x = pair(fmaxf(__uint_as_float(w[2 * q]), kFloor), fmaxf(__uint_as_float(w[2 * q + 1]), kFloor));
          }
          const uint64_t d = fma2(x, aa, mm);
          float d0, d1;
          unpair(d, d0, d1);
          const uint64_t e = pair(ex2_approx(d0), ex2_approx(d1));
          s2 = add2(s2, e);
          t2 = fma2(e, d, t2);
        }
      }
    } else if (st.m > -INFINITY) {
      float s0, s1, t0, t1;
      unpair(s2, s0, s1);
      unpair(t2, t0, t1);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        float f[kVec];
        unpack<T>(cur[j], f);
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          const float d = (f[k] - st.m) * a, e = exp2f(d);
          s0 += e;
          if (e > 0.f) t0 = fmaf(e, d, t0);
        }
      }
      s2 = pair(s0, s1);
      t2 = pair(t0, t1);
    }
  }
  // While this row's sums are joined, the two first batches of the row that one of the SM's CTAs takes
  // next come to L2 (4096 x 128256 bf16, when it was brought in: 188 us without, 185 with; 2047 with the gradient: 286 and 280).
  if (CLUSTER == 1 && threadIdx.x == 0 && r + ahead < gridDim.x) {
    const Row next(logits + (r + ahead) * ld, V);
    const int bytes = min(next.nv, 2 * kBatch * kThreads) * 16;
    if (bytes > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(next.vec(0)), "r"(bytes));
  }
  {
    float s0, s1, t0, t1;
    unpair(s2, s0, s1);
    unpair(t2, t0, t1);
    const float off = carried(st.m, a, near_to), f = 1.f / ex2_approx(off);   // a lone token's sum is this 2^off
    st.s = f * (s0 + s1);
    st.t = f * fmaf(-off, s0 + s1, t0 + t1);
  }
  // what this thread's vectors can rank: at best (its maximum, first index of the batch), surely
  // no worse than (its maximum, last index)
  uint64_t upper = 0, lower = 0;
  if (top > 0 && best >= 0) {
    int last = best;   // the thread's own last vector of the batch: no two threads may share a lower key
#pragma unroll
    for (int j = 1; j < kBatch; ++j)
      if (best + j * kThreads < v1) last = best + j * kThreads;
    upper = rank_key(st.m, row.head + best * kVec);
    lower = rank_key(st.m, row.head + last * kVec + kVec - 1);
  }
  // elements outside of the vectors: one a thread of the first CTA
  const int edges = rank == 0 ? row.head + row.tail : 0;
  uint64_t edge_key = 0;
  if (threadIdx.x < edges) {
    const int i = row.edge(threadIdx.x);
    const float x = logit(row.x + i);
    if (!(x < INFINITY)) bad = true;
    edge_key = rank_key(x, i);
    if (x > -INFINITY) st.join(x, 1.f, 0.f, a);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st.join(__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
            __shfl_xor_sync(0xffffffffu, st.t, o), a);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) sm.stats[warp] = st;
  // every warp's few largest lower keys
  const int pick = (top + kWarps - 1) / kWarps + 2;
  if (top > 0) {
    const uint64_t sorted = falling(lower, lane);
    if (lane < pick) sm.maxima[warp * pick + lane] = sorted;
  }
  __syncthreads();
  if (lane == 0 && bad) sm.bad = 1;
  if (top > 0 && threadIdx.x < kWarps * pick) {
    // the one that top - 1 others exceed
    const uint64_t mine = sm.maxima[threadIdx.x];
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kWarps * pick; ++i) above += sm.maxima[i] > mine;
    if (above == top - 1 && mine > 0) sm.least = mine;
  }
  __syncthreads();
  bad = sm.bad;

  // ---- the most likely tokens of this CTA
  if (top > 0) {
    const uint64_t least = sm.least;
    if (upper >= least && upper > 0) sm.slots[atomicAdd(&sm.nslots, 1)] = threadIdx.x;
    __syncthreads();
    auto offer = [&](uint64_t key) {
      if (key < least) return;
      const int at = atomicAdd(&sm.ncand, 1);
      if (at < kCand) sm.cand[at] = key;
    };
    if (!bad) {
      const int per = (v1 - v0 + kThreads - 1) / kThreads;
      for (int i = threadIdx.x; i < sm.nslots * per; i += kThreads) {
        const int slot = i / per, at = v0 + sm.slots[slot] + (i - slot * per) * kThreads;
        if (at >= v1) continue;
        float f[kVec];
        unpack<T>(*row.vec(at), f);
#pragma unroll
        for (int k = 0; k < kVec; ++k) offer(rank_key(f[k], row.head + at * kVec + k));
      }
      if (threadIdx.x < edges) offer(edge_key);
    }
    __syncthreads();
    const int n = sm.ncand;
    if (bad || n > kCand) {
      // more equal logits than places, or NaN or +inf, where the maxima say nothing: every vector again
      __syncthreads();   // `lists` takes the place of `cand`
      TopList list;
      for (int v = v0 + warp * 32; v < v1; v += kThreads) {
        const int at = v + lane;
        float f[kVec];
        if (at < v1) unpack<T>(*row.vec(at), f);
#pragma unroll
        for (int k = 0; k < kVec; ++k) list.take(at < v1 ? rank_key(f[k], row.head + at * kVec + k) : 0, top, lane);
      }
      if (warp == 0) list.take(edge_key, top, lane);   // the edges are all in the first warp
      sm.lists[warp][lane] = list.key;
      __syncthreads();
      if (warp == 0) {
        for (int w = 1; w < kWarps; ++w) list.merge(sm.lists[w][lane], lane);
        sm.cta_keys[lane] = list.key;
      }
    } else if (warp == 0) {
      TopList list;
      for (int i = 0; i < n; i += 32) list.merge_unsorted(i + lane < n ? sm.cand[i + lane] : 0, lane);
      sm.cta_keys[lane] = list.key;
    }
  }
  if (warp == 0) {
    if (lane == 0) {
      Stats all = sm.stats[0];
      for (int w = 1; w < kWarps; ++w) all.join(sm.stats[w].m, sm.stats[w].s, sm.stats[w].t, a);
      sm.cta = all;
      sm.cta_bad = bad;
    }
  }
  if constexpr (CLUSTER > 1) cg::this_cluster().sync();
  if (rank == 0 && warp == 0) {
    __syncwarp();
    Stats all = sm.cta;
    TopList list;
    if (top > 0) list.key = sm.cta_keys[lane];
    if constexpr (CLUSTER > 1) {
      Stats part[CLUSTER];
      uint64_t keys[CLUSTER];
#pragma unroll
      for (int c = 1; c < CLUSTER; ++c) {
        const RowSmem* o = cg::this_cluster().map_shared_rank(&sm, c);
        part[c] = o->cta;
        if (o->cta_bad) bad = true;
        keys[c] = top > 0 ? o->cta_keys[lane] : 0;
      }
#pragma unroll
      for (int c = 1; c < CLUSTER; ++c) {
        all.join(part[c].m, part[c].s, part[c].t, a);
        if (top > 0) list.merge(keys[c], lane);
      }
    }
    const bool empty = all.m == -INFINITY;
    const float ls = logf(fmaxf(all.s, 1.f));   // the maximum's own term is 1
    const float lse = bad ? NAN : empty ? -INFINITY : fmaf(all.m, scale, ls);
    // log probability of a logit: the difference to the maximum first, so that nothing large cancels,
    // unless it is beyond the float range and its product with a scale below 1 is not
    auto log_p = [&](float x) {
      if (bad) return NAN;
      if (empty) return -INFINITY;
      const float d = (x - all.m) * scale;
      return (d > -INFINITY || x == -INFINITY ? d : fmaf(x, scale, -(all.m * scale))) - ls;
    };
    if (lane == 0) {
      lse_out[r] = lse;
      if (entropy) entropy[r] = bad ? NAN : empty ? 0.f : fmaf(-kLn2, all.t / all.s, ls);
      if (targets) {
        int g = targets[r];
        if (g >= V) {
          if (err) atomicOr(err, GLT_DEVERR_BAD_SHAPE);
          g = -1;
        }
        logp[r] = g < 0 ? 0.f : log_p(logit(row.x + g));
      }
    }
    if (lane < top) {
      const uint32_t id = key_index(list.key);
      top_ids[r * top + lane] = static_cast<int32_t>(id);
      top_logp[r * top + lane] = log_p(logit(row.x + id));
    }
  }
  if constexpr (CLUSTER > 1) cg::this_cluster().sync();   // the others' shared memory was read
}

// Rows from the last one back: right after the forward, L2 still holds those.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(
    const T* logits, int64_t ld, int rows, int V, const int32_t* __restrict__ targets, float scale,
    const float* __restrict__ lse, const float* __restrict__ entropy, const float* __restrict__ d_logp,
    const float* __restrict__ d_entropy, T* dlogits, int64_t ld_d) {
  constexpr int kVec = 16 / sizeof(T);
  const int64_t r = rows - 1 - static_cast<int64_t>(blockIdx.x);
  const int g = targets ? targets[r] : -1;
  const bool given = g >= 0 && g < V;
  const float dl = d_logp && given ? d_logp[r] : 0.f;
  const float de = d_entropy ? d_entropy[r] : 0.f;
  const float l = lse[r], h = d_entropy ? entropy[r] : 0.f;
  const float base = fmaf(de, h, dl);   // dl + de * (log p + H) = base + de * log p
  // log p = z - lse.  Below -200 (it may be -inf) p is 0 in 32 bits, and the floor keeps the product with
  // it 0; NaN stays NaN.
  const float w = -scale * de, w0 = -scale * base, from = l == -INFINITY ? 0.f : -l;
  auto grad = [&](float x) {
    float lp = fmaf(x, scale, from);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(lp) : "f"(-200.f));
    return ex2_approx(lp * kLog2e) * fmaf(w, lp, w0);
  };
  const RowView<T> row(logits + r * ld, V);
  T* out = dlogits + r * ld_d;
  const int step = gridDim.y * kThreads;
  const int first = blockIdx.y * kThreads + threadIdx.x;
  auto one = [&](int i) { put(out + i, grad(logit(row.x + i)) + (i == g && l != -INFINITY ? scale * dl : 0.f)); };
  if (((reinterpret_cast<uintptr_t>(row.x) ^ reinterpret_cast<uintptr_t>(out)) & 15) != 0) {
    for (int i = first; i < V; i += step) one(i);   // no common vectors
    return;
  }
  const int hot = given && l != -INFINITY ? g - row.head : -1;
  for (int v = first; v < row.nv; v += kBatch * step) {
    uint4 b[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (v + j * step < row.nv) b[j] = __ldcs(row.vec(v + j * step));
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int at = v + j * step;
      if (at >= row.nv) break;
      float f[kVec];
      unpack<T>(b[j], f);
#pragma unroll
      for (int k = 0; k < kVec; ++k) f[k] = grad(f[k]);
      if (hot >= 0 && hot / kVec == at)
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (hot - at * kVec == k) f[k] += scale * dl;
      uint4 u;
      if constexpr (sizeof(T) == 2)
        u = make_uint4(pack_bf16x2_rn(f[0], f[1]), pack_bf16x2_rn(f[2], f[3]), pack_bf16x2_rn(f[4], f[5]), pack_bf16x2_rn(f[6], f[7]));
      else
        u = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      __stcs(reinterpret_cast<uint4*>(out + row.head) + at, u);
    }
  }
  if (first < row.head + row.tail) one(row.edge(first));
}

int check(const void* logits, int dtype, int64_t ld, int rows, int V, float scale) {
  if (dtype != 0 && dtype != 1) return fail(GLT_EINVAL, "token_logprobs: dtype %d (0 fp32, 1 bf16)", dtype);
  if (rows < 0 || V < 1 || ld < V) return fail(GLT_EINVAL, "token_logprobs: rows %d, V %d, ld %lld", rows, V, (long long)ld);
  if (!(scale > 0.f) || !(scale <= FLT_MAX)) return fail(GLT_EINVAL, "token_logprobs: scale must be positive and finite");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype ? 2 : 4)) return fail(GLT_EINVAL, "token_logprobs: logits not aligned to their type");
  return GLT_OK;
}

struct Args {
  const void* logits;
  int64_t ld;
  int rows, V;
  const int32_t* targets;
  float scale;
  int top;
  float *logp, *entropy, *lse;
  int32_t* top_ids;
  float* top_logp;
};

template <typename T, int CLUSTER>
int launch_forward(const Args& f, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(f.rows) * CLUSTER);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CLUSTER;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  GLT_CUDA_TRY(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, CLUSTER>, static_cast<const T*>(f.logits), f.ld, f.V,
                                  f.targets, f.scale, f.top, f.logp, f.entropy, f.lse, f.top_ids, f.top_logp,
                                  kCtasPerSm * num_sms(), device_error_word()));
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

// CTAs a row: while the rows alone leave SMs idle, as long as each CTA keeps two batches a thread.
template <typename T>
int forward(const Args& f, cudaStream_t st) {
  const int64_t batch = static_cast<int64_t>(kBatch) * kThreads * 16 / sizeof(T);
  int c = 1;
  while (c < 8 && static_cast<int64_t>(f.rows) * c < num_sms() && f.V >= 4 * c * batch) c *= 2;
  if (c == 8) return launch_forward<T, 8>(f, st);
  if (c == 4) return launch_forward<T, 4>(f, st);
  if (c == 2) return launch_forward<T, 2>(f, st);
  return launch_forward<T, 1>(f, st);
}

template <typename T>
int backward(const void* logits, int64_t ld, int rows, int V, const int32_t* targets, float scale, const float* lse,
             const float* entropy, const float* d_logp, const float* d_entropy, void* dlogits, int64_t ld_d, cudaStream_t st) {
  // CTAs a row: enough for all SMs, each with a batch a thread
  const int64_t batch = static_cast<int64_t>(kBatch) * kThreads * 16 / sizeof(T);
  int64_t y = (8ll * num_sms() + rows - 1) / rows;
  const int64_t most = (V + batch - 1) / batch;
  if (y > most) y = most;
  if (y > 65535) y = 65535;
  token_logprobs_bwd_kernel<T><<<dim3(rows, static_cast<unsigned>(y)), kThreads, 0, st>>>(
      static_cast<const T*>(logits), ld, rows, V, targets, scale, lse, entropy, d_logp, d_entropy,
      static_cast<T*>(dlogits), ld_d);
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

}  // namespace
}  // namespace glt

extern "C" int glt_token_logprobs(const void* logits, int dtype, int64_t ld, int rows, int V,
                                  const int32_t* targets, float scale, int top, float* logp,
                                  float* entropy, float* lse, int32_t* top_ids, float* top_logp,
                                  void* stream) {
  if (rows > 0 && (!logits || !lse)) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check(logits, dtype, ld, rows, V, scale));
  if (rows > INT_MAX / 8) return glt::fail(GLT_EINVAL, "token_logprobs: rows %d (at most %d)", rows, INT_MAX / 8);
  if (top < 0 || top > glt::kMaxTop || top > V)
    return glt::fail(GLT_EINVAL, "token_logprobs: top %d (0..%d, at most V)", top, glt::kMaxTop);
  if (rows > 0 && top > 0 && (!top_ids || !top_logp)) return glt::fail(GLT_EINVAL, "token_logprobs: top without outputs");
  if (rows > 0 && (targets != nullptr) != (logp != nullptr))
    return glt::fail(GLT_EINVAL, "token_logprobs: targets and logp go together");
  if (rows == 0) return GLT_OK;
  const glt::Args f{logits, ld, rows, V, targets, scale, top, logp, entropy, lse, top_ids, top_logp};
  return dtype ? glt::forward<uint16_t>(f, static_cast<cudaStream_t>(stream))
               : glt::forward<float>(f, static_cast<cudaStream_t>(stream));
}

extern "C" int glt_token_logprobs_bwd(const void* logits, int dtype, int64_t ld, int rows, int V,
                                      const int32_t* targets, float scale, const float* lse,
                                      const float* entropy, const float* d_logp,
                                      const float* d_entropy, void* dlogits, int64_t ld_d,
                                      void* stream) {
  if (rows > 0 && (!logits || !lse || !dlogits)) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check(logits, dtype, ld, rows, V, scale));
  if (ld_d < V) return glt::fail(GLT_EINVAL, "token_logprobs: ld_d %lld below V %d", (long long)ld_d, V);
  if (d_logp && !targets) return glt::fail(GLT_EINVAL, "token_logprobs: d_logp without targets");
  if (d_entropy && !entropy) return glt::fail(GLT_EINVAL, "token_logprobs: d_entropy without the forward's entropy");
  if (reinterpret_cast<uintptr_t>(dlogits) % (dtype ? 2 : 4))
    return glt::fail(GLT_EINVAL, "token_logprobs: dlogits not aligned to their type");
  if (logits == dlogits && ld != ld_d) return glt::fail(GLT_EINVAL, "token_logprobs: in place needs ld = ld_d");
  if (rows == 0) return GLT_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype)
    return glt::backward<uint16_t>(logits, ld, rows, V, targets, scale, lse, entropy, d_logp, d_entropy, dlogits, ld_d, st);
  return glt::backward<float>(logits, ld, rows, V, targets, scale, lse, entropy, d_logp, d_entropy, dlogits, ld_d, st);
}
