// Attention of a step's queries over the 8-bit key/value cache: the kernels of glt_kv8_attention,
// glt_kv8_window_attention (kv8_attention.cu) and, for the sequences' own tokens, glt_kv8_prefix_attention
// (kv8_prefix.cu), which differ in Mode.
//
//   o_i = sum_t p_it v_t / sum_t p_it,   p_it = exp(scale q_i.k_t - m_i),   m_i a running maximum
//
// A few queries meet a long cache, so the cache's bytes bound the kernel: each is
// read once for all query heads that share its KV head.
//
// Work.  A unit is one KV head of one sequence with up to 8 NT of its query rows
// (query token x head of the group); its tokens are cut into steps of 32.  The
// steps of all units, laid end to end, are dealt to the CTAs in equal runs, so a
// batch of any lengths loads all SMs alike; the four warps of a CTA take the steps
// of its run in turn, each with its own maximum and sum, and join at the end of a
// unit.  A unit that crosses CTAs leaves partial results, which a second kernel
// joins.  All sizes are read on the device: a captured graph follows the lengths.
//
// Tensor cores.  Both products have the cache as operand A (16 tokens, or 16
// channels, by 16) and the few queries as operand B (N = 8), in f16 with 32-bit sums:
//   S^T = K . Q^T:  8-bit codes become f16 exactly; a query row is brought to f16 by a
//                   power of two (its bf16 mantissa fits), the block's scale multiplies S.
//   O^T = V^T . P^T: P is rounded to f16 (11 bits), V's codes are exact, the block's scale
//                   multiplies the 32-bit sums of a step.  P is taken from the step's own
//                   maximum times 2^15; a weight still below f16's normal range (2^-29 of
//                   that maximum) is added in 32 bits on the side, so each weight keeps its
//                   11 bits, whatever the values it meets.
// The order of a contraction's index is free, so a lane loads 16 contiguous bytes and
// uses them for four k-steps of S or eight rows of O.
//
// Loads.  A warp keeps its own ring of stages in shared memory: one lane starts two TMA
// copies a step (K and V, 32 rows each, one with blocks of 16 tokens: four), swizzled so
// that the fragment reads meet no bank twice, and the warp waits on the stage's mbarrier.
// No warp waits for another inside a unit, and the copies run ahead across units.
//
// Measured (32 heads over 8, head_dim 128): 4 sequences of 65537 tokens e4m3 91.4 us, 5.9 TB/s of cache; 32 ragged
// sequences of up to 8191 tokens int8 62 us, 5.0 TB/s, the ends of units being the difference.  Many query rows (5 new
// tokens x 8 heads a KV head) are bound by the instructions and their latency: 39 us for 12 sequences, 0.8 TB/s; the
// kernels for 16 query rows of 128 channels hold all 255 registers and spill 188 to 284 bytes a thread.
#pragma once

#include <float.h>
#include <limits.h>

#include <type_traits>

#include "kv8.cuh"

namespace glt {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 32;   // tokens of a step
constexpr float kF16Min = 6.103515625e-05f;   // 2^-14, the smallest normal f16

constexpr int kCtasPerSm = 2;   // three, with smaller rings, took 108 us for the long caches where two took 99
// What beginning and ending a unit costs a CTA, in steps (0.39 us each; measured on 32 ragged
// sequences: 4.5 us a unit, and 76 us in all with 3 where 12 gave 64).
constexpr int kUnitCost = 12;

// kPlain: all earlier tokens, or those of a window.  kSinks: of a window and the first `sinks` tokens.
// kPrefix: all earlier tokens, in 32 bits and not divided by the sum of weights, for a join with a prefix's parts.
enum class Mode { kPlain, kSinks, kPrefix };

struct AttnArgs {
  GltKv8Cache c;
  GltKv8Batch b;
  const uint16_t* q;
  int64_t ld_q;
  uint16_t* o;
  int64_t ld_o;
  float* lse;
  int nh, group;
  float scale;
  int window;
  const uint8_t* mask;
  int64_t ld_mask;
  void* workspace;
  unsigned int* err;
  int sinks;    // kSinks
  float* own;   // kPrefix: dev [rows, num_heads, head_dim] sums of values, then [rows, num_heads] maxima (base 2) and sums of weights
  bool chained; // kPrefix: the launch before is the prefix's, so that this one may start while it runs
};

// Steps that hold a sequence's first tokens.
__device__ __forceinline__ int sink_steps(const AttnArgs& a) { return a.sinks / kStep + (a.sinks % kStep != 0); }

// What one sequence has to do: `steps` steps from token `lo` on, for `units` units.  kSinks: the first sink_steps of them are from
// token 0 on, and lo is 0 where the window's follow without a gap.
struct SeqWork {
  int past, n, row0, lo, steps, units;
  template <Mode M>
  __device__ __forceinline__ int token(const AttnArgs& a, int step) const {
    return (M == Mode::kSinks && step < sink_steps(a) ? 0 : lo) + step * kStep;
  }
  __device__ __forceinline__ int64_t cost() const { return static_cast<int64_t>(steps + kUnitCost) * units; }
};
template <int ROWS, Mode M>
__device__ __forceinline__ SeqWork seq_work(const AttnArgs& a, int seq, unsigned int* err) {
  const Kv8Span s = kv8_span(a.b, seq, a.c.block_tokens, err);
  SeqWork w;
  w.past = s.past;
  w.n = s.n;
  w.row0 = s.row0;
  w.lo = a.window > 0 ? max(0, s.past - a.window + 1) & ~(kStep - 1) : 0;
  if (M == Mode::kSinks) w.lo = max(0, w.lo / kStep - sink_steps(a)) * kStep;
  w.steps = (s.past + s.n - w.lo + kStep - 1) / kStep;
  w.units = s.n > 0 ? a.c.num_kv_heads * ((s.n * a.group + ROWS - 1) / ROWS) : 0;   // n * group is checked on the host
  return w;
}

// a / b by the much shorter 32-bit division where that is enough.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// How the cost of all sequences, laid end to end, is shared: each of `ctas` CTAs gets
// `each`, the first `more` of them one more.
struct Shares {
  int64_t each;
  int ctas, more;
  __device__ __forceinline__ Shares(int64_t total, int grid) {
    const int64_t n = (total + kWarps - 1) / kWarps;   // at least a step for every warp
    ctas = n < grid ? static_cast<int>(n) : grid;
    each = ctas > 0 ? quotient(total, ctas) : 0;
    more = static_cast<int>(total - each * ctas);
  }
  __device__ __forceinline__ int64_t begin(int i) const { return each * i + min(i, more); }
  __device__ __forceinline__ int owner(int64_t x) const {
    const int64_t head = (each + 1) * more;
    return static_cast<int>(x < head ? quotient(x, each + 1) : more + quotient(x - head, each));
  }
};

// A CTA's run of the whole: where it begins, and what it costs.
struct Run {
  int64_t begin, end;   // in the whole
  int64_t base;         // of its first sequence
  int seq;
  SeqWork w;            // of that sequence
};
struct ScanSmem {
  int64_t warp[kWarps];
  Run run;
};
template <int ROWS, Mode M>
__device__ __forceinline__ Shares find_run(const AttnArgs& a, ScanSmem& sm) {
  const int per = (a.b.num_seqs + kThreads - 1) / kThreads;
  const int first = min(a.b.num_seqs, static_cast<int>(threadIdx.x) * per), last = min(a.b.num_seqs, first + per);
  int64_t mine = 0;
  SeqWork w;
  for (int s = first; s < last; ++s) {
    w = seq_work<ROWS, M>(a, s, blockIdx.x == 0 ? a.err : nullptr);
    mine += w.cost();
  }
  int64_t scan = mine, total = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) sm.warp[warp] = scan;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) scan += sm.warp[i];
    total += sm.warp[i];
  }
  const Shares sh(total, gridDim.x);
  const int64_t begin = static_cast<int>(blockIdx.x) < sh.ctas ? sh.begin(blockIdx.x) : total;
  const int64_t end = static_cast<int>(blockIdx.x) < sh.ctas ? sh.begin(blockIdx.x + 1) : total;
  int64_t base = scan - mine;
  if (begin >= base && begin < scan) {   // one thread's, for begin < total
    for (int s = first; s < last; ++s) {
      if (last - first > 1) w = seq_work<ROWS, M>(a, s, nullptr);
      if (begin < base + w.cost()) {
        sm.run.begin = begin;
        sm.run.end = end;
        sm.run.base = base;
        sm.run.seq = s;
        sm.run.w = w;
        break;
      }
      base += w.cost();
    }
  } else if (begin == total && threadIdx.x == 0) {
    sm.run.begin = sm.run.end = total;
  }
  __syncthreads();
  return sh;
}

// Walks a run unit by unit: steps [s0, s1) of each (none where the run only holds a part
// of the unit's kUnitCost).
template <int ROWS, Mode M>
struct Cursor {
  int seq, unit, s0, s1;
  int kvh, tile;   // of the unit
  int64_t at, left;   // position in the sequence's unit, rest of the run
  SeqWork w;
  __device__ __forceinline__ void start(const AttnArgs& a, const Run& r) {
    seq = r.seq;
    left = r.end - r.begin;
    if (left <= 0) return;
    w = r.w;
    const int64_t offset = r.begin - r.base;
    unit = static_cast<int>(quotient(offset, w.steps + kUnitCost));
    tile = unit / a.c.num_kv_heads;
    kvh = unit - tile * a.c.num_kv_heads;
    at = offset - static_cast<int64_t>(unit) * (w.steps + kUnitCost);
    bounds();
  }
  __device__ __forceinline__ void bounds() {
    s0 = max(0, static_cast<int>(at) - kUnitCost);
    s1 = static_cast<int>(min(static_cast<int64_t>(w.steps), at + left - kUnitCost));
  }
  __device__ __forceinline__ void next(const AttnArgs& a) {
    left -= w.steps + kUnitCost - at;
    if (left <= 0) return;
    ++unit;
    if (++kvh == a.c.num_kv_heads) {
      kvh = 0;
      ++tile;
    }
    if (unit == w.units) {
      unit = kvh = tile = 0;
      do {
        if (++seq >= a.b.num_seqs) {   // only if the lengths changed under the kernel
          left = 0;
          return;
        }
        w = seq_work<ROWS, M>(a, seq, nullptr);
      } while (w.units == 0);
    }
    at = 0;
    bounds();
  }
  __device__ __forceinline__ bool whole() const { return s0 == 0 && s1 == w.steps; }
};

// The workspace: what to join (one task a CTA, that begins a unit it does not end), then two
// partial results a CTA: rows x hd sums, rows maxima (base 2), rows sums of weights.
struct JoinTask {
  int parts;        // CTAs that hold a part: this one and the next parts - 1; 0: nothing to join
  int first_slot;   // of this CTA; the others used their first
  int row0, tile, kvh, rows;
  int pad[2];
};
struct Workspace {
  int* ctas;
  JoinTask* tasks;
  float* slots;
  int64_t bytes;
  __host__ __device__ Workspace(void* p, int grid, int rows, int hd) {
    uint8_t* b = static_cast<uint8_t*>(p);
    ctas = reinterpret_cast<int*>(b);
    tasks = reinterpret_cast<JoinTask*>(b + 32);
    slots = reinterpret_cast<float*>(b + 32 + grid * sizeof(JoinTask));
    bytes = 32 + grid * sizeof(JoinTask) + static_cast<int64_t>(grid) * 2 * (rows * hd + 2 * rows) * 4;
  }
};

// Copies 4 bytes (zero where !on: the source is not read then).
__device__ __forceinline__ void copy_async4(void* dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(tc::smem_u32(dst)), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_groups() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from sums of 0.
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// Bytes 0, 1 (HI = 0) or 2, 3 of a word of codes as two f16 numbers.  An int8 code u
// in the low mantissa bits of 1024 is 1024 + u; 1152 less is u - 128.
template <int FMT, int HI>
__device__ __forceinline__ uint32_t two_codes(uint32_t w) {
  if constexpr (FMT == GLT_KV8_INT8) {
    uint32_t r;
    const uint32_t x = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));
    return r;
  } else {
    return e4m3x2_to_f16x2(HI ? w >> 16 : w & 0xFFFFu);
  }
}

// 2^(m - top) for partial results: weights that saw nothing are 0 (or NaN) already.
__device__ __forceinline__ float join_factor(float m, float top) { return top == -INFINITY ? 1.f : ex2_approx(m - top); }

// Where scales of V join the exponents, a number that leaves 32 bits (below 2^-126, counted 2^10 at least at the reference) has less than
// 2^-72 of the weight of the token that made the reference, if their scales lie within a window of 2^64: from 2^-52 (not below
// 2^-90, where values count as 0) to 2^12 of the first one.  Values of 0 weigh as the least scale, 2^-90, so that no reference is
// theirs where a summand is near: beside scales up to 2^8 they have less than 2^-38 then.
// Else weights are summed from numbers 2^kWideLift as large, which the largest, 2^15 and some, bear: they have
// less than 2^-32 of that weight where they leave 32 bits.  (All steps that way: 4096 rows behind 65537 tokens 367 us for 193.)
constexpr float kLeastScale = 0x1p-90f, kMostBesideNone = 0x1p8f;
struct ScaleWindow {
  float low, high;
  __device__ __forceinline__ explicit ScaleWindow(float first) {
    const int e = first >= kLeastScale && first <= FLT_MAX ? static_cast<int>(__float_as_uint(first) >> 23) - 127 : -8;
    low = __int_as_float((max(e - 52, -90) + 127) << 23);
    high = __int_as_float((min(e + 12, 127) + 127) << 23);
  }
};
constexpr float kWideLift = 108.f;
// The sum of weights of tokens whose numbers sum up to `lifted`; log_v and inv_v are their scale's.
__device__ __forceinline__ float wide_weights(float lifted, float log_v, float inv_v) {
  return log_v < 0.f ? lifted * (inv_v * 0x1p-108f) : lifted * inv_v * 0x1p-108f;
}
// 2^d, d <= 0, as two factors, the second 1 down to 2^-120: a sum of weights is taken times both, since where scales of V join the
// exponents it may be as far above 1 as 2^d is below.
struct TwoFactors {
  float a, b;
  __device__ __forceinline__ explicit TwoFactors(float d)
      : a(ex2_approx(fmaxf(d, -120.f))), b(ex2_approx(fminf(d + 120.f, 0.f))) {}
};

// Four channels of a query row from their sum z, the row's maximum (base 2) and sum of
// weights.  A row that saw nothing has weight 0 and gives 0; NaN stays NaN.
template <Mode M>
__device__ __forceinline__ void write_out(const AttnArgs& a, int row0, int r, int kvh, int hd, int d, float4 z,
                                          float top, float sum) {
  const int i = r / a.group, head = kvh * a.group + r - i * a.group;
  const int64_t tok = row0 + i;
  if (M == Mode::kPrefix) {
    const int64_t at = tok * a.nh + head;
    *reinterpret_cast<float4*>(a.own + at * hd + d) = z;
    if (d == 0) *reinterpret_cast<float2*>(a.own + static_cast<int64_t>(a.b.rows) * a.nh * hd + 2 * at) = make_float2(top, sum);
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(a.o + tok * a.ld_o + static_cast<int64_t>(head) * hd + d) =
      make_uint2(pack_bf16x2_rn(z.x * inv, z.y * inv), pack_bf16x2_rn(z.z * inv, z.w * inv));
  if (a.lse && d == 0) a.lse[tok * a.nh + head] = sum == 0.f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
}

// One warp's ring: stages of 32 rows of K, then 32 rows of V; scales and flags beside them.
template <int HD>
struct Ring {
  static constexpr int kStages = HD == 128 ? 2 : 3;
  static constexpr int kPart = kStep * HD;          // bytes of K (or V) of a stage
  static constexpr int kStage = 2 * kPart;
  static constexpr int kWarp = kStages * kStage;
};
struct StageNote {
  float scale[4];   // K, V of the first fold unit; K, V of the second
  int valid;        // bit u: the block of tokens 16 u .. 16 u + 15 is in the pool
  int pad[3];
};
template <int HD, int NT>
constexpr int smem_bytes() {
  return 1024 /* alignment */ + kWarps * Ring<HD>::kWarp + 2 * 8 * NT * (HD + 4) * 4 + kWarps * 8 * NT * 8 +
         kWarps * Ring<HD>::kStages * static_cast<int>(sizeof(StageNote) + 8) + static_cast<int>(sizeof(ScanSmem));
}

template <int HD, int FMT, int NT, bool BT16, Mode M>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv8_attention_kernel(const __grid_constant__ AttnArgs a,
                                                                                   const __grid_constant__ CUtensorMap map_k,
                                                                                   const __grid_constant__ CUtensorMap map_v) {
  constexpr bool kSinks = M == Mode::kSinks;
  constexpr int ROWS = 8 * NT, LU = BT16 ? 2 : 1, kJoinRow = HD + 4;
  // the sums of a step's second half join those of the first, unless each half has its own scale
  // or (NT = 2) holding them would not leave registers enough
  constexpr bool kFoldEach = LU == 2 || NT == 2;
  using R = Ring<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-tc::smem_u32(smem_raw) & 1023u);   // the swizzle goes by address
  float* join_o = reinterpret_cast<float*>(smem + kWarps * R::kWarp);            // [2][ROWS][kJoinRow]
  float2* join_ml = reinterpret_cast<float2*>(join_o + 2 * ROWS * kJoinRow);     // [warp][ROWS]
  StageNote* notes = reinterpret_cast<StageNote*>(join_ml + kWarps * ROWS);
  uint64_t* bars = reinterpret_cast<uint64_t*>(notes + kWarps * R::kStages);
  ScanSmem& scan = *reinterpret_cast<ScanSmem*>(bars + kWarps * R::kStages);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;");
  uint8_t* ring = smem + warp * R::kWarp;
  notes += warp * R::kStages;
  bars += warp * R::kStages;
  if (lane == 0) {
    for (int i = 0; i < R::kStages; ++i) tc::mbar_init(bars + i, 1);
    tc::fence_mbar_init();
  }

  const Shares shares = find_run<ROWS, M>(a, scan);
  const Workspace ws(a.workspace, gridDim.x, ROWS, HD);
  if (blockIdx.x == 0 && threadIdx.x == 0) *ws.ctas = shares.ctas;
  if (scan.run.end <= scan.run.begin) {
    if (M == Mode::kPrefix) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }

  // The copies run kStages steps ahead of the arithmetic, and the block ids one step ahead of
  // the copies: `ld` stands on the next step to copy, whose ids are on their way.
  const int bt_log = 31 - __clz(a.c.block_tokens);
  Cursor<ROWS, M> ld;
  ld.start(a, scan.run);
  int ld_step = ld.s0 + warp, ld_stage = 0, ld_id[LU];
  bool ld_on[LU];   // some query may see tokens of it
  auto seek = [&]() {
    while (ld.left > 0 && ld_step >= ld.s1) {
      ld.next(a);
      ld_step = ld.s0 + warp;
    }
    if (ld.left > 0) {
      const int t = ld.w.template token<M>(a, ld_step);
      const int32_t* ids = a.b.block_table + static_cast<int64_t>(ld.seq) * a.b.max_blocks;
      // of a step's two blocks of 16 the first may lie before the window, and the last beyond the tokens
      ld_on[0] = LU == 1 || a.window == 0 || t + 15 > ld.w.past - a.window || (kSinks && t < a.sinks);
      if (LU == 2) ld_on[LU - 1] = t + 16 < ld.w.past + ld.w.n;
      // (and between first tokens and window may lie more)
      if (LU == 2 && kSinks && t + 16 >= a.sinks && t + 31 <= ld.w.past - a.window) ld_on[LU - 1] = false;
#pragma unroll
      for (int f = 0; f < LU; ++f) ld_id[f] = ld_on[f] ? ids[(t + 16 * f) >> bt_log] : -1;
    }
  };
  // Copies this warp's next step into the next stage.
  int issued = 0;
  auto issue = [&]() {
    if (ld.left > 0) {
      const int t0 = ld.w.template token<M>(a, ld_step);
      uint64_t* bar = bars + ld_stage;
      uint8_t* dst = ring + ld_stage * R::kStage;
      int valid = 0;
#pragma unroll
      for (int f = 0; f < LU; ++f) {
        const bool on = ld_id[f] >= 0 && ld_id[f] < a.c.num_blocks;
        if (on) valid |= LU == 2 ? 1 << f : 3;
        if (!on && ld_on[f] && lane == 0 && a.err) atomicOr(a.err, GLT_DEVERR_BAD_SHAPE);
        const int64_t hb = on ? static_cast<int64_t>(ld_id[f]) * a.c.num_kv_heads + ld.kvh : 0;
        if (lane < 2) copy_async4(notes[ld_stage].scale + f * 2 + lane, (lane ? a.c.v_scale : a.c.k_scale) + hb, on);
      }
      if (lane == 0) {
        notes[ld_stage].valid = valid;
        const int units = LU == 2 ? (valid & 1) + (valid >> 1) : valid ? 1 : 0;
        tc::mbar_arrive_expect_tx(bar, units * (R::kStage / LU));
#pragma unroll
        for (int f = 0; f < LU; ++f) {
          if (!(valid >> f & 1)) continue;
          const int64_t hb = static_cast<int64_t>(ld_id[f]) * a.c.num_kv_heads + ld.kvh;
          const int row = static_cast<int>((hb << bt_log) + ((t0 + 16 * f) & (a.c.block_tokens - 1)));
          tc::tma_load_2d(dst + f * (R::kPart / LU), &map_k, bar, 0, row);
          tc::tma_load_2d(dst + R::kPart + f * (R::kPart / LU), &map_v, bar, 0, row);
        }
      }
      ld_step += kWarps;
      ++issued;
      seek();
    }
    commit();
    ld_stage = ld_stage + 1 == R::kStages ? 0 : ld_stage + 1;
  };
  __syncwarp();   // the barriers are ready
  seek();
#pragma unroll 1
  for (int i = 0; i < R::kStages; ++i) issue();

  Cursor<ROWS, M> cu;
  cu.start(a, scan.run);
  int stage = 0, taken = 0;
  uint32_t phase = 0;
  bool lost = false;   // a copy did not arrive in time
  int done = 0;        // units of the run with steps here
  int64_t base = scan.run.begin - cu.at;   // of the unit in the whole
  JoinTask task = {};
  // A lane's fragment bytes in a stage.  K: rows g + 8 r + 16 u, chunk 2c + h (64-byte rows: c);
  // V: rows 2c + e + 8 r + 16 u, the g-th eighth.
  int off_k[HD / 64], off_v[2];
  if (HD == 128) {
#pragma unroll
    for (int h = 0; h < HD / 64; ++h) off_k[h] = g * HD + (((2 * c + h) ^ g) << 4);
#pragma unroll
    for (int e = 0; e < 2; ++e) off_v[e] = R::kPart + (2 * c + e) * HD + ((g ^ (2 * c + e)) << 4);
  } else {
    off_k[0] = g * HD + ((c ^ (g >> 1)) << 4);
#pragma unroll
    for (int e = 0; e < 2; ++e) off_v[e] = R::kPart + (2 * c + e) * HD + (((g >> 1) ^ c) << 4) + (g & 1) * 8;
  }
  // The queries of the unit that `cu` stands on: operand B's bytes, as they lie in memory.
  auto load_queries = [&](uint4 (&v)[NT][HD / 64][2]) {
    const int rows = min(ROWS, cu.w.n * a.group - cu.tile * ROWS);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = cu.tile * ROWS + nt * 8 + g, i = r / a.group;
      const uint16_t* src = a.q + (cu.w.row0 + static_cast<int64_t>(i)) * a.ld_q + (cu.kvh * a.group + r - i * a.group) * HD;
#pragma unroll
      for (int h = 0; h < HD / 64; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          v[nt][h][j] = nt * 8 + g < rows ? *reinterpret_cast<const uint4*>(src + (HD == 128 ? 2 * c + h : c) * 16 + j * 8)
                                          : make_uint4(0, 0, 0, 0);
    }
  };
  auto power = [](int e) { return __int_as_float((e + 127) << 23); };   // 2^e, |e| < 127
  auto skip = [&]() {   // to the next unit with steps here
    while (cu.left > 0 && cu.s1 <= cu.s0) {
      base += cu.w.steps + kUnitCost;
      cu.next(a);
    }
  };
  skip();
  uint4 queries[NT][HD / 64][2];
  if (cu.left > 0) load_queries(queries);
  while (cu.left > 0) {
    const int kvh = cu.kvh, tile = cu.tile;
    const int rows = min(ROWS, cu.w.n * a.group - tile * ROWS);
    // ---- queries: operand B, and the factor that takes S to log2 units
    uint32_t qb[NT][HD / 16][2];
    float qs[NT][2];
    int pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float peak = 0.f;
#pragma unroll
      for (int h = 0; h < HD / 64; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float f[8];
          unpack8(queries[nt][h][j], f);
#pragma unroll
          for (int k = 0; k < 8; ++k) peak = fmaxf(peak, fabsf(f[k]));
        }
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
      // 2^e takes the largest magnitude to [2^13, 2^14) (below it for subnormals): bf16's 8 bits
      // stay exact in f16 down to 2^-27 of it, and smaller ones keep an absolute 2^-38 of it
      int e = 0;
      if (peak > 0.f && peak <= FLT_MAX) e = 13 - (static_cast<int>(__float_as_uint(peak) >> 23) - 127);
      const float f1 = power(e >> 1), f2 = power(e - (e >> 1));   // 2^e may be out of range
#pragma unroll
      for (int h = 0; h < HD / 64; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float f[8];
          unpack8(queries[nt][h][j], f);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = f[k] * f1 * f2;
          const int s = h * 4 + j * 2;
          qb[nt][s][0] = pack_f16x2(f[0], f[1]);
          qb[nt][s][1] = pack_f16x2(f[2], f[3]);
          qb[nt][s + 1][0] = pack_f16x2(f[4], f[5]);
          qb[nt][s + 1][1] = pack_f16x2(f[6], f[7]);
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // columns 2c, 2c + 1 of S^T: the rows that lanes 8c and 8c + 4 loaded
        const int ec = __shfl_sync(0xffffffffu, e, 8 * c + 4 * j);
        qs[nt][j] = a.scale * 1.4426950408889634f * power(-(ec >> 1)) * power(-(ec - (ec >> 1)));
        pos[nt][j] = cu.w.past + (tile * ROWS + nt * 8 + 2 * c + j) / a.group;
      }
    }
    const int pos_lo = cu.w.past + tile * ROWS / a.group;
    const int pos_hi = cu.w.past + (tile * ROWS + rows - 1) / a.group;
    const int before = a.window > 0 ? pos_lo - a.window : -1;   // the last token before every query's window
    float acc[HD / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < HD / 16; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[j][nt][k] = 0.f;
    }
    const uint8_t* mrow = a.mask ? a.mask + cu.seq * a.ld_mask : nullptr;
    // A lane's token of a step, read a step early and looked at only then.
    auto mask_byte = [&](int step) {
      const int t = cu.w.template token<M>(a, step) + lane;
      return step < cu.s1 && t <= pos_hi ? mrow[t] : static_cast<uint8_t>(0);
    };
    uint8_t ahead = mrow ? mask_byte(cu.s0 + warp) : 0;

    for (int step = cu.s0 + warp; step < cu.s1; step += kWarps) {
      if (lost) continue;
      uint32_t seen = 0xFFFFFFFFu;   // bit: a token of the step
      if (mrow) {
        seen = __ballot_sync(0xffffffffu, ahead != 0);
        ahead = mask_byte(step + kWarps);
      }
      wait_groups<R::kStages - 1>();
      __syncwarp();   // the note comes from other lanes
      if (!__all_sync(0xffffffffu, tc::mbar_wait(bars + stage, phase, a.err))) {
        lost = true;
        continue;
      }
      ++taken;
      uint8_t* sg = ring + stage * R::kStage;
      const float4 sc = *reinterpret_cast<const float4*>(notes[stage].scale);
      const int valid = notes[stage].valid;
      const int t0 = cu.w.template token<M>(a, step);
      // ---- S^T
      float s[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) {
          const uint4 r0 = *reinterpret_cast<const uint4*>(sg + off_k[h] + 16 * u * HD);
          const uint4 r1 = *reinterpret_cast<const uint4*>(sg + off_k[h] + (16 * u + 8) * HD);
          const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t fa[4] = {two_codes<FMT, 0>(w0[k]), two_codes<FMT, 0>(w1[k]), two_codes<FMT, 1>(w0[k]),
                                    two_codes<FMT, 1>(w1[k])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (h == 0 && k == 0)
                mma_f16_zero(s[u][nt], fa, qb[nt][0][0], qb[nt][0][1]);
              else
                mma_f16(s[u][nt], fa, qb[nt][h * 4 + k][0], qb[nt][h * 4 + k][1]);
            }
          }
        }
      }
      // ---- masks.  z = s * unit is the score in log2 units; the units are kept above 0 so that
      // a masked -inf stays one
      const bool edge = valid != 3 || mrow || t0 + kStep - 1 > pos_lo ||
                        (a.window > 0 && t0 <= pos_hi - a.window && !(kSinks && t0 + kStep <= a.sinks));
      uint32_t live[4] = {};
      if (edge) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = t0 + 8 * i + g;
          // a query of the tile sees it
          const bool on = (valid >> (i >> 1) & 1) && (seen >> (8 * i + g) & 1) && t <= pos_hi &&
                          (kSinks ? t > before || t < a.sinks : t > before);
          if (FMT == GLT_KV8_E4M3) live[i] = __ballot_sync(0xffffffffu, on);   // bit 4g: token 8 i + g
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (!(on && t <= pos[nt][j] &&
                    (a.window == 0 || t > pos[nt][j] - a.window || (kSinks && t < a.sinks))))
                s[i >> 1][nt][(i & 1) * 2 + j] = -INFINITY;
        }
      }
      // A fold unit is what shares a scale of V in this step: its halves with blocks of 16
      // tokens, else the whole step.  Its weights are taken from its own maximum `peak`
      // (2^15 at most, in f16's range), and join the running sums by a 32-bit factor.
      bool moved = false;
      float peak[LU][NT][2], unit[LU][NT][2], ref[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = m[nt][j];
#pragma unroll
          for (int f = 0; f < LU; ++f) {
            unit[f][nt][j] = fmaxf((f ? sc.z : sc.x) * qs[nt][j], 1e-37f);
            float x = fmaxf(s[f][nt][j], s[f][nt][2 + j]);
            if (LU == 1) x = fmaxf(x, fmaxf(s[1][nt][j], s[1][nt][2 + j]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            x *= unit[f][nt][j];
            peak[f][nt][j] = x;
            top = fmaxf(top, x);
          }
          moved |= top > m[nt][j];
          ref[nt][j] = top;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float corr = ref[nt][j] == -INFINITY ? 1.f : ex2_approx(m[nt][j] - ref[nt][j]);
            m[nt][j] = ref[nt][j];
            l[nt][j] *= corr;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
              acc[k][nt][j] *= corr;
              acc[k][nt][2 + j] *= corr;
            }
          }
      }
      // ---- P^T as operand B.  Weights below f16's normal range go the 32-bit way below.
      uint32_t pb[2][NT][2];
      float fold[LU][NT][2];   // from a unit's sums to the running ones
      bool small = false;
#pragma unroll
      for (int f = 0; f < LU; ++f)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // (a scale of K that is NaN comes back in here: the units above drop it)
            const float r = peak[f][nt][j] == -INFINITY ? 0.f : fmaf(f ? sc.z : sc.x, 0.f, peak[f][nt][j] - 15.f);
            const float w = peak[f][nt][j] == -INFINITY ? 0.f : ex2_approx(r - m[nt][j]);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (LU == 2 && (i >> 1) != f) continue;
              float& p = s[i >> 1][nt][(i & 1) * 2 + j];
              p = ex2_approx(fmaf(p, unit[f][nt][j], -r));
              sum += p;
              small |= p < kF16Min && p > 0.f;
            }
            l[nt][j] = fmaf(sum, w, l[nt][j]);
            // a unit that the row sees nothing of may have any scale
            fold[f][nt][j] = peak[f][nt][j] == -INFINITY ? 0.f : w * (f ? sc.w : sc.y);
          }
      if (__any_sync(0xffffffffu, small)) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {   // tokens 8 i + g of the step
          float p[NT][2];
          bool mine = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float x = s[0][nt][j];
              if (i == 1) x = s[0][nt][2 + j];
              if (i == 2) x = s[1][nt][j];
              if (i == 3) x = s[1][nt][2 + j];
              if (!(x < kF16Min)) x = 0.f;
              mine |= x > 0.f;
              p[nt][j] = x * fold[LU == 2 ? i >> 1 : 0][nt][j];
            }
          uint32_t lanes = __ballot_sync(0xffffffffu, mine);
          while (lanes) {
            const int tg = (__ffs(lanes) - 1) >> 2;
            lanes &= ~(0xFu << (4 * tg));
            // row 8 i + tg, the g-th eighth of its channels
            const uint8_t* vc = sg + R::kPart + (8 * i + tg) * HD +
                                (HD == 128 ? (g ^ tg) << 4 : (((g >> 1) ^ (tg >> 1)) << 4) + (g & 1) * 8);
            float pt[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) pt[nt][j] = __shfl_sync(0xffffffffu, p[nt][j], tg * 4 + c);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float v = kv8_decode(vc[2 * k + e], FMT);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int j = 0; j < 2; ++j) acc[k][nt][2 * e + j] = fmaf(pt[nt][j], v, acc[k][nt][2 * e + j]);
              }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (s[u][nt][k] < kF16Min) s[u][nt][k] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pb[u][nt][0] = transpose_8x8(pack_f16x2(s[u][nt][0], s[u][nt][1]));
          pb[u][nt][1] = transpose_8x8(pack_f16x2(s[u][nt][2], s[u][nt][3]));
        }
      // ---- O^T
      float part[HD / 16][NT][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t w[4][HD / 32];   // four tokens, four channels a word
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (HD == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(sg + off_v[i & 1] + (16 * u + 8 * (i >> 1)) * HD);
            w[i][0] = x.x, w[i][1] = x.y, w[i][2] = x.z, w[i][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(sg + off_v[i & 1] + (16 * u + 8 * (i >> 1)) * HD);
            w[i][0] = x.x, w[i][1] = x.y;
          }
        }
        if (FMT == GLT_KV8_E4M3 && edge) {
          // bytes of tokens that no row sees may be NaN codes, and 0 times NaN is NaN
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(live[2 * u + (i >> 1)] >> (4 * (2 * c + (i & 1))) & 1))
#pragma unroll
              for (int k = 0; k < HD / 32; ++k) w[i][k] = 0;
        }
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t x = __byte_perm(w[0][k >> 1], w[1][k >> 1], (k & 1) ? 0x7362 : 0x5140);
          const uint32_t y = __byte_perm(w[2][k >> 1], w[3][k >> 1], (k & 1) ? 0x7362 : 0x5140);
          const uint32_t fa[4] = {two_codes<FMT, 0>(x), two_codes<FMT, 1>(x), two_codes<FMT, 0>(y), two_codes<FMT, 1>(y)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (kFoldEach || u == 0)
              mma_f16_zero(part[k][nt], fa, pb[u][nt][0], pb[u][nt][1]);
            else
              mma_f16(part[k][nt], fa, pb[u][nt][0], pb[u][nt][1]);
            if (kFoldEach || u == 1)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[k][nt][e] = fmaf(part[k][nt][e], fold[LU == 2 ? u : 0][nt][e & 1], acc[k][nt][e]);
          }
        }
      }
      __syncwarp();   // all lanes are done with the stage
      if (++stage == R::kStages) {
        stage = 0;
        phase ^= 1;
      }
      issue();
    }

    // ---- on to the next unit, whose queries come while this one is joined
    const bool whole = cu.whole();
    const int row0 = cu.w.row0;
    const int slot_index = blockIdx.x * 2 + (done > 0 ? 1 : 0);   // only the first and last unit can be cut
    if (!whole && cu.s0 == 0) {
      task.parts = shares.owner(base + cu.w.steps + kUnitCost - 1) - blockIdx.x + 1;
      task.first_slot = slot_index;
      task.row0 = row0;
      task.tile = tile;
      task.kvh = kvh;
      task.rows = rows;
    }
    base += cu.w.steps + kUnitCost;
    cu.next(a);
    skip();
    if (cu.left > 0) load_queries(queries);
    // ---- join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = l[nt][j];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        l[nt][j] = x;
        if (g == 0) join_ml[warp * ROWS + nt * 8 + 2 * c + j] = make_float2(m[nt][j], x);
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, join_ml[w * ROWS + nt * 8 + 2 * c + j].x);
        const float f = join_factor(m[nt][j], top);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          acc[k][nt][j] *= f;
          acc[k][nt][2 + j] *= f;
        }
      }
    // O^T tile k, row g (+8) is channel g hd / 8 + 2k (+1); column 2c + j is a query row.  Two channels
    // lie where neither this nor the reading below meets a bank twice: rows are 4 floats longer
    // (eight banks from one c to the next), and tiles 2i and 2i + 1 share 32, turned by 8i.
    auto turned = [](int k, int g) { return (k >> 1) * 32 + (((k & 1) * 16 + 2 * g + 8 * (k >> 1)) & 31); };
    auto place = [&](int k, int nt, int j) { return (nt * 8 + 2 * c + j) * kJoinRow + turned(k, g); };
    if (warp >= 2) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            *reinterpret_cast<float2*>(join_o + (warp - 2) * ROWS * kJoinRow + place(k, nt, j)) =
                make_float2(acc[k][nt][j], acc[k][nt][2 + j]);
    }
    __syncthreads();
    if (warp < 2) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float2* d = reinterpret_cast<float2*>(join_o + warp * ROWS * kJoinRow + place(k, nt, j));
            const float2 x = *d;
            *d = make_float2(x.x + acc[k][nt][j], x.y + acc[k][nt][2 + j]);
          }
    }
    __syncthreads();
    float* slot = ws.slots + static_cast<int64_t>(slot_index) * (ROWS * HD + 2 * ROWS);
    for (int i = threadIdx.x; i < rows * (HD / 4); i += kThreads) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, join_ml[w * ROWS + r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += join_ml[w * ROWS + r].y * join_factor(join_ml[w * ROWS + r].x, top);
      float4 z;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float* from = join_o + r * kJoinRow + turned((d % (HD / 8)) / 2 + h, d / (HD / 8));
        const float2 x = *reinterpret_cast<const float2*>(from), y = *reinterpret_cast<const float2*>(from + ROWS * kJoinRow);
        (h ? z.z : z.x) = x.x + y.x;
        (h ? z.w : z.y) = x.y + y.y;
      }
      if (whole) {
        write_out<M>(a, row0, tile * ROWS + r, kvh, HD, d, z, top, sum);
      } else {
        *reinterpret_cast<float4*>(slot + r * HD + d) = z;
        if (d == 0) {
          slot[ROWS * HD + r] = top;
          slot[ROWS * HD + ROWS + r] = sum;
        }
      }
    }
    __syncthreads();   // the join buffers are free again
    ++done;
  }
  if (M == Mode::kPrefix) asm volatile("griddepcontrol.wait;" ::: "memory");   // who waits for this kernel waits for the prefix's
  if (threadIdx.x == 0) ws.tasks[blockIdx.x] = task;
  wait_groups<0>();
  // after a lost copy: the copies still under way end before the shared memory does
  for (; taken < issued; ++taken) {
    tc::mbar_wait(bars + stage, phase, a.err);
    if (++stage == R::kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
}

// A task to the CTAs of a column of the grid: they join the parts of a unit, four channels of a row a thread
// (with four turns a thread for 16 rows of 128 channels instead, the 12 x 5 draft tokens' join took 4 us longer).
constexpr int kJoinBatch = 8;   // parts whose loads are in flight at once
template <int HD, int NT, Mode M>
__global__ void __launch_bounds__(kThreads) kv8_join_kernel(const __grid_constant__ AttnArgs a, int grid) {
  constexpr int ROWS = 8 * NT, kSlot = ROWS * HD + 2 * ROWS;
  const Workspace ws(a.workspace, grid, ROWS, HD);
  if (M == Mode::kPrefix) asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int ctas = *ws.ctas;
  const JoinTask task = ws.tasks[blockIdx.x];   // read before it is known to be one: within the workspace
  if (static_cast<int>(blockIdx.x) >= ctas || task.parts < 2) return;
  auto slot = [&](int k) {
    return ws.slots + (k == 0 ? static_cast<int64_t>(task.first_slot) : 2 * (static_cast<int64_t>(blockIdx.x) + k)) * kSlot;
  };
  const int e = blockIdx.y * kThreads + threadIdx.x;
  if (e < task.rows * (HD / 4)) {
    const int r = e / (HD / 4), d = e % (HD / 4) * 4;
    float top = -INFINITY, sum = 0.f;
    float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < task.parts; k0 += kJoinBatch) {
      float m[kJoinBatch], l[kJoinBatch];
      float4 x[kJoinBatch];
      float peak = top;
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        const float* p = slot(min(k0 + k, task.parts - 1));
        m[k] = p[ROWS * HD + r];
        l[k] = p[ROWS * HD + ROWS + r];
        x[k] = *reinterpret_cast<const float4*>(p + r * HD + d);
      }
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k)
        if (k0 + k < task.parts) peak = fmaxf(peak, m[k]);
      const float old = join_factor(top, peak);
      sum *= old;
      z = make_float4(z.x * old, z.y * old, z.z * old, z.w * old);
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        if (k0 + k >= task.parts) continue;
        const float f = join_factor(m[k], peak);
        sum = fmaf(l[k], f, sum);
        z.x = fmaf(x[k].x, f, z.x);
        z.y = fmaf(x[k].y, f, z.y);
        z.z = fmaf(x[k].z, f, z.z);
        z.w = fmaf(x[k].w, f, z.w);
      }
      top = peak;
    }
    write_out<M>(a, task.row0, task.tile * ROWS + r, task.kvh, HD, d, z, top, sum);
  }
}

int check_heads(const GltKv8Cache* c, const GltKv8Batch* b, int nh) {
  GLT_TRY(kv8_check(c, b));
  if (nh < 1 || nh % c->num_kv_heads || nh > 65535)
    return fail(GLT_EINVAL, "kv8: num_heads %d must be a multiple of num_kv_heads %d", nh, c->num_kv_heads);
  if (static_cast<int64_t>(kv8_most_new(*c, *b)) * nh > INT_MAX / 2)
    return fail(GLT_EINVAL, "kv8: %d new rows of a sequence with %d heads", kv8_most_new(*c, *b), nh);
  return GLT_OK;
}

// Row tiles of 8 fill the tensor core's N for up to 8 rows a KV head; more rows go 16 at a
// time, which reads and decodes the cache half as often (40 rows, when measured: 44.6 us against 46.1, at the
// price of 16 rows' sums, which leave no registers).
struct Plan {
  int nt, grid;
  int64_t bytes;
};
Plan plan(const GltKv8Cache& c, const GltKv8Batch& b, int nh) {
  Plan p;
  const int64_t rows = static_cast<int64_t>(kv8_most_new(c, b)) * (nh / c.num_kv_heads);
  p.nt = rows <= 8 ? 1 : 2;
  // no more CTAs than the fullest cache could feed
  const int64_t tiles = (rows + 8 * p.nt - 1) / (8 * p.nt);
  const int64_t steps = (static_cast<int64_t>(b.max_blocks) * c.block_tokens + kStep - 1) / kStep;
  const double most = static_cast<double>(tiles) * c.num_kv_heads * b.num_seqs * (steps + kUnitCost) / kWarps + 1;
  p.grid = num_sms() * kCtasPerSm;
  if (most < p.grid) p.grid = static_cast<int>(most);
  p.bytes = Workspace(nullptr, p.grid, 8 * p.nt, c.head_dim).bytes;
  return p;
}

template <int HD, int FMT, int NT, bool BT16, Mode M>
int launch(const AttnArgs& a, int grid, cudaStream_t st) {
  constexpr int bytes = smem_bytes<HD, NT>();
  GLT_TRY(ensure_smem_attr(reinterpret_cast<const void*>(&kv8_attention_kernel<HD, FMT, NT, BT16, M>), bytes));
  // rows of the pools; a copy is a step's rows, or a block's where blocks are shorter
  const uint64_t pool_rows = static_cast<uint64_t>(a.c.num_blocks) * a.c.num_kv_heads * a.c.block_tokens;
  CUtensorMap map_k, map_v;
  GLT_TRY(make_tmap_u8(&map_k, a.c.k, HD, pool_rows, BT16 ? 16 : kStep));
  GLT_TRY(make_tmap_u8(&map_v, a.c.v, HD, pool_rows, BT16 ? 16 : kStep));
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  if (M == Mode::kPrefix) {
    cfg.gridDim = dim3(grid);
    cfg.dynamicSmemBytes = bytes;
    cfg.numAttrs = a.chained ? 1 : 0;   // behind any other kernel, its writes would not be awaited
    GLT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv8_attention_kernel<HD, FMT, NT, BT16, M>, a, map_k, map_v));
  } else {
    kv8_attention_kernel<HD, FMT, NT, BT16, M><<<grid, kThreads, bytes, st>>>(a, map_k, map_v);
  }
  GLT_LAUNCH_CHECK();
  if (grid < 2) return GLT_OK;
  // starts while the first kernel runs and waits for its end
  cfg.gridDim = dim3(grid - 1, 8 * NT * HD / 4 / kThreads);   // the last CTA ends every unit it begins
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  GLT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv8_join_kernel<HD, NT, M>, a, grid));
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

template <int HD, int FMT, Mode M>
int launch_rows(const AttnArgs& a, const Plan& p, cudaStream_t st) {
  if (a.c.block_tokens == 16)
    return p.nt == 1 ? launch<HD, FMT, 1, true, M>(a, p.grid, st) : launch<HD, FMT, 2, true, M>(a, p.grid, st);
  return p.nt == 1 ? launch<HD, FMT, 1, false, M>(a, p.grid, st) : launch<HD, FMT, 2, false, M>(a, p.grid, st);
}
template <Mode M>
int launch_all(const AttnArgs& a, const Plan& p, cudaStream_t st) {
  const bool int8 = a.c.format == GLT_KV8_INT8;
  if (a.c.head_dim == 128)
    return int8 ? launch_rows<128, GLT_KV8_INT8, M>(a, p, st) : launch_rows<128, GLT_KV8_E4M3, M>(a, p, st);
  return int8 ? launch_rows<64, GLT_KV8_INT8, M>(a, p, st) : launch_rows<64, GLT_KV8_E4M3, M>(a, p, st);
}

// The checks and arguments that every form of the call shares; p is its plan.
int prepare(const GltKv8Cache* cache, const GltKv8Batch* batch, const uint16_t* q, int64_t ld_q, uint16_t* o, int64_t ld_o,
            float* lse, int num_heads, float scale, int window, const uint8_t* token_mask, int64_t ld_mask,
            void* workspace, int64_t workspace_bytes, AttnArgs* a, Plan* p) {
  if (!q || !o) return fail(GLT_EINVAL, "null argument");
  const int64_t width = static_cast<int64_t>(num_heads) * cache->head_dim;
  if (ld_q < width || ld_o < width || ld_q % 8 || ld_o % 8 || !aligned16(q) || !aligned16(o))
    return fail(GLT_EINVAL, "kv8: q and o rows must be 16-byte aligned (strides multiples of 8, at least %lld)", (long long)width);
  if (!(scale >= 0.f) || scale > FLT_MAX) return fail(GLT_EINVAL, "kv8: scale must be finite and not negative");
  if (window < 0) return fail(GLT_EINVAL, "kv8: negative window");
  if (token_mask && ld_mask < static_cast<int64_t>(batch->max_blocks) * cache->block_tokens)
    return fail(GLT_EINVAL, "kv8: mask row stride below max_blocks * block_tokens");
  *p = plan(*cache, *batch, num_heads);
  if (workspace_bytes < p->bytes || !workspace || !aligned16(workspace))
    return fail(GLT_EINVAL, "kv8: workspace must be 16-byte aligned and hold %lld bytes", (long long)p->bytes);
  *a = {};
  a->c = *cache;
  a->b = *batch;
  a->q = q;
  a->ld_q = ld_q;
  a->o = o;
  a->ld_o = ld_o;
  a->lse = lse;
  a->nh = num_heads;
  a->group = num_heads / cache->num_kv_heads;
  a->scale = scale > 0.f ? scale : 1.f / sqrtf(static_cast<float>(cache->head_dim));
  a->window = window;
  a->mask = token_mask;
  a->ld_mask = ld_mask;
  a->workspace = workspace;
  a->err = device_error_word();
  return GLT_OK;
}

}  // namespace
}  // namespace glt
