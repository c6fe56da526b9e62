// Attention of a batch of sequences that share a long prefix (glt_kv8_prefix_attention).
//
//   o = (sum over the prefix + sum over own tokens of p v) / (the same of p)
//
// Every query of the batch sees the whole prefix, so its cache is read once for all of them: the queries
// that share a KV head are the rows of tcgen05 products with it.
//
// A CTA (see kv8_prefix.cuh for its share of the work) goes through steps of 64 tokens:
//   warp 14     looks up the blocks, copies their codes in bulk into a ring of K or V of a step each, and notes the scales.
//   warps 8-11  turn codes into f16, which holds them exactly, and lay K and V out as the products read them.
//   warps 12-13 issue the products of a lane each: S = Q K^T, and O += P V with P in TMEM, as P was written over S.  (From one
//               warp, the tensor cores ran dry whenever it went from one barrier to the next.)
//   warps 0-7   softmax, a thread a query row, in two lanes of 128 rows with an S and an O each: the tensor core works
//               for one lane while the other's softmax runs.  With more than 128 rows a KV head the lanes are two
//               tiles of rows at the same tokens; else every second step of the same rows.
// A query row is brought to f16 by a power of two, as in kv8_attention.cuh.  The scale of K multiplies S in 32 bits.  The
// scale of V joins the exponent: a token counts 2^(s + log2 scale - ref) in the sum of values, ref a running
// reference near the maximum of that exponent, so that f16 has what one token can add at most near its top whatever the
// scales of the blocks are: 11 bits down to 2^-24 of the reference, and below that within 2^-35 of it.  Over 1 / scale,
// in 32 bits, the same numbers make the sum of weights; where scales lie so far apart that they would leave 32 bits, larger
// ones do (ScaleWindow).  (P as the sum of two bf16 numbers needs no such
// reference, but half as many products and instructions again: 306 us where f16 took 258, other things equal.)
// The reference moves only when the weights come near f16's top.
//
// What bounds it: 4 rows hd operations a token are 83 us at the measured bf16 rate for 4096 rows (128 sequences, 32 heads over 8,
// head_dim 128) behind 65537 tokens, of 193 us the call takes.  A step of 64 tokens and 256 rows takes a CTA 2400 cycles
// where its products need 1300 of the tensor cores and its exponentials 1000 of their units: each of the
// softmax's two warps a scheduler waits 700 of them for what it has just read or issued, at 0.4 instructions a cycle.  Sixteen
// softmax warps of half a row each (72 registers) were slower, 234 us.  One result after the other: loops as short as here instead of
// unrolled code 306 us for 423; scores ahead of the softmax, sums instead of maxima 204 for 258.
// Few sequences are bound by beginnings and ends: 64 sequences behind 8193 tokens 55 us, of which the units' first loads, the
// parts' way through memory (19 MB) and the own tokens' kernel are three quarters.
#include <float.h>

#include <algorithm>

#include "kv8_attention.cuh"
#include "kv8_own.cuh"
#include "kv8_prefix.cuh"

namespace glt {
namespace {

constexpr int kSoftmaxWarps = 8, kDecodeWarps = 4, kIssueWarp = kSoftmaxWarps + kDecodeWarps;
constexpr int kCopyWarp = kIssueWarp + 2;   // an issuing warp for each lane
constexpr int kPrefixThreads = 32 * (kCopyWarp + 1);
constexpr int kAhead = 2;   // steps that K is laid out ahead of V
constexpr int kDecodeThreads = 32 * kDecodeWarps;
constexpr float kLift = 10.f;         // base 2: what the reference counts in f16, whose top is 2^16 and last normal 2^-14
constexpr float kMostSum = 0x1p15f;   // of 16 tokens, before the reference moves: over the least scale, 2^26 of them stay within 32 bits

struct PrefixArgs {
  GltKv8Cache c;
  const int32_t* block_ids;
  const uint16_t* q;
  int64_t ld_q;
  int rows, group;   // query rows a KV head: rows = tokens * group
  float scale;
  PrefixParts parts;
  unsigned int* err;
};

// Scales of a step's groups of 16 tokens, and flags of each: kLost, its block is not in the pool; kNone, its values are 0; kWide, a scale
// of V so far was outside the run's ScaleWindow.
constexpr int kLost = 1, kNone = 2, kWide = 4, kEach = 0x01010101;
struct alignas(16) PrefixNote {
  float k[4], log_v[4], inv_v[4];
  uint8_t flags[4];
  int pad[3];
  __device__ __forceinline__ int all_flags() const { return *reinterpret_cast<const int*>(flags); }
};
constexpr int kNotes = 16;   // steps whose scales are held: more than can be under way
constexpr int kSlots = 3;    // steps of K, and of V, that are laid out

template <int HD, int LANES>
struct PrefixSmem {
  static constexpr int kQ = kPrefixRows * HD * 2;
  static constexpr int kPart = kPrefixStep * HD * 2;   // K (or V) of a step
  static constexpr int kRaw = kPrefixStep * HD;        // its codes
  static constexpr int kRaws = LANES == 2 ? 8 : 12;
  static constexpr int kOffK = LANES * kQ;
  static constexpr int kOffV = kOffK + kSlots * kPart;
  static constexpr int kOffRaw = kOffV + kSlots * kPart;
  static constexpr int kOffNotes = kOffRaw + kRaws * kRaw;
  static constexpr int kOffBars = kOffNotes + kNotes * static_cast<int>(sizeof(PrefixNote));
  static constexpr int kBars = 2 * kRaws + 4 * kSlots + 8 + 2 + 3;
  static constexpr int kOffUnits = kOffBars + (kBars + 2) * 8;
  static constexpr int kTotal = 1024 + kOffUnits + (LANES == 1 ? kPrefixRows * 4 : 0);
};
static_assert(PrefixSmem<128, 1>::kTotal <= 232448 && PrefixSmem<128, 2>::kTotal <= 232448, "shared memory");

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 64 columns of the thread's lane.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  uint32_t r[64];
#pragma unroll
  for (int h = 0; h < 64; h += 32)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[h + 0]), "=r"(r[h + 1]), "=r"(r[h + 2]), "=r"(r[h + 3]), "=r"(r[h + 4]), "=r"(r[h + 5]), "=r"(r[h + 6]),
          "=r"(r[h + 7]), "=r"(r[h + 8]), "=r"(r[h + 9]), "=r"(r[h + 10]), "=r"(r[h + 11]), "=r"(r[h + 12]),
          "=r"(r[h + 13]), "=r"(r[h + 14]), "=r"(r[h + 15]), "=r"(r[h + 16]), "=r"(r[h + 17]), "=r"(r[h + 18]),
          "=r"(r[h + 19]), "=r"(r[h + 20]), "=r"(r[h + 21]), "=r"(r[h + 22]), "=r"(r[h + 23]), "=r"(r[h + 24]),
          "=r"(r[h + 25]), "=r"(r[h + 26]), "=r"(r[h + 27]), "=r"(r[h + 28]), "=r"(r[h + 29]), "=r"(r[h + 30]),
          "=r"(r[h + 31])
        : "r"(taddr + h));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
// Two floats in one instruction.
__device__ __forceinline__ uint64_t two_floats(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float low(uint64_t x) { return __uint_as_float(static_cast<uint32_t>(x)); }
__device__ __forceinline__ float high(uint64_t x) { return __uint_as_float(static_cast<uint32_t>(x >> 32)); }
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
__device__ __forceinline__ void four(const float* p, float (&f)[4]) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&v)[16]) {
  uint32_t u[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(v[i]);
  tmem_st16(taddr, u);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Copies 16 bytes (zero where !on: the source is not read then).
__device__ __forceinline__ void copy_async16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}
// O (+)= P . V with P in TMEM.
__device__ __forceinline__ void umma_p(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc));
}

// Sixteen codes as f16 numbers, in two vectors.
template <int FMT>
__device__ __forceinline__ void sixteen_f16(const uint4& x, uint4& a, uint4& b) {
  a = make_uint4(two_codes<FMT, 0>(x.x), two_codes<FMT, 1>(x.x), two_codes<FMT, 0>(x.y), two_codes<FMT, 1>(x.y));
  b = make_uint4(two_codes<FMT, 0>(x.z), two_codes<FMT, 1>(x.z), two_codes<FMT, 0>(x.w), two_codes<FMT, 1>(x.w));
}

// Walks a CTA's run: steps [s0, s1) of unit `unit`.
struct PrefixRun {
  int64_t left;   // of the run, from the unit's first place here on
  int steps, place, unit, s0, s1;
  __device__ __forceinline__ PrefixRun(const PrefixShares& sh, int cta) : left(0), steps(sh.steps) {
    if (cta >= sh.ctas) return;
    const int64_t begin = sh.begin(cta);
    left = sh.begin(cta + 1) - begin;
    unit = static_cast<int>(PrefixShares::quotient(begin, steps + kPrefixUnitCost));
    place = static_cast<int>(begin - static_cast<int64_t>(unit) * (steps + kPrefixUnitCost));
    bounds();
  }
  __device__ __forceinline__ void bounds() {
    s0 = max(0, place - kPrefixUnitCost);
    s1 = static_cast<int>(min(static_cast<int64_t>(steps), place + left - kPrefixUnitCost));
    if (left > 0 && s1 <= s0) next();   // only a part of the unit's cost
  }
  __device__ __forceinline__ bool on() const { return left > 0; }
  // On to the next step.
  __device__ __forceinline__ void step(int& s) {
    if (++s < s1) return;
    next();
    s = on() ? s0 : 0;
  }
  __device__ __forceinline__ void next() {
    left -= steps + kPrefixUnitCost - place;
    ++unit;
    place = 0;
    if (left > 0) bounds();
  }
};

// A step where scales of V lie far apart (kWide): 16 tokens at a time, by their maximum, P over what is read of S.  done: the barrier of
// the lane's last product with V, if there was one.  (Not inline: with its code in the loop
// of ordinary steps 64 sequences behind 8193 tokens took 55.8 us for 54.8, and 128 behind 65537 191.8 for 192.7.)
struct RowSums {
  float m, l;   // the reference, the sum of weights
  bool ok;
};
template <int HD>
__device__ __noinline__ RowSums wide_step(const PrefixNote& note, int left, float unit_q, float m, float l, uint32_t s_buf, uint32_t o_at,
                                          uint64_t* done, uint32_t parity, unsigned int* err, volatile int* abort) {
  const int flags = note.all_flags();
  auto group = [&](int g, float (&v)[16]) {
    tmem_ld16(s_buf + 16 * g, v);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (16 * g + j >= left || (flags >> (8 * g) & kLost)) v[j] = -INFINITY;
    return fmaxf(note.k[g] * unit_q, 1e-37f);
  };
  float peak = m;
#pragma unroll 1
  for (int g = 0; g < 4; ++g) {
    float v[16], top = -INFINITY;
    const float u = group(g, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) top = fmaxf(top, v[j]);
    peak = fmaxf(peak, fmaf(top, u, note.log_v[g]));
  }
  if (__any_sync(0xffffffffu, peak > m)) {
    const TwoFactors f(peak > m ? m - peak : 0.f);
    if (done) {
      if (!__all_sync(0xffffffffu, tc::mbar_wait(done, parity, err, abort))) return {m, l, false};
      tc::tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        float o[16];
        tmem_ld16(o_at + c, o);
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = o[j] * f.a * f.b;
        tmem_st16(o_at + c, o);
      }
    }
    l = l * f.a * f.b;
    m = peak;
  }
  const float ref = kLift - (m == -INFINITY ? 0.f : m);
#pragma unroll 1
  for (int g = 0; g < 4; ++g) {
    float v[16], lifted = 0.f;
    uint32_t p[8];
    const float u = group(g, v), log_v = note.log_v[g], r = ref + log_v;
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float e0 = fmaf(v[j], u, r), e1 = fmaf(v[j + 1], u, r);
      p[j / 2] = pack_f16x2(ex2_approx(e0), ex2_approx(e1));
      lifted += ex2_approx(e0 + kWideLift) + ex2_approx(e1 + kWideLift);
    }
    tmem_st8(s_buf + 8 * g, p);
    l += wide_weights(lifted, log_v, note.inv_v[g]);
  }
  return {m, l, true};
}

template <int HD, int FMT, int LANES>
__global__ void __launch_bounds__(kPrefixThreads, 1) kv8_prefix_kernel(const __grid_constant__ PrefixArgs a) {
  using L = PrefixSmem<HD, LANES>;
  constexpr uint32_t kBf16 = (1u << 7) | (1u << 10);   // operand types of a descriptor: f16 is 0
  constexpr uint32_t kIdescS = tc::make_idesc(kPrefixStep, false, false) & ~kBf16, kIdescO = tc::make_idesc(HD, false, true) & ~kBf16;
  constexpr uint32_t kColO = 256;   // TMEM: two S of lane 0, of lane 1 (64 columns each), O of lane 0, of lane 1 (128 each)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-tc::smem_u32(smem_raw) & 1023u);   // the swizzle goes by address
  PrefixNote* notes = reinterpret_cast<PrefixNote*>(smem + L::kOffNotes);
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
  uint64_t* raw_empty = raw_full + L::kRaws;
  uint64_t* k_full = raw_empty + L::kRaws;   // K of a step is laid out, is read (and so on for V)
  uint64_t* k_empty = k_full + kSlots;
  uint64_t* v_full = k_empty + kSlots;
  uint64_t* v_empty = v_full + kSlots;
  uint64_t* s_full = v_empty + kSlots;       // [lane][2] S is there
  uint64_t* p_full = s_full + 4;             // [lane][2] P is there
  uint64_t* o_full = p_full + 4;             // [lane] O has a P more
  uint64_t* q_full = o_full + 2;             // the unit's queries are laid out
  uint64_t* unit_done = q_full + 1;          // all products of the unit are done
  uint64_t* drain = unit_done + 1;
  uint32_t* slot = reinterpret_cast<uint32_t*>(drain + 1);
  float* unit_rows = reinterpret_cast<float*>(smem + L::kOffUnits);   // LANES = 1: what lane 0 found for each row
  __shared__ int abort_storage;
  volatile int& abort = abort_storage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;");
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kRaws; ++i) {
      tc::mbar_init(raw_full + i, 1);
      tc::mbar_init(raw_empty + i, kDecodeWarps);
    }
    for (int i = 0; i < kSlots; ++i) {
      tc::mbar_init(k_full + i, kDecodeWarps);
      tc::mbar_init(k_empty + i, LANES);
      tc::mbar_init(v_full + i, kDecodeWarps);
      tc::mbar_init(v_empty + i, LANES);
    }
    for (int i = 0; i < 2; ++i) tc::mbar_init(o_full + i, 1);
    for (int i = 0; i < 4; ++i) {
      tc::mbar_init(s_full + i, 2);   // the products, and their issuer, who has seen the step's note
      tc::mbar_init(p_full + i, 4);
    }
    tc::mbar_init(q_full, kSoftmaxWarps);   // both lanes', so that neither falls a unit behind
    tc::mbar_init(unit_done, 2);
    tc::mbar_init(drain, 2);
    abort = 0;
    tc::fence_mbar_init();
  }
  if (warp == kIssueWarp) {
    tc::tmem_alloc(slot, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot;
  const int tokens = a.parts.tokens(blockIdx.x == 0 && threadIdx.x == 0 ? a.err : nullptr);
  const PrefixShares shares(a.parts, tokens);
  PrefixRun run(shares, blockIdx.x);
  int copied = 0;   // elements of the ring that this thread has armed

  if (warp < kSoftmaxWarps) {
    // ------------------------------- softmax -------------------------------
    const int mine = warp >> 2;                            // lane of the pipeline
    const int r = (warp & 3) * 32 + lane;                  // query row in the tile
    const uint32_t at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_at = at + mine * 128, o_at = at + kColO + mine * 128;
    // x / group for x < group + 4: the quotient is at most 4, and no multiple lies as near as 2^-32 of it
    const uint32_t group_inverse = a.group > 1 ? 0xFFFFFFFFu / static_cast<uint32_t>(a.group) + 1 : 0;
    int seg = 0, base = 0, products = 0;   // steps before the unit's, the lane's steps so far
    for (; run.on() && !abort; run.next(), ++seg) {
      const int kvh = run.unit % a.parts.kv_heads, pair = run.unit / a.parts.kv_heads;
      // ---- queries: a warp its threads' rows, kPer lanes to a row
      // (one lane for both where they are the same)
      const int n = run.s1 - run.s0;
      float unit_q = 0.f;   // takes S to log2 units
      if (LANES == 2 || mine == 0) {
        // into their places as they are, a warp its threads' rows, kPer lanes to a row, all at once (the loads' latency is the
        // unit's); then a thread takes its row to f16
        constexpr int kPer = HD / 8, kRows = 32 / kPer, kTurns = 32 / kRows;
        const int tile_row = (LANES == 2 ? pair * 2 + mine : pair) * kPrefixRows;
        uint8_t* q_smem = smem + (LANES == 2 ? mine * L::kQ : 0);
        auto place = [&](int row, int c) { return q_smem + (c >> 3) * (kPrefixRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4); };
        int row = (warp & 3) * 32 + lane / kPer;
        int tok = (tile_row + row) / a.group, head = tile_row + row - tok * a.group;   // head of the group
#pragma unroll 4
        for (int i = 0; i < kTurns; ++i) {
          copy_async16(place(row, lane % kPer), a.q + static_cast<int64_t>(tok) * a.ld_q + (kvh * a.group + head) * HD + lane % kPer * 8,
                       tile_row + row < a.rows);
          row += kRows;
          head += kRows;
          const int more = a.group > 1 ? static_cast<int>(__umulhi(static_cast<uint32_t>(head), group_inverse)) : head;   // head / group
          tok += more;
          head -= more * a.group;
        }
        commit();
        wait_groups<0>();
        __syncwarp();
        uint32_t tops = 0;   // of bf16 numbers without their signs, the larger is the larger integer
#pragma unroll 4
        for (int c = 0; c < HD / 8; ++c) {
          const uint4 x = *reinterpret_cast<const uint4*>(place(r, c));
          tops = __vmaxu2(tops, __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu), __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu)));
        }
        const float peak = fmaxf(bf16_lo(tops), bf16_hi(tops));
        // 2^e takes the largest magnitude to [2^13, 2^14)
        auto power = [](int e) { return __int_as_float((e + 127) << 23); };   // 2^e, |e| < 127
        int e = 0;
        if (peak > 0.f && peak <= FLT_MAX) e = 13 - (static_cast<int>(__float_as_uint(peak) >> 23) - 127);
        const float f1 = power(e >> 1), f2 = power(e - (e >> 1));   // 2^e may be out of range
        unit_q = a.scale * 1.4426950408889634f * power(-(e >> 1)) * power(-(e - (e >> 1)));
#pragma unroll 2
        for (int c = 0; c < HD / 8; ++c) {
          float f[8];
          unpack8(*reinterpret_cast<const uint4*>(place(r, c)), f);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = f[j] * f1 * f2;
          *reinterpret_cast<uint4*>(place(r, c)) =
              make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7]));
        }
        if (LANES == 1) unit_rows[r] = unit_q;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(q_full);
      } else {
        if (lane == 0) tc::mbar_arrive(q_full);
        if (!__all_sync(0xffffffffu, tc::mbar_wait(q_full, seg & 1, a.err, &abort))) {
          abort = 1;
          break;
        }
        unit_q = unit_rows[r];
      }
      float m = -INFINITY, l = 0.f;
      bool any = false;
      for (int i = LANES == 2 ? 0 : mine; i < n && !abort; i += LANES == 2 ? 1 : 2) {
        const int it = base + i, buf = products & 1;
        const PrefixNote& note = notes[it % kNotes];
        if (!__all_sync(0xffffffffu, tc::mbar_wait(s_full + 2 * mine + buf, products >> 1 & 1, a.err, &abort))) {
          abort = 1;
          break;
        }
        tc::tc_fence_after();
        float u[4], w[4];   // of the groups of 16 tokens
        four(note.k, u);
        four(note.log_v, w);
        const int flags = note.all_flags(), left = tokens - (run.s0 + i) * kPrefixStep;   // tokens of the step
        const uint32_t s_buf = s_at + buf * kPrefixStep;
        float v[kPrefixStep];
        tmem_ld64(s_buf, v);
#pragma unroll
        for (int g = 0; g < 4; ++g) u[g] = fmaxf(u[g] * unit_q, 1e-37f);   // above 0, so that a masked -inf stays one
        if (left < kPrefixStep || (flags & (kLost | kWide) * kEach)) {
          if (flags & kWide * kEach) {
            const RowSums x = wide_step<HD>(note, left, unit_q, m, l, s_buf, o_at, any ? o_full + mine : nullptr, (products - 1) & 1,
                                            a.err, &abort);
            if (!x.ok) {
              abort = 1;
              break;
            }
            m = x.m;
            l = x.l;
            any = true;
            ++products;
            tmem_wait_st();
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(p_full + 2 * mine + buf);
            continue;
          }
#pragma unroll
          for (int j = 0; j < kPrefixStep; ++j)
            if (j >= left || (flags >> (j / 16 * 8) & kLost)) v[j] = -INFINITY;
        }
        // P by the reference as it stands.  A unit's first S moves it, and one whose weights would come near f16's
        // top, which the sums show: the maximum is taken then, and only then.
        float sums[4];
        bool moved = false;
#pragma unroll 1
        while (true) {
          const float ref = kLift - (m == -INFINITY ? 0.f : m);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t p[8];
            const float r = ref + w[g];
            const uint64_t u2 = two_floats(u[g], u[g]), r2 = two_floats(r, r);
            uint64_t sum = 0;
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const uint64_t e = fma2(two_floats(v[16 * g + j], v[16 * g + j + 1]), u2, r2);
              const float p0 = ex2_approx(low(e)), p1 = ex2_approx(high(e));
              sum = add2(sum, two_floats(p0, p1));
              p[j / 2] = pack_f16x2(p0, p1);
            }
            sums[g] = low(sum) + high(sum);
            tmem_st8(s_buf + 8 * g, p);   // over S, which is read
          }
          const bool high = fmaxf(fmaxf(sums[0], sums[1]), fmaxf(sums[2], sums[3])) > kMostSum;
          if (moved || !__any_sync(0xffffffffu, high || m == -INFINITY)) break;
          moved = true;
          float peak = -INFINITY;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float x[4] = {v[16 * g], v[16 * g + 1], v[16 * g + 2], v[16 * g + 3]};
#pragma unroll
            for (int j = 4; j < 16; ++j) x[j & 3] = fmaxf(x[j & 3], v[16 * g + j]);
            peak = fmaxf(peak, fmaf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), u[g], w[g]));
          }
          const bool grow = peak > m;   // rows of the warp that need not move do no harm
          const float f = grow ? (m == -INFINITY ? 0.f : ex2_approx(m - peak)) : 1.f;
          if (any) {
            // the lane's last product with V is done, and the next one waits for this P
            if (!__all_sync(0xffffffffu, tc::mbar_wait(o_full + mine, (products - 1) & 1, a.err, &abort))) {
              abort = 1;
              break;
            }
            tc::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              float o[16];
              tmem_ld16(o_at + c, o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] *= f;
              tmem_st16(o_at + c, o);
            }
          }
          if (grow) {
            l *= f;
            m = peak;
          }
        }
        if (abort) break;
        any = true;
        ++products;
        four(note.inv_v, u);
#pragma unroll
        for (int g = 0; g < 4; ++g) l = fmaf(sums[g], u[g], l);
        tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full + 2 * mine + buf);
      }
      // ---- the unit's result
      if (abort || !__all_sync(0xffffffffu, tc::mbar_wait(unit_done, seg & 1, a.err, &abort))) {
        abort = 1;
        break;
      }
      tc::tc_fence_after();
      float* out = a.parts.slots + (static_cast<int64_t>(run.unit) + blockIdx.x) * PrefixParts::slot_floats(HD);
      const int row = mine * kPrefixRows + r;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float o[32];
        if (any) {
          tc::tmem_ld32(o_at + c, o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + row * HD + c + j), "f"(o[j]),
                       "f"(o[j + 1]), "f"(o[j + 2]), "f"(o[j + 3]), "f"(o[j + 4]), "f"(o[j + 5]), "f"(o[j + 6]), "f"(o[j + 7])
                       : "memory");
      }
      out[2 * kPrefixRows * HD + row] = m - kLift;
      out[2 * kPrefixRows * (HD + 1) + row] = l;
      tc::tc_fence_before();   // the next unit's products write O once P of its first step has come
      base += n;
    }
  } else if (warp < kIssueWarp) {
    // ------------------------------- codes ---------------------------------
    constexpr int kChunks = HD / 16;                                    // 16 channels of a token
    constexpr int kMine = kPrefixStep * kChunks / kDecodeThreads;       // of a thread, of an element of the ring
    const int tid = threadIdx.x - 32 * kSoftmaxWarps;
    const int chunk = tid % kChunks, tok0 = tid / kChunks;
    int raw = 0;
    uint32_t raw_phase = 0;
    static_assert(kDecodeThreads / kChunks % 8 == 0, "a thread's tokens are swizzled alike");
    const int c = 2 * (chunk & 3), turn = tok0 & 7;
    const int off_lo = (chunk >> 2) * (kPrefixStep * 128) + tok0 * 128 + ((c ^ turn) << 4), off_hi = off_lo ^ 16;
    // The next element of the ring, once it is there.
    auto take = [&](uint4 (&x)[kMine], int& from) {
      if (!__all_sync(0xffffffffu, tc::mbar_wait(raw_full + raw, raw_phase, a.err, &abort))) return false;
      const uint8_t* src = smem + L::kOffRaw + raw * L::kRaw + tid * 16;
#pragma unroll
      for (int i = 0; i < kMine; ++i) x[i] = *reinterpret_cast<const uint4*>(src + i * (kDecodeThreads * 16));
      from = raw;
      if (++raw == L::kRaws) {
        raw = 0;
        raw_phase ^= 1;
      }
      return true;
    };
    // Tokens that are not there become 0 (P is 0 there, and 0 times a NaN would not be).
    auto lay = [&](const uint4 (&x)[kMine], uint8_t* dst, int left, int flags) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int tok = tok0 + i * (kDecodeThreads / kChunks);
        uint4 lo, hi;
        sixteen_f16<FMT>(x[i], lo, hi);
        if (tok >= left || (flags >> ((tok >> 4) * 8) & 1)) lo = hi = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + off_lo + i * (kDecodeThreads / kChunks * 128)) = lo;
        *reinterpret_cast<uint4*>(dst + off_hi + i * (kDecodeThreads / kChunks * 128)) = hi;
      }
    };
    int step = run.on() ? run.s0 : 0, left[kAhead + 1] = {};
    // K of a step goes with V of the step kAhead before: one turn's latencies for both
    for (int it = 0, end = INT_MAX - kAhead; !abort && it < end + kAhead; ++it) {
#pragma unroll
      for (int i = kAhead; i > 0; --i) left[i] = left[i - 1];
      if (it < end && !run.on()) end = it;
      const bool with_k = it < end, with_v = it >= kAhead && it < end + kAhead;
      if (with_k) {
        left[0] = tokens - step * kPrefixStep;
        run.step(step);
      }
      const int v = it - kAhead, slot_k = it % kSlots, slot_v = v % kSlots;
      uint4 xk[kMine], xv[kMine];
      int from_k = 0, from_v = 0;
      bool ok = true;
      if (with_k)
        ok = __all_sync(0xffffffffu, tc::mbar_wait(k_empty + slot_k, (it / kSlots & 1) ^ 1, a.err, &abort)) && take(xk, from_k);
      if (ok && with_v)
        ok = __all_sync(0xffffffffu, tc::mbar_wait(v_empty + slot_v, (v / kSlots & 1) ^ 1, a.err, &abort)) && take(xv, from_v);
      if (!ok) {
        abort = 1;
        break;
      }
      if (with_k) lay(xk, smem + L::kOffK + slot_k * L::kPart, left[0], notes[it % kNotes].all_flags());
      if (with_v) {
        const int flags = notes[v % kNotes].all_flags();
        lay(xv, smem + L::kOffV + slot_v * L::kPart, left[kAhead], flags | flags >> 1);   // kLost or kNone
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (with_k) {
          tc::mbar_arrive(k_full + slot_k);
          tc::mbar_arrive(raw_empty + from_k);
        }
        if (with_v) {
          tc::mbar_arrive(v_full + slot_v);
          tc::mbar_arrive(raw_empty + from_v);
        }
      }
    }
  } else if (warp == kCopyWarp) {
    // ------------------------------- copies --------------------------------
    const int bt = a.c.block_tokens, bt_log = 31 - __clz(bt);
    const int piece = min(bt, kPrefixStep);   // tokens of a copy
    int raw = 0;
    uint32_t raw_phase = 1;
    // Lane g < 4 has tokens 16 g .. of a step.  Its block's id is read two steps ahead, its scales one.
    struct Place {
      bool on, in;     // the run has the step; its block is in the pool
      int step, unit;
      int64_t row;     // id, then block and head in the pool, then token
      float k, v;
    };
    constexpr int64_t kNoTokens = INT64_MIN;   // no group of the step, or one behind the last token
    int step = run.on() ? run.s0 : 0;
    auto read_id = [&]() {
      Place x = {run.on(), false, step, run.unit, kNoTokens, 0.f, 0.f};
      if (x.on && lane < 4 && step * kPrefixStep + 16 * lane < tokens)
        x.row = a.block_ids[(step * kPrefixStep + 16 * lane) >> bt_log];
      if (x.on) run.step(step);
      return x;
    };
    auto read_scales = [&](Place& x) {
      x.in = x.row >= 0 && x.row < a.c.num_blocks;
      const int64_t hb = x.in ? x.row * a.c.num_kv_heads + x.unit % a.parts.kv_heads : 0;
      x.k = x.in ? a.c.k_scale[hb] : 0.f;
      x.v = x.in ? a.c.v_scale[hb] : x.row == kNoTokens ? 0x1p-8f : 0.f;   // (an ordinary one)
      x.row = (hb << bt_log) + ((x.step * kPrefixStep + 16 * lane) & (bt - 1));
    };
    // one lane for each copy: that of the copy's first 16 tokens
    const bool leads = lane < 4 && 16 * lane % piece == 0;
    auto copy = [&](const uint8_t* pool, bool in, int64_t row) {
      const int copies = __popc(__ballot_sync(0xffffffffu, leads && in));
      if (lane == 0) tc::mbar_arrive_expect_tx(raw_full + raw, copies * piece * HD);
      __syncwarp();
      if (leads && in) bulk_load(smem + L::kOffRaw + raw * L::kRaw + 16 * lane * HD, pool + row * HD, piece * HD, raw_full + raw);
      ++copied;
      if (++raw == L::kRaws) {
        raw = 0;
        raw_phase ^= 1;
      }
    };
    auto free = [&]() { return __all_sync(0xffffffffu, tc::mbar_wait(raw_empty + raw, raw_phase, a.err, &abort)) != 0; };
    Place now = read_id();
    read_scales(now);
    Place next = read_id();
    const ScaleWindow window(__shfl_sync(0xffffffffu, now.v, 0));
    int wide = 0;   // kWide, once a scale of the lane's groups was outside the window
    bool in_v[kAhead + 1] = {};
    int64_t row_v[kAhead + 1] = {};
    for (int it = 0, end = INT_MAX - kAhead; !abort && it < end + kAhead; ++it) {
      bool ok = true;
#pragma unroll
      for (int i = kAhead; i > 0; --i) in_v[i] = in_v[i - 1], row_v[i] = row_v[i - 1];
      if (it < end && !now.on) end = it;
      if (it < end) {
        in_v[0] = now.in;
        row_v[0] = now.row;
        const float ks = now.k;
        float vs = now.v;
        int flags = wide;
        if (!(vs >= window.low && vs <= window.high)) {
          const bool none = vs < kLeastScale;
          if (now.in) {
            if (!none || window.high > kMostBesideNone) flags = wide = kWide;
          } else if (none) {   // (not a group without tokens)
            flags |= kLost;
            if (a.err) atomicOr(a.err, GLT_DEVERR_BAD_SHAPE);
          }
          if (none) {
            flags |= kNone;
            vs = kLeastScale;
          }
        }
        read_scales(next);
        now = next;
        next = read_id();
        ok = free();
        if (ok) {
          PrefixNote& note = notes[it % kNotes];
          if (lane < 4) {
            note.k[lane] = ks;
            note.log_v[lane] = log2f(vs) + ks * 0.f;   // NaN where the scale of K is one (which the softmax drops)
            note.inv_v[lane] = 1.f / vs;
            note.flags[lane] = static_cast<uint8_t>(flags);
          }
          __syncwarp();
          copy(a.c.k, in_v[0], row_v[0]);
        }
      }
      if (ok && it >= kAhead && it < end + kAhead) {
        ok = free();
        if (ok) copy(a.c.v, in_v[kAhead], row_v[kAhead]);
      }
      if (!ok) abort = 1;
    }
  } else if (warp < kCopyWarp && lane == 0) {
    // ------------------------------- products ------------------------------
    const int mine = warp - kIssueWarp;
    const uint32_t q = tc::smem_u32(smem) + (LANES == 2 ? mine * L::kQ : 0), k_at = tc::smem_u32(smem + L::kOffK),
                   v_at = tc::smem_u32(smem + L::kOffV), s = tmem + mine * 128, o = tmem + kColO + mine * 128;
    bool ok = true;
    int base = 0, scored = 0, summed = 0;   // steps before the unit's; the lane's S and P so far
    for (int seg = 0; ok && run.on() && !abort; run.next(), ++seg) {
      const int n = run.s1 - run.s0, first = LANES == 2 ? 0 : mine, by = LANES == 2 ? 1 : 2;
      ok = tc::mbar_wait(q_full, seg & 1, a.err, &abort);
      // S runs two of the lane's steps ahead of its P, so that the softmax of one has the time between
      auto scores = [&](int i) {
        const int it = base + i, slot = it % kSlots;
        if (!tc::mbar_wait(k_full + slot, it / kSlots & 1, a.err, &abort)) return false;
        tc::tc_fence_after();
        const uint32_t kk = k_at + slot * L::kPart, buf = scored++ & 1;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
          tc::umma_bf16(s + buf * kPrefixStep, tc::desc_kmajor(q + (j >> 2) * (kPrefixRows * 128), j & 3),
                        tc::desc_kmajor(kk + (j >> 2) * (kPrefixStep * 128), j & 3), kIdescS, j > 0);
        tc::mbar_arrive(s_full + 2 * mine + buf);
        tc::umma_commit(s_full + 2 * mine + buf);
        tc::umma_commit(k_empty + slot);
        return true;
      };
      if (ok && first < n) ok = scores(first);
      if (ok && first + by < n) ok = scores(first + by);
      for (int i = first; ok && i < n; i += by) {
        const int it = base + i, slot = it % kSlots, buf = summed & 1;
        ok = tc::mbar_wait(v_full + slot, it / kSlots & 1, a.err, &abort) &&
             tc::mbar_wait(p_full + 2 * mine + buf, summed >> 1 & 1, a.err, &abort);
        if (!ok) break;
        ++summed;
        tc::tc_fence_after();
        const uint32_t vv = v_at + slot * L::kPart;
#pragma unroll
        for (int j = 0; j < kPrefixStep / 16; ++j)
          umma_p(o, s + buf * kPrefixStep + 8 * j, tc::make_sdesc(vv + j * 2048, kPrefixStep * 128, 1024), kIdescO,
                 !(i == first && j == 0));
        tc::umma_commit(o_full + mine);
        tc::umma_commit(v_empty + slot);
        if (i + 2 * by < n) ok = scores(i + 2 * by);
      }
      if (ok) tc::umma_commit(unit_done);
      base += n;
    }
    if (!ok) abort = 1;
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == kCopyWarp && lane == 0 && abort) {
    // copies still under way end before the shared memory does
    for (int d = 0; d < L::kRaws && d < copied; ++d) {
      const int j = copied - 1 - d;
      tc::mbar_wait(raw_full + j % L::kRaws, (j / L::kRaws) & 1, a.err);
    }
  }
  if (abort) {
    // no product may still write TMEM when it is given back
    if (lane == 0 && (warp == kIssueWarp || warp == kIssueWarp + 1)) {
      tc::umma_commit(drain);
      tc::mbar_wait(drain, 0, a.err);
    }
    __syncthreads();
  }
  if (warp == kIssueWarp) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Joins what the prefix and the sequences' own tokens gave the query rows: a lane eight channels of a row, SPLIT warps
// a share of its parts each.  blockIdx.y is the sequence.  REPORT: the prefix has no blocks, and so no kernel that would report
// a length.
constexpr int kJoinWarps = 4;
template <int SPLIT, bool REPORT>
__global__ void __launch_bounds__(32 * kJoinWarps, SPLIT > 1 ? 7 : 6) kv8_prefix_join_kernel(const __grid_constant__ AttnArgs a,
                                                                         const __grid_constant__ PrefixParts p) {
  constexpr int kSets = kJoinWarps / SPLIT;   // of rows, of a CTA
  __shared__ float4 sm_z[kJoinWarps][2][32];
  __shared__ float2 sm_ml[kJoinWarps][32];
  const int hd = a.c.head_dim, slot = PrefixParts::slot_floats(hd);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % SPLIT;
  const int per_log = hd == 128 ? 4 : 3, rows = 32 >> per_log;   // of a set
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Kv8Span s = kv8_span(a.b, blockIdx.y, a.c.block_tokens, nullptr);
  const PrefixShares sh(p, p.tokens(REPORT && (blockIdx.x | blockIdx.y | threadIdx.x) == 0 ? a.err : nullptr));
  const int count = s.n * a.nh, first_row = s.row0 * a.nh;   // rows of heads: checked on the host
  const float* own_ml = a.own + static_cast<int64_t>(a.b.rows) * a.nh * hd;
  const int d = (lane & ((1 << per_log) - 1)) * 8;
  // (the CTA's warps take as many turns as its first)
  for (int i0 = blockIdx.x * kSets * rows; i0 < count; i0 += gridDim.x * kSets * rows) {
    const int i = i0 + warp / SPLIT * rows + (lane >> per_log);
    const bool on = i < count;
    const int at = first_row + (on ? i : i0);   // row and head
    const int tok = at / a.nh, head = at - tok * a.nh, kvh = head / a.group, in_group = head - kvh * a.group;
    const int rho = tok * a.group + in_group, tile = rho / kPrefixRows, row = rho % kPrefixRows;
    const int unit = (p.lanes == 2 ? tile >> 1 : tile) * p.kv_heads + kvh;
    // the row's parts: one a CTA, or two; the last is the sequence's own
    const int lane0 = p.lanes == 2 ? tile & 1 : 0, twice = p.lanes == 2 ? 0 : 1;
    int first = 0, parts = 1;
    if (sh.ctas > 0) {
      const int64_t begin = static_cast<int64_t>(unit) * (sh.steps + kPrefixUnitCost);
      first = sh.owner(begin + kPrefixUnitCost);
      parts = ((sh.owner(begin + sh.steps + kPrefixUnitCost - 1) - first + 1) << twice) + 1;
    }
    const float* base = p.slots + static_cast<int64_t>(unit + first) * slot;
    float z[8] = {}, top = -INFINITY, sum = 0.f;
    constexpr int kBatch = 3;   // parts whose loads are in flight at once
    for (int k0 = share; k0 < parts; k0 += kBatch * SPLIT) {
      float m[kBatch], l[kBatch];
      float4 x[kBatch][2];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int part = k0 + k * SPLIT;
        m[k] = -INFINITY;
        l[k] = 0.f;
        x[k][0] = x[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        const float* from;
        if (part < parts - 1) {
          const float* part_at = base + static_cast<int64_t>(part >> twice) * slot;
          const int r = (twice ? part & 1 : lane0) * kPrefixRows + row;
          from = part_at + r * hd + d;
          m[k] = part_at[2 * kPrefixRows * hd + r];
          l[k] = part_at[2 * kPrefixRows * (hd + 1) + r];
        } else {
          from = a.own + static_cast<int64_t>(at) * hd + d;
          if (part == parts - 1) {
            const float2 ml = *reinterpret_cast<const float2*>(own_ml + 2 * static_cast<int64_t>(at));
            m[k] = ml.x;
            l[k] = ml.y;
          }
        }
        if (part < parts) {
          x[k][0] = reinterpret_cast<const float4*>(from)[0];
          x[k][1] = reinterpret_cast<const float4*>(from)[1];
        }
      }
      float peak = top;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) peak = fmaxf(peak, m[k]);
      const TwoFactors old(peak == -INFINITY ? 0.f : top - peak);
      sum = sum * old.b * old.a;
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = z[j] * old.b * old.a;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const TwoFactors f(peak == -INFINITY ? 0.f : m[k] - peak);
        sum = fmaf(l[k] * f.b, f.a, sum);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          z[4 * h] = fmaf(x[k][h].x * f.b, f.a, z[4 * h]);
          z[4 * h + 1] = fmaf(x[k][h].y * f.b, f.a, z[4 * h + 1]);
          z[4 * h + 2] = fmaf(x[k][h].z * f.b, f.a, z[4 * h + 2]);
          z[4 * h + 3] = fmaf(x[k][h].w * f.b, f.a, z[4 * h + 3]);
        }
      }
      top = peak;
    }
    if constexpr (SPLIT > 1) {
      sm_z[warp][0][lane] = make_float4(z[0], z[1], z[2], z[3]);
      sm_z[warp][1][lane] = make_float4(z[4], z[5], z[6], z[7]);
      sm_ml[warp][lane] = make_float2(top, sum);
      __syncthreads();
      if (share == 0) {
        float peak = top;
#pragma unroll
        for (int w = 1; w < SPLIT; ++w) peak = fmaxf(peak, sm_ml[warp + w][lane].x);
        const TwoFactors old(peak == -INFINITY ? 0.f : top - peak);
        sum = sum * old.b * old.a;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = z[j] * old.b * old.a;
#pragma unroll
        for (int w = 1; w < SPLIT; ++w) {
          const float2 ml = sm_ml[warp + w][lane];
          const TwoFactors f(peak == -INFINITY ? 0.f : ml.x - peak);
          sum = fmaf(ml.y * f.b, f.a, sum);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 x = sm_z[warp + w][h][lane];
            z[4 * h] = fmaf(x.x * f.b, f.a, z[4 * h]);
            z[4 * h + 1] = fmaf(x.y * f.b, f.a, z[4 * h + 1]);
            z[4 * h + 2] = fmaf(x.z * f.b, f.a, z[4 * h + 2]);
            z[4 * h + 3] = fmaf(x.w * f.b, f.a, z[4 * h + 3]);
          }
        }
        top = peak;
      }
    }
    if (on && share == 0) {
      write_out<Mode::kPlain>(a, tok, in_group, kvh, hd, d, make_float4(z[0], z[1], z[2], z[3]), top, sum);
      write_out<Mode::kPlain>(a, tok, in_group, kvh, hd, d + 4, make_float4(z[4], z[5], z[6], z[7]), top, sum);
    }
    if (SPLIT > 1) __syncthreads();
  }
}

template <int HD, int FMT>
int launch_prefix(const PrefixArgs& a, cudaStream_t st) {
  auto go = [&](auto kern, int bytes) {
    GLT_TRY(ensure_smem_attr(reinterpret_cast<const void*>(kern), bytes));
    kern<<<a.parts.grid, kPrefixThreads, bytes, st>>>(a);
    GLT_LAUNCH_CHECK();
    return static_cast<int>(GLT_OK);
  };
  return a.parts.lanes == 2 ? go(kv8_prefix_kernel<HD, FMT, 2>, PrefixSmem<HD, 2>::kTotal)
                            : go(kv8_prefix_kernel<HD, FMT, 1>, PrefixSmem<HD, 1>::kTotal);
}

int check_prefix(const GltKv8Cache* c, const GltKv8Prefix* p) {
  if (!p) return fail(GLT_EINVAL, "null argument");
  if (p->num_blocks < 0 || static_cast<int64_t>(p->num_blocks) * c->block_tokens > INT_MAX - 4096)
    return fail(GLT_EINVAL, "kv8: a prefix of %d blocks", p->num_blocks);
  if (!p->length || (p->num_blocks > 0 && !p->block_ids)) return fail(GLT_EINVAL, "kv8: null prefix length or block ids");
  return GLT_OK;
}

// The shares of the prefix; `slots` is left to the caller.
PrefixParts plan_prefix(const GltKv8Cache& c, const GltKv8Batch& b, const GltKv8Prefix& p, int nh) {
  PrefixParts s = {};
  s.length = p.length;
  s.capacity = p.num_blocks * c.block_tokens;
  s.kv_heads = c.num_kv_heads;
  const int64_t rows = static_cast<int64_t>(b.rows) * (nh / c.num_kv_heads);
  s.tiles = static_cast<int>((rows + kPrefixRows - 1) / kPrefixRows);
  s.lanes = s.tiles > 1 ? 2 : 1;
  const int64_t most = static_cast<int64_t>(s.units()) * ((s.capacity + kPrefixStep - 1) / kPrefixStep);
  s.grid = num_sms();
  if (most < s.grid) s.grid = static_cast<int>(most);
  return s;
}
int64_t align32(int64_t n) { return (n + 31) / 32 * 32; }
int64_t own_bytes(const GltKv8Cache& c, const GltKv8Batch& b, int nh) {
  return align32(static_cast<int64_t>(b.rows) * nh * (c.head_dim + 2) * 4);
}
template <int SPLIT, bool REPORT>
int launch_join(const AttnArgs& a, const PrefixParts& parts, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(kv8_most_new(a.c, a.b)) * a.nh, set = kJoinWarps / SPLIT * (256 / a.c.head_dim);
  // as many CTAs as are resident at once go through all rows, if they are enough for a sequence each
  const int64_t resident = (static_cast<int64_t>(num_sms()) * 8 + a.b.num_seqs - 1) / a.b.num_seqs;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min((rows + set - 1) / set, resident)), a.b.num_seqs);
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  GLT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv8_prefix_join_kernel<SPLIT, REPORT>, a, parts));
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

}  // namespace
}  // namespace glt

extern "C" int glt_kv8_prefix_attention_workspace(const GltKv8Cache* cache, const GltKv8Batch* batch,
                                                  const GltKv8Prefix* prefix, int num_heads, int64_t* bytes) {
  if (!bytes) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_heads(cache, batch, num_heads));
  GLT_TRY(glt::check_prefix(cache, prefix));
  *bytes = batch->rows > 0 && batch->max_new > 0
               ? glt::align32(glt::plan(*cache, *batch, num_heads).bytes) +
                     glt::own_bytes(*cache, *batch, num_heads) +
                     glt::plan_prefix(*cache, *batch, *prefix, num_heads).bytes(cache->head_dim)
               : 0;
  return GLT_OK;
}

extern "C" int glt_kv8_prefix_attention(const GltKv8Cache* cache, const GltKv8Batch* batch, const GltKv8Prefix* prefix,
                                        const uint16_t* q, int64_t ld_q, uint16_t* o, int64_t ld_o, float* lse,
                                        int num_heads, float scale, const uint8_t* token_mask, int64_t ld_mask,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  GLT_TRY(glt::check_heads(cache, batch, num_heads));
  GLT_TRY(glt::check_prefix(cache, prefix));
  if (batch->rows == 0 || batch->max_new == 0) return GLT_OK;
  if (static_cast<int64_t>(batch->rows) * num_heads > INT_MAX / 2)
    return glt::fail(GLT_EINVAL, "kv8: %d rows of %d heads", batch->rows, num_heads);
  glt::AttnArgs a;
  glt::Plan p;
  GLT_TRY(glt::prepare(cache, batch, q, ld_q, o, ld_o, lse, num_heads, scale, 0, token_mask, ld_mask, workspace,
                       workspace_bytes, &a, &p));
  glt::PrefixParts parts = glt::plan_prefix(*cache, *batch, *prefix, num_heads);
  const int64_t first = glt::align32(p.bytes), second = first + glt::own_bytes(*cache, *batch, num_heads),
                need = second + parts.bytes(cache->head_dim);
  if (workspace_bytes < need)
    return glt::fail(GLT_EINVAL, "kv8: workspace must be 32-byte aligned and hold %lld bytes", (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) & 31) return glt::fail(GLT_EINVAL, "kv8: workspace must be 32-byte aligned");
  a.own = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + first);
  parts.slots = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + second);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  a.chained = parts.grid > 0;
  if (a.chained) {
    const glt::PrefixArgs x = {*cache, prefix->block_ids, q, ld_q, batch->rows * a.group, a.group, a.scale, parts, a.err};
    const bool int8 = cache->format == GLT_KV8_INT8;
    if (cache->head_dim == 128)
      GLT_TRY((int8 ? glt::launch_prefix<128, GLT_KV8_INT8>(x, st) : glt::launch_prefix<128, GLT_KV8_E4M3>(x, st)));
    else
      GLT_TRY((int8 ? glt::launch_prefix<64, GLT_KV8_INT8>(x, st) : glt::launch_prefix<64, GLT_KV8_E4M3>(x, st)));
  }
  if (glt::own_is_short(a))
    GLT_TRY(glt::launch_own(a, st));
  else
    GLT_TRY(glt::launch_all<glt::Mode::kPrefix>(a, p, st));
  if (parts.grid == 0) return glt::launch_join<1, true>(a, parts, st);
  // Rows of many parts go to four warps, others to one (whole calls, four warps / one, in us, by the parts of a unit: 64 sequences of 4
  // heads over each of 6, 8, 10, 12, 16 and 20 KV heads, 25 parts 51.2 / 57.5, 19 55.9 / 61.0, 15 69.7 / 70.3, 12 76.3 / 75.5, 9 86.8 / 85.4,
  // 7 102.7 / 98.1; 3 sequences, units of up to 26 parts 14.5 / 17.6; 128 sequences, 10 parts 197 / 195; 18944 rows of 3 107.4 / 87.3).
  return (parts.lanes == 2 ? 1 : 2) * parts.grid > 12 * parts.units() ? glt::launch_join<4, false>(a, parts, st) : glt::launch_join<1, false>(a, parts, st);
}
