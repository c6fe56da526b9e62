// Attention over few own tokens of each sequence behind a shared prefix: sums of values, maxima and sums of weights in
// 32 bits, as Mode::kPrefix of kv8_attention.cuh leaves them.
//
// A warp takes 16 query rows (token x head of the group) of a KV head through all tokens that they see, 16 at a time. Nothing
// is shared or joined, so a unit's beginning and end cost next to nothing, and there is one launch less.  Queries are operand A of
// mma.sync, and codes go from memory to operand B in registers.  The order of a contraction's index and of
// the channels is free: a lane loads 16 contiguous bytes of K for four k-steps of S, and 16 of V
// (8 with head_dim 64) for a column of as many products.  P stays in the registers that S came in.
// The scale of V joins the exponent, and P is rounded to f16, counted 2^15 at the running maximum of the exponents:
// 11 bits down to 2^-29 of the row's largest summand, and below that within 2^-40 of it.  Over the scale, the same numbers make
// the sum of weights, unless scales lie far apart (ScaleWindow).
//
// What bounds it: latency, about 0.8 us a step of 16 tokens, of which the next step's codes are on their way during one
// (fetching four steps ahead to L2 gained nothing).  So it is for short tables (own_is_short).
#pragma once

#include <algorithm>

#include "kv8_attention.cuh"

namespace glt {
namespace {

constexpr int kOwnWarps = 4;
constexpr int kOwnRows = 16;
constexpr int kOwnStep = 16;   // tokens: blocks hold a multiple of them
constexpr float kOwnLift = 15.f;   // (over the least scale, a weight's 2^15 stay within 32 bits)

template <int HD, int FMT>
__global__ void __launch_bounds__(32 * kOwnWarps, 2) kv8_own_kernel(const __grid_constant__ AttnArgs a, int tiles) {
  constexpr int kWords = HD / 32;   // of V, of a token, of a lane
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  // neighbouring warps have the tiles of a KV head, or its neighbours
  const int unit = static_cast<int>(blockIdx.x) * kOwnWarps + (threadIdx.x >> 5), kvh = unit / tiles, tile = unit - kvh * tiles;
  const int seq = blockIdx.y;
  const Kv8Span s = kv8_span(a.b, seq, a.c.block_tokens, unit == 0 && lane == 0 ? a.err : nullptr);
  const int rows = s.n * a.group, r0 = tile * kOwnRows;   // checked on the host
  if (kvh < a.c.num_kv_heads && r0 < rows) {
    const int bt_log = 31 - __clz(a.c.block_tokens);
    const int end = s.past + min(r0 + kOwnRows - 1, rows - 1) / a.group + 1;   // tokens that some row sees
    const int32_t* ids = a.b.block_table + static_cast<int64_t>(seq) * a.b.max_blocks;
    const uint8_t* mask = a.mask ? a.mask + seq * a.ld_mask : nullptr;

    // ---- queries, brought to f16 by a power of two as in kv8_attention.cuh
    uint32_t qa[HD / 16][4];
    float qs[2];
    int pos[2];
    auto power = [](int e) { return __int_as_float((e + 127) << 23); };   // 2^e, |e| < 127
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + g + 8 * h, i = r / a.group;
      pos[h] = s.past + i;
      uint4 v[HD / 64][2];
      const uint16_t* src = a.q + (s.row0 + static_cast<int64_t>(i)) * a.ld_q + (kvh * a.group + r - i * a.group) * HD;
#pragma unroll
      for (int k = 0; k < HD / 64; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          v[k][j] = r < rows ? *reinterpret_cast<const uint4*>(src + (HD == 128 ? 2 * c + k : c) * 16 + j * 8) : make_uint4(0, 0, 0, 0);
      float peak = 0.f;
#pragma unroll
      for (int k = 0; k < HD / 64; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float f[8];
          unpack8(v[k][j], f);
#pragma unroll
          for (int x = 0; x < 8; ++x) peak = fmaxf(peak, fabsf(f[x]));
        }
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
      int e = 0;
      if (peak > 0.f && peak <= FLT_MAX) e = 13 - (static_cast<int>(__float_as_uint(peak) >> 23) - 127);
      const float f1 = power(e >> 1), f2 = power(e - (e >> 1));   // 2^e may be out of range
      qs[h] = a.scale * 1.4426950408889634f * power(-(e >> 1)) * power(-(e - (e >> 1)));
#pragma unroll
      for (int k = 0; k < HD / 64; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float f[8];
          unpack8(v[k][j], f);
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] = f[x] * f1 * f2;
          const int at = k * 4 + j * 2;   // k-steps: of four channels of each lane of the row
          qa[at][h] = pack_f16x2(f[0], f[1]);
          qa[at][2 + h] = pack_f16x2(f[2], f[3]);
          qa[at + 1][h] = pack_f16x2(f[4], f[5]);
          qa[at + 1][2 + h] = pack_f16x2(f[6], f[7]);
        }
    }

    // ---- tokens: the codes of a step come while the one before is worked on, and its block's id a step earlier
    struct Step {
      uint4 k[2][HD / 64];       // tokens g, 8 + g
      uint32_t v[4][kWords];     // tokens 2c, 2c + 1, 2c + 8, 2c + 9
      float ks, vs;
      int seen;                  // of these: bit i, some row may see it
    };
    auto id_of = [&](int t0) { return t0 < end ? ids[t0 >> bt_log] : 0; };
    auto load = [&](int t0, int id, Step& x) {
      const bool on = id >= 0 && id < a.c.num_blocks;
      if (!on && lane == 0 && a.err) atomicOr(a.err, GLT_DEVERR_BAD_SHAPE);
      const int64_t hb = on ? static_cast<int64_t>(id) * a.c.num_kv_heads + kvh : 0;
      const int64_t row = (hb << bt_log) + (t0 & (a.c.block_tokens - 1));
      x.ks = a.c.k_scale[hb];
      x.vs = a.c.v_scale[hb];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int k = 0; k < HD / 64; ++k)
          x.k[n][k] = *reinterpret_cast<const uint4*>(a.c.k + (row + 8 * n + g) * HD + (HD == 128 ? 2 * c + k : c) * 16);
      x.seen = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = (i >> 1) * 8 + 2 * c + (i & 1);
        const uint8_t* src = a.c.v + (row + t) * HD + g * (HD / 8);
        if constexpr (HD == 128) {
          const uint4 w = *reinterpret_cast<const uint4*>(src);
          x.v[i][0] = w.x, x.v[i][1] = w.y, x.v[i][2] = w.z, x.v[i][3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(src);
          x.v[i][0] = w.x, x.v[i][1] = w.y;
        }
        if (on && t0 + t < end && (!mask || mask[t0 + t])) x.seen |= 1 << i;
      }
    };

    float acc[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool wide = false;   // a scale of V so far was outside the window
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    Step now, ahead;
    int id = id_of(kOwnStep);
    load(0, id_of(0), ahead);
    const ScaleWindow window(ahead.vs);
#pragma unroll 1
    for (int t0 = 0; t0 < end; t0 += kOwnStep) {
      now = ahead;
      if (t0 + kOwnStep < end) {
        load(t0 + kOwnStep, id, ahead);
        id = id_of(t0 + 2 * kOwnStep);
      }
      if (!__any_sync(0xffffffffu, now.seen != 0)) continue;   // its scales may be anything
      float z[2][4] = {};   // S: tokens 2c, 2c + 1 of row g and of row 8 + g; the same 8 tokens on
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int k = 0; k < HD / 64; ++k) {
          const uint32_t w[4] = {now.k[n][k].x, now.k[n][k].y, now.k[n][k].z, now.k[n][k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_f16(z[n], qa[k * 4 + j], two_codes<FMT, 0>(w[j]), two_codes<FMT, 1>(w[j]));
        }
      const bool some = !(now.vs < kLeastScale);
      const float vs = some ? now.vs : kLeastScale, log_v = log2f(vs), inv_v = 1.f / vs;
      wide |= some ? !(now.vs >= window.low && now.vs <= window.high) : window.high > kMostBesideNone;
      uint32_t p[4];
      float factor[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float u = now.ks * qs[h];
        float x[4], peak = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = t0 + (i >> 1) * 8 + 2 * c + (i & 1);
          x[i] = (now.seen >> i & 1) && t <= pos[h] ? fmaf(z[i >> 1][2 * h + (i & 1)], u, log_v) : -INFINITY;
          peak = fmaxf(peak, x[i]);
        }
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
        const float top = fmaxf(m[h], peak), ref = kOwnLift - (top == -INFINITY ? 0.f : top);
        factor[h] = m[h] == -INFINITY ? 1.f : ex2_approx(m[h] - top);   // (without a maximum the sums are 0, or NaN)
        const float before = m[h];
        m[h] = top;
        float y[4], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = ex2_approx(x[i] + ref);
          sum += y[i];
        }
        if (wide) {
          const TwoFactors f(before == -INFINITY ? 0.f : before - top);
          float lifted = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) lifted += ex2_approx(x[i] + ref + kWideLift);
          l[h] = l[h] * f.a * f.b + wide_weights(lifted, log_v, inv_v);
        } else {
          l[h] = fmaf(sum, inv_v, l[h] * factor[h]);
        }
        p[h] = pack_f16x2(y[0], y[1]);
        p[2 + h] = pack_f16x2(y[2], y[3]);
      }
      if (__any_sync(0xffffffffu, factor[0] != 1.f || factor[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) acc[j][0] *= factor[0], acc[j][1] *= factor[0], acc[j][2] *= factor[1], acc[j][3] *= factor[1];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!some || !(now.seen >> i & 1)) {   // what no row sees may hold anything
#pragma unroll
          for (int w = 0; w < kWords; ++w) now.v[i][w] = FMT == GLT_KV8_INT8 ? 0x80808080u : 0u;
        }
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        uint32_t lo[4], hi[4];   // channels 4w, 4w + 1 and 4w + 2, 4w + 3 of the four tokens
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] = two_codes<FMT, 0>(now.v[i][w]), hi[i] = two_codes<FMT, 1>(now.v[i][w]);
        mma_f16(acc[4 * w], p, __byte_perm(lo[0], lo[1], 0x5410), __byte_perm(lo[2], lo[3], 0x5410));
        mma_f16(acc[4 * w + 1], p, __byte_perm(lo[0], lo[1], 0x7632), __byte_perm(lo[2], lo[3], 0x7632));
        mma_f16(acc[4 * w + 2], p, __byte_perm(hi[0], hi[1], 0x5410), __byte_perm(hi[2], hi[3], 0x5410));
        mma_f16(acc[4 * w + 3], p, __byte_perm(hi[0], hi[1], 0x7632), __byte_perm(hi[2], hi[3], 0x7632));
      }
    }

    // ---- the rows' results: column 2c + x of the product j is channel (2c + x) HD / 8 + j
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int r = r0 + g + 8 * h;
      if (r < rows) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int j = 0; j < HD / 8; j += 4)
            write_out<Mode::kPrefix>(a, s.row0, r, kvh, HD, (2 * c + x) * (HD / 8) + j,
                                     make_float4(acc[j][2 * h + x], acc[j + 1][2 * h + x], acc[j + 2][2 * h + x], acc[j + 3][2 * h + x]),
                                     m[h] - kOwnLift, l[h]);
      }
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // who waits for this kernel waits for the prefix's
}

int own_tiles(const AttnArgs& a) { return (kv8_most_new(a.c, a.b) * a.group + kOwnRows - 1) / kOwnRows; }   // 32 bits: check_heads
// Whether the sequences' tables hold so few tokens that this kernel is the faster one: the more warps there are, the more the ends of units
// cost the other.  Whole calls behind 777 tokens, head_dim 128, e4m3, other kernel / this one in us, by the tokens of a table:
//                                                            256            320            384            512
//   1 sequence, 1 token, 32 heads over 8: 8 warps        21.9 / 22.5    22.4 / 25.3    22.8 / 28.7    21.7 / 34.7
//   2 sequences, 37 tokens, 32 heads over 4: 152 warps   37.9 / 33.9    40.2 / 37.6    40.2 / 41.7    42.3 / 49.5
//   64 sequences, 1 token, 32 heads over 8: 512          38.9 / 32.5    42.3 / 36.9    42.8 / 41.2    47.3 / 49.9
//   128 sequences: 1024                                  55.4 / 48.4    62.2 / 54.4    64.1 / 59.9    70.5 / 68.2
//   100 sequences, 5 tokens, 64 heads over 8: 2400       145 / 108      161 / 120      165 / 132      186 / 153
// (Next to its bound the rule is off by up to 7 %: 152 warps with 320 tokens, 512 with 384, 1024 with 512.)  It goes by the room of a
// table, since what the sequences hold is known on the device alone: tables as tight as the lengths allow are the faster ones.
bool own_is_short(const AttnArgs& a) {
  const int64_t warps = static_cast<int64_t>(a.b.num_seqs) * a.c.num_kv_heads * own_tiles(a);
  return static_cast<int64_t>(a.b.max_blocks) * a.c.block_tokens <= std::min<int64_t>(512, 256 + warps / 8);
}
template <int HD, int FMT>
int launch_own(const AttnArgs& a, cudaStream_t st) {
  const int tiles = own_tiles(a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((tiles * a.c.num_kv_heads + kOwnWarps - 1) / kOwnWarps, a.b.num_seqs);
  cfg.blockDim = dim3(32 * kOwnWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.chained ? 1 : 0;   // behind any other kernel, its writes would not be awaited
  GLT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv8_own_kernel<HD, FMT>, a, tiles));
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}
int launch_own(const AttnArgs& a, cudaStream_t st) {
  const bool int8 = a.c.format == GLT_KV8_INT8;
  if (a.c.head_dim == 128) return int8 ? launch_own<128, GLT_KV8_INT8>(a, st) : launch_own<128, GLT_KV8_E4M3>(a, st);
  return int8 ? launch_own<64, GLT_KV8_INT8>(a, st) : launch_own<64, GLT_KV8_E4M3>(a, st);
}

}  // namespace
}  // namespace glt
