// Products in 8-bit integers with a scale for each token and each channel (glt_w8_*).
//
//   y[m, n] = s_m t_n sum_k c[m, k] w[n, k] (+ r[m, n]),   c[m, k] = nearest(x[m, k] / s_m),   s_m = max_k |x[m, k]| / 127
//
// The sum of products of bytes is an integer and exact, in any order.  What is rounded: x to its codes (that is
// the operator), the integer to 24 bits, two products with the scales, the residual's sum, and y.
//
// Quantising: one CTA a token keeps the row in registers between the maximum and the codes (with a norm, between
// the sum of squares, the maximum and the codes), so x is read once; bound by HBM for many tokens.
//
// Product: weights are operand A of tcgen05.mma kind::i8 (128 or 256 channels), tokens operand B, so that a
// thread of the epilogue owns a channel, a warp writes 32 neighbouring channels of a token whatever their alignment,
// and few tokens cost few columns.  Two kernels:
//   * w8_stream_kernel, bound by the weights' bytes.  A CTA takes 128 channels, up to 64 tokens and a share of K; the CTAs
//     of a cluster share K and add their integers through distributed shared memory.  It starts
//     (programmatic dependent launch) while the tokens are quantised and fills its ring with weights.
//     8 tokens by 28672 x 4096: 22.7 us, 5.2 TB/s; 60 tokens by 32001 x 4097: 30.8 us, where every CTA's tokens come through L2 too.
//   * the CTA-pair kernel of tc_gemm_pair.cuh with byte operands, bound by the tensor cores and, in long runs, the power
//     limit: 8192 tokens by 28672 x 4096 654 us (2.9e15 operations a second), 2047 by 4096 x 14336 95 us (2.5e15: 128 tiles are
//     1.7 rounds of 74 pairs).
// The first goes on while all its tiles are resident at once: 64 / 65 tokens by 28672 x 4096 27.4 / 41.0 us against 33.8 / 34.8 by
// pairs, 512 by 4096 x 4096 18.9 against 21.7, 400 by 6144 x 4096 30.1 against 21.7.
#include <float.h>
#include <limits.h>

#include "gemm.cuh"

namespace glt {
namespace {

// --------------------------------------------------------------------------- quantising rows
struct QuantArgs {
  const uint16_t* x;
  int64_t ld_x;
  int rows, K;
  const uint16_t* norm;   // NULL: none
  float eps;
  int8_t* codes;
  int64_t ld_codes;
  float* scales;
};

__device__ __forceinline__ uint4 load_vec(const uint16_t* row, int v, int K, bool aligned) {
  const int k = v * 8;
  if (aligned && k + 8 <= K) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t w[4] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < K) w[i >> 1] |= static_cast<uint32_t>(row[k + i]) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The largest (or the sum) of all threads' values of a row, in every thread.
template <int THREADS, bool MAX>
__device__ __forceinline__ float block_join(float v, float* sm) {
  v = MAX ? warp_max(v) : warp_sum(v);
  __syncthreads();   // sm may still be read
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = sm[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) r = MAX ? fmaxf(r, sm[i]) : r + sm[i];
  return r;
}

// Codes of eight values.  Common: y inv with inv = fl(1 / s) is within two units in the last place of the quotient, one
// correction by the remainder brings it within one, and a second gives the quotient rounded to nearest
// (Markstein's theorem, IBM Journal of Research and Development 34, 1990); 1.5 * 2^23 added to it leaves the
// nearest integer, ties to even, in the low bits.  |q| <= 127 (1 + 2^-23), so nothing needs a clamp.
__device__ __forceinline__ uint2 encode8(const float (&y)[8], float s, float inv, bool common) {
  uint32_t c[8];
  if (common) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q = y[i] * inv;
      q = fmaf(fmaf(-q, s, y[i]), inv, q);
      c[i] = __float_as_uint(fmaf(fmaf(-q, s, y[i]), inv, q) + 12582912.f);
    }
  } else {   // a scale of 0 (or one that is no number), or so small that its reciprocal or the remainders leave the float range
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c[i] = s > 0.f && s <= FLT_MAX ? static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(__fdiv_rn(y[i], s), -127.f), 127.f))) : 0u;
  }
  auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
  };
  return make_uint2(four(c[0], c[1], c[2], c[3]), four(c[4], c[5], c[6], c[7]));
}

// VECS vectors of eight values a thread; VECS = 0: any length, read again for each pass.  A CTA takes one row after the
// other; the next one's loads are under way while a row is worked on, whose values stay in registers from the norm to the
// codes: for many tokens instructions and the latency between barriers bound it (8192 rows of 4096 with their norm: 34 us,
// 0.44 of the copy rate; a warp a row, without barriers, took 64).
template <int THREADS, int VECS, bool NORM>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) w8_quantize_kernel(const QuantArgs a) {
  __shared__ float sm[THREADS / 32];
  asm volatile("griddepcontrol.launch_dependents;");
  const int vecs = (a.K + 15) / 16 * 2;   // codes are written up to a multiple of 16
  const bool g_aligned = NORM && (reinterpret_cast<uintptr_t>(a.norm) & 15u) == 0;
  constexpr int kHeld = VECS > 0 ? VECS : 1;
  uint4 ahead[kHeld];
  auto row_of = [&](int64_t r) { return a.x + r * a.ld_x; };
  auto is_aligned = [&](int64_t r) { return (reinterpret_cast<uintptr_t>(row_of(r)) & 15u) == 0; };
  auto load = [&](int64_t r) {
    const bool aligned = is_aligned(r);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = threadIdx.x + i * THREADS;
      ahead[i] = v < vecs ? load_vec(row_of(r), v, a.K, aligned) : make_uint4(0, 0, 0, 0);
    }
  };
  if (VECS > 0) load(blockIdx.x);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    float y[kHeld][8];
    if constexpr (VECS > 0) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) unpack8(ahead[i], y[i]);
      if (r + gridDim.x < a.rows) load(r + gridDim.x);
    }
    // f(vector's index, its eight values as they stand)
    float factor = 1.f, lift = 1.f;
    bool normed = false;
    auto for_each = [&](auto&& f) {
      if constexpr (VECS > 0) {
#pragma unroll
        for (int i = 0; i < VECS; ++i) f(threadIdx.x + i * THREADS, y[i]);
      } else {
        const bool aligned = is_aligned(r);
        for (int v = threadIdx.x; v < vecs; v += THREADS) {
          unpack8(load_vec(row_of(r), v, a.K, aligned), y[0]);
          if (lift != 1.f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[0][j] *= lift;
          }
          if (normed) {
            float g[8];
            unpack8(load_vec(a.norm, v, a.K, g_aligned), g);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[0][j] = y[0][j] * factor * g[j];
          }
          f(v, y[0]);
        }
      }
    };
    if constexpr (NORM) {
      auto mean_square = [&]() {
        float sum = 0.f;
        for_each([&](int, float (&f)[8]) {
#pragma unroll
          for (int j = 0; j < 8; ++j) sum = fmaf(f[j], f[j], sum);
        });
        return block_join<THREADS, false>(sum, sm) / a.K;
      };
      float mean = mean_square() + a.eps;
      // A mean that leaves the float range is taken again of x / 2^80, whose squares sum up to 2^(96 + 17) at most, and one below
      // 2^-100, where squares lose bits, of 2^100 x: so a row of any finite bf16 has its norm.  Its values stay multiplied.
      if (!(mean <= FLT_MAX) || mean < 0x1p-100f) {
        lift = mean < 0x1p-100f ? 0x1p100f : 0x1p-80f;
        if constexpr (VECS > 0) {
#pragma unroll
          for (int i = 0; i < VECS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) y[i][j] *= lift;
        }
        mean = mean_square() + a.eps * lift * lift;
      }
      factor = rsqrtf(mean);
      normed = true;
      if constexpr (VECS > 0) {
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
          const int v = threadIdx.x + i * THREADS;
          float g[8];
          unpack8(v < vecs ? load_vec(a.norm, v, a.K, g_aligned) : make_uint4(0, 0, 0, 0), g);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[i][j] = y[i][j] * factor * g[j];
        }
      }
    }
    float peak = 0.f, odd = 0.f;   // odd: NaN when a value is NaN or infinite
    for_each([&](int, float (&f)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        peak = fmaxf(peak, fabsf(f[j]));
        odd = fmaf(f[j], 0.f, odd);
      }
    });
    peak = block_join<THREADS, true>(odd == 0.f ? peak : INFINITY, sm);
    // a row that holds an infinity or NaN has no scale: it says so
    const float s = peak <= FLT_MAX ? __fdiv_rn(peak, 127.f) : __uint_as_float(0x7FC00000u);
    if (threadIdx.x == 0) a.scales[r] = s;
    const bool common = s >= 0x1p-100f && s <= 0x1p100f;   // reciprocals and remainders are normal numbers
    const float inv = __frcp_rn(s);
    int8_t* out = a.codes + r * a.ld_codes;
    for_each([&](int v, float (&f)[8]) {
      if (v < vecs) *reinterpret_cast<uint2*>(out + v * 8) = encode8(f, s, inv, common);
    });
  }
}

// A row goes to as many threads as hold it with up to four vectors each.
int quantize(const QuantArgs& a, cudaStream_t st) {
  auto go = [&](auto threads, auto vecs) {
    constexpr int T = decltype(threads)::value, V = decltype(vecs)::value;
    const int most = num_sms() * (1024 / T);   // as many as are resident
    const int grid = a.rows < most ? a.rows : most;
    if (a.norm)
      w8_quantize_kernel<T, V, true><<<grid, T, 0, st>>>(a);
    else
      w8_quantize_kernel<T, V, false><<<grid, T, 0, st>>>(a);
  };
  if (a.K <= 4096)
    go(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  else if (a.K <= 8192)
    go(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
  else if (a.K <= 16384)
    go(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
  else
    go(std::integral_constant<int, 512>{}, std::integral_constant<int, 0>{});
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

// --------------------------------------------------------------------------- products
struct ProductArgs {
  const float* x_scales;
  const float* w_scales;
  void* y;
  int64_t ld_y;
  const uint16_t* resid;
  int64_t ld_r;
  int M, N;
};

// A sum is below 2^31, so times a channel's scale t below 2^96 it stays within 32 bits; a larger t is multiplied last, so that only a
// result that leaves the range does.  LARGE: such a t may be among the warp's channels (with the choice for every element in
// the pair kernel, 8192 tokens by 28672 x 4096 took 688 us for 672).  Underflow takes nothing: a product with an integer is a
// multiple of the other factor's last place.
constexpr float kLargeScale = 0x1p96f;
template <bool BF16, bool RESID, bool LARGE>
__device__ __forceinline__ void put(const ProductArgs& a, int m, int n, int sum, float t, float s, uint16_t r) {
  float z = static_cast<float>(sum) * t * s;
  if (LARGE && t >= kLargeScale) z = static_cast<float>(sum) * s * t;
  if (RESID) z += bf16_bits_to_f32(r);
  if (BF16)
    static_cast<uint16_t*>(a.y)[m * a.ld_y + n] = bf16_bits_rn(z);
  else
    static_cast<float*>(a.y)[m * a.ld_y + n] = z;
}

// The pair kernel's epilogue: rows are channels, columns tokens.
template <bool BF16, bool RESID>
struct EpiW8 {
  static constexpr int kParts = 2;
  ProductArgs a;
  __device__ __forceinline__ void operator()(const tc::EpiCtx<256>& c) const {
    const bool on = c.row < a.N;
    const float t = on ? a.w_scales[c.row] : 0.f;
    if (__any_sync(0xffffffffu, t >= kLargeScale))
      write<true>(c, on, t);
    else
      write<false>(c, on, t);
  }
  template <bool LARGE>
  __device__ __forceinline__ void write(const tc::EpiCtx<256>& c, bool on, float t) const {
#pragma unroll 1
    for (int j = c.part * 128; j < c.part * 128 + 128; j += 32) {
      if (c.n0 + j >= a.M) break;
      const int m0 = c.n0 + j, m1 = min(a.M, m0 + 32) - 1;
      float v[32];
      uint16_t r[32];   // all reads before the first write, and none behind a branch of its own
      if (RESID) {
        const uint16_t* from = a.resid + (on ? c.row : 0);
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = from[min(m0 + i, m1) * a.ld_r];
      }
      const float s = a.x_scales[min(m0 + static_cast<int>(threadIdx.x & 31), m1)];   // a lane's token
      c.load(j, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float si = __shfl_sync(0xffffffffu, s, i);
        if (on && m0 + i <= m1) put<BF16, RESID, LARGE>(a, m0 + i, c.row, __float_as_int(v[i]), t, si, RESID ? r[i] : 0);
      }
    }
  }
};

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void umma_s8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

constexpr int kChannels = 128;   // of a CTA of the stream kernel
constexpr int kStreamThreads = 192;
constexpr int kMaxShares = 8;    // CTAs of a cluster

template <int NT>
struct Stream {
  static constexpr int kA = kChannels * 128, kB = NT * 128, kStage = kA + kB;
  static constexpr int kCtasPerSm = 2;
  static constexpr int kStages = 110 * 1024 / kStage;
  static constexpr int kSmem = 1024 + kStages * kStage + (2 * kStages + 2) * 8 + 16;
  static constexpr int kTmem = NT < 32 ? 32 : NT;
};

// shares: CTAs of the cluster, blockIdx.x % shares is the CTA's.
template <int NT, bool BF16, bool RESID>
__global__ void __launch_bounds__(kStreamThreads) w8_stream_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                  const __grid_constant__ CUtensorMap map_x, int blocks,
                                                                  int shares, const ProductArgs a, unsigned int* err) {
  using S = Stream<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-tc::smem_u32(smem_raw) & 1023u);   // the swizzle goes by address
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kStages * S::kStage);
  uint64_t* empty = full + S::kStages;
  uint64_t* done = empty + S::kStages;
  uint64_t* drain = done + 1;
  uint32_t* slot = reinterpret_cast<uint32_t*>(drain + 1);
  __shared__ int abort_storage;
  volatile int& abort = abort_storage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = static_cast<int>(blockIdx.x % shares);
  const int n0 = static_cast<int>(blockIdx.x / shares) * kChannels, m0 = static_cast<int>(blockIdx.y) * NT;
  const int begin = static_cast<int>(static_cast<int64_t>(blocks) * share / shares);
  const int end = static_cast<int>(static_cast<int64_t>(blocks) * (share + 1) / shares);
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      tc::mbar_init(full + i, 1);
      tc::mbar_init(empty + i, 1);
    }
    tc::mbar_init(done, 1);
    tc::mbar_init(drain, 1);
    abort = 0;
    tc::fence_mbar_init();
    tc::tma_prefetch_desc(&map_w);
    tc::tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tc::tmem_alloc(slot, S::kTmem);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot;
  int issued = 0;

  if (warp == 0) {
    if (lane == 0) {
      // the weights are not the kernel before's: they come while it runs
      const int first = min(end - begin, S::kStages);
      for (int i = 0; i < first; ++i) {
        tc::mbar_arrive_expect_tx(full + i, S::kStage);
        tc::tma_load_2d(smem + i * S::kStage, &map_w, full + i, (begin + i) * 64, n0);
      }
      asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int i = 0; i < first; ++i)
        tc::tma_load_2d(smem + i * S::kStage + S::kA, &map_x, full + i, (begin + i) * 64, m0);
      issued = first;
      for (int b = begin + first; b < end; ++b, ++issued) {
        const int s = issued % S::kStages;
        if (!tc::mbar_wait(empty + s, ((issued / S::kStages) & 1) ^ 1, err, &abort)) {
          abort = 1;
          break;
        }
        uint8_t* dst = smem + s * S::kStage;
        tc::mbar_arrive_expect_tx(full + s, S::kStage);
        tc::tma_load_2d(dst, &map_w, full + s, b * 64, n0);
        tc::tma_load_2d(dst + S::kA, &map_x, full + s, b * 64, m0);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = tc::make_idesc_s8(kChannels, NT);
      uint32_t acc = 0;
      int it = 0;
      for (int b = begin; b < end; ++b, ++it) {
        const int s = it % S::kStages;
        if (!tc::mbar_wait(full + s, (it / S::kStages) & 1, err, &abort)) {
          abort = 1;
          break;
        }
        tc::tc_fence_after();
        const uint32_t at = tc::smem_u32(smem + s * S::kStage);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          umma_s8(tmem, tc::desc_kmajor(at, k), tc::desc_kmajor(at + S::kA, k), idesc, acc);
          acc = 1;
        }
        tc::umma_commit(empty + s);
      }
      if (!abort) tc::umma_commit(done);
    }
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the tokens' scales
  }
  // The cluster's integers.  Each CTA adds up a run of `chunk` tokens and takes the others' parts of it into the
  // memory of its ring, which is free once all its products are done.
  const int tokens = min(NT, a.M - m0), chunk = ((tokens + shares - 1) / shares + 7) & ~7;
  bool good = true;
  if (warp >= 2) {
    good = __all_sync(0xffffffffu, tc::mbar_wait(done, 0, err, &abort));
    if (!good) abort = 1;
    tc::tc_fence_after();
  }
  const int sub = warp & 3, ch = sub * 32 + lane, n = n0 + ch;
  const uint32_t from = tmem + (static_cast<uint32_t>(sub * 32) << 16);
  if (shares > 1) {
    __syncwarp();
    tc::cluster_sync_all();
    if (warp >= 2 && good) {
      for (int to = 0; to < shares; ++to) {
        const int c0 = to * chunk, c1 = min(tokens, c0 + chunk);
        if (to == share || c0 >= c1) continue;
        // part `share` (less one behind the receiver's own) of the receiver's memory: [part][four tokens][channel][token]
        const uint32_t dst = tc::mapa_shared(
            tc::smem_u32(smem) + ((share - (share > to ? 1 : 0)) * chunk * kChannels + ch * 4) * 4, static_cast<uint32_t>(to));
        for (int c = c0; c < c1; c += 8) {
          uint32_t v[8];
          tmem_ld8(from + static_cast<uint32_t>(c), v);
#pragma unroll
          for (int i = 0; i < 8; i += 4)
            asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (c + i - c0) * kChannels * 4),
                         "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
                         : "memory");
        }
      }
    }
    __syncwarp();
    tc::cluster_sync_all();
  }
  if (warp >= 2 && good) {
    const int c0 = share * chunk, c1 = min(tokens, c0 + chunk);
    const float t = n < a.N ? a.w_scales[n] : 0.f;
    for (int c = c0; c < c1; c += 8) {
      uint32_t v[8];
      uint16_t r[8] = {};   // (y may be the residual: all reads before the first write)
      float s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int m = m0 + min(c + i, c1 - 1);
        s[i] = a.x_scales[m];
        if (RESID) r[i] = a.resid[m * a.ld_r + min(n, a.N - 1)];
      }
      tmem_ld8(from + static_cast<uint32_t>(c), v);
      const int4* part = reinterpret_cast<const int4*>(smem) + (c - c0) / 4 * kChannels + ch;
      for (int p = 0; p < shares - 1; ++p) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int4 x = part[p * (chunk / 4) * kChannels + h * kChannels];
          v[4 * h] += x.x, v[4 * h + 1] += x.y, v[4 * h + 2] += x.z, v[4 * h + 3] += x.w;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n < a.N && c + i < c1) put<BF16, RESID, true>(a, m0 + c + i, n, static_cast<int>(v[i]), t, s[i], r[i]);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (abort) {
    // copies still under way end before the shared memory does, and products before their accumulator
    if (threadIdx.x == 0)
      for (int d = 0; d < S::kStages && d < issued; ++d) {
        const int j = issued - 1 - d;
        tc::mbar_wait(full + j % S::kStages, (j / S::kStages) & 1, err);
      }
    if (threadIdx.x == 32) {
      tc::umma_commit(drain);
      tc::mbar_wait(drain, 0, err);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, S::kTmem);
  }
}

// Operands as maps of pairs of bytes: K is padded with zeros to a multiple of 16.
struct Codes {
  const int8_t* p;
  int64_t ld;
};

template <int NT, bool BF16, bool RESID>
int launch_stream(const Codes& w, const Codes& x, int K16, const ProductArgs& a, bool after_quantize, cudaStream_t st) {
  using S = Stream<NT>;
  auto kern = w8_stream_kernel<NT, BF16, RESID>;
  GLT_TRY(ensure_smem_attr(reinterpret_cast<const void*>(kern), S::kSmem));
  CUtensorMap map_w, map_x;
  GLT_TRY(make_tmap_bf16(&map_w, w.p, K16 / 2, a.N, w.ld / 2, kChannels));
  GLT_TRY(make_tmap_bf16(&map_x, x.p, K16 / 2, a.M, x.ld / 2, NT));
  unsigned int* err = device_error_word();
  if (!err) return fail(GLT_ECUDA, "device error word unavailable");
  const int blocks = (K16 + 127) / 128;
  const int rows = (a.N + kChannels - 1) / kChannels, cols = (a.M + NT - 1) / NT;
  // K is shared so that all CTAs are resident at once, each with four blocks of it at least.  (Clusters of 6
  // for 48 tiles took 21.2 us with 64 tokens where 4 take 12.6.)
  int shares = kMaxShares;
  while (shares > 1 && (static_cast<int64_t>(rows) * cols * shares > static_cast<int64_t>(num_sms()) * S::kCtasPerSm || shares > blocks / 4))
    shares /= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * shares, cols);
  cfg.blockDim = dim3(kStreamThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = shares;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_quantize ? 2 : 1;
  GLT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, map_w, map_x, blocks, shares, a, err));
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

template <bool BF16, bool RESID>
int product(const Codes& w, const Codes& x, int K16, const ProductArgs& a, bool after_quantize, cudaStream_t st) {
  if (a.M <= 16) return launch_stream<16, BF16, RESID>(w, x, K16, a, after_quantize, st);
  if (a.M <= 32) return launch_stream<32, BF16, RESID>(w, x, K16, a, after_quantize, st);
  // more tokens go 64 at a time while all tiles are resident at once
  const int64_t tiles = static_cast<int64_t>((a.N + kChannels - 1) / kChannels) * ((a.M + 63) / 64);
  if (tiles <= 2 * num_sms()) return launch_stream<64, BF16, RESID>(w, x, K16, a, after_quantize, st);
  // 16 tiles of 256 channels a raster group: the group's weights stay in L2 while all tokens pass
  return launch_gemm_pair<false, false, tc::PairS8>({w.p, w.ld / 2, false}, {x.p, x.ld / 2, false}, a.N, a.M, K16 / 2,
                                                    EpiW8<BF16, RESID>{a}, st, 1, nullptr, INT_MAX, 16, nullptr, 0, nullptr,
                                                    tc::GLT_MBAR_TIMEOUT_NS);
}

int product(const Codes& w, const Codes& x, int K16, const ProductArgs& a, int y_dtype, bool after_quantize, cudaStream_t st) {
  if (a.resid)
    return y_dtype ? product<true, true>(w, x, K16, a, after_quantize, st) : product<false, true>(w, x, K16, a, after_quantize, st);
  return y_dtype ? product<true, false>(w, x, K16, a, after_quantize, st) : product<false, false>(w, x, K16, a, after_quantize, st);
}

int round16(int k) { return (k + 15) / 16 * 16; }
// 131071 products of two bytes stay within 32 bits
constexpr int kMaxK = 131071;
constexpr int kMaxRows = INT_MAX - 255;   // rounded up to tiles they are 32-bit numbers still

int check_sizes(int M, int N, int K) {
  if (M < 0 || M > kMaxRows || N < 1 || N > kMaxRows || K < 1 || K > kMaxK)
    return fail(GLT_EINVAL, "w8: sizes M %d, N %d (at most %d), K %d (at most %d)", M, N, kMaxRows, K, kMaxK);
  return GLT_OK;
}
int check_codes(const int8_t* p, int64_t ld, int K, const char* what) {
  if (!p || !aligned16(p) || ld % 16 || ld < round16(K))
    return fail(GLT_EINVAL, "w8: %s must be 16-byte aligned with a row stride that is a multiple of 16 and at least %d", what, round16(K));
  return GLT_OK;
}
int check_out(const void* y, int64_t ld_y, int y_dtype, const uint16_t* resid, int64_t ld_r, int N) {
  if (!y || ld_y < N || (resid && ld_r < N)) return fail(GLT_EINVAL, "w8: y (and resid) need rows of %d", N);
  if (y_dtype != 0 && y_dtype != 1) return fail(GLT_EINVAL, "w8: y_dtype %d (0 fp32, 1 bf16)", y_dtype);
  return GLT_OK;
}
int64_t codes_bytes(int M, int K) { return (static_cast<int64_t>(M) * round16(K) + 255) / 256 * 256; }

}  // namespace
}  // namespace glt

extern "C" int glt_w8_quantize_rows(const uint16_t* x, int64_t ld_x, int rows, int K, const uint16_t* norm, float eps,
                                    int8_t* codes, int64_t ld_codes, float* scales, void* stream) {
  GLT_TRY(glt::check_sizes(rows, 1, K));
  if (rows == 0) return GLT_OK;
  GLT_TRY(glt::check_codes(codes, ld_codes, K, "codes"));
  if (!x || !scales || ld_x < K) return glt::fail(GLT_EINVAL, "w8: null argument, or rows of x closer than %d", K);
  if (norm && !(eps >= 0.f && eps <= FLT_MAX)) return glt::fail(GLT_EINVAL, "w8: eps must be finite and not negative");
  return glt::quantize({x, ld_x, rows, K, norm, eps, codes, ld_codes, scales}, static_cast<cudaStream_t>(stream));
}

extern "C" int glt_w8_linear_rows(const int8_t* codes, int64_t ld_codes, const float* scales, int M, const int8_t* w,
                                  int64_t ld_w, const float* w_scales, int N, int K, void* y, int64_t ld_y, int y_dtype,
                                  const uint16_t* resid, int64_t ld_r, void* stream) {
  GLT_TRY(glt::check_sizes(M, N, K));
  if (M == 0) return GLT_OK;
  GLT_TRY(glt::check_codes(codes, ld_codes, K, "codes"));
  GLT_TRY(glt::check_codes(w, ld_w, K, "w"));
  GLT_TRY(glt::check_out(y, ld_y, y_dtype, resid, ld_r, N));
  if (!scales || !w_scales) return glt::fail(GLT_EINVAL, "null argument");
  const glt::ProductArgs a = {scales, w_scales, y, ld_y, resid, ld_r, M, N};
  return glt::product({w, ld_w}, {codes, ld_codes}, glt::round16(K), a, y_dtype, false, static_cast<cudaStream_t>(stream));
}

extern "C" int glt_w8_linear_workspace(int M, int K, int64_t* bytes) {
  if (!bytes) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_sizes(M, 1, K));
  *bytes = glt::codes_bytes(M, K) + 4ll * M;
  return GLT_OK;
}

extern "C" int glt_w8_linear(const uint16_t* x, int64_t ld_x, int M, const uint16_t* norm, float eps, const int8_t* w,
                             int64_t ld_w, const float* w_scales, int N, int K, void* y, int64_t ld_y, int y_dtype,
                             const uint16_t* resid, int64_t ld_r, void* workspace, int64_t workspace_bytes, void* stream) {
  GLT_TRY(glt::check_sizes(M, N, K));
  if (M == 0) return GLT_OK;
  GLT_TRY(glt::check_codes(w, ld_w, K, "w"));
  GLT_TRY(glt::check_out(y, ld_y, y_dtype, resid, ld_r, N));
  if (!w_scales) return glt::fail(GLT_EINVAL, "null argument");
  const int64_t codes_bytes = glt::codes_bytes(M, K);
  if (!workspace || !glt::aligned16(workspace) || workspace_bytes < codes_bytes + 4ll * M)
    return glt::fail(GLT_EINVAL, "w8: workspace must be 16-byte aligned and hold %lld bytes", (long long)(codes_bytes + 4ll * M));
  int8_t* codes = static_cast<int8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(codes + codes_bytes);
  const int K16 = glt::round16(K);
  GLT_TRY(glt_w8_quantize_rows(x, ld_x, M, K, norm, eps, codes, K16, scales, stream));
  const glt::ProductArgs a = {scales, w_scales, y, ld_y, resid, ld_r, M, N};
  return glt::product({w, ld_w}, {codes, K16}, K16, a, y_dtype, true, static_cast<cudaStream_t>(stream));
}
