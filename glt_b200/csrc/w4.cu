// Products with 4-bit weights and group scales (glt_w4_*).
//
// Packed layout of W [N, K]: rows in tiles of 16, columns in chunks of 64 (the last
// ones filled up with zero scales).  A chunk of a tile is 128 words of eight codes,
// in the order the A fragments of mma.m16n8k16 want them: lane 4g + c of a warp owns
// words 4 * lane + s, s = 0..3, and word s holds, for the k-step s of the chunk, rows
// g and g + 8 at columns col(c, s, 0..3) = (s / 2) * 32 + c * 8 + (s % 2) * 4 + 0..3.
// So a warp reads a chunk as one 16-byte load a lane, 512 contiguous bytes, and each
// 32-column half of the chunk (the smallest group) is two whole k-steps.
// Register i of the fragment (row half i % 2, column pair i / 2) takes its two codes
// from bits 4i + 3 .. 4i + 6 and 16 further up (modulo 32): a rotation by 4i brings
// them to mantissa bits 3..6 of two bf16 numbers 1 + code / 16, exactly.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "gemm.cuh"

namespace cg = cooperative_groups;

namespace glt {
namespace {

__host__ __device__ inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// Offsets of the three parts of a packed matrix.
struct W4Layout {
  int N, K, group, asym;
  int tiles, chunks, groups;  // groups: of the filled-up columns
  int64_t scale_off, zero_off, bytes;
  W4Layout(int N_, int K_, int group_, int asym_) : N(N_), K(K_), group(group_), asym(asym_) {
    tiles = (N + 15) / 16;
    chunks = (K + 63) / 64;
    groups = static_cast<int>(up(static_cast<int64_t>(chunks) * 64, group) / group);
    scale_off = up(static_cast<int64_t>(tiles) * chunks * 512, 256);
    // [tile][group][g][row half] bf16, then the zeros as bf16 1 + zero / 16 in the same order
    zero_off = up(scale_off + static_cast<int64_t>(tiles) * groups * 32, 256);
    bytes = zero_off + (asym ? up(static_cast<int64_t>(tiles) * groups * 32, 256) : 0);
  }
};

int check_shape(int N, int K, int group) {
  if (group != 32 && group != 64 && group != 128) return fail(GLT_EINVAL, "w4: group %d (32, 64 or 128)", group);
  if (N < 1 || K < 1 || K % group) return fail(GLT_EINVAL, "w4: N %d, K %d (a positive multiple of the group %d)", N, K, group);
  return GLT_OK;
}

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) < INFINITY ? x : 0.f; }

// One warp a group: the group's largest magnitude (or range), then its codes.
__global__ void __launch_bounds__(256) w4_quantize_kernel(const uint16_t* __restrict__ w, int64_t ld, int N,
                                                          int K, int group, int asym, uint8_t* __restrict__ codes,
                                                          uint16_t* __restrict__ scales, uint8_t* __restrict__ zeros) {
  const int lane = threadIdx.x & 31;
  const int ng = K / group;
  const int64_t total = static_cast<int64_t>(N) * ng;
  for (int64_t u = blockIdx.x * 8ll + (threadIdx.x >> 5); u < total; u += gridDim.x * 8ll) {
    const int64_t n = u / ng;
    const int k0 = static_cast<int>(u - n * ng) * group;
    float x[4];
    float lo = 0.f, hi = 0.f;
    for (int j = 0; j < group / 32; ++j) {
      x[j] = bf16_bits_to_f32(w[n * ld + k0 + j * 32 + lane]);
      const float f = finite_or_zero(x[j]);
      lo = fminf(lo, f);
      hi = fmaxf(hi, f);
    }
    lo = -warp_max(-lo);
    hi = warp_max(hi);
    const uint16_t sb = bf16_bits_rn(asym ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f);
    const float s = bf16_bits_to_f32(sb);
    const float z = !asym ? 8.f : s > 0.f ? fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0.f;
    if (lane == 0) {
      scales[u] = sb;
      if (asym) zeros[u] = static_cast<uint8_t>(z);
    }
    for (int j = 0; j < group / 32; ++j) {
      // a NaN (or a group of zeros) takes the code of 0
      const float q = s > 0.f && x[j] == x[j] ? rintf(x[j] / s) : 0.f;
      codes[n * K + k0 + j * 32 + lane] = static_cast<uint8_t>(fminf(fmaxf(q + z, 0.f), 15.f));
    }
  }
}

__device__ __forceinline__ int chunk_col(int c, int s, int e) { return (s >> 1) * 32 + c * 8 + (s & 1) * 4 + e; }
__device__ __forceinline__ int code_bit(int i, int h) { return (3 + 16 * h + 4 * i) & 31; }

__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* __restrict__ codes,
                                                      const uint16_t* __restrict__ scales,
                                                      const uint8_t* __restrict__ zeros, W4Layout L,
                                                      uint8_t* __restrict__ packed) {
  const int ng = L.K / L.group;
  const int64_t words = static_cast<int64_t>(L.tiles) * L.chunks * 128;
  const int64_t scs = static_cast<int64_t>(L.tiles) * L.groups * 16;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t first = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  for (int64_t q = first; q < words; q += step) {
    const int s = q & 3, lane = (q >> 2) & 31;
    const int64_t tc = q >> 7;
    const int64_t tile = tc / L.chunks;
    const int chunk = static_cast<int>(tc - tile * L.chunks);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t n = tile * 16 + (lane >> 2) + 8 * (i & 1);
        const int k = chunk * 64 + chunk_col(lane & 3, s, 2 * (i >> 1) + h);
        const uint32_t u = n < L.N && k < L.K ? codes[n * L.K + k] & 15u : 0u;
        const int b = code_bit(i, h);
        word |= b <= 28 ? u << b : (u << b) | (u >> (32 - b));
      }
    reinterpret_cast<uint32_t*>(packed)[q] = word;
  }
  for (int64_t q = first; q < scs; q += step) {
    const int64_t tg = q >> 4;
    const int64_t tile = tg / L.groups;
    const int grp = static_cast<int>(tg - tile * L.groups);
    const int64_t n = tile * 16 + ((q >> 1) & 7) + 8 * (q & 1);
    const bool in = n < L.N && grp < ng;
    reinterpret_cast<uint16_t*>(packed + L.scale_off)[q] = in ? scales[n * ng + grp] : 0;
    if (L.asym)
      reinterpret_cast<uint16_t*>(packed + L.zero_off)[q] = 0x3F80u | (in ? (zeros[n * ng + grp] & 15u) << 3 : 0u);
  }
}

__global__ void __launch_bounds__(256) w4_unpack_kernel(const uint8_t* __restrict__ packed, W4Layout L,
                                                        uint16_t* __restrict__ w, int64_t ld) {
  const int64_t total = static_cast<int64_t>(L.N) * L.K;
  for (int64_t q = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; q < total;
       q += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t n = q / L.K;
    const int k = static_cast<int>(q - n * L.K);
    const int r = n & 15, kk = k & 63;
    const int s = (kk >> 5) * 2 + ((kk >> 2) & 1), c = (kk >> 3) & 3, e = kk & 3;
    const int64_t word = (((n >> 4) * L.chunks + (k >> 6)) * 32 + (r & 7) * 4 + c) * 4 + s;
    const int b = code_bit((r >> 3) + 2 * (e >> 1), e & 1);
    const uint32_t v = reinterpret_cast<const uint32_t*>(packed)[word];
    const float u = static_cast<float>(__funnelshift_r(v, v, b) & 15u);
    const int64_t sc = ((n >> 4) * L.groups + k / L.group) * 16 + (r & 7) * 2 + (r >> 3);
    const float z = L.asym ? static_cast<float>((reinterpret_cast<const uint16_t*>(packed + L.zero_off)[sc] >> 3) & 15u) : 8.f;
    w[n * ld + k] = bf16_bits_rn((u - z) * bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(packed + L.scale_off)[sc]));
  }
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from other sums.
__device__ __forceinline__ void mma_bf16_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                              float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

struct LinearArgs {
  const uint8_t* packed;
  W4Layout L;
  const uint16_t* x;
  int64_t ld_x;
  int M;
  void* y;
  int64_t ld_y;
  int y_bf16;
  const uint16_t* resid;
  int64_t ld_r;
};

constexpr int kLinWarps = 4;
constexpr int kLinThreads = 32 * kLinWarps;

// y = x . W^T for up to 8 NT rows of x: the weights are operand A (16 rows by 16 columns),
// the rows of x operand B (N = 8).  A cluster of S CTAs takes 16 TILES rows of W; its CTAs
// split the columns, and a CTA's warps take the pieces of its part in turn, TILES tiles at
// once so that a fragment of x serves them all.  A piece is a chunk, or two with groups of
// 128, so that a group's sums meet its scale once.  Partial sums meet in shared memory, then
// over the cluster, in a fixed order.
//
// Half a byte a weight leaves about 22 cycles of an SM for a tile's chunk, so instructions
// count.  A register of two weights takes a rotation (three in four) and one AND-OR to become
// 1 + code / 16.  Taking 1 + zero / 16 off costs one more; with the constant zero 8 it is left
// to the tensor core: a product with -1.5 everywhere gives -1.5 sum x, from which the sums of
// every tile start.  (Then |x| counts 1.5 to 1.94 times in 32-bit sums instead of about 0.25
// times.)  Infinities would not survive that, so a piece of x whose sum is not finite goes
// the exact way.
template <int NT, int TILES, bool ASYM, int GROUP>
__global__ void __launch_bounds__(kLinThreads) w4_linear_kernel(const __grid_constant__ LinearArgs a) {
  constexpr int kSub = GROUP == 128 ? 2 : 1;                    // chunks of a piece
  constexpr int kGroups = GROUP == 32 ? 2 : 1;                  // groups of a piece
  constexpr int kAhead = NT == 1 ? 4 / kSub : NT == 2 ? 2 : 1;  // pieces on their way
  constexpr int kRows = 16 * TILES, kCols = 8 * NT, kOut = kRows * kCols;
  extern __shared__ float red[];   // [warp][column][row], then the CTA's sums
  cg::cluster_group cluster = cg::this_cluster();
  const int S = cluster.num_blocks(), rank = cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const W4Layout& L = a.L;
  const int tile0 = static_cast<int>(blockIdx.x / S) * TILES;
  const int m0 = blockIdx.y * kCols;
  const int pieces = L.chunks / kSub;   // K is a multiple of the group
  const int p0 = static_cast<int>(static_cast<int64_t>(pieces) * rank / S);
  const int p1 = static_cast<int>(static_cast<int64_t>(pieces) * (rank + 1) / S);

  // A warp's pieces are p0 + warp + kLinWarps j; from j to j + 1 everything it reads moves on
  // by a fixed number of bytes.  Tiles past the last one repeat it, rows of x past the last one
  // the first: nothing of theirs is written.
  const int first = p0 + warp;
  const int steps = first < p1 ? (p1 - first + kLinWarps - 1) / kLinWarps : 0;
  const uint4* cw[TILES];
  const uint32_t *sw[TILES], *zw[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int64_t tile = min(tile0 + t, L.tiles - 1);
    const int64_t grp = (tile * L.groups + first * kGroups) * 8 + g;
    cw[t] = reinterpret_cast<const uint4*>(a.packed) + (tile * L.chunks + first * kSub) * 32 + lane;
    sw[t] = reinterpret_cast<const uint32_t*>(a.packed + L.scale_off) + grp;
    zw[t] = reinterpret_cast<const uint32_t*>(a.packed + L.zero_off) + grp;
  }
  const uint16_t* xr[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    xr[n] = a.x + (m0 + n * 8 + g < a.M ? m0 + n * 8 + g : 0) * a.ld_x + static_cast<int64_t>(first) * kSub * 64 + c * 8;

  struct Piece {
    uint4 w[TILES][kSub];
    uint32_t sc[TILES][kGroups], z[TILES][kGroups];
    uint4 x[NT][2 * kSub];
  };
  Piece ahead[kAhead];
  // Loads the piece `d` steps on from where the pointers stand; half: only 32 of its 64 columns
  // exist (the last of a K that is an odd multiple of 32).
  auto load = [&](Piece& k, int d, bool half) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
#pragma unroll
      for (int i = 0; i < kSub; ++i) k.w[t][i] = __ldcs(cw[t] + (d * kLinWarps * kSub + i) * 32);
#pragma unroll
      for (int h = 0; h < kGroups; ++h) {
        k.sc[t][h] = sw[t][(d * kLinWarps * kGroups + h) * 8];
        if (ASYM) k.z[t][h] = zw[t][(d * kLinWarps * kGroups + h) * 8];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2 * kSub; ++h) {
        if (GROUP == 32 && h == 1 && half)
          k.x[n][h] = make_uint4(0, 0, 0, 0);
        else
          k.x[n][h] = *reinterpret_cast<const uint4*>(xr[n] + d * kLinWarps * kSub * 64 + h * 32);
      }
  };
  const int odd_step = GROUP == 32 && (L.K & 32) && p1 == pieces && steps > 0 && first + (steps - 1) * kLinWarps == pieces - 1
                           ? steps - 1 : -1;

  float acc[TILES][NT][4] = {};
  // The k-steps of a group: `start` what its sums begin with, SUB whether zeros are taken off.
  auto group_of = [&](const Piece& k, int h, const float (&start)[NT][2], auto sub) {
    constexpr int kSteps = GROUP / 16;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      float part[NT][4];
      uint32_t z0 = 0x3FC03FC0u, z1 = 0x3FC03FC0u;
      if (ASYM) {
        z0 = __byte_perm(k.z[t][h], 0, 0x1010);
        z1 = __byte_perm(k.z[t][h], 0, 0x3232);
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int s = h * kSteps + i;   // k-step of the piece
        const uint4& wv = k.w[t][s >> 2];
        const uint32_t word = (s & 3) == 0 ? wv.x : (s & 3) == 1 ? wv.y : (s & 3) == 2 ? wv.z : wv.w;
        uint32_t f[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f[r] = (__funnelshift_r(word, word, 4 * r) & 0x00780078u) | 0x3F803F80u;
          if (decltype(sub)::value) f[r] = sub_bf16x2(f[r], (r & 1) ? z1 : z0);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4& x = k.x[n][s >> 1];
          const uint32_t b0 = s & 1 ? x.z : x.x, b1 = s & 1 ? x.w : x.y;
          if (i == 0)
            mma_bf16_from(part[n], f, b0, b1, start[n][0], start[n][1], start[n][0], start[n][1]);
          else
            mma_bf16(part[n], f, b0, b1);
        }
      }
      const float s0 = bf16_lo(k.sc[t][h]), s1 = bf16_hi(k.sc[t][h]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[t][n][0] = fmaf(s0, part[n][0], acc[t][n][0]);
        acc[t][n][1] = fmaf(s0, part[n][1], acc[t][n][1]);
        acc[t][n][2] = fmaf(s1, part[n][2], acc[t][n][2]);
        acc[t][n][3] = fmaf(s1, part[n][3], acc[t][n][3]);
      }
    }
  };
  auto use = [&](const Piece& k) {
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      float start[NT][2] = {};
      bool exact = ASYM;
      if (!ASYM) {
        const uint32_t minus[4] = {0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u};   // -1.5
        float sum[NT][4];
#pragma unroll
        for (int i = 0; i < GROUP / 16; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int s = h * (GROUP / 16) + i;
            const uint4& x = k.x[n][s >> 1];
            const uint32_t b0 = s & 1 ? x.z : x.x, b1 = s & 1 ? x.w : x.y;
            if (i == 0)
              mma_bf16_from(sum[n], minus, b0, b1, 0.f, 0.f, 0.f, 0.f);
            else
              mma_bf16(sum[n], minus, b0, b1);
          }
        float big = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          start[n][0] = sum[n][0];
          start[n][1] = sum[n][1];
          big = fmaf(sum[n][0], 0.f, fmaf(sum[n][1], 0.f, big));   // 0, or NaN
        }
        exact = __any_sync(0xffffffffu, big != 0.f);
      }
      if (exact) {
        const float none[NT][2] = {};
        group_of(k, h, none, std::true_type());
      } else {
        group_of(k, h, start, std::false_type());
      }
    }
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d)
    if (d < steps) load(ahead[d], d, d == odd_step);
  for (int j = 0; j < steps; j += kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      if (j + d < steps) {
        use(ahead[d]);
        if (j + d + kAhead < steps) load(ahead[d], d + kAhead, j + d + kAhead == odd_step);
      }
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      cw[t] += kAhead * kLinWarps * kSub * 32;
      sw[t] += kAhead * kLinWarps * kGroups * 8;
      if (ASYM) zw[t] += kAhead * kLinWarps * kGroups * 8;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) xr[n] += kAhead * kLinWarps * kSub * 64;
  }

  // ---- join the warps, then the cluster
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        red[warp * kOut + (n * 8 + 2 * c + (q & 1)) * kRows + t * 16 + g + 8 * (q >> 1)] = acc[t][n][q];
  __syncthreads();
  for (int e = threadIdx.x; e < kOut; e += kLinThreads)
    red[e] = (red[e] + red[kOut + e]) + (red[2 * kOut + e] + red[3 * kOut + e]);
  if (S > 1)
    cluster.sync();
  else
    __syncthreads();
  const int e0 = kOut * rank / S, e1 = kOut * (rank + 1) / S;
  for (int e = e0 + threadIdx.x; e < e1; e += kLinThreads) {
    const int m = m0 + e / kRows;
    const int64_t n = static_cast<int64_t>(tile0) * 16 + e % kRows;
    float o = 0.f;
    for (int r = 0; r < S; ++r) o += S > 1 ? cluster.map_shared_rank(red, r)[e] : red[e];
    if (m >= a.M || n >= L.N) continue;
    o *= 16.f;   // the products are of code / 16
    if (a.resid) o += bf16_bits_to_f32(a.resid[m * a.ld_r + n]);
    if (a.y_bf16)
      static_cast<uint16_t*>(a.y)[m * a.ld_y + n] = bf16_bits_rn(o);
    else
      static_cast<float*>(a.y)[m * a.ld_y + n] = o;
  }
  if (S > 1) cluster.sync();   // the others have read this CTA's sums
}

template <int NT, int TILES, bool ASYM, int GROUP>
int launch_linear(const LinearArgs& a, cudaStream_t st) {
  const auto kernel = w4_linear_kernel<NT, TILES, ASYM, GROUP>;
  constexpr int bytes = kLinWarps * 16 * TILES * 8 * NT * 4;
  const int groups = (a.L.tiles + TILES - 1) / TILES, blocks = (a.M + 8 * NT - 1) / (8 * NT);
  // CTAs a group of tiles: until the SMs hold six each, while every warp keeps two chunks
  int S = 1;
  while (S < 8 && static_cast<int64_t>(groups) * blocks * S < 6ll * num_sms() && a.L.chunks >= 4 * S * kLinWarps) S *= 2;
  if (blocks > 65535) return fail(GLT_EINVAL, "w4: %d rows", a.M);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups) * S, blocks);
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  GLT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

template <int NT, int TILES>
int launch_linear_as(const LinearArgs& a, cudaStream_t st) {
  if (a.L.asym) {
    if (a.L.group == 32) return launch_linear<NT, TILES, true, 32>(a, st);
    return a.L.group == 64 ? launch_linear<NT, TILES, true, 64>(a, st) : launch_linear<NT, TILES, true, 128>(a, st);
  }
  if (a.L.group == 32) return launch_linear<NT, TILES, false, 32>(a, st);
  return a.L.group == 64 ? launch_linear<NT, TILES, false, 64>(a, st) : launch_linear<NT, TILES, false, 128>(a, st);
}

int grid_for(int64_t units, int per_cta) {
  const int64_t b = (units + per_cta - 1) / per_cta, cap = static_cast<int64_t>(num_sms()) * 16;
  return static_cast<int>(b < 1 ? 1 : b < cap ? b : cap);
}

}  // namespace
}  // namespace glt

using glt::W4Layout;

extern "C" int glt_w4_packed_bytes(int N, int K, int group, int asym, int64_t* bytes) {
  if (!bytes) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_shape(N, K, group));
  *bytes = W4Layout(N, K, group, asym).bytes;
  return GLT_OK;
}

extern "C" int glt_w4_quantize(const uint16_t* w, int64_t ld_w, int N, int K, int group, int asym,
                               uint8_t* codes, uint16_t* scales, uint8_t* zeros, void* stream) {
  if (!w || !codes || !scales || (asym && !zeros)) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_shape(N, K, group));
  if (ld_w < K) return glt::fail(GLT_EINVAL, "w4: row stride %lld below K %d", (long long)ld_w, K);
  const int64_t units = static_cast<int64_t>(N) * (K / group);
  glt::w4_quantize_kernel<<<glt::grid_for(units, 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      w, ld_w, N, K, group, asym, codes, scales, zeros);
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

extern "C" int glt_w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int N,
                           int K, int group, void* packed, void* stream) {
  if (!codes || !scales || !packed) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_shape(N, K, group));
  if (!glt::aligned16(packed)) return glt::fail(GLT_EINVAL, "w4: packed weights must be 16-byte aligned");
  const W4Layout L(N, K, group, zeros != nullptr);
  glt::w4_pack_kernel<<<glt::grid_for(static_cast<int64_t>(L.tiles) * L.chunks * 128, 256), 256, 0,
                        static_cast<cudaStream_t>(stream)>>>(codes, scales, zeros, L, static_cast<uint8_t*>(packed));
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

extern "C" int glt_w4_unpack(const void* packed, int N, int K, int group, int asym, uint16_t* w,
                             int64_t ld_w, void* stream) {
  if (!packed || !w) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_shape(N, K, group));
  if (ld_w < K) return glt::fail(GLT_EINVAL, "w4: row stride %lld below K %d", (long long)ld_w, K);
  if (!glt::aligned16(packed)) return glt::fail(GLT_EINVAL, "w4: packed weights must be 16-byte aligned");
  glt::w4_unpack_kernel<<<glt::grid_for(static_cast<int64_t>(N) * K, 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(packed), W4Layout(N, K, group, asym), w, ld_w);
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

extern "C" int glt_w4_linear(const void* packed, int N, int K, int group, int asym, const uint16_t* x,
                             int64_t ld_x, int M, void* y, int64_t ld_y, int y_dtype,
                             const uint16_t* resid, int64_t ld_r, void* stream) {
  GLT_TRY(glt::check_shape(N, K, group));
  if (!packed || (M > 0 && (!x || !y))) return glt::fail(GLT_EINVAL, "null argument");
  if (M < 0) return glt::fail(GLT_EINVAL, "w4: negative rows");
  if (y_dtype != 0 && y_dtype != 1) return glt::fail(GLT_EINVAL, "w4: output type %d (0 fp32, 1 bf16)", y_dtype);
  if (ld_x < K || ld_x % 8 || !glt::aligned16(x))
    return glt::fail(GLT_EINVAL, "w4: x needs 16-byte aligned rows (row stride a multiple of 8, at least K)");
  if (ld_y < N || (resid && ld_r < N)) return glt::fail(GLT_EINVAL, "w4: output or residual row stride below N %d", N);
  if (!glt::aligned16(packed)) return glt::fail(GLT_EINVAL, "w4: packed weights must be 16-byte aligned");
  if (M == 0) return GLT_OK;
  const glt::LinearArgs a{static_cast<const uint8_t*>(packed), W4Layout(N, K, group, asym), x, ld_x, M, y, ld_y,
                          y_dtype, resid, ld_r};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (M <= 8) return glt::launch_linear_as<1, 2>(a, st);
  if (M <= 16) return glt::launch_linear_as<2, 2>(a, st);
  if (M <= 24) return glt::launch_linear_as<3, 2>(a, st);
  return glt::launch_linear_as<4, 2>(a, st);
}
