// Products with 4-bit weights and group scales (glt_w4_*).
//
// Packed layout of W [N, K]: rows in tiles of 16, columns in blocks of 128 (the last
// one filled up with zero scales).  A block of a tile is one record, a tile's records follow
// one another.  A record: two chunks of 64 columns, 128 words of eight codes each, then the
// scales of the block's groups, [group][g][row half] bf16, then with asym 15 - zero alike, as bytes
// of a 32-bit word (row g, row g + 8, 0, 0).
// Lane 4g + c of a warp owns words 4 * lane + s, s = 0..3, of a chunk; byte b of word s holds
// the codes of row g (low nibble) and row g + 8 (high nibble) at column
// (s / 2) * 32 + 8 c + (s % 2) * 4 + b.  So one AND (and a shift) makes four codes a register
// of operand A of mma.m16n8k32 on bytes, and a word is operand A of mma.m16n8k16 on f16, columns
// b = 0, 2 and b = 1, 3 side by side.
#include <math.h>

#include <climits>
#include <type_traits>

#include "common.cuh"
#include "gemm.cuh"

namespace glt {
namespace {

struct W4Layout {
  int N, K, group, asym;
  int tiles, blocks;
  int per_block;   // groups of a block
  int record;      // bytes
  int64_t bytes;
  W4Layout(int N_, int K_, int group_, int asym_) : N(N_), K(K_), group(group_), asym(asym_ != 0) {
    tiles = (N + 15) / 16;
    blocks = (K + 127) / 128;
    per_block = 128 / group;
    record = 1024 + per_block * 32 * (1 + asym);
    bytes = static_cast<int64_t>(tiles) * blocks * record;
  }
};

// a / b by the much shorter 32-bit division where that is enough.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

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
    float step = asym ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f;
    if (!(step < INFINITY)) step = hi / 15.f - lo / 15.f;   // the range is beyond a float, a step of it is not
    const uint16_t sb = bf16_bits_rn(step);
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

__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* __restrict__ codes,
                                                      const uint16_t* __restrict__ scales,
                                                      const uint8_t* __restrict__ zeros, W4Layout L,
                                                      uint8_t* __restrict__ packed) {
  const int ng = L.K / L.group, words = L.record / 4;
  const int64_t total = static_cast<int64_t>(L.tiles) * L.blocks * words;
  for (int64_t q = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; q < total;
       q += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t rec = q / words;
    const int i = static_cast<int>(q - rec * words);
    const int64_t tile = rec / L.blocks;
    const int block = static_cast<int>(rec - tile * L.blocks);
    uint32_t word = 0;
    if (i < 256) {
      const int s = i & 3, lane = (i >> 2) & 31;
#pragma unroll
      for (int e = 0; e < 8; ++e) {   // nibble e: byte e / 2, row half e % 2
        const int64_t n = tile * 16 + (lane >> 2) + 8 * (e & 1);
        const int k = block * 128 + (i >> 7) * 64 + (s >> 1) * 32 + (lane & 3) * 8 + (s & 1) * 4 + (e >> 1);
        word |= (n < L.N && k < L.K ? codes[n * L.K + k] & 15u : 0u) << (4 * e);
      }
    } else {
      const int j = (i - 256) % (L.per_block * 8);
      const bool zero = i - 256 >= L.per_block * 8;
      const int grp = block * L.per_block + (j >> 3);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t n = tile * 16 + (j & 7) + 8 * e;
        if (n >= L.N || grp >= ng) continue;
        word |= zero ? (15u - (zeros[n * ng + grp] & 15u)) << (8 * e) : static_cast<uint32_t>(scales[n * ng + grp]) << (16 * e);
      }
    }
    reinterpret_cast<uint32_t*>(packed)[q] = word;
  }
}

// code - zero and scale of one weight.
__device__ __forceinline__ float w4_code(const uint8_t* packed, const W4Layout& L, int64_t n, int k, float* scale) {
  const uint8_t* rec = packed + ((n >> 4) * L.blocks + (k >> 7)) * L.record;
  const int r = n & 15, kk = k & 63;
  const int s = (kk >> 5) * 2 + ((kk >> 2) & 1), c = (kk >> 3) & 3;
  const int word = ((k >> 6) & 1) * 128 + ((r & 7) * 4 + c) * 4 + s;
  const uint32_t u = reinterpret_cast<const uint32_t*>(rec)[word] >> (8 * (kk & 3) + 4 * (r >> 3)) & 15u;
  const uint16_t* sc = reinterpret_cast<const uint16_t*>(rec + 1024) + ((k & 127) / L.group) * 16 + (r & 7) * 2 + (r >> 3);
  *scale = bf16_bits_to_f32(sc[0]);
  const int zero = L.asym ? 15 - rec[1024 + L.per_block * 32 + ((k & 127) / L.group) * 32 + (r & 7) * 4 + (r >> 3)] : 8;
  return static_cast<float>(static_cast<int>(u) - zero);
}

__global__ void __launch_bounds__(256) w4_unpack_kernel(const uint8_t* __restrict__ packed, W4Layout L,
                                                        uint16_t* __restrict__ w, int64_t ld) {
  const int64_t total = static_cast<int64_t>(L.N) * L.K;
  for (int64_t q = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; q < total;
       q += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t n = q / L.K;
    const int k = static_cast<int>(q - n * L.K);
    float scale;
    const float u = w4_code(packed, L, n, k, &scale);
    w[n * ld + k] = bf16_bits_rn(u * scale);
  }
}

__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
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
// Both halves of a register as f16 numbers.
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// 2^n for -149 <= n <= 127.
__device__ __forceinline__ float power_of_two(int n) { return __int_as_float(n >= -126 ? (n + 127) << 23 : 1 << (n + 149)); }

// ---- operand B: the image of x.  Within a block of 128 columns a row of x is multiplied by a power of two,
// 2^a, that its largest magnitude chooses, and held in one of two forms.  Both keep every bf16 number down to
// 2^-22 of that magnitude exactly, and round off only what lies below 2^-30 of it: outliers a million times
// the other columns cost these nothing, also where an outlier's own weight is 0.
//
// HALF: one f16 number a value, the largest in [2^15, 2^16): 8 rows of x are a tile of N = 8 columns.  Codes
// less their zero are f16 too, exactly; products are exact and sums in 32 bits.
//
// Bytes: fixed-point numbers v = round(x 2^a), the largest in [2^30, 2^31), as four signed bytes, a column of
// operand B each: 2 rows are a tile.  Products with the codes are exact integers until a group's end.
//
// Which.  A matrix instruction of bytes takes twice the columns of one of f16 at the same cost, and eight codes
// need three instructions where f16 needs nine; but a row takes four columns, and a group's end six instructions
// for two rows of W where f16 takes two.  So bytes for up to 4 rows, with groups of 32 for up to 2 (28672 x 4096,
// us, bytes and f16: groups of 128, 1 row 14.8 and 18.6, 4 rows 18.3 and 20.8; of 32, 1 row 16.7 and 19.8,
// 4 rows 23.8 and 22.4).
//
// Image: [chunk of 64][tile of rows] with, for bytes, [lane][16 bytes], high byte first, and for f16
// [half][lane][16 bytes]; lane 4g + c holds column g at the k of operand A's lanes c.
constexpr int kPrepThreads = 256;
constexpr int kMagic = 0x4B400000;   // 1.5 2^23 as a float: kMagic + i is the float 1.5 2^23 + i
// Bytes: what lane c needs at the ends of a group: what its two columns' sums begin with, kMagic - 8 (asym: 15)
// times the sum of the bytes, and 2^-a of its row's block.  (f16: two factors 2^-a a lane and block.)
// A factor is NaN where the block holds something that is not finite; such a row's products are then done the
// plain way.
struct __align__(16) GroupNote {
  int start[2];
  float factor;
  int pad;
};
template <bool HALF>
struct XImage {
  static constexpr int kRows = HALF ? 8 : 2;          // a tile's
  static constexpr int kChunk = HALF ? 1024 : 512;    // bytes of a tile's chunk,
  static constexpr int kNote = HALF ? 32 : 64;        // of its notes
  int per_cta;   // tiles of rows of x that a CTA takes
  int tiles, chunks, noted;   // tiles filled up to per_cta's multiple; chunks and blocks (bytes: groups) to the end of the last block
  int64_t notes, bytes;   // offset in the workspace, after the image; of both
  __host__ __device__ XImage(const W4Layout& L, int M) {
    const int need = (M + kRows - 1) / kRows, ctas = (need + kMaxTiles - 1) / kMaxTiles;
    per_cta = (need + ctas - 1) / ctas;
    tiles = per_cta * ctas;
    chunks = L.blocks * 2;
    noted = HALF ? L.blocks : L.blocks * L.per_block;
    notes = static_cast<int64_t>(chunks) * tiles * kChunk;
    bytes = notes + static_cast<int64_t>(noted) * tiles * kNote;   // [block or group][tile][lane c]
  }
  static constexpr int kMaxTiles = 4;
};
bool half_image(const W4Layout& L, int M) { return M > (L.group == 32 ? 2 : 4); }
int64_t image_bytes(const W4Layout& L, int M) { return half_image(L, M) ? XImage<true>(L, M).bytes : XImage<false>(L, M).bytes; }

// Eight columns (vector v) of row m of x into the image at ws; the threads of a block's 16 vectors are
// neighbours and all here.
template <bool HALF, int GROUP>
__device__ __forceinline__ void prepare_vector(const uint16_t* __restrict__ x, int64_t ld_x, const W4Layout& L,
                                               const XImage<HALF>& I, int m, int v, uint8_t* ws) {
  using Image = XImage<HALF>;
  const bool in = v < I.chunks * 8;
  uint4 u = make_uint4(0, 0, 0, 0);
  if (in && v * 8 < L.K) u = *reinterpret_cast<const uint4*>(x + m * ld_x + v * 8);
  float f[8];
  unpack8(u, f);
  float peak = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) peak = fabsf(f[k]) <= peak ? peak : fabsf(f[k]) < INFINITY ? fabsf(f[k]) : INFINITY;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
  const bool finite = peak < INFINITY;
  const int chunk = v >> 3, step = (v >> 2) & 1, c = v & 3, tile = m / Image::kRows, row = m % Image::kRows;
  int a = 0;
  if (HALF) {
    if (peak > 0.f && finite) a = 15 - ilogbf(peak);
  } else if (peak > 0.f && finite) {
    // one less for the one mantissa whose high byte would be 128; 2^149 makes every number an integer, and its
    // reciprocal is the smallest float
    const int e = ilogbf(peak);
    const bool top = (__float_as_uint(peak) >> 16 & 0x7F) == 0x7F && e > -127;
    a = min(30 - e - (top ? 1 : 0), 149);
  }
  // in two factors: 2^a may be out of range
  const float a0 = power_of_two(a / 2), a1 = power_of_two(a - a / 2);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = finite ? f[k] * a0 * a1 : 0.f;
  const float factor = finite ? power_of_two(-a) : NAN;
  if constexpr (HALF) {
    if (!in) return;
    uint8_t* dst = ws + (static_cast<int64_t>(chunk) * I.tiles + tile) * Image::kChunk + step * 512 + (row * 4 + c) * 16;
    *reinterpret_cast<uint4*>(dst) =
        make_uint4(pack_f16x2(f[0], f[2]), pack_f16x2(f[1], f[3]), pack_f16x2(f[4], f[6]), pack_f16x2(f[5], f[7]));
    if (v % 16 == 0)   // of the block: two rows a lane
      reinterpret_cast<float*>(ws + I.notes + (static_cast<int64_t>(v / 16) * I.tiles + tile) * Image::kNote)[row] = factor;
  } else {
    constexpr int kLanes = GROUP / 8;   // of a group; 16 of a block
    uint32_t limb[4][2] = {};
    int sum[4] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      int i = __float2int_rn(f[k]);
#pragma unroll
      for (int l = 3; l >= 0; --l) {
        const int up = l > 0 ? (i + 128) >> 8 : 0;   // what the next higher byte takes
        const int b = i - up * 256;
        limb[l][k >> 2] |= (static_cast<uint32_t>(b) & 0xFFu) << (8 * (k & 3));
        sum[l] += b;
        i = up;
      }
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1)
#pragma unroll
      for (int l = 0; l < 4; ++l) sum[l] += __shfl_xor_sync(0xffffffffu, sum[l], o);
    if (!in) return;
    uint8_t* dst = ws + (static_cast<int64_t>(chunk) * I.tiles + tile) * Image::kChunk + (row * 16 + c) * 16 + step * 8;
#pragma unroll
    for (int l = 0; l < 4; ++l) *reinterpret_cast<uint2*>(dst + l * 64) = make_uint2(limb[l][0], limb[l][1]);
    if (v % kLanes == 0) {
      GroupNote* note = reinterpret_cast<GroupNote*>(ws + I.notes + (static_cast<int64_t>(v / kLanes) * I.tiles + tile) * Image::kNote) + row * 2;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        note[j] = GroupNote{{kMagic - (L.asym ? 15 : 8) * sum[2 * j], kMagic - (L.asym ? 15 : 8) * sum[2 * j + 1]}, factor, 0};
    }
  }
}

template <bool HALF, int GROUP>
__global__ void __launch_bounds__(kPrepThreads) w4_prepare_kernel(const uint16_t* __restrict__ x, int64_t ld_x, int M,
                                                                  W4Layout L, uint8_t* __restrict__ ws) {
  asm volatile("griddepcontrol.launch_dependents;");
  prepare_vector<HALF, GROUP>(x, ld_x, L, XImage<HALF>(L, M), blockIdx.y, blockIdx.x * kPrepThreads + threadIdx.x, ws);
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
  uint8_t* ws;
  unsigned int* err;
  // 1024 twice in f16.  An argument, since the compiler makes two instructions of an AND and an OR with constants
  // and one where one of them is in a register.
  uint32_t f16_1024;
};

// One contiguous copy (16-byte aligned, a multiple of 16 bytes) into shared memory.
__device__ __forceinline__ void copy_bulk(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}

// One product the plain way, for rows of x that are not finite.
__device__ __noinline__ float plain_product(const LinearArgs& a, int64_t n, int m) {
  float sum = 0.f;
  for (int k0 = 0; k0 < a.L.K && sum == sum; k0 += 32)   // a sum that is NaN stays so; a group is 32 columns at least
    for (int k = k0; k < k0 + 32; ++k) {
      float scale;
      const float u = w4_code(a.packed, a.L, n, k, &scale);
      sum = fmaf(bf16_bits_to_f32(a.x[m * a.ld_x + k]) * scale, u, sum);
    }
  return sum;
}

// y = x . W^T for up to NT tiles of rows of x: the weights are operand A (16 rows by 32 columns, or twice 16),
// the image of x operand B.
//
// Work.  One CTA a SM.  A unit is TILES tiles of 16 rows of W, all fed by a load of the
// image.  A CTA takes a run of units, and its warps equal runs of their blocks, laid end to
// end.  Each warp has a ring of stages, filled by TMA with a record (of every tile) a stage,
// that runs ahead across units.  A unit that one warp holds whole is written from registers;
// the parts of a unit that warps share go through shared memory to the warp that begins
// it, which adds them in order.  (Clusters that split a unit's columns over SMs balance better
// on paper, 12.25 tiles a CTA for 13 at 28672 rows, and measured 14.2 us for 13.6.)
//
// Half a byte a weight leaves about 22 cycles of an SM for a tile's chunk, so instructions
// count.  Bytes: 12 integer ones make a chunk's fragments (8 AND, 4 shifts).  Zeros: sum v (u - 8) = sum v u - 8 sum v,
// the second part, and the number that turns the integer into a float, being what a group's sums begin with; with
// stored zeros the codes become u + (15 - z), 0..30, by one addition a register, and 15 takes the place of 8.
// f16: a code in the low mantissa bits of 1024 is 1024 + u, four bits further up 1024 + 16 u; one f16 instruction
// takes off the zero, exactly, so that a weight of 0 is 0 whatever x it meets.
//
// Bytes, and one tile of f16, a warp reads with its notes into registers, one chunk and one group ahead; more tiles
// come by the ring (kRingX), since there are neither the registers nor the warps to hide their latency.  As many warps
// as have the registers and two stages: two tiles, 16 rows by 28672 x 4096, 10, 12 and 14 warps 30.1, 26.3 and 27.9 us;
// four tiles, 32 rows by 4096 x 4096, 6 and 8 warps 13.4 and 12.5; three tiles, 24 rows, 8 and 11 warps 10.6 either way.
//
// Measured, in a graph whose calls use different weights (more than L2 holds together): one row by 28672 x 4096 14.7 us,
// 4.1 TB/s of packed weights, by 4096 x 4096 6.7; 8 rows by 4096 x 4096 7.3, 16 rows 9.1, 32 rows 12.5; 19 rows by
// 4096 x 14336 in groups of 32 with zeros 23.7.  One row is bound by the copies and the launch; many rows by the
// codes' way to f16 and the latency of the image, which each warp copies for itself.
__host__ __device__ constexpr int linear_warps(bool half, int nt) { return !half || nt == 1 ? 16 : nt == 2 ? 12 : nt == 3 ? 11 : 8; }

template <bool HALF, int NT, int TILES, bool ASYM, int GROUP>
struct LinearSmem {
  using Image = XImage<HALF>;
  static constexpr int kWarps = linear_warps(HALF, NT);
  static constexpr bool kRingX = HALF && NT > 1;
  static constexpr int kRecord = 1024 + 128 / GROUP * 32 * (ASYM ? 2 : 1);
  static constexpr int kBlocks = TILES == 1 ? 2 : 1;           // of a stage: with one tile they lie side by side
  static constexpr int kImage = kBlocks * TILES * kRecord;     // where a stage's part of the image begins,
  static constexpr int kNotes = kImage + (kRingX ? NT * 2 * Image::kChunk : 0);   // and its notes
  static constexpr int kStage = kNotes + (kRingX ? NT * Image::kNote : 0);
  static constexpr int kSums = HALF ? 4 : 2;                   // of a lane, tile of W and tile of x
  static constexpr int kPart = TILES * NT * kSums * 32;        // floats of a part of a unit
  static constexpr int kFit = (227 * 1024 / kWarps - kPart * 4 - 32) / kStage;
  static constexpr int kStages = kFit < 4 ? kFit : 4;
  static_assert(kStages >= 2, "a warp needs two stages");
  static constexpr int kRing = kStages * kStage;               // a warp's
  static constexpr int kBytes = (kWarps * (kRing + kPart * 4 + kStages * 8) + 127) / 128 * 128;
};

template <bool HALF, int NT, int TILES, bool ASYM, int GROUP, bool FUSED>
__global__ void __launch_bounds__(32 * linear_warps(HALF, NT), 1) w4_linear_kernel(const __grid_constant__ LinearArgs a) {
  using Smem = LinearSmem<HALF, NT, TILES, ASYM, GROUP>;
  constexpr int kWarps = Smem::kWarps, kRecord = Smem::kRecord, kPart = Smem::kPart, kStages = Smem::kStages, kSums = Smem::kSums;
  constexpr bool kRingX = Smem::kRingX;
  using Image = XImage<HALF>;
  constexpr int kPer = 128 / GROUP, kSteps = GROUP / 32;        // groups of a block, steps of 32 columns of a group
  constexpr int kVecs = HALF ? 2 : 1;                           // 16-byte vectors of a lane, tile and chunk of the image
  constexpr int kLeast = 4;                                     // blocks: shorter runs cost more to join than to read
  extern __shared__ __align__(128) uint8_t smem[];
  float* parts = reinterpret_cast<float*>(smem + kWarps * Smem::kRing);   // [warp], of the unit that it goes on with
  uint64_t* bars = reinterpret_cast<uint64_t*>(parts + kWarps * kPart);
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, warp = threadIdx.x >> 5;
  const W4Layout& L = a.L;
  const Image I(L, a.M);
  const int P = L.blocks;
  const int units = (L.tiles + TILES - 1) / TILES;
  const int u0 = static_cast<int>(quotient(static_cast<int64_t>(units) * blockIdx.x, gridDim.x));
  const int u1 = static_cast<int>(quotient(static_cast<int64_t>(units) * (blockIdx.x + 1), gridDim.x));
  const int64_t all = static_cast<int64_t>(u1 - u0) * P;
  const int warps = static_cast<int>(min(static_cast<int64_t>(kWarps), (all + kLeast - 1) / kLeast));
  const int64_t each = quotient(all, warps), more = all - each * warps;
  auto begin_of = [&](int w) { return each * w + min(static_cast<int64_t>(w), more); };
  const int64_t begin = warp < warps ? begin_of(warp) : all, end = warp < warps ? begin_of(warp + 1) : all;
  const int count = static_cast<int>(end - begin);
  int unit = u0, piece = 0;
  if (count > 0) {
    const int64_t u = quotient(begin, P);
    unit += static_cast<int>(u);
    piece = static_cast<int>(begin - u * P);
  }

  // ---- the ring
  uint8_t* ring = smem + warp * Smem::kRing;
  bars += warp * kStages;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) tc::mbar_init(bars + i, 1);
    tc::fence_mbar_init();
  }
  __syncwarp();
  int to_issue = count, ld_piece = piece, ld_unit = unit;
  const uint8_t* src = a.packed + (static_cast<int64_t>(unit) * TILES * P + piece) * kRecord;
  auto issue = [&](int stage) {
    if (to_issue <= 0) return;
    const int n = min(to_issue, Smem::kBlocks);
    if (lane == 0) {
      tc::mbar_arrive_expect_tx(bars + stage, n * TILES * kRecord + Smem::kStage - Smem::kImage);
      uint8_t* dst = ring + stage * Smem::kStage;
      if (kRingX) {
        // of one block: its two chunks of the image, NT tiles of each, and their notes
        const int first = blockIdx.y * NT, at_once = I.tiles == NT ? 1 : 0;
        for (int h = 0; h < 2; h += 1 + at_once)
          copy_bulk(dst + Smem::kImage + h * NT * Image::kChunk,
                    a.ws + (static_cast<int64_t>(ld_piece * 2 + h) * I.tiles + first) * Image::kChunk,
                    NT * Image::kChunk << at_once, bars + stage);
        copy_bulk(dst + Smem::kNotes, a.ws + I.notes + (static_cast<int64_t>(ld_piece) * I.tiles + first) * Image::kNote,
                  NT * Image::kNote, bars + stage);
      }
      copy_bulk(dst, src, n * kRecord, bars + stage);
      if (TILES == 2)   // a tile past the last one repeats it: nothing of it is written
        copy_bulk(dst + kRecord, ld_unit * 2 + 1 < L.tiles ? src + static_cast<int64_t>(P) * kRecord : src, kRecord, bars + stage);
    }
    to_issue -= n;
    src += n * kRecord;
    if (TILES == 2 && ++ld_piece == P) {
      ld_piece = 0;
      ++ld_unit;
      src += static_cast<int64_t>(P) * kRecord;
    }
  };
  if (kRingX) asm volatile("griddepcontrol.wait;" ::: "memory");   // the image is ready
#pragma unroll 1
  for (int i = 0; i < kStages; ++i) issue(i);

  // ---- the image: the workspace's, or (FUSED) made here, in shared memory, while the ring fills
  const uint8_t* img = a.ws;
  if (FUSED) {
    uint8_t* own = smem + Smem::kBytes;
    for (int m = 0; m < a.M; ++m)
      for (int v = 0; v < I.chunks * 8; v += 32 * kWarps)
        prepare_vector<HALF, GROUP>(a.x, a.ld_x, L, I, m, v + threadIdx.x, own);
    __syncthreads();
    img = own;
  }
  // image and notes are read one chunk and one group (f16: one block) ahead
  const int image_chunk = I.tiles * (Image::kChunk / 16), note_stride = I.tiles * Image::kNote;
  const uint4* image = reinterpret_cast<const uint4*>(img) + blockIdx.y * NT * (Image::kChunk / 16) + lane;
  const uint8_t* notes = img + I.notes + blockIdx.y * NT * Image::kNote + c * (Image::kNote / 4);
  using Note = typename std::conditional<HALF, float2, uint4>::type;
  auto load_image = [&](uint4 (&x)[NT][kVecs], int chunk) {
    const uint4* p = image + chunk * image_chunk;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < kVecs; ++j) x[n][j] = p[(n * kVecs + j) * 32];
  };
  auto load_note = [&](Note (&x)[NT], int at) {
    const uint8_t* p = notes + static_cast<int64_t>(at) * note_stride;
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] = *reinterpret_cast<const Note*>(p + n * Image::kNote);
  };
  // bytes: a lane's two columns are the high or the low half of a row's four
  const float high = c & 1 ? 256.f : 16777216.f, low = c & 1 ? 1.f : 65536.f, back = -12582912.f * (high + low);

  float acc[TILES][NT][kSums] = {};   // rows g, g + 8 of W by a row (f16: two rows) of a tile of x
  float sum[TILES][NT][kSums];        // of a block's groups
  using Part = typename std::conditional<HALF, float, int>::type;
  Part part[TILES][NT][4];
  // Step s of 32 columns, of group grp, of the record(s) at `rec`, with the image's chunk x and (bytes) the group's note.
  auto step = [&](const uint8_t* rec, int grp, int s, const uint4 (&x)[NT][kVecs], const Note (&note)[NT]) {
    const bool first = s % kSteps == 0, last = s % kSteps == kSteps - 1;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const uint8_t* sc = rec + t * kRecord + 1024 + grp * 32 + g * 4;
      const uint2 w = *reinterpret_cast<const uint2*>(rec + t * kRecord + (s >> 1) * 512 + lane * 16 + (s & 1) * 8);
      const uint32_t z = ASYM ? *reinterpret_cast<const uint32_t*>(sc + kPer * 32) : 0;   // 15 - zero of rows g, g + 8
      if constexpr (HALF) {
        // 1024 + zero and 1024 + 16 zero, twice each
        uint32_t z0 = 0x64086408u, z1 = 0x64806480u;
        if (ASYM) {
          z0 = (__byte_perm(z, 0, 0x4040) ^ 0x000F000Fu) | 0x64006400u;
          z1 = ((__byte_perm(z, 0, 0x4141) ^ 0x000F000Fu) << 4) | 0x64006400u;
        }
        const uint32_t words[2] = {w.x, w.y};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t lo = words[h], hi = words[h] >> 8;
          const uint32_t f[4] = {sub_f16x2((lo & 0x000F000Fu) | a.f16_1024, z0), sub_f16x2((lo & 0x00F000F0u) | a.f16_1024, z1),
                                 sub_f16x2((hi & 0x000F000Fu) | a.f16_1024, z0), sub_f16x2((hi & 0x00F000F0u) | a.f16_1024, z1)};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint4 b = x[n][kRingX ? 0 : s & 1];
            if (kRingX)
              b = *reinterpret_cast<const uint4*>(rec + Smem::kImage + ((s >> 1) * NT + n) * Image::kChunk + (s & 1) * 512 + lane * 16);
            if (first && h == 0)
              mma_f16_zero(part[t][n], f, b.x, b.y);
            else
              mma_f16(part[t][n], f, h ? b.z : b.x, h ? b.w : b.y);
          }
        }
      } else {
        uint32_t f[4] = {w.x & 0x0F0F0F0Fu, (w.x >> 4) & 0x0F0F0F0Fu, w.y & 0x0F0F0F0Fu, (w.y >> 4) & 0x0F0F0F0Fu};
        if (ASYM) {
          const uint32_t z0 = __byte_perm(z, 0, 0x0000), z1 = __byte_perm(z, 0, 0x1111);
          f[0] += z0, f[1] += z1, f[2] += z0, f[3] += z1;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (first) {
            part[t][n][0] = part[t][n][2] = static_cast<int>(note[n].x);
            part[t][n][1] = part[t][n][3] = static_cast<int>(note[n].y);
          }
          if (s & 1)
            mma_u8s8(part[t][n], f, x[n][0].z, x[n][0].w);
          else
            mma_u8s8(part[t][n], f, x[n][0].x, x[n][0].y);
        }
      }
      if (last) {
        const uint32_t two = *reinterpret_cast<const uint32_t*>(sc);
        const float w2[2] = {bf16_lo(two), HALF ? bf16_hi(two) * 0.0625f : bf16_hi(two)};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int q = 0; q < kSums; ++q) {
            float v;
            if constexpr (HALF)
              v = part[t][n][q];
            else   // high h + low l of the floats 1.5 2^23 + h and + l: the first product and its constant are
                   // multiples of `high`, and exact
              v = fmaf(__int_as_float(part[t][n][2 * q + 1]), low, fmaf(__int_as_float(part[t][n][2 * q]), high, back));
            sum[t][n][q] = fmaf(v, w2[q / (kSums / 2)], sum[t][n][q]);
          }
      }
    }
  };
  auto begin_block = [&]() {
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < kSums; ++q) sum[t][n][q] = 0.f;
  };
  // the row's 2^-a belongs to the block: its groups' sums meet it together
  auto end_block = [&](const uint8_t* rec, const Note (&note)[NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float factor[2];
      if constexpr (HALF) {
        float2 two = note[n];
        if (kRingX) two = *reinterpret_cast<const float2*>(rec + Smem::kNotes + n * Image::kNote + c * 8);
        factor[0] = two.x, factor[1] = two.y;
      } else {
        factor[0] = factor[1] = __uint_as_float(note[n].z);
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int q = 0; q < kSums; ++q) acc[t][n][q] = fmaf(sum[t][n][q], factor[q & 1], acc[t][n][q]);
    }
  };
  // Sum q of a lane: row g (+ 8) of W by row `col` of a tile of x.
  auto row_of = [](int q) { return q / (kSums / 2) * 8; };
  auto col_of = [&](int q) { return HALF ? 2 * c + (q & 1) : c >> 1; };
  auto write = [&](int u) {
    const int m0 = static_cast<int>(blockIdx.y) * NT * Image::kRows;
    const int64_t row0 = static_cast<int64_t>(u) * TILES * 16 + g;
    float resid[NT][TILES][kSums];   // all on their way before the first store, which may be to the same place
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int q = 0; q < kSums; ++q) {
          const int m = m0 + n * Image::kRows + col_of(q);
          const int64_t row = row0 + t * 16 + row_of(q);
          resid[n][t][q] = a.resid && m < a.M && row < L.N ? bf16_bits_to_f32(a.resid[m * a.ld_r + row]) : 0.f;
        }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (!HALF) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int q = 0; q < kSums; ++q) acc[t][n][q] += __shfl_xor_sync(0xffffffffu, acc[t][n][q], 1);   // the other bytes' lane
        if (c & 1) continue;
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int q = 0; q < kSums; ++q) {
          const int m = m0 + n * Image::kRows + col_of(q);
          const int64_t row = row0 + t * 16 + row_of(q);
          if (m >= a.M || row >= L.N) continue;
          const float v = acc[t][n][q];
          const float y = (fabsf(v) < INFINITY ? v : plain_product(a, row, m)) + resid[n][t][q];
          if (a.y_bf16)
            static_cast<uint16_t*>(a.y)[m * a.ld_y + row] = bf16_bits_rn(y);
          else
            static_cast<float*>(a.y)[m * a.ld_y + row] = y;
        }
    }
  };
  float* mine = parts + warp * kPart + lane;
  auto clear = [&]() {
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < kSums; ++q) acc[t][n][q] = 0.f;
  };
  auto leave = [&]() {
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < kSums; ++q) mine[((t * NT + n) * kSums + q) * 32] = acc[t][n][q];
    clear();
  };

  if (!FUSED && !kRingX) asm volatile("griddepcontrol.wait;" ::: "memory");   // the image is ready
  bool begun = piece == 0;   // this warp holds its unit's first block
  bool lost = false;         // a copy did not arrive in time
  int stage = 0, left = count;
  uint32_t phase = 0;
  uint4 x0[NT][kVecs], x1[NT][kVecs];
  Note note[2][NT];
  constexpr int kNotesPer = HALF ? 1 : kPer;   // of a block
  if (!kRingX && count > 0) {
    load_image(x0, piece * 2);
    load_note(note[0], piece * kNotesPer);
  }
#pragma unroll 1
  while (left > 0) {
    if (!__all_sync(0xffffffffu, tc::mbar_wait(bars + stage, phase, a.err))) {
      lost = true;
      break;
    }
#pragma unroll
    for (int b = 0; b < Smem::kBlocks; ++b) {
      if (b > 0 && left <= 0) break;
      const uint8_t* rec = ring + stage * Smem::kStage + b * kRecord;
      const int after = piece + 1 == P ? 0 : piece + 1;
      if (!kRingX) load_image(x1, piece * 2 + 1);
      begin_block();
      if constexpr (kRingX) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
          for (int s = 0; s < kSteps; ++s) step(rec, i, i * kSteps + s, x0, note[0]);
        end_block(rec, note[0]);
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          // note[..] of group i of the block: with one note a block they change places from block to block
          const int i = s / kSteps, k = kNotesPer == 1 ? 0 : i, at = kNotesPer == 1 ? b & 1 : i & 1;
          if (kNotesPer == 1 ? s == 0 : s % kSteps == 0)
            load_note(note[at ^ 1], k + 1 < kNotesPer ? piece * kNotesPer + k + 1 : after * kNotesPer);
          step(rec, i, s, s < 2 ? x0 : x1, note[at]);
          if (s == 1) load_image(x0, after * 2);
          if (s == 3) end_block(rec, note[at]);
        }
        static_assert(kNotesPer > 1 || Smem::kBlocks == 2, "notes change places from block to block");
      }
      --left;
      piece = after;
      if (piece == 0) {
        if (begun) {
          write(unit);
          clear();
        } else {
          leave();
        }
        ++unit;
        begun = true;
      }
    }
    __syncwarp();   // all lanes are done with the stage
    issue(stage);
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  // after a lost copy: the copies still under way end before the shared memory does
  for (int under_way = lost ? (left - to_issue + Smem::kBlocks - 1) / Smem::kBlocks : 0; under_way > 0; --under_way) {
    tc::mbar_wait(bars + stage, phase, a.err);
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  // A unit goes on in the next warp: this one keeps what it began, and leaves what it only goes on with.
  const bool goes_on = piece > 0 && count > 0, joins = goes_on && begun;
  if (goes_on && !begun) leave();
  __syncthreads();
  if (joins) {
    const int64_t unit_end = static_cast<int64_t>(unit - u0 + 1) * P;
    auto add = [&](const float* from) {
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int q = 0; q < kSums; ++q) acc[t][n][q] += from[((t * NT + n) * kSums + q) * 32];
    };
#pragma unroll 4
    for (int w = warp + 1; w < warps && begin_of(w) < unit_end; ++w)
      add(parts + w * kPart + lane);
    write(unit);
  }
}

template <bool HALF, int NT, int TILES, bool ASYM, int GROUP, bool FUSED>
int launch_linear_one(const LinearArgs& a, const XImage<HALF>& I, cudaStream_t st) {
  const auto kernel = w4_linear_kernel<HALF, NT, TILES, ASYM, GROUP, FUSED>;
  const int bytes = LinearSmem<HALF, NT, TILES, ASYM, GROUP>::kBytes + (FUSED ? static_cast<int>(I.bytes) : 0);
  GLT_TRY(ensure_smem_attr(reinterpret_cast<const void*>(kernel), bytes));
  const int units = (a.L.tiles + TILES - 1) / TILES;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units < num_sms() ? units : num_sms(), I.tiles / NT);
  cfg.blockDim = dim3(32 * linear_warps(HALF, NT));
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = FUSED ? 0 : 1;   // with a preparation: starts beside it and waits for its end after the first copies
  GLT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  GLT_LAUNCH_CHECK();
  return GLT_OK;
}

template <bool HALF, int NT, int TILES, bool ASYM, int GROUP>
int launch_linear(const LinearArgs& a, cudaStream_t st) {
  const XImage<HALF> I(a.L, a.M);
  if (I.tiles / NT > 65535 || a.M > 65535) return fail(GLT_EINVAL, "w4: %d rows (at most 65535)", a.M);
  // A small x of one tile is turned into its bytes by every CTA for itself: one launch less, 2.1 us of the host's time.
  // On the device one row by 28672 x 4096 takes 14.5 us so and 15.6 with a launch before, by 896 x 4864 6.6 and 5.9;
  // two rows by 896 x 4864 8.8 and 5.9.  Its f16 image takes longer to make (8 rows by 4864 x 896 10.1 us and 5.2).
  if constexpr (!HALF && NT == 1)
    if (static_cast<int64_t>(a.M) * a.L.K <= 16384 && LinearSmem<HALF, NT, TILES, ASYM, GROUP>::kBytes + I.bytes <= 227 * 1024)
      return launch_linear_one<HALF, NT, TILES, ASYM, GROUP, true>(a, I, st);
  w4_prepare_kernel<HALF, GROUP><<<dim3((I.chunks * 8 + kPrepThreads - 1) / kPrepThreads, a.M), kPrepThreads, 0, st>>>(a.x, a.ld_x, a.M, a.L, a.ws);
  GLT_LAUNCH_CHECK();
  return launch_linear_one<HALF, NT, TILES, ASYM, GROUP, false>(a, I, st);
}

template <bool HALF, int NT, int TILES>
int launch_linear_as(const LinearArgs& a, cudaStream_t st) {
  if (a.L.asym) {
    if (a.L.group == 32) return launch_linear<HALF, NT, TILES, true, 32>(a, st);
    return a.L.group == 64 ? launch_linear<HALF, NT, TILES, true, 64>(a, st) : launch_linear<HALF, NT, TILES, true, 128>(a, st);
  }
  if (a.L.group == 32) return launch_linear<HALF, NT, TILES, false, 32>(a, st);
  return a.L.group == 64 ? launch_linear<HALF, NT, TILES, false, 64>(a, st) : launch_linear<HALF, NT, TILES, false, 128>(a, st);
}

int launch_rows(const LinearArgs& a, cudaStream_t st) {
  if (!half_image(a.L, a.M)) return a.M <= 2 ? launch_linear_as<false, 1, 1>(a, st) : launch_linear_as<false, 2, 1>(a, st);
  const int n = XImage<true>(a.L, a.M).per_cta;
  if (n == 1) return launch_linear_as<true, 1, 1>(a, st);
  if (n == 2) return launch_linear_as<true, 2, 2>(a, st);
  return n == 3 ? launch_linear_as<true, 3, 2>(a, st) : launch_linear_as<true, 4, 2>(a, st);
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
  glt::w4_pack_kernel<<<glt::grid_for(L.bytes / 4, 256), 256, 0,
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

extern "C" int glt_w4_linear_workspace(int M, int N, int K, int group, int y_dtype, int64_t* bytes) {
  if (!bytes) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_shape(N, K, group));
  if (M < 0) return glt::fail(GLT_EINVAL, "w4: negative rows");
  if (y_dtype != 0 && y_dtype != 1) return glt::fail(GLT_EINVAL, "w4: output type %d (0 fp32, 1 bf16)", y_dtype);
  const W4Layout L(N, K, group, 0);
  *bytes = M == 0 ? 0 : glt::image_bytes(L, M);
  return GLT_OK;
}

extern "C" int glt_w4_linear(const void* packed, int N, int K, int group, int asym, const uint16_t* x,
                             int64_t ld_x, int M, void* y, int64_t ld_y, int y_dtype,
                             const uint16_t* resid, int64_t ld_r, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  GLT_TRY(glt::check_shape(N, K, group));
  if (!packed || (M > 0 && (!x || !y))) return glt::fail(GLT_EINVAL, "null argument");
  if (M < 0) return glt::fail(GLT_EINVAL, "w4: negative rows");
  if (y_dtype != 0 && y_dtype != 1) return glt::fail(GLT_EINVAL, "w4: output type %d (0 fp32, 1 bf16)", y_dtype);
  if (ld_x < K || ld_x % 8 || !glt::aligned16(x))
    return glt::fail(GLT_EINVAL, "w4: x needs 16-byte aligned rows (row stride a multiple of 8, at least K)");
  if (ld_y < N || (resid && ld_r < N)) return glt::fail(GLT_EINVAL, "w4: output or residual row stride below N %d", N);
  if (!glt::aligned16(packed)) return glt::fail(GLT_EINVAL, "w4: packed weights must be 16-byte aligned");
  if (M == 0) return GLT_OK;
  const W4Layout L(N, K, group, asym);
  const int64_t need = glt::image_bytes(L, M);
  if (workspace_bytes < need || !workspace || !glt::aligned16(workspace))
    return glt::fail(GLT_EINVAL, "w4: workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
  if (need / 4 > INT_MAX) return glt::fail(GLT_EINVAL, "w4: %d rows of %d columns", M, K);
  const glt::LinearArgs a{static_cast<const uint8_t*>(packed), L, x, ld_x, M, y, ld_y, y_dtype, resid, ld_r,
                          static_cast<uint8_t*>(workspace), glt::device_error_word(), 0x64006400u};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return glt::launch_rows(a, st);
}
