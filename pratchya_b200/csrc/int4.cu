// Weights in 4 bits with a scale, and where wanted a zero point, for each group of 32, 64 or 128 values along the contraction:
//   w[k][n] = scale[n][k / g] * (u[k][n] - zero[n][k / g])        u in 0..15, zero 8 where none is stored
// the quantizer, its inverse, and products of few rows with such a weight, y[m][n] = sum_k x[m][k] w[k][n].
//
// Stored by tiles of 16 columns n and 128 values of k, in the order in which a warp's matrix instruction takes them, so that a warp reads a tile
// as two 512-byte rows of 16 bytes a lane:
//   q [ceil(N/16)][ceil(K/128)][1024]: byte half * 512 + (g * 4 + t) * 16 + c * 4 + b, column 16 A + 8 half + g; the four bytes of a word hold
//     k = 128 B + 32 c + 8 t + i, i = 0..7, at nibbles 0, 4, 1, 5, 2, 6, 3, 7 (the lower nibble of a byte first);
//   scale bf16 [ceil(N/16)][ceil(K/128)][16][128 / g], zero uint8 the same.
// k beyond K holds the code of 0, columns beyond N scales of 0.
#include "common.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

namespace pb {
namespace {

namespace cg = cooperative_groups;

// ---- the quantizer -----------------------------------------------------------------------------------------------------
constexpr int kQuantThreads = 256, kQuantCols = 64;      // 128 x 64 weights a CTA
constexpr int kHalf = 160;             // words of eight columns in shared memory, 20 a column; a word's place among four goes by the eight: a warp's columns meet no bank twice

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// where word (t, quarter) of a CTA's column is in shared memory, and a tile's sixteen bytes `slot` there
__device__ __forceinline__ uint32_t staged_at(uint32_t col, uint32_t t, uint32_t quarter) { return col / 8 * kHalf + col % 8 * 20 + t * 4 + (quarter ^ (col / 8 & 3)); }
__device__ __forceinline__ uint4* staged_slot(uint32_t* staged, uint32_t eight, uint32_t slot) { return reinterpret_cast<uint4*>(staged + eight * kHalf + slot / 4 * 20 + slot % 4 * 4); }
__device__ __forceinline__ uint4 turned(uint4 o, uint32_t eight) {      // its words to their places, and back
  if (eight & 1) o = make_uint4(o.y, o.x, o.w, o.z);
  if (eight & 2) o = make_uint4(o.z, o.w, o.x, o.y);
  return o;
}
constexpr float kRound = 12582912.0f;      // added to a number below 2^22 in size, it leaves that number's nearest integer (of two the even one) in the last bits
constexpr uint32_t kRoundBits = 0x4b400000u;

// ZERO: scale = bf16((max(w, 0) - min(w, 0)) / 15), zero = rint(-min / scale), u = rint(w / scale) + zero, both within 0..15;
// otherwise scale = bf16(max|w| / 7), u = rint(w / scale) + 8 within 0..15: a normal scale is 2^-9 of itself too small at most, and u within 1..15 by itself; a subnormal
// one may be a third too small, and there, alone, the values are brought to its reach first.
// A group of nothing but zeros has scale 0.  The scale is rounded before the codes are taken: they are the nearest ones for the scale that is stored.
// A group that holds a NaN or an infinity has a scale that is no finite number.
// A thread has COLS neighbouring columns (two where one load brings two bf16) and 32 / COLS values of k of each.  f32 [2048, 8192] in 16.1 us (floor 11.6), [2048, 65536]
// in 105 (92, HBM); bf16 [2048, 8192] in 15.3.  With a division per weight, __fdiv_rn, and words staged without regard to banks 22.
template <typename T, bool ZERO, int COLS>
__global__ void __launch_bounds__(kQuantThreads) quantize_int4_kernel(const T* __restrict__ w, int64_t depth, int64_t cols, int per_group, uint32_t kblocks,
                                                                      uint32_t* __restrict__ q, __nv_bfloat16* __restrict__ scale, uint8_t* __restrict__ zero) {
  grid_wait();
  constexpr int kRows = 32 / COLS, kRuns = 4 * COLS, kWords = kRows / 8;      // of a thread; threads along k
  __shared__ float lows[ZERO ? kRuns : 1][kQuantCols], highs[kRuns][kQuantCols];
  __shared__ __align__(16) uint32_t staged[8 * kHalf];
  const uint32_t pair = threadIdx.x % (kQuantCols / COLS), run = threadIdx.x / (kQuantCols / COLS);      // a warp has neighbouring columns
  const uint32_t kb = blockIdx.x;
  const int64_t n0 = (int64_t)blockIdx.y * kQuantCols + pair * COLS, k0 = (int64_t)kb * 128 + run * kRows;
  float v[COLS][kRows], low[COLS], high[COLS];
  const T* from = w + k0 * cols + n0;
  const int rows = n0 >= cols ? 0 : (int)min((int64_t)kRows, depth - k0);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const T* at = from + i * cols;
    if constexpr (COLS == 2) {      // of an even number of columns, two bf16 at four bytes
      const uint32_t two = i < rows ? __ldg(reinterpret_cast<const uint32_t*>(at)) : 0u;
      v[0][i] = __uint_as_float(two << 16);
      v[1][i] = __uint_as_float(two & 0xffff0000u);
    } else {
      v[0][i] = i < rows ? Elem<T>::to_f32(*at) : 0.0f;
    }
  }
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    low[c] = high[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (ZERO) {
        low[c] = -max_nan(-low[c], -v[c][i]);
        high[c] = max_nan(high[c], v[c][i]);
      } else {
        high[c] = max_nan(high[c], fabsf(v[c][i]));
      }
    }
    if (ZERO) lows[run][pair * COLS + c] = low[c];
    highs[run][pair * COLS + c] = high[c];
  }
  __syncthreads();
  const int runs = kRuns / per_group, first = (int)run / runs * runs;      // of a group
  const int64_t tiles = (cols + 15) / 16;
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    const uint32_t col = pair * COLS + c;
    for (int o = 0; o < runs; ++o) {
      if (ZERO) low[c] = -max_nan(-low[c], -lows[first + o][col]);
      high[c] = max_nan(high[c], highs[first + o][col]);
    }
    float span = ZERO ? __fsub_rn(high[c], low[c]) : high[c], steps = ZERO ? 15.0f : 7.0f;
    if (ZERO && span == INFINITY) { span = 0.5f * high[c] - 0.5f * low[c]; steps = 7.5f; }      // of finite weights, twice what the type holds
    const float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(span, steps)));
    if (!ZERO && s < 0x1p-126f && s > 0.0f)
#pragma unroll
      for (int i = 0; i < kRows; ++i) v[c][i] = fminf(fmaxf(v[c][i], -8.0f * s), 7.0f * s);
    const float z = !ZERO ? 8.0f : s != 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(-low[c], s)), 0.0f), 15.0f) : 0.0f;
    // Correctly rounded quotients by a reciprocal and two corrections, of numbers that a power of two has taken from the ends of the range (what it loses of a
    // number below 2^-62 is nothing beside a scale above 2^90).  A scale of zero or no number: codes of 0, or any.
    const float f = s < 0x1p-90f ? 0x1p64f : s > 0x1p90f ? 0x1p-64f : 1.0f, d = s * f, r = s > 0.0f && s < INFINITY ? __frcp_rn(d) : 0.0f;
    const float2 f2 = make_float2(f, f), r2 = make_float2(r, r), nd2 = make_float2(-d, -d), round2 = make_float2(kRound, kRound), z2 = make_float2(z, z);
#pragma unroll
    for (int word = 0; word < kWords; ++word) {
      float2 u[4];      // of k = 2 i and 2 i + 1
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = __fmul2_rn(make_float2(v[c][word * 8 + 2 * i], v[c][word * 8 + 2 * i + 1]), f2);
        u[i] = __fadd2_rn(__fadd2_rn(div_hoisted_unsigned2(x, nd2, r2), round2), z2);
        if (ZERO) u[i] = make_float2(fminf(fmaxf(u[i].x, kRound), kRound + 15.0f), fminf(fmaxf(u[i].y, kRound), kRound + 15.0f));
      }
      // nibbles 7..0 hold k = 7, 5, 3, 1, 6, 4, 2, 0; the bits of kRound come out of all eight together
      uint32_t packed = __float_as_uint(u[3].y);
      packed = packed * 16 + __float_as_uint(u[2].y);
      packed = packed * 16 + __float_as_uint(u[1].y);
      packed = packed * 16 + __float_as_uint(u[0].y);
      packed = packed * 16 + __float_as_uint(u[3].x);
      packed = packed * 16 + __float_as_uint(u[2].x);
      packed = packed * 16 + __float_as_uint(u[1].x);
      packed = packed * 16 + __float_as_uint(u[0].x);
      const uint32_t k8 = run * kWords + word, t = k8 % 4, quarter = k8 / 4;      // k = 32 quarter + 8 t + ..
      staged[staged_at(col, t, quarter)] = packed - kRoundBits * 0x11111111u;
    }
    const int64_t at = (int64_t)blockIdx.y * 4 + col / 16;
    if (at < tiles && (int)run == first) {
      const int64_t i = ((at * kblocks + kb) * 16 + col % 16) * per_group + run / runs;
      scale[i] = __float2bfloat16_rn(s);
      if (ZERO) zero[i] = (uint8_t)z;
    }
  }
  __syncthreads();
  const uint32_t part = threadIdx.x / 64;      // a tile's 1024 bytes, 16 a thread
  const int64_t a = (int64_t)blockIdx.y * 4 + part;
  if (a < tiles) {
    const uint32_t slot = threadIdx.x % 64, eight = threadIdx.x / 32;
    reinterpret_cast<uint4*>(q + (a * kblocks + kb) * 256)[slot] = turned(*staged_slot(staged, eight, slot % 32), eight);
  }
}

// A thread has COLS neighbouring columns (two of bf16, which one store takes) and 32 / COLS values of k of each.  f32 [2048, 8192] in 12.6 us, [2048, 65536] in 101
// (floor 92); bf16 [2048, 8192] in 9.7.  With the words straight from global memory, 64 bytes apart, bf16 took 13.8; with every code shifted to the bottom of its word 11.1.
template <typename T, int COLS>
__global__ void __launch_bounds__(kQuantThreads) dequantize_int4_kernel(const uint32_t* __restrict__ q, const __nv_bfloat16* __restrict__ scale, const uint8_t* __restrict__ zero,
                                                                        int64_t depth, int64_t cols, int per_group, uint32_t kblocks, T* __restrict__ w) {
  grid_wait();
  constexpr int kRows = 32 / COLS, kWords = kRows / 8;
  __shared__ __align__(16) uint32_t staged[8 * kHalf];
  const uint32_t pair = threadIdx.x % (kQuantCols / COLS), run = threadIdx.x / (kQuantCols / COLS), kb = blockIdx.x, quarter = run * kWords / 4;
  const int64_t n = (int64_t)blockIdx.y * kQuantCols + pair * COLS, k0 = (int64_t)kb * 128 + run * kRows, tiles = (cols + 15) / 16;
  float s[COLS], z[COLS];
  if (n < cols)
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const int64_t i = (((n / 16 * kblocks + kb) * 16) + (n + c) % 16) * per_group + quarter * per_group / 4;
      s[c] = __bfloat162float(scale[i]);
      z[c] = zero ? (float)zero[i] : 8.0f;
    }
  const int64_t a = (int64_t)blockIdx.y * 4 + threadIdx.x / 64;
  const uint32_t eight = threadIdx.x / 32;
  if (a < tiles) *staged_slot(staged, eight, threadIdx.x % 32) = turned(__ldg(reinterpret_cast<const uint4*>(q + (a * kblocks + kb) * 256) + threadIdx.x % 64), eight);
  __syncthreads();
  if (n >= cols) return;
  uint32_t word[COLS][kWords];
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int t = 0; t < kWords; ++t) word[c][t] = staged[staged_at(pair * COLS + c, (run * kWords + t) % 4, quarter)];
  // A code at nibble p of a word (or, p > 4, of its upper half) is 16^p times itself there: it is taken as that, and the scale is so much smaller.
  float scales[COLS][5], zeros[COLS][5];
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int p = 0; p < 5; ++p) {
      scales[c][p] = s[c] * (1.0f / (1 << 4 * p));
      zeros[c][p] = kRound + z[c] * (1 << 4 * p);
    }
  T* to = w + k0 * cols + n;
  const uint32_t pitch = (uint32_t)cols;      // columns are fewer than 2^22 (the grid's second dimension): offsets within a run of k take 32 bits, one operation
  const int rows = (int)min((int64_t)kRows, depth - k0);
#pragma unroll
  for (int t = 0; t < kWords; ++t)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int nibble = j / 2 + 4 * (j % 2), p = nibble > 4 ? nibble - 4 : nibble;
      float v[COLS];
#pragma unroll
      for (int c = 0; c < COLS; ++c) v[c] = scales[c][p] * (__uint_as_float(((nibble > 4 ? word[c][t] >> 16 : word[c][t]) & (15u << 4 * p)) | kRoundBits) - zeros[c][p]);
      if (t * 8 + j < rows) {
        T* at = to + (uint32_t)(t * 8 + j) * pitch;
        if constexpr (COLS == 2) *reinterpret_cast<uint32_t*>(at) = pack_bf16x2(v[0], v[1]);
        else *at = Elem<T>::from_f32(v[0]);
      }
    }
}

// ---- products of few rows ------------------------------------------------------------------------------------------------
// A warp's matrix instruction takes 16 columns n of the weight as its rows and 8 rows of x as its columns: the weight, of which there is much, fills it, and
// x, of which there is little, is what may be padded.  (tcgen05's tiles of 64 rows and more would want codes unpacked into shared memory for one to thirty-two
// columns; the tensor core is busy a fifth of the time here.)  Two forms of x:
//  - whole numbers: every block of 128 values of a row gets a scale, a power of two, and its values become whole numbers of three (bf16) or four (f32) digits of
//    eight bits with a sign, each digit a column of its own.  Codes become bytes of 16 (u - 8) by one operation on four of them, products and sums of a group
//    are exact in int32 (m16n8k32), and meet the scales in f32.  24 operations unpack a kilobyte of codes.
//  - bf16 as it is (m16n8k16): codes become bf16 by their bits (0x4300 | u is 128 + u) less 128 + zero, both exact, 88 operations a kilobyte; a row of x is one column.
// Sums over a group meet the group's scale in f32, groups and warps add in f32.
// Floor: the weight's bytes from HBM, 10.6 us for 2048 x 65536.  On one B200, us:
//   one row, f32: 2048 x 65536 15.6 (68 %), 2048 x 8192 4.2, 2048 x 2048 3.0, 2048 x 128 2.9 (a launch, x's way to the digits and one barrier)
//   bf16 rows x depth x columns: 8 x 2048 x 8192 5.8, 32 x 8192 x 2048 11.0, 32 x 2048 x 65536 53 (with so much of x in shared
//   memory an SM has one CTA, two warps a scheduler: tensor pipe 30 %, issue slots 35 %; two blocks ahead instead of four 57)
// What a row of 65536 columns takes beside the stream of codes (9.4 us at 7.3 TB/s): 2.7 until x is in digits, 0.9 for the sums of the warps, a launch.
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPad = 32;               // values behind a row of x in shared memory: neighbouring rows' 64 bytes then lie in other banks
constexpr int kPadDigits = 16;         // the same for digits: neighbouring rows' sixteen bytes of four lanes in turn
constexpr int kMaxCluster = 8;
constexpr int kMaxChunk = 16;
constexpr uint32_t kNoTile = 0xffffffffu;
// tiles of a chunk that one warp's run can touch
__host__ __device__ constexpr uint32_t segments_of(uint32_t chunk) { return (chunk + kWarps - 1) / kWarps + 1; }

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// two codes of a word, less 128 + zero of `bias`
template <int SHIFT> __device__ __forceinline__ uint32_t pair_of(uint32_t word, uint32_t bias) {
  uint32_t r;      // (word >> SHIFT & mask) | 128s in one operation behind the shift
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(r) : "r"(word >> SHIFT), "r"(0x43004300u));
  return sub_bf16x2(r, bias);
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mma_from_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A whole number below 2^22 in size as the low bits of an f32: kWhole + i, whose value less kWholeValue is i
constexpr int kWhole = 0x4b400000;
constexpr float kWholeValue = 12582912.0f;

// The whole numbers that a block of 128 values of x becomes: x = scale * t in DIGITS digits of eight bits with a sign each.  The scale is a power of two, and
// |t| < 2^22 or 2^30: a bf16 within 2^-14 of its block's largest and an f32 within 2^-6 are exact, smaller ones to 2^-22 and 2^-30 of the largest.
template <int DIGITS> struct Whole {
  static constexpr uint32_t kBits = 8 * DIGITS - 3;
  float up, scale;
  __device__ __forceinline__ explicit Whole(uint32_t largest) {      // the bits of the block's largest |x|
    const uint32_t e = max(largest >> 23, 30u);                      // below 2^-97 digits of 2^-126 and more are left
    const bool finite = largest < 0x7f800000u;                       // with an infinity or a NaN every product of the row is NaN
    up = finite ? __uint_as_float((254u + kBits - e) << 23) : 0.0f;
    scale = __uint_as_float(finite ? (e - kBits) << 23 : 0x7fc00000u);
  }
  // the digits of x as bytes, each with its sign, the lowest first: halves of their range are added, so that none borrows, and turned into signs
  __device__ __forceinline__ uint32_t digits(float x) const {
    constexpr uint32_t kHalves = DIGITS == 4 ? 0x00808080u : 0x00008080u;
    return ((uint32_t)(up == 0.0f ? 0 : __float2int_rn(x * up)) + kHalves) ^ kHalves;
  }
};

struct Product {
  const void* x;
  int64_t stride;                        // of x's rows
  const uint8_t* q;
  const __nv_bfloat16* scale;
  const uint8_t* zero;
  void* out;
  uint32_t rows, depth, cols;
  uint32_t kblocks, tiles;               // of the weight
  uint32_t rows_per_pass;                // rows of x that one pass over the weight serves (blockIdx.y)
  uint32_t chunk;                        // tiles between two barriers
  uint32_t per_cta;                      // blocks of k of a CTA of a cluster
  FastDiv by_per_cta;
  uint32_t tiles_each, tiles_over;       // tiles of a cluster; the first tiles_over clusters have one more
  int out_f32;
};

// 128 values of k of 16 columns as a lane has them: the codes of two columns (g and g + 8 of the tile), 32 values of k each, and these columns' scales and
// zero points
template <int PER_GROUP, bool ZERO> struct Block {
  uint4 lower, upper;
  uint16_t scale[2][PER_GROUP];
  uint8_t zero[2][PER_GROUP];
  __device__ __forceinline__ void load(const Product& p, uint32_t unit, uint32_t lane) {
    const uint4* codes = reinterpret_cast<const uint4*>(p.q + (uint64_t)unit * 1024) + lane;
    lower = __ldg(codes);
    upper = __ldg(codes + 32);
    const uint16_t* s = reinterpret_cast<const uint16_t*>(p.scale) + (uint64_t)unit * (16 * PER_GROUP) + (lane >> 2) * PER_GROUP;
    vector(scale[0], s);
    vector(scale[1], s + 8 * PER_GROUP);
    if (ZERO) {
      const uint8_t* z = p.zero + (uint64_t)unit * (16 * PER_GROUP) + (lane >> 2) * PER_GROUP;
      vector(zero[0], z);
      vector(zero[1], z + 8 * PER_GROUP);
    }
  }
  template <typename E> static __device__ __forceinline__ void vector(E (&to)[PER_GROUP], const E* from) {      // one load of 1 to 8 bytes
    constexpr int kBytes = PER_GROUP * sizeof(E);
    using W = std::conditional_t<kBytes == 1, uint8_t, std::conditional_t<kBytes == 2, uint16_t, std::conditional_t<kBytes == 4, uint32_t, uint2>>>;
    const W w = __ldg(reinterpret_cast<const W*>(from));
    memcpy(to, &w, kBytes);
  }
};

// DIGITS: 0 takes a bf16 x as it is, 3 and 4 take x as whole numbers; MT: sets of 8 columns of the instruction.  The CTAs of a cluster split k; a cluster has a
// run of the weight's tiles, `chunk` of them at a time.  A CTA's blocks of a chunk, tile after tile, are cut evenly over its eight warps wherever the cut
// falls: a warp reads one run of memory, blocks ahead of the one that it computes, and leaves its sum of each tile (or part of one) in shared
// memory.  They meet behind one barrier a chunk.  (A tile per warp leaves SMs with four CTAs beside others with three; a tile split over a CTA's warps has a
// barrier for every 16 columns: 2048 x 65536 20.1 and 23.6 us where this took 19.8.  Sixteen warps a CTA repeat more of what every warp does once: 20.7.)
template <typename TX, int DIGITS, int MT, int PER_GROUP, bool ZERO>
__global__ void __launch_bounds__(kThreads, DIGITS == 0 && MT == 4 ? 1 : 2) int4_product_kernel(const Product p) {
  grid_wait();
  constexpr int kParts = DIGITS ? DIGITS : 1;      // columns of the instruction that a row of x takes, the first with its uppermost digits
  constexpr int kAhead = MT <= 2 || DIGITS == 0 ? 4 : 2;      // blocks that a warp has on the way or in hand
  extern __shared__ __align__(16) uint8_t smem[];
  // of a chunk: the tile that a warp's run begins in (none: kNoTile), and the warps that have a tile's first and last block
  __shared__ uint32_t tiles_at[kWarps], first_warp[kMaxChunk], last_warp[kMaxChunk];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank(), id = blockIdx.x / ctas;
  const uint32_t kb0 = min(rank * p.per_cta, p.kblocks), kbn = min(p.per_cta, p.kblocks - kb0);
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t row0 = blockIdx.y * p.rows_per_pass, rows = min(p.rows_per_pass, p.rows - row0), columns = rows * kParts;
  const uint32_t first = id * p.tiles_each + min(id, p.tiles_over), last = first + p.tiles_each + (id < p.tiles_over ? 1 : 0);
  const uint32_t sum_floats = columns * 16, segments = segments_of(p.chunk);
  float* sums = reinterpret_cast<float*>(smem);                                     // [warp][segment][column][16 n]
  float* joined = sums + kWarps * segments * sum_floats;                            // a cluster's: [tile][column][16 n]
  // x: a column's bf16 values or digits, [column][k]; of the digits also, of every column, the scale of each block, and of each group the sum, for the weight's zero points
  uint8_t* xs = reinterpret_cast<uint8_t*>(joined + (ctas > 1 ? p.chunk * sum_floats : 0));
  const uint32_t pitch = DIGITS ? p.per_cta * 128 + kPadDigits : (p.per_cta * 128 + kPad) * 2;
  float* x_scales = reinterpret_cast<float*>(xs + columns * pitch);                 // [block][8 MT]
  int* x_sums = reinterpret_cast<int*>(x_scales + p.per_cta * 8 * MT);              // [block][group][8 MT]

  uint32_t unit = 0, run = 0, kb = 0;      // of this warp: the next block's number in the weight, blocks of the chunk, and where the first one is in its tile
  auto start_chunk = [&](uint32_t tile0, uint32_t count) {
    const uint32_t all = count * kbn, begin = all * warp / kWarps;
    run = all * (warp + 1) / kWarps - begin;
    const uint32_t tile = kbn ? begin / kbn : 0;
    kb = begin - tile * kbn;
    if (lane == 0) tiles_at[warp] = run ? tile : kNoTile;
    if (tid < count && kbn) {      // block b is of the last warp w whose run begins, at all * w / kWarps, no later
      first_warp[tid] = ((tid * kbn + 1) * kWarps + all - 1) / all - 1;
      last_warp[tid] = ((tid + 1) * kbn * kWarps + all - 1) / all - 1;
    }
    unit = (tile0 + tile) * p.kblocks + kb0 + kb;
  };
  start_chunk(first, min(p.chunk, last - first));
  Block<PER_GROUP, ZERO> ahead[kAhead];
  uint32_t asked = kb;      // the place in its tile of the block to be loaded next
  auto load = [&](Block<PER_GROUP, ZERO>& to) {
    to.load(p, unit, lane);
    ++unit;
    if (++asked == kbn) { asked = 0; unit += p.kblocks - kbn; }
  };
  auto load_ahead = [&] {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (run > (uint32_t)i) load(ahead[i]);
  };

  // This CTA's part of x.  It is asked for before the weight: behind four blocks of every warp's it would come 3000 cycles later.
  const TX* x = static_cast<const TX*>(p.x) + (int64_t)row0 * p.stride + kb0 * 128;
  const uint32_t depth = p.depth - min(p.depth, kb0 * 128);
  if constexpr (DIGITS != 0) {      // a warp takes a row's block at a time, a lane four values of it: two pairs of the eight that a word of codes meets
    const uint32_t word = lane / 2, at = word * 8 + (lane & 1) * 2;
    const bool pairs = ((reinterpret_cast<uintptr_t>(x) | (uint64_t)p.stride * sizeof(TX)) & (2 * sizeof(TX) - 1)) == 0;
    constexpr int kBatch = MT == 1 ? 2 : 4;      // row blocks on the way; the last one again where there is none
    const uint32_t all = rows * p.per_cta;
    float batch[kBatch][4];
    auto load_batch = [&](uint32_t i0) {
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const uint32_t i = min(i0 + q * kWarps, all - 1), m = p.by_per_cta.div(i), k = (i - m * p.per_cta) * 128 + at;
        const TX* from = x + (int64_t)m * p.stride + k;
        float (&v)[4] = batch[q];
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
          const TX* pair = from + j * 4;
          if (pairs && k + j * 4 + 1 < depth) {
            if constexpr (sizeof(TX) == 4) {
              const float2 w = *reinterpret_cast<const float2*>(pair);
              v[2 * j] = w.x; v[2 * j + 1] = w.y;
            } else {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(pair);
              v[2 * j] = __uint_as_float(w << 16); v[2 * j + 1] = __uint_as_float(w & 0xffff0000u);
            }
          } else {
            v[2 * j] = k + j * 4 < depth ? Elem<TX>::to_f32(pair[0]) : 0.0f;
            v[2 * j + 1] = k + j * 4 + 1 < depth ? Elem<TX>::to_f32(pair[1]) : 0.0f;
          }
        }
      }
    };
    load_batch(warp);
    load_ahead();
    for (uint32_t i0 = warp; i0 < all; i0 += kWarps * kBatch) {
      if (i0 != warp) load_batch(i0);
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const uint32_t i = min(i0 + q * kWarps, all - 1), m = p.by_per_cta.div(i), b = i - m * p.per_cta;
        float (&v)[4] = batch[q];
        uint32_t size = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) size = max(size, __float_as_uint(v[e]) & 0x7fffffffu);
        const Whole<kParts> whole(__reduce_max_sync(0xffffffffu, size));
        uint32_t d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = whole.digits(v[e]);
        // the j-th digits of k = 0, 4, 1, 5 of the word or of 2, 6, 3, 7: as a byte's lower and upper nibbles have the codes
        uint32_t part[4];
        const uint32_t l02 = __byte_perm(d[0], d[2], 0x5140), l13 = __byte_perm(d[1], d[3], 0x5140), u02 = __byte_perm(d[0], d[2], 0x7362), u13 = __byte_perm(d[1], d[3], 0x7362);
        part[0] = __byte_perm(l02, l13, 0x5410); part[1] = __byte_perm(l02, l13, 0x7632); part[2] = __byte_perm(u02, u13, 0x5410); part[3] = __byte_perm(u02, u13, 0x7632);
        constexpr int kLanes = 32 / PER_GROUP;
        uint32_t two[2] = {0, 0};      // a group's sums of two digits each, of 16 bits with their signs
        if constexpr (ZERO) {
#pragma unroll
          for (int j = 0; j < 2; ++j) two[j] = (uint32_t)__dp4a((int)part[2 * j], 0x01010101, 0) + ((uint32_t)__dp4a((int)part[2 * j + 1], 0x01010101, 0) << 16);
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1)
#pragma unroll
            for (int j = 0; j < 2; ++j) two[j] += __shfl_xor_sync(0xffffffffu, two[j], o);
        }
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          const uint32_t column = m * kParts + kParts - 1 - j;
          *reinterpret_cast<uint32_t*>(xs + column * pitch + b * 128 + (word % 4) * 32 + (word / 4) * 8 + (lane & 1) * 4) = part[j];
          if constexpr (ZERO) {
            const int lower = (int)(int16_t)two[j / 2], sum = j % 2 ? (int)(two[j / 2] - (uint32_t)lower) >> 16 : lower;
            if (lane % kLanes == 0) x_sums[(b * PER_GROUP + lane / kLanes) * (8 * MT) + column] = 16 * sum;
          }
          if (lane == 0) x_scales[b * (8 * MT) + column] = whole.scale * ((float)(1u << 8 * j) * 0.0625f);      // the codes are sixteen times theirs
        }
      }
    }
  } else {      // bf16, eight values at a time
    const bool whole = ((reinterpret_cast<uintptr_t>(x) | (uint64_t)p.stride * 2) & 15) == 0;
    // rows over the warps, and where there are fewer of them a row over several
    const uint32_t over = rows >= (uint32_t)kWarps ? 1 : rows > kWarps / 2 ? 1 : rows > kWarps / 4 ? 2 : rows > kWarps / 8 ? 4 : 8;
    for (uint32_t m = warp / over; m < rows; m += kWarps / over) {
      const uint16_t* row = reinterpret_cast<const uint16_t*>(x) + (int64_t)m * p.stride;
      uint8_t* to = xs + m * pitch;
#pragma unroll 4
      for (uint32_t k = (warp % over * 32 + lane) * 8; k < kbn * 128; k += over * 256) {
        if (whole && k + 8 <= depth) {
          copy16(shared_address(to + k * 2), row + k);
        } else {
          uint32_t w[4];
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) w[e] = (k + 2 * e < depth ? row[k + 2 * e] : 0u) | (k + 2 * e + 1 < depth ? (uint32_t)row[k + 2 * e + 1] << 16 : 0u);
          *reinterpret_cast<uint4*>(to + k * 2) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    load_ahead();
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncthreads();

  // a column of the instruction that is none of x's has another's values: nobody reads its sums
  const uint8_t* mine[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) mine[i] = xs + min(i * 8 + g, columns - 1) * pitch + t * (DIGITS ? 32 : 16);
  for (uint32_t tile0 = first; tile0 < last; tile0 += p.chunk) {
    const uint32_t count = min(p.chunk, last - tile0);
    float total[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) total[i][0] = total[i][1] = total[i][2] = total[i][3] = 0.0f;
    float* own = sums + warp * segments * sum_floats + t * 32 + g;
    auto multiply = [&](const Block<PER_GROUP, ZERO>& w, bool ends) {
      const uint32_t lo[4] = {w.lower.x, w.lower.y, w.lower.z, w.lower.w}, up[4] = {w.upper.x, w.upper.y, w.upper.z, w.upper.w};
      constexpr int kRun = 4 / PER_GROUP;                                   // 32-value runs of a group
      if constexpr (DIGITS != 0) {
        int sum[MT][4];
        float of_block[MT][4];
        uint4 x4[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          x4[i][0] = *reinterpret_cast<const uint4*>(mine[i] + kb * 128);
          x4[i][1] = *reinterpret_cast<const uint4*>(mine[i] + kb * 128 + 16);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int of = c / kRun;
          if (c % kRun == 0)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              sum[i][0] = sum[i][1] = sum[i][2] = sum[i][3] = kWhole;
              if (ZERO) {      // what the zero points take off beside the eight that the codes are less, in the sum from its start
                const int2 s = *reinterpret_cast<const int2*>(x_sums + (kb * PER_GROUP + of) * (8 * MT) + i * 8 + t * 2);
                const int z_lo = 8 - (int)w.zero[0][of], z_up = 8 - (int)w.zero[1][of];
                sum[i][0] += z_lo * s.x; sum[i][1] += z_lo * s.y; sum[i][2] += z_up * s.x; sum[i][3] += z_up * s.y;
              }
            }
          // codes u as bytes of 16 (u - 8): a nibble in the upper half of its byte with its highest bit turned
          const uint32_t a0 = (lo[c] << 4 & 0xf0f0f0f0u) ^ 0x80808080u, a1 = (up[c] << 4 & 0xf0f0f0f0u) ^ 0x80808080u;
          const uint32_t a2 = (lo[c] & 0xf0f0f0f0u) ^ 0x80808080u, a3 = (up[c] & 0xf0f0f0f0u) ^ 0x80808080u;
#pragma unroll
          for (int i = 0; i < MT; ++i) mma(sum[i], a0, a1, a2, a3, c % 2 ? x4[i][c / 2].z : x4[i][c / 2].x, c % 2 ? x4[i][c / 2].w : x4[i][c / 2].y);
          if (c % kRun == kRun - 1) {
            const float s_lo = __uint_as_float((uint32_t)w.scale[0][of] << 16), s_up = __uint_as_float((uint32_t)w.scale[1][of] << 16);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) {      // exact until it meets the scale
                const float whole = __int_as_float(sum[i][e]) - kWholeValue, s = e < 2 ? s_lo : s_up;
                of_block[i][e] = of == 0 ? s * whole : fmaf(s, whole, of_block[i][e]);
              }
          }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const float2 s = *reinterpret_cast<const float2*>(x_scales + kb * (8 * MT) + i * 8 + t * 2);
#pragma unroll
          for (int e = 0; e < 4; ++e) total[i][e] = fmaf(e & 1 ? s.y : s.x, of_block[i][e], total[i][e]);
        }
      } else {
        constexpr int kChains = MT == 1 && PER_GROUP == 1 ? 2 : 1;            // sums under way at once where one would wait for itself
        float sum[MT][kChains][4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int of = c / kRun, chain = c % kChains;
          uint32_t bias_lo = 0x43084308u, bias_up = 0x43084308u;
          if (ZERO) {
            bias_lo = (0x4300u | w.zero[0][of]) * 0x10001u;
            bias_up = (0x4300u | w.zero[1][of]) * 0x10001u;
          }
          const uint32_t a[8] = {pair_of<0>(lo[c], bias_lo), pair_of<0>(up[c], bias_up), pair_of<4>(lo[c], bias_lo), pair_of<4>(up[c], bias_up),
                                 pair_of<8>(lo[c], bias_lo), pair_of<8>(up[c], bias_up), pair_of<12>(lo[c], bias_lo), pair_of<12>(up[c], bias_up)};
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const uint4 x4 = *reinterpret_cast<const uint4*>(mine[i] + kb * 256 + c * 64);
            if (c % kRun < kChains) mma_from_zero(sum[i][chain], a[0], a[1], a[2], a[3], x4.x, x4.y);
            else mma(sum[i][chain], a[0], a[1], a[2], a[3], x4.x, x4.y);
            mma(sum[i][chain], a[4], a[5], a[6], a[7], x4.z, x4.w);
          }
          if (c % kRun == kRun - 1) {
            const float s_lo = __uint_as_float((uint32_t)w.scale[0][of] << 16), s_up = __uint_as_float((uint32_t)w.scale[1][of] << 16);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) total[i][e] = fmaf(e < 2 ? s_lo : s_up, kChains == 2 ? sum[i][0][e] + sum[i][kChains - 1][e] : sum[i][0][e], total[i][e]);
          }
        }
      }
      if (++kb == kbn || ends) {      // a tile's end, or the run's
        kb = 0;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (i * 8 + (e & 1) + t * 2 < columns) own[i * 128 + (e & 1) * 16 + (e & 2) * 4] = total[i][e];
            total[i][e] = 0.0f;
          }
        own += sum_floats;
      }
    };
    for (uint32_t b = run; b > 0;) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (b > 0) {
          multiply(ahead[i], b == 1);
          if (b > (uint32_t)kAhead) load(ahead[i]);
          --b;
        }
    }
    __syncthreads();
    // the sums of a tile's entries over the warps that have a part of it: ENTRIES of them, 16 apart
    auto over_warps = [&](uint32_t j, uint32_t at, auto& y) {
      constexpr int kEntries = sizeof(y) / sizeof(float);
#pragma unroll
      for (int e = 0; e < kEntries; ++e) y[e] = 0.0f;
      if (kbn) {
        const uint32_t end = last_warp[j];
#pragma unroll 2
        for (uint32_t w = first_warp[j]; w <= end; ++w) {
          const uint32_t tile = tiles_at[w];
          const float* from = sums + (w * segments + (tile == kNoTile ? 0 : j - tile)) * sum_floats + at;
#pragma unroll
          for (int e = 0; e < kEntries; ++e) {
            const float s = from[e * 16];
            y[e] += tile == kNoTile ? 0.0f : s;
          }
        }
      }
    };
    auto write = [&](uint32_t j, uint32_t m, uint32_t n, float y) {
      const uint32_t col = (tile0 + j) * 16 + n;
      if (col >= p.cols) return;
      const int64_t at = (int64_t)(row0 + m) * p.cols + col;
      if (p.out_f32) static_cast<float*>(p.out)[at] = y;
      else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
    };
    const uint32_t outputs = rows * 16;      // of a tile; a term's and a row's sums lie 16 apart
    if (ctas == 1) {
      for (uint32_t i = tid; i < count * outputs; i += kThreads) {
        const uint32_t j = i / outputs, m = (i - j * outputs) / 16, n = i % 16;
        float of[kParts], y = 0.0f;
        over_warps(j, m * (kParts * 16) + n, of);
#pragma unroll
        for (int part = kParts - 1; part >= 0; --part) y += of[part];      // the small ones first
        write(j, m, n, y);
      }
    } else {
      const uint32_t fours = (columns + 3) / 4 * 16;      // of a tile, four columns' sums at a time
      for (uint32_t i = tid; i < count * fours; i += kThreads) {
        const uint32_t j = i / fours, column = (i - j * fours) / 16 * 4, at = column * 16 + i % 16;
        float of[4];
        over_warps(j, at, of);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          if (column + e < columns) joined[j * sum_floats + at + e * 16] = of[e];
      }
      cluster.sync();
      for (uint32_t i = rank * kThreads + tid; i < count * outputs; i += ctas * kThreads) {      // each rank finishes a part
        const uint32_t j = i / outputs, m = (i - j * outputs) / 16, n = i % 16;
        float y = 0.0f;
#pragma unroll
        for (int term = kParts - 1; term >= 0; --term) {
          float of[kMaxCluster];
#pragma unroll
          for (uint32_t r = 0; r < kMaxCluster; ++r) of[r] = r < ctas ? *cluster.map_shared_rank(joined + j * sum_floats + (m * kParts + term) * 16 + n, r) : 0.0f;
#pragma unroll
          for (uint32_t r = 0; r < kMaxCluster; ++r) y += of[r];
        }
        write(j, m, n, y);
      }
    }
    const uint32_t next = tile0 + p.chunk;
    if (ctas > 1) cluster.sync();                 // nobody leaves or writes its sums again while they are read
    else if (next < last) __syncthreads();
    if (next < last) {
      start_chunk(next, min(p.chunk, last - next));
      asked = kb;
      load_ahead();
    }
  }
}

template <int DIGITS, int MT, int PER_GROUP> size_t shared_bytes(uint32_t columns, uint32_t kblocks_of_cta, uint32_t chunk, uint32_t ctas) {
  const size_t sums = (size_t)columns * 64 * (kWarps * segments_of(chunk) + (ctas > 1 ? chunk : 0));
  return sums + (DIGITS ? (size_t)columns * (kblocks_of_cta * 128 + kPadDigits) + (size_t)kblocks_of_cta * 32 * MT * (1 + PER_GROUP) : (size_t)columns * (kblocks_of_cta * 128 + kPad) * 2);
}

constexpr size_t kMaxShared = 226 * 1024;      // of 227 KB, beside the kernel's own few bytes

template <typename TX, int DIGITS, int MT, int PER_GROUP, bool ZERO> int launch_product(Product p, cudaStream_t st) {
  constexpr uint32_t kParts = DIGITS ? DIGITS : 1;
  auto kernel = int4_product_kernel<TX, DIGITS, MT, PER_GROUP, ZERO>;
  uint32_t ctas = 1, per_pass = std::min<uint32_t>(p.rows, 8 * MT / kParts), clusters, bytes;
  const uint32_t sms = sm_count(), force = env_switch("PB_INT4_CTAS", 0), force_sm = env_switch("PB_INT4_PERSM", 0);
  // x in shared memory: split k over a cluster, and where that is not enough serve fewer rows with a pass.  Few tiles of a long contraction (`few`) are split, too, us, one
  // CTA | by the rule: one f32 row, 16384 x 256 10.1 | 4.1, 16384 x 2048 10.3 | 6.9, 8192 x 2048 6.2 | 5.5, 8192 x 4096 7.9 | 6.7; 8 bf16 rows, 8192 x 2048 7.3 | 6.5; at the
  // rule's edge it takes longer, 4096 x 2048 4.1 | 4.4.  So is x where making its digits takes a CTA more than its products (`heavy`): 8 f32 rows, 2048 x 256 6.8 | 4.9,
  // 2048 x 2048 6.9 | 6.4, 2048 x 4096 7.7 | 7.7; of four rows it takes longer where the contraction is short, 1024 x 2048 3.4 | 4.6.
  while (true) {
    const uint32_t per = (p.kblocks + ctas - 1) / ctas;
    uint32_t room = sms / ctas;      // clusters that are resident at once with a CTA an SM; 33 of four and 15 of eight CTAs on 148 SMs
    if (ctas >= 4) room -= room / (ctas == 4 ? 9 : 6);
    const uint64_t x_bytes = (uint64_t)per_pass * kParts * per * (DIGITS ? 128 : 256);
    // two CTAs on an SM where one of them has more to read of the weight than of x
    uint32_t per_sm = force_sm ? force_sm : (uint64_t)p.tiles * p.kblocks * 1024 / (2 * sms) >= 2 * x_bytes ? 2 : 1;
    size_t need;
    while (true) {
      clusters = std::max<uint32_t>(1, std::min<uint32_t>(p.tiles, room * per_sm));
      p.chunk = std::min<uint32_t>(kMaxChunk, (p.tiles + clusters - 1) / clusters);
      need = shared_bytes<DIGITS, MT, PER_GROUP>(per_pass * kParts, per, p.chunk, ctas);
      if (per_sm == 1 || per_sm * (need + 1024) <= 228 * 1024) break;
      --per_sm;
    }
    bytes = (uint32_t)std::min<size_t>(need, kMaxShared + 1);
    const bool few = p.tiles * ctas < 4 * sms && p.kblocks > ctas * kWarps * 2;
    const bool heavy = DIGITS && per_pass >= 4 && per_pass > MT * ((p.tiles + clusters - 1) / clusters);      // more digits to make than products
    if (bytes <= kMaxShared && (force ? ctas == force : ctas == kMaxCluster || !(few || heavy))) break;
    if (ctas < kMaxCluster) ctas *= 2;
    else if (per_pass > 1) { per_pass /= 2; ctas = 1; }
    else return fail(PB_ERR_UNSUPPORTED, "pb_int4_product: a contraction of %u does not fit", p.depth);
  }
  p.rows_per_pass = per_pass;
  p.per_cta = (p.kblocks + ctas - 1) / ctas;
  p.by_per_cta = FastDiv(p.per_cta);
  p.tiles_each = p.tiles / clusters;
  p.tiles_over = p.tiles % clusters;
  static std::atomic<uint64_t> allowed{0};      // devices on which this kernel may have so much
  int device = 0;
  PB_CUDA_TRY(cudaGetDevice(&device));
  if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
    PB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxShared));
    if (device < 64) allowed.fetch_or(1ull << device, std::memory_order_relaxed);
  }
  const uint32_t passes = (p.rows + per_pass - 1) / per_pass;
  if (passes > 65535) return fail(PB_ERR_UNSUPPORTED, "pb_int4_product: %u rows", p.rows);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(clusters * ctas, passes);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = ctas; attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = 2;
  cudaLaunchKernelEx(&config, kernel, p);
  PB_LAUNCH_CHECK("int4_product_kernel");
  return PB_OK;
}

template <typename TX, int DIGITS, int MT> int launch_of(const Product& p, int per_group, cudaStream_t st) {
  if (p.zero)
    return per_group == 1 ? launch_product<TX, DIGITS, MT, 1, true>(p, st) : per_group == 2 ? launch_product<TX, DIGITS, MT, 2, true>(p, st) : launch_product<TX, DIGITS, MT, 4, true>(p, st);
  return per_group == 1 ? launch_product<TX, DIGITS, MT, 1, false>(p, st) : per_group == 2 ? launch_product<TX, DIGITS, MT, 2, false>(p, st) : launch_product<TX, DIGITS, MT, 4, false>(p, st);
}

int check_int4(const char* who, int64_t depth, int64_t cols, int group) {
  if (group != 32 && group != 64 && group != 128) return fail(PB_ERR_BAD_GRID, "%s: groups of %d (32, 64 or 128)", who, group);
  if (depth <= 0 || cols <= 0 || depth > 0x7fffff00ll || cols > 0x3fffffffll) return fail(PB_ERR_BAD_SHAPE, "%s: depth=%lld cols=%lld", who, (long long)depth, (long long)cols);
  return PB_OK;
}

}  // namespace
}  // namespace pb

using namespace pb;

extern "C" int pb_quantize_int4(const void* w, int dtype, int64_t depth, int64_t cols, int group, uint8_t* q, void* scale, uint8_t* zero, void* stream) {
  if (!w || !q || !scale) return fail(PB_ERR_NULL_POINTER, "pb_quantize_int4: null argument");
  if (dtype != PB_F32 && dtype != PB_BF16) return fail(PB_ERR_BAD_DTYPE, "pb_quantize_int4: dtype %d", dtype);
  if (int s = check_int4("pb_quantize_int4", depth, cols, group)) return s;
  if (off_by(q, 16) || off_by(w, dtype == PB_F32 ? 4 : 2) || off_by(scale, 2)) return fail(PB_ERR_MISALIGNED, "pb_quantize_int4: q 16 bytes, w and scale their types");
  const uint32_t kblocks = (uint32_t)((depth + 127) / 128), col_blocks = (uint32_t)((cols + kQuantCols - 1) / kQuantCols);
  if (col_blocks > 65535) return fail(PB_ERR_UNSUPPORTED, "pb_quantize_int4: %lld columns", (long long)cols);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(kblocks, col_blocks);
  auto* words = reinterpret_cast<uint32_t*>(q);
  auto* s = static_cast<__nv_bfloat16*>(scale);
  const int per_group = 128 / group;
  auto launch = [&](auto* in, auto cols_of_thread) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(in)>>;
    constexpr int kCols = decltype(cols_of_thread)::value;
    if (zero) launch_behind(quantize_int4_kernel<T, true, kCols>, grid, kQuantThreads, 0, st, in, depth, cols, per_group, kblocks, words, s, zero);
    else launch_behind(quantize_int4_kernel<T, false, kCols>, grid, kQuantThreads, 0, st, in, depth, cols, per_group, kblocks, words, s, zero);
  };
  const bool pairs = cols % 2 == 0 && (reinterpret_cast<uintptr_t>(w) & 3) == 0;
  if (dtype == PB_F32) launch(static_cast<const float*>(w), std::integral_constant<int, 1>());
  else if (pairs) launch(static_cast<const __nv_bfloat16*>(w), std::integral_constant<int, 2>());
  else launch(static_cast<const __nv_bfloat16*>(w), std::integral_constant<int, 1>());
  PB_LAUNCH_CHECK("quantize_int4_kernel");
  return PB_OK;
}

extern "C" int pb_dequantize_int4(const uint8_t* q, const void* scale, const uint8_t* zero, int64_t depth, int64_t cols, int group, void* out, int dtype, void* stream) {
  if (!q || !scale || !out) return fail(PB_ERR_NULL_POINTER, "pb_dequantize_int4: null argument");
  if (dtype != PB_F32 && dtype != PB_BF16) return fail(PB_ERR_BAD_DTYPE, "pb_dequantize_int4: dtype %d", dtype);
  if (int s = check_int4("pb_dequantize_int4", depth, cols, group)) return s;
  if (off_by(q, 16) || off_by(out, dtype == PB_F32 ? 4 : 2) || off_by(scale, 2)) return fail(PB_ERR_MISALIGNED, "pb_dequantize_int4: q 16 bytes, scale and out their types");
  const uint32_t kblocks = (uint32_t)((depth + 127) / 128), col_blocks = (uint32_t)((cols + kQuantCols - 1) / kQuantCols);
  if (col_blocks > 65535) return fail(PB_ERR_UNSUPPORTED, "pb_dequantize_int4: %lld columns", (long long)cols);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(kblocks, col_blocks);
  const auto* words = reinterpret_cast<const uint32_t*>(q);
  const auto* s = static_cast<const __nv_bfloat16*>(scale);
  auto launch = [&](auto kernel, auto* to) { launch_behind(kernel, grid, kQuantThreads, 0, st, words, s, zero, depth, cols, 128 / group, kblocks, to); };
  if (dtype == PB_F32) launch(dequantize_int4_kernel<float, 1>, static_cast<float*>(out));
  else if (cols % 2 == 0 && (reinterpret_cast<uintptr_t>(out) & 3) == 0) launch(dequantize_int4_kernel<__nv_bfloat16, 2>, static_cast<__nv_bfloat16*>(out));
  else launch(dequantize_int4_kernel<__nv_bfloat16, 1>, static_cast<__nv_bfloat16*>(out));
  PB_LAUNCH_CHECK("dequantize_int4_kernel");
  return PB_OK;
}

extern "C" int pb_int4_product(const void* x, int x_dtype, int64_t rows, int64_t depth, int64_t stride, const uint8_t* q, const void* scale, const uint8_t* zero, int group,
                               int64_t cols, void* out, int out_dtype, void* stream) {
  if (int s = check_int4("pb_int4_product", depth, cols, group)) return s;
  if (rows < 0 || rows > 0x7fffffffll || stride < 0) return fail(PB_ERR_BAD_SHAPE, "pb_int4_product: rows=%lld stride=%lld", (long long)rows, (long long)stride);
  if ((x_dtype != PB_F32 && x_dtype != PB_BF16) || (out_dtype != PB_F32 && out_dtype != PB_BF16)) return fail(PB_ERR_BAD_DTYPE, "pb_int4_product: dtypes %d, %d", x_dtype, out_dtype);
  if (rows == 0) return PB_OK;
  if (!x || !q || !scale || !out) return fail(PB_ERR_NULL_POINTER, "pb_int4_product: null argument");
  const int per_group = 128 / group;      // a lane loads as many scales, and zero points, at once
  if (off_by(q, 16) || off_by(scale, 2 * per_group) || off_by(zero, per_group) || off_by(x, x_dtype == PB_F32 ? 4 : 2) || off_by(out, out_dtype == PB_F32 ? 4 : 2))
    return fail(PB_ERR_MISALIGNED, "pb_int4_product: q 16, scale %d and zero %d bytes, x and out their types", 2 * per_group, per_group);
  if ((uint64_t)((cols + 15) / 16) * ((depth + 127) / 128) > 0x7fffffffull) return fail(PB_ERR_BAD_SHAPE, "pb_int4_product: depth=%lld cols=%lld", (long long)depth, (long long)cols);
  Product p{x, stride, q, static_cast<const __nv_bfloat16*>(scale), zero, out, (uint32_t)rows, (uint32_t)depth, (uint32_t)cols, (uint32_t)((depth + 127) / 128),
            (uint32_t)((cols + 15) / 16), 0, 0, 0, FastDiv(), 0, 0, out_dtype == PB_F32};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (x_dtype == PB_F32) return rows <= 2 ? launch_of<float, 4, 1>(p, per_group, st) : rows <= 4 ? launch_of<float, 4, 2>(p, per_group, st) : launch_of<float, 4, 4>(p, per_group, st);
  // A bf16 x as it is or in digits, us, 2048 values deep: 2048 columns 2.97 | 3.22 (one row) and 3.06 | 3.98 (two), 8192 columns 4.80 | 4.38 and 5.43 | 5.26 (with zero
  // points, 8192 deep and 2048 columns, 5.70 | 6.44), 65536 columns 18.8 | 15.6 and 19.4 | 17.0, four rows 20.1 | 21.7: making digits is made good by many columns
  if (rows <= 2 && (int64_t)p.tiles * p.kblocks >= 16384) return launch_of<__nv_bfloat16, 3, 1>(p, per_group, st);
  return rows <= 8 ? launch_of<__nv_bfloat16, 0, 1>(p, per_group, st) : rows <= 16 ? launch_of<__nv_bfloat16, 0, 2>(p, per_group, st) : launch_of<__nv_bfloat16, 0, 4>(p, per_group, st);
}
