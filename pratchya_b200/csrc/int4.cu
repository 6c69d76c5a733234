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

namespace pb {
namespace {

namespace cg = cooperative_groups;

// ---- the quantizer -----------------------------------------------------------------------------------------------------
constexpr int kQuantThreads = 256, kQuantCols = 64;      // 128 x 64 weights a CTA, 32 values of one column a thread

// the word that holds eight codes, the i-th of them k = i
__device__ __forceinline__ uint32_t pack_codes(const uint32_t (&u)[8]) {
  return u[0] | u[2] << 4 | u[4] << 8 | u[6] << 12 | u[1] << 16 | u[3] << 20 | u[5] << 24 | u[7] << 28;
}
__device__ __forceinline__ uint32_t code_at(uint32_t word, int i) { return word >> (4 * (i / 2 + 4 * (i % 2))) & 15u; }
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// ZERO: scale = bf16((max(w, 0) - min(w, 0)) / 15), zero = rint(-min / scale), u = rint(w / scale) + zero, both within 0..15;
// otherwise scale = bf16(max|w| / 7), u = rint(w / scale) within -8..7, plus 8.  A group of nothing but zeros has scale 0.
// The scale is rounded before the codes are taken: they are the nearest ones for the scale that is stored.
// A group that holds a NaN or an infinity has a scale that is no finite number.
template <typename T, bool ZERO>
__global__ void __launch_bounds__(kQuantThreads) quantize_int4_kernel(const T* __restrict__ w, int64_t depth, int64_t cols, int per_group, uint32_t kblocks,
                                                                      uint32_t* __restrict__ q, __nv_bfloat16* __restrict__ scale, uint8_t* __restrict__ zero) {
  grid_wait();
  __shared__ float lows[4][kQuantCols], highs[4][kQuantCols];
  __shared__ __align__(16) uint32_t staged[4 * 256];
  const uint32_t col = threadIdx.x % kQuantCols, c = threadIdx.x / kQuantCols;      // a warp has 32 neighbouring columns
  const uint32_t kb = blockIdx.x;
  const int64_t n = (int64_t)blockIdx.y * kQuantCols + col, k0 = (int64_t)kb * 128 + c * 32;
  float v[32];
  float low = 0.0f, high = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i] = n < cols && k0 + i < depth ? Elem<T>::to_f32(w[(k0 + i) * cols + n]) : 0.0f;
    if (ZERO) {
      low = -max_nan(-low, -v[i]);
      high = max_nan(high, v[i]);
    } else {
      high = max_nan(high, fabsf(v[i]));
    }
  }
  lows[c][col] = low;
  highs[c][col] = high;
  __syncthreads();
  const int quarters = 4 / per_group;      // 32-value runs of a group
  const int first = (int)c / quarters * quarters;
  for (int o = 0; o < quarters; ++o) {
    if (ZERO) low = -max_nan(-low, -lows[first + o][col]);
    high = max_nan(high, highs[first + o][col]);
  }
  const float s = __bfloat162float(__float2bfloat16_rn(ZERO ? __fdiv_rn(__fsub_rn(high, low), 15.0f) : __fdiv_rn(high, 7.0f)));
  const bool some = s != 0.0f;
  const float z = !ZERO ? 8.0f : some ? fminf(fmaxf(rintf(__fdiv_rn(-low, s)), 0.0f), 15.0f) : 0.0f;
  const uint32_t half = col % 16 / 8, g = col % 8, tile = col / 16;
#pragma unroll
  for (uint32_t t = 0; t < 4; ++t) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float r = some ? rintf(__fdiv_rn(v[t * 8 + i], s)) : 0.0f;
      u[i] = (uint32_t)(int)(ZERO ? fminf(fmaxf(r + z, 0.0f), 15.0f) : fminf(fmaxf(r, -8.0f), 7.0f) + 8.0f);
    }
    staged[tile * 256 + half * 128 + (g * 4 + t) * 4 + c] = pack_codes(u);
  }
  const int64_t tiles = (cols + 15) / 16, at = (int64_t)blockIdx.y * 4 + tile;
  if (at < tiles && (int)c == first) {
    const int64_t i = ((at * kblocks + kb) * 16 + col % 16) * per_group + c / quarters;
    scale[i] = __float2bfloat16_rn(s);
    if (ZERO) zero[i] = (uint8_t)z;
  }
  __syncthreads();
  const uint32_t part = threadIdx.x / 64;      // a tile's 1024 bytes, 16 a thread
  const int64_t a = (int64_t)blockIdx.y * 4 + part;
  if (a < tiles)
    reinterpret_cast<uint4*>(q + (a * kblocks + kb) * 256)[threadIdx.x % 64] = reinterpret_cast<const uint4*>(staged + part * 256)[threadIdx.x % 64];
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) dequantize_int4_kernel(const uint32_t* __restrict__ q, const __nv_bfloat16* __restrict__ scale, const uint8_t* __restrict__ zero,
                                                                        int64_t depth, int64_t cols, int per_group, uint32_t kblocks, T* __restrict__ w) {
  grid_wait();
  const uint32_t col = threadIdx.x % kQuantCols, c = threadIdx.x / kQuantCols, kb = blockIdx.x;
  const int64_t n = (int64_t)blockIdx.y * kQuantCols + col, k0 = (int64_t)kb * 128 + c * 32;
  if (n >= cols) return;
  const int64_t tile = n / 16 * kblocks + kb, i = (tile * 16 + n % 16) * per_group + c * per_group / 4;
  const float s = __bfloat162float(scale[i]), z = zero ? (float)zero[i] : 8.0f;
  const uint32_t* words = q + tile * 256 + (n % 16 / 8) * 128 + (n % 8) * 16 + c;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t word = words[t * 4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + t * 8 + j < depth) w[(k0 + t * 8 + j) * cols + n] = Elem<T>::from_f32(s * ((float)code_at(word, j) - z));
  }
}

// ---- products of few rows ------------------------------------------------------------------------------------------------
// A warp's matrix instruction m16n8k16 takes 16 columns n of the weight as its rows and 8 rows of x as its columns: the weight, of which there is much,
// fills it, and x, of which there is little, is what may be padded.  Codes become bf16 by their bits (0x4300 | u is 128 + u) and are taken less
// 128 + zero, both exact; sums over a group are f32, and meet the group's scale in f32.  An f32 x goes as three bf16 terms, 8 bits of its 24 each, in
// three columns of the instruction whose sums meet at the end: for one or two rows they cost nothing.
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kStages = 4;             // tiles that a warp has on the way
constexpr int kPad = 32;               // values behind a row of x in shared memory: neighbouring rows' 64 bytes then lie in other banks
constexpr int kMaxCluster = 8;

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
  return sub_bf16x2((word >> SHIFT & 0x000f000fu) | 0x43004300u, bias);
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t to, const void* from) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 8 bits of an f32 after another: x = hi + mid + lo (but for the last bits of numbers below 2^-110); an infinity or a NaN is hi alone
__device__ __forceinline__ void three_terms(float x, uint16_t& hi, uint16_t& mid, uint16_t& lo) {
  const uint32_t h = __float_as_uint(x) & 0xffff0000u;
  hi = x != x ? 0x7fc0 : (uint16_t)(h >> 16);
  const float r = (h & 0x7f800000u) == 0x7f800000u ? 0.0f : x - __uint_as_float(h);
  const uint32_t m = __float_as_uint(r) & 0xffff0000u;
  mid = (uint16_t)(m >> 16);
  lo = (uint16_t)(__float_as_uint(r - __uint_as_float(m)) >> 16);
}

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
  int out_f32;
};

// A warp's ring of tiles: codes, scales and zero points of PER_GROUP groups
template <int PER_GROUP, bool ZERO> struct Stage {
  static constexpr int kScales = 1024, kZeros = kScales + 32 * PER_GROUP, kBytes = kZeros + (ZERO ? 16 * PER_GROUP : 0);
};

// MT: sets of 8 columns.  A CTA's warps share a tile's 16 columns n and split its 128-blocks of k; the CTAs of a cluster split k before that.
// Each warp copies its tiles ahead into a ring of its own.
template <typename TX, int MT, int PER_GROUP, bool ZERO>
__global__ void __launch_bounds__(kThreads) int4_product_kernel(const Product p) {
  grid_wait();
  using S = Stage<PER_GROUP, ZERO>;
  constexpr int kTerms = sizeof(TX) == 4 ? 3 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const uint32_t per = (p.kblocks + ctas - 1) / ctas, kb0 = min(rank * per, p.kblocks), kbn = min(per, p.kblocks - kb0);
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t row0 = blockIdx.y * p.rows_per_pass, rows = min(p.rows_per_pass, p.rows - row0), columns = rows * kTerms;
  uint8_t* ring = smem + warp * (kStages * S::kBytes);
  float* sums = reinterpret_cast<float*>(smem + kWarps * kStages * S::kBytes);      // [warps][16][8 MT]; the CTA's at its beginning
  uint16_t* xs = reinterpret_cast<uint16_t*>(sums + kWarps * 16 * 8 * MT);
  const uint32_t pitch = per * 128 + kPad;

  // the tiles of this warp: tile after tile of the grid's stride, in each its blocks of k
  uint32_t ahead_tile = blockIdx.x / ctas, ahead_kb = warp;
  const uint32_t tile_step = gridDim.x / ctas;
  const uint32_t ring_at = shared_address(ring);
  auto ask = [&](uint32_t stage) {
    while (ahead_kb >= kbn && ahead_tile < p.tiles) { ahead_kb = warp; ahead_tile += tile_step; if (warp >= kbn) ahead_tile = p.tiles; }
    if (ahead_tile < p.tiles) {
      const uint64_t unit = (uint64_t)ahead_tile * p.kblocks + kb0 + ahead_kb;
      const uint32_t to = ring_at + stage * S::kBytes;
      copy16(to + lane * 16, p.q + unit * 1024 + lane * 16);
      copy16(to + 512 + lane * 16, p.q + unit * 1024 + 512 + lane * 16);
      if (lane < 8 * PER_GROUP) copy4(to + S::kScales + lane * 4, reinterpret_cast<const uint8_t*>(p.scale) + unit * (32 * PER_GROUP) + lane * 4);
      if (ZERO && lane < 4 * PER_GROUP) copy4(to + S::kZeros + lane * 4, p.zero + unit * (16 * PER_GROUP) + lane * 4);
      ahead_kb += kWarps;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) ask(s);

  // this CTA's part of x, as bf16
  const TX* x = static_cast<const TX*>(p.x) + (int64_t)row0 * p.stride;
  for (uint32_t m = 0; m < rows; ++m)
    for (uint32_t k = tid; k < kbn * 128; k += kThreads) {
      const uint32_t at = kb0 * 128 + k;
      if constexpr (kTerms == 3) {
        uint16_t* to = xs + (uint64_t)(m * 3) * pitch + k;
        three_terms(at < p.depth ? x[m * p.stride + at] : 0.0f, to[0], to[pitch], to[2 * pitch]);
      } else {
        xs[(uint64_t)m * pitch + k] = at < p.depth ? reinterpret_cast<const uint16_t*>(x)[m * p.stride + at] : (uint16_t)0;
      }
    }
  __syncthreads();

  uint32_t stage = 0;
  for (uint32_t tile = blockIdx.x / ctas; tile < p.tiles; tile += tile_step) {
    float total[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) total[i][0] = total[i][1] = total[i][2] = total[i][3] = 0.0f;
    for (uint32_t kb = warp; kb < kbn; kb += kWarps) {
      ask((stage + kStages - 1) % kStages);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const uint8_t* in = ring + stage * S::kBytes;
      const uint4 lower = *reinterpret_cast<const uint4*>(in + lane * 16), upper = *reinterpret_cast<const uint4*>(in + 512 + lane * 16);
      const uint16_t* scales = reinterpret_cast<const uint16_t*>(in + S::kScales);
      const uint32_t lo[4] = {lower.x, lower.y, lower.z, lower.w}, up[4] = {upper.x, upper.y, upper.z, upper.w};
      float sum[MT][4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        constexpr int kRun = 4 / PER_GROUP;      // 32-value runs of a group
        const int of = c / kRun;
        uint32_t bias_lo = 0x43084308u, bias_up = 0x43084308u;
        if (ZERO) {
          bias_lo = (0x4300u | in[S::kZeros + g * PER_GROUP + of]) * 0x10001u;
          bias_up = (0x4300u | in[S::kZeros + (g + 8) * PER_GROUP + of]) * 0x10001u;
        }
        if (c % kRun == 0)
#pragma unroll
          for (int i = 0; i < MT; ++i) sum[i][0] = sum[i][1] = sum[i][2] = sum[i][3] = 0.0f;
        const uint32_t a[8] = {pair_of<0>(lo[c], bias_lo), pair_of<0>(up[c], bias_up), pair_of<4>(lo[c], bias_lo), pair_of<4>(up[c], bias_up),
                               pair_of<8>(lo[c], bias_lo), pair_of<8>(up[c], bias_up), pair_of<12>(lo[c], bias_lo), pair_of<12>(up[c], bias_up)};
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint4 b = make_uint4(0, 0, 0, 0);
          if (i * 8 + g < columns) b = *reinterpret_cast<const uint4*>(xs + (uint64_t)(i * 8 + g) * pitch + kb * 128 + c * 32 + t * 8);
          mma(sum[i], a[0], a[1], a[2], a[3], b.x, b.y);
          mma(sum[i], a[4], a[5], a[6], a[7], b.z, b.w);
        }
        if (c % kRun == kRun - 1) {
          const float s_lo = __uint_as_float((uint32_t)scales[g * PER_GROUP + of] << 16), s_up = __uint_as_float((uint32_t)scales[(g + 8) * PER_GROUP + of] << 16);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            total[i][0] = fmaf(s_lo, sum[i][0], total[i][0]);
            total[i][1] = fmaf(s_lo, sum[i][1], total[i][1]);
            total[i][2] = fmaf(s_up, sum[i][2], total[i][2]);
            total[i][3] = fmaf(s_up, sum[i][3], total[i][3]);
          }
        }
      }
      __syncwarp();      // the stage is free for the next copy
      stage = (stage + 1) % kStages;
    }
    // the warps' sums, column by column of the instruction: [column][16 n]
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t column = i * 8 + t * 2 + (e & 1);
        if (column < columns) sums[warp * (128 * MT) + column * 16 + g + (e & 2) * 4] = total[i][e];
      }
    __syncthreads();
    for (uint32_t i = tid; i < columns * 16; i += kThreads) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s += sums[w * (128 * MT) + i];
      sums[i] = s;
    }
    if (ctas > 1) cluster.sync(); else __syncthreads();
    // the ranks' sums: each rank finishes a part of the rows
    for (uint32_t i = rank * kThreads + tid; i < rows * 16; i += ctas * kThreads) {
      const uint32_t m = i / 16, n = i % 16;
      float y = 0.0f;
#pragma unroll
      for (int term = kTerms - 1; term >= 0; --term) {      // the small ones first
        const uint32_t at = (m * kTerms + term) * 16 + n;
        if (ctas == 1) y += sums[at];
        else for (uint32_t r = 0; r < ctas; ++r) y += *cluster.map_shared_rank(sums + at, r);
      }
      const uint32_t col = tile * 16 + n;
      if (col < p.cols) {
        const int64_t at = (int64_t)(row0 + m) * p.cols + col;
        if (p.out_f32) static_cast<float*>(p.out)[at] = y;
        else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
      }
    }
    if (ctas > 1) cluster.sync(); else __syncthreads();      // the sums' memory is free, and nobody leaves while it is read
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename TX, int MT, int PER_GROUP, bool ZERO> size_t shared_bytes(uint32_t columns, uint32_t kblocks_of_cta) {
  return kWarps * kStages * Stage<PER_GROUP, ZERO>::kBytes + kWarps * 16 * 8 * MT * 4 + (size_t)columns * (kblocks_of_cta * 128 + kPad) * 2;
}

constexpr size_t kMaxShared = 227 * 1024;

template <typename TX, int MT, int PER_GROUP, bool ZERO> int launch_product(Product p, cudaStream_t st) {
  constexpr uint32_t kTerms = sizeof(TX) == 4 ? 3 : 1;
  auto kernel = int4_product_kernel<TX, MT, PER_GROUP, ZERO>;
  uint32_t ctas = 1, per_pass = p.rows < 8 * MT / kTerms ? p.rows : 8 * MT / kTerms;
  size_t bytes;
  while (true) {      // x in shared memory: split k over a cluster, and where that is not enough serve fewer rows with a pass
    bytes = shared_bytes<TX, MT, PER_GROUP, ZERO>(per_pass * kTerms, (p.kblocks + ctas - 1) / ctas);
    if (bytes <= kMaxShared) break;
    if (ctas < kMaxCluster) ctas *= 2;
    else if (per_pass > 1) { per_pass /= 2; ctas = 1; }
    else return fail(PB_ERR_UNSUPPORTED, "pb_int4_product: a contraction of %u does not fit", p.depth);
  }
  p.rows_per_pass = per_pass;
  PB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxShared));
  const uint32_t per_sm = (uint32_t)std::max<size_t>(1, std::min<size_t>(4, (size_t)(228 * 1024) / (bytes + 1024)));
  const uint32_t room = std::max<uint32_t>(1, sm_count() * per_sm / ctas);
  const uint32_t passes = (p.rows + per_pass - 1) / per_pass;
  if (passes > 65535) return fail(PB_ERR_UNSUPPORTED, "pb_int4_product: %u rows", p.rows);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(std::min(p.tiles, room) * ctas, passes);
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

template <typename TX, int MT> int launch_of(const Product& p, int per_group, cudaStream_t st) {
  if (p.zero) return per_group == 1 ? launch_product<TX, MT, 1, true>(p, st) : per_group == 2 ? launch_product<TX, MT, 2, true>(p, st) : launch_product<TX, MT, 4, true>(p, st);
  return per_group == 1 ? launch_product<TX, MT, 1, false>(p, st) : per_group == 2 ? launch_product<TX, MT, 2, false>(p, st) : launch_product<TX, MT, 4, false>(p, st);
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
  if (reinterpret_cast<uintptr_t>(q) & 15) return fail(PB_ERR_MISALIGNED, "pb_quantize_int4: q must be 16-byte aligned");
  const uint32_t kblocks = (uint32_t)((depth + 127) / 128), col_blocks = (uint32_t)((cols + kQuantCols - 1) / kQuantCols);
  if (col_blocks > 65535) return fail(PB_ERR_UNSUPPORTED, "pb_quantize_int4: %lld columns", (long long)cols);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(kblocks, col_blocks);
  auto* words = reinterpret_cast<uint32_t*>(q);
  auto* s = static_cast<__nv_bfloat16*>(scale);
  const int per_group = 128 / group;
  if (dtype == PB_F32) {
    const float* in = static_cast<const float*>(w);
    if (zero) launch_behind(quantize_int4_kernel<float, true>, grid, kQuantThreads, 0, st, in, depth, cols, per_group, kblocks, words, s, zero);
    else launch_behind(quantize_int4_kernel<float, false>, grid, kQuantThreads, 0, st, in, depth, cols, per_group, kblocks, words, s, zero);
  } else {
    const __nv_bfloat16* in = static_cast<const __nv_bfloat16*>(w);
    if (zero) launch_behind(quantize_int4_kernel<__nv_bfloat16, true>, grid, kQuantThreads, 0, st, in, depth, cols, per_group, kblocks, words, s, zero);
    else launch_behind(quantize_int4_kernel<__nv_bfloat16, false>, grid, kQuantThreads, 0, st, in, depth, cols, per_group, kblocks, words, s, zero);
  }
  PB_LAUNCH_CHECK("quantize_int4_kernel");
  return PB_OK;
}

extern "C" int pb_dequantize_int4(const uint8_t* q, const void* scale, const uint8_t* zero, int64_t depth, int64_t cols, int group, void* out, int dtype, void* stream) {
  if (!q || !scale || !out) return fail(PB_ERR_NULL_POINTER, "pb_dequantize_int4: null argument");
  if (dtype != PB_F32 && dtype != PB_BF16) return fail(PB_ERR_BAD_DTYPE, "pb_dequantize_int4: dtype %d", dtype);
  if (int s = check_int4("pb_dequantize_int4", depth, cols, group)) return s;
  if (reinterpret_cast<uintptr_t>(q) & 15) return fail(PB_ERR_MISALIGNED, "pb_dequantize_int4: q must be 16-byte aligned");
  const uint32_t kblocks = (uint32_t)((depth + 127) / 128), col_blocks = (uint32_t)((cols + kQuantCols - 1) / kQuantCols);
  if (col_blocks > 65535) return fail(PB_ERR_UNSUPPORTED, "pb_dequantize_int4: %lld columns", (long long)cols);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(kblocks, col_blocks);
  const auto* words = reinterpret_cast<const uint32_t*>(q);
  const auto* s = static_cast<const __nv_bfloat16*>(scale);
  if (dtype == PB_F32) launch_behind(dequantize_int4_kernel<float>, grid, kQuantThreads, 0, st, words, s, zero, depth, cols, 128 / group, kblocks, static_cast<float*>(out));
  else launch_behind(dequantize_int4_kernel<__nv_bfloat16>, grid, kQuantThreads, 0, st, words, s, zero, depth, cols, 128 / group, kblocks, static_cast<__nv_bfloat16*>(out));
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
  if ((reinterpret_cast<uintptr_t>(q) & 15) || ((reinterpret_cast<uintptr_t>(scale) | reinterpret_cast<uintptr_t>(zero)) & 3) ||
      (reinterpret_cast<uintptr_t>(x) % (x_dtype == PB_F32 ? 4 : 2)) || (reinterpret_cast<uintptr_t>(out) % (out_dtype == PB_F32 ? 4 : 2)))
    return fail(PB_ERR_MISALIGNED, "pb_int4_product: q 16, scale and zero 4 bytes, x and out their types");
  Product p{x, stride, q, static_cast<const __nv_bfloat16*>(scale), zero, out, (uint32_t)rows, (uint32_t)depth, (uint32_t)cols, (uint32_t)((depth + 127) / 128),
            (uint32_t)((cols + 15) / 16), 0, out_dtype == PB_F32};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t columns = rows * (x_dtype == PB_F32 ? 3 : 1);
  if (x_dtype == PB_F32) return columns <= 8 ? launch_of<float, 1>(p, 128 / group, st) : columns <= 16 ? launch_of<float, 2>(p, 128 / group, st) : launch_of<float, 4>(p, 128 / group, st);
  return columns <= 8 ? launch_of<__nv_bfloat16, 1>(p, 128 / group, st) : columns <= 16 ? launch_of<__nv_bfloat16, 2>(p, 128 / group, st) : launch_of<__nv_bfloat16, 4>(p, 128 / group, st);
}
