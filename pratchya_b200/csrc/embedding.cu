// The token embedding (EmbeddingScaled, pratchya/_nnx_impl/_module.py:21-37) and its gradient:
//   rows[i] = scale * table[ids[i]],      d_table[v] = scale * sum of g[i] over the i with ids[i] = v, in their order.
// Both are bound by bytes: rows read and written; g read once and every row of d_table written once, most of them zeros.
//
// The gradient goes by sorted tokens and has no float atomics, so that its bits do not depend on the order of threads: (id, position) pairs are sorted by id, stable, with
// digits of up to nine bits (two passes below 2^18 words); a block of up to kRun sorted positions is then one CTA's for a slab of columns: runs of one id that
// lie in it go to d_table at once, and what of a run crosses its ends leaves as partial sums in f32, which another kernel adds up in their order.  Which rows no
// token has is a bitmap; they are zeroed by CTAs beside those of the first pass that moves pairs, so that the sort is behind bytes that have to be written anyway.
// Up to 4096 tokens one CTA sorts in its shared memory, and the zeros are written beside the sums.
#include <algorithm>

#include "common.cuh"

namespace pb {
namespace {

constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32;
constexpr int kWarpKeys = 128, kTile = kWarpKeys * kSortWarps;      // keys a CTA sorts
constexpr int kMostBits = 9, kBins = 1 << kMostBits;
constexpr int kRun = 32, kShortRun = 8;      // sorted positions a CTA adds up: the fewer where there are few, that CTAs ask for all of them at once
constexpr int kFewTiles = 320, kChunk = 256;      // up to kFewTiles a tile adds up the others' counts by itself; else they are summed first, kChunk tiles a CTA
constexpr int kAlone = 4096, kAloneThreads = 1024, kAloneWarps = kAloneThreads / 32;      // pairs that one CTA sorts
constexpr int kSumThreads = 128;
constexpr int kAhead = 8;             // rows of g that a thread asks for at once
constexpr int kLooks = 4;             // 16-byte vectors of a lane of the lookup
constexpr int kZeroRows = 16, kZeroBeside = 4;      // a CTA's, of 512 threads beside the sort and of 128 beside the sums

// A token's row: ids below zero count from the end; -1 for padding, -2 for what lies beyond the table on either side.
__device__ __forceinline__ int64_t row_of(int64_t id, int64_t vocab, int64_t padding) {
  if (id < 0) id += vocab;
  return id < 0 || id >= vocab ? -2 : id == padding ? -1 : id;
}

template <typename T, bool VECTORS>
struct Columns {
  static constexpr int kN = VECTORS ? 16 / (int)sizeof(T) : 1;      // that a thread takes at once
  static __device__ __forceinline__ void load(const T* p, float (&x)[kN]) {
    if constexpr (!VECTORS) {
      x[0] = Elem<T>::to_f32(*p);
    } else {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) x[j] = __uint_as_float(w[j]);
        else { x[2 * j] = __uint_as_float(w[j] << 16); x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[kN]) {
    if constexpr (!VECTORS) {
      *p = Elem<T>::from_f32(x[0]);
    } else if constexpr (sizeof(T) == 4) {
      __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
    } else {
      __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])));
    }
  }
};

// ---- the lookup -----------------------------------------------------------------------------------------------------
struct LookupParams {
  const void* table;
  const int64_t* ids;
  void* out;
  int64_t vocab, channels, padding;
  uint32_t items;             // of a warp: a row's part of 32 x kLooks vectors
  FastDiv per_row;
  float scale;
};
template <typename T, bool VECTORS>
__global__ void __launch_bounds__(128) lookup_kernel(const __grid_constant__ LookupParams p) {
  grid_wait();
  using C = Columns<T, VECTORS>;
  const uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const uint32_t i = p.per_row.div(item);
  const int64_t first = ((int64_t)(item - i * p.per_row.d) * 32 * kLooks + (threadIdx.x & 31)) * C::kN;
  const int64_t row = row_of(__ldg(p.ids + i), p.vocab, p.padding);
  const T* from = static_cast<const T*>(p.table) + max(row, (int64_t)0) * p.channels;
  T* to = static_cast<T*>(p.out) + (int64_t)i * p.channels;
  float x[kLooks][C::kN];
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    const int64_t c = first + k * 32 * C::kN;
#pragma unroll
    for (int j = 0; j < C::kN; ++j) x[k][j] = row == -2 ? nanf("") : 0.0f;
    if (row >= 0 && c < p.channels) C::load(from + c, x[k]);
  }
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    const int64_t c = first + k * 32 * C::kN;
    if (c >= p.channels) break;
    if (row >= 0) {
#pragma unroll
      for (int j = 0; j < C::kN; ++j) x[k][j] *= p.scale;
    }
    C::store(to + c, x[k]);
  }
}

// ---- the sort -------------------------------------------------------------------------------------------------------
// rows that no token has
struct ZeroParams {
  const uint32_t* present;
  void* d_table;
  int64_t vocab, row_bytes;
  bool vectors;
};
struct SortParams {
  const int64_t* ids;              // the first pass: keys are made of them
  const uint32_t *keys, *order;    // later ones
  uint32_t *keys_out, *order_out;
  uint32_t* counts;                // [tiles][kBins]
  uint32_t* sums;                  // of many tiles: [chunks + 1][kBins], see scan_kernel
  uint32_t* present;               // the first pass: a bit for each row that a token has
  int64_t vocab, padding;
  uint32_t n, tiles, shift, bits;
  ZeroParams zero;                 // for the CTAs behind the tiles'
};
__device__ __forceinline__ uint32_t key_at(const SortParams& p, uint32_t i) {
  if (!p.ids) return p.keys[i];
  const int64_t row = row_of(p.ids[i], p.vocab, p.padding);
  return row < 0 ? (uint32_t)p.vocab : (uint32_t)row;      // sorts behind every row
}

__global__ void __launch_bounds__(kSortThreads) count_kernel(const __grid_constant__ SortParams p) {
  grid_wait();
  __shared__ uint32_t bins[kBins];
  bins[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t first = blockIdx.x * kTile, mask = (1u << p.bits) - 1;
#pragma unroll
  for (int k = 0; k < kTile / kSortThreads; ++k) {
    const uint32_t i = first + k * kSortThreads + threadIdx.x;
    if (i < p.n) {
      const uint32_t key = key_at(p, i);
      atomicAdd(&bins[key >> p.shift & mask], 1u);
      if (p.present && key < p.vocab) atomicOr(p.present + key / 32, 1u << (key % 32));
    }
  }
  __syncthreads();
  p.counts[(size_t)blockIdx.x * kBins + threadIdx.x] = bins[threadIdx.x];
}

// the pairs of lower digits than this thread's, of which there are `all`
__device__ __forceinline__ uint32_t below_digit(uint32_t all) {
  __shared__ uint32_t sums[kSortWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t upto = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t below = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += below;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  uint32_t base = upto - all;
  for (int w = 0; w < warp; ++w) base += sums[w];
  return base;
}

// Counts of many tiles: where each of them reads all others' the work grows with the square of the tokens.  The gradient of 65536 words of 8 channels, us, by every tile | by the
// kernels here: 2^19 tokens (256 tiles) 187 | 199, 2^20 352 | 322, 2^22 1807 | 961, 2^23 5100 | 1680.
// A CTA's chunk of tiles: each one's counts become those of the chunk's tiles before it, and the chunk's own go to sums[chunk].
__global__ void __launch_bounds__(kSortThreads) scan_kernel(const __grid_constant__ SortParams p) {
  grid_wait();
  const uint32_t end = min(p.tiles, (blockIdx.x + 1) * kChunk);
  uint32_t before = 0;
  for (uint32_t t0 = blockIdx.x * kChunk; t0 < end; t0 += 16) {
    uint32_t c[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) c[k] = t0 + k < end ? p.counts[(size_t)(t0 + k) * kBins + threadIdx.x] : 0u;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      if (t0 + k < end) p.counts[(size_t)(t0 + k) * kBins + threadIdx.x] = before;
      before += c[k];
    }
  }
  p.sums[blockIdx.x * kBins + threadIdx.x] = before;
}
// One CTA: the same for the chunks, of which the last row is that of a digit's first pair.
__global__ void __launch_bounds__(kSortThreads) scan_chunks_kernel(const __grid_constant__ SortParams p) {
  grid_wait();
  const uint32_t chunks = (p.tiles + kChunk - 1) / kChunk;
  uint32_t before = 0;
#pragma unroll 8
  for (uint32_t k = 0; k < chunks; ++k) {
    const uint32_t c = p.sums[k * kBins + threadIdx.x];
    p.sums[k * kBins + threadIdx.x] = before;
    before += c;
  }
  p.sums[chunks * kBins + threadIdx.x] = below_digit(before);
}

template <int THREADS, int ROWS>
__device__ __forceinline__ void zero_rows(const ZeroParams& p, uint32_t block) {
  const int64_t first = (int64_t)block * ROWS;
  const uint32_t word = p.present[first / 32] >> (first % 32);
  for (int r = 0; r < ROWS && first + r < p.vocab; ++r) {
    if (word >> r & 1) continue;
    char* row = static_cast<char*>(p.d_table) + (first + r) * p.row_bytes;
    if (p.vectors) for (int64_t c = (int64_t)threadIdx.x * 16; c < p.row_bytes; c += THREADS * 16) __stcs(reinterpret_cast<uint4*>(row + c), make_uint4(0u, 0u, 0u, 0u));
    else for (int64_t c = (int64_t)threadIdx.x * 2; c < p.row_bytes; c += THREADS * 2) *reinterpret_cast<unsigned short*>(row + c) = 0;
  }
}

// a tile's pairs to where they go: behind the pairs of lower digits, of the tiles before, of the warps before, and of the lanes before
__global__ void __launch_bounds__(kSortThreads) scatter_kernel(const __grid_constant__ SortParams p) {
  grid_wait();
  if (blockIdx.x >= p.tiles) return zero_rows<kSortThreads, kZeroRows>(p.zero, blockIdx.x - p.tiles);
  __shared__ uint32_t at[kSortWarps][kBins];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t bin = threadIdx.x, mask = (1u << p.bits) - 1;
  for (int w = 0; w < kSortWarps; ++w) at[w][bin] = 0;
  uint32_t base = 0;
  if (p.sums) {
    base = p.counts[(size_t)blockIdx.x * kBins + bin] + p.sums[blockIdx.x / kChunk * kBins + bin] + p.sums[(p.tiles + kChunk - 1) / kChunk * kBins + bin];
    __syncthreads();
  } else {
    uint32_t all = 0;
#pragma unroll 8
    for (uint32_t t = 0; t < p.tiles; ++t) {
      const uint32_t c = p.counts[(size_t)t * kBins + bin];
      all += c;
      if (t < blockIdx.x) base += c;
    }
    base += below_digit(all);
  }
  uint32_t keys[kWarpKeys / 32], digits[kWarpKeys / 32];
  const uint32_t first = blockIdx.x * kTile + warp * kWarpKeys + lane;
#pragma unroll
  for (int k = 0; k < kWarpKeys / 32; ++k) {
    const uint32_t i = first + 32 * k;
    keys[k] = i < p.n ? key_at(p, i) : 0u;
    digits[k] = i < p.n ? keys[k] >> p.shift & mask : kBins;
    if (i < p.n) atomicAdd(&at[warp][digits[k]], 1u);
  }
  __syncthreads();
  for (int w = 0; w < kSortWarps; ++w) {
    const uint32_t c = at[w][bin];
    at[w][bin] = base;
    base += c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWarpKeys / 32; ++k) {
    const uint32_t i = first + 32 * k, same = __match_any_sync(0xffffffffu, digits[k]);
    const uint32_t rank = __popc(same & ((1u << lane) - 1));
    uint32_t to = 0;
    if (i < p.n) to = at[warp][digits[k]] + rank;
    __syncwarp();
    if (i < p.n && rank == 0) at[warp][digits[k]] += __popc(same);
    __syncwarp();
    if (i < p.n) {
      p.keys_out[to] = keys[k];
      p.order_out[to] = p.ids ? i : p.order[i];
    }
  }
}

// All passes of up to kAlone pairs: by one CTA, pairs and the warps' numbers of each digit in its shared memory.
struct AloneParams {
  const int64_t* ids;
  uint32_t *keys, *order, *present;
  int64_t vocab, padding;
  uint32_t n, words, bits, passes;      // words: of the bitmap
};
constexpr int kAloneSmem = (kAloneWarps * kBins + 4 * kAlone) * 4;
__global__ void __launch_bounds__(kAloneThreads) sort_alone_kernel(const __grid_constant__ AloneParams p) {
  grid_wait();
  extern __shared__ uint32_t alone_smem[];
  __shared__ uint32_t sums[kAloneWarps];
  uint32_t(*at)[kBins] = reinterpret_cast<uint32_t(*)[kBins]>(alone_smem);
  uint32_t* pairs = alone_smem + kAloneWarps * kBins;      // two times keys and order
  constexpr int kEach = kAlone / kAloneThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t first = warp * (32 * kEach) + lane;
  uint32_t keys[kEach], order[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const uint32_t i = first + 32 * k;
    const int64_t row = i < p.n ? row_of(p.ids[i], p.vocab, p.padding) : -1;
    keys[k] = row < 0 ? (uint32_t)p.vocab : (uint32_t)row;
    order[k] = i;
  }
  for (uint32_t w = threadIdx.x; w < p.words; w += kAloneThreads) p.present[w] = 0;
  uint32_t shift = 0;
  for (uint32_t pass = 0; pass < p.passes; ++pass) {
    const uint32_t width = (p.bits - shift + p.passes - pass - 1) / (p.passes - pass), mask = (1u << width) - 1;
    for (int w = threadIdx.x; w < kAloneWarps * kBins; w += kAloneThreads) alone_smem[w] = 0;
    __syncthreads();      // and the bitmap is zero
    if (pass == 0) {
#pragma unroll
      for (int k = 0; k < kEach; ++k)
        if (keys[k] < p.vocab) atomicOr(p.present + keys[k] / 32, 1u << (keys[k] % 32));
    }
    uint32_t digits[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      digits[k] = first + 32 * k < p.n ? keys[k] >> shift & mask : kBins;
      if (digits[k] < kBins) atomicAdd(&at[warp][digits[k]], 1u);
    }
    __syncthreads();
    uint32_t all = 0, upto = 0;
    if (threadIdx.x < kBins) {
#pragma unroll 8
      for (int w = 0; w < kAloneWarps; ++w) all += at[w][threadIdx.x];
      upto = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t below = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += below;
      }
      if (lane == 31) sums[warp] = upto;
    }
    __syncthreads();
    if (threadIdx.x < kBins) {
      uint32_t base = upto - all;
      for (int w = 0; w < warp; ++w) base += sums[w];
#pragma unroll 8
      for (int w = 0; w < kAloneWarps; ++w) {
        const uint32_t c = at[w][threadIdx.x];
        at[w][threadIdx.x] = base;
        base += c;
      }
    }
    __syncthreads();
    const bool last = pass + 1 == p.passes;
    uint32_t* to_keys = last ? p.keys : pairs + (pass & 1) * 2 * kAlone;
    uint32_t* to_order = last ? p.order : pairs + ((pass & 1) * 2 + 1) * kAlone;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const uint32_t same = __match_any_sync(0xffffffffu, digits[k]), rank = __popc(same & ((1u << lane) - 1));
      const bool there = digits[k] < kBins;
      uint32_t to = 0;
      if (there) to = at[warp][digits[k]] + rank;
      __syncwarp();
      if (there && rank == 0) at[warp][digits[k]] += __popc(same);
      __syncwarp();
      if (there) { to_keys[to] = keys[k]; to_order[to] = order[k]; }
    }
    __syncthreads();
    if (!last) {
#pragma unroll
      for (int k = 0; k < kEach; ++k) { keys[k] = to_keys[first + 32 * k]; order[k] = to_order[first + 32 * k]; }      // behind the n-th whatever was there
    }
    shift += width;
  }
}

// ---- the sums -------------------------------------------------------------------------------------------------------
struct SumParams {
  const void* g;
  const uint32_t *keys, *order;
  void* d_table;
  float* partial;            // [blocks][2][channels]: of the run that reaches into a block from before, and of the one that leaves it
  int64_t vocab, channels;
  uint32_t n, run, blocks, items;      // items: blocks times slabs
  float scale;
  ZeroParams zero;           // for the CTAs behind the items'
};
template <typename T, bool VECTORS>
__global__ void __launch_bounds__(kSumThreads) sum_kernel(const __grid_constant__ SumParams p) {
  grid_wait();
  using C = Columns<T, VECTORS>;
  if (blockIdx.x >= p.items) return zero_rows<kSumThreads, kZeroBeside>(p.zero, blockIdx.x - p.items);
  const uint32_t slab = blockIdx.x / p.blocks, block = blockIdx.x - slab * p.blocks;
  __shared__ uint32_t keys[kRun + 2], order[kRun];      // keys: of the position before, too, and of the one behind
  const uint32_t first = block * p.run, n = min(p.run, p.n - first);
  if (threadIdx.x < n + 2) {
    const int64_t i = (int64_t)first + threadIdx.x - 1;
    keys[threadIdx.x] = i >= 0 && i < p.n ? p.keys[i] : 0xffffffffu;
  }
  if (threadIdx.x < n) order[threadIdx.x] = p.order[first + threadIdx.x];
  __syncthreads();
  const int64_t c = ((int64_t)slab * kSumThreads + threadIdx.x) * C::kN;
  if (c >= p.channels || keys[1] >= p.vocab) return;
  const T* g = static_cast<const T*>(p.g) + c;
  float sum[C::kN];
#pragma unroll
  for (int j = 0; j < C::kN; ++j) sum[j] = 0.0f;
  bool whole = keys[0] != keys[1];          // the run began in this block
  for (uint32_t i0 = 0; i0 < n; i0 += kAhead) {
    float x[kAhead][C::kN];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i0 + k < n && keys[i0 + k + 1] < p.vocab) C::load(g + (int64_t)order[i0 + k] * p.channels, x[k]);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint32_t i = i0 + k;
      if (i >= n) break;
      const uint32_t key = keys[i + 1];
      if (key >= p.vocab) return;           // and all behind it
#pragma unroll
      for (int j = 0; j < C::kN; ++j) sum[j] += x[k][j];
      const bool ends = keys[i + 2] != key;
      if (!ends && i + 1 < n) continue;
      if (ends && whole) {
#pragma unroll
        for (int j = 0; j < C::kN; ++j) sum[j] *= p.scale;
        C::store(static_cast<T*>(p.d_table) + (int64_t)key * p.channels + c, sum);
      } else {
        float* to = p.partial + ((int64_t)block * 2 + (whole ? 1 : 0)) * p.channels + c;
        if constexpr (VECTORS) {
#pragma unroll
          for (int j = 0; j < C::kN; j += 4) *reinterpret_cast<float4*>(to + j) = make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
        } else {
          to[0] = sum[0];
        }
      }
#pragma unroll
      for (int j = 0; j < C::kN; ++j) sum[j] = 0.0f;
      whole = true;
    }
  }
}

// Runs of several blocks, by the block where they begin: kJoin groups of threads take the blocks behind it in turn, and meet in their order.  A thread has four columns, or one.
constexpr int kJoin = 4, kJoinThreads = 128;
template <typename T, bool VECTORS>
__global__ void __launch_bounds__(kJoin * kJoinThreads) join_kernel(const __grid_constant__ SumParams p) {
  grid_wait();
  constexpr int kN = VECTORS ? 4 : 1;
  __shared__ float sums[kJoin][kJoinThreads][kN];
  __shared__ uint32_t last;
  const uint32_t block = blockIdx.x, end = block * p.run + p.run;
  const uint32_t key = p.keys[end - 1], behind = p.keys[end], before = block ? p.keys[block * p.run - 1] : 0xffffffffu;
  if (key >= p.vocab || behind != key || before == key) return;                  // nothing leaves this block, or it came from before
  if (threadIdx.x < 32) {                                                        // the last block that the run reaches: 32 places at a time
    uint32_t lo = end, hi = p.n - 1;                                             // keys[lo] == key, and none behind hi
    while (lo < hi) {
      const uint32_t step = (hi - lo + 31) / 32, at = min(hi, lo + step * (threadIdx.x + 1));
      const uint32_t reach = __popc(__ballot_sync(0xffffffffu, p.keys[at] == key));
      hi = reach == 32 ? hi : min(hi, lo + step * (reach + 1) - 1);
      lo = reach == 32 ? hi : lo + step * reach;
    }
    if (threadIdx.x == 0) last = lo / p.run;
  }
  __syncthreads();
  const int group = threadIdx.x / kJoinThreads, column = threadIdx.x % kJoinThreads;
  const int64_t c = ((int64_t)blockIdx.y * kJoinThreads + column) * kN;
  float sum[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j) sum[j] = 0.0f;
  auto add = [&](int64_t slot) {
    const float* from = p.partial + slot * p.channels + c;
    if constexpr (VECTORS) {
      const float4 v = *reinterpret_cast<const float4*>(from);
      sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
    } else {
      sum[0] += from[0];
    }
  };
  if (c < p.channels) {
    if (group == 0) add((int64_t)block * 2 + 1);
#pragma unroll 8
    for (uint32_t b = block + 1 + group; b <= last; b += kJoin) add((int64_t)b * 2);
  }
#pragma unroll
  for (int j = 0; j < kN; ++j) sums[group][column][j] = sum[j];
  __syncthreads();
  if (group != 0 || c >= p.channels) return;
  T* to = static_cast<T*>(p.d_table) + (int64_t)key * p.channels + c;
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    float s = sum[j];
#pragma unroll
    for (int k = 1; k < kJoin; ++k) s += sums[k][column][j];
    to[j] = Elem<T>::from_f32(s * p.scale);
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct Plan {
  uint32_t tiles, run, blocks;
  size_t off_keys[2], off_order[2], off_counts, off_sums, off_partial, bytes;
};
int make_plan(int64_t n, int64_t vocab, int64_t channels, Plan* q) {
  if (n < 0 || n > (1 << 28) || vocab <= 0 || vocab > (1 << 30) || channels <= 0 || channels > (1 << 21))
    return fail(PB_ERR_BAD_SHAPE, "pb_embedding: %lld tokens, table [%lld, %lld]", (long long)n, (long long)vocab, (long long)channels);
  q->tiles = (uint32_t)((n + kTile - 1) / kTile);
  q->run = n <= kAlone ? kShortRun : kRun;
  q->blocks = (uint32_t)((n + q->run - 1) / q->run);
  size_t at = (size_t)((vocab + 31) / 32 + 63) / 64 * 256;
  auto take = [&](size_t bytes) { const size_t was = at; at += (bytes + 255) / 256 * 256; return was; };
  for (int i = 0; i < 2; ++i) { q->off_keys[i] = take((size_t)n * 4); q->off_order[i] = take((size_t)n * 4); }
  q->off_counts = take((size_t)q->tiles * kBins * 4);
  q->off_sums = take(q->tiles > kFewTiles ? ((size_t)(q->tiles + kChunk - 1) / kChunk + 1) * kBins * 4 : 0);
  q->off_partial = take((size_t)q->blocks * 2 * channels * 4);
  q->bytes = at;
  return PB_OK;
}
int check(const char* name, int dtype, int64_t n, const int64_t* ids, int64_t vocab, int64_t channels, Plan* q) {
  if (int s = make_plan(n, vocab, channels, q)) return s;
  if (dtype != PB_F32 && dtype != PB_BF16) return fail(PB_ERR_BAD_DTYPE, "%s: dtype %d", name, dtype);
  if (n && !ids) return fail(PB_ERR_NULL_POINTER, "%s: null argument", name);
  if (off_by(ids, 8)) return fail(PB_ERR_MISALIGNED, "%s: misaligned ids", name);
  return PB_OK;
}

template <typename T, bool VECTORS>
int sum_runs(SumParams p, const Plan& q, bool zero, cudaStream_t st) {
  const int64_t slab = (int64_t)kSumThreads * Columns<T, VECTORS>::kN, items = q.blocks * ((p.channels + slab - 1) / slab);
  const int64_t grid = items + (zero ? (p.vocab + kZeroBeside - 1) / kZeroBeside : 0);
  if (grid > kMaxIndexed) return fail(PB_ERR_BAD_SHAPE, "pb_embedding_lookup_bwd: %u tokens of %lld channels", p.n, (long long)p.channels);
  p.run = q.run; p.blocks = q.blocks; p.items = (uint32_t)items;
  launch_behind(sum_kernel<T, VECTORS>, (unsigned)grid, kSumThreads, 0, st, p);
  PB_LAUNCH_CHECK("embedding sum_kernel");
  if (q.blocks > 1) {
    const int64_t columns = kJoinThreads * (VECTORS ? 4 : 1);
    launch_behind(join_kernel<T, VECTORS>, dim3(q.blocks - 1, (unsigned)((p.channels + columns - 1) / columns)), kJoin * kJoinThreads, 0, st, p);
    PB_LAUNCH_CHECK("embedding join_kernel");
  }
  return PB_OK;
}

}  // namespace
}  // namespace pb

using namespace pb;

extern "C" int pb_embedding_lookup(const void* table, int dtype, int64_t vocab, int64_t channels, const int64_t* ids, int64_t n, float scale, int64_t padding_id, void* out, void* stream) {
  Plan q;
  if (int s = check("pb_embedding_lookup", dtype, n, ids, vocab, channels, &q)) return s;
  if (n == 0) return PB_OK;
  if (!table || !out) return fail(PB_ERR_NULL_POINTER, "pb_embedding_lookup: null argument");
  const int64_t size = dtype == PB_F32 ? 4 : 2;
  if (off_by(table, size) || off_by(out, size)) return fail(PB_ERR_MISALIGNED, "pb_embedding_lookup: misaligned array");
  const bool vectors = channels * size % 16 == 0 && !off_by(table, 16) && !off_by(out, 16);
  const int64_t part = 32 * kLooks * (vectors ? 16 / size : 1), per_row = (channels + part - 1) / part, items = n * per_row;
  if (items > kMaxIndexed) return fail(PB_ERR_BAD_SHAPE, "pb_embedding_lookup: %lld tokens of %lld channels", (long long)n, (long long)channels);
  const LookupParams p{table, ids, out, vocab, channels, padding_id, (uint32_t)items, FastDiv((uint32_t)per_row), scale};
  const unsigned grid = (unsigned)((items + 3) / 4);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) { launch_behind(kernel, grid, 128, 0, st, p); };
  if (dtype == PB_F32) vectors ? go(lookup_kernel<float, true>) : go(lookup_kernel<float, false>);
  else vectors ? go(lookup_kernel<__nv_bfloat16, true>) : go(lookup_kernel<__nv_bfloat16, false>);
  PB_LAUNCH_CHECK("lookup_kernel");
  return PB_OK;
}

extern "C" size_t pb_embedding_lookup_bwd_workspace_size(int64_t n, int64_t vocab, int64_t channels) {
  Plan q;
  return make_plan(n, vocab, channels, &q) ? 0 : q.bytes;
}

extern "C" int pb_embedding_lookup_bwd(const void* g, int dtype, const int64_t* ids, int64_t n, int64_t vocab, int64_t channels, float scale, int64_t padding_id, void* d_table,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  Plan q;
  if (int s = check("pb_embedding_lookup_bwd", dtype, n, ids, vocab, channels, &q)) return s;
  if (!d_table || (n && (!g || !workspace))) return fail(PB_ERR_NULL_POINTER, "pb_embedding_lookup_bwd: null argument");
  const int64_t size = dtype == PB_F32 ? 4 : 2;
  if (off_by(g, size) || off_by(d_table, size) || off_by(workspace, 256)) return fail(PB_ERR_MISALIGNED, "pb_embedding_lookup_bwd: misaligned array");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    PB_CUDA_TRY(cudaMemsetAsync(d_table, 0, (size_t)(vocab * channels * size), st));
    return PB_OK;
  }
  if (workspace_bytes < q.bytes) return fail(PB_ERR_WORKSPACE_TOO_SMALL, "pb_embedding_lookup_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, q.bytes);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  uint32_t* present = reinterpret_cast<uint32_t*>(ws);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(ws + q.off_keys[0]), reinterpret_cast<uint32_t*>(ws + q.off_keys[1])};
  uint32_t* order[2] = {reinterpret_cast<uint32_t*>(ws + q.off_order[0]), reinterpret_cast<uint32_t*>(ws + q.off_order[1])};
  const uint32_t words = (uint32_t)((vocab + 31) / 32);
  uint32_t bits = 1;
  while ((vocab >> bits) != 0) ++bits;          // of the keys, `vocab` itself among them
  const int passes = (int)((bits + kMostBits - 1) / kMostBits);
  const bool vectors = channels * size % 16 == 0 && !off_by(d_table, 16) && !off_by(g, 16), alone = n <= kAlone;
  const ZeroParams zero{present, d_table, vocab, channels * size, vectors};
  if (alone) {
    PB_CUDA_TRY(cudaFuncSetAttribute(sort_alone_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kAloneSmem));      // per device
    launch_behind(sort_alone_kernel, 1, kAloneThreads, kAloneSmem, st, AloneParams{ids, keys[(passes - 1) & 1], order[(passes - 1) & 1], present, vocab, padding_id, (uint32_t)n, words, bits, (uint32_t)passes});
    PB_LAUNCH_CHECK("embedding sort_alone_kernel");
  } else {
    PB_CUDA_TRY(cudaMemsetAsync(present, 0, (size_t)words * 4, st));
    SortParams p{};
    p.counts = reinterpret_cast<uint32_t*>(ws + q.off_counts);
    p.sums = q.tiles > kFewTiles ? reinterpret_cast<uint32_t*>(ws + q.off_sums) : nullptr;
    p.vocab = vocab; p.padding = padding_id; p.n = (uint32_t)n; p.tiles = q.tiles; p.zero = zero;
    for (int k = 0, shift = 0; k < passes; ++k) {
      const int width = ((int)bits - shift + passes - k - 1) / (passes - k);
      p.ids = k == 0 ? ids : nullptr;
      p.keys = keys[(k + 1) & 1]; p.order = order[(k + 1) & 1];
      p.keys_out = keys[k & 1]; p.order_out = order[k & 1];
      p.present = k == 0 ? present : nullptr;
      p.shift = (uint32_t)shift; p.bits = (uint32_t)width;
      launch_behind(count_kernel, q.tiles, kSortThreads, 0, st, p);
      PB_LAUNCH_CHECK("embedding count_kernel");
      if (p.sums) {
        launch_behind(scan_kernel, (q.tiles + kChunk - 1) / kChunk, kSortThreads, 0, st, p);
        PB_LAUNCH_CHECK("embedding scan_kernel");
        launch_behind(scan_chunks_kernel, 1, kSortThreads, 0, st, p);
        PB_LAUNCH_CHECK("embedding scan_chunks_kernel");
      }
      launch_behind(scatter_kernel, q.tiles + (k == 0 ? (unsigned)((vocab + kZeroRows - 1) / kZeroRows) : 0u), kSortThreads, 0, st, p);
      PB_LAUNCH_CHECK("embedding scatter_kernel");
      shift += width;
    }
  }
  SumParams sp{};
  sp.g = g; sp.keys = keys[(passes - 1) & 1]; sp.order = order[(passes - 1) & 1]; sp.d_table = d_table; sp.partial = reinterpret_cast<float*>(ws + q.off_partial);
  sp.vocab = vocab; sp.channels = channels; sp.n = (uint32_t)n; sp.scale = scale; sp.zero = zero;
  if (dtype == PB_F32) return vectors ? sum_runs<float, true>(sp, q, alone, st) : sum_runs<float, false>(sp, q, alone, st);
  return vectors ? sum_runs<__nv_bfloat16, true>(sp, q, alone, st) : sum_runs<__nv_bfloat16, false>(sp, q, alone, st);
}
