// Products of 16-bit operands on the tensor cores for the operators that are built around one: D[m, n] = sum_k A[m, k] B[n, k] in f32, handed to
// an epilogue of the operator's own (loss statistics, a gradient, a polynomial's term) in the registers that read the accumulator.
//
// A and B are both bf16 or both fp16, each with k or with its rows lying together in memory (K-major, or M/N-major): TMA takes either
// into 128-byte swizzled tiles and the matrix descriptors say which, so that no operand is ever transposed.  A tile is 128 CTAS x N:
//   CTAS = 2: a cluster of two CTAs makes 256 x 256; each loads its own 128 rows of A and its own 128 of B (32 KB per 64 of k and
//             SM, where one CTA's 128 x 256 takes 48: what a tile loads from L2 is the nearest bound beside the tensor core);
//   the same pair with 256 x 128, and CTAS = 1 with 128 x 128 or 128 x 256: for products that have few tiles, or few rows.
// Persistent: warp 0 loads, a lane of warp 1 (of the leading CTA) issues tcgen05.mma, eight warps empty one accumulator of TMEM while the
// other fills, each thread one row and half of the columns.  Every wait is bounded and reported by pb_gemm_check.
// The tensor core's own additions do not round to nearest: an accumulator takes `group` stages of k, and the sums of a tile's groups are added up in the
// registers that read them.  2-norm errors of the loss of 64 positions of 2048 against 64 bits: one group 1.4e-6, groups of 512 of k 2.4e-7.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace pb {
namespace products {
namespace {

constexpr int kDepth = 64;                        // k per stage: 128 bytes, a swizzled row
constexpr uint32_t kWaitPolls = 1u << 21;         // a poll parks for up to 2 us: about four seconds at most

constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 128 + 32 * kEpilogueWarps;
constexpr int kBlock = 64;                        // columns that an epilogue takes at a time: 128 bytes
constexpr int kSlotBytes = 32 * kBlock * 2;       // of an epilogue warp's 32 rows of them

// SLOTS: of shared memory for each epilogue warp
template <int CTAS, int N, int SLOTS>
struct Form {
  static constexpr int kRows = 128 * CTAS;        // of a tile
  static constexpr int kBRows = N / CTAS;         // of B that a CTA loads
  static constexpr int kABytes = 128 * kDepth * 2, kBBytes = kBRows * kDepth * 2, kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = kStageBytes > 32768 ? 4 : SLOTS == 2 ? 5 : 6;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kEpilogueWarps * SLOTS * kSlotBytes;      // 1024: the tiles start on a swizzle atom
  static constexpr int kCols = N / 2;             // of an epilogue thread
  static_assert(kSmem + 512 <= 232448 && kCols % kBlock == 0, "an SM's shared memory, whole blocks");
};

constexpr int kFirstStage = 1, kEightAtMost = 2, kAsked = 4;      // bits of what the diagnostics build withholds, see pb_debug_product_control

__device__ unsigned int g_status;                 // 0, or PB_ERR_DEVICE_TIMEOUT once a bounded wait ran out

struct Params {
  const int* count;         // where `counted` says so, the rows of D (1) or the extent of k (2) on the device
  int counted;
  int rows, cols, depth;    // extents of D and k; with `counted` the most that count may say
  int batch;
  int upper;                // only tiles that reach the diagonal or lie above it; where a block is stored once more transposed is the epilogue's affair
  int band;                 // tile rows that are walked down before the next column
  int bf16;                 // else fp16
  int group;                // stages of k that an accumulator takes
  int cuts, cut;            // 0: whole tiles; else the parts that a tile's stages are cut into, and their length
  uint32_t polls;
  int withhold;             // diagnostics build: kFirstStage, kAsked
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded: false, and the status word set, when the poll budget ran out.  One block of PTX, so that the loops that wait keep their state in registers.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t polls) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .u32 n;\n\tmov.u32 n, 0;\n"
      "WAIT_%=:\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, 2000;\n\t"
      "@p bra DONE_%=;\n\t"
      "add.u32 n, n, 1;\n\t"
      "setp.lt.u32 p, n, %3;\n\t"
      "@p bra WAIT_%=;\n\t"
      "setp.ne.u32 p, n, n;\n"
      "DONE_%=:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity), "r"(polls) : "memory");
  if (!ok) atomicExch(&g_status, (unsigned int)PB_ERR_DEVICE_TIMEOUT);
  return ok;
}
// the address of the same place in shared memory in the cluster's first CTA
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_in_cluster(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }
template <int CTAS>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if (CTAS == 2)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// arrives, when what this thread has issued is done, on the barrier at this place in every CTA of the tile
template <int CTAS>
__device__ __forceinline__ void commit_to(uint32_t bar) {
  if (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, uint32_t accumulate) {
  if (CTAS == 2)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(instr), "r"(accumulate) : "memory");
}
// Operand tiles (descriptor version 1, 128-byte swizzle).  K-major: rows of 128 bytes (64 of k), 8-row groups 1024 bytes apart.  M/N-major: for each 64
// of the operand's rows 64 k of 128 bytes, eight k 1024 bytes apart, the next 64 rows 8192.
template <bool MN>
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
  const uint64_t start = (uint64_t)((addr & 0x3ffffu) >> 4) | (1ull << 46) | ((uint64_t)(1024 >> 4) << 32) | (2ull << 61);
  return start | (MN ? (uint64_t)(8192 >> 4) << 16 : 1ull << 16);
}
template <bool MN> constexpr uint32_t kStep16 = MN ? 16 * 128 / 16 : 32 / 16;      // 16 of k further, in descriptor units
// kind::f16, f32 accumulator
template <int CTAS, int N, bool A_MN, bool B_MN>
constexpr uint32_t kInstr = (1u << 4) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 * CTAS >> 4) << 24);
constexpr uint32_t kBf16Operands = (1u << 7) | (1u << 10);

__device__ __forceinline__ void ld_acc32(uint32_t taddr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr) : "memory");
}
// until the load has arrived; the registers pass through, so that nothing reads them before
__device__ __forceinline__ void wait_acc32(float (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                 "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
                 "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
               :: "memory");
}

__device__ __forceinline__ void ld_acc16(uint32_t taddr, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void wait_acc16(float (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
               :: "memory");
}
template <int BLOCK>
__device__ __forceinline__ void ld_acc(uint32_t taddr, float (&r)[BLOCK]) {
#pragma unroll
  for (int j = 0; j < BLOCK; j += 32) ld_acc32(taddr + j, *reinterpret_cast<float(*)[32]>(&r[j]));
}
template <int BLOCK>
__device__ __forceinline__ void wait_acc(float (&r)[BLOCK]) {
#pragma unroll
  for (int j = 0; j < BLOCK; j += 32) wait_acc32(*reinterpret_cast<float(*)[32]>(&r[j]));
}

// by an instruction that no compiler makes without the condition (a volatile load in a conditional expression was made, of a null pointer)
__device__ __forceinline__ int counted_on_device(const Params& p) {
  int n = 0;
  if (p.counted) asm volatile("ld.global.b32 %0, [%1];" : "=r"(n) : "l"(p.count) : "memory");
  return n;
}

// What an epilogue is told of a thread's part of a tile: its row, its first column, and where they are on the chip.
struct Place {
  int batch, row, col;      // of D; the columns are col .. col + Form::kCols
  int rows, cols;           // D's extents
  int slice;                // of columns, Form::kCols
  bool beside_diagonal;     // with `upper`: the tile is not on the diagonal
  int lane;
  uint32_t slots, own, bar; // this warp's shared memory, the lane's row there (Slots), and a barrier for what is asked for
  uint32_t polls;
  bool withheld;            // diagnostics build: nothing that is asked for is sent for
  int part;                 // a number for this warp's part of the tile, among all of D
};

// ---- what epilogues share -------------------------------------------------------------------------------------------
struct Bf16 {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
struct Fp16 {
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t p;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
    return p;
  }
  static __device__ __forceinline__ float2 open(uint32_t p) { return __half22float2(*reinterpret_cast<const __half2*>(&p)); }
};
// A warp's blocks of 32 rows x kBlock 16-bit elements between registers, where a lane has a row, and memory: through slots of 4 KB in shared memory, as TMA's 128-byte swizzle lays
// them (16-byte pieces of a row exchanged by its number, so that neither side meets a bank twice).  TMA moves them: the same by loads and stores of the lanes, 64
// bytes of eight rows each, took the last product of a step of four 2048 x 8192 updates 282 us for 222, and a single 2048 x 2048 matrix's 31 for 22.5.
struct Slots {
  static constexpr int kBytes = 32 * kBlock * 2, kPieces = kBlock / 8;
  static __device__ __forceinline__ uint32_t own(const Place& at, int slot, int k) { return (at.own + slot * kBytes) ^ (k << 4); }      // the lane's row's k-th piece
  static __device__ __forceinline__ void put(uint32_t to, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
  }
  static __device__ __forceinline__ uint4 get(uint32_t from) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
    return v;
  }
  template <class T>
  static __device__ __forceinline__ void stage(const Place& at, int slot, const float (&v)[kBlock]) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k)
      put(own(at, slot, k), T::pack(v[8 * k], v[8 * k + 1]), T::pack(v[8 * k + 2], v[8 * k + 3]), T::pack(v[8 * k + 4], v[8 * k + 5]), T::pack(v[8 * k + 6], v[8 * k + 7]));
  }
  // the block's columns as rows of 32, without a swizzle
  static __device__ __forceinline__ void stage_transposed(const Place& at, int slot, const float (&v)[kBlock]) {
#pragma unroll
    for (int j = 0; j < kBlock; ++j)
      asm volatile("st.shared.b16 [%0], %1;" ::"r"(at.slots + slot * kBytes + j * 64 + at.lane * 2), "h"(__half_as_ushort(__float2half_rn(v[j]))) : "memory");
  }
  // Between a warp's accesses to its slots and TMA's: by all lanes.
  static __device__ __forceinline__ void hand_over() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
  }
  // by one lane
  static __device__ __forceinline__ void send(const Place& at, int slot, const CUtensorMap* map, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(at.slots + slot * kBytes), "r"(x), "r"(y), "r"(z) : "memory");
  }
  static __device__ __forceinline__ void sent() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
  static __device__ __forceinline__ void wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }      // until what was sent has left the slots
  static __device__ __forceinline__ void wait_sent() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
  static __device__ __forceinline__ void ask(const Place& at, int slot, const CUtensorMap* map, int x, int y, int z) { load_box<1>(at.slots + slot * kBytes, map, x, y, z, at.bar); }
  // A staged block to rows that TMA does not reach: row `to_row` of each lane's (below 0 none), `ld` elements apart from `first` on; n columns are there; vectors: rows begin at whole 16 bytes.
  static __device__ __noinline__ void scatter(uint32_t own, int lane, unsigned short* first, int64_t ld, int to_row, int n, bool vectors) {
    const uint32_t base = own - (lane * (kBlock * 2) + ((lane & 7) << 4));
    if (vectors && n >= kBlock) {
      const int piece = lane & 7;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3), to = __shfl_sync(0xffffffffu, to_row, r);
        const uint4 v = get(base + r * (kBlock * 2) + ((piece ^ (r & 7)) << 4));
        if (to >= 0) *reinterpret_cast<uint4*>(first + to * ld + 8 * piece) = v;
      }
    } else {
#pragma unroll 2
      for (int r = 0; r < 32; ++r) {
        const int row = __shfl_sync(0xffffffffu, to_row, r);
        unsigned short* to = first + row * ld;
#pragma unroll
        for (int c0 = 0; c0 < kBlock; c0 += 32) {
          const int c = c0 + lane;
          unsigned short x;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(base + r * (kBlock * 2) + (((c >> 3) ^ (r & 7)) << 4) + 2 * (c & 7)) : "memory");
          if (row >= 0 && c < n) to[c] = x;
        }
      }
    }
    __syncwarp();
  }
};

// Tiles of D, band by band.  upper: those with anything on or above the diagonal, column after column; a tile is `ratio` times as high as wide.
struct Tiles {
  int tiles_m, tiles_n, per_batch, band, upper, ratio;
  __host__ __device__ __forceinline__ Tiles(const Params& p, int rows, int tile_rows, int tile_cols) {
    tiles_m = (rows + tile_rows - 1) / tile_rows; tiles_n = (p.cols + tile_cols - 1) / tile_cols;
    band = p.band; upper = p.upper; ratio = tile_rows > tile_cols ? tile_rows / tile_cols : 1;
    const int high = tiles_n / ratio;
    per_batch = upper ? ratio * high * (high + 1) / 2 + tiles_n % ratio * (high + 1) : tiles_m * tiles_n;
  }
  __device__ __forceinline__ void at(int t, int& batch, int& tm, int& tn) const {
    batch = t / per_batch;
    t -= batch * per_batch;
    if (upper) {            // `ratio` columns of one tile, as many of two, ...
      int high = (int)((sqrtf(8.0f * (float)(t / ratio) + 1.0f) - 1.0f) * 0.5f);
      while (ratio * high * (high + 1) / 2 > t) --high;
      while (ratio * (high + 1) * (high + 2) / 2 <= t) ++high;
      t -= ratio * high * (high + 1) / 2;
      tn = high * ratio + t / (high + 1);
      tm = t % (high + 1);
      return;
    }
    const int whole = band * tiles_n, b = t / whole, within = t - b * whole, rows = min(band, tiles_m - b * band);
    tn = within / rows;
    tm = b * band + (within - tn * rows);
  }
};

// What a cluster works on: tiles in turn, or with p.cuts parts of `cut` stages of them: all tiles' first parts, then all tiles' second ones, ..., so that what is under way
// at a time reads the same of k.  (Runs of stages of one length for all clusters balance best, but then nothing is read twice from L2: 16384 of k, 8192 x
// 2048 sums 500 us for 370.)
struct Work {
  int at, items, stride, steps, tiles, cut, part;
  __device__ __forceinline__ Work(const Params& p, int tiles_, int steps_, int cluster, int clusters)
      : at(cluster), items(tiles_ * max(1, p.cuts)), stride(clusters), steps(steps_), tiles(tiles_), cut(p.cuts ? p.cut : steps_), part(0) {}
  // stages [k0, k1) of a tile; none where the last ones are not there
  __device__ __forceinline__ bool next(int& tile, int& k0, int& k1) {
    if (at >= items) return false;
    part = at / tiles;
    tile = at - part * tiles;
    k0 = min(steps, part * cut); k1 = min(steps, k0 + cut);
    at += stride;
    return true;
  }
};

// Epilogue: constructed from its Params by every thread of the epilogue warps, then for each tile, by whole warps, begin(place) before its sums are there, block(place, c, v) for each kBlock columns
// from place.col + c on (whatever lies outside of D zeros; not called for columns beyond it), and end(place); at last finish(place), in an abort too.  kSlots: 4 KB a warp each.
// kGrouped: sums of groups of stages are added up in registers, 128 of a thread, and the warps that load and issue hand over some of theirs.
template <int CTAS, int N, bool A_MN, bool B_MN, class Epilogue>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Params p,
               const __grid_constant__ typename Epilogue::Params e) {
  constexpr bool GROUPED = Epilogue::kGrouped;
  using F = Form<CTAS, N, Epilogue::kSlots>;
  extern __shared__ unsigned char product_smem[];
  __shared__ __align__(8) uint64_t bars[2 * F::kStages + 4 + kEpilogueWarps];
  __shared__ uint32_t tmem_slot;
  const uint32_t base = (smem_u32(product_smem) + 1023u) & ~1023u;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = CTAS == 2 ? (int)(blockIdx.x & 1) : 0;
  const bool leader = rank == 0;
  auto full = [&](int s) { return smem_u32(&bars[s]); };                            // used in the leader
  auto empty = [&](int s) { return smem_u32(&bars[F::kStages + s]); };              // one set per CTA
  auto acc_full = [&](int a) { return smem_u32(&bars[2 * F::kStages + a]); };       // one set per CTA
  auto acc_empty = [&](int a) { return smem_u32(&bars[2 * F::kStages + 2 + a]); };  // used in the leader
  if (tid == 0) {
    for (int s = 0; s < F::kStages; ++s) { bar_init(full(s), 1); bar_init(empty(s), 1); }
    for (int a = 0; a < 2; ++a) { bar_init(acc_full(a), 1); bar_init(acc_empty(a), CTAS * kEpilogueWarps); }
    for (int w = 0; w < kEpilogueWarps; ++w) bar_init(smem_u32(&bars[2 * F::kStages + 4 + w]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 32 * 2) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
  }
  if (warp == 1) {
    if (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((uint32_t)(2 * N)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((uint32_t)(2 * N)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_before();
  __syncthreads();
  if (CTAS == 2) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");      // both CTAs' barriers are there before any remote signal
  tc_after();
  const uint32_t tmem = *(volatile uint32_t*)&tmem_slot;
  grid_wait();
  const int count = counted_on_device(p);
  const int rows = p.counted == 1 ? count : p.rows, depth = p.counted == 2 ? count : p.depth;
  const int steps = (depth + kDepth - 1) / kDepth;
  const Tiles tiles(p, rows, F::kRows, N);
  const int items = tiles.per_batch * p.batch;
  Work work(p, items, steps, blockIdx.x / CTAS, gridDim.x / CTAS);

  // registers with GROUPED: 128 x 56 + 256 x 216 of the 384 x 168 that the block has
  if (warp < 4) {
    if (GROUPED) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        int w, k, k1;
        while (ok && work.next(w, k, k1)) {
          int batch, tm, tn;
          tiles.at(w, batch, tm, tn);
          const int m0 = tm * F::kRows + rank * 128, n0 = tn * N + rank * F::kBRows;
          for (; k < k1; ++k, ++it) {
            const int s = it % F::kStages;
            if (!bar_wait(empty(s), ((it / F::kStages) & 1) ^ 1, p.polls)) { ok = false; break; }
            if ((p.withhold & kFirstStage) && it == 0) continue;
            const uint32_t bar = CTAS == 2 ? in_leader(full(s)) : full(s), a = base + s * F::kStageBytes, b = a + F::kABytes;
            if (leader) bar_expect(full(s), CTAS * F::kStageBytes);
            if (A_MN) {
              load_box<CTAS>(a, &map_a, m0, k * kDepth, batch, bar);
              load_box<CTAS>(a + 8192, &map_a, m0 + 64, k * kDepth, batch, bar);
            } else {
              load_box<CTAS>(a, &map_a, k * kDepth, m0, batch, bar);
            }
            if (B_MN) {
#pragma unroll
              for (int j = 0; j < F::kBRows / 64; ++j) load_box<CTAS>(b + j * 8192, &map_b, n0 + 64 * j, k * kDepth, batch, bar);
            } else {
              load_box<CTAS>(b, &map_b, k * kDepth, n0, batch, bar);
            }
          }
        }
        // leave only when every copy that this pair started has landed (bounded)
        if (leader)
          for (uint32_t k = it > (uint32_t)F::kStages ? it - F::kStages : 0; k < it; ++k)
            if (!((p.withhold & kFirstStage) && k == 0)) (void)bar_wait(full(k % F::kStages), (k / F::kStages) & 1, p.polls);
      }
    } else if (warp == 1) {
      if (lane == 0 && leader) {
        const uint32_t instr = kInstr<CTAS, N, A_MN, B_MN> | (p.bf16 ? kBf16Operands : 0u);
        uint32_t it = 0, n = 0;
        bool ok = true;
        int w, begin, k1;
        while (ok && work.next(w, begin, k1)) {
          for (int k0 = begin; ok && (k0 == begin || k0 < k1); k0 += p.group, ++n) {
            const uint32_t ab = n & 1, d = tmem + ab * N;
            ok = bar_wait(acc_empty(ab), ((n >> 1) & 1) ^ 1, p.polls);
            tc_after();
            const int end = k1 - k0 < p.group ? k1 : k0 + p.group;
            for (int k = k0; ok && k < end; ++k, ++it) {
              const int s = it % F::kStages;
              if (!bar_wait(full(s), (it / F::kStages) & 1, p.polls)) { ok = false; break; }
              tc_after();
              const uint64_t a = tile_desc<A_MN>(base + s * F::kStageBytes), b = tile_desc<B_MN>(base + s * F::kStageBytes + F::kABytes);
#pragma unroll
              for (int j = 0; j < kDepth / 16; ++j) mma<CTAS>(d, a + (uint64_t)(j * kStep16<A_MN>), b + (uint64_t)(j * kStep16<B_MN>), instr, k > k0 || j > 0);
              commit_to<CTAS>(empty(s));
            }
            if (ok) commit_to<CTAS>(acc_full(ab));
          }
        }
      }
    }
  } else {
    if (GROUPED) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int quad = warp & 3, slice = (warp - 4) >> 2;      // rows 32 quad .., columns kCols slice ..
    Epilogue epilogue(e);
    Place at;
    at.rows = rows; at.cols = p.cols; at.lane = lane; at.slice = F::kCols;
    at.slots = base + F::kStages * F::kStageBytes + (warp - 4) * Epilogue::kSlots * kSlotBytes;
    at.own = at.slots + lane * (kBlock * 2) + ((lane & 7) << 4);
    at.bar = smem_u32(&bars[2 * F::kStages + 4 + warp - 4]);
    at.polls = p.polls; at.withheld = p.withhold & kAsked;
    uint32_t n = 0;
    bool ok = true;
    int w, begin, k1;
    while (ok && work.next(w, begin, k1)) {
      int tm, tn;
      tiles.at(w, at.batch, tm, tn);
      at.row = tm * F::kRows + rank * 128 + quad * 32 + lane;
      at.col = tn * N + slice * F::kCols;
      at.beside_diagonal = tm != tn / tiles.ratio;
      at.part = ((work.part * items + w) * CTAS + rank) * kEpilogueWarps + warp - 4;
      epilogue.begin(at);
      float acc[GROUPED ? F::kCols / kBlock : 1][kBlock];
      auto from = [&](uint32_t ab, int c) { return tmem + ((uint32_t)(quad * 32) << 16) + ab * N + slice * F::kCols + c; };
      auto release = [&](uint32_t ab) {
        tc_before();
        __syncwarp();
        if (lane == 0) arrive_in_cluster(CTAS == 2 ? in_leader(acc_empty(ab)) : acc_empty(ab));
      };
      for (int k0 = begin; k0 == begin || k0 < k1; k0 += p.group, ++n) {
        const uint32_t ab = n & 1;
        ok = __all_sync(0xffffffffu, bar_wait(acc_full(ab), (n >> 1) & 1, p.polls));
        if (!ok) break;
        tc_after();
        if constexpr (!GROUPED) {
#pragma unroll
          for (int c = 0; c < F::kCols; c += kBlock) {
            ld_acc(from(ab, c), acc[0]);
            wait_acc(acc[0]);
            if (begin == k1)          // nothing was added up
#pragma unroll
              for (int j = 0; j < kBlock; ++j) acc[0][j] = 0.0f;
            if (c + kBlock == F::kCols) release(ab);
            if (at.col + c < p.cols) epilogue.block(at, c, acc[0]);
          }
        } else {
          if (k0 == begin) {
#pragma unroll
            for (int c = 0; c < F::kCols / kBlock; ++c) ld_acc(from(ab, c * kBlock), acc[c]);
#pragma unroll
            for (int c = 0; c < F::kCols / kBlock; ++c) wait_acc(acc[c]);
          } else {
#pragma unroll
            for (int c = 0; c < F::kCols / 16; ++c) {
              float v[16];
              ld_acc16(from(ab, 16 * c), v);
              wait_acc16(v);
              float* sum = acc[16 * c / kBlock] + 16 * c % kBlock;
#pragma unroll
              for (int j = 0; j < 16; j += 2) {
                const float2 s = __fadd2_rn(make_float2(sum[j], sum[j + 1]), make_float2(v[j], v[j + 1]));
                sum[j] = s.x; sum[j + 1] = s.y;
              }
            }
          }
          release(ab);
        }
      }
      if (!ok) break;
      if constexpr (GROUPED) {
#pragma unroll
        for (int c = 0; c < F::kCols / kBlock; ++c) {
          if (begin == k1)            // nothing was added up
#pragma unroll
            for (int j = 0; j < kBlock; ++j) acc[c][j] = 0.0f;
          if (at.col + c * kBlock < p.cols) epilogue.block(at, c * kBlock, acc[c]);
        }
      }
      epilogue.end(at);
    }
    epilogue.finish(at);
  }
  // Neither CTA leaves, or frees TMEM, while the other can still signal its barriers or issue into its TMEM.
  tc_before();
  __syncthreads();
  if (CTAS == 2) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == 1) {
    tc_after();
    if (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(2 * N)) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(2 * N)) : "memory");
  }
}

// ---- products whose tiles are cut -----------------------------------------------------------------------------------
// The sums of a part of a tile's stages, 16 bytes a lane in a row; `add`: onto what is there, of a product before.
template <bool GROUPED>
struct PartEpilogue {
  static constexpr bool kGrouped = GROUPED;
  static constexpr int kSlots = 1;
  struct Params { float4* parts; bool add; };
  const Params& p;
  __device__ __forceinline__ explicit PartEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void begin(const Place&) {}
  __device__ __forceinline__ void block(const Place& at, int c, float (&v)[kBlock]) {
    float4* to = p.parts + ((int64_t)at.part * at.slice + c) * 8 + at.lane;
#pragma unroll
    for (int j = 0; j < kBlock / 4; ++j) {
      float4 f = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      if (p.add) {
        const float4 g = to[32 * j];
        f.x += g.x; f.y += g.y; f.z += g.z; f.w += g.w;
      }
      to[32 * j] = f;
    }
  }
  __device__ __forceinline__ void end(const Place&) {}
  __device__ __forceinline__ void finish(const Place&) {}
};
// A tile's parts together, in their order, and its epilogue: a CTA for 128 rows of a tile and one block of each of the epilogue's warps.
template <int CTAS, int N, class Epilogue>
__global__ void __launch_bounds__(32 * kEpilogueWarps) finish_kernel(const float4* parts, const __grid_constant__ Params p, const __grid_constant__ typename Epilogue::Params e) {
  using F = Form<CTAS, N, Epilogue::kSlots>;
  extern __shared__ unsigned char finish_smem[];
  __shared__ __align__(8) uint64_t bars[kEpilogueWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = warp & 3, slice = warp >> 2;
  if (threadIdx.x < kEpilogueWarps) bar_init(smem_u32(&bars[threadIdx.x]), 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();
  grid_wait();
  const int count = counted_on_device(p);
  const int rows = p.counted == 1 ? count : p.rows;
  const Tiles tiles(p, rows, F::kRows, N);
  const int items = tiles.per_batch * p.batch, w = blockIdx.x / CTAS, rank = blockIdx.x % CTAS;
  if (w >= items) return;
  Epilogue epilogue(e);
  Place at;
  int tm, tn;
  tiles.at(w, at.batch, tm, tn);
  at.rows = rows; at.cols = p.cols; at.lane = lane; at.slice = F::kCols; at.polls = p.polls; at.withheld = false;
  at.slots = ((smem_u32(finish_smem) + 1023u) & ~1023u) + warp * Epilogue::kSlots * kSlotBytes;
  at.own = at.slots + lane * (kBlock * 2) + ((lane & 7) << 4);
  at.bar = smem_u32(&bars[warp]);
  at.row = tm * F::kRows + rank * 128 + quad * 32 + lane;
  at.col = tn * N + slice * F::kCols;
  at.beside_diagonal = tm != tn / tiles.ratio;
  at.part = 0;
  epilogue.begin(at);
  const int c = blockIdx.y * kBlock;
  if (at.col + c < p.cols) {
    float v[kBlock];
#pragma unroll
    for (int j = 0; j < kBlock; ++j) v[j] = 0.0f;
#pragma unroll 2
    for (int k = 0; k < p.cuts; ++k) {
      const float4* from = parts + (((int64_t)k * items + w) * CTAS + rank) * kEpilogueWarps * (F::kCols * 8) + (warp * F::kCols + c) * 8 + lane;
#pragma unroll
      for (int j = 0; j < kBlock / 4; ++j) {
        const float4 f = from[32 * j];
        v[4 * j] += f.x; v[4 * j + 1] += f.y; v[4 * j + 2] += f.z; v[4 * j + 3] += f.w;
      }
    }
    epilogue.block(at, c, v);
  }
  epilogue.end(at);
  epilogue.finish(at);
}

// ---- host side --------------------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// `batch` matrices of [outer, inner] 16-bit elements, rows `ld` apart (a multiple of 8), matrices `plane`; boxes of 64 (inner) x box_outer, swizzled, or of fewer (inner), as they are
inline int make_map(CUtensorMap* map, const void* base, bool bf16, int64_t inner, int64_t outer, int64_t ld, int64_t batch, int64_t plane, int box_outer, int box_inner = kDepth) {
  EncodeFn encode = reinterpret_cast<EncodeFn>(tensor_map_encoder());
  if (!encode) return fail(PB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)batch};
  const cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(plane * 2)};
  const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, box_inner == kDepth ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(PB_ERR_CUDA, "cuTensorMapEncodeTiled (products) failed with CUresult %d", (int)r);
  return PB_OK;
}

#ifdef PB_DIAGNOSTICS
std::atomic<uint32_t> g_polls{kWaitPolls};
std::atomic<int> g_withhold{0};
inline void control(uint32_t polls, int withhold) {
  g_polls.store(polls ? polls : kWaitPolls);
  g_withhold.store(withhold);
}
#endif

// An operand: `rows` (of D's rows or columns) x depth, its k lying together or (mn) its rows
struct Operand {
  const void* at;
  bool mn;
  int64_t rows, depth, ld, plane;
};

template <int CTAS> int64_t clusters_of() { return sm_count() / CTAS; }
template <int CTAS, int N>
int64_t tiles_of(const Params& p) {      // with `counted` rows: at most
  const int64_t tm = (p.rows + 128 * CTAS - 1) / (128 * CTAS), tn = (p.cols + N - 1) / N, ratio = 128 * CTAS > N ? 128 * CTAS / N : 1, high = tn / ratio;
  return p.batch * (p.upper ? ratio * high * (high + 1) / 2 + tn % ratio * (high + 1) : tm * tn);
}
template <int CTAS, int N>
void set_common(Params* p) {
  // a band's rows of A, some 16 MB, stay in L2 while its columns go by
  p->band = (int)std::min<int64_t>((p->rows + 128 * CTAS - 1) / (128 * CTAS), std::max<int64_t>(1, (16 << 20) / (128 * CTAS * 2 * std::max<int64_t>(1, p->cuts ? (int64_t)p->cut * kDepth : p->depth))));
  p->polls = kWaitPolls; p->withhold = 0;
#ifdef PB_DIAGNOSTICS
  p->polls = g_polls.load(); p->withhold = g_withhold.load();
#endif
}

template <int CTAS, int N, bool A_MN, bool B_MN, class Epilogue>
int launch(const Operand& a, const Operand& b, Params p, const typename Epilogue::Params& e, cudaStream_t st) {
  using F = Form<CTAS, N, Epilogue::kSlots>;
  CUtensorMap map_a, map_b;
  auto map = [&](CUtensorMap* m, const Operand& o, int box_rows) {
    return o.mn ? make_map(m, o.at, p.bf16, o.rows, o.depth, o.ld, p.batch, o.plane, kDepth) : make_map(m, o.at, p.bf16, o.depth, o.rows, o.ld, p.batch, o.plane, box_rows);
  };
  if (int s = map(&map_a, a, 128)) return s;
  if (int s = map(&map_b, b, F::kBRows)) return s;
  const int64_t items = tiles_of<CTAS, N>(p);
  if (items > kMaxIndexed / 2) return fail(PB_ERR_BAD_SHAPE, "%lld tiles of a product", (long long)items);
  if (items == 0) return PB_OK;
  if (!Epilogue::kGrouped) p.group = 1 << 24;      // more stages than there are, and added to one of them within an int
  set_common<CTAS, N>(&p);
  auto kernel = product_kernel<CTAS, N, A_MN, B_MN, Epilogue>;
  PB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem));      // per device
  const int64_t clusters = std::min<int64_t>(items * std::max(1, p.cuts), clusters_of<CTAS>());
  launch_behind(kernel, (unsigned)(clusters * CTAS), kThreads, F::kSmem, st, map_a, map_b, p, e);
  PB_LAUNCH_CHECK("product_kernel");
  return PB_OK;
}

// Cuts a product of few tiles, or of a few more than whole rounds of them, where that pays: a part costs its rounds and, for its accumulators, about kPartCost stages more, and the
// joining of all parts a stage for every kJoinParts of them.  At most kMostCuts parts of eight stages at least.
constexpr int kPartCost = 10, kJoinParts = 6, kMostCuts = 32;
template <int CTAS, int N>
void cut_stages(Params* p, int stages) {
  const int64_t tiles = tiles_of<CTAS, N>(*p), clusters = clusters_of<CTAS>();
  int64_t best = 0;
  for (int n = 1; n <= kMostCuts && (n == 1 || stages / n >= 8); ++n) {
    const int64_t cut = (stages + n - 1) / n, cost = (tiles * n + clusters - 1) / clusters * (cut + kPartCost) + tiles * n / kJoinParts;
    if (n > 1 && cost >= best) continue;
    best = cost; p->cuts = n; p->cut = (int)cut;
  }
  p->cuts = (stages + p->cut - 1) / std::max(1, p->cut);
}
// float4s that the parts of a cut product take
template <int CTAS, int N>
int64_t parts_of(const Params& p) { return tiles_of<CTAS, N>(p) * p.cuts * CTAS * (128 * N / 4); }

template <int CTAS, int N, class Epilogue>
int launch_finish(const float4* parts, Params p, const typename Epilogue::Params& e, cudaStream_t st) {
  const int64_t items = tiles_of<CTAS, N>(p);
  if (items == 0) return PB_OK;
  set_common<CTAS, N>(&p);
  constexpr int kSmem = 1024 + kEpilogueWarps * Epilogue::kSlots * kSlotBytes;
  auto kernel = finish_kernel<CTAS, N, Epilogue>;
  PB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  launch_behind(kernel, dim3((unsigned)(items * CTAS), Form<CTAS, N, Epilogue::kSlots>::kCols / kBlock), 32 * kEpilogueWarps, kSmem, st, parts, p, e);
  PB_LAUNCH_CHECK("finish_kernel");
  return PB_OK;
}

inline int status_fetch(unsigned int* out) {
  const unsigned int zero = 0;
  PB_CUDA_TRY(cudaMemcpyFromSymbol(out, g_status, sizeof(*out)));
  if (*out != 0) PB_CUDA_TRY(cudaMemcpyToSymbol(g_status, &zero, sizeof(zero)));
  return PB_OK;
}

}  // namespace
}  // namespace products
}  // namespace pb
