// Products of 16-bit operands on the tensor cores for the operators that are built around one: D[m, n] = sum_k A[m, k] B[n, k] in f32, handed to
// an epilogue of the operator's own (loss statistics, a gradient, a polynomial's term) in the registers that read the accumulator.
//
// A and B are both bf16 or both fp16, each with k or with its rows lying together in memory (K-major, or M/N-major): TMA takes either
// into 128-byte swizzled tiles and the matrix descriptors say which, so that no operand is ever transposed.  A tile is 128 CTAS x N:
//   CTAS = 2: a cluster of two CTAs makes 256 x 256; each loads its own 128 rows of A and its own 128 of B (32 KB per 64 of k and
//             SM, where one CTA's 128 x 256 takes 48: what a tile loads from L2 is the nearest bound beside the tensor core);
//   CTAS = 1: 128 x 128, for products that have few tiles.
// Persistent: warp 0 loads, a lane of warp 1 (of the leading CTA) issues tcgen05.mma, eight warps empty one accumulator of TMEM while the
// other fills, each thread one row and half of the columns.  Every wait is bounded and reported by pb_gemm_check.
// The tensor core's own additions do not round to nearest: an accumulator takes `group` stages of k, and the sums of a tile's groups are added up in the
// registers that read them.  2-norm errors of the loss of 64 positions of 2048 against 64 bits: one group 1.4e-6, groups of 512 of k GROUP_ERROR.
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
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 128 + 32 * kEpilogueWarps;
constexpr uint32_t kWaitPolls = 1u << 21;         // a poll parks for up to 2 us: about four seconds at most

template <int CTAS, int N>
struct Form {
  static constexpr int kRows = 128 * CTAS;        // of a tile
  static constexpr int kBRows = N / CTAS;         // of B that a CTA loads
  static constexpr int kABytes = 128 * kDepth * 2, kBBytes = kBRows * kDepth * 2, kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 6;
  static constexpr int kPitch = 34;               // 16-bit elements of a staged row: odd in words, so that columns of it meet no bank twice
  static constexpr int kStaging = 32 * kPitch * 2;                                       // of an epilogue warp: 32 x 32 elements
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kEpilogueWarps * kStaging;      // 1024: the tiles start on a swizzle atom
  static constexpr int kCols = N / 2;             // of an epilogue thread
  static_assert(kSmem + 512 <= 232448, "an SM's shared memory");
};

__device__ unsigned int g_status;                 // 0, or PB_ERR_DEVICE_TIMEOUT once a bounded wait ran out

struct Params {
  const int* count;         // where `counted` says so, the rows of D (1) or the extent of k (2) on the device
  int counted;
  int rows, cols, depth;    // extents of D and k; with `counted` the most that count may say
  int batch;
  int upper;                // only tiles on and above the diagonal (CTAS * 128 == N)
  int band;                 // tile rows that are walked down before the next column
  int bf16;                 // else fp16
  int group;                // stages of k that an accumulator takes
  uint32_t polls;
  int withhold;             // diagnostics build: the first stage is never filled
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

// What an epilogue is told of a thread's part of a tile: its row, its first column, and where they are on the chip.
struct Place {
  int batch, row, col;      // of D; the columns are col .. col + Form::kCols
  int rows, cols;           // D's extents
  bool beside;              // with `upper`: the tile is not on the diagonal
  int lane;
  uint32_t staging;         // this warp's shared memory, Form::kStaging bytes
};

struct Tiles {
  int tiles_m, tiles_n, per_batch, band, upper;
  __device__ __forceinline__ Tiles(const Params& p, int rows, int tile_rows, int tile_cols) {
    tiles_m = (rows + tile_rows - 1) / tile_rows; tiles_n = (p.cols + tile_cols - 1) / tile_cols;
    per_batch = p.upper ? tiles_n * (tiles_n + 1) / 2 : tiles_m * tiles_n;
    band = p.band; upper = p.upper;
  }
  __device__ __forceinline__ void at(int t, int& batch, int& tm, int& tn) const {
    batch = t / per_batch;
    t -= batch * per_batch;
    if (upper) {            // column after column down to the diagonal
      tn = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
      while (tn * (tn + 1) / 2 > t) --tn;
      while ((tn + 1) * (tn + 2) / 2 <= t) ++tn;
      tm = t - tn * (tn + 1) / 2;
      return;
    }
    const int whole = band * tiles_n, b = t / whole, within = t - b * whole, rows = min(band, tiles_m - b * band);
    tn = within / rows;
    tm = b * band + (within - tn * rows);
  }
};

// Epilogue: constructed from its Params by every thread of the epilogue warps, then for each tile begin(place), chunk<C>(place, c, v) for each 32 columns from
// place.col + c on (D's own sums, whatever lies outside of it zeros; not called for columns beyond it), and end(place), by whole warps.
template <int CTAS, int N, bool A_MN, bool B_MN, class Epilogue>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Params p,
               const __grid_constant__ typename Epilogue::Params e) {
  using F = Form<CTAS, N>;
  extern __shared__ unsigned char product_smem[];
  __shared__ __align__(8) uint64_t bars[2 * F::kStages + 4];
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
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
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
  const int count = p.counted ? *(const volatile int*)p.count : 0;
  const int rows = p.counted == 1 ? count : p.rows, depth = p.counted == 2 ? count : p.depth;
  const int steps = (depth + kDepth - 1) / kDepth;
  const Tiles tiles(p, rows, F::kRows, N);
  const int items = tiles.per_batch * p.batch, first = blockIdx.x / CTAS, stride = gridDim.x / CTAS;

  // registers: 128 x 56 + 256 x 216 of the 384 x 168 that the block has
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int w = first; w < items && ok; w += stride) {
          int batch, tm, tn;
          tiles.at(w, batch, tm, tn);
          const int m0 = tm * F::kRows + rank * 128, n0 = tn * N + rank * F::kBRows;
          for (int k = 0; k < steps; ++k, ++it) {
            const int s = it % F::kStages;
            if (!bar_wait(empty(s), ((it / F::kStages) & 1) ^ 1, p.polls)) { ok = false; break; }
            if (p.withhold && it == 0) continue;
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
            if (!(p.withhold && k == 0)) (void)bar_wait(full(k % F::kStages), (k / F::kStages) & 1, p.polls);
      }
    } else if (warp == 1) {
      if (lane == 0 && leader) {
        const uint32_t instr = kInstr<CTAS, N, A_MN, B_MN> | (p.bf16 ? kBf16Operands : 0u);
        uint32_t it = 0, n = 0;
        bool ok = true;
        for (int w = first; w < items && ok; w += stride) {
          for (int k0 = 0; ok && (k0 == 0 || k0 < steps); k0 += p.group, ++n) {
            const uint32_t ab = n & 1, d = tmem + ab * N;
            ok = bar_wait(acc_empty(ab), ((n >> 1) & 1) ^ 1, p.polls);
            tc_after();
            const int end = min(steps, k0 + p.group);
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int quad = warp & 3, half = (warp - 4) >> 2;      // rows 32 quad .., columns kCols half ..
    Epilogue epilogue(e);
    Place at;
    at.rows = rows; at.cols = p.cols; at.lane = lane;
    at.staging = base + F::kStages * F::kStageBytes + (warp - 4) * F::kStaging;
    uint32_t n = 0;
    bool ok = true;
    for (int w = first; w < items && ok; w += stride) {
      int tm, tn;
      tiles.at(w, at.batch, tm, tn);
      at.row = tm * F::kRows + rank * 128 + quad * 32 + lane;
      at.col = tn * N + half * F::kCols;
      at.beside = tm != tn;
      float acc[F::kCols / 32][32];
      for (int k0 = 0; k0 == 0 || k0 < steps; k0 += p.group, ++n) {
        const uint32_t ab = n & 1;
        ok = __all_sync(0xffffffffu, bar_wait(acc_full(ab), (n >> 1) & 1, p.polls));
        if (!ok) break;
        tc_after();
        const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + ab * N + half * F::kCols;
        const uint32_t freed = CTAS == 2 ? in_leader(acc_empty(ab)) : acc_empty(ab);
        if (k0 == 0) {
#pragma unroll
          for (int c = 0; c < F::kCols / 32; ++c) ld_acc32(from + 32 * c, acc[c]);
#pragma unroll
          for (int c = 0; c < F::kCols / 32; ++c) wait_acc32(acc[c]);
        } else {
#pragma unroll
          for (int c = 0; c < F::kCols / 32; ++c) {
            float v[32];
            ld_acc32(from + 32 * c, v);
            wait_acc32(v);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 s = __fadd2_rn(make_float2(acc[c][j], acc[c][j + 1]), make_float2(v[j], v[j + 1]));
              acc[c][j] = s.x; acc[c][j + 1] = s.y;
            }
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) arrive_in_cluster(freed);
      }
      if (!ok) break;
      if (steps == 0) {             // nothing was added up
#pragma unroll
        for (int c = 0; c < F::kCols / 32; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c][j] = 0.0f;
      }
      epilogue.begin(at);
#pragma unroll
      for (int c = 0; c < F::kCols / 32; ++c)
        if (at.col + 32 * c < p.cols) epilogue.chunk(at, 32 * c, acc[c]);
      epilogue.end(at);
    }
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
__device__ __forceinline__ void st_global_32bytes(void* at, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// 32 elements of a row as two whole 32-byte stores
template <class T>
__device__ __forceinline__ void store_row32(void* at, const float (&v)[32]) {
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = T::pack(v[2 * j], v[2 * j + 1]);
  st_global_32bytes(at, w);
  st_global_32bytes(static_cast<char*>(at) + 32, w + 8);
}
// A warp's 32 x 32 elements to rows that lie anywhere: through shared memory, so that a warp's store is 64 bytes of one row.  row_of(r): where lane r's row begins at these
// columns, or null.
template <class T>
__device__ __forceinline__ void store_block32(const Place& at, unsigned short* row, int n, const float (&v)[32]) {
  constexpr int kWords = Form<1, 128>::kPitch / 2;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at.staging + 4 * (at.lane * kWords + j)), "r"(T::pack(v[2 * j], v[2 * j + 1])) : "memory");
  __syncwarp();
  const unsigned long long mine = reinterpret_cast<unsigned long long>(row);
#pragma unroll 8
  for (int r = 0; r < 32; ++r) {
    unsigned short* to = reinterpret_cast<unsigned short*>(__shfl_sync(0xffffffffu, mine, r));
    unsigned short x;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at.staging + 4 * r * kWords + 2 * at.lane));
    if (to && at.lane < n) to[at.lane] = x;
  }
  __syncwarp();
}

// ---- host side --------------------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// `batch` matrices of [outer, inner] 16-bit elements, rows `ld` apart (a multiple of 8), matrices `plane`; boxes of 64 (inner) x box_outer
inline int make_map(CUtensorMap* map, const void* base, bool bf16, int64_t inner, int64_t outer, int64_t ld, int64_t batch, int64_t plane, int box_outer) {
  EncodeFn encode = reinterpret_cast<EncodeFn>(tensor_map_encoder());
  if (!encode) return fail(PB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)batch};
  const cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(plane * 2)};
  const cuuint32_t box[3] = {(cuuint32_t)kDepth, (cuuint32_t)box_outer, 1}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(PB_ERR_CUDA, "cuTensorMapEncodeTiled (products) failed with CUresult %d", (int)r);
  return PB_OK;
}

#ifdef PB_DIAGNOSTICS
std::atomic<uint32_t> g_polls{kWaitPolls};
std::atomic<int> g_withhold{0};
#endif

// An operand: `rows` (of D's rows or columns) x depth, its k lying together or (mn) its rows
struct Operand {
  const void* at;
  bool mn;
  int64_t rows, depth, ld, plane;
};

template <int CTAS, int N, bool A_MN, bool B_MN, class Epilogue>
int launch(const Operand& a, const Operand& b, Params p, const typename Epilogue::Params& e, cudaStream_t st) {
  using F = Form<CTAS, N>;
  CUtensorMap map_a, map_b;
  auto map = [&](CUtensorMap* m, const Operand& o, int box_rows) {
    return o.mn ? make_map(m, o.at, p.bf16, o.rows, o.depth, o.ld, p.batch, o.plane, kDepth) : make_map(m, o.at, p.bf16, o.depth, o.rows, o.ld, p.batch, o.plane, box_rows);
  };
  if (int s = map(&map_a, a, 128)) return s;
  if (int s = map(&map_b, b, F::kBRows)) return s;
  const int64_t tm = (p.rows + F::kRows - 1) / F::kRows, tn = (p.cols + N - 1) / N, items = p.batch * (p.upper ? tn * (tn + 1) / 2 : tm * tn);
  if (items > kMaxIndexed / 2) return fail(PB_ERR_BAD_SHAPE, "%lld tiles of a product", (long long)items);
  if (items == 0) return PB_OK;
  // a band's rows of A, some 16 MB, stay in L2 while its columns go by
  p.band = (int)std::max<int64_t>(1, (16 << 20) / (F::kRows * 2 * std::max<int64_t>(1, p.depth)));
  if (p.group == 0) p.group = kMaxIndexed;
  p.polls = kWaitPolls; p.withhold = 0;
#ifdef PB_DIAGNOSTICS
  p.polls = g_polls.load(); p.withhold = g_withhold.load();
#endif
  auto kernel = product_kernel<CTAS, N, A_MN, B_MN, Epilogue>;
  PB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem));      // per device
  const int64_t clusters = std::min<int64_t>(items, sm_count() / CTAS);
  launch_behind(kernel, (unsigned)(clusters * CTAS), kThreads, F::kSmem, st, map_a, map_b, p, e);
  PB_LAUNCH_CHECK("product_kernel");
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
