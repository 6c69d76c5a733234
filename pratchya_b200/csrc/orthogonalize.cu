// The orthogonalised update of a weight by Newton-Schulz products, the step of the reference's optimizer that follows its momentum for 2-D weights
// (newton_schulz, pratchya/_nnx_impl/_optimizer.py:11-29): X = G / (|G| + eps), then `steps` times
//   A = X X^T,   X <- a X + (b A + c A A) X       (rows <= cols; else A = X^T X and X <- a X + X (b A + c A A)),
// an odd polynomial of X's singular values that draws them all towards 1.
//
// X is kept as two fp16 terms of 2^12 X (22 bits), of which the products take the first; A and B = b A + c A A as one fp16 term of 2^10 times
// them.  What rounding leaves in directions that G does not have is the reason: there A and B vanish, only a X acts, and
// it multiplies what is there by 3.44 a step, 485 in five.  With X in one term a rank-1 update was 15 % off (in bf16 150 %); with two, 3e-4, while
// what the products' operands lose stays with the direction it belongs to (1.2e-3 of a full-rank update, 1.66e-3 is the output's own bf16).
// fp16 and not bf16: three more bits, and the polynomial keeps every value within range.
//
// Three products a step (products.cuh).  A and B are symmetric: only tiles on and above the diagonal are made, and stored to both places.
#include <cmath>
#include <mutex>
#include <utility>

#include "products.cuh"

namespace pb {
namespace {
using namespace products;

constexpr float kScaleX = 0x1p12f, kScaleA = 0x1p10f;
constexpr int kParts = 256;           // of a matrix, for its sum of squares
constexpr float kMostX = 4.0f, kMostB = 32.0f;      // of the polynomial on [0, 1] and what it makes of that: half of fp16's range at most

// ---- G -> X -------------------------------------------------------------------------------------------------------
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void open(const uint4& v, float* x) { x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void open(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[2 * j] = __uint_as_float(w[j] << 16); x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
  }
};

// sums[batch][kParts]: in 64 bits, so that no square of an f32 leaves the range
template <typename T>
__global__ void __launch_bounds__(256) square_sums_kernel(const T* g, int64_t n, bool vectors, double* sums) {
  grid_wait();
  __shared__ double red[8];
  const T* x = g + (int64_t)blockIdx.y * n;
  double s = 0.0;
  if (vectors) {
    constexpr int kN = Vec<T>::kN;
    const uint4* v = reinterpret_cast<const uint4*>(x);
    const int64_t whole = n / kN;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < whole; i += kParts * 256 * 4) {
      uint4 w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = i + k * kParts * 256 < whole ? __ldg(v + i + k * kParts * 256) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[kN];
        Vec<T>::open(w[k], f);
#pragma unroll
        for (int j = 0; j < kN; ++j) s = fma((double)f[j], (double)f[j], s);
      }
    }
  } else {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += kParts * 256) {
      const double f = (double)Elem<T>::to_f32(x[i]);
      s = fma(f, f, s);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) s += red[w];
    sums[(int64_t)blockIdx.y * kParts + blockIdx.x] = s;
  }
}

// 2^12 / (|G| + eps), of |G|^2 = s, as two powers of two and a rest in [1, 2): each within f32 where the whole may not be (2^161 for the least f32 alone).  NaN for an infinity or a NaN
// anywhere.  Nothing but zeros stays so by any factor that is a number; under a tiny eps the formula's own is none.
__device__ __forceinline__ void scale_factors(double s, double eps, float* factors) {
  const double by = s == 0.0 && eps > 0.0 ? 1.0 : (double)kScaleX / (sqrt(s) + eps);
  int e = 0;
  const double rest = 2.0 * frexp(by, &e);
  const bool fine = isfinite(by) && isfinite(s);
  e -= 1;
  factors[0] = fine ? (float)rest : nanf("");
  factors[1] = fine ? ldexpf(1.0f, e / 2) : 1.0f;
  factors[2] = fine ? ldexpf(1.0f, e - e / 2) : 1.0f;
}

__device__ __forceinline__ void two_terms(float x, __half& hi, __half& lo) {
  hi = __float2half_rn(x);
  lo = __float2half_rn(x - __half2float(hi));
}

struct SplitParams {
  const void* g;
  const double* sums;
  __half *hi, *lo;
  int64_t rows, cols, ld;
  double eps;
  bool vectors;
};
// eight columns of a row a thread
template <typename T>
__global__ void __launch_bounds__(256) normalise_kernel(const __grid_constant__ SplitParams p) {
  grid_wait();
  __shared__ float factors[3];
  if (threadIdx.x < 32) {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kParts / 32; ++k) s += p.sums[(int64_t)blockIdx.y * kParts + 32 * k + threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) {
      scale_factors(s, p.eps, factors);
    }
  }
  __syncthreads();
  const int64_t per_row = p.ld / 8, v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = v / per_row, col = (v - row * per_row) * 8;
  if (row >= p.rows || col >= p.cols) return;
  const T* x = static_cast<const T*>(p.g) + ((int64_t)blockIdx.y * p.rows + row) * p.cols + col;
  float f[8];
  if (p.vectors) {
#pragma unroll
    for (int j = 0; j < 8; j += Vec<T>::kN) Vec<T>::open(__ldg(reinterpret_cast<const uint4*>(x + j)), f + j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = col + j < p.cols ? Elem<T>::to_f32(x[j]) : 0.0f;
  }
  __align__(16) __half hi[8], lo[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) two_terms(f[j] * factors[1] * factors[2] * factors[0], hi[j], lo[j]);
  const int64_t to = ((int64_t)blockIdx.y * p.rows + row) * p.ld + col;
  *reinterpret_cast<uint4*>(p.hi + to) = *reinterpret_cast<const uint4*>(hi);
  *reinterpret_cast<uint4*>(p.lo + to) = *reinterpret_cast<const uint4*>(lo);
}

// ---- the epilogues ------------------------------------------------------------------------------------------------
struct Ungrouped { static constexpr bool kGrouped = false; static constexpr int kSlots = 2; };

// where a symmetric matrix's blocks go: by its rows, and where the tile is beside the diagonal the same numbers by its columns
struct Symmetric { CUtensorMap rows, columns; };
__device__ __forceinline__ void store_both(const Place& at, int c, const Symmetric& to, const float (&v)[kBlock]) {
  Slots::stage<Fp16>(at, 0, v);
  if (at.beside_diagonal) Slots::stage_transposed(at, 1, v);
  Slots::hand_over();
  if (at.lane == 0 && at.row < at.rows) {
    Slots::send(at, 0, &to.rows, at.col + c, at.row, at.batch);
    if (at.beside_diagonal) Slots::send(at, 1, &to.columns, at.row, at.col + c, at.batch);
    Slots::sent();
  }
}
// until the slots can be written to again
__device__ __forceinline__ void wait_slots(const Place& at) {
  if (at.lane == 0) Slots::wait_read();
  __syncwarp();
}
// v = of_v * v + by * the lane's row of what a slot holds
__device__ __forceinline__ void add_rows(const Place& at, int slot, float of_v, float by, float (&v)[kBlock]) {
#pragma unroll
  for (int k = 0; k < Slots::kPieces; ++k) {
    const uint4 w = Slots::get(Slots::own(at, slot, k));
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 x = Fp16::open(words[j]), y = make_float2(v[8 * k + 2 * j], v[8 * k + 2 * j + 1]);
      if (of_v != 1.0f) y = __fmul2_rn(y, make_float2(of_v, of_v));
      y = __ffma2_rn(x, make_float2(by, by), y);
      v[8 * k + 2 * j] = y.x; v[8 * k + 2 * j + 1] = y.y;
    }
  }
}

struct GramEpilogue : Ungrouped {
  struct Params { Symmetric a; };
  const Params& p;
  __device__ __forceinline__ explicit GramEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void begin(const Place&) {}
  __device__ __forceinline__ void block(const Place& at, int c, float (&v)[kBlock]) {
    wait_slots(at);
#pragma unroll
    for (int j = 0; j < kBlock; ++j) v[j] *= kScaleA / (kScaleX * kScaleX);
    store_both(at, c, p.a, v);
  }
  __device__ __forceinline__ void end(const Place&) {}
  __device__ __forceinline__ void finish(const Place& at) { if (at.lane == 0) Slots::wait_sent(); }
};

// Blocks that are read before they are written: asked for a block ahead, as soon as the slots have been read out.  `pending`: on their way.  `lost`: the wait for one ran out; its
// barrier's phase stays open, so nothing more is asked for, read or written, and the end waits for it once more.
struct Reading : Ungrouped {
  uint32_t phase = 0;
  bool pending = false, lost = false;
  __device__ __forceinline__ bool arrived(const Place& at) {
    if (lost) return false;
    lost = !__all_sync(0xffffffffu, bar_wait(at.bar, phase, at.polls));
    if (lost) return false;
    phase ^= 1; pending = false;
    return true;
  }
  __device__ __forceinline__ bool asks(const Place& at, int c) {
    if (lost || c >= at.slice || at.col + c >= at.cols) return false;
    pending = true;
    return at.lane == 0 && !at.withheld;
  }
  __device__ __forceinline__ void finish(const Place& at) {
    if (pending) (void)bar_wait(at.bar, phase, at.polls);
    if (at.lane == 0) Slots::wait_sent();
  }
};

struct SquareEpilogue : Reading {
  struct Params { CUtensorMap a; Symmetric b; float of_a, of_square; };
  const Params& p;
  __device__ __forceinline__ explicit SquareEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void ask(const Place& at, int c) {
    if (!asks(at, c)) return;
    Slots::wait_read();
    bar_expect(at.bar, kSlotBytes);
    Slots::ask(at, 0, &p.a, at.col + c, at.row, at.batch);
  }
  __device__ __forceinline__ void begin(const Place& at) { ask(at, 0); }
  __device__ __forceinline__ void block(const Place& at, int c, float (&v)[kBlock]) {
    if (!arrived(at)) return;
    add_rows(at, 0, p.of_square, p.of_a, v);
    __syncwarp();
    store_both(at, c, p.b, v);
    ask(at, c + kBlock);
  }
  __device__ __forceinline__ void end(const Place&) {}
};

// LAST: X leaves as bf16, by TMA or, where its rows do not begin at whole 16 bytes, by the lanes
template <bool LAST>
struct UpdateEpilogue : Reading {
  struct Params { CUtensorMap hi, lo, hi_out, lo_out; __nv_bfloat16* out; int64_t out_ld, out_plane; bool whole; float of_x; };
  const Params& p;
  __device__ __forceinline__ explicit UpdateEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void ask(const Place& at, int c) {
    if (!asks(at, c)) return;
    Slots::wait_read();
    bar_expect(at.bar, 2 * kSlotBytes);
    Slots::ask(at, 0, &p.hi, at.col + c, at.row, at.batch);
    Slots::ask(at, 1, &p.lo, at.col + c, at.row, at.batch);
  }
  __device__ __forceinline__ void begin(const Place& at) { ask(at, 0); }
  __device__ __forceinline__ void block(const Place& at, int c, float (&v)[kBlock]) {
    constexpr float kDown = LAST ? 1.0f / kScaleX : 1.0f;
    if (!arrived(at)) return;
    add_rows(at, 1, kDown / kScaleA, kDown * p.of_x, v);
    add_rows(at, 0, 1.0f, kDown * p.of_x, v);
    __syncwarp();
    if constexpr (LAST) {
      Slots::stage<Bf16>(at, 0, v);
      Slots::hand_over();
      if (p.whole) {
        if (at.lane == 0 && at.row < at.rows) { Slots::send(at, 0, &p.hi_out, at.col + c, at.row, at.batch); Slots::sent(); }
      } else {
        Slots::scatter(at.own, at.lane, reinterpret_cast<unsigned short*>(p.out + at.batch * p.out_plane + at.col + c), p.out_ld, at.row < at.rows ? at.row : -1, at.cols - at.col - c, false);
        Slots::hand_over();
      }
    } else {
      Slots::stage<Fp16>(at, 0, v);
#pragma unroll
      for (int j = 0; j < kBlock; j += 2) {
        const float2 h = Fp16::open(Fp16::pack(v[j], v[j + 1]));
        const float2 l = __ffma2_rn(h, make_float2(-1.0f, -1.0f), make_float2(v[j], v[j + 1]));
        v[j] = l.x; v[j + 1] = l.y;
      }
      Slots::stage<Fp16>(at, 1, v);
      Slots::hand_over();
      if (at.lane == 0 && at.row < at.rows) {
        Slots::send(at, 0, &p.hi_out, at.col + c, at.row, at.batch);
        Slots::send(at, 1, &p.lo_out, at.col + c, at.row, at.batch);
        Slots::sent();
      }
    }
    ask(at, c + kBlock);
  }
  __device__ __forceinline__ void end(const Place&) {}
};

// ---- matrices of up to 128 columns (or rows) ----------------------------------------------------------------------
// All steps in one launch, X never in memory: a cluster of CTAs shares the other direction, 256 of it each; a thread has one of these, 128 numbers of X in f32, and their fp16
// roundings lie in shared memory as an operand, the same tile as X (rows by k) and as X^T (k by rows).  A step: the cluster's CTAs make their parts of
// A = X^T X and send each other the rows that they add up (S CTAs 128 / S each); these go to all as fp16; every CTA makes A A, B and its own rows of X B.  The low-rank layers' weights,
// 2048 x 128: one 127 us by three products a step, 54 so; 120 of them 917 and 452 (fifteen clusters of eight run at a time).
// What it is bound by: a step's chain of 17000 cycles, half of them the cluster's sums (16 bytes a clock into an SM, two barriers); the rest are tensor core round trips and fp16 rows
// through shared memory, with nothing of another matrix beside them.
constexpr int kNarrow = 128, kSlab = 256, kMostClusters = 16;
constexpr int kNarrowSmem = 1024 + kSlab * kNarrow * 2 + 2 * kNarrow * kNarrow * 2 + kNarrow * kNarrow * 4;      // X, A and B, sums from the others

struct NarrowParams {
  const void* g;
  __nv_bfloat16* out;
  int64_t length;           // of the long direction
  int width, size, steps;   // of the short one; CTAs of a cluster
  bool tall;                // the long direction is rows
  bool vectors, out_vectors;
  double eps;
  float coefficients[64 * 3];
  uint32_t polls;
};
__device__ __forceinline__ void cluster_sync_all() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ uint64_t narrow_desc(uint32_t addr, uint32_t next) {      // 128-byte swizzle; K-major (next: unused), or M/N-major with the next 64 rows `next` bytes on
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// the 16-byte piece of row r at columns 8 k .. of a matrix of `rows` rows by 128 columns: two panels of 64 columns
__device__ __forceinline__ uint32_t piece_at(uint32_t base, int rows, int r, int k) { return base + (k >> 3) * (rows * 128) + r * 128 + (((k & 7) ^ (r & 7)) << 4); }

template <typename T>
__global__ void __launch_bounds__(kSlab, 1) narrow_kernel(const __grid_constant__ NarrowParams p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bar;
  __shared__ uint32_t tmem_slot;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, x_at = base, a_at = x_at + kSlab * kNarrow * 2, sums_at = a_at + kNarrow * kNarrow * 2, b_at = sums_at + kNarrow * kNarrow * 4;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = warp & 3, half = warp >> 2;
  if (tid == 0) {
    bar_init(smem_u32(&bar), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  cluster_sync_all();          // the others run, and can be written to
  tc_after();
  const uint32_t tmem = *(volatile uint32_t*)&tmem_slot, lanes = tmem + ((uint32_t)(quad * 32) << 16);
  grid_wait();
  __shared__ double squares[8], of_cluster[kMostClusters];
  __shared__ float factors[3];
  const int rank = (int)(blockIdx.x % p.size), share = kNarrow / p.size;      // rows of A that this CTA adds up

  // this thread's numbers
  const int64_t matrix = (int64_t)(blockIdx.x / p.size) * p.length * p.width, at = (int64_t)rank * kSlab + tid;
  const T* g = static_cast<const T*>(p.g) + matrix;
  float x[kNarrow];
  if (p.tall && p.vectors) {
    constexpr int kN = Vec<T>::kN;
#pragma unroll
    for (int j = 0; j < kNarrow; j += kN) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (at < p.length && j < p.width) v = __ldg(reinterpret_cast<const uint4*>(g + at * p.width + j));
      Vec<T>::open(v, x + j);
    }
  } else {
    const T* from = p.tall ? g + at * p.width : g + at;
    const int64_t step = p.tall ? 1 : p.length;
#pragma unroll
    for (int j = 0; j < kNarrow; ++j) x[j] = at < p.length && j < p.width ? Elem<T>::to_f32(from[j * step]) : 0.0f;
  }
  float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < kNarrow; ++j) part[j & 3] = fmaf(x[j], x[j], part[j & 3]);
  double s = (double)((part[0] + part[1]) + (part[2] + part[3]));
  if (!(s < 0x1p120) || s < 0x1p-60) {          // squares that leave f32, or lose their bits in it
    s = 0.0;
#pragma unroll
    for (int j = 0; j < kNarrow; ++j) s = fma((double)x[j], (double)x[j], s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) squares[warp] = s;
  __syncthreads();
  if (tid < p.size) {
    for (int w = 1; w < 8; ++w) s = w == 1 ? squares[0] + squares[1] : s + squares[w];
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(in_cta(smem_u32(&of_cluster[rank]), tid)), "d"(s) : "memory");
  }
  cluster_sync_all();
  if (tid == 0) {
    s = 0.0;
    for (int r = 0; r < p.size; ++r) s += of_cluster[r];
    scale_factors(s, p.eps, factors);
  }
  __syncthreads();
  const float f1 = factors[1], f2 = factors[2], f0 = factors[0];
#pragma unroll
  for (int j = 0; j < kNarrow; ++j) x[j] = x[j] * f1 * f2 * f0;

  constexpr uint32_t kSquare = (1u << 4) | ((uint32_t)(kNarrow >> 3) << 17) | ((uint32_t)(128 >> 4) << 24), kTransposed = kSquare | (3u << 15);
  uint32_t phase = 0;
  auto products_done = [&] {
    (void)bar_wait(smem_u32(&bar), phase, p.polls);      // where it runs out, the status says so and the barriers below are still met
    phase ^= 1;
    tc_after();
  };
  for (int step = 0; step < p.steps; ++step) {
    const float a = p.coefficients[3 * step], b = p.coefficients[3 * step + 1], c = p.coefficients[3 * step + 2];
    // X's first terms as an operand
#pragma unroll
    for (int k = 0; k < kNarrow / 8; ++k) {
      const float* v = x + 8 * k;
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at(x_at, kSlab, tid, k)), "r"(Fp16::pack(v[0], v[1])), "r"(Fp16::pack(v[2], v[3])), "r"(Fp16::pack(v[4], v[5])),
                   "r"(Fp16::pack(v[6], v[7])) : "memory");
    }
    async_fence();
    tc_before();
    __syncthreads();
    if (tid == 0) {          // A = X^T X of this CTA's 256
      tc_after();
#pragma unroll 4
      for (int k = 0; k < kSlab / 16; ++k) {
        const uint64_t d = narrow_desc(x_at + k * 2048, kSlab * 128);
        mma<1>(tmem, d, d, kTransposed, k > 0);
      }
      commit_to<1>(smem_u32(&bar));
    }
    products_done();
    {                        // row quad * 32 + lane of it, 64 columns, to whom adds that row up; 16-byte pieces of a row exchanged by its number
      const int row = quad * 32 + lane;
      const uint32_t to = in_cta(sums_at + ((uint32_t)(rank * share + row % share) * kNarrow) * 4, row / share);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        ld_acc32(lanes + half * 64 + h * 32, v);
        wait_acc32(v);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + (((half * 16 + h * 8 + k) ^ lane) << 4)), "f"(v[4 * k]), "f"(v[4 * k + 1]), "f"(v[4 * k + 2]), "f"(v[4 * k + 3]) : "memory");
      }
      tc_before();
    }
    cluster_sync_all();
    for (int i = tid; i < share * (kNarrow / 4); i += kSlab) {      // four columns of a row, in the CTAs' order, to all of them
      const int row = i / (kNarrow / 4), piece = i % (kNarrow / 4), whole = rank * share + row;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int r = 0; r < p.size; ++r) {
        float4 w;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(w.x), "=f"(w.y), "=f"(w.z), "=f"(w.w)
                     : "r"(sums_at + (uint32_t)(r * share + row) * kNarrow * 4 + ((piece ^ (whole & 31)) << 4)) : "memory");
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      constexpr float kDown = kScaleA / (kScaleX * kScaleX);
      const uint32_t lo = Fp16::pack(v.x * kDown, v.y * kDown), hi = Fp16::pack(v.z * kDown, v.w * kDown), to = piece_at(a_at, kNarrow, whole, piece >> 1) + (piece & 1) * 8;
      for (int r = 0; r < p.size; ++r) asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(in_cta(to, r)), "r"(lo), "r"(hi) : "memory");
    }
    async_fence();
    cluster_sync_all();
    async_fence();
    if (tid == 0) {          // A A
      tc_after();
#pragma unroll
      for (int k = 0; k < kNarrow / 16; ++k) {
        const uint64_t d = narrow_desc(a_at + (k >> 2) * (kNarrow * 128) + (k & 3) * 32, 16);
        mma<1>(tmem + kNarrow, d, d, kSquare, k > 0);
      }
      commit_to<1>(smem_u32(&bar));
    }
    products_done();
    {                        // B = b A + c A A
      const int row = quad * 32 + lane;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        ld_acc32(lanes + kNarrow + half * 64 + h * 32, v);
        wait_acc32(v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int piece = half * 8 + h * 4 + k;
          const uint4 w = Slots::get(piece_at(a_at, kNarrow, row, piece));
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
          uint32_t to[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = Fp16::open(words[j]);
            to[j] = Fp16::pack(fmaf(v[8 * k + 2 * j], c / kScaleA, f.x * b), fmaf(v[8 * k + 2 * j + 1], c / kScaleA, f.y * b));
          }
          Slots::put(piece_at(b_at, kNarrow, row, piece), to[0], to[1], to[2], to[3]);
        }
      }
    }
    async_fence();
    tc_before();
    __syncthreads();
    if (tid == 0) {          // X B, 128 of X at a time
      tc_after();
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int k = 0; k < kNarrow / 16; ++k)
          mma<1>(tmem + (2 + t) * kNarrow, narrow_desc(x_at + (k >> 2) * (kSlab * 128) + t * (128 * 128) + (k & 3) * 32, 16), narrow_desc(b_at + (k >> 2) * (kNarrow * 128) + (k & 3) * 32, 16), kSquare, k > 0);
      commit_to<1>(smem_u32(&bar));
    }
    products_done();
#pragma unroll
    for (int h = 0; h < kNarrow / 32; ++h) {
      float v[32];
      ld_acc32(lanes + (2 + half) * kNarrow + h * 32, v);
      wait_acc32(v);
#pragma unroll
      for (int j = 0; j < 32; ++j) x[32 * h + j] = fmaf(x[32 * h + j], a, v[j] * (1.0f / kScaleA));
    }
  }
  constexpr float kDown = 1.0f / kScaleX;
  if (p.tall) {              // the CTA's rows lie together: through shared memory, 16 or two bytes a thread
    const int here = (int)max((int64_t)0, min((int64_t)kSlab, p.length - (int64_t)rank * kSlab)) * p.width;
    __nv_bfloat16 *to = p.out + matrix + (int64_t)rank * kSlab * p.width, *from = reinterpret_cast<__nv_bfloat16*>(smem_raw + (base - smem_u32(smem_raw)));
    if (p.out_vectors) {     // where a row's 16-byte pieces are a multiple of eight, they are exchanged by its number, against bank conflicts
      const int pieces = p.width / 8, turn = pieces % 8 == 0 ? 7 : 0;
#pragma unroll
      for (int k = 0; k < kNarrow / 8; ++k) {
        const float* v = x + 8 * k;
        if (k < pieces)
          reinterpret_cast<uint4*>(from)[tid * pieces + (k ^ (tid & turn))] = make_uint4(pack_bf16x2(v[0] * kDown, v[1] * kDown), pack_bf16x2(v[2] * kDown, v[3] * kDown), pack_bf16x2(v[4] * kDown, v[5] * kDown), pack_bf16x2(v[6] * kDown, v[7] * kDown));
      }
      __syncthreads();
      for (int i = tid; i < here / 8; i += kSlab) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(from)[i ^ (i / pieces & turn)];
    } else {
#pragma unroll
      for (int j = 0; j < kNarrow; ++j)
        if (j < p.width) from[tid * p.width + j] = __float2bfloat16_rn(x[j] * kDown);
      __syncthreads();
      for (int i = tid; i < here; i += kSlab) to[i] = from[i];
    }
  } else if (at < p.length) {
    __nv_bfloat16* to = p.out + matrix + at;
#pragma unroll
    for (int j = 0; j < kNarrow; ++j)
      if (j < p.width) to[j * p.length] = __float2bfloat16_rn(x[j] * kDown);
  }
  tc_before();
  __syncthreads();
  if (warp == 0) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// The CTAs that a cluster may have on the current device.  Every GPU that runs the kernel has room for eight; sixteen, an SM each in one GPC, may be more than a part of a GPU has.
int most_clusters() {
#ifdef PB_DIAGNOSTICS
  if (g_withhold.load() & kEightAtMost) return 8;
#endif
  static std::mutex mu;
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 8;
  std::lock_guard<std::mutex> lock(mu);
  if (cached[dev] == 0) {
    auto fits = [](auto kernel) {
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(kMostClusters); config.blockDim = dim3(kSlab); config.dynamicSmemBytes = kNarrowSmem;
      cudaLaunchAttribute size;
      size.id = cudaLaunchAttributeClusterDimension;
      size.val.clusterDim.x = kMostClusters; size.val.clusterDim.y = size.val.clusterDim.z = 1;
      config.attrs = &size; config.numAttrs = 1;
      int clusters = 0;
      return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNarrowSmem) == cudaSuccess &&
             cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
             cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) == cudaSuccess && clusters > 0;
    };
    cached[dev] = fits(narrow_kernel<float>) && fits(narrow_kernel<__nv_bfloat16>) ? kMostClusters : 8;
    if (cached[dev] == 8) (void)cudaGetLastError();      // no error of the call
  }
  return cached[dev];
}
// A cluster's CTAs for a matrix; 0: too long, or too wide.  2048 x 128 | 129: 54 | 132 us, 4096 x 128 | 4097 x 128: 59 | 142
int narrow_size(int64_t rows, int64_t cols) {
  const int64_t length = std::max(rows, cols), width = std::min(rows, cols);
  if (width > kNarrow || length > kMostClusters * kSlab || (length > 8 * kSlab && most_clusters() < kMostClusters)) return 0;
  int size = 1;
  while (size * kSlab < length) size *= 2;
  return size;
}

int run_narrow(const void* update, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps, const float* coefficients, double eps, void* out, cudaStream_t st) {
  NarrowParams p{};
  p.g = update; p.out = static_cast<__nv_bfloat16*>(out);
  p.tall = rows >= cols; p.length = std::max(rows, cols); p.width = (int)std::min(rows, cols); p.size = narrow_size(rows, cols); p.steps = steps; p.eps = eps;
  p.vectors = !off_by(update, 16) && p.width * (dtype == PB_F32 ? 4 : 2) % 16 == 0;
  p.out_vectors = !off_by(out, 16) && p.width % 8 == 0;
  std::copy(coefficients, coefficients + 3 * steps, p.coefficients);
  p.polls = kWaitPolls;
#ifdef PB_DIAGNOSTICS
  p.polls = g_polls.load();
#endif
  auto kernel = dtype == PB_F32 ? narrow_kernel<float> : narrow_kernel<__nv_bfloat16>;
  PB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNarrowSmem));      // per device
  if (p.size > 8) PB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(batch * p.size)); config.blockDim = dim3(kSlab); config.dynamicSmemBytes = kNarrowSmem; config.stream = st;
  cudaLaunchAttribute how[2];
  how[0].id = cudaLaunchAttributeClusterDimension;
  how[0].val.clusterDim.x = (unsigned)p.size; how[0].val.clusterDim.y = how[0].val.clusterDim.z = 1;
  how[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  how[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = how; config.numAttrs = 2;
  cudaLaunchKernelEx(&config, kernel, p);
  PB_LAUNCH_CHECK("narrow_kernel");
  return PB_OK;
}

// ---- host side ----------------------------------------------------------------------------------------------------
// Forms of a product's tiles: 256 x 256 and 256 x 128 of a CTA pair, 128 x 128 of a CTA.  A tile's stage of 64 of k is bound by its loads from L2, some 58 bytes a clock into an SM: 563, 413 and 540 cycles, and
// a tile takes 9000, 6000 and 5000 more until its sums have left.  So the wide pair's is the best wherever its tiles fill the chip, and the others where it
// would leave half of it idle: A of 2048 x 2048, 36 tiles | 72, 22.4 us | 17.3.
enum Tile { kPair256, kPair128, kSingle };
double cost_of(Tile tile, const Params& p) {
  const int64_t stages = (p.depth + kDepth - 1) / kDepth;
  auto rounds = [](int64_t tiles, int64_t clusters) { return (tiles + clusters - 1) / clusters; };
  return tile == kPair256 ? rounds(tiles_of<2, 256>(p), clusters_of<2>()) * (563.0 * stages + 9000) : tile == kPair128 ? rounds(tiles_of<2, 128>(p), clusters_of<2>()) * (413.0 * stages + 6000)
                          : rounds(tiles_of<1, 128>(p), clusters_of<1>()) * (540.0 * stages + 5000);
}
Tile tile_of(const Params& p) {
  Tile best = kPair256;
  for (Tile t : {kPair128, kSingle})
    if (cost_of(t, p) < cost_of(best, p)) best = t;
  return best;
}
template <bool A_MN, bool B_MN, class E>
int run(const Operand& a, const Operand& b, const Params& p, const typename E::Params& e, cudaStream_t st) {
  const Tile tile = tile_of(p);
  return tile == kPair256 ? launch<2, 256, A_MN, B_MN, E>(a, b, p, e, st) : tile == kPair128 ? launch<2, 128, A_MN, B_MN, E>(a, b, p, e, st) : launch<1, 128, A_MN, B_MN, E>(a, b, p, e, st);
}

struct Plan {
  int64_t d, ld, ld_a, plane, plane_a;
  Params gram;              // A's product; cut where its tiles are few and long
  size_t off_hi[2], off_lo[2], off_a, off_b, off_parts, bytes;
};
int make_plan(int64_t batch, int64_t rows, int64_t cols, Plan* q) {
  if (batch <= 0 || rows <= 0 || cols <= 0 || rows > (1 << 24) || cols > (1 << 24) || batch > 65535 || rows * cols > (1ll << 36))
    return fail(PB_ERR_BAD_SHAPE, "pb_orthogonalize: batch=%lld rows=%lld cols=%lld", (long long)batch, (long long)rows, (long long)cols);
  if (narrow_size(rows, cols)) {
    q->bytes = 256;         // never written to
    return PB_OK;
  }
  q->d = std::min(rows, cols);
  q->ld = (cols + 63) / 64 * 64; q->ld_a = (q->d + 63) / 64 * 64;
  q->plane = rows * q->ld; q->plane_a = q->d * q->ld_a;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t was = at; at += (bytes + 255) / 256 * 256; return was; };
  take((size_t)batch * kParts * sizeof(double));
  for (int i = 0; i < 2; ++i) { q->off_hi[i] = take((size_t)batch * q->plane * 2); q->off_lo[i] = take((size_t)batch * q->plane * 2); }
  q->off_a = take((size_t)batch * q->plane_a * 2);
  q->off_b = take((size_t)batch * q->plane_a * 2);
  q->gram = Params{};
  Params& p = q->gram;
  p.batch = (int)batch; p.rows = p.cols = (int)q->d; p.depth = (int)std::max(rows, cols); p.upper = 1;
  Params cut = p;
  cut_stages<2, 256>(&cut, (p.depth + kDepth - 1) / kDepth);
  const int64_t clusters = clusters_of<2>(), tiles = tiles_of<2, 256>(p);
  const double cut_cost = 563.0 * ((tiles * cut.cuts + clusters - 1) / clusters * (cut.cut + kPartCost) + tiles * cut.cuts / kJoinParts) + 8000;      // and another launch
  if (cut.cuts > 1 && cut_cost < cost_of(tile_of(p), p)) p = cut;
  q->off_parts = take(p.cuts ? (size_t)parts_of<2, 256>(p) * 16 : 0);
  q->bytes = at;
  return PB_OK;
}

template <bool LAST>
int run_update(bool tall, const Operand& x_rows, const Operand& x_cols, const Operand& poly, const Params& p, const typename UpdateEpilogue<LAST>::Params& e, cudaStream_t st) {
  return tall ? run<false, false, UpdateEpilogue<LAST>>(x_rows, poly, p, e, st) : run<false, true, UpdateEpilogue<LAST>>(poly, x_cols, p, e, st);
}

}  // namespace

int orthogonalize_status_fetch(unsigned int* out) { return status_fetch(out); }
#ifdef PB_DIAGNOSTICS
void orthogonalize_control(uint32_t polls, int withhold) { control(polls, withhold); }
#endif
}  // namespace pb

using namespace pb;

extern "C" size_t pb_orthogonalize_workspace_size(int64_t batch, int64_t rows, int64_t cols) {
  Plan q;
  return make_plan(batch, rows, cols, &q) ? 0 : q.bytes;
}

extern "C" int pb_orthogonalize(const void* update, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps, const float* coefficients, double eps,
                                void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (!update || !coefficients || !out || !workspace) return fail(PB_ERR_NULL_POINTER, "pb_orthogonalize: null argument");
  if (dtype != PB_F32 && dtype != PB_BF16) return fail(PB_ERR_BAD_DTYPE, "pb_orthogonalize: dtype %d", dtype);
  Plan q;
  if (int s = make_plan(batch, rows, cols, &q)) return s;
  if (steps < 1 || steps > 64 || !(eps >= 0.0)) return fail(PB_ERR_BAD_SHAPE, "pb_orthogonalize: %d steps, eps %g", steps, eps);
  if (off_by(update, dtype == PB_F32 ? 4 : 2) || off_by(out, 2) || off_by(workspace, 256)) return fail(PB_ERR_MISALIGNED, "pb_orthogonalize: misaligned array");
  if (workspace_bytes < q.bytes) return fail(PB_ERR_WORKSPACE_TOO_SMALL, "pb_orthogonalize: workspace of %zu bytes, %zu needed", workspace_bytes, q.bytes);
  // what singular values of up to 1 become has to stay within what the terms hold
  double most = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
    double next = 0.0, gram = 0.0;
    for (int i = 0; i <= 1024; ++i) {
      const double s = most * i / 1024, s2 = s * s;
      next = std::max(next, std::fabs(s * (a + s2 * (b + s2 * c))));
      gram = std::max(gram, std::fabs(s2 * (b + s2 * c)));
    }
    if (!std::isfinite(a + b + c) || !(next <= kMostX) || !(gram <= kMostB))
      return fail(PB_ERR_UNSUPPORTED, "pb_orthogonalize: coefficients %g %g %g of step %d take singular values beyond %g", a, b, c, k, (double)kMostX);
    most = next;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (narrow_size(rows, cols)) return run_narrow(update, dtype, batch, rows, cols, steps, coefficients, eps, out, st);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  double* sums = reinterpret_cast<double*>(ws);
  __half* hi[2] = {reinterpret_cast<__half*>(ws + q.off_hi[0]), reinterpret_cast<__half*>(ws + q.off_hi[1])};
  __half* lo[2] = {reinterpret_cast<__half*>(ws + q.off_lo[0]), reinterpret_cast<__half*>(ws + q.off_lo[1])};
  __half *gram = reinterpret_cast<__half*>(ws + q.off_a), *poly = reinterpret_cast<__half*>(ws + q.off_b);

  const int64_t n = rows * cols;
  const size_t element = dtype == PB_F32 ? 4 : 2;
  const bool vectors = !off_by(update, 16) && n * element % 16 == 0;
  SplitParams sp{update, sums, hi[0], lo[0], rows, cols, q.ld, eps, vectors && cols % 8 == 0};
  const int64_t blocks = (rows * (q.ld / 8) + 255) / 256;
  if (blocks > kMaxIndexed) return fail(PB_ERR_BAD_SHAPE, "pb_orthogonalize: %lld x %lld", (long long)rows, (long long)cols);
  if (dtype == PB_F32) {
    launch_behind(square_sums_kernel<float>, dim3(kParts, (unsigned)batch), 256, 0, st, static_cast<const float*>(update), n, vectors, sums);
    PB_LAUNCH_CHECK("square_sums_kernel");
    launch_behind(normalise_kernel<float>, dim3((unsigned)blocks, (unsigned)batch), 256, 0, st, sp);
  } else {
    launch_behind(square_sums_kernel<__nv_bfloat16>, dim3(kParts, (unsigned)batch), 256, 0, st, static_cast<const __nv_bfloat16*>(update), n, vectors, sums);
    PB_LAUNCH_CHECK("square_sums_kernel");
    launch_behind(normalise_kernel<__nv_bfloat16>, dim3((unsigned)blocks, (unsigned)batch), 256, 0, st, sp);
  }
  PB_LAUNCH_CHECK("normalise_kernel");

  const bool tall = rows > cols;
  // blocks of 32 rows of X's terms, of A and of B for the epilogues, and their transposes
  CUtensorMap hi_blocks[2], lo_blocks[2], out_blocks{};
  for (int i = 0; i < 2; ++i) {
    if (int s = make_map(&hi_blocks[i], hi[i], false, cols, rows, q.ld, batch, q.plane, 32)) return s;
    if (int s = make_map(&lo_blocks[i], lo[i], false, cols, rows, q.ld, batch, q.plane, 32)) return s;
  }
  const bool whole = !off_by(out, 16) && cols % 8 == 0;
  if (whole)
    if (int s = make_map(&out_blocks, out, true, cols, rows, cols, batch, n, 32)) return s;
  Symmetric gram_blocks, poly_blocks;
  for (auto [blocks, at] : {std::pair{&gram_blocks, gram}, std::pair{&poly_blocks, poly}}) {
    if (int s = make_map(&blocks->rows, at, false, q.d, q.d, q.ld_a, batch, q.plane_a, 32)) return s;
    if (int s = make_map(&blocks->columns, at, false, q.d, q.d, q.ld_a, batch, q.plane_a, kBlock, 32)) return s;
  }
  Params p{};
  p.batch = (int)batch; p.bf16 = 0;
  for (int k = 0; k < steps; ++k) {
    const int now = k & 1;
    const float a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
    const Operand x_rows{hi[now], false, rows, cols, q.ld, q.plane}, x_cols{hi[now], true, cols, rows, q.ld, q.plane};      // X by its rows, and by its columns
    const GramEpilogue::Params ge{gram_blocks};
    if (q.gram.cuts) {
      float4* parts = reinterpret_cast<float4*>(ws + q.off_parts);
      const PartEpilogue<false>::Params pe{parts, false};
      if (int s = tall ? launch<2, 256, true, true, PartEpilogue<false>>(x_cols, x_cols, q.gram, pe, st) : launch<2, 256, false, false, PartEpilogue<false>>(x_rows, x_rows, q.gram, pe, st)) return s;
      if (int s = launch_finish<2, 256, GramEpilogue>(parts, q.gram, ge, st)) return s;
    } else if (int s = tall ? run<true, true, GramEpilogue>(x_cols, x_cols, q.gram, ge, st) : run<false, false, GramEpilogue>(x_rows, x_rows, q.gram, ge, st)) {
      return s;
    }
    p.rows = p.cols = p.depth = (int)q.d; p.upper = 1;
    const Operand gram_rows{gram, false, q.d, q.d, q.ld_a, q.plane_a}, poly_rows{poly, false, q.d, q.d, q.ld_a, q.plane_a};
    if (int s = run<false, false, SquareEpilogue>(gram_rows, gram_rows, p, SquareEpilogue::Params{gram_blocks.rows, poly_blocks, b, c / kScaleA}, st)) return s;
    p.rows = (int)rows; p.cols = (int)cols; p.upper = 0;
    if (int s = k == steps - 1 ? run_update<true>(tall, x_rows, x_cols, poly_rows, p, {hi_blocks[now], lo_blocks[now], out_blocks, out_blocks, static_cast<__nv_bfloat16*>(out), cols, n, whole, a}, st)
                               : run_update<false>(tall, x_rows, x_cols, poly_rows, p, {hi_blocks[now], lo_blocks[now], hi_blocks[now ^ 1], lo_blocks[now ^ 1], nullptr, 0, 0, true, a}, st))
      return s;
  }
  return PB_OK;
}
