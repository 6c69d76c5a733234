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
      // 2^12 / (|G| + eps) as two powers of two and a rest in [1, 2): each within f32 where the whole may not be
      const double by = (double)kScaleX / (sqrt(s) + p.eps);
      int e = 0;
      const double rest = 2.0 * frexp(by, &e);
      const bool fine = isfinite(by) && isfinite(s);
      e -= 1;
      factors[0] = fine ? (float)rest : nanf("");      // an infinity or a NaN anywhere: nothing else
      factors[1] = ldexpf(1.0f, e / 2);
      factors[2] = ldexpf(1.0f, e - e / 2);
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

// Blocks that are read before they are written: asked for a block ahead, as soon as the slots have been read out.  `pending`: on their way.
struct Reading : Ungrouped {
  uint32_t phase = 0;
  bool pending = false;
  __device__ __forceinline__ bool arrived(const Place& at) {
    const bool ok = bar_wait(at.bar, phase, at.polls);
    phase ^= 1; pending = false;
    return __all_sync(0xffffffffu, ok);
  }
  __device__ __forceinline__ void finish(const Place& at) {
    if (pending) (void)arrived(at);
    if (at.lane == 0) Slots::wait_sent();
  }
};

struct SquareEpilogue : Reading {
  struct Params { CUtensorMap a; Symmetric b; float of_a, of_square; };
  const Params& p;
  __device__ __forceinline__ explicit SquareEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void ask(const Place& at, int c) {
    if (c >= at.slice || at.col + c >= at.cols) return;
    pending = true;
    if (at.lane == 0) {
      Slots::wait_read();
      bar_expect(at.bar, kSlotBytes);
      Slots::ask(at, 0, &p.a, at.col + c, at.row, at.batch);
    }
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
    if (c >= at.slice || at.col + c >= at.cols) return;
    pending = true;
    if (at.lane == 0) {
      Slots::wait_read();
      bar_expect(at.bar, 2 * kSlotBytes);
      Slots::ask(at, 0, &p.hi, at.col + c, at.row, at.batch);
      Slots::ask(at, 1, &p.lo, at.col + c, at.row, at.batch);
    }
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

// ---- host side ----------------------------------------------------------------------------------------------------
struct Plan {
  int64_t d, ld, ld_a, plane, plane_a;
  size_t off_hi[2], off_lo[2], off_a, off_b, bytes;
};
int make_plan(int64_t batch, int64_t rows, int64_t cols, Plan* q) {
  if (batch <= 0 || rows <= 0 || cols <= 0 || rows > (1 << 24) || cols > (1 << 24) || batch > 65535 || rows * cols > (1ll << 36))
    return fail(PB_ERR_BAD_SHAPE, "pb_orthogonalize: batch=%lld rows=%lld cols=%lld", (long long)batch, (long long)rows, (long long)cols);
  q->d = std::min(rows, cols);
  q->ld = (cols + 63) / 64 * 64; q->ld_a = (q->d + 63) / 64 * 64;
  q->plane = rows * q->ld; q->plane_a = q->d * q->ld_a;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t was = at; at += (bytes + 255) / 256 * 256; return was; };
  take((size_t)batch * kParts * sizeof(double));
  for (int i = 0; i < 2; ++i) { q->off_hi[i] = take((size_t)batch * q->plane * 2); q->off_lo[i] = take((size_t)batch * q->plane * 2); }
  q->off_a = take((size_t)batch * q->plane_a * 2);
  q->off_b = take((size_t)batch * q->plane_a * 2);
  q->bytes = at;
  return PB_OK;
}

// 256 x 256 tiles of a CTA pair, or 128 x 128 ones of a CTA where pairs would leave most SMs without any
bool small_tiles(int64_t rows, int64_t cols, int64_t batch, bool upper) {
  const int64_t tm = (rows + 255) / 256, tn = (cols + 255) / 256;
  return batch * (upper ? tn * (tn + 1) / 2 : tm * tn) * 4 <= sm_count() / 2;
}
template <bool A_MN, bool B_MN, class E>
int run(const Operand& a, const Operand& b, const Params& p, const typename E::Params& e, cudaStream_t st) {
  return small_tiles(p.rows, p.cols, p.batch, p.upper) ? launch<1, 128, A_MN, B_MN, E>(a, b, p, e, st) : launch<2, 256, A_MN, B_MN, E>(a, b, p, e, st);
}

template <bool LAST>
int run_update(bool tall, const Operand& x_rows, const Operand& x_cols, const Operand& poly, const Params& p, const typename UpdateEpilogue<LAST>::Params& e, cudaStream_t st) {
  return tall ? run<false, false, UpdateEpilogue<LAST>>(x_rows, poly, p, e, st) : run<false, true, UpdateEpilogue<LAST>>(poly, x_cols, p, e, st);
}

}  // namespace

int orthogonalize_status_fetch(unsigned int* out) { return status_fetch(out); }
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
    p.rows = p.cols = (int)q.d; p.depth = (int)(tall ? rows : cols); p.upper = 1;
    const GramEpilogue::Params ge{gram_blocks};
    if (int s = tall ? run<true, true, GramEpilogue>(x_cols, x_cols, p, ge, st) : run<false, false, GramEpilogue>(x_rows, x_rows, p, ge, st)) return s;
    p.depth = (int)q.d;
    const Operand gram_rows{gram, false, q.d, q.d, q.ld_a, q.plane_a}, poly_rows{poly, false, q.d, q.d, q.ld_a, q.plane_a};
    if (int s = run<false, false, SquareEpilogue>(gram_rows, gram_rows, p, SquareEpilogue::Params{gram_blocks.rows, poly_blocks, b, c / kScaleA}, st)) return s;
    p.rows = (int)rows; p.cols = (int)cols; p.upper = 0;
    if (int s = k == steps - 1 ? run_update<true>(tall, x_rows, x_cols, poly_rows, p, {hi_blocks[now], lo_blocks[now], out_blocks, out_blocks, static_cast<__nv_bfloat16*>(out), cols, n, whole, a}, st)
                               : run_update<false>(tall, x_rows, x_cols, poly_rows, p, {hi_blocks[now], lo_blocks[now], hi_blocks[now ^ 1], lo_blocks[now ^ 1], nullptr, 0, 0, true, a}, st))
      return s;
  }
  return PB_OK;
}
