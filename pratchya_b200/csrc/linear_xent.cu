// Softmax cross entropy of hidden states against a vocabulary's weight, without the logits: the reference's lm_head and compute_loss
// (pratchya/_nnx_impl/_model.py:77, _utils.py:7-13) in one operator for a weight in bf16.  For a position x with target t, z = x W:
//   lse = log sum_j exp z_j,   loss = lse - (1 - a) z_t - a mean_j z_j,   dz_j = g (exp(z_j - lse) - (1 - a) [j = t] - a / V),
//   dx = dz W^T,   dW = x^T dz.
// Forward: one product (products.cuh) whose epilogue keeps of each 128 logits of a position a maximum, a sum of exponentials and, with smoothing, a sum,
// and of all of them the target's; a small kernel joins these.  Exponentials are of differences from the maximum, which are exact where they matter (a fused z log2(e) - m
// saves an instruction of two logits, but from logits of 10^9 on what rounding m leaves takes every term to 0).
// Backward: the logits once more, a piece of the vocabulary at a time, left as dz / (g (1 - a)) in bf16, and two products of the piece: dx, added up over the pieces in
// f32, and the piece's part of dW.  An operand of a bf16 product is rounded once; divided so, the target's element, the largest, is p_t / (1 - a) - 1 and next to
// exact while p_t is small, where g's and a's own bits would round all of a position's gradient one way (2.7e-3 of dx and dW, 1.66e-3 of
// which is the results' own rounding; now GRADIENT_ERROR).  dx takes g (1 - a) in f32 at its end; for dW the hidden states are multiplied by g over the largest g, exactly 1
// where all are one.
//
// Positions without a target do no work: a first kernel numbers those that have one, a second brings their hidden states together (rows
// of zeros up to a whole tile behind them), and the products read the number of rows on the device.  So what lies in a padded position, a NaN too, reaches nothing.
#include "products.cuh"

namespace pb {
namespace {
using namespace products;

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kRowTile = 256;                           // hidden states come in whole tiles of them
constexpr int kGroup = 8;                                // stages, 512 of k, of an accumulator
constexpr int kPart = 128;                              // logits of a position that an epilogue thread adds up
constexpr size_t kMostGradient = (size_t)256 << 20;     // bytes of dz at a time

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- which positions there are ------------------------------------------------------------------------------------
struct SelectParams {
  const int64_t* targets;
  int64_t vocab;
  int rows;
  int *count, *place, *origin, *target;      // place[row]: its number or -1; origin, target[number]
  const float *lse, *g;                      // backward: brought together, too, and the g of the largest magnitude
  float *lse_out, *g_out, *g_most;
  float* loss;                               // forward: of positions without a target 0, beyond the vocabulary NaN; and their lse
  float* lse_none;
};
// one CTA: a thread takes a run of positions and counts, the runs' sums meet, and it numbers its own in their order
__global__ void __launch_bounds__(1024) select_kernel(const __grid_constant__ SelectParams p) {
  grid_wait();
  __shared__ int sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int run = (p.rows + 1023) / 1024, first = min(p.rows, (int)threadIdx.x * run), last = min(p.rows, first + run);
  int mine = 0;
  float most = 0.0f;
  for (int i = first; i < last; ++i) {
    const bool there = p.targets[i] >= 0 && p.targets[i] < p.vocab;
    mine += there;
    if (p.g && there) most = fmaxf(most, fabsf(p.g[i]));
  }
  if (p.g) {
    __shared__ float tops[32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) tops[warp] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 32; ++w) most = fmaxf(most, tops[w]);
      *p.g_most = most;
    }
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int below = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += below;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  int at = before + upto - mine;
  if (threadIdx.x == 0) *p.count = all;
  for (int i = first; i < last; ++i) {
    const int64_t t = p.targets[i];
    const bool there = t >= 0 && t < p.vocab;
    p.place[i] = there ? at : -1;
    if (there) {
      p.origin[at] = i; p.target[at] = (int)t;
      if (p.lse) { p.lse_out[at] = p.lse[i]; p.g_out[at] = p.g[i]; }
      ++at;
    } else if (p.loss) {
      p.loss[i] = t < 0 ? 0.0f : nanf("");
      p.lse_none[i] = 0.0f;
    }
  }
}

struct GatherParams {
  const unsigned short* x;
  int64_t inner, stride_outer, stride_inner;
  const int *count, *place;
  unsigned short* out;
  // backward: the rows times g / g_most, and dx's of zeros for positions without a target
  unsigned short *scaled, *dx;
  const float *g, *g_most;
  int rows, depth, ld;
  bool vectors, dx_vectors;
};
// a warp a row, and kRowTile more for the zeros behind the last
__global__ void __launch_bounds__(256) gather_kernel(const __grid_constant__ GatherParams p) {
  grid_wait();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= p.rows) {
    const int count = *p.count, to = count + row - p.rows;
    if (to >= (count + kRowTile - 1) / kRowTile * kRowTile) return;
    for (int c = lane * 8; c < p.ld; c += 256) {
      *reinterpret_cast<uint4*>(p.out + (int64_t)to * p.ld + c) = make_uint4(0u, 0u, 0u, 0u);
      if (p.scaled) *reinterpret_cast<uint4*>(p.scaled + (int64_t)to * p.ld + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  const int to = p.place[row];
  if (to >= 0) {
    const unsigned short* from = p.x + row / p.inner * p.stride_outer + row % p.inner * p.stride_inner;
    unsigned short* out = p.out + (int64_t)to * p.ld;
    unsigned short* scaled = p.scaled ? p.scaled + (int64_t)to * p.ld : nullptr;
    float by = 1.0f;
    if (scaled) {
      const float most = *p.g_most, g = p.g[to];
      by = most == 0.0f ? g : __fdiv_rn(g, most);          // every g is zero, or none is a number
    }
    auto times = [&](uint32_t x) { return pack_bf16x2(__uint_as_float(x << 16) * by, __uint_as_float(x & 0xffff0000u) * by); };
    if (p.vectors) {
#pragma unroll 4
      for (int c = lane * 8; c < p.depth; c += 256) {
        const uint4 v = *reinterpret_cast<const uint4*>(from + c);
        *reinterpret_cast<uint4*>(out + c) = v;
        if (scaled) *reinterpret_cast<uint4*>(scaled + c) = make_uint4(times(v.x), times(v.y), times(v.z), times(v.w));
      }
    } else {
      for (int c = lane; c < p.ld; c += 32) {
        const unsigned short v = c < p.depth ? from[c] : (unsigned short)0;
        out[c] = v;
        if (scaled) scaled[c] = (unsigned short)times(v);
      }
    }
  } else if (p.dx) {
    unsigned short* out = p.dx + (int64_t)row * p.depth;
    if (p.dx_vectors) for (int c = lane * 8; c < p.depth; c += 256) *reinterpret_cast<uint4*>(out + c) = make_uint4(0u, 0u, 0u, 0u);
    else for (int c = lane; c < p.depth; c += 32) out[c] = 0;
  }
}

// a weight whose rows do not lie as TMA wants them, to rows that do
__global__ void __launch_bounds__(256) pad_kernel(const unsigned short* from, int64_t inner, int64_t ld_from, unsigned short* to, int64_t ld_to) {
  grid_wait();
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < inner; c += (int64_t)gridDim.x * 256) to[row * ld_to + c] = from[row * ld_from + c];
}

// ---- the epilogues ------------------------------------------------------------------------------------------------
struct Grouped { static constexpr bool kGrouped = true; static constexpr int kSlots = 1; };
// terms[part][row] = (m, s): the largest z of a part and the sum of exp(z - m); sums[part][row] of z; hit[row] the target's z
template <bool MEAN>
struct StatsEpilogue : Grouped {
  struct Params { const int* target; float2* terms; float* sums; float* hit; int64_t cap; };
  const Params& p;
  float m, s, sum, hit;
  int t;
  __device__ __forceinline__ explicit StatsEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void begin(const Place& at) {
    m = -INFINITY; s = 0.0f; sum = 0.0f;
    t = at.row < at.rows ? p.target[at.row] - at.col : -1;
  }
  __device__ __forceinline__ void block(const Place& at, int c, float (&v)[kBlock]) {
    const int n = at.cols - at.col - c;
    if (__any_sync(0xffffffffu, t >= c && t < c + kBlock)) {
#pragma unroll
      for (int j = 0; j < kBlock; ++j)
        if (t == c + j) p.hit[at.row] = v[j];
    }
    if (MEAN) {
      float2 a = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < kBlock; j += 2) a = __fadd2_rn(a, make_float2(v[j], v[j + 1]));      // beyond the vocabulary: zeros
      sum += a.x + a.y;
    }
    if (n < kBlock) {
#pragma unroll
      for (int j = 0; j < kBlock; ++j)
        if (j >= n) v[j] = -INFINITY;
    }
    float top = v[0];
#pragma unroll
    for (int j = 1; j < kBlock; ++j) top = fmaxf(top, v[j]);
    if (top > m) { s *= exp2_approx((m - top) * kLog2E); m = top; }
    const float base = m == -INFINITY ? 0.0f : -m;
    float2 a = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < kBlock; j += 2) {
      const float2 d = __fmul2_rn(__fadd2_rn(make_float2(v[j], v[j + 1]), make_float2(base, base)), make_float2(kLog2E, kLog2E));
      a = __fadd2_rn(a, make_float2(exp2_approx(d.x), exp2_approx(d.y)));
    }
    s += a.x + a.y;
  }
  __device__ __forceinline__ void end(const Place& at) {
    if (at.row >= at.rows) return;
    const int64_t to = (int64_t)(at.col / kPart) * p.cap + at.row;
    p.terms[to] = make_float2(m, s);
    if (MEAN) p.sums[to] = sum;
  }
  __device__ __forceinline__ void finish(const Place&) {}
};

// dz / (g by)[row][col], rows of `ld` elements: zeros behind the last position, up to the end of its tile.  up = 1 / by, mean = a / V / by, hit = (1 - a) / by
struct GradientEpilogue : Grouped {
  struct Params { CUtensorMap dz; const int* target; const float* lse; int first; float up, mean, hit; };
  const Params& p;
  float lse;
  int t;
  __device__ __forceinline__ explicit GradientEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void begin(const Place& at) {
    const bool there = at.row < at.rows;
    t = there ? p.target[at.row] - p.first - at.col : -1;
    lse = there ? -p.lse[at.row] : 0.0f;
  }
  __device__ __forceinline__ void block(const Place& at, int c, float (&v)[kBlock]) {
    const bool there = at.row < at.rows;
#pragma unroll
    for (int j = 0; j < kBlock; j += 2) {
      const float2 d = __fmul2_rn(__fadd2_rn(make_float2(v[j], v[j + 1]), make_float2(lse, lse)), make_float2(kLog2E, kLog2E));
      const float2 r = __ffma2_rn(make_float2(exp2_approx(d.x), exp2_approx(d.y)), make_float2(p.up, p.up), make_float2(-p.mean, -p.mean));
      v[j] = there ? r.x : 0.0f; v[j + 1] = there ? r.y : 0.0f;
    }
    if (__any_sync(0xffffffffu, t >= c && t < c + kBlock)) {
#pragma unroll
      for (int j = 0; j < kBlock; ++j)
        if (t == c + j) v[j] -= p.hit;
    }
    if (at.lane == 0) Slots::wait_read();
    __syncwarp();
    Slots::stage<Bf16>(at, 0, v);
    Slots::hand_over();
    if (at.lane == 0) { Slots::send(at, 0, &p.dz, at.col + c, at.row, 0); Slots::sent(); }
  }
  __device__ __forceinline__ void end(const Place&) {}
  __device__ __forceinline__ void finish(const Place& at) { if (at.lane == 0) Slots::wait_sent(); }
};

enum { kOnly, kFirst, kMore, kLast };      // of the products that are added up: a single one to bf16; into acc, onto acc, with acc to bf16
template <int MODE>
struct StoreEpilogue : Grouped {
  // what leaves as bf16 is multiplied by `by` and by scale[row], or scale[0] without origin; acc: a warp's parts of the tiles, 16 bytes a lane in a row
  struct Params { __nv_bfloat16* out; float4* acc; const int* origin; const float* scale; float by; int64_t ld; bool vectors; };
  const Params& p;
  int row;
  float scale;
  __device__ __forceinline__ explicit StoreEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void begin(const Place& at) {
    row = at.row < at.rows ? (p.origin ? p.origin[at.row] : at.row) : -1;
    scale = row < 0 || MODE == kFirst || MODE == kMore ? 0.0f : p.by * p.scale[p.origin ? at.row : 0];
  }
  __device__ __forceinline__ void block(const Place& at, int c, float (&v)[kBlock]) {
    if constexpr (MODE != kOnly) {
      float4* a = p.acc + ((int64_t)at.part * (kPart / 4) + c / 4) * 32 + at.lane;
#pragma unroll
      for (int j = 0; j < kBlock / 4; ++j) {
        float4 f = MODE == kFirst ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : a[32 * j];
        f.x += v[4 * j]; f.y += v[4 * j + 1]; f.z += v[4 * j + 2]; f.w += v[4 * j + 3];
        if (MODE == kLast) { v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w; }
        else a[32 * j] = f;
      }
    }
    if constexpr (MODE == kOnly || MODE == kLast) {
#pragma unroll
      for (int j = 0; j < kBlock; ++j) v[j] *= scale;
      Slots::stage<Bf16>(at, 0, v);
      __syncwarp();
      Slots::scatter(at.own, at.lane, reinterpret_cast<unsigned short*>(p.out + at.col + c), p.ld, row, at.cols - at.col - c, p.vectors);
    }
  }
  __device__ __forceinline__ void end(const Place&) {}
  __device__ __forceinline__ void finish(const Place&) {}
};

// ---- the parts of a position's logits together ----------------------------------------------------------------------
// 32 positions a CTA, a warp's lanes one each, 32 warps that take every 32nd part
template <bool MEAN>
__global__ void __launch_bounds__(1024) join_kernel(const float2* terms, const float* sums, const float* hit, const int* origin, const int* count, int64_t cap, int parts, float smoothing,
                                                    float inv_vocab, float* loss, float* lse) {
  grid_wait();
  __shared__ float red[3][32][33];
  const int n = *count, row = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x * 32 >= n) return;
  float m = -INFINITY, s = 0.0f, sum = 0.0f;
#pragma unroll 4
  for (int k = warp; k < parts; k += 32) {      // rows up to cap are there, if not told of
    const float2 t = terms[(int64_t)k * cap + row];
    if (MEAN) sum += sums[(int64_t)k * cap + row];
    const float top = fmaxf(m, t.x), base = top == -INFINITY ? 0.0f : top;
    s = s * exp2_approx((m - base) * kLog2E) + t.y * exp2_approx((t.x - base) * kLog2E);
    m = top;
  }
  red[0][warp][lane] = m; red[1][warp][lane] = s; red[2][warp][lane] = sum;
  __syncthreads();
  // warp w: position w, a lane each of its 32 sums
  m = red[0][lane][warp]; s = red[1][lane][warp]; sum = red[2][lane][warp];
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  s *= exp2_approx((m - (top == -INFINITY ? 0.0f : top)) * kLog2E);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  const int number = blockIdx.x * 32 + warp;
  if (lane == 0 && number < n) {
    const float l = top + logf(s);
    const int to = origin[number];
    lse[to] = l;
    loss[to] = MEAN ? l - (1.0f - smoothing) * hit[number] - smoothing * (sum * inv_vocab) : l - hit[number];
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------
struct Weight {
  const void* at;
  int64_t ld;
  bool by_word;      // [vocab, depth], else [depth, vocab]
};

struct Plan {
  int64_t cap, ld_x, piece, ld_w, inner_w, outer_w, parts;
  int pieces;
  bool pad;
  size_t off_place, off_origin, off_target, off_lse, off_g, off_x, off_scaled, off_w, off_terms, off_sums, off_hit, off_dz, off_acc, bytes;
};
int make_plan(const char* name, int64_t rows, int64_t depth, const Weight& w, int64_t vocab, bool backward, Plan* q) {
  if (rows < 0 || rows > (1 << 24) || depth <= 0 || depth > (1 << 20) || vocab <= 0 || vocab > (1 << 28) || w.ld < (w.by_word ? depth : vocab))
    return fail(PB_ERR_BAD_SHAPE, "%s: rows=%lld depth=%lld vocab=%lld, rows of the weight %lld apart", name, (long long)rows, (long long)depth, (long long)vocab, (long long)w.ld);
  q->cap = (rows + kRowTile - 1) / kRowTile * kRowTile;
  q->ld_x = (depth + 7) / 8 * 8;
  q->inner_w = w.by_word ? depth : vocab; q->outer_w = w.by_word ? vocab : depth;
  q->pad = w.ld % 8 != 0 || off_by(w.at, 16);
  q->ld_w = q->pad ? (q->inner_w + 7) / 8 * 8 : w.ld;
  q->parts = (vocab + 255) / 256 * (256 / kPart);
  const int64_t most = std::max<int64_t>(256, (int64_t)(kMostGradient / 2) / std::max<int64_t>(1, q->cap) / 256 * 256);
  q->pieces = (int)((vocab + most - 1) / most);
  q->piece = ((vocab + q->pieces - 1) / q->pieces + 255) / 256 * 256;
  q->pieces = (int)((vocab + q->piece - 1) / q->piece);
  size_t at = 256;
  auto take = [&](size_t bytes) { const size_t was = at; at += (bytes + 255) / 256 * 256; return was; };
  q->off_place = take((size_t)rows * 4); q->off_origin = take((size_t)q->cap * 4); q->off_target = take((size_t)q->cap * 4);
  q->off_x = take((size_t)q->cap * q->ld_x * 2);
  q->off_w = take(q->pad ? (size_t)q->outer_w * q->ld_w * 2 : 0);
  q->off_lse = q->off_g = q->off_scaled = q->off_dz = q->off_acc = q->off_terms = q->off_sums = q->off_hit = 0;
  if (backward) {
    q->off_lse = take((size_t)q->cap * 4); q->off_g = take((size_t)q->cap * 4);
    q->off_scaled = take((size_t)q->cap * q->ld_x * 2);
    q->off_dz = take((size_t)q->cap * q->piece * 2);
    q->off_acc = take(q->pieces > 1 ? (size_t)q->cap * ((depth + 255) / 256 * 256) * 4 : 0);
  } else {
    q->off_terms = take((size_t)q->parts * q->cap * 8); q->off_sums = take((size_t)q->parts * q->cap * 4); q->off_hit = take((size_t)q->cap * 4);
  }
  q->bytes = at;
  return PB_OK;
}

struct Positions {
  const void* x;
  int64_t outer, inner, stride_outer, stride_inner, depth;
  const int64_t* targets;
};
int checks(const char* name, const Positions& x, const Weight& w, int64_t vocab, float smoothing, const void* workspace, size_t bytes, bool backward, Plan* q) {
  if (x.outer < 0 || x.inner < 0 || x.stride_outer < 0 || x.stride_inner < 0 || (x.outer > 0 && x.inner > (1 << 24) / x.outer))
    return fail(PB_ERR_BAD_SHAPE, "%s: %lld x %lld positions, %lld and %lld apart", name, (long long)x.outer, (long long)x.inner, (long long)x.stride_outer, (long long)x.stride_inner);
  const int64_t rows = x.outer * x.inner;
  if (int s = make_plan(name, rows, x.depth, w, vocab, backward, q)) return s;
  if (!(smoothing >= 0.0f && smoothing <= 1.0f)) return fail(PB_ERR_BAD_SHAPE, "%s: smoothing %g", name, (double)smoothing);
  if (!w.at || (rows && (!x.x || !x.targets || !workspace))) return fail(PB_ERR_NULL_POINTER, "%s: null argument", name);
  if (off_by(x.x, 2) || off_by(w.at, 2) || off_by(x.targets, 8) || off_by(workspace, 256)) return fail(PB_ERR_MISALIGNED, "%s: misaligned array", name);
  if (rows && bytes < q->bytes) return fail(PB_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu needed", name, bytes, q->bytes);
  return PB_OK;
}

template <typename T> T* part(void* workspace, size_t off) { return reinterpret_cast<T*>(static_cast<unsigned char*>(workspace) + off); }

// numbers the positions, brings their hidden states together and the weight where TMA reads it
int make_ready(const Positions& x, Weight* w, int64_t vocab, const Plan& q, void* ws, float* loss, float* lse_none, const float* lse, const float* g, void* dx, bool scaled, cudaStream_t st) {
  const int rows = (int)(x.outer * x.inner);
  const SelectParams sp{x.targets, vocab, rows, part<int>(ws, 0), part<int>(ws, q.off_place), part<int>(ws, q.off_origin), part<int>(ws, q.off_target), lse, g,
                        part<float>(ws, q.off_lse), part<float>(ws, q.off_g), part<float>(ws, 64), loss, lse_none};
  launch_behind(select_kernel, 1, 1024, 0, st, sp);
  PB_LAUNCH_CHECK("select_kernel");
  const bool vectors = x.depth % 8 == 0 && !off_by(x.x, 16) && (x.outer == 1 || x.stride_outer % 8 == 0) && (x.inner == 1 || x.stride_inner % 8 == 0);
  const GatherParams gp{static_cast<const unsigned short*>(x.x), x.inner, x.stride_outer, x.stride_inner, part<int>(ws, 0), part<int>(ws, q.off_place), part<unsigned short>(ws, q.off_x),
                        scaled ? part<unsigned short>(ws, q.off_scaled) : nullptr, static_cast<unsigned short*>(dx), part<float>(ws, q.off_g), part<float>(ws, 64), rows, (int)x.depth, (int)q.ld_x, vectors, x.depth % 8 == 0 && !off_by(dx, 16)};
  launch_behind(gather_kernel, (unsigned)((rows + kRowTile + 7) / 8), 256, 0, st, gp);
  PB_LAUNCH_CHECK("gather_kernel");
  if (q.pad) {
    const unsigned x_blocks = (unsigned)std::min<int64_t>(8, (q.inner_w + 255) / 256), y = (unsigned)std::min<int64_t>(65535, q.outer_w), z = (unsigned)((q.outer_w + 65534) / 65535);
    for (unsigned k = 0; k < z; ++k) {          // the last round has fewer rows
      const int64_t first = (int64_t)k * 65535, n = std::min<int64_t>(y, q.outer_w - first);
      launch_behind(pad_kernel, dim3(x_blocks, (unsigned)n), 256, 0, st, static_cast<const unsigned short*>(w->at) + first * w->ld, q.inner_w, w->ld, part<unsigned short>(ws, q.off_w) + first * q.ld_w, q.ld_w);
      PB_LAUNCH_CHECK("pad_kernel");
    }
    w->at = part<unsigned short>(ws, q.off_w);
    w->ld = q.ld_w;
  }
  return PB_OK;
}

bool in_vectors(const void* p, int64_t ld) { return !off_by(p, 16) && ld % 8 == 0; }

const unsigned short* words(const Weight& w, int64_t first) { return static_cast<const unsigned short*>(w.at) + (w.by_word ? first * w.ld : first); }

template <class E>
int logits(const Plan& q, const Weight& w, int64_t first, int64_t n, int64_t depth, void* ws, const typename E::Params& e, cudaStream_t st) {
  Params p{};
  p.count = part<int>(ws, 0); p.counted = 1; p.rows = (int)q.cap; p.cols = (int)n; p.depth = (int)depth; p.batch = 1; p.bf16 = 1; p.group = kGroup;
  const Operand x{part<void>(ws, q.off_x), false, q.cap, depth, q.ld_x, q.cap * q.ld_x}, words_of{words(w, first), !w.by_word, n, depth, w.ld, w.ld * 8};
  return w.by_word ? launch<2, 256, false, false, E>(x, words_of, p, e, st) : launch<2, 256, false, true, E>(x, words_of, p, e, st);
}
template <int MODE>
int to_hidden(const Plan& q, const Weight& w, int64_t first, int64_t n, int64_t depth, void* ws, const typename StoreEpilogue<MODE>::Params& e, cudaStream_t st) {
  Params p{};
  p.count = part<int>(ws, 0); p.counted = 1; p.rows = (int)q.cap; p.cols = (int)depth; p.depth = (int)n; p.batch = 1; p.bf16 = 1; p.group = kGroup;
  const Operand dz{part<void>(ws, q.off_dz), false, q.cap, n, q.piece, q.cap * q.piece}, words_of{words(w, first), w.by_word, depth, n, w.ld, w.ld * 8};
  return w.by_word ? launch<2, 256, false, true, StoreEpilogue<MODE>>(dz, words_of, p, e, st) : launch<2, 256, false, false, StoreEpilogue<MODE>>(dz, words_of, p, e, st);
}

}  // namespace

int linear_xent_status_fetch(unsigned int* out) { return status_fetch(out); }
}  // namespace pb

using namespace pb;

extern "C" size_t pb_linear_xent_workspace_size(int64_t rows, int64_t depth, const void* weight, int64_t ld, int by_word, int64_t vocab, int backward) {
  Plan q;
  return make_plan("pb_linear_xent", rows, depth, Weight{weight, ld, by_word != 0}, vocab, backward != 0, &q) ? 0 : q.bytes;
}

extern "C" int pb_linear_xent(const void* x, int64_t outer, int64_t inner, int64_t stride_outer, int64_t stride_inner, int64_t depth, const void* weight, int64_t ld, int by_word, int64_t vocab,
                              const int64_t* targets, float smoothing, float* loss, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  const Positions at{x, outer, inner, stride_outer, stride_inner, depth, targets};
  Weight w{weight, ld, by_word != 0};
  Plan q;
  if (int s = checks("pb_linear_xent", at, w, vocab, smoothing, workspace, workspace_bytes, false, &q)) return s;
  if (outer * inner == 0) return PB_OK;
  if (!loss || !lse) return fail(PB_ERR_NULL_POINTER, "pb_linear_xent: null argument");
  if (off_by(loss, 4) || off_by(lse, 4)) return fail(PB_ERR_MISALIGNED, "pb_linear_xent: misaligned array");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int s = make_ready(at, &w, vocab, q, workspace, loss, lse, nullptr, nullptr, nullptr, false, st)) return s;
  int* target = part<int>(workspace, q.off_target);
  float2* terms = part<float2>(workspace, q.off_terms);
  float *sums = part<float>(workspace, q.off_sums), *hit = part<float>(workspace, q.off_hit);
  const unsigned blocks = (unsigned)(q.cap / 32);
  if (smoothing != 0.0f) {
    if (int s = logits<StatsEpilogue<true>>(q, w, 0, vocab, depth, workspace, {target, terms, sums, hit, q.cap}, st)) return s;
    launch_behind(join_kernel<true>, blocks, 1024, 0, st, terms, sums, hit, part<int>(workspace, q.off_origin), part<int>(workspace, 0), q.cap, (int)q.parts, smoothing, 1.0f / (float)vocab, loss, lse);
  } else {
    if (int s = logits<StatsEpilogue<false>>(q, w, 0, vocab, depth, workspace, {target, terms, sums, hit, q.cap}, st)) return s;
    launch_behind(join_kernel<false>, blocks, 1024, 0, st, terms, sums, hit, part<int>(workspace, q.off_origin), part<int>(workspace, 0), q.cap, (int)q.parts, 0.0f, 0.0f, loss, lse);
  }
  PB_LAUNCH_CHECK("join_kernel");
  return PB_OK;
}

extern "C" int pb_linear_xent_bwd(const void* x, int64_t outer, int64_t inner, int64_t stride_outer, int64_t stride_inner, int64_t depth, const void* weight, int64_t ld, int by_word, int64_t vocab,
                                  const int64_t* targets, float smoothing, const float* lse, const float* g, void* dx, void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  const Positions at{x, outer, inner, stride_outer, stride_inner, depth, targets};
  Weight w{weight, ld, by_word != 0};
  Plan q;
  if (int s = checks("pb_linear_xent_bwd", at, w, vocab, smoothing, workspace, workspace_bytes, true, &q)) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (off_by(lse, 4) || off_by(g, 4) || off_by(dx, 2) || off_by(dweight, 2)) return fail(PB_ERR_MISALIGNED, "pb_linear_xent_bwd: misaligned array");
  if (outer * inner == 0) {
    if (dweight) PB_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)depth * vocab * 2, st));
    return PB_OK;
  }
  if (!lse || !g) return fail(PB_ERR_NULL_POINTER, "pb_linear_xent_bwd: null argument");
  if (!dx && !dweight) return PB_OK;
  if (int s = make_ready(at, &w, vocab, q, workspace, nullptr, nullptr, lse, g, dx, dweight != nullptr, st)) return s;
  int *origin = part<int>(workspace, q.off_origin), *target = part<int>(workspace, q.off_target);
  __nv_bfloat16 *dz = part<__nv_bfloat16>(workspace, q.off_dz), *d_hidden = static_cast<__nv_bfloat16*>(dx);
  float4* acc = part<float4>(workspace, q.off_acc);
  const float* gs = part<float>(workspace, q.off_g);
  const float by = smoothing <= 0.5f ? 1.0f - smoothing : 1.0f;      // without a target's share to speak of, any
  CUtensorMap dz_blocks;
  if (int s = make_map(&dz_blocks, dz, true, q.piece, q.cap, q.piece, 1, q.cap * q.piece, 32)) return s;
  for (int k = 0; k < q.pieces; ++k) {
    const int64_t first = k * q.piece, n = std::min(q.piece, vocab - first);
    if (int s = logits<GradientEpilogue>(q, w, first, n, depth, workspace,
                                         {dz_blocks, target, part<float>(workspace, q.off_lse), (int)first, 1.0f / by, smoothing / (float)vocab / by, (1.0f - smoothing) / by}, st))
      return s;
    if (dx) {
      const bool vectors = in_vectors(dx, depth);
      if (int s = q.pieces == 1       ? to_hidden<kOnly>(q, w, first, n, depth, workspace, {d_hidden, acc, origin, gs, by, depth, vectors}, st)
                : k == 0              ? to_hidden<kFirst>(q, w, first, n, depth, workspace, {d_hidden, acc, origin, gs, by, depth, vectors}, st)
                : k < q.pieces - 1    ? to_hidden<kMore>(q, w, first, n, depth, workspace, {d_hidden, acc, origin, gs, by, depth, vectors}, st)
                                      : to_hidden<kLast>(q, w, first, n, depth, workspace, {d_hidden, acc, origin, gs, by, depth, vectors}, st))
        return s;
    }
    if (dweight) {
      Params p{};
      p.count = part<int>(workspace, 0); p.counted = 2; p.depth = (int)q.cap; p.batch = 1; p.bf16 = 1; p.group = kGroup;
      p.rows = (int)(w.by_word ? n : depth); p.cols = (int)(w.by_word ? depth : n);
      const Operand hidden{part<void>(workspace, q.off_scaled), true, depth, q.cap, q.ld_x, q.cap * q.ld_x}, gradient{dz, true, n, q.cap, q.piece, q.cap * q.piece};
      const int64_t ld_out = w.by_word ? depth : vocab;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(dweight) + (w.by_word ? first * depth : first);
      const StoreEpilogue<kOnly>::Params e{out, nullptr, nullptr, part<float>(workspace, 64), by, ld_out, in_vectors(out, ld_out)};
      if (int s = w.by_word ? launch<2, 256, true, true, StoreEpilogue<kOnly>>(gradient, hidden, p, e, st) : launch<2, 256, true, true, StoreEpilogue<kOnly>>(hidden, gradient, p, e, st)) return s;
    }
  }
  return PB_OK;
}
