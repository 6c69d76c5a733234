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
// which is the results' own rounding; now 2.3e-3).  dx takes g (1 - a) in f32 at its end; for dW the hidden states are multiplied by g over the largest g, exactly 1
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
// One CTA: 8192 positions at a time, a warp's by ballot, the warps' numbers added up.
__global__ void __launch_bounds__(1024) select_kernel(const __grid_constant__ SelectParams p) {
  grid_wait();
  constexpr int kRounds = 8;
  __shared__ int sums[kRounds * 32];
  __shared__ float tops[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  float most = 0.0f;
  for (int first = 0; first < p.rows; first += kRounds * 1024) {
    int64_t t[kRounds];
    float l[kRounds], g[kRounds];
    uint32_t there[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = first + r * 1024 + threadIdx.x;
      t[r] = i < p.rows ? p.targets[i] : -1;
      l[r] = p.lse && i < p.rows ? p.lse[i] : 0.0f;
      g[r] = p.lse && i < p.rows ? p.g[i] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const bool is = t[r] >= 0 && t[r] < p.vocab;
      there[r] = __ballot_sync(0xffffffffu, is);
      if (is) most = fmaxf(most, fabsf(g[r]));
      if (lane == 0) sums[r * 32 + warp] = __popc(there[r]);
    }
    __syncthreads();
    if (warp == 0) {
      int upto = 0;
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        int n = sums[r * 32 + lane], all = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int below = __shfl_up_sync(0xffffffffu, all, o);
          if (lane >= o) all += below;
        }
        sums[r * 32 + lane] = upto + all - n;
        upto += __shfl_sync(0xffffffffu, all, 31);
      }
      if (lane == 0) tops[0] = __int_as_float(upto);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = first + r * 1024 + threadIdx.x;
      if (i >= p.rows) break;
      if (there[r] >> lane & 1) {
        const int at = before + sums[r * 32 + warp] + __popc(there[r] & ((1u << lane) - 1));
        p.place[i] = at; p.origin[at] = i; p.target[at] = (int)t[r];
        if (p.lse) { p.lse_out[at] = l[r]; p.g_out[at] = g[r]; }
      } else {
        p.place[i] = -1;
        if (p.loss) {
          p.loss[i] = t[r] < 0 ? 0.0f : nanf("");
          p.lse_none[i] = 0.0f;
        }
      }
    }
    before += __float_as_int(tops[0]);
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.count = before;
  if (!p.lse) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (lane == 0) tops[warp] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) most = fmaxf(most, tops[w]);
    *p.g_most = most;
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
  uint32_t items;
  FastDiv per_row;
};
// A warp takes kGather elements of a row; kRowTile rows more are zeros behind the last.
constexpr int kGather = 1024;
__global__ void __launch_bounds__(128) gather_kernel(const __grid_constant__ GatherParams p) {
  grid_wait();
  const uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const int row = (int)p.per_row.div(item), lane = threadIdx.x & 31;
  const int c0 = (int)(item - row * p.per_row.d) * kGather, c1 = min(c0 + kGather, p.ld), behind = *p.count + row - p.rows;
  const int to = row < p.rows ? p.place[row] : behind < (*p.count + kRowTile - 1) / kRowTile * kRowTile ? behind : -1;
  unsigned short *out = p.out + (int64_t)to * p.ld, *scaled = p.scaled ? p.scaled + (int64_t)to * p.ld : nullptr;
  if (row >= p.rows) {
    if (to < 0) return;
    for (int c = c0 + lane * 8; c < c1; c += 256) {
      *reinterpret_cast<uint4*>(out + c) = make_uint4(0u, 0u, 0u, 0u);
      if (scaled) *reinterpret_cast<uint4*>(scaled + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  if (to < 0) {
    if (!p.dx) return;
    unsigned short* none = p.dx + (int64_t)row * p.depth;
    if (p.dx_vectors) for (int c = c0 + lane * 8; c < min(c1, p.depth); c += 256) *reinterpret_cast<uint4*>(none + c) = make_uint4(0u, 0u, 0u, 0u);
    else for (int c = c0 + lane; c < min(c1, p.depth); c += 32) none[c] = 0;
    return;
  }
  const unsigned short* from = p.x + row / p.inner * p.stride_outer + row % p.inner * p.stride_inner;
  float by = 1.0f;
  if (scaled) {
    const float most = *p.g_most, g = p.g[to];
    by = most == 0.0f ? g : __fdiv_rn(g, most);          // every g is zero, or none is a number
  }
  auto times = [&](uint32_t x) { return pack_bf16x2(__uint_as_float(x << 16) * by, __uint_as_float(x & 0xffff0000u) * by); };
  if (p.vectors) {
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = c0 + lane * 8 + 256 * k;
      v[k] = c < p.depth ? *reinterpret_cast<const uint4*>(from + c) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = c0 + lane * 8 + 256 * k;
      if (c >= c1) break;
      *reinterpret_cast<uint4*>(out + c) = v[k];
      if (scaled) *reinterpret_cast<uint4*>(scaled + c) = make_uint4(times(v[k].x), times(v[k].y), times(v[k].z), times(v[k].w));
    }
  } else {
#pragma unroll 4
    for (int c = c0 + lane; c < c1; c += 32) {
      const unsigned short v = c < p.depth ? from[c] : (unsigned short)0;
      out[c] = v;
      if (scaled) scaled[c] = (unsigned short)times(v);
    }
  }
}

// A weight whose rows do not lie as TMA wants them, to rows that do: a thread takes eight elements, out of the two aligned vectors that hold them wherever both lie in [begin, end), the weight's own
// memory.  65537 words of 2048: 81 us, where
// two bytes a thread took 240.
struct PadParams {
  const unsigned short *from, *begin, *end;
  int64_t inner, ld_from;
  unsigned short* to;
  int64_t ld_to;
};
__global__ void __launch_bounds__(256) pad_kernel(const __grid_constant__ PadParams p) {
  grid_wait();
  const int64_t row = blockIdx.y;
  const unsigned short* from = p.from + row * p.ld_from;
  unsigned short* to = p.to + row * p.ld_to;
  const int off = (int)(reinterpret_cast<uintptr_t>(from) / 2 % 8);      // of every eight elements in their first vector
#pragma unroll 4
  for (int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; c < p.inner; c += (int64_t)gridDim.x * 256 * 8) {
    const unsigned short* at = from + c - off;
    uint32_t w[9];
    if (at >= p.begin && at + 16 <= p.end) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(at)), b = __ldg(reinterpret_cast<const uint4*>(at) + 1);
      const uint32_t all[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 5; ++k) w[k] = off & 4 ? (off & 2 ? all[min(k + 3, 7)] : all[min(k + 2, 7)]) : (off & 2 ? all[k + 1] : all[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = off & 1 ? __funnelshift_r(w[k], w[k + 1], 16) : w[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = c + 2 * k < p.inner ? from[c + 2 * k] : 0u, hi = c + 2 * k + 1 < p.inner ? from[c + 2 * k + 1] : 0u;
        w[k] = lo | hi << 16;
      }
    }
    *reinterpret_cast<uint4*>(to + c) = make_uint4(w[0], w[1], w[2], w[3]);      // rows end at whole vectors
  }
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

// D times `by` and scale[row], or scale[0] without origin, as bf16 in rows of `ld`; with origin row r goes to row origin[r].  By TMA where that reaches the rows (`blocks`), else by the lanes.
struct StoreEpilogue : Grouped {
  struct Params { CUtensorMap blocks; __nv_bfloat16* out; const int* origin; const float* scale; float by; int64_t ld; bool vectors; };
  const Params& p;
  int row;
  float scale;
  __device__ __forceinline__ explicit StoreEpilogue(const Params& e) : p(e) {}
  __device__ __forceinline__ void begin(const Place& at) {
    row = at.row < at.rows ? (p.origin ? p.origin[at.row] : at.row) : -1;
    scale = row < 0 ? 0.0f : p.by * p.scale[p.origin ? at.row : 0];
  }
  __device__ __forceinline__ void block(const Place& at, int c, float (&v)[kBlock]) {
#pragma unroll
    for (int j = 0; j < kBlock; ++j) v[j] *= scale;
    if (!p.origin && p.vectors) {
      if (at.lane == 0) Slots::wait_read();
      __syncwarp();
      Slots::stage<Bf16>(at, 0, v);
      Slots::hand_over();
      if (at.lane == 0 && at.row < at.rows) { Slots::send(at, 0, &p.blocks, at.col + c, at.row, 0); Slots::sent(); }
      return;
    }
    Slots::stage<Bf16>(at, 0, v);
    __syncwarp();
    Slots::scatter(at.own, at.lane, reinterpret_cast<unsigned short*>(p.out + at.col + c), p.ld, row, at.cols - at.col - c, p.vectors);
  }
  __device__ __forceinline__ void end(const Place&) {}
  __device__ __forceinline__ void finish(const Place& at) { if (at.lane == 0) Slots::wait_sent(); }
};

// ---- the parts of a position's logits together ----------------------------------------------------------------------
// POSITIONS a CTA, a lane of each so many one of them; the others, 1024 / POSITIONS, take a part in turn.  65536 words: 64 positions by 32 | 8 10.8 | 6.5 us, 8192 of them 12.7 | 20.1
constexpr int kManyPositions = 2048;      // from there on 32 fill the chip
template <bool MEAN, int POSITIONS>
__global__ void __launch_bounds__(1024) join_losses_kernel(const float2* terms, const float* sums, const float* hit, const int* origin, const int* count, int64_t cap, int parts, float smoothing,
                                                    float inv_vocab, float* loss, float* lse) {
  grid_wait();
  __shared__ float red[3][32][POSITIONS + 1];
  const int n = *count, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * POSITIONS + lane % POSITIONS;
  if (blockIdx.x * POSITIONS >= n) return;
  float m = -INFINITY, s = 0.0f, sum = 0.0f;
  auto add = [&](float m2, float s2, float sum2) {
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
    s = s * exp2_approx((m - base) * kLog2E) + s2 * exp2_approx((m2 - base) * kLog2E);
    m = top; sum += sum2;
  };
#pragma unroll 8
  for (int k = threadIdx.x / POSITIONS; k < parts; k += 1024 / POSITIONS) {      // rows up to cap are there, if not told of
    const float2 t = terms[(int64_t)k * cap + row];
    add(t.x, t.y, MEAN ? sums[(int64_t)k * cap + row] : 0.0f);
  }
#pragma unroll
  for (int o = POSITIONS; o < 32; o <<= 1) add(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), __shfl_xor_sync(0xffffffffu, sum, o));
  if (lane < POSITIONS) { red[0][warp][lane] = m; red[1][warp][lane] = s; red[2][warp][lane] = sum; }
  __syncthreads();
  if (warp >= POSITIONS) return;
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
  const int number = blockIdx.x * POSITIONS + warp;
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
  int64_t rows;
  int pieces;
  bool pad;
  size_t off_place, off_origin, off_target, off_lse, off_g, off_x, off_scaled, off_w, off_terms, off_sums, off_hit, off_dz, off_parts, bytes;
};
template <typename T> T* part(void* workspace, size_t off) { return reinterpret_cast<T*>(static_cast<unsigned char*>(workspace) + off); }
// Where there is one tile of rows, half of a pair's 256 would be idle: a CTA's 128 x 256.  The product of 64 positions of 2048 with 65536 words:
// 62 us by a pair's, 50 so (41 are the weight's bytes).
bool few_rows(const Plan& q) { return q.rows <= 128; }

// dx's product of a piece: few tiles of many stages, so they are cut, by the most positions that may count; how many do is known on the device alone
Params hidden_params(const Plan& q, int64_t n, int64_t depth, void* ws) {
  Params p{};
  p.count = part<int>(ws, 0); p.counted = 1; p.rows = (int)(few_rows(q) ? 128 : q.cap); p.cols = (int)depth; p.depth = (int)n; p.batch = 1; p.bf16 = 1; p.group = kGroup;
  if (few_rows(q)) cut_stages<1, 256>(&p, (int)(q.piece / kDepth));
  else cut_stages<2, 256>(&p, (int)(q.piece / kDepth));
  return p;
}
int make_plan(const char* name, int64_t rows, int64_t depth, const Weight& w, int64_t vocab, bool backward, Plan* q) {
  if (rows < 0 || rows > (1 << 24) || depth <= 0 || depth > (1 << 20) || vocab <= 0 || vocab > (1 << 28) || w.ld < (w.by_word ? depth : vocab))
    return fail(PB_ERR_BAD_SHAPE, "%s: rows=%lld depth=%lld vocab=%lld, rows of the weight %lld apart", name, (long long)rows, (long long)depth, (long long)vocab, (long long)w.ld);
  q->rows = rows;
  q->cap = (rows + kRowTile - 1) / kRowTile * kRowTile;
  q->ld_x = (depth + 63) / 64 * 64;      // rows of whole 128-byte lines
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
  q->off_lse = q->off_g = q->off_scaled = q->off_dz = q->off_parts = q->off_terms = q->off_sums = q->off_hit = 0;
  if (backward) {
    q->off_lse = take((size_t)q->cap * 4); q->off_g = take((size_t)q->cap * 4);
    q->off_scaled = take((size_t)q->cap * q->ld_x * 2);
    q->off_dz = take((size_t)q->cap * q->piece * 2);
    const Params p = hidden_params(*q, q->piece, depth, nullptr);
    q->off_parts = take((size_t)(few_rows(*q) ? parts_of<1, 256>(p) : parts_of<2, 256>(p)) * 16);
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


// numbers the positions, brings their hidden states together and the weight where TMA reads it
int make_ready(const Positions& x, Weight* w, int64_t vocab, const Plan& q, void* ws, float* loss, float* lse_none, const float* lse, const float* g, void* dx, bool scaled, cudaStream_t st) {
  const int rows = (int)(x.outer * x.inner);
  const SelectParams sp{x.targets, vocab, rows, part<int>(ws, 0), part<int>(ws, q.off_place), part<int>(ws, q.off_origin), part<int>(ws, q.off_target), lse, g,
                        part<float>(ws, q.off_lse), part<float>(ws, q.off_g), part<float>(ws, 64), loss, lse_none};
  launch_behind(select_kernel, 1, 1024, 0, st, sp);
  PB_LAUNCH_CHECK("select_kernel");
  const bool vectors = x.depth % 8 == 0 && !off_by(x.x, 16) && (x.outer == 1 || x.stride_outer % 8 == 0) && (x.inner == 1 || x.stride_inner % 8 == 0);
  const int64_t per_row = (q.ld_x + kGather - 1) / kGather;
  if ((rows + kRowTile) * per_row > kMaxIndexed) return fail(PB_ERR_BAD_SHAPE, "pb_linear_xent: %d positions of %lld", rows, (long long)x.depth);
  const GatherParams gp{static_cast<const unsigned short*>(x.x), x.inner, x.stride_outer, x.stride_inner, part<int>(ws, 0), part<int>(ws, q.off_place), part<unsigned short>(ws, q.off_x),
                        scaled ? part<unsigned short>(ws, q.off_scaled) : nullptr, static_cast<unsigned short*>(dx), part<float>(ws, q.off_g), part<float>(ws, 64), rows, (int)x.depth, (int)q.ld_x, vectors, x.depth % 8 == 0 && !off_by(dx, 16), (uint32_t)((rows + kRowTile) * per_row), FastDiv((uint32_t)per_row)};
  launch_behind(gather_kernel, (gp.items + 3) / 4, 128, 0, st, gp);
  PB_LAUNCH_CHECK("gather_kernel");
  if (q.pad) {
    const unsigned short* begin = static_cast<const unsigned short*>(w->at);
    const unsigned short* end = begin + (q.outer_w - 1) * w->ld + q.inner_w;
    const unsigned x_blocks = (unsigned)std::min<int64_t>(8, (q.inner_w + 2047) / 2048), y = (unsigned)std::min<int64_t>(65535, q.outer_w), z = (unsigned)((q.outer_w + 65534) / 65535);
    for (unsigned k = 0; k < z; ++k) {          // the last round has fewer rows
      const int64_t first = (int64_t)k * 65535, n = std::min<int64_t>(y, q.outer_w - first);
      launch_behind(pad_kernel, dim3(x_blocks, (unsigned)n), 256, 0, st, PadParams{begin + first * w->ld, begin, end, q.inner_w, w->ld, part<unsigned short>(ws, q.off_w) + first * q.ld_w, q.ld_w});
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
  p.count = part<int>(ws, 0); p.counted = 1; p.rows = (int)(few_rows(q) ? 128 : q.cap); p.cols = (int)n; p.depth = (int)depth; p.batch = 1; p.bf16 = 1; p.group = kGroup;
  const Operand x{part<void>(ws, q.off_x), false, q.cap, depth, q.ld_x, q.cap * q.ld_x}, words_of{words(w, first), !w.by_word, n, depth, w.ld, w.ld * 8};
  if (few_rows(q)) return w.by_word ? launch<1, 256, false, false, E>(x, words_of, p, e, st) : launch<1, 256, false, true, E>(x, words_of, p, e, st);
  return w.by_word ? launch<2, 256, false, false, E>(x, words_of, p, e, st) : launch<2, 256, false, true, E>(x, words_of, p, e, st);
}
int to_hidden(const Plan& q, const Weight& w, int64_t first, int64_t n, int64_t depth, void* ws, cudaStream_t st) {
  const Params p = hidden_params(q, n, depth, ws);
  const Operand dz{part<void>(ws, q.off_dz), false, q.cap, n, q.piece, q.cap * q.piece}, words_of{words(w, first), w.by_word, depth, n, w.ld, w.ld * 8};
  using E = PartEpilogue<true>;
  const E::Params e{part<float4>(ws, q.off_parts), first > 0};
  if (few_rows(q)) return w.by_word ? launch<1, 256, false, true, E>(dz, words_of, p, e, st) : launch<1, 256, false, false, E>(dz, words_of, p, e, st);
  return w.by_word ? launch<2, 256, false, true, E>(dz, words_of, p, e, st) : launch<2, 256, false, false, E>(dz, words_of, p, e, st);
}

}  // namespace

int linear_xent_status_fetch(unsigned int* out) { return status_fetch(out); }
#ifdef PB_DIAGNOSTICS
void linear_xent_control(uint32_t polls, int withhold) { control(polls, withhold); }
#endif
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
  const bool many = q.rows >= kManyPositions;
  const unsigned blocks = (unsigned)(q.cap / (many ? 32 : 8));
  auto go = [&](auto kernel) {
    launch_behind(kernel, blocks, 1024, 0, st, terms, sums, hit, part<int>(workspace, q.off_origin), part<int>(workspace, 0), q.cap, (int)q.parts, smoothing, 1.0f / (float)vocab, loss, lse);
  };
  if (smoothing != 0.0f) {
    if (int s = logits<StatsEpilogue<true>>(q, w, 0, vocab, depth, workspace, {target, terms, sums, hit, q.cap}, st)) return s;
    many ? go(join_losses_kernel<true, 32>) : go(join_losses_kernel<true, 8>);
  } else {
    if (int s = logits<StatsEpilogue<false>>(q, w, 0, vocab, depth, workspace, {target, terms, sums, hit, q.cap}, st)) return s;
    many ? go(join_losses_kernel<false, 32>) : go(join_losses_kernel<false, 8>);
  }
  PB_LAUNCH_CHECK("join_losses_kernel");
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
  const float* gs = part<float>(workspace, q.off_g);
  const float by = smoothing <= 0.5f ? 1.0f - smoothing : 1.0f;      // without a target's share to speak of, any
  CUtensorMap dz_blocks;
  if (int s = make_map(&dz_blocks, dz, true, q.piece, q.cap, q.piece, 1, q.cap * q.piece, 32)) return s;
  for (int k = 0; k < q.pieces; ++k) {
    const int64_t first = k * q.piece, n = std::min(q.piece, vocab - first);
    if (int s = logits<GradientEpilogue>(q, w, first, n, depth, workspace,
                                         {dz_blocks, target, part<float>(workspace, q.off_lse), (int)first, 1.0f / by, smoothing / (float)vocab / by, (1.0f - smoothing) / by}, st))
      return s;
    if (dx)
      if (int s = to_hidden(q, w, first, n, depth, workspace, st)) return s;
    if (dweight) {
      Params p{};
      p.count = part<int>(workspace, 0); p.counted = 2; p.depth = (int)q.cap; p.batch = 1; p.bf16 = 1; p.group = kGroup;
      p.rows = (int)(w.by_word ? n : depth); p.cols = (int)(w.by_word ? depth : n);
      const Operand hidden{part<void>(workspace, q.off_scaled), true, depth, q.cap, q.ld_x, q.cap * q.ld_x}, gradient{dz, true, n, q.cap, q.piece, q.cap * q.piece};
      const int64_t ld_out = w.by_word ? depth : vocab;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(dweight) + (w.by_word ? first * depth : first);
      StoreEpilogue::Params e{{}, out, nullptr, part<float>(workspace, 64), by, ld_out, in_vectors(out, ld_out)};
      if (e.vectors)
        if (int s = make_map(&e.blocks, out, true, p.cols, p.rows, ld_out, 1, (int64_t)p.rows * ld_out, 32)) return s;
      if (int s = w.by_word ? launch<2, 256, true, true, StoreEpilogue>(gradient, hidden, p, e, st) : launch<2, 256, true, true, StoreEpilogue>(hidden, gradient, p, e, st)) return s;
    }
  }
  if (dx) {
    const StoreEpilogue::Params e{{}, d_hidden, origin, gs, by, depth, in_vectors(dx, depth)};
    const Params p = hidden_params(q, q.piece, depth, workspace);
    const float4* parts = part<float4>(workspace, q.off_parts);
    if (int s = few_rows(q) ? launch_finish<1, 256, StoreEpilogue>(parts, p, e, st) : launch_finish<2, 256, StoreEpilogue>(parts, p, e, st)) return s;
  }
  return PB_OK;
}
