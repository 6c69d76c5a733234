// Log probabilities of given tokens with the entropy and the best alternatives of every position, and the logits' gradient.
//
// A row of logits z:  m = max z,  d_j = z_j - m,  S = sum_j exp(d_j)
//   logp_j  = d_j - log S
//   entropy = log S - sum_j exp(d_j) d_j / S          (both terms are at or above zero: nothing cancels)
//   top     = the k largest z, equal ones in the order of their indices
// m and log S are kept apart for the backward pass: their sum rounds at the size of the logits, and exp(z - sum) would carry that error into
// every probability of the row.
//   dz_j = sum_i g_i [j == t_i] + sum_i h_i [j == top_i] - p_j (sum_i g_i + sum_i h_i + g_entropy (logp_j + entropy))
// with g the cotangents of the given tokens' log probabilities and h those of the alternatives'.
//
// Exponentials are ex2.approx.ftz of a difference times log2 e: within 2^-22, and a probability below 2^-126 is 0, also as the gradient's factor.
//
// Floor: HBM.  The forward pass reads the logits once (4 or 2 bytes each), the backward pass once more and writes dz.  What it takes beside that is an
// exponential per logit (16 a cycle and SM: 73 % of a bf16 logit's time at 6.5 TB/s) and six to seven instructions, so packed f32x2 arithmetic, and for the
// alternatives no more than a thread's two best vectors while the row goes by.  On one B200, us (and of the measured 6.53 TB/s):
//   2000 x 65536 bf16     48 (84 %) without alternatives, 55 with five, 68 with 64
//   1000 x 65536 f32      43.5 (92 %), 60 with 64;  4096 x 65536 f32, forward and gradient 509 (97 %)
//   one row of 65536 f32, five alternatives: 5.5, a launch and some ten dependent steps of 0.2 to 0.8 each
#include "common.cuh"

#include <cooperative_groups.h>

namespace pb {
namespace {

namespace cg = cooperative_groups;

constexpr int kLoads = 4;                  // 16-byte loads that a thread has in flight
constexpr int kBackThreads = 256;
constexpr int kMaxTop = 128, kMaxTokens = 128;
constexpr int kCandidates = 1024;          // keys of a row that are looked at together
constexpr uint32_t kHalve = 16;            // alternatives up to which the bound is a group's key
constexpr uint32_t kNarrow = 256;          // more keys than this become fewer before they are ranked
constexpr int kMaxCluster = 8;             // CTAs that share a row; kMaxCluster * kMaxTop <= kCandidates

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {      // unlike fmaxf, a NaN stays one
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
constexpr float kFar = -1e30f;             // a difference below it weighs nothing, and times a weight of zero it is zero where -inf is NaN

// 16 bytes of logits as numbers, two at a time, and their largest
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kSize = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float2 (&v)[2]) {
    v[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y)); v[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[2]) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
  static __device__ __forceinline__ float at(const uint4& r, uint32_t i) { return __uint_as_float(i < 2 ? i == 0 ? r.x : r.y : i == 2 ? r.z : r.w); }
  static __device__ __forceinline__ float top(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kSize = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float2 (&v)[4]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[4]) {
    return make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y), pack_bf16x2(v[2].x, v[2].y), pack_bf16x2(v[3].x, v[3].y));
  }
  static __device__ __forceinline__ float at(const uint4& r, uint32_t i) {
    const uint32_t w = i < 4 ? i < 2 ? r.x : r.y : i < 6 ? r.z : r.w;
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
  static __device__ __forceinline__ float top(const uint4& r) {
    auto both = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2(__hmax2(both(r.x), both(r.y)), __hmax2(both(r.z), both(r.w)));      // of a number and a NaN the number
    return fmaxf(__low2float(m), __high2float(m));
  }
};

// A maximum, the sum of exp(z - maximum) and the sum of exp(z - maximum) (z - maximum).  While the maximum is -inf (nothing but -inf seen) the
// differences are taken from 0, so that -inf - -inf does not make a NaN of a logit that only weighs nothing.
struct Sums { float m, s, w; };
struct Terms : Sums {
  __device__ __forceinline__ Terms() : Sums{-INFINITY, 0.0f, 0.0f} {}
  __device__ __forceinline__ Terms(const Sums& o) : Sums(o) {}
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.0f : m; }
  __device__ __forceinline__ void raise(float top) {
    const float by = m - top, c = exp2_fast(by * kLog2e);
    w = c == 0.0f ? c * s : c * (w + s * by);      // c = 0: by may be infinite (s may be NaN and stays so)
    s *= c;
    m = top;
  }
  __device__ __forceinline__ void add(float z, float from) {
    const float d = max_nan(z - from, kFar), e = exp2_fast(d * kLog2e);
    s += e;
    w += e * d;
  }
  // the terms of LANES lanes of a warp together, in each of them
  template <int LANES> __device__ __forceinline__ void over_lanes() {
    float top = m;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float by = max_nan(m - (top == -INFINITY ? 0.0f : top), kFar), c = exp2_fast(by * kLog2e);      // m = -inf: sums of zero
    w = c * (w + s * by);
    s *= c;
    m = top;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      w += __shfl_xor_sync(0xffffffffu, w, o);
    }
  }
};

// A logit and its index as one number: larger for a larger logit, and among equal ones for a lower index.  -0 is 0; NaN ranks with -inf.
// No key is 0.
__device__ __forceinline__ uint32_t order_of(float z) {
  const uint32_t b = __float_as_uint(z != z ? -INFINITY : z + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ uint64_t key_of(float z, uint32_t index) { return (uint64_t)order_of(z) << 32 | (uint32_t)~index; }

struct Rows {      // row r at (r / inner) * stride_outer + (r % inner) * stride_inner
  FastDiv by_inner;
  int64_t stride_outer, stride_inner;
  __device__ __forceinline__ int64_t at(uint32_t r) const {
    const uint32_t o = by_inner.div(r);
    return o * stride_outer + (r - o * by_inner.d) * stride_inner;
  }
};

// A row as elements up to the first 16-byte boundary, whole 16-byte vectors and the rest; CTA `rank` of `ctas` has every vector of its slice, the
// first CTA also the elements before and the last one those behind.
template <typename T> struct Slice {
  static constexpr int kVec = Vec<T>::kSize;
  const T* z;
  uint32_t head, tail, tail_at, first, count;      // count vectors from vector `first` on
  __device__ __forceinline__ Slice(const T* row, uint32_t vocab, uint32_t rank, uint32_t ctas) : z(row) {
    head = min((uint32_t)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (uint32_t)sizeof(T), vocab);
    const uint32_t vecs = (vocab - head) / kVec, per = ctas == 1 ? vecs : (vecs + ctas - 1) / ctas;
    tail_at = head + vecs * kVec;
    tail = vocab - tail_at;
    first = min(rank * per, vecs);
    count = min(per, vecs - first);
    if (rank != 0) head = 0;
    if (rank != ctas - 1) tail = 0;
  }
  // index of its first vector's first element: tail_at is a number of whole vectors behind the elements before the first one
  __device__ __forceinline__ uint32_t at0() const { return first * kVec + tail_at % kVec; }
  __device__ __forceinline__ uint32_t elements() const { return head + tail + count * kVec; }
};

struct Halving { uint32_t counts[3], lowest, highest; };      // `lowest` ~0, the others 0 behind a barrier

template <int THREADS> struct Shared {
  uint64_t cand[kCandidates];
  uint64_t groups[32];             // the best keys of groups of threads
  uint64_t sorted[kMaxTop];
  uint64_t gathered[kMaxCluster * kMaxTop];      // of a cluster's CTAs, in its first one
  uint64_t bound;
  Sums terms[THREADS / 32], cta, of_cta[kMaxCluster];
  uint32_t n_cand, n_hot;
  Halving halving;
  uint16_t hot[THREADS];
};

// For every key in[0, n), which lie at 16 bytes, how many are above it, as done(index, key, above) in one thread.  Where there are fewer keys than threads, neighbouring threads share one.
template <int THREADS, typename Done> __device__ __forceinline__ void rank_keys(const uint64_t* in, uint32_t n, Done done) {
  const uint32_t tid = threadIdx.x, share = n <= THREADS / 8 ? 8 : n <= THREADS / 4 ? 4 : n <= THREADS / 2 ? 2 : 1;
  const uint32_t part = tid % share, step = THREADS / share;
  for (uint32_t i0 = tid / 32 * 32 / share; i0 < n; i0 += step) {      // a warp's threads go round together
    const uint32_t i = i0 + tid % 32 / share;
    const uint64_t key = i < n ? in[i] : ~0ull;
    uint32_t above = 0;
#pragma unroll 4
    for (uint32_t j = part * 2; j + 1 < n; j += share * 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(in + j);
      above += (two.x > key) + (two.y > key);
    }
    if ((n & 1) && part == 0) above += in[n - 1] > key;
    for (uint32_t o = 1; o < share; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (i < n && part == 0) done(i, key, above);
  }
}

__device__ __forceinline__ void reset(Halving& h) {
  if (threadIdx.x < 3) h.counts[threadIdx.x] = 0;
  if (threadIdx.x == 0) { h.lowest = ~0u; h.highest = 0; }
}

// A bound that at least k and, where it is above -inf, at most `most` of the threads' keys reach, found by halving between the lowest and the highest of them.  Where those are far apart (masks
// of the type's lowest value, -inf), thirty halvings would only come to where the others are: there it goes down from the highest, four times as far each time, until k reach it, and halves
// then (48 rows of 65536 under such masks, 20 alternatives, us: 13.9 | 9.8; without masks going down takes more steps, 9.1 | 9.6).  k of the keys are not 0, none of those is another's like, and their
// indices are below vocab; every(f) is f(key) for all of a thread's.
template <typename Every> __device__ __forceinline__ uint64_t bound_by_halving(Halving& h, uint32_t k, uint32_t most, uint32_t vocab, Every every) {
  const uint32_t tid = threadIdx.x, nothing = order_of(-INFINITY);
  const uint64_t something = (uint64_t)(nothing + 1) << 32;
  uint32_t lowest = ~0u, highest = 0;
  every([&](uint64_t key) {
    if (key) lowest = min(lowest, (uint32_t)(key >> 32));
    highest = max(highest, (uint32_t)(key >> 32));
  });
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  highest = __reduce_max_sync(0xffffffffu, highest);
  if (tid % 32 == 0) { atomicMin(&h.lowest, lowest); atomicMax(&h.highest, highest); }
  __syncthreads();
  uint64_t low = (uint64_t)h.lowest << 32 | ~(vocab - 1), high = ((uint64_t)h.highest + 1) << 32;      // none reach high (an order is below 2^32 - 1)
  uint32_t slot = 0;
  auto reached = [&](uint64_t bound) {
    uint32_t reach = 0;
    every([&](uint64_t key) { reach += key >= bound; });
    reach = __reduce_add_sync(0xffffffffu, reach);
    if (tid % 32 == 0 && reach) atomicAdd(&h.counts[slot], reach);
    const uint32_t next = slot == 2 ? 0 : slot + 1;
    if (tid == 0) h.counts[next] = 0;      // those who read it are past the barrier before
    __syncthreads();
    const uint32_t all = h.counts[slot];
    slot = next;
    return all;
  };
  if (high - low >= 1ull << 58 || low < something) {
    for (uint64_t step = 1ull << 52;; step = step < 1ull << 62 ? step << 2 : ~0ull) {
      low = high - something > step ? high - step : something;
      const uint32_t all = reached(low);
      if (all >= k) {
        if (all <= most) return low;
        break;
      }
      if (low == something) return (uint64_t)nothing << 32;      // fewer than k are more than -inf
      high = low;
    }
  }
  while (high - low > 1) {
    const uint64_t middle = low + (high - low) / 2;
    const uint32_t all = reached(middle);
    if (all < k) { high = middle; continue; }
    low = max(middle, middle >> 32 << 32 | ~(vocab - 1));      // as many reach the last index's key
    if (all <= most) break;
  }
  return low;
}

// What a thread knows of its logits: the largest and the last index of the vector that it first came in (its own index before and behind the vectors), and the largest
// of its other vectors' largest.
struct Best {
  float top = -INFINITY, second = -INFINITY;
  uint32_t at;
  __device__ __forceinline__ void meet(float t, uint32_t index) {
    second = fmaxf(second, fminf(top, t));
    if (t > top) { top = t; at = index; }
  }
};

// sorted[0, k) of the slice's k best logits; sh.bound = 1, sh.n_cand = sh.n_hot = 0 and sh.halving reset behind a barrier.  Every thread brings the best of its own as a
// key, `mine`, 0 where it has none.  A bound that at least k of the threads' keys reach and few more: for small k the k-th largest of the keys of groups of threads,
// of twice k groups or more, else one found by halving (2000 rows of 65536 bf16, us, ranked groups | halving: 64 of them 75 | 68, 20 69 | 61, five 55 | 59).  So at
// least k logits of the slice reach it, and all of the k best are those threads': vectors do not overlap, so another thread's logit of the same value lies
// behind.  Such a thread looks at its best vector again, which is in `raw` or else is read again; where its second one reaches the bound, too, the CTA reads all of
// that thread's.  The logits that reach the bound are ranked, unless they are so many (rows of few vectors, ties, best logits that crowd into a few threads) that
// it is better raised first: eight rows of 1000, 128 of them, 148 -> 14 us.
template <typename T, int THREADS, bool MANY>
__device__ void best_of_slice(Shared<THREADS>& sh, const Slice<T>& sl, const Best& best, uint64_t mine, const uint4 (&raw)[kLoads], uint32_t k, uint32_t vocab) {
  constexpr int kVec = Vec<T>::kSize;
  const uint32_t tid = threadIdx.x;
  const uint32_t rounds = (sl.count + THREADS - 1) / THREADS, at0 = sl.at0();
  const uint32_t groups = k <= 4 ? 8 : 32, lanes = THREADS / groups;
  uint4 best_vector;      // asked for before it is known whether it is wanted: most of the time that takes is then over
  const bool vector = rounds > kLoads && best.at >= at0 && best.at < sl.tail_at;
  // the key of the first logit that `mine` may stand for: an index of a vector is its last one's
  const uint64_t reach = mine + (mine != 0 && best.at >= at0 && best.at < sl.tail_at ? kVec - 1 : 0);
  if (vector) best_vector = *reinterpret_cast<const uint4*>(sl.z + best.at - (kVec - 1));
  if constexpr (MANY) {
    if (min(max(max(sl.head, sl.tail), sl.count), (uint32_t)THREADS) >= k) {      // as many threads have a key
      const uint64_t bound = bound_by_halving(sh.halving, k, k + 8, vocab, [&](auto f) { f(mine); });
      if (tid == 0) sh.bound = bound;
    }
    __syncthreads();
  } else {
    uint64_t key = mine;
    for (uint32_t o = 1; o < min(lanes, 32u); o <<= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, key, o);
      key = other > key ? other : key;
    }
    const uint32_t held = max(groups, (uint32_t)THREADS / 32);      // a group is a warp at most
    if (tid % (THREADS / held) == 0) sh.groups[tid / (THREADS / held)] = key;
    __syncthreads();
    rank_keys<THREADS>(sh.groups, held, [&](uint32_t, uint64_t own, uint32_t above) {
      if (own != 0 && above == k - 1) sh.bound = own;      // no two of the others are equal
    });
    __syncthreads();
  }
  while (true) {      // once, but for rows whose best logits crowd into a few threads: the bound rises until what reaches it has room
    uint64_t bound = sh.bound;
    if (bound >> 32 == order_of(-INFINITY)) {      // -inf is wanted only where fewer than k are more: those that are lie before 2 k - 1 others
      uint32_t last = at0 - sl.head + 2 * k - 2;
      if (last >= at0) last += kVec - 1 - (last - at0) % kVec;
      if (last < sl.tail_at) bound = max(bound, key_of(-INFINITY, last));
    }
    const float bound_z = value_of((uint32_t)(bound >> 32));
    auto offer = [&](float z, uint32_t index) {
      if (z < bound_z) return;      // a NaN is not: it ranks with -inf
      const uint64_t c = key_of(z, index);
      if (c >= bound) {
        const uint32_t at = atomicAdd(&sh.n_cand, 1u);
        if (at < kCandidates) sh.cand[at] = c;
      }
    };
    auto offer_all = [&](const uint4& r, uint32_t at) {      // few reach it, in most vectors one
      float2 v[kVec / 2];
      Vec<T>::unpack(r, v);
      uint32_t reach = 0;
#pragma unroll
      for (int e = 0; e < kVec / 2; ++e) reach |= (v[e].x < bound_z ? 0u : 1u << (2 * e)) | (v[e].y < bound_z ? 0u : 2u << (2 * e));
      for (; reach; reach &= reach - 1) {
        const uint32_t e = __ffs(reach) - 1;
        offer(Vec<T>::at(r, e), at + e);
      }
    };
    if (reach >= bound) {
      if (tid < sl.head) offer(Elem<T>::to_f32(sl.z[tid]), tid);
      if (tid < sl.tail) offer(Elem<T>::to_f32(sl.z[sl.tail_at + tid]), sl.tail_at + tid);
      // a bound of -inf has the index of a thread's first vector: of other -inf only those of first vectors reach it
      const bool nothing = bound_z == -INFINITY, several = nothing ? best.second > -INFINITY : !(best.second < bound_z);
      if (rounds <= kLoads) {
#pragma unroll
        for (int l = 0; l < kLoads; ++l) {
          const uint32_t at = at0 + (tid + l * THREADS) * kVec;
          if (tid + l * THREADS < sl.count && (several || best.at == at + kVec - 1 || (nothing && l == 0))) offer_all(raw[l], at);
        }
      } else if (several) {
        sh.hot[atomicAdd(&sh.n_hot, 1u)] = (uint16_t)tid;
      } else {
        if (vector) offer_all(best_vector, best.at - (kVec - 1));
        const uint32_t first = at0 + tid * kVec;
        if (nothing && tid < sl.count && !(vector && best.at == first + kVec - 1)) offer_all(*reinterpret_cast<const uint4*>(sl.z + first), first);
      }
    }
    __syncthreads();
    if (sh.n_hot != 0) {
      const uint32_t bits = rounds >= 32 ? 5 : 32 - __clz(rounds - 1), lane = tid & ((1u << bits) - 1);      // a warp or a part of it for each
      for (uint32_t h = tid >> bits; h < sh.n_hot; h += THREADS >> bits)
        for (uint32_t vec = lane * THREADS + sh.hot[h]; vec < sl.count; vec += THREADS << bits) {
          const uint32_t at = at0 + vec * kVec;
          const uint4 r = *reinterpret_cast<const uint4*>(sl.z + at);
          if (!(Vec<T>::top(r) < bound_z)) offer_all(r, at);      // of nothing but NaN the top is one
        }
      __syncthreads();
    }
    const uint32_t n = sh.n_cand;
    if (n > kNarrow) {
      reset(sh.halving);
      __syncthreads();
      const uint64_t raised = bound_by_halving(sh.halving, k, k + 32, vocab, [&](auto f) {
        for (uint32_t i = tid; i < min(n, (uint32_t)kCandidates); i += THREADS) f(sh.cand[i]);
      });
      if (raised > bound) {      // fewer reach it: `most` of those looked at.  Else fewer than k are more than -inf, and there is room for as many of those as may be wanted
        if (tid == 0) { sh.bound = raised; sh.n_cand = 0; sh.n_hot = 0; }
        __syncthreads();
        continue;
      }
    }
    rank_keys<THREADS>(sh.cand, min(n, (uint32_t)kCandidates), [&](uint32_t, uint64_t key, uint32_t above) {
      if (above < k) sh.sorted[above] = key;
    });
    __syncthreads();
    break;
  }
}

// A CTA's shared memory may be written from the others of its cluster once it runs: every thread says so at its kernel's start, and waits for the others' word where
// they have long given it (none is late by more than the launch).  Between the two nothing is ordered, so the first is relaxed.
__device__ __forceinline__ void cluster_here() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_all_here() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

struct Forward {
  const void* logits;
  Rows rows;
  uint32_t vocab, n_tokens, top;
  const int64_t* tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  float2* stats;
};

// One row per cluster of CTAs (of one CTA where there are rows enough to fill the chip); its CTAs' terms and best logits meet in the first one, which the
// others write to: behind one barrier they are done (reading from the first CTA took two, and 1.2 us more for a single row).  That the first CTA runs
// they know from a barrier that is begun at the kernel's start and ended in front of the writes, a whole stream later.
// With alternatives a row is two phases, the stream (22000 cycles of a 128 KB row among three others on the SM) and the selection (half as many for 64 of them, a
// quarter for five), which other rows' streams hide in part: more, smaller CTAs are better until the selection is longer than they can hide.
// TOP: 0 for no alternatives, 1 for up to kHalve, 2 for more (in one kernel few of them took 1 to 3 % longer).
template <typename T, int THREADS, int TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(const Forward p) {
  grid_wait();
  __shared__ __align__(16) Shared<THREADS> sh;
  constexpr int kVec = Vec<T>::kSize, kWarps = THREADS / 32;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x;
  if (ctas > 1) cluster_here();
  const uint32_t row = ctas == 1 ? blockIdx.x : blockIdx.x / ctas;
  const T* z = static_cast<const T*>(p.logits) + p.rows.at(row);
  const Slice<T> sl(z, p.vocab, rank, ctas);
  const uint32_t at0 = sl.at0();
  const uint4* vecs = reinterpret_cast<const uint4*>(z + at0);

  // a given token's logit, asked for ahead of the row
  int64_t token = -1;
  float token_z = 0.0f;
  if (rank == 0 && tid < p.n_tokens) {
    token = p.tokens[(int64_t)row * p.n_tokens + tid];
    if (token >= 0) token_z = token < p.vocab ? Elem<T>::to_f32(z[token]) : NAN;
  }

  Terms t;
  Best best;
  best.at = tid < sl.head ? tid : tid < sl.count ? at0 + tid * kVec + kVec - 1 : sl.tail_at + tid;
  const bool any = tid < sl.head || tid < sl.count || tid < sl.tail;
  bool masked = false;      // this warp has met a logit that is no number
  if (tid < sl.head) {
    const float v = Elem<T>::to_f32(sl.z[tid]);
    if (v > t.m) t.m = v;
    best.meet(v, tid);
    t.add(v, t.base());
  }
  // Four vectors at a time; each is asked for while the ones before it are added up.
  uint4 raw[kLoads];
  const uint4* ahead = vecs + tid;      // of the next four, and how many vectors are left from there on
  int left = (int)(sl.count - tid);
#pragma unroll
  for (int l = 0; l < kLoads; ++l)
    if (l * THREADS < left) raw[l] = __ldg(ahead + l * THREADS);
  for (uint32_t j0 = 0; j0 < sl.count; j0 += kLoads * THREADS) {
    const uint32_t j = j0 + tid;
    const bool full = j0 + kLoads * THREADS <= sl.count;
    ahead += kLoads * THREADS;
    left -= kLoads * THREADS;
    float tops[kLoads];
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      tops[l] = full || j + l * THREADS < sl.count ? Vec<T>::top(raw[l]) : -INFINITY;
      if constexpr (TOP) best.meet(tops[l], at0 + (j + l * THREADS) * kVec + kVec - 1);
    }
    static_assert(kLoads == 4, "the largest of four");
    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (top > t.m) t.raise(top);
    const float from = t.base();
    float2 v[kVec / 2];
    if (full && !masked) {
      const float2 minus = make_float2(-from, -from), scale = make_float2(kLog2e, kLog2e);
      float2 sum = make_float2(t.s, 0.0f), weighted = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        Vec<T>::unpack(raw[l], v);
        if (l * THREADS < left) raw[l] = __ldg(ahead + l * THREADS);
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
          const float2 d = __fadd2_rn(v[i], minus), a = __fmul2_rn(d, scale), e = make_float2(exp2_fast(a.x), exp2_fast(a.y));
          sum = __fadd2_rn(sum, e);
          weighted = __ffma2_rn(e, d, weighted);
        }
      }
      t.s = sum.x + sum.y;
      float w = weighted.x + weighted.y;
      if (__any_sync(0xffffffffu, w != w)) {      // 0 * -inf: the warp goes on with differences that are kept finite, and adds these logits up once more
        masked = true;
        Terms again;
#pragma unroll 1
        for (int l = 0; l < kLoads; ++l) {
          Vec<T>::unpack(__ldg(vecs + j + l * THREADS), v);
#pragma unroll
          for (int i = 0; i < kVec / 2; ++i) { again.add(v[i].x, from); again.add(v[i].y, from); }
        }
        w = again.w;
      }
      t.w += w;
    } else {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const bool has = full || j + l * THREADS < sl.count;
        if (has) Vec<T>::unpack(raw[l], v);
        if (l * THREADS < left) raw[l] = __ldg(ahead + l * THREADS);
        if (has)
#pragma unroll
          for (int i = 0; i < kVec / 2; ++i) { t.add(v[i].x, from); t.add(v[i].y, from); }
      }
    }
  }
  if (tid < sl.tail) {
    const float v = Elem<T>::to_f32(sl.z[sl.tail_at + tid]);
    if (v > t.m) t.raise(v);
    best.meet(v, sl.tail_at + tid);
    t.add(v, t.base());
  }
  const uint64_t mine = any ? key_of(best.top, best.at) : 0;

  t.template over_lanes<32>();
  if ((tid & 31) == 0) sh.terms[tid >> 5] = t;
  if (TOP && tid == 0) { sh.bound = 1; sh.n_cand = 0; sh.n_hot = 0; }
  if (TOP) reset(sh.halving);
  __syncthreads();
  if (tid / 32 == kWarps - 1) {      // the last warp: the first ones have a bound to find
    const uint32_t lane = tid & 31;
    Terms r;
    if (lane < kWarps) r = sh.terms[lane];
    r.template over_lanes<kWarps>();
    if (lane == 0) sh.cta = r;
  }
  const uint32_t own = TOP ? min(p.top, sl.elements()) : 0;
  if (TOP && own) best_of_slice<T, THREADS, TOP == 2>(sh, sl, best, mine, raw, own, p.vocab);
  else __syncthreads();
  if (ctas > 1) {      // everyone hands what it has to the first CTA
    cluster_all_here();
    Shared<THREADS>* to = cluster.map_shared_rank(&sh, 0);
    if (TOP)
      for (uint32_t i = tid; i < p.top; i += THREADS) to->gathered[rank * p.top + i] = i < own ? sh.sorted[i] : 0;
    if (tid == 0) to->of_cta[rank] = sh.cta;
    cluster.sync();
    if (rank != 0) return;
    if (tid < 32) {
      Terms r;
      if (tid < ctas) r = sh.of_cta[tid];
      r.template over_lanes<kMaxCluster>();
      if (tid == 0) sh.cta = r;
    }
    if (TOP) {
      const uint64_t* all = sh.gathered;
      uint32_t n = ctas * p.top;
      if (n > kNarrow) {      // into cand, which is free again
        if (tid == 0) sh.n_cand = 0;
        reset(sh.halving);
        __syncthreads();
        uint64_t bound = bound_by_halving(sh.halving, p.top, p.top + 32, p.vocab, [&](auto f) {
          for (uint32_t i = tid; i < n; i += THREADS) f(sh.gathered[i]);
        });
        bound = max(bound, key_of(-INFINITY, 2 * p.top - 2));      // where fewer than k are more than -inf, those that are wanted lie before 2 k - 1 others
        for (uint32_t i = tid; i < n; i += THREADS)
          if (sh.gathered[i] >= bound) sh.cand[atomicAdd(&sh.n_cand, 1u)] = sh.gathered[i];
        __syncthreads();
        all = sh.cand;
        n = sh.n_cand;
      }
      rank_keys<THREADS>(all, n, [&](uint32_t, uint64_t key, uint32_t above) {
        if (above < p.top && key != 0) sh.sorted[above] = key;
      });
    }
    __syncthreads();
  }
  if (tid >= max(max(p.n_tokens, p.top), 1u)) return;
  const Sums r = sh.cta;
  const bool dead = r.s == 0.0f;      // nothing but -inf: every token's log probability is -inf
  const float log_s = dead ? INFINITY : logf(r.s), from = dead ? 0.0f : r.m;
  if (tid == 0) {
    if (p.entropy) p.entropy[row] = dead ? 0.0f : log_s - r.w / r.s;
    if (p.stats) p.stats[row] = make_float2(from, log_s);
  }
  if (tid < p.n_tokens) p.logprobs[(int64_t)row * p.n_tokens + tid] = token < 0 ? 0.0f : (token_z - from) - log_s;
  if (TOP && tid < p.top) {
    const uint64_t key = sh.sorted[tid];
    p.top_tokens[(int64_t)row * p.top + tid] = (int64_t)(uint32_t)~(uint32_t)key;
    p.top_logprobs[(int64_t)row * p.top + tid] = (value_of((uint32_t)(key >> 32)) - from) - log_s;
  }
}

constexpr float kNothing = -1000.0f;       // a log probability below it is a probability of 0, and times an entropy's cotangent of up to 2^117 it is finite

struct Backward {
  const void* logits;
  Rows rows;
  uint32_t vocab, n_tokens, top;
  const int64_t *tokens, *top_tokens;
  const float2* stats;
  const float *entropy, *g_logprobs, *g_entropy, *g_top;
  void* dlogits;
};

// sizeof(T) * kVec bytes of logits from an address that is a multiple of sizeof(T) only
template <typename T> __device__ __forceinline__ uint4 load_anywhere(const T* from) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(from);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
  const uint32_t a = __ldg(w), b = __ldg(w + 1), c = __ldg(w + 2), d = __ldg(w + 3);
  if ((at & 3) == 0) return make_uint4(a, b, c, d);
  const uint32_t e = __ldg(reinterpret_cast<const uint16_t*>(w + 4));      // the last one, and nothing behind it
  return make_uint4(__funnelshift_r(a, b, 16), __funnelshift_r(b, c, 16), __funnelshift_r(c, d, 16), __funnelshift_r(d, e, 16));
}

// Bound by HBM: 4096 x 65536 f32 in 333 us (6.45 TB/s, read and written); 1023 x 32003 bf16, rows of logits and of dz at different places of 16 bytes (a view that
// leaves every sequence's last position out), 26 us with five 4-byte loads for a vector, 80 with an element a load and store.
// A row's slice per CTA (gridDim.y slices of a row), in vectors of dz.  Few logits have a cotangent of their own: they are written again behind the slice's.
template <typename T>
__global__ void __launch_bounds__(kBackThreads) token_logprobs_bwd_kernel(const Backward p) {
  grid_wait();
  constexpr int kVec = Vec<T>::kSize;
  __shared__ int64_t at[kMaxTokens + kMaxTop];
  __shared__ float own[kMaxTokens + kMaxTop];
  __shared__ float total;
  const uint32_t tid = threadIdx.x;
  const uint32_t row = blockIdx.x;
  const T* z = static_cast<const T*>(p.logits) + p.rows.at(row);
  T* dz = static_cast<T*>(p.dlogits) + (int64_t)row * p.vocab;
  const uint32_t n = p.n_tokens + p.top;
  const float2 st = p.stats[row];
  const bool dead = st.y == INFINITY;
  const float g_entropy = p.g_entropy && !dead ? p.g_entropy[row] : 0.0f, entropy = p.g_entropy ? p.entropy[row] : 0.0f;
  for (uint32_t i = tid; i < n; i += kBackThreads) {
    const bool given = i < p.n_tokens;
    int64_t j = given ? p.tokens[(int64_t)row * p.n_tokens + i] : p.top_tokens[(int64_t)row * p.top + i - p.n_tokens];
    const float* g = given ? p.g_logprobs : p.g_top;
    const bool counts = j >= 0 && j < p.vocab && g != nullptr;
    at[i] = counts ? j : -1;
    own[i] = counts ? (given ? g[(int64_t)row * p.n_tokens + i] : g[(int64_t)row * p.top + i - p.n_tokens]) : 0.0f;
  }
  __syncthreads();
  if (tid < 32) {
    float sum = 0.0f;
    for (uint32_t i = tid; i < n; i += 32) sum += own[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (tid == 0) total = sum;
  }
  __syncthreads();
  // p_j (c - g_entropy log p_j), with everything that a row has one of in c.  A row without any logit has no gradient, whatever its cotangents.
  const float c = dead ? 0.0f : fmaf(-g_entropy, entropy, -total);
  const float2 minus_m = make_float2(-st.x, -st.x), minus_s = make_float2(-st.y, -st.y), scale = make_float2(kLog2e, kLog2e), minus_g = make_float2(-g_entropy, -g_entropy), c2 = make_float2(c, c);
  auto gradient = [&](const float2& v) {
    float2 x = __fadd2_rn(__fadd2_rn(v, minus_m), minus_s);
    x = make_float2(max_nan(x.x, kNothing), max_nan(x.y, kNothing));
    const float2 a = __fmul2_rn(x, scale);
    return __fmul2_rn(make_float2(exp2_fast(a.x), exp2_fast(a.y)), __ffma2_rn(minus_g, x, c2));
  };
  auto one = [&](uint32_t j) { return gradient(make_float2(Elem<T>::to_f32(z[j]), 0.0f)).x; };
  const Slice<T> sl(dz, p.vocab, blockIdx.y, gridDim.y);
  const uint32_t at0 = sl.at0(), lo = blockIdx.y == 0 ? 0 : at0, hi = at0 + sl.count * kVec + sl.tail;      // elements of this CTA
  const bool same = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
  if (tid < sl.head) dz[tid] = Elem<T>::from_f32(one(tid));
  if (tid < sl.tail) dz[sl.tail_at + tid] = Elem<T>::from_f32(one(sl.tail_at + tid));
  uint4* out = reinterpret_cast<uint4*>(dz + at0);
#pragma unroll 2
  for (uint32_t j = tid; j < sl.count; j += kBackThreads) {
    const uint4 r = same ? __ldg(reinterpret_cast<const uint4*>(z + at0) + j) : load_anywhere(z + at0 + j * kVec);
    float2 v[kVec / 2];
    Vec<T>::unpack(r, v);
#pragma unroll
    for (int e = 0; e < kVec / 2; ++e) v[e] = gradient(v[e]);
    out[j] = Vec<T>::pack(v);
  }
  if (n == 0 || dead) return;
  __syncthreads();
  for (uint32_t i = tid; i < n; i += kBackThreads) {
    const int64_t j = at[i];
    if (j < (int64_t)lo || j >= (int64_t)hi) continue;
    float g = 0.0f;
    bool first = true;
    for (uint32_t o = 0; o < n; ++o)
      if (at[o] == j) {
        first = first && o >= i;
        g += own[o];
      }
    if (first) dz[j] = Elem<T>::from_f32(one((uint32_t)j) + g);
  }
}

// CTAs that share a row: where rows alone do not fill the chip
int ctas_of_row(int64_t rows, int64_t bytes) {
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= 2 * (int64_t)sm_count() && bytes / (c * 2) >= 8192) c *= 2;
  return c;
}

template <typename T, int THREADS, int TOP> cudaError_t launch_forward(const Forward& p, int64_t rows, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(rows * ctas)); config.blockDim = dim3(THREADS); config.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = ctas; attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, token_logprobs_kernel<T, THREADS, TOP>, p);
}
template <typename T> cudaError_t forward_of(const Forward& p, int64_t rows, cudaStream_t st) {
  const int64_t bytes = (int64_t)p.vocab * sizeof(T);
  const int64_t sms = sm_count();
  int ctas = 1;
  while (ctas < kMaxCluster && rows * ctas * 2 <= sms && bytes / (ctas * 2) >= 32768) ctas *= 2;
  // us, 128 | 256 | 512 threads a row: 4096 rows of 16 KB 26 | 39 | 71 (five alternatives), 17.5 | 21.5 | 38 (none), 122 | 89 | 144 (128), of 8 KB 41 | 57 | 117 (64);
  // 2000 rows of 128 KB 55 | 56 | 67 (five), 50 | 48 | 52 (none), 88 | 68 | 85 (64); 148 rows of 256 KB 20.2 | 18.2 | 13.5 (20); one such row over eight CTAs 6.6 | 5.7 | 6.1
  int threads;
  if (rows * ctas <= sms) threads = bytes / ctas > 32768 ? 512 : bytes / ctas > 8192 || p.top > 64 ? 256 : 128;
  else threads = p.top <= 64 && (bytes <= 32768 || (bytes <= 131072 && p.top > 0 && p.top <= 32)) ? 128 : 256;
  if (int v = env_switch("PB_LP_CTAS", 0)) ctas = v;
  if (int v = env_switch("PB_LP_WIDE", 0)) threads = v;
  if (threads == 128) return p.top > kHalve ? launch_forward<T, 128, 2>(p, rows, ctas, st) : p.top ? launch_forward<T, 128, 1>(p, rows, ctas, st) : launch_forward<T, 128, 0>(p, rows, ctas, st);
  if (threads == 512) return p.top > kHalve ? launch_forward<T, 512, 2>(p, rows, ctas, st) : p.top ? launch_forward<T, 512, 1>(p, rows, ctas, st) : launch_forward<T, 512, 0>(p, rows, ctas, st);
  return p.top > kHalve ? launch_forward<T, 256, 2>(p, rows, ctas, st) : p.top ? launch_forward<T, 256, 1>(p, rows, ctas, st) : launch_forward<T, 256, 0>(p, rows, ctas, st);
}

int check_rows(const char* who, const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer, int64_t stride_inner, int64_t vocab,
               const int64_t* tokens, int n_tokens, int top) {
  if (dtype != PB_F32 && dtype != PB_BF16) return fail(PB_ERR_BAD_DTYPE, "%s: dtype %d", who, dtype);
  if (outer < 0 || inner < 0 || vocab <= 0 || vocab > 0x7fffffffll || stride_outer < 0 || stride_inner < 0)
    return fail(PB_ERR_BAD_SHAPE, "%s: outer=%lld inner=%lld vocab=%lld strides %lld, %lld", who, (long long)outer, (long long)inner, (long long)vocab, (long long)stride_outer, (long long)stride_inner);
  if (n_tokens < 0 || n_tokens > kMaxTokens || top < 0 || top > kMaxTop || top > vocab)
    return fail(PB_ERR_BAD_SHAPE, "%s: %d tokens and %d alternatives of %lld (at most %d and %d)", who, n_tokens, top, (long long)vocab, kMaxTokens, kMaxTop);
  if (inner > 0 && outer > 0x7fffffffll / kMaxCluster / inner) return fail(PB_ERR_BAD_SHAPE, "%s: too many rows (%lld x %lld)", who, (long long)outer, (long long)inner);
  if (outer * inner > 0 && (!logits || (n_tokens && !tokens))) return fail(PB_ERR_NULL_POINTER, "%s: null argument", who);
  if (off_by(logits, dtype == PB_F32 ? 4 : 2) || off_by(tokens, 8)) return fail(PB_ERR_MISALIGNED, "%s: logits and tokens lie at their types' bytes", who);
  return PB_OK;
}

}  // namespace
}  // namespace pb

using namespace pb;

extern "C" int pb_token_logprobs(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer, int64_t stride_inner, int64_t vocab,
                                 const int64_t* tokens, int n_tokens, int top, float* logprobs, float* entropy, float* top_logprobs, int64_t* top_tokens,
                                 float* stats, void* stream) {
  if (int s = check_rows("pb_token_logprobs", logits, dtype, outer, inner, stride_outer, stride_inner, vocab, tokens, n_tokens, top)) return s;
  const int64_t rows = outer * inner;
  if (rows == 0) return PB_OK;
  if ((n_tokens && !logprobs) || (top && (!top_logprobs || !top_tokens))) return fail(PB_ERR_NULL_POINTER, "pb_token_logprobs: null argument");
  if (off_by(stats, 8) || off_by(top_tokens, 8) || off_by(logprobs, 4) || off_by(entropy, 4) || off_by(top_logprobs, 4))
    return fail(PB_ERR_MISALIGNED, "pb_token_logprobs: stats 8 bytes, the others their types");
  const Forward p{logits, {FastDiv((uint32_t)inner), stride_outer, stride_inner}, (uint32_t)vocab, (uint32_t)n_tokens, (uint32_t)top, tokens, logprobs, entropy, top_logprobs, top_tokens,
                  reinterpret_cast<float2*>(stats)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_F32) forward_of<float>(p, rows, st);
  else forward_of<__nv_bfloat16>(p, rows, st);
  PB_LAUNCH_CHECK("token_logprobs_kernel");
  return PB_OK;
}

extern "C" int pb_token_logprobs_bwd(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer, int64_t stride_inner, int64_t vocab,
                                     const int64_t* tokens, int n_tokens, const int64_t* top_tokens, int top, const float* stats, const float* entropy,
                                     const float* g_logprobs, const float* g_entropy, const float* g_top, void* dlogits, void* stream) {
  if (int s = check_rows("pb_token_logprobs_bwd", logits, dtype, outer, inner, stride_outer, stride_inner, vocab, tokens, n_tokens, top)) return s;
  const int64_t rows = outer * inner;
  if (rows == 0) return PB_OK;
  if (!stats || !dlogits || (top && !top_tokens) || (g_entropy && !entropy)) return fail(PB_ERR_NULL_POINTER, "pb_token_logprobs_bwd: null argument");
  if (off_by(stats, 8) || off_by(dlogits, 16) || off_by(top_tokens, 8) || off_by(entropy, 4) || off_by(g_logprobs, 4) || off_by(g_entropy, 4) || off_by(g_top, 4))
    return fail(PB_ERR_MISALIGNED, "pb_token_logprobs_bwd: stats 8 and dlogits 16 bytes, the others their types");
  const Backward p{logits, {FastDiv((uint32_t)inner), stride_outer, stride_inner}, (uint32_t)vocab, (uint32_t)n_tokens, (uint32_t)top, tokens, top_tokens,
                   reinterpret_cast<const float2*>(stats), entropy, g_logprobs, g_entropy, g_top, dlogits};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)rows, (unsigned)ctas_of_row(rows, vocab * (dtype == PB_F32 ? 4 : 2)));
  if (dtype == PB_F32) launch_behind(token_logprobs_bwd_kernel<float>, grid, kBackThreads, 0, st, p);
  else launch_behind(token_logprobs_bwd_kernel<__nv_bfloat16>, grid, kBackThreads, 0, st, p);
  PB_LAUNCH_CHECK("token_logprobs_bwd_kernel");
  return PB_OK;
}
