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
// Bound by HBM: the forward pass reads the logits once (4 or 2 bytes each), the backward pass once more and writes dz.
#include "common.cuh"

#include <cooperative_groups.h>

namespace pb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kLoads = 4;                  // 16-byte loads that a thread has in flight
constexpr int kMaxTop = 128, kMaxTokens = 128;
constexpr int kCandidates = 1024;          // keys of a row that are ranked against one another
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

// 16 bytes of logits as numbers
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kSize = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kSize = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};
template <int N> __device__ __forceinline__ float top_of(const float (&v)[N]) {
  float t = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) t = fmaxf(t, v[i]);
  return t;
}

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
  __device__ __forceinline__ void join(const Terms& o) {      // o's maximum and this one's may be -inf: sums of zero then
    const float top = fmaxf(m, o.m), from = top == -INFINITY ? 0.0f : top;
    const float a = max_nan(m - from, kFar), b = max_nan(o.m - from, kFar);
    const float ca = exp2_fast(a * kLog2e), cb = exp2_fast(b * kLog2e);
    w = ca * (w + s * a) + cb * (o.w + o.s * b);
    s = ca * s + cb * o.s;
    m = top;
  }
  template <int LANES> __device__ __forceinline__ void over_lanes() {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      Terms t;
      t.m = __shfl_xor_sync(0xffffffffu, m, o); t.s = __shfl_xor_sync(0xffffffffu, s, o); t.w = __shfl_xor_sync(0xffffffffu, w, o);
      join(t);
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

struct Rows {
  int64_t inner, stride_outer, stride_inner;      // row r at (r / inner) * stride_outer + (r % inner) * stride_inner
  __device__ __forceinline__ int64_t at(int64_t r) const { return (r / inner) * stride_outer + (r % inner) * stride_inner; }
};

// A row as elements up to the first 16-byte boundary, whole 16-byte vectors and the rest; CTA `rank` of `ctas` has every vector of its slice, the
// first CTA also the elements before and the last one those behind.
template <typename T> struct Slice {
  static constexpr int kVec = Vec<T>::kSize;
  const T* z;
  uint32_t head, tail, tail_at, first, count;      // count vectors from vector `first` on
  __device__ __forceinline__ Slice(const T* row, uint32_t vocab, uint32_t rank, uint32_t ctas) : z(row) {
    head = min((uint32_t)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (uint32_t)sizeof(T), vocab);
    const uint32_t vecs = (vocab - head) / kVec, per = (vecs + ctas - 1) / ctas;
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

struct Shared {
  uint64_t cand[kCandidates];
  uint64_t lists[kThreads];             // the threads' best keys, 32 of a warp in order
  uint64_t sorted[kMaxTop];
  Sums terms[kWarps], cta;
  uint64_t threshold;
  uint32_t n_cand, n_hot;
  uint16_t hot[kThreads];
};

// The keys in[0, n) that are among the k largest, in order
__device__ __forceinline__ void rank_keys(const uint64_t* in, uint32_t n, uint32_t k, uint64_t* out) {
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t key = in[i];
    uint32_t above = 0;
    for (uint32_t j = 0; j < n; ++j) above += in[j] > key;
    if (above < k) out[above] = key;
  }
}

// sorted[0, k) of the slice's k best logits.  Every thread brings the best of its own: `mine` is that logit's value with the last index of the vector
// that it first came in.  Of these keys, the k-th largest is a bound that at least k logits of the slice reach, and they all belong to
// the k threads whose keys reach it: vectors do not overlap, so another thread's logit of the same value lies behind.  Those threads' logits
// (k / 256 of the slice) are read again, from L2, and the ones that reach the bound are ranked.
template <typename T>
__device__ void best_of_slice(Shared& sh, const Slice<T>& sl, uint64_t mine, uint32_t k) {
  constexpr int kVec = Vec<T>::kSize;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // 32 keys of a warp in falling order
  uint64_t key = mine;
#pragma unroll
  for (uint32_t size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (uint32_t step = size >> 1; step > 0; step >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, key, step);
      const bool larger = ((lane & step) == 0) == ((lane & size) == 0);      // of the two, whether this lane takes the larger
      key = (key > other) == larger ? key : other;
    }
  sh.lists[tid] = key;
  if (tid == 0) { sh.threshold = 1; sh.n_hot = 0; }
  __syncthreads();
  if (key != 0) {      // no two of the others are equal
    uint32_t above = lane;
    for (uint32_t l = 1; l < kWarps; ++l) {
      const uint64_t* list = sh.lists + ((warp + l) % kWarps) * 32;
      uint32_t at = 0;
#pragma unroll
      for (uint32_t step = 16; step > 0; step >>= 1)
        if (list[at + step - 1] > key) at += step;
      above += at + (list[at] > key);
    }
    if (above == k - 1) sh.threshold = key;
  }
  __syncthreads();
  const uint32_t rounds = (sl.count + kThreads - 1) / kThreads;
  while (true) {      // once, but for rows whose best logits crowd into a few threads: the bound rises until what reaches it has room
    const uint64_t bound = sh.threshold;
    if (tid == 0) sh.n_cand = 0;
    __syncthreads();
    auto offer = [&](float z, uint32_t index) {
      const uint64_t c = key_of(z, index);
      if (c >= bound) {
        const uint32_t at = atomicAdd(&sh.n_cand, 1u);
        if (at < kCandidates) sh.cand[at] = c;
      }
    };
    if (mine >= bound) {
      sh.hot[atomicAdd(&sh.n_hot, 1u)] = (uint16_t)tid;
      if (tid < sl.head) offer(Elem<T>::to_f32(sl.z[tid]), tid);
      if (tid < sl.tail) offer(Elem<T>::to_f32(sl.z[sl.tail_at + tid]), sl.tail_at + tid);
    }
    __syncthreads();
    const uint32_t items = sh.n_hot * rounds;
    const uint32_t at0 = sl.at0();
    for (uint32_t i = tid; i < items; i += kThreads) {
      const uint32_t h = i / rounds, vec = (i - h * rounds) * kThreads + sh.hot[h];
      if (vec < sl.count) {
        const uint32_t at = at0 + vec * kVec;
        float v[kVec];
        Vec<T>::unpack(*reinterpret_cast<const uint4*>(sl.z + at), v);
#pragma unroll
        for (int e = 0; e < kVec; ++e) offer(v[e], at + e);
      }
    }
    __syncthreads();
    const uint32_t n = sh.n_cand, kept = min(n, (uint32_t)kCandidates);
    rank_keys(sh.cand, kept, k, sh.sorted);
    __syncthreads();
    if (n <= kCandidates) break;
    if (tid == 0) { sh.threshold = sh.sorted[k - 1]; sh.n_hot = 0; }
    __syncthreads();
  }
}

struct Forward {
  const void* logits;
  Rows rows;
  uint32_t vocab, n_tokens, top;
  const int64_t* tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  float2* stats;
};

// One row per cluster of CTAs (of one CTA where there are rows enough to fill the chip); its CTAs' terms and best logits meet in the first one.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const Forward p) {
  grid_wait();
  __shared__ Shared sh;
  constexpr int kVec = Vec<T>::kSize;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x;
  const int64_t row = blockIdx.x / ctas;
  const T* z = static_cast<const T*>(p.logits) + p.rows.at(row);
  const Slice<T> sl(z, p.vocab, rank, ctas);
  const uint4* vecs = reinterpret_cast<const uint4*>(z + sl.at0());

  // a given token's logit, asked for ahead of the row
  int64_t token = -1;
  float token_z = 0.0f;
  if (rank == 0 && tid < p.n_tokens) {
    token = p.tokens[row * p.n_tokens + tid];
    if (token >= 0) token_z = token < p.vocab ? Elem<T>::to_f32(z[token]) : NAN;
  }

  Terms t;
  const uint32_t at0 = sl.at0();
  // where the thread's best logit is: the last index of its vector
  uint32_t best = tid < sl.head ? tid : tid < sl.count ? at0 + tid * kVec + kVec - 1 : sl.tail_at + tid;
  const bool any = tid < sl.head || tid < sl.count || tid < sl.tail;
  if (tid < sl.head) {
    const float v = Elem<T>::to_f32(sl.z[tid]);
    if (v > t.m) t.m = v;
    t.add(v, t.base());
  }
  uint32_t j = tid;
  for (; j + (kLoads - 1) * kThreads < sl.count; j += kLoads * kThreads) {
    uint4 raw[kLoads];
#pragma unroll
    for (int l = 0; l < kLoads; ++l) raw[l] = __ldg(vecs + j + l * kThreads);
    float tops[kLoads];
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      float v[kVec];
      Vec<T>::unpack(raw[l], v);
      tops[l] = top_of(v);
    }
    const float top = top_of(tops);
    if (top > t.m) {
      t.raise(top);
      if constexpr (TOP) {
        uint32_t l = kLoads - 1;
#pragma unroll
        for (int i = kLoads - 2; i >= 0; --i) l = tops[i] == top ? i : l;
        best = at0 + (j + l * kThreads) * kVec + kVec - 1;
      }
    }
    const float from = t.base();
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      float v[kVec];
      Vec<T>::unpack(raw[l], v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) t.add(v[e], from);
    }
  }
  for (; j < sl.count; j += kThreads) {
    float v[kVec];
    Vec<T>::unpack(__ldg(vecs + j), v);
    const float top = top_of(v);
    if (top > t.m) {
      t.raise(top);
      best = at0 + j * kVec + kVec - 1;
    }
    const float from = t.base();
#pragma unroll
    for (int e = 0; e < kVec; ++e) t.add(v[e], from);
  }
  if (tid < sl.tail) {
    const float v = Elem<T>::to_f32(sl.z[sl.tail_at + tid]);
    if (v > t.m) {
      t.raise(v);
      best = sl.tail_at + tid;
    }
    t.add(v, t.base());
  }
  const uint64_t mine = any ? key_of(t.m, best) : 0;

  t.over_lanes<32>();
  if ((tid & 31) == 0) sh.terms[tid >> 5] = t;
  __syncthreads();
  if (tid < 32) {
    Terms r;
    if (tid < kWarps) r = sh.terms[tid];
    r.over_lanes<kWarps>();
    if (tid == 0) sh.cta = r;
  }
  const uint32_t own = TOP ? min(p.top, sl.elements()) : 0;
  if (TOP && own) best_of_slice(sh, sl, mine, own);
  __syncthreads();
  if (ctas > 1) {
    cluster.sync();
    if (rank == 0) {
      if (tid < 32) {
        Terms r;
        if (tid < ctas) r = cluster.map_shared_rank(&sh, tid)->cta;
        r.over_lanes<kMaxCluster>();
        __syncwarp();
        if (tid == 0) sh.cta = r;      // every lane has read its CTA's, this one's among them
      }
      if (TOP) {
        uint32_t n = 0;
        for (uint32_t r = 0; r < ctas; ++r) {
          const uint32_t of = min(p.top, Slice<T>(z, p.vocab, r, ctas).elements());
          if (tid < of) sh.cand[n + tid] = cluster.map_shared_rank(&sh, r)->sorted[tid];
          n += of;
        }
        __syncthreads();
        rank_keys(sh.cand, n, p.top, sh.sorted);
      }
    }
    cluster.sync();      // nobody leaves while its memory is read
    if (rank != 0) return;
  }
  const Sums r = sh.cta;
  const bool dead = r.s == 0.0f;      // nothing but -inf: every token's log probability is -inf
  const float log_s = dead ? INFINITY : logf(r.s), from = dead ? 0.0f : r.m;
  if (tid == 0) {
    if (p.entropy) p.entropy[row] = dead ? 0.0f : log_s - r.w / r.s;
    if (p.stats) p.stats[row] = make_float2(from, log_s);
  }
  if (tid < p.n_tokens) p.logprobs[row * p.n_tokens + tid] = token < 0 ? 0.0f : (token_z - from) - log_s;
  if (TOP && tid < p.top) {
    const uint64_t key = sh.sorted[tid];
    p.top_tokens[row * p.top + tid] = (int64_t)(uint32_t)~(uint32_t)key;
    p.top_logprobs[row * p.top + tid] = (value_of((uint32_t)(key >> 32)) - from) - log_s;
  }
}

struct Backward {
  const void* logits;
  Rows rows;
  uint32_t vocab, n_tokens, top;
  const int64_t *tokens, *top_tokens;
  const float2* stats;
  const float *entropy, *g_logprobs, *g_entropy, *g_top;
  void* dlogits;
};

// A row's slice per CTA (gridDim.y slices of a row).  Few logits have a cotangent of their own: they are written again behind the slice's.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(const Backward p) {
  grid_wait();
  constexpr int kVec = Vec<T>::kSize;
  __shared__ int64_t at[kMaxTokens + kMaxTop];
  __shared__ float own[kMaxTokens + kMaxTop];
  __shared__ float total;
  const uint32_t tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(p.logits) + p.rows.at(row);
  T* dz = static_cast<T*>(p.dlogits) + row * p.vocab;
  const uint32_t n = p.n_tokens + p.top;
  const float2 st = p.stats[row];
  const float g_entropy = p.g_entropy ? p.g_entropy[row] : 0.0f, entropy = p.g_entropy ? p.entropy[row] : 0.0f;
  for (uint32_t i = tid; i < n; i += kThreads) {
    const bool given = i < p.n_tokens;
    int64_t j = given ? p.tokens[row * p.n_tokens + i] : p.top_tokens[row * p.top + i - p.n_tokens];
    const float* g = given ? p.g_logprobs : p.g_top;
    const bool counts = j >= 0 && j < p.vocab && g != nullptr;
    at[i] = counts ? j : -1;
    own[i] = counts ? (given ? g[row * p.n_tokens + i] : g[row * p.top + i - p.n_tokens]) : 0.0f;
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
  const float all = total;
  auto gradient = [&](float v) {
    const float x = max_nan((v - st.x) - st.y, kFar), pr = exp2_fast(x * kLog2e);
    return -pr * (all + g_entropy * (x + entropy));
  };
  uint32_t lo, hi;      // elements of this CTA
  if (((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0) {
    const Slice<T> sl(z, p.vocab, blockIdx.y, gridDim.y);
    const uint32_t at0 = sl.at0();
    lo = blockIdx.y == 0 ? 0 : at0;
    hi = at0 + sl.count * kVec + sl.tail;
    if (tid < sl.head) dz[tid] = Elem<T>::from_f32(gradient(Elem<T>::to_f32(z[tid])));
    if (tid < sl.tail) dz[sl.tail_at + tid] = Elem<T>::from_f32(gradient(Elem<T>::to_f32(z[sl.tail_at + tid])));
    const uint4* in = reinterpret_cast<const uint4*>(z + at0);
    uint4* out = reinterpret_cast<uint4*>(dz + at0);
    for (uint32_t j = tid; j < sl.count; j += kThreads) {
      float v[kVec];
      Vec<T>::unpack(__ldg(in + j), v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = gradient(v[e]);
      out[j] = Vec<T>::pack(v);
    }
  } else {      // rows of logits and of dz that start at other places of 16 bytes
    const uint32_t per = (p.vocab + gridDim.y - 1) / gridDim.y;
    lo = min(blockIdx.y * per, p.vocab);
    hi = min(lo + per, p.vocab);
    for (uint32_t j = lo + tid; j < hi; j += kThreads) dz[j] = Elem<T>::from_f32(gradient(Elem<T>::to_f32(z[j])));
  }
  if (n == 0 || st.y == INFINITY) return;      // a row without any logit has no gradient
  __syncthreads();
  for (uint32_t i = tid; i < n; i += kThreads) {
    const int64_t j = at[i];
    if (j < (int64_t)lo || j >= (int64_t)hi) continue;
    float g = 0.0f;
    bool first = true;
    for (uint32_t o = 0; o < n; ++o)
      if (at[o] == j) {
        first = first && o >= i;
        g += own[o];
      }
    if (first) dz[j] = Elem<T>::from_f32(gradient(Elem<T>::to_f32(z[j])) + g);
  }
}

// CTAs that share a row: where rows alone do not fill the chip
int ctas_of_row(int64_t rows, int64_t bytes) {
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= 2 * (int64_t)sm_count() && bytes / (c * 2) >= 8192) c *= 2;
  return c;
}

template <typename T, bool TOP> cudaError_t launch_forward(const Forward& p, int64_t rows, cudaStream_t st) {
  const int ctas = ctas_of_row(rows, (int64_t)p.vocab * sizeof(T));
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(rows * ctas)); config.blockDim = dim3(kThreads); config.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = ctas; attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, token_logprobs_kernel<T, TOP>, p);
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
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == PB_F32 ? 4 : 2)) return fail(PB_ERR_MISALIGNED, "%s: logits are not aligned to their type", who);
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
  if (reinterpret_cast<uintptr_t>(stats) & 7) return fail(PB_ERR_MISALIGNED, "pb_token_logprobs: stats must be 8-byte aligned");
  const Forward p{logits, {inner, stride_outer, stride_inner}, (uint32_t)vocab, (uint32_t)n_tokens, (uint32_t)top, tokens, logprobs, entropy, top_logprobs, top_tokens,
                  reinterpret_cast<float2*>(stats)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_F32) top ? launch_forward<float, true>(p, rows, st) : launch_forward<float, false>(p, rows, st);
  else top ? launch_forward<__nv_bfloat16, true>(p, rows, st) : launch_forward<__nv_bfloat16, false>(p, rows, st);
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
  if ((reinterpret_cast<uintptr_t>(stats) & 7) || (reinterpret_cast<uintptr_t>(dlogits) & 15)) return fail(PB_ERR_MISALIGNED, "pb_token_logprobs_bwd: stats 8 and dlogits 16 bytes");
  const Backward p{logits, {inner, stride_outer, stride_inner}, (uint32_t)vocab, (uint32_t)n_tokens, (uint32_t)top, tokens, top_tokens,
                   reinterpret_cast<const float2*>(stats), entropy, g_logprobs, g_entropy, g_top, dlogits};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)rows, (unsigned)ctas_of_row(rows, vocab * (dtype == PB_F32 ? 4 : 2)));
  if (dtype == PB_F32) launch_behind(token_logprobs_bwd_kernel<float>, grid, kThreads, 0, st, p);
  else launch_behind(token_logprobs_bwd_kernel<__nv_bfloat16>, grid, kThreads, 0, st, p);
  PB_LAUNCH_CHECK("token_logprobs_bwd_kernel");
  return PB_OK;
}
