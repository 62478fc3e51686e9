// Log probabilities of given tokens with the entropy of each row and its top alternatives,
// and the gradient of all three, over (vocab-padded) logits.
//
// Row m with logits z[0..V), temperature τ, target y:
//   l_j = z_j / τ - log Σ exp(z / τ);  logp = l_y;  H = -Σ p_j l_j  (p = e^l);
//   the k largest z by value, the lowest id first among equals, and their l.
//   dz_j = (1 / τ) (g_y [j = y] + Σ_i g_i [j = id_i] - (g_y + Σ_i g_i) p_j - g_H p_j (l_j + H))
// A row counts nothing where its target is outside [0, V) (ignore_index among them; its logits
// are not read) or where no logit is above -inf: zeros, ids -1, a gradient of 0.  NaN or +inf
// make the row's numbers NaN (NaN is the largest value for the top alternatives).
//
// Forward: one pass over a row with a running maximum m and S = Σ 2^t, A = Σ t 2^t,
// t = (z - m) log2(e) / τ; H = ln2 (log2 S - A / S).  Where m rises by d powers of two,
// A' = (A - d S) 2^-d, S' = S 2^-d.  The top alternatives cost that pass the maximum of every
// chunk of columns (8 of them, or a warp's tile where the row is long): the k best of the row
// lie in the k chunks with the best maxima, so the k-th best of those is a bound, and only
// chunks above it are looked at again.
// Backward: one pass, p from the row's m, S and H; the columns with a g term are written a
// second time by their block (each sum rounded once; no atomics).
//
// What bounds it: memory, next to 16 exponentials a cycle and SM.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>

#include <type_traits>

#include "rows.cuh"

namespace zq {

constexpr int kLpMaxTop = 256;
constexpr int kLpCandidates = 1024;      // of the list in shared memory, besides k ties
constexpr int kLpFine = 65536;           // rows of at most this many columns: chunks of 8
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpLn2 = 0.6931471805599453f;

struct LogprobParams {
  const void* z;
  const int64_t* targets;   // [M] or null: every row counts, no logp
  float *logp, *entropy;    // [M]
  float* top;               // [M, K]
  int64_t* ids;             // [M, K]
  float* stats;             // [M, 3]: m, log2 S, H of counted rows; log2 S = inf of the others
  const float *gp, *gh, *gt;   // gradients, or null
  void* dz;
  int64_t M, stride, gstride, width, V;
  int K, chunks;            // chunks of a row at most
  float scale;              // log2(e) / τ
  double tau;
};

__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// t of a logit: exact difference first, so nothing overflows that is finite in the end, and a
// bound from below, under which 2^t is 0 (t 2^t would be 0 · -inf).  NaN stays.
__device__ __forceinline__ float lp_t(float z, float m, float scale) { return max_nan((z - m) * scale, -1000.0f); }

// 16 bytes of a row
template <typename T>
struct LpVec {
  static constexpr int N = 16 / (int)sizeof(T);
  uint4 u;
  __device__ __forceinline__ void values(float (&v)[N]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 f;
        if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else f = bf16x2_to_f2(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(v[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      }
    }
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// A row's vectors start at the 16-byte boundary at or before its first element: vector i
// holds columns [i N - lead, i N - lead + N); those outside [0, V) are -inf.
template <typename T>
struct LpRow {
  static constexpr int N = LpVec<T>::N;
  const T* z;
  int lead;
  int64_t V, vecs;
  __device__ __forceinline__ LpRow(const void* base, int64_t row, int64_t stride, int64_t V_) : V(V_) {
    z = reinterpret_cast<const T*>(base) + row * stride;
    lead = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
    vecs = (lead + V + N - 1) / N;
  }
  __device__ __forceinline__ int64_t col(int64_t i) const { return i * N - lead; }
  __device__ __forceinline__ bool whole(int64_t i) const { return col(i) >= 0 && col(i) + N <= V; }
  __device__ __forceinline__ LpVec<T> load(int64_t i) const {
    LpVec<T> r;
    if (whole(i)) {
      r.u = __ldg(reinterpret_cast<const uint4*>(z + col(i)));
    } else {
      float v[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int64_t c = col(i) + j;
        v[j] = c >= 0 && c < V ? to_f32<T>(z[c]) : -INFINITY;
      }
      r.set(v);
    }
    return r;
  }
};

struct LpSums {
  float m, s, a;
};

// the sums when the maximum goes to `to` (above m)
__device__ __forceinline__ void lp_raise(LpSums& x, float to, float scale) {
  if (x.m == -INFINITY) {   // nothing yet
    x.m = to;
    return;
  }
  const float d = lp_t(x.m, to, scale);   // <= 0
  const float f = lp_exp2(d);
  x.a = f * fmaf(d, x.s, x.a);
  x.s *= f;
  x.m = to;
}

__device__ __forceinline__ LpSums lp_join(LpSums a, LpSums b, float scale) {
  // (a NaN is in the sums of its lane; maxima that are NaN there are not compared)
  const float to = fmaxf(a.m, b.m);
  if (to > a.m) lp_raise(a, to, scale);
  if (to > b.m) lp_raise(b, to, scale);
  a.s += b.s;
  a.a += b.a;
  return a;
}

__device__ __forceinline__ LpSums lp_warp_join(LpSums x, float scale) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpSums y;
    y.m = __shfl_xor_sync(0xffffffffu, x.m, o);
    y.s = __shfl_xor_sync(0xffffffffu, x.s, o);
    y.a = __shfl_xor_sync(0xffffffffu, x.a, o);
    x = lp_join(x, y, scale);
  }
  return x;
}

// (z - m) / τ - log S, in 64 bits for a row's few numbers
__device__ __forceinline__ float lp_log(float z, float m, double tau, double log_s) {
  return (float)(((double)z - (double)m) / tau - log_s);
}

// Whole numbers in the values' order (0 and -0 equal, NaN above all), without the places that
// are the same for all values of the type.
template <typename T>
struct LpKey {
  static constexpr int kLow = std::is_same<T, __nv_bfloat16>::value ? 16 : std::is_same<T, __half>::value ? 13 : 0;
  static constexpr int kBits = 32 - kLow;
  static __device__ __forceinline__ uint32_t of(float v) {
    if (v != v) return 0xffffffffu >> kLow;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u ? ~b : b | 0x80000000u) >> kLow;
  }
};

template <int NT>
__device__ __forceinline__ uint32_t lp_block_sum(uint32_t v, uint32_t* s_n, int turn) {
  // s_n[3]: the word of two turns ahead is cleared while this one's is in use
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) atomicAdd(&s_n[turn % 3], v);
  __syncthreads();
  if (threadIdx.x == 0) s_n[(turn + 2) % 3] = 0u;
  return s_n[turn % 3];
}

// The top alternatives of a row, by the block that has all chunks' maxima.
template <typename T, int NT, bool FINE>
__device__ void lp_top(const LogprobParams& p, const LpRow<T>& row, int64_t m, const float* s_max, int chunks, float high,
                       double log_s, bool nan, uint32_t* s_n, uint64_t* s_list, uint32_t* s_count) {
  constexpr int N = LpVec<T>::N, kVecs = FINE ? 1 : 32;   // vectors of a chunk
  using Key = LpKey<T>;
  const int tid = threadIdx.x, lane = tid & 31;
  const uint32_t K = (uint32_t)p.K;
  if (tid < 3) s_n[tid] = 0u;
  if (tid == 0) *s_count = 0u;
  __syncthreads();
  int turn = 0;
  // the K-th best of the chunks' maxima (0, below all, where there are fewer chunks)
  uint32_t bound = 0;
  if (chunks >= p.K) {
#pragma unroll 1
    for (int bit = Key::kBits - 1; bit >= 0; --bit) {
      const uint32_t up = bound | (1u << bit);
      uint32_t n = 0;
      for (int i = tid; i < chunks; i += NT) n += Key::of(s_max[i]) >= up ? 1u : 0u;
      if (lp_block_sum<NT>(n, s_n, turn++) >= K) bound = up;
    }
  }
  // Elements above the bound, in any order (they are ranked below).  Where they do not fit the
  // list (a row whose best lie side by side), the bound rises to the K-th best element.
  auto each = [&](uint32_t at_least, auto&& f) {   // elements of chunks whose maximum reaches it
    for (int c = tid / kVecs; c < chunks; c += NT / kVecs) {
      if (Key::of(s_max[c]) < at_least) continue;
      const int64_t i = (int64_t)c * kVecs + tid % kVecs;
      if (i >= row.vecs) continue;
      float v[N];
      row.load(i).values(v);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int64_t col = row.col(i) + j;
        if (col >= 0 && col < row.V) f(Key::of(v[j]), (uint32_t)col);
      }
    }
  };
  auto collect = [&] {
    each(bound + 1, [&](uint32_t key, uint32_t col) {
      if (key > bound) {
        const uint32_t at = atomicAdd(s_count, 1u);
        if (at < kLpCandidates) s_list[at] = ((uint64_t)key << 32) | (uint32_t)~col;
      }
    });
    __syncthreads();
  };
  collect();
  if (*s_count > kLpCandidates) {
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = Key::kBits - 1; bit >= 0; --bit) {
      const uint32_t up = t | (1u << bit);
      uint32_t n = 0;
      each(up, [&](uint32_t key, uint32_t) { n += key >= up ? 1u : 0u; });
      if (lp_block_sum<NT>(n, s_n, turn++) >= K) t = up;
    }
    bound = t;
    __syncthreads();
    if (tid == 0) *s_count = 0u;
    __syncthreads();
    collect();   // fewer than K
  }
  const uint32_t above = *s_count;
  // elements at the bound, in the order of their columns, until there are K
  uint32_t n = above;
  if (tid < 32 && n < K) {
    constexpr int kStep = 32 / kVecs;   // chunks that a warp looks at at once
    for (int c0 = 0; c0 < chunks && n < K; c0 += kStep) {
      const int c = c0 + lane / kVecs;
      const bool look = c < chunks && Key::of(s_max[c]) >= bound;
      if (!__any_sync(0xffffffffu, look)) continue;
      const int64_t i = (int64_t)c * kVecs + lane % kVecs;
      uint32_t ties = 0;
      float v[N];
      if (look && i < row.vecs) {
        row.load(i).values(v);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int64_t col = row.col(i) + j;
          if (col >= 0 && col < row.V && Key::of(v[j]) == bound) ties |= 1u << j;
        }
      }
      uint32_t before = __popc(ties);   // of lower lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      const uint32_t all = __shfl_sync(0xffffffffu, before, 31);
      uint32_t at = n + before - __popc(ties);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if ((ties >> j & 1u) && at < K) s_list[at] = ((uint64_t)bound << 32) | (uint32_t)~(uint32_t)(row.col(i) + j);
        at += ties >> j & 1u;
      }
      n = min(K, n + all);
    }
  }
  if (tid == 0) *s_count = max(n, above);   // (above K only where the list holds it)
  __syncthreads();
  n = *s_count;
  // each candidate's rank is the number of better ones: all keys differ by their column
  for (uint32_t i = tid; i < n; i += NT) {
    const uint64_t mine = s_list[i];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += s_list[j] > mine ? 1u : 0u;
    if (rank < K) {
      const uint32_t col = ~(uint32_t)mine;
      p.ids[m * p.K + rank] = col;
      p.top[m * p.K + rank] = nan ? NAN : lp_log(to_f32<T>(row.z[col]), high, p.tau, log_s);
    }
  }
}

// A block (a cluster of them, each with a slice of the columns, where there are fewer rows
// than places) works on one row.
template <typename T, int NT, bool TOP, bool FINE>
__global__ void __launch_bounds__(NT) logprob_fwd_kernel(const __grid_constant__ LogprobParams p) {
  constexpr int N = LpVec<T>::N, U = 4, kWarps = NT / 32;
  namespace cg = cooperative_groups;
  auto cluster = cg::this_cluster();
  const int csize = (int)cluster.num_blocks(), crank = (int)cluster.block_rank();
  extern __shared__ float lp_smem[];   // chunks' maxima (rank 0: of the whole row), the list
  __shared__ LpSums s_part[8 * kWarps];
  __shared__ uint32_t s_n[3], s_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t m = blockIdx.x / (unsigned)csize;
  const int64_t y = p.targets != nullptr ? p.targets[m] : 0;
  const bool counted = y >= 0 && y < p.V;
  if (!counted) {   // (all blocks of the cluster)
    if (crank == 0) {
      for (int i = tid; i < p.K; i += NT) p.ids[m * p.K + i] = -1, p.top[m * p.K + i] = 0.0f;
      if (tid == 0) {
        if (p.targets != nullptr) p.logp[m] = 0.0f;
        p.entropy[m] = 0.0f;
        p.stats[3 * m] = 0.0f, p.stats[3 * m + 1] = INFINITY, p.stats[3 * m + 2] = 0.0f;
      }
    }
    return;
  }
  const LpRow<T> row(p.z, m, p.stride, p.V);
  float* s_max = lp_smem;
  if (csize > 1) {
    if constexpr (TOP) s_max = cluster.map_shared_rank(lp_smem, 0);
    cluster.sync();   // rank 0, to which the others write, is there
  }
  // tiles of 32 vectors; a warp takes U of them at a time
  const int64_t tiles = (row.vecs + 31) / 32, per = (tiles + csize - 1) / csize;
  const int64_t t0 = min(tiles, per * crank), t1 = min(tiles, t0 + per);
  LpSums x{-INFINITY, 0.0f, 0.0f};
  const float scale = p.scale;
  for (int64_t t = t0 + warp * U; t < t1; t += kWarps * U) {
    LpVec<T> r[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int64_t i = (t + j) * 32 + lane;
      if (t + j < t1 && i < row.vecs) r[j] = row.load(i);
      else {
        float none[N];
#pragma unroll
        for (int e = 0; e < N; ++e) none[e] = -INFINITY;
        r[j].set(none);
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float v[N];
      r[j].values(v);
      float top = v[0];
#pragma unroll
      for (int e = 1; e < N; ++e) top = max_nan(top, v[e]);
      if constexpr (TOP) {
        if constexpr (FINE) {
          if (t + j < t1 && (t + j) * 32 + lane < row.vecs) s_max[(t + j) * 32 + lane] = top;
        } else {
          float all;
          asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(all) : "f"(top));
          if (lane == 0 && t + j < t1) s_max[t + j] = all;
        }
      }
      if (top > x.m) lp_raise(x, top, scale);
      const float from = x.m == -INFINITY ? 0.0f : x.m;   // nothing but -inf so far: weights of 0
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float tt = lp_t(v[e], from, scale), w = lp_exp2(tt);
        x.s += w;
        x.a = fmaf(w, tt, x.a);
      }
    }
  }
  x = lp_warp_join(x, scale);
  if (lane == 0) {
    LpSums* to = s_part;
    if (csize > 1) to = cluster.map_shared_rank(s_part, 0);
    to[crank * kWarps + warp] = x;
  }
  if (csize > 1) {
    cluster.sync();
    if (crank > 0) return;
  } else {
    __syncthreads();
  }
  x = LpSums{-INFINITY, 0.0f, 0.0f};
  for (int i = 0; i < csize * kWarps; ++i) x = lp_join(x, s_part[i], scale);   // the same in every thread
  if (x.m == -INFINITY && !(x.s != x.s)) {   // no logit above -inf
    for (int i = tid; i < p.K; i += NT) p.ids[m * p.K + i] = -1, p.top[m * p.K + i] = 0.0f;
    if (tid == 0) {
      if (p.targets != nullptr) p.logp[m] = 0.0f;
      p.entropy[m] = 0.0f;
      p.stats[3 * m] = 0.0f, p.stats[3 * m + 1] = INFINITY, p.stats[3 * m + 2] = 0.0f;
    }
    return;
  }
  const bool nan = !(x.s < INFINITY) || x.m == INFINITY;
  const double log_s = log((double)x.s);
  if (tid == 0) {
    const double l2 = log2((double)x.s);
    const float h = nan ? NAN : fmaxf(0.0f, (float)((l2 - (double)x.a / (double)x.s) * 0.6931471805599453));
    if (p.targets != nullptr) p.logp[m] = nan ? NAN : lp_log(to_f32<T>(row.z[y]), x.m, p.tau, log_s);
    p.entropy[m] = h;
    p.stats[3 * m] = nan ? NAN : x.m;
    p.stats[3 * m + 1] = nan ? NAN : (float)l2;
    p.stats[3 * m + 2] = h;
  }
  if constexpr (TOP) {
    uint64_t* s_list = reinterpret_cast<uint64_t*>(lp_smem + (p.chunks + 1) / 2 * 2);
    lp_top<T, NT, FINE>(p, row, m, lp_smem, (int)(FINE ? row.vecs : tiles), x.m, log_s, nan, s_n, s_list, &s_count);
  }
}

// Gradient: a block takes kLpSeg vectors of a row.
constexpr int kLpBwdThreads = 256, kLpBwdVecs = 4;
constexpr int kLpSeg = kLpBwdThreads * kLpBwdVecs;

template <typename T>
__global__ void __launch_bounds__(kLpBwdThreads) logprob_bwd_kernel(const __grid_constant__ LogprobParams p, int segs) {
  constexpr int N = LpVec<T>::N;
  __shared__ float s_g[kLpBwdThreads / 32];
  __shared__ int s_hit;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t m = blockIdx.x / (unsigned)segs, seg = blockIdx.x - m * segs;
  // the gradient's row has the logits' alignment; its vectors, the columns behind V among them
  const LpRow<T> row(p.z, m, p.stride, p.V);
  T* out = reinterpret_cast<T*>(p.dz) + m * p.gstride;
  const float high = p.stats[3 * m], l2 = p.stats[3 * m + 1], h = p.stats[3 * m + 2];
  const bool counted = !(l2 == INFINITY);
  const int64_t i0 = seg * kLpSeg + tid;
  LpVec<T> r[kLpBwdVecs];
#pragma unroll
  for (int j = 0; j < kLpBwdVecs; ++j) {
    const int64_t i = i0 + j * kLpBwdThreads;
    r[j].u = make_uint4(0u, 0u, 0u, 0u);
    if (counted && i < row.vecs) r[j] = row.load(i);
  }
  const float gh = p.gh != nullptr && counted ? p.gh[m] : 0.0f;
  const float gy = p.gp != nullptr && counted ? p.gp[m] : 0.0f;
  float g = 0.0f;   // of all entries
  if (p.gt != nullptr && counted) {
    for (int i = tid; i < p.K; i += kLpBwdThreads) g += p.gt[m * p.K + i];
    g = warp_sum(g);
    if (lane == 0) s_g[warp] = g;
    __syncthreads();
    g = 0.0f;
#pragma unroll
    for (int i = 0; i < kLpBwdThreads / 32; ++i) g += s_g[i];
  }
  // dz = p (c0 + c1 log2 p) + g terms
  const float inv = (float)(1.0 / p.tau);
  const float c0 = -(g + gy + gh * h) * inv, c1 = -gh * kLpLn2 * inv;
  auto smooth = [&](float z) {
    const float t = max_nan((z - high) * p.scale - l2, -1000.0f);
    return lp_exp2(t) * fmaf(c1, t, c0);
  };
#pragma unroll
  for (int j = 0; j < kLpBwdVecs; ++j) {
    const int64_t i = i0 + j * kLpBwdThreads, col = row.col(i);
    if (col >= p.width) continue;
    float v[N];
    r[j].values(v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = counted && col + e < p.V ? smooth(v[e]) : 0.0f;
    if (col >= 0 && col + N <= p.width) {
      LpVec<T> o;
      o.set(v);
      *reinterpret_cast<uint4*>(out + col) = o.u;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (col + e >= 0 && col + e < p.width) out[col + e] = from_f32<T>(v[e]);
    }
  }
  if (!counted) return;
  // columns with g terms
  const int64_t y = p.targets != nullptr && p.gp != nullptr ? p.targets[m] : -1;
  const int64_t c_begin = row.col(seg * kLpSeg), c_end = row.col((seg + 1) * kLpSeg);
  if (tid == 0) s_hit = 0;
  __syncthreads();   // the vectors are written
  if (p.gt != nullptr) {
    for (int i = tid; i < p.K; i += kLpBwdThreads) {
      const int64_t c = p.ids[m * p.K + i];
      if (c == y) s_hit = 1;
      if (c < c_begin || c >= c_end || c < 0) continue;
      const float more = p.gt[m * p.K + i] + (c == y ? gy : 0.0f);
      out[c] = from_f32<T>(smooth(to_f32<T>(row.z[c])) + more * inv);
    }
    __syncthreads();
  }
  if (tid == 0 && y >= c_begin && y < c_end && y >= 0 && s_hit == 0)
    out[y] = from_f32<T>(smooth(to_f32<T>(row.z[y])) + gy * inv);
}

}  // namespace zq

using namespace zq;

namespace {

LogprobParams lp_params(const at::Tensor& z, const c10::optional<at::Tensor>& targets, const at::Tensor& top,
                        const at::Tensor& ids, const at::Tensor& stats, int64_t vocab, double temperature) {
  TORCH_CHECK(z.is_cuda() && z.dim() == 2 && z.size(0) > 0 && z.size(1) > 0 && (z.stride(1) == 1 || z.size(1) == 1),
              "token_logprobs: logits [M, V] on the GPU with unit column stride");
  TORCH_CHECK(vocab > 0 && vocab <= z.size(1) && vocab <= (1LL << 22), "token_logprobs: vocab must be 1 to the logits' width, at most 2^22");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(z.data_ptr()) % z.element_size() == 0, "token_logprobs: alignment");
  const int64_t M = z.size(0);
  const int dev = z.get_device();
  auto here = [&](const at::Tensor& t, at::ScalarType type, int64_t n) {
    return t.is_cuda() && t.get_device() == dev && t.is_contiguous() && t.scalar_type() == type && t.numel() == n;
  };
  LogprobParams p = {};
  p.K = (int)top.size(-1);
  TORCH_CHECK(p.K <= kLpMaxTop && p.K <= vocab, "token_logprobs: at most ", kLpMaxTop, " alternatives of the vocabulary");
  TORCH_CHECK(here(top, at::kFloat, M * p.K) && here(ids, at::kLong, M * p.K) && here(stats, at::kFloat, 3 * M),
              "token_logprobs: top fp32 [M, K], ids int64 [M, K], stats fp32 [M, 3]");
  if (targets.has_value()) {
    TORCH_CHECK(here(*targets, at::kLong, M), "token_logprobs: targets int64 [M], contiguous, on the logits' device");
    p.targets = targets->data_ptr<int64_t>();
  }
  p.z = z.data_ptr();
  p.top = top.data_ptr<float>();
  p.ids = ids.data_ptr<int64_t>();
  p.stats = stats.data_ptr<float>();
  p.M = M;
  p.stride = z.stride(0);
  p.width = z.size(1);
  p.V = vocab;
  p.scale = (float)(1.4426950408889634 / temperature);
  p.tau = temperature;
  return p;
}

template <typename T, int NT, bool TOP, bool FINE>
void lp_launch(LogprobParams& p, cudaStream_t stream) {
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  constexpr int N = LpVec<T>::N;
  const int64_t vecs = (p.V + 2 * N - 2) / N;   // at the worst alignment
  p.chunks = FINE ? (int)vecs : (int)((vecs + 31) / 32);
  auto kern = logprob_fwd_kernel<T, NT, TOP, FINE>;
  const size_t smem = TOP ? ((size_t)p.chunks + 1) / 2 * 8 + 8 * (size_t)(kLpCandidates + p.K) : 0;
  // a cluster to a row where that leaves SMs without a block, down to 4 warp tiles a warp
  int csize = 1;
  while (csize < 8 && p.M * csize * 2 <= 2 * sms && vecs / (2 * csize) >= 4 * NT) csize *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.M * csize));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)csize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (smem > 48 * 1024)
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
}

}  // namespace

#define ZQ_LP_TYPES(TYPE, ...)                                                 \
  switch (TYPE) {                                                              \
    case at::kBFloat16: { using T = __nv_bfloat16; __VA_ARGS__; break; }       \
    case at::kHalf: { using T = __half; __VA_ARGS__; break; }                  \
    case at::kFloat: { using T = float; __VA_ARGS__; break; }                  \
    default: TORCH_CHECK(false, "token_logprobs: bf16, fp16 or fp32 logits");  \
  }

void logprob_fwd(at::Tensor z, c10::optional<at::Tensor> targets, c10::optional<at::Tensor> logp, at::Tensor entropy,
                 at::Tensor top, at::Tensor ids, at::Tensor stats, int64_t vocab, double temperature) {
  LogprobParams p = lp_params(z, targets, top, ids, stats, vocab, temperature);
  TORCH_CHECK(targets.has_value() == logp.has_value(), "token_logprobs: log probabilities go with targets");
  TORCH_CHECK(entropy.is_cuda() && entropy.get_device() == z.get_device() && entropy.is_contiguous() &&
                  entropy.scalar_type() == at::kFloat && entropy.numel() == p.M,
              "token_logprobs: entropy fp32 [M]");
  p.entropy = entropy.data_ptr<float>();
  if (logp.has_value()) {
    TORCH_CHECK(logp->is_cuda() && logp->get_device() == z.get_device() && logp->is_contiguous() &&
                    logp->scalar_type() == at::kFloat && logp->numel() == p.M,
                "token_logprobs: log probabilities fp32 [M]");
    p.logp = logp->data_ptr<float>();
  }
  TORCH_CHECK(p.M < (1LL << 28), "token_logprobs: too many rows");
  const c10::cuda::CUDAGuard guard(z.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  ZQ_LP_TYPES(z.scalar_type(), {
    if (p.K == 0) lp_launch<T, 256, false, false>(p, stream);
    else if (p.V <= kLpFine) lp_launch<T, 256, true, true>(p, stream);
    else lp_launch<T, 256, true, false>(p, stream);
  });
}

// dz [M, W] (the columns behind vocab are 0) from gradients of logp, entropy and top
void logprob_bwd(at::Tensor z, c10::optional<at::Tensor> targets, at::Tensor top, at::Tensor ids, at::Tensor stats,
                 c10::optional<at::Tensor> gp, c10::optional<at::Tensor> gh, c10::optional<at::Tensor> gt, at::Tensor dz,
                 int64_t vocab, double temperature) {
  LogprobParams p = lp_params(z, targets, top, ids, stats, vocab, temperature);
  const int dev = z.get_device();
  auto grad = [&](const c10::optional<at::Tensor>& g, int64_t n) -> const float* {
    if (!g.has_value()) return nullptr;
    TORCH_CHECK(g->is_cuda() && g->get_device() == dev && g->is_contiguous() && g->scalar_type() == at::kFloat && g->numel() == n,
                "token_logprobs: gradients fp32, contiguous, like the outputs");
    return g->data_ptr<float>();
  };
  p.gp = grad(gp, p.M);
  p.gh = grad(gh, p.M);
  p.gt = p.K > 0 ? grad(gt, p.M * p.K) : nullptr;
  TORCH_CHECK(p.gp == nullptr || p.targets != nullptr, "token_logprobs: a gradient of log probabilities needs targets");
  TORCH_CHECK(dz.is_cuda() && dz.get_device() == dev && dz.scalar_type() == z.scalar_type() && dz.sizes() == z.sizes() &&
                  (dz.stride(1) == 1 || p.width == 1) && (p.M == 1 || dz.stride(0) >= p.width),
              "token_logprobs: the gradient is like the logits, rows apart");
  p.dz = dz.data_ptr();
  p.gstride = dz.stride(0);
  const int64_t es = z.element_size();
  TORCH_CHECK(((reinterpret_cast<uintptr_t>(p.z) ^ reinterpret_cast<uintptr_t>(p.dz)) & 15) == 0 &&
                  (p.M == 1 || ((p.stride - p.gstride) * es) % 16 == 0),
              "token_logprobs: logits rows must be aligned as the gradient's");
  const int64_t N = 16 / es, vecs = (p.width + 2 * N - 2) / N, segs = (vecs + kLpSeg - 1) / kLpSeg;
  TORCH_CHECK(p.M * segs < (1LL << 31), "token_logprobs: too many rows");
  const c10::cuda::CUDAGuard guard(z.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  ZQ_LP_TYPES(z.scalar_type(), {
    logprob_bwd_kernel<T><<<(unsigned)(p.M * segs), kLpBwdThreads, 0, stream>>>(p, (int)segs);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
