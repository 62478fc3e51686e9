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
// Forward: one pass over a row with a running reference m (the maximum, or up to 12 powers of
// two less) and S = Σ 2^t, A = Σ t 2^t, t = z s - m s, s = log2(e) / τ; H = ln2 (log2 S - A / S).
// Where m rises by d powers of two, A' = (A - d S) 2^-d, S' = S 2^-d.  The shift m s is rounded
// and the same one wherever it enters, so t carries one rounding of a small number and no
// error of the size of m s.  Rows whose maximum is far from 0 (all masked by the type's lowest
// value) are summed again from differences.  The top alternatives cost that pass the maximum of every
// chunk of columns: the k best of the row lie in the k chunks with the best maxima, so the k-th
// best of those is a bound, and a second launch looks at the chunks that reach it alone.
// Backward: one pass, p from the row's m, S and H; the columns with a g term are written a
// second time by their warp (each sum rounded once; no atomics).
//
// What bounds it: memory, next to 16 exponentials a cycle and SM.  8192 x 152064 bf16: forward
// 372 us (a copy's rate), 403 and 81 for the ranking with 32 alternatives; gradient 785 us (0.97).
// 4096 x 50257 with an eighth of the rows not counted: 78 and 137 us (0.71, 0.86): a row's start and
// end weigh more, and 3584 rows are three and a bit rounds of blocks.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>

#include <type_traits>

#include "rows.cuh"

namespace zq {

constexpr int kLpMaxTop = 256;
constexpr int kLpCandidates = 512;      // of the list in shared memory, besides k ties
constexpr int kLpHits = 512;             // chunks of the list of those that reach the bound
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpLn2 = 0.6931471805599453f;

struct LogprobParams {
  const void* z;
  const int64_t* targets;   // [M] or null: every row counts, no logp
  float *logp, *entropy;    // [M]
  float* top;               // [M, K]
  int64_t* ids;             // [M, K]
  float* stats;             // [M, 3]: m, S, H of counted rows; S = inf of the others
  uint8_t* maxima;          // [M, row_maxima] bytes: see LpMaxima
  int64_t row_maxima;
  const float *gp, *gh, *gt;   // gradients, or null
  void* dz;
  int64_t M, stride, gstride, width, V;
  int K;
  float scale;              // log2(e) / τ
  double inv_tau, inv_scale;
};

__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// t of a logit for any row: exact difference first, so nothing overflows that is finite in the
// end, and a bound from below, under which 2^t is 0 (t 2^t would be 0 · -inf).  NaN stays.
__device__ __forceinline__ float lp_t(float z, float m, float scale) { return max_nan((z - m) * scale, -1000.0f); }

// The shift of a reference m, the rounded product -m s.  It is rounded down: where m is a mask's
// value so far (-1e9, the type's lowest) what the rounding leaves may be any power of two, but
// none above 1, and sums of 0 go when the reference moves up.
__device__ __forceinline__ float lp_shift(float m, float scale) { return __fmul_rd(-m, scale); }

// Logits from here down are taken as this: they weigh 0 in a row whose reference is in the range
// where what the shift's rounding leaves is small (t < -1.3e7 at a temperature of 1e6), and t stays
// finite, also times up to |g_H| / τ in the gradient: 2^t = 0 times what overflows would be NaN
// (-1e13 · 1.44 ln 2 |g_H| / τ² does from |g_H| / τ² = 3e25 on, -1e30 did from 3e8).  Other rows take
// the form above.
constexpr float kLpFloor = -1e13f;
__device__ __forceinline__ bool lp_plain(float m, float scale) { return fabsf(m * scale) < 1e6f; }

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
  // the largest; NaN where there is one
  __device__ __forceinline__ float largest() const {
    if constexpr (sizeof(T) == 4) {
      return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)), max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2 a = __hmax2_nan(*reinterpret_cast<const T2*>(&u.x), *reinterpret_cast<const T2*>(&u.y));
      const T2 b = __hmax2_nan(*reinterpret_cast<const T2*>(&u.z), *reinterpret_cast<const T2*>(&u.w));
      const T2 c = __hmax2_nan(a, b);
      return max_nan(to_f32<T>(c.x), to_f32<T>(c.y));
    }
  }
  // bounded from below by the floor (bf16 has it: before the values are spread); NaN stays
  __device__ __forceinline__ void floored_pairs(uint64_t (&p)[N / 2]) const {
    float v[N];
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      __nv_bfloat162 low;
      low.x = low.y = __float2bfloat16_rn(kLpFloor);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), low);
        const float2 f = bf16x2_to_f2(*reinterpret_cast<const uint32_t*>(&m));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    } else {
      values(v);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = max_nan(v[i], kLpFloor);
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) p[i] = f2_pack(v[2 * i], v[2 * i + 1]);
  }
  __device__ __forceinline__ void set_pairs(const uint64_t (&p)[N / 2]) {
    float v[N];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) f2_unpack(p[i], v[2 * i], v[2 * i + 1]);
    set(v);
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
  int lead, V, vecs;
  __device__ __forceinline__ LpRow(const void* base, int64_t row, int64_t stride, int V_) : V(V_) {
    z = reinterpret_cast<const T*>(base) + row * stride;
    lead = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
    vecs = (lead + V + N - 1) / N;
  }
  __device__ __forceinline__ int col(int i) const { return i * N - lead; }
  __device__ __forceinline__ bool whole(int i) const { return col(i) >= 0 && col(i) + N <= V; }
  // vectors [i, i + n) are whole
  __device__ __forceinline__ bool inside(int i, int n) const { return col(i) >= 0 && col(i + n) <= V; }
  __device__ __forceinline__ LpVec<T> load_whole(int i) const {
    LpVec<T> r;
    r.u = __ldg(reinterpret_cast<const uint4*>(z - lead) + i);
    return r;
  }
  __device__ __forceinline__ void ahead(int i) const {
    if (whole(i)) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint4*>(z - lead) + i));
  }
  __device__ __forceinline__ LpVec<T> load(int i) const {   // (-inf behind the row's last, too)
    if (whole(i)) return load_whole(i);
    LpVec<T> r;
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = col(i) + j;
      v[j] = c >= 0 && c < V ? to_f32<T>(z[c]) : -INFINITY;
    }
    r.set(v);
    return r;
  }
};

struct LpSums {
  float m, s, a;
};

// How far the largest may leave the reference behind, in powers of two: 2^t stays below 2^12
// (S and A are relative to m in any case), and the rescaling, which one of a warp's lanes
// would nearly always want, becomes rare.
constexpr float kLpBehind = 12.0f;

// Factors of S and A where the reference goes up from m to `to`: PLAIN as their shifts differ
template <bool PLAIN>
__device__ __forceinline__ void lp_raise(LpSums& x, float to, float scale) {
  if (x.m != -INFINITY) {   // (otherwise nothing yet, or a NaN, which stays)
    const float d = PLAIN ? lp_shift(to, scale) - lp_shift(x.m, scale) : lp_t(x.m, to, scale);   // <= 0
    const float f = lp_exp2(d);
    x.a = f * fmaf(d, x.s, x.a);
    x.s *= f;
  }
  x.m = to;
}

template <bool PLAIN>
__device__ __forceinline__ LpSums lp_join(LpSums a, LpSums b, float scale) {
  const float to = fmaxf(a.m, b.m);
  if (to > a.m) lp_raise<PLAIN>(a, to, scale);
  if (to > b.m) lp_raise<PLAIN>(b, to, scale);
  a.s += b.s;
  a.a += b.a;
  return a;
}

template <bool PLAIN>
__device__ __forceinline__ LpSums lp_warp_join(LpSums x, float scale) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpSums y;
    y.m = __shfl_xor_sync(0xffffffffu, x.m, o);
    y.s = __shfl_xor_sync(0xffffffffu, x.s, o);
    y.a = __shfl_xor_sync(0xffffffffu, x.a, o);
    x = lp_join<PLAIN>(x, y, scale);
  }
  return x;
}

// log of a positive number: its exponent's part in 64 bits, its mantissa's (below 0.35) in 32
__device__ __forceinline__ double lp_log(float s) {
  const int e = (__float_as_int(s) - 0x3f3504f3) >> 23;   // mantissa in [sqrt(1/2), sqrt(2))
  return (double)e * 0.69314718055994531 + (double)logf(__int_as_float(__float_as_int(s) - (e << 23)));
}
// A row's few numbers, in 64 bits (sums and products; divisions and logarithms would take longer
// than a short row): l = (z - m) / τ - log S.  Plain sums are relative to the rounded shift: m is
// what it stands for.
struct LpLog {
  double m, log_s, inv_tau;
  __device__ __forceinline__ LpLog(const LogprobParams& p, float high, float sum)
      : m(lp_plain(high, p.scale) ? -(double)lp_shift(high, p.scale) * p.inv_scale : (double)high),
        log_s(sum < INFINITY ? lp_log(sum) : 0.0), inv_tau(p.inv_tau) {}
  // At most 0, as p is at most 1: a certain token's S may be below 1 by the exponential's error.
  __device__ __forceinline__ float of(float z) const { return (float)fmin(((double)z - m) * inv_tau - log_s, 0.0); }
};

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
  static __device__ __forceinline__ float value(uint32_t key) {
    if (key == 0xffffffffu >> kLow) return NAN;
    const uint32_t b = key << kLow;
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~(b | ((1u << kLow) - 1u)));
  }
};

// What the pass over a row keeps for its top alternatives: the maxima of its chunks.  A chunk is a
// vector (G = 1, rows of few vectors for the alternatives wanted), or a lane's vectors of the four
// tiles that a warp takes at a time (G = 4); 9.5 KB for a row of 152064 columns of bf16.
template <typename T, int G>
struct LpMaxima {
  static constexpr int kPad = 16 / (int)sizeof(T);
  T* chunk;
  static __host__ __device__ constexpr int chunks(int vecs) { return G == 1 ? vecs : (vecs + 127) / 128 * 32; }
  static __host__ __device__ constexpr int64_t bytes(int vecs) {   // of a row
    return (int64_t)((chunks(vecs) + kPad - 1) / kPad * kPad) * (int64_t)sizeof(T);
  }
  __device__ __forceinline__ LpMaxima(const LogprobParams& p, int64_t m) : chunk(reinterpret_cast<T*>(p.maxima + m * p.row_maxima)) {}
  static __device__ __forceinline__ int vector(int c, int j) { return G == 1 ? c : (c / 32 * 4 + j) * 32 + c % 32; }
  static __device__ __forceinline__ int chunk_of(int i) { return G == 1 ? i : i / 128 * 32 + i % 32; }
};

constexpr int kLpParts = 512;   // a row's chunks in at most this many parts
struct LpLists {                 // of a warp that ranks a row's alternatives
  uint64_t cand[kLpCandidates + kLpMaxTop];
  uint32_t key[kLpParts];        // of the parts; then the parts that reach the bound
  uint32_t hits[kLpHits];        // chunks that do
  uint32_t vecs[128];            // vectors that do, of a step
};

// 16 bytes where `there`, without a branch: several such loads are under way at once
__device__ __forceinline__ uint4 lp_load_if(const void* p, bool there) {
  uint4 r = make_uint4(0u, 0u, 0u, 0u);
  asm volatile(
      "{\n"
      "  .reg .pred p;\n"
      "  setp.ne.u32 p, %5, 0;\n"
      "  @p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n"
      "}\n"
      : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)
      : "l"(p), "r"((uint32_t)there));
  return r;
}

// The top alternatives of a row, by one warp, in a launch of its own: what it waits for (the
// row's maxima, its candidates from memory) is 5 to 10 us, in which the pass over the logits would
// have one warp of its blocks at work (8192 x 152064 with 32 alternatives: 542 us).
template <typename T, int G>
__device__ void lp_top(const LogprobParams& p, const LpRow<T>& row, int64_t m, const LpMaxima<T, G>& s_max, const LpLog& log,
                       bool nan, LpLists& list) {
  constexpr int N = LpVec<T>::N;
  using Key = LpKey<T>;
  using Max = LpMaxima<T, G>;
  const int lane = threadIdx.x & 31, chunks = Max::chunks(row.vecs);
  const uint32_t K = (uint32_t)p.K, below = (1u << lane) - 1u;
  auto chunk_key = [&](int i) { return Key::of(to_f32<T>(s_max.chunk[i])); };
  // Parts of `size` consecutive chunks.  The K-th best of the parts' maxima (0, below all, where
  // there are fewer) is the bound: of n parts some -n log(1 - K / n) elements reach it.
  // (One warp at work waits for its instructions too: loops here are short and rolled.)
  int shift = 0;
  while ((kLpParts << shift) < chunks) ++shift;
  const int size = 1 << shift, parts = (chunks + size - 1) >> shift;
  for (int i = lane; i < parts; i += 32) list.key[i] = 0u;
  __syncwarp();
  constexpr int A = 4;   // loads of a lane under way
  for (int c0 = 0; c0 < chunks; c0 += 32 * N * A) {   // (a row's chunks end in a whole vector)
    LpVec<T> r[A];
#pragma unroll
    for (int j = 0; j < A; ++j) {
      const int c = c0 + (j * 32 + lane) * N;
      r[j].u = lp_load_if(s_max.chunk + c, c < chunks);
    }
#pragma unroll
    for (int j = 0; j < A; ++j) {
      const int c = c0 + (j * 32 + lane) * N;
      if (c >= chunks) continue;
      if (size >= N) {
        atomicMax(&list.key[c >> shift], Key::of(r[j].largest()));
      } else {
        float v[N];
        r[j].values(v);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (c + e < chunks) atomicMax(&list.key[(c + e) >> shift], Key::of(v[e]));
      }
    }
  }
  __syncwarp();
  uint32_t bound = 0;
  if (parts >= p.K) {
#pragma unroll 1
    for (int bit = Key::kBits - 1; bit >= 0; --bit) {
      const uint32_t up = bound | (1u << bit);   // (above 0, the key of no part)
      uint32_t n = 0;
#pragma unroll 8
      for (int i = lane; i < parts; i += 32) n += list.key[i] >= up ? 1u : 0u;
      if (__reduce_add_sync(0xffffffffu, n) >= K) bound = up;
    }
  }
  // the parts that reach it, and their chunks that do
  auto push = [&](bool in, uint32_t what, uint32_t* to, int& n, int room) {
    const uint32_t all = __ballot_sync(0xffffffffu, in);
    const int at = n + __popc(all & below);
    if (in && at < room) to[at] = what;
    n += __popc(all);
  };
  int n_parts = 0, hits = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < parts; i0 += 32) {   // (in place: no further than what has been read)
    const bool in = i0 + lane < parts && list.key[min(i0 + lane, kLpParts - 1)] >= bound;
    __syncwarp();
    push(in, (uint32_t)(i0 + lane), list.key, n_parts, kLpParts);
    __syncwarp();
  }
#pragma unroll 1
  for (int i0 = 0; i0 < n_parts << shift; i0 += 32 * A) {
    uint32_t k[A];
    int c[A];
#pragma unroll
    for (int j = 0; j < A; ++j) {
      const int i = i0 + j * 32 + lane;
      c[j] = i < n_parts << shift ? ((int)list.key[min(i >> shift, n_parts - 1)] << shift) + (i & (size - 1)) : chunks;
      k[j] = chunk_key(min(c[j], chunks - 1));
    }
#pragma unroll
    for (int j = 0; j < A; ++j) push(c[j] < chunks && k[j] >= bound, (uint32_t)c[j], list.hits, hits, kLpHits);
  }
  __syncwarp();
  // A lane's vector of those that hold elements that reach `at_least` (no less than the bound of
  // the list of chunks): f(vector, values, bits of its elements that do); in every lane.
  auto each = [&](uint32_t at_least, auto&& f) {
    const bool listed = hits <= kLpHits;   // (otherwise many equal maxima: all chunks)
    const int vecs = listed ? hits * G : row.vecs;
#pragma unroll 1
    for (int v0 = 0; v0 < vecs; v0 += 32 * A) {
      LpVec<T> r[A];
      int i[A], n = 0;
#pragma unroll
      for (int j = 0; j < A; ++j) {
        const int v = v0 + j * 32 + lane;
        i[j] = v >= vecs ? row.vecs : listed ? Max::vector((int)list.hits[v / G], v % G) : v;
        r[j].u = lp_load_if(row.z + row.col(i[j]), row.whole(i[j]));
      }
#pragma unroll
      for (int j = 0; j < A; ++j)   // (the row's edges are looked at below)
        push(i[j] < row.vecs && (!row.whole(i[j]) || Key::of(r[j].largest()) >= at_least), (uint32_t)i[j], list.vecs, n, 128);
      __syncwarp();
#pragma unroll 1
      for (int u = 0; u < n; u += 32) {
        uint32_t bits = 0;
        const int at = u + lane < n ? (int)list.vecs[u + lane] : row.vecs;
        float v[N];
        if (at < row.vecs) {
          row.load(at).values(v);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int col = row.col(at) + e;
            bits |= (Key::of(v[e]) >= at_least && col >= 0 && col < row.V ? 1u : 0u) << e;
          }
        }
        f(at, v, bits);
      }
      __syncwarp();
    }
  };
  // Places for the lanes' numbers of elements, in the order of the lanes; all of them in `sum`.
  auto places = [&](uint32_t count, uint32_t& sum) {
    uint32_t to = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += up;
    }
    sum = __shfl_sync(0xffffffffu, to, 31);
    return to - count;
  };
  auto collect = [&](uint32_t from) {
    uint32_t n = 0;
    __syncwarp();
    each(from, [&](int i, const float (&v)[N], uint32_t bits) {
      uint32_t sum, at = n + places(__popc(bits), sum);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (bits >> e & 1u) {
          if (at < kLpCandidates) list.cand[at] = ((uint64_t)Key::of(v[e]) << 32) | (uint32_t)~(uint32_t)(row.col(i) + e);
          ++at;
        }
      }
      n += sum;
    });
    __syncwarp();
    return n;
  };
  // Elements that reach the bound, in any order (they are ranked below).  Where they do not fit
  // the list, those above it, and then those at it in the order of their columns as far as they
  // are wanted (a row of many equal ones); where the former do not fit either (a row whose best
  // lie side by side), the bound rises to the K-th best element before.
  uint32_t n = collect(bound);
  if (n > kLpCandidates) {
    auto above = [&] { return bound < 0xffffffffu ? collect(bound + 1) : 0u; };   // (the largest key: NaN)
    n = above();
    if (n > kLpCandidates) {
      uint32_t t = 0;
#pragma unroll 1
      for (int bit = Key::kBits - 1; bit >= 0; --bit) {
        const uint32_t up = t | (1u << bit);
        uint32_t c = 0;
        each(up, [&](int, const float (&)[N], uint32_t bits) { c += __popc(bits); });
        if (__reduce_add_sync(0xffffffffu, c) >= K) t = up;
      }
      bound = t;
      n = above();   // fewer than K
    }
    // a vector a lane at a time, until there are K
    for (int i0 = 0; i0 < row.vecs && n < K; i0 += 32) {
      const int i = i0 + lane;
      uint32_t ties = 0;
      if (i < row.vecs && chunk_key(Max::chunk_of(i)) >= bound) {
        float v[N];
        row.load(i).values(v);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int col = row.col(i) + e;
          ties |= (Key::of(v[e]) == bound && col >= 0 && col < row.V ? 1u : 0u) << e;
        }
      }
      if (!__any_sync(0xffffffffu, ties != 0)) continue;
      uint32_t sum, at = n + places(__popc(ties), sum);
      for (; ties != 0 && at < K; ties &= ties - 1, ++at)
        list.cand[at] = ((uint64_t)bound << 32) | (uint32_t)~(uint32_t)(row.col(i) + __ffs(ties) - 1);
      n = min(K, n + sum);
    }
    __syncwarp();
  }
  // each candidate's rank is the number of better ones: all keys differ by their column
  for (uint32_t i = lane; i < n; i += 32) {
    const uint64_t mine = list.cand[i];
    const uint32_t col = ~(uint32_t)mine;
    uint32_t rank = 0;
#pragma unroll 4
    for (uint32_t j = 0; j < n; ++j) rank += list.cand[j] > mine ? 1u : 0u;
    if (rank < K) {
      p.ids[m * p.K + rank] = col;
      p.top[m * p.K + rank] = nan ? NAN : log.of(Key::value((uint32_t)(mine >> 32)));
    }
  }
}

// A warp's tiles [t0, t1) of 32 vectors of a row (t0 a multiple of 4): its sums, and its chunks'
// maxima.  Tiles that lie inside the row go in groups of U, the next group's loads ahead of this one's arithmetic,
// in packed pairs.
template <typename T, int G>
__device__ __forceinline__ LpSums lp_slice(const LpRow<T>& row, int t0, int t1, float scale, const LpMaxima<T, G>& s_max) {
  constexpr int N = LpVec<T>::N, P = N / 2, U = 4;
  const int lane = threadIdx.x & 31;
  const float behind = kLpBehind / scale;
  float m = -INFINITY;
  uint64_t s2 = 0ull, a2 = 0ull;
  auto add = [&](const LpVec<T> (&r)[U], int tile, int n) {
    float cm = -INFINITY;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (j < n) {
        const float top = r[j].largest();
        if constexpr (G == 1)   // (exact: one of the type's values; -inf up to a whole vector of them)
          if ((tile + j) * 32 + lane < (row.vecs + N - 1) / N * N) s_max.chunk[(tile + j) * 32 + lane] = from_f32<T>(top);
        cm = max_nan(cm, top);
      }
    }
    if constexpr (G > 1) s_max.chunk[tile / U * 32 + lane] = from_f32<T>(cm);
    cm = fmaxf(cm, kLpFloor);   // (a NaN is left to the sums)
    if (cm > m + behind || m == -INFINITY) {
      float s, a, lo, hi;
      f2_unpack(s2, lo, hi), s = lo + hi;
      f2_unpack(a2, lo, hi), a = lo + hi;
      LpSums x{m, s, a};
      lp_raise<true>(x, cm, scale);
      m = x.m, s2 = f2_pack(x.s, 0.0f), a2 = f2_pack(x.a, 0.0f);
    }
    const float shift = lp_shift(m, scale);
    const uint64_t sc = f2_pack(scale, scale), sh = f2_pack(shift, shift);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (j < n) {
        uint64_t z[P];
        r[j].floored_pairs(z);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const uint64_t t = f2_fma(z[i], sc, sh);
          float lo, hi;
          f2_unpack(t, lo, hi);
          const uint64_t w = f2_pack(lp_exp2(lo), lp_exp2(hi));
          s2 = f2_add(s2, w);
          a2 = f2_fma(w, t, a2);
        }
      }
    }
  };
  int t = t0;
  auto inside = [&](int t) { return t + U <= t1 && row.inside(t * 32, 32 * U); };
  auto fetch = [&](LpVec<T> (&r)[U], int t) {
#pragma unroll
    for (int j = 0; j < U; ++j) r[j] = row.load_whole((t + j) * 32 + lane);
  };
  while (t < t1) {
    if (inside(t)) {
      LpVec<T> next[U];
      fetch(next, t);
      for (;;) {
        LpVec<T> r[U];
#pragma unroll
        for (int j = 0; j < U; ++j) r[j] = next[j];
        const int here = t;
        t += U;
        const bool more = inside(t);
        if (more) fetch(next, t);
        add(r, here, U);
        if (!more) break;
      }
    } else {
      LpVec<T> r[U];
#pragma unroll
      for (int j = 0; j < U; ++j) r[j] = row.load((t + j) * 32 + lane);
      add(r, t, min(U, t1 - t));
      t += U;
    }
  }
  float lo, hi;
  LpSums x{m, 0.0f, 0.0f};
  f2_unpack(s2, lo, hi), x.s = lo + hi;
  f2_unpack(a2, lo, hi), x.a = lo + hi;
  return x;
}

// The sums of a whole row from differences, for rows whose maximum is far from 0.
template <typename T, int NT>
__device__ LpSums lp_far(const LpRow<T>& row, float scale, LpSums* s_part) {
  constexpr int N = LpVec<T>::N;
  LpSums x{-INFINITY, 0.0f, 0.0f};
  for (int i = threadIdx.x; i < row.vecs; i += NT) {
    const LpVec<T> r = row.load(i);
    float v[N];
    r.values(v);
    const float top = r.largest();
    if (top > x.m) lp_raise<false>(x, top, scale);
    const float from = x.m == -INFINITY ? 0.0f : x.m;   // nothing but -inf so far: weights of 0
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float t = lp_t(v[e], from, scale), w = lp_exp2(t);
      x.s += w;
      x.a = fmaf(w, t, x.a);
    }
  }
  x = lp_warp_join<false>(x, scale);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = x;
  __syncthreads();
  x = s_part[0];
  for (int i = 1; i < NT / 32; ++i) x = lp_join<false>(x, s_part[i], scale);
  return x;
}

// A block (a cluster of them, each with a slice of the columns, where there are fewer rows
// than places) works on one row.
template <typename T, int NT, int G>   // G: 0 without alternatives
__global__ void __launch_bounds__(NT, NT == 32 ? 24 : 1024 / NT) logprob_fwd_kernel(const __grid_constant__ LogprobParams p) {
  constexpr int kWarps = NT / 32;
  namespace cg = cooperative_groups;
  auto cluster = cg::this_cluster();
  const int csize = (int)cluster.num_blocks(), crank = (int)cluster.block_rank();
  __shared__ LpSums s_part[8 * kWarps];
  __shared__ LpSums s_row;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t m = blockIdx.x / (unsigned)csize;
  const LpRow<T> row(p.z, m, p.stride, (int)p.V);
  const LpMaxima<T, G> s_max(p, m);
  // consecutive groups of four tiles to a warp, as equal as they can be
  const int tiles = (row.vecs + 31) / 32, groups = (tiles + 3) / 4, part = crank * kWarps + warp, parts = csize * kWarps;
  const int t0 = 4 * (int)((int64_t)groups * part / parts), t1 = min(tiles, 4 * (int)((int64_t)groups * (part + 1) / parts));
  const int64_t y = p.targets != nullptr ? p.targets[m] : 0;
  row.ahead(t0 * 32 + lane);   // on its way while the target is read
  auto nothing = [&] {   // the row does not count
    if (tid == 0) {
      if (p.targets != nullptr) p.logp[m] = 0.0f;
      p.entropy[m] = 0.0f;
      p.stats[3 * m] = 0.0f, p.stats[3 * m + 1] = INFINITY, p.stats[3 * m + 2] = 0.0f;
    }
  };
  if (y < 0 || y >= p.V) {   // (all blocks of the cluster)
    if (crank == 0) nothing();
    return;
  }
  const float zy = tid == 0 && p.targets != nullptr ? to_f32<T>(row.z[y]) : 0.0f;
  LpSums* to = s_part;
  if (csize > 1) {
    to = cluster.map_shared_rank(s_part, 0);
    cluster.sync();   // rank 0, to which the others write, is there
  }
  const float scale = p.scale;
  LpSums x = lp_warp_join<true>(lp_slice<T, G>(row, t0, t1, scale, s_max), scale);
  if (lane == 0) to[crank * kWarps + warp] = x;
  if (csize > 1) {
    cluster.sync();
    if (crank > 0) return;
  } else {
    __syncthreads();
  }
  // the first warp joins the parts (at most 64), the others wait
  if (warp == 0) {
    x = lane < parts ? s_part[lane] : LpSums{-INFINITY, 0.0f, 0.0f};
    if (lane + 32 < parts) x = lp_join<true>(x, s_part[lane + 32], scale);
    x = lp_warp_join<true>(x, scale);
    if (lane == 0) s_row = x;
  }
  __syncthreads();
  x = s_row;
  const bool plain = lp_plain(x.m, scale);
  if (!plain) x = lp_far<T, NT>(row, scale, s_part);
  if (x.m == -INFINITY && x.s == x.s) return nothing();   // no logit above -inf
  const bool nan = !(x.s < INFINITY) || !(x.m < INFINITY);
  if (tid == 0) {
    const LpLog log(p, x.m, x.s);
    const float h = nan ? NAN : fmaxf(0.0f, (float)(log.log_s - (double)(x.a / x.s) * 0.69314718055994531));
    if (p.targets != nullptr) p.logp[m] = nan ? NAN : log.of(zy);
    p.entropy[m] = h;
    p.stats[3 * m] = nan ? NAN : x.m;
    p.stats[3 * m + 1] = nan ? NAN : x.s;
    p.stats[3 * m + 2] = h;
  }
}

constexpr int kLpTopWarps = 4;   // rows of a block

template <typename T, int G>
__global__ void __launch_bounds__(kLpTopWarps * 32) logprob_top_kernel(const __grid_constant__ LogprobParams p) {
  __shared__ LpLists s_lists[kLpTopWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t m = (int64_t)blockIdx.x * kLpTopWarps + warp;
  if (m >= p.M) return;
  const float high = p.stats[3 * m], sum = p.stats[3 * m + 1];
  if (sum == INFINITY) {   // the row does not count
    for (int i = lane; i < p.K; i += 32) p.ids[m * p.K + i] = -1, p.top[m * p.K + i] = 0.0f;
    return;
  }
  const LpRow<T> row(p.z, m, p.stride, (int)p.V);
  lp_top<T, G>(p, row, m, LpMaxima<T, G>(p, m), LpLog(p, high, sum), sum != sum, s_lists[warp]);
}

// Gradient: a warp takes U tiles of 32 vectors of a row and needs no other: it sums the row's
// entries of g itself, and the columns of its tiles with a g term it writes a second time.
constexpr int kLpBwdWarps = 8, kLpBwdTiles = 8;

template <typename T>
__global__ void __launch_bounds__(kLpBwdWarps * 32, 3) logprob_bwd_kernel(const __grid_constant__ LogprobParams p, uint32_t segs) {
  constexpr int N = LpVec<T>::N, P = N / 2, U = kLpBwdTiles;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * kLpBwdWarps + (threadIdx.x >> 5);
  const int64_t m = (uint32_t)unit / segs;   // (checked: below 2^32)
  if (m >= p.M) return;
  const int i0 = (int)((uint32_t)unit - (uint32_t)m * segs) * 32 * U;   // first vector
  // the gradient's row has the logits' alignment; its vectors, the columns behind V among them
  const LpRow<T> row(p.z, m, p.stride, (int)p.V);
  T* out = reinterpret_cast<T*>(p.dz) + m * p.gstride;
  const float high = p.stats[3 * m], sum = p.stats[3 * m + 1], h = p.stats[3 * m + 2];
  const int64_t y = p.gp != nullptr && p.targets != nullptr ? p.targets[m] : -1;
  const float gh = p.gh != nullptr ? p.gh[m] : 0.0f, gy = p.gp != nullptr ? p.gp[m] : 0.0f;
  // the first 32 alternatives, one a lane
  const bool mine = p.gt != nullptr && lane < p.K;
  const float gt = mine ? p.gt[m * p.K + lane] : 0.0f;
  const int64_t id = mine ? p.ids[m * p.K + lane] : -1;
  const bool counted = !(sum == INFINITY);
  LpVec<T> r[U];
  const bool inside = row.inside(i0, 32 * U);
  if (counted) {
#pragma unroll
    for (int j = 0; j < U; ++j) r[j] = inside ? row.load_whole(i0 + j * 32 + lane) : row.load(i0 + j * 32 + lane);
  }
  float g = gt;   // of all entries
  if (p.gt != nullptr) {
    for (int i = lane + 32; i < p.K; i += 32) g += p.gt[m * p.K + i];
    g = warp_sum(g);
  }
  // dz = p (c0 + c1 log2 p) + g terms
  const float l2 = log2f(sum);
  const float inv = (float)p.inv_tau;
  const float c0 = -(g + gy + gh * h) * inv, c1 = -gh * kLpLn2 * inv;
  const bool plain = lp_plain(high, p.scale);
  const float shift = lp_shift(high, p.scale);
  auto smooth = [&](float z) {
    const float t = plain ? fmaf(max_nan(z, kLpFloor), p.scale, shift) - l2 : max_nan((z - high) * p.scale - l2, -1000.0f);
    return lp_exp2(t) * fmaf(c1, t, c0);
  };
  if (inside && counted && plain) {
    const uint64_t sc = f2_pack(p.scale, p.scale), sh = f2_pack(shift, shift), l = f2_pack(-l2, -l2);
    const uint64_t d0 = f2_pack(c0, c0), d1 = f2_pack(c1, c1);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      uint64_t z[P];
      r[j].floored_pairs(z);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint64_t t = f2_add(f2_fma(z[i], sc, sh), l);
        float lo, hi;
        f2_unpack(t, lo, hi);
        z[i] = f2_mul(f2_pack(lp_exp2(lo), lp_exp2(hi)), f2_fma(d1, t, d0));
      }
      LpVec<T> o;
      o.set_pairs(z);
      reinterpret_cast<uint4*>(out - row.lead)[i0 + j * 32 + lane] = o.u;
    }
  } else {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int col = row.col(i0 + j * 32 + lane);
      if (col >= p.width) continue;
      float v[N];
      if (counted) r[j].values(v);
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
  }
  if (!counted) return;
  // columns with g terms: this warp's, once its vectors are written
  const int c_begin = max(0, row.col(i0)), c_end = row.col(i0 + 32 * U);
  bool hit = false;
  auto again = [&](int64_t c, float more) {
    hit = hit || c == y;
    if (c >= c_begin && c < c_end)
      out[c] = from_f32<T>(smooth(to_f32<T>(row.z[c])) + (more + (c == y ? gy : 0.0f)) * inv);
  };
  __syncwarp();
  if (p.gt != nullptr) {
    if (mine) again(id, gt);
    for (int i = lane + 32; i < p.K; i += 32) again(p.ids[m * p.K + i], p.gt[m * p.K + i]);
    hit = __any_sync(0xffffffffu, hit);
  }
  if (lane == 0 && !hit && y >= c_begin && y < c_end) out[y] = from_f32<T>(smooth(to_f32<T>(row.z[y])) + gy * inv);
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
  p.inv_tau = 1.0 / temperature;
  p.inv_scale = 1.0 / (double)p.scale;
  return p;
}

template <typename T, int NT, int G>
void lp_launch(LogprobParams& p, const at::Tensor& like, cudaStream_t stream) {
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  constexpr int N = LpVec<T>::N;
  const int64_t vecs = (p.V + 2 * N - 2) / N;   // at the worst alignment
  auto kern = logprob_fwd_kernel<T, NT, G>;
  // a cluster to a row where that leaves SMs without a block, down to 4 warp tiles a warp
  int csize = 1;
  while (csize < 8 && p.M * csize * 2 <= 2 * sms && vecs / (2 * csize) >= 4 * NT) csize *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.M * csize));
  cfg.blockDim = dim3(NT);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)csize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = csize > 1 ? 1 : 0;
  at::Tensor maxima;
  if constexpr (G > 0) {
    p.row_maxima = LpMaxima<T, G>::bytes((int)vecs);
    maxima = at::empty({p.M * p.row_maxima}, like.options().dtype(at::kByte));
    p.maxima = reinterpret_cast<uint8_t*>(maxima.data_ptr());
  }
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
  if constexpr (G > 0) {
    logprob_top_kernel<T, G><<<(unsigned)((p.M + kLpTopWarps - 1) / kLpTopWarps), kLpTopWarps * 32, 0, stream>>>(p);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
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
    // What a row costs beside its columns (a load before the first, joins) is latency: blocks of
    // 4 warps, or of one for short rows, leave more of them on an SM to cover it, where there are
    // rows for twice as many (4096 x 50257: 86 us with 8 warps, 78 with 4).
    const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    auto shape = [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      if (p.K == 0) lp_launch<T, NT, 0>(p, z, stream);
      else if (2 * (p.V / (4 * LpVec<T>::N)) >= 3 * p.K) lp_launch<T, NT, 4>(p, z, stream);
      else lp_launch<T, NT, 1>(p, z, stream);
    };
    if (p.V <= 4096 && p.M >= 4 * sms) shape(std::integral_constant<int, 32>{});
    else if (p.M >= 8 * sms) shape(std::integral_constant<int, 128>{});
    else shape(std::integral_constant<int, 256>{});
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
  const int64_t N = 16 / es, vecs = (p.width + 2 * N - 2) / N, segs = (vecs + 32 * kLpBwdTiles - 1) / (32 * kLpBwdTiles);
  TORCH_CHECK(p.M * segs < (1LL << 32) - kLpBwdWarps && p.width < (1LL << 30), "token_logprobs: too many rows or columns");
  const c10::cuda::CUDAGuard guard(z.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  ZQ_LP_TYPES(z.scalar_type(), {
    logprob_bwd_kernel<T><<<(unsigned)((p.M * segs + kLpBwdWarps - 1) / kLpBwdWarps), kLpBwdWarps * 32, 0, stream>>>(
        p, (uint32_t)segs);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
