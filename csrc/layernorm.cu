// Layer norm of rows of D columns, forward and backward, optionally after a residual
// addition and with its input kept in 8 bits for the backward.
//
//   h = x (+ delta, rounded to the type);  mu = mean h;  v = mean (h - mu)^2;
//   r = (v + eps)^-1/2;  n = (h - mu) r;  y = n w + b
// and with a = dy w (n from the kept h, which may be the 8-bit one):
//   dx = r (a - mean a - n mean(a n)) (+ dh);  dw = sum over rows dy n;  db = sum over rows dy
//
// Forward: a team of W warps takes one row at a time and holds it in registers, K tiles of 256
// columns a warp; w and b are in shared memory.  Backward: a team takes two rows at a time, holds
// their sums and those of dw and db, and reads the rows twice from shared memory.  Teams go over
// the rows with a fixed stride, and the loads of the next row are under way while this one is
// reduced.  A mean that is large next to the deviation costs nothing but its own roundings: a warp's
// sums are of differences from its first value, the row's mean is formed by differences from the
// first warp's, and n by subtracting before r is multiplied (r h - r mu rounds r mu: n = 0.08 in a
// row of 10000).  A row of one value has n = 0.  The variance is the joined sum of squares about
// each warp's own mean (columns n_i, mean m_i, squares q_i: q = sum q_i + n_i (m_i - mu)^2), so
// one exchange gives both and nothing cancels.  dw and db: a block's teams add up in team order in
// shared memory, the blocks' rows of partial sums are added in block order by a second kernel: no
// atomics.
//
// What bounds it: memory in the plain forward (8192 x 3584 with residual 39 us, 0.92 of a copy's
// rate); arithmetic and the latency of reductions and barriers with codes (16384 x 5120: 106 us,
// 0.61) and in the backward (52 us, 0.70, and 112 us from codes, 0.57), at half to two thirds of the
// issue slots and no pipe above 0.46.
// Rows that are not whole 16-byte vectors go by single elements and without rows under way: 16384 x
// 5003 bf16 111 us forward (0.45), 289 backward (0.26), with codes 224 and 395 (0.28, 0.16).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>

#include "rows.cuh"

namespace zq {

constexpr int kLnMaxWarps = 16;     // of a team
constexpr int kLnBlockWarps = 24;   // of a block at most: 80 registers a thread (20: 96, 16: 128)
constexpr int kLnMaxTeams = kLnBlockWarps / 2;   // of several warps

struct LnParams {
  const void *x, *delta, *dy, *dh;   // rows of pitch xs, ds, dys, dhs
  int64_t xs, ds, dys, dhs;
  void *h, *y, *dx;                  // dense
  const void *w, *b;                 // type wt: 0 fp32, 1 bf16, 2 fp16
  float *mean, *rstd;                // [M]
  int8_t* codes;                     // [M, P], or null
  float* steps;                      // [M, G]
  float* part;                       // [grid, 2, D]
  int64_t M, P, G;
  int D, wt, W, R;                   // warps of a team, teams of a block
  int slots, slots_at;               // groups of rows under way in shared memory, where they begin
  const void* src[3];                // the tensors that go through it, in the kernel's order
  int64_t pitch[3];
  float eps;
};

__device__ __forceinline__ float ln_param(const void* p, int type, int i) {
  if (type == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (type == 2) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}

// w or b in shared memory, in 32 bits and in the lanes' order (a lane's 8 columns of a tile in
// two runs of 4, so that a warp's 16-byte reads fall on different banks)
template <bool VEC>
__device__ __forceinline__ int ln_place(int c) {   // of column c
  const int i = c & (kTile - 1);
  return VEC ? (c - i) + ((i >> 2) & 1) * 128 + (i >> 3) * 4 + (i & 3) : c;
}
template <bool VEC>
__device__ __forceinline__ void ln_stage(float* s, const void* p, int type, float absent, int D) {
  const int whole = (D + kTile - 1) / kTile * kTile;
  // four columns at a time; a run of four stays one
  if (p != nullptr && type == 0 && D % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const float4* v = reinterpret_cast<const float4*>(p);
#pragma unroll 4
    for (int c = threadIdx.x * 4; c < whole; c += blockDim.x * 4) {
      const float4 f = c < D ? __ldg(v + c / 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      *reinterpret_cast<float4*>(s + ln_place<VEC>(c)) = f;
    }
    return;
  }
#pragma unroll 4
  for (int c = threadIdx.x; c < whole; c += blockDim.x)
    s[ln_place<VEC>(c)] = c >= D ? 0.0f : p == nullptr ? absent : ln_param(p, type, c);
}
template <bool VEC>
__device__ __forceinline__ void ln_staged(const float* s, int base, int lane, uint64_t (&v)[4]) {
  if constexpr (VEC) {
    const float4 a = *reinterpret_cast<const float4*>(s + base + lane * 4);
    const float4 b = *reinterpret_cast<const float4*>(s + base + 128 + lane * 4);
    v[0] = f2_pack(a.x, a.y), v[1] = f2_pack(a.z, a.w), v[2] = f2_pack(b.x, b.y), v[3] = f2_pack(b.z, b.w);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f2_pack(s[base + 64 * i + lane], s[base + 64 * i + 32 + lane]);
  }
}

__device__ __forceinline__ float f2_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

// A lane's mask of values that are columns of the row.
template <bool VEC>
__device__ __forceinline__ uint32_t ln_mask(int base, int lane, int D) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m |= (base + tile_col<VEC>(lane, i) < D ? 1u : 0u) << i;
  return m;
}

// Every warp's pair of numbers, lane i getting warp i's (0 past the last).  Buffers alternate
// from row to row: a thread that writes one again has passed the other's barrier, to which its
// readers came after they had read.
__device__ __forceinline__ float2 ln_exchange(float2 (&buf)[kLnMaxWarps], float2 mine, int wt, int lane, int team, int W) {
  if (lane == 0) buf[wt] = mine;
  named_barrier(1 + team, W * 32);
  return lane < W ? buf[lane] : make_float2(0.0f, 0.0f);
}
// the sum of the first 16 lanes' values, in every lane
__device__ __forceinline__ float ln_sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return __shfl_sync(0xffffffffu, v, 0);
}

// Rows on their way: every warp copies its own columns of NS tensors of T (and, CODES, of the 8-bit
// input, STATS, the row's mean and deviation) into its own places of shared memory, S groups of
// rows ahead, and reads them back itself, so no barrier belongs to it and nothing waits in
// registers.  A lane copies its own vectors; codes go 16 bytes a lane, the few single numbers by a
// few lanes (copies of 4 and 8 bytes by all of them took as long as the vectors).
template <typename T, int K, int NS, bool CODES, bool STATS>
struct LnSlots {
  static constexpr int kVecs = (int)sizeof(T) / 2;   // 16-byte vectors of a lane's 8 elements
  static constexpr int kBytes = K * (16 * kVecs * NS + (CODES ? 8 : 0)) + (CODES || STATS ? 4 : 0);   // of a thread
  uint32_t mine;       // shared address of this thread's vectors in the first slot
  uint32_t slot_bytes; // from slot to slot
  uint32_t there;      // bit k: tile k has columns here
  int first;           // the warp's first column

  // A warp's places in a slot: [tensor][tile][vector][lane] of 16 bytes; codes [tile][256]; numbers:
  // steps [tile][2], mean, deviation.
  static constexpr int kCodes = 512 * K * kVecs * NS, kNumbers = kCodes + (CODES ? 256 * K : 0), kStats = CODES ? 2 * K : 0;
  static __device__ __forceinline__ uint32_t vec(int i) { return 512u * i; }
  static __device__ __forceinline__ int lane() { return threadIdx.x & 31; }
  __device__ __forceinline__ uint32_t number(int i) const { return kNumbers + 4u * i - 16u * lane(); }

  __device__ __forceinline__ void init(uint8_t* smem, const LnParams& p, int first_, int n) {
    first = first_;
    there = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) there |= (first + lane() * 8 + k * p.W * kTile < p.D ? 1u : 0u) << k;
    mine = smem_u32(smem) + (threadIdx.x >> 5) * (32u * kBytes) + 16u * lane();
    slot_bytes = (uint32_t)kBytes * blockDim.x;
    if (first + ((K - 1) * p.W + 1) * kTile > p.D) {   // places that are never filled hold zeros
      for (int s = 0; s < n; ++s) {
        const uint32_t at = mine + s * slot_bytes;
#pragma unroll
        for (int i = 0; i < NS * K * kVecs; ++i)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + vec(i)), "r"(0) : "memory");
        if constexpr (CODES) {
#pragma unroll
          for (int k = 0; k < K; ++k)
            asm volatile("st.shared.v2.b32 [%0], {%1, %1};" ::"r"(at + kCodes + 256u * k - 8u * lane()), "r"(0) : "memory");
          if (lane() < 2 * K) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + number(lane())), "r"(0) : "memory");
        }
      }
      __syncwarp();
    }
  }
  // fetches rows [row, row + B) of M into slots [group B, group B + B), as one group of copies
  template <int B>
  __device__ __forceinline__ void fetch(const LnParams& p, int group, int64_t first_row) const {
    if constexpr (CODES || STATS) __syncwarp();   // (the slots are read)
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const uint32_t at = mine + (group * B + b) * slot_bytes;
      const int64_t row = first_row + b;
      if (row >= p.M) continue;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const T* from = reinterpret_cast<const T*>(p.src[i]) + row * p.pitch[i] + first + lane() * 8;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int v = 0; v < kVecs; ++v)
            if (there >> k & 1u)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + vec((i * K + k) * kVecs + v)),
                           "l"(from + k * p.W * kTile + v * (16 / (int)sizeof(T)))
                           : "memory");
      }
      if constexpr (CODES) {
        const int8_t* codes = p.codes + row * p.P + first + lane() * 16;
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (lane() < 16 && first + k * p.W * kTile + lane() * 16 < p.D)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + kCodes + 256u * k), "l"(codes + k * p.W * kTile)
                         : "memory");
      }
      if constexpr (CODES || STATS) {
        const int group_at = (first + (lane() >> 1) * p.W * kTile) / kGroup + (lane() & 1);   // of the lane's step
        const float* from = nullptr;
        if (CODES && lane() < 2 * K && group_at < p.G) from = p.steps + row * p.G + group_at;
        if (STATS && lane() == kStats) from = p.mean + row;
        if (STATS && lane() == kStats + 1) from = p.rstd + row;
        if (from != nullptr)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at + number(lane())), "l"(from) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void get_stats(int slot, float& mu, float& r) const {
    const uint32_t at = mine + slot * slot_bytes;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(mu) : "r"(at + number(kStats)) : "memory");
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(at + number(kStats + 1)) : "memory");
  }
  // until all but the last S - 1 fetches are there
  static __device__ __forceinline__ void wait(int S) {
    if (S == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (S == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else asm volatile("cp.async.wait_group 3;" ::: "memory");
    if constexpr (CODES || STATS) __syncwarp();   // other lanes' copies
  }
  __device__ __forceinline__ void get(int slot, int i, int k, RawTile<T, true>& t) const {
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(t.w[4 * v]), "=r"(t.w[4 * v + 1]), "=r"(t.w[4 * v + 2]), "=r"(t.w[4 * v + 3])
                   : "r"(mine + slot * slot_bytes + vec((i * K + k) * kVecs + v))
                   : "memory");
  }
  __device__ __forceinline__ void get(int slot, int k, RawCodes<true>& c) const {
    const uint32_t at = mine + slot * slot_bytes;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(c.w.x), "=r"(c.w.y) : "r"(at + kCodes + 256u * k - 8u * lane()) : "memory");
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(c.step[0]) : "r"(at + number(2 * k + (lane() >> 4))) : "memory");
  }
};

// PIPE: rows come through shared memory; otherwise (not on 16-byte boundaries, or too wide for
// two of them) they are read where they are.  KEEP: h is kept in 8 bits.
template <typename T, bool VEC, int K, bool RES, bool KEEP, bool PIPE>
__global__ void __launch_bounds__(kLnMaxWarps * 32) ln_fwd_kernel(const __grid_constant__ LnParams p) {
  __shared__ float2 s_red[kLnMaxTeams][2][kLnMaxWarps];
  extern __shared__ __align__(16) float s_wb[];   // w and b; the slots
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int W = p.W, team = warp / W, wt = warp - team * W, D = p.D, S = p.slots;
  const int whole = (D + kTile - 1) / kTile * kTile;
  const int64_t step = (int64_t)gridDim.x * p.R;
  int64_t row = (int64_t)blockIdx.x * p.R + team;
  LnSlots<T, K, RES ? 2 : 1, false, false> rows;
  if constexpr (PIPE) {
    rows.init(reinterpret_cast<uint8_t*>(s_wb) + p.slots_at, p, wt * kTile, S);
    for (int i = 0; i < S; ++i) rows.template fetch<1>(p, i, row + i * step);
  }
  ln_stage<VEC>(s_wb, p.w, p.wt, 1.0f, D);
  ln_stage<VEC>(s_wb + whole, p.b, p.wt, 0.0f, D);
  // columns of warp i of a team, in lane i; of this warp
  auto columns = [&](int i) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) n += max(0, min(kTile, D - (i + k * W) * kTile));
    return (float)n;
  };
  const float cols = columns(wt), cols_of = columns(lane), inv_cols = cols > 0.0f ? 1.0f / cols : 0.0f, inv_d = 1.0f / (float)D;
  __syncthreads();
  int at = 0;
  for (int turn = 0; row < p.M; row += step, turn ^= 1) {
    uint64_t v[K][4];
    if constexpr (PIPE) rows.wait(S);
    auto tile = [&](int stream, const void* from, int64_t pitch, int k, uint64_t (&u)[4]) {
      RawTile<T, VEC> t;
      if constexpr (PIPE) rows.get(at, stream, k, t);
      else t.load(reinterpret_cast<const T*>(from) + row * pitch, (wt + k * W) * kTile, lane, D);
      t.pairs(u);
    };
    auto read = [&](bool again) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        tile(0, p.x, p.xs, k, v[k]);
        if constexpr (RES) {
          const int base = (wt + k * W) * kTile;
          RawTile<T, VEC> t;
          uint64_t d[4];
          tile(1, p.delta, p.ds, k, d);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[k][i] = f2_add(v[k][i], d[i]);
          t.set(v[k]);
          if (!again && base < D) t.store(reinterpret_cast<T*>(p.h) + row * D, base, lane, D);
          t.pairs(v[k]);   // as the next layer and the backward see it
        }
      }
    };
    read(false);
    if constexpr (KEEP) {
      int8_t* c[K];
      float* t[K];
      int base[K];
#pragma unroll
      for (int k = 0; k < K; ++k) c[k] = p.codes + row * p.P, t[k] = p.steps + row * p.G, base[k] = (wt + k * W) * kTile;
      keep_tiles<VEC, K>(v, c, t, base, lane, D);
    }
    // The warp's mean and its sum of squares about it, from differences from its first value, which are
    // small or exact: one pass and one reduction.  q = sum d^2 - n (mean d)^2 cancels, and differences
    // are rounded as that value is, where it lies far out; from 2.8 deviations on once more, from the
    // mean and the row read again, so that the 22 roundings of a sum weigh 9-fold at most (16384 x 5120
    // kept in 8 bits: 107 us from 2 deviations on, 104 from 5.5).  v: the differences.  (Read again from
    // its slot, filled anew behind this only; from memory, with the slot given up before: 110 us.)
    float mu, q, from, rest;
    f2_unpack(v[0][0], from, rest);
    from = __shfl_sync(0xffffffffu, from, 0);
    float away = -from;
    for (bool again = false;; again = true) {
      const uint64_t away2 = f2_pack(away, away);
      uint64_t s2 = 0ull, q2 = 0ull;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int base = (wt + k * W) * kTile;
        if (base + kTile <= D) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[k][i] = f2_add(v[k][i], away2);
        } else if (base < D) {   // the row ends in this tile: 0 behind it
          const uint32_t mask = ln_mask<VEC>(base, lane, D);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a, b;
            f2_unpack(f2_add(v[k][i], away2), a, b);
            v[k][i] = f2_pack(mask >> (2 * i) & 1u ? a : 0.0f, mask >> (2 * i + 1) & 1u ? b : 0.0f);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s2 = f2_add(s2, v[k][i]);
          q2 = f2_fma(v[k][i], v[k][i], q2);
        }
      }
      const float d = warp_sum(f2_sum(s2)) * inv_cols, nd2 = cols * d * d;
      q = warp_sum(f2_sum(q2)) - nd2;
      mu = from + d;
      if (again || nd2 <= 8.0f * q) break;   // (sums beyond 32 bits, too: infinity - infinity is NaN)
      read(true);
      away = -mu;
      from = mu;
    }
    q = max_nan(q, 0.0f);
    if constexpr (PIPE) {   // the slot is read
      rows.template fetch<1>(p, at, row + S * step);
      at = at + 1 == S ? 0 : at + 1;
    }
    if (W > 1) {
      const float2 o = ln_exchange(s_red[team][turn], make_float2(mu, q), wt, lane, team, W);
      const float first = __shfl_sync(0xffffffffu, o.x, 0);   // (again from differences)
      mu = fmaf(ln_sum16(lane < W ? cols_of * (o.x - first) : 0.0f), inv_d, first);
      const float d = o.x - mu;
      q = ln_sum16(lane < W ? fmaf(cols_of * d, d, o.y) : 0.0f);
    }
    const float r = rsqrtf(fmaf(q, inv_d, p.eps));
    if (wt == 0 && lane == 0 && p.mean != nullptr) p.mean[row] = mu, p.rstd[row] = r;
    const float off = (from - mu) * r;   // (of a few deviations' size)
    const uint64_t off2 = f2_pack(off, off), r2 = f2_pack(r, r);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int base = (wt + k * W) * kTile;
      if (base >= D) continue;
      uint64_t w[4], b[4];
      ln_staged<VEC>(s_wb, base, lane, w);
      ln_staged<VEC>(s_wb + whole, base, lane, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k][i] = f2_fma(f2_fma(v[k][i], r2, off2), w[i], b[i]);
      RawTile<T, VEC> y;
      y.set(v[k]);
      y.store(reinterpret_cast<T*>(p.y) + row * D, base, lane, D);
    }
  }
}

// KEPT: h in 8 bits; RES: dh is added.  A team takes two consecutive rows at a time, which share
// the reductions' barrier and latencies.  A row is read twice (through shared memory, or from the
// caches): for its sums, and for dx once they are known; there are no registers to hold it.
constexpr int kLnRows = 2;
template <typename T, bool VEC, int K, bool KEPT, bool RES, bool PIPE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) ln_bwd_kernel(const __grid_constant__ LnParams p) {
  constexpr int B = kLnRows;
  __shared__ float s_red[kLnMaxTeams][2][kLnMaxWarps][2 * B];
  extern __shared__ __align__(16) float s_wb[];   // w, at the end [2, D]: teams add up; the slots
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int W = p.W, team = warp / W, wt = warp - team * W, D = p.D, S = p.slots;
  const int64_t step = (int64_t)gridDim.x * p.R * B;
  int64_t row = ((int64_t)blockIdx.x * p.R + team) * B;
  constexpr int kH = 1, kX = RES ? 2 : 1;   // tensors behind dy
  LnSlots<T, K, 1 + (RES ? 1 : 0) + (KEPT ? 0 : 1), KEPT, true> rows;
  if constexpr (PIPE) {
    rows.init(reinterpret_cast<uint8_t*>(s_wb) + p.slots_at, p, wt * kTile, S * B);
    for (int i = 0; i < S; ++i) rows.template fetch<B>(p, i, row + i * step);
  }
  ln_stage<VEC>(s_wb, p.w, p.wt, 1.0f, D);
  uint64_t dw[K][4], db[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[k][i] = db[k][i] = 0ull;
  const float inv_d = 1.0f / (float)D;
  __syncthreads();

  int at = 0;   // the rows' group of slots
  for (int turn = 0; row < p.M; row += step, turn ^= 1) {
    const bool second = row + 1 < p.M;
    float mu[B], r[B];
    if constexpr (PIPE) {   // (of a second row that is not there: not used)
      rows.wait(S);
      rows.get_stats(at * B, mu[0], r[0]);
      rows.get_stats(at * B + 1, mu[1], r[1]);
    } else {
      mu[0] = p.mean[row], r[0] = p.rstd[row];
      mu[1] = second ? p.mean[row + 1] : 0.0f, r[1] = second ? p.rstd[row + 1] : 0.0f;
    }
    auto gradient = [&](const void* from, int64_t pitch, int stream, int b, int k, uint64_t (&g)[4]) {
      RawTile<T, VEC> t;
      if constexpr (PIPE) rows.get(at * B + b, stream, k, t);
      else t.load(reinterpret_cast<const T*>(from) + (row + b) * pitch, (wt + k * W) * kTile, lane, D);
      t.pairs(g);
    };
    auto away = [&](int b, int k, uint64_t (&d)[4]) {   // h - mu
      const int base = (wt + k * W) * kTile;
      if constexpr (KEPT) {
        RawCodes<VEC> c;
        if constexpr (PIPE) rows.get(at * B + b, k, c);
        else c.load(p.codes + (row + b) * p.P, p.steps + (row + b) * p.G, base, lane, D);
        c.away(mu[b], d);
      } else {
        RawTile<T, VEC> t;
        if constexpr (PIPE) rows.get(at * B + b, kX, k, t);
        else t.load(reinterpret_cast<const T*>(p.x) + (row + b) * p.xs, base, lane, D);
        t.pairs(d);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = f2_add(d[i], f2_pack(-mu[b], -mu[b]));
      }
    };
    float s[2 * B];   // sums of a and a (h - mu) of each row
    {
      uint64_t t[2 * B];
#pragma unroll
      for (int i = 0; i < 2 * B; ++i) t[i] = 0ull;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int base = (wt + k * W) * kTile;
        if (base >= D) continue;
        uint64_t w[4];
        ln_staged<VEC>(s_wb, base, lane, w);
#pragma unroll
        for (int b = 0; b < B; ++b) {
          if (b > 0 && !second) continue;
          uint64_t g[4], d[4];
          gradient(p.dy, p.dys, 0, b, k, g);
          away(b, k, d);
          const uint64_t r2 = f2_pack(r[b], r[b]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {   // (past the row's end dy and w are 0)
            dw[k][i] = f2_fma(g[i], f2_mul(d[i], r2), dw[k][i]);
            db[k][i] = f2_add(db[k][i], g[i]);
            g[i] = f2_mul(g[i], w[i]);
            t[2 * b] = f2_add(t[2 * b], g[i]);
            t[2 * b + 1] = f2_fma(g[i], d[i], t[2 * b + 1]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * B; ++i) s[i] = f2_sum(t[i]);
    }
    // Four sums over a warp: lanes swap what they do not go on with, so that lane i ends with
    // number i & 3; then over the team.
    static_assert(B == 2, "four sums");
    float v;
    {
      const bool odd = lane & 1, high = lane & 2;
      const float a = (odd ? s[1] : s[0]) + __shfl_xor_sync(0xffffffffu, odd ? s[0] : s[1], 1);
      const float c = (odd ? s[3] : s[2]) + __shfl_xor_sync(0xffffffffu, odd ? s[2] : s[3], 1);
      v = (high ? c : a) + __shfl_xor_sync(0xffffffffu, high ? a : c, 2);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    if (W > 1) {   // (buffers in turn: see ln_exchange)
      float(&buf)[kLnMaxWarps][2 * B] = s_red[team][turn];
      if (lane < 2 * B) buf[wt][lane] = v;
      named_barrier(1 + team, W * 32);
      v = 0.0f;
#pragma unroll
      for (int i = 0; i < kLnMaxWarps; i += 8) {
        const int from = i + (lane >> 2);
        if (from < W) v += buf[from][lane & 3];
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
#pragma unroll
    for (int i = 0; i < 2 * B; ++i) s[i] = __shfl_sync(0xffffffffu, v, i) * inv_d;
    // dx = r a - r mean a - (h - mu) r^2 mean(a n)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int base = (wt + k * W) * kTile;
      if (base >= D) continue;
      uint64_t w[4];
      ln_staged<VEC>(s_wb, base, lane, w);
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (b > 0 && !second) continue;
        const float c0 = -r[b] * s[2 * b], c1 = -r[b] * (r[b] * (r[b] * s[2 * b + 1]));
        const uint64_t c02 = f2_pack(c0, c0), c12 = f2_pack(c1, c1), r2 = f2_pack(r[b], r[b]);
        uint64_t g[4], d[4];
        gradient(p.dy, p.dys, 0, b, k, g);
        away(b, k, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = f2_fma(f2_mul(g[i], w[i]), r2, f2_fma(d[i], c12, c02));
        if constexpr (RES) {
          uint64_t h[4];
          gradient(p.dh, p.dhs, kH, b, k, h);
#pragma unroll
          for (int i = 0; i < 4; ++i) g[i] = f2_add(g[i], h[i]);
        }
        RawTile<T, VEC> o;
        o.set(g);
        o.store(reinterpret_cast<T*>(p.dx) + (row + b) * D, base, lane, D);
      }
    }
    if constexpr (PIPE) {   // the slots are read: the rows S groups behind these
      rows.template fetch<B>(p, at, row + S * step);
      at = at + 1 == S ? 0 : at + 1;
    }
  }
  if (p.part == nullptr) return;
  float* out = p.part + (int64_t)blockIdx.x * 2 * D;
  for (int j = 0; j < p.R; ++j) {
    __syncthreads();
    if (team != j) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = (wt + k * W) * kTile + tile_col<VEC>(lane, i);
        if (c < D) {
          float a, b, u, v;
          f2_unpack(dw[k][i / 2], a, b);
          u = i & 1 ? b : a;
          f2_unpack(db[k][i / 2], a, b);
          v = i & 1 ? b : a;
          if (j > 0) u += s_wb[c], v += s_wb[D + c];
          if (j == p.R - 1) out[c] = u, out[D + c] = v;
          else s_wb[c] = u, s_wb[D + c] = v;
        }
      }
    }
  }
}

// Sums of the blocks' partial rows: 32 columns a block, its 16 warps take rows in turn and
// are added in warp order.
constexpr int kLnSumWarps = 16;
template <typename T>
__global__ void __launch_bounds__(kLnSumWarps * 32) ln_sum_kernel(const float* __restrict__ part, int rows, int D,
                                                                  T* __restrict__ dw, T* __restrict__ db) {
  __shared__ float s[kLnSumWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;   // of dw and db behind one another
  float v = 0.0f;
  if (c < 2 * D)
#pragma unroll 8
    for (int i = warp; i < rows; i += kLnSumWarps) v += part[(int64_t)i * 2 * D + c];
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < 2 * D) {
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < kLnSumWarps; ++i) v += s[i][lane];
    if (c < D) {
      if (dw != nullptr) dw[c] = from_f32<T>(v);
    } else if (db != nullptr) {
      db[c - D] = from_f32<T>(v);
    }
  }
}

}  // namespace zq

using namespace zq;

namespace {

int64_t ln_rows(const at::Tensor& t, const at::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == like.get_device() && t.dim() == 2 && t.sizes() == like.sizes() &&
                  t.scalar_type() == like.scalar_type() && (t.stride(1) == 1 || t.size(1) == 1),
              "layer_norm: ", what, " must be [M, D] like the input, unit column stride");
  return t.stride(0);
}

bool ln_aligned(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 &&
         (t.size(0) < 2 || t.stride(0) * t.element_size() % 16 == 0);
}

void ln_vector(const at::Tensor& t, const at::Tensor& x, at::ScalarType type, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == x.get_device() && t.is_contiguous() && t.numel() == x.size(1) &&
                  t.scalar_type() == type,
              "layer_norm: ", what, " must be [D] on the input's device, contiguous, of the weight's type");
}

LnParams ln_base(const at::Tensor& x, const c10::optional<at::Tensor>& w, const c10::optional<at::Tensor>& b, bool& vec) {
  LnParams p = {};
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(0) > 0 && x.size(1) > 0, "layer_norm: [M, D] on the GPU");
  p.M = x.size(0);
  const int64_t D = x.size(1);
  TORCH_CHECK(D <= 4 * kLnMaxWarps * kTile, "layer_norm: at most ", 4 * kLnMaxWarps * kTile, " columns, got ", D);
  p.D = (int)D;
  p.P = (D + 15) / 16 * 16;
  p.G = (D + kGroup - 1) / kGroup;
  at::ScalarType wt = at::kFloat;
  if (w.has_value()) wt = w->scalar_type();
  else if (b.has_value()) wt = b->scalar_type();
  TORCH_CHECK(wt == at::kFloat || wt == at::kBFloat16 || wt == at::kHalf, "layer_norm: weight and bias in fp32, bf16 or fp16");
  if (w.has_value()) ln_vector(*w, x, wt, "weight"), p.w = w->data_ptr();
  if (b.has_value()) ln_vector(*b, x, wt, "bias"), p.b = b->data_ptr();
  p.wt = wt == at::kFloat ? 0 : wt == at::kBFloat16 ? 1 : 2;
  vec = D % 8 == 0;
  return p;
}

void ln_kept(LnParams& p, const at::Tensor& x, const at::Tensor& codes, const at::Tensor& steps) {
  TORCH_CHECK(codes.is_cuda() && codes.get_device() == x.get_device() && codes.scalar_type() == at::kChar &&
                  codes.is_contiguous() && codes.numel() == p.M * p.P && steps.is_cuda() &&
                  steps.get_device() == x.get_device() && steps.scalar_type() == at::kFloat && steps.is_contiguous() &&
                  steps.numel() == p.M * p.G && (reinterpret_cast<uintptr_t>(codes.data_ptr()) & 15) == 0,
              "layer_norm: codes int8 [M, D up to 16s], steps fp32 [M, D / 128]");
  p.codes = codes.data_ptr<int8_t>();
  p.steps = steps.data_ptr<float>();
}

void ln_stats(LnParams& p, const at::Tensor& x, const at::Tensor& stats) {
  TORCH_CHECK(stats.is_cuda() && stats.get_device() == x.get_device() && stats.scalar_type() == at::kFloat &&
                  stats.is_contiguous() && stats.numel() == 2 * p.M,
              "layer_norm: statistics fp32 [2, M]");
  p.mean = stats.data_ptr<float>();
  p.rstd = p.mean + p.M;
}

// Tiles of a warp, warps of a team.  What a row costs beside its columns - reductions, a
// barrier, addresses - is shared by a warp's tiles: four in the forward (16384 x 5120 kept in 8
// bits with two: 136 us); in the backward, whose sums of dw and db take the registers, two and
// two rows, and four where 16 warps do not reach.
int ln_shape(LnParams& p, int most) {
  const int tiles = (p.D + kTile - 1) / kTile;
  const int K = tiles <= 2 ? tiles : tiles <= most * kLnMaxWarps ? most : 4;
  p.W = (tiles + K - 1) / K;
  return K;
}

// Teams of a block, as many as `warps` hold, fewer where there are no rows for them, and groups of
// `rows` rows under way in shared memory behind `front` bytes: 2 to 4, as many as leave `blocks`
// blocks to an SM; fewer blocks, then fewer teams, where two do not fit.  Returns the bytes in
// all, 0 where not even one team has room for two groups.
//   The backward has one block of many teams to an SM (w and a block's row of partial sums are
// there once), the forward three small ones (its warps have more registers that way: 8192 x 3584
// with residual 38 us against 46).
size_t ln_block(LnParams& p, size_t front, size_t thread_bytes, int warps, int rows, int blocks) {
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount, groups = (p.M + rows - 1) / rows;
  const size_t fixed = 1024 + sizeof(float) * kLnMaxTeams * 2 * kLnMaxWarps * 4;   // (the system's, the static arrays)
  p.slots_at = (int)front;
  p.slots = 0;
  for (p.R = (int)std::max<int64_t>(1, std::min<int64_t>(warps / p.W, (groups + sms - 1) / sms)); p.R > 0; --p.R) {
    const size_t slot = thread_bytes * p.W * p.R * 32 * rows;
    for (int n = blocks; n > 0; --n) {
      const size_t room = (size_t)(228 * 1024) / n - fixed;
      if (front + 2 * slot > room) continue;
      p.slots = (int)std::min<size_t>(4, (room - front) / slot);
      return front + p.slots * slot;
    }
  }
  p.R = 1;
  return 0;
}

// Teams of a block without slots: as many as 16 warps hold, and rows are there for
int ln_teams(const LnParams& p, int rows) {
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount, groups = (p.M + rows - 1) / rows;
  return (int)std::max<int64_t>(1, std::min<int64_t>(kLnMaxWarps / p.W, (groups + sms - 1) / sms));
}

// Blocks that are resident at once (a kernel's, by its shape), no more than there are rows for
template <typename F>
unsigned ln_grid(F kern, const LnParams& p, size_t smem, int rows) {
  int n = 0;
  if (smem > 32 * 1024)   // (48 KB with the static arrays go without)
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, p.W * p.R * 32, smem));
  TORCH_CHECK(n > 0, "layer_norm: a block does not fit the device");
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  return (unsigned)std::min<int64_t>((p.M + p.R * rows - 1) / (p.R * rows), n * sms);
}

}  // namespace

#define ZQ_LN_TYPES(TYPE, ...)                                                 \
  switch (TYPE) {                                                              \
    case at::kBFloat16: { using T = __nv_bfloat16; __VA_ARGS__; break; }       \
    case at::kHalf: { using T = __half; __VA_ARGS__; break; }                  \
    case at::kFloat: { using T = float; __VA_ARGS__; break; }                  \
    default: TORCH_CHECK(false, "layer_norm: bf16, fp16 or fp32");             \
  }

template <typename F>
static void ln_flags(bool a, bool b, F f) {
  const std::true_type yes;
  const std::false_type no;
  if (a && b) f(yes, yes);
  else if (a) f(yes, no);
  else if (b) f(no, yes);
  else f(no, no);
}

template <typename T, bool VEC, int K>
static void ln_fwd_launch(LnParams& p, cudaStream_t stream) {
  const size_t front = (size_t)2 * ((p.D + kTile - 1) / kTile * kTile) * 4;   // w and b
  auto go = [&](auto kern, size_t smem) {
    const unsigned grid = ln_grid(kern, p, smem, 1);
    kern<<<grid, p.W * p.R * 32, smem, stream>>>(p);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  };
  ln_flags(p.delta != nullptr, p.codes != nullptr, [&](auto res, auto keep) {
    constexpr bool RES = decltype(res)::value, KEEP = decltype(keep)::value;
    if constexpr (VEC) {
      p.src[0] = p.x, p.pitch[0] = p.xs;
      p.src[1] = p.delta, p.pitch[1] = p.ds;
      const size_t smem = ln_block(p, front, LnSlots<T, K, RES ? 2 : 1, false, false>::kBytes, 8, 1, 3);
      if (smem > 0) return go(ln_fwd_kernel<T, VEC, K, RES, KEEP, true>, smem);
    }
    if constexpr (!VEC || K == 4) {
      p.R = VEC ? 1 : ln_teams(p, 1);
      go(ln_fwd_kernel<T, VEC, K, RES, KEEP, false>, front);
    }
  });
}

// h and y [M, D]; stats [2, M] (mean, 1 / deviation), codes and steps where a backward follows
void layernorm_fwd(at::Tensor x, c10::optional<at::Tensor> delta, c10::optional<at::Tensor> w, c10::optional<at::Tensor> b,
                   c10::optional<at::Tensor> h, at::Tensor y, c10::optional<at::Tensor> stats,
                   c10::optional<at::Tensor> codes, c10::optional<at::Tensor> steps, double eps) {
  bool vec;
  LnParams p = ln_base(x, w, b, vec);
  p.eps = (float)eps;
  p.x = x.data_ptr();
  p.xs = ln_rows(x, x, "x");
  vec = vec && ln_aligned(x);
  if (delta.has_value()) {
    p.delta = delta->data_ptr();
    p.ds = ln_rows(*delta, x, "delta");
    TORCH_CHECK(h.has_value() && h->is_contiguous(), "layer_norm: h is contiguous");
    ln_rows(*h, x, "h");
    p.h = h->data_ptr();
    vec = vec && ln_aligned(*delta) && ln_aligned(*h);
  }
  ln_rows(y, x, "y");
  TORCH_CHECK(y.is_contiguous(), "layer_norm: y is contiguous");
  p.y = y.data_ptr();
  vec = vec && ln_aligned(y);
  if (stats.has_value()) ln_stats(p, x, *stats);
  if (codes.has_value()) ln_kept(p, x, *codes, *steps);
  const c10::cuda::CUDAGuard guard(x.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int K = ln_shape(p, 4);
  ZQ_LN_TYPES(x.scalar_type(), {
    if (vec) {
      if (K == 1) ln_fwd_launch<T, true, 1>(p, stream);
      else if (K == 2) ln_fwd_launch<T, true, 2>(p, stream);
      else ln_fwd_launch<T, true, 4>(p, stream);
    } else {
      if (K == 1) ln_fwd_launch<T, false, 1>(p, stream);
      else if (K == 2) ln_fwd_launch<T, false, 2>(p, stream);
      else ln_fwd_launch<T, false, 4>(p, stream);
    }
  });
}

template <typename T, bool VEC, int K>
static void ln_bwd_launch(LnParams& p, const at::Tensor& dy, c10::optional<at::Tensor>& dw, c10::optional<at::Tensor>& db,
                          cudaStream_t stream) {
  const bool sums = dw.has_value() || db.has_value();
  // w; [2, D] where teams' sums are added
  const size_t row = (size_t)((p.D + kTile - 1) / kTile * kTile) * 4, front = sums && p.W <= kLnBlockWarps / 2 ? 2 * row : row;
  auto go = [&](auto kern, size_t smem) {
    const unsigned grid = ln_grid(kern, p, smem, kLnRows);
    at::Tensor part;
    if (sums) {
      part = at::empty({(int64_t)grid * 2 * p.D}, dy.options().dtype(at::kFloat));
      p.part = part.data_ptr<float>();
    }
    kern<<<grid, p.W * p.R * 32, smem, stream>>>(p);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    if (!sums) return;
    const at::ScalarType type = dw.has_value() ? dw->scalar_type() : db->scalar_type();
    const unsigned blocks = (unsigned)((2 * p.D + 31) / 32);
    auto finish = [&](auto zero) {
      using W = decltype(zero);
      ln_sum_kernel<W><<<blocks, kLnSumWarps * 32, 0, stream>>>(
          p.part, (int)grid, p.D, dw.has_value() ? reinterpret_cast<W*>(dw->data_ptr()) : nullptr,
          db.has_value() ? reinterpret_cast<W*>(db->data_ptr()) : nullptr);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    };
    if (type == at::kFloat) finish(float{});
    else if (type == at::kBFloat16) finish(__nv_bfloat16{});
    else finish(__half{});
  };
  ln_flags(p.codes != nullptr, p.dh != nullptr, [&](auto kept, auto res) {
    constexpr bool KEPT = decltype(kept)::value, RES = decltype(res)::value;
    if constexpr (VEC) {
      p.src[0] = p.dy, p.pitch[0] = p.dys;
      p.src[1] = RES ? p.dh : p.x, p.pitch[1] = RES ? p.dhs : p.xs;
      p.src[2] = p.x, p.pitch[2] = p.xs;
      constexpr int kBytes = LnSlots<T, K, 1 + (RES ? 1 : 0) + (KEPT ? 0 : 1), KEPT, true>::kBytes;
      // as many warps as two groups of rows leave room for, and the registers that they do
      constexpr int kRoom = 227 * 1024 / (kBytes * 32 * kLnRows * 2);
      constexpr int kWarps = K > 2 || kRoom <= kLnMaxWarps ? kLnMaxWarps : kRoom < kLnBlockWarps ? 20 : kLnBlockWarps;
      const size_t smem = ln_block(p, front, kBytes, kWarps, kLnRows, 1);
      if constexpr (K == 2 && kWarps > 20)   // (16384 x 5120 from codes, 20 warps: 131 us with 80 registers, 112 with 96)
        if (smem > 0 && p.W * p.R <= 20) return go(ln_bwd_kernel<T, VEC, K, KEPT, RES, true, 20>, smem);
      if (smem > 0) return go(ln_bwd_kernel<T, VEC, K, KEPT, RES, true, kWarps>, smem);
    }
    p.R = VEC ? 1 : ln_teams(p, kLnRows);
    go(ln_bwd_kernel<T, VEC, K, KEPT, RES, false, kLnMaxWarps>, front);
  });
}

// dx [M, D], dw and db [D] from dy, the kept input (x, or codes and steps) and stats
void layernorm_bwd(at::Tensor dy, c10::optional<at::Tensor> dh, c10::optional<at::Tensor> x, c10::optional<at::Tensor> codes,
                   c10::optional<at::Tensor> steps, c10::optional<at::Tensor> w, at::Tensor stats, at::Tensor dx,
                   c10::optional<at::Tensor> dw, c10::optional<at::Tensor> db) {
  bool vec;
  LnParams p = ln_base(dy, w, c10::nullopt, vec);
  TORCH_CHECK(x.has_value() != codes.has_value(), "layer_norm: the input, or its codes");
  p.dy = dy.data_ptr();
  p.dys = ln_rows(dy, dy, "dy");
  vec = vec && ln_aligned(dy);
  if (dh.has_value()) {
    p.dh = dh->data_ptr();
    p.dhs = ln_rows(*dh, dy, "dh");
    vec = vec && ln_aligned(*dh);
  }
  if (x.has_value()) {
    p.x = x->data_ptr();
    p.xs = ln_rows(*x, dy, "x");
    vec = vec && ln_aligned(*x);
  } else {
    ln_kept(p, dy, *codes, *steps);
  }
  ln_stats(p, dy, stats);
  ln_rows(dx, dy, "dx");
  TORCH_CHECK(dx.is_contiguous(), "layer_norm: dx is contiguous");
  p.dx = dx.data_ptr();
  vec = vec && ln_aligned(dx);
  const at::ScalarType wt = w.has_value() ? w->scalar_type() : db.has_value() ? db->scalar_type() : at::kFloat;
  if (dw.has_value()) ln_vector(*dw, dy, wt, "dw");
  if (db.has_value()) ln_vector(*db, dy, wt, "db");
  const c10::cuda::CUDAGuard guard(dy.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int K = ln_shape(p, 2);
  ZQ_LN_TYPES(dy.scalar_type(), {
    if (vec) {
      if (K == 1) ln_bwd_launch<T, true, 1>(p, dy, dw, db, stream);
      else if (K == 2) ln_bwd_launch<T, true, 2>(p, dy, dw, db, stream);
      else ln_bwd_launch<T, true, 4>(p, dy, dw, db, stream);
    } else {
      if (K == 1) ln_bwd_launch<T, false, 1>(p, dy, dw, db, stream);
      else if (K == 2) ln_bwd_launch<T, false, 2>(p, dy, dw, db, stream);
      else ln_bwd_launch<T, false, 4>(p, dy, dw, db, stream);
    }
  });
}
