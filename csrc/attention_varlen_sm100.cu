// Attention over packed sequences on the 5th-generation tensor cores (sm_100a):
// forward, and the backward that recomputes the probabilities.
//
// q, o: [T, Hq, D], k, v: [T, Hk, D], bf16 or fp16, D <= 128 a multiple of 8 (q, k,
// v, do through TMA maps: any 16-byte-multiple strides), GQA (Hq a multiple of Hk).
// Sequence i holds rows [cu[i], cu[i+1]); a query sees the keys of its own sequence,
// with `causal` those up to its own position.  lse: [Hq, T] fp32, natural log.
//
//   S = scale·Q Kᵀ, P = softmax(S), O = P V
//   dP = dO Vᵀ, dS = P ∘ (dP - delta), delta = rowsum(dO ∘ O)
//   dQ = scale·dS K, dK = scale·dSᵀ Q, dV = Pᵀ dO
//
// A plan (packed_plan below) lists the row tiles of all sequences, longest work
// first: the grid is (entries, heads) with as many entries as any division of T
// rows into n sequences can have; blocks past the real count leave at once, but
// for the first of them, which writes zeros to the rows of no sequence.
//
// Ragged ends: tiles are loaded whole, so rows past a sequence's end hold the next
// sequence's values (or the TMA fill).  Scores of such keys are replaced (never
// multiplied) and such queries' outputs are not stored; rows that enter a product
// as its K dimension (V forward, K in dQ, Q and dO in dK/dV) are zeroed in shared
// memory first, so that 0 · NaN of a neighbour or of unset padding cannot arise.
//
// MMAs are issued by a whole warp that stays converged, with one elected lane
// inside: the descriptors then are warp-uniform values.  Measured for M = 128, K = 16 on
// one SM, back to back: N / 2 + 10 cycles with A in tensor memory, N / 2 + 43 with A in
// shared memory (N = 128: 74 and 107, N = 64: 42 and 75) against N / 2 of arithmetic.
//
// Measured (bf16, D = 128, causal, inputs not in L2; the multiply rate counts the visible pairs):
//   9 sequences, 8080 rows, 28/4 heads    forward 127 us, dQ 161, dK/dV 207
//   7 sequences, 6004 rows, 24/24 heads   forward 77 us, dQ 89, dK/dV 123
//   8191 + 1037 rows, 8/2 heads           forward 130 us (1.1 PFLOP/s), dQ 192, dK/dV 268
// and fp16, D = 64, bidirectional, 8 sequences, 2393 rows, 12/12 heads: 18.5, 22, 32.6.
// Short sequences are bound by what a block does around its loop (launch, first loads,
// pipeline fill, output: 7-8 us of a block's 15-20 us, with one block to an SM by its
// registers and tensor memory; dQ runs part of it under the block before), long ones by
// the chain of MMAs and exponentials.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "attention_common.cuh"

// defined in gemm_sm100.cu
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();
zq::DeviceStatus* status_buffer(int device);

namespace zq {

constexpr int kVlRows = 128;
enum VlErr { kErrVlLoad = 321, kErrVlMma = 322, kErrVlCompute = 323, kErrVlPlan = 324 };

// One tile of a sequence.  slot: number of this tile over all sequences.
struct __align__(16) VlTile {
  int start, len, tile, slot;
};
// Where a sequence's row statistics begin in a head's row of them: at its first row and four
// more for every 128-row tile before it, rounded down to 16 bytes (they are loaded in bulk).
// A sequence with rows has a tile, so the next one begins behind its last row.
__device__ __forceinline__ int vl_stats_at(const VlTile& w) { return (w.start + 4 * (w.slot - w.tile)) & ~3; }
static int64_t vl_stats_row(int64_t T, int64_t tiles) { return (T + 4 * tiles + 64 + 3) / 4 * 4; }   // (a whole load behind the last)
// meta words: [0] 256-row tiles, [1] 128-row query tiles, [2] 128-row key tiles,
// [3] first row of a sequence, [4] row behind the last sequence
constexpr int kVlMeta = 8;

struct VlParams {
  const VlTile* tiles;
  const int* meta;        // the plan's meta words
  int count_at;           // which of them counts these tiles
  int T, Hq, Hk, D, causal, stats_row;
  int split;              // CTAs of a cluster that share a key tile (dK/dV)
  float scale, scale_log2;
  DeviceStatus* status;
};

template <bool FP16>
__device__ __forceinline__ uint32_t vl_pack(float lo, float hi) {
  if constexpr (FP16) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    return pack_bf16x2(lo, hi);
  }
}
template <bool FP16>
__device__ __forceinline__ float2 vl_unpack(uint32_t w) {
  if constexpr (FP16) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
  } else {
    return bf16x2_to_f2(w);
  }
}
// kind::f16, fp32 accumulators; both operands of one type; `bmn`: B MN-major
template <bool FP16>
__host__ __device__ constexpr uint32_t vl_idesc(int M, int N, bool bmn) {
  return (1u << 4) | (FP16 ? 0u : (1u << 7) | (1u << 10)) | (bmn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t c0, int32_t c1,
                                            int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// a tile of ROWS rows x DP columns: one swizzled atom per 64 columns
template <int DP, int ROWS>
__device__ __forceinline__ void vl_load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int row) {
#pragma unroll
  for (int a = 0; a < DP / 64; ++a) tma_load_3d(dst + a * ROWS * 128, map, bar, a * 64, head, row);
}

// zeros to rows [from, ROWS) of such a tile, by 256 threads; then visible to the MMAs
template <int DP, int ROWS>
__device__ __forceinline__ void vl_zero_rows(uint8_t* tile, int from, int thread) {
  for (int i = thread; i < (DP / 64) * ROWS; i += 256) {
    const int row = i % ROWS;
    if (row >= from) {
      uint4* r = reinterpret_cast<uint4*>(tile + (i / ROWS) * ROWS * 128 + row * 128);
#pragma unroll
      for (int c = 0; c < 8; ++c) r[c] = make_uint4(0, 0, 0, 0);
    }
  }
  fence_proxy_async_smem();
}

// wait by all lanes, decided as one
__device__ __forceinline__ bool vl_wait(uint64_t* bar, uint32_t parity, DeviceStatus* st, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, st, code));
}

// zeros to the rows of no sequence of one head of out [T, H, D] (contiguous)
__device__ __forceinline__ void vl_zero_outside(uint16_t* out, int T, int H, int h, int D, const int* meta) {
  const int first = meta[3], last = meta[4], per = D / 8;
  const int64_t n = (int64_t)(first + (T - last)) * per;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    int row = (int)(i / per);
    if (row >= first) row = row - first + last;
    *reinterpret_cast<uint4*>(out + ((int64_t)row * H + h) * D + (i % per) * 8) = make_uint4(0, 0, 0, 0);
  }
}

// The forward's O in 32 bits, as its rounded value and one more byte: the 8 bits
// behind the kept ones of the 32-bit pattern, read as a signed number they are the
// difference to the value rounded to nearest (bits 8-15 for bf16, 5-12 for fp16; a tie
// rounded down reads as one rounded up, and below fp16's normal range the byte is worth
// 2^-11 of the value at most).  delta = rowsum(dO ∘ O) is formed from both: from the
// rounded O alone it has an error of the size of dS's own rounding where a row sees few
// keys (dQ and dK of 88-row sequences: 1.60 times the error of one rounding, with the
// byte 1.41).
// the bytes of four values
template <bool FP16>
__device__ __forceinline__ uint32_t vl_low_bytes(float a, float b, float c, float d) {
  uint32_t x[4] = {__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d)};
  if constexpr (FP16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] <<= 3;   // to byte 1
  }
  return __byte_perm(__byte_perm(x[0], x[1], 0x0051), __byte_perm(x[2], x[3], 0x0051), 0x5410);
}
// byte K of `bytes` back onto a rounded value
template <bool FP16, int K>
__device__ __forceinline__ float vl_with_low(float rounded, uint32_t bytes) {
  int d;   // byte k, sign-extended, from byte 1 on (a selector's top bit copies the sign; __byte_perm has none)
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(d) : "r"(bytes), "n"(0x8804 | (K << 4) | (K << 8) | (K << 12)));
  if constexpr (FP16) d >>= 3;
  return rounded == 0.0f ? 0.0f : __int_as_float(__float_as_int(rounded) + d);   // (below 0's pattern lies NaN)
}

// A warp's 32 accumulator rows (one a lane) of N columns times f, rounded, to rows `out`
// (ld elements apart; the first `live` exist, and columns below D).  They go through
// `stage` (64 N bytes of the warp's own), so that a store covers whole lines of a few
// rows instead of 16 bytes of 32 rows each.  `low` (optional): the low bytes, likewise.
template <bool FP16, int N>
__device__ __forceinline__ void vl_store_rows(uint32_t taddr, float f, uint8_t* stage, uint16_t* out, int64_t ld, int col0, int D,
                                              int live, uint8_t* low = nullptr) {
  const int lane = threadIdx.x & 31;
  constexpr int per = N / 8;                       // 16-byte chunks of a row, and lanes to a row
  // a row's chunks, their places turned by the row against bank conflicts
  auto at = [&](int r, int c) { return stage + r * (N * 2) + ((c ^ (r & (per - 1))) << 4); };
  uint32_t lb[N / 4];
#pragma unroll
  for (int c = 0; c < N; c += 32) {
    uint32_t o[32];
    tmem_ld_32x32b_x32(taddr + (uint32_t)c, o);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 v;
      v.x = vl_pack<FP16>(__uint_as_float(o[8 * i + 0]), __uint_as_float(o[8 * i + 1]));
      v.y = vl_pack<FP16>(__uint_as_float(o[8 * i + 2]), __uint_as_float(o[8 * i + 3]));
      v.z = vl_pack<FP16>(__uint_as_float(o[8 * i + 4]), __uint_as_float(o[8 * i + 5]));
      v.w = vl_pack<FP16>(__uint_as_float(o[8 * i + 6]), __uint_as_float(o[8 * i + 7]));
      *reinterpret_cast<uint4*>(at(lane, c / 8 + i)) = v;
    }
    if (low != nullptr)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        lb[c / 4 + i] = vl_low_bytes<FP16>(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                           __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
  }
  __syncwarp();
  const int chunk = lane % per;
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 32 / per) {
    const int r = r0 + lane / per;
    const uint4 v = *reinterpret_cast<const uint4*>(at(r, chunk));
    if (r < live && col0 + 8 * chunk < D) *reinterpret_cast<uint4*>(out + r * ld + col0 + 8 * chunk) = v;
  }
  if (low != nullptr) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N / 8; ++i)
      *reinterpret_cast<uint2*>(at(lane, i)) = make_uint2(lb[2 * i], lb[2 * i + 1]);
    __syncwarp();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 32 / per) {
      const int r = r0 + lane / per;
      const uint2 v = *reinterpret_cast<const uint2*>(at(r, chunk));
      if (r < live && col0 + 8 * chunk < D) *reinterpret_cast<uint2*>(low + r * ld + col0 + 8 * chunk) = v;
    }
  }
}

// ============================================================================
// Plan: tile tables of the packed sequences and each row's position.
//
// Blocks 0-2 build the tables (256-row tiles, 128-row query tiles, 128-row key
// tiles), each sorted by the tile's causal work, longest first (a counting sort
// over at most 1024 classes; the order inside a class only moves blocks about).
// The other blocks write positions.  cu is taken as it is on the device: values
// are clamped to [0, T] and to rising order, and a division that needs more tiles
// than the table has loses what does not fit, with an error status.
// ============================================================================
constexpr int kPlanThreads = 1024;
constexpr int kPlanClasses = 1024;

__device__ __forceinline__ int plan_bound(const int* cu, int i, int T) { return min(max(cu[i], 0), T); }

__global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(const int* __restrict__ cu, int n, int T, int cap256,
                                                                   int cap128, VlTile* __restrict__ tiles,
                                                                   int* __restrict__ base, int* __restrict__ meta,
                                                                   int* __restrict__ positions, DeviceStatus* status) {
  const int tid = threadIdx.x;
  if (blockIdx.x >= 3) {
    const int row = (blockIdx.x - 3) * kPlanThreads + tid;
    if (row >= T) return;
    int lo = 0, hi = n;   // the last i with cu[i] <= row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu[mid] <= row) lo = mid; else hi = mid - 1;
    }
    const int begin = plan_bound(cu, lo, T);
    positions[row] = (lo < n && row >= begin) ? row - begin : 0;
    return;
  }
  __shared__ int s_warp[32];
  __shared__ int s_class[kPlanClasses];
  __shared__ int s_run;
  const int kind = blockIdx.x;                       // 0: 256-row tiles, 1: queries, 2: keys
  const int rows = kind == 0 ? 256 : 128, cap = kind == 0 ? cap256 : cap128;
  VlTile* out = tiles + (kind == 0 ? 0 : cap256 + (kind - 1) * cap128);
  int* b = base + kind * (n + 1);
  auto bounds = [&](int i, int& begin, int& len) {
    begin = plan_bound(cu, i, T);
    len = max(plan_bound(cu, i + 1, T) - begin, 0);
  };
  // b[i] = tiles of the sequences before i, or cap + 1 where these are more (a rising
  // division has no more than cap; one out of order can ask for more than 2^31, so every
  // sum is cut off there: cap < 2^25, 32 of them fit)
  if (tid == 0) s_run = 0;
  for (int i = tid; i < kPlanClasses; i += kPlanThreads) s_class[i] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int c = 0;
    if (i < n) {
      int begin, len;
      bounds(i, begin, len);
      c = min((len + rows - 1) / rows, cap + 1);
    }
    int x = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if ((tid & 31) >= o) x += y;
    }
    if ((tid & 31) == 31) s_warp[tid >> 5] = min(x, cap + 1);
    __syncthreads();
    int before = s_run;
    for (int w = 0; w < (tid >> 5); ++w) before = min(before + s_warp[w], cap + 1);
    if (i < n) b[i] = min(before + x - c, cap + 1);
    __syncthreads();
    if (tid == kPlanThreads - 1) s_run = min(before + x, cap + 1);
    __syncthreads();
  }
  const int want = s_run, total = min(want, cap);
  if (tid == 0) {
    b[n] = want;
    meta[kind] = 0;
    if (kind == 0) {
      meta[3] = n > 0 ? plan_bound(cu, 0, T) : 0;
      meta[4] = n > 0 ? max(plan_bound(cu, n, T), plan_bound(cu, 0, T)) : 0;
    }
    bool bad = want > cap;
    if (bad) record_error(status, kErrVlPlan, want);
  }
  __syncthreads();
  // classes of work, in units of 64 rows, halved until they fit
  int shift = 0;
  while (((T + 63) / 64 >> shift) >= kPlanClasses) ++shift;
  auto tile_at = [&](int s, VlTile& t, int& cls) -> bool {
    int lo = 0, hi = n - 1;   // the last sequence with b[i] <= s
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (b[mid] <= s) lo = mid; else hi = mid - 1;
    }
    bounds(lo, t.start, t.len);
    t.tile = s - b[lo];
    t.slot = s;
    // a sequence whose tiles do not all fit is left out (its row statistics would not either)
    if (b[lo + 1] > cap || t.tile < 0 || t.tile * rows >= t.len) return false;
    const int row = t.tile * rows;
    const int work = kind == 2 ? t.len - row : min(row + rows, t.len);
    cls = kPlanClasses - 1 - min(kPlanClasses - 1, (work + 63) / 64 >> shift);   // longest first
    return true;
  };
  for (int s = tid; s < total; s += kPlanThreads) {
    VlTile t;
    int cls;
    if (tile_at(s, t, cls)) atomicAdd(&s_class[cls], 1);
  }
  __syncthreads();
  {   // exclusive scan over the classes (one per thread)
    static_assert(kPlanClasses == kPlanThreads, "one class per thread");
    const int c = s_class[tid];
    int x = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if ((tid & 31) >= o) x += y;
    }
    if ((tid & 31) == 31) s_warp[tid >> 5] = x;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < (tid >> 5); ++w) before += s_warp[w];
    s_class[tid] = before + x - c;
    if (tid == kPlanThreads - 1) meta[kind] = before + x;
  }
  __syncthreads();
  for (int s = tid; s < total; s += kPlanThreads) {
    VlTile t;
    int cls;
    if (tile_at(s, t, cls)) out[atomicAdd(&s_class[cls], 1)] = t;
  }
}

// ============================================================================
// Forward: two query tiles (256 rows of one sequence and head) per CTA.
//
// Tensor memory: S_A 0-127, S_B 128-255, O_A 256.., O_B 384..; P (16-bit pairs)
// is written over S's own columns.  Q_A and Q_B stay in shared memory, K and V tiles
// of 128 keys stream through two-stage rings read by both query tiles.  576 threads:
// warps 0-7 / 8-15 are the softmax warps of tile A / B, two threads to a query row (=
// TMEM lane) with 64 keys each, which exchange their maxima through shared memory;
// warp 16 issues the MMAs in the order
//     PV_A(j), S_A(j+1) | PV_B(j), S_B(j+1) | ...
// so one tile's exponentials run beside the other's products; warp 17 loads.
// (The loop of a tile - scores, softmax, P V, next scores - is serial, so the time from
// scores to P counts in full.)  A step of 128 keys for both tiles takes about 3400 cycles,
// of which the MMAs need 2900 (Q from shared memory; for Q in tensor memory too the scores
// and O of two tiles leave no columns) and the exponentials 1500 of the special-function
// unit.  One thread a row measured the same.
// The running maximum moves only when a row's maximum grows by more than 2^8 (O is
// rescaled then); O / l and lse use the same one, so the result is exact.
// When the sequence ends inside tile A, tile B does not exist and is skipped.
// ============================================================================
constexpr int kVfThreads = 576;   // 16 softmax warps, MMA warp, loader warp
constexpr int kVfStages = 2;
constexpr float kVlRescale = 8.0f;
// exp2_poly3_x2 of anything up to -120, to the bit: taken off its results, a masked key weighs
// 0 (a value behind the mask is weighed by it), and what exceeds 2^-96 does not change
constexpr float kVlPolyFloor = 0.9999289512634277f * 0x1p-120f;

template <int DP>
struct VfSmem {
  static constexpr int kTile = 128 * DP * 2;
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + kVfStages * kTile;
  static constexpr int kX = kV + kVfStages * kTile;     // [2 tiles][2 parities][2 halves][128 rows] fp32
  static constexpr int kBar = kX + 2 * 2 * 2 * 128 * 4;
  static constexpr int kBytes = kBar + 256 + 1024;
};

template <bool FP16, int DP>
__global__ void __launch_bounds__(kVfThreads, 1)
attn_varlen_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ VlParams p,
                       uint16_t* __restrict__ O, float* __restrict__ lse, uint8_t* __restrict__ low) {
  using L = VfSmem<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;     // [kVfStages]
  uint64_t* k_empty = bars + 3;
  uint64_t* v_full = bars + 5;
  uint64_t* v_empty = bars + 7;
  uint64_t* s_full = bars + 9;     // [tile]
  uint64_t* p_full = bars + 11;    // [tile], one arrival per softmax warp
  uint64_t* pv_done = bars + 13;   // [tile]
  uint64_t* drain = bars + 15;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int entry = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
  const VlTile w = p.tiles[entry];   // (read beside the count; past it the plan's other words)
  const int count = p.meta[p.count_at];
  if (entry >= count) {
    if (entry == count) vl_zero_outside(O, p.T, p.Hq, h, p.D, p.meta);
    return;
  }
  const int hk = h / (p.Hq / p.Hk);
  const int row_a = w.tile * 256, row_b = row_a + 128;
  const int nkt = (w.len + 127) / 128;
  const int n_a = p.causal ? min(2 * w.tile + 1, nkt) : nkt;
  const int n_b = row_b >= w.len ? 0 : p.causal ? min(2 * w.tile + 2, nkt) : nkt;   // n_b >= n_a, or none
  const int n_max = max(n_a, n_b);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kVfStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 16) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 17) {
    // ------------------------------------------------------------ TMA loader (one thread)
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, (n_b > 0 ? 2 : 1) * L::kTile);
      vl_load_tile<DP, 128>(smem + L::kQ, &tmQ, q_full, h, w.start + row_a);
      if (n_b > 0) vl_load_tile<DP, 128>(smem + L::kQ + L::kTile, &tmQ, q_full, h, w.start + row_b);
      int k_issued = 0, v_issued = 0;
      bool ok = true;
      for (int j = 0; j < n_max && ok; ++j) {
        const int st = j % kVfStages;
        const uint32_t ph = ((j / kVfStages) & 1) ^ 1;
        if (!mbar_wait(&k_empty[st], ph, p.status, kErrVlLoad)) { ok = false; break; }
        mbar_arrive_expect_tx(&k_full[st], L::kTile);
        vl_load_tile<DP, 128>(smem + L::kK + st * L::kTile, &tmK, &k_full[st], hk, w.start + j * 128);
        k_issued = j + 1;
        if (!mbar_wait(&v_empty[st], ph, p.status, kErrVlLoad)) { ok = false; break; }
        mbar_arrive_expect_tx(&v_full[st], L::kTile);
        vl_load_tile<DP, 128>(smem + L::kV + st * L::kTile, &tmV, &v_full[st], hk, w.start + j * 128);
        v_issued = j + 1;
      }
      if (!ok) {  // let every copy this thread issued land before the CTA can exit
        mbar_wait(q_full, 0, nullptr, 0);
        for (int j = max(k_issued - kVfStages, 0); j < k_issued; ++j)
          mbar_wait(&k_full[j % kVfStages], (j / kVfStages) & 1, nullptr, 0);
        for (int j = max(v_issued - kVfStages, 0); j < v_issued; ++j)
          mbar_wait(&v_full[j % kVfStages], (j / kVfStages) & 1, nullptr, 0);
      }
    }
  } else if (warp == 16) {
    // ------------------------------------------------------------ MMA issuer (whole warp)
    constexpr uint32_t idesc_s = vl_idesc<FP16>(128, 128, false);
    constexpr uint32_t idesc_pv = vl_idesc<FP16>(128, DP, true);
    const uint32_t q_base = smem_u32(smem + L::kQ), k_base = smem_u32(smem + L::kK), v_base = smem_u32(smem + L::kV);
    auto wait_k = [&](int j) { return vl_wait(&k_full[j % kVfStages], (j / kVfStages) & 1, p.status, kErrVlMma); };
    // S_x = Q_x K_jᵀ; `last`: nobody reads K_j after it
    auto issue_s = [&](int x, int j, bool last) {
      const uint64_t qd = umma_desc_sw128_kmajor(q_base + x * L::kTile);
      const uint64_t kd = umma_desc_sw128_kmajor(k_base + (j % kVfStages) * L::kTile);
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint64_t off = (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
          umma_f16_ss(tmem + (uint32_t)(x * 128), qd + off, kd + off, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[x]);
        if (last) umma_commit(&k_empty[j % kVfStages]);
      }
      __syncwarp();
    };
    // O_x += P_x V_j: P from tensor memory, V read MN-major
    auto issue_pv = [&](int x, int j, bool last) {
      const uint64_t vd = umma_desc_sw128_mnmajor(v_base + (j % kVfStages) * L::kTile, 16384u);
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_f16_ts(tmem + 256u + (uint32_t)(x * 128), tmem + (uint32_t)(x * 128 + (kk >> 2) * 64 + (kk & 3) * 8),
                      vd + (uint64_t)(kk * 128),
                      idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&pv_done[x]);
        if (last) umma_commit(&v_empty[j % kVfStages]);
      }
      __syncwarp();
    };
    bool ok = vl_wait(q_full, 0, p.status, kErrVlMma) && wait_k(0);
    if (ok) {
      tc_fence_after();
      issue_s(0, 0, n_b == 0);
      if (n_b > 0) issue_s(1, 0, true);
    }
    for (int j = 0; j < n_max && ok; ++j) {
      if (!vl_wait(&v_full[j % kVfStages], (j / kVfStages) & 1, p.status, kErrVlMma)) { ok = false; break; }
      if (j < n_a) {
        if (!vl_wait(&p_full[0], j & 1, p.status, kErrVlMma)) { ok = false; break; }
        tc_fence_after();
        issue_pv(0, j, n_b == 0);
        if (j + 1 < n_a) {
          if (!wait_k(j + 1)) { ok = false; break; }
          tc_fence_after();
          issue_s(0, j + 1, n_b == 0);
        }
      }
      if (j < n_b) {
        if (!vl_wait(&p_full[1], j & 1, p.status, kErrVlMma)) { ok = false; break; }
        tc_fence_after();
        issue_pv(1, j, true);
        if (j + 1 < n_b) {
          if (!wait_k(j + 1)) { ok = false; break; }
          tc_fence_after();
          issue_s(1, j + 1, true);
        }
      }
    }
    // every MMA issued has completed before TMEM can be freed
    if (elect_one_sync()) umma_commit(drain);
    __syncwarp();
    mbar_wait(drain, 0, nullptr, 0);
  } else {
    // ------------------------------------------------------------ softmax + epilogue
    const int x = warp >> 3;                        // 0: tile A, 1: tile B
    const int half = (warp >> 2) & 1;               // keys (and O columns) of this thread's half row
    const int quad = warp & 3;                      // TMEM lane quadrant
    const int row = quad * 32 + lane;               // row in the tile = TMEM lane
    const int pair_bar = 1 + x * 4 + quad;          // the two warps of these rows
    const int q = (x == 0 ? row_a : row_b) + row;   // row in the sequence
    const int n_kv = x == 0 ? n_a : n_b;
    const int limit = (p.causal ? min(q + 1, w.len) : w.len) - 64 * half;   // keys that the row sees, from this half's first
    const uint32_t t_s = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(x * 128 + half * 64);
    const uint32_t t_o = tmem + ((uint32_t)(quad * 32) << 16) + 256u + (uint32_t)(x * 128 + half * (DP / 2));
    float* xs = reinterpret_cast<float*>(smem + L::kX) + x * 512;
    float m_used = -INFINITY;
    float l = 0.0f;                                 // this half's share of the row sum
    bool ok = true;
    // a wait that ran out makes the later ones return at once: the two warps of a row meet
    // at their barrier in every step all the same
    auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && vl_wait(bar, parity, p.status, kErrVlCompute); };
    for (int j = 0; j < n_kv; ++j) {
      wait(&s_full[x], j & 1);
      tc_fence_after();
      uint32_t r[64];
      tmem_ld64(t_s, r);
      tmem_ld_wait();
      const int seen = limit - j * 128;
      if (__any_sync(0xffffffffu, seen < 64)) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c >= seen) r[c] = __float_as_uint(-INFINITY);
      }
      // row max: 8 independent chains of 3-input maxima over columns 8..55, then the rest
      float pm[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) pm[i] = __uint_as_float(r[i]);
#pragma unroll
      for (int c = 8; c < 56; c += 16)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          pm[i] = fmax3(pm[i], __uint_as_float(r[c + i]), __uint_as_float(r[c + 8 + i]));
      const float mine = fmax3(fmax3(pm[0], pm[1], __uint_as_float(r[56])),
                               fmax3(pm[2], pm[3], __uint_as_float(r[57])),
                               fmax3(fmax3(pm[4], pm[5], __uint_as_float(r[58])),
                                     fmax3(pm[6], pm[7], __uint_as_float(r[59])),
                                     fmax3(__uint_as_float(r[60]), __uint_as_float(r[61]),
                                           fmaxf(__uint_as_float(r[62]), __uint_as_float(r[63])))));
      float* xm = xs + (j & 1) * 256 + row;
      xm[half * 128] = mine;
      named_barrier(pair_bar, 64);
      const float mx = fmaxf(mine, xm[(half ^ 1) * 128]) * p.scale_log2;
      const bool need = mx > m_used + kVlRescale;
      const bool rescale = __any_sync(0xffffffffu, need);   // (the same in both warps of the rows)
      float factor = 1.0f;
      if (rescale) {
        const float m_new = need ? mx : m_used;
        factor = (m_used == -INFINITY) ? 0.0f : fast_exp2(m_used - m_new);
        m_used = m_new;
      }
      // (a row whose scores so far are all -inf: shifted by nothing they weigh 0, not NaN)
      const float shift = m_used == -INFINITY ? 0.0f : -m_used;
      const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nm2 = f2_pack(shift, shift);
      uint64_t ps2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int i = 0; i < 32; ++i) {  // masked keys hold -inf: 2^x gives 0
        float a0, a1;
        f2_unpack(f2_fma(f2_pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), sc2, nm2), a0, a1);
        float p0, p1;
        if (i % 4 == 3) {
          exp2_poly3_x2(a0, a1, p0, p1);
          f2_unpack(f2_sub(f2_pack(p0, p1), f2_pack(kVlPolyFloor, kVlPolyFloor)), p0, p1);
        } else {
          p0 = fast_exp2(a0);
          p1 = fast_exp2(a1);
        }
        ps2[i & 3] = f2_add(ps2[i & 3], f2_pack(p0, p1));
        r[i] = vl_pack<FP16>(p0, p1);
      }
      tmem_st_32x32b_x32(t_s, *reinterpret_cast<const uint32_t(*)[32]>(&r[0]));   // over this half's own scores
      float ps[4];
      f2_unpack(f2_add(ps2[0], ps2[1]), ps[0], ps[1]);
      f2_unpack(f2_add(ps2[2], ps2[3]), ps[2], ps[3]);
      l = l * factor + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
      if (rescale && j > 0) {
        // O holds PV_0..PV_{j-1}: wait for PV_{j-1}, then scale this thread's half row
        wait(&pv_done[x], (j - 1) & 1);
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < DP / 64; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_o + (uint32_t)(c * 32), o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
          tmem_st_32x32b_x32(t_o + (uint32_t)(c * 32), o);
        }
      }
      // the sequence ends inside this key tile: zero V's other rows, by the first
      // query tile that uses it (PV_B(j) is issued after PV_A(j))
      if (w.len - j * 128 < 128 && (x == 0 || j >= n_a)) {
        wait(&v_full[j % kVfStages], (j / kVfStages) & 1);
        vl_zero_rows<DP, 128>(smem + L::kV + (j % kVfStages) * L::kTile, w.len - j * 128, threadIdx.x & 255);
      }
      tmem_st_wait();
      tc_fence_before();          // TMEM loads/stores of this step ordered before the arrive
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[x]);
    }
    if (n_kv > 0) {
      const int jl = n_kv - 1;
      float* xl = xs + (n_kv & 1) * 256 + row;      // (the other parity than the last step's)
      xl[half * 128] = l;
      named_barrier(pair_bar, 64);
      l += xl[(half ^ 1) * 128];
      wait(&pv_done[x], jl & 1);
      if (ok) {
        tc_fence_after();
        // 1 / l, a last bit up: where few keys have equal weights O would often lie at a tie of
        // its rounding, which its byte cannot tell apart; with the bit it lies above it
        const float inv = __uint_as_float(__float_as_uint(1.0f / l) + 1u);
        // (this tile's Q has given all its scores: its memory stages the output)
        const int64_t at = ((int64_t)(w.start + q - lane) * p.Hq + h) * p.D;
        vl_store_rows<FP16, DP / 2>(t_o, inv, smem + L::kQ + x * L::kTile + (warp & 7) * (L::kTile / 8), O + at,
                                    (int64_t)p.Hq * p.D, half * (DP / 2), p.D, w.len - (q - lane),
                                    low != nullptr ? low + at : nullptr);
        if (q < w.len && half == 0) lse[(int64_t)h * p.T + w.start + q] = (m_used + __log2f(l)) * 0.69314718055994531f;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ============================================================================
// dQ: an item is a 128-query tile of a head, its steps are key tiles of 64.
//
// A CTA does one item after another: when the loader comes to the last key tiles of one it
// asks the hardware for a block of the grid that has not started, and takes that block's
// item over (no counter in memory, and the longest-first order of the grid still evens
// out; asked for at the item's start, the items of 8191 + 1037 rows took 201 us, not
// 192).  So Q, dO and the first K and V of the next item are on their way during the
// last steps of this one, its O comes to L2, its first scores are formed while dQ of
// this one leaves, and tensor memory and barriers are set up once.  One item to a CTA,
// which paid for all this between any two: 184 us against 157 (8080 rows, 28/4 heads),
// 100 against 87 (6004 rows, 24/24 heads), 181 both at 8191 + 1037 rows.
// Q and dO are copied into tensor memory once, so that S = Q Kᵀ and dP = dO Vᵀ
// (N = 64) read only K and V from shared memory.  S and dP are double-buffered:
// two groups of eight warps take alternate key tiles (two threads to a query row, 32
// columns each: no exchange between warps), the MMA warp issues the scores of tile t + 1
// before it waits for dS of tile t.  dS (16-bit pairs, over S's own columns) times
// K (read MN-major) adds into dQ; dQ is written once: no atomics.
// Tensor memory: S 64 b, dP 128 + 64 b (b = t & 1), dQ 256.., Q 384.., dO 448...
// A key tile takes about 1400 cycles, of which its MMAs need 970.
// The kernel also forms delta = rowsum(dO ∘ O) and -lse·log2(e) of its rows and
// stores them for the dK/dV kernel, which runs after it.
// ============================================================================
constexpr int kVlMaxSplit = 4;      // CTAs that share a key tile at most (dK/dV)
constexpr int kVbThreads = 608;     // two groups of eight compute warps, MMA warp, two loader warps

// Asks for a block of this grid that has not started: it then never starts, and its
// index comes to `answer` (16 bytes; -1 in vl_answered_block: none was left, and no
// further request may be made).
__device__ __forceinline__ void vl_request_block(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ int vl_answered_block(const void* answer) {
  int x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 a;\n\t"
      "ld.shared.b128 a, [%1];\n\t"
      "mov.u32 %0, -1;\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, a;\n\t}"
      : "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return x;
}
// threadIdx.x, read where it is written
__device__ __forceinline__ int vl_tid() {
  int t;
  asm volatile("mov.u32 %0, %%tid.x;" : "=r"(t));
  return t;
}
__device__ __forceinline__ void vl_prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// loads that stay where they are written
__device__ __forceinline__ float vl_ld_f32(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 vl_ld_u2(const void* p) {
  uint2 v;
  asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 vl_ld_u4(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <int DP>
struct VqSmem {
  static constexpr int kKStages = 5, kVStages = 3;
  static constexpr int kTile = 128 * DP * 2, kHalf = 64 * DP * 2;
  static constexpr int kQ = 0, kDO = kTile, kK = 2 * kTile, kV = kK + kKStages * kHalf;
  static constexpr int kStage = kV + kVStages * kHalf;   // dQ on its way out, 2 KB a warp
  static constexpr int kX = kStage + 256 * DP;           // [2][128] fp32
  static constexpr int kBar = kX + 1024;
  static constexpr int kBytes = kBar + 288 + 1024;
  static_assert(kBytes <= 232448, "shared memory of a block");
};

template <bool FP16, int DP>
__global__ void __launch_bounds__(kVbThreads, 1)
attn_varlen_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                      const __grid_constant__ VlParams p, const uint16_t* __restrict__ O,
                      const uint8_t* __restrict__ low, const float* __restrict__ lse, float* __restrict__ delta, float* __restrict__ nlse2,
                      uint16_t* __restrict__ dQ) {
  using L = VqSmem<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* q_full = bars;                     // Q and dO landed
  uint64_t* in_tmem = bars + 1;                // Q and dO copied (one arrival per compute warp)
  uint64_t* k_full = bars + 2;                 // [kKStages]
  uint64_t* k_empty = k_full + L::kKStages;
  uint64_t* v_full = k_empty + L::kKStages;    // [kVStages]
  uint64_t* v_empty = v_full + L::kVStages;
  uint64_t* s_full = v_empty + L::kVStages;    // [2]
  uint64_t* ds_full = s_full + 2;              // [2], eight arrivals
  uint64_t* dq_done = ds_full + 2;
  uint64_t* q_empty = dq_done + 1;             // the tile of Q and dO may be loaded over, the note is copied
  uint64_t* dq_read = dq_done + 2;             // dQ left tensor memory
  uint64_t* next_full = dq_done + 3;           // the answer to a request for another block's item
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dq_done + 4);
  // the loader's note of an item, for the other warps (two: an item's epilogue comes under the next)
  VlTile* s_tile = reinterpret_cast<VlTile*>(smem + L::kBar + 224);
  int* s_head = reinterpret_cast<int*>(s_tile + 2);                  // [2], -1: no more
  int* s_zero = s_head + 2;                                          // head whose outside rows are left, or -1
  uint8_t* answer = smem + L::kBar + 272;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = p.meta[p.count_at];
  const int own = blockIdx.x;   // item (entry, head)
  if (own / p.Hq >= count) {
    if (own / p.Hq == count) vl_zero_outside(dQ, p.T, p.Hq, own % p.Hq, p.D, p.meta);
    return;
  }
  auto key_tiles = [&](const VlTile& w) { return ((p.causal ? min(w.tile * 128 + 128, w.len) : w.len) + 63) / 64; };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(in_tmem, 16);
    for (int i = 0; i < L::kKStages; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < L::kVStages; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&ds_full[i], 8); }
    mbar_init(dq_done, 1);
    mbar_init(q_empty, 17);
    mbar_init(dq_read, 16);
    mbar_init(next_full, 1);
    *s_zero = -1;
    fence_mbar_init();
    prefetch_tmap(&tmQ); prefetch_tmap(&tmK); prefetch_tmap(&tmV); prefetch_tmap(&tmDO);
  }
  if (warp == 16) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 17) {
    // ------------------------------------------------------------ TMA loader of Q, dO and K; items
    int t = 0, it = 0, i = own, asked = -1;   // key tiles of all items so far; items; this one; requests
    bool ok = true;
    for (;; ++it) {
      if (it > 0 && !vl_wait(q_empty, (it - 1) & 1, p.status, kErrVlLoad)) { ok = false; break; }
      if (i < 0) {
        if (lane == 0) {
          s_head[it & 1] = -1;
          mbar_arrive(q_full);
        }
        break;
      }
      const VlTile w = p.tiles[i / p.Hq];
      const int h = i % p.Hq, hk = h / (p.Hq / p.Hk), n_kv = key_tiles(w), row0 = w.tile * 128;
      if (lane == 0) {
        s_tile[it & 1] = w;
        s_head[it & 1] = h;
        mbar_arrive_expect_tx(q_full, 2 * L::kTile);   // (releases the note)
        vl_load_tile<DP, 128>(smem + L::kQ, &tmQ, q_full, h, w.start + row0);
        vl_load_tile<DP, 128>(smem + L::kDO, &tmDO, q_full, h, w.start + row0);
      }
      for (int r = lane; r < min(128, w.len - row0); r += 32) {   // O, read between two items, to L2
        const int64_t at = ((int64_t)(w.start + row0 + r) * p.Hq + h) * p.D;
        vl_prefetch(O + at);
        vl_prefetch(O + at + p.D - 8);
        vl_prefetch(low + at);
      }
      __syncwarp();
      if (lane == 0)
        for (int j = 0; j < n_kv; ++j, ++t) {
          const int st = t % L::kKStages;
          ok = mbar_wait(&k_empty[st], ((t / L::kKStages) & 1) ^ 1, p.status, kErrVlLoad);
          if (!ok) break;
          mbar_arrive_expect_tx(&k_full[st], L::kHalf);
          vl_load_tile<DP, 64>(smem + L::kK + st * L::kHalf, &tmK, &k_full[st], hk, w.start + j * 64);
          if (j == max(n_kv - 2, 0)) {   // (not sooner: the items then even out over the SMs)
            asked = it;
            mbar_arrive_expect_tx(next_full, 16);
            vl_request_block(answer, next_full);
          }
        }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok || !vl_wait(next_full, it & 1, p.status, kErrVlLoad)) { ok = false; ++it; break; }
      i = vl_answered_block(answer);
      if (i >= 0 && i / p.Hq >= count) {   // a block with no tile: no more requests after it
        if (lane == 0 && i / p.Hq == count) *s_zero = i % p.Hq;
        i = -1;
      }
      fence_proxy_async_smem();            // the answer is read before the next is written
      __syncwarp();
    }
    if (!ok && lane == 0) {  // let every copy this thread issued land before the CTA can exit
      if (asked >= 0) mbar_wait(next_full, asked & 1, nullptr, 0);
      if (it > 0) mbar_wait(q_full, (it - 1) & 1, nullptr, 0);
      for (int u = max(t - L::kKStages, 0); u < t; ++u) mbar_wait(&k_full[u % L::kKStages], (u / L::kKStages) & 1, nullptr, 0);
    }
  } else if (warp == 18) {
    // ------------------------------------------------------------ TMA loader of V, by the other's notes
    if (lane == 0) {
      int t = 0;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        if (!mbar_wait(q_full, it & 1, p.status, kErrVlLoad)) { ok = false; break; }
        if (s_head[it & 1] < 0) break;
        const VlTile w = s_tile[it & 1];
        const int hk = s_head[it & 1] / (p.Hq / p.Hk), n_kv = key_tiles(w);
        // (an item whose K fits the ring needs no V for the next one's Q and dO to come: without
        // this arrival q_full could complete twice before this thread has looked at it once)
        mbar_arrive(q_empty);
        for (int j = 0; j < n_kv; ++j, ++t) {
          const int st = t % L::kVStages;
          ok = mbar_wait(&v_empty[st], ((t / L::kVStages) & 1) ^ 1, p.status, kErrVlLoad);
          if (!ok) break;
          mbar_arrive_expect_tx(&v_full[st], L::kHalf);
          vl_load_tile<DP, 64>(smem + L::kV + st * L::kHalf, &tmV, &v_full[st], hk, w.start + j * 64);
        }
      }
      if (!ok)
        for (int u = max(t - L::kVStages, 0); u < t; ++u) mbar_wait(&v_full[u % L::kVStages], (u / L::kVStages) & 1, nullptr, 0);
    }
  } else if (warp == 16) {
    // ------------------------------------------------------------ MMA issuer (whole warp)
    constexpr uint32_t idesc_s = vl_idesc<FP16>(128, 64, false);
    constexpr uint32_t idesc_q = vl_idesc<FP16>(128, DP, true);
    const uint32_t k_base = smem_u32(smem + L::kK), v_base = smem_u32(smem + L::kV);
    auto issue_scores = [&](int t) -> bool {
      const int ks = t % L::kKStages, vs = t % L::kVStages, b = t & 1;
      if (!vl_wait(&k_full[ks], (t / L::kKStages) & 1, p.status, kErrVlMma)) return false;
      if (!vl_wait(&v_full[vs], (t / L::kVStages) & 1, p.status, kErrVlMma)) return false;
      tc_fence_after();
      const uint64_t kd = umma_desc_sw128_kmajor(k_base + ks * L::kHalf), vd = umma_desc_sw128_kmajor(v_base + vs * L::kHalf);
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint64_t off = (uint64_t)(((kk >> 2) * 8192 + (kk & 3) * 32) >> 4);
          umma_f16_ts(tmem + (uint32_t)(64 * b), tmem + 384u + (uint32_t)(kk * 8), kd + off, idesc_s, kk > 0 ? 1u : 0u);
          umma_f16_ts(tmem + 128u + (uint32_t)(64 * b), tmem + 448u + (uint32_t)(kk * 8), vd + off, idesc_s,
                      kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[b]);
        umma_commit(&v_empty[vs]);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    int base = 0, it = 0;   // key tiles of the items before, items
    for (; ok; ++it) {
      if (!vl_wait(in_tmem, it & 1, p.status, kErrVlMma)) break;
      // (reduced over the warp: with it the descriptors below are known to be warp-uniform)
      const int n_kv = (int)__reduce_max_sync(0xffffffffu, s_head[it & 1] < 0 ? 0u : (unsigned)key_tiles(s_tile[it & 1]));
      if (n_kv == 0) break;
      const int end = base + n_kv;
      ok = issue_scores(base);
      for (int t = base; t < end && ok; ++t) {
        if (t + 1 < end && !issue_scores(t + 1)) { ok = false; break; }
        const int b = t & 1, ks = t % L::kKStages;
        if (!vl_wait(&ds_full[b], (t >> 1) & 1, p.status, kErrVlMma)) { ok = false; break; }
        if (t == base && it > 0 && !vl_wait(dq_read, (it - 1) & 1, p.status, kErrVlMma)) { ok = false; break; }
        tc_fence_after();
        const uint64_t kd = umma_desc_sw128_mnmajor(k_base + ks * L::kHalf, 8192u);
        if (elect_one_sync()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_f16_ts(tmem + 256u, tmem + (uint32_t)(64 * b + (kk >> 1) * 32 + (kk & 1) * 8), kd + (uint64_t)(kk * 128), idesc_q,
                        (t > base || kk > 0) ? 1u : 0u);
          umma_commit(&k_empty[ks]);
        }
        __syncwarp();
      }
      if (elect_one_sync()) umma_commit(dq_done);
      __syncwarp();
      base = end;
    }
    if (it > 0) mbar_wait(dq_done, (it - 1) & 1, nullptr, 0);   // every MMA issued has completed before TMEM can be freed
  } else {
    // ------------------------------------------------------------ dS + epilogue
    constexpr int LR = DP / 8, RI = 32 / LR, NI = 8 / RI;        // delta: lanes to a row, rows at once, steps
    int base = 0;              // key tiles of the items before
    for (int it = 0;; ++it) {
      // (the thread's places are formed again for each item: over the loop below they would
      // not fit beside its scores)
      const int tid = vl_tid(), wp = tid >> 5, lane = tid & 31;
      const int quad = wp & 3, half = (wp >> 2) & 1, g = wp >> 3, part = wp >> 2;
      const int row = quad * 32 + lane;
      const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
      const VlTile& w = s_tile[it & 1];
      float* xs = reinterpret_cast<float*>(smem + L::kX) + 128 * (it & 1);
      float lse_row = 0.0f;
      // eight rows of delta a warp: DP / 8 lanes to a row (whole lines), O from global, dO from the tile
      const int dchunk = lane % LR, drow0 = wp * 8 + lane / LR;
      // with the last scores of the item before, Q and dO may leave tensor memory
      if (it > 0 && !vl_wait(&s_full[(base - 1) & 1], ((base - 1) >> 1) & 1, p.status, kErrVlCompute)) break;
      if (!vl_wait(q_full, it & 1, p.status, kErrVlCompute)) break;
      const int h = s_head[it & 1];
      const bool more = h >= 0;
      if (more) {   // group 0 copies Q, group 1 dO, an atom each half: the first scores can start
        tc_fence_after();
        if (half < DP / 64)
          copy_row_to_tmem(smem + (g == 0 ? L::kQ : L::kDO) + half * 16384 + row * 128, row,
                           lane_base + 384u + (uint32_t)(64 * g + 32 * half));
        tmem_st_wait();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(in_tmem);
      if (more) {
        const int row0 = w.tile * 128;
        if (row0 + row < w.len) lse_row = vl_ld_f32(lse + (int64_t)h * p.T + w.start + row0 + row);
        uint4 ov[NI];
        uint2 lv[NI];
        const int left = dchunk * 8 < p.D ? w.len - row0 - drow0 : 0;   // rows from this lane's first
        int64_t at = ((int64_t)(w.start + row0 + drow0) * p.Hq + h) * p.D + dchunk * 8;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          ov[i] = make_uint4(0, 0, 0, 0);
          lv[i] = make_uint2(0, 0);
          if (i * RI < left) {
            ov[i] = vl_ld_u4(O + at);
            lv[i] = vl_ld_u2(low + at);
          }
          at += (int64_t)RI * p.Hq * p.D;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int r = drow0 + i * RI;
          const uint4 du = *reinterpret_cast<const uint4*>(smem + L::kDO + (dchunk >> 3) * 16384 + r * 128 +
                                                           (((dchunk & 7) ^ (r & 7)) << 4));
          const uint32_t dw[4] = {du.x, du.y, du.z, du.w}, ow[4] = {ov[i].x, ov[i].y, ov[i].z, ov[i].w};
          float acc = 0.0f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t lw = j == 0 ? lv[i].x : lv[i].y;
            const float2 a0 = vl_unpack<FP16>(dw[2 * j]), b0 = vl_unpack<FP16>(ow[2 * j]);
            const float2 a1 = vl_unpack<FP16>(dw[2 * j + 1]), b1 = vl_unpack<FP16>(ow[2 * j + 1]);
            acc = fmaf(a0.x, vl_with_low<FP16, 0>(b0.x, lw), acc);
            acc = fmaf(a0.y, vl_with_low<FP16, 1>(b0.y, lw), acc);
            acc = fmaf(a1.x, vl_with_low<FP16, 2>(b1.x, lw), acc);
            acc = fmaf(a1.y, vl_with_low<FP16, 3>(b1.y, lw), acc);
          }
          // (a row past the sequence's end: whatever its dO holds, O is 0 there, and NaN stays in the row)
#pragma unroll
          for (int o = LR / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
          if (dchunk == 0) xs[r] = acc;
        }
      }
      if (it > 0) {   // dQ of the item before, while the first scores of this one are formed
        if (!vl_wait(dq_done, (it - 1) & 1, p.status, kErrVlCompute)) break;
        tc_fence_after();
        const VlTile& b = s_tile[(it - 1) & 1];
        const int first = b.tile * 128 + quad * 32;
        uint16_t* out = dQ + ((int64_t)(b.start + first) * p.Hq + s_head[(it - 1) & 1]) * p.D;
        if (part < DP / 32)   // 32 columns a warp
          vl_store_rows<FP16, 32>(lane_base + 256u + (uint32_t)(part * 32), p.scale,
                                  smem + L::kStage + (part * 4 + quad) * 2048, out, (int64_t)p.Hq * p.D, part * 32, p.D,
                                  b.len - first);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dq_read);
      }
      if (!more) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(q_empty);   // (with the note of the item before read)
      if (!vl_wait(q_empty, it & 1, p.status, kErrVlCompute)) break;   // the other warps' delta
      const int len = w.len;
      const bool live = w.tile * 128 + row < len;
      const float l2 = lse_row * 1.4426950408889634f;
      const float dl = live ? xs[row] : 0.0f;
      if (g == 0 && half == 0 && live) {
        const int64_t at = (int64_t)h * p.stats_row + vl_stats_at(w) + w.tile * 128 + row;
        delta[at] = dl;
        nlse2[at] = -l2;
      }
      const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nl2 = f2_pack(-l2, -l2), dl2 = f2_pack(dl, dl);
      const uint32_t t_s = lane_base + (uint32_t)(64 * g + 32 * half);
      // keys that the row sees, from this half's first, and the sequence's end, both counted
      // from the CTA's first key tile
      const uint32_t limit = (live ? (p.causal ? w.tile * 128 + row + 1 : len) : 0) - 32 * half + base * 64u;
      const uint32_t keys = len + base * 64u;
      const int first = base;
      base += key_tiles(w);
      bool ok = true;
      for (int t = first + (g ^ (first & 1)); t < base; t += 2) {
        if (!vl_wait(&s_full[g], (t >> 1) & 1, p.status, kErrVlCompute)) { ok = false; break; }
        tc_fence_after();
        uint32_t s[32], dp[32];
        tmem_ld_32x32b_x32(t_s, s);
        tmem_ld_32x32b_x32(t_s + 128u, dp);
        tmem_ld_wait();
        const int seen = (int)(limit - t * 64u);
        const bool cut = __any_sync(0xffffffffu, seen < 32);
        uint32_t pk[16];
        // (with and without the mask apart: a branch in every step would keep the steps apart)
        auto form = [&](auto masked) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int c = 2 * i;
            float a0, a1, g0, g1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2, nl2), a0, a1);
            f2_unpack(f2_mul(f2_pack(fast_exp2(a0), fast_exp2(a1)),
                             f2_sub(f2_pack(__uint_as_float(dp[c]), __uint_as_float(dp[c + 1])), dl2)), g0, g1);
            if constexpr (decltype(masked)::value) {
              g0 = c >= seen ? 0.0f : g0;
              g1 = c + 1 >= seen ? 0.0f : g1;
            }
            pk[i] = vl_pack<FP16>(g0, g1);
          }
        };
        if (cut) form(std::true_type());
        else form(std::false_type());
        tmem_st_32x32b_x16(t_s, pk);   // over this half's own scores
        if (keys - t * 64u < 64u)   // the sequence ends inside this key tile (K_t has given its scores)
          vl_zero_rows<DP, 64>(smem + L::kK + (t % L::kKStages) * L::kHalf, (int)(keys - t * 64u), tid & 255);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[g]);
      }
      if (!ok) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 16) { tc_fence_after(); tmem_dealloc(tmem, 512); }
  if (*s_zero >= 0) vl_zero_outside(dQ, p.T, p.Hq, *s_zero, p.D, p.meta);
}

// ============================================================================
// dK and dV: one CTA per (128-key tile, kv head), over the query heads that share
// the kv head and their query tiles of 64.
//
//   Sᵀ_t = K Q_tᵀ, dPᵀ_t = V dO_tᵀ       M = 128 keys, N = 64 queries
//   dV += Pᵀ_t dO_t, dK += dSᵀ_t Q_t      A = Pᵀ / dSᵀ from tensor memory, B MN-major
// Two groups of eight warps take alternate query tiles (two threads to a key row, 32
// queries each);
// the scores of tile t + 1 are issued before the wait for Pᵀ/dSᵀ of tile t.
// Tensor memory: dV 0.., dK 128.., Sᵀ 256 + 128 b, dPᵀ 320 + 128 b (b = t & 1),
// Pᵀ and dSᵀ over the scores that they were formed from.  Q and dO come through rings of
// four tiles with the tile's -lse·log2(e) and delta.
//
// A query tile takes about 2200 cycles, of which its MMAs need 1800 (K and V from shared
// memory).  With K and V in tensor memory and steps of 32 queries they would need 1400, but
// the shorter steps' latency outweighs it: 231 us against 205 on the first case above.
//
// Where there are few key tiles a cluster of S CTAs shares one: CTA r takes every
// S-th of its query tiles, and at the end each writes its dV and dK (32 bits) into
// its own rings' memory, and sums one S-th of the columns over the cluster, in rank
// order - no atomics, the same result every time (8191 + 1037 rows, 8/2 heads: 589 us
// without clusters, 308 with two CTAs a tile, at that step of the kernel).
// ============================================================================
template <int DP>
struct VkSmem {
  static constexpr int kStages = 4;
  static constexpr int kTile = 128 * DP * 2, kHalf = 64 * DP * 2;
  static constexpr int kK = 0, kV = kTile, kQ = 2 * kTile, kDO = kQ + kStages * kHalf;
  static constexpr int kLD = kDO + kStages * kHalf;      // per stage: -lse·log2(e) [64], delta [64]
  static constexpr int kBar = kLD + kStages * 512;
  static constexpr int kBytes = kBar + 256 + 1024;
};

template <bool FP16, int DP>
__global__ void __launch_bounds__(kVbThreads, 1)
attn_varlen_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                       const __grid_constant__ VlParams p, const float* __restrict__ nlse2,
                       const float* __restrict__ delta, uint16_t* __restrict__ dK, uint16_t* __restrict__ dV) {
  using L = VkSmem<DP>;
  static_assert(2 * L::kStages * L::kHalf >= 2 * 128 * DP * 4, "the rings hold dV and dK in 32 bits");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* kv_full = bars;                          // K and V landed
  uint64_t* q_full = bars + 1;                       // [kStages]
  uint64_t* q_empty = q_full + L::kStages;
  uint64_t* o_full = q_empty + L::kStages;           // dO with the rows' statistics
  uint64_t* o_empty = o_full + L::kStages;
  uint64_t* s_full = o_empty + L::kStages;           // [2]
  uint64_t* p_full = s_full + 2;                     // [2], eight arrivals
  uint64_t* acc_done = p_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.split, rank = (int)(blockIdx.x % (unsigned)S);
  const int entry = blockIdx.x / (unsigned)S / p.Hk, hk = blockIdx.x / (unsigned)S % p.Hk;
  const VlTile w = p.tiles[entry];   // (read beside the count; past it the plan's other words)
  const int count = p.meta[p.count_at];
  if (entry >= count) {   // (all of a cluster)
    if (entry == count && rank == 0) {
      vl_zero_outside(dK, p.T, p.Hk, hk, p.D, p.meta);
      vl_zero_outside(dV, p.T, p.Hk, hk, p.D, p.meta);
    }
    return;
  }
  const int group = p.Hq / p.Hk, key0 = w.tile * 128;
  const int i0 = p.causal ? 2 * w.tile : 0;          // first 64-query tile that sees this key tile
  const int per_head = (w.len + 63) / 64 - i0;
  const int n_it = (group * per_head - rank + S - 1) / S;   // this CTA's; 0 where there are fewer tiles than CTAs
  const int stats_at = vl_stats_at(w);

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1);
      mbar_init(&o_full[i], 1); mbar_init(&o_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 8); }
    mbar_init(acc_done, 1);
    fence_mbar_init();
    prefetch_tmap(&tmQ); prefetch_tmap(&tmK); prefetch_tmap(&tmV); prefetch_tmap(&tmDO);
  }
  if (warp == 16) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 17) {
    // ------------------------------------------------------------ TMA loaders (Q with K and V; dO)
    if (lane == 0) {
      const bool is_q = warp == 17;
      if (is_q) {
        mbar_arrive_expect_tx(kv_full, 2 * L::kTile);
        vl_load_tile<DP, 128>(smem + L::kK, &tmK, kv_full, hk, w.start + key0);
        vl_load_tile<DP, 128>(smem + L::kV, &tmV, kv_full, hk, w.start + key0);
      }
      const CUtensorMap* map = is_q ? &tmQ : &tmDO;
      uint64_t* empty = is_q ? q_empty : o_empty;
      uint64_t* full = is_q ? q_full : o_full;
      uint8_t* ring = smem + (is_q ? L::kQ : L::kDO);
      int issued = 0, h = hk * group, it = i0 + rank;
      bool ok = true;
      for (int t = 0; t < n_it; ++t) {
        while (it >= i0 + per_head) { it -= per_head; ++h; }
        const int st = t % L::kStages;
        if (!mbar_wait(&empty[st], ((t / L::kStages) & 1) ^ 1, p.status, kErrVlLoad)) { ok = false; break; }
        mbar_arrive_expect_tx(&full[st], L::kHalf + (is_q ? 0 : 512));
        vl_load_tile<DP, 64>(ring + st * L::kHalf, map, &full[st], h, w.start + it * 64);
        if (!is_q) {  // this query tile's -lse·log2(e) and delta (256 B each)
          const int64_t at = (int64_t)h * p.stats_row + stats_at + it * 64;
          bulk_load(smem + L::kLD + st * 512, nlse2 + at, 256, &full[st]);
          bulk_load(smem + L::kLD + st * 512 + 256, delta + at, 256, &full[st]);
        }
        issued = t + 1;
        it += S;
      }
      if (is_q && n_it == 0) mbar_wait(kv_full, 0, nullptr, 0);   // nobody else waits for K and V
      if (!ok) {  // let every copy this thread issued land before the CTA can exit
        if (is_q) mbar_wait(kv_full, 0, nullptr, 0);
        for (int t = max(issued - L::kStages, 0); t < issued; ++t)
          mbar_wait(&full[t % L::kStages], (t / L::kStages) & 1, nullptr, 0);
      }
    }
  } else if (warp == 16) {
    // ------------------------------------------------------------ MMA issuer (whole warp)
    constexpr uint32_t idesc_s = vl_idesc<FP16>(128, 64, false);
    constexpr uint32_t idesc_g = vl_idesc<FP16>(128, DP, true);
    const uint64_t kd = umma_desc_sw128_kmajor(smem_u32(smem + L::kK)), vd = umma_desc_sw128_kmajor(smem_u32(smem + L::kV));
    const uint32_t q_base = smem_u32(smem + L::kQ), o_base = smem_u32(smem + L::kDO);
    auto issue_scores = [&](int t) -> bool {
      const int st = t % L::kStages;
      const uint32_t ph = (t / L::kStages) & 1, sc = tmem + 256u + 128u * (uint32_t)(t & 1);
      if (!vl_wait(&q_full[st], ph, p.status, kErrVlMma)) return false;
      if (!vl_wait(&o_full[st], ph, p.status, kErrVlMma)) return false;
      tc_fence_after();
      const uint64_t qd = umma_desc_sw128_kmajor(q_base + st * L::kHalf), od = umma_desc_sw128_kmajor(o_base + st * L::kHalf);
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint64_t ka = (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
          const uint64_t qa = (uint64_t)(((kk >> 2) * 8192 + (kk & 3) * 32) >> 4);
          umma_f16_ss(sc, kd + ka, qd + qa, idesc_s, kk > 0 ? 1u : 0u);
          umma_f16_ss(sc + 64u, vd + ka, od + qa, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t & 1]);
      }
      __syncwarp();
      return true;
    };
    bool ok = n_it > 0 && vl_wait(kv_full, 0, p.status, kErrVlMma) && issue_scores(0);
    for (int t = 0; t < n_it && ok; ++t) {
      if (t + 1 < n_it && !issue_scores(t + 1)) { ok = false; break; }
      if (!vl_wait(&p_full[t & 1], (t >> 1) & 1, p.status, kErrVlMma)) { ok = false; break; }
      tc_fence_after();
      const int st = t % L::kStages;
      const uint32_t sc = tmem + 256u + 128u * (uint32_t)(t & 1);
      const uint64_t qd = umma_desc_sw128_mnmajor(q_base + st * L::kHalf, 8192u);
      const uint64_t od = umma_desc_sw128_mnmajor(o_base + st * L::kHalf, 8192u);
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {   // dV += Pᵀ dO and dK += dSᵀ Q
          umma_f16_ts(tmem, sc + (uint32_t)((kk >> 1) * 32 + (kk & 1) * 8), od + (uint64_t)(kk * 128), idesc_g, (t > 0 || kk > 0) ? 1u : 0u);
          umma_f16_ts(tmem + 128u, sc + 64u + (uint32_t)((kk >> 1) * 32 + (kk & 1) * 8), qd + (uint64_t)(kk * 128), idesc_g,
                      (t > 0 || kk > 0) ? 1u : 0u);
        }
        umma_commit(&q_empty[st]);
        umma_commit(&o_empty[st]);
      }
      __syncwarp();
    }
    if (elect_one_sync()) umma_commit(acc_done);
    __syncwarp();
    mbar_wait(acc_done, 0, nullptr, 0);   // every MMA issued has completed before TMEM can be freed
  } else {
    // ------------------------------------------------------------ Pᵀ, dSᵀ + epilogue
    const int quad = warp & 3, half = (warp >> 2) & 1, g = warp >> 3;
    const int row = quad * 32 + lane, key = key0 + row;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t sc = lane_base + 256u + 128u * (uint32_t)g + 32u * (uint32_t)half;
    bool ok = true;
    int it = i0 + (rank + S * g) % per_head;
    for (int t = g; t < n_it; t += 2) {
      const int st = t % L::kStages;
      const float* sl = reinterpret_cast<const float*>(smem + L::kLD + st * 512) + 32 * half;
      // (o_full has completed by then; waiting on it makes the row statistics visible here)
      if (!vl_wait(&s_full[g], (t >> 1) & 1, p.status, kErrVlCompute) ||
          !vl_wait(&o_full[st], (t / L::kStages) & 1, p.status, kErrVlCompute)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t s[32], dp[32];
      tmem_ld_32x32b_x32(sc, s);
      tmem_ld_32x32b_x32(sc + 64u, dp);
      tmem_ld_wait();
      // queries [from, to) of the tile see this key (this half's first is 0)
      const int to = w.len - it * 64 - 32 * half;
      const int from = p.causal ? key - it * 64 - 32 * half : 0;
      const bool cut = to < 32 || __any_sync(0xffffffffu, from > 0);
      uint32_t pp[16], dsp[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // 4 queries per step: shared-memory broadcasts
        const float4 l4 = reinterpret_cast<const float4*>(sl)[i];
        const float4 d4 = reinterpret_cast<const float4*>(sl + 64)[i];
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
        float pr[4], ds[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = 4 * i + 2 * u;
          const uint64_t lv = u == 0 ? f2_pack(l4.x, l4.y) : f2_pack(l4.z, l4.w);
          const uint64_t dv2 = u == 0 ? f2_pack(d4.x, d4.y) : f2_pack(d4.z, d4.w);
          float a0, a1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2, lv), a0, a1);
          pr[2 * u] = fast_exp2(a0);
          pr[2 * u + 1] = fast_exp2(a1);
          f2_unpack(f2_mul(f2_pack(pr[2 * u], pr[2 * u + 1]),
                           f2_sub(f2_pack(__uint_as_float(dp[c]), __uint_as_float(dp[c + 1])), dv2)),
                    ds[2 * u], ds[2 * u + 1]);
        }
        if (cut) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (4 * i + u < from || 4 * i + u >= to) pr[u] = ds[u] = 0.0f;
        }
        pp[2 * i] = vl_pack<FP16>(pr[0], pr[1]);
        pp[2 * i + 1] = vl_pack<FP16>(pr[2], pr[3]);
        dsp[2 * i] = vl_pack<FP16>(ds[0], ds[1]);
        dsp[2 * i + 1] = vl_pack<FP16>(ds[2], ds[3]);
      }
      tmem_st_32x32b_x16(sc, pp);
      tmem_st_32x32b_x16(sc + 64u, dsp);
      if (w.len - it * 64 < 64) {   // the sequence ends inside this query tile (it has given its scores)
        vl_zero_rows<DP, 64>(smem + L::kQ + st * L::kHalf, w.len - it * 64, threadIdx.x & 255);
        vl_zero_rows<DP, 64>(smem + L::kDO + st * L::kHalf, w.len - it * 64, threadIdx.x & 255);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[g]);
      it += 2 * S;
      while (it >= i0 + per_head) it -= per_head;
    }
    ok = ok && vl_wait(acc_done, 0, p.status, kErrVlCompute);
    tc_fence_after();
    // group 0 has dV, group 1 dK; half of the columns a warp
    const int col0 = half * (DP / 2);
    const uint32_t acc = lane_base + (uint32_t)(128 * g + col0);
    if (S == 1) {
      // (K and V have given all their products: their memory stages the output)
      const int64_t at = ((int64_t)(w.start + key - lane) * p.Hk + hk) * p.D;
      if (ok)
        vl_store_rows<FP16, DP / 2>(acc, g == 0 ? 1.0f : p.scale, smem + L::kK + warp * (L::kTile / 8), (g == 0 ? dV : dK) + at,
                                    (int64_t)p.Hk * p.D, col0, p.D, w.len - (key - lane));
    } else {   // [column][row]: the lanes of a warp write one line
      float* mine = reinterpret_cast<float*>(smem + L::kQ) + g * DP * 128 + col0 * 128 + row;
#pragma unroll 1
      for (int c = 0; c < DP / 2; c += 32) {
        uint32_t o[32];
        if (n_it > 0) {
          tmem_ld_32x32b_x32(acc + (uint32_t)c, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) mine[(c + i) * 128] = n_it > 0 ? __uint_as_float(o[i]) : 0.0f;
      }
    }
  }

  if (S > 1) {
    __syncwarp();
    cluster_sync_all();   // every CTA's dV and dK are in its shared memory
    if (warp < 16) {
      const int g = warp >> 3, half = (warp >> 2) & 1, row = (warp & 3) * 32 + lane, key = key0 + row;
      const float f = g == 0 ? 1.0f : p.scale;
      const uint32_t mine = smem_u32(smem + L::kQ) + (uint32_t)((g * DP * 128 + row) * 4);
      uint16_t* out = (g == 0 ? dV : dK) + ((int64_t)(w.start + key) * p.Hk + hk) * p.D;
      const int cols = DP / S / 2;   // of each half
#pragma unroll 1
      for (int c = (2 * rank + half) * cols; c < (2 * rank + half + 1) * cols; c += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        for (int r = 0; r < S; ++r) {
          const uint32_t from = map_to_cta(mine, (uint32_t)r) + (uint32_t)(c * 512);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float x;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(from + (uint32_t)(i * 512)) : "memory");
            v[i] += x;
          }
        }
        if (key < w.len && c < p.D)
          *reinterpret_cast<uint4*>(out + c) =
              make_uint4(vl_pack<FP16>(v[0] * f, v[1] * f), vl_pack<FP16>(v[2] * f, v[3] * f),
                         vl_pack<FP16>(v[4] * f, v[5] * f), vl_pack<FP16>(v[6] * f, v[7] * f));
      }
    }
    __syncwarp();
    cluster_sync_all();   // read by all before a CTA's memory goes
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

}  // namespace zq

using namespace zq;

// The plan's integers: tile tables, scratch, meta (see the sizes in packed_plan_words).
static int64_t vl_cap(int64_t T, int64_t n, int rows) { return (T + rows - 1) / rows + n; }

int64_t packed_plan_words(int64_t T, int64_t n) {
  return 4 * (vl_cap(T, n, 256) + 2 * vl_cap(T, n, 128)) + kVlMeta + 3 * (n + 1);
}

// plan: int32 [packed_plan_words(T, n)], 16-byte aligned; positions (optional): int32 [T]
void packed_plan(at::Tensor cu, int64_t T, at::Tensor plan, c10::optional<at::Tensor> positions) {
  TORCH_CHECK(cu.is_cuda() && cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.dim() == 1 && cu.numel() >= 1,
              "packed_plan: cu_seqlens int32 [n + 1] on the GPU");
  const int64_t n = cu.numel() - 1;
  TORCH_CHECK(T >= 0 && T < (1LL << 30) && n < (1 << 24), "packed_plan: too many rows or sequences");
  TORCH_CHECK(plan.is_cuda() && plan.get_device() == cu.get_device() && plan.scalar_type() == at::kInt && plan.is_contiguous() &&
                  plan.numel() == packed_plan_words(T, n) && (reinterpret_cast<uintptr_t>(plan.data_ptr()) & 15) == 0,
              "packed_plan: plan int32 [packed_plan_words]");
  const bool rows = positions.has_value() && T > 0;
  TORCH_CHECK(!rows || (positions->is_cuda() && positions->get_device() == cu.get_device() &&
                        positions->scalar_type() == at::kInt && positions->is_contiguous() && positions->numel() == T),
              "packed_plan: positions int32 [T]");
  const c10::cuda::CUDAGuard guard(cu.device());
  const int64_t c256 = vl_cap(T, n, 256), c128 = vl_cap(T, n, 128);
  int* words = plan.data_ptr<int>();
  int* meta = words + 4 * (c256 + 2 * c128);
  const unsigned grid = 3 + (rows ? (unsigned)((T + kPlanThreads - 1) / kPlanThreads) : 0u);
  packed_plan_kernel<<<grid, kPlanThreads, 0, at::cuda::getCurrentCUDAStream()>>>(
      cu.data_ptr<int>(), (int)n, (int)T, (int)c256, (int)c128, reinterpret_cast<VlTile*>(words), meta + kVlMeta, meta,
      rows ? positions->data_ptr<int>() : nullptr, status_buffer(cu.get_device()));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// [T, H, D] as a 3-D map (D, H, T) with boxes of 64 columns x 1 head x box_rows rows
static CUtensorMap vl_tmap(const at::Tensor& t, int box_rows) {
  CUtensorMap map;
  const int64_t T = t.size(0), H = t.size(1), D = t.size(2);
  // the stride of an axis of one is never taken; the map wants a real one all the same
  const int64_t sh = H > 1 ? t.stride(1) : D, st = T > 1 ? t.stride(0) : H * D;
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 && t.stride(2) == 1 && sh % 8 == 0 && st % 8 == 0 && sh > 0 &&
                  st > 0,
              "attention: 16-byte aligned rows with unit stride");
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)(sh * 2), (cuuint64_t)(st * 2)};
  cuuint32_t box[3] = {64u, 1u, (cuuint32_t)box_rows};
  cuuint32_t estr[3] = {1u, 1u, 1u};
  const auto type = t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUresult r = get_encode_fn()(&map, type, 3, t.data_ptr(), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "attention: cuTensorMapEncodeTiled failed with code ", (int)r);
  return map;
}

struct VlCall {
  VlParams p;
  int64_t c256, c128, n;
  bool fp16, narrow;
};

static VlCall vl_check(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& plan, int64_t n,
                       bool causal, double scale) {
  TORCH_CHECK(q.is_cuda() && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) && q.dim() == 3,
              "attention: bf16 or fp16 [T, H, D] CUDA tensors");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), Hk = k.dim() == 3 ? k.size(1) : 0;
  for (const at::Tensor* t : {&k, &v})
    TORCH_CHECK(t->is_cuda() && t->get_device() == q.get_device() && t->scalar_type() == q.scalar_type() && t->dim() == 3 &&
                    t->size(0) == T && t->size(1) == Hk && t->size(2) == D,
                "attention: k and v [T, Hk, D] like q");
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "attention: head width a multiple of 8 up to 128");
  TORCH_CHECK(T > 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0, "attention: rows, and Hq a multiple of Hk");
  TORCH_CHECK(scale > 0, "attention: scale must be positive");
  TORCH_CHECK(plan.is_cuda() && plan.get_device() == q.get_device() && plan.scalar_type() == at::kInt && plan.is_contiguous() &&
                  n >= 0 && plan.numel() == packed_plan_words(T, n),
              "attention: the plan is another division's");
  VlCall c;
  c.c256 = vl_cap(T, n, 256);
  c.c128 = vl_cap(T, n, 128);
  c.n = n;
  TORCH_CHECK((c.c128 + 1) * Hq * kVlMaxSplit < (1LL << 31), "attention: grid too large");
  const int* words = plan.data_ptr<int>();
  c.p = VlParams{reinterpret_cast<const VlTile*>(words), words + 4 * (c.c256 + 2 * c.c128), 0, (int)T, (int)Hq, (int)Hk,
                 (int)D, causal ? 1 : 0, (int)vl_stats_row(T, c.c128), 1, (float)scale, (float)(scale * 1.4426950408889634),
                 status_buffer(q.get_device())};
  c.fp16 = q.scalar_type() == at::kHalf;
  c.narrow = D <= 64;
  return c;
}

static uint16_t* vl_out(const at::Tensor& t, const at::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == like.get_device() && t.scalar_type() == like.scalar_type() && t.is_contiguous() &&
                  t.sizes() == like.sizes() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
              "attention: outputs are contiguous and like their inputs");
  return reinterpret_cast<uint16_t*>(t.data_ptr());
}

template <typename K>
static void vl_smem(K kern, int bytes, bool (&done)[64], int dev) {
  if (done[dev]) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done[dev] = true;
}

template <bool FP16, int DP>
static void vl_launch_fwd(const VlCall& c, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, uint16_t* o,
                          float* lse, uint8_t* low, int dev) {
  static bool done[64] = {false};
  auto kern = attn_varlen_fwd_kernel<FP16, DP>;
  vl_smem(kern, VfSmem<DP>::kBytes, done, dev);
  kern<<<(unsigned)((c.c256 + 1) * c.p.Hq), kVfThreads, VfSmem<DP>::kBytes, at::cuda::getCurrentCUDAStream()>>>(tq, tk, tv, c.p,
                                                                                                               o, lse, low);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

static uint8_t* vl_low(const at::Tensor& low, const at::Tensor& q) {
  TORCH_CHECK(low.is_cuda() && low.get_device() == q.get_device() && low.scalar_type() == at::kChar && low.is_contiguous() &&
                  low.sizes() == q.sizes() && (reinterpret_cast<uintptr_t>(low.data_ptr()) & 7) == 0,
              "attention: the low bytes of o are int8, contiguous, like q");
  return reinterpret_cast<uint8_t*>(low.data_ptr());
}

// o [T, Hq, D] contiguous; lse [Hq, T] fp32 and, for a backward, low [T, Hq, D] int8
// (the rows of no sequence are not written in these)
void attn_varlen_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor plan, int64_t n, at::Tensor o, at::Tensor lse,
                     c10::optional<at::Tensor> low, bool causal, double scale) {
  VlCall c = vl_check(q, k, v, plan, n, causal, scale);
  uint16_t* op = vl_out(o, q);
  TORCH_CHECK(lse.is_cuda() && lse.get_device() == q.get_device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.numel() == q.size(0) * q.size(1),
              "attention: lse [Hq, T] fp32");
  const c10::cuda::CUDAGuard guard(q.device());
  const CUtensorMap tq = vl_tmap(q, 128), tk = vl_tmap(k, 128), tv = vl_tmap(v, 128);
  c.p.count_at = 0;
  auto go = c.fp16 ? (c.narrow ? vl_launch_fwd<true, 64> : vl_launch_fwd<true, 128>)
                   : (c.narrow ? vl_launch_fwd<false, 64> : vl_launch_fwd<false, 128>);
  go(c, tq, tk, tv, op, lse.data_ptr<float>(), low.has_value() ? vl_low(*low, q) : nullptr, q.get_device());
}

struct VlBwd {
  CUtensorMap q128, do128, k64, v64, q64, do64, k128, v128;
  const uint16_t* o;
  const uint8_t* low;
  const float* lse;
  float *delta, *nlse2;
  uint16_t *dq, *dk, *dv;
};

template <bool FP16, int DP>
static void vl_launch_bwd(VlCall& c, const VlBwd& b, int dev) {
  static bool done_q[64] = {false}, done_k[64] = {false};
  auto kq = attn_varlen_dq_kernel<FP16, DP>;
  auto kk = attn_varlen_dkv_kernel<FP16, DP>;
  vl_smem(kq, VqSmem<DP>::kBytes, done_q, dev);
  vl_smem(kk, VkSmem<DP>::kBytes, done_k, dev);
  auto stream = at::cuda::getCurrentCUDAStream();
  const VlTile* tiles = c.p.tiles;
  c.p.count_at = 1;
  c.p.tiles = tiles + c.c256;
  kq<<<(unsigned)((c.c128 + 1) * c.p.Hq), kVbThreads, VqSmem<DP>::kBytes, stream>>>(b.q128, b.k64, b.v64, b.do128, c.p, b.o, b.low,
                                                                                   b.lse,
                                                                                   b.delta, b.nlse2, b.dq);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  c.p.count_at = 2;
  c.p.tiles = tiles + c.c256 + c.c128;
  // A cluster to a key tile where the tiles are too few to even out over the SMs, as
  // long as each of its CTAs keeps about eight query tiles of 64 on average (the exchange
  // at the end takes about 3 us).
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int64_t work = c.c128 * c.p.Hk;
  const int64_t each = (int64_t)(c.p.Hq / c.p.Hk) * c.p.T / std::max<int64_t>(c.n, 1) / (c.p.causal ? 128 : 64);
  c.p.split = work <= sms && each >= 32 ? 4 : work <= 3 * sms && each >= 16 ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((c.c128 + 1) * c.p.Hk * c.p.split));
  cfg.blockDim = dim3(kVbThreads);
  cfg.dynamicSmemBytes = VkSmem<DP>::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c.p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kk, b.q64, b.k128, b.v128, b.do64, c.p, (const float*)b.nlse2, (const float*)b.delta,
                                    b.dk, b.dv));
}

// dq, dk, dv (contiguous) from dout, the forward's inputs, o, lse and low: two launches
void attn_varlen_bwd(at::Tensor dout, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o, at::Tensor lse, at::Tensor low,
                     at::Tensor plan, int64_t n, at::Tensor dq, at::Tensor dk, at::Tensor dv, bool causal, double scale) {
  VlCall c = vl_check(q, k, v, plan, n, causal, scale);
  TORCH_CHECK(dout.is_cuda() && dout.get_device() == q.get_device() && dout.scalar_type() == q.scalar_type() &&
                  dout.sizes() == q.sizes(),
              "attention backward: dout like q");
  TORCH_CHECK(lse.is_cuda() && lse.get_device() == q.get_device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.numel() == q.size(0) * q.size(1),
              "attention: lse [Hq, T] fp32");
  const c10::cuda::CUDAGuard guard(q.device());
  auto stats = at::empty({2, q.size(1), c.p.stats_row}, lse.options());
  VlBwd b{vl_tmap(q, 128), vl_tmap(dout, 128), vl_tmap(k, 64), vl_tmap(v, 64), vl_tmap(q, 64), vl_tmap(dout, 64), vl_tmap(k, 128),
          vl_tmap(v, 128), vl_out(o, q), vl_low(low, q), lse.data_ptr<float>(), stats.data_ptr<float>(),
          stats.data_ptr<float>() + stats.numel() / 2, vl_out(dq, q), vl_out(dk, k), vl_out(dv, v)};
  auto go = c.fp16 ? (c.narrow ? vl_launch_bwd<true, 64> : vl_launch_bwd<true, 128>)
                   : (c.narrow ? vl_launch_bwd<false, 64> : vl_launch_bwd<false, 128>);
  go(c, b, q.get_device());
}
