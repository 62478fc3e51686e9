// Embedding lookup with scaling, and the gradient of its table by sorted tokens.
//
//   y_i = s W[id_i], rounded once; an id outside [0, V) gives a row of zeros
//   dW_v = s sum over i with id_i = v of dy_i, in 32 bits, rounded once; other rows 0
//
// Backward.  The (id, token) pairs are sorted by id, equal ids in token order (a radix sort of
// 9-bit digits, least significant first, each pass stable): in one block's shared memory up
// to kSortTile tokens, in passes over all blocks' tiles above that.  Then a warp takes kPiece
// sorted tokens and 256 columns and adds the tokens' rows up in order; a run of one id inside a
// piece is a finished row of dW.  Blocks beyond these write zeros over the rows that no token
// has (each lane looks its row up among the sorted ids); the table's first rows are filled with
// zeros as a whole by blocks beyond the sort's, as many as memory takes while it sorts.  Runs that cross pieces leave partial
// sums, which a last kernel adds in piece order.  No atomics on values, so a gradient is the same
// bits from run to run, and no run is longer than a piece for any warp, however often an id
// occurs.
//
// What bounds it: memory; the zeros of a large table are most of it.  Measured: 8192 tokens
// against 152064 x 3584 bf16: lookup 17 us, sort 20 (zeros meanwhile), sums and zeros 162 to 174, joins 7;
// 40013 x 1001 fp32, rows on odd boundaries: sums 81 us, four sort launches 60.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>

#include "rows.cuh"

namespace zq {

constexpr int kEmbWarps = 8;
constexpr int kPiece = 32;             // sorted tokens of a warp
constexpr int kRadixBits = 9, kRadix = 1 << kRadixBits;
constexpr int kSortWarps = 32, kSortItems = 8;
constexpr int kSortTile = kSortWarps * 32 * kSortItems;   // tokens that a block ranks: 8192

__device__ __forceinline__ int emb_id(const void* ids, int ids64, int64_t i, int V) {
  const int64_t v = ids64 ? reinterpret_cast<const int64_t*>(ids)[i] : (int64_t)reinterpret_cast<const int32_t*>(ids)[i];
  return v >= 0 && v < V ? (int)v : -1;
}

// A unit is one token and 256 columns; a warp takes U of them.
template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kEmbWarps * 32) embedding_fwd_kernel(const void* __restrict__ ids, int ids64,
                                                                       const T* __restrict__ w, int64_t ws,
                                                                       T* __restrict__ y, int64_t units, int tiles, int V,
                                                                       int D, float scale) {
  const int lane = threadIdx.x & 31;
  const int64_t first = ((int64_t)blockIdx.x * kEmbWarps + (threadIdx.x >> 5)) * U;
  if (first >= units) return;
  const int n = (int)min((int64_t)U, units - first);
  uint32_t row = (uint32_t)first / (uint32_t)tiles, tile = (uint32_t)first - row * (uint32_t)tiles;
  int64_t at[U];
  int base[U], id[U];
  uint32_t here = 0;   // bit j: the id is in the table
#pragma unroll
  for (int j = 0; j < U; ++j) {
    at[j] = row;
    base[j] = (int)tile * kTile;
    if (++tile == (uint32_t)tiles) tile = 0, ++row;
    id[j] = j < n ? emb_id(ids, ids64, at[j], V) : -1;
    here |= (id[j] >= 0 ? 1u : 0u) << j;
  }
  RawTile<T, VEC> t[U];
#pragma unroll
  for (int j = 0; j < U; ++j) t[j].load(w + max(id[j], 0) * ws, base[j], lane, id[j] >= 0 ? D : 0);
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      float v[8];
      t[j].values(v);
      // (an absent id's zeros times a scale that is not finite, or negative, would be NaN or -0)
      const float s = here >> j & 1u ? scale : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= s;
      store_tile<T, VEC>(y + at[j] * D, base[j], lane, D, v);
    }
  }
}

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------
// Ids outside the table sort behind all others (as V).
__device__ __forceinline__ uint32_t sort_key(const void* ids, int ids64, int64_t i, int V) {
  const int v = emb_id(ids, ids64, i, V);
  return v < 0 ? (uint32_t)V : (uint32_t)v;
}

// Ranks of a block's items by a digit, in order: every warp has kSortItems * 32 consecutive
// items, `count` of its digits so far in its row of s_count; the lanes of a step with equal
// digits are found by ballots over the digit's bits.
struct SortRank {
  uint32_t peers_before, peers;
};
__device__ __forceinline__ SortRank digit_peers(uint32_t digit, bool valid, int lane) {
  uint32_t m = __ballot_sync(0xffffffffu, valid);
#pragma unroll
  for (int b = 0; b < kRadixBits; ++b) {
    const uint32_t set = __ballot_sync(0xffffffffu, (digit >> b) & 1u);
    m &= (digit >> b) & 1u ? set : ~set;
  }
  return SortRank{(uint32_t)__popc(m & ((1u << lane) - 1u)), (uint32_t)__popc(m)};
}

// (digits of this warp before the step) + (of the lanes before); counts go up
__device__ __forceinline__ uint32_t rank_step(uint16_t* mine, uint32_t digit, bool valid, int lane) {
  const SortRank r = digit_peers(digit, valid, lane);
  uint32_t before = 0;
  if (valid) before = mine[digit];
  __syncwarp();
  if (valid && r.peers_before == 0) mine[digit] = (uint16_t)(before + r.peers);
  __syncwarp();
  return before + r.peers_before;
}

// Zeros over `bytes` bytes by a warp.
__device__ __forceinline__ void zero_range(uint8_t* p, int64_t bytes, int lane) {
  const int64_t head = min(bytes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15));
  for (int64_t i = lane; i < head; i += 32) p[i] = 0;
  p += head, bytes -= head;
  const int64_t vecs = bytes / 16;
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 4
  for (int64_t i = lane; i < vecs; i += 32) reinterpret_cast<uint4*>(p)[i] = z;
  for (int64_t i = vecs * 16 + lane; i < bytes; i += 32) p[i] = 0;
}

// Zeros over `bytes` bytes by the blocks from `first` on.
struct ZeroShare {
  uint8_t* p;
  int64_t bytes;
};
constexpr int64_t kZeroChunk = 16384;
__device__ __forceinline__ void zero_share(const ZeroShare& z, int first) {
  const int warps = blockDim.x / 32, lane = threadIdx.x & 31;
  const int64_t step = (int64_t)(gridDim.x - first) * warps * kZeroChunk;
  for (int64_t at = ((int64_t)(blockIdx.x - first) * warps + threadIdx.x / 32) * kZeroChunk; at < z.bytes; at += step)
    zero_range(z.p + at, min(kZeroChunk, z.bytes - at), lane);
}

// Exclusive sums of s_count[warp][digit] in the order digit, warp (u16: at most kSortTile),
// by 1024 threads: each takes a digit's run of kRun warps.
__device__ __forceinline__ void scan_counts(uint16_t (*s_count)[kRadix], uint32_t* s_sum) {
  constexpr int kRun = kSortWarps * kRadix / (kSortWarps * 32);   // counters of a thread: 16
  constexpr int kRuns = kSortWarps / kRun;                        // threads of a digit: 2
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int digit = tid / kRuns, w0 = (tid % kRuns) * kRun;
  uint32_t sum = 0, v[kRun];
#pragma unroll
  for (int i = 0; i < kRun; ++i) v[i] = s_count[w0 + i][digit], sum += v[i];
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    uint32_t w = s_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    s_sum[lane] = w;
  }
  __syncthreads();
  uint32_t at = incl - sum + (warp > 0 ? s_sum[warp - 1] : 0u);
#pragma unroll
  for (int i = 0; i < kRun; ++i) s_count[w0 + i][digit] = (uint16_t)at, at += v[i];
  __syncthreads();
}

// One block sorts up to kSortTile tokens.  (n_cross: see the sums)
__global__ void __launch_bounds__(kSortWarps * 32) embedding_sort_block_kernel(const void* __restrict__ ids, int ids64, int T,
                                                                               int V, int passes, int32_t* __restrict__ keys,
                                                                               int32_t* __restrict__ order,
                                                                               int32_t* __restrict__ n_cross, const ZeroShare zero) {
  if (blockIdx.x > 0) return zero_share(zero, 1);
  if (threadIdx.x == 0) *n_cross = 0;
  extern __shared__ uint8_t emb_smem[];
  uint16_t(*s_count)[kRadix] = reinterpret_cast<uint16_t(*)[kRadix]>(emb_smem);           // 32 KB
  uint32_t* s_key = reinterpret_cast<uint32_t*>(emb_smem + kSortWarps * kRadix * 2);      // 32 KB
  uint16_t* s_at = reinterpret_cast<uint16_t*>(s_key + kSortTile);                        // 16 KB
  __shared__ uint32_t s_sum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per_warp = ((T + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;   // consecutive items of a warp
  uint32_t key[kSortItems], token[kSortItems];
  bool valid[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int i = warp * per_warp + j * 32 + lane;
    valid[j] = j * 32 < per_warp && i < T;
    key[j] = valid[j] ? sort_key(ids, ids64, i, V) : 0u;
    token[j] = (uint32_t)i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * kRadixBits;
    for (int i = lane; i < kRadix / 2; i += 32) reinterpret_cast<uint32_t*>(s_count[warp])[i] = 0u;
    __syncwarp();
    uint32_t rank[kSortItems];
#pragma unroll
    for (int j = 0; j < kSortItems; ++j)
      if (j * 32 < per_warp) rank[j] = rank_step(s_count[warp], (key[j] >> shift) & (kRadix - 1), valid[j], lane);
    __syncthreads();
    scan_counts(s_count, s_sum);
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      if (valid[j]) {
        const uint32_t to = s_count[warp][(key[j] >> shift) & (kRadix - 1)] + rank[j];
        s_key[to] = key[j];
        s_at[to] = (uint16_t)token[j];
      }
    }
    __syncthreads();
    if (pass + 1 < passes) {
#pragma unroll
      for (int j = 0; j < kSortItems; ++j) {
        const int i = warp * per_warp + j * 32 + lane;
        if (valid[j]) key[j] = s_key[i], token[j] = s_at[i];
      }
    }
  }
  for (int i = tid; i < T; i += blockDim.x) keys[i] = (int32_t)s_key[i], order[i] = (int32_t)s_at[i];
}

// One pass over many tiles: the tiles' counts of a digit's values ...
template <bool FIRST>
__global__ void __launch_bounds__(kSortWarps * 32) embedding_count_kernel(const void* __restrict__ ids, int ids64, int64_t T,
                                                                          int V, int shift,
                                                                          uint32_t* __restrict__ counts,
                                                                          int32_t* __restrict__ n_cross, int tiles,
                                                                          const ZeroShare zero) {
  if ((int)blockIdx.x >= tiles) return zero_share(zero, tiles);
  if (FIRST && blockIdx.x == 0 && threadIdx.x == 0) *n_cross = 0;
  __shared__ uint32_t s_n[kRadix];
  const int tid = threadIdx.x;
  if (tid < kRadix) s_n[tid] = 0u;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = first + j * kSortWarps * 32 + tid;
    if (i < T) {
      const uint32_t key = FIRST ? sort_key(ids, ids64, i, V) : (uint32_t)reinterpret_cast<const int32_t*>(ids)[i];
      atomicAdd(&s_n[(key >> shift) & (kRadix - 1)], 1u);   // (a count: the same whatever the order)
    }
  }
  __syncthreads();
  if (tid < kRadix) counts[(int64_t)blockIdx.x * kRadix + tid] = s_n[tid];
}

// ... and the tiles' items to their places: each block sums the counts before its own.
template <bool FIRST>
__global__ void __launch_bounds__(kSortWarps * 32) embedding_place_kernel(const void* __restrict__ ids, int ids64,
                                                                          const int32_t* __restrict__ from, int64_t T, int V,
                                                                          int shift, int tiles,
                                                                          const uint32_t* __restrict__ counts,
                                                                          int32_t* __restrict__ keys,
                                                                          int32_t* __restrict__ order, const ZeroShare zero) {
  if ((int)blockIdx.x >= tiles) return zero_share(zero, tiles);
  extern __shared__ uint8_t emb_smem[];
  uint16_t(*s_count)[kRadix] = reinterpret_cast<uint16_t(*)[kRadix]>(emb_smem);
  __shared__ uint32_t s_base[kRadix], s_total[kRadix];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kRadix) {   // a digit's tiles: those before this one, and all
    uint32_t before = 0, all = 0;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
      const uint32_t c = counts[(int64_t)t * kRadix + tid];
      all += c;
      before += t < (int)blockIdx.x ? c : 0u;
    }
    s_base[tid] = before, s_total[tid] = all;
  }
  const int64_t first = (int64_t)blockIdx.x * kSortTile + warp * kSortItems * 32;
  uint32_t key[kSortItems], token[kSortItems], rank[kSortItems];
  bool valid[kSortItems];
  for (int i = lane; i < kRadix / 2; i += 32) reinterpret_cast<uint32_t*>(s_count[warp])[i] = 0u;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = first + j * 32 + lane;
    valid[j] = i < T;
    key[j] = !valid[j] ? 0u : FIRST ? sort_key(ids, ids64, i, V) : (uint32_t)reinterpret_cast<const int32_t*>(ids)[i];
    token[j] = !valid[j] ? 0u : FIRST ? (uint32_t)i : (uint32_t)from[i];
  }
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) rank[j] = rank_step(s_count[warp], (key[j] >> shift) & (kRadix - 1), valid[j], lane);
  __syncthreads();
  // digits before this one, over all tiles; then this tile's warps before this one
  if (warp == 0) {
    uint32_t run = 0;
    for (int d = lane * (kRadix / 32); d < (lane + 1) * (kRadix / 32); ++d) run += s_total[d];
    uint32_t incl = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    uint32_t at = incl - run;
    for (int d = lane * (kRadix / 32); d < (lane + 1) * (kRadix / 32); ++d) {
      s_base[d] += at;
      at += s_total[d];
    }
  }
  if (tid < kRadix) {
    uint32_t at = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = s_count[w][tid];
      s_count[w][tid] = (uint16_t)at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    if (valid[j]) {
      const uint32_t digit = (key[j] >> shift) & (kRadix - 1);
      const uint32_t to = s_base[digit] + s_count[warp][digit] + rank[j];
      keys[to] = (int32_t)key[j];
      order[to] = (int32_t)token[j];
    }
  }
}

// ---------------------------------------------------------------------------
// sums
// ---------------------------------------------------------------------------
// 32 rows of the table from `first` on: zeros over those that no token has.
__device__ __forceinline__ void zero_rows(const int32_t* __restrict__ keys, int64_t tokens, uint8_t* dw, int64_t row_bytes,
                                          int64_t first, int V, int lane) {
  const int64_t row = first + lane;
  int64_t lo = 0, hi = tokens;   // first token whose id is not below the row's
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < row) lo = mid + 1;
    else hi = mid;
  }
  uint32_t absent = __ballot_sync(0xffffffffu, row < V && (lo == tokens || keys[lo] != row));
  while (absent != 0) {   // consecutive ones are one range
    const int from = __ffs(absent) - 1;
    const uint32_t run = ~(absent >> from);
    const int n = run == 0u ? 32 : __ffs(run) - 1;
    zero_range(dw + (first + from) * row_bytes, n * row_bytes, lane);
    absent = from + n >= 32 ? 0u : absent >> (from + n) << (from + n);
  }
}

// Partial sums [pieces, 2, D]: of the run that a piece starts with and that began before it
// (0; also where it goes on behind the piece), and of the one that it starts and that goes
// on behind it (1).  Pieces with one of the latter are listed for the join (in any order).
// Warps behind the pieces' write zeros.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kEmbWarps * 32) embedding_sum_kernel(const int32_t* __restrict__ keys,
                                                                       const int32_t* __restrict__ order, int64_t tokens,
                                                                       const T* __restrict__ dy, int64_t dys,
                                                                       T* __restrict__ dw, float* __restrict__ part,
                                                                       int32_t* __restrict__ n_cross,
                                                                       int32_t* __restrict__ cross, int sum_blocks,
                                                                       int64_t zero_from, int tiles,
                                                                       int V, int D, float scale) {
  const int lane = threadIdx.x & 31;
  if ((int)blockIdx.x >= sum_blocks) {
    const int64_t first = zero_from + ((int64_t)(blockIdx.x - sum_blocks) * kEmbWarps + (threadIdx.x >> 5)) * 32;
    if (first < V) zero_rows(keys, tokens, reinterpret_cast<uint8_t*>(dw), (int64_t)D * sizeof(T), first, V, lane);
    return;
  }
  const int64_t unit = (int64_t)blockIdx.x * kEmbWarps + (threadIdx.x >> 5);
  const int64_t piece = unit / tiles, begin = piece * kPiece;
  if (begin >= tokens) return;
  const int base = (int)(unit - piece * tiles) * kTile;
  const int n = (int)min((int64_t)kPiece, tokens - begin);
  // lane i holds sorted token i; the ids on both sides of the piece
  const int key = lane < n ? keys[begin + lane] : -1;
  const int tok = lane < n ? order[begin + lane] : 0;
  const int before = begin > 0 ? keys[begin - 1] : -1;
  const int after = begin + n < tokens ? keys[begin + n] : -1;
  constexpr int B = 8;   // rows under way
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
  int run = 0;   // first token of the run
#pragma unroll 1
  for (int j0 = 0; j0 < n; j0 += B) {
    RawTile<T, VEC> t[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int64_t row = __shfl_sync(0xffffffffu, tok, (j0 + j) & 31);
      const int k = __shfl_sync(0xffffffffu, key, (j0 + j) & 31);
      t[j].load(dy + row * dys, base, lane, j0 + j < n && k < V ? D : 0);
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int at = j0 + j;
      if (at < n) {
        float v[8];
        t[j].values(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += v[i];
        const int k = __shfl_sync(0xffffffffu, key, at);
        const int next = at + 1 < n ? __shfl_sync(0xffffffffu, key, (at + 1) & 31) : after;
        if (at + 1 == n || next != k) {   // the run ends here, or goes on behind the piece
          if (k < V) {
            const bool began_before = run == 0 && before == k, goes_on = at + 1 == n && next == k;
            if (began_before || goes_on) {
              if (!began_before && base == 0 && lane == 0) cross[atomicAdd(n_cross, 1)] = (int32_t)piece;
              store_tile<float, VEC>(part + (piece * 2 + (began_before ? 0 : 1)) * D, base, lane, D, sum);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) sum[i] *= scale;
              store_tile<T, VEC>(dw + (int64_t)k * D, base, lane, D, sum);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
          run = at + 1;
        }
      }
    }
  }
}

// A block takes a listed piece and 256 columns: the pieces' partial sums of the run that starts
// there and goes on.  Its warps take the pieces in turn and are added in warp order.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kEmbWarps * 32) embedding_join_kernel(const int32_t* __restrict__ keys, int64_t tokens,
                                                                        const float* __restrict__ part, T* __restrict__ dw,
                                                                        const int32_t* __restrict__ n_cross,
                                                                        const int32_t* __restrict__ cross, int tiles, int D,
                                                                        float scale) {
  __shared__ float s_sum[kEmbWarps][kTile];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t units = (int64_t)*n_cross * tiles;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int64_t piece = cross[unit / tiles];
    const int base = (int)(unit % tiles) * kTile;
    const int k = keys[(piece + 1) * kPiece - 1];
    // pieces behind this one that the run goes through or ends in: those that start with k
    const int64_t pieces = (tokens + kPiece - 1) / kPiece;
    int64_t n = 0;
    for (;;) {
      const int64_t q = piece + 1 + n + lane;
      const uint32_t in = __ballot_sync(0xffffffffu, q < pieces && keys[q * kPiece] == k);
      const int got = in == 0xffffffffu ? 32 : __ffs(~in) - 1;
      n += got;
      if (got < 32) break;
    }
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
#pragma unroll 4
    for (int64_t j = warp; j <= n; j += kEmbWarps) {
      RawTile<float, VEC> t;
      t.load(part + ((piece + j) * 2 + (j == 0 ? 1 : 0)) * D, base, lane, D);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += __uint_as_float(t.w[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s_sum[warp][i * 32 + lane] = sum[i];
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int w = 1; w < kEmbWarps; ++w)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += s_sum[w][i * 32 + lane];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] *= scale;
      store_tile<T, VEC>(dw + (int64_t)k * D, base, lane, D, sum);
    }
    __syncthreads();   // (before the next one's sums)
  }
}

}  // namespace zq

using namespace zq;

namespace {

bool emb_aligned(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 &&
         (t.size(0) < 2 || t.stride(0) * t.element_size() % 16 == 0);
}

void emb_check(const at::Tensor& ids, const at::Tensor& table, const at::Tensor& rows) {
  TORCH_CHECK(table.is_cuda() && table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0 &&
                  (table.stride(1) == 1 || table.size(1) == 1),
              "embedding: weight [V, D] on the GPU, unit column stride");
  TORCH_CHECK(table.size(0) < (1LL << 31) && table.size(1) < (1LL << 30), "embedding: less than 2^31 rows, 2^30 columns");
  TORCH_CHECK(ids.is_cuda() && ids.get_device() == table.get_device() && ids.is_contiguous() &&
                  (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong) && ids.numel() > 0 &&
                  ids.numel() < (1LL << 31),
              "embedding: ids int32 or int64, contiguous, on the weight's device");
  TORCH_CHECK(rows.is_cuda() && rows.get_device() == table.get_device() && rows.scalar_type() == table.scalar_type() &&
                  rows.dim() == 2 && rows.size(0) == ids.numel() && rows.size(1) == table.size(1) &&
                  (rows.stride(1) == 1 || rows.size(1) == 1),
              "embedding: rows [T, D] of the weight's type");
}

}  // namespace

#define ZQ_EMB_TYPES(TYPE, ...)                                                \
  switch (TYPE) {                                                              \
    case at::kBFloat16: { using T = __nv_bfloat16; __VA_ARGS__; break; }       \
    case at::kHalf: { using T = __half; __VA_ARGS__; break; }                  \
    case at::kFloat: { using T = float; __VA_ARGS__; break; }                  \
    default: TORCH_CHECK(false, "embedding: bf16, fp16 or fp32");              \
  }

// y [T, D]
void embedding_fwd(at::Tensor ids, at::Tensor w, at::Tensor y, double scale) {
  emb_check(ids, w, y);
  TORCH_CHECK(y.is_contiguous(), "embedding: contiguous output");
  const c10::cuda::CUDAGuard guard(w.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int V = (int)w.size(0), D = (int)w.size(1), tiles = (D + kTile - 1) / kTile;
  const int64_t units = ids.numel() * tiles;
  TORCH_CHECK(units < (1LL << 32), "embedding: too many tokens");
  const int ids64 = ids.scalar_type() == at::kLong;
  constexpr int U = 4;
  const unsigned grid = (unsigned)((units + kEmbWarps * U - 1) / (kEmbWarps * U));
  ZQ_EMB_TYPES(w.scalar_type(), {
    const T* wp = reinterpret_cast<const T*>(w.data_ptr());
    T* yp = reinterpret_cast<T*>(y.data_ptr());
    if (D % 8 == 0 && emb_aligned(w) && emb_aligned(y))
      embedding_fwd_kernel<T, true, U><<<grid, kEmbWarps * 32, 0, stream>>>(ids.data_ptr(), ids64, wp, w.stride(0), yp, units,
                                                                            tiles, V, D, (float)scale);
    else
      embedding_fwd_kernel<T, false, U><<<grid, kEmbWarps * 32, 0, stream>>>(ids.data_ptr(), ids64, wp, w.stride(0), yp, units,
                                                                             tiles, V, D, (float)scale);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// dw [V, D] from dy [T, D]
void embedding_bwd(at::Tensor ids, at::Tensor dy, at::Tensor dw, double scale) {
  emb_check(ids, dw, dy);
  TORCH_CHECK(dw.is_contiguous() && (reinterpret_cast<uintptr_t>(dw.data_ptr()) & 15) == 0,
              "embedding: contiguous gradient on a 16-byte boundary");
  const c10::cuda::CUDAGuard guard(dw.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int64_t T_ = ids.numel();
  const int V = (int)dw.size(0), D = (int)dw.size(1), tiles = (D + kTile - 1) / kTile;
  const int ids64 = ids.scalar_type() == at::kLong;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  int passes = 1;   // digits of 0 .. V
  while (passes < 4 && ((uint64_t)V >> (passes * kRadixBits)) != 0) ++passes;
  const int64_t pieces = (T_ + kPiece - 1) / kPiece;
  TORCH_CHECK(pieces * tiles < (1LL << 31), "embedding: too many tokens");
  const auto i32 = ids.options().dtype(at::kInt);
  at::Tensor sorted, crossing = at::empty({1 + pieces}, i32);
  int32_t *keys, *order, *n_cross = crossing.data_ptr<int32_t>(), *cross = n_cross + 1;
  // the table's first rows, zeroed meanwhile: `bytes` a launch
  const int64_t row_bytes = (int64_t)D * dw.element_size();
  int64_t zeroed = 0;   // rows
  auto share = [&](int64_t bytes) {
    const int64_t rows = std::min<int64_t>(V - zeroed, bytes / row_bytes);
    const ZeroShare z{reinterpret_cast<uint8_t*>(dw.data_ptr()) + zeroed * row_bytes, rows * row_bytes};
    zeroed += rows;
    return z;
  };
  auto share_blocks = [&](const ZeroShare& z) {
    return (unsigned)std::min<int64_t>(2 * sms, (z.bytes + 32 * kZeroChunk - 1) / (32 * kZeroChunk));
  };
  if (T_ <= kSortTile) {
    sorted = at::empty({2 * T_}, i32);
    keys = sorted.data_ptr<int32_t>();
    order = keys + T_;
    constexpr int smem = kSortWarps * kRadix * 2 + kSortTile * 6;
    static bool configured[64] = {false};
    const int dev = dw.get_device();
    if (!configured[dev]) {
      C10_CUDA_CHECK(cudaFuncSetAttribute(embedding_sort_block_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      configured[dev] = true;
    }
    // (8192 tokens in two passes take 19 us)
    const ZeroShare z = share((int64_t)passes * 3500 * (T_ + 4096));
    embedding_sort_block_kernel<<<1 + share_blocks(z), kSortWarps * 32, smem, stream>>>(ids.data_ptr(), ids64, (int)T_, V, passes,
                                                                                        keys, order, n_cross, z);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  } else {
    const int64_t n = (T_ + kSortTile - 1) / kSortTile;
    sorted = at::empty({4 * T_ + kRadix * n}, i32);   // two buffers in turn, the counts
    int32_t* buf[2] = {sorted.data_ptr<int32_t>(), sorted.data_ptr<int32_t>() + 2 * T_};
    uint32_t* counts = reinterpret_cast<uint32_t*>(buf[1] + 2 * T_);
    constexpr int smem = kSortWarps * kRadix * 2;
    // A launch takes a tile's latency, 4 to 10 us to count and 16 to 20 to place, from 8193 tokens to
    // 524288 (22 to place 2^20), so the zeros beside one are as many at any number of tokens.
    for (int pass = 0; pass < passes; ++pass) {
      const ZeroShare z0 = share(24 << 20), z1 = share(72 << 20);
      const unsigned b0 = (unsigned)n + share_blocks(z0), b1 = (unsigned)n + share_blocks(z1);
      int32_t *in = buf[pass & 1], *out = buf[(pass + 1) & 1];
      const int shift = pass * kRadixBits;
      if (pass == 0) {
        embedding_count_kernel<true><<<b0, kSortWarps * 32, 0, stream>>>(ids.data_ptr(), ids64, T_, V, shift, counts, n_cross, (int)n, z0);
        C10_CUDA_KERNEL_LAUNCH_CHECK();
        embedding_place_kernel<true><<<b1, kSortWarps * 32, smem, stream>>>(ids.data_ptr(), ids64, nullptr, T_, V, shift, (int)n,
                                                                             counts, out, out + T_, z1);
      } else {
        embedding_count_kernel<false><<<b0, kSortWarps * 32, 0, stream>>>(in, 0, T_, V, shift, counts, nullptr, (int)n, z0);
        C10_CUDA_KERNEL_LAUNCH_CHECK();
        embedding_place_kernel<false><<<b1, kSortWarps * 32, smem, stream>>>(in, 0, in + T_, T_, V, shift, (int)n, counts, out,
                                                                              out + T_, z1);
      }
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
    keys = buf[passes & 1];
    order = keys + T_;
  }
  at::Tensor part = at::empty({pieces * 2 * D}, ids.options().dtype(at::kFloat));
  float* pp = part.data_ptr<float>();
  const int64_t sums = (pieces * tiles + kEmbWarps - 1) / kEmbWarps, zeros = (V - zeroed + 32 * kEmbWarps - 1) / (32 * kEmbWarps);
  ZQ_EMB_TYPES(dw.scalar_type(), {
    const T* dyp = reinterpret_cast<const T*>(dy.data_ptr());
    T* dwp = reinterpret_cast<T*>(dw.data_ptr());
    auto go = [&](auto sum, auto join) {
      sum<<<(unsigned)(sums + zeros), kEmbWarps * 32, 0, stream>>>(keys, order, T_, dyp, dy.stride(0), dwp, pp, n_cross, cross,
                                                                   (int)sums, zeroed, tiles, V, D, (float)scale);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      if (pieces > 1) {
        const unsigned grid = (unsigned)std::min<int64_t>(pieces * tiles, 16 * sms);
        join<<<grid, kEmbWarps * 32, 0, stream>>>(keys, T_, pp, dwp, n_cross, cross, tiles, D, (float)scale);
      }
    };
    if (D % 8 == 0 && emb_aligned(dy)) go(embedding_sum_kernel<T, true>, embedding_join_kernel<T, true>);
    else go(embedding_sum_kernel<T, false>, embedding_join_kernel<T, false>);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
