// Distillation from a teacher's top logits, mixed with the hard targets: loss
// rows, their mean, and the gradient of the mean, over (vocab-padded) logits.
//
// Row m with student logits z[0..V), teacher entries (id_k, t_k), k < K, and
// target y, temperature τ:
//   p = softmax over the row's entries of t / τ        (ids < 0 or >= V: no entry)
//   q = softmax(z / τ), r = softmax(z)                 (over the whole vocabulary)
//   loss = α τ² Σ_k p_k (log p_k - log q[id_k]) + (1 - α) (-log r[y])
//   dloss/dz_j = α τ (q_j - Σ_{k: id_k = j} p_k) + (1 - α) (r_j - [j = y])
// A row whose target is outside [0, V) (ignore_index among them) counts nothing;
// a row without entries has no first term.  The mean is over the n counted rows.
//
// A block (a cluster of blocks, each with a slice of the columns, where a row does not
// fit into one block's shared memory or there are fewer rows than SMs) works on one
// row at a time, with three kinds of warps:
//   one loads: bulk copies of the row into a ring of chunks, running ahead into the
//     next rows as far as chunks are free;
//   NT / 32 compute: pass 1 over the chunks takes the running maximum and the sums of
//     exponentials, pass 2 over the same chunks, still in shared memory, writes the
//     gradient and frees them.  The logits are read from memory once and the gradient
//     is written once, and loads go on while a row is being worked on;
//   one follows the teacher: its distribution during pass 1, the loss during pass 2,
//     and after it the K + 1 columns whose gradient has a p or one-hot term (written a
//     second time, each with its terms summed in 32 bits and rounded once; entries
//     with the same id add up in entry order, so there are no atomics on values).
// The mean's n is counted by every block from the targets beforehand.
//
// What bounds it: memory, next to the special-function unit's 16 exponentials a cycle
// and SM: two a logit at τ = 1 (0.57 ms of 8192 x 152064 against 0.76 ms of memory).  At
// τ = 2 and 4 the hard softmax's exponential is the soft one's square or fourth power;
// other τ take four a logit.  Measured with a fifth of the rows not counted, which are not
// read (so 0.9 of the bytes of all logits and gradients move): 8192 x 152064 bf16 870 us,
// 5.2 TB/s, 0.79 of a copy; 4096 x 50257 at τ = 2 178 us, 4.2 TB/s, 0.64 (a row's joins,
// about 4000 cycles next to 8000 of its passes, are what is left), at τ = 1.5 250 us.  One
// block a row that read it twice, the second time from L2, took 1130 and 350 us.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>

#include "common.cuh"

// defined in gemm_sm100.cu
zq::DeviceStatus* status_buffer(int device);

namespace zq {

constexpr int kDistMaxK = 1024;
constexpr int kDistMaxCluster = 8;
constexpr int kDistSeen = 8192;          // bits of the map of entries' ids
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
enum DistErr { kErrDistLoad = 331, kErrDistChunk = 332, kErrDistPeer = 333 };

struct DistillParams {
  const void* logits;
  const void* ids;          // int32 or int64 [M, K]
  const void* teacher;      // fp32, bf16 or fp16 [M, K]
  const int64_t* targets;   // [M] or null
  float* rows;              // [M] loss rows (written unless grad_only)
  float* sums;              // [M, 3]: maximum and the two sums of a row; written, or read by grad_only
  const float* g;           // grad_only: gradient of each loss row, or one of their mean
  void* grad;               // [M, width]; null: forward alone
  int64_t M, stride, grad_stride, width, vocab;
  int K, ids64, teacher_type;
  float soft_scale;         // log2(e) / τ; with one softmax, its scale
  float alpha, tau;
  bool grad_only, g_mean, two;   // two: two softmaxes
  DeviceStatus* status;
};

__device__ __forceinline__ float dist_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's reference m (its maximum or somewhat less, in the logits' own units) and the sums of
// 2^(x·s + shift(m, s)) at the softmaxes' scales s.  The shift is the ROUNDED product
// -m·s, everywhere the same one: x·s + shift is then one exact product and one
// rounding of a small number, and no error of the size of m·s enters.  It is rounded down:
// where m is a mask's value so far (-1e9, the type's lowest) what the rounding leaves may
// be any power of two, but none above 1, and sums of 0 go when the maximum moves up.
struct RowSums {
  float m, soft, hard;
};

// (a maximum of -inf shifts by nothing: sums of 0, not NaN.  The product is kept from the
// compiler's own fma, which would round one of two shifts and not the other: a maximum
// that stays would raise its sum by 2^(|m·s| 2^-25))
__device__ __forceinline__ float dist_shift(float m, float s) { return m == -INFINITY ? 0.0f : __fmul_rd(-m, s); }

// factor of a sum when the maximum goes from `from` up to `to`
__device__ __forceinline__ float dist_raise(float from, float to, float s) {
  return from == -INFINITY ? 0.0f : dist_exp2(dist_shift(to, s) - dist_shift(from, s));
}

// The softmaxes of a kernel.  MODE 1: one, at the scale ss (`soft` holds its sum: τ = 1,
// α = 1 or α = 0).  MODE 2, 4: τ = MODE, the hard exponential is the soft one's power
// (scale and shift of the hard one are MODE times the soft one's).  MODE 0: two.
template <int MODE>
__device__ __forceinline__ float dist_power(float e) {
  return MODE == 2 ? e * e : (e * e) * (e * e);
}

// A thread's sums while it goes over its columns: two partial sums each, so that the
// arithmetic is in packed pairs.
struct LaneSums {
  float m;
  uint64_t soft, hard;
};

template <int MODE>
__device__ __forceinline__ void lane_raise(LaneSums& a, float to, float ss) {
  const float f = dist_raise(a.m, to, ss);
  a.soft = f2_mul(a.soft, f2_pack(f, f));
  float fh = 1.0f;
  if constexpr (MODE == 0) fh = dist_raise(a.m, to, kLog2e);
  if constexpr (MODE >= 2) fh = dist_power<MODE>(f);
  if constexpr (MODE != 1) a.hard = f2_mul(a.hard, f2_pack(fh, fh));
  a.m = to;
}

__device__ __forceinline__ uint64_t f2_exp2(uint64_t x) {
  float lo, hi;
  f2_unpack(x, lo, hi);
  return f2_pack(dist_exp2(lo), dist_exp2(hi));
}

// The maximum of a thread moves only when it is left behind by this many powers of two
// of the faster softmax: exponentials stay below 2^12 (their sums are relative to m and
// exact in any case), and the rescaling, which one of a warp's 32 threads would nearly
// always want, becomes rare.
constexpr float kDistBehind = 12.0f;

// P pairs of columns with the largest value cm; behind: kDistBehind in logits
template <int MODE, int P>
__device__ __forceinline__ void lane_add(LaneSums& a, const uint64_t (&x)[P], float cm, float ss, float behind) {
  if (cm > a.m + behind) lane_raise<MODE>(a, cm, ss);   // (from -inf: always)
  const float bs = dist_shift(a.m, ss), bh = dist_shift(a.m, kLog2e);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const uint64_t e = f2_exp2(f2_fma(x[i], f2_pack(ss, ss), f2_pack(bs, bs)));
    a.soft = f2_add(a.soft, e);
    if constexpr (MODE == 0) a.hard = f2_add(a.hard, f2_exp2(f2_fma(x[i], f2_pack(kLog2e, kLog2e), f2_pack(bh, bh))));
    if constexpr (MODE == 2) a.hard = f2_fma(e, e, a.hard);
    if constexpr (MODE == 4) {
      const uint64_t e2 = f2_mul(e, e);
      a.hard = f2_fma(e2, e2, a.hard);
    }
  }
}

// maximum over a warp, in every lane
__device__ __forceinline__ float warp_max_f32(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Joins the lanes' partial results; the same one in every lane.
template <int MODE>
__device__ __forceinline__ RowSums warp_join(RowSums a, float ss) {
  const float m = warp_max_f32(a.m);   // (sums over nothing but -inf are 0, or NaN, which stays)
  const float f = dist_raise(a.m, m, ss);
  RowSums r{m, warp_sum(a.soft * f), 0.0f};
  if constexpr (MODE == 0) r.hard = warp_sum(a.hard * dist_raise(a.m, m, kLog2e));
  if constexpr (MODE >= 2) r.hard = warp_sum(a.hard * dist_power<MODE>(f));
  return r;
}

// Gradient entries without their p and one-hot terms; the softmaxes' denominators are in
// the factors fs and fh.
template <int MODE>
__device__ __forceinline__ uint64_t dist_smooth(uint64_t v, float ss, float shift_s, float shift_h, float fs, float fh) {
  const uint64_t e = f2_exp2(f2_fma(v, f2_pack(ss, ss), f2_pack(shift_s, shift_s)));
  const uint64_t f = f2_pack(fs, fs), g = f2_pack(fh, fh);
  if constexpr (MODE == 0)
    return f2_fma(g, f2_exp2(f2_fma(v, f2_pack(kLog2e, kLog2e), f2_pack(shift_h, shift_h))), f2_mul(f, e));
  if constexpr (MODE == 2) return f2_mul(e, f2_fma(g, e, f));
  if constexpr (MODE == 4) return f2_mul(e, f2_fma(g, f2_mul(f2_mul(e, e), e), f));
  return f2_mul(f, e);
}
template <int MODE>
__device__ __forceinline__ float dist_smooth1(float v, float ss, float shift_s, float shift_h, float fs, float fh) {
  float lo, hi;
  f2_unpack(dist_smooth<MODE>(f2_pack(v, v), ss, shift_s, shift_h, fs, fh), lo, hi);
  return lo;
}

// mbar_wait whose looks hint at a long sleep: the other block of the SM has work to
// issue meanwhile
__device__ __forceinline__ bool dist_wait_long(uint64_t* bar, uint32_t parity, DeviceStatus* st) {
  unsigned long long t0 = 0;
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n"
        "  .reg .pred p;\n"
        "  mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "  selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(2000u)
        : "memory");
    if (ok != 0) return true;
    if (t0 == 0) {
      t0 = globaltimer();
    } else if (globaltimer() - t0 > kWaitTimeoutNs) {
      record_error(st, kErrDistPeer, (int)parity);
      return false;
    }
  }
}

// 16 bytes into the shared memory of block `rank` of the cluster, which complete that
// many bytes of its barrier.  (An arrival with a release at cluster scope would wait
// for the gradient stores of the row before.)
__device__ __forceinline__ void dist_send(float* to, uint64_t* bar, int rank, float x, float y, float z) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
          map_to_cta(smem_u32(to), (uint32_t)rank)),
      "r"(__float_as_uint(x)), "r"(__float_as_uint(y)), "r"(__float_as_uint(z)), "r"(0u),
      "r"(map_to_cta(smem_u32(bar), (uint32_t)rank))
      : "memory");
}

// 16 bytes of a row
template <typename T>
struct DistVec {
  static constexpr int N = 16 / (int)sizeof(T), P = N / 2;
  uint4 u;
  __device__ __forceinline__ void pairs(uint64_t* x) const {
    if constexpr (sizeof(T) == 4) {
      x[0] = f2_pack(__uint_as_float(u.x), __uint_as_float(u.y));
      x[1] = f2_pack(__uint_as_float(u.z), __uint_as_float(u.w));
    } else {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 f;
        if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else f = bf16x2_to_f2(w[i]);
        x[i] = f2_pack(f.x, f.y);
      }
    }
  }
  __device__ __forceinline__ float largest() const {
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2 a = __hmax2(*reinterpret_cast<const T2*>(&u.x), *reinterpret_cast<const T2*>(&u.y));
      const T2 b = __hmax2(*reinterpret_cast<const T2*>(&u.z), *reinterpret_cast<const T2*>(&u.w));
      const T2 c = __hmax2(a, b);
      return fmaxf(to_f32<T>(c.x), to_f32<T>(c.y));
    }
  }
  __device__ __forceinline__ void set(int i, uint64_t pair) {   // columns 2i, 2i + 1
    float lo, hi;
    f2_unpack(pair, lo, hi);
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(lo);
      w[2 * i + 1] = __float_as_uint(hi);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(lo, hi);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      w[i] = pack_bf16x2(lo, hi);
    }
  }
};

__device__ __forceinline__ float dist_teacher(const DistillParams& p, int64_t i) {
  if (p.teacher_type == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.teacher)[i]);
  if (p.teacher_type == 2) return __half2float(reinterpret_cast<const __half*>(p.teacher)[i]);
  return reinterpret_cast<const float*>(p.teacher)[i];
}

// The shapes of a block: NT compute threads, chunks of V vectors a thread, SLOTS chunks,
// BLOCKS of them on an SM.  Several to an SM, so that one row's reductions and exchanges
// overlap with another's passes; short rows take the smaller ones.
template <int NT, int V, int SLOTS, int BLOCKS>
struct DistShape {
  static constexpr int kNT = NT, kV = V, kBlocks = BLOCKS;
  static constexpr int kThreads = NT + 64, kWarps = NT / 32;
  static constexpr int kVecs = V * NT, kBytes = kVecs * 16;
  static constexpr uint32_t kSlots = SLOTS;
  static constexpr int64_t kRing = (int64_t)SLOTS * kBytes;
};
using DistSmall = DistShape<128, 2, 8, 5>;      //  32 KB
using DistWide = DistShape<256, 4, 4, 3>;       //  64 KB
using DistWidest = DistShape<512, 4, 6, 1>;     // 192 KB

template <typename T, typename S, int MODE>
__global__ void __launch_bounds__(S::kThreads, S::kBlocks) distill_kernel(const __grid_constant__ DistillParams p) {
  constexpr int NT = S::kNT, N = DistVec<T>::N, P = DistVec<T>::P;
  extern __shared__ __align__(128) uint8_t dist_smem[];
  uint8_t* ring = dist_smem;
  // the teacher's entries of two rows, and the target as the last of each: log2 of the
  // probability, the column (or -1) and its logit
  float* s_p2 = reinterpret_cast<float*>(ring + S::kRing);
  int* s_id2 = reinterpret_cast<int*>(s_p2 + 2 * (p.K + 1));
  float* s_z2 = reinterpret_cast<float*>(s_id2 + 2 * (p.K + 1));
  __shared__ uint64_t full[S::kSlots], empty[S::kSlots], joined[2];
  // of all the cluster's compute warps; behind them a token of each teacher warp
  __shared__ __align__(16) float s_part[2][kDistMaxCluster * (S::kWarps + 1)][4];
  __shared__ float s_some[2];
  __shared__ uint32_t s_seen[kDistSeen / 32], s_twice[kDistSeen / 32];
  __shared__ int s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t csize_u;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize_u));
  const int csize = (int)csize_u, clog = 31 - __clz(csize);   // 1, 2, 4 or 8
  const int crank = csize > 1 ? (int)cluster_ctarank() : 0;
  const int64_t row0 = blockIdx.x / csize_u, row_step = gridDim.x / csize_u;
  const float ss = p.soft_scale;

  if (tid == 0) {
    for (uint32_t i = 0; i < S::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], S::kWarps);
    }
    // the compute and teacher warps of the whole cluster: none of them is more than a row
    // ahead of another, so a row's parts are read before the next but one overwrites them
    // (in a cluster by the bytes that they send)
    mbar_init(&joined[0], csize > 1 ? 1u : (uint32_t)(S::kWarps + 1));
    mbar_init(&joined[1], csize > 1 ? 1u : (uint32_t)(S::kWarps + 1));
    fence_mbar_init();
    s_count = 0;
  }
  for (int i = tid; i < kDistSeen / 32; i += S::kThreads) s_seen[i] = s_twice[i] = 0u;
  __syncthreads();
  float inv_n = 1.0f;
  if (p.grad != nullptr && (!p.grad_only || p.g_mean)) {   // rows counted, for the mean's gradient
    if (p.targets != nullptr) {
      int c = 0;
      for (int64_t i = tid; i < p.M; i += S::kThreads) {
        const int64_t y = p.targets[i];
        c += (y >= 0 && y < p.vocab) ? 1 : 0;
      }
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) atomicAdd(&s_count, c);
      __syncthreads();
    }
    inv_n = 1.0f / fmaxf(p.targets != nullptr ? (float)s_count : (float)p.M, 1.0f);
    if (p.g_mean) inv_n *= p.g[0];
  }
  if (csize > 1) cluster_sync_all();   // the peers' barriers are set up

  // a row's columns: `head` up to the first 16-byte boundary, whole vectors, then a tail
  // (this block's vectors [v0, v1) go through the ring, the edges are rank 0's)
  struct Cut {
    int64_t head, tail, v0, v1;
  };
  auto cut = [&](const T* z) {
    Cut c;
    const int mis = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
    c.head = min((int64_t)(mis == 0 ? 0 : N - mis), p.vocab);
    const int64_t nvec = (p.vocab - c.head) / N, per = (nvec + csize - 1) >> clog;
    c.tail = c.head + nvec * N;
    c.v0 = min(nvec, per * crank);
    c.v1 = min(nvec, c.v0 + per);
    return c;
  };
  auto target = [&](int64_t row) { return p.targets != nullptr && row < p.M ? p.targets[row] : (int64_t)-1; };
  auto counts = [&](int64_t y) { return p.targets == nullptr || (y >= 0 && y < p.vocab); };
  auto logits_row = [&](int64_t row) { return reinterpret_cast<const T*>(p.logits) + row * p.stride; };
  // a wait that ran out once makes the others return at once: results are lost, nothing hangs
  bool dead = false;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (!dead && !mbar_wait(bar, parity, p.status, code)) dead = true;
  };

  // the end of pass 1: every warp's sums, the teacher's distribution
  auto wait_joined = [&](uint32_t turn) {
    if (!dead && !dist_wait_long(&joined[turn & 1u], (turn >> 1) & 1u, p.status)) dead = true;
    __syncwarp();
  };
  struct Factors {
    RowSums a;
    float shift_s, shift_h, cs, ch, fs, fh;
  };
  auto joined_row = [&](int64_t row, uint32_t turn) {
    const int par = (int)(turn & 1u);
    Factors f;
    float g = p.grad == nullptr ? 0.0f : p.grad_only && !p.g_mean ? p.g[row] : inv_n;
    wait_joined(turn);
    if (!p.grad_only) {   // joined in the same order by every warp
      RowSums a{-INFINITY, 0.0f, 0.0f};
      const int parts = csize * S::kWarps;
      for (int i = lane; i < parts; i += 32) a.m = fmaxf(a.m, s_part[par][i][0]);
      for (int i = lane; i < parts; i += 32) {
        const float* b = s_part[par][i];
        const float r = dist_raise(b[0], a.m, ss);
        a.soft += b[1] * r;
        if constexpr (MODE == 0) a.hard += b[2] * dist_raise(b[0], a.m, kLog2e);
        if constexpr (MODE >= 2) a.hard += b[2] * dist_power<MODE>(r);
      }
      f.a = warp_join<MODE>(a, ss);
    } else {
      f.a = RowSums{p.sums[3 * row], p.sums[3 * row + 1], p.sums[3 * row + 2]};
    }
    f.shift_s = dist_shift(f.a.m, ss);
    f.shift_h = dist_shift(f.a.m, kLog2e);
    // a row without entries has no soft term; one softmax stands for both terms
    f.cs = p.alpha * p.tau * s_some[par] * g;
    f.ch = (1.0f - p.alpha) * g;
    f.fs = (MODE == 1 ? f.cs + f.ch : f.cs) / f.a.soft;
    f.fh = MODE == 1 ? 0.0f : f.ch / f.a.hard;
    return f;
  };

  int64_t y_next = target(row0);
  if (warp == S::kWarps) {
    // ------------------------------------------------------------ loader (one thread)
    if (lane == 0) {
      uint32_t n = 0;   // chunks so far
      for (int64_t row = row0; row < p.M; row += row_step) {
        const int64_t y = y_next;
        y_next = target(row + row_step);
        if (!counts(y)) continue;
        const T* z = logits_row(row);
        const Cut c = cut(z);
        for (int64_t v = c.v0; v < c.v1; v += S::kVecs, ++n) {
          const int slot = (int)(n % S::kSlots);
          wait(&empty[slot], ((n / S::kSlots) & 1u) ^ 1u, kErrDistLoad);
          if (dead) break;
          const uint32_t bytes = (uint32_t)min((int64_t)S::kVecs, c.v1 - v) * 16u;
          mbar_arrive_expect_tx(&full[slot], bytes);
          bulk_load(ring + slot * S::kBytes, reinterpret_cast<const uint8_t*>(z + c.head) + v * 16, bytes, &full[slot]);
        }
        if (dead) break;
      }
      // copies in flight land before the block can go (where nothing ran out, all have been waited for)
      if (dead)
        for (uint32_t i = n > S::kSlots ? n - S::kSlots : 0; i < n; ++i)
          mbar_wait(&full[i % S::kSlots], (i / S::kSlots) & 1u, nullptr, 0);
    }
  } else if (warp < S::kWarps) {
    // ------------------------------------------------------------ compute
    uint32_t slot = 0, phase = 0;                 // of the row's first chunk
    uint32_t turn = 0;                            // counted rows so far
    const float behind = kDistBehind / fmaxf(ss, kLog2e);
    for (int64_t row = row0; row < p.M; row += row_step) {
      const T* z = logits_row(row);
      const int64_t y = y_next;
      y_next = target(row + row_step);
      const Cut c = cut(z);
      T* dz = p.grad != nullptr ? reinterpret_cast<T*>(p.grad) + row * p.grad_stride : nullptr;
      uint4* dv = reinterpret_cast<uint4*>(dz + c.head);   // (rows of logits and gradient are aligned alike)

      if (!counts(y)) {   // a gradient of zeros
        if (dz != nullptr) {
          for (int64_t i = c.v0 + tid; i < c.v1; i += NT) __stcs(dv + i, make_uint4(0, 0, 0, 0));
          if (crank == 0) {
            for (int64_t i = tid; i < c.head; i += NT) dz[i] = from_f32<T>(0.0f);
            for (int64_t i = c.tail + tid; i < p.width; i += NT) dz[i] = from_f32<T>(0.0f);
          }
        }
        continue;   // (the same in every warp of the cluster)
      }
      const int par = (int)(turn & 1u);
      const int vecs = (int)(c.v1 - c.v0);
      RowSums a{-INFINITY, 0.0f, 0.0f};
      float edge = 0.0f;       // this thread's column of the row's edges, loaded ahead of its use
      int64_t edge_col = -1;
      if (crank == 0 && tid < 2 * N) {
        if (tid < c.head) edge_col = tid;
        else if (c.tail + (tid - c.head) < p.vocab) edge_col = c.tail + (tid - c.head);
        if (edge_col >= 0) edge = to_f32<T>(z[edge_col]);
      }
      if (!p.grad_only) {
        LaneSums ls{-INFINITY, 0ull, 0ull};
        uint32_t sl = slot, ph = phase;
        for (int left = vecs; left > 0; left -= S::kVecs) {
          wait(&full[sl], ph, kErrDistChunk);
          const uint4* src = reinterpret_cast<const uint4*>(ring + sl * S::kBytes) + tid;
          DistVec<T> w[S::kV];
          if (left >= S::kVecs) {
            uint64_t x[S::kV * P];
#pragma unroll
            for (int u = 0; u < S::kV; ++u) w[u].u = src[u * NT];
            float cm = w[0].largest();
#pragma unroll
            for (int u = 1; u < S::kV; ++u) cm = fmaxf(cm, w[u].largest());
#pragma unroll
            for (int u = 0; u < S::kV; ++u) w[u].pairs(x + u * P);
            lane_add<MODE, S::kV * P>(ls, x, cm, ss, behind);
          } else {
            for (int j = tid; j < left; j += NT) {
              w[0].u = src[j - tid];
              uint64_t y2[P];
              w[0].pairs(y2);
              lane_add<MODE, P>(ls, y2, w[0].largest(), ss, behind);
            }
          }
          if (dz == nullptr) {   // forward alone: the chunk is done with
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[sl]);
          }
          if (++sl == S::kSlots) { sl = 0; ph ^= 1u; }
        }
        float s0, s1, h0, h1;
        f2_unpack(ls.soft, s0, s1);
        f2_unpack(ls.hard, h0, h1);
        a = RowSums{ls.m, s0 + s1, h0 + h1};
        if (edge_col >= 0) {
          const float m = fmaxf(a.m, edge), f = dist_raise(a.m, m, ss);
          const float e = dist_exp2(fmaf(edge, ss, dist_shift(m, ss)));
          a.soft = a.soft * f + e;
          if constexpr (MODE == 0)
            a.hard = a.hard * dist_raise(a.m, m, kLog2e) + dist_exp2(fmaf(edge, kLog2e, dist_shift(m, kLog2e)));
          if constexpr (MODE >= 2) a.hard = a.hard * dist_power<MODE>(f) + dist_power<MODE>(e);
          a.m = m;
        }
        __syncwarp();
        a = warp_join<MODE>(a, ss);
      }
      // this warp's sums to every block of the cluster
      if (csize == 1) {
        if (lane == 0) {
          float* to = s_part[par][warp];
          to[0] = a.m;
          to[1] = a.soft;
          to[2] = a.hard;
          mbar_arrive(&joined[par]);
        }
      } else if (lane < csize) {
        dist_send(s_part[par][crank * S::kWarps + warp], &joined[par], lane, a.m, a.soft, a.hard);
      }
      __syncwarp();
      if (dz != nullptr) {
        const Factors f = joined_row(row, turn);
        uint4* dst = dv + c.v0 + tid;
        uint32_t sl = slot, ph = phase;
        for (int left = vecs; left > 0; left -= S::kVecs) {
          wait(&full[sl], ph, kErrDistChunk);   // (grad_only: the first look at it)
          const uint4* src = reinterpret_cast<const uint4*>(ring + sl * S::kBytes) + tid;
          auto turn_out = [&](int u, const DistVec<T>& w) {
            DistVec<T> o;
            uint64_t x[P];
            w.pairs(x);
#pragma unroll
            for (int e = 0; e < P; ++e) o.set(e, dist_smooth<MODE>(x[e], ss, f.shift_s, f.shift_h, f.fs, f.fh));
            __stcs(dst + u * NT, o.u);
          };
          if (left >= S::kVecs) {
            DistVec<T> w[S::kV];
#pragma unroll
            for (int u = 0; u < S::kV; ++u) w[u].u = src[u * NT];
#pragma unroll
            for (int u = 0; u < S::kV; ++u) turn_out(u, w[u]);
          } else {
            for (int u = 0; u * NT + tid < left; ++u) turn_out(u, DistVec<T>{src[u * NT]});
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[sl]);
          if (++sl == S::kSlots) { sl = 0; ph ^= 1u; }
          dst += S::kVecs;
        }
        if (edge_col >= 0) dz[edge_col] = from_f32<T>(dist_smooth1<MODE>(edge, ss, f.shift_s, f.shift_h, f.fs, f.fh));
        if (crank == 0)
          for (int64_t i = p.vocab + tid; i < p.width; i += NT) dz[i] = from_f32<T>(0.0f);
        __syncwarp();
        asm volatile("bar.arrive %0, %1;" ::"r"(2 + par), "r"(NT + 32) : "memory");
      } else {   // (nobody runs more than a row ahead)
        wait_joined(turn);
      }
      slot += (uint32_t)((vecs + S::kVecs - 1) / S::kVecs);
      if (slot >= S::kSlots) { slot -= S::kSlots; phase ^= 1u; }
      ++turn;
    }
  } else {
    // ------------------------------------------------------------ the teacher's warp
    // Its loads take long and its work is short, so it is a row ahead with the entries.
    int64_t y = y_next, y_after = 0;
    // the first counted row from `row` on, its target in y; the others count nothing
    auto next_counted = [&](int64_t row) {
      for (; row < p.M; row += row_step) {
        y_after = target(row + row_step);
        if (counts(y)) return row;
        if (lane == 0 && crank == 0 && !p.grad_only)
          p.rows[row] = p.sums[3 * row] = p.sums[3 * row + 1] = p.sums[3 * row + 2] = 0.0f;
        y = y_after;
      }
      return row;
    };
    // a row's entries as columns and log2 p (-inf: no entry, or none of the mass)
    auto entries = [&](int64_t row, uint32_t turn) {
      const int par = (int)(turn & 1u);
      float* s_p = s_p2 + par * (p.K + 1);
      int* s_id = s_id2 + par * (p.K + 1);
      float* s_z = s_z2 + par * (p.K + 1);
      const T* z = logits_row(row);
      float tm = -INFINITY;
      for (int k0 = lane; k0 < p.K; k0 += 128) {   // four of each lane at once
        int64_t v[4];
        float t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t e = row * p.K + k0 + 32 * u;
          const bool in = k0 + 32 * u < p.K;
          v[u] = !in ? -1 : p.ids64 ? reinterpret_cast<const int64_t*>(p.ids)[e] : (int64_t)reinterpret_cast<const int32_t*>(p.ids)[e];
          t[u] = in ? dist_teacher(p, e) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (k0 + 32 * u >= p.K) break;
          const bool in = v[u] >= 0 && v[u] < p.vocab;
          const float x = in ? t[u] : -INFINITY;
          s_z[k0 + 32 * u] = in ? to_f32<T>(z[v[u]]) : 0.0f;
          s_id[k0 + 32 * u] = in ? (int)v[u] : -1;
          s_p[k0 + 32 * u] = x;
          tm = fmaxf(tm, x);
        }
      }
      if (lane == 0) {
        s_id[p.K] = p.targets != nullptr ? (int)y : -1;
        s_p[p.K] = -INFINITY;
        s_z[p.K] = p.targets != nullptr ? to_f32<T>(z[y]) : 0.0f;
      }
      __syncwarp();
      tm = -dist_shift(warp_max(tm), 1.0f);
      // (the largest taken off before the scale: entries near the type's lowest value stay finite)
      const float c = kLog2e / p.tau;
      float mass = 0.0f;
      for (int k = lane; k < p.K; k += 32) mass += dist_exp2((s_p[k] - tm) * c);
      mass = warp_sum(mass);
      const bool some = !(mass == 0.0f);
      const float lm = log2f(mass);
      for (int k = lane; k < p.K; k += 32) s_p[k] = some ? (s_p[k] - tm) * c - lm : -INFINITY;
      if (lane == 0) s_some[par] = some ? 1.0f : 0.0f;
      __syncwarp();
      if (csize == 1) {
        if (lane == 0) mbar_arrive(&joined[par]);
      } else {
        if (lane == 0) mbar_arrive_expect_tx(&joined[par], (uint32_t)(csize * (S::kWarps + 1)) * 16u);
        if (lane < csize) dist_send(s_part[par][csize * S::kWarps + crank], &joined[par], lane, 0.0f, 0.0f, 0.0f);
      }
      __syncwarp();
    };
    uint32_t turn = 0;
    int64_t row = next_counted(row0);
    if (row < p.M) entries(row, 0);
    while (row < p.M) {
      const int64_t y_row = y;
      y = y_after;
      const Factors f = joined_row(row, turn);
      const int64_t next = next_counted(row + row_step);
      if (next < p.M) entries(next, turn + 1);
      const float* s_p = s_p2 + (turn & 1u) * (p.K + 1);
      const int* s_id = s_id2 + (turn & 1u) * (p.K + 1);
      const float* s_z = s_z2 + (turn & 1u) * (p.K + 1);
      const Cut c = cut(logits_row(row));
      if (!p.grad_only && crank == 0) {
        const float log_s = log2f(f.a.soft);
        float kl = 0.0f;
#pragma unroll 4
        for (int k = lane; k < p.K; k += 32) {
          const float lp = s_p[k], pk = dist_exp2(lp);
          if (s_id[k] >= 0 && !(pk == 0.0f)) kl += pk * (lp - (fmaf(s_z[k], ss, f.shift_s) - log_s));
        }
        kl = warp_sum(kl);
        if (lane == 0) {
          float loss = 0.0f;
          if (p.alpha > 0.0f) loss = p.alpha * p.tau * p.tau * kLn2 * kl;
          if (p.alpha < 1.0f) {
            const float zy = s_z[p.K];
            const float at = MODE == 0 ? fmaf(zy, kLog2e, f.shift_h) : (MODE == 1 ? 1.0f : (float)MODE) * fmaf(zy, ss, f.shift_s);
            loss += (1.0f - p.alpha) * kLn2 * (log2f(MODE == 1 ? f.a.soft : f.a.hard) - at);
          }
          p.rows[row] = loss;
          p.sums[3 * row] = f.a.m;
          p.sums[3 * row + 1] = f.a.soft;
          p.sums[3 * row + 2] = f.a.hard;
        }
        __syncwarp();
      }
      if (p.grad != nullptr) {
        T* dz = reinterpret_cast<T*>(p.grad) + row * p.grad_stride;
        // which entries may share their column with another one
        auto bit = [&](int id) { return (uint32_t)id * 2654435761u >> 19; };   // 13 bits
        static_assert(kDistSeen == 1 << 13, "bits of the hash");
        for (int k = lane; k <= p.K; k += 32) {
          const int id = s_id[k];
          if (id < 0) continue;
          const uint32_t h = bit(id), m = 1u << (h & 31u);
          if (atomicOr(&s_seen[h >> 5], m) & m) atomicOr(&s_twice[h >> 5], m);
        }
        __syncwarp();
        // the smooth part of these columns is written (a barrier for even rows and one for odd
        // ones: the compute warps may be a row further already)
        named_barrier(2 + (int)(turn & 1u), NT + 32);
        for (int k = lane; k <= p.K; k += 32) {
          const int id = s_id[k];
          if (id < 0) continue;
          const bool at_edge = id < c.head || id >= c.tail;
          const int64_t vec = at_edge ? 0 : (id - c.head) / N;
          if (at_edge ? crank != 0 : (vec < c.v0 || vec >= c.v1)) continue;   // another block's column
          const uint32_t h = bit(id);
          float pk = dist_exp2(s_p[k]);
          if (s_twice[h >> 5] >> (h & 31u) & 1u) {
            pk = 0.0f;
            for (int j = 0; j < p.K; ++j)
              if (s_id[j] == id) pk += dist_exp2(s_p[j]);
          }
          float d = dist_smooth1<MODE>(s_z[k], ss, f.shift_s, f.shift_h, f.fs, f.fh) - f.cs * pk;
          if (p.targets != nullptr && id == (int)y_row) d -= f.ch;
          dz[id] = from_f32<T>(d);
        }
        __syncwarp();
        for (int k = lane; k <= p.K; k += 32) {   // clear the maps
          const int id = s_id[k];
          if (id >= 0) s_seen[bit(id) >> 5] = s_twice[bit(id) >> 5] = 0u;
        }
        __syncwarp();
      }
      row = next;
      ++turn;
    }
  }
  if (csize > 1) {   // a block's memory stays until no peer can write to it
    __syncwarp();
    cluster_sync_all();
  }
}

// ============================================================================
// After the rows: those whose mask left nothing, and the mean.
//
// Where a row's largest logit is a mask's value (-1e9, the type's lowest), so that m·s is
// beyond 2^26, the rounded shift is off by more than the sums' range allows for.  Such a
// row, which the kernel above leaves unusable, is formed again here from (x - m)·s, a row
// at a time by the whole block.  The mean (`loss`, one block) is the sum of the rows over
// the number of counted ones, in 64 bits and a fixed order.
// ============================================================================
constexpr int kDistFinish = 1024;

__device__ __forceinline__ float dist_block(float v, bool max, float* part) {   // over the block, in every thread
  v = max ? warp_max(v) : warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[threadIdx.x & 31];
  return max ? warp_max(v) : warp_sum(v);
}

template <typename T>
__global__ void __launch_bounds__(kDistFinish) distill_finish_kernel(const __grid_constant__ DistillParams p,
                                                                     float* __restrict__ loss) {
  __shared__ double s_sum[32];
  __shared__ int s_n[32], s_row;
  __shared__ float s_part[32], s_p[kDistMaxK + 1], s_z[kDistMaxK + 1];
  __shared__ int s_id[kDistMaxK + 1];
  const int tid = threadIdx.x, warp = tid >> 5;
  const float ss = p.soft_scale, fast = fmaxf(ss, kLog2e);
  auto far = [&](int64_t row) {   // (rows that count nothing have m = 0)
    const float m = p.sums[3 * row];
    return (m != -INFINITY) & (fabsf(m) * fast > 67108864.0f);
  };
  auto counted = [&](int64_t row) {
    const int64_t y = p.targets != nullptr ? p.targets[row] : 0;
    return ((y >= 0) & (y < p.vocab)) ? 1 : 0;
  };
  double s = 0.0;
  int n = 0;
  bool some_far = false;
  if (loss != nullptr) {
#pragma unroll 4
    for (int64_t i = tid; i < p.M; i += kDistFinish) {   // (nothing here waits for a load before the next one)
      s += p.rows[i];
      n += counted(i);
      some_far |= far(i);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if ((tid & 31) == 0) s_n[warp] = n;
  } else {
#pragma unroll 1
    for (int64_t i = blockIdx.x + (int64_t)tid * gridDim.x; i < p.M; i += (int64_t)gridDim.x * kDistFinish) some_far |= far(i);
  }
  if (__syncthreads_or(some_far)) {
    if (loss == nullptr) {   // (wanted by the gradient of a mean alone)
#pragma unroll 1
      for (int64_t i = tid; p.g_mean && i < p.M; i += kDistFinish) n += counted(i);
      n = __reduce_add_sync(0xffffffffu, n);
      if ((tid & 31) == 0) s_n[warp] = n;
      __syncthreads();
    }
    n = 0;
    for (int w = 0; w < 32; ++w) n += s_n[w];
    const float inv_n = 1.0f / fmaxf((float)n, 1.0f);
    auto redo = [&](int64_t row) {
      const T* z = reinterpret_cast<const T*>(p.logits) + row * p.stride;
      const float m = p.sums[3 * row];
      auto near = [&](int64_t j) { return to_f32<T>(z[j]) - m; };
      float soft = 0.0f, hard = 0.0f;
      for (int64_t j = tid; j < p.vocab; j += kDistFinish) {
        const float x = near(j);
        soft += dist_exp2(x * ss);
        hard += p.two ? dist_exp2(x * kLog2e) : 0.0f;
      }
      soft = dist_block(soft, false, s_part);
      hard = p.two ? dist_block(hard, false, s_part) : soft;
      // the entries as columns, log2 p and logits; the target behind them
      const int y = p.targets != nullptr ? (int)p.targets[row] : -1;
      float tm = -INFINITY;
      for (int k = tid; k <= p.K; k += kDistFinish) {
        const int64_t e = row * p.K + k;
        int64_t id = y;
        float t = -INFINITY;
        if (k < p.K) {
          id = p.ids64 ? reinterpret_cast<const int64_t*>(p.ids)[e] : (int64_t)reinterpret_cast<const int32_t*>(p.ids)[e];
          if (id < 0 || id >= p.vocab) id = -1;
          if (id >= 0) t = dist_teacher(p, e);
        }
        s_id[k] = (int)id;
        s_p[k] = t;
        s_z[k] = id >= 0 ? near(id) : 0.0f;
        tm = fmaxf(tm, t);
      }
      tm = -dist_shift(dist_block(tm, true, s_part), 1.0f);
      const float c = kLog2e / p.tau;
      float mass = 0.0f;
      for (int k = tid; k < p.K; k += kDistFinish) mass += dist_exp2((s_p[k] - tm) * c);
      mass = dist_block(mass, false, s_part);
      const bool some = !(mass == 0.0f);
      const float lm = log2f(mass), log_s = log2f(soft);
      float kl = 0.0f;
      for (int k = tid; k < p.K; k += kDistFinish) {
        const float lp = some ? (s_p[k] - tm) * c - lm : -INFINITY, pk = dist_exp2(lp);
        s_p[k] = lp;
        if (s_id[k] >= 0 && !(pk == 0.0f)) kl += pk * (lp - (s_z[k] * ss - log_s));
      }
      kl = dist_block(kl, false, s_part);
      if (tid == 0 && !p.grad_only) {
        float v = 0.0f;
        if (p.alpha > 0.0f) v = p.alpha * p.tau * p.tau * kLn2 * kl;
        if (p.alpha < 1.0f) v += (1.0f - p.alpha) * kLn2 * (log2f(hard) - s_z[p.K] * (p.two ? kLog2e : ss));
        p.rows[row] = v;
      }
      if (p.grad != nullptr) {
        const float g = !p.grad_only ? inv_n : p.g_mean ? p.g[0] * inv_n : p.g[row];
        const float cs = p.alpha * p.tau * (some ? 1.0f : 0.0f) * g, ch = (1.0f - p.alpha) * g;
        const float fs = (p.two ? cs : cs + ch) / soft, fh = p.two ? ch / hard : 0.0f;
        auto smooth = [&](float x) { return fs * dist_exp2(x * ss) + (p.two ? fh * dist_exp2(x * kLog2e) : 0.0f); };
        T* dz = reinterpret_cast<T*>(p.grad) + row * p.grad_stride;
        for (int64_t j = tid; j < p.vocab; j += kDistFinish) dz[j] = from_f32<T>(smooth(near(j)));
        __syncthreads();
        for (int k = tid; k <= p.K; k += kDistFinish) {
          const int id = s_id[k];
          if (id < 0) continue;
          float pk = 0.0f;
          for (int j = 0; j < p.K; ++j)
            if (s_id[j] == id) pk += dist_exp2(s_p[j]);
          dz[id] = from_f32<T>(smooth(s_z[k]) - cs * pk - (id == y ? ch : 0.0f));
        }
      }
      __syncthreads();
    };
    for (int64_t base = blockIdx.x; base < p.M; base += (int64_t)gridDim.x * kDistFinish) {
      const int64_t row = base + (int64_t)tid * gridDim.x;
      bool left = row < p.M && far(row);
      for (;;) {   // the block's far rows, lowest first
        if (tid == 0) s_row = kDistFinish;
        __syncthreads();
        if (left) atomicMin(&s_row, tid);
        __syncthreads();
        const int t = s_row;
        __syncthreads();
        if (t == kDistFinish) break;
        redo(base + (int64_t)t * gridDim.x);
        left = left && t != tid;
      }
    }
    if (loss != nullptr) {
      s = 0.0;
      for (int64_t i = tid; i < p.M; i += kDistFinish) s += p.rows[i];
    }
  }
  if (loss == nullptr) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((tid & 31) == 0) s_sum[warp] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.0;
    n = 0;
    for (int w = 0; w < 32; ++w) {
      s += s_sum[w];
      n += s_n[w];
    }
    loss[0] = (float)(s / (double)max(n, 1));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) scale_by_scalar_kernel(T* __restrict__ x, const float* __restrict__ g, int64_t n) {
  const float f = g[0];
  if (f == 1.0f) return;
  constexpr int N = DistVec<T>::N;
  const int64_t nv = n / N;
  const int64_t step = (int64_t)gridDim.x * blockDim.x, first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t i = first; i < nv; i += step) {
    const DistVec<T> w{reinterpret_cast<const uint4*>(x)[i]};
    DistVec<T> o;
    uint64_t v[N / 2];
    w.pairs(v);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) o.set(j, f2_mul(v[j], f2_pack(f, f)));
    reinterpret_cast<uint4*>(x)[i] = o.u;
  }
  for (int64_t i = nv * N + first; i < n; i += step) x[i] = from_f32<T>(to_f32<T>(x[i]) * f);
}

template <typename T, typename S, int MODE>
static void launch_distill(const DistillParams& p, int csize, cudaStream_t stream) {
  auto kern = distill_kernel<T, S, MODE>;
  int dev;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  static bool configured[64] = {false};
  // clusters at once, by the power of two that holds K + 1 entries
  static int resident[64][kDistMaxCluster + 1][12] = {{{0}}};
  int kpow = 0;
  while ((1 << kpow) < p.K + 1) ++kpow;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(S::kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)csize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const size_t smem = (size_t)S::kRing + 24 * std::min((size_t)1 << kpow, (size_t)kDistMaxK + 1);
  const size_t most = (size_t)S::kRing + 24 * (kDistMaxK + 1);
  if (!configured[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    configured[dev] = true;
  }
  if (resident[dev][csize][kpow] == 0) {   // a cluster that waits for a place would do its rows after all others
    cfg.gridDim = dim3((unsigned)csize);
    cfg.dynamicSmemBytes = smem;
    int n = 0;
    C10_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    TORCH_CHECK(n > 0, "distill: a cluster of ", csize, " blocks does not fit the device");
    resident[dev][csize][kpow] = n;
  }
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(p.M, resident[dev][csize][kpow]) * csize));
  cfg.dynamicSmemBytes = smem;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
}

template <typename T, typename S>
static void launch_distill_mode(DistillParams& p, int csize, cudaStream_t stream) {
  const bool both = p.alpha > 0.0f && p.alpha < 1.0f && p.tau != 1.0f;
  p.two = both;
  if (!both) {
    if (p.alpha == 0.0f) p.soft_scale = kLog2e;   // the hard softmax alone
    launch_distill<T, S, 1>(p, csize, stream);
  } else if (p.tau == 2.0f) {
    launch_distill<T, S, 2>(p, csize, stream);
  } else if (p.tau == 4.0f) {
    launch_distill<T, S, 4>(p, csize, stream);
  } else {
    launch_distill<T, S, 0>(p, csize, stream);
  }
}

template <typename T>
static void launch_distill_shape(DistillParams& p, cudaStream_t stream) {
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int64_t row = p.vocab * (int64_t)sizeof(T);
  auto slice = [&](int c) { return (row + c - 1) / c + 16; };
  // A row's slices have to fit into the rings.  Three blocks to an SM where that takes at
  // most two slices (50257 columns of bf16: 187 us against 197 with one block to an SM,
  // 4096 rows at τ = 2; 16384 x 32003: 546 against 1094), otherwise one (152064 columns,
  // 8192 rows: 877 us with two slices against 1238 with eight smaller ones; a cluster of
  // eight leaves SMs without a place for it).
  int csize = slice(1) <= DistWide::kRing ? 1 : 2;
  if (slice(2) > DistWide::kRing) {
    csize = 1;
    while (csize < kDistMaxCluster && slice(csize) > DistWidest::kRing) csize *= 2;
  }
  TORCH_CHECK(slice(csize) <= DistWidest::kRing, "distill: a row of logits may have up to ",
              kDistMaxCluster * (DistWidest::kRing - 16), " bytes, got ", row);
  // more slices where the rows leave SMs idle, down to 8 KB of logits a block
  while (csize < kDistMaxCluster && p.M * csize * 2 <= sms && slice(2 * csize) >= 8192) csize *= 2;
  const int64_t mine = slice(csize);
  if (2 * mine <= DistSmall::kRing) launch_distill_mode<T, DistSmall>(p, csize, stream);
  else if (mine <= DistWide::kRing) launch_distill_mode<T, DistWide>(p, csize, stream);
  else launch_distill_mode<T, DistWidest>(p, csize, stream);
}

}  // namespace zq

using namespace zq;

static DistillParams distill_params(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher,
                                    const c10::optional<at::Tensor>& targets, const at::Tensor& sums,
                                    const at::Tensor* grad, int64_t vocab, int64_t ignore_index, double temperature,
                                    double alpha) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(0) > 0 && logits.size(1) > 0 &&
                  (logits.stride(1) == 1 || logits.size(1) == 1),
              "distill: logits [M, V] on the GPU with unit column stride");
  const int64_t M = logits.size(0), W = logits.size(1);
  TORCH_CHECK(vocab > 0 && vocab <= W && W < (1LL << 31), "distill: vocab must be 1 to the logits' width");
  TORCH_CHECK(ignore_index < 0 || ignore_index >= vocab, "distill: ignore_index must be outside the vocabulary");
  TORCH_CHECK(temperature > 0 && alpha >= 0 && alpha <= 1, "distill: temperature > 0, alpha in [0, 1]");
  const int dev = logits.get_device();
  auto here = [&](const at::Tensor& t) { return t.is_cuda() && t.get_device() == dev && t.is_contiguous(); };
  TORCH_CHECK(here(ids) && ids.dim() == 2 && ids.size(0) == M && ids.size(1) <= kDistMaxK &&
                  (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong),
              "distill: ids [M, K <= ", kDistMaxK, "] int32 or int64, contiguous, on the logits' device");
  TORCH_CHECK(here(teacher) && teacher.sizes() == ids.sizes() &&
                  (teacher.scalar_type() == at::kFloat || teacher.scalar_type() == at::kBFloat16 ||
                   teacher.scalar_type() == at::kHalf),
              "distill: teacher logits [M, K] fp32, bf16 or fp16, contiguous, on the logits' device");
  const bool has_targets = targets.has_value() && targets->defined();
  TORCH_CHECK(!has_targets || (here(*targets) && targets->scalar_type() == at::kLong && targets->numel() == M),
              "distill: targets [M] int64, contiguous, on the logits' device");
  TORCH_CHECK(has_targets || alpha == 1.0, "distill: alpha below 1 needs targets");
  TORCH_CHECK(here(sums) && sums.scalar_type() == at::kFloat && sums.numel() == 3 * M, "distill: sums [M, 3] fp32");
  if (grad != nullptr) {
    TORCH_CHECK(grad->is_cuda() && grad->get_device() == dev && grad->scalar_type() == logits.scalar_type() &&
                    grad->sizes() == logits.sizes() && (grad->stride(1) == 1 || W == 1) && (M == 1 || grad->stride(0) >= W),
                "distill: the gradient is like the logits, rows apart");
    // a logits row and its gradient row have one alignment: the kernel takes both by the same vectors
    const int64_t es = logits.element_size();
    TORCH_CHECK(((reinterpret_cast<uintptr_t>(logits.data_ptr()) ^ reinterpret_cast<uintptr_t>(grad->data_ptr())) & 15) == 0 &&
                    (M == 1 || ((logits.stride(0) - grad->stride(0)) * es) % 16 == 0),
                "distill: logits rows must be aligned as the gradient's");
  }
  TORCH_CHECK((reinterpret_cast<uintptr_t>(logits.data_ptr()) % logits.element_size()) == 0, "distill: alignment");
  DistillParams p = {};
  p.logits = logits.data_ptr();
  p.ids = ids.data_ptr();
  p.teacher = teacher.data_ptr();
  p.targets = has_targets ? targets->data_ptr<int64_t>() : nullptr;
  p.sums = sums.data_ptr<float>();
  p.grad = grad != nullptr ? grad->data_ptr() : nullptr;
  p.M = M;
  p.stride = logits.stride(0);
  p.grad_stride = grad != nullptr ? grad->stride(0) : 0;
  p.width = W;
  p.vocab = vocab;
  p.K = (int)ids.size(1);
  p.ids64 = ids.scalar_type() == at::kLong;
  p.teacher_type = teacher.scalar_type() == at::kFloat ? 0 : teacher.scalar_type() == at::kBFloat16 ? 1 : 2;
  p.soft_scale = (float)(1.4426950408889634 / temperature);
  p.alpha = (float)alpha;
  p.tau = (float)temperature;
  p.status = status_buffer(dev);
  return p;
}

template <typename T>
static void launch_distill_rows(DistillParams& p, float* loss, cudaStream_t stream) {
  launch_distill_shape<T>(p, stream);
  // (without a mean the rows are divided over a few blocks)
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const unsigned grid = loss != nullptr ? 1u : (unsigned)std::min<int64_t>(sms, (p.M + 31) / 32);
  distill_finish_kernel<T><<<grid, kDistFinish, 0, stream>>>(p, loss);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

static void launch_distill_typed(const at::Tensor& logits, DistillParams& p, float* loss) {
  auto stream = at::cuda::getCurrentCUDAStream();
  switch (logits.scalar_type()) {
    case at::kBFloat16: launch_distill_rows<__nv_bfloat16>(p, loss, stream); break;
    case at::kHalf: launch_distill_rows<__half>(p, loss, stream); break;
    case at::kFloat: launch_distill_rows<float>(p, loss, stream); break;
    default: TORCH_CHECK(false, "distill: bf16, fp16 or fp32 logits");
  }
}

// rows [M] and sums [M, 3] (fp32) are written; grad (optional): the gradient of the
// mean of the counted rows; loss (optional, [1]): that mean.
void distill(at::Tensor logits, at::Tensor ids, at::Tensor teacher, c10::optional<at::Tensor> targets,
             at::Tensor rows, at::Tensor sums, c10::optional<at::Tensor> grad, c10::optional<at::Tensor> loss,
             int64_t vocab, int64_t ignore_index, double temperature, double alpha) {
  const bool want = grad.has_value() && grad->defined();
  DistillParams p = distill_params(logits, ids, teacher, targets, sums, want ? &*grad : nullptr, vocab, ignore_index,
                                   temperature, alpha);
  TORCH_CHECK(rows.is_cuda() && rows.get_device() == logits.get_device() && rows.is_contiguous() &&
                  rows.scalar_type() == at::kFloat && rows.numel() == p.M,
              "distill: rows [M] fp32");
  p.rows = rows.data_ptr<float>();
  float* mean = nullptr;
  if (loss.has_value() && loss->defined()) {
    TORCH_CHECK(loss->is_cuda() && loss->get_device() == logits.get_device() && loss->scalar_type() == at::kFloat &&
                    loss->numel() == 1,
                "distill: loss is one fp32 value");
    mean = loss->data_ptr<float>();
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  launch_distill_typed(logits, p, mean);
}

// The gradient of the loss rows times g [M], or of their mean times g [1] (`mean`),
// from the sums that distill() wrote.
void distill_grad(at::Tensor logits, at::Tensor ids, at::Tensor teacher, c10::optional<at::Tensor> targets,
                  at::Tensor sums, at::Tensor g, at::Tensor grad, int64_t vocab, int64_t ignore_index,
                  double temperature, double alpha, bool mean) {
  DistillParams p = distill_params(logits, ids, teacher, targets, sums, &grad, vocab, ignore_index, temperature, alpha);
  TORCH_CHECK(g.is_cuda() && g.get_device() == logits.get_device() && g.is_contiguous() && g.scalar_type() == at::kFloat &&
                  g.numel() == (mean ? 1 : p.M),
              "distill: g fp32, [M] or one value for the mean");
  p.g = g.data_ptr<float>();
  p.grad_only = true;
  p.g_mean = mean;
  const c10::cuda::CUDAGuard guard(logits.device());
  launch_distill_typed(logits, p, nullptr);
}

// x *= g[0] in place (one more rounding); where g[0] is 1 the kernel returns at once
// and x is not touched.
void scale_by_scalar(at::Tensor x, at::Tensor g) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous() && (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0 && g.is_cuda() &&
                  g.get_device() == x.get_device() && g.scalar_type() == at::kFloat && g.numel() == 1,
              "scale_by_scalar: contiguous x, one fp32 value g on its device");
  if (x.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const unsigned grid = (unsigned)std::min<int64_t>((x.numel() + 2047) / 2048, 8 * (int64_t)sms);
  auto stream = at::cuda::getCurrentCUDAStream();
  const float* gp = g.data_ptr<float>();
  switch (x.scalar_type()) {
    case at::kBFloat16:
      scale_by_scalar_kernel<<<grid, 256, 0, stream>>>(reinterpret_cast<__nv_bfloat16*>(x.data_ptr()), gp, x.numel());
      break;
    case at::kFloat: scale_by_scalar_kernel<<<grid, 256, 0, stream>>>(x.data_ptr<float>(), gp, x.numel()); break;
    default: TORCH_CHECK(false, "scale_by_scalar: bf16 or fp32");
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
