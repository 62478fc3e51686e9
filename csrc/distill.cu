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
// One block (or a cluster of blocks that split the columns, when there are fewer
// rows than SMs) works on one row at a time:
//   pass 1  running maximum and sums of exp2 in 32 bits, one read of the row;
//   pass 2  the gradient, from the row read again - it is still in L2: all rows
//           in flight are grid x V x 2 B = 90 MB at V = 152064, and the
//           gradient is written with streaming stores so as not to push them
//           out.  So the logits come from HBM once and the gradient goes there
//           once; n is counted by every block from the targets beforehand.
// The K + 1 columns whose gradient has a p or one-hot term are written a second
// time by the block that owns the column, each with its terms summed in 32 bits
// and rounded once; entries with the same id sum their p in entry order, so
// there are no atomics.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"

namespace zq {

constexpr int kDistThreads = 512;
constexpr int kDistWarps = kDistThreads / 32;
constexpr int kDistMaxK = 1024;
constexpr int kDistMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DistillParams {
  const void* logits;
  const void* ids;          // int32 or int64 [M, K]
  const void* teacher;      // fp32, bf16 or fp16 [M, K]
  const int64_t* targets;   // [M] or null
  float* rows;              // [M] loss rows (written unless GRAD)
  float* sums;              // [M, 3]: maximum and the two sums of a row; written, or read by GRAD
  const float* g;           // GRAD: gradient of each loss row
  void* grad;               // [M, width]; null: forward alone
  int64_t M, stride, grad_stride, width, vocab;
  int K, ids64, teacher_type;
  float soft_scale;         // log2(e) / τ
  float alpha, tau;
  bool grad_only;
};

__device__ __forceinline__ float dist_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's running maximum m (in the logits' own units) and the sums of
// 2^(x·s + shift(m, s)) at the two scales s.  The shift is the ROUNDED product
// -m·s, everywhere the same one: x·s + shift is then one exact product and one
// rounding of a small number, and no error of the size of m·s enters.
struct RowSums {
  float m, soft, hard;
};

// (a maximum of -inf shifts by nothing: sums of 0, not NaN)
__device__ __forceinline__ float dist_shift(float m, float s) { return m == -INFINITY ? 0.0f : -m * s; }

// factor of the sums when the maximum goes from `from` up to `to`
__device__ __forceinline__ float dist_raise(float from, float to, float s) {
  return from == -INFINITY ? 0.0f : dist_exp2(dist_shift(to, s) - dist_shift(from, s));
}

template <bool SOFT, bool HARD>
__device__ __forceinline__ void sums_merge(RowSums& a, const RowSums& b, float ss) {
  const float m = fmaxf(a.m, b.m);
  // sums over nothing but -inf are 0 (or NaN, which stays)
  if constexpr (SOFT)
    a.soft = (a.m == m ? a.soft : a.soft * dist_raise(a.m, m, ss)) + (b.m == m ? b.soft : b.soft * dist_raise(b.m, m, ss));
  if constexpr (HARD)
    a.hard = (a.m == m ? a.hard : a.hard * dist_raise(a.m, m, kLog2e)) + (b.m == m ? b.hard : b.hard * dist_raise(b.m, m, kLog2e));
  a.m = m;
}

template <bool SOFT, bool HARD, int N>
__device__ __forceinline__ void sums_add(RowSums& a, const float (&v)[N], float ss) {
  float cm = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) cm = fmaxf(cm, v[i]);
  if (cm > a.m) {
    if constexpr (SOFT) a.soft *= dist_raise(a.m, cm, ss);
    if constexpr (HARD) a.hard *= dist_raise(a.m, cm, kLog2e);
    a.m = cm;
  }
  const float bs = dist_shift(a.m, ss), bh = dist_shift(a.m, kLog2e);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (SOFT) a.soft += dist_exp2(fmaf(v[i], ss, bs));
    if constexpr (HARD) a.hard += dist_exp2(fmaf(v[i], kLog2e, bh));
  }
}

template <typename T>
struct DistVec {
  static constexpr int N = 16 / (int)sizeof(T);
  union { uint4 u; T t[N]; } w;
  __device__ __forceinline__ void floats(float (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32<T>(w.t[i]);
  }
};

__device__ __forceinline__ float dist_teacher(const DistillParams& p, int64_t i) {
  if (p.teacher_type == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.teacher)[i]);
  if (p.teacher_type == 2) return __half2float(reinterpret_cast<const __half*>(p.teacher)[i]);
  return reinterpret_cast<const float*>(p.teacher)[i];
}

// shared-memory words of another block of the cluster
__device__ __forceinline__ float dist_peer_f32(const float* local, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(smem_u32(local), rank)) : "memory");
  return v;
}

// SOFT: α > 0 and τ != 1, or α = 1: the sums at 1/τ; HARD: the sums at 1 (with
// τ = 1 one set of sums serves both terms and is the HARD one).
template <typename T, bool SOFT, bool HARD>
__global__ void __launch_bounds__(kDistThreads, 2) distill_kernel(const __grid_constant__ DistillParams p) {
  constexpr int N = DistVec<T>::N;
  extern __shared__ uint8_t dist_smem[];
  float* s_p = reinterpret_cast<float*>(dist_smem);         // [K + 1] teacher probability
  int* s_id = reinterpret_cast<int*>(s_p + p.K + 1);        // [K + 1] column, or -1
  __shared__ float s_part[kDistWarps][3];
  __shared__ float s_block[4];                              // m, soft, hard of this block; mass
  __shared__ float s_kl;
  __shared__ int s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t csize;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
  const int crank = csize > 1 ? (int)cluster_ctarank() : 0;
  const int64_t row0 = blockIdx.x / csize, row_step = gridDim.x / csize;
  const float ss = p.soft_scale;

  float inv_n = 0.0f;
  if (p.grad != nullptr && !p.grad_only) {   // rows counted, for the mean's gradient
    float n = (float)p.M;
    if (p.targets != nullptr) {
      if (tid == 0) s_count = 0;
      __syncthreads();
      int c = 0;
      for (int64_t i = tid; i < p.M; i += kDistThreads) {
        const int64_t y = p.targets[i];
        c += (y >= 0 && y < p.vocab) ? 1 : 0;
      }
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) atomicAdd(&s_count, c);
      __syncthreads();
      n = (float)s_count;
    }
    inv_n = 1.0f / fmaxf(n, 1.0f);
  }

  for (int64_t row = row0; row < p.M; row += row_step) {
    const T* z = reinterpret_cast<const T*>(p.logits) + row * p.stride;
    const int64_t y = p.targets != nullptr ? p.targets[row] : -1;
    const bool counted = p.targets == nullptr || (y >= 0 && y < p.vocab);
    const float gscale = p.grad == nullptr ? 0.0f : p.grad_only ? (counted ? p.g[row] : 0.0f) : (counted ? inv_n : 0.0f);
    T* dz = p.grad != nullptr ? reinterpret_cast<T*>(p.grad) + row * p.grad_stride : nullptr;
    // columns: `head` up to the first 16-byte boundary, then whole vectors, then a tail
    const int mis = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
    const int64_t head = min((int64_t)(mis == 0 ? 0 : N - mis), p.vocab);
    const int64_t nvec = (p.vocab - head) / N;
    const int64_t tail = head + nvec * N;
    // this block's vectors
    const int64_t per = (nvec + csize - 1) / csize;
    const int64_t v0 = min(nvec, per * crank), v1 = min(nvec, v0 + per);
    const uint4* zv = reinterpret_cast<const uint4*>(z + head);

    if (!counted) {   // nothing counts: no loss, a gradient of zeros
      if (tid == 0 && crank == 0 && !p.grad_only) {
        p.rows[row] = 0.0f;
        p.sums[3 * row] = p.sums[3 * row + 1] = p.sums[3 * row + 2] = 0.0f;
      }
      if (dz != nullptr) {
        // the gradient rows have the logits' alignment (checked by the host)
        uint4* dv = reinterpret_cast<uint4*>(dz + head);
        for (int64_t i = v0 + tid; i < v1; i += kDistThreads) __stcs(dv + i, make_uint4(0, 0, 0, 0));
        if (crank == 0) {
          for (int64_t c = tid; c < head; c += kDistThreads) dz[c] = from_f32<T>(0.0f);
          for (int64_t c = tail + tid; c < p.width; c += kDistThreads) dz[c] = from_f32<T>(0.0f);
        }
      }
      continue;   // the same in every block of the cluster
    }

    // teacher entries
    __syncthreads();   // the last row's entries have been read
    for (int k = tid; k <= p.K; k += kDistThreads) {
      int id = -1;
      float t = -INFINITY;
      if (k == p.K) {
        id = (p.targets != nullptr) ? (int)y : -1;
      } else {
        const int64_t e = row * p.K + k;
        const int64_t v = p.ids64 ? reinterpret_cast<const int64_t*>(p.ids)[e]
                                  : (int64_t)reinterpret_cast<const int32_t*>(p.ids)[e];
        if (v >= 0 && v < p.vocab) {
          id = (int)v;
          t = dist_teacher(p, e) * ss;   // t / τ in log2 units
        }
      }
      s_id[k] = id;
      s_p[k] = t;
    }

    if (!p.grad_only) {
      RowSums a{-INFINITY, 0.0f, 0.0f};
      int64_t i = v0 + tid;
      for (; i + 3 * kDistThreads < v1; i += 4 * kDistThreads) {   // four loads in flight
        DistVec<T> w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u].w.u = __ldg(zv + i + u * kDistThreads);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float v[N];
          w[u].floats(v);
          sums_add<SOFT, HARD>(a, v, ss);
        }
      }
      for (; i < v1; i += kDistThreads) {
        DistVec<T> w;
        w.w.u = __ldg(zv + i);
        float v[N];
        w.floats(v);
        sums_add<SOFT, HARD>(a, v, ss);
      }
      if (crank == 0) {
        for (int64_t c = tid; c < head; c += kDistThreads) {
          const float v[1] = {to_f32<T>(z[c])};
          sums_add<SOFT, HARD>(a, v, ss);
        }
        for (int64_t c = tail + tid; c < p.vocab; c += kDistThreads) {
          const float v[1] = {to_f32<T>(z[c])};
          sums_add<SOFT, HARD>(a, v, ss);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        RowSums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.soft = SOFT ? __shfl_xor_sync(0xffffffffu, a.soft, o) : 0.0f;
        b.hard = HARD ? __shfl_xor_sync(0xffffffffu, a.hard, o) : 0.0f;
        sums_merge<SOFT, HARD>(a, b, ss);
      }
      if (lane == 0) {
        s_part[warp][0] = a.m;
        s_part[warp][1] = a.soft;
        s_part[warp][2] = a.hard;
      }
    }
    __syncthreads();   // entries and the warps' sums
    RowSums a{-INFINITY, 0.0f, 0.0f};
    if (!p.grad_only) {
      // every thread joins the parts in the same order
#pragma unroll 4
      for (int w = 0; w < kDistWarps; ++w)
        sums_merge<SOFT, HARD>(a, RowSums{s_part[w][0], s_part[w][1], s_part[w][2]}, ss);
      if (csize > 1) {
        if (tid == 0) {
          s_block[0] = a.m;
          s_block[1] = a.soft;
          s_block[2] = a.hard;
        }
        cluster_sync_all();
        a = RowSums{-INFINITY, 0.0f, 0.0f};
        for (uint32_t r = 0; r < csize; ++r)
          sums_merge<SOFT, HARD>(a, RowSums{dist_peer_f32(&s_block[0], r), dist_peer_f32(&s_block[1], r),
                                            dist_peer_f32(&s_block[2], r)}, ss);
        cluster_sync_all();   // read by all before the next row (or the exit)
      }
    } else {
      a = RowSums{p.sums[3 * row], p.sums[3 * row + 1], p.sums[3 * row + 2]};
    }
    // shifts and sums of the two softmaxes; with one of them it stands for both
    const float shift_h = dist_shift(a.m, kLog2e), shift_s = SOFT ? dist_shift(a.m, ss) : shift_h;
    const float sum_h = a.hard, sum_s = SOFT ? a.soft : a.hard;

    // warp 0: the teacher's distribution (in place of its logits) and the loss
    if (warp == 0) {
      float tm = -INFINITY;
      for (int k = lane; k < p.K; k += 32) tm = fmaxf(tm, s_p[k]);
      tm = -dist_shift(warp_max(tm), 1.0f);
      float mass = 0.0f;
      for (int k = lane; k < p.K; k += 32) mass += dist_exp2(s_p[k] - tm);
      mass = warp_sum(mass);
      const bool some = !(mass == 0.0f);
      const float lm = log2f(mass), inv = 1.0f / mass;
      const float log_s = log2f(sum_s);
      float kl = 0.0f;
      for (int k = lane; k < p.K; k += 32) {
        const float d = s_p[k] - tm, pk = some ? dist_exp2(d) * inv : 0.0f;
        if (s_id[k] >= 0 && !(pk == 0.0f) && !p.grad_only)
          kl += pk * ((d - lm) - (fmaf(to_f32<T>(z[s_id[k]]), ss, shift_s) - log_s));
        s_p[k] = pk;
      }
      if (!p.grad_only) {
        kl = warp_sum(kl);
        if (lane == 0 && crank == 0) {
          float loss = 0.0f;
          if (p.alpha > 0.0f) loss = p.alpha * p.tau * p.tau * kLn2 * kl;
          if (p.alpha < 1.0f)
            loss += (1.0f - p.alpha) * kLn2 * (log2f(sum_h) - fmaf(to_f32<T>(z[y]), kLog2e, shift_h));
          p.rows[row] = loss;
          p.sums[3 * row] = a.m;
          p.sums[3 * row + 1] = a.soft;
          p.sums[3 * row + 2] = a.hard;
        }
      }
      if (lane == 0) {
        s_p[p.K] = 0.0f;
        s_block[3] = some ? 1.0f : 0.0f;
      }
    }
    if (dz == nullptr) continue;   // the next row's first barrier keeps the entries
    __syncthreads();
    // a row without entries has no soft term
    const float cs = p.alpha * p.tau * s_block[3] * gscale, ch = (1.0f - p.alpha) * gscale;
    // the softmaxes' denominators go into the factors; τ = 1: both terms share one softmax
    const float fs = cs / sum_s, fh = (SOFT ? ch : ch + cs) / sum_h;
    auto smooth = [&](float v) {
      float d = 0.0f;
      if constexpr (SOFT) d = fs * dist_exp2(fmaf(v, ss, shift_s));
      if constexpr (HARD) d = fmaf(fh, dist_exp2(fmaf(v, kLog2e, shift_h)), d);
      return d;
    };
    uint4* dv = reinterpret_cast<uint4*>(dz + head);
    int64_t i = v0 + tid;
    auto store = [&](int64_t at, const DistVec<T>& w) {
      float v[N];
      w.floats(v);
      DistVec<T> o;
#pragma unroll
      for (int j = 0; j < N; ++j) o.w.t[j] = from_f32<T>(smooth(v[j]));
      __stcs(dv + at, o.w.u);
    };
    for (; i + 3 * kDistThreads < v1; i += 4 * kDistThreads) {
      DistVec<T> w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u].w.u = __ldcs(zv + i + u * kDistThreads);
#pragma unroll
      for (int u = 0; u < 4; ++u) store(i + u * kDistThreads, w[u]);
    }
    for (; i < v1; i += kDistThreads) {
      DistVec<T> w;
      w.w.u = __ldcs(zv + i);
      store(i, w);
    }
    if (crank == 0) {
      for (int64_t c = tid; c < head; c += kDistThreads) dz[c] = from_f32<T>(smooth(to_f32<T>(z[c])));
      for (int64_t c = tail + tid; c < p.vocab; c += kDistThreads) dz[c] = from_f32<T>(smooth(to_f32<T>(z[c])));
      for (int64_t c = p.vocab + tid; c < p.width; c += kDistThreads) dz[c] = from_f32<T>(0.0f);
    }
    __syncthreads();   // the smooth part of these columns is written (by this block)
    for (int k = tid; k <= p.K; k += kDistThreads) {
      const int id = s_id[k];
      if (id < 0) continue;
      const bool edge = id < head || id >= tail;
      const int64_t vec = edge ? 0 : (id - head) / N;
      if (edge ? crank != 0 : (vec < v0 || vec >= v1)) continue;   // another block's column
      float pk = 0.0f;
      for (int j = 0; j < p.K; ++j) pk += s_id[j] == id ? s_p[j] : 0.0f;
      float d = smooth(to_f32<T>(z[id])) - cs * pk;
      if (p.targets != nullptr && id == (int)y) d -= ch;
      dz[id] = from_f32<T>(d);
    }
  }
}

// loss = sum of the rows over the number of counted ones, in 64 bits and a fixed order
__global__ void __launch_bounds__(1024) distill_mean_kernel(const float* __restrict__ rows,
                                                            const int64_t* __restrict__ targets,
                                                            float* __restrict__ loss, int64_t M, int64_t vocab) {
  __shared__ double s_sum[32];
  __shared__ int s_n[32];
  double s = 0.0;
  int n = 0;
  for (int64_t i = threadIdx.x; i < M; i += 1024) {
    s += rows[i];
    n += (targets == nullptr || (targets[i] >= 0 && targets[i] < vocab)) ? 1 : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = s;
    s_n[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
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
    DistVec<T> w;
    w.w.u = reinterpret_cast<const uint4*>(x)[i];
#pragma unroll
    for (int j = 0; j < N; ++j) w.w.t[j] = from_f32<T>(to_f32<T>(w.w.t[j]) * f);
    reinterpret_cast<uint4*>(x)[i] = w.w.u;
  }
  for (int64_t i = nv * N + first; i < n; i += step) x[i] = from_f32<T>(to_f32<T>(x[i]) * f);
}

template <typename T>
static void launch_distill(const DistillParams& p, cudaStream_t stream) {
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // fewer rows than SMs: clusters split a row's columns, down to 8 KB of logits a
  // block (below that the exchange costs more than the shorter pass saves)
  int csize = 1;
  while (csize < kDistMaxCluster && p.M * csize * 2 <= sms && p.vocab * (int64_t)sizeof(T) / (2 * csize) >= 8192) csize *= 2;
  const unsigned rows = (unsigned)std::min<int64_t>(p.M, 2 * (int64_t)sms);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * csize);
  cfg.blockDim = dim3(kDistThreads);
  cfg.dynamicSmemBytes = (size_t)(p.K + 1) * 8;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool hard = p.alpha < 1.0f || p.tau == 1.0f, soft = p.alpha > 0.0f && p.tau != 1.0f;
  auto kern = soft && hard ? distill_kernel<T, true, true> : soft ? distill_kernel<T, true, false> : distill_kernel<T, false, true>;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
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
  return p;
}

static void launch_distill_typed(const at::Tensor& logits, const DistillParams& p) {
  auto stream = at::cuda::getCurrentCUDAStream();
  switch (logits.scalar_type()) {
    case at::kBFloat16: launch_distill<__nv_bfloat16>(p, stream); break;
    case at::kHalf: launch_distill<__half>(p, stream); break;
    case at::kFloat: launch_distill<float>(p, stream); break;
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
  const c10::cuda::CUDAGuard guard(logits.device());
  launch_distill_typed(logits, p);
  if (loss.has_value() && loss->defined()) {
    TORCH_CHECK(loss->is_cuda() && loss->get_device() == logits.get_device() && loss->scalar_type() == at::kFloat &&
                    loss->numel() == 1,
                "distill: loss is one fp32 value");
    distill_mean_kernel<<<1, 1024, 0, at::cuda::getCurrentCUDAStream()>>>(p.rows, p.targets, loss->data_ptr<float>(), p.M,
                                                                          p.vocab);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

// The gradient of the loss rows times g [M], from the sums that distill() wrote.
void distill_grad(at::Tensor logits, at::Tensor ids, at::Tensor teacher, c10::optional<at::Tensor> targets,
                  at::Tensor sums, at::Tensor g, at::Tensor grad, int64_t vocab, int64_t ignore_index,
                  double temperature, double alpha) {
  DistillParams p = distill_params(logits, ids, teacher, targets, sums, &grad, vocab, ignore_index, temperature, alpha);
  TORCH_CHECK(g.is_cuda() && g.get_device() == logits.get_device() && g.is_contiguous() && g.scalar_type() == at::kFloat &&
                  g.numel() == p.M,
              "distill: g [M] fp32");
  p.g = g.data_ptr<float>();
  p.grad_only = true;
  const c10::cuda::CUDAGuard guard(logits.device());
  launch_distill_typed(logits, p);
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
