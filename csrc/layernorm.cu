// Layer norm of rows of D columns, forward and backward, optionally after a residual
// addition and with its input kept in 8 bits for the backward.
//
//   h = x (+ delta, rounded to the type);  mu = mean h;  v = mean (h - mu)^2;
//   r = (v + eps)^-1/2;  n = (h - mu) r;  y = n w + b
// and with a = dy w (n from the kept h, which may be the 8-bit one):
//   dx = r (a - mean a - n mean(a n)) (+ dh);  dw = sum over rows dy n;  db = sum over rows dy
//
// A team of W warps takes one row at a time and holds it in registers, K tiles of 256 columns
// a warp, with w (and b, and the sums of dw and db) of the same columns beside it; teams go
// over the rows with a fixed stride, and the loads of the next row are under way while this
// one is reduced.  The variance is the joined sum of squares about each warp's own mean
// (columns n_i, mean m_i, squares q_i: q = sum q_i + n_i (m_i - mu)^2), so one exchange gives
// both and nothing cancels.  dw and db: a block's teams add up in team order in shared memory,
// the blocks' rows of partial sums are added in block order by a second kernel: no atomics.
//
// What bounds it: memory.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>

#include "rows.cuh"

namespace zq {

constexpr int kLnMaxWarps = 16;   // of a team
constexpr int kLnMaxTeams = 8;    // of a block

struct LnParams {
  const void *x, *delta, *dy, *dh;   // rows of pitch xs, deltas, dys, dhs
  int64_t xs, ds, dys, dhs;
  void *h, *y, *dx;                  // dense
  const void *w, *b;                 // type wt: 0 fp32, 1 bf16, 2 fp16
  float *mean, *rstd;                // [M]
  int8_t* codes;                     // [M, P], or null
  float* steps;                      // [M, G]
  float* part;                       // [grid, 2, D]
  int64_t M, P, G;
  int D, wt, W, R;                   // warps of a team, teams of a block
  float eps;
};

__device__ __forceinline__ float ln_param(const void* p, int type, int i) {
  if (type == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (type == 2) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}

template <bool VEC, int K>
__device__ __forceinline__ void ln_params(const void* p, int type, float absent, int wt, int W, int lane, int D,
                                          float (&v)[K][8]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (wt + k * W) * kTile + tile_col<VEC>(lane, i);
      v[k][i] = c >= D ? 0.0f : p == nullptr ? absent : ln_param(p, type, c);
    }
  }
}

// Every warp's pair of numbers, in every thread of the team.  Buffers alternate from row to
// row: a thread that writes one again has passed the other's barrier, to which its readers
// came after they had read.
__device__ __forceinline__ void ln_exchange(float2 (&buf)[kLnMaxWarps], float2 mine, int wt, int lane, int team, int W) {
  if (lane == 0) buf[wt] = mine;
  named_barrier(1 + team, W * 32);
}

template <typename T, bool VEC, int K, bool RES>
__global__ void __launch_bounds__(kLnMaxWarps * 32) ln_fwd_kernel(const __grid_constant__ LnParams p) {
  __shared__ float2 s_red[kLnMaxTeams][2][kLnMaxWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int W = p.W, team = warp / W, wt = warp - team * W, D = p.D;
  float w[K][8], b[K][8];
  ln_params<VEC, K>(p.w, p.wt, 1.0f, wt, W, lane, D, w);
  ln_params<VEC, K>(p.b, p.wt, 0.0f, wt, W, lane, D, b);
  float cols = 0.0f;   // of this warp
#pragma unroll
  for (int k = 0; k < K; ++k) cols += (float)max(0, min(kTile, D - (wt + k * W) * kTile));
  const float inv_cols = cols > 0.0f ? 1.0f / cols : 0.0f, inv_d = 1.0f / (float)D;

  const int64_t step = (int64_t)gridDim.x * p.R;
  RawTile<T, VEC> rx[K], rd[RES ? K : 1];
  auto load = [&](int64_t row) {
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.xs;
#pragma unroll
    for (int k = 0; k < K; ++k) rx[k].load(x, (wt + k * W) * kTile, lane, D);
    if constexpr (RES) {
      const T* d = reinterpret_cast<const T*>(p.delta) + row * p.ds;
#pragma unroll
      for (int k = 0; k < K; ++k) rd[k].load(d, (wt + k * W) * kTile, lane, D);
    }
  };
  int64_t row = (int64_t)blockIdx.x * p.R + team;
  if (row < p.M) load(row);
  for (int turn = 0; row < p.M; row += step, turn ^= 1) {
    float v[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rx[k].values(v[k]);
      if constexpr (RES) {
        float d[8];
        rd[k].values(d);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] += d[i];
        RawTile<T, VEC> h;
        h.set(v[k]);
        h.store(reinterpret_cast<T*>(p.h) + row * D, (wt + k * W) * kTile, lane, D);
        h.values(v[k]);   // as the next layer and the backward see it
      }
    }
    if (row + step < p.M) load(row + step);
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[k][i];
    float mu = warp_sum(s) * inv_cols;
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = v[k][i] - mu;
        if ((wt + k * W) * kTile + tile_col<VEC>(lane, i) < D) q = fmaf(d, d, q);
      }
    q = warp_sum(q);
    if (W > 1) {
      float2(&buf)[kLnMaxWarps] = s_red[team][turn];
      ln_exchange(buf, make_float2(mu, q), wt, lane, team, W);
      // columns of a warp: as above
      float m = 0.0f;
      auto columns = [&](int i) {
        float n = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) n += (float)max(0, min(kTile, D - (i + k * W) * kTile));
        return n;
      };
      for (int i = 0; i < W; ++i) m = fmaf(columns(i), buf[i].x, m);
      m *= inv_d;
      q = 0.0f;
      for (int i = 0; i < W; ++i) {
        const float d = buf[i].x - m;
        q += buf[i].y + columns(i) * d * d;
      }
      mu = m;
    }
    const float r = 1.0f / sqrtf(q * inv_d + p.eps);
    if (wt == 0 && lane == 0 && p.mean != nullptr) p.mean[row] = mu, p.rstd[row] = r;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int base = (wt + k * W) * kTile;
      if (p.codes != nullptr && base < D) keep_tile<VEC>(v[k], p.codes + row * p.P, p.steps + row * p.G, base, lane, D);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = fmaf((v[k][i] - mu) * r, w[k][i], b[k][i]);
      store_tile<T, VEC>(reinterpret_cast<T*>(p.y) + row * D, base, lane, D, v[k]);
    }
  }
}

// KEPT: h in 8 bits; RES: dh is added
template <typename T, bool VEC, int K, bool KEPT, bool RES>
__global__ void __launch_bounds__(kLnMaxWarps * 32) ln_bwd_kernel(const __grid_constant__ LnParams p) {
  __shared__ float2 s_red[kLnMaxTeams][2][kLnMaxWarps];
  extern __shared__ float s_part[];   // [2, D], teams add up
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int W = p.W, team = warp / W, wt = warp - team * W, D = p.D;
  float w[K][8], dw[K][8], db[K][8];
  ln_params<VEC, K>(p.w, p.wt, 1.0f, wt, W, lane, D, w);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[k][i] = db[k][i] = 0.0f;
  const float inv_d = 1.0f / (float)D;

  const int64_t step = (int64_t)gridDim.x * p.R;
  RawTile<T, VEC> rg[K], rx[KEPT ? 1 : K], rh[RES ? K : 1];
  RawCodes<VEC> rc[KEPT ? K : 1];
  float mu_next = 0.0f, r_next = 0.0f;
  auto load = [&](int64_t row) {
    const T* g = reinterpret_cast<const T*>(p.dy) + row * p.dys;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int base = (wt + k * W) * kTile;
      rg[k].load(g, base, lane, D);
      if constexpr (KEPT) rc[k].load(p.codes + row * p.P, p.steps + row * p.G, base, lane, D);
      else rx[k].load(reinterpret_cast<const T*>(p.x) + row * p.xs, base, lane, D);
      if constexpr (RES) rh[k].load(reinterpret_cast<const T*>(p.dh) + row * p.dhs, base, lane, D);
    }
    mu_next = p.mean[row];
    r_next = p.rstd[row];
  };
  int64_t row = (int64_t)blockIdx.x * p.R + team;
  if (row < p.M) load(row);
  for (int turn = 0; row < p.M; row += step, turn ^= 1) {
    const float mu = mu_next, r = r_next;
    float a[K][8], n[K][8];
    RawTile<T, VEC> h[RES ? K : 1];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rg[k].values(a[k]);
      if constexpr (KEPT) rc[k].values(n[k]);
      else rx[k].values(n[k]);
      if constexpr (RES) h[k] = rh[k];
    }
    if (row + step < p.M) load(row + step);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // (past the row's end dy and w are 0)
        n[k][i] = (n[k][i] - mu) * r;
        dw[k][i] = fmaf(a[k][i], n[k][i], dw[k][i]);
        db[k][i] += a[k][i];
        a[k][i] *= w[k][i];
        s1 += a[k][i];
        s2 = fmaf(a[k][i], n[k][i], s2);
      }
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (W > 1) {
      float2(&buf)[kLnMaxWarps] = s_red[team][turn];
      ln_exchange(buf, make_float2(s1, s2), wt, lane, team, W);
      s1 = s2 = 0.0f;
      for (int i = 0; i < W; ++i) s1 += buf[i].x, s2 += buf[i].y;
    }
    s1 *= inv_d;
    s2 *= inv_d;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float add[8];
      if constexpr (RES) h[k].values(add);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = r * (a[k][i] - s1 - n[k][i] * s2);
        a[k][i] = RES ? d + add[i] : d;
      }
      store_tile<T, VEC>(reinterpret_cast<T*>(p.dx) + row * D, (wt + k * W) * kTile, lane, D, a[k]);
    }
  }
  if (p.part == nullptr) return;
  float* out = p.part + (int64_t)blockIdx.x * 2 * D;
  for (int t = 0; t < p.R; ++t) {
    if (t > 0) __syncthreads();
    if (team != t) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = (wt + k * W) * kTile + tile_col<VEC>(lane, i);
        if (c < D) {
          const float u = t > 0 ? s_part[c] + dw[k][i] : dw[k][i];
          const float v = t > 0 ? s_part[D + c] + db[k][i] : db[k][i];
          if (t == p.R - 1) out[c] = u, out[D + c] = v;
          else s_part[c] = u, s_part[D + c] = v;
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
  TORCH_CHECK(wt == at::kFloat || wt == at::kBFloat16 || wt == at::kHalf, "layer_norm: weight in fp32, bf16 or fp16");
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

// Tiles of a warp, warps of a team, teams of a block: two tiles a warp where 16 warps reach
// (more columns in flight per barrier than one, and the sums of the backward fit beside them),
// about 8 warps a block.
int ln_shape(LnParams& p) {
  const int tiles = (p.D + kTile - 1) / kTile;
  const int K = tiles == 1 ? 1 : tiles <= 2 * kLnMaxWarps ? 2 : 4;
  p.W = (tiles + K - 1) / K;
  p.R = std::max(1, kLnMaxTeams / p.W);
  return K;
}

// Blocks that are resident at once (a kernel's, by its shape), no more than there are rows for
template <typename F>
unsigned ln_grid(F kern, const LnParams& p, size_t smem) {
  int n = 0;
  C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, p.W * p.R * 32, smem));
  TORCH_CHECK(n > 0, "layer_norm: a block does not fit the device");
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  return (unsigned)std::min<int64_t>((p.M + p.R - 1) / p.R, n * sms);
}

}  // namespace

#define ZQ_LN_TYPES(TYPE, ...)                                                 \
  switch (TYPE) {                                                              \
    case at::kBFloat16: { using T = __nv_bfloat16; __VA_ARGS__; break; }       \
    case at::kHalf: { using T = __half; __VA_ARGS__; break; }                  \
    case at::kFloat: { using T = float; __VA_ARGS__; break; }                  \
    default: TORCH_CHECK(false, "layer_norm: bf16, fp16 or fp32");             \
  }

template <typename T, bool VEC, int K>
static void ln_fwd_launch(const LnParams& p, cudaStream_t stream) {
  auto go = [&](auto kern) {
    kern<<<ln_grid(kern, p, 0), p.W * p.R * 32, 0, stream>>>(p);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  };
  if (p.delta != nullptr) go(ln_fwd_kernel<T, VEC, K, true>);
  else go(ln_fwd_kernel<T, VEC, K, false>);
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
  const int K = ln_shape(p);
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
  const size_t smem = sums && p.R > 1 ? (size_t)2 * p.D * 4 : 0;
  auto go = [&](auto kern) {
    const unsigned grid = ln_grid(kern, p, smem);
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
  if (p.codes != nullptr) {
    if (p.dh != nullptr) go(ln_bwd_kernel<T, VEC, K, true, true>);
    else go(ln_bwd_kernel<T, VEC, K, true, false>);
  } else {
    if (p.dh != nullptr) go(ln_bwd_kernel<T, VEC, K, false, true>);
    else go(ln_bwd_kernel<T, VEC, K, false, false>);
  }
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
  const int K = ln_shape(p);
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
