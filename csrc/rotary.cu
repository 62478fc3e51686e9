// Rotary positions with explicit positions, either pair layout, part of the
// head, and context scaling, for q and k in one launch.
//
//   y = f · (a cos φ - b sin φ, b cos φ + a sin φ),   φ = 2π · pos · turns[i]
//
// for the pair (a, b) = (x[i], x[i + R/2]) (half layout) or (x[2i], x[2i + 1])
// (interleaved), i < R/2; columns R.. pass through.  The gradient is the same
// map with the angle negated (sign = -1).
//
// Angles: pos · turns[i] is formed in 64 bits and reduced to a fraction of a
// turn there (at position 262144 an angle held in 32 bits is off by up to 2^-6
// radians), then sin and cos are taken in 32 bits of an argument in [-1, 1] half
// turns.  They are computed once for each (token, pair)
// into shared memory and used by all heads of the token: R/2 evaluations for
// (Hq + Hk) · D elements, so the kernel stays bound by memory.  turns travels in
// the kernel's parameters: no table in global memory to keep or to fill.
//
// A block takes `tile` tokens at a time; a thread moves 16 bytes of each half of
// the pair range (one 16-byte vector when interleaved).  Rows that are not
// 16-byte aligned, or whose widths are not whole vectors, take the element-wise
// form of the same code.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"

namespace zq {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 128;   // rotary width up to 256
constexpr int kRotMaxTile = 16;     // tokens per block iteration

struct RotarySide {
  const void* x;
  void* y;                   // contiguous [T, heads, D]
  int64_t token_stride, head_stride;
  int heads;
};

struct RotaryParams {
  RotarySide side[2];        // q, k
  const void* positions;
  int64_t tokens, pos_len;   // token t sits at positions[t % pos_len]
  int dim, rot, tile, pos64;
  float sin_factor, factor;
  double turns[kRotMaxPairs];
};

template <typename T, int VEC, bool WIDE>
__device__ __forceinline__ void rot_load(const T* p, float (&v)[VEC]) {
  if constexpr (WIDE) {
    static_assert(VEC * sizeof(T) == 16, "one 16-byte vector");
    union { uint4 u; T t[VEC]; } w;
    w.u = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32<T>(w.t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32<T>(p[i]);
  }
}

template <typename T, int VEC, bool WIDE>
__device__ __forceinline__ void rot_store(T* p, const float (&v)[VEC]) {
  if constexpr (WIDE) {
    union { uint4 u; T t[VEC]; } w;
#pragma unroll
    for (int i = 0; i < VEC; ++i) w.t[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = w.u;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = from_f32<T>(v[i]);
  }
}

// VEC elements per access: 16 bytes (WIDE), or 1 (half layout) / 2 (interleaved)
template <typename T, int VEC, bool WIDE, bool INTER>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 cs[];   // [tile][R/2] (cos, sin), times the factor
  const int half = p.rot / 2;
  const int turn_items = INTER ? p.rot / VEC : half / VEC;
  constexpr int PASS = (INTER && !WIDE) ? 1 : VEC;   // widths past R need not be whole pairs
  const int items = turn_items + (p.dim - p.rot) / PASS;
  const int heads = p.side[0].heads + p.side[1].heads;
  const int per_token = heads * items;
  for (int64_t t0 = (int64_t)blockIdx.x * p.tile; t0 < p.tokens; t0 += (int64_t)gridDim.x * p.tile) {
    const int nt = (int)min((int64_t)p.tile, p.tokens - t0);
    for (int i = threadIdx.x; i < nt * half; i += kRotThreads) {
      const int64_t at = (t0 + i / half) % p.pos_len;
      const int64_t pos = p.pos64 ? reinterpret_cast<const int64_t*>(p.positions)[at]
                                  : (int64_t)reinterpret_cast<const int32_t*>(p.positions)[at];
      const double turn = (double)pos * p.turns[i % half];
      float s, c;
      sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
      cs[i] = make_float2(c * p.factor, s * p.sin_factor);
    }
    __syncthreads();
    for (int n = threadIdx.x; n < nt * per_token; n += kRotThreads) {
      const int tok = n / per_token, in = n - tok * per_token;
      const int hd = in / items, it = in - hd * items;
      const bool second = hd >= p.side[0].heads;
      const RotarySide& sd = p.side[second ? 1 : 0];
      const int h = second ? hd - p.side[0].heads : hd;
      const T* x = reinterpret_cast<const T*>(sd.x) + (t0 + tok) * sd.token_stride + h * sd.head_stride;
      T* y = reinterpret_cast<T*>(sd.y) + ((t0 + tok) * sd.heads + h) * (int64_t)p.dim;
      if (it >= turn_items) {   // columns past the rotary width
        const int c = p.rot + (it - turn_items) * PASS;
        if constexpr (WIDE) {
          *reinterpret_cast<uint4*>(y + c) = *reinterpret_cast<const uint4*>(x + c);
        } else {
#pragma unroll
          for (int i = 0; i < PASS; ++i) y[c + i] = x[c + i];
        }
        continue;
      }
      if constexpr (INTER) {
        const float2* w = cs + tok * half + it * (VEC / 2);
        float v[VEC], o[VEC];
        rot_load<T, VEC, WIDE>(x + it * VEC, v);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          o[2 * i] = rope_lo(v[2 * i], v[2 * i + 1], w[i].x, w[i].y);
          o[2 * i + 1] = rope_hi(v[2 * i], v[2 * i + 1], w[i].x, w[i].y);
        }
        rot_store<T, VEC, WIDE>(y + it * VEC, o);
      } else {
        const float2* w = cs + tok * half + it * VEC;
        float a[VEC], b[VEC], lo[VEC], hi[VEC];
        rot_load<T, VEC, WIDE>(x + it * VEC, a);
        rot_load<T, VEC, WIDE>(x + half + it * VEC, b);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          lo[i] = rope_lo(a[i], b[i], w[i].x, w[i].y);
          hi[i] = rope_hi(a[i], b[i], w[i].x, w[i].y);
        }
        rot_store<T, VEC, WIDE>(y + it * VEC, lo);
        rot_store<T, VEC, WIDE>(y + half + it * VEC, hi);
      }
    }
    __syncthreads();   // the next tokens' angles overwrite these
  }
}

template <typename T>
static void launch_rotary(const RotaryParams& p, bool wide, bool inter, unsigned grid, cudaStream_t stream) {
  constexpr int W = 16 / (int)sizeof(T);
  const size_t smem = (size_t)p.tile * (p.rot / 2) * sizeof(float2);
  if (wide)
    inter ? rotary_kernel<T, W, true, true><<<grid, kRotThreads, smem, stream>>>(p)
          : rotary_kernel<T, W, true, false><<<grid, kRotThreads, smem, stream>>>(p);
  else
    inter ? rotary_kernel<T, 2, false, true><<<grid, kRotThreads, smem, stream>>>(p)
          : rotary_kernel<T, 1, false, false><<<grid, kRotThreads, smem, stream>>>(p);
}

}  // namespace zq

using namespace zq;

// q [T, Hq, D] and (optional) k [T, Hk, D], unit stride inside a head; qo, ko
// contiguous; positions int32 / int64 (1-D); turns: fp64 CPU tensor [R/2] of
// turns per position; factor scales cos and sin, sign = -1 turns back.
void rotary(at::Tensor q, c10::optional<at::Tensor> k, at::Tensor positions, at::Tensor turns, at::Tensor qo,
            c10::optional<at::Tensor> ko, bool interleaved, double factor, double sign) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && (!k.has_value() || (k->is_cuda() && k->dim() == 3 && ko.has_value())),
              "rotary: q and k are [T, H, D] CUDA tensors");
  TORCH_CHECK(turns.device().is_cpu() && turns.scalar_type() == at::kDouble && turns.is_contiguous() &&
                  turns.numel() >= 1 && turns.numel() <= kRotMaxPairs && 2 * turns.numel() <= q.size(2),
              "rotary: turns must be 1 to ", kRotMaxPairs, " fp64 values on the CPU, two columns of the head each");
  TORCH_CHECK(positions.is_cuda() && positions.get_device() == q.get_device() && positions.is_contiguous() &&
                  (positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt),
              "rotary: positions must be contiguous int32 or int64 on q's device");
  const int64_t T = q.size(0), D = q.size(2);
  if (T == 0) return;
  TORCH_CHECK(positions.numel() > 0 && T % positions.numel() == 0, "rotary: one position per token");
  RotaryParams p;
  const int64_t esize = q.element_size();
  const int64_t W = 16 / esize, R = 2 * turns.numel();
  bool wide = D % W == 0 && (D - R) % W == 0 && (interleaved ? R : R / 2) % W == 0;
  const at::Tensor* xs[2] = {&q, k.has_value() ? &*k : nullptr};
  const at::Tensor* ys[2] = {&qo, k.has_value() ? &*ko : nullptr};
  int64_t heads = 0;
  for (int i = 0; i < 2; ++i) {
    if (xs[i] == nullptr) {
      p.side[i] = RotarySide{nullptr, nullptr, 0, 0, 0};
      continue;
    }
    const at::Tensor &x = *xs[i], &y = *ys[i];
    TORCH_CHECK(x.scalar_type() == q.scalar_type() && y.scalar_type() == q.scalar_type() && x.get_device() == q.get_device() &&
                    y.is_cuda() && y.get_device() == q.get_device() && x.size(0) == T && x.size(2) == D && y.sizes() == x.sizes() &&
                    y.is_contiguous() && (x.stride(2) == 1 || D == 1),
                "rotary: q, k and their outputs have one type, device, token count and head width");
    wide = wide && (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0 &&
           (reinterpret_cast<uintptr_t>(y.data_ptr()) & 15) == 0 && x.stride(0) % W == 0 && x.stride(1) % W == 0;
    p.side[i] = RotarySide{x.data_ptr(), y.data_ptr(), x.stride(0), x.stride(1), (int)x.size(1)};
    heads += x.size(1);
  }
  if (heads == 0) return;
  TORCH_CHECK(heads * D < (1 << 24), "rotary: heads x width too large");
  p.positions = positions.data_ptr();
  p.pos64 = positions.scalar_type() == at::kLong;
  p.tokens = T;
  p.pos_len = positions.numel();
  p.dim = (int)D;
  p.rot = (int)R;
  p.factor = (float)factor;
  p.sin_factor = (float)(factor * sign);
  for (int64_t i = 0; i < turns.numel(); ++i) p.turns[i] = turns.data_ptr<double>()[i];
  const c10::cuda::CUDAGuard guard(q.device());
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // few tokens: one a block, so that the call is spread over the SMs; many: enough
  // of them that a block's threads have about four vectors each between two barriers
  const int64_t vectors = heads * std::max<int64_t>(1, D / (wide ? 2 * W : 2));
  const int64_t most = std::min<int64_t>(kRotMaxTile, (4 * kRotThreads + vectors - 1) / vectors);
  p.tile = (int)std::max<int64_t>(1, std::min<int64_t>(most, T / (8 * (int64_t)sms)));
  const int64_t tiles = (T + p.tile - 1) / p.tile;
  const unsigned grid = (unsigned)std::min<int64_t>(tiles, 8 * (int64_t)sms);
  auto stream = at::cuda::getCurrentCUDAStream();
  switch (q.scalar_type()) {
    case at::kBFloat16: launch_rotary<__nv_bfloat16>(p, wide, interleaved, grid, stream); break;
    case at::kHalf: launch_rotary<__half>(p, wide, interleaved, grid, stream); break;
    case at::kFloat: launch_rotary<float>(p, wide, interleaved, grid, stream); break;
    default: TORCH_CHECK(false, "rotary: bf16, fp16 or fp32");
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
