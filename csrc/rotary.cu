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
// turns.  turns travels in the kernel's parameters: no table in global memory to
// keep or to fill.
//
// A thread owns one 16-byte column of one token (two of them, one in each half, in
// the half layout): it evaluates its pairs' angles once, keeps them in registers and
// walks over the heads, so there is no shared memory and no barrier, and the
// evaluations are R/2 per token for (Hq + Hk) · D elements.  Bound by memory: 65537
// tokens x 18 heads x 128 (64 rotary columns, interleaved, fp16) take 102.5 us, 5.9 TB/s,
// 0.90 of a copy; with the angles in shared memory and blocks of a few tokens it was
// 153 us.  With few tokens the heads are divided over the grid's second axis.  Rows that
// are not 16-byte aligned, or whose widths are not whole vectors, take the element-wise
// form of the same code.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cstring>

#include "common.cuh"

namespace zq {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 128;   // rotary width up to 256

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
  int dim, rot, heads_per_block, pos64;
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

// U heads of one side at once: loads, then turns, then stores.
// VEC elements per access: 16 bytes (WIDE), or 1 (half layout) / 2 (interleaved).
template <typename T, int VEC, bool WIDE, bool INTER, int U>
__device__ __forceinline__ void rot_heads(const T* x, T* y, int64_t head_stride, int dim, int half, const float* c,
                                          const float* s) {
  float a[U][VEC], b[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    rot_load<T, VEC, WIDE>(x + u * head_stride, a[u]);
    if constexpr (!INTER) rot_load<T, VEC, WIDE>(x + u * head_stride + half, b[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float lo[VEC], hi[VEC];
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        lo[2 * i] = rope_lo(a[u][2 * i], a[u][2 * i + 1], c[i], s[i]);
        lo[2 * i + 1] = rope_hi(a[u][2 * i], a[u][2 * i + 1], c[i], s[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        lo[i] = rope_lo(a[u][i], b[u][i], c[i], s[i]);
        hi[i] = rope_hi(a[u][i], b[u][i], c[i], s[i]);
      }
      rot_store<T, VEC, WIDE>(y + (int64_t)u * dim + half, hi);
    }
    rot_store<T, VEC, WIDE>(y + (int64_t)u * dim, lo);
  }
}

template <typename T, int VEC, bool WIDE, bool INTER>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int PAIRS = INTER ? VEC / 2 : VEC;       // pairs of one thread
  constexpr int PASS = (INTER && !WIDE) ? 1 : VEC;   // widths past R need not be whole pairs
  const int half = p.rot / 2;
  const int turn_items = half / PAIRS;
  const int items = turn_items + (p.dim - p.rot) / PASS;
  // threads of one kind together: first all tokens' pairs, then all tokens' other columns
  const int64_t n = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  const bool turns = n < p.tokens * turn_items;
  const int kind = turns ? turn_items : items - turn_items;
  const int64_t left = turns ? n : n - p.tokens * turn_items;
  if (left >= p.tokens * kind) return;
  const int64_t tok = left / kind;
  const int it = (int)(left - tok * kind);
  float c[PAIRS], s[PAIRS];
  if (turns) {
    const int64_t at = p.pos_len == p.tokens ? tok : tok % p.pos_len;
    const int64_t pos = p.pos64 ? reinterpret_cast<const int64_t*>(p.positions)[at]
                                : (int64_t)reinterpret_cast<const int32_t*>(p.positions)[at];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const double turn = (double)pos * p.turns[it * PAIRS + i];
      sincospif(2.0f * (float)(turn - rint(turn)), &s[i], &c[i]);
      c[i] *= p.factor;
      s[i] *= p.sin_factor;
    }
  }
  const int col = turns ? it * (INTER ? VEC : PAIRS) : p.rot + it * PASS;
  // this block's heads [h0, h1) of both sides in a row
  const int heads = p.side[0].heads + p.side[1].heads;
  const int h0 = blockIdx.y * p.heads_per_block, h1 = min(heads, h0 + p.heads_per_block);
#pragma unroll
  for (int sd = 0; sd < 2; ++sd) {
    const RotarySide& side = p.side[sd];
    const int first = sd == 0 ? 0 : p.side[0].heads;
    int h = max(h0 - first, 0);
    const int end = min(h1 - first, side.heads);
    if (h >= end) continue;
    const T* x = reinterpret_cast<const T*>(side.x) + tok * side.token_stride + h * side.head_stride + col;
    T* y = reinterpret_cast<T*>(side.y) + (tok * side.heads + h) * (int64_t)p.dim + col;
    if (turns) {
      constexpr int U = 4;
      for (; h + U <= end; h += U) {
        rot_heads<T, VEC, WIDE, INTER, U>(x, y, side.head_stride, p.dim, half, c, s);
        x += U * side.head_stride;
        y += U * (int64_t)p.dim;
      }
      for (; h < end; ++h) {
        rot_heads<T, VEC, WIDE, INTER, 1>(x, y, side.head_stride, p.dim, half, c, s);
        x += side.head_stride;
        y += p.dim;
      }
    } else {   // columns past the rotary width
      constexpr int U = 4;
      for (; h < end; h += U) {
        const int m = min(U, end - h);
        if constexpr (WIDE) {
          uint4 v[U];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (u < m) v[u] = *reinterpret_cast<const uint4*>(x + u * side.head_stride);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (u < m) *reinterpret_cast<uint4*>(y + u * (int64_t)p.dim) = v[u];
        } else {
          for (int u = 0; u < m; ++u)
            for (int i = 0; i < PASS; ++i) y[u * (int64_t)p.dim + i] = x[u * side.head_stride + i];
        }
        x += U * side.head_stride;
        y += U * (int64_t)p.dim;
      }
    }
  }
}

template <typename T>
static void launch_rotary(RotaryParams& p, bool wide, bool inter, int sms, cudaStream_t stream) {
  constexpr int W = 16 / (int)sizeof(T);
  const int vec = wide ? W : inter ? 2 : 1, pairs = inter ? vec / 2 : vec, pass = inter && !wide ? 1 : vec;
  const int64_t items = p.rot / 2 / pairs + (p.dim - p.rot) / pass;
  const int64_t blocks = (p.tokens * items + kRotThreads - 1) / kRotThreads;
  const int heads = p.side[0].heads + p.side[1].heads;
  // all heads in one thread where the tokens alone fill the SMs (eight blocks each);
  // otherwise the heads are divided until they do, down to four (the angles are
  // evaluated once for each part), or to one where that still leaves SMs idle
  const int64_t least = blocks * ((heads + 3) / 4) < sms ? 1 : 4;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>((heads + least - 1) / least, 8 * sms / blocks));
  p.heads_per_block = (int)((heads + parts - 1) / parts);
  const dim3 grid((unsigned)blocks, (unsigned)((heads + p.heads_per_block - 1) / p.heads_per_block));
  auto kern = wide ? (inter ? rotary_kernel<T, W, true, true> : rotary_kernel<T, W, true, false>)
                   : (inter ? rotary_kernel<T, 2, false, true> : rotary_kernel<T, 1, false, false>);
  kern<<<grid, kRotThreads, 0, stream>>>(p);
}

}  // namespace zq

using namespace zq;

// q [T, Hq, D] and (optional) k [T, Hk, D], unit stride inside a head; qo, ko
// contiguous; positions int32 / int64 (1-D); turns: `pairs` 64-bit turns per
// position, on the host; factor scales cos and sin, sign = -1 turns back.
void rotary_turns(const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& positions, const void* turns,
                  int64_t pairs, const at::Tensor& qo, const c10::optional<at::Tensor>& ko, bool interleaved, double factor,
                  double sign) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && (!k.has_value() || (k->is_cuda() && k->dim() == 3 && ko.has_value())),
              "rotary: q and k are [T, H, D] CUDA tensors");
  TORCH_CHECK(pairs >= 1 && pairs <= kRotMaxPairs && 2 * pairs <= q.size(2),
              "rotary: turns must be 1 to ", kRotMaxPairs, " values, two columns of the head each");
  TORCH_CHECK(positions.is_cuda() && positions.get_device() == q.get_device() && positions.is_contiguous() &&
                  (positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt),
              "rotary: positions must be contiguous int32 or int64 on q's device");
  const int64_t T = q.size(0), D = q.size(2);
  if (T == 0) return;
  TORCH_CHECK(positions.numel() > 0 && T % positions.numel() == 0, "rotary: one position per token");
  RotaryParams p;
  const int64_t esize = q.element_size();
  const int64_t W = 16 / esize, R = 2 * pairs;
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
  TORCH_CHECK(heads < 65536 && T * D < (1LL << 38), "rotary: too many rows or heads");
  p.positions = positions.data_ptr();
  p.pos64 = positions.scalar_type() == at::kLong;
  p.tokens = T;
  p.pos_len = positions.numel();
  p.dim = (int)D;
  p.rot = (int)R;
  p.factor = (float)factor;
  p.sin_factor = (float)(factor * sign);
  std::memcpy(p.turns, turns, (size_t)pairs * sizeof(double));
  const c10::cuda::CUDAGuard guard(q.device());
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  auto stream = at::cuda::getCurrentCUDAStream();
  switch (q.scalar_type()) {
    case at::kBFloat16: launch_rotary<__nv_bfloat16>(p, wide, interleaved, sms, stream); break;
    case at::kHalf: launch_rotary<__half>(p, wide, interleaved, sms, stream); break;
    case at::kFloat: launch_rotary<float>(p, wide, interleaved, sms, stream); break;
    default: TORCH_CHECK(false, "rotary: bf16, fp16 or fp32");
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// the same with the turns as an fp64 CPU tensor [R/2]
void rotary(at::Tensor q, c10::optional<at::Tensor> k, at::Tensor positions, at::Tensor turns, at::Tensor qo,
            c10::optional<at::Tensor> ko, bool interleaved, double factor, double sign) {
  TORCH_CHECK(turns.device().is_cpu() && turns.scalar_type() == at::kDouble && turns.is_contiguous(),
              "rotary: turns must be fp64 values on the CPU");
  rotary_turns(q, k, positions, turns.data_ptr(), turns.numel(), qo, ko, interleaved, factor, sign);
}
