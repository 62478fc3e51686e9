// Activations kept in 8 bits for the backward pass: quantise and read back, and GELU and
// SwiGLU whose inputs are kept that way.
//
// Groups of 128 consecutive columns of a row (the last may be short), a = max |x| of one:
//   inv = 127 / a (one 32-bit division), code = nearest integer to x inv, ties to even (the
//   product is not rounded before), step = a (1/127) in 32 bits; read back as code * step.
// Codes are whole numbers of exact products, so they are the same on every device.
// The error is at most half a step, a / 254, of the group's largest.
//   gelu:   y = x Phi(x);            dx = dy (Phi(xq) + xq phi(xq))
//   swiglu: y = g sigma(g) u;        du = dy gq s,  dg = dy uq s (1 + gq (1 - s)),  s = sigma(gq)
//
// What bounds them: memory, but for GELU.  A warp takes 256 columns at a time (rows.cuh) and loads several
// such tiles before it works on the first.  Measured: 16384 x 5120 bf16 50 us to keep, 45 us to
// read back (0.77 and 0.85 of a copy's rate); SwiGLU of 8192 x 18944 213 us forward, 208 backward
// (0.89 and 0.91).  GELU is bound by its arithmetic: 8192 x 18944 210 us forward (0.57, at 0.85 of the
// issue slots), 234 backward (0.51, 0.76).
// Rows that are not whole 16-byte vectors go by single elements: 16384 x 5003 bf16 137 us to keep,
// 128 to read back, SwiGLU 355 and 332, GELU 263 and 256 (0.24 to 0.30).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>

#include "gelu.cuh"
#include "rows.cuh"
#include "swiglu.cuh"

namespace zq {

constexpr int kActWarps = 8;

// rows of the tensors of a launch, in elements (codes in bytes)
struct ActShape {
  int64_t M, D, tiles, P, G;   // tiles of a row
  uint32_t units;              // M * tiles
};

// The U units of a warp: unit u is tile u % tiles of row u / tiles.
struct ActUnit {
  int64_t row;
  int base;
};
template <int U>
__device__ __forceinline__ int act_units(const ActShape& s, ActUnit (&out)[U]) {
  const uint64_t first = ((uint64_t)blockIdx.x * kActWarps + (threadIdx.x >> 5)) * U;
  if (first >= s.units) {   // a warp behind the last unit: tiles past every row's end
#pragma unroll
    for (int j = 0; j < U; ++j) out[j].row = 0, out[j].base = (int)s.D;
    return 0;
  }
  uint32_t row = (uint32_t)first / (uint32_t)s.tiles, tile = (uint32_t)first - row * (uint32_t)s.tiles;
  const int n = (int)min((uint64_t)U, s.units - first);
#pragma unroll
  for (int j = 0; j < U; ++j) {
    out[j].row = row;
    out[j].base = j < n ? (int)tile * kTile : (int)s.D;
    if (++tile == (uint32_t)s.tiles) tile = 0, ++row;
  }
  return n;
}

template <bool VEC, int U>
__device__ __forceinline__ void keep_units(const uint64_t (&v)[U][4], const ActUnit (&u)[U], int8_t* codes, float* steps,
                                           int lane, const ActShape& s) {
  int8_t* c[U];
  float* t[U];
  int base[U];
#pragma unroll
  for (int j = 0; j < U; ++j) c[j] = codes + u[j].row * s.P, t[j] = steps + u[j].row * s.G, base[j] = u[j].base;
  keep_tiles<VEC, U>(v, c, t, base, lane, (int)s.D);
}

// fp32 activations take CUDA's accurate functions; 16-bit ones those of the kernels that
// keep their inputs as they are, so that the outputs are the same bits
template <typename T>
__device__ __forceinline__ GeluCP act_gelu(float x) {
  if constexpr (sizeof(T) == 4) return GeluCP{normcdff(x), expf(-0.5f * x * x) * 0.39894228040143268f};
  else return gelu_cdf_pdf(x);
}
template <typename T>
__device__ __forceinline__ float act_sigmoid(float x) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-x));
  else return swiglu_sigmoid(x);
}

template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kActWarps * 32) act8_keep_kernel(const T* __restrict__ x, int64_t xs,
                                                                   int8_t* __restrict__ codes, float* __restrict__ steps,
                                                                   const ActShape s) {
  const int lane = threadIdx.x & 31;
  ActUnit u[U];
  if (act_units<U>(s, u) == 0) return;
  RawTile<T, VEC> t[U];
#pragma unroll
  for (int j = 0; j < U; ++j)
    if (u[j].base < s.D) t[j].load(x + u[j].row * xs, u[j].base, lane, (int)s.D);
  uint64_t v[U][4];
#pragma unroll
  for (int j = 0; j < U; ++j) t[j].pairs(v[j]);
  keep_units<VEC, U>(v, u, codes, steps, lane, s);
}

template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kActWarps * 32) act8_read_kernel(const int8_t* __restrict__ codes,
                                                                   const float* __restrict__ steps, T* __restrict__ x,
                                                                   const ActShape s) {
  const int lane = threadIdx.x & 31;
  ActUnit u[U];
  const int n = act_units<U>(s, u);
  RawCodes<VEC> c[U];
#pragma unroll
  for (int j = 0; j < U; ++j)
    if (j < n) c[j].load(codes + u[j].row * s.P, steps + u[j].row * s.G, u[j].base, lane, (int)s.D);
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      float v[8];
      c[j].values(v);
      store_tile<T, VEC>(x + u[j].row * s.D, u[j].base, lane, (int)s.D, v);
    }
  }
}

template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kActWarps * 32) gelu8_fwd_kernel(const T* __restrict__ x, int64_t xs, T* __restrict__ y,
                                                                   int8_t* __restrict__ codes, float* __restrict__ steps,
                                                                   const ActShape s) {
  const int lane = threadIdx.x & 31;
  ActUnit u[U];
  const int n = act_units<U>(s, u);
  RawTile<T, VEC> t[U];
#pragma unroll
  for (int j = 0; j < U; ++j)
    if (j < n) t[j].load(x + u[j].row * xs, u[j].base, lane, (int)s.D);
  {
    uint64_t v[U][4];
#pragma unroll
    for (int j = 0; j < U; ++j) t[j].pairs(v[j]);
    keep_units<VEC, U>(v, u, codes, steps, lane, s);
  }
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      float v[8], o[8];
      t[j].values(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = v[i] * act_gelu<T>(v[i]).cdf;
      store_tile<T, VEC>(y + u[j].row * s.D, u[j].base, lane, (int)s.D, o);
    }
  }
}

template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kActWarps * 32) gelu8_bwd_kernel(const T* __restrict__ dy, int64_t ds,
                                                                   const int8_t* __restrict__ codes,
                                                                   const float* __restrict__ steps, T* __restrict__ dx,
                                                                   const ActShape s) {
  const int lane = threadIdx.x & 31;
  ActUnit u[U];
  const int n = act_units<U>(s, u);
  RawTile<T, VEC> t[U];
  RawCodes<VEC> c[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      t[j].load(dy + u[j].row * ds, u[j].base, lane, (int)s.D);
      c[j].load(codes + u[j].row * s.P, steps + u[j].row * s.G, u[j].base, lane, (int)s.D);
    }
  }
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      float d[8], v[8];
      t[j].values(d);
      c[j].values(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const GeluCP p = act_gelu<T>(v[i]);
        d[i] *= p.cdf + v[i] * p.pdf;
      }
      store_tile<T, VEC>(dx + u[j].row * s.D, u[j].base, lane, (int)s.D, d);
    }
  }
}

template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kActWarps * 32) swiglu8_fwd_kernel(const T* __restrict__ g, int64_t gs,
                                                                     const T* __restrict__ up, int64_t us,
                                                                     T* __restrict__ y, int8_t* __restrict__ gcodes,
                                                                     float* __restrict__ gsteps, int8_t* __restrict__ ucodes,
                                                                     float* __restrict__ usteps, const ActShape s) {
  const int lane = threadIdx.x & 31;
  ActUnit u[U];
  const int n = act_units<U>(s, u);
  RawTile<T, VEC> a[U], b[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      a[j].load(g + u[j].row * gs, u[j].base, lane, (int)s.D);
      b[j].load(up + u[j].row * us, u[j].base, lane, (int)s.D);
    }
  }
  {   // both inputs' tiles at once
    uint64_t v[2 * U][4];
    int8_t* c[2 * U];
    float* t[2 * U];
    int base[2 * U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      a[j].pairs(v[2 * j]);
      b[j].pairs(v[2 * j + 1]);
      c[2 * j] = gcodes + u[j].row * s.P, t[2 * j] = gsteps + u[j].row * s.G;
      c[2 * j + 1] = ucodes + u[j].row * s.P, t[2 * j + 1] = usteps + u[j].row * s.G;
      base[2 * j] = base[2 * j + 1] = u[j].base;
    }
    keep_tiles<VEC, 2 * U>(v, c, t, base, lane, (int)s.D);
  }
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      float v[8], w[8];
      a[j].values(v);
      b[j].values(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] *= v[i] * act_sigmoid<T>(v[i]);
      store_tile<T, VEC>(y + u[j].row * s.D, u[j].base, lane, (int)s.D, w);
    }
  }
}

template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kActWarps * 32) swiglu8_bwd_kernel(
    const T* __restrict__ dy, int64_t ds, const int8_t* __restrict__ gcodes, const float* __restrict__ gsteps,
    const int8_t* __restrict__ ucodes, const float* __restrict__ usteps, T* __restrict__ dg, T* __restrict__ du,
    const ActShape s) {
  const int lane = threadIdx.x & 31;
  ActUnit u[U];
  const int n = act_units<U>(s, u);
  RawTile<T, VEC> t[U];
  RawCodes<VEC> a[U], b[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      t[j].load(dy + u[j].row * ds, u[j].base, lane, (int)s.D);
      a[j].load(gcodes + u[j].row * s.P, gsteps + u[j].row * s.G, u[j].base, lane, (int)s.D);
      b[j].load(ucodes + u[j].row * s.P, usteps + u[j].row * s.G, u[j].base, lane, (int)s.D);
    }
  }
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (j < n) {
      float d[8], v[8], w[8];
      t[j].values(d);
      a[j].values(v);
      b[j].values(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = act_sigmoid<T>(v[i]);
        w[i] *= d[i] * q * (1.0f + v[i] * (1.0f - q));
        v[i] *= d[i] * q;
      }
      store_tile<T, VEC>(dg + u[j].row * s.D, u[j].base, lane, (int)s.D, w);
      store_tile<T, VEC>(du + u[j].row * s.D, u[j].base, lane, (int)s.D, v);
    }
  }
}

}  // namespace zq

using namespace zq;

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
namespace {

struct ActLaunch {
  ActShape s;
  bool vec;
  cudaStream_t stream;
};

bool aligned16(const at::Tensor& t, int64_t pitch) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 && (t.size(0) < 2 || pitch * t.element_size() % 16 == 0);
}

// [M, D] rows of unit stride
int64_t act_rows(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == like.get_device() && t.dim() == 2 && t.sizes() == like.sizes() &&
                  t.scalar_type() == like.scalar_type() && (t.stride(1) == 1 || t.size(1) == 1),
              name, ": [M, D] on one device, of one type and shape, unit column stride");
  return t.stride(0);
}

// shape of a launch over x's rows; `rows`: the dense tensors of that shape
ActLaunch act_launch(const at::Tensor& x, std::initializer_list<const at::Tensor*> rows,
                     std::initializer_list<const at::Tensor*> codes, std::initializer_list<const at::Tensor*> steps,
                     const char* name) {
  ActLaunch l;
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(0) > 0 && x.size(1) > 0, name, ": [M, D] on the GPU");
  l.s.M = x.size(0);
  l.s.D = x.size(1);
  TORCH_CHECK(l.s.D < (1LL << 30), name, ": rows of less than 2^30 columns");
  l.s.tiles = (l.s.D + kTile - 1) / kTile;
  l.s.P = (l.s.D + 15) / 16 * 16;
  l.s.G = (l.s.D + kGroup - 1) / kGroup;
  TORCH_CHECK(l.s.M * l.s.tiles < (1LL << 32), name, ": too many rows");
  l.s.units = (uint32_t)(l.s.M * l.s.tiles);
  l.vec = l.s.D % 8 == 0;
  for (const at::Tensor* t : rows) {
    const int64_t pitch = act_rows(*t, x, name);
    l.vec = l.vec && aligned16(*t, pitch);
  }
  for (const at::Tensor* t : codes) {
    TORCH_CHECK(t->is_cuda() && t->get_device() == x.get_device() && t->scalar_type() == at::kChar && t->is_contiguous() &&
                    t->dim() == 2 && t->size(0) == l.s.M && t->size(1) == l.s.P,
                name, ": codes int8 [M, D up to 16s]");
    TORCH_CHECK((reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0, name, ": codes on a 16-byte boundary");
  }
  for (const at::Tensor* t : steps)
    TORCH_CHECK(t->is_cuda() && t->get_device() == x.get_device() && t->scalar_type() == at::kFloat && t->is_contiguous() &&
                    t->dim() == 2 && t->size(0) == l.s.M && t->size(1) == l.s.G,
                name, ": steps fp32 [M, D / 128]");
  l.stream = at::cuda::getCurrentCUDAStream(x.get_device());
  return l;
}

unsigned act_grid(const ActLaunch& l, int U) {
  return (unsigned)(((int64_t)l.s.units + kActWarps * U - 1) / (kActWarps * U));
}

template <typename T>
T* ptr(const at::Tensor& t) {
  return reinterpret_cast<T*>(t.data_ptr());
}

}  // namespace

#define ZQ_ACT_TYPES(TENSOR, NAME, ...)                                                    \
  switch ((TENSOR).scalar_type()) {                                                        \
    case at::kBFloat16: { using T = __nv_bfloat16; __VA_ARGS__; break; }                   \
    case at::kHalf: { using T = __half; __VA_ARGS__; break; }                              \
    case at::kFloat: { using T = float; __VA_ARGS__; break; }                              \
    default: TORCH_CHECK(false, NAME, ": bf16, fp16 or fp32");                             \
  }
#define ZQ_ACT_LAUNCH(KERNEL, U, ...)                                                      \
  do {                                                                                     \
    if (l.vec) KERNEL<T, true, U><<<act_grid(l, U), kActWarps * 32, 0, l.stream>>>(__VA_ARGS__); \
    else KERNEL<T, false, U><<<act_grid(l, U), kActWarps * 32, 0, l.stream>>>(__VA_ARGS__);      \
    C10_CUDA_KERNEL_LAUNCH_CHECK();                                                        \
  } while (0)

void act8_keep(at::Tensor x, at::Tensor codes, at::Tensor steps) {
  const c10::cuda::CUDAGuard guard(x.device());
  const ActLaunch l = act_launch(x, {&x}, {&codes}, {&steps}, "quantize_activation");
  ZQ_ACT_TYPES(x, "quantize_activation",
               ZQ_ACT_LAUNCH(act8_keep_kernel, 4, ptr<T>(x), x.stride(0), codes.data_ptr<int8_t>(), steps.data_ptr<float>(), l.s));
}

void act8_read(at::Tensor codes, at::Tensor steps, at::Tensor x) {
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.is_contiguous(), "dequantize_activation: contiguous output");
  const ActLaunch l = act_launch(x, {&x}, {&codes}, {&steps}, "dequantize_activation");
  ZQ_ACT_TYPES(x, "dequantize_activation",
               ZQ_ACT_LAUNCH(act8_read_kernel, 4, codes.data_ptr<int8_t>(), steps.data_ptr<float>(), ptr<T>(x), l.s));
}

void gelu8_fwd(at::Tensor x, at::Tensor y, at::Tensor codes, at::Tensor steps) {
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(y.is_contiguous(), "gelu: contiguous output");
  const ActLaunch l = act_launch(x, {&x, &y}, {&codes}, {&steps}, "gelu");
  ZQ_ACT_TYPES(x, "gelu", ZQ_ACT_LAUNCH(gelu8_fwd_kernel, 4, ptr<T>(x), x.stride(0), ptr<T>(y), codes.data_ptr<int8_t>(),
                                        steps.data_ptr<float>(), l.s));
}

void gelu8_bwd(at::Tensor dy, at::Tensor codes, at::Tensor steps, at::Tensor dx) {
  const c10::cuda::CUDAGuard guard(dy.device());
  TORCH_CHECK(dx.is_contiguous(), "gelu: contiguous output");
  const ActLaunch l = act_launch(dy, {&dy, &dx}, {&codes}, {&steps}, "gelu");
  ZQ_ACT_TYPES(dy, "gelu", ZQ_ACT_LAUNCH(gelu8_bwd_kernel, 4, ptr<T>(dy), dy.stride(0), codes.data_ptr<int8_t>(),
                                         steps.data_ptr<float>(), ptr<T>(dx), l.s));
}

void swiglu8_fwd(at::Tensor g, at::Tensor u, at::Tensor y, at::Tensor gcodes, at::Tensor gsteps, at::Tensor ucodes,
                 at::Tensor usteps) {
  const c10::cuda::CUDAGuard guard(g.device());
  TORCH_CHECK(y.is_contiguous(), "swiglu: contiguous output");
  const ActLaunch l = act_launch(g, {&g, &u, &y}, {&gcodes, &ucodes}, {&gsteps, &usteps}, "swiglu");
  ZQ_ACT_TYPES(g, "swiglu", ZQ_ACT_LAUNCH(swiglu8_fwd_kernel, 2, ptr<T>(g), g.stride(0), ptr<T>(u), u.stride(0), ptr<T>(y),
                                          gcodes.data_ptr<int8_t>(), gsteps.data_ptr<float>(), ucodes.data_ptr<int8_t>(),
                                          usteps.data_ptr<float>(), l.s));
}

void swiglu8_bwd(at::Tensor dy, at::Tensor gcodes, at::Tensor gsteps, at::Tensor ucodes, at::Tensor usteps, at::Tensor dg,
                 at::Tensor du) {
  const c10::cuda::CUDAGuard guard(dy.device());
  TORCH_CHECK(dg.is_contiguous() && du.is_contiguous(), "swiglu: contiguous outputs");
  const ActLaunch l = act_launch(dy, {&dy, &dg, &du}, {&gcodes, &ucodes}, {&gsteps, &usteps}, "swiglu");
  ZQ_ACT_TYPES(dy, "swiglu", ZQ_ACT_LAUNCH(swiglu8_bwd_kernel, 2, ptr<T>(dy), dy.stride(0), gcodes.data_ptr<int8_t>(),
                                           gsteps.data_ptr<float>(), ucodes.data_ptr<int8_t>(), usteps.data_ptr<float>(),
                                           ptr<T>(dg), ptr<T>(du), l.s));
}
