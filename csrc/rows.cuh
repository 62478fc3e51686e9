// Tiles of a row: what the row-wise operators (8-bit activations, layer norm, embedding)
// share.
//
// A warp takes 256 columns of a row at a time, 8 a lane.  VEC: rows that start on a 16-byte
// boundary and have a multiple of 8 columns; a lane holds 8 consecutive ones (one 16-byte
// access, two in fp32).  Otherwise the lanes are interleaved (column 32 i + lane), so that
// an access of single elements still covers whole sectors.  Groups of 128 columns, which
// share a step in 8 bits, are half a warp's lanes or half of every lane's values.
#pragma once

#include "common.cuh"

namespace zq {

constexpr int kTile = 256;    // columns of a warp's tile
constexpr int kGroup = 128;   // columns of a step

template <bool VEC>
__device__ __forceinline__ int tile_col(int lane, int i) {
  return VEC ? lane * 8 + i : i * 32 + lane;
}

// A tile as it is loaded, so that several can be under way at once.
template <typename T, bool VEC>
struct RawTile {
  static constexpr int kWords = (int)sizeof(T) * 2;   // of 8 elements
  uint32_t w[kWords];

  // columns [base, base + 256) of a row of D; those past its end are 0
  __device__ __forceinline__ void load(const T* row, int base, int lane, int D) {
    if constexpr (VEC) {
      const int c = base + lane * 8;
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 u = c < D ? __ldg(reinterpret_cast<const uint4*>(row + c) + i) : make_uint4(0u, 0u, 0u, 0u);
        w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
      }
    } else {
      T* e = reinterpret_cast<T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = base + i * 32 + lane;
        e[i] = c < D ? row[c] : from_f32<T>(0.0f);
      }
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = bf16x2_to_f2(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  }
  // the same as packed pairs (2i, 2i + 1)
  __device__ __forceinline__ void pairs(uint64_t (&v)[4]) const {
    float f[8];
    values(f);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f2_pack(f[2 * i], f[2 * i + 1]);
  }
  __device__ __forceinline__ void set(const uint64_t (&v)[4]) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) f2_unpack(v[i], f[2 * i], f[2 * i + 1]);
    set(f);
  }
  // rounds to the type, once
  __device__ __forceinline__ void set(const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void store(T* row, int base, int lane, int D) const {
    if constexpr (VEC) {
      const int c = base + lane * 8;
      if (c < D) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i)
          reinterpret_cast<uint4*>(row + c)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      }
    } else {
      const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = base + i * 32 + lane;
        if (c < D) row[c] = e[i];
      }
    }
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void store_tile(T* row, int base, int lane, int D, const float (&v)[8]) {
  RawTile<T, VEC> t;
  t.set(v);
  t.store(row, base, lane, D);
}

// ---------------------------------------------------------------------------
// 8 bits: codes int8 [M, P] (P: D up to a multiple of 16), steps fp32 [M, ceil(D / 128)]
// ---------------------------------------------------------------------------
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where one is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Step and factor of a group from the largest size a of its elements.  Below 2^-119 the
// factor 127 / a leaves the range: the group reads back as 0.  A NaN or an infinity makes
// the whole group read back as NaN.
struct GroupScale {
  float step, inv;
};
__device__ __forceinline__ GroupScale group_scale(float a) {
  GroupScale g;
  const bool zero = a < 0x1p-119f, bad = !(a < INFINITY);
  g.inv = zero || bad ? 0.0f : __fdiv_rn(127.0f, a);
  g.step = bad ? __int_as_float(0x7fc00000) : zero ? 0.0f : __fmul_rn(a, 1.0f / 127.0f);
  return g;
}

// The nearest whole number to v * inv, ties to even, in the low byte: one fma onto a number
// whose last place is 1 (the product is not rounded before).
__device__ __forceinline__ uint32_t code_of(float v, float inv) {
  return __float_as_uint(__fmaf_rn(v, inv, 12582912.0f));
}

// Writes the codes and steps of K tiles of one warp: tile k holds columns [base[k], base[k] + 256)
// of row `codes[k]`, `steps[k]`; tiles with base[k] >= D are none.
template <bool VEC, int K>
__device__ __forceinline__ void keep_tiles(const uint64_t (&v)[K][4], int8_t* const (&codes)[K], float* const (&steps)[K],
                                           const int (&base)[K], int lane, int D) {
  const uint64_t magic = f2_pack(12582912.0f, 12582912.0f);
  if constexpr (VEC) {
    float a[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) f2_unpack(v[k][i], f[2 * i], f[2 * i + 1]);
      a[k] = max_nan(max_nan(max_nan(fabsf(f[0]), fabsf(f[1])), max_nan(fabsf(f[2]), fabsf(f[3]))),
                     max_nan(max_nan(fabsf(f[4]), fabsf(f[5])), max_nan(fabsf(f[6]), fabsf(f[7]))));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) a[k] = max_nan(a[k], __shfl_xor_sync(0xffffffffu, a[k], o));
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const GroupScale g = group_scale(a[k]);
      if ((lane & 15) == 0 && base[k] + lane * 8 < D) steps[k][(base[k] + lane * 8) / kGroup] = g.step;
      const float inv = g.inv;
      const uint64_t inv2 = f2_pack(inv, inv);
      uint32_t c[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float lo, hi;
        f2_unpack(f2_fma(v[k][i], inv2, magic), lo, hi);
        c[2 * i] = __float_as_uint(lo), c[2 * i + 1] = __float_as_uint(hi);
      }
      const int col = base[k] + lane * 8;
      if (col < D) {
        uint2 w;
        w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        w.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
        *reinterpret_cast<uint2*>(codes[k] + col) = w;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) f2_unpack(v[k][i], f[2 * i], f[2 * i + 1]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float a = max_nan(max_nan(fabsf(f[4 * h]), fabsf(f[4 * h + 1])), max_nan(fabsf(f[4 * h + 2]), fabsf(f[4 * h + 3])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        const GroupScale g = group_scale(a);
        const int first = base[k] + h * kGroup;
        if (lane == 0 && first < D) steps[k][first / kGroup] = g.step;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = first + i * 32 + lane;
          if (col < D) codes[k][col] = (int8_t)(code_of(f[4 * h + i], g.inv) & 0xffu);
        }
      }
    }
  }
}

// A tile of codes as it is loaded.
template <bool VEC>
struct RawCodes {
  uint2 w;
  float step[VEC ? 1 : 2];
  __device__ __forceinline__ void load(const int8_t* codes, const float* steps, int base, int lane, int D) {
    if constexpr (VEC) {
      const int at = base + lane * 8;
      w = at < D ? __ldg(reinterpret_cast<const uint2*>(codes + at)) : make_uint2(0u, 0u);
      step[0] = at < D ? __ldg(steps + at / kGroup) : 0.0f;
    } else {
      uint8_t* b = reinterpret_cast<uint8_t*>(&w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = base + i * 32 + lane;
        b[i] = at < D ? (uint8_t)codes[at] : (uint8_t)0;
      }
      step[0] = base < D ? steps[base / kGroup] : 0.0f;
      step[1] = base + kGroup < D ? steps[base / kGroup + 1] : 0.0f;
    }
  }
  // code * step, rounded once in 32 bits.  (A byte plus 128 in the last places of 2^23: the
  // conversion instruction runs at an eighth of the rate.)
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = __uint_as_float(__byte_perm(i < 4 ? x : y, 0x4b000000u, 0x7540u + (i & 3)));
      v[i] = __fmul_rn(__fadd_rn(f, -8388736.0f), step[VEC ? 0 : i / 4]);
    }
  }
  // code * step - mu, rounded once, in packed pairs
  __device__ __forceinline__ void away(float mu, uint64_t (&v)[4]) const {
    const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u;
    const uint64_t back = f2_pack(-8388736.0f, -8388736.0f), mu2 = f2_pack(-mu, -mu);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t s = i < 2 ? x : y;
      const float lo = __uint_as_float(__byte_perm(s, 0x4b000000u, 0x7540u + (2 * i & 3)));
      const float hi = __uint_as_float(__byte_perm(s, 0x4b000000u, 0x7540u + ((2 * i + 1) & 3)));
      const float t = step[VEC ? 0 : i / 2];
      v[i] = f2_fma(f2_add(f2_pack(lo, hi), back), f2_pack(t, t), mu2);
    }
  }
};

}  // namespace zq
