// Device helpers shared by the attention kernels.
#pragma once

#include "common.cuh"

namespace zq {

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x for a pair, x <= 64, by range reduction x = j + f, f in [-1/2, 1/2], and a
// degree-3 polynomial (a relative-error least-squares fit on 4000 Chebyshev nodes
// of [-1/2, 1/2]; max relative error 7.8e-5 in fp32); x below -120 is clamped
// there (2^-120 ~ 7.5e-37 instead of 0).
__device__ __forceinline__ void exp2_poly3_x2(float a0, float a1, float& p0, float& p1) {
  const uint64_t x = f2_pack(fmaxf(a0, -120.0f), fmaxf(a1, -120.0f));
  const uint64_t magic = f2_pack(12582912.0f, 12582912.0f);   // 1.5 * 2^23
  const uint64_t t = f2_add(x, magic);        // round(x) in the low mantissa bits
  const uint64_t f = f2_sub(x, f2_sub(t, magic));   // [-1/2, 1/2]
  uint64_t p = f2_fma(f2_pack(0.05508868396282196f, 0.05508868396282196f), f,
                      f2_pack(0.24260404706001282f, 0.24260404706001282f));
  p = f2_fma(p, f, f2_pack(0.6932762265205383f, 0.6932762265205383f));
  p = f2_fma(p, f, f2_pack(0.9999289512634277f, 0.9999289512634277f));
  float q0, q1, t0, t1;
  f2_unpack(p, q0, q1);
  f2_unpack(t, t0, t1);
  // the bits of t are (0x4B400000 + round(x)); shifted by 23 only round(x) << 23 remains
  p0 = __int_as_float(__float_as_int(q0) + (__float_as_int(t0) << 23));
  p1 = __int_as_float(__float_as_int(q1) + (__float_as_int(t1) << 23));
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// 64 consecutive columns of one TMEM row (this thread's lane) -> registers
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  tmem_ld_32x32b_x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
  tmem_ld_32x32b_x32(taddr + 32u, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
}

// one 128-byte row of a 128-byte-swizzled smem atom (64 bf16) -> 32 TMEM columns
__device__ __forceinline__ void copy_row_to_tmem(const uint8_t* atom_row, int row, uint32_t taddr) {
  uint32_t v[32];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint4 u = *reinterpret_cast<const uint4*>(atom_row + ((c ^ (row & 7)) << 4));
    v[4 * c + 0] = u.x;
    v[4 * c + 1] = u.y;
    v[4 * c + 2] = u.z;
    v[4 * c + 3] = u.w;
  }
  tmem_st_32x32b_x32(taddr, v);
}

}  // namespace zq
