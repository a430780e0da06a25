// Softmax building blocks of the attention kernels on tcgen05: special functions, pairs of floats, rows of scores in tensor memory.
#pragma once
#include "tcgen05.cuh"

#define FT_LOG2E 1.4426950408889634f

__device__ __forceinline__ float ft_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(x) = 1 - 2 / (1 + 2^(2 x log2 e)): two special-function instructions, absolute error of a few 1e-7, exact limits
__device__ __forceinline__ float ft_tanh(float x) {
  float t = ft_ex2(x * (2.0f * FT_LOG2E)), r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + t));
  return fmaf(-2.0f, r, 1.0f);
}
// A raw score s (the product's sum, before the scale) capped in place: the softmax below multiplies by the scale, so the
// capped score is handed on as (cap / scale) * tanh(s * scale / cap).
__device__ __forceinline__ uint32_t ft_cap(uint32_t s, float cap_out, float cap_in) {
  return __float_as_uint(cap_out * ft_tanh(__uint_as_float(s) * cap_in));
}
// the first n of 32 output elements (n a multiple of 8) times the sigmoid of their gate logits (16-byte aligned)
__device__ __forceinline__ void ft_gate(uint32_t (&v)[32], const bf16* g, int n) {
#pragma unroll
  for (int c = 0; c < 4; c++) {
    if (8 * c >= n) break;
    const uint4 w = *(const uint4*)(g + 8 * c);
    const bf16* e = (const bf16*)&w;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float s;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + ft_ex2(-FT_LOG2E * __bfloat162float(e[i]))));
      v[8 * c + i] = __float_as_uint(__uint_as_float(v[8 * c + i]) * s);
    }
  }
}
__device__ __forceinline__ float ft_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// two floats at once: d = a * b + c and d = a + b on pairs held in 64-bit registers
__device__ __forceinline__ uint64_t ft_pack2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void ft_unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t ft_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t ft_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// two floats as the packed upper halves of their bits, and what that leaves of them (exactly): bfloat16 parts by truncation
__device__ __forceinline__ uint32_t ft_cut_pair(float& u, float& v) {
  const uint32_t a = __float_as_uint(u), b = __float_as_uint(v);
  u -= __uint_as_float(a & 0xffff0000u);
  v -= __uint_as_float(b & 0xffff0000u);
  return __byte_perm(a, b, 0x7632);
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]: A's row m in lane m, two bfloat16 of K per 32-bit column
__device__ __forceinline__ void umma_bf16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}

// maximum of a row's 64 scores, four chains of three-input maxima
__device__ __forceinline__ float ft_rowmax(const uint32_t (&s)[64]) {
  float m[4];
#pragma unroll
  for (int c = 0; c < 4; c++) m[c] = ft_max3(__uint_as_float(s[16 * c]), __uint_as_float(s[16 * c + 1]), __uint_as_float(s[16 * c + 2]));
#pragma unroll
  for (int i = 3; i < 15; i += 2)
#pragma unroll
    for (int c = 0; c < 4; c++) m[c] = ft_max3(m[c], __uint_as_float(s[16 * c + i]), __uint_as_float(s[16 * c + i + 1]));
#pragma unroll
  for (int c = 0; c < 4; c++) m[c] = fmaxf(m[c], __uint_as_float(s[16 * c + 15]));
  return fmaxf(ft_max3(m[0], m[1], m[2]), m[3]);
}
__device__ __forceinline__ void ft_ld64(uint32_t taddr, uint32_t (&s)[64]) {
  tmem_ld32(taddr, *(uint32_t(*)[32])&s[0]);
  tmem_ld32(taddr + 32, *(uint32_t(*)[32])&s[32]);
}
