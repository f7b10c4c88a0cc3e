// Device helpers of the products with 4-bit weights: conversion, matrix instruction, the outputs' last step.
#pragma once

#include "mx4_internal.h"

namespace t2w {

namespace {

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// eight codes (columns 0 .. 7, the lowest nibble first) times the scale, as the matrix unit's operand
template <bool BF>
__device__ __forceinline__ uint4 widen(uint32_t c, float scale) {
  if constexpr (BF)
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3)));
  else
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3)));
}

template <bool BF>
__device__ __forceinline__ f32x4 mma(uint4 a, uint4 b, f32x4 c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// the float 2^(byte i of w - 127)
__device__ __forceinline__ float scale_of(uint32_t w, int i) { return __uint_as_float(((w >> (8 * i)) & 0xffu) << 23); }

template <bool BF>
__device__ __forceinline__ float load1(const void* p, long long i) {
  const uint16_t h = ((const uint16_t*)p)[i];
  return BF ? bf2f(h) : h2f(h);
}
template <bool BF>
__device__ __forceinline__ uint16_t round1(float v) {
  return BF ? f2bf(v) : f2h(v);
}

__device__ __forceinline__ float gate_act(float g, int act) { return act == T2W_MX4_SILU ? silu(g) : gelu_tanh(g); }

// What outputs n .. n + 3 of row m need besides their sums, as loaded: ahead of the stores (the compiler may not move a load
// across them, as the residual may be y itself), so that an epilogue waits for memory once and not for every block.  Places
// behind the last read the last.
struct Extra {
  float bias[4];
  uint32_t res[4];  // quad: two words, else four values
};

template <bool BF>
__device__ __forceinline__ Extra fetch(const Mx4Args& a, int m, int n) {
  Extra x = {{0.f, 0.f, 0.f, 0.f}, {0, 0, 0, 0}};
  const uint16_t* res = (const uint16_t*)a.residual + (long long)min(m, a.m - 1) * a.ldr;
  if (a.quad) {
    const int c = min(n, a.n - 4);
    if (a.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x.bias[e] = a.bias[c + e];
    }
    if (a.residual) {
      const uint2 h = *(const uint2*)(res + c);
      x.res[0] = h.x, x.res[1] = h.y;
    }
    return x;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = min(n + e, a.n - 1);
    if (a.bias) x.bias[e] = a.bias[c];
    if (a.residual) x.res[e] = res[c];
  }
  return x;
}

// Outputs n .. n + 3 of row m from their sums
template <bool BF>
__device__ __forceinline__ void finish(const Mx4Args& a, int m, int n, const float (&v)[4], const Extra& x) {
  if (m >= a.m || n >= a.n) return;
  uint16_t* y = (uint16_t*)a.y + (long long)m * a.ldy + n;
  float r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = v[e] + x.bias[e];
  if (a.quad) {
    r[0] += BF ? lo2f(x.res[0]) : lo2h(x.res[0]);
    r[1] += BF ? hi2f(x.res[0]) : hi2h(x.res[0]);
    r[2] += BF ? lo2f(x.res[1]) : lo2h(x.res[1]);
    r[3] += BF ? hi2f(x.res[1]) : hi2h(x.res[1]);
    *(uint2*)y = BF ? make_uint2(pack2(r[0], r[1]), pack2(r[2], r[3])) : make_uint2(pack2h(r[0], r[1]), pack2h(r[2], r[3]));
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.n) y[e] = round1<BF>(r[e] + (BF ? lo2f(x.res[e]) : lo2h(x.res[e])));
}

}  // namespace

}  // namespace t2w
