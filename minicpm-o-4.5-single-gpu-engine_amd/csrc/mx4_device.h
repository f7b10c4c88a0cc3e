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
  uint2 res;  // the residual's four values
};

// of N places (row of x, first channel); the branches, the same for all, stand outside.  Two wide rows share an output's.
template <Form F, int N>
__device__ __forceinline__ void fetch(const Mx4Args& a, const int2 (&at)[N], Extra (&x)[N]) {
  constexpr int S = F == Form::WIDE ? 1 : 0;
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = Extra{};
  const uint16_t* res = (const uint16_t*)a.residual;
  if (a.quad) {
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j].bias[e] = a.bias[min(at[j].y, a.n - 4) + e];
    }
    if (a.residual) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        x[j].res = *(const uint2*)(res + (long long)(min(at[j].x, a.m - 1) >> S) * a.ldr + min(at[j].y, a.n - 4));
    }
    return;
  }
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j].bias[e] = a.bias[min(at[j].y + e, a.n - 1)];
  }
  if (a.residual) {
    uint32_t r[N][4];
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) r[j][e] = res[(long long)(min(at[j].x, a.m - 1) >> S) * a.ldr + min(at[j].y + e, a.n - 1)];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j].res = make_uint2(r[j][0] | r[j][1] << 16, r[j][2] | r[j][3] << 16);
  }
}

// r[0 .. 3] at channels n .. n + 3 of a row
template <bool BF>
__device__ __forceinline__ void put(const Mx4Args& a, uint16_t* y, int n, const float (&r)[4]) {
  if (a.quad) {
    *(uint2*)y = BF ? make_uint2(pack2(r[0], r[1]), pack2(r[2], r[3])) : make_uint2(pack2h(r[0], r[1]), pack2h(r[2], r[3]));
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.n) y[e] = round1<BF>(r[e]);
}

template <bool BF>
__device__ __forceinline__ void add(float (&v)[4], const Extra& x) {
  const float h[4] = {BF ? lo2f(x.res.x) : lo2h(x.res.x), BF ? hi2f(x.res.x) : hi2h(x.res.x), BF ? lo2f(x.res.y) : lo2h(x.res.y), BF ? hi2f(x.res.y) : hi2h(x.res.y)};
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = v[e] + x.bias[e] + h[e];
}

// Outputs n .. n + 3 of row m from their sums
template <bool BF, bool GATED, Form F>
__device__ __forceinline__ void finish(const Mx4Args& a, int m, int n, float (&v)[4], const Extra& x) {
  if (m >= a.m || n >= a.n) return;
  if constexpr (F == Form::PLAIN) {
    if constexpr (!GATED) add<BF>(v, x);
    put<BF>(a, (uint16_t*)a.y + (long long)m * a.ldy + n, n, v);
  } else if constexpr (GATED) {
    // The nearest bf16 of a value held within bf16's largest, and the rest: of an infinite value the rest is infinite, so that it
    // meets codes of zero as an infinity does.
    float lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float top = __uint_as_float(0x7f7f0000u);
      const float hi = bf2f(f2bf(__builtin_amdgcn_fmed3f(v[e], -top, top)));
      lo[e] = v[e] - hi, v[e] = hi;
    }
    uint16_t* y = (uint16_t*)a.y + 2LL * m * a.ldy + n;
    put<true>(a, y, n, v);
    put<true>(a, y + a.ldy, n, lo);
  } else {
    // rows 2 r and 2 r + 1 are neighbouring lanes, inside a.m together
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v[e]), 0xB1, 0xF, 0xF, false));  // quad_perm 1,0,3,2
    if (m & 1) return;
    uint16_t* y = (uint16_t*)a.y + (long long)(m >> 1) * a.ldy + n;
    if (a.half) {
      add<false>(v, x);
      put<false>(a, y, n, v);
    } else {
      add<true>(v, x);
      put<true>(a, y, n, v);
    }
  }
}

}  // namespace

}  // namespace t2w
