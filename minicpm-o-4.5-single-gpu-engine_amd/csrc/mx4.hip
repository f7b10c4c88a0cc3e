// Operators on 4-bit weights (e2m1 codes, a power-of-two scale for every 32 columns): laying a matrix out, quantizing one, and
// the products with few rows.
//
// y = x W^T: a code times its scale is exact in bf16 and in fp16, so the matrix unit's products are exact and the sums fp32: the
// only roundings are the fp32 additions' and the output's.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "mx4_device.h"

namespace t2w {

namespace {

// --- few rows --------------------------------------------------------------------------------------------------------
// A workgroup owns RB blocks of 16 channels (GATED: the same block of both matrices) and 16 CB rows of x; its waves take the units
// of 512 columns in turn, each converting its codes in registers, and their sums meet in LDS in the order of the waves.
template <bool BF, int CB, int RB, bool GATED>
__global__ __launch_bounds__(1024) void mx4_rows_kernel(const Mx4Args a) {
  extern __shared__ float4 part[];  // [waves][RB][CB][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int steps = (a.k + 127) >> 7, units = (a.k + 511) >> 9, q = lane >> 4;
  const int nb = (a.n + 15) >> 4;
  f32x4 acc[RB][CB];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int c = 0; c < CB; ++c) acc[r][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint4* w[RB];
  const uint32_t* s[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int b = GATED ? (int)blockIdx.x : min((int)blockIdx.x * RB + r, nb - 1);
    w[r] = (const uint4*)a.w[GATED ? r : 0] + (size_t)b * steps * 64 + lane;
    s[r] = (const uint32_t*)a.s[GATED ? r : 0] + (size_t)b * units * 64 + lane;
  }
  const uint16_t* x[CB];
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    const int m = min((int)blockIdx.y * 16 * CB + 16 * c + (lane & 15), a.m - 1);  // rows behind the last repeat it: not stored
    x[c] = (const uint16_t*)a.x + (long long)m * a.ldx + 32 * q;
  }
  for (int u = wave; u < units; u += waves) {
    const int n_steps = min(4, steps - 4 * u);
    uint32_t sc[RB];
    uint4 code[RB][4];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      sc[r] = s[r][(size_t)u * 64];
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (t < n_steps) code[r][t] = w[r][(size_t)(4 * u + t) * 64];
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t >= n_steps) break;
      const int k0 = 512 * u + 128 * t;
      uint4 xf[CB][4];
      const bool whole = k0 + 128 <= a.k;
#pragma unroll
      for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          xf[c][j] = make_uint4(0, 0, 0, 0);
          if (whole || k0 + 32 * q + 8 * j < a.k) xf[c][j] = *(const uint4*)(x[c] + k0 + 8 * j);
        }
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float f = scale_of(sc[r], t);
        const uint32_t cw[4] = {code[r][t].x, code[r][t].y, code[r][t].z, code[r][t].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 wf = widen<BF>(cw[j], f);
#pragma unroll
          for (int c = 0; c < CB; ++c) acc[r][c] = mma<BF>(wf, xf[c][j], acc[r][c]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int c = 0; c < CB; ++c) part[((wave * RB + r) * CB + c) * 64 + lane] = __builtin_bit_cast(float4, acc[r][c]);
  __syncthreads();
  constexpr int TILES = GATED ? CB : RB * CB;
  for (int t = wave; t < TILES; t += waves) {
    float v[GATED ? 2 : 1][4];
#pragma unroll
    for (int g = 0; g < (GATED ? 2 : 1); ++g) {
      const int at = GATED ? g * CB + t : t;
      float4 p = part[at * 64 + lane];
      for (int i = 1; i < waves; ++i) {
        const float4 o = part[(i * RB * CB + at) * 64 + lane];
        p.x += o.x, p.y += o.y, p.z += o.z, p.w += o.w;
      }
      v[g][0] = p.x, v[g][1] = p.y, v[g][2] = p.z, v[g][3] = p.w;
    }
    const int c = GATED ? t : t % CB, r = GATED ? 0 : t / CB;
    const int n = ((int)blockIdx.x * (GATED ? 1 : RB) + r) * 16 + 4 * q, m = (int)blockIdx.y * 16 * CB + 16 * c + (lane & 15);
    if (m >= a.m || n >= a.n) continue;
    if constexpr (GATED) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] = gate_act(v[0][e], a.act) * v[1][e];
    }
    finish<BF>(a, m, n, v[0]);
  }
}

template <bool BF, int CB, int RB, bool GATED>
hipError_t launch_rows(const Mx4Args& a, hipStream_t st) {
  constexpr int MOST = RB * CB > 4 ? 8 : 16;  // 64 KB of sums
  const int units = mx4_units(a.k), rounds = (units + MOST - 1) / MOST, waves = (units + rounds - 1) / rounds;
  const int nb = mx4_blocks(a.n);
  const dim3 grid(GATED ? nb : (nb + RB - 1) / RB, (a.m + 16 * CB - 1) / (16 * CB));
  mx4_rows_kernel<BF, CB, RB, GATED><<<grid, waves * 64, (size_t)waves * RB * CB * 1024, st>>>(a);
  return hipGetLastError();
}

// --- layout ----------------------------------------------------------------------------------------------------------
// status bits: 1 a scale outside 2^MX4_EMIN .. 2^MX4_EMAX on a group that is not zero, 2 a weight that is not finite or too large

// A thread per lane and step: 32 columns of a channel
__global__ void mx4_pack_kernel(const uint32_t* codes, const uint8_t* scales, int n, int k, uint4* w, uint8_t* s, int* status) {
  const int steps = (k + 127) >> 7, units = (k + 511) >> 9, groups = (k + 31) >> 5;
  const size_t total = (size_t)((n + 15) >> 4) * units * 256;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
    const int lane = (int)(i & 63), t = (int)(i >> 6) & 3;
    const size_t bu = i >> 8;
    const int u = (int)(bu % units), b = (int)(bu / units), step = 4 * u + t;
    const int ch = 16 * b + (lane & 15), g = 4 * step + (lane >> 4);
    uint32_t c[4] = {0, 0, 0, 0};
    int e = 127;
    if (ch < n && g < groups) {
      const size_t row = (size_t)ch * (k >> 3);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * g + j < (k >> 3)) c[j] = codes[row + 4 * g + j];
      if ((c[0] | c[1] | c[2] | c[3]) & 0x77777777u) {
        e = scales[(size_t)ch * groups + g];
        if (e < 127 + MX4_EMIN || e > 127 + MX4_EMAX) atomicOr(status, 1);
      }
    }
    if (step < steps) w[((size_t)b * steps + step) * 64 + lane] = make_uint4(c[0], c[1], c[2], c[3]);
    s[(bu * 64 + lane) * 4 + t] = (uint8_t)e;
  }
}

// The same from 16- or 32-bit weights: a group's scale is the smallest power of two, at least 2^MX4_EMIN, that keeps its largest
// magnitude within 6; codes are rounded to nearest, ties to even.
template <int DT>
__global__ void mx4_quantize_kernel(const void* src, long long ld, int n, int k, uint4* w, uint8_t* s, int* status) {
  const int steps = (k + 127) >> 7, units = (k + 511) >> 9;
  const size_t total = (size_t)((n + 15) >> 4) * units * 256;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
    const int lane = (int)(i & 63), t = (int)(i >> 6) & 3;
    const size_t bu = i >> 8;
    const int u = (int)(bu % units), b = (int)(bu / units), step = 4 * u + t;
    const int ch = 16 * b + (lane & 15), col = 128 * step + 32 * (lane >> 4);
    float v[32];
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = 0.f;
      if (ch < n && col + j < k) {
        const long long at = (long long)ch * ld + col + j;
        v[j] = DT == T2W_MX4_FP32 ? ((const float*)src)[at] : load1<DT == T2W_MX4_BF16>(src, at);
      }
      bad |= !(fabsf(v[j]) <= 6.0f * (1 << MX4_EMAX));
      top = fmaxf(top, fabsf(v[j]));
    }
    uint32_t c[4] = {0, 0, 0, 0};
    int e = 0;
    if (bad) {
      atomicOr(status, 2);
    } else if (top > 0.f) {
      // top = 1.m 2^E, 6 = 1.5 2^2
      const uint32_t bits = __float_as_uint(top);
      e = (int)(bits >> 23) - 127 - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0);
      e = e < MX4_EMIN ? MX4_EMIN : e;
      const float f = __uint_as_float((uint32_t)(e + 127) << 23);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t o = 0;
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[8 * j], v[8 * j + 1], f, 0);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[8 * j + 2], v[8 * j + 3], f, 1);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[8 * j + 4], v[8 * j + 5], f, 2);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[8 * j + 6], v[8 * j + 7], f, 3);
        c[j] = o;
      }
    }
    if (step < steps) w[((size_t)b * steps + step) * 64 + lane] = make_uint4(c[0], c[1], c[2], c[3]);
    s[(bu * 64 + lane) * 4 + t] = (uint8_t)(e + 127);
  }
}

dim3 layout_grid(int n, int k) {
  const size_t g = (size_t)mx4_blocks(n) * mx4_units(k);  // 256 threads each
  return dim3((unsigned)(g < 65536 ? g : 65536));
}

}  // namespace

hipError_t mx4_pack(const t2w_mx4_pack_args& a, hipStream_t st) {
  mx4_pack_kernel<<<layout_grid(a.n, a.k), 256, 0, st>>>((const uint32_t*)a.codes, (const uint8_t*)a.scales, a.n, a.k, (uint4*)a.w_codes,
                                                         (uint8_t*)a.w_scales, a.status);
  return hipGetLastError();
}

hipError_t mx4_quantize(const t2w_mx4_quantize_args& a, hipStream_t st) {
  const auto go = [&](auto dt) {
    mx4_quantize_kernel<decltype(dt)::value><<<layout_grid(a.n, a.k), 256, 0, st>>>(a.w, a.ldw, a.n, a.k, (uint4*)a.w_codes, (uint8_t*)a.w_scales, a.status);
  };
  if (a.dtype == T2W_MX4_BF16) go(std::integral_constant<int, T2W_MX4_BF16>{});
  else if (a.dtype == T2W_MX4_FP16) go(std::integral_constant<int, T2W_MX4_FP16>{});
  else go(std::integral_constant<int, T2W_MX4_FP32>{});
  return hipGetLastError();
}

hipError_t mx4_rows(const Mx4Args& a, bool bf, bool gated, hipStream_t st) {
  if (gated) {
    if (a.m <= 16) return bf ? launch_rows<true, 1, 2, true>(a, st) : launch_rows<false, 1, 2, true>(a, st);
    return bf ? launch_rows<true, 4, 2, true>(a, st) : launch_rows<false, 4, 2, true>(a, st);
  }
  if (a.m <= 16) return bf ? launch_rows<true, 1, 1, false>(a, st) : launch_rows<false, 1, 1, false>(a, st);
  return bf ? launch_rows<true, 4, 1, false>(a, st) : launch_rows<false, 4, 1, false>(a, st);
}

}  // namespace t2w
