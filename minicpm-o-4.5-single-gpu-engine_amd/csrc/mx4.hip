// Operators on 4-bit weights (e2m1 codes, a power-of-two scale for every 32 columns): laying a matrix out, quantizing one, and
// the products with few rows.
//
// y = x W^T: a code times its scale is exact in bf16 and in fp16, so the matrix unit's products are exact and the sums fp32: the
// only roundings are the fp32 additions' and the output's.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mx4_device.h"

namespace t2w {

namespace {

// --- few rows --------------------------------------------------------------------------------------------------------
// Up to 16 rows of x (a grid's y: 16 more).  A workgroup takes blocks of 16 channels in turn; each of its waves has units of 512
// columns (GATED: even waves of the gate's matrix, odd ones of the other), whose codes it converts in registers, and the waves'
// sums meet in LDS in the order of the waves.  The stream of codes is what bounds it: a step's registers are loaded again, with
// the wave's next unit, as soon as the step is converted, so that a wave always has about 4 KB in flight, across units and blocks.
// x lies in LDS, brought there once by each workgroup (16-byte chunk c of a step of row r at c ^ r: 16 rows' reads cover all
// banks), zero behind k.  A wave reads 4 KB of it a step's 1 KB of codes; from memory that alone takes the L1 cache's whole
// bandwidth: one row x 14336 x 2 gates of 4096 columns 18.3 us, from LDS 12.4.  Of rows too long for LDS (ALL false) the first `held`
// units are there and the others are read from memory.
// Measured (kernel times, codes from HBM): 1 row x 6144 x 4096 4.7 us, 3 rows x 128001 x 4096 49 us (5.6 TB/s), one row's gated
// 14336 x 4096 x 2 12.6 us (5.0 TB/s) and 4096 x 14336 6.7 us (one block a CU: 4.7 TB/s).  Two blocks a wave at a time (half the
// reads of x) took 10% longer; 4 or 8 waves a workgroup instead of 16 gain nothing at one row and take 26.7 and 18.3 us instead of
// 16.5 at 16 rows' gated 14336 x 4096 x 2.
template <bool BF, bool GATED, Form F, bool ALL>
__global__ __launch_bounds__(1024) void mx4_rows_kernel(const Mx4Args a, int held) {
  extern __shared__ uint4 lds[];  // x [rows][held][4][16], then sums [2][waves][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int steps = (a.k + 127) >> 7, units = (a.k + 511) >> 9, q = lane >> 4, nb = (a.n + 15) >> 4;
  const int first = GATED ? wave >> 1 : wave, stride = GATED ? waves >> 1 : waves;  // this wave's units
  const int m0 = 16 * blockIdx.y, rows = min(16, a.m - m0), row = min(lane & 15, rows - 1);  // lanes behind the last row repeat it: not stored
  const uint16_t* x = (const uint16_t*)a.x + (long long)m0 * a.ldx;
  uint4* xs = lds;
  f32x4* part = (f32x4*)(lds + rows * held * 64);
  const uint8_t* w = GATED && (wave & 1) ? a.w[1] : a.w[0];
  const uint8_t* s = GATED && (wave & 1) ? a.s[1] : a.s[0];

  uint4 code[4];
  uint32_t sc, scn = 0;
  // step t of unit u of block g; behind the last step the last again, against columns of x that are zero
  const auto load = [&](int g, int u, int t) {
    code[t] = *(const uint4*)(w + ((size_t)g * steps + min(4 * u + t, steps - 1)) * 1024 + (uint32_t)(lane * 16));
  };
  const auto load_scales = [&](int g, int u) { return *(const uint32_t*)(s + ((size_t)g * units + u) * 256 + (uint32_t)(lane * 4)); };

  int g = blockIdx.x, u = first;
  // a unit's 1 KB of a row at a time, straight to LDS, all in flight together; columns behind k are out of the row's bounds: zeros
  for (int r = GATED ? wave & 1 : 0; r < rows; r += GATED ? 2 : 1) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(x + (long long)r * a.ldx), 0, a.k * 2, 0x00020000);
    const int c = (lane & ~15) | ((lane ^ r) & 15);
    for (int b = first; b < held; b += stride)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(xs + (r * held + b) * 64), 16, c * 16, b * 1024, 0, 0);
  }
  asm volatile("" ::: "memory");
  sc = load_scales(g, u);
#pragma unroll
  for (int t = 0; t < 4; ++t) load(g, u, t);
  asm volatile("s_waitcnt vmcnt(5)" ::: "memory");  // x is there, the codes may still be on their way
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  const uint16_t* xrow = x + (long long)row * a.ldx + 32 * q;

  f32x4 acc[2];
  const auto unit_of = [&](auto more, auto in, int gn, int un) {
    constexpr bool MORE = decltype(more)::value, IN = decltype(in)::value;
    if (MORE) scn = load_scales(gn, un);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint4 xf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (IN) {
          xf[j] = xs[(row * held + u) * 64 + 16 * t + ((4 * q + j) ^ row)];
        } else {
          xf[j] = make_uint4(0, 0, 0, 0);
          const int k0 = 512 * u + 128 * t + 8 * j;
          if (k0 + 32 * q < a.k) xf[j] = *(const uint4*)(xrow + k0);
        }
      }
      const float f = scale_of(sc, t);
      const uint4 w0 = widen<BF>(code[t].x, f), w1 = widen<BF>(code[t].y, f), w2 = widen<BF>(code[t].z, f), w3 = widen<BF>(code[t].w, f);
      if (MORE) {
        load(gn, un, t);
        asm volatile("" ::: "memory");
      }
      acc[0] = mma<BF>(w0, xf[0], acc[0]);
      acc[1] = mma<BF>(w1, xf[1], acc[1]);
      acc[0] = mma<BF>(w2, xf[2], acc[0]);
      acc[1] = mma<BF>(w3, xf[3], acc[1]);
    }
    if (MORE) sc = scn;
  };
  const auto unit = [&](auto more, int gn, int un) {
    if (ALL || u < held) unit_of(more, std::true_type{}, gn, un);
    else unit_of(more, std::false_type{}, gn, un);
  };

  for (int turn = 0; g < nb; turn ^= 1) {
    acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (; u + stride < units; u += stride) unit(std::true_type{}, g, u + stride);
    const int gn = g + gridDim.x;
    if (gn < nb) unit(std::true_type{}, gn, first);
    else unit(std::false_type{}, 0, 0);
    u = first;
    const int n = g * 16 + 4 * q, m = m0 + (lane & 15);
    Extra ex[1] = {};
    if (!GATED && wave == 0) fetch<F>(a, {make_int2(m, n)}, ex);
    f32x4* p = part + turn * waves * 64;
    p[wave * 64 + lane] = acc[0] + acc[1];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the codes in flight are not waited for
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (wave == 0) {  // the others go on; the sums' other half is theirs until the next barrier
      f32x4 v = p[lane], o = p[GATED ? 64 + lane : lane];
      for (int i = 1; i < stride; ++i) {
        v += p[(GATED ? 2 * i : i) * 64 + lane];
        if constexpr (GATED) o += p[(2 * i + 1) * 64 + lane];
      }
      float r[4] = {v[0], v[1], v[2], v[3]};
      if constexpr (GATED) {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = gate_act(r[e], a.act) * o[e];
      }
      finish<BF, GATED, F>(a, m, n, r, ex[0]);
    }
    g = gn;
  }
}

constexpr size_t LDS_CU = 160 * 1024;

struct RowsPlan {
  int waves, held;  // units of x in LDS
  size_t bytes;     // of LDS
};

RowsPlan rows_plan(int m, int k, bool gated) {
  const int units = mx4_units(k), two = gated ? 2 : 1, rows = std::min(m, 16);
  const int rounds = (units * two + 15) / 16, waves = (units + rounds - 1) / rounds * two;
  const size_t sums = (size_t)2 * waves * 1024;
  const int held = (int)std::min<size_t>(units, (LDS_CU - sums) / ((size_t)rows * 1024));
  return {waves, held, (size_t)rows * held * 1024 + sums};
}

template <bool BF, bool GATED, Form F, bool ALL>
hipError_t launch_rows(const Mx4Args& a, const RowsPlan& p, hipStream_t st) {
  if (p.bytes > 64 * 1024) {  // beyond the default a function has to be told, on each device
    static std::atomic<uint64_t> told{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(told.load(std::memory_order_acquire) & bit)) {
      e = hipFuncSetAttribute((const void*)mx4_rows_kernel<BF, GATED, F, ALL>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_CU);
      if (e != hipSuccess) return e;
      told.fetch_or(bit, std::memory_order_release);
    }
  }
  const int nb = mx4_blocks(a.n), fit = std::max(1, std::min(16 / p.waves, (int)(LDS_CU / p.bytes)));  // workgroups a CU
  const int rounds = (nb + 256 * fit - 1) / (256 * fit);
  mx4_rows_kernel<BF, GATED, F, ALL><<<dim3((nb + rounds - 1) / rounds, (a.m + 15) / 16), p.waves * 64, p.bytes, st>>>(a, p.held);
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

int mx4_rows_outside(int m, int k, bool gated) { return mx4_units(k) - rows_plan(m, k, gated).held; }

hipError_t mx4_rows(const Mx4Args& a, bool bf, bool gated, Form form, hipStream_t st) {
  const RowsPlan p = rows_plan(a.m, a.k, gated);
  return mx4_dispatch(bf, gated, form, [&](auto b, auto g, auto f) {
    constexpr bool BF = decltype(b)::value, GATED = decltype(g)::value;
    constexpr Form F = decltype(f)::value;
    return p.held == mx4_units(a.k) ? launch_rows<BF, GATED, F, true>(a, p, st) : launch_rows<BF, GATED, F, false>(a, p, st);
  });
}

}  // namespace t2w
