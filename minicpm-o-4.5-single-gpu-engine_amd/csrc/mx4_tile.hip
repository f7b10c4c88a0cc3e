// Products with 4-bit weights over many rows: tiles of x in LDS, codes from memory to registers, conversion beside the MFMAs.
//
// A workgroup of WM x WN waves owns 16 TM WM rows of x and TN WN blocks of 16 weight channels (gated: half of them of each
// matrix), a wave TM x TN blocks of 16 x 16.  K advances in stages of 128 columns: x is copied into LDS by buffer loads (two
// buffers, 16-byte chunk c of row r at c ^ (r % 16): the 16 rows of a fragment read cover all 64 banks), a lane's 16 bytes of
// codes of each block go straight into registers, already in operand order.  A stage is four steps of 32 columns; next to a
// step's MFMAs the next step's fragments are read and its codes converted.  The barrier stands in front of a stage's last step,
// whose fragments every wave holds by then: the loads of the stage after next are issued right behind it and have a stage's time.
// Rows behind the last and columns behind k are out of the buffer's bounds and read as zeros.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx4_device.h"

namespace t2w {

namespace {

typedef __attribute__((address_space(3))) void* lds_ptr_t;
constexpr uint32_t OUTSIDE = 0x80000000u, BOUND = 0x7fffff00u;  // byte offsets in the tile's rows of x

template <bool BF, bool GATED, int TM, int TN, int WM, int WN>
struct MxTile {
  static constexpr int NW = WM * WN, BM = 16 * TM * WM, NB = TN * WN;   // waves; rows; weight blocks
  static constexpr int CB = GATED ? NB / 2 : NB;                         // blocks of output channels
  static constexpr int LD = BM / 4 / NW;                                 // 1 KB copies a stage and wave
  static_assert(BM % (4 * NW) == 0, "copies spread evenly");
  const Mx4Args& a;
  __amdgpu_buffer_rsrc_t xr;
  uint32_t off[LD];
  int lane, wave, wm, wn, steps, units;
  const uint4* w[TN];      // scalar: this wave's blocks
  const uint32_t* s[TN];
  f32x4 acc[TN][TM];
  uint4 xf[TM];

  __device__ __forceinline__ MxTile(const Mx4Args& a_, int mt, int nt) : a(a_) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wave / WN, wn = wave % WN;
    steps = (a.k + 127) >> 7, units = (a.k + 511) >> 9;
    const int m0 = mt * BM;
    xr = __builtin_amdgcn_make_buffer_rsrc((void*)((const uint16_t*)a.x + (long long)m0 * a.ldx), 0, (int)BOUND, 0x00020000);
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int r = (wave * LD + i) * 4 + (lane >> 4);
      off[i] = m0 + r < a.m ? (uint32_t)r * (uint32_t)(a.ldx * 2) + (uint32_t)(((lane & 15) ^ (r & 15)) * 16) : OUTSIDE;
    }
    const int nb = (a.n + 15) >> 4;
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const int g = GATED && t >= TN / 2 ? 1 : 0;
      const int b = min(nt * CB + wn * (GATED ? TN / 2 : TN) + (GATED ? t % (TN / 2) : t), nb - 1);
      w[t] = (const uint4*)a.w[g] + (size_t)b * steps * 64;
      s[t] = (const uint32_t*)a.s[g] + (size_t)b * units * 64;
    }
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  struct Codes {
    uint4 c[TN];
    uint32_t e[TN];
  };

  // the loads of stage st
  __device__ __forceinline__ void issue(uint4* xs, Codes& cd, int st) const {
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int r = (wave * LD + i) * 4 + (lane >> 4);
      const uint32_t o = 128 * st + 8 * ((lane & 15) ^ (r & 15)) < a.k ? off[i] : OUTSIDE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_ptr_t)(xs + (wave * LD + i) * 64), 16, o, st * 256, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      cd.c[t] = *(const uint4*)((const uint8_t*)(w[t] + (size_t)st * 64) + (uint32_t)(lane * 16));
      cd.e[t] = *(const uint32_t*)((const uint8_t*)(s[t] + (size_t)(st >> 2) * 64) + (uint32_t)(lane * 4));
    }
    asm volatile("" ::: "memory");  // the loads stay here: left to itself the compiler sinks them to their use, a stage later
  }

  __device__ __forceinline__ uint4 xread(const uint4* xs, int i, int j) const {
    const int c = lane & 15, q = lane >> 4;
    return xs[((wm * TM + i) * 16 + c) * 16 + ((4 * q + j) ^ c)];
  }
  static __device__ __forceinline__ uint32_t word(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

  // the MFMAs of one step on wf and xf; next to them the fragments (xf in place, wn_) of step jn of the stage in xs / cd
  __device__ __forceinline__ void step(const uint4 (&wf)[TN], uint4 (&wnx)[TN], const uint4* xs, const Codes& cd, int st, int jn) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int t = 0; t < TN; ++t) acc[t][i] = mma<BF>(wf[t], xf[i], acc[t][i]);
      xf[i] = xread(xs, i, jn);
#pragma unroll
      for (int t = i * TN / TM; t < (i + 1) * TN / TM; ++t)
        wnx[t] = widen<BF>(word(cd.c[t], jn), __uint_as_float(((cd.e[t] >> (8 * (st & 3))) & 0xffu) << 23));
    }
    constexpr int EVERY = TM > 4 ? TM / 4 : 1;  // 4 TN conversions to TM TN MFMAs
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int t = 0; t < TN; ++t) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if ((i * TN + t) % EVERY == 0) __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  }

  // stage st in (xc, cc), the next one in (xn, cn); s1: behind the last
  __device__ __forceinline__ void stage(uint4* xc, uint4* xn, Codes& cc, Codes& cn, uint4 (&w0)[TN], uint4 (&w1)[TN], int st, int s1) {
    step(w0, w1, xc, cc, st, 1);
    step(w1, w0, xc, cc, st, 2);
    step(w0, w1, xc, cc, st, 3);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    const int nx = min(st + 1, s1 - 1);
    issue(xc, cc, min(st + 2, s1 - 1));
    step(w1, w0, xn, cn, nx, 0);
  }

  __device__ __forceinline__ void run(uint4* x0, uint4* x1, int s0, int s1) {
    Codes c0, c1;
    uint4 w0[TN], w1[TN];
    issue(x0, c0, s0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    issue(x1, c1, min(s0 + 1, s1 - 1));
#pragma unroll
    for (int i = 0; i < TM; ++i) xf[i] = xread(x0, i, 0);
#pragma unroll
    for (int t = 0; t < TN; ++t) w0[t] = widen<BF>(c0.c[t].x, __uint_as_float(((c0.e[t] >> (8 * (s0 & 3))) & 0xffu) << 23));
    int st = s0;
    for (; st + 1 < s1; st += 2) {
      stage(x0, x1, c0, c1, w0, w1, st, s1);
      stage(x1, x0, c1, c0, w0, w1, st + 1, s1);
    }
    if (st < s1) stage(x0, x1, c0, c1, w0, w1, st, s1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last stage's repeated loads into LDS
  }
};

// outputs of block (t, i) of a wave from its sums p (and u of the second matrix)
template <bool BF, bool GATED, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void block_store(const Mx4Args& a, int mt, int nt, int wave, int t, int i, f32x4 p, f32x4 u) {
  const int lane = threadIdx.x & 63, wm = wave / WN, wn = wave % WN;
  constexpr int OT = GATED ? TN / 2 : TN;
  const int m = (mt * WM + wm) * 16 * TM + 16 * i + (lane & 15), n = ((nt * WN + wn) * OT + t) * 16 + 4 * (lane >> 4);
  if (m >= a.m || n >= a.n) return;
  float o[4] = {p[0], p[1], p[2], p[3]};
  if constexpr (GATED) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = gate_act(o[e], a.act) * u[e];
  }
  finish<BF>(a, m, n, o);
}

// tile number b of tm x tn tiles -> (row, column): an XCD gets a run of tiles (workgroups go round the 8 XCDs), which walks
// groups of 4 rows column by column, so that the tiles at work on an XCD share rows of x and columns of W in its L2
__device__ __forceinline__ int2 tile_at(int b, int tm, int tn) {
  const int total = tm * tn, q = total >> 3, r = total & 7, x = b & 7;
  const int t = x * q + min(x, r) + (b >> 3);
  const int grp = t / (4 * tn), rows = min(4, tm - 4 * grp), in = t - grp * 4 * tn;
  return make_int2(4 * grp + in % rows, in / rows);
}

template <bool BF, bool GATED, int TM, int TN, int WM, int WN, bool PART>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx4_tile_kernel(const Mx4Args a, int tm, int tn, int splits, f32x4* part) {
  typedef MxTile<BF, GATED, TM, TN, WM, WN> T;
  __shared__ uint4 x0[T::BM * 16], x1[T::BM * 16];
  const int total = tm * tn;
  const int split = PART ? (int)blockIdx.x / total : 0, b = (int)blockIdx.x - split * total;
  const int2 at = tile_at(b, tm, tn);
  T t(a, at.x, at.y);
  const int s0 = PART ? (int)((long long)t.steps * split / splits) : 0, s1 = PART ? (int)((long long)t.steps * (split + 1) / splits) : t.steps;
  t.run(x0, x1, s0, s1);
  if constexpr (PART) {
    f32x4* p = part + (size_t)(blockIdx.x * T::NW + t.wave) * (TM * TN * 64) + t.lane;
#pragma unroll
    for (int y = 0; y < TN; ++y)
#pragma unroll
      for (int i = 0; i < TM; ++i) p[(y * TM + i) * 64] = t.acc[y][i];
  } else {
    constexpr int OT = GATED ? TN / 2 : TN;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int y = 0; y < OT; ++y) block_store<BF, GATED, TM, TN, WM, WN>(a, at.x, at.y, t.wave, y, i, t.acc[y][i], t.acc[GATED ? y + OT : y][i]);
  }
}

// sums of the parts in the order of the splits; a wave has one block of one wave of one tile (gated: of both matrices)
template <bool BF, bool GATED, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(256) void mx4_join_kernel(const Mx4Args a, int tm, int tn, int splits, const f32x4* part) {
  constexpr int NW = WM * WN, OT = GATED ? TN / 2 : TN;
  const int id = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int blk = id % (OT * TM), w = id / (OT * TM);  // w: tile and wave
  if (w >= tm * tn * NW) return;
  const int2 at = tile_at(w / NW, tm, tn);
  const size_t stride = (size_t)tm * tn * NW * (TM * TN * 64);
  const f32x4* p = part + ((size_t)w * (TM * TN) + blk) * 64 + lane;
  f32x4 v = p[0], u = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (GATED) u = p[OT * TM * 64];
#pragma unroll 4
  for (int s = 1; s < splits; ++s) {
    v += p[s * stride];
    if constexpr (GATED) u += p[s * stride + OT * TM * 64];
  }
  block_store<BF, GATED, TM, TN, WM, WN>(a, at.x, at.y, w % NW, blk / TM, blk % TM, v, u);
}

template <bool BF, bool GATED, int TM, int TN, int WM, int WN>
hipError_t launch(const Mx4Args& a, int splits, float* part, hipStream_t st) {
  typedef MxTile<BF, GATED, TM, TN, WM, WN> T;
  const int tm = (a.m + T::BM - 1) / T::BM, tn = (mx4_blocks(a.n) + T::CB - 1) / T::CB;
  if (splits <= 1) {
    mx4_tile_kernel<BF, GATED, TM, TN, WM, WN, false><<<tm * tn, 64 * T::NW, 0, st>>>(a, tm, tn, 1, nullptr);
    return hipGetLastError();
  }
  mx4_tile_kernel<BF, GATED, TM, TN, WM, WN, true><<<tm * tn * splits, 64 * T::NW, 0, st>>>(a, tm, tn, splits, (f32x4*)part);
  mx4_join_kernel<BF, GATED, TM, TN, WM, WN><<<(tm * tn * T::NW * TM * (GATED ? TN / 2 : TN) + 3) / 4, 256, 0, st>>>(a, tm, tn, splits, (const f32x4*)part);
  return hipGetLastError();
}

// The one tile: 64 rows by 256 weight channels (gated: 128 of each matrix), four waves of 64 x 64, two workgroups a CU.
constexpr int TILE_M = 64, TILE_N = 256, SLOTS = 512;

struct Plan {
  int tiles, splits;
};

// k is split where the tiles do not fill the chip's places, into parts of four stages at least
Plan plan(int m, int n, int k, bool gated) {
  const int tn = gated ? (n + TILE_N / 2 - 1) / (TILE_N / 2) : (n + TILE_N - 1) / TILE_N;
  const long long tiles = (long long)((m + TILE_M - 1) / TILE_M) * tn;
  if (tiles > SLOTS / 2) return {(int)tiles, 1};
  const int by_k = mx4_steps(k) / 4, by_n = SLOTS / (int)tiles;
  return {(int)tiles, std::max(1, std::min(by_k, by_n))};
}

}  // namespace

// a row's place in its tile is a 31-bit byte offset
bool mx4_takes_tiles(int m, long long ldx) { return m > 16 && ldx < (1 << 24); }

size_t mx4_tiles_workspace(int m, int n, int k, bool gated) {
  const Plan p = plan(m, n, k, gated);
  return p.splits > 1 ? (size_t)p.tiles * p.splits * TILE_M * TILE_N * 4 : 0;
}

hipError_t mx4_tiles(const Mx4Args& a, bool bf, bool gated, void* workspace, hipStream_t st) {
  const int splits = plan(a.m, a.n, a.k, gated).splits;
  float* part = (float*)workspace;
  if (gated) return bf ? launch<true, true, 4, 4, 1, 4>(a, splits, part, st) : launch<false, true, 4, 4, 1, 4>(a, splits, part, st);
  return bf ? launch<true, false, 4, 4, 1, 4>(a, splits, part, st) : launch<false, false, 4, 4, 1, 4>(a, splits, part, st);
}

}  // namespace t2w
