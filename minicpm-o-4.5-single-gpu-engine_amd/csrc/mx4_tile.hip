// Products with 4-bit weights over many rows: tiles of x in LDS, codes from memory to registers, conversion beside the MFMAs.
//
// A workgroup of WN waves side by side owns 16 TM rows of x and TN WN blocks of 16 weight channels (gated: half of them of each
// matrix), a wave TM x TN blocks of 16 x 16.  K advances in stages of 128 columns: x is copied into LDS by buffer loads (two
// buffers, 16-byte chunk c of row r at c ^ (r % 16): the 16 rows of a fragment read cover all 64 banks), a lane's 16 bytes of
// codes of each block go straight into registers, already in operand order.  A stage is four steps of 32 columns; next to a
// step's MFMAs the next step's fragments are read and its codes converted.  The barrier stands in front of a stage's last step,
// whose fragments every wave holds by then: the loads of the stage after next are issued right behind it and have a stage's time.
// Rows behind the last and columns behind k are out of the buffer's bounds and read as zeros.  The buffers are objects of their own,
// named at compile time: behind one indexed array the compiler would wait for all copies before every read.
//
// The conversion is one instruction for two weights and shares the wave's time with the MFMAs; the codes come to a CU at a quarter
// of bf16's bytes, which is why a tile of only 64 rows reaches the rate of a large bf16 product: 64 x 256 tiles run 4001 rows x
// 6144 x 4096 in 156 to 176 us (1.15 to 1.29 PFLOP/s, by machine) and 2005 rows' gated 14336 x 4096 x 2 in 359 to 396 (1.19 to 1.31).
// There the matrix units are busy for 53 to 62% of the cycles at a clock of 2.0 GHz, vector instructions issue in 40% and the waves
// wait for a quarter of theirs.  With two workgroups a CU the barriers of one fall into the other's MFMAs: 128 x 256 tiles of eight waves, one
// workgroup a CU, took 9% longer, 256 x 256 (spilling) 21%, waves of 128 x 64 (half the conversions a product) alone on a SIMD 18%.
// Few tiles are bound by what one CU takes in, about 65 bytes a ns whatever its waves: hence the split of k over workgroups.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx4_device.h"

namespace t2w {

namespace {

constexpr uint32_t OUTSIDE = 0x80000000u, BOUND = 0x7fffff00u;  // byte offsets in the tile's rows of x

template <bool BF, bool GATED, int TM, int TN, int WN>
struct MxTile {
  static constexpr int NW = WN, BM = 16 * TM, NB = TN * WN;   // waves; rows; weight blocks
  static constexpr int CB = GATED ? NB / 2 : NB;                         // blocks of output channels
  static constexpr int LD = BM / 4 / NW;                                 // 1 KB copies a stage and wave
  static constexpr int LOADS = LD + 2 * TN;                              // a stage's, of a wave
  static_assert(BM % (4 * NW) == 0, "copies spread evenly");
  const Mx4Args& a;
  __amdgpu_buffer_rsrc_t xr;
  uint32_t off[LD];
  int lane, wave, steps, units;
  __amdgpu_buffer_rsrc_t wr[GATED ? 2 : 1], sr[GATED ? 2 : 1];  // this wave's blocks of each matrix
  f32x4 acc[TN][TM];

  __device__ __forceinline__ MxTile(const Mx4Args& a_, int mt, int nt) : a(a_) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % NW;
    steps = (a.k + 127) >> 7, units = (a.k + 511) >> 9;
    const int m0 = mt * BM;
    xr = __builtin_amdgcn_make_buffer_rsrc((void*)((const uint16_t*)a.x + (long long)m0 * a.ldx), 0, (int)BOUND, 0x00020000);
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int r = (wave * LD + i) * 4 + (lane >> 4);
      off[i] = m0 + r < a.m ? (uint32_t)r * (uint32_t)(a.ldx * 2) + (uint32_t)(((lane & 15) ^ (r & 15)) * 16) : OUTSIDE;
    }
    // blocks behind the last are out of bounds as well
    constexpr int WB = GATED ? TN / 2 : TN;
    const int b0 = __builtin_amdgcn_readfirstlane(nt * CB + wave * WB), have = __builtin_amdgcn_readfirstlane(max(0, min(WB, ((a.n + 15) >> 4) - b0)));
#pragma unroll
    for (int g = 0; g < (GATED ? 2 : 1); ++g) {
      wr[g] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w[g] + (size_t)b0 * steps * 1024), 0, have * steps * 1024, 0x00020000);
      sr[g] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.s[g] + (size_t)b0 * units * 256), 0, have * units * 256, 0x00020000);
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

  // the loads of stage st; none of a stage from s1 on (the registers and LDS get zeros, so that no branch parts the loop)
  __device__ __forceinline__ void issue(uint4* xs, Codes& cd, int st, int s1) const {
    const int end = st < s1 ? a.k : 0;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int r = (wave * LD + i) * 4 + (lane >> 4);
      const uint32_t o = 128 * st + 8 * ((lane & 15) ^ (r & 15)) < end ? off[i] : OUTSIDE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_ptr_t)(xs + (wave * LD + i) * 64), 16, o, st * 256, 0, 0);
    }
    const uint32_t at = st < s1 ? (uint32_t)lane * 16 : OUTSIDE;
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      constexpr int WB = GATED ? TN / 2 : TN;
      const int g = t / WB, b = t % WB;
      cd.c[t] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(wr[g], at, (b * steps + st) * 1024, 0));
      cd.e[t] = __builtin_amdgcn_raw_buffer_load_b32(sr[g], at >> 2, (b * units + (st >> 2)) * 256, 0);
    }
    asm volatile("" ::: "memory");  // the loads stay here: left to itself the compiler sinks them to their use, a stage later
  }

  __device__ __forceinline__ uint4 xread(const uint4* xs, int i, int j) const {
    const int c = lane & 15, q = lane >> 4;
    return xs[(i * 16 + c) * 16 + ((4 * q + j) ^ c)];
  }
  static __device__ __forceinline__ uint32_t word(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

  // The MFMAs of one step on wf and xf; next to them xf's place is filled with the fragments of step jx in xs and wnx with the
  // codes of step jn of stage st in cd.
  __device__ __forceinline__ void step(const uint4 (&wf)[TN], uint4 (&wnx)[TN], uint4 (&xf)[TM], const uint4* xs, int jx, const Codes& cd, int st, int jn) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int t = 0; t < TN; ++t) acc[t][i] = mma<BF>(wf[t], xf[i], acc[t][i]);
      xf[i] = xread(xs, i, jx);
#pragma unroll
      for (int t = i * TN / TM; t < (i + 1) * TN / TM; ++t)
        wnx[t] = widen<BF>(word(cd.c[t], jn), __uint_as_float(((cd.e[t] >> (8 * (st & 3))) & 0xffu) << 23));
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int t = 0; t < TN; ++t) {  // an MFMA, a conversion; then a read
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  }

  // Stage st in (xc, cc), the next one in (xn, cn); the loads of stage st + D go to (xl, cl).
  // AHEAD 1: fragments are read a step ahead, which 16 MFMAs a step cover; the barrier stands in front of the last step, when every
  // wave holds its fragments of the stage, and the freed buffer is the one to load (xl is xc).
  // AHEAD 2: with 2 or 4 MFMAs a step a fragment's way from LDS takes longer than a step, so they are read two ahead into two sets in
  // turn; the barrier stands in the stage's middle, and a buffer more than D lets xl be one that was read a stage ago.
  // TAIL: the (TAIL + 1)th stage behind the loop.  Nothing is left to load there, so it loads nothing and knows how many loads are
  // behind the next stage's (loads that the compiler may drop, as nobody reads what they bring, could not be counted on).
  template <int D, int AHEAD, int TAIL>
  __device__ __forceinline__ void stage(uint4* xc, uint4* xn, uint4* xl, Codes& cc, Codes& cn, Codes& cl, uint4 (&w0)[TN], uint4 (&w1)[TN], uint4 (&xa)[TM],
                                        uint4 (&xb)[TM], int st, int s1) {
    constexpr int LATER = (TAIL < 0 ? D - 2 : TAIL < D - 2 ? D - 2 - TAIL : 0) * LOADS;  // in flight behind the next stage's
    if constexpr (AHEAD == 1) {
      step(w0, w1, xa, xc, 1, cc, st, 1);
      step(w1, w0, xa, xc, 2, cc, st, 2);
      step(w0, w1, xa, xc, 3, cc, st, 3);
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LATER) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (TAIL < 0) issue(xl, cl, st + D, s1);
      step(w1, w0, xa, xn, 0, cn, st + 1, 0);
    } else {
      step(w0, w1, xa, xc, 2, cc, st, 1);
      step(w1, w0, xb, xc, 3, cc, st, 2);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (TAIL < 0) issue(xl, cl, st + D, s1);
      step(w0, w1, xa, xn, 0, cc, st, 3);
      step(w1, w0, xb, xn, 1, cn, st + 1, 0);
    }
  }

  // n stages from s0 on, those from s1 on of zeros; D in flight over XB buffers
  template <int D, int XB>
  __device__ __forceinline__ void run(uint4* const (&x)[XB], int s0, int s1, int n) {
    constexpr int AHEAD = XB > D ? 2 : 1;
    Codes c[XB];
    uint4 w0[TN], w1[TN], xa[TM], xb[TM];
#pragma unroll
    for (int d = 0; d < D; ++d) issue(x[d], c[d], s0 + d, s1);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * LOADS) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      xa[i] = xread(x[0], i, 0);
      if (AHEAD == 2) xb[i] = xread(x[0], i, 1);
    }
#pragma unroll
    for (int t = 0; t < TN; ++t) w0[t] = widen<BF>(c[0].c[t].x, __uint_as_float(((c[0].e[t] >> (8 * (s0 & 3))) & 0xffu) << 23));
    int i = 0;
    for (; i + XB <= n; i += XB) {
#pragma unroll
      for (int d = 0; d < XB; ++d)
        stage<D, AHEAD, -1>(x[d], x[(d + 1) % XB], x[(d + D) % XB], c[d], c[(d + 1) % XB], c[(d + D) % XB], w0, w1, xa, xb, s0 + i + d, s1);
    }
    static_assert((XB == 2 || XB == 4) && XB - 1 <= D, "the stages behind the loop are all on their way when it ends");
    if (i < n) stage<D, AHEAD, 0>(x[0], x[1], x[0], c[0], c[1], c[0], w0, w1, xa, xb, s0 + i, s1);
    if constexpr (XB == 4) {
      if (i + 1 < n) stage<D, AHEAD, 1>(x[1], x[2], x[0], c[1], c[2], c[0], w0, w1, xa, xb, s0 + i + 1, s1);
      if (i + 2 < n) stage<D, AHEAD, 2>(x[2], x[3], x[0], c[2], c[3], c[0], w0, w1, xa, xb, s0 + i + 2, s1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was issued into LDS behind the last stage
  }
};

// first output (row, channel) of this lane in block (t, i) of a wave
template <bool GATED, int TM, int TN, int WN>
__device__ __forceinline__ int2 place(int mt, int nt, int wave, int t, int i) {
  const int lane = threadIdx.x & 63;
  constexpr int OT = GATED ? TN / 2 : TN;
  return make_int2((mt * TM + i) * 16 + (lane & 15), ((nt * WN + wave) * OT + t) * 16 + 4 * (lane >> 4));
}

// the outputs at a place from their sums p (and u of the second matrix)
template <bool BF, bool GATED, Form F>
__device__ __forceinline__ void block_store(const Mx4Args& a, int2 at, f32x4 p, f32x4 u, const Extra& ex) {
  float o[4] = {p[0], p[1], p[2], p[3]};
  if constexpr (GATED) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = gate_act(o[e], a.act) * u[e];
  }
  finish<BF, GATED, F>(a, at.x, at.y, o, ex);
}

// tile number b of tm x tn tiles -> (row, column): an XCD gets a run of tiles (workgroups go round the 8 XCDs), which walks
// groups of 4 rows column by column, so that the tiles at work on an XCD share rows of x and columns of W in its L2
__device__ __forceinline__ int2 tile_at(int b, int tm, int tn) {
  const int total = tm * tn, q = total >> 3, r = total & 7, x = b & 7;
  const int t = x * q + min(x, r) + (b >> 3);
  const int grp = t / (4 * tn), rows = min(4, tm - 4 * grp), in = t - grp * 4 * tn;
  return make_int2(4 * grp + in % rows, in / rows);
}

// KG groups of waves share a tile, each with its run of the stages and buffers of its own; their sums meet in LDS, and each group
// finishes its share of the blocks.
template <bool BF, bool GATED, Form F, int TM, int TN, int WN, int D, int XB, int KG, bool PART>
__global__ __launch_bounds__(64 * WN * KG, 2) void mx4_tile_kernel(const Mx4Args a, int tm, int tn, int splits, f32x4* part) {
  typedef MxTile<BF, GATED, TM, TN, WN> T;
  constexpr int XS = T::BM * 16;
  __shared__ uint4 x0[KG * XS], x1[KG * XS], x2[XB == 4 ? KG * XS : 1], x3[XB == 4 ? KG * XS : 1];  // objects of their own: see the top
  const int total = tm * tn;
  const int split = PART ? (int)blockIdx.x / total : 0, b = (int)blockIdx.x - split * total;
  const int2 at = tile_at(b, tm, tn);
  T t(a, at.x, at.y);
  int s0 = PART ? (int)((long long)t.steps * split / splits) : 0, s1 = PART ? (int)((long long)t.steps * (split + 1) / splits) : t.steps;
  int n = s1 - s0;  // stages to go through: the same for all groups, whose barriers are common
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / (64 * T::NW)) : 0;
  if constexpr (KG > 1) {
    n = (n + KG - 1) / KG;
    s0 += kg * n, s1 = min(s1, s0 + n);
  }
  const int xo = kg * XS;
  if constexpr (XB == 2) t.template run<D, 2>({x0 + xo, x1 + xo}, s0, s1, n);
  else t.template run<D, 4>({x0 + xo, x1 + xo, x2 + xo, x3 + xo}, s0, s1, n);
  constexpr int OT = GATED ? TN / 2 : TN, BLOCKS = TM * TN, OUT = OT * TM;  // blocks of sums and of outputs of a wave
  constexpr int MINE = (OUT + KG - 1) / KG;                                  // this group's: kg, kg + KG, ..
  f32x4 sum[GATED ? 2 : 1][MINE];
  if constexpr (KG > 1) {
    static_assert((OUT % KG == 0 || OUT == 1) && KG % 2 == 0 && KG / 2 * T::NW * BLOCKS * 64 <= KG * XS, "whole shares; half of the groups' sums fit a buffer");
    __syncthreads();  // every wave is through with the buffers
    const auto red = [&](int g) { return (f32x4*)(g < KG / 2 ? x0 : x1) + ((g % (KG / 2)) * T::NW + t.wave) * BLOCKS * 64 + t.lane; };
    f32x4* own = red(kg);
#pragma unroll
    for (int y = 0; y < TN; ++y)
#pragma unroll
      for (int i = 0; i < TM; ++i) own[(y * TM + i) * 64] = t.acc[y][i];
    __syncthreads();
    if (OUT == 1 && kg > 0) return;
#pragma unroll
    for (int j = 0; j < MINE; ++j)
#pragma unroll
      for (int h = 0; h < (GATED ? 2 : 1); ++h) {
        const int at_ = (kg + j * KG + h * OUT) * 64;
        sum[h][j] = red(0)[at_];
#pragma unroll
        for (int g = 1; g < KG; ++g) sum[h][j] += red(g)[at_];
      }
  } else {
#pragma unroll
    for (int j = 0; j < MINE; ++j)
#pragma unroll
      for (int h = 0; h < (GATED ? 2 : 1); ++h) sum[h][j] = t.acc[j / TM + h * OT][j % TM];
  }
  if constexpr (PART) {
    f32x4* p = part + (size_t)(blockIdx.x * T::NW + t.wave) * (BLOCKS * 64) + t.lane;
#pragma unroll
    for (int j = 0; j < MINE; ++j)
#pragma unroll
      for (int h = 0; h < (GATED ? 2 : 1); ++h) p[(kg + j * KG + h * OUT) * 64] = sum[h][j];
  } else {
    Extra ex[MINE] = {};
    int2 o[MINE];
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int b_ = kg + j * KG;
      o[j] = place<GATED, TM, TN, WN>(at.x, at.y, t.wave, b_ / TM, b_ % TM);
    }
    if (!GATED) fetch<F>(a, o, ex);
#pragma unroll
    for (int j = 0; j < MINE; ++j) block_store<BF, GATED, F>(a, o[j], sum[0][j], sum[GATED ? 1 : 0][j], ex[j]);
  }
}

// sums of the parts in the order of the splits; a wave has one block of one wave of one tile (gated: of both matrices)
template <bool BF, bool GATED, Form F, int TM, int TN, int WN>
__global__ __launch_bounds__(256) void mx4_join_kernel(const Mx4Args a, int tm, int tn, int splits, const f32x4* part) {
  constexpr int NW = WN, OT = GATED ? TN / 2 : TN;
  const int id = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int blk = id % (OT * TM), w = id / (OT * TM);  // w: tile and wave
  if (w >= tm * tn * NW) return;
  const int2 at = tile_at(w / NW, tm, tn);
  const size_t stride = (size_t)tm * tn * NW * (TM * TN * 64);
  const f32x4* p = part + ((size_t)w * (TM * TN) + blk) * 64 + lane;
  const int2 o = place<GATED, TM, TN, WN>(at.x, at.y, w % NW, blk / TM, blk % TM);
  Extra ex[1] = {};
  if (!GATED) fetch<F>(a, {o}, ex);
  f32x4 v = p[0], u = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (GATED) u = p[OT * TM * 64];
#pragma unroll 4
  for (int s = 1; s < splits; ++s) {
    v += p[s * stride];
    if constexpr (GATED) u += p[s * stride + OT * TM * 64];
  }
  block_store<BF, GATED, F>(a, o, v, u, ex[0]);
}

template <bool BF, bool GATED, Form F, int TM, int TN, int WN, int D, int XB, int KG>
hipError_t launch(const Mx4Args& a, int splits, float* part, hipStream_t st) {
  typedef MxTile<BF, GATED, TM, TN, WN> T;
  const int tm = (a.m + T::BM - 1) / T::BM, tn = (mx4_blocks(a.n) + T::CB - 1) / T::CB;
  if (splits <= 1) {
    mx4_tile_kernel<BF, GATED, F, TM, TN, WN, D, XB, KG, false><<<tm * tn, 64 * T::NW * KG, 0, st>>>(a, tm, tn, 1, nullptr);
    return hipGetLastError();
  }
  mx4_tile_kernel<BF, GATED, F, TM, TN, WN, D, XB, KG, true><<<tm * tn * splits, 64 * T::NW * KG, 0, st>>>(a, tm, tn, splits, (f32x4*)part);
  mx4_join_kernel<BF, GATED, F, TM, TN, WN><<<(tm * tn * T::NW * TM * (GATED ? TN / 2 : TN) + 3) / 4, 256, 0, st>>>(a, tm, tn, splits, (const f32x4*)part);
  return hipGetLastError();
}

// The tiles, each with four waves side by side: rows, weight channels (gated: half of each matrix), groups of waves that split k, and
// the microseconds of a pass (a stage of each group) with one workgroup on a CU and, of each, with several.  Measured with codes from
// HBM (more matrices in turn than a cache holds): 6144 channels x 4096 columns x 64 rows take 11.4 / 13.9 / 25 / 37 us (the first 9.6
// with a matrix in the last-level cache), 28000 x 4096 x 32 20 / 16 / 27 / 36, x 100 45 / 38 / 33 / 39; the wide two take 396 / 368 for
// 2005 rows of 14336 x 4096 x 2, gated, and 395 / 364 for 4010 rows of 4096 x 14336.
struct Shape {
  int bm, bn, kg;
  float one, many;
};
constexpr Shape SHAPES[4] = {{16, 128, 2, 0.42f, 0.42f}, {32, 128, 2, 0.52f, 0.60f}, {64, 128, 1, 0.70f, 0.44f}, {64, 256, 1, 0.90f, 0.79f}};

struct Plan {
  int shape, tiles, splits;
  float us;
};

// The cheapest by that model: 5 us for a launch, its first loads and stores; where k is split over workgroups 4.5 us and the
// parts' way to memory and back (8 TB/s) more.  k is split so that the workgroups fill the 256 CUs once or twice, 512 at most.
Plan plan(int m, int n, int k, bool gated) {
  Plan best{0, 0, 1, 3e38f};
  const int steps = mx4_steps(k), cols = gated ? 2 * n : n;
  for (int i = 0; i < 4; ++i) {
    const Shape& s = SHAPES[i];
    const long long tiles = (long long)((m + s.bm - 1) / s.bm) * ((cols + s.bn - 1) / s.bn);
    int last = 0;
    for (const int fill : {0, 128, 256, 512}) {
      const int splits = fill == 0 ? 1 : (int)std::min<long long>(fill / tiles, steps / (2 * s.kg));
      if (splits <= last) continue;
      last = splits;
      const int passes = (steps + splits * s.kg - 1) / (splits * s.kg);
      const long long wgs = tiles * splits;
      // several workgroups a CU share it; the last round counts whole while rounds are few
      const float turns = wgs <= 256 ? s.one : s.many * (wgs < 2048 ? (float)((wgs + 255) / 256) : (float)wgs / 256);
      float us = 5.f + passes * turns;
      if (splits > 1) us += 4.5f + (float)wgs * s.bm * s.bn * 8 / 8e6f;
      if (us < best.us) best = {i, (int)std::min<long long>(tiles, 1 << 30), splits, us};
    }
  }
  return best;
}

template <bool BF, bool GATED, Form F>
hipError_t launch_plan(const Mx4Args& a, const Plan& p, float* part, hipStream_t st) {
  switch (p.shape) {
    case 0: return launch<BF, GATED, F, 1, 2, 4, 3, 4, 2>(a, p.splits, part, st);
    case 1: return launch<BF, GATED, F, 2, 2, 4, 3, 4, 2>(a, p.splits, part, st);
    case 2: return launch<BF, GATED, F, 4, 2, 4, 2, 2, 1>(a, p.splits, part, st);
    default: return launch<BF, GATED, F, 4, 4, 4, 2, 2, 1>(a, p.splits, part, st);
  }
}

}  // namespace

bool mx4_takes_tiles(int m, int n, int k, long long ldx, bool gated) {
  if (ldx >= (1 << 24)) return false;  // a row's place in its tile is a 31-bit byte offset
  if (m > 16) return true;
  const int outside = mx4_rows_outside(m, k, gated);
  if (outside == 0) return false;
  // few rows, too long for the LDS: by the stream (5.5 TB/s) and what comes from memory for every block of a CU.  4096 channels x 14336
  // columns x 6, 10 and 16 rows take 10.6, 13.9 and 17.9 us (tiles 12.4 to 12.6), 2048 x 5464 x 16 6.5 (8.5), 20000 x 8192 x 16 34.9 (24.1).
  const float mb = (gated ? 2 : 1) * 0.53f * n * (k * 1e-6f);
  return plan(m, n, k, gated).us < 2.5f + mb / 5.5f + 0.45f * outside * ((mx4_blocks(n) + 255) / 256);
}

size_t mx4_tiles_workspace(int m, int n, int k, bool gated) {
  const Plan p = plan(m, n, k, gated);
  return p.splits > 1 ? (size_t)p.tiles * p.splits * SHAPES[p.shape].bm * SHAPES[p.shape].bn * 4 : 0;
}

t2w_mx4_form mx4_tiles_form(int m, int n, int k, bool gated) {
  const Plan p = plan(m, n, k, gated);
  return {SHAPES[p.shape].bm, SHAPES[p.shape].bn / (gated ? 2 : 1), p.splits};
}

hipError_t mx4_tiles(const Mx4Args& a, bool bf, bool gated, Form form, void* workspace, hipStream_t st) {
  const Plan p = plan(a.m, a.n, a.k, gated);
  return mx4_dispatch(bf, gated, form, [&](auto b, auto g, auto f) {
    return launch_plan<decltype(b)::value, decltype(g)::value, decltype(f)::value>(a, p, (float*)workspace, st);
  });
}

}  // namespace t2w
