// Rotary positions of several axes (time, height, width): pair p of a head turns by pos[axis[p]][token] * inv_freq[p].
//
// The angle is computed in turns as 64-bit fixed point: freq[p] is inv_freq[p] / 2 pi in units of 2^-64 turns (wrapped), an integer
// product wraps whole turns away by itself, and its upper 32 bits are the angle to 2^-32 turns at every int32 position.  Sine and
// cosine take it in fp32, which rounds it by at most 2^-26 turns (10^-7 radians, less than their own error), at any position alike;
// fp32 products lose the angle of far positions (position 10^6 at frequency 1: 0.06 radians).
//
// Bound by memory: 37,433 tokens of 40 heads x 128 take 140 us (5.4 TB/s read and written; a copy of that size 5.2).  A lane keeps its
// eight pairs' sines and cosines for all heads of its token: computed for each head they would be most of the work.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/t2w.h"
#include "common.h"
#include "rows_overlap.h"

namespace t2w {

int set_error(const char* what, hipError_t e);

namespace {

// Lanes: rot / 16 lanes a head, each 8 pairs (16 channels); a wave turns 64 / LPH heads of one token at a time.
template <bool BF, bool HALVES>
__global__ __launch_bounds__(256) void rope_kernel(const t2w_rope_args a, int head_splits) {
  const int lane = threadIdx.x & 63, lph = a.rot >> 4, sub = lane / lph, i = lane - sub * lph, hpw = 64 / lph;
  const int wid = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int total = (int)gridDim.x * 4;
  if (sub >= hpw) return;
  const int heads = a.q_heads + a.k_heads, at0 = HALVES ? 8 * i : 16 * i, at1 = HALVES ? 8 * i + (a.rot >> 1) : 16 * i + 8;
  uint64_t freq[8];
  int axis[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) freq[e] = a.freq[8 * i + e], axis[e] = min((int)a.axis[8 * i + e], a.n_axes - 1);
  for (int item = wid; item < a.n_tok * head_splits; item += total) {
    const int tok = item / head_splits, split = item - tok * head_splits;
    const auto source = [&](int h) {
      return h < a.q_heads ? (const uint16_t*)a.q + (long long)tok * a.ldq + h * a.head_dim
                           : (const uint16_t*)a.k + (long long)tok * a.ldk + (h - a.q_heads) * a.head_dim;
    };
    int h = split * hpw + sub;
    if (h >= heads) continue;
    // a head's channels are on their way while the angles, then while the head before are worked on
    const uint16_t* src = source(h);
    uint4 u0 = *(const uint4*)(src + at0), u1 = *(const uint4*)(src + at1);
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t p = a.pos[(long long)axis[e] * a.ld_pos + tok];
      const int32_t turn = (int32_t)((uint64_t)p * freq[e] >> 32);
      sincospif((float)turn * 0x1p-31f, &sn[e], &cs[e]);
      sn[e] *= a.scale, cs[e] *= a.scale;
    }
    while (true) {
      const int next = h + head_splits * hpw;
      const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
      const uint16_t* here = src;
      if (next < heads) {
        src = source(next);
        u0 = *(const uint4*)(src + at0), u1 = *(const uint4*)(src + at1);
      }
      uint16_t* dst = h < a.q_heads ? (uint16_t*)a.q_out + (long long)tok * a.ldq_out + h * a.head_dim
                                    : (uint16_t*)a.k_out + (long long)tok * a.ldk_out + (h - a.q_heads) * a.head_dim;
      float v[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[2 * e] = BF ? lo2f(w[e]) : lo2h(w[e]), v[2 * e + 1] = BF ? hi2f(w[e]) : hi2h(w[e]);
      float o[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c0 = HALVES ? e : 2 * e, c1 = HALVES ? e + 8 : 2 * e + 1;
        o[c0] = v[c0] * cs[e] - v[c1] * sn[e];
        o[c1] = v[c0] * sn[e] + v[c1] * cs[e];
      }
      uint32_t r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = BF ? pack2(o[2 * e], o[2 * e + 1]) : pack2h(o[2 * e], o[2 * e + 1]);
      *(uint4*)(dst + at0) = make_uint4(r[0], r[1], r[2], r[3]);
      *(uint4*)(dst + at1) = make_uint4(r[4], r[5], r[6], r[7]);
      if (here != dst)
        for (int c = a.rot + 8 * i; c < a.head_dim; c += 8 * lph) *(uint4*)(dst + c) = *(const uint4*)(here + c);
      if (next >= heads) break;
      h = next;
    }
  }
}

hipError_t rope_launch(const t2w_rope_args& a, hipStream_t st) {
  const int hpw = 64 / (a.rot >> 4), turns = (a.q_heads + a.k_heads + hpw - 1) / hpw;
  // A token's heads go to waves of their own while there are few tokens, though each wave then computes the angles: 64 tokens of 40
  // heads x 128 take 3.9 us (one wave a token: 5.0), 500 5.3 (5.4), 1000 8.0 (6.1); of 32 heads x 64 3.6 (3.9), 3.8 (4.1), 4.5 (4.4).
  const int splits = a.n_tok <= 512 ? turns : 1;
  const long long waves = (long long)a.n_tok * splits;
  const unsigned grid = (unsigned)((waves + 3) / 4 < 8192 ? (waves + 3) / 4 : 8192);
  const bool halves = a.pairs == T2W_ROPE_HALVES;
  if (a.dtype == T2W_ROPE_BF16) {
    if (halves) rope_kernel<true, true><<<grid, 256, 0, st>>>(a, splits);
    else rope_kernel<true, false><<<grid, 256, 0, st>>>(a, splits);
  } else {
    if (halves) rope_kernel<false, true><<<grid, 256, 0, st>>>(a, splits);
    else rope_kernel<false, false><<<grid, 256, 0, st>>>(a, splits);
  }
  return hipGetLastError();
}

// what a call may not be, null if nothing
const char* rope_check(const t2w_rope_args& a) {
  if (a.dtype != T2W_ROPE_BF16 && a.dtype != T2W_ROPE_FP16) return "rope: dtype must be bf16 or fp16";
  if (a.pairs != T2W_ROPE_HALVES && a.pairs != T2W_ROPE_NEIGHBOURS) return "rope: pairs must be halves or neighbours";
  if (a.head_dim < 16 || a.head_dim > 1024 || a.head_dim % 8) return "rope: head_dim must be 16 to 1024, a multiple of 8";
  if (a.rot < 16 || a.rot > a.head_dim || a.rot % 16) return "rope: rotated channels must be 16 to head_dim, a multiple of 16";
  if (a.n_tok < 0 || a.n_tok > (1 << 24)) return "rope: at most 2^24 tokens";
  if (a.q_heads < 0 || a.k_heads < 0 || a.q_heads > 4096 || a.k_heads > 4096) return "rope: at most 4096 heads";
  // one row for all axes (text) has stride 0; rows that overlap in part are taken for a mistake
  if (a.n_axes < 1 || a.n_axes > 16 || (a.n_axes > 1 && a.ld_pos != 0 && a.ld_pos < a.n_tok)) return "rope: 1 to 16 axes, their positions in rows of n_tok";
  if (!std::isfinite(a.scale)) return "rope: scale must be finite";
  if (a.n_tok == 0 || a.q_heads + a.k_heads == 0) return nullptr;
  if (!a.freq || !a.axis || !a.pos) return "rope: null table or positions";
  const struct { const void* p; const void* o; long long ld, ldo; int h; } t[2] = {{a.q, a.q_out, a.ldq, a.ldq_out, a.q_heads}, {a.k, a.k_out, a.ldk, a.ldk_out, a.k_heads}};
  for (const auto& x : t) {
    if (!x.h) continue;
    if (!x.p || !x.o) return "rope: null heads";
    if (((uintptr_t)x.p & 15) || ((uintptr_t)x.o & 15) || x.ld % 8 || x.ldo % 8) return "rope: rows must be 16-byte aligned, their strides multiples of 8";
    const long long w = (long long)x.h * a.head_dim;
    if (a.n_tok > 1 && (x.ld < w || x.ldo < w)) return "rope: token rows overlap";
  }
  // an output may be its own input (the same rows) and meets nothing else
  for (int i = 0; i < 2; ++i) {
    if (!t[i].h) continue;
    const Rows out{t[i].o, t[i].ldo * 2, (long long)t[i].h * a.head_dim * 2, a.n_tok};
    if (i == 1 && t[0].h && rows_meet(out, Rows{t[0].o, t[0].ldo * 2, (long long)t[0].h * a.head_dim * 2, a.n_tok})) return "rope: the outputs overlap";
    for (int j = 0; j < 2; ++j) {
      if (!t[j].h) continue;
      if (i == j && t[i].p == t[i].o && (t[i].ld == t[i].ldo || a.n_tok == 1)) continue;
      if (rows_meet(out, Rows{t[j].p, t[j].ld * 2, (long long)t[j].h * a.head_dim * 2, a.n_tok})) return "rope: an output overlaps an input";
    }
    for (int j = 0; j < a.n_axes; ++j)
      if (rows_meet(out, Rows{a.pos + j * a.ld_pos, 4LL * a.n_tok, 4LL * a.n_tok, 1})) return "rope: an output overlaps the positions";
  }
  return nullptr;
}

}  // namespace

}  // namespace t2w

extern "C" int t2w_rope(const t2w_rope_args* a, void* stream) {
  using namespace t2w;
  if (!a) return set_error("rope: null arguments", hipSuccess);
  if (const char* e = rope_check(*a)) return set_error(e, hipSuccess);
  if (a->n_tok == 0 || a->q_heads + a->k_heads == 0) return 0;
  const hipError_t e = rope_launch(*a, (hipStream_t)stream);
  return e == hipSuccess ? 0 : set_error("rope", e);
}
