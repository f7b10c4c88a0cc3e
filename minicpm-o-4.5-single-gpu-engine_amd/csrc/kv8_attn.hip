// Attention over the paged 8-bit key/value cache: out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that query
// i sees, key and value codes times their blocks' scales.  Block format: kv8_internal.h.
#include "kv8_internal.h"

#include <atomic>
#include <cmath>
#include <type_traits>

namespace t2w {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// Work of one launch.  A tile is `tt` tokens of a row, its packed rows (token, query head of the group), m = token * G +
// head, sharing one key head; a part is a run of key blocks of a tile's row.
struct KV8Split {
  int G;        // query heads of a key head
  int tt;       // tokens of a tile
  int per_row;  // tile slots of a row, 0: tiles listed over all rows (find_tile)
  int n_tiles;  // tile slots of the call
  int bps;      // key blocks of a part, more where a row would have over `parts` of them
  int parts;    // most parts of a tile; 1: the kernel writes the outputs itself
  int cap;      // tile form: (tile, key head, part)s that the workspace holds, whatever the number of tiles; 0: all of `parts`
  float cm;     // scale log2(e) = cm 2^ce, cm in [0.72, 1.45): the product itself may leave fp32's range, or its normal one
  int ce;
};

// Workspace of split calls, parts joined by kv8_join_kernel: the parts' outputs, fp32 [tile slot][kv head][part][m][D],
// then (maximum, sum) [tile slot][kv head][part][m][2].
__host__ __device__ __forceinline__ size_t part_rows(const KV8Split& s, int kv_heads) {
  return (s.cap > 0 ? (size_t)s.cap : (size_t)s.n_tiles * kv_heads * s.parts) * (s.tt * s.G);
}

struct Tile {
  int row, start, i0, rows;  // its row, the row's first token, the tile's first token in it, packed rows
  int cached, n_new, total;  // total = cached + n_new keys; cached < 0 where the row has fewer keys than queries
  int end;                   // keys [0, end) are visible to some query of the tile
  int slot, parts;           // its slot, and its most parts
  bool bad;                  // the row is longer than its table, or than max_new tokens: NaN outputs
};

// The tile of a slot, by the whole wave; false: nothing there.
__device__ __forceinline__ bool find_tile(const t2w_kv8_attention_args& a, const KV8Split& s, int slot, Tile& t) {
  int at, next, live = 1;  // live: the call's tiles, where s.cap asks for them
  if (s.per_row > 0) {
    t.row = slot / s.per_row;
    at = slot - t.row * s.per_row;
    t.start = a.row_start[t.row];
    next = a.row_start[t.row + 1];
    t.total = a.kv_total[t.row];
  } else if (a.n_rows <= 64) {
    // All rows at once, one a lane.  Slots go by the tile's place in its row, the last ones first: the tiles of a causal
    // prompt that see most start first.  With N(x) the tiles at place x or later, slot s is at the largest x with N(x) > s.
    const int lane = threadIdx.x & 63, r = min(lane, a.n_rows - 1);
    const int start = a.row_start[r], stop = a.row_start[r + 1], total = a.kv_total[r];
    const int tiles = lane < a.n_rows && stop > start ? min((stop - start - 1) / s.tt + 1, 1 << 24) : 0;
    auto from = [&](int x) { return __builtin_amdgcn_readlane(wave_scan(max(tiles - x, 0)), 63); };
    live = from(0);
    if (live <= slot) return false;
    int lo = 0, hi = s.n_tiles + 1;  // no row has more tiles than the call has slots
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (from(mid) > slot) lo = mid; else hi = mid;
    }
    const uint64_t have = __builtin_amdgcn_ballot_w64(tiles > lo);
    const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0));
    const int nth = slot - from(lo + 1);  // of the rows with a tile there
    t.row = min((int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(tiles > lo && rank == nth) | (1ull << 63)), a.n_rows - 1);
    t.start = __builtin_amdgcn_readlane(start, t.row);
    next = __builtin_amdgcn_readlane(stop, t.row);
    t.total = __builtin_amdgcn_readlane(total, t.row);
    at = lo;
  } else if (s.cap > 0) {
    // More rows, the tiles counted, the last rows' last ones first: each lane sums a run of rows, then the rows of the run
    // that holds the tile go one to a lane.
    const int lane = threadIdx.x & 63, step = (a.n_rows + 63) / 64;
    auto tiles_of = [&](int r) {
      if (r >= a.n_rows) return 0;
      const int start = a.row_start[r], stop = a.row_start[r + 1];
      return stop > start ? min((stop - start - 1) / s.tt + 1, 1 << 18) : 0;  // at most 128 where starts are well formed: no sum wraps
    };
    int mine = 0;
    for (int i = 0; i < step; ++i) mine += tiles_of(lane * step + i);
    const int upto = wave_scan(mine);
    live = __builtin_amdgcn_readlane(upto, 63);
    if (live <= slot) return false;
    const int back = live - 1 - slot, run = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > back) | (1ull << 63));
    const int n = lane < step ? tiles_of(run * step + lane) : 0, to = wave_scan(n) + __builtin_amdgcn_readlane(upto - mine, run);
    const int nth = __builtin_ctzll(__builtin_amdgcn_ballot_w64(to > back) | (1ull << 63));
    t.row = min(run * step + nth, a.n_rows - 1);
    at = back - __builtin_amdgcn_readlane(to - n, nth);
    t.start = a.row_start[t.row];
    next = a.row_start[t.row + 1];
    t.total = a.kv_total[t.row];
  } else {  // the last rows' last tiles first
    const int back = s.n_tiles - 1 - slot;
    t.row = kv8_find_row(a.row_start, a.n_rows, s.tt, 1, back);
    t.start = a.row_start[t.row];
    next = a.row_start[t.row + 1];
    t.total = a.kv_total[t.row];
    at = back - (t.start / s.tt + t.row);
  }
  // the same in every lane, which the compiler does not see on every way here
  t.row = __builtin_amdgcn_readfirstlane(t.row);
  t.start = __builtin_amdgcn_readfirstlane(t.start);
  t.n_new = __builtin_amdgcn_readfirstlane(next) - t.start;
  t.total = __builtin_amdgcn_readfirstlane(t.total);
  at = __builtin_amdgcn_readfirstlane(at);
  t.i0 = at * s.tt;
  if (t.start < 0 || t.n_new <= 0 || t.start > a.n_tok - t.n_new || at < 0 || t.i0 >= t.n_new) return false;
  t.bad = t.total < 0 || t.total > a.width * KV8_BLOCK || (s.per_row > 0 && t.n_new > s.per_row * s.tt);
  const int n = min(s.tt, t.n_new - t.i0);
  t.rows = n * s.G;
  t.cached = t.total - t.n_new;
  const int last = t.i0 + n - 1;
  const int seen = a.chunk > 0 ? (int)min((long long)t.n_new, ((long long)(last / a.chunk) + 1) * a.chunk) : t.n_new;
  t.end = max(t.cached + seen, 0);
  t.slot = slot;
  t.parts = s.cap > 0 ? min(s.parts, max(1, s.cap / a.pages.kv_heads / live)) : s.parts;  // slot < live: all partials lie within s.cap
  return true;
}

// keys that query i (a token of the tile's row) sees
__device__ __forceinline__ int seen_by(const t2w_kv8_attention_args& a, const Tile& t, int i) {
  const int seen = a.chunk > 0 ? (int)min((long long)t.n_new, ((long long)(i / a.chunk) + 1) * a.chunk) : t.n_new;
  return max(t.cached + seen, 0);
}

// parts of a tile and the blocks of one
__device__ __forceinline__ int tile_parts(const KV8Split& s, const Tile& t, int& per) {
  const int nb = (t.end + KV8_BLOCK - 1) / KV8_BLOCK;
  per = max(s.bps, (nb + t.parts - 1) / t.parts);
  return max(1, (nb + per - 1) / per);
}

// NaN to the tile's outputs, by `threads` threads; to the whole row's where it has more tokens than the bound
template <bool BF, int D>
__device__ void nan_tile(const t2w_kv8_attention_args& a, const KV8Split& s, const Tile& t, int kv_head, int thread, int threads) {
  const int n = s.per_row > 0 && t.n_new > s.per_row * s.tt ? t.n_new : t.rows / s.G;
  for (int i = 0; i < n; ++i)
    for (int x = thread; x < s.G * D; x += threads)
      ((uint16_t*)a.out)[(long long)(t.start + t.i0 + i) * a.ldo + kv_head * s.G * D + x] = BF ? 0x7fc0 : 0x7e00;
}

__device__ __forceinline__ f16x8 as_f16x8(uint4 v) { return __builtin_bit_cast(f16x8, v); }

__device__ __forceinline__ bf16x8 codes_bf16(uint32_t lo, uint32_t hi) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  return as_bf16x8(make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)));
}
// codes times a power of two
__device__ __forceinline__ f16x8 codes_f16(uint32_t lo, uint32_t hi, float s) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, true);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, true);
  return as_f16x8(make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)));
}

// K . Q^T of 8 key codes a lane and the query operand in the queries' own type: e4m3 codes are exact in both
template <bool BF>
__device__ __forceinline__ f32x4 mfma_qk(uint32_t lo, uint32_t hi, uint4 q, f32x4 c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_bf16(lo, hi), as_bf16x8(q), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16(lo, hi, 1.f), as_f16x8(q), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ f32x16 mfma_qk(uint32_t lo, uint32_t hi, uint4 q, f32x16 c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(codes_bf16(lo, hi), as_bf16x8(q), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_f16(lo, hi, 1.f), as_f16x8(q), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_pv(f16x8 v, f16x8 p, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma_pv(f16x8 v, f16x8 p, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p, c, 0, 0, 0); }

// maximum over the lanes that hold the same query: lanes l, l ^ 32 (32-query tiles) and l ^ 16 (16-query tiles).  Through
// the LDS crossbar: it runs only when the reference moves, and hipcc drops the maximum of a v_permlane32_swap's two results.
template <int MR>
__device__ __forceinline__ float query_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 32, 64));
  if constexpr (MR == 16) v = fmaxf(v, __shfl_xor(v, 16, 64));
  return v;
}

// Exponent bytes of a block, in scalar registers: an E8M0 NaN among the values' is one among the keys', whose NaN scores reach
// who sees the block and nobody else, and counts for no unit
__device__ __forceinline__ void nan_scales(int& kx, int& vx) {
  kx = vx == 255 ? 255 : kx;
  vx = kx == 255 ? -1 : vx;
}

__device__ __forceinline__ float pow2_bits(int biased) { return __uint_as_float((uint32_t)min(max(biased, 0), 254) << 23); }

// Softmax and output state of a wave's MR packed rows (lane column = query), shared by both kernels.  Scores are in units of
// log2, s = q . k times c = scale log2(e) 2^(key exponent), a normal number or applied to the scores themselves (scale_scores).
//  * m is a reference that the running maximum may pass by 8 before it is moved (then to the true maximum so far):
//    probabilities are 2^(s - m + 7) <= 2^15 in fp16, so most blocks need no exchange between lanes and no rescaling of the
//    outputs, and a probability keeps fp16's 11 bits down to 2^-21 of the largest and 2^-32 of it absolutely.  fp16 and not
//    bf16: bf16's 8 bits would cost as much again as the output's own rounding.
//  * value codes enter as fp16, exact, times 2^(their exponent - E + 7), E the largest value exponent so far, while the exponents
//    span at most NEAR; a block that nobody sees yet can change nothing but E, which scales o exactly.
//  * from the first block on that lies further apart (`wide`) the scale is a part of the weight: the operands of P . V are
//    2^(s - m + exponent - k + 7) <= 2^15 and the codes times 2^7, with k a reference of each query that moves as m does.  What
//    counts is then a term's own size, p times its scale, however far scales lie apart: a block of large values and no weight
//    takes no bits from the others, nor the other way round.  l takes its exponentials in fp32 there.
//  * a weight is off by 2^-12 of it or by 2^-25, half of fp16's smallest step, where the largest is 2^7 and more (2^(7 - NEAR)
//    of those before the exponents span more than that): 2^-32 of the largest p times scale, 2^-22 at worst, a key.
//  * sums of probabilities are of the same rounded fp16 values as the outputs' (fp32 dot products, a lane its own keys').
constexpr int NEAR = 10;

constexpr int WIDE = 1 << 20;    // in place of a value unit: exponents lie far apart

// Value exponents (biased) of the blocks so far, -1 where one counts for nobody.  The unit that the block's values need:
// the largest of them, or WIDE from where they span more than NEAR on.
struct Units {
  int hi = -1;
  unsigned lo = 255;
  __device__ __forceinline__ int add(int e) {
    hi = max(hi, e);
    lo = min(lo, (unsigned)e);
    return hi - (int)lo > NEAR ? WIDE : hi;
  }
  // exponent of the factor of the block's codes, 7 above what its values are in units of it
  static __device__ __forceinline__ int factor(int e, int unit) { return (unit == WIDE ? 0 : e - unit) + 127 + 7; }
};

template <int MR, int D>
struct State {
  static constexpr int AR = MR == 16 ? 4 : 16;     // values of an accumulator
  static constexpr int KG = MR == 16 ? 2 : 1;      // score tiles of a block
  static constexpr int NP = MR == 16 ? 1 : 2;      // probability operands of a block
  static constexpr int NT = D / (2 * MR);          // output tile pairs: channels 2 p and 2 p + 1, p = MR t + i
  typedef typename std::conditional<MR == 16, f32x4, f32x16>::type Acc;
  Acc o[NT][2];
  float l = 0.f;                // sum of the lane's probabilities; of the query's when the lane groups are added
  float m = -__builtin_inff();  // reference
  float nb = 7.f;               // 7 - m, 7 where m is -inf; 0 where `big`; -k where `wide`
  bool big = false;             // some query of the wave has a large |m|
  int E = -1;                   // biased value exponent that o is in units of (0 is 2^-127); -1: none yet
  bool wide = false;            // value exponents lie far apart: o is in units of 2^k, each query's own
  uint32_t one = 0x3c003c00;    // a pair of fp16 ones, for the sums of probabilities; zeros where `wide`
  bool slow = false;            // big or wide: `move` computes the exponentials' arguments itself

  __device__ __forceinline__ State() {
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < AR; ++r) o[x][j][r] = 0.f;
  }
  __device__ __forceinline__ void scale_o(float f) {
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < AR; ++r) o[x][j][r] *= f;
  }
  // key of score r of tile x within its block
  static __device__ __forceinline__ int key_of(int x, int r, int g) { return MR == 16 ? 8 * g + 4 * x + r : 16 * (r >> 3) + 8 * g + (r & 7); }

  static __device__ __forceinline__ float top(const Acc (&sc)[KG]) {
    float mx = sc[0][0];
#pragma unroll
    for (int x = 0; x < KG; ++x)
#pragma unroll
      for (int r = 0; r < AR; ++r) mx = fmaxf(mx, sc[x][r]);
    return mx;
  }
  // A block's factor c = cm 2^ex is a normal number for |ex| <= NORMAL; where it is not, its scores are scaled themselves, in
  // fp32's whole range (a factor of 0 would make NaN of an invisible score's -inf).
  static constexpr int NORMAL = 125;
  static __device__ __forceinline__ void scale_scores(Acc (&sc)[KG], float cm, int ex) {
#pragma unroll
    for (int x = 0; x < KG; ++x)
#pragma unroll
      for (int r = 0; r < AR; ++r) sc[x][r] = __builtin_amdgcn_ldexpf(sc[x][r] * cm, ex);
  }
  // Scores of keys from `lim` on are -inf, the others NaN where `off`.
  static __device__ __forceinline__ void mask(Acc (&sc)[KG], bool off, int key0, int lim, int g) {
#pragma unroll
    for (int x = 0; x < KG; ++x)
#pragma unroll
      for (int r = 0; r < AR; ++r) sc[x][r] = key0 + key_of(x, r, g) < lim ? (off ? __builtin_nanf("") : sc[x][r]) : -__builtin_inff();
  }
  // (Branches that few blocks take are marked unlikely, out of the loops' way: 1,106 -> 1,095 us on the long chunk.)
  // Moves the reference where a block's scores, in units 1 / c and -inf where invisible, of maximum mx, pass it.  Where |m| is
  // large, s - m + 7 in one fma is not what the scores' own rounding allows: 7 - m rounds too, and a score of m + 8 could reach
  // 2^16, infinite in fp16.  There s is rounded first, as mx was, and s - m is exact where it counts; nothing may be contracted.
  // Each query by its own m alone, so that its bits do not depend on the others of the wave.
  __device__ __forceinline__ void move(Acc (&sc)[KG], float& c, float mx, int vx, int e) {
#pragma clang fp contract(off)
    mx *= c;
    // one comparison for both: some maximum passes the reference by 8, or the unit rises (then every lane's does)
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(fmaxf(mx - m, -1.f) > (e > E ? -2.f : 8.f)) != 0, 0)) {
      nb = e == WIDE && !wide ? -(float)E : nb;
      wide = wide || e == WIDE;
      const bool up = !wide && e > E;
      float seen = mx;
      if (wide || __builtin_amdgcn_ballot_w64(mx - m > 8.f)) seen = query_max<MR>(mx);
      const float mn = seen - m > 8.f ? seen : m;  // each query by its own scores alone
      const float alpha = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      big = big || __builtin_amdgcn_ballot_w64(large(mn)) != 0;
      // wide: scores count from mn now, and k with them; then k moves to the largest weight where that passes it by 8
      const float n = nb + (mn == m ? 0.f : fminf(mn - m, 1e30f)), need = mn == -__builtin_inff() ? -1e30f : seen - mn + (float)vx;
      const float nk = need + n > 8.f ? -need : n;
      const float f = wide ? __builtin_amdgcn_exp2f(nk - n) : up ? (E < 0 ? 0.f : alpha * pow2_bits(E - e + 127)) : alpha;
      nb = wide ? nk : big ? 0.f : mn == -__builtin_inff() ? 7.f : 7.f - mn;
      E = up ? e : E;
      slow = big || wide;
      one = wide ? 0 : one;  // `move` sums them, below
      m = mn;
      l *= alpha;
      scale_o(f);
    }
    if (__builtin_expect(slow, 0)) {
      const float m0 = m == -__builtin_inff() ? 0.f : m, add = wide ? (float)vx : 0.f;
      const bool own = large(m0);
#pragma unroll
      for (int x = 0; x < KG; ++x)
#pragma unroll
        for (int r = 0; r < AR; ++r) {
          const float s = sc[x][r] * c, arg = own ? (s - m0) + 7.f : fmaf(sc[x][r], c, 7.f - m0);
          if (wide) l += __builtin_amdgcn_exp2f(arg);
          sc[x][r] = arg + add;
        }
      c = 1.f;
    }
  }
  static __device__ __forceinline__ bool large(float m) { return fabsf(m) > 4194304.f && m != -__builtin_inff(); }
  // a block's probabilities, the operands of P . V
  __device__ __forceinline__ void exps(const Acc (&sc)[KG], float c, f16x8 (&p)[NP]) const {
#pragma unroll
    for (int x = 0; x < NP; ++x)
#pragma unroll
      for (int z = 0; z < 8; z += 2) {
        float e[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const float s = MR == 16 ? sc[(z + w) / 4 % KG][(z + w) % 4] : sc[0][8 * x + z + w];
          e[w] = __builtin_amdgcn_exp2f(fmaf(s, c, nb));
        }
        const f16x2_t h = __builtin_convertvector((f32x2_t{e[0], e[1]}), f16x2_t);
        p[x][z] = h[0];
        p[x][z + 1] = h[1];
      }
  }
  __device__ __forceinline__ void sum(f16x8 p) {
#pragma unroll
    for (int z = 0; z < 8; z += 2) l = __builtin_amdgcn_fdot2(f16x2_t{p[z], p[z + 1]}, __builtin_bit_cast(f16x2_t, one), l, false);
  }

  // the other state of the same rows, left in LDS by another wave (`put`), folded into this one
  static constexpr int WORDS = NT * 2 * AR + 3;
  __device__ __forceinline__ int unit() const { return wide ? WIDE : E; }
  __device__ __forceinline__ void put(float (*dst)[64], int lane) const {
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < AR; ++r) dst[(x * 2 + j) * AR + r][lane] = o[x][j][r];
    dst[WORDS - 3][lane] = m;
    dst[WORDS - 2][lane] = l;
    dst[WORDS - 1][lane] = nb;
  }
  __device__ __forceinline__ void fold(const float (*src)[64], int e2, int lane) {
    const float m2 = src[WORDS - 3][lane], l2 = src[WORDS - 2][lane];
    const float mn = fmaxf(m, m2);
    const float f1 = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    const float f2 = m2 == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m2 - mn);
    float g1, g2;
    if (!wide && e2 != WIDE && (E < 0 || e2 < 0 || abs(E - e2) <= 60)) {
      const int en = max(E, e2);
      g1 = E == en ? f1 : f1 * (E < 0 ? 0.f : pow2_bits(E - en + 127));
      g2 = e2 == en ? f2 : f2 * (e2 < 0 ? 0.f : pow2_bits(e2 - en + 127));
      E = en;
    } else {  // each query's unit: the larger one, as above, or where they lie far apart that of the larger weight times scale
      float k1 = wide ? -nb : (float)E, k2 = e2 == WIDE ? -src[WORDS - 1][lane] : (float)e2;
      k1 = m == -__builtin_inff() ? k2 : k1;
      k2 = m2 == -__builtin_inff() ? k1 : k2;
      const bool near = fabsf(k1 - k2) <= 60.f;
      const float a1 = near ? k1 : (m - mn) + k1, a2 = near ? k2 : (m2 - mn) + k2, kn = fmaxf(a1, a2);
      g1 = (near ? f1 : 1.f) * __builtin_amdgcn_exp2f(a1 - kn);
      g2 = (near ? f2 : 1.f) * __builtin_amdgcn_exp2f(a2 - kn);
      wide = true;
      nb = -kn;
    }
    l = l * f1 + l2 * f2;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < AR; ++r) o[x][j][r] = o[x][j][r] * g1 + src[(x * 2 + j) * AR + r][lane] * g2;
    m = mn;
  }

  // Row mrow of the tile (lane group g): to the outputs, or to the call's workspace where the tile has several parts
  template <bool BF>
  __device__ __forceinline__ void store(const t2w_kv8_attention_args& a, const KV8Split& sp, const Tile& t, int kv_head, int part, int parts,
                                        int mrow, int g) const {
    float sum = l + __shfl_xor(l, 32, 64);
    if constexpr (MR == 16) sum += __shfl_xor(sum, 16, 64);
    float inv = sum == 0.f ? 0.f : 1.f / sum;
    int unit = E - 127 - 7;  // o counts 2^unit
    if (wide) {
      const float k = fmaxf(-nb, -1000.f), whole = rintf(k);
      unit = (int)whole - 127 - 7;
      inv *= __builtin_amdgcn_exp2f(k - whole);
    }
    // values r .. r + 3 of both tiles of a pair are 8 consecutive channels, from d on
    if (parts == 1) {
      const int tok = mrow / sp.G, hq = mrow - tok * sp.G;
      uint16_t* out = (uint16_t*)a.out + (long long)(t.start + t.i0 + tok) * a.ldo + (kv_head * sp.G + hq) * D;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int r = 0; r < AR; r += 4) {
          const int d = MR == 16 ? 32 * x + 8 * g : 64 * x + 4 * r + 8 * g;
          uint32_t w[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float u = __builtin_amdgcn_ldexpf(o[x][0][r + y] * inv, unit), v = __builtin_amdgcn_ldexpf(o[x][1][r + y] * inv, unit);
            w[y] = BF ? pack2(u, v) : pack2h(u, v);
          }
          *(uint4*)(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
      const size_t pr = ((size_t)t.slot * a.pages.kv_heads + kv_head) * t.parts + part, rows = sp.tt * sp.G;
      float* po = (float*)a.workspace + (pr * rows + mrow) * D;
      float* ml = (float*)a.workspace + part_rows(sp, a.pages.kv_heads) * D + (pr * rows + mrow) * 2;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int r = 0; r < AR; r += 4) {
          const int d = MR == 16 ? 32 * x + 8 * g : 64 * x + 4 * r + 8 * g;
#pragma unroll
          for (int y = 0; y < 4; y += 2)
            *(float4*)(po + d + 2 * y) = make_float4(__builtin_amdgcn_ldexpf(o[x][0][r + y] * inv, unit), __builtin_amdgcn_ldexpf(o[x][1][r + y] * inv, unit),
                                                     __builtin_amdgcn_ldexpf(o[x][0][r + y + 1] * inv, unit), __builtin_amdgcn_ldexpf(o[x][1][r + y + 1] * inv, unit));
        }
      if (g == 0) *(float2*)ml = make_float2(m, sum);
    }
  }
};

// Direct form, for tiles of few packed rows (steps, draft checks, windows of up to 64 packed rows): every wave loads its key
// and value fragments from the pages into registers and converts them there; no LDS and no barrier before the end.  RW waves
// of MR packed rows each, times 4 / RW waves that take every (4 / RW)-th block; their states are merged through LDS.
//
// Bound by memory: 2 D codes a token and key head are read once and meet at least MR query columns of the matrix unit, whose
// unused columns cost nothing that matters (64 rows of up to 8,192 keys, 32 heads over 8 of 128: 735 MB in 137 us, 5.35 TB/s
// where a copy reaches 5.14 and reads alone 5.87).  One register set a block: the next block's keys load as soon as the
// scores have used these, its values after P . V; two sets spilled and took 221 us.  MR = 16 (16x16x32 MFMA) has half the
// softmax work of MR = 32 (32x32x16) where rows allow it.  Heads of 64 run four workgroups a CU, so that 1,024 workgroups of
// windows are all resident (64 rows of 50 tokens over 370 keys: 17.1 us; 16.5 against 19.7 with three a CU when both were built).
//
// With S^T = K . Q^T the score MFMA leaves a lane scores of its own query only; the rows of K are fed in an order that makes
// them the 8 (MR = 16) or 2 x 8 keys whose value bytes the same lane loads as the P . V operand:
//   MR 16: lane (i = l % 16, g = l / 16); key operand kg row i = key 8 (i / 4) + 4 kg + i % 4, its scores: keys 8 g + 4 kg + r
//   MR 32: lane (i = l % 32, g = l / 32); row i = key with bits 2 and 3 of i swapped, scores r: keys 16 (r / 8) + 8 g + r % 8
// Channels are paired the same way on both sides: lane group x loads the 16-channel chunk n x' + x of keys and queries.
template <bool BF, int D, int MR, int RW, int OCC>
__global__ void __launch_bounds__(256, OCC) kv8_attn_direct_kernel(t2w_kv8_attention_args a, KV8Split sp) {
  typedef State<MR, D> St;
  constexpr int KW = 4 / RW;                       // waves that share the keys of the same packed rows
  constexpr int LG = 64 / MR;                      // lane groups: 4 or 2
  constexpr int NQ = D / (8 * LG), NL = D / 32;    // query operands; 16-byte loads of a block's keys, and of its values
  constexpr int KG = St::KG, AR = St::AR, NP = St::NP;
  __shared__ float s_acc[KW / 2 * RW][St::WORDS][64];
  __shared__ int s_e[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % RW, kw = wave / RW;
  const int slot = blockIdx.x / a.pages.kv_heads, kv_head = blockIdx.x - slot * a.pages.kv_heads, part = blockIdx.y;
  // the first ids are under way with the row's lengths where its number is known and parts have their planned size
  const int ahead = part * sp.bps + kw;
  int id_ahead = 0;
  if (sp.per_row > 0 && ahead + lane * KW < a.width) id_ahead = a.table[(size_t)(slot / sp.per_row) * a.ld_table + ahead + lane * KW];
  Tile t;
  if (!find_tile(a, sp, slot, t)) return;
  if (t.bad) {
    if (part == 0) nan_tile<BF, D>(a, sp, t, kv_head, threadIdx.x, 256);
    return;
  }
  int per;
  const int parts = tile_parts(sp, t, per);
  if (part >= parts) return;
  const int b0 = part * per, b1 = min(b0 + per, (t.end + KV8_BLOCK - 1) / KV8_BLOCK);
  const int i = lane % MR, g = lane / MR;
  const int m0 = rw * MR;
  const bool idle = m0 >= t.rows;  // a wave without rows still meets the barriers
  const int mrow = m0 + i;
  const int tok = min(mrow, t.rows - 1) / sp.G, hq = min(mrow, t.rows - 1) - tok * sp.G;
  const int lim = seen_by(a, t, t.i0 + tok);
  const int lim_lo = seen_by(a, t, t.i0 + min(m0, t.rows - 1) / sp.G);  // the wave's first query sees least

  uint4 q[NQ];
  {
    const uint16_t* src = (const uint16_t*)a.q + (long long)(t.start + t.i0 + tok) * a.ldq + (kv_head * sp.G + hq) * D;
#pragma unroll
    for (int n = 0; n < NQ; ++n) q[n] = *(const uint4*)(src + (LG * (n >> 1) + g) * 16 + (n & 1) * 8);
  }
  St st;
  Units units;

  // the lane's place in a block's keys and values; its loads lie at constant distances from there (load offsets)
  const uint32_t koff = MR == 16 ? g * 512 + (8 * (i >> 2) + (i & 3)) * 16 : g * 512 + ((i & 0x13) | ((i & 4) << 1) | ((i & 8) >> 1)) * 16;
  const uint32_t voff = g * 8 * D + i * 16;
  const size_t stride = (size_t)a.pages.kv_heads * (KV8_BLOCK * D);
  const uint8_t* kbase = (const uint8_t*)a.pages.k + (size_t)kv_head * (KV8_BLOCK * D);
  const uint8_t* vbase = (const uint8_t*)a.pages.v + (size_t)kv_head * (KV8_BLOCK * D);
  const int* table = a.table + (size_t)t.row * a.ld_table;

  // one block's codes; the next block's keys are loaded as soon as the scores have used these, its values after P . V
  uint4 kf[NL], vf[NL];
  auto load_k = [&](int id) {
    const uint8_t* kp = kbase + (size_t)id * stride;
#pragma unroll
    for (int n = 0; n < NL; ++n) kf[n] = *(const uint4*)(kp + koff + (MR == 16 ? (n / 2) * 2048 + (n % 2) * 64 : n * 1024));
  };
  auto load_v = [&](int id) {
    const uint8_t* vp = vbase + (size_t)id * stride;
#pragma unroll
    for (int n = 0; n < NL; ++n) vf[n] = *(const uint4*)(vp + voff + (MR == 16 ? n * 256 : (n % 2) * 16 * D + (n / 2) * 512));
  };

  if (!idle) {
    // the wave's blocks b0 + kw, + KW, ...: ids and exponents of the next 64 of them one a lane
    for (int base = b0 + kw; base < b1; base += 64 * KW) {
      const int mine = base + lane * KW;
      int id = mine >= b1 ? 0 : sp.per_row > 0 && base == ahead ? id_ahead : table[mine], ke = 255, ve = -1;
      if ((unsigned)id < (unsigned)a.pages.n_blocks) {
        ke = a.pages.k_exp[(size_t)id * a.pages.kv_heads + kv_head];
        ve = a.pages.v_exp[(size_t)id * a.pages.kv_heads + kv_head];
      } else {
        id = 0;
      }
      const int n = min(64, (b1 - base + KW - 1) / KW);
      load_k(__builtin_amdgcn_readlane(id, 0));
      load_v(__builtin_amdgcn_readlane(id, 0));
      for (int x = 0; x < n; ++x) {
        int kx = __builtin_amdgcn_readlane(ke, x), vx = __builtin_amdgcn_readlane(ve, x);
        nan_scales(kx, vx);
        const int next = x + 1 < n ? __builtin_amdgcn_readlane(id, x + 1) : -1, key0 = (base + x * KW) * KV8_BLOCK;
        typename St::Acc sc[KG];
#pragma unroll
        for (int z = 0; z < KG; ++z)
#pragma unroll
          for (int r = 0; r < AR; ++r) sc[z][r] = 0.f;
#pragma unroll
        for (int w = 0; w < NL; ++w) {
          const int z = MR == 16 ? w % 2 : 0, j = MR == 16 ? w / 2 : w;
          sc[z] = mfma_qk<BF>(kf[w].x, kf[w].y, q[2 * j], sc[z]);
          sc[z] = mfma_qk<BF>(kf[w].z, kf[w].w, q[2 * j + 1], sc[z]);
        }
        if (next >= 0) load_k(next);
        const bool off = kx > 254;  // a block id outside the pages, or an E8M0 NaN
        const int ex = sp.ce + kx - 127;
        float c = __builtin_amdgcn_ldexpf(sp.cm, ex);
        if (__builtin_expect(max(key0 + KV8_BLOCK - lim_lo, kx - 254) > 0, 0)) St::mask(sc, off, key0, lim, g);  // or some query of the wave does not see all of the block
        if (__builtin_expect(abs(ex) > St::NORMAL, 0)) {
          St::scale_scores(sc, sp.cm, ex);
          c = 1.f;
        }
        if (off || key0 + KV8_BLOCK > t.total) {  // values behind the last token count as zeros, whatever they are
#pragma unroll
          for (int w = 0; w < NL; ++w) {
            const int left = off ? 0 : t.total - key0 - 8 * (MR == 16 ? g : 2 * (w % 2) + g);
            const uint64_t keep = left >= 8 ? ~0ull : left <= 0 ? 0ull : (1ull << (8 * left)) - 1ull;
            vf[w].x &= (uint32_t)keep; vf[w].y &= (uint32_t)(keep >> 32);
            vf[w].z &= (uint32_t)keep; vf[w].w &= (uint32_t)(keep >> 32);
          }
        }
        const int unit = units.add(vx);
        st.move(sc, c, St::top(sc), vx, unit);
        f16x8 p[NP];
        st.exps(sc, c, p);
#pragma unroll
        for (int w = 0; w < NP; ++w) st.sum(p[w]);
        const float vs = pow2_bits(Units::factor(vx, unit));
#pragma unroll
        for (int w = 0; w < NL; ++w) {
          const int z = MR == 16 ? w : w / 2, kk = MR == 16 ? 0 : w % 2;
          st.o[z][0] = mfma_pv(codes_f16(vf[w].x, vf[w].y, vs), p[kk], st.o[z][0]);
          st.o[z][1] = mfma_pv(codes_f16(vf[w].z, vf[w].w, vs), p[kk], st.o[z][1]);
        }
        if (next >= 0) load_v(next);
      }
    }
  }
  // merge the key waves pairwise: the upper half leaves its state, the lower half folds it in
#pragma unroll
  for (int w = KW / 2; w >= 1; w /= 2) {
    if (kw >= w && kw < 2 * w) {
      st.put(s_acc[(kw - w) * RW + rw], lane);
      if (lane == 0) s_e[wave] = st.unit();
    }
    __syncthreads();
    if (kw < w) st.fold(s_acc[kw * RW + rw], s_e[wave + w * RW], lane);
    if (w > 1) __syncthreads();
  }
  if (kw == 0 && mrow < t.rows) st.template store<BF>(a, sp, t, kv_head, part, parts, mrow, g);
}

// Tile form, for tiles of many packed rows (prompts): RW waves of 32 packed rows each share the keys, two blocks a step.  The
// workgroup loads a step's codes (one step ahead, in registers), converts them once, and leaves them in LDS as the MFMA
// operands; every wave then reads whole fragments, 16 consecutive bytes a lane.  Three LDS steps: one is read, the next one
// written, and with one barrier in the middle of a step no wave writes what another may still read of the step before.
//
// A 32x32x16 MFMA keeps the matrix unit for 32 cycles and the vector issue port for 16: four vector instructions behind each
// are free.  So a block's exponentials run between the next block's score MFMAs, and the conversion and the next maximum
// between the value MFMAs.  2,048 tokens over 32,000 (32 heads over 8 of 128, fp16, causal): 1,094 us, 1.01 PFLOP/s against
// 1.17 of a large library product on the same card; 44% of the cycles on the matrix unit, 42% issuing vector instructions,
// the LDS reads (16 KB a wave and block) about half.  Without the interleaving 1,190 us against 1,115 then; four waves and two
// workgroups a CU 1,174 against 1,096 in the same run.
template <bool BF, int D, int RW>
__global__ void __launch_bounds__(64 * RW, 2) kv8_attn_tile_kernel(t2w_kv8_attention_args a, KV8Split sp) {
  typedef State<32, D> St;
  constexpr int CB = 2 * D, T = 64 * RW;      // 16-byte code chunks of a block's keys, and of its values; threads
  constexpr int NC = 2 * CB / T;              // chunks of a step (two blocks) a thread
  extern __shared__ uint4 s_kv[];
  uint4 (*s_k)[2][2 * CB] = (uint4 (*)[2][2 * CB])s_kv, (*s_v)[2][2 * CB] = s_k + 3;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slot = blockIdx.x / a.pages.kv_heads, kv_head = blockIdx.x - slot * a.pages.kv_heads, part = blockIdx.y;
  Tile t;
  if (!find_tile(a, sp, slot, t)) return;
  if (t.bad) {
    if (part == 0) nan_tile<BF, D>(a, sp, t, kv_head, tid, T);
    return;
  }
  int per;
  const int parts = tile_parts(sp, t, per);
  if (part >= parts) return;
  const int b0 = part * per, b1 = min(b0 + per, (t.end + KV8_BLOCK - 1) / KV8_BLOCK), steps = (b1 - b0 + 1) / 2;
  const int i = lane & 31, g = lane >> 5;
  const int m0 = wave * 32, mrow = m0 + i, last = min(m0 + 31, t.rows - 1);
  const int tok = min(mrow, t.rows - 1) / sp.G, hq = min(mrow, t.rows - 1) - tok * sp.G;
  const int lim = min(seen_by(a, t, t.i0 + tok), b1 * KV8_BLOCK);
  const int lim_lo = min(seen_by(a, t, t.i0 + min(m0, t.rows - 1) / sp.G), b1 * KV8_BLOCK);
  const int lim_hi = m0 >= t.rows ? 0 : min(seen_by(a, t, t.i0 + last / sp.G), b1 * KV8_BLOCK);  // the wave's rows see no key from there on
  const int v_end = min(t.total, b1 * KV8_BLOCK);

  uint4 q[D / 16];
  {
    const uint16_t* src = (const uint16_t*)a.q + (long long)(t.start + t.i0 + tok) * a.ldq + (kv_head * sp.G + hq) * D;
#pragma unroll
    for (int n = 0; n < D / 16; ++n) q[n] = *(const uint4*)(src + (2 * (n >> 1) + g) * 16 + (n & 1) * 8);
  }
  St st;
  const size_t stride = (size_t)a.pages.kv_heads * (KV8_BLOCK * D);
  const uint8_t* kbase = (const uint8_t*)a.pages.k + (size_t)kv_head * (KV8_BLOCK * D);
  const uint8_t* vbase = (const uint8_t*)a.pages.v + (size_t)kv_head * (KV8_BLOCK * D);
  const int* table = a.table + (size_t)t.row * a.ld_table;

  // ids and exponents of 64 blocks (32 steps) one a lane, the next 64's on the way
  auto ids_of = [&](int chunk) {
    const int b = b0 + chunk * 64 + lane;
    return b < b1 ? table[b] : 0;
  };
  auto exps_of = [&](int chunk, int& id, int& ke, int& ve) {
    ke = 127;
    ve = -1;
    if (b0 + chunk * 64 + lane >= b1) return;  // a last step's second block beyond the part: nobody sees it
    if ((unsigned)id < (unsigned)a.pages.n_blocks) {
      ke = a.pages.k_exp[(size_t)id * a.pages.kv_heads + kv_head];
      ve = a.pages.v_exp[(size_t)id * a.pages.kv_heads + kv_head];
    } else {
      id = 0;
      ke = 255;
    }
  };
  int id = ids_of(0), ke, ve;
  exps_of(0, id, ke, ve);
  int id2 = ids_of(1), ke2 = 127, ve2 = -1;

  uint4 rk[NC], rv[NC];
  int nke[2], nve[2];  // exponents of the step in registers
  Units units;         // of the blocks that were converted
  int nE[2], nS[2];    // value units of the step in registers, and the exponents of its codes' factors
  auto load = [&](int s) {
    const int x = 2 * (s & 31);
    if (s > 0 && x == 0) { id = id2; ke = ke2; ve = ve2; id2 = ids_of(s / 32 + 1); }
    if (x == 32) exps_of(s / 32 + 1, id2, ke2, ve2);
    nke[0] = __builtin_amdgcn_readlane(ke, x); nke[1] = __builtin_amdgcn_readlane(ke, x + 1);
    nve[0] = __builtin_amdgcn_readlane(ve, x); nve[1] = __builtin_amdgcn_readlane(ve, x + 1);
    nan_scales(nke[0], nve[0]);
    nan_scales(nke[1], nve[1]);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int y = __builtin_amdgcn_readfirstlane((tid + T * n) / CB), r = (tid + T * n) % CB;
      const size_t page = (size_t)__builtin_amdgcn_readlane(id, x + y) * stride;
      rk[n] = *(const uint4*)(kbase + page + (uint32_t)(r * 16));
      rv[n] = *(const uint4*)(vbase + page + (uint32_t)(r * 16));
    }
  };
  // the step in registers to LDS, in four pieces a chunk; `unit` comes first
  auto unit = [&](int s) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      nE[y] = units.add(nve[y]);
      nS[y] = Units::factor(nve[y], nE[y]);
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int y = __builtin_amdgcn_readfirstlane((tid + T * n) / CB), r = (tid + T * n) % CB, key0 = (b0 + 2 * s + y) * KV8_BLOCK;
      if (nke[y] > 254 || key0 + KV8_BLOCK > v_end) {  // values behind the last token count as zeros, whatever they are
        const int left = nke[y] > 254 ? 0 : v_end - key0 - 8 * (r / (D / 2));
        const uint64_t keep = left >= 8 ? ~0ull : left <= 0 ? 0ull : (1ull << (8 * left)) - 1ull;
        rv[n].x &= (uint32_t)keep; rv[n].y &= (uint32_t)(keep >> 32);
        rv[n].z &= (uint32_t)keep; rv[n].w &= (uint32_t)(keep >> 32);
      }
    }
  };
  auto convert = [&](int piece, int buf) {
    const int n = piece >> 2;
    const int y = __builtin_amdgcn_readfirstlane((tid + T * n) / CB), r = (tid + T * n) % CB;
    if ((piece & 3) < 2) {  // keys: chunk c of 16 channels, key k -> two operands of 8 channels, at the key's operand row
      const int c = r >> 5, k = r & 31, row = (k & 0x13) | ((k & 4) << 1) | ((k & 8) >> 1);
      const uint32_t lo = (piece & 1) ? rk[n].z : rk[n].x, hi = (piece & 1) ? rk[n].w : rk[n].y;
      uint4* kd = &s_k[buf][y][c * 64 + (piece & 1) * 32 + row];
      if constexpr (BF) *kd = __builtin_bit_cast(uint4, codes_bf16(lo, hi));
      else *kd = __builtin_bit_cast(uint4, codes_f16(lo, hi, 1.f));
    } else {  // values: group of 8 keys, channel pair -> an operand of 8 keys for each channel
      const float vs = pow2_bits(y ? nS[1] : nS[0]);
      const uint32_t lo = (piece & 1) ? rv[n].z : rv[n].x, hi = (piece & 1) ? rv[n].w : rv[n].y;
      s_v[buf][y][r / (D / 2) * D + (piece & 1) * (D / 2) + r % (D / 2)] = __builtin_bit_cast(uint4, codes_f16(lo, hi, vs));
    }
  };
  uint4 kf[D / 16], vf[2][St::NT][2];
  auto read_k = [&](int buf, int y) {
#pragma unroll
    for (int n = 0; n < D / 16; ++n) kf[n] = s_k[buf][y][(2 * (n >> 1) + g) * 64 + (n & 1) * 32 + i];
  };
  auto scores = [&](typename St::Acc& sc) {
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      if constexpr (BF) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(kf[n]), as_bf16x8(q[n]), sc, 0, 0, 0);
      else sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_f16x8(kf[n]), as_f16x8(q[n]), sc, 0, 0, 0);
    }
  };
  // One block: its scores are in `sc`, their maximum in mx; the next block's go into `sn` while its probabilities are made,
  // and into mx while P . V runs, where the next step's codes are converted too (cbuf >= 0).  The order within a phase is
  // pinned, a few vector instructions behind each MFMA, so that both units work at once.
  float mx;
  auto block = [&](int buf, int y, int key0, int kx, int vx, int E, typename St::Acc (&sc)[1], int nbuf, int ny, typename St::Acc (&sn)[1], auto conv, int cbuf) {
    read_k(nbuf, ny);
    const int ex = sp.ce + kx - 127;
    float c = __builtin_amdgcn_ldexpf(sp.cm, ex);
    if (__builtin_expect(max(key0 + KV8_BLOCK - lim_lo, kx - 254) > 0, 0)) {
      St::mask(sc, kx > 254, key0, lim, g);
      mx = St::top(sc);
    }
    if (__builtin_expect(abs(ex) > St::NORMAL, 0)) {
      St::scale_scores(sc, sp.cm, ex);
      c = 1.f;
      mx = St::top(sc);
    }
    st.move(sc, c, mx, vx, E);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int x = 0; x < St::NT; ++x)
#pragma unroll
        for (int j = 0; j < 2; ++j) vf[kk][x][j] = s_v[buf][y][(2 * kk + g) * D + j * (D / 2) + 32 * x + i];
    constexpr int NQ = D / 16, NE = 16 / NQ;
    f16x8 p[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) sn[0][r] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      if constexpr (BF) sn[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(kf[n]), as_bf16x8(q[n]), sn[0], 0, 0, 0);
      else sn[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_f16x8(kf[n]), as_f16x8(q[n]), sn[0], 0, 0, 0);
#pragma unroll
      for (int z = NE * n; z < NE * (n + 1); z += 2) {
        const f16x2_t h = __builtin_convertvector((f32x2_t{__builtin_amdgcn_exp2f(fmaf(sc[0][z], c, st.nb)), __builtin_amdgcn_exp2f(fmaf(sc[0][z + 1], c, st.nb))}), f16x2_t);
        p[z >> 3][z & 7] = h[0];
        p[z >> 3][(z & 7) + 1] = h[1];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    constexpr int NV = 2 * St::NT, NM = 2 * NV;  // P . V products of half a block, of all of it
    constexpr int CP = decltype(conv)::value ? 4 * NC : 0;
#pragma unroll
    for (int n = 0; n < NM; ++n) {
      const int kk = n / NV, w = n % NV;
      st.o[w >> 1][w & 1] = mfma_pv(as_f16x8(vf[kk][w >> 1][w & 1]), p[kk], st.o[w >> 1][w & 1]);
      if (w == 0) st.sum(p[kk]);
#pragma unroll
      for (int z = CP * n / NM; z < CP * (n + 1) / NM; ++z) convert(z, cbuf);
      if (n == NM - 4) mx = fmaxf(fmaxf(sn[0][0], sn[0][1]), fmaxf(sn[0][2], sn[0][3]));
      if (n > NM - 4) {
#pragma unroll
        for (int z = 4 * (n - NM + 4); z < 4 * (n - NM + 5); ++z) mx = fmaxf(mx, sn[0][z]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  load(0);
  unit(0);
#pragma unroll
  for (int z = 0; z < 4 * NC; ++z) convert(z, 0);
  int kx0 = nke[0], kx1 = nke[1], vx0 = nve[0], vx1 = nve[1], E0 = nE[0], E1 = nE[1];
  if (steps > 1) load(1);
  __syncthreads();
  typename St::Acc s0[1], s1[1];
  read_k(0, 0);
  scores(s0[0]);
  mx = St::top(s0);
  int cur = 0;
  for (int s = 0; s < steps; ++s) {
    const int nxt = cur == 2 ? 0 : cur + 1, key0 = (b0 + 2 * s) * KV8_BLOCK;
    const bool on = key0 < lim_hi, more = s + 1 < steps;
    int nkx0 = 127, nkx1 = 127, nvx0 = -1, nvx1 = -1;
    if (more) {
      unit(s + 1);
      nkx0 = nke[0]; nkx1 = nke[1];
      nvx0 = nve[0]; nvx1 = nve[1];
    }
    if (on) {
      block(cur, 0, key0, kx0, vx0, E0, s0, cur, 1, s1, std::true_type(), nxt);  // after the last step: into a buffer that nobody reads
    } else {
#pragma unroll
      for (int z = 0; z < 4 * NC; ++z) convert(z, nxt);
    }
    if (s + 2 < steps) load(s + 2);
    __syncthreads();
    if (on) block(cur, 1, key0 + KV8_BLOCK, kx1, vx1, E1, s1, nxt, 0, s0, std::false_type(), 0);
    kx0 = nkx0; kx1 = nkx1; vx0 = nvx0; vx1 = nvx1; E0 = nE[0]; E1 = nE[1];
    cur = nxt;
  }
  if (mrow < t.rows) st.template store<BF>(a, sp, t, kv_head, part, parts, mrow, g);
}

// Joins the parts of split tiles, WR waves to a packed row: each wave sums its share of them, a lane D / 64 channels.  Four
// waves where a row has more than 8 parts: 47 parts 24.9 us a call, 32.7 with one wave; 4 parts 21.2 and 20.7.
template <bool BF, int D, int WR>
__global__ void __launch_bounds__(256) kv8_join_kernel(t2w_kv8_attention_args a, KV8Split sp) {
  constexpr int NV = D / 64;
  __shared__ float s_acc[WR > 1 ? 4 : 1][NV][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave % WR;
  const int slot = blockIdx.x / a.pages.kv_heads, kv_head = blockIdx.x - slot * a.pages.kv_heads, m = blockIdx.y * (4 / WR) + wave / WR;
  Tile t;
  if (!find_tile(a, sp, slot, t) || t.bad) return;
  int per;
  const int parts = tile_parts(sp, t, per);
  if (parts == 1 || m >= t.rows) return;  // with WR == 4 the whole workgroup
  const size_t rows = sp.tt * sp.G, pr = ((size_t)slot * a.pages.kv_heads + kv_head) * t.parts;
  const float* po = (const float*)a.workspace + (pr * rows + m) * D + lane * NV;
  const float* ml = (const float*)a.workspace + part_rows(sp, a.pages.kv_heads) * D + (pr * rows + m) * 2;
  // every lane its parts' (maximum, sum): up to 256 parts
  float2 x[4];
  float top = -__builtin_inff();
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int p = n * 64 + lane;
    x[n] = p < parts ? *(const float2*)(ml + (size_t)p * rows * 2) : make_float2(-__builtin_inff(), 0.f);
    top = fmaxf(top, x[n].x);
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
  float sum = 0.f, acc[NV] = {};
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if (n * 64 >= parts) break;
    const float f = x[n].y != x[n].y ? __builtin_nanf("") : x[n].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(x[n].x - top) * x[n].y;
    sum += f;
    const int cnt = min(64, parts - n * 64);
#pragma unroll 8
    for (int p = w; p < cnt; p += WR) {
      const float fp = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), p));
      const float* src = po + (size_t)(n * 64 + p) * rows * D;
#pragma unroll
      for (int v = 0; v < NV; ++v) acc[v] += fp * src[v];
    }
  }
  sum = wave_sum(sum);
  if constexpr (WR > 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v) s_acc[w][v][lane] = acc[v];
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int v = 0; v < NV; ++v) acc[v] = (s_acc[0][v][lane] + s_acc[1][v][lane]) + (s_acc[2][v][lane] + s_acc[3][v][lane]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int tok = m / sp.G;
  uint16_t* out = (uint16_t*)a.out + (long long)(t.start + t.i0 + tok) * a.ldo + (kv_head * sp.G + m - tok * sp.G) * D + lane * NV;
#pragma unroll
  for (int v = 0; v < NV; ++v) out[v] = BF ? f2bf(acc[v] * inv) : f2h(acc[v] * inv);
}

// Which form, tile and split a call takes: from its sizes and bounds alone, so that the workspace's size is known too.
struct Choice {
  int mr, rw;  // packed rows of a wave, waves that share the keys' loads
  bool tile;   // the tile form
  KV8Split s;
};

Choice choose(const t2w_kv8_attention_args& a) {
  Choice c;
  const int G = c.s.G = a.heads / a.pages.kv_heads;
  const long max_new = a.max_new > 0 ? min(a.max_new, a.n_tok) : a.n_tok, packed = max_new * G;
  const long max_kv = a.max_kv > 0 ? min((long)a.max_kv, (long)a.width * KV8_BLOCK) : (long)a.width * KV8_BLOCK;
  const long nb = (max_kv + KV8_BLOCK - 1) / KV8_BLOCK;
  // The direct form on as few packed rows as hold the longest row, up to 64.  With heads of 128 the tile form takes calls
  // whose 256-row tiles (and parts) fill the chip, one workgroup a CU, and are mostly full: 32 heads over 8 (us, direct /
  // tile): one row of 8,000 tokens 625 / 550, 2,048 behind 32,000 1,250 / 1,095, four of 500 30.7 / 27.8; a row of 1,000
  // tokens alone (128 workgroups) 24.7 / 37.8, 32 of 70 behind 2,000 (tiles 55% full) 130 / 161.  With heads of 64 the
  // direct form was the faster one of those tried (tiles of 128 rows, four waves: 1,000 tokens of 16 heads 14.8 / 24.6, 8,000
  // 202 / 214).
  c.mr = packed <= 16 ? 16 : 32;
  c.rw = packed <= 32 ? 1 : 2;
  c.tile = false;
  // Tiles: as many rows as there can be of the longest; without a bound every row may end in a part of one.
  const long tt = 256 / G, rows = a.max_new > 0 ? (a.n_tok + max_new - 1) / max_new : 1, slots = a.n_tok / tt + min(a.n_rows, a.n_tok);
  const long tiles = a.max_new > 0 || a.n_rows == 1 ? rows * ((max_new + tt - 1) / tt) : slots, groups = tiles * a.pages.kv_heads;
  const long fit = groups >= 256 ? 1 : min(256 / max(groups, 1L), max(nb / 64, 1L));
  if (a.pages.head_dim == 128 && packed > 64 && groups * fit >= 224 && a.n_tok * 10L >= tiles * tt * 7) {
    c.tile = true;
    c.rw = 8;
  }
  c.s.tt = c.mr * c.rw / G;
  // How many tiles there are only the GPU knows (rows may rest): the tile form's workspace is that of one round of workgroups,
  // and the kernel counts the tiles and takes fewer parts where there are more of them (parts for every slot took 2.2 GB for 64
  // rows of a token without bounds, tables 2,048 wide, and 35 GB for 4,096 rows of which one has 256 tokens).
  c.s.cap = c.tile && fit > 1 ? 256 : 0;
  c.s.cm = std::frexp(a.scale, &c.s.ce) * 1.4426950408889634f;
  c.s.per_row = a.max_new > 0 && a.max_new <= c.s.tt && c.s.cap == 0 ? 1 : 0;
  c.s.n_tiles = c.s.cap > 0 ? (int)slots : c.s.per_row ? a.n_rows : a.n_tok / c.s.tt + a.n_rows;
  // Parts: the tile form's, so that one round of workgroups fills the chip.  The direct form's lists of up to 48 blocks stay
  // whole (a second launch costs more: one row of 1,500 keys 9.6 us whole, 10.5 split); longer ones are cut where
  // workgroups are few, to 512 in all and 16 blocks or more a part (two rows of 131,072 keys: 103 us with 512 workgroups,
  // 111 with 1,024, 120 with 2,048; 64 rows of up to 8,192: 139, 152, 150).
  long parts = 1;
  if (c.tile) {
    parts = fit;
  } else if (nb > 48) {
    const long g = (long)c.s.n_tiles * a.pages.kv_heads;
    parts = min((512 + g - 1) / g, (nb + 15) / 16);
  }
  c.s.bps = (int)((nb + parts - 1) / parts);
  c.s.parts = (int)min((nb + c.s.bps - 1) / c.s.bps, 256L);
  return c;
}

}  // namespace

size_t kv8_attention_workspace(const t2w_kv8_attention_args& a) {
  const Choice c = choose(a);
  return c.s.parts > 1 ? part_rows(c.s, a.pages.kv_heads) * (a.pages.head_dim + 2) * sizeof(float) : 0;
}

template <bool BF, int D>
static hipError_t launch(const t2w_kv8_attention_args& a, const Choice& c, hipStream_t st) {
  const dim3 grid((unsigned)(c.s.n_tiles * a.pages.kv_heads), c.s.parts);
  if (c.tile) {
    if constexpr (D == 128) {
      constexpr int LDS = 3 * 2 * 2 * KV8_BLOCK * D * 2;  // three steps of two blocks, keys and values in 16 bits
      static std::atomic<uint64_t> done{0};  // devices whose LDS limit of this kernel is raised above 64 KB
      int dev = 0;
      hipError_t e = hipGetDevice(&dev);
      if (e != hipSuccess) return e;
      const uint64_t bit = dev < 64 ? 1ull << dev : 0;
      if (!(done.load(std::memory_order_acquire) & bit)) {
        e = hipFuncSetAttribute((const void*)kv8_attn_tile_kernel<BF, D, 8>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return e;
        done.fetch_or(bit, std::memory_order_release);
      }
      hipLaunchKernelGGL((kv8_attn_tile_kernel<BF, D, 8>), grid, dim3(512), LDS, st, a, c.s);
    }
  } else if (c.mr == 16) {
    hipLaunchKernelGGL((kv8_attn_direct_kernel<BF, D, 16, 1, D == 64 ? 6 : 4>), grid, dim3(256), 0, st, a, c.s);
  } else if (c.rw == 1) {
    hipLaunchKernelGGL((kv8_attn_direct_kernel<BF, D, 32, 1, D == 64 ? 4 : 2>), grid, dim3(256), 0, st, a, c.s);
  } else {
    hipLaunchKernelGGL((kv8_attn_direct_kernel<BF, D, 32, 2, D == 64 ? 4 : 2>), grid, dim3(256), 0, st, a, c.s);
  }
  // counted tiles have parts only where they are few (and cap / 2 is at least the key heads where there are parts at all)
  const int joined = c.s.cap > 0 ? min(c.s.n_tiles, c.s.cap / 2 / a.pages.kv_heads) : c.s.n_tiles;
  const unsigned groups = (unsigned)(joined * a.pages.kv_heads), rows = (unsigned)(c.s.tt * c.s.G);
  if (c.s.parts > 8) hipLaunchKernelGGL((kv8_join_kernel<BF, D, 4>), dim3(groups, rows), dim3(256), 0, st, a, c.s);
  else if (c.s.parts > 1) hipLaunchKernelGGL((kv8_join_kernel<BF, D, 1>), dim3(groups, (rows + 3) / 4), dim3(256), 0, st, a, c.s);
  return hipGetLastError();
}

hipError_t kv8_attention(const t2w_kv8_attention_args& a, hipStream_t st) {
  if (a.n_tok <= 0 || a.n_rows <= 0) return hipSuccess;
  const Choice c = choose(a);
  if ((long)c.s.n_tiles * a.pages.kv_heads > 0x7fffffffL) return hipErrorInvalidValue;
  if (a.dtype == T2W_KV8_BF16) return a.pages.head_dim == 64 ? launch<true, 64>(a, c, st) : launch<true, 128>(a, c, st);
  return a.pages.head_dim == 64 ? launch<false, 64>(a, c, st) : launch<false, 128>(a, c, st);
}

}  // namespace t2w
