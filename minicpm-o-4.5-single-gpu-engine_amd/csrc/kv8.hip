// Paged 8-bit key/value cache: block tables and slot maps built on the GPU from request lengths, and the append that
// quantizes new keys and values into the cache.  Block format: kv8_internal.h.
#include "kv8_internal.h"

namespace t2w {

namespace {

// ---------------------------------------------------------------- tables
// Row r holds kv_len[r] tokens in ceil(kv_len[r] / 32) blocks and gets new_len[r] more.  With the exclusive sums S of the
// new lengths and B of the blocks that each row needs beyond its own, token n of the call belongs to the row with
// S[r] <= n < S[r + 1], stands at position p = kv_len[r] + n - S[r], and its block p / 32 is the row's own or the new
// block free_ids[head + B[r] + p / 32 - own blocks].
//
// One launch and no wait between workgroups: every workgroup sums all rows by itself (PER rows a thread, loaded together, a
// scan within each wave and one over the four waves), keeps S, B and kv_len in LDS, and then writes the tables of its own
// PLAN_TOKENS tokens.  The token at a block's first place writes that block into the table, so each new entry has one
// writer and none is read in the same call.  Bound by latency: a launch, the lengths' load, an id's load, the stores
// (64 rows of a token 4.2 us, 2,048 rows 6.0, 512 rows of 277,805 tokens 5.8; shuffles instead of DPP moves and lengths
// loaded one by one: 4.5, 10.0, 7.9).
constexpr int PLAN_TOKENS = 1024;  // tokens of a workgroup

// T threads of PER rows and PLAN_TOKENS / T tokens.  VEC: the lengths and the token tables are 16-byte aligned.
template <int T, int PER, bool VEC>
__global__ void __launch_bounds__(T) kv8_plan_kernel(t2w_kv8_plan_args a) {
  constexpr int W = T / 64, NT = PLAN_TOKENS / T;
  __shared__ int s_tok[T * PER + 1], s_blk[T * PER], s_kv[T * PER];
  __shared__ int w_tok[W], w_blk[W], w_bad[W];
  __shared__ long long w_tot[W][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r0 = tid * PER;
  const int head = a.free_head[0];
  int kv[PER], nw[PER];
  if (VEC && PER == 4 && r0 + 4 <= a.n_rows) {
    const int4 x = *(const int4*)(a.kv_len + r0), y = *(const int4*)(a.new_len + r0);
    kv[0] = x.x; kv[1 % PER] = x.y; kv[2 % PER] = x.z; kv[3 % PER] = x.w;
    nw[0] = y.x; nw[1 % PER] = y.y; nw[2 % PER] = y.z; nw[3 % PER] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = r0 + i < a.n_rows;
      kv[i] = in ? a.kv_len[r0 + i] : 0;
      nw[i] = in ? a.new_len[r0 + i] : 0;
    }
  }
  int tok = 0, blk = 0, bad = 0, at[PER], ab[PER];
  long long tok64 = 0, blk64 = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    bad |= (kv[i] < 0 || nw[i] < 0) ? 1 : 0;
    const long long want = ((long long)kv[i] + nw[i] + KV8_BLOCK - 1) / KV8_BLOCK, have = ((long long)kv[i] + KV8_BLOCK - 1) / KV8_BLOCK;
    bad |= want > a.width ? 4 : 0;
    at[i] = tok;
    ab[i] = blk;
    tok += nw[i];
    blk += (int)(want - have);
    tok64 += nw[i];
    blk64 += want - have;
  }
  const int it = wave_scan(tok), ib = wave_scan(blk);
  // The 32-bit sums are exact where every thread's are small (at most 1024 threads of 2^20); else they may wrap, and
  // the 64-bit totals say that the call fails.
  long long t64 = __builtin_amdgcn_readlane(it, 63), b64 = __builtin_amdgcn_readlane(ib, 63);
  if (__builtin_amdgcn_ballot_w64(tok64 > (1 << 20) || tok64 < 0 || blk64 > (1 << 20) || blk64 < 0)) {
    t64 = tok64;
    b64 = blk64;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      t64 += __shfl_xor(t64, o, 64);
      b64 += __shfl_xor(b64, o, 64);
    }
  }
  bad = (__builtin_amdgcn_ballot_w64(bad & 1) ? 1 : 0) | (__builtin_amdgcn_ballot_w64(bad & 4) ? 4 : 0);
  if (lane == 63) {
    w_tok[wave] = it;
    w_blk[wave] = ib;
    w_tot[wave][0] = t64;
    w_tot[wave][1] = b64;
    w_bad[wave] = bad;
  }
  __syncthreads();
  int bt = it - tok, bb = ib - blk;
  for (int w = 0; w < wave; ++w) { bt += w_tok[w]; bb += w_blk[w]; }
  long long n_tok = 0, n_blk = 0;
  int status = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    n_tok += w_tot[w][0];
    n_blk += w_tot[w][1];
    status |= w_bad[w];
  }
  status |= n_tok > a.n_tok ? 2 : 0;
  status |= (head < 0 || head + n_blk > a.n_free) ? 8 : 0;
  const bool ok = status == 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    s_tok[r0 + i] = at[i] + bt;  // rows from n_rows on start at the total
    s_blk[r0 + i] = ab[i] + bb;
    s_kv[r0 + i] = kv[i];
    if (blockIdx.x == 0 && r0 + i < a.n_rows) {
      a.row_start[r0 + i] = ok ? at[i] + bt : 0;
      a.kv_total[r0 + i] = ok ? kv[i] + nw[i] : kv[i];
    }
  }
  if (tid == 0) {
    s_tok[T * PER] = (int)n_tok;
    if (blockIdx.x == 0) {
      a.row_start[a.n_rows] = ok ? (int)n_tok : 0;
      a.free_head_out[0] = ok ? head + (int)n_blk : head;
      a.status[0] = status;
    }
  }
  __syncthreads();
  const int n0 = blockIdx.x * PLAN_TOKENS + tid * NT;
  if (n0 >= a.n_tok) return;
  const int total = ok ? (int)n_tok : 0;
  int r = 0;
  if (n0 < total) {  // the last row that starts at or before n0: rows without tokens start where the next one does
    int lo = 0, hi = a.n_rows;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_tok[mid] <= n0) lo = mid; else hi = mid;
    }
    r = lo;
  }
  int row[NT], pos[NT], slot[NT];
  int* entry[NT];
  const int* from[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + j;
    row[j] = pos[j] = slot[j] = -1;
    entry[j] = nullptr;
    from[j] = nullptr;
    if (n < total) {
      while (s_tok[r + 1] <= n) ++r;  // n < total: ends at the row that holds n
      const int k = s_kv[r], p = k + n - s_tok[r], b = p / KV8_BLOCK, have = (k + KV8_BLOCK - 1) / KV8_BLOCK;
      entry[j] = a.table + (size_t)r * a.ld_table + b;
      from[j] = b < have ? entry[j] : a.free_ids + (head + s_blk[r] + b - have);
      row[j] = r;
      pos[j] = p;
    }
  }
  int id[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) id[j] = from[j] ? *from[j] : 0;
#pragma unroll
  for (int j = 0; j < NT; ++j)
    if (from[j]) {
      if (pos[j] % KV8_BLOCK == 0) *entry[j] = id[j];
      slot[j] = (int)((unsigned)id[j] * KV8_BLOCK + pos[j] % KV8_BLOCK);
    }
  if (VEC && NT == 4 && n0 + 4 <= a.n_tok) {
    *(int4*)(a.tok_row + n0) = make_int4(row[0], row[1 % NT], row[2 % NT], row[3 % NT]);
    *(int4*)(a.tok_pos + n0) = make_int4(pos[0], pos[1 % NT], pos[2 % NT], pos[3 % NT]);
    *(int4*)(a.slots + n0) = make_int4(slot[0], slot[1 % NT], slot[2 % NT], slot[3 % NT]);
  } else {
#pragma unroll
    for (int j = 0; j < NT; ++j)
      if (n0 + j < a.n_tok) {
        a.tok_row[n0 + j] = row[j];
        a.tok_pos[n0 + j] = pos[j];
        a.slots[n0 + j] = slot[j];
      }
  }
}

// ---------------------------------------------------------------- append
// A block's scale is 2^e with the smallest e that keeps its largest magnitude within e4m3's 448 (mx_exp), so a code is
// e4m3(x / 2^e) and nothing clips.  A block that holds tokens already takes max(e_old, e_new); where that is larger than
// e_old, its codes c become e4m3(c * 2^(e_old - e)), which is exact except where a code leaves e4m3's normal range: that
// is why the scales are powers of two.  A token with a key or value that is not finite counts for no scale and is stored
// as a key of NaN codes and a value of zeros: a query that sees it gets NaN, through its score, and no other query does
// (a NaN among the values would reach every query of a tile through 0 * NaN).  A new block is zero behind its last token.
//
// Memory bound (2 bytes read and 1 written a value).  A workgroup takes one touched block of two heads, a wave the keys or
// the values of one of them.  The keys' wave loads 16 channels of a key per lane (32 bytes) and stores them as 16; the
// values' wave loads a channel pair of every key (rows of D values are read whole, 4 bytes a lane) and so holds eight keys
// of two channels, the stored order, in its own registers: no LDS, no shuffles.  37,433 tokens of 8 heads of 128 in fp16: 230 MB in
// 51 us, 88% of a copy's rate; a step of 64 tokens 5 us, a launch and four loads that wait for each other.
template <bool BF>
__device__ __forceinline__ float lo16(uint32_t w) { if constexpr (BF) return lo2f(w); else return lo2h(w); }
template <bool BF>
__device__ __forceinline__ float hi16(uint32_t w) { if constexpr (BF) return hi2f(w); else return hi2h(w); }

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// four values times inv, clamped to +-448 and rounded to nearest even e4m3, packed low byte first: mx_pack4 with the factor itself,
// which is subnormal for scales of 2^127
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float inv) {
  auto cl = [](float x) { return fminf(fmaxf(x, -448.0f), 448.0f); };
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(cl(a * inv), cl(b * inv), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cl(c * inv), cl(d * inv), w, true);
}

// codes of four bytes times f (a power of two <= 1), rounded to nearest even; NaN stays NaN
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  int o = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, o, true);
}

// maximum over the wave, the same in every lane: the scan's lane moves, whose last lane then holds it
__device__ __forceinline__ int wave_max_i(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}

// the largest magnitude of packed maxima (sign bits cleared), as the bits of one 16-bit value
__device__ __forceinline__ int top16(uint32_t m) { return wave_max_i(max((int)(m & 0xffffu), (int)(m >> 16))); }

template <bool BF, int D>
__global__ void __launch_bounds__(256) kv8_append_kernel(t2w_kv8_append_args a, int per_row) {
  constexpr int INF = BF ? 0x7f80 : 0x7c00;  // magnitudes from here on are not finite
  __shared__ uint32_t s_bad[2][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hw = wave >> 1;
  const bool is_v = wave & 1;
  // a block's heads next to each other: they share the tokens' rows
  const int pairs = (a.pages.kv_heads + 1) / 2, item = blockIdx.x / pairs, head = (blockIdx.x - item * pairs) * 2 + hw;
  const bool live = head < a.pages.kv_heads;
  int row, at;
  if (per_row > 0) {
    row = item / per_row;
    at = item - row * per_row;
  } else {
    row = kv8_find_row(a.row_start, a.n_rows, KV8_BLOCK, 2, item);
    at = item - (a.row_start[row] / KV8_BLOCK + 2 * row);
    if (at < 0) return;  // in front of the first row, whose tokens need not be the call's first ones
  }
  const int start = a.row_start[row], n_new = a.row_start[row + 1] - start, total = a.kv_total[row];
  if (start < 0 || n_new <= 0 || start > a.n_tok - n_new || total < n_new) return;  // nothing new, or a malformed table
  const int old = total - n_new;
  const int b_first = old / KV8_BLOCK, b_last = min((total - 1) / KV8_BLOCK, a.width - 1);
  // a row's last workgroup goes on to its end: rows longer than the caller's bound are still stored whole
  const bool on = per_row > 0 && at == per_row - 1;
  for (int b = b_first + at; b <= b_last; ++b) {
    const int id = a.table[(size_t)row * a.ld_table + b];  // waited for where the stores begin
    const int first = max(old - b * KV8_BLOCK, 0), end = min(total - b * KV8_BLOCK, KV8_BLOCK);  // new tokens [first, end)
    const int tok0 = start + b * KV8_BLOCK - old;  // token of place 0 (may lie before the row's first one)
    constexpr int NC = D / 16, KP = 64 / NC, NP = NC / 2;  // the keys' wave: NC lanes a key, KP keys a pass
    constexpr int VK = D == 128 ? 32 : 16;                // the values' wave: keys of a lane
    const int c = lane % NC, kl = lane / NC;
    const int p = D == 128 ? lane : lane & 31, g0 = D == 128 ? 0 : 2 * (lane >> 5);
    uint4 xk[NP][2];
    uint32_t xv[VK];
    uint32_t m = 0;
    if (live) {
      if (!is_v) {
        const uint16_t* src = (const uint16_t*)a.k + head * D + c * 16;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          const int t = n * KP + kl;
          xk[n][0] = xk[n][1] = make_uint4(0, 0, 0, 0);
          if (t >= first && t < end) {
            const uint4* q = (const uint4*)(src + (long long)(tok0 + t) * a.ldk);
            xk[n][0] = q[0];
            xk[n][1] = q[1];
          }
        }
#pragma unroll
        for (int n = 0; n < NP; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w[4] = {xk[n][h].x, xk[n][h].y, xk[n][h].z, xk[n][h].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) m = max_u16x2(m, w[j] & 0x7fff7fffu);
          }
      } else {
        const uint16_t* src = (const uint16_t*)a.v + head * D + 2 * p;
#pragma unroll
        for (int j = 0; j < VK; ++j) {
          const int t = g0 * 8 + j;
          xv[j] = 0;
          if (t >= first && t < end) xv[j] = *(const uint32_t*)(src + (long long)(tok0 + t) * a.ldv);
        }
#pragma unroll
        for (int j = 0; j < VK; ++j) m = max_u16x2(m, xv[j] & 0x7fff7fffu);
      }
    }
    // the block's scale so far, under way while the tokens arrive
    const bool fresh = first == 0, mine = live && (unsigned)id < (unsigned)a.pages.n_blocks;
    uint8_t* exps = (is_v ? a.pages.v_exp : a.pages.k_exp) + (size_t)(mine ? id : 0) * a.pages.kv_heads + (live ? head : 0);
    const int was = mine && !fresh ? (int)*exps - 127 : 0;
    int top = top16(m);
    uint32_t bad = 0;  // tokens of this head with a key (the keys' wave) or value (the values') that is not finite
    auto off16 = [&](uint32_t w) { return (int)(w & 0x7fffu) >= INF || (int)((w >> 16) & 0x7fffu) >= INF; };
    if (top >= INF) {
      if (!is_v) {
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          bool f = false;
#pragma unroll
          for (int h = 0; h < 2; ++h) f |= off16(xk[n][h].x) || off16(xk[n][h].y) || off16(xk[n][h].z) || off16(xk[n][h].w);
          const uint64_t bits = __builtin_amdgcn_ballot_w64(f);
#pragma unroll
          for (int q = 0; q < KP; ++q) bad |= ((bits >> (q * NC)) & ((1u << NC) - 1u)) ? 1u << (n * KP + q) : 0u;
        }
      } else {
#pragma unroll
        for (int j = 0; j < VK; ++j) {
          const uint64_t bits = __builtin_amdgcn_ballot_w64(off16(xv[j]));
          if constexpr (D == 128) {
            bad |= bits ? 1u << j : 0u;
          } else {
            bad |= (uint32_t)bits ? 1u << j : 0u;
            bad |= (uint32_t)(bits >> 32) ? 1u << (16 + j) : 0u;
          }
        }
      }
    }
    if (lane == 0) s_bad[hw][is_v] = bad;
    __syncthreads();
    bad = s_bad[hw][0] | s_bad[hw][1];
    __syncthreads();  // before the next block's flags
    if (bad) {        // the maximum again, without the tokens that are not finite
      m = 0;
      if (!is_v) {
#pragma unroll
        for (int n = 0; n < NP; ++n)
          if (!((bad >> (n * KP + kl)) & 1u)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w[4] = {xk[n][h].x, xk[n][h].y, xk[n][h].z, xk[n][h].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) m = max_u16x2(m, w[j] & 0x7fff7fffu);
            }
          }
      } else {
#pragma unroll
        for (int j = 0; j < VK; ++j) {
          if ((bad >> (g0 * 8 + j)) & 1u) xv[j] = 0;  // stored as zeros
          m = max_u16x2(m, xv[j] & 0x7fff7fffu);
        }
      }
      top = top16(m);
    }
    if (mine) {
      const size_t page = ((size_t)id * a.pages.kv_heads + head) * (size_t)(KV8_BLOCK * D);
      int e = mx_exp(lo16<BF>((uint32_t)top)), shift = 0;
      if (!fresh) {
        shift = max(e - was, 0);
        e = max(e, was);
      }
      // a block that was filled elsewhere may have the scale 2^127, or an E8M0 NaN (128 here): it keeps it
      const float inv = __builtin_amdgcn_ldexpf(1.f, -e);
      const float f = shift < 126 ? __uint_as_float((uint32_t)(127 - shift) << 23) : 0.f;
      if (lane == 0) *exps = (uint8_t)(e + 127);
      if (!is_v) {
        uint4* dst = (uint4*)((uint8_t*)a.pages.k + page) + c * 32;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          const int t = n * KP + kl;
          uint4 o = make_uint4(0, 0, 0, 0);
          if (t >= first && t < end) {
            uint32_t r[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint4 u = xk[n][h];
              r[2 * h] = pack4(lo16<BF>(u.x), hi16<BF>(u.x), lo16<BF>(u.y), hi16<BF>(u.y), inv);
              r[2 * h + 1] = pack4(lo16<BF>(u.z), hi16<BF>(u.z), lo16<BF>(u.w), hi16<BF>(u.w), inv);
            }
            o = make_uint4(r[0], r[1], r[2], r[3]);
            if ((bad >> t) & 1u) o = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
            dst[t] = o;
          } else if (fresh) {
            dst[t] = o;
          } else if (shift > 0 && t < first) {
            const uint4 u = dst[t];
            dst[t] = make_uint4(rescale4(u.x, f), rescale4(u.y, f), rescale4(u.z, f), rescale4(u.w, f));
          }
        }
      } else {
        uint4* dst = (uint4*)((uint8_t*)a.pages.v + page) + p;
#pragma unroll
        for (int gg = 0; gg < VK / 8; ++gg) {
          const int g = g0 + gg, t0 = g * 8;
          const bool has_new = t0 < end && t0 + 8 > first, has_old = t0 < first;
          if (!(fresh || has_new || (has_old && shift > 0))) continue;
          uint32_t r[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t* x = xv + gg * 8 + 4 * h;
            r[h] = pack4(lo16<BF>(x[0]), lo16<BF>(x[1]), lo16<BF>(x[2]), lo16<BF>(x[3]), inv);
            r[2 + h] = pack4(hi16<BF>(x[0]), hi16<BF>(x[1]), hi16<BF>(x[2]), hi16<BF>(x[3]), inv);
          }
          if (!fresh) {  // the group's other places keep what they hold; its old tokens at the new scale
            const uint4 u = dst[g * (D / 2)];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t s = shift > 0 ? rescale4(w[j], f) : w[j];
              uint32_t o = 0;
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const int t = t0 + 4 * (j & 1) + y;
                const uint32_t mask = 0xffu << (8 * y);
                o |= (t < first ? s : t < end ? r[j] : w[j]) & mask;
              }
              r[j] = o;
            }
          }
          dst[g * (D / 2)] = make_uint4(r[0], r[1], r[2], r[3]);
        }
      }
    }
    if (!on) break;
  }
}

}  // namespace

hipError_t kv8_plan(const t2w_kv8_plan_args& a, hipStream_t st) {
  const int wgs = a.n_tok > 0 ? (a.n_tok + PLAN_TOKENS - 1) / PLAN_TOKENS : 1;
  const bool vec = (((uintptr_t)a.kv_len | (uintptr_t)a.new_len | (uintptr_t)a.tok_row | (uintptr_t)a.tok_pos | (uintptr_t)a.slots) & 15) == 0;
#define T2W_KV8_PLAN(T, PER)                                                                       \
  if (vec) hipLaunchKernelGGL((kv8_plan_kernel<T, PER, true>), dim3(wgs), dim3(T), 0, st, a);      \
  else hipLaunchKernelGGL((kv8_plan_kernel<T, PER, false>), dim3(wgs), dim3(T), 0, st, a);
  if (a.n_rows <= 256) { T2W_KV8_PLAN(256, 1) }
  else if (a.n_rows <= 1024) { T2W_KV8_PLAN(256, 4) }
  else { T2W_KV8_PLAN(1024, 4) }  // 2048 rows: 6.0 us against 9.8 with 256 threads of 16 rows
#undef T2W_KV8_PLAN
  return hipGetLastError();
}

hipError_t kv8_append(const t2w_kv8_append_args& a, hipStream_t st) {
  if (a.n_tok <= 0 || a.n_rows <= 0) return hipSuccess;
  // blocks that a row of up to max_new new tokens touches; more than the whole call's list would be: the list
  const long list = a.n_tok / KV8_BLOCK + 2L * a.n_rows;
  int per_row = a.max_new > 0 ? (int)(((long)a.max_new + KV8_BLOCK - 2) / KV8_BLOCK + 1) : 0;
  if (per_row > 0 && (long)per_row * a.n_rows > list) per_row = 0;
  const long wgs = (per_row > 0 ? (long)per_row * a.n_rows : list) * ((a.pages.kv_heads + 1) / 2);
  if (wgs > 0x7fffffffL) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs);
#define T2W_KV8_APPEND(BF, D) hipLaunchKernelGGL((kv8_append_kernel<BF, D>), grid, dim3(256), 0, st, a, per_row)
  if (a.dtype == T2W_KV8_BF16) {
    if (a.pages.head_dim == 64) T2W_KV8_APPEND(true, 64); else T2W_KV8_APPEND(true, 128);
  } else {
    if (a.pages.head_dim == 64) T2W_KV8_APPEND(false, 64); else T2W_KV8_APPEND(false, 128);
  }
#undef T2W_KV8_APPEND
  return hipGetLastError();
}

}  // namespace t2w
