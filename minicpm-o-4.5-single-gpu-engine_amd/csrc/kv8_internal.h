// Launch interfaces of the paged 8-bit key/value cache: device-built tables (kv8.hip), the quantizing append (kv8.hip)
// and attention over the cache (kv8_attn.hip).  The arguments are checked in kv8_capi.hip.
//
// Block format: 32 tokens of one key/value head, D channels (64 or 128), e4m3 codes and an E8M0 scale byte (exponent +
// 127) for the keys and one for the values.
//   key   (t, d)  byte (d / 16) * 512 + t * 16 + d % 16                     a lane's 16 channels of one key are 16 bytes
//   value (t, d)  byte (t / 8) * 8 D + (d / 2) * 16 + (d % 2) * 8 + t % 8    a lane's 8 keys of two channels are 16 bytes
// Both are the MFMA operand orders of the attention: its lanes load whole fragments 16 bytes wide, a wave 512 contiguous
// bytes or more, with no transposition on the way.
#pragma once

#include "../../include/t2w.h"
#include "common.h"

namespace t2w {

constexpr int KV8_BLOCK = 32;
constexpr int KV8_MAX_ROWS = 4096;  // rows of a call: the tables kernel holds three integers of each in LDS

// sum over lanes 0 .. l of the wave, in lane l: shifts within the 16-lane rows, then each row's last lane to those behind it
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// Row that owns entry t of a list in which row r starts at row_start[r] / div + mult * r (the starts ascend with r): the
// last row whose start is at most t, 0 if there is none.  All 64 lanes of a wave call it together; two dependent loads at
// most (n_rows <= 4096), one up to 64 rows.
__device__ __forceinline__ int kv8_find_row(const int* row_start, int n_rows, int div, int mult, int t) {
  const int lane = threadIdx.x & 63;
  const int step = (n_rows + 63) / 64;
  int r = lane * step;
  bool le = r < n_rows && row_start[r] / div + mult * r <= t;
  int at = (__popcll(__builtin_amdgcn_ballot_w64(le)) - 1) * step;
  at = at < 0 ? 0 : at;
  if (step > 1) {
    r = at + lane;
    le = lane < step && r < n_rows && row_start[r] / div + mult * r <= t;
    const int n = __popcll(__builtin_amdgcn_ballot_w64(le));
    at += n > 0 ? n - 1 : 0;
  }
  return __builtin_amdgcn_readfirstlane(at);
}

hipError_t kv8_plan(const t2w_kv8_plan_args& a, hipStream_t st);
hipError_t kv8_append(const t2w_kv8_append_args& a, hipStream_t st);
hipError_t kv8_attention(const t2w_kv8_attention_args& a, hipStream_t st);
size_t kv8_attention_workspace(const t2w_kv8_attention_args& a);

}  // namespace t2w
