// Launch interfaces of the operators on 4-bit weights (mx4.hip: layout and few-row products).  The arguments are checked in
// mx4_capi.hip.
//
// A weight matrix [n, k] in the order its kernels read, made once by t2w_mx4_pack or t2w_mx4_quantize: blocks of 16 output
// channels by steps of 128 columns, 1,024 bytes each:
//   codes   [ceil(n / 16)][ceil(k / 128)][64 lanes][16 bytes]   lane l: channel l % 16, the 32 columns (one group) from
//           32 (l / 16) of the step on, two codes a byte, the even column in the lower nibble
//   scales  [ceil(n / 16)][ceil(k / 512)][64 lanes][4]          lane l's group scales of four steps
// A lane's 16 bytes are its operand of four 16 x 16 x 32 matrix instructions: instruction j takes bytes 4 j .. 4 j + 3, that is
// columns 32 (l / 16) + 8 j .. + 7, and the other operand's lanes take the same columns.  A wave loads 1,024 contiguous bytes, and
// every lane converts with one scale of its own.  Channels and columns behind the last hold zero codes.
#pragma once

#include <type_traits>

#include "../../include/t2w.h"
#include "common.h"

namespace t2w {

constexpr int MX4_EMIN = -23, MX4_EMAX = 13;  // scales' exponents: 0.5 * 2^-23 and 6 * 2^13 are exact in fp16 (and bf16)

inline int mx4_blocks(int n) { return (n + 15) / 16; }
inline int mx4_steps(int k) { return (k + 127) / 128; }
inline int mx4_units(int k) { return (k + 511) / 512; }

// One product (or the two of a gated block) over the rows of x.
//
// Wide inner values (Form::WIDE) stand between a gated block and the product behind it: the block writes each value h as two bf16
// rows, 2 r the nearest bf16 and 2 r + 1 the nearest to what that leaves (h to 2^-16 of it, over fp32's range), and the product runs
// on those 2 m rows (of bf16, whatever the outputs' type: the weights are exact in both) and adds two rows' sums at the end.
enum class Form { PLAIN, WIDE };

struct Mx4Args {
  const uint8_t* w[2];  // codes and scales; [1]: the second matrix of a gated block
  const uint8_t* s[2];
  const void* x;
  long long ldx;
  int m, n, k;
  const float* bias;
  const void* residual;
  long long ldr;
  void* y;
  long long ldy;
  int act;   // of a gated block: T2W_MX4_SILU, T2W_MX4_GELU
  int quad;  // y's (and residual's) groups of four columns are whole and 8-byte aligned
  int half;  // of a product on wide rows: y and the residual are fp16, else bf16
};

hipError_t mx4_pack(const t2w_mx4_pack_args& a, hipStream_t st);
hipError_t mx4_quantize(const t2w_mx4_quantize_args& a, hipStream_t st);
// The products: few rows (mx4.hip) and tiles (mx4_tile.hip), which may split k over workgroups (fp32 parts in the workspace,
// joined by a second kernel).
hipError_t mx4_rows(const Mx4Args& a, bool bf, bool gated, Form form, hipStream_t st);
int mx4_rows_outside(int m, int k, bool gated);  // units of 512 columns of x that do not fit the LDS
bool mx4_takes_tiles(int m, int n, int k, long long ldx, bool gated);
size_t mx4_tiles_workspace(int m, int n, int k, bool gated);
t2w_mx4_form mx4_tiles_form(int m, int n, int k, bool gated);
hipError_t mx4_tiles(const Mx4Args& a, bool bf, bool gated, Form form, void* workspace, hipStream_t st);

// f(bf16 operands?, gated?, form) with compile-time arguments
template <class F>
hipError_t mx4_dispatch(bool bf, bool gated, Form form, F&& f) {
  constexpr std::true_type y{};
  constexpr std::false_type n{};
  constexpr std::integral_constant<Form, Form::PLAIN> plain{};
  constexpr std::integral_constant<Form, Form::WIDE> wide{};
  if (form == Form::WIDE) {
    if (!gated) return f(y, n, wide);
    return bf ? f(y, y, wide) : f(n, y, wide);
  }
  if (gated) return bf ? f(y, y, plain) : f(n, y, plain);
  return bf ? f(y, n, plain) : f(n, n, plain);
}

}  // namespace t2w
