// C-ABI of the operators on 4-bit weights: argument checks in front of mx4.hip.
#include <hip/hip_runtime.h>

#include "../../include/t2w.h"
#include "mx4_internal.h"
#include "rows_overlap.h"

using namespace t2w;

namespace t2w {
int set_error(const char* what, hipError_t e);
}

namespace {

int xerr(const char* what, hipError_t e = hipSuccess) { return set_error(what, e); }

constexpr int MAX_ROWS = 1 << 20, MAX_N = 1 << 24, MAX_K = 1 << 20;

const char* check_size(int n, int k) {
  if (n < 1 || n > MAX_N) return "mx4: n must be 1 to 2^24";
  if (k < 8 || k > MAX_K || k % 8) return "mx4: k must be 8 to 2^20, a multiple of 8";
  return nullptr;
}

const char* check_weight(const t2w_mx4_weight& w) {
  if (const char* e = check_size(w.n, w.k)) return e;
  if (!w.codes || !w.scales) return "mx4: null weight";
  if (((uintptr_t)w.codes & 15) || ((uintptr_t)w.scales & 3)) return "mx4: the weight's codes must be 16-byte aligned, its scales 4-byte";
  return nullptr;
}

// x [m, k] and y [m, n] in 16 bits
const char* check_rows(const void* x, long long ldx, int k, void* y, long long ldy, int n, const void* residual, long long ldr, int dtype, int m) {
  if (dtype != T2W_MX4_BF16 && dtype != T2W_MX4_FP16) return "mx4: dtype must be bf16 or fp16";
  if (m < 0 || m > MAX_ROWS) return "mx4: m must be 0 to 2^20";
  if (m == 0) return nullptr;
  if (!x || !y) return "mx4: null rows";
  if (((uintptr_t)x & 15) || (m > 1 && ldx % 8)) return "mx4: x must be 16-byte aligned, its row stride a multiple of 8";
  if (((uintptr_t)y & 1) || ((uintptr_t)residual & 1)) return "mx4: misaligned outputs or residual";
  if (m > 1 && (ldx < k || ldy < n || (residual && ldr < n))) return "mx4: rows overlap";
  const Rows out{y, ldy * 2, 2LL * n, m};
  if (rows_meet(out, Rows{x, ldx * 2, 2LL * k, m})) return "mx4: the outputs overlap x";
  if (residual && !(residual == y && (ldr == ldy || m == 1)) && rows_meet(out, Rows{residual, ldr * 2, 2LL * n, m})) return "mx4: the outputs overlap the residual";
  return nullptr;
}

// a weight's memory as one row
bool on_weight(const Rows& r, const t2w_mx4_weight& w) {
  const long long c = (long long)t2w_mx4_codes_bytes(w.n, w.k), s = (long long)t2w_mx4_scales_bytes(w.n, w.k);
  return rows_meet(r, Rows{w.codes, c, c, 1}) || rows_meet(r, Rows{w.scales, s, s, 1});
}

// bytes of the parts that a product splits into
size_t part_bytes(int m, int n, int k, long long ldx, bool gated) { return mx4_takes_tiles(m, n, k, ldx, gated) ? mx4_tiles_workspace(m, n, k, gated) : 0; }

// the workspace against what a call needs and its other operands
const char* check_workspace(const void* ws, size_t have, size_t need, const Rows& out, const Rows& x, const void* residual, long long ldr) {
  if (need == 0) return nullptr;
  if (!ws || have < need) return "mx4: workspace too small";
  if ((uintptr_t)ws & 15) return "mx4: workspace must be 16-byte aligned";
  const Rows w{ws, (long long)need, (long long)need, 1};
  if (rows_meet(w, out) || rows_meet(w, x) || (residual && rows_meet(w, Rows{residual, ldr * 2, out.width, out.n}))) return "mx4: the workspace overlaps an operand";
  return nullptr;
}

int run(const Mx4Args& g, int dtype, bool gated, Form form, void* workspace, void* stream, const char* what) {
  Mx4Args a = g;
  const int rows = form == Form::PLAIN ? a.m : gated ? 2 * a.m : a.m / 2;  // of y
  const auto whole = [&](const void* p, long long ld) { return !((uintptr_t)p & 7) && (rows == 1 || ld % 4 == 0); };
  a.quad = a.n % 4 == 0 && whole(a.y, a.ldy) && (!a.residual || whole(a.residual, a.ldr));
  a.half = dtype == T2W_MX4_FP16;
  const bool bf = dtype == T2W_MX4_BF16;
  const hipError_t e = mx4_takes_tiles(a.m, a.n, a.k, a.ldx, gated) ? mx4_tiles(a, bf, gated, form, workspace, (hipStream_t)stream)
                                                                    : mx4_rows(a, bf, gated, form, (hipStream_t)stream);
  return e == hipSuccess ? 0 : xerr(what, e);
}

}  // namespace

namespace {

// what laying a matrix out may not be given: outputs that share bytes with each other or with the `n_in` inputs
const char* check_layout(int n, int k, void* w_codes, void* w_scales, int* status, const Rows* in, int n_in) {
  const long long c = (long long)t2w_mx4_codes_bytes(n, k), s = (long long)t2w_mx4_scales_bytes(n, k);
  const Rows out[3] = {{w_codes, c, c, 1}, {w_scales, s, s, 1}, {status, 4, 4, 1}};
  for (int i = 0; i < 3; ++i) {
    for (int j = 0; j < i; ++j)
      if (rows_meet(out[i], out[j])) return "mx4: the laid out codes, scales and status overlap";
    for (int j = 0; j < n_in; ++j)
      if (rows_meet(out[i], in[j])) return "mx4: an output overlaps an input";
  }
  return nullptr;
}

}  // namespace

extern "C" {

size_t t2w_mx4_codes_bytes(int n, int k) { return check_size(n, k) ? 0 : (size_t)mx4_blocks(n) * mx4_steps(k) * 1024; }
size_t t2w_mx4_scales_bytes(int n, int k) { return check_size(n, k) ? 0 : (size_t)mx4_blocks(n) * mx4_units(k) * 256; }

int t2w_mx4_product_form(int m, int n, int k, long long ldx, int gated, t2w_mx4_form* form) {
  if (const char* e = check_size(n, k)) return xerr(e);
  if (m < 1 || m > 2 * MAX_ROWS || !form) return xerr("mx4 form: 1 to 2^21 rows and a place for the form");
  *form = mx4_takes_tiles(m, n, k, ldx, gated != 0) ? mx4_tiles_form(m, n, k, gated != 0) : t2w_mx4_form{0, 0, 1};
  return 0;
}

int t2w_mx4_pack(const t2w_mx4_pack_args* a, void* stream) {
  if (!a) return xerr("mx4 pack: null arguments");
  if (const char* e = check_size(a->n, a->k)) return xerr(e);
  if (!a->codes || !a->scales || !a->w_codes || !a->w_scales || !a->status) return xerr("mx4 pack: null operand");
  if (((uintptr_t)a->codes & 3) || ((uintptr_t)a->w_codes & 15) || ((uintptr_t)a->w_scales & 3) || ((uintptr_t)a->status & 3)) return xerr("mx4 pack: misaligned operand");
  const long long c = (long long)a->n * (a->k / 2), s = (long long)a->n * ((a->k + 31) / 32);
  const Rows in[2] = {{a->codes, c, c, 1}, {a->scales, s, s, 1}};
  if (const char* e = check_layout(a->n, a->k, a->w_codes, a->w_scales, a->status, in, 2)) return xerr(e);
  const hipError_t e = mx4_pack(*a, (hipStream_t)stream);
  return e == hipSuccess ? 0 : xerr("mx4 pack", e);
}

int t2w_mx4_quantize(const t2w_mx4_quantize_args* a, void* stream) {
  if (!a) return xerr("mx4 quantize: null arguments");
  if (const char* e = check_size(a->n, a->k)) return xerr(e);
  if (a->dtype != T2W_MX4_BF16 && a->dtype != T2W_MX4_FP16 && a->dtype != T2W_MX4_FP32) return xerr("mx4 quantize: dtype must be bf16, fp16 or fp32");
  if (!a->w || !a->w_codes || !a->w_scales || !a->status) return xerr("mx4 quantize: null operand");
  if (((uintptr_t)a->w & (a->dtype == T2W_MX4_FP32 ? 3 : 1)) || ((uintptr_t)a->w_codes & 15) || ((uintptr_t)a->w_scales & 3) || ((uintptr_t)a->status & 3)) return xerr("mx4 quantize: misaligned operand");
  if (a->n > 1 && a->ldw < a->k) return xerr("mx4 quantize: rows overlap");
  const long long size = a->dtype == T2W_MX4_FP32 ? 4 : 2;
  const Rows in{a->w, a->ldw * size, a->k * size, a->n};
  if (const char* e = check_layout(a->n, a->k, a->w_codes, a->w_scales, a->status, &in, 1)) return xerr(e);
  const hipError_t e = mx4_quantize(*a, (hipStream_t)stream);
  return e == hipSuccess ? 0 : xerr("mx4 quantize", e);
}

size_t t2w_mx4_linear_workspace_bytes(const t2w_mx4_linear_args* a) {
  if (!a || check_weight(a->w) || a->m < 1 || a->m > MAX_ROWS) return 0;
  return part_bytes(a->m, a->w.n, a->w.k, a->ldx, false);
}

int t2w_mx4_linear(const t2w_mx4_linear_args* a, void* stream) {
  if (!a) return xerr("mx4 linear: null arguments");
  if (const char* e = check_weight(a->w)) return xerr(e);
  if (const char* e = check_rows(a->x, a->ldx, a->w.k, a->y, a->ldy, a->w.n, a->residual, a->ldr, a->dtype, a->m)) return xerr(e);
  if (a->m == 0) return 0;
  if ((uintptr_t)a->bias & 3) return xerr("mx4: misaligned bias");
  const Rows out{a->y, a->ldy * 2, 2LL * a->w.n, a->m};
  if (on_weight(out, a->w) || (a->bias && rows_meet(out, Rows{a->bias, 4LL * a->w.n, 4LL * a->w.n, 1}))) return xerr("mx4: the outputs overlap the weight or bias");
  const size_t need = t2w_mx4_linear_workspace_bytes(a);
  if (const char* e = check_workspace(a->workspace, a->workspace_bytes, need, out, Rows{a->x, a->ldx * 2, 2LL * a->w.k, a->m}, a->residual, a->ldr)) return xerr(e);
  if (need) {
    const Rows ws{a->workspace, (long long)need, (long long)need, 1};
    if (on_weight(ws, a->w) || (a->bias && rows_meet(ws, Rows{a->bias, 4LL * a->w.n, 4LL * a->w.n, 1}))) return xerr("mx4: the workspace overlaps an operand");
  }
  Mx4Args g{};
  g.w[0] = (const uint8_t*)a->w.codes, g.s[0] = (const uint8_t*)a->w.scales;
  g.x = a->x, g.ldx = a->ldx, g.m = a->m, g.n = a->w.n, g.k = a->w.k;
  g.bias = a->bias, g.residual = a->residual, g.ldr = a->ldr, g.y = a->y, g.ldy = a->ldy;
  return run(g, a->dtype, false, Form::PLAIN, a->workspace, stream, "mx4 linear");
}

static const char* check_gated(const t2w_mx4_weight& gate, const t2w_mx4_weight& up, int act) {
  if (const char* e = check_weight(gate)) return e;
  if (const char* e = check_weight(up)) return e;
  if (gate.n != up.n || gate.k != up.k) return "mx4: the gate's and the up projection's sizes differ";
  if (act != T2W_MX4_SILU && act != T2W_MX4_GELU) return "mx4: act must be silu or gelu";
  return nullptr;
}

static Mx4Args gated_args(const t2w_mx4_weight& gate, const t2w_mx4_weight& up, const void* x, long long ldx, int m, int act, void* y, long long ldy) {
  Mx4Args g{};
  g.w[0] = (const uint8_t*)gate.codes, g.s[0] = (const uint8_t*)gate.scales;
  g.w[1] = (const uint8_t*)up.codes, g.s[1] = (const uint8_t*)up.scales;
  g.x = x, g.ldx = ldx, g.m = m, g.n = gate.n, g.k = gate.k, g.y = y, g.ldy = ldy, g.act = act;
  return g;
}

size_t t2w_mx4_gated_workspace_bytes(const t2w_mx4_gated_args* a) {
  if (!a || check_gated(a->gate, a->up, a->act) || a->m < 1 || a->m > MAX_ROWS) return 0;
  return part_bytes(a->m, a->gate.n, a->gate.k, a->ldx, true);
}

int t2w_mx4_gated(const t2w_mx4_gated_args* a, void* stream) {
  if (!a) return xerr("mx4 gated: null arguments");
  if (const char* e = check_gated(a->gate, a->up, a->act)) return xerr(e);
  if (const char* e = check_rows(a->x, a->ldx, a->gate.k, a->y, a->ldy, a->gate.n, nullptr, 0, a->dtype, a->m)) return xerr(e);
  if (a->m == 0) return 0;
  const Rows out{a->y, a->ldy * 2, 2LL * a->gate.n, a->m};
  if (on_weight(out, a->gate) || on_weight(out, a->up)) return xerr("mx4: the outputs overlap a weight");
  const size_t need = t2w_mx4_gated_workspace_bytes(a);
  if (const char* e = check_workspace(a->workspace, a->workspace_bytes, need, out, Rows{a->x, a->ldx * 2, 2LL * a->gate.k, a->m}, nullptr, 0)) return xerr(e);
  const Rows ws{a->workspace, (long long)need, (long long)need, 1};
  if (need && (on_weight(ws, a->gate) || on_weight(ws, a->up))) return xerr("mx4: the workspace overlaps an operand");
  return run(gated_args(a->gate, a->up, a->x, a->ldx, a->m, a->act, a->y, a->ldy), a->dtype, true, Form::PLAIN, a->workspace, stream, "mx4 gated");
}

// The inner rows lie in the workspace, each at a 16-byte boundary: the second product's matrix operand, of 16 bits.  Wide, a value is two
// rows' sum, which doubles that product (a third of the block's work) and leaves the outputs' errors at their own rounding's.  Rounded
// to x's type once, errors grow to up to sqrt(2) of that (bf16 1.7e-3 to 2.0-2.3e-3, fp16 2.1e-4 to 2.5-3.1e-4, relative) and fp16 loses
// what is beyond 65504.  Wide and rounded, a call: 1 x 4096 x 14336 20.4 and 19.7 us, 16 x 2048 x 5464 16.4 and 13.6, 200 x 4096 x
// 14336 106 and 86, 2005 rows 729 and 543.
static long long inner_ld(const t2w_mx4_ffn_args& a) { return (a.gate.n + 7) / 8 * 8; }
static int inner_rows(const t2w_mx4_ffn_args& a) { return a.inner == T2W_MX4_INNER_WIDE ? 2 * a.m : a.m; }

static const char* check_ffn(const t2w_mx4_ffn_args* a) {
  if (!a) return "mx4 ffn: null arguments";
  if (const char* e = check_gated(a->gate, a->up, a->act)) return e;
  if (const char* e = check_weight(a->down)) return e;
  if (a->inner != T2W_MX4_INNER_ROUNDED && a->inner != T2W_MX4_INNER_WIDE) return "mx4 ffn: inner must be rounded or wide";
  if (a->down.k != a->gate.n) return "mx4 ffn: the down projection's columns are not the gate's channels";
  return check_rows(a->x, a->ldx, a->gate.k, a->y, a->ldy, a->down.n, a->residual, a->ldr, a->dtype, a->m);
}

// the inner rows, then (16-byte aligned: rows are) the parts of whichever product needs more
static size_t inner_bytes(const t2w_mx4_ffn_args& a) { return (size_t)inner_rows(a) * inner_ld(a) * 2; }

size_t t2w_mx4_ffn_workspace_bytes(const t2w_mx4_ffn_args* a) {
  if (!a || check_gated(a->gate, a->up, a->act) || check_weight(a->down) || a->m < 1 || a->m > MAX_ROWS) return 0;
  const size_t p = part_bytes(a->m, a->gate.n, a->gate.k, a->ldx, true), q = part_bytes(inner_rows(*a), a->down.n, a->down.k, inner_ld(*a), false);
  return inner_bytes(*a) + (p > q ? p : q);
}

int t2w_mx4_ffn(const t2w_mx4_ffn_args* a, void* stream) {
  if (const char* e = check_ffn(a)) return xerr(e);
  if (a->m == 0) return 0;
  const size_t need = t2w_mx4_ffn_workspace_bytes(a);
  const Rows out{a->y, a->ldy * 2, 2LL * a->down.n, a->m}, ws{a->workspace, (long long)need, (long long)need, 1};
  if (on_weight(out, a->gate) || on_weight(out, a->up) || on_weight(out, a->down)) return xerr("mx4: the outputs overlap a weight");
  if (const char* e = check_workspace(a->workspace, a->workspace_bytes, need, out, Rows{a->x, a->ldx * 2, 2LL * a->gate.k, a->m}, a->residual, a->ldr)) return xerr(e);
  if (on_weight(ws, a->gate) || on_weight(ws, a->up) || on_weight(ws, a->down)) return xerr("mx4: the workspace overlaps an operand");
  const long long ldh = inner_ld(*a);
  const Form form = a->inner == T2W_MX4_INNER_WIDE ? Form::WIDE : Form::PLAIN;
  void* part = (uint8_t*)a->workspace + inner_bytes(*a);
  if (int rc = run(gated_args(a->gate, a->up, a->x, a->ldx, a->m, a->act, a->workspace, ldh), a->dtype, true, form, part, stream, "mx4 ffn")) return rc;
  Mx4Args g{};
  g.w[0] = (const uint8_t*)a->down.codes, g.s[0] = (const uint8_t*)a->down.scales;
  g.x = a->workspace, g.ldx = ldh, g.m = inner_rows(*a), g.n = a->down.n, g.k = a->down.k;
  g.residual = a->residual, g.ldr = a->ldr, g.y = a->y, g.ldy = a->ldy;
  return run(g, a->dtype, false, form, part, stream, "mx4 ffn");
}

}  // extern "C"
