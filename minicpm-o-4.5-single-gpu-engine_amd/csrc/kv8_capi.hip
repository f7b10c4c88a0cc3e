// C-ABI of the paged 8-bit key/value cache: argument checks in front of kv8.hip and kv8_attn.hip.  What depends on device
// data (lengths, block ids) is checked by the kernels themselves.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/t2w.h"
#include "kv8_internal.h"

using namespace t2w;

namespace t2w {
int set_error(const char* what, hipError_t e);
}

namespace {

int kerr(const char* what, hipError_t e = hipSuccess) { return set_error(what, e); }

bool meet(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + nb && y < x + na;
}

const char* check_pages(const t2w_kv8_pages& p) {
  if (!p.k || !p.v || !p.k_exp || !p.v_exp) return "kv8: null pages";
  if (p.head_dim != 64 && p.head_dim != 128) return "kv8: head_dim must be 64 or 128";
  if (p.kv_heads < 1 || p.kv_heads > 1024) return "kv8: kv_heads must be 1 to 1024";
  if (p.n_blocks < 1 || p.n_blocks > (1 << 26)) return "kv8: n_blocks must be 1 to 2^26";
  if (((uintptr_t)p.k & 15) || ((uintptr_t)p.v & 15)) return "kv8: pages must be 16-byte aligned";
  return nullptr;
}

const char* check_rows(int n_rows, int width, int ld_table) {
  if (n_rows < 0 || n_rows > KV8_MAX_ROWS) return "kv8: n_rows must be 0 to 4096";
  if (width < 1 || width >= (1 << 26) || ld_table < width) return "kv8: table width must be 1 to 2^26 - 1 and at most its row stride";
  return nullptr;
}

}  // namespace

extern "C" {

int t2w_kv8_plan(const t2w_kv8_plan_args* a, void* stream) {
  if (!a) return kerr("kv8 plan: null arguments");
  if (const char* e = check_rows(a->n_rows, a->width, a->ld_table)) return kerr(e);
  if (a->n_tok < 0 || a->n_free < 0) return kerr("kv8 plan: negative n_tok or n_free");
  if (a->n_rows > 0 && (!a->kv_len || !a->new_len || !a->table || !a->kv_total)) return kerr("kv8 plan: null rows");
  if (!a->free_head || !a->free_head_out || !a->row_start || !a->status || (a->n_free > 0 && !a->free_ids)) return kerr("kv8 plan: null free list or output");
  if (a->n_tok > 0 && (!a->tok_row || !a->tok_pos || !a->slots)) return kerr("kv8 plan: null token tables");
  // every workgroup reads the lengths and the head for itself: what is written must not be what another still reads
  const size_t rb = (size_t)a->n_rows * 4, tb = (size_t)a->n_tok * 4;
  const struct { const void* p; size_t n; } in[4] = {{a->kv_len, rb}, {a->new_len, rb}, {a->free_head, 4}, {a->free_ids, (size_t)a->n_free * 4}},
      out[7] = {{a->kv_total, rb}, {a->row_start, rb + 4}, {a->free_head_out, 4}, {a->status, 4}, {a->tok_row, tb}, {a->tok_pos, tb}, {a->slots, tb}};
  for (const auto& x : in)
    for (const auto& y : out)
      if (x.p && y.p && x.n && y.n && meet(x.p, x.n, y.p, y.n)) return kerr("kv8 plan: an output lies on an input");
  const size_t span = a->n_rows > 0 ? ((size_t)(a->n_rows - 1) * a->ld_table + a->width) * 4 : 0;
  for (const auto& x : in)
    if (span && x.n && meet(x.p, x.n, a->table, span)) return kerr("kv8 plan: the table lies on an input");
  for (const auto& y : out)
    if (span && y.n && meet(y.p, y.n, a->table, span)) return kerr("kv8 plan: an output lies on the table");
  const hipError_t e = kv8_plan(*a, (hipStream_t)stream);
  return e == hipSuccess ? 0 : kerr("kv8 plan", e);
}

int t2w_kv8_append(const t2w_kv8_append_args* a, void* stream) {
  if (!a) return kerr("kv8 append: null arguments");
  if (const char* e = check_pages(a->pages)) return kerr(e);
  if (const char* e = check_rows(a->n_rows, a->width, a->ld_table)) return kerr(e);
  if (a->dtype != T2W_KV8_BF16 && a->dtype != T2W_KV8_FP16) return kerr("kv8 append: dtype must be bf16 or fp16");
  if (a->n_tok < 0 || a->max_new < 0) return kerr("kv8 append: negative n_tok or max_new");
  if (a->n_tok == 0 || a->n_rows == 0) return 0;
  if (!a->k || !a->v || !a->table || !a->row_start || !a->kv_total) return kerr("kv8 append: null operand");
  const long long row = (long long)a->pages.kv_heads * a->pages.head_dim;
  if (a->n_tok > 1 && (a->ldk < row || a->ldv < row)) return kerr("kv8 append: token rows overlap");
  if (a->ldk % 8 || a->ldv % 8 || ((uintptr_t)a->k & 15) || ((uintptr_t)a->v & 15)) return kerr("kv8 append: keys and values must be 16-byte aligned, their row strides multiples of 8");
  const hipError_t e = kv8_append(*a, (hipStream_t)stream);
  return e == hipSuccess ? 0 : kerr("kv8 append", e);
}

static const char* check_attention(const t2w_kv8_attention_args* a) {
  if (!a) return "kv8 attention: null arguments";
  if (const char* e = check_pages(a->pages)) return e;
  if (const char* e = check_rows(a->n_rows, a->width, a->ld_table)) return e;
  if (a->dtype != T2W_KV8_BF16 && a->dtype != T2W_KV8_FP16) return "kv8 attention: dtype must be bf16 or fp16";
  if (a->heads < 1 || a->heads % a->pages.kv_heads || a->heads / a->pages.kv_heads > 16) return "kv8 attention: heads must be 1 to 16 times kv_heads";
  if (a->n_tok < 0 || a->chunk < 0 || a->max_new < 0 || a->max_kv < 0) return "kv8 attention: negative n_tok, chunk, max_new or max_kv";
  if (a->n_tok > (1 << 24)) return "kv8 attention: at most 2^24 new tokens";
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return "kv8 attention: scale must be positive and finite";
  return nullptr;
}

size_t t2w_kv8_attention_workspace_bytes(const t2w_kv8_attention_args* a) {
  if (check_attention(a) || a->n_tok == 0 || a->n_rows == 0) return 0;
  return kv8_attention_workspace(*a);
}

int t2w_kv8_attention(const t2w_kv8_attention_args* a, void* stream) {
  if (const char* e = check_attention(a)) return kerr(e);
  if (a->n_tok == 0 || a->n_rows == 0) return 0;
  if (!a->q || !a->out || !a->table || !a->row_start || !a->kv_total) return kerr("kv8 attention: null operand");
  const long long row = (long long)a->heads * a->pages.head_dim;
  if (a->n_tok > 1 && (a->ldq < row || a->ldo < row)) return kerr("kv8 attention: token rows overlap");
  if (a->ldq % 8 || a->ldo % 8 || ((uintptr_t)a->q & 15) || ((uintptr_t)a->out & 15)) return kerr("kv8 attention: q and out must be 16-byte aligned, their row strides multiples of 8");
  const size_t need = kv8_attention_workspace(*a);
  if (need && (!a->workspace || a->workspace_bytes < need)) return kerr("kv8 attention: workspace too small");
  if ((uintptr_t)a->workspace & 15) return kerr("kv8 attention: workspace must be 16-byte aligned");
  const hipError_t e = kv8_attention(*a, (hipStream_t)stream);
  return e == hipSuccess ? 0 : kerr("kv8 attention", e);
}

}  // extern "C"
