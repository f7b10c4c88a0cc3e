// Attention over the paged 8-bit key/value cache: out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that query
// i sees, key and value codes times their blocks' scales.  Block format: kv8_internal.h.
#include "kv8_internal.h"

namespace t2w {

namespace {

// One wave per (token, head), 32 keys of a block at a time: lane (key, half) sums every other 16-channel chunk of its key
// in fp32, the wave keeps the running maximum and sum, and each lane the output of one or two channels.
template <bool BF, int D>
__global__ void __launch_bounds__(256) kv8_attn_token_kernel(t2w_kv8_attention_args a) {
  __shared__ float s_q[4][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = blockIdx.x, head = blockIdx.y * 4 + wave;
  if (head >= a.heads) return;
  const int kv_head = head / (a.heads / a.pages.kv_heads);
  int lo = 0, hi = a.n_rows;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.row_start[mid] <= n) lo = mid; else hi = mid;
  }
  const int row = lo, start = a.row_start[row], n_new = a.row_start[row + 1] - start, total = a.kv_total[row];
  const int i = n - start;
  if (i < 0 || i >= n_new) return;  // behind the last row
  const int seen_new = a.chunk > 0 ? (int)min((long long)n_new, ((long long)i / a.chunk + 1) * a.chunk) : n_new;
  const int seen = min(max(total - n_new + seen_new, 0), total);
  const bool bad_row = total < 0 || total > a.width * KV8_BLOCK;
  const uint16_t* q = (const uint16_t*)a.q + (long long)n * a.ldq + head * D;
  for (int d = lane; d < D; d += 64) s_q[wave][d] = BF ? bf2f(q[d]) : h2f(q[d]);
  __builtin_amdgcn_wave_barrier();
  constexpr int NV = D / 64;
  float o[NV] = {}, m = -__builtin_inff(), l = 0.f;
  const float c = a.scale * 1.4426950408889634f;
  const int key = lane & 31, half = lane >> 5;
  for (int b = 0; !bad_row && b * KV8_BLOCK < seen; ++b) {
    int id = a.table[(size_t)row * a.ld_table + b];
    const bool bad = (unsigned)id >= (unsigned)a.pages.n_blocks;
    if (bad) id = 0;
    const size_t pg = (size_t)id * a.pages.kv_heads + kv_head;
    const uint8_t* kp = (const uint8_t*)a.pages.k + pg * (KV8_BLOCK * D);
    const uint8_t* vp = (const uint8_t*)a.pages.v + pg * (KV8_BLOCK * D);
    const float ks = ldexpf(1.f, (int)a.pages.k_exp[pg] - 127), vs = ldexpf(1.f, (int)a.pages.v_exp[pg] - 127);
    float s = 0.f;
    for (int ch = half; ch < D / 16; ch += 2) {
      const uint4 u = *(const uint4*)(kp + ch * 512 + key * 16);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto x = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], false);
        const auto y = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], true);
        const float* qq = s_q[wave] + ch * 16 + j * 4;
        s += x[0] * qq[0] + x[1] * qq[1] + y[0] * qq[2] + y[1] * qq[3];
      }
    }
    s += xor32(s);
    s = b * KV8_BLOCK + key < seen ? (bad ? __builtin_nanf("") : s * ks * c) : -__builtin_inff();
    float mx = s;
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w, 64));
    const float mn = fmaxf(m, mx), mr = mn == -__builtin_inff() ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - mr), p = __builtin_amdgcn_exp2f(s - mr);
    float ps = half ? 0.f : p;
    l = l * alpha + wave_sum(ps);
    m = mn;
#pragma unroll
    for (int v = 0; v < NV; ++v) o[v] *= alpha;
    const int left = seen - b * KV8_BLOCK;
    for (int t = 0; t < KV8_BLOCK && t < left; ++t) {
      const float pt = __shfl(p, t, 64) * vs;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int d = lane + 64 * v;
        const int code = vp[(t >> 3) * (8 * D) + (d >> 1) * 16 + (d & 1) * 8 + (t & 7)];
        o[v] += pt * __builtin_amdgcn_cvt_pk_f32_fp8(code, false)[0];
      }
    }
  }
  uint16_t* out = (uint16_t*)a.out + (long long)n * a.ldo + head * D;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const float x = bad_row ? __builtin_nanf("") : l == 0.f ? 0.f : o[v] / l;
    out[lane + 64 * v] = BF ? f2bf(x) : f2h(x);
  }
}

}  // namespace

size_t kv8_attention_workspace(const t2w_kv8_attention_args&) { return 0; }

hipError_t kv8_attention(const t2w_kv8_attention_args& a, hipStream_t st) {
  if (a.n_tok <= 0 || a.n_rows <= 0) return hipSuccess;
  const dim3 grid((unsigned)a.n_tok, (unsigned)((a.heads + 3) / 4));
#define T2W_KV8_ATTN(BF, D) hipLaunchKernelGGL((kv8_attn_token_kernel<BF, D>), grid, dim3(256), 0, st, a)
  if (a.dtype == T2W_KV8_BF16) {
    if (a.pages.head_dim == 64) T2W_KV8_ATTN(true, 64); else T2W_KV8_ATTN(true, 128);
  } else {
    if (a.pages.head_dim == 64) T2W_KV8_ATTN(false, 64); else T2W_KV8_ATTN(false, 128);
  }
#undef T2W_KV8_ATTN
  return hipGetLastError();
}

}  // namespace t2w
