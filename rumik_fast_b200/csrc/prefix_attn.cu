// prefix_attn.cu - decode attention of a batch of sequences that share a prefix (rb_prefix_attn), grouped-query heads,
// over KV caches in any of rb_kv_cache's formats:
//   out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, h] . k_j),
//   j over the prefix's slots [0, *prefix_len) and sequence b's own slots [0, own_len[b]); no slot at all: zeros.
// A quantised row enters the products as its codes, exact small integers: q . (s c + m) = s (q . c) + m sum(q) for a
// key, p (s c + m) = (p s) c + p m for a value, so the scales multiply scores and probabilities, never elements.
#include "common.cuh"
#include "kernels.h"

namespace rb {

namespace pfx {

struct Side {
  const void* k;
  const void* v;
  const void* k_par;
  const void* v_par;
  const int64_t* len;
  int64_t cache_len;
};

struct Params {
  const void* q;
  void* out;
  int64_t ldq, ldo;
  Side pre, own;
  int n_seqs, n_q, n_kv, bf16;
  float scale;
};

constexpr int kWarps = 8;

// One CTA per (query head, sequence): each warp takes every eighth slot, a lane holds head_dim / 32 columns.
template <int kHd, int kFmt>
__global__ void __launch_bounds__(kWarps * 32) prefix_attn_kernel(const __grid_constant__ Params p) {
  constexpr int kE = kHd / 32;
  __shared__ float so[kWarps][kHd], sm[kWarps], sl[kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x, b = blockIdx.y, kv = h / (p.n_q / p.n_kv);
  const int64_t np = p.pre.k ? *p.pre.len : 0, no = p.own.k ? p.own.len[b] : 0;
  if (np < 0 || np > p.pre.cache_len || no < 0 || no > p.own.cache_len) {
    if (threadIdx.x == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
    return;
  }
  float q[kE], o[kE], qs = 0.f, m = -INFINITY, l = 0.f;
  for (int e = 0; e < kE; ++e) {
    q[e] = load_act(p.q, b * p.ldq + static_cast<int64_t>(h) * kHd + lane * kE + e, p.bf16) * p.scale;
    qs += q[e];
    o[e] = 0.f;
  }
  for (int64_t j = warp; j < np + no; j += kWarps) {
    const Side& S = j < np ? p.pre : p.own;
    const int64_t row = j < np ? kv * S.cache_len + j : (static_cast<int64_t>(b) * p.n_kv + kv) * S.cache_len + j - np;
    float k[kE], v[kE], ks = 1.f, km = 0.f, vs = 1.f, vm = 0.f;
    for (int e = 0; e < kE; ++e) {
      const int64_t at = row * kHd + lane * kE + e;
      if (kFmt == RB_KV_PLAIN) {
        k[e] = load_act(S.k, at, p.bf16);
        v[e] = load_act(S.v, at, p.bf16);
      } else if (kFmt == RB_KV_INT8) {
        k[e] = static_cast<float>(static_cast<const uint8_t*>(S.k)[at]) - 128.f;
        v[e] = static_cast<float>(static_cast<const uint8_t*>(S.v)[at]) - 128.f;
      } else {
        k[e] = static_cast<float>((static_cast<const uint8_t*>(S.k)[at / 2] >> (4 * (at & 1))) & 15);
        v[e] = static_cast<float>((static_cast<const uint8_t*>(S.v)[at / 2] >> (4 * (at & 1))) & 15);
      }
    }
    if (kFmt == RB_KV_INT8) {
      ks = load_act(S.k_par, row, true);
      vs = load_act(S.v_par, row, true);
    } else if (kFmt == RB_KV_INT4) {
      ks = load_act(S.k_par, 2 * row, true);
      vs = load_act(S.v_par, 2 * row, true);
      km = load_act(S.k_par, 2 * row + 1, p.bf16);
      vm = load_act(S.v_par, 2 * row + 1, p.bf16);
    }
    float s = 0.f;
    for (int e = 0; e < kE; ++e) s += q[e] * (k[e] * ks + km);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.f : expf(m - mn), pr = s == -INFINITY ? 0.f : expf(s - mn);
    m = mn;
    l = l * f + pr;
    for (int e = 0; e < kE; ++e) o[e] = o[e] * f + pr * (v[e] * vs + vm);
  }
  for (int e = 0; e < kE; ++e) so[warp][lane * kE + e] = o[e];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kHd; d += kWarps * 32) {
    float mx = -INFINITY, lt = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm[w]);
    for (int w = 0; w < kWarps; ++w) {
      const float f = sm[w] == -INFINITY ? 0.f : expf(sm[w] - mx);
      lt += sl[w] * f;
      acc += so[w][d] * f;
    }
    store_out(p.out, b * p.ldo + static_cast<int64_t>(h) * kHd + d, np + no == 0 ? 0.f : acc / lt, p.bf16);
  }
}

}  // namespace pfx

int64_t prefix_attn_workspace(const rb_prefix_attn_args*, int) { return 16; }

int launch_prefix_attn(const rb_prefix_attn_args* a, int num_sms, int flags, cudaStream_t stream) {
  using namespace pfx;
  const rb_kv_cache* any = a->prefix ? a->prefix : a->own;
  Params p = {};
  p.q = a->q;
  p.out = a->out;
  p.ldq = a->ldq;
  p.ldo = a->ldo;
  if (a->prefix) p.pre = {a->prefix->k, a->prefix->v, a->prefix->k_par, a->prefix->v_par, a->prefix_len, a->prefix->cache_len};
  if (a->own) p.own = {a->own->k, a->own->v, a->own->k_par, a->own->v_par, a->own_len, a->own->cache_len};
  p.n_seqs = static_cast<int>(a->n_seqs);
  p.n_q = a->n_q_heads;
  p.n_kv = any->n_kv_heads;
  p.bf16 = any->dtype == RB_BF16;
  p.scale = a->scale;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_q, p.n_seqs);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (flags & RB_FLAG_PDL) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void (*kern)(Params);
  if (any->head_dim == 128)
    kern = any->fmt == RB_KV_INT8 ? prefix_attn_kernel<128, RB_KV_INT8>
                                  : (any->fmt == RB_KV_INT4 ? prefix_attn_kernel<128, RB_KV_INT4> : prefix_attn_kernel<128, RB_KV_PLAIN>);
  else
    kern = any->fmt == RB_KV_INT8 ? prefix_attn_kernel<64, RB_KV_INT8>
                                  : (any->fmt == RB_KV_INT4 ? prefix_attn_kernel<64, RB_KV_INT4> : prefix_attn_kernel<64, RB_KV_PLAIN>);
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? RB_OK : RB_ERR_LAUNCH;
}

}  // namespace rb
