// kv_cache.cu - key and value rows of a batch of sequences, quantised as they are written into the cache and read
// back as the values they stand for (rb_kv_write, rb_kv_read). One row is the head_dim values of one (sequence,
// slot, key-value head):
//   RB_KV_INT8   s = bf16(max|x| / 127), c = clamp(rint(x / s), -127, 127); the cache holds c + 128 and s
//   RB_KV_INT4   m = min x (exact in the activation dtype), s = bf16((max x - m) / 15), c = clamp(rint((x - m) / s),
//                0, 15); the cache holds two codes a byte (low nibble = even column) and the pair (s, m)
//   RB_KV_PLAIN  the row as it is
// The scale is rounded to bf16 BEFORE the codes are computed against it, so its 8 bits cost nothing (127 s and 15 s
// stay within half a step of the largest value) and it keeps fp32's range, which an fp16 scale would not. x (11 bits)
// over s (8 bits) is either exactly a half-integer or at least 2^-16 of itself away from one, so the codes do not
// depend on how wide the quotient is computed.
// A row with a NaN or an infinity gets s = NaN and codes of zero: all of it reads back as NaN, in this kernel and in
// the attention. s == 0 (a row of equal values, or of zeros) gives codes of zero.
#include "common.cuh"
#include "kernels.h"

namespace rb {

namespace kvc {

constexpr int kThreads = 256;

struct Rows {  // one of k, v: the row source (or destination) and the cache side
  const void* x;
  int64_t s_seq, s_tok, s_head;  // elements
  void* c;
  void* par;
};

struct WriteParams {
  Rows r[2];
  const int64_t* pos;
  int64_t n_seqs, n_tokens, cache_len;
  int n_heads, bf16;
};

struct ReadParams {
  const void* c[2];
  const void* par[2];
  void* out[2];
  int64_t n_seqs, start, count, cache_len;
  int n_heads, bf16;
};

// Largest value of the group of kLanes lanes that share a row.
template <int kLanes>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int kLanes>
__device__ __forceinline__ bool group_any(bool b) {
  const unsigned m = __ballot_sync(0xffffffffu, b);
  const int first = (threadIdx.x & 31) / kLanes * kLanes;
  return (m >> first) & (kLanes == 32 ? 0xffffffffu : (1u << kLanes) - 1u);
}

__device__ __forceinline__ float bf16_round(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }

// kLanes lanes hold a row, 8 values each (one 16-byte load).
template <int kHd, int kFmt>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const __grid_constant__ WriteParams p) {
  constexpr int kLanes = kHd / 8;
  griddep_wait();
  griddep_launch_dependents();
  const int sub = threadIdx.x % kLanes;
  const int64_t rows = 2 * p.n_seqs * p.n_tokens * p.n_heads;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kLanes);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads / kLanes);
  // every lane of a warp takes part in the row reductions: the loop bound is the same for the whole CTA
  for (int64_t base = first; base < rows; base += step) {
    const int64_t row = base + threadIdx.x / kLanes;
    const bool in = row < rows;
    int64_t i = in ? row : 0;
    const int h = static_cast<int>(i % p.n_heads);
    i /= p.n_heads;
    const int64_t t = i % p.n_tokens;
    i /= p.n_tokens;
    const int64_t b = i % p.n_seqs;
    const Rows& R = p.r[i / p.n_seqs];
    const int64_t at = p.pos[b];
    const bool fits = at >= -t && at < p.cache_len - t;  // 0 <= at + t < cache_len, without the sum (at may be any)
    if (in && !fits && sub == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
    const int64_t slot = fits ? at + t : 0;
    const uint4 raw = ldg_cg_128(reinterpret_cast<const uint16_t*>(R.x) + b * R.s_seq + t * R.s_tok + h * R.s_head + sub * 8);
    const int64_t dst = (b * p.n_heads + h) * p.cache_len + slot;
    const bool store = in && fits;
    if constexpr (kFmt == RB_KV_PLAIN) {
      if (store) reinterpret_cast<uint4*>(R.c)[dst * kLanes + sub] = raw;
      continue;
    }
    float x[8];
    raw_to_f32(raw, p.bf16 != 0, x);
    if constexpr (kFmt == RB_KV_INT8) {
      float top = 0.f;
      bool odd = false;  // NaN or infinity
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = fmaxf(top, fabsf(x[e]));
        odd |= !(fabsf(x[e]) <= 3.402823466e38f);
      }
      top = group_max<kLanes>(top);
      odd = group_any<kLanes>(odd);
      const float s = odd ? __int_as_float(0x7fc00000) : bf16_round(__fdiv_rn(top, 127.f));
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[e], s)), -127.f), 127.f) : 0.f;
        w[e >> 2] |= static_cast<uint32_t>(static_cast<int>(q) + 128) << (8 * (e & 3));
      }
      if (store) {
        reinterpret_cast<uint2*>(R.c)[dst * kLanes + sub] = make_uint2(w[0], w[1]);
        if (sub == 0) reinterpret_cast<__nv_bfloat16*>(R.par)[dst] = __float2bfloat16_rn(s);
      }
    } else {
      float hi = x[0], lo = -x[0];
      bool odd = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        hi = fmaxf(hi, x[e]);
        lo = fmaxf(lo, -x[e]);
        odd |= !(fabsf(x[e]) <= 3.402823466e38f);
      }
      hi = group_max<kLanes>(hi);
      const float m = -group_max<kLanes>(lo);
      odd = group_any<kLanes>(odd);
      const float range = hi - m;
      const float s = odd || !(range <= 3.402823466e38f) ? __int_as_float(0x7fc00000) : bf16_round(__fdiv_rn(range, 15.f));
      uint32_t w = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[e] - m, s)), 0.f), 15.f) : 0.f;
        w |= static_cast<uint32_t>(static_cast<int>(q)) << (4 * e);
      }
      if (store) {
        reinterpret_cast<uint32_t*>(R.c)[dst * kLanes + sub] = w;
        if (sub == 0) {
          const uint32_t mb = p.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(m)) : __half_as_ushort(__float2half_rn(m));
          reinterpret_cast<uint32_t*>(R.par)[dst] = __bfloat16_as_ushort(__float2bfloat16_rn(s)) | (mb << 16);
        }
      }
    }
  }
}

// fp32 -> the activation dtype, clamped to its finite range (15 s + m of a row that reaches fp16's largest value may
// round past it); NaN stays NaN.
__device__ __forceinline__ uint32_t pack_act2(float a, float b, bool bf16) {
  const float top = bf16 ? 3.3895313892515355e38f : 65504.f;
  a = a > top ? top : (a < -top ? -top : a);
  b = b > top ? top : (b < -top ? -top : b);
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int kHd, int kFmt>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int kLanes = kHd / 8;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t units = 2 * p.n_seqs * p.n_heads * p.count * kLanes;  // 8 values each
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; u < units; u += step) {
    const int sub = static_cast<int>(u % kLanes);
    const int64_t row = u / kLanes;
    const int64_t t = row % p.count;
    int64_t i = row / p.count;
    const int64_t bh = i % (p.n_seqs * p.n_heads);
    const int which = static_cast<int>(i / (p.n_seqs * p.n_heads));
    const int64_t src = bh * p.cache_len + p.start + t;
    uint4* out = reinterpret_cast<uint4*>(p.out[which]) + (bh * p.count + t) * kLanes + sub;
    if constexpr (kFmt == RB_KV_PLAIN) {
      *out = ldg_cg_128(reinterpret_cast<const uint4*>(p.c[which]) + src * kLanes + sub);
    } else {
      float v[8];
      if constexpr (kFmt == RB_KV_INT8) {
        const uint2 w = __ldcg(reinterpret_cast<const uint2*>(p.c[which]) + src * kLanes + sub);
        const float s = __uint_as_float(static_cast<uint32_t>(__ldcg(reinterpret_cast<const unsigned short*>(p.par[which]) + src)) << 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t c = ((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 255u;
          v[e] = static_cast<float>(static_cast<int>(c) - 128) * s;
        }
      } else {
        const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(p.c[which]) + src * kLanes + sub);
        const uint32_t sm = __ldcg(reinterpret_cast<const uint32_t*>(p.par[which]) + src);
        const float s = __uint_as_float(sm << 16);
        const float m = p.bf16 ? __uint_as_float(sm & 0xffff0000u) : __half2float(__ushort_as_half(static_cast<unsigned short>(sm >> 16)));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(static_cast<float>((w >> (4 * e)) & 15u), s, m);
      }
      *out = make_uint4(pack_act2(v[0], v[1], p.bf16), pack_act2(v[2], v[3], p.bf16), pack_act2(v[4], v[5], p.bf16),
                        pack_act2(v[6], v[7], p.bf16));
    }
  }
}

template <typename P>
int launch(void (*kern)(P), const P& p, int64_t blocks, int num_sms, int flags, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 16 * static_cast<int64_t>(num_sms))));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (flags & RB_FLAG_PDL) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? RB_OK : RB_ERR_LAUNCH;
}

}  // namespace kvc

int launch_kv_write(const rb_kv_cache* c, const void* k, const void* v, const int64_t* ks, const int64_t* vs,
                    int64_t n_tokens, const int64_t* pos, int num_sms, int flags, cudaStream_t stream) {
  using namespace kvc;
  WriteParams p = {};
  p.r[0] = {k, ks[0], ks[1], ks[2], c->k, c->k_par};
  p.r[1] = {v, vs[0], vs[1], vs[2], c->v, c->v_par};
  p.pos = pos;
  p.n_seqs = c->n_seqs;
  p.n_tokens = n_tokens;
  p.cache_len = c->cache_len;
  p.n_heads = c->n_kv_heads;
  p.bf16 = c->dtype == RB_BF16;
  const int64_t per = kThreads / (c->head_dim / 8);
  const int64_t blocks = (2 * c->n_seqs * n_tokens * c->n_kv_heads + per - 1) / per;
  void (*kern)(WriteParams) = nullptr;
  if (c->head_dim == 128)
    kern = c->fmt == RB_KV_INT8 ? kv_write_kernel<128, RB_KV_INT8>
                                : (c->fmt == RB_KV_INT4 ? kv_write_kernel<128, RB_KV_INT4> : kv_write_kernel<128, RB_KV_PLAIN>);
  else
    kern = c->fmt == RB_KV_INT8 ? kv_write_kernel<64, RB_KV_INT8>
                                : (c->fmt == RB_KV_INT4 ? kv_write_kernel<64, RB_KV_INT4> : kv_write_kernel<64, RB_KV_PLAIN>);
  return launch(kern, p, blocks, num_sms, flags, stream);
}

int launch_kv_read(const rb_kv_cache* c, void* k_out, void* v_out, int64_t start, int64_t count, int num_sms, int flags,
                   cudaStream_t stream) {
  using namespace kvc;
  ReadParams p = {};
  p.c[0] = c->k;
  p.c[1] = c->v;
  p.par[0] = c->k_par;
  p.par[1] = c->v_par;
  p.out[0] = k_out;
  p.out[1] = v_out;
  p.n_seqs = c->n_seqs;
  p.start = start;
  p.count = count;
  p.cache_len = c->cache_len;
  p.n_heads = c->n_kv_heads;
  p.bf16 = c->dtype == RB_BF16;
  const int64_t blocks = (2 * c->n_seqs * c->n_kv_heads * count * (c->head_dim / 8) + kThreads - 1) / kThreads;
  void (*kern)(ReadParams) = nullptr;
  if (c->head_dim == 128)
    kern = c->fmt == RB_KV_INT8 ? kv_read_kernel<128, RB_KV_INT8>
                                : (c->fmt == RB_KV_INT4 ? kv_read_kernel<128, RB_KV_INT4> : kv_read_kernel<128, RB_KV_PLAIN>);
  else
    kern = c->fmt == RB_KV_INT8 ? kv_read_kernel<64, RB_KV_INT8>
                                : (c->fmt == RB_KV_INT4 ? kv_read_kernel<64, RB_KV_INT4> : kv_read_kernel<64, RB_KV_PLAIN>);
  return launch(kern, p, blocks, num_sms, flags, stream);
}

}  // namespace rb
