// kv_cache.cu - key and value rows of a batch of sequences, quantised as they are written into the cache and read
// back as the values they stand for (rb_kv_write, rb_kv_read). One row is the head_dim values of one (sequence,
// slot, key-value head):
//   RB_KV_INT8   s = bf16(max|x| / 127), c = clamp(rint(x / s), -127, 127); the cache holds c + 128 and s
//   RB_KV_INT4   m = min x (exact in the activation dtype), s = bf16((max x - m) (1 / 15)), the product in fp32,
//                c = clamp(rint((x - m) / s), 0, 15); the cache holds two codes a byte (low nibble = even column) and the
//                pair (s, m). One fp16 row in 200 has a range midway between two scales, which are then equally good: by
//                the product with fp32's 1 / 15, a little above it, the larger one is taken, and no division is needed
//   RB_KV_PLAIN  the row as it is
// The scale is rounded to bf16 BEFORE the codes are computed against it, so its 8 bits cost nothing (127 s and 15 s
// stay within half a step of the largest value) and it keeps fp32's range, which an fp16 scale would not. x (11 bits)
// over s (8 bits) is either exactly a half-integer or at least 2^-16 of itself away from one, so the codes do not
// depend on how wide the quotient is computed.
// A row with a NaN or an infinity gets s = NaN and codes of zero: all of it reads back as NaN, in this kernel and in
// the attention. s == 0 (a row of equal values, or of zeros) gives codes of zero.
// Bound: HBM for prompts, each byte moved once. 65,536 tokens of 8 heads of 128 in int8, written and read back: 135 us
// for 0.81 GB, 0.92 of the measured copy bandwidth; 4,099 tokens in int4 12 us for 42 MB (0.55: a few waves of CTAs). One token of 16 sequences is two launches of 2 us, all latency.
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
  int64_t n_tokens, cache_len;
  uint32_t n_seqs, n_heads, tiles;  // tiles: CTAs of one (key or value, sequence)
};

struct ReadParams {
  const void* c[2];
  const void* par[2];
  void* out[2];
  int64_t start, count, cache_len;
  uint32_t heads, tiles;  // sequences x heads; CTAs of one (key or value, sequence, head)
  int bf16;
};

__device__ __forceinline__ float bf16_round(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }

// The row's result in every one of the kLanes lanes that share it.
template <int kLanes, typename Op>
__device__ __forceinline__ uint32_t row_all(uint32_t v, Op op) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Largest and smallest of a thread's eight values as the 16-bit types order them, NaN winning.
template <bool kBf16, bool kMax>
__device__ __forceinline__ uint32_t pick2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (kBf16) {
    if constexpr (kMax) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  } else {
    if constexpr (kMax) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  }
  return d;
}

__device__ __forceinline__ float act_of(uint32_t bits16, bool bf16) {
  return bf16 ? __uint_as_float(bits16 << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits16)));
}

// The 16-bit pair as fp32.
template <bool kBf16>
__device__ __forceinline__ float2 pair_of(uint32_t w) {
  if constexpr (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

constexpr float kRint = 12582912.f;  // 1.5 2^23: a sum with it is rounded to an integer, held in its low bits

// rint(x / s) of a thread's eight values, clamped to [lo, hi], as integers in the low byte; s > 0. The quotient is the
// product with the reciprocal, corrected once by its exact remainder x - t s (Markstein's method, IBM J. Res. Dev. 34,
// 1990): it is x / s rounded to fp32, so that exact half-integers, 0.3 % of 16-bit values, go to the even code. Rounding
// by the sum with kRint and keeping the integer bits takes no conversion instruction (a quarter of the rate).
__device__ __forceinline__ void quantise8(const float2 (&x)[4], float s, float lo, float hi, uint32_t (&q)[8]) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float2 inv2 = make_float2(inv, inv), s2 = make_float2(-s, -s), c2 = make_float2(kRint, kRint);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 t = fma2(x[e], inv2, make_float2(0.f, 0.f));
    const float2 r = add2(fma2(fma2(t, s2, x[e]), inv2, t), c2);
    q[2 * e] = __float_as_uint(r.x);
    q[2 * e + 1] = __float_as_uint(r.y);
  }
  // a scale so small that the remainder or the scale itself is not a normal number: divide and clamp. Above it
  // |x| <= 127.25 s (15.03 s), so that no code is out of range.
  if (s < 1e-28f) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      q[e] = static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn((e & 1) ? x[e >> 1].y : x[e >> 1].x, s)), lo), hi)));
  }
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// A row of kLanes lanes, eight values (16 bytes) each: its codes to `c` (this lane's) and, from lane 0, its parameters'
// word through `out`.
template <int kLanes, int kFmt, bool kBf16, typename Out>
__device__ __forceinline__ void quantise_row(const uint4 raw, bool store, void* c, Out out) {
  if constexpr (kFmt == RB_KV_PLAIN) {
    if (store) *reinterpret_cast<uint4*>(c) = raw;
  } else {
    const uint32_t r4[4] = {raw.x, raw.y, raw.z, raw.w};
    float2 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = pair_of<kBf16>(r4[e]);
    float s;
    uint32_t word = 0u;
    if constexpr (kFmt == RB_KV_INT8) {
      uint32_t top = r4[0] & 0x7fff7fffu;
#pragma unroll
      for (int e = 1; e < 4; ++e) top = pick2<kBf16, true>(top, r4[e] & 0x7fff7fffu);
      top = row_all<kLanes>(top, [](uint32_t a, uint32_t d) { return pick2<kBf16, true>(a, d); });
      top = pick2<kBf16, true>(top, top >> 16) & 0xffffu;
      // no 11-bit value is 127 times a 9-bit one: top / 127 is never near a tie of bf16, and the product rounds as it does
      s = bf16_round(act_of(top, kBf16) * (1.f / 127.f));
      if (top >= (kBf16 ? 0x7f80u : 0x7c00u)) s = __int_as_float(0x7fc00000);
    } else {
      uint32_t hi2 = r4[0], lo2 = r4[0];
#pragma unroll
      for (int e = 1; e < 4; ++e) hi2 = pick2<kBf16, true>(hi2, r4[e]), lo2 = pick2<kBf16, false>(lo2, r4[e]);
      hi2 = row_all<kLanes>(hi2, [](uint32_t a, uint32_t d) { return pick2<kBf16, true>(a, d); });
      lo2 = row_all<kLanes>(lo2, [](uint32_t a, uint32_t d) { return pick2<kBf16, false>(a, d); });
      const uint32_t lo = pick2<kBf16, false>(lo2, lo2 >> 16) & 0xffffu;
      const float m = act_of(lo, kBf16), range = act_of(pick2<kBf16, true>(hi2, hi2 >> 16) & 0xffffu, kBf16) - m;
      s = range <= 3.402823466e38f ? bf16_round(range * (1.f / 15.f)) : __int_as_float(0x7fc00000);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = add2(x[e], make_float2(-m, -m));
      word = lo << 16;
    }
    word |= __bfloat16_as_ushort(__float2bfloat16_rn(s));
    uint32_t q[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
    if (s > 0.f) quantise8(x, s, kFmt == RB_KV_INT8 ? -127.f : 0.f, kFmt == RB_KV_INT8 ? 127.f : 15.f, q);
    if constexpr (kFmt == RB_KV_INT8) {  // + 128 of a signed byte: its top bit turned over
      if (store)
        *reinterpret_cast<uint2*>(c) =
            make_uint2(low_bytes(q[0], q[1], q[2], q[3]) ^ 0x80808080u, low_bytes(q[4], q[5], q[6], q[7]) ^ 0x80808080u);
    } else {
      const uint32_t even = low_bytes(q[0], q[2], q[4], q[6]), odd = low_bytes(q[1], q[3], q[5], q[7]);
      if (store) *reinterpret_cast<uint32_t*>(c) = even | (odd << 4);
    }
    out(word);
  }
}

// A CTA takes kGroups x kRows rows of one (key or value, sequence); all of a thread's loads go out first, four of 16 bytes,
// which keep HBM busy while other rows' codes are computed. Bound by instructions: 65,536 tokens in int8 84 us, 4.8 TB/s,
// the schedulers busy four cycles of five, with 130 instructions a warp and 32 x 8 values, a quarter of them indices. (Four
// tiles a CTA, with and without the next one's loads under way, save those and took 85 us.) kByHead: consecutive tokens of one head - addresses a
// constant apart, the parameters one contiguous store. Otherwise (fewer than kGroups tokens, a decode step) rows in
// (token, head) order, so that a step of one token is not one row a CTA.
constexpr int kRows = 4;

template <int kHd, int kFmt, bool kBf16, bool kByHead>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const __grid_constant__ WriteParams p) {
  constexpr int kLanes = kHd / 8, kGroups = kThreads / kLanes, kTile = kGroups * kRows;
  constexpr int kRowBytes = kFmt == RB_KV_PLAIN ? 2 * kHd : (kFmt == RB_KV_INT8 ? kHd : kHd / 2);
  constexpr int kParBytes = kFmt == RB_KV_INT8 ? 2 : 4;
  __shared__ uint32_t par[kByHead ? kTile : 1];
  griddep_wait();
  griddep_launch_dependents();
  const int sub = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const uint32_t which_seq = blockIdx.x / p.tiles, tile = blockIdx.x - which_seq * p.tiles;
  const bool second = which_seq >= p.n_seqs;
  const int64_t b = second ? which_seq - p.n_seqs : which_seq;
  const Rows& R = p.r[second];
  const int64_t at = __ldcg(p.pos + b);
  // the tokens with a slot: 0 <= at + t < cache_len (at may be any value: no sum of it is formed before it is known)
  const int64_t t_lo = at >= 0 ? 0 : (at < -p.n_tokens ? p.n_tokens : -at);
  const int64_t t_end = at >= p.cache_len ? 0 : min(p.n_tokens, at < 0 ? p.cache_len + t_lo : p.cache_len - at);
  if (tile == 0 && threadIdx.x == 0 && (t_lo > 0 || t_end < p.n_tokens)) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
  const uint16_t* src = reinterpret_cast<const uint16_t*>(R.x) + b * R.s_seq + sub * 8;
  uint8_t* codes = static_cast<uint8_t*>(R.c) + sub * (kRowBytes / kLanes);
  uint4 raw[kRows];
  if constexpr (kByHead) {
    const uint32_t tt = tile / p.n_heads, h = tile - tt * p.n_heads;
    const int64_t t0 = static_cast<int64_t>(tt) * kTile;
    // relative to the tile: rows [lo, hi) have a slot
    const int lo = static_cast<int>(min(max(t_lo - t0, int64_t(0)), int64_t(kTile)));
    const int hi = static_cast<int>(min(max(t_end - t0, int64_t(0)), int64_t(kTile)));
    if (lo >= hi) return;
    const int64_t row = (b * p.n_heads + h) * p.cache_len + at + t0;  // of the tile's first token; used from `lo` on
    src += h * R.s_head + (t0 + grp) * R.s_tok;
    codes += (row + grp) * kRowBytes;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int x = i * kGroups + grp;
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (x >= lo && x < hi) raw[i] = ldg_cg_128(src + i * kGroups * R.s_tok);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int x = i * kGroups + grp;
      quantise_row<kLanes, kFmt, kBf16>(raw[i], x >= lo && x < hi, codes + i * kGroups * kRowBytes, [&](uint32_t word) {
        if (sub == 0) par[x] = word;
      });
    }
    if constexpr (kFmt != RB_KV_PLAIN) {
      __syncthreads();
      uint8_t* dst = static_cast<uint8_t*>(R.par) + row * kParBytes;
      for (int x = threadIdx.x; x < hi; x += kThreads) {
        if (x < lo) continue;
        if constexpr (kFmt == RB_KV_INT8) reinterpret_cast<uint16_t*>(dst)[x] = static_cast<uint16_t>(par[x]);
        else reinterpret_cast<uint32_t*>(dst)[x] = par[x];
      }
    }
  } else {
    int64_t dst[kRows];  // the row in the cache; -1: nothing to store
    const uint32_t rows = static_cast<uint32_t>(p.n_tokens) * p.n_heads;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const uint32_t x = tile * kTile + i * kGroups + grp;
      const uint32_t t = x / p.n_heads, h = x - t * p.n_heads;
      const bool on = x < rows && t >= t_lo && t < t_end;
      dst[i] = on ? (b * p.n_heads + h) * p.cache_len + at + t : -1;
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (on) raw[i] = ldg_cg_128(src + t * R.s_tok + h * R.s_head);
    }
#pragma unroll 1
    for (int i = 0; i < kRows; ++i) {
      const int64_t d = i < 2 ? (i ? dst[1] : dst[0]) : (i == 2 ? dst[2] : dst[3]);
      const uint4 v = i < 2 ? (i ? raw[1] : raw[0]) : (i == 2 ? raw[2] : raw[3]);
      if (__all_sync(0xffffffffu, d < 0)) continue;  // a step of one token leaves most of the tile empty
      quantise_row<kLanes, kFmt, kBf16>(v, d >= 0, codes + d * kRowBytes, [&](uint32_t word) {
        if (sub != 0 || d < 0) return;
        if constexpr (kFmt == RB_KV_INT8) reinterpret_cast<uint16_t*>(R.par)[d] = static_cast<uint16_t>(word);
        else reinterpret_cast<uint32_t*>(R.par)[d] = word;
      });
    }
  }
}

// fp32 -> the activation dtype, clamped to its finite range (15 s + m of a row that reaches fp16's largest value may
// round past it); NaN stays NaN.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack_act2(float2 v) {
  uint32_t d;
  if constexpr (kBf16) asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(v.y), "f"(v.x));
  else asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(v.y), "f"(v.x));
  return d;
}

// The values of eight codes in `raw` (int8: two words; int4: one) under the row's parameters.
template <int kFmt, bool kBf16>
__device__ __forceinline__ uint4 values_of(const uint2 raw, uint32_t word) {
  const float s = __uint_as_float(word << 16);
  uint32_t o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (kFmt == RB_KV_INT8) {  // a byte under 2^23's exponent, less 2^23 + 128
      const uint32_t w = e < 2 ? raw.x : raw.y, at = 2 * (e & 1);
      const float2 c = make_float2(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 + at)), __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7441 + at)));
      o[e] = pack_act2<kBf16>(mul2(add2(c, make_float2(-8388736.f, -8388736.f)), make_float2(s, s)));
    } else {
      const float m = act_of(word >> 16, kBf16);
      const float2 c = make_float2(__uint_as_float(((raw.x >> (8 * e)) & 15u) | 0x4B000000u), __uint_as_float(((raw.x >> (8 * e + 4)) & 15u) | 0x4B000000u));
      o[e] = pack_act2<kBf16>(fma2(add2(c, make_float2(-8388608.f, -8388608.f)), make_float2(s, s), make_float2(m, m)));
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// A CTA reads kThreads x kUnits pieces of eight values of one (key or value, sequence, head); its loads go out first.
// HBM-bound: the values that it writes are two to four times the codes it reads. A thread's pieces are kThreads apart, so
// their addresses and their rows' differ by constants.
constexpr int kUnits = 4;

template <int kHd, int kFmt>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int kLanes = kHd / 8, kRowsApart = kThreads / kLanes;
  griddep_wait();
  griddep_launch_dependents();
  const uint32_t line = blockIdx.x / p.tiles;
  const int64_t u0 = static_cast<int64_t>(blockIdx.x - line * p.tiles) * (kThreads * kUnits) + threadIdx.x, units = p.count * kLanes;
  const int which = line >= p.heads;
  const int64_t bh = which ? line - p.heads : line, src = bh * p.cache_len + p.start;
  const int left = static_cast<int>(min(max(units - u0, int64_t(0)), int64_t(kThreads * kUnits)));  // piece i is there: i kThreads < left
  uint4* out = reinterpret_cast<uint4*>(p.out[which]) + bh * units + u0;
  const int64_t at = src * kLanes + u0, row = src + u0 / kLanes;
  if constexpr (kFmt == RB_KV_PLAIN) {
    const uint4* from = reinterpret_cast<const uint4*>(p.c[which]) + at;
    uint4 raw[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
      if (i * kThreads < left) raw[i] = ldg_cg_128(from + i * kThreads);
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
      if (i * kThreads < left) out[i * kThreads] = raw[i];
  } else {
    uint2 raw[kUnits];
    uint32_t word[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      raw[i] = make_uint2(0u, 0u);
      word[i] = 0u;
      if (i * kThreads >= left) continue;
      if constexpr (kFmt == RB_KV_INT8) {
        raw[i] = __ldcg(reinterpret_cast<const uint2*>(p.c[which]) + at + i * kThreads);
        word[i] = __ldcg(reinterpret_cast<const unsigned short*>(p.par[which]) + row + i * kRowsApart);
      } else {
        raw[i].x = __ldcg(reinterpret_cast<const unsigned int*>(p.c[which]) + at + i * kThreads);
        word[i] = __ldcg(reinterpret_cast<const unsigned int*>(p.par[which]) + row + i * kRowsApart);
      }
    }
    if (p.bf16) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        if (i * kThreads < left) out[i * kThreads] = values_of<kFmt, true>(raw[i], word[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        if (i * kThreads < left) out[i * kThreads] = values_of<kFmt, false>(raw[i], word[i]);
    }
  }
}

template <typename P>
int launch(void (*kern)(P), const P& p, int64_t blocks, int flags, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (flags & RB_FLAG_PDL) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? RB_OK : RB_ERR_LAUNCH;
}

template <bool kByHead>
auto write_kernel(int fmt, bool wide, bool bf) -> void (*)(WriteParams) {
  if (fmt == RB_KV_PLAIN) return wide ? kv_write_kernel<128, RB_KV_PLAIN, false, kByHead> : kv_write_kernel<64, RB_KV_PLAIN, false, kByHead>;
  if (fmt == RB_KV_INT8)
    return wide ? (bf ? kv_write_kernel<128, RB_KV_INT8, true, kByHead> : kv_write_kernel<128, RB_KV_INT8, false, kByHead>)
                : (bf ? kv_write_kernel<64, RB_KV_INT8, true, kByHead> : kv_write_kernel<64, RB_KV_INT8, false, kByHead>);
  return wide ? (bf ? kv_write_kernel<128, RB_KV_INT4, true, kByHead> : kv_write_kernel<128, RB_KV_INT4, false, kByHead>)
              : (bf ? kv_write_kernel<64, RB_KV_INT4, true, kByHead> : kv_write_kernel<64, RB_KV_INT4, false, kByHead>);
}

}  // namespace kvc

int launch_kv_write(const rb_kv_cache* c, const void* k, const void* v, const int64_t* ks, const int64_t* vs,
                    int64_t n_tokens, const int64_t* pos, int flags, cudaStream_t stream) {
  using namespace kvc;
  WriteParams p = {};
  p.r[0] = {k, ks[0], ks[1], ks[2], c->k, c->k_par};
  p.r[1] = {v, vs[0], vs[1], vs[2], c->v, c->v_par};
  p.pos = pos;
  p.n_tokens = n_tokens;
  p.cache_len = c->cache_len;
  p.n_heads = static_cast<uint32_t>(c->n_kv_heads);
  p.n_seqs = static_cast<uint32_t>(c->n_seqs);
  const int64_t groups = kThreads / (c->head_dim / 8), tile = groups * kRows;
  const bool by_head = n_tokens >= groups;
  const int64_t tiles = by_head ? (n_tokens + tile - 1) / tile * c->n_kv_heads : (n_tokens * c->n_kv_heads + tile - 1) / tile;
  const int64_t blocks = 2 * c->n_seqs * tiles;
  if (blocks > (int64_t(1) << 31) - 1) return RB_ERR_SHAPE;
  p.tiles = static_cast<uint32_t>(tiles);
  const bool bf = c->dtype == RB_BF16, wide = c->head_dim == 128;
  void (*kern)(WriteParams) = by_head ? write_kernel<true>(c->fmt, wide, bf) : write_kernel<false>(c->fmt, wide, bf);
  return launch(kern, p, blocks, flags, stream);
}

int launch_kv_read(const rb_kv_cache* c, void* k_out, void* v_out, int64_t start, int64_t count, int flags,
                   cudaStream_t stream) {
  using namespace kvc;
  ReadParams p = {};
  p.c[0] = c->k;
  p.c[1] = c->v;
  p.par[0] = c->k_par;
  p.par[1] = c->v_par;
  p.out[0] = k_out;
  p.out[1] = v_out;
  p.start = start;
  p.count = count;
  p.cache_len = c->cache_len;
  p.heads = static_cast<uint32_t>(c->n_seqs * c->n_kv_heads);
  p.bf16 = c->dtype == RB_BF16;
  const int64_t tiles = (count * (c->head_dim / 8) + kThreads * kUnits - 1) / (kThreads * kUnits);
  const int64_t blocks = 2 * c->n_seqs * c->n_kv_heads * tiles;
  if (blocks > (int64_t(1) << 31) - 1) return RB_ERR_SHAPE;
  p.tiles = static_cast<uint32_t>(tiles);
  void (*kern)(ReadParams) = nullptr;
  if (c->head_dim == 128)
    kern = c->fmt == RB_KV_INT8 ? kv_read_kernel<128, RB_KV_INT8>
                                : (c->fmt == RB_KV_INT4 ? kv_read_kernel<128, RB_KV_INT4> : kv_read_kernel<128, RB_KV_PLAIN>);
  else
    kern = c->fmt == RB_KV_INT8 ? kv_read_kernel<64, RB_KV_INT8>
                                : (c->fmt == RB_KV_INT4 ? kv_read_kernel<64, RB_KV_INT4> : kv_read_kernel<64, RB_KV_PLAIN>);
  return launch(kern, p, blocks, flags, stream);
}

}  // namespace rb
