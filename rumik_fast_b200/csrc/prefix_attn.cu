// prefix_attn.cu - decode attention of a batch of sequences that share a prefix (rb_prefix_attn), grouped-query heads,
// over KV caches in any of rb_kv_cache's formats:
//   out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, h] . k_j),
//   j over the prefix's slots [0, *prefix_len) and sequence b's own slots [0, own_len[b]); no slot at all: zeros.
// A quantised row enters the products as its codes, exact small integers: q . (s c + m) = s (q . c) + m sum(q) for a
// key, p (s c + m) = (p s) c + p m for a value, so the scales multiply scores and probabilities, never elements, and
// no rounding is added to the codes'.
//
// The query rows of one key-value head, r = b rep + j over the whole batch, share its keys: they are the M side of the
// two products. One pass over the slots keeps, per row, a reference R (log2 units), l = sum 2^(t - R) and
// O = sum 2^(t - R) v in fp32 (t: the score times log2 e). Any R gives the same O / l. It is chosen for the 16-bit factor
// of the second product, 2^(t - R) s: R is the largest t + e so far, e the exponent of the slot's value scale (0 for 16-bit
// rows), less kRoom, and is only raised when a slot exceeds it by kSlack more, so the accumulators are rarely rescaled. So
// what counts is a slot's weight times its values: one of large values and no weight takes no accuracy from the others,
// nor does one of much weight and no values (a reference from the scores and the largest scale by themselves would).
//
// 16 bits hold, beside the caches' own rounding: the factors 2^(t - R) s, rounded to fp16 (2^-11 of themselves, 2^-31 of the
// row's largest where they are subnormal; 4-bit rows add the remainder as a second term), or for bf16 rows to bf16 (2^-8:
// products on the tensor cores take both operands in one type); and bf16 queries over codes, as fp16 under a power of
// two of their row. l sums the factors before they are rounded, in fp32 like the scores and O.
//
// Work is cut along the slots so that every SM streams a share of the caches: CTAs take (key-value head, 16 wm rows,
// split of the prefix) or (sequence, key-value head, split of its own rows) items and leave an fp32 partial
// (R, l, O) each, which prefix_attn_merge joins in split order (deterministic).
//
// Bound: the latency of a split's stages and of the launches (attention and merge) where the caches are small - 4 sequences
// on 301 slots 10 us - and beyond some 16 rows the conversion of the codes to 16 bits, once a warp: 8 heads, 40,000 slots
// of int8 30 us with 8 rows (2.7 TB/s), 65 with 48. From there on prefix_attn_tc.cu, which converts a tile once for 128
// rows, takes the prefix.
#include "common.cuh"
#include "tc.cuh"
#include "kernels.h"

namespace rb {

namespace pfx {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// CTAs of an SM, by registers: codes of 128 columns run two, with stages of 128 slots and steps of 32; everything else
// three, with 64 and 16. (int8, 16 sequences of 4,096 slots: 44 us so, 48 with three CTAs of 64-slot stages; 64 sequences
// of 700: 20 against 26.)
constexpr bool wide_steps(int fmt, int hd) { return fmt != RB_KV_PLAIN && hd == 128; }
constexpr int ctas_per_sm(int fmt, int hd) { return wide_steps(fmt, hd) ? 2 : 3; }
constexpr float kLog2e = 1.4426950408889634f;
// A row's factor from scores to log2 units, within the normal numbers: a masked slot's -inf stays -inf, a score of zero zero.
__device__ __forceinline__ float factor_in_range(float f) { return fminf(fmaxf(f, 1.17549435e-38f), 3.402823466e38f); }
// t + e of a row's slots stays below R + kRoom + kSlack, so that 2^(t - R) s < 2^15 and fits fp16; the largest is at least
// 2^kRoom, which keeps factors down to 2^-20 of it normal numbers.
constexpr float kRoom = 6.f, kSlack = 8.f;
constexpr int kLeastE = -80;      // of e: 2^(t - R) is at most 2^94, and sums of 2^27 of them are finite
constexpr int kBelowM = 60;       // e is at least the exponent of a 4-bit row's m less this: 2^(t - R) m is finite, too

struct Side {
  const uint8_t* k;
  const uint8_t* v;
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
  int n_seqs, n_q, n_kv, rep, bf16;
  float scale;
  int wm, tiles_m;   // warps along the rows of a tile, row tiles of the prefix's M = n_seqs rep rows
  int max_np;        // most splits of the prefix
  int parts;         // partials a prefix split leaves: 1, or 2 (prefix_attn_tc.cu)
  int max_ns;        // most splits of a sequence's own rows
  float* o;          // partials: prefix items [n_kv][tiles_m][max_np][rows][hd], then own [n_seqs][n_kv][max_ns][rep][hd]
  float2* rl;        // the same without hd: (R, l)
  int64_t own_o, own_rl;  // offsets of the own partials
  int* plan;         // {prefix splits, own splits, tiles of a prefix split, tiles of an own split}
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// v 2^d for d <= 0, also where 2^d is below fp32's range: references lie as far apart as value scales do, and the sums under
// the lower one as far above one.
__device__ __forceinline__ float lowered(float v, float d) {
  const float h = ex2(0.5f * d);
  return v * h * h;
}

// A value row's e, from its scale and (4-bit rows, else 0) the middle of its range. A NaN scale shows by itself.
__device__ __forceinline__ float value_exponent(float s, float m) {
  const int es = static_cast<int>(__float_as_uint(s) >> 23), em = static_cast<int>((__float_as_uint(m) >> 23) & 255u) - kBelowM;
  return s == s ? static_cast<float>(max(max(es, em) - 127, kLeastE)) : static_cast<float>(kLeastE);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;  // 0: the 16 bytes are filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
// Shared-memory loads without a memory clobber: volatile keeps them between the barriers that guard the data, and
// nothing that is held in registers is loaded again after them.
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float2 lds64f(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint4 lds128v(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    mma_f16_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// One format at one head size: the tile's shared-memory layout and the MMA fragments it yields. The order of the
// columns inside a product's k16 step is free as long as both operands share it, and so is the order of the output
// columns: both are chosen so that a lane's codes are contiguous bytes.
template <int kHd_, int kFmt_, bool kBf16_>
struct Fmt {
  static constexpr int kHd = kHd_, kFmt = kFmt_;
  static constexpr bool kBf16 = kBf16_;          // bf16 products: plain bf16 rows only
  static constexpr bool kPlain = kFmt == RB_KV_PLAIN;
  static constexpr int kKs = kHd / 16;           // k16 steps of q . k
  static constexpr int kNv = kHd / 8;            // n8 tiles of p v
  static constexpr int kRow = kPlain ? 2 * kHd : (kFmt == RB_KV_INT8 ? kHd : kHd / 2);  // bytes of a row
  static constexpr int kChunks = kRow / 16;
  static constexpr int kCtas = ctas_per_sm(kFmt, kHd);
  static constexpr int kTile = wide_steps(kFmt, kHd) ? 128 : 64;  // slots of a stage
  static constexpr int kSide = kTile * kRow;       // bytes of a stage's keys (or values)
  static constexpr int kE = kFmt == RB_KV_INT4 ? 4 : 2;  // a stage's parameters in fp32, kTile each: s of keys, of values, (m of keys, of values,) e of values
  static constexpr int kPar = kPlain ? 0 : kTile * 4 * (kE + 1);
  static constexpr int kStage = 2 * kSide + kPar;

  // 16-byte chunk `ch` of row `r` in the key (value) tile; conflict-free for the loads below
  __device__ static uint32_t k_at(int r, int ch) {
    if constexpr (kPlain) return r * kRow + ((ch ^ (r & 7)) << 4);
    if constexpr (kRow == 128) return r * kRow + ((ch ^ ((r & 1) << 2)) << 4);
    return r * kRow + (ch << 4);
  }
  __device__ static uint32_t v_at(int r, int ch) {
    if constexpr (kPlain) return r * kRow + ((ch ^ (r & 7)) << 4);
    const uint32_t byte = r * kRow + (ch << 4);
    const uint32_t x = kRow == 32 ? ((r >> 2) & 1) << 1 : ((r >> 1) & 3) << 1;
    return byte ^ (x << 4);
  }

  // The query columns that lane column c holds at k16 step ks as register pair q (k = 2c, 2c + 1 | 2c + 8, 2c + 9).
  __device__ static uint32_t q_pair(const uint16_t* row, int ks, int c, int q) {
    if constexpr (kPlain) return __ldcg(reinterpret_cast<const unsigned int*>(row + ks * 16 + q * 8 + 2 * c));
    if constexpr (kFmt == RB_KV_INT8)
      return __ldcg(reinterpret_cast<const unsigned int*>(row + (ks >> 2) * 64 + c * 16 + (ks & 3) * 4 + q * 2));
    // a word of eight 4-bit codes: nibbles i and i + 4 are the pair
    const uint16_t* at = row + c * (kHd / 4) + (ks >> 1) * 8 + (ks & 1) * 2 + q;
    return static_cast<uint32_t>(__ldcg(at)) | (static_cast<uint32_t>(__ldcg(at + 4)) << 16);
  }
  // Output column of accumulator tile u, column n
  __device__ static int o_col(int u, int n) { return kPlain ? u * 8 + n : n * kNv + u; }

  // Key fragments of 16 slots from row0 at k16 step ks: b[t] for slots 8 t .. 8 t + 7. `raw` carries a lane's key
  // bytes of the 16 slots (quantised formats), loaded once by k_raw.
  struct KRaw {
    uint32_t w[2][kPlain ? 1 : kRow / 16];
  };
  __device__ static void k_raw(uint32_t tile, int row0, int lane, KRaw& raw) {
    if constexpr (!kPlain) {
      const int g = lane >> 2, c = lane & 3;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = row0 + 8 * t + g;
        if constexpr (kRow == 32) {
          const uint2 v = lds64(tile + k_at(r, c >> 1) + (c & 1) * 8);
          raw.w[t][0] = v.x, raw.w[t][1] = v.y;
        } else {
#pragma unroll
          for (int i = 0; i < kRow / 64; ++i) {
            const uint4 v = lds128v(tile + k_at(r, c + 4 * i));
            raw.w[t][4 * i] = v.x, raw.w[t][4 * i + 1] = v.y, raw.w[t][4 * i + 2] = v.z, raw.w[t][4 * i + 3] = v.w;
          }
        }
      }
    }
  }
  __device__ static void k_frag(uint32_t tile, int row0, int lane, int ks, const KRaw& raw, uint32_t (&b)[2][2]) {
    if constexpr (kPlain) {
      uint32_t r[4];
      const int row = row0 + (lane & 7) + ((lane >> 4) << 3);
      ldsm4(tile + k_at(row, 2 * ks + ((lane >> 3) & 1)), r);
      b[0][0] = r[0], b[0][1] = r[1], b[1][0] = r[2], b[1][1] = r[3];
    } else if constexpr (kFmt == RB_KV_INT8) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t w = raw.w[t][ks];
        b[t][0] = mm4::hsub2_u(__byte_perm(w, 0x64646464u, 0x4140), 0x64806480u);  // 1024 + (c + 128) - 1152
        b[t][1] = mm4::hsub2_u(__byte_perm(w, 0x64646464u, 0x4342), 0x64806480u);
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t w = raw.w[t][ks >> 1] >> (8 * (ks & 1));
        b[t][0] = mm4::hsub2_u((w & 0x000F000Fu) | 0x64006400u, 0x64086408u);  // 1024 + c - 1032
        b[t][1] = mm4::hsub2_u((w & 0x00F000F0u) | 0x54005400u, 0x54805480u);  // 64 + c - 72
      }
    }
  }

  // Value fragments of 16 slots from row0: for every accumulator tile u, f(u, b0, b1).
  template <typename F>
  __device__ static void v_frags(uint32_t tile, int row0, int lane, F f) {
    if constexpr (kPlain) {
      const int row = row0 + (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
      for (int u = 0; u < kNv; u += 2) {
        uint32_t r[4];
        ldsm4t(tile + v_at(row, u + (lane >> 4)), r);
        f(u, r[0], r[1]);
        f(u + 1, r[2], r[3]);
      }
    } else {
      constexpr int kB = kRow / 8;  // bytes of a lane in each of its four rows
      const int g = lane >> 2, c = lane & 3;
      uint32_t w[4][kB / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = row0 + 2 * c + (i & 1) + ((i >> 1) << 3);
        if constexpr (kB == 16) {
          const uint4 v = lds128v(tile + v_at(r, g));
          w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
        } else if constexpr (kB == 8) {
          const uint2 v = lds64(tile + v_at(r, g >> 1) + (g & 1) * 8);
          w[i][0] = v.x, w[i][1] = v.y;
        } else {
          w[i][0] = lds32(tile + v_at(r, g >> 2) + (g & 3) * 4);
        }
      }
      if constexpr (kFmt == RB_KV_INT8) {
#pragma unroll
        for (int x = 0; x < kB / 4; ++x) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // bytes 2 hf, 2 hf + 1 of the word
            const uint32_t lo = __byte_perm(w[0][x], w[1][x], hf ? 0x7362 : 0x5140);  // (r0 b, r1 b, r0 b', r1 b')
            const uint32_t hi = __byte_perm(w[2][x], w[3][x], hf ? 0x7362 : 0x5140);
            f(4 * x + 2 * hf, mm4::hsub2_u(__byte_perm(lo, 0x64646464u, 0x4140), 0x64806480u),
              mm4::hsub2_u(__byte_perm(hi, 0x64646464u, 0x4140), 0x64806480u));
            f(4 * x + 2 * hf + 1, mm4::hsub2_u(__byte_perm(lo, 0x64646464u, 0x4342), 0x64806480u),
              mm4::hsub2_u(__byte_perm(hi, 0x64646464u, 0x4342), 0x64806480u));
          }
        }
      } else {
#pragma unroll
        for (int x = 0; x < kB / 4; ++x) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // halves of the word: nibbles 4 hf .. 4 hf + 3
            uint32_t lo = __byte_perm(w[0][x], w[1][x], hf ? 0x7632 : 0x5410);
            uint32_t hi = __byte_perm(w[2][x], w[3][x], hf ? 0x7632 : 0x5410);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              f(8 * x + 4 * hf + 2 * q, mm4::hsub2_u((lo & 0x000F000Fu) | 0x64006400u, 0x64086408u),
                mm4::hsub2_u((hi & 0x000F000Fu) | 0x64006400u, 0x64086408u));
              f(8 * x + 4 * hf + 2 * q + 1, mm4::hsub2_u((lo & 0x00F000F0u) | 0x54005400u, 0x54805480u),
                mm4::hsub2_u((hi & 0x00F000F0u) | 0x54005400u, 0x54805480u));
              lo >>= 8, hi >>= 8;
            }
          }
        }
      }
    }
  }
};

// Tiles of a split in the tcgen05 kernel: at least two, one for each of its groups.
__device__ __forceinline__ int tiles_of_split(int tiles, int max_np) { return max(2, (tiles + max_np - 1) / max_np); }

// What one item reads and where its partial goes.
struct Item {
  const uint8_t* k;  // the head's first row
  const uint8_t* v;
  const void* k_par;
  const void* v_par;
  int64_t par0;      // index of the first row's parameters
  int64_t n;         // visible slots
  int t0, t1;        // stages [t0, t1)
  int seq, row0, rows;  // seq < 0: rows row0 .. row0 + rows - 1 of the batch's; else sequence seq's rep rows
  int kv;
  float* o;
  float2* rl;
};

// A CTA's four warps: each takes 16 query rows; wm of them stand along the rows (1, 2 or 4), the other 4 / wm along the
// slots of a stage. Two or three CTAs an SM: one's loads and barriers hide behind the others' products.
template <typename F>
struct Tile {
  static constexpr int kBlock = wide_steps(F::kFmt, F::kHd) ? 32 : 16;  // slots of one softmax step
  static constexpr int kNt = kBlock / 8;
  static_assert(F::kTile / kWarps % kBlock == 0, "a warp's slots of a stage are whole steps");
  static constexpr int kMergeRow = (F::kNv * 33) * 16;        // a warp's 16-row accumulator tile, padded
  static constexpr int kFit = (227 * 1024 / F::kCtas - 2048) / F::kStage;  // of a CTA's share of the shared memory
  static constexpr int kStages = kFit < 2 ? 2 : (kFit > 5 ? 5 : kFit);
  static constexpr int kRing = kStages * F::kStage;
  static constexpr int kMerge = kWarps * kMergeRow;
  static constexpr int kOffRl = kRing > kMerge ? kRing : kMerge;  // the merge reuses the ring; (R, l) [4][16]
  static constexpr int kSmem = kOffRl + kWarps * 16 * 8;
};

template <typename F>
__device__ __forceinline__ void run_item(const Params& p, const Item it, const int wm_n, uint8_t* smem) {
  using T = Tile<F>;
  constexpr int kHd = F::kHd;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int wm = warp & (wm_n - 1), wk = warp / wm_n, per_warp = F::kTile * wm_n / kWarps;
  const uint32_t s0 = smem_u32(smem);
  float2* rl = reinterpret_cast<float2*>(smem + T::kOffRl);

  uint32_t ld_slot = 0, rd_slot = 0;  // byte offsets of the stage to fill and of the stage to read in the ring
  auto load_rows = [&](int t) {       // stage t's keys and values
    const uint32_t dst = s0 + ld_slot;
    const int64_t left = it.n - static_cast<int64_t>(t) * F::kTile;
    const uint8_t* k = it.k + static_cast<int64_t>(t) * F::kSide + tid * 16;
    const uint8_t* v = it.v + static_cast<int64_t>(t) * F::kSide + tid * 16;
    // a stage's rows are contiguous; kThreads chunks on, the swizzle of a chunk is the same
    static_assert(kThreads / F::kChunks % 8 == 0, "the swizzle repeats every eight rows");
    const uint32_t kd = dst + F::k_at(tid / F::kChunks, tid % F::kChunks), vd = dst + F::kSide + F::v_at(tid / F::kChunks, tid % F::kChunks);
    if (left >= F::kTile) {
#pragma unroll
      for (int i = 0; i < F::kSide / 16 / kThreads; ++i) {
        cp_async16(kd + i * kThreads * 16, k + i * kThreads * 16, true);
        cp_async16(vd + i * kThreads * 16, v + i * kThreads * 16, true);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < F::kSide / 16 / kThreads; ++i) {
        const bool on = (i * kThreads + tid) / F::kChunks < left;
        cp_async16(kd + i * kThreads * 16, on ? k + i * kThreads * 16 : it.k, on);
        cp_async16(vd + i * kThreads * 16, on ? v + i * kThreads * 16 : it.v, on);
      }
    }
  };
  // A stage's row parameters: loaded into registers ahead, stored as fp32 behind its rows (2-byte scales of an odd
  // cache length have no alignment that an asynchronous copy takes).
  constexpr int kWords = 2 * F::kTile / kThreads;  // a thread's: the keys' parameters first, then the values'
  uint32_t par[kWords];
  auto load_par = [&](int t) {
    if constexpr (!F::kPlain) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const int x = i * kThreads + tid;
        const int64_t r = static_cast<int64_t>(t) * F::kTile + (x & (F::kTile - 1));
        const void* src = x < F::kTile ? it.k_par : it.v_par;
        par[i] = 0u;
        if (r < it.n) par[i] = F::kFmt == RB_KV_INT8 ? static_cast<uint32_t>(__ldcg(reinterpret_cast<const unsigned short*>(src) + it.par0 + r))
                                                     : __ldcg(reinterpret_cast<const unsigned int*>(src) + it.par0 + r);
      }
    }
  };
  auto store_par = [&]() {  // behind the rows of the stage last loaded
    if constexpr (!F::kPlain) {
      float* dst = reinterpret_cast<float*>(smem + ld_slot + 2 * F::kSide);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const int x = i * kThreads + tid;
        const float sc = __uint_as_float(par[i] << 16);
        dst[x] = sc;
        float mid = 0.f;
        if constexpr (F::kFmt == RB_KV_INT4) {  // codes enter as c - 8: m + 8 s stands for the middle of the row's range
          mid = fmaf(8.f, sc, p.bf16 ? __uint_as_float(par[i] & 0xffff0000u) : __half2float(__ushort_as_half(static_cast<unsigned short>(par[i] >> 16))));
          dst[2 * F::kTile + x] = mid;
        }
        if (x >= F::kTile) dst[(F::kE - 1) * F::kTile + x] = value_exponent(sc, mid);
      }
    }
  };
  auto next = [](uint32_t slot) { return slot + F::kStage == T::kRing ? 0u : slot + F::kStage; };

  __syncthreads();  // the previous item's merge has been read
  load_rows(it.t0);
  cp_commit();
  load_par(it.t0);

  // ---- the warp's queries (rows g, g + 8 of its 16) as A fragments, straight from global memory ----
  uint32_t qa[F::kKs][4];
  float fr[2], qs[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = wm * 16 + x * 8 + g;
    const bool on = r < it.rows;
    const int row = it.row0 + r;
    const int b = it.seq >= 0 ? it.seq : (on ? row / p.rep : 0), j = it.seq >= 0 ? r : row % p.rep;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + b * p.ldq + static_cast<int64_t>(it.kv * p.rep + (on ? j : 0)) * kHd;
#pragma unroll
    for (int ks = 0; ks < F::kKs; ++ks)
#pragma unroll
      for (int q = 0; q < 2; ++q) qa[ks][2 * q + x] = on ? F::q_pair(src, ks, c, q) : 0u;
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    float f = fabsf(p.scale) * kLog2e;
    float sum = 0.f;
    if (!F::kPlain && p.bf16) {
      // fp16 queries for the codes' product: scaled by a power of two so that the row's largest is in [1, 2) - exact
      // but for elements 2^-24 below it
      uint32_t top = 0u;
#pragma unroll
      for (int ks = 0; ks < F::kKs; ++ks)
#pragma unroll
        for (int q = 0; q < 2; ++q) top = __vmaxu2(top, qa[ks][2 * q + x] & 0x7fff7fffu);
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t t16 = max(top & 0xffffu, top >> 16);
      const uint32_t ex = t16 >> 7;  // the exponent of a bf16
      const uint32_t exc = ex < 30u ? 30u : (ex > 220u ? 220u : ex);
      const float down = __uint_as_float((254u - exc) << 23);
      f *= __uint_as_float(exc << 23);
#pragma unroll
      for (int ks = 0; ks < F::kKs; ++ks)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t u = qa[ks][2 * q + x];
          qa[ks][2 * q + x] = pack2<false>(__uint_as_float(u << 16) * down, __uint_as_float(u & 0xffff0000u) * down);
        }
    }
    if (flip) {
#pragma unroll
      for (int ks = 0; ks < F::kKs; ++ks) qa[ks][x] ^= flip, qa[ks][2 + x] ^= flip;
    }
    if constexpr (F::kFmt == RB_KV_INT4) {
#pragma unroll
      for (int ks = 0; ks < F::kKs; ++ks)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&qa[ks][2 * q + x]));
          sum += v.x + v.y;
        }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    }
    fr[x] = factor_in_range(f);
    qs[x] = sum;
  }
  store_par();
  ld_slot = next(ld_slot);
#pragma unroll 1
  for (int i = 1; i < T::kStages - 1; ++i) {
    if (it.t0 + i < it.t1) {
      load_rows(it.t0 + i);
      load_par(it.t0 + i);
      store_par();
      ld_slot = next(ld_slot);
    }
    cp_commit();
  }

  float o[F::kNv][4], l[2], w[2], ref[2];
#pragma unroll
  for (int u = 0; u < F::kNv; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[u][e] = 0.f;
#pragma unroll
  for (int x = 0; x < 2; ++x) l[x] = w[x] = 0.f, ref[x] = -INFINITY;

#pragma unroll 1
  for (int t = it.t0; t < it.t1; ++t) {
    cp_wait<T::kStages - 2>();
    __syncthreads();  // stage t is there for everybody, stage t - 1 is free
    const bool more = t + T::kStages - 1 < it.t1;
    if (more) {
      load_rows(t + T::kStages - 1);
      load_par(t + T::kStages - 1);
    }
    cp_commit();
    const uint32_t kt = s0 + rd_slot, vt = kt + F::kSide, pt = vt + F::kSide;
    rd_slot = next(rd_slot);
    const int64_t left64 = it.n - static_cast<int64_t>(t) * F::kTile;
    const int left = left64 < F::kTile ? static_cast<int>(left64) : F::kTile;
    const int b1 = min((wk + 1) * per_warp, left);
#pragma unroll 1
    for (int b0 = wk * per_warp; b0 < b1; b0 += T::kBlock) {
      float s[T::kNt][4];
#pragma unroll
      for (int n = 0; n < T::kNt; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
      // ---- scores ----
      typename F::KRaw raw[T::kNt / 2];
#pragma unroll
      for (int n = 0; n < T::kNt / 2; ++n) F::k_raw(kt, b0 + 16 * n, lane, raw[n]);
#pragma unroll
      for (int ks = 0; ks < F::kKs; ++ks)
#pragma unroll
        for (int n = 0; n < T::kNt / 2; ++n) {
          uint32_t b[2][2];
          F::k_frag(kt, b0 + 16 * n, lane, ks, raw[n], b);
          mma16816<F::kBf16>(s[2 * n], qa[ks], b[0][0], b[0][1]);
          mma16816<F::kBf16>(s[2 * n + 1], qa[ks], b[1][0], b[1][1]);
        }
      // ---- scales, mask, largest ----
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < T::kNt; ++n) {
        if constexpr (!F::kPlain) {
          const int col = b0 + 8 * n + 2 * c;
          const float2 ks = lds64f(pt + col * 4);
          float2 km = make_float2(0.f, 0.f);
          if constexpr (F::kFmt == RB_KV_INT4) km = lds64f(pt + (2 * F::kTile + col) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float sc = (e & 1) ? ks.y : ks.x;
            if constexpr (F::kFmt == RB_KV_INT4)
              s[n][e] = fmaf(s[n][e], sc, ((e & 1) ? km.y : km.x) * qs[e >> 1]);
            else
              s[n][e] *= sc;
          }
        }
      }
      if (b0 + T::kBlock > left) {
#pragma unroll
        for (int n = 0; n < T::kNt; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (b0 + 8 * n + 2 * c + (e & 1) >= left) s[n][e] = -INFINITY;
      }
#pragma unroll
      for (int n = 0; n < T::kNt; ++n) {
        float2 ev = make_float2(0.f, 0.f);
        if constexpr (!F::kPlain) ev = lds64f(pt + (F::kE * F::kTile + b0 + 8 * n + 2 * c) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], F::kPlain ? s[n][e] : fmaf(s[n][e], fr[e >> 1], (e & 1) ? ev.y : ev.x));
      }
      if constexpr (F::kPlain) top[0] *= fr[0], top[1] *= fr[1];
      if (__any_sync(0xffffffffu, top[0] > ref[0] + (kRoom + kSlack) || top[1] > ref[1] + (kRoom + kSlack))) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float v = top[x];
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
          const float nr = fmaxf(ref[x], v - kRoom);
          const float d = ref[x] == -INFINITY ? -INFINITY : ref[x] - nr, f = ex2(d);
          ref[x] = nr;
          l[x] = lowered(l[x], d);
          if constexpr (F::kFmt == RB_KV_INT4) w[x] = lowered(w[x], d);
#pragma unroll
          for (int u = 0; u < F::kNv; ++u) o[u][2 * x] *= f, o[u][2 * x + 1] *= f;
        }
      }
      // ---- probabilities ----
      float base[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) base[x] = ref[x] == -INFINITY ? 0.f : -ref[x];
#pragma unroll
      for (int n = 0; n < T::kNt; ++n) {
        const int col = b0 + 8 * n + 2 * c;
        float2 vs = make_float2(1.f, 1.f), vm = make_float2(0.f, 0.f);
        if constexpr (!F::kPlain) vs = lds64f(pt + (F::kTile + col) * 4);
        if constexpr (F::kFmt == RB_KV_INT4) vm = lds64f(pt + (3 * F::kTile + col) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float pr = ex2(fmaf(s[n][e], fr[e >> 1], base[e >> 1]));
          l[e >> 1] += pr;
          if constexpr (F::kFmt == RB_KV_INT4) w[e >> 1] = fmaf(pr, (e & 1) ? vm.y : vm.x, w[e >> 1]);
          if constexpr (!F::kPlain) pr *= (e & 1) ? vs.y : vs.x;
          s[n][e] = pr;
        }
      }
      // ---- O += p v ----
#pragma unroll
      for (int n = 0; n < T::kNt / 2; ++n) {
        uint32_t a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = pack2<F::kBf16>(s[2 * n + (e >> 1)][2 * (e & 1)], s[2 * n + (e >> 1)][2 * (e & 1) + 1]);
        // 4-bit rows: a value's part s (c - 8) may be far larger than the value, so the rounding of p s to fp16 is
        // made up for by a second term
        uint32_t a2[4] = {0u, 0u, 0u, 0u};
        if constexpr (F::kFmt == RB_KV_INT4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&a[e]));
            a2[e] = pack2<false>(s[2 * n + (e >> 1)][2 * (e & 1)] - hi.x, s[2 * n + (e >> 1)][2 * (e & 1) + 1] - hi.y);
          }
        }
        F::v_frags(vt, b0 + 16 * n, lane, [&](int u, uint32_t f0, uint32_t f1) {
          mma16816<F::kBf16>(o[u], a, f0, f1);
          if constexpr (F::kFmt == RB_KV_INT4) mma16816<false>(o[u], a2, f0, f1);
        });
      }
    }
    if (more) {
      store_par();
      ld_slot = next(ld_slot);
    }
  }
  cp_wait<0>();

  // ---- join the warps along the slots, in their order, and leave the item's partial ----
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    if constexpr (F::kFmt == RB_KV_INT4) {
      w[x] += __shfl_xor_sync(0xffffffffu, w[x], 1);
      w[x] += __shfl_xor_sync(0xffffffffu, w[x], 2);
    }
    if (c == 0)
      rl[warp * 16 + x * 8 + g] =
          make_float2(ref[x] == -INFINITY && l[x] == 0.f ? -INFINITY : (ref[x] == -INFINITY ? 0.f : ref[x]), l[x]);
  }
  __syncthreads();
  {
    float f[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float hi = -INFINITY;
      for (int k = wm; k < kWarps; k += wm_n) hi = fmaxf(hi, rl[k * 16 + x * 8 + g].x);
      const float mine = rl[warp * 16 + x * 8 + g].x;
      // 4-bit rows: half of the way, to be taken twice, as in lowered(); without p m in them, the sums of a warp whose factor
      // is below fp32's range are nothing beside the others'
      f[x] = mine == -INFINITY ? 0.f : ex2((F::kFmt == RB_KV_INT4 ? 0.5f : 1.f) * (mine - hi));
    }
    uint8_t* dst = smem + warp * T::kMergeRow;
#pragma unroll
    for (int u = 0; u < F::kNv; ++u)
      *reinterpret_cast<float4*>(dst + (u * 33 + lane) * 16) =
          F::kFmt == RB_KV_INT4 ? make_float4((o[u][0] + w[0]) * f[0] * f[0], (o[u][1] + w[0]) * f[0] * f[0], (o[u][2] + w[1]) * f[1] * f[1], (o[u][3] + w[1]) * f[1] * f[1])
                                : make_float4(o[u][0] * f[0], o[u][1] * f[0], o[u][2] * f[1], o[u][3] * f[1]);
  }
  __syncthreads();
#pragma unroll 2
  for (int x = tid; x < it.rows * (kHd / 2); x += kThreads) {
    const int r = x / (kHd / 2), d2 = x % (kHd / 2);
    // columns o_col(u, n), o_col(u, n + 1) of the fragments: a pair in the plain order, strided in the codes' order
    float2 acc = make_float2(0.f, 0.f);
    const int u = F::kPlain ? d2 >> 2 : d2 % F::kNv, n = F::kPlain ? (d2 & 3) * 2 : (d2 / F::kNv) * 2;
    const uint8_t* src = smem + (r >> 4) * T::kMergeRow + (u * 33 + (r & 7) * 4 + n / 2) * 16 + ((r >> 3) & 1) * 8;
    for (int k = 0; k < kWarps; k += wm_n) {
      const float2 v = *reinterpret_cast<const float2*>(src + k * T::kMergeRow);
      acc.x += v.x, acc.y += v.y;
    }
    float* dst = it.o + static_cast<int64_t>(r) * kHd;
    if constexpr (F::kPlain) {
      *reinterpret_cast<float2*>(dst + F::o_col(u, n)) = acc;
    } else {
      dst[F::o_col(u, n)] = acc.x;
      dst[F::o_col(u, n + 1)] = acc.y;
    }
  }
  for (int r = tid; r < it.rows; r += kThreads) {
    float hi = -INFINITY, sum = 0.f;
    for (int k = r >> 4; k < kWarps; k += wm_n) hi = fmaxf(hi, rl[k * 16 + (r & 15)].x);
    for (int k = r >> 4; k < kWarps; k += wm_n) {
      const float2 v = rl[k * 16 + (r & 15)];
      sum += v.x == -INFINITY ? 0.f : lowered(v.y, v.x - hi);
    }
    it.rl[r] = make_float2(hi, sum);
  }
}

// How the lengths on the device are dealt to the grid. Every CTA computes the same plan.
struct Plan {
  int np, ns, pt, ot;    // splits of the prefix and of own rows, stages a split
  int prefix_items, own_items;
  bool prefix_ok;
};

template <int kTile>
__device__ __forceinline__ Plan make_plan(const Params& p, int grid) {
  // every warp by itself: no barrier, and the loads of all lengths go out together. The launch before may have written the
  // lengths while this one was resident: loads that stay behind the wait (__ldg's may not), as everywhere below
  const int lane = threadIdx.x & 31;
  const int64_t np_raw = p.pre.k ? __ldcg(p.pre.len) : 0;
  int sum = 0, most = 0;
  if (p.own.k) {
#pragma unroll 2
    for (int b = lane; b < p.n_seqs; b += 32) {
      const int64_t n = __ldcg(p.own.len + b);
      if (n <= 0 || n > p.own.cache_len) continue;
      const int t = static_cast<int>((n + kTile - 1) / kTile);
      sum += min(t + 2, 1 << 20);  // an item's start and end cost about two stages
      most = max(most, t);
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    most = __reduce_max_sync(0xffffffffu, most);
  }
  Plan pl;
  pl.prefix_ok = np_raw >= 0 && np_raw <= p.pre.cache_len;
  const int64_t n = pl.prefix_ok ? np_raw : 0;
  const int tiles = static_cast<int>((n + kTile - 1) / kTile), lanes = p.n_kv * p.tiles_m;
  const float own = static_cast<float>(sum) * static_cast<float>(p.n_kv), pre = static_cast<float>(tiles) * static_cast<float>(lanes);
  pl.ns = most ? min(p.max_ns, (most + 3) / 4) : 0;  // at least four stages a split
  pl.ot = pl.ns ? (most + pl.ns - 1) / pl.ns : 0;
  pl.ns = pl.ot ? (most + pl.ot - 1) / pl.ot : 0;
  pl.own_items = p.n_seqs * p.n_kv * pl.ns;
  // the own items' share of the CTAs, at most one each; the rest for the prefix
  int g_own = sum > 0 ? static_cast<int>(__fdividef(own, own + pre) * static_cast<float>(grid) + 0.5f) : 0;
  g_own = min(max(g_own, sum > 0 ? 1 : 0), pl.own_items);
  if (tiles > 0 && g_own >= grid) g_own = grid - 1;
  pl.np = tiles ? max(1, min(min((grid - g_own) / lanes, tiles), p.max_np)) : 0;
  pl.pt = pl.np ? (tiles + pl.np - 1) / pl.np : 0;
  pl.np = pl.pt ? (tiles + pl.pt - 1) / pl.pt : 0;
  pl.prefix_items = lanes * pl.np;
  return pl;
}

template <typename F>
__global__ void __launch_bounds__(kThreads, F::kCtas) prefix_attn_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  // Behind the tcgen05 kernel (parts == 2) the own rows need not wait for it: it let this launch start only after its own
  // wait, so what comes before both is complete. They start on the SMs that it leaves, and wait for it at their end, so
  // that the merge, which waits for this launch, finds both kernels' partials.
  const bool beside = p.parts == 2;
  if (!beside) griddep_wait();
  griddep_launch_dependents();
  const int grid = gridDim.x, cta = blockIdx.x;
  const Plan pl = make_plan<F::kTile>(p, grid);
  if (cta == 0 && threadIdx.x == 0) {
    p.plan[0] = pl.np, p.plan[1] = pl.ns, p.plan[2] = pl.pt, p.plan[3] = pl.ot;
    if (!pl.prefix_ok) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
  }
  if (!pl.prefix_ok) return;
  // with fewer prefix items than CTAs, those beyond take the own items among themselves
  const bool apart = pl.prefix_items < grid;
  int i = cta, step = grid;
  if (apart && cta >= pl.prefix_items) step = grid - pl.prefix_items;
  const int end = apart && cta < pl.prefix_items ? pl.prefix_items : pl.prefix_items + pl.own_items;
#pragma unroll 1
  for (; i < end; i += step) {
    Item it;
    int wm = 1;
    const bool pre = i < pl.prefix_items;
    const Side& S = pre ? p.pre : p.own;
    int64_t head;
    if (pre) {
      const int lane_i = i / pl.np, sp = i % pl.np;
      it.kv = lane_i / p.tiles_m;
      const int rt = lane_i % p.tiles_m;
      head = it.kv;
      it.n = __ldcg(S.len);
      it.t0 = sp * pl.pt;
      it.t1 = it.t0 + pl.pt;
      it.seq = -1;
      wm = p.wm;
      const int tile = 16 * wm;
      it.row0 = rt * tile;
      it.rows = min(tile, p.n_seqs * p.rep - it.row0);
      const int64_t slot = (static_cast<int64_t>(lane_i) * p.max_np + sp) * tile;
      it.o = p.o + slot * F::kHd;
      it.rl = p.rl + slot;
    } else {
      const int x = i - pl.prefix_items, sp = x % pl.ns;
      it.kv = (x / pl.ns) % p.n_kv;
      it.seq = x / pl.ns / p.n_kv;
      it.n = __ldcg(S.len + it.seq);
      if (it.n < 0 || it.n > S.cache_len) {
        if (threadIdx.x == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
        continue;
      }
      it.t0 = sp * pl.ot;
      it.t1 = it.t0 + pl.ot;
      head = static_cast<int64_t>(it.seq) * p.n_kv + it.kv;
      it.row0 = 0;
      it.rows = p.rep;
      const int64_t slot = (head * p.max_ns + sp) * p.rep;
      it.o = p.o + p.own_o + slot * F::kHd;
      it.rl = p.rl + p.own_rl + slot;
    }
    it.t1 = min(static_cast<int>((it.n + F::kTile - 1) / F::kTile), it.t1);
    if (it.t0 >= it.t1) continue;
    it.par0 = head * S.cache_len;
    it.k = S.k + it.par0 * F::kRow;
    it.v = S.v + it.par0 * F::kRow;
    it.k_par = S.k_par;
    it.v_par = S.v_par;
    run_item<F>(p, it, wm, smem);
  }
  if (beside) griddep_wait();
  // an own length outside its cache with no item of its own (no split at all) is reported here
  if (cta == 0 && pl.ns == 0 && p.own.k)
    for (int b = threadIdx.x; b < p.n_seqs; b += kThreads)
      if (const int64_t n = __ldcg(p.own.len + b); n < 0 || n > p.own.cache_len) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
}

// A CTA joins the partials of one (sequence, query head): prefix splits, then own splits. Warp w takes every fourth
// one, eight loads at a time, under a reference of its own (one for all would be another round trip to L2 before the
// loads); the warps' sums are joined in warp order. Latency-bound: the launch and two dependent loads.
template <int kHd>
__global__ void __launch_bounds__(kThreads) prefix_attn_merge(const __grid_constant__ Params p, int tile_rows, int stage) {
  constexpr int kE = kHd / 32;
  __shared__ float so[kWarps][kHd], sl[kWarps], sr[kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / p.n_q, h = blockIdx.x % p.n_q, kv = h / p.rep, j = h % p.rep;
  const int64_t n_pre = p.pre.len ? __ldcg(p.pre.len) : 0, n_own = p.own.len ? __ldcg(p.own.len + b) : 0;
  // prefix_attn_kernel leaves the plan, and runs where there are rows for it: a cache without slots has no kernel
  const bool planned = p.own.k || (p.pre.k && p.parts == 1);
  const int ot = planned ? __ldcg(p.plan + 3) : 0;
  int np = planned ? __ldcg(p.plan) : 0;
  if (n_pre < 0 || n_pre > p.pre.cache_len || n_own < 0 || n_own > p.own.cache_len) {
    if (threadIdx.x == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
    return;
  }
  if (p.parts == 2) {  // the tcgen05 kernel's splits: the tiles dealt evenly, two partials each
    const int tiles = static_cast<int>((n_pre + 127) / 128), per = tiles_of_split(tiles, p.max_np);
    np = 2 * ((tiles + per - 1) / per);
  }
  const int ns = n_own ? static_cast<int>(((n_own + stage - 1) / stage + ot - 1) / ot) : 0;
  const int r = b * p.rep + j, rt = r / tile_rows;
  // partial i: row x0 + i xs of the prefix's, then own row y0 + (i - np) rep
  const int64_t x0 = (static_cast<int64_t>(kv) * p.tiles_m + rt) * p.max_np * p.parts * tile_rows + r % tile_rows;
  const int64_t y0 = p.own_rl + (static_cast<int64_t>(b) * p.n_kv + kv) * p.max_ns * p.rep + j;
  auto at = [&](int i) { return i < np ? x0 + static_cast<int64_t>(i) * tile_rows : y0 + static_cast<int64_t>(i - np) * p.rep; };
  const int n = np + ns;
  float acc[kE], l = 0.f, hi = -INFINITY;
#pragma unroll
  for (int e = 0; e < kE; ++e) acc[e] = 0.f;
  for (int i0 = warp; i0 < n; i0 += 8 * kWarps) {
    float2 v[8];
    float x[8][kE];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = i0 + k * kWarps;
      v[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int e = 0; e < kE; ++e) x[k][e] = 0.f;
      if (i < n) {
        const int64_t a = at(i);
        v[k] = __ldcg(p.rl + a);
        if constexpr (kE == 4) {
          const float4 y = __ldcg(reinterpret_cast<const float4*>(p.o + a * kHd) + lane);
          x[k][0] = y.x, x[k][1] = y.y, x[k][2] = y.z, x[k][3] = y.w;
        } else {
          const float2 y = __ldcg(reinterpret_cast<const float2*>(p.o + a * kHd) + lane);
          x[k][0] = y.x, x[k][1] = y.y;
        }
      }
    }
    float top = hi;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, v[k].x);
    if (hi != -INFINITY) {  // not the first eight: l and acc hold something
      l = lowered(l, hi - top);
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[e] = lowered(acc[e], hi - top);
    }
    hi = top;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (v[k].x == -INFINITY) continue;  // nothing there: its sums may not have been written
      const float h = ex2(0.5f * (v[k].x - hi));
      l = fmaf(v[k].y * h, h, l);
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[e] = fmaf(x[k][e] * h, h, acc[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) so[warp][lane * kE + e] = acc[e];
  if (lane == 0) sl[warp] = l, sr[warp] = hi;
  __syncthreads();
  if (threadIdx.x < kHd / 2) {
    const int d = 2 * threadIdx.x;
    float x = 0.f, y = 0.f, lt = 0.f;
    const float top = fmaxf(fmaxf(sr[0], sr[1]), fmaxf(sr[2], sr[3]));
    static_assert(kWarps == 4, "the warps' references");
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const float h = sr[k] == -INFINITY ? 0.f : ex2(0.5f * (sr[k] - top));
      x = fmaf(so[k][d] * h, h, x), y = fmaf(so[k][d + 1] * h, h, y), lt = fmaf(sl[k] * h, h, lt);
    }
    const bool none = n_pre + n_own == 0;
    x = none ? 0.f : x / lt;
    y = none ? 0.f : y / lt;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + b * p.ldo + static_cast<int64_t>(h) * kHd + d;
    *reinterpret_cast<uint32_t*>(dst) = p.bf16 ? pack2<true>(x, y) : pack2<false>(x, y);
  }
}

}  // namespace pfx

}  // namespace rb
