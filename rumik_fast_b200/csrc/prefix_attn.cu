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
// O = sum 2^(t - R) v in fp32 (t: the score times log2 e). R is only raised when a score exceeds it by more than 2^8,
// so the accumulators are rarely rescaled; any R gives the same O / l.
//
// Work is cut along the slots so that every SM streams a share of the caches: CTAs take (key-value head, 16 kMt kWm
// rows, split of the prefix) or (sequence, key-value head, split of its own rows) items and leave an fp32 partial
// (R, l, O) each, which prefix_attn_merge joins in split order (deterministic).
#include "common.cuh"
#include "tc.cuh"
#include "kernels.h"

namespace rb {

namespace pfx {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxSeqs = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;     // a row's reference is raised when a score exceeds it by this (log2)
constexpr float kLowestE = -90.f; // exponent range of the value scales folded into the reference
constexpr float kHighestE = 90.f;

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
  int tiles_m;       // row tiles of the prefix's M = n_seqs rep rows
  int max_np;        // most splits of the prefix
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;  // 0: the 16 bytes are filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
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
  static constexpr int kTile = kPlain ? 64 : 128;  // slots of a stage
  static constexpr int kSide = kTile * kRow;       // bytes of a stage's keys (or values)
  static constexpr int kPar = kPlain ? 0 : kTile * 4 * (kFmt == RB_KV_INT4 ? 4 : 2);  // fp32 s (and m) of keys, values
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

  // Column of q . k held by lane column c at k16 step ks, register pair p (k = 2c, 2c+1 | 2c+8, 2c+9), element e;
  // inverse: where column d goes.
  __device__ static void q_place(int d, int& ks, int& c, int& p, int& e) {
    if constexpr (kPlain) {
      ks = d >> 4, p = (d >> 3) & 1, c = (d >> 1) & 3, e = d & 1;
    } else if constexpr (kFmt == RB_KV_INT8) {
      ks = ((d >> 6) << 2) | ((d >> 2) & 3), c = (d >> 4) & 3, p = (d >> 1) & 1, e = d & 1;
    } else {
      const int per = kHd / 4;  // columns of a lane: kHd / 32 words of eight
      c = d / per, e = (d >> 2) & 1, p = d & 1;
      ks = (((d % per) >> 3) << 1) | ((d >> 1) & 1);
    }
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
            const uint4 v = lds128_a(tile + k_at(r, c + 4 * i));
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
          const uint4 v = lds128_a(tile + v_at(r, g));
          w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
        } else if constexpr (kB == 8) {
          const uint2 v = lds64(tile + v_at(r, g >> 1) + (g & 1) * 8);
          w[i][0] = v.x, w[i][1] = v.y;
        } else {
          w[i][0] = lds32_a(tile + v_at(r, g >> 2) + (g & 3) * 4);
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

// kMt 16-row tiles a warp, kWm warps along the rows, kWk = 4 / kWm along the slots of a stage.
template <typename F, int kMt, int kWm>
struct Tile {
  static constexpr int kWk = kWarps / kWm;
  static constexpr int kRows = 16 * kMt * kWm;
  static constexpr int kPerWarp = F::kTile / kWk;             // slots of a warp in a stage
  static constexpr int kBlock = kPerWarp < 32 ? kPerWarp : 32;  // slots of one softmax step
  static constexpr int kNt = kBlock / 8;
  static constexpr int kQ = kRows * F::kHd * 2;
  static constexpr int kMergeRow = (F::kNv * 33) * 16;        // a warp's 16-row accumulator tile, padded
  static constexpr int kMerge = kWarps * kMt * kMergeRow;
  static constexpr int kStages = (kQ + 3 * F::kStage > 108 * 1024) ? 2 : 3;
  static constexpr int kRing = kStages * F::kStage;
  static constexpr int kOffQ = kRing > kMerge ? kRing : kMerge;  // the merge reuses the ring
  static constexpr int kOffRow = kOffQ + kQ;                  // rowf, qsum [kRows], then (R, l) [kWk][kRows]
  static constexpr int kSmem = kOffRow + kRows * 8 + kWk * kRows * 8;
};

template <typename F, int kMt, int kWm>
__device__ __noinline__ void run_item(const Params& p, const Item& it, uint8_t* smem) {
  using T = Tile<F, kMt, kWm>;
  constexpr int kHd = F::kHd;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int wm = warp % kWm, wk = warp / kWm;
  const uint32_t s0 = smem_u32(smem);
  float* rowf = reinterpret_cast<float*>(smem + T::kOffRow);
  float* qsum = rowf + T::kRows;
  float2* rl = reinterpret_cast<float2*>(qsum + T::kRows);

  auto stage = [&](int i) { return s0 + (i % T::kStages) * F::kStage; };
  auto load_rows = [&](int t) {  // stage t's keys and values
    const uint32_t dst = stage(t - it.t0);
    const int64_t first = static_cast<int64_t>(t) * F::kTile;
#pragma unroll
    for (int i = 0; i < F::kTile * F::kChunks / kThreads; ++i) {
      const int x = i * kThreads + tid, r = x / F::kChunks, ch = x % F::kChunks;
      const bool on = first + r < it.n;
      const int64_t off = on ? (first + r) * F::kRow + ch * 16 : 0;
      cp_async16(dst + F::k_at(r, ch), it.k + off, on);
      cp_async16(dst + F::kSide + F::v_at(r, ch), it.v + off, on);
    }
  };
  // A stage's row parameters: loaded into registers ahead, stored as fp32 behind its rows (2-byte scales of an odd
  // cache length have no alignment that an asynchronous copy takes).
  uint32_t par[2] = {0u, 0u};
  auto load_par = [&](int t) {
    if constexpr (!F::kPlain) {
      const int64_t r = static_cast<int64_t>(t) * F::kTile + tid;
      const bool on = r < it.n;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const void* src = s ? it.v_par : it.k_par;
        par[s] = 0u;
        if (on) par[s] = F::kFmt == RB_KV_INT8 ? static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(src) + it.par0 + r))
                                               : __ldg(reinterpret_cast<const uint32_t*>(src) + it.par0 + r);
      }
    }
  };
  auto store_par = [&](int t) {
    if constexpr (!F::kPlain) {
      float* dst = reinterpret_cast<float*>(smem + ((t - it.t0) % T::kStages) * F::kStage + 2 * F::kSide);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float sc = __uint_as_float(par[s] << 16);
        dst[s * F::kTile + tid] = sc;
        if constexpr (F::kFmt == RB_KV_INT4)  // codes enter as c - 8: m + 8 s stands for the middle of the row's range
          dst[(2 + s) * F::kTile + tid] = fmaf(
              8.f, sc, p.bf16 ? __uint_as_float(par[s] & 0xffff0000u) : __half2float(__ushort_as_half(static_cast<unsigned short>(par[s] >> 16))));
      }
    }
  };
  static_assert(F::kPlain || F::kTile == kThreads, "one thread a slot's parameters");

  __syncthreads();  // the previous item's merge has been read
#pragma unroll
  for (int i = 0; i < T::kStages - 1; ++i) {
    if (it.t0 + i < it.t1) {
      load_rows(it.t0 + i);
      load_par(it.t0 + i);
      store_par(it.t0 + i);
    }
    cp_commit();
  }

  // ---- the queries, in the order of the A fragments ----
  for (int r = warp; r < T::kRows; r += kWarps) {
    const bool on = r < it.rows;
    const int row = it.row0 + r;
    const int b = it.seq >= 0 ? it.seq : (on ? row / p.rep : 0), j = it.seq >= 0 ? r : row % p.rep;
    constexpr int kE = kHd / 32;
    const int64_t at = b * p.ldq + static_cast<int64_t>(it.kv * p.rep + (on ? j : 0)) * kHd + lane * kE;
    uint32_t raw[kE / 2];
#pragma unroll
    for (int e = 0; e < kE / 2; ++e) raw[e] = on ? __ldcg(reinterpret_cast<const unsigned int*>(reinterpret_cast<const uint16_t*>(p.q) + at) + e) : 0u;
    if (p.scale < 0.f) {
#pragma unroll
      for (int e = 0; e < kE / 2; ++e) raw[e] ^= 0x80008000u;
    }
    float f = fmaxf(fabsf(p.scale) * kLog2e, 1e-30f);
    if constexpr (!F::kPlain) {
      // fp16 queries for the codes' product: scaled by a power of two so that the row's largest is in [1, 2) - exact
      // but for elements 2^-24 below it
      float v[kE], top = 0.f, sum = 0.f;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const uint32_t u = raw[e / 2] >> (16 * (e & 1)) & 0xffffu;
        v[e] = p.bf16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(u)));
        top = fmaxf(top, fabsf(v[e]));
      }
      const uint32_t ex = __reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23;
      const uint32_t exc = ex < 30u ? 30u : (ex > 220u ? 220u : ex);
      const float down = __uint_as_float((254u - exc) << 23);
      f *= __uint_as_float(exc << 23);
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const __half h = __float2half_rn(v[e] * down);
        sum += __half2float(h);
        const uint32_t u = __half_as_ushort(h);
        raw[e / 2] = (e & 1) ? raw[e / 2] | (u << 16) : u;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) qsum[r] = sum;
    }
    if (lane == 0) rowf[r] = f;
    uint16_t* qf = reinterpret_cast<uint16_t*>(smem + T::kOffQ);
    const int mt = r >> 4, half = (r >> 3) & 1;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      int ks, qc, qp, qe;
      F::q_place(lane * kE + e, ks, qc, qp, qe);
      qf[(((mt * F::kKs + ks) * 32 + (r & 7) * 4 + qc) * 4 + qp * 2 + half) * 2 + qe] =
          static_cast<uint16_t>(raw[e / 2] >> (16 * (e & 1)));
    }
  }

  float o[kMt][F::kNv][4], l[kMt][2], w[kMt][2], ref[kMt][2], fr[kMt][2], qs[kMt][2];
  float ve = F::kPlain ? 0.f : kLowestE;  // exponent of the value scales seen, part of every row's reference
#pragma unroll
  for (int m = 0; m < kMt; ++m) {
#pragma unroll
    for (int u = 0; u < F::kNv; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][u][e] = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) l[m][x] = w[m][x] = 0.f, ref[m][x] = -INFINITY;
  }
  uint32_t qreg[kMt == 1 ? F::kKs : 1][4];

  for (int t = it.t0; t < it.t1; ++t) {
    cp_wait<T::kStages - 2>();
    __syncthreads();  // stage t is there for everybody, stage t - 1 is free
    const int ahead = t + T::kStages - 1;
    if (ahead < it.t1) {
      load_rows(ahead);
      load_par(ahead);
    }
    cp_commit();
    if (t == it.t0) {
#pragma unroll
      for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = (wm * kMt + m) * 16 + x * 8 + g;
          fr[m][x] = rowf[r];
          qs[m][x] = F::kFmt == RB_KV_INT4 ? qsum[r] : 0.f;
        }
      if constexpr (kMt == 1) {
#pragma unroll
        for (int ks = 0; ks < F::kKs; ++ks) {
          const uint4 v = lds128_a(s0 + T::kOffQ + ((wm * F::kKs + ks) * 32 + lane) * 16);
          qreg[ks][0] = v.x, qreg[ks][1] = v.y, qreg[ks][2] = v.z, qreg[ks][3] = v.w;
        }
      }
    }
    const uint32_t kt = stage(t - it.t0), vt = kt + F::kSide, pt = vt + F::kSide;
    const int64_t left = it.n - static_cast<int64_t>(t) * F::kTile;
#pragma unroll 1
    for (int b0 = wk * T::kPerWarp; b0 < (wk + 1) * T::kPerWarp; b0 += T::kBlock) {
      if (b0 >= left) break;
      float s[kMt][T::kNt][4];
#pragma unroll
      for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int n = 0; n < T::kNt; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] = 0.f;
      // ---- scores ----
      typename F::KRaw raw[T::kNt / 2];
#pragma unroll
      for (int n = 0; n < T::kNt / 2; ++n) F::k_raw(kt, b0 + 16 * n, lane, raw[n]);
#pragma unroll
      for (int ks = 0; ks < F::kKs; ++ks) {
        uint32_t a[kMt][4];
        if constexpr (kMt == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) a[0][e] = qreg[ks][e];
        } else {
#pragma unroll
          for (int m = 0; m < kMt; ++m) {
            const uint4 v = lds128_a(s0 + T::kOffQ + (((wm * kMt + m) * F::kKs + ks) * 32 + lane) * 16);
            a[m][0] = v.x, a[m][1] = v.y, a[m][2] = v.z, a[m][3] = v.w;
          }
        }
#pragma unroll
        for (int n = 0; n < T::kNt / 2; ++n) {
          uint32_t b[2][2];
          F::k_frag(kt, b0 + 16 * n, lane, ks, raw[n], b);
#pragma unroll
          for (int m = 0; m < kMt; ++m) {
            mma16816<F::kBf16>(s[m][2 * n], a[m], b[0][0], b[0][1]);
            mma16816<F::kBf16>(s[m][2 * n + 1], a[m], b[1][0], b[1][1]);
          }
        }
      }
      // ---- scales, mask, largest ----
      bool raise = false;
      float top[kMt][2];
#pragma unroll
      for (int m = 0; m < kMt; ++m) top[m][0] = top[m][1] = -INFINITY;
#pragma unroll
      for (int n = 0; n < T::kNt; ++n) {
        const int col = b0 + 8 * n + 2 * c;
        if constexpr (!F::kPlain) {
          const float2 ks = lds64f_a(pt + col * 4);
          float2 km = make_float2(0.f, 0.f);
          if constexpr (F::kFmt == RB_KV_INT4) km = lds64f_a(pt + (2 * F::kTile + col) * 4);
#pragma unroll
          for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float sc = (e & 1) ? ks.y : ks.x;
              if constexpr (F::kFmt == RB_KV_INT4)
                s[m][n][e] = fmaf(s[m][n][e], sc, ((e & 1) ? km.y : km.x) * qs[m][e >> 1]);
              else
                s[m][n][e] *= sc;
            }
        }
        if (b0 + T::kBlock > left) {
#pragma unroll
          for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + (e & 1) >= left) s[m][n][e] = -INFINITY;
        }
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[m][e >> 1] = fmaxf(top[m][e >> 1], s[m][n][e]);
      }
#pragma unroll
      for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int x = 0; x < 2; ++x) raise |= top[m][x] * fr[m][x] > ref[m][x] + kSlack;
      float ven = ve;
      if constexpr (!F::kPlain) {
        // the block's largest value scale (NaN left out: it shows by itself): its exponent goes into the reference,
        // so that the 16-bit p s stay within fp16's range whatever the size of the values
        const float vs = lane < T::kBlock ? __uint_as_float(lds32_a(pt + (F::kTile + b0 + lane) * 4)) : 0.f;
        const uint32_t hi = __reduce_max_sync(0xffffffffu, vs == vs ? __float_as_uint(vs) : 0u);
        ven = fmaxf(ve, fminf(fmaxf(static_cast<float>(static_cast<int>(hi >> 23) - 127), kLowestE), kHighestE));
        raise |= ven > ve;
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float v = top[m][x];
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
            const float nr = fmaxf(ref[m][x], v * fr[m][x]);
            const float f = ref[m][x] == -INFINITY ? 0.f : ex2((ref[m][x] - nr) + (ve - ven));
            ref[m][x] = nr;
            l[m][x] *= f;
            w[m][x] *= f;
#pragma unroll
            for (int u = 0; u < F::kNv; ++u) o[m][u][2 * x] *= f, o[m][u][2 * x + 1] *= f;
          }
        ve = ven;
      }
      // ---- probabilities ----
      float base[kMt][2];
#pragma unroll
      for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int x = 0; x < 2; ++x) base[m][x] = ref[m][x] == -INFINITY ? 0.f : -(ref[m][x] + ve);
#pragma unroll
      for (int n = 0; n < T::kNt; ++n) {
        const int col = b0 + 8 * n + 2 * c;
        float2 vs = make_float2(1.f, 1.f), vm = make_float2(0.f, 0.f);
        if constexpr (!F::kPlain) vs = lds64f_a(pt + (F::kTile + col) * 4);
        if constexpr (F::kFmt == RB_KV_INT4) vm = lds64f_a(pt + (3 * F::kTile + col) * 4);
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float pr = ex2(fmaf(s[m][n][e], fr[m][e >> 1], base[m][e >> 1]));
            l[m][e >> 1] += pr;
            if constexpr (F::kFmt == RB_KV_INT4) w[m][e >> 1] = fmaf(pr, (e & 1) ? vm.y : vm.x, w[m][e >> 1]);
            if constexpr (!F::kPlain) pr *= (e & 1) ? vs.y : vs.x;
            s[m][n][e] = pr;
          }
      }
      // ---- O += p v ----
#pragma unroll
      for (int n = 0; n < T::kNt / 2; ++n) {
        uint32_t a[kMt][4];
#pragma unroll
        for (int m = 0; m < kMt; ++m) {
          a[m][0] = pack2<F::kBf16>(s[m][2 * n][0], s[m][2 * n][1]);
          a[m][1] = pack2<F::kBf16>(s[m][2 * n][2], s[m][2 * n][3]);
          a[m][2] = pack2<F::kBf16>(s[m][2 * n + 1][0], s[m][2 * n + 1][1]);
          a[m][3] = pack2<F::kBf16>(s[m][2 * n + 1][2], s[m][2 * n + 1][3]);
        }
        // 4-bit rows: a value's part s (c - 8) may be far larger than the value, so the rounding of p s to fp16 is
        // made up for by a second term
        uint32_t a2[F::kFmt == RB_KV_INT4 ? kMt : 1][4];
        if constexpr (F::kFmt == RB_KV_INT4) {
#pragma unroll
          for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&a[m][e]));
              a2[m][e] = pack2<false>(s[m][2 * n + (e >> 1)][2 * (e & 1)] - hi.x, s[m][2 * n + (e >> 1)][2 * (e & 1) + 1] - hi.y);
            }
        }
        F::v_frags(vt, b0 + 16 * n, lane, [&](int u, uint32_t f0, uint32_t f1) {
#pragma unroll
          for (int m = 0; m < kMt; ++m) mma16816<F::kBf16>(o[m][u], a[m], f0, f1);
          if constexpr (F::kFmt == RB_KV_INT4) {
#pragma unroll
            for (int m = 0; m < kMt; ++m) mma16816<false>(o[m][u], a2[m], f0, f1);
          }
        });
      }
    }
    if (ahead < it.t1) store_par(ahead);
  }
  cp_wait<0>();

  // ---- join the warps along the slots, in their order, and leave the item's partial ----
#pragma unroll
  for (int m = 0; m < kMt; ++m)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[m][x] += __shfl_xor_sync(0xffffffffu, l[m][x], 1);
      l[m][x] += __shfl_xor_sync(0xffffffffu, l[m][x], 2);
      if constexpr (F::kFmt == RB_KV_INT4) {
        w[m][x] += __shfl_xor_sync(0xffffffffu, w[m][x], 1);
        w[m][x] += __shfl_xor_sync(0xffffffffu, w[m][x], 2);
      }
      if (c == 0) rl[wk * T::kRows + (wm * kMt + m) * 16 + x * 8 + g] =
          make_float2(ref[m][x] == -INFINITY && l[m][x] == 0.f ? -INFINITY : (ref[m][x] == -INFINITY ? 0.f : ref[m][x] + ve), l[m][x]);
    }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < kMt; ++m) {
    float f[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = (wm * kMt + m) * 16 + x * 8 + g;
      float hi = -INFINITY;
#pragma unroll
      for (int k = 0; k < T::kWk; ++k) hi = fmaxf(hi, rl[k * T::kRows + r].x);
      const float mine = rl[wk * T::kRows + r].x;
      f[x] = mine == -INFINITY ? 0.f : ex2(mine - hi);
    }
    uint8_t* dst = smem + (warp * kMt + m) * T::kMergeRow;
#pragma unroll
    for (int u = 0; u < F::kNv; ++u)
      *reinterpret_cast<float4*>(dst + (u * 33 + lane) * 16) =
          make_float4((o[m][u][0] + w[m][0]) * f[0], (o[m][u][1] + w[m][0]) * f[0], (o[m][u][2] + w[m][1]) * f[1],
                      (o[m][u][3] + w[m][1]) * f[1]);
  }
  __syncthreads();
  for (int x = tid; x < it.rows * (kHd / 2); x += kThreads) {
    const int r = x / (kHd / 2), d2 = x % (kHd / 2);
    const int mt = r >> 4, m = mt % kMt, rw = mt / kMt, half = (r >> 3) & 1;
    // columns o_col(u, n), o_col(u, n + 1) of the fragments: a pair in the plain order, strided in the codes' order
    float2 acc = make_float2(0.f, 0.f);
    const int u = F::kPlain ? d2 >> 2 : d2 % F::kNv, n = F::kPlain ? (d2 & 3) * 2 : (d2 / F::kNv) * 2;
#pragma unroll
    for (int k = 0; k < T::kWk; ++k) {
      const float2 v = *reinterpret_cast<const float2*>(smem + ((k * kWm + rw) * kMt + m) * T::kMergeRow +
                                                        (u * 33 + (r & 7) * 4 + n / 2) * 16 + half * 8);
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
#pragma unroll
    for (int k = 0; k < T::kWk; ++k) hi = fmaxf(hi, rl[k * T::kRows + r].x);
#pragma unroll
    for (int k = 0; k < T::kWk; ++k) {
      const float2 v = rl[k * T::kRows + r];
      sum += v.x == -INFINITY ? 0.f : v.y * ex2(v.x - hi);
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
  __shared__ unsigned long long sum_s;
  __shared__ int most_s;
  if (threadIdx.x == 0) sum_s = 0, most_s = 0;
  const int64_t np_raw = p.pre.k ? *p.pre.len : 0;
  __syncthreads();
  if (p.own.k) {
    unsigned long long sum = 0;
    int most = 0;
    for (int b = threadIdx.x; b < p.n_seqs; b += blockDim.x) {
      const int64_t n = p.own.len[b];
      if (n <= 0 || n > p.own.cache_len) continue;
      const int t = static_cast<int>((n + kTile - 1) / kTile);
      sum += t + 2;  // an item's start and end cost about two stages
      most = most > t ? most : t;
    }
    if (sum) atomicAdd(&sum_s, sum), atomicMax(&most_s, most);
  }
  __syncthreads();
  Plan pl;
  pl.prefix_ok = np_raw >= 0 && np_raw <= p.pre.cache_len;
  const int64_t n = pl.prefix_ok ? np_raw : 0;
  const int tiles = static_cast<int>((n + kTile - 1) / kTile), lanes = p.n_kv * p.tiles_m;
  const double own = static_cast<double>(sum_s) * p.n_kv, pre = static_cast<double>(tiles) * lanes;
  int g_own = own > 0 ? static_cast<int>(grid * (own / (own + pre)) + 0.5) : 0;
  if (own > 0 && g_own < 1) g_own = 1;
  if (tiles > 0 && g_own >= grid) g_own = grid - 1;
  pl.np = tiles ? max(1, min(min((grid - g_own) / lanes, tiles), p.max_np)) : 0;
  pl.pt = pl.np ? (tiles + pl.np - 1) / pl.np : 0;
  pl.np = pl.pt ? (tiles + pl.pt - 1) / pl.pt : 0;
  pl.ns = most_s ? min(p.max_ns, (most_s + 3) / 4) : 0;  // at least four stages a split
  pl.ot = pl.ns ? (most_s + pl.ns - 1) / pl.ns : 0;
  pl.ns = pl.ot ? (most_s + pl.ot - 1) / pl.ot : 0;
  pl.prefix_items = lanes * pl.np;
  pl.own_items = p.n_seqs * p.n_kv * pl.ns;
  return pl;
}

template <typename F, int kMt, int kWm>
__global__ void __launch_bounds__(kThreads, 2) prefix_attn_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  griddep_wait();
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
  for (; i < end; i += step) {
    Item it;
    if (i < pl.prefix_items) {
      const int lane_i = i / pl.np, sp = i % pl.np;
      it.kv = lane_i / p.tiles_m;
      const int rt = lane_i % p.tiles_m;
      constexpr int kRows = Tile<F, kMt, kWm>::kRows;
      const int64_t row = static_cast<int64_t>(it.kv) * p.pre.cache_len;
      it.k = p.pre.k + row * F::kRow;
      it.v = p.pre.v + row * F::kRow;
      it.k_par = p.pre.k_par;
      it.v_par = p.pre.v_par;
      it.par0 = row;
      it.n = *p.pre.len;
      it.t0 = sp * pl.pt;
      it.t1 = min(static_cast<int>((it.n + F::kTile - 1) / F::kTile), it.t0 + pl.pt);
      it.seq = -1;
      it.row0 = rt * kRows;
      it.rows = min(kRows, p.n_seqs * p.rep - it.row0);
      const int64_t slot = static_cast<int64_t>(lane_i) * p.max_np + sp;
      it.o = p.o + slot * kRows * F::kHd;
      it.rl = p.rl + slot * kRows;
      run_item<F, kMt, kWm>(p, it, smem);
    } else {
      const int x = i - pl.prefix_items, sp = x % pl.ns;
      it.kv = (x / pl.ns) % p.n_kv;
      it.seq = x / pl.ns / p.n_kv;
      it.n = p.own.len[it.seq];
      if (it.n < 0 || it.n > p.own.cache_len) {
        if (threadIdx.x == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
        continue;
      }
      it.t0 = sp * pl.ot;
      it.t1 = min(static_cast<int>((it.n + F::kTile - 1) / F::kTile), it.t0 + pl.ot);
      if (it.t0 >= it.t1) continue;
      const int64_t head = static_cast<int64_t>(it.seq) * p.n_kv + it.kv, row = head * p.own.cache_len;
      it.k = p.own.k + row * F::kRow;
      it.v = p.own.v + row * F::kRow;
      it.k_par = p.own.k_par;
      it.v_par = p.own.v_par;
      it.par0 = row;
      it.row0 = 0;
      it.rows = p.rep;
      const int64_t slot = head * p.max_ns + sp;
      it.o = p.o + p.own_o + slot * p.rep * F::kHd;
      it.rl = p.rl + p.own_rl + slot * p.rep;
      run_item<F, 1, 1>(p, it, smem);
    }
  }
  // an own length outside its cache with no item of its own (no split at all) is reported here
  if (cta == 0 && pl.ns == 0 && p.own.k)
    for (int b = threadIdx.x; b < p.n_seqs; b += kThreads)
      if (p.own.len[b] < 0 || p.own.len[b] > p.own.cache_len) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
}

// One warp joins the partials of one (sequence, query head): prefix splits, then own splits, in order.
template <int kHd>
__global__ void __launch_bounds__(kThreads) prefix_attn_merge(const __grid_constant__ Params p, int tile_rows, int stage) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= p.n_seqs * p.n_q) return;
  const int b = row / p.n_q, h = row % p.n_q, kv = h / p.rep, j = h % p.rep;
  const int64_t n_pre = p.pre.k ? *p.pre.len : 0, n_own = p.own.k ? p.own.len[b] : 0;
  if (n_pre < 0 || n_pre > p.pre.cache_len || n_own < 0 || n_own > p.own.cache_len) return;
  const int np = p.plan[0], ot = p.plan[3];
  const int ns = n_own ? static_cast<int>(((n_own + stage - 1) / stage + ot - 1) / ot) : 0;
  const int r = b * p.rep + j, rt = r / tile_rows;
  const int64_t slot0 = (static_cast<int64_t>(kv) * p.tiles_m + rt) * p.max_np;
  const int64_t own0 = (static_cast<int64_t>(b) * p.n_kv + kv) * p.max_ns;
  auto rl_of = [&](int i) {
    return i < np ? p.rl + (slot0 + i) * tile_rows + r % tile_rows : p.rl + p.own_rl + (own0 + i - np) * p.rep + j;
  };
  auto o_of = [&](int i) {
    return i < np ? p.o + ((slot0 + i) * tile_rows + r % tile_rows) * kHd : p.o + p.own_o + ((own0 + i - np) * p.rep + j) * kHd;
  };
  const int n = np + ns;
  float hi = -INFINITY;
  for (int i = lane; i < n; i += 32) hi = fmaxf(hi, __ldcg(rl_of(i)).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  constexpr int kE = kHd / 32;
  float acc[kE], l = 0.f;
#pragma unroll
  for (int e = 0; e < kE; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float2 v = __ldcg(rl_of(i));
    const float f = v.x == -INFINITY ? 0.f : ex2(v.x - hi);
    l = fmaf(v.y, f, l);
    const float* src = o_of(i) + lane * kE;
    if constexpr (kE == 4) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
      acc[0] = fmaf(x.x, f, acc[0]), acc[1] = fmaf(x.y, f, acc[1]), acc[2] = fmaf(x.z, f, acc[2]), acc[3] = fmaf(x.w, f, acc[3]);
    } else {
      const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
      acc[0] = fmaf(x.x, f, acc[0]), acc[1] = fmaf(x.y, f, acc[1]);
    }
  }
  const float inv = n_pre + n_own == 0 ? 0.f : 1.f / l;
  uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.out) + b * p.ldo + static_cast<int64_t>(h) * kHd + lane * kE);
#pragma unroll
  for (int e = 0; e < kE; e += 2) {
    const float x = n_pre + n_own == 0 ? 0.f : acc[e] * inv, y = n_pre + n_own == 0 ? 0.f : acc[e + 1] * inv;
    dst[e / 2] = p.bf16 ? pack2<true>(x, y) : pack2<false>(x, y);
  }
}

struct Config {
  int mt, wm;
};
// The narrowest tile that holds the batch's rows: a warp of one or two 16-row tiles reads each key once; beyond 32 rows
// two or four warps share the keys.
inline Config config_of(int64_t rows) {
  if (rows <= 16) return {1, 1};
  if (rows <= 32) return {2, 1};
  if (rows <= 64) return {2, 2};
  return {2, 4};
}

struct Layout {
  int grid, tile_rows, tiles_m, max_np, max_ns;
  int64_t pre_slots, own_slots, rl_bytes, o_bytes, total;
};
inline Layout layout_of(const rb_prefix_attn_args* a, int num_sms) {
  const rb_kv_cache* c = a->prefix ? a->prefix : a->own;
  const int rep = a->n_q_heads / c->n_kv_heads;
  const int64_t rows = a->n_seqs * rep;
  const Config cf = config_of(rows);
  Layout L = {};
  L.grid = 2 * num_sms;
  L.tile_rows = 16 * cf.mt * cf.wm;
  L.tiles_m = static_cast<int>((rows + L.tile_rows - 1) / L.tile_rows);
  const int64_t lanes = static_cast<int64_t>(c->n_kv_heads) * L.tiles_m, heads = a->n_seqs * c->n_kv_heads;
  L.max_np = a->prefix ? static_cast<int>(std::max<int64_t>(1, L.grid / std::max<int64_t>(lanes, 1))) : 0;
  L.max_ns = a->own ? static_cast<int>(std::max<int64_t>(1, L.grid / std::max<int64_t>(heads, 1))) : 0;
  L.pre_slots = lanes * L.max_np * L.tile_rows;
  L.own_slots = heads * L.max_ns * rep;
  L.rl_bytes = ((L.pre_slots + L.own_slots) * 8 + 255) / 256 * 256;
  L.o_bytes = (L.pre_slots + L.own_slots) * c->head_dim * 4;
  L.total = 256 + L.rl_bytes + L.o_bytes;
  return L;
}

template <typename F, int kMt, int kWm>
int launch_main(const Params& p, int grid, int flags, cudaStream_t stream) {
  constexpr int smem = Tile<F, kMt, kWm>::kSmem > Tile<F, 1, 1>::kSmem ? Tile<F, kMt, kWm>::kSmem : Tile<F, 1, 1>::kSmem;
  static_assert(smem <= 113 * 1024, "two CTAs an SM");
  void (*kern)(Params) = prefix_attn_kernel<F, kMt, kWm>;
  if (ensure_smem_limit(reinterpret_cast<const void*>(kern), smem) != cudaSuccess) return RB_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (flags & RB_FLAG_PDL) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? RB_OK : RB_ERR_LAUNCH;
}

template <typename F>
int launch_format(const Params& p, const Layout& L, Config cf, int flags, cudaStream_t stream) {
  int st;
  if (cf.mt == 1) st = launch_main<F, 1, 1>(p, L.grid, flags, stream);
  else if (cf.wm == 1) st = launch_main<F, 2, 1>(p, L.grid, flags, stream);
  else if (cf.wm == 2) st = launch_main<F, 2, 2>(p, L.grid, flags, stream);
  else st = launch_main<F, 2, 4>(p, L.grid, flags, stream);
  if (st != RB_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.n_seqs * p.n_q + kWarps - 1) / kWarps);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (flags & RB_FLAG_PDL) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, prefix_attn_merge<F::kHd>, p, L.tile_rows, F::kTile) == cudaSuccess ? RB_OK : RB_ERR_LAUNCH;
}

}  // namespace pfx

int64_t prefix_attn_workspace(const rb_prefix_attn_args* a, int num_sms) { return pfx::layout_of(a, num_sms).total; }

int launch_prefix_attn(const rb_prefix_attn_args* a, int num_sms, int flags, cudaStream_t stream) {
  using namespace pfx;
  const rb_kv_cache* c = a->prefix ? a->prefix : a->own;
  const Layout L = layout_of(a, num_sms);
  Params p = {};
  p.q = a->q;
  p.out = a->out;
  p.ldq = a->ldq;
  p.ldo = a->ldo;
  auto side = [](const rb_kv_cache* s, const int64_t* len) {
    return Side{static_cast<const uint8_t*>(s->k), static_cast<const uint8_t*>(s->v), s->k_par, s->v_par, len, s->cache_len};
  };
  if (a->prefix) p.pre = side(a->prefix, a->prefix_len);
  if (a->own) p.own = side(a->own, a->own_len);
  p.n_seqs = static_cast<int>(a->n_seqs);
  p.n_q = a->n_q_heads;
  p.n_kv = c->n_kv_heads;
  p.rep = p.n_q / p.n_kv;
  p.bf16 = c->dtype == RB_BF16;
  p.scale = a->scale;
  p.tiles_m = L.tiles_m;
  p.max_np = L.max_np;
  p.max_ns = L.max_ns;
  uint8_t* w = static_cast<uint8_t*>(a->ws);
  p.plan = reinterpret_cast<int*>(w);
  p.rl = reinterpret_cast<float2*>(w + 256);
  p.o = reinterpret_cast<float*>(w + 256 + L.rl_bytes);
  p.own_rl = L.pre_slots;
  p.own_o = L.pre_slots * c->head_dim;
  const Config cf = config_of(a->n_seqs * p.rep);
  const bool wide = c->head_dim == 128;
  switch (c->fmt) {
    case RB_KV_INT8:
      return wide ? launch_format<Fmt<128, RB_KV_INT8, false>>(p, L, cf, flags, stream)
                  : launch_format<Fmt<64, RB_KV_INT8, false>>(p, L, cf, flags, stream);
    case RB_KV_INT4:
      return wide ? launch_format<Fmt<128, RB_KV_INT4, false>>(p, L, cf, flags, stream)
                  : launch_format<Fmt<64, RB_KV_INT4, false>>(p, L, cf, flags, stream);
    default:
      if (p.bf16)
        return wide ? launch_format<Fmt<128, RB_KV_PLAIN, true>>(p, L, cf, flags, stream)
                    : launch_format<Fmt<64, RB_KV_PLAIN, true>>(p, L, cf, flags, stream);
      return wide ? launch_format<Fmt<128, RB_KV_PLAIN, false>>(p, L, cf, flags, stream)
                  : launch_format<Fmt<64, RB_KV_PLAIN, false>>(p, L, cf, flags, stream);
  }
}

}  // namespace rb
