// prefix_attn_tc.cu - the shared prefix's part of rb_prefix_attn on the tcgen05 tensor cores, for batches with more query
// rows per key-value head than the warp-level kernel (prefix_attn.cu) streams at HBM rate. The mathematics, the formats'
// rules and the partials are those of prefix_attn.cu.
//
// One CTA takes 128 query rows of one key-value head and a split of the prefix, in tiles of 128 slots. M = 128 rows:
//   S = Q K^T    Q and K in shared memory (K-major, 128-byte swizzle), S in tensor memory
//   O += P V     P in tensor memory as 16-bit values over the columns of S it came from, V in shared memory as its rows
//                lie (MN-major), O in tensor memory
// Two groups of four softmax warps (thread = row = tensor-memory lane) take the tiles in turn, each with its own S, its
// own O and its own references: 4 x 128 columns fill the tensor memory, and a group only waits for the tensor core. They
// leave two partials. One thread issues every MMA, in the order QK(0) QK(1) PV(0) QK(2) PV(1) ...: MMAs of one thread
// complete in order, so QK(t + 2) may overwrite the columns that PV(t) read. Eight loader warps fill rings of two key
// and three value tiles: 16-bit rows by asynchronous copies, codes through registers, converted to 16-bit integers on
// the way (a tile ahead, so that a whole tile of codes is always in flight).
#include "common.cuh"
#include "tc.cuh"
#include "kernels.h"

namespace rb {

namespace pfxt {

using pfx::ex2;
using pfx::Item;
using pfx::Params;

constexpr int kTile = 128;        // slots of a tile, and query rows of a CTA
constexpr int kSoftWarps = 8;
constexpr int kMmaWarp = 8;
constexpr int kFirstLoad = 9;
constexpr int kLoadWarps = 8;
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int kThreads = (kFirstLoad + kLoadWarps) * 32;
constexpr int kKRing = 2, kVRing = 3;
constexpr uint32_t kTmemCols = 512;

template <int kHd_, int kFmt_, bool kBf16_>
struct Fmt {
  static constexpr int kHd = kHd_, kFmt = kFmt_;
  static constexpr bool kBf16 = kBf16_, kPlain = kFmt == RB_KV_PLAIN;
  static constexpr int kRow = kPlain ? 2 * kHd : (kFmt == RB_KV_INT8 ? kHd : kHd / 2);
  static constexpr int kAtom = kTile * 128;              // 64 columns of 128 rows
  static constexpr int kTileBytes = kTile * kHd * 2;     // a tile of 16-bit values
  static constexpr int kPar = kTile * 4 * 4;             // fp32 s of keys, s of values, m of keys, m of values
  static constexpr int kOffK = kTileBytes, kOffV = kOffK + kKRing * kTileBytes, kOffPar = kOffV + kVRing * kTileBytes;
  static constexpr int kOffBar = kOffPar + kVRing * kPar;
  static constexpr int kBars = 2 * kKRing + 2 * kVRing + 3 * 2 + 1;
  static constexpr int kSmem = 1024 + kOffBar + kBars * 8 + 16;
  static constexpr int kRaw = kPlain ? 1 : kTile * kRow / 16 / kLoadThreads;  // 16-byte pieces of a thread in a tile of codes
  static constexpr uint32_t kType = kBf16 ? 1u : 0u;
  static constexpr uint32_t kIdesc = (1u << 4) | (kType << 7) | (kType << 10) | (static_cast<uint32_t>(kTile >> 4) << 24);
  static constexpr uint32_t kIdescQk = kIdesc | (static_cast<uint32_t>(kTile >> 3) << 17);
  static constexpr uint32_t kIdescPv = kIdesc | (static_cast<uint32_t>(kHd >> 3) << 17) | (1u << 16);  // B is MN-major
};

// Descriptor of V: MN-major, 128-byte swizzle; 64-column atoms kAtom bytes apart, groups of eight slots 1024.
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr, uint32_t atom) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(atom >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t a, float (&f)[32]) {
  uint32_t v[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(a)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ float4 lds128f(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}

// Byte offset of the 16-byte piece `ch` (eight 16-bit columns) of row r in a swizzled tile.
__device__ __forceinline__ uint32_t piece_at(int r, int ch) { return (ch >> 3) * (kTile * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4); }

template <typename F>
__global__ void __launch_bounds__(kThreads, 1) prefix_attn_tc_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s0 = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + F::kOffBar);
  uint64_t* kempty = kfull + kKRing;
  uint64_t* vfull = kempty + kKRing;
  uint64_t* vempty = vfull + kVRing;
  uint64_t* sfull = vempty + kVRing;  // [2] S of the group's tile is there
  uint64_t* pfull = sfull + 2;        // [2] the group has written P (four warps)
  uint64_t* pvdone = pfull + 2;       // [2] the group's last PV is complete
  uint64_t* qfull = pvdone + 2;       // Q is in shared memory (four warps)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(qfull + 1);

  griddep_wait();
  griddep_launch_dependents();
  const int64_t n = *p.pre.len;
  const int lane_i = blockIdx.x / p.max_np, sp = blockIdx.x % p.max_np;
  const int kv = lane_i / p.tiles_m, row0 = (lane_i % p.tiles_m) * kTile;
  if (n < 0 || n > p.pre.cache_len) {
    if (blockIdx.x == 0 && tid == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
    return;
  }
  const int tiles = static_cast<int>((n + kTile - 1) / kTile);
  const int per = (tiles + p.max_np - 1) / p.max_np;
  const int t0 = sp * per, t1 = min(tiles, t0 + per), nt = t1 - t0;
  if (nt <= 0) return;  // the merge knows which splits there are

  if (tid == 0) {
    for (int i = 0; i < kKRing; ++i) {
      mbar_init(kfull + i, kLoadWarps);
      mbar_init(kempty + i, 1);
    }
    for (int i = 0; i < kVRing; ++i) {
      mbar_init(vfull + i, kLoadWarps);
      mbar_init(vempty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull + i, 1);
      mbar_init(pfull + i, 4);
      mbar_init(pvdone + i, 1);
    }
    mbar_init(qfull, 4);
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  mm4::tc_fence_before();
  __syncthreads();
  mm4::tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // S of group 0, S of group 1, O of group 0, O of group 1: 128 columns each
  const int64_t head = static_cast<int64_t>(kv) * p.pre.cache_len;  // the head's first row

  if (warp == kMmaWarp) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      bool ok = mbar_wait(qfull, 0, ERR_PFX_WAIT);
      mm4::tc_fence_after();
      for (int t = 0; t <= nt && ok; ++t) {
        if (t < nt) {
          const int ks = t % kKRing;
          ok = mbar_wait(kfull + ks, (t / kKRing) & 1, ERR_PFX_WAIT);
          if (!ok) break;
          mm4::tc_fence_after();
          const uint32_t kt = s0 + F::kOffK + ks * F::kTileBytes;
#pragma unroll
          for (int i = 0; i < F::kHd / 16; ++i)
            umma_ss(tmem + (t & 1) * kTile, mm4::sw128_desc(s0 + (i >> 2) * F::kAtom + (i & 3) * 32),
                    mm4::sw128_desc(kt + (i >> 2) * F::kAtom + (i & 3) * 32), F::kIdescQk, i != 0);
          mm4::umma_commit(sfull + (t & 1));
          mm4::umma_commit(kempty + ks);
        }
        if (t > 0) {
          const int u = t - 1, vs = u % kVRing, g = u & 1;
          ok = mbar_wait(vfull + vs, (u / kVRing) & 1, ERR_PFX_WAIT) && mbar_wait(pfull + g, (u >> 1) & 1, ERR_PFX_WAIT);
          if (!ok) break;
          mm4::tc_fence_after();
          const uint32_t vt = s0 + F::kOffV + vs * F::kTileBytes, s = tmem + g * kTile, o = tmem + (2 + g) * kTile;
#pragma unroll
          for (int i = 0; i < kTile / 16; ++i)
            umma_ts(o, s + 32 * (i >> 1) + 8 * (i & 1), v_desc(vt + i * 2048, F::kAtom), F::kIdescPv, u >= 2 || i != 0);
          if constexpr (F::kFmt == RB_KV_INT4) {
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
              umma_ts(o, s + 32 * (i >> 1) + 16 + 8 * (i & 1), v_desc(vt + i * 2048, F::kAtom), F::kIdescPv, 1);
          }
          mm4::umma_commit(vempty + vs);
          mm4::umma_commit(pvdone + g);
        }
      }
    }
  } else if (warp >= kFirstLoad) {
    // ---------------- loaders ----------------
    const int lt = tid - kFirstLoad * 32;
    bool ok = true;
    auto arrive = [&](uint64_t* bar) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    const uint8_t* k = p.pre.k + head * F::kRow;
    const uint8_t* v = p.pre.v + head * F::kRow;
    if constexpr (F::kPlain) {
      constexpr int kPieces = F::kRow / 16, kEach = kTile * kPieces / kLoadThreads;
      auto load = [&](const uint8_t* src, uint32_t dst, int t) {
        const int64_t first = static_cast<int64_t>(t0 + t) * kTile;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int x = i * kLoadThreads + lt, r = x / kPieces, ch = x % kPieces;
          const bool on = first + r < n;
          pfx::cp_async16(dst + piece_at(r, ch), on ? src + (first + r) * F::kRow + ch * 16 : src, on);
        }
        pfx::cp_commit();
      };
      for (int t = 0; t <= nt; ++t) {
        if (t < nt) {
          if (t >= kKRing && ok) ok = mbar_wait(kempty + t % kKRing, (t / kKRing - 1) & 1, ERR_PFX_WAIT);
          if (ok) load(k, s0 + F::kOffK + (t % kKRing) * F::kTileBytes, t);
          if (t >= kVRing && ok) ok = mbar_wait(vempty + t % kVRing, (t / kVRing - 1) & 1, ERR_PFX_WAIT);
          if (ok) load(v, s0 + F::kOffV + (t % kVRing) * F::kTileBytes, t);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        if (t > 0) {  // the tile before has landed
          if (t < nt) pfx::cp_wait<2>();
          else pfx::cp_wait<0>();
          arrive(kfull + (t - 1) % kKRing);
          arrive(vfull + (t - 1) % kVRing);
        }
      }
      pfx::cp_wait<0>();
    } else {
      constexpr int kPieces = F::kRow / 16;
      uint4 kr[F::kRaw], vr[F::kRaw];
      uint32_t par = 0u;
      auto fetch = [&](const uint8_t* src, int t, uint4 (&raw)[F::kRaw]) {
        const int64_t first = static_cast<int64_t>(t0 + t) * kTile;
#pragma unroll
        for (int i = 0; i < F::kRaw; ++i) {
          const int x = i * kLoadThreads + lt;
          raw[i] = make_uint4(0u, 0u, 0u, 0u);
          if (first + x / kPieces < n) raw[i] = ldg_cg_128(src + first * F::kRow + x * 16);
        }
      };
      auto fetch_par = [&](int t) {  // threads 0..127: a key's, 128..255: a value's
        const int64_t r = static_cast<int64_t>(t0 + t) * kTile + (lt & (kTile - 1));
        const void* src = lt < kTile ? p.pre.k_par : p.pre.v_par;
        par = 0u;
        if (r < n)
          par = F::kFmt == RB_KV_INT8 ? static_cast<uint32_t>(__ldcg(reinterpret_cast<const unsigned short*>(src) + head + r))
                                      : __ldcg(reinterpret_cast<const unsigned int*>(src) + head + r);
      };
      auto store = [&](uint32_t dst, const uint4 (&raw)[F::kRaw]) {
#pragma unroll
        for (int i = 0; i < F::kRaw; ++i) {
          const int x = i * kLoadThreads + lt, r = x / kPieces, ch = x % kPieces;
          const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          if constexpr (F::kFmt == RB_KV_INT8) {
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              h[2 * e] = mm4::hsub2_u(__byte_perm(w[e], 0x64646464u, 0x4140), 0x64806480u);  // 1024 + (c + 128) - 1152
              h[2 * e + 1] = mm4::hsub2_u(__byte_perm(w[e], 0x64646464u, 0x4342), 0x64806480u);
            }
            sts128(dst + piece_at(r, 2 * ch), h[0], h[1], h[2], h[3]);
            sts128(dst + piece_at(r, 2 * ch + 1), h[4], h[5], h[6], h[7]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // a word: eight columns
              uint32_t h[4];
#pragma unroll
              for (int b = 0; b < 4; ++b)  // (1024 + low nibble, 64 + high nibble) - (1032, 72): c - 8
                h[b] = mm4::hsub2_u(and_or(__byte_perm(w[e], 0u, 0x4040u | (0x0101u * b)), 0x00F0000Fu, 0x54006400u), 0x54806408u);
              sts128(dst + piece_at(r, 4 * ch + e), h[0], h[1], h[2], h[3]);
            }
          }
        }
      };
      auto store_par = [&](int t) {
        float* dst = reinterpret_cast<float*>(smem + F::kOffPar + (t % kVRing) * F::kPar);
        const float s = __uint_as_float(par << 16);
        dst[lt] = s;
        if constexpr (F::kFmt == RB_KV_INT4)
          dst[2 * kTile + lt] =
              fmaf(8.f, s, p.bf16 ? __uint_as_float(par & 0xffff0000u) : __half2float(__ushort_as_half(static_cast<unsigned short>(par >> 16))));
      };
      fetch(k, 0, kr);
      fetch(v, 0, vr);
      fetch_par(0);
      for (int t = 0; t < nt; ++t) {
        if (t >= kKRing && ok) ok = mbar_wait(kempty + t % kKRing, (t / kKRing - 1) & 1, ERR_PFX_WAIT);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        store(s0 + F::kOffK + (t % kKRing) * F::kTileBytes, kr);
        if (t + 1 < nt) fetch(k, t + 1, kr);
        arrive(kfull + t % kKRing);
        if (t >= kVRing && ok) ok = mbar_wait(vempty + t % kVRing, (t / kVRing - 1) & 1, ERR_PFX_WAIT);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        store_par(t);
        store(s0 + F::kOffV + (t % kVRing) * F::kTileBytes, vr);
        if (t + 1 < nt) {
          fetch(v, t + 1, vr);
          fetch_par(t + 1);
        }
        arrive(vfull + t % kVRing);
      }
    }
  } else {
    // ---------------- softmax: group g takes the tiles t % 2 == g; thread = row ----------------
    const int g = warp >> 2, quad = warp & 3, r = quad * 32 + lane, row = row0 + r;
    const int rows = min(kTile, p.n_seqs * p.rep - row0);
    const bool on = r < rows, busy = quad * 32 < rows;  // busy: the warp has a row of the batch
    const uint32_t tq = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t ts = tq + g * kTile, to = tq + (2 + g) * kTile;
    float fr = fmaxf(fabsf(p.scale) * pfx::kLog2e, 1e-30f), qs = 0.f;
    {
      // the row of Q: group 0 writes it to shared memory, both keep its factor and sum
      const int b = on ? row / p.rep : 0, j = on ? row % p.rep : 0;
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + b * p.ldq + static_cast<int64_t>(kv * p.rep + j) * F::kHd);
      const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
      float down = 1.f;
      if constexpr (!F::kPlain) {
        uint32_t top = 0u;
#pragma unroll 4
        for (int i = 0; i < F::kHd / 8; ++i) {
          const uint4 x = on ? __ldcg(src + i) : make_uint4(0u, 0u, 0u, 0u);
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
        }
        const uint32_t t16 = max(top & 0xffffu, top >> 16);
        const uint32_t ex = __float_as_uint(p.bf16 ? __uint_as_float(t16 << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(t16)))) >> 23;
        const uint32_t exc = ex < 30u ? 30u : (ex > 220u ? 220u : ex);
        down = __uint_as_float((254u - exc) << 23);
        fr *= __uint_as_float(exc << 23);
      }
#pragma unroll 4
      for (int i = 0; i < F::kHd / 8; ++i) {
        const uint4 x = on ? __ldcg(src + i) : make_uint4(0u, 0u, 0u, 0u);
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (!F::kPlain) {
            float2 f;
            if (p.bf16) f = make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
            else f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
            w[e] = pfx::pack2<false>(f.x * down, f.y * down);
            if constexpr (F::kFmt == RB_KV_INT4) {
              f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
              qs += f.x + f.y;
            }
          }
          w[e] ^= flip;
        }
        if (g == 0) sts128(s0 + piece_at(r, i), w[0], w[1], w[2], w[3]);
      }
      if (flip) qs = -qs;
      if (g == 0) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull);
      }
    }
    float ref = -INFINITY, ve = F::kPlain ? 0.f : pfx::kLowestE;
    float2 l2 = make_float2(0.f, 0.f), w2 = make_float2(0.f, 0.f);
    bool ok = true;
    for (int t = g; t < nt && ok; t += 2) {
      ok = mbar_wait(sfull + g, (t >> 1) & 1, ERR_PFX_WAIT);
      if (!F::kPlain && ok) ok = mbar_wait(vfull + t % kVRing, (t / kVRing) & 1, ERR_PFX_WAIT);  // its parameters
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      mm4::tc_fence_after();
      const uint32_t par = s0 + F::kOffPar + (t % kVRing) * F::kPar;
      const int left = static_cast<int>(min(n - static_cast<int64_t>(t0 + t) * kTile, int64_t(kTile)));
      if (busy) {
        // 32 columns of the row's scores from column c0: scaled by the keys' scales, -inf beyond the prefix
        auto scores = [&](int c0, float2 (&x)[16]) {
          float f[32];
          tmem_ld32(ts + c0, f);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = make_float2(f[2 * i], f[2 * i + 1]);
          if constexpr (!F::kPlain) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 s = lds128f(par + (c0 + 4 * i) * 4);
              if constexpr (F::kFmt == RB_KV_INT4) {
                const float4 m = lds128f(par + (2 * kTile + c0 + 4 * i) * 4);
                const float2 q2 = make_float2(qs, qs);
                x[2 * i] = fma2(x[2 * i], make_float2(s.x, s.y), mul2(make_float2(m.x, m.y), q2));
                x[2 * i + 1] = fma2(x[2 * i + 1], make_float2(s.z, s.w), mul2(make_float2(m.z, m.w), q2));
              } else {
                x[2 * i] = mul2(x[2 * i], make_float2(s.x, s.y));
                x[2 * i + 1] = mul2(x[2 * i + 1], make_float2(s.z, s.w));
              }
            }
          }
          if (c0 + 32 > left) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (c0 + 2 * i >= left) x[i].x = -INFINITY;
              if (c0 + 2 * i + 1 >= left) x[i].y = -INFINITY;
            }
          }
        };
        float top = -INFINITY;
#pragma unroll 1
        for (int c0 = 0; c0 < kTile; c0 += 32) {
          float2 x[16];
          scores(c0, x);
#pragma unroll
          for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(x[i].x, x[i].y));
        }
        float ven = ve;
        if constexpr (!F::kPlain) {
          const float4 s = lds128f(par + (kTile + 4 * lane) * 4);
          auto bits = [](float f) { return f == f ? __float_as_uint(f) : 0u; };  // a NaN shows by itself
          const uint32_t hi = __reduce_max_sync(0xffffffffu, max(max(bits(s.x), bits(s.y)), max(bits(s.z), bits(s.w))));
          ven = fmaxf(ve, fminf(fmaxf(static_cast<float>(static_cast<int>(hi >> 23) - 127), pfx::kLowestE), pfx::kHighestE));
        }
        if (__any_sync(0xffffffffu, top * fr > ref + pfx::kSlack || ven > ve)) {
          const float nr = fmaxf(ref, top * fr);
          const float f = ref == -INFINITY ? 0.f : ex2((ref - nr) + (ve - ven));
          ref = nr;
          ve = ven;
          l2 = mul2(l2, make_float2(f, f));
          w2 = mul2(w2, make_float2(f, f));
          if (t >= 2) {  // the group's O holds something: all of it is there, and the next PV waits for this tile's P
            ok = __all_sync(0xffffffffu, mbar_wait(pvdone + g, ((t >> 1) - 1) & 1, ERR_PFX_WAIT));
            mm4::tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < F::kHd && ok; c0 += 16) {
              uint32_t v[16];
              asm volatile(
                  "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
                  "[%16];\n\ttcgen05.wait::ld.sync.aligned;"
                  : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                    "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                  : "r"(to + c0)
                  : "memory");
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
              tmem_st16(to + c0, v);
            }
          }
        }
        const float base = ref == -INFINITY ? 0.f : -(ref + ve);
        const float2 f2 = make_float2(fr, fr), b2 = make_float2(base, base);
#pragma unroll 1
        for (int c0 = 0; c0 < kTile && ok; c0 += 32) {
          float2 x[16];
          scores(c0, x);
          uint32_t hi[16], lo[F::kFmt == RB_KV_INT4 ? 16 : 1];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 pr = fma2(x[i], f2, b2);
            pr.x = ex2(pr.x);
            pr.y = ex2(pr.y);
            l2 = add2(l2, pr);
            x[i] = pr;
          }
          if constexpr (!F::kPlain) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 s = lds128f(par + (kTile + c0 + 4 * i) * 4);
              if constexpr (F::kFmt == RB_KV_INT4) {
                const float4 m = lds128f(par + (3 * kTile + c0 + 4 * i) * 4);
                w2 = fma2(x[2 * i], make_float2(m.x, m.y), w2);
                w2 = fma2(x[2 * i + 1], make_float2(m.z, m.w), w2);
              }
              x[2 * i] = mul2(x[2 * i], make_float2(s.x, s.y));
              x[2 * i + 1] = mul2(x[2 * i + 1], make_float2(s.z, s.w));
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            hi[i] = pfx::pack2<F::kBf16>(x[i].x, x[i].y);
            if constexpr (F::kFmt == RB_KV_INT4) {  // what the rounding of p s left, as a second term
              const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
              lo[i] = pfx::pack2<false>(x[i].x - h.x, x[i].y - h.y);
            }
          }
          tmem_st16(ts + c0, hi);
          if constexpr (F::kFmt == RB_KV_INT4) tmem_st16(ts + c0 + 16, lo);
        }
        tmem_wait_st();
      }
      if (!ok) break;
      mm4::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull + g);
    }
    // ---- the group's partial ----
    const int mine = nt > g ? (nt - g + 1) / 2 : 0;  // tiles of this group
    if (mine && ok) ok = __all_sync(0xffffffffu, mbar_wait(pvdone + g, (mine - 1) & 1, ERR_PFX_WAIT));
    mm4::tc_fence_after();
    const int64_t slot = (static_cast<int64_t>(lane_i) * p.max_np + sp) * 2 + g;
    const float l = l2.x + l2.y, w = w2.x + w2.y;
    if (on) p.rl[slot * kTile + r] = make_float2(!mine || (ref == -INFINITY && l == 0.f) ? -INFINITY : (ref == -INFINITY ? 0.f : ref + ve), l);
    if (mine && busy && ok) {
      float4* dst = reinterpret_cast<float4*>(p.o + (slot * kTile + r) * F::kHd);
#pragma unroll 1
      for (int c0 = 0; c0 < F::kHd; c0 += 32) {
        float f[32];
        tmem_ld32(to + c0, f);
        if (on) {
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[c0 / 4 + i] = make_float4(f[4 * i] + w, f[4 * i + 1] + w, f[4 * i + 2] + w, f[4 * i + 3] + w);
        }
      }
    }
    mm4::tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    mm4::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

}  // namespace pfxt

namespace pfx {

// Warps along the rows: the fewest whose 16-row tiles hold the batch's rows, at most four.
inline int warps_m(int64_t rows) { return rows <= 16 ? 1 : (rows <= 32 ? 2 : 4); }

// Which kernel streams the prefix, when the flags do not say.
inline bool use_tc(const rb_prefix_attn_args* a, int rep, int flags) {
  if (!a->prefix || (flags & RB_FLAG_KERNEL_MMA)) return false;
  if (flags & RB_FLAG_KERNEL_TC) return true;
  return a->n_seqs * rep > 32 && a->prefix->cache_len >= 2048;
}

struct Layout {
  int grid, wm, tile_rows, tiles_m, max_np, max_ns, parts;
  int64_t pre_slots, rl_bytes, total;
};
inline Layout layout_of(const rb_prefix_attn_args* a, int num_sms, bool tc) {
  const rb_kv_cache* c = a->prefix ? a->prefix : a->own;
  const int rep = a->n_q_heads / c->n_kv_heads;
  const int64_t rows = a->n_seqs * rep;
  Layout L = {};
  L.grid = kCtasPerSm * num_sms;
  L.wm = warps_m(rows);
  L.parts = tc ? 2 : 1;
  L.tile_rows = tc ? pfxt::kTile : 16 * L.wm;
  L.tiles_m = static_cast<int>((rows + L.tile_rows - 1) / L.tile_rows);
  const int64_t lanes = static_cast<int64_t>(c->n_kv_heads) * L.tiles_m, heads = a->n_seqs * c->n_kv_heads;
  // the warp-level kernel deals its items to kCtasPerSm CTAs an SM, the tcgen05 kernel has one CTA an item and SM
  L.max_np = a->prefix ? static_cast<int>(std::max<int64_t>(1, (tc ? num_sms : L.grid) / std::max<int64_t>(lanes, 1))) : 0;
  L.max_ns = a->own ? static_cast<int>(std::max<int64_t>(1, L.grid / std::max<int64_t>(heads, 1))) : 0;
  L.pre_slots = lanes * L.max_np * L.parts * L.tile_rows;
  const int64_t own_slots = heads * L.max_ns * rep;
  L.rl_bytes = ((L.pre_slots + own_slots) * 8 + 255) / 256 * 256;
  L.total = 256 + L.rl_bytes + (L.pre_slots + own_slots) * c->head_dim * 4;
  return L;
}

inline cudaLaunchConfig_t launch_config(int grid, int threads, int smem, int flags, cudaStream_t stream, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (flags & RB_FLAG_PDL) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

template <int kHd, int kFmt, bool kBf16>
int launch_format(const Params& p, const Layout& L, bool tc, int flags, cudaStream_t stream) {
  using F = Fmt<kHd, kFmt, kBf16>;
  using T = pfxt::Fmt<kHd, kFmt, kBf16>;
  constexpr int smem = Tile<F>::kSmem;
  static_assert((smem + 1024) * kCtasPerSm <= 227 * 1024, "CTAs an SM");
  static_assert(T::kSmem <= 227 * 1024, "the tcgen05 kernel's shared memory");
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg;
  Params rest = p;
  if (tc) {
    auto* kern = pfxt::prefix_attn_tc_kernel<T>;
    if (ensure_smem_limit(reinterpret_cast<const void*>(kern), T::kSmem) != cudaSuccess) return RB_ERR_LAUNCH;
    cfg = launch_config(p.n_kv * p.tiles_m * p.max_np, pfxt::kThreads, T::kSmem, flags, stream, attr);
    if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) return RB_ERR_LAUNCH;
    rest.pre.k = nullptr;  // only the own rows are left for the warp-level kernel
  }
  if (rest.pre.k || rest.own.k) {
    if (ensure_smem_limit(reinterpret_cast<const void*>(prefix_attn_kernel<F>), smem) != cudaSuccess) return RB_ERR_LAUNCH;
    cfg = launch_config(L.grid, kThreads, smem, flags, stream, attr);
    if (cudaLaunchKernelEx(&cfg, prefix_attn_kernel<F>, rest) != cudaSuccess) return RB_ERR_LAUNCH;
  }
  cfg = launch_config(p.n_seqs * p.n_q, kThreads, 0, flags, stream, attr);
  return cudaLaunchKernelEx(&cfg, prefix_attn_merge<kHd>, p, L.tile_rows, F::kTile) == cudaSuccess ? RB_OK : RB_ERR_LAUNCH;
}

}  // namespace pfx

int64_t prefix_attn_workspace(const rb_prefix_attn_args* a, int num_sms) {
  // enough for either kernel: a call's flags may name the other one
  return std::max(pfx::layout_of(a, num_sms, false).total, a->prefix ? pfx::layout_of(a, num_sms, true).total : 0);
}

int launch_prefix_attn(const rb_prefix_attn_args* a, int num_sms, int flags, cudaStream_t stream) {
  using namespace pfx;
  const rb_kv_cache* c = a->prefix ? a->prefix : a->own;
  Params p = {};
  p.q = a->q;
  p.out = a->out;
  p.ldq = a->ldq;
  p.ldo = a->ldo;
  auto side = [](const rb_kv_cache* s, const int64_t* len) {
    return Side{static_cast<const uint8_t*>(s->k), static_cast<const uint8_t*>(s->v), s->k_par, s->v_par, len, s->cache_len};
  };
  if (a->prefix && a->prefix->cache_len) p.pre = side(a->prefix, a->prefix_len);
  if (a->own && a->own->cache_len) p.own = side(a->own, a->own_len);
  p.n_seqs = static_cast<int>(a->n_seqs);
  p.n_q = a->n_q_heads;
  p.n_kv = c->n_kv_heads;
  p.rep = p.n_q / p.n_kv;
  const bool tc = p.pre.k && use_tc(a, p.rep, flags);
  const Layout L = layout_of(a, num_sms, tc);
  p.bf16 = c->dtype == RB_BF16;
  p.scale = a->scale;
  p.wm = L.wm;
  p.tiles_m = L.tiles_m;
  p.max_np = L.max_np;
  p.max_ns = L.max_ns;
  p.parts = L.parts;
  uint8_t* w = static_cast<uint8_t*>(a->ws);
  p.plan = reinterpret_cast<int*>(w);
  p.rl = reinterpret_cast<float2*>(w + 256);
  p.o = reinterpret_cast<float*>(w + 256 + L.rl_bytes);
  p.own_rl = L.pre_slots;
  p.own_o = L.pre_slots * c->head_dim;
  const bool wide = c->head_dim == 128;
  switch (c->fmt) {
    case RB_KV_INT8:
      return wide ? launch_format<128, RB_KV_INT8, false>(p, L, tc, flags, stream) : launch_format<64, RB_KV_INT8, false>(p, L, tc, flags, stream);
    case RB_KV_INT4:
      return wide ? launch_format<128, RB_KV_INT4, false>(p, L, tc, flags, stream) : launch_format<64, RB_KV_INT4, false>(p, L, tc, flags, stream);
    default:
      if (p.bf16)
        return wide ? launch_format<128, RB_KV_PLAIN, true>(p, L, tc, flags, stream) : launch_format<64, RB_KV_PLAIN, true>(p, L, tc, flags, stream);
      return wide ? launch_format<128, RB_KV_PLAIN, false>(p, L, tc, flags, stream) : launch_format<64, RB_KV_PLAIN, false>(p, L, tc, flags, stream);
  }
}

}  // namespace rb
