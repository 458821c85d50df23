// prefix_attn_tc.cu - the shared prefix's part of rb_prefix_attn on the tcgen05 tensor cores, for batches with more query
// rows per key-value head than the warp-level kernel (prefix_attn.cu) streams at HBM rate. The mathematics, the formats'
// rules and the partials are those of prefix_attn.cu.
//
// One CTA takes 128 query rows of one key-value head and a split of the prefix, in tiles of 128 slots. M = 128 rows:
//   S = Q K^T    Q and K in shared memory (K-major, 128-byte swizzle), S in tensor memory
//   O += P V     P in tensor memory as 16-bit values over the columns of S it came from, V in shared memory as its rows
//                lie (MN-major), O in tensor memory
// Two groups of four softmax warps take the tiles in turn, each with its own S, its own O and its own references: 4 x 128
// columns fill the tensor memory, and a group only waits for the tensor core. They leave two partials. A warp reads its
// 32 lanes of S as 16 x 256-bit fragments: a thread then holds every fourth pair of columns of four rows, and needs a
// quarter of the tile's scales - delivering all of them to every thread took longer than the exponentials. Rows lie on
// lanes 32 (r % 4) + r / 4, so that a batch of up to 64 rows uses half of each warp's lanes, not two of the four warps.
// A group's first warp issues its MMAs, PV(t) and then QK(t + 2): MMAs of one thread complete in order, so QK(t + 2) may
// overwrite the columns that PV(t) reads. Four warps fill a ring of key tiles and four a ring of value tiles: 16-bit rows
// by asynchronous copies, two tiles ahead; codes through registers, converted to 16-bit integers on the way, the next
// tile's already in flight. (One warp for all MMAs made 17 warps, which leaves 96 registers a thread and spills; four
// loader warps for both rings paced the whole kernel at 4,100 cycles a tile.)
//
// Bound: 16-bit rows by HBM in the loop over the tiles (64 KB in 2,950 cycles on every SM: 6.1 TB/s), beside 10 us of start
// and merge (32,768 slots of 8 heads with 48 rows: 46 us). 8-bit codes of up to 64 rows by the loaders, 2,100 cycles a tile of keys or values: conversion, the
// proxy fence and the loads' latency in turn. More rows by a group's chain of QK, softmax and PV, 6,000 cycles for each of
// two tiles under way, with codes somewhat more (100,001 slots of 4 heads with 256 rows, int8: 121 us, 105 without the own
// rows, 500 TFLOP/s; 6 of them for the largest t + e of the rows slot by slot, which the largest t and e apart would save).
#include "common.cuh"
#include "tc.cuh"
#include "kernels.h"

namespace rb {

namespace pfxt {

using pfx::ex2;
using pfx::Params;

constexpr int kTile = 128;        // slots of a tile, and query rows of a CTA
constexpr int kFirstK = 8, kFirstV = 12;  // warps 0 .. 7: two softmax groups; 8 .. 11 and 12 .. 15: loaders
constexpr int kLoadWarps = 4;
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int kThreads = 512;
// Registers by warpgroup, and the tiles of codes that a loader holds ahead. kH 16-lane halves of a warp hold rows: the
// softmax warps keep a tile's scores, 64 kH a thread; what they leave goes to the loaders.
template <int kFmt, int kH>
struct Regs {
  static constexpr int kSoft = kH == 1 ? 144 : (kFmt == RB_KV_INT4 ? 200 : 192), kLoad = 256 - kSoft, kAhead = kH == 1 ? 2 : 1;
  static_assert(2 * kSoft + 2 * kLoad <= 4 * (65536 / kThreads), "the launch's registers");
};
constexpr int kVRing = 3, kKParRing = 4;
constexpr uint32_t kTmemCols = 512;

template <int kHd_, int kFmt_, bool kBf16_>
struct Fmt {
  static constexpr int kHd = kHd_, kFmt = kFmt_;
  static constexpr bool kBf16 = kBf16_, kPlain = kFmt == RB_KV_PLAIN;
  static constexpr int kRow = kPlain ? 2 * kHd : (kFmt == RB_KV_INT8 ? kHd : kHd / 2);
  static constexpr int kAtom = kTile * 128;              // 64 columns of 128 rows
  static constexpr int kTileBytes = kTile * kHd * 2;     // a tile of 16-bit values
  static constexpr int kKRing = kPlain ? 3 : 2;          // copies two tiles ahead need three
  // fp32 s and m of a tile's keys (values), in the order in which the fragments need them: slot 8 u + 2 c + e at
  // c kParC + 2 u + e, so that a lane reads its columns in sixteen-byte pieces and the four c fall on different banks
  static constexpr int kParC = kTile / 4 + 4, kParN = 4 * kParC;
  static constexpr int kPar = kPlain ? 0 : kParN * 4 * 2, kVPar = kPlain ? 0 : kParN * 4 * 3;  // of the values e, too
  static constexpr int kOffK = kTileBytes, kOffV = kOffK + kKRing * kTileBytes, kOffPar = kOffV + kVRing * kTileBytes;
  static constexpr int kOffVPar = kOffPar + kKParRing * kPar;
  static constexpr int kOffRow = kOffVPar + kVRing * kVPar;  // factor and sum of the rows' queries
  static constexpr int kOffBar = kOffRow + kTile * 8;
  static constexpr int kBars = 2 * kKRing + 2 * kVRing + 3 * 2;
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

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ float4 lds128f(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}

// One lane of a converged warp; the compiler keeps what is computed for it in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on != 0;
}

// Byte offset of the 16-byte piece `ch` (eight 16-bit columns) of row r in a swizzled tile.
__device__ __forceinline__ uint32_t piece_at(int r, int ch) { return (ch >> 3) * (kTile * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4); }

constexpr int kBarSoft = 1, kBarGroup = 2;  // named barriers: all softmax warps; a group (2, 3)

// 16 lanes x 128 columns as fragments: x[4 u + e] is column 8 u + 2 c + (e & 1) of lane l + 8 (e >> 1), with l = lane / 4 and
// c = lane % 4. Valid after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld_frag(uint32_t a, float (&x)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
      : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15]), "=f"(x[16]), "=f"(x[17]), "=f"(x[18]), "=f"(x[19]), "=f"(x[20]), "=f"(x[21]), "=f"(x[22]), "=f"(x[23]), "=f"(x[24]), "=f"(x[25]), "=f"(x[26]), "=f"(x[27]), "=f"(x[28]), "=f"(x[29]), "=f"(x[30]), "=f"(x[31]), "=f"(x[32]), "=f"(x[33]), "=f"(x[34]), "=f"(x[35]), "=f"(x[36]), "=f"(x[37]), "=f"(x[38]), "=f"(x[39]), "=f"(x[40]), "=f"(x[41]), "=f"(x[42]), "=f"(x[43]), "=f"(x[44]), "=f"(x[45]), "=f"(x[46]), "=f"(x[47]), "=f"(x[48]), "=f"(x[49]), "=f"(x[50]), "=f"(x[51]), "=f"(x[52]), "=f"(x[53]), "=f"(x[54]), "=f"(x[55]), "=f"(x[56]), "=f"(x[57]), "=f"(x[58]), "=f"(x[59]), "=f"(x[60]), "=f"(x[61]), "=f"(x[62]), "=f"(x[63])
      : "r"(a));
}
// The same of 16 columns.
__device__ __forceinline__ void tmem_ld_frag16(uint32_t a, float (&x)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
               : "r"(a));
}
__device__ __forceinline__ void tmem_st_frag16(uint32_t a, const float (&x)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(a), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}
// 16 lanes x 16 columns of packed pairs: v[2 i + h] is column 4 i + c of lane l + 8 h.
__device__ __forceinline__ void tmem_st_pairs(uint32_t a, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_wait_ld(float (&x)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(x[i]));
}

// The softmax warps' work on the CTA's tiles. kH: 16-lane halves of a warp that hold rows of the batch.
template <typename F, int kH>
__device__ __forceinline__ void run_softmax(const Params& p, uint32_t s0, uint8_t* smem, uint32_t tmem, int g, int quad, int lane, int nt,
                                            int64_t n, int rows, int64_t split) {
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + F::kOffBar);
  uint64_t* kempty = kfull + F::kKRing;
  uint64_t* vfull = kempty + F::kKRing;
  uint64_t* vempty = vfull + kVRing;
  uint64_t* sfull = vempty + kVRing + g;
  uint64_t* pvdone = sfull + 2;
  uint64_t* ended = pvdone + 2;
  const float* rowf = reinterpret_cast<const float*>(smem + F::kOffRow);
  const int l0 = lane >> 2, c = lane & 3;
  const uint32_t tq = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  const uint32_t ts = tq + g * kTile, to = tq + (2 + g) * kTile, half = 16u << 16;  // the second half's lanes
  const bool busy = quad < rows;
  float fr[2 * kH], qs[2 * kH], ref[2 * kH];  // row y of the thread: lane 16 (y / 2) + 8 (y % 2) + l0
  float l[2 * kH], w[2 * kH];
#pragma unroll
  for (int y = 0; y < 2 * kH; ++y) {
    const int at = quad * 32 + 8 * y + l0;
    fr[y] = rowf[at];
    qs[y] = F::kFmt == RB_KV_INT4 ? rowf[kTile + at] : 0.f;
    ref[y] = -INFINITY;
    l[y] = w[y] = 0.f;
  }
  bool ok = true;
  // The group's first warp: S = Q K^T of tile t, once its keys are there.
  auto issue_qk = [&](int t) {
    const int ks = t % F::kKRing;
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(kfull + ks, (t / F::kKRing) & 1, ERR_PFX_WAIT));
    mm4::tc_fence_after();
    if (ok && elect_one()) {
      const uint64_t qd = mm4::sw128_desc(s0), kd = mm4::sw128_desc(s0 + F::kOffK + ks * F::kTileBytes);
#pragma unroll
      for (int i = 0; i < F::kHd / 16; ++i) {
        const uint32_t at = ((i >> 2) * F::kAtom + (i & 3) * 32) >> 4;
        umma_ss(tmem + g * kTile, qd + at, kd + at, F::kIdescQk, i != 0);
      }
      mm4::umma_commit(sfull);
      mm4::umma_commit(kempty + ks);
    }
    __syncwarp();
  };
  if (quad == 0 && g < nt) issue_qk(g);
  // Every warp goes through every tile, also after a wait that ran out, so that the group's barrier is complete.
#pragma unroll 1
  for (int t = g; t < nt; t += 2) {
    if (ok) ok = mbar_wait(sfull, (t >> 1) & 1, ERR_PFX_WAIT);
    if (ok) ok = mbar_wait(vfull + t % kVRing, (t / kVRing) & 1, ERR_PFX_WAIT);  // its parameters; the PV below needs them
    ok = __all_sync(0xffffffffu, ok);
    mm4::tc_fence_after();
    if (busy && ok) {
      const uint32_t kpar = s0 + F::kOffPar + (t % kKParRing) * F::kPar + c * (F::kParC * 4);
      const uint32_t vpar = s0 + F::kOffVPar + (t % kVRing) * F::kVPar + c * (F::kParC * 4);
      // A lane's row parameters of the columns 8 u + 2 c, two u at a time, loaded kAhead steps before they are used: a load
      // from shared memory takes long while the tensor core reads its operands there.
      constexpr int kAhead = F::kFmt == RB_KV_INT4 ? 1 : 2;
      float4 ps[kAhead], pm[F::kFmt == RB_KV_INT4 ? kAhead : 1], pe;
      auto ahead = [&](uint32_t base, int i) {
        if constexpr (!F::kPlain) {
          ps[i % kAhead] = lds128f(base + 16 * i);
          if constexpr (F::kFmt == RB_KV_INT4) pm[i % kAhead] = lds128f(base + F::kParN * 4 + 16 * i);
        }
      };
      auto ahead_e = [&](int i) {
        if constexpr (!F::kPlain) pe = lds128f(vpar + 2 * F::kParN * 4 + 16 * i);
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ahead(kpar, i);
      ahead_e(0);
      const int left = static_cast<int>(min(n - static_cast<int64_t>(t) * kTile, int64_t(kTile)));
      // the rows' scores, scaled by the keys' scales, -inf beyond the prefix; and the largest score plus exponent of the
      // value's scale (-inf beyond the prefix), in log2 units
      float top[2 * kH];
#pragma unroll
      for (int y = 0; y < 2 * kH; ++y) top[y] = -INFINITY;
      float x[kH][64];
#pragma unroll
      for (int h = 0; h < kH; ++h) tmem_ld_frag(ts + h * half, x[h]);
#pragma unroll
      for (int h = 0; h < kH; ++h) tmem_wait_ld(x[h]);
      if constexpr (!F::kPlain) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 k4 = ps[i % kAhead], m4 = F::kFmt == RB_KV_INT4 ? pm[i % (F::kFmt == RB_KV_INT4 ? kAhead : 1)] : k4, e4 = pe;
          if (i + kAhead < 8) ahead(kpar, i + kAhead);
          if (i < 7) ahead_e(i + 1);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int u = 2 * i + q;
            const float2 ks = q ? make_float2(k4.z, k4.w) : make_float2(k4.x, k4.y), km = q ? make_float2(m4.z, m4.w) : make_float2(m4.x, m4.y);
            const float2 ev = q ? make_float2(e4.z, e4.w) : make_float2(e4.x, e4.y);
#pragma unroll
            for (int y = 0; y < 2 * kH; ++y) {
              float& a = x[y >> 1][4 * u + 2 * (y & 1)];
              float& b = x[y >> 1][4 * u + 2 * (y & 1) + 1];
              float2 v = make_float2(a, b);
              if constexpr (F::kFmt == RB_KV_INT8) v = mul2(v, ks);
              else v = fma2(v, ks, mul2(km, make_float2(qs[y], qs[y])));
              a = v.x, b = v.y;
              v = fma2(v, make_float2(fr[y], fr[y]), ev);
              top[y] = fmaxf(top[y], fmaxf(v.x, v.y));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ahead(vpar, i);
      }
      if (left < kTile) {
#pragma unroll
        for (int h = 0; h < kH; ++h)
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (8 * (i >> 2) + 2 * c + (i & 1) >= left) x[h][i] = -INFINITY;
      }
      bool raise = false;
#pragma unroll
      for (int y = 0; y < 2 * kH; ++y) {
        if constexpr (F::kPlain) {
#pragma unroll
          for (int u = 0; u < 16; ++u) top[y] = fmaxf(top[y], fmaxf(x[y >> 1][4 * u + 2 * (y & 1)], x[y >> 1][4 * u + 2 * (y & 1) + 1]));
          top[y] *= fr[y];
        }
        raise |= top[y] > ref[y] + (pfx::kRoom + pfx::kSlack);
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int y = 0; y < 2 * kH; ++y) {
          float v = top[y];
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
          const float nr = fmaxf(ref[y], v - pfx::kRoom), d = ref[y] == -INFINITY ? -INFINITY : ref[y] - nr;
          top[y] = ex2(d);  // O's factor from here on
          ref[y] = nr;
          l[y] = pfx::lowered(l[y], d);
          w[y] = pfx::lowered(w[y], d);
        }
        if (t >= 2) {  // the group's O holds something: all of it is there, and the next PV waits for this tile's P
          ok = __all_sync(0xffffffffu, mbar_wait(pvdone, ((t >> 1) - 1) & 1, ERR_PFX_WAIT));
          mm4::tc_fence_after();
#pragma unroll 1
          for (int c0 = 0; c0 < F::kHd && ok; c0 += 16) {
#pragma unroll
            for (int h = 0; h < kH; ++h) {
              float v[8];
              tmem_ld_frag16(to + h * half + c0, v);
              tmem_wait_ld(v);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] *= top[2 * h + ((i >> 1) & 1)];
              tmem_st_frag16(to + h * half + c0, v);
            }
          }
        }
      }
      // P = 2^(t - R), over the columns that S came from
      float base[2 * kH];
#pragma unroll
      for (int y = 0; y < 2 * kH; ++y) base[y] = ref[y] == -INFINITY ? 0.f : -ref[y];
#pragma unroll
      for (int u0 = 0; u0 < 16; u0 += 4) {  // 32 columns: sixteen of packed pairs, and sixteen for their remainders
        uint32_t hi[kH][8], lo[F::kFmt == RB_KV_INT4 ? kH : 1][8];
#pragma unroll
        for (int u = u0; u < u0 + 4; ++u) {
          float2 vs = make_float2(1.f, 1.f), vm = make_float2(0.f, 0.f);
          if constexpr (!F::kPlain) {
            const int i = u >> 1;
            const float4 s4 = ps[i % kAhead];
            vs = (u & 1) ? make_float2(s4.z, s4.w) : make_float2(s4.x, s4.y);
            if constexpr (F::kFmt == RB_KV_INT4) {
              const float4 m4 = pm[i % kAhead];
              vm = (u & 1) ? make_float2(m4.z, m4.w) : make_float2(m4.x, m4.y);
            }
            if ((u & 1) && i + kAhead < 8) ahead(vpar, i + kAhead);
          }
#pragma unroll
          for (int y = 0; y < 2 * kH; ++y) {
            float2 v = make_float2(x[y >> 1][4 * u + 2 * (y & 1)], x[y >> 1][4 * u + 2 * (y & 1) + 1]);
            v = fma2(v, make_float2(fr[y], fr[y]), make_float2(base[y], base[y]));
            v.x = ex2(v.x);
            v.y = ex2(v.y);
            l[y] += v.x + v.y;
            if constexpr (F::kFmt == RB_KV_INT4) w[y] = fmaf(v.x, vm.x, fmaf(v.y, vm.y, w[y]));
            if constexpr (!F::kPlain) v = mul2(v, vs);
            uint32_t& out = hi[y >> 1][2 * (u - u0) + (y & 1)];
            out = pfx::pack2<F::kBf16>(v.x, v.y);
            if constexpr (F::kFmt == RB_KV_INT4) {  // what the rounding of p s left, as a second term
              const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&out));
              lo[y >> 1][2 * (u - u0) + (y & 1)] = pfx::pack2<false>(v.x - r.x, v.y - r.y);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < kH; ++h) {
          tmem_st_pairs(ts + h * half + 8 * u0, hi[h]);
          if constexpr (F::kFmt == RB_KV_INT4) tmem_st_pairs(ts + h * half + 8 * u0 + 16, lo[h]);
        }
      }
      tmem_wait_st();
    }
    mm4::tc_fence_before();
    named_bar_sync(kBarGroup + g, 128);  // the group's P is complete
    if (quad == 0) {
      mm4::tc_fence_after();
      const int vs = t % kVRing;
      if (ok && elect_one()) {
        const uint64_t vd = v_desc(s0 + F::kOffV + vs * F::kTileBytes, F::kAtom);
        const uint32_t s = tmem + g * kTile, o = tmem + (2 + g) * kTile;
#pragma unroll
        for (int i = 0; i < kTile / 16; ++i)
          umma_ts(o, s + 32 * (i >> 1) + 8 * (i & 1), vd + i * (2048 >> 4), F::kIdescPv, t >= 2 || i != 0);
        if constexpr (F::kFmt == RB_KV_INT4) {
#pragma unroll
          for (int i = 0; i < kTile / 16; ++i)
            umma_ts(o, s + 32 * (i >> 1) + 16 + 8 * (i & 1), vd + i * (2048 >> 4), F::kIdescPv, 1);
        }
        mm4::umma_commit(vempty + vs);
        mm4::umma_commit(pvdone);
      }
      __syncwarp();
      if (t + 2 < nt) issue_qk(t + 2);
    }
  }
  // ---- the group's partial ----
  const int mine = nt > g ? (nt - g + 1) / 2 : 0;  // tiles of this group
  if (mine && ok) ok = __all_sync(0xffffffffu, mbar_wait(pvdone, (mine - 1) & 1, ERR_PFX_WAIT));
  if (!ok && quad == 0) {
    // A wait ran out, whatever the limit in force: the products that this warp has issued still end before their shared and
    // tensor memory is given back. One more commit tells when; they wait for nothing, and the bound is the longest limit.
    if (elect_one()) mm4::umma_commit(ended);
    __syncwarp();
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_wait(ended, 0) && globaltimer_ns() - t0 < kMaxWaitNs) {
    }
  }
  mm4::tc_fence_after();
  const int64_t first = (split * 2 + g) * kTile;
#pragma unroll
  for (int y = 0; y < 2 * kH; ++y) {
    l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
    l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
    w[y] += __shfl_xor_sync(0xffffffffu, w[y], 1);
    w[y] += __shfl_xor_sync(0xffffffffu, w[y], 2);
    const int r = (8 * y + l0) * 4 + quad;
    if (c == 0 && r < rows)
      p.rl[first + r] = make_float2(!mine || (ref[y] == -INFINITY && l[y] == 0.f) ? -INFINITY : (ref[y] == -INFINITY ? 0.f : ref[y]), l[y]);
  }
  if (mine && busy && ok) {
#pragma unroll 2
    for (int c0 = 0; c0 < F::kHd; c0 += 16) {
#pragma unroll
      for (int h = 0; h < kH; ++h) {
        float v[8];
        tmem_ld_frag16(to + h * half + c0, v);
        tmem_wait_ld(v);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int y = 2 * h + ((i >> 1) & 1), r = (8 * y + l0) * 4 + quad;
          if (r < rows)
            *reinterpret_cast<float2*>(p.o + (first + r) * F::kHd + c0 + 8 * (i >> 2) + 2 * c) = make_float2(v[i] + w[y], v[i + 1] + w[y]);
        }
      }
    }
  }
  mm4::tc_fence_before();
}

template <typename F, int kH>
__global__ void __launch_bounds__(kThreads, 1) prefix_attn_tc_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s0 = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + F::kOffBar);
  uint64_t* kempty = kfull + F::kKRing;
  uint64_t* vfull = kempty + F::kKRing;
  uint64_t* vempty = vfull + kVRing;
  uint64_t* sfull = vempty + kVRing;  // [2] S of the group's tile is there
  uint64_t* pvdone = sfull + 2;       // [2] the group's last PV is complete
  uint64_t* ended = pvdone + 2;       // [2] all that the group issued is complete: waited for where another wait ran out
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ended + 2);

  griddep_wait();
  griddep_launch_dependents();
  const int64_t n = __ldcg(p.pre.len);
  const int lane_i = blockIdx.x / p.max_np, sp = blockIdx.x % p.max_np;
  const int kv = lane_i / p.tiles_m, row0 = (lane_i % p.tiles_m) * kTile;
  if (n < 0 || n > p.pre.cache_len) {
    if (blockIdx.x == 0 && tid == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
    return;
  }
  const int tiles = static_cast<int>((n + kTile - 1) / kTile);
  const int per = pfx::tiles_of_split(tiles, p.max_np);
  const int t0 = sp * per, t1 = min(tiles, t0 + per), nt = t1 - t0;
  if (nt <= 0) return;  // the merge knows which splits there are

  if (tid == 0) {
    for (int i = 0; i < F::kKRing; ++i) {
      mbar_init(kfull + i, kLoadWarps);
      mbar_init(kempty + i, 1);
    }
    for (int i = 0; i < kVRing; ++i) {
      mbar_init(vfull + i, kLoadWarps);
      mbar_init(vempty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull + i, 1);
      mbar_init(pvdone + i, 1);
      mbar_init(ended + i, 1);
    }
    fence_mbar_init();
  }
  if (warp == kFirstK) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  mm4::tc_fence_before();
  __syncthreads();
  mm4::tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // S of group 0, S of group 1, O of group 0, O of group 1: 128 columns each
  const int64_t head = static_cast<int64_t>(kv) * p.pre.cache_len;  // the head's first row

  if (warp >= kFirstK) {
    // ---------------- loaders: four warps of keys, four of values ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<F::kFmt, kH>::kLoad));
    const bool keys = warp < kFirstV;
    const int lw = warp - (keys ? kFirstK : kFirstV), lt = lw * 32 + lane;
    const int ring = keys ? F::kKRing : kVRing;
    uint64_t* full = keys ? kfull : vfull;
    uint64_t* empty = keys ? kempty : vempty;
    const uint8_t* src = (keys ? p.pre.k : p.pre.v) + head * F::kRow;
    const uint32_t base = s0 + (keys ? F::kOffK : F::kOffV);
    bool ok = true;
    auto arrive = [&](int slot) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + slot);
    };
    int slot = 0, phase = 1;  // of the tile to fill: its slot, and the parity of the release that it waits for
    auto free_slot = [&](int t) {
      if (t >= ring && ok) ok = mbar_wait(empty + slot, phase, ERR_PFX_WAIT);
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    auto next_slot = [&] {
      if (++slot == ring) slot = 0, phase ^= 1;
    };
    if constexpr (F::kPlain) {
      constexpr int kPieces = F::kRow / 16, kEach = kTile * kPieces / kLoadThreads;
      int landed = 0;  // slot of the tile to release
      for (int t = 0; t < nt + 2; ++t) {
        if (t < nt) {
          if (!free_slot(t)) break;
          const int64_t first = static_cast<int64_t>(t0 + t) * kTile;
          const uint32_t dst = base + slot * F::kTileBytes;
          const uint8_t* from = src + first * F::kRow + lt * 16;
          if (first + kTile <= n) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
              const int x = i * kLoadThreads + lt;
              pfx::cp_async16(dst + piece_at(x / kPieces, x % kPieces), from + i * kLoadThreads * 16, true);
            }
          } else {
#pragma unroll 1
            for (int i = 0; i < kEach; ++i) {
              const int x = i * kLoadThreads + lt;
              const bool on = first + x / kPieces < n;
              pfx::cp_async16(dst + piece_at(x / kPieces, x % kPieces), on ? from + i * kLoadThreads * 16 : src, on);
            }
          }
          next_slot();
        }
        pfx::cp_commit();
        if (t > 1) {  // two tiles may still be under way: tile t - 2 has landed
          pfx::cp_wait<2>();
          arrive(landed);
          landed = landed + 1 == ring ? 0 : landed + 1;
        }
      }
      pfx::cp_wait<0>();
    } else {
      constexpr int kPieces = F::kRow / 16;
      // A tile's pieces of sixteen bytes lie one after another and are dealt so: a warp's load is 512 bytes in a row, a
      // thread's pieces are the same columns, ch, of rows kStep apart, and the swizzle of their stores does not change.
      // Eight lanes that store together hold whole rows; where those span two atoms (128 columns), whose banks are the
      // same, the lanes of the second one store the halves of their piece in the other order: no two share a bank.
      constexpr int kStep = kLoadThreads / kPieces, kChunks = F::kFmt == RB_KV_INT8 ? 2 : 4;  // 16-byte chunks of values a piece
      static_assert(kStep % 8 == 0 && F::kRaw * kStep == kTile, "whole periods of the swizzle");
      const int lr = lt / kPieces, ch = lt % kPieces;
      const bool turn = kChunks * ch >= 8;
      uint32_t at_chunk[kChunks];  // offset of the chunk that is stored e-th, in a tile
#pragma unroll
      for (int e = 0; e < kChunks; ++e) at_chunk[e] = piece_at(lr, kChunks * ch + (turn ? e ^ (kChunks / 2) : e));
      constexpr int kParBytes = F::kFmt == RB_KV_INT8 ? 2 : 4;
      constexpr int kAhead = Regs<F::kFmt, kH>::kAhead;
      uint4 raws[kAhead][F::kRaw];
      uint32_t pars[kAhead];
      const uint8_t* from = src + static_cast<int64_t>(t0) * kTile * F::kRow + lt * 16;
      const uint8_t* par_from = static_cast<const uint8_t*>(keys ? p.pre.k_par : p.pre.v_par) + (head + static_cast<int64_t>(t0) * kTile + lt) * kParBytes;
      int seen = static_cast<int>(n - static_cast<int64_t>(t0) * kTile);  // slots from the tile to fetch on
      // Tile t (in order, none left out): piece i of a thread is of row lr + i kStep, its parameters' word of slot lt.
      auto fetch = [&](int t, uint4 (&raw)[F::kRaw], uint32_t& par) {
        if (t >= nt) return;
#pragma unroll
        for (int i = 0; i < F::kRaw; ++i) {
          raw[i] = make_uint4(0u, 0u, 0u, 0u);
          if (lr + i * kStep < seen) raw[i] = ldg_cg_128(from + i * kLoadThreads * 16);
        }
        par = 0u;
        if (lt < seen)
          par = F::kFmt == RB_KV_INT8 ? static_cast<uint32_t>(__ldcg(reinterpret_cast<const unsigned short*>(par_from)))
                                      : __ldcg(reinterpret_cast<const unsigned int*>(par_from));
        // registers hold less than is on the way from HBM: the tiles behind are called to L2 by the thread whose
        // addresses start a tile (each of them is loaded before the CTA ends). Line by line by all threads it took longer.
        constexpr int kFar = 4;
        if (t + kFar < nt && lt == 0) {
          const int rows = min(seen - kFar * kTile, kTile);
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from + kFar * kTile * F::kRow), "r"(rows * F::kRow) : "memory");
          const uint8_t* what = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(par_from + kFar * kTile * kParBytes) & ~uintptr_t(15));
          if (rows * kParBytes >= 16) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(what), "r"(rows * kParBytes & ~15) : "memory");
        }
        from += kTile * F::kRow;
        par_from += kTile * kParBytes;
        seen -= kTile;
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fetch(i, raws[i], pars[i]);
      auto convert = [&](int t, uint4 (&raw)[F::kRaw], uint32_t& par) {
        // The keys' parameters lie in a ring of four: tile t - 4's are free once QK(t - 2), which its group issued behind
        // PV(t - 4), has released the keys' slot.
        if (!free_slot(t)) return;
        const uint32_t dst = base + slot * F::kTileBytes;
#pragma unroll
        for (int i = 0; i < F::kRaw; ++i) {
          uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          if (F::kHd == 128 && turn) w[0] = raw[i].z, w[1] = raw[i].w, w[2] = raw[i].x, w[3] = raw[i].y;
          const uint32_t to = dst + i * (kStep * 128);
          if constexpr (F::kFmt == RB_KV_INT8) {
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              h[2 * e] = mm4::hsub2_u(__byte_perm(w[e], 0x64646464u, 0x4140), 0x64806480u);  // 1024 + (c + 128) - 1152
              h[2 * e + 1] = mm4::hsub2_u(__byte_perm(w[e], 0x64646464u, 0x4342), 0x64806480u);
            }
            sts128(to + at_chunk[0], h[0], h[1], h[2], h[3]);
            sts128(to + at_chunk[1], h[4], h[5], h[6], h[7]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // a word: eight columns
              uint32_t h[4];
#pragma unroll
              for (int b = 0; b < 4; ++b)  // (1024 + low nibble, 64 + high nibble) - (1032, 72): c - 8
                h[b] = mm4::hsub2_u(and_or(__byte_perm(w[e], 0u, 0x4040u | (0x0101u * b)), 0x00F0000Fu, 0x54006400u), 0x54806408u);
              sts128(to + at_chunk[e], h[0], h[1], h[2], h[3]);
            }
          }
        }
        float* pd = reinterpret_cast<float*>(smem + (keys ? F::kOffPar + (t % kKParRing) * F::kPar : F::kOffVPar + slot * F::kVPar));
        const float s = __uint_as_float(par << 16);
        const int at = ((lt >> 1) & 3) * F::kParC + 2 * (lt >> 3) + (lt & 1);
        float mid = 0.f;
        pd[at] = s;
        if constexpr (F::kFmt == RB_KV_INT4) {
          mid = fmaf(8.f, s, p.bf16 ? __uint_as_float(par & 0xffff0000u) : __half2float(__ushort_as_half(static_cast<unsigned short>(par >> 16))));
          pd[F::kParN + at] = mid;
        }
        if (!keys) pd[2 * F::kParN + at] = lt < n - static_cast<int64_t>(t0 + t) * kTile ? pfx::value_exponent(s, mid) : -INFINITY;
        arrive(slot);
        next_slot();
        fetch(t + kAhead, raw, par);
      };
      for (int t = 0; t < nt && ok; t += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (t + i < nt && ok) convert(t + i, raws[i], pars[i]);
      }
    }
  } else {
    // ---------------- softmax: group g takes the tiles t % 2 == g ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs<F::kFmt, kH>::kSoft));
    const int g = warp >> 2, quad = warp & 3;
    const int rows = min(kTile, p.n_seqs * p.rep - row0);
    float* rowf = reinterpret_cast<float*>(smem + F::kOffRow);
    float* qsum = rowf + kTile;
    if (g == 0) {
      // group 0 brings the queries: thread = lane, its row's loads all at once
      const int r = lane * 4 + quad, lane_row = quad * 32 + lane, row = row0 + r;
      const bool on = r < rows;
      const int b = on ? row / p.rep : 0, j = on ? row % p.rep : 0;
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + b * p.ldq + static_cast<int64_t>(kv * p.rep + j) * F::kHd);
      uint4 q[F::kHd / 8];
#pragma unroll
      for (int i = 0; i < F::kHd / 8; ++i) q[i] = on ? ldg_cg_128(src + i) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
      float f = fabsf(p.scale) * pfx::kLog2e, sum = 0.f, down = 1.f;
      if constexpr (!F::kPlain) {
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < F::kHd / 8; ++i)
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(q[i].x & 0x7fff7fffu, q[i].y & 0x7fff7fffu), __vmaxu2(q[i].z & 0x7fff7fffu, q[i].w & 0x7fff7fffu)));
        const uint32_t t16 = max(top & 0xffffu, top >> 16);
        const uint32_t ex = __float_as_uint(p.bf16 ? __uint_as_float(t16 << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(t16)))) >> 23;
        const uint32_t exc = ex < 30u ? 30u : (ex > 220u ? 220u : ex);
        down = __uint_as_float((254u - exc) << 23);
        f *= __uint_as_float(exc << 23);
      }
#pragma unroll
      for (int i = 0; i < F::kHd / 8; ++i) {
        uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (!F::kPlain) {
            float2 v;
            if (p.bf16) v = make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
            else v = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
            w[e] = pfx::pack2<false>(v.x * down, v.y * down);
            if constexpr (F::kFmt == RB_KV_INT4) {
              v = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
              sum += v.x + v.y;
            }
          }
          w[e] ^= flip;
        }
        sts128(s0 + piece_at(lane_row, i), w[0], w[1], w[2], w[3]);
      }
      rowf[lane_row] = pfx::factor_in_range(f);
      qsum[lane_row] = flip ? -sum : sum;
      fence_proxy_async_smem();
    }
    named_bar_sync(kBarSoft, 256);
    run_softmax<F, kH>(p, s0, smem, tmem, g, quad, lane, nt, n - static_cast<int64_t>(t0) * kTile, rows, lane_i * p.max_np + sp);
  }
  __syncthreads();
  if (warp == kFirstK) {
    mm4::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

}  // namespace pfxt

namespace pfx {

// Warps along the rows: the fewest whose 16-row tiles hold the batch's rows, at most four.
inline int warps_m(int64_t rows) { return rows <= 16 ? 1 : (rows <= 32 ? 2 : 4); }

// Which kernel streams the prefix, when the flags do not say: by its capacity, the lengths being on the device. us of the
// warp-level kernel / the tcgen05 kernel, 20 own slots a sequence:
//   The tcgen05 kernel's start costs about what one to two thousand slots cost the other one (128 columns, 16 bits, 8 heads:
//   24 rows 1,100 slots 12.8 / 10.9, 10,000 21.6 / 18.4; 128 rows 18.2 / 17.7, 36.8 / 29.9; 64 columns, int8, 2 heads: 16 rows
//   1,100 slots 9.2 / 9.5, 10,000 23.0 / 12.6; 128 rows 2,100 slots 13.1 / 12.7, 10,000 17.9 / 15.7).
//   With one tile of 16 rows over rows of up to 128 bytes the warp-level kernel, which converts in registers what the
//   products read, keeps up as long as it has slots for all SMs: from some 98,304 of all heads together (64 columns, 4 rows of
//   8 heads, 40,000 slots: plain 19.9 / 26.7, int8 21.3 / 27.3, int4 25.4 / 35.7; 8 rows of 2 heads, 10,000: plain 21.1 / 11.7,
//   int8 19.2 / 12.6), and with 8-bit codes of 128 columns on the whole (8 rows: 2 heads 2,100 slots 9.7 / 11.0, 10,000 15.2 /
//   14.0; 8 heads 11.4 / 11.8, 14.7 / 20.4). Over 2,700 sizes of 1 to 16 heads, 1 to 128 rows and 600 to 40,000 slots this
//   choice takes 2.3 % longer than the better kernel each time would, 1.5 times as long at worst.
inline bool use_tc(const rb_prefix_attn_args* a, int rep, int flags) {
  if (!a->prefix || (flags & RB_FLAG_KERNEL_MMA)) return false;
  if (flags & RB_FLAG_KERNEL_TC) return true;
  const rb_kv_cache* c = a->prefix;
  const int64_t rows = a->n_seqs * rep;
  const bool int8 = c->fmt == RB_KV_INT8, wide = c->head_dim == 128;
  if (rows <= 16 && !(c->fmt == RB_KV_PLAIN && wide) && ((int8 && wide) || c->n_kv_heads * c->cache_len >= 98304)) return false;
  return c->cache_len >= (rows > 32 ? 1024 : 2048);
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
  L.grid = ctas_per_sm(c->fmt, c->head_dim) * num_sms;
  L.wm = warps_m(rows);
  L.parts = tc ? 2 : 1;
  L.tile_rows = tc ? pfxt::kTile : 16 * L.wm;
  L.tiles_m = static_cast<int>((rows + L.tile_rows - 1) / L.tile_rows);
  const int64_t lanes = static_cast<int64_t>(c->n_kv_heads) * L.tiles_m, heads = a->n_seqs * c->n_kv_heads;
  // the warp-level kernel deals its items to two or three CTAs an SM, the tcgen05 kernel has one CTA an item and SM
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
  static_assert((smem + 1024) * F::kCtas <= 227 * 1024, "CTAs an SM");
  static_assert(T::kSmem <= 227 * 1024, "the tcgen05 kernel's shared memory");
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg;
  Params rest = p;
  if (tc) {
    auto* kern = p.n_seqs * p.rep <= pfxt::kTile / 2 ? pfxt::prefix_attn_tc_kernel<T, 1> : pfxt::prefix_attn_tc_kernel<T, 2>;
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
  // k is null where there is no row to read, len where there is no cache: a cache without slots still has its lengths checked
  auto side = [](const rb_kv_cache* s, const int64_t* len) {
    const bool rows = s->cache_len > 0;
    return Side{rows ? static_cast<const uint8_t*>(s->k) : nullptr, static_cast<const uint8_t*>(s->v), s->k_par, s->v_par, len, s->cache_len};
  };
  if (a->prefix) p.pre = side(a->prefix, a->prefix_len);
  if (a->own) p.own = side(a->own, a->own_len);
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
