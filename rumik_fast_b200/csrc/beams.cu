// beams.cu - one step of a beam search on the device: the selection of the best beams over every beam's vocabulary
// (rb_beam_select) and the reordering of the beams' cache rows by their parents, in place (rb_beam_reorder).
//
// Selection, per request of nb beams:
//   cand[b, v] = (x[b, v] - m_b) - log sum_v exp(x[b, v] - m_b) + score_b,  m_b = max_v x[b, v]        (a live beam)
//   cand[b, end] = score_b and nothing else                                           (a finished beam)
// and the nb best of the nb V candidates. Within a beam the order of the candidates is the order of the logits, so no
// normaliser is needed to find a beam's nb best rows: one pass over the logits yields each chunk's maximum, sum of
// exponentials and nb best (value, row) keys. A CTA takes its chunk in batches of 4096 rows, the next one's loads in
// flight; the first batch gives a bound that nb keys reach, and of later ones only the keys above it are looked at: two
// barriers a batch instead of a selection. The last chunk of a beam to finish merges them, and the last beam
// of a request picks the winners: one launch, every logit read once.
// A key is the logit's order-preserving 32 bits above the row's complement, so the largest key is the largest logit,
// the lower row among equals, and no two keys are equal: the result does not depend on the order of arrival.
// Bound: 8 requests of 16 beams over 130,001 fp32 logits take 30 us, 0.34 of the measured copy bandwidth: half of the time
// in barriers of the batches, the rest in the 17 instructions a warp spends on 32 logits (45 us with one batch a CTA and
// its selection for each). Four beams over 16,385 rows: 10 us, three dependent steps of latency (chunk, beam, request).
#include "common.cuh"
#include "kernels.h"

namespace rb {

namespace bm {

using Key = unsigned long long;
constexpr int kThreads = 256;
constexpr int kPer = 16;                       // logits of a thread, held in registers
constexpr int kChunk = kThreads * kPer;        // 4096 rows a batch
constexpr int kSelectCtas = 4;                 // of an SM, by registers and shared memory
constexpr int kFew = 64;                        // threads whose keys a list takes before it is cut back to the nb best (144: 32 us, not 30)
constexpr int kMaxBeams = 32;
constexpr int kCap = kThreads / 32 * kMaxBeams * kPer;                // keys that may pass a bound: 4096
// Keys of the lists that a beam's or a request's last CTA merges: nb of each of a beam's chunks, of which a launch has no more
// than kMaxCtas over all rows unless each row has just one (select_per); or nb of each beam.
constexpr int kMaxCtas = 4096;
static_assert(kCap >= kChunk && kCap >= kFew * kPer && kMaxCtas <= kThreads * kPer && kMaxBeams * kMaxBeams <= kThreads * kPer,
              "at most kPer keys a thread, as in a batch");

struct SelectParams {
  const void* logits;
  int64_t ld;
  const float* scores;
  const uint8_t* done;
  const int64_t* ids;
  const int64_t* step;
  float* out_scores;
  int64_t* out_parents;
  int64_t* out_tokens;
  uint8_t* out_done;
  unsigned int* tickets;   // [R nb] chunks done, then [R] beams done: zero between launches
  float2* part;            // [R nb][chunks] (maximum, sum of exponentials)
  Key* keys;               // [R nb][chunks][nb]
  float* row_cand;         // [R nb][nb] a beam's best candidates, best first
  int* row_idx;            // [R nb][nb] their rows (-1: none)
  int64_t end_idx, min_new;
  int nb, V, chunks, per;  // per: batches of kChunk logits a CTA takes
};

__device__ __forceinline__ Key make_key(float x, uint32_t row) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 -> +0
  const uint32_t k = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (static_cast<Key>(k) << 32) | (0xffffffffu - row);
}
__device__ __forceinline__ float key_value(Key key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint32_t key_row(Key key) { return 0xffffffffu - static_cast<uint32_t>(key); }

struct Shared {
  Key cand[kCap + kMaxBeams];  // a batch's keys and those that were kept of the ones before
  Key top[kThreads];
  Key bound[kThreads / 32], each[kThreads / 32];
  float2 red[kThreads / 32];
  int n;
  int last;
};

// A bound that at least k of the CTA's keys reach. `best` is this thread's largest key (0: none). From the ranks within the
// warps, the larger of two such bounds: the largest over the warps of a warp's k-th (at most k lanes of each warp reach
// it), and the smallest over the warps of a warp's ceil(k / 8)-th (8 ceil(k / 8) keys do), which is the closer one on
// ordinary logits - about 2 k keys pass it.
__device__ __forceinline__ Key cta_bound(Shared& sh, int k, Key best) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  sh.top[threadIdx.x] = best;
  if (lane == 0) sh.bound[warp] = 1, sh.each[warp] = 0;
  __syncwarp();
  int rank = 0;
  const ulonglong2* all = reinterpret_cast<const ulonglong2*>(sh.top + warp * 32);
#pragma unroll 8
  for (int j = 0; j < 16; ++j) {
    const ulonglong2 v = all[j];
    rank += v.x > best;
    rank += v.y > best;
  }
  if (rank == k - 1 && best != 0) sh.bound[warp] = best;  // keys differ: one thread has this rank
  if (rank == (k + kThreads / 32 - 1) / (kThreads / 32) - 1) sh.each[warp] = best;
  __syncthreads();
  Key lim = 1, least = ~Key(0);
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    lim = sh.bound[w] > lim ? sh.bound[w] : lim;
    least = sh.each[w] < least ? sh.each[w] : least;
  }
  return least > lim ? least : lim;
}

// The k largest of the keys in sh.cand, best first, through out(rank, key); ranks without a key get 0.
template <typename Out>
__device__ __forceinline__ void cta_rank(Shared& sh, int k, Out out) {
  __syncthreads();
  const int n = sh.n;
#pragma unroll 1
  for (int c = threadIdx.x; c < n; c += kThreads) {
    const Key v = sh.cand[c];
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) r += sh.cand[j] > v;
    if (r < k) out(r, v);
  }
  for (int r = n + threadIdx.x; r < k; r += kThreads) out(r, Key(0));
  __syncthreads();
}

// The k largest of n <= kPer kThreads keys get(0) .. get(n - 1) (0: none).
template <typename Get, typename Out>
__device__ __forceinline__ void cta_top(Shared& sh, int k, int n, Get get, Out out) {
  if (n <= kThreads) {  // a key a thread: all of them are ranked
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    const Key v = threadIdx.x < n ? get(threadIdx.x) : Key(0);
    if (v) sh.cand[atomicAdd(&sh.n, 1)] = v;
  } else {
    Key best = 0;
    if (threadIdx.x == 0) sh.n = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const Key v = get(i);
      best = v > best ? v : best;
    }
    const Key lim = cta_bound(sh, k, best);
    if (best >= lim) {
#pragma unroll 1
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const Key v = get(i);
        if (v >= lim) sh.cand[atomicAdd(&sh.n, 1)] = v;
      }
    }
  }
  cta_rank(sh, k, out);
}

// Whether this CTA is the last of `of` to arrive at the ticket, which is then zero again. What the others wrote
// before they arrived is visible to the last one's loads: the barrier puts a CTA's writes before its one thread's
// release, and that thread's acquire before the loads.
__device__ __forceinline__ bool last_to_arrive(Shared& sh, unsigned int* ticket, int of) {
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned int before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
    const bool last = before + 1u == static_cast<unsigned>(of);
    if (last) *ticket = 0u;
    sh.last = last;
  }
  __syncthreads();
  return sh.last != 0;
}

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) {  // the hardware's 2^x (relative error 2^-22)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp_of(float x) { return ex2(x * kLog2e); }
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// (maximum, sum of exponentials) of two parts; a maximum of +inf marks a part without a distribution.
__device__ __forceinline__ float2 merge_sums(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY || m == INFINITY) return make_float2(m, 0.f);
  return make_float2(m, a.y * exp_of(a.x - m) + b.y * exp_of(b.x - m));
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kSelectCtas) beam_select_kernel(const __grid_constant__ SelectParams p) {
  __shared__ Shared sh;
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y, chunk = blockIdx.x, nb = p.nb;
  const int req = row / nb;
  const bool early = p.step && *p.step < p.min_new;
  const float score = p.scores[row];
  const bool done = p.done[row] != 0;
  const bool dead = !(score > -INFINITY && score < INFINITY);  // no candidate of this beam counts
  if (!done && !dead) {
    const int begin = chunk * p.per * kChunk, end = min(p.V, begin + p.per * kChunk);
    const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
    T raw[kPer];
    auto load = [&](int from) {
      if (from + kChunk <= end) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) raw[i] = x[from + tid + i * kThreads];
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) raw[i] = from + tid + i * kThreads < end ? x[from + tid + i * kThreads] : T(-INFINITY);
      }
    };
    load(begin);
    float2 ms = make_float2(-INFINITY, 0.f);
    bool odd = false;
    Key lim = 1;         // at least nb keys so far reach it (1: fewer keys than that)
    float least = 0.f;   // its logit (NaN for 1)
    int held = 0;        // threads whose keys are in sh.cand, about the keys there
    if (tid == 0) sh.n = 0;
#pragma unroll 1
    for (int from = begin; from < end; from += kChunk) {
      const int first = from + tid;
      float v[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = static_cast<float>(raw[i]);
      if (from + kChunk < end) load(from + kChunk);
      if (early) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (first + i * kThreads == p.end_idx) v[i] = -INFINITY;
      }
      float top = v[0];
#pragma unroll
      for (int i = 1; i < kPer; ++i) top = max_nan(top, v[i]);
      odd |= !(top < INFINITY);  // NaN or +inf: the row has no distribution
      if (!odd && top > -INFINITY) {
        const float m = fmaxf(ms.x, top);
        float2 sum = make_float2(ms.y * exp_of(ms.x - m), 0.f);
        const float2 off = make_float2(-m, -m), unit = make_float2(kLog2e, kLog2e);
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
          const float2 t = mul2(add2(make_float2(v[i], v[i + 1]), off), unit);
          sum = add2(sum, make_float2(ex2(t.x), ex2(t.y)));
        }
        ms = make_float2(m, sum.x + sum.y);
      }
      auto best = [&] {  // this thread's largest key: the lowest row among equals
        int at = 0;
#pragma unroll
        for (int i = kPer - 1; i > 0; --i)
          if (v[i] == top) at = i;
        if (v[0] == top) at = 0;
        return first < end ? make_key(top, first + at * kThreads) : Key(0);
      };
      // rows past the vocabulary hold -inf like masked ones, but no key
      auto reaches = [&] { return first < end && !(top < least); };
      if (from == begin) {
        lim = cta_bound(sh, nb, best());
        least = key_value(lim);
      }
      int many = __syncthreads_count(reaches());
      if (from > begin && held + many > kFew) {
        // the list's nb best stay, and the last of them is the new bound
        cta_rank(sh, nb, [&](int r, Key key) { sh.top[r] = key; });
        if (tid < nb) sh.cand[tid] = sh.top[tid];
        if (tid == 0) sh.n = min(sh.n, nb);
        lim = max(lim, sh.top[nb - 1]);
        least = key_value(lim);
        held = nb;
        many = __syncthreads_count(reaches());
        if (many > kFew) {  // rising logits, for one: this batch's own bound is closer
          lim = max(lim, cta_bound(sh, nb, best()));
          least = key_value(lim);
          many = __syncthreads_count(reaches());
        }
      }
      held += many;
      if (reaches()) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (!(v[i] < least)) {
            const Key key = make_key(v[i], first + i * kThreads);
            if (key >= lim && first + i * kThreads < end) sh.cand[atomicAdd(&sh.n, 1)] = key;
          }
      }
    }
    if (odd) ms = make_float2(INFINITY, 0.f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      ms = merge_sums(ms, make_float2(__shfl_xor_sync(0xffffffffu, ms.x, o), __shfl_xor_sync(0xffffffffu, ms.y, o)));
    if (lane == 0) sh.red[warp] = ms;
    Key* dst = p.keys + (static_cast<int64_t>(row) * p.chunks + chunk) * nb;
    cta_rank(sh, nb, [&](int r, Key key) { dst[r] = key; });
    if (tid == 0) {
#pragma unroll 1
      for (int w = 1; w < kThreads / 32; ++w) ms = merge_sums(ms, sh.red[w]);
      p.part[static_cast<int64_t>(row) * p.chunks + chunk] = ms;
    }
  }
  if (!last_to_arrive(sh, p.tickets + row, p.chunks)) return;

  // ---- the beam's nb best candidates ----
  float* cand = p.row_cand + static_cast<int64_t>(row) * nb;
  int* idx = p.row_idx + static_cast<int64_t>(row) * nb;
  float2 ms = make_float2(-INFINITY, 0.f);
  bool odd = false;
  if (!done && !dead) {
    // every warp merges the chunks' sums, lane l those of chunks l, l + 32, ...
#pragma unroll 1
    for (int c = lane; c < p.chunks; c += 32) ms = merge_sums(ms, __ldcg(p.part + static_cast<int64_t>(row) * p.chunks + c));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      ms = merge_sums(ms, make_float2(__shfl_xor_sync(0xffffffffu, ms.x, o), __shfl_xor_sync(0xffffffffu, ms.y, o)));
    // lane 0's: the lanes add in different orders, and which thread writes which candidate is not fixed
    ms = make_float2(__shfl_sync(0xffffffffu, ms.x, 0), __shfl_sync(0xffffffffu, ms.y, 0));
    odd = ms.x == INFINITY;
    if (odd && tid == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
  }
  if (!done && !dead && !odd && ms.x > -INFINITY) {
    // ms.y >= 1 up to rounding: the largest logit's own term. The largest logit is taken off first: rounded to a sum with
    // it, the logarithm would lose what logits far from zero leave no bits for.
    const float log_sum = logf(ms.y);
    const Key* src = p.keys + static_cast<int64_t>(row) * p.chunks * nb;
    cta_top(
        sh, nb, p.chunks * nb, [&](int i) { return __ldcg(src + i); },
        [&](int r, Key key) {
          cand[r] = key ? ((key_value(key) - ms.x) - log_sum) + score : -INFINITY;
          idx[r] = key ? static_cast<int>(key_row(key)) : -1;
        });
  } else {
    // a finished beam: its end row with the score it has; then, and for a beam without any candidate, rows of -inf
    // in their order (all of them where the score is not finite)
    const int end = static_cast<int>(p.end_idx);
    const bool counts = done && !dead;
    for (int r = tid; r < nb; r += kThreads) {
      const int rest = counts ? (r - 1 >= end ? r : r - 1) : r;
      const int at = counts && r == 0 ? end : rest;
      cand[r] = counts && r == 0 ? score : -INFINITY;
      idx[r] = at < p.V ? at : -1;
    }
  }
  if (!last_to_arrive(sh, p.tickets + gridDim.y + req, nb)) return;

  // ---- the request's nb best: keys of (candidate, place in the order beam, rank within the beam) ----
  const int64_t base = static_cast<int64_t>(req) * nb * nb;
  cta_top(
      sh, nb, nb * nb,
      [&](int i) { return __ldcg(p.row_idx + base + i) >= 0 ? make_key(__ldcg(p.row_cand + base + i), i) : Key(0); },
      [&](int r, Key key) {
        if (key == 0) return;  // not reached: every beam gives min(nb, V) rows
        const int at = static_cast<int>(key_row(key)), parent = at / nb;
        const int tok = __ldcg(p.row_idx + base + at);
        const int64_t o = static_cast<int64_t>(req) * nb + r;
        p.out_scores[o] = key_value(key);
        p.out_parents[o] = parent;
        p.out_tokens[o] = p.ids ? p.ids[tok] : tok;
        p.out_done[o] = p.done[req * nb + parent] != 0 || tok == p.end_idx;
      });
}

// ---- reordering ----

// Of every (tensor, beam head) line the columns are independent: a thread holds one column of all beams, so any permutation
// or copying of beams is done in place and each row is read once, however many beams take it over. HBM-bound: 72 tensors
// of 8 beams with 701 slots, 0.72 GB, 130 to 139 us (0.79 to 0.85 of the measured copy bandwidth). One launch for up to kMaxTensors
// tensors, which is what counts for small states: 8 tensors of 61 slots 3 us.
constexpr int kReorderThreads = 128;

struct Tensor {
  uint8_t* p;
  int64_t line;   // bytes of one (beam, head): cache_len rows
  int heads, row_bytes, unit, line0;  // unit: bytes of one access; line0: the tensor's first line in the launch
};
constexpr int kMaxTensors = 100;
struct ReorderParams {
  Tensor t[kMaxTensors];
  const int64_t* parents;
  const int64_t* slots;
  int count, nb;
  int64_t cache_len;
};
static_assert(sizeof(ReorderParams) < 4096, "kernel parameters");

template <typename U, int kBeams>
__device__ __forceinline__ void reorder_line(uint8_t* base, int64_t beam_bytes, const int* parent, const int64_t* bytes,
                                             uint32_t needed, int nb, int64_t most, int piece, int pieces) {
  for (int64_t at = (static_cast<int64_t>(piece) * kReorderThreads + threadIdx.x) * sizeof(U); at < most;
       at += static_cast<int64_t>(pieces) * kReorderThreads * sizeof(U)) {
    // one column of every beam that another one takes over, all read before any is written: the columns of a line
    // are independent, so the beams change places in place
    U v[kBeams];
#pragma unroll
    for (int b = 0; b < kBeams; ++b)
      if ((needed >> b) & 1u) v[b] = *reinterpret_cast<const U*>(base + b * beam_bytes + at);
#pragma unroll
    for (int b = 0; b < kBeams; ++b) {
      if (!((needed >> b) & 1u) || at >= bytes[b]) continue;
      for (int c = 0; c < nb; ++c)
        if (parent[c] == b && c != b) *reinterpret_cast<U*>(base + c * beam_bytes + at) = v[b];
    }
  }
}

template <int kBeams>
__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(const __grid_constant__ ReorderParams p) {
  __shared__ int parent[kMaxBeams];
  __shared__ int64_t bytes[kMaxBeams];
  griddep_wait();
  griddep_launch_dependents();
  const int nb = p.nb, req = blockIdx.z;
  int t = 0;
  while (t + 1 < p.count && static_cast<int>(blockIdx.x) >= p.t[t + 1].line0) ++t;
  const Tensor& T = p.t[t];
  const int head = blockIdx.x - T.line0;
  bool ok = true;
  if (threadIdx.x < nb) {
    const int64_t q = p.parents[req * nb + threadIdx.x], n = p.slots[req * nb + threadIdx.x];
    ok = q >= 0 && q < nb && n >= 0 && n <= p.cache_len;
    parent[threadIdx.x] = ok ? static_cast<int>(q) : 0;
    bytes[threadIdx.x] = ok ? n * T.row_bytes : 0;
  }
  if (__syncthreads_or(!ok)) {  // an index that is none: the request's rows stay as they are
    if (threadIdx.x == 0) atomicOr(&g_device_error, static_cast<unsigned>(ERR_ARG));
    return;
  }
  uint32_t needed = 0;
  int64_t most = 0;
  for (int c = 0; c < nb; ++c) {
    const int b = parent[c];
    if (b == c) continue;
    needed |= 1u << b;
    most = bytes[b] > most ? bytes[b] : most;
  }
  if (!needed) return;
  const int64_t beam_bytes = T.line * T.heads;
  uint8_t* base = T.p + static_cast<int64_t>(req) * nb * beam_bytes + head * T.line;
  switch (T.unit) {
    case 16: reorder_line<uint4, kBeams>(base, beam_bytes, parent, bytes, needed, nb, most, blockIdx.y, gridDim.y); break;
    case 8: reorder_line<uint2, kBeams>(base, beam_bytes, parent, bytes, needed, nb, most, blockIdx.y, gridDim.y); break;
    case 4: reorder_line<uint32_t, kBeams>(base, beam_bytes, parent, bytes, needed, nb, most, blockIdx.y, gridDim.y); break;
    default: reorder_line<uint16_t, kBeams>(base, beam_bytes, parent, bytes, needed, nb, most, blockIdx.y, gridDim.y); break;
  }
}

}  // namespace bm

namespace {
int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }
// Batches of kChunk logits that a CTA takes: one while the CTAs of all rows are no more than `ctas`, else the fewest that
// make them so (all of a row's, if need be).
int64_t select_per(int64_t rows, int64_t V, int64_t ctas) {
  const int64_t batches = (V + bm::kChunk - 1) / bm::kChunk;
  int64_t per = 1;
  while (per < batches && rows * ((batches + per - 1) / per) > std::min<int64_t>(ctas, bm::kMaxCtas)) ++per;
  return per;
}
int64_t select_chunks(int64_t V, int64_t per) { return (V + per * bm::kChunk - 1) / (per * bm::kChunk); }
}  // namespace

int64_t beam_select_tickets(int64_t requests, int nb) { return align16((requests * nb + requests) * 4); }

int64_t beam_select_workspace(int64_t requests, int nb, int64_t V) {
  // for the most CTAs that a launch has, however many the device holds: more of them have no fewer chunks a row
  const int64_t rows = requests * nb, ch = select_chunks(V, select_per(rows, V, bm::kMaxCtas));
  return beam_select_tickets(requests, nb) + align16(rows * ch * 8) + align16(rows * ch * nb * 8) + 2 * align16(rows * nb * 4);
}

int launch_beam_select(const rb_beam_select_args* a, int num_sms, int flags, cudaStream_t stream) {
  using namespace bm;
  const int64_t rows = a->requests * a->n_beams;
  SelectParams p = {};
  p.logits = a->logits;
  p.ld = a->ld;
  p.scores = a->scores;
  p.done = a->done;
  p.ids = a->ids;
  p.step = a->step;
  p.out_scores = a->out_scores;
  p.out_parents = a->out_parents;
  p.out_tokens = a->out_tokens;
  p.out_done = a->out_done;
  p.end_idx = a->end_idx;
  p.min_new = a->min_new;
  p.nb = a->n_beams;
  p.V = static_cast<int>(a->n_vocab);
  p.per = static_cast<int>(select_per(rows, a->n_vocab, kSelectCtas * static_cast<int64_t>(num_sms)));  // the CTAs fit on the SMs at once
  p.chunks = static_cast<int>(select_chunks(a->n_vocab, p.per));
  uint8_t* w = static_cast<uint8_t*>(a->ws);
  p.tickets = reinterpret_cast<unsigned int*>(w);
  w += beam_select_tickets(a->requests, a->n_beams);
  p.part = reinterpret_cast<float2*>(w);
  w += align16(rows * p.chunks * 8);
  p.keys = reinterpret_cast<Key*>(w);
  w += align16(rows * p.chunks * a->n_beams * 8);
  p.row_cand = reinterpret_cast<float*>(w);
  w += align16(rows * a->n_beams * 4);
  p.row_idx = reinterpret_cast<int*>(w);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.chunks, static_cast<unsigned>(rows));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (flags & RB_FLAG_PDL) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void (*kern)(SelectParams) = a->logits_dtype == RB_F32    ? beam_select_kernel<float>
                               : a->logits_dtype == RB_BF16 ? beam_select_kernel<__nv_bfloat16>
                                                            : beam_select_kernel<__half>;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? RB_OK : RB_ERR_LAUNCH;
}

int launch_beam_reorder(const rb_beam_tensor* t, int count, int64_t requests, int nb, int64_t cache_len,
                        const int64_t* parents, const int64_t* slots, int num_sms, int flags, cudaStream_t stream) {
  using namespace bm;
  for (int done = 0; done < count;) {
    ReorderParams p = {};
    p.parents = parents;
    p.slots = slots;
    p.nb = nb;
    p.cache_len = cache_len;
    int lines = 0;
    int64_t widest = 0;
    for (; done < count && p.count < kMaxTensors; ++done) {
      const rb_beam_tensor& s = t[done];
      Tensor& d = p.t[p.count++];
      d.p = static_cast<uint8_t*>(s.p);
      d.heads = s.n_heads;
      d.row_bytes = s.row_bytes;
      d.line = cache_len * s.row_bytes;
      d.line0 = lines;
      // the widest access that every (beam, head) of the tensor is aligned to
      const uint64_t mix = static_cast<uint64_t>(reinterpret_cast<uintptr_t>(s.p)) | static_cast<uint64_t>(d.line) |
                           static_cast<uint64_t>(s.row_bytes);
      d.unit = mix % 16 == 0 ? 16 : mix % 8 == 0 ? 8 : mix % 4 == 0 ? 4 : 2;
      lines += s.n_heads;
      widest = std::max<int64_t>(widest, d.line / d.unit);
    }
    // about eight CTAs an SM, and no more pieces of a line than it has columns for
    int64_t pieces = (8 * static_cast<int64_t>(num_sms) + lines * requests - 1) / (lines * requests);
    pieces = std::max<int64_t>(1, std::min<int64_t>(pieces, (widest + kReorderThreads - 1) / kReorderThreads));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(lines, static_cast<unsigned>(pieces), static_cast<unsigned>(requests));
    cfg.blockDim = dim3(kReorderThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = (flags & RB_FLAG_PDL) ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void (*kern)(ReorderParams) = nb <= 4    ? beam_reorder_kernel<4>
                                  : nb <= 8  ? beam_reorder_kernel<8>
                                  : nb <= 16 ? beam_reorder_kernel<16>
                                             : beam_reorder_kernel<32>;
    if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) return RB_ERR_LAUNCH;
  }
  return RB_OK;
}

}  // namespace rb
