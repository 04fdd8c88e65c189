// tg_beam.cu -- beam search's selection over beams and vocabulary.
//
// Two launches.  scan_kernel streams the logits once: a block takes a part of a row,
// sums exp(x - max) and finds the part's `beams` largest logits.  merge_kernel takes a
// batch row: lse from its parts, score = (x - lse) + scores[beam] for the parts'
// candidates, the `beams` best of them, and the histories.
//
// The candidates of a part cost the stream almost nothing: each thread keeps the
// maximum of every 4 vectors it reads in shared memory.  The (beams + 4)-th largest of
// the maxima of 64 sets of threads bounds the part's (beams + 4)-th largest logit from
// below, so only the few groups that reach it (1.2 to 1.5 times beams + 4, of thousands)
// are read again.
//
// Order is by score in fp32, then index, while a part's list is cut by logit.  The two
// differ only where rounding gives two different logits one score; merge_kernel looks
// for that at every list's cut, among the kept logits and below the cut, and then, as for rows with NaN or +inf or with more ties
// than a list holds, finds the row's list from the logits themselves (row_exact).
//
// Bound and figures (B200): HBM bytes for many rows, each logit once; 1024 rows of 128,256
// bf16 logits take 61 us (263 MB, 4.4 TB/s): the stream itself runs at 6.4 TB/s, the lists
// at its blocks' ends and merge_kernel take a third of the time.  Latency for few: 4 rows
// of 50,257 fp32 logits 11 us, half of it the merge.  A batch row with rows for row_exact
// takes far longer: 0.13 ms with one row of 50,257 and 4 beams, 0.7 ms with one of 128,256 and
// 8 beams, 5 ms with all 8; 64 x 16 such rows 20 ms.
//
// One launch instead of two, the last block of a batch row merging it, was slower on the
// device (66 and 12 us: every block waits for its fence and its arrival, and the merge
// has fewer threads).  Persistent blocks with a ring of bulk copies were slower too (86 us:
// a block per SM hides the ends of its rows less well than 4).
#include "tg_host.h"

#include <cuda_bf16.h>

#include <cfloat>
#include <cmath>
#include <new>

namespace tg {
namespace {

constexpr int kThreads = 256;
constexpr int kMergeThreads = 512;
constexpr int kQuads = kThreads / 4;
constexpr int kVecs = 4;         // 16-byte vectors of a group
constexpr int kMaxGroups = 32;   // groups of a thread in a part
constexpr int kListMax = 1024;   // candidates of a part before its cut
constexpr int kExtra = 4;        // candidates past `beams`: the first one cut is then known exactly
constexpr int kWave = 592;       // blocks that run at a time: 148 SMs x 4
constexpr float kLog2e = 1.44269504f;
constexpr int kKeep = TG_MAX_BEAMS * TG_MAX_BEAMS;  // keys that the merge ranks
constexpr int kMergeSmem = 200 * 1024;

constexpr uint32_t kBadState = 1, kBadHistory = 2;

struct PartHead {
  float t, l;     // sum over the part of 2^(x log2e - t)
  float cut;      // the largest logit left out of the list (-inf: none)
  int32_t count;  // entries of the list; -1: the row needs row_exact
};

struct Candidate {
  float x;
  int32_t id;
};

struct BeamArgs {
  const void* logits;
  int64_t row_stride;
  int32_t vocab, beams, batch, parts, num_states, mask_words, eos_id, pad_id, history_stride;
  const float* scores;
  const int32_t* finished;
  const uint32_t* mask_table;
  const int32_t* state_id;
  const int32_t* history;
  const int32_t* history_len;
  int32_t *out_parent, *out_token, *out_finished, *out_history, *out_history_len;
  float* out_score;
  PartHead* heads;         // [rows, parts]
  Candidate* candidates;   // [rows, parts, beams]
  uint32_t* status;
};

__device__ __forceinline__ void after_previous_work() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row adds no candidates of its own when its beam is finished or dead.
__device__ __forceinline__ bool row_scores(const BeamArgs& a, int row) {
  const float s = a.scores[row];
  return s > -INFINITY && !(a.finished && a.finished[row]);
}

__device__ __forceinline__ const uint32_t* row_mask(const BeamArgs& a, int row) {
  if (!a.state_id) return nullptr;
  const int s = a.state_id[row];
  return s < 0 || s >= a.num_states ? nullptr : a.mask_table + static_cast<size_t>(s) * a.mask_words;
}

__device__ __forceinline__ bool allowed(const uint32_t* mask, int v) { return !mask || (mask[v >> 5] >> (v & 31) & 1); }

template <int DT>
struct Elem;
template <>
struct Elem<TG_DTYPE_F32> {
  static constexpr int kPer = 4;
  using T = float;
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  // the next smaller value of the type
  static __device__ __forceinline__ float below(float x) { return nextafterf(x, -INFINITY); }
  static __device__ __forceinline__ uint4 masked(const uint4& v, uint32_t bits) {
    return make_uint4(bits & 1 ? v.x : 0xff800000u, bits & 2 ? v.y : 0xff800000u, bits & 4 ? v.z : 0xff800000u, bits & 8 ? v.w : 0xff800000u);
  }
  // the largest of N vectors; NaN does not count
  template <int N>
  static __device__ __forceinline__ float most(const uint4* d) {
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < N; v++) {
      float x[4];
      unpack(d[v], x);
      m = fmaxf(fmaxf(m, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
    }
    return m;
  }
};
template <>
struct Elem<TG_DTYPE_BF16> {
  static constexpr int kPer = 8;
  using T = uint16_t;
  static __device__ __forceinline__ float get(const uint16_t* p) { return __uint_as_float(static_cast<uint32_t>(*p) << 16); }
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  static __device__ __forceinline__ float below(float x) {
    const uint32_t b = __float_as_uint(x);
    return __uint_as_float(x == 0.0f ? 0x80010000u : x > 0.0f ? b - 0x10000u : b + 0x10000u);
  }
  static __device__ __forceinline__ uint32_t masked_word(uint32_t w, uint32_t bits) {
    return (bits & 1 ? w & 0xffffu : 0xff80u) | (bits & 2 ? w & 0xffff0000u : 0xff800000u);
  }
  static __device__ __forceinline__ uint4 masked(const uint4& v, uint32_t bits) {
    return make_uint4(masked_word(v.x, bits), masked_word(v.y, bits >> 2), masked_word(v.z, bits >> 4), masked_word(v.w, bits >> 6));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t m;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    return m;
  }
  template <int N>
  static __device__ __forceinline__ float most(const uint4* d) {
    uint32_t m = 0xff80ff80u;
#pragma unroll
    for (int v = 0; v < N; v++) m = max2(max2(m, max2(d[v].x, d[v].y)), max2(d[v].z, d[v].w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
};

__device__ __forceinline__ uint4 load_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// The bits of `kPer` tokens from token v on (v + kPer <= vocab).
template <int kPer>
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* mask, int v) {
  const uint32_t lo = mask[v >> 5];
  const uint32_t hi = (v & 31) + kPer > 32 ? mask[(v >> 5) + 1] : 0;
  return __funnelshift_r(lo, hi, v & 31);
}

__device__ __forceinline__ uint64_t two(float lo, float hi) { return static_cast<uint64_t>(__float_as_uint(hi)) << 32 | __float_as_uint(lo); }
__device__ __forceinline__ float low_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// sum 2^(x log2e - t), rescaled when a group exceeds t: t is a rounded x log2e, so
// the largest term is 1 but for t's rounding, which lse = t / log2e + ln(sum) takes out
// again.  From logits of about 2^30 on that rounding alone is a hundred binary orders and
// more: the sum is then 0 or infinite, and the row is left to row_exact.
struct Sum {
  float t = -INFINITY, l = 0.0f;
  __device__ __forceinline__ void raise(float top) {
    // finite for every finite logit: with t = -inf the terms of the lowest values, as masks
    // have them, would be infinite and not 0 beside ordinary ones
    const float at = top > -INFINITY ? fmaxf(top * kLog2e, -FLT_MAX) : top;
    if (at > t) {
      l *= exp2_fast(t - at);
      t = at;
    }
  }
  __device__ __forceinline__ void add(float x, float top) {
    raise(top);
    if (top > -INFINITY) l += exp2_fast(__fmaf_rn(x, kLog2e, -t));
  }
  // N vectors, whose largest is `top`; two elements an instruction where it exists
  template <typename E, int N>
  __device__ __forceinline__ void add(const uint4* d, float top) {
    raise(top);
    if (!(top > -INFINITY)) return;
    const uint64_t scale = two(kLog2e, kLog2e), from = two(-t, -t);
    uint64_t s[2] = {0, 0};
#pragma unroll
    for (int v = 0; v < N; v++) {
      float x[E::kPer];
      E::unpack(d[v], x);
#pragma unroll
      for (int i = 0; i < E::kPer; i += 2) {
        const uint64_t y = fma2(two(x[i], x[i + 1]), scale, from);
        s[i / 2 & 1] = add2(s[i / 2 & 1], two(exp2_fast(low_of(y)), exp2_fast(high_of(y))));
      }
    }
    s[0] = add2(s[0], s[1]);
    l += low_of(s[0]) + high_of(s[0]);
  }
};

// The 32 lanes' sums as one, in every lane.
__device__ __forceinline__ void join_lanes(Sum& s) {
  float t = s.t;
  for (int d = 16; d; d >>= 1) t = fmaxf(t, __shfl_xor_sync(~0u, t, d));
  float l = s.t > -INFINITY ? s.l * exp2_fast(s.t - t) : 0.0f;
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
  s.t = t, s.l = l;
}

__device__ __forceinline__ bool before(float xa, int ia, float xb, int ib) { return xa > xb || (xa == xb && ia < ib); }

template <int DT, bool kMasked>
__global__ void __launch_bounds__(kThreads, 4) scan_kernel(BeamArgs a) {
  using E = Elem<DT>;
  constexpr int kPer = E::kPer;
  __shared__ float group_max[kMaxGroups + 1][kThreads];
  __shared__ __align__(16) float quad_max[kQuads];
  __shared__ Candidate list[kListMax];
  __shared__ int32_t hits[kListMax];  // groups to read again: group * kThreads + thread
  __shared__ float warp_t[kThreads / 32], warp_l[kThreads / 32];
  __shared__ int n_list, n_hits;
  __shared__ float bound;
  const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  after_previous_work();
  if (!row_scores(a, row)) return;
  const uint32_t* mask = kMasked ? row_mask(a, row) : nullptr;
  const typename E::T* p = static_cast<const typename E::T*>(a.logits) + row * a.row_stride;
  // the row's 16-byte-aligned middle in equal parts; the first part also has the
  // elements before it, the last those after it
  const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(typename E::T)), a.vocab);
  const int vecs = (a.vocab - head) / kPer;
  const int per = (vecs + a.parts - 1) / a.parts;
  const int v0 = min(part * per, vecs), v1 = min(v0 + per, vecs);
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  const int groups = (v1 - v0 + kThreads * kVecs - 1) / (kThreads * kVecs);

  Sum sum;
  float most = -INFINITY;
  // the odd elements: one per thread, kept as a group of their own
  int odd = -1;
  if (part == 0 && tid < head) odd = tid;
  if (part == a.parts - 1 && tid >= 32) {
    const int v = head + vecs * kPer + tid - 32;
    if (v < a.vocab) odd = v;
  }
  float odd_x = -INFINITY;
  if (odd >= 0 && allowed(mask, odd)) {
    odd_x = fmaxf(E::get(p + odd), -INFINITY);  // NaN: -inf
    const float raw = E::get(p + odd);
    sum.add(raw, odd_x);
  }
  group_max[groups][tid] = odd_x;
  most = odd_x;

  const auto fetch = [&](int g, uint4* d) {
#pragma unroll
    for (int u = 0; u < kVecs; u++) {
      const int i = v0 + (g * kVecs + u) * kThreads + tid;
      d[u] = i < v1 ? load_stream(pv + i) : E::nothing();
    }
  };
  const auto mask_group = [&](int g, uint4* d) {
    if (!kMasked || !mask) return;
    uint32_t bits[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; u++) {
      const int i = v0 + (g * kVecs + u) * kThreads + tid;
      bits[u] = i < v1 ? mask_bits<kPer>(mask, head + i * kPer) : 0;
    }
#pragma unroll
    for (int u = 0; u < kVecs; u++) d[u] = E::masked(d[u], bits[u]);
  };
  uint4 next[kVecs];
  if (groups > 0) fetch(0, next);
  for (int g = 0; g < groups; g++) {
    uint4 now[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; u++) now[u] = next[u];
    if (g + 1 < groups) fetch(g + 1, next);
    mask_group(g, now);
    const float top = E::template most<kVecs>(now);
    sum.add<E, kVecs>(now, top);
    group_max[g][tid] = top;
    most = fmaxf(most, top);
  }
  join_lanes(sum);
  if ((tid & 31) == 0) warp_t[tid >> 5] = sum.t, warp_l[tid >> 5] = sum.l;
  // the maxima of 4 threads each, 64 in all
  float quad = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
  quad = fmaxf(quad, __shfl_xor_sync(~0u, quad, 2));
  if ((tid & 3) == 0) quad_max[tid >> 2] = quad;
  if (tid == 0) {
    n_list = n_hits = 0;
    bound = -INFINITY;
  }
  __syncthreads();
  // the (beams + kExtra)-th largest of them, which as many logits reach: each thread
  // counts those before its own
  if (tid < kQuads) {
    const float mine = quad_max[tid];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < kQuads; i += 4) {
      const float4 o = *reinterpret_cast<const float4*>(&quad_max[i]);
      rank += before(o.x, i, mine, tid) + before(o.y, i + 1, mine, tid) + before(o.z, i + 2, mine, tid) + before(o.w, i + 3, mine, tid);
    }
    if (rank == a.beams + kExtra - 1) bound = mine;
  }
  __syncthreads();
  // the groups that reach it, then their vectors, one per thread: all re-reads at once
  const float low = bound;
  if (most >= low && most > -INFINITY)
    for (int g = 0; g < groups; g++) {
      const float top = group_max[g][tid];
      if (top >= low && top > -INFINITY) {
        const int at = atomicAdd(&n_hits, 1);
        if (at < kListMax) hits[at] = g * kThreads + tid;
      }
    }
  __syncthreads();
  const auto put = [&](float x, int id) {
    const int at = atomicAdd(&n_list, 1);
    if (at < kListMax) list[at] = Candidate{x, id};
  };
  const int n_groups = min(n_hits, kListMax);
  for (int h = tid; h < n_groups * kVecs; h += kThreads) {
    const int hit = hits[h / kVecs], i = v0 + (hit / kThreads * kVecs + h % kVecs) * kThreads + hit % kThreads;
    if (i >= v1) continue;
    uint4 d = load_stream(pv + i);
    const int id = head + i * kPer;
    if (kMasked && mask) d = E::masked(d, mask_bits<kPer>(mask, id));
    float x[kPer];
    E::unpack(d, x);
#pragma unroll
    for (int e = 0; e < kPer; e++)
      if (x[e] >= low && x[e] > -INFINITY) put(x[e], id + e);
  }
  if (odd_x >= low && odd_x > -INFINITY) put(odd_x, odd);
  __syncthreads();
  const int n = n_hits > kListMax ? kListMax + 1 : n_list, kept = min(n, a.beams);  // a group has one at least
  const int64_t at = static_cast<int64_t>(row) * a.parts + part;
  if (n <= kListMax) {
    for (int i = tid; i < n; i += kThreads) {
      const Candidate c = list[i];
      int r = 0;
      for (int j = 0; j < n; j++) r += before(list[j].x, list[j].id, c.x, c.id);
      if (r < a.beams) a.candidates[at * a.beams + r] = c;
      if (r == a.beams) a.heads[at].cut = c.x;
    }
    if (tid == 0 && n <= a.beams) a.heads[at].cut = -INFINITY;
  }
  if (tid < 32) {
    Sum s;
    if (tid < kThreads / 32) s.t = warp_t[tid], s.l = warp_l[tid];
    join_lanes(s);
    if (tid == 0) {
      a.heads[at].t = s.t;
      a.heads[at].l = s.l;
      // NaN, +inf or logits far beyond what t can tell apart in the part: its sum is not finite
      a.heads[at].count = n <= kListMax && s.l < INFINITY && s.t < INFINITY ? kept : -1;
    }
  }
}

// 64-bit keys in the order of the result: score, then the lower index.
__device__ __forceinline__ uint64_t key_of(float s, uint32_t index) {
  const uint32_t b = __float_as_uint(s);
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<uint64_t>(o) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float score_of(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xffffffffu - static_cast<uint32_t>(key); }

// -0 and +0 are one score.
__device__ __forceinline__ float score(float x, float lse, float beam) { return ((x - lse) + beam) + 0.0f; }

// The block's largest key; every thread gets it.
__device__ uint64_t block_max(uint64_t k, uint64_t* warp_keys) {
  for (int d = 16; d; d >>= 1) {
    const uint64_t o = __shfl_xor_sync(~0u, k, d);
    k = o > k ? o : k;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warp_keys[threadIdx.x >> 5] = k;
  __syncthreads();
  uint64_t best = 0;
  for (int w = 0; w < kMergeThreads / 32; w++) best = warp_keys[w] > best ? warp_keys[w] : best;
  return best;
}

template <int DT>
__device__ __forceinline__ float logit(const typename Elem<DT>::T* p, const uint32_t* mask, int v) {
  if (!allowed(mask, v)) return -INFINITY;
  return fminf(fmaxf(Elem<DT>::get(p + v), -INFINITY), FLT_MAX);  // NaN: -inf, +inf: the largest finite value
}

// A row's lse and its `beams` best keys from the logits, by `beams` + 2 passes of the
// block over the row: what the lists cannot settle.
template <int DT>
__device__ void row_exact(const BeamArgs& a, int row, int w, float* lse_out, uint64_t* keys, uint64_t* warp_keys) {
  const typename Elem<DT>::T* p = static_cast<const typename Elem<DT>::T*>(a.logits) + row * a.row_stride;
  const uint32_t* mask = row_mask(a, row);
  const int tid = threadIdx.x;
  float top = -INFINITY;
  for (int v = tid; v < a.vocab; v += kMergeThreads) top = fmaxf(top, logit<DT>(p, mask, v));
  top = score_of(block_max(key_of(top, 0), warp_keys));
  double sum = 0.0;
  if (top > -INFINITY)
    for (int v = tid; v < a.vocab; v += kMergeThreads) sum += exp(static_cast<double>(logit<DT>(p, mask, v)) - static_cast<double>(top));
  // the block's sum, in a fixed order
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
  __syncthreads();
  if ((tid & 31) == 0) warp_keys[tid >> 5] = __double_as_longlong(sum);
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < kMergeThreads / 32; i++) sum += __longlong_as_double(warp_keys[i]);
  const float lse = static_cast<float>(static_cast<double>(top) + log(sum));
  const float beam = a.scores[row];
  uint64_t prev = ~0ull;
  for (int r = 0; r < a.beams; r++) {
    uint64_t best = 0;
    if (top > -INFINITY)
      for (int v = tid; v < a.vocab; v += kMergeThreads) {
        const float x = logit<DT>(p, mask, v);
        if (x == -INFINITY) continue;
        const float s = score(x, lse, beam);
        if (!(s > -INFINITY)) continue;
        const uint64_t k = key_of(s, static_cast<uint32_t>(w) * a.vocab + v);
        if (k < prev && k > best) best = k;
      }
    best = block_max(best, warp_keys);
    if (tid == 0) keys[r] = best;
    prev = best;
    if (best == 0) {  // no more: the same for every thread
      for (int i = r + 1 + tid; i < a.beams; i += kMergeThreads) keys[i] = 0;
      break;
    }
  }
  if (tid == 0) *lse_out = lse;
  __syncthreads();
}

// Key 0: no candidate.
template <int DT>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(BeamArgs a) {
  extern __shared__ uint64_t keys[];  // [beams, parts, beams], then PartHead [beams, parts]
  __shared__ uint64_t warp_keys[kMergeThreads / 32], best[TG_MAX_BEAMS], keep[kKeep];
  __shared__ unsigned long long bound;
  __shared__ int n_keys;
  __shared__ float lse[TG_MAX_BEAMS], row_sum[TG_MAX_BEAMS], beam[TG_MAX_BEAMS];
  __shared__ int live[TG_MAX_BEAMS];    // 1: the row adds candidates, 2: it goes on as it is, 0: neither
  __shared__ int exact[TG_MAX_BEAMS];   // 1: the row needs row_exact, 2: it had it
  __shared__ int from_row[TG_MAX_BEAMS], from_len[TG_MAX_BEAMS], grow[TG_MAX_BEAMS];
  const int b = blockIdx.x, tid = threadIdx.x, W = a.beams, P = a.parts, row0 = b * W, lane = tid & 31;
  after_previous_work();
  const int per_row = P * W, total = W * per_row;
  PartHead* heads = reinterpret_cast<PartHead*>(keys + total);
  // what the first key of each thread needs, on its way while the heads are read
  Candidate first{0.0f, 0};
  if (tid < total) first = a.candidates[static_cast<int64_t>(row0) * per_row + tid];
  if (tid < W) {
    const int row = row0 + tid;
    const float s = a.scores[row];
    const bool done = a.finished && a.finished[row];
    beam[tid] = s;
    live[tid] = s > -INFINITY ? (done ? 2 : 1) : 0;
    exact[tid] = 0;
    if (a.state_id && live[tid] == 1 && a.state_id[row] >= a.num_states) atomicOr(a.status, kBadState);
  }
  for (int i = tid; i < W * P; i += kMergeThreads) heads[i] = a.heads[static_cast<int64_t>(row0) * P + i];
  __syncthreads();
  for (int i = tid; i < W * P; i += kMergeThreads) {
    if (live[i / P] != 1) heads[i] = PartHead{-INFINITY, 0.0f, -INFINITY, 0};
    if (heads[i].count < 0) exact[i / P] = 1;
  }
  __syncthreads();
  // lse of a row: a warp adds its parts, a thread takes the logarithm
  for (int w = tid >> 5; w < W; w += kMergeThreads / 32) {
    float top = -INFINITY, sum = 0.0f;
    for (int p = lane; p < P; p += 32) top = fmaxf(top, heads[w * P + p].t);
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    for (int p = lane; p < P; p += 32)
      if (heads[w * P + p].t > -INFINITY) sum += heads[w * P + p].l * exp2_fast(heads[w * P + p].t - top);
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    if (lane == 0) lse[w] = top, row_sum[w] = sum;
  }
  __syncthreads();
  // a sum that fp32 does not hold (see Sum): row_exact
  if (tid < W && lse[tid] > -INFINITY && !(row_sum[tid] > 0.0f && row_sum[tid] < INFINITY)) exact[tid] = 1;
  if (tid < W && lse[tid] > -INFINITY)
    lse[tid] = static_cast<float>(static_cast<double>(lse[tid]) * (1.0 / static_cast<double>(kLog2e)) + log(static_cast<double>(row_sum[tid])));
  __syncthreads();
  for (int i = tid; i < total; i += kMergeThreads) {
    const int w = i / per_row, list = i / W, r = i - list * W;
    uint64_t k = 0;
    if (live[w] == 1) {
      if (r < heads[list].count) {
        const Candidate c = i == tid ? first : a.candidates[static_cast<int64_t>(row0) * per_row + i];
        const float s = score(c.x, lse[w], beam[w]);
        if (s > -INFINITY) k = key_of(s, static_cast<uint32_t>(w) * a.vocab + c.id);
      }
    } else if (live[w] == 2 && i == w * per_row) {  // finished: it stays as it is
      k = key_of(beam[w] + 0.0f, static_cast<uint32_t>(w) * a.vocab + a.pad_id);
    }
    keys[i] = k;
  }
  __syncthreads();
  for (bool again = true; again;) {
    again = false;
    for (int w = 0; w < W; w++)
      if (exact[w] == 1) {  // the same for every thread
        for (int i = W + tid; i < per_row; i += kMergeThreads) keys[w * per_row + i] = 0;
        row_exact<DT>(a, row0 + w, w, &lse[w], keys + w * per_row, warp_keys);
        if (tid == 0) exact[w] = 2;
        __syncthreads();
      }
    // Bounds of the beams-th best key: the beams-th best of the lists' first keys, and the
    // beams/2-th best of the lists' pairs of first keys, by the lesser.  Lists fall but for
    // rounding, so at most about beams * beams keys reach them.  Each of these counts those
    // before it.
    if (tid == 0) n_keys = 0, bound = 0;
    if (tid < W) best[tid] = 0;
    __syncthreads();
    const int lists = W * P;
    const auto front = [&](int list, bool pair) {
      const uint64_t k = keys[list * W];
      return pair ? min(k, keys[list * W + 1]) : k;
    };
    for (int i = tid; i < (W > 1 ? 2 * lists : lists); i += kMergeThreads) {
      const bool pair = i >= lists;
      const uint64_t k = front(pair ? i - lists : i, pair);
      int r = 0;
      if (k != 0) {
#pragma unroll 4
        for (int j = 0; j < lists; j++) r += front(j, pair) > k;
        if (r + 1 == (pair ? (W + 1) / 2 : W)) atomicMax(&bound, static_cast<unsigned long long>(k));
      }
    }
    __syncthreads();
    for (int i0 = 0; i0 < total; i0 += kMergeThreads) {
      const uint64_t k = i0 + tid < total ? keys[i0 + tid] : 0;
      const bool in = k != 0 && k >= bound;
      const uint32_t all = __ballot_sync(~0u, in);
      int at = 0;
      if (lane == 0 && all) at = atomicAdd(&n_keys, __popc(all));
      at = __shfl_sync(~0u, at, 0) + __popc(all & ((1u << lane) - 1));
      if (in && at < kKeep) keep[at] = k;
    }
    __syncthreads();
    if (n_keys <= kKeep) {
      for (int i = tid; i < n_keys; i += kMergeThreads) {
        const uint64_t k = keep[i];
        int r = 0;
#pragma unroll 4
        for (int j = 0; j < n_keys; j++) r += keep[j] > k;
        if (r < W) best[r] = k;
      }
    } else {
      uint64_t prev = ~0ull;
      for (int r = 0; r < W; r++) {
        uint64_t k = 0;
        for (int i = tid; i < total; i += kMergeThreads) {
          const uint64_t o = keys[i];
          if (o < prev && o > k) k = o;
        }
        k = block_max(k, warp_keys);
        if (tid == 0) best[r] = k;
        prev = k;
      }
    }
    __syncthreads();
    // A logit that a list left out matters only if it has the score of one that the
    // list kept with a larger logit, and that score reaches the selection.  The largest
    // left out has it then; beside kept ones of its own logit, which come before it, a
    // smaller one may.
    const uint64_t last = best[W - 1];
    for (int i = tid; i < W * P; i += kMergeThreads) {
      const int w = i / P;
      const PartHead h = heads[i];
      if (exact[w] || live[w] != 1 || h.cut == -INFINITY || h.count <= 0) continue;
      // the list's kept logits with the cut one's score, if any, are at its end
      const float s = score(h.cut, lse[w], beam[w]);
      if (!(s > -INFINITY) || (last != 0 && s < score_of(last))) continue;
      for (int r = h.count - 1; r >= 0; r--) {
        const uint64_t k = keys[i * W + r];
        if (k == 0 || score_of(k) != s) break;
        const Candidate c = a.candidates[(static_cast<int64_t>(row0) * P + i) * W + r];
        if (c.x != h.cut || score(Elem<DT>::below(h.cut), lse[w], beam[w]) == s) {
          exact[w] = 1;
          break;
        }
      }
    }
    __syncthreads();
    for (int w = 0; w < W; w++) again |= exact[w] == 1;
    __syncthreads();
  }
  if (tid < W) {
    const uint64_t k = best[tid];
    const uint32_t index = index_of(k);
    const int parent = k ? static_cast<int>(index / a.vocab) : -1, token = k ? static_cast<int>(index % a.vocab) : -1;
    const int at = row0 + tid;
    a.out_parent[at] = parent;
    a.out_token[at] = token;
    a.out_score[at] = k ? score_of(k) : -INFINITY;
    const bool was = k && live[parent] == 2;
    if (a.out_finished) a.out_finished[at] = !k || was || (a.eos_id >= 0 && token == a.eos_id);
    if (a.history) {
      int len = k ? a.history_len[row0 + parent] : 0;
      if (len < 0 || len > a.history_stride) {
        atomicOr(a.status, kBadHistory);
        len = min(max(len, 0), a.history_stride);
      }
      const bool more = k && len < a.history_stride && !was;
      a.out_history_len[at] = len + more;
      from_row[tid] = row0 + max(parent, 0);
      from_len[tid] = len;
      grow[tid] = more ? token : -1;
    }
  }
  if (!a.history) return;
  __syncthreads();
  // 8 loads of 4 entries on their way per lane where rows are aligned, 16 of one where not
  const auto copy = [&](auto type) {
    using T = decltype(type);
    constexpr int kPer = sizeof(T) / 4, kLoads = kPer > 1 ? 8 : 16, kStep = 32 * kPer * kLoads;
    const int pieces = (a.history_stride + kStep - 1) / kStep;
    for (int u = tid >> 5; u < W * pieces; u += kMergeThreads / 32) {
      const int w = u / pieces, j0 = (u - w * pieces) * kStep + lane * kPer, len = from_len[w];
      const int32_t* from = a.history + static_cast<int64_t>(from_row[w]) * a.history_stride;
      int32_t* to = a.out_history + static_cast<int64_t>(row0 + w) * a.history_stride;
      __align__(16) int32_t x[kPer * kLoads];
#pragma unroll
      for (int e = 0; e < kLoads; e++) {
        const int j = j0 + 32 * kPer * e;
        if (j < len) *reinterpret_cast<T*>(x + e * kPer) = *reinterpret_cast<const T*>(from + j);
      }
#pragma unroll
      for (int e = 0; e < kLoads; e++) {
        const int j = j0 + 32 * kPer * e;
        if (j >= a.history_stride) break;
#pragma unroll
        for (int i = 0; i < kPer; i++)
          if (j + i >= len) x[e * kPer + i] = j + i == len ? grow[w] : -1;
        *reinterpret_cast<T*>(to + j) = *reinterpret_cast<const T*>(x + e * kPer);
      }
    }
  };
  if (a.history_stride % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.history) | reinterpret_cast<uintptr_t>(a.out_history)) & 15) == 0) copy(int4{});
  else copy(int32_t{});
}

// Parts of a row: the number with the least waves x (groups of a part + 3.5), since what
// follows a part's last group takes as long as 3.5 groups (9,000 of 2,700 cycles with 4
// blocks on an SM).  1024 rows of 16 groups: 62 us in one part, 66 in two, 73 in four; 128
// rows: 22.7 us in 4 parts, 24.6 in 3, 26.1 in 2; 4 rows of 13 groups: 10.5 us in 13 parts,
// 12.1 in 2, 14.0 in one.  Never more groups than a block keeps.
int parts_of(int vocab, int per, int rows) {
  const int step = kThreads * kVecs * per;  // elements of one group of every thread
  const int most = (vocab + step - 1) / step, least = (most + kMaxGroups - 1) / kMaxGroups;
  const int limit = kWave / rows > 4 ? kWave / rows : 4;
  int best = least;
  float cost = FLT_MAX;
  for (int p = least; p <= most && (p <= limit || p == least); p++) {
    const float waves = static_cast<float>((static_cast<int64_t>(rows) * p + kWave - 1) / kWave);
    const float c = waves * (static_cast<float>((most + p - 1) / p) + 3.5f);
    if (c < cost) cost = c, best = p;
  }
  return best;
}

}  // namespace
}  // namespace tg

struct tg_beam {
  int device = 0;
  int vocab = 0;
  int beams = 0;
  int max_batch = 0;
  size_t slots = 0;  // (row, part) pairs that the workspace holds
  tg::PartHead* heads = nullptr;
  tg::Candidate* candidates = nullptr;
  uint32_t* status = nullptr;
};

using tg::set_error;

extern "C" {

int32_t tg_beam_destroy(tg_beam* h) {
  if (!h) return TG_OK;
  {
    tg::CurrentDevice g(h->device);
    if (h->heads) cudaFree(h->heads);
  }
  delete h;
  return TG_OK;
}

int32_t tg_beam_create(int32_t device, int32_t vocab, int32_t beams, int32_t max_batch, tg_beam** out) {
  if (!out) return set_error(TG_ERR_INVALID_ARG, "out is NULL");
  *out = nullptr;
  if (vocab <= 0 || vocab > TG_MAX_VOCAB) return set_error(TG_ERR_UNSUPPORTED, "vocab outside [1, TG_MAX_VOCAB]");
  if (beams <= 0 || beams > TG_MAX_BEAMS) return set_error(TG_ERR_UNSUPPORTED, "beams outside [1, TG_MAX_BEAMS]");
  if (max_batch <= 0) return set_error(TG_ERR_INVALID_ARG, "max_batch must be positive");
  if (max_batch > 65535 / beams) return set_error(TG_ERR_UNSUPPORTED, "max_batch * beams beyond 65535");
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) return set_error(TG_ERR_NO_DEVICE, "CUDA device not present");
  tg::CurrentDevice g(device);
  tg_beam* h = new (std::nothrow) tg_beam();
  if (!h) return set_error(TG_ERR_CUDA, "out of host memory");
  h->device = device;
  h->vocab = vocab;
  h->beams = beams;
  h->max_batch = max_batch;
  const size_t rows = static_cast<size_t>(max_batch) * beams;
  // the parts of any number of rows up to `rows`: at most 4 each, or one wave, or what a block's groups ask for
  const size_t least = tg::parts_of(vocab, 4, 1 << 20);
  h->slots = rows * (least > 4 ? least : 4) + tg::kWave;
  char* base = nullptr;
  const size_t list_bytes = h->slots * beams * sizeof(tg::Candidate);
  cudaError_t e = cudaMalloc(&base, h->slots * sizeof(tg::PartHead) + list_bytes + 4);
  if (e == cudaSuccess) {
    h->heads = reinterpret_cast<tg::PartHead*>(base);
    h->candidates = reinterpret_cast<tg::Candidate*>(base + h->slots * sizeof(tg::PartHead));
    h->status = reinterpret_cast<uint32_t*>(base + h->slots * sizeof(tg::PartHead) + list_bytes);
    e = cudaMemset(h->status, 0, 4);
  }
  if (e == cudaSuccess) e = cudaFuncSetAttribute(tg::merge_kernel<TG_DTYPE_F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, tg::kMergeSmem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(tg::merge_kernel<TG_DTYPE_BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, tg::kMergeSmem);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();  // calls may come on any stream
  if (e != cudaSuccess) {
    tg_beam_destroy(h);
    return tg::set_cuda_error(e, "tg_beam_create");
  }
  *out = h;
  return TG_OK;
}

int32_t tg_beam_device_status(tg_beam* h, uint32_t* out_bits) {
  if (!h || !out_bits) return set_error(TG_ERR_INVALID_ARG, "NULL argument");
  tg::CurrentDevice g(h->device);
  TG_TRY(cudaDeviceSynchronize());
  TG_TRY(cudaMemcpy(out_bits, h->status, 4, cudaMemcpyDeviceToHost));
  TG_TRY(cudaMemset(h->status, 0, 4));
  TG_TRY(cudaDeviceSynchronize());
  return TG_OK;
}

int32_t tg_beam_select(tg_beam* h, const void* logits, int32_t dtype, int64_t row_stride, int32_t batch, const float* scores,
                       const int32_t* finished, const uint32_t* mask_table, int32_t num_states, const int32_t* state_id,
                       int32_t eos_id, int32_t pad_id, const int32_t* history, const int32_t* history_len,
                       int32_t history_stride, int32_t* out_parent, int32_t* out_token, float* out_score,
                       int32_t* out_finished, int32_t* out_history, int32_t* out_history_len, void* stream) {
  if (!h) return set_error(TG_ERR_INVALID_ARG, "beam handle is NULL");
  if (dtype != TG_DTYPE_F32 && dtype != TG_DTYPE_BF16) return set_error(TG_ERR_INVALID_ARG, "dtype must be TG_DTYPE_F32 or TG_DTYPE_BF16");
  if (batch < 0 || batch > h->max_batch) return set_error(TG_ERR_INVALID_ARG, "batch outside [0, max_batch]");
  if (batch == 0) return TG_OK;
  if (!logits || !scores || !out_parent || !out_token || !out_score)
    return set_error(TG_ERR_INVALID_ARG, "logits, scores, out_parent, out_token and out_score are required");
  if (row_stride < h->vocab) return set_error(TG_ERR_INVALID_ARG, "row_stride < vocab");
  if (state_id && (!mask_table || num_states <= 0)) return set_error(TG_ERR_INVALID_ARG, "state_id given without mask_table / num_states");
  if (eos_id < -1 || eos_id >= h->vocab || pad_id < 0 || pad_id >= h->vocab) return set_error(TG_ERR_INVALID_ARG, "eos_id outside [-1, vocab) or pad_id outside [0, vocab)");
  if (history && (!history_len || !out_history || !out_history_len || history_stride <= 0))
    return set_error(TG_ERR_INVALID_ARG, "history given without history_len, history_stride, out_history and out_history_len");
  if (history && (history == out_history || history_len == out_history_len)) return set_error(TG_ERR_INVALID_ARG, "out_history must not be history");
  const uintptr_t es = dtype == TG_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % es) return set_error(TG_ERR_INVALID_ARG, "logits is not aligned to its elements");
  tg::CurrentDevice g(h->device);
  tg::BeamArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.vocab = h->vocab;
  a.beams = h->beams;
  a.batch = batch;
  a.parts = tg::parts_of(h->vocab, dtype == TG_DTYPE_F32 ? 4 : 8, batch * h->beams);
  a.num_states = num_states;
  a.mask_words = (h->vocab + 31) / 32;
  a.eos_id = eos_id;
  a.pad_id = pad_id;
  a.history_stride = history_stride;
  a.scores = scores;
  a.finished = finished;
  a.mask_table = mask_table;
  a.state_id = state_id;
  a.history = history;
  a.history_len = history_len;
  a.out_parent = out_parent;
  a.out_token = out_token;
  a.out_score = out_score;
  a.out_finished = out_finished;
  a.out_history = out_history;
  a.out_history_len = out_history_len;
  a.heads = h->heads;
  a.candidates = h->candidates;
  a.status = h->status;
  static_assert((TG_MAX_VOCAB - 1) / (tg::kThreads * tg::kVecs * 4 * tg::kMaxGroups) + 1 <= tg::kMergeSmem / (TG_MAX_BEAMS * TG_MAX_BEAMS * 8 + TG_MAX_BEAMS * sizeof(tg::PartHead)),
                "the parts that the longest row asks for fit the merge");
  // the merge holds beams x parts x beams keys, and the parts' heads, in shared memory
  const size_t per_part = static_cast<size_t>(a.beams) * a.beams * 8 + a.beams * sizeof(tg::PartHead), most = tg::kMergeSmem / per_part;
  if (static_cast<size_t>(a.parts) > most) a.parts = static_cast<int>(most);
  const size_t smem = a.parts * per_part;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(a.parts, batch * h->beams);
  if (dtype == TG_DTYPE_F32) {
    TG_TRY(tg::launch_after(state_id ? tg::scan_kernel<TG_DTYPE_F32, true> : tg::scan_kernel<TG_DTYPE_F32, false>, grid, tg::kThreads, 0, st, 1, a));
    TG_TRY(tg::launch_after(tg::merge_kernel<TG_DTYPE_F32>, dim3(batch), tg::kMergeThreads, smem, st, 1, a));
  } else {
    TG_TRY(tg::launch_after(state_id ? tg::scan_kernel<TG_DTYPE_BF16, true> : tg::scan_kernel<TG_DTYPE_BF16, false>, grid, tg::kThreads, 0, st, 1, a));
    TG_TRY(tg::launch_after(tg::merge_kernel<TG_DTYPE_BF16>, dim3(batch), tg::kMergeThreads, smem, st, 1, a));
  }
  return TG_OK;
}

}  // extern "C"
