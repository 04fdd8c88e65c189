// tg_cache.cu -- bookkeeping of the paged key/value cache: pages reserved, shared,
// copied on write, freed, and a drafted tree's accepted path moved together.
//
// State: lens, counts, tables, refs and a bitmap of the free pages.  Allocation is
// "the lowest-numbered free pages, row after row": the state is then a function of
// the calls alone, whatever order atomics ran in, and a free page needs no list whose
// order could differ.  A bitmap of 128 K pages is 16 KB: one block scans it in
// registers.
//
// What bounds these calls: the bookkeeping is latency, a few dependent loads and block
// scans, 4 to 6 us a launch on B200 (16 rows forked, extended and copied in two small
// layers: 12 us in 3 launches; 64 trees accepted in 32 layers, with truncate and extend:
// 20 us in 5).  The copies are HBM bytes, 2 x (tokens x kv_heads x head_dim x 2 B x 2
// pools x layers): 64 pages in 32 layers, 603 MB, 87 us for fork and extend together,
// 6.9 TB/s; 64 x 512 tokens of 8 heads appended, 268 MB, 43 us, 6.2 TB/s.
#include "tg_cache.h"

#include <climits>
#include <cstring>
#include <new>

#include <cooperative_groups.h>

namespace tg {
namespace {

constexpr int kBlock = 1024;       // threads of the one-block calls
constexpr int kForkBlocks = 8;     // fork: one cluster of this many blocks
constexpr int kCopyThreads = 256;
constexpr int kCopyUnit = 4096;    // bytes a warp copies at a time: 8 x 16 B in flight per lane

__device__ __forceinline__ void after_previous_work() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void report(const CacheView& c, uint32_t bits) {
  if (bits) atomicOr(c.status, bits);
}

// Exclusive prefix sum over the block (kBlock threads); *total = the block's sum.
// `warp_sums`: 33 ints of shared memory, free again after the call.
__device__ int block_prefix(int x, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(~0u, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int s = warp_sums[lane];
    int w = s;
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(~0u, w, d);
      if (lane >= d) w += y;
    }
    warp_sums[lane] = w - s;
    if (lane == 31) warp_sums[32] = w;
  }
  __syncthreads();
  const int r = warp_sums[warp] + inc - x;
  *total = warp_sums[32];
  __syncthreads();
  return r;
}

constexpr int kShort = -1;               // in `first`: a row's copy of this page does not fit
constexpr int kKeeperShort = 1 << 30;    // in `need`: the row would keep such a page (a table row has at most 2^28 pages)

// One block, since rows take pages in order: two prefix sums over the block, one over the
// rows' wishes and one over the bitmap, are all that orders them.  Pages for each row's next
// counts[i] tokens.  Latency, about 6 us with 64 rows.
__global__ void __launch_bounds__(kBlock) extend_kernel(CacheView c, int n, const int32_t* seqs, const int32_t* counts) {
  __shared__ int sums[33];
  __shared__ int n_copies;
  const int tid = threadIdx.x, ps = c.page_size;
  after_previous_work();
  if (tid == 0) n_copies = 0;
  uint32_t bad = 0;
  // the rows' wishes; a partly filled last page learns how many rows of this call would write to it
  for (int i = tid; i < n; i += kBlock) {
    const int s = seqs[i];
    int need = -1, last = -1;
    if (s < 0 || s >= c.max_seqs || atomicExch(&c.claim[s], 1) != 0) {
      bad |= kBadSlot;
    } else {
      const int len = c.lens[s], have = c.counts[s], more = counts[i];
      const int64_t want = (static_cast<int64_t>(len) + more + ps - 1) >> c.page_log2;
      need = 0;
      if (more < 0 || want > c.width) {
        bad |= kBadLength;
      } else if (more > 0) {
        need = want > have ? static_cast<int>(want - have) : 0;
        if (len & (ps - 1)) {
          last = c.tables[static_cast<size_t>(s) * c.width + (len >> c.page_log2)];
          atomicAdd(&c.shared[last], 1);
          atomicMin(&c.first[last], i);
        }
      }
    }
    c.need[i] = need < 0 ? -1 : 2 * need;
    c.last[i] = last;
  }
  __syncthreads();
  // a row copies its last page when others hold it; of the only holders the first keeps it
  int total = 0;
  for (int base = 0; base < n; base += kBlock) {
    const int i = base + tid;
    int takes = 0;
    if (i < n && c.need[i] >= 0) {
      const int last = c.last[i];
      int copy = 0;
      if (last >= 0) {
        const int held = __ldcg(&c.refs[last]);
        copy = !(held == 1 || (__ldcg(&c.shared[last]) == held && __ldcg(&c.first[last]) == i));
      }
      takes = (c.need[i] >> 1) + copy;
      c.need[i] |= copy;
    }
    int sum;
    const int at = block_prefix(takes, sums, &sum);
    if (i < n) c.start[i] = total + at;
    total += sum;
  }
  // the `total` lowest free pages: each thread owns a run of the bitmap's words
  int avail = 0;
  if (total > 0) {  // the same for every thread
    const int words = (c.num_pages + 31) >> 5, per = (words + kBlock - 1) / kBlock;
    const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
    int mine = 0;
    for (int w = w0; w < w1; w++) mine += __popc(__ldcg(&c.free_map[w]));
    int rank = block_prefix(mine, sums, &avail);
    for (int w = w0; w < w1 && rank < total; w++) {
      for (uint32_t m = __ldcg(&c.free_map[w]); m && rank < total; m &= m - 1) c.list[rank++] = (w << 5) + __ffs(m) - 1;
    }
    if (total > avail) {
      // the first of a shared page's only holders keeps it if the others copy it: where a copy
      // does not fit, the page has two holders left and the first, who may not store, is not served either
      for (int i = tid; i < n; i += kBlock) {
        const int need = c.need[i], takes = (need >> 1) + (need & 1);
        if (need > 0 && (need & 1) && c.start[i] + takes > avail) c.first[c.last[i]] = kShort;
      }
      __syncthreads();
      for (int i = tid; i < n; i += kBlock) {
        const int need = c.need[i], last = c.last[i];
        if (need >= 0 && !(need & 1) && last >= 0 && c.first[last] == kShort) c.need[i] = need | kKeeperShort;
      }
    }
    __syncthreads();
    const int given = min(total, avail);
    for (int e = tid; e < given; e += kBlock) {
      int lo = 0, hi = n - 1;  // the last row that starts at or before e has page e
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (c.start[mid] <= e) lo = mid; else hi = mid - 1;
      }
      const int need = c.need[lo], copy = need & 1, k = e - c.start[lo];
      if ((need & kKeeperShort) || c.start[lo] + (need >> 1) + copy > avail) continue;  // the row is not served
      const int s = seqs[lo], p = c.list[e], len = c.lens[s];
      int32_t* row = c.tables + static_cast<size_t>(s) * c.width;
      c.refs[p] = 1;
      atomicAnd(&c.free_map[p >> 5], ~(1u << (p & 31)));
      if (copy && k == 0) {
        const int from = c.last[lo];
        row[len >> c.page_log2] = p;
        atomicSub(&c.refs[from], 1);
        c.copies[atomicAdd(&n_copies, 1)] = make_int4(from, p, len & (ps - 1), 0);
      } else {
        row[c.counts[s] + k - copy] = p;
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < n; i += kBlock) {
    const int need = c.need[i];
    if (need < 0) continue;
    const int s = seqs[i], last = c.last[i], takes = ((need & ~kKeeperShort) >> 1) + (need & 1);
    if (last >= 0) {
      c.shared[last] = 0;
      c.first[last] = INT_MAX;
    }
    if ((need & kKeeperShort) || (takes > 0 && c.start[i] + takes > avail)) bad |= kNoPages;
    else c.counts[s] += need >> 1;
    c.claim[s] = 0;
  }
  if (tid == 0) *c.n_copies = n_copies;
  report(c, bad);
}

// The page copies that extend_kernel listed, all layers: a warp per 4 KB piece of a
// (copy, layer, pool, head)'s tokens, which are contiguous, so that 8 loads of 16 bytes per
// lane are on their way before the first store.  HBM, 6.9 TB/s at 603 MB; 3 us when there
// is nothing to copy.
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(CacheView c) {
  after_previous_work();
  const int n = __ldcg(c.n_copies);
  if (n == 0) return;
  const int lane = threadIdx.x & 31;
  const int row_bytes = c.head_dim * 2, head_bytes = row_bytes << c.page_log2;
  const int pieces = (head_bytes + kCopyUnit - 1) / kCopyUnit;
  const int per_copy = c.layers * 2 * c.kv_heads * pieces;
  const int64_t units = static_cast<int64_t>(n) * per_copy;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCopyThreads / 32);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kCopyThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
    const int4 job = c.copies[u / per_copy];
    int r = static_cast<int>(u % per_copy);
    const int piece = r % pieces;
    r /= pieces;
    const int head = r % c.kv_heads;
    r /= c.kv_heads;
    char* pool = (r & 1) ? c.v : c.k;
    const int64_t layer = static_cast<int64_t>(r >> 1) * c.num_pages;
    const int begin = piece * kCopyUnit, end = min(begin + kCopyUnit, job.z * row_bytes);
    const char* from = pool + ((layer + job.x) * c.kv_heads + head) * head_bytes;
    char* to = pool + ((layer + job.y) * c.kv_heads + head) * head_bytes;
    int4 buf[kCopyUnit / 512];
#pragma unroll
    for (int k = 0; k < kCopyUnit / 512; k++) {
      const int b = begin + (k * 32 + lane) * 16;
      if (b < end) buf[k] = __ldcs(reinterpret_cast<const int4*>(from + b));
    }
#pragma unroll
    for (int k = 0; k < kCopyUnit / 512; k++) {
      const int b = begin + (k * 32 + lane) * 16;
      if (b < end) __stcs(reinterpret_cast<int4*>(to + b), buf[k]);
    }
  }
}

// Whether the page that slot s's length ends in is its alone: a fork shares it until one of
// the two is extended, and what one stored there the other would read.
__device__ __forceinline__ bool owns_end(const CacheView& c, int s, int len) {
  return !(len & (c.page_size - 1)) || c.refs[c.tables[static_cast<size_t>(s) * c.width + (len >> c.page_log2)]] == 1;
}

__device__ __forceinline__ void release_page(const CacheView& c, int p) {
  if (atomicSub(&c.refs[p], 1) == 1) atomicOr(&c.free_map[p >> 5], 1u << (p & 31));
}

// One cluster of 8 blocks: the phases need a barrier over all rows, and 8 SMs' loads are
// enough for tables (6.5 us for 64 rows).  dst[i]'s row becomes src[i]'s.  Every new hold is counted before any
// old one is given back, so no page that stays in use passes through "free"; pages
// that dst holds at the same place already (a common prefix) are not touched.
__global__ void __launch_bounds__(kBlock) fork_kernel(CacheView c, int n, const int32_t* src, const int32_t* dst) {
  auto cluster = cooperative_groups::this_cluster();
  const int threads = kForkBlocks * kBlock, gid = blockIdx.x * kBlock + threadIdx.x;
  after_previous_work();
  uint32_t bad = 0;
  for (int i = gid; i < n; i += threads) {
    const int s = src[i], d = dst[i];
    int4 r = make_int4(0, 0, 0, 0);
    if (d < 0 || d >= c.max_seqs || s < -1 || s >= c.max_seqs) {
      bad |= kBadSlot;
    } else if (atomicExch(&c.claim[d], 1) != 0) {
      bad |= kBadSlot;
    } else {
      const int len = s < 0 ? 0 : c.lens[s];
      r = make_int4((len + c.page_size - 1) >> c.page_log2, c.counts[d], len, 1);
    }
    c.info[i] = r;
  }
  cluster.sync();
  // warps per row: all of them when there are few rows
  const int all = threads / 32, lane = threadIdx.x & 31;
  const int per = n >= all ? 1 : all / n;
  for (int u = gid >> 5; u < n * per; u += all) {
    const int i = u / per;
    const int4 r = __ldcg(&c.info[i]);
    if (!r.w) continue;
    const int32_t* from = c.tables + static_cast<size_t>(max(src[i], 0)) * c.width;
    const int32_t* to = c.tables + static_cast<size_t>(dst[i]) * c.width;
    for (int j = (u % per) * 32 + lane; j < max(r.x, r.y); j += 32 * per) {
      const int p = j < r.x ? from[j] : -1, old = j < r.y ? to[j] : -1;
      c.staged[static_cast<size_t>(i) * c.width + j] = p;
      if (p >= 0 && p != old) atomicAdd(&c.refs[p], 1);
    }
  }
  cluster.sync();
  for (int u = gid >> 5; u < n * per; u += all) {
    const int i = u / per, part = u % per;
    const int4 r = __ldcg(&c.info[i]);
    if (!r.w) continue;
    const int d = dst[i];
    int32_t* to = c.tables + static_cast<size_t>(d) * c.width;
    for (int j = part * 32 + lane; j < max(r.x, r.y); j += 32 * per) {
      const int p = c.staged[static_cast<size_t>(i) * c.width + j], old = j < r.y ? to[j] : -1;
      if (p != old) {
        to[j] = p;
        if (old >= 0) release_page(c, old);
      }
    }
    if (part == 0 && lane == 0) {
      c.lens[d] = r.z;
      c.counts[d] = r.x;
      c.claim[d] = 0;
    }
  }
  report(c, bad);
}

// Lane-parallel: gives back a row's pages from `keep` on.  Taking the count down with
// atomicMin makes each page go back once even if a slot were given twice.
__device__ void release_from(const CacheView& c, int s, int keep, int lane) {
  int had = 0;
  if (lane == 0) had = atomicMin(&c.counts[s], keep);
  had = __shfl_sync(~0u, had, 0);
  int32_t* row = c.tables + static_cast<size_t>(s) * c.width;
  for (int j = keep + lane; j < had; j += 32) {
    const int p = row[j];
    row[j] = -1;
    release_page(c, p);
  }
}

// A warp per row; 4 us.
__global__ void __launch_bounds__(kCopyThreads) truncate_kernel(CacheView c, int n, const int32_t* seqs, const int32_t* lens) {
  const int i = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  after_previous_work();
  if (i >= n) return;
  const int s = seqs[i];
  if (s < 0 || s >= c.max_seqs) {
    if (lane == 0) report(c, kBadSlot);
    return;
  }
  const int len = lens ? lens[i] : 0;
  if (len < 0 || len > c.lens[s]) {
    if (lane == 0) report(c, kBadLength);
    return;
  }
  __syncwarp();
  if (lane == 0) atomicMin(&c.lens[s], len);  // a slot given twice: the shorter, as its pages
  release_from(c, s, (len + c.page_size - 1) >> c.page_log2, lane);
}

__global__ void __launch_bounds__(kCopyThreads) commit_kernel(CacheView c, int n, const int32_t* seqs, const int32_t* counts) {
  const int i = blockIdx.x * kCopyThreads + threadIdx.x;
  after_previous_work();
  if (i >= n) return;
  const int s = seqs[i], more = counts[i];
  if (s < 0 || s >= c.max_seqs) {
    report(c, kBadSlot);
    return;
  }
  if (more < 0) {
    report(c, kBadLength);
    return;
  }
  // checked and stored at once: a slot given twice must not pass its pages, whose ids later
  // calls follow up to the length.  A failed exchange means that another row advanced.
  const int64_t room = static_cast<int64_t>(c.counts[s]) << c.page_log2;
  for (int len = __ldcg(&c.lens[s]);;) {
    if (static_cast<int64_t>(len) + more > room) {
      report(c, kNotReserved);
      return;
    }
    const int now = atomicCAS(&c.lens[s], len, len + more);
    if (now == len) return;
    len = now;
  }
}

struct Tokens {  // [n, tokens, kv_heads, head_dim]: strides in bytes
  const char* p;
  int64_t row, token, head;
};

// A thread per 16 bytes of a token's keys and values; kAligned: their rows are 16-byte
// aligned, else they are read by elements.
template <bool kAligned>
__global__ void __launch_bounds__(kCopyThreads) append_kernel(CacheView c, int layer, const int32_t* seqs, const int32_t* counts,
                                                              int tokens, Tokens k, Tokens v) {
  const int i = blockIdx.y, cols = c.head_dim >> 3;
  after_previous_work();
  const int s = seqs[i];
  if (s < 0 || s >= c.max_seqs) {
    if (threadIdx.x == 0 && blockIdx.x == 0) report(c, kBadSlot);
    return;
  }
  int count = counts ? counts[i] : tokens;
  const int64_t room = (static_cast<int64_t>(c.counts[s]) << c.page_log2) - c.lens[s];
  uint32_t bad = 0;
  if (count < 0 || count > tokens) {
    bad |= kBadLength;
    count = 0;
  }
  if (count > room) {
    bad |= kNotReserved;
    count = static_cast<int>(room);
  }
  if (count > 0 && !owns_end(c, s, c.lens[s])) {
    bad |= kNotReserved;
    count = 0;
  }
  if (threadIdx.x == 0 && blockIdx.x == 0) report(c, bad);
  const int64_t work = static_cast<int64_t>(count) * c.kv_heads * cols, step = static_cast<int64_t>(gridDim.x) * kCopyThreads;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x; u < work; u += step) {
    const int col = static_cast<int>(u % cols), head = static_cast<int>(u / cols % c.kv_heads);
    const int64_t t = u / cols / c.kv_heads;
    const int64_t pos = c.lens[s] + t;
    const int64_t page = c.tables[static_cast<size_t>(s) * c.width + (pos >> c.page_log2)] + static_cast<int64_t>(layer) * c.num_pages;
    const int64_t at = (((page * c.kv_heads + head) << c.page_log2) + (pos & (c.page_size - 1))) * c.head_dim * 2 + col * 16;
    const char* a = k.p + i * k.row + t * k.token + head * k.head + col * 16;
    const char* b = v.p + i * v.row + t * v.token + head * v.head + col * 16;
    int4 x, y;
    if (kAligned) {
      x = *reinterpret_cast<const int4*>(a);
      y = *reinterpret_cast<const int4*>(b);
    } else {
      uint16_t e[8], f[8];
#pragma unroll
      for (int m = 0; m < 8; m++) {
        e[m] = reinterpret_cast<const uint16_t*>(a)[m];
        f[m] = reinterpret_cast<const uint16_t*>(b)[m];
      }
      memcpy(&x, e, 16);
      memcpy(&y, f, 16);
    }
    *reinterpret_cast<int4*>(c.k + at) = x;
    *reinterpret_cast<int4*>(c.v + at) = y;
  }
}

// A warp per row, which holds the tree in its lanes: a step of the walk is a shuffle and two
// ballots (5.5 us for 64 trees of 64 nodes).  The walk, the length, the surplus pages; the moves are resolved to
// (page, slot) before any page goes back and left to move_kernel.
__global__ void __launch_bounds__(kCopyThreads) accept_kernel(CacheView c, int n, const int32_t* seqs, int nodes, const int32_t* n_nodes,
                                                              const int32_t* parents, const int32_t* tokens, const int32_t* ids,
                                                              int32_t* out_ids, int32_t* out_n) {
  const int i = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  after_previous_work();
  if (i >= n) return;
  const int s = seqs[i];
  int count = n_nodes ? n_nodes[i] : nodes;
  uint32_t bad = 0;
  // a slot given twice is served once: of two warps on one row, one would follow page
  // ids that the other gives back.  move_kernel ends the claim.
  int claimed = 1;
  if (lane == 0 && s >= 0 && s < c.max_seqs) claimed = atomicExch(&c.claim[s], 1);
  if (__shfl_sync(~0u, claimed, 0) != 0) {
    bad |= kBadSlot;
    count = 0;
  } else if (count < 0 || count > nodes) {
    bad |= kBadTree;
    count = 0;
  }
  const int64_t base = static_cast<int64_t>(i) * nodes;
  // lane l holds nodes l and l + 32
  int up[2], tok[2], id[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int j = lane + 32 * h;
    const bool in = j < count;
    up[h] = in && j > 0 ? parents[base + j] : -1;
    tok[h] = in ? tokens[base + j] : 0;
    id[h] = in ? ids[base + j] : 0;
  }
  int len = 0;
  if (!bad) {
    len = c.lens[s];
    if (static_cast<int64_t>(len) + count > static_cast<int64_t>(c.counts[s]) << c.page_log2 || (count > 0 && !owns_end(c, s, len))) {
      bad |= kNotReserved;
      count = 0;
    }
  }
  // a child has a higher number than its parent, so the path ascends and ends
  int taken = 0, mine[2] = {-1, -1}, out[2] = {-1, -1};  // the path's entries l and l + 32, and their ids
  for (int at = count > 0 ? 0 : -1; at >= 0;) {
    const int want = __shfl_sync(~0u, at < 32 ? id[0] : id[1], at & 31);
    if (lane == (taken & 31)) {
      mine[taken >> 5] = at;
      out[taken >> 5] = want;
    }
    taken++;
    const unsigned lo = __ballot_sync(~0u, up[0] == at && lane > at && tok[0] == want);
    const unsigned hi = __ballot_sync(~0u, up[1] == at && lane + 32 > at && tok[1] == want);
    at = lo ? __ffs(lo) - 1 : hi ? __ffs(hi) + 31 : -1;
  }
  int moved = 0;
  if (!bad) {  // else the row stays as it is, what it has reserved included
    const int32_t* row = c.tables + static_cast<size_t>(s) * c.width;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int j = lane + 32 * h;
      // the moves form the path's tail: once a node is off its place, all after it are
      const bool off = mine[h] >= 0 && mine[h] != j;
      const unsigned m = __ballot_sync(~0u, off);
      if (off) {
        const int from = len + mine[h], to = len + j;
        c.moves[static_cast<size_t>(i) * TG_MAX_TREE_NODES + moved + __popc(m & ((1u << lane) - 1))] =
            make_int4(row[from >> c.page_log2], from & (c.page_size - 1), row[to >> c.page_log2], to & (c.page_size - 1));
      }
      moved += __popc(m);
    }
    __syncwarp();
    if (lane == 0) c.lens[s] = len + taken;
    release_from(c, s, (len + taken + c.page_size - 1) >> c.page_log2, lane);
  }
  if (lane == 0) {
    c.n_moves[i] = moved;
    out_n[i] = taken;
    report(c, bad);
  }
#pragma unroll
  for (int h = 0; h < 2; h++)
    if (lane + 32 * h < nodes) out_ids[base + lane + 32 * h] = out[h];
}

// A thread per 16-byte column of a (row, layer, pool, head): it moves that column of
// the path's tokens in ascending order, up to 8 loads ahead of the stores.  The path
// ascends, so a source is never a place stored to by an earlier move of the same
// thread, and no other thread touches the column.  4 us for a few rows, 10 us for 64 trees
// in 32 layers.
__global__ void __launch_bounds__(kCopyThreads) move_kernel(CacheView c, const int32_t* seqs) {
  after_previous_work();
  const int i = blockIdx.y, n = c.n_moves[i];
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const int s = seqs[i];
    if (s >= 0 && s < c.max_seqs) c.claim[s] = 0;
  }
  if (n == 0) return;
  const int cols = c.head_dim >> 3;
  const int u = blockIdx.x * kCopyThreads + threadIdx.x;
  if (u >= c.layers * 2 * c.kv_heads * cols) return;
  const int col = u % cols, head = u / cols % c.kv_heads, r = u / cols / c.kv_heads;
  char* pool = ((r & 1) ? c.v : c.k) + col * 16;
  const int64_t layer = static_cast<int64_t>(r >> 1) * c.num_pages;
  const int4* jobs = c.moves + static_cast<size_t>(i) * TG_MAX_TREE_NODES;
  for (int j = 0; j < n; j += 8) {
    int4 buf[8];
#pragma unroll
    for (int m = 0; m < 8; m++)
      if (j + m < n) {
        const int4 job = jobs[j + m];
        buf[m] = *reinterpret_cast<const int4*>(pool + ((((layer + job.x) * c.kv_heads + head) << c.page_log2) + job.y) * c.head_dim * 2);
      }
#pragma unroll
    for (int m = 0; m < 8; m++)
      if (j + m < n) {
        const int4 job = jobs[j + m];
        *reinterpret_cast<int4*>(pool + ((((layer + job.z) * c.kv_heads + head) << c.page_log2) + job.w) * c.head_dim * 2) = buf[m];
      }
  }
}

// A warp per tree.  Bits by pointer jumping: after k rounds a node's set holds its
// next 2^k ancestors; 6 rounds cover 64 nodes.
__global__ void __launch_bounds__(kCopyThreads) masks_kernel(int n, int nodes, const int32_t* n_nodes, const int32_t* parents, uint64_t* masks) {
  const int i = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  after_previous_work();
  if (i >= n) return;
  const int count = n_nodes ? min(max(n_nodes[i], 0), nodes) : nodes;
  uint64_t set[2];
  int up[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int j = lane + 32 * h;
    set[h] = j < count ? 1ull << j : 0;
    const int p = j > 0 && j < count ? parents[static_cast<int64_t>(i) * nodes + j] : -1;
    up[h] = p < j ? p : -1;
  }
  for (int round = 0; round < 6; round++) {
    uint64_t s[2];
    int u[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int at = up[h] < 0 ? 0 : up[h];
      const uint64_t s0 = __shfl_sync(~0u, set[0], at & 31), s1 = __shfl_sync(~0u, set[1], at & 31);
      const int u0 = __shfl_sync(~0u, up[0], at & 31), u1 = __shfl_sync(~0u, up[1], at & 31);
      s[h] = up[h] < 0 ? 0 : at < 32 ? s0 : s1;
      u[h] = up[h] < 0 ? -1 : at < 32 ? u0 : u1;
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      set[h] |= s[h];
      up[h] = u[h];
    }
  }
#pragma unroll
  for (int h = 0; h < 2; h++)
    if (lane + 32 * h < nodes) masks[static_cast<int64_t>(i) * nodes + lane + 32 * h] = set[h];
}

int32_t check_rows(const tg_cache* c, int32_t n) {
  if (!c) return set_error(TG_ERR_INVALID_ARG, "cache is NULL");
  if (n < 0 || n > c->view.max_seqs) return set_error(TG_ERR_INVALID_ARG, "n outside [0, max_seqs]");
  return TG_OK;
}

int blocks_of_warps(int n) { return (n + kCopyThreads / 32 - 1) / (kCopyThreads / 32); }

}  // namespace
}  // namespace tg

using tg::set_error;

extern "C" {

int32_t tg_cache_destroy(tg_cache* c) {
  if (!c) return TG_OK;
  {
    tg::CurrentDevice g(c->device);
    if (c->arena) cudaFree(c->arena);
    if (c->partial) cudaFree(c->partial);
  }
  delete c;
  return TG_OK;
}

int32_t tg_cache_create(int32_t device, const tg_cache_config* config, void* k_pool, void* v_pool, tg_cache** out) {
  if (!out) return set_error(TG_ERR_INVALID_ARG, "out is NULL");
  *out = nullptr;
  if (!config || !k_pool || !v_pool) return set_error(TG_ERR_INVALID_ARG, "config, k_pool and v_pool are required");
  const tg_cache_config& f = *config;
  if (f.layers <= 0 || f.kv_heads <= 0 || f.num_pages <= 0 || f.max_seqs <= 0 || f.max_pages_per_seq <= 0)
    return set_error(TG_ERR_INVALID_ARG, "layers, kv_heads, num_pages, max_seqs and max_pages_per_seq must be positive");
  if (f.dtype != TG_DTYPE_BF16 && f.dtype != TG_DTYPE_F16) return set_error(TG_ERR_UNSUPPORTED, "dtype must be TG_DTYPE_BF16 or TG_DTYPE_F16");
  if (f.head_dim < 8 || f.head_dim > 128 || f.head_dim % 8) return set_error(TG_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 in [8, 128]");
  if (f.page_size < 8 || f.page_size > 256 || (f.page_size & (f.page_size - 1)))
    return set_error(TG_ERR_UNSUPPORTED, "page_size must be a power of two in [8, 256]");
  // limits of the 32-bit page, token and copy indices (byte offsets are 64-bit)
  const int64_t seqs = f.max_seqs, width = f.max_pages_per_seq, pages = f.num_pages;
  if (seqs > 65535 || seqs * (width + 1) > INT32_MAX || width * f.page_size > INT32_MAX || pages > (1 << 24) ||
      pages * f.layers * f.kv_heads > INT32_MAX || static_cast<int64_t>(f.layers) * 2 * f.kv_heads * 16 > INT32_MAX || f.kv_heads > 65535)
    return set_error(TG_ERR_UNSUPPORTED, "cache beyond the limits: 65535 slots, 2^24 pages, 2^31 table entries, tokens per row and layers x pages x kv_heads");
  if ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15)
    return set_error(TG_ERR_INVALID_ARG, "k_pool and v_pool must be 16-byte aligned");
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) return set_error(TG_ERR_NO_DEVICE, "CUDA device not present");
  tg::CurrentDevice g(device);
  tg_cache* c = new (std::nothrow) tg_cache();
  if (!c) return set_error(TG_ERR_CUDA, "out of host memory");
  c->device = device;
  c->dtype = f.dtype;
  tg::CacheView& v = c->view;
  v.layers = f.layers;
  v.kv_heads = f.kv_heads;
  v.head_dim = f.head_dim;
  v.page_size = f.page_size;
  while ((1 << v.page_log2) < f.page_size) v.page_log2++;
  v.num_pages = f.num_pages;
  v.max_seqs = f.max_seqs;
  v.width = f.max_pages_per_seq;
  v.k = static_cast<char*>(k_pool);
  v.v = static_cast<char*>(v_pool);
  const size_t words = (pages + 31) / 32;
  size_t size = 0;
  const auto place = [&size](size_t bytes) {
    const size_t at = size;
    size += (bytes + 255) & ~static_cast<size_t>(255);
    return at;
  };
  const size_t lens = place(seqs * 4), counts = place(seqs * 4), claim = place(seqs * 4), n_copies = place(8), status = place(4),
               shared = place(pages * 4), refs = place(pages * 4), zeros = size,  // 0 up to here
               tables = place(seqs * width * 4), start = place(seqs * 4), need = place(seqs * 4), last = place(seqs * 4),
               list = place(pages * 4), copies = place(seqs * 16), info = place(seqs * 16), staged = place(seqs * width * 4),
               moves = place(seqs * TG_MAX_TREE_NODES * 16), n_moves = place(seqs * 4), first = place(pages * 4), free_map = place(words * 4);
  cudaError_t e = cudaDeviceGetAttribute(&c->sms, cudaDevAttrMultiProcessorCount, device);
  if (e == cudaSuccess) e = cudaMalloc(&c->arena, size);
  if (e == cudaSuccess) {
    char* a = static_cast<char*>(c->arena);
    const auto ints = [a](size_t at) { return reinterpret_cast<int32_t*>(a + at); };
    v.lens = ints(lens), v.counts = ints(counts), v.claim = ints(claim), v.n_copies = ints(n_copies);
    v.status = reinterpret_cast<uint32_t*>(a + status);
    v.shared = ints(shared), v.refs = ints(refs), v.tables = ints(tables), v.start = ints(start), v.need = ints(need), v.last = ints(last);
    v.list = ints(list), v.staged = ints(staged), v.n_moves = ints(n_moves), v.first = ints(first);
    v.copies = reinterpret_cast<int4*>(a + copies), v.info = reinterpret_cast<int4*>(a + info), v.moves = reinterpret_cast<int4*>(a + moves);
    v.free_map = reinterpret_cast<uint32_t*>(a + free_map);
    e = cudaMemset(a, 0, zeros);
    if (e == cudaSuccess) e = cudaMemset(v.tables, 0xff, seqs * width * 4);
    if (e == cudaSuccess) e = cudaMemset(v.first, 0x7f, pages * 4);  // 0x7f7f7f7f: past every row
    if (e == cudaSuccess) e = cudaMemset(v.free_map, 0xff, words * 4);
    if (e == cudaSuccess && pages % 32) {
      const uint32_t tail = (1u << (pages % 32)) - 1;
      e = cudaMemcpy(v.free_map + words - 1, &tail, 4, cudaMemcpyHostToDevice);
    }
    if (e == cudaSuccess) e = cudaDeviceSynchronize();  // calls may come on any stream
  }
  if (e != cudaSuccess) {
    tg_cache_destroy(c);
    return tg::set_cuda_error(e, "tg_cache_create");
  }
  const int32_t rc = tg::tree_setup(c);
  if (rc != TG_OK) {
    tg_cache_destroy(c);
    return rc;
  }
  *out = c;
  return TG_OK;
}

int32_t tg_cache_get_state(tg_cache* c, tg_cache_state* out) {
  if (!c || !out) return set_error(TG_ERR_INVALID_ARG, "NULL argument");
  *out = tg_cache_state{c->view.lens, c->view.counts, c->view.tables, c->view.refs};
  return TG_OK;
}

int32_t tg_cache_device_status(tg_cache* c, uint32_t* out_bits) {
  if (!c || !out_bits) return set_error(TG_ERR_INVALID_ARG, "NULL argument");
  tg::CurrentDevice g(c->device);
  TG_TRY(cudaDeviceSynchronize());
  TG_TRY(cudaMemcpy(out_bits, c->view.status, 4, cudaMemcpyDeviceToHost));
  TG_TRY(cudaMemset(c->view.status, 0, 4));
  TG_TRY(cudaDeviceSynchronize());  // cleared before the next call on any stream
  return TG_OK;
}

int32_t tg_cache_extend(tg_cache* c, int32_t n, const int32_t* seqs, const int32_t* counts, void* stream) {
  if (const int32_t rc = tg::check_rows(c, n)) return rc;
  if (n == 0) return TG_OK;
  if (!seqs || !counts) return set_error(TG_ERR_INVALID_ARG, "seqs and counts are required");
  tg::CurrentDevice g(c->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TG_TRY(tg::launch_after(tg::extend_kernel, dim3(1), tg::kBlock, 0, st, 1, c->view, n, seqs, counts));
  TG_TRY(tg::launch_after(tg::copy_kernel, dim3(c->sms * 4), tg::kCopyThreads, 0, st, 1, c->view));
  return TG_OK;
}

int32_t tg_cache_fork(tg_cache* c, int32_t n, const int32_t* src, const int32_t* dst, void* stream) {
  if (const int32_t rc = tg::check_rows(c, n)) return rc;
  if (n == 0) return TG_OK;
  if (!src || !dst) return set_error(TG_ERR_INVALID_ARG, "src and dst are required");
  tg::CurrentDevice g(c->device);
  TG_TRY(tg::launch_after(tg::fork_kernel, dim3(tg::kForkBlocks), tg::kBlock, 0, static_cast<cudaStream_t>(stream), tg::kForkBlocks, c->view, n, src, dst));
  return TG_OK;
}

int32_t tg_cache_truncate(tg_cache* c, int32_t n, const int32_t* seqs, const int32_t* lens, void* stream) {
  if (const int32_t rc = tg::check_rows(c, n)) return rc;
  if (n == 0) return TG_OK;
  if (!seqs) return set_error(TG_ERR_INVALID_ARG, "seqs is required");
  tg::CurrentDevice g(c->device);
  TG_TRY(tg::launch_after(tg::truncate_kernel, dim3(tg::blocks_of_warps(n)), tg::kCopyThreads, 0, static_cast<cudaStream_t>(stream), 1, c->view, n, seqs, lens));
  return TG_OK;
}

int32_t tg_cache_commit(tg_cache* c, int32_t n, const int32_t* seqs, const int32_t* counts, void* stream) {
  if (const int32_t rc = tg::check_rows(c, n)) return rc;
  if (n == 0) return TG_OK;
  if (!seqs || !counts) return set_error(TG_ERR_INVALID_ARG, "seqs and counts are required");
  tg::CurrentDevice g(c->device);
  TG_TRY(tg::launch_after(tg::commit_kernel, dim3((n + tg::kCopyThreads - 1) / tg::kCopyThreads), tg::kCopyThreads, 0, static_cast<cudaStream_t>(stream), 1, c->view, n, seqs, counts));
  return TG_OK;
}

int32_t tg_cache_append(tg_cache* c, int32_t layer, int32_t n, const int32_t* seqs, const int32_t* counts, int32_t tokens,
                        const void* k, int64_t k_row, int64_t k_token, int64_t k_head, const void* v, int64_t v_row,
                        int64_t v_token, int64_t v_head, void* stream) {
  if (const int32_t rc = tg::check_rows(c, n)) return rc;
  if (layer < 0 || layer >= c->view.layers) return set_error(TG_ERR_INVALID_ARG, "layer outside [0, layers)");
  if (tokens < 0) return set_error(TG_ERR_INVALID_ARG, "tokens < 0");
  if (n == 0 || tokens == 0) return TG_OK;
  if (!seqs || !k || !v) return set_error(TG_ERR_INVALID_ARG, "seqs, k and v are required");
  tg::CurrentDevice g(c->device);
  const tg::Tokens a{static_cast<const char*>(k), k_row * 2, k_token * 2, k_head * 2};
  const tg::Tokens b{static_cast<const char*>(v), v_row * 2, v_token * 2, v_head * 2};
  const bool aligned = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | static_cast<uintptr_t>(a.row | a.token | a.head | b.row | b.token | b.head)) & 15) == 0;
  const int64_t work = static_cast<int64_t>(tokens) * c->view.kv_heads * (c->view.head_dim / 8);
  const int64_t want = (work + tg::kCopyThreads - 1) / tg::kCopyThreads;
  const dim3 grid(static_cast<unsigned>(want < 4096 ? want : 4096), n);
  TG_TRY(tg::launch_after(aligned ? tg::append_kernel<true> : tg::append_kernel<false>, grid, tg::kCopyThreads, 0, static_cast<cudaStream_t>(stream), 1, c->view,
                          layer, seqs, counts, tokens, a, b));
  return TG_OK;
}

int32_t tg_cache_accept(tg_cache* c, int32_t n, const int32_t* seqs, int32_t nodes, const int32_t* n_nodes, const int32_t* parents,
                        const int32_t* tokens, const int32_t* ids, int32_t* out_ids, int32_t* out_n, void* stream) {
  if (const int32_t rc = tg::check_rows(c, n)) return rc;
  if (nodes < 1 || nodes > TG_MAX_TREE_NODES) return set_error(TG_ERR_UNSUPPORTED, "nodes outside [1, TG_MAX_TREE_NODES]");
  if (n == 0) return TG_OK;
  if (!seqs || !parents || !tokens || !ids || !out_ids || !out_n)
    return set_error(TG_ERR_INVALID_ARG, "seqs, parents, tokens, ids, out_ids and out_n are required");
  tg::CurrentDevice g(c->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TG_TRY(tg::launch_after(tg::accept_kernel, dim3(tg::blocks_of_warps(n)), tg::kCopyThreads, 0, st, 1, c->view, n, seqs, nodes, n_nodes, parents, tokens, ids, out_ids, out_n));
  const int columns = c->view.layers * 2 * c->view.kv_heads * (c->view.head_dim / 8);
  TG_TRY(tg::launch_after(tg::move_kernel, dim3((columns + tg::kCopyThreads - 1) / tg::kCopyThreads, n), tg::kCopyThreads, 0, st, 1, c->view, seqs));
  return TG_OK;
}

int32_t tg_tree_masks(int32_t n, int32_t nodes, const int32_t* n_nodes, const int32_t* parents, uint64_t* masks, void* stream) {
  if (n < 0) return set_error(TG_ERR_INVALID_ARG, "n < 0");
  if (nodes < 1 || nodes > TG_MAX_TREE_NODES) return set_error(TG_ERR_UNSUPPORTED, "nodes outside [1, TG_MAX_TREE_NODES]");
  if (n == 0) return TG_OK;
  if (!parents || !masks) return set_error(TG_ERR_INVALID_ARG, "parents and masks are required");
  TG_TRY(tg::launch_after(tg::masks_kernel, dim3(tg::blocks_of_warps(n)), tg::kCopyThreads, 0, static_cast<cudaStream_t>(stream), 1, n, nodes, n_nodes, parents, masks));
  return TG_OK;
}

}  // extern "C"
