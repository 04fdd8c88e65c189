// tg_tree.cu -- attention of drafted nodes over a paged cache (tg_tree_attention).
//
//   s_ij = scale q_i . k_j over the cached tokens and the nodes that i sees,
//   o_i = sum_j 2^(c s_ij - t_i) v_j / sum_j 2^(c s_ij - t_i),  c = scale log2 e
// in one pass over the keys with a running bound t_i of the row's maximum.
//
// Rows.  All query heads of a key head and all nodes read the same keys, so they form
// the rows of one matrix: row = node * group + head in group.  A work item is (sequence,
// key head, block of rows); its tiles are the nodes themselves (up to 64 keys, tile 0)
// and 128 cached tokens each.  Keys and values are read once per item; a single
// token with 4 heads per key head uses 4 of a tile's 128 rows, which costs no time while
// the bytes bound it (128 rows need 1050 tensor cycles a tile, its 64 KB 2800).
//
// Split.  The tiles of all items, in order, are cut into equal runs, one per block, one
// block per SM: any mix of lengths is balanced to a tile.  An item that is cut
// leaves (t, sum, unnormalised o) of its runs in a workspace, and join_kernel puts
// them together in the order of the runs: the result does not depend on timing.
//
// A block.  16 warps with roles that meet at mbarriers only:
//   8       pages by tiled TMA into a ring of 128-byte-swizzled slots, 128 keys or values each
//   9       one lane issues tcgen05.mma: S = Q K^T into TMEM, O += P V with P read from TMEM
//   0-7     two groups that turn S into P, a thread per row, so no row needs a shuffle; they
//           work on two S buffers: on two blocks of 128 rows of the same tile when the item
//           has more than 128 rows (kWide), else on alternate tiles of the same rows, joined
//           at the item's end.  While one group exponentiates, the tensor cores work for
//           the other
//   10, 11  walk over the run's segments (the part of an item that is in it), Q and the
//           nodes of a segment ahead, the nodes also into the cache
//   12-15   join a segment's two groups and write its rows, while the others go on
//
// Bound and figures (B200; 6.5 TB/s and 1.65 PFLOP/s by the card's own copy and GEMM; in
// bursts of some ms, and in brackets over a second of calls, which the card runs slower):
//   HBM for decoding: 64 sequences, 1 node, 115 (130) us for 622 MB, 5.4 TB/s (4.8).  Pages
//   below 64 tokens cost more: the copy engine takes about 75 cycles a box and a box is a page's
//   part of a tile (16,000 tokens, 32 sequences: 93 us, in pages of 16 118, of 8 153)
//   the chain S -> P -> O -> S of a group for many rows: 4300 cycles a tile, of which the
//   weights take 2400 (the exponentials' unit 1024 of them), the products 770, and the waits
//   between warps the rest: 1 sequence, 64 nodes x 4 heads, 95 (105) us, 0.72 PFLOP/s (0.66)
//   the card's power limit for the largest call (64 sequences, 16 nodes): 240 to 267 (281) us,
//   by the clock that the card holds, 1.66 to 1.78 GHz of 1.96
//   latency for small calls: 15 us, of which join_kernel's launch takes 3
// Tried and slower: exponentials of 32 scores beside the next 32's maxima (one vote more a
// half tile: +5%), a tile's loop unrolled with more registers (the code left the
// instruction caches: twice as slow), runs handed out in small pieces by a counter.
//
// Rounding: S, the sums and O are fp32; P is rounded to the cache's type for the tensor
// cores (the products with V take 16-bit operands), relative 2^-8 (bf16) or 2^-11
// (f16, down to 2^-21 of the row's largest weight, below that to 2^-32 of it) of a weight, and
// the output once.  t moves only when a row's maximum exceeds its first by more than 8, so P
// stays below 2^8 (f16: 2^15) and O is rarely rescaled.
#include "tg_cache.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

namespace tg {
namespace {

constexpr int kThreads = 512;    // 8 softmax warps, a TMA, an issuing and two loading warps, 4 that write results
constexpr int kTile = 128;       // cached tokens of a tile, rows of a row block
constexpr int kTreeTile = TG_MAX_TREE_NODES;
constexpr int kWaitLimit = 1 << 24;
constexpr long long kWaitCycles = 1ll << 31;
constexpr float kSlack = 8.0f;   // log2 of how far P may exceed its first maximum
// log2 of that: f16 weights use the type's range, since those below 2^-14 lose bits and those
// below 2^-25 are 0.  2^(7 + 8) is below its largest value; a row's largest weight is at
// least 2^7, so bits are lost below 2^-21 of it, all of a weight below 2^-32.
template <bool kBf16>
constexpr float kFirst = kBf16 ? 0.0f : 7.0f;
constexpr float kLog2e = 1.44269504f;

// x / group by ceil(2^32 / group) (0: group 1): exact while x group^2 < 2^32, as rows below
// 64 x group and groups up to 256 are.
__device__ __forceinline__ int divide(int x, uint32_t inverse) { return inverse ? static_cast<int>(__umulhi(x, inverse)) : x; }

struct Rows {  // [n, nodes, heads, head_dim]: strides in elements
  const uint16_t* p;
  int64_t row, node, head;
};

struct TreeArgs {
  int32_t layer, n, nodes, q_heads, group, blocks, min_tiles, vec;  // vec: all rows are 16-byte aligned
  uint32_t group_inverse;  // ceil(2^32 / group)
  int32_t q_rows, tree_rows, slots;  // shared memory: rows of a row block, of the nodes' tile, ring slots
  int32_t buffers;                   // of Q and the nodes: 1 or 2
  int32_t q_box;                     // nodes of a box of Q's tensor map; 0: Q comes by 16-byte copies
  uint32_t ring_block, ring_group;   // bytes from one 64-column block of a slot to the next, from 8 tokens to the next 8
  const int32_t* seqs;
  const int32_t* n_nodes;
  const uint64_t* masks;
  Rows q, k, v;
  float scale;
  uint16_t* out;
  float* out_lse;
  struct CutItem* cuts;    // [blocks of the grid] for join_kernel
  float* partial;          // [runs, 2] parts of items (see part_floats)
};

// An item that runs cut, written by the block whose run has its first tile: its parts are
// `part`, then the first ones of the runs after that up to `last`.
struct CutItem {
  int32_t b, head, block, nodes;  // b < 0: none in this run
  int32_t part, last;
};

// ---- PTX -----------------------------------------------------------------------------

__device__ __forceinline__ void after_previous_work() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two floats an instruction.
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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_poll(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// The same from lane 0 alone, by predicate: the warp stays together.
__device__ __forceinline__ bool bar_poll_lane0(uint32_t bar, uint32_t parity, uint32_t lane) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.eq.u32 q, %3, 0;\n mov.u32 %0, 0;\n @q mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @q selp.u32 %0, 1, 0, p;\n}"
      : "=&r"(ok)
      : "r"(bar), "r"(parity), "r"(lane)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void tma_load(uint32_t to, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %4, %5, %6}], [%2];" ::"r"(to), "l"(map), "r"(bar), "r"(x), "r"(0),
      "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_load_q(uint32_t to, const CUtensorMap* map, uint32_t bar, int x, int head, int node, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(to), "l"(map), "r"(bar), "r"(x), "r"(head),
      "r"(node), "r"(b)
      : "memory");
}
// Bytes that the phase waits for, beside its arrivals.
__device__ __forceinline__ void bar_more_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

#define TG_R32(v, o) \
  "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7]), "=r"(v[o + 8]), "=r"(v[o + 9]), \
      "=r"(v[o + 10]), "=r"(v[o + 11]), "=r"(v[o + 12]), "=r"(v[o + 13]), "=r"(v[o + 14]), "=r"(v[o + 15]), "=r"(v[o + 16]), "=r"(v[o + 17]), "=r"(v[o + 18]), \
      "=r"(v[o + 19]), "=r"(v[o + 20]), "=r"(v[o + 21]), "=r"(v[o + 22]), "=r"(v[o + 23]), "=r"(v[o + 24]), "=r"(v[o + 25]), "=r"(v[o + 26]), "=r"(v[o + 27]), \
      "=r"(v[o + 28]), "=r"(v[o + 29]), "=r"(v[o + 30]), "=r"(v[o + 31])
#define TG_REGS32 \
  "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}"

// 32 columns of this warp's 32 lanes, a lane per thread.
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " TG_REGS32 ", [%32];" : TG_R32(v, 0) : "r"(at));
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                 "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(at)
               : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle: start, leading and stride byte
// offsets in 16-byte units, version 1, layout 2.  K-major operands: stride = 8 rows;
// the N-major V: leading = the next 64 columns, stride = 8 keys.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t leading, uint32_t stride) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | static_cast<uint64_t>(leading >> 4) << 16 | static_cast<uint64_t>(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: fp32 result, 16-bit operands (0: f16, 1: bf16), M = 128.
__device__ __forceinline__ constexpr uint32_t instruction(int bf16, int n, int n_major_b) {
  return 1u << 4 | static_cast<uint32_t>(bf16) << 7 | static_cast<uint32_t>(bf16) << 10 | static_cast<uint32_t>(n_major_b) << 16 | static_cast<uint32_t>(n >> 3) << 17 |
         static_cast<uint32_t>(kTile >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add)
               : "memory");
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  if (kBf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The sign bits of the halves of w that are not finite: an exponent of ones carries into it.
template <bool kBf16>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  return kBf16 ? ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
// w with zeros in their place.
template <bool kBf16>
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  const uint32_t odd = odd_halves<kBf16>(w);
  return w & ~((odd >> 15) * 0xffffu);
}
template <bool kBf16>
__device__ __forceinline__ bool not_finite(uint16_t x) {
  return kBf16 ? (x & 0x7f80) == 0x7f80 : (x & 0x7c00) == 0x7c00;
}
template <bool kBf16>
__device__ __forceinline__ float widen(uint16_t x) {
  return kBf16 ? __uint_as_float(static_cast<uint32_t>(x) << 16) : __half2float(__ushort_as_half(x));
}

// ---- the division of the work ---------------------------------------------------------

// Quotient of numbers that are nearly always below 2^32 (the 64-bit division is long).
__device__ __noinline__ int64_t long_quotient(int64_t x, int64_t d) { return x / d; }
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t d) {
  return ((x | d) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(d)) : long_quotient(x, d);
}

// A sequence's part of the work.  An item counts as its tiles and kOverhead more, for
// what a block does once per item: runs are cut in this measure, so that a run of many
// short items has as much to do as one of a few long ones.
constexpr int kOverhead = 2;
struct Seq {
  int slot, len, nodes;  // nodes 0 where the row cannot be served
  int ctx;               // tiles of cached tokens
  int active;            // row blocks with rows
  int per_head;          // measure of a key head's items
  uint32_t bad;
};

template <int kRows>
__device__ __forceinline__ Seq sequence(const CacheView& c, const TreeArgs& a, int b) {
  Seq q;
  q.slot = a.seqs[b];
  q.nodes = a.n_nodes ? a.n_nodes[b] : a.nodes;
  q.bad = 0;
  if (q.nodes < 0 || q.nodes > a.nodes) q.bad |= kBadTree;
  if (q.slot < 0 || q.slot >= c.max_seqs) q.bad |= kBadSlot;
  if (q.bad) q.nodes = 0;
  q.len = q.bad ? 0 : c.lens[q.slot];
  q.ctx = (q.len + kTile - 1) / kTile;
  q.active = (q.nodes * a.group + kRows - 1) / kRows;
  q.per_head = q.active * (q.ctx + 1 + kOverhead) + (a.blocks - q.active) * (1 + kOverhead);
  return q;
}

// Walks over the segments of a run: over [t0, t1) of an item's tiles, item after item.
// A segment may be empty, where a run's end falls into an item's overhead.
template <int kRows>
struct Walk {
  int64_t left;  // what is left of the run from this item on
  int64_t at;    // where the run enters the item, in the sequence's measure
  int into;      // where in the item's measure that is
  int b, head, block, tiles;
  bool fresh;    // a sequence not looked at yet
  Seq q;

  __device__ __forceinline__ void start(int b0, int64_t at0, int64_t count) { b = b0, at = at0, left = count, fresh = true; }
  // Fills in the item.
  __device__ __forceinline__ void enter(const CacheView& c, const TreeArgs& a) {
    if (fresh) q = sequence<kRows>(c, a, b);
    fresh = false;
    head = static_cast<int>(quotient(at, q.per_head));
    int r = static_cast<int>(at - static_cast<int64_t>(head) * q.per_head);
    const int full = q.active * (q.ctx + 1 + kOverhead);
    if (r < full) {
      tiles = q.ctx + 1;
      block = static_cast<uint32_t>(r) / static_cast<uint32_t>(tiles + kOverhead);
      into = r - block * (tiles + kOverhead);
    } else {
      r -= full;
      tiles = 1;
      block = q.active + r / (1 + kOverhead);
      into = r % (1 + kOverhead);
    }
  }
  __device__ int t0() const { return max(0, into - kOverhead); }
  __device__ int t1() const { return static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(tiles), into + left - kOverhead))); }
  // To the next item of the run; false: there is none.
  __device__ __forceinline__ bool advance(const CacheView& c) {
    const int rest = tiles + kOverhead - into;
    if (left <= rest) return false;
    left -= rest;
    at += rest;
    if (at == static_cast<int64_t>(q.per_head) * c.kv_heads) b++, at = 0, fresh = true;
    return true;
  }
};

// The measure of a run.
__device__ __forceinline__ int64_t run_length(int64_t total, int blocks, int min_tiles) {
  const int64_t run = quotient(total + blocks - 1, blocks);
  return run < min_tiles ? min_tiles : run;
}

// ---- shared memory ----------------------------------------------------------------------

// In front the control block, then Q (each row block [64-column blocks][q_rows][128 bytes])
// and the nodes' keys and values ([64-column blocks][tree_rows][128 bytes] each), twice
// in a narrow block that keeps kMinSlots slots then (the next segment's are loaded while
// this one runs), and the ring ([64-column blocks][128][128 bytes] per slot).  Q takes only the rows that the call
// has: the products read 128 rows from its start, and what the rows past the last hold
// reaches only results that nothing reads.  The space saved is ring: bytes in flight.
template <int kDim, bool kWide>
struct Layout {
  static constexpr int kBlocks = kDim / 64;       // 64-column blocks of a row
  static constexpr int kSlot = kTile * kDim * 2;  // 128 keys or values
  static constexpr int kRows = kWide ? 2 * kTile : kTile;
  static constexpr int kBuffers = kWide ? 1 : 2;  // of Q and the nodes at most; of the sets and the sums
};
constexpr int kMaxSlots = 9;
// Keys and values take the slots in turn.  A softmax group waits for the last tile's values
// by parity, which tells a slot's load from the one two before it only if the one before is
// known to have landed.  From 3 slots on that was a load whose product came before the tile's
// scores; of 2 slots all values take the second, and the load before may be under way.
constexpr int kMinSlots = 3;

// A part of an item in the workspace: float4 o[kDim / 4][kRows], float2 (t, sum)[kRows].
template <int kDim, int kRows>
__device__ __forceinline__ constexpr int part_floats() { return kRows * (kDim + 2); }

// A run of tiles of one item, as the walking warp hands it to the others.
struct Segment {
  int32_t b, head, block;         // the item; b < 0: there are no more
  int32_t t0, t1;                 // [t0, t1) of the item's tiles
  int32_t slot, len, nodes;       // the sequence
  int32_t part;                   // the part that its rows make; -1: they are whole
};
constexpr int kSegments = 2;      // in hand: this one and the next

struct Control {
  uint64_t full[kMaxSlots], empty[kMaxSlots], q_full[2], q_empty[2], s_full[2], p_half[2], p_full[2], half_done[2], stats, done, read, drain;
  uint64_t seg_full[kSegments], seg_empty[kSegments];
  uint64_t odd[4][2];  // nodes with a value that is not finite, by segment modulo 4 and loading warp
  int64_t total, run_off;
  Segment seg[kSegments];
  int32_t run_b, give_up;
  uint32_t tmem;
};
// After it, by segment modulo kBuffers: the nodes' sets, and t and sum of each row in each
// group.  All in front of the 1024-byte-aligned tiles, within 3 KB for a wide block, which
// leaves it 4 ring slots with 64 nodes.
struct Sets {
  uint64_t of[TG_MAX_TREE_NODES];
};
struct Sums {
  float t[2][kTile], sum[2][kTile];
};
constexpr int kSetsAt = 512;
static_assert(sizeof(Control) <= kSetsAt, "the control block outgrew its space");
template <int kBuffers>
__host__ __device__ constexpr int control_bytes() {
  return (kSetsAt + kBuffers * static_cast<int>(sizeof(Sets) + sizeof(Sums)) + 1023) / 1024 * 1024;
}
static_assert(control_bytes<1>() == 3072, "a wide block's share");

// A wait gives up after kWaitLimit polls or kWaitCycles cycles (about a second),
// whichever is first.
struct Patience {
  int polls = 0;
  long long since = 0;
  __device__ __forceinline__ bool over() {
    if (++polls == 16) since = clock64();
    return polls > kWaitLimit || (polls > 16 && (polls & 63) == 0 && clock64() - since > kWaitCycles);
  }
};

// The long way of the waits below.  Not inlined, like other rare paths here: the code of
// all roles has to fit the instruction caches (at 140 KB everything ran half as fast).
__device__ __noinline__ bool wait_on(Control* ctl, uint32_t at, uint32_t parity) {
  const uint32_t lane = threadIdx.x & 31;
  for (Patience p;;) {
    if (__any_sync(~0u, bar_poll_lane0(at, parity, lane))) return true;
    if (__any_sync(~0u, *reinterpret_cast<volatile int32_t*>(&ctl->give_up) || p.over())) break;
  }
  *reinterpret_cast<volatile int32_t*>(&ctl->give_up) = 1;
  return false;
}
__device__ __noinline__ bool wait_on_alone(Control* ctl, uint32_t at, uint32_t parity) {
  for (Patience p;;) {
    if (bar_poll(at, parity)) return true;
    if (*reinterpret_cast<volatile int32_t*>(&ctl->give_up) || p.over()) break;
  }
  *reinterpret_cast<volatile int32_t*>(&ctl->give_up) = 1;
  return false;
}

// Waits for a phase, by a whole warp that stays together (its tcgen05 instructions need
// that).  False: the block gives up (this wait or another took too long).
__device__ __forceinline__ bool wait(Control* ctl, uint64_t* bar, uint32_t parity) {
  const bool ok = wait_on(ctl, smem_addr(bar), parity);
  __syncwarp();
  return ok;
}
// The same by one lane.
__device__ __forceinline__ bool wait_alone(Control* ctl, uint64_t* bar, uint32_t parity) {
  const uint32_t at = smem_addr(bar);
  return bar_poll(at, parity) || wait_on_alone(ctl, at, parity);
}
// For what is under way when a block gives up.
__device__ __noinline__ void wait_out(uint64_t* bar, uint32_t parity) {
  const uint32_t at = smem_addr(bar);
  for (Patience p; !bar_poll(at, parity) && !p.over();) {
  }
}

// One lane of the warp, the same in every call.
__device__ __forceinline__ bool elect() {
  uint32_t yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
  return yes != 0;
}

__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) bar_arrive(smem_addr(bar));
}

// 16 bytes to shared memory, asynchronously; zeros where `there` is false.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// 8 elements of a row from column `col` on.
__device__ __noinline__ uint4 load8_by_element(const uint16_t* row, int col) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = row[col + 2 * i] | static_cast<uint32_t>(row[col + 2 * i + 1]) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// A row's fp32 columns in TMEM by f, by whole warps.
__device__ __forceinline__ void scale_columns(uint32_t at, int columns, float f) {
#pragma unroll 1
  for (int i = 0; i < columns; i += 16) {
    uint32_t o[16];
    tmem_load16(at + i, o);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
    tmem_store16(at + i, o);
  }
}

// Scores of keys that a row does not see (their bit is clear): -inf.
__device__ __forceinline__ void unseen(uint32_t* v, uint32_t seen) {
#pragma unroll
  for (int e = 0; e < 32; e++) v[e] = seen >> e & 1 ? v[e] : 0xff800000u;
}

// A place in the queue of segments, and the parity of its phase.
struct Turn {
  uint32_t at = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++at == kSegments) at = 0, phase ^= 1;
  }
};

// Adds the values that are not finite of the nodes in `seen` to a row that was written:
// to its result, or (out null) to its part, 4 columns at each `stride`.
template <bool kBf16>
__device__ __noinline__ void add_odd(const uint16_t* v, int64_t v_node, uint64_t seen, int dim, uint16_t* out, float* part, int stride) {
  for (; seen; seen &= seen - 1) {
    const uint16_t* row = v + (__ffsll(seen) - 1) * v_node;
    for (int d = 0; d < dim; d++)
      if (not_finite<kBf16>(row[d])) {
        const float y = widen<kBf16>(row[d]);
        if (out) out[d] = static_cast<uint16_t>(pack<kBf16>(widen<kBf16>(out[d]) + y, 0.0f));
        else part[(d >> 2) * stride + (d & 3)] += y;
      }
  }
}

// The factor of a part (t, sum) of a row in the whole: nothing where the part saw
// nothing; NaN where all that it saw were NaN.
__device__ __forceinline__ float weight(float t, float sum, float t_all) { return t == -INFINITY ? sum : exp2_fast(t - t_all); }

// ln 2^t sum, with ln 2 in two parts.
__device__ __forceinline__ float log_sum(float t, float sum) {
  return sum == 0.0f ? -INFINITY : __fmaf_rn(t, 0.693147182f, __fmaf_rn(t, -1.90465421e-9f, logf(sum)));
}

template <int kDim, bool kWide, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1) tree_kernel(CacheView c, TreeArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                                                            const __grid_constant__ CUtensorMap q_map) {
  using L = Layout<kDim, kWide>;
  constexpr int kRows = L::kRows, kChunks = kDim / 8;
  extern __shared__ __align__(1024) uint8_t raw[];
  Control& ctl = *reinterpret_cast<Control*>(raw);
  Sets* sets = reinterpret_cast<Sets*>(raw + kSetsAt);
  Sums* sums = reinterpret_cast<Sums*>(raw + kSetsAt + L::kBuffers * sizeof(Sets));
  int64_t* scan = reinterpret_cast<int64_t*>(sums);  // before the roles begin
  constexpr int kBuffers = L::kBuffers;
  const uint32_t buffers = kWide ? 1 : a.buffers, buffers_log2 = buffers - 1;
  const uint32_t q_block = a.q_rows * 128, q_tile = L::kBlocks * q_block, tree_block = a.tree_rows * 128;  // bytes
  const uint32_t q_at = control_bytes<L::kBuffers>(), tk_at = q_at + (kWide ? 2 : 1) * q_tile, tv_at = tk_at + L::kBlocks * tree_block;
  const uint32_t q_size = tv_at + L::kBlocks * tree_block - q_at, ring_at = q_at + buffers * q_size;  // of a buffer: Q and the nodes
  const uint32_t base = smem_addr(raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (base & 1023) {  // the swizzle needs it; shared memory starts on such a boundary
    if (tid == 0) atomicOr(c.status, kGaveUp);
    return;
  }

  if (tid == 0) {
    for (int i = 0; i < kMaxSlots; i++) {
      bar_init(smem_addr(&ctl.full[i]), 1);
      bar_init(smem_addr(&ctl.empty[i]), 1);
    }
    for (int i = 0; i < 2; i++) {
      bar_init(smem_addr(&ctl.q_full[i]), 2);
      bar_init(smem_addr(&ctl.q_empty[i]), 1);
      bar_init(smem_addr(&ctl.s_full[i]), 1);
      bar_init(smem_addr(&ctl.p_half[i]), 4);
      bar_init(smem_addr(&ctl.p_full[i]), 4);
      bar_init(smem_addr(&ctl.half_done[i]), 1);
    }
    bar_init(smem_addr(&ctl.done), 1);
    bar_init(smem_addr(&ctl.stats), 8);
    bar_init(smem_addr(&ctl.read), 4);
    bar_init(smem_addr(&ctl.drain), 1);
    for (int i = 0; i < kSegments; i++) {
      bar_init(smem_addr(&ctl.seg_full[i]), 1);
      bar_init(smem_addr(&ctl.seg_empty[i]), 16);  // every warp
    }
    ctl.give_up = 0;
    ctl.run_b = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == 1) {  // all 512 columns: shared memory allows one block per SM
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&ctl.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (warp == 8 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map));
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map));
  }
  after_previous_work();

  // this block's first run: each thread adds up some sequences' tiles, the one whose sum
  // reaches the run's first tile finds its place
  {
    const int per = (a.n + kThreads - 1) / kThreads, b0 = min(tid * per, a.n), b1 = min(b0 + per, a.n);
    int64_t mine = 0;
    uint32_t bad = 0;
    for (int b = b0; b < b1; b++) {
      const Seq q = sequence<kRows>(c, a, b);
      mine += static_cast<int64_t>(q.per_head) * c.kv_heads;
      bad |= q.bad;
    }
    int64_t inc = mine;
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += y;
    }
    if (lane == 31) scan[warp] = inc;
    tmem_before();
    __syncthreads();
    tmem_after();
    int64_t before = 0, total = 0;
    for (int w = 0; w < kThreads / 32; w++) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    int64_t at = before + inc - mine;
    const int64_t run = run_length(total, gridDim.x, a.min_tiles), first = run * blockIdx.x;
    if (tid == 0) ctl.total = total;
    if (blockIdx.x == 0 && bad) atomicOr(c.status, bad);
    if (first < total && first >= at && first < at + mine) {
      for (int b = b0; b < b1; b++) {
        const int64_t n = static_cast<int64_t>(sequence<kRows>(c, a, b).per_head) * c.kv_heads;
        if (first >= at && first < at + n) {
          ctl.run_b = b;
          ctl.run_off = first - at;
        }
        at += n;
      }
    }
    __syncthreads();
  }
  constexpr uint32_t tmem = 0;  // where 512 columns start
  const bool work = ctl.run_b >= 0 && ctl.tmem == tmem;
  if (ctl.tmem != tmem && tid == 0) ctl.give_up = 1;
  if (!work && tid == 0) a.cuts[blockIdx.x].b = -1;

  // Q of a segment and, with tile 0, the nodes' keys and values into a buffer, the nodes'
  // also into the cache: by the two warps 10 and 11.
  const auto load_rows = [&](const Segment& w, uint32_t segment) {
    const uint32_t buffer = segment & buffers_log2;
    if (segment >= buffers && !wait(&ctl, &ctl.q_empty[buffer], ((segment >> buffers_log2) - 1) & 1)) return false;
    const uint32_t to = buffer * q_size;
    const int rows0 = w.block * kRows, rows = min(kRows, w.nodes * a.group - rows0);  // rows that are there
    const bool tree = w.t0 == 0;
    const int me = tid - 320, ch = me % kChunks, first_row = me / kChunks;  // a thread keeps its column of chunks
    constexpr int kRowStep = 64 / kChunks;
    // 8 columns of a row to shared memory; zeros past the head's dimension and where the row is not there
    const auto bring = [&](uint32_t at, const uint16_t* row, bool there) {
      there = there && ch * 8 < c.head_dim;
      if (a.vec) copy16(base + at, row + (there ? ch * 8 : 0), there);
      else *reinterpret_cast<uint4*>(raw + at) = there ? load8_by_element(row, ch * 8) : make_uint4(0, 0, 0, 0);
    };
    // what the nodes' places in the cache take to find is on its way before the copies are
    const bool stores = tree && w.block == 0 && w.nodes > 0;
    const int first_page = w.len >> c.page_log2, in_page = w.len & (c.page_size - 1);
    int page = -1, room = 0, holders = 1;  // page: this lane's among those that the nodes go to; 64 nodes reach 9 at most
    uint64_t seen = 0;
    if (stores) {
      room = (c.counts[w.slot] << c.page_log2) - w.len;
      if (lane < 9 && first_page + lane < c.width) page = c.tables[static_cast<size_t>(w.slot) * c.width + first_page + lane];
    }
    if (tree && me < w.nodes) seen = a.masks ? a.masks[static_cast<int64_t>(w.b) * a.nodes + me] : ~0ull >> (63 - me);
    const uint16_t* q_from = a.q.p + w.b * a.q.row + static_cast<int64_t>(w.head) * a.group * a.q.head;
    if (a.q_box) {
      if (warp == 10) {
        const uint32_t bar = smem_addr(&ctl.q_full[buffer]);
        // no rows are there where a row block is all past the sequence's nodes
        const int blocks = rows > 0 ? (rows + kTile - 1) / kTile : 0, node0 = rows0 >= kTile ? rows0 / a.group : 0;
        if (blocks > 0 && elect()) {
          bar_more_bytes(bar, blocks * L::kBlocks * a.q_box * a.group * 128);
          for (int block = 0; block < blocks; block++)
#pragma unroll
            for (int x = 0; x < L::kBlocks; x++)
              tma_load_q(base + q_at + to + block * q_tile + x * q_block, &q_map, bar, x * 64, w.head * a.group, node0 + block * a.q_box, w.b);
        }
        __syncwarp();
      }
    } else
#pragma unroll 4
    for (int r = first_row; r < rows; r += kRowStep) {
      const int node = divide(rows0 + r, a.group_inverse), h = rows0 + r - node * a.group, rr = r & (kTile - 1);
      bring(q_at + to + (r / kTile) * q_tile + (ch >> 3) * q_block + rr * 128 + ((ch ^ rr) & 7) * 16, q_from + node * a.q.node + h * a.q.head, true);
    }
    if (tree) {
      const uint16_t* k_from = a.k.p + w.b * a.k.row + w.head * a.k.head;
      const uint16_t* v_from = a.v.p + w.b * a.v.row + w.head * a.v.head;
#pragma unroll 4
      for (int j = first_row; j < a.tree_rows; j += kRowStep) {
        const uint32_t at = to + (ch >> 3) * tree_block + j * 128 + ((ch ^ j) & 7) * 16;
        const int node = j < w.nodes ? j : 0;
        bring(tk_at + at, k_from + node * a.k.node, j < w.nodes);
        bring(tv_at + at, v_from + node * a.v.node, j < w.nodes);
      }
      if (me < w.nodes) sets[segment % kBuffers].of[me] = seen & (w.nodes < 64 ? (1ull << w.nodes) - 1 : ~0ull);
      // the page that the length ends in may be another row's too, forked and not yet copied
      if (lane == 0 && page >= 0 && in_page) holders = c.refs[page];
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    uint32_t odd_lo = 0, odd_hi = 0;
    if (tree) {
      holders = __shfl_sync(~0u, holders, 0);
      const int keep = stores && holders == 1 ? min(w.nodes, room) : 0;
      if (me == 0 && stores && w.head == 0 && keep < w.nodes) atomicOr(c.status, kNotReserved);
      const int64_t pages = static_cast<int64_t>(a.layer) * c.num_pages;
#pragma unroll 2
      for (int j = first_row; j < a.tree_rows; j += kRowStep) {  // as often in every lane
        const uint32_t at = to + (ch >> 3) * tree_block + j * 128 + ((ch ^ j) & 7) * 16;
        const int there = __shfl_sync(~0u, page, (in_page + j) >> c.page_log2 & 31);
        uint4 v = *reinterpret_cast<const uint4*>(raw + tv_at + at);
        if (j < keep && ch * 8 < c.head_dim) {
          const int64_t in_pool = (((pages + there) * c.kv_heads + w.head) << c.page_log2) + ((w.len + j) & (c.page_size - 1));
          *reinterpret_cast<uint4*>(c.k + in_pool * c.head_dim * 2 + ch * 16) = *reinterpret_cast<const uint4*>(raw + tk_at + at);
          *reinterpret_cast<uint4*>(c.v + in_pool * c.head_dim * 2 + ch * 16) = v;
        }
        // a value that is not finite would reach every row as 0 * inf: it is taken out
        // here and added to the rows that see it at the end
        if (odd_halves<kBf16>(v.x) | odd_halves<kBf16>(v.y) | odd_halves<kBf16>(v.z) | odd_halves<kBf16>(v.w)) {
          (j < 32 ? odd_lo : odd_hi) |= 1u << (j & 31);
          *reinterpret_cast<uint4*>(raw + tv_at + at) = make_uint4(finite_halves<kBf16>(v.x), finite_halves<kBf16>(v.y), finite_halves<kBf16>(v.z), finite_halves<kBf16>(v.w));
        }
      }
    }
    odd_lo = __reduce_or_sync(~0u, odd_lo);
    odd_hi = __reduce_or_sync(~0u, odd_hi);
    if (lane == 0) ctl.odd[segment % 4][warp & 1] = static_cast<uint64_t>(odd_hi) << 32 | odd_lo;
    if (a.scale < 0.0f) {  // scale's sign goes into Q (by copies then)
      for (int r = first_row; r < rows; r += kRowStep) {
        const int rr = r & (kTile - 1);
        uint4* q = reinterpret_cast<uint4*>(raw + q_at + to + (r / kTile) * q_tile + (ch >> 3) * q_block + rr * 128 + ((ch ^ rr) & 7) * 16);
        *q = make_uint4(q->x ^ 0x80008000u, q->y ^ 0x80008000u, q->z ^ 0x80008000u, q->w ^ 0x80008000u);
      }
    }
    fence_async();
    warp_arrive(&ctl.q_full[buffer]);
    return true;
  };

  if (work && warp == 8) {
    // ---- loading warp: a lane per page of a tile
    const int box = min(c.page_size, kTile);  // tokens of a page in a tile
    uint32_t slot = 0, turn = 0;
    int tiles = 0;  // of the first segment
    bool ok = true;
    for (Turn k; ok; k.next()) {
      ok = wait(&ctl, &ctl.seg_full[k.at], k.phase);
      if (!ok) break;
      const Segment g = ctl.seg[k.at];
      if (g.b < 0) break;
      for (int t = max(g.t0, 1); ok && t < g.t1; t++) {
        const int token = (t - 1) * kTile, here = min(kTile, g.len - token), n = (here + box - 1) / box;
        int page = 0;
        if (lane < n) page = c.tables[static_cast<size_t>(g.slot) * c.width + ((token + lane * box) >> c.page_log2)];
        const int z = (a.layer * c.num_pages + page) * c.kv_heads + g.head, y = ((token + lane * box) & (c.page_size - 1)) >> 3;
        // past the first tile the run's first Q goes before: behind a full ring of
        // copies its loads would wait for all of them
        if (tiles >= 0 && ++tiles == 2) ok = wait(&ctl, &ctl.q_full[0], 0);
#pragma unroll 1
        for (int kv = 0; ok && kv < 2; kv++) {
          if (turn > 0) ok = wait(&ctl, &ctl.empty[slot], (turn - 1) & 1);
          if (!ok) break;
          const uint32_t bar = smem_addr(&ctl.full[slot]), to = base + ring_at + slot * L::kSlot;
          if (lane == 0) bar_expect(bar, n * box * L::kBlocks * 128);
          __syncwarp();
          if (lane < n) {
            for (uint32_t x = 0; x < L::kBlocks; x += a.ring_block == 1024 ? 2 : 1)
              tma_load(to + x * a.ring_block + lane * (box >> 3) * a.ring_group, kv ? &v_map : &k_map, bar, x * 64, y, z);
          }
          __syncwarp();
          if (++slot == static_cast<uint32_t>(a.slots)) slot = 0, turn++;
        }
      }
      tiles = -1;
      warp_arrive(&ctl.seg_empty[k.at]);
    }
    // on giving up, no copy may still be under way when the block ends
    if (lane == 0 && *reinterpret_cast<volatile int32_t*>(&ctl.give_up)) {
      for (uint32_t i = 0; i < static_cast<uint32_t>(a.slots); i++) {
        const uint32_t loads = turn + (i < slot ? 1 : 0);  // copies that this slot was given
        if (loads > 0) wait_out(&ctl.full[i], (loads - 1) & 1);
      }
    }
  } else if (work && warp == 9) {
    // ---- issuing lane: S = Q K^T two steps ahead of O += P V
    if (elect()) {
      constexpr uint32_t s_inst = instruction(kBf16, kTile, 0), o_inst = instruction(kBf16, kDim, 1);
      const uint32_t tree_inst = s_inst - (static_cast<uint32_t>((kTile - a.tree_rows) >> 3) << 17);
      const uint64_t k_desc = operand(base + ring_at, 16, a.ring_group), v_desc = operand(base + ring_at, a.ring_block, a.ring_group);
      const uint32_t ring_step = a.ring_block / 16, ring_keys = a.ring_group / 8;
      uint64_t q_desc = operand(base + q_at, 16, 1024), tk_desc = operand(base + tk_at, 16, 1024), tv_desc = operand(base + tv_at, tree_block, 1024);
      const uint32_t slots = a.slots, q_step = q_block / 16, tree_step = tree_block / 16;
      uint32_t k_slot = 0, k_turn = 0, v_slot = 1, v_turn = 0;  // the next keys and values in the ring
      // steps of a segment from which on the last scores come after the nodes' products, and
      // so Q and the nodes are free with them
      constexpr int kEarly = kWide ? 4 : 3;
      uint32_t segment = 0, p_turn = 0;  // p_turn: bit s is group s's parity
      bool ok = true;
      for (Turn k; ok; k.next()) {
        ok = wait_alone(&ctl, &ctl.seg_full[k.at], k.phase);
        if (!ok || ctl.seg[k.at].b < 0) break;
        const int t0 = ctl.seg[k.at].t0, t1 = ctl.seg[k.at].t1, len = ctl.seg[k.at].len, nodes = ctl.seg[k.at].nodes;
        const int n = (t1 - t0) * (kWide ? 2 : 1);
        ok = wait_alone(&ctl, &ctl.q_full[segment & buffers_log2], segment >> buffers_log2 & 1);
        tmem_after();
        bool k_ready = false;  // the next keys were seen in the ring
        // Step j, a tile for group s, makes the output of its tile, 64 keys as soon as their
        // weights are there, then the scores of step j + 2, the group's next.
        for (int j = -2; ok && j < n; j++) {
          const int s = j & 1;
          const bool last_use = !kWide || s == 1;  // of the tile's keys or values
          if (j >= 0) {
            const int t = t0 + (kWide ? j >> 1 : j), keys = t > 0 ? min(kTile, len - (t - 1) * kTile) : nodes;
            if (t > 0 && !(kWide && s)) {
              ok = wait_alone(&ctl, &ctl.full[v_slot], v_turn & 1);
              if (!ok) break;
            }
            // look for the next keys before P is there, not between its product and theirs
            if (j + 2 < n && !(kWide && s)) k_ready = bar_poll(smem_addr(&ctl.full[k_slot]), k_turn & 1);
            const uint64_t vd = t > 0 ? v_desc + v_slot * (L::kSlot / 16) : tv_desc;
            const uint32_t step = t > 0 ? ring_keys : 2048 / 16;  // 16 keys
            const uint32_t d = 2 * kTile + s * kDim, p = s * kTile, turn = p_turn >> s & 1;
            const int steps = max(1, (keys + 15) / 16);
            ok = wait_alone(&ctl, &ctl.p_half[s], turn);
            if (!ok) break;
            tmem_after();
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (i < steps) mma_ts(d, p + i * 8, vd + i * step, o_inst, j >= 2 || i > 0);
            tmem_commit(smem_addr(&ctl.half_done[s]));
            ok = wait_alone(&ctl, &ctl.p_full[s], turn);
            if (!ok) break;
            p_turn ^= 1u << s;
            if (steps > 4) {
              tmem_after();
#pragma unroll
              for (int i = 4; i < 8; i++)
                if (i < steps) mma_ts(d, p + i * 8, vd + i * step, o_inst, 1);
            }
            if (t > 0 && last_use) {
              tmem_commit(smem_addr(&ctl.empty[v_slot]));
              v_slot += 2;
              if (v_slot >= slots) v_slot -= slots, v_turn++;
            }
            if (j == n - 1) {
              tmem_commit(smem_addr(&ctl.done));
              if (n < kEarly) tmem_commit(smem_addr(&ctl.q_empty[segment & buffers_log2]));
            }
          }
          if (j + 2 < n) {
            const int t = t0 + (kWide ? (j + 2) >> 1 : j + 2);
            if (t > 0) {
              ok = k_ready || wait_alone(&ctl, &ctl.full[k_slot], k_turn & 1);
              if (!ok) break;
              k_ready = kWide && s == 0;
              tmem_after();
            }
            const uint64_t qd = q_desc + (kWide ? s * (q_tile / 16) : 0), kd = t > 0 ? k_desc + k_slot * (L::kSlot / 16) : tk_desc;
            const uint32_t d = s * kTile, step = t > 0 ? ring_step : tree_step, inst = t > 0 ? s_inst : tree_inst;
#pragma unroll
            for (int i = 0; i < kDim / 16; i++) mma_ss(d, qd + (i >> 2) * q_step + (i & 3) * 2, kd + (i >> 2) * step + (i & 3) * 2, inst, i > 0);
            tmem_commit(smem_addr(&ctl.s_full[s]));
            if (j == n - 3 && n >= kEarly) tmem_commit(smem_addr(&ctl.q_empty[segment & buffers_log2]));
            if (t > 0 && last_use) {
              tmem_commit(smem_addr(&ctl.empty[k_slot]));
              k_slot += 2;
              if (k_slot >= slots) k_slot -= slots, k_turn++;
            }
          }
        }
        segment++;
        if (buffers == 2) {
          const uint64_t to = segment & 1 ? q_size / 16 : -static_cast<uint64_t>(q_size / 16);  // the other buffer
          q_desc += to, tk_desc += to, tv_desc += to;
        }
        if (ok) bar_arrive(smem_addr(&ctl.seg_empty[k.at]));
      }
      if (!ok) {  // what was issued ends before the block does
        tmem_commit(smem_addr(&ctl.drain));
        wait_out(&ctl.drain, 0);
      }
    }
  } else if (work && warp < 12 && warp >= 10) {
    // ---- the warps that load Q and the nodes; the first of them walks: it hands the block's
    // segments over, ahead of the others
    Walk<kRows> w;
    const int64_t run = run_length(ctl.total, gridDim.x, a.min_tiles), first = run * blockIdx.x;
    w.start(ctl.run_b, ctl.run_off, min(run, ctl.total - first));
    uint32_t segment = 0;
    bool ok = true, more = true, opening = true;
    CutItem cut;
    cut.b = -1;
    for (Turn k; ok; k.next(), segment++) {
      if (warp == 10) {
        Segment g;
        g.b = -1;
        while (more && g.b < 0) {
          w.enter(c, a);
          const int t0 = w.t0(), t1 = w.t1();
          if (t0 < t1) {
            const int me = blockIdx.x, part = t0 == 0 && t1 == w.tiles ? -1 : 2 * me + (opening ? 0 : 1);
            g = Segment{w.b, w.head, w.block, t0, t1, w.q.slot, w.q.len, w.q.nodes, part};
            if (t0 == 0 && t1 < w.tiles) {  // the run's last segment
              cut = CutItem{w.b, w.head, w.block, w.q.nodes, part, me + static_cast<int>(quotient(w.tiles - t1 + run - 1, run))};
            }
          }
          more = w.advance(c);
          opening = false;
        }
        if (segment >= kSegments) ok = wait(&ctl, &ctl.seg_empty[k.at], k.phase ^ 1);
        if (!ok) break;
        if (lane == 0) {
          ctl.seg[k.at] = g;
          bar_arrive(smem_addr(&ctl.seg_full[k.at]));
        }
        __syncwarp();
      }
      ok = wait(&ctl, &ctl.seg_full[k.at], k.phase);
      if (!ok) break;
      const Segment g = ctl.seg[k.at];
      if (g.b < 0) break;
      ok = load_rows(g, segment);
      warp_arrive(&ctl.seg_empty[k.at]);
    }
    if (warp == 10 && lane == 0) {
      a.cuts[blockIdx.x] = cut;
      if (a.q_box && *reinterpret_cast<volatile int32_t*>(&ctl.give_up))  // no copy may be under way when the block ends
        for (uint32_t i = 0; i < buffers && i < segment; i++) wait_out(&ctl.q_full[i], (segment - 1 - i) >> buffers_log2 & 1);
    }
  } else if (work && warp < 8) {
    // ---- softmax warps: a thread per row
    const int g = warp >> 2, row = tid & (kTile - 1);       // group, row of its row block
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    const uint32_t s_at = tmem + lanes + g * kTile, o_at = tmem + lanes + 2 * kTile + g * kDim;
    const float cs = fmaxf(fabsf(a.scale) * kLog2e, 1.17549435e-38f);  // not 0: a masked -inf stays -inf
    uint32_t loaded = 0, segment = 0, s_turn = 0;
    bool ok = true;
    for (Turn k; ok; k.next()) {
      ok = wait(&ctl, &ctl.seg_full[k.at], k.phase);
      if (!ok) break;
      const Segment& w = ctl.seg[k.at];  // read where it is needed: registers are for the scores
      if (w.b < 0) break;
      const int rows0 = w.block * kRows, rows = min(kRows, w.nodes * a.group - rows0);
      const int r = row + (kWide ? g * kTile : 0);
      const bool mine = r < rows, any = (r & ~31) < rows;  // this row, this warp's rows are there
      const int node = mine ? divide(rows0 + r, a.group_inverse) : 0, h = w.head * a.group + (mine ? rows0 + r - node * a.group : 0);
      uint64_t sees = 0;
      float t_ref = -INFINITY;
      uint64_t sum = 0;
      bool clear = segment == 0;  // the last segment's O has been read
      const int step = kWide ? 1 : 2;
      for (int t = w.t0 + (kWide ? 0 : g); ok && t < w.t1; t += step) {
        const int keys = t > 0 ? min(kTile, w.len - (t - 1) * kTile) : w.nodes;
        ok = wait(&ctl, &ctl.s_full[g], s_turn & 1);
        if (!ok) break;
        if (t == 0 && mine) sees = sets[segment % kBuffers].of[node];
        tmem_after();
        if (t > 0 && keys < kTile) {
          // the rows of V past the sequence's end that the last 16-key step reads are not
          // its tokens: zeros in their place
          const uint32_t e = loaded + 2 * (t - max(w.t0, 1)) + 1, slot = e % a.slots;
          ok = wait(&ctl, &ctl.full[slot], (e / a.slots) & 1);
          if (!ok) break;
          const int end = (keys + 15) & ~15;
          for (int i = row; i < (end - keys) * kChunks; i += kTile) {
            const int j = keys + i / kChunks, ch = i % kChunks;
            *reinterpret_cast<uint4*>(raw + ring_at + slot * L::kSlot + (ch >> 3) * a.ring_block + (j >> 3) * a.ring_group + (j & 7) * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async();
          __syncwarp();
        }
#pragma unroll 1
        for (int half = 0; half < 2; half++) {
          if (any && (!half || keys > 64)) {
            // 64 scores: if their maximum exceeds the bound by more than the slack, the
            // bound moves, and with it the output so far (rare after a row's first
            // scores); then their weights, which go over the scores.  A loop, not unrolled
            // over the tile: that did not fit the instruction caches beside the other roles.
            const uint32_t at = s_at + half * 64;
            uint32_t v[64];
            tmem_load32(at, v);
            tmem_load32(at + 32, v + 32);
            tmem_wait_ld();
            if (t == 0 || keys < kTile) {
              const int here = keys - 64 * half;
              const uint64_t seen = t == 0 ? sees : here >= 64 ? ~0ull : here > 0 ? (1ull << here) - 1 : 0ull;
              unseen(v, static_cast<uint32_t>(seen));
              unseen(v + 32, static_cast<uint32_t>(seen >> 32));
            }
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 64; e += 2) m[e >> 1 & 3] = max3(m[e >> 1 & 3], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
            const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * cs;
            // the difference, not a sum with t: that would be rounded where scores are huge
            const bool move = top - t_ref > kFirst<kBf16> + kSlack;
            if (__any_sync(~0u, move)) {
              const float to = top - kFirst<kBf16>, f = move ? exp2_fast(t_ref - to) : 1.0f;
              if (move) t_ref = to;
              sum = mul2(sum, two(f, f));
              if (half) {  // the products with the first half's weights are to end first; those
                           // of the tiles before had when this one's scores were made
                ok = wait(&ctl, &ctl.half_done[g], s_turn & 1);
                if (!ok) break;
                tmem_after();
              }
              if (half || t >= w.t0 + step) scale_columns(o_at, kDim, f);
            }
            const float t_use = t_ref == -INFINITY ? 0.0f : t_ref;
            const uint64_t scale = two(cs, cs), from = two(-t_use, -t_use);
            uint64_t part[2] = {0, 0};  // small weights add up before they meet the row's sum
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const uint64_t x = fma2(two(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), scale, from);
              const float p0 = exp2_fast(low_of(x)), p1 = exp2_fast(high_of(x));
              part[e >> 1 & 1] = add2(part[e >> 1 & 1], two(p0, p1));
              v[e / 2] = pack<kBf16>(p0, p1);
            }
            sum = add2(sum, add2(part[0], part[1]));
            tmem_store16(s_at + half * 32, v);
            tmem_store16(s_at + half * 32 + 16, v + 16);
            tmem_wait_st();
          }
          if (!clear) {  // the last segment's O has been read before a product writes it again
            ok = wait(&ctl, &ctl.read, (segment - 1) & 1);
            if (!ok) break;
            clear = true;
          }
          tmem_before();
          warp_arrive(half ? &ctl.p_full[g] : &ctl.p_half[g]);
        }
        s_turn++;
      }
      if (ok && !clear) ok = wait(&ctl, &ctl.read, (segment - 1) & 1);
      if (!ok) break;
      loaded += 2 * (w.t1 - max(w.t0, 1));
      sums[segment % kBuffers].t[g][row] = t_ref;
      sums[segment % kBuffers].sum[g][row] = low_of(sum) + high_of(sum);
      warp_arrive(&ctl.stats);
      segment++;
      warp_arrive(&ctl.seg_empty[k.at]);
    }
  } else if (work && warp >= 12) {
    // ---- writing warps: a segment's rows are joined over the two groups and written, or
    // left to be joined over blocks, while the others begin the next segment
    const int row = tid & (kTile - 1);
    const uint32_t o_at = tmem + (static_cast<uint32_t>(warp & 3) << 21) + 2 * kTile;
    uint32_t segment = 0;
    bool ok = true;
    for (Turn k; ok; k.next()) {
      ok = wait(&ctl, &ctl.seg_full[k.at], k.phase);
      if (!ok) break;
      const Segment& w = ctl.seg[k.at];
      if (w.b < 0) break;
      ok = wait(&ctl, &ctl.stats, segment & 1) && wait(&ctl, &ctl.done, segment & 1);
      if (!ok) break;
      tmem_after();
      const int rows0 = w.block * kRows, rows = min(kRows, w.nodes * a.group - rows0);
      const bool whole = w.part < 0;
      const bool one = kWide || w.t1 - w.t0 == 1;  // a row's O is in one group only
      const uint64_t odd = w.t0 == 0 ? ctl.odd[segment % 4][0] | ctl.odd[segment % 4][1] : 0;
      const Sums& of = sums[segment % kBuffers];
      float* part = a.partial + static_cast<int64_t>(w.part) * part_floats<kDim, kRows>();
#pragma unroll 1
      for (int g = 0; g < (kWide ? 2 : 1); g++) {
        const int r = row + g * kTile;
        const bool mine = r < rows, any = (r & ~31) < rows;  // this row, this warp's rows are there
        if (!any) break;
        const float ta = of.t[g][row], sa = of.sum[g][row];
        float t_ref = ta, sum = sa, f0 = 1.0f, f1 = 0.0f;  // factors of the two groups' O
        if (!kWide) {
          const float tb = of.t[1][row], sb = of.sum[1][row];
          t_ref = fmaxf(ta, tb);
          f0 = weight(ta, sa, t_ref);
          f1 = weight(tb, sb, t_ref);
          sum = sa * f0 + sb * f1;
        }
        const int node = mine ? divide(rows0 + r, a.group_inverse) : 0, h = w.head * a.group + (mine ? rows0 + r - node * a.group : 0);
        const int64_t at = (static_cast<int64_t>(w.b) * a.nodes + node) * a.q_heads + h;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint64_t seen = 0;
        if (odd && mine) seen = odd & (a.masks ? a.masks[static_cast<int64_t>(w.b) * a.nodes + node] : ~0ull >> (63 - node));
#pragma unroll 1
        for (int col = 0; col < kDim; col += 32) {
          float x[32];
          {
            uint32_t o[32];
            __syncwarp();
            tmem_load32(o_at + (kWide ? g * kDim : 0) + col, o);
            tmem_wait_ld();
            // a factor of 0 must not meet what an unused accumulator holds
#pragma unroll
            for (int e = 0; e < 32; e++) x[e] = kWide ? __uint_as_float(o[e]) : f0 == 0.0f ? 0.0f : __uint_as_float(o[e]) * f0;
            if (!one) {
              tmem_load32(o_at + kDim + col, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; e++) x[e] += f1 == 0.0f ? 0.0f : __uint_as_float(o[e]) * f1;
            }
          }
          if (mine) {
            if (whole) {
              uint4* out = reinterpret_cast<uint4*>(a.out + at * c.head_dim + col);
#pragma unroll
              for (int e = 0; e < 32; e += 8)
                if (col + e < c.head_dim)
                  out[e / 8] = make_uint4(pack<kBf16>(x[e] * inv, x[e + 1] * inv), pack<kBf16>(x[e + 2] * inv, x[e + 3] * inv), pack<kBf16>(x[e + 4] * inv, x[e + 5] * inv),
                                          pack<kBf16>(x[e + 6] * inv, x[e + 7] * inv));
            } else {
              float4* to = reinterpret_cast<float4*>(part) + (col / 4) * kRows + r;
#pragma unroll
              for (int e = 0; e < 32; e += 4) to[e / 4 * kRows] = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
            }
          }
        }
        if (mine) {
          if (!whole) reinterpret_cast<float2*>(part + kDim * kRows)[r] = make_float2(t_ref, sum);
          else if (a.out_lse) a.out_lse[at] = log_sum(t_ref, sum);
          if (seen)  // rare: the values that were taken out
            add_odd<kBf16>(a.v.p + w.b * a.v.row + w.head * a.v.head, a.v.node, seen, c.head_dim, whole ? a.out + at * c.head_dim : nullptr, part + 4 * r, 4 * kRows);
        }
      }
      tmem_before();
      warp_arrive(&ctl.read);
      if (w.t0 == 0) {  // rows of nodes that are not there: zeros
        const int have = max(rows, 0), want = min(kRows, a.nodes * a.group - rows0), chunks = c.head_dim >> 3;
        for (int i = row; i < (want - have) * chunks; i += kTile) {
          const int q = rows0 + have + i / chunks, node = divide(q, a.group_inverse);
          const int64_t at = (static_cast<int64_t>(w.b) * a.nodes + node) * a.q_heads + w.head * a.group + q - node * a.group;
          reinterpret_cast<uint4*>(a.out + at * c.head_dim)[i % chunks] = make_uint4(0, 0, 0, 0);
          if (i % chunks == 0 && a.out_lse) a.out_lse[at] = -INFINITY;
        }
      }
      __syncwarp();
      segment++;
      warp_arrive(&ctl.seg_empty[k.at]);
    }
  }
  __syncwarp();
  tmem_before();
  __syncthreads();
  if (tid == 0 && ctl.give_up) atomicOr(c.status, kGaveUp);
  __syncwarp();
  if (warp == 1) {
    tmem_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(ctl.tmem));
  }
}

// Joins the rows of the items that runs cut: a thread per row and 4 columns, a warp per 32
// rows, so that parts are read in whole lines, 8 parts at a time.  Grid: runs, 32 rows,
// 32 columns.
template <int kDim, bool kWide, bool kBf16>
__global__ void __launch_bounds__(256) join_kernel(CacheView c, TreeArgs a) {
  constexpr int kRows = Layout<kDim, kWide>::kRows, kBatch = 8;
  after_previous_work();
  const CutItem w = a.cuts[blockIdx.x];
  if (w.b < 0) return;
  const int rows0 = w.block * kRows, rows = min(kRows, w.nodes * a.group - rows0);
  const int r = blockIdx.y * 32 + (threadIdx.x & 31), col4 = blockIdx.z * 8 + (threadIdx.x >> 5);
  if (r >= rows || col4 * 4 >= c.head_dim) return;
  const int first = blockIdx.x, n = w.last - first + 1;
  const auto part = [&](int i) { return a.partial + static_cast<int64_t>(i == 0 ? w.part : 2 * (first + i)) * part_floats<kDim, kRows>(); };
  float t = -INFINITY, sum = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kBatch) {
    float2 ts[kBatch];
    float4 y[kBatch];
    float top = t;
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      ts[i] = make_float2(-INFINITY, 0.0f);
      if (i0 + i < n) {
        ts[i] = __ldcg(reinterpret_cast<const float2*>(part(i0 + i) + kDim * kRows) + r);
        y[i] = __ldcg(reinterpret_cast<const float4*>(part(i0 + i)) + col4 * kRows + r);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++) top = fmaxf(top, ts[i].x);
    const float before = weight(t, sum, top);
    if (before != 1.0f) {
      sum = before == 0.0f ? 0.0f : sum * before;
      o.x *= before, o.y *= before, o.z *= before, o.w *= before;
      t = top;
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const float f = weight(ts[i].x, ts[i].y, top);
      if (f != 0.0f) {
        sum += f * ts[i].y;
        o.x += f * y[i].x, o.y += f * y[i].y, o.z += f * y[i].z, o.w += f * y[i].w;
      }
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int q = rows0 + r, node = divide(q, a.group_inverse);
  const int64_t at = (static_cast<int64_t>(w.b) * a.nodes + node) * a.q_heads + w.head * a.group + q - node * a.group;
  *reinterpret_cast<uint2*>(a.out + at * c.head_dim + col4 * 4) = make_uint2(pack<kBf16>(o.x * inv, o.y * inv), pack<kBf16>(o.z * inv, o.w * inv));
  if (col4 == 0 && a.out_lse) a.out_lse[at] = log_sum(t, sum);
}

constexpr int kMaxSmem = 227 * 1024;

template <int kDim, bool kWide, bool kBf16>
cudaError_t allow_smem() {
  return cudaFuncSetAttribute(tree_kernel<kDim, kWide, kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
}

template <int kDim, bool kWide, bool kBf16>
cudaError_t launch(tg_cache* c, TreeArgs a, const CUtensorMap& q_map, cudaStream_t st) {
  using L = Layout<kDim, kWide>;
  const int rows = a.nodes * a.group < L::kRows ? a.nodes * a.group : L::kRows;
  a.q_rows = kWide ? kTile : (rows + 7) & ~7;
  a.tree_rows = (a.nodes + 15) & ~15;
  constexpr int kRowBlocks = kWide ? 2 : 1, kRoom = kMaxSmem - control_bytes<L::kBuffers>();
  static_assert((kRoom - (kRowBlocks * kTile + 2 * kTreeTile) * kDim * 2) / L::kSlot >= kMinSlots, "one buffer of any call leaves enough slots");
  const int buffer = (kRowBlocks * a.q_rows + 2 * a.tree_rows) * kDim * 2;
  // 16 sequences of 8192 tokens, 8 key heads: 64 nodes x 2 heads in one buffer beside 4 slots
  // 121 us, the calls beside them (64 x 1, 48 x 2, 40 x 3, 32 x 4) in two beside 3 slots 146 to 153
  a.buffers = L::kBuffers;
  if (kRoom - a.buffers * buffer < kMinSlots * L::kSlot) a.buffers = 1;
  const int fixed = control_bytes<L::kBuffers>() + a.buffers * buffer;
  a.slots = (kMaxSmem - fixed) / L::kSlot;
  const bool joined = c->view.head_dim == 128;  // as tree_setup's boxes
  a.ring_block = joined ? 1024 : kTile * 128;
  a.ring_group = joined ? 2048 : 1024;
  if (a.slots > kMaxSlots) a.slots = kMaxSlots;
  // the last row block's 128 rows, read from its start, end inside the block's memory:
  // at least kMinSlots slots of 128 rows follow it
  cudaError_t e = launch_after(tree_kernel<kDim, kWide, kBf16>, dim3(c->sms), kThreads, fixed + a.slots * L::kSlot, st, 1, c->view, a, c->k_map, c->v_map, q_map);
  const dim3 grid(c->sms, (rows + 31) / 32, kDim / 32);
  if (e == cudaSuccess) e = launch_after(join_kernel<kDim, kWide, kBf16>, grid, 256, 0, st, 1, c->view, a);
  return e;
}

template <int kDim>
cudaError_t launch_dim(tg_cache* c, const TreeArgs& a, const CUtensorMap& q, bool wide, cudaStream_t st) {
  const bool bf16 = c->dtype == TG_DTYPE_BF16;
  if (wide) return bf16 ? launch<kDim, true, true>(c, a, q, st) : launch<kDim, true, false>(c, a, q, st);
  return bf16 ? launch<kDim, false, true>(c, a, q, st) : launch<kDim, false, false>(c, a, q, st);
}

// The workspace: the cut items, then the parts, two per run.
constexpr size_t cut_bytes(int sms) { return (static_cast<size_t>(sms) * sizeof(CutItem) + 255) / 256 * 256; }
constexpr size_t part_bytes(int sms) { return static_cast<size_t>(sms) * 2 * 2 * kTile * (128 + 2) * sizeof(float); }

}  // namespace

int32_t tree_setup(tg_cache* c) noexcept {
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult found;
  TG_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
  if (found != cudaDriverEntryPointSuccess || !fn) return set_error(TG_ERR_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
  c->encode = reinterpret_cast<EncodeTiled>(fn);
  const CacheView& v = c->view;
  // A box is what a tile needs of a page: 8-token groups of 64-column blocks, as they lie in
  // a slot.  A head dimension of 128 comes as one box of both blocks (dimension 2), since
  // the copy engine takes about 75 cycles a box whatever its size; other dimensions past
  // 64 take a box per block, for the columns past the end to read as zeros.
  const cuuint64_t d = v.head_dim, ps = v.page_size, joined = d == 128 ? 2 : 1;
  const cuuint64_t dims[5] = {joined == 2 ? 64 : d, 8, joined, ps / 8, static_cast<cuuint64_t>(v.num_pages) * v.layers * v.kv_heads};
  const cuuint64_t strides[4] = {d * 2, 128, d * 16, d * 2 * ps};
  const cuuint32_t box[5] = {64, 8, static_cast<cuuint32_t>(joined), static_cast<cuuint32_t>((ps < kTile ? ps : kTile) / 8), 1}, ones[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < 2; i++) {
    const CUresult r = c->encode(i ? &c->v_map : &c->k_map, c->dtype == TG_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                                 i ? v.v : v.k, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(TG_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  }
  TG_TRY((allow_smem<64, false, false>()));
  TG_TRY((allow_smem<64, false, true>()));
  TG_TRY((allow_smem<64, true, false>()));
  TG_TRY((allow_smem<64, true, true>()));
  TG_TRY((allow_smem<128, false, false>()));
  TG_TRY((allow_smem<128, false, true>()));
  TG_TRY((allow_smem<128, true, false>()));
  TG_TRY((allow_smem<128, true, true>()));
  TG_TRY(cudaMalloc(&c->partial, cut_bytes(c->sms) + part_bytes(c->sms)));
  return TG_OK;
}

}  // namespace tg

using tg::set_error;

extern "C" {

int32_t tg_tree_attention(tg_cache* c, int32_t layer, int32_t n, const int32_t* seqs, int32_t nodes, const int32_t* n_nodes,
                          const uint64_t* masks, int32_t q_heads, const void* q, int64_t q_row, int64_t q_node, int64_t q_head,
                          const void* k, int64_t k_row, int64_t k_node, int64_t k_head, const void* v, int64_t v_row,
                          int64_t v_node, int64_t v_head, float scale, void* out, float* out_lse, void* stream) {
  if (!c) return set_error(TG_ERR_INVALID_ARG, "cache is NULL");
  if (n < 0 || n > c->view.max_seqs) return set_error(TG_ERR_INVALID_ARG, "n outside [0, max_seqs]");
  if (layer < 0 || layer >= c->view.layers) return set_error(TG_ERR_INVALID_ARG, "layer outside [0, layers)");
  if (nodes < 1 || nodes > TG_MAX_TREE_NODES) return set_error(TG_ERR_UNSUPPORTED, "nodes outside [1, TG_MAX_TREE_NODES]");
  if (q_heads <= 0 || q_heads % c->view.kv_heads) return set_error(TG_ERR_INVALID_ARG, "q_heads must be a multiple of kv_heads");
  if (q_heads / c->view.kv_heads > 256) return set_error(TG_ERR_UNSUPPORTED, "more than 256 query heads per key head");
  if (!std::isfinite(scale)) return set_error(TG_ERR_INVALID_ARG, "scale must be finite");
  if (n == 0) return TG_OK;
  if (!seqs || !q || !k || !v || !out) return set_error(TG_ERR_INVALID_ARG, "seqs, q, k, v and out are required");
  if (reinterpret_cast<uintptr_t>(out) & 15) return set_error(TG_ERR_INVALID_ARG, "out must be 16-byte aligned");
  tg::CurrentDevice g(c->device);
  tg::TreeArgs a{};
  a.layer = layer;
  a.n = n;
  a.nodes = nodes;
  a.q_heads = q_heads;
  a.group = q_heads / c->view.kv_heads;
  a.group_inverse = a.group == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + a.group - 1) / a.group);
  const bool wide = nodes * a.group > tg::kTile;  // more rows than one block of the tensor cores takes
  const int rows = wide ? 2 * tg::kTile : tg::kTile;
  a.blocks = (nodes * a.group + rows - 1) / rows;
  a.min_tiles = 2 + tg::kOverhead;
  a.vec = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
            static_cast<uintptr_t>((q_row | q_node | q_head | k_row | k_node | k_head | v_row | v_node | v_head) * 2)) & 15) == 0;
  a.seqs = seqs;
  a.n_nodes = n_nodes;
  a.masks = masks;
  a.q = {static_cast<const uint16_t*>(q), q_row, q_node, q_head};
  a.k = {static_cast<const uint16_t*>(k), k_row, k_node, k_head};
  a.v = {static_cast<const uint16_t*>(v), v_row, v_node, v_head};
  a.scale = scale;
  a.out = static_cast<uint16_t*>(out);
  a.out_lse = out_lse;
  char* space = static_cast<char*>(c->partial);
  a.cuts = reinterpret_cast<tg::CutItem*>(space);
  a.partial = reinterpret_cast<float*>(space + tg::cut_bytes(c->sms));
  // Q comes in boxes of whole nodes, heads inside nodes, as its rows lie in shared memory: two
  // warps' 16-byte copies take 170 cycles an instruction of 512 bytes, 11,000 for 256 rows
  // (91 short sequences of 64 nodes x 8 heads: 88 us by copies, 67 by boxes; with 4 rows both
  // take the same).  Copies stay for rows that a map cannot describe (not 16-byte aligned,
  // a stride of 0, heads that do not fill 128 rows evenly) and for a negative scale.
  CUtensorMap q_map{};
  if (a.vec && scale >= 0.0f && tg::kTile % a.group == 0 && q_row > 0 && q_node > 0 && q_head > 0) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c->view.head_dim), static_cast<cuuint64_t>(q_heads), static_cast<cuuint64_t>(nodes), static_cast<cuuint64_t>(n)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(q_head) * 2, static_cast<cuuint64_t>(q_node) * 2, static_cast<cuuint64_t>(q_row) * 2};
    const int box_nodes = nodes < tg::kTile / a.group ? nodes : tg::kTile / a.group;
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(box_nodes), 1}, ones[4] = {1, 1, 1, 1};
    if (c->encode(&q_map, c->dtype == TG_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(q), dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS)
      a.q_box = box_nodes;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TG_TRY(c->view.head_dim <= 64 ? tg::launch_dim<64>(c, a, q_map, wide, st) : tg::launch_dim<128>(c, a, q_map, wide, st));
  return TG_OK;
}

}  // extern "C"
