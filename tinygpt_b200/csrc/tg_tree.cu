// tg_tree.cu -- attention of drafted nodes over a paged cache (tg_tree_attention).
#include "tg_cache.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

namespace tg {
namespace {

__device__ __forceinline__ void after_previous_work() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Rows {  // [n, nodes, heads, head_dim]: strides in elements
  const void* p;
  int64_t row, node, head;
};

struct TreeArgs {
  int32_t layer, n, nodes, q_heads;
  const int32_t* seqs;
  const int32_t* n_nodes;
  const uint64_t* masks;
  Rows q, k, v;
  float scale;
  void* out;
  float* out_lse;
};

constexpr int kThreads = 128;

// A block per (row, node, query head); a warp per key, lanes over the head's
// dimensions; each warp with its own running maximum and sum.
template <class T>
__global__ void __launch_bounds__(kThreads) tree_kernel(CacheView c, TreeArgs a) {
  __shared__ float wm[4], wl[4], wo[4][128];
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  after_previous_work();
  const int D = c.head_dim, kvh = h / (a.q_heads / c.kv_heads);
  T* out = static_cast<T*>(a.out) + ((static_cast<int64_t>(b) * a.nodes + i) * a.q_heads + h) * D;
  const int64_t at = (static_cast<int64_t>(b) * a.nodes + i) * a.q_heads + h;
  const int s = a.seqs[b], given = a.n_nodes ? a.n_nodes[b] : a.nodes;
  const bool bad = given < 0 || given > a.nodes;
  const int count = bad ? 0 : given;
  if (bad && threadIdx.x == 0) atomicOr(c.status, kBadTree);
  if (s < 0 || s >= c.max_seqs || i >= count) {
    for (int d = threadIdx.x; d < D; d += kThreads) out[d] = T(0.0f);
    if (threadIdx.x == 0 && a.out_lse) a.out_lse[at] = -INFINITY;
    return;
  }
  const int len = c.lens[s];
  const uint64_t mask = a.masks ? a.masks[static_cast<int64_t>(b) * a.nodes + i] : (i == 63 ? ~0ull : (2ull << i) - 1);
  const T* q = static_cast<const T*>(a.q.p) + b * a.q.row + i * a.q.node + h * a.q.head;
  float qr[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
  for (int e = 0; e < 4; e++) qr[e] = lane + 32 * e < D ? float(q[lane + 32 * e]) : 0.0f;
  for (int j = warp; j < len + count; j += 4) {
    const T *k, *v;
    if (j < len) {
      const int64_t page = c.tables[static_cast<size_t>(s) * c.width + (j >> c.page_log2)] + static_cast<int64_t>(a.layer) * c.num_pages;
      const int64_t off = (((page * c.kv_heads + kvh) << c.page_log2) + (j & (c.page_size - 1))) * D;
      k = reinterpret_cast<const T*>(c.k) + off;
      v = reinterpret_cast<const T*>(c.v) + off;
    } else {
      if (!(mask >> (j - len) & 1)) continue;
      k = static_cast<const T*>(a.k.p) + b * a.k.row + (j - len) * a.k.node + kvh * a.k.head;
      v = static_cast<const T*>(a.v.p) + b * a.v.row + (j - len) * a.v.node + kvh * a.v.head;
    }
    float dot = 0;
    for (int e = 0; e < 4; e++)
      if (lane + 32 * e < D) dot = fmaf(qr[e], float(k[lane + 32 * e]), dot);
    for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(~0u, dot, d);
    dot *= a.scale;
    const float nm = fmaxf(m, dot), f = expf(m - nm), p = expf(dot - nm);
    m = nm;
    l = l * f + p;
    for (int e = 0; e < 4; e++)
      if (lane + 32 * e < D) o[e] = o[e] * f + p * float(v[lane + 32 * e]);
  }
  if (lane == 0) wm[warp] = m, wl[warp] = l;
  for (int e = 0; e < 4; e++) wo[warp][lane + 32 * e] = o[e];
  __syncthreads();
  float top = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
  float total = 0, f[4];
  for (int w = 0; w < 4; w++) {
    f[w] = wm[w] == -INFINITY ? 0.0f : expf(wm[w] - top);
    total += wl[w] * f[w];
  }
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float x = 0;
    for (int w = 0; w < 4; w++) x += f[w] == 0.0f ? 0.0f : f[w] * wo[w][d];
    out[d] = T(total == 0.0f ? 0.0f : x / total);
  }
  if (threadIdx.x == 0 && a.out_lse) a.out_lse[at] = total == 0.0f ? -INFINITY : top + logf(total);
}

}  // namespace

int32_t tree_setup(tg_cache*) noexcept { return TG_OK; }

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
  if (!(scale == scale) || std::isinf(scale)) return set_error(TG_ERR_INVALID_ARG, "scale must be finite");
  if (n == 0) return TG_OK;
  if (!seqs || !q || !k || !v || !out) return set_error(TG_ERR_INVALID_ARG, "seqs, q, k, v and out are required");
  tg::CurrentDevice g(c->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const tg::TreeArgs a{layer, n, nodes, q_heads, seqs, n_nodes, masks, {q, q_row, q_node, q_head}, {k, k_row, k_node, k_head},
                       {v, v_row, v_node, v_head}, scale, out, out_lse};
  const int32_t rc = tg_cache_append(c, layer, n, seqs, n_nodes, nodes, k, k_row, k_node, k_head, v, v_row, v_node, v_head, stream);
  if (rc != TG_OK) return rc;
  const dim3 grid(q_heads, nodes, n);
  TG_TRY(tg::launch_after(c->dtype == TG_DTYPE_BF16 ? tg::tree_kernel<__nv_bfloat16> : tg::tree_kernel<__half>, grid, tg::kThreads, 0, st, 1, c->view, a));
  return TG_OK;
}

}  // extern "C"
