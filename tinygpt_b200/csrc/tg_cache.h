// tg_cache.h -- the paged cache's handle, shared by tg_cache.cu (bookkeeping,
// page copies) and tg_tree.cu (attention).
#ifndef TG_CACHE_H
#define TG_CACHE_H

#include <cuda.h>

#include "tg_host.h"

namespace tg {

// Status bits (tg_cache_device_status).
constexpr uint32_t kBadSlot = 1, kNoPages = 2, kBadLength = 4, kNotReserved = 8, kGaveUp = 16, kBadTree = 32;

// What the kernels see of a cache.
struct CacheView {
  int32_t layers, kv_heads, head_dim, page_size, page_log2, num_pages, max_seqs, width;  // width: pages per table row
  char* k;  // pools, 2-byte elements
  char* v;
  int32_t* lens;
  int32_t* counts;
  int32_t* tables;
  int32_t* refs;
  uint32_t* free_map;  // bit p: page p is held by no row
  uint32_t* status;
  // scratch of single calls; claim, shared and first are back at 0, 0, INT_MAX after each
  int32_t* claim;    // [max_seqs]  a row of the call has this slot
  int32_t* shared;   // [num_pages] rows of the call that would write to this page
  int32_t* first;    // [num_pages] the first of them
  int32_t* start;    // [max_seqs]  row -> its first page in `list`
  int32_t* need;     // [max_seqs]  row -> 2 * new pages + (1 if its last page is copied), -1: not in the call
  int32_t* last;     // [max_seqs]  row -> its partly filled last page or -1
  int32_t* list;     // [num_pages] pages handed out by the call
  int4* copies;      // [max_seqs]  (from, to, tokens, -)
  int32_t* n_copies;
  int4* info;        // [max_seqs]  fork: (new pages, old pages, length, served)
  int32_t* staged;   // [max_seqs, width] fork: the new table rows
  int4* moves;       // [max_seqs, TG_MAX_TREE_NODES] accept: (from page, slot, to page, slot)
  int32_t* n_moves;  // [max_seqs]
};

}  // namespace tg

// cuTensorMapEncodeTiled
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct tg_cache {
  int device = 0;
  int sms = 0;
  tg::CacheView view{};
  int32_t dtype = 0;
  void* arena = nullptr;   // every device array of the view
  void* partial = nullptr; // attention: outputs of split rows (tg_tree.cu)
  CUtensorMap k_map{}, v_map{};
  EncodeTiled encode = nullptr;
};

namespace tg {
// tg_tree.cu: the attention's share of a handle (tensor maps, workspace).
__attribute__((visibility("hidden"))) int32_t tree_setup(tg_cache* c) noexcept;
}  // namespace tg

#endif  // TG_CACHE_H
