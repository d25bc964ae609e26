// The int8 cache and a call's sequences as the kernels see them (kv_cache.cu, cached_attention.cu).
#ifndef TGCB_KV_CACHE_CUH_
#define TGCB_KV_CACHE_CUH_

#include <cstdint>

#include "tgcb.h"

namespace tgcb_kv {

constexpr int kMaxBatch = 4096;

struct Cache {
  int8_t* keys;
  int8_t* values;
  float* key_scales;
  float* value_scales;
  int* faults;
  int pages, heads, page, width, page_bits;  // page == 1 << page_bits
};

struct Batch {
  const int* table;
  const int* starts;
  const int* offsets;
  long long table_stride, tokens;
  int batch, max_pages, each;
};

// Fills *c and *b, or reports why the call is refused (kv_cache.cu).
int checked(const tgcb_cache* cache, const tgcb_batch* batch, int dtype, Cache* c, Batch* b, const char* what);

// Token rows [first, last) of sequence s, whatever the offsets hold.
__device__ __forceinline__ void range_of(const Batch& b, int s, long long* first, long long* last) {
  long long f, l;
  if (b.offsets == nullptr) {
    f = (long long)s * b.each, l = f + b.each;
  } else {
    f = __ldg(b.offsets + s), l = __ldg(b.offsets + s + 1);
    f = f < 0 ? 0 : f;
    l = l > b.tokens ? b.tokens : l;
  }
  *first = f, *last = l < f ? f : l;
}

// The page of a position, -1 where the position or the entry is out of range.
__device__ __forceinline__ int page_of(const Cache& c, const Batch& b, int s, long long position) {
  const long long slot = position >> c.page_bits;
  if (position < 0 || slot >= b.max_pages) return -1;
  const int page = __ldg(b.table + s * b.table_stride + slot);
  return page < 0 || page >= c.pages ? -1 : page;
}

}  // namespace tgcb_kv

#endif  // TGCB_KV_CACHE_CUH_
