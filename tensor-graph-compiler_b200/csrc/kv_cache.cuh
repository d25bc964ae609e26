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

// Where a token row lies: its sequence (-1: none), and the page and place of its position
// (page -1: the position or the table's entry is out of range).
struct Place {
  int sequence, page, row;
  long long position;
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

// The whole CTA looks for `token`'s place; *out (shared, sequence -1 before) holds it after a barrier.
__device__ __forceinline__ void find(const Cache& c, const Batch& b, long long token, Place* out) {
  const bool even = b.offsets == nullptr;
  if (even && threadIdx.x != 0) return;
  for (int s = even ? (int)(token / b.each) : threadIdx.x; s < b.batch; s += blockDim.x) {
    long long first, last;
    range_of(b, s, &first, &last);
    if (token >= first && token < last) {
      const long long position = (long long)__ldg(b.starts + s) + token - first;
      out->page = page_of(c, b, s, position);
      out->row = (int)(position & (c.page - 1));
      out->position = position;
      out->sequence = s;
      if (out->page < 0) atomicAdd(c.faults, 1);
      return;
    }
  }
}

// *later (shared, 0 before) becomes 1 where a later token row of the call has the same place.
__device__ __forceinline__ void find_later(const Cache& c, const Batch& b, long long token, const Place& place, int* later) {
  for (int s = place.sequence + threadIdx.x; s < b.batch; s += blockDim.x) {
    long long first, last;
    range_of(b, s, &first, &last);
    const long long start = __ldg(b.starts + s);
    if (last <= first || start < 0) continue;
    for (long long slot = start >> c.page_bits; slot <= (start + last - first - 1) >> c.page_bits && slot < b.max_pages; ++slot) {
      const long long at = first + (slot << c.page_bits) + place.row - start;
      if (at > token && at >= first && at < last && __ldg(b.table + s * b.table_stride + slot) == place.page) *later = 1;
    }
  }
}

}  // namespace tgcb_kv

#endif  // TGCB_KV_CACHE_CUH_
