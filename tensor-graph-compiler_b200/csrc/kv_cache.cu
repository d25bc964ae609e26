// The int8 cache of keys and values: rows quantised as they are written, and read back.
//
// A row x of one head becomes codes rint(x / scale) with scale = float(double(max|x|) / 127), 1 for a
// row of zeros: the rule of tgcb_quantise_rows_i8, bit for bit, so a row quantised there and a row
// written here are the same.
#include <cuda_runtime.h>

#include <cstdint>

#include "elements.cuh"
#include "internal.h"
#include "kv_cache.cuh"
#include "tgcb.h"

namespace {

using namespace tgcb_elem;
using tgcb_kv::Batch;
using tgcb_kv::Cache;
using tgcb_kv::Place;

struct Rows {
  char* data;
  long long t, h;
};

constexpr int kThreads = 256;

// One CTA per token, a warp per row of it.
template <typename T>
__global__ void __launch_bounds__(kThreads) append_rows(const Cache c, const Batch b, const Rows keys, const Rows values) {
  __shared__ Place place;
  __shared__ int later;
  const long long token = blockIdx.x;
  if (threadIdx.x == 0) later = 0, place.sequence = -1;
  __syncthreads();
  tgcb_kv::find(c, b, token, &place);
  __syncthreads();
  if (place.sequence < 0 || place.page < 0) return;
  tgcb_kv::find_later(c, b, token, place, &later);
  __syncthreads();
  if (later) return;
  const int lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < 2 * c.heads; r += kThreads / 32) {
    const bool value = r >= c.heads;
    const int h = value ? r - c.heads : r;
    const Rows& rows = value ? values : keys;
    const T* x = reinterpret_cast<const T*>(rows.data) + token * rows.t + h * rows.h;
    unsigned m = 0;
    for (int i = lane; i < c.width; i += 32) m = max(m, __float_as_uint(to_float(x[i])) & 0x7fffffffu);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float largest = __uint_as_float(m);
    const float scale = largest == 0.0f ? 1.0f : (float)((double)largest / 127.0);
    const long long at = ((long long)place.page * c.heads + h) * c.page + place.row;
    if (lane == 0) (value ? c.value_scales : c.key_scales)[at] = scale;
    int8_t* q = (value ? c.values : c.keys) + at * c.width;
    for (int i = lane; i < c.width; i += 32) {
      const float t = fminf(fmaxf(rintf(__fdiv_rn(to_float(x[i]), scale)), -128.0f), 127.0f);
      q[i] = (int8_t)(int)t;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) read_rows(const Cache c, const Batch b, const Rows keys, const Rows values) {
  __shared__ Place place;
  const long long token = blockIdx.x;
  if (threadIdx.x == 0) place.sequence = -1;
  __syncthreads();
  tgcb_kv::find(c, b, token, &place);
  __syncthreads();
  if (place.sequence < 0) return;
  const int lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < 2 * c.heads; r += kThreads / 32) {
    const bool value = r >= c.heads;
    const int h = value ? r - c.heads : r;
    const Rows& rows = value ? values : keys;
    T* x = reinterpret_cast<T*>(rows.data) + token * rows.t + h * rows.h;
    const long long at = ((long long)place.page * c.heads + h) * c.page + place.row;
    const float scale = place.page < 0 ? __int_as_float(0x7fffffff) : (value ? c.value_scales : c.key_scales)[at];
    const int8_t* q = (value ? c.values : c.keys) + at * c.width;
    for (int i = lane; i < c.width; i += 32) x[i] = from_float<T>(place.page < 0 ? scale : (float)q[i] * scale);
  }
}

template <typename T>
int run(const Cache& c, const Batch& b, const Rows& k, const Rows& v, bool read, cudaStream_t s) {
  if (b.tokens == 0) return TGCB_OK;
  if (read)
    read_rows<T><<<(unsigned)b.tokens, kThreads, 0, s>>>(c, b, k, v);
  else
    append_rows<T><<<(unsigned)b.tokens, kThreads, 0, s>>>(c, b, k, v);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, "kv_cache", cudaGetErrorString(e));
  return TGCB_OK;
}

int entry(const tgcb_cache* cache, const tgcb_batch* batch, int dtype, const tgcb_heads* keys, const tgcb_heads* values,
          bool read, void* stream, const char* what) {
  Cache c;
  Batch b;
  const int rc = tgcb_kv::checked(cache, batch, dtype, &c, &b, what);
  if (rc != TGCB_OK) return rc;
  if (keys == nullptr || values == nullptr || (b.tokens > 0 && (keys->data == nullptr || values->data == nullptr)))
    return tgcb_internal_fail(TGCB_E_INVALID, what, "null pointer");
  const Rows k = {static_cast<char*>(keys->data), keys->token_stride, keys->head_stride};
  const Rows v = {static_cast<char*>(values->data), values->token_stride, values->head_stride};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TGCB_F32: return run<float>(c, b, k, v, read, s);
    case TGCB_BF16: return run<__nv_bfloat16>(c, b, k, v, read, s);
    default: return run<__half>(c, b, k, v, read, s);
  }
}

}  // namespace

namespace tgcb_kv {

int checked(const tgcb_cache* cache, const tgcb_batch* batch, int dtype, Cache* c, Batch* b, const char* what) {
  auto bad = [&](const char* why) { return tgcb_internal_fail(TGCB_E_INVALID, what, why); };
  if (cache == nullptr || batch == nullptr) return bad("null descriptor");
  if (dtype < TGCB_F32 || dtype > TGCB_F16) return bad("unknown element type");
  if (cache->keys == nullptr || cache->values == nullptr || cache->key_scales == nullptr || cache->value_scales == nullptr ||
      cache->faults == nullptr)
    return bad("null pointer in the cache");
  if ((reinterpret_cast<uintptr_t>(cache->keys) | reinterpret_cast<uintptr_t>(cache->values)) & 15u)
    return bad("the cache's codes must be 16-byte aligned");
  if (cache->width != 32 && cache->width != 64 && cache->width != 128 && cache->width != 256)
    return bad("the cache's width must be 32, 64, 128 or 256");
  if (cache->page != 16 && cache->page != 32 && cache->page != 64 && cache->page != 128)
    return bad("a page has 16, 32, 64 or 128 places");
  if (cache->kv_heads < 1 || cache->kv_heads > 1024) return bad("a cache has 1 to 1024 heads");
  if (cache->pages < 1 || cache->pages > 0x7fffffffll) return bad("a cache has 1 to 2^31 - 1 pages");
  if (batch->tokens < 0 || batch->tokens > 0x7fffffffll) return bad("too many tokens");
  if (batch->batch < 1 || batch->batch > kMaxBatch) return bad("a call has 1 to 4096 sequences");
  if (batch->max_pages < 1 || (long long)batch->max_pages * cache->page > (1ll << 30)) return bad("a page table holds 1 to 2^30 positions a sequence");
  if (batch->table == nullptr || batch->starts == nullptr) return bad("null pointer in the batch");
  if (batch->offsets == nullptr && batch->tokens % batch->batch != 0)
    return bad("without offsets every sequence has the same number of tokens");
  *c = Cache{cache->keys, cache->values, cache->key_scales, cache->value_scales, cache->faults,
             (int)cache->pages, cache->kv_heads, cache->page, cache->width, __builtin_ctz((unsigned)cache->page)};
  *b = Batch{batch->table, batch->starts, batch->offsets, batch->table_stride, batch->tokens,
             batch->batch, batch->max_pages, (int)(batch->tokens / batch->batch)};
  return TGCB_OK;
}

}  // namespace tgcb_kv

extern "C" {

int tgcb_cache_append(const tgcb_cache* cache, const tgcb_batch* batch, int dtype, const tgcb_heads* keys,
                      const tgcb_heads* values, void* stream) {
  return entry(cache, batch, dtype, keys, values, false, stream, "tgcb_cache_append");
}

int tgcb_cache_read(const tgcb_cache* cache, const tgcb_batch* batch, int dtype, const tgcb_heads* keys,
                    const tgcb_heads* values, void* stream) {
  return entry(cache, batch, dtype, keys, values, true, stream, "tgcb_cache_read");
}

}  // extern "C"
