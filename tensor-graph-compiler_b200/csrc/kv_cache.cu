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

struct Rows {
  char* data;
  long long t, h;
};

constexpr int kThreads = 256;
constexpr int kTokens = 32;  // tokens a CTA takes at most: a warp has a thread for each

// Where a token row lies: the page and place of its position. Page -1: the position or the table's
// entry is out of range; kNoSequence: the row belongs to no sequence.
struct __align__(8) Place {
  int page, row;
};
constexpr int kNoSequence = -2;

// The places of token rows [token0, token0 + count), by the whole CTA; a barrier must be before and follow. Threads
// look at their share of the sequences for the rows that are theirs, then a thread a row looks up its place: a
// sequence's thread doing that row by row waited for one page number after another, 4 of append's 40 us and of read's 37.
// *least: the first sequence met.
__device__ __forceinline__ void find_places(const Cache& c, const Batch& b, long long token0, int count, Place* places, int* least) {
  if (b.offsets != nullptr) {
    for (int s = threadIdx.x; s < b.batch; s += kThreads) {
      long long first, last;
      tgcb_kv::range_of(b, s, &first, &last);
      for (long long t = first > token0 ? first : token0; t < last && t < token0 + count; ++t) places[t - token0].row = s;
    }
    __syncthreads();
  }
  if (threadIdx.x >= 32) return;
  const int i = threadIdx.x;
  const int s = i >= count ? -1 : b.offsets == nullptr ? (int)((token0 + i) / b.each) : places[i].row;
  if (s >= 0) {
    long long first, last;
    tgcb_kv::range_of(b, s, &first, &last);
    const long long position = (long long)__ldg(b.starts + s) + token0 + i - first;
    const int page = tgcb_kv::page_of(c, b, s, position);
    if (page < 0) atomicAdd(c.faults, 1);
    places[i] = Place{page, (int)(position & (c.page - 1))};
  }
  const int smallest = __reduce_min_sync(0xffffffffu, s < 0 ? b.batch : s);
  if (i == 0) *least = smallest;
}

// later[i] becomes 1 where a later row of the call has row i's place: two sequences that share a page both
// write to, or a page twice in one table row. The call's written pages are few beside its rows; a
// thread takes a sequence, and a sequence of many pages is taken by its warp. Rows that follow one another in a
// page are compared as one: looking at each took 10 of append's 54 us.
__device__ __forceinline__ void find_later(const Cache& c, const Batch& b, long long token0, int count, const Place* places, int least, int* later) {
  const int lane = threadIdx.x & 31;
  if (least + (int)(threadIdx.x & ~31) >= b.batch) return;  // whole warps
  const int page_here = lane < count ? places[lane].page : kNoSequence, page_before = __shfl_up_sync(0xffffffffu, page_here, 1);
  const unsigned runs = __ballot_sync(0xffffffffu, lane < count && (lane == 0 || page_here != page_before));
  auto look = [&](int page, long long slot, long long first, long long last, long long start) {
    if (page < 0) return;
    for (unsigned r = runs; r; r &= r - 1) {
      for (int i = __ffs(r) - 1; i < count && places[i].page == page; ++i) {
        const long long at = first + (slot << c.page_bits) + places[i].row - start;
        if (at > token0 + i && at >= first && at < last) later[i] = 1;
      }
    }
  };
  for (int s0 = least + (threadIdx.x & ~31); s0 < b.batch; s0 += kThreads) {
    const int s = s0 + lane;
    long long first = 0, last = 0, start = 0, slot = 0, end = 0;
    if (s < b.batch) {
      tgcb_kv::range_of(b, s, &first, &last);
      start = __ldg(b.starts + s);
      if (last > first && start + last - first > 0) {
        slot = start < 0 ? 0 : start >> c.page_bits;
        end = ((start + last - first - 1) >> c.page_bits) + 1;
        end = end > b.max_pages ? b.max_pages : end;
      }
    }
    const int* pages = b.table + s * b.table_stride;
    const int page0 = slot < end ? __ldg(pages + slot) : -1, page1 = slot + 1 < end ? __ldg(pages + slot + 1) : -1;
    look(page0, slot, first, last, start);
    look(page1, slot + 1, first, last, start);
    unsigned more = __ballot_sync(0xffffffffu, slot + 2 < end);
    while (more) {
      const int from = __ffs(more) - 1;
      more &= more - 1;
      const long long f = __shfl_sync(0xffffffffu, first, from), l = __shfl_sync(0xffffffffu, last, from);
      const long long st = __shfl_sync(0xffffffffu, start, from), e = __shfl_sync(0xffffffffu, end, from);
      const int* row = b.table + (s0 + from) * b.table_stride;
      for (long long k = __shfl_sync(0xffffffffu, slot, from) + 2 + lane; k < e; k += 128) {
        int page[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) page[i] = k + 32 * i < e ? __ldg(row + k + 32 * i) : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) look(page[i], k + 32 * i, f, l, st);
      }
    }
  }
}

// Eight values of a row, a thread's share of it: eight in a row of 16-bit values, and of float32 four in each
// half of the row, so that neighbouring threads' 16 bytes lie side by side. WHOLE: rows are 16-byte aligned.
template <typename T, bool WHOLE>
struct Eight {
  static constexpr bool HALVES = sizeof(T) == 4;
  union {
    uint4 raw[sizeof(T) / 2];
    T e[8];
  };
  __device__ Eight() {}
  static __device__ __forceinline__ int column(int item, int i, int width) {
    return HALVES ? 4 * item + (i & 3) + (i >> 2) * (width / 2) : 8 * item + i;
  }
  __device__ __forceinline__ void load(const T* row, int item, int width) {
    if constexpr (WHOLE) {
      raw[0] = *reinterpret_cast<const uint4*>(row + column(item, 0, width));
      if constexpr (HALVES) raw[1] = *reinterpret_cast<const uint4*>(row + column(item, 4, width));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = row[column(item, i, width)];
    }
  }
  __device__ __forceinline__ void store(T* row, int item, int width) const {
    if constexpr (WHOLE) {
      *reinterpret_cast<uint4*>(row + column(item, 0, width)) = raw[0];
      if constexpr (HALVES) *reinterpret_cast<uint4*>(row + column(item, 4, width)) = raw[1];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) row[column(item, i, width)] = e[i];
    }
  }
  static __device__ __forceinline__ uint2 load_codes(const int8_t* row, int item, int width) {
    if constexpr (HALVES)
      return make_uint2(*reinterpret_cast<const unsigned*>(row + 4 * item), *reinterpret_cast<const unsigned*>(row + 4 * item + width / 2));
    return *reinterpret_cast<const uint2*>(row + 8 * item);
  }
  static __device__ __forceinline__ void store_codes(int8_t* row, int item, int width, uint2 q) {
    if constexpr (HALVES) {
      *reinterpret_cast<unsigned*>(row + 4 * item) = q.x;
      *reinterpret_cast<unsigned*>(row + 4 * item + width / 2) = q.y;
    } else {
      *reinterpret_cast<uint2*>(row + 8 * item) = q;
    }
  }
};

// Codes of eight values: rint(x / scale). With the approximate reciprocal (2 ulp for scales of normal size) x * (1 / scale)
// is off by 2^-22 + 2^-24 of the quotient, 3.8e-5 at most, so away from half-integers (5e-5) it rounds
// as the quotient does, and values near one are divided (normal bfloat16 values have some in 45% of the warps:
// max / 2 is 63.5 scales). There |x / scale| <= 127 (1 + 2^-21):
// no clamp; other rows divide and clamp. Adding 1.5 2^23 rounds to an integer, ties to even, in the sum's low bits.
template <bool SIXTEEN>
__device__ __forceinline__ uint2 codes_of(const float* x, float scale) {
  unsigned q[8];
  if (scale >= 0x1p-126f && scale <= 0x1p126f) {  // not NaN, not infinite
    const float inverse = __fdividef(1.0f, scale);
    float near = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = x[i] * inverse, rounded = t + 12582912.0f;
      near = fmaxf(near, fabsf(t - (rounded - 12582912.0f)));
      q[i] = __float_as_uint(rounded);
    }
    if (near >= 0.49995f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = x[i] * inverse;
        if (!SIXTEEN || fabsf(d - (__uint_as_float(q[i]) - 12582912.0f)) >= 0.49995f) q[i] = __float_as_uint(__fdiv_rn(x[i], scale) + 12582912.0f);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = (unsigned)(int)fminf(fmaxf(rintf(__fdiv_rn(x[i], scale)), -128.0f), 127.0f);
  }
  uint2 r;
  r.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  r.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return r;
}

// The larger magnitude, NaN if either is.
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// Bound by HBM: append reads a row and writes width + 4 bytes, read the reverse. width / 8 threads have a
// row; a CTA takes `each` tokens with all their heads, keys then values, and has the values of kAhead
// rounds on their way at once. Measured, 16384 tokens of 8 + 8 float32 heads of 128 (169 MB each way): read 29 us,
// 5.8 TB/s; append 37 us, 4.6 TB/s, held by the look-up of its tokens' places before its first store (with 16 tokens a
// CTA 2 us more, for two rounds of it) and by instructions: 190 a warp for 32 eights of values. The same tokens in
// bfloat16 (102 MB): append 39 us, read 20 us. Each CTA of an append looks through the pages that the sequences from its own
// on write to, so that part grows with the square of the call: hidden at 16384 tokens, not at millions in small pages.
template <typename T>
constexpr int kAhead = 8 / sizeof(T);  // 64 bytes a thread, within the registers of four CTAs an SM

// The rows of one thread group: a side and head of the keys and values, and every step-th token from the
// first. A CTA whose groups are fewer than a token's rows goes over its tokens several times.
struct Group {
  int row, rows, token, step;
  __device__ __forceinline__ Group(int group, int groups, int rows) : rows(rows) {
    const int at_once = min(groups, rows);
    step = groups / at_once;
    token = group / at_once, row = group - token * at_once;
    if (token >= step) token = 1 << 30;  // more groups than whole tokens' rows: idle
  }
};

template <typename T, int W, bool WHOLE>
__global__ void __launch_bounds__(kThreads, WHOLE ? 4 : 2) append_rows(const Cache c, const Batch b, const Rows keys, const Rows values, int each) {
  __shared__ Place places[kTokens];
  __shared__ int later[kTokens], least;
  const long long token0 = (long long)blockIdx.x * each;
  const int count = (int)min((long long)each, b.tokens - token0);
  constexpr int lanes = W / 8, groups = kThreads / lanes;
  const int item = threadIdx.x % lanes;
  const Group g(threadIdx.x / lanes, groups, 2 * c.heads);
  if (threadIdx.x < kTokens) places[threadIdx.x] = Place{kNoSequence, -1}, later[threadIdx.x] = 0;

  for (int row0 = 0; row0 < g.rows; row0 += groups) {
    const int row = row0 + g.row;
    const bool real = row < g.rows, value = row >= c.heads;
    const int head = value ? row - c.heads : row;
    const Rows& rows = value ? values : keys;
    const T* from = reinterpret_cast<const T*>(rows.data) + (real ? token0 * rows.t + head * rows.h : 0);
    const long long t = rows.t;
    int8_t* codes = value ? c.values : c.keys;
    float* scales = value ? c.value_scales : c.key_scales;
    // each row's registers take the next round's row as soon as its values are out of them
    Eight<T, WHOLE> x[kAhead<T>];
    auto load = [&](int i, int token) {
      if (real && token < count) x[i].load(from + token * t, item, W);
    };
#pragma unroll
    for (int i = 0; i < kAhead<T>; ++i) load(i, i * g.step + g.token);
    if (row0 == 0) {
      __syncthreads();
      find_places(c, b, token0, count, places, &least);
      __syncthreads();
      find_later(c, b, token0, count, places, least, later);
      __syncthreads();
    }
    for (int base = 0; base < count; base += kAhead<T> * g.step) {
#pragma unroll
      for (int i = 0; i < kAhead<T>; ++i) {
        float v[8], largest = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float(x[i].e[j]), largest = larger(largest, v[j]);
        const int token = base + i * g.step + g.token;
        load(i, token + kAhead<T> * g.step);
#pragma unroll
        for (int o = lanes / 2; o > 0; o /= 2) largest = larger(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        if (!real || token >= count || later[token]) continue;
        const Place place = places[token];
        if (place.page < 0) continue;
        // float(double(largest) / 127) of the rule: a quotient of 24-bit numbers rounded to 53 bits on the
        // way is never moved to another float32 by it
        const float scale = largest == 0.0f ? 1.0f : __fdiv_rn(largest, 127.0f);
        const long long at = ((long long)place.page * c.heads + head) * c.page + place.row;
        Eight<T, WHOLE>::store_codes(codes + at * W, item, W, codes_of<sizeof(T) == 2>(v, scale));
        if (item == 0) scales[at] = scale;
      }
    }
  }
}

template <typename T, int W, bool WHOLE>
__global__ void __launch_bounds__(kThreads) read_rows(const Cache c, const Batch b, const Rows keys, const Rows values, int each) {
  __shared__ Place places[kTokens];
  __shared__ int least;
  const long long token0 = (long long)blockIdx.x * each;
  const int count = (int)min((long long)each, b.tokens - token0);
  constexpr int lanes = W / 8, groups = kThreads / lanes;
  const int item = threadIdx.x % lanes;
  const Group g(threadIdx.x / lanes, groups, 2 * c.heads);
  if (threadIdx.x < kTokens) places[threadIdx.x] = Place{kNoSequence, -1};
  __syncthreads();
  find_places(c, b, token0, count, places, &least);
  __syncthreads();
  for (int row = g.row; row < g.rows; row += groups) {
    const bool value = row >= c.heads;
    const int head = value ? row - c.heads : row;
    const Rows& rows = value ? values : keys;
    T* to = reinterpret_cast<T*>(rows.data) + token0 * rows.t + head * rows.h;
    const long long t = rows.t;
    const int8_t* codes = value ? c.values : c.keys;
    const float* scales = value ? c.value_scales : c.key_scales;
    for (int base = g.token; base < count; base += kAhead<T> * g.step) {
      uint2 q[kAhead<T>];
      float scale[kAhead<T>];
      bool mine[kAhead<T>];
#pragma unroll
      for (int i = 0; i < kAhead<T>; ++i) {
        q[i] = make_uint2(0, 0);
        scale[i] = __int_as_float(0x7fffffff);
        const int token = base + i * g.step;
        const Place place = token < count ? places[token] : Place{kNoSequence, 0};
        mine[i] = place.page != kNoSequence;
        if (place.page >= 0) {
          const long long at = ((long long)place.page * c.heads + head) * c.page + place.row;
          q[i] = Eight<T, WHOLE>::load_codes(codes + at * W, item, W);
          scale[i] = scales[at];
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead<T>; ++i) {
        Eight<T, WHOLE> x;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int code = (int)(signed char)((j < 4 ? q[i].x : q[i].y) >> (8 * (j & 3)));
          x.e[j] = from_float<T>((float)code * scale[i]);
        }
        if (mine[i]) x.store(to + (base + i * g.step) * t, item, W);
      }
    }
  }
}

template <typename T, int W>
int run(const Cache& c, const Batch& b, const Rows& k, const Rows& v, bool read, cudaStream_t s) {
  if (b.tokens == 0) return TGCB_OK;
  // whole rounds of the 592 CTAs that are resident at once, of at most kTokens tokens each
  const long long rounds = (b.tokens + 592 * kTokens - 1) / (592 * kTokens);
  const int each = (int)((b.tokens + 592 * rounds - 1) / (592 * rounds));
  const unsigned grid = (unsigned)((b.tokens + each - 1) / each);
  bool whole = true;
  for (const Rows& r : {k, v})
    whole = whole && ((reinterpret_cast<uintptr_t>(r.data) | (unsigned long long)(r.t * (long long)sizeof(T)) |
                       (unsigned long long)(r.h * (long long)sizeof(T))) & 15u) == 0;
  if (read)
    (whole ? read_rows<T, W, true> : read_rows<T, W, false>)<<<grid, kThreads, 0, s>>>(c, b, k, v, each);
  else
    (whole ? append_rows<T, W, true> : append_rows<T, W, false>)<<<grid, kThreads, 0, s>>>(c, b, k, v, each);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, "kv_cache", cudaGetErrorString(e));
  return TGCB_OK;
}

template <typename T>
int by_width(const Cache& c, const Batch& b, const Rows& k, const Rows& v, bool read, cudaStream_t s) {
  switch (c.width) {
    case 32: return run<T, 32>(c, b, k, v, read, s);
    case 64: return run<T, 64>(c, b, k, v, read, s);
    case 128: return run<T, 128>(c, b, k, v, read, s);
    default: return run<T, 256>(c, b, k, v, read, s);
  }
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
    case TGCB_F32: return by_width<float>(c, b, k, v, read, s);
    case TGCB_BF16: return by_width<__nv_bfloat16>(c, b, k, v, read, s);
    default: return by_width<__half>(c, b, k, v, read, s);
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
