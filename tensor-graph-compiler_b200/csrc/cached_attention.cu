// Attention of single tokens, prompt pieces and drafted trees over the int8 cache.
//
// For a token at position P of its sequence and query head h, reading key head h / group: s_j = scale (q . k_j),
// capped to cap tanh(s_j / cap) on request, over the positions j the token sees; out = sum_j e^(s_j - m) v_j
// / sum_j e^(s_j - m) with m the largest s_j, found in one pass by rescaling what has been added
// whenever a larger score arrives.
#include <cuda_runtime.h>

#include <cmath>
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

struct Args {
  const char* q;
  char* out;
  long long q_t, q_h, out_t, out_h;
  const long long* visible;
  int q_heads;
  float scale, cap;
};

constexpr int kWarps = 4;

// One warp per token and query head, one key at a time.
template <typename T, int W>
__global__ void __launch_bounds__(32 * kWarps) attend_rows(const Cache c, const Batch b, const Args a) {
  __shared__ Place place;
  const long long token = blockIdx.x;
  if (threadIdx.x == 0) place.sequence = -1;
  __syncthreads();
  tgcb_kv::find(c, b, token, &place);
  __syncthreads();
  if (place.sequence < 0) return;
  const int lane = threadIdx.x & 31;
  constexpr int E = W / 32;
  long long first, last;
  tgcb_kv::range_of(b, place.sequence, &first, &last);
  const long long start = place.position - (token - first);
  const long long end = a.visible ? start + (last - first) : place.position + 1;
  const unsigned long long bits = a.visible ? (unsigned long long)a.visible[token] : 0ull;
  for (int head = threadIdx.x >> 5; head < a.q_heads; head += kWarps) {
    const T* q = reinterpret_cast<const T*>(a.q) + token * a.q_t + head * a.q_h;
    T* out = reinterpret_cast<T*>(a.out) + token * a.out_t + head * a.out_h;
    const int h = head / (a.q_heads / c.heads);
    float x[E], o[E], m = -INFINITY, sum = 0.f;
    bool any = false;
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = to_float(q[lane * E + i]), o[i] = 0.f;
    for (long long j = 0; j < end; ++j) {
      if (a.visible && j >= start && (j - start >= 64 || !((bits >> (j - start)) & 1))) continue;
      const int page = tgcb_kv::page_of(c, b, place.sequence, j);
      if (page < 0) continue;
      any = true;
      const long long at = ((long long)page * c.heads + h) * c.page + (j & (c.page - 1));
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) s = fmaf(x[i], (float)c.keys[at * W + lane * E + i], s);
#pragma unroll
      for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
      s = s * c.key_scales[at] * a.scale;
      if (a.cap > 0) s = a.cap * tanhf(s / a.cap);
      const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
      const float keep = expf(m - base), p = expf(s - base);
      m = mn;
      sum = sum * keep + p;
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = o[i] * keep + p * c.value_scales[at] * (float)c.values[at * W + lane * E + i];
    }
#pragma unroll
    for (int i = 0; i < E; ++i) out[lane * E + i] = from_float<T>(any ? o[i] / sum : 0.f);
  }
}

template <typename T, int W>
int launch(const Cache& c, const Batch& b, const Args& a, cudaStream_t s) {
  attend_rows<T, W><<<(unsigned)b.tokens, 32 * kWarps, 0, s>>>(c, b, a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, "cached_attention", cudaGetErrorString(e));
  return TGCB_OK;
}

template <typename T>
int run(const Cache& c, const Batch& b, const Args& a, cudaStream_t s) {
  switch (c.width) {
    case 32: return launch<T, 32>(c, b, a, s);
    case 64: return launch<T, 64>(c, b, a, s);
    case 128: return launch<T, 128>(c, b, a, s);
    default: return launch<T, 256>(c, b, a, s);
  }
}

}  // namespace

extern "C" {

size_t tgcb_cached_attention_scratch_bytes(const tgcb_cache* cache, const tgcb_batch* batch, int q_heads) {
  (void)cache, (void)batch, (void)q_heads;
  return 0;
}

int tgcb_cached_attention(const tgcb_cache* cache, const tgcb_batch* batch, int dtype, int q_heads,
                          const tgcb_heads* queries, const int64_t* visible, float scale, float cap,
                          const tgcb_heads* out, void* scratch, size_t scratch_bytes, void* stream) {
  const char* what = "tgcb_cached_attention";
  Cache c;
  Batch b;
  const int rc = tgcb_kv::checked(cache, batch, dtype, &c, &b, what);
  if (rc != TGCB_OK) return rc;
  auto bad = [&](const char* why) { return tgcb_internal_fail(TGCB_E_INVALID, what, why); };
  if (queries == nullptr || out == nullptr || (b.tokens > 0 && (queries->data == nullptr || out->data == nullptr)))
    return bad("null pointer");
  if (q_heads < 1 || q_heads % c.heads) return bad("the query heads must be a multiple of the cache's heads");
  if (!std::isfinite(scale)) return bad("the scale must be finite");
  if (!(cap >= 0) || std::isinf(cap)) return bad("the cap must be finite and not negative");
  if (b.tokens == 0) return TGCB_OK;
  (void)scratch, (void)scratch_bytes;
  const Args a = {static_cast<const char*>(queries->data), static_cast<char*>(out->data), queries->token_stride,
                  queries->head_stride, out->token_stride, out->head_stride,
                  reinterpret_cast<const long long*>(visible), q_heads, scale, cap};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TGCB_F32: return run<float>(c, b, a, s);
    case TGCB_BF16: return run<__nv_bfloat16>(c, b, a, s);
    default: return run<__half>(c, b, a, s);
  }
}

}  // extern "C"
