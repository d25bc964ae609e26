// What the kernels of attention over the int8 cache share: a call's arguments, how its work is cut into equal
// pieces, and the joining of units that were cut (cached_attention.cu, cached_attention_tc.cu).
#ifndef TGCB_CACHED_ATTENTION_CUH_
#define TGCB_CACHED_ATTENTION_CUH_

#include <cuda_runtime.h>

#include <cstdint>

#include "elements.cuh"
#include "internal.h"
#include "kv_cache.cuh"
#include "tgcb.h"

namespace tgcb_attend {

using namespace tgcb_elem;
using tgcb_kv::Batch;
using tgcb_kv::Cache;

struct Args {
  const char* q;
  char* out;
  long long q_t, q_h, out_t, out_h;
  const long long* visible;
  float* parts;   // [2 * CTAs][ROWS * (W + 2)]: weighted sums, then each row's maximum and sum of weights
  int4* cuts;     // [CTAs]: sequence (-1: none), head, row tile and last CTA of the unit that is cut at this CTA's end
  int group;      // query heads that share a key head
  float scale, cap;
  int capacity;   // positions a table row holds
  int whole;      // units are not cut
};

// Bytes 0 and 2 of a word of int8 codes as two bfloat16, each x / 64. With the sign bit flipped a byte is x + 128,
// and the bfloat16 whose low byte it is and whose high byte is zero has the value (x + 128) 2^-133, subnormal
// below 128 and normal from there; times 2^127, minus 2, is x 2^-6, exactly (the usual way to a float through its
// exponent's bits, in multiply-add form). `flip` and `mask` are
// 0x00800080 and 0x00ff00ff in registers, for with two constants in it the logic operation is issued twice.
// Against cutting the byte into its sign and its other bits and subtracting the two as
// bfloat16 numbers around 128: 1.5 arithmetic-logic instructions fewer for every two codes.
constexpr float kCodeScale = 64.f;
__device__ __forceinline__ unsigned codes(unsigned w, unsigned mask, unsigned flip) {
  unsigned u, r;
  asm("lop3.b32 %0, %1, %2, %3, 0x78;" : "=r"(u) : "r"(flip), "r"(w), "r"(mask));  // flip ^ (w & mask)
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(0x7f007f00u), "r"(0xc000c000u));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// float32 rows take CUDA's tanh (a few units in the last place). For 16-bit rows 1 - 2 / (1 + e^2x) is off by 2^-22, which
// is 2^-19 of the tangent from |x| = 1/4 on; below that the series x - x^3/3 + 2x^5/15 - 17x^7/315, off by 2^-21 of it, so
// that a cap far above the scores leaves them as they are (without the series caps from 10^6 on were wrong, and at 10^8 all
// scores 0). One tree of 13 nodes with a cap: 37 us, 35 without the series.
template <typename T>
__device__ __forceinline__ float tanh_of(float x) {
  if constexpr (sizeof(T) == 4) return tanhf(x);
  const float y = x * x, far = 1.f - __fdividef(2.f, 1.f + exp2_fast(2.885390081777927f * x));
  const float near = x * fmaf(y, fmaf(y, fmaf(y, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  return fabsf(x) < 0.25f ? near : far;
}

// Weighted values are added up before they are divided by the weights' sum, and up to 2^30 of them with values above 2^87 (a
// scale above 2^80) could leave float32's range. Such a key's weight is kept 2^kLargeMargin below one: its row's
// reference, against which weights and their sum are taken, is at least the key's score plus the margin, in units of
// log2 e. Other weights need none: 2^30 keys, 2^8 for a reference that may lag behind (cached_attention_tc.cu), 2^87.
constexpr float kLargeScale = 0x1p80f, kLargeMargin = 40.f;

// Two floats as N pairs of bfloat16 whose sums they are: the leading 8 bits cut off N - 1 times (exact
// remainders), the rest rounded.
template <int N>
__device__ __forceinline__ void split(float x, float y, unsigned* parts) {
#pragma unroll
  for (int i = 0; i < N - 1; ++i) {
    parts[i] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
  }
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(parts[N - 1]) : "f"(y), "f"(x));
}

// A sequence's rows, units and steps.
struct Sequence {
  long long first;  // its first token row
  int rows, tiles;  // token rows; tiles of ROWS query rows
  long long start;
  int end;    // positions that its last row may see
  int steps;  // of STEP positions, of one unit
};

template <int ROWS, int STEP>
__device__ __forceinline__ Sequence sequence_of(const Batch& b, const Args& a, int s) {
  Sequence q;
  long long last;
  tgcb_kv::range_of(b, s, &q.first, &last);
  q.rows = (int)(last - q.first);
  q.tiles = (int)(((long long)q.rows * a.group + ROWS - 1) / ROWS);
  q.start = __ldg(b.starts + s);
  const long long end = q.start + q.rows;
  q.end = (int)(end < 0 ? 0 : end > a.capacity ? a.capacity : end);
  q.steps = max(1, (q.end + STEP - 1) / STEP);
  return q;
}

// Counts a sequence that has positions before the first or past its table, once.
__device__ __forceinline__ void count_outside(const Cache& c, const Sequence& q, const Args& a, bool once) {
  if (once && (q.start < 0 || q.start + q.rows > a.capacity)) atomicAdd(c.faults, 1);
}

template <int ROWS, int STEP>
__device__ __forceinline__ long long work_of(const Cache& c, const Batch& b, const Args& a, int s) {
  const Sequence q = sequence_of<ROWS, STEP>(b, a, s);
  return (long long)c.heads * q.tiles * (a.whole ? 1 : q.steps);
}

struct Begin {
  long long total, offset;  // all work; this CTA's first piece within its first sequence
  int sequence;
};

// Where this CTA's share of the work begins: the threads add up consecutive sequences, the CTA
// scans the sums, and the thread in whose sequences the share begins walks to it.
template <int ROWS, int STEP, int WARPS>
__device__ __forceinline__ void begin_at(const Cache& c, const Batch& b, const Args& a, int least, long long* chunk, Begin* out) {
  __shared__ long long warp_sums[WARPS];
  const int per = (b.batch + 32 * WARPS - 1) / (32 * WARPS);
  const int s0 = min(threadIdx.x * per, b.batch), s1 = min(s0 + per, b.batch);
  long long mine = 0;
  for (int s = s0; s < s1; ++s) mine += work_of<ROWS, STEP>(c, b, a, s);
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if ((threadIdx.x & 31) >= o) upto += v;
  }
  if ((threadIdx.x & 31) == 31) warp_sums[threadIdx.x >> 5] = upto;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < (int)(threadIdx.x >> 5)) upto += warp_sums[w];
    total += warp_sums[w];
  }
  long long share = (total + gridDim.x - 1) / gridDim.x;
  share = share < (a.whole ? 1 : least) ? (a.whole ? 1 : least) : share;
  *chunk = share;
  const long long target = blockIdx.x * share;
  if (threadIdx.x == 0) out->total = total;
  if (target >= upto - mine && target < upto) {
    long long left = target - (upto - mine);
    int s = s0;
    for (;; ++s) {
      const long long w = work_of<ROWS, STEP>(c, b, a, s);
      if (left < w) break;
      left -= w;
    }
    out->sequence = s;
    out->offset = left;
  }
  __syncthreads();
}

// Sums of weights of parts, where -1 marks a part whose scores were all -infinity: its factor is 0 beside
// any other part, and a row with nothing else has no answer (NaN, as 0 / 0). Without branches, which
// would hold back the loads of the parts behind them.
struct Weights {
  float all = 0.f;
  bool lowest = false;
  __device__ __forceinline__ void add(float sum, float factor) {
    lowest |= sum < 0.f;
    all = fmaf(sum < 0.f ? 0.f : sum, factor, all);
  }
  __device__ __forceinline__ float sum() const { return all == 0.f && lowest ? -1.f : all; }
};
__device__ __forceinline__ float answer(float v, float sum) {
  return sum == 0.f ? 0.f : sum < 0.f ? __int_as_float(0x7fffffff) : v / sum;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float* v, bool wide) {
  if (wide) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      union {
        uint2 raw;
        T e[4];
      } x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.e[i] = from_float<T>(v[i]);
      *reinterpret_cast<uint2*>(p) = x.raw;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = from_float<T>(v[i]);
  }
}

template <typename T>
__device__ __forceinline__ T* out_row(const Args& a, const Sequence& q, int head, int row) {
  const int token = row / a.group, in_group = row - token * a.group;
  return reinterpret_cast<T*>(a.out) + (q.first + token) * a.out_t + (long long)(head * a.group + in_group) * a.out_h;
}

template <typename T>
__device__ __forceinline__ bool out_wide(const Args& a) {
  return ((reinterpret_cast<uintptr_t>(a.out) | (unsigned long long)(a.out_t * sizeof(T)) | (unsigned long long)(a.out_h * sizeof(T))) &
          (4 * sizeof(T) - 1)) == 0;
}

// Joins the parts of the unit that begins in CTA blockIdx.x of `attend` and was cut at its end, in the
// order of the keys: a warp per row, first the parts' maxima and sums (a lane per part), then the
// weighted sums (a lane per four columns), eight parts' loads in flight.
template <typename T, int W, int RN>
__global__ void __launch_bounds__(256) combine(const Cache c, const Batch b, const Args a) {
  constexpr int ROWS = 8 * RN, QUADS = W / 4, PER = (QUADS + 31) / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.x < 0) return;
  const Sequence q = sequence_of<ROWS, 32>(b, a, cut.x);
  const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (r >= q.rows * a.group - cut.z * ROWS) return;
  const int n = cut.w - blockIdx.x + 1;
  auto part = [&](int i) { return a.parts + (i == 0 ? 2ll * blockIdx.x + 1 : 2ll * (blockIdx.x + i)) * ROWS * (W + 2); };
  float mm = -INFINITY;
  for (int k = lane; k < n; k += 32) mm = fmaxf(mm, part(k)[ROWS * W + 2 * r]);
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
  const float base = mm == -INFINITY ? 0.f : mm;
  Weights all;
  float v[PER][4];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
  for (int k0 = 0; k0 < n; k0 += 32) {
    float mine = 0.f, weights = 0.f;
    if (k0 + lane < n) {
      const float2 ml = *reinterpret_cast<const float2*>(part(k0 + lane) + ROWS * W + 2 * r);
      mine = exp2_fast(ml.x - base), weights = ml.y;
    }
    const int some = min(32, n - k0);
#pragma unroll 8
    for (int k = 0; k < some; ++k) {
      const float f = __shfl_sync(0xffffffffu, mine, k);
      all.add(__shfl_sync(0xffffffffu, weights, k), f);
      const float* p = part(k0 + k) + r * W;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (QUADS >= 32 || lane < QUADS) {
          const float4 x = *reinterpret_cast<const float4*>(p + 4 * (lane + 32 * i));
          v[i][0] = fmaf(x.x, f, v[i][0]), v[i][1] = fmaf(x.y, f, v[i][1]);
          v[i][2] = fmaf(x.z, f, v[i][2]), v[i][3] = fmaf(x.w, f, v[i][3]);
        }
    }
  }
  const bool wide = out_wide<T>(a);
  const float all_sum = all.sum();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (QUADS >= 32 || lane < QUADS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = answer(v[i][j], all_sum);
      store4<T>(out_row<T>(a, q, cut.y, cut.z * ROWS + r) + 4 * (lane + 32 * i), v[i], wide);
    }
}

// Queues `combine` behind the kernel whose CTAs left the parts.
template <typename T, int W, int RN>
cudaError_t launch_combine(const Cache& c, const Batch& b, const Args& a, unsigned ctas, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, RN);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, combine<T, W, RN>, c, b, a);
}

// Units of up to 128 query rows on tcgen05 (cached_attention_tc.cu): 16-bit rows, widths 64 and 128.
constexpr int kTensorRows = 128;
constexpr int kTensorCtas = 148;
int attend_tensor(const Cache& c, const Batch& b, const Args& a, int dtype, cudaStream_t s);

}  // namespace tgcb_attend

#endif  // TGCB_CACHED_ATTENTION_CUH_
