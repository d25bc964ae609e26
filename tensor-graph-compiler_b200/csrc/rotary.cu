// RMS norm of query and key heads with the position rotation in the same pass, forward and backward.
//
// A head row x of `width` columns: r = 1 / sqrt(mean(x^2) + eps), y = x r g, and for the first
// `rotary` columns each pair (a, b) of y becomes (a cos t - b sin t, a sin t + b cos t) with
// t = position * frequency. The rotation is orthogonal, so the backward pass turns the output
// gradients by -t: d = rotate(dout, -t); dgain = sum over rows of d x r; with e = g d,
// dx = r (e - x r^2 mean(e x)).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "elements.cuh"
#include "internal.h"
#include "tgcb.h"

namespace {

using namespace tgcb_elem;

constexpr int kMaxWidth = 1024;
constexpr int kPartials = 592;  // CTAs of a backward pass, each with one partial row of gain gradients per side

struct Side {
  const void* in;
  const void* grad;
  void* out;
  const void* gain;
  void* gain_grad;
  long long in_t, in_h, grad_t, grad_h, out_t, out_h;
  int heads;
};

struct Params {
  Side side[2];
  const void* positions;
  const double* frequencies;
  float* partials;
  long long tokens;
  int gain_dtype, position_bytes, interleaved, width, rotary;
  float epsilon, by_width;
};

// cos and sin of position * frequency. The half turns are taken in float64 (a far position has many of them
// and float32 would lose the angle) and reduced to one either way, so that rounding the rest to
// float32 costs 2^-25 of a half turn at most.
__device__ __forceinline__ void turn(double position, double frequency, float* c, float* s) {
  const double halves = position * (frequency * 0.31830988618379067154);  // 1 / pi
  sincospif((float)(halves - 2.0 * rint(0.5 * halves)), s, c);
}

__device__ __forceinline__ double position_of(const Params& p, long long token) {
  return p.position_bytes == 8 ? (double)static_cast<const long long*>(p.positions)[token]
                               : (double)static_cast<const int*>(p.positions)[token];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Any width, stride and alignment: one warp per row, elements one by one, each pair's angle computed
// where it is used. A lane reads a pair whole before it writes it, so the output may be the input.
constexpr int kRowWarps = 4;

template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(32 * kRowWarps) norm_rotate_rows(const Params p) {
  extern __shared__ float sums[];  // backward: [warp][side][width], each lane adding to its own columns
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = p.rotary / 2, heads = p.side[0].heads + p.side[1].heads;
  const long long rows = p.tokens * heads;
  if (BACKWARD) {
    for (int i = threadIdx.x; i < kRowWarps * 2 * p.width; i += 32 * kRowWarps) sums[i] = 0.f;
    __syncthreads();
  }
  for (long long row = (long long)blockIdx.x * kRowWarps + warp; row < rows; row += (long long)gridDim.x * kRowWarps) {
    const long long token = row / heads;
    int head = (int)(row - token * heads);
    const int which = head >= p.side[0].heads;
    const Side& s = p.side[which];
    if (which) head -= p.side[0].heads;
    const T* x = static_cast<const T*>(s.in) + token * s.in_t + head * s.in_h;
    const T* g = BACKWARD ? static_cast<const T*>(s.grad) + token * s.grad_t + head * s.grad_h : nullptr;
    T* y = static_cast<T*>(s.out) + token * s.out_t + head * s.out_h;
    const double position = position_of(p, token);

    float square = 0.f;
    for (int c = lane; c < p.width; c += 32) {
      const float v = to_float(x[c]);
      square = fmaf(v, v, square);
    }
    const float r = rsqrtf(fmaf(warp_sum(square), p.by_width, p.epsilon));

    // items: `half` pairs, then the single columns behind them
    const int items = half + p.width - p.rotary;
    float ex = 0.f;  // backward: sum of e x
    for (int phase = BACKWARD ? 0 : 1; phase < 2; ++phase) {
      for (int i = lane; i < items; i += 32) {
        const bool pair = i < half;
        const int c0 = pair ? (p.interleaved ? 2 * i : i) : p.rotary + i - half;
        const int c1 = p.interleaved ? c0 + 1 : c0 + half;
        float cs = 1.f, sn = 0.f;
        if (pair) turn(position, p.frequencies[i], &cs, &sn);
        const float x0 = to_float(x[c0]), x1 = pair ? to_float(x[c1]) : 0.f;
        const float g0 = load_any(s.gain, p.gain_dtype, c0), g1 = pair ? load_any(s.gain, p.gain_dtype, c1) : 0.f;
        if (!BACKWARD) {
          const float a = x0 * r * g0, b = x1 * r * g1;
          y[c0] = from_float<T>(a * cs - b * sn);
          if (pair) y[c1] = from_float<T>(a * sn + b * cs);
        } else {
          const float u = to_float(g[c0]), v = pair ? to_float(g[c1]) : 0.f;
          const float d0 = u * cs + v * sn, d1 = v * cs - u * sn;
          if (phase == 0) {
            ex += d0 * g0 * x0 + d1 * g1 * x1;
            float* mine = sums + (warp * 2 + which) * p.width;
            mine[c0] += d0 * x0 * r;
            if (pair) mine[c1] += d1 * x1 * r;
          } else {
            const float m = ex * r * r * p.by_width;
            y[c0] = from_float<T>(r * (d0 * g0 - x0 * m));
            if (pair) y[c1] = from_float<T>(r * (d1 * g1 - x1 * m));
          }
        }
      }
      if (BACKWARD && phase == 0) ex = warp_sum(ex);
    }
  }
  if (BACKWARD) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.width; i += 32 * kRowWarps) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) v += sums[w * 2 * p.width + i];
      p.partials[(long long)blockIdx.x * 2 * p.width + i] = v;
    }
  }
}

// Rows of 16-byte vectors. A group of `lanes` threads has one row: thread i of it holds two vectors, which in the turned
// columns are the two halves of its pairs (or, interleaved, two vectors of whole pairs), so that a
// pair never leaves its thread, and neighbouring threads' vectors lie side by side. A CTA takes `tokens_each` tokens at a time, with `groups[side]` groups a side for each
// (a side's heads in `passes` rounds); a group always has the same side and columns.
//
// Bound by HBM: each row is read and written once (backward: two read, one written). What has to be
// hidden is the latency of the rows and of the angles (float64 products, once a token for all
// heads). So CTAs are persistent, and each thread copies its own vectors kStages - 1 steps ahead into slots of
// shared memory that no other thread touches. Angles are computed for as many tiles of tokens at a time (a
// batch) as gives every thread one, a batch ahead, so that there is one barrier a batch. Measured, 8192 tokens
// of 32 + 8 bfloat16 heads of 128: forward 40 us (168 MB, 4.2 TB/s), backward 56 us (252 MB, 4.5 TB/s), held by
// their instructions (some 350 a warp and step, for 16-bit elements twice the float32 ones' a byte; instructions on pairs of
// float32 values are not used); 4095 tokens
// of 16 + 4 float32 heads, backward: 20 us (126 MB, 6.2 TB/s).
// Threads a CTA has at most, and the CTAs of that size that fit an SM's registers: 64 a thread forward, 102 backward.
constexpr int kVecThreads[2] = {512, 320};
constexpr int kVecResident = 2;
constexpr int kStages = 4;
constexpr size_t kMaxShared = 200 * 1024;

struct Layout {
  int items, lanes_log, groups[2], tokens_each, passes, threads, batch;
  size_t shared;
};

__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

template <int N>
__device__ __forceinline__ void load_floats(const float* p, float* out) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + i);
      out[i] = x.x, out[i + 1] = x.y, out[i + 2] = x.z, out[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 x = *reinterpret_cast<const float2*>(p + i);
      out[i] = x.x, out[i + 1] = x.y;
    }
  }
}

// Turns the pairs of two vectors, by the angles that begin at `cosines` + turn_a and + turn_b (-1: not turned).
template <int V, bool INTERLEAVED, bool BACK>
__device__ __forceinline__ void turn_vectors(float* a, float* b, const float* cosines, int sines, int turn_a, int turn_b) {
  auto pair = [](float* x, float* y, float c, float s) {
    const float u = *x, v = *y;
    *x = BACK ? u * c + v * s : u * c - v * s;
    *y = BACK ? v * c - u * s : u * s + v * c;
  };
  if constexpr (!INTERLEAVED) {
    if (turn_a < 0) return;
    float c[V], s[V];
    load_floats<V>(cosines + turn_a, c), load_floats<V>(cosines + sines + turn_a, s);
#pragma unroll
    for (int i = 0; i < V; ++i) pair(a + i, b + i, c[i], s[i]);
  } else {
    float c[V / 2], s[V / 2];
    if (turn_a >= 0) {
      load_floats<V / 2>(cosines + turn_a, c), load_floats<V / 2>(cosines + sines + turn_a, s);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) pair(a + 2 * i, a + 2 * i + 1, c[i], s[i]);
    }
    if (turn_b >= 0) {
      load_floats<V / 2>(cosines + turn_b, c), load_floats<V / 2>(cosines + sines + turn_b, s);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) pair(b + 2 * i, b + 2 * i + 1, c[i], s[i]);
    }
  }
}

template <typename T, bool INTERLEAVED, bool BACKWARD>
__global__ void __launch_bounds__(kVecThreads[BACKWARD], kVecResident) norm_rotate_vectors(const Params p, const Layout layout) {
  constexpr int V = Vec<T>::N, SLOTS = BACKWARD ? 4 : 2;
  if (BACKWARD) asm volatile("griddepcontrol.launch_dependents;");  // gain_sums, which waits for the end
  // slots [stage][vector][thread] of 16 bytes, gains [side][width], cosines and sines [2 buffers][batch][tokens_each]
  // [cos, sin][half rounded up to 4]; at the end the sums
  extern __shared__ __align__(16) float shared[];
  const int half = p.rotary / 2, sines = (half + 3) & ~3, lanes = 1 << layout.lanes_log, per_token = layout.groups[0] + layout.groups[1];
  const int group = threadIdx.x >> layout.lanes_log, item = threadIdx.x & (lanes - 1);
  const int token_in = group / per_token, in_token = group - token_in * per_token;
  const int which = in_token >= layout.groups[0];
  const Side& s = p.side[which];
  const int head0 = which ? in_token - layout.groups[0] : in_token, heads_step = layout.groups[which];
  const bool working = token_in < layout.tokens_each;

  // this thread's columns a and b, V of each, and the first of the frequencies that turn them (-1: none)
  int a, b, turn_a, turn_b;
  if (INTERLEAVED) {
    a = item * V, b = a + layout.items * V;
    turn_a = a < p.rotary ? a / 2 : -1, turn_b = b < p.rotary ? b / 2 : -1;
  } else {
    const int pairs = half / V;
    const bool paired = item < pairs;
    a = paired ? item * V : p.rotary + (item - pairs) * V;
    b = paired ? half + item * V : a + (layout.items - pairs) * V;
    turn_a = turn_b = paired ? item * V : -1;
  }
  const bool has_a = working && item < layout.items, has_b = has_a && b < p.width;
  if (!has_a) a = 0;
  if (!has_b) b = 0;
  const unsigned slots_at = static_cast<unsigned>(__cvta_generic_to_shared(shared)) + threadIdx.x * 16, slot = blockDim.x * 16;
  const unsigned stage_bytes = SLOTS * slot, ring_end = kStages * stage_bytes;
  float* gains = shared + kStages * SLOTS * blockDim.x * 4;
  float* all_angles = gains + 2 * p.width;
  for (int i = threadIdx.x; i < 2 * p.width; i += blockDim.x)
    gains[i] = load_any(p.side[i >= p.width].gain, p.gain_dtype, i >= p.width ? i - p.width : i);
  const float *gain_a = gains + which * p.width + a, *gain_b = gains + which * p.width + b;
  float sum_a[V], sum_b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum_a[i] = sum_b[i] = 0.f;

  const long long tiles = (p.tokens + layout.tokens_each - 1) / layout.tokens_each;
  const long long tile_step = (long long)gridDim.x * layout.tokens_each, tile0 = (long long)blockIdx.x * layout.tokens_each;
  const int mine = (int)((tiles - blockIdx.x + gridDim.x - 1) / gridDim.x);  // this CTA's tiles, one at least
  const long long in_step = tile_step * s.in_t, grad_step = tile_step * s.grad_t, out_step = tile_step * s.out_t;

  // angles of the batch of tiles that begins at token row token0; a thread's first is the same each time
  const int per_tile = layout.tokens_each * half;
  auto angle_at = [&](int i, long long* token, int* f, int* at) {
    const int tile = i / per_tile, in_tile = i - tile * per_tile, t = in_tile / half;
    *f = in_tile - t * half;
    *token = tile * tile_step + t;
    *at = (tile * layout.tokens_each + t) * 2 * sines + *f;
  };
  long long angle_token = 0;
  int angle_f = 0, angle_to = 0;
  angle_at(threadIdx.x, &angle_token, &angle_f, &angle_to);
  const double angle_frequency = p.frequencies[angle_f];
  auto angles_of = [&](long long token0, float* to) {
    if (threadIdx.x >= layout.batch * per_tile) return;
    if (token0 + angle_token < p.tokens) turn(position_of(p, token0 + angle_token), angle_frequency, to + angle_to, to + angle_to + sines);
    for (int i = threadIdx.x + blockDim.x; i < layout.batch * per_tile; i += blockDim.x) {  // only where one tile has more angles than the CTA threads
      long long token;
      int f, at;
      angle_at(i, &token, &f, &at);
      if (token0 + token < p.tokens) turn(position_of(p, token0 + token), p.frequencies[f], to + at, to + at + sines);
    }
  };
  const int token_floats = layout.tokens_each * 2 * sines, batch_floats = layout.batch * token_floats;

  for (int pass = 0; pass < layout.passes; ++pass) {
    const int head = head0 + pass * heads_step;
    const bool mine_too = working && head < s.heads;
    const int h = mine_too ? head : 0;
    // rows of this pass that are this thread's: the tokens tile0 + token_in, a tile_step further each
    const int tokens_left = mine_too && tile0 + token_in < p.tokens ? (int)((p.tokens - tile0 - token_in + tile_step - 1) / tile_step) : 0;
    const long long first = tokens_left ? tile0 + token_in : 0;
    const T* x = static_cast<const T*>(s.in) + first * s.in_t + h * s.in_h;
    const T* d = BACKWARD ? static_cast<const T*>(s.grad) + first * s.grad_t + h * s.grad_h : nullptr;
    T* y = static_cast<T*>(s.out) + first * s.out_t + h * s.out_h;
    int ahead_left = tokens_left;
    unsigned ahead_at = 0, now_at = 0;
    auto copy_ahead = [&]() {
      const bool row = ahead_left > 0;
      --ahead_left;
      const unsigned to = slots_at + ahead_at;
      ahead_at = ahead_at + stage_bytes == ring_end ? 0 : ahead_at + stage_bytes;
      copy16(to, x + a, row && has_a);
      copy16(to + slot, x + b, row && has_b);
      if (BACKWARD) {
        copy16(to + 2 * slot, d + a, row && has_a);
        copy16(to + 3 * slot, d + b, row && has_b);
        if (ahead_left > 0) d += grad_step;
      }
      if (ahead_left > 0) x += in_step;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) copy_ahead();
    __syncthreads();  // the last pass's angles are used up
    angles_of(tile0, all_angles);
    int buffer = 0, in_batch = 0;

    for (int tile = 0; tile < mine; ++tile) {
      if (in_batch == 0) {
        __syncthreads();  // this batch's angles are there, and the other buffer's are used up
        if (tile + layout.batch < mine) angles_of(tile0 + (tile + layout.batch) * tile_step, all_angles + (buffer ^ 1) * batch_floats);
      }
      // (cos, sin) of vector a's and vector b's pairs; of the half-split order a pair is (a[i], b[i])
      const float* cs = all_angles + buffer * batch_floats + in_batch * token_floats + (working ? token_in : 0) * 2 * sines;
      if (++in_batch == layout.batch) in_batch = 0, buffer ^= 1;
      copy_ahead();
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      const bool row = tile < tokens_left;
      const char* from = reinterpret_cast<const char*>(shared) + threadIdx.x * 16 + now_at;
      now_at = now_at + stage_bytes == ring_end ? 0 : now_at + stage_bytes;
      Vec<T> xa, xb;
      xa.raw = *reinterpret_cast<const uint4*>(from), xb.raw = *reinterpret_cast<const uint4*>(from + slot);
      float fa[V], fb[V], wa[V], wb[V], square = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        fa[i] = to_float(xa.e[i]), fb[i] = to_float(xb.e[i]);
        square = fmaf(fa[i], fa[i], square);
        square = fmaf(fb[i], fb[i], square);
      }
      load_floats<V>(gain_a, wa), load_floats<V>(gain_b, wb);
      if (!BACKWARD) {
        for (int o = lanes >> 1; o > 0; o >>= 1) square += __shfl_xor_sync(0xffffffffu, square, o);
        const float r = rsqrtf(fmaf(square, p.by_width, p.epsilon));
#pragma unroll
        for (int i = 0; i < V; ++i) fa[i] = fa[i] * r * wa[i], fb[i] = fb[i] * r * wb[i];
        turn_vectors<V, INTERLEAVED, false>(fa, fb, cs, sines, turn_a, turn_b);
      } else {
        Vec<T> da, db;
        da.raw = *reinterpret_cast<const uint4*>(from + 2 * slot), db.raw = *reinterpret_cast<const uint4*>(from + 3 * slot);
        float ga[V], gb[V], ex = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) ga[i] = to_float(da.e[i]), gb[i] = to_float(db.e[i]);
        turn_vectors<V, INTERLEAVED, true>(ga, gb, cs, sines, turn_a, turn_b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          ex = fmaf(ga[i] * wa[i], fa[i], ex);
          ex = fmaf(gb[i] * wb[i], fb[i], ex);
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) {
          square += __shfl_xor_sync(0xffffffffu, square, o);
          ex += __shfl_xor_sync(0xffffffffu, ex, o);
        }
        const float r = rsqrtf(fmaf(square, p.by_width, p.epsilon)), m = ex * r * r * p.by_width;
        if (row) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            sum_a[i] = fmaf(ga[i] * r, fa[i], sum_a[i]);
            sum_b[i] = fmaf(gb[i] * r, fb[i], sum_b[i]);
            fa[i] = r * (ga[i] * wa[i] - fa[i] * m);
            fb[i] = r * (gb[i] * wb[i] - fb[i] * m);
          }
        }
      }
      if (row) {
        if (has_a) store_vec<T>(y + a, fa);
        if (has_b) store_vec<T>(y + b, fb);
        y += out_step;
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  if (BACKWARD) {  // this CTA's gain gradients: the groups of a side added up in order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (has_a) shared[group * p.width + a + i] = sum_a[i];
      if (has_b) shared[group * p.width + b + i] = sum_b[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.width; c += blockDim.x) {
      const int side = c >= p.width, column = c - side * p.width;
      float v = 0.f;
      for (int t = 0; t < layout.tokens_each; ++t)
        for (int g = side ? layout.groups[0] : 0; g < (side ? per_token : layout.groups[0]); ++g)
          v += shared[(t * per_token + g) * p.width + column];
      p.partials[(long long)blockIdx.x * 2 * p.width + c] = v;
    }
  }
}

// Whether the vector kernel takes these rows, and how. Other rows (widths that are no multiple of 16 bytes, odd halves,
// rows off a 16-byte boundary) take norm_rotate_rows: the same 8192 tokens there in 150 us forward and 519 us backward.
template <typename T>
bool vectors(const Params& p, bool backward, Layout* out) {
  constexpr int V = Vec<T>::N;
  const int half = p.rotary / 2;
  if (p.width % V || (p.interleaved ? p.rotary % V : half % V)) return false;
  auto whole = [](const void* data, long long t, long long h) {
    return ((reinterpret_cast<uintptr_t>(data) | (unsigned long long)(t * (long long)sizeof(T)) | (unsigned long long)(h * (long long)sizeof(T))) & 15u) == 0;
  };
  for (const Side& s : p.side)
    if (!whole(s.in, s.in_t, s.in_h) || !whole(s.out, s.out_t, s.out_h) || (backward && !whole(s.grad, s.grad_t, s.grad_h))) return false;
  const int single = p.width / V, items = p.interleaved ? (single + 1) / 2 : half / V + (single - p.rotary / V + 1) / 2;
  Layout l = {};
  l.items = items;
  while ((1 << l.lanes_log) < items) ++l.lanes_log;
  if (l.lanes_log > 5) return false;
  const int most = kVecThreads[backward] >> l.lanes_log;
  for (l.passes = 1;; ++l.passes) {
    for (int i = 0; i < 2; ++i) l.groups[i] = (p.side[i].heads + l.passes - 1) / l.passes;
    if (l.groups[0] + l.groups[1] <= most) break;
  }
  // several tokens a CTA where one has few heads and there are tiles enough
  const int per_token = l.groups[0] + l.groups[1];
  l.tokens_each = 1;
  while (2 * l.tokens_each * per_token <= most / 2 && p.tokens / (2 * l.tokens_each) >= 148 * 8) l.tokens_each *= 2;
  l.threads = ((l.tokens_each * per_token << l.lanes_log) + 31) / 32 * 32;
  l.batch = std::max(1, l.threads / (l.tokens_each * half));
  l.shared = (2ull * p.width + 2ull * l.batch * l.tokens_each * 2 * ((half + 3) & ~3)) * sizeof(float) + (size_t)kStages * (backward ? 4 : 2) * l.threads * 16;
  const size_t sums = backward ? (size_t)(l.threads >> l.lanes_log) * p.width * sizeof(float) : 0;
  if (sums > l.shared) l.shared = sums;
  *out = l;
  return l.shared <= kMaxShared;
}

// The gain gradients: column sums of the CTAs' partial rows, in float64 and in a fixed order. 32 warps
// for 32 columns, each with all its rows' loads in flight; with 8 warps that waited for every
// load 592 partial rows took 30 us.
__global__ void __launch_bounds__(1024) gain_sums(const Params p, int partials) {
  __shared__ double part[32][33];
  constexpr int PER = (kPartials + 31) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float x[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = warp + 32 * i;
    x[i] = c < 2 * p.width && row < partials ? __ldcg(p.partials + (long long)row * 2 * p.width + c) : 0.f;
  }
  double v = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) v += (double)x[i];
  part[warp][lane] = v;
  __syncthreads();
  // warp w adds up column w
  v = part[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
  const int column = blockIdx.x * 32 + warp;
  if (lane == 0 && column < 2 * p.width) {
    const int which = column >= p.width;
    store_any(p.side[which].gain_grad, p.gain_dtype, column - which * p.width, (float)v);
  }
}

int check(const tgcb_rotary_desc* d, bool backward, const char* what) {
  auto bad = [&](const char* why) { return tgcb_internal_fail(TGCB_E_INVALID, what, why); };
  if (d == nullptr) return bad("null descriptor");
  if (d->dtype < TGCB_F32 || d->dtype > TGCB_F16) return bad("unknown element type");
  if (d->gain_dtype != TGCB_F32 && d->gain_dtype != d->dtype) return bad("the gains are float32 or of the rows' type");
  if (d->position_bytes != 4 && d->position_bytes != 8) return bad("positions are 4- or 8-byte integers");
  if (d->tokens < 0) return bad("negative token count");
  if (d->heads[0] < 1 || d->heads[1] < 1 || d->heads[0] > (1 << 20) || d->heads[1] > (1 << 20))
    return bad("there is at least one query head and one key head, and at most 2^20");
  if (d->tokens > (1ll << 40)) return bad("too many tokens");
  if (d->width < 2 || d->width > kMaxWidth) return bad("width must be from 2 to 1024");
  if (d->rotary < 2 || d->rotary > d->width || d->rotary % 2) return bad("rotary must be even, from 2 to width");
  if (!(d->epsilon > 0) || !((float)d->epsilon > 0) || std::isinf((float)d->epsilon)) return bad("epsilon must be a positive float32");
  for (int i = 0; i < 2; ++i) {
    if (d->gain[i] == nullptr || d->frequencies == nullptr) return bad("null pointer");
    if (backward && d->gain_grad[i] == nullptr) return bad("null pointer");
    if (d->tokens > 0 && (d->in[i].data == nullptr || d->out[i].data == nullptr || d->positions == nullptr ||
                          (backward && d->grad[i].data == nullptr)))
      return bad("null pointer");
  }
  if (backward && (d->scratch == nullptr || d->scratch_bytes < tgcb_norm_rotate_scratch_bytes(d->width)))
    return bad("scratch is smaller than tgcb_norm_rotate_scratch_bytes");
  if (backward && (reinterpret_cast<uintptr_t>(d->scratch) & 15u)) return bad("scratch must be 16-byte aligned");
  return TGCB_OK;
}

Params params_of(const tgcb_rotary_desc* d) {
  Params p = {};
  for (int i = 0; i < 2; ++i) {
    Side& s = p.side[i];
    s.in = d->in[i].data, s.in_t = d->in[i].token_stride, s.in_h = d->in[i].head_stride;
    s.grad = d->grad[i].data, s.grad_t = d->grad[i].token_stride, s.grad_h = d->grad[i].head_stride;
    s.out = d->out[i].data, s.out_t = d->out[i].token_stride, s.out_h = d->out[i].head_stride;
    s.gain = d->gain[i], s.gain_grad = d->gain_grad[i], s.heads = d->heads[i];
  }
  p.positions = d->positions, p.frequencies = d->frequencies, p.partials = static_cast<float*>(d->scratch);
  p.tokens = d->tokens, p.gain_dtype = d->gain_dtype, p.position_bytes = d->position_bytes;
  p.interleaved = d->interleaved != 0, p.width = d->width, p.rotary = d->rotary, p.epsilon = (float)d->epsilon;
  p.by_width = (float)(1.0 / d->width);
  return p;
}

int failed(cudaError_t e) { return e == cudaSuccess ? TGCB_OK : tgcb_internal_fail(TGCB_E_CUDA, "norm_rotate", cudaGetErrorString(e)); }

// Queued behind the kernel that writes the partial rows, and resident before it ends.
int run_gain_sums(const Params& p, unsigned partials, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((2 * p.width + 31) / 32);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return failed(cudaLaunchKernelEx(&cfg, gain_sums, p, (int)partials));
}

template <typename T, bool INTERLEAVED, bool BACKWARD>
int run_vectors(const Params& p, const Layout& l, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return failed(e);
  static std::atomic<unsigned long long> configured{0};
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    e = cudaFuncSetAttribute(norm_rotate_vectors<T, INTERLEAVED, BACKWARD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxShared);
    if (e != cudaSuccess) return failed(e);
    configured.fetch_or(bit);
  }
  const long long tiles = (p.tokens + l.tokens_each - 1) / l.tokens_each;
  // one CTA for each that fits
  const long long by_registers = kVecThreads[BACKWARD] * kVecResident / l.threads, by_shared = 227 * 1024 / (l.shared + 1024);
  const long long resident = 148 * std::max(1ll, std::min({by_registers, by_shared, 2048ll / l.threads}));
  const unsigned grid = (unsigned)std::min({tiles, resident, (long long)kPartials});
  norm_rotate_vectors<T, INTERLEAVED, BACKWARD><<<grid, l.threads, l.shared, s>>>(p, l);
  e = cudaGetLastError();
  if (e != cudaSuccess) return failed(e);
  return BACKWARD ? run_gain_sums(p, grid, s) : TGCB_OK;
}

template <typename T>
int run(const Params& p, bool backward, cudaStream_t s) {
  Layout l;
  if (p.tokens > 0 && vectors<T>(p, backward, &l)) {
    if (backward) return p.interleaved ? run_vectors<T, true, true>(p, l, s) : run_vectors<T, false, true>(p, l, s);
    return p.interleaved ? run_vectors<T, true, false>(p, l, s) : run_vectors<T, false, false>(p, l, s);
  }
  const long long rows = p.tokens * (p.side[0].heads + p.side[1].heads);
  const long long ctas = (rows + kRowWarps - 1) / kRowWarps;
  if (!backward) {
    const unsigned grid = (unsigned)(ctas < 148 * 64 ? ctas : 148 * 64);
    if (grid) norm_rotate_rows<T, false><<<grid, 32 * kRowWarps, 0, s>>>(p);
    return failed(cudaGetLastError());
  }
  const unsigned grid = (unsigned)(ctas < kPartials ? ctas : kPartials);
  if (grid) norm_rotate_rows<T, true><<<grid, 32 * kRowWarps, kRowWarps * 2 * p.width * sizeof(float), s>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? failed(e) : run_gain_sums(p, grid, s);
}

int dispatch(const tgcb_rotary_desc* d, bool backward, void* stream) {
  const Params p = params_of(d);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (d->dtype) {
    case TGCB_F32: return run<float>(p, backward, s);
    case TGCB_BF16: return run<__nv_bfloat16>(p, backward, s);
    default: return run<__half>(p, backward, s);
  }
}

}  // namespace

extern "C" {

int tgcb_norm_rotate(const tgcb_rotary_desc* d, void* stream) {
  const int rc = check(d, false, "tgcb_norm_rotate");
  if (rc != TGCB_OK) return rc;
  return dispatch(d, false, stream);
}

size_t tgcb_norm_rotate_scratch_bytes(int width) {
  return width < 1 || width > kMaxWidth ? 0 : (size_t)kPartials * 2 * width * sizeof(float);
}

int tgcb_norm_rotate_backward(const tgcb_rotary_desc* d, void* stream) {
  const int rc = check(d, true, "tgcb_norm_rotate_backward");
  if (rc != TGCB_OK) return rc;
  return dispatch(d, true, stream);
}

}  // extern "C"
