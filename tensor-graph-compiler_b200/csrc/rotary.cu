// RMS norm of query and key heads with the position rotation in the same pass, forward and backward.
//
// A head row x of `width` columns: r = 1 / sqrt(mean(x^2) + eps), y = x r g, and for the first
// `rotary` columns each pair (a, b) of y becomes (a cos t - b sin t, a sin t + b cos t) with
// t = position * frequency. The rotation is orthogonal, so the backward pass turns the output
// gradients by -t: d = rotate(dout, -t); dgain = sum over rows of d x r; with e = g d,
// dx = r (e - x r^2 mean(e x)).
#include <cuda_runtime.h>

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
  float epsilon;
};

// cos and sin of position * frequency. The turns are taken in float64 (a far position has many of them
// and float32 would lose the angle), reduced to a quarter turn and an eighth of a turn either way,
// so that rounding the rest to float32 costs 2^-25 of an eighth of a turn at most.
__device__ __forceinline__ void turn(double position, double frequency, float* c, float* s) {
  const double quarters = position * (frequency * 0.63661977236758134308);  // 2 / pi
  const double whole = rint(quarters);
  float sv, cv;
  sincospif(0.5f * (float)(quarters - whole), &sv, &cv);
  const int k = (int)((long long)whole & 3);
  const float a = (k & 1) ? sv : cv, b = (k & 1) ? cv : sv;
  *c = (k == 1 || k == 2) ? -a : a;
  *s = (k >= 2) ? -b : b;
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
    const float r = 1.f / sqrtf(warp_sum(square) / (float)p.width + p.epsilon);

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
            const float m = ex * r * r / (float)p.width;
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

// The gain gradients: column sums of the CTAs' partial rows, in float64 and in a fixed order.
__global__ void __launch_bounds__(256) gain_sums(const Params p, int partials) {
  __shared__ double part[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  double v = 0.0;
  if (c < 2 * p.width)
    for (int i = warp; i < partials; i += 8) v += (double)p.partials[(long long)i * 2 * p.width + c];
  part[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < 2 * p.width) {
#pragma unroll
    for (int w = 1; w < 8; ++w) v += part[w][lane];
    const int which = c >= p.width;
    store_any(p.side[which].gain_grad, p.gain_dtype, c - which * p.width, (float)v);
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
  if (!(d->epsilon > 0)) return bad("epsilon must be positive");
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
  return p;
}

template <typename T>
int run(const Params& p, bool backward, cudaStream_t s) {
  const long long rows = p.tokens * (p.side[0].heads + p.side[1].heads);
  const long long ctas = (rows + kRowWarps - 1) / kRowWarps;
  if (!backward) {
    const unsigned grid = (unsigned)(ctas < 148 * 64 ? ctas : 148 * 64);
    if (grid) norm_rotate_rows<T, false><<<grid, 32 * kRowWarps, 0, s>>>(p);
  } else {
    const unsigned grid = (unsigned)(ctas < kPartials ? ctas : kPartials);
    if (grid) norm_rotate_rows<T, true><<<grid, 32 * kRowWarps, kRowWarps * 2 * p.width * sizeof(float), s>>>(p);
    gain_sums<<<(2 * p.width + 31) / 32, 256, 0, s>>>(p, (int)grid);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, "norm_rotate", cudaGetErrorString(e));
  return TGCB_OK;
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
