// Attention of single tokens, prompt pieces and drafted trees over the int8 cache.
//
// For a token at position P of its sequence and query head h, reading key head h / group: s_j = scale (q . k_j),
// capped to cap tanh(s_j / cap) on request, over the positions j the token sees; out = sum_j e^(s_j - m) v_j
// / sum_j e^(s_j - m) with m the largest s_j, found in one pass by rescaling what has been added
// whenever a larger score arrives.
//
// A unit is one sequence, one key head and up to ROWS = 8 RN query rows (tokens x the heads that
// share the key head, token by token). Both products run on mma.sync with the cache as the left
// operand: S^T [16 keys x 8 rows] = K Q^T and O^T [16 columns x 8 rows] += V^T P^T. With the rows as the narrow
// side a single token's few query heads fill an 8-wide tile instead of a 16-wide one, and a
// warp's codes are converted once for all its rows. The codes are exact in bfloat16; what
// multiplies them is split into bfloat16 parts: the queries exactly (1 part from bfloat16, 2 from
// float16, 3 from float32), the weights p_j * value scale into 2 parts (16 bits) for 16-bit rows, below their
// own rounding, and 3 (24 bits) for float32 rows.
//
// What bounds it with few rows is reading the cache, 2 W + 8 bytes a position and head, and next to that
// the instructions for a key, of which the conversion of its codes is half (25 a key for bfloat16 rows, 32
// for float32 ones). Measured: 64 tokens of 32 heads on 8 over 1024 to 4096 positions of width 128 (347 MB) in
// 71 us, 4.9 TB/s; 2 float32 tokens over 131072 positions (554 MB) with a cap in 125 us, 4.4 TB/s. Each
// warp streams its own 32-key steps through a private ring in shared memory (cp.async), with no
// barrier between warps until a unit ends. The work is the list of all units' steps, cut into
// equal pieces, one per CTA, whatever the sequences' lengths are (they are known on the device alone):
// a unit that lies in one piece is finished there, one that is cut leaves its parts in scratch and
// `combine` joins them in order, so results do not depend on timing.
//
// Four row tiles at width 128 spill (296 to 420 bytes of stores a thread, bfloat16 to float32), as do two at width 256 (164
// to 244) and four at width 64 in bfloat16 and float32 (60 and 44). A row tile's steps end at its last row's position, but
// the pieces are cut as if all tiles of a sequence had the last one's.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "cached_attention.cuh"

namespace {

using namespace tgcb_attend;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 32;       // keys a warp takes at once; pages hold 16 or more, so a step touches at most two
// Three per SM, which fit at once with one row tile and widths up to 128 (with 888 the long float32 case took 160 instead of
// 142 us). Two fit with more row tiles and one at width 256, for registers and shared memory: there the equal pieces run in one
// and a half and in three rounds. Scratch is for this many.
constexpr int kMaxCtas = 444;
constexpr int kMinSteps = 8;    // steps a CTA takes at least: two per warp
constexpr int kWholeBelow = 512;  // positions up to which units are not cut, which saves the second launch

template <typename T>
struct Parts;
template <>
struct Parts<__nv_bfloat16> {
  static constexpr int Q = 1, P = 2;
};
template <>
struct Parts<__half> {
  static constexpr int Q = 2, P = 2;
};
template <>
struct Parts<float> {
  static constexpr int Q = 3, P = 3;
};

template <typename T, int W, int RN>
struct Shape {
  static constexpr int ROWS = 8 * RN;
  static constexpr int STAGE = kStep * (2 * W + 8);
  static constexpr int STAGES = 2;
  static constexpr int RING = kWarps * STAGES * STAGE;
  static constexpr int OP = W + 4;  // pitch of a warp's sums in floats when the warps are joined
  static constexpr int JOIN = kWarps * ROWS * (OP + 2) * 4;
  static constexpr int QUERIES = RN * Parts<T>::Q * (W / 16) * 32 * 8;
  static constexpr int BYTES = QUERIES + (RING > JOIN ? RING : JOIN);
};

// Where 16-byte piece `piece` of row `row` of a step lies in its row: permuted so that one piece of eight
// consecutive rows, which ldmatrix reads at once, lies on all banks.
template <int W>
__device__ __forceinline__ int piece_at(int row, int piece) {
  return piece ^ (W >= 128 ? row & 7 : W == 64 ? (row >> 1) & 3 : (row >> 2) & 1);
}

// One 16-byte piece of 32 rows of bytes, whose addresses the lanes give. Plain: word i is bytes
// 4 (lane % 4) .. + 3 of row 8 i + lane / 4. Transposed: bytes 2 (lane / 4) and + 1 of row 8 i + 2 (lane % 4), then
// the same two of the next row.
__device__ __forceinline__ void load_rows(unsigned address, unsigned* w) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void load_rows_transposed(unsigned address, unsigned* w) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(address)
               : "memory");
}

__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(unsigned dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}

__device__ __forceinline__ void mma(float* d, const unsigned* a, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned transposed(unsigned x) {
  unsigned r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

template <typename T, int W, int RN>
__global__ void __launch_bounds__(kThreads, RN == 1 && W <= 128 ? 3 : 2) attend(const Cache c, const Batch b, const Args a) {
  using S = Shape<T, W, RN>;
  constexpr int NQ = Parts<T>::Q, NP = Parts<T>::P, ROWS = S::ROWS, TILES = W / 16;
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ __align__(16) unsigned char memory[];
  __shared__ Begin begin;
  asm volatile("griddepcontrol.launch_dependents;");
  long long chunk;
  begin_at<ROWS, kStep, kWarps>(c, b, a, kMinSteps, &chunk, &begin);
  const long long total = begin.total;
  long long at = blockIdx.x * chunk;
  const long long stop = at + chunk < total ? at + chunk : total;
  if (!a.whole && threadIdx.x == 0) a.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (at >= stop) return;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, l4 = lane & 3;
  uint2* queries = reinterpret_cast<uint2*>(memory);
  unsigned char* ring = memory + S::QUERIES + warp * S::STAGES * S::STAGE;
  const unsigned ring_at = static_cast<unsigned>(__cvta_generic_to_shared(ring));
  const bool wide = out_wide<T>(a);
  // a score's factor beside its key's scale: for the hyperbolic tangent of the cap, or in units of log2 e
  const float factor = kCodeScale * (a.cap > 0 ? a.scale / a.cap : a.scale * kLog2e), cap2 = a.cap * kLog2e;
  unsigned mask, flip;
  asm volatile("mov.u32 %0, 0x00ff00ff;" : "=r"(mask));
  asm volatile("mov.u32 %0, 0x00800080;" : "=r"(flip));

  int s = begin.sequence;
  Sequence q = sequence_of<ROWS, kStep>(b, a, s);
  const int per_unit0 = a.whole ? 1 : q.steps;
  long long unit = begin.offset / per_unit0;
  int from = (int)(begin.offset - unit * per_unit0);

  while (at < stop) {
    while (unit >= (long long)c.heads * q.tiles) {  // on to the next sequence that has rows
      q = sequence_of<ROWS, kStep>(b, a, ++s);
      unit = 0;
    }
    const int head = (int)(unit / q.tiles), tile = (int)(unit - (long long)head * q.tiles);
    int to = q.steps;
    if (!a.whole) to = stop - at < to - from ? from + (int)(stop - at) : to;
    const int rows = min(ROWS, q.rows * a.group - tile * ROWS);

    count_outside(c, q, a, head == 0 && tile == 0 && from == 0 && threadIdx.x == 0);
    // The unit's queries as right-hand fragments: word pair (part, k, lane) holds row lane / 4's columns
    // 16 k + 4 (lane % 4) + {0, 2} and {1, 3}, as `codes` delivers the keys' columns.
    __syncthreads();
    for (int i = threadIdx.x; i < RN * TILES * 32; i += kThreads) {
      const int ln = i & 31, k = (i >> 5) % TILES, rn = (i >> 5) / TILES;
      const int r = rn * 8 + (ln >> 2);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < rows) {
        const int row = tile * ROWS + r, token = row / a.group, in_group = row - token * a.group;
        const T* p = reinterpret_cast<const T*>(a.q) + (q.first + token) * a.q_t + (long long)(head * a.group + in_group) * a.q_h +
                     16 * k + 4 * (ln & 3);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_float(p[j]);
      }
      unsigned even[NQ], odd[NQ];
      split<NQ>(v[0], v[2], even);
      split<NQ>(v[1], v[3], odd);
#pragma unroll
      for (int j = 0; j < NQ; ++j) queries[((rn * NQ + j) * TILES + k) * 32 + ln] = make_uint2(even[j], odd[j]);
    }
    __syncthreads();

    // What this lane's rows 2 l4 + {0, 1} of each row tile see: positions below `limit`, and with
    // `visible` those whose bit is set. Positions below `all` are seen by every row.
    int limit[RN][2];
    unsigned long long bits[RN][2];
    int all;
    {
      const int token0 = tile * ROWS / a.group;
      const long long seen = a.visible ? q.start : q.start + token0 + 1;
      all = (int)(seen < 0 ? 0 : seen > a.capacity ? a.capacity : seen);
#pragma unroll
      for (int rn = 0; rn < RN; ++rn)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = tile * ROWS + min(rn * 8 + 2 * l4 + j, rows - 1), token = row / a.group;
          const long long sees = a.visible ? q.start : q.start + token + 1;
          limit[rn][j] = (int)(sees < 0 ? 0 : sees > a.capacity ? a.capacity : sees);
          bits[rn][j] = a.visible ? (unsigned long long)__ldg(a.visible + q.first + token) : 0ull;
        }
    }
    const int in_tree = a.visible ? min(q.rows, 64) : 0;
    // a tile's rows need no step behind the last position that one of them sees
    int end = to;
    if (!a.visible) {
      const long long sees = q.start + (tile * ROWS + rows - 1) / a.group + 1;
      end = min(to, (int)(((sees < 0 ? 0 : sees > q.end ? q.end : sees) + kStep - 1) / kStep));
    }

    float m[RN][2], sum[RN][2], o[RN][TILES][4];
    unsigned seen_rows = 0;
#pragma unroll
    for (int rn = 0; rn < RN; ++rn) {
      m[rn][0] = m[rn][1] = -INFINITY, sum[rn][0] = sum[rn][1] = 0.f;
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[rn][t][0] = o[rn][t][1] = o[rn][t][2] = o[rn][t][3] = 0.f;
    }

    // pages of a step's two halves, -1: none of it is read
    auto pages_of = [&](int step) {
      int2 p = make_int2(-1, -1);
      if (step < end) {
        const int position = step * kStep;
        p.x = tgcb_kv::page_of(c, b, s, position);
        if (p.x < 0 && lane == 0 && position < q.end) atomicAdd(c.faults, 1);
        if (position + 16 < q.end) {
          p.y = c.page_bits >= 5 ? p.x : tgcb_kv::page_of(c, b, s, position + 16);
          if (p.y < 0 && lane == 0) atomicAdd(c.faults, 1);
        }
      }
      return p;
    };
    constexpr int CH = W / 16;                    // 16-byte pieces of a row
    constexpr int LANES = CH < 16 ? 32 / CH : 2;  // rows a warp copies at once; divides 16
    // the permutation goes by a row's last three bits, so copies 8 rows apart share their offsets
    constexpr int KINDS = LANES < 8 ? 8 / LANES : 1;
    unsigned copy_to[KINDS];
#pragma unroll
    for (int i = 0; i < KINDS; ++i) {
      const int r = i * LANES + lane / CH;
      copy_to[i] = ring_at + r * W + 16 * piece_at<W>(r, lane % CH);
    }
    const unsigned scale_to = ring_at + 2 * kStep * W + 4 * lane;
    const int lane_from = lane * 16;
    auto issue = [&](int step, int stage, int2 p) {
      if (step < end) {
        const int place = (step * kStep) & (c.page - 1);
        const long long row0 = ((long long)max(p.x, 0) * c.heads + head) * c.page + place;
        const long long row1 = ((long long)max(p.y, 0) * c.heads + head) * c.page + ((place + 16) & (c.page - 1));
        const unsigned at_stage = stage * S::STAGE;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const long long row = half ? row1 : row0;
          const bool valid = (half ? p.y : p.x) >= 0;
          const int8_t* k = c.keys + row * W + lane_from;
          const int8_t* v = c.values + row * W + lane_from;
#pragma unroll
          for (int r0 = 0; r0 < 16; r0 += LANES) {
            const int kind = r0 / LANES % KINDS, group = r0 / LANES / KINDS * KINDS * LANES + 16 * half;
            copy16(copy_to[kind] + at_stage + group * W, k + r0 * W, valid);
            copy16(copy_to[kind] + at_stage + (kStep + group) * W, v + r0 * W, valid);
          }
        }
        const long long row = lane < 16 ? row0 + lane : row1 + (lane - 16);
        const bool valid = (lane < 16 ? p.x : p.y) >= 0;
        copy4(scale_to + at_stage, c.key_scales + row, valid);
        copy4(scale_to + at_stage + 4 * kStep, c.value_scales + row, valid);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    int2 held[S::STAGES];
    const int first = from + warp;
#pragma unroll
    for (int i = 0; i < S::STAGES; ++i) {
      held[i] = pages_of(first + i * kWarps);
      issue(first + i * kWarps, i, held[i]);
    }
    int2 next = pages_of(first + S::STAGES * kWarps);
    int stage = 0;
    for (int step = first; step < end; step += kWarps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 1) : "memory");
      __syncwarp();
      const unsigned rows_at = ring_at + stage * S::STAGE + lane * W;  // of the keys; the values follow
      const float* key_scale = reinterpret_cast<const float*>(ring + stage * S::STAGE + 2 * kStep * W);
      const float* value_scale = key_scale + kStep;
      const int position = step * kStep;
      const bool inside = position + kStep <= all && held[0].x >= 0 && held[0].y >= 0;

      // scores: [half of the step][row tile]{key g row 2 l4, same row 2 l4 + 1, key g + 8 ..}
      float sc[2][RN][4], low[2][RN][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int rn = 0; rn < RN; ++rn)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[h][rn][j] = low[h][rn][j] = 0.f;
#pragma unroll
      for (int k = 0; k < TILES; ++k) {
        unsigned raw[4], ka[2][4];
        load_rows(rows_at + 16 * piece_at<W>(lane, k), raw);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ka[h][0] = codes(raw[2 * h], mask, flip), ka[h][1] = codes(raw[2 * h + 1], mask, flip);
          ka[h][2] = codes(raw[2 * h] >> 8, mask, flip), ka[h][3] = codes(raw[2 * h + 1] >> 8, mask, flip);
        }
#pragma unroll
        for (int rn = 0; rn < RN; ++rn)
#pragma unroll
          for (int part = 0; part < NQ; ++part) {
            const uint2 qb = queries[((rn * NQ + part) * TILES + k) * 32 + lane];
#pragma unroll
            for (int h = 0; h < 2; ++h) mma(part == 0 ? sc[h][rn] : low[h][rn], ka[h], qb.x, qb.y);
          }
      }

      // scores in units of log2 e
      float vs[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float ks = key_scale[16 * h + 8 * k + g] * factor;
          vs[h][k] = value_scale[16 * h + 8 * k + g] * kCodeScale;
#pragma unroll
          for (int rn = 0; rn < RN; ++rn)
#pragma unroll
            for (int j = 2 * k; j < 2 * k + 2; ++j) {
              if (NQ > 1) sc[h][rn][j] += low[h][rn][j];
              sc[h][rn][j] *= ks;
            }
        }
      if (a.cap > 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int rn = 0; rn < RN; ++rn)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[h][rn][j] = cap2 * tanh_of<T>(sc[h][rn][j]);
      }
      unsigned hidden = 0;  // bit (h RN + rn) 4 + j: a score that its row does not see
      if (!inside) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int key = position + 16 * h + 8 * k + g;
            const bool there = (h ? held[0].y : held[0].x) >= 0;
            const int since = (int)min((long long)key - q.start, 1ll << 30);
            const bool in_call = since >= 0 && since < in_tree;
#pragma unroll
            for (int rn = 0; rn < RN; ++rn)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const bool sees = key < limit[rn][j] || (in_call && ((bits[rn][j] >> since) & 1));
                if (sees && there) {
                  seen_rows |= 1u << (rn * 2 + j);
                } else {
                  sc[h][rn][2 * k + j] = -INFINITY;
                  hidden |= 1u << ((h * RN + rn) * 4 + 2 * k + j);
                }
              }
          }
      } else {
        seen_rows = ~0u;
      }
      float keep[RN][2], base[RN][2], top[RN][2];
      bool moved = false;
#pragma unroll
      for (int rn = 0; rn < RN; ++rn)
#pragma unroll
        for (int j = 0; j < 2; ++j) top[rn][j] = fmaxf(fmaxf(sc[0][rn][j], sc[0][rn][2 + j]), fmaxf(sc[1][rn][j], sc[1][rn][2 + j]));
      const float largest = fmaxf(fmaxf(fabsf(vs[0][0]), fabsf(vs[0][1])), fmaxf(fabsf(vs[1][0]), fabsf(vs[1][1])));
      if (__any_sync(0xffffffffu, largest > kLargeScale * kCodeScale)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (fabsf(vs[h][k]) > kLargeScale * kCodeScale) {
#pragma unroll
              for (int rn = 0; rn < RN; ++rn)
#pragma unroll
                for (int j = 0; j < 2; ++j) top[rn][j] = fmaxf(top[rn][j], sc[h][rn][2 * k + j] + kLargeMargin);
            }
      }
#pragma unroll
      for (int rn = 0; rn < RN; ++rn)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float t = top[rn][j];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
          const float mn = fmaxf(m[rn][j], t);
          keep[rn][j] = mn == m[rn][j] ? 1.f : exp2_fast(m[rn][j] - mn);
          moved |= mn != m[rn][j];
          m[rn][j] = mn;
          base[rn][j] = mn == -INFINITY ? 0.f : mn;
          sum[rn][j] *= keep[rn][j];
        }
      // float32 rows: each step's products in accumulators of their own, added in float32. The tensor cores cut off
      // what does not fit their sums, which over thousands of steps would all err to the same side.
      constexpr bool FRESH = NP == 3;
      if (!FRESH && __any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int rn = 0; rn < RN; ++rn)
#pragma unroll
          for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[rn][t][j] *= keep[rn][j & 1];
      }

      // weights, and the products with the values
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int rn = 0; rn < RN; ++rn)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = exp2_fast(sc[h][rn][j] - base[rn][j & 1]);
            sum[rn][j & 1] += p;
            sc[h][rn][j] = p * vs[h][j >> 1];
          }
      if (hidden) {  // whatever lies there
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int rn = 0; rn < RN; ++rn)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if ((hidden >> ((h * RN + rn) * 4 + j)) & 1) sc[h][rn][j] = 0.f;
      }
      unsigned pb[2][RN][NP][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int rn = 0; rn < RN; ++rn) {
          unsigned lo[NP], hi[NP];
          split<NP>(sc[h][rn][0], sc[h][rn][1], lo);
          split<NP>(sc[h][rn][2], sc[h][rn][3], hi);
#pragma unroll
          for (int part = 0; part < NP; ++part) {
            pb[h][rn][part][0] = transposed(lo[part]);
            pb[h][rn][part][1] = transposed(hi[part]);
          }
        }
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        unsigned raw[4];
        float fresh[RN][4];
#pragma unroll
        for (int rn = 0; rn < RN; ++rn) fresh[rn][0] = fresh[rn][1] = fresh[rn][2] = fresh[rn][3] = 0.f;
        load_rows_transposed(rows_at + kStep * W + 16 * piece_at<W>(lane, t), raw);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          unsigned va[4];  // tile rows lane / 4 and + 8: columns 16 t + 2 (lane / 4) and the next
          va[0] = codes(raw[2 * h], mask, flip), va[1] = codes(raw[2 * h] >> 8, mask, flip);
          va[2] = codes(raw[2 * h + 1], mask, flip), va[3] = codes(raw[2 * h + 1] >> 8, mask, flip);
#pragma unroll
          for (int rn = 0; rn < RN; ++rn)
#pragma unroll
            for (int part = 0; part < NP; ++part)
              mma(FRESH ? fresh[rn] : o[rn][t], va, pb[h][rn][part][0], pb[h][rn][part][1]);
        }
        if (FRESH) {
#pragma unroll
          for (int rn = 0; rn < RN; ++rn)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[rn][t][j] = fmaf(o[rn][t][j], keep[rn][j & 1], fresh[rn][j]);
        }
      }
      __syncwarp();
      issue(step + S::STAGES * kWarps, stage, next);
#pragma unroll
      for (int i = 0; i + 1 < S::STAGES; ++i) held[i] = held[i + 1];
      held[S::STAGES - 1] = next;
      next = pages_of(step + (S::STAGES + 1) * kWarps);
      stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // join the warps: maxima and sums, then the weighted sums of each row
#pragma unroll
    for (int rn = 0; rn < RN; ++rn)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum[rn][j] += __shfl_xor_sync(0xffffffffu, sum[rn][j], x);
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) seen_rows |= __shfl_xor_sync(0xffffffffu, seen_rows, x);
    __syncthreads();  // the rings are free
    float* joined = reinterpret_cast<float*>(memory + S::QUERIES);
    float* own = joined + warp * ROWS * (S::OP + 2);
#pragma unroll
    for (int rn = 0; rn < RN; ++rn)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = rn * 8 + 2 * l4 + j;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
          *reinterpret_cast<float2*>(own + r * S::OP + 16 * t + 2 * g) = make_float2(o[rn][t][j], o[rn][t][2 + j]);
        if (g == 0) {
          // a row that saw nothing has sum 0, one that saw scores of -infinity alone is marked with -1
          const bool lowest = ((seen_rows >> (rn * 2 + j)) & 1) && m[rn][j] == -INFINITY;
          own[ROWS * S::OP + 2 * r] = m[rn][j];
          own[ROWS * S::OP + 2 * r + 1] = lowest ? -1.f : sum[rn][j];
        }
      }
    __syncthreads();
    const bool complete = from == 0 && to == q.steps;
    // a piece that began in an earlier CTA goes to slot 0 of this CTA, one that ends in a later to slot 1
    float* part = complete ? nullptr : a.parts + (2ll * blockIdx.x + (from == 0)) * ROWS * (W + 2);
    constexpr int QUADS = W / 4;
    for (int i = threadIdx.x; i < rows * QUADS; i += kThreads) {
      const int r = i / QUADS, quad = i - r * QUADS;
      const float* ml = joined + ROWS * S::OP + 2 * r;
      float mm = -INFINITY, f[kWarps];
      Weights all;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ml[w * ROWS * (S::OP + 2)]);
      const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        f[w] = exp2_fast(ml[w * ROWS * (S::OP + 2)] - base);
        all.add(ml[w * ROWS * (S::OP + 2) + 1], f[w]);
      }
      const float all_sum = all.sum();
      const int col = 4 * quad;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(joined + w * ROWS * (S::OP + 2) + r * S::OP + col);
        v[0] = fmaf(x.x, f[w], v[0]), v[1] = fmaf(x.y, f[w], v[1]), v[2] = fmaf(x.z, f[w], v[2]), v[3] = fmaf(x.w, f[w], v[3]);
      }
      if (complete) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = answer(v[j], all_sum);
        store4<T>(out_row<T>(a, q, head, tile * ROWS + r) + col, v, wide);
      } else {
        *reinterpret_cast<float4*>(part + r * W + col) = make_float4(v[0], v[1], v[2], v[3]);
        if (quad == 0) *reinterpret_cast<float2*>(part + ROWS * W + 2 * r) = make_float2(mm, all_sum);
      }
    }
    if (!complete && from == 0 && threadIdx.x == 0) {
      const long long last = (at + q.steps - 1) / chunk;
      a.cuts[blockIdx.x] = make_int4(s, head, tile, (int)last);
    }
    at += a.whole ? 1 : to - from;
    ++unit;
    from = 0;
  }
}

// Row tiles of 8 a unit takes: as many as the call's sequences have rows on average, since a unit
// reads and converts its keys once for all its rows.
int row_tiles(const Batch& b, int group, int width) {
  const long long rows = (b.tokens + b.batch - 1) / b.batch * group;
  if (rows <= 8) return 1;
  if (rows <= 16 || width > 128) return 2;
  return 4;
}

// Calls in 16 bits and widths 64 and 128 take the tcgen05 kernel, with units of 128 rows, where sequences have more than
// 32 query rows a key head on average and the call may have four tiles of 128 keys for every SM. Measured there and
// here: 2 x 509 tokens behind 4000 positions 132 and 367 us, 32 trees of 1 to 31 nodes over 2000 to 8000 positions 273
// and 515 us; one tree of 13 nodes over 2047 positions, too little to fill the longer pipeline, 50 and 42 us (each
// from a cold L2, a single call). Below 52 rows the two were not compared. Lengths are on the device, so the
// choice goes by the call's average: 512 tokens beside 200 single ones (32 heads on 8 of 128, over 2000 positions) take
// 456 us, and 89 + 151 us in two calls.
bool for_tensor(const Cache& c, const Batch& b, int group) {
  if ((c.width != 64 && c.width != 128) || (b.tokens + b.batch - 1) / b.batch * group <= 32) return false;
  if ((long long)c.pages * c.heads * c.page > 0x7fffffffll) return false;  // it numbers rows in 32 bits
  const long long units = (b.tokens * group + kTensorRows - 1) / kTensorRows * c.heads;
  return units * ((long long)b.max_pages * c.page / 128) >= 4 * kTensorCtas;
}

size_t cuts_bytes() { return kMaxCtas * sizeof(int4); }

size_t scratch_bytes(const Cache& c, const Batch& b, int q_heads) {
  if (b.tokens == 0 || (long long)b.max_pages * c.page <= kWholeBelow) return 0;
  size_t rows = 2ull * kMaxCtas * 8 * row_tiles(b, q_heads / c.heads, c.width);
  if (for_tensor(c, b, q_heads / c.heads)) rows = std::max<size_t>(rows, 2ull * kTensorCtas * kTensorRows);
  return cuts_bytes() + rows * (c.width + 2) * sizeof(float);
}

template <typename T, int W, int RN>
int launch(const Cache& c, const Batch& b, const Args& a, cudaStream_t s) {
  using S = Shape<T, W, RN>;
  const char* what = "tgcb_cached_attention";
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, what, cudaGetErrorString(e));
  static std::atomic<unsigned long long> configured{0};
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    e = cudaFuncSetAttribute(attend<T, W, RN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES);
    if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, what, cudaGetErrorString(e));
    configured.fetch_or(bit);
  }
  // no more CTAs than there can be pieces of work
  const long long tiles = (b.tokens * a.group + S::ROWS - 1) / S::ROWS + b.batch;
  const long long steps = a.whole ? 1 : (a.capacity + kStep - 1) / kStep;
  const long long pieces = (tiles * c.heads * steps + (a.whole ? 0 : kMinSteps - 1)) / (a.whole ? 1 : kMinSteps);
  const unsigned grid = (unsigned)(pieces < kMaxCtas ? pieces : kMaxCtas);
  attend<T, W, RN><<<grid, kThreads, S::BYTES, s>>>(c, b, a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, what, cudaGetErrorString(e));
  if (a.whole) return TGCB_OK;
  e = launch_combine<T, W, RN>(c, b, a, grid, s);
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, what, cudaGetErrorString(e));
  return TGCB_OK;
}

template <typename T, int W>
int by_rows(const Cache& c, const Batch& b, const Args& a, cudaStream_t s) {
  switch (row_tiles(b, a.group, W)) {
    case 1: return launch<T, W, 1>(c, b, a, s);
    case 2: return launch<T, W, 2>(c, b, a, s);
    default:
      if constexpr (W <= 128) return launch<T, W, 4>(c, b, a, s);
      return launch<T, W, 2>(c, b, a, s);
  }
}

template <typename T>
int run(const Cache& c, const Batch& b, const Args& a, cudaStream_t s) {
  switch (c.width) {
    case 32: return by_rows<T, 32>(c, b, a, s);
    case 64: return by_rows<T, 64>(c, b, a, s);
    case 128: return by_rows<T, 128>(c, b, a, s);
    default: return by_rows<T, 256>(c, b, a, s);
  }
}

}  // namespace

extern "C" {

size_t tgcb_cached_attention_scratch_bytes(const tgcb_cache* cache, const tgcb_batch* batch, int q_heads) {
  Cache c;
  Batch b;
  if (tgcb_kv::checked(cache, batch, TGCB_F32, &c, &b, "tgcb_cached_attention_scratch_bytes") != TGCB_OK) return 0;
  return q_heads < 1 || q_heads % c.heads ? 0 : scratch_bytes(c, b, q_heads);
}

int tgcb_cached_attention(const tgcb_cache* cache, const tgcb_batch* batch, int dtype, int q_heads,
                          const tgcb_heads* queries, const int64_t* visible, float scale, float cap,
                          const tgcb_heads* out, void* scratch, size_t scratch_size, void* stream) {
  const char* what = "tgcb_cached_attention";
  Cache c;
  Batch b;
  const int rc = tgcb_kv::checked(cache, batch, dtype, &c, &b, what);
  if (rc != TGCB_OK) return rc;
  auto bad = [&](const char* why) { return tgcb_internal_fail(TGCB_E_INVALID, what, why); };
  if (queries == nullptr || out == nullptr || (b.tokens > 0 && (queries->data == nullptr || out->data == nullptr)))
    return bad("null pointer");
  if (q_heads < 1 || q_heads % c.heads) return bad("the query heads must be a multiple of the cache's heads");
  if (b.tokens * q_heads > 0x7fffffffll) return bad("too many tokens");
  if (!std::isfinite(scale)) return bad("the scale must be finite");
  if (!(cap >= 0) || std::isinf(cap)) return bad("the cap must be finite and not negative");
  // the largest factors that the kernels form of them, with room for their constants; a score over a cap of at most 1e30
  // that is no normal float32 is off by less than 2^-20 of a unit as long as q . code is below 2^30
  if (cap > 1.1e30f) return bad("a cap is at most 1e30: 0 for none");
  if (std::fabs(scale) > 1.1e30f || (cap > 0 && !(std::fabs(scale / cap) <= 1.1e30f))) return bad("the scale under the cap is beyond float32");
  if (b.tokens == 0) return TGCB_OK;
  const size_t need = scratch_bytes(c, b, q_heads);
  if (need && (scratch == nullptr || scratch_size < need || (reinterpret_cast<uintptr_t>(scratch) & 15u)))
    return bad("scratch must be 16-byte aligned and hold tgcb_cached_attention_scratch_bytes");
  Args a = {};
  a.q = static_cast<const char*>(queries->data), a.q_t = queries->token_stride, a.q_h = queries->head_stride;
  a.out = static_cast<char*>(out->data), a.out_t = out->token_stride, a.out_h = out->head_stride;
  a.visible = reinterpret_cast<const long long*>(visible);
  a.cuts = static_cast<int4*>(scratch);
  a.parts = need ? reinterpret_cast<float*>(static_cast<char*>(scratch) + cuts_bytes()) : nullptr;
  a.group = q_heads / c.heads, a.scale = scale, a.cap = cap;
  a.capacity = b.max_pages * c.page, a.whole = need == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype != TGCB_F32 && for_tensor(c, b, a.group)) return attend_tensor(c, b, a, dtype, s);
  switch (dtype) {
    case TGCB_F32: return run<float>(c, b, a, s);
    case TGCB_BF16: return run<__nv_bfloat16>(c, b, a, s);
    default: return run<__half>(c, b, a, s);
  }
}

}  // extern "C"
