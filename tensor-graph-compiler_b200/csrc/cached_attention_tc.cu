// Attention over the int8 cache for many query rows at once (prompt pieces, larger trees) on tcgen05.
//
// A unit is one sequence, one key head and up to 128 query rows (tokens x the heads that share the
// key head). One CTA an SM; its keys come in tiles of 128, even tiles to group 0 and odd ones to
// group 1, two halves of the CTA that each keep their own maxima, sums and accumulator for the
// same rows and are joined at the unit's end. While one group is in its softmax, the other's products run.
//
//   converters (4 warps for the keys, 4 for the values): codes from the cache to 16-bit matrices in shared memory
//     (128-byte swizzle; the next tile's codes are in registers by then); the first also bring the scales, the
//     others a unit's queries.
//   products (1 thread): S = Q K^T into the group's 128 columns of tensor memory; O += P V with P read from tensor
//     memory and V as it lies (columns contiguous).
//   softmax (2 x 4 warps, a thread per row): the row's maximum, then weights e^(s - m) times the value's
//     scale as two bfloat16 parts (16 bits, as in the kernel for few rows), written over the scores
//     they came from: 16 scores' columns hold 8 columns of leading and 8 of remaining parts.
//     The accumulator is rescaled only when a maximum grows by more than 2^8, since the weights' sum
//     and the products share whatever reference they were taken against.
//
// Bound by its 20 warps of three codes, which issue 0.53 instructions a cycle and scheduler and wait for one another,
// tensor memory and instruction fetch (4.1 to 4.3 us for 128 rows x 128 keys at width 128, of which the products, the
// second in two parts, take 1.1), with 320 to 454 bytes of spill stores and 548 to 580 of spill loads a thread under the
// launch's 96 registers. Loops are kept short for that reason. Every tile of codes is converted for 128 rows alone, both
// groups having the same ones, and a sequence's tiles of rows count alike in the division of the work although early rows
// see fewer keys: one prompt of 8192 tokens behind nothing, 32 heads on 8, takes 2477 us (222 TFLOP/s; its busiest CTA has
// 1.9 times the average's tiles). Measured: 2 x 509 tokens of 16 heads on 4 behind 4000 positions 122 us, 290 TFLOP/s; 32
// trees of 1 to 31 nodes, 32 heads on 8, over 2000 to 8000 positions 242 to 270 us (calls in a row).
// All waits are bounded (4 s); a CTA that gives up records status 6 and unwinds.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "cached_attention.cuh"

namespace {

using namespace tgcb_attend;

constexpr int kKeys = 128;
constexpr int kGroupThreads = 128;
constexpr int kKeyThreads = 2 * kGroupThreads;           // first thread of the keys' converters
constexpr int kValueThreads = kKeyThreads + 128;         // of the values'
constexpr int kProducts = kValueThreads + 128;           // of the four warps of which one thread issues products
constexpr int kTensorThreads = kProducts + 128;
// Registers a thread: the launch gives 96 to each of the five groups of 128, 480 in all, which the
// roles share out between them.
constexpr int kSoftmaxRegisters = 136, kConverterRegisters = 80, kProductRegisters = 48, kLaunchRegisters = 96;
static_assert(2 * kSoftmaxRegisters + 2 * kConverterRegisters + kProductRegisters <= 5 * kLaunchRegisters, "the launch has no more registers");
static_assert(kSoftmaxRegisters >= kLaunchRegisters && kConverterRegisters <= kLaunchRegisters && kProductRegisters <= kLaunchRegisters,
              "more_registers only goes up, fewer_registers only down");
constexpr int kLeastTiles = 2;                           // one for each group
constexpr int kStatusTimeout = 6;                        // device status code (the kernels' TGCB_STATUS_* family)
constexpr float kGrowth = 8.f;                           // of a maximum, in powers of two, before anything is rescaled

template <int W>
struct Memory {
  static constexpr int TILE = kKeys * W * 2;
  static constexpr int QUERIES = 0;
  static constexpr int STAGES = kTensorRows * W * 2;     // group g: keys, then values
  static constexpr int KEY_SCALES = STAGES + 4 * TILE;   // float [group][turn][128]
  static constexpr int VALUE_SCALES = KEY_SCALES + 4 * kKeys * 4;
  static constexpr int EXCHANGE = VALUE_SCALES + 4 * kKeys * 4;  // float [128][33]
  static constexpr int ROWS = EXCHANGE + 128 * 33 * 4;   // float2 [parity][group][128]: maximum and sum
  static constexpr int BYTES = ROWS + 4 * 128 * 8 + 1024;  // and room to begin on a 1024-byte boundary
};

struct Shared {
  unsigned long long q_full, q_free, k_full[2], scaled[2][2], v_full[2], s_full[2], p_ready[2], pv_done[2], rows_full, x_full, x_free, drained;
  unsigned tmem, valid[2][2];  // of 32 keys of a tile a byte: a bit for each 16 whose page is there, and bit 2 where `large` has a bit
  unsigned large[2][2][4];     // a bit for each key of a tile whose value's scale is above kLargeScale
  int abort;
};

__device__ __forceinline__ unsigned at(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(at(bar)) : "memory");
}

// Waits for a barrier's phase; false when the CTA gives up.
__device__ __forceinline__ bool wait(unsigned long long* bar, unsigned parity, Shared* sh, int* status) {
  unsigned long long start = 0;
  for (unsigned it = 0;; ++it) {
    unsigned ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(at(bar)), "r"(parity)
                 : "memory");
    if (ok) return true;
    if ((it & 255u) == 255u) {
      if (*reinterpret_cast<volatile int*>(&sh->abort)) return false;
      unsigned long long now;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
      if (start == 0) {
        start = now;
      } else if (now - start > 4000000000ull) {
        *reinterpret_cast<volatile int*>(&sh->abort) = 1;
        atomicCAS(status, 0, kStatusTimeout);
        return false;
      }
    }
  }
}

// The same for a whole warp, of which one thread polls.
__device__ __forceinline__ bool wait_warp(unsigned long long* bar, unsigned parity, Shared* sh, int* status) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = wait(bar, parity, sh, status);
  ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
  __syncwarp();
  return ok;
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void commit(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(at(bar)) : "memory");
}

#define TGCB_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define TGCB_S8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])

// 32 columns of a warp's 32 rows of tensor memory, a row a thread.
__device__ __forceinline__ void load32(unsigned tmem, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32]; tcgen05.wait::ld.sync.aligned;"
      : TGCB_R8(r, 0), TGCB_R8(r, 8), TGCB_R8(r, 16), TGCB_R8(r, 24)
      : "r"(tmem)
      : "memory");
}
__device__ __forceinline__ void load16(unsigned tmem, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16]; tcgen05.wait::ld.sync.aligned;"
      : TGCB_R8(r, 0), TGCB_R8(r, 8)
      : "r"(tmem)
      : "memory");
}
__device__ __forceinline__ void store16(unsigned tmem, const unsigned* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(tmem),
               TGCB_S8(r, 0), TGCB_S8(r, 8)
               : "memory");
}
__device__ __forceinline__ void store32(unsigned tmem, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(tmem),
      TGCB_S8(r, 0), TGCB_S8(r, 8), TGCB_S8(r, 16), TGCB_S8(r, 24)
      : "memory");
}
__device__ __forceinline__ void stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A matrix in shared memory with the 128-byte swizzle: rows of 128 bytes, eight to an atom. The lower half of its
// description, to which steps in 16-byte units are added; `lbo`: from one 128-byte column block to the next where
// the columns are not the summed dimension. The upper half is the same for all.
__device__ __forceinline__ unsigned matrix(unsigned start, unsigned lbo) { return ((start >> 4) & 0x3fffu) | (lbo >> 4) << 16; }
constexpr unsigned kMatrixHigh = 64u | 1u << 14 | 2u << 29;

__device__ __forceinline__ void product_ss(unsigned d, unsigned a, unsigned b, unsigned how, bool add) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 a, b; setp.ne.b32 p, %4, 0; mov.b64 a, {%1, %6}; mov.b64 b, {%2, %6};"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, {%5, %5, %5, %5}, p; }" ::"r"(d),
      "r"(a), "r"(b), "r"(how), "r"((unsigned)add), "r"(0u), "r"(kMatrixHigh)
      : "memory");
}
__device__ __forceinline__ void product_ts(unsigned d, unsigned a, unsigned b, unsigned how, bool add) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 b; setp.ne.b32 p, %4, 0; mov.b64 b, {%2, %6};"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, {%5, %5, %5, %5}, p; }" ::"r"(d),
      "r"(a), "r"(b), "r"(how), "r"((unsigned)add), "r"(0u), "r"(kMatrixHigh)
      : "memory");
}

// Two codes as float16, bytes 0 and 2 of a word: with the sign bit flipped they are x + 128, the low bits of 1024 + x
// + 128.
__device__ __forceinline__ unsigned half_codes(unsigned w, unsigned mask, unsigned magic) {
  unsigned u, r;
  asm("lop3.b32 %0, %1, %2, %3, 0x78;" : "=r"(u) : "r"(magic), "r"(w), "r"(mask));  // magic ^ (w & mask)
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x64806480u));
  return r;
}

// 16 bytes of codes, loaded where it stands: a plain load of constant memory may be moved down to its use, which is a
// tile later.
__device__ __forceinline__ void load_now(uint4* to, const int8_t* from) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(to->x), "=r"(to->y), "=r"(to->z), "=r"(to->w) : "l"(from));
}

// The pieces of this CTA's share of the work, as every role walks through them.
struct Walk {
  const Cache& c;
  const Batch& b;
  const Args& a;
  long long place, stop, chunk, unit;
  Sequence q;
  int s, from;
  int head, tile, to, rows, tiles, all;  // of the present piece: `tiles` of 128 keys from `from`; positions below `all` are seen by all rows

  __device__ __forceinline__ Walk(const Cache& c, const Batch& b, const Args& a, const Begin& begin, long long chunk)
      : c(c), b(b), a(a), chunk(chunk) {
    place = blockIdx.x * chunk;
    stop = min(place + chunk, begin.total);
    s = begin.sequence;
    q = sequence_of<kTensorRows, kKeys>(b, a, s);
    const int per = a.whole ? 1 : q.steps;
    unit = begin.offset / per;
    from = (int)(begin.offset - unit * per);
  }
  __device__ __forceinline__ bool next() {
    if (place >= stop) return false;
    while (unit >= (long long)c.heads * q.tiles) {
      q = sequence_of<kTensorRows, kKeys>(b, a, ++s);
      unit = 0;
    }
    head = (int)(unit / q.tiles), tile = (int)(unit - (long long)head * q.tiles);
    to = q.steps;
    if (!a.whole) to = stop - place < to - from ? from + (int)(stop - place) : to;
    rows = min(kTensorRows, q.rows * a.group - tile * kTensorRows);
    const int first = tile * kTensorRows / a.group, last = (tile * kTensorRows + rows - 1) / a.group;
    auto clip = [&](long long v, int most) { return (int)(v < 0 ? 0 : v > most ? most : v); };
    all = clip(a.visible ? q.start : q.start + first + 1, a.capacity);
    const int end = a.visible ? to : min(to, (clip(q.start + last + 1, q.end) + kKeys - 1) / kKeys);
    tiles = max(0, end - from);
    return true;
  }
  __device__ __forceinline__ void advance() {
    place += a.whole ? 1 : to - from;
    ++unit;
    from = 0;
  }
};

template <typename T, int W>
__device__ __forceinline__ void convert(const Cache& c, const Batch& b, const Args& a, Walk walk, Shared* sh, unsigned char* memory, int* status,
                                        bool VALUES) {
  using M = Memory<W>;
  // 16-code pieces of a row; rows a pass copies. Eight neighbouring threads have four pieces of two rows, whose halves lie on
  // different banks.
  constexpr int CH = W / 16, PASSES = CH, PER = 128 / CH;
  const bool HALF = !VALUES && !std::is_same_v<T, __nv_bfloat16>;  // the values meet bfloat16 weights
  const int tid = threadIdx.x - (VALUES ? kValueThreads : kKeyThreads), piece = tid % 4 + (W == 128 ? tid / 64 * 4 : 0), in_pass = W == 128 ? tid % 64 / 4 : tid / 4;
  const float factor = (HALF ? 1.f : kCodeScale) * (a.cap > 0 ? a.scale / a.cap : a.scale * 1.4426950408889634f);
  unsigned mask, flip, magic;
  asm volatile("mov.u32 %0, 0x00ff00ff;" : "=r"(mask));
  asm volatile("mov.u32 %0, 0x00800080;" : "=r"(flip));
  asm volatile("mov.u32 %0, 0x64806480;" : "=r"(magic));
  const bool wide_q = ((reinterpret_cast<uintptr_t>(a.q) | (unsigned long long)(a.q_t * 2) | (unsigned long long)(a.q_h * 2)) & 15u) == 0;
  unsigned turns[2] = {0, 0}, units = 0;

  while (walk.next()) {
    if (walk.tiles > 0) {
      const Sequence& q = walk.q;
      const int head = walk.head;
      // A tile's pages, a lane for each 16 keys (one page holds them), and, once they are there, the rows of the first of
      // those keys: -1 where they are not there or not read. There are fewer than 2^31 rows.
      constexpr int kUnread = -2;
      auto pages_of = [&](int tile) {
        const int lane = tid & 31, position = (walk.from + tile) * kKeys + 16 * lane;
        if (lane >= kKeys / 16 || tile >= walk.tiles || position >= q.end) return kUnread;
        return max(__ldg(b.table + walk.s * b.table_stride + (position >> c.page_bits)), -1);  // no entry is kUnread
      };
      auto rows_of = [&](int tile, int page) {
        const bool there = page >= 0 && page < c.pages;
        if (!VALUES && !there && page != kUnread && tid < 32) atomicAdd(c.faults, 1);
        return there ? (page * c.heads + head) * c.page + (((walk.from + tile) * kKeys + 16 * (tid & 31)) & (c.page - 1)) : -1;
      };
      const int8_t* from = VALUES ? c.values : c.keys;
      auto load = [&](int rows, uint4* raw) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int row = __shfl_sync(0xffffffffu, rows, W == 128 ? i : 2 * i + tid / 64);
          raw[i] = make_uint4(0, 0, 0, 0);
          if (row >= 0) load_now(raw + i, from + (long long)(row + in_pass % 16) * W + 16 * piece);
        }
      };
      auto scales_of = [&](int rows, float* ks, float* vs) {  // of key tid; whether its page is there
        const int row = __shfl_sync(0xffffffffu, rows, tid / 16);
        *ks = row < 0 ? 0.f : c.key_scales[row + tid % 16], *vs = row < 0 ? 0.f : c.value_scales[row + tid % 16];
        return row >= 0;
      };
      auto store = [&](unsigned char* to, const uint4* raw) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int key = i * PER + in_pass;
          const unsigned w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          uint4 out[2];
          unsigned* o = reinterpret_cast<unsigned*>(out);
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // columns 4 j + {0, 2} and {1, 3}
            o[2 * j] = HALF ? half_codes(w[j], mask, magic) : codes(w[j], mask, flip);
            o[2 * j + 1] = HALF ? half_codes(w[j] >> 8, mask, magic) : codes(w[j] >> 8, mask, flip);
          }
          unsigned char* row = to + (piece / 4) * (kKeys * 128) + key * 128;
          *reinterpret_cast<uint4*>(row + 16 * ((2 * (piece % 4)) ^ (key & 7))) = out[0];
          *reinterpret_cast<uint4*>(row + 16 * ((2 * (piece % 4) + 1) ^ (key & 7))) = out[1];
        }
      };
      uint4 raw[PASSES];
      float ks = 0.f, vs = 0.f;
      bool held = false;
      {
        const int rows = rows_of(0, pages_of(0));
        if (!VALUES) held = scales_of(rows, &ks, &vs);
        load(rows, raw);
      }
      int pages = pages_of(1);

      if (VALUES) {
      // the unit's queries, their columns in the order in which `codes` leaves the keys'
      if (units && !wait_warp(&sh->q_free, (units - 1) & 1, sh, status)) return;
      constexpr int EIGHTS = W / 8, ROUNDS = kTensorRows * EIGHTS / 128, SOME = 8;  // 8-column pieces of a row; SOME in flight
#pragma unroll 1
      for (int i0 = 0; i0 < ROUNDS; i0 += SOME) {
        uint4 v[SOME];
#pragma unroll
        for (int i = 0; i < SOME; ++i) {
          const int r = ((i0 + i) * 128 + tid) / EIGHTS, eight = tid % EIGHTS;
          v[i] = make_uint4(0, 0, 0, 0);
          if (r < walk.rows) {
            const int row = walk.tile * kTensorRows + r, token = row / a.group, in_group = row - token * a.group;
            const T* p = reinterpret_cast<const T*>(a.q) + (q.first + token) * a.q_t + (long long)(head * a.group + in_group) * a.q_h + 8 * eight;
            if (wide_q) {
              v[i] = *reinterpret_cast<const uint4*>(p);
            } else {
              const unsigned short* e = reinterpret_cast<const unsigned short*>(p);
              v[i] = make_uint4(e[0] | (unsigned)e[1] << 16, e[2] | (unsigned)e[3] << 16, e[4] | (unsigned)e[5] << 16, e[6] | (unsigned)e[7] << 16);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < SOME; ++i) {
          const int r = ((i0 + i) * 128 + tid) / EIGHTS, eight = tid % EIGHTS;
          const uint4 x = v[i];  // each four columns as (0, 2), (1, 3)
          *reinterpret_cast<uint4*>(memory + M::QUERIES + (eight / 8) * (kTensorRows * 128) + r * 128 + 16 * ((eight % 8) ^ (r & 7))) =
              make_uint4(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.x, x.y, 0x7632), __byte_perm(x.z, x.w, 0x5410), __byte_perm(x.z, x.w, 0x7632));
        }
      }
      fence_async();
      arrive(&sh->q_full);
      ++units;
      }

      for (int t = 0; t < walk.tiles; ++t) {
        const int g = t & 1;
        const unsigned turn = turns[g]++;
        unsigned char* stage = memory + M::STAGES + (2 * g + VALUES) * M::TILE;
        // the group's last scores (outputs) are there: their keys (values) are used up
        if (turn && !wait_warp(VALUES ? &sh->pv_done[g] : &sh->s_full[g], (turn - 1) & 1, sh, status)) return;
        store(stage, raw);
        if (!VALUES) {
          float* scales = reinterpret_cast<float*>(memory + M::KEY_SCALES) + (g * 2 + (turn & 1)) * kKeys;
          scales[tid] = ks * factor;
          scales[tid + (M::VALUE_SCALES - M::KEY_SCALES) / 4] = vs * kCodeScale;
          const unsigned there = __ballot_sync(0xffffffffu, held);
          const unsigned large = __ballot_sync(0xffffffffu, fabsf(vs) > kLargeScale);
          if ((tid & 31) == 0) {
            reinterpret_cast<unsigned char*>(&sh->valid[g][turn & 1])[tid / 32] = (unsigned char)((there & 1) | (there >> 16 & 1) << 1 | (large ? 4 : 0));
            sh->large[g][turn & 1][tid / 32] = large;
          }
        }
        fence_async();
        arrive(VALUES ? &sh->v_full[g] : &sh->k_full[g]);
        if (!VALUES) arrive(&sh->scaled[g][turn & 1]);  // of the softmax; k_full may be a phase further when it gets there
        if (t + 1 < walk.tiles) {
          const int rows = rows_of(t + 1, pages);
          if (!VALUES) held = scales_of(rows, &ks, &vs);
          load(rows, raw);
          pages = pages_of(t + 2);
        }
      }
    }
    walk.advance();
  }
}

template <typename T, int W>
__device__ __forceinline__ void multiply(Walk walk, Shared* sh, unsigned char* memory, unsigned tmem, int* status) {
  using M = Memory<W>;
  constexpr bool HALF = !std::is_same_v<T, __nv_bfloat16>;
  // float32 results; both factors float16 or both bfloat16; the values with their columns contiguous
  constexpr unsigned kScores = 1u << 4 | (HALF ? 0u : 1u << 7 | 1u << 10) | (unsigned)(kKeys >> 3) << 17 | 8u << 24;
  constexpr unsigned kOutputs = 1u << 4 | 1u << 7 | 1u << 10 | 1u << 16 | (unsigned)(W >> 3) << 17 | 8u << 24;
  const unsigned queries = matrix(at(memory + M::QUERIES), 16);
  unsigned score_turns[2] = {0, 0}, output_turns[2] = {0, 0}, units = 0;
  while (walk.next()) {
    if (walk.tiles > 0) {
      if (!wait(&sh->q_full, units++ & 1, sh, status)) return;
      for (int t = 0; t <= walk.tiles; ++t) {
        if (t < walk.tiles) {
          const int g = t & 1;
          const unsigned turn = score_turns[g]++;
          if (!wait(&sh->k_full[g], turn & 1, sh, status)) return;
          if (turn && !wait(&sh->pv_done[g], (turn - 1) & 1, sh, status)) return;  // the weights there are used up
          fence_after();
          const unsigned keys = matrix(at(memory + M::STAGES + g * 2 * M::TILE), 16);
#pragma unroll
          for (int k = 0; k < W / 16; ++k) {
            const unsigned to = ((k / 4) * (kKeys * 128) + (k % 4) * 32) / 16;
            product_ss(tmem + 2 * W + g * kKeys, queries + to, keys + to, kScores, k > 0);
          }
          commit(&sh->s_full[g]);
          if (t + 1 == walk.tiles) commit(&sh->q_free);
        }
        if (t > 0) {
          const int g = (t - 1) & 1;
          const unsigned turn = output_turns[g]++;
          if (!wait(&sh->p_ready[g], turn & 1, sh, status)) return;
          if (!wait(&sh->v_full[g], turn & 1, sh, status)) return;
          fence_after();
          const unsigned values = matrix(at(memory + M::STAGES + g * 2 * M::TILE + M::TILE), kKeys * 128), weights = tmem + 2 * W + g * kKeys;
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
#pragma unroll
            for (int part = 0; part < 2; ++part)
              product_ts(tmem + g * W, weights + 16 * k + 8 * part, values + k * 16 * 128 / 16, kOutputs,
                         t > 2 || k > 0 || part > 0);
          commit(&sh->pv_done[g]);
        }
      }
    }
    walk.advance();
  }
}

// Whether rows of 16-bit outputs lie on 16-byte boundaries, and eight of their columns stored.
__device__ __forceinline__ bool out_whole(const Args& a) {
  return ((reinterpret_cast<uintptr_t>(a.out) | (unsigned long long)(a.out_t * 2) | (unsigned long long)(a.out_h * 2)) & 15u) == 0;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v, bool whole) {
  if (whole) {
    store_vec<T>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_float<T>(v[i]);
  }
}

// The largest of a row's 128 scaled scores, of those alone that `seen_of` shows where MASKED.
template <bool MASKED, class Seen>
__device__ __forceinline__ float top_of(unsigned scores, const float* ks, Seen seen_of) {
  float top[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
  for (int ch = 0; ch < 8; ++ch) {
    unsigned r[16];
    load16(scores + 16 * ch, r);
    const unsigned see = MASKED ? seen_of(ch / 2) >> (16 * (ch & 1)) : 0;
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const float4 k = *reinterpret_cast<const float4*>(ks + 16 * ch + j);
      float x[4] = {__uint_as_float(r[j]) * k.x, __uint_as_float(r[j + 1]) * k.y, __uint_as_float(r[j + 2]) * k.z, __uint_as_float(r[j + 3]) * k.w};
      if (MASKED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (see >> (j + i)) & 1 ? x[i] : -INFINITY;
      }
      top[0] = fmaxf(top[0], fmaxf(x[0], x[1])), top[1] = fmaxf(top[1], fmaxf(x[2], x[3]));
    }
  }
  return fmaxf(top[0], top[1]);
}

// The same of capped scores, with the margin for the keys of `large`. Rare: short rather than fast.
template <typename T, class Seen>
__device__ __forceinline__ float top_of_large(unsigned scores, const float* ks, const unsigned* large, float cap2, Seen seen_of) {
  float top = -INFINITY;
#pragma unroll 1
  for (int ch = 0; ch < 8; ++ch) {
    unsigned r[16];
    load16(scores + 16 * ch, r);
    const unsigned see = seen_of(ch / 2) >> (16 * (ch & 1)), more = large[ch / 2] >> (16 * (ch & 1));
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float x = __uint_as_float(r[j]) * ks[16 * ch + j];
      if (cap2 > 0) x = cap2 * tanh_of<T>(x);
      if ((more >> j) & 1) x += kLargeMargin;
      if ((see >> j) & 1) top = fmaxf(top, x);
    }
  }
  return top;
}

// Writes a row's 128 weights times the values' scales over its scores, 16 at a time as 8 columns of leading and 8 of
// remaining parts, and returns the weights' sum.
template <typename T, bool CAP, bool MASKED, class Seen>
__device__ __forceinline__ float weights(unsigned scores, const float* ks, const float* vs, float base, float cap2, Seen seen_of) {
  float some[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int ch = 0; ch < 8; ++ch) {
    unsigned r[16], parts[16];
    load16(scores + 16 * ch, r);
    const unsigned see = MASKED ? seen_of(ch / 2) >> (16 * (ch & 1)) : 0;
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const float4 k = *reinterpret_cast<const float4*>(ks + 16 * ch + j), v = *reinterpret_cast<const float4*>(vs + 16 * ch + j);
      const float by[4] = {k.x, k.y, k.z, k.w}, scale[4] = {v.x, v.y, v.z, v.w};
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float s = __uint_as_float(r[j + i]);
        float p = exp2_fast(CAP ? fmaf(cap2, tanh_of<T>(s * by[i]), -base) : fmaf(s, by[i], -base));
        w[i] = p * scale[i];
        if (MASKED && !((see >> (j + i)) & 1)) p = 0.f, w[i] = 0.f;  // whatever lies there
        some[i] += p;
      }
      unsigned two[2];
      split<2>(w[0], w[1], two);
      parts[j / 2] = two[0], parts[8 + j / 2] = two[1];
      split<2>(w[2], w[3], two);
      parts[j / 2 + 1] = two[0], parts[8 + j / 2 + 1] = two[1];
    }
    store16(scores + 16 * ch, parts);
  }
  return (some[0] + some[1]) + (some[2] + some[3]);
}

template <typename T, int W>
__device__ __forceinline__ void weigh(const Cache& c, const Batch& b, const Args& a, Walk walk, Shared* sh, unsigned char* memory, unsigned tmem,
                                      int* status) {
  using M = Memory<W>;
  const int g = threadIdx.x / kGroupThreads, row = threadIdx.x % kGroupThreads;
  const unsigned lanes = (unsigned)(row & ~31) << 16;
  const unsigned scores = tmem + lanes + 2 * W + g * kKeys, sums = tmem + lanes + g * W;
  const float cap2 = a.cap * 1.4426950408889634f;
  const bool wide = out_whole(a);
  float* exchange = reinterpret_cast<float*>(memory + M::EXCHANGE) + row * 33;
  unsigned turns = 0, pieces = 0, chunks = 0;

  while (walk.next()) {
    const Sequence& q = walk.q;
    count_outside(c, q, a, walk.head == 0 && walk.tile == 0 && walk.from == 0 && threadIdx.x == 0);
    const int mine = walk.tile * kTensorRows + min(row, walk.rows - 1), token = mine / a.group;
    const long long sees = a.visible ? q.start : q.start + token + 1;
    const int limit = (int)(sees < 0 ? 0 : sees > a.capacity ? a.capacity : sees);
    unsigned long long bits = 0;
    if (a.visible) {
      bits = (unsigned long long)__ldg(a.visible + q.first + token);
      if (q.rows < 64) bits &= (1ull << q.rows) - 1;
    }
    float m = -INFINITY, sum = 0.f;
    bool seen = false;
    for (int t = g; t < walk.tiles; t += 2) {
      const unsigned turn = turns++;
      const int position = (walk.from + t) * kKeys;
      if (!wait_warp(&sh->scaled[g][turn & 1], turn >> 1 & 1, sh, status) || !wait_warp(&sh->s_full[g], turn & 1, sh, status)) return;
      fence_after();
      const float* ks = reinterpret_cast<const float*>(memory + M::KEY_SCALES) + (g * 2 + (turn & 1)) * kKeys;
      const float* vs = ks + (M::VALUE_SCALES - M::KEY_SCALES) / 4;
      const unsigned word = sh->valid[g][turn & 1];
      const bool inside = position + kKeys <= walk.all && word == 0x03030303u;
      // the keys of 32 from column 32 ch that this row sees
      auto seen_of = [&](int ch) -> unsigned {
        const int first = position + 32 * ch, below = limit - first;
        unsigned s = below >= 32 ? 0xffffffffu : below <= 0 ? 0u : (1u << below) - 1;
        if (a.visible) {
          const long long since = first - q.start;
          if (since >= 0 && since < 64) s |= (unsigned)(bits >> since);
          if (since < 0 && since > -32) s |= (unsigned)(bits << -since);
        }
        const unsigned halves = word >> (8 * ch);
        return s & ((halves & 1 ? 0xffffu : 0u) | (halves & 2 ? 0xffff0000u : 0u));
      };
      float top = -INFINITY;
      const bool margin = word & 0x04040404u;
      if (inside) {
        top = top_of<false>(scores, ks, seen_of);
        seen = true;
      } else {
        top = margin ? top_of_large<T>(scores, ks, sh->large[g][turn & 1], cap2, seen_of) : top_of<true>(scores, ks, seen_of);
        seen = seen || seen_of(0) || seen_of(1) || seen_of(2) || seen_of(3);
      }
      if (a.cap > 0 && !margin) top = top == -INFINITY ? top : cap2 * tanh_of<T>(top);
      const bool grown = top > m + kGrowth || (m == -INFINITY && top > m);
      if (__any_sync(0xffffffffu, grown)) {
        const float keep = grown ? exp2_fast(m - top) : 1.f;
        m = grown ? top : m;
        sum *= keep;
        if (t > 1) {
          if (!wait_warp(&sh->pv_done[g], (turn - 1) & 1, sh, status)) return;
          fence_after();
#pragma unroll 1
          for (int ch = 0; ch < W / 32; ++ch) {
            unsigned r[32];
            load32(sums + 32 * ch, r);
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
            store32(sums + 32 * ch, r);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : m;
      if (a.cap > 0)
        sum += inside ? weights<T, true, false>(scores, ks, vs, base, cap2, seen_of) : weights<T, true, true>(scores, ks, vs, base, cap2, seen_of);
      else
        sum += inside ? weights<T, false, false>(scores, ks, vs, base, cap2, seen_of) : weights<T, false, true>(scores, ks, vs, base, cap2, seen_of);
      stored();
      fence_before();
      arrive(&sh->p_ready[g]);
    }

    // join the groups: maxima and sums through shared memory, then 32 columns at a time
    const bool any = g < walk.tiles;
    if (any && !wait_warp(&sh->pv_done[g], (turns - 1) & 1, sh, status)) return;
    fence_after();
    float2* rows = reinterpret_cast<float2*>(memory + M::ROWS) + (pieces & 1) * 256;
    rows[g * 128 + row] = make_float2(m, seen && m == -INFINITY ? -1.f : sum);
    arrive(&sh->rows_full);
    if (!wait_warp(&sh->rows_full, pieces++ & 1, sh, status)) return;
    const float2 other = rows[(g ^ 1) * 128 + row], own = rows[g * 128 + row];
    const float mm = fmaxf(own.x, other.x), base = mm == -INFINITY ? 0.f : mm;
    const float factor = exp2_fast(own.x - base);
    const bool complete = walk.from == 0 && walk.to == q.steps;
    float* part = complete ? nullptr : a.parts + (2ll * blockIdx.x + (walk.from == 0)) * kTensorRows * (W + 2);
    Weights all;
    all.add(own.y, factor);
    all.add(other.y, exp2_fast(other.x - base));
    const float all_sum = all.sum();
    const bool two = walk.tiles > 1;
    T* out = out_row<T>(a, q, walk.head, mine);
#pragma unroll 1
    for (int ch = 0; ch < W / 32; ++ch) {
      unsigned r[32];
      if (any) load32(sums + 32 * ch, r);
      if (g == 1) {
        if (!two) break;
        if (chunks && !wait_warp(&sh->x_free, (chunks - 1) & 1, sh, status)) return;
#pragma unroll
        for (int j = 0; j < 32; ++j) exchange[j] = __uint_as_float(r[j]) * factor;
        arrive(&sh->x_full);
        ++chunks;
        continue;
      }
      float v[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = any ? __uint_as_float(r[j]) * factor : 0.f;
      if (two) {
        if (!wait_warp(&sh->x_full, chunks++ & 1, sh, status)) return;
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += exchange[j];
        arrive(&sh->x_free);
      }
#pragma unroll
      for (int j = 0; j < 32; j += 4) {  // the columns' order
        const float x = v[j + 1];
        v[j + 1] = v[j + 2], v[j + 2] = x;
      }
      if (complete) {
        const float by = all_sum > 0.f ? 1.f / all_sum : answer(0.f, all_sum);  // nothing seen: times zero
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j + i] *= by;
          if (row < walk.rows) store8<T>(out + 32 * ch + j, v + j, wide);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) part[(32 * ch + j) * kTensorRows + row] = v[j];
      }
      __syncwarp();
    }
    __syncwarp();
    fence_before();
    if (!complete && g == 0) {
      part[W * kTensorRows + row] = mm, part[(W + 1) * kTensorRows + row] = all_sum;
      if (walk.from == 0 && row == 0) a.cuts[blockIdx.x] = make_int4(walk.s, walk.head, walk.tile, (int)((walk.place + q.steps - 1) / walk.chunk));
    }
    walk.advance();
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(kTensorThreads, 1) attend_tiles(const Cache c, const Batch b, const Args a, int* status) {
  extern __shared__ unsigned char raw[];
  __shared__ Shared sh;
  __shared__ Begin begin;
  asm volatile("griddepcontrol.launch_dependents;");
  unsigned char* memory = raw + ((1024u - (at(raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    auto init = [](unsigned long long* bar, unsigned count) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(at(bar)), "r"(count));
    };
    init(&sh.q_full, 128), init(&sh.q_free, 1), init(&sh.rows_full, 256), init(&sh.x_full, 128), init(&sh.x_free, 128), init(&sh.drained, 1);
    for (int g = 0; g < 2; ++g) {
      init(&sh.k_full[g], 128), init(&sh.scaled[g][0], 128), init(&sh.scaled[g][1], 128), init(&sh.v_full[g], 128), init(&sh.s_full[g], 1), init(&sh.p_ready[g], 128), init(&sh.pv_done[g], 1);
      sh.valid[g][0] = sh.valid[g][1] = 0;
    }
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kProducts / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at(&sh.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  long long chunk;
  fence_before();
  begin_at<kTensorRows, kKeys, kTensorThreads / 32>(c, b, a, kLeastTiles, &chunk, &begin);  // ends with a barrier
  fence_after();
  const unsigned tmem = sh.tmem;
  if (!a.whole && threadIdx.x == 0) a.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
  __syncthreads();  // a cut that is written below comes after
  if (blockIdx.x * chunk < begin.total) {
    const Walk walk(c, b, a, begin, chunk);
    if (threadIdx.x < kKeyThreads) {
      more_registers<kSoftmaxRegisters>();
      weigh<T, W>(c, b, a, walk, &sh, memory, tmem, status);
    } else if (threadIdx.x < kProducts) {
      fewer_registers<kConverterRegisters>();
      convert<T, W>(c, b, a, walk, &sh, memory, status, threadIdx.x >= kValueThreads);
    } else {
      fewer_registers<kProductRegisters>();
      if (threadIdx.x == kProducts) {
        multiply<T, W>(walk, &sh, memory, tmem, status);
        commit(&sh.drained);  // whatever was queued has ended before the memory is given back
        wait(&sh.drained, 0, &sh, status);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kProducts / 32) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Joins the parts of the unit that begins in CTA blockIdx.x and was cut at its end, in the order of the keys: a thread per
// row, kColumns columns a CTA, since the parts lie column by column (a row is a thread where they are made).
constexpr int kColumns = 16;

template <typename T, int W>
__global__ void __launch_bounds__(kTensorRows) join_columns(const Cache c, const Batch b, const Args a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.x < 0) return;
  const Sequence q = sequence_of<kTensorRows, kKeys>(b, a, cut.x);
  const int row = threadIdx.x, column = blockIdx.y * kColumns, n = cut.w - blockIdx.x + 1;
  auto part = [&](int i) { return a.parts + (i == 0 ? 2ll * blockIdx.x + 1 : 2ll * (blockIdx.x + i)) * kTensorRows * (W + 2) + row; };
  float mm = -INFINITY;
#pragma unroll 8
  for (int k = 0; k < n; ++k) mm = fmaxf(mm, part(k)[W * kTensorRows]);
  const float base = mm == -INFINITY ? 0.f : mm;
  Weights all;
  float v[kColumns];
#pragma unroll
  for (int i = 0; i < kColumns; ++i) v[i] = 0.f;
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    const float* p = part(k);
    const float f = exp2_fast(p[W * kTensorRows] - base);
    all.add(p[(W + 1) * kTensorRows], f);
#pragma unroll
    for (int i = 0; i < kColumns; ++i) v[i] = fmaf(p[(column + i) * kTensorRows], f, v[i]);
  }
  if (row >= q.rows * a.group - cut.z * kTensorRows) return;
  const float all_sum = all.sum();
#pragma unroll
  for (int i = 0; i < kColumns; ++i) v[i] = answer(v[i], all_sum);
  T* out = out_row<T>(a, q, cut.y, cut.z * kTensorRows + row) + column;
  const bool whole = out_whole(a);
#pragma unroll
  for (int i = 0; i < kColumns; i += 8) store8<T>(out + i, v + i, whole);
}

template <typename T, int W>
int launch(const Cache& c, const Batch& b, const Args& a, cudaStream_t s) {
  const char* what = "tgcb_cached_attention";
  int dev = 0, *status = nullptr;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, what, cudaGetErrorString(e));
  const int rc = tgcb_internal_status_word(&status);
  if (rc != TGCB_OK) return rc;
  static std::atomic<unsigned long long> configured{0};
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    e = cudaFuncSetAttribute(attend_tiles<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, Memory<W>::BYTES);
    if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, what, cudaGetErrorString(e));
    configured.fetch_or(bit);
  }
  const long long tiles = (b.tokens * a.group + kTensorRows - 1) / kTensorRows + b.batch;
  const long long steps = a.whole ? 1 : (a.capacity + kKeys - 1) / kKeys;
  const long long pieces = (tiles * c.heads * steps + (a.whole ? 0 : kLeastTiles - 1)) / (a.whole ? 1 : kLeastTiles);
  const unsigned grid = (unsigned)(pieces < kTensorCtas ? pieces : kTensorCtas);
  attend_tiles<T, W><<<grid, kTensorThreads, Memory<W>::BYTES, s>>>(c, b, a, status);
  e = cudaGetLastError();
  if (e == cudaSuccess && !a.whole) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, W / kColumns);
    cfg.blockDim = dim3(kTensorRows);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, join_columns<T, W>, c, b, a);
  }
  if (e != cudaSuccess) return tgcb_internal_fail(TGCB_E_CUDA, what, cudaGetErrorString(e));
  return TGCB_OK;
}

}  // namespace

int tgcb_attend::attend_tensor(const Cache& c, const Batch& b, const Args& a, int dtype, cudaStream_t s) {
  if (dtype == TGCB_BF16) return c.width == 128 ? launch<__nv_bfloat16, 128>(c, b, a, s) : launch<__nv_bfloat16, 64>(c, b, a, s);
  return c.width == 128 ? launch<__half, 128>(c, b, a, s) : launch<__half, 64>(c, b, a, s);
}
