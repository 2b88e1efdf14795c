// Attention of new tokens over a paged key-value cache.
//
// Mathematics: with s = scale * q . k in log2 units, a pass over the slots
// keeps m = max s, l = sum 2^(s - m) and o = sum 2^(s - m) v; two such states
// join as m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m), o likewise, and
// out = o / l.  m, l, o, s are fp32.  The products run on the tensor cores
// with fp32 accumulation; q, k, v enter exactly (they are 16-bit) and the
// probabilities as two 16-bit terms, hi cut off and lo rounded (bf16: within 2^-16
// relative; fp16, taken times 2^15 for its short range: 2^-21 relative, or 2^-38 of
// the row's largest where that is more), so the output is rounded once.
//
// Bound: memory.  A cached token costs 4 * head_dim bytes per kv head and
// 4 * head_dim * rows flops; with few rows (query heads of a kv head times
// step tokens) warp-level MMAs at m = 16 rows keep far ahead of HBM, and
// their operands come straight from the shared-memory tiles.
//
// Split: the tiles (128 tokens, 64 above head_dim 128) of all (sequence, row
// tile, kv head) items form one index space (an item's tiles follow kItemCost positions that stand for
// its fixed cost), cut into equal runs, one per resident CTA; lengths are read
// on the device, so ragged batches balance by themselves.  A run that ends
// inside an item leaves (m, l, o) in the workspace and the item's last CTA to
// arrive (a counter at the item's first CTA) joins them in run order, so the
// result does not depend on timing.
//
// Tile: four producer warps fetch a tile's K and V as tensor (TMA) boxes of
// min(16, page_size) tokens, page ids one tile ahead, through a ring of stages;
// the hardware's 128-byte swizzle makes the fragment loads conflict-free.  Up to 16 rows, each consumer warp takes its own 16 tokens;
// with more, MT row tiles of 16 take W/MT warps each.  Consumers meet only
// where an item ends.  An item's queries go from memory straight to the
// registers of the products, fetched while the item before is joined.  Slots
// that a row does not see may hold anything: their scores are replaced and
// their V zeroed in registers, in the blocks where that can happen.
//
// Measured (B200): one sequence of 131071 tokens, 64 query and 8 kv heads of
// 128, 86 us = 6.2 TB/s (0.95 of the measured HBM rate); 64 sequences of 100 to
// 8000 tokens, 32 / 8 heads, 84 us = 5.8 TB/s (0.88); one of 1024 tokens 7.9 us,
// a chain of latencies (launch, lengths, page ids, tile, part, join); 64 rows
// over 32000 tokens 66 us (the warps' products).  One producer warp instead of
// four held the ragged batch at 90 us: a warp issues a box every 90 cycles or so.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "tp_decode.cuh"
#include "tp_paged.cuh"

using namespace tp;

namespace {

// An item costs about two tiles beside its own (its queries, the join of the
// warps), so the split counts it as that many tiles more: 64 sequences of 100 to
// 8000 tokens 81 us, against 101 us with equal tile counts.
constexpr int kItemCost = 2;
constexpr int kPaMaxCtas = 512;
constexpr int64_t kPaStoredMax = int64_t(1) << 30;  // bytes of stored scores
constexpr int kWtThreads = 128;
constexpr int kWtRound = 32;  // row tiles whose weights are summed before they join the slot's
constexpr int kPaStatusOff = kPaMaxCtas * 4;      // status word after the counters
constexpr int kPaCounterBytes = kPaStatusOff + 256;

struct AttnParams {
  CUtensorMap k_map, v_map;  // {64 elements, token, panel, head, page}, or without panels {head_dim, token, 1, head, page}
  const void* q;
  void* out;
  float* lse;
  const int32_t* block_table;
  const int32_t* lengths;
  float* scores;
  int64_t num_pages, table_stride;
  int panels;       // boxes hold all panels of 64 elements
  int lg_box;       // log2 of the tokens per box: min(16, page_size)
  int batch, tokens, q_heads, kv_heads, group, head_dim;
  int lg_page, capacity;
  uint64_t group_inv;  // ceil(2^64 / group), 0 for a group of 1
  int rows;      // tokens * group: query rows of a kv head
  int row_tiles;
  float scale_log2;
  unsigned* counters;
  unsigned* status;
  unsigned polls;  // limit of a wait
  int hold;        // a test's: one producer stops before tile hold - 1 of its block (0: none does)
  float* part_o;   // [ctas][2][16*MT][HD]
  float2* part_ml; // [ctas][2][16*MT]
  float* lse2;     // log2 units (accumulate only): [batch][tokens][q_heads], with stored scores [batch][kv_heads][rows]
  float* sbuf;     // [index space][16*MT][TILE] scores in log2 units (stored scores only)
  // the weights kernel's
  float lse_unit;        // what lse2 is taken times
  const int32_t* counts; // [batch] step tokens whose weights are added, or NULL: all
  const void* k_pages;   // and its strides, in elements
  int64_t page_stride, head_stride, token_stride;
};

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int token, int head, int page,
                                        uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(dst), "l"(map), "r"(x), "r"(token), "r"(0), "r"(head), "r"(page), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}

// Mma<T>::split: x = hi + lo for x, y >= 0.  hi is x cut off and lo the rest, both
// raised to the type's least positive (bf16: normal) value: an infinite V times a
// term of 0, or of the other sign, would make NaN of an infinite output.
template <class T>
struct Mma;
template <>
struct Mma<__half> {
  // What the probabilities are taken times: at most 2^15 then, so fp16 keeps
  // them down to 2^-39 of the row's largest (1 in its place would lose all
  // below 2^-25, a long flat tail under one large score).
  static constexpr float kScale = 32768.f;
  // either half infinite or NaN: its exponent is all ones
  static __device__ __forceinline__ bool not_finite(uint32_t v) {
    constexpr uint32_t E = 0x7c007c00u;
    return (v & E & 0xffffu) == (E & 0xffffu) || (v & E & 0xffff0000u) == (E & 0xffff0000u);
  }
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    __half2 h;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(reinterpret_cast<uint32_t&>(h)) : "f"(y), "f"(x));
    const __half2 least = __halves2half2(__ushort_as_half(1), __ushort_as_half(1));
    const float2 f = __half22float2(h);
    const __half2 r = __hmax2(__floats2half2_rn(x - f.x, y - f.y), least);
    h = __hmax2(h, least);
    hi = reinterpret_cast<const uint32_t&>(h);
    lo = reinterpret_cast<const uint32_t&>(r);
  }
};
template <>
struct Mma<__nv_bfloat16> {
  static constexpr float kScale = 1.f;  // fp32's range
  // either half infinite or NaN: its exponent is all ones
  static __device__ __forceinline__ bool not_finite(uint32_t v) {
    constexpr uint32_t E = 0x7f807f80u;
    return (v & E & 0xffffu) == (E & 0xffffu) || (v & E & 0xffff0000u) == (E & 0xffff0000u);
  }
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    __nv_bfloat162 h;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(reinterpret_cast<uint32_t&>(h)) : "f"(y), "f"(x));
    const __nv_bfloat162 least = __halves2bfloat162(__ushort_as_bfloat16(0x80), __ushort_as_bfloat16(0x80));
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 r = __hmax2(__floats2bfloat162_rn(x - f.x, y - f.y), least);
    h = __hmax2(h, least);
    hi = reinterpret_cast<const uint32_t&>(h);
    lo = reinterpret_cast<const uint32_t&>(r);
  }
};

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// 2^(a - b) for a <= b, 0 where a is -inf (also where both are).
__device__ __forceinline__ float exp2_diff(float a, float b) { return a == -INFINITY ? 0.f : exp2f(a - b); }

// ---------------------------------------------------------------------------
// the index space of tiles
// ---------------------------------------------------------------------------
// Step token of query row `row`.
__device__ __forceinline__ int token_of(const AttnParams& p, int row) {
  return p.group_inv ? static_cast<int>(__umul64hi(static_cast<uint64_t>(row), p.group_inv)) : row;
}
// Slots that query row `row` of sequence length `len` (before the step) sees.
__device__ __forceinline__ int visible(const AttnParams& p, int len, int row) {
  return len < 0 ? 0 : static_cast<int>(min((int64_t)len + token_of(p, row) + 1, (int64_t)p.capacity));
}
// Tiles of an item: one at least, so that every output row is written.
template <class S>
__device__ __forceinline__ int item_tiles(const AttnParams& p, int len, int rt) {
  const int vis = visible(p, len, min(p.rows, (rt + 1) * S::RT) - 1);
  return max(1, (vis + S::TILE - 1) / S::TILE);
}
// Positions of a sequence's items.
template <class S>
__device__ __forceinline__ int seq_size(const AttnParams& p, int len) {
  int n = 0;
  for (int rt = 0; rt < p.row_tiles; ++rt) n += kItemCost + item_tiles<S>(p, len, rt);
  return n * p.kv_heads;
}

struct Cursor {  // one tile: sequence, row tile, kv head, tile of the item, the item's tiles and last seen slot + 1
  int b, rt, h, tile, n, hi, len;
};

template <class S>
__device__ __forceinline__ void set_item(const AttnParams& p, Cursor& c) {
  c.hi = visible(p, c.len, min(p.rows, (c.rt + 1) * S::RT) - 1);
  c.n = max(1, (c.hi + S::TILE - 1) / S::TILE);
}

template <class S>
__device__ __forceinline__ void step_cursor(const AttnParams& p, Cursor& c) {
  if (++c.tile < c.n) return;
  c.tile = 0;
  if (++c.h < p.kv_heads) return;
  c.h = 0;
  if (++c.rt == p.row_tiles) {
    c.rt = 0;
    c.len = p.lengths[++c.b];
  }
  set_item<S>(p, c);
}

// Sum over a block of W warps of one value per thread (all threads call it).
template <int W>
__device__ __forceinline__ int block_sum(int v, int* s_tmp) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_tmp[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) t += s_tmp[w];
  return t;
}

// This CTA's equal share [t0, t1) of the concatenation of `count(len)`
// positions per sequence, `per` positions each; the sequence holding t0, its
// length and the positions before it.  False (in every thread) where the share
// is empty.  s_tmp: W + 3 words.
template <int W, class F>
__device__ __forceinline__ bool find_share(const AttnParams& p, F count, int* s_tmp, int& per, int& t0, int& t1, int& b_out,
                                           int& len_out, int& before) {
  constexpr int N = 32 * W;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int rest = 0;  // sequences past the first block of the scan
  if (p.batch > N) {
    for (int b = threadIdx.x + N; b < p.batch; b += N) rest += count(p.lengths[b]);
    rest = block_sum<W>(rest, s_tmp);
  }
  int run = 0;
  for (int base = 0; base < p.batch; base += N) {
    const int b = base + threadIdx.x;
    const int len = b < p.batch ? p.lengths[b] : 0, own = b < p.batch ? count(len) : 0;
    int inc = own;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, m);
      if (lane >= m) inc += o;
    }
    __syncthreads();
    if (lane == 31) s_tmp[warp] = inc;
    if (threadIdx.x == 0) s_tmp[W] = -1;
    __syncthreads();
    int part = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) inc += s_tmp[w];
      part += s_tmp[w];
    }
    if (base == 0) {
      const int total = part + rest;
      per = (total + gridDim.x - 1) / gridDim.x;
      t0 = min((int)blockIdx.x * per, total);
      t1 = min(t0 + per, total);
      if (t0 >= t1) return false;
    }
    if (own > 0 && run + inc - own <= t0 && t0 < run + inc) {
      s_tmp[W] = b;
      s_tmp[W + 1] = run + inc - own;
      s_tmp[W + 2] = len;
    }
    __syncthreads();
    if (s_tmp[W] >= 0) break;
    run += part;
  }
  b_out = s_tmp[W];
  before = s_tmp[W + 1];
  len_out = s_tmp[W + 2];
  return true;
}

// ---------------------------------------------------------------------------
// the attention kernel
// ---------------------------------------------------------------------------
template <int HD, int MT>
struct PaShape {
  static constexpr int W = HD == 256 ? 4 : 8;        // consumer warps
  static constexpr int THREADS = 32 * (W + 4);       // and four producers
  static constexpr int TILE = 16 * W;                // tokens
  static constexpr int RT = 16 * MT;                 // rows of an item
  static constexpr int WT = W / MT;                  // warps along the tokens
  static constexpr int kPanels = HD / 64;            // 128-byte columns of a block of 16 tokens
  static constexpr int kBlock = 16 * HD * 2;         // its K (or V): [panel][16][128 bytes], swizzled
  static constexpr int kKV = W * kBlock;
  static constexpr int kStage = 2 * kKV;             // 32 to 64 KB
  static constexpr int kStages = HD == 64 ? 6 : 3;
  static constexpr int kSmem = kStages * kStage;
  static_assert(kSmem <= 225 * 1024, "shared memory");
  static_assert(kStage % 1024 == 0, "the swizzle repeats every 1024 bytes");
  static_assert(W * 16 * HD * 4 == kStage, "the join buffer reuses a consumed stage");
};

// A stage's barrier; false when the wait runs out.
//
// What happens then: a consumer that gave up neither waits nor hands stages back
// any more, so the producers run dry within the ring and give up too, and the
// rows it has a part in become NaN.  Consumers still go through their items
// (they meet at the ends, and other blocks may wait to be counted), and before
// the block ends the producers make up the arrivals of the tiles that some of
// them had begun and wait, with a limit, for what is in flight.
__device__ __forceinline__ bool stage_wait(uint64_t* bar, unsigned parity, unsigned polls) {
  const uint32_t a = smem_u32(bar);
  for (unsigned i = 0; i < polls; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}

template <int N>
__device__ __forceinline__ void block_end_sync() {  // of all N threads, producers and consumers
  asm volatile("bar.sync 2, %0;" ::"n"(N) : "memory");
}

// The producers' end of a block that gave up: the arrivals of the tiles [fetched,
// most) that others began and this one did not (no stage is more than a round
// ahead, and none of these was handed back), then a wait for what is in flight.
__device__ __noinline__ void settle(uint64_t* full, int stages, int fetched, const int* all_fetched, unsigned* status) {
  int most = 0;
  for (int i = 0; i < 4; ++i) most = max(most, all_fetched[i]);
  for (int i = fetched; i < most; ++i)
    if ((threadIdx.x & 31) == 0) mbar_arrive(&full[i % stages]);
  for (int i = max(0, most - stages); i < most; ++i)
    if (!mbar_wait(&full[i % stages], (i / stages) & 1)) atomicOr(status, 2u);
}
// A test's held wait: until another of the block's waits runs out.
__device__ __noinline__ void hold_wait(unsigned polls, const volatile int& gone) {
  for (unsigned i = 0; i < polls && !gone; ++i) __nanosleep(1000);
}

template <int N>
__device__ __forceinline__ void consumers_sync() {  // of N threads; the producers never join
  asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}

// STORE: the scores go to the workspace.
template <class T, int HD, int MT, bool STORE>
__global__ void __launch_bounds__(PaShape<HD, MT>::THREADS, 1) paged_attn_kernel(const __grid_constant__ AttnParams p) {
  using S = PaShape<HD, MT>;
  constexpr int RT = S::RT, W = S::W, WT = S::WT, NB = MT == 1 || HD == 256 ? 1 : 2, kStages = S::kStages;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ int s_tmp[W + 8];
  __shared__ __align__(8) uint64_t s_full[kStages], s_empty[kStages];
  __shared__ uint32_t s_valid[kStages][W];  // the tokens of a block of 16 that have a page
  __shared__ float s_m[W][16], s_l[W][16];
  __shared__ bool s_last;
  __shared__ volatile int s_gone;  // a wait ran out
  __shared__ int s_fetched[4];     // tiles that each producer began
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t sbase = smem_u32(smem);
  if (tid == 0) {
    s_gone = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.v_map) : "memory");
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s_full[i], 4);
      mbar_init(&s_empty[i], W);
    }
    fence_mbar_init();
  }

  // ---- this CTA's run [t0, t1) of the index space ----
  int per, t0, t1, before;
  Cursor c;
  pdl_wait();
  pdl_trigger();  // after the wait: the weights kernel of stored scores reads the lengths at once
  // (its barriers also publish the mbarriers and s_gone)
  if (!find_share<W + 4>(p, [&](int len) { return seq_size<S>(p, len); }, s_tmp, per, t0, t1, c.b, c.len, before)) return;
  int rem = t0 - before;
  for (c.rt = 0;; ++c.rt) {
    set_item<S>(p, c);
    if (rem < p.kv_heads * (kItemCost + c.n)) break;
    rem -= p.kv_heads * (kItemCost + c.n);
  }
  c.h = rem / (kItemCost + c.n);
  c.tile = rem - c.h * (kItemCost + c.n) - kItemCost;
  if (c.tile < 0) {  // the run begins in the item's fixed part
    t0 -= c.tile;
    c.tile = 0;
  }
  if (t0 >= t1) return;
  int stage = 0, t = t0;
  unsigned phase = 0;  // parity of the stage's round; a consumer's has kGaveUp set once its wait ran out
  constexpr unsigned kGaveUp = 2;
  auto next_stage = [&] {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1u;
    }
  };

  // Of the 168 registers that 384 threads get each, the producers' warpgroup
  // gives up 112: 256 * 224 + 128 * 56 = 384 * 168.  (256 threads have 255.)
  if (warp >= W) {
    if (W == 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // the producers: a quarter of a tile's boxes each, a box per lane (a warp
    // issues its lanes' copies one after the other, some 90 cycles apart)
    constexpr int B = W / 4;  // blocks of 16 tokens per producer
    const int lg_boxes = 4 - p.lg_box, page_mask = (1 << p.lg_page) - 1;
    const int at = (warp - W) * (16 * B) + (lane << p.lg_box);  // the lane's token of the tile
    const bool mine = lane < (B << lg_boxes);
    auto page_of = [&] {
      const int tok = c.tile * S::TILE + at;
      return mine && tok < p.capacity ? p.block_table[c.b * p.table_stride + (tok >> p.lg_page)] : -1;
    };
    int pid = page_of(), fetched = 0;
    while (true) {
      bool go = stage_wait(&s_empty[stage], phase ^ 1u, p.polls);  // (the first round of the ring does not wait)
      if (p.hold && p.hold == fetched + 1 && warp == W + 1) {
        hold_wait(p.polls, s_gone);
        go = false;
      }
      if (!__all_sync(0xffffffffu, go)) {
        s_gone = 1;
        if (lane == 0) atomicOr(p.status, 1u);
        break;
      }
      const uint32_t bar = smem_u32(&s_full[stage]);
      const int tok = c.tile * S::TILE + at;
      const bool ok = mine && tok < c.hi && pid >= 0 && pid < p.num_pages;
      const uint32_t got = __ballot_sync(0xffffffffu, ok);
      if (lane < B) {
        uint32_t valid = 0;
        for (int i = 0; i < 1 << lg_boxes; ++i)
          if ((got >> ((lane << lg_boxes) + i)) & 1u) valid |= ((1u << (1 << p.lg_box)) - 1u) << (i << p.lg_box);
        s_valid[stage][(warp - W) * B + lane] = valid;
      }
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                     "r"(__popc(got) * (S::kPanels * 2 * 128 << p.lg_box))
                     : "memory");
      __syncwarp();
      if (ok) {
        const uint32_t d = sbase + stage * S::kStage + (at >> 4) * S::kBlock + ((at & 15) << 7);
        for (int i = 0; i < (p.panels ? 1 : S::kPanels); ++i) {
          tma_box(d + i * 2048, &p.k_map, i * 64, tok & page_mask, c.h, pid, bar);
          tma_box(d + S::kKV + i * 2048, &p.v_map, i * 64, tok & page_mask, c.h, pid, bar);
        }
      }
      ++fetched;
      t += c.tile + 1 == c.n ? 1 + kItemCost : 1;
      if (t >= t1) break;
      step_cursor<S>(p, c);
      pid = page_of();
      next_stage();
    }
    if (lane == 0) s_fetched[warp - W] = fetched;
    block_end_sync<S::THREADS>();
    if (s_gone) settle(s_full, kStages, fetched, s_fetched, p.status);
    return;
  }
  if (W == 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");

  // ---- the consumers: this warp's 16 rows ----
  const int mt = warp / WT, tw = warp % WT;
  const int r0 = lane >> 2, cq = lane & 3;  // this thread: rows r0, r0 + 8, columns 2 cq + {0, 1} of each 8
  // Fragments of the queries.  A product may take the columns in any order
  // that both operands share: this thread holds the 16-byte chunks 2 cq and
  // 2 cq + 1 of each 64 columns, so both operands load 16 bytes at a time.
  uint32_t qf[HD / 16][4];
  auto load_queries = [&] {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = c.rt * RT + mt * 16 + r0 + 8 * e, j = token_of(p, row);
      const T* q = static_cast<const T*>(p.q) +
                   (((int64_t)c.b * p.tokens + j) * p.q_heads + c.h * p.group + row - j * p.group) * p.head_dim;
#pragma unroll
      for (int kk = 0; kk < HD / 32; ++kk) {
        const int chunk = (kk >> 1) * 8 + 2 * cq + (kk & 1);
        const uint4 x = row < p.rows && chunk * 8 < p.head_dim ? __ldg(reinterpret_cast<const uint4*>(q + chunk * 8))
                                                                : make_uint4(0u, 0u, 0u, 0u);
        qf[2 * kk][e] = x.x;
        qf[2 * kk][2 + e] = x.y;
        qf[2 * kk + 1][e] = x.z;
        qf[2 * kk + 1][2 + e] = x.w;
      }
    }
  };
  load_queries();

  while (true) {  // an item, or this run's part of it
    float o[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int row0 = c.rt * RT + mt * 16, last_row = min(row0 + 16, p.rows) - 1;
    int jr[2], vis[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = row0 + r0 + 8 * e;
      jr[e] = token_of(p, row);
      vis[e] = row < p.rows ? visible(p, c.len, row) : 0;
    }
    const int j_lo = token_of(p, row0), j_hi = token_of(p, max(last_row, 0));
    const int vis_lo = last_row >= row0 ? visible(p, c.len, row0) : 0;  // slots seen by every row,
    const int vis_hi = last_row >= row0 ? visible(p, c.len, last_row) : 0;  // and by any
    const int t_end = min(t1, t + c.n - c.tile);
    // the rows' scores of a block, in log2 units, for the accumulated weights
    auto store_scores = [&](int blk, const float (*s)[4]) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (row0 + r0 + 8 * e < p.rows)
#pragma unroll
          for (int n = 0; n < 2; ++n)
            *reinterpret_cast<float2*>(p.sbuf + ((size_t)t * RT + mt * 16 + r0 + 8 * e) * S::TILE + blk * 16 + n * 8 + cq * 2) =
                s ? make_float2(s[n][2 * e], s[n][2 * e + 1]) : make_float2(-INFINITY, -INFINITY);
    };

    while (true) {
      const uint32_t st = sbase + stage * S::kStage;
      if (phase < kGaveUp && !stage_wait(&s_full[stage], phase, p.polls)) {
        phase |= kGaveUp;  // reported through the status word
        s_gone = 1;
        atomicOr(p.status, 1u);
      }
      // this warp's MT blocks of 16 tokens, NB at a time
#pragma unroll 1
      for (int blk = tw * MT; blk < (tw + 1) * MT; blk += NB) {
        const int tok0 = c.tile * S::TILE + blk * 16;
        if (tok0 >= vis_hi) {  // nothing here for these rows
          if (STORE)
            for (int i = 0; i < NB; ++i) store_scores(blk + i, nullptr);
          continue;
        }
        uint32_t valid[NB];
        bool whole = true;  // every slot seen by every row
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          valid[i] = phase >= kGaveUp ? 0xffffu : s_valid[stage][blk + i];
          whole = whole && valid[i] == 0xffffu && tok0 + 16 * (i + 1) <= vis_lo;
        }
        const uint32_t kb = st + blk * S::kBlock;
        float s[2 * NB][4], s2[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s2[0][e] = s2[1][e] = 0.f;
#pragma unroll
          for (int n = 0; n < 2 * NB; ++n) s[n][e] = 0.f;
        }
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk) {  // four chains of products
          const int chunk = 2 * cq + (kk & 1);
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            uint4 kf[2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
              kf[n] = lds16(kb + i * S::kBlock + (kk >> 1) * 2048 + (n * 8 + r0) * 128 + (((chunk ^ r0) & 7) << 4));
            Mma<T>::run(s[2 * i], qf[2 * kk], kf[0].x, kf[0].y);
            Mma<T>::run(s[2 * i + 1], qf[2 * kk], kf[1].x, kf[1].y);
            Mma<T>::run(NB == 1 ? s2[0] : s[2 * i], qf[2 * kk + 1], kf[0].z, kf[0].w);
            Mma<T>::run(NB == 1 ? s2[1] : s[2 * i + 1], qf[2 * kk + 1], kf[1].z, kf[1].w);
          }
        }
#pragma unroll
        for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = (NB == 1 ? s[n][e] + s2[n % 2][e] : s[n][e]) * p.scale_log2;
        if (!whole) {
#pragma unroll
          for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int col = n * 8 + cq * 2 + (e & 1);
              if (!((valid[n / 2] >> (col & 15)) & 1u) || tok0 + col >= vis[e >> 1]) s[n][e] = -INFINITY;
            }
        }
        if (STORE) {
          if (phase >= kGaveUp) {  // (what the slots hold is anything: their weights become NaN)
#pragma unroll
            for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[n][e] = s[n][e] == -INFINITY ? s[n][e] : __int_as_float(0x7fc00000);
          }
#pragma unroll
          for (int i = 0; i < NB; ++i) store_scores(blk + i, s + 2 * i);
        }
        // running maximum: the quad of four lanes shares a row
        float mn[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[0][2 * e], s[0][2 * e + 1]);
#pragma unroll
          for (int n = 1; n < 2 * NB; ++n) x = fmaxf(x, fmaxf(s[n][2 * e], s[n][2 * e + 1]));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          mn[e] = fmaxf(m[e], x);
        }
        if (__any_sync(0xffffffffu, mn[0] != m[0] || mn[1] != m[1])) {
          const float a0 = exp2_diff(m[0], mn[0]), a1 = exp2_diff(m[1], mn[1]);
          m[0] = mn[0];
          m[1] = mn[1];
          l[0] *= a0;
          l[1] *= a1;
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) {
            o[n][0] *= a0;
            o[n][1] *= a0;
            o[n][2] *= a1;
            o[n][3] *= a1;
          }
        }
        const float b0 = m[0] == -INFINITY ? 0.f : m[0], b1 = m[1] == -INFINITY ? 0.f : m[1];
        uint32_t ph[NB][4], pl[NB][4];
        float add[2] = {0.f, 0.f};  // (the block's sum first: many small terms beside a large l then lose little)
#pragma unroll
        for (int n = 0; n < 2 * NB; ++n) {
          s[n][0] = exp2f(s[n][0] - b0);
          s[n][1] = exp2f(s[n][1] - b0);
          s[n][2] = exp2f(s[n][2] - b1);
          s[n][3] = exp2f(s[n][3] - b1);
          add[0] += s[n][0] + s[n][1];
          add[1] += s[n][2] + s[n][3];
          constexpr float C = Mma<T>::kScale;
          Mma<T>::split(s[n][0] * C, s[n][1] * C, ph[n / 2][n % 2 * 2], pl[n / 2][n % 2 * 2]);
          Mma<T>::split(s[n][2] * C, s[n][3] * C, ph[n / 2][n % 2 * 2 + 1], pl[n / 2][n % 2 * 2 + 1]);
        }
        l[0] += add[0];
        l[1] += add[1];
        if (!whole) {  // slots that a row does not see have no weight at all
#pragma unroll
          for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t some = (s[n][2 * e] > 0.f ? 0x0000ffffu : 0u) | (s[n][2 * e + 1] > 0.f ? 0xffff0000u : 0u);
              ph[n / 2][n % 2 * 2 + e] &= some;
              pl[n / 2][n % 2 * 2 + e] &= some;
            }
        }
        // o += P V, 16-column pairs at a time (independent products in a row);
        // `keep` masks the V fragments' two tokens of each 8 where MASKED
        auto v_frag = [&](int i, int nn, uint32_t (&vf)[4]) {
          const int r = lane & 15, chunk = nn * 2 + (lane >> 4);
          ldsm4t(vf, kb + i * S::kBlock + S::kKV + (chunk >> 3) * 2048 + r * 128 + (((chunk ^ r) & 7) << 4));
        };
        auto keep_of = [&](int i, int see, uint32_t (&k)[2]) {  // tokens of block i below `see` that have a page
          see -= tok0 + 16 * i;
          const uint32_t seen = (see >= 16 ? valid[i] : see <= 0 ? 0u : valid[i] & ((1u << see) - 1u)) >> (cq * 2);
          k[0] = (seen & 1u ? 0x0000ffffu : 0u) | (seen & 2u ? 0xffff0000u : 0u);
          k[1] = (seen & 0x100u ? 0x0000ffffu : 0u) | (seen & 0x200u ? 0xffff0000u : 0u);
        };
        auto product = [&](int i, const uint32_t (&k)[2], auto masked) {
#pragma unroll
          for (int nn = 0; nn < HD / 16; nn += 2) {
            uint32_t vf[2][4];
            v_frag(i, nn, vf[0]);
            v_frag(i, nn + 1, vf[1]);
            if constexpr (decltype(masked)::value) {
#pragma unroll
              for (int e = 0; e < 8; ++e) vf[e / 4][e % 4] &= k[e & 1];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) Mma<T>::run(o[2 * nn + e], ph[i], vf[e / 2][e % 2 * 2], vf[e / 2][e % 2 * 2 + 1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) Mma<T>::run(o[2 * nn + e], pl[i], vf[e / 2][e % 2 * 2], vf[e / 2][e % 2 * 2 + 1]);
          }
        };
        if (whole) {
          const uint32_t all[2] = {~0u, ~0u};
#pragma unroll
          for (int i = 0; i < NB; ++i) product(i, all, std::false_type{});
        } else {
          // Slots that no row sees are zeroed (0 * what they hold may be NaN).
          // Slots that some rows see and others do not are harmless while V is
          // finite there; where it is not, each step token's product takes only
          // what the token sees, and only its own rows of the result.
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            uint32_t k[2];
            keep_of(i, vis_hi, k);
            bool apart = false;
            if (j_lo < j_hi) {
#pragma unroll
              for (int nn = 0; nn < HD / 16; ++nn) {
                uint32_t vf[4];
                v_frag(i, nn, vf);
#pragma unroll
                for (int e = 0; e < 4; ++e) apart = apart || Mma<T>::not_finite(vf[e] & k[e & 1]);
              }
              apart = __any_sync(0xffffffffu, apart);
            }
            if (!apart) {
              product(i, k, std::true_type{});
              continue;
            }
#pragma unroll 1
            for (int j = j_lo; j <= j_hi; ++j) {
              keep_of(i, visible(p, c.len, j * p.group), k);
#pragma unroll
              for (int nn = 0; nn < HD / 16; ++nn) {
                uint32_t vf[4];
                v_frag(i, nn, vf);
                float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
                Mma<T>::run(x, ph[i], vf[0] & k[0], vf[1] & k[1]);
                Mma<T>::run(y, ph[i], vf[2] & k[0], vf[3] & k[1]);
                Mma<T>::run(x, pl[i], vf[0] & k[0], vf[1] & k[1]);
                Mma<T>::run(y, pl[i], vf[2] & k[0], vf[3] & k[1]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (jr[e >> 1] == j) {
                    o[2 * nn][e] += x[e];
                    o[2 * nn + 1][e] += y[e];
                  }
              }
            }
          }
        }
      }
      if (t + 1 == t_end) break;
      __syncwarp();
      if (lane == 0 && phase < kGaveUp) mbar_arrive(&s_empty[stage]);
      ++t;
      ++c.tile;
      next_stage();
    }

    // ---- the end of this CTA's part of the item ----
    const int nrow = min(RT, p.rows - c.rt * RT);
    const Cursor done = c;
    const int t_next = t + (c.tile + 1 == c.n ? 1 + kItemCost : 1);
    if (t_next < t1) {  // the next item's queries, on their way while this one is joined
      step_cursor<S>(p, c);
      load_queries();
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (__any_sync(0xffffffffu, phase >= kGaveUp)) l[e] = __int_as_float(0x7fc00000);  // (the products are the warp's)
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (cq == 0) s_m[warp][r0 + 8 * e] = m[e];
    }
    consumers_sync<32 * W>();  // every warp is done with this tile: its stage becomes the join buffer
    float* buf = reinterpret_cast<float*>(smem + stage * S::kStage);  // [warp][16][HD], 32-byte groups swizzled
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = r0 + 8 * e;
      if (mt * 16 + r < nrow) {  // the warp's sums, to the row's maximum over its warps
        float M = s_m[mt * WT][r];
#pragma unroll
        for (int w = 1; w < WT; ++w) M = fmaxf(M, s_m[mt * WT + w][r]);
        const float f = exp2_diff(m[e], M);
        if (cq == 0) s_l[warp][r] = l[e] == 0.f ? 0.f : l[e] * f;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
          *reinterpret_cast<float2*>(buf + (warp * 16 + r) * HD + ((n * 8 + cq * 2) ^ ((r & 7) << 3))) =
              make_float2(o[n][2 * e] * f, o[n][2 * e + 1] * f);
      }
    }
    consumers_sync<32 * W>();
    const int begin = t - done.tile, end = begin + done.n;  // the item's tiles
    const int c0 = begin / per, c1 = (end - 1) / per; // CTAs that share it
    const bool alone = c0 == c1;
    const int slot = blockIdx.x == c0 ? 1 : 0;  // an item that began in an earlier CTA: slot 0
    float* po = p.part_o + (size_t)(blockIdx.x * 2 + slot) * RT * HD;
    float2* pml = p.part_ml + (blockIdx.x * 2 + slot) * RT;
    const int64_t out0 = ((int64_t)done.b * p.tokens) * p.q_heads + done.h * p.group;
    auto finish = [&](int r, int d, const auto& v, float M, float L) {  // row r, elements d..
      constexpr int N = sizeof(v) / sizeof(float);
      const int row = done.rt * RT + r, j = token_of(p, row);
      const int64_t at = out0 + (int64_t)j * p.q_heads + row - j * p.group;
      const float inv = L > 0.f || L != L ? 1.f / (L * Mma<T>::kScale) : 0.f;
      if (d < p.head_dim) {
        Pack<T, N> w;
#pragma unroll
        for (int e = 0; e < N; ++e) w.v[e] = Elem<T>::from(v[e] * inv);
        *reinterpret_cast<Pack<T, N>*>(static_cast<T*>(p.out) + at * p.head_dim + d) = w;
      }
      if (d == 0) {
        const float lg = L > 0.f || L != L ? M + log2f(L) : -INFINITY;
        if (p.lse) p.lse[at] = lg * 0.6931471805599453f;
        if (STORE) p.lse2[((int64_t)done.b * p.kv_heads + done.h) * p.rows + row] = lg;
        else if (p.lse2) p.lse2[at] = lg;
      }
    };
    for (int i = tid; i < nrow * (HD / 4); i += 32 * W) {
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
      const int w0 = (r / 16) * WT, rr = r % 16;
      float M = s_m[w0][rr], L = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WT; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(buf + ((w0 + w) * 16 + rr) * HD + (d ^ ((rr & 7) << 3)));
        M = fmaxf(M, s_m[w0 + w][rr]);
        L += s_l[w0 + w][rr];
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
      }
      if (alone) {
        const float vv[4] = {v.x, v.y, v.z, v.w};
        finish(r, d, vv, M, L);
      } else {
        *reinterpret_cast<float4*>(po + r * HD + d) = v;
        if (d == 0) pml[r] = make_float2(M, L);
      }
    }
    if (!alone) {
      consumers_sync<32 * W>();
      if (tid == 0) {  // one acq_rel add publishes this part and orders the last arriver's reads
        unsigned n;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(p.counters + c0) : "memory");
        s_last = n == static_cast<unsigned>(c1 - c0);
        if (s_last) p.counters[c0] = 0u;
      }
      consumers_sync<32 * W>();
      if (s_last) {
        // a warp per row, each lane HD / 32 neighbouring elements
        constexpr int E = HD / 32;
        for (int r = warp; r < nrow; r += W) {
          float M = -INFINITY, L = 0.f, v[E];
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = 0.f;
          constexpr int U = HD == 256 ? 10 : 24;  // parts whose loads are in flight together
          for (int k0 = c0; k0 <= c1; k0 += U) {
            auto part = [&](int k) { return static_cast<size_t>(min(k, c1) * 2 + (k == c0 ? 1 : 0)) * RT + r; };
            float2 ml[2];
            float x[U][E];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const int i = 32 * w + lane;
              ml[w] = i < U && k0 + i <= c1 ? __ldcg(p.part_ml + part(k0 + i)) : make_float2(-INFINITY, 0.f);
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
#pragma unroll
              for (int e = 0; e < E; ++e) x[i][e] = 0.f;
              if (k0 + i <= c1) {
                const float* src = p.part_o + part(k0 + i) * HD + lane * E;
                if constexpr (E == 2) {
                  const float2 y = __ldcg(reinterpret_cast<const float2*>(src));
                  x[i][0] = y.x;
                  x[i][1] = y.y;
                } else {
#pragma unroll
                  for (int e = 0; e < E; e += 4) {
                    const float4 y = __ldcg(reinterpret_cast<const float4*>(src + e));
                    x[i][e] = y.x;
                    x[i][e + 1] = y.y;
                    x[i][e + 2] = y.z;
                    x[i][e + 3] = y.w;
                  }
                }
              }
            }
            float top = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
            for (int q = 16; q; q >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, q));
            top = fmaxf(top, M);
            const float f = exp2_diff(M, top), g[2] = {exp2_diff(ml[0].x, top), exp2_diff(ml[1].x, top)};
            float lg = (ml[0].y == 0.f ? 0.f : ml[0].y * g[0]) + (ml[1].y == 0.f ? 0.f : ml[1].y * g[1]);
#pragma unroll
            for (int q = 16; q; q >>= 1) lg += __shfl_xor_sync(0xffffffffu, lg, q);
            M = top;
            L = L * f + lg;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] *= f;
#pragma unroll
            for (int i = 0; i < U; ++i) {
              const float w = __shfl_sync(0xffffffffu, g[i / 32], i % 32);
#pragma unroll
              for (int e = 0; e < E; ++e) v[e] = fmaf(x[i][e], w, v[e]);
            }
          }
          finish(r, lane * E, v, M, L);
        }
      }
    }
    // the join buffer goes back to the producers
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    consumers_sync<32 * W>();
    if (lane == 0 && phase < kGaveUp) mbar_arrive(&s_empty[stage]);
    t = t_next;
    if (t >= t1) break;
    next_stage();
  }
  block_end_sync<S::THREADS>();
}

// ---------------------------------------------------------------------------
// accumulated weights: scores[b][h][s] += sum over the rows of 2^(s - lse)
//
// The normaliser is known only when a row has met all its slots, so every slot
// is looked at twice.  Few rows leave their scores in the workspace (two
// kernels below, plan_attn has the rule); else the scores are computed again,
// from K and the rows' log-sum-exp: a warp holds the K of its slots in registers
// as the products' second operand and walks the rows, 16 at a time, that see
// any of them.  Either way a slot's sum is made by one warp or thread, so the
// result does not depend on timing.
//
// Measured: 512 tokens of 32 / 8 heads over 8000 slots 823 us, of which 366 are
// the attention; from stored scores 955 us and 580 MB of workspace, where the
// sequence's K and V take 35 MB.
// ---------------------------------------------------------------------------
struct WtShape {
  static constexpr int W = kWtThreads / 32;
  static constexpr int NS = 2;  // blocks of 8 slots per warp (four: 16 % slower, fewer CTAs fit)
  static constexpr int SLOTS = 8 * NS;
  static constexpr int TILE = W * SLOTS;
};

template <class T, int HD>
__global__ void __launch_bounds__(kWtThreads) paged_weights_kernel(const __grid_constant__ AttnParams p) {
  using S = WtShape;
  constexpr int W = S::W, NS = S::NS;
  __shared__ int s_tmp[W + 4];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = lane >> 2, cq = lane & 3;  // as in the attention kernel
  auto tiles = [&](int len) { return (visible(p, len, p.rows - 1) + S::TILE - 1) / S::TILE; };
  int per, t0, t1, b, len, before;
  if (!find_share<W>(p, [&](int n) { return p.kv_heads * tiles(n); }, s_tmp, per, t0, t1, b, len, before)) return;
  int n = tiles(len);
  for (int t = t0; t < t1; ++t) {
    while (t - before >= p.kv_heads * n) {
      before += p.kv_heads * n;
      len = p.lengths[++b];
      n = tiles(len);
    }
    const int h = (t - before) / n, slot0 = ((t - before) - h * n) * S::TILE + warp * S::SLOTS;
    const int rows = p.counts ? max(0, min(p.counts[b], p.tokens)) * p.group : p.rows;
    const int hi = rows ? visible(p, len, rows - 1) : 0;
    if (slot0 >= hi) continue;
    // the slots' K: this lane's row of each block, the chunks of 8 columns as in the attention kernel
    uint4 kf[NS][HD / 32];
    uint32_t got[NS];  // bit 4 i: slot i of the block is there
    bool all = true;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int slot = slot0 + 8 * i + r0;
      const int page = slot < hi ? p.block_table[b * p.table_stride + (slot >> p.lg_page)] : -1;
      const bool ok = page >= 0 && page < p.num_pages;
      got[i] = __ballot_sync(0xffffffffu, ok);
      all = all && got[i] == 0xffffffffu;
      const T* k = static_cast<const T*>(p.k_pages) + (ok ? page * p.page_stride + h * p.head_stride +
                                                                (slot & ((1 << p.lg_page) - 1)) * p.token_stride : 0);
#pragma unroll
      for (int kk = 0; kk < HD / 32; ++kk) {
        const int chunk = (kk >> 1) * 8 + 2 * cq + (kk & 1);
        kf[i][kk] = ok && chunk * 8 < p.head_dim ? *reinterpret_cast<const uint4*>(k + chunk * 8) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
    float* score = p.scores + ((int64_t)b * p.kv_heads + h) * p.capacity + slot0;
    float was[NS][2], sum[NS][2];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = 8 * i + 2 * cq + e;
        was[i][e] = r0 == 0 && slot0 + at < hi ? score[at] : 0.f;
        sum[i][e] = 0.f;
      }
    // rows from the first step token that sees the first slot; sums in two levels
    for (int base = max(0, slot0 - len) * p.group & ~15; base < rows; base += 16 * kWtRound) {
      float part[NS][2];
#pragma unroll
      for (int i = 0; i < NS; ++i) part[i][0] = part[i][1] = 0.f;
      const int end = min(rows, base + 16 * kWtRound);
#pragma unroll 1
      for (int row0 = base; row0 < end; row0 += 16) {
        uint32_t qf[HD / 16][4];
        float z[2];
        int see[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = row0 + r0 + 8 * e, j = token_of(p, row);
          const int64_t at = ((int64_t)b * p.tokens + j) * p.q_heads + h * p.group + row - j * p.group;
          const bool on = row < rows;
          const T* q = static_cast<const T*>(p.q) + at * p.head_dim;
          z[e] = on ? p.lse2[at] * p.lse_unit : 0.f;
          see[e] = on ? visible(p, len, row) : 0;
#pragma unroll
          for (int kk = 0; kk < HD / 32; ++kk) {
            const int chunk = (kk >> 1) * 8 + 2 * cq + (kk & 1);
            const uint4 x = on && chunk * 8 < p.head_dim ? __ldg(reinterpret_cast<const uint4*>(q + chunk * 8))
                                                         : make_uint4(0u, 0u, 0u, 0u);
            qf[2 * kk][e] = x.x;
            qf[2 * kk][2 + e] = x.y;
            qf[2 * kk + 1][e] = x.z;
            qf[2 * kk + 1][2 + e] = x.w;
          }
        }
        float s[NS][4];
#pragma unroll
        for (int i = 0; i < NS; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk) {
#pragma unroll
          for (int i = 0; i < NS; ++i) Mma<T>::run(s[i], qf[2 * kk], kf[i][kk].x, kf[i][kk].y);
#pragma unroll
          for (int i = 0; i < NS; ++i) Mma<T>::run(s[i], qf[2 * kk + 1], kf[i][kk].z, kf[i][kk].w);
        }
        const bool whole = all && row0 + 16 <= rows && slot0 + S::SLOTS <= visible(p, len, row0);
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = 2 * cq + (e & 1);
            const bool seen = whole || (((got[i] >> (4 * col)) & 1u) && slot0 + 8 * i + col < see[e >> 1]);
            if (seen) part[i][e & 1] += exp2_diff(s[i][e] * p.scale_log2, z[e >> 1]);
          }
      }
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        sum[i][0] += part[i][0];
        sum[i][1] += part[i][1];
      }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int m = 4; m < 32; m <<= 1) sum[i][e] += __shfl_xor_sync(0xffffffffu, sum[i][e], m);
        const int at = 8 * i + 2 * cq + e;
        if (r0 == 0 && slot0 + at < hi) score[at] = was[i][e] + sum[i][e];
      }
  }
}

// From the scores that the attention kernel left in the workspace (16 bytes a
// slot and four rows, against head_dim * 2 for reading K again).  Five tokens of
// eight sequences, 7900 slots: 4 us of 24, a chain of round trips (30 us with
// eight rows' loads together, i.e. one round trip more; 28 us in all from K).
template <class S>
__global__ void __launch_bounds__(kWtThreads) paged_stored_weights_kernel(const __grid_constant__ AttnParams p) {
  constexpr int W = kWtThreads / 32, RT = S::RT, TILE = S::TILE;
  __shared__ int s_tmp[W + 4];
  pdl_trigger();
  // The lengths are as old as the attention kernel's own inputs, which it had
  // waited for before it let this one begin.  (All rows are in one row tile.)
  auto count = [&](int len) { return p.kv_heads * item_tiles<S>(p, len, 0); };
  int per, t0, t1, b, len, before;
  if (!find_share<W>(p, count, s_tmp, per, t0, t1, b, len, before)) return;
  int base = before + b * p.kv_heads * kItemCost;  // positions of the attention kernel's index space before sequence b
  int n = item_tiles<S>(p, len, 0);
  pdl_wait();
  const int sub = threadIdx.x / TILE, tok = threadIdx.x % TILE;
  for (int t = t0 + sub; t < t1; t += kWtThreads / TILE) {
    while (t - before >= p.kv_heads * n) {
      before += p.kv_heads * n;
      base += p.kv_heads * (kItemCost + n);
      len = p.lengths[++b];
      n = item_tiles<S>(p, len, 0);
    }
    const int h = (t - before) / n, tile = (t - before) - h * n;
    const int slot = tile * TILE + tok;
    if (slot >= visible(p, len, p.rows - 1)) continue;
    float* score = p.scores + ((int64_t)b * p.kv_heads + h) * p.capacity + slot;
    const float was = *score;
    float w = 0.f;
    const float* s = p.sbuf + (size_t)(base + h * (kItemCost + n) + kItemCost + tile) * RT * TILE + tok;
    const float* z = p.lse2 + ((int64_t)b * p.kv_heads + h) * p.rows;
    const int rows = min(RT, p.rows);  // (all of them; the bound lets the loop go where RT is 16)
    for (int r = 0; r < rows; r += 16) {  // sixteen rows' loads together: one round trip for most calls
      float a[16], m[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int at = min(r + k, rows - 1);
        a[k] = s[at * TILE];
        m[k] = z[at];
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) w += r + k < rows ? exp2_diff(a[k], m[k]) : 0.f;
    }
    *score = was + w;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct PaPlan {
  int hd, mt, tile;
  bool store;  // scores for the accumulated weights go through the workspace
  int64_t max_tiles, positions, ml_off, o_off, lse_off, s_off, bytes;
};

// Sizes of the call's index space and workspace (no device work).
tp_status plan_attn(const tp_paged_cache* c, int tokens, int q_heads, int accumulate, PaPlan* out) {
  if (tokens < 1 || q_heads < 1 || c->kv_heads < 1 || q_heads % c->kv_heads)
    return fail(TP_ERR_ARG, "tp_paged_attn: need tokens >= 1 and q_heads a multiple of kv_heads");
  PaPlan pl{};
  pl.hd = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  const int64_t rows = (int64_t)tokens * (q_heads / c->kv_heads);
  // rows of an item: as few 16-row tiles as hold them, four at most (each item
  // reads the keys and values once)
  pl.mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int64_t rt = 16 * pl.mt, row_tiles = (rows + rt - 1) / rt;
  const int64_t cap = (int64_t)c->max_pages * c->page_size;
  const int64_t items = (int64_t)c->batch * c->kv_heads * row_tiles;
  pl.tile = pl.hd == 256 ? 64 : 128;
  pl.max_tiles = items * std::max<int64_t>(1, (cap + pl.tile - 1) / pl.tile);
  pl.positions = pl.max_tiles + items * kItemCost;
  if (rows > (1 << 24) || items > (1 << 30) || pl.positions > (int64_t(1) << 30))
    return fail(TP_ERR_UNSUPPORTED, "tp_paged_attn: too many rows, sequences or slots");
  int64_t at = kPaCounterBytes;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  pl.ml_off = take((int64_t)kPaMaxCtas * 2 * rt * 8);
  pl.o_off = take((int64_t)kPaMaxCtas * 2 * rt * pl.hd * 4);
  // Stored scores take rt * 4 bytes per slot of the capacity: for up to 32 rows
  // (8000 slots of one sequence 32 us with the attention, 35 us from K; 16
  // sequences, four rows 114 against 171 us; with 64 rows 45 against 38 us), and
  // not where that workspace would grow past 1 GiB.
  const int64_t stored = pl.positions * rt * pl.tile * 4;
  pl.store = accumulate && rows <= 32 && stored <= kPaStoredMax;
  if (accumulate) pl.lse_off = take((int64_t)c->batch * c->kv_heads * rows * 4);
  if (pl.store) pl.s_off = take(stored);
  pl.bytes = at;
  *out = pl;
  return TP_OK;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once.
tp_status encoder(EncodeTiled* out) {
  static void* cached;
  void* fn = __atomic_load_n(&cached, __ATOMIC_ACQUIRE);
  if (!fn) {
    cudaDriverEntryPointQueryResult found;
    TP_CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found),
                "cuTensorMapEncodeTiled");
    if (found != cudaDriverEntryPointSuccess || !fn) return fail(TP_ERR_CUDA, "cuTensorMapEncodeTiled: not in this driver");
    __atomic_store_n(&cached, fn, __ATOMIC_RELEASE);
  }
  *out = reinterpret_cast<EncodeTiled>(fn);
  return TP_OK;
}

// The pages as a tensor of boxes of min(16, page_size) tokens: all of a token's
// 64-element panels where they are whole and a box has 16 tokens (it is then
// the block's layout in shared memory), else one panel, zero-filled past
// head_dim.
tp_status page_map(const tp_paged_cache* c, void* base, bool panels, int box, CUtensorMap* map) {
  EncodeTiled encode;
  const tp_status s = encoder(&encode);
  if (s != TP_OK) return s;
  const auto u64 = [](int64_t v) { return static_cast<cuuint64_t>(v); };
  const cuuint32_t np = panels ? static_cast<cuuint32_t>(c->head_dim / 64) : 1u;
  const cuuint64_t dims[5] = {panels ? u64(64) : u64(c->head_dim), u64(c->page_size), np, u64(c->kv_heads),
                              u64(std::max<int64_t>(1, c->num_pages))};
  const cuuint64_t strides[4] = {u64(c->token_stride * 2), 128, u64(c->head_stride * 2), u64(c->page_stride * 2)};
  const cuuint32_t boxes[5] = {64u, static_cast<cuuint32_t>(box), np, 1u, 1u};
  const cuuint32_t ones[5] = {1u, 1u, 1u, 1u, 1u};
  const CUresult r = encode(map, c->dtype == TP_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                            base, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(TP_ERR_UNSUPPORTED, "tp_paged_attn: the pages' sizes and strides make no tensor map (error %d)", (int)r);
  return TP_OK;
}

template <class T, int HD>
tp_status launch_weights(const AttnParams& p, cudaStream_t st) {
  int sms = 0;
  const tp_status s = device_sms(&sms);
  if (s != TP_OK) return s;
  const int64_t tiles = (int64_t)p.batch * p.kv_heads * ((p.capacity + WtShape::TILE - 1) / WtShape::TILE);
  return launch_early(paged_weights_kernel<T, HD>, dim3(static_cast<unsigned>(std::min<int64_t>(8 * sms, tiles))), kWtThreads, 0,
                      st, "paged_weights launch", p);
}

template <class T, int HD, int MT, bool STORE>
tp_status launch_attn(const AttnParams& p, const PaPlan& pl, cudaStream_t st) {
  using S = PaShape<HD, MT>;
  static_assert(S::TILE == (HD == 256 ? 64 : 128), "as plan_attn");
  const auto kern = paged_attn_kernel<T, HD, MT, STORE>;
  static int smem_set[64];
  static int ctas[64];  // resident CTAs per SM
  tp_status s = ensure_smem(kern, S::kSmem, smem_set, "paged_attn: shared memory attribute");
  if (s != TP_OK) return s;
  int sms = 0, dev = 0;
  s = device_sms(&sms);
  if (s != TP_OK) return s;
  TP_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
  int occ = __atomic_load_n(&ctas[dev], __ATOMIC_RELAXED);
  if (!occ) {
    TP_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, S::THREADS, S::kSmem), "paged_attn: occupancy");
    if (occ < 1) return fail(TP_ERR_CUDA, "paged_attn: the kernel does not fit this device");
    __atomic_store_n(&ctas[dev], occ, __ATOMIC_RELAXED);
  }
  const int grid = static_cast<int>(std::min<int64_t>(std::min(kPaMaxCtas, sms * occ), pl.positions));
  s = launch_early(kern, dim3(grid), S::THREADS, S::kSmem, st, "paged_attn launch", p);
  if (s != TP_OK || !p.lse2) return s;
  if constexpr (STORE)
    return launch_early(paged_stored_weights_kernel<S>, dim3(static_cast<unsigned>(std::min<int64_t>(8 * sms, pl.max_tiles))),
                        kWtThreads, 0, st, "paged_stored_weights launch", p);
  else
    return launch_weights<T, HD>(p, st);
}

template <class T, int HD>
tp_status dispatch_rows(const AttnParams& p, const PaPlan& pl, cudaStream_t st) {
  if (pl.mt == 1) return pl.store ? launch_attn<T, HD, 1, true>(p, pl, st) : launch_attn<T, HD, 1, false>(p, pl, st);
  if (pl.mt == 2) return pl.store ? launch_attn<T, HD, 2, true>(p, pl, st) : launch_attn<T, HD, 2, false>(p, pl, st);
  return launch_attn<T, HD, 4, false>(p, pl, st);
}

template <class T>
tp_status dispatch_dim(const AttnParams& p, const PaPlan& pl, cudaStream_t st) {
  if (pl.hd == 64) return dispatch_rows<T, 64>(p, pl, st);
  if (pl.hd == 128) return dispatch_rows<T, 128>(p, pl, st);
  return dispatch_rows<T, 256>(p, pl, st);
}

// What both launches need of a call.
void fill_params(const tp_paged_cache* c, int tokens, int q_heads, float scale, AttnParams* p) {
  p->block_table = c->block_table;
  p->lengths = c->lengths;
  p->scores = c->scores;
  p->num_pages = c->num_pages;
  p->table_stride = c->table_stride;
  p->batch = c->batch;
  p->tokens = tokens;
  p->q_heads = q_heads;
  p->kv_heads = c->kv_heads;
  p->group = q_heads / c->kv_heads;
  p->head_dim = c->head_dim;
  p->lg_page = log2_int(c->page_size);
  p->capacity = c->max_pages * c->page_size;
  p->group_inv = p->group == 1 ? 0 : ~uint64_t(0) / p->group + 1;
  p->rows = tokens * p->group;
  p->scale_log2 = scale * 1.4426950408889634f;
  p->lse_unit = 1.f;
  p->k_pages = c->k_pages;
  p->page_stride = c->page_stride;
  p->head_stride = c->head_stride;
  p->token_stride = c->token_stride;
}

}  // namespace

extern "C" {

TP_API int64_t tp_paged_attn_workspace_bytes(const tp_paged_cache* cache, int tokens, int q_heads, int accumulate) {
  PaPlan pl;
  tp_status s = check_cache(cache, "tp_paged_attn_workspace_bytes");
  if (s == TP_OK) s = plan_attn(cache, tokens, q_heads, accumulate, &pl);
  return s == TP_OK ? pl.bytes : -static_cast<int64_t>(s);
}

TP_API tp_status tp_paged_attn(const tp_paged_attn_args* args, const tp_paged_cache* cache, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  if (!args || !args->q || !args->out) return fail(TP_ERR_ARG, "tp_paged_attn: null pointer");
  const tp_paged_attn_args& a = *args;
  tp_status s = check_cache(cache, "tp_paged_attn");
  if (s != TP_OK) return s;
  PaPlan pl;
  s = plan_attn(cache, a.tokens, a.q_heads, a.accumulate, &pl);
  if (s != TP_OK) return s;
  if (a.accumulate && !cache->scores) return fail(TP_ERR_ARG, "tp_paged_attn: the cache has no scores to accumulate in");
  if (a.wait_polls < 0 || a.wait_hold < 0 || (a.wait_hold && !a.wait_polls))
    return fail(TP_ERR_ARG, "tp_paged_attn: bad wait limit (a held wait needs one of its own)");
  if (!aligned(a.q, 16) || !aligned(a.out, 16))
    return fail(TP_ERR_ALIGN, "tp_paged_attn: q and out must be 16-byte aligned");
  if (!workspace || workspace_bytes < pl.bytes || !aligned(workspace, 256))
    return fail(TP_ERR_WORKSPACE, "tp_paged_attn: workspace missing, not 256-byte aligned or smaller than %lld bytes",
                (long long)pl.bytes);
  AttnParams p{};
  const int box = std::min(16, cache->page_size);
  p.lg_box = log2_int(box);
  p.panels = box == 16 && cache->head_dim == pl.hd;
  s = page_map(cache, cache->k_pages, p.panels, box, &p.k_map);
  if (s == TP_OK) s = page_map(cache, cache->v_pages, p.panels, box, &p.v_map);
  if (s != TP_OK) return s;
  fill_params(cache, a.tokens, a.q_heads, a.softmax_scale, &p);
  p.q = a.q;
  p.out = a.out;
  p.lse = a.lse;
  p.row_tiles = (p.rows + 16 * pl.mt - 1) / (16 * pl.mt);
  auto* ws = static_cast<unsigned char*>(workspace);
  p.counters = reinterpret_cast<unsigned*>(ws);
  p.status = reinterpret_cast<unsigned*>(ws + kPaStatusOff);
  p.polls = a.wait_polls > 0 ? static_cast<unsigned>(a.wait_polls) : kMaxPolls;
  p.hold = a.wait_hold;
  p.part_ml = reinterpret_cast<float2*>(ws + pl.ml_off);
  p.part_o = reinterpret_cast<float*>(ws + pl.o_off);
  if (a.accumulate) p.lse2 = reinterpret_cast<float*>(ws + pl.lse_off);
  if (pl.store) p.sbuf = reinterpret_cast<float*>(ws + pl.s_off);
  cudaStream_t st = as_stream(stream);
  return cache->dtype == TP_F16 ? dispatch_dim<__half>(p, pl, st) : dispatch_dim<__nv_bfloat16>(p, pl, st);
}

TP_API tp_status tp_paged_weights(const tp_paged_weights_args* args, const tp_paged_cache* cache, void* stream) {
  if (!args || !args->q || !args->lse) return fail(TP_ERR_ARG, "tp_paged_weights: null pointer");
  const tp_paged_weights_args& a = *args;
  tp_status s = check_cache(cache, "tp_paged_weights");
  if (s != TP_OK) return s;
  PaPlan pl;
  s = plan_attn(cache, a.tokens, a.q_heads, 1, &pl);
  if (s != TP_OK) return s;
  if (!cache->scores) return fail(TP_ERR_ARG, "tp_paged_weights: the cache has no scores to accumulate in");
  if (!aligned(a.q, 16)) return fail(TP_ERR_ALIGN, "tp_paged_weights: q must be 16-byte aligned");
  AttnParams p{};
  fill_params(cache, a.tokens, a.q_heads, a.softmax_scale, &p);
  p.q = a.q;
  p.lse2 = const_cast<float*>(a.lse);  // (only read)
  p.lse_unit = 1.4426950408889634f;
  p.counts = a.counts;
  cudaStream_t st = as_stream(stream);
  const auto launch = [&](auto t) {
    using T = decltype(t);
    return pl.hd == 64 ? launch_weights<T, 64>(p, st) : pl.hd == 128 ? launch_weights<T, 128>(p, st) : launch_weights<T, 256>(p, st);
  };
  return cache->dtype == TP_F16 ? launch(__half{}) : launch(__nv_bfloat16{});
}

TP_API tp_status tp_paged_attn_status(void* workspace, void* stream) {
  if (!workspace) return fail(TP_ERR_ARG, "tp_paged_attn_status: null workspace");
  auto* word = reinterpret_cast<unsigned*>(static_cast<unsigned char*>(workspace) + kPaStatusOff);
  cudaStream_t st = as_stream(stream);
  unsigned v = 0;
  TP_CUDA_TRY(cudaMemcpyAsync(&v, word, 4, cudaMemcpyDeviceToHost, st), "status copy");
  TP_CUDA_TRY(cudaStreamSynchronize(st), "status sync");
  if (!v) return clear_ok();
  TP_CUDA_TRY(cudaMemsetAsync(word, 0, 4, st), "status clear");
  return fail(TP_ERR_DEVICE, "tp_paged_attn: a bounded device wait ran out, outputs are NaN (status %u)", v);
}

}  // extern "C"
