// Eviction from a paged cache by accumulated attention weight.
//
// Mathematics: the `budget` largest of n keys per (sequence, kv head), a key
// being the score's order-preserving 32-bit image (guarded slots above all,
// the lower slot first on equality).  A radix selection finds the budget-th
// key in three counting passes over 11, 11 and 10 bits; one ordered pass over
// bit words (a thread per 32 slots) marks the kept slots.  With the kept slots above the budget s_0 < s_1 < ... and the
// freed ones below it h_0 < h_1 < ..., slot s_i moves to h_i: as many rows as
// must move, every source at or above the budget and every destination below
// it, so the moves are independent of each other.
//
// Bound: the moves, 4 * head_dim bytes read and as many written per row, for
// many of them; the chain of passes of one CTA for few.  The selection reads a
// slot's 8 bytes once and keeps the keys in shared memory (up to 40960 slots;
// above, it forms them again in each pass).  Few rows are moved by the CTA
// that selected them; many by a second launch over the whole GPU.
//
// Measured (B200, whole calls): 64 of 1088 slots in each of 64 heads 8.0 us;
// 16 sequences of up to 16384 slots cut to 2048 35 us, of which the longest
// heads' selection about 20 (the passes' barriers and collisions) and the moves
// 14 (86 MB, 6 TB/s).  A cluster of CTAs per head that adds its counts up
// through distributed shared memory was slower (65 us).
#include <algorithm>

#include "tp_decode.cuh"
#include "tp_paged.cuh"

using namespace tp;

namespace {

constexpr int kEvMaxSlots = 1 << 19;
constexpr int kEvCached = 40960;   // slots whose keys fit in shared memory
constexpr int kEvBins = 2048;
// Threads of the selection: few where few slots are (its barriers cost less).
// Eight sequences of 1088 slots take 7.9 us with 256, 8.8 us with 1024; of 2000
// slots 9.7 against 10.1 us.
constexpr int kEvSmall = 2048;      // capacity up to which 256 threads do
constexpr int kMvThreads = 256;
// Rows in flight per group of lanes: four where one CTA moves its own few (one
// round for 64), two in the launch over the GPU (more CTAs instead).
constexpr int kMvOwn = 4, kMvRows = 2;
// Moves per head up to which the selecting CTA does them itself: 64 moves in
// each of 64 heads take 7.9 us in all so and 11.6 us with the second launch,
// 256 moves 10.3 against 14.6 us, 512 the same in both.
constexpr int kMvFused = 256;

struct EvictParams {
  tp_evict_args a;
  unsigned char* k_pages;
  unsigned char* v_pages;
  const int32_t* block_table;
  const int32_t* lengths;
  const float* scores;
  const int32_t* positions;
  int64_t num_pages, page_stride, head_stride, token_stride, table_stride;
  int batch, kv_heads, head_dim, lg_page, capacity;
  int max_moves;   // per (sequence, kv head)
  int* moved;      // [batch][kv_heads]
  longlong2* moves;  // [batch][kv_heads][max_moves]: element offsets (from, to) in the pages, -1 where a page is missing
  int lg_lanes;      // lanes per row
  int cached;        // keys in shared memory
  int fused;         // moves by the selecting CTA
  int vectors;       // rows of scores and positions are 16-byte aligned
};

__device__ __forceinline__ uint32_t slot_key(const EvictParams& p, float v, int at, int64_t next) {
  if (at < p.a.sinks || at >= next - p.a.recent) return 0xFFFFFFFFu;
  if (v != v) return 0xFFFFFFFEu;
  if (v == 0.f) v = 0.f;  // -0 equals 0
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sums over the block of N values per thread, and the sums.
template <int N, int WARPS>
__device__ __forceinline__ void block_prefix(const uint32_t (&v)[N], uint32_t (*s_tmp)[32], uint32_t (&before)[N],
                                             uint32_t (&all)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) inc[k] = v[k];
#pragma unroll
  for (int m = 1; m < 32; m <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, inc[k], m);
      if (lane >= m) inc[k] += o;
    }
  __syncthreads();
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < N; ++k) s_tmp[k][warp] = inc[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t x = lane < WARPS ? s_tmp[k][lane] : 0u;
    all[k] = __reduce_add_sync(0xffffffffu, x);
    before[k] = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0u) + inc[k] - v[k];
  }
}

// Moves rows [first, n) step by step: K and V of a slot by a group of lanes,
// R rows in flight.
template <int R>
__device__ __forceinline__ void move_rows(const EvictParams& p, const longlong2* moves, int n, int first, int step, int chunk) {
  if (chunk * 8 >= p.head_dim) return;
  for (int i0 = first; i0 < n; i0 += R * step) {
    longlong2 m[R];
    uint4 kv[R], vv[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int i = i0 + u * step;
      m[u] = i < n ? moves[i] : make_longlong2(-1, -1);
    }
#pragma unroll
    for (int u = 0; u < R; ++u)
      if (m[u].x >= 0 && m[u].y >= 0) {
        kv[u] = *reinterpret_cast<const uint4*>(p.k_pages + 2 * (m[u].x + chunk * 8));
        vv[u] = *reinterpret_cast<const uint4*>(p.v_pages + 2 * (m[u].x + chunk * 8));
      }
#pragma unroll
    for (int u = 0; u < R; ++u)
      if (m[u].x >= 0 && m[u].y >= 0) {
        *reinterpret_cast<uint4*>(p.k_pages + 2 * (m[u].y + chunk * 8)) = kv[u];
        *reinterpret_cast<uint4*>(p.v_pages + 2 * (m[u].y + chunk * 8)) = vv[u];
      }
  }
}

// COPIES: of the histogram, against collisions.
template <int THREADS, int COPIES>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const __grid_constant__ EvictParams p) {
  constexpr int WARPS = THREADS / 32, D = kEvBins / THREADS;  // D: digits per thread
  extern __shared__ __align__(16) uint32_t s_dyn[];
  uint32_t* hist = s_dyn;                              // [copies][bins]; then the (to, from) slots of fused moves
  uint32_t* kept = s_dyn + COPIES * kEvBins;           // a bit per slot: key above the threshold
  uint32_t* level = kept + (p.capacity + 31) / 32;     // a bit per slot: key equal to it
  uint32_t* keys = level + (p.capacity + 31) / 32;     // [capacity] where cached
  __shared__ uint32_t s_sum[2][32];
  __shared__ uint32_t s_pick[2];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, h = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t bh = (int64_t)b * p.kv_heads + h;
  const float* sc = p.scores + bh * p.capacity;
  const int32_t* pos = p.positions + bh * p.capacity;
  float* nsc = p.a.new_scores + bh * p.capacity;
  int32_t* npos = p.a.new_positions + bh * p.capacity;
  const int len = p.lengths[b], budget = p.a.budget;
  const int64_t next = p.a.next_pos[b];
  const int n = max(0, min(len, p.capacity)), live = min(n, budget);
  if (h == 0 && tid == 0) p.a.new_lengths[b] = min(len, min(budget, p.capacity));
  // f(i, score, position) for this thread's slots below `end`, four
  // neighbouring ones at a time where rows of the arrays are 16-byte aligned
  auto each_slot = [&](int end, auto f) {
    constexpr int U = 2;  // groups of four whose loads are in flight together
    if (p.vectors) {
      for (int i0 = 4 * tid; i0 < end; i0 += 4 * U * THREADS) {
        float4 v[U];
        int4 at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = min(i0 + 4 * u * THREADS, (end - 1) & ~3);  // (within the capacity, a multiple of four)
          v[u] = *reinterpret_cast<const float4*>(sc + i);
          at[u] = *reinterpret_cast<const int4*>(pos + i);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + 4 * u * THREADS;
          if (i < end) f(i, v[u].x, at[u].x);
          if (i + 1 < end) f(i + 1, v[u].y, at[u].y);
          if (i + 2 < end) f(i + 2, v[u].z, at[u].z);
          if (i + 3 < end) f(i + 3, v[u].w, at[u].w);
        }
      }
    } else {
      constexpr int S = 4 * U;
      for (int i0 = tid; i0 < end; i0 += S * THREADS) {
        float v[S];
        int at[S];
#pragma unroll
        for (int u = 0; u < S; ++u) {
          const int i = min(i0 + u * THREADS, end - 1);
          v[u] = sc[i];
          at[u] = pos[i];
        }
#pragma unroll
        for (int u = 0; u < S; ++u)
          if (i0 + u * THREADS < end) f(i0 + u * THREADS, v[u], at[u]);
      }
    }
  };
  auto copy = [&] {  // the kept range as it was (freed slots are overwritten later), zeros past it
    int first = live;  // of the zeros
    if (p.vectors) {
      first = (live + 3) & ~3;
      for (int i = first + 4 * tid; i < p.capacity; i += 4 * THREADS) {
        *reinterpret_cast<float4*>(nsc + i) = make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<int4*>(npos + i) = make_int4(-1, -1, -1, -1);
      }
      if (tid < first - live) {
        nsc[live + tid] = 0.f;
        npos[live + tid] = -1;
      }
    } else {
      for (int i = first + tid; i < p.capacity; i += THREADS) {
        nsc[i] = 0.f;
        npos[i] = -1;
      }
    }
    each_slot(live, [&](int i, float v, int at) {
      nsc[i] = v;
      npos[i] = at;
    });
  };
  if (n <= budget) {
    copy();
    if (tid == 0) p.moved[bh] = 0;
    return;
  }
  if (p.cached) each_slot(n, [&](int i, float v, int at) { keys[i] = slot_key(p, v, at, next); });
  auto key = [&](int i) { return p.cached ? keys[i] : slot_key(p, sc[i], pos[i], next); };

  // ---- the budget-th largest key: digits of 11, 11 and 10 bits ----
  // (a digit's count lies where the threads that sum D digits each meet no bank twice)
  auto place = [](uint32_t digit) { return digit % D * THREADS + digit / D; };
  uint32_t prefix = 0, want = budget;  // keys that match `prefix` above the digit hold the want-th largest
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < COPIES * kEvBins; i += THREADS) hist[i] = 0;
    __syncthreads();
    uint32_t* mine = hist + (warp % COPIES) * kEvBins;
    auto count = [&](uint32_t k) {
      if (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits))) atomicAdd(&mine[place((k >> shift) & ((1u << bits) - 1))], 1u);
    };
    if (p.cached) {
#pragma unroll 4
      for (int i = tid; i < n; i += THREADS) count(keys[i]);
    } else {
      each_slot(n, [&](int, float v, int at) { count(slot_key(p, v, at, next)); });
    }
    __syncthreads();
    // thread t holds D digits down from kEvBins - 1 - D t
    uint32_t own[D], sum[1] = {0}, pre[1], all[1];
#pragma unroll
    for (int e = 0; e < D; ++e) {
      own[e] = 0;
#pragma unroll
      for (int w = 0; w < COPIES; ++w) own[e] += hist[w * kEvBins + place(kEvBins - 1 - D * tid - e)];
      sum[0] += own[e];
    }
    block_prefix<1, WARPS>(sum, s_sum, pre, all);
    uint32_t above = pre[0];
    if (above < want && want <= above + sum[0]) {
#pragma unroll
      for (int e = 0; e < D; ++e) {
        if (above < want && want <= above + own[e]) {
          s_pick[0] = kEvBins - 1 - D * tid - e;
          s_pick[1] = want - above;
        }
        above += own[e];
      }
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    want = s_pick[1];
  }
  // keys above `prefix` are kept, and of those equal to it the first `want`

  const int words = (n + 31) / 32;
#pragma unroll 4
  for (int w = warp; w < words; w += WARPS) {
    const int i = w * 32 + lane;
    const uint32_t k = key(min(i, n - 1));
    const uint32_t gt = __ballot_sync(0xffffffffu, i < n && k > prefix), eq = __ballot_sync(0xffffffffu, i < n && k == prefix);
    if (lane == 0) {
      kept[w] = gt;
      level[w] = eq;
    }
  }
  __syncthreads();
  // the slots of move m: in the shared memory of the counts where few, else in
  // the words of its entry of the list
  longlong2* mv = p.moves + bh * p.max_moves;
  int2* pairs = reinterpret_cast<int2*>(hist);
  uint32_t equal = 0, moves = 0, freed = 0;  // equal keys, late slots and holes in the words before
  for (int c0 = 0; c0 < words; c0 += THREADS) {  // a word per thread
    const int w = c0 + tid;
    uint32_t word = w < words ? kept[w] : 0, eq = w < words ? level[w] : 0;
    uint32_t c[1] = {static_cast<uint32_t>(__popc(eq))}, at[1], all[1];
    block_prefix<1, WARPS>(c, s_sum, at, all);
    at[0] += equal;
    equal += all[0];
    int take = at[0] >= want ? 0 : static_cast<int>(min(want - at[0], c[0]));
    if (take == (int)c[0]) {
      word |= eq;
    } else {
      for (; take > 0; --take, eq &= eq - 1) word |= eq & (0u - eq);
    }
    const int below = budget - w * 32;  // of the word's slots, those under the budget
    const uint32_t low = below >= 32 ? 0xffffffffu : below <= 0 ? 0u : (1u << below) - 1;
    uint32_t holes = ~word & low, late = word & ~low;  // (the budget is below n: every hole is a slot)
    uint32_t two[2] = {static_cast<uint32_t>(__popc(holes)), static_cast<uint32_t>(__popc(late))}, from[2], sum[2];
    block_prefix<2, WARPS>(two, s_sum, from, sum);
    for (uint32_t m = freed + from[0]; holes; holes &= holes - 1, ++m) {
      const int i = w * 32 + __ffs(holes) - 1;
      if (p.fused) pairs[m].y = i;
      else mv[m].y = i;
    }
    for (uint32_t m = moves + from[1]; late; late &= late - 1, ++m) {
      const int i = w * 32 + __ffs(late) - 1;
      if (p.fused) pairs[m].x = i;
      else mv[m].x = i;
    }
    freed += sum[0];
    moves += sum[1];
  }
  copy();
  __syncthreads();
  // ---- the moved slots' entries, and where their rows lie ----
  const int32_t* table = p.block_table + b * p.table_stride;
  const int mask = (1 << p.lg_page) - 1;
  auto offset = [&](int slot) -> long long {
    const int page = table[slot >> p.lg_page];
    if (page < 0 || page >= p.num_pages) return -1;
    return page * p.page_stride + h * p.head_stride + (slot & mask) * p.token_stride;
  };
  longlong2* list = p.fused ? reinterpret_cast<longlong2*>(hist) + kMvFused : mv;  // (past the pairs)
  constexpr int M = 2;  // moves whose loads are in flight together
  for (int i0 = tid; i0 < (int)moves; i0 += M * THREADS) {
    int2 m[M];
    float v[M];
    int at[M];
    longlong2 rows[M];
#pragma unroll
    for (int u = 0; u < M; ++u) {
      const int i = i0 + u * THREADS;  // (an entry is read and replaced by one thread)
      m[u] = i >= (int)moves ? make_int2(0, 0)
             : p.fused       ? pairs[i]
                             : make_int2(static_cast<int>(mv[i].x), static_cast<int>(mv[i].y));
    }
#pragma unroll
    for (int u = 0; u < M; ++u) {
      v[u] = sc[m[u].x];
      at[u] = pos[m[u].x];
      rows[u] = make_longlong2(offset(m[u].x), offset(m[u].y));
    }
#pragma unroll
    for (int u = 0; u < M; ++u)
      if (i0 + u * THREADS < (int)moves) {
        nsc[m[u].y] = v[u];
        npos[m[u].y] = at[u];
        list[i0 + u * THREADS] = rows[u];
      }
  }
  if (!p.fused) {
    if (tid == 0) p.moved[bh] = static_cast<int>(moves);
    return;
  }
  __syncthreads();
  move_rows<kMvOwn>(p, list, moves, tid >> p.lg_lanes, THREADS >> p.lg_lanes, tid & ((1 << p.lg_lanes) - 1));
}

template <int THREADS, int COPIES>
tp_status launch_select(const EvictParams& p, cudaStream_t st) {
  const int smem = (COPIES * kEvBins + 2 * ((p.capacity + 31) / 32) + (p.cached ? p.capacity : 0)) * 4;
  static int smem_set[64];
  // (the default dynamic limit is 48 KB less the static shared memory)
  const tp_status s = ensure_smem(evict_select_kernel<THREADS, COPIES>, smem > 47 * 1024 ? smem + 1024 : smem, smem_set,
                                  "evict: shared memory attribute");
  if (s != TP_OK) return s;
  return launch_early(evict_select_kernel<THREADS, COPIES>, dim3(p.kv_heads, p.batch), THREADS, smem, st,
                      "evict_select launch", p);
}

__global__ void __launch_bounds__(kMvThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t bh = blockIdx.y;
  const int rows = kMvThreads >> p.lg_lanes;
  move_rows<kMvRows>(p, p.moves + bh * p.max_moves, p.moved[bh], blockIdx.x * rows + (threadIdx.x >> p.lg_lanes), gridDim.x * rows,
            threadIdx.x & ((1 << p.lg_lanes) - 1));
}

int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

tp_status plan_evict(const tp_paged_cache* c, int64_t budget, const char* who, int64_t* max_moves, int64_t* bytes) {
  const tp_status s = check_cache(c, who);
  if (s != TP_OK) return s;
  if (budget < 1) return fail(TP_ERR_ARG, "%s: budget must be positive", who);
  const int64_t cap = (int64_t)c->max_pages * c->page_size;
  if (cap > kEvMaxSlots) return fail(TP_ERR_UNSUPPORTED, "%s: more than %d slots per sequence", who, kEvMaxSlots);
  const int64_t heads = (int64_t)c->batch * c->kv_heads;
  if (c->kv_heads > 65535 || c->batch > 65535 || heads > 65535)
    return fail(TP_ERR_UNSUPPORTED, "%s: more than 65535 sequences times kv heads", who);
  *max_moves = std::max<int64_t>(0, std::min(budget, cap - budget));
  *bytes = round256(heads * 4) + round256(heads * *max_moves * (int64_t)sizeof(longlong2));
  return TP_OK;
}

}  // namespace

extern "C" {

TP_API int64_t tp_cache_evict_workspace_bytes(const tp_paged_cache* cache, int budget) {
  int64_t moves, bytes;
  const tp_status s = plan_evict(cache, budget, "tp_cache_evict_workspace_bytes", &moves, &bytes);
  return s == TP_OK ? bytes : -static_cast<int64_t>(s);
}

TP_API tp_status tp_cache_evict(const tp_evict_args* args, const tp_paged_cache* cache, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (!args) return fail(TP_ERR_ARG, "tp_cache_evict: null arguments");
  const tp_evict_args& a = *args;
  int64_t max_moves, bytes;
  tp_status s = plan_evict(cache, a.budget, "tp_cache_evict", &max_moves, &bytes);
  if (s != TP_OK) return s;
  if (!cache->scores || !cache->positions || !a.next_pos || !a.new_lengths || !a.new_scores || !a.new_positions)
    return fail(TP_ERR_ARG, "tp_cache_evict: null pointer");
  if (a.recent < 0 || a.sinks < 0 || (int64_t)a.recent + a.sinks > a.budget)
    return fail(TP_ERR_ARG, "tp_cache_evict: recent and sinks must be >= 0 and fit in the budget");
  if (a.new_scores == cache->scores || a.new_positions == cache->positions)
    return fail(TP_ERR_ARG, "tp_cache_evict: the new scores and positions need buffers of their own");
  if (!workspace || workspace_bytes < bytes || !aligned(workspace, 256))
    return fail(TP_ERR_WORKSPACE, "tp_cache_evict: workspace missing, not 256-byte aligned or smaller than %lld bytes",
                (long long)bytes);
  EvictParams p{};
  p.a = a;
  p.k_pages = static_cast<unsigned char*>(cache->k_pages);
  p.v_pages = static_cast<unsigned char*>(cache->v_pages);
  p.block_table = cache->block_table;
  p.lengths = cache->lengths;
  p.scores = cache->scores;
  p.positions = cache->positions;
  p.num_pages = cache->num_pages;
  p.page_stride = cache->page_stride;
  p.head_stride = cache->head_stride;
  p.token_stride = cache->token_stride;
  p.table_stride = cache->table_stride;
  p.batch = cache->batch;
  p.kv_heads = cache->kv_heads;
  p.head_dim = cache->head_dim;
  p.lg_page = log2_int(cache->page_size);
  p.capacity = cache->max_pages * cache->page_size;
  p.max_moves = static_cast<int>(max_moves);
  auto* ws = static_cast<unsigned char*>(workspace);
  const int heads = cache->batch * cache->kv_heads;
  p.moved = reinterpret_cast<int*>(ws);
  p.moves = reinterpret_cast<longlong2*>(ws + round256((int64_t)heads * 4));
  cudaStream_t st = as_stream(stream);
  p.lg_lanes = log2_int((cache->head_dim + 7) / 8);
  p.cached = p.capacity <= kEvCached;
  p.vectors = p.capacity % 4 == 0 && aligned(p.scores, 16) && aligned(p.positions, 16) && aligned(a.new_scores, 16) &&
              aligned(a.new_positions, 16);
  p.fused = max_moves <= kMvFused;
  s = p.capacity <= kEvSmall ? launch_select<256, 2>(p, st) : launch_select<1024, 4>(p, st);
  if (s != TP_OK || p.fused) return s;
  int sms = 0;
  s = device_sms(&sms);
  if (s != TP_OK) return s;
  // about 32 CTAs per SM in all (many end at once: their heads move little), never
  // more than the rows that may move; with 8 and four rows in flight 7 % slower
  const int rows = (kMvThreads >> p.lg_lanes) * kMvRows;
  const int64_t per_head = std::max<int64_t>(1, std::min<int64_t>((max_moves + rows - 1) / rows, (32 * sms + heads - 1) / heads));
  return launch_early(evict_move_kernel, dim3(static_cast<unsigned>(per_head), heads), kMvThreads, 0, st, "evict_move launch", p);
}

}  // extern "C"
