// Eviction from a paged cache by accumulated attention weight.
//
// Mathematics: the `budget` largest of n keys per (sequence, kv head), a key
// being the score's order-preserving 32-bit image (guarded slots above all,
// the lower slot first on equality).  A radix selection finds the budget-th
// key in three counting passes over 11, 11 and 10 bits; one ordered pass marks
// the kept slots.  With the kept slots above the budget s_0 < s_1 < ... and the
// freed ones below it h_0 < h_1 < ..., slot s_i moves to h_i: as many rows as
// must move, every source at or above the budget and every destination below
// it, so the moves are independent of each other.
//
// Bound: the moves, 4 * head_dim bytes read and as many written per row, for
// many of them; the chain of passes of one CTA for few.  The selection reads a
// slot's 8 bytes once and keeps the keys in shared memory (up to 40960 slots;
// above, it forms them again in each pass).  Few rows are moved by the CTA
// that selected them; many by a second launch over the whole GPU.
#include <algorithm>

#include "tp_decode.cuh"
#include "tp_paged.cuh"

using namespace tp;

namespace {

constexpr int kEvThreads = 1024;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvMaxSlots = 1 << 20;
constexpr int kEvCached = 40960;   // slots whose keys fit in shared memory
constexpr int kEvBins = 2048;
constexpr int kEvCopies = 4;        // of the histogram: fewer collisions
constexpr int kMvThreads = 256;
constexpr int kMvRows = 4;          // rows in flight per group of lanes
// Moves per head up to which the selecting CTA does them itself.  EVNOTE
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
};

__device__ __forceinline__ uint32_t slot_key(const EvictParams& p, float v, int at, int next) {
  if (at < p.a.sinks || at >= next - p.a.recent) return 0xFFFFFFFFu;
  if (v != v) return 0xFFFFFFFEu;
  if (v == 0.f) v = 0.f;  // -0 equals 0
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum of one value per warp (call with the value in every
// lane); returns this warp's prefix.
__device__ __forceinline__ int warps_prefix(int v, int* s_tmp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) s_tmp[warp] = v;
  __syncthreads();
  int x = lane < warp ? s_tmp[lane] : 0;
#pragma unroll
  for (int m = 16; m; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

// Moves rows [first, n) step by step: K and V of a slot by a group of lanes,
// kMvRows rows in flight.
__device__ __forceinline__ void move_rows(const EvictParams& p, const longlong2* moves, int n, int first, int step, int chunk) {
  if (chunk * 8 >= p.head_dim) return;
  for (int i0 = first; i0 < n; i0 += kMvRows * step) {
    longlong2 m[kMvRows];
    uint4 kv[kMvRows], vv[kMvRows];
#pragma unroll
    for (int u = 0; u < kMvRows; ++u) {
      const int i = i0 + u * step;
      m[u] = i < n ? moves[i] : make_longlong2(-1, -1);
    }
#pragma unroll
    for (int u = 0; u < kMvRows; ++u)
      if (m[u].x >= 0 && m[u].y >= 0) {
        kv[u] = *reinterpret_cast<const uint4*>(p.k_pages + 2 * (m[u].x + chunk * 8));
        vv[u] = *reinterpret_cast<const uint4*>(p.v_pages + 2 * (m[u].x + chunk * 8));
      }
#pragma unroll
    for (int u = 0; u < kMvRows; ++u)
      if (m[u].x >= 0 && m[u].y >= 0) {
        *reinterpret_cast<uint4*>(p.k_pages + 2 * (m[u].y + chunk * 8)) = kv[u];
        *reinterpret_cast<uint4*>(p.v_pages + 2 * (m[u].y + chunk * 8)) = vv[u];
      }
  }
}

__global__ void __launch_bounds__(kEvThreads, 1) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t s_dyn[];
  uint32_t* hist = s_dyn;                              // [copies][bins]; then the (to, from) slots of fused moves
  uint32_t* kept = s_dyn + kEvCopies * kEvBins;        // a bit per slot
  uint32_t* keys = kept + (p.capacity + 31) / 32;      // [capacity] where cached
  __shared__ uint32_t s_warp[kEvWarps];
  __shared__ uint32_t s_pick[2];
  __shared__ int s_tmp[kEvWarps];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, h = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t bh = (int64_t)b * p.kv_heads + h;
  const float* sc = p.scores + bh * p.capacity;
  const int32_t* pos = p.positions + bh * p.capacity;
  float* nsc = p.a.new_scores + bh * p.capacity;
  int32_t* npos = p.a.new_positions + bh * p.capacity;
  const int len = p.lengths[b], next = p.a.next_pos[b], budget = p.a.budget;
  const int n = max(0, min(len, p.capacity)), live = min(n, budget);
  if (h == 0 && tid == 0) p.a.new_lengths[b] = min(len, min(budget, p.capacity));
  for (int i0 = tid; i0 < p.capacity; i0 += 4 * kEvThreads) {  // (four slots' loads in flight)
    float v[4];
    int at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kEvThreads;
      v[u] = i < n ? sc[i] : 0.f;
      at[u] = i < n ? pos[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kEvThreads;
      if (i >= p.capacity) break;
      if (p.cached) keys[i] = slot_key(p, v[u], at[u], next);
      nsc[i] = i < live ? v[u] : 0.f;
      npos[i] = i < live ? at[u] : -1;
    }
  }
  if (n <= budget) {
    if (tid == 0) p.moved[bh] = 0;
    return;
  }
  auto key = [&](int i) { return p.cached ? keys[i] : slot_key(p, sc[i], pos[i], next); };

  // ---- the budget-th largest key: digits of 11, 11 and 10 bits ----
  uint32_t prefix = 0, want = budget;  // keys that match `prefix` above the digit hold the want-th largest
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kEvCopies * kEvBins; i += kEvThreads) hist[i] = 0;
    __syncthreads();
    uint32_t* mine = hist + (warp % kEvCopies) * kEvBins;
    for (int i = tid; i < n; i += kEvThreads) {
      const uint32_t k = key(i);
      if (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits))) atomicAdd(&mine[(k >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // thread t holds the digits kEvBins - 1 - 2 t and the one below, from the top
    uint32_t own[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int w = 0; w < kEvCopies; ++w) own[e] += hist[w * kEvBins + kEvBins - 1 - 2 * tid - e];
    uint32_t inc = own[0] + own[1];
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, inc, m);
      if (lane >= m) inc += o;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    uint32_t above = lane < warp ? s_warp[lane] : 0;
    above = __reduce_add_sync(0xffffffffu, above) + inc - own[0] - own[1];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (above < want && want <= above + own[e]) {
        s_pick[0] = kEvBins - 1 - 2 * tid - e;
        s_pick[1] = want - above;
      }
      above += own[e];
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    want = s_pick[1];
  }
  // keys above `prefix` are kept, and of those equal to it the first `want`

  // ---- kept bits, in slot order: each warp walks a run of whole words ----
  const int words = (n + 31) / 32, run = (words + kEvWarps - 1) / kEvWarps;
  const int w0 = min(warp * run, words), w1 = min(w0 + run, words);
  int equal = 0;
  for (int w = w0; w < w1; ++w) {
    const int i = w * 32 + lane;
    equal += __popc(__ballot_sync(0xffffffffu, i < n && key(min(i, n - 1)) == prefix));
  }
  int taken = warps_prefix(equal, s_tmp);
  int holes = 0, late = 0;
  for (int w = w0; w < w1; ++w) {
    const int i = w * 32 + lane;
    const uint32_t k = key(min(i, n - 1));
    const uint32_t eq = __ballot_sync(0xffffffffu, i < n && k == prefix);
    const int rank = taken + __popc(eq & ((1u << lane) - 1));
    const bool keep = i < n && (k > prefix || (k == prefix && rank < (int)want));
    const uint32_t word = __ballot_sync(0xffffffffu, keep);
    taken += __popc(eq);
    if (lane == 0) kept[w] = word;
    const int below = budget - w * 32;  // of the word's slots, those under the budget
    const uint32_t low = below >= 32 ? 0xffffffffu : below <= 0 ? 0u : (1u << below) - 1;
    holes += __popc(~word & low);  // (the budget is below n: every such slot exists)
    late += __popc(word & ~low);
  }
  int hole_at = warps_prefix(holes, s_tmp);
  int late_at = warps_prefix(late, s_tmp);
  // the slots of move m: in the shared memory of the counts where few, else in
  // the words of its entry of the list
  longlong2* mv = p.moves + bh * p.max_moves;
  int2* pairs = reinterpret_cast<int2*>(hist);
  for (int w = w0; w < w1; ++w) {
    const int i = w * 32 + lane;
    const uint32_t word = kept[w];
    const int below = budget - w * 32;
    const uint32_t low = below >= 32 ? 0xffffffffu : below <= 0 ? 0u : (1u << below) - 1;
    const uint32_t hb = ~word & low, lb = word & ~low, under = (1u << lane) - 1;
    if ((hb >> lane) & 1u) {
      const int m = hole_at + __popc(hb & under);
      if (p.fused) pairs[m].y = i;
      else mv[m].y = i;
    }
    if ((lb >> lane) & 1u) {
      const int m = late_at + __popc(lb & under);
      if (p.fused) pairs[m].x = i;
      else mv[m].x = i;
    }
    hole_at += __popc(hb);
    late_at += __popc(lb);
  }
  __syncthreads();
  if (warp == kEvWarps - 1 && lane == 0) s_tmp[0] = late_at;  // the number of moves
  __syncthreads();
  const int moves = s_tmp[0];
  // ---- the slots' entries, and where their rows lie ----
  const int32_t* table = p.block_table + b * p.table_stride;
  const int mask = (1 << p.lg_page) - 1;
  auto offset = [&](int slot) -> long long {
    const int page = table[slot >> p.lg_page];
    if (page < 0 || page >= p.num_pages) return -1;
    return page * p.page_stride + h * p.head_stride + (slot & mask) * p.token_stride;
  };
  longlong2* list = p.fused ? reinterpret_cast<longlong2*>(hist) + kMvFused : mv;  // (past the pairs)
  for (int i = tid; i < moves; i += kEvThreads) {
    const int2 m = p.fused ? pairs[i] : make_int2(static_cast<int>(mv[i].x), static_cast<int>(mv[i].y));
    nsc[m.y] = sc[m.x];
    npos[m.y] = pos[m.x];
    list[i] = make_longlong2(offset(m.x), offset(m.y));
  }
  if (!p.fused) {
    if (tid == 0) p.moved[bh] = moves;
    return;
  }
  __syncthreads();
  move_rows(p, list, moves, tid >> p.lg_lanes, kEvThreads >> p.lg_lanes, tid & ((1 << p.lg_lanes) - 1));
}

__global__ void __launch_bounds__(kMvThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t bh = blockIdx.y;
  const int rows = kMvThreads >> p.lg_lanes;
  move_rows(p, p.moves + bh * p.max_moves, p.moved[bh], blockIdx.x * rows + (threadIdx.x >> p.lg_lanes), gridDim.x * rows,
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
  p.fused = max_moves <= kMvFused;
  const int smem = (kEvCopies * kEvBins + (p.capacity + 31) / 32 + (p.cached ? p.capacity : 0)) * 4;
  static int smem_set[64];
  s = ensure_smem(evict_select_kernel, smem, smem_set, "evict: shared memory attribute");
  if (s != TP_OK) return s;
  s = launch_early(evict_select_kernel, dim3(cache->kv_heads, cache->batch), kEvThreads, smem, st, "evict_select launch", p);
  if (s != TP_OK || p.fused) return s;
  int sms = 0;
  s = device_sms(&sms);
  if (s != TP_OK) return s;
  // about eight CTAs per SM in all, never more than the rows that may move
  const int rows = (kMvThreads >> p.lg_lanes) * kMvRows;
  const int64_t per_head = std::max<int64_t>(1, std::min<int64_t>((max_moves + rows - 1) / rows, (8 * sms + heads - 1) / heads));
  return launch_early(evict_move_kernel, dim3(static_cast<unsigned>(per_head), heads), kMvThreads, 0, st, "evict_move launch", p);
}

}  // extern "C"
