// Eviction from a paged cache by accumulated attention weight.
//
// Mathematics: the `budget` largest of n keys per (sequence, kv head), a key
// being the score's order-preserving 32-bit image (guarded slots above all,
// the lower slot first on equality).  A radix selection finds the budget-th
// key in four counting passes; one ordered pass marks the kept slots.  With
// the kept slots above the budget s_0 < s_1 < ... and the freed ones below it
// h_0 < h_1 < ..., slot s_i moves to h_i: as many rows as must move, every
// source at or above the budget and every destination below it, so the moves
// are independent of each other.
//
// Bound: the moves, 4 * head_dim bytes read and as many written per row; the
// selection reads 8 bytes a slot (and counts in L1 / L2).  Two launches: the
// selection per head, then all rows of all heads spread over the GPU.
#include <algorithm>

#include "tp_decode.cuh"
#include "tp_paged.cuh"

using namespace tp;

namespace {

constexpr int kEvThreads = 1024;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvMaxSlots = 1 << 20;
constexpr int kMvThreads = 256;

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
  int2* moves;     // [batch][kv_heads][max_moves]: (from, to)
};

__device__ __forceinline__ uint32_t slot_key(const EvictParams& p, const float* sc, const int32_t* pos, int next, int i) {
  const int at = pos[i];
  if (at < p.a.sinks || at >= next - p.a.recent) return 0xFFFFFFFFu;
  float v = sc[i];
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

__global__ void __launch_bounds__(kEvThreads, 1) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t s_dyn[];
  uint32_t* hist = s_dyn;                        // [warps][256]
  uint32_t* kept = s_dyn + kEvWarps * 256;       // a bit per slot
  __shared__ uint32_t s_sum[256];
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
  const int len = p.lengths[b], n = max(0, min(len, p.capacity)), budget = p.a.budget;
  if (h == 0 && tid == 0) p.a.new_lengths[b] = min(len, min(budget, p.capacity));
  const int live = min(n, budget);
  for (int i = tid; i < p.capacity; i += kEvThreads) {
    nsc[i] = i < live ? sc[i] : 0.f;
    npos[i] = i < live ? pos[i] : -1;
  }
  if (n <= budget) {
    if (tid == 0) p.moved[bh] = 0;
    return;
  }
  const int next = p.a.next_pos[b];

  // ---- the budget-th largest key, eight bits at a time ----
  uint32_t prefix = 0, want = budget;  // keys that match `prefix` above `shift` hold the want-th largest
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < kEvWarps * 256; i += kEvThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kEvThreads) {
      const uint32_t k = slot_key(p, sc, pos, next, i);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[warp * 256 + ((k >> shift) & 255)], 1u);
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t s = 0;
      for (int w = 0; w < kEvWarps; ++w) s += hist[w * 256 + tid];
      s_sum[tid] = s;
    }
    __syncthreads();
    if (warp == 0) {  // lane l holds digits 255 - 8 l - 7 .. 255 - 8 l, from the top
      uint32_t own[8], mine = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) mine += own[e] = s_sum[255 - 8 * lane - e];
      uint32_t inc = mine;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, inc, m);
        if (lane >= m) inc += o;
      }
      uint32_t above = inc - mine;
      if (above < want && want <= inc) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (above < want && want <= above + own[e]) {
            s_pick[0] = 255 - 8 * lane - e;
            s_pick[1] = want - above;
          }
          above += own[e];
        }
      }
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
    const uint32_t k = i < n ? slot_key(p, sc, pos, next, i) : 0;
    equal += __popc(__ballot_sync(0xffffffffu, i < n && k == prefix));
  }
  int taken = warps_prefix(equal, s_tmp);
  int holes = 0, late = 0;
  for (int w = w0; w < w1; ++w) {
    const int i = w * 32 + lane;
    const uint32_t k = i < n ? slot_key(p, sc, pos, next, i) : 0;
    const uint32_t eq = __ballot_sync(0xffffffffu, i < n && k == prefix);
    const int rank = taken + __popc(eq & ((1u << lane) - 1));
    const bool keep = i < n && (k > prefix || (k == prefix && rank < (int)want));
    const uint32_t word = __ballot_sync(0xffffffffu, keep);
    taken += __popc(eq);
    if (lane == 0) kept[w] = word;
    holes += __popc(__ballot_sync(0xffffffffu, !keep && i < budget));
    late += __popc(__ballot_sync(0xffffffffu, keep && i >= budget));
  }
  int hole_at = warps_prefix(holes, s_tmp);
  int late_at = warps_prefix(late, s_tmp);
  int2* mv = p.moves + bh * p.max_moves;
  for (int w = w0; w < w1; ++w) {
    const int i = w * 32 + lane;
    const bool keep = (kept[w] >> lane) & 1u;
    const bool hole = !keep && i < budget, over = keep && i >= budget;
    const uint32_t hb = __ballot_sync(0xffffffffu, hole), lb = __ballot_sync(0xffffffffu, over);
    if (hole) mv[hole_at + __popc(hb & ((1u << lane) - 1))].y = i;
    if (over) mv[late_at + __popc(lb & ((1u << lane) - 1))].x = i;
    hole_at += __popc(hb);
    late_at += __popc(lb);
  }
  __syncthreads();
  if (warp == kEvWarps - 1) s_tmp[0] = late_at;  // every lane the same: the number of moves
  __syncthreads();
  const int moves = s_tmp[0];
  for (int i = tid; i < moves; i += kEvThreads) {
    const int2 m = mv[i];
    nsc[m.y] = sc[m.x];
    npos[m.y] = pos[m.x];
  }
  if (tid == 0) p.moved[bh] = moves;
}

// One row (K and V of a slot) per group of head_dim / 8 lanes.
__global__ void __launch_bounds__(kMvThreads) evict_move_kernel(const __grid_constant__ EvictParams p, int lg_lanes) {
  pdl_trigger();
  pdl_wait();
  const int64_t bh = blockIdx.y;
  const int b = static_cast<int>(bh / p.kv_heads), h = static_cast<int>(bh - (int64_t)b * p.kv_heads);
  const int n = p.moved[bh];
  const int chunk = threadIdx.x & ((1 << lg_lanes) - 1);
  const int rows = kMvThreads >> lg_lanes;
  const int32_t* table = p.block_table + b * p.table_stride;
  const int mask = (1 << p.lg_page) - 1;
  for (int i = blockIdx.x * rows + (threadIdx.x >> lg_lanes); i < n; i += gridDim.x * rows) {
    const int2 m = p.moves[bh * p.max_moves + i];
    const int from = table[m.x >> p.lg_page], to = table[m.y >> p.lg_page];
    if (from < 0 || from >= p.num_pages || to < 0 || to >= p.num_pages || chunk * 8 >= p.head_dim) continue;
    const int64_t src = from * p.page_stride + h * p.head_stride + (m.x & mask) * p.token_stride + chunk * 8;
    const int64_t dst = to * p.page_stride + h * p.head_stride + (m.y & mask) * p.token_stride + chunk * 8;
    const uint4 kv = *reinterpret_cast<const uint4*>(p.k_pages + 2 * src);
    const uint4 vv = *reinterpret_cast<const uint4*>(p.v_pages + 2 * src);
    *reinterpret_cast<uint4*>(p.k_pages + 2 * dst) = kv;
    *reinterpret_cast<uint4*>(p.v_pages + 2 * dst) = vv;
  }
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
  *bytes = round256(heads * 4) + round256(heads * *max_moves * (int64_t)sizeof(int2));
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
  p.moves = reinterpret_cast<int2*>(ws + round256((int64_t)heads * 4));
  cudaStream_t st = as_stream(stream);
  const int smem = (kEvWarps * 256 + (p.capacity + 31) / 32) * 4;
  static int smem_set[64];
  s = ensure_smem(evict_select_kernel, smem, smem_set, "evict: shared memory attribute");
  if (s != TP_OK) return s;
  s = launch_early(evict_select_kernel, dim3(cache->kv_heads, cache->batch), kEvThreads, smem, st, "evict_select launch", p);
  if (s != TP_OK || max_moves == 0) return s;
  int sms = 0;
  s = device_sms(&sms);
  if (s != TP_OK) return s;
  int lg_lanes = log2_int((cache->head_dim + 7) / 8);
  const int rows = kMvThreads >> lg_lanes;
  // about eight CTAs per SM in all, never more than the rows that may move
  const int64_t per_head = std::max<int64_t>(1, std::min<int64_t>((max_moves + rows - 1) / rows, (8 * sms + heads - 1) / heads));
  return launch_early(evict_move_kernel, dim3(static_cast<unsigned>(per_head), heads), kMvThreads, 0, st, "evict_move launch",
                      p, lg_lanes);
}

}  // extern "C"
