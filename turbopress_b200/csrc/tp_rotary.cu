// Rotary positions of queries and keys, with the optional per-head RMS norm
// before them and the append of keys and values to a paged cache.
//
// Mathematics: pair (i, j) of a head turns by the angle 2 pi * p * f, where f
// (turns per position) is held as a 64-bit fixed-point fraction: p * f modulo
// 2^64 is the angle modulo one turn, within the p * 2^-65 turns that rounding f
// leaves.  A 32-bit product loses 0.004 rad at position 100000.  cos and sin then come from sincospif of a value in
// [-1, 1).  Everything is fp32, rounded once on the way out.
//
// Bound: memory.  Each element of q, k, v is read once and written once; the
// 64 sincospif of a token cost as much as moving ~10 heads, so a CTA computes
// them once per token into shared memory and all its heads use them.
//
// Layout: a unit is the 2*VEC elements one thread turns: two VEC-element
// vectors (16 bytes each where VEC = 8) at p and p + rot/2, or adjacent ones
// in the interleaved layout and in the part that is not turned.  G lanes (a
// power of two) hold one head, so the norm's sum of squares is a shuffle
// reduction and q, k can be turned in place.
#include <algorithm>

#include "tp_decode.cuh"
#include "tp_paged.cuh"

using namespace tp;

namespace {

constexpr int kRtThreads = 256;
constexpr int kRtMaxTokens = 8;  // tokens per CTA

struct RotaryParams {
  tp_rotary_args a;
  const int32_t* block_table;
  const int32_t* lengths;
  float* scores;
  int32_t* slot_pos;
  void* k_pages;
  void* v_pages;
  int64_t num_pages, page_stride, head_stride, token_stride, table_stride;
  int capacity, lg_page, paged;
  int tpc;         // tokens per CTA
  int heads;       // q + k (+ v) heads of a token
  int heads_cta;   // heads per CTA (grid.y)
  int units;       // units per head
  int rot_units;   // of those, turned
  int lg_group;    // log2 G
};

// Positions the unit's two vectors start at.
template <int VEC>
__device__ __forceinline__ void unit_at(const RotaryParams& p, int u, int& lo, int& hi) {
  if (u < p.rot_units && !p.a.interleaved) {
    lo = u * VEC;
    hi = lo + p.a.rot_dim / 2;
  } else {
    lo = u * 2 * VEC;
    hi = lo + VEC;
  }
}

// UPL: units per lane (more than one only where a head has over 32 units).
template <class T, int VEC, int UPL>
__global__ void __launch_bounds__(kRtThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 cs[];  // [tpc][rot/2]
  __shared__ int64_t s_dst[kRtMaxTokens];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const int64_t tok0 = (int64_t)blockIdx.x * p.tpc;
  const int nt = static_cast<int>(min((int64_t)p.tpc, p.a.tokens - tok0));
  const int h0 = blockIdx.y * p.heads_cta, nh = min(p.heads_cta, p.heads - h0);
  const int half = p.a.rot_dim / 2;
  const int G = 1 << p.lg_group;
  const int u0 = tid & (G - 1), slot0 = tid >> p.lg_group, nslots = kRtThreads >> p.lg_group;
  const int total = nt * nh;

  // a lane's units of one head
  auto source = [&](int idx, const T*& src, int& t, int& head) {
    t = idx / nh;
    head = h0 + idx - t * nh;
    const int64_t n = tok0 + t;
    if (head < p.a.q_heads) src = static_cast<const T*>(p.a.q) + n * p.a.q_token_stride + head * p.a.q_head_stride;
    else if (head < p.a.q_heads + p.a.kv_heads)
      src = static_cast<const T*>(p.a.k) + n * p.a.k_token_stride + (head - p.a.q_heads) * p.a.k_head_stride;
    else
      src = static_cast<const T*>(p.a.v) + n * p.a.v_token_stride + (head - p.a.q_heads - p.a.kv_heads) * p.a.v_head_stride;
  };
  auto load = [&](int idx, Pack<T, VEC> (&x)[UPL][2]) {
    if (idx >= total) return;
    const T* src;
    int t, head;
    source(idx, src, t, head);
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int u = u0 + i * G;
      if (u < p.units) {
        int lo, hi;
        unit_at<VEC>(p, u, lo, hi);
        x[i][0] = *reinterpret_cast<const Pack<T, VEC>*>(src + lo);
        x[i][1] = *reinterpret_cast<const Pack<T, VEC>*>(src + hi);
      }
    }
  };

  Pack<T, VEC> x[UPL][2], nx[UPL][2];
  load(slot0, x);  // in flight while the angles are computed

  if (p.paged && tid < nt) {
    const int64_t n = tok0 + tid;
    const int b = static_cast<int>(n / p.a.seq), i = static_cast<int>(n - (int64_t)b * p.a.seq);
    const int len = p.lengths[b];
    int64_t dst = -1;
    if (len >= 0 && i < p.capacity - len) {
      const int slot = len + i;
      const int page = p.block_table[b * p.table_stride + (slot >> p.lg_page)];
      if (page >= 0 && page < p.num_pages) dst = page * p.page_stride + (slot & ((1 << p.lg_page) - 1)) * p.token_stride;
      if (blockIdx.y == 0) {
        const int64_t at = (int64_t)b * p.a.kv_heads * p.capacity + slot;
        const int pos = static_cast<int>(p.a.positions ? p.a.positions[n] : (int64_t)p.a.base[b] + i);
        for (int h = 0; h < p.a.kv_heads; ++h) {
          if (p.slot_pos) p.slot_pos[at + (int64_t)h * p.capacity] = pos;
          if (p.scores) p.scores[at + (int64_t)h * p.capacity] = 0.f;
        }
      }
    }
    s_dst[tid] = dst;
  }
  for (int i = tid; i < nt * half; i += kRtThreads) {
    const int t = i / half, n = i - t * half;
    const int64_t tok = tok0 + t;
    int64_t pos;
    if (p.a.positions) {
      pos = p.a.positions[tok];
    } else {
      const int64_t b = tok / p.a.seq;
      pos = (int64_t)p.a.base[b] + (tok - b * p.a.seq);
    }
    const int64_t turn = static_cast<int64_t>(static_cast<uint64_t>(pos) * p.a.freq[n]);  // [-1/2, 1/2) turns
    float s, c;
    sincospif(__ll2float_rn(turn) * 1.0842021724855044e-19f /* 2^-63 */, &s, &c);
    cs[i] = make_float2(c * p.a.scale, (p.a.inverse ? -s : s) * p.a.scale);
  }
  __syncthreads();

  // every warp makes the same number of rounds: the norm's shuffles need all lanes
  for (int base = 0; base < total; base += nslots) {
    const int idx = base + slot0;
    load(idx + nslots, nx);
    const bool on = idx < total;
    const T* src;
    int t = 0, head = 0;
    if (on) source(idx, src, t, head);
    const int kind = head < p.a.q_heads ? 0 : head < p.a.q_heads + p.a.kv_heads ? 1 : 2;
    const T* w = static_cast<const T*>(kind == 0 ? p.a.q_norm : kind == 1 ? p.a.k_norm : nullptr);
    float rinv = 1.f;
    if (p.a.q_norm || p.a.k_norm) {  // the same in every thread
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < UPL; ++i)
        if (on && u0 + i * G < p.units)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float a = Elem<T>::to(x[i][0].v[e]), b = Elem<T>::to(x[i][1].v[e]);
            sq = fmaf(a, a, fmaf(b, b, sq));
          }
      for (int m = G >> 1; m; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m);
      if (w) rinv = rsqrtf(sq / p.a.head_dim + p.a.eps);
    }
    T* dst = nullptr;
    if (on) {
      const int64_t n = tok0 + t;
      if (kind == 0) {
        dst = static_cast<T*>(p.a.q_out) + (n * p.a.q_heads + head) * p.a.head_dim;
      } else {
        const int h = kind == 1 ? head - p.a.q_heads : head - p.a.q_heads - p.a.kv_heads;
        if (!p.paged) {
          dst = static_cast<T*>(p.a.k_out) + (n * p.a.kv_heads + h) * p.a.head_dim;
        } else if (s_dst[t] >= 0) {
          dst = static_cast<T*>(kind == 1 ? p.k_pages : p.v_pages) + s_dst[t] + h * p.head_stride;
        }
      }
    }
    if (dst) {
#pragma unroll
      for (int i = 0; i < UPL; ++i) {
        const int u = u0 + i * G;
        if (u >= p.units) continue;
        int lo, hi;
        unit_at<VEC>(p, u, lo, hi);
        if (kind < 2 && (w || u < p.rot_units)) {
          float a[VEC], b[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            a[e] = Elem<T>::to(x[i][0].v[e]);
            b[e] = Elem<T>::to(x[i][1].v[e]);
          }
          if (w) {
            const Pack<T, VEC> wa = *reinterpret_cast<const Pack<T, VEC>*>(w + lo);
            const Pack<T, VEC> wb = *reinterpret_cast<const Pack<T, VEC>*>(w + hi);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              a[e] *= rinv * Elem<T>::to(wa.v[e]);
              b[e] *= rinv * Elem<T>::to(wb.v[e]);
            }
          }
          if (u < p.rot_units) {
            const float2* c = cs + t * half + u * VEC;
            if (!p.a.interleaved || VEC == 1) {  // VEC = 1: both layouts pair the unit's two elements
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                const float2 f = c[e];
                const float y = a[e] * f.x - b[e] * f.y;
                b[e] = b[e] * f.x + a[e] * f.y;
                a[e] = y;
              }
            } else {
#pragma unroll
              for (int e = 0; e < VEC; e += 2) {
                const float2 f = c[e / 2], g = c[VEC / 2 + e / 2];
                const float y = a[e] * f.x - a[(e + 1) % VEC] * f.y;
                a[(e + 1) % VEC] = a[(e + 1) % VEC] * f.x + a[e] * f.y;
                a[e] = y;
                const float z = b[e] * g.x - b[(e + 1) % VEC] * g.y;
                b[(e + 1) % VEC] = b[(e + 1) % VEC] * g.x + b[e] * g.y;
                b[e] = z;
              }
            }
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            x[i][0].v[e] = Elem<T>::from(a[e]);
            x[i][1].v[e] = Elem<T>::from(b[e]);
          }
        }
        *reinterpret_cast<Pack<T, VEC>*>(dst + lo) = x[i][0];
        *reinterpret_cast<Pack<T, VEC>*>(dst + hi) = x[i][1];
      }
    }
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      x[i][0] = nx[i][0];
      x[i][1] = nx[i][1];
    }
  }
}

template <class T, int VEC, int UPL>
tp_status launch_rotary(RotaryParams& p, cudaStream_t st) {
  p.units = p.a.head_dim / (2 * VEC);
  p.rot_units = p.a.rot_dim / (2 * VEC);
  p.lg_group = std::min(5, log2_int(p.units));
  // One token per CTA, and its heads over several CTAs, while that keeps the
  // grid under four CTAs per SM (short calls: latency); else several tokens
  // per CTA, which share the launch's fixed costs.
  int sms = 0;
  const tp_status s = device_sms(&sms);
  if (s != TP_OK) return s;
  const int nslots = kRtThreads >> p.lg_group;
  const int64_t want = 4 * (int64_t)sms;
  p.tpc = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kRtMaxTokens, p.a.tokens / want)));
  int split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want / p.a.tokens, (p.heads + nslots - 1) / nslots)));
  p.heads_cta = (p.heads + split - 1) / split;
  split = (p.heads + p.heads_cta - 1) / p.heads_cta;
  const int64_t grid = (p.a.tokens + p.tpc - 1) / p.tpc;
  if (grid > 0x7FFFFFFF) return fail(TP_ERR_UNSUPPORTED, "tp_rotary: too many tokens");
  const int smem = p.tpc * (p.a.rot_dim / 2) * static_cast<int>(sizeof(float2));
  return launch_early(rotary_kernel<T, VEC, UPL>, dim3(static_cast<unsigned>(grid), split), kRtThreads, smem, st,
                      "rotary launch", p);
}

template <class T>
tp_status dispatch_rotary(RotaryParams& p, cudaStream_t st) {
  const tp_rotary_args& a = p.a;
  // the widest vector that divides the head, its turned part, every stride and address
  auto fits = [&](int vec) {
    const int64_t strides[] = {a.q_token_stride, a.q_head_stride, a.k_token_stride, a.k_head_stride,
                               p.paged ? a.v_token_stride : 0, p.paged ? a.v_head_stride : 0};
    for (int64_t s : strides)
      if (s % vec) return false;
    const void* ptrs[] = {a.q, a.k, p.paged ? a.v : nullptr, a.q_out, p.paged ? nullptr : a.k_out, a.q_norm, a.k_norm};
    const uintptr_t bytes = std::min<uintptr_t>(16, vec * sizeof(T));
    for (const void* q : ptrs)
      if (!aligned(q, bytes)) return false;
    return a.head_dim % (2 * vec) == 0 && a.rot_dim % (2 * vec) == 0;
  };
  if (fits(8)) return launch_rotary<T, 8, 1>(p, st);
  if (fits(4)) return launch_rotary<T, 4, 1>(p, st);
  return launch_rotary<T, 1, 4>(p, st);
}

}  // namespace

extern "C" {

TP_API tp_status tp_rotary(const tp_rotary_args* args, const tp_paged_cache* cache, void* stream) {
  if (!args) return fail(TP_ERR_ARG, "tp_rotary: null arguments");
  const tp_rotary_args& a = *args;
  if (a.tokens < 0 || a.seq < 1 || a.tokens % a.seq || a.q_heads < 0 || a.kv_heads < 0 || a.q_heads > 65535 ||
      a.kv_heads > 65535 || a.q_heads + a.kv_heads < 1)
    return fail(TP_ERR_ARG, "tp_rotary: bad token or head counts");
  if (a.head_dim < 2 || a.head_dim > 256 || a.head_dim % 2 || a.rot_dim < 2 || a.rot_dim % 2 || a.rot_dim > a.head_dim)
    return fail(TP_ERR_UNSUPPORTED, "tp_rotary: head_dim %d and rot_dim %d must be even, rot_dim <= head_dim <= 256",
                a.head_dim, a.rot_dim);
  if (!valid_dtype(a.dtype)) return fail(TP_ERR_ARG, "tp_rotary: bad dtype %d", a.dtype);
  if (cache) {
    const tp_status s = check_cache(cache, "tp_rotary");
    if (s != TP_OK) return s;
    if (cache->dtype != a.dtype || cache->head_dim != a.head_dim || cache->kv_heads != a.kv_heads ||
        (int64_t)cache->batch * a.seq != a.tokens)
      return fail(TP_ERR_ARG, "tp_rotary: the cache's dtype, heads, head_dim or batch differ from the tokens'");
  }
  if (a.tokens == 0) return clear_ok();
  if ((a.q_heads && (!a.q || !a.q_out)) || (a.kv_heads && (!a.k || (cache ? !a.v : !a.k_out))) || !a.freq ||
      (!a.positions && !a.base))
    return fail(TP_ERR_ARG, "tp_rotary: null pointer");
  RotaryParams p{};
  p.a = a;
  p.paged = cache != nullptr;
  p.heads = a.q_heads + a.kv_heads * (cache ? 2 : 1);
  if (cache) {
    p.block_table = cache->block_table;
    p.lengths = cache->lengths;
    p.scores = cache->scores;
    p.slot_pos = cache->positions;
    p.k_pages = cache->k_pages;
    p.v_pages = cache->v_pages;
    p.num_pages = cache->num_pages;
    p.page_stride = cache->page_stride;
    p.head_stride = cache->head_stride;
    p.token_stride = cache->token_stride;
    p.table_stride = cache->table_stride;
    p.capacity = cache->max_pages * cache->page_size;
    p.lg_page = log2_int(cache->page_size);
  }
  cudaStream_t st = as_stream(stream);
  if (a.dtype == TP_F16) return dispatch_rotary<__half>(p, st);
  if (a.dtype == TP_BF16) return dispatch_rotary<__nv_bfloat16>(p, st);
  return dispatch_rotary<float>(p, st);
}

}  // extern "C"
