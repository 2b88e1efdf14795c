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
// reduction and q, k can be turned in place.  A thread keeps its unit and head
// through the CTA's tokens (addresses advance by one addition), with several
// tokens' loads in flight.
//
// Measured (B200): 8192 tokens of 64 + 8 + 8 heads of 128 with the append, bf16,
// 62 us = 5.4 TB/s (0.83 of the measured HBM rate; issue slots 58 % busy); one
// token of 32 + 8 + 8 heads with head norms 3.3 us, the launch and two round
// trips.
#include <algorithm>
#include <type_traits>

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

// A vector's elements as floats, and back, two at a time.
template <class T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& x, float (&v)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = Elem<T>::to(x.v[e]);
}
template <class T, int N>
__device__ __forceinline__ void pack(const float (&v)[N], Pack<T, N>& x) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    if constexpr (N > 1 && sizeof(T) == 2) {
      if constexpr (std::is_same<T, __half>::value)
        *reinterpret_cast<__half2*>(&x.v[e]) = __floats2half2_rn(v[e], v[(e + 1) % N]);
      else
        *reinterpret_cast<__nv_bfloat162*>(&x.v[e]) = __floats2bfloat162_rn(v[e], v[(e + 1) % N]);
    } else {
      x.v[e] = Elem<T>::from(v[e]);
      if (N > 1) x.v[(e + 1) % N] = Elem<T>::from(v[(e + 1) % N]);
    }
  }
}

// N floats of shared memory, 16 bytes at a time (a unit's are so aligned).
template <int N>
__device__ __forceinline__ void read_floats(const float* p, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + e);
      v[e] = x.x;
      v[e + 1] = x.y;
      v[e + 2] = x.z;
      v[e + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = p[e];
  }
}

// UPL: units per lane (more than one only where a head has over 32 units).
template <class T, int VEC, int UPL>
__global__ void __launch_bounds__(kRtThreads, VEC == 1 ? 2 : 4) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ __align__(16) float cs[];  // [tpc][cos, sin][rot/2]
  __shared__ int64_t s_dst[kRtMaxTokens];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const int64_t tok0 = (int64_t)blockIdx.x * p.tpc;
  const int nt = static_cast<int>(min((int64_t)p.tpc, p.a.tokens - tok0));
  const int h0 = blockIdx.y * p.heads_cta, h1 = min(h0 + p.heads_cta, p.heads);
  const int half = p.a.rot_dim / 2;
  const int G = 1 << p.lg_group;
  const int u0 = tid & (G - 1), slot0 = tid >> p.lg_group, nslots = kRtThreads >> p.lg_group;

  // The source row of `head` at the CTA's first token, and its step per token.
  auto source = [&](int head, int64_t& step) -> const T* {
    const int k = head - p.a.q_heads, v = k - p.a.kv_heads;
    if (k < 0) {
      step = p.a.q_token_stride;
      return static_cast<const T*>(p.a.q) + tok0 * step + head * p.a.q_head_stride;
    }
    if (v < 0) {
      step = p.a.k_token_stride;
      return static_cast<const T*>(p.a.k) + tok0 * step + k * p.a.k_head_stride;
    }
    step = p.a.v_token_stride;
    return static_cast<const T*>(p.a.v) + tok0 * step + v * p.a.v_head_stride;
  };
  constexpr int TB = UPL == 1 ? 2 : 1;  // tokens whose loads are in flight
  Pack<T, VEC> x[TB][UPL][2];
  auto load = [&](const T* src, int64_t step, int t0) {
#pragma unroll
    for (int t = 0; t < TB; ++t)
      if (t0 + t < nt)
#pragma unroll
        for (int i = 0; i < UPL; ++i) {
          const int u = u0 + i * G;
          if (u < p.units) {
            int lo, hi;
            unit_at<VEC>(p, u, lo, hi);
            x[t][i][0] = *reinterpret_cast<const Pack<T, VEC>*>(src + t * step + lo);
            x[t][i][1] = *reinterpret_cast<const Pack<T, VEC>*>(src + t * step + hi);
          }
        }
  };
  int64_t step = 0;
  const T* src = h0 + slot0 < h1 ? source(h0 + slot0, step) : nullptr;
  if (src) load(src, step, 0);  // in flight while the angles are computed

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
    cs[(2 * t) * half + n] = c * p.a.scale;
    cs[(2 * t + 1) * half + n] = (p.a.inverse ? -s : s) * p.a.scale;
  }
  __syncthreads();

  const bool norms = p.a.q_norm || p.a.k_norm;
  // every warp makes the same number of rounds: the norm's shuffles need all lanes
  for (int base = h0; base < h1; base += nslots) {
    const int head = base + slot0;
    const bool on = head < h1;
    const int kind = head < p.a.q_heads ? 0 : head < p.a.q_heads + p.a.kv_heads ? 1 : 2;
    const int h = kind == 0 ? head : kind == 1 ? head - p.a.q_heads : head - p.a.q_heads - p.a.kv_heads;
    const T* w = static_cast<const T*>(kind == 0 ? p.a.q_norm : kind == 1 ? p.a.k_norm : nullptr);
    if (base != h0) src = on ? source(head, step) : nullptr;
    // contiguous outputs advance by a row of heads; pages are looked up
    const int64_t out_step = (int64_t)(kind == 0 ? p.a.q_heads : p.a.kv_heads) * p.a.head_dim;
    T* out = kind == 0 ? static_cast<T*>(p.a.q_out) : p.paged ? nullptr : static_cast<T*>(p.a.k_out);
    if (out) out += tok0 * out_step + h * p.a.head_dim;
    T* pages = static_cast<T*>(kind == 1 ? p.k_pages : p.v_pages) + (p.paged ? h * p.head_stride : 0);
    for (int t0 = 0; t0 < nt; t0 += TB) {
      if (src && (base != h0 || t0)) load(src, step, t0);
#pragma unroll
      for (int tt = 0; tt < TB; ++tt) {
        const int t = t0 + tt;
        if (t >= nt) break;
        float rinv = 1.f;
        if (norms) {
          float sq = 0.f;
#pragma unroll
          for (int i = 0; i < UPL; ++i)
            if (on && u0 + i * G < p.units)
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                const float a = Elem<T>::to(x[tt][i][0].v[e]), b = Elem<T>::to(x[tt][i][1].v[e]);
                sq = fmaf(a, a, fmaf(b, b, sq));
              }
          for (int m = G >> 1; m; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m);
          if (w) rinv = rsqrtf(sq / p.a.head_dim + p.a.eps);
        }
        T* dst = out ? out + t * out_step : s_dst[t] >= 0 ? pages + s_dst[t] : nullptr;
        if (!on || !dst) continue;
#pragma unroll
        for (int i = 0; i < UPL; ++i) {
          const int u = u0 + i * G;
          if (u >= p.units) continue;
          int lo, hi;
          unit_at<VEC>(p, u, lo, hi);
          if (kind < 2 && (w || u < p.rot_units)) {
            float a[VEC], b[VEC];
            unpack(x[tt][i][0], a);
            unpack(x[tt][i][1], b);
            if (w) {
              float wa[VEC], wb[VEC];
              unpack(*reinterpret_cast<const Pack<T, VEC>*>(w + lo), wa);
              unpack(*reinterpret_cast<const Pack<T, VEC>*>(w + hi), wb);
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                a[e] *= rinv * wa[e];
                b[e] *= rinv * wb[e];
              }
            }
            if (u < p.rot_units) {
              const float* co = cs + (2 * t) * half + u * VEC;
              float c[VEC], s[VEC];
              read_floats(co, c);
              read_floats(co + half, s);
              if (!p.a.interleaved || VEC == 1) {  // VEC = 1: both layouts pair the unit's two elements
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                  const float y = a[e] * c[e] - b[e] * s[e];
                  b[e] = b[e] * c[e] + a[e] * s[e];
                  a[e] = y;
                }
              } else {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                  constexpr int O = VEC > 1 ? 1 : 0, H = VEC / 2;
                  const float ca = c[e / 2], sa = s[e / 2], cb = c[H + e / 2], sb = s[H + e / 2];
                  const float y = a[e] * ca - a[e + O] * sa;
                  a[e + O] = a[e + O] * ca + a[e] * sa;
                  a[e] = y;
                  const float z = b[e] * cb - b[e + O] * sb;
                  b[e + O] = b[e + O] * cb + b[e] * sb;
                  b[e] = z;
                }
              }
            }
            pack(a, x[tt][i][0]);
            pack(b, x[tt][i][1]);
          }
          *reinterpret_cast<Pack<T, VEC>*>(dst + lo) = x[tt][i][0];
          *reinterpret_cast<Pack<T, VEC>*>(dst + hi) = x[tt][i][1];
        }
      }
      if (src) src += TB * step;
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
  // per CTA, which share the fixed costs (8192 tokens: 62 us, 65 us at eight
  // CTAs per SM, i.e. half the tokens each).
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
  const int smem = p.tpc * p.a.rot_dim * static_cast<int>(sizeof(float));
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
