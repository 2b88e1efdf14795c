// Verification of drafted tokens against the target's logits.
//
// Mathematics: with p = softmax(x / t) and u uniform, accepting a draft d ~ q
// while u q(d) < p(d) and drawing a replacement from max(p - q, 0) at the first
// rejection leaves the tokens distributed as the target's own.  The draw is an
// exponential race: with independent exponentials e, argmax r_i / e_i is i with
// probability r_i / sum r, needs no normaliser and no prefix sums, and a
// maximum does not depend on the order it is taken in.
//
// Bound: memory.  One pass over the logits (running maximum m and sum of
// 2^((x - m) c), or the argmax for a greedy sequence), one pass over the one
// row that decides (in L2 for small batches), its draft row and its noise.
//
// Split: rows are cut into slices of equal length over the GPU; the last CTA
// of a sequence joins its rows' slices, walks the drafts and leaves the row to
// draw from; a second launch races over it, its last CTA writing the token.
// Counters and keys in the workspace return to zero.
//
// Measured (B200, whole calls): four greedy drafts over 151936 fp32 logits
// 7.4 us; 32 sequences of seven drafts over 128256 fp16 logits with draft
// probabilities 32 us = 3.1 TB/s (rows 17: exponentials and the joins' tail; race
// 12); five sequences of three drafts over 5003 10 us, latencies.
#include <algorithm>

#include "tp_decode.cuh"
#include "tp_paged.cuh"

using namespace tp;

namespace {

constexpr int kVfThreads = 256;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfResident = 6;    // CTAs per SM
constexpr int kVfMaxRows = 64;    // drafts + 1
constexpr int kVfMaxSplits = 128;
constexpr float kVfLeast = 1.17549435e-38f;  // temperatures below count as 0 (1 / t would pass fp32's range)
// Vocabulary up to which the CTA that decides on a sequence also draws, without
// a second launch: five sequences of 5003 tokens 9.8 us of GPU time so, 11.8 us
// with it; of 16000 tokens 12.8 against 11.3 us.
constexpr int kVfAlone = 8192;

struct Part {  // one slice of a row
  float m, l;               // sampled: maximum and sum of 2^((x - m) c),
  float draft, need;        // in slice 0 the draft's logit and uniform * q (infinite for a draft that cannot stand)
  unsigned long long key;   // greedy: argmax key
};

struct Choice {  // what a sequence draws from
  float m, c, inv_l;  // p_i = 2^((x_i - m) c) * inv_l
  int row;            // of its logits; -1: nothing to draw
  int residual;       // 1: from max(p - q, 0)
};

struct VerifyParams {
  tp_verify_args a;
  int splits, race_splits;
  Part* part;                 // [batch][rows][splits]
  Choice* choice;             // [batch]
  unsigned long long* key;    // [batch]: the race's leader
  unsigned* done;             // [batch][2]: CTAs that have arrived
};

__device__ __forceinline__ unsigned long long argmax_key(float v, unsigned idx) {
  unsigned u;
  if (v != v) {
    u = 0xFFFFFFFFu;
  } else {
    if (v == 0.f) v = 0.f;
    u = __float_as_uint(v);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  }
  return (static_cast<unsigned long long>(u) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ unsigned key_index(unsigned long long k) { return 0xFFFFFFFFu - static_cast<unsigned>(k); }

__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, k, m);
    k = o > k ? o : k;
  }
  return k;
}

// Elements [lo, hi) of a row that fall to this thread, in ascending order:
// vec(i, w) for U 16-byte vectors of the aligned middle (vector u at
// i + u * kVfThreads vectors) or one, each(i, x) for single elements at ragged
// ends.
template <int U, class T, class F, class G>
__device__ __forceinline__ void for_slice(const T* row, int lo, int hi, F each, G vec) {
  constexpr int V = 16 / sizeof(T);
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(T));
  const int head = min(hi, lo + (mis ? V - mis : 0));
  if (lo + (int)threadIdx.x < head) each(lo + threadIdx.x, Elem<T>::to(row[lo + threadIdx.x]));
  const int nvec = (hi - head) / V;
  const uint4* mid = reinterpret_cast<const uint4*>(row + head);
  int i = threadIdx.x;
  if constexpr (U > 1) {
    for (; i + (U - 1) * kVfThreads < nvec; i += U * kVfThreads) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = __ldg(mid + i + u * kVfThreads);
      vec(head + i * V, w);
    }
  }
  for (; i < nvec; i += kVfThreads) {
    const uint4 w[1] = {__ldg(mid + i)};
    vec(head + i * V, w);
  }
  const int tail = head + nvec * V + threadIdx.x;
  if (tail < hi) each(tail, Elem<T>::to(row[tail]));
}

// Two neighbouring elements of a vector's word pair w[e].
template <class T>
struct Two;
template <>
struct Two<__half> {
  static __device__ __forceinline__ float2 at(const uint4& w, int e) {
    return __half22float2(reinterpret_cast<const __half2*>(&w)[e]);
  }
  template <int N>
  static __device__ __forceinline__ float largest(const uint4 (&w)[N]) {
    const __half2* h = reinterpret_cast<const __half2*>(w);
    __half2 x = h[0];
#pragma unroll
    for (int e = 1; e < 4 * N; ++e) x = __hmax2(x, h[e]);
    const float2 f = __half22float2(x);
    return fmaxf(f.x, f.y);
  }
};
template <>
struct Two<__nv_bfloat16> {
  static __device__ __forceinline__ float2 at(const uint4& w, int e) {
    return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&w)[e]);
  }
  template <int N>
  static __device__ __forceinline__ float largest(const uint4 (&w)[N]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
    __nv_bfloat162 x = h[0];
#pragma unroll
    for (int e = 1; e < 4 * N; ++e) x = __hmax2(x, h[e]);
    const float2 f = __bfloat1622float2(x);
    return fmaxf(f.x, f.y);
  }
};
template <>
struct Two<float> {
  static __device__ __forceinline__ float2 at(const uint4& w, int e) { return reinterpret_cast<const float2*>(&w)[e]; }
  template <int N>
  static __device__ __forceinline__ float largest(const uint4 (&w)[N]) {
    const float* f = reinterpret_cast<const float*>(w);
    float x = f[0];
#pragma unroll
    for (int e = 1; e < 4 * N; ++e) x = fmaxf(x, f[e]);
    return x;
  }
};

// Packed fp32 pairs (one instruction for two elements).
__device__ __forceinline__ uint64_t pack2(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x to 2 ulp; below 2^-126 it gives 0, which no sum or comparison here notices.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Joins two (m, l) with 2^((x - m) c) terms.
__device__ __forceinline__ void join(float& m, float& l, float m2, float l2, float c) {
  const float top = fmaxf(m, m2);
  const float f = m == top ? 1.f : exp2f((m - top) * c), g = m2 == top ? 1.f : exp2f((m2 - top) * c);
  l = (l == 0.f ? 0.f : l * f) + (l2 == 0.f ? 0.f : l2 * g);
  m = top;
}

// Largest key of the block, in every thread.
__device__ __forceinline__ unsigned long long block_max(unsigned long long k, unsigned long long* s_k) {
  k = warp_max(k);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_k[threadIdx.x >> 5] = k;
  __syncthreads();
  k = s_k[0];
#pragma unroll
  for (int w = 1; w < kVfWarps; ++w) k = s_k[w] > k ? s_k[w] : k;
  return k;
}
// *at, in every thread of the block, and 0 in its place.
__device__ __forceinline__ unsigned long long take_key(unsigned long long* at, unsigned long long* s_k) {
  __syncthreads();
  if (threadIdx.x == 0) s_k[0] = atomicExch(at, 0ull);
  __syncthreads();
  return s_k[0];
}
// N neighbouring floats, 16 bytes at a time where the address allows.
template <int N>
__device__ __forceinline__ void load_floats(const float* p, float (&v)[N]) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
      v[i] = x.x;
      v[i + 1] = x.y;
      v[i + 2] = x.z;
      v[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __ldg(p + i);
  }
}

// The race over elements [lo, hi) of the choice's row, from max(p - q, 0)
// (`residual`) or from p: the block's largest key, in every thread.
template <class T>
__device__ __forceinline__ unsigned long long race_slice(const VerifyParams& p, int b, const Choice& ch, int lo, int hi,
                                                         bool residual, unsigned long long* s_k) {
  const T* row = static_cast<const T*>(p.a.logits) + (int64_t)b * p.a.batch_stride + (int64_t)ch.row * p.a.row_stride;
  const float* noise = p.a.noise + (int64_t)b * p.a.vocab;
  const float* q = residual && p.a.draft_probs
                       ? p.a.draft_probs + ((int64_t)b * p.a.drafts + ch.row) * p.a.vocab
                       : nullptr;
  const int64_t hot = residual && !q ? p.a.draft_tokens[(int64_t)b * p.a.drafts + ch.row] : -1;
  float top = 0.f;  // the largest r / e, and where
  int at = -1;
  auto chance = [&](float x) { return exp2f((x - ch.m) * ch.c) * ch.inv_l; };
  auto enter = [&](int i, float r, float e) {  // the exact quotient
    const float f = r / e;
    if (f > top) {
      top = f;
      at = i;
    }
  };
  auto one = [&](int i, float x) {
    const float qi = q ? q[i] : i == hot ? 1.f : 0.f;
    enter(i, fmaxf(chance(x) - qi, 0.f), noise[i]);
  };
  constexpr int V = 16 / sizeof(T);
  for_slice<1>(row, lo, hi, one, [&](int i, const uint4 (&w)[1]) {
    float e[V], r[V];
    if (q) {
      load_floats<V>(q + i, r);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) r[k] = i + k == hot ? 1.f : 0.f;
    }
    load_floats<V>(noise + i, e);
    // The exact divisions are for quotients near the vector's largest, if that
    // is near the best or above; where the largest is below 1e-30 (no
    // approximation holds there), for all.
    float near = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float2 x = Two<T>::at(w[0], k / 2);
      r[k] = fmaxf(exp2_fast(((k & 1 ? x.y : x.x) - ch.m) * ch.c) * ch.inv_l - r[k], 0.f);
      float inv;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(e[k]));
      e[k] = r[k] * inv;
      near = fmaxf(near, e[k]);
    }
    if (near >= top * 0.999f || top < 1e-30f) {
      unsigned some = 0;
#pragma unroll
      for (int k = 0; k < V; ++k) some |= (near < 1e-30f ? r[k] > 0.f : e[k] >= near * 0.999f) ? 1u << k : 0u;
      for (; some; some &= some - 1) {
        const int k = __ffs(some) - 1;
        one(i + k, Elem<T>::to(row[i + k]));
      }
    }
  });
  return block_max(at >= 0 ? argmax_key(top, at) : 0ull, s_k);
}

// The whole row's race by one block, out of line: where it ends the rows kernel
// (its registers are not the streaming loop's) and where it hardly occurs.
template <class T>
__device__ __noinline__ unsigned long long race_row(const VerifyParams& p, int b, Choice ch, bool residual,
                                                    unsigned long long* s_k) {
  return race_slice<T>(p, b, ch, 0, p.a.vocab, residual, s_k);
}

// ALONE: the CTA that decides on a sequence also draws.
template <class T, bool ALONE>
__global__ void __launch_bounds__(kVfThreads, kVfResident) verify_rows_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ float s_m[kVfWarps], s_l[kVfWarps];
  __shared__ unsigned long long s_k[kVfWarps];
  __shared__ bool s_last;
  __shared__ bool s_ok[kVfMaxRows];
  __shared__ float s_rm[kVfMaxRows], s_rl[kVfMaxRows];
  __shared__ unsigned s_arg[kVfMaxRows];
  pdl_trigger();
  pdl_wait();
  const int rows = p.a.drafts + 1;
  const int b = blockIdx.y / rows, k = blockIdx.y - b * rows;
  const int used = p.a.counts ? max(0, min(p.a.counts[b], p.a.drafts)) : p.a.drafts;
  if (k > used) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float heat = p.a.temperature ? p.a.temperature[b] : 0.f;
  const bool greedy = !(heat >= kVfLeast);
  const float c = greedy ? 0.f : 1.4426950408889634f / heat;
  const T* row = static_cast<const T*>(p.a.logits) + (int64_t)b * p.a.batch_stride + (int64_t)k * p.a.row_stride;
  const int per = (p.a.vocab + p.splits - 1) / p.splits;
  const int lo = min((int)blockIdx.x * per, p.a.vocab), hi = min(lo + per, p.a.vocab);

  // what decides on the row's draft, fetched while the row streams
  float draft = 0.f, need = INFINITY;
  if (blockIdx.x == 0 && tid == 0 && k < used && !greedy) {
    const int64_t d = p.a.draft_tokens[(int64_t)b * p.a.drafts + k];
    if (d >= 0 && d < p.a.vocab) {
      const float qd = p.a.draft_probs ? p.a.draft_probs[((int64_t)b * p.a.drafts + k) * p.a.vocab + d] : 1.f;
      draft = Elem<T>::to(row[d]);
      need = p.a.uniforms[(int64_t)b * p.a.drafts + k] * qd;
    }
  }

  float m = -INFINITY, l = 0.f;
  unsigned long long best = 0ull;
  if (greedy) {
    float top = -INFINITY;
    int at = -1;
    auto one = [&](int i, float x) {
      if (at < 0 || (!(x <= top) && top == top)) {  // a larger value, or the first NaN
        top = x;
        at = i;
      }
    };
    for_slice<4>(row, lo, hi, one, [&](int i, const auto& w) {
      constexpr int N = sizeof(w) / 16, V = 16 / sizeof(T);
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 x = Two<T>::at(w[u], e / 2);
          one(i + u * kVfThreads * V + e, x.x);
          one(i + u * kVfThreads * V + e + 1, x.y);
        }
    });
    if (at >= 0) best = argmax_key(top, at);
  } else {
    // Elements two at a time: 2^((x - m) c), the sum in four parts.  (x c - m c
    // in one instruction would lose 2^-24 |m c|, much at low temperatures.)
    uint64_t sum[2] = {0ull, 0ull}, less = 0ull;
    const uint64_t c2 = pack2(make_float2(c, c));
    auto raise = [&](float t) {  // to a new maximum
      const float f = m == -INFINITY ? 0.f : exp2f((m - t) * c);
      l *= f;
      const uint64_t f2 = pack2(make_float2(f, f));
      sum[0] = mul2(sum[0], f2);
      sum[1] = mul2(sum[1], f2);
      m = t;
      less = pack2(make_float2(-t, -t));
    };
    auto one = [&](int, float x) {
      if (x == -INFINITY) return;
      if (x > m) raise(x);
      l += exp2f((x - m) * c);
    };
    for_slice<4>(row, lo, hi, one, [&](int, const auto& w) {
      constexpr int N = sizeof(w) / 16;
      const float t = Two<T>::largest(w);
      if (t > m) raise(t);
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < 8 / (int)sizeof(T); ++e) {
          const float2 y = unpack2(mul2(add2(pack2(Two<T>::at(w[u], e)), less), c2));
          sum[e & 1] = add2(sum[e & 1], pack2(make_float2(exp2_fast(y.x), exp2_fast(y.y))));
        }
    });
    const float2 s = unpack2(add2(sum[0], sum[1]));
    l += s.x + s.y;
  }
  if (greedy) {
    best = warp_max(best);
    if (lane == 0) s_k[warp] = best;
  } else {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
      join(m, l, m2, l2, c);
    }
    if (lane == 0) {
      s_m[warp] = m;
      s_l[warp] = l;
    }
  }
  __syncthreads();
  if (tid == 0) {
    Part out{-INFINITY, 0.f, draft, need, 0ull};
    for (int w = 0; w < kVfWarps; ++w) {
      if (greedy) out.key = s_k[w] > out.key ? s_k[w] : out.key;
      else join(out.m, out.l, s_m[w], s_l[w], c);
    }
    p.part[((int64_t)b * rows + k) * p.splits + blockIdx.x] = out;
    __threadfence();
    s_last = atomicAdd(&p.done[2 * b], 1u) == static_cast<unsigned>((used + 1) * p.splits - 1);
    if (s_last) p.done[2 * b] = 0u;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();

  // ---- the sequence's rows, a warp each: statistics, and whether the draft stands ----
  const int64_t* drafts = p.a.draft_tokens + (int64_t)b * p.a.drafts;
  for (int r = warp; r <= used; r += kVfWarps) {
    const Part* q = p.part + ((int64_t)b * rows + r) * p.splits;
    float rm = -INFINITY, rl = 0.f;
    unsigned long long rk = 0ull;
    const float draft_r = __ldcg(&q[0].draft), need_r = __ldcg(&q[0].need);
    for (int i = lane; i < p.splits; i += 32) {
      const float qm = __ldcg(&q[i].m), ql = __ldcg(&q[i].l);
      const unsigned long long qk = __ldcg(&q[i].key);
      rk = qk > rk ? qk : rk;
      if (!greedy) join(rm, rl, qm, ql, c);
    }
    rk = warp_max(rk);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, rm, o), l2 = __shfl_xor_sync(0xffffffffu, rl, o);
      join(rm, rl, m2, l2, c);
    }
    if (lane == 0) {
      s_rm[r] = rm;
      s_rl[r] = rl;
      s_arg[r] = key_index(rk);
      if (r < used)  // an infinite need (and NaN) never stands
        s_ok[r] = greedy ? drafts[r] == (int64_t)key_index(rk) : need_r < exp2f((draft_r - rm) * c) / rl;
    }
  }
  __syncthreads();
  int n = 0;
  while (n < used && s_ok[n]) ++n;
  if (tid < rows) {
    const int64_t at = (int64_t)b * rows + tid;
    if (tid < n) p.a.tokens[at] = drafts[tid];
    else p.a.tokens[at] = tid == n && greedy ? (int64_t)s_arg[n] : -1;
  }
  const Choice ch{s_rm[n], c, 1.f / s_rl[n], greedy ? -1 : n, n < used};
  if (tid == 0) {
    p.a.accepted[b] = n;
    p.choice[b] = ch;
  }
  if (!ALONE || greedy) return;
  // a short row: drawn here, and not in a launch of its own
  unsigned long long won = race_row<T>(p, b, ch, ch.residual, s_k);
  if (!won && ch.residual) won = race_row<T>(p, b, ch, false, s_k);
  if (tid == 0) p.a.tokens[(int64_t)b * rows + n] = won ? (int64_t)key_index(won) : -1;
}

template <class T>
__global__ void __launch_bounds__(kVfThreads, kVfResident) verify_race_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ unsigned long long s_k[kVfWarps];
  __shared__ bool s_last;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, tid = threadIdx.x;
  const Choice ch = p.choice[b];
  if (ch.row < 0) return;
  const int per = (p.a.vocab + p.race_splits - 1) / p.race_splits;
  const int lo = min((int)blockIdx.x * per, p.a.vocab), hi = min(lo + per, p.a.vocab);
  const unsigned long long key = race_slice<T>(p, b, ch, lo, hi, ch.residual, s_k);
  if (tid == 0) {
    if (key) atomicMax(&p.key[b], key);
    __threadfence();
    s_last = atomicAdd(&p.done[2 * b + 1], 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  unsigned long long won = take_key(&p.key[b], s_k);
  // Nothing left of p - q anywhere (q is not normalised): the draw is from p,
  // by this CTA alone, since it hardly occurs.
  if (!won && ch.residual) won = race_row<T>(p, b, ch, false, s_k);
  if (tid == 0) {
    p.a.tokens[(int64_t)b * (p.a.drafts + 1) + ch.row] = won ? (int64_t)key_index(won) : -1;
    p.done[2 * b + 1] = 0u;
  }
}

int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

struct VfPlan {
  int64_t choice_off, part_off, bytes;
};

tp_status plan_verify(int64_t batch, int64_t drafts, int64_t vocab, VfPlan* pl) {
  if (batch < 1 || drafts < 0 || vocab < 1) return fail(TP_ERR_ARG, "tp_verify_drafts: bad sizes");
  if (drafts + 1 > kVfMaxRows) return fail(TP_ERR_UNSUPPORTED, "tp_verify_drafts: more than %d drafts", kVfMaxRows - 1);
  if (batch * (drafts + 1) > 65535) return fail(TP_ERR_UNSUPPORTED, "tp_verify_drafts: more than 65535 rows");
  if (vocab > 0x7FFFFFF0) return fail(TP_ERR_UNSUPPORTED, "tp_verify_drafts: vocabulary too large");
  // counters and keys of up to 65535 sequences at a fixed place, so that calls
  // of other sizes find them zero
  pl->choice_off = round256(65536 * (8 + 2 * 4));
  pl->part_off = pl->choice_off + round256(batch * (int64_t)sizeof(Choice));
  pl->bytes = pl->part_off + round256(batch * (drafts + 1) * kVfMaxSplits * (int64_t)sizeof(Part));
  return TP_OK;
}

template <class T>
tp_status launch_verify(VerifyParams& p, cudaStream_t st) {
  int sms = 0;
  tp_status s = device_sms(&sms);
  if (s != TP_OK) return s;
  const int rows = p.a.batch * (p.a.drafts + 1);
  // slices: all CTAs resident at once, 4096 elements each at
  // least (16 a thread): more and smaller ones cost more in the joins
  auto slices = [&](int n) {
    const int64_t most = (p.a.vocab + 4095) / 4096;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kVfResident * sms / n, most, kVfMaxSplits})));
  };
  const bool alone = p.a.vocab <= kVfAlone;
  p.splits = slices(rows);
  p.race_splits = slices(p.a.batch);
  s = launch_early(alone ? verify_rows_kernel<T, true> : verify_rows_kernel<T, false>, dim3(p.splits, rows), kVfThreads, 0,
                   st, "verify_rows launch", p);
  if (s != TP_OK || !p.a.temperature || alone) return s;  // (all greedy: the tokens are written)
  return launch_early(verify_race_kernel<T>, dim3(p.race_splits, p.a.batch), kVfThreads, 0, st, "verify_race launch", p);
}

}  // namespace

extern "C" {

TP_API int64_t tp_verify_workspace_bytes(int batch, int drafts, int vocab) {
  VfPlan pl;
  const tp_status s = plan_verify(batch, drafts, vocab, &pl);
  return s == TP_OK ? pl.bytes : -static_cast<int64_t>(s);
}

TP_API tp_status tp_verify_drafts(const tp_verify_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!args) return fail(TP_ERR_ARG, "tp_verify_drafts: null arguments");
  const tp_verify_args& a = *args;
  VfPlan pl;
  const tp_status s = plan_verify(a.batch, a.drafts, a.vocab, &pl);
  if (s != TP_OK) return s;
  if (!a.logits || !a.accepted || !a.tokens || (a.drafts && !a.draft_tokens) ||
      (a.temperature && (!a.noise || (a.drafts && !a.uniforms))))
    return fail(TP_ERR_ARG, "tp_verify_drafts: null pointer");
  if (!valid_dtype(a.dtype)) return fail(TP_ERR_ARG, "tp_verify_drafts: bad dtype %d", a.dtype);
  if (!aligned(a.logits, a.dtype == TP_F32 ? 4 : 2))
    return fail(TP_ERR_ALIGN, "tp_verify_drafts: logits are not aligned to their elements");
  if (!workspace || workspace_bytes < pl.bytes || !aligned(workspace, 256))
    return fail(TP_ERR_WORKSPACE, "tp_verify_drafts: workspace missing, not 256-byte aligned or smaller than %lld bytes",
                (long long)pl.bytes);
  VerifyParams p{};
  p.a = a;
  auto* ws = static_cast<unsigned char*>(workspace);
  p.key = reinterpret_cast<unsigned long long*>(ws);
  p.done = reinterpret_cast<unsigned*>(ws + 65536 * 8);
  p.choice = reinterpret_cast<Choice*>(ws + pl.choice_off);
  p.part = reinterpret_cast<Part*>(ws + pl.part_off);
  cudaStream_t st = as_stream(stream);
  if (a.dtype == TP_F16) return launch_verify<__half>(p, st);
  if (a.dtype == TP_BF16) return launch_verify<__nv_bfloat16>(p, st);
  return launch_verify<float>(p, st);
}

}  // extern "C"
