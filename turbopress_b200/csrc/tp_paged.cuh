// Shared by the paged-cache kernels: argument checks of a cache, slot lookup.
#pragma once

#include "tp_common.cuh"

namespace tp {

constexpr int64_t kMaxSlots = int64_t(1) << 30;  // per sequence: slot numbers are 32-bit

// Host checks of what is not device data.
inline tp_status check_cache(const tp_paged_cache* c, const char* who) {
  if (!c || !c->k_pages || !c->v_pages || !c->block_table || !c->lengths)
    return fail(TP_ERR_ARG, "%s: null cache pointer", who);
  if (c->batch < 1 || c->kv_heads < 1 || c->max_pages < 1 || c->num_pages < 0 || c->table_stride < c->max_pages)
    return fail(TP_ERR_ARG, "%s: bad cache sizes", who);
  if (c->page_size < 1 || (c->page_size & (c->page_size - 1)))
    return fail(TP_ERR_UNSUPPORTED, "%s: page_size %d is not a power of two", who, c->page_size);
  if ((int64_t)c->max_pages * c->page_size > kMaxSlots)
    return fail(TP_ERR_UNSUPPORTED, "%s: more than %lld slots per sequence", who, (long long)kMaxSlots);
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8)
    return fail(TP_ERR_UNSUPPORTED, "%s: head_dim %d is not a multiple of 8 up to 256", who, c->head_dim);
  if (c->dtype != TP_F16 && c->dtype != TP_BF16)
    return fail(TP_ERR_UNSUPPORTED, "%s: pages must be fp16 or bf16", who);
  if (c->page_stride < 0 || c->head_stride < 0 || c->token_stride < 0)
    return fail(TP_ERR_ARG, "%s: negative cache stride", who);
  if (!aligned(c->k_pages, 16) || !aligned(c->v_pages, 16) || c->page_stride % 8 || c->head_stride % 8 ||
      c->token_stride % 8)
    return fail(TP_ERR_ALIGN, "%s: pages and their strides must be multiples of 16 bytes", who);
  return TP_OK;
}

inline int log2_int(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}

// Multiprocessors of the current device (queried once per device).
inline tp_status device_sms(int* sms) {
  static int cached[64];
  int dev = 0;
  TP_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(TP_ERR_UNSUPPORTED, "device index %d out of range", dev);
  int n = __atomic_load_n(&cached[dev], __ATOMIC_RELAXED);
  if (!n) {
    TP_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "SM count");
    __atomic_store_n(&cached[dev], n, __ATOMIC_RELAXED);
  }
  *sms = n;
  return TP_OK;
}

// Launch that may begin while the kernel before it in the stream ends: every
// kernel launched this way waits (griddepcontrol.wait) for that kernel's
// completion before its first access to memory that others write.
template <class... Params, class... Args>
inline tp_status launch_early(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream,
                              const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...), what);
  return clear_ok();
}

// N neighbouring elements, accessed 16 bytes at a time at most.
template <class T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Pack {
  T v[VEC];
};

// Element types of the kernels.
template <class T>
struct Elem;
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};

}  // namespace tp
