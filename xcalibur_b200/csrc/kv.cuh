// What the attention-side kernels share: the cache as a kernel sees it, its argument checks, small device helpers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/xcb_attn.h"

namespace xcb {

constexpr int kMaxDevices = 64;

inline int kv_elem_bytes(int dtype) { return dtype == XCB_DTYPE_E4M3 ? 1 : 2; }

// Division by a run-time constant (page size, group size) as a multiply: exact for 0 <= n < 2^31.
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return FastDiv{d, (uint32_t)((((1ull << s) - d) << 32) / d + 1), s};
}
__device__ __forceinline__ int fdiv(int n, FastDiv f) {
  return (int)((__umulhi(f.mul, (uint32_t)n) + (uint32_t)n) >> f.shift);
}

// One layer of the cache for a kernel.
struct KvLayer {
  uint8_t* k;           // keys of the layer; values lie `plane` bytes further
  int64_t plane;
  const int32_t* table;
  const int32_t* lens;
  const float* k_scale;
  const float* v_scale;
  int32_t* status;
  int32_t num_pages, kv_heads, page_size, max_seqs, max_pages;
  FastDiv page_div;
};

inline bool kv_aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// Sizes whose products stay inside the index arithmetic of the kernels: a row of a page table and a sequence's
// length fit 31 bits, byte offsets are 64-bit.
inline int kv_check(const XcbKvCache* c) {
  if (!c || !c->kv || !c->page_table || !c->seq_lens || !c->status) return XCB_ERR_INVALID_ARG;
  if (c->layers <= 0 || c->num_pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0 || c->head_dim <= 0 ||
      c->max_seqs <= 0 || c->max_pages <= 0)
    return XCB_ERR_INVALID_ARG;
  if (c->dtype != XCB_DTYPE_BF16 && c->dtype != XCB_DTYPE_F16 && c->dtype != XCB_DTYPE_E4M3) return XCB_ERR_INVALID_ARG;
  if (c->head_dim > 256 || (c->head_dim * kv_elem_bytes(c->dtype)) % 16) return XCB_ERR_UNSUPPORTED;
  if (c->page_size > 65536 || c->kv_heads > 65536) return XCB_ERR_UNSUPPORTED;
  if ((int64_t)c->max_pages * c->page_size >= (1ll << 31) - 65536) return XCB_ERR_UNSUPPORTED;
  if ((int64_t)c->max_pages * c->max_seqs >= 1ll << 31 || c->num_pages > 1 << 30) return XCB_ERR_UNSUPPORTED;
  if (!kv_aligned(c->kv, 16) || !kv_aligned(c->page_table, 4) || !kv_aligned(c->seq_lens, 4) ||
      !kv_aligned(c->refcounts, 4) || !kv_aligned(c->status, 4) || !kv_aligned(c->k_scale, 4) ||
      !kv_aligned(c->v_scale, 4))
    return XCB_ERR_INVALID_ARG;
  return XCB_OK;
}

inline KvLayer kv_layer(const XcbKvCache* c, int layer) {
  KvLayer l;
  l.plane = (int64_t)c->num_pages * c->kv_heads * c->page_size * c->head_dim * kv_elem_bytes(c->dtype);
  l.k = (uint8_t*)c->kv + 2 * l.plane * layer;
  l.table = c->page_table;
  l.lens = c->seq_lens;
  const bool scaled = c->dtype == XCB_DTYPE_E4M3;
  l.k_scale = scaled ? c->k_scale : nullptr;
  l.v_scale = scaled ? c->v_scale : nullptr;
  l.status = c->status;
  l.num_pages = c->num_pages;
  l.kv_heads = c->kv_heads;
  l.page_size = c->page_size;
  l.max_seqs = c->max_seqs;
  l.max_pages = c->max_pages;
  l.page_div = fast_div((uint32_t)c->page_size);
  return l;
}

// Streaming multiprocessors of the current device (looked up once per device), or 0 on a CUDA error.
inline int sm_count() {
  static int cached[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < kMaxDevices && cached[dev]) return cached[dev];
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < kMaxDevices) cached[dev] = n;
  return n;
}

// ------------------------------------------------------------------------------------------------ element types
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&r);
}

}  // namespace xcb
