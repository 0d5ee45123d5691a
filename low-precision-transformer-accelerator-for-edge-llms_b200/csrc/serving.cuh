// serving.cuh -- element types and addressing shared by the paged-cache and
// log-probability operators (paged.cu, paged_attn.cu, logprobs.cu).
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/tl_api.h"
#include "common.cuh"
#include "once.cuh"

namespace tl {

inline tl_status cuda_status(cudaError_t e) { return e == cudaSuccess ? TL_OK : TL_ERR_CUDA; }

// Launches with programmatic serialization: a kernel's CTAs may be placed while
// the kernel before it drains. Every thread of such a kernel calls pdl_begin()
// before it touches global memory. Calls in a row, with and without, when it
// came in: append of 16 prompts 32.2 and 34.2 us, attention of 64 contexts over
// INT8 19.0 and 20.5, log probabilities of 2048 rows 53.0 and 53.7.
template <typename... P, typename... A>
tl_status launch_serving(void (*kernel)(P...), unsigned grid, int threads, size_t smem, int cluster, cudaStream_t s,
                         const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args...));
}
// Raises a kernel's limit of dynamic shared memory on the current device.
template <typename K>
bool allow_shared(K* kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}
// All that the kernels before have written is there; from here on the next one
// may be placed (not earlier: what it must not overtake has ended by then).
TL_DEV void pdl_begin() {
  pdl_wait();
  pdl_launch_dependents();
}

inline bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int dtype_bytes(int32_t dt) { return dt == TL_F32 ? 4 : dt == TL_I8 ? 1 : 2; }
inline bool is_float_dtype(int32_t dt) { return dt == TL_F32 || dt == TL_BF16 || dt == TL_F16; }

template <typename T>
TL_DEV float to_f32(T x);
template <>
TL_DEV float to_f32<float>(float x) { return x; }
template <>
TL_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
TL_DEV float to_f32<__half>(__half x) { return __half2float(x); }

template <typename T>
TL_DEV T from_f32(float x);
template <>
TL_DEV float from_f32<float>(float x) { return x; }
template <>
TL_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
TL_DEV __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Division of a position by the page size, which is any positive number: for
// n < 2^31 and 1 <= d < 2^31 with s = ceil(log2 d), m = floor(2^(31+s) / d) + 1
// fits 33 bits at most 2^32 and floor(n m / 2^(31+s)) = floor(n / d) (Granlund
// and Montgomery, "Division by invariant integers using multiplication").
struct PageDiv {
  uint32_t d;
  uint32_t shift;
  uint64_t mul;
};
inline PageDiv page_div(int32_t d) {
  PageDiv r;
  r.d = static_cast<uint32_t>(d);
  uint32_t s = 0;
  while ((1ull << s) < r.d) ++s;
  r.shift = 31 + s;
  r.mul = (1ull << r.shift) / r.d + 1;
  return r;
}
TL_DEV uint32_t div_page(uint32_t n, const PageDiv& p) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * p.mul) >> p.shift);
}

// The pool and the table as the kernels see them.
struct PagedView {
  void* k;
  void* v;
  float* ks;
  float* vs;
  int32_t pages, hkv, ps;
  PageDiv div;
  const int32_t* table;
  int32_t n_seqs, max_pages;
  int64_t table_stride;
};

// Row index (in rows of head_dim elements) of kv head 0 of position p of
// sequence s, or -1 where none exists; head h is h * ps rows further.
TL_DEV int64_t paged_row(const PagedView& c, int s, int p) {
  if (s < 0 || s >= c.n_seqs || p < 0) return -1;
  const uint32_t pg = div_page(static_cast<uint32_t>(p), c.div);
  if (pg >= static_cast<uint32_t>(c.max_pages)) return -1;
  const int page = c.table[static_cast<int64_t>(s) * c.table_stride + pg];
  if (page < 0 || page >= c.pages) return -1;
  return static_cast<int64_t>(page) * c.hkv * c.ps + (static_cast<uint32_t>(p) - pg * c.div.d);
}

// Checks shared by the paged entry points; fills the view.
tl_status paged_view(const tl_paged_kv* cache, const int32_t* table, int32_t n_seqs, int32_t max_pages,
                     int64_t table_stride, PagedView* out);

}  // namespace tl
