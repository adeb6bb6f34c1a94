// Shared by the paged serving operators (rope_append.cu, paged_attn.cu, copy_pages.cu, sample.cu):
// element conversions, the checks of a page pool's descriptor, and how a refusal is reported.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/mllm.h"

namespace mllm {

void set_global_error(const char* msg);  // engine.cu: message for mllm_last_error(NULL)

namespace paged {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline bool is_float_kind(int dt) { return dt == MLLM_DTYPE_F32 || dt == MLLM_DTYPE_F16 || dt == MLLM_DTYPE_BF16; }
inline int esize(int dt) { return dt == MLLM_DTYPE_F32 ? 4 : 2; }

inline int refuse(int code, const char* why) {
  try {
    set_global_error(why);
  } catch (...) {  // the message did not fit memory: the code still says what happened
  }
  return code;
}

// MLLM_OK, or the status of the first thing wrong with a pool's descriptor.
inline int check_kv(const mllm_paged_kv* kv) {
  if (!kv) return refuse(MLLM_ERR_ARG, "paged cache: null descriptor");
  if (!is_float_kind(kv->dtype)) return refuse(MLLM_ERR_UNSUPPORTED, "paged cache: dtype must be f32, f16 or bf16");
  if (!kv->k || !kv->v) return refuse(MLLM_ERR_ARG, "paged cache: null pool");
  if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8)
    return refuse(MLLM_ERR_UNSUPPORTED, "paged cache: head_dim must be a multiple of 8, 8 to 256");
  if (kv->n_pages < 1 || kv->page_len < 1 || kv->n_kv_heads < 1)
    return refuse(MLLM_ERR_ARG, "paged cache: non-positive page count, page length or kv heads");
  if (kv->page_stride < kv->head_dim || kv->head_stride < kv->head_dim || kv->pos_stride < kv->head_dim)
    return refuse(MLLM_ERR_ARG, "paged cache: a stride is below head_dim");
  const int per = 16 / esize(kv->dtype);
  if (((uintptr_t)kv->k & 15) || ((uintptr_t)kv->v & 15) || kv->page_stride % per || kv->head_stride % per ||
      kv->pos_stride % per)
    return refuse(MLLM_ERR_ARG, "paged cache: pools and strides must be 16-byte aligned");
  return MLLM_OK;
}

inline int launched(const char* what) {
  return cudaGetLastError() == cudaSuccess ? MLLM_OK : refuse(MLLM_ERR_CUDA, what);
}

}  // namespace paged
}  // namespace mllm
