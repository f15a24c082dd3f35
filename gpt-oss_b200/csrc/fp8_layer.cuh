// What the operators of an FP8 expert layer (routed_rows.cu, fp8_quant.cu, fp8_gemm_sm100.cu) share: argument checks of
// their C entries, and loads and stores of the three row types.
#pragma once
#include <cstdarg>
#include <cstdio>

#include "moe_internal.cuh"

namespace moe {

constexpr int kScaleBlock = 128;   // columns (of weights also rows) that share a scale

// Records the message in the handle and returns the code.
inline int op_fail(moe_ctx *c, int code, const char *fmt, ...) {
  char buf[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  try { c->err = buf; } catch (...) {}   // out of host memory: the code alone has to do
  return code;
}

inline int dtype_size(int dtype) { return dtype == MOE_F32 ? 4 : dtype == MOE_BF16 || dtype == MOE_F16 ? 2 : 0; }
inline bool aligned_to(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Makes the handle's device current; every entry calls it after its own checks.
inline int use_device(moe_ctx *c, const char *who) {
  int current = -1;
  if (cudaGetDevice(&current) == cudaSuccess && current == c->cfg.device) return MOE_OK;
  const cudaError_t e = cudaSetDevice(c->cfg.device);
  return e == cudaSuccess ? MOE_OK : op_fail(c, MOE_ERR_CUDA, "%s: cudaSetDevice(%d): %s", who, c->cfg.device, cudaGetErrorString(e));
}
// Dynamic shared memory above 48 KB has to be asked for, once per kernel and device: bits of moe_ctx::smem_asked.
enum : unsigned { kSmemGemm16 = 1u, kSmemGemm64 = 2u, kSmemGemm128 = 4u, kSmemGemmWide = 8u, kSmemGemmWideSplit = 16u, kSmemGroup = 32u };
inline cudaError_t allow_smem(moe_ctx *c, const void *kernel, int bytes, unsigned bit) {
  if (c->smem_asked & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) c->smem_asked |= bit;
  return e;
}
inline int launched(moe_ctx *c, const char *who, cudaError_t e) {
  if (e != cudaSuccess) {
    (void)cudaGetLastError();   // a refused launch is not left for the next call to find
    return op_fail(c, MOE_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  }
  c->launches += 1;
  return MOE_OK;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void store_as(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_as(__half *p, float v) { *p = __float2half_rn(v); }

}  // namespace moe
