// Rows and weights -> e4m3 codes with one fp32 scale per 128 columns (moe_quantize_fp8) or per 128 x 128 block
// (moe_quantize_fp8_blocks).
//
// Of a block with the largest magnitude m (at least 2^-96, so that 448 / m is finite):  scale = m / 448,
// code = e4m3(v * (448 / m)), each operation rounded to nearest; 448 is the largest e4m3 magnitude.  Only finite values
// count towards m: a NaN becomes a NaN code, an infinity +-448, and neither takes its block along.
//
// Rows may pass through a gated activation on the way in (what lies between the two products of an expert), and may be
// written at several places (the rows of a token's experts): the values are read and converted once.
#include <cuda_fp8.h>

#include "fp8_layer.cuh"

namespace moe {

constexpr float kFp8Max = 448.f;
constexpr float kAmaxFloor = 1.262177448e-29f;   // 2^-96
constexpr int kQuantLanes = 16;                  // lanes that share a block, eight columns each

__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int off = kQuantLanes / 2; off; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
__device__ __forceinline__ uint2 encode8(const float (&v)[8], float inv) {
  uint32_t p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
}

// gate * sigmoid(alpha * gate) * (up + 1) with the gate clamped from above and up on both sides (ACT_SWIGLU), or
// gate * sigmoid(gate) * up (ACT_SILU_MUL).  Comparisons, not fminf: a NaN stays one.
template <int kAct>
__device__ __forceinline__ float gated(float gate, float up, float limit, float alpha) {
  if (kAct == MOE_ACT_SWIGLU) {
    gate = gate > limit ? limit : gate;
    up = up > limit ? limit : up < -limit ? -limit : up;
    return gate / (1.f + expf(-alpha * gate)) * (up + 1.f);
  }
  return gate / (1.f + expf(-gate)) * up;
}

template <class T, int kAct>
__global__ void __launch_bounds__(256)
quantize_fp8_kernel(const T *x, size_t ld_x, int rows, int cols, float limit, float alpha, const int *pair_row, int fanout, int out_rows,
                    const int *n_rows, uint8_t *codes, size_t ld_codes, float *scales, size_t ld_scales) {
  const int lane16 = threadIdx.x % kQuantLanes;
  const int n_blocks = (cols + kScaleBlock - 1) / kScaleBlock;
  const size_t unit = (static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x) / kQuantLanes;
  const size_t row = unit / n_blocks;
  const int kb = static_cast<int>(unit % n_blocks), c0 = kb * kScaleBlock + lane16 * 8;
  int live = rows;
  if (n_rows != nullptr) live = min(live, *n_rows);
  const bool on = row < static_cast<size_t>(max(live, 0));
  float v[8], m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = 0.f;
    if (on && c0 + i < cols) {
      const T *src = x + row * ld_x;
      if (kAct == MOE_ACT_NONE) v[i] = to_f32(src[c0 + i]);
      else if (kAct == MOE_ACT_SWIGLU) v[i] = gated<kAct>(to_f32(src[2 * (c0 + i)]), to_f32(src[2 * (c0 + i) + 1]), limit, alpha);
      else v[i] = gated<kAct>(to_f32(src[c0 + i]), to_f32(src[cols + c0 + i]), limit, alpha);
    }
    const float a = fabsf(v[i]);
    if (a < __int_as_float(0x7f800000)) m = fmaxf(m, a);
  }
  m = fmaxf(half_warp_max(m), kAmaxFloor);
  if (!on) return;
  const uint2 q = encode8(v, __fdiv_rn(kFp8Max, m));
  for (int j = 0; j < fanout; ++j) {
    const int r = pair_row != nullptr ? pair_row[row * fanout + j] : static_cast<int>(row);
    if (r < 0 || r >= out_rows) continue;
    uint8_t *dst = codes + static_cast<size_t>(r) * ld_codes + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < cols) dst[i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
    if (lane16 == 0) scales[static_cast<size_t>(r) * ld_scales + kb] = __fdiv_rn(m, kFp8Max);
  }
}

// A CTA per 128 x 128 block: half-warp h takes rows h, h + 16, ... of it.
template <class T>
__global__ void __launch_bounds__(256)
quantize_fp8_blocks_kernel(const T *w, size_t ld_w, int rows, int cols, uint8_t *codes, size_t ld_codes, float *scales) {
  __shared__ float s_max[8];
  const int lane16 = threadIdx.x % kQuantLanes, half = threadIdx.x / kQuantLanes;
  const int r0 = blockIdx.y * kScaleBlock, c0 = blockIdx.x * kScaleBlock + lane16 * 8;
  const size_t mat = blockIdx.z;
  const T *src = w + mat * rows * ld_w;
  float v[8][8], m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + half + 16 * j;
      v[j][i] = r < rows && c0 + i < cols ? to_f32(src[static_cast<size_t>(r) * ld_w + c0 + i]) : 0.f;
      const float a = fabsf(v[j][i]);
      if (a < __int_as_float(0x7f800000)) m = fmaxf(m, a);
    }
  for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int i = 0; i < 8; ++i) m = fmaxf(m, s_max[i]);
  m = fmaxf(m, kAmaxFloor);
  const float inv = __fdiv_rn(kFp8Max, m);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = r0 + half + 16 * j;
    if (r >= rows) continue;
    const uint2 q = encode8(v[j], inv);
    uint8_t *dst = codes + (mat * rows + r) * ld_codes + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < cols) dst[i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
  if (threadIdx.x == 0) scales[(mat * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = __fdiv_rn(m, kFp8Max);
}

}  // namespace moe

using namespace moe;

extern "C" {

int moe_quantize_fp8(moe_handle c, const void *x_dev, int dtype, long long ld_x, int rows, int cols, int act, float limit, float alpha,
                     const int *pair_row_dev, int fanout, int out_rows, const int *n_rows_dev, uint8_t *codes_dev, long long ld_codes,
                     float *scales_dev, long long ld_scales, void *stream) {
  if (!c) return MOE_ERR_INVALID;
  const int size = dtype_size(dtype);
  if (act != MOE_ACT_NONE && act != MOE_ACT_SWIGLU && act != MOE_ACT_SILU_MUL) return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: activation %d", act);
  if (act == MOE_ACT_SWIGLU && !(limit >= 0.f && alpha - alpha == 0.f))
    return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: limit %g, alpha %g", static_cast<double>(limit), static_cast<double>(alpha));
  const long long n_blocks = (static_cast<long long>(cols) + kScaleBlock - 1) / kScaleBlock, wide = act == MOE_ACT_NONE ? cols : 2ll * cols;
  if (!size || rows < 0 || cols < 1 || ld_x < wide || ld_codes < cols || ld_scales < n_blocks)
    return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: dtype %d, %d rows of %d columns, strides %lld, %lld, %lld", dtype, rows, cols, ld_x, ld_codes, ld_scales);
  if (fanout < 1 || out_rows < 0 || static_cast<long long>(rows) * fanout > 0x7fffffffll || (!pair_row_dev && (fanout != 1 || out_rows < rows)))
    return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: %d rows to %d places each among %d%s", rows, fanout, out_rows, pair_row_dev ? "" : ", without a map");
  if (rows == 0 || out_rows == 0) return MOE_OK;
  if (!x_dev || !codes_dev || !scales_dev) return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: null tensor");
  if (!aligned_to(x_dev, size) || !aligned_to(pair_row_dev, 4) || !aligned_to(n_rows_dev, 4) || !aligned_to(scales_dev, 4))
    return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: a tensor is not aligned to its elements");
  if (int rc = use_device(c, "moe_quantize_fp8")) return rc;
  const size_t threads = static_cast<size_t>(rows) * n_blocks * kQuantLanes, grid = (threads + 255) / 256;
  if (grid > 0x7fffffffu) return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: %d rows of %d columns in one call", rows, cols);
  auto go = [&](auto type, auto kernel_of) {
    using T = decltype(type);
    kernel_of<<<static_cast<unsigned>(grid), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T *>(x_dev), static_cast<size_t>(ld_x), rows, cols, limit, alpha, pair_row_dev, fanout, out_rows, n_rows_dev,
        codes_dev, static_cast<size_t>(ld_codes), scales_dev, static_cast<size_t>(ld_scales));
    return cudaGetLastError();
  };
  auto by_act = [&](auto type) {
    using T = decltype(type);
    return act == MOE_ACT_NONE     ? go(type, quantize_fp8_kernel<T, MOE_ACT_NONE>)
           : act == MOE_ACT_SWIGLU ? go(type, quantize_fp8_kernel<T, MOE_ACT_SWIGLU>)
                                   : go(type, quantize_fp8_kernel<T, MOE_ACT_SILU_MUL>);
  };
  return launched(c, "moe_quantize_fp8", dtype == MOE_F32 ? by_act(float()) : dtype == MOE_BF16 ? by_act(__nv_bfloat16()) : by_act(__half()));
}

int moe_quantize_fp8_blocks(moe_handle c, const void *w_dev, int dtype, long long ld_w, int n_mats, int rows, int cols, uint8_t *codes_dev,
                            long long ld_codes, float *scales_dev, void *stream) {
  if (!c) return MOE_ERR_INVALID;
  const int size = dtype_size(dtype);
  if (!size || n_mats < 0 || n_mats > 65535 || rows < 1 || rows > 65535 * kScaleBlock || cols < 1 || ld_w < cols || ld_codes < cols)
    return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8_blocks: dtype %d, %d matrices of %d x %d, strides %lld, %lld", dtype, n_mats, rows, cols, ld_w, ld_codes);
  if (n_mats == 0) return MOE_OK;
  if (!w_dev || !codes_dev || !scales_dev) return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8_blocks: null tensor");
  if (!aligned_to(w_dev, size) || !aligned_to(scales_dev, 4)) return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8_blocks: a tensor is not aligned to its elements");
  if (int rc = use_device(c, "moe_quantize_fp8_blocks")) return rc;
  const dim3 grid((cols - 1) / kScaleBlock + 1, (rows - 1) / kScaleBlock + 1, n_mats);
  auto go = [&](auto type) {
    using T = decltype(type);
    quantize_fp8_blocks_kernel<T><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T *>(w_dev), static_cast<size_t>(ld_w), rows, cols, codes_dev, static_cast<size_t>(ld_codes), scales_dev);
    return cudaGetLastError();
  };
  return launched(c, "moe_quantize_fp8_blocks", dtype == MOE_F32 ? go(float()) : dtype == MOE_BF16 ? go(__nv_bfloat16()) : go(__half()));
}

}  // extern "C"
