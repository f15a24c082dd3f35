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
// gate * sigmoid(gate) * up (ACT_SILU_MUL).  Comparisons, not fminf: a NaN stays one.  The fast exponential and quotient are off
// by 2^-20 at |alpha * gate| = 8 and 2^-18 at 32, next to a code's half step of 2^-4: with expf and a rounded division 17.7 M
// values took 46 us, the instructions being the bound, with these HBM is.
template <int kAct>
__device__ __forceinline__ float gated(float gate, float up, float limit, float alpha) {
  if (kAct == MOE_ACT_SWIGLU) {
    gate = gate > limit ? limit : gate;
    up = up > limit ? limit : up < -limit ? -limit : up;
    return __fdividef(gate, 1.f + __expf(-alpha * gate)) * (up + 1.f);
  }
  return __fdividef(gate, 1.f + __expf(-gate)) * up;
}

// Eight consecutive values of a row, of which `n` (any number) exist; wide: 16-byte loads.
template <class T>
__device__ __forceinline__ void read8(const T *p, int n, bool wide, float (&v)[8]) {
  if (wide && n >= 8) {
    uint4 raw[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) raw[i] = reinterpret_cast<const uint4 *>(p)[i];
    const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}
__device__ __forceinline__ void write8(uint8_t *p, int n, bool wide, uint2 q) {
  if (wide && n >= 8) {
    *reinterpret_cast<uint2 *>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}
__device__ __forceinline__ float finite_max(const float (&v)[8], float m) {
  float a = m;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[i]));   // drops a NaN
  if (a < __int_as_float(0x7f800000)) return a;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (fabsf(v[i]) < __int_as_float(0x7f800000)) m = fmaxf(m, fabsf(v[i]));
  return m;
}

// Sixteen lanes per block of 128 columns, eight columns each; the (row, block) pairs of a call are dealt to the half-warps.
constexpr int kQuantThreads = 256, kQuantHalves = kQuantThreads / kQuantLanes;

template <class T, int kAct>
__global__ void __launch_bounds__(kQuantThreads)
quantize_fp8_kernel(const T *x, size_t ld_x, int rows, int cols, unsigned n_blocks, float limit, float alpha, const int *pair_row, int fanout,
                    int out_rows, const int *n_rows, uint8_t *codes, size_t ld_codes, float *scales, size_t ld_scales, int wide_in, int wide_out) {
  grid_dep_sync();
  const int lane16 = threadIdx.x % kQuantLanes;
  int live = rows;
  if (n_rows != nullptr) live = max(min(live, *n_rows), 0);
  const unsigned units = static_cast<unsigned>(live) * n_blocks;      // (row, block) pairs; the host bounds rows * n_blocks
  const unsigned stride = gridDim.x * kQuantHalves;
  for (unsigned unit = blockIdx.x * kQuantHalves + threadIdx.x / kQuantLanes; ; unit += stride) {
    // (the two halves of a warp leave together: shuffles are the whole warp's)
    const bool on = unit < units;
    if (!__any_sync(0xffffffffu, on)) break;
    const unsigned row = on ? unit / n_blocks : 0, kb = unit - row * n_blocks;
    const int c0 = static_cast<int>(kb) * kScaleBlock + lane16 * 8, n = on ? cols - c0 : 0;
    const T *src = x + static_cast<size_t>(row) * ld_x;
    float v[8];
    if (kAct == MOE_ACT_NONE) {
      read8(src + c0, n, wide_in, v);
    } else {
      float a[8], b[8];
      if (kAct == MOE_ACT_SWIGLU) {
        read8(src + 2 * c0, 2 * n, wide_in, a);
        read8(src + 2 * c0 + 8, 2 * n - 8, wide_in, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = gated<kAct>(a[2 * i], a[2 * i + 1], limit, alpha);
          v[i + 4] = gated<kAct>(b[2 * i], b[2 * i + 1], limit, alpha);
        }
      } else {
        read8(src + c0, n, wide_in, a);
        read8(src + cols + c0, n, wide_in, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = gated<kAct>(a[i], b[i], limit, alpha);
      }
    }
    const float m = half_warp_max(finite_max(v, kAmaxFloor));
    if (!on) continue;
    const uint2 q = encode8(v, __fdiv_rn(kFp8Max, m));
    const float scale = __fdiv_rn(m, kFp8Max);
    for (int j = 0; j < fanout; ++j) {
      const int r = pair_row != nullptr ? pair_row[static_cast<size_t>(row) * fanout + j] : static_cast<int>(row);
      if (r < 0 || r >= out_rows) continue;
      write8(codes + static_cast<size_t>(r) * ld_codes + c0, n, wide_out, q);
      if (lane16 == 0) scales[static_cast<size_t>(r) * ld_scales + kb] = scale;
    }
  }
}

// A CTA per 128 x 128 block: half-warp h takes rows h, h + 16, ... of it.
template <class T>
__global__ void __launch_bounds__(256)
quantize_fp8_blocks_kernel(const T *w, size_t ld_w, int rows, int cols, uint8_t *codes, size_t ld_codes, float *scales, int wide_in, int wide_out) {
  __shared__ float s_max[8];
  grid_dep_sync();
  const int lane16 = threadIdx.x % kQuantLanes, half = threadIdx.x / kQuantLanes;
  const int r0 = blockIdx.y * kScaleBlock, c0 = blockIdx.x * kScaleBlock + lane16 * 8, n = cols - c0;
  const size_t mat = blockIdx.z;
  const T *src = w + mat * rows * ld_w;
  float v[8][8], m = kAmaxFloor;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = r0 + half + 16 * j;
    read8(src + static_cast<size_t>(min(r, rows - 1)) * ld_w + c0, r < rows ? n : 0, wide_in, v[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) m = finite_max(v[j], m);
#pragma unroll
  for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, s_max[i]);
  const float inv = __fdiv_rn(kFp8Max, m);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = r0 + half + 16 * j;
    if (r < rows) write8(codes + (mat * rows + r) * ld_codes + c0, n, wide_out, encode8(v[j], inv));
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
  const long long units = static_cast<long long>(rows) * n_blocks;
  if (units > 0x3fffffffll) return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: %d rows of %d columns in one call", rows, cols);
  // wide accesses: rows of 16-byte pieces in (with MOE_ACT_SILU_MUL the second half of a row too), of 8-byte pieces out
  const int wide_in = aligned_to(x_dev, 16) && ld_x * size % 16 == 0 && (act != MOE_ACT_SILU_MUL || static_cast<long long>(cols) * size % 16 == 0);
  const int wide_out = aligned_to(codes_dev, 8) && ld_codes % 8 == 0;
  const unsigned grid = static_cast<unsigned>(std::min<long long>((units + kQuantHalves - 1) / kQuantHalves, static_cast<long long>(c->sm_count) * 64));
  auto go = [&](auto type, auto kernel) {
    using T = decltype(type);
    return launch_kernel(kernel, dim3(grid), kQuantThreads, 0, static_cast<cudaStream_t>(stream), true, 0, static_cast<const T *>(x_dev),
                         static_cast<size_t>(ld_x), rows, cols, static_cast<unsigned>(n_blocks), limit, alpha, pair_row_dev, fanout, out_rows, n_rows_dev,
                         codes_dev, static_cast<size_t>(ld_codes), scales_dev, static_cast<size_t>(ld_scales), wide_in, wide_out);
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
  const int wide_in = aligned_to(w_dev, 16) && ld_w * size % 16 == 0, wide_out = aligned_to(codes_dev, 8) && ld_codes % 8 == 0;
  auto go = [&](auto type) {
    using T = decltype(type);
    return launch_kernel(quantize_fp8_blocks_kernel<T>, grid, 256, 0, static_cast<cudaStream_t>(stream), true, 0, static_cast<const T *>(w_dev),
                         static_cast<size_t>(ld_w), rows, cols, codes_dev, static_cast<size_t>(ld_codes), scales_dev, wide_in, wide_out);
  };
  return launched(c, "moe_quantize_fp8_blocks", dtype == MOE_F32 ? go(float()) : dtype == MOE_BF16 ? go(__nv_bfloat16()) : go(__half()));
}

}  // extern "C"
