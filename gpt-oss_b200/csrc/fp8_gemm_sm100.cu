// Product of e4m3 rows with e4m3 weights under a scale for every 128 columns of a row and every 128 x 128 block of the
// weights, dense or with the rows grouped by expert (moe_gemm_fp8):
//
//   out[m, n] = bias[g, n] + sum over blocks b of  sa[m, b] * sb[g, n / 128, b] * (sum over k in b of a[m, k] * w[g, n, k])
//
// with g the group of row m.
#include <cuda_fp8.h>

#include "fp8_layer.cuh"

namespace moe {

struct Fp8GemmArgs {
  const uint8_t *a, *b;
  size_t ld_a, ld_b;         // bytes between rows
  const float *sa, *sb;
  size_t ld_sa;
  int rows, n, k, n_groups;
  const int *offsets;        // [n_groups + 1], rows of group g: [offsets[g], offsets[g + 1]); nullptr: one group of all rows
  const __nv_bfloat16 *bias;
  void *out;
  size_t ld_out;
};

// Rows [begin, end) of a group, whatever the offsets say inside [0, rows].
__device__ __forceinline__ void group_rows(const Fp8GemmArgs &p, int g, int &begin, int &end) {
  begin = 0;
  end = p.rows;
  if (p.offsets != nullptr) {
    begin = min(max(p.offsets[g], 0), p.rows);
    end = min(max(p.offsets[g + 1], begin), p.rows);
  }
}

__device__ __forceinline__ float e4m3_to_f32(uint8_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(v), __NV_E4M3)));
}

// 64 rows x 64 weight rows per CTA on the CUDA cores, a scale block of k at a time through shared memory.
template <class T>
__global__ void __launch_bounds__(256)
fp8_gemm_simt_kernel(const Fp8GemmArgs p) {
  __shared__ float s_a[32][65], s_b[32][65];
  int begin, end;
  group_rows(p, blockIdx.z, begin, end);
  const int n0 = blockIdx.x * 64, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int n_kb = (p.k + kScaleBlock - 1) / kScaleBlock, n_nb = (p.n + kScaleBlock - 1) / kScaleBlock;
  for (int m0 = begin + blockIdx.y * 64; m0 < end; m0 += gridDim.y * 64) {
    float acc[4][4] = {};
    for (int kb = 0; kb < n_kb; ++kb) {
      float part[4][4] = {};
      for (int k0 = kb * kScaleBlock; k0 < min(p.k, (kb + 1) * kScaleBlock); k0 += 32) {
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * 32; i += 256) {
          const int r = i / 32, kk = i % 32;
          const bool in = k0 + kk < p.k;
          s_a[kk][r] = in && m0 + r < end ? e4m3_to_f32(p.a[static_cast<size_t>(m0 + r) * p.ld_a + k0 + kk]) : 0.f;
          s_b[kk][r] = in && n0 + r < p.n ? e4m3_to_f32(p.b[(static_cast<size_t>(blockIdx.z) * p.n + n0 + r) * p.ld_b + k0 + kk]) : 0.f;
        }
        __syncthreads();
        for (int kk = 0; kk < 32; ++kk)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[i][j] = fmaf(s_a[kk][ty + 16 * i], s_b[kk][tx + 16 * j], part[i][j]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
          if (m < end && n < p.n)
            acc[i][j] = fmaf(part[i][j], p.sa[static_cast<size_t>(m) * p.ld_sa + kb] * p.sb[(static_cast<size_t>(blockIdx.z) * n_nb + n / kScaleBlock) * n_kb + kb], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
        if (m < end && n < p.n) {
          const float b = p.bias != nullptr ? __bfloat162float(p.bias[static_cast<size_t>(blockIdx.z) * p.n + n]) : 0.f;
          store_as(static_cast<T *>(p.out) + static_cast<size_t>(m) * p.ld_out + n, acc[i][j] + b);
        }
      }
  }
}

}  // namespace moe

using namespace moe;

extern "C" {

int moe_gemm_fp8(moe_handle c, const uint8_t *a_dev, long long ld_a, const float *sa_dev, long long ld_sa, int rows, const uint8_t *b_dev,
                 long long ld_b, const float *sb_dev, int n, int k, int n_groups, const int *offsets_dev, const void *bias_dev, void *out_dev,
                 int out_dtype, long long ld_out, void *stream) {
  if (!c) return MOE_ERR_INVALID;
  const int size = dtype_size(out_dtype);
  const long long n_kb = (static_cast<long long>(k) + kScaleBlock - 1) / kScaleBlock;
  if (!size || rows < 0 || n < 1 || k < 1 || ld_a < k || ld_b < k || ld_sa < n_kb || ld_out < n)
    return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: %d x %d x %d, output type %d, strides %lld, %lld, %lld, %lld", rows, n, k, out_dtype, ld_a, ld_sa, ld_b, ld_out);
  if (n_groups < 1 || n_groups > 1024 || (!offsets_dev && n_groups != 1))
    return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: %d groups%s", n_groups, offsets_dev ? "" : " without offsets");
  if (ld_a % 16 || ld_b % 16 || !aligned_to(a_dev, 16) || !aligned_to(b_dev, 16))
    return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: codes need 16-byte aligned rows (strides %lld, %lld)", ld_a, ld_b);
  if (rows == 0) return MOE_OK;
  if (!a_dev || !sa_dev || !b_dev || !sb_dev || !out_dev) return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: null tensor");
  if (!aligned_to(sa_dev, 4) || !aligned_to(sb_dev, 4) || !aligned_to(offsets_dev, 4) || !aligned_to(bias_dev, 2) || !aligned_to(out_dev, size))
    return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: a tensor is not aligned to its elements");
  if (int rc = use_device(c, "moe_gemm_fp8")) return rc;
  Fp8GemmArgs p = {};
  p.a = a_dev; p.b = b_dev; p.ld_a = static_cast<size_t>(ld_a); p.ld_b = static_cast<size_t>(ld_b);
  p.sa = sa_dev; p.sb = sb_dev; p.ld_sa = static_cast<size_t>(ld_sa);
  p.rows = rows; p.n = n; p.k = k; p.n_groups = n_groups; p.offsets = offsets_dev;
  p.bias = static_cast<const __nv_bfloat16 *>(bias_dev); p.out = out_dev; p.ld_out = static_cast<size_t>(ld_out);
  const dim3 grid((n - 1) / 64 + 1, std::min((rows - 1) / 64 + 1, 128), n_groups);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (out_dtype == MOE_F32) fp8_gemm_simt_kernel<float><<<grid, 256, 0, s>>>(p);
  else if (out_dtype == MOE_BF16) fp8_gemm_simt_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
  else fp8_gemm_simt_kernel<__half><<<grid, 256, 0, s>>>(p);
  return launched(c, "moe_gemm_fp8", cudaGetLastError());
}

}  // extern "C"
