// Row movement around a layer of routed experts, as calls of their own: routing by scores (moe_route_scored), the
// permutation that sorts (token, expert) pairs by expert (moe_group_pairs), and the weighted sum of a token's expert rows
// (moe_combine_pairs).  The MXFP4 block has fixed forms of all three inside (route.cu); these take any router rule, any
// row types and strides, and pairs without an expert.
#include "fp8_layer.cuh"

namespace moe {

// ---------------------------------------------------------------------------
// Routing.  Of a row's logits x:  s = sigmoid(x), or softmax over the experts that are on;  p = s + bias;  the groups
// with the highest sum of their group_top largest p stay;  the top_k largest p of what stays are selected, ties to the
// lower index;  weight = s [/ sum of the selected s] * scale.  An expert is off where x or its bias is -inf or NaN.
// Scores are held in 64 bits: which of two neighbouring p is larger is part of the answer, and s + bias is where
// 32 bits would tie or swap them.
// A warp per row; lane l owns the per_lane consecutive experts from l * per_lane, so that a lower lane is a lower index.
// ---------------------------------------------------------------------------
constexpr int kRouteWarps = 4;
constexpr int kMaxScoredExperts = 512, kMaxScoredTopK = 32, kMaxScoredGroups = 32;

// 64-bit integers in the order of the doubles; 0 is below every one of them and means "off".
__device__ __forceinline__ unsigned long long ordered_key(double p) {
  const long long b = __double_as_longlong(p == 0.0 ? 0.0 : p);   // -0 and 0 are equal
  return b < 0 ? ~static_cast<unsigned long long>(b) : static_cast<unsigned long long>(b) | 0x8000000000000000ull;
}
__device__ __forceinline__ double key_value(unsigned long long k) {
  return __longlong_as_double(static_cast<long long>((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
}

template <class T, int kPer>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_scored_kernel(const T *logits, size_t ld, const float *bias, int rows, moe_route_rule rule, int per_lane, int *idx, float *w) {
  __shared__ unsigned long long s_keys[kRouteWarps][kPer * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t row = static_cast<size_t>(blockIdx.x) * kRouteWarps + warp;
  if (row >= static_cast<size_t>(rows)) return;
  const int E = rule.n_experts, first = lane * per_lane;
  const float inf = __int_as_float(0x7f800000);
  double s[kPer];
  unsigned long long key[kPer];
  double top = -1e300;   // largest logit of the experts that are on
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool mine = i < per_lane && first + i < E;
    float x = mine ? to_f32(logits[row * ld + first + i]) : -inf;
    if (x > 3.402823466e38f) x = 3.402823466e38f;   // +inf counts as the largest finite value
    key[i] = x > -inf ? 1 : 0;
    s[i] = x;
    if (key[i]) top = fmax(top, s[i]);
  }
  if (rule.score == MOE_SCORE_SOFTMAX) {
    for (int off = 16; off; off >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, off));
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      s[i] = key[i] ? exp(s[i] - top) : 0.0;
      sum += s[i];
    }
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (key[i]) s[i] /= sum;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) s[i] = key[i] ? 1.0 / (1.0 + exp(-s[i])) : 0.0;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (!key[i]) continue;
    const float b = bias != nullptr ? bias[first + i] : 0.f;
    key[i] = b > -inf ? ordered_key(s[i] + static_cast<double>(b)) : 0;
  }
  if (rule.n_groups > 1) {
    // lane g takes group g: the group_top largest of its members, then its rank among the groups
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < per_lane && first + i < E) s_keys[warp][first + i] = key[i];
    __syncwarp();
    const int size = E / rule.n_groups;
    unsigned long long k1 = 0, k2 = 0;
    if (lane < rule.n_groups)
      for (int j = 0; j < size; ++j) {
        const unsigned long long k = s_keys[warp][lane * size + j];
        if (k > k1) { k2 = k1; k1 = k; }
        else if (k > k2) k2 = k;
      }
    unsigned long long g_key = k1;
    if (rule.group_top == 2 && k2) g_key = ordered_key(key_value(k1) + key_value(k2));
    int better = 0;
    for (int g = 0; g < rule.n_groups; ++g) {
      const unsigned long long k = __shfl_sync(0xffffffffu, g_key, g);
      better += k > g_key || (k == g_key && g < lane);
    }
    const unsigned stays = __ballot_sync(0xffffffffu, lane < rule.n_groups && better < rule.top_groups);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < per_lane && first + i < E && !(stays >> ((first + i) / size) & 1u)) key[i] = 0;
  }
  // top_k rounds: the largest key of a lane, then of the warp; the lowest lane of equal ones
  int sel = -1;
  double sel_s = 0.0;
  for (int k = 0; k < rule.top_k; ++k) {
    unsigned long long best = 0;
    int at = 0;
    double best_s = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (key[i] > best) { best = key[i]; at = i; best_s = s[i]; }
    const unsigned hi = static_cast<unsigned>(best >> 32), lo = static_cast<unsigned>(best);
    const unsigned hi_max = __reduce_max_sync(0xffffffffu, hi);
    if (hi_max == 0) break;   // nothing left (a key that is on has its sign bit or a large complement set)
    const unsigned lo_max = __reduce_max_sync(0xffffffffu, hi == hi_max ? lo : 0u);
    const int owner = __ffs(__ballot_sync(0xffffffffu, hi == hi_max && lo == lo_max)) - 1;
    const int e = __shfl_sync(0xffffffffu, first + at, owner);
    const double es = __shfl_sync(0xffffffffu, best_s, owner);
    if (lane == k) { sel = e; sel_s = es; }
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i == at) key[i] = 0;
    }
  }
  double sum = sel_s;
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane < rule.top_k) {
    const double share = !rule.renormalise ? sel_s : sum > 0.0 ? sel_s / sum : 0.0;
    idx[row * rule.top_k + lane] = sel;
    w[row * rule.top_k + lane] = static_cast<float>(share * static_cast<double>(rule.scale));
  }
}

template <class T>
cudaError_t launch_route_scored(const moe_route_rule &r, const void *logits, size_t ld, const float *bias, int rows, int *idx, float *w,
                                cudaStream_t s) {
  const int per = (r.n_experts + 31) / 32;
  const unsigned grid = static_cast<unsigned>((static_cast<size_t>(rows) + kRouteWarps - 1) / kRouteWarps);
  const T *x = static_cast<const T *>(logits);
  auto go = [&](auto kernel) { kernel<<<grid, kRouteWarps * 32, 0, s>>>(x, ld, bias, rows, r, per, idx, w); };
  if (per <= 1) go(route_scored_kernel<T, 1>);
  else if (per <= 2) go(route_scored_kernel<T, 2>);
  else if (per <= 4) go(route_scored_kernel<T, 4>);
  else if (per <= 8) go(route_scored_kernel<T, 8>);
  else go(route_scored_kernel<T, 16>);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Stable counting sort of the pairs (token * top_k + slot) by expert.  One CTA: every warp owns a contiguous range of
// pairs and counts it into a histogram of its own; prefixes over experts and warps give every warp its place in every
// expert's rows; a second walk over the same pairs hands the places out, so that they ascend with the pair.
// ---------------------------------------------------------------------------
constexpr int kGroupThreads = 1024, kGroupWarps = kGroupThreads / 32;
constexpr int kMaxGroupedExperts = 1024;

__global__ void __launch_bounds__(kGroupThreads)
group_pairs_kernel(const int *idx, size_t n_pairs, int E, int *offsets, int *pair_row, int *row_pair) {
  extern __shared__ int s_hist[];   // [kGroupWarps][E]
  __shared__ int s_scan[kGroupWarps], s_total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int *mine = s_hist + warp * E;
  for (int i = threadIdx.x; i < kGroupWarps * E; i += kGroupThreads) s_hist[i] = 0;
  __syncthreads();
  const size_t per = (n_pairs + kGroupThreads - 1) / kGroupThreads * 32;
  const size_t begin = min(per * warp, n_pairs), end = min(begin + per, n_pairs);
  for (size_t p = begin + lane; p < end; p += 32) {
    const int e = idx[p];
    if (e >= 0 && e < E) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  // thread e: exclusive prefix over the warps, then over the experts
  int total = 0;
  if (threadIdx.x < E)
    for (int v = 0; v < kGroupWarps; ++v) {
      const int n = s_hist[v * E + threadIdx.x];
      s_hist[v * E + threadIdx.x] = total;
      total += n;
    }
  int incl = total;
  for (int off = 1; off < 32; off <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += up;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int v = s_scan[lane], t = v;
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, t, off);
      if (lane >= off) t += up;
    }
    s_scan[lane] = t - v;
    if (lane == 31) s_total = t;
  }
  __syncthreads();
  const int start = s_scan[warp] + incl - total;
  if (threadIdx.x < E) {
    offsets[threadIdx.x] = start;
    for (int v = 0; v < kGroupWarps; ++v) s_hist[v * E + threadIdx.x] += start;
  }
  if (threadIdx.x == 0) offsets[E] = s_total;
  __syncthreads();
  for (size_t p0 = begin; p0 < end; p0 += 32) {
    const size_t p = p0 + lane;
    int e = p < end ? idx[p] : -1;
    if (e < 0 || e >= E) e = -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int row = -1;
    if (e >= 0) row = mine[e] + rank;
    __syncwarp();
    if (e >= 0 && rank == 0) mine[e] += __popc(same);
    __syncwarp();
    if (p < end) pair_row[p] = row;
    if (row >= 0 && row_pair != nullptr) row_pair[row] = static_cast<int>(p);
  }
  if (row_pair != nullptr)
    for (size_t r = static_cast<size_t>(s_total) + threadIdx.x; r < n_pairs; r += kGroupThreads) row_pair[r] = -1;
}

// ---------------------------------------------------------------------------
// out[t] = residual[t] + sum over k of w[t, k] * y[pair_row[t, k]], added in the order of k in fp32 and rounded once.
// A pair whose row is negative or not below n_y_rows adds nothing, whatever its weight.
// ---------------------------------------------------------------------------
template <class TY, class TO>
__global__ void __launch_bounds__(256)
combine_pairs_kernel(const TY *y, size_t ld_y, int n_y_rows, const int *pair_row, const float *w, int top_k, int cols, const TO *residual,
                     size_t ld_residual, TO *out, size_t ld_out) {
  const size_t t = blockIdx.x;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    float sum = 0.f;
    for (int k = 0; k < top_k; ++k) {
      const int r = pair_row[t * top_k + k];
      if (r >= 0 && r < n_y_rows) sum = fmaf(w[t * top_k + k], to_f32(y[static_cast<size_t>(r) * ld_y + c]), sum);
    }
    if (residual != nullptr) sum += to_f32(residual[t * ld_residual + c]);
    store_as(out + t * ld_out + c, sum);
  }
}

template <class TY, class TO>
cudaError_t launch_combine_pairs(const void *y, size_t ld_y, int n_y_rows, const int *pair_row, const float *w, int rows, int top_k, int cols,
                                 const void *residual, size_t ld_residual, void *out, size_t ld_out, cudaStream_t s) {
  combine_pairs_kernel<TY, TO><<<rows, 256, 0, s>>>(static_cast<const TY *>(y), ld_y, n_y_rows, pair_row, w, top_k, cols,
                                                    static_cast<const TO *>(residual), ld_residual, static_cast<TO *>(out), ld_out);
  return cudaGetLastError();
}

}  // namespace moe

using namespace moe;

extern "C" {

int moe_route_scored(moe_handle c, const moe_route_rule *rule, const void *logits_dev, int dtype, long long ld, const float *bias_dev,
                     int rows, int *idx_dev, float *w_dev, void *stream) {
  if (!c) return MOE_ERR_INVALID;
  if (!rule) return op_fail(c, MOE_ERR_INVALID, "moe_route_scored: null rule");
  const moe_route_rule &r = *rule;
  if (r.n_experts < 1 || r.n_experts > kMaxScoredExperts || r.top_k < 1 || r.top_k > kMaxScoredTopK || r.top_k > r.n_experts)
    return op_fail(c, MOE_ERR_INVALID, "moe_route_scored: %d of %d experts (at most %d of %d)", r.top_k, r.n_experts, kMaxScoredTopK, kMaxScoredExperts);
  if (r.score != MOE_SCORE_SOFTMAX && r.score != MOE_SCORE_SIGMOID) return op_fail(c, MOE_ERR_INVALID, "moe_route_scored: score %d", r.score);
  if (r.n_groups < 1 || r.n_groups > kMaxScoredGroups || r.n_experts % r.n_groups || r.top_groups < 1 || r.top_groups > r.n_groups ||
      (r.group_top != 1 && r.group_top != 2))
    return op_fail(c, MOE_ERR_INVALID, "moe_route_scored: %d of %d groups of %d experts, by their %d best", r.top_groups, r.n_groups, r.n_experts, r.group_top);
  if (!(r.scale - r.scale == 0.f)) return op_fail(c, MOE_ERR_INVALID, "moe_route_scored: scale is not finite");
  const int size = dtype_size(dtype);
  if (!size || ld < r.n_experts || rows < 0) return op_fail(c, MOE_ERR_INVALID, "moe_route_scored: dtype %d, row stride %lld, %d rows", dtype, ld, rows);
  if (rows == 0) return MOE_OK;
  if (!logits_dev || !idx_dev || !w_dev) return op_fail(c, MOE_ERR_INVALID, "moe_route_scored: null tensor");
  if (!aligned_to(logits_dev, size) || !aligned_to(bias_dev, 4) || !aligned_to(idx_dev, 4) || !aligned_to(w_dev, 4))
    return op_fail(c, MOE_ERR_INVALID, "moe_route_scored: a tensor is not aligned to its elements");
  if (int rc = use_device(c, "moe_route_scored")) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t l = static_cast<size_t>(ld);
  return launched(c, "moe_route_scored",
                  dtype == MOE_F32    ? launch_route_scored<float>(r, logits_dev, l, bias_dev, rows, idx_dev, w_dev, s)
                  : dtype == MOE_BF16 ? launch_route_scored<__nv_bfloat16>(r, logits_dev, l, bias_dev, rows, idx_dev, w_dev, s)
                                      : launch_route_scored<__half>(r, logits_dev, l, bias_dev, rows, idx_dev, w_dev, s));
}

int moe_group_pairs(moe_handle c, const int *idx_dev, int rows, int top_k, int n_experts, int *offsets_dev, int *pair_row_dev,
                    int *row_pair_dev, void *stream) {
  if (!c) return MOE_ERR_INVALID;
  if (rows < 0 || top_k < 1 || n_experts < 1 || n_experts > kMaxGroupedExperts || static_cast<long long>(rows) * top_k > 0x7fffffffll)
    return op_fail(c, MOE_ERR_INVALID, "moe_group_pairs: %d rows x %d, %d experts (at most %d)", rows, top_k, n_experts, kMaxGroupedExperts);
  if (!offsets_dev || (rows > 0 && (!idx_dev || !pair_row_dev))) return op_fail(c, MOE_ERR_INVALID, "moe_group_pairs: null tensor");
  if (!aligned_to(idx_dev, 4) || !aligned_to(offsets_dev, 4) || !aligned_to(pair_row_dev, 4) || !aligned_to(row_pair_dev, 4))
    return op_fail(c, MOE_ERR_INVALID, "moe_group_pairs: a tensor is not aligned to its elements");
  if (int rc = use_device(c, "moe_group_pairs")) return rc;
  const size_t smem = static_cast<size_t>(kGroupWarps) * n_experts * sizeof(int);
  cudaError_t e = allow_smem(c, reinterpret_cast<const void *>(group_pairs_kernel), kGroupWarps * kMaxGroupedExperts * 4, kSmemGroup);
  if (e == cudaSuccess) {
    group_pairs_kernel<<<1, kGroupThreads, smem, static_cast<cudaStream_t>(stream)>>>(idx_dev, static_cast<size_t>(rows) * top_k, n_experts,
                                                                                      offsets_dev, pair_row_dev, row_pair_dev);
    e = cudaGetLastError();
  }
  return launched(c, "moe_group_pairs", e);
}

int moe_combine_pairs(moe_handle c, const void *y_dev, int y_dtype, long long ld_y, int n_y_rows, const int *pair_row_dev, const float *w_dev,
                      int rows, int top_k, int cols, const void *residual_dev, long long ld_residual, void *out_dev, int out_dtype,
                      long long ld_out, void *stream) {
  if (!c) return MOE_ERR_INVALID;
  const int ys = dtype_size(y_dtype), os = dtype_size(out_dtype);
  if (!ys || !os || rows < 0 || top_k < 1 || cols < 1 || n_y_rows < 0 || ld_y < cols || ld_out < cols || (residual_dev && ld_residual < cols) ||
      static_cast<long long>(rows) * top_k > 0x7fffffffll)
    return op_fail(c, MOE_ERR_INVALID, "moe_combine_pairs: dtypes %d and %d, %d rows x %d of %d columns, strides %lld, %lld, %lld", y_dtype, out_dtype,
                   rows, top_k, cols, ld_y, ld_residual, ld_out);
  if (rows == 0) return MOE_OK;
  if ((!y_dev && n_y_rows > 0) || !pair_row_dev || !w_dev || !out_dev) return op_fail(c, MOE_ERR_INVALID, "moe_combine_pairs: null tensor");
  if (!aligned_to(y_dev, ys) || !aligned_to(pair_row_dev, 4) || !aligned_to(w_dev, 4) || !aligned_to(residual_dev, os) || !aligned_to(out_dev, os))
    return op_fail(c, MOE_ERR_INVALID, "moe_combine_pairs: a tensor is not aligned to its elements");
  if (int rc = use_device(c, "moe_combine_pairs")) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t ly = static_cast<size_t>(ld_y), lr = residual_dev ? static_cast<size_t>(ld_residual) : 0, lo = static_cast<size_t>(ld_out);
  auto from = [&](auto y_type) {
    using TY = decltype(y_type);
    switch (out_dtype) {
      case MOE_F32: return launch_combine_pairs<TY, float>(y_dev, ly, n_y_rows, pair_row_dev, w_dev, rows, top_k, cols, residual_dev, lr, out_dev, lo, s);
      case MOE_BF16: return launch_combine_pairs<TY, __nv_bfloat16>(y_dev, ly, n_y_rows, pair_row_dev, w_dev, rows, top_k, cols, residual_dev, lr, out_dev, lo, s);
      default: return launch_combine_pairs<TY, __half>(y_dev, ly, n_y_rows, pair_row_dev, w_dev, rows, top_k, cols, residual_dev, lr, out_dev, lo, s);
    }
  };
  return launched(c, "moe_combine_pairs", y_dtype == MOE_F32 ? from(float()) : y_dtype == MOE_BF16 ? from(__nv_bfloat16()) : from(__half()));
}

}  // extern "C"
