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

#include <algorithm>
#include <type_traits>

#include "fp8_layer.cuh"

namespace moe {

constexpr float kFp8Max = 448.f;
constexpr float kAmaxFloor = 1.262177448e-29f;   // 2^-96
constexpr int kQuantCols = 16;                   // columns of a lane
constexpr int kQuantLanes = 128 / kQuantCols;    // lanes that share a block

// Largest value of the lanes that share a block.
__device__ __forceinline__ float block_max(float v) {
#pragma unroll
  for (int off = kQuantLanes / 2; off; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
// Two values side by side, two operations at a time, each rounded to nearest.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint4 encode16(const float (&v)[16], float inv) {
  const uint64_t by = pair(inv, inv);
  uint32_t p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(halves(mul2(pair(v[4 * i], v[4 * i + 1]), by)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(halves(mul2(pair(v[4 * i + 2], v[4 * i + 3]), by)), __NV_SATFINITE, __NV_E4M3);
    p[i] = lo | (hi << 16);
  }
  return make_uint4(p[0], p[1], p[2], p[3]);
}

// gate * sigmoid(alpha * gate) * (up + 1) with the gate clamped from above and up on both sides (ACT_SWIGLU), or
// gate * sigmoid(gate) * up (ACT_SILU_MUL); `rate` is -alpha * log2(e).  Minimum and maximum keep a NaN.  The fast exponential
// and reciprocal are off by 2^-20 at |alpha * gate| = 8 and 2^-18 at 32, next to a code's half step of 2^-4: 137 of 71 M codes are not
// those of 64 bits.  With a division corrected by its remainder 134 for 1.9 us more (6144 x 2880), with expf too 132 for 3.6.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_fast(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float rcp_fast(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}
template <int kAct>
__device__ __forceinline__ float2 gated(float gate0, float gate1, float up0, float up1, float limit, float rate) {
  if (kAct == MOE_ACT_SWIGLU) {
    gate0 = min_nan(gate0, limit);
    gate1 = min_nan(gate1, limit);
    up0 = max_nan(min_nan(up0, limit), -limit);
    up1 = max_nan(min_nan(up1, limit), -limit);
  }
  const uint64_t gate = pair(gate0, gate1), one = pair(1.f, 1.f);
  uint64_t up = pair(up0, up1);
  if (kAct == MOE_ACT_SWIGLU) up = add2(up, one);
  const float2 t = halves(mul2(gate, pair(rate, rate)));
  const float2 d = halves(add2(pair(exp2_fast(t.x), exp2_fast(t.y)), one));
  return halves(mul2(mul2(gate, pair(rcp_fast(d.x), rcp_fast(d.y))), up));
}

// Sixteen values of a row as they lie in memory: consecutive ones in 16-byte loads, or every eighth (eight lanes read neighbours).
// `n`: how many columns there are from the first on.
template <class T>
struct Raw16 {
  uint4 v[sizeof(T)];
  __device__ __forceinline__ void load(const T *p, bool there) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) v[i] = there ? reinterpret_cast<const uint4 *>(p)[i] : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void load_spread(const T *p, int n, int step) {
    T *e = reinterpret_cast<T *>(v);
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = kQuantLanes * i < n ? p[step * i] : T(0.f);
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f32(reinterpret_cast<const T *>(v)[i]); }
};
// Codes of every eighth column -> those of the lane's sixteen neighbours.  Bytes 2 m, 2 m + 1 of lane l are columns 16 m + l and
// 16 m + 8 + l: an 8 x 8 transpose of byte pairs over the eight lanes.
__device__ __forceinline__ uint4 gather_codes(uint4 q) {
  const unsigned lane = threadIdx.x % kQuantLanes;
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t lo[2] = {0, 0}, hi[2] = {0, 0};
#pragma unroll
  for (unsigned step = 0; step < kQuantLanes; ++step) {
    const unsigned other = lane ^ step;
    const uint32_t pair_word = (other & 4) ? ((other & 2) ? w[3] : w[2]) : ((other & 2) ? w[1] : w[0]);
    const uint32_t got = __shfl_xor_sync(0xffffffffu, pair_word >> (16 * (other & 1)), step);   // byte pair `lane` of lane `other`
    const unsigned shift = 8 * (other & 3);
    const uint32_t first = (got & 0xffu) << shift, second = ((got >> 8) & 0xffu) << shift;
    if (other & 4) { lo[1] |= first; hi[1] |= second; }
    else { lo[0] |= first; hi[0] |= second; }
  }
  return make_uint4(lo[0], lo[1], hi[0], hi[1]);
}
__device__ __forceinline__ void write_spread(uint8_t *p, int n, uint4 q) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (kQuantLanes * i < n) p[kQuantLanes * i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i & 3)));
}
__device__ __forceinline__ float finite_max(const float (&v)[16], float m) {
  float a = m;
#pragma unroll
  for (int i = 0; i < 16; i += 2) asm("max.abs.f32 %0, %0, %1, %2;" : "+f"(a) : "f"(v[i]), "f"(v[i + 1]));   // drops a NaN
  if (a < __int_as_float(0x7f800000)) return a;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (fabsf(v[i]) < __int_as_float(0x7f800000)) m = fmaxf(m, fabsf(v[i]));
  return m;
}

// Eight lanes per block of 128 columns, sixteen columns each; the (row, block) pairs of a call are dealt to the groups of lanes.
// Bound by instructions (addresses, places, the two quotients of a block cost the same whatever a lane converts; two values to an
// instruction where there is one).  6144 x 2880 values through SwiGLU 18.1 us, 1856 rows to four places each 6.5; with eight columns a
// lane 24 and 8.5, without the pairs of values 19.0, with four CTAs to an SM in place of five 19.5 and 7.4.  More pairs of a thread
// under way together cost registers and time.  A grid of up to 16 CTAs an SM: with 5, 2048 x 7168 to eight places takes 30.5 us
// instead of 26.6, with 40 the SwiGLU 19.1.
constexpr int kQuantThreads = 256, kQuantGroups = kQuantThreads / kQuantLanes, kPlaces = 4;

template <class T, int kAct, bool kWideIn>
__global__ void __launch_bounds__(kQuantThreads, 5)
quantize_fp8_kernel(const T *x, unsigned ld_x, int rows, int cols, unsigned n_blocks, float limit, float rate, const int *pair_row, unsigned fanout,
                    int out_rows, const int *n_rows, uint8_t *codes, unsigned ld_codes, float *scales, unsigned ld_scales, int wide_out) {
  grid_dep_sync();
  const unsigned lane = threadIdx.x % kQuantLanes;
  int live = rows;
  if (n_rows != nullptr) live = max(min(live, *n_rows), 0);
  const unsigned units = static_cast<unsigned>(live) * n_blocks;      // (row, block) pairs; the host bounds rows * n_blocks
  const unsigned stride = gridDim.x * kQuantGroups;
  // (the groups of a warp leave together: the shuffles are the whole warp's)
  const unsigned row_step = stride / n_blocks, kb_step = stride - row_step * n_blocks;
  unsigned unit = blockIdx.x * kQuantGroups + threadIdx.x / kQuantLanes, at_row = unit / n_blocks, at_kb = unit - at_row * n_blocks;
  auto next = [&]() {
    unit += stride;
    at_row += row_step;
    at_kb += kb_step;
    if (at_kb >= n_blocks) { at_kb -= n_blocks; ++at_row; }
  };
  for (; __any_sync(0xffffffffu, unit < units); next()) {
    const bool on = unit < units;
    const unsigned row = on ? at_row : 0, kb = on ? at_kb : n_blocks;   // no column of block n_blocks exists
    // a lane's columns: sixteen neighbours, or, where rows of x are not 16-byte aligned and in a last part of a block that is not made
    // of sixteens, every eighth
    const int left = cols - static_cast<int>(kb * kScaleBlock);
    const bool packed_out = wide_out && (left >= kScaleBlock || cols % kQuantCols == 0), whole = kWideIn && packed_out;
    const int c0 = static_cast<int>(kb * kScaleBlock + lane * (whole ? kQuantCols : 1)), n = cols - c0;
    const T *src = x + static_cast<size_t>(row) * ld_x;
    float v[16];
    int place[kPlaces];
#pragma unroll
    for (int j = 0; j < kPlaces; ++j) place[j] = -1;
    if (pair_row == nullptr) {
      if (on) place[0] = static_cast<int>(row);
    } else {
#pragma unroll
      for (int j = 0; j < kPlaces; ++j)
        if (on && j < static_cast<int>(fanout)) place[j] = pair_row[static_cast<size_t>(row) * fanout + j];
    }
    if (kAct == MOE_ACT_NONE) {
      Raw16<T> a;
      if (whole) a.load(src + c0, n > 0);
      else a.load_spread(src + c0, n, kQuantLanes);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = a[i];
    } else {
      Raw16<T> a, b;
      if (!whole) {   // gates in a, ups in b
        const int at = kAct == MOE_ACT_SWIGLU ? 2 * c0 : c0, step = kAct == MOE_ACT_SWIGLU ? 2 * kQuantLanes : kQuantLanes;
        a.load_spread(src + at, n, step);
        b.load_spread(src + at + (kAct == MOE_ACT_SWIGLU ? 1 : cols), n, step);
      } else if (kAct == MOE_ACT_SWIGLU) {
        a.load(src + 2 * c0, n > 0);
        b.load(src + 2 * c0 + 16, n > 0);
      } else {
        a.load(src + c0, n > 0);
        b.load(src + cols + c0, n > 0);
      }
      if (kAct == MOE_ACT_SWIGLU && whole) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float2 p = gated<kAct>(a[2 * i], a[2 * i + 2], a[2 * i + 1], a[2 * i + 3], limit, rate);
          const float2 q = gated<kAct>(b[2 * i], b[2 * i + 2], b[2 * i + 1], b[2 * i + 3], limit, rate);
          v[i] = p.x; v[i + 1] = p.y;
          v[i + 8] = q.x; v[i + 9] = q.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 p = gated<kAct>(a[i], a[i + 1], b[i], b[i + 1], limit, rate);
          v[i] = p.x; v[i + 1] = p.y;
        }
      }
    }
    const float m = block_max(finite_max(v, kAmaxFloor));
    uint4 q = encode16(v, __fdiv_rn(kFp8Max, m));
    if (!kWideIn && wide_out) {   // (all lanes: one block of the warp's is reason enough)
      const uint4 packed = gather_codes(q);
      if (packed_out) q = packed;
    }
    const float scale = __fdiv_rn(m, kFp8Max);
    auto put = [&](int r) {
      if (static_cast<unsigned>(r) >= static_cast<unsigned>(out_rows)) return;
      uint8_t *dst = codes + static_cast<size_t>(static_cast<unsigned>(r)) * ld_codes;
      if (!packed_out) write_spread(dst + c0, n, q);
      else if (static_cast<int>(lane * kQuantCols) < left) *reinterpret_cast<uint4 *>(dst + kb * kScaleBlock + lane * kQuantCols) = q;
      if (lane == 0) scales[static_cast<size_t>(static_cast<unsigned>(r)) * ld_scales + kb] = scale;
    };
    put(place[0]);
    if (fanout > 1) {
#pragma unroll
      for (int j = 1; j < kPlaces; ++j) put(place[j]);
    }
    if (on)
      for (unsigned j = kPlaces; j < fanout; ++j) put(pair_row[static_cast<size_t>(row) * fanout + j]);
  }
}

// A CTA per 128 x 128 block: lane group g takes rows g, g + 32, ... of it.  32 x 5760 x 2880 from fp32 374 us: 7.1 TB/s, HBM.  From
// bf16 476 us, 3.4 TB/s: two CTAs fit an SM, and with half the bytes of a load under way they wait for them (issue slots 23 % used).
template <class T>
__global__ void __launch_bounds__(kQuantThreads)
quantize_fp8_blocks_kernel(const T *w, size_t ld_w, int rows, int cols, uint8_t *codes, size_t ld_codes, float *scales, int wide) {
  __shared__ float s_max[kQuantThreads / 32];
  grid_dep_sync();
  constexpr int kRows = kScaleBlock / kQuantGroups;   // of a thread
  const int lane = threadIdx.x % kQuantLanes, group = threadIdx.x / kQuantLanes;
  const int r0 = blockIdx.y * kScaleBlock;
  const bool whole = wide && (cols - static_cast<int>(blockIdx.x * kScaleBlock) >= kScaleBlock || cols % kQuantCols == 0);   // (quantize_fp8_kernel)
  const int c0 = blockIdx.x * kScaleBlock + lane * (whole ? kQuantCols : 1), n = cols - c0;
  const size_t mat = blockIdx.z;
  const T *src = w + mat * rows * ld_w;
  Raw16<T> raw[kRows];
  float m = kAmaxFloor;
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int r = r0 + group + kQuantGroups * j;
    const T *from = src + static_cast<size_t>(min(r, rows - 1)) * ld_w + c0;   // (a row again, where there is none: no other maximum)
    if (whole) raw[j].load(from, n > 0);
    else raw[j].load_spread(from, n, kQuantLanes);
  }
  float v[16];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = raw[j][i];
    m = finite_max(v, m);
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuantThreads / 32; ++i) m = fmaxf(m, s_max[i]);
  const float inv = __fdiv_rn(kFp8Max, m);
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int r = r0 + group + kQuantGroups * j;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = raw[j][i];
    if (r >= rows) continue;
    uint8_t *dst = codes + (mat * rows + r) * ld_codes + c0;
    if (!whole) write_spread(dst, n, encode16(v, inv));
    else if (n > 0) *reinterpret_cast<uint4 *>(dst) = encode16(v, inv);
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
  if (!size || rows < 0 || cols < 1 || ld_x < wide || ld_codes < cols || ld_scales < n_blocks || std::max({ld_x, ld_codes, ld_scales}) > 0x7fffffffll)
    return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: dtype %d, %d rows of %d columns, strides %lld, %lld, %lld", dtype, rows, cols, ld_x, ld_codes, ld_scales);
  if (fanout < 1 || out_rows < 0 || static_cast<long long>(rows) * fanout > 0x7fffffffll || (!pair_row_dev && (fanout != 1 || out_rows < rows)))
    return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: %d rows to %d places each among %d%s", rows, fanout, out_rows, pair_row_dev ? "" : ", without a map");
  if (rows == 0 || out_rows == 0) return MOE_OK;
  if (!x_dev || !codes_dev || !scales_dev) return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: null tensor");
  if (!aligned_to(x_dev, size) || !aligned_to(pair_row_dev, 4) || !aligned_to(n_rows_dev, 4) || !aligned_to(scales_dev, 4))
    return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: a tensor is not aligned to its elements");
  const long long units = static_cast<long long>(rows) * n_blocks;
  if (units > 0x3fffffffll) return op_fail(c, MOE_ERR_INVALID, "moe_quantize_fp8: %d rows of %d columns in one call", rows, cols);
  if (int rc = use_device(c, "moe_quantize_fp8")) return rc;
  // wide accesses: rows of 16-byte pieces (with MOE_ACT_SILU_MUL the second half of a row of x too)
  const int wide_in = aligned_to(x_dev, 16) && ld_x * size % 16 == 0 && (act != MOE_ACT_SILU_MUL || static_cast<long long>(cols) * size % 16 == 0);
  const int wide_out = aligned_to(codes_dev, 16) && ld_codes % 16 == 0;
  // (an alpha whose rate would be infinite: gates next to 0 are below the smallest maximum, but 0 * inf would be a NaN)
  const float rate = std::clamp(-1.44269504088896341f * (act == MOE_ACT_SWIGLU ? alpha : 1.f), -3.402823466e38f, 3.402823466e38f);
  const unsigned grid = static_cast<unsigned>(std::min<long long>((units + kQuantGroups - 1) / kQuantGroups, static_cast<long long>(c->sm_count) * 16));
  auto go = [&](auto type, auto kernel) {
    using T = decltype(type);
    return launch_kernel(kernel, dim3(grid), kQuantThreads, 0, static_cast<cudaStream_t>(stream), true, 0, static_cast<const T *>(x_dev),
                         static_cast<unsigned>(ld_x), rows, cols, static_cast<unsigned>(n_blocks), limit, rate, pair_row_dev, static_cast<unsigned>(fanout),
                         out_rows, n_rows_dev, codes_dev, static_cast<unsigned>(ld_codes), scales_dev, static_cast<unsigned>(ld_scales), wide_out);
  };
  auto by_act = [&](auto type) {
    using T = decltype(type);
    auto by_alignment = [&](auto wide) {
      constexpr bool kWide = decltype(wide)::value;
      return act == MOE_ACT_NONE     ? go(type, quantize_fp8_kernel<T, MOE_ACT_NONE, kWide>)
             : act == MOE_ACT_SWIGLU ? go(type, quantize_fp8_kernel<T, MOE_ACT_SWIGLU, kWide>)
                                     : go(type, quantize_fp8_kernel<T, MOE_ACT_SILU_MUL, kWide>);
    };
    return wide_in ? by_alignment(std::true_type()) : by_alignment(std::false_type());
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
  const int wide_in = aligned_to(w_dev, 16) && ld_w * size % 16 == 0, wide_out = aligned_to(codes_dev, 16) && ld_codes % 16 == 0;
  auto go = [&](auto type) {
    using T = decltype(type);
    return launch_kernel(quantize_fp8_blocks_kernel<T>, grid, kQuantThreads, 0, static_cast<cudaStream_t>(stream), true, 0, static_cast<const T *>(w_dev),
                         static_cast<size_t>(ld_w), rows, cols, codes_dev, static_cast<size_t>(ld_codes), scales_dev, wide_in && wide_out);
  };
  return launched(c, "moe_quantize_fp8_blocks", dtype == MOE_F32 ? go(float()) : dtype == MOE_BF16 ? go(__nv_bfloat16()) : go(__half()));
}

}  // extern "C"
