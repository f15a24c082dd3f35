// Product of e4m3 rows with e4m3 weights under a scale for every 128 columns of a row and every 128 x 128 block of the
// weights, dense or with the rows grouped by expert (moe_gemm_fp8):
//
//   out[m, n] = bias[g, n] + sum over blocks b of  sa[m, b] * sb[g, n / 128, b] * (sum over k in b of a[m, k] * w[g, n, k])
//
// with g the group of row m.  The inner sum is a tcgen05.mma of K = 128 (four instructions) into a fresh fp32 accumulator in
// tensor memory; the outer one, with its two scales, is one multiply-add per element and block on the CUDA cores, in fp32
// registers.
//
// That outer sum is what these kernels are shaped by.  The codes of a block of k go from HBM through TMA to the tensor core
// untouched, but every fp32 partial product comes back through registers once per 128 of k.
//
// Few rows per group (fp8_gemm_kernel).  The weights are the M operand: a tile is one row of scale blocks (128 weight rows, a lane of
// tensor memory each) against up to kTok token rows on N, which follows the number of rows of the group in steps of 16.  sb is
// then one number per tile and block, and sa * sb a vector over the columns of the accumulator that a warp of its own forms in
// shared memory.  The accumulators are read as fragments (a thread has two neighbouring columns of four rows): an 8-byte load of
// scales then serves four packed multiply-adds.  With a row per thread every scale of the tile is loaded in every thread, and a
// block of 128 x 128 took 700 cycles for its multiply-adds instead of 120, although the tensor-memory loads of fragments are
// slower (128 cycles of a quadrant for 64 columns, 35 for rows).  Bound by HBM: 256 rows over 32 experts of 5760 x 2880 85 us =
// 6.3 TB/s in a graph, 92 called one after the other.  One decode step (16 x 4096 x 7168) 8.6 us in a graph, 9.8 called, for the 4.5
// that its weights take: launch, 14 blocks of k, and the sum of four CTAs' parts.
//
// Many rows per group (fp8_gemm_wide_kernel).  128 token rows x 256 weight rows; the token rows are the M operand, so that sa * sb
// is one number per thread and block.  8192 x 4096 x 7168 263 us = 1.83 PFLOP/s, 6144 rows over 32 experts of 5760 x 2880 208 us,
// called one after the other, at the power cap: the clock falls to 1.36 GHz (short runs in a graph begin at a higher one: 218 to 255
// and 175; the figures below are of those).  In cycles a block of k takes 775 (dense) for 512 of tensor pipe; two
// accumulators of 256 columns are all that tensor memory holds, and one comes back for its next block after the MMA (512), the
// wait that sees it done (180), eight loads of 16 columns with their multiply-adds (600) and the wait of the MMA warp (150).
// Measured and set aside: pairs of CTAs (cta_group::2, 256 x 256), which move a third less through shared memory, 226 us for the
// experts (tiles of 256 rows waste 62 % on groups of 192, those of 128 32 %) and 260 for the dense case; halves of 128 columns
// with an MMA warp each, the same; the next barrier looked up ahead of time, 4 to 8 % slower; loads of 32 columns in two
// buffers, slower by what spills (the accumulators are 128 registers of 168).
#include <cuda_fp8.h>

#include "fp8_layer.cuh"
#include "sm100_ptx.cuh"

namespace moe {

using namespace sm100;

struct Fp8GemmArgs {
  const float *sa, *sb;
  size_t ld_sa;
  int rows, n, n_kb, n_groups;
  const int *offsets;        // [n_groups + 1], rows of group g: [offsets[g], offsets[g + 1]); nullptr: one group of all rows
  const __nv_bfloat16 *bias;
  void *out;
  size_t ld_out;
  int out_dtype;
  int splits;                // CTAs of a cluster that share the reduction of a tile
  unsigned int *status;
};

constexpr int kMaxGemmGroups = 1024;
constexpr int kGemmRingBytes = 218 * 1024;               // of shared memory for tiles, scales and outputs
constexpr int kScaleBlocks = 8, kScaleSlots = 2;         // blocks of k whose scales are handed over at once
constexpr int kWeightTile = kScaleBlock * kScaleBlock;   // bytes of a tile's weights per block of k

template <int kTok>
struct GemmShape {
  static_assert(kTok == 16 || kTok == 64 || kTok == 128, "the forms of gemm_form");
  static constexpr int kBoxRows = kTok == 16 ? 16 : kTok / 2;     // token rows of a copy
  static constexpr int kStageBytes = kWeightTile + kTok * kScaleBlock;
  static constexpr int kEpiWarps = kTok <= 64 ? 4 : 8;
  static constexpr int kCols = kTok / (kEpiWarps / 4);            // accumulator columns of a warp
  static constexpr int kBufCols = kTok < 32 ? 32 : kTok;
  static constexpr int kAccBufs = 4;                              // accumulators: blocks of k under way
  static constexpr int kTmemCols = kAccBufs * kBufCols;
  static constexpr int kThreads = (kEpiWarps + 3) * 32;           // + copies, MMA, scales
  static constexpr int kPartPitch = kScaleBlock + 4;              // floats of a token's partial sums: no bank conflicts
  static constexpr int kOutPitch = 80;                            // bytes of 32 16-bit outputs of a token, the same
  static constexpr int kOutCols = kCols < 32 ? kCols : 32;        // tokens of a warp that are on their way out at once
  static constexpr int kOutWarp = kOutCols * kOutPitch;
  static constexpr int kRing = kGemmRingBytes - kEpiWarps * kOutWarp - kScaleSlots * kScaleBlocks * kTok * 4;
  static constexpr int kStages = kRing / kStageBytes < 12 ? kRing / kStageBytes : 12;
  static constexpr int kScaleOff = kStages * kStageBytes;
  static constexpr int kOutOff = kScaleOff + kScaleSlots * kScaleBlocks * kTok * 4;
  static constexpr int kPlanOff = kOutOff + kEpiWarps * kOutWarp;  // [2]: a tile's GemmTile and the bias of its weight rows
  static constexpr int kPlanBytes = 16 + kScaleBlock * 4;
  static constexpr int kBarOff = kPlanOff + 2 * kPlanBytes;
  static constexpr int kBars = 2 * kStages + 2 * kAccBufs + 2 * kScaleSlots + 4;
  static constexpr int kSmem = kBarOff + 8 * kBars + 1024;        // + slack to align the ring
  static_assert(kTok * kPartPitch * 4 <= kStages * kStageBytes, "a split's partial tile reuses the ring");
  static_assert(kSmem + 4608 <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void fma_f32x2(uint64_t &acc, uint32_t lo, uint32_t hi, uint64_t f) {
  asm("{\n\t.reg .b64 v;\n\tmov.b64 v, {%1, %2};\n\tfma.rn.f32x2 %0, v, %3, %0;\n\t}" : "+l"(acc) : "r"(lo), "r"(hi), "l"(f));
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void store_out(const Fp8GemmArgs &p, size_t at, float v) {
  if (p.out_dtype == MOE_BF16) store_as(static_cast<__nv_bfloat16 *>(p.out) + at, v);
  else if (p.out_dtype == MOE_F16) store_as(static_cast<__half *>(p.out) + at, v);
  else store_as(static_cast<float *>(p.out) + at, v);
}

// Two neighbouring 16-bit outputs, of which `left` exist, where rows are aligned to `bytes`.
__device__ __forceinline__ void store_word16(uint16_t *dst, uint32_t w, int left, int bytes) {
  if (left >= 2 && bytes >= 4) {
    *reinterpret_cast<uint32_t *>(dst) = w;
  } else {
    if (left >= 1) dst[0] = static_cast<uint16_t>(w);
    if (left >= 2) dst[1] = static_cast<uint16_t>(w >> 16);
  }
}

constexpr int kMaxSplits = 8;   // CTAs of a cluster that share the reduction of a tile

// One tile: rows [row0, row0 + ntok) of group g against weight rows [128 nb, 128 nb + 128).
struct GemmTile {
  int g, nb, row0, ntok;
};

// A CTA's share of a split tile, kWidth output columns from n0: rows split, split + splits, ..., `mine` of them.  kAhead places of a
// thread are under way together: a load from another CTA's shared memory takes about a microsecond.  The few rows of the narrow
// kernel want less code instead: 128 x 4096 x 7168 13.6 us with one place, 14.2 with four.
template <int kWidth, int kThreads, int kAhead, int kMost>
__device__ __forceinline__ void add_up_splits(const Fp8GemmArgs &p, const GemmTile &t, uint32_t part, int pitch, int mine, int split, int n0, int out_bytes) {
  constexpr int kQuads = kWidth / 4;
  for (int e0 = threadIdx.x; e0 < mine * kQuads; e0 += kAhead * kThreads) {
    float4 v[kAhead][kMost];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int e = e0 + i * kThreads;
#pragma unroll
      for (int r = 0; r < kMost; ++r)
        if (e < mine * kQuads && r < p.splits)
          v[i][r] = ld_cluster_f32x4(map_to_cta(part + 4u * ((split + e / kQuads * p.splits) * pitch + e % kQuads * 4), r));
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int e = e0 + i * kThreads, row = split + e / kQuads * p.splits, n = n0 + e % kQuads * 4;
      if (e >= mine * kQuads) break;
      float4 sum = v[i][0];
#pragma unroll
      for (int r = 1; r < kMost; ++r)
        if (r < p.splits) { sum.x += v[i][r].x; sum.y += v[i][r].y; sum.z += v[i][r].z; sum.w += v[i][r].w; }   // in the order of k
      float o[4] = {sum.x, sum.y, sum.z, sum.w};
      if (p.bias != nullptr) {
        const __nv_bfloat16 *bias = p.bias + static_cast<size_t>(t.g) * p.n + n;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += n + j < p.n ? __bfloat162float(bias[j]) : 0.f;
      }
      const size_t at = static_cast<size_t>(t.row0 + row) * p.ld_out + n;
      if (p.out_dtype == MOE_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.n) static_cast<float *>(p.out)[at + j] = o[j];
      } else {
        uint16_t *dst = static_cast<uint16_t *>(p.out) + at;
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          store_word16(dst + j, p.out_dtype == MOE_BF16 ? pack2<__nv_bfloat16>(o[j], o[j + 1]) : pack2<__half>(o[j], o[j + 1]), p.n - n - j, out_bytes);
      }
    }
  }
}

// Offsets that are not ascending give wrong rows or none, never rows outside.
__device__ __forceinline__ int group_begin(const Fp8GemmArgs &p, int g) { return p.offsets == nullptr ? 0 : min(max(p.offsets[g], 0), p.rows); }
__device__ __forceinline__ int group_end(const Fp8GemmArgs &p, int g) { return p.offsets == nullptr ? p.rows : min(max(p.offsets[g + 1], 0), p.rows); }

// Token tiles of a group of cnt rows, and the rows of each of them: equal but for the last, in steps of 16.  (Unsigned: cnt may be
// near 2^31.)
__host__ __device__ constexpr int tiles_of(int cnt, unsigned tok) { return static_cast<int>((static_cast<unsigned>(cnt > 0 ? cnt : 0) + tok - 1) / tok); }
__host__ __device__ constexpr int rows_of_tile(unsigned cnt, unsigned tiles) { return static_cast<int>(((cnt + tiles - 1) / tiles + 15) / 16 * 16); }
constexpr int kMostRows = 0x7fffff00;   // of a call, and columns: with a tile more an index still fits an int
static_assert(tiles_of(0, 64) == 0 && tiles_of(-5, 64) == 0 && tiles_of(1, 64) == 1 && tiles_of(64, 64) == 1 && tiles_of(65, 64) == 2, "tiles");
static_assert(rows_of_tile(1, 1) == 16 && rows_of_tile(16, 1) == 16 && rows_of_tile(65, 2) == 48 && rows_of_tile(129, 2) == 80, "rows of a tile");
static_assert(rows_of_tile(kMostRows, tiles_of(kMostRows, 64)) == 64 && rows_of_tile(kMostRows, tiles_of(kMostRows, 128)) == 128, "the largest call");

// s_tiles[g] = token tiles of the groups before g, g = 0..n_groups.  Called by all threads, ends with a barrier.
template <int kTok>
__device__ __forceinline__ void count_tiles(const Fp8GemmArgs &p, int *s_tiles) {
  for (int g = threadIdx.x; g < p.n_groups; g += blockDim.x) s_tiles[g + 1] = tiles_of(group_end(p, g) - group_begin(p, g), kTok);
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int before = 0;
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
      int v = g0 + lane < p.n_groups ? s_tiles[g0 + lane + 1] : 0;
      for (int off = 1; off < 32; off <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += up;
      }
      if (g0 + lane < p.n_groups) s_tiles[g0 + lane + 1] = before + v;
      before += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) {
      s_tiles[0] = 0;
      // ascending offsets cannot give more (and what the host sized the grid for stays true)
      if (before < 0 || before > p.rows / kTok + p.n_groups) s_tiles[p.n_groups] = 0;
    }
  }
  __syncthreads();
}
// Item -> tile, of n_nb weight blocks per group: the token tiles of a weight block follow one another, in runs of kRunTiles of a
// group's tiles.  So the CTAs that are at work share a dozen token tiles and a dozen weight blocks: with all tiles of a group in
// one run 65536 x 4096 x 4096 took 1465 us (token rows again from HBM for every weight block), with 8 / 12 / 16 / 32 of them
// 1170 / 1140 / 1180 / 1170, 8192 x 4096 x 7168 233 and 226 / 224 / 227 / 226.  The tiles of a group are of equal size in steps of
// 16 rows; none is empty.
constexpr int kRunTiles = 12;
__device__ __forceinline__ GemmTile tile_at(const Fp8GemmArgs &p, const int *s_tiles, int item, int n_nb) {
  // (every role finds its first tile before anything else can happen: the divisions below are half a microsecond of a decode step)
  if (p.n_groups == 1 && s_tiles[1] == 1) return GemmTile{0, item, group_begin(p, 0), group_end(p, 0) - group_begin(p, 0)};
  const int q = item / n_nb;
  int lo = 0, hi = p.n_groups;   // s_tiles[lo] <= q < s_tiles[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_tiles[mid] <= q) lo = mid; else hi = mid;
  }
  const int tiles = s_tiles[lo + 1] - s_tiles[lo];
  const int local = item - s_tiles[lo] * n_nb;
  const int begin = group_begin(p, lo), cnt = group_end(p, lo) - begin;
  const int per = rows_of_tile(cnt, tiles);
  if (tiles <= kRunTiles) {
    const int nb = local / tiles, row = (local - nb * tiles) * per;
    return GemmTile{lo, nb, begin + row, min(per, cnt - row)};
  }
  const int run = local / (kRunTiles * n_nb), in_run = local - run * kRunTiles * n_nb, width = min(kRunTiles, tiles - run * kRunTiles);
  const int nb = in_run / width, row = (run * kRunTiles + in_run - nb * width) * per;
  return GemmTile{lo, nb, begin + row, min(per, cnt - row)};
}

template <int kTok>
__global__ void __launch_bounds__(GemmShape<kTok>::kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const Fp8GemmArgs p, const int out_bytes) {
  using S = GemmShape<kTok>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_tiles[kMaxGemmGroups + 1];   // token tiles of the groups before g
  __shared__ uint32_t s_tmem, s_abort;
  volatile uint32_t *abort_flag = &s_abort;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *ring_ptr = smem_raw + (ring - smem_u32(smem_raw));
  const uint32_t bars = ring + S::kBarOff;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (S::kStages + s); };
  auto dfull = [&](int d) { return bars + 8u * (2 * S::kStages + d); };
  auto dempty = [&](int d) { return bars + 8u * (2 * S::kStages + S::kAccBufs + d); };
  auto sfull = [&](int s) { return bars + 8u * (2 * S::kStages + 2 * S::kAccBufs + s); };
  auto sempty = [&](int s) { return bars + 8u * (2 * S::kStages + 2 * S::kAccBufs + kScaleSlots + s); };
  auto pfull = [&](int i) { return bars + 8u * (2 * S::kStages + 2 * S::kAccBufs + 2 * kScaleSlots + i); };
  auto pempty = [&](int i) { return bars + 8u * (2 * S::kStages + 2 * S::kAccBufs + 2 * kScaleSlots + 2 + i); };
  constexpr int kCopyWarp = S::kEpiWarps, kMmaWarp = kCopyWarp + 1, kScaleWarp = kCopyWarp + 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
    for (int d = 0; d < S::kAccBufs; ++d) { mbar_init(dfull(d), 1); mbar_init(dempty(d), S::kEpiWarps); }
    for (int s = 0; s < kScaleSlots; ++s) { mbar_init(sfull(s), 1); mbar_init(sempty(s), S::kEpiWarps); }
    for (int i = 0; i < 2; ++i) { mbar_init(pfull(i), 1); mbar_init(pempty(i), S::kEpiWarps); }
    s_abort = 0u;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&s_tmem), S::kTmemCols);
    tmem_relinquish();
  }
  if (warp == kCopyWarp && lane == 0) {
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
  }
  grid_dep_sync();   // from here on what other kernels wrote is read
  tc_fence_before();
  count_tiles<kTok>(p, s_tiles);
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  const int n_nb = (p.n + kScaleBlock - 1) / kScaleBlock;
  const int n_items = s_tiles[p.n_groups] * n_nb;   // far below 2^31: every tile has outputs
  // A split launch has a cluster per tile; otherwise the CTAs walk through the tiles, the token tiles of a weight block next
  // to one another, so that its weights come from L2 after the first.
  const int split = p.splits > 1 ? static_cast<int>(blockIdx.y) : 0;
  const int kb0 = static_cast<int>(static_cast<long long>(p.n_kb) * split / p.splits);
  const int kb1 = static_cast<int>(static_cast<long long>(p.n_kb) * (split + 1) / p.splits);
  const int stride = p.splits > 1 ? n_items : gridDim.x;   // a split CTA takes one tile
  auto tile_of = [&](int item) { return tile_at(p, s_tiles, item, n_nb); };
  bool ok = true;

  if (warp == kCopyWarp) {
    // ---- copies: the weights of a block of k, and as many boxes of token rows as the tile has
    uint32_t s = 0, par = 1u;
    for (int it = blockIdx.x; ok && it < n_items; it += stride) {
      const GemmTile t = tile_of(it);
      const int boxes = (t.ntok + S::kBoxRows - 1) / S::kBoxRows;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_warp(empty(s), par, abort_flag, p.status, ST_WAIT_EMPTY)) { ok = false; break; }
        if (elect_one()) {
          const uint32_t stage = ring + s * S::kStageBytes;
          mbar_arrive_expect_tx(full(s), kWeightTile + boxes * S::kBoxRows * kScaleBlock);
          tma_load_3d(stage, &tm_b, kb * kScaleBlock, t.nb * kScaleBlock, t.g, full(s));
          for (int i = 0; i < boxes; ++i)
            tma_load_2d(stage + kWeightTile + i * S::kBoxRows * kScaleBlock, &tm_a, kb * kScaleBlock, t.row0 + i * S::kBoxRows, full(s));
        }
        __syncwarp();
        if (++s == S::kStages) { s = 0; par ^= 1u; }
      }
    }
  } else if (warp == kMmaWarp) {
    // ---- MMA: every block of k into the next of the accumulators
    uint32_t s = 0, par = 0, d = 0, dpar = 1u;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t desc = smem_desc_sw128(0);
    for (int it = blockIdx.x; ok && it < n_items; it += stride) {
      const uint32_t idesc = __shfl_sync(0xffffffffu, idesc_e4m3(kScaleBlock, (tile_of(it).ntok + 15) / 16 * 16), 0);   // uniform
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_warp(full(s), par, abort_flag, p.status, ST_WAIT_FULL)) { ok = false; break; }
        if (!mbar_wait_warp(dempty(d), dpar, abort_flag, p.status, ST_WAIT_DEMPTY)) { ok = false; break; }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t stage = ring + s * S::kStageBytes, acc = tm + d * S::kBufCols;
          const uint64_t wd = desc | (stage >> 4), xd = desc | ((stage + kWeightTile) >> 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) mma_f8(acc, wd + 2 * i, xd + 2 * i, idesc, i > 0);
          mma_commit(empty(s));
          mma_commit(dfull(d));
        }
        __syncwarp();
        if (++s == S::kStages) { s = 0; par ^= 1u; }
        if (++d == S::kAccBufs) { d = 0; dpar ^= 1u; }
      }
    }
  } else if (warp == kScaleWarp) {
    // ---- scales of the tile's tokens times the block's own, kScaleBlocks blocks of k to a slot
    constexpr int kPer = kTok < 32 ? 1 : kTok / 32;   // tokens of a lane
    uint32_t s = 0, par = 1u, plan = 0, ppar = 1u;
    float *slots = reinterpret_cast<float *>(ring_ptr + S::kScaleOff);
    for (int it = blockIdx.x; ok && it < n_items; it += stride) {
      const GemmTile t = tile_of(it);
      float bias[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = t.nb * kScaleBlock + 32 * i + lane;
        bias[i] = p.bias != nullptr && n < p.n ? __bfloat162float(p.bias[static_cast<size_t>(t.g) * p.n + n]) : 0.f;
      }
      if (!mbar_wait_warp(pempty(plan), ppar, abort_flag, p.status, ST_WAIT_AFREE)) { ok = false; break; }
      uint8_t *at = ring_ptr + S::kPlanOff + plan * S::kPlanBytes;
      if (lane == 0) *reinterpret_cast<GemmTile *>(at) = t;
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<float *>(at + 16)[32 * i + lane] = bias[i];
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull(plan));
      if (plan ^= 1u; plan == 0) ppar ^= 1u;
      const float *sb = p.sb + (static_cast<size_t>(t.g) * n_nb + t.nb) * p.n_kb;
      for (int k0 = kb0; ok && k0 < kb1; k0 += kScaleBlocks) {
        const float b = lane < kScaleBlocks && k0 + lane < kb1 ? sb[k0 + lane] : 0.f;
        float v[kPer][kScaleBlocks];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int tok = lane + 32 * i;
          const float *sa = p.sa + static_cast<size_t>(t.row0 + tok) * p.ld_sa + k0;
#pragma unroll
          for (int j = 0; j < kScaleBlocks; ++j) v[i][j] = tok < t.ntok && k0 + j < kb1 ? sa[j] : 0.f;
        }
        if (!mbar_wait_warp(sempty(s), par, abort_flag, p.status, ST_WAIT_AFREE)) { ok = false; break; }
#pragma unroll
        for (int j = 0; j < kScaleBlocks; ++j) {
          const float f = __shfl_sync(0xffffffffu, b, j);
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (lane + 32 * i < kTok) slots[(s * kScaleBlocks + j) * kTok + lane + 32 * i] = v[i][j] * f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(sfull(s));
        if (++s == kScaleSlots) { s = 0; par ^= 1u; }
      }
    }
  } else {
    // ---- sums over the blocks: warp w has weight rows 32 (w % 4) .. + 31 and kCols token columns, as fragments: of the columns
    // 8 j .. 8 j + 7 and rows 16 h + 8 i + lane / 4 the pair 2 (lane % 4), + 1 is acc[j][h][i]
    const int quad = warp & 3, col0 = (warp >> 2) * S::kCols, pair0 = 2 * (lane & 3);
    const uint32_t lane_field = static_cast<uint32_t>(quad * 32) << 16;
    const float *slots = reinterpret_cast<const float *>(ring_ptr + S::kScaleOff) + col0 + pair0;
    uint32_t d = 0, dpar = 0, s = 0, spar = 0, plan = 0, ppar = 0;
    for (int it = blockIdx.x; ok && it < n_items; it += stride) {
      if (!mbar_wait_warp(pfull(plan), ppar, abort_flag, p.status, ST_WAIT_AREADY)) { ok = false; break; }
      const uint8_t *at = ring_ptr + S::kPlanOff + plan * S::kPlanBytes;
      const GemmTile t = *reinterpret_cast<const GemmTile *>(at);
      uint64_t acc[S::kCols / 8][2][2];
#pragma unroll
      for (int j = 0; j < S::kCols / 8; ++j) acc[j][0][0] = acc[j][0][1] = acc[j][1][0] = acc[j][1][1] = 0ull;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int kq = (kb - kb0) % kScaleBlocks;
        if (kq == 0 && !mbar_wait_warp(sfull(s), spar, abort_flag, p.status, ST_WAIT_AREADY)) { ok = false; break; }
        if (!mbar_wait_warp(dfull(d), dpar, abort_flag, p.status, ST_WAIT_DFULL)) { ok = false; break; }
        tc_fence_after();
        const uint32_t src = tmem + lane_field + d * S::kBufCols + col0;
        const float *f = slots + (s * kScaleBlocks + kq) * kTok;
        constexpr int kLd = S::kCols < 32 ? 16 : 32;   // columns of a load
        uint32_t v[S::kCols / kLd][2][kLd / 2];
#pragma unroll
        for (int l = 0; l < S::kCols / kLd; ++l)
          if (col0 + l * kLd < t.ntok) {
            tmem_ld_frag(src + l * kLd, v[l][0]);
            tmem_ld_frag(src + l * kLd + (16u << 16), v[l][1]);
          }
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dempty(d));
#pragma unroll
        for (int l = 0; l < S::kCols / kLd; ++l)
          if (col0 + l * kLd < t.ntok) {
#pragma unroll
            for (int j = 0; j < kLd / 8; ++j) {
              const uint64_t f2 = *reinterpret_cast<const uint64_t *>(f + l * kLd + 8 * j);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) fma_f32x2(acc[l * kLd / 8 + j][h][i], v[l][h][4 * j + 2 * i], v[l][h][4 * j + 2 * i + 1], f2);
            }
          }
        if (kq == kScaleBlocks - 1 || kb + 1 == kb1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty(s));
          if (++s == kScaleSlots) { s = 0; spar ^= 1u; }
        }
        if (++d == S::kAccBufs) { d = 0; dpar ^= 1u; }
      }
      if (!ok) break;
      const int n_w = t.nb * kScaleBlock + quad * 32;   // first weight row of the warp
      auto value = [&](int j, int h, int i, int c) { return __uint_as_float(static_cast<uint32_t>(acc[j][h][i] >> (32 * c))); };
      if (p.splits > 1) {
        // every MMA of this CTA is complete: the ring takes the partial tile, [token][weight row]
        float *part = reinterpret_cast<float *>(ring_ptr);
#pragma unroll
        for (int j = 0; j < S::kCols / 8; ++j)
          if (col0 + 8 * j < t.ntok) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int h = e >> 2, i = (e >> 1) & 1, c = e & 1;
              part[(col0 + 8 * j + pair0 + c) * S::kPartPitch + quad * 32 + 16 * h + 8 * i + (lane >> 2)] = value(j, h, i, c);
            }
          }
        break;   // a split CTA has one tile
      }
      float b[2][2];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e >> 1][e & 1] = reinterpret_cast<const float *>(at + 16)[quad * 32 + 8 * e + (lane >> 2)];
      __syncwarp();
      if (lane == 0) mbar_arrive(pempty(plan));
      if (plan ^= 1u; plan == 0) ppar ^= 1u;
      if (p.out_dtype != MOE_F32) {
        // 16-bit outputs: blocks of 8 tokens x 32 weight rows are transposed in shared memory and leave as 16 bytes a lane, or as 4 (2
        // where the output's rows are not aligned to that)
        const uint32_t stage = ring + S::kOutOff + warp * S::kOutWarp;
        const uint32_t st_at = stage + (lane & 7) * S::kOutPitch + (lane >> 3) * 16;
        const int ntok = t.ntok - col0;
#pragma unroll
        for (int j0 = 0; j0 < S::kCols / 8; j0 += S::kOutCols / 8) {
          if (8 * j0 >= ntok) break;
          __syncwarp();
#pragma unroll
          for (int j = 0; j < S::kOutCols / 8; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int h = e >> 1, i = e & 1;
              const float x = value(j0 + j, h, i, 0) + b[h][i], y = value(j0 + j, h, i, 1) + b[h][i];
              w[e] = p.out_dtype == MOE_BF16 ? pack2<__nv_bfloat16>(x, y) : pack2<__half>(x, y);
            }
            stmatrix_trans_x4(st_at + j * 8 * S::kOutPitch, w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          // (32 experts of 1440 x 2880: 48 rows each 33.4 us with 16 bytes, 35.4 with 4; but 32 rows each, in the smaller form, 34.1 and
          // 32.8, and 64 x 4096 x 7168 11.3 and 10.7: there the code's size counts more)
          if (kTok == 128 && out_bytes == 16) {
            const int n = n_w + (lane & 3) * 8;
            const uint32_t ld_at = stage + (lane >> 2) * S::kOutPitch + (lane & 3) * 16;
            uint16_t *dst = static_cast<uint16_t *>(p.out) + static_cast<size_t>(t.row0 + col0 + 8 * j0 + (lane >> 2)) * p.ld_out + n;
#pragma unroll
            for (int j = 0; j < S::kOutCols / 8; ++j, dst += 8 * p.ld_out) {
              if (8 * (j0 + j) + (lane >> 2) >= ntok || n >= p.n) continue;
              uint32_t o[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(ld_at + j * 8 * S::kOutPitch) : "memory");
              if (n + 8 <= p.n) {
                *reinterpret_cast<uint4 *>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (n + e < p.n) dst[e] = static_cast<uint16_t>(o[e / 2] >> (16 * (e & 1)));
              }
            }
            continue;
          }
          const int here = min(ntok - 8 * j0, S::kOutCols), n = (lane & 15) * 2;
          uint16_t *dst = static_cast<uint16_t *>(p.out) + static_cast<size_t>(t.row0 + col0 + 8 * j0 + (lane >> 4)) * p.ld_out + n_w + n;
          for (int tok = lane >> 4; tok < here; tok += 2, dst += 2 * p.ld_out) {
            uint32_t o;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(o) : "r"(stage + tok * S::kOutPitch + n * 2) : "memory");
            store_word16(dst, o, p.n - n_w - n, out_bytes);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < S::kCols / 8; ++j) {
          if (col0 + 8 * j >= t.ntok) break;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int h = e >> 2, i = (e >> 1) & 1, c = e & 1, tok = col0 + 8 * j + pair0 + c, n = n_w + 16 * h + 8 * i + (lane >> 2);
            if (tok < t.ntok && n < p.n) store_out(p, static_cast<size_t>(t.row0 + tok) * p.ld_out + n, value(j, h, i, c) + b[h][i]);
          }
        }
      }
    }
  }
  __syncwarp();
  if (p.splits > 1) {
    // the CTAs of the cluster add up the tile, each its share of the tokens, in the order of k
    cluster_sync_all();
    const int it = blockIdx.x;
    if (it < n_items) {
      const GemmTile t = tile_of(it);
      const uint32_t base = smem_u32(ring_ptr);
      const int mine = (t.ntok - split + p.splits - 1) / p.splits;
      if (p.splits <= 4) add_up_splits<kScaleBlock, S::kThreads, 1, 4>(p, t, base, S::kPartPitch, mine, split, t.nb * kScaleBlock, out_bytes);
      else add_up_splits<kScaleBlock, S::kThreads, 1, kMaxSplits>(p, t, base, S::kPartPitch, mine, split, t.nb * kScaleBlock, out_bytes);
    }
    cluster_sync_all();   // no CTA leaves while another may still read its part
  }
  if (!ok && warp == kCopyWarp)   // give copies in flight time to land before shared memory is released
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Many rows per group: 128 token rows (a lane of tensor memory each) x 256 weight rows.  Eight epilogue warps: a quadrant of the rows
// and a half of the columns, which is a row of scale blocks; a warp each for copies, MMAs, and scales and bias.
// ---------------------------------------------------------------------------
constexpr int kWideTok = 128, kWideN = 256;
constexpr int kWideTile = kWideTok * kScaleBlock;                       // bytes of the token rows of a block of k
constexpr int kWideStage = kWideTile + kWideN * kScaleBlock, kWideStages = 3, kWideAccBufs = 2;
constexpr int kWideEpiWarps = 8, kWideThreads = (kWideEpiWarps + 3) * 32;
constexpr int kWidePart = kWideN + 4;                      // floats of a row of a split's partial tile: no bank conflicts
constexpr int kWideCols = kWideN / (kWideEpiWarps / 4);
constexpr int kOutBox = 32 * 128;                          // outputs of a warp on their way out: 32 rows of 128 bytes
constexpr int kWideOutOff = kWideStages * kWideStage;
constexpr int kWideBiasOff = kWideOutOff + kWideEpiWarps * kOutBox;
constexpr int kWideScaleOff = kWideBiasOff + 2 * kWideN * 4;
constexpr int kWideScaleSlot = 2 * kScaleBlocks * 128;
constexpr int kWideBarOff = kWideScaleOff + kScaleSlots * kWideScaleSlot * 4;
constexpr int kWideBars = 2 * kWideStages + 2 * kWideAccBufs + 2 * kScaleSlots + 4;
constexpr int kWideSmem = kWideBarOff + 8 * kWideBars + 1024;
static_assert(kWideCols == kScaleBlock, "one sb per warp and block of k");
static_assert(kWideTok * kWidePart * 4 <= kWideStages * kWideStage, "a split's partial tile reuses the ring");
static_assert(kWideSmem + 4608 <= 227 * 1024, "shared memory");

// What the copy engine would do with a box of staged outputs (128-byte swizzle), by a warp: rows [0, rows) to output rows row0..
// and columns n..; 16 bytes a lane where the output's rows are aligned to that, else 4 or 2.
__device__ __forceinline__ void copy_box(const Fp8GemmArgs &p, const uint8_t *box, int row0, int rows, int n, int out_bytes) {
  const int lane = threadIdx.x & 31, size = p.out_dtype == MOE_F32 ? 4 : 2, per = 16 / size;
  if (out_bytes == 16) {
    for (int i = lane; i < rows * 8; i += 32) {   // (row, 16-byte piece)
      const int r = i / 8, piece = i % 8, col = n + piece * per;
      const uint4 v = *reinterpret_cast<const uint4 *>(box + r * 128 + ((piece ^ (r & 7)) << 4));
      const size_t at = static_cast<size_t>(row0 + r) * p.ld_out + col;
      if (col + per <= p.n) {
        *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(p.out) + at * size) = v;
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= per || col + j >= p.n) break;
          if (size == 4) static_cast<uint32_t *>(p.out)[at + j] = w[j & 3];
          else static_cast<uint16_t *>(p.out)[at + j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
        }
      }
    }
    return;
  }
  const int col = n + lane * 4 / size;   // a 4-byte word a lane, eight rows at a time
  for (int r0 = 0; r0 < rows; r0 += 8) {
    uint32_t w[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) w[r] = *reinterpret_cast<const uint32_t *>(box + (r0 + r) * 128 + ((lane / 4 ^ r) << 4) + lane % 4 * 4);
    size_t at = static_cast<size_t>(row0 + r0) * p.ld_out + col;
#pragma unroll
    for (int r = 0; r < 8; ++r, at += p.ld_out) {
      if (r0 + r >= rows) break;
      if (size == 2) store_word16(static_cast<uint16_t *>(p.out) + at, w[r], p.n - col, out_bytes);
      else if (col < p.n) static_cast<uint32_t *>(p.out)[at] = w[r];
    }
  }
}

// Boxes that leave by the copy engine: none, those that lie in the output whole, all.
enum { kTiledNone = 0, kTiledWhole = 1, kTiledAll = 2 };

// kSplit: a cluster of p.splits CTAs, blockIdx.y of them, shares the reduction of one tile.
template <bool kSplit>
__global__ void __launch_bounds__(kWideThreads, 1)
fp8_gemm_wide_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_out,
                     const Fp8GemmArgs p, const int tiled_out, const int out_bytes) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_tiles[kMaxGemmGroups + 1];
  __shared__ uint32_t s_tmem, s_abort;
  volatile uint32_t *abort_flag = &s_abort;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float *s_bias = reinterpret_cast<float *>(smem_raw + (ring - smem_u32(smem_raw)) + kWideBiasOff);   // [2][kWideN]
  float *s_scales = reinterpret_cast<float *>(smem_raw + (ring - smem_u32(smem_raw)) + kWideScaleOff);
  const uint32_t bars = ring + kWideBarOff;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (kWideStages + s); };
  auto dfull = [&](int d) { return bars + 8u * (2 * kWideStages + d); };
  auto dempty = [&](int d) { return bars + 8u * (2 * kWideStages + kWideAccBufs + d); };
  constexpr int kSideBars = 2 * kWideStages + 2 * kWideAccBufs;
  auto bfull = [&](int i) { return bars + 8u * (kSideBars + i); };
  auto bempty = [&](int i) { return bars + 8u * (kSideBars + 2 + i); };
  auto sfull = [&](int i) { return bars + 8u * (kSideBars + 4 + i); };
  auto sempty = [&](int i) { return bars + 8u * (kSideBars + 4 + kScaleSlots + i); };
  constexpr int kCopyWarp = kWideEpiWarps, kSideWarp = kCopyWarp + 1, kMmaWarp = kCopyWarp + 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kWideStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
    for (int d = 0; d < kWideAccBufs; ++d) { mbar_init(dfull(d), 1); mbar_init(dempty(d), kWideEpiWarps); }
    for (int i = 0; i < 2; ++i) { mbar_init(bfull(i), 1); mbar_init(bempty(i), kWideEpiWarps); }
    for (int i = 0; i < kScaleSlots; ++i) { mbar_init(sfull(i), 1); mbar_init(sempty(i), kWideEpiWarps); }
    s_abort = 0u;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&s_tmem), kWideAccBufs * kWideN);
    tmem_relinquish();
  }
  if (warp == kCopyWarp && lane == 0) {
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
    if (tiled_out) prefetch_tensormap(&tm_out);
  }
  grid_dep_sync();   // from here on what other kernels wrote is read
  tc_fence_before();
  count_tiles<kWideTok>(p, s_tiles);
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int n_nb = (p.n + kWideN - 1) / kWideN, n_sb = (p.n + kScaleBlock - 1) / kScaleBlock;
  const int n_items = s_tiles[p.n_groups] * n_nb;
  const int first = blockIdx.x, stride = kSplit ? n_items : gridDim.x;   // a split CTA takes one tile
  const int split = kSplit ? static_cast<int>(blockIdx.y) : 0;
  const int kb0 = kSplit ? static_cast<int>(static_cast<long long>(p.n_kb) * split / p.splits) : 0;
  const int kb1 = kSplit ? static_cast<int>(static_cast<long long>(p.n_kb) * (split + 1) / p.splits) : p.n_kb;
  bool ok = true;

  if (warp >= kWideEpiWarps) {
    if (warp == kCopyWarp) {
      uint32_t s = 0, par = 1u;
      for (int it = first; ok && it < n_items; it += stride) {
        const GemmTile t = tile_at(p, s_tiles, it, n_nb);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_warp(empty(s), par, abort_flag, p.status, ST_WAIT_EMPTY)) { ok = false; break; }
          if (elect_one()) {
            const uint32_t stage = ring + s * kWideStage;
            mbar_arrive_expect_tx(full(s), kWideStage);
            tma_load_2d(stage, &tm_a, kb * kScaleBlock, t.row0, full(s));
            tma_load_3d(stage + kWideTile, &tm_b, kb * kScaleBlock, t.nb * kWideN, t.g, full(s));
          }
          __syncwarp();
          if (++s == kWideStages) { s = 0; par ^= 1u; }
        }
      }
    } else if (warp == kMmaWarp) {
      uint32_t s = 0, par = 0, d = 0, dpar = 1u;
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t desc = smem_desc_sw128(0);
      constexpr uint32_t idesc = idesc_e4m3(128, kWideN);
      for (int it = first; ok && it < n_items; it += stride) {
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_warp(full(s), par, abort_flag, p.status, ST_WAIT_FULL)) { ok = false; break; }
          if (!mbar_wait_warp(dempty(d), dpar, abort_flag, p.status, ST_WAIT_DEMPTY)) { ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t stage = ring + s * kWideStage, acc = tm + d * kWideN;
            const uint64_t xd = desc | (stage >> 4), wd = desc | ((stage + kWideTile) >> 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma_f8(acc, xd + 2 * i, wd + 2 * i, idesc, i > 0);
            mma_commit(dfull(d));
            mma_commit(empty(s));
          }
          __syncwarp();
          if (++s == kWideStages) { s = 0; par ^= 1u; }
          if (++d == kWideAccBufs) { d = 0; dpar ^= 1u; }
        }
      }
    }
    if (warp == kSideWarp) {
      // ---- bias as fp32, and the products of both scales: for every row of this CTA and either half of the columns
      uint32_t buf = 0, bpar = 1u, s = 0, par = 1u;
      for (int it = first; ok && it < n_items; it += stride) {
        const GemmTile t = tile_at(p, s_tiles, it, n_nb);
        // rows and weight blocks that do not exist take the scales of the last one: their sums go nowhere
        const float *sb0 = p.sb + (static_cast<size_t>(t.g) * n_sb + 2 * t.nb) * p.n_kb, *sb1 = 2 * t.nb + 1 < n_sb ? sb0 + p.n_kb : sb0;
        float bias[kWideN / 32];
#pragma unroll
        for (int i = 0; i < kWideN / 32; ++i) {
          const int n = t.nb * kWideN + 32 * i + lane;
          bias[i] = p.bias != nullptr && n < p.n ? __bfloat162float(p.bias[static_cast<size_t>(t.g) * p.n + n]) : 0.f;
        }
        for (int k0 = kb0; ok && k0 < kb1; k0 += kScaleBlocks) {
          const bool mine = lane < kScaleBlocks && k0 + lane < kb1;
          const float b0 = mine ? sb0[k0 + lane] : 0.f, b1 = mine ? sb1[k0 + lane] : 0.f;
          float v[4][kScaleBlocks];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float *sa = p.sa + static_cast<size_t>(t.row0 + min(32 * r + lane, t.ntok - 1)) * p.ld_sa + k0;
#pragma unroll
            for (int j = 0; j < kScaleBlocks; ++j) v[r][j] = k0 + j < kb1 ? sa[j] : 0.f;
          }
          if (!mbar_wait_warp(sempty(s), par, abort_flag, p.status, ST_WAIT_AFREE)) { ok = false; break; }
          float *dst = s_scales + s * kWideScaleSlot + lane;
#pragma unroll
          for (int j = 0; j < kScaleBlocks; ++j) {
            const float f0 = __shfl_sync(0xffffffffu, b0, j), f1 = __shfl_sync(0xffffffffu, b1, j);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              dst[j * 128 + 32 * r] = v[r][j] * f0;
              dst[(kScaleBlocks + j) * 128 + 32 * r] = v[r][j] * f1;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(sfull(s));
          if (++s == kScaleSlots) { s = 0; par ^= 1u; }
        }
        if (!ok || !mbar_wait_warp(bempty(buf), bpar, abort_flag, p.status, ST_WAIT_AFREE)) { ok = false; break; }
#pragma unroll
        for (int i = 0; i < kWideN / 32; ++i) s_bias[buf * kWideN + 32 * i + lane] = bias[i];
        __syncwarp();
        if (lane == 0) mbar_arrive(bfull(buf));
        if (buf ^= 1u; buf == 0) bpar ^= 1u;
      }
    }
  } else {
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t src0 = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * kWideCols;
    const uint32_t out_smem = ring + kWideOutOff + warp * kOutBox;
    const uint32_t out_lane = out_smem + lane * 128 + ((lane & 7) << 4);   // piece i of the lane's row: at this address ^ 16 i
    const uint8_t *out_gen = smem_raw + (out_smem - smem_u32(smem_raw));
    uint32_t d = 0, dpar = 0, buf = 0, bpar = 0, s = 0, spar = 0;
    for (int it = first; it < n_items; it += stride) {
      const GemmTile t = tile_at(p, s_tiles, it, n_nb);
      const int n0 = t.nb * kWideN + half * kWideCols;
      uint64_t acc[kWideCols / 2];
#pragma unroll
      for (int c = 0; c < kWideCols / 2; ++c) acc[c] = 0ull;
      for (int kb = kb0; kb < kb1; ++kb) {
        if ((kb - kb0) % kScaleBlocks == 0 && !mbar_wait_warp(sfull(s), spar, abort_flag, p.status, ST_WAIT_AREADY)) { ok = false; break; }
        const float scale = s_scales[s * kWideScaleSlot + (half * kScaleBlocks + (kb - kb0) % kScaleBlocks) * 128 + quad * 32 + lane];
        uint64_t f;
        asm("mov.b64 %0, {%1, %1};" : "=l"(f) : "r"(__float_as_uint(scale)));
        if (!mbar_wait_warp(dfull(d), dpar, abort_flag, p.status, ST_WAIT_DFULL)) { ok = false; break; }
        tc_fence_after();
        const uint32_t src = src0 + d * kWideN;
        uint32_t v[2][16];
        tmem_ld16(src, v[0]);
#pragma unroll
        for (int c = 0; c < kWideCols / 16; ++c) {   // the next 16 columns are on their way while these are added
          tmem_wait_ld();
          if (c + 1 < kWideCols / 16) {
            tmem_ld16(src + 16 * (c + 1), v[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(dempty(d));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) fma_f32x2(acc[8 * c + i], v[c & 1][2 * i], v[c & 1][2 * i + 1], f);
        }
        if ((kb - kb0) % kScaleBlocks == kScaleBlocks - 1 || kb + 1 == kb1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty(s));
          if (++s == kScaleSlots) { s = 0; spar ^= 1u; }
        }
        if (++d == kWideAccBufs) { d = 0; dpar ^= 1u; }
      }
      if (!ok) break;
      if constexpr (kSplit) {   // every MMA of this CTA is complete: the ring takes the partial tile
        float4 *part = reinterpret_cast<float4 *>(smem_raw + (ring - smem_u32(smem_raw))) + (quad * 32 + lane) * (kWidePart / 4) + half * (kWideCols / 4);
#pragma unroll
        for (int c = 0; c < kWideCols / 4; ++c)
          part[c] = make_float4(__uint_as_float(static_cast<uint32_t>(acc[2 * c])), __uint_as_float(static_cast<uint32_t>(acc[2 * c] >> 32)),
                                __uint_as_float(static_cast<uint32_t>(acc[2 * c + 1])), __uint_as_float(static_cast<uint32_t>(acc[2 * c + 1] >> 32)));
        break;
      }
      // Through shared memory, a box of 32 rows x 128 bytes at a time: 64 16-bit columns or 32 fp32 ones.  Rows that all exist
      // leave by the copy engine while the next box, or tile, is under way, others (and outputs that it cannot address) by the warp.
      // The engine writes whole 16-byte pieces, so a last box that ends inside one leaves by the warp too (8192 x 512 deep, rows of 4104
      // bf16: 4104 columns 38.3 us, 4097 to 4103 39.7 to 40.6).
      const int rows_here = t.ntok - quad * 32, row_out = t.row0 + quad * 32;
      const bool by_copy = tiled_out && rows_here >= 32;
      if (!mbar_wait_warp(bfull(buf), bpar, abort_flag, p.status, ST_WAIT_AREADY)) { ok = false; break; }
      const float4 *bias = reinterpret_cast<const float4 *>(s_bias + buf * kWideN + half * kWideCols);
      auto sums = [&](int c) {   // four columns with their bias
        const float4 b = bias[c];
        return make_float4(__uint_as_float(static_cast<uint32_t>(acc[2 * c])) + b.x, __uint_as_float(static_cast<uint32_t>(acc[2 * c] >> 32)) + b.y,
                           __uint_as_float(static_cast<uint32_t>(acc[2 * c + 1])) + b.z, __uint_as_float(static_cast<uint32_t>(acc[2 * c + 1] >> 32)) + b.w);
      };
      // (the address is formed inside the statement: eight of them, kept across the loop over k, would cost registers there)
      auto stage = [&](int piece, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
        asm volatile("{\n\t.reg .b32 at;\n\txor.b32 at, %0, %1;\n\tst.shared.v4.b32 [at], {%2, %3, %4, %5};\n\t}" ::"r"(out_lane), "r"(piece << 4),
                     "r"(w0), "r"(w1), "r"(w2), "r"(w3)
                     : "memory");
      };
      auto box_free = [&]() {
        if (lane == 0) tma_store_wait_read();
        __syncwarp();
      };
      auto leave = [&](int n, int box_cols) {
        fence_proxy_async_smem();
        __syncwarp();
        if (by_copy && (tiled_out == kTiledAll || n + box_cols <= p.n)) {
          if (lane == 0 && n < p.n) {
            tma_store_2d(&tm_out, n, row_out, out_smem);
            tma_store_commit();
          }
        } else {
          copy_box(p, out_gen, row_out, min(rows_here, 32), n, out_bytes);
        }
      };
      if (p.out_dtype == MOE_F32) {
#pragma unroll
        for (int c = 0; c < kWideCols / 4; ++c) {
          if (c % 8 == 0) box_free();
          const float4 v = sums(c);
          stage(c % 8, __float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w));
          if (c % 8 == 7) leave(n0 + 4 * (c - 7), 32);
        }
      } else {
        const bool bf16 = p.out_dtype == MOE_BF16;
        auto pack = [&](float lo, float hi) { return bf16 ? pack2<__nv_bfloat16>(lo, hi) : pack2<__half>(lo, hi); };
#pragma unroll
        for (int c = 0; c < kWideCols / 8; ++c) {
          if (c % 8 == 0) box_free();
          const float4 v = sums(2 * c), u = sums(2 * c + 1);
          stage(c % 8, pack(v.x, v.y), pack(v.z, v.w), pack(u.x, u.y), pack(u.z, u.w));
          if (c % 8 == 7) leave(n0 + 8 * (c - 7), 64);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bempty(buf));
      if (buf ^= 1u; buf == 0) bpar ^= 1u;
    }
    if (lane == 0) tma_store_wait_all();
  }
  __syncwarp();
  if constexpr (kSplit) {
    // the CTAs of the cluster add up the tile, each its share of the rows, in the order of k
    cluster_sync_all();
    if (first < n_items) {
      const GemmTile t = tile_at(p, s_tiles, first, n_nb);
      const int mine = (t.ntok - split + p.splits - 1) / p.splits;
      if (p.splits <= 4) add_up_splits<kWideN, kWideThreads, 4, 4>(p, t, ring, kWidePart, mine, split, t.nb * kWideN, out_bytes);
      else add_up_splits<kWideN, kWideThreads, 2, kMaxSplits>(p, t, ring, kWidePart, mine, split, t.nb * kWideN, out_bytes);
    }
    cluster_sync_all();   // no CTA leaves while another may still read its part
  }
  if (!ok && warp == kCopyWarp)   // give copies in flight time to land before shared memory is released
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kWideAccBufs * kWideN);
  }
}

namespace {

// Codes as rows of k bytes with the 128-byte swizzle of the tensor core: [groups, rows, k], a copy takes box_rows x 128.
bool encode_codes(CUtensorMap *m, const uint8_t *base, int k, long long ld, int rows, int groups, int box_rows) {
  TensorMapEncodeFn fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(groups)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld), static_cast<cuuint64_t>(ld) * rows};
  const cuuint32_t box[3] = {kScaleBlock, static_cast<cuuint32_t>(box_rows), 1}, es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, groups > 0 ? 3 : 2, const_cast<uint8_t *>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Outputs [rows, n], stored as boxes of 32 rows x 128 bytes.
bool encode_out(CUtensorMap *m, const Fp8GemmArgs &p) {
  TensorMapEncodeFn fn = tensor_map_encoder();
  if (!fn) return false;
  const int size = dtype_size(p.out_dtype);
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.n), static_cast<cuuint64_t>(p.rows)}, strides[1] = {static_cast<cuuint64_t>(p.ld_out) * size};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / size), 32}, es[2] = {1, 1};
  return fn(m, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.out, dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Bytes that the output's rows are aligned to: 16, 4 or the size of an element.
int out_alignment(const Fp8GemmArgs &p) {
  const int size = dtype_size(p.out_dtype);
  for (int bytes : {16, 4})
    if (aligned_to(p.out, bytes) && p.ld_out * size % bytes == 0) return bytes;
  return size;
}

struct GemmCall {
  const uint8_t *a, *b;
  long long ld_a, ld_b;
  int k;
  Fp8GemmArgs p;
};

// CTAs that share the reduction of a tile where the call has at most `tiles`: 1, 2 or 4, as many as give no SM more than one, and 8 of
// up to a dozen tiles with four blocks of k for each.  More clusters of eight, and any of three, do not all fit the device at once
// although their CTAs would: 393 x 3011 x 6502 (48 tiles) in two 32 us, in three 42; 512 x 512 x 2048 (16 tiles) in four 8.5 us, in
// eight 17.5; 16 rows of 1536 (12 tiles): 7168 deep 7.6 in four and 6.4 in eight, 2048 deep 5.2 and 5.6.
int k_splits(long long tiles, int n_kb, int sm_count) {
  int splits = 1;
  while (splits < 4 && tiles * splits * 2 <= sm_count && splits * 2 <= n_kb) splits *= 2;
  return splits == 4 && tiles <= 12 && tiles * kMaxSplits <= sm_count && n_kb >= 4 * kMaxSplits ? kMaxSplits : splits;
}

// Which kernel.  Groups: by the rows that one has on average (their numbers are on the device).  us, the kernel with 64 / 128 token
// columns / the wide one, 32 groups of 5760 x 2880: 8 rows each 85 / 89 / 96, 32 rows 93 / 94 / 100, 64 rows 137 / 104 / 102, 96 rows
// 191 / 113 / 104.  A tile narrower than its group reads the weights again, from L2; with a tail of groups above the average, columns
// for twice the average pay.
// One product: 16 rows or fewer in the smallest tile (1 row of 4096 x 7168 8.2 us, in the next 9.0); else by what the blocks of k of the
// busiest CTA cost, and the start and the end of a call.  64 / 128 / wide, measured: 128 x 4096 x 7168 17.0 / 12.9 / 16.9, 214 x 225 x
// 7912 9.7 / 11.1 / 15.3, 256 x 1536 x 7168 16.4 / 13.3 / 13.9, 512 x 512 x 2048 8.0 / 8.5 / 11.0, 512 x 1536 x 7168 24.6 / 19.7 / 16.7,
// 886 x 637 x 382 8.3 / 9.0 / 11.9, 1024 x 576 x 7168 24.8 / 19.7 / 16.7; the sums below are within 3 us of all of them.
enum GemmForm { kForm16, kForm64, kForm128, kFormWide };
GemmForm gemm_form(int rows, int n_groups, int n, int n_kb, int sm_count) {
  if (n_groups > 1) {
    const int per_group = (rows - 1) / n_groups + 1;
    return per_group <= 32 ? kForm64 : per_group <= 80 || n <= kScaleBlock ? kForm128 : kFormWide;
  }
  if (rows <= 16) return kForm16;
  auto cost = [&](int tok, int width, double split_ends, double ends, double block) {
    const long long tiles = ((rows - 1ll) / tok + 1) * ((n - 1ll) / width + 1);
    const int splits = k_splits(tiles, n_kb, sm_count);
    const long long rounds = (tiles * splits - 1) / sm_count + 1, blocks = (n_kb + splits - 1) / splits;
    return (splits > 1 ? split_ends : ends) + block * static_cast<double>(rounds * blocks);
  };
  const double c64 = cost(64, kScaleBlock, 6.8, 6.8, 0.36), c128 = cost(128, kScaleBlock, 7.0, 7.0, 0.43), wide = cost(kWideTok, kWideN, 11.0, 8.0, 0.42);
  return c64 <= c128 && c64 <= wide ? kForm64 : c128 <= wide ? kForm128 : kFormWide;
}

template <int kTok>
cudaError_t launch_fp8_gemm(moe_ctx *h, const GemmCall &c, cudaStream_t s, bool &maps_ok) {
  const int sm_count = h->sm_count;
  using S = GemmShape<kTok>;
  CUtensorMap ma, mb;
  maps_ok = encode_codes(&ma, c.a, c.k, c.ld_a, c.p.rows, 0, S::kBoxRows) && encode_codes(&mb, c.b, c.k, c.ld_b, c.p.n, c.p.n_groups, kScaleBlock);
  if (!maps_ok) return cudaSuccess;
  const cudaError_t e = allow_smem(h, reinterpret_cast<const void *>(fp8_gemm_kernel<kTok>), S::kSmem, kTok == 16 ? kSmemGemm16 : kTok == 64 ? kSmemGemm64 : kSmemGemm128);
  if (e != cudaSuccess) return e;
  // Most tiles that the call can have: a group of cnt rows has at most 1 + (cnt - 1) / kTok.
  const long long groups = std::min(c.p.n_groups, c.p.rows), n_nb = (c.p.n + kScaleBlock - 1) / kScaleBlock;
  const long long most = (groups + (c.p.rows - groups) / kTok) * n_nb;
  Fp8GemmArgs p = c.p;
  p.splits = k_splits(most, p.n_kb, sm_count);
  const dim3 grid(static_cast<unsigned>(p.splits > 1 ? most : std::min<long long>(most, sm_count)), p.splits, 1);
  return launch_kernel(fp8_gemm_kernel<kTok>, grid, S::kThreads, S::kSmem, s, true, p.splits > 1 ? p.splits : 0, ma, mb, p, out_alignment(p));
}

cudaError_t launch_fp8_gemm_wide(moe_ctx *h, const GemmCall &c, cudaStream_t s, bool &maps_ok) {
  const int sm_count = h->sm_count;
  CUtensorMap ma, mb;
  maps_ok = encode_codes(&ma, c.a, c.k, c.ld_a, c.p.rows, 0, 128) && encode_codes(&mb, c.b, c.k, c.ld_b, c.p.n, c.p.n_groups, kWideN);
  if (!maps_ok) return cudaSuccess;
  const long long groups = std::min(c.p.n_groups, c.p.rows), n_nb = (c.p.n + kWideN - 1) / kWideN;
  const long long most = (groups + (c.p.rows - groups) / kWideTok) * n_nb;
  Fp8GemmArgs p = c.p;
  p.splits = k_splits(most, p.n_kb, sm_count);
  const auto kernel = p.splits > 1 ? fp8_gemm_wide_kernel<true> : fp8_gemm_wide_kernel<false>;
  const cudaError_t e = allow_smem(h, reinterpret_cast<const void *>(kernel), kWideSmem, p.splits > 1 ? kSmemGemmWideSplit : kSmemGemmWide);
  if (e != cudaSuccess) return e;
  // outputs through the copy engine: rows 16-byte aligned
  CUtensorMap mo = ma;
  const int tiled = out_alignment(c.p) != 16 || !encode_out(&mo, c.p) ? kTiledNone
                    : static_cast<long long>(c.p.n) * dtype_size(c.p.out_dtype) % 16 == 0 ? kTiledAll : kTiledWhole;
  const dim3 grid(static_cast<unsigned>(p.splits > 1 ? most : std::min<long long>(most, sm_count)), p.splits, 1);
  return launch_kernel(kernel, grid, kWideThreads, kWideSmem, s, true, p.splits > 1 ? p.splits : 0, ma, mb, mo, p, tiled, out_alignment(p));
}

}  // namespace

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
  if (rows > kMostRows || n > kMostRows) return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: %d rows x %d columns in one call", rows, n);
  if (ld_a % 16 || ld_b % 16 || !aligned_to(a_dev, 16) || !aligned_to(b_dev, 16))
    return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: codes need 16-byte aligned rows (strides %lld, %lld)", ld_a, ld_b);
  if (rows == 0) return MOE_OK;
  if (!a_dev || !sa_dev || !b_dev || !sb_dev || !out_dev) return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: null tensor");
  if (!aligned_to(sa_dev, 4) || !aligned_to(sb_dev, 4) || !aligned_to(offsets_dev, 4) || !aligned_to(bias_dev, 2) || !aligned_to(out_dev, size))
    return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: a tensor is not aligned to its elements");
  if (int rc = use_device(c, "moe_gemm_fp8")) return rc;
  GemmCall call = {a_dev, b_dev, ld_a, ld_b, k, {}};
  Fp8GemmArgs &p = call.p;
  p.sa = sa_dev; p.sb = sb_dev; p.ld_sa = static_cast<size_t>(ld_sa);
  p.rows = rows; p.n = n; p.n_kb = static_cast<int>(n_kb); p.n_groups = n_groups; p.offsets = offsets_dev;
  p.bias = static_cast<const __nv_bfloat16 *>(bias_dev); p.out = out_dev; p.ld_out = static_cast<size_t>(ld_out);
  p.out_dtype = out_dtype; p.status = c->status;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const GemmForm form = gemm_form(rows, n_groups, n, p.n_kb, c->sm_count);
  bool maps_ok = true;
  const cudaError_t e = form == kForm16    ? launch_fp8_gemm<16>(c, call, s, maps_ok)
                        : form == kForm64  ? launch_fp8_gemm<64>(c, call, s, maps_ok)
                        : form == kForm128 ? launch_fp8_gemm<128>(c, call, s, maps_ok)
                                           : launch_fp8_gemm_wide(c, call, s, maps_ok);
  if (!maps_ok) return op_fail(c, MOE_ERR_INVALID, "moe_gemm_fp8: no tensor map for %d x %d and %d x %d x %d codes", rows, k, n_groups, n, k);
  return launched(c, "moe_gemm_fp8", e);
}

}  // extern "C"
