// Row movement around a layer of routed experts, as calls of their own: routing by scores (moe_route_scored), the
// permutation that sorts (token, expert) pairs by expert (moe_group_pairs), and the weighted sum of a token's expert rows
// (moe_combine_pairs).  The MXFP4 block has fixed forms of all three inside (route.cu); these take any router rule, any
// row types and strides, and pairs without an expert.
#include <type_traits>

#include "fp8_layer.cuh"
#include "sm100_ptx.cuh"

namespace moe {

// ---------------------------------------------------------------------------
// Routing.  Of a row's logits x:  s = sigmoid(x), or softmax over the experts that are on;  p = s + bias;  the groups
// with the highest sum of their group_top largest p stay;  the top_k largest p of what stays are selected, ties to the
// lower index;  weight = s [/ sum of the selected s] * scale.  An expert is off where x is -inf or NaN.  Where its bias is, it is
// not selected, but its x counts in the softmax: a bias does not change the scores.
//
// Which of two neighbouring p is larger is part of the answer, so the comparisons are those of 64 bits.  A row is tried in
// 32 bits first.  Without a bias the scores are in the order of the logits, and these are compared; only where 64 bits themselves
// no longer tell scores apart (a sigmoid above 16, logits within 1e-9) is the order not theirs.  With a bias a sigmoid in 32 bits
// is off by less than 2^-21 (s (1 - s) times the exponential's (2 + 1.2 |x|) 2^-23, and the roundings of sum and quotient), a
// softmax by less than 2^-18 of the row's largest (exponentials, a sum of up to 512, a quotient); so an order is certain where two
// values differ by 2^-20, or 2^-17 of that largest, and 2^-22 of their own magnitudes (sums of two by twice that, and by twice
// 2^-22 of their parts' magnitudes, which may have opposite signs), or where both logits and both biases are equal: then the index
// decides.  A row with a closer call is done again in 64 bits.  Of 8192 rows of 256 experts some 18 are: 10.4 us without them, 15.2
// with them, which is the time of one such row at the end (eight rounds on 64-bit keys 1.6 us, the exponentials 0.3; with the first
// rows sent through that code, to have it in the caches, 17.0).
// Settling only the calls in doubt, with one exponential a lane, took the same 15.2, and 0.6 us more on a single row.
//
// A warp per row; lane l owns the per_lane consecutive experts from l * per_lane, so that a lower lane is a lower index.
// ---------------------------------------------------------------------------
constexpr int kRouteWarps = 4;
constexpr int kMaxScoredExperts = 512, kMaxScoredTopK = 32, kMaxScoredGroups = 32;

// Unsigned integers in the order of the values; 0 is below every one of them and means "off".
__device__ __forceinline__ unsigned ordered_key(float p) {
  const unsigned b = __float_as_uint(p + 0.f);   // -0 and 0 are equal
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long ordered_key(double p) {
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(p + 0.0));
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ double key_value(unsigned long long k) {
  return __longlong_as_double(static_cast<long long>((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
}
// Largest key of the warp and the lanes that have it.
__device__ __forceinline__ unsigned warp_best(unsigned k, unsigned &owners) {
  const unsigned top = __reduce_max_sync(0xffffffffu, k);
  owners = __ballot_sync(0xffffffffu, k == top);
  return top;
}
__device__ __forceinline__ unsigned long long warp_best(unsigned long long k, unsigned &owners) {
  const unsigned hi = static_cast<unsigned>(k >> 32), lo = static_cast<unsigned>(k);
  const unsigned hi_top = __reduce_max_sync(0xffffffffu, hi);
  const unsigned lo_top = __reduce_max_sync(0xffffffffu, hi == hi_top ? lo : 0u);
  owners = __ballot_sync(0xffffffffu, hi == hi_top && lo == lo_top);
  return static_cast<unsigned long long>(hi_top) << 32 | lo_top;
}
template <class R>
__device__ __forceinline__ R warp_sum(R v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The two largest keys of a lane -> those of its group, in all of the group's lanes: `lanes` whole ones, a power of two.
template <class Key>
__device__ __forceinline__ void two_best(int lanes, Key &k1, Key &k2) {
  for (int off = 1; off < lanes; off <<= 1) {
    const Key o1 = __shfl_xor_sync(0xffffffffu, k1, off), o2 = __shfl_xor_sync(0xffffffffu, k2, off);
    k2 = max(max(k2, o2), min(k1, o1));
    k1 = max(k1, o1);
  }
}
// Lane g < n_groups holds what group g is worth: its rank, equal ones by the lower index.
template <class Key>
__device__ __forceinline__ int group_rank(Key worth, int n_groups, int lane) {
  int better = 0;
  for (int g = 0; g < n_groups; ++g) {
    const Key k = __shfl_sync(0xffffffffu, worth, g);
    better += k > worth || (k == worth && g < lane);
  }
  return lane < n_groups ? better : 32;
}
// One round of the selection: the largest key left in the warp, of the lowest lane that has it, and in that lane the lowest expert.
// Returns the key (0: nothing left); the owner's key is taken out.
template <class Key, int kPer>
__device__ __forceinline__ Key take_best(Key (&key)[kPer], Key &best, int lane, int &at, int &owner) {
  unsigned owners;
  const Key top = warp_best(best, owners);
  if (top == 0) return 0;
  owner = __ffs(owners) - 1;
  at = 0;
  if (lane == owner) {
    Key next = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool hit = !found && key[i] == top;
      if (hit) {
        at = i;
        key[i] = 0;
      }
      found = found || hit;
      next = max(next, key[i]);
    }
    best = next;
  }
  at = __shfl_sync(0xffffffffu, at, owner);
  return top;
}

// Largest first, by a network of fixed comparisons (odd-even merges).
template <int kPer>
__device__ __forceinline__ void sort_keys(unsigned (&key)[kPer]) {
#pragma unroll
  for (int p = 1; p < kPer; p *= 2)
#pragma unroll
    for (int d = p; d >= 1; d /= 2)
#pragma unroll
      for (int a = 0; a + d < kPer; ++a)
        if (a >= d % p && (a - d % p) % (2 * d) < d && a / (2 * p) == (a + d) / (2 * p)) {
          const unsigned low = min(key[a], key[a + d]);
          key[a] = max(key[a], key[a + d]);
          key[a + d] = low;
        }
}

// kDivide: a softmax that is not renormalised.  Its weights are divided by the row's sum, which is then one of whole exponentials in 64
// bits: with fast ones added in 32, weights were off by up to 9.5 x 2^-24 (512 experts), now by 3.3, and 8192 rows of 512 take 20.3 us
// in place of 19.1.  In the other kernels the sum only serves the selection.
//
// One row in 32 bits.  x[i]: the lane's logits, -inf where there is none; b[i]: its biases, -inf where there is no expert.  Lane
// k < top_k receives the k-th selected expert (or -1) in `sel`.  `top` and `sum`: of the softmax.  Returns false where 32 bits do
// not settle a comparison.  Groups are `group_lanes` whole lanes.
//
// The low bits of a key give way to the place in the lane (a lower place is a higher key), and a lane sorts its keys once: a round
// of the selection is then a maximum over the lanes' first keys and a shift in the lane that has it.  With unsorted keys, of
// which a round looked for its winner again, 8192 rows of 256 experts took 17.5 us instead of 15.2.
template <class T, int kPer, bool kDivide>
__device__ __forceinline__ bool select_fast(const T *src, const float (&x)[kPer], const float *bias, const float (&b)[kPer], const moe_route_rule &rule,
                                            int per_lane, int group_lanes, int lane, float top, float &sum, int &sel) {
  const float inf = __int_as_float(0x7f800000);
  constexpr unsigned kPlace = kPer - 1;       // bits of a place
  constexpr bool kExact = sizeof(T) == 2;     // logits whose keys lose nothing to the place
  const bool softmax = rule.score == MOE_SCORE_SOFTMAX;
  auto score = [&](float v) { return softmax ? __expf(v - top) : __fdividef(1.f, 1.f + __expf(-v)); };
  float over = 1.f;   // a softmax is score * over
  unsigned key[kPer];
  if (bias != nullptr || kDivide) {
    float s[kPer];
    if (softmax) {
      std::conditional_t<kDivide, double, float> all = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        s[i] = x[i] > -inf ? (kDivide ? expf(x[i] - top) : __expf(x[i] - top)) : 0.f;
        all += s[i];
      }
      sum = static_cast<float>(warp_sum(all));
      over = sum > 0.f ? __fdividef(1.f, sum) : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) s[i] = __fdividef(1.f, 1.f + __expf(-x[i]));
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) key[i] = bias != nullptr ? ordered_key(fmaf(s[i], over, b[i])) : ordered_key(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) key[i] = ordered_key(x[i]);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) key[i] = x[i] > -inf && b[i] > -inf ? (key[i] & ~kPlace) | (kPlace - i) : 0;   // (a finite value's key is above 2^22)
  sort_keys(key);
  // what a key stands for, off by less than `lost` of its magnitude (towards zero)
  auto value = [&](unsigned k) { return __uint_as_float(((k >> 31) ? k & 0x7fffffffu : ~k) & ~kPlace); };
  constexpr float lost = kPlace * 1.1920928955078125e-07f;                        // 2^-23 a place
  constexpr float rel = lost + 2.384185791015625e-07f;                            // and 2^-22
  const float close = softmax ? over * 7.62939453125e-06f : 9.5367431640625e-07f;   // 2^-17, 2^-20
  // the order of two keys (the first is not the smaller) is that of 64 bits
  auto certain = [&](unsigned ka, unsigned kc) {
    const float a = value(ka), c = value(kc);
    if (bias != nullptr) return a - c > close + rel * (fabsf(a) + fabsf(c));
    return (softmax ? a > top - 600.f : c < 16.f && a > -600.f) && a - c > 1e-9f + (kExact ? 0.f : lost * (fabsf(a) + fabsf(c)));
  };
  bool settled = true;
  if (rule.n_groups > 1) {
    unsigned k1 = key[0], k2 = kPer > 1 ? key[kPer > 1 ? 1 : 0] : 0;
    two_best(group_lanes, k1, k2);
    k1 = __shfl_sync(0xffffffffu, k1, lane * group_lanes & 31) & ~kPlace;   // lane g: those of group g
    k2 = __shfl_sync(0xffffffffu, k2, lane * group_lanes & 31) & ~kPlace;
    if (lane >= rule.n_groups) k1 = k2 = 0;
    unsigned worth = k1;
    float off = 0.f;   // how far a sum may be off for its parts' roundings and for what their logits lost
    const bool sums = rule.group_top == 2;
    if (sums && k1 != 0) {
      auto part = [&](unsigned k) {
        if (k == 0) return 0.f;
        const float v = value(k);
        float p = v;
        if (bias == nullptr) {
          const float d = lost * fabsf(v);
          p = score(v) * over;
          if (!kExact) off += d < 0.1f ? 1.1f * d * p : inf;
        }
        off += 2.f * rel * fabsf(p);
        return p;
      };
      worth = ordered_key(part(k1) + part(k2));
    }
    const int rank = group_rank(worth, rule.n_groups, lane);
    const unsigned stays = __ballot_sync(0xffffffffu, rank < rule.top_groups);
    if (rule.top_groups < rule.n_groups) {   // every group against the last that stays: above it, below it, or made of the same
      const int in = __ffs(__ballot_sync(0xffffffffu, rank == rule.top_groups - 1)) - 1;
      const unsigned a1 = __shfl_sync(0xffffffffu, k1, in), a2 = __shfl_sync(0xffffffffu, k2, in), wa = __shfl_sync(0xffffffffu, worth, in);
      const float off_in = __shfl_sync(0xffffffffu, off, in);
      if (worth != 0 && wa != 0) {
        const unsigned hi = max(worth, wa), lo = min(worth, wa);
        const bool same = lane == in || (kExact && bias == nullptr && k1 == a1 && (!sums || k2 == a2));
        settled = same || (sums ? key_value(hi) - key_value(lo) > 2.f * close + (off + off_in) : certain(hi, lo));
      }
    }
    if (!(stays >> (lane / group_lanes) & 1u)) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) key[i] = 0;
    }
  }
  // lane k keeps the k-th; the lowest lane wins among equal ones
  unsigned kept = 0;
  int from = 0;
  for (int k = 0; k < rule.top_k; ++k) {
    const unsigned best = __reduce_max_sync(0xffffffffu, key[0]);
    if (best == 0) break;
    const int owner = __ffs(__ballot_sync(0xffffffffu, (key[0] ^ best) <= kPlace)) - 1;
    const unsigned won = __shfl_sync(0xffffffffu, key[0], owner);
    if (lane == k) { kept = won; from = owner; }
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i + 1 < kPer; ++i) key[i] = key[i + 1];
      key[kPer - 1] = 0;
    }
  }
  sel = kept != 0 ? from * per_lane + static_cast<int>(kPlace - (kept & kPlace)) : -1;
  // neighbours among the selected, and the last of them against all that is left.  Equal logits under equal biases: the index decided
  auto same = [&](int e, int f) { return to_f32(src[e]) == to_f32(src[f]) && (bias == nullptr || bias[e] == bias[f]); };
  const unsigned after = __shfl_down_sync(0xffffffffu, kept, 1), last = __shfl_sync(0xffffffffu, kept, rule.top_k - 1);
  const int after_sel = __shfl_down_sync(0xffffffffu, sel, 1), last_sel = __shfl_sync(0xffffffffu, sel, rule.top_k - 1);
  if (lane + 1 < rule.top_k && after != 0 && !certain(kept, after) && !same(sel, after_sel)) settled = false;
  if (key[0] != 0 && !certain(last, key[0])) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (key[i] != 0 && !certain(last, key[i]) && !same(last_sel, lane * per_lane + static_cast<int>(kPlace - (key[i] & kPlace)))) settled = false;
  }
  return __all_sync(0xffffffffu, settled);
}

// One row in 64 bits; sel_s: the score of the selected.  With group_lanes = 0 groups are any runs of experts, through `shared`.
template <int kPer>
__device__ __forceinline__ void select_exact(const float (&x)[kPer], const float (&b)[kPer], const moe_route_rule &rule, int per_lane, int group_lanes,
                                             unsigned long long *shared, int lane, float top, int &sel, double &sel_s) {
  using Key = unsigned long long;
  const float inf = __int_as_float(0x7f800000);
  const int first = lane * per_lane;
  double s[kPer];
  Key key[kPer];
  if (rule.score == MOE_SCORE_SOFTMAX) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      s[i] = x[i] > -inf ? exp(static_cast<double>(x[i]) - static_cast<double>(top)) : 0.0;
      sum += s[i];
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (sum > 0.0) s[i] /= sum;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) s[i] = 1.0 / (1.0 + exp(-static_cast<double>(x[i])));
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    key[i] = ordered_key(s[i] + static_cast<double>(b[i]));
    if (!(x[i] > -inf) || !(b[i] > -inf)) key[i] = 0;
  }
  if (rule.n_groups > 1) {
    const int size = rule.n_experts / rule.n_groups;
    Key k1 = 0, k2 = 0;
    if (group_lanes > 0) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        k2 = max(k2, min(k1, key[i]));
        k1 = max(k1, key[i]);
      }
      two_best(group_lanes, k1, k2);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i < per_lane && first + i < rule.n_experts) shared[first + i] = key[i];
      __syncwarp();
      if (lane < rule.n_groups)
        for (int j = 0; j < size; ++j) {
          const Key k = shared[lane * size + j];
          k2 = max(k2, min(k1, k));
          k1 = max(k1, k);
        }
    }
    Key worth = k1;
    if (rule.group_top == 2 && k2) worth = ordered_key(key_value(k1) + key_value(k2));
    if (group_lanes > 0) worth = __shfl_sync(0xffffffffu, worth, lane * group_lanes & 31);
    if (lane >= rule.n_groups) worth = 0;
    const unsigned stays = __ballot_sync(0xffffffffu, group_rank(worth, rule.n_groups, lane) < rule.top_groups);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < per_lane && first + i < rule.n_experts && !(stays >> ((first + i) / size) & 1u)) key[i] = 0;
  }
  sel = -1;
  sel_s = 0.0;
  Key best = key[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) best = max(best, key[i]);
  for (int k = 0; k < rule.top_k; ++k) {
    int at, owner;
    if (take_best(key, best, lane, at, owner) == 0) break;
    double mine = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i == at) mine = s[i];
    mine = __shfl_sync(0xffffffffu, mine, owner);
    if (lane == k) {
      sel = owner * per_lane + at;
      sel_s = mine;
    }
  }
}

template <class T, int kPer, bool kDivide>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_scored_kernel(const T *logits, size_t ld, const float *bias, int rows, moe_route_rule rule, int per_lane, int group_lanes, int vec, int vec_bias,
                    int *idx, float *w) {
  __shared__ unsigned long long s_keys[kRouteWarps][kPer * 32];   // groups that are not whole lanes
  grid_dep_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t row = static_cast<size_t>(blockIdx.x) * kRouteWarps + warp;
  if (row >= static_cast<size_t>(rows)) return;
  const int E = rule.n_experts, first = lane * per_lane;
  const float inf = __int_as_float(0x7f800000);
  float x[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = -inf;
  const T *src = logits + row * ld;
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  if (kPer >= kVec && vec) {   // per_lane is a multiple of kVec, rows are 16-byte aligned
#pragma unroll
    for (int i = 0; i + kVec <= kPer; i += kVec)
      if (i < per_lane && first + i < E) {
        const uint4 v = *reinterpret_cast<const uint4 *>(src + first + i);
        const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[i + j] = to_f32(e[j]);
      }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < per_lane && first + i < E) x[i] = to_f32(src[first + i]);
  }
  float b[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) b[i] = i < per_lane && first + i < E ? 0.f : -inf;
  if (bias != nullptr) {
    if (kPer >= 4 && vec_bias) {
#pragma unroll
      for (int i = 0; i + 4 <= kPer; i += 4)
        if (i < per_lane && first + i < E) {
          const float4 v = *reinterpret_cast<const float4 *>(bias + first + i);
          b[i] = v.x; b[i + 1] = v.y; b[i + 2] = v.z; b[i + 3] = v.w;
        }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i < per_lane && first + i < E) b[i] = bias[first + i];
    }
  }
  if (bias != nullptr) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (b[i] > 3.402823466e38f) b[i] = 3.402823466e38f;   // +inf counts as the largest finite value (a NaN stays)
  }
  float top = -inf;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (x[i] > 3.402823466e38f) x[i] = 3.402823466e38f;
    if (x[i] != x[i]) x[i] = -inf;                         // NaN is off
    top = fmaxf(top, x[i]);
  }
  if (rule.score == MOE_SCORE_SOFTMAX) {
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (!(top > -inf)) top = 0.f;
  }
  int sel;
  double share = 0.0;
  float sum = 0.f;
  if ((rule.n_groups == 1 || group_lanes > 0) && select_fast<T, kPer, kDivide>(src, x, bias, b, rule, per_lane, group_lanes, lane, top, sum, sel)) {
    // weights of the selected from their logits, within a few roundings of 32 bits
    float s = 0.f, v = 0.f;
    if (sel >= 0) {
      v = to_f32(src[sel]);
      if (v > 3.402823466e38f) v = 3.402823466e38f;
      if (rule.score == MOE_SCORE_SOFTMAX) {
        const float d = v - top, r = d - v, lost = (v - (d - r)) - (top + r);   // v - top is d + lost exactly
        s = expf(d);
        if (fabsf(lost) < 1.f) s = fmaf(s, lost, s);
      } else {
        s = __fdiv_rn(1.f, 1.f + expf(-v));
      }
    }
    if (__all_sync(0xffffffffu, sel < 0 || s >= 7.888609052210118e-31f)) {   // 2^-100
      if (rule.renormalise) {
        const float all = warp_sum(s);
        share = all > 0.f ? __fdiv_rn(s, all) : 0.f;
      } else {
        share = rule.score != MOE_SCORE_SOFTMAX ? s : sum > 0.f ? __fdiv_rn(s, sum) : 0.f;
      }
    } else {
      // Scores next to the smallest normal number of 32 bits (a sigmoid below -69, a softmax whose bias selects as far below the
      // largest logit) lose their places, or are all 0 where their quotients are not: 64 bits
      if (sel >= 0) share = rule.score == MOE_SCORE_SOFTMAX ? exp(static_cast<double>(v) - static_cast<double>(top)) : 1.0 / (1.0 + exp(-static_cast<double>(v)));
      const double all = rule.renormalise ? warp_sum(share) : rule.score == MOE_SCORE_SOFTMAX ? static_cast<double>(sum) : 1.0;
      share = all > 0.0 ? share / all : 0.0;
    }
  } else {
    double s;
    select_exact(x, b, rule, per_lane, group_lanes, s_keys[warp], lane, top, sel, s);
    share = s;
    if (rule.renormalise) {
      const double all = warp_sum(s);
      share = all > 0.0 ? s / all : 0.0;
    }
  }
  if (lane < rule.top_k) {
    idx[row * rule.top_k + lane] = sel;
    w[row * rule.top_k + lane] = static_cast<float>(share * static_cast<double>(rule.scale));
  }
}

template <class T>
cudaError_t launch_route_scored(const moe_route_rule &r, const void *logits, size_t ld, const float *bias, int rows, int *idx, float *w,
                                cudaStream_t s) {
  // Experts of a lane: enough for all in 32 lanes; with groups, up to 16 such that a group is a power of two of whole lanes.
  int per = (r.n_experts + 31) / 32, group_lanes = 0;
  if (r.n_groups > 1) {
    const int size = r.n_experts / r.n_groups;
    for (int p = per; p <= 16 && group_lanes == 0; ++p)
      if (size % p == 0 && ((size / p) & (size / p - 1)) == 0) { per = p; group_lanes = size / p; }
  }
  const unsigned grid = static_cast<unsigned>((static_cast<size_t>(rows) + kRouteWarps - 1) / kRouteWarps);
  const T *x = static_cast<const T *>(logits);
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  const int vec = per % kVec == 0 && r.n_experts % kVec == 0 && ld % kVec == 0 && aligned_to(x, 16);
  const int vec_bias = per % 4 == 0 && r.n_experts % 4 == 0 && aligned_to(bias, 16);
  auto go = [&](auto kernel) {
    return launch_kernel(kernel, dim3(grid), kRouteWarps * 32, 0, s, true, 0, x, ld, bias, rows, r, per, group_lanes, vec, vec_bias, idx, w);
  };
  auto by_experts = [&](auto divide) {
    constexpr bool kDivide = decltype(divide)::value;
    if (per <= 1) return go(route_scored_kernel<T, 1, kDivide>);
    if (per <= 2) return go(route_scored_kernel<T, 2, kDivide>);
    if (per <= 4) return go(route_scored_kernel<T, 4, kDivide>);
    if (per <= 8) return go(route_scored_kernel<T, 8, kDivide>);
    return go(route_scored_kernel<T, 16, kDivide>);
  };
  return r.score == MOE_SCORE_SOFTMAX && !r.renormalise ? by_experts(std::true_type()) : by_experts(std::false_type());
}

// ---------------------------------------------------------------------------
// Stable counting sort of the pairs (token * top_k + slot) by expert, in one launch of one cluster: the CTAs own contiguous
// ranges of pairs and their warps contiguous parts of them, each with a histogram of its own.  Every CTA reads the others'
// totals from their shared memory; prefixes over experts, CTAs and warps then give every warp its place in every expert's rows,
// and a second walk over the same pairs hands the places out, so that they ascend with the pair.  Latency is all there is to
// it: 8192 x 8 pairs of 256 experts 80 us on one CTA, 10.7 on eight (launch and cluster 3, pairs and histograms 2, prefixes and the
// other CTAs' totals 3, places 2).
// ---------------------------------------------------------------------------
constexpr int kGroupThreads = 1024, kGroupWarps = kGroupThreads / 32, kGroupMaxCtas = 8;
constexpr int kMaxGroupedExperts = 1024;

__global__ void __launch_bounds__(kGroupThreads)
group_pairs_kernel(const int *idx, size_t n_pairs, int E, int *offsets, int *pair_row, int *row_pair) {
  extern __shared__ int s_hist[];   // [kGroupWarps][E], then the totals of this CTA [E]
  __shared__ int s_scan[kGroupWarps], s_all, s_start[kMaxGroupedExperts];   // s_start: first row of this CTA's pairs of an expert
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = gridDim.y, rank = blockIdx.y;   // the cluster is the grid
  int *mine = s_hist + warp * E, *totals = s_hist + kGroupWarps * E;
  for (int i = threadIdx.x; i < kGroupWarps * E; i += kGroupThreads) s_hist[i] = 0;
  __syncthreads();
  grid_dep_sync();
  const size_t per = (n_pairs + static_cast<size_t>(ctas) * kGroupThreads - 1) / (static_cast<size_t>(ctas) * kGroupThreads) * 32;
  const size_t begin = min(per * (rank * kGroupWarps + warp), n_pairs), end = min(begin + per, n_pairs);
  // the first eight steps of a warp stay in registers for the second walk
  constexpr int kKept = 8;
  int kept[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    const size_t p = begin + 32 * i + lane;
    kept[i] = p < end ? idx[p] : -1;
    if (kept[i] >= E) kept[i] = -1;
  }
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (kept[i] >= 0) atomicAdd(&mine[kept[i]], 1);
  for (size_t p = begin + 32 * kKept + lane; p < end; p += 32) {
    const int e = idx[p];
    if (e >= 0 && e < E) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  // thread e: exclusive prefix over the warps of this CTA, then over the CTAs and the experts
  int total = 0;
  if (threadIdx.x < E) {
    int n[kGroupWarps];
#pragma unroll
    for (int v = 0; v < kGroupWarps; ++v) n[v] = s_hist[v * E + threadIdx.x];
#pragma unroll
    for (int v = 0; v < kGroupWarps; ++v) {
      s_hist[v * E + threadIdx.x] = total;
      total += n[v];
    }
    totals[threadIdx.x] = total;
  }
  int before = 0, all = total;
  if (ctas > 1) {
    sm100::cluster_sync_all();
    all = 0;
    if (threadIdx.x < E)
#pragma unroll
      for (int r = 0; r < kGroupMaxCtas; ++r)
        if (r < ctas) {
          const int n = static_cast<int>(sm100::ld_cluster_u32(sm100::map_to_cta(sm100::smem_u32(&totals[threadIdx.x]), r)));
          all += n;
          if (r < rank) before += n;
        }
  }
  int incl = all;
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
    if (lane == 31) s_all = t;
  }
  __syncthreads();
  const int start = s_scan[warp] + incl - all;
  if (threadIdx.x < E) {
    if (rank == 0) offsets[threadIdx.x] = start;
    s_start[threadIdx.x] = start + before;
  }
  if (rank == 0 && threadIdx.x == 0) offsets[E] = s_all;
  __syncthreads();
  // lanes with the same expert, from a ballot for each bit of its number (__match_any_sync takes ~60 cycles for every distinct
  // number of the warp: 2000 a step with 256 experts, 14 of the 22 us that the call took)
  const int bits = 32 - __clz(E);
  auto place = [&](size_t p, int e) {
    unsigned same = __ballot_sync(0xffffffffu, e >= 0);
    for (int i = 0; i < bits; ++i) {
      const unsigned set = __ballot_sync(0xffffffffu, e >> i & 1);
      same &= (e >> i & 1) ? set : ~set;
    }
    const int rank_here = __popc(same & ((1u << lane) - 1u));
    int row = -1;
    if (e >= 0) row = s_start[e] + mine[e] + rank_here;
    __syncwarp();
    if (e >= 0 && rank_here == 0) mine[e] += __popc(same);   // one lane of each expert
    __syncwarp();
    if (p < end) pair_row[p] = row;
    if (row >= 0 && row_pair != nullptr) row_pair[row] = static_cast<int>(p);
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (begin + 32 * i < end) place(begin + 32 * i + lane, kept[i]);
  for (size_t p0 = begin + 32 * kKept; p0 < end; p0 += 32) {
    const size_t p = p0 + lane;
    int e = p < end ? idx[p] : -1;
    if (e < 0 || e >= E) e = -1;
    place(p, e);
  }
  if (row_pair != nullptr)
    for (size_t r = static_cast<size_t>(s_all) + rank * kGroupThreads + threadIdx.x; r < n_pairs; r += static_cast<size_t>(ctas) * kGroupThreads)
      row_pair[r] = -1;
  if (ctas > 1) sm100::cluster_sync_all();   // no CTA leaves while another may still read its totals
}

// ---------------------------------------------------------------------------
// out[t] = residual[t] + sum over k of w[t, k] * y[pair_row[t, k]], added in the order of k in fp32 and rounded once.
// A pair whose row is negative or not below n_y_rows adds nothing, whatever its weight.
// ---------------------------------------------------------------------------
// Bound by HBM.  A CTA per row (per part of one where there are few rows); a thread has eight neighbouring columns a step.  With
// every row 16-byte aligned (vec) they are one or two wide loads, and the loads of four pairs are requested together and a step
// ahead of their use.  8192 rows of 2880 bf16 columns, four pairs each, us: a CTA per 1024 columns 61 (the loads of an index and
// of the row behind it are then most of a CTA's life), per row, a step ahead 40.
constexpr int kCombineThreads = 128, kCombineCols = 8;

template <class T>
struct Raw8 {   // eight values as they lie in memory
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = reinterpret_cast<const uint4 *>(p)[i];
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f32(reinterpret_cast<const T *>(v)[i]); }
};
template <class T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  uint4 raw[sizeof(T) / 2];
  T *e = reinterpret_cast<T *>(raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) store_as(e + i, v[i]);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = raw[i];
}

template <class TY, class TO>
__global__ void __launch_bounds__(kCombineThreads)
combine_pairs_kernel(const TY *y, size_t ld_y, int n_y_rows, const int *pair_row, const float *w, int top_k, int cols, const TO *residual,
                     size_t ld_residual, TO *out, size_t ld_out, int vec) {
  grid_dep_sync();
  const size_t t = blockIdx.x;
  const int *rows = pair_row + t * top_k;
  const float *weights = w + t * top_k;
  const int first = (blockIdx.y * blockDim.x + threadIdx.x) * kCombineCols, step = gridDim.y * blockDim.x * kCombineCols;
  const int whole = vec ? cols / kCombineCols * kCombineCols : 0;   // columns that are read and written in vectors
  constexpr int kAhead = 4;
  // the first four pairs: their rows' vectors of the next step are on their way while those of this step are added
  const TY *src[kAhead];
  float f[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int r = k < top_k ? rows[k] : -1;
    const bool on = r >= 0 && r < n_y_rows;
    src[k] = on ? y + static_cast<size_t>(r) * ld_y : nullptr;
    f[k] = on ? weights[k] : 0.f;
  }
  Raw8<TY> v[kAhead];
  Raw8<TO> res;
  auto fetch = [&](int c0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (src[k] != nullptr) v[k].load(src[k] + c0);
    if (residual != nullptr) res.load(residual + t * ld_residual + c0);
  };
  int c0 = first;
  if (c0 < whole) fetch(c0);
  for (; c0 < whole; c0 += step) {
    float sum[8] = {}, plus[8] = {};
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (src[k] != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = fmaf(f[k], v[k][i], sum[i]);
      }
    if (residual != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) plus[i] = res[i];
    }
    if (c0 + step < whole) fetch(c0 + step);
    for (int k = kAhead; k < top_k; ++k) {
      const int r = rows[k];
      if (r < 0 || r >= n_y_rows) continue;
      Raw8<TY> u;
      u.load(y + static_cast<size_t>(r) * ld_y + c0);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = fmaf(weights[k], u[i], sum[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += plus[i];
    store8(out + t * ld_out + c0, sum);
  }
  for (; c0 < cols; c0 += step) {
    float sum[8] = {};
    for (int k = 0; k < top_k; ++k) {
      const int r = rows[k];
      if (r < 0 || r >= n_y_rows) continue;
      const TY *from = y + static_cast<size_t>(r) * ld_y + c0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < cols) sum[i] = fmaf(weights[k], to_f32(from[i]), sum[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < cols) store_as(out + t * ld_out + c0 + i, residual != nullptr ? sum[i] + to_f32(residual[t * ld_residual + c0 + i]) : sum[i]);
  }
}

template <class TY, class TO>
cudaError_t launch_combine_pairs(const void *y, size_t ld_y, int n_y_rows, const int *pair_row, const float *w, int rows, int top_k, int cols,
                                 const void *residual, size_t ld_residual, void *out, size_t ld_out, cudaStream_t s) {
  const int vec = aligned_to(y, 16) && aligned_to(residual, 16) && aligned_to(out, 16) && ld_y * sizeof(TY) % 16 == 0 &&
                  ld_residual * sizeof(TO) % 16 == 0 && ld_out * sizeof(TO) % 16 == 0;
  const int vectors = (cols + kCombineCols - 1) / kCombineCols;
  const int parts = rows >= 1024 ? 1 : (vectors + kCombineThreads - 1) / kCombineThreads;
  const int steps = (vectors + kCombineThreads * parts - 1) / (kCombineThreads * parts);
  const int threads = ((vectors + steps * parts - 1) / (steps * parts) + 31) / 32 * 32;
  const dim3 grid(rows, parts, 1);
  return launch_kernel(combine_pairs_kernel<TY, TO>, grid, threads, 0, s, true, 0, static_cast<const TY *>(y), ld_y, n_y_rows, pair_row, w,
                       top_k, cols, static_cast<const TO *>(residual), ld_residual, static_cast<TO *>(out), ld_out, vec);
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
  const size_t smem = static_cast<size_t>(kGroupWarps + 1) * n_experts * sizeof(int), n_pairs = static_cast<size_t>(rows) * top_k;
  int ctas = 1;   // one step of 32 pairs for every warp, then more steps
  while (ctas < kGroupMaxCtas && n_pairs > static_cast<size_t>(ctas) * kGroupThreads) ctas *= 2;
  cudaError_t e = allow_smem(c, reinterpret_cast<const void *>(group_pairs_kernel), (kGroupWarps + 1) * kMaxGroupedExperts * 4, kSmemGroup);
  if (e == cudaSuccess)
    e = launch_kernel(group_pairs_kernel, dim3(1, ctas, 1), kGroupThreads, smem, static_cast<cudaStream_t>(stream), true, ctas > 1 ? ctas : 0, idx_dev,
                      n_pairs, n_experts, offsets_dev, pair_row_dev, row_pair_dev);
  return launched(c, "moe_group_pairs", e);
}

int moe_combine_pairs(moe_handle c, const void *y_dev, int y_dtype, long long ld_y, int n_y_rows, const int *pair_row_dev, const float *w_dev,
                      int rows, int top_k, int cols, const void *residual_dev, long long ld_residual, void *out_dev, int out_dtype,
                      long long ld_out, void *stream) {
  if (!c) return MOE_ERR_INVALID;
  const int ys = dtype_size(y_dtype), os = dtype_size(out_dtype);
  if (!ys || !os || rows < 0 || top_k < 1 || cols < 1 || n_y_rows < 0 || cols > 65535 * kCombineThreads * kCombineCols || ld_y < cols || ld_out < cols || (residual_dev && ld_residual < cols) ||
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
