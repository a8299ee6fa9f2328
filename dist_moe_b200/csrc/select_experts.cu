// Expert ids and scores of every token from the router's logits, forward and backward.
//
//   p = softmax(l) over the experts, or sigmoid(l);   c = p + b (b: optional bias, for the choice alone)
//   with groups: a group's value is the sum of its one or two largest c, and the experts of the `kept` best groups remain
//   ids = the K largest c in falling order, equal values by index;   v_k = p[ids_k]
//   score_k = scale * v_k, or scale * v_k / sum_j v_j
// An expert whose logit or c is -inf or NaN is not chosen (a NaN logit counts as -inf); where fewer than K are left, and for masked
// tokens, ids are -1 and scores 0, which is how the routed experts take a route that goes nowhere.  +inf logits share the softmax.
//
// The choice is the one of 64-bit arithmetic.  Without a bias p is monotone in l, so experts are compared by their logits.  Otherwise c
// in 32 bits carries an error of a few units in the last place; where two values that decide something lie nearer than that, which is so
// in under one row in a hundred of normally distributed logits, the experts in question, or for groups the whole row, are compared once
// more in 64 bits.
//
// Backward, w_k = v_k / sum v, g_k = scale * grad_k:
//   softmax            dl_i = p_i (g_i [i chosen] - sum_k p_k g_k)
//   sigmoid            dl_k = g_k p_k (1 - p_k)
//   softmax, normalised  dl_k = w_k (g_k - sum_j w_j g_j);   sigmoid, normalised: the same times 1 - p_k
//
// A warp per token: its logits sit in registers, expert 32 j + lane in register j.  Each of the K rounds is two warp reductions over the
// lanes' largest remaining values; a lane keeps its two largest, and looks through its registers again where a third is asked for.
//
// Instruction bound: the logits are read once (4096 x 256 in 0.6 us at the copy rate).  Measured, events included (some 6 us), K = 8:
// 4096 x 256 12 us from the logits alone, 14 with a bias, 18 with 4 of 8 groups too, 16384 x 256 27 and 46; backward 8 to 10 and 18.
// The backward is bound by instructions too, at one element a load and store: the softmax walks over a row three times and takes each
// exponential twice (65536 x 256 52 us, 20 at the copy rate), the other forms fill with zeros and write K values (25 us, 10).
#include <type_traits>

#include "common.cuh"
#include "../../include/dist_moe_b200.h"

namespace dm {

constexpr int kSelectWarps = 4;

struct SelectParams {
  const void* logits;
  int64_t stride;  // elements between rows
  int64_t T;
  int E, K, groups, kept, group_top;
  int sigmoid, renormalize;
  float scale;
  const float* bias;            // null: none
  const unsigned char* mask;    // null: every token is live
  void* ids;
  void* scores;
  int ids_are_int64, scores_are_bf16;
};

__device__ __forceinline__ float select_load(const float* p) { return *p; }
__device__ __forceinline__ float select_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void select_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void select_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Floats as unsigned words of the same order; 0 for what cannot be chosen.  Adding zero makes -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > neg_inf())) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ (static_cast<int32_t>(b) < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k ^ (static_cast<int32_t>(k) < 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t order_key(double v) {
  if (!(v > static_cast<double>(neg_inf()))) return 0;
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return b ^ (static_cast<int64_t>(b) < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, k, d);
    k = o > k ? o : k;
  }
  return k;
}

// What the softmax's exponential is taken of: +inf logits, which are the largest then, share it.
template <typename V>
__device__ __forceinline__ V below(float l, float top) {
  return l == top ? V(0) : V(l) - V(top);
}

// The two largest values seen, falling.
template <typename V>
struct Top2 {
  V first, second;  // -inf: nothing
  __device__ __forceinline__ void add(V v) {
    if (v > first) {
      second = first;
      first = v;
    } else if (v > second) {
      second = v;
    }
  }
};

// The choice in V arithmetic.  `values` (shared memory of this warp, E of them) are compared between groups, `keys`, in registers, between
// experts; whether two values are nearer than `tolerance` allows is looked at between groups and between experts where the `near_...` are
// set.  The chosen index of round k ends up in lane k; between experts that are near one another there are more rounds than K, up to
// the first one that stands clear of those before it.
struct Found {
  bool near_groups, near_experts;
  int rounds;  // experts found, 32 at the most
};
template <int kPer, typename Key, typename V>
__device__ __forceinline__ Found choose(Key (&keys)[kPer], const V* values, V tolerance, bool near_groups, bool near_experts,
                                        const SelectParams& p, int lane, int& chosen) {
  Found found{false, false, 0};
  const V nothing = static_cast<V>(neg_inf());
  if (p.groups > 1) {
    const int size = p.E / p.groups;
    int shift = 5;  // 2^shift lanes look through a group
    while ((32 >> shift) < p.groups) --shift;
    const int lanes_per = 1 << shift, group = lane >> shift, sub = lane & (lanes_per - 1);
    Top2<V> best{nothing, nothing};
    if (group < p.groups) {
      const int rounds = (size + lanes_per - 1) >> shift;
      int k = group % rounds;  // groups start at different members: their banks differ
      for (int i = 0; i < rounds; ++i) {
        const int member = sub + (k << shift);
        if (member < size) best.add(values[group * size + member]);
        k = k + 1 == rounds ? 0 : k + 1;
      }
    }
    for (int d = 1; d < lanes_per; d <<= 1) {
      const V a = __shfl_xor_sync(0xffffffffu, best.first, d), b = __shfl_xor_sync(0xffffffffu, best.second, d);
      best.add(a);
      best.add(b);
    }
    const bool two = p.group_top == 2 && best.second > nothing;
    const V value = two ? best.first + best.second : best.first;
    int rank = 0;  // groups of larger value, or of equal value and lower index
    for (int g = 0; g < p.groups; ++g) {
      const V other = __shfl_sync(0xffffffffu, value, g << shift);
      if (other > value || (other == value && g < group)) ++rank;
    }
    const bool keep = group < p.groups && rank < p.kept;
    if (near_groups && p.kept < p.groups) {
      // the smallest kept value, the largest other one, and the largest size of what was added
      V above = keep ? value : static_cast<V>(-neg_inf()), under = keep || group >= p.groups ? nothing : value;
      V span = group < p.groups && best.first > nothing ? fabs(best.first) + (two ? fabs(best.second) : V(0)) : V(0);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        const V a = __shfl_xor_sync(0xffffffffu, above, d), u = __shfl_xor_sync(0xffffffffu, under, d), w = __shfl_xor_sync(0xffffffffu, span, d);
        above = a < above ? a : above;
        under = u > under ? u : under;
        span = w > span ? w : span;
      }
      // sums of two values each: two errors on either side.  Written so that infinities on both sides count as near.
      found.near_groups = under > nothing && !(above - under > 4 * (tolerance + static_cast<V>(0x1p-23f) * span));
    }
    const uint32_t kept_lanes = __ballot_sync(0xffffffffu, keep && sub == 0);
    const uint32_t per_group = ((1u << 20) + size - 1) / size;  // e / size, exactly for e < 1024
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = 32 * j + lane;
      if (e < p.E && !(kept_lanes >> ((e * per_group >> 20) << shift) & 1)) keys[j] = 0;
    }
  }
  Key mine = 0, next = 0;  // the lane's largest remaining key and the one after it
  int at = 0, at_next = 0;
  uint32_t gone = 0;       // registers already chosen
  bool stale = false;      // `next` is not known
  auto scan = [&] {
    mine = next = 0;
    at = at_next = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const Key k = gone >> j & 1 ? 0 : keys[j];
      if (k > mine) {
        next = mine;
        at_next = at;
        mine = k;
        at = j;
      } else if (k > next) {
        next = k;
        at_next = j;
      }
    }
    stale = false;
  };
  scan();
  chosen = -1;
  Key last = 0;
  auto near_last = [&](Key key) {
    const float a = key_value(static_cast<uint32_t>(last)), b = key_value(static_cast<uint32_t>(key));
    return !(a - b > 2.0f * (static_cast<float>(tolerance) + 0x1p-23f * fabsf(a)));
  };
  for (int k = 0; k < 32; ++k) {
    if (k >= p.K && !near_experts) break;
    const Key top = warp_max_key(mine);
    if (top == 0) break;
    const int e = static_cast<int>(__reduce_min_sync(0xffffffffu, mine == top ? static_cast<uint32_t>(32 * at + lane) : 0xffffffffu));
    if (near_experts && k > 0 && sizeof(Key) == 4) {
      const bool near = near_last(top);
      if (k >= p.K && !near) break;
      found.near_experts = found.near_experts || near;
    }
    found.rounds = k + 1;
    last = top;
    if (lane == k) chosen = e;
    const bool won = lane == (e & 31);
    if (won) gone |= 1u << at;
    if (__any_sync(0xffffffffu, won && stale)) {
      if (won) scan();
    } else if (won) {
      mine = next;
      at = at_next;
      next = 0;
      stale = kPer > 2;
    }
  }
  if (near_experts && found.rounds == 32) {  // and what would come after them
    const Key top = warp_max_key(mine);
    found.near_experts = found.near_experts || (top != 0 && near_last(top));
  }
  return found;
}

// The sum of the softmax, in 64 bits.
template <int kPer, typename L>
__device__ __noinline__ double sum_again(const SelectParams& p, const L* row, float top, int lane) {
  double z = 0.0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = 32 * j + lane;
    const float l = e < p.E ? select_load(row + e) : neg_inf();
    const bool in = l > neg_inf();
    const double x = exp(in ? below<double>(l, top) : 0.0);
    z += in ? x : 0.0;
  }
  return warp_sum(z);
}

// The order of the experts found, lane k the k-th, by their values in 64 bits: any expert that is not among them is clear of the K best.
template <typename L>
__device__ __noinline__ int order_again(const SelectParams& p, const L* row, float top, double z, int found, int expert, int lane) {
  uint64_t key = 0;
  if (lane < found) {
    const float l = select_load(row + expert);
    const double x = exp(p.sigmoid ? -static_cast<double>(l) : below<double>(l, top));
    key = order_key((p.sigmoid ? 1.0 / (1.0 + x) : x / z) + static_cast<double>(p.bias[expert]));
  }
  int rank = 0;
  for (int i = 0; i < found; ++i) {
    const uint64_t other = __shfl_sync(0xffffffffu, key, i);
    const int e = __shfl_sync(0xffffffffu, expert, i);
    if (other > key || (other == key && e < expert)) ++rank;
  }
  int chosen = -1;
  for (int k = 0; k < p.K && k < found; ++k) {
    const uint32_t who = __ballot_sync(0xffffffffu, lane < found && rank == k);
    const int e = __shfl_sync(0xffffffffu, expert, __ffs(static_cast<int>(who)) - 1);
    if (lane == k) chosen = e;
  }
  return chosen;
}

// The row in 64 bits: its values go through `values64`, shared memory of this warp (E doubles).  No branch among a lane's values: their
// exponentials run side by side.  (One after another they took such a row 10 us, twice the time of all others: 4096 tokens of 256 experts
// with a bias 20 us, without one 10.)
template <int kPer, typename L>
__device__ __noinline__ int choose_again(const SelectParams& p, const L* row, float top, double* values64, int lane) {
  double c[kPer];
  double z = 0.0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = 32 * j + lane;
    const float l = e < p.E ? select_load(row + e) : neg_inf();
    const bool in = l > neg_inf();
    const double x = exp(p.sigmoid ? (in ? -static_cast<double>(l) : 0.0) : (in ? below<double>(l, top) : 0.0));
    c[j] = in ? x : -1.0;  // -1: not to be chosen
    z += in ? x : 0.0;
  }
  if (!p.sigmoid) z = warp_sum(z);
  uint64_t keys[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = 32 * j + lane;
    const bool in = c[j] >= 0.0;
    double v = p.sigmoid ? 1.0 / (1.0 + (in ? c[j] : 0.0)) : (in ? c[j] : 0.0) / z;
    if (p.bias != nullptr && e < p.E) v += static_cast<double>(p.bias[e]);
    keys[j] = in ? order_key(v) : 0;
    if (e < p.E) {
      values64[e] = keys[j] != 0 ? v : static_cast<double>(neg_inf());
      // without a bias logits are compared, as in the 32-bit form
      if (p.bias == nullptr && keys[j] != 0) keys[j] = order_key(static_cast<double>(select_load(row + e)));
    }
  }
  __syncwarp();
  int chosen;
  choose<kPer, uint64_t, double>(keys, values64, 0.0, false, false, p, lane, chosen);
  return chosen;
}

template <int kPer, typename L>
__global__ void __launch_bounds__(32 * kSelectWarps) select_experts_kernel(const SelectParams p) {
  extern __shared__ double select_smem[];  // a row of E doubles per warp where values are compared
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kSelectWarps + warp;
  if (t >= p.T) return;
  const L* row = static_cast<const L*>(p.logits) + t * p.stride;
  int chosen = -1;
  float score = 0.f;
  if (p.mask == nullptr || p.mask[t] != 0) {
    float l[kPer];
    float top = neg_inf();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = 32 * j + lane;
      l[j] = e < p.E ? select_load(row + e) : neg_inf();
      if (!(l[j] > neg_inf())) l[j] = neg_inf();  // NaN
      top = fmaxf(top, l[j]);
    }
    const bool by_value = p.bias != nullptr;
    const bool values = by_value || p.groups > 1;
    float z = 1.f;
    if (!p.sigmoid) {
      top = warp_max(top);
      if (values || !p.renormalize) {
        z = 0.f;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (l[j] > neg_inf()) z += expf(below<float>(l[j], top));
        z = warp_sum(z);
      }
    }
    double* row64 = select_smem + static_cast<int64_t>(warp) * p.E;
    float* row32 = reinterpret_cast<float*>(row64);
    uint32_t keys[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = 32 * j + lane;
      keys[j] = order_key(l[j]);
      if (values && e < p.E) {
        float c = neg_inf();
        if (keys[j] != 0) {
          c = p.sigmoid ? 1.0f / (1.0f + expf(-l[j])) : expf(below<float>(l[j], top)) / z;
          if (by_value) c += p.bias[e];
          if (!(c > neg_inf())) c = neg_inf();
          if (by_value) keys[j] = order_key(c);
        }
        if (p.groups > 1) row32[e] = c;
      }
    }
    if (p.groups > 1) __syncwarp();
    // Error of p, in units of 2^-24.  Sigmoid: exponential 4 times p (1 - p), sum and quotient 1 each times p: under 3.  Softmax, relative
    // to p <= 1 / z: rounding of the exponent d e^-d <= 0.4, exponential 4, a sum of up to 1024 such terms in 37 roundings, quotient 1:
    // under 64.  The bias' addition is half a unit of c in the last place.
    const float tolerance = p.sigmoid ? 0x1p-22f : 0x1p-18f / z;
    // without a bias experts go by their logits, exactly
    const Found found = choose<kPer, uint32_t, float>(keys, row32, tolerance, values, by_value, p, lane, chosen);
    if (found.near_groups || (found.near_experts && found.rounds == 32)) {
      __syncwarp();
      chosen = choose_again<kPer, L>(p, row, top, row64, lane);
    } else if (found.near_experts) {
      chosen = order_again<L>(p, row, top, p.sigmoid ? 1.0 : sum_again<kPer, L>(p, row, top, lane), found.rounds, chosen, lane);
    }
    // lane k: the score of the k-th
    const bool have = lane < p.K && chosen >= 0;
    const float lk = have ? select_load(row + chosen) : neg_inf();
    if (p.renormalize) {
      // relative to the largest chosen logit, so that nothing underflows together: p_k = e^(l - m) (softmax) or e^(l - m) / (1 + e^l)
      float m = warp_max(lk);
      if (p.sigmoid && m > 0.f) m = 0.f;
      float v = 0.f;
      if (have) v = !p.sigmoid ? expf(below<float>(lk, m)) : lk >= 0.f ? 1.0f / (1.0f + expf(-lk)) : expf(below<float>(lk, m)) / (1.0f + expf(lk));
      const float sum = warp_sum(v);
      if (have) score = p.scale * (v / sum);
    } else if (have) {
      score = p.scale * (p.sigmoid ? 1.0f / (1.0f + expf(-lk)) : expf(below<float>(lk, top)) / z);
    }
  }
  if (lane < p.K) {
    const int64_t at = t * p.K + lane;
    if (p.ids_are_int64)
      static_cast<int64_t*>(p.ids)[at] = chosen;
    else
      static_cast<int32_t*>(p.ids)[at] = chosen;
    if (p.scores_are_bf16)
      static_cast<__nv_bfloat16*>(p.scores)[at] = __float2bfloat16_rn(score);
    else
      static_cast<float*>(p.scores)[at] = score;
  }
}

struct SelectGradParams {
  const void* logits;
  int64_t stride, T;
  int E, K, sigmoid, renormalize;
  float scale;
  const void* ids;
  const void* grad_scores;
  int ids_are_int64, scores_are_bf16;
  void* grad_logits;  // [T, E]
};

template <typename L>
__global__ void __launch_bounds__(32 * kSelectWarps) select_experts_bwd_kernel(const SelectGradParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kSelectWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  const L* row = static_cast<const L*>(p.logits) + t * p.stride;
  L* out = static_cast<L*>(p.grad_logits) + t * p.E;
  int id = -1;
  float g = 0.f, l = neg_inf();
  if (lane < p.K) {
    const int64_t at = t * p.K + lane;
    id = static_cast<int>(p.ids_are_int64 ? static_cast<const int64_t*>(p.ids)[at] : static_cast<const int32_t*>(p.ids)[at]);
    if (id >= p.E) id = -1;
    if (id >= 0) {
      l = select_load(row + id);
      g = p.scale * (p.scores_are_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.grad_scores)[at])
                                       : static_cast<const float*>(p.grad_scores)[at]);
    }
  }
  const bool have = id >= 0;
  float own = 0.f;  // gradient of the lane's chosen logit
  if (p.renormalize || p.sigmoid) {
    const float q = have ? 1.0f / (1.0f + expf(l)) : 0.f;  // 1 - sigmoid
    if (p.renormalize) {
      float m = warp_max(l);
      if (p.sigmoid && m > 0.f) m = 0.f;
      float v = 0.f;
      if (have) v = !p.sigmoid ? expf(below<float>(l, m)) : l >= 0.f ? 1.0f / (1.0f + expf(-l)) : expf(below<float>(l, m)) * q;
      const float sum = warp_sum(v);
      const float w = have ? v / sum : 0.f;
      const float mean = warp_sum(w * g);
      own = w * (g - mean) * (p.sigmoid ? q : 1.0f);
    } else if (have) {
      own = g * q / (1.0f + expf(-l));
    }
    for (int e = lane; e < p.E; e += 32) select_store(out + e, 0.f);
  } else {
    float top = neg_inf();
    for (int e = lane; e < p.E; e += 32) {
      const float x = select_load(row + e);
      if (x > top) top = x;
    }
    top = warp_max(top);
    float z = 0.f;
    for (int e = lane; e < p.E; e += 32) {
      const float x = select_load(row + e);
      if (x > neg_inf()) z += expf(below<float>(x, top));
    }
    z = warp_sum(z);
    const float v = have ? expf(below<float>(l, top)) / z : 0.f;
    const float dot = warp_sum(v * g);
    own = v * (g - dot);
    for (int e = lane; e < p.E; e += 32) {
      const float x = select_load(row + e);
      select_store(out + e, x > neg_inf() ? -dot * (expf(below<float>(x, top)) / z) : 0.f);
    }
  }
  __syncwarp();  // the chosen ones over what was just written
  if (have) select_store(out + id, own);
}

}  // namespace dm

using namespace dm;

constexpr int kSelectMaxExperts = 1024;

extern "C" int dm_select_experts(const void* logits, int logits_are_bf16, int64_t stride, int64_t T, int E, int K, int sigmoid,
                                 const float* bias, int groups, int kept, int group_top, int renormalize, float scale,
                                 const void* mask, void* ids, int ids_are_int64, void* scores, int scores_are_bf16, void* stream) {
  if (T < 0 || T > (int64_t{1} << 32) || E <= 0 || K <= 0 || K > 32 || K > E || stride < 0) return kRcBadArg;
  if (groups <= 0 || groups > 32 || E % groups != 0 || kept <= 0 || kept > groups || (group_top != 1 && group_top != 2)) return kRcBadArg;
  if (E > kSelectMaxExperts) return kRcTooLarge;
  if (T == 0) return kRcOk;
  if (!logits || !ids || !scores) return kRcBadArg;
  SelectParams p{logits, stride, T, E, K, groups, kept, group_top, sigmoid, renormalize, scale, bias,
                 static_cast<const unsigned char*>(mask), ids, scores, ids_are_int64, scores_are_bf16};
  const unsigned blocks = static_cast<unsigned>(ceil_div64(T, kSelectWarps));
  const size_t smem = bias != nullptr || groups > 1 ? static_cast<size_t>(kSelectWarps) * E * sizeof(double) : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&](auto per) {
    if (logits_are_bf16)
      select_experts_kernel<decltype(per)::value, __nv_bfloat16><<<blocks, 32 * kSelectWarps, smem, st>>>(p);
    else
      select_experts_kernel<decltype(per)::value, float><<<blocks, 32 * kSelectWarps, smem, st>>>(p);
    return static_cast<int>(cudaGetLastError());
  };
  if (E <= 32) return run(std::integral_constant<int, 1>{});
  if (E <= 64) return run(std::integral_constant<int, 2>{});
  if (E <= 128) return run(std::integral_constant<int, 4>{});
  if (E <= 256) return run(std::integral_constant<int, 8>{});
  if (E <= 512) return run(std::integral_constant<int, 16>{});
  return run(std::integral_constant<int, 32>{});
}

extern "C" int dm_select_experts_bwd(const void* logits, int logits_are_bf16, int64_t stride, int64_t T, int E, int K, int sigmoid,
                                     int renormalize, float scale, const void* ids, int ids_are_int64, const void* grad_scores,
                                     int scores_are_bf16, void* grad_logits, void* stream) {
  if (T < 0 || T > (int64_t{1} << 32) || E <= 0 || K <= 0 || K > 32 || K > E || stride < 0) return kRcBadArg;
  if (E > kSelectMaxExperts) return kRcTooLarge;
  if (T == 0) return kRcOk;
  if (!logits || !ids || !grad_scores || !grad_logits) return kRcBadArg;
  const SelectGradParams p{logits, stride, T, E, K, sigmoid, renormalize, scale, ids, grad_scores, ids_are_int64, scores_are_bf16, grad_logits};
  const unsigned blocks = static_cast<unsigned>(ceil_div64(T, kSelectWarps));
  if (logits_are_bf16)
    select_experts_bwd_kernel<__nv_bfloat16><<<blocks, 32 * kSelectWarps, 0, static_cast<cudaStream_t>(stream)>>>(p);
  else
    select_experts_bwd_kernel<float><<<blocks, 32 * kSelectWarps, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return static_cast<int>(cudaGetLastError());
}
