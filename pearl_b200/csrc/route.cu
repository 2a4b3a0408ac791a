// route.cu -- the router of a MoE layer: the top_k experts of every token and
// their weights from the router's logits (see pb2_route_tokens).
//
// A warp per token; lane l holds the kPer = ceil(experts / 32) consecutive
// experts from l * kPer on, so that the lowest lane with a key holds the
// lowest expert with it.  Each lane sorts its keys (bare values: min and max
// only); a round of the choice is then one warp-wide maximum of the lanes'
// heads, one ballot and a pop in the winner's lane.  Which of the winner's
// experts a key belongs to is looked up once at the end, one lane per chosen
// expert, as are the scores: a softmax needs every exponential only for its
// sum, sigmoids without a bias only those of the chosen.
//
// Bound by instruction issue (a few hundred per token), not by the logits'
// bytes: carrying indices through the rounds and computing all scores took
// 27 us for 32768 tokens of 128 experts and 19 us for 4099 of 256 in groups.
#include <algorithm>

#include "pb2_epilogue.cuh"

namespace pb2 {
namespace {

constexpr int kRouteWarps = 4;
constexpr int kMaxExperts = 256;
constexpr int kMaxTopK = 32;
constexpr unsigned kAll = 0xffffffffu;
// Keys: floats as unsigned integers in the same order (-inf, which masks an
// expert, is 0x007fffff); 0 is an expert that does not take part -- one of an
// excluded group, or one already chosen.
constexpr uint32_t kOut = 0u;

struct RouteArgs {
  const void* logits;
  const float* bias;
  float* weights;
  int32_t* ids;
  int tokens, experts, top_k, groups, kept;
  int type, sigmoid, renorm, vec;
  int group_lanes;  // lanes of a group where that is a whole power of two, else 0
  float scaling;
};

__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }

__device__ __forceinline__ float load_logit(const RouteArgs& a, int64_t i) {
  if (a.type == PB2_TYPE_F32) return clean(static_cast<const float*>(a.logits)[i]);
  return clean(half_at(a.logits, i, a.type == PB2_TYPE_F16));
}

// This lane's kPer logits of the row starting at element `row` (-inf past
// the last expert).  a.vec: whole lanes and aligned rows, wide loads.
template <int kPer>
__device__ __forceinline__ void load_lane(const RouteArgs& a, int64_t row, int lane, float* x) {
  const int e0 = lane * kPer;
  if (a.vec && e0 < a.experts) {
    if (a.type == PB2_TYPE_F32) {
      const float* p = static_cast<const float*>(a.logits) + row + e0;
      if constexpr (kPer == 1) {
        x[0] = p[0];
      } else if constexpr (kPer == 2) {
        const float2 v = *reinterpret_cast<const float2*>(p);
        x[0] = v.x; x[1] = v.y;
      } else {
#pragma unroll
        for (int j = 0; j < kPer; j += 4) {
          const float4 v = *reinterpret_cast<const float4*>(p + j);
          x[j] = v.x; x[j + 1] = v.y; x[j + 2] = v.z; x[j + 3] = v.w;
        }
      }
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(a.logits) + row + e0;
      const bool f16 = a.type == PB2_TYPE_F16;
      if constexpr (kPer == 1) {
        x[0] = half_at(p, 0, f16);
      } else {
        uint32_t w[kPer / 2];
        if constexpr (kPer == 2) {
          w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (kPer == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(p);
          w[0] = v.x; w[1] = v.y;
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(p);
          w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j) {
          const float2 f = unpack_half2(w[j], f16);
          x[2 * j] = f.x; x[2 * j + 1] = f.y;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = clean(x[j]);
    return;
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) x[j] = e0 + j < a.experts ? load_logit(a, row + e0 + j) : -INFINITY;
}

__device__ __forceinline__ uint32_t order_key(float x) {
  const int b = __float_as_int(clean(x) + 0.0f);  // -0 and +0 tie
  return uint32_t(b) ^ (uint32_t(b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ float sigmoid_exact(float x) { return x == -INFINITY ? 0.f : 1.0f / (1.0f + expf(-x)); }

// e^(v - top) with 0 for a masked logit and 1 for the top one (also where
// both are infinite).
__device__ __forceinline__ float softmax_term(float v, float top) {
  return v == -INFINITY ? 0.f : v == top ? 1.f : __expf(v - top);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Keys of a lane in descending order: minimal networks of 0, 1, 5 and 19
// comparators.
template <int kPer>
__device__ __forceinline__ void sort_lane(uint32_t* k) {
  auto order = [&](int i, int j) {
    const uint32_t hi = max(k[i], k[j]);
    k[j] = min(k[i], k[j]);
    k[i] = hi;
  };
  if constexpr (kPer == 2) order(0, 1);
  if constexpr (kPer == 4) { order(0, 2); order(1, 3); order(0, 1); order(2, 3); order(1, 2); }
  if constexpr (kPer == 8) {
    order(0, 2); order(1, 3); order(4, 6); order(5, 7);
    order(0, 4); order(1, 5); order(2, 6); order(3, 7);
    order(0, 1); order(2, 3); order(4, 5); order(6, 7);
    order(2, 4); order(3, 5);
    order(1, 4); order(3, 6);
    order(1, 2); order(3, 4); order(5, 6);
  }
}

template <int kPer, bool kGroups>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const RouteArgs a) {
  __shared__ __align__(16) uint32_t s_key[kRouteWarps][32 * kPer];
  __shared__ uint32_t s_group[kRouteWarps][kGroups ? 32 * kPer : 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int t = blockIdx.x * kRouteWarps + warp;
  griddep_wait();
  griddep_launch_dependents();
  if (t >= a.tokens) return;
  const int64_t row = int64_t(t) * a.experts;
  float x[kPer];
  load_lane<kPer>(a, row, lane, x);
  // The row's softmax statistics, where they are needed: renormalized
  // weights are a softmax over the chosen experts alone.
  float top = -INFINITY, sum = 0.f;
  const bool full = !a.sigmoid && (!a.renorm || a.bias);
  if (full) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) top = fmaxf(top, x[j]);
    top = key_value(__reduce_max_sync(kAll, order_key(top)));
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += softmax_term(x[j], top);
    sum = warp_sum(sum);
  }
  auto score = [&](float v) {
    if (a.sigmoid) return sigmoid_exact(v);
    return softmax_term(v, top) / sum;
  };
  uint32_t key[kPer];
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = lane * kPer + j;
      key[j] = e >= a.experts ? kOut : order_key(x[j] == -INFINITY ? x[j] : score(x[j]) + a.bias[e]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) key[j] = lane * kPer + j >= a.experts ? kOut : order_key(x[j]);
  }
  if constexpr (kPer == 1) {
    s_key[warp][lane] = key[0];
  } else if constexpr (kPer == 2) {
    *reinterpret_cast<uint2*>(&s_key[warp][2 * lane]) = make_uint2(key[0], key[1]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; j += 4)
      *reinterpret_cast<uint4*>(&s_key[warp][lane * kPer + j]) = make_uint4(key[j], key[j + 1], key[j + 2], key[j + 3]);
  }
  if (kGroups && a.group_lanes == 0) {
    __syncwarp();
    const int width = a.experts / a.groups;
    // Group g's value in lane g % 32, element g / 32.
    uint32_t value[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = lane + 32 * i;
      value[i] = kOut;
      s_group[warp][g] = 0u;
      if (g < a.groups) {
        uint32_t first = kOut, second = kOut;
        for (int j = 0; j < width; ++j) {
          const uint32_t k = s_key[warp][g * width + j];
          second = max(second, min(first, k));
          first = max(first, k);
        }
        value[i] = a.bias && width > 1 ? order_key(key_value(first) + key_value(second)) : first;
      }
    }
    __syncwarp();
    for (int r = 0; r < a.kept; ++r) {
      uint32_t best = value[0];
#pragma unroll
      for (int i = 1; i < kPer; ++i) best = max(best, value[i]);
      best = __reduce_max_sync(kAll, best);
      unsigned at = 0x7fffffffu;
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i)
        if (value[i] == best) at = lane + 32 * i;
      at = __reduce_min_sync(kAll, at);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (at == unsigned(lane + 32 * i)) { value[i] = kOut; s_group[warp][at] = 1u; }
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = lane * kPer + j;
      if (e < a.experts && !s_group[warp][e / width]) {
        key[j] = kOut;
        s_key[warp][e] = kOut;
      }
    }
  }
  sort_lane<kPer>(key);
  if (kGroups && a.group_lanes) {
    // A group is a power of two of whole lanes: its two best keys by a
    // butterfly over them.
    uint32_t first = key[0], second = kPer > 1 ? key[1 % kPer] : kOut;
    for (int o = a.group_lanes >> 1; o > 0; o >>= 1) {
      const uint32_t f = __shfl_xor_sync(kAll, first, o), n = __shfl_xor_sync(kAll, second, o);
      second = max(max(second, n), min(first, f));
      first = max(first, f);
    }
    uint32_t value = first;
    if (a.bias && a.experts > a.groups && first != kOut) value = order_key(key_value(first) + key_value(second));
    const int group = lane / a.group_lanes;
    bool in = false;
    for (int r = 0; r < a.kept; ++r) {
      const uint32_t best = __reduce_max_sync(kAll, value);
      const int from = __ffs(__ballot_sync(kAll, value == best)) - 1;
      if (from / a.group_lanes == group) { in = true; value = kOut; }
    }
    if (!in) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        key[j] = kOut;
        s_key[warp][lane * kPer + j] = kOut;
      }
    }
  }
  // Lane r learns the r-th chosen key and which lanes' heads it was (the
  // lowest of them gives it up).
  uint32_t my_key = 0, my_heads = 0;
  const uint32_t bit = 1u << lane, up_to = bit | (bit - 1u);
  for (int r = 0; r < a.top_k; ++r) {
    const uint32_t best = __reduce_max_sync(kAll, key[0]);
    const uint32_t heads = __ballot_sync(kAll, key[0] == best);
    const bool mine = (heads & up_to) == bit;
    my_key = lane == r ? best : my_key;
    my_heads = lane == r ? heads : my_heads;
#pragma unroll
    for (int j = 0; j + 1 < kPer; ++j) key[j] = mine ? key[j + 1] : key[j];
    key[kPer - 1] = mine ? kOut : key[kPer - 1];
  }
  // Equal keys of one lane follow one another in the rounds; the n-th of them
  // is the n-th of the lane's experts with that key.
  const int from = __ffs(my_heads) - 1;
  const uint32_t last_key = __shfl_up_sync(kAll, my_key, 1);
  const int last_from = __shfl_up_sync(kAll, from, 1);
  const uint32_t again = __ballot_sync(kAll, lane > 0 && lane < a.top_k && my_key == last_key && from == last_from);
  int skip = __clz(~(again << (31 - lane)));
  __syncwarp();
  int id = 0;
  float v = -INFINITY;
  if (lane < a.top_k) {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (s_key[warp][from * kPer + j] == my_key && skip-- == 0) id = from * kPer + j;
    v = load_logit(a, row + id);
  }
  if (!a.sigmoid && !full) top = key_value(__reduce_max_sync(kAll, order_key(v)));
  float w = a.sigmoid ? sigmoid_exact(v) : full ? softmax_term(v, top) / sum : softmax_term(v, top);
  if (lane >= a.top_k || !(w > 0.f)) w = 0.f;  // 0 / 0: a row that masks every expert
  if (a.renorm) {
    const float total = warp_sum(w);
    w = total > 0.f ? w / total : 0.f;
  }
  if (lane < a.top_k) {
    a.weights[int64_t(t) * a.top_k + lane] = w * a.scaling;
    a.ids[int64_t(t) * a.top_k + lane] = id;
  }
}

template <int kPer>
int launch_route(const RouteArgs& a, cudaStream_t s) {
  const dim3 grid(unsigned((a.tokens + kRouteWarps - 1) / kRouteWarps));
  if (a.groups > 1) return launch_programmatic(route_kernel<kPer, true>, grid, 32 * kRouteWarps, 0, s, 1, a);
  return launch_programmatic(route_kernel<kPer, false>, grid, 32 * kRouteWarps, 0, s, 1, a);
}

}  // namespace
}  // namespace pb2

extern "C" int pb2_route_tokens(const pb2_route_params* pp, void* stream) {
  pb2::NvtxRange nvtx_range("pb2_route_tokens");
  using namespace pb2;
  if (!pp) return PB2_ERR_INVALID_ARGUMENT;
  const pb2_route_params& p = *pp;
  if (p.num_tokens < 0 || p.num_tokens > INT32_MAX || p.num_experts <= 0 || p.num_experts > kMaxExperts || p.top_k <= 0 ||
      p.top_k > kMaxTopK)
    return PB2_ERR_INVALID_ARGUMENT;
  if (p.num_groups <= 0 || p.num_experts % p.num_groups != 0 || p.topk_groups <= 0 || p.topk_groups > p.num_groups ||
      p.top_k > p.topk_groups * (p.num_experts / p.num_groups))
    return PB2_ERR_INVALID_ARGUMENT;
  if (p.logits_type < PB2_TYPE_F32 || p.logits_type > PB2_TYPE_F16) return PB2_ERR_INVALID_ARGUMENT;
  if (p.scoring != PB2_SCORE_SOFTMAX && p.scoring != PB2_SCORE_SIGMOID) return PB2_ERR_INVALID_ARGUMENT;
  if (p.num_tokens > 0 && (!p.logits || !p.topk_weights || !p.topk_ids)) return PB2_ERR_INVALID_ARGUMENT;
  int st = set_device(p.device);
  if (st) return st;
  if (p.num_tokens == 0) return PB2_OK;
  RouteArgs a;
  a.logits = p.logits;
  a.bias = p.bias;
  a.weights = p.topk_weights;
  a.ids = p.topk_ids;
  a.tokens = int(p.num_tokens);
  a.experts = int(p.num_experts);
  a.top_k = int(p.top_k);
  a.groups = p.topk_groups < p.num_groups ? int(p.num_groups) : 1;
  a.kept = int(p.topk_groups);
  a.type = p.logits_type;
  a.sigmoid = p.scoring == PB2_SCORE_SIGMOID;
  a.renorm = p.renormalize;
  a.scaling = p.scaling;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int per = a.experts <= 32 ? 1 : a.experts <= 64 ? 2 : a.experts <= 128 ? 4 : 8;
  const int lane_bytes = per * (a.type == PB2_TYPE_F32 ? 4 : 2);
  a.vec = a.experts % per == 0 && reinterpret_cast<uintptr_t>(p.logits) % std::min(lane_bytes, 16) == 0;
  const int width = a.experts / a.groups, lanes = width / per;
  a.group_lanes = a.groups > 1 && width % per == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  switch (per) {
    case 1: return launch_route<1>(a, s);
    case 2: return launch_route<2>(a, s);
    case 4: return launch_route<4>(a, s);
    default: return launch_route<8>(a, s);
  }
}
