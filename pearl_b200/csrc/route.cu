// route.cu -- the router of a MoE layer: the top_k experts of every token and
// their weights from the router's logits (see pb2_route_tokens).
//
// kLanes lanes work on a token (a warp on 32 / kLanes of them); lane l of
// them holds the kPer consecutive experts from l * kPer on, so that the
// lowest lane with a key holds the lowest expert with it.  Each lane sorts
// its keys (bare values: min and max only); a round of the choice is then a
// maximum over the lanes' heads, one ballot and a pop in the winner's lane.
// Which of the winner's experts a key belongs to is looked up once at the
// end, one lane per chosen expert, as are the scores: sigmoids without a
// bias are taken of the chosen alone, and renormalized softmax weights are a
// softmax over the chosen, which needs no other exponential.
//
// 32768 tokens of 128 f32 logits take 12.1 us (1.6 TB/s of 6.5).  An SM at work
// issues in 61% of its slots, with 7.7 warps a scheduler of which 2.2 could go
// on; what the others wait for is, in this order, their logits, the integer
// pipe (minima, maxima and selects, 53% busy), shuffles.  Over the whole launch
// 44% of the slots: the rest is its start and its last blocks.  A warp per
// token with indices carried through the rounds and all scores computed took
// 27 us, bare keys 20, no exponentials beside the chosen 16, eight lanes a
// token 11.4, the full exponential 12.1.  4099 tokens of 256 experts in 8
// groups with a bias: 8.2 us; 4 tokens of 8 experts: 1.9 us.
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

// The kPer logits from e0 on of the row starting at element `row` (-inf past
// the last expert).  a.vec: whole vectors of min(kPer, 4) logits, aligned.
template <int kPer>
__device__ __forceinline__ void load_lane(const RouteArgs& a, int64_t row, int e0, float* x) {
  constexpr int kVec = kPer < 4 ? kPer : 4;
  if (kVec > 1 && a.vec) {
    const bool f16 = a.type == PB2_TYPE_F16;
#pragma unroll
    for (int j = 0; j < kPer; j += kVec) {
      float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (e0 + j < a.experts) {
        if (a.type == PB2_TYPE_F32) {
          const float* p = static_cast<const float*>(a.logits) + row + e0 + j;
          if constexpr (kVec == 4) {
            const float4 w = *reinterpret_cast<const float4*>(p);
            v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
          } else {
            const float2 w = *reinterpret_cast<const float2*>(p);
            v[0] = w.x; v[1] = w.y;
          }
        } else {
          const uint16_t* p = static_cast<const uint16_t*>(a.logits) + row + e0 + j;
          uint2 w = make_uint2(0u, 0u);
          if constexpr (kVec == 4) w = *reinterpret_cast<const uint2*>(p);
          else w.x = *reinterpret_cast<const uint32_t*>(p);
          const float2 f = unpack_half2(w.x, f16), g = unpack_half2(w.y, f16);
          v[0] = f.x; v[1] = f.y; v[2] = g.x; v[3] = g.y;
        }
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) x[j + i] = clean(v[i]);
    }
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
// both are infinite).  In full f32: the one-instruction exponential loses
// 2^-17 at 80 below the top, and with a bias the scores decide the choice.
__device__ __forceinline__ float softmax_term(float v, float top) {
  return v == -INFINITY ? 0.f : v == top ? 1.f : expf(v - top);
}

// Sum and maximum over the kLanes lanes of a token.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (kLanes == 32) return __reduce_max_sync(kAll, v);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// Keys of a lane in descending order: Batcher's odd-even merge sort (1, 5,
// 19, 63 comparators).
template <int kPer>
__device__ __forceinline__ void sort_lane(uint32_t* key) {
#pragma unroll
  for (int p = 1; p < kPer; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < kPer; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < kPer && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint32_t hi = max(key[i + j], key[i + j + k]);
            key[i + j + k] = min(key[i + j], key[i + j + k]);
            key[i + j] = hi;
          }
}

template <int kLanes, int kPer, bool kGroups>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const RouteArgs a) {
  constexpr int kTokens = 32 / kLanes * kRouteWarps;  // of a CTA
  constexpr int kKept = kPer < kLanes ? kPer : kLanes;  // top_k <= kLanes: no lane gives up more keys
  constexpr uint32_t kMask = kLanes == 32 ? kAll : (1u << kLanes) - 1u;
  __shared__ __align__(16) uint32_t s_key[kTokens][kLanes * kPer];
  __shared__ uint32_t s_group[kTokens][kGroups ? kLanes * kPer : 1];
  const int lane = threadIdx.x % kLanes, slot = threadIdx.x / kLanes;
  const int base = threadIdx.x % 32 - lane;  // the token's first lane in its warp
  const int t = blockIdx.x * kTokens + slot;
  const bool live = t < a.tokens;
  griddep_wait();
  griddep_launch_dependents();
  uint32_t* keys = s_key[slot];
  const int64_t row = int64_t(live ? t : 0) * a.experts;
  float x[kPer];
  load_lane<kPer>(a, row, lane * kPer, x);
  // The row's softmax statistics, where they are needed.
  float top = -INFINITY, sum = 0.f;
  const bool full = !a.sigmoid && (!a.renorm || a.bias);
  if (full) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) top = fmaxf(top, x[j]);
    top = key_value(lanes_max<kLanes>(order_key(top)));
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += softmax_term(x[j], top);
    sum = lanes_sum<kLanes>(sum);
  }
  uint32_t key[kPer];
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = lane * kPer + j;
      float c = x[j];
      if (c != -INFINITY) c = (a.sigmoid ? sigmoid_exact(c) : softmax_term(c, top) / sum) + a.bias[e];
      key[j] = e >= a.experts ? kOut : order_key(c);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) key[j] = lane * kPer + j >= a.experts ? kOut : order_key(x[j]);
  }
  if constexpr (kPer == 1) {
    keys[lane] = key[0];
  } else if constexpr (kPer == 2) {
    *reinterpret_cast<uint2*>(keys + 2 * lane) = make_uint2(key[0], key[1]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; j += 4)
      *reinterpret_cast<uint4*>(keys + lane * kPer + j) = make_uint4(key[j], key[j + 1], key[j + 2], key[j + 3]);
  }
  if (kGroups && a.group_lanes == 0) {
    __syncwarp();
    const int width = a.experts / a.groups;
    uint32_t* kept = s_group[slot];
    // Group g's value in lane g % kLanes, element g / kLanes.
    uint32_t value[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = lane + kLanes * i;
      value[i] = kOut;
      kept[g] = 0u;
      if (g < a.groups) {
        uint32_t first = kOut, second = kOut;
        for (int j = 0; j < width; ++j) {
          const uint32_t k = keys[g * width + j];
          second = max(second, min(first, k));
          first = max(first, k);
        }
        value[i] = a.bias && width > 1 ? order_key(key_value(first) + key_value(second)) : first;
      }
    }
    for (int r = 0; r < a.kept; ++r) {
      uint32_t best = value[0];
#pragma unroll
      for (int i = 1; i < kPer; ++i) best = max(best, value[i]);
      best = lanes_max<kLanes>(best);
      uint32_t at = 0x7fffffffu;
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i)
        if (value[i] == best) at = lane + kLanes * i;
      at = ~lanes_max<kLanes>(~at);  // the lowest
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (at == uint32_t(lane + kLanes * i)) { value[i] = kOut; kept[at] = 1u; }
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = lane * kPer + j;
      if (e < a.experts && !kept[e / width]) {
        key[j] = kOut;
        keys[e] = kOut;
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
      const uint32_t best = lanes_max<kLanes>(value);
      const uint32_t heads = (__ballot_sync(kAll, value == best) >> base) & kMask;
      if ((__ffs(heads) - 1) / a.group_lanes == group) { in = true; value = kOut; }
    }
    if (!in) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        key[j] = kOut;
        keys[lane * kPer + j] = kOut;
      }
    }
  }
  // Lane r learns the r-th chosen key and which lanes' heads it was (the
  // lowest of them gives it up).
  uint32_t my_key = 0, my_heads = 0;
  const uint32_t bit = 1u << lane, up_to = bit | (bit - 1u);
  for (int r = 0; r < a.top_k; ++r) {
    const uint32_t best = lanes_max<kLanes>(key[0]);
    const uint32_t heads = (__ballot_sync(kAll, key[0] == best) >> base) & kMask;
    const bool mine = (heads & up_to) == bit;
    my_key = lane == r ? best : my_key;
    my_heads = lane == r ? heads : my_heads;
#pragma unroll
    for (int j = 0; j + 1 < kKept; ++j) key[j] = mine ? key[j + 1] : key[j];
    key[kKept - 1] = mine ? kOut : key[kKept - 1];
  }
  // Equal keys of one lane follow one another in the rounds; the n-th of them
  // is the n-th of the lane's experts with that key.
  const int from = __ffs(my_heads) - 1;
  const uint32_t last_key = __shfl_up_sync(kAll, my_key, 1, kLanes);
  const int last_from = __shfl_up_sync(kAll, from, 1, kLanes);
  const uint32_t again =
      __ballot_sync(kAll, lane > 0 && lane < a.top_k && my_key == last_key && from == last_from) >> base;
  int skip = __clz(~(again << (31 - lane)));
  __syncwarp();
  int id = 0;
  float v = -INFINITY;
  if (lane < a.top_k) {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (keys[from * kPer + j] == my_key && skip-- == 0) id = from * kPer + j;
    v = load_logit(a, row + id);
  }
  if (!a.sigmoid && !full) top = key_value(lanes_max<kLanes>(order_key(v)));
  float w = a.sigmoid ? sigmoid_exact(v) : full ? softmax_term(v, top) / sum : softmax_term(v, top);
  if (lane >= a.top_k || !(w > 0.f)) w = 0.f;  // 0 / 0: a row that masks every expert
  if (a.renorm) {
    const float total = lanes_sum<kLanes>(w);
    w = total > 0.f ? w / total : 0.f;
  }
  if (live && lane < a.top_k) {
    a.weights[int64_t(t) * a.top_k + lane] = w * a.scaling;
    a.ids[int64_t(t) * a.top_k + lane] = id;
  }
}

template <int kLanes, int kPer>
int launch_route(RouteArgs& a, cudaStream_t s) {
  constexpr int kTokens = 32 / kLanes * kRouteWarps;
  const int width = a.experts / a.groups, lanes = width / kPer;
  a.group_lanes = a.groups > 1 && width % kPer == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  constexpr int kVec = kPer < 4 ? kPer : 4;
  a.vec = a.experts % kVec == 0 &&
          reinterpret_cast<uintptr_t>(a.logits) % (kVec * (a.type == PB2_TYPE_F32 ? 4 : 2)) == 0;
  const dim3 grid(unsigned((a.tokens + kTokens - 1) / kTokens));
  if (a.groups > 1) return launch_programmatic(route_kernel<kLanes, kPer, true>, grid, 32 * kRouteWarps, 0, s, 1, a);
  return launch_programmatic(route_kernel<kLanes, kPer, false>, grid, 32 * kRouteWarps, 0, s, 1, a);
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
  // Many tokens: as few lanes a token as the choice allows (a lane per chosen
  // expert), whose rounds' instructions then serve several tokens at once.
  // Few tokens: a warp a token, whose chain is shorter (fewer experts a lane
  // to score, sort and look up).  8 lanes | 32 lanes, us: 64 experts, top 6,
  // 2048 tokens 2.64 | 2.53, 4099 2.78 | 3.07, 32768 6.9 | 12.8; 128 experts,
  // top 8, 512 tokens 3.2 | 2.3, 4099 3.7 | 3.6, 8192 4.9 | 5.7, and with a
  // bias, which takes every expert's score, 512 5.8 | 3.0, 8192 7.3 | 6.8,
  // 32768 16 | 19; 256 experts in 16 lanes | 32, 64 tokens 3.5 | 2.4, 32768
  // 22.8 | 22.1, and with groups and a bias 7.1 | 4.4 and 41 | 38.  (Where it
  // is off most: a whole softmax over 128 at 9000 tokens, 5.8 | 6.4.)
  const bool scores = a.bias || (!a.sigmoid && !a.renorm);
  const int64_t few = int64_t(sm_count(p.device)) * (a.experts <= 64 ? 16 : 32) * (scores ? 2 : 1);
  if (a.tokens > few && a.top_k <= 8 && a.experts <= 128) {
    if (a.experts <= 32) return launch_route<8, 4>(a, s);
    return a.experts <= 64 ? launch_route<8, 8>(a, s) : launch_route<8, 16>(a, s);
  }
  if (a.tokens > few && a.top_k <= 16 && a.experts > 64 && a.experts <= 128) return launch_route<16, 8>(a, s);
  if (a.experts <= 32) return launch_route<32, 1>(a, s);
  if (a.experts <= 64) return launch_route<32, 2>(a, s);
  return a.experts <= 128 ? launch_route<32, 4>(a, s) : launch_route<32, 8>(a, s);
}
