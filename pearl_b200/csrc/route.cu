// route.cu -- the router of a MoE layer: the top_k experts of every token and
// their weights from the router's logits (see pb2_route_tokens).
//
// A warp per token; lane l holds the experts l, l + 32, ...  The choice is
// top_k rounds of a warp-wide maximum over (key, index).
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
  int type, sigmoid, renorm;
  float scaling;
};

__device__ __forceinline__ float load_logit(const RouteArgs& a, int64_t i) {
  float x;
  if (a.type == PB2_TYPE_F32) x = static_cast<const float*>(a.logits)[i];
  else x = half_at(a.logits, i, a.type == PB2_TYPE_F16);
  return x == x ? x : -INFINITY;
}

__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 and +0 tie
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

// The largest of the warp's keys (kPer a lane, element i of lane l being
// number l + 32 i), the lowest number at equal keys; it leaves the keys.
template <int kPer>
__device__ __forceinline__ int take_best(uint32_t* key, int lane) {
  uint32_t best = key[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) best = max(best, key[i]);
  best = __reduce_max_sync(kAll, best);
  unsigned at = 0x7fffffffu;
#pragma unroll
  for (int i = kPer - 1; i >= 0; --i)
    if (key[i] == best) at = lane + 32 * i;
  at = __reduce_min_sync(kAll, at);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (at == unsigned(lane + 32 * i)) key[i] = kOut;
  return int(at);
}

template <int kPer>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const RouteArgs a) {
  __shared__ uint32_t s_key[kRouteWarps][32 * kPer];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int t = blockIdx.x * kRouteWarps + warp;
  griddep_wait();
  griddep_launch_dependents();
  if (t >= a.tokens) return;
  float x[kPer], score[kPer];
  uint32_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 32 * i;
    x[i] = e < a.experts ? load_logit(a, int64_t(t) * a.experts + e) : -INFINITY;
  }
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) score[i] = x[i] == -INFINITY ? 0.f : 1.0f / (1.0f + expf(-x[i]));
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) top = fmaxf(top, x[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      score[i] = x[i] == -INFINITY ? 0.f : x[i] == top ? 1.f : expf(x[i] - top);
      sum += score[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
#pragma unroll
    for (int i = 0; i < kPer; ++i) score[i] = sum > 0.f ? score[i] / sum : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 32 * i;
    key[i] = e >= a.experts ? kOut : order_key(x[i] == -INFINITY || !a.bias ? x[i] : score[i] + a.bias[e]);
  }
  if (a.groups > 1) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) s_key[warp][lane + 32 * i] = key[i];
    __syncwarp();
    const int width = a.experts / a.groups;
    uint32_t value[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = lane + 32 * i;
      value[i] = kOut;
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
    for (int r = 0; r < a.kept; ++r) {  // s_key: kept groups, by group
      const int g = take_best<kPer>(value, lane);
      if (r == 0) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) s_key[warp][lane + 32 * i] = 0u;
        __syncwarp();
      }
      if (lane == 0) s_key[warp][g] = 1u;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      if (e < a.experts && !s_key[warp][e / width]) key[i] = kOut;
    }
  }
  float sum = 0.f, mine = 0.f;
  int my_id = 0;
  for (int r = 0; r < a.top_k; ++r) {
    const int at = take_best<kPer>(key, lane);
    float s = score[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i)
      if (at / 32 == i) s = score[i];
    s = __shfl_sync(kAll, s, at & 31);
    sum += s;
    if (lane == r) { mine = s; my_id = at; }
  }
  if (lane < a.top_k) {
    if (a.renorm) mine = sum > 0.f ? mine / sum : 0.f;
    a.weights[int64_t(t) * a.top_k + lane] = mine * a.scaling;
    a.ids[int64_t(t) * a.top_k + lane] = my_id;
  }
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
  const dim3 grid(unsigned((p.num_tokens + kRouteWarps - 1) / kRouteWarps));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.experts <= 32) return launch_programmatic(route_kernel<1>, grid, 32 * kRouteWarps, 0, s, 1, a);
  if (a.experts <= 64) return launch_programmatic(route_kernel<2>, grid, 32 * kRouteWarps, 0, s, 1, a);
  if (a.experts <= 128) return launch_programmatic(route_kernel<4>, grid, 32 * kRouteWarps, 0, s, 1, a);
  return launch_programmatic(route_kernel<8>, grid, 32 * kRouteWarps, 0, s, 1, a);
}
