// Top-k expert router with counts, a balance loss and a z loss, for sm_100a.
//
//   p = softmax(logits[t]);  experts[t] = k largest, weights = p at them
//   balance = mean over frames of  E / (k n_s^2) sum_e counts[s, e] P[s, e],
//   P[s, e] = sum over the valid tokens of s of p[t, e];  z = mean lse^2
//
// Gradient, with a_e the cotangent of p_e (share[s, e] grad_balance, plus the
// weight's where it is p_e itself):
//   dlogit_e = p_e (a_e - sum_j p_j a_j) + 2 / n grad_z lse p_e
//   and, for renormalised weights w, + w_i (gw_i - sum_j w_j gw_j) at expert i.
//
// One warp per token with the row in registers.  Largest logits are found in
// an order-preserving integer form by warp-wide integer reductions; ties go to
// the lowest index.  P and the counts are sums of integers: p is rounded to a
// multiple of 2^-shift (shift such that all tokens fit 62 bits, 40 at most),
// so integer atomics give the same sum in any order, with an absolute error
// of 2^-shift a token, below that of a float sum.
#include "launch.cuh"

namespace bysj {
namespace {

struct RouteArgs {
  const void* logits;
  int64_t tokens;
  int experts, k;
  const uint8_t* mask;
  const int64_t* offsets;
  int64_t frames;
  int renormalize;
  float* weights;
  int64_t* chosen;
  int64_t* counts;
  float* balance;
  float* z;
  float* z_scale;
  float* denom;
  float* share;
  unsigned long long* mass;    // [frames][experts] sum of p in units of 2^-shift
  unsigned long long* number;  // [frames] valid tokens
  unsigned* poison;            // a probability was not a number
  double* square;              // [CTAs] sum of lse^2
  int shift;
  int ctas;
  const float* grad_weights;
  const float* grad_balance;
  const float* grad_z;
  void* grad_logits;
};

__device__ __forceinline__ float load_f32(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

// Unsigned key in the order of the logits, with 0 for -inf (never chosen) and
// NaN above all; + 0.0f makes the two zeros equal.
__device__ __forceinline__ unsigned order_key(float v) {
  if (v == -INFINITY) return 0u;
  if (isnan(v)) return 0xffffffffu;
  const unsigned b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Frame of token t: the last whose offset is <= t.
__device__ __forceinline__ int64_t frame_of(const RouteArgs& a, int64_t t) {
  if (a.offsets == nullptr) return 0;
  int64_t lo = 0, hi = a.frames - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (__ldg(a.offsets + mid) <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float warp_max(float v) { return xor_max(v, 1); }
__device__ __forceinline__ float warp_sum(float v) { return xor_sum(v, 1); }

template <typename T, int NV>
__global__ void __launch_bounds__(kBlock) route_forward_kernel(RouteArgs a) {
  __shared__ double s_square[kWarpsPerBlock];
  const int lane = lane_id();
  const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarpsPerBlock;
  const float unit = static_cast<float>(int64_t{1} << a.shift);
  double square = 0.0;
  for (int64_t t = global_warp(); t < a.tokens; t += warps) {
    const T* row = static_cast<const T*>(a.logits) + t * a.experts;
    const bool on = a.mask == nullptr || __ldg(a.mask + t) != 0;
    float x[NV];
    unsigned key[NV];
    float top = -INFINITY;
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + i * kWarp;
      x[i] = on && e < a.experts ? load_f32(row + e) : -INFINITY;
      key[i] = order_key(x[i]);
      any |= key[i];
      top = fmaxf(top, x[i]);
    }
    top = warp_max(top);
    const bool valid = __any_sync(kFull, any != 0);
    if (!valid) {
      for (int i = lane; i < a.k; i += kWarp) {
        a.weights[t * a.k + i] = 0.0f;
        a.chosen[t * a.k + i] = -1;
      }
      if (lane == 0) a.denom[t] = 1.0f;
      continue;
    }
    float total = 0.0f, p[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      p[i] = x[i] == -INFINITY ? 0.0f : expf(x[i] - top);
      total += p[i];
    }
    total = warp_sum(total);
    const int64_t s = frame_of(a, t);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + i * kWarp;
      p[i] /= total;
      if (e < a.experts && p[i] != 0.0f) {
        if (isnan(p[i])) atomicOr(a.poison, 1u);
        else atomicAdd(a.mass + s * a.experts + e, static_cast<unsigned long long>(
                                                       __float2ull_rn(p[i] * unit)));
      }
    }
    // k times the largest remaining key, the lowest index among equals; lane i
    // keeps slot i
    float mine = 0.0f, picked = 0.0f;
    int64_t index = -1;
    for (int slot = 0; slot < a.k; ++slot) {
      unsigned best = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(kFull, best);
      if (best == 0) break;
      unsigned where = 0xffffffffu;
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
        if (key[i] == best) where = lane + i * kWarp;
      where = __reduce_min_sync(kFull, where);
      float value = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (lane + i * kWarp == static_cast<int>(where)) {
          key[i] = 0;
          value = p[i];
          atomicAdd(reinterpret_cast<unsigned long long*>(a.counts) + s * a.experts + where, 1ull);
        }
      value = __shfl_sync(kFull, value, where & 31);
      picked += value;
      if (lane == slot) {
        mine = value;
        index = where;
      }
    }
    if (lane < a.k) {
      a.weights[t * a.k + lane] = a.renormalize && index >= 0 ? mine / picked : mine;
      a.chosen[t * a.k + lane] = index;
    }
    if (lane == 0) {
      a.denom[t] = total;
      atomicAdd(a.number + s, 1ull);
      const float lse = top + logf(total);
      square += static_cast<double>(lse) * lse;
    }
  }
  if (lane == 0) s_square[threadIdx.x / kWarp] = square;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kWarpsPerBlock; ++i) square += s_square[i];
    a.square[blockIdx.x] = square;
  }
}

__device__ __forceinline__ double block_sum(double v, double* scratch) {
  v = xor_sum(v, 1);
  __syncthreads();
  if (lane_id() == 0) scratch[threadIdx.x / kWarp] = v;
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < kWarpsPerBlock; ++i) total += scratch[i];
  return total;
}

__global__ void __launch_bounds__(kBlock) route_losses_kernel(RouteArgs a) {
  __shared__ double scratch[kWarpsPerBlock];
  double used = 0.0, valid = 0.0, square = 0.0, balance = 0.0;
  for (int64_t s = threadIdx.x; s < a.frames; s += kBlock) {
    used += a.number[s] > 0;
    valid += static_cast<double>(a.number[s]);
  }
  for (int i = threadIdx.x; i < a.ctas; i += kBlock) square += a.square[i];
  used = block_sum(used, scratch);
  valid = block_sum(valid, scratch);
  square = block_sum(square, scratch);
  const double unit = 1.0 / static_cast<double>(int64_t{1} << a.shift);
  for (int64_t i = threadIdx.x; i < a.frames * a.experts; i += kBlock) {
    const double n = static_cast<double>(a.number[i / a.experts]);
    const double share =
        n > 0.0 ? a.experts * static_cast<double>(a.counts[i]) / (a.k * n * n * used) : 0.0;
    a.share[i] = static_cast<float>(share);
    balance += share * (static_cast<double>(a.mass[i]) * unit);
  }
  balance = block_sum(balance, scratch);
  if (threadIdx.x == 0) {
    *a.balance = *a.poison ? NAN : static_cast<float>(balance);
    *a.z = valid > 0.0 ? static_cast<float>(square / valid) : 0.0f;
    *a.z_scale = valid > 0.0 ? static_cast<float>(2.0 / valid) : 0.0f;
  }
}

template <typename T, int NV>
__global__ void __launch_bounds__(kBlock) route_backward_kernel(RouteArgs a) {
  const int lane = lane_id();
  const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarpsPerBlock;
  const float gb = a.grad_balance ? __ldg(a.grad_balance) : 0.0f;
  const float gz = a.grad_z ? __ldg(a.grad_z) * *a.z_scale : 0.0f;
  for (int64_t t = global_warp(); t < a.tokens; t += warps) {
    const T* row = static_cast<const T*>(a.logits) + t * a.experts;
    T* out = static_cast<T*>(a.grad_logits) + t * a.experts;
    const int64_t first = a.chosen[t * a.k];
    if (first < 0) {  // not a valid token
      for (int e = lane; e < a.experts; e += kWarp) store_value(out + e, 0.0f);
      continue;
    }
    const float top = load_f32(row + first), total = a.denom[t];
    const int64_t s = frame_of(a, t);
    float p[NV], cot[NV], direct[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + i * kWarp;
      const float x = e < a.experts ? load_f32(row + e) : -INFINITY;
      p[i] = x == -INFINITY ? 0.0f : expf(x - top) / total;
      cot[i] = e < a.experts ? gb * a.share[s * a.experts + e] : 0.0f;
      direct[i] = 0.0f;
    }
    if (a.grad_weights != nullptr) {
      const float gw = lane < a.k ? a.grad_weights[t * a.k + lane] : 0.0f;
      const float w = lane < a.k ? a.weights[t * a.k + lane] : 0.0f;
      const int index = lane < a.k ? static_cast<int>(a.chosen[t * a.k + lane]) : -1;
      const float along = a.renormalize ? warp_sum(w * gw) : 0.0f;
      for (int slot = 0; slot < a.k; ++slot) {
        const int e = __shfl_sync(kFull, index, slot);
        const float g = __shfl_sync(kFull, a.renormalize ? w * (gw - along) : gw, slot);
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (lane + i * kWarp == e) {
            if (a.renormalize) direct[i] = g;
            else cot[i] += g;
          }
      }
    }
    float along = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) along += p[i] * cot[i];
    along = warp_sum(along);
    const float pull = gz * (top + logf(total)) - along;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + i * kWarp;
      if (e < a.experts) store_value(out + e, p[i] * (cot[i] + pull) + direct[i]);
    }
  }
}

int route_ctas(int64_t tokens) {
  int64_t blocks = (tokens + kWarpsPerBlock - 1) / kWarpsPerBlock;
  const int64_t cap = static_cast<int64_t>(current_device_info().sm_count) * 8;
  if (blocks > cap) blocks = cap;
  return blocks < 1 ? 1 : static_cast<int>(blocks);
}

// The zeroed part comes first: mass, number, poison.
size_t carve_workspace(RouteArgs& a, void* workspace, size_t* zeroed) {
  Carver carve(workspace);
  a.mass = carve.take<unsigned long long>(static_cast<size_t>(a.frames) * a.experts);
  a.number = carve.take<unsigned long long>(static_cast<size_t>(a.frames));
  a.poison = carve.take<unsigned>(1);
  *zeroed = carve.need;
  a.square = carve.take<double>(static_cast<size_t>(a.ctas));
  return carve.need;
}

using RouteKernel = void (*)(RouteArgs);

template <typename T, bool BACKWARD>
RouteKernel route_pick(int experts) {
#define BYSJ_ROUTE_CASE(NV) \
  if (experts <= NV * kWarp) return BACKWARD ? route_backward_kernel<T, NV> : route_forward_kernel<T, NV>;
  BYSJ_ROUTE_CASE(1)
  BYSJ_ROUTE_CASE(2)
  BYSJ_ROUTE_CASE(4)
  BYSJ_ROUTE_CASE(8)
  BYSJ_ROUTE_CASE(16)
  BYSJ_ROUTE_CASE(32)
#undef BYSJ_ROUTE_CASE
  return nullptr;
}

int check_sizes(int dtype, int64_t tokens, int64_t n_experts, int64_t k, const int64_t* offsets,
                int64_t frames) {
  if (dtype != BYSJ_F32 && dtype != BYSJ_BF16)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "route: unknown dtype %d", dtype);
  if (tokens < 0 || n_experts < 1 || frames < 0)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "route: invalid sizes");
  if (n_experts > BYSJ_ROUTE_MAX_EXPERTS)
    return fail(BYSJ_ERR_UNSUPPORTED, "route: at most %d experts", BYSJ_ROUTE_MAX_EXPERTS);
  if (k < 1 || k > n_experts || k > BYSJ_ROUTE_MAX_K)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "route: k must be 1 .. min(experts, %d)",
                BYSJ_ROUTE_MAX_K);
  if (offsets == nullptr ? frames != 1 : frames < 1 && tokens > 0)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "route: invalid number of frames");
  return BYSJ_OK;
}

}  // namespace
}  // namespace bysj

using namespace bysj;

extern "C" {

size_t bysj_route_forward_workspace_size(int64_t tokens, int64_t n_experts, int64_t frames) {
  if (tokens < 0 || n_experts < 1 || frames < 0) return 0;
  RouteArgs a{};
  a.experts = static_cast<int>(n_experts);
  a.frames = frames;
  a.ctas = route_ctas(tokens);
  size_t zeroed = 0;
  return carve_workspace(a, nullptr, &zeroed);
}

int bysj_route_forward(const void* logits, int dtype, int64_t tokens, int64_t n_experts,
                       int64_t k, const uint8_t* mask, const int64_t* offsets, int64_t frames,
                       int renormalize, float* weights, int64_t* experts, int64_t* counts,
                       float* balance, float* z, float* z_scale, float* denom, float* share,
                       void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int st = check_sizes(dtype, tokens, n_experts, k, offsets, frames);
  if (st) return st;
  if (balance == nullptr || z == nullptr || z_scale == nullptr ||
      (frames > 0 && (counts == nullptr || share == nullptr)) ||
      (tokens > 0 && (logits == nullptr || weights == nullptr || experts == nullptr ||
                      denom == nullptr)))
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "route: NULL pointer");
  RouteArgs a{};
  a.experts = static_cast<int>(n_experts);
  a.frames = frames;
  a.ctas = route_ctas(tokens);
  size_t zeroed = 0;
  const size_t need = carve_workspace(a, workspace, &zeroed);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(BYSJ_ERR_WORKSPACE, "route: workspace of %zu bytes needed, %zu given", need,
                workspace_bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = cuda_check(cudaMemsetAsync(workspace, 0, zeroed, s), "route: zero workspace");
  if (st == BYSJ_OK && frames > 0)
    st = cuda_check(cudaMemsetAsync(counts, 0, sizeof(int64_t) * frames * n_experts, s),
                    "route: zero counts");
  if (st) return st;
  a.logits = logits;
  a.tokens = tokens;
  a.k = static_cast<int>(k);
  a.mask = mask;
  a.offsets = offsets;
  a.renormalize = renormalize;
  a.weights = weights;
  a.chosen = experts;
  a.counts = counts;
  a.balance = balance;
  a.z = z;
  a.z_scale = z_scale;
  a.denom = denom;
  a.share = share;
  a.shift = 40;
  while ((tokens >> (62 - a.shift)) != 0) --a.shift;
  const RouteKernel kernel = dtype == BYSJ_F32 ? route_pick<float, false>(a.experts)
                                               : route_pick<__nv_bfloat16, false>(a.experts);
  kernel<<<a.ctas, kBlock, 0, s>>>(a);
  st = launch_check("route_forward_kernel");
  if (st) return st;
  route_losses_kernel<<<1, kBlock, 0, s>>>(a);
  return launch_check("route_losses_kernel");
}

int bysj_route_backward(const void* logits, int dtype, int64_t tokens, int64_t n_experts,
                        int64_t k, const int64_t* offsets, int64_t frames, int renormalize,
                        const float* weights, const int64_t* experts, const float* denom,
                        const float* share, const float* z_scale, const float* grad_weights,
                        const float* grad_balance, const float* grad_z, void* grad_logits,
                        void* stream) {
  clear_error();
  const int st = check_sizes(dtype, tokens, n_experts, k, offsets, frames);
  if (st) return st;
  if (tokens == 0) return BYSJ_OK;
  if (logits == nullptr || weights == nullptr || experts == nullptr || denom == nullptr ||
      share == nullptr || z_scale == nullptr || grad_logits == nullptr)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "route backward: NULL pointer");
  RouteArgs a{};
  a.logits = logits;
  a.tokens = tokens;
  a.experts = static_cast<int>(n_experts);
  a.k = static_cast<int>(k);
  a.offsets = offsets;
  a.frames = frames;
  a.renormalize = renormalize;
  a.weights = const_cast<float*>(weights);
  a.chosen = const_cast<int64_t*>(experts);
  a.denom = const_cast<float*>(denom);
  a.share = const_cast<float*>(share);
  a.z_scale = const_cast<float*>(z_scale);
  a.grad_weights = grad_weights;
  a.grad_balance = grad_balance;
  a.grad_z = grad_z;
  a.grad_logits = grad_logits;
  const RouteKernel kernel = dtype == BYSJ_F32 ? route_pick<float, true>(a.experts)
                                               : route_pick<__nv_bfloat16, true>(a.experts);
  kernel<<<route_ctas(tokens), kBlock, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_check("route_backward_kernel");
}

}  // extern "C"
