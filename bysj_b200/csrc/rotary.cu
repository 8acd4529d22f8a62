// Rotary positions with several axes for sm_100a, fp32 or bf16 heads.
//
//   theta[t, p] = positions[t, axis(p)] * inv_freq[p]
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin
//
// The gradient of x is the same rotation by -theta; a rotation keeps the cross
// product, so the gradient of theta is sum_h (gx2 x1 - gx1 x2) with x the
// forward input and gx the gradient just computed: neither y nor the angles
// are kept between the passes.
//
// One warp per token; a lane takes pairs p = lane, lane + 32, ..., evaluates
// sin and cos of its angle once and turns that pair of every head of q and k.
#include "launch.cuh"

namespace bysj {
namespace {

struct RotaryArgs {
  bysj_rotary_side side[2];
  const void* positions;
  int integer_positions;
  const float* inv_freq;
  int end[BYSJ_ROTARY_MAX_AXES];  // pairs before the end of each axis
  int axes;
  int pairs;
  int64_t tokens, dim;
  int interleaved;
  float sign;
  float* grad_positions;
};

__device__ __forceinline__ float load_f32(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

__device__ __forceinline__ int axis_of(const RotaryArgs& a, int p) {
  int axis = 0;
#pragma unroll
  for (int i = 0; i < BYSJ_ROTARY_MAX_AXES - 1; ++i)
    if (i < a.axes - 1 && p >= a.end[i]) axis = i + 1;
  return axis;
}

__device__ __forceinline__ float position_of(const RotaryArgs& a, int64_t t, int axis) {
  const int64_t i = t * a.axes + axis;
  if (a.integer_positions)
    return static_cast<float>(__ldg(static_cast<const long long*>(a.positions) + i));
  return __ldg(static_cast<const float*>(a.positions) + i);
}

template <typename T, bool POS_GRAD>
__global__ void __launch_bounds__(kBlock) rotary_kernel(RotaryArgs a) {
  const int lane = lane_id();
  const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarpsPerBlock;
  for (int64_t t = global_warp(); t < a.tokens; t += warps) {
    float grad[BYSJ_ROTARY_MAX_AXES] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = lane; p < a.pairs; p += kWarp) {
      const int axis = axis_of(a, p);
      const float freq = __ldg(a.inv_freq + p);
      float sine, cosine;
      sincosf(position_of(a, t, axis) * freq, &sine, &cosine);
      sine *= a.sign;
      const int64_t c1 = a.interleaved ? 2 * p : p;
      const int64_t c2 = a.interleaved ? 2 * p + 1 : p + a.pairs;
      float dtheta = 0.0f;
      for (int s = 0; s < 2; ++s) {
        const bysj_rotary_side& side = a.side[s];
        for (int64_t h = 0; h < side.heads; ++h) {
          const T* x = static_cast<const T*>(side.x) + t * side.x_token_stride +
                       h * side.x_head_stride;
          T* y = static_cast<T*>(side.y) + (t * side.heads + h) * a.dim;
          const float x1 = load_f32(x + c1), x2 = load_f32(x + c2);
          const float y1 = x1 * cosine - x2 * sine, y2 = x2 * cosine + x1 * sine;
          store_value(y + c1, y1);
          store_value(y + c2, y2);
          if constexpr (POS_GRAD) {
            const T* v = static_cast<const T*>(side.saved) + t * side.saved_token_stride +
                         h * side.saved_head_stride;
            dtheta += y2 * load_f32(v + c1) - y1 * load_f32(v + c2);
          }
        }
      }
      if constexpr (POS_GRAD) {
#pragma unroll
        for (int i = 0; i < BYSJ_ROTARY_MAX_AXES; ++i)
          if (i == axis) grad[i] += freq * dtheta;
      }
    }
    for (int s = 0; s < 2; ++s) {
      const bysj_rotary_side& side = a.side[s];
      for (int64_t h = 0; h < side.heads; ++h) {
        const T* x = static_cast<const T*>(side.x) + t * side.x_token_stride +
                     h * side.x_head_stride;
        T* y = static_cast<T*>(side.y) + (t * side.heads + h) * a.dim;
        for (int64_t c = 2 * a.pairs + lane; c < a.dim; c += kWarp) y[c] = x[c];
      }
    }
    if constexpr (POS_GRAD) {
#pragma unroll
      for (int i = 0; i < BYSJ_ROTARY_MAX_AXES; ++i) {
        const float total = xor_sum(grad[i], 1);
        if (lane == 0 && i < a.axes) a.grad_positions[t * a.axes + i] = total;
      }
    }
  }
}

}  // namespace
}  // namespace bysj

using namespace bysj;

extern "C" int bysj_rotary_axes(const bysj_rotary_side* q, const bysj_rotary_side* k, int dtype,
                                const void* positions, int integer_positions,
                                const float* inv_freq, const int64_t* sections, int axes,
                                int64_t tokens, int64_t dim, int interleaved, int inverse,
                                float* grad_positions, void* stream) {
  clear_error();
  if (dtype != BYSJ_F32 && dtype != BYSJ_BF16)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "rotary: unknown dtype %d", dtype);
  if (tokens < 0 || dim <= 0 || dim > (int64_t{1} << 30) || q == nullptr || k == nullptr ||
      q->heads < 0 || k->heads < 0)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "rotary: invalid sizes");
  if (axes < 1 || axes > BYSJ_ROTARY_MAX_AXES || sections == nullptr)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "rotary: 1 to %d axes", BYSJ_ROTARY_MAX_AXES);
  if (grad_positions != nullptr && (!inverse || integer_positions))
    return fail(BYSJ_ERR_INVALID_ARGUMENT,
                "rotary: a position gradient needs the inverse rotation and float positions");
  RotaryArgs a{};
  int64_t pairs = 0;
  for (int i = 0; i < BYSJ_ROTARY_MAX_AXES; ++i) {
    if (i < axes) {
      if (sections[i] < 0 || sections[i] > dim)
        return fail(BYSJ_ERR_INVALID_ARGUMENT, "rotary: invalid section");
      pairs += sections[i];
    }
    a.end[i] = static_cast<int>(pairs);
  }
  if (2 * pairs > dim)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "rotary: the sections hold more pairs than dim / 2");
  if (tokens == 0 || q->heads + k->heads == 0) {
    if (grad_positions != nullptr && tokens > 0)
      return cuda_check(cudaMemsetAsync(grad_positions, 0, sizeof(float) * tokens * axes,
                                        static_cast<cudaStream_t>(stream)),
                        "rotary: zero grad_positions");
    return BYSJ_OK;
  }
  if (positions == nullptr || (pairs > 0 && inv_freq == nullptr))
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "rotary: NULL pointer");
  for (const bysj_rotary_side* side : {q, k})
    if (side->heads > 0 && (side->x == nullptr || side->y == nullptr ||
                            (grad_positions != nullptr && side->saved == nullptr)))
      return fail(BYSJ_ERR_INVALID_ARGUMENT, "rotary: NULL pointer");
  a.side[0] = *q;
  a.side[1] = *k;
  a.positions = positions;
  a.integer_positions = integer_positions;
  a.inv_freq = inv_freq;
  a.axes = axes;
  a.pairs = static_cast<int>(pairs);
  a.tokens = tokens;
  a.dim = dim;
  a.interleaved = interleaved;
  a.sign = inverse ? -1.0f : 1.0f;
  a.grad_positions = grad_positions;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int64_t blocks = (tokens + kWarpsPerBlock - 1) / kWarpsPerBlock;
  const int64_t cap = static_cast<int64_t>(current_device_info().sm_count) * 16;
  if (blocks > cap) blocks = cap;
  const auto kernel = dtype == BYSJ_F32
                          ? (grad_positions ? rotary_kernel<float, true>
                                            : rotary_kernel<float, false>)
                          : (grad_positions ? rotary_kernel<__nv_bfloat16, true>
                                            : rotary_kernel<__nv_bfloat16, false>);
  kernel<<<static_cast<unsigned>(blocks), kBlock, 0, s>>>(a);
  return launch_check("rotary_kernel");
}
