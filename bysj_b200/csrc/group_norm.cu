// Group norm over frames with an activation, channels last, for sm_100a.
//
//   z = (x - mean[b, g]) rstd[b, g] w[c] + b[c],  y = act(z)
//   dz = dy act'(z), d = dz w
//   dx = rstd (d - mean(d) - xhat mean(d xhat)),  dw = sum dz xhat,  db = sum dz
//
// The rows of all frames are cut into chunks of equal length, whatever the
// frames' lengths; the part of a frame inside a chunk is a piece.  Pieces are
// numbered chunk + frame, which is unique because going from one piece to the
// next advances at least one of the two.  A first kernel leaves two numbers
// per piece and channel (mean and centred square sum; in the backward pass
// sum dz and sum dz xhat, from which the group's sums and the gradients of
// weight and bias both follow), a second joins the pieces of each frame in
// their order, a third writes the result.  No atomics: results repeat bit
// for bit.
#include "launch.cuh"

namespace bysj {
namespace {

struct Frames {
  const int64_t* offsets;  // NULL: equal frames
  int64_t count, inner, rows;
  // First row of frame b (b == count: all rows).  Offsets are clamped to the
  // tensor, so a wrong prefix sum gives wrong numbers, not a wild access.
  __device__ __forceinline__ int64_t begin(int64_t b) const {
    if (offsets == nullptr) return b * (rows / count);
    int64_t r = __ldg(offsets + b) * inner;
    r = r < 0 ? 0 : r;
    return r > rows ? rows : r;
  }
  // Last frame that begins at or before row r.
  __device__ __forceinline__ int64_t of_row(int64_t r) const {
    if (offsets == nullptr) return r / (rows / count);
    int64_t lo = 0, hi = count - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) >> 1;
      if (begin(mid) <= r) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

struct GroupArgs {
  const void* x;
  const void* grad_out;
  void* out;
  Frames frames;
  int64_t channels, groups, group_channels;
  int64_t chunk_rows, chunks;
  const float* weight;
  const float* bias;
  float* mean;
  float* rstd;
  float eps;
  int activation;
  float2* partial;  // [chunks + frames][channels]
  float2* sums;     // [frames][groups]: mean(d), mean(d xhat)
  float* grad_weight;
  float* grad_bias;
};

__device__ __forceinline__ float load_f32(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float activate(float z, int activation) {
  if (activation == BYSJ_ACT_NONE) return z;
  const float s = 1.0f / (1.0f + expf(-z));
  return activation == BYSJ_ACT_SILU ? z * s : s;
}

__device__ __forceinline__ float activate_grad(float z, int activation) {
  if (activation == BYSJ_ACT_NONE) return 1.0f;
  const float s = 1.0f / (1.0f + expf(-z));
  return activation == BYSJ_ACT_SILU ? s * (1.0f + z * (1.0f - s)) : s * (1.0f - s);
}

// Threads of a CTA: `tx` channels side by side, `ty` rows at a time.
struct Tile {
  int tx, ty, cx, ry;
  __device__ explicit Tile(int64_t channels) {
    tx = channels < kBlock ? static_cast<int>(channels) : kBlock;
    ty = kBlock / tx;
    cx = threadIdx.x % tx;
    ry = threadIdx.x / tx;
  }
};

// Sum over the CTA's rows of one channel column; the total is returned to the
// threads of row 0.
__device__ __forceinline__ double column_sum(double v, const Tile& t, double* scratch) {
  __syncthreads();
  if (t.ry < t.ty) scratch[t.ry * t.tx + t.cx] = v;
  __syncthreads();
  double total = 0.0;
  if (t.ry == 0)
    for (int i = 0; i < t.ty; ++i) total += scratch[i * t.tx + t.cx];
  return total;
}

// Per piece and channel: forward, the mean and the sum of squares about it;
// backward, sum dz and sum dz xhat.
template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(kBlock) group_partial_kernel(GroupArgs a) {
  __shared__ double scratch[kBlock];
  const Tile t(a.channels);
  const int64_t chunk = blockIdx.x;
  const int64_t r0 = chunk * a.chunk_rows;
  const int64_t r1 = min(r0 + a.chunk_rows, a.frames.rows);
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.grad_out);
  int64_t lo = r0;
  for (int64_t b = a.frames.of_row(r0); b < a.frames.count && lo < r1; ++b) {
    const int64_t hi = min(a.frames.begin(b + 1), r1);
    if (hi <= lo) continue;
    for (int64_t c0 = 0; c0 < a.channels; c0 += t.tx) {
      const int64_t c = c0 + t.cx;
      const bool on = t.ry < t.ty && c < a.channels;
      double s1 = 0.0, s2 = 0.0;
      float pivot = 0.0f;
      if (on) {
        if constexpr (BACKWARD) {
          const int64_t g = c / a.group_channels;
          const float mean = a.mean[b * a.groups + g], rstd = a.rstd[b * a.groups + g];
          const float w = a.weight ? a.weight[c] : 1.0f, bias = a.bias ? a.bias[c] : 0.0f;
          for (int64_t r = lo + t.ry; r < hi; r += t.ty) {
            const float xhat = (load_f32(x + r * a.channels + c) - mean) * rstd;
            const float dz = load_f32(dy + r * a.channels + c) *
                             activate_grad(xhat * w + bias, a.activation);
            s1 += dz;
            s2 += static_cast<double>(dz * xhat);
          }
        } else {
          // squares about a value of the piece, not about 0: a mean far from
          // 0 takes no digits from the variance
          pivot = load_f32(x + lo * a.channels + c);
          for (int64_t r = lo + t.ry; r < hi; r += t.ty) {
            const float d = load_f32(x + r * a.channels + c) - pivot;
            s1 += d;
            s2 += static_cast<double>(d * d);
          }
        }
      }
      s1 = column_sum(s1, t, scratch);
      s2 = column_sum(s2, t, scratch);
      if (on && t.ry == 0) {
        float2 v;
        if constexpr (BACKWARD) {
          v = make_float2(static_cast<float>(s1), static_cast<float>(s2));
        } else {
          const double n = static_cast<double>(hi - lo);
          v = make_float2(static_cast<float>(pivot + s1 / n),
                          static_cast<float>(s2 - s1 * s1 / n));
        }
        a.partial[(chunk + b) * a.channels + c] = v;
      }
    }
    lo = hi;
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

// Joins the pieces of frame blockIdx.x for group blockIdx.y.
template <bool BACKWARD>
__global__ void __launch_bounds__(kBlock) group_join_kernel(GroupArgs a) {
  __shared__ double scratch[kWarpsPerBlock];
  const int64_t b = blockIdx.x;
  const int64_t r0 = a.frames.begin(b), r1 = a.frames.begin(b + 1);
  const double n = static_cast<double>(r1 - r0) * static_cast<double>(a.group_channels);
  for (int64_t g = blockIdx.y; g < a.groups; g += gridDim.y) {
    if (r1 <= r0) {
      if (threadIdx.x == 0) {
        if constexpr (BACKWARD) {
          a.sums[b * a.groups + g] = make_float2(0.0f, 0.0f);
        } else {
          a.mean[b * a.groups + g] = 0.0f;
          a.rstd[b * a.groups + g] = 0.0f;
        }
      }
      continue;
    }
    const int64_t first = r0 / a.chunk_rows, last = (r1 - 1) / a.chunk_rows;
    const int64_t items = (last - first + 1) * a.group_channels;
    double s1 = 0.0, s2 = 0.0;
    for (int64_t i = threadIdx.x; i < items; i += kBlock) {
      const int64_t chunk = first + i / a.group_channels;
      const int64_t c = g * a.group_channels + i % a.group_channels;
      const float2 v = a.partial[(chunk + b) * a.channels + c];
      if constexpr (BACKWARD) {
        const double w = a.weight ? a.weight[c] : 1.0;
        s1 += w * v.x;
        s2 += w * v.y;
      } else {
        const int64_t begin = max(chunk * a.chunk_rows, r0);
        const int64_t end = min((chunk + 1) * a.chunk_rows, r1);
        s1 += static_cast<double>(end - begin) * v.x;
      }
    }
    const double mean = block_sum(s1, scratch) / n;
    if constexpr (BACKWARD) {
      s2 = block_sum(s2, scratch) / n;
      if (threadIdx.x == 0)
        a.sums[b * a.groups + g] =
            make_float2(static_cast<float>(mean), static_cast<float>(s2));
    } else {
      for (int64_t i = threadIdx.x; i < items; i += kBlock) {
        const int64_t chunk = first + i / a.group_channels;
        const int64_t c = g * a.group_channels + i % a.group_channels;
        const float2 v = a.partial[(chunk + b) * a.channels + c];
        const int64_t begin = max(chunk * a.chunk_rows, r0);
        const int64_t end = min((chunk + 1) * a.chunk_rows, r1);
        const double d = v.x - mean;
        s2 += v.y + static_cast<double>(end - begin) * d * d;
      }
      s2 = block_sum(s2, scratch) / n;
      if (threadIdx.x == 0) {
        a.mean[b * a.groups + g] = static_cast<float>(mean);
        a.rstd[b * a.groups + g] = static_cast<float>(1.0 / sqrt(s2 + a.eps));
      }
    }
  }
}

template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(kBlock) group_apply_kernel(GroupArgs a) {
  const Tile t(a.channels);
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.chunk_rows;
  const int64_t r1 = min(r0 + a.chunk_rows, a.frames.rows);
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.grad_out);
  T* out = static_cast<T*>(a.out);
  int64_t lo = r0;
  for (int64_t b = a.frames.of_row(r0); b < a.frames.count && lo < r1; ++b) {
    const int64_t hi = min(a.frames.begin(b + 1), r1);
    if (hi <= lo) continue;
    for (int64_t c = t.cx; c < a.channels && t.ry < t.ty; c += t.tx) {
      const int64_t g = c / a.group_channels;
      const float mean = a.mean[b * a.groups + g], rstd = a.rstd[b * a.groups + g];
      const float w = a.weight ? a.weight[c] : 1.0f, bias = a.bias ? a.bias[c] : 0.0f;
      float2 sums = make_float2(0.0f, 0.0f);
      if constexpr (BACKWARD) sums = a.sums[b * a.groups + g];
      for (int64_t r = lo + t.ry; r < hi; r += t.ty) {
        const int64_t i = r * a.channels + c;
        const float xhat = (load_f32(x + i) - mean) * rstd;
        const float z = xhat * w + bias;
        if constexpr (BACKWARD) {
          const float d = load_f32(dy + i) * activate_grad(z, a.activation) * w;
          store_value(out + i, rstd * (d - sums.x - xhat * sums.y));
        } else {
          store_value(out + i, activate(z, a.activation));
        }
      }
    }
    lo = hi;
  }
}

// grad_weight and grad_bias: the pieces of all frames, channel by channel.
__global__ void __launch_bounds__(kBlock) group_affine_grad_kernel(GroupArgs a) {
  __shared__ double scratch[kWarpsPerBlock];
  const int64_t c = blockIdx.x;
  double s1 = 0.0, s2 = 0.0;
  for (int64_t chunk = threadIdx.x; chunk < a.chunks; chunk += kBlock) {
    const int64_t r0 = chunk * a.chunk_rows;
    const int64_t r1 = min(r0 + a.chunk_rows, a.frames.rows);
    int64_t lo = r0;
    for (int64_t b = a.frames.of_row(r0); b < a.frames.count && lo < r1; ++b) {
      const int64_t hi = min(a.frames.begin(b + 1), r1);
      if (hi <= lo) continue;
      const float2 v = a.partial[(chunk + b) * a.channels + c];
      s1 += v.x;
      s2 += v.y;
      lo = hi;
    }
  }
  s1 = block_sum(s1, scratch);
  s2 = block_sum(s2, scratch);
  if (threadIdx.x == 0) {
    if (a.grad_bias) a.grad_bias[c] = static_cast<float>(s1);
    if (a.grad_weight) a.grad_weight[c] = static_cast<float>(s2);
  }
}

// Rows of a chunk: about four chunks for each SM, 16 to 512 rows.
int64_t chunk_rows_of(int64_t rows) {
  const int64_t want = rows / (static_cast<int64_t>(current_device_info().sm_count) * 4);
  return want < 16 ? 16 : want > 512 ? 512 : want;
}

size_t carve_workspace(GroupArgs& a, void* workspace, bool backward) {
  Carver carve(workspace);
  a.partial = carve.take<float2>(static_cast<size_t>(a.chunks + a.frames.count) * a.channels);
  if (backward) a.sums = carve.take<float2>(static_cast<size_t>(a.frames.count) * a.groups);
  return carve.need;
}

void plan(GroupArgs& a, int64_t rows, int64_t channels, int64_t groups, int64_t frames) {
  a.frames.rows = rows;
  a.frames.count = frames;
  a.channels = channels;
  a.groups = groups;
  a.group_channels = channels / groups;
  a.chunk_rows = chunk_rows_of(rows);
  a.chunks = (rows + a.chunk_rows - 1) / a.chunk_rows;
}

size_t workspace_size(int64_t rows, int64_t channels, int64_t groups, int64_t frames,
                      bool backward) {
  if (rows <= 0 || channels <= 0 || groups <= 0 || frames <= 0) return 0;
  GroupArgs a{};
  plan(a, rows, channels, groups, frames);
  return carve_workspace(a, nullptr, backward);
}

int check_shape(const char* name, int dtype, int64_t rows, int64_t channels, int64_t groups,
                const int64_t* offsets, int64_t frames, int64_t inner, int activation) {
  if (dtype != BYSJ_F32 && dtype != BYSJ_BF16)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", name, dtype);
  if (rows < 0 || channels <= 0 || groups <= 0 || channels % groups != 0 || frames < 0)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "%s: invalid sizes", name);
  if (offsets != nullptr && inner < 1)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "%s: inner must be positive", name);
  if (offsets == nullptr && frames > 0 && rows % frames != 0)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "%s: rows must be a multiple of frames", name);
  if (rows > 0 && frames == 0)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "%s: rows without a frame", name);
  if (activation != BYSJ_ACT_NONE && activation != BYSJ_ACT_SILU &&
      activation != BYSJ_ACT_SIGMOID)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", name, activation);
  if (frames > 0x7fffffff)
    return fail(BYSJ_ERR_TOO_LARGE, "%s: more than 2^31 - 1 frames", name);
  return BYSJ_OK;
}

template <typename T, bool BACKWARD>
int launch(const GroupArgs& a, cudaStream_t s) {
  const unsigned chunks = static_cast<unsigned>(a.chunks);
  const dim3 joins(static_cast<unsigned>(a.frames.count),
                   static_cast<unsigned>(a.groups < 65535 ? a.groups : 65535));
  group_partial_kernel<T, BACKWARD><<<chunks, kBlock, 0, s>>>(a);
  int st = launch_check("group_partial_kernel");
  if (st) return st;
  group_join_kernel<BACKWARD><<<joins, kBlock, 0, s>>>(a);
  st = launch_check("group_join_kernel");
  if (st) return st;
  group_apply_kernel<T, BACKWARD><<<chunks, kBlock, 0, s>>>(a);
  return launch_check("group_apply_kernel");
}

}  // namespace
}  // namespace bysj

using namespace bysj;

extern "C" {

size_t bysj_group_norm_forward_workspace_size(int64_t rows, int64_t channels, int64_t groups,
                                              int64_t frames) {
  return workspace_size(rows, channels, groups, frames, false);
}

size_t bysj_group_norm_backward_workspace_size(int64_t rows, int64_t channels, int64_t groups,
                                               int64_t frames) {
  return workspace_size(rows, channels, groups, frames, true);
}

int bysj_group_norm_forward(const void* x, int dtype, int64_t rows, int64_t channels,
                            int64_t groups, const int64_t* offsets, int64_t frames,
                            int64_t inner, const float* weight, const float* bias, float eps,
                            int activation, void* y, float* mean, float* rstd, void* workspace,
                            size_t workspace_bytes, void* stream) {
  clear_error();
  const int st = check_shape("group norm", dtype, rows, channels, groups, offsets, frames, inner,
                             activation);
  if (st) return st;
  if (!(eps > 0.0f)) return fail(BYSJ_ERR_INVALID_ARGUMENT, "group norm: eps must be positive");
  if (frames == 0) return BYSJ_OK;
  if (mean == nullptr || rstd == nullptr)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "group norm: NULL statistics");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    const size_t bytes = sizeof(float) * static_cast<size_t>(frames) * groups;
    const int zero = cuda_check(cudaMemsetAsync(mean, 0, bytes, s), "group norm: zero mean");
    return zero ? zero : cuda_check(cudaMemsetAsync(rstd, 0, bytes, s), "group norm: zero rstd");
  }
  if (x == nullptr || y == nullptr)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "group norm: NULL pointer");
  GroupArgs a{};
  plan(a, rows, channels, groups, frames);
  const size_t need = carve_workspace(a, workspace, false);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(BYSJ_ERR_WORKSPACE, "group norm: workspace of %zu bytes needed, %zu given", need,
                workspace_bytes);
  a.frames.offsets = offsets;
  a.frames.inner = inner;
  a.x = x;
  a.out = y;
  a.weight = weight;
  a.bias = bias;
  a.mean = mean;
  a.rstd = rstd;
  a.eps = eps;
  a.activation = activation;
  return dtype == BYSJ_F32 ? launch<float, false>(a, s) : launch<__nv_bfloat16, false>(a, s);
}

int bysj_group_norm_backward(const void* grad_out, const void* x, int dtype, int64_t rows,
                             int64_t channels, int64_t groups, const int64_t* offsets,
                             int64_t frames, int64_t inner, const float* weight,
                             const float* bias, const float* mean, const float* rstd,
                             int activation, void* grad_x, float* grad_weight, float* grad_bias,
                             void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int st = check_shape("group norm backward", dtype, rows, channels, groups, offsets, frames,
                       inner, activation);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    for (float* grad : {grad_weight, grad_bias})
      if (grad != nullptr && st == BYSJ_OK)
        st = cuda_check(cudaMemsetAsync(grad, 0, sizeof(float) * channels, s),
                        "group norm backward: zero gradients");
    return st;
  }
  if (grad_out == nullptr || x == nullptr || grad_x == nullptr || mean == nullptr ||
      rstd == nullptr)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "group norm backward: NULL pointer");
  GroupArgs a{};
  plan(a, rows, channels, groups, frames);
  const size_t need = carve_workspace(a, workspace, true);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(BYSJ_ERR_WORKSPACE,
                "group norm backward: workspace of %zu bytes needed, %zu given", need,
                workspace_bytes);
  a.frames.offsets = offsets;
  a.frames.inner = inner;
  a.x = x;
  a.grad_out = grad_out;
  a.out = grad_x;
  a.weight = weight;
  a.bias = bias;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.activation = activation;
  a.grad_weight = grad_weight;
  a.grad_bias = grad_bias;
  st = dtype == BYSJ_F32 ? launch<float, true>(a, s) : launch<__nv_bfloat16, true>(a, s);
  if (st || (grad_weight == nullptr && grad_bias == nullptr)) return st;
  group_affine_grad_kernel<<<static_cast<unsigned>(channels), kBlock, 0, s>>>(a);
  return launch_check("group_affine_grad_kernel");
}

}  // extern "C"
