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
// A CTA takes a few tokens at a time.  It evaluates sine and cosine of each
// (token, pair) once into shared memory; then a thread holds the 8 (bfloat16)
// or 4 (float32) pairs of one 16-byte vector in registers and turns them in
// every HS-th head of q and k, four heads requested at a time.  Consecutive
// threads take consecutive vectors, then consecutive heads, so a warp reads and
// writes whole lines.  98304 tokens of 16 + 4 heads of 64 bfloat16 channels (506 MB)
// take 105 us, 0.73 of the measured copy bandwidth: a CTA's loads begin after its
// angles and a barrier, so neither HBM (54 % of its peak) nor issue (49 %) is full.
// Angles evaluated by each lane for its own pairs took 178 us; a
// fourth CTA on an SM, with half the loads in flight for each thread, 114 us.
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
  // a CTA's tile: tokens and pairs, and threads side by side
  int tile_tokens, tile_pairs, heads_abreast, vectors_abreast;
};

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

// The pairs that a thread turns in one head: VP pairs as loaded.
template <typename T, int VP, bool INTERLEAVED>
struct Pairs {
  RowVec<T, VP> a, b;  // channels p .. and pairs + p .., or 2 p .. and on
  __device__ __forceinline__ void load(const T* head, int p, int pairs) {
    if constexpr (INTERLEAVED) {
      a.load(head + 2 * p, 0);
      b.load(head + 2 * p + VP, 0);
    } else {
      a.load(head + p, 0);
      b.load(head + pairs + p, 0);
    }
  }
  __device__ __forceinline__ float first(int i) const {
    if constexpr (INTERLEAVED && VP > 1) return i < VP / 2 ? a.get(2 * i) : b.get(2 * i - VP);
    else return a.get(i);
  }
  __device__ __forceinline__ float second(int i) const {
    if constexpr (INTERLEAVED && VP > 1)
      return i < VP / 2 ? a.get(2 * i + 1) : b.get(2 * i + 1 - VP);
    else return b.get(i);
  }
};

template <int VP>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[VP]) {
  if constexpr (VP == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else p[0] = v[0];
}
template <int VP>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[VP]) {
  if constexpr (VP == 8) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
  } else {
    p[0] = __float2bfloat16_rn(v[0]);
  }
}

template <typename T, int VP, bool INTERLEAVED>
__device__ __forceinline__ void store_pairs(T* head, int p, int pairs, const float (&y1)[VP],
                                            const float (&y2)[VP]) {
  if constexpr (!INTERLEAVED) {
    store_vec<VP>(head + p, y1);
    store_vec<VP>(head + pairs + p, y2);
  } else if constexpr (VP == 1) {
    store_vec<1>(head + 2 * p, y1);
    store_vec<1>(head + 2 * p + 1, y2);
  } else {
    float v[VP];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < VP / 2; ++i) {
        v[2 * i] = y1[half * VP / 2 + i];
        v[2 * i + 1] = y2[half * VP / 2 + i];
      }
      store_vec<VP>(head + 2 * p + half * VP, v);
    }
  }
}

// Shared memory: sine and cosine [2][tokens][tile pairs] (two tiles, so one
// barrier each), and with a position gradient the threads' angle gradients
// [tokens][heads side by side][tile pairs] and the axes' sums [tokens][4].
template <typename T, int VP, bool INTERLEAVED, bool POS_GRAD>
__global__ void __launch_bounds__(kBlock, 3) rotary_kernel(RotaryArgs a) {
  extern __shared__ __align__(16) float2 s_turn[];
  const int tile_pairs = a.tile_pairs, tt = a.tile_tokens, hs = a.heads_abreast;
  float* s_dtheta = reinterpret_cast<float*>(s_turn + 2 * tt * tile_pairs);
  float* s_axis = s_dtheta + tt * hs * tile_pairs;
  const int heads_q = static_cast<int>(a.side[0].heads);
  const int heads = heads_q + static_cast<int>(a.side[1].heads);
  // thread -> (token, first head, vector of pairs)
  const int vectors = a.vectors_abreast;
  const int vector = threadIdx.x % vectors, rest = threadIdx.x / vectors;
  const int h0 = rest % hs, tok = rest / hs;
  const int64_t token_tiles = (a.tokens + tt - 1) / tt;
  int buffer = 0;
  for (int64_t tile = blockIdx.x; tile < token_tiles; tile += gridDim.x) {
    const int64_t t0 = tile * tt;
    const int count = static_cast<int>(min(static_cast<int64_t>(tt), a.tokens - t0));
    if constexpr (POS_GRAD) {
      __syncthreads();
      for (int i = threadIdx.x; i < tt * BYSJ_ROTARY_MAX_AXES; i += kBlock) s_axis[i] = 0.0f;
    }
    for (int p0 = 0; p0 < a.pairs; p0 += tile_pairs) {
      const int np = min(tile_pairs, a.pairs - p0);
      float2* turn = s_turn + buffer * tt * tile_pairs;
      buffer ^= 1;
      for (int i = threadIdx.x; i < count * np; i += kBlock) {
        const int t = i / np, p = i - t * np;
        const float theta =
            position_of(a, t0 + t, axis_of(a, p0 + p)) * __ldg(a.inv_freq + p0 + p);
        float sine, cosine;
        sincosf(theta, &sine, &cosine);
        turn[t * tile_pairs + p] = make_float2(cosine, sine * a.sign);
      }
      __syncthreads();
      if (tok < count) {
        const int64_t t = t0 + tok;
        const int64_t stride_q = a.side[0].x_head_stride, stride_k = a.side[1].x_head_stride;
        const T* xq = static_cast<const T*>(a.side[0].x) + t * a.side[0].x_token_stride;
        const T* xk = static_cast<const T*>(a.side[1].x) + t * a.side[1].x_token_stride;
        T* yq = static_cast<T*>(a.side[0].y) + t * heads_q * a.dim;
        T* yk = static_cast<T*>(a.side[1].y) + t * (heads - heads_q) * a.dim;
        const T *sq = nullptr, *sk = nullptr;
        if constexpr (POS_GRAD) {
          sq = static_cast<const T*>(a.side[0].saved) + t * a.side[0].saved_token_stride;
          sk = static_cast<const T*>(a.side[1].saved) + t * a.side[1].saved_token_stride;
        }
        for (int v = vector; v * VP < np; v += vectors) {
          const int pl = v * VP, p = p0 + pl;
          float cosine[VP], sine[VP], dtheta[VP];
#pragma unroll
          for (int i = 0; i < VP; ++i) {
            const float2 q = turn[tok * tile_pairs + pl + i];
            cosine[i] = q.x;
            sine[i] = q.y;
            dtheta[i] = 0.0f;
          }
          using PairsT = Pairs<T, VP, INTERLEAVED>;
          auto finish = [&](const PairsT& x, const PairsT& saved, T* y) {
            float y1[VP], y2[VP];
#pragma unroll
            for (int i = 0; i < VP; ++i) {
              const float x1 = x.first(i), x2 = x.second(i);
              // spelled out, so that every variant of the kernel gives the same bits
              y1[i] = fmaf(x1, cosine[i], -__fmul_rn(x2, sine[i]));
              y2[i] = fmaf(x2, cosine[i], __fmul_rn(x1, sine[i]));
              if constexpr (POS_GRAD)
                dtheta[i] += y2[i] * saved.first(i) - y1[i] * saved.second(i);
            }
            store_pairs<T, VP, INTERLEAVED>(y, p, a.pairs, y1, y2);
          };
          // kAhead heads are requested before the first is turned
          constexpr int kAhead = POS_GRAD ? 2 : 4;
          for (int h = h0; h < heads; h += kAhead * hs) {
            PairsT x[kAhead], saved[POS_GRAD ? kAhead : 1];
            T* y[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
              const int head = h + j * hs;
              if (head >= heads) continue;
              const bool k = head >= heads_q;
              const int at = k ? head - heads_q : head;
              x[j].load((k ? xk : xq) + at * (k ? stride_k : stride_q), p, a.pairs);
              y[j] = (k ? yk : yq) + at * a.dim;
              if constexpr (POS_GRAD)
                saved[j].load((k ? sk : sq) + at * (k ? a.side[1].saved_head_stride
                                                      : a.side[0].saved_head_stride),
                              p, a.pairs);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
              if (h + j * hs < heads) finish(x[j], saved[POS_GRAD ? j : 0], y[j]);
          }
          if constexpr (POS_GRAD)
#pragma unroll
            for (int i = 0; i < VP; ++i)
              s_dtheta[(tok * hs + h0) * tile_pairs + pl + i] = dtheta[i];
        }
      }
      if constexpr (POS_GRAD) {
        __syncthreads();
        // a warp joins a token's heads and pairs, in their order
        for (int t = threadIdx.x / kWarp; t < count; t += kWarpsPerBlock) {
          float sums[BYSJ_ROTARY_MAX_AXES] = {0.0f, 0.0f, 0.0f, 0.0f};
          for (int p = lane_id(); p < np; p += kWarp) {
            float d = 0.0f;
            for (int h = 0; h < hs; ++h) d += s_dtheta[(t * hs + h) * tile_pairs + p];
            d *= __ldg(a.inv_freq + p0 + p);
            const int axis = axis_of(a, p0 + p);
#pragma unroll
            for (int i = 0; i < BYSJ_ROTARY_MAX_AXES; ++i)
              if (i == axis) sums[i] += d;
          }
#pragma unroll
          for (int i = 0; i < BYSJ_ROTARY_MAX_AXES; ++i) {
            const float total = xor_sum(sums[i], 1);
            if (lane_id() == 0) s_axis[t * BYSJ_ROTARY_MAX_AXES + i] += total;
          }
        }
        __syncthreads();
      }
    }
    if constexpr (POS_GRAD) {
      __syncthreads();
      for (int i = threadIdx.x; i < count * a.axes; i += kBlock) {
        const int t = i / a.axes, axis = i - t * a.axes;
        a.grad_positions[(t0 + t) * a.axes + axis] = s_axis[t * BYSJ_ROTARY_MAX_AXES + axis];
      }
    }
    // channels without an angle
    const int tail = static_cast<int>(a.dim) - 2 * a.pairs;
    if (tail > 0)
      for (int64_t i = threadIdx.x; i < static_cast<int64_t>(count) * heads * tail; i += kBlock) {
        const int c = 2 * a.pairs + static_cast<int>(i % tail);
        const int h = static_cast<int>(i / tail % heads);
        const int64_t t = t0 + i / tail / heads;
        const bysj_rotary_side& side = a.side[h >= heads_q ? 1 : 0];
        const int64_t at = h >= heads_q ? h - heads_q : h;
        static_cast<T*>(side.y)[(t * side.heads + at) * a.dim + c] =
            static_cast<const T*>(side.x)[t * side.x_token_stride + at * side.x_head_stride + c];
      }
  }
}

using RotaryKernel = void (*)(RotaryArgs);

template <typename T, int VP>
RotaryKernel rotary_pick(bool interleaved, bool pos_grad) {
  if (interleaved)
    return pos_grad ? rotary_kernel<T, VP, true, true> : rotary_kernel<T, VP, true, false>;
  return pos_grad ? rotary_kernel<T, VP, false, true> : rotary_kernel<T, VP, false, false>;
}

// Whole 16-byte vectors of every head are aligned.
bool side_aligned(const bysj_rotary_side& side, int64_t dim, int64_t vec, bool saved) {
  if (side.heads == 0) return true;
  bool ok = aligned16(side.x) && aligned16(side.y) && dim % vec == 0 &&
            side.x_token_stride % vec == 0 && side.x_head_stride % vec == 0;
  if (saved)
    ok = ok && aligned16(side.saved) && side.saved_token_stride % vec == 0 &&
         side.saved_head_stride % vec == 0;
  return ok;
}

// Tiles: up to 256 pairs; threads over the vectors of a tile, then over heads
// (up to 64 threads, so that a request covers lines of several heads), then over
// tokens.  Of the numbers of heads side by side the one that leaves the fewest
// threads without work.
size_t plan_tiles(RotaryArgs& a, int vp, bool pos_grad) {
  const int heads = static_cast<int>(a.side[0].heads + a.side[1].heads);
  a.tile_pairs = a.pairs < 1 ? 1 : a.pairs < 256 ? a.pairs : 256;
  a.vectors_abreast = (a.tile_pairs + vp - 1) / vp;
  const int want = 64 / a.vectors_abreast < 1 ? 1 : 64 / a.vectors_abreast;
  double best = 0.0;
  for (int hs = heads < want ? heads : want; hs >= 1; --hs) {
    const int tokens = kBlock / (a.vectors_abreast * hs), rounds = (heads + hs - 1) / hs;
    const double busy = static_cast<double>(tokens) * a.vectors_abreast * heads / rounds;
    if (busy > best * 1.01) {
      best = busy;
      a.heads_abreast = hs;
      a.tile_tokens = tokens;
    }
  }
  const size_t turn = sizeof(float2) * 2 * a.tile_tokens * a.tile_pairs;
  if (!pos_grad) return turn;
  return turn + sizeof(float) * a.tile_tokens *
                    (a.heads_abreast * a.tile_pairs + BYSJ_ROTARY_MAX_AXES);
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
  if (tokens < 0 || dim <= 0 || dim > (int64_t{1} << 20) || q == nullptr || k == nullptr ||
      q->heads < 0 || k->heads < 0 || q->heads + k->heads > (int64_t{1} << 20))
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
  const int64_t vec = dtype == BYSJ_F32 ? 4 : 8;
  const bool pos_grad = grad_positions != nullptr;
  const bool vectors = pairs > 0 && pairs % vec == 0 && side_aligned(*q, dim, vec, pos_grad) &&
                       side_aligned(*k, dim, vec, pos_grad);
  const size_t smem = plan_tiles(a, vectors ? static_cast<int>(vec) : 1, pos_grad);
  const RotaryKernel kernel =
      dtype == BYSJ_F32 ? (vectors ? rotary_pick<float, 4>(interleaved, pos_grad)
                                   : rotary_pick<float, 1>(interleaved, pos_grad))
                        : (vectors ? rotary_pick<__nv_bfloat16, 8>(interleaved, pos_grad)
                                   : rotary_pick<__nv_bfloat16, 1>(interleaved, pos_grad));
  const int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (st) return st;
  int64_t blocks = (tokens + a.tile_tokens - 1) / a.tile_tokens;
  const int64_t cap = static_cast<int64_t>(current_device_info().sm_count) *
                      resident_blocks(reinterpret_cast<const void*>(kernel), smem);
  if (blocks > cap) blocks = cap;
  kernel<<<static_cast<unsigned>(blocks), kBlock, smem, s>>>(a);
  return launch_check("rotary_kernel");
}
