// One AdamW step over many tensors for sm_100a, states in 32 or 8 bits.
//
//   m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
//   p = decay p - size m / (correct sqrt(v) + eps)
//
// Work is counted in blocks of 256 elements, the unit that shares one scale
// of an 8-bit state.  The tensor table travels in the kernel's parameters
// (no copy to the device); a warp finds the tensor of its block by a binary
// search and takes 8 elements per lane, four side by side twice, so that each
// array is read and written in whole lines (16 bytes a lane of float32, 8 of
// bfloat16, 4 of codes).  Every tensor's states begin at a block boundary of
// the shared state buffers, so the table holds no state pointers and their
// loads are always aligned; a parameter or gradient that is not, and a tensor's
// last block, goes element by element.
//
// Each product and sum is rounded to fp32 on its own (no fused
// multiply-add), so a step gives the same bits as the formula evaluated one
// operation at a time.
//
// 104.7 M float32 parameters, 32-bit states: 443 us, 28 B an element at the
// measured copy bandwidth (448 us).  39.5 M bfloat16 parameters with masters and
// 8-bit states: 160 us (16 B an element, 97 us at that bandwidth), bound by issue:
// about 100 lane operations an element, of which the correctly rounded root and
// quotient are a good part.  Random rounding adds 39 us for sqrt(v), 41 us for both:
// an eighth more instructions, and registers for three CTAs on an SM instead of
// four.  Values of 8-bit states: 75 us (10 B, 60 us).
//
// 8-bit states.  m keeps a sign and a 7-bit magnitude with 3 mantissa bits
// (a relative rounding of at most 1/16 down to 2^-16 of the block's
// largest); sqrt(v) an 8-bit code with 4 mantissa bits (1/32).  The step
// divides by sqrt(v), so its root is what is kept: 2^-16 there spans 2^-32 of
// v.  A positive v never becomes 0: its code is at least 1, so no rounding makes
// a step divide by eps alone.  The scale is the block's largest magnitude itself
// and value(top) = 1, so that element is kept exactly, and a decay by beta of the
// whole block is carried by the scale.
//
// A step takes at most 1 - beta1 off m and (1 - beta2) / 2 off sqrt(v).  Where
// that is less than half the gap between two codes, an element whose gradients
// change beside others that do not would stay at its code for ever if it were
// rounded to the nearest.  Such a moment is rounded at random instead, up with the
// probability that keeps its mean: the code's bits plus a uniform number of one
// unit, cut.  Random words come from a counter (the step and the element), so a
// step repeats and resumes bit for bit.  m: where 1 - beta1 < 1/16 (half a gap is
// up to 1/18 of m).  sqrt(v): where 1 - beta2 < 1/64; 6000 steps of random
// gradients, half a block's changed by 0.1 or 4 after 2000, give sqrt(v) beside
// 32-bit states within 0.84 .. 1.23 (nearest) and 0.73 .. 1.29 (random) at beta2 =
// 0.97, 0.84 .. 1.24 and 0.74 .. 1.40 at 0.98, up to 3.6 and 1.36 at 0.99, up to
// 9.7 and 2.2 at 0.999 (0.11 root mean square of its logarithm).
#include "launch.cuh"

namespace bysj {
namespace {

constexpr int kStateBlock = BYSJ_ADAMW_BLOCK;
constexpr int kPerLane = kStateBlock / kWarp;
constexpr int kTopM = 127, kMantM = 3;
constexpr int kTopV = 255, kMantV = 4;

struct AdamEntry {
  void* param;
  const void* grad;
  int64_t n;
  int64_t state_block;  // first block in the state buffers
  int64_t work_block;   // first block of this launch's work list
};

template <int CAP>
struct AdamArgs {
  AdamEntry entry[CAP];
  int count;
  int64_t work_blocks;
  void* exp_avg;
  void* exp_avg_sq;
  float* exp_avg_scale;
  float* exp_avg_sq_scale;
  float* master;
  const float* grad_scale;
  bysj_adamw_hyper h;
  uint64_t counter;            // of the step, for random rounding
  bool random_m, random_v;     // round the moment's codes at random
};

// Kernel parameters hold 32,764 bytes; most models need far fewer entries and
// a shorter parameter block costs less to launch.
constexpr int kSmallTable = 96;
constexpr int kLargeTable = 800;

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

// The i-th of a lane's elements in its block.
__device__ __forceinline__ int element(int lane, int i) {
  return lane * 4 + i / 4 * 4 * kWarp + i % 4;
}
__device__ __forceinline__ void load4(const float* p, float* v) {
  const float4 q = *reinterpret_cast<const float4*>(p);
  v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float* v) {
  const uint2 q = *reinterpret_cast<const uint2*>(p);
  v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
}
__device__ __forceinline__ void store4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* v) {
  __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
}

// Byte j of a word moved to the bits above 23 - MANT of a float, cut by `mask`.
template <int MANT>
__device__ __forceinline__ unsigned byte_bits(unsigned word, int j, unsigned mask) {
  const int up = 23 - MANT - 8 * j;
  return (up >= 0 ? word << up : word >> -up) & mask;
}
template <int TOP, int MANT>
__device__ __forceinline__ float code_value(unsigned bits) {
  const float v = __uint_as_float(bits + (((127u << MANT) - TOP) << (23 - MANT)));
  return bits != 0 ? v : 0.0f;
}

// What byte j of a word of codes stands for.
__device__ __forceinline__ float value_m(unsigned word, int j, float scale) {
  const float size = __fmul_rn(
      code_value<kTopM, kMantM>(byte_bits<kMantM>(word, j, 127u << (23 - kMantM))), scale);
  const unsigned sign = (word << (24 - 8 * j)) & 0x80000000u;
  return __uint_as_float(__float_as_uint(size) | sign);
}
__device__ __forceinline__ float value_v(unsigned word, int j, float scale) {
  const float root = __fmul_rn(
      code_value<kTopV, kMantV>(byte_bits<kMantV>(word, j, 255u << (23 - kMantV))), scale);
  return __fmul_rn(root, root);
}

// How a ratio is rounded to a code: to nearest (ties to even), or at random by a
// 16-bit number, taken at the middle of its 2^-16.
struct Rounding {
  bool random;
  unsigned r;
  // Added below the last kept bit before the cut, in units of 2^-shift of it.
  template <int SHIFT>
  __device__ __forceinline__ unsigned addend(unsigned bits) const {
    const unsigned nearest = (1u << (SHIFT - 1)) - 1u + ((bits >> SHIFT) & 1u);
    return random ? (r << (SHIFT - 16)) | (1u << (SHIFT - 17)) : nearest;
  }
  // Part of the smallest code's value from which on a ratio below it takes it.
  __device__ __forceinline__ float threshold() const {
    return random ? static_cast<float>(131071u - 2u * r) * (1.0f / 131072.0f) : 0.5f;
  }
};

// Four random words for the elements 4 quad .. 4 quad + 3 at step `counter`:
// Philox 4x32 with seven rounds (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011).
__device__ __forceinline__ uint4 random_words(uint64_t quad, uint64_t counter) {
  uint4 c = make_uint4(static_cast<unsigned>(quad), static_cast<unsigned>(quad >> 32), 0u, 0u);
  unsigned k0 = static_cast<unsigned>(counter), k1 = static_cast<unsigned>(counter >> 32);
#pragma unroll
  for (int round = 0; round < 7; ++round) {
    const unsigned hi0 = __umulhi(0xd2511f53u, c.x), lo0 = 0xd2511f53u * c.x;
    const unsigned hi1 = __umulhi(0xcd9e8d57u, c.z), lo1 = 0xcd9e8d57u * c.z;
    c = make_uint4(hi1 ^ c.y ^ k0, lo1, hi0 ^ c.w ^ k1, lo0);
    k0 += 0x9e3779b9u;
    k1 += 0xbb67ae85u;
  }
  return c;
}

// Code of a ratio from the smallest code's value on: the bits of the float
// rounded to MANT mantissa bits, counted down from TOP.
template <int TOP, int MANT>
__device__ __forceinline__ unsigned ratio_code(float ratio, Rounding how) {
  constexpr int kShift = 23 - MANT;
  const unsigned bits = __float_as_uint(ratio);
  return ((bits + how.addend<kShift>(bits)) >> kShift) - ((127u << MANT) - TOP);
}

// Largest magnitude over the warp's block; for non-negative floats the order
// of the bits is the order of the values (NaN above all).
__device__ __forceinline__ float block_max(const float (&v)[kPerLane]) {
  unsigned best = 0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    best = max(best, static_cast<unsigned>(__float_as_int(v[i])) & 0x7fffffffu);
  return __uint_as_float(__reduce_max_sync(kFull, best));
}

__device__ __forceinline__ float inverse_scale(float scale) {
  return scale > 0.0f ? __frcp_rn(scale) : 0.0f;
}

// Ratios are at most 1 up to a rounding that the code drops, unless the scale
// is so small that its inverse is infinite: then every value but 0 takes the
// top code (0 times it is not a number and compares as below the least).  A block
// with a NaN or an infinity has it for its scale, and no finite value of any code.
constexpr float kLeastM = 1.25f / 65536.0f, kLeastV = 1.125f / 65536.0f;  // value(1)

// Below the smallest code's value: to it or to 0.
__device__ __forceinline__ unsigned encode_m(float m, float inv, Rounding how) {
  const float ratio = __fmul_rn(fabsf(m), inv);
  const unsigned code = ratio_code<kTopM, kMantM>(fminf(fmaxf(ratio, kLeastM), 1.0f), how);
  return (ratio >= how.threshold() * kLeastM ? code : 0u) | (m < 0.0f ? 128u : 0u);
}
__device__ __forceinline__ unsigned encode_v(float root, float inv, Rounding how) {
  const float ratio = fminf(__fmul_rn(root, inv), 1.0f);
  const unsigned code = ratio_code<kTopV, kMantV>(fmaxf(ratio, kLeastV), how);
  return root > 0.0f ? code : 0u;
}
__device__ __forceinline__ unsigned pack4(const unsigned (&c)[4]) {
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

// Resident CTAs: with 32-bit states three leave 80 registers a thread and four 64;
// three keep more of a lane's 16-byte loads in flight (104.7 M float32 parameters:
// 443 against 452 us).  The 8-bit step is bound by issue and wants the warps, at
// the price of 5 spilled registers (39.5 M bfloat16: 160 us with four, 181 with
// three).  With random numbers it needs 72 to 78 registers and takes three.
// RANDOM: a moment of the 8-bit states may be rounded at random.
template <typename T, int BITS, bool MASTER, int CAP, bool RANDOM>
__global__ void __launch_bounds__(kBlock, BITS == 8 && !RANDOM ? 4 : 3)
    adamw_kernel(const __grid_constant__ AdamArgs<CAP> a) {
  const int lane = lane_id();
  const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarpsPerBlock;
  const float scale = a.grad_scale != nullptr ? __ldg(a.grad_scale) : 1.0f;
  const bool scaled = a.grad_scale != nullptr;
  int lo = 0;  // last entry whose work_block <= work
  for (int64_t work = global_warp(); work < a.work_blocks; work += warps) {
    if (lo + 1 < a.count && a.entry[lo + 1].work_block <= work) {
      ++lo;
      int hi = a.count - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.entry[mid].work_block <= work) lo = mid;
        else hi = mid - 1;
      }
    }
    const int64_t local = work - a.entry[lo].work_block;
    const int64_t block = a.entry[lo].state_block + local;
    const int64_t begin = local * kStateBlock;
    const int64_t left = a.entry[lo].n - begin;
    T* param = static_cast<T*>(a.entry[lo].param) + begin;
    const T* grad = static_cast<const T*>(a.entry[lo].grad) + begin;
    const int64_t state = block * kStateBlock;
    float p[kPerLane], g[kPerLane], m[kPerLane], v[kPerLane];
    const bool whole = left >= kStateBlock &&
                       ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad)) &
                        (4 * sizeof(T) - 1)) == 0;
    if (whole) {
#pragma unroll
      for (int i = 0; i < kPerLane; i += 4) {
        load4(grad + element(lane, i), g + i);
        if constexpr (!MASTER) load4(param + element(lane, i), p + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int j = element(lane, i);
        g[i] = j < left ? load_f32(grad + j) : 0.0f;
        if constexpr (!MASTER) p[i] = j < left ? load_f32(param + j) : 0.0f;
      }
    }
    float scale_m = 0.0f, scale_v = 0.0f;
    if constexpr (BITS == 8) {
      scale_m = a.exp_avg_scale[block];
      scale_v = a.exp_avg_sq_scale[block];
    }
#pragma unroll
    for (int i = 0; i < kPerLane; i += 4) {
      const int64_t at = state + element(lane, i);
      if constexpr (MASTER) load4(a.master + at, p + i);
      if constexpr (BITS == 32) {
        load4(static_cast<const float*>(a.exp_avg) + at, m + i);
        load4(static_cast<const float*>(a.exp_avg_sq) + at, v + i);
      } else {
        const unsigned cm =
            *reinterpret_cast<const unsigned*>(static_cast<uint8_t*>(a.exp_avg) + at);
        const unsigned cv =
            *reinterpret_cast<const unsigned*>(static_cast<uint8_t*>(a.exp_avg_sq) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m[i + j] = value_m(cm, j, scale_m);
          v[i + j] = value_v(cv, j, scale_v);
        }
      }
    }
    float root[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const float gi = scaled ? __fmul_rn(g[i], scale) : g[i];
      m[i] = __fadd_rn(__fmul_rn(m[i], a.h.beta1), __fmul_rn(gi, a.h.one_minus_beta1));
      v[i] = __fadd_rn(__fmul_rn(v[i], a.h.beta2),
                       __fmul_rn(__fmul_rn(gi, a.h.one_minus_beta2), gi));
      root[i] = __fsqrt_rn(v[i]);
      const float den = __fadd_rn(__fmul_rn(root[i], a.h.correct), a.h.eps);
      p[i] = __fsub_rn(__fmul_rn(p[i], a.h.decay), __fmul_rn(__fdiv_rn(m[i], den), a.h.size));
    }
    if (whole) {
#pragma unroll
      for (int i = 0; i < kPerLane; i += 4) {
        store4(param + element(lane, i), p + i);
        if constexpr (MASTER) store4(a.master + state + element(lane, i), p + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int j = element(lane, i);
        if (j < left) {
          store_value(param + j, p[i]);
          if constexpr (MASTER) a.master[state + j] = p[i];
        }
      }
    }
    if constexpr (BITS == 32) {
#pragma unroll
      for (int i = 0; i < kPerLane; i += 4) {
        store4(static_cast<float*>(a.exp_avg) + state + element(lane, i), m + i);
        store4(static_cast<float*>(a.exp_avg_sq) + state + element(lane, i), v + i);
      }
    } else {
      const float sm = block_max(m), sv = block_max(root);
      const float im = inverse_scale(sm), iv = inverse_scale(sv);
#pragma unroll
      for (int i = 0; i < kPerLane; i += 4) {
        unsigned codes_m[4], codes_v[4];
        const int64_t at = state + element(lane, i);
        uint4 words = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (RANDOM) words = random_words(static_cast<uint64_t>(at) / 4, a.counter);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned word = j == 0 ? words.x : j == 1 ? words.y : j == 2 ? words.z : words.w;
          codes_m[j] = encode_m(m[i + j], im, {RANDOM && a.random_m, word & 0xffffu});
          codes_v[j] = encode_v(root[i + j], iv, {RANDOM && a.random_v, word >> 16});
        }
        *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(a.exp_avg) + at) = pack4(codes_m);
        *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(a.exp_avg_sq) + at) = pack4(codes_v);
      }
      if (lane == 0) {
        a.exp_avg_scale[block] = sm;
        a.exp_avg_sq_scale[block] = sv;
      }
    }
  }
}

// Four elements a lane, four times in steps of the grid.
__global__ void __launch_bounds__(kBlock)
    adamw_values_kernel(const uint8_t* exp_avg, const uint8_t* exp_avg_sq, const float* scale_m,
                        const float* scale_v, int64_t quads, float* out_m, float* out_v) {
  constexpr int kQuadsBlock = kStateBlock / 4, kUnroll = 4;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kBlock;
  for (int64_t q0 = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; q0 < quads;
       q0 += step * kUnroll) {
    unsigned cm[kUnroll], cv[kUnroll];
    float sm[kUnroll], sv[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t q = q0 + u * step;
      if (q >= quads) continue;
      cm[u] = reinterpret_cast<const unsigned*>(exp_avg)[q];
      cv[u] = reinterpret_cast<const unsigned*>(exp_avg_sq)[q];
      sm[u] = __ldg(scale_m + q / kQuadsBlock);
      sv[u] = __ldg(scale_v + q / kQuadsBlock);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t q = q0 + u * step;
      if (q >= quads) continue;
      float m[4], v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = value_m(cm[u], j, sm[u]);
        v[j] = value_v(cv[u], j, sv[u]);
      }
      store4(out_m + 4 * q, m);
      store4(out_v + 4 * q, v);
    }
  }
}

template <typename T, int BITS, bool MASTER, int CAP, bool RANDOM>
int launch_chunk(const bysj_adamw_tensor* tensors, int64_t count, AdamArgs<CAP>& a,
                 cudaStream_t s) {
  a.count = 0;
  a.work_blocks = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (tensors[i].n == 0) continue;
    AdamEntry& e = a.entry[a.count++];
    e.param = tensors[i].param;
    e.grad = tensors[i].grad;
    e.n = tensors[i].n;
    e.state_block = tensors[i].first_block;
    e.work_block = a.work_blocks;
    a.work_blocks += (tensors[i].n + kStateBlock - 1) / kStateBlock;
  }
  if (a.work_blocks == 0) return BYSJ_OK;
  int64_t blocks = (a.work_blocks + kWarpsPerBlock - 1) / kWarpsPerBlock;
  const int64_t cap = static_cast<int64_t>(current_device_info().sm_count) * 16;
  if (blocks > cap) blocks = cap;
  adamw_kernel<T, BITS, MASTER, CAP, RANDOM><<<static_cast<unsigned>(blocks), kBlock, 0, s>>>(a);
  return launch_check("adamw_kernel");
}

template <typename T, int BITS, bool MASTER, int CAP, bool RANDOM>
int launch_all(const bysj_adamw_tensor* tensors, int64_t count, const AdamArgs<1>& base,
               cudaStream_t s) {
  AdamArgs<CAP> a;
  a.exp_avg = base.exp_avg;
  a.exp_avg_sq = base.exp_avg_sq;
  a.exp_avg_scale = base.exp_avg_scale;
  a.exp_avg_sq_scale = base.exp_avg_sq_scale;
  a.master = base.master;
  a.grad_scale = base.grad_scale;
  a.h = base.h;
  a.counter = base.counter;
  a.random_m = base.random_m;
  a.random_v = base.random_v;
  for (int64_t at = 0; at < count; at += CAP) {
    const int64_t part = count - at < CAP ? count - at : CAP;
    const int st = launch_chunk<T, BITS, MASTER, CAP, RANDOM>(tensors + at, part, a, s);
    if (st != BYSJ_OK) return st;
  }
  return BYSJ_OK;
}

template <typename T, int BITS, bool RANDOM>
int launch_bits(const bysj_adamw_tensor* tensors, int64_t count, const AdamArgs<1>& base,
                cudaStream_t s) {
  const bool small = count <= kSmallTable;
  if (base.master != nullptr)
    return small ? launch_all<T, BITS, true, kSmallTable, RANDOM>(tensors, count, base, s)
                 : launch_all<T, BITS, true, kLargeTable, RANDOM>(tensors, count, base, s);
  return small ? launch_all<T, BITS, false, kSmallTable, RANDOM>(tensors, count, base, s)
               : launch_all<T, BITS, false, kLargeTable, RANDOM>(tensors, count, base, s);
}

template <typename T>
int launch_type(const bysj_adamw_tensor* tensors, int64_t count, int bits,
                const AdamArgs<1>& base, cudaStream_t s) {
  if (bits == 32) return launch_bits<T, 32, false>(tensors, count, base, s);
  return base.random_m || base.random_v ? launch_bits<T, 8, true>(tensors, count, base, s)
                                        : launch_bits<T, 8, false>(tensors, count, base, s);
}

// Moments of 8-bit states that a step moves by less than half a code.
constexpr float kSlowM = 1.0f / 16.0f, kSlowV = 1.0f / 64.0f;

int adamw_step(const bysj_adamw_tensor* tensors, int64_t n_tensors, int dtype, int state_bits,
               void* exp_avg, void* exp_avg_sq, float* exp_avg_scale, float* exp_avg_sq_scale,
               float* master, const float* grad_scale, const bysj_adamw_hyper* hyper,
               const uint64_t* counter, void* stream) {
  clear_error();
  if (dtype != BYSJ_F32 && dtype != BYSJ_BF16)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "adamw: unknown dtype %d", dtype);
  if (state_bits != 8 && state_bits != 32)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "adamw: states have 8 or 32 bits");
  if (n_tensors < 0 || (n_tensors > 0 && tensors == nullptr) || hyper == nullptr)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "adamw: no tensors or hyper parameters");
  int64_t elements = 0;
  for (int64_t i = 0; i < n_tensors; ++i) {
    if (tensors[i].n < 0 || tensors[i].first_block < 0)
      return fail(BYSJ_ERR_INVALID_ARGUMENT, "adamw: tensor %lld has an invalid size",
                  (long long)i);
    if (tensors[i].n > 0 && (tensors[i].param == nullptr || tensors[i].grad == nullptr))
      return fail(BYSJ_ERR_INVALID_ARGUMENT, "adamw: tensor %lld is NULL", (long long)i);
    elements += tensors[i].n;
  }
  if (elements == 0) return BYSJ_OK;
  if (exp_avg == nullptr || exp_avg_sq == nullptr ||
      (state_bits == 8 && (exp_avg_scale == nullptr || exp_avg_sq_scale == nullptr)))
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "adamw: NULL state");
  AdamArgs<1> base{};
  if (state_bits == 8) {
    base.random_m = hyper->one_minus_beta1 < kSlowM;
    base.random_v = hyper->one_minus_beta2 < kSlowV;
    if ((base.random_m || base.random_v) && counter == nullptr)
      return fail(BYSJ_ERR_INVALID_ARGUMENT,
                  "adamw: 8-bit states at these betas need bysj_adamw_step_counted");
  }
  if (counter != nullptr) base.counter = *counter;
  base.exp_avg = exp_avg;
  base.exp_avg_sq = exp_avg_sq;
  base.exp_avg_scale = exp_avg_scale;
  base.exp_avg_sq_scale = exp_avg_sq_scale;
  base.master = master;
  base.grad_scale = grad_scale;
  base.h = *hyper;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == BYSJ_F32 ? launch_type<float>(tensors, n_tensors, state_bits, base, s)
                           : launch_type<__nv_bfloat16>(tensors, n_tensors, state_bits, base, s);
}

}  // namespace
}  // namespace bysj

using namespace bysj;

extern "C" {

int bysj_adamw_step(const bysj_adamw_tensor* tensors, int64_t n_tensors, int dtype,
                    int state_bits, void* exp_avg, void* exp_avg_sq, float* exp_avg_scale,
                    float* exp_avg_sq_scale, float* master, const float* grad_scale,
                    const bysj_adamw_hyper* hyper, void* stream) {
  return adamw_step(tensors, n_tensors, dtype, state_bits, exp_avg, exp_avg_sq, exp_avg_scale,
                    exp_avg_sq_scale, master, grad_scale, hyper, nullptr, stream);
}

int bysj_adamw_step_counted(const bysj_adamw_tensor* tensors, int64_t n_tensors, int dtype,
                            int state_bits, void* exp_avg, void* exp_avg_sq,
                            float* exp_avg_scale, float* exp_avg_sq_scale, float* master,
                            const float* grad_scale, const bysj_adamw_hyper* hyper,
                            uint64_t counter, void* stream) {
  return adamw_step(tensors, n_tensors, dtype, state_bits, exp_avg, exp_avg_sq, exp_avg_scale,
                    exp_avg_sq_scale, master, grad_scale, hyper, &counter, stream);
}

int bysj_adamw_state_values(const uint8_t* exp_avg, const uint8_t* exp_avg_sq,
                            const float* exp_avg_scale, const float* exp_avg_sq_scale,
                            int64_t blocks, float* exp_avg_values, float* exp_avg_sq_values,
                            void* stream) {
  clear_error();
  if (blocks < 0) return fail(BYSJ_ERR_INVALID_ARGUMENT, "adamw values: invalid size");
  if (blocks == 0) return BYSJ_OK;
  if (exp_avg == nullptr || exp_avg_sq == nullptr || exp_avg_scale == nullptr ||
      exp_avg_sq_scale == nullptr || exp_avg_values == nullptr || exp_avg_sq_values == nullptr)
    return fail(BYSJ_ERR_INVALID_ARGUMENT, "adamw values: NULL pointer");
  const int64_t quads = blocks * (kStateBlock / 4);
  int64_t grid = (quads + kBlock - 1) / kBlock;
  const int64_t cap = static_cast<int64_t>(current_device_info().sm_count) * 8;
  if (grid > cap) grid = cap;
  adamw_values_kernel<<<static_cast<unsigned>(grid), kBlock, 0,
                        static_cast<cudaStream_t>(stream)>>>(
      exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, quads, exp_avg_values,
      exp_avg_sq_values);
  return launch_check("adamw_values_kernel");
}

}  // extern "C"
