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
// A group of L lanes holds a token's row in registers (M logits a lane), so a
// warp routes 32 / L tokens at once.  The row's order is that of unsigned keys
// with the column in the low bits: a key is unique, ties fall to the lowest
// column.  A bfloat16 logit and its column fit 32 bits; a float32 key drops as
// many mantissa bits as the column needs, and a warp in which two neighbours
// of the order agree in what is left, or in which a NaN occurs, orders its
// tokens again by full value and column.  For k = 3 .. 8 each lane sorts its
// keys in lists of eight and keeps the upper half of bitonic merges, first of
// its own lists, then with the other lanes of the group; for other k the next
// largest below `prev` is the maximum of key - prev in wrapping arithmetic
// (the keys still to come wrap to the top), one add-and-max a logit and slot.
//
// P and the counts are sums of integers.  A lane adds its columns' p over the
// tokens of a piece (the part of a frame inside a CTA's range) in float32; a
// CTA adds its warps in their order, rounds to a multiple of 2^-shift (shift
// such that all tokens fit 62 bits, 40 at most) and adds that to the frame's
// total.  Integer atomics give the same sum in any order, so results repeat
// bit for bit.
//
// 500000 x 128 bfloat16 logits, k = 8, renormalised: forward 94 us, bound by the
// integer pipe of the comparators (122 warp instructions a token; the pass a slot
// takes 217 and 168 us; HBM would need 27 us), backward 84 us, bound by issue
// (HBM 49 us).  With an atomic for each probability the pair took 4.7 ms.
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
  unsigned long long* taken;   // [frames][experts] slots
  unsigned long long* number;  // [frames] valid tokens
  unsigned* poison;            // a probability was not a number
  unsigned* ticket;
  int64_t zeroed;              // words from mass on that start at 0
  double* square;              // [CTAs] sum of lse^2
  double* part;                // [CTAs of the losses kernel]
  int shift;
  int ctas;
  int64_t tokens_per_cta;
  bool fused_losses;
  int k_magic;                 // it / k == (it k_magic) >> 16 for it < 32 k
  size_t stage_bytes;
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

template <int V>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[V]) {
  if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else p[0] = v[0];
}
template <int V>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
  } else {
    p[0] = __float2bfloat16_rn(v[0]);
  }
}
template <int V, typename T>
__device__ __forceinline__ void copy_vec(T* to, const T* from) {
  if constexpr (V * sizeof(T) == 16)
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
  else *to = *from;
}
template <int V, typename T>
__device__ __forceinline__ void zero_vec(T* to) {
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(to) = make_uint4(0u, 0u, 0u, 0u);
  else *to = T(0.0f);
}

// Cotangents in shared memory, so that the L lanes of a row read 16 bytes each
// side by side: vector n of V columns keeps its quarters apart, [n][V / 4][L][4].
template <int V, int L>
__device__ __forceinline__ int cot_place(int c) {
  if constexpr (V <= 4) return c;
  else return c / (V * L) * V * L + (c % V / 4 * L + c / V % L) * 4 + c % 4;
}
// Those of vector n of lane l.
template <int V, int L>
__device__ __forceinline__ void load_cot(const float* s, int n, int l, float (&v)[V]) {
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(s + n * V * L + (i / 4 * L + l) * 4);
      v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
    }
  } else {
    v[0] = s[n * L + l];
  }
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

__device__ __forceinline__ int64_t frame_end(const RouteArgs& a, int64_t s) {
  return a.offsets == nullptr || s + 1 >= a.frames ? a.tokens : __ldg(a.offsets + s + 1);
}

// The logits of one token that a lane holds: NV vectors of V, element i of
// vector v at column (v L + l) V + i, as loaded (a bfloat16 row in flight
// takes half the registers).
template <typename T, int V, int NV, int L>
struct Row {
  RowVec<T, V> v[NV];
  __device__ __forceinline__ void load(const T* row, int l, int experts, bool on) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (n * L + l) * V;
      if (on && c < experts) v[n].load(row, n * L + l);
      else fill(v[n]);
    }
  }
  __device__ __forceinline__ float get(int i) const { return v[i / V].get(i % V); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NV; ++n) fill(v[n]);
  }
  // Largest of the lane's logits (a NaN yields to a number).
  __device__ __forceinline__ float top() const {
    if constexpr (sizeof(T) == 2 && V == 8) {  // two at a time
      __nv_bfloat162 m = pair(0);
#pragma unroll
      for (int w = 1; w < 4 * NV; ++w) m = __hmax2(m, pair(w));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      float m = get(0);
#pragma unroll
      for (int i = 1; i < V * NV; ++i) m = fmaxf(m, get(i));
      return m;
    }
  }
  // Logits 2 w and 2 w + 1 of a bfloat16 row.
  __device__ __forceinline__ __nv_bfloat162 pair(int w) const {
    const uint4& r = v[w / 4].r;
    const uint32_t u = w % 4 == 0 ? r.x : w % 4 == 1 ? r.y : w % 4 == 2 ? r.z : r.w;
    return *reinterpret_cast<const __nv_bfloat162*>(&u);
  }
  __device__ static constexpr int column(int i, int l) { return ((i / V) * L + l) * V + i % V; }
  // -inf: what lies beyond the row's end, or belongs to a token left out
  __device__ static __forceinline__ void fill(RowVec<float, 4>& r) {
    r.r = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  }
  __device__ static __forceinline__ void fill(RowVec<float, 1>& r) { r.r = -INFINITY; }
  __device__ static __forceinline__ void fill(RowVec<__nv_bfloat16, 8>& r) {
    r.r = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  }
  __device__ static __forceinline__ void fill(RowVec<__nv_bfloat16, 1>& r) { r.r = 0xff80u; }
};

template <int L>
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int s = 1; s < L; s <<= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, s));
  return v;
}
template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int s = 1; s < L; s <<= 1) v += __shfl_xor_sync(kFull, v, s);
  return v;
}
template <int L>
__device__ __forceinline__ unsigned row_max(unsigned v) {
#pragma unroll
  for (int s = 1; s < L; s <<= 1) v = max(v, __shfl_xor_sync(kFull, v, s));
  return v;
}

// Keys.  order_bits: the bits of a float in the order of the values (+ 0.0f
// makes the two zeros equal).  A key replaces the bits under `mask` by
// mask - column; column (n L + l) V + i has the lane l in bits of its own, so
// a lane orders its own keys without them and adds them before it meets others.
constexpr unsigned kBarred = 0x007fffffu;  // order_bits(-inf)

template <typename T, int V, int NV, int L>
struct Keys {
  static constexpr int M = V * NV;
  static constexpr unsigned kMask = sizeof(T) == 2 ? 0xffffu : M * L - 1;
  static constexpr unsigned kLane = (L - 1) * V;  // the lane's bits of a column
  static constexpr unsigned kBar = kBarred | kMask;
  __device__ static __forceinline__ unsigned order_bits(float v) {
    const unsigned b = __float_as_uint(v + 0.0f);
    return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
  }
  // Keys of a lane's row, without the lane's own bits.
  __device__ static __forceinline__ void make(const Row<T, V, NV, L>& row, unsigned (&key)[M]) {
    if constexpr (sizeof(T) == 2 && V == 8) {  // two at a time, off the integer pipe where it goes
#pragma unroll
      for (int w = 0; w < M / 2; ++w) {
        const __nv_bfloat162 z = __hadd2(row.pair(w), __float2bfloat162_rn(0.0f));
        const unsigned b = *reinterpret_cast<const unsigned*>(&z);
        const unsigned o = b ^ (((b >> 15) & 0x00010001u) * 0x7fffu | 0x80008000u);
        key[2 * w] = o * 65536u + rest(2 * w);
        key[2 * w + 1] = (o & 0xffff0000u) | rest(2 * w + 1);
      }
    } else {
#pragma unroll
      for (int i = 0; i < M; ++i) key[i] = (order_bits(row.get(i)) & ~kMask) | rest(i);
    }
  }
  __device__ static constexpr unsigned rest(int i) {
    return (kMask - (i / V) * L * V - i % V) & ~kLane;
  }
  __device__ static __forceinline__ unsigned lane_part(int l) {
    return kLane - static_cast<unsigned>(l * V);
  }
  __device__ static __forceinline__ bool barred(unsigned key) { return (key | kMask) <= kBar; }
  __device__ static __forceinline__ int column(unsigned key) {
    return static_cast<int>(kMask - (key & kMask));
  }
  // The logit of a key: in the key itself for bfloat16, else read again.
  __device__ static __forceinline__ float logit(unsigned key, const T* row) {
    if constexpr (sizeof(T) == 2) {
      const unsigned b = key & 0xffff0000u;
      return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : b ^ 0xffff0000u);
    } else {
      return load_f32(row + column(key));
    }
  }
};

// Comparators of sorting networks, larger first.
__device__ __forceinline__ void order2(unsigned& a, unsigned& b) {
  const unsigned hi = max(a, b);
  b = min(a, b);
  a = hi;
}
__device__ __forceinline__ void sort8(unsigned (&v)[8]) {  // odd-even merge sort
  order2(v[0], v[1]); order2(v[2], v[3]); order2(v[4], v[5]); order2(v[6], v[7]);
  order2(v[0], v[2]); order2(v[1], v[3]); order2(v[4], v[6]); order2(v[5], v[7]);
  order2(v[1], v[2]); order2(v[5], v[6]);
  order2(v[0], v[4]); order2(v[1], v[5]); order2(v[2], v[6]); order2(v[3], v[7]);
  order2(v[2], v[4]); order2(v[3], v[5]);
  order2(v[1], v[2]); order2(v[3], v[4]); order2(v[5], v[6]);
}
__device__ __forceinline__ void merge8(unsigned (&v)[8]) {  // a bitonic list in order
#pragma unroll
  for (int s = 4; s > 0; s >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((i & s) == 0) order2(v[i], v[i + s]);
}

// exp(x - ref) on the transcendental pipe: the rounding of the product adds
// |x - ref| 2^-24 relative to the 2 units of ex2.  The difference comes first,
// so rows of any magnitude (all at the type's lowest value, say) are safe.
__device__ __forceinline__ float exp_from(float x, float ref) {
  return ex2_ftz((x - ref) * 1.4426950408889634f);
}

// Exact order for a warp's rows: the next in (value, then column) after
// (prev, at); NaN is largest.  Slow: two reductions a slot.
template <typename T, int V, int NV, int L>
__device__ __noinline__ void pick_exact(const Row<T, V, NV, L>& row, int l, int experts, int k,
                                        unsigned* picks) {
  using Key = Keys<T, V, NV, L>;
  constexpr int M = V * NV;
  unsigned prev = 0;
  int at = -1;
  for (int slot = 0; slot < k; ++slot) {
    unsigned best = 0;
    int where = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int c = row.column(i, l);
      const float x = row.get(i);
      const unsigned key = c >= experts ? 0u : isnan(x) ? 0xffffffffu : Key::order_bits(x);
      const bool left = slot == 0 || key < prev || (key == prev && c > at);
      if (left && (key > best || (key == best && c < where))) {
        best = key;
        where = c;
      }
    }
#pragma unroll
    for (int s = 1; s < L; s <<= 1) {
      const unsigned other = __shfl_xor_sync(kFull, best, s);
      const int there = __shfl_xor_sync(kFull, where, s);
      if (other > best || (other == best && there < where)) {
        best = other;
        where = there;
      }
    }
    if (l == 0)
      picks[slot] = best <= kBarred ? 0u : (best & ~Key::kMask) | (Key::kMask - where);
    prev = best;
    at = where;
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

// share, counts and the losses from the totals, by CTA `cta` of `ctas`; reads
// through L2, where the other CTAs' totals are.
__device__ void route_losses(const RouteArgs& a, int cta, int ctas) {
  __shared__ double scratch[kWarpsPerBlock];
  __shared__ bool s_join;
  double used = 0.0, valid = 0.0;
  for (int64_t s = threadIdx.x; s < a.frames; s += kBlock) {
    const unsigned long long n = __ldcg(a.number + s);
    used += n > 0;
    valid += static_cast<double>(n);
  }
  used = block_sum(used, scratch);
  valid = block_sum(valid, scratch);
  const double unit = 1.0 / static_cast<double>(int64_t{1} << a.shift);
  double balance = 0.0;
  for (int64_t i = static_cast<int64_t>(cta) * kBlock + threadIdx.x; i < a.frames * a.experts;
       i += static_cast<int64_t>(ctas) * kBlock) {
    const double n = static_cast<double>(__ldcg(a.number + i / a.experts));
    const unsigned long long taken = __ldcg(a.taken + i);
    const double share =
        n > 0.0 ? a.experts * static_cast<double>(taken) / (a.k * n * n * used) : 0.0;
    a.share[i] = static_cast<float>(share);
    a.counts[i] = static_cast<int64_t>(taken);
    balance += share * (static_cast<double>(__ldcg(a.mass + i)) * unit);
  }
  balance = block_sum(balance, scratch);
  if (ctas > 1) {  // join the CTAs' parts in their order
    if (threadIdx.x == 0) {
      __stcg(a.part + cta, balance);
      __threadfence();
      s_join = atomicAdd(a.ticket, 1u) + 1 == static_cast<unsigned>(ctas);
      __threadfence();
    }
    __syncthreads();
    if (!s_join) return;
    balance = 0.0;
    for (int i = threadIdx.x; i < ctas; i += kBlock) balance += __ldcg(a.part + i);
    balance = block_sum(balance, scratch);
  }
  double square = 0.0;
  for (int i = threadIdx.x; i < a.ctas; i += kBlock) square += __ldcg(a.square + i);
  square = block_sum(square, scratch);
  if (threadIdx.x == 0) {
    *a.balance = __ldcg(a.poison) ? NAN : static_cast<float>(balance);
    *a.z = valid > 0.0 ? static_cast<float>(square / valid) : 0.0f;
    *a.z_scale = valid > 0.0 ? static_cast<float>(2.0 / valid) : 0.0f;
  }
}

// Shared memory of the forward kernel, per CTA: counts [E], one row of mass a
// warp [warps][E], and per warp the picks and their values [32 / L][k].
// TOP 8: networks, k <= 8; TOP 0: a pass a slot.
template <typename T, int V, int NV, int L, int TOP>
__global__ void __launch_bounds__(kBlock, 2) route_forward_kernel(RouteArgs a) {
  constexpr int M = V * NV, R = kWarp / L;
  using RowT = Row<T, V, NV, L>;
  using Key = Keys<T, V, NV, L>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int E = a.experts, k = a.k, items = R * k;
  unsigned* s_count = reinterpret_cast<unsigned*>(smem);
  float* s_mass = reinterpret_cast<float*>(s_count + E);
  unsigned* s_pick = reinterpret_cast<unsigned*>(s_mass + kWarpsPerBlock * E);
  const int lane = lane_id(), warp = threadIdx.x / kWarp, l = lane % L, g = lane / L;
  unsigned* picks = s_pick + warp * 2 * items;
  float* values = reinterpret_cast<float*>(picks + items);
  __shared__ double s_square[kWarpsPerBlock];
  __shared__ int s_valid[kWarpsPerBlock];
  __shared__ bool s_last;
  const T* logits = static_cast<const T*>(a.logits);
  const float unit = static_cast<float>(int64_t{1} << a.shift);
  const unsigned lane_part = Key::lane_part(l);
  const int64_t t0 = a.tokens_per_cta * blockIdx.x;
  const int64_t t1 = min(t0 + a.tokens_per_cta, a.tokens);

  if (gridDim.x == 1) {  // alone: no memset ran before
    for (int64_t i = threadIdx.x; i < a.zeroed; i += kBlock) a.mass[i] = 0;
  }
  for (int i = threadIdx.x; i < E; i += kBlock) s_count[i] = 0;
  __syncthreads();

  double square = 0.0;
  int64_t s = t0 < t1 ? frame_of(a, t0) : 0;
  for (int64_t lo = t0; lo < t1; ++s) {
    const int64_t hi = min(frame_end(a, s), t1);
    if (hi <= lo) {
      if (s + 1 >= a.frames) break;
      continue;
    }
    float mass[M];
#pragma unroll
    for (int i = 0; i < M; ++i) mass[i] = 0.0f;
    int valid_rows = 0;
    auto fetch = [&](int64_t base, RowT& row) {
      const int64_t t = base + g;
      const bool on = t < hi && (a.mask == nullptr || __ldg(a.mask + t) != 0);
      row.load(logits + t * E, l, E, on);
    };
    RowT next;
    fetch(lo + warp * R, next);
    for (int64_t base = lo + warp * R; base < hi; base += kWarpsPerBlock * R) {
      const RowT row = next;
      if (base + kWarpsPerBlock * R < hi) fetch(base + kWarpsPerBlock * R, next);
      const int64_t t = base + g;
      const float top = row_max<L>(row.top());
      const float ref = top > -INFINITY ? top : 0.0f;
      float total = 0.0f, inv;
      {
        float e[M];
#pragma unroll
        for (int i = 0; i < M; ++i) {
          e[i] = exp_from(row.get(i), ref);
          total += e[i];
        }
        total = row_sum<L>(total);
        inv = total != 0.0f ? 1.0f / total : 0.0f;  // 0: every logit is -inf
#pragma unroll
        for (int i = 0; i < M; ++i) mass[i] = fmaf(e[i], inv, mass[i]);
      }
      bool unclear = isnan(total);
      constexpr bool kExact = sizeof(T) == 2;
      if constexpr (TOP == 8) {
        unsigned list[8];
        int above = 0;  // keys that reach the last pick's kept bits
        {
          unsigned key[M];
          Key::make(row, key);
#pragma unroll
          for (int i = 0; i < 8; ++i) list[i] = i < M ? key[i < M ? i : 0] : 0u;
          sort8(list);
#pragma unroll
          for (int n = 8; n < M; n += 8) {
            unsigned other[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) other[i] = key[n + i];
            sort8(other);
#pragma unroll
            for (int i = 0; i < 8; ++i) list[i] = max(list[i], other[7 - i]);
            merge8(list);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) list[i] |= lane_part;
#pragma unroll
          for (int d = 1; d < L; d <<= 1) {
            unsigned other[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) other[i] = __shfl_xor_sync(kFull, list[7 - i], d);
#pragma unroll
            for (int i = 0; i < 8; ++i) list[i] = max(list[i], other[i]);
            merge8(list);
          }
          if constexpr (!kExact) {
            unsigned last = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (i == k - 1) last = list[i] & ~Key::kMask;
#pragma unroll
            for (int i = 0; i < M; ++i) above += key[i] >= last;
            if (last <= kBarred) above = 0;  // barred either way
          }
        }
        if constexpr (!kExact) {
#pragma unroll
          for (int d = 1; d < L; d <<= 1) above += __shfl_xor_sync(kFull, above, d);
          unclear |= above > k;
#pragma unroll
          for (int i = 1; i < 8; ++i)
            unclear |= i < k && !Key::barred(list[i]) &&
                       (list[i] | Key::kMask) == (list[i - 1] | Key::kMask);
        }
        if (__any_sync(kFull, unclear)) {
          pick_exact<T, V, NV, L>(row, l, E, k, picks + g * k);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) list[i] = i < k ? picks[g * k + i] : 0u;
          __syncwarp();
        }
        // slots l, l + L, ... of the row are this lane's to finish
        constexpr int kMine = L >= 8 ? 1 : 8 / L;
        unsigned mine[kMine];
        float w[kMine], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          mine[i] = 0u;
#pragma unroll
          for (int q = 0; q < (L < 8 ? L : 8); ++q)
            if (l == q) mine[i] = list[i * L + q];
          const bool on = l + i * L < k && t < hi && !Key::barred(mine[i]);
          if (!on) mine[i] = 0u;
          w[i] = on ? exp_from(Key::logit(mine[i], logits + t * E), ref) * inv : 0.0f;
          sum += w[i];
          if (on) atomicAdd(s_count + Key::column(mine[i]), 1u);
        }
        if (a.renormalize) {
          sum = row_sum<L>(sum);
#pragma unroll
          for (int i = 0; i < kMine; ++i)
            if (mine[i] != 0u) w[i] /= sum;
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          if (l + i * L < k && t < hi) {
            const int64_t at = t * k + l + i * L;
            a.weights[at] = w[i];
            a.chosen[at] = mine[i] == 0u ? int64_t{-1} : Key::column(mine[i]);
          }
        }
      } else {
        unsigned key[M];
        Key::make(row, key);
#pragma unroll
        for (int i = 0; i < M; ++i) key[i] |= lane_part;
        unsigned prev = 0;
        const int rounds = kExact ? k : k + 1;  // one more: is the last one clear?
        for (int slot = 0; slot < rounds; ++slot) {
          unsigned m = 0;
#pragma unroll
          for (int i = 0; i < M; ++i) m = __viaddmax_u32(key[i], 0u - prev, m);
          const unsigned best = row_max<L>(m) + prev;
          if constexpr (!kExact)
            unclear |= slot > 0 && best < prev && !Key::barred(best) &&
                       (best | Key::kMask) == (prev | Key::kMask);
          if (l == 0 && slot < k) picks[g * k + slot] = best;
          prev = best;
        }
        if (__any_sync(kFull, unclear)) pick_exact<T, V, NV, L>(row, l, E, k, picks + g * k);
        __syncwarp();
        // weights and indices, the warp's R k slots side by side
        for (int it0 = 0; it0 < items; it0 += kWarp) {
          const int it = it0 + lane;
          const int r = min((it * a.k_magic) >> 16, R - 1);
          const float ref_r = __shfl_sync(kFull, ref, r * L);
          const float inv_r = __shfl_sync(kFull, inv, r * L);
          if (it < items) {
            unsigned pick = picks[it];
            float p = 0.0f;
            if (base + r >= hi || Key::barred(pick)) pick = 0u;
            if (pick != 0u) {
              p = exp_from(Key::logit(pick, logits + (base + r) * E), ref_r) * inv_r;
              atomicAdd(s_count + Key::column(pick), 1u);
            }
            picks[it] = pick;
            values[it] = p;
          }
        }
        __syncwarp();
        for (int it = lane; it < items; it += kWarp) {
          const int r = (it * a.k_magic) >> 16;
          if (base + r < hi) {
            float w = values[it];
            const unsigned pick = picks[it];
            if (a.renormalize && pick != 0u) {
              float sum = 0.0f;
              for (int j = 0; j < k; ++j) sum += values[r * k + j];
              w /= sum;
            }
            a.weights[base * k + it] = w;
            a.chosen[base * k + it] = pick == 0u ? int64_t{-1} : Key::column(pick);
          }
        }
        __syncwarp();
      }
      if (l == 0 && t < hi) {
        a.denom[t] = total;
        if (total != 0.0f) {  // a NaN counts
          const float lse = ref + logf(total);
          square += static_cast<double>(lse) * lse;
          ++valid_rows;
        }
      }
    }

    // flush the piece into its frame's totals
#pragma unroll
    for (int i = 0; i < M; ++i) {
      mass[i] = xor_sum(mass[i], L);
      const int c = RowT::column(i, l);
      if (g == 0 && c < E) s_mass[warp * E + c] = mass[i];
    }
    for (int o = L; o < kWarp; o <<= 1) valid_rows += __shfl_xor_sync(kFull, valid_rows, o);
    if (lane == 0) s_valid[warp] = valid_rows;
    __syncthreads();
    for (int c = threadIdx.x; c < E; c += kBlock) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarpsPerBlock; ++w) sum += s_mass[w * E + c];
      if (isnan(sum)) atomicOr(a.poison, 1u);
      else if (sum != 0.0f)
        atomicAdd(a.mass + s * E + c, static_cast<unsigned long long>(__float2ull_rn(sum * unit)));
      if (s_count[c] != 0) {
        atomicAdd(a.taken + s * E + c, static_cast<unsigned long long>(s_count[c]));
        s_count[c] = 0;
      }
    }
    if (threadIdx.x == 0) {
      int n = 0;
      for (int w = 0; w < kWarpsPerBlock; ++w) n += s_valid[w];
      if (n != 0) atomicAdd(a.number + s, static_cast<unsigned long long>(n));
    }
    __syncthreads();
    lo = hi;
  }

  square = xor_sum(square, 1);
  if (lane == 0) s_square[warp] = square;
  __syncthreads();
  if (threadIdx.x == 0) {
    square = 0.0;
    for (int w = 0; w < kWarpsPerBlock; ++w) square += s_square[w];
    __stcg(a.square + blockIdx.x, square);
  }
  if (!a.fused_losses) return;
  // the last CTA to arrive turns the totals into the losses
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(a.ticket, 1u) + 1 == gridDim.x;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  route_losses(a, 0, 1);
}

__global__ void __launch_bounds__(kBlock) route_losses_kernel(RouteArgs a) {
  route_losses(a, blockIdx.x, gridDim.x);
}

// Shared memory, per CTA: the rows on their way out [warps][32 / L][E] and the
// cotangents share[s, e] grad_balance [M L] (see cot_place).
template <typename T, int V, int NV, int L>
__global__ void __launch_bounds__(kBlock, V * NV <= 16 ? 3 : 2)
    route_backward_kernel(RouteArgs a) {
  constexpr int M = V * NV, R = kWarp / L;
  using RowT = Row<T, V, NV, L>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int E = a.experts, k = a.k;
  const int lane = lane_id(), warp = threadIdx.x / kWarp, l = lane % L, g = lane / L;
  float* s_cot = reinterpret_cast<float*>(smem + a.stage_bytes);  // 16-byte aligned
  T* stage = reinterpret_cast<T*>(smem) + (warp * R + g) * E;
  const T* logits = static_cast<const T*>(a.logits);
  T* out = static_cast<T*>(a.grad_logits);
  const bool gated = a.grad_weights != nullptr;
  const float gb = a.grad_balance ? __ldg(a.grad_balance) : 0.0f;
  const float gz = a.grad_z ? __ldg(a.grad_z) * __ldg(a.z_scale) : 0.0f;
  const int64_t t0 = a.tokens_per_cta * blockIdx.x;
  const int64_t t1 = min(t0 + a.tokens_per_cta, a.tokens);

  // What a token needs, requested one step ahead; slots l, l + L, ... of its k
  // belong to lane l, those of the first eight here.
  constexpr int kMine = L >= 8 ? 1 : 8 / L;
  struct Fetch {
    RowT row;
    float total, w[kMine], gw[kMine];
    int slot[kMine], first;  // experts of the lane's slots; of slot 0
  };
  auto fetch = [&](int64_t t, int64_t hi) {
    Fetch f;
    const bool in = t < hi;
    f.row.load(logits + t * E, l, E, in);
    f.total = in ? __ldg(a.denom + t) : 1.0f;
    f.first = in ? static_cast<int>(__ldg(a.chosen + t * k)) : -1;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int j = l + i * L;
      const bool mine = gated && in && j < k;
      f.slot[i] = mine ? static_cast<int>(__ldg(a.chosen + t * k + j)) : -1;
      f.w[i] = mine ? __ldg(a.weights + t * k + j) : 0.0f;
      f.gw[i] = mine ? __ldg(a.grad_weights + t * k + j) : 0.0f;
    }
    return f;
  };

  int64_t s = t0 < t1 ? frame_of(a, t0) : 0;
  for (int64_t lo = t0; lo < t1; ++s) {
    const int64_t hi = min(frame_end(a, s), t1);
    if (hi <= lo) {
      if (s + 1 >= a.frames) break;
      continue;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < M * L; c += kBlock)
      s_cot[cot_place<V, L>(c)] = c < E ? gb * __ldg(a.share + s * E + c) : 0.0f;
    __syncthreads();
    Fetch next = fetch(lo + warp * R + g, hi);
    for (int64_t base = lo + warp * R; base < hi; base += kWarpsPerBlock * R) {
      const int64_t t = base + g;
      Fetch f = next;
      if (base + kWarpsPerBlock * R < hi) next = fetch(t + kWarpsPerBlock * R, hi);
      if (f.first < 0) {  // not a valid token: its gradient is 0 whatever comes back
        f.row.clear();
        f.total = 1.0f;
      }
      const float inv = 1.0f / f.total;
      const float top = row_max<L>(f.row.top());
      const float ref = top > -INFINITY ? top : 0.0f;
      float along_w = 0.0f;
#pragma unroll
      for (int i = 0; i < kMine; ++i)  // an empty slot's cotangent may hold anything
        along_w = fmaf(f.w[i], f.slot[i] >= 0 ? f.gw[i] : 0.0f, along_w);
      if (gated && k > kMine * L && t < hi)
        for (int j = l + kMine * L; j < k; j += L)
          if (__ldg(a.chosen + t * k + j) >= 0)
            along_w += __ldg(a.weights + t * k + j) * __ldg(a.grad_weights + t * k + j);
      along_w = row_sum<L>(along_w);
      // p_e and the sum of p_e a_e; a weight that is p itself adds gw p at its expert
      float p[M], along = 0.0f;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        float cot[V];
        load_cot<V, L>(s_cot, n, l, cot);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          p[n * V + i] = exp_from(f.row.get(n * V + i), ref) * inv;
          along = fmaf(p[n * V + i], cot[i], along);
        }
      }
      along = row_sum<L>(along);
      if (!a.renormalize) along += along_w;
      const float pull = gz * (ref + logf(f.total)) - along;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = (n * L + l) * V;
        float v[V];
        load_cot<V, L>(s_cot, n, l, v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = p[n * V + i] * (v[i] + pull);
        if (c < E) store_vec<V>(stage + c, v);
      }
      if (gated) {  // the chosen experts once more, with the weights' part
        __syncwarp();
        auto fix = [&](int c, float w, float gw) {
          const float pe = a.renormalize
                               ? exp_from(load_f32(logits + t * E + c), ref) * inv
                               : w;
          const float cot = s_cot[cot_place<V, L>(c)];
          store_value(stage + c, a.renormalize ? fmaf(pe, cot + pull, w * (gw - along_w))
                                               : pe * (cot + gw + pull));
        };
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (f.slot[i] >= 0) fix(f.slot[i], f.w[i], f.gw[i]);
        if (t < hi)
          for (int j = l + kMine * L; j < k; j += L) {
            const int c = static_cast<int>(__ldg(a.chosen + t * k + j));
            if (c >= 0) fix(c, __ldg(a.weights + t * k + j), __ldg(a.grad_weights + t * k + j));
          }
      }
      __syncwarp();
      if (t < hi) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          const int c = (n * L + l) * V;
          if (c >= E) continue;
          if (f.first >= 0) copy_vec<V>(out + t * E + c, stage + c);
          else zero_vec<V>(out + t * E + c);
        }
      }
      __syncwarp();
    }
    lo = hi;
  }
}

// Launch shapes by the number of experts: L lanes a token and M logits a lane.
// Few lanes a token mean few shuffles: M = 32 for the networks.  The other
// kernels take M = 16, which leaves registers for more warps (backward pass of
// 500000 x 128 bfloat16: 87 us, 98 us with M = 32).  Rows whose length is
// not a multiple of the vector width, or that are not aligned to 16 bytes, are
// read one logit at a time.
using RouteKernel = void (*)(RouteArgs);
struct RouteShape {
  RouteKernel kernel;
  int lanes, columns;  // of a token: lanes, and logits they hold
};

enum RoutePass { kForwardSlots, kForwardNetwork, kBackward };

template <typename T, int V, int NV, int L, RoutePass P>
RouteShape route_shape() {
  if constexpr (P == kBackward) return {route_backward_kernel<T, V, NV, L>, L, V * NV * L};
  else return {route_forward_kernel<T, V, NV, L, P == kForwardNetwork ? 8 : 0>, L, V * NV * L};
}

template <typename T, RoutePass P>
RouteShape route_pick(int experts, bool vectors) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  constexpr int W = P == kForwardNetwork ? 2 : 1;  // 16 W logits a lane
  if (vectors) {
    if (experts <= 16) return route_shape<T, V, 1, 16 / V, P>();
    if (experts <= 32) return route_shape<T, V, 8 / V, 4, P>();
    if (experts <= 64) return route_shape<T, V, 16 / V, 4, P>();
    if (experts <= 128) return route_shape<T, V, 16 * W / V, 8 / W, P>();
    if (experts <= 256) return route_shape<T, V, 16 * W / V, 16 / W, P>();
    if (experts <= 512) return route_shape<T, V, 16 * W / V, 32 / W, P>();
    return route_shape<T, V, 32 / V, 32, P>();
  }
  if constexpr (P == kForwardNetwork) {
    return route_pick<T, kForwardSlots>(experts, false);
  } else {
    if (experts <= 16) return route_shape<T, 1, 4, 4, P>();
    if (experts <= 64) return route_shape<T, 1, 8, 8, P>();
    if (experts <= 256) return route_shape<T, 1, 16, 16, P>();
    if (experts <= 512) return route_shape<T, 1, 16, 32, P>();
    return route_shape<T, 1, 32, 32, P>();
  }
}

template <typename T>
RouteShape route_pick_pass(int experts, bool vectors, RoutePass pass) {
  if (pass == kBackward) return route_pick<T, kBackward>(experts, vectors);
  return pass == kForwardNetwork ? route_pick<T, kForwardNetwork>(experts, vectors)
                                 : route_pick<T, kForwardSlots>(experts, vectors);
}

RouteShape route_pick_any(int dtype, int experts, const void* a, const void* b, RoutePass pass) {
  const int v = dtype == BYSJ_F32 ? 4 : 8;
  const bool vectors = experts % v == 0 && aligned16(a) && aligned16(b);
  return dtype == BYSJ_F32 ? route_pick_pass<float>(experts, vectors, pass)
                           : route_pick_pass<__nv_bfloat16>(experts, vectors, pass);
}

// A CTA's tokens: at least 64, so that its flush into the frames' totals is
// small beside them; one wave of the forward's two CTAs for each SM.
int route_ctas(int64_t tokens) {
  int64_t ctas = (tokens + 63) / 64;
  const int64_t cap = static_cast<int64_t>(current_device_info().sm_count) * 2;
  if (ctas > cap) ctas = cap;
  return ctas < 1 ? 1 : static_cast<int>(ctas);
}

// One CTA's worth of losses rides along in the forward kernel; more cells than
// this get a kernel of their own.
constexpr int64_t kFusedLossCells = 16384;

int loss_ctas(int64_t cells) {
  const int64_t ctas = (cells + 8 * kBlock - 1) / (8 * kBlock);
  const int64_t cap = current_device_info().sm_count;
  return static_cast<int>(ctas < cap ? ctas : cap);
}

// The zeroed part comes first, in whole 8-byte words.
size_t carve_workspace(RouteArgs& a, void* workspace) {
  Carver carve(workspace);
  const size_t cells = static_cast<size_t>(a.frames) * a.experts;
  a.zeroed = static_cast<int64_t>(2 * cells + a.frames + 1);
  a.mass = carve.take<unsigned long long>(static_cast<size_t>(a.zeroed));
  a.taken = a.mass + cells;
  a.number = a.taken + cells;
  a.poison = reinterpret_cast<unsigned*>(a.number + a.frames);
  a.ticket = a.poison + 1;
  a.square = carve.take<double>(static_cast<size_t>(a.ctas));
  a.part = carve.take<double>(static_cast<size_t>(current_device_info().sm_count));
  return carve.need;
}

void plan_tokens(RouteArgs& a) {
  a.ctas = route_ctas(a.tokens);
  a.tokens_per_cta = ((a.tokens + a.ctas - 1) / a.ctas + 63) / 64 * 64;
  a.k_magic = 65536 / a.k + 1;
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
  return carve_workspace(a, nullptr);
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
  a.tokens = tokens;
  a.experts = static_cast<int>(n_experts);
  a.k = static_cast<int>(k);
  a.frames = frames;
  plan_tokens(a);
  const size_t need = carve_workspace(a, workspace);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(BYSJ_ERR_WORKSPACE, "route: workspace of %zu bytes needed, %zu given", need,
                workspace_bytes);
  a.logits = logits;
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
  a.fused_losses = frames * n_experts <= kFusedLossCells;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.ctas > 1) {
    st = cuda_check(cudaMemsetAsync(a.mass, 0, sizeof(unsigned long long) * a.zeroed, s),
                    "route: zero workspace");
    if (st) return st;
  }
  const RouteShape shape = route_pick_any(dtype, a.experts, logits, logits,
                                          k >= 3 && k <= 8 ? kForwardNetwork : kForwardSlots);
  const size_t smem = sizeof(unsigned) * (a.experts * (1 + kWarpsPerBlock) +
                                          kWarpsPerBlock * 2 * (kWarp / shape.lanes) * a.k);
  st = allow_dynamic_smem(reinterpret_cast<const void*>(shape.kernel), smem);
  if (st) return st;
  shape.kernel<<<a.ctas, kBlock, smem, s>>>(a);
  st = launch_check("route_forward_kernel");
  if (st || a.fused_losses) return st;
  route_losses_kernel<<<loss_ctas(frames * n_experts), kBlock, 0, s>>>(a);
  return launch_check("route_losses_kernel");
}

int bysj_route_backward(const void* logits, int dtype, int64_t tokens, int64_t n_experts,
                        int64_t k, const int64_t* offsets, int64_t frames, int renormalize,
                        const float* weights, const int64_t* experts, const float* denom,
                        const float* share, const float* z_scale, const float* grad_weights,
                        const float* grad_balance, const float* grad_z, void* grad_logits,
                        void* stream) {
  clear_error();
  int st = check_sizes(dtype, tokens, n_experts, k, offsets, frames);
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
  plan_tokens(a);
  // no flush here: smaller ranges, three CTAs for each SM and four waves
  const int64_t per = (tokens + current_device_info().sm_count * 12 - 1) /
                      (current_device_info().sm_count * 12);
  a.tokens_per_cta = (per + 63) / 64 * 64;
  a.ctas = static_cast<int>((tokens + a.tokens_per_cta - 1) / a.tokens_per_cta);
  const RouteShape shape = route_pick_any(dtype, a.experts, logits, grad_logits, kBackward);
  const size_t rows = static_cast<size_t>(kWarpsPerBlock) * (kWarp / shape.lanes);
  a.stage_bytes = (rows * a.experts * (dtype == BYSJ_F32 ? 4 : 2) + 15) / 16 * 16;
  const size_t smem = a.stage_bytes + sizeof(float) * shape.columns;
  st = allow_dynamic_smem(reinterpret_cast<const void*>(shape.kernel), smem);
  if (st) return st;
  shape.kernel<<<a.ctas, kBlock, smem, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_check("route_backward_kernel");
}

}  // extern "C"
