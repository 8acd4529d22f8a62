// Group norm over frames with an activation, channels last, for sm_100a.
//
//   z = (x - mean[b, g]) rstd[b, g] w[c] + b[c],  y = act(z)
//   dz = dy act'(z), d = dz w
//   dx = rstd (d - mean(d) - xhat mean(d xhat)),  dw = sum dz xhat,  db = sum dz
//
// By the mean size of a frame (the lengths themselves are on the device only):
//
// Small frames: a CTA takes whole frames, reads each twice (the second time
// from L1 or L2, if it is small) and needs no other CTA.  A long frame among many
// short ones is then one CTA's work, at a small part of the bandwidth.
//
// Larger frames: the rows of all frames are cut into one chunk for each
// resident CTA, whatever the frames' lengths; the part of a frame inside a
// chunk is a piece.  Pieces are numbered chunk + frame, which is unique because
// going from one piece to the next advances at least one of the two.  A first
// kernel leaves two numbers per piece and channel (mean and centred square
// sum; in the backward pass sum dz and sum dz xhat, from which the group's sums
// and the gradients of weight and bias both follow); numbers that no piece has
// are zero.  A second kernel joins the pieces of each frame and group, a third
// writes the result.  It walks each chunk from its end, where the first stopped,
// so that what L2 still holds is read from there (39 of 101 MB of x forward, 23 of
// 201 MB of x and dy backward, at 393216 x 128 bfloat16).
//
// Sums are float32, of a few tens of terms at a time (rows of a thread, threads
// of a channel, pieces of a frame), so their rounding does not grow with the
// rows; float64 arithmetic cost tens of microseconds a kernel here.  The variance
// loses no digits to outliers or to channels that lie apart: a thread takes
// squares about the mean of its own rows nearby, and means and squares of threads,
// pieces and channels are joined as such, where only squares add.  No atomics:
// results repeat bit for bit.
//
// Bound by HBM in the results, by instruction issue and loads in flight in the
// statistics.  16 frames of 24576 x 128 bfloat16 with SiLU: forward 34 us
// statistics, 5 us join, 35 us result (302 MB with x read twice: 46 us at the
// measured copy bandwidth), backward 53, 4 and 59 us (503 MB: 77 us).  One kernel
// that meets its CTAs for each frame (slabs of shared memory, or drawn chunks)
// took 2 to 3 times as long: a meeting costs several microseconds, and a frame
// of megabytes needs many.
//
// z is one multiply-add, x A + B with A = rstd w and B = b - mean A: B's
// rounding is 2^-24 |mean| rstd w, as large as that of the stored mean.
#include <type_traits>

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
  // Last frame that begins at or before row r; a whole warp, 32 probes a step.
  __device__ __forceinline__ int64_t of_row(int64_t r) const {
    if (offsets == nullptr) return r / (rows / count);
    int64_t lo = 0, hi = count;
    while (hi - lo > 1) {
      const int64_t step = (hi - lo + kWarp - 1) / kWarp, probe = lo + lane_id() * step;
      const bool before = probe < hi && (probe == lo || begin(probe) <= r);
      const int64_t next = lo + (__popc(__ballot_sync(kFull, before)) - 1) * step;
      hi = min(hi, next + step);
      lo = next;
    }
    return lo;
  }
};

struct GroupArgs {
  const void* x;
  const void* grad_out;
  void* out;
  Frames frames;
  int channels, groups, group_channels;
  const float* weight;
  const float* bias;
  float* mean;  // forward: outputs
  float* rstd;
  float eps;
  int activation;
  float* grad_weight;
  float* grad_bias;
  float2* affine;  // backward, frame kernel: [CTAs][channels] sum dz, sum dz xhat
  // chunks
  int64_t chunk_rows, chunks;
  int64_t apply_rows;   // of a CTA of the result
  float2* partial;      // [chunks + frames][channels]
  float2* sums;         // backward: [frames][groups] mean(d), mean(d xhat)
};

// VEC values at p (global or shared memory).
template <int VEC>
__device__ __forceinline__ void load_vec(const float* p, float (&v)[VEC]) {
  if constexpr (VEC == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
    v[0] = *p;
  }
}
template <int VEC>
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&v)[VEC]) {
  if constexpr (VEC == 4) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
  } else {
    v[0] = __bfloat162float(*p);
  }
}
template <int VEC>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  else __stcs(p, v[0]);
}
template <int VEC>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
    __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<uint2*>(h));
  } else {
    p[0] = __float2bfloat16_rn(v[0]);
  }
}

// VEC values as loaded.
template <typename T, int VEC>
struct Raw {
  static constexpr int kBytes = VEC * sizeof(T);
  using Word = std::conditional_t<
      kBytes == 16, uint4,
      std::conditional_t<kBytes == 8, uint2,
                         std::conditional_t<kBytes == 4, uint32_t, uint16_t>>>;
  Word word;
  __device__ __forceinline__ void load(const T* p) { word = *reinterpret_cast<const Word*>(p); }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    load_vec<VEC>(reinterpret_cast<const T*>(&word), v);
  }
};

// A thread's rows of one or two arrays, kRows at a time (of BYTES together).
template <typename T, int VEC, bool TWO, int BYTES>
struct Rows {
  static constexpr int kRows =
      VEC == 1 ? 8 : BYTES / static_cast<int>(VEC * sizeof(T) * (TWO ? 2 : 1));
  Raw<T, VEC> a[kRows], b[TWO ? kRows : 1];
  __device__ __forceinline__ void load(const T*& pa, const T*& pb, int64_t step) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      a[j].load(pa);
      pa += step;
      if constexpr (TWO) {
        b[j].load(pb);
        pb += step;
      }
    }
  }
  // The last 1 .. kRows - 1 rows.
  __device__ __forceinline__ void load(const T* pa, const T* pb, int64_t step, int count) {
#pragma unroll
    for (int j = 0; j < kRows - 1; ++j) {
      if (j >= count) continue;
      a[j].load(pa);
      pa += step;
      if constexpr (TWO) {
        b[j].load(pb);
        pb += step;
      }
    }
  }
};

// use(a, b) for n rows of a thread in order, the next kRows requested before
// the last ones are used, which batch(rows, their number) sees first.
template <typename T, int VEC, bool TWO, int BYTES, typename Batch, typename Use>
__device__ __forceinline__ void each_row(const T* pa, const T* pb, int64_t step, int64_t n,
                                         Batch batch, Use use) {
  using RowsT = Rows<T, VEC, TWO, BYTES>;
  constexpr int kRows = RowsT::kRows;
  const int rest = static_cast<int>(n % kRows);
  auto apply = [&](const RowsT& rows, int j) {
    float a[VEC], b[VEC];
    rows.a[j].get(a);
    rows.b[TWO ? j : 0].get(b);
    use(a, b);
  };
  RowsT next;
  if (n >= kRows) next.load(pa, pb, step);
  else next.load(pa, pb, step, rest);
  for (; n >= kRows; n -= kRows) {
    const RowsT now = next;
    if (n >= 2 * kRows) next.load(pa, pb, step);
    else next.load(pa, pb, step, rest);
    batch(now, kRows);
#pragma unroll
    for (int j = 0; j < kRows; ++j) apply(now, j);
  }
  if (rest > 0) batch(next, rest);
#pragma unroll
  for (int j = 0; j < kRows - 1; ++j)
    if (j < rest) apply(next, j);
}

// 1 / (1 + exp(-z)) by the approximate exponential and reciprocal (2 units
// and 1 unit in the last place; the product adds |z| 2^-24).
__device__ __forceinline__ float sigmoid(float z) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2_ftz(z * -1.4426950408889634f)));
  return r;
}
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == BYSJ_ACT_NONE) return z;
  const float s = sigmoid(z);
  return ACT == BYSJ_ACT_SILU ? z * s : s;
}
template <int ACT>
__device__ __forceinline__ float activate_grad(float z) {
  if constexpr (ACT == BYSJ_ACT_NONE) return 1.0f;
  const float s = sigmoid(z), t = 1.0f - s;
  return ACT == BYSJ_ACT_SILU ? fmaf(s * t, z, s) : s * t;
}

// Threads over a tile of channels: cv vectors side by side, ty rows at a time.
template <int VEC, int THREADS>
struct Tile {
  int c0, width, ty, ry, c;  // c: first channel of this thread
  bool on;
  __device__ Tile(int begin, int channels) {
    c0 = begin;
    width = min(channels - begin, THREADS * VEC);
    const int cv = width / VEC;
    ty = THREADS / cv;
    ry = threadIdx.x / cv;
    c = begin + (threadIdx.x % cv) * VEC;
    on = ry < ty;
  }
};

// Per channel of a thread: xhat = x r + o, z = xhat w + b (forward: z = x r + o
// with weight and bias in r and o), and dx = dz k - xhat s - t.
template <int VEC>
struct Columns {
  float r[VEC], o[VEC], w[VEC], b[VEC], k[VEC], s[VEC], t[VEC];
  template <bool BACKWARD>
  __device__ __forceinline__ void set(const GroupArgs& a, int c, int i, float mean, float rstd,
                                      float2 sums) {
    w[i] = a.weight ? __ldg(a.weight + c) : 1.0f;
    b[i] = a.bias ? __ldg(a.bias + c) : 0.0f;
    if constexpr (BACKWARD) {
      r[i] = rstd;
      o[i] = -mean * rstd;
      k[i] = rstd * w[i];
      s[i] = rstd * sums.y;
      t[i] = rstd * sums.x;
    } else {
      r[i] = rstd * w[i];
      o[i] = fmaf(-mean, r[i], b[i]);
    }
  }
};

// Number, mean and sum of squares about the mean of some values.  Joining two of
// them only adds squares, so no digits cancel wherever the means lie.  The part is
// an approximate quotient, of which a difference of means is taken; beside nothing
// it is 1 or 0 exactly, so that a mean keeps its bits.
struct Moments {
  float n = 0.0f, mean = 0.0f, m2 = 0.0f;
  __device__ __forceinline__ void join(const Moments& o) {
    const float sum = n + o.n, d = o.mean - mean;
    const float part = o.n > 0.0f ? (n > 0.0f ? __fdividef(o.n, sum) : 1.0f) : 0.0f;
    mean = fmaf(d, part, mean);
    m2 += fmaf(d * (n * part), d, o.m2);  // d first: its square may overflow beside n = 0
    n = sum;
  }
};

// Adds n terms term(i) for i = first, first + step, ...: eight at a time, the
// eights then to the sum, so that the rounding grows with n / 8 + 8 terms.
template <typename Term>
__device__ __forceinline__ void add_terms(int first, int n, int step, float& s1, float& s2,
                                          Term term) {
  for (int i = first; i < n;) {
    float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u, i += step) {
      if (i >= n) continue;
      const float2 v = term(i);
      t1 += v.x;
      t2 += v.y;
    }
    s1 += t1;
    s2 += t2;
  }
}

// Terms of a thread's inner sums before they join the outer ones; a multiple of
// the rows that each_row takes at a time.
constexpr int kInner = 64;

// Channel sums over a slab's rows into chan[] (forward: mean and the sum of
// squares about it; backward: sum dz, sum dz xhat).  Ends synchronised.
//
// Forward: a thread sums kInner rows at a time about a pivot, the mean of its rows
// before them; they move the pivot by off = s1 / rows so far, and what squares about
// the old pivot exceed those about the new one is s1 off.  The first pivot is the
// mean of the first batch of rows (of four or eight: an outlier there enters it by a
// quarter or less, so that squares cancel by a factor of 5 at most).
template <typename T, int VEC, int THREADS, bool BACKWARD, int ACT>
__device__ __forceinline__ void column_stats(const Tile<VEC, THREADS>& t, const T* x, const T* dy,
                                             int64_t rows, int channels, const Columns<VEC>& q,
                                             float* scratch, float2* level, float2* chan) {
  if (t.on) {
    float s1[VEC], s2[VEC], o1[VEC], o2[VEC];  // inner and outer sums; forward: o1 is the pivot
#pragma unroll
    for (int i = 0; i < VEC; ++i) s1[i] = s2[i] = o1[i] = o2[i] = 0.0f;
    const int64_t step = static_cast<int64_t>(t.ty) * channels;
    const T* px = x + t.ry * static_cast<int64_t>(channels) + t.c;
    const T* pg = dy + t.ry * static_cast<int64_t>(channels) + t.c;
    const int64_t n = rows > t.ry ? (rows - t.ry + t.ty - 1) / t.ty : 0;  // of this thread
    int terms = 0;      // of the inner sums
    float done = 0.0f;  // forward: rows of the outer ones
    auto flush = [&] {
      done += static_cast<float>(terms);
      const float inv = 1.0f / done;
      terms = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if constexpr (BACKWARD) {
          o1[i] += s1[i];
          o2[i] += s2[i];
        } else {
          const float off = s1[i] * inv;
          o1[i] += off;
          o2[i] += fmaf(-s1[i], off, s2[i]);
        }
        s1[i] = s2[i] = 0.0f;
      }
    };
    auto batch = [&](const auto& now, int count) {
      if constexpr (BACKWARD) return;
      if (terms == 0) {  // the first of all
#pragma unroll
        for (int j = 0; j < now.kRows; ++j) {
          if (j >= count) continue;
          float v[VEC];
          now.a[j].get(v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) o1[i] += v[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) o1[i] /= static_cast<float>(count);
      }
      if (terms == kInner) flush();
      terms += count;
    };
    each_row<T, VEC, BACKWARD, BACKWARD ? 128 : 64>(px, pg, step, n, batch, [&](const float(&v)[VEC], const float(&g)[VEC]) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if constexpr (BACKWARD) {
          const float xhat = fmaf(v[i], q.r[i], q.o[i]);
          const float dz = g[i] * activate_grad<ACT>(fmaf(xhat, q.w[i], q.b[i]));
          s1[i] += dz;
          s2[i] = fmaf(dz, xhat, s2[i]);
        } else {
          const float d = v[i] - o1[i];
          s1[i] += d;
          s2[i] = fmaf(d, d, s2[i]);
        }
      }
      if constexpr (BACKWARD)
        if (++terms == kInner) flush();
    });
    if (terms > 0) flush();
    float* place = scratch + t.ry * t.width + t.c - t.c0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      place[i] = o1[i];
      place[THREADS * VEC + i] = o2[i];
    }
  }
  __syncthreads();
  // THREADS / width parts of the rows side by side, then the parts in order
  const int parts = t.width < THREADS ? THREADS / t.width : 1;
  const int share = (t.ty + parts - 1) / parts;
  // forward: rows of thread row r, and of all before it
  const int64_t each = rows / t.ty;
  const int more = static_cast<int>(rows - each * t.ty);
  const auto before = [&](int r) { return each * r + min(r, more); };
  for (int i = threadIdx.x; i < parts * t.width; i += THREADS) {
    const int part = i / t.width, c = i - part * t.width;
    const int end = min((part + 1) * share, t.ty);
    float2 v;
    if constexpr (BACKWARD) {
      v = make_float2(0.0f, 0.0f);
      for (int r = part * share; r < end; ++r) {
        v.x += scratch[r * t.width + c];
        v.y += scratch[THREADS * VEC + r * t.width + c];
      }
    } else {
      Moments m;
      for (int r = part * share; r < end; ++r)
        m.join({static_cast<float>(r < more ? each + 1 : each), scratch[r * t.width + c],
                scratch[THREADS * VEC + r * t.width + c]});
      v = make_float2(m.mean, m.m2);
    }
    if (parts > 1) level[i] = v;
    else chan[t.c0 + c] = v;
  }
  __syncthreads();
  if (parts > 1) {
    for (int c = threadIdx.x; c < t.width; c += THREADS) {
      if constexpr (BACKWARD) {
        float2 v = make_float2(0.0f, 0.0f);
        for (int part = 0; part < parts; ++part) {
          v.x += level[part * t.width + c].x;
          v.y += level[part * t.width + c].y;
        }
        chan[t.c0 + c] = v;
      } else {
        Moments m;
        for (int part = 0; part < parts; ++part) {
          const float2 v = level[part * t.width + c];
          const int from = min(part * share, t.ty), to = min(from + share, t.ty);
          m.join({static_cast<float>(before(to) - before(from)), v.x, v.y});
        }
        chan[t.c0 + c] = make_float2(m.mean, m.m2);
      }
    }
    __syncthreads();
  }
}

// One warp: the channels of group g joined.  Forward: mean and sum of squares
// about it of `rows` rows; backward: sum d and sum d xhat, d = dz w.
template <bool BACKWARD>
__device__ __forceinline__ float2 join_channels(const GroupArgs& a, const float2* chan, int g,
                                                int64_t rows) {
  const int lane = lane_id(), c0 = g * a.group_channels;
  float s1 = 0.0f, s2 = 0.0f;
  for (int c = c0 + lane; c < c0 + a.group_channels; c += kWarp) {
    const float w = BACKWARD && a.weight ? __ldg(a.weight + c) : 1.0f;
    s1 += w * chan[c].x;
    s2 += w * chan[c].y;
  }
  s1 = xor_sum(s1, 1);
  if constexpr (!BACKWARD) {
    s1 /= static_cast<float>(a.group_channels);
    for (int c = c0 + lane; c < c0 + a.group_channels; c += kWarp) {
      const float d = chan[c].x - s1;
      s2 += static_cast<float>(rows) * d * d;
    }
  }
  s2 = xor_sum(s2, 1);
  return make_float2(s1, s2);
}

// y or dx of `rows` rows, the last first.  The result is written past L1 with
// the first place in line to leave L2: nothing here reads it again.
template <typename T, int VEC, int THREADS, bool BACKWARD, int ACT>
__device__ __forceinline__ void apply_rows(const Tile<VEC, THREADS>& t, const T* x, const T* dy,
                                           T* out, int64_t rows, int channels,
                                           const Columns<VEC>& q) {
  if (!t.on) return;
  const int64_t step = static_cast<int64_t>(t.ty) * channels;
  const int64_t n = rows > t.ry ? (rows - t.ry + t.ty - 1) / t.ty : 0;
  if (n == 0) return;
  const int64_t at = (t.ry + (n - 1) * t.ty) * static_cast<int64_t>(channels) + t.c;
  const T* px = x + at;
  const T* pg = dy + at;
  T* py = out + at;
  const auto nothing = [](const auto&, int) {};
  each_row<T, VEC, BACKWARD, 64>(px, pg, -step, n, nothing, [&](const float(&v)[VEC], const float(&g)[VEC]) {
    float y[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (BACKWARD) {
        const float xhat = fmaf(v[i], q.r[i], q.o[i]);
        const float dz = g[i] * activate_grad<ACT>(fmaf(xhat, q.w[i], q.b[i]));
        y[i] = fmaf(dz, q.k[i], -fmaf(xhat, q.s[i], q.t[i]));
      } else {
        y[i] = activate<ACT>(fmaf(v[i], q.r[i], q.o[i]));
      }
    }
    store_vec<VEC>(py, y);
    py -= step;
  });
}

// Shared memory of both kernels: level [THREADS], scratch [2][THREADS * VEC],
// chan [channels], stats [groups] and, backward, the affine sums [channels].
template <int VEC, int THREADS>
__host__ __device__ constexpr size_t fixed_smem(int channels, int groups, bool backward) {
  return sizeof(float) * 2 * THREADS * VEC + sizeof(float2) * THREADS +
         sizeof(float2) * (static_cast<size_t>(channels) * (backward ? 2 : 1) + groups);
}

template <int VEC, int THREADS>
struct Smem {
  float2* level;
  float* scratch;
  float2 *chan, *stats, *affine;
  __device__ Smem(unsigned char* base, int channels, int groups) {
    level = reinterpret_cast<float2*>(base);
    scratch = reinterpret_cast<float*>(level + THREADS);
    chan = reinterpret_cast<float2*>(scratch + 2 * THREADS * VEC);
    stats = chan + channels;
    affine = stats + groups;
  }
};

// A variance that is not a number (an infinity among the values) stays one: the mean
// alone may be infinite, which an activation turns into a number.
__device__ __forceinline__ float2 moments(const GroupArgs& a, float mean, float variance) {
  return make_float2(mean, 1.0f / sqrtf((variance < 0.0f ? 0.0f : variance) + a.eps));
}

// Statistics of one tile's thread: mean and rstd of frame b, and its sums.
template <int VEC, int THREADS, bool BACKWARD>
__device__ __forceinline__ void set_columns(const GroupArgs& a, const Tile<VEC, THREADS>& t,
                                            int64_t b, const float2* sums, Columns<VEC>& q) {
  if (!t.on) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int64_t at = b * a.groups + (t.c + i) / a.group_channels;
    q.template set<BACKWARD>(a, t.c + i, i, a.mean[at], a.rstd[at],
                             sums ? sums[at] : make_float2(0.0f, 0.0f));
  }
}

// Whole frames, one CTA each, in steps of the grid.
template <typename T, int VEC, int THREADS, bool BACKWARD, int ACT>
__global__ void __launch_bounds__(THREADS) group_frame_kernel(GroupArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  const Smem<VEC, THREADS> m(smem, a.channels, a.groups);
  const int warp = threadIdx.x / kWarp;
  if constexpr (BACKWARD)
    for (int c = threadIdx.x; c < a.channels; c += THREADS) m.affine[c] = make_float2(0.f, 0.f);
  for (int64_t b = blockIdx.x; b < a.frames.count; b += gridDim.x) {
    const int64_t begin = a.frames.begin(b), rows = a.frames.begin(b + 1) - begin;
    const T* x = static_cast<const T*>(a.x) + begin * a.channels;
    const T* dy = static_cast<const T*>(BACKWARD ? a.grad_out : a.x) + begin * a.channels;
    T* out = static_cast<T*>(a.out) + begin * a.channels;
    if (rows <= 0) {
      if constexpr (!BACKWARD)
        for (int g = threadIdx.x; g < a.groups; g += THREADS)
          a.mean[b * a.groups + g] = a.rstd[b * a.groups + g] = 0.0f;
      continue;
    }
    __syncthreads();
    Columns<VEC> q;
    for (int c0 = 0; c0 < a.channels; c0 += THREADS * VEC) {
      const Tile<VEC, THREADS> t(c0, a.channels);
      if constexpr (BACKWARD) set_columns<VEC, THREADS, true>(a, t, b, nullptr, q);
      column_stats<T, VEC, THREADS, BACKWARD, ACT>(t, x, dy, rows, a.channels, q, m.scratch,
                                                   m.level, m.chan);
    }
    for (int g = warp; g < a.groups; g += THREADS / kWarp) {
      const float2 v = join_channels<BACKWARD>(a, m.chan, g, rows);
      const float n = static_cast<float>(rows) * static_cast<float>(a.group_channels);
      if (lane_id() == 0) {
        if constexpr (BACKWARD) {
          m.stats[g] = make_float2(v.x / n, v.y / n);
        } else {
          m.stats[g] = moments(a, v.x, v.y / n);
          a.mean[b * a.groups + g] = m.stats[g].x;
          a.rstd[b * a.groups + g] = m.stats[g].y;
        }
      }
    }
    if constexpr (BACKWARD)
      for (int c = threadIdx.x; c < a.channels; c += THREADS) {
        m.affine[c].x += m.chan[c].x;
        m.affine[c].y += m.chan[c].y;
      }
    __syncthreads();
    for (int c0 = 0; c0 < a.channels; c0 += THREADS * VEC) {
      const Tile<VEC, THREADS> t(c0, a.channels);
      if (t.on) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int g = (t.c + i) / a.group_channels;
          const float2 v = m.stats[g];
          if constexpr (BACKWARD)
            q.template set<true>(a, t.c + i, i, a.mean[b * a.groups + g],
                                 a.rstd[b * a.groups + g], v);
          else q.template set<false>(a, t.c + i, i, v.x, v.y, v);
        }
      }
      apply_rows<T, VEC, THREADS, BACKWARD, ACT>(t, x, dy, out, rows, a.channels, q);
    }
  }
  if constexpr (BACKWARD) {
    __syncthreads();
    for (int c = threadIdx.x; c < a.channels; c += THREADS)
      a.affine[static_cast<int64_t>(blockIdx.x) * a.channels + c] = m.affine[c];
  }
}

// ---- chunks of all frames ---------------------------------------------------

__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = xor_sum(v, 1);
  __syncthreads();
  if (lane_id() == 0) scratch[threadIdx.x / kWarp] = v;
  __syncthreads();
  float total = 0.0f;
  for (int i = 0; i < kWarpsPerBlock; ++i) total += scratch[i];
  return total;
}

// Sums rows of channel pairs in a fixed order into the gradients of weight
// and bias: 8 channels a CTA, 32 rows at a time.
constexpr int kAffineChannels = 8;

__device__ __forceinline__ void affine_grad(const GroupArgs& a, int tile, const float2* rows,
                                            int64_t count) {
  constexpr int kAbreast = kBlock / kAffineChannels;
  __shared__ float2 part[kAbreast][kAffineChannels];
  const int rank = threadIdx.x / kAffineChannels, lane = threadIdx.x % kAffineChannels;
  const int c = tile * kAffineChannels + lane;
  float s1 = 0.0f, s2 = 0.0f;
  if (c < a.channels)
    add_terms(rank, static_cast<int>(count), kAbreast, s1, s2,
              [&](int i) { return rows[static_cast<int64_t>(i) * a.channels + c]; });
  part[rank][lane] = make_float2(s1, s2);
  __syncthreads();
  if (rank == 0 && c < a.channels) {
    for (int i = 1; i < kAbreast; ++i) {
      s1 += part[i][lane].x;
      s2 += part[i][lane].y;
    }
    if (a.grad_bias) a.grad_bias[c] = s1;
    if (a.grad_weight) a.grad_weight[c] = s2;
  }
}

constexpr int kChunkThreads = 256;
static_assert(kChunkThreads == kBlock, "affine_grad and block_sum run in both kernels");

// The pieces of a frame: what each of its channels left there.
struct Pieces {
  const GroupArgs& a;
  int64_t r0, r1, first;
  int count;
  float n;                // values of a group
  const float2* partial;  // the first piece's channels
  __device__ Pieces(const GroupArgs& args, int64_t b) : a(args) {
    r0 = a.frames.begin(b);
    r1 = a.frames.begin(b + 1);
    first = r0 / a.chunk_rows;
    count = static_cast<int>((r1 - 1) / a.chunk_rows - first) + 1;
    n = static_cast<float>(r1 - r0) * static_cast<float>(a.group_channels);
    partial = a.partial + (first + b) * a.channels;
  }
  __device__ __forceinline__ float2 at(int p, int c) const {
    return partial[static_cast<int64_t>(p) * a.channels + c];
  }
  // Forward: pieces from, from + step, ... of channel c joined to m, eight at a time.
  __device__ void join(int c, int from, int step, Moments& m) const {
    for (int p = from; p < count;) {
      Moments eight;
#pragma unroll
      for (int u = 0; u < 8; ++u, p += step) {
        if (p >= count) continue;
        const int64_t chunk = first + p;
        const float rows = static_cast<float>(
            static_cast<int>(min((chunk + 1) * a.chunk_rows, r1) - max(chunk * a.chunk_rows, r0)));
        const float2 v = at(p, c);
        eight.join({rows, v.x, v.y});
      }
      m.join(eight);
    }
  }
  // Backward: their sums of d and d xhat, d = dz w.
  __device__ void add(int c, int from, int step, float& s1, float& s2) const {
    const float w = a.weight ? __ldg(a.weight + c) : 1.0f;
    add_terms(from, count, step, s1, s2, [&](int p) {
      const float2 v = at(p, c);
      return make_float2(v.x * w, v.y * w);
    });
  }
};

// The block's moments joined in a fixed order; on thread 0.
template <int LANES>
__device__ __forceinline__ void lanes_join(Moments& v) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d >>= 1)
    v.join({__shfl_down_sync(kFull, v.n, d), __shfl_down_sync(kFull, v.mean, d),
            __shfl_down_sync(kFull, v.m2, d)});
}
__device__ __forceinline__ Moments block_join(Moments v, Moments* scratch) {
  lanes_join<kWarp>(v);
  __syncthreads();
  if (lane_id() == 0) scratch[threadIdx.x / kWarp] = v;
  __syncthreads();
  if (threadIdx.x < kWarp) {
    v = threadIdx.x < kWarpsPerBlock ? scratch[threadIdx.x] : Moments();
    lanes_join<kWarpsPerBlock>(v);
  }
  return v;
}

// CTAs of the kernel below on one SM.  In the statistics of the backward pass
// more rows in flight for each thread do better than a third CTA (180001 x 96
// float32: 35 us against 44; 393216 x 128 bfloat16: 53 - 54 us either way); in the
// results it is the other way round (bfloat16: 59 us against 71).
__host__ __device__ constexpr int chunk_ctas(bool backward, bool apply) {
  return backward ? (apply ? 3 : 2) : 4;
}

// APPLY: y or dx; otherwise the pieces' numbers.  One chunk a CTA.
template <typename T, int VEC, bool BACKWARD, int ACT, bool APPLY>
__global__ void __launch_bounds__(kChunkThreads, chunk_ctas(BACKWARD, APPLY))
    group_chunk_kernel(GroupArgs a) {
  constexpr int kThreads = kChunkThreads;
  extern __shared__ __align__(128) unsigned char smem[];
  const Smem<VEC, kThreads> m(smem, a.channels, a.groups);
  const int C = a.channels;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(BACKWARD ? a.grad_out : a.x);
  const int64_t chunk = blockIdx.x;
  const int64_t chunk_rows = APPLY ? a.apply_rows : a.chunk_rows;
  const int64_t r0 = chunk * chunk_rows, r1 = min(r0 + chunk_rows, a.frames.rows);
  const int64_t b0 = a.frames.of_row(r0);
  auto no_piece = [&](int64_t from, int64_t to) {  // numbers [from, to)
    if constexpr (!APPLY)
      for (int64_t i = from * C + threadIdx.x; i < to * C; i += kThreads)
        a.partial[i] = make_float2(0.0f, 0.0f);
  };
  no_piece(chunk == 0 ? 0 : chunk + b0, chunk + b0);
  int64_t lo = r0, b = b0;
  for (; b < a.frames.count && lo < r1; ++b) {
    const int64_t hi = min(a.frames.begin(b + 1), r1);
    if (hi <= lo) {
      no_piece(chunk + b, chunk + b + 1);
      continue;
    }
    for (int c0 = 0; c0 < C; c0 += kThreads * VEC) {
      const Tile<VEC, kThreads> t(c0, C);
      Columns<VEC> q;
      if constexpr (APPLY) {
        set_columns<VEC, kThreads, BACKWARD>(a, t, b, BACKWARD ? a.sums : nullptr, q);
        apply_rows<T, VEC, kThreads, BACKWARD, ACT>(t, x + lo * C, dy + lo * C,
                                                    static_cast<T*>(a.out) + lo * C, hi - lo, C,
                                                    q);
      } else {
        if constexpr (BACKWARD) set_columns<VEC, kThreads, true>(a, t, b, nullptr, q);
        column_stats<T, VEC, kThreads, BACKWARD, ACT>(t, x + lo * C, dy + lo * C, hi - lo, C, q,
                                                      m.scratch, m.level, m.chan);
        for (int c = threadIdx.x; c < t.width; c += kThreads)
          a.partial[(chunk + b) * C + c0 + c] = m.chan[c0 + c];
        __syncthreads();
      }
    }
    lo = hi;
  }
  if constexpr (!APPLY) {  // up to the next chunk's first number
    const int64_t next =
        r1 < a.frames.rows ? chunk + 1 + a.frames.of_row(r1) : a.chunks + a.frames.count;
    no_piece(chunk + b, next);
  }
}

__global__ void __launch_bounds__(kBlock) group_affine_kernel(GroupArgs a, int ctas) {
  affine_grad(a, blockIdx.x, a.affine, ctas);
}

// Joins the pieces of one frame and group a CTA, in steps of the grid; the
// first `tiles` CTAs take the gradients of weight and bias, from all pieces.
template <bool BACKWARD>
__global__ void __launch_bounds__(kBlock) group_join_kernel(GroupArgs a, int tiles) {
  using Part = std::conditional_t<BACKWARD, float, Moments>;
  __shared__ __align__(16) unsigned char memory[kWarpsPerBlock * sizeof(Part)];
  Part* scratch = reinterpret_cast<Part*>(memory);
  if constexpr (BACKWARD) {
    if (static_cast<int>(blockIdx.x) < tiles) {
      affine_grad(a, blockIdx.x, a.partial, a.chunks + a.frames.count);
      return;
    }
  }
  const int64_t units = a.frames.count * a.groups;
  for (int64_t unit = blockIdx.x - tiles; unit < units; unit += gridDim.x - tiles) {
    const int64_t b = unit / a.groups;
    const int g = static_cast<int>(unit % a.groups), c0 = g * a.group_channels;
    if (a.frames.begin(b + 1) <= a.frames.begin(b)) {
      if constexpr (!BACKWARD)
        if (threadIdx.x == 0) a.mean[unit] = a.rstd[unit] = 0.0f;
      continue;
    }
    const Pieces pieces(a, b);
    const int width = a.group_channels < kBlock ? a.group_channels : kBlock;
    const int lanes = kBlock / width, rank = threadIdx.x / width;
    const int c_first = rank < lanes ? threadIdx.x % width : a.group_channels;
    if constexpr (BACKWARD) {
      float s1 = 0.0f, s2 = 0.0f;
      for (int c = c_first; c < a.group_channels; c += width) pieces.add(c0 + c, rank, lanes, s1, s2);
      s1 = block_sum(s1, scratch);
      s2 = block_sum(s2, scratch);
      if (threadIdx.x == 0) a.sums[unit] = make_float2(s1 / pieces.n, s2 / pieces.n);
    } else {
      Moments m;
      for (int c = c_first; c < a.group_channels; c += width) pieces.join(c0 + c, rank, lanes, m);
      m = block_join(m, scratch);
      if (threadIdx.x == 0) {
        const float2 v = moments(a, m.mean, m.m2 / pieces.n);
        a.mean[unit] = v.x;
        a.rstd[unit] = v.y;
      }
    }
  }
}

// ---- host -------------------------------------------------------------------

// A frame of at most this many bytes is one CTA's work: two passes over it
// through L1 cost less than a meeting of CTAs.
constexpr int64_t kSmallFrame = 64 * 1024;

struct Plan {
  bool chunked = false;
  int ctas = 1;
  int threads = 256;  // frame kernel
  int64_t chunk_rows = 1, chunks = 0, apply_rows = 1;
};

// Depends on sizes only, so that the workspace size follows from them; `item`
// is the element size.
Plan make_plan(int64_t rows, int64_t channels, int64_t frames, int item, bool backward) {
  Plan p;
  const int64_t sms = current_device_info().sm_count;
  const int64_t row_bytes = channels * item;
  p.chunked = rows * row_bytes / (frames > 0 ? frames : 1) > kSmallFrame;
  // few frames: more threads for each
  p.threads = frames <= sms ? 512 : 256;
  p.ctas = static_cast<int>(frames < sms * 4 ? frames : sms * 4);
  if (!p.chunked) return p;
  // one chunk for each resident CTA, of 16 KB at least
  const int64_t least = (16384 + row_bytes - 1) / row_bytes;
  const auto cut = [&](bool apply) {
    const int64_t ctas = sms * chunk_ctas(backward, apply), each = (rows + ctas - 1) / ctas;
    return each < least ? least : each;
  };
  p.chunk_rows = cut(false);
  p.apply_rows = cut(true);
  p.chunks = (rows + p.chunk_rows - 1) / p.chunk_rows;
  return p;
}

size_t carve_workspace(GroupArgs& a, const Plan& p, void* workspace, bool backward) {
  Carver carve(workspace);
  if (p.chunked) {
    a.partial =
        carve.take<float2>(static_cast<size_t>(p.chunks + a.frames.count) * a.channels);
    if (backward) a.sums = carve.take<float2>(static_cast<size_t>(a.frames.count) * a.groups);
  } else if (backward) {
    a.affine = carve.take<float2>(static_cast<size_t>(p.ctas) * a.channels);
  }
  return carve.need;
}

void set_sizes(GroupArgs& a, int64_t rows, int64_t channels, int64_t groups,
               const int64_t* offsets, int64_t frames, int64_t inner) {
  a.frames.offsets = offsets;
  a.frames.count = frames;
  a.frames.inner = inner;
  a.frames.rows = rows;
  a.channels = static_cast<int>(channels);
  a.groups = static_cast<int>(groups);
  a.group_channels = static_cast<int>(channels / groups);
}

// The larger of what the plans of either element size need.
size_t workspace_size(int64_t rows, int64_t channels, int64_t groups, int64_t frames,
                      bool backward) {
  if (rows <= 0 || channels <= 0 || groups <= 0 || frames <= 0) return 0;
  size_t most = 0;
  for (int item : {2, 4}) {
    GroupArgs a{};
    set_sizes(a, rows, channels, groups, nullptr, frames, 1);
    const size_t need = carve_workspace(a, make_plan(rows, channels, frames, item, backward),
                                        nullptr, backward);
    if (need > most) most = need;
  }
  return most;
}

using GroupKernel = void (*)(GroupArgs);

int launch_one(GroupKernel kernel, const char* name, unsigned ctas, int threads, size_t smem,
               const GroupArgs& a, cudaStream_t s) {
  const int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (st) return st;
  kernel<<<ctas, threads, smem, s>>>(a);
  return launch_check(name);
}

template <typename T, int VEC, bool BACKWARD, int ACT>
int launch_act(const GroupArgs& a, const Plan& p, cudaStream_t s) {
  const bool affine = BACKWARD && (a.grad_weight != nullptr || a.grad_bias != nullptr);
  const int tiles = affine ? (a.channels + kAffineChannels - 1) / kAffineChannels : 0;
  if (!p.chunked) {
    const int st =
        p.threads == 512
            ? launch_one(group_frame_kernel<T, VEC, 512, BACKWARD, ACT>, "group_frame_kernel",
                         p.ctas, 512, fixed_smem<VEC, 512>(a.channels, a.groups, BACKWARD), a, s)
            : launch_one(group_frame_kernel<T, VEC, 256, BACKWARD, ACT>, "group_frame_kernel",
                         p.ctas, 256, fixed_smem<VEC, 256>(a.channels, a.groups, BACKWARD), a, s);
    if (st || !affine) return st;
    group_affine_kernel<<<tiles, kBlock, 0, s>>>(a, p.ctas);
    return launch_check("group_affine_kernel");
  }
  const unsigned chunks = static_cast<unsigned>(p.chunks);
  const size_t smem = fixed_smem<VEC, kChunkThreads>(a.channels, a.groups, BACKWARD);
  int st = launch_one(group_chunk_kernel<T, VEC, BACKWARD, ACT, false>, "group_chunk_kernel",
                      chunks, kChunkThreads, smem, a, s);
  if (st) return st;
  const int64_t units = a.frames.count * a.groups;
  group_join_kernel<BACKWARD>
      <<<static_cast<unsigned>((units < 65536 ? units : 65536) + tiles), kBlock, 0, s>>>(a, tiles);
  st = launch_check("group_join_kernel");
  if (st) return st;
  return launch_one(group_chunk_kernel<T, VEC, BACKWARD, ACT, true>, "group_chunk_kernel",
                    static_cast<unsigned>((a.frames.rows + p.apply_rows - 1) / p.apply_rows),
                    kChunkThreads, 0, a, s);
}

template <typename T, int VEC, bool BACKWARD>
int launch_vec(const GroupArgs& a, const Plan& p, cudaStream_t s) {
  switch (a.activation) {
    case BYSJ_ACT_SILU: return launch_act<T, VEC, BACKWARD, BYSJ_ACT_SILU>(a, p, s);
    case BYSJ_ACT_SIGMOID: return launch_act<T, VEC, BACKWARD, BYSJ_ACT_SIGMOID>(a, p, s);
    default: return launch_act<T, VEC, BACKWARD, BYSJ_ACT_NONE>(a, p, s);
  }
}

template <typename T, bool BACKWARD>
int launch(GroupArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  // four channels a thread: 16 or 8 bytes
  constexpr uintptr_t kAlign = 4 * sizeof(T) - 1;
  const uintptr_t all = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out) |
                        (BACKWARD ? reinterpret_cast<uintptr_t>(a.grad_out) : 0);
  const bool vectors = a.channels % 4 == 0 && (all & kAlign) == 0;
  const Plan p = make_plan(a.frames.rows, a.channels, a.frames.count, sizeof(T), BACKWARD);
  const size_t need = carve_workspace(a, p, workspace, BACKWARD);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(BYSJ_ERR_WORKSPACE, "group norm: workspace of %zu bytes needed, %zu given", need,
                workspace_bytes);
  a.chunk_rows = p.chunk_rows;
  a.chunks = p.chunks;
  a.apply_rows = p.apply_rows;
  return vectors ? launch_vec<T, 4, BACKWARD>(a, p, s) : launch_vec<T, 1, BACKWARD>(a, p, s);
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
  if (channels > BYSJ_GROUP_NORM_MAX_CHANNELS)
    return fail(BYSJ_ERR_UNSUPPORTED, "%s: at most %d channels", name,
                BYSJ_GROUP_NORM_MAX_CHANNELS);
  return BYSJ_OK;
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
  set_sizes(a, rows, channels, groups, offsets, frames, inner);
  a.x = x;
  a.out = y;
  a.weight = weight;
  a.bias = bias;
  a.mean = mean;
  a.rstd = rstd;
  a.eps = eps;
  a.activation = activation;
  return dtype == BYSJ_F32 ? launch<float, false>(a, workspace, workspace_bytes, s)
                           : launch<__nv_bfloat16, false>(a, workspace, workspace_bytes, s);
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
  set_sizes(a, rows, channels, groups, offsets, frames, inner);
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
  return dtype == BYSJ_F32 ? launch<float, true>(a, workspace, workspace_bytes, s)
                           : launch<__nv_bfloat16, true>(a, workspace, workspace_bytes, s);
}

}  // extern "C"
