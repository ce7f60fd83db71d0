// The fitting step over a list of tensors: the global gradient norm, clipping by it, and the Adam
// update with decoupled weight decay.
//
//   norm = sqrt(sum g^2) or max |g| over every entry of every tensor,
//   coef = min(1, max_norm / (norm + 1e-6)),   g' = coef g,
//   m = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2,
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps).
// The squares are added in fp64 and in an order fixed by the sizes and alignments alone: the norm neither
// overflows for entries past 1.8e19 nor changes from run to run.  A non-finite norm goes through
// the formula (NaN everywhere for a NaN, zeros and NaN for an infinity).
//
// The tensors are cut into chunks, one a warp at a time; a table says which tensor a chunk belongs
// to.  A short table travels as a kernel parameter, a long one is written to the workspace by launches
// that carry it in pieces as THEIR parameters: no host buffer is read after the call returns, so
// the call can be captured in a graph.
//
// Memory bounds the work: one read for the norm, then a read and a write.  Few entries are done by
// one cluster, whose CTAs join their sums over distributed shared memory, in one launch (one family of
// 1,023 columns 5 us).  Else a first kernel leaves a partial sum a CTA, and the second, whose CTAs each
// join them, goes through every warp's chunks backwards, from what the first left in L2.
// Measured, call after call: 201 M bf16 entries 81 + 124 us, 5.0 and 6.5 TB/s (76 and 99 % of the copy
// bandwidth); Adam over 104 M fp32 entries 83 + 507 us, 5.0 and 5.7 TB/s (76 and 87 %), with bf16 gradients 45 + 540
// us (4.6 and 5.0 TB/s).  The norm's pass also writes back what the call before left dirty in L2: with L2 flushed it
// takes 64, 69 and 39 us (6.3, 6.0 and 5.3 TB/s).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kb_common.cuh"
#include "kb_solver.h"

namespace {

using namespace kb;

constexpr float kClipEps = 1e-6f;
constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 256;
// CTAs of the norm kernel and of the second one, all resident: more bytes under way help a kernel that
// only reads, and fewer streams one that also writes (with L2 flushed, 201 M bf16: norm 66 us with 5 an SM, 72
// with 8; clip 127 with 3, 137 with 2; Adam 104 M: 500 us with 3, 514 with 4).
constexpr int kNormCtas = 148 * 5;
constexpr int kApplyCtas = 148 * 3;
constexpr int kClusterThreads = 512;  // a CTA of the one-cluster form
constexpr int kClusterChunks = 128;   // chunks it takes at most: one a warp
constexpr int kInline = 32;           // tensors whose table travels with the kernel itself
constexpr int kPieceBytes = 32000;    // records of one table-writing launch,
constexpr int kSmallPiece = 96;       // and how many a last one has (a launch costs the host 6 us with the former,
                                      // under 3 with the latter)

struct alignas(16) Entry {
  void* p[4];         // clip: source, destination; Adam: gradient, parameter, m, v
  long long n;
  int chunk0;         // first chunk of this tensor
  short dtype;        // of p[0]: 0 fp32, 1 bf16, 2 fp16
  signed char shift;  // entries from the 16-byte boundary at or before p[0] to p[0]; -1: the arrays'
                      // boundaries do not fall together and entries go one by one
};

struct Table {
  Entry e[kInline];
  const Entry* far;  // the table in the workspace (NULL: e)
  int n, n_chunks, log2_chunk;
};

// An entry without the arrays that clipping has not.
struct alignas(16) SlimEntry {
  void* p[2];
  long long n;
  int chunk0;
  short dtype;
  signed char shift;
};
__device__ __forceinline__ Entry expand(const Entry& e) { return e; }
__device__ __forceinline__ Entry expand(const SlimEntry& s) {
  return Entry{{s.p[0], s.p[1], nullptr, nullptr}, s.n, s.chunk0, s.dtype, s.shift};
}

template <typename R, int N = kPieceBytes / (int)sizeof(R)>
struct Piece {
  static constexpr int kRecords = N;
  R e[N];
  Entry* dst;
  int n;
};
static_assert(sizeof(Entry) == 48 && sizeof(SlimEntry) == 32 && sizeof(Piece<Entry>) <= 32764 &&
                  sizeof(Piece<SlimEntry>) <= 32764,
              "kernel parameters end at 32,764 bytes");

template <typename P>
__global__ void write_table_kernel(const __grid_constant__ P piece) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < piece.n) piece.dst[i] = expand(piece.e[i]);
}

// The last entry whose first chunk is <= chunk, by a warp: 32 probes a round.
__device__ __forceinline__ int find_entry(const Entry* e, int n, int chunk, int lane) {
  int lo = 0;
  while (n > 1) {  // the entry is among e[lo .. lo + n)
    const int step = (n + 31) / 32, i = lane * step;
    const unsigned below = __ballot_sync(kAll, i < n && e[lo + i].chunk0 <= chunk);
    const int k = 31 - __clz(below);  // probe 0 always is
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

// 16 bytes of a tensor as floats, and back; the entry-wise forms.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
  static __device__ __forceinline__ void decode(const uint4& q, float* f) {
    f[0] = __uint_as_float(q.x); f[1] = __uint_as_float(q.y); f[2] = __uint_as_float(q.z); f[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 encode(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ void decode(const uint4& q, float* f) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 encode(const float* f) {
    uint4 q;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    return q;
  }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void decode(const uint4& q, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 v = __half22float2(h[j]);
      f[2 * j] = v.x;
      f[2 * j + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 encode(const float* f) {
    uint4 q;
    __half2* h = reinterpret_cast<__half2*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
    return q;
  }
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ double max_nan(double a, double b) { return (a != a) ? a : ((b != b) ? b : fmax(a, b)); }

// What a warp gathers of the norm.  The squares of a vector are added in fp32 (at most 8 terms, 2^-21 of
// their sum) and join the fp64 total with one conversion; a sum that is not well inside fp32's range
// is formed again in fp64.
struct Gathered {
  double squares = 0.0;
  float largest = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float* f, bool square) {
    if (square) {
      float q = f[0] * f[0];
#pragma unroll
      for (int i = 1; i < N; ++i) q = fmaf(f[i], f[i], q);
      if (q > 1e-30f && q < 1e37f) {
        squares += (double)q;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) squares = fma((double)f[i], (double)f[i], squares);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) largest = max_nan(largest, fabsf(f[i]));
    }
  }
  __device__ __forceinline__ double value(bool square) const { return square ? squares : (double)largest; }
};

// Goes through chunk k of a tensor by a warp.  f(whole, i, m): entries [i, i + m) of the tensor, m <= N,
// in the first m places; whole: the vector at entry i may be moved as 16 bytes (m = N).
template <int N, typename F>
__device__ __forceinline__ void for_chunk(const Entry& e, long long k, int log2_chunk, int lane, const F& f) {
  const int shift = e.shift < 0 ? 0 : e.shift;
  const long long begin = (k << log2_chunk) - shift;  // the tensor's entry at the chunk's first place
  const long long end = min(e.n, begin + (1ll << log2_chunk));
#pragma unroll 4
  for (long long i = begin + lane * N; i < end; i += 32 * N) {
    if (e.shift >= 0 && i >= 0 && i + N <= e.n) {
      f(true, i, N);
    } else {
      const long long a = i < 0 ? 0 : i;
      f(false, a, (int)(min(e.n, i + N) - a));
    }
  }
}

// (Plain loads: the same kernel may write there later.)
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, bool whole, long long i, int m, float* f) {
  constexpr int N = Vec<T>::N;
  if (whole) {
    Vec<T>::decode(*reinterpret_cast<const uint4*>(p + i), f);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = j < m ? Vec<T>::up(p[i + j]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, bool whole, long long i, int m, const float* f) {
  constexpr int N = Vec<T>::N;
  if (whole) {
    *reinterpret_cast<uint4*>(p + i) = Vec<T>::encode(f);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < m) p[i + j] = Vec<T>::down(f[j]);
  }
}

// Whether chunk k is made of whole vectors only, `steps` a lane, in groups of U: *begin its first entry.
template <int N, int U>
__device__ __forceinline__ bool whole_chunk(const Entry& e, long long k, int log2_chunk, long long* begin) {
  *begin = (k << log2_chunk) - e.shift;
  return e.shift >= 0 && *begin >= 0 && *begin + (1ll << log2_chunk) <= e.n && (1 << log2_chunk) % (32 * N * U) == 0;
}

template <typename T>
__device__ __forceinline__ void gather_chunk(const Entry& e, long long k, int log2_chunk, bool square, int lane,
                                             Gathered& to) {
  constexpr int N = Vec<T>::N, U = 4;
  const T* p = static_cast<const T*>(e.p[0]);
  long long begin;
  if (whole_chunk<N, U>(e, k, log2_chunk, &begin)) {
    const uint4* v = reinterpret_cast<const uint4*>(p + begin) + lane;
    for (int i = 0; i < (1 << log2_chunk) / N; i += 32 * U) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = v[i + 32 * u];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        Vec<T>::decode(q[u], f);
        to.add<N>(f, square);
      }
    }
    return;
  }
  for_chunk<N>(e, k, log2_chunk, lane, [&](bool whole, long long i, int m) {
    float f[N];
    load_vec(p, whole, i, m, f);
    to.add<N>(f, square);
  });
}

// The clip coefficient as head * tail: fp32 holds one below 2^-126 with few bits or not at all, and beside
// entries of 1e38 the product is an ordinary number.  tail is 1, or 2^-64 for what is below 2^-100.
struct Coef {
  float head = 1.f, tail = 1.f;
  __device__ __forceinline__ float operator*(float x) const { return (x * head) * tail; }
};

// The second pass reads the gradient for the last time and what else it moves but once: all of it is
// marked to leave L2 first (ld.cs, st.cs), so that the gradient's end stays there until it is reached.
template <typename T>
__device__ __forceinline__ void clip_chunk(const Entry& e, long long k, int log2_chunk, Coef coef, int lane) {
  constexpr int N = Vec<T>::N, U = 4;
  const T* p = static_cast<const T*>(e.p[0]);
  T* o = static_cast<T*>(e.p[1]);
  long long begin;
  if (whole_chunk<N, U>(e, k, log2_chunk, &begin)) {
    const uint4* v = reinterpret_cast<const uint4*>(p + begin) + lane;
    uint4* w = reinterpret_cast<uint4*>(o + begin) + lane;
    for (int i = 0; i < (1 << log2_chunk) / N; i += 32 * U) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = __ldcs(v + i + 32 * u);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        Vec<T>::decode(q[u], f);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = coef * f[j];
        __stcs(w + i + 32 * u, Vec<T>::encode(f));
      }
    }
    return;
  }
  for_chunk<N>(e, k, log2_chunk, lane, [&](bool whole, long long i, int m) {
    float f[N];
    load_vec(p, whole, i, m, f);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = coef * f[j];
    store_vec(o, whole, i, m, f);
  });
}

struct AdamArgs {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, decay, size, inv_root;
};

__device__ __forceinline__ void adam_entry(const AdamArgs& k, float g, float& p, float& m, float& v) {
  m = fmaf(k.one_minus_beta1, g, k.beta1 * m);
  v = fmaf(k.one_minus_beta2 * g, g, k.beta2 * v);  // g * g is out of range from 1.8e19 on
  // the decay is a term of the update, not a factor 1 - lr wd, which fp32 holds to 6e-8 of 1:
  // 0.6 % of a decay of 1e-5
  p -= fmaf(k.decay, p, k.size * (m / fmaf(sqrtf(v), k.inv_root, k.eps)));
}

template <typename T>
__device__ __forceinline__ void adam_chunk(const Entry& e, long long k, int log2_chunk, Coef coef, const AdamArgs& a,
                                           int lane) {
  constexpr int N = Vec<T>::N;
  const T* gp = static_cast<const T*>(e.p[0]);
  float *pp = static_cast<float*>(e.p[1]), *mp = static_cast<float*>(e.p[2]), *vp = static_cast<float*>(e.p[3]);
  constexpr int U = N == 4 ? 2 : 1;
  long long begin;
  if (whole_chunk<N, U>(e, k, log2_chunk, &begin)) {
    for (long long i = begin + lane * N; i < begin + (1ll << log2_chunk); i += 32 * N * U) {
      uint4 gq[U], pq[U * N / 4], mq[U * N / 4], vq[U * N / 4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long at = i + 32 * N * u;
        gq[u] = __ldcs(reinterpret_cast<const uint4*>(gp + at));
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
          pq[u * N / 4 + j] = __ldcs(reinterpret_cast<const uint4*>(pp + at) + j);
          mq[u * N / 4 + j] = __ldcs(reinterpret_cast<const uint4*>(mp + at) + j);
          vq[u * N / 4 + j] = __ldcs(reinterpret_cast<const uint4*>(vp + at) + j);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long at = i + 32 * N * u;
        float g[N];
        Vec<T>::decode(gq[u], g);
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
          float p[4], m[4], v[4];
          Vec<float>::decode(pq[u * N / 4 + j], p);
          Vec<float>::decode(mq[u * N / 4 + j], m);
          Vec<float>::decode(vq[u * N / 4 + j], v);
#pragma unroll
          for (int l = 0; l < 4; ++l) adam_entry(a, coef * g[4 * j + l], p[l], m[l], v[l]);
          __stcs(reinterpret_cast<uint4*>(pp + at) + j, Vec<float>::encode(p));
          __stcs(reinterpret_cast<uint4*>(mp + at) + j, Vec<float>::encode(m));
          __stcs(reinterpret_cast<uint4*>(vp + at) + j, Vec<float>::encode(v));
        }
      }
    }
    return;
  }
  for_chunk<N>(e, k, log2_chunk, lane, [&](bool whole, long long i, int n) {
    float g[N];
    load_vec(gp, whole, i, n, g);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) adam_entry(a, coef * g[j], pp[i + j], mp[i + j], vp[i + j]);
  });
}

// The chunks of warp w of n: w, w + n, ..., so that the grid moves through memory as one front
// (a stretch of chunks a warp: clip 201 M bf16 227 us, Adam 104 M entries 695).
struct Share {
  int w, n;
};
__device__ __forceinline__ const Entry* entries(const Table& t) { return t.far ? t.far : t.e; }

// The entry of a chunk, looked for from the one before.
__device__ __forceinline__ int entry_of(const Table& t, const Entry* e, int at, int chunk, int lane) {
  if (at >= 0 && e[at].chunk0 <= chunk && (at + 1 == t.n || e[at + 1].chunk0 > chunk)) return at;
  return find_entry(e, t.n, chunk, lane);
}

__device__ __forceinline__ double gather_share(const Table& t, Share w, bool square, int lane) {
  Gathered to;
  const Entry* e = entries(t);
  int at = -1;
  for (int c = w.w; c < t.n_chunks; c += w.n) {
    at = entry_of(t, e, at, c, lane);
    const Entry& x = e[at];
    const long long k = c - x.chunk0;
    if (x.dtype == 0) gather_chunk<float>(x, k, t.log2_chunk, square, lane, to);
    else if (x.dtype == 1) gather_chunk<__nv_bfloat16>(x, k, t.log2_chunk, square, lane, to);
    else gather_chunk<__half>(x, k, t.log2_chunk, square, lane, to);
  }
  return to.value(square);
}

// Backwards, so that what the norm's pass read last comes first.
template <bool ADAM>
__device__ __forceinline__ void apply_share(const Table& t, Share w, Coef coef, const AdamArgs& a, int lane) {
  if (w.w >= t.n_chunks) return;
  const Entry* e = entries(t);
  int at = -1;
  for (int c = w.w + (t.n_chunks - 1 - w.w) / w.n * w.n; c >= 0; c -= w.n) {
    at = entry_of(t, e, at, c, lane);
    const Entry& x = e[at];
    const long long k = c - x.chunk0;
    if constexpr (ADAM) {
      if (x.dtype == 0) adam_chunk<float>(x, k, t.log2_chunk, coef, a, lane);
      else if (x.dtype == 1) adam_chunk<__nv_bfloat16>(x, k, t.log2_chunk, coef, a, lane);
      else adam_chunk<__half>(x, k, t.log2_chunk, coef, a, lane);
    } else {
      if (x.dtype == 0) clip_chunk<float>(x, k, t.log2_chunk, coef, lane);
      else if (x.dtype == 1) clip_chunk<__nv_bfloat16>(x, k, t.log2_chunk, coef, lane);
      else clip_chunk<__half>(x, k, t.log2_chunk, coef, lane);
    }
  }
}

// Sum (or maximum) over the block, in a fixed order; every thread gets it.
__device__ __forceinline__ double block_join(double v, bool square, double* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double y = __shfl_xor_sync(kAll, v, o);
    v = square ? v + y : max_nan(v, y);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  double r = 0.0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) r = square ? r + scratch[w] : max_nan(r, scratch[w]);
  return r;
}

__device__ __forceinline__ Coef clip_coefficient(double norm, double max_norm) {
  const double c = max_norm / (norm + (double)kClipEps);
  if (c >= 1.0) return Coef{};
  if (c < 0x1p-100) return Coef{(float)(c * 0x1p64), 0x1p-64f};
  return Coef{(float)c, 1.f};  // a NaN stays
}

struct Step {
  bool square, apply, clip;  // which norm; whether anything is written; whether the norm is wanted at all
  double max_norm;
  float* norm_out;
  AdamArgs adam;
};

__global__ void __launch_bounds__(kThreads, 5) norm_partials_kernel(const __grid_constant__ Table t, bool square,
                                                                  double* partials) {
  __shared__ double scratch[kThreads / 32];
  const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Share r{(int)blockIdx.x * (kThreads / 32) + wid, (int)gridDim.x * (kThreads / 32)};
  const double v = block_join(gather_share(t, r, square, lane), square, scratch);
  if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

template <bool ADAM>
__global__ void __launch_bounds__(kThreads, 3) apply_kernel(const __grid_constant__ Table t, const Step s,
                                                          const double* partials, int n_partials) {
  __shared__ double scratch[kThreads / 32];
  Coef coef;
  if (s.clip) {  // every CTA joins the partials itself, in the same order
    double v = 0.0;
    for (int i = threadIdx.x; i < n_partials; i += kThreads) v = s.square ? v + partials[i] : max_nan(v, partials[i]);
    v = block_join(v, s.square, scratch);
    const double norm = s.square ? sqrt(v) : v;
    if (blockIdx.x == 0 && threadIdx.x == 0) *s.norm_out = (float)norm;
    coef = clip_coefficient(norm, s.max_norm);
  }
  if (!s.apply) return;
  const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  apply_share<ADAM>(t, Share{(int)blockIdx.x * (kThreads / 32) + wid, (int)gridDim.x * (kThreads / 32)}, coef, s.adam,
                    lane);
}

// All of it by one cluster.
template <bool ADAM>
__global__ void __launch_bounds__(kClusterThreads, 1) cluster_kernel(const __grid_constant__ Table t, const Step s) {
  namespace cg = cooperative_groups;
  __shared__ double scratch[kClusterThreads / 32];
  __shared__ double mine;
  cg::cluster_group cluster = cg::this_cluster();
  const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const Share r{cta * (kClusterThreads / 32) + wid, n_ctas * (kClusterThreads / 32)};
  Coef coef;
  if (s.clip) {
    double v = block_join(gather_share(t, r, s.square, lane), s.square, scratch);
    if (n_ctas > 1) {
      if (threadIdx.x == 0) mine = v;
      cluster.sync();
      v = 0.0;
      for (int o = 0; o < n_ctas; ++o) {
        const double y = *cluster.map_shared_rank(&mine, o);
        v = s.square ? v + y : max_nan(v, y);
      }
    }
    const double norm = s.square ? sqrt(v) : v;
    if (cta == 0 && threadIdx.x == 0) *s.norm_out = (float)norm;
    coef = clip_coefficient(norm, s.max_norm);
  }
  if (s.apply) apply_share<ADAM>(t, r, coef, s.adam, lane);
  if (n_ctas > 1 && s.clip) cluster.sync();  // no CTA leaves while its sum is read
}

long long align16(long long x) { return (x + 15) & ~15ll; }
long long table_offset() { return align16((long long)kNormCtas * sizeof(double)); }
long long workspace_bytes(int n) { return table_offset() + (n > kInline ? (long long)n * (long long)sizeof(Entry) : 0); }

template <typename P>
cudaError_t write_piece(const P& piece, cudaStream_t st) {
  write_table_kernel<P><<<(piece.n + 127) / 128, 128, 0, st>>>(piece);
  return cudaGetLastError();
}

void shorten(const Entry& e, Entry& r) { r = e; }
void shorten(const Entry& e, SlimEntry& r) { r = SlimEntry{{e.p[0], e.p[1]}, e.n, e.chunk0, e.dtype, e.shift}; }

// Fills the table from the HOST lists (tensors without entries are left out) and, past kInline
// tensors, enqueues its writing to the workspace in records R.  ptrs[j] may be NULL (no such array).
template <typename R>
int make_table(Table& t, const long long* const ptrs[4], const long long* counts, const int* dtypes, int n, char* ws,
               cudaStream_t st) {
  static const int log2_size[3] = {2, 1, 1};
  const auto log2_of = [&](int i, int j) {  // bytes of an entry of array j of tensor i: Adam's p, m, v are fp32
    return j == 0 || ptrs[2] == nullptr ? log2_size[dtypes[i]] : 2;
  };
  long long total = 0;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0 || dtypes[i] < 0 || dtypes[i] > 2) return KB_ERR_ARG;
    total += counts[i];
    for (int j = 0; j < 4 && counts[i] > 0; ++j) {
      if (ptrs[j] == nullptr) continue;
      if (ptrs[j][i] == 0 || (ptrs[j][i] & ((1 << log2_of(i, j)) - 1)) != 0) return KB_ERR_ARG;
    }
  }
  // chunks of 2,048 entries, smaller ones where that leaves warps without one
  t.log2_chunk = 11;
  while (t.log2_chunk > 8 && (total >> t.log2_chunk) < kNormCtas * (kThreads / 32)) --t.log2_chunk;
  const bool far = n > kInline;
  Entry* dst = reinterpret_cast<Entry*>(ws + table_offset());
  Piece<R> piece;
  piece.n = 0;
  long long chunks = 0;
  t.n = 0;
  for (int i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    Entry e{};
    // entries past the 16-byte boundary: address mod 16 in entries, which has to be the same in all arrays
    int shift = (int)(ptrs[0][i] & 15) >> log2_of(i, 0);
    for (int j = 0; j < 4; ++j) {
      if (ptrs[j] == nullptr) continue;
      const int l = log2_of(i, j);
      if (shift >= 0 && ((int)(ptrs[j][i] & 15) >> l) != (shift & ((16 >> l) - 1))) shift = -1;
      e.p[j] = reinterpret_cast<void*>(ptrs[j][i]);
    }
    e.n = counts[i];
    e.dtype = (short)dtypes[i];
    e.shift = (signed char)shift;
    e.chunk0 = (int)chunks;
    chunks += (counts[i] + (shift > 0 ? shift : 0) + (1ll << t.log2_chunk) - 1) >> t.log2_chunk;
    if (chunks > 0x7fffffffll) return KB_ERR_SIZE;
    ++t.n;
    if (!far) {
      t.e[t.n - 1] = e;
      continue;
    }
    shorten(e, piece.e[piece.n++]);
    if (piece.n == piece.kRecords) {
      piece.dst = dst;
      if (write_piece(piece, st) != cudaSuccess) return KB_ERR_LAUNCH;
      dst += piece.n;
      piece.n = 0;
    }
  }
  for (int i = 0; i < piece.n;) {
    cudaError_t e;
    if (piece.n - i > 3 * kSmallPiece) {  // i = 0
      piece.dst = dst;
      e = write_piece(piece, st);
      i = piece.n;
    } else {
      Piece<R, kSmallPiece> small;
      small.dst = dst + i;
      small.n = piece.n - i < kSmallPiece ? piece.n - i : kSmallPiece;
      for (int j = 0; j < small.n; ++j) small.e[j] = piece.e[i + j];
      e = write_piece(small, st);
      i += small.n;
    }
    if (e != cudaSuccess) return KB_ERR_LAUNCH;
  }
  t.far = far ? reinterpret_cast<const Entry*>(ws + table_offset()) : nullptr;
  t.n_chunks = (int)chunks;
  return KB_OK;
}

template <bool ADAM>
int launch_step(const Table& t, const Step& s, void* ws, cudaStream_t st) {
  if (t.n_chunks <= kClusterChunks) {
    unsigned ctas = 1;
    while (ctas < 8 && (int)ctas * (kClusterThreads / 32) < t.n_chunks) ctas *= 2;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kClusterThreads);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, cluster_kernel<ADAM>, t, s) == cudaSuccess ? KB_OK : KB_ERR_LAUNCH;
  }
  double* partials = static_cast<double*>(ws);
  const int wanted = (t.n_chunks + kThreads / 32 - 1) / (kThreads / 32);
  const int norm_ctas = wanted < kNormCtas ? wanted : kNormCtas, ctas = wanted < kApplyCtas ? wanted : kApplyCtas;
  if (s.clip) norm_partials_kernel<<<norm_ctas, kThreads, 0, st>>>(t, s.square, partials);
  apply_kernel<ADAM><<<s.apply ? ctas : 1, kThreads, 0, st>>>(t, s, partials, norm_ctas);
  return cudaGetLastError() == cudaSuccess ? KB_OK : KB_ERR_LAUNCH;
}

}  // namespace

extern "C" int kb_fit_workspace(int n_tensors, long long* bytes_out) {
  if (n_tensors < 0 || !bytes_out) return KB_ERR_ARG;
  *bytes_out = workspace_bytes(n_tensors);
  return KB_OK;
}

extern "C" int kb_clip_gradients(const long long* grads, const long long* outs, const long long* counts,
                                 const int* dtypes, int n_tensors, int kind, double max_norm, float* norm_out,
                                 void* ws, long long ws_bytes, void* stream) {
  if (n_tensors < 0 || (kind != 0 && kind != 2) || !norm_out || !ws || ws_bytes < workspace_bytes(n_tensors) ||
      (n_tensors > 0 && (!grads || !counts || !dtypes)) || (outs && !(max_norm >= 0.0)) ||
      !on_boundary(ws, 16) || !on_boundary(norm_out, 4))
    return KB_ERR_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  Table t{};
  const long long* const ptrs[4] = {grads, outs, nullptr, nullptr};
  const int status = make_table<SlimEntry>(t, ptrs, counts, dtypes, n_tensors, static_cast<char*>(ws), st);
  if (status != KB_OK) return status;
  const Step s{kind == 2, outs != nullptr, true, max_norm, norm_out, AdamArgs{}};
  return launch_step<false>(t, s, ws, st);
}

extern "C" int kb_adam_step(const long long* params, const long long* grads, const long long* exp_avg,
                            const long long* exp_avg_sq, const long long* counts, const int* grad_dtypes,
                            int n_tensors, double lr, double beta1, double beta2, double eps, double weight_decay,
                            double correction1, double correction2, int kind, double max_norm, float* norm_out,
                            void* ws, long long ws_bytes, void* stream) {
  if (n_tensors < 0 || (kind != -1 && kind != 0 && kind != 2) || !ws || ws_bytes < workspace_bytes(n_tensors) ||
      (kind >= 0 && (!norm_out || !(max_norm >= 0.0))) || !(correction1 > 0.0) || !(correction2 > 0.0) ||
      (n_tensors > 0 && (!params || !grads || !exp_avg || !exp_avg_sq || !counts || !grad_dtypes)) ||
      !on_boundary(ws, 16) || !on_boundary(norm_out, 4))
    return KB_ERR_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  Table t{};
  const long long* const ptrs[4] = {grads, params, exp_avg, exp_avg_sq};
  const int status = make_table<Entry>(t, ptrs, counts, grad_dtypes, n_tensors, static_cast<char*>(ws), st);
  if (status != KB_OK) return status;
  const AdamArgs k{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps,
                   (float)(lr * weight_decay), (float)(lr / correction1), (float)(1.0 / sqrt(correction2))};
  return launch_step<true>(t, Step{kind == 2, true, kind >= 0, max_norm, norm_out, k}, ws, st);
}
