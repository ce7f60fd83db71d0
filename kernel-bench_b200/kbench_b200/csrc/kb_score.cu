// Row scores: what a row of log values over S columns (a clade's species placements; any row of
// unnormalised log probabilities) says about its columns, and the gradient of that.
//
// For base u in {2, e}, a row x with m = max x and Sigma = sum_s u^(x_s - m):
//   log_mass = m + log_u Sigma,   log p_s = (x_s - m) - log_u Sigma,
//   entropy  = -sum p_s log_u p_s = log_u Sigma - (sum u^(x_s - m) (x_s - m)) / Sigma,
//   top      = the k largest entries, equal ones by the lower column.
// The row's log probabilities are formed from m and Sigma, never from log_mass: a row's offset is
// hundreds of binades, where log_mass has lost the bits that tell Sigma apart.
// Everything is evaluated in base 2 (z = (x - m) * scale, scale = 1 or log2 e) in fp32.
// -inf is an impossible column (p = 0); a row with nothing else has log_mass = -inf, entropy 0 and
// no gradient; a row that holds NaN or +inf scores NaN and has no top columns.
//
// Reading a row once.  A warp reads batches of 128 16-byte vectors (four a lane, the next batch's
// loads issued before this one is worked on); a lane keeps the running (m, Sigma, T), T = sum 2^z z,
// rescaled when its maximum grows, and adds a batch's terms apart first, so that the chain of fp32
// additions is short.  For the top list a lane only leaves its largest entry of every group of batches
// in shared memory on the way.  The k-th largest of the 32 lanes' maxima is a lower bound tau of the
// row's k-th entry (k lanes have one at least that large, and few entries are), so afterwards the
// groups whose maximum reaches tau -- about k of them -- are read again, from L1 or L2, and their
// entries from tau up become candidates, cut back to the best k by counting the larger ones of each.
// Rows start at any entry: vectors are taken at 16-byte boundaries, and the entries of the first
// and the last that are not the row's count as -inf.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>

#include "kb_common.cuh"
#include "kb_solver.h"

namespace {

using namespace kb;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFarBelow = -1.0e4f;  // finite stand-in for z = -inf beside its weight 2^z = 0

// Values as unsigned integers in the same order (-0 as +0), and back.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned b = __float_as_uint(x + 0.0f);  // -0 ties with +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(unsigned o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ unsigned ordered16(unsigned b) {
  if (b == 0x8000u) b = 0u;
  return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
}
__device__ __forceinline__ unsigned short unordered16(unsigned o) {
  return (unsigned short)((o & 0x8000u) ? (o & 0x7fffu) : (~o & 0xffffu));
}

// 16 bytes of a row as floats, and back.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr unsigned kNegInf = 0xff800000u;  // a word of -inf
  static __device__ __forceinline__ void decode(const uint4& q, float* f) {
    f[0] = __uint_as_float(q.x); f[1] = __uint_as_float(q.y); f[2] = __uint_as_float(q.z); f[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 encode(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
  static __device__ __forceinline__ unsigned order(float x) { return ordered(x); }
  static __device__ __forceinline__ float value(unsigned o) { return unordered(o); }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr unsigned kNegInf = 0xff80ff80u;
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
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ unsigned order(float x) { return ordered16(__float_as_uint(x) >> 16); }
  static __device__ __forceinline__ float value(unsigned o) { return __uint_as_float((unsigned)unordered16(o) << 16); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr unsigned kNegInf = 0xfc00fc00u;
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
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ unsigned order(float x) { return ordered16(__half_as_ushort(__float2half_rn(x))); }
  static __device__ __forceinline__ float value(unsigned o) { return __half2float(__ushort_as_half(unordered16(o))); }
};

constexpr unsigned kAll = 0xffffffffu;
constexpr int kWarps = 8;             // warps of a CTA
constexpr int kRowWarps = 2;          // and of one whose warps take a row each
constexpr int kSteps = 4;             // vectors of a lane in a batch
constexpr int kBatch = 32 * kSteps;   // vectors of a batch
constexpr int kGroups = 32;           // groups of batches a lane keeps the maximum of
constexpr int kCand = 64;             // candidates a warp holds: the best 32 and a ballot's 32

// A row's vectors: `vec` starts at the 16-byte boundary at or before the row, `shift` entries early.
template <typename T>
struct Row {
  const T* x;
  const uint4* vec;
  int S, shift, n_vec, n_batch;
  __device__ __forceinline__ Row(const T* x_, int S_) : x(x_), S(S_) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x_);
    shift = (int)((a & 15) / sizeof(T));
    vec = reinterpret_cast<const uint4*>(a & ~(uintptr_t)15);
    n_vec = S > 0 ? (S + shift + Vec<T>::N - 1) / Vec<T>::N : 0;
    n_batch = (n_vec + kBatch - 1) / kBatch;
  }
  // Vector v; one past the row holds -inf.
  __device__ __forceinline__ uint4 load_one(int v) const {
    constexpr unsigned w = Vec<T>::kNegInf;
    return v < n_vec ? __ldg(vec + v) : make_uint4(w, w, w, w);
  }
  // A lane's vectors of batch b.
  __device__ __forceinline__ void load(uint4 (&q)[kSteps], int b, int lane) const {
#pragma unroll
    for (int u = 0; u < kSteps; ++u) q[u] = load_one((b * kSteps + u) * 32 + lane);
  }
  __device__ __forceinline__ int column(int b, int i, int lane) const {
    return ((b * kSteps + i / Vec<T>::N) * 32 + lane) * Vec<T>::N - shift + i % Vec<T>::N;
  }
  // Their entries; those of the row's first and last vector that are not the row's count as -inf.
  __device__ __forceinline__ void decode(const uint4 (&q)[kSteps], float (&f)[kSteps * Vec<T>::N], int b,
                                         int lane) const {
#pragma unroll
    for (int u = 0; u < kSteps; ++u) Vec<T>::decode(q[u], f + u * Vec<T>::N);
    if (b == 0 || b == n_batch - 1) {
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int v = (b * kSteps + u) * 32 + lane;
        if (v == 0 || v == n_vec - 1) {
#pragma unroll
          for (int e = 0; e < Vec<T>::N; ++e)
            if ((unsigned)(v * Vec<T>::N - shift + e) >= (unsigned)S) f[u * Vec<T>::N + e] = neg_inf();
        }
      }
    }
  }
};

// 2^z with results below 2^-126 as 0: one instruction, where the form that keeps subnormal results takes
// four (bf16 rows of 4,095 without a top list: 76 -> 68 us for 32,071).  Beside a sum of at least 1
// such a weight is nothing.
__device__ __forceinline__ float weight(float z) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(z));
  return y;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
  return m;
}
// -2^z z for z <= 0, given w = 2^z.  The value is in [0, 0.54), so saturation to [0, 1] leaves it as it
// is, and makes the NaN of an impossible column's 0 * inf the 0 it stands for.
__device__ __forceinline__ float weighted(float w, float z) {
  float y;
  asm("mul.rn.sat.f32 %0, %1, %2;" : "=f"(y) : "f"(w), "f"(-z));
  return y;
}

// Running sums relative to a maximum: Sigma = sum 2^z, T = sum 2^z z, z = (x - m) scale.
struct Sums {
  float m, sum, wsum;
};
// The factor of sums taken relative to a smaller maximum.  A difference below kFarBelow (from -inf
// or from a type's lowest value) has factor 0 and stays finite beside it; a NaN sum survives.
__device__ __forceinline__ void rebase(Sums& a, float m, float scale) {
  const float d = fmaxf((a.m - m) * scale, kFarBelow), r = weight(d);
  a.wsum = r * fmaf(d, a.sum, a.wsum);
  a.sum *= r;
  a.m = m;
}
// The maximum of the lanes' values (redux; a NaN is passed over).
__device__ __forceinline__ float lanes_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ Sums warp_join(Sums a, float scale) {
  const float m = lanes_max(a.m);
  rebase(a, safe_max(m), scale);
  a.m = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.sum += __shfl_xor_sync(kAll, a.sum, o);
    a.wsum += __shfl_xor_sync(kAll, a.wsum, o);
  }
  return a;
}

// Two floats side by side: the packed fp32 instructions take half the issue slots of two plain ones.
struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair pack(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ void unpack(Pair p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p.v)); }
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair c;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair c;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}

// Keys whose unsigned order is the order of the top list: by value, then by the lower column.
typedef unsigned long long Key;
__device__ __forceinline__ Key top_key(float x, int col) { return ((Key)ordered(x) << 32) | (0xffffffffu - (unsigned)col); }
__device__ __forceinline__ float key_value(Key k) { return unordered((unsigned)(k >> 32)); }
__device__ __forceinline__ int key_column(Key k) { return (int)(0xffffffffu - (unsigned)k); }

// Keeps the best k of a warp's `count` <= kCand keys, in order: a key's place is the number of larger
// keys.  Returns how many are kept.
__device__ __noinline__ int cut_keys(Key* keys, int count, int k, int lane) {
  __syncwarp();
  const Key a = lane < count ? keys[lane] : 0;
  int ra = 0;
  if (count <= 32) {
#pragma unroll 4
    for (int j = 0; j < count; ++j) ra += keys[j] > a;
    __syncwarp();
  } else {
    const Key b = lane + 32 < count ? keys[lane + 32] : 0;
    int rb = 0;
    for (int j = 0; j < count; ++j) {
      const Key y = keys[j];
      ra += y > a;
      rb += y > b;
    }
    __syncwarp();
    if (lane + 32 < count && rb < k) keys[rb] = b;
  }
  if (lane < count && ra < k) keys[ra] = a;
  __syncwarp();
  return count < k ? count : k;
}

// The k-th largest of the values of each G lanes, k <= G, by sorting them (a bitonic network: 15
// exchanges for 32).
template <int G = 32>
__device__ __forceinline__ float kth_of_lanes(float v, int k, int lane) {
#pragma unroll
  for (int size = 2; size <= G; size *= 2) {
#pragma unroll
    for (int o = size / 2; o > 0; o >>= 1) {
      // falling where `size` is clear in the lane (everywhere, at last): the lower lane keeps the larger
      const bool larger = ((lane & size & (G - 1)) == 0) == ((lane & o) == 0);
      const float y = __shfl_xor_sync(kAll, v, o);
      v = larger ? fmaxf(v, y) : fminf(v, y);
    }
  }
  return __shfl_sync(kAll, v, (threadIdx.x & 31 & ~(G - 1)) + k - 1);
}

// Adds the lanes' marked entries (bit i of `mine`: column col_of(i)) to a warp's candidates, one a lane
// at a time; least: the k-th key of the last cut, below which nothing is in the list.
template <typename T, typename ColumnOf>
__device__ __forceinline__ void take(const T* x, int S, unsigned mine, const ColumnOf& col_of, Key* keys, int& count,
                                     Key& least, int k, int lane) {
  while (__any_sync(kAll, mine != 0)) {
    const int col = mine ? col_of(__ffs(mine) - 1) : -1;
    mine &= mine - 1;
    bool c = (unsigned)col < (unsigned)S;
    const Key key = c ? top_key(Vec<T>::up(x[col]), col) : 0;
    c = c && key > least;
    unsigned in = __ballot_sync(kAll, c);
    if (count + __popc(in) > kCand) {
      count = cut_keys(keys, count, k, lane);  // count was above kCand - 32 >= k
      least = keys[k - 1];
      c = c && key > least;
      in = __ballot_sync(kAll, c);
    }
    if (c) keys[count + __popc(in & ((1u << lane) - 1))] = key;
    count += __popc(in);
  }
}

// The bound that candidates are taken from: all finite entries where fewer than k lanes have one.
__device__ __forceinline__ float finite_bound(float tau) { return fmaxf(tau, -3.402823466e38f); }

// Completes a list that the finite entries of columns [c0, c1) leave short: the lowest of the other
// columns, all -inf.  Of any 64 columns at least 64 - 31 are among those.
template <typename T>
__device__ __forceinline__ void fill(const T* x, int c0, int c1, Key* keys, int& count, int k, int lane) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (count >= k) return;
    const int col = c0 + j * 32 + lane;
    const bool c = col < c1 && is_neg_inf(Vec<T>::up(x[col]));
    const unsigned in = __ballot_sync(kAll, c);
    if (c) keys[count + __popc(in & ((1u << lane) - 1))] = top_key(neg_inf(), col);
    count += __popc(in);
  }
}

// The best k of a row's batches [b0, b1), all of them at least tau, to keys[0 .. returned) in order.
// maxima[g * 32 + lane]: that lane's maximum of the g-th `group` batches.  Each lane goes through its
// own groups that reach tau; the lanes' candidates are taken one a lane at a time.
template <typename T>
__device__ __forceinline__ int collect(const Row<T>& row, const float* maxima, int group, float tau, int b0, int b1,
                                       Key* keys, int k, int lane) {
  constexpr int E = kSteps * Vec<T>::N;
  const bool few = is_neg_inf(tau);  // fewer than k lanes have a finite entry
  tau = finite_bound(tau);
  int count = 0;
  Key least = 0;
  unsigned hot = 0;  // this lane's groups that reach tau
  for (int g = 0; b0 + g * group < b1; ++g) hot |= (unsigned)(maxima[g * 32 + lane] >= tau) << g;
  while (__any_sync(kAll, hot != 0)) {
    // the lane's lowest hot group may hold an entry of the list: its maximum in its first column
    const int g = __ffs(hot) - 1, first = b0 + g * group;
    const bool may = hot != 0 && (least == 0 || top_key(maxima[g * 32 + lane], row.column(first, 0, lane)) > least);
    hot &= hot - 1;
    for (int j = 0; j < group; ++j) {
      const int b = first + j;
      unsigned mine = 0;
      if (may && b < b1) {
        uint4 q[kSteps];
        float f[E];
        row.load(q, b, lane);
#pragma unroll
        for (int u = 0; u < kSteps; ++u) Vec<T>::decode(q[u], f + u * Vec<T>::N);
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (f[i] >= tau) mine |= 1u << i;
      }
      take<T>(row.x, row.S, mine, [&](int i) { return row.column(b, i, lane); }, keys, count, least, k, lane);
    }
  }
  if (few && count < k && b0 < b1)
    fill(row.x, max(0, row.column(b0, 0, 0)), min(row.S, row.column(b1, 0, 0)), keys, count, k, lane);
  return cut_keys(keys, count, k, lane);
}

struct ScoreArgs {
  const void* rows;
  long long row_stride, n_rows;
  int n_cols, n_given, n_top;
  float scale, unit;  // log2 u and its reciprocal: 1, 1 or log2 e, ln 2
  const long long* given;
  float *log_mass, *entropy, *given_lp, *top_lp, *stats;
  long long* top_col;
};

// Batches of a group that lanes keep one maximum of, for a warp's n batches.
__device__ __forceinline__ int group_size(int n) { return (n + kGroups - 1) / kGroups; }

// Batches [b0, b1) of a row by one warp: each lane's sums, its maximum of every `group` batches
// (maxima[g * 32 + lane]) and over all of them (top_most).  AHEAD batches are under way.
template <typename T, bool TOP, bool NATURAL, int AHEAD = 1>
__device__ __forceinline__ Sums scan(const Row<T>& row, int b0, int b1, float scale, int group, float* maxima,
                                     float& top_most, int lane) {
  constexpr int E = kSteps * Vec<T>::N;
  top_most = neg_inf();
  Sums a{neg_inf(), 0.f, 0.f};
  float group_most = neg_inf();
  int left = group, slot = lane;
  uint4 next[AHEAD][kSteps];
#pragma unroll
  for (int d = 0; d < AHEAD; ++d)
    if (b0 + d < b1) row.load(next[d], b0 + d, lane);
  const auto take_batch = [&](int b, uint4 (&q)[kSteps]) {
    float f[E];
    row.decode(q, f, b, lane);
    if (b + AHEAD < b1) row.load(q, b + AHEAD, lane);
    float most = f[0];
#pragma unroll
    for (int i = 1; i + 1 < E; i += 2) most = max3(most, f[i], f[i + 1]);
    most = fmaxf(most, f[E - 1]);
    if constexpr (TOP) {
      group_most = fmaxf(group_most, most);
      if (--left == 0 || b + 1 == b1) {
        maxima[slot] = group_most;
        top_most = fmaxf(top_most, group_most);
        group_most = neg_inf();
        left = group;
        slot += 32;
      }
    }
    if (most > a.m) rebase(a, most, scale);
    const float ms = safe_max(a.m);
    const Pair minus = pack(-ms, -ms), factor = pack(scale, scale);
    Pair sum = pack(0.f, 0.f), less = sum;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      Pair z = pack(f[i], f[i + 1]) + minus;
      if constexpr (NATURAL) z = z * factor;
      float z0, z1;
      unpack(z, z0, z1);
      const float w0 = weight(z0), w1 = weight(z1);
      sum = sum + pack(w0, w1);
      less = less + pack(weighted(w0, z0), weighted(w1, z1));
    }
    float s0, s1, t0, t1;
    unpack(sum, s0, s1);
    unpack(less, t0, t1);
    a.sum += s0 + s1;
    a.wsum -= t0 + t1;
  };
  for (int b = b0; b < b1; b += AHEAD) {
#pragma unroll
    for (int d = 0; d < AHEAD; ++d)
      if (d == 0 || b + d < b1) take_batch(b + d, next[d]);
  }
  return a;
}

// Place j of a row's top list (not there: none).
__device__ __forceinline__ void write_top(const ScoreArgs& a, long long r, int j, bool there, float v, int col,
                                          float ms, float log_sum, bool bad, bool empty) {
  a.top_col[r * a.n_top + j] = there && !bad ? col : -1;
  a.top_lp[r * a.n_top + j] =
      bad ? __int_as_float(0x7fc00000) : (there && !empty ? (v - ms) - log_sum : neg_inf());
}

// One warp writes a row's outputs; keys: the best n_keys in order.
template <typename T, bool TOP>
__device__ __forceinline__ void write_scores(const ScoreArgs& a, long long r, const T* x, const Sums& s,
                                             const Key* keys, int n_keys, int lane) {
  const float nan = __int_as_float(0x7fc00000);
  const bool empty = s.sum == 0.f, bad = !(s.sum < __int_as_float(0x7f800000));
  const float ms = safe_max(s.m), bits = log2f(s.sum), log_sum = bad ? nan : bits * a.unit;
  if (lane == 0) {
    a.log_mass[r] = bad ? nan : ms + log_sum;
    a.entropy[r] = bad ? nan : (empty ? 0.f : (bits - s.wsum / s.sum) * a.unit);
    a.stats[2 * r] = bad ? nan : s.m;
    a.stats[2 * r + 1] = bad ? nan : s.sum;
  }
  if (lane < a.n_given) {
    const long long t = a.given[r * a.n_given + lane];
    a.given_lp[r * a.n_given + lane] =
        (t < 0 || t >= a.n_cols) ? 0.f : (empty ? neg_inf() : (Vec<T>::up(x[t]) - ms) - log_sum);
  }
  if constexpr (TOP) {
    if (lane < a.n_top) {
      const Key key = lane < n_keys ? keys[lane] : 0;
      write_top(a, r, lane, lane < n_keys, key_value(key), key_column(key), ms, log_sum, bad, empty);
    }
  }
}

// Short rows: G lanes a row (32 / G rows a warp), its entries in their registers (entry i of lane l: column
// i G + l), the top list as above with k <= G.  What a row costs beside its entries -- the bound, the
// candidates' loop, the cut, the outputs -- is paid once for the warp's rows.
// 16-bit values and their column make a 32-bit key.
template <typename T>
struct ShortKey {
  typedef unsigned type;
  static __device__ __forceinline__ unsigned make(float x, int col) {
    return (Vec<T>::order(x) << 16) | (0xffffu - (unsigned)col);
  }
  static __device__ __forceinline__ float value(unsigned k) { return Vec<T>::value(k >> 16); }
  static __device__ __forceinline__ int column(unsigned k) { return (int)(0xffffu - (k & 0xffffu)); }
};
template <>
struct ShortKey<float> {
  typedef Key type;
  static __device__ __forceinline__ Key make(float x, int col) { return top_key(x, col); }
  static __device__ __forceinline__ float value(Key k) { return key_value(k); }
  static __device__ __forceinline__ int column(Key k) { return key_column(k); }
};

// One row's list, kept by G lanes; every lane of the warp calls every function.
template <typename T, int G>
struct ShortList {
  typedef typename ShortKey<T>::type KeyT;
  KeyT *keys, *best;  // kCand candidates; room for 32 of them
  int k, lane, count;
  KeyT least;  // the k-th key of the last cut: nothing below it is in the list
  __device__ __forceinline__ ShortList(KeyT* keys_, KeyT* best_, int k_, int lane_)
      : keys(keys_), best(best_), k(k_), lane(lane_), count(0), least(0) {}

  static __device__ __forceinline__ unsigned group_ballot(bool c) {
    const unsigned b = __ballot_sync(kAll, c);
    return G == 32 ? b : (b >> (threadIdx.x & 31 & ~(G - 1))) & ((1u << (G & 31)) - 1);
  }
  // Keeps the best k, in order, of the lists that are `on`: a key's place is the number of larger keys.
  __device__ __forceinline__ void cut(bool on) {
    __syncwarp();
    const int n = on ? count : 0, most = __reduce_max_sync(kAll, n);
    for (int base = 0; base < most; base += G) {
      const KeyT a = base + lane < n ? keys[base + lane] : 0;
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < most; ++j) rank += (G == 32 || j < n) && keys[j] > a;
      if (base + lane < n && rank < k) best[rank] = a;
    }
    __syncwarp();
    if (on) {
      count = min(count, k);
      for (int j = lane; j < count; j += G) keys[j] = best[j];
    }
    __syncwarp();
    if (on && count == k) least = keys[k - 1];
  }
  __device__ __forceinline__ void push(bool c, KeyT key) {
    c = c && key > least;
    unsigned in = group_ballot(c);
    const bool over = count + __popc(in) > kCand;
    if (__any_sync(kAll, over)) {
      cut(over);
      c = c && key > least;
      in = group_ballot(c);
    }
    if (c) keys[count + __popc(in & ((1u << lane) - 1))] = key;
    count += __popc(in);
  }
};

template <int G>
__device__ __forceinline__ float group_max(float x) {
  if constexpr (G == 32) {
    return lanes_max(x);
  } else {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(kAll, x, o));
    return x;
  }
}

template <typename T, int G, int E>
__global__ void __launch_bounds__(32 * kWarps) score_short_kernel(const ScoreArgs a) {
  typedef ShortList<T, G> List;
  typedef ShortKey<T> K;
  const int lane = threadIdx.x & (G - 1);
  const long long at = ((long long)blockIdx.x * (32 * kWarps) + threadIdx.x) / G;
  const bool live = at < a.n_rows;  // lanes past the last row work on it and write nothing
  const long long r = live ? at : a.n_rows - 1;
  const T* x = static_cast<const T*>(a.rows) + r * a.row_stride;
  const float nan = __int_as_float(0x7fc00000);
  float f[E];
  if (a.n_cols > G * (E - 1)) {  // only a lane's last entry may be missing (trees of 2^j leaves: S = 2^(j+1) - 1)
#pragma unroll
    for (int i = 0; i + 1 < E; ++i) f[i] = Vec<T>::up(x[i * G + lane]);
    f[E - 1] = (E - 1) * G + lane < a.n_cols ? Vec<T>::up(x[(E - 1) * G + lane]) : neg_inf();
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = i * G + lane < a.n_cols ? Vec<T>::up(x[i * G + lane]) : neg_inf();
  }
  float most = fmaxf(f[0], f[1]);
#pragma unroll
  for (int i = 2; i < E; i += 2) most = max3(most, f[i], f[i + 1]);
  const float m = group_max<G>(most), ms = safe_max(m);
  float sum, less;
  {
    const Pair minus = pack(-ms, -ms), factor = pack(a.scale, a.scale);
    Pair sums = pack(0.f, 0.f), lesses = sums;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      float z0, z1;
      unpack((pack(f[i], f[i + 1]) + minus) * factor, z0, z1);
      const float w0 = weight(z0), w1 = weight(z1);
      sums = sums + pack(w0, w1);
      lesses = lesses + pack(weighted(w0, z0), weighted(w1, z1));
    }
    float s0, s1, t0, t1;
    unpack(sums, s0, s1);
    unpack(lesses, t0, t1);
    sum = s0 + s1;
    less = t0 + t1;
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(kAll, sum, o);
    less += __shfl_xor_sync(kAll, less, o);
  }
  const bool empty = sum == 0.f, bad = !(sum < __int_as_float(0x7f800000));
  const float bits = log2f(sum), log_sum = bad ? nan : bits * a.unit;
  if (live) {
    if (lane == 0) {
      a.log_mass[r] = bad ? nan : ms + log_sum;
      a.entropy[r] = bad ? nan : (empty ? 0.f : (bits + less / sum) * a.unit);
    }
    if (lane < 2) a.stats[2 * r + lane] = bad ? nan : (lane == 0 ? m : sum);
    for (int j = lane; j < a.n_given; j += G) {
      const long long t = a.given[r * a.n_given + j];
      a.given_lp[r * a.n_given + j] =
          (t < 0 || t >= a.n_cols) ? 0.f : (empty ? neg_inf() : (Vec<T>::up(x[t]) - ms) - log_sum);
    }
  }
  if (a.n_top == 0) return;
  __shared__ typename K::type keys[kWarps * 32 / G][kCand], best[kWarps * 32 / G][32];
  List list(keys[threadIdx.x / G], best[threadIdx.x / G], a.n_top, lane);
  const float tau = finite_bound(kth_of_lanes<G>(most, a.n_top, lane));
  unsigned mine = 0;
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (f[i] >= tau) mine |= 1u << i;
  while (__any_sync(kAll, mine != 0)) {
    const int col = mine ? (__ffs(mine) - 1) * G + lane : 0;
    const bool c = mine != 0;
    mine &= mine - 1;
    list.push(c, c ? K::make(Vec<T>::up(x[col]), col) : 0);
  }
  if (__any_sync(kAll, list.count < a.n_top)) {  // too few finite entries: the lowest of the others
    for (int j = 0; j < 64; j += G) {
      const bool c = list.count < a.n_top && j + lane < a.n_cols && is_neg_inf(Vec<T>::up(x[j + lane]));
      list.push(c, c ? K::make(neg_inf(), j + lane) : 0);
    }
  }
  list.cut(true);
  if (live)
    for (int j = lane; j < a.n_top; j += G) {
      const bool there = j < list.count;
      const typename K::type key = there ? list.keys[j] : 0;
      write_top(a, r, j, there, K::value(key), K::column(key), ms, log_sum, bad, empty);
    }
}

// A warp a row, in CTAs of two warps: a finished row makes room for the next without waiting for six
// others (128,282 x 4,095 fp32, 8 columns: 446 us in CTAs of 8 warps, 435 of 4, 430 of 2; persistent
// warps 462, and 610 with the next row asked into L2 by bulk prefetches).  More rows under way help
// too: at 64 registers (32 warps an SM) 367 us where 76 (24 warps) take 411.  16-bit rows, whose
// batches hold twice the entries, are bound by their instructions and keep 80.
// Measured: 128,282 x 4,095 fp32 with 8 columns 354 us, 6.0 TB/s, 91 % of the copy bandwidth; after a second of
// nothing else, at 1.6 GHz under the power cap, 390 us a call, 5.4 TB/s, 83 %.
// Where all rows are under way at once the warps are too few to fill memory with one batch each; with
// AHEAD = 2 they ask for two (2,300 x 32,001 fp32: 76 us, 82 with one; 1,700 x 4,095: 16 and 18).
template <typename T, bool TOP, bool NATURAL, int AHEAD>
__global__ void __launch_bounds__(32 * kRowWarps, (AHEAD == 2 ? 16 : sizeof(T) == 4 ? 32 : 24) / kRowWarps)
    score_warp_kernel(const ScoreArgs a) {
  __shared__ Key keys[kRowWarps][TOP ? kCand : 1];
  __shared__ float maxima[kRowWarps][TOP ? 32 * kGroups : 1];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long long r = (long long)blockIdx.x * kRowWarps + wid;
  if (r >= a.n_rows) return;
  const Row<T> row(static_cast<const T*>(a.rows) + r * a.row_stride, a.n_cols);
  const int group = group_size(row.n_batch);
  float most;
  Sums s = scan<T, TOP, NATURAL, AHEAD>(row, 0, row.n_batch, a.scale, group, maxima[wid], most, lane);
  s = warp_join(s, a.scale);
  int count = 0;
  if constexpr (TOP)
    count = collect(row, maxima[wid], group, kth_of_lanes(most, a.n_top, lane), 0, row.n_batch, keys[wid], a.n_top,
                    lane);
  write_scores<T, TOP>(a, r, row.x, s, keys[wid], count, lane);
}

struct Part {      // what a warp, and then a CTA, hands on
  Key keys[32];    // in order
  Sums s;
  int count;
};

// The best k of n <= kWarps sorted lists: a key's place is its place in its own list and the larger keys
// of the others, found by bisection.  All threads call; out.count and out.keys are set.
__device__ __forceinline__ void merge_lists(const Part* parts, int n, int k, Part& out) {
  const int w = threadIdx.x >> 5, p = threadIdx.x & 31;
  if (w < n && p < parts[w].count) {
    const Key key = parts[w].keys[p];
    int rank = p;
    for (int o = 0; o < n; ++o) {
      if (o == w) continue;
      int lo = 0, hi = parts[o].count;  // keys[0 .. lo) are larger
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (parts[o].keys[mid] > key) lo = mid + 1; else hi = mid;
      }
      rank += lo;
    }
    if (rank < k) out.keys[rank] = key;
  }
  if (threadIdx.x == 0) {
    int c = 0;
    for (int o = 0; o < n; ++o) c += parts[o].count;
    out.count = c < k ? c : k;
  }
}
__device__ __forceinline__ Sums join_parts(const Part* parts, int n, float scale, int lane) {
  return warp_join(lane < n ? parts[lane].s : Sums{neg_inf(), 0.f, 0.f}, scale);
}

// What score_group_kernel keeps in (dynamic) shared memory, for CTAs of W warps.
struct GroupSpace {
  Part* parts;       // [W + 1]: the warps', then the CTAs'; the CTA's own
  Key* keys;         // [W][kCand]
  float* maxima;     // [W][32 kGroups]
  float* lane_most;  // [W][32]
  __device__ __forceinline__ GroupSpace(unsigned char* at, int W)
      : parts(reinterpret_cast<Part*>(at)), keys(reinterpret_cast<Key*>(parts + W + 1)),
        maxima(reinterpret_cast<float*>(keys + W * kCand)), lane_most(maxima + W * 32 * kGroups) {}
  static int bytes(int W, bool top) {
    return (W + 1) * (int)sizeof(Part) + (top ? W * (kCand * (int)sizeof(Key) + (32 * kGroups + 32) * (int)sizeof(float)) : 0);
  }
};

// A cluster a row: each warp of its CTAs (8 warps, or 4 where the row has one CTA) takes a
// stretch of the row's batches; the CTA's lists and sums are joined in shared memory, the cluster's in
// the first CTA's, read over distributed shared memory.
template <typename T, bool TOP, bool NATURAL>
__global__ void __launch_bounds__(32 * kWarps, 3) score_group_kernel(const ScoreArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) unsigned char space[];
  const int W = blockDim.x >> 5;
  const GroupSpace sm(space, W);
  Part *parts = sm.parts, &mine = parts[W];
  cg::cluster_group cluster = cg::this_cluster();
  const int n_ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long long r = blockIdx.x / n_ctas;
  const Row<T> row(static_cast<const T*>(a.rows) + r * a.row_stride, a.n_cols);
  const long long w = cta * W + wid, n_warps = n_ctas * W;
  Key* keys = sm.keys + wid * kCand;
  float* maxima = sm.maxima + wid * 32 * kGroups;
  const int b0 = (int)(row.n_batch * w / n_warps), b1 = (int)(row.n_batch * (w + 1) / n_warps);
  const int group = group_size(b1 - b0);
  float most;
  Sums s = scan<T, TOP, NATURAL>(row, b0, b1, a.scale, group, maxima, most, lane);
  s = warp_join(s, a.scale);
  if (lane == 0) parts[wid].s = s;
  if constexpr (TOP) {
    // the bound is the CTA's: of the maxima that equal lanes of its warps share
    sm.lane_most[wid * 32 + lane] = most;
    __syncthreads();
    for (int o = 0; o < W; ++o) most = fmaxf(most, sm.lane_most[o * 32 + lane]);
    const int count = collect(row, maxima, group, kth_of_lanes(most, a.n_top, lane), b0, b1, keys, a.n_top, lane);
    if (lane < count) parts[wid].keys[lane] = keys[lane];
    if (lane == 0) parts[wid].count = count;
  }
  __syncthreads();
  if constexpr (TOP) merge_lists(parts, W, a.n_top, mine);
  if (wid == 0) {
    s = join_parts(parts, W, a.scale, lane);
    if (lane == 0) mine.s = s;
  }
  if (n_ctas > 1) {
    cluster.sync();
    if (cta == 0 && wid < n_ctas) {
      const Part* other = cluster.map_shared_rank(&mine, wid);
      if constexpr (TOP) {
        const int count = other->count;
        if (lane < count) parts[wid].keys[lane] = other->keys[lane];
        if (lane == 0) parts[wid].count = count;
      }
      if (lane == 0) parts[wid].s = other->s;
    }
    cluster.sync();  // no CTA leaves while its part is read
    if (cta != 0) return;
    if constexpr (TOP) merge_lists(parts, n_ctas, a.n_top, mine);
    s = join_parts(parts, n_ctas, a.scale, lane);
  }
  __syncthreads();
  if (wid == 0) write_scores<T, TOP>(a, r, row.x, s, mine.keys, TOP ? mine.count : 0, lane);
}

struct ScoreGradArgs {
  const void* rows;
  long long row_stride, n_rows;
  int n_cols, n_given;
  float scale;
  const float *stats, *entropy;
  const long long* given;
  const float *g_mass, *g_given, *g_entropy;
  void* out;
  long long out_stride;
};

// dL/dx_s = p_s (a - sum_t g_t - h ln2 (z_s - log2 Sigma + H)) + sum_{t: given_t = s} g_t, with the
// cotangents a of log_mass, g of the given columns and h of the entropy, H in bits (the factor
// ln u of d log_u and the one of d u^x cancel, so both bases share it).  Impossible columns are
// constants: no gradient at them, none through a given column that is one.  That holds beside cotangents
// that are not finite too (functions of an empty row's log mass, -inf, have such).
struct Gradient {
  float m, scale, direct, bend;
  __device__ __forceinline__ Gradient(const ScoreGradArgs& a, long long r, float m_row, float sum, float g_all) {
    const bool empty = sum == 0.f;
    const float h = a.g_entropy ? a.g_entropy[r] * kLn2 : 0.f;
    const float bits = (a.g_entropy ? a.entropy[r] * a.scale : 0.f) - (empty ? 0.f : log2f(sum));
    const float inv = empty ? 0.f : 1.f / sum;
    m = empty ? 0.f : m_row;
    scale = a.scale;
    // p (base - h (z + bits)) = 2^z direct - 2^z z bend
    direct = ((a.g_mass ? a.g_mass[r] : 0.f) - g_all - h * bits) * inv;
    bend = h * inv;
    if (empty) direct = bend = 0.f;
  }
  // Whether the row is a distribution (else its stats are NaN) beside which a factor is not finite: 0 times it
  // is NaN at the impossible columns.
  __device__ __forceinline__ bool odd() const {
    return m == m && !(fabsf(direct) + fabsf(bend) < __int_as_float(0x7f800000));
  }
  // without the given columns' own terms
  __device__ __forceinline__ float operator()(float x) const {
    const float z = (x - m) * scale, w = weight(z);
    return fmaf(w, direct, weighted(w, z) * bend);
  }
};

// A warp takes `chunk` batches of a row: one read and one write of each entry, so memory bounds it
// (32,071 x 4,095 fp32: 171 us, 6.1 TB/s, 94 % of the copy bandwidth; 4 CTAs an SM, 3 and 5 take 7 % and
// 15 % longer).
// A vector is worked on as soon as it is there and its registers take the next batch's.
// The entries at given columns are written once more, by the lane that holds the column.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps, 4) score_rows_backward_kernel(const ScoreGradArgs a, const int chunk,
                                                                          const unsigned chunks) {
  constexpr int N = Vec<T>::N;
  const int lane = threadIdx.x & 31;
  const unsigned long long task = (unsigned long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const long long r = (long long)(chunks == 1 ? task : task / chunks);
  if (r >= a.n_rows) return;
  const T* x = static_cast<const T*>(a.rows) + r * a.row_stride;
  T* out = static_cast<T*>(a.out) + r * a.out_stride;
  const Row<T> row(x, a.n_cols);
  const int b0 = (int)(task - (unsigned long long)r * chunks) * chunk, b1 = min(row.n_batch, b0 + chunk);
  if (b0 >= b1) return;
  uint4 next[kSteps];
  row.load(next, b0, lane);

  const float m_row = a.stats[2 * r], sum = a.stats[2 * r + 1];
  const bool empty = sum == 0.f;
  int t = -1;
  float g = 0.f, g_all = 0.f;
  if (a.n_given > 0) {
    if (lane < a.n_given) {
      const long long tt = a.given[r * a.n_given + lane];
      if (tt >= 0 && tt < a.n_cols && !empty && !is_neg_inf(Vec<T>::up(x[tt]))) {
        t = (int)tt;
        g = a.g_given[r * a.n_given + lane];
      }
    }
    g_all = warp_sum(g);
  }
  const Gradient gradient(a, r, m_row, sum, g_all);

  // whether the output's 16-byte boundaries fall where the input's do
  const uintptr_t to = reinterpret_cast<uintptr_t>(out);
  const bool even = (int)((to & 15) / sizeof(T)) == row.shift;
  uint4* out_vec = reinterpret_cast<uint4*>(to & ~(uintptr_t)15);
  for (int b = b0; b < b1; ++b) {
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const int v = (b * kSteps + u) * 32 + lane;
      float f[N];
      Vec<T>::decode(next[u], f);
      if (b + 1 < b1) next[u] = row.load_one(v + kBatch);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = gradient(f[e]);
      if (v >= row.n_vec) continue;
      if (even && (v > 0 || row.shift == 0) && (v + 1) * (long long)N <= (long long)row.S + row.shift) {
        out_vec[v] = Vec<T>::encode(f);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int col = v * N - row.shift + e;
          if ((unsigned)col < (unsigned)row.S) out[col] = Vec<T>::down(f[e]);
        }
      }
    }
  }
  if (gradient.odd()) {
    __syncwarp();  // after the stores above
    for (int col = max(0, row.column(b0, 0, 0)) + lane; col < min(row.S, row.column(b1, 0, 0)); col += 32)
      if (is_neg_inf(Vec<T>::up(x[col]))) out[col] = Vec<T>::down(0.f);
  }
  if (a.n_given == 0) return;
  // equal columns are added up by the first lane that has one, in the lanes' order
  float add = 0.f;
  bool first = true;
  for (int j = 0; j < a.n_given; ++j) {
    const int tj = __shfl_sync(kAll, t, j);
    const float gj = __shfl_sync(kAll, g, j);
    if (tj == t) {
      add += gj;
      first = first && j >= lane;
    }
  }
  __syncwarp();  // after the stores above
  if (t >= 0 && first && t >= row.column(b0, 0, 0) && t < row.column(b1, 0, 0))
    out[t] = Vec<T>::down(gradient(Vec<T>::up(x[t])) + add);
}

// Rows of up to 256 columns: G lanes a row, E of its entries each, as in score_short_kernel.
template <typename T, int G, int E>
__global__ void __launch_bounds__(32 * kWarps) score_short_backward_kernel(const ScoreGradArgs a) {
  const int lane = threadIdx.x & (G - 1), S = a.n_cols;
  const long long r = ((long long)blockIdx.x * (32 * kWarps) + threadIdx.x) / G;
  if (r >= a.n_rows) return;
  const T* x = static_cast<const T*>(a.rows) + r * a.row_stride;
  T* out = static_cast<T*>(a.out) + r * a.out_stride;
  float f[E], add[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    f[i] = i * G + lane < S ? Vec<T>::up(x[i * G + lane]) : neg_inf();
    add[i] = 0.f;
  }
  const float m_row = a.stats[2 * r], sum = a.stats[2 * r + 1];
  const bool empty = sum == 0.f;
  float g_all = 0.f;
  for (int j = 0; j < a.n_given; ++j) {
    const long long t = a.given[r * a.n_given + j];
    if (t < 0 || t >= S || empty || is_neg_inf(Vec<T>::up(x[t]))) continue;
    const float g = a.g_given[r * a.n_given + j];
    g_all += g;
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i * G + lane == (int)t) add[i] += g;
  }
  const Gradient gradient(a, r, m_row, sum, g_all);
  const bool odd = gradient.odd();
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (i * G + lane < S)
      out[i * G + lane] = Vec<T>::down(odd && is_neg_inf(f[i]) ? 0.f : gradient(f[i]) + add[i]);
}

template <typename T>
cudaError_t launch_backward(const ScoreGradArgs& a, cudaStream_t st) {
  // (300,000 x 63 fp32: 52 us, 264 by vectors; 120,000 x 255: 78 and 103)
  if (a.n_cols <= 256) {
    const auto ctas = [&](int g) { return (unsigned)((a.n_rows + 32 * kWarps / g - 1) / (32 * kWarps / g)); };
    if (a.n_cols <= 64) score_short_backward_kernel<T, 8, 8><<<ctas(8), 32 * kWarps, 0, st>>>(a);
    else if (a.n_cols <= 128) score_short_backward_kernel<T, 16, 8><<<ctas(16), 32 * kWarps, 0, st>>>(a);
    else score_short_backward_kernel<T, 16, 16><<<ctas(16), 32 * kWarps, 0, st>>>(a);
    return cudaGetLastError();
  }
  const long long batches = ((long long)a.n_cols * sizeof(T) + 15 + 16 * kBatch - 1) / (16 * kBatch);
  // about 4,096 entries a warp in equal chunks (a row of 4,095 fp32 entries that starts off a boundary
  // is 9 batches: one chunk of 9 takes 177 us, one of 8 and one of 1 188), or a batch where that leaves
  // fewer warps than the GPU holds
  constexpr int kPer = 4096 / (kBatch * Vec<T>::N);
  long long chunks = batches < kPer ? 1 : (batches + kPer / 2) / kPer;
  if (a.n_rows * chunks < 148 * 32) chunks = batches;
  const int chunk = (int)((batches + chunks - 1) / chunks);
  const long long ctas = (a.n_rows * chunks + kWarps - 1) / kWarps;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  score_rows_backward_kernel<T><<<(unsigned)ctas, 32 * kWarps, 0, st>>>(a, chunk, (unsigned)chunks);
  return cudaGetLastError();
}

// By the row's length and the number of rows (times between events around the call, L2 flushed: about 4 us
// above the kernel's own):
//  * up to 1,024 columns: the registers of a warp, or of 16 or 8 lanes where they hold the row
//    and no more alternatives are asked for than lanes take part (300,000 x 63 fp32: 70 us, 161 with a
//    warp a row; 200,000 x 127: 86 and 141; 60,000 x 511: 49 and 59);
//  * a warp a row, unless the rows are few beside their length (fewer than 25 for each 2 KB of a row):
//    a warp then reads too long after the others, and a CTA a row is faster (1,200 x 32,001 fp32: 55 us, 66
//    with a warp a row; 1,200 x 16,383: 39 and 35; 5,000 x 131,071: 469 and 549; 3,000 x 60,000: 162 and 153);
//  * four warps a row where all rows then fit at once (800 x 32,001 fp32: 35 us, 39 with eight, 61 with one;
//    500 x 8,191: 15, 18 and 17; two a row for up to 1,776 rows are slower than one: 1,200 x 32,001 67);
//  * as many warps a row as give every SM 16 of them, in CTAs of 8 and clusters of up to 8 CTAs, as
//    long as each has a batch (2 KB) to read (16 x 131,071 bf16: 17 us; 26 in clusters of 16).
template <typename T, bool TOP, bool NATURAL>
cudaError_t launch_scores(const ScoreArgs& a, cudaStream_t st) {
  if (a.n_cols <= 1024) {
    const auto rows_a_cta = [&](int g) { return (unsigned)((a.n_rows + 32 * kWarps / g - 1) / (32 * kWarps / g)); };
    if (a.n_cols <= 64 && a.n_top <= 8) score_short_kernel<T, 8, 8><<<rows_a_cta(8), 32 * kWarps, 0, st>>>(a);
    else if (a.n_cols <= 128 && a.n_top <= 16) score_short_kernel<T, 16, 8><<<rows_a_cta(16), 32 * kWarps, 0, st>>>(a);
    else if (a.n_cols <= 256 && a.n_top <= 16) score_short_kernel<T, 16, 16><<<rows_a_cta(16), 32 * kWarps, 0, st>>>(a);
    else if (a.n_cols <= 256) score_short_kernel<T, 32, 8><<<rows_a_cta(32), 32 * kWarps, 0, st>>>(a);
    else if (a.n_cols <= 512 && a.n_top <= 16) score_short_kernel<T, 16, 32><<<rows_a_cta(16), 32 * kWarps, 0, st>>>(a);
    else if (a.n_cols <= 512) score_short_kernel<T, 32, 16><<<rows_a_cta(32), 32 * kWarps, 0, st>>>(a);
    else score_short_kernel<T, 32, 32><<<rows_a_cta(32), 32 * kWarps, 0, st>>>(a);
    return cudaGetLastError();
  }
  const long long batches = ((long long)a.n_cols * sizeof(T) + 16 * kBatch - 1) / (16 * kBatch);
  const long long wanted = (148 * 16 + a.n_rows - 1) / a.n_rows;
  const long long warps = wanted < batches ? wanted : batches;
  constexpr long long one_wave = 148 * 24;  // warps that the GPU holds of the grouped kernel
  const bool few = 4 * a.n_rows <= one_wave && batches >= 4;
  if (warps < kWarps && !few && (batches < kWarps || 25 * batches < a.n_rows)) {
    const unsigned ctas = (unsigned)((a.n_rows + kRowWarps - 1) / kRowWarps);
    if (a.n_rows <= 148 * 16) score_warp_kernel<T, TOP, NATURAL, 2><<<ctas, 32 * kRowWarps, 0, st>>>(a);
    else score_warp_kernel<T, TOP, NATURAL, 1><<<ctas, 32 * kRowWarps, 0, st>>>(a);
    return cudaGetLastError();
  }
  unsigned ctas = 1;
  while (ctas < kWarps && 2 * ctas * kWarps <= warps) ctas *= 2;
  const int W = few && a.n_rows * ctas * kWarps > one_wave ? 4 : kWarps;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.n_rows * ctas));
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = GroupSpace::bytes(W, TOP);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, score_group_kernel<T, TOP, NATURAL>, a);
}

template <typename T>
cudaError_t launch_scores_of(const ScoreArgs& a, bool natural, cudaStream_t st) {
  if (a.n_top > 0) return natural ? launch_scores<T, true, true>(a, st) : launch_scores<T, true, false>(a, st);
  return natural ? launch_scores<T, false, true>(a, st) : launch_scores<T, false, false>(a, st);
}

}  // namespace

static bool floats_on_boundary(std::initializer_list<const float*> ps) {
  for (const float* p : ps)
    if (!kb::on_boundary(p, 4)) return false;
  return true;
}

extern "C" int kb_score_rows(const void* rows, long long row_stride, int dtype, long long n_rows, int n_cols,
                             int natural, const long long* given, int n_given, int n_top, float* log_mass,
                             float* entropy, float* given_log_prob, float* top_log_prob, long long* top_column,
                             float* stats, void* stream) {
  if (n_rows < 0 || n_cols < 0 || row_stride < 0 || n_given < 0 || n_given > KB_MAX_GIVEN || n_top < 0 ||
      n_top > KB_MAX_TOP || dtype < 0 || dtype > 2)
    return KB_ERR_ARG;
  if (n_rows == 0) return KB_OK;
  if ((!rows && n_cols > 0) || !log_mass || !entropy || !stats || (n_given > 0 && (!given || !given_log_prob)) ||
      (n_top > 0 && (!top_log_prob || !top_column)))
    return KB_ERR_ARG;
  if (!on_boundary(rows, dtype == 0 ? 4 : 2) || !on_boundary(given, 8) || !on_boundary(top_column, 8) ||
      !floats_on_boundary({log_mass, entropy, given_log_prob, top_log_prob, stats}))
    return KB_ERR_ARG;
  if (n_rows > 0x7fffffffll || n_cols > KB_MAX_SCORE_COLS) return KB_ERR_SIZE;
  ScoreArgs a{rows, row_stride, n_rows, n_cols, n_given, n_top, natural ? kLog2e : 1.f, natural ? kLn2 : 1.f,
              given, log_mass, entropy, given_log_prob, top_log_prob, stats, top_column};
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == 0   ? launch_scores_of<float>(a, natural, st)
                        : dtype == 1 ? launch_scores_of<__nv_bfloat16>(a, natural, st)
                                     : launch_scores_of<__half>(a, natural, st);
  return e == cudaSuccess ? KB_OK : KB_ERR_LAUNCH;
}

extern "C" int kb_score_rows_backward(const void* rows, long long row_stride, int dtype, long long n_rows, int n_cols,
                                      int natural, const float* stats, const float* entropy, const long long* given,
                                      int n_given, const float* grad_log_mass, const float* grad_given,
                                      const float* grad_entropy, void* grad_rows, long long grad_stride,
                                      void* stream) {
  if (n_rows < 0 || n_cols < 0 || row_stride < 0 || grad_stride < 0 || n_given < 0 || n_given > KB_MAX_GIVEN ||
      dtype < 0 || dtype > 2)
    return KB_ERR_ARG;
  if (n_rows == 0 || n_cols == 0) return KB_OK;
  if (!rows || !grad_rows || !stats || (grad_entropy && !entropy) || (n_given > 0 && grad_given && !given) ||
      (n_rows > 1 && grad_stride < n_cols))
    return KB_ERR_ARG;
  const unsigned width = dtype == 0 ? 4 : 2;
  if (!on_boundary(rows, width) || !on_boundary(grad_rows, width) || !on_boundary(given, 8) ||
      !floats_on_boundary({stats, entropy, grad_log_mass, grad_given, grad_entropy}))
    return KB_ERR_ARG;
  if (n_rows > 0x7fffffffll || n_cols > KB_MAX_SCORE_COLS) return KB_ERR_SIZE;
  ScoreGradArgs a{rows, row_stride, n_rows, n_cols, grad_given ? n_given : 0, natural ? kLog2e : 1.f, stats, entropy,
                  given, grad_log_mass, grad_given, grad_entropy, grad_rows, grad_stride};
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == 0   ? launch_backward<float>(a, st)
                        : dtype == 1 ? launch_backward<__nv_bfloat16>(a, st)
                                     : launch_backward<__half>(a, st);
  return e == cudaSuccess ? KB_OK : KB_ERR_LAUNCH;
}
