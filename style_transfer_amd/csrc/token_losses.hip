// Losses over rows of logits for gfx950: the labels' log-probabilities, the preference loss of paired sequences, the
// clipped policy loss with its KL and entropy terms, and the distillation from a teacher's top logits.  HBM-bound.
//
// One row of logits x[0..V) at temperature tau, in the base-2 domain of the hardware's exponential:
//
//   c = log2(e) / tau     m = max x     d_j = (x_j - m) c     e_j = 2^d_j     S = sum e_j     W = sum e_j d_j
//   log q_j = ln2 d_j - ln S            entropy H = ln S - ln2 W / S
//
// Every loss here reaches x through the label's log-probability and the entropy, or through a short list of entries, so
// every gradient row is   g_j = (alpha + gamma d_j) e_j   plus a few patched entries:
//
//   dL/dlogp = a, dL/dH = b:  alpha = -(a + b (H - ln S)) / (tau S)   gamma = -b ln2 / (tau S)   patch: + a / tau at the label
//
// The difference x - m comes before the factor c: the lowest value of a type used as a mask cannot overflow against
// itself, and a row that holds nothing else is the uniform distribution that the formula gives.  A row of -inf only has
// S = 0: no distribution, log-probability -inf, entropy 0, gradient 0.
//
// Sums of a row are fp32 per thread and over a fixed tree; what a row is reduced to is finished in fp64 (one thread or
// one wave a row), because a sequence's sum of hundreds of log-probabilities is compared with another model's: c's own
// rounding (relative 2^-25) shifts every term the same way, and W, which is d ln S / d ln c, takes that shift out again.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "common.h"

namespace {

constexpr int NT = 256;                  // threads of a streaming block
constexpr int MAX_SPLITS = 64;           // parts of a row: one wave joins them
constexpr float D_MIN = -200.f;          // 2^-200 is 0 in fp32: keeps 0 * inf out of e_j d_j where x_j = -inf
constexpr double LN2 = 0.6931471805599453094;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_u __attribute__((aligned(2)));      // a row of another alignment than the one loaded

struct Logits {
  const void* x;
  const void* labels;                    // int64 or int32, null for the distillation
  int labels64;
  int ignore;
  unsigned inner;                        // row r starts at (r / inner) * s_outer + (r % inner) * s_inner
  long long s_outer, s_inner;
  int vocab;
  unsigned rows;
  float c;
  double tau;
};

// what a gradient pass needs of a row (float4): reference m, alpha, gamma, patch
typedef f32x4 RowGrad;

__device__ __forceinline__ long long row_offset(const Logits& p, unsigned r) {
  return (long long)(r / p.inner) * p.s_outer + (long long)(r % p.inner) * p.s_inner;
}

__device__ __forceinline__ long long load_index(const void* t, int is64, size_t i) {
  return is64 ? reinterpret_cast<const long long*>(t)[i] : (long long)reinterpret_cast<const int*>(t)[i];
}

// ---- the three storage types: 16 bytes <-> VEC floats ------------------------------------------------------------------
template <typename T> struct Type;
template <> struct Type<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ void unpack(const u32x4& v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[i]);
    return v;
  }
};
template <> struct Type<__bf16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ void unpack(const u32x4& v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    typedef __bf16 h8 __attribute__((ext_vector_type(8)));
    h8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (__bf16)f[i];
    return __builtin_bit_cast(u32x4, h);
  }
};
template <> struct Type<_Float16> {
  static constexpr int VEC = 8;
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void unpack(const u32x4& v, float* f) {
    const h8 h = __builtin_bit_cast(h8, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    h8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)f[i];
    return __builtin_bit_cast(u32x4, h);
  }
};

// ---- running statistics ----------------------------------------------------------------------------------------------
// (m, S, W) of a part of a row; an empty part has m = -inf, S = W = 0.
struct Part {
  float m, s, w;
};

__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }

// A part seen from another reference: d' = d + t, t = (m_old - m_new) c <= 0.
__device__ __forceinline__ void rebase(float& s, float& w, float m_old, float m_new, float c) {
  const float t = (m_old - finite_ref(m_new)) * c;
  const float f = __builtin_amdgcn_exp2f(t);
  w = f * fmaf(fmaxf(t, D_MIN), s, w);
  s *= f;
}

__device__ __forceinline__ Part join(Part a, Part b, float c) {
  const float m = fmaxf(a.m, b.m);
  rebase(a.s, a.w, a.m, m, c);
  rebase(b.s, b.w, b.m, m, c);
  return {m, a.s + b.s, a.w + b.w};
}

__device__ __forceinline__ Part wave_join(Part p, float c) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    p = join(p, Part{__shfl_xor(p.m, off, 64), __shfl_xor(p.s, off, 64), __shfl_xor(p.w, off, 64)}, c);
  return p;
}

// N more elements into a thread's part
template <int N>
__device__ __forceinline__ void take(Part& p, const float* x, float c) {
  float m = p.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
  if (m > p.m) {
    rebase(p.s, p.w, p.m, m, c);
    p.m = m;
  }
  const float ref = finite_ref(p.m);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = (x[i] - ref) * c;
    const float e = __builtin_amdgcn_exp2f(d);
    p.s += e;
    p.w = fmaf(fmaxf(d, D_MIN), e, p.w);
  }
}

// ---- what the logits of a row say once its parts are joined ----------------------------------------------------------------
struct RowStat {
  double ln_s;       // ln S, with the rounding of c taken out
  float h;           // entropy
  float inv_ts;      // 1 / (tau S); 0 for a row without a distribution
  float ref;         // m, or 0
};

__device__ __forceinline__ RowStat finish(const Part& q, float c, double tau) {
  RowStat r;
  r.ref = finite_ref(q.m);
  if (q.s == 0.f) {
    r.ln_s = -INFINITY;
    r.h = 0.f;
    r.inv_ts = 0.f;
    return r;
  }
  const double eps = (double)c * LN2 * tau - 1.0;          // c = (1 + eps) log2(e) / tau
  r.ln_s = log((double)q.s - eps * LN2 * (double)q.w);
  r.h = (float)(r.ln_s - LN2 * (double)q.w / (double)q.s);
  r.inv_ts = (float)(1.0 / (tau * (double)q.s));
  return r;
}

// natural logarithm of q at a logit
__device__ __forceinline__ double log_prob(float x, const RowStat& r, double tau) {
  return r.inv_ts == 0.f ? -INFINITY : ((double)x - (double)r.ref) / tau - r.ln_s;
}

template <typename T>
__device__ __forceinline__ float load_one(const void* base, long long i) {
  return (float)reinterpret_cast<const T*>(base)[i];
}

// A row's outputs from its joined statistics: log-probability, entropy, and what the gradient needs.  `state`:
// (m, 1 / (tau S), H - ln S, -).
template <typename T>
__device__ __forceinline__ void write_row(const Logits& p, unsigned r, long long label, const Part& q, float* logp, float* entropy,
                                          f32x4* state) {
  const RowStat st = finish(q, p.c, p.tau);
  float lp = NAN, h = st.h, inv = st.inv_ts;
  if (label >= 0 && label < p.vocab) lp = (float)log_prob(load_one<T>(p.x, row_offset(p, r) + label), st, p.tau);
  else inv = NAN;                                              // a label outside the vocabulary: visible, never an access
  logp[r] = lp;
  if (entropy) entropy[r] = h;
  if (state) state[r] = f32x4{st.ref, inv, st.inv_ts == 0.f ? 0.f : (float)((double)st.h - st.ln_s), 0.f};
}

__device__ __forceinline__ void write_no_row(unsigned r, float* logp, float* entropy, f32x4* state) {
  logp[r] = 0.f;
  if (entropy) entropy[r] = 0.f;
  if (state) state[r] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// ---- pass 1: the statistics of rows, or of parts of rows ------------------------------------------------------------------
// TPR threads share a part; every part of a row streams its elements once, 16 bytes a load, aligned on the input.
template <typename T, int TPR>
__device__ __forceinline__ Part stream_part(const T* x, int n, float c, int t) {
  constexpr int VEC = Type<T>::VEC;
  Part p{-INFINITY, 0.f, 0.f};
  const int head = std::min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int nv = (n - head) / VEC;
  const u32x4* v = reinterpret_cast<const u32x4*>(x + head);
  int i = t;
  for (; i + 3 * TPR < nv; i += 4 * TPR) {                     // four loads in flight
    u32x4 b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = __builtin_nontemporal_load(v + i + k * TPR);
    float f[4 * VEC];
#pragma unroll
    for (int k = 0; k < 4; ++k) Type<T>::unpack(b[k], f + k * VEC);
    take<4 * VEC>(p, f, c);
  }
  for (; i < nv; i += TPR) {
    float f[VEC];
    Type<T>::unpack(v[i], f);
    take<VEC>(p, f, c);
  }
  if (t < head) {
    const float f = (float)x[t];
    take<1>(p, &f, c);
  }
  const int done = head + nv * VEC;
  if (t < n - done) {
    const float f = (float)x[done + t];
    take<1>(p, &f, c);
  }
  return p;
}

struct StatsOut {
  float* logp;
  float* entropy;
  f32x4* state;
  f32x4* parts;          // [rows][splits], used where splits > 1
  unsigned* counter;     // cleared for the loss kernel behind this one
  RowGrad* clear;        // row gradients that a loss kernel fills in for the rows it owns
};

template <typename T, int TPR>
__global__ __launch_bounds__(NT) void stats_kernel(Logits p, int splits, int chunk, StatsOut o) {
  constexpr int WPR = TPR / 64;                                // waves of a part
  __shared__ Part red[NT / 64];
  const int t = threadIdx.x % TPR;
  const unsigned long long part = (unsigned long long)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const unsigned r = (unsigned)(part / splits);
  const int sp = (int)(part % splits);
  if (blockIdx.x == 0 && threadIdx.x == 0 && o.counter) *o.counter = 0;
  const bool live = r < p.rows;
  const long long label = live && p.labels ? load_index(p.labels, p.labels64, r) : p.ignore;
  if (live && label != p.ignore) {
    const int lo = std::min((long long)sp * chunk, (long long)p.vocab), hi = std::min((long long)lo + chunk, (long long)p.vocab);
    const T* x = reinterpret_cast<const T*>(p.x) + row_offset(p, r) + lo;
    Part q = wave_join(stream_part<T, TPR>(x, hi - lo, p.c, t), p.c);
    if (WPR > 1) {                                             // the whole block has this row: the barriers are uniform
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = q;
      __syncthreads();
      q = red[0];
#pragma unroll
      for (int w = 1; w < WPR; ++w) q = join(q, red[w], p.c);
    }
    if (t == 0) {
      if (splits > 1) o.parts[part] = f32x4{q.m, q.s, q.w, 0.f};
      else write_row<T>(p, r, label, q, o.logp, o.entropy, o.state);
    }
  } else if (live && t == 0 && sp == 0) {
    write_no_row(r, o.logp, o.entropy, o.state);
  }
  if (live && t == 0 && sp == 0 && o.clear) o.clear[r] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// joins the parts of each row: a wave a row
template <typename T>
__global__ __launch_bounds__(NT) void join_kernel(Logits p, int splits, StatsOut o) {
  const unsigned r = blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (r >= p.rows) return;
  const long long label = load_index(p.labels, p.labels64, r);
  if (label == p.ignore) return;
  Part q{-INFINITY, 0.f, 0.f};
  if (lane < splits) {
    const f32x4 v = o.parts[(size_t)r * splits + lane];
    q = Part{v[0], v[1], v[2]};
  }
  q = wave_join(q, p.c);
  if (lane == 0) write_row<T>(p, r, label, q, o.logp, o.entropy, o.state);
}

// ---- pass 2: gradient rows -----------------------------------------------------------------------------------------------
// g_j = (alpha + gamma d_j) e_j, the label's entry + patch.  A row with alpha = gamma = patch = 0 is zero whatever its
// logits hold, and they are not read.
struct GradIn {
  const RowGrad* row;        // losses: coefficients for an upstream gradient of 1 ...
  const float* gout;         // ... and that upstream gradient (device scalar, null = 1)
  int skip_if_one;           // grad already holds the rows for an upstream gradient of 1
  const f32x4* state;        // log-probabilities: statistics and the rows' own upstream gradients
  const float* g_logp;
  const float* g_entropy;
};

__device__ __forceinline__ RowGrad row_grad(const Logits& p, const GradIn& g, unsigned r, float scale, bool counts) {
  RowGrad v{0.f, 0.f, 0.f, 0.f};
  if (!counts) return v;
  if (g.row) {
    v = g.row[r];
    v[1] *= scale; v[2] *= scale; v[3] *= scale;
    return v;
  }
  const f32x4 s = g.state[r];
  const float a = g.g_logp ? g.g_logp[r] : 0.f, b = g.g_entropy ? g.g_entropy[r] : 0.f;
  if (s[1] == 0.f) return v;
  v[0] = s[0];
  v[1] = -(a + b * s[2]) * s[1];
  v[2] = -b * (float)LN2 * s[1];
  v[3] = a / (float)p.tau;
  return v;
}

template <typename T, int TPR>
__global__ __launch_bounds__(NT) void grad_kernel(Logits p, GradIn g, int splits, int chunk, T* __restrict__ grad) {
  constexpr int VEC = Type<T>::VEC;
  const float scale = g.gout ? g.gout[0] : 1.f;
  if (g.skip_if_one && scale == 1.f) return;
  const int t = threadIdx.x % TPR;
  const unsigned long long part = (unsigned long long)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const unsigned r = (unsigned)(part / splits);
  if (r >= p.rows) return;
  const int lo = std::min((long long)(part % splits) * chunk, (long long)p.vocab);
  const int n = std::min((long long)chunk, (long long)p.vocab - lo);
  const long long label = load_index(p.labels, p.labels64, r);
  const RowGrad k = row_grad(p, g, r, scale, label != p.ignore);
  T* out = grad + (size_t)r * p.vocab + lo;
  const T* x = reinterpret_cast<const T*>(p.x) + row_offset(p, r) + lo;
  const bool zero = k[1] == 0.f && k[2] == 0.f && k[3] == 0.f;
  const int at = zero ? -1 : (int)std::max(-1ll, std::min(label - lo, (long long)n));
  // aligned on the output where the row is only written, on the input otherwise
  const int head = std::min(n, (int)((16 - (reinterpret_cast<uintptr_t>(zero ? out : x) & 15)) & 15) / (int)sizeof(T));
  const int nv = (n - head) / VEC;
  const u32x4* v = reinterpret_cast<const u32x4*>(x + head);
  u32x4_u* o = reinterpret_cast<u32x4_u*>(out + head);
  const auto one = [&](float f, int j) {
    const float d = (f - k[0]) * p.c, e = __builtin_amdgcn_exp2f(d);
    return fmaf(fmaxf(d, D_MIN), k[2], k[1]) * e + (j == at ? k[3] : 0.f);
  };
  for (int i = t; i < nv; i += TPR) {
    u32x4 w = {0u, 0u, 0u, 0u};
    if (!zero) {
      float f[VEC];
      Type<T>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = one(f[j], head + i * VEC + j);
      w = Type<T>::pack(f);
    }
    o[i] = w;
  }
  if (t < head) out[t] = zero ? (T)0.f : (T)one((float)x[t], t);
  const int done = head + nv * VEC;
  if (t < n - done) out[done + t] = zero ? (T)0.f : (T)one((float)x[done + t], done + t);
}

// ---- sequences ----------------------------------------------------------------------------------------------------------
// Rows [start, end) of sequence s: cu[s], cu[s + 1] of a packed batch (clamped to the rows that are there), or the s-th
// `inner` rows of a padded one.
struct Sequences {
  const int* cu;
  unsigned count;
  unsigned inner;
  unsigned rows;
};

__device__ __forceinline__ unsigned clamp_row(int v, unsigned rows) { return v < 0 ? 0u : std::min((unsigned)v, rows); }

__device__ __forceinline__ void sequence(const Sequences& q, unsigned s, unsigned& start, unsigned& end) {
  if (q.cu) {
    start = clamp_row(q.cu[s], q.rows);
    end = std::max(start, clamp_row(q.cu[s + 1], q.rows));
  } else {
    start = s * q.inner;
    end = start + q.inner;
  }
}

// the sequence of row r of a packed batch, or -1: the last s with cu[s] <= r, found by halving
__device__ __forceinline__ int sequence_of(const Sequences& q, unsigned r) {
  if (!q.cu) return (int)(r / q.inner);
  unsigned lo = 0, hi = q.count;
  while (lo < hi) {                                             // first s with cu[s + 1] > r
    const unsigned mid = (lo + hi) / 2;
    if (q.cu[mid + 1] > (int)r) hi = mid;
    else lo = mid + 1;
  }
  return lo < q.count && q.cu[lo] <= (int)r ? (int)lo : -1;
}

__device__ __forceinline__ double block_sum64(double v, double* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) t += red[w];
  return t;
}

// True in exactly one block: the last one to come here.  What the other blocks wrote before is visible to it.
__device__ __forceinline__ bool last_block(unsigned* counter) {
  __shared__ unsigned seen;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) seen = atomicAdd(counter, 1u);
  __syncthreads();
  const bool last = seen == gridDim.x - 1;
  if (last) __threadfence();
  return last;
}

// ---- preference loss ---------------------------------------------------------------------------------------------------
struct PrefIn {
  Sequences seq;             // 2 P sequences: the chosen ones, then the rejected ones
  const float* logp;
  const f32x4* state;
  const float* ref;          // [2 P] or null
  int kind, average;
  double beta, smoothing, scale;
  double* each;              // [P] workspace
  unsigned* counter;
  float* loss;
  float* rewards;            // beta (L - ref) of each sequence
  RowGrad* row;              // null without a gradient
};

__device__ __forceinline__ double log1p_exp(double v) { return v > 0 ? v + log1p(exp(-v)) : log1p(exp(v)); }

// A block a pair: the two sums in fp64, the pair's loss and its slope, the rows' coefficients; the last block takes the mean.
__global__ __launch_bounds__(1024) void pref_kernel(Logits p, PrefIn q) {
  __shared__ double red[16];
  const unsigned pairs = q.seq.count / 2, pair = blockIdx.x;
  double ratio[2];
  double inv[2];
  for (int side = 0; side < 2; ++side) {
    unsigned start, end;
    sequence(q.seq, pair + side * pairs, start, end);
    double sum = 0, n = 0;
    for (unsigned r = start + threadIdx.x; r < end; r += blockDim.x) {
      sum += (double)q.logp[r];
      if (load_index(p.labels, p.labels64, r) != p.ignore) n += 1;
    }
    sum = block_sum64(sum, red);
    n = q.average ? block_sum64(n, red) : 1.0;
    inv[side] = n > 0 ? 1.0 / n : 0.0;
    ratio[side] = sum * (n > 0 ? 1.0 / n : 1.0) - (q.ref ? (double)q.ref[pair + side * pairs] : 0.0);
  }
  const double h = ratio[0] - ratio[1], z = q.beta * h;
  double loss, slope;
  if (q.kind == ST_PREF_SIGMOID) {
    loss = (1 - q.smoothing) * log1p_exp(-z) + q.smoothing * log1p_exp(z);
    slope = q.beta * (q.smoothing / (1 + exp(-z)) - (1 - q.smoothing) / (1 + exp(z)));
  } else if (q.kind == ST_PREF_IPO) {
    const double v = h - 0.5 / q.beta;
    loss = v * v;
    slope = 2 * v;
  } else {
    loss = z < 1 ? 1 - z : (z >= 1 ? 0.0 : z);                  // a NaN stays one
    slope = z < 1 ? -q.beta : (z >= 1 ? 0.0 : z);
  }
  if (threadIdx.x == 0) {
    q.each[pair] = loss;
    q.rewards[pair] = (float)(q.beta * ratio[0]);
    q.rewards[pairs + pair] = (float)(q.beta * ratio[1]);
  }
  if (q.row)
    for (int side = 0; side < 2; ++side) {
      unsigned start, end;
      sequence(q.seq, pair + side * pairs, start, end);
      const float a = (float)((side ? -slope : slope) * inv[side] * q.scale / pairs);
      for (unsigned r = start + threadIdx.x; r < end; r += blockDim.x) {
        const f32x4 s = q.state[r];
        const bool counts = load_index(p.labels, p.labels64, r) != p.ignore && s[1] != 0.f;
        q.row[r] = counts ? f32x4{s[0], -a * s[1], 0.f, a / (float)p.tau} : f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  if (last_block(q.counter)) {
    double sum = 0;
    for (unsigned i = threadIdx.x; i < pairs; i += blockDim.x) sum += __hip_atomic_load(q.each + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sum = block_sum64(sum, red);
    if (threadIdx.x == 0) q.loss[0] = (float)(q.scale * sum / pairs);
  }
}

// ---- clipped policy loss --------------------------------------------------------------------------------------------------
struct PolicyIn {
  Sequences seq;
  const float* logp;
  const float* entropy;
  const f32x4* state;
  const float* old_logp;
  const float* adv;
  int adv_per_sequence;
  const float* ref;          // null: no KL term
  double low, high, kl, ent, scale;
  int per_sequence;          // mean of the sequences' means; else the mean over tokens
  int* count;                // [sequences] labels of each (per_sequence)
  double* norm;              // 1 / tokens or 1 / sequences that hold any
  double* sums;              // [4][blocks]
  unsigned* counter;
  float* loss;
  float* stats;              // surrogate, KL, entropy, clipped share
  RowGrad* row;
};

// How many labels count, over all rows or a sequence each (one block; whole numbers, so their order does not matter).
__global__ __launch_bounds__(1024) void count_kernel(Logits p, PolicyIn q) {
  __shared__ double red[16];
  double n = 0;
  if (q.per_sequence) {
    for (unsigned s = threadIdx.x >> 6; s < q.seq.count; s += blockDim.x >> 6) {
      unsigned start, end;
      sequence(q.seq, s, start, end);
      int c = 0;
      for (unsigned r = start + (threadIdx.x & 63); r < end; r += 64) c += load_index(p.labels, p.labels64, r) != p.ignore;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) c += __shfl_xor(c, off, 64);
      if ((threadIdx.x & 63) == 0) {
        q.count[s] = c;
        n += c > 0;
      }
    }
  } else {
    unsigned first = 0, end = q.seq.rows, unused;
    if (q.seq.cu) {                                             // rows outside every sequence do not count
      sequence(q.seq, 0, first, unused);
      sequence(q.seq, q.seq.count - 1, unused, end);
    }
    for (unsigned r = first + threadIdx.x; r < end; r += blockDim.x) n += load_index(p.labels, p.labels64, r) != p.ignore;
  }
  n = block_sum64(n, red);
  if (threadIdx.x == 0) {
    *q.norm = n > 0 ? 1.0 / n : 0.0;
    *q.counter = 0;
  }
}

struct TokenTerms {
  double part, kl, clipped;  // surrogate, KL estimate, 1 where the clip holds the ratio
  double a;                  // d (surrogate + kl_coef KL) / d logp
};

__device__ __forceinline__ TokenTerms token_terms(const PolicyIn& q, unsigned r, double logp, double adv) {
  TokenTerms t;
  const double ratio = exp(logp - (double)q.old_logp[r]);
  const bool over = adv > 0 && ratio > 1 + q.high, under = adv < 0 && ratio < 1 - q.low;
  t.clipped = over || under;
  t.part = -adv * (over ? 1 + q.high : under ? 1 - q.low : ratio);
  t.a = t.clipped != 0 ? 0.0 : -adv * ratio;
  t.kl = 0;
  if (q.ref) {
    const double d = (double)q.ref[r] - logp, e = expm1(d);     // exp(d) - 1 - d without its cancellation near 0
    t.kl = e - d;
    t.a -= q.kl * e;
  }
  return t;
}

// a thread a row; the last block sums the blocks' sums in order
__global__ __launch_bounds__(NT) void policy_kernel(Logits p, PolicyIn q) {
  __shared__ double red[NT / 64];
  const unsigned r = blockIdx.x * NT + threadIdx.x;
  double sum[4] = {0, 0, 0, 0};
  if (r < p.rows) {
    RowGrad g{0.f, 0.f, 0.f, 0.f};
    const int s = sequence_of(q.seq, r);
    if (s >= 0 && load_index(p.labels, p.labels64, r) != p.ignore) {
      const double w = q.per_sequence ? *q.norm / q.count[s] : *q.norm;
      const TokenTerms t = token_terms(q, r, (double)q.logp[r], (double)q.adv[q.adv_per_sequence ? s : r]);
      sum[0] = w * t.part;
      sum[1] = w * t.kl;
      sum[2] = w * (double)q.entropy[r];
      sum[3] = w * t.clipped;
      const f32x4 st = q.state[r];
      const double a = q.scale * w * t.a, b = -q.scale * w * q.ent;
      if (st[1] != 0.f)
        g = f32x4{st[0], (float)(-(a + b * (double)st[2]) * (double)st[1]), (float)(-b * LN2 * (double)st[1]), (float)(a / p.tau)};
    }
    if (q.row) q.row[r] = g;
  }
  for (int k = 0; k < 4; ++k) {
    const double v = block_sum64(sum[k], red);
    if (threadIdx.x == 0) q.sums[(size_t)k * gridDim.x + blockIdx.x] = v;
  }
  if (last_block(q.counter)) {
    double tot[4];
    for (int k = 0; k < 4; ++k) {
      double v = 0;
      for (unsigned i = threadIdx.x; i < gridDim.x; i += NT)
        v += __hip_atomic_load(q.sums + (size_t)k * gridDim.x + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      tot[k] = block_sum64(v, red);
    }
    if (threadIdx.x == 0) {
      q.loss[0] = (float)(q.scale * (tot[0] + (q.ref ? q.kl * tot[1] : 0.0) - (q.ent != 0 ? q.ent * tot[2] : 0.0)));
      for (int k = 0; k < 4; ++k) q.stats[k] = (float)tot[k];
    }
  }
}

// ---- distillation from a teacher's top logits ---------------------------------------------------------------------------------
// The list of a row is K pairs (index, value); an index below 0 is unused.  p_k is the teacher's probability of entry k,
// P their sum, and with a bucket for all that is not listed rest = max(0, 1 - P) and q_rest the student's mass off the list:
//   loss / tau^2 = sum p_k (ln p_k - ln q_k) + rest (ln rest - ln q_rest)
//   d / dx_j = tau g (Q q_j - p_j) on the list,  tau g q_j (Q - rest / q_rest) off it,  Q = P + rest
// q_rest comes from its own sum over the elements off the list (a bitmap in LDS tells them apart): 1 - sum q_k would keep
// no digit of it where the student is sure of a listed token.  Entries that name the same token add up.
struct ListIn {
  const void* idx;           // [rows][k] int64 or int32
  int idx64;
  const float* val;          // [rows][k]
  int k;
  const unsigned char* mask; // [rows] or null
  int tail;
  double scale;
  const double* norm;        // 1 / rows that count
  f32x4* off;                // [rows][splits]: statistics of the elements off the list; [3]: an index twice
  f32x4* row;                // [rows][2]: (m_off, alpha_off, m, alpha_on), (vref, gz, repeated, -)
  double* sums;              // [blocks]
  unsigned* counter;
  float* loss;
};

struct WaveGroup {
  static constexpr int SIZE = 64;
  int t;
  __device__ WaveGroup() : t(threadIdx.x & 63) {}
  __device__ double sum(double v) const {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
  }
  __device__ float max(float v) const {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
  }
};

// The loss of row r and what its gradient needs, from the statistics `off` of the elements off the list.  Every thread of
// the group gets the same result.
template <typename T, typename G>
__device__ double list_terms(const Logits& p, const ListIn& q, unsigned r, Part off, bool repeated, const G& g, f32x4* row) {
  const T* x = reinterpret_cast<const T*>(p.x) + row_offset(p, r);
  const size_t first = (size_t)r * q.k;
  float m = off.m, vref = -INFINITY;
  double bad = 0;
  for (int k = g.t; k < q.k; k += G::SIZE) {
    const long long j = load_index(q.idx, q.idx64, first + k);
    if (j < 0) continue;
    if (j >= p.vocab) { bad = 1; continue; }
    m = fmaxf(m, (float)x[j]);
    const float v = q.val[first + k];
    vref = fmaxf(vref, v == v ? v : INFINITY);
  }
  m = g.max(m);
  vref = q.tail ? 0.f : g.max(vref);
  const float ref = finite_ref(m);
  if (vref == -INFINITY) vref = 0.f;                            // an empty list, or one without mass
  const double it = q.tail ? 1.0 : 1.0 / p.tau;
  double z = 0, s_list = 0, w_list = 0, listed = 0;
  for (int k = g.t; k < q.k; k += G::SIZE) {
    const long long j = load_index(q.idx, q.idx64, first + k);
    if (j < 0 || j >= p.vocab) continue;
    z += exp(((double)q.val[first + k] - (double)vref) * it);
    bool again = false;                                         // counted under an earlier entry
    if (repeated)
      for (int i = 0; i < k && !again; ++i) again = load_index(q.idx, q.idx64, first + i) == j;
    if (again) continue;
    const float d = ((float)x[j] - ref) * p.c, e = __builtin_amdgcn_exp2f(d);
    s_list += (double)e;
    w_list += (double)(fmaxf(d, D_MIN) * e);
    listed += 1;
  }
  z = g.sum(z);
  s_list = g.sum(s_list);
  w_list = g.sum(w_list);
  listed = g.sum(listed);
  bad = g.sum(bad);
  // the whole row from the two parts, seen from ref
  float s_off = off.s, w_off = off.w;
  rebase(s_off, w_off, off.m, ref, p.c);
  const double eps = (double)p.c * LN2 * p.tau - 1.0;
  const double s = s_list + (double)s_off;
  const double ln_s = s == 0 ? -INFINITY : log(s - eps * LN2 * (w_list + (double)w_off));
  double mass = 0, loss = 0;
  for (int k = g.t; k < q.k; k += G::SIZE) {
    const long long j = load_index(q.idx, q.idx64, first + k);
    if (j < 0 || j >= p.vocab) continue;
    const double lv = ((double)q.val[first + k] - (double)vref) * it;
    const double pk = q.tail ? exp(lv) : (z > 0 ? exp(lv) / z : (z == 0 ? 0.0 : z));
    mass += pk;
    if (pk != 0) loss += pk * ((q.tail ? lv : lv - log(z)) - (((double)(float)x[j] - (double)ref) / p.tau - ln_s));
  }
  mass = g.sum(mass);
  loss = g.sum(loss);
  const double rest = q.tail && listed < (double)p.vocab ? (mass < 1 ? 1 - mass : (mass >= 1 ? 0.0 : mass)) : 0.0;
  double to_rest = 0;
  if (rest != 0) {
    const double ln_off = off.s == 0.f ? -INFINITY : log((double)off.s - eps * LN2 * (double)off.w) + ((double)finite_ref(off.m) - (double)ref) / p.tau;
    loss += rest * (log(rest) - (ln_off - ln_s));
    if (off.s != 0.f) to_rest = rest / (double)off.s;
  }
  const double w = q.scale * *q.norm, gr = w * p.tau, total = mass + rest;
  const double on = s == 0 ? 0.0 : gr * total / s;
  const double shift = exp2((double)((finite_ref(off.m) - ref) * p.c));
  float a_off = s == 0 || off.s == 0.f ? 0.f : (float)(on * shift - gr * to_rest);
  float a_on = (float)on, gz = s == 0 ? 0.f : (float)(q.tail ? gr : (z > 0 ? gr / z : (z == 0 ? 0.0 : z)));
  if (bad != 0) {
    loss = NAN;
    a_off = a_on = NAN;
  }
  if (row) {
    row[0] = f32x4{finite_ref(off.m), a_off, ref, a_on};
    row[1] = f32x4{vref, gz, repeated ? 1.f : 0.f, (s == 0 || total == 0) && bad == 0 ? 0.f : 1.f};
  }
  return w * p.tau * p.tau * loss;
}

// Bits of the listed elements of [lo, lo + n), shifted so that a 16-byte vector's elements start at a multiple of VEC;
// returns whether this thread met an index that was set before.
__device__ __forceinline__ bool mark(uint32_t* bits, const ListIn& q, unsigned r, int lo, int n, int shift, int t, int threads) {
  bool twice = false;
  for (int k = t; k < q.k; k += threads) {
    const long long j = load_index(q.idx, q.idx64, (size_t)r * q.k + k) - lo;
    if (j < 0 || j >= n) continue;
    const unsigned at = (unsigned)j + shift, bit = 1u << (at & 31);
    twice |= (atomicOr(bits + (at >> 5), bit) & bit) != 0;
  }
  return twice;
}

__device__ __forceinline__ bool marked(const uint32_t* bits, unsigned at) { return bits[at >> 5] >> (at & 31) & 1; }

template <typename T, int TPR>
__global__ __launch_bounds__(NT) void list_stats_kernel(Logits p, ListIn q, int splits, int chunk) {
  constexpr int VEC = Type<T>::VEC, WPR = TPR / 64;
  extern __shared__ uint32_t all_bits[];
  __shared__ Part red[NT / 64];
  __shared__ int any[NT / 64];
  const int t = threadIdx.x % TPR, words = (chunk + VEC + 31) / 32;
  uint32_t* bits = all_bits + (threadIdx.x / TPR) * words;
  const unsigned long long part = (unsigned long long)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const unsigned r = (unsigned)(part / splits);
  const bool live = r < p.rows && (!q.mask || q.mask[r]);
  const int lo = live ? std::min((long long)(part % splits) * chunk, (long long)p.vocab) : 0;
  const int n = live ? std::min((long long)chunk, (long long)p.vocab - lo) : 0;
  const T* x = reinterpret_cast<const T*>(p.x) + (live ? row_offset(p, r) + lo : 0);
  const int head = std::min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int shift = (VEC - head % VEC) % VEC;
  for (int i = t; i < words; i += TPR) bits[i] = 0;
  __syncthreads();
  const bool twice = live && mark(bits, q, r, lo, n, shift, t, TPR);
  __syncthreads();
  Part s{-INFINITY, 0.f, 0.f};
  const int nv = (n - head) / VEC;
  const u32x4* v = reinterpret_cast<const u32x4*>(x + head);
  for (int i = t; i < nv; i += TPR) {
    float f[VEC];
    Type<T>::unpack(__builtin_nontemporal_load(v + i), f);
    const unsigned at = head + i * VEC + shift;
    const uint32_t on = bits[at >> 5] >> (at & 31) & ((1u << VEC) - 1);
    if (on)
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = on >> j & 1 ? -INFINITY : f[j];
    take<VEC>(s, f, p.c);
  }
  const int done = head + nv * VEC;
  for (int part_of = 0; part_of < 2; ++part_of) {               // the elements before and behind the vectors
    const int j = part_of ? done + t : t;
    if (j < (part_of ? n : head) && !marked(bits, j + shift)) {
      const float f = (float)x[j];
      take<1>(s, &f, p.c);
    }
  }
  s = wave_join(s, p.c);
  int flag = __any(twice) ? 1 : 0;
  if (WPR > 1) {
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6] = s;
      any[threadIdx.x >> 6] = flag;
    }
    __syncthreads();
    s = red[0];
    flag = any[0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      s = join(s, red[w], p.c);
      flag |= any[w];
    }
  }
  if (live && t == 0) q.off[part] = f32x4{s.m, s.s, s.w, flag ? 1.f : 0.f};
}

// a wave a row; the last block sums
template <typename T>
__global__ __launch_bounds__(NT) void list_kernel(Logits p, ListIn q, int splits) {
  __shared__ double red[NT / 64];
  const WaveGroup g;
  double sum = 0;
  for (unsigned r = blockIdx.x * (NT / 64) + (threadIdx.x >> 6); r < p.rows; r += gridDim.x * (NT / 64)) {
    f32x4* row = q.row ? q.row + 2 * (size_t)r : nullptr;
    if (q.mask && !q.mask[r]) {
      if (row && g.t < 2) row[g.t] = f32x4{0.f, 0.f, 0.f, 0.f};
      continue;
    }
    Part s{-INFINITY, 0.f, 0.f};
    bool repeated = false;
    if (g.t < splits) {
      const f32x4 v = q.off[(size_t)r * splits + g.t];
      s = Part{v[0], v[1], v[2]};
      repeated = v[3] != 0.f;
    }
    s = wave_join(s, p.c);
    f32x4 to[2];
    const double loss = list_terms<T>(p, q, r, s, __any(repeated), g, to);
    if (row && g.t < 2) row[g.t] = to[g.t];
    if (g.t == 0) sum += loss;
  }
  sum = block_sum64(sum, red);
  if (threadIdx.x == 0) q.sums[blockIdx.x] = sum;
  if (last_block(q.counter)) {
    double v = 0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += NT) v += __hip_atomic_load(q.sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    v = block_sum64(v, red);
    if (threadIdx.x == 0) q.loss[0] = (float)v;
  }
}

// the rows that the mask counts (one block)
__global__ __launch_bounds__(1024) void count_mask_kernel(const unsigned char* mask, unsigned rows, double* norm, unsigned* counter) {
  __shared__ double red[16];
  double n = 0;
  if (mask) {
    for (unsigned r = threadIdx.x; r < rows; r += blockDim.x) n += mask[r] != 0;
    n = block_sum64(n, red);
  } else {
    n = rows;
  }
  if (threadIdx.x == 0) {
    *norm = n > 0 ? 1.0 / n : 0.0;
    *counter = 0;
  }
}

// The entries of a row's list that lie in [lo, lo + n), over the stream that wrote them as if they were off it.
template <typename T>
__device__ __forceinline__ void patch_list(const Logits& p, const ListIn& q, unsigned r, const f32x4& a, const f32x4& b, float scale, int lo,
                                           int n, const T* x, T* out, int t, int threads) {
  const float cv = q.tail ? (float)(1.0 / LN2) : p.c;
  const size_t first = (size_t)r * q.k;
  for (int k = t; k < q.k; k += threads) {
    const long long j = load_index(q.idx, q.idx64, first + k) - lo;
    if (j < 0 || j >= n) continue;
    float pk = 0.f;
    if (b[2] != 0.f) {                                          // an index twice in this row: its entries' sum, in order
      for (int i = 0; i < q.k; ++i)
        if (load_index(q.idx, q.idx64, first + i) - lo == j) pk += __builtin_amdgcn_exp2f((q.val[first + i] - b[0]) * cv);
    } else {
      pk = __builtin_amdgcn_exp2f((q.val[first + k] - b[0]) * cv);
    }
    const float e = __builtin_amdgcn_exp2f(((float)x[j] - a[2]) * p.c);
    out[j] = (T)(scale * (a[3] * e - b[1] * pk));
  }
}

template <typename T, int TPR>
__global__ __launch_bounds__(NT) void list_grad_kernel(Logits p, ListIn q, const float* gout, int skip_if_one, int splits, int chunk,
                                                       T* __restrict__ grad) {
  constexpr int VEC = Type<T>::VEC;
  const float scale = gout ? gout[0] : 1.f;
  if (skip_if_one && scale == 1.f) return;
  const int t = threadIdx.x % TPR;
  const unsigned long long part = (unsigned long long)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const unsigned r = (unsigned)(part / splits);
  const bool live = r < p.rows;
  const int lo = live ? std::min((long long)(part % splits) * chunk, (long long)p.vocab) : 0;
  const int n = live ? std::min((long long)chunk, (long long)p.vocab - lo) : 0;
  const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
  const f32x4 a = live ? q.row[2 * (size_t)r] : zero4, b = live ? q.row[2 * (size_t)r + 1] : zero4;
  const bool zero = b[3] == 0.f;
  T* out = grad + (live ? (size_t)r * p.vocab + lo : 0);
  const T* x = reinterpret_cast<const T*>(p.x) + (live ? row_offset(p, r) + lo : 0);
  const int head = std::min(n, (int)((16 - (reinterpret_cast<uintptr_t>(zero ? out : x) & 15)) & 15) / (int)sizeof(T));
  const int nv = (n - head) / VEC;
  const u32x4* v = reinterpret_cast<const u32x4*>(x + head);
  u32x4_u* o = reinterpret_cast<u32x4_u*>(out + head);
  const float alpha = a[1] * scale;
  const auto one = [&](float f) { return alpha * __builtin_amdgcn_exp2f((f - a[0]) * p.c); };
  for (int i = t; i < nv; i += TPR) {
    u32x4 w = {0u, 0u, 0u, 0u};
    if (!zero) {
      float f[VEC];
      Type<T>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = one(f[j]);
      w = Type<T>::pack(f);
    }
    o[i] = w;
  }
  if (t < head) out[t] = zero ? (T)0.f : (T)one((float)x[t]);
  const int done = head + nv * VEC;
  if (t < n - done) out[done + t] = zero ? (T)0.f : (T)one((float)x[done + t]);
  __syncthreads();                                              // a listed element is written twice, in this order
  if (!zero) patch_list<T>(p, q, r, a, b, scale, lo, n, x, out, t, TPR);
}

// ---- host side --------------------------------------------------------------------------------------------------------------
struct Split {
  int tpr, splits, chunk;
};

// Threads of a part and parts of a row.  A row of up to 4 KB is a wave's work (four rows a block share no barrier); a
// longer one is a block's.  Where the rows alone would leave compute units idle, a row is cut until there are about four
// blocks for each of the 256, in parts of 8 KB at least (two 16-byte loads a thread).
Split split_of(unsigned rows, int vocab, int size) {
  const long long bytes = (long long)vocab * size;
  if (bytes <= 4096) return {64, 1, vocab};
  int s = 1;
  if (rows < 1024) s = (int)std::min<long long>(MAX_SPLITS, std::min(st::cdivll(1024, std::max(1u, rows)), bytes / 8192));
  s = std::max(1, s);
  const int per = 16 / size;
  const int chunk = (int)(st::cdivll(st::cdivll(vocab, s), per) * per);
  return {NT, (int)st::cdivll(vocab, chunk), chunk};
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

bool bad_logits(const char* who, const Logits& p, int dtype, long long rows, long long inner, long long so, long long si, int* rc) {
  *rc = ST_OK;
  if (dtype != ST_F32 && dtype != ST_BF16 && dtype != ST_F16) *rc = st::fail(ST_ERR_BAD_ARG, "%s: dtype %d", who, dtype);
  else if (rows < 0 || rows > 0x7fffffffLL || inner <= 0 || inner > 0x7fffffffLL) *rc = st::fail(ST_ERR_BAD_ARG, "%s: rows=%lld inner=%lld", who, rows, inner);
  else if (p.vocab <= 0) *rc = st::fail(ST_ERR_BAD_ARG, "%s: vocab=%d", who, p.vocab);
  else if (!(p.tau > 0) || !std::isfinite(p.tau) || !std::isfinite(p.c) || p.c == 0.f) *rc = st::fail(ST_ERR_BAD_ARG, "%s: temperature %g", who, p.tau);
  else if (so < 0 || si < 0) *rc = st::fail(ST_ERR_BAD_ARG, "%s: negative stride", who);
  else if (rows > 0 && !p.x) *rc = st::fail(ST_ERR_BAD_ARG, "%s: null logits", who);
  else if (reinterpret_cast<uintptr_t>(p.x) % (dtype == ST_F32 ? 4 : 2)) *rc = st::fail(ST_ERR_BAD_ARG, "%s: logits not aligned to their type", who);
  return *rc != ST_OK;
}

Logits make_logits(const void* x, long long rows, long long inner, long long so, long long si, int vocab, const void* labels,
                   int labels64, int ignore, double tau) {
  Logits p{};
  p.x = x;
  p.labels = labels;
  p.labels64 = labels64;
  p.ignore = ignore;
  p.inner = (unsigned)inner;
  p.s_outer = so;
  p.s_inner = si;
  p.vocab = vocab;
  p.rows = (unsigned)rows;
  p.tau = tau;
  p.c = (float)(1.0 / (LN2 * tau));
  return p;
}

int size_of(int dtype) { return dtype == ST_F32 ? 4 : 2; }

// what every forward pass needs of the workspace, one after another
struct Space {
  char* at;
  size_t used = 0;
  template <typename V>
  V* take(size_t n) {
    V* p = reinterpret_cast<V*>(at + used);
    used += align256(n * sizeof(V));
    return p;
  }
};

template <typename T>
int launch_stats_t(const char* who, const Logits& p, const StatsOut& o, hipStream_t s) {
  const Split k = split_of(p.rows, p.vocab, (int)sizeof(T));
  const long long parts = (long long)p.rows * k.splits, blocks = st::cdivll(parts, NT / k.tpr);
  if (blocks > 0x7fffffffLL) return st::fail(ST_ERR_BAD_ARG, "%s: too many rows", who);
  if (k.tpr == 64) hipLaunchKernelGGL((stats_kernel<T, 64>), dim3((unsigned)blocks), dim3(NT), 0, s, p, k.splits, k.chunk, o);
  else hipLaunchKernelGGL((stats_kernel<T, NT>), dim3((unsigned)blocks), dim3(NT), 0, s, p, k.splits, k.chunk, o);
  if (k.splits > 1) hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)st::cdivll(p.rows, NT / 64)), dim3(NT), 0, s, p, k.splits, o);
  return st::check_launch(who);
}

int launch_stats(const char* who, int dtype, const Logits& p, const StatsOut& o, hipStream_t s) {
  if (dtype == ST_F32) return launch_stats_t<float>(who, p, o, s);
  if (dtype == ST_BF16) return launch_stats_t<__bf16>(who, p, o, s);
  return launch_stats_t<_Float16>(who, p, o, s);
}

template <typename T>
int launch_grad_t(const char* who, const Logits& p, const GradIn& g, void* grad, hipStream_t s) {
  // parts of 16 KB: four 16-byte loads a thread, and enough blocks whatever the number of rows
  const long long bytes = (long long)p.vocab * (long long)sizeof(T);
  const int tpr = bytes <= 4096 ? 64 : NT;
  const int chunk = bytes <= 4096 ? p.vocab : 16384 / (int)sizeof(T);
  const int splits = (int)st::cdivll(p.vocab, chunk);
  const long long blocks = st::cdivll((long long)p.rows * splits, NT / tpr);
  if (blocks > 0x7fffffffLL) return st::fail(ST_ERR_BAD_ARG, "%s: too many rows", who);
  if (tpr == 64) hipLaunchKernelGGL((grad_kernel<T, 64>), dim3((unsigned)blocks), dim3(NT), 0, s, p, g, splits, chunk, (T*)grad);
  else hipLaunchKernelGGL((grad_kernel<T, NT>), dim3((unsigned)blocks), dim3(NT), 0, s, p, g, splits, chunk, (T*)grad);
  return st::check_launch(who);
}

int launch_grad(const char* who, int dtype, const Logits& p, const GradIn& g, void* grad, hipStream_t s) {
  if (dtype == ST_F32) return launch_grad_t<float>(who, p, g, grad, s);
  if (dtype == ST_BF16) return launch_grad_t<__bf16>(who, p, g, grad, s);
  return launch_grad_t<_Float16>(who, p, g, grad, s);
}

size_t parts_bytes(long long rows, int vocab, int size) {
  if (rows <= 0 || rows > 0x7fffffffLL || vocab <= 0) return 0;
  const Split k = split_of((unsigned)rows, vocab, size);
  return k.splits > 1 ? align256((size_t)rows * k.splits * sizeof(f32x4)) : 0;
}

// Parts of a row for the distillation: as split_of, and no part larger than a bitmap of 16 KB (131072 elements).
Split list_split_of(unsigned rows, int vocab, int size) {
  Split k = split_of(rows, vocab, size);
  const int most = 131072;
  if (k.chunk > most) {
    k.splits = (int)st::cdivll(vocab, most);
    const int per = 16 / size;
    k.chunk = (int)(st::cdivll(st::cdivll(vocab, k.splits), per) * per);
    k.splits = (int)st::cdivll(vocab, k.chunk);
  }
  return k;
}

constexpr unsigned LIST_BLOCKS = 1024;   // blocks of list_kernel, each with one sum

template <typename T>
int launch_list_t(const char* who, const Logits& p, const ListIn& q, hipStream_t s) {
  const Split k = list_split_of(p.rows, p.vocab, (int)sizeof(T));
  const long long blocks = st::cdivll((long long)p.rows * k.splits, NT / k.tpr);
  if (blocks > 0x7fffffffLL || k.splits > MAX_SPLITS) return st::fail(ST_ERR_BAD_ARG, "%s: rows=%u vocab=%d is too large", who, p.rows, p.vocab);
  const size_t lds = (size_t)(NT / k.tpr) * ((k.chunk + Type<T>::VEC + 31) / 32) * 4;
  hipLaunchKernelGGL(count_mask_kernel, dim3(1), dim3(1024), 0, s, q.mask, p.rows, const_cast<double*>(q.norm), q.counter);
  if (k.tpr == 64) hipLaunchKernelGGL((list_stats_kernel<T, 64>), dim3((unsigned)blocks), dim3(NT), lds, s, p, q, k.splits, k.chunk);
  else hipLaunchKernelGGL((list_stats_kernel<T, NT>), dim3((unsigned)blocks), dim3(NT), lds, s, p, q, k.splits, k.chunk);
  const unsigned rows4 = (unsigned)st::cdivll(p.rows, NT / 64);
  hipLaunchKernelGGL(list_kernel<T>, dim3(std::min(rows4, LIST_BLOCKS)), dim3(NT), 0, s, p, q, k.splits);
  return st::check_launch(who);
}

template <typename T>
int launch_list_grad_t(const char* who, const Logits& p, const ListIn& q, const float* gout, int skip, void* grad, hipStream_t s) {
  const long long bytes = (long long)p.vocab * (long long)sizeof(T);
  const int tpr = bytes <= 4096 ? 64 : NT;
  const int chunk = bytes <= 4096 ? p.vocab : 16384 / (int)sizeof(T);
  const int splits = (int)st::cdivll(p.vocab, chunk);
  const long long blocks = st::cdivll((long long)p.rows * splits, NT / tpr);
  if (blocks > 0x7fffffffLL) return st::fail(ST_ERR_BAD_ARG, "%s: too many rows", who);
  if (tpr == 64) hipLaunchKernelGGL((list_grad_kernel<T, 64>), dim3((unsigned)blocks), dim3(NT), 0, s, p, q, gout, skip, splits, chunk, (T*)grad);
  else hipLaunchKernelGGL((list_grad_kernel<T, NT>), dim3((unsigned)blocks), dim3(NT), 0, s, p, q, gout, skip, splits, chunk, (T*)grad);
  return st::check_launch(who);
}

}  // namespace

extern "C" size_t st_token_workspace_bytes(int dtype, long long rows, int vocab, long long sequences) {
  if (rows < 0 || sequences < 0) return 0;
  const size_t r = (size_t)rows, q = (size_t)sequences;
  return parts_bytes(rows, vocab, size_of(dtype)) + 2 * align256(r * 4) + align256(r * 16) +   // parts, logp, entropy, state
         align256(q * 8) + align256(8) + 4 * align256((r / NT + 1) * 8) + 1024;
}

extern "C" int st_token_logprobs_fwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner,
                                     int vocab, const void* labels, int labels64, int ignore, double tau, float* logp, float* entropy,
                                     float* state, void* workspace, st_stream_t stream) {
  const char* who = "st_token_logprobs_fwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, labels, labels64, ignore, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  if (rows == 0) return ST_OK;
  ST_REQUIRE(labels && logp && workspace, "%s: null pointer", who);
  StatsOut o{};
  o.logp = logp;
  o.entropy = entropy;
  o.state = reinterpret_cast<f32x4*>(state);
  o.parts = reinterpret_cast<f32x4*>(workspace);
  return launch_stats(who, dtype, p, o, (hipStream_t)stream);
}

extern "C" int st_token_logprobs_bwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner,
                                     int vocab, const void* labels, int labels64, int ignore, double tau, const float* state,
                                     const float* g_logp, const float* g_entropy, void* grad, st_stream_t stream) {
  const char* who = "st_token_logprobs_bwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, labels, labels64, ignore, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  if (rows == 0) return ST_OK;
  ST_REQUIRE(labels && state && grad, "%s: null pointer", who);
  GradIn g{};
  g.state = reinterpret_cast<const f32x4*>(state);
  g.g_logp = g_logp;
  g.g_entropy = g_entropy;
  return launch_grad(who, dtype, p, g, grad, (hipStream_t)stream);
}

extern "C" int st_preference_loss_fwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner,
                                      int vocab, const void* labels, int labels64, int ignore, const int* cu_seqlens, int pairs,
                                      const float* ref_logps, int kind, int average, double beta, double label_smoothing, double scale,
                                      float* loss, float* rewards, float* row_grad, void* workspace, st_stream_t stream) {
  const char* who = "st_preference_loss_fwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, labels, labels64, ignore, 1.0);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  ST_REQUIRE(loss && rewards && workspace && (rows == 0 || labels), "%s: null pointer", who);
  ST_REQUIRE(rows > 0 && pairs > 0 && (cu_seqlens || rows == 2LL * pairs * inner), "%s: pairs=%d rows=%lld inner=%lld", who, pairs, rows, inner);
  ST_REQUIRE(kind >= ST_PREF_SIGMOID && kind <= ST_PREF_HINGE && beta > 0 && label_smoothing >= 0 && label_smoothing < 0.5,
             "%s: kind=%d beta=%g label_smoothing=%g", who, kind, beta, label_smoothing);
  hipStream_t s = (hipStream_t)stream;
  Space w{reinterpret_cast<char*>(workspace)};
  StatsOut o{};
  PrefIn q{};
  o.parts = w.take<f32x4>(parts_bytes(rows, vocab, size_of(dtype)) / sizeof(f32x4));
  o.logp = w.take<float>((size_t)rows);
  o.state = w.take<f32x4>((size_t)rows);
  q.each = w.take<double>((size_t)pairs);
  q.counter = w.take<unsigned>(1);
  o.counter = q.counter;
  o.clear = reinterpret_cast<RowGrad*>(row_grad);
  q.seq = Sequences{cu_seqlens, 2u * (unsigned)pairs, (unsigned)inner, (unsigned)rows};
  q.logp = o.logp;
  q.state = o.state;
  q.ref = ref_logps;
  q.kind = kind;
  q.average = average;
  q.beta = beta;
  q.smoothing = label_smoothing;
  q.scale = scale;
  q.loss = loss;
  q.rewards = rewards;
  q.row = o.clear;
  if ((rc = launch_stats(who, dtype, p, o, s)) != ST_OK) return rc;
  hipLaunchKernelGGL(pref_kernel, dim3((unsigned)pairs), dim3(1024), 0, s, p, q);
  return st::check_launch(who);
}

extern "C" int st_policy_loss_fwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner, int vocab,
                                  const void* labels, int labels64, int ignore, double tau, const int* cu_seqlens, int sequences,
                                  const float* old_logps, const float* advantages, int adv_per_sequence, const float* ref_logps,
                                  double clip_low, double clip_high, double kl_coef, double entropy_coef, int per_sequence, double scale,
                                  float* loss, float* stats, float* row_grad, void* workspace, st_stream_t stream) {
  const char* who = "st_policy_loss_fwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, labels, labels64, ignore, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  ST_REQUIRE(loss && stats && workspace && (rows == 0 || (labels && old_logps && advantages)), "%s: null pointer", who);
  ST_REQUIRE(rows > 0 && sequences > 0 && (cu_seqlens || rows == (long long)sequences * inner), "%s: sequences=%d rows=%lld inner=%lld", who,
             sequences, rows, inner);
  ST_REQUIRE(clip_low >= 0 && clip_low <= 1 && clip_high >= 0, "%s: clip [%g, %g]", who, clip_low, clip_high);
  hipStream_t s = (hipStream_t)stream;
  Space w{reinterpret_cast<char*>(workspace)};
  StatsOut o{};
  PolicyIn q{};
  const unsigned blocks = (unsigned)st::cdivll(rows, NT);
  o.parts = w.take<f32x4>(parts_bytes(rows, vocab, size_of(dtype)) / sizeof(f32x4));
  o.logp = w.take<float>((size_t)rows);
  o.entropy = w.take<float>((size_t)rows);
  o.state = w.take<f32x4>((size_t)rows);
  q.count = w.take<int>((size_t)sequences);
  q.norm = w.take<double>(1);
  q.sums = w.take<double>(4 * (size_t)blocks);
  q.counter = w.take<unsigned>(1);
  q.seq = Sequences{cu_seqlens, (unsigned)sequences, (unsigned)inner, (unsigned)rows};
  q.logp = o.logp;
  q.entropy = o.entropy;
  q.state = o.state;
  q.old_logp = old_logps;
  q.adv = advantages;
  q.adv_per_sequence = adv_per_sequence;
  q.ref = ref_logps;
  q.low = clip_low;
  q.high = clip_high;
  q.kl = kl_coef;
  q.ent = entropy_coef;
  q.scale = scale;
  q.per_sequence = per_sequence;
  q.loss = loss;
  q.stats = stats;
  q.row = reinterpret_cast<RowGrad*>(row_grad);
  hipLaunchKernelGGL(count_kernel, dim3(1), dim3(1024), 0, s, p, q);
  if ((rc = launch_stats(who, dtype, p, o, s)) != ST_OK) return rc;
  hipLaunchKernelGGL(policy_kernel, dim3(blocks), dim3(NT), 0, s, p, q);
  return st::check_launch(who);
}

extern "C" int st_token_loss_bwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner, int vocab,
                                 const void* labels, int labels64, int ignore, double tau, const float* row_grad, const float* gout,
                                 void* grad, st_stream_t stream) {
  const char* who = "st_token_loss_bwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, labels, labels64, ignore, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  if (rows == 0) return ST_OK;
  ST_REQUIRE(labels && row_grad && grad, "%s: null pointer", who);
  GradIn g{};
  g.row = reinterpret_cast<const RowGrad*>(row_grad);
  g.gout = gout;
  return launch_grad(who, dtype, p, g, grad, (hipStream_t)stream);
}

extern "C" size_t st_distill_workspace_bytes(int dtype, long long rows, int vocab) {
  if (rows <= 0 || rows > 0x7fffffffLL || vocab <= 0) return 0;
  const Split k = list_split_of((unsigned)rows, vocab, size_of(dtype));
  return align256((size_t)rows * k.splits * sizeof(f32x4)) + align256(LIST_BLOCKS * sizeof(double)) + 1024;
}

extern "C" int st_distill_loss_fwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner, int vocab,
                                   const void* teacher_idx, int idx64, const float* teacher_val, int k, const unsigned char* mask, double tau,
                                   int tail, double scale, float* loss, float* row_grad, void* workspace, st_stream_t stream) {
  const char* who = "st_distill_loss_fwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, nullptr, 0, 0, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  ST_REQUIRE(rows > 0 && k > 0, "%s: rows=%lld k=%d", who, rows, k);
  ST_REQUIRE(teacher_idx && teacher_val && loss && workspace, "%s: null pointer", who);
  hipStream_t s = (hipStream_t)stream;
  const Split sp = list_split_of(p.rows, vocab, size_of(dtype));
  Space w{reinterpret_cast<char*>(workspace)};
  ListIn q{};
  q.idx = teacher_idx;
  q.idx64 = idx64;
  q.val = teacher_val;
  q.k = k;
  q.mask = mask;
  q.tail = tail;
  q.scale = scale;
  q.off = w.take<f32x4>((size_t)rows * sp.splits);
  q.sums = w.take<double>(LIST_BLOCKS);
  q.norm = w.take<double>(1);
  q.counter = w.take<unsigned>(1);
  q.row = reinterpret_cast<f32x4*>(row_grad);
  q.loss = loss;
  if (dtype == ST_F32) return launch_list_t<float>(who, p, q, s);
  if (dtype == ST_BF16) return launch_list_t<__bf16>(who, p, q, s);
  return launch_list_t<_Float16>(who, p, q, s);
}

extern "C" int st_distill_loss_bwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner, int vocab,
                                   const void* teacher_idx, int idx64, const float* teacher_val, int k, double tau, int tail,
                                   const float* row_grad, const float* gout, void* grad, st_stream_t stream) {
  const char* who = "st_distill_loss_bwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, nullptr, 0, 0, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  if (rows == 0) return ST_OK;
  ST_REQUIRE(teacher_idx && teacher_val && row_grad && grad && k > 0, "%s: null pointer", who);
  ListIn q{};
  q.idx = teacher_idx;
  q.idx64 = idx64;
  q.val = teacher_val;
  q.k = k;
  q.tail = tail;
  q.row = const_cast<f32x4*>(reinterpret_cast<const f32x4*>(row_grad));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == ST_F32) return launch_list_grad_t<float>(who, p, q, gout, 0, grad, s);
  if (dtype == ST_BF16) return launch_list_grad_t<__bf16>(who, p, q, gout, 0, grad, s);
  return launch_list_grad_t<_Float16>(who, p, q, gout, 0, grad, s);
}
