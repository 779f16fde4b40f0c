// Shared device code of the losses over rows of logits (token_losses.hip, token_distill.hip) for gfx950.
//
// One row of logits x[0..V) at temperature tau, in the base-2 domain of the hardware's exponential:
//
//   c = log2(e) / tau     m = max x     d_j = (x_j - m) c     e_j = 2^d_j     S = sum e_j     W = sum e_j d_j
//   log q_j = ln2 d_j - ln S            entropy H = ln S - ln2 W / S
//
// Every loss here reaches x through the label's log-probability and the entropy, or through a short list of entries, so
// every gradient row is   g_j = (alpha + gamma d_j) e_j   plus a few patched entries.
//
// The difference x - m comes before the factor c: the lowest value of a type used as a mask cannot overflow against
// itself, and a row that holds nothing else is the uniform distribution that the formula gives.  A row of -inf only has
// S = 0: no distribution, log-probability -inf, entropy 0, gradient 0.
//
// Sums of a row are fp32 per thread and over a fixed tree; what a row is reduced to is finished in fp64 (one wave a row),
// because a sequence's sum of hundreds of log-probabilities is compared with another model's: c's own rounding (relative
// 2^-25) shifts every term the same way, and W, which is d S / d ln c up to a factor, takes that shift out again.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "common.h"

namespace st_token {

constexpr int NT = 256;                  // threads of a streaming block
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

// e_j and e_j d_j of N elements, each group of four summed by itself first: where one element is most of S, what it is
// added to loses the small ones' last digits all in one direction, and a row of 131072 has hundreds of them a thread
// (measured on rows with one such element: ln S 1.3e-6 too small on average with one running sum).
template <int N>
__device__ __forceinline__ void add_up(const float* x, float ref, float c, float& s, float& w) {
  float ss = 0.f, ww = 0.f;
#pragma unroll
  for (int g = 0; g < N; g += 4) {
    float e[4], a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float d = g + i < N ? (x[g + i < N ? g + i : 0] - ref) * c : -INFINITY;
      e[i] = __builtin_amdgcn_exp2f(d);
      a[i] = fmaxf(d, D_MIN);
    }
    const float s4 = (e[0] + e[1]) + (e[2] + e[3]);
    const float w4 = fmaf(a[1], e[1], a[0] * e[0]) + fmaf(a[3], e[3], a[2] * e[2]);
    ss = g == 0 ? s4 : ss + s4;
    ww = g == 0 ? w4 : ww + w4;
  }
  s += ss;
  w += ww;
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
  add_up<N>(x, finite_ref(p.m), c, p.s, p.w);
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


// ---- gradient entries: (alpha + gamma d_j) e_j, at the label + patch.  BOTH: gamma is not 0.  One form for every kernel that
// writes them, with its roundings spelled out: a gradient computed again is the same to the bit. --------------------------------
template <bool BOTH>
__device__ __forceinline__ float gradient_entry(float f, const f32x4& k, float c) {
  const float d = (f - k[0]) * c, e = __builtin_amdgcn_exp2f(d);
  return (BOTH ? fmaf(fmaxf(d, D_MIN), k[2], k[1]) : k[1]) * e;
}
template <typename T, bool BOTH>
__device__ __forceinline__ T gradient_one(float f, const f32x4& k, float c, bool label) {
#pragma clang fp contract(off)
  const float g = gradient_entry<BOTH>(f, k, c);
  return (T)(label ? g + k[3] : g);
}
template <typename T, bool BOTH>
__device__ __forceinline__ u32x4 gradient_vector(const u32x4& w, const f32x4& k, float c, int label) {
#pragma clang fp contract(off)
  constexpr int VEC = Type<T>::VEC;
  float f[VEC];
  Type<T>::unpack(w, f);
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = gradient_entry<BOTH>(f[j], k, c);
  if (label >= 0 && label < VEC)
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = j == label ? f[j] + k[3] : f[j];
  return Type<T>::pack(f);
}

// ---- a row held by its threads -------------------------------------------------------------------------------------------
// TPR threads hold up to TPR * NCH 16-byte vectors of a row in registers, so that its statistics and its gradient need one
// read of memory; vectors beyond that (rows of more than 256 KB) are read again.  Vectors are aligned on the input; the up
// to 2 (VEC - 1) elements before and behind them are one more register of the first threads.
template <typename T> __device__ __forceinline__ u32x4 no_elements();       // -inf: adds nothing, changes no maximum
template <> __device__ __forceinline__ u32x4 no_elements<float>() { return u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}; }
template <> __device__ __forceinline__ u32x4 no_elements<__bf16>() { return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}; }
template <> __device__ __forceinline__ u32x4 no_elements<_Float16>() { return u32x4{0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u}; }

template <typename T, int TPR, int NCH>
struct Row {
  static constexpr int VEC = Type<T>::VEC;
  u32x4 v[NCH];
  float extra;               // the element `extra_at` (-1: none)
  int extra_at, t, n, head, nv;
  const T* x;

  __device__ __forceinline__ const u32x4* body() const { return reinterpret_cast<const u32x4*>(x + head); }

  __device__ __forceinline__ void load(const T* row, int vocab, int thread) {
    x = row;
    n = vocab;
    t = thread;
    head = std::min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
    nv = (n - head) / VEC;
    const u32x4* b = body();
#pragma unroll
    for (int i = 0; i < NCH; ++i) v[i] = t + i * TPR < nv ? __builtin_nontemporal_load(b + t + i * TPR) : no_elements<T>();
    const int behind = head + nv * VEC;
    extra_at = t < head ? t : (t < head + n - behind ? behind + t - head : -1);
    extra = extra_at >= 0 ? (float)x[extra_at] : -INFINITY;
  }

  // Between two passes over the registers: what a pass made of them (twice as many floats of a 16-bit type) is made again
  // by the next one, not kept.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < NCH; ++i) asm volatile("" : "+v"(v[i]));
  }

  __device__ __forceinline__ Part stats(float c) {
    float m = extra;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float f[VEC];
      Type<T>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) m = fmaxf(m, f[j]);
    }
    forget();
    const float ref = finite_ref(m);
    Part p{m, 0.f, 0.f};
    add_up<1>(&extra, ref, c, p.s, p.w);
#pragma unroll
    for (int i = 0; i < NCH; i += 4) {
      float s = 0.f, w = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[VEC];
        Type<T>::unpack(v[i + k], f);
        add_up<VEC>(f, ref, c, s, w);
      }
      p.s += s;
      p.w += w;
    }
    return p;
  }

  template <bool BOTH>
  __device__ __forceinline__ void store_as(T* out, const f32x4& k, float c, int at) const {
    u32x4_u* o = reinterpret_cast<u32x4_u*>(out + head);
#pragma unroll
    for (int q = 0; q < NCH; ++q) {
      const int i = t + q * TPR;
      if (i < nv) o[i] = gradient_vector<T, BOTH>(v[q], k, c, at - head - i * VEC);
    }
    for (int i = t + NCH * TPR; i < nv; i += TPR) o[i] = gradient_vector<T, BOTH>(body()[i], k, c, at - head - i * VEC);
    if (extra_at >= 0) out[extra_at] = gradient_one<T, BOTH>(extra, k, c, extra_at == at);
  }
  __device__ __forceinline__ void store(T* out, const f32x4& k, float c, int at) {
    forget();
    if (k[2] == 0.f) store_as<false>(out, k, c, at);
    else store_as<true>(out, k, c, at);
  }
};

// a gradient row without a gradient
template <typename T, int TPR>
__device__ __forceinline__ void store_zeros(T* out, int n, int t) {
  constexpr int VEC = Type<T>::VEC;
  const int head = std::min(n, (int)((16 - (reinterpret_cast<uintptr_t>(out) & 15)) & 15) / (int)sizeof(T));
  const int nv = (n - head) / VEC, behind = head + nv * VEC;
  u32x4* o = reinterpret_cast<u32x4*>(out + head);
  for (int i = t; i < nv; i += TPR) o[i] = u32x4{0u, 0u, 0u, 0u};
  if (t < head) out[t] = (T)0.f;
  if (t < n - behind) out[behind + t] = (T)0.f;
}

__device__ __forceinline__ float first_lane(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// The parts of a row's waves; the result is in the first wave (TPR > 64: through LDS, one barrier).
template <int TPR>
__device__ __forceinline__ Part row_join(Part p, float c, Part* red) {
  p = wave_join(p, c);
  if (TPR > 64) {
    constexpr int WAVES = TPR / 64;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = p;
    __syncthreads();
    if (threadIdx.x < 64) {
      p = threadIdx.x < WAVES ? red[threadIdx.x] : Part{-INFINITY, 0.f, 0.f};
#pragma unroll
      for (int off = WAVES / 2; off > 0; off >>= 1)
        p = join(p, Part{__shfl_xor(p.m, off, 64), __shfl_xor(p.s, off, 64), __shfl_xor(p.w, off, 64)}, c);
    }
  }
  // the lanes' sums differ in the last bit (each rounds its own part first): the first lane's is the row's
  return Part{first_lane(p.m), first_lane(p.s), first_lane(p.w)};
}

// ---- counts and sums over rows --------------------------------------------------------------------------------------------------
// Up to 64 blocks count what the mean divides by; every row's wave adds up their counts itself (whole numbers: any order).
constexpr int COUNT_BLOCKS = 64;

struct Sums {
  double* counted;           // [COUNT_BLOCKS]
  int blocks;                // of them used
  f32x4* terms;              // [rows]: a row's weighted terms
  double* partial;           // [4][COUNT_BLOCKS]
  unsigned* counter;
  unsigned rows;
  float* loss;               // scale * (terms[0] + kl terms[1] - ent terms[2])
  float* stats;              // the four sums, or null
  double scale, kl, ent;
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// 1 / what counts, in every lane of a wave; 0 where nothing does
__device__ __forceinline__ double one_over_counted(const Sums& q) {
  const int lane = threadIdx.x & 63;
  const double n = wave_sum64(lane < q.blocks ? q.counted[lane] : 0.0);
  return n > 0 ? 1.0 / n : 0.0;
}

// Adds the rows' terms in a fixed order; the last block adds the blocks' sums.
static __global__ __launch_bounds__(1024) void sum_terms_kernel(Sums q) {
  __shared__ double red[16];
  double sum[4] = {0, 0, 0, 0};
  for (unsigned r = blockIdx.x * 1024 + threadIdx.x; r < q.rows; r += gridDim.x * 1024) {
    const f32x4 v = q.terms[r];
    for (int k = 0; k < 4; ++k) sum[k] += (double)v[k];
  }
  for (int k = 0; k < 4; ++k) {
    sum[k] = block_sum64(sum[k], red);
    if (threadIdx.x == 0) q.partial[k * COUNT_BLOCKS + blockIdx.x] = sum[k];
  }
  if (gridDim.x > 1) {
    if (!last_block(q.counter)) return;
    for (int k = 0; k < 4; ++k) {
      const double v = threadIdx.x < gridDim.x
                           ? __hip_atomic_load(q.partial + k * COUNT_BLOCKS + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
      sum[k] = block_sum64(v, red);
    }
  }
  if (threadIdx.x == 0) {
    q.loss[0] = (float)(q.scale * (sum[0] + (q.kl != 0 ? q.kl * sum[1] : 0.0) - (q.ent != 0 ? q.ent * sum[2] : 0.0)));
    if (q.stats)
      for (int k = 0; k < 4; ++k) q.stats[k] = (float)sum[k];
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
inline size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

inline bool bad_logits(const char* who, const Logits& p, int dtype, long long rows, long long inner, long long so, long long si, int* rc) {
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

inline Logits make_logits(const void* x, long long rows, long long inner, long long so, long long si, int vocab, const void* labels,
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

inline int size_of(int dtype) { return dtype == ST_F32 ? 4 : 2; }

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


inline Sums make_sums(Space& w, long long rows, float* loss, float* stats, double scale, double kl, double ent) {
  Sums q{};
  q.counted = w.take<double>(COUNT_BLOCKS);
  q.partial = w.take<double>(4 * COUNT_BLOCKS);
  q.counter = w.take<unsigned>(1);
  q.terms = w.take<f32x4>((size_t)rows);
  q.rows = (unsigned)rows;
  q.loss = loss;
  q.stats = stats;
  q.scale = scale;
  q.kl = kl;
  q.ent = ent;
  return q;
}

inline size_t sums_bytes(long long rows) { return align256(COUNT_BLOCKS * 8) * 5 + 256 + align256((size_t)rows * sizeof(f32x4)); }

inline void launch_sum_terms(const Sums& q, hipStream_t s) {
  hipLaunchKernelGGL(sum_terms_kernel, dim3(std::min<unsigned>(COUNT_BLOCKS, (unsigned)st::cdivll(q.rows, 4096))), dim3(1024), 0, s, q);
}

// Which of the row kernels takes a row of `bytes`: the smallest (threads, vectors a thread) that holds it, so that as many
// rows as possible share a compute unit; the largest holds 256 KB (64 registers of 1024 threads) and reads again what is
// beyond.  `kernel` is called with the two as integral constants.
template <int A, int B> struct Shape {
  static constexpr int TPR = A, NCH = B, BLOCK = A < NT ? NT : A, ROWS = BLOCK / A;
};
template <typename F>
auto with_shape(long long bytes, F kernel) {
  if (bytes <= 4 << 10) return kernel(Shape<64, 4>{});
  if (bytes <= 16 << 10) return kernel(Shape<256, 4>{});
  if (bytes <= 32 << 10) return kernel(Shape<256, 8>{});
  if (bytes <= 64 << 10) return kernel(Shape<512, 8>{});
  if (bytes <= 128 << 10) return kernel(Shape<1024, 8>{});
  return kernel(Shape<1024, 16>{});
}
template <typename F>
auto with_type(int dtype, F f) {
  if (dtype == ST_F32) return f(float{});
  if (dtype == ST_BF16) return f(__bf16{});
  return f(_Float16{});
}

}  // namespace st_token
