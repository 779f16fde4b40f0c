// Shared device code of the losses over rows of logits (token_losses.hip, token_distill.hip) for gfx950.
//
// One row of logits x[0..V) at temperature tau, in the base-2 domain of the hardware's exponential, seen from a reference m:
//
//   c = log2(e) / tau     d_j = x_j c - m c     e_j = 2^d_j     S = sum e_j     W = sum e_j d_j
//   log q_j = ln2 d_j - ln S                    entropy H = ln S - ln2 W / S
//
// Every loss here reaches x through the label's log-probability and the entropy, or through a short list of entries, so
// every gradient row is   g_j = (alpha + gamma d_j) e_j   plus a few patched entries.
//
// m is a value near the maximum, not the maximum itself: a wave takes the largest of its first vector and another one where an
// element lies more than a bit above it.  That saves a pass over the row, and lets the exponentials begin while the row is
// still arriving; and since no d_j is above 1.5, the elements that S mostly consists of have hardly any rounding in their
// exponents.  (With the first reference kept as long as S stays below 2^80 a dominant element's d_j reaches 80, whose rounding is
// 2.6e-6 of S.)  m c is rounded to a whole number, which then stands for the reference everywhere: d_j is one fused multiply-add
// with no error but its own, and a part seen from another reference is multiplied by a power of two, exactly.  (The hardware's
// exponential is 3.4e-9 too small on average, and an element would go through four of them on its way into S.)
//
// Where |m c| reaches 2^24 ("low" rows: nothing but a mask's value, -1e9 or the lowest of the type) the next whole number can be
// far from it, and the difference comes first, d_j = (x_j - m) c: such a row is the uniform distribution that the formula gives,
// whatever the value.  A row of -inf only has S = 0: no distribution, log-probability -inf, entropy 0, gradient 0.
//
// Sums of a row are fp32 per thread and over a fixed tree; what a row is reduced to is finished in fp64 (one wave a row),
// because a sequence's sum of hundreds of log-probabilities is compared with another model's: c's own rounding (relative 2^-24
// at most) shifts every term the same way, and W, which is d S / d ln c up to a factor, takes that shift out again.
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
typedef double f64x4 __attribute__((ext_vector_type(4)));
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
  float eps_ln2;                         // c = (1 + eps) log2(e) / tau: eps ln2
  double tau, inv_tau, inv_ct;           // 1 / tau, 1 / (c tau)
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

constexpr float LOW = 0x1p24f;

// A reference and its product with c as a whole number.
struct Ref {
  float m, mc;
  bool low;
};
__device__ __forceinline__ Ref make_ref(float m, float c) {
  const float f = m == -INFINITY ? 0.f : m;
  const float mc = rintf(f * c);
  return {f, mc, !(fabsf(mc) < LOW)};
}
template <bool IS_LOW>
__device__ __forceinline__ float distance(float x, const Ref& r, float c) {
  return IS_LOW ? (x - r.m) * c : fmaf(x, c, -r.mc);
}
__device__ __forceinline__ float distance(float x, const Ref& r, float c) { return r.low ? distance<true>(x, r, c) : distance<false>(x, r, c); }

// From an old reference to a new one; -inf where the old part is empty.  One of them may be low and the other not: the whole
// number is the reference then, not the m that it came from, which is up to half a bit away.
__device__ __forceinline__ float step(float m_old, const Ref& to, float c) {
  if (m_old == -INFINITY) return -INFINITY;
  const Ref from = make_ref(m_old, c);
  if (from.low) return distance(m_old, to, c);
  return to.low ? -fmaf(to.m, c, -from.mc) : from.mc - to.mc;
}

// A part seen from another reference: d' = d + t.
__device__ __forceinline__ void rebase(float& s, float& w, float m_old, const Ref& to, float c) {
  const float t = step(m_old, to, c);
  const float f = __builtin_amdgcn_exp2f(t);
  w = f * fmaf(fmaxf(t, D_MIN), s, w);
  s *= f;
}

// Reductions over a wave by lane moves of the vector unit; the result is in every lane.  LANES = 16: over the first row of
// sixteen lanes alone.
template <int CTRL, int ROWS>
__device__ __forceinline__ float lane_move(float v, float none) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(none), __float_as_uint(v), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double lane_move(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int SHR1 = 0x111, SHR2 = 0x112, SHR4 = 0x114, SHR8 = 0x118, BCAST15 = 0x142, BCAST31 = 0x143;

__device__ __forceinline__ float from_lane(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

template <int LANES = 64>
__device__ __forceinline__ float lanes_max(float v) {
  v = fmaxf(v, lane_move<SHR1, 0xf>(v, -INFINITY));
  v = fmaxf(v, lane_move<SHR2, 0xf>(v, -INFINITY));
  v = fmaxf(v, lane_move<SHR4, 0xf>(v, -INFINITY));
  v = fmaxf(v, lane_move<SHR8, 0xf>(v, -INFINITY));
  if (LANES == 16) return from_lane(v, 15);
  v = fmaxf(v, lane_move<BCAST15, 0xa>(v, -INFINITY));
  v = fmaxf(v, lane_move<BCAST31, 0xc>(v, -INFINITY));
  return from_lane(v, 63);
}
template <int LANES = 64>
__device__ __forceinline__ float lanes_sum(float v) {
  v += lane_move<SHR1, 0xf>(v, 0.f);
  v += lane_move<SHR2, 0xf>(v, 0.f);
  v += lane_move<SHR4, 0xf>(v, 0.f);
  v += lane_move<SHR8, 0xf>(v, 0.f);
  if (LANES == 16) return from_lane(v, 15);
  v += lane_move<BCAST15, 0xa>(v, 0.f);
  v += lane_move<BCAST31, 0xc>(v, 0.f);
  return from_lane(v, 63);
}
__device__ __forceinline__ double lanes_sum(double v) {
  v += lane_move<SHR1, 0xf>(v);
  v += lane_move<SHR2, 0xf>(v);
  v += lane_move<SHR4, 0xf>(v);
  v += lane_move<SHR8, 0xf>(v);
  v += lane_move<BCAST15, 0xa>(v);
  v += lane_move<BCAST31, 0xc>(v);
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(u >> 32), 63) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((uint32_t)u, 63));
}

// the parts of a wave's lanes (of its first 16), seen from their maximum
template <int LANES = 64>
__device__ __forceinline__ Part wave_join(Part p, float c) {
  const float m = lanes_max<LANES>(p.m);
  rebase(p.s, p.w, p.m, make_ref(m, c), c);
  return {m, lanes_sum<LANES>(p.s), lanes_sum<LANES>(p.w)};
}

// The parts of a row's waves; every lane of the row's first wave gets the result (TPR > 64: through LDS, one barrier).
template <int TPR>
__device__ __forceinline__ Part row_join(Part p, float c, Part* red) {
  p = wave_join(p, c);
  if (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = p;
    __syncthreads();
    if (threadIdx.x < 64) p = wave_join<16>(threadIdx.x < TPR / 64 ? red[threadIdx.x] : Part{-INFINITY, 0.f, 0.f}, c);
  }
  return p;
}

// e_j and e_j d_j of N elements, each group of four summed by itself first: where one element is most of S, what it is
// added to loses the small ones' last digits all in one direction, and a row of 131072 has hundreds of them a thread
// (measured on rows with one such element: ln S 1.3e-6 too small on average with one running sum).
template <int N, bool IS_LOW>
__device__ __forceinline__ void add_up(const float* x, const Ref& ref, float c, float& s, float& w) {
  float ss = 0.f, ww = 0.f;
#pragma unroll
  for (int g = 0; g < N; g += 4) {
    float e[4], a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float d = g + i < N ? distance<IS_LOW>(x[g + i < N ? g + i : 0], ref, c) : -INFINITY;
      e[i] = __builtin_amdgcn_exp2f(d);
      a[i] = fmaxf(d, D_MIN);
    }
    const float s4 = (e[0] + e[1]) + (e[2] + e[3]);
    ss = g == 0 ? s4 : ss + s4;
    const float w4 = fmaf(a[1], e[1], a[0] * e[0]) + fmaf(a[3], e[3], a[2] * e[2]);
    ww = g == 0 ? w4 : ww + w4;
  }
  s += ss;
  w += ww;
}

// N more elements into a thread's part, whose reference is the largest that it has seen
template <int N>
__device__ __forceinline__ void take(Part& p, const float* x, float c) {
  float m = p.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
  const Ref ref = make_ref(m, c);
  if (m > p.m) {
    rebase(p.s, p.w, p.m, ref, c);
    p.m = m;
  }
  if (ref.low) add_up<N, true>(x, ref, c, p.s, p.w);
  else add_up<N, false>(x, ref, c, p.s, p.w);
}

// ---- what the logits of a row say once its parts are joined ----------------------------------------------------------------
struct RowStat {
  double z;          // the reference as a logit over tau
  double ln_s;       // ln S, with the rounding of c taken out
  float h;           // entropy
  float inv_ts;      // 1 / (tau S); 0 for a row without a distribution
  float ref;
};

// ln of a positive number with the logarithm's own error, not that of a result of up to 88 in fp32
__device__ __forceinline__ double ln_wide(float v) {
  const float f = __builtin_amdgcn_frexp_mantf(v);              // [1/2, 1)
  const int up = f < 0.70710678f;                               // to [0.7, 1.42): a small logarithm has a small error
  return (double)(__builtin_amdgcn_frexp_expf(v) - up) * LN2 + (double)(__builtin_amdgcn_logf(up ? 2 * f : f) * (float)LN2);
}

// exp(v), relative error below 2^-46: the 16th root's series (the term left out is below 2^-47 of the result), squared four times with
// 1 left out.  (The library's exp is exact to the last bit and takes 24 registers more of kernels that hold a row in theirs.)
__device__ __forceinline__ double exp64(double v) {
  if (v != v) return v;
  v = fmax(fmin(v, 1400.0), -1400.0);                             // inf and 0 from here on
  const double k = rint(v * (1.0 / LN2)), r = fma(-k, LN2, v) * 0.0625;
  double p = fma(fma(fma(fma(r, 1.0 / 720, 1.0 / 120), r, 1.0 / 24), r, 1.0 / 6), r, 0.5);
  p = fma(p * r, r, r);
#pragma unroll
  for (int i = 0; i < 4; ++i) p = p * (2.0 + p);
  return ldexp(1.0 + p, (int)k);
}

// ln v, absolute error below 2^-46: what exp64 leaves of the logarithm above, to second order (of 1e-7)
__device__ __forceinline__ double ln64(double v) {
  const double y = ln_wide((float)v), left = fma(v, exp64(-y), -1.0);
  return fma(-0.5 * left, left, left) + y;
}

__device__ __forceinline__ float reciprocal(float v) {
  const float r = __builtin_amdgcn_rcpf(v);
  return fmaf(fmaf(-v, r, 1.f), r, r);
}

// what a reference is in x / tau
__device__ __forceinline__ double logit_of(const Ref& r, const Logits& p) { return r.low ? (double)r.m * p.inv_tau : (double)r.mc * p.inv_ct; }

__device__ __forceinline__ RowStat finish(const Part& q, const Logits& p) {
  RowStat r;
  const Ref ref = make_ref(q.m, p.c);
  const float inv = reciprocal(q.s);
  r.ref = ref.m;
  r.z = logit_of(ref, p);
  r.ln_s = ln64((double)q.s - (double)p.eps_ln2 * (double)q.w);
  r.h = (float)(r.ln_s - p.inv_ct * (double)q.w * (double)inv);
  r.inv_ts = (float)(p.inv_tau * (double)inv);
  if (q.s == 0.f) {
    r.ln_s = -INFINITY;
    r.h = 0.f;
    r.inv_ts = 0.f;
  }
  return r;
}

// natural logarithm of q at a logit (not fused: what the reference itself is over tau leaves nothing)
__device__ __forceinline__ double log_prob(float x, const RowStat& r, const Logits& p) {
#pragma clang fp contract(off)
  return r.inv_ts == 0.f ? -INFINITY : (double)x * p.inv_tau - r.z - r.ln_s;
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
  v = lanes_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) t += red[w];
  return t;
}

// ---- gradient entries: (alpha + gamma d_j) e_j, at the label + patch --------------------------------------------------------
// BOTH: gamma is not 0 (the form with gamma = 0 has the same value).  One form for every kernel that writes them: a gradient
// computed again is the same to the bit.
template <bool BOTH, bool IS_LOW>
__device__ __forceinline__ float gradient_entry(float f, const f32x4& k, const Ref& ref, float c) {
  const float d = distance<IS_LOW>(f, ref, c), e = __builtin_amdgcn_exp2f(d);
  return (BOTH ? fmaf(fmaxf(d, D_MIN), k[2], k[1]) : k[1]) * e;
}
template <typename T, bool BOTH, bool IS_LOW>
__device__ __forceinline__ u32x4 gradient_vector(const u32x4& w, const f32x4& k, const Ref& ref, float c) {
  constexpr int VEC = Type<T>::VEC;
  float f[VEC];
  Type<T>::unpack(w, f);
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = gradient_entry<BOTH, IS_LOW>(f[j], k, ref, c);
  return Type<T>::pack(f);
}

template <bool PAST>
__device__ __forceinline__ void put(u32x4_u* at, const u32x4& w) {
  if (PAST) __builtin_nontemporal_store((u32x4_u)w, at);
  else *at = w;
}

// What a row, or a part of one, is for the threads that share it: 16-byte vectors aligned on the input, in turn, and the up
// to 2 (VEC - 1) elements before and behind them, one for each of the first threads.
template <typename T, int TPR>
struct Span {
  static constexpr int VEC = Type<T>::VEC;
  // Loads in flight where a row is read again: 16 elements a thread where rows are larger than their threads' registers (32 spill:
  // 2048 rows of 160000 bf16 take 297 us instead of 263; fp32 with 8: 1024 of 131072, 242 us instead of 238), one load where that
  // happens to rare rows only (more would cost every row the registers).
  static constexpr int AGAIN = TPR == 1024 ? 16 / VEC : 1;
  const T* x;
  int n, t, head, nv;
  __device__ __forceinline__ Span() {}
  __device__ __forceinline__ Span(const T* row, int elements, int thread) : x(row), n(elements), t(thread) {
    head = std::min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
    nv = (n - head) / VEC;
  }
  __device__ __forceinline__ const u32x4* body() const { return reinterpret_cast<const u32x4*>(x + head); }
  __device__ __forceinline__ int extra_at() const {             // this thread's element outside the vectors, or -1
    const int j = t < head ? t : t + nv * VEC;
    return j < n && t < head + n - (head + nv * VEC) ? j : -1;
  }
  __device__ __forceinline__ int owner(int at) const {          // the thread that has element `at`
    const int in = at - head;
    return in < 0 ? at : in < nv * VEC ? in / VEC % TPR : at - nv * VEC;
  }

  // Gradient of the vectors from `first` on and of the element outside them.  PAST: stores go past the caches, which keep the
  // logits that are still to be read (4096 rows of 32768 bf16, both passes: 154 -> 129 us; where the row is in registers there
  // is nothing to keep, and such stores are 10 % slower).
  template <bool BOTH, bool IS_LOW, bool PAST = false>
  __device__ __forceinline__ void stream(T* out, const f32x4& k, const Ref& ref, float c, int first) const {
    u32x4_u* o = reinterpret_cast<u32x4_u*>(out + head);
    for (int i = t + first; i < nv; i += AGAIN * TPR) {
      u32x4 b[AGAIN];
#pragma unroll
      for (int q = 0; q < AGAIN; ++q) b[q] = body()[std::min(i + q * TPR, nv - 1)];
#pragma unroll
      for (int q = 0; q < AGAIN; ++q)
        if (i + q * TPR < nv) put<PAST>(o + i + q * TPR, gradient_vector<T, BOTH, IS_LOW>(b[q], k, ref, c));
    }
    const int j = extra_at();
    if (j >= 0) out[j] = (T)gradient_entry<BOTH, IS_LOW>((float)x[j], k, ref, c);
  }
  __device__ __forceinline__ void stream_all(T* out, const f32x4& k, const Ref& ref, float c) const {
    if (ref.low) stream<true, true, true>(out, k, ref, c, 0);
    else if (k[2] != 0.f) stream<true, false, true>(out, k, ref, c, 0);
    else stream<false, false, true>(out, k, ref, c, 0);
  }
  // the label's entry, by the thread that wrote it as any other before: its two stores keep their order
  __device__ __forceinline__ void label(T* out, const f32x4& k, const Ref& ref, float c, int at) const {
#pragma clang fp contract(off)
    if (at < 0 || at >= n || t != owner(at)) return;
    const float f = (float)x[at];
    out[at] = (T)((ref.low ? gradient_entry<true, true>(f, k, ref, c) : gradient_entry<true, false>(f, k, ref, c)) + k[3]);
  }
};

// ---- a row held by its threads -------------------------------------------------------------------------------------------
// TPR threads hold up to TPR * NCH vectors of a row in registers, so that its statistics and its gradient need one read of
// memory; vectors beyond that (rows of more than 320 KB) are read again.  A wave passes over the vectors that none of its
// lanes has.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

struct Whole {                // nothing of a row is left out
  __device__ __forceinline__ void vector(int, int, float*) const {}
  __device__ __forceinline__ float extra(int, float v) const { return v; }
};

template <typename T, int TPR, int NCH>
struct Row : Span<T, TPR> {
  using Base = Span<T, TPR>;
  using Base::AGAIN;
  using Base::VEC;
  using Base::body;
  using Base::n;
  using Base::nv;
  using Base::t;
  using Base::x;
  u32x4 v[NCH];
  T outside;                  // the element outside the vectors
  int slots, full;            // vectors of v that any lane of the wave has; that all its lanes have

  __device__ __forceinline__ void place(const T* row, int elements, int thread) { static_cast<Base&>(*this) = Base(row, elements, thread); }

  // Buffer loads: one after the other without a branch between them, so that the first vector can be waited for alone; what
  // lies behind the row is not asked for and comes back as 0.
  __device__ __forceinline__ void load() {
    outside = x[std::max(0, this->extra_at())];                // first, since loads return in order
    const int first = scalar(t), last = nv - 1 - first;
    slots = last < 0 ? 0 : last / TPR + 1;
    full = last < 63 ? 0 : (last - 63) / TPR + 1;
    const uint64_t at = reinterpret_cast<uint64_t>(body());
    const uint64_t base = (uint64_t)(uint32_t)scalar((int)(at >> 32)) << 32 | (uint32_t)scalar((int)at);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base), 0, scalar(std::min(nv, NCH * TPR)) * 16, 0x00020000);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, t * 16 + i * TPR * 16, 0, 2));
      __builtin_amdgcn_sched_barrier(0);                        // in this order
    }
  }
  __device__ __forceinline__ float extra() const { return this->extra_at() >= 0 ? (float)outside : -INFINITY; }
  // the elements of vector i; -inf where the lane has none
  __device__ __forceinline__ void elements(int i, float* f) const {
    Type<T>::unpack(v[i], f);
    if (i >= full)
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = t + i * TPR < nv ? f[j] : -INFINITY;
  }

  // Between two passes over the registers: what a pass made of them (twice as many floats of a 16-bit type) is made again
  // by the next one, not kept.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < NCH; ++i) asm volatile("" : "+v"(v[i]));
  }

  // The thread's part of the row's statistics.  `leave_out` puts -inf in place of what does not belong: among the elements f of
  // the thread's `slot`-th vector, and of the element outside the vectors.
  template <typename F>
  __device__ __forceinline__ Part stats(float c, const F& leave_out) {
    const float beside = leave_out.extra(t, extra());
    Part p{-INFINITY, 0.f, 0.f};                                // an empty part, which no other one is seen from
    Ref ref = make_ref(-INFINITY, c);
    float limit = -INFINITY;
    const float bit = __builtin_amdgcn_rcpf(c);
    // One reference for the wave, in a scalar register, and another where any lane has an element more than a bit above it; what
    // was added up before is multiplied by a power of two.
    const auto raise = [&](float g, float& s, float& w) {
      if (!__any(g > limit)) return;
      const float m = lanes_max(g);
      ref = make_ref(m, c);
      rebase(p.s, p.w, p.m, ref, c);
      rebase(s, w, p.m, ref, c);
      p.m = m;
      limit = m + bit;
    };
    float none = 0.f, none_w = 0.f;
    raise(beside, none, none_w);
    if (!ref.low) add_up<1, false>(&beside, ref, c, p.s, p.w);
#pragma unroll
    for (int i = 0; i < NCH; i += 4) {
      float s = 0.f, w = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < slots && !ref.low) {
          float f[VEC];
          elements(i + k, f);
          leave_out.vector(i + k, t, f);
          float g = f[0];
#pragma unroll
          for (int j = 1; j < VEC; ++j) g = fmaxf(g, f[j]);
          raise(g, s, w);
          if (!ref.low) add_up<VEC, false>(f, ref, c, s, w);
        }
      p.s += s;
      p.w += w;
    }
    int from = NCH;
    if (ref.low) {                                              // element by element, from the beginning
      p = Part{-INFINITY, 0.f, 0.f};
      take<1>(p, &beside, c);
      from = 0;
    }
    for (int slot = from; t + slot * TPR < nv; slot += AGAIN) {
      u32x4 b[AGAIN];
      float f[AGAIN * VEC];
#pragma unroll
      for (int k = 0; k < AGAIN; ++k) b[k] = body()[std::min(t + (slot + k) * TPR, nv - 1)];
#pragma unroll
      for (int k = 0; k < AGAIN; ++k) {
        Type<T>::unpack(b[k], f + k * VEC);
        if (t + (slot + k) * TPR < nv) {
          leave_out.vector(slot + k, t, f + k * VEC);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[k * VEC + j] = -INFINITY;
        }
      }
      take<AGAIN * VEC>(p, f, c);
    }
    return p;
  }

  template <bool BOTH>
  __device__ __forceinline__ void store_as(T* out, const f32x4& k, const Ref& ref, float c) const {
    u32x4_u* o = reinterpret_cast<u32x4_u*>(out + this->head);
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      if (i < slots) {
        const u32x4 w = gradient_vector<T, BOTH, false>(v[i], k, ref, c);
        if (t + i * TPR < nv) o[t + i * TPR] = w;
      }
    this->template stream<BOTH, false>(out, k, ref, c, NCH * TPR);
  }
  __device__ __forceinline__ void store(T* out, const f32x4& k, float c, int at) {
    forget();
    const Ref ref = make_ref(k[0], c);
    if (ref.low) this->template stream<true, true>(out, k, ref, c, 0);
    else if (k[2] != 0.f) store_as<true>(out, k, ref, c);
    else store_as<false>(out, k, ref, c);
    this->label(out, k, ref, c, at);
  }
};

// a gradient row without a gradient
template <typename T, int TPR, bool PAST = false>
__device__ __forceinline__ void store_zeros(T* out, int n, int t) {
  constexpr int VEC = Type<T>::VEC;
  const int head = std::min(n, (int)((16 - (reinterpret_cast<uintptr_t>(out) & 15)) & 15) / (int)sizeof(T));
  const int nv = (n - head) / VEC, behind = head + nv * VEC;
  u32x4* o = reinterpret_cast<u32x4*>(out + head);
  for (int i = t; i < nv; i += TPR) put<PAST>(o + i, u32x4{0u, 0u, 0u, 0u});
  if (t < head) out[t] = (T)0.f;
  if (t < n - behind) out[behind + t] = (T)0.f;
}

// ---- counts and sums over rows --------------------------------------------------------------------------------------------------
// Up to 64 blocks count what the mean divides by; every row's wave adds up their counts itself (whole numbers: any order).
constexpr int COUNT_BLOCKS = 64;

struct Sums {
  double* counted;           // [COUNT_BLOCKS]
  int blocks;                // of them used
  f64x4* terms;              // [rows]: a row's weighted terms; of both signs, their sum may be far smaller than they are
  double* partial;           // [4][COUNT_BLOCKS]
  unsigned rows;
  float* loss;               // scale * (terms[0] + kl terms[1] - ent terms[2])
  float* stats;              // the four sums, or null
  double scale, kl, ent;
};

// A lane's share of what counts (asked for early), and 1 / their sum in every lane of a wave; 0 where nothing counts.
__device__ __forceinline__ double counted_share(const Sums& q) {
  const int lane = threadIdx.x & 63;
  return lane < q.blocks ? q.counted[lane] : 0.0;
}
__device__ __forceinline__ double one_over(double share) {
  const double n = lanes_sum(share);
  return n > 0 ? 1.0 / n : 0.0;
}

__device__ __forceinline__ void write_sums(const Sums& q, const double* sum) {
  q.loss[0] = (float)(q.scale * (sum[0] + (q.kl != 0 ? q.kl * sum[1] : 0.0) - (q.ent != 0 ? q.ent * sum[2] : 0.0)));
  if (q.stats)
    for (int k = 0; k < 4; ++k) q.stats[k] = (float)sum[k];
}

// Adds the rows' terms in a fixed order: one block all of them, or COUNT_BLOCKS blocks a share each and a block more behind
// them.  (A last block that waits for the others' fences costs 13 us here: the gradient's lines are still in the caches.)
static __global__ __launch_bounds__(1024) void sum_terms_kernel(Sums q) {
  __shared__ double red[16];
  double sum[4] = {0, 0, 0, 0};
  for (unsigned r = blockIdx.x * 1024 + threadIdx.x; r < q.rows; r += gridDim.x * 1024) {
    const f64x4 v = q.terms[r];
    for (int k = 0; k < 4; ++k) sum[k] += v[k];
  }
  for (int k = 0; k < 4; ++k) sum[k] = block_sum64(sum[k], red);
  if (threadIdx.x != 0) return;
  if (gridDim.x == 1) write_sums(q, sum);
  else
    for (int k = 0; k < 4; ++k) q.partial[k * COUNT_BLOCKS + blockIdx.x] = sum[k];
}

static __global__ __launch_bounds__(64) void sum_partial_kernel(Sums q) {
  double sum[4];
  for (int k = 0; k < 4; ++k) sum[k] = lanes_sum(q.partial[k * COUNT_BLOCKS + threadIdx.x]);
  if (threadIdx.x == 0) write_sums(q, sum);
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
  p.inv_tau = 1.0 / tau;
  p.c = (float)(1.0 / (LN2 * tau));
  p.inv_ct = 1.0 / ((double)p.c * tau);
  p.eps_ln2 = (float)(((double)p.c * LN2 * tau - 1.0) * LN2);
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

// HIP counts the threads of a launch in 32 bits.
inline bool fits_a_launch(long long blocks, int threads) { return blocks * threads <= 0xffffffffLL; }

inline Sums make_sums(Space& w, long long rows, float* loss, float* stats, double scale, double kl, double ent) {
  Sums q{};
  q.counted = w.take<double>(COUNT_BLOCKS);
  q.partial = w.take<double>(4 * COUNT_BLOCKS);
  q.terms = w.take<f64x4>((size_t)rows);
  q.rows = (unsigned)rows;
  q.loss = loss;
  q.stats = stats;
  q.scale = scale;
  q.kl = kl;
  q.ent = ent;
  return q;
}

inline size_t sums_bytes(long long rows) { return align256(COUNT_BLOCKS * 8) * 5 + align256((size_t)rows * sizeof(f64x4)); }

inline void launch_sum_terms(const Sums& q, hipStream_t s) {
  const bool one = q.rows <= 16384;                             // 16 rows a thread
  hipLaunchKernelGGL(sum_terms_kernel, dim3(one ? 1 : COUNT_BLOCKS), dim3(1024), 0, s, q);
  if (!one) hipLaunchKernelGGL(sum_partial_kernel, dim3(1), dim3(64), 0, s, q);
}

// Which of the row kernels takes a row of `bytes`: the fewest threads that hold it with 16 vectors each, so that as many
// rows as possible share a compute unit, each in another phase of its work (16 vectors and about 50 more registers leave
// room for 16 waves, 256 KB of rows); rows of up to 16 KB are a wave's and meet no barrier.  Up to 160 KB 20 vectors let two rows
// share a compute unit where 1024 threads would have it alone (4096 rows of 80000 bf16, policy 284 -> 258 us, distillation 341 ->
// 270; at the other sizes 20 instead of 16 are 1 to 5 % slower).  The largest reads again what is beyond 320 KB.  `kernel` is
// called with the two numbers as a type; it takes 128 registers at most, 4 waves a SIMD.
template <int A, int B> struct Shape {
  static constexpr int TPR = A, NCH = B, BLOCK = A == 64 ? 256 : A, ROWS = BLOCK / A;
};
template <typename F>
auto with_shape(long long bytes, F kernel) {
  if (bytes <= 4 << 10) return kernel(Shape<64, 4>{});
  if (bytes <= 8 << 10) return kernel(Shape<64, 8>{});
  if (bytes <= 16 << 10) return kernel(Shape<64, 16>{});
  if (bytes <= 32 << 10) return kernel(Shape<128, 16>{});
  if (bytes <= 64 << 10) return kernel(Shape<256, 16>{});
  if (bytes <= 128 << 10) return kernel(Shape<512, 16>{});
  if (bytes <= 160 << 10) return kernel(Shape<512, 20>{});
  if (bytes <= 256 << 10) return kernel(Shape<1024, 16>{});
  return kernel(Shape<1024, 20>{});                             // 320 KB of it
}
template <typename F>
auto with_type(int dtype, F f) {
  if (dtype == ST_F32) return f(float{});
  if (dtype == ST_BF16) return f(__bf16{});
  return f(_Float16{});
}

}  // namespace st_token
