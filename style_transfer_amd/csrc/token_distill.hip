// Distillation from a teacher's top logits for gfx950 (token_rows.h: the row kernels' shared code).  HBM-bound.
//
// The list of a row is K pairs (index, value); an index below 0 is unused.  p_k is the teacher's probability of entry k,
// P their sum, and with a bucket for all that is not listed rest = max(0, 1 - P) and q_rest the student's mass off the list:
//   loss / tau^2 = sum p_k (ln p_k - ln q_k) + rest (ln rest - ln q_rest)
//   d / dx_j = tau (Q q_j - p_j) on the list,  tau q_j (Q - rest / q_rest) off it,  Q = P + rest
// q_rest comes from its own sum over the elements off the list (a bitmap in LDS tells them apart): 1 - sum q_k would keep
// no digit of it where the student is sure of a listed token.  Entries that name the same token add up.
//
// One kernel holds a row in registers, with -inf in place of the listed elements, so that its statistics are those off the
// list, and writes the gradient in two steps: the stream as if nothing were listed, then the K entries over it.  A thread of
// the row has one entry of the list (more where K is larger than the threads); entries and their logits are asked for before
// the row, since loads return in order, and stay in registers until they are written.
#include "token_rows.h"

namespace {

using namespace st_token;

constexpr int MAX_VOCAB = 1 << 20;       // the bitmap of a row: 128 KB of LDS
constexpr int MAX_LIST = 4096;           // a list that names a token twice is gone through once for each entry: 1024 rows of 32768
                                         // bf16, value and gradient, 132 -> 188 us with K = 256, 0.12 -> 1.8 ms with 1024, 0.23 -> 28 ms with 4096
constexpr size_t MAX_PLAIN_LDS = 48 << 10;   // dynamic LDS that a kernel gets without asking (64 KB with what it declares)

// what the list of a row, or a wave's part of it, says by itself
struct ListSum {
  double z;                  // sum of exp((v - vref) / tau); tail: the mass itself
  double gap;                // sum of exp((v - vref) / tau) ((v - vref) / tau - (x - m) / tau)
  float m, s, w;             // the listed logits' maximum, S and W of the listed tokens seen from it (once each entry)
  float vref;                // the values' maximum, -inf without any; tail: 0
  int used, bad;             // entries; any outside the vocabulary
};

struct ListIn {
  const void* idx;           // [rows][k] int64 or int32
  int idx64;
  const float* val;          // [rows][k]
  int k;
  const unsigned char* mask; // [rows] or null
  int tail;
  double scale;
  f32x4* row;                // [rows][2]: (m_off, alpha_off, m, alpha_on), (vref, g / Z, an index twice, not zero) or null
};

// index of entry k: -1 unused, -2 outside the vocabulary
__device__ __forceinline__ int entry_index(const ListIn& q, size_t at, int vocab) {
  const long long j = load_index(q.idx, q.idx64, at);
  return j < 0 ? -1 : j >= vocab ? -2 : (int)j;
}

template <typename T>
struct Entry {
  int j;                     // entry_index
  float v;                   // its value
  T x;                       // its logit
};

template <typename T>
__device__ __forceinline__ Entry<T> load_entry(const Logits& p, const ListIn& q, unsigned r, int k, const T* x) {
  Entry<T> e{-1, 0.f, (T)0.f};
  if (k < q.k) {
    e.j = entry_index(q, (size_t)r * q.k + k, p.vocab);
    e.v = q.val[(size_t)r * q.k + k];
    e.x = x[std::max(0, e.j)];
  }
  return e;
}

// A wave's part of the list: entry k of each lane (in `mine`), k + threads, ...  The whole wave calls it.
template <typename T>
__device__ __forceinline__ ListSum sum_list(const Logits& p, const ListIn& q, unsigned r, const T* x, const Entry<T>& mine, int k, int threads) {
  ListSum o;
  float m = -INFINITY, vref = -INFINITY;
  int used = 0, bad = 0;
  Entry<T> e = mine;
  for (int i = k;;) {
    bad |= e.j == -2;
    if (e.j >= 0) {
      m = fmaxf(m, (float)e.x);
      vref = fmaxf(vref, e.v == e.v ? e.v : INFINITY);
      ++used;
    }
    if ((i += threads) >= q.k) break;
    e = load_entry(p, q, r, i, x);
  }
  o.m = lanes_max(m);
  o.vref = q.tail ? 0.f : lanes_max(vref);
  o.used = q.k <= threads ? (int)__popcll(__ballot(used)) : (int)lanes_sum((float)used);
  o.bad = __any(bad);
  const Ref ref = make_ref(o.m, p.c);
  const double it = q.tail ? 1.0 : p.inv_tau, from = o.vref == -INFINITY ? 0.0 : (double)o.vref;
  float s = 0.f, w = 0.f;
  double z = 0.0, gap = 0.0;
  e = mine;
  for (int i = k;;) {
    if (e.j >= 0) {
      const float d = distance((float)e.x, ref, p.c), ex = __builtin_amdgcn_exp2f(d);
      const double lv = ((double)e.v - from) * it, ev = exp64(lv);      // 64 bits: 1 - sum p has no digit left of a p rounded to 32
      s += ex;
      w = fmaf(fmaxf(d, D_MIN), ex, w);
      z += ev;
      if (ev != 0.0) gap += ev * (lv - ((double)(float)e.x - (double)ref.m) * p.inv_tau);
    }
    if ((i += threads) >= q.k) break;
    e = load_entry(p, q, r, i, x);
  }
  o.s = lanes_sum(s);
  o.w = lanes_sum(w);
  o.z = lanes_sum(z);
  o.gap = lanes_sum(gap);
  return o;
}

// the waves' parts as one; lane i of the calling wave has wave i's (a part without entries: m = vref = -inf, the rest 0)
__device__ __forceinline__ ListSum join_lists(const Logits& p, const ListIn& q, const ListSum& part) {
  ListSum o;
  o.m = lanes_max<16>(part.m);
  o.vref = q.tail ? 0.f : lanes_max<16>(part.vref);
  const Ref ref = make_ref(o.m, p.c);
  float s = part.s, w = part.w;
  rebase(s, w, part.m, ref, p.c);
  // (v - vref) / tau and (x - m) / tau of the part's entries change by a and b
  const bool any = part.z != 0;
  const double a = !any || q.tail ? 0.0 : ((double)part.vref - (double)o.vref) * p.inv_tau;
  const double b = any && part.m > -INFINITY ? ((double)part.m - (double)ref.m) * p.inv_tau : 0.0;
  const double f = any ? exp64(a) : 0.0;
  o.s = lanes_sum<16>(s);
  o.w = lanes_sum<16>(w);
  o.z = lanes_sum(any ? f * part.z : 0.0);
  o.gap = lanes_sum(f != 0.0 ? f * (part.gap + part.z * (a - b)) : 0.0);      // an entry without mass does not count: its logit may be -inf
  o.used = (int)lanes_sum<16>((float)part.used);
  o.bad = __any(part.bad);
  return o;
}

// the rows that the mean is over
__global__ __launch_bounds__(1024) void count_mask_kernel(const unsigned char* mask, Sums u) {
  __shared__ double red[16];
  double n = 0;
  for (unsigned r = blockIdx.x * 1024 + threadIdx.x; r < u.rows; r += u.blocks * 1024) n += mask[r] != 0;
  n = block_sum64(n, red);
  if (threadIdx.x == 0) u.counted[blockIdx.x] = n;
}

// A bit for each element of a row, a word of a thread's vectors behind the other: the words of a row's threads lie side by
// side, so that a wave reads them without conflicts, and 32 / VEC vectors cost a thread one read.  The elements outside the
// vectors have the last word.
template <typename T, int TPR>
struct Marks {
  static constexpr int VEC = Type<T>::VEC, PER = 32 / VEC, THREADS = TPR;      // PER: vectors of a word
  uint32_t* bits;

  static __host__ __device__ int words(int vocab) {             // of a row, whatever its alignment
    const int slots = (vocab / VEC + TPR - 1) / TPR;
    return (slots + PER - 1) / PER * TPR + 1;
  }
  // whether it was set before
  __device__ __forceinline__ bool set(const Span<T, TPR>& row, int j, int last) const {
    const int in = j - row.head, i = in / VEC;
    const bool body = in >= 0 && i < row.nv;
    const int slot = i / TPR, at = body ? slot / PER * TPR + i % TPR : last;
    const uint32_t bit = 1u << (body ? slot % PER * VEC + in % VEC : row.owner(j));
    return (atomicOr(bits + at, bit) & bit) != 0;
  }
  // the bits of the PER vectors from slot `slot` on (a multiple of PER)
  __device__ __forceinline__ uint32_t word(int slot, int t) const { return bits[slot / PER * TPR + t]; }
};

// -inf in place of the listed elements.  (Their gradient is written as any other's first and then over it, so that the
// registers keep the row as it is.)
template <typename M>
struct Unlisted {
  M marks;
  int last;                  // the word of the elements outside the vectors
  __device__ __forceinline__ void vector(int slot, int t, float* f) const {
    const uint32_t on = marks.word(slot / M::PER * M::PER, t) >> (slot % M::PER * M::VEC) & ((1u << M::VEC) - 1);
    if (on)
#pragma unroll
      for (int j = 0; j < M::VEC; ++j) f[j] = on >> j & 1 ? -INFINITY : f[j];
  }
  __device__ __forceinline__ float extra(int t, float v) const { return t < 32 && marks.bits[last] >> t & 1 ? -INFINITY : v; }
};

// exp((v - vref) / tau) with the exponent in two numbers, so that it has no rounding: what the difference leaves, and what c (with
// c_lo) leaves of log2(e) / tau.  Most of a gradient's norm is in the listed entries; in 64 bits this is 6 to 15 % of the time of
// short rows (65536 of 1000 bf16, 16384 of 4096).
__device__ __forceinline__ float listed_mass(float v, float vref, float c, float c_lo) {
#pragma clang fp contract(off)
  const float t = v - vref, back = t - v, left = (v - (t - back)) - (vref + back);
  const float y = t * c, k = rintf(y);
  if (y < D_MIN) return 0.f;
  return ldexpf(__builtin_amdgcn_exp2f(fmaf(t, c, -k) + fmaf(left, c, t * c_lo)), (int)k);
}

// The entries of a row's list that lie in [lo, lo + n), over the stream that wrote them as if they were off it: entry t of
// each thread (in `mine`), t + threads, ...  x and out are the row's beginning.
template <typename T>
__device__ __forceinline__ void patch_list(const Logits& p, const ListIn& q, unsigned r, const f32x4& a, const f32x4& b, float scale, int lo,
                                           int n, const T* x, T* out, const Entry<T>& mine, int t, int threads) {
  const double log2e = (q.tail ? 1.0 : p.inv_tau) * (1.0 / LN2);
  const float cv = (float)log2e, cv_lo = (float)(log2e - (double)cv);
  const Ref ref = make_ref(a[2], p.c);
  const size_t first = (size_t)r * q.k;
  Entry<T> e = mine;
  for (int k = t;;) {
    if (e.j >= lo && e.j - lo < n) {
      float pk = 0.f;
      if (b[2] != 0.f) {                                        // an index twice in this row: its entries' sum, in order
        for (int i = 0; i < q.k; ++i)
          if (entry_index(q, first + i, p.vocab) == e.j) pk += listed_mass(q.val[first + i], b[0], cv, cv_lo);
      } else {
        pk = listed_mass(e.v, b[0], cv, cv_lo);
      }
      const float ex = __builtin_amdgcn_exp2f(distance((float)e.x, ref, p.c));
      out[e.j] = (T)(scale * (a[3] * ex - b[1] * pk));
    }
    if ((k += threads) >= q.k) break;
    e = load_entry(p, q, r, k, x);
  }
}

// the list's own sums without what later entries of a token added to the student's side (a whole wave calls it)
template <typename T>
__device__ __forceinline__ ListSum without_repeats(const Logits& p, const ListIn& q, unsigned r, const T* x, ListSum o) {
  const size_t first = (size_t)r * q.k;
  const Ref ref = make_ref(o.m, p.c);
  float s = 0, w = 0, n = 0;
  for (int k = threadIdx.x & 63; k < q.k; k += 64) {
    const int j = entry_index(q, first + k, p.vocab);
    bool again = false;
    if (j >= 0)
      for (int i = 0; i < k; ++i) again |= entry_index(q, first + i, p.vocab) == j;      // no exit: the loads overlap
    if (again) n += 1;
    else if (j >= 0) {
      const float d = distance((float)x[j], ref, p.c), ex = __builtin_amdgcn_exp2f(d);
      s += ex;
      w = fmaf(fmaxf(d, D_MIN), ex, w);
    }
  }
  o.s = lanes_sum(s);
  o.w = lanes_sum(w);
  o.used -= (int)lanes_sum(n);
  return o;
}

// A row's loss (not yet times its weight) and coefficients, from the statistics off the list and the list's own sums.
__device__ __forceinline__ double finish_list(const Logits& p, const ListIn& q, const Part& off, const ListSum& o, double weight, bool repeated,
                                              f32x4& a, f32x4& b) {
#pragma clang fp contract(off)                                  // two equal references over tau have no difference
  const Ref ref = make_ref(fmaxf(off.m, o.m), p.c), ref_off = make_ref(off.m, p.c);
  float s_off = off.s, w_off = off.w, s_list = o.s, w_list = o.w;
  rebase(s_off, w_off, off.m, ref, p.c);
  rebase(s_list, w_list, o.m, ref, p.c);
  const float s = s_list + s_off;
  const double eps = (double)p.eps_ln2;                         // takes c's rounding out of ln S
  const double from = logit_of(ref, p), ln_s = ln64((double)s - eps * (double)(w_list + w_off));      // their sum is ln of the sum of
                                                                // exp(x / tau); references are subtracted from each other first: they may be -1e14
  const double mass = q.tail ? o.z : o.z == 0 ? 0.0 : o.z / o.z;                       // 1, or NaN
  double loss = 0;
  if (mass != 0) {
    loss = (q.tail ? o.gap : o.gap / o.z - ln64(o.z)) + mass * (from - (double)make_ref(o.m, p.c).m * p.inv_tau + ln_s);
    if (s == 0.f) loss = INFINITY;
  }
  const double rest = q.tail && o.used < p.vocab ? (mass < 1 ? 1 - mass : mass >= 1 ? 0.0 : mass) : 0.0;
  const float inv = reciprocal(s), inv_off = reciprocal(off.s);
  if (rest != 0) loss += off.s == 0.f ? INFINITY : rest * (ln64(rest) - (logit_of(ref_off, p) - from + (ln64((double)off.s - eps * (double)off.w) - ln_s)));
  const double gr = q.scale * weight * p.tau, total = mass + rest;
  const float on = s == 0.f ? 0.f : (float)(gr * total * (double)inv);
  const double back = (double)__builtin_amdgcn_exp2f(step(off.m, ref, p.c));
  a = f32x4{ref_off.m, s == 0.f || off.s == 0.f ? 0.f : (float)(gr * (total * (double)inv * back - rest * (double)inv_off)), ref.m, on};
  b = f32x4{o.vref == -INFINITY ? 0.f : o.vref, s == 0.f || mass == 0 ? 0.f : (float)(q.tail ? gr : gr / o.z), repeated ? 1.f : 0.f, s == 0.f || total == 0 ? 0.f : 1.f};
  if (o.used == 0) {                                            // nothing is listed: nothing to learn, whatever the logits hold
    loss = 0;
    a = b = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (o.bad) {
    loss = NAN;
    a[1] = a[3] = NAN;
    b[3] = 1.f;
  }
  return loss;
}

__device__ __forceinline__ void no_list(const ListIn& q, const Sums& u, unsigned r, int t) {
  if (t == 0) u.terms[r] = f64x4{0.0, 0.0, 0.0, 0.0};
  if (t < 2 && q.row) q.row[2 * (size_t)r + t] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// LDS, and for its own stores memory, of a row's threads in order: they are a block, or a wave, whose accesses keep their
// order by themselves.
template <int TPR>
__device__ __forceinline__ void sync_row() {
  if (TPR > 64) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}
template <int TPR>
__device__ __forceinline__ bool sync_row_or(bool v) {
  if (TPR > 64) return __syncthreads_or(v);
  sync_row<TPR>();
  return __any(v);
}

// The logits are read once and the gradient written once: 4096 rows of 32768 bf16, K = 64, in 122 us, 4.4 TB/s (a copy reaches
// 6.4); of 131072 in 507 us, 4.2 TB/s, where one row fills a compute unit and its reading and writing take turns; 1024 rows of
// 131072 fp32, of which the last 192 KB each are read twice (K = 256: 200 MB of that from beyond the L2), in 251 us, 4.3 TB/s.
template <typename T, typename S>
__global__ __launch_bounds__(S::BLOCK, 4) void distill_kernel(Logits p, ListIn q, Sums u, int words, T* __restrict__ grad) {
  constexpr int TPR = S::TPR, VEC = Type<T>::VEC;
  using M = Marks<T, TPR>;
  extern __shared__ uint32_t all_bits[];
  __shared__ Part red[TPR / 64];
  __shared__ ListSum lists[TPR / 64];
  __shared__ f32x4 told[2];
  const int t = threadIdx.x % TPR;
  const M marks{all_bits + (threadIdx.x / TPR) * words};
  const unsigned r = blockIdx.x * S::ROWS + (S::ROWS > 1 ? scalar(threadIdx.x / TPR) : 0);      // the same for a wave
  const bool counts = r < p.rows && (!q.mask || q.mask[r]);
  if (!counts) {                                                // all threads of the row
    if (r >= p.rows) return;
    no_list(q, u, r, t);
    if (grad) store_zeros<T, TPR>(grad + (size_t)r * p.vocab, p.vocab, t);
    return;
  }
  const T* x = reinterpret_cast<const T*>(p.x) + row_offset(p, r);
  const Entry<T> mine = load_entry(p, q, r, t, x);
  for (int i = t; i < words; i += TPR) marks.bits[i] = 0;
  Row<T, TPR, S::NCH> row;
  row.place(x, p.vocab, t);
  sync_row<TPR>();
  bool twice = false;
  const bool has_entries = scalar(t) < q.k;                     // of the wave
  if (has_entries) {
    if (mine.j >= 0) twice = marks.set(row, mine.j, words - 1);
    for (int k = t + TPR; k < q.k; k += TPR) {
      const int j = entry_index(q, (size_t)r * q.k + k, p.vocab);
      if (j >= 0) twice |= marks.set(row, j, words - 1);
    }
  }
  row.load();
  const double share = q.mask ? counted_share(u) : 0.0;
  twice = sync_row_or<TPR>(twice);
  ListSum list{0.0, 0.0, -INFINITY, 0.f, 0.f, -INFINITY, 0, 0};
  if (has_entries) list = sum_list(p, q, r, x, mine, t, TPR);
  if (TPR > 64 && (threadIdx.x & 63) == 0) lists[threadIdx.x >> 6] = list;     // read behind row_join's barrier
  const Part m = row_join<TPR>(row.stats(p.c, Unlisted<M>{marks, words - 1}), p.c, red);
  f32x4 a{0.f, 0.f, 0.f, 0.f}, b{0.f, 0.f, 0.f, 0.f};
  if (TPR == 64 || threadIdx.x < 64) {
    if (TPR > 64) list = join_lists(p, q, threadIdx.x < TPR / 64 ? lists[threadIdx.x] : ListSum{0.0, 0.0, -INFINITY, 0.f, 0.f, -INFINITY, 0, 0});
    if (twice) list = without_repeats(p, q, r, x, list);
    const double w = q.mask ? one_over(share) : 1.0 / u.rows;
    const double loss = w * p.tau * p.tau * finish_list(p, q, m, list, w, twice, a, b);
    if (t == 0) {
      u.terms[r] = f64x4{loss, 0.0, 0.0, 0.0};
      if (q.row) {
        q.row[2 * (size_t)r] = a;
        q.row[2 * (size_t)r + 1] = b;
      }
      if (TPR > 64) {
        told[0] = a;
        told[1] = b;
      }
    }
  }
  if (!grad) return;
  if (TPR > 64) {
    __syncthreads();
    a = told[0];
    b = told[1];
  }
  T* out = grad + (size_t)r * p.vocab;
  const bool zero = b[3] == 0.f;
  if (zero) {
    store_zeros<T, TPR>(out, p.vocab, t);
    return;
  }
  row.store(out, f32x4{a[0], a[1], 0.f, 0.f}, p.c, -1);
  sync_row<TPR>();                                              // a listed element is written twice, in this order
  if (has_entries) patch_list<T>(p, q, r, a, b, 1.f, 0, p.vocab, x, out, mine, t, TPR);
}

// the gradient again, for another upstream gradient or a second time
template <typename T, int TPR>
__global__ __launch_bounds__(NT) void list_grad_kernel(Logits p, ListIn q, const float* gout, int skip_if_one, int splits, int chunk,
                                                       T* __restrict__ grad) {
  const float scale = gout ? gout[0] : 1.f;
  if (skip_if_one && scale == 1.f) return;
  const int t = threadIdx.x % TPR;
  const unsigned long long parts = (unsigned long long)p.rows * splits, step = (unsigned long long)gridDim.x * (NT / TPR);
  for (unsigned long long first = (unsigned long long)blockIdx.x * (NT / TPR); first < parts; first += step) {     // the same for a block's threads
    const unsigned long long part = first + threadIdx.x / TPR;
    const unsigned r = (unsigned)(part / splits);
    const bool live = part < parts;
    const int lo = live ? std::min((long long)(part % splits) * chunk, (long long)p.vocab) : 0;
    const int n = live ? std::min((long long)chunk, (long long)p.vocab - lo) : 0;
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    const f32x4 a = live ? q.row[2 * (size_t)r] : none, b = live ? q.row[2 * (size_t)r + 1] : none;
    const bool zero = b[3] == 0.f;
    T* out = grad + (live ? (size_t)r * p.vocab + lo : 0);
    const T* x = reinterpret_cast<const T*>(p.x) + (live ? row_offset(p, r) + lo : 0);
    if (zero) {
      store_zeros<T, TPR>(out, n, t);
    } else {
      Span<T, TPR>(x, n, t).stream_all(out, f32x4{a[0], a[1] * scale, 0.f, 0.f}, make_ref(a[0], p.c), p.c);
    }
    __syncthreads();                                            // a listed element is written twice, in this order
    if (!zero) patch_list<T>(p, q, r, a, b, scale, lo, n, x - lo, out - lo, load_entry(p, q, r, t, x - lo), t, TPR);
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------------
template <typename T>
int launch_list_grad_t(const char* who, const Logits& p, const ListIn& q, const float* gout, int skip, void* grad, hipStream_t s) {
  const long long bytes = (long long)p.vocab * (long long)sizeof(T);
  const int tpr = bytes <= 4096 ? 64 : NT;
  const int chunk = bytes <= 4096 ? p.vocab : 16384 / (int)sizeof(T);
  const int splits = (int)st::cdivll(p.vocab, chunk);
  // a launch that may have nothing to do is kept small
  const long long blocks = std::min<long long>(st::cdivll((long long)p.rows * splits, NT / tpr), skip ? 4096 : 1LL << 23);
  if (tpr == 64) hipLaunchKernelGGL((list_grad_kernel<T, 64>), dim3((unsigned)blocks), dim3(NT), 0, s, p, q, gout, skip, splits, chunk, (T*)grad);
  else hipLaunchKernelGGL((list_grad_kernel<T, NT>), dim3((unsigned)blocks), dim3(NT), 0, s, p, q, gout, skip, splits, chunk, (T*)grad);
  return st::check_launch(who);
}

}  // namespace

extern "C" size_t st_distill_workspace_bytes(long long rows) {
  if (rows <= 0 || rows > 0x7fffffffLL) return 0;
  return sums_bytes(rows);
}

extern "C" int st_distill_loss_fwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner, int vocab,
                                   const void* teacher_idx, int idx64, const float* teacher_val, int k, const unsigned char* mask, double tau,
                                   int tail, double scale, float* loss, float* row_grad, void* grad, void* workspace, st_stream_t stream) {
  const char* who = "st_distill_loss_fwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, nullptr, 0, 0, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  ST_REQUIRE(rows > 0 && k > 0, "%s: rows=%lld k=%d", who, rows, k);
  ST_REQUIRE(vocab <= MAX_VOCAB && k <= MAX_LIST, "%s: vocab=%d (at most %d), k=%d (at most %d)", who, vocab, MAX_VOCAB, k, MAX_LIST);
  ST_REQUIRE(teacher_idx && teacher_val && loss && workspace, "%s: null pointer", who);
  hipStream_t s = (hipStream_t)stream;
  Space w{reinterpret_cast<char*>(workspace)};
  Sums u = make_sums(w, rows, loss, nullptr, scale, 0.0, 0.0);
  ListIn q{};
  q.idx = teacher_idx;
  q.idx64 = idx64;
  q.val = teacher_val;
  q.k = k;
  q.mask = mask;
  q.tail = tail;
  q.scale = scale;
  q.row = reinterpret_cast<f32x4*>(row_grad);
  u.blocks = (int)std::min<long long>(COUNT_BLOCKS, st::cdivll(rows, 4096));
  if (mask) hipLaunchKernelGGL(count_mask_kernel, dim3(u.blocks), dim3(1024), 0, s, mask, u);
  return with_type(dtype, [&](auto type) {
    using T = decltype(type);
    const int launched = with_shape((long long)vocab * (long long)sizeof(T), [&](auto shape) -> int {
      using S = decltype(shape);
      const int words = Marks<T, S::TPR>::words(vocab);
      const size_t lds = (size_t)words * 4 * S::ROWS;
      if (lds > MAX_PLAIN_LDS) {                                // the attribute is set once a device: to the most that any call needs
        static st::DynLdsOptIn opt_in;
        const int rc = st::allow_dynamic_lds(distill_kernel<T, S>, (size_t)(MAX_VOCAB / 8 + 64), opt_in, who);
        if (rc != ST_OK) return rc;
      }
      const long long blocks = st::cdivll(rows, S::ROWS);
      if (!fits_a_launch(blocks, S::BLOCK)) return st::fail(ST_ERR_BAD_ARG, "%s: rows=%lld vocab=%d: too many for a launch", who, rows, vocab);
      hipLaunchKernelGGL((distill_kernel<T, S>), dim3((unsigned)blocks), dim3(S::BLOCK), lds, s, p, q, u, words, (T*)grad);
      return ST_OK;
    });
    if (launched != ST_OK) return launched;
    launch_sum_terms(u, s);
    return st::check_launch(who);
  });
}

extern "C" int st_distill_loss_bwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner, int vocab,
                                   const void* teacher_idx, int idx64, const float* teacher_val, int k, double tau, int tail,
                                   const float* row_grad, const float* gout, int grad_is_for_one, void* grad, st_stream_t stream) {
  const char* who = "st_distill_loss_bwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, nullptr, 0, 0, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  if (rows == 0) return ST_OK;
  ST_REQUIRE(vocab <= MAX_VOCAB && k > 0 && k <= MAX_LIST, "%s: vocab=%d (at most %d), k=%d (at most %d)", who, vocab, MAX_VOCAB, k, MAX_LIST);
  ST_REQUIRE(teacher_idx && teacher_val && row_grad && grad, "%s: null pointer", who);
  ListIn q{};
  q.idx = teacher_idx;
  q.idx64 = idx64;
  q.val = teacher_val;
  q.k = k;
  q.tail = tail;
  q.row = const_cast<f32x4*>(reinterpret_cast<const f32x4*>(row_grad));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == ST_F32) return launch_list_grad_t<float>(who, p, q, gout, grad_is_for_one, grad, s);
  if (dtype == ST_BF16) return launch_list_grad_t<__bf16>(who, p, q, gout, grad_is_for_one, grad, s);
  return launch_list_grad_t<_Float16>(who, p, q, gout, grad_is_for_one, grad, s);
}
