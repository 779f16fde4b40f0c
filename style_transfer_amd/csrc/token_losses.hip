// Losses over rows of logits for gfx950: the labels' log-probabilities, the preference loss of paired sequences and the
// clipped policy loss with its KL and entropy terms (token_distill.hip: the distillation).  HBM-bound.
//
//   dL/dlogp = a, dL/dH = b:  alpha = -(a + b (H - ln S)) / (tau S)   gamma = -b ln2 / (tau S)   patch: + a / tau at the label
//
// The policy loss of a row decides the row's gradient, so one kernel reads a row once, holds it in registers and writes its
// gradient.  A preference loss couples all rows of a pair: one pass for the statistics, one for the gradient.
#include "token_rows.h"

namespace {

using namespace st_token;

constexpr int MAX_SPLITS = 64;           // parts of a row: one wave joins them

template <typename T>
__device__ __forceinline__ float load_one(const void* base, long long i) {
  return (float)reinterpret_cast<const T*>(base)[i];
}

struct StatsOut {
  float* logp;           // or
  double* wide;          // for sums over sequences, of which a loss takes differences
  float* entropy;
  f32x4* state;
  f32x4* parts;          // [rows][splits], used where splits > 1
  RowGrad* clear;        // row gradients that a loss kernel fills in for the rows it owns
  int again;             // a gradient pass will read the logits again
};

// A row's outputs from its joined statistics: log-probability, entropy, and what the gradient needs.  `state`:
// (m, 1 / (tau S), H - ln S, -).
template <typename T>
__device__ __forceinline__ void write_row(const Logits& p, unsigned r, long long label, const Part& q, const StatsOut& o) {
  const RowStat st = finish(q, p);
  double lp = NAN;
  float inv = st.inv_ts;
  if (label >= 0 && label < p.vocab) lp = log_prob(load_one<T>(p.x, row_offset(p, r) + label), st, p);
  else inv = NAN;                                              // a label outside the vocabulary: visible, never an access
  if (o.logp) o.logp[r] = (float)lp;
  if (o.wide) o.wide[r] = lp;
  if (o.entropy) o.entropy[r] = st.h;
  if (o.state) o.state[r] = f32x4{st.ref, inv, st.inv_ts == 0.f ? 0.f : (float)((double)st.h - st.ln_s), 0.f};
}

__device__ __forceinline__ void write_no_row(unsigned r, const StatsOut& o) {
  if (o.logp) o.logp[r] = 0.f;
  if (o.wide) o.wide[r] = 0.0;
  if (o.entropy) o.entropy[r] = 0.f;
  if (o.state) o.state[r] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// ---- pass 1: the statistics of rows, or of parts of rows ------------------------------------------------------------------
// TPR threads share a part; every part of a row streams its elements once, 16 bytes a load, aligned on the input.
template <typename T, int TPR, bool KEEP>
__device__ __forceinline__ Part stream_part(const T* x, int n, float c, int t) {
  constexpr int VEC = Type<T>::VEC;
  Part p{-INFINITY, 0.f, 0.f};
  const Span<T, TPR> span(x, n, t);
  const u32x4* v = span.body();
  const int nv = span.nv;
  int i = t;
  for (; i + 3 * TPR < nv; i += 4 * TPR) {                     // four loads in flight
    u32x4 b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = KEEP ? v[i + k * TPR] : __builtin_nontemporal_load(v + i + k * TPR);
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
  const int j = span.extra_at();
  if (j >= 0) {
    const float f = (float)x[j];
    take<1>(p, &f, c);
  }
  return p;
}

// One read of the logits, a running reference a thread, no more than a few floats written a row: 4096 rows of 131072 bf16 in
// 175 us, 6.1 TB/s (a kernel that only reads reaches 7.2); one such row, cut into 32 parts, with join_kernel in 6 us.
template <typename T, int TPR, bool KEEP>
__global__ __launch_bounds__(NT) void stats_kernel(Logits p, int splits, int chunk, StatsOut o) {
  __shared__ Part red[NT / 64];
  const int t = threadIdx.x % TPR;
  const unsigned long long part = (unsigned long long)blockIdx.x * (NT / TPR) + scalar(threadIdx.x / TPR);    // the same for a wave
  const unsigned r = (unsigned)(part / splits);
  const int sp = (int)(part % splits);
  const bool live = r < p.rows;
  const long long label = live ? load_index(p.labels, p.labels64, r) : p.ignore;
  if (live && label != p.ignore) {
    const int lo = std::min((long long)sp * chunk, (long long)p.vocab), hi = std::min((long long)lo + chunk, (long long)p.vocab);
    const T* x = reinterpret_cast<const T*>(p.x) + row_offset(p, r) + lo;
    const Part q = row_join<TPR>(stream_part<T, TPR, KEEP>(x, hi - lo, p.c, t), p.c, red);     // TPR > 64: one row, so the barrier is uniform
    if (t == 0) {
      if (splits > 1) o.parts[part] = f32x4{q.m, q.s, q.w, 0.f};
      else write_row<T>(p, r, label, q, o);
    }
  } else if (live && t == 0 && sp == 0) {
    write_no_row(r, o);
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
  if (lane == 0) write_row<T>(p, r, label, q, o);
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
  int backwards;             // from the last row to the first
};

__device__ __forceinline__ RowGrad row_grad(const Logits& p, const GradIn& g, unsigned r, float scale, bool counts) {
  RowGrad v{0.f, 0.f, 0.f, 0.f};
  if (!counts) return v;
  if (g.row) {
    v = g.row[r];
    for (int i = 1; i < 4; ++i) v[i] = v[i] == 0.f ? 0.f : v[i] * scale;      // a row without a gradient has none, whatever comes from above
    return v;
  }
  const f32x4 s = g.state[r];
  const float a = g.g_logp ? g.g_logp[r] : 0.f, b = g.g_entropy ? g.g_entropy[r] : 0.f;
  if (s[1] == 0.f) return v;
  v[0] = s[0];
  v[1] = -(a + b * s[2]) * s[1];
  v[2] = -b * (float)p.inv_ct * s[1];
  v[3] = a * (float)p.inv_tau;
  return v;
}

// Reads the logits again and writes the gradient, 16 KB a block: 4096 rows of 131072 bf16 in 357 us, 6.0 TB/s
// (a copy reaches 6.4).
template <typename T, int TPR>
__global__ __launch_bounds__(NT) void grad_kernel(Logits p, GradIn g, int splits, int chunk, T* __restrict__ grad) {
  const float scale = g.gout ? g.gout[0] : 1.f;
  if (g.skip_if_one && scale == 1.f) return;
  const int t = threadIdx.x % TPR;
  const unsigned long long parts = (unsigned long long)p.rows * splits;
  for (unsigned long long part = (unsigned long long)blockIdx.x * (NT / TPR) + threadIdx.x / TPR; part < parts;
       part += (unsigned long long)gridDim.x * (NT / TPR)) {
    const unsigned at_row = (unsigned)(part / splits), r = g.backwards ? p.rows - 1 - at_row : at_row;
    const int lo = std::min((long long)(part % splits) * chunk, (long long)p.vocab);
    const int n = std::min((long long)chunk, (long long)p.vocab - lo);
    const long long label = load_index(p.labels, p.labels64, r);
    const RowGrad k = row_grad(p, g, r, scale, label != p.ignore);
    T* out = grad + (size_t)r * p.vocab + lo;
    const T* x = reinterpret_cast<const T*>(p.x) + row_offset(p, r) + lo;
    if (k[1] == 0.f && k[2] == 0.f && k[3] == 0.f) {
      store_zeros<T, TPR, true>(out, n, t);
      continue;
    }
    const Span<T, TPR> part_of(x, n, t);
    const Ref ref = make_ref(k[0], p.c);
    part_of.stream_all(out, k, ref, p.c);
    part_of.label(out, k, ref, p.c, (int)std::max(-1ll, std::min(label - lo, (long long)n)));
  }
}

// ---- preference loss ---------------------------------------------------------------------------------------------------
struct PrefIn {
  Sequences seq;             // 2 P sequences: the chosen ones, then the rejected ones
  const double* logp;
  const f32x4* state;
  const float* ref;          // [2 P] or null
  int kind, average;
  double beta, smoothing, scale;
  double* each;              // [P] workspace
  float* loss;
  float* rewards;            // beta (L - ref) of each sequence
  RowGrad* row;              // null without a gradient
};

// A block a pair: the two sums in fp64, the pair's loss and its slope (first wave), the rows' coefficients.
__global__ __launch_bounds__(1024) void pref_kernel(Logits p, PrefIn q) {
  __shared__ double red[16];
  __shared__ double slopes[2];
  const unsigned pairs = q.seq.count / 2, pair = blockIdx.x;
  double sum[2], n[2];
  unsigned start[2], end[2];
  for (int side = 0; side < 2; ++side) {
    sequence(q.seq, pair + side * pairs, start[side], end[side]);
    sum[side] = n[side] = 0;
    for (unsigned r = start[side] + threadIdx.x; r < end[side]; r += blockDim.x) {
      sum[side] += q.logp[r];
      n[side] += load_index(p.labels, p.labels64, r) != p.ignore;
    }
    sum[side] = block_sum64(sum[side], red);
    n[side] = q.average ? block_sum64(n[side], red) : 1.0;
  }
  if (threadIdx.x < 64) {
    double ratio[2], inv[2];
    for (int side = 0; side < 2; ++side) {
      inv[side] = n[side] > 0 ? 1.0 / n[side] : 0.0;
      ratio[side] = sum[side] * (n[side] > 0 ? inv[side] : 1.0) - (q.ref ? (double)q.ref[pair + side * pairs] : 0.0);
    }
    const double h = ratio[0] - ratio[1], z = q.beta * h;
    double loss, slope;
    if (q.kind == ST_PREF_SIGMOID) {
      const double e = exp(-fabs(z)), soft = log1p(e), small = e / (1 + e), large = 1 / (1 + e);
      loss = (1 - q.smoothing) * (soft + fmax(-z, 0.0));
      if (q.smoothing != 0) loss += q.smoothing * (soft + fmax(z, 0.0));       // z is +inf where a rejected label is masked
      slope = q.beta * (q.smoothing * (z > 0 ? large : small) - (1 - q.smoothing) * (z > 0 ? small : large));
      if (z != z) loss = slope = z;
    } else if (q.kind == ST_PREF_IPO) {
      const double v = h - 0.5 / q.beta;
      loss = v * v;
      slope = 2 * v;
    } else {
      loss = z < 1 ? 1 - z : (z >= 1 ? 0.0 : z);                // a NaN stays one
      slope = z < 1 ? -q.beta : (z >= 1 ? 0.0 : z);
    }
    if (threadIdx.x < 2) {
      const int side = threadIdx.x;
      q.rewards[pair + side * pairs] = (float)(q.beta * ratio[side]);
      slopes[side] = (side ? -slope : slope) * inv[side] * q.scale / pairs;
      if (side == 0) q.each[pair] = loss;
    }
  }
  __syncthreads();
  if (q.row)
    for (int side = 0; side < 2; ++side) {
      const float a = (float)slopes[side], patch = (float)(slopes[side] * p.inv_tau);
      for (unsigned r = start[side] + threadIdx.x; r < end[side]; r += blockDim.x) {
        const f32x4 s = q.state[r];
        const bool counts = load_index(p.labels, p.labels64, r) != p.ignore && s[1] != 0.f;
        q.row[r] = counts ? f32x4{s[0], -a * s[1], 0.f, patch} : f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
}

__global__ __launch_bounds__(256) void pref_mean_kernel(PrefIn q) {
  __shared__ double red[4];
  const unsigned pairs = q.seq.count / 2;
  double sum = 0;
  for (unsigned i = threadIdx.x; i < pairs; i += 256) sum += q.each[i];
  sum = block_sum64(sum, red);
  if (threadIdx.x == 0) q.loss[0] = (float)(q.scale * sum / pairs);
}

// ---- clipped policy loss --------------------------------------------------------------------------------------------------
struct PolicyIn {
  Sequences seq;
  const float* old_logp;
  const float* adv;
  int adv_per_sequence;
  const float* ref;          // null: no KL term
  double low, high, kl, ent, scale;
  int per_sequence;          // mean of the sequences' means; else the mean over tokens
  int* count;                // [sequences] labels of each (per_sequence)
  RowGrad* row;
};

struct TokenTerms {
  double part, kl, clipped;  // surrogate, KL estimate, 1 where the clip holds the ratio
  double a;                  // d (surrogate + kl_coef KL) / d logp
};

// exp(d) - 1 - d, which is all that is left of it near 0: its series up to |d| = 1/4 (the term left out is below 2^-36 of it)
__device__ __forceinline__ double kl_estimate(double d) {
  if (!(fabs(d) <= 0.25)) {
    const double e = exp64(d);
    return e == INFINITY ? e : e - 1.0 - d;
  }
  double s = 1.0;
#pragma unroll
  for (int n = 9; n > 2; --n) s = fma(s * d, 1.0 / n, 1.0);
  return 0.5 * d * d * s;
}

__device__ __forceinline__ TokenTerms token_terms(double log_ratio, double d, const PolicyIn& q, double adv) {
  TokenTerms t;
  const double ratio = exp64(log_ratio);
  const bool over = adv > 0 && ratio > 1 + q.high, under = adv < 0 && ratio < 1 - q.low;
  t.clipped = over || under;
  t.part = -adv * (over ? 1 + q.high : under ? 1 - q.low : ratio);
  t.a = t.clipped != 0 ? 0.0 : -adv * ratio;
  t.kl = 0;
  if (q.ref) {
    t.kl = kl_estimate(d);
    if (q.kl != 0) t.a -= q.kl * (d == -INFINITY ? -1.0 : t.kl + d);     // exp(d) - 1
  }
  return t;
}

// The sequence of row r, or -1 outside of all: how many sequences end at or before r, found by 64 probes at a time (8192
// sequences: three steps; one after another they were 128, and 32768 rows of 4096 bf16 took 168 us instead of 92).  A whole
// wave calls it.
__device__ __forceinline__ int sequence_of(const Sequences& q, unsigned r) {
  if (!q.cu) return (int)(r / q.inner);
  unsigned lo = 0, hi = q.count;                                // the answer lies in [lo, hi]
  while (lo < hi) {
    const unsigned step = (hi - lo + 63) / 64, i = lo + ((threadIdx.x & 63) + 1) * step - 1;
    lo += step * (unsigned)__popcll(__ballot(i < hi && q.cu[i + 1] <= (int)r));
    hi = std::min(hi, lo + step - 1);
  }
  return lo < q.count && q.cu[lo] <= (int)r ? (int)lo : -1;
}

// What the mean divides by: labels of all rows, or of each sequence and how many sequences have any.
__global__ __launch_bounds__(1024) void count_kernel(Logits p, PolicyIn q, Sums u) {
  __shared__ double red[16];
  double n = 0;
  if (q.per_sequence) {
    // a wave a sequence; of up to 64 sequences, which may be long, a block each (one of 32768 rows: the loss 230 us -> 108)
    const bool alone = q.seq.count <= COUNT_BLOCKS;
    const unsigned threads = alone ? 1024 : 64, t = threadIdx.x % threads, each = 1024 / threads;
    for (unsigned s = blockIdx.x * each + threadIdx.x / threads; s < q.seq.count; s += gridDim.x * each) {
      unsigned start, end;
      sequence(q.seq, s, start, end);
      double c = 0;
      for (unsigned r = start + t; r < end; r += threads) c += load_index(p.labels, p.labels64, r) != p.ignore;
      c = alone ? block_sum64(c, red) : lanes_sum(c);           // alone: the same s for the whole block
      if (t == 0) {
        q.count[s] = (int)c;
        n += c > 0;
      }
    }
  } else {
    unsigned first = 0, end = q.seq.rows, unused;
    if (q.seq.cu) {                                             // rows outside every sequence do not count
      sequence(q.seq, 0, first, unused);
      sequence(q.seq, q.seq.count - 1, unused, end);
    }
    for (unsigned r = first + blockIdx.x * 1024 + threadIdx.x; r < end; r += gridDim.x * 1024) n += load_index(p.labels, p.labels64, r) != p.ignore;
  }
  n = block_sum64(n, red);
  if (threadIdx.x == 0) u.counted[blockIdx.x] = n;
}

// One pass: a row's statistics, its terms and, where the caller wants one, its gradient (for an upstream gradient of 1).  With
// the row in registers the logits are read once: 4096 rows of 131072 bf16 in 412 to 452 us, 4.8 to 5.2 TB/s read and written (two passes
// take 532), of 32768 in 111 us, 4.9 TB/s; 1024 rows of 131072 fp32, of which the last 192 KB each are read twice, in 254 us, 4.2 TB/s.
// Rows of 2 KB are bound by what a wave does once a row (65536 of 1000 bf16: 79 us, 3.3 TB/s; 5 us of them for a row's
// logarithm, ratio and estimate in 64 bits).
template <typename T, typename S>
__global__ __launch_bounds__(S::BLOCK, 4) void policy_kernel(Logits p, PolicyIn q, Sums u, T* __restrict__ grad) {
  constexpr int TPR = S::TPR;
  __shared__ Part red[TPR / 64];
  __shared__ f32x4 told;
  const int t = threadIdx.x % TPR;
  const unsigned r = blockIdx.x * S::ROWS + (S::ROWS > 1 ? scalar(threadIdx.x / TPR) : 0);      // the same for a wave
  if (r >= p.rows) return;                                      // whole waves (TPR = 64) or the whole block
  const long long label = load_index(p.labels, p.labels64, r);
  const int s = sequence_of(q.seq, r);
  T* out = grad ? grad + (size_t)r * p.vocab : nullptr;
  if (label == p.ignore || s < 0) {
    if (t == 0) {
      u.terms[r] = f64x4{0.0, 0.0, 0.0, 0.0};
      if (q.row) q.row[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (out) store_zeros<T, TPR>(out, p.vocab, t);
    return;
  }
  const T* x = reinterpret_cast<const T*>(p.x) + row_offset(p, r);
  Row<T, TPR, S::NCH> row;
  row.place(x, p.vocab, t);
  row.load();
  // asked for before they are needed: they arrive with the row
  const bool inside = label >= 0 && label < p.vocab;
  const T x_label = x[inside ? label : 0];
  const float old = q.old_logp[r], ref = q.ref ? q.ref[r] : 0.f, adv = q.adv[q.adv_per_sequence ? s : r];
  const double share = counted_share(u);
  const int own = q.per_sequence ? q.count[s] : 1;
  const Part m = row_join<TPR>(row.stats(p.c, Whole{}), p.c, red);
  f32x4 g{0.f, 0.f, 0.f, 0.f};
  if (TPR == 64 || threadIdx.x < 64) {
    const double w = one_over(share) / own;
    const RowStat st = finish(m, p);
    const double logp = inside ? log_prob((float)x_label, st, p) : NAN;
    const TokenTerms k = token_terms(logp - (double)old, (double)ref - logp, q, (double)adv);
    if (st.inv_ts != 0.f) {
      const double a = q.scale * w * k.a, b = -q.scale * w * q.ent, over = (double)st.inv_ts;
      g = f32x4{st.ref, (float)(-(a + b * ((double)st.h - st.ln_s)) * over), (float)(-b * p.inv_ct * over), (float)(a * p.inv_tau)};
    }
    if (t == 0) {
      u.terms[r] = f64x4{w * k.part, w * k.kl, w * (double)st.h, w * k.clipped};
      if (q.row) q.row[r] = g;
      if (TPR > 64) told = g;
    }
  }
  if (!out) return;
  if (TPR > 64) {
    __syncthreads();
    g = told;
  }
  if (g[1] == 0.f && g[2] == 0.f && g[3] == 0.f) store_zeros<T, TPR>(out, p.vocab, t);
  else row.store(out, g, p.c, inside ? (int)label : -1);
}

// ---- host side --------------------------------------------------------------------------------------------------------------
struct Split {
  int tpr, splits, chunk;
};

// Threads of a part and parts of a row.  A row of up to 4 KB is a wave's work (four rows a block share no barrier), and one of up
// to 32 KB where there are enough rows to fill the compute units with waves (forward, bf16: 16384 x 4096 37 -> 26 us, 10300 x
// 6618 37 -> 27, 2048 x 16380 16.7 -> 15.3; 1024 x 8190 7.0 against 7.5, 8192 x 32768 97 against 105); a longer one is a block's.  Where the rows alone would leave compute units idle, a row is cut until there are about four
// blocks for each of the 256, in parts of 8 KB at least (two 16-byte loads a thread).
Split split_of(unsigned rows, int vocab, int size) {
  const long long bytes = (long long)vocab * size;
  if (bytes <= 4096 || (bytes <= 32768 && rows >= 2048)) return {64, 1, vocab};
  int s = 1;
  if (rows < 1024) s = (int)std::min<long long>(MAX_SPLITS, std::min(st::cdivll(1024, std::max(1u, rows)), bytes / 8192));
  s = std::max(1, s);
  const int per = 16 / size;
  const int chunk = (int)std::min<long long>(vocab, st::cdivll(st::cdivll(vocab, s), per) * per);
  return {NT, (int)st::cdivll(vocab, chunk), chunk};
}

// Two passes over logits of up to 512 MB meet in the 256 MB of the memory-side cache if the first leaves them there and the
// second begins with what it read last (4096 rows of 32768 bf16: 142 -> 129 us, 8192: 271 -> 266); of larger ones too little
// is left, and loads past the caches are faster (16384 rows: 532 us against 545).
bool read_twice_from_cache(const Logits& p, int size) { return (long long)p.rows * p.vocab * size <= 512LL << 20; }

template <typename T>
int launch_stats_t(const char* who, const Logits& p, const StatsOut& o, hipStream_t s) {
  const Split k = split_of(p.rows, p.vocab, (int)sizeof(T));
  const long long parts = (long long)p.rows * k.splits, blocks = st::cdivll(parts, NT / k.tpr);
  if (!fits_a_launch(blocks, NT)) return st::fail(ST_ERR_BAD_ARG, "%s: rows=%u vocab=%d: too many for a launch", who, p.rows, p.vocab);
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(NT), 0, s, p, k.splits, k.chunk, o); };
  const bool keep = o.again && read_twice_from_cache(p, (int)sizeof(T));
  if (k.tpr == 64) keep ? launch(stats_kernel<T, 64, true>) : launch(stats_kernel<T, 64, false>);
  else keep ? launch(stats_kernel<T, NT, true>) : launch(stats_kernel<T, NT, false>);
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
  // parts of 16 KB: four 16-byte loads a thread, and enough blocks whatever the number of rows; rows of up to 8 KB are a wave's
  // (16384 x 2500 bf16: 29 us against 33; of 13 KB, 10300 x 6618: 54 against 47)
  const long long bytes = (long long)p.vocab * (long long)sizeof(T);
  const int tpr = bytes <= 8192 ? 64 : NT;
  const int chunk = bytes <= 8192 ? p.vocab : 16384 / (int)sizeof(T);
  const int splits = (int)st::cdivll(p.vocab, chunk);
  // a launch that may have nothing to do is kept small: 131072 blocks that end at once take 28 us, 4096 take 3
  const long long blocks = std::min<long long>(st::cdivll((long long)p.rows * splits, NT / tpr), g.skip_if_one ? 4096 : 1LL << 23);
  if (tpr == 64) hipLaunchKernelGGL((grad_kernel<T, 64>), dim3((unsigned)blocks), dim3(NT), 0, s, p, g, splits, chunk, (T*)grad);
  else hipLaunchKernelGGL((grad_kernel<T, NT>), dim3((unsigned)blocks), dim3(NT), 0, s, p, g, splits, chunk, (T*)grad);
  return st::check_launch(who);
}

int launch_grad(const char* who, int dtype, const Logits& p, GradIn g, void* grad, hipStream_t s) {
  g.backwards = !g.skip_if_one && read_twice_from_cache(p, size_of(dtype));
  if (dtype == ST_F32) return launch_grad_t<float>(who, p, g, grad, s);
  if (dtype == ST_BF16) return launch_grad_t<__bf16>(who, p, g, grad, s);
  return launch_grad_t<_Float16>(who, p, g, grad, s);
}

size_t parts_bytes(long long rows, int vocab, int size) {
  if (rows <= 0 || rows > 0x7fffffffLL || vocab <= 0) return 0;
  const Split k = split_of((unsigned)rows, vocab, size);
  return k.splits > 1 ? align256((size_t)rows * k.splits * sizeof(f32x4)) : 0;
}

}  // namespace

extern "C" size_t st_token_workspace_bytes(int dtype, long long rows, int vocab, long long sequences) {
  if (rows < 0 || sequences < 0) return 0;
  const size_t r = (size_t)rows, q = (size_t)sequences;
  // parts, log-probabilities, statistics, pairs' losses; or rows' terms and sequences' counts
  return std::max(parts_bytes(rows, vocab, size_of(dtype)) + align256(r * 8) + align256(r * 16) + align256(q * 8),
                  sums_bytes(rows) + align256(q * 4));
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
  o.again = state != nullptr;
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
  const int pair_threads = rows <= 512LL * pairs ? 256 : 1024;
  ST_REQUIRE(fits_a_launch(pairs, pair_threads), "%s: pairs=%d: too many for a launch", who, pairs);
  ST_REQUIRE(kind >= ST_PREF_SIGMOID && kind <= ST_PREF_HINGE && beta > 0 && label_smoothing >= 0 && label_smoothing < 0.5,
             "%s: kind=%d beta=%g label_smoothing=%g", who, kind, beta, label_smoothing);
  hipStream_t s = (hipStream_t)stream;
  Space w{reinterpret_cast<char*>(workspace)};
  StatsOut o{};
  PrefIn q{};
  o.parts = w.take<f32x4>(parts_bytes(rows, vocab, size_of(dtype)) / sizeof(f32x4));
  o.wide = w.take<double>((size_t)rows);
  o.state = w.take<f32x4>((size_t)rows);
  q.each = w.take<double>((size_t)pairs);
  o.clear = reinterpret_cast<RowGrad*>(row_grad);
  o.again = row_grad != nullptr;
  q.seq = Sequences{cu_seqlens, 2u * (unsigned)pairs, (unsigned)inner, (unsigned)rows};
  q.logp = o.wide;
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
  // 4096 pairs of 8 tokens: 90 us with 256 threads a pair, 126 with 1024 (32768 rows of 4096 bf16)
  hipLaunchKernelGGL(pref_kernel, dim3((unsigned)pairs), dim3(pair_threads), 0, s, p, q);
  hipLaunchKernelGGL(pref_mean_kernel, dim3(1), dim3(256), 0, s, q);
  return st::check_launch(who);
}

extern "C" int st_policy_loss_fwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner, int vocab,
                                  const void* labels, int labels64, int ignore, double tau, const int* cu_seqlens, int sequences,
                                  const float* old_logps, const float* advantages, int adv_per_sequence, const float* ref_logps,
                                  double clip_low, double clip_high, double kl_coef, double entropy_coef, int per_sequence, double scale,
                                  float* loss, float* stats, float* row_grad, void* grad, void* workspace, st_stream_t stream) {
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
  Sums u = make_sums(w, rows, loss, stats, scale, ref_logps ? kl_coef : 0.0, entropy_coef);
  PolicyIn q{};
  q.count = w.take<int>((size_t)sequences);
  q.seq = Sequences{cu_seqlens, (unsigned)sequences, (unsigned)inner, (unsigned)rows};
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
  q.row = reinterpret_cast<RowGrad*>(row_grad);
  // a block of 1024 threads: a sequence or 16 at a time, or four labels a thread
  u.blocks = (int)std::min<long long>(COUNT_BLOCKS, !per_sequence ? st::cdivll(rows, 4096) : sequences <= COUNT_BLOCKS ? sequences
                                                                                                               : st::cdivll(sequences, 16));
  hipLaunchKernelGGL(count_kernel, dim3(u.blocks), dim3(1024), 0, s, p, q, u);
  rc = with_type(dtype, [&](auto type) {
    using T = decltype(type);
    return with_shape((long long)vocab * (long long)sizeof(T), [&](auto shape) -> int {
      using S = decltype(shape);
      const long long blocks = st::cdivll(rows, S::ROWS);
      if (!fits_a_launch(blocks, S::BLOCK)) return st::fail(ST_ERR_BAD_ARG, "%s: rows=%lld vocab=%d: too many for a launch", who, rows, vocab);
      hipLaunchKernelGGL((policy_kernel<T, S>), dim3((unsigned)blocks), dim3(S::BLOCK), 0, s, p, q, u, (T*)grad);
      return ST_OK;
    });
  });
  if (rc != ST_OK) return rc;
  launch_sum_terms(u, s);
  return st::check_launch(who);
}

extern "C" int st_token_loss_bwd(const void* x, int dtype, long long rows, long long inner, long long s_outer, long long s_inner, int vocab,
                                 const void* labels, int labels64, int ignore, double tau, const float* row_grad, const float* gout,
                                 int grad_is_for_one, void* grad, st_stream_t stream) {
  const char* who = "st_token_loss_bwd";
  Logits p = make_logits(x, rows, inner, s_outer, s_inner, vocab, labels, labels64, ignore, tau);
  int rc;
  if (bad_logits(who, p, dtype, rows, inner, s_outer, s_inner, &rc)) return rc;
  if (rows == 0) return ST_OK;
  ST_REQUIRE(labels && row_grad && grad, "%s: null pointer", who);
  GradIn g{};
  g.row = reinterpret_cast<const RowGrad*>(row_grad);
  g.gout = gout;
  g.skip_if_one = grad_is_for_one;
  return launch_grad(who, dtype, p, g, grad, (hipStream_t)stream);
}

