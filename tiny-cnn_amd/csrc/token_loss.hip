// token_loss.hip — losses of language models on logits: log-probabilities of given tokens, the clipped
// policy loss and the paired preference loss, and their gradients with respect to the logits.
//
// All of them stand on one row operation. With m = max_j x_j, s = sum_j exp(x_j - m) and a target t,
//   logp = x_t - m - log s,    d logp / d x_j = [j = t] - exp(x_j - m) / s,
// so a row's gradient is d ([j = t] - p_j) with one number d per row. A row is read in 16-byte words; a thread
// that holds its words in registers has read the row once when it writes the gradient. m is exact, s is summed
// in fp32 per thread (128 terms at most, or a running sum) and in 64 bits across threads, and what a row makes of
// them (its logarithm, the ratio of two policies, the loss, d) is computed in 64 bits: ratios next to a clipping
// bound decide whether a whole row has a gradient.
#include "lm_types.h"

#include <cfloat>

namespace tdh {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -FLT_MAX;   // the running maximum of nothing: finite, so that -inf - LOWEST is -inf and not NaN

__device__ __forceinline__ float exp_base2(const float x) { return __builtin_amdgcn_exp2f(x); }

// A row's 16-byte words: word k holds elements k * N - shift ... of the row, the first and the last one perhaps
// only partly.
template <class T>
struct Row {
  static constexpr int N = Word<T>::N;
  const T *p;
  int shift, words, len;
  __device__ __forceinline__ Row(const T *row, const int len_) : p(row), len(len_) {
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    words = (shift + len + N - 1) / N;
  }
  __device__ __forceinline__ bool whole(const int k) const { return k * N >= shift && k * N + N <= shift + len; }
  // elements outside the row read as -inf
  template <bool ONCE>
  __device__ __forceinline__ Word<T> load(const int k) const {
    const T *at = p + (static_cast<long>(k) * N - shift);
    if (whole(k)) return load_word<T, ONCE>(at);
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = k * N - shift + e;
      v[e]        = i >= 0 && i < len ? to_f32(at[e]) : -INFINITY;
    }
    return Word<T>::from(v);
  }
};

// Writes word k (in the numbering of the row of logits) of the gradient's row.
template <class T>
__device__ __forceinline__ void store_row_word(const Row<T> &r, T *out, const int k, const float (&v)[Word<T>::N]) {
  T *at = out + (static_cast<long>(k) * Word<T>::N - r.shift);
  if (r.whole(k) && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
    store_word<true>(at, Word<T>::from(v).raw);
    return;
  }
#pragma unroll
  for (int e = 0; e < Word<T>::N; ++e) {
    const int i = k * Word<T>::N - r.shift + e;
    if (i >= 0 && i < r.len) at[e] = from_f32<T>(v[e]);
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// (m, s) of a part of a row: its maximum and the sum of exp(x - m)
struct Part {
  float m;
  double s;
};
__device__ __forceinline__ Part join(const Part a, const Part b) {
  const float m = fmaxf(a.m, b.m);
  return Part{m, a.s * static_cast<double>(exp_base2((a.m - m) * LOG2E)) + b.s * static_cast<double>(exp_base2((b.m - m) * LOG2E))};
}
__device__ __forceinline__ Part wave_join(Part p) {
#pragma unroll
  for (int o = 32; o; o >>= 1) p = join(p, Part{__shfl_xor(p.m, o), __shfl_xor(p.s, o)});
  return p;
}

template <class T>
__device__ __forceinline__ float word_max(const Word<T> &w, float m) {
#pragma unroll
  for (int e = 0; e < Word<T>::N; ++e) m = fmaxf(m, w[e]);
  return m;
}
template <class T>
__device__ __forceinline__ float word_sum(const Word<T> &w, const float m, float s) {
#pragma unroll
  for (int e = 0; e < Word<T>::N; ++e) s += exp_base2((w[e] - m) * LOG2E);
  return s;
}

// What is made of a row: MODE. A row that is read once goes past the caches where nothing reads it again soon: 8192 x
// 65536 logits in bf16, log-probabilities alone 167 us without that and 159 with it; with the gradient's pass behind them
// 476 and 488.
enum { ROW_LOGP, ROW_POLICY };
struct RowArgs {
  const void *logits;
  size_t ld;
  const int32_t *target;
  int rows, vocab;
  float *logp;
  float *stats;     // (m, s) of every row, for the gradient
  double *logp64;   // (preference) the log-probability in 64 bits
  const int32_t *seq_start;   // (preference) rows outside the sequences are neither read nor written
  int sequences;
  // policy
  const float *old_logp, *ref_logp, *advantage, *weight;
  float clip_low, clip_high, kl_coef;
  float *row_loss;
  void *dlogits;
  size_t ld_d;
};

// d, the factor of the gradient, of one row of the policy loss, and the loss itself
__device__ __forceinline__ double policy_row(const RowArgs &a, const int row, const double logp, double *loss) {
  const double w = a.weight ? a.weight[row] : 1.0, adv = a.advantage[row];
  const double ratio = exp(logp - static_cast<double>(a.old_logp[row]));
  const double low = 1.0 - static_cast<double>(a.clip_low), high = 1.0 + static_cast<double>(a.clip_high);
  const double free = ratio * adv, held = (ratio < low ? low : ratio > high ? high : ratio) * adv;
  double l = -(free <= held || free != free ? free : held), d = free <= held ? -free : free > held ? 0.0 : free;
  if (a.ref_logp && a.kl_coef != 0.0f) {   // (a coefficient of 0 leaves the term out, which may be infinite)
    const double gap = static_cast<double>(a.ref_logp[row]) - logp, e = expm1(gap), k = a.kl_coef;
    l += k * (e - gap);
    d -= k * e;
  }
  *loss = w * l;
  return w * d;
}

// What one thread makes of its row, whose maximum and sum it has: d and d / s of the policy loss's gradient
template <class T, int MODE>
__device__ __forceinline__ void finish_row(const RowArgs &a, const int row, const T *x, const int t, const Part p, float *d, float *scale) {
  const bool in = t < a.vocab;
  // (x_t - m first: m + log s would lose the logarithm beside a large m)
  const double lp = in ? static_cast<double>(to_f32(x[in ? t : 0])) - static_cast<double>(p.m) - log(p.s) : __builtin_nan("");
  if (a.logp) a.logp[row] = static_cast<float>(lp);
  if (a.logp64) a.logp64[row] = lp;
  if (a.stats) {
    const bool none = p.s == 0.0;   // nothing but -inf: exp(x - m) is exp(-inf + inf)
    a.stats[2 * static_cast<size_t>(row)]     = none ? -INFINITY : p.m;
    a.stats[2 * static_cast<size_t>(row) + 1] = none ? __builtin_nanf("") : static_cast<float>(p.s);
  }
  if constexpr (MODE == ROW_POLICY) {
    double loss, dd = policy_row(a, row, lp, &loss);
    if (a.row_loss) a.row_loss[row] = static_cast<float>(loss);
    *d     = static_cast<float>(dd);
    *scale = static_cast<float>(dd / p.s);
  }
}
// ... of a row that does not count
template <int MODE>
__device__ __forceinline__ void skip_row(const RowArgs &a, const int row) {
  if (a.logp) a.logp[row] = 0.0f;
  if (a.stats) a.stats[2 * static_cast<size_t>(row)] = a.stats[2 * static_cast<size_t>(row) + 1] = 0.0f;
  if (a.logp64) a.logp64[row] = 0.0;
  if (MODE == ROW_POLICY && a.row_loss) a.row_loss[row] = 0.0f;
}

// WAVES waves a row; W 16-byte words a thread in registers, or W = 0: any number, read once more for the gradient. Rows in
// registers of few waves are fastest as long as several workgroups fit a compute unit (policy loss of 8192 x 32000 in
// bf16, 4000 words: 4 waves 198 us, 8 waves 208, 16 waves 258, read twice 214). Longer rows do not fit 4 waves; 16 of them hold
// up to 16384 words, beyond which the 16 read twice. us so / with 8 waves that read twice: 4096 x 50001 in bf16 197 / 190, 4096 x 32001 in
// fp32 202 / 230, 1024 x 100000 in bf16 88 / 107, 4096 x 131072 in bf16 424 / 452, 2048 x 131075 in fp32 478 / 554.
template <class T, int MODE, int WAVES, int W, bool ONCE>
__global__ void __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256)
row_kernel(const RowArgs a) {
  constexpr int NT = 64 * WAVES, ROWS = WAVES >= 4 ? 1 : 4 / WAVES;   // threads and rows of a workgroup
  constexpr int N = Word<T>::N;
  __shared__ Part parts[WAVES > 1 ? WAVES : 1];
  __shared__ float shared_out[2];
  const int row = blockIdx.x * ROWS + (WAVES == 1 ? threadIdx.x >> 6 : 0);
  const int tid = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  if (row >= a.rows) return;   // (WAVES > 1: the whole workgroup)
  if (a.seq_start && (row < a.seq_start[0] || row >= a.seq_start[a.sequences])) return;
  const T *x = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * a.ld;
  T *dx      = MODE == ROW_POLICY && a.dlogits ? static_cast<T *>(a.dlogits) + static_cast<size_t>(row) * a.ld_d : nullptr;
  const Row<T> r(x, a.vocab);
  const int t = a.target[row];
  if (t < 0) {   // not counted, and not read
    if (tid == 0) skip_row<MODE>(a, row);
    if (dx) {
      const float zero[N] = {};
      for (int k = tid; k < r.words; k += NT) store_row_word(r, dx, k, zero);
    }
    return;
  }

  Word<T> held[W ? W : 1];
  Part p;
  if constexpr (W > 0) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int k = tid + i * NT;
      if (k < r.words) held[i] = r.template load<MODE == ROW_POLICY || ONCE>(k);
    }
    p.m = LOWEST;
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (tid + i * NT < r.words) p.m = word_max(held[i], p.m);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (tid + i * NT < r.words) s = word_sum(held[i], p.m, s);
    p.s = s;
  } else {
    p = Part{LOWEST, 0.0};
    for (int k = tid; k < r.words; k += NT) {
      const Word<T> w = r.template load<MODE == ROW_LOGP && ONCE>(k);
      const float m   = word_max(w, p.m);
      p.s = p.s * static_cast<double>(exp_base2((p.m - m) * LOG2E)) + static_cast<double>(word_sum(w, m, 0.0f));
      p.m = m;
    }
  }
  p = wave_join(p);
  float scale = 0.0f, d = 0.0f;   // d / s and d
  auto finish = [&]() { finish_row<T, MODE>(a, row, x, t, p, &d, &scale); };
  if constexpr (WAVES == 1) {
    if (tid == 0) finish();
    if (MODE != ROW_POLICY || !dx) return;
    d     = __shfl(d, 0);
    scale = __shfl(scale, 0);
  } else {
    if ((tid & 63) == 0) parts[tid >> 6] = p;
    __syncthreads();
    if (tid < 64) {
      p = parts[tid < WAVES ? tid : 0];
      if (tid >= WAVES) p.s = 0.0;
      p = wave_join(p);
      if (tid == 0) {
        finish();
        if (MODE == ROW_POLICY) {
          shared_out[0] = d;
          shared_out[1] = scale;
          parts[0].m    = p.m;
        }
      }
    }
    if (MODE != ROW_POLICY || !dx) return;
    __syncthreads();
    d     = shared_out[0];
    scale = shared_out[1];
    p.m   = parts[0].m;
  }

  if constexpr (MODE == ROW_POLICY) {
    auto grad = [&](const Word<T> &w, const int k) {
      float g[N];
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = -scale * exp_base2((w[e] - p.m) * LOG2E);
      const int at = t - (k * N - r.shift);
      if (at >= 0 && at < N) {
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = e == at ? g[e] + d : g[e];
      }
      store_row_word(r, dx, k, g);
    };
    if constexpr (W > 0) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (tid + i * NT < r.words) grad(held[i], tid + i * NT);
    } else {
      for (int k = tid; k < r.words; k += NT) grad(r.template load<true>(k), k);
    }
  }
}

// Rows of a few logits (small policy nets), a thread each. With `loss` one workgroup has all of them, and adds up the
// losses as well: 6 us, which is a launch and the logarithms and exponentials in 64 bits behind each other; a launch of its own for
// the sum is 4 more.
constexpr int SHORT_ROW = 32, SHORT_NT = 1024;
template <class T, int MODE>
__global__ void __launch_bounds__(SHORT_NT)
short_row_kernel(const RowArgs a, float *__restrict__ loss) {
  __shared__ double part[SHORT_NT / 64];
  const int row = blockIdx.x * blockDim.x + threadIdx.x;
  const bool in = row < a.rows && !(a.seq_start && (row < a.seq_start[0] || row >= a.seq_start[a.sequences]));
  if (in) {
    const T *x  = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * a.ld;
    T *dx       = MODE == ROW_POLICY && a.dlogits ? static_cast<T *>(a.dlogits) + static_cast<size_t>(row) * a.ld_d : nullptr;
    const int t = a.target[row];
    if (t < 0) {
      skip_row<MODE>(a, row);
      if (dx)
        for (int j = 0; j < a.vocab; ++j) dx[j] = T{};
    } else {
      Part p{LOWEST, 0.0};
      for (int j = 0; j < a.vocab; ++j) p.m = fmaxf(p.m, to_f32(x[j]));
      for (int j = 0; j < a.vocab; ++j) p.s += static_cast<double>(exp_base2((to_f32(x[j]) - p.m) * LOG2E));
      float d = 0.0f, scale = 0.0f;
      finish_row<T, MODE>(a, row, x, t, p, &d, &scale);
      if (dx)
        for (int j = 0; j < a.vocab; ++j) {
          const float g = -scale * exp_base2((to_f32(x[j]) - p.m) * LOG2E);
          dx[j] = from_f32<T>(j == t ? g + d : g);
        }
    }
  }
  if (!loss) return;
  double s = in && a.row_loss ? a.row_loss[row] : 0.0;   // (what this thread has just written)
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int w = 0; w < static_cast<int>(blockDim.x / 64); ++w) sum += part[w];
    loss[0] = static_cast<float>(sum);
  }
}

// What the sequences of a pair come to.
struct PairArgs {
  const double *logp64;
  const int32_t *seq_start;
  const float *ref_logp;
  int pairs, rows, kind;
  double beta, smoothing;
  float *seq_logp, *margin, *pair_loss, *d;
};
struct PairValue {
  double margin, loss, d;   // d: of the chosen sequence's gradient, -d of the rejected one's
};
// ... of the sums c and r over the two sequences
__device__ __forceinline__ PairValue pair_value(const PairArgs &a, const int pair, const double c, const double r) {
  const double rc = a.ref_logp ? a.ref_logp[2 * pair] : 0.0, rr = a.ref_logp ? a.ref_logp[2 * pair + 1] : 0.0;
  const double m = a.beta * ((c - rc) - (r - rr));
  double loss, dm;
  switch (a.kind) {
    case TDH_PREF_SIGMOID: {
      // log(1 + exp(-|m|)) on the side where it cannot overflow, and the linear part of the other
      const double e = exp(-fabs(m)), l = log1p(e);
      const double neg = m > 0 ? l : l - m, pos = m > 0 ? l + m : l;   // softplus(-m), softplus(m)
      const double up = (m > 0 ? e : 1.0) / (1.0 + e);                 // sigmoid(-m)
      // (a share of 0 leaves its side out: at an infinite margin the other one is infinite)
      loss = (a.smoothing == 1.0 ? 0.0 : (1.0 - a.smoothing) * neg) + (a.smoothing == 0.0 ? 0.0 : a.smoothing * pos);
      dm   = a.smoothing * ((m > 0 ? 1.0 : e) / (1.0 + e)) - (1.0 - a.smoothing) * up;
    } break;
    case TDH_PREF_SQUARED: {
      const double v = (m - 0.5) / a.beta;
      loss = v * v;
      dm   = 2.0 * v / a.beta;
    } break;
    default:
      loss = m < 1.0 ? 1.0 - m : m >= 1.0 ? 0.0 : m;   // (NaN stays)
      dm   = m < 1.0 ? -1.0 : m >= 1.0 ? 0.0 : m;
      break;
  }
  return PairValue{m, loss, a.beta * dm / a.pairs};
}
// a lane's share of the sum over sequence s, `lanes` of them
__device__ __forceinline__ double sequence_share(const PairArgs &a, const int s, const int t, const int lanes) {
  const int beg = max(0, min(a.rows, a.seq_start[s])), end = max(beg, min(a.rows, a.seq_start[s + 1]));
  double sum = 0.0;
#pragma unroll 4
  for (int i = beg + t; i < end; i += lanes) sum += a.logp64[i];
  return sum;
}
__device__ __forceinline__ void keep_pair(const PairArgs &a, const int pair, const double c, const double r, const PairValue &v) {
  if (a.seq_logp) {
    a.seq_logp[2 * pair]     = static_cast<float>(c);
    a.seq_logp[2 * pair + 1] = static_cast<float>(r);
  }
  if (a.margin) a.margin[pair] = static_cast<float>(v.margin);
}

// dlogits = d ([j = t] - exp(x - m) / s), row by row; workgroups of 256 threads take SPAN words of a row, each of its threads
// GRAD_WORDS that are on their way together. Bound by memory: 4096 x 131072 in bf16 308 us, 7.0 TB/s (the last rows of the pass
// before are still in the memory-side cache).
constexpr int GRAD_NT = 256, GRAD_WORDS = 4, GRAD_SPAN = GRAD_NT * GRAD_WORDS;
struct GradArgs {
  const void *logits;
  size_t ld;
  const int32_t *target;
  int rows, vocab, blocks_per_row;
  const float *stats;       // (m, s) per row
  const float *d;           // per row, or (seq_start) per sequence
  const int32_t *seq_start;
  int sequences;
  void *dlogits;
  size_t ld_d;
  // the mean of these, which a workgroup behind the others computes (null: none)
  const float *pair_loss;
  float *loss;
  PairArgs pair;   // WITH_PAIRS: what d comes from
};
// out[0] = scale * (v[0] + ... + v[n-1]), by one workgroup, in an order that n and its size set
template <int NT>
__device__ __forceinline__ void sum_of(const float *v, const int n, const double scale, float *out) {
  __shared__ double part[NT / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += NT) s += v[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int w = 0; w < NT / 64; ++w) sum += part[w];
    out[0] = static_cast<float>(scale * sum);
  }
}
// WITH_PAIRS: few short sequences, every workgroup adds up those of its row's pair itself, and one behind the others leaves what
// belongs to the pairs: a launch less. us of a loss with a launch for the pairs / so: 3 pairs of up to 41 rows of 1003 logits 12.0 / 9.0; 8 of
// 20 rows of 30000 17.2 / 14.9; 16 of 60 rows of 1000 14.1 / 14.2; one of 1000 rows 13.4 / 15.0; 60 of 10 rows 13.4 / 27.2.
template <class T, bool WITH_PAIRS>
__global__ void __launch_bounds__(GRAD_NT)
dlogits_kernel(const GradArgs a) {
  constexpr int N = Word<T>::N;
  __shared__ double sums[GRAD_NT / 64];
  if (WITH_PAIRS && blockIdx.x == gridDim.x - 1) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double loss = 0.0;
    for (int p = wave; p < a.pair.pairs; p += GRAD_NT / 64) {
      const double c = wave_sum(sequence_share(a.pair, 2 * p, lane, 64)), r = wave_sum(sequence_share(a.pair, 2 * p + 1, lane, 64));
      const PairValue v = pair_value(a.pair, p, c, r);
      loss += v.loss;
      if (lane == 0) keep_pair(a.pair, p, c, r, v);
    }
    if (lane == 0) sums[wave] = loss;
    __syncthreads();
    if (threadIdx.x == 0 && a.loss) {
      for (int w = 1; w < GRAD_NT / 64; ++w) loss += sums[w];
      a.loss[0] = static_cast<float>(loss / a.pair.pairs);
    }
    return;
  }
  if (!WITH_PAIRS && a.loss && blockIdx.x == gridDim.x - 1) {
    sum_of<GRAD_NT>(a.pair_loss, a.sequences / 2, 2.0 / a.sequences, a.loss);
    return;
  }
  const int row = blockIdx.x / a.blocks_per_row, part = blockIdx.x % a.blocks_per_row, tid = threadIdx.x;
  float d = 0.0f;
  if (a.seq_start) {
    // the sequence that the row belongs to: the last one that starts at or before it
    int lo = 0, hi = a.sequences;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.seq_start[mid] <= row) lo = mid; else hi = mid;
    }
    if (row < a.seq_start[0] || row >= a.seq_start[a.sequences]) return;   // in no sequence: left as it is
    if constexpr (WITH_PAIRS) {
      if (tid < 128) {
        const double sum = wave_sum(sequence_share(a.pair, (lo & ~1) + (tid >> 6), tid & 63, 64));
        if ((tid & 63) == 0) sums[tid >> 6] = sum;
      }
      __syncthreads();
      d = static_cast<float>(pair_value(a.pair, lo >> 1, sums[0], sums[1]).d);
      if (lo & 1) d = -d;
    } else {
      d = a.d[lo];
    }
  } else {
    d = a.d[row];
  }
  const T *x = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * a.ld;
  T *dx      = static_cast<T *>(a.dlogits) + static_cast<size_t>(row) * a.ld_d;
  const Row<T> r(x, a.vocab);
  const int t = a.target[row], k0 = part * GRAD_SPAN + tid;
  if (t < 0) {
    const float zero[N] = {};
#pragma unroll
    for (int i = 0; i < GRAD_WORDS; ++i)
      if (k0 + i * GRAD_NT < r.words) store_row_word(r, dx, k0 + i * GRAD_NT, zero);
    return;
  }
  if (t >= a.vocab) d = __builtin_nanf("");
  const float m = a.stats[2 * static_cast<size_t>(row)], scale = d / a.stats[2 * static_cast<size_t>(row) + 1];
  Word<T> w[GRAD_WORDS];
#pragma unroll
  for (int i = 0; i < GRAD_WORDS; ++i)
    if (k0 + i * GRAD_NT < r.words) w[i] = r.template load<true>(k0 + i * GRAD_NT);
#pragma unroll
  for (int i = 0; i < GRAD_WORDS; ++i) {
    const int k = k0 + i * GRAD_NT;
    if (k >= r.words) break;
    float g[N];
#pragma unroll
    for (int e = 0; e < N; ++e) g[e] = -scale * exp_base2((w[i][e] - m) * LOG2E);
    const int at = t - (k * N - r.shift);
    if (at >= 0 && at < N) {
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = e == at ? g[e] + d : g[e];
    }
    store_row_word(r, dx, k, g);
  }
}

constexpr int SUM_NT = 1024;
__global__ void __launch_bounds__(SUM_NT)
sum_kernel(const float *__restrict__ v, const int n, const double scale, float *__restrict__ out) {
  sum_of<SUM_NT>(v, n, scale, out);
}

constexpr int PAIR_NT = 256;
// One workgroup a pair: the sums over its two sequences, its margin, its loss and the factors of its gradient. 4 us, a launch.
__global__ void __launch_bounds__(PAIR_NT)
pair_kernel(const PairArgs a) {
  __shared__ double part[PAIR_NT / 64];
  const int pair = blockIdx.x, tid = threadIdx.x;
  const double sum = wave_sum(sequence_share(a, 2 * pair + (tid >> 7), tid & 127, 128));
  if ((tid & 63) == 0) part[tid >> 6] = sum;
  __syncthreads();
  if (tid) return;
  const double c = part[0] + part[1], r = part[2] + part[3];
  const PairValue v = pair_value(a, pair, c, r);
  keep_pair(a, pair, c, r, v);
  a.pair_loss[pair]   = static_cast<float>(v.loss);
  const float d       = static_cast<float>(v.d);
  a.d[2 * pair]       = d;
  a.d[2 * pair + 1]   = -d;
}

// `again`: the logits are read again soon
template <class T, int MODE>
int launch_rows(const RowArgs &a, bool again) {
  const int words = static_cast<int>((static_cast<long>(a.vocab) * sizeof(T) + 15 + 15) / 16);   // at any alignment
  auto go = [&](auto kernel, int waves) {
    const int rows_per = waves >= 4 ? 1 : 4 / waves;
    TDH_LAUNCH(kernel, dim3(ceil_div(a.rows, rows_per)), dim3(waves > 4 ? 64 * waves : 256), 0, ctx().stream, a);
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  };
  if (a.vocab <= SHORT_ROW) {
    TDH_LAUNCH((short_row_kernel<T, MODE>), dim3(ceil_div(a.rows, 256)), dim3(256), 0, ctx().stream, a, static_cast<float *>(nullptr));
    TDH_LAUNCH_CHECK();
    return TDH_OK;
  }
  if (words <= 64) return go(row_kernel<T, MODE, 1, 1, false>, 1);
  if (words <= 128) return go(row_kernel<T, MODE, 1, 2, false>, 1);
  if (words <= 256) return go(row_kernel<T, MODE, 1, 4, false>, 1);
  // fewer rows than compute units: all the waves there are for each
  if (a.rows > 256) {
    if (words <= 512) return go(row_kernel<T, MODE, 1, 8, false>, 1);
    if (words <= 1024) return go(row_kernel<T, MODE, 4, 4, false>, 4);
    if (words <= 2048) return go(row_kernel<T, MODE, 4, 8, false>, 4);
    if (words <= 4096) return go(row_kernel<T, MODE, 4, 16, false>, 4);
    if constexpr (MODE == ROW_LOGP) return again ? go(row_kernel<T, MODE, 8, 0, false>, 8) : go(row_kernel<T, MODE, 8, 0, true>, 8);
  }
  if (words <= 1024) return go(row_kernel<T, MODE, 16, 1, false>, 16);
  if (words <= 4096) return go(row_kernel<T, MODE, 16, 4, false>, 16);
  if constexpr (MODE == ROW_POLICY) {
    if (words <= 8192) return go(row_kernel<T, MODE, 16, 8, false>, 16);
    if (words <= 16384) return go(row_kernel<T, MODE, 16, 16, false>, 16);
  }
  return go(row_kernel<T, MODE, 16, 0, false>, 16);
}

// workgroups of a row at any alignment
int grad_blocks(int vocab, size_t size) { return ceil_div(static_cast<int>((vocab * size + 15 + 15) / 16), GRAD_SPAN); }
template <class T>
int launch_dlogits(GradArgs a) {
  a.blocks_per_row = grad_blocks(a.vocab, sizeof(T));
  const dim3 grid(a.rows * a.blocks_per_row + (a.loss || a.pair.pairs ? 1 : 0));
  if (a.pair.pairs)
    TDH_LAUNCH((dlogits_kernel<T, true>), grid, dim3(GRAD_NT), 0, ctx().stream, a);
  else
    TDH_LAUNCH((dlogits_kernel<T, false>), grid, dim3(GRAD_NT), 0, ctx().stream, a);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

int launch_sum(const float *v, int n, double scale, float *out) {
  ProfScope prof("loss_sum", 4.0 * n, WORK_BYTE);
  TDH_LAUNCH(sum_kernel, dim3(1), dim3(SUM_NT), 0, ctx().stream, v, n, scale, out);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

constexpr int WITH_PAIRS_PAIRS = 8, WITH_PAIRS_ROWS = 1024, WITH_PAIRS_BLOCKS = 2048;

double logits_bytes(int dtype, int rows, int vocab, int passes) {
  return static_cast<double>(dtype_size(dtype)) * rows * vocab * passes;
}

constexpr size_t LONG_ROW = 65536 - 32;   // bytes of a row that is 4096 words at any alignment
int check_logits(const char *who, int dtype, int rows, int vocab, const void *logits, size_t ld, const int32_t *target) {
  TDH_CHECK_ARG(dtype_known(dtype), "%s: element type %d", who, dtype);
  TDH_CHECK_ARG(rows >= 0 && rows <= GRID_X_MAX && vocab > 0 && vocab <= (1 << 30), "%s: %d rows of %d logits", who, rows, vocab);
  // (a long row has up to 1024 threads, and a launch fewer than 2^32)
  TDH_CHECK_ARG(rows < (1 << 22) || vocab * dtype_size(dtype) <= LONG_ROW, "%s: %d rows of %d logits, more than 64 KB each", who, rows, vocab);
  TDH_CHECK_ARG(ld >= static_cast<size_t>(vocab) && ld <= (static_cast<size_t>(1) << 40), "%s: rows of %d logits %zu elements apart", who, vocab, ld);
  TDH_CHECK_ARG(rows == 0 || (logits && target), "%s: null tensor", who);
  TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(logits) & (dtype_size(dtype) - 1)) == 0, "%s: logits not aligned to their elements", who);
  return TDH_OK;
}

// The gradient may take the logits' place (the same address and row distance), and is apart from them otherwise.
int check_dlogits(const char *who, int dtype, int rows, int vocab, const void *logits, size_t ld, const void *dlogits, size_t ld_d) {
  TDH_CHECK_ARG(ld_d >= static_cast<size_t>(vocab) && ld_d <= (static_cast<size_t>(1) << 40),
                "%s: rows of %d gradients %zu elements apart", who, vocab, ld_d);
  TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(dlogits) & (dtype_size(dtype) - 1)) == 0, "%s: gradient not aligned to its elements", who);
  TDH_CHECK_ARG(static_cast<long>(rows) * grad_blocks(vocab, dtype_size(dtype)) < GRID_X_MAX, "%s: %d rows of %d logits are too many", who, rows, vocab);
  if (rows == 0 || (dlogits == logits && ld_d == ld)) return TDH_OK;
  const uintptr_t x = reinterpret_cast<uintptr_t>(logits), g = reinterpret_cast<uintptr_t>(dlogits), size = dtype_size(dtype);
  TDH_CHECK_ARG(x + size * ((rows - 1) * ld + vocab) <= g || g + size * ((rows - 1) * ld_d + vocab) <= x,
                "%s: the gradient overlaps the logits without taking their place", who);
  return TDH_OK;
}

// the memory that `rows` rows of logits or gradients take
Span span_of(int dtype, int rows, int vocab, const void *p, size_t ld) {
  return Span{p, rows > 0 ? dtype_size(dtype) * ((rows - 1) * ld + vocab) : 0};
}

}  // namespace
}  // namespace tdh

using namespace tdh;

extern "C" {

int tdh_token_logprob_fwd(int dtype, int rows, int vocab, const void *logits, size_t ld, const int32_t *target, float *logp,
                          float *stats) {
  TDH_TRY(check_logits("tdh_token_logprob_fwd", dtype, rows, vocab, logits, ld, target));
  TDH_CHECK_ARG(rows == 0 || logp, "tdh_token_logprob_fwd: null tensor");
  const size_t r4 = 4 * static_cast<size_t>(rows);
  TDH_TRY(check_apart("tdh_token_logprob_fwd", {{logp, r4}, {stats, 2 * r4}}, {span_of(dtype, rows, vocab, logits, ld), {target, r4}}));
  TDH_REQUIRE_INIT();
  if (rows == 0) return TDH_OK;
  RowArgs a{};
  a.logits = logits; a.ld = ld; a.target = target; a.rows = rows; a.vocab = vocab;
  a.logp = logp; a.stats = stats;
  ProfScope prof("token_logprob_fwd", logits_bytes(dtype, rows, vocab, 1), WORK_BYTE);
  return with_dtype(dtype, [&](auto t) { return launch_rows<decltype(t), ROW_LOGP>(a, stats != nullptr); });
}

int tdh_token_logprob_bwd(int dtype, int rows, int vocab, const void *logits, size_t ld, const int32_t *target,
                          const float *stats, const float *dlogp, void *dlogits, size_t ld_d) {
  TDH_TRY(check_logits("tdh_token_logprob_bwd", dtype, rows, vocab, logits, ld, target));
  TDH_TRY(check_dlogits("tdh_token_logprob_bwd", dtype, rows, vocab, logits, ld, dlogits, ld_d));
  TDH_CHECK_ARG(rows == 0 || (stats && dlogp && dlogits), "tdh_token_logprob_bwd: null tensor");
  const size_t r4 = 4 * static_cast<size_t>(rows);
  TDH_TRY(check_apart("tdh_token_logprob_bwd", {span_of(dtype, rows, vocab, dlogits, ld_d)}, {{target, r4}, {stats, 2 * r4}, {dlogp, r4}}));
  TDH_REQUIRE_INIT();
  if (rows == 0) return TDH_OK;
  GradArgs g{};
  g.logits = logits; g.ld = ld; g.target = target; g.rows = rows; g.vocab = vocab;
  g.stats = stats; g.d = dlogp; g.dlogits = dlogits; g.ld_d = ld_d;
  ProfScope prof("token_logprob_bwd", logits_bytes(dtype, rows, vocab, 2), WORK_BYTE);
  return with_dtype(dtype, [&](auto t) { return launch_dlogits<decltype(t)>(g); });
}

int tdh_policy_loss(const tdh_policy_desc *p, int dtype, int rows, int vocab, const void *logits, size_t ld,
                    const int32_t *target, const float *old_logp, const float *ref_logp, const float *advantage,
                    const float *weight, float *logp, float *row_loss, float *loss, void *dlogits, size_t ld_d) {
  TDH_TRY(check_logits("tdh_policy_loss", dtype, rows, vocab, logits, ld, target));
  TDH_CHECK_ARG(p != nullptr, "tdh_policy_loss: null descriptor");
  TDH_CHECK_ARG(p->clip_low >= 0.0f && p->clip_low <= 1.0f && p->clip_high >= 0.0f && p->clip_high <= FLT_MAX,
                "tdh_policy_loss: clipping to 1 - %g .. 1 + %g", p->clip_low, p->clip_high);
  TDH_CHECK_ARG(p->kl_coef >= 0.0f && p->kl_coef <= FLT_MAX, "tdh_policy_loss: KL coefficient %g", p->kl_coef);
  TDH_CHECK_ARG(rows == 0 || (old_logp && advantage), "tdh_policy_loss: null tensor");
  if (dlogits) TDH_TRY(check_dlogits("tdh_policy_loss", dtype, rows, vocab, logits, ld, dlogits, ld_d));
  const size_t r4 = 4 * static_cast<size_t>(rows);
  TDH_TRY(check_apart("tdh_policy_loss", {{logp, r4}, {row_loss, r4}, {loss, 4}, span_of(dtype, rows, vocab, dlogits, ld_d)},
                      {{target, r4}, {old_logp, r4}, {ref_logp, r4}, {advantage, r4}, {weight, r4}}));
  TDH_TRY(check_apart("tdh_policy_loss", {{logp, r4}, {row_loss, r4}, {loss, 4}}, {span_of(dtype, rows, vocab, logits, ld)}));
  TDH_REQUIRE_INIT();
  if (rows == 0) return loss ? launch_sum(nullptr, 0, 1.0, loss) : static_cast<int>(TDH_OK);
  if (loss && !row_loss) {
    TDH_TRY(ws_begin(ws_align(sizeof(float) * rows)));
    void *ws = nullptr;
    TDH_TRY(ws_take(sizeof(float) * rows, &ws));
    row_loss = static_cast<float *>(ws);
  }
  RowArgs a{};
  a.logits = logits; a.ld = ld; a.target = target; a.rows = rows; a.vocab = vocab;
  a.logp = logp;
  a.old_logp = old_logp; a.ref_logp = ref_logp; a.advantage = advantage; a.weight = weight;
  a.clip_low = p->clip_low; a.clip_high = p->clip_high; a.kl_coef = p->kl_coef;
  a.row_loss = row_loss; a.dlogits = dlogits; a.ld_d = ld_d;
  {
    ProfScope prof("policy_loss", logits_bytes(dtype, rows, vocab, dlogits ? 2 : 1), WORK_BYTE);
    if (vocab <= SHORT_ROW && rows <= SHORT_NT && loss)   // one workgroup does it all
      return with_dtype(dtype, [&](auto t) {
        TDH_LAUNCH((short_row_kernel<decltype(t), ROW_POLICY>), dim3(1), dim3((rows + 63) / 64 * 64), 0, ctx().stream, a, loss);
        TDH_LAUNCH_CHECK();
        return static_cast<int>(TDH_OK);
      });
    TDH_TRY(with_dtype(dtype, [&](auto t) { return launch_rows<decltype(t), ROW_POLICY>(a, false); }));
  }
  return loss ? launch_sum(row_loss, rows, 1.0, loss) : static_cast<int>(TDH_OK);
}

int tdh_preference_loss(const tdh_preference_desc *p, int dtype, int pairs, int rows, int vocab, const void *logits, size_t ld,
                        const int32_t *target, const int32_t *seq_start, const float *ref_logp, float *logp,
                        float *seq_logp, float *margin, float *loss, void *dlogits, size_t ld_d) {
  TDH_TRY(check_logits("tdh_preference_loss", dtype, rows, vocab, logits, ld, target));
  TDH_CHECK_ARG(p != nullptr, "tdh_preference_loss: null descriptor");
  TDH_CHECK_ARG(p->kind == TDH_PREF_SIGMOID || p->kind == TDH_PREF_SQUARED || p->kind == TDH_PREF_HINGE,
                "tdh_preference_loss: kind %d", p->kind);
  TDH_CHECK_ARG(p->beta > 0.0f && p->beta <= FLT_MAX, "tdh_preference_loss: beta %g", p->beta);
  TDH_CHECK_ARG(p->smoothing >= 0.0f && p->smoothing <= 1.0f, "tdh_preference_loss: label smoothing %g", p->smoothing);
  TDH_CHECK_ARG(pairs >= 0 && pairs <= (1 << 23), "tdh_preference_loss: %d pairs", pairs);
  TDH_CHECK_ARG(pairs == 0 || seq_start, "tdh_preference_loss: null tensor");
  if (dlogits) TDH_TRY(check_dlogits("tdh_preference_loss", dtype, rows, vocab, logits, ld, dlogits, ld_d));
  const size_t r4 = 4 * static_cast<size_t>(rows), p4 = 4 * static_cast<size_t>(pairs);
  TDH_TRY(check_apart("tdh_preference_loss", {{logp, r4}, {seq_logp, 2 * p4}, {margin, p4}, {loss, 4}, span_of(dtype, rows, vocab, dlogits, ld_d)},
                      {{target, r4}, {seq_start, 2 * p4 + 4}, {ref_logp, 2 * p4}}));
  TDH_TRY(check_apart("tdh_preference_loss", {{logp, r4}, {seq_logp, 2 * p4}, {margin, p4}, {loss, 4}}, {span_of(dtype, rows, vocab, logits, ld)}));
  TDH_REQUIRE_INIT();
  if (pairs == 0) return loss ? launch_sum(nullptr, 0, 1.0, loss) : static_cast<int>(TDH_OK);
  const size_t nr = static_cast<size_t>(rows), np = static_cast<size_t>(pairs);
  TDH_TRY(ws_begin(2 * ws_align(8 * nr) + ws_align(4 * np) + ws_align(8 * np)));
  void *logp64 = nullptr, *stats = nullptr, *pair_loss = nullptr, *d = nullptr;
  TDH_TRY(ws_take(8 * nr, &logp64));
  TDH_TRY(ws_take(8 * nr, &stats));
  TDH_TRY(ws_take(4 * np, &pair_loss));
  TDH_TRY(ws_take(8 * np, &d));
  if (rows) {
    RowArgs a{};
    a.logits = logits; a.ld = ld; a.target = target; a.rows = rows; a.vocab = vocab;
    a.logp = logp; a.logp64 = static_cast<double *>(logp64);
    a.stats = static_cast<float *>(stats);
    a.seq_start = seq_start; a.sequences = 2 * pairs;
    ProfScope prof("preference_logprob", logits_bytes(dtype, rows, vocab, 1), WORK_BYTE);
    TDH_TRY(with_dtype(dtype, [&](auto t) { return launch_rows<decltype(t), ROW_LOGP>(a, dlogits != nullptr); }));
  }
  PairArgs pa{};
  pa.logp64 = static_cast<const double *>(logp64); pa.seq_start = seq_start; pa.ref_logp = ref_logp;
  pa.pairs = pairs; pa.rows = rows; pa.kind = p->kind; pa.beta = p->beta; pa.smoothing = p->smoothing;
  pa.seq_logp = seq_logp; pa.margin = margin; pa.pair_loss = static_cast<float *>(pair_loss); pa.d = static_cast<float *>(d);
  // few pairs, short sequences, and a gradient whose workgroups are all on the chip at once
  const bool with_pairs = dlogits && rows && pairs <= WITH_PAIRS_PAIRS && rows <= WITH_PAIRS_ROWS &&
                          static_cast<long>(rows) * grad_blocks(vocab, dtype_size(dtype)) <= WITH_PAIRS_BLOCKS;
  if (!with_pairs) {
    ProfScope prof("preference_pairs", 8.0 * rows, WORK_BYTE);
    TDH_LAUNCH(pair_kernel, dim3(pairs), dim3(PAIR_NT), 0, ctx().stream, pa);
    TDH_LAUNCH_CHECK();
  }
  if (dlogits && rows) {
    GradArgs g{};
    g.logits = logits; g.ld = ld; g.target = target; g.rows = rows; g.vocab = vocab;
    g.stats = static_cast<const float *>(stats); g.d = static_cast<const float *>(d);
    g.seq_start = seq_start; g.sequences = 2 * pairs; g.dlogits = dlogits; g.ld_d = ld_d;
    g.pair_loss = static_cast<const float *>(pair_loss); g.loss = loss;
    if (with_pairs) g.pair = pa;
    ProfScope prof("preference_grad", logits_bytes(dtype, rows, vocab, 2), WORK_BYTE);
    return with_dtype(dtype, [&](auto t) { return launch_dlogits<decltype(t)>(g); });
  }
  return loss ? launch_sum(static_cast<const float *>(pair_loss), pairs, 1.0 / pairs, loss) : static_cast<int>(TDH_OK);
}

}  // extern "C"
