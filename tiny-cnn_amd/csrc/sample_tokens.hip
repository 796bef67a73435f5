// sample_tokens.hip — a token of every row of logits from a given random number, with temperature, top-k, top-p and min-p.
//
// With the maximum m, token i weighs w_i = exp((x_i - m) / temperature), held as a whole multiple of 2^-fix. Sums of them are sums of integers:
// exact, the same in any order, and so the same wherever a row's sums are split, which is what finds the token: the weights left up to token i are at most u
// times the weights left in all, those up to and with it are more. fix leaves the sum of a row below 2^62.
//
// A filter leaves a beginning of the tokens ordered by logit (and index): those with a logit above V and the first `ties` with V. V is found by
// histograms over ever finer ranges of logits: of counts for top-k, of weights for top-p (select()). min-p is a bound on the logit itself. Nothing is
// sorted.
//
// A workgroup has a row, whose words it keeps in LDS (up to 128 KB of them, else it reads them again in every pass). A few long rows have several
// workgroups in the passes that look at all of a row. Bound by the exponentials in 64 bits, some 20 instructions a logit that counts, and by the
// latency of a chain of passes on one compute unit. bf16, us: 64 rows of 131072 with top_p 0.9 73, with top_k 50 50; 2048 rows of 65536 as they are
// 148, with top_k 50 268, with top_p 0.9 547.
#include "lm_types.h"

#include <cfloat>

namespace tdh {

namespace {

typedef unsigned long long u64;

struct SampleArgs {
  const void *logits;
  size_t ld;
  const float *u;
  const tdh_sample_desc *settings;   // or null: p for all rows
  tdh_sample_desc p;
  int vocab, fix;
  int32_t *token, *kept;
  float *logp, *logq;
};

// 2^t for -1000 <= t < 1000, to 2e-12 of the value: the fit is of (2^f - 1) / f for |f| <= 1/2 (Chebyshev nodes), so that 2^0 is 1. Adding 1.5 * 2^52 leaves
// t to the nearest whole number in the low bits, which go to the exponent as they are.
__device__ __forceinline__ double exp2_64(const double t) {
  constexpr double MAGIC = 6755399441055744.0;
  const double big = t + MAGIC, f = t - (big - MAGIC);
  double p = 1.325080551750225e-06;
  p = __builtin_fma(p, f, 1.5303700711365693e-05);
  p = __builtin_fma(p, f, 0.00015403475186530786);
  p = __builtin_fma(p, f, 0.0013333478473685416);
  p = __builtin_fma(p, f, 0.00961812913523614);
  p = __builtin_fma(p, f, 0.055504109063258665);
  p = __builtin_fma(p, f, 0.24022650695888503);
  p = __builtin_fma(p, f, 0.6931471805568324);
  p = __builtin_fma(p, f, 1.0);
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  u32x2 b = __builtin_bit_cast(u32x2, p);
  b.y += __builtin_bit_cast(u32x2, big).x << 20;
  return __builtin_bit_cast(double, b);
}
constexpr double LOG2E_64 = 1.4426950408889634;

// exp(d) in fp32, d <= 0: the product with log2(e) with its rounding
__device__ __forceinline__ float exp_32(float d) {
  d = fmaxf(d, -200.0f);
  const float t = d * 1.44269504f, r = __builtin_fmaf(d, 1.44269504f, -t) + d * 1.925963033e-8f, e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, 0.69314718f * r, e);
}

// logits in an order of whole numbers, -0 as 0
__device__ __forceinline__ uint32_t key_of(const float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(const uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

template <class V>
__device__ __forceinline__ V wave_total(V v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <class V>
__device__ __forceinline__ V wave_scan(V v) {   // with this lane's own
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V w = __shfl_up(v, o);
    if ((threadIdx.x & 63) >= o) v += w;
  }
  return v;
}
__device__ __forceinline__ float wave_top(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ void no_token(const SampleArgs &a, const int row) {
  a.token[row] = -1;
  if (a.kept) a.kept[row] = 0;
  if (a.logp) a.logp[row] = __builtin_nanf("");
  if (a.logq) a.logq[row] = __builtin_nanf("");
}

// The words of a row, each wave's behind each other: word(i) of this thread, i < per, and a wave's share of the row's words.
template <class T, int NT, bool HELD>
struct RowWords {
  static constexpr int N = Word<T>::N;
  const T *x;
  uint4 *held;   // (HELD) in LDS, where load() put them
  int vocab, words, per, first;
  __device__ __forceinline__ RowWords(const SampleArgs &a, uint4 *lds) : held(lds) {
    x     = static_cast<const T *>(a.logits) + static_cast<size_t>(blockIdx.x) * a.ld;
    vocab = a.vocab;
    words = (vocab + N - 1) / N;
    per   = (words + NT - 1) / NT;
    first = (static_cast<int>(threadIdx.x) >> 6) * per * 64 + (threadIdx.x & 63);
  }
  __device__ __forceinline__ Word<T> load(const int k) const { return row_word(x, k, vocab, -INFINITY); }
  __device__ __forceinline__ Word<T> at(const int k) const { return HELD ? Word<T>{held[k]} : load(k); }
  // f(word, i) of every word that this wave has, the next two on their way meanwhile. All lanes take part in all of them; behind the
  // row's end a word is nothing but -inf.
  template <class F>
  __device__ __forceinline__ void each_word(const F &f) const {
    const int begin = first - (threadIdx.x & 63), mine = min(per, (words - begin + 63) >> 6), last = words - 1;
    if (mine <= 0) return;
    auto get = [&](int i) { return at(min(first + 64 * i, last)); };
    Word<T> now = get(0), next = get(min(1, mine - 1));
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      const Word<T> then = get(min(i + 2, mine - 1));
      if (first + 64 * i > last) {
        constexpr uint32_t nothing = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, bf16>::value ? 0xff80ff80u : 0xfc00fc00u;
        now.raw = make_uint4(nothing, nothing, nothing, nothing);
      }
      f(now, i);
      now  = next;
      next = then;
    }
  }
  template <class F>
  __device__ __forceinline__ void each(const F &f) const {
    each_word([&](const Word<T> &w, int) {
#pragma unroll
      for (int e = 0; e < N; ++e) f(w[e]);
    });
  }
};

// u times all, which the weights up to and with the drawn token's exceed. A u below 0 or NaN is 0, of 1 or more fp32's last number below 1, so that
// less than all comes out (the maximum alone weighs 2^32 or more).
__device__ __forceinline__ u64 place_of(const float u, const u64 all) {
  return static_cast<u64>(static_cast<double>(u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f) * static_cast<double>(all));
}
// (a single maximum: the logarithm of 1 + rest has rest's precision)
__device__ __forceinline__ double log_of_sum(const double tops, const double rest) { return tops == 1.0 ? log1p(rest) : log(tops + rest); }

// --------------------------------------------------------------- without filters
// Long rows without top-k, top-p and min-p. The weights are taken by a reference near the maximum, the largest logit among every thread's first
// words, so that one pass over the row gives the sums of its waves. A second pass has the maximum itself for its reference: where the first one was
// too far below it for whole numbers of 62 bits, or where what is left beside the likeliest token has lost its figures beside that one's weight.
// That wave's words, read once more, give the token.
template <class T, int NT>
__global__ void __launch_bounds__(NT, 2)
sample_all_kernel(const SampleArgs a) {
  constexpr int WAVES = NT / 64, N = Word<T>::N;
  __shared__ float tops[WAVES];
  __shared__ int bads[WAVES], counts[WAVES], top_counts[WAVES];
  __shared__ double sums[WAVES], raws[WAVES];
  __shared__ u64 wholes[WAVES], wholes2[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
  const RowWords<T, NT, false> words(a, nullptr);
  const double temperature = a.p.temperature, rate = LOG2E_64 / temperature, unit = __builtin_ldexp(1.0, min(a.fix, 45));
  const bool with_raw = a.logp && temperature != 1.0;

  float ref = -INFINITY;
  if (words.first < words.words) {
    const Word<T> w = words.load(words.first);
#pragma unroll
    for (int e = 0; e < N; ++e) ref = fmaxf(ref, w[e]);
  }
  ref = wave_top(ref);
  if (lane == 0) tops[wave] = ref;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) ref = fmaxf(ref, tops[w]);
  ref = fabsf(ref) <= FLT_MAX ? ref : 0.0f;

  auto weight = [&](float v) { return exp2_64(__builtin_fmax((static_cast<double>(v) - static_cast<double>(ref)) * rate, -1000.0)); };
  constexpr double SHIFT = 4503599627370496.0;   // 2^52: the sum's low bits are the rounded product
  constexpr u64 SHIFT_BITS = 0x4330000000000000ull;
  // (weights of 2^6 and more of the reference's: to 2^6 of the unit)
  auto whole = [&](double w) {
    return w < 64.0 ? __builtin_bit_cast(u64, __builtin_fma(w, unit, SHIFT)) - SHIFT_BITS
                    : (__builtin_bit_cast(u64, __builtin_fma(w, unit * 0x1p-10, SHIFT)) - SHIFT_BITS) << 10;
  };
  float top = -INFINITY;
  double sum = 0.0, raw = 0.0;   // (second pass: of what is below the maximum)
  int kept = 0, top_n = 0;
  bool second = false;
#pragma unroll 1
  for (;;) {
    u64 s = 0;
    double f = 0.0, q = 0.0;
    int n = 0, tn = 0;
    bool bad = false;
    float t = -INFINITY;
    // e^4 of the reference's weight, or the next smaller number: rounded up by half a place of the reference's it may weigh e^8, for whose whole number
    // 52 bits are too few
    const double border = static_cast<double>(ref) + 4.0 * temperature;
    float large = static_cast<float>(border);
    if (static_cast<double>(large) > border) large = of_key(key_of(large) - 1);
    words.each_word([&](const Word<T> &w, int) {
      float m = w[0];
#pragma unroll
      for (int e = 1; e < N; ++e) m = fmaxf(m, w[e]);
      t = fmaxf(t, m);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        bad = bad || !(w[e] < INFINITY);
        n += __builtin_popcountll(__ballot(w[e] > -INFINITY));
      }
      if (__builtin_expect(second || m > large, 0)) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float v  = w[e];
          const double x = weight(v);
          s += whole(x);
          f += second && v == ref ? 0.0 : x;
          tn += v == ref;
          if (with_raw) q += second && v == ref ? 0.0 : static_cast<double>(exp_32(v - ref));
        }
      } else {
        u64 c = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const double x = weight(w[e]);
          c += __builtin_bit_cast(u64, __builtin_fma(x, unit, SHIFT));
          f += x;
        }
        s += c - N * SHIFT_BITS;
        if (with_raw)
#pragma unroll
          for (int e = 0; e < N; ++e) q += static_cast<double>(exp_32(w[e] - ref));
      }
    });
    t  = wave_top(t);
    s  = wave_total(s);
    f  = wave_total(f);
    tn = wave_total(tn);
    if (with_raw) q = wave_total(q);
    const int any_bad = __any(bad);
    __syncthreads();   // (what was there before has been read)
    if (lane == 0) {
      tops[wave] = t;
      bads[wave] = any_bad;
      counts[wave] = n;
      top_counts[wave] = tn;
      wholes[wave] = s;
      sums[wave] = f;
      raws[wave] = q;
    }
    __syncthreads();
    sum = raw = 0.0;
    kept = top_n = 0;
    int all_bad = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      top = fmaxf(top, tops[w]);
      all_bad |= bads[w];
      kept += counts[w];
      top_n += top_counts[w];
      sum += sums[w];
      raw += raws[w];
    }
    if (all_bad || top == -INFINITY) {   // (the whole workgroup)
      if (tid == 0) no_token(a, row);
      return;
    }
    if (second) break;
    // whole numbers that add up to less than 2^62, and no reference above the maximum (0, where the first words hold nothing but -inf);
    // the likeliest's share below 1 - 10^-4, of fp32's exponentials 0.9
    const double beyond = (static_cast<double>(top) - static_cast<double>(ref)) * rate;
    if (beyond >= 0.0 && beyond < 60.0 && sum * unit < 0x1p61 && sum > 1.0001 * weight(top) &&
        (!with_raw || (top - ref < 80.0f && raw > 1.1 * static_cast<double>(exp_32(top - ref)))))
      break;
    ref    = top;
    second = true;
  }
  u64 all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) all += wholes[w];
  const u64 r = place_of(a.u[row], all);
  u64 before = 0;
  int where = 0;
#pragma unroll 1
  for (; where < WAVES - 1 && before + wholes[where] <= r; ++where) before += wholes[where];
  const int span = words.per * 64, share = (span + NT - 1) / NT, beg = where * span + tid * share;
  const int end = min(min(beg + share, (where + 1) * span), words.words);
  u64 mine = 0;
  for (int k = beg; k < end; ++k) {
    const Word<T> w = words.load(k);
#pragma unroll
    for (int e = 0; e < N; ++e) mine += whole(weight(w[e]));
  }
  const u64 scan = wave_scan(mine);
  if (lane == 63) wholes2[wave] = scan;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    if (w < wave) before += wholes2[w];
  before += scan - mine;
  if (before > r || before + mine <= r) return;
  // one thread is left
  int token = -1;
  float chosen = 0.0f;
  for (int k = beg; k < end && token < 0; ++k) {
    const Word<T> w = words.load(k);
    u64 g[N];
#pragma unroll
    for (int e = 0; e < N; ++e) g[e] = whole(weight(w[e]));
#pragma unroll
    for (int e = 0; e < N; ++e) {
      before += g[e];
      if (token < 0 && before > r) {
        token  = k * N + e;
        chosen = w[e];
      }
    }
  }
  a.token[row] = token;
  if (a.kept) a.kept[row] = kept;
  const double d = static_cast<double>(chosen) - static_cast<double>(ref);
  const double lq = d / temperature - (second ? log_of_sum(top_n, sum) : log(sum));
  if (a.logq) a.logq[row] = static_cast<float>(lq);
  if (a.logp) a.logp[row] = static_cast<float>(!with_raw ? lq : d - (second ? log_of_sum(top_n, raw) : log(raw)));
}

// ------------------------------------------------------------------ with filters
struct RowSettings {
  tdh_sample_desc p;
  bool with_k, with_p, with_q, same;   // same: what is left is all, by its probability under the logits as they are
  int top_k;
  double temperature, rate, share_p;
};
__device__ __forceinline__ RowSettings row_settings(const SampleArgs &a, const int row) {
  RowSettings s;
  s.p = a.settings ? a.settings[row] : a.p;
  const bool greedy = !(s.p.temperature > 0.0f);
  s.temperature     = greedy ? 1.0 : static_cast<double>(s.p.temperature);
  s.rate            = LOG2E_64 / s.temperature;
  s.top_k           = greedy ? 1 : s.p.top_k;
  s.with_k          = s.top_k > 0 && s.top_k < a.vocab;
  s.with_p          = !greedy && s.p.top_p < 1.0f;
  s.with_q          = !greedy && s.p.min_p > 0.0f;
  s.same            = !(s.with_k || s.with_p || s.with_q) && s.temperature == 1.0;
  s.share_p         = fmaxf(s.p.top_p, 0.0f);
  return s;
}
// weights as whole numbers
struct Weights {
  double top, rate, unit;
  // (of 2^-1000 nothing is left, nor where t is 0 times an infinity)
  __device__ __forceinline__ double operator()(const float v) const { return exp2_64(__builtin_fmax((static_cast<double>(v) - top) * rate, -1000.0)); }
  __device__ __forceinline__ u64 whole(const double w) const {
    constexpr double SHIFT = 4503599627370496.0;   // 2^52: the sum's low bits are the rounded product
    return __builtin_bit_cast(u64, __builtin_fma(w, unit, SHIFT)) - __builtin_bit_cast(u64, SHIFT);
  }
};
// What is left of a wave's or a workgroup's words: weight and number above V, number with V; of the weights below the maximum, and of the exponentials of
// all logits below it, the sums in floating point; number of maxima.
struct Left {
  u64 gt;
  double rest, raw;
  int gt_n, ties, tops;
  __device__ __forceinline__ void add(const Left &o) {
    gt += o.gt;
    rest += o.rest;
    raw += o.raw;
    gt_n += o.gt_n;
    ties += o.ties;
    tops += o.tops;
  }
};
// ... of a wave, whose words `each(f)` gives to f, by all of its lanes. Those above V are put behind each other in a queue of the wave's own, and weighed 64
// at a time.
constexpr int LEFT_QUEUE = 256;
template <class Each>
__device__ __forceinline__ Left weigh_left(const Each &each, const float V, const float top, const Weights &weight, const bool with_raw, float *queue) {
  const int lane = threadIdx.x & 63;
  Left l{};
  int queued = 0;
  auto weigh = [&](const int m) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    queued -= m;
    if (lane < m) {
      const float v  = queue[queued + lane];
      const double x = weight(v);
      l.gt += weight.whole(x);
      l.rest += v < top ? x : 0.0;
      l.tops += v == top;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  each([&](const auto &w) {
    constexpr int N = std::remove_reference_t<decltype(w)>::N;
    float m = w[0];
#pragma unroll
    for (int e = 1; e < N; ++e) m = fmaxf(m, w[e]);
    if (__any(m >= V))
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v  = w[e];
        const u64 keep = __ballot(v > V);
        l.ties += __builtin_popcountll(__ballot(v == V));
        if (v > V) queue[queued + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(keep >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(keep), 0))] = v;
        queued += __builtin_popcountll(keep);
        l.gt_n += __builtin_popcountll(keep);
        if (e & 1)
          while (queued >= 64) weigh(64);
      }
    if (with_raw) {
      float r = 0.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) r += w[e] < top ? exp_32(w[e] - top) : 0.0f;
      l.raw += static_cast<double>(r);
    }
  });
  weigh(queued);
  l.gt   = wave_total(l.gt);
  l.tops = V == top ? l.ties : wave_total(l.tops);
  l.rest = wave_total(l.rest);
  l.raw  = wave_total(l.raw);
  return l;
}
// The token, of what is left in `count` pieces of `span` words each, and all results of the row. By the whole workgroup; get(k): word k.
template <class T, int NT, class Get>
__device__ __forceinline__ void draw_token(const SampleArgs &a, const RowSettings &set, const Weights &weight, const float top, const float V, const u64 ties,
                                           const Left *left, const int count, const int span, const int words, const Get &get, u64 (&gt2)[NT / 64],
                                           int (&ties2)[NT / 64]) {
  constexpr int WAVES = NT / 64, N = Word<T>::N;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
  const double v_weight64 = weight(V);
  const u64 v_weight = weight.whole(v_weight64);
  u64 gt_all = 0, ties_all = 0;
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    gt_all += left[i].gt;
    ties_all += left[i].ties;
  }
  const u64 ties_left = min(ties, ties_all), all = gt_all + v_weight * ties_left;
  const u64 r = place_of(a.u[row], all);
  // the weights left up to a place with `g` above V and `t` with V in front of it
  auto upto = [&](u64 g, u64 t) { return g + v_weight * min(t, ties_left); };
  u64 g0 = 0, t0 = 0;
  int where = 0;
#pragma unroll 1
  for (; where < count - 1; ++where) {
    const u64 g1 = g0 + left[where].gt, t1 = t0 + left[where].ties;
    if (upto(g1, t1) > r) break;
    g0 = g1;
    t0 = t1;
  }
  // that piece's words, a share for every thread
  const int share = (span + NT - 1) / NT, beg = where * span + tid * share, end = min(min(beg + share, (where + 1) * span), words);
  u64 gt = 0;
  int at = 0;
  for (int k = beg; k < end; ++k) {
    const Word<T> w = get(k);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (w[e] > V) gt += weight.whole(weight(w[e]));
      at += w[e] == V;
    }
  }
  const u64 gt_scan = wave_scan(gt);
  const int at_scan = wave_scan(at);
  if (lane == 63) {
    gt2[wave]   = gt_scan;
    ties2[wave] = at_scan;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    if (w < wave) {
      g0 += gt2[w];
      t0 += ties2[w];
    }
  g0 += gt_scan - gt;
  t0 += at_scan - at;
  if (upto(g0, t0) > r || upto(g0 + gt, t0 + at) <= r) return;
  // one thread is left
  int token = -1;
  float chosen = V;
  for (int k = beg; k < end && token < 0; ++k) {
    const Word<T> w = get(k);
    u64 g[N];
#pragma unroll
    for (int e = 0; e < N; ++e) g[e] = w[e] > V ? weight.whole(weight(w[e])) : 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      g0 += g[e];
      t0 += w[e] == V;
      if (token < 0 && w[e] >= V && upto(g0, t0) > r) {
        token  = k * N + e;
        chosen = w[e];
      }
    }
  }
  a.token[row] = token;
  Left sum{};
#pragma unroll 1
  for (int i = 0; i < count; ++i) sum.add(left[i]);
  if (a.kept) a.kept[row] = static_cast<int>(sum.gt_n + ties_left);
  const double d = static_cast<double>(chosen) - weight.top;
  if (a.logq) a.logq[row] = static_cast<float>(V == top ? -log(static_cast<double>(ties_left))
                                                        : d / set.temperature - log_of_sum(sum.tops, sum.rest + v_weight64 * static_cast<double>(ties_left)));
  if (a.logp) a.logp[row] = static_cast<float>(d - log_of_sum(sum.tops, set.same ? sum.rest : sum.raw));
}
constexpr int SAMPLE_LIST = 2048, SAMPLE_SHORT = 128;   // logits that a list takes, and that one wave goes through by itself
// LDS of a row's workgroup
template <int NT>
struct SampleShared {
  static constexpr int WAVES = NT / 64, BINS = 2 * NT;
  u64 hist[BINS];   // (counts: the first half of it)
  float list[SAMPLE_LIST];
  u64 sum[WAVES];
  u64 found_above, found_upto, found_ties;
  float found_v;
  int found_bin, listed;
  float top[WAVES], far[WAVES];
  int bad[WAVES], n[WAVES];
  Left left[WAVES];
  u64 gt2[WAVES];
  int ties2[WAVES];
};

// The ranges of a first round: equal ones of the distance from the maximum, the last for what is beyond. That one's sum takes no atomics, so it
// begins behind the average where a target is likely to be nearer. bf16, top_p 0.9, us, by 1.2 and by 4 times the average: 64 rows of 131072 75 and 81, 256 of
// 32000 47 and 53, but 2048 of 65536 545 and 515: it pays where few rows wait for it. Finite masks count in the average and leave all that matters in the first few ranges: the
// results are the same, but 2048 rows of 65536, half of them masked, take with top_p 0.9 780 where the mask is -1e4, 880 of -1e9 and 1170 of the lowest number, of -inf 500; with top_k 50
// 490, 730, 1120 and 270.
template <int BINS>
struct FirstBins {
  float top, scale;
  __device__ __forceinline__ FirstBins(const float top, const float mean, const bool near) : top(top) {
    const float reach = (near ? 1.2f : 4.0f) * mean;
    scale             = reach > 0.0f ? BINS / reach : 0.0f;
  }
  __device__ __forceinline__ int operator()(const float v) const { return static_cast<int>(fminf((top - v) * scale, static_cast<float>(BINS - 1))); }
};
__device__ __forceinline__ bool near_p(const RowSettings &s) { return s.p.top_p <= 0.95f; }

// Few long rows: what needs all of a row's logits and is the same in any order comes from several workgroups a row, in two launches ahead of the row's
// own: the maximum, and by it the sums of exponentials and the first histogram of top-p's.
struct SamplePart {
  float top, far;   // the largest logit, and the sum of `n` finite ones
  int n, bad;
};
struct SampleBound {   // logits above v are left, and the first `ties` that are v
  float v;
  u64 ties;
};
struct SampleAhead {
  SamplePart *parts;   // [rows][count]
  double *raw;         // [rows][count]
  u64 *hist;           // [rows][2048]
  SampleBound *bounds; // [rows]
  Left *left;          // [rows][count]
  int count, chunk;    // workgroups of a row, words of each
};
constexpr int SAMPLE_BINS = 2048, AHEAD_NT = 512, AHEAD_MOST = 32;
struct RowTop {
  float top, mean;
  bool bad;
};
__device__ __forceinline__ RowTop row_top(const float top, const float far, const int n, const bool bad) {
  return RowTop{top, n ? top - far / static_cast<float>(n) : 16.0f, bad || top == -INFINITY};
}
// (a lane a part: one after the other they take their way from memory each, 8 parts 4 us)
__device__ __forceinline__ RowTop row_top(const SampleAhead &ahead, const int row) {
  const int lane = threadIdx.x & 63;
  SamplePart p{-INFINITY, 0.0f, 0, 0};
  if (lane < ahead.count) p = ahead.parts[row * ahead.count + lane];
  return row_top(wave_top(p.top), wave_total(p.far), wave_total(p.n), __any(p.bad));
}
template <class T>
__global__ void __launch_bounds__(AHEAD_NT)
sample_top_kernel(const SampleArgs a, const SampleAhead ahead) {
  constexpr int WAVES = AHEAD_NT / 64, N = Word<T>::N;
  __shared__ SamplePart waves[WAVES];
  const int tid = threadIdx.x, row = blockIdx.y, part = blockIdx.x, words = (a.vocab + N - 1) / N;
  const int beg = min(words, part * ahead.chunk), end = min(words, beg + ahead.chunk);
  const T *x = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * a.ld;
  for (int b = part * AHEAD_NT + tid; b < SAMPLE_BINS; b += ahead.count * AHEAD_NT) ahead.hist[static_cast<size_t>(row) * SAMPLE_BINS + b] = 0;
  float top = -INFINITY, far = 0.0f;
  int n = 0;
  bool strange = false;
#pragma unroll 4
  for (int k = beg + tid; k < end; k += AHEAD_NT) {
    const Word<T> w = row_word(x, k, a.vocab, -INFINITY);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      top     = fmaxf(top, w[e]);
      strange = strange || !(w[e] < INFINITY);
    }
    if (k < beg + AHEAD_NT)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        far += w[e] > -INFINITY ? w[e] : 0.0f;
        n += w[e] > -INFINITY;
      }
  }
  top = wave_top(top);
  far = wave_total(far);
  n   = wave_total(n);
  const int bad = __any(strange);
  if ((tid & 63) == 0) waves[tid >> 6] = SamplePart{top, far, n, bad};
  __syncthreads();
  if (tid) return;
  SamplePart all = waves[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    all.top = fmaxf(all.top, waves[w].top);
    all.far += waves[w].far;
    all.n += waves[w].n;
    all.bad |= waves[w].bad;
  }
  ahead.parts[row * ahead.count + part] = all;
}
template <class T>
__global__ void __launch_bounds__(AHEAD_NT)
sample_sums_kernel(const SampleArgs a, const SampleAhead ahead) {
  constexpr int WAVES = AHEAD_NT / 64, N = Word<T>::N;
  __shared__ u64 hist[SAMPLE_BINS];
  __shared__ double raws[WAVES];
  const int tid = threadIdx.x, row = blockIdx.y, part = blockIdx.x, words = (a.vocab + N - 1) / N;
  const int beg = min(words, part * ahead.chunk), end = min(words, beg + ahead.chunk);
  const T *x = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * a.ld;
  const RowSettings s = row_settings(a, row);
  const RowTop r      = row_top(ahead, row);
  const bool with_raw = a.logp && !s.same, with_hist = s.with_p && !s.with_k;
  if (tid == 0) ahead.raw[row * ahead.count + part] = 0.0;
  if (r.bad || !(with_raw || with_hist)) return;   // (the whole workgroup)
  const Weights weight{r.top, s.rate, __builtin_ldexp(1.0, a.fix)};
  const FirstBins<SAMPLE_BINS> bin_of(r.top, r.mean, near_p(s));
  for (int b = tid; b < SAMPLE_BINS; b += AHEAD_NT) hist[b] = 0;
  __syncthreads();
  double raw = 0.0;
  u64 last   = 0;
#pragma unroll 1
  for (int k = beg + tid; k < end; k += AHEAD_NT) {
    const Word<T> w = row_word(x, k, a.vocab, -INFINITY);
    if (with_hist)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const u64 v = weight.whole(weight(w[e]));
        const int b = bin_of(w[e]);
        last += b == SAMPLE_BINS - 1 ? v : 0;
        if (b < SAMPLE_BINS - 1) atomicAdd(&hist[b], v);
      }
    if (with_raw) {
      float f = 0.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) f += w[e] < r.top ? exp_32(w[e] - r.top) : 0.0f;
      raw += static_cast<double>(f);
    }
  }
  last = wave_total(last);
  raw  = wave_total(raw);
  if ((tid & 63) == 0) {
    if (last) atomicAdd(&hist[SAMPLE_BINS - 1], last);
    raws[tid >> 6] = raw;
  }
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < WAVES; ++w) raw += raws[w];
    ahead.raw[row * ahead.count + part] = raw;
  }
  if (with_hist)
    for (int b = tid; b < SAMPLE_BINS; b += AHEAD_NT)
      if (hist[b]) atomicAdd(&ahead.hist[static_cast<size_t>(row) * SAMPLE_BINS + b], hist[b]);
}

// the two of them for the rows of several workgroups
template <class T>
__global__ void __launch_bounds__(AHEAD_NT)
sample_left_kernel(const SampleArgs a, const SampleAhead ahead) {
  constexpr int WAVES = AHEAD_NT / 64, N = Word<T>::N;
  __shared__ float queues[WAVES][LEFT_QUEUE];
  __shared__ Left waves[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y, part = blockIdx.x, words = (a.vocab + N - 1) / N;
  const int beg = min(words, part * ahead.chunk), end = min(words, beg + ahead.chunk);
  const RowSettings s = row_settings(a, row);
  const RowTop r      = row_top(ahead, row);
  if (r.bad) return;   // (the whole workgroup)
  const T *x = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * a.ld;
  const Weights weight{r.top, s.rate, __builtin_ldexp(1.0, a.fix)};
  const Left mine = weigh_left(
      [&](auto f) {
#pragma unroll 1
        for (int k0 = beg + 64 * wave; k0 < end; k0 += AHEAD_NT) {
          float none[N];
#pragma unroll
          for (int e = 0; e < N; ++e) none[e] = -INFINITY;
          f(k0 + lane < end ? row_word(x, k0 + lane, a.vocab, -INFINITY) : Word<T>::from(none));
        }
      },
      ahead.bounds[row].v, r.top, weight, false, queues[wave]);
  if (lane == 0) waves[wave] = mine;
  __syncthreads();
  if (tid) return;
  Left all = waves[0];
  for (int w = 1; w < WAVES; ++w) all.add(waves[w]);
  all.raw = ahead.raw[row * ahead.count + part];
  ahead.left[row * ahead.count + part] = all;
}
constexpr int DRAW_NT = 1024;
template <class T>
__global__ void __launch_bounds__(DRAW_NT)
sample_draw_kernel(const SampleArgs a, const SampleAhead ahead) {
  constexpr int N = Word<T>::N;
  __shared__ u64 gt2[DRAW_NT / 64];
  __shared__ int ties2[DRAW_NT / 64];
  __shared__ Left left[AHEAD_MOST];
  const int row = blockIdx.x;
  if (threadIdx.x < ahead.count) left[threadIdx.x] = ahead.left[row * ahead.count + threadIdx.x];
  __syncthreads();
  const RowSettings s = row_settings(a, row);
  const RowTop r      = row_top(ahead, row);
  if (r.bad) return;   // (the whole workgroup; the row has its results)
  const SampleBound b = ahead.bounds[row];
  const Weights weight{r.top, s.rate, __builtin_ldexp(1.0, a.fix)};
  const T *x = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * a.ld;
  draw_token<T, DRAW_NT>(a, s, weight, r.top, b.v, b.ties, left, ahead.count, ahead.chunk, (a.vocab + N - 1) / N,
                         [&](int k) { return row_word(x, k, a.vocab, -INFINITY); }, gt2, ties2);
}

template <class T, int NT, bool HELD, bool AHEAD>
__global__ void __launch_bounds__(NT)
sample_kernel(const SampleArgs a, const SampleAhead ahead) {
  using Shared = SampleShared<NT>;
  constexpr int WAVES = Shared::WAVES, BINS = Shared::BINS, N = Word<T>::N;
  extern __shared__ uint4 row_lds[];
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x, vocab = a.vocab;
  const RowWords<T, NT, HELD> words(a, row_lds);

  const RowSettings set = row_settings(a, row);
  const tdh_sample_desc &p = set.p;
  const bool with_k = set.with_k, with_p = set.with_p, with_q = set.with_q;
  const int top_k = set.top_k;
  const double temperature = set.temperature, share_p = set.share_p;

  // maximum, and how far others lie from it on average: those of every thread's first word will do
  RowTop all_top;
  if constexpr (AHEAD) {
    all_top = row_top(ahead, row);
    if (tid == 0) sh.listed = 0;
    __syncthreads();
  } else {
    float top = -INFINITY, far = 0.0f;
    int n = 0;
    bool strange = false;
    RowWords<T, NT, false>(a, nullptr).each_word([&](const Word<T> &w, int i) {
      if (HELD && words.first + 64 * i < words.words) row_lds[words.first + 64 * i] = w.raw;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        top     = fmaxf(top, w[e]);
        strange = strange || !(w[e] < INFINITY);
      }
      if (i == 0)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          far += w[e] > -INFINITY ? w[e] : 0.0f;
          n += w[e] > -INFINITY;
        }
    });
    top = wave_top(top);
    far = wave_total(far);
    n   = wave_total(n);
    int bad = __any(strange);
    if (lane == 0) {
      sh.top[wave] = top;
      sh.far[wave] = far;
      sh.bad[wave] = bad;
      sh.n[wave]   = n;
    }
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    far = 0.0f;
    n = bad = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      top = fmaxf(top, sh.top[w]);
      far += sh.far[w];
      n += sh.n[w];
      bad |= sh.bad[w];
    }
    all_top = row_top(top, far, n, bad);
  }
  const float top = all_top.top, mean = all_top.mean;
  if (all_top.bad) {   // (the whole workgroup)
    if (tid == 0) no_token(a, row);
    return;
  }
  const double top64 = top;
  const Weights weight{top64, set.rate, __builtin_ldexp(1.0, a.fix)};
  auto whole = [&](double w) { return weight.whole(w); };

  // What is left: logits above V, and the first `ties` of those that are V
  float V  = -INFINITY;
  u64 ties = 0;
  bool in_list = false;   // all that is left is in the list

  // The logit at which the sum over what is left, from the largest logit on, reaches a target: top_k (counts) or the share top_p of
  // all (weights). V becomes that logit and ties what is missing there. The first round is over the row, those behind it over the logits that the first
  // one leaves in question, in the list if they fit.
  auto select = [&](auto zero) {
    using M = decltype(zero);
    constexpr bool MASS = sizeof(M) == 8;
    M *hist = reinterpret_cast<M *>(sh.hist);
    const FirstBins<BINS> bin_of(top, mean, MASS ? near_p(set) : top_k <= vocab / 8);
    // the smallest logit, as a key, in range b or one before it; by all the lanes of every wave
    auto first_in = [&](const int b) {
      uint32_t from = key_of(-FLT_MAX), to = key_of(top);
      while (from < to) {
        const uint32_t at = from + static_cast<uint32_t>((static_cast<u64>(to - from) * lane) / 63);
        const int hit = __builtin_ctzll(__ballot(bin_of(of_key(at)) <= b));   // (the last lane's is the maximum, or known to be)
        to = __shfl(at, hit);
        if (hit == 0) break;
        from = __shfl(at, hit - 1) + 1;
      }
      return to;
    };
    const u64 v_weight = MASS ? whole(weight(V)) : 0;
    u64 above = 0, target = MASS ? 0 : static_cast<u64>(top_k);
    int shift = 0;
    uint32_t lo = 0, hi = 0;
    bool listed = in_list;
    // A short list in one wave: each lane has a logit, and what the larger ones come to. `whole_sum`: the list has all that is left.
    auto in_short_list = [&](const bool whole_sum) {
      __syncthreads();
      if (wave == 0) {
        const int m = sh.listed;
        float v_new = V;
        u64 here = 0;
        bool done = false;
        for (int i0 = 0; !done && (i0 == 0 || i0 < m); i0 += 64) {
          const bool in = i0 + lane < m && sh.list[i0 + lane] > V;
          const float v = in ? sh.list[i0 + lane] : 0.0f;
          u64 larger = above, equal = 0, total = above;
          for (int j = 0; j < m; ++j) {
            const float o = sh.list[j];
            const u64 w = !(o > V) ? 0 : MASS ? sh.hist[j] : 1;
            total += w;
            larger += o > v ? w : 0;
            equal += o == v ? w : 0;
          }
          if (MASS && whole_sum) {
            const u64 all = total + ties * v_weight;
            target = max(1ull, min(all, static_cast<u64>(__builtin_ceil(share_p * static_cast<double>(all)))));
          }
          const u64 hit = __ballot(in && larger < target && larger + equal >= target);
          if (hit) {
            const int from = __builtin_ctzll(hit);
            v_new = __shfl(v, from);
            here  = target - __shfl(larger, from);
            if (MASS) {
              const u64 w = whole(weight(v_new));
              here = (here + w - 1) / w;
            }
            done = true;
          } else if (MASS && total < target && total + ties * v_weight >= target) {   // among those that are V already
            here = min(ties, (target - total + v_weight - 1) / max(1ull, v_weight));
            done = true;
          }
        }
        if (lane == 0) {
          sh.found_v    = v_new;
          sh.found_ties = here;
        }
      }
      __syncthreads();
      V    = sh.found_v;
      ties = sh.found_ties;
    };
    auto weigh_list = [&] {
      if (MASS) {
        __syncthreads();
        for (int i = tid; i < sh.listed; i += NT) sh.hist[i] = whole(weight(sh.list[i]));
      }
    };
    if (listed && sh.listed <= SAMPLE_SHORT) {   // (what top-k left; more than one of them)
      weigh_list();
      return in_short_list(true);
    }
    auto clear = [&] {
      __syncthreads();   // (the histogram of before has been read)
      hist[tid] = hist[tid + NT] = 0;
      __syncthreads();
    };
    M last = 0;   // (the first round's last range has the most, and one sum a lane)
    auto first_round = [&](float v, M what) {
      const int b = bin_of(v);
      last += b == BINS - 1 ? what : 0;
      if (b < BINS - 1) atomicAdd(&hist[b], what);
    };
    auto add_last = [&] {
      last = wave_total(last);
      if (lane == 0 && last) atomicAdd(&hist[BINS - 1], last);
    };
    // where the sums over the ranges reach what `want(total)` says (or false: they do not)
    auto find = [&](auto want_of) {
      __syncthreads();
      const u64 first = hist[2 * tid], second = hist[2 * tid + 1];
      u64 upto = wave_scan(first + second);
      if (lane == 63) sh.sum[wave] = upto;
      __syncthreads();
      u64 total = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        if (w == wave) upto += total;
        total += sh.sum[w];
      }
      const u64 want = want_of(total);
      if (total < want) return false;
      if (upto >= want && upto - first - second < want) {
        const bool later = upto - second < want;
        sh.found_bin   = 2 * tid + later;
        sh.found_above = upto - second - (later ? 0 : first);
        sh.found_upto  = upto - (later ? 0 : second);
      }
      __syncthreads();
      return true;
    };
    // all from `least` to `most` (and above V) into the list
    auto gather = [&](const float least, const float most) {
      words.each_word([&](const Word<T> &w, int) {
        float m = w[0];
#pragma unroll
        for (int e = 1; e < N; ++e) m = fmaxf(m, w[e]);
        if (!__any(m >= least)) return;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (w[e] >= least && w[e] <= most && w[e] > V) {   // (few)
            const int at = atomicAdd(&sh.listed, 1);
            if (at < SAMPLE_LIST) sh.list[at] = w[e];
          }
      });
      __syncthreads();
    };
    // (of GRAIN neighbouring keys one is a number of the logits' type)
    constexpr int GRAIN = sizeof(T) == 4 ? 0 : std::is_same<T, bf16>::value ? 16 : 13;
    auto finer = [&] { shift = max(GRAIN, (32 - __builtin_clz((hi - lo) | 1)) - (31 - __builtin_clz(BINS))); };

    int round = 0;
    if constexpr (!MASS) {
      // A rough bound first, from every thread's first word: where as many of those lie as top_k takes of them, and then some. Between top_k
      // and SAMPLE_LIST of all logits are above it nearly always, and nothing else has to be looked at.
      const float share = static_cast<float>(top_k) / words.per;
      const int rough = static_cast<int>(1.3f * share + 4.0f * sqrtf(share)) + 7;
      if (words.per >= 4 && static_cast<long>(rough) * words.per <= SAMPLE_LIST * 3 / 4) {
        clear();
        const int k = words.first;
        if (k < words.words) {
          const Word<T> w = words.at(k);
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (w[e] > -INFINITY) first_round(w[e], 1u);
        }
        last = 0;   // (a bound there would be none)
        if (find([&](u64) { return static_cast<u64>(rough); })) {
          lo = first_in(sh.found_bin);
          hi = key_of(top);
          gather(of_key(lo), top);
          const int m = sh.listed;
          if (m >= top_k && m <= SAMPLE_LIST) {
            in_list = listed = true;
            if (m <= SAMPLE_SHORT) return in_short_list(false);
            finer();
            round = 1;
          } else {
            __syncthreads();
            if (tid == 0) sh.listed = 0;
          }
        }
      }
    }
    for (; round < 6; ++round) {   // (32 bits of logits, 7 or more a round behind the first)
      clear();
      auto later_round = [&](float v, auto what) {
        const uint32_t k = key_of(v);
        if (k >= lo && k <= hi) atomicAdd(&hist[(hi - k) >> shift], what());
      };
      auto one = [&](float v) {
        if constexpr (MASS) {
          if (v > V) {
            if (round) later_round(v, [&] { return whole(weight(v)); }); else first_round(v, whole(weight(v)));
          }
        } else if (v > -INFINITY) {
          if (round) later_round(v, [] { return 1u; }); else first_round(v, 1u);
        }
      };
      if (listed) {
        const int m = sh.listed;
        for (int i = tid; i < m; i += NT) one(sh.list[i]);
      } else if (AHEAD && MASS && round == 0 && !with_k) {
        if constexpr (AHEAD && MASS) {
          const u64 *from = ahead.hist + static_cast<size_t>(row) * BINS;
          hist[tid]      = from[tid];
          hist[tid + NT] = from[tid + NT];
        }
      } else {
        words.each(one);
      }
      if (MASS && ties && tid == 0) {
        if (round) later_round(V, [&] { return ties * v_weight; }); else first_round(V, ties * v_weight);
      }
      if (round == 0) add_last();
      const bool there = find([&](u64 total) {
        if (MASS && round == 0)
          target = max(1ull, min(total, static_cast<u64>(__builtin_ceil(share_p * static_cast<double>(total)))));
        return target - above;
      });
      if (!there) return;   // fewer than top_k (the whole workgroup)
      above += sh.found_above;
      const int b = sh.found_bin;
      if (round == 0) {
        hi = bin_of(top) < b ? first_in(b - 1) - 1 : key_of(top);
        lo = first_in(b);
        // Of top-k all from the maximum on, which is what top-p looks at next; of weights that range alone.
        if (!listed && (MASS || sh.found_upto <= SAMPLE_LIST)) {
          gather(of_key(lo), MASS ? of_key(hi) : top);
          listed = sh.listed <= SAMPLE_LIST;
          if (!MASS) in_list = true;
          if (sh.listed <= SAMPLE_SHORT) {
            if (!MASS) above = 0;
            weigh_list();
            return in_short_list(false);
          }
        }
      } else {
        hi -= static_cast<uint32_t>(b) << shift;
        if (shift == GRAIN) {
          if (GRAIN) {   // positive numbers' keys end in zeros, negative ones' in ones
            const uint32_t down = hi >> GRAIN << GRAIN;
            hi = down & 0x80000000u ? down : ((hi + 1) >> GRAIN << GRAIN) - 1;
          }
          break;
        }
        // (keys of numbers are 2^23 and more, and 512 ranges 2^23 wide at most; of 128 one may be wider than the lowest numbers' keys are large)
        const uint32_t width = (1u << shift) - 1;
        lo = max(lo, BINS >= 512 || hi > width ? hi - width : 0u);
      }
      finer();
    }
    const float before = V;
    V = of_key(hi);
    u64 here = target - above;
    if (MASS) {
      const u64 w = whole(weight(V));
      here = w ? (here + w - 1) / w : 1;
      if (V == before) here = min(here, ties);
    }
    ties = here;
  };
  if (with_k) select(0u);
  if (with_p && in_list && top_k <= SAMPLE_SHORT && sh.listed > SAMPLE_SHORT) {   // what is above V in a short list again
    float mine[SAMPLE_LIST / NT];
    const int m = sh.listed;
#pragma unroll
    for (int i = 0; i < SAMPLE_LIST / NT; ++i) mine[i] = tid + i * NT < m ? sh.list[tid + i * NT] : -INFINITY;
    __syncthreads();
    if (tid == 0) sh.listed = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SAMPLE_LIST / NT; ++i)
      if (mine[i] > V) sh.list[atomicAdd(&sh.listed, 1)] = mine[i];
    __syncthreads();
  }
  if (with_p) select(0ull);
  if (with_q) {
    const double cut = top64 + temperature * log(static_cast<double>(fminf(p.min_p, 1.0f)));
    float f = static_cast<float>(cut);
    if (static_cast<double>(f) < cut) f = of_key(key_of(f) + 1);
    f = fminf(fmaxf(f, -FLT_MAX), top);
    if (f > V) {
      V    = f;
      ties = ~0ull >> 2;
    }
  }

  if constexpr (AHEAD) {   // the rest is other launches'
    if (tid == 0) ahead.bounds[row] = SampleBound{V, ties};
  } else {
    __syncthreads();   // (the histogram has been read)
    const Left mine = weigh_left([&](auto f) { words.each_word([&](const Word<T> &w, int) { f(w); }); }, V, top, weight, a.logp && !set.same,
                                 reinterpret_cast<float *>(sh.hist) + wave * LEFT_QUEUE);
    if (lane == 0) sh.left[wave] = mine;
    __syncthreads();
    draw_token<T, NT>(a, set, weight, top, V, ties, sh.left, WAVES, words.per * 64, words.words, [&](int k) { return words.at(k); }, sh.gt2, sh.ties2);
  }
}

// Logits of a row, and a share of the compute units in rows, from and up to which several workgroups have a row where top-p looks at all of it; twice
// as many logits where the settings are the rows' own and may not ask for that. bf16, one workgroup and several, us:
//   top_p 0.9          33000           66000           100000           131072           200000 logits
//   1 row              48 and 43       76 and 52        96 and 55       101 and  49      110 and  43
//   32 rows            50 and 48       79 and 63        99 and 67       115 and  71      152 and  74
//   64                 51 and 53       79 and 66       100 and 75       115 and  81      152 and  91
//   65                 51 and 53       80 and 67       100 and 75       116 and  85      152 and  94
//   128                51 and 58       80 and 77       100 and 93       116 and 105      154 and 128
//   192                50 and 69       80 and 101      102 and 129      119 and 151      156 and 205
//   top_k 50 in settings of their own, 64 rows         39 and 43 (66000)  46 and 47       51 and  50       68 and  62
// So the rows could be twice as many, and rows with settings of their own as many logits less as top-k is rare among them.
constexpr int SAMPLE_AHEAD_VOCAB = 1 << 16, SAMPLE_AHEAD_SHARE = 4;
constexpr size_t SAMPLE_HELD = 128 << 10;   // bytes of a row that stay in LDS
template <class T>
int launch_sample(const SampleArgs &a, int rows) {
  const int words = static_cast<int>((static_cast<long>(a.vocab) + Word<T>::N - 1) / Word<T>::N), cus = std::max(1, ctx().compute_units);
  const size_t bytes = 16 * static_cast<size_t>(words);
  const bool with_k = a.p.top_k > 0 && a.p.top_k < a.vocab, with_p = a.p.top_p < 1.0f;
  auto go = [&](auto kernel, int nt, size_t lds, auto... more) {
    if (lds > (32 << 10))
      TDH_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SAMPLE_HELD)));
    TDH_LAUNCH(kernel, dim3(rows), dim3(nt), lds, ctx().stream, a, more...);
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  };
  SampleAhead ahead{};
  if (words <= 128) return go(sample_kernel<T, 64, true, false>, 64, bytes, ahead);
  if (words <= 1024) return go(sample_kernel<T, 256, true, false>, 256, bytes, ahead);
  const bool filters = a.settings || !(a.p.temperature > 0.0f) || with_k || with_p || a.p.min_p > 0.0f;
  if (!filters) return rows > 2 * cus ? go(sample_all_kernel<T, 512>, 512, 0) : go(sample_all_kernel<T, 1024>, 1024, 0);
  if (rows <= cus / SAMPLE_AHEAD_SHARE && (a.settings ? a.vocab >= 2 * SAMPLE_AHEAD_VOCAB : with_p && !with_k && a.vocab >= SAMPLE_AHEAD_VOCAB)) {
    ahead.count = std::min({2 * cus / rows, ceil_div(words, AHEAD_NT), AHEAD_MOST});
    ahead.chunk = ceil_div(words, ahead.count);
    const size_t parts = static_cast<size_t>(rows) * ahead.count;
    const size_t sizes[5] = {sizeof(SamplePart) * parts, sizeof(double) * parts, sizeof(u64) * SAMPLE_BINS * rows, sizeof(SampleBound) * rows,
                             sizeof(Left) * parts};
    size_t total = 0;
    for (size_t bytes : sizes) total += ws_align(bytes);
    TDH_TRY(ws_begin(total));
    void *mem[5] = {};
    for (int i = 0; i < 5; ++i) TDH_TRY(ws_take(sizes[i], &mem[i]));
    ahead.parts  = static_cast<SamplePart *>(mem[0]);
    ahead.raw    = static_cast<double *>(mem[1]);
    ahead.hist   = static_cast<u64 *>(mem[2]);
    ahead.bounds = static_cast<SampleBound *>(mem[3]);
    ahead.left   = static_cast<Left *>(mem[4]);
    const dim3 grid(ahead.count, rows);
    TDH_LAUNCH((sample_top_kernel<T>), grid, dim3(AHEAD_NT), 0, ctx().stream, a, ahead);
    TDH_LAUNCH_CHECK();
    TDH_LAUNCH((sample_sums_kernel<T>), grid, dim3(AHEAD_NT), 0, ctx().stream, a, ahead);
    TDH_LAUNCH_CHECK();
    TDH_TRY(go(sample_kernel<T, 1024, false, true>, 1024, 0, ahead));
    TDH_LAUNCH((sample_left_kernel<T>), grid, dim3(AHEAD_NT), 0, ctx().stream, a, ahead);
    TDH_LAUNCH_CHECK();
    return go(sample_draw_kernel<T>, DRAW_NT, 0, ahead);
  }
  if (bytes <= SAMPLE_HELD) return go(sample_kernel<T, 1024, true, false>, 1024, bytes, ahead);
  return go(sample_kernel<T, 1024, false, false>, 1024, 0, ahead);
}

}  // namespace
}  // namespace tdh

using namespace tdh;

extern "C" {

int tdh_sample_tokens(const tdh_sample_desc *p, const tdh_sample_desc *settings, int dtype, int rows, int vocab, const void *logits, size_t ld,
                      const float *u, int32_t *token, float *logp, float *logq, int32_t *kept) {
  const char *who = "tdh_sample_tokens";
  TDH_CHECK_ARG(dtype_known(dtype), "%s: element type %d", who, dtype);
  TDH_CHECK_ARG(rows >= 0 && rows < (1 << 22) && vocab > 0 && vocab <= (1 << 30), "%s: %d rows of %d logits", who, rows, vocab);
  TDH_CHECK_ARG(ld >= static_cast<size_t>(vocab) && ld <= (static_cast<size_t>(1) << 40), "%s: rows of %d logits %zu elements apart", who, vocab, ld);
  TDH_CHECK_ARG(p || settings, "%s: null descriptor", who);
  TDH_CHECK_ARG(rows == 0 || (logits && u && token), "%s: null tensor", who);
  TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(logits) & (dtype_size(dtype) - 1)) == 0, "%s: logits not aligned to their elements", who);
  const uintptr_t four = reinterpret_cast<uintptr_t>(settings) | reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(token) |
                         reinterpret_cast<uintptr_t>(logp) | reinterpret_cast<uintptr_t>(logq) | reinterpret_cast<uintptr_t>(kept);
  TDH_CHECK_ARG((four & 3) == 0, "%s: a tensor that is not aligned to its elements", who);
  if (!settings) {
    TDH_CHECK_ARG(p->temperature >= 0.0f && p->temperature <= FLT_MAX, "%s: temperature %g", who, p->temperature);
    TDH_CHECK_ARG(p->top_k >= 0, "%s: top_k %d", who, p->top_k);
    TDH_CHECK_ARG(p->top_p > 0.0f && p->top_p <= 1.0f, "%s: top_p %g", who, p->top_p);
    TDH_CHECK_ARG(p->min_p >= 0.0f && p->min_p <= 1.0f, "%s: min_p %g", who, p->min_p);
  }
  const size_t r4 = 4 * static_cast<size_t>(rows);
  const Span in{logits, rows > 0 ? dtype_size(dtype) * ((rows - 1) * ld + vocab) : 0};
  TDH_TRY(check_apart(who, {{token, r4}, {logp, r4}, {logq, r4}, {kept, r4}}, {in, {u, r4}, {settings, 4 * r4}}));
  TDH_REQUIRE_INIT();
  if (rows == 0) return TDH_OK;
  SampleArgs a{};
  a.logits = logits; a.ld = ld; a.u = u; a.settings = settings;
  if (p) a.p = *p;
  a.vocab = vocab;
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  a.fix = std::min(50, 62 - bits);
  a.token = token; a.kept = kept; a.logp = logp; a.logq = logq;
  ProfScope prof("sample_tokens", static_cast<double>(dtype_size(dtype)) * rows * vocab, WORK_BYTE);
  return with_dtype(dtype, [&](auto t) { return launch_sample<decltype(t)>(a, rows); });
}

}  // extern "C"
