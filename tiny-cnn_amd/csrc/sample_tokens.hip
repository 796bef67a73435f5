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
// A workgroup has a row, whose words stay in its registers (of up to 16384 words, else they are read in every pass). Bound by the exponentials in
// 64 bits, some 20 instructions a logit that counts, and by the latency of a chain of passes on one compute unit.
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

// 2^t for t <= 0, to 4e-14 of the value: the fit is of (2^f - 1) / f for |f| <= 1/2 (Chebyshev nodes), so that 2^0 is 1
__device__ __forceinline__ double exp2_64(double t) {
  t = __builtin_fmax(t, -1000.0);   // (and where t is 0 times an infinity: nothing)
  const double n = __builtin_rint(t), f = t - n;
  double p = 1.0203121063391729e-07;
  p = __builtin_fma(p, f, 1.3255224878668817e-06);
  p = __builtin_fma(p, f, 1.525268684626772e-05);
  p = __builtin_fma(p, f, 0.00015403455852453838);
  p = __builtin_fma(p, f, 0.0013333558179043112);
  p = __builtin_fma(p, f, 0.009618129159402558);
  p = __builtin_fma(p, f, 0.055504108664760424);
  p = __builtin_fma(p, f, 0.2402265069581299);
  p = __builtin_fma(p, f, 0.6931471805599453);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, static_cast<int>(n));
}
constexpr double LOG2E_64 = 1.4426950408889634;

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

// LDS of a row's workgroup
template <int NT>
struct SampleShared {
  static constexpr int WAVES = NT / 64, BINS = 2 * NT;
  u64 hist[BINS];   // (counts: the first half of it)
  u64 sum[WAVES];
  u64 found_above;
  int found_bin;
  float top[WAVES], far[WAVES];
  int bad[WAVES], n[WAVES];
  // what is left, wave by wave: weight and number above V, number with V; weights below the maximum in floating point, number of maxima
  u64 gt[WAVES], gt2[WAVES];
  int gt_n[WAVES], ties[WAVES], ties2[WAVES], tops[WAVES];
  double rest[WAVES], raw[WAVES];
};

// W words a thread, each wave's behind each other (W = 0: any number, read in every pass)
template <class T, int NT, int W>
__global__ void __launch_bounds__(NT)
sample_kernel(const SampleArgs a) {
  using Shared = SampleShared<NT>;
  constexpr int WAVES = Shared::WAVES, BINS = Shared::BINS, N = Word<T>::N;
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x, vocab = a.vocab;
  const T *x = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * a.ld;
  const int words = (vocab + N - 1) / N, per = (words + NT - 1) / NT;   // words a thread
  const int first_word = wave * per * 64 + lane;
  auto load = [&](int k) { return row_word(x, k, vocab, -INFINITY); };
  Word<T> held[W ? W : 1];
  if constexpr (W > 0) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < per && first_word + 64 * i < words) held[i] = load(first_word + 64 * i);
  }
  // f(logit) of every logit that this thread has
  auto each = [&](auto f) {
    if constexpr (W > 0) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        // (a word at a time: left alone the compiler keeps what it unpacks from one pass to the next, and spills)
        asm volatile("" : "+v"(held[i].raw.x), "+v"(held[i].raw.y), "+v"(held[i].raw.z), "+v"(held[i].raw.w));
        if (i < per && first_word + 64 * i < words)
#pragma unroll
          for (int e = 0; e < N; ++e) f(held[i][e]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      for (int i = 0; i < per && first_word + 64 * i < words; ++i) {
        const Word<T> w = load(first_word + 64 * i);
#pragma unroll
        for (int e = 0; e < N; ++e) f(w[e]);
      }
    }
  };

  // the row's settings
  const tdh_sample_desc p = a.settings ? a.settings[row] : a.p;
  const bool greedy = !(p.temperature > 0.0f);
  const double temperature = greedy ? 1.0 : static_cast<double>(p.temperature), rate = LOG2E_64 / temperature;
  const int top_k = greedy ? 1 : p.top_k;
  const bool with_k = top_k > 0 && top_k < vocab, with_p = !greedy && p.top_p < 1.0f, with_q = !greedy && p.min_p > 0.0f;

  // maximum, and how far the others lie from it on average
  float top = -INFINITY, far = 0.0f;
  int bad = 0, n = 0;
  each([&](float v) {
    top = fmaxf(top, v);
    bad |= !(v < INFINITY);
  });
  if (with_k || with_p)
    each([&](float v) {
      far += v > -INFINITY ? v : 0.0f;
      n += v > -INFINITY;
    });
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  far = wave_total(far);
  n   = wave_total(n);
  bad = __any(bad);
  if (lane == 0) {
    sh.top[wave] = top;
    sh.far[wave] = far;
    sh.bad[wave] = bad;
    sh.n[wave]   = n;
  }
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
  if (bad || top == -INFINITY) {   // (the whole workgroup)
    if (tid == 0) {
      a.token[row] = -1;
      if (a.kept) a.kept[row] = 0;
      if (a.logp) a.logp[row] = __builtin_nanf("");
      if (a.logq) a.logq[row] = __builtin_nanf("");
    }
    return;
  }
  const double top64 = top, unit = __builtin_ldexp(1.0, a.fix);
  auto weight = [&](float v) { return exp2_64((static_cast<double>(v) - top64) * rate); };
  constexpr double SHIFT = 4503599627370496.0;   // 2^52: the sum's low bits are the rounded product
  auto whole = [&](double w) { return __builtin_bit_cast(u64, __builtin_fma(w, unit, SHIFT)) - __builtin_bit_cast(u64, SHIFT); };

  // What is left: logits above V, and the first `ties` of those that are V
  float V  = -INFINITY;
  u64 ties = 0;

  // The logit at which the sum over what is left, from the largest logit on, reaches a target: top_k (counts) or the share top_p of
  // all (weights). V becomes that logit and ties what is missing there.
  auto select = [&](auto zero) {
    using M = decltype(zero);
    constexpr bool MASS = sizeof(M) == 8;
    M *hist = reinterpret_cast<M *>(sh.hist);
    const float mean = top - far / static_cast<float>(n), scale = mean > 0.0f ? BINS / (4.0f * mean) : 0.0f;
    // the first round's ranges: equal ones of the distance from the maximum, the last for what is beyond four times the average
    auto bin_of = [&](float v) { return static_cast<int>(fminf((top - v) * scale, static_cast<float>(BINS - 1))); };
    const u64 v_weight = MASS ? whole(weight(V)) : 0;
    u64 above = 0, target = MASS ? 0 : static_cast<u64>(top_k);
    int bin = 0, shift = 0;
    uint32_t lo = 0, hi = 0;
    for (int round = 0; round < 6; ++round) {   // (32 bits of logits, 7 or more a round behind the first)
      __syncthreads();   // (the histogram of before has been read)
      hist[tid] = hist[tid + NT] = 0;
      __syncthreads();
      M last = 0;   // (the first round's last range has the most, and one sum a lane)
      auto add = [&](float v, M what) {
        if (round == 0) {
          const int b = bin_of(v);
          if (b == BINS - 1)
            last += what;
          else
            atomicAdd(&hist[b], what);
        } else {
          const uint32_t k = key_of(v);
          if (k >= lo && k <= hi && bin_of(v) == bin) atomicAdd(&hist[(hi - k) >> shift], what);
        }
      };
      if constexpr (MASS) {
        const float from = round ? of_key(lo) : V;
        each([&](float v) {
          if (v > V && v >= from) add(v, whole(weight(v)));
        });
        if (ties && tid == 0) add(V, ties * v_weight);
      } else {
        each([&](float v) {
          if (v > -INFINITY) add(v, 1);
        });
      }
      if (round == 0) {
        last = wave_total(last);
        if (lane == 0 && last) atomicAdd(&hist[BINS - 1], last);
      }
      __syncthreads();
      const u64 one = hist[2 * tid], two = hist[2 * tid + 1];
      u64 upto = wave_scan(one + two);
      if (lane == 63) sh.sum[wave] = upto;
      __syncthreads();
      u64 total = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        if (w == wave) upto += total;
        total += sh.sum[w];
      }
      if (round == 0) {
        if (MASS) target = max(1ull, min(total, static_cast<u64>(__builtin_ceil(static_cast<double>(p.top_p) * static_cast<double>(total)))));
        if (total < target) return;   // fewer than top_k (the whole workgroup)
      }
      const u64 want = target - above;
      if (upto >= want && upto - one - two < want) {
        const bool second = upto - two < want;
        sh.found_bin   = 2 * tid + second;
        sh.found_above = above + upto - two - (second ? 0 : one);
      }
      __syncthreads();
      above = sh.found_above;
      const int b = sh.found_bin;
      if (round == 0) {
        bin = b;
        // the logits of that range lie between these (and other ranges' beside it)
        const double s = scale, x1 = top64 - b * 0.999999 / s, x0 = top64 - (b + 1) * 1.000001 / s;
        hi = scale > 0.0f ? key_of(static_cast<float>(x1 + 1e-6 * __builtin_fabs(x1) + 1e-37)) : key_of(top);
        lo = scale > 0.0f && b < BINS - 1 ? key_of(__builtin_fmaxf(static_cast<float>(x0 - 1e-6 * __builtin_fabs(x0) - 1e-37), -FLT_MAX)) : key_of(-FLT_MAX);
        hi = min(hi, key_of(top));
      } else {
        hi -= static_cast<uint32_t>(b) << shift;
        if (shift == 0) break;
        lo = max(lo, hi - ((1u << shift) - 1));
      }
      shift = max(0, (32 - __builtin_clz((hi - lo) | 1)) - (31 - __builtin_clz(BINS)));
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

  // the weights that are left, wave by wave
  const double v_weight64 = weight(V);
  const u64 v_weight = whole(v_weight64);
  {
    u64 gt = 0;
    int gt_n = 0, at = 0, tops = 0;
    double rest = 0.0, raw = 0.0;
    each([&](float v) {
      if (v > V) {
        const double w = weight(v);
        gt += whole(w);
        ++gt_n;
        rest += v < top ? w : 0.0;
      }
      at += v == V;
      tops += v == top;
    });
    const bool same = a.logp && !(with_k || with_p || with_q) && temperature == 1.0;
    if (a.logp && !same) {
      // exp(v - top) in fp32, the product with log2(e) with its rounding
      each([&](float v) {
        const float d = fmaxf(v - top, -200.0f), t = d * 1.44269504f, r = __builtin_fmaf(d, 1.44269504f, -t) + d * 1.925963033e-8f;
        const float e = __builtin_amdgcn_exp2f(t);
        raw += v < top && v > -INFINITY ? static_cast<double>(__builtin_fmaf(e, 0.69314718f * r, e)) : 0.0;
      });
    }
    gt   = wave_total(gt);
    gt_n = wave_total(gt_n);
    at   = wave_total(at);
    tops = wave_total(tops);
    rest = wave_total(rest);
    raw  = wave_total(same ? rest : raw);
    if (lane == 0) {
      sh.gt[wave]   = gt;
      sh.gt_n[wave] = gt_n;
      sh.ties[wave] = at;
      sh.tops[wave] = tops;
      sh.rest[wave] = rest;
      sh.raw[wave]  = same ? rest : raw;
    }
  }
  __syncthreads();
  u64 gt_all = 0, ties_all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    gt_all += sh.gt[w];
    ties_all += sh.ties[w];
  }
  const u64 ties_left = min(ties, ties_all), all = gt_all + v_weight * ties_left;
  const double u = a.u[row];
  u64 r = static_cast<u64>((u > 0.0 ? fmin(u, 1.0) : 0.0) * static_cast<double>(all));
  r = min(r, all - 1);
  // the weights left up to a place with `g` above V and `t` with V in front of it
  auto upto = [&](u64 g, u64 t) { return g + v_weight * min(t, ties_left); };
  u64 g0 = 0, t0 = 0;
  int where = 0;
#pragma unroll 1
  for (; where < WAVES - 1; ++where) {
    const u64 g1 = g0 + sh.gt[where], t1 = t0 + sh.ties[where];
    if (upto(g1, t1) > r) break;
    g0 = g1;
    t0 = t1;
  }
  // that wave's words, a share for every thread
  const int share = (per * 64 + NT - 1) / NT, beg = where * per * 64 + tid * share, end = min(min(beg + share, (where + 1) * per * 64), words);
  u64 gt = 0;
  int at = 0;
  for (int k = beg; k < end; ++k) {
    const Word<T> w = load(k);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (w[e] > V) gt += whole(weight(w[e]));
      at += w[e] == V;
    }
  }
  const u64 gt_scan = wave_scan(gt);
  const int at_scan = wave_scan(at);
  if (lane == 63) {
    sh.gt2[wave]   = gt_scan;
    sh.ties2[wave] = at_scan;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    if (w < wave) {
      g0 += sh.gt2[w];
      t0 += sh.ties2[w];
    }
  g0 += gt_scan - gt;
  t0 += at_scan - at;
  if (upto(g0, t0) > r || upto(g0 + gt, t0 + at) <= r) return;
  // one thread is left
  int token = -1;
  float chosen = V;
  for (int k = beg; k < end && token < 0; ++k) {
#pragma unroll 1
    for (int e = 0; e < N && token < 0; ++e) {
      const float v = to_f32(x[min(k * N + e, vocab - 1)]);
      if (k * N + e >= vocab || v < V) continue;
      if (v > V) g0 += whole(weight(v)); else ++t0;
      if (upto(g0, t0) > r) {
        token  = k * N + e;
        chosen = v;
      }
    }
  }
  a.token[row] = token;
  u64 gt_count = 0;
  int tops = 0;
  double rest = 0.0, raw = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    gt_count += sh.gt_n[w];
    tops += sh.tops[w];
    rest += sh.rest[w];
    raw += sh.raw[w];
  }
  if (a.kept) a.kept[row] = static_cast<int>(gt_count + ties_left);
  const double d = static_cast<double>(chosen) - top64;
  // (a single maximum: the logarithm of 1 + rest has rest's precision)
  auto log_of = [](double tops, double rest) { return tops == 1.0 ? log1p(rest) : log(tops + rest); };
  if (a.logq) a.logq[row] = static_cast<float>(V == top ? -log(static_cast<double>(ties_left))
                                                        : d / temperature - log_of(tops, rest + v_weight64 * static_cast<double>(ties_left)));
  if (a.logp) a.logp[row] = static_cast<float>(d - log_of(tops, raw));
}

template <class T>
int launch_sample(const SampleArgs &a, int rows) {
  const int words = static_cast<int>((static_cast<long>(a.vocab) + Word<T>::N - 1) / Word<T>::N);
  auto go = [&](auto kernel, int nt) {
    TDH_LAUNCH(kernel, dim3(rows), dim3(nt), 0, ctx().stream, a);
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  };
  if (words <= 64) return go(sample_kernel<T, 64, 1>, 64);
  if (words <= 512) return go(sample_kernel<T, 256, 2>, 256);
  if (words <= 1024) return go(sample_kernel<T, 1024, 1>, 1024);
  if (words <= 4096) return go(sample_kernel<T, 1024, 4>, 1024);
  if (words <= 8192) return go(sample_kernel<T, 1024, 8>, 1024);
  if (words <= 16384) return go(sample_kernel<T, 1024, 16>, 1024);
  return go(sample_kernel<T, 1024, 0>, 1024);
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
