// layernorm.hip — layer normalisation of rows, and its gradients.
//
//   mean = sum x / n, rstd = 1 / sqrt(sum (x - mean)^2 / n + eps), xhat = (x - mean) rstd, y = xhat gamma + beta
//   g = dy gamma, dx = rstd (g - sum g / n - xhat sum(g xhat) / n), dgamma = sum over rows of dy xhat, dbeta = sum over rows of dy
//
// A row stays in the registers of the lanes that have it, so each direction reads its tensors once; the backward pass adds up the
// gradients of gamma and beta on the way, every thread for the columns that it has in all of its rows. Sums are fp32. What rounding takes
// from the mean (a row far from zero) is put back from the sum of the deviations: with d = x - mean as computed and e = sum d / n, the
// deviations are d - e and their mean square is sum d^2 / n - e^2.
#include "lm_types.h"

#include <cfloat>

namespace tdh {

namespace {

struct NormFwdArgs {
  const void *x, *gamma, *beta;
  void *y;
  float *stats;
  size_t ld, ld_y;
  int rows, len;
  float eps, inv_len;
};
struct NormBwdArgs {
  const void *x, *gamma, *dy;
  const float *stats;
  void *dx;
  size_t ld, ld_dy, ld_dx;
  int rows, len;
  float inv_len;
  float *partial;        // [workgroups][2][len]: the gradients of gamma and beta (null: nobody wants them), or, of one workgroup,
  void *dgamma, *dbeta;  // the gradients themselves
  int accumulate;
};

// Sums over the LANES lanes that have a row (a power of two; more than a wave: LANES / 64 whole waves, through LDS). `turn` tells two
// calls behind each other apart, which need no barrier between them then; every thread of the workgroup calls.
template <int LANES, int K, int NT>
struct GroupSum {
  static constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
  float part[WAVES > 1 ? 2 : 1][WAVES > 1 ? NT / 64 : 1][K];
  __device__ __forceinline__ void operator()(float (&v)[K], const int turn) {
#pragma unroll
    for (int o = (LANES < 64 ? LANES : 64) / 2; o; o >>= 1)
#pragma unroll
      for (int i = 0; i < K; ++i) v[i] += __shfl_xor(v[i], o);
    if constexpr (WAVES > 1) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < K; ++i) part[turn & 1][wave][i] = v[i];
      __syncthreads();
      const int first = wave / WAVES * WAVES;
#pragma unroll
      for (int i = 0; i < K; ++i) {
        v[i] = part[turn & 1][first][i];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v[i] += part[turn & 1][first + w][i];
      }
    }
  }
};

// LANES lanes a row, W words a lane. W = 0: any number of words, the row is read three times.
template <class T, int LANES, int W, bool ONCE>
__global__ void __launch_bounds__(LANES > 256 ? LANES : 256)
layernorm_fwd_kernel(const NormFwdArgs a) {
  constexpr int NT = LANES > 256 ? LANES : 256, ROWS = NT / LANES, N = Word<T>::N;
  __shared__ GroupSum<LANES, 2, NT> sum;
  const int lane = threadIdx.x % LANES, words = (a.len + N - 1) / N;
  const T *gamma = static_cast<const T *>(a.gamma), *beta = static_cast<const T *>(a.beta);
  int turn = 0;
  for (long first = static_cast<long>(blockIdx.x) * ROWS; first < a.rows; first += static_cast<long>(gridDim.x) * ROWS) {
    const long row  = first + threadIdx.x / LANES;
    const bool live = row < a.rows;   // (the others take part in the sums)
    const T *x      = static_cast<const T *>(a.x) + (live ? row : 0) * a.ld;
    Word<T> held[W ? W : 1];
    // f(word index, word) of every word that this lane has
    auto each = [&](const float rest, auto f) {
      if constexpr (W > 0) {
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (lane + i * LANES < words) f(lane + i * LANES, held[i]);
      } else {
        for (int k = lane; k < words; k += LANES) f(k, row_word(x, k, a.len, rest));
      }
    };
    if constexpr (W > 0) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (lane + i * LANES < words) held[i] = row_word(x, lane + i * LANES, a.len, 0.0f);
    }
    float s[2] = {0.0f, 0.0f};
    each(0.0f, [&](int, const Word<T> &w) {
#pragma unroll
      for (int e = 0; e < N; ++e) s[0] += w[e];
    });
    sum(s, turn++);
    float mean = s[0] * a.inv_len;
    s[0] = s[1] = 0.0f;
    each(0.0f, [&](int k, const Word<T> &w) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = k * N + e < a.len ? w[e] - mean : 0.0f;
        s[0] += d;
        s[1] = __builtin_fmaf(d, d, s[1]);
      }
    });
    sum(s, turn++);
    float off = s[0] * a.inv_len, var = s[1] * a.inv_len - off * off;
    // Beyond fp32: the sum of the values, or the squares of what the mean's rounding makes of the deviations. Then every element's share of the mean is added up, and
    // the mean taken nearer (a sum of 2^24 terms is off by 1e-3 of them at most, so four times do from any start); the squares are those of d - e. By all
    // lanes of a row or none of them, from memory, so that nothing of it takes registers from the others.
    if (__builtin_expect(!(var <= FLT_MAX), 0)) {
      mean = __builtin_fabsf(mean) <= FLT_MAX ? mean : 0.0f;
      off  = 0.0f;
#pragma unroll 1
      for (int pass = 0; pass < 6; ++pass) {   // four times the mean, once what it is still off by, the squares
        s[0] = s[1] = 0.0f;
#pragma unroll 1
        for (int k = lane; k < words; k += LANES) {
          const Word<T> w = row_word(x, k, a.len, 0.0f);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float d = k * N + e < a.len ? (w[e] - mean) - off : 0.0f;
            s[0] += d * (0.5f * a.inv_len);
            s[1] = __builtin_fmaf(d, d, s[1]);
          }
        }
        sum(s, turn++);
        if (pass < 4)
          mean = __builtin_amdgcn_fmed3f(mean + 2.0f * s[0], -FLT_MAX, FLT_MAX);
        else if (pass < 5)
          off = 2.0f * s[0];
        else
          var = s[1] * a.inv_len;
      }
    }
    const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + a.eps);
    if (!live) continue;
    if (a.stats && lane == 0) {
      a.stats[2 * row]     = mean + off;
      a.stats[2 * row + 1] = rstd;
    }
    T *y = static_cast<T *>(a.y) + row * a.ld_y;
    each(0.0f, [&](int k, const Word<T> &w) {
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = ((w[e] - mean) - off) * rstd;
      if (gamma) {
        const Word<T> g = row_word(gamma, k, a.len, 0.0f);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= g[e];
      }
      if (beta) {
        const Word<T> b = row_word(beta, k, a.len, 0.0f);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] += b[e];
      }
      put_row_word<T, ONCE>(y, k, a.len, v);
    });
  }
}

// out (+)= v
template <class T>
__device__ __forceinline__ void leave(void *out, const int c, const float v, const int accumulate) {
  T *p = static_cast<T *>(out);
  if (p) p[c] = from_f32<T>(accumulate ? v + to_f32(p[c]) : v);
}

// Backward, LANES lanes a row, W words a lane, 512 / LANES rows of a workgroup at a time, the next ones on their way meanwhile.
constexpr int NB_NT = 512;
template <class T, int LANES, int W, bool ONCE>
__global__ void __launch_bounds__(NB_NT)
layernorm_bwd_kernel(const NormBwdArgs a) {
  constexpr int ROWS = NB_NT / LANES, N = Word<T>::N, E = W * N, COLS = LANES * E;
  // a wave's lanes that have the same columns are added up by shuffles, so LDS holds a set of columns for every wave or group of waves
  constexpr int SETS = LANES < 64 ? NB_NT / 64 : ROWS;
  __shared__ GroupSum<LANES, 3, NB_NT> sum;
  __shared__ float sets[SETS * COLS];
  const int tid = threadIdx.x, lane = tid % LANES, words = (a.len + N - 1) / N;
  Word<T> gamma[W];
  float dg[E] = {}, db[E] = {};
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int k = lane + i * LANES;
    if (a.gamma && k < words) {
      gamma[i] = row_word(static_cast<const T *>(a.gamma), k, a.len, 0.0f);
    } else {
      float one[N];
#pragma unroll
      for (int e = 0; e < N; ++e) one[e] = 1.0f;
      gamma[i] = Word<T>::from(one);
    }
  }
  Word<T> x[W], dy[W];
  float mean = 0.0f, rstd = 0.0f;
  // (what is not there is zero in dy, and adds nothing)
  auto fetch = [&](const long row) {
    const bool live = row < a.rows;
    const long r    = live ? row : 0;
    mean = live ? a.stats[2 * r] : 0.0f;
    rstd = live ? a.stats[2 * r + 1] : 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int k = lane + i * LANES;
      x[i].raw = dy[i].raw = make_uint4(0, 0, 0, 0);
      if (live && k < words) {
        x[i]  = row_word(static_cast<const T *>(a.x) + r * a.ld, k, a.len, 0.0f);
        dy[i] = row_word(static_cast<const T *>(a.dy) + r * a.ld_dy, k, a.len, 0.0f);
      }
    }
  };
  const long step = static_cast<long>(gridDim.x) * ROWS;
  int turn = 0;
  fetch(static_cast<long>(blockIdx.x) * ROWS + tid / LANES);
  for (long first = static_cast<long>(blockIdx.x) * ROWS; first < a.rows; first += step) {
    const long row = first + tid / LANES;
    const float m = mean, rs = rstd;
    Word<T> xw[W], dw[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      xw[i] = x[i];
      dw[i] = dy[i];
    }
    if (first + step < a.rows) fetch(row + step);
    float s[3] = {0.0f, 0.0f, 0.0f};   // of d, g and g d
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const bool in = (lane + i * LANES) * N + e < a.len;
        const float d = in ? xw[i][e] - m : 0.0f, g = dw[i][e] * gamma[i][e];
        s[0] += d;
        s[1] += g;
        s[2] = __builtin_fmaf(g, d, s[2]);
      }
    sum(s, turn++);
    const float off = s[0] * a.inv_len, c1 = s[1] * a.inv_len, c2 = (s[2] * a.inv_len - off * c1) * rs;
    const bool live = row < a.rows;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int k = lane + i * LANES;
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float xhat = ((xw[i][e] - m) - off) * rs, d = dw[i][e];
        db[i * N + e] += d;
        dg[i * N + e] = __builtin_fmaf(d, xhat, dg[i * N + e]);
        v[e] = rs * ((d * gamma[i][e] - c1) - xhat * c2);
      }
      if (a.dx && live && k < words) put_row_word<T, ONCE>(static_cast<T *>(a.dx) + row * a.ld_dx, k, a.len, v);
    }
  }
  if (!a.partial && !a.dgamma && !a.dbeta) return;
  // the sets of columns together, first gamma's, then beta's
  auto join = [&](float (&v)[E], float *partial, void *out) {
#pragma unroll
    for (int o = LANES; o < 64; o <<= 1)
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] += __shfl_xor(v[e], o);
    const int set = LANES < 64 ? tid / 64 : tid / LANES;
    __syncthreads();
    if (LANES >= 64 || (tid & 63) < LANES) {
#pragma unroll
      for (int i = 0; i < W; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) sets[set * COLS + (lane + i * LANES) * N + e] = v[i * N + e];
    }
    __syncthreads();
    for (int c = tid; c < a.len; c += NB_NT) {
      float t = sets[c];
#pragma unroll
      for (int q = 1; q < SETS; ++q) t += sets[q * COLS + c];
      if (a.partial)
        partial[c] = t;
      else
        leave<T>(out, c, t, a.accumulate);
    }
  };
  float *p = a.partial ? a.partial + static_cast<size_t>(blockIdx.x) * 2 * a.len : nullptr;
  join(dg, p, a.dgamma);
  join(db, p + a.len, a.dbeta);
}

// Rows that a workgroup does not hold: the three sums of every row first, which give (off, sum g / n, sum(g xhat) / n) ...
constexpr int NS_NT = 1024;
template <class T>
__global__ void __launch_bounds__(NS_NT)
layernorm_long_sums_kernel(const NormBwdArgs a, float *__restrict__ out) {
  constexpr int N = Word<T>::N;
  __shared__ GroupSum<NS_NT, 3, NS_NT> sum;
  const int tid = threadIdx.x, words = (a.len + N - 1) / N;
  const T *gamma = static_cast<const T *>(a.gamma);
  int turn = 0;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.ld, *dy = static_cast<const T *>(a.dy) + row * a.ld_dy;
    const float m = a.stats[2 * row], rs = a.stats[2 * row + 1];
    float s[3] = {0.0f, 0.0f, 0.0f};
    for (int k = tid; k < words; k += NS_NT) {
      const Word<T> xw = row_word(x, k, a.len, 0.0f), dw = row_word(dy, k, a.len, 0.0f);
      Word<T> gw = dw;
      if (gamma) gw = row_word(gamma, k, a.len, 0.0f);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = k * N + e < a.len ? xw[e] - m : 0.0f, g = gamma ? dw[e] * gw[e] : dw[e];
        s[0] += d;
        s[1] += g;
        s[2] = __builtin_fmaf(g, d, s[2]);
      }
    }
    sum(s, turn++);
    if (tid == 0) {
      const float off = s[0] * a.inv_len, c1 = s[1] * a.inv_len;
      out[3 * row]     = off;
      out[3 * row + 1] = c1;
      out[3 * row + 2] = (s[2] * a.inv_len - off * c1) * rs;
    }
  }
}
// ... and then everything else, a thread a word of the columns, down a band of `band` rows.
constexpr int NL_NT = 256;
template <class T>
__global__ void __launch_bounds__(NL_NT)
layernorm_long_bwd_kernel(const NormBwdArgs a, const float *__restrict__ sums, const int band) {
  constexpr int N = Word<T>::N;
  const int k = blockIdx.x * NL_NT + threadIdx.x;
  if (k * N >= a.len) return;
  const long beg = static_cast<long>(blockIdx.y) * band, end = min(static_cast<long>(a.rows), beg + band);
  Word<T> gamma{};
  if (a.gamma) gamma = row_word(static_cast<const T *>(a.gamma), k, a.len, 0.0f);
  float dg[N] = {}, db[N] = {};
  for (long row = beg; row < end; ++row) {
    const Word<T> x = row_word(static_cast<const T *>(a.x) + row * a.ld, k, a.len, 0.0f);
    const Word<T> dy = row_word(static_cast<const T *>(a.dy) + row * a.ld_dy, k, a.len, 0.0f);
    const float m = a.stats[2 * row], rs = a.stats[2 * row + 1], off = sums[3 * row], c1 = sums[3 * row + 1], c2 = sums[3 * row + 2];
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float xhat = ((x[e] - m) - off) * rs, d = dy[e];
      db[e] += d;
      dg[e] = __builtin_fmaf(d, xhat, dg[e]);
      v[e]  = rs * (((a.gamma ? d * gamma[e] : d) - c1) - xhat * c2);
    }
    if (a.dx) put_row_word(static_cast<T *>(a.dx) + row * a.ld_dx, k, a.len, v);
  }
  if (!a.partial) return;
  float *p = a.partial + static_cast<size_t>(blockIdx.y) * 2 * a.len;
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (k * N + e < a.len) {
      p[k * N + e]         = dg[e];
      p[a.len + k * N + e] = db[e];
    }
}

// The gradients of gamma and beta from `parts` partial sums, in an order that their number sets: a workgroup 32 columns, of which every
// thread adds up each 32nd part.
constexpr int NS_COLS = 32, NS_GROUPS = 32;
template <class T>
__global__ void __launch_bounds__(NS_COLS * NS_GROUPS)
layernorm_sum_kernel(const float *__restrict__ partial, const int parts, const int len, void *dgamma, void *dbeta, const int accumulate) {
  __shared__ float lds[NS_GROUPS][NS_COLS + 1];
  const int c = threadIdx.x % NS_COLS, g = threadIdx.x / NS_COLS;
  const long col = static_cast<long>(blockIdx.x) * NS_COLS + c;   // of [gamma's, beta's]
  float s = 0.0f;
  if (col < 2L * len)
    for (int p = g; p < parts; p += NS_GROUPS) s += partial[static_cast<size_t>(p) * 2 * len + col];
  lds[g][c] = s;
  __syncthreads();
  if (g || col >= 2L * len) return;
#pragma unroll
  for (int q = 1; q < NS_GROUPS; ++q) s += lds[q][c];
  if (col < len)
    leave<T>(dgamma, static_cast<int>(col), s, accumulate);
  else
    leave<T>(dbeta, static_cast<int>(col - len), s, accumulate);
}

// ------------------------------------------------------------------ launches
// Results that the L2 caches do not hold go past them: 8192 x 4096 in bf16 forward 37.7 us through them, 30.6 past them; 4096 x 4096 in fp32 34.5
// and 25.9.
// So 8192 x 4096 in bf16 goes forward at 4.4 TB/s and back, 40 us and 4.1 for the sums of its partial gradients, at 5.0: bound by memory. Not kept, us: the
// backward pass of two workgroups a compute unit without rows ahead 54.6 (one with the next row ahead 40), with two rows ahead 44.8, reads past
// the caches 34.5 forward, 256 lanes a row 39.6 forward.
constexpr double NORM_ONCE_BYTES = 32 << 20;
constexpr int NORM_HELD = 8192;   // elements of a row that a workgroup of the backward pass holds

template <class T>
int launch_norm_fwd(const NormFwdArgs &a) {
  const int words = ceil_div(a.len, Word<T>::N), cus = std::max(1, ctx().compute_units);
  const bool once = static_cast<double>(sizeof(T)) * a.rows * a.len > NORM_ONCE_BYTES;
  auto go = [&](auto l, auto w) {
    constexpr int LANES = decltype(l)::value, W = decltype(w)::value, NT = LANES > 256 ? LANES : 256;
    const dim3 grid(std::min(ceil_div(a.rows, NT / LANES), 64 * cus));
    if (once)
      TDH_LAUNCH((layernorm_fwd_kernel<T, LANES, W, true>), grid, dim3(NT), 0, ctx().stream, a);
    else
      TDH_LAUNCH((layernorm_fwd_kernel<T, LANES, W, false>), grid, dim3(NT), 0, ctx().stream, a);
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  };
  if (words <= 8) return go(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
  if (words <= 32) return go(std::integral_constant<int, 32>(), std::integral_constant<int, 1>());
  if (words <= 64) return go(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
  if (words <= 128) return go(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
  // fewer rows than there are compute units: as many lanes for each as it has words
  if (a.rows > 4 * cus && words <= 256) return go(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
  if (a.rows > 4 * cus && words <= 512) return go(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
  if (words <= 256) return go(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
  if (words <= 1024) return go(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
  if (words <= 2048) return go(std::integral_constant<int, 256>(), std::integral_constant<int, 8>());
  if (words <= 8192) return go(std::integral_constant<int, 1024>(), std::integral_constant<int, 8>());
  return go(std::integral_constant<int, 1024>(), std::integral_constant<int, 0>());
}

// how the backward pass is laid out: lanes of a row (0: the long rows' kernels), workgroups or bands
struct NormBwdPlan {
  int lanes, parts, band;
};
NormBwdPlan norm_bwd_plan(int rows, int len) {
  const int cus = std::max(1, ctx().compute_units);
  NormBwdPlan p{};
  if (len > NORM_HELD) {
    // bands of rows until the chip is full or a band is down to eight
    const int strips = ceil_div(len, NL_NT * 4), want = std::max(1, 8 * cus / strips);
    p.band  = std::max(8, ceil_div(rows, want));
    p.parts = ceil_div(rows, p.band);
    return p;
  }
  p.lanes = len <= 64 ? 8 : len <= 256 ? 32 : len <= 1024 ? 64 : len <= 2048 ? 128 : len <= 4096 ? 256 : 512;
  p.parts = std::min(ceil_div(rows, NB_NT / p.lanes), cus);
  return p;
}
size_t norm_bwd_bytes(const NormBwdPlan &p, int rows, int len, bool grads) {
  const size_t part = grads && (p.parts > 1 || !p.lanes) ? ws_align(sizeof(float) * 2 * len * static_cast<size_t>(p.parts)) : 0;
  return part + (p.lanes ? 0 : ws_align(sizeof(float) * 3 * static_cast<size_t>(rows)));
}

template <class T>
int launch_norm_sum(const NormBwdArgs &a, int parts) {
  ProfScope prof("layernorm_grads", 8.0 * a.len * parts, WORK_BYTE);
  TDH_LAUNCH((layernorm_sum_kernel<T>), dim3(static_cast<unsigned>(ceil_div_sz(2 * static_cast<size_t>(a.len), NS_COLS))),
             dim3(NS_COLS * NS_GROUPS), 0, ctx().stream, a.partial, parts, a.len, a.dgamma, a.dbeta, a.accumulate);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

template <class T>
int launch_norm_bwd(NormBwdArgs a) {
  const NormBwdPlan p = norm_bwd_plan(a.rows, a.len);
  const bool grads = a.dgamma || a.dbeta;
  TDH_TRY(ws_begin(norm_bwd_bytes(p, a.rows, a.len, grads)));
  if (grads && (p.parts > 1 || !p.lanes)) {
    void *part = nullptr;
    TDH_TRY(ws_take(sizeof(float) * 2 * a.len * static_cast<size_t>(p.parts), &part));
    a.partial = static_cast<float *>(part);
  }
  {
    ProfScope prof("layernorm_bwd", static_cast<double>(sizeof(T)) * a.rows * a.len * (a.dx ? 3 : 2), WORK_BYTE);
    if (!p.lanes) {
      void *sums = nullptr;
      TDH_TRY(ws_take(sizeof(float) * 3 * static_cast<size_t>(a.rows), &sums));
      TDH_LAUNCH((layernorm_long_sums_kernel<T>), dim3(std::min(a.rows, 65536)), dim3(NS_NT), 0, ctx().stream, a, static_cast<float *>(sums));
      TDH_LAUNCH_CHECK();
      TDH_LAUNCH((layernorm_long_bwd_kernel<T>), dim3(ceil_div(ceil_div(a.len, Word<T>::N), NL_NT), p.parts), dim3(NL_NT), 0, ctx().stream, a,
                 static_cast<const float *>(sums), p.band);
      TDH_LAUNCH_CHECK();
    } else {
      constexpr int W = 16 / Word<T>::N;
      const bool once = static_cast<double>(sizeof(T)) * a.rows * a.len > NORM_ONCE_BYTES;
      auto go = [&](auto l, auto w) {
        constexpr int LANES = decltype(l)::value, WORDS = decltype(w)::value;
        if (once)
          TDH_LAUNCH((layernorm_bwd_kernel<T, LANES, WORDS, true>), dim3(p.parts), dim3(NB_NT), 0, ctx().stream, a);
        else
          TDH_LAUNCH((layernorm_bwd_kernel<T, LANES, WORDS, false>), dim3(p.parts), dim3(NB_NT), 0, ctx().stream, a);
        TDH_LAUNCH_CHECK();
        return static_cast<int>(TDH_OK);
      };
      const std::integral_constant<int, W / 2> half;
      const std::integral_constant<int, W> all;
      switch (p.lanes) {
        case 8: TDH_TRY(go(std::integral_constant<int, 8>(), half)); break;
        case 32: TDH_TRY(go(std::integral_constant<int, 32>(), half)); break;
        case 64: TDH_TRY(go(std::integral_constant<int, 64>(), all)); break;
        case 128: TDH_TRY(go(std::integral_constant<int, 128>(), all)); break;
        case 256: TDH_TRY(go(std::integral_constant<int, 256>(), all)); break;
        default: TDH_TRY(go(std::integral_constant<int, 512>(), all)); break;
      }
    }
  }
  return a.partial ? launch_norm_sum<T>(a, p.parts) : static_cast<int>(TDH_OK);
}

Span rows_span(int dtype, int rows, int len, const void *p, size_t ld) {
  return Span{p, rows > 0 ? dtype_size(dtype) * ((rows - 1) * ld + len) : 0};
}
int check_norm(const char *who, int dtype, int rows, int len) {
  TDH_CHECK_ARG(dtype_known(dtype), "%s: element type %d", who, dtype);
  TDH_CHECK_ARG(rows >= 0 && rows <= GRID_X_MAX && len > 0 && len <= (1 << 24), "%s: %d rows of %d elements", who, rows, len);
  return TDH_OK;
}
int check_norm_rows(const char *who, const char *what, int dtype, int rows, int len, const void *p, size_t ld) {
  TDH_CHECK_ARG(ld >= static_cast<size_t>(len) && ld <= (static_cast<size_t>(1) << 40), "%s: rows of %d elements of %s %zu apart", who, len, what, ld);
  TDH_CHECK_ARG(rows == 0 || p, "%s: null tensor", who);
  TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) == 0, "%s: %s not aligned to its elements", who, what);
  return TDH_OK;
}
// `out` is `in` itself, row for row, or apart from it
int check_in_place(const char *who, const Span &out, const Span &in, size_t ld_out, size_t ld_in) {
  return out.p == in.p && ld_out == ld_in ? static_cast<int>(TDH_OK) : check_apart(who, {out}, {in});
}

}  // namespace
}  // namespace tdh

using namespace tdh;

extern "C" {

int tdh_layernorm_fwd(int dtype, int rows, int len, float eps, const void *x, size_t ld, const void *gamma, const void *beta, void *y,
                      size_t ld_y, float *stats) {
  const char *who = "tdh_layernorm_fwd";
  TDH_TRY(check_norm(who, dtype, rows, len));
  TDH_CHECK_ARG(eps >= FLT_MIN && eps <= FLT_MAX, "%s: eps %g", who, eps);
  TDH_TRY(check_norm_rows(who, "x", dtype, rows, len, x, ld));
  TDH_TRY(check_norm_rows(who, "y", dtype, rows, len, y, ld_y));
  const uintptr_t align = dtype_size(dtype) - 1;
  TDH_CHECK_ARG(((reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(beta)) & align) == 0 && (reinterpret_cast<uintptr_t>(stats) & 3) == 0,
                "%s: a tensor that is not aligned to its elements", who);
  const Span sx = rows_span(dtype, rows, len, x, ld), sy = rows_span(dtype, rows, len, y, ld_y);
  const Span st{rows ? stats : nullptr, 8 * static_cast<size_t>(rows)}, sg{gamma, dtype_size(dtype) * len}, sb{beta, dtype_size(dtype) * len};
  TDH_TRY(check_apart(who, {sy, st}, {sg, sb}));
  TDH_TRY(check_apart(who, {st}, {sx}));
  TDH_TRY(check_in_place(who, sy, sx, ld_y, ld));
  TDH_REQUIRE_INIT();
  if (rows == 0) return TDH_OK;
  const NormFwdArgs a{x, gamma, beta, y, stats, ld, ld_y, rows, len, eps, 1.0f / static_cast<float>(len)};
  ProfScope prof("layernorm_fwd", 2.0 * dtype_size(dtype) * rows * len, WORK_BYTE);
  return with_dtype(dtype, [&](auto t) { return launch_norm_fwd<decltype(t)>(a); });
}

int tdh_layernorm_bwd(int dtype, int rows, int len, const void *x, size_t ld, const void *gamma, const float *stats, const void *dy,
                      size_t ld_dy, void *dx, size_t ld_dx, void *dgamma, void *dbeta, int accumulate) {
  const char *who = "tdh_layernorm_bwd";
  TDH_TRY(check_norm(who, dtype, rows, len));
  TDH_TRY(check_norm_rows(who, "x", dtype, rows, len, x, ld));
  TDH_TRY(check_norm_rows(who, "dy", dtype, rows, len, dy, ld_dy));
  if (dx) TDH_TRY(check_norm_rows(who, "dx", dtype, rows, len, dx, ld_dx));
  TDH_CHECK_ARG(rows == 0 || stats, "%s: null tensor", who);
  const size_t size = dtype_size(dtype), row = size * len;
  TDH_CHECK_ARG(((reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(dgamma) | reinterpret_cast<uintptr_t>(dbeta)) & (size - 1)) == 0 &&
                    (reinterpret_cast<uintptr_t>(stats) & 3) == 0,
                "%s: a tensor that is not aligned to its elements", who);
  const Span sx = rows_span(dtype, rows, len, x, ld), sdy = rows_span(dtype, rows, len, dy, ld_dy), sdx = rows_span(dtype, dx ? rows : 0, len, dx, ld_dx);
  const Span st{stats, 8 * static_cast<size_t>(rows)}, sg{gamma, row}, sdg{dgamma, row}, sdb{dbeta, row};
  TDH_TRY(check_apart(who, {sdx, sdg, sdb}, {sx, st, sg}));
  TDH_TRY(check_apart(who, {sdg, sdb}, {sdy}));
  TDH_TRY(check_in_place(who, sdx, sdy, ld_dx, ld_dy));
  TDH_REQUIRE_INIT();
  if (rows == 0 ? accumulate || (!dgamma && !dbeta) : !dx && !dgamma && !dbeta) return TDH_OK;
  const NormBwdArgs a{x, gamma, dy, stats, dx, ld, ld_dy, ld_dx, rows, len, 1.0f / static_cast<float>(len), nullptr, dgamma, dbeta, accumulate};
  return with_dtype(dtype, [&](auto t) {
    return rows ? launch_norm_bwd<decltype(t)>(a) : launch_norm_sum<decltype(t)>(a, 0);   // (sums of nothing)
  });
}

}  // extern "C"
