// gated_ff.hip — the gated feed-forward block: z = x W + b with W = [in][2 hidden], gate columns first, and
// h = act(z_gate) * z_up; on the way back dz = (dh * z_up * act'(z_gate), dh * act(z_gate)),
// dx = dz W^T, dW = x^T dz, db = the column sums of dz.
//
//   up to FEW_ROWS samples   the weights are read once, as they lie, by vector kernels (few_fwd_kernel, few_bwd_kernel)
//   16-bit types             three products on the matrix cores (gemm16.h); the forward one takes gate and up columns in
//                            pairs and leaves h, and z for the way back
//   fp32                     products of many samples on operands in three bf16 parts (gemm_x3.h), at any row length, the
//                            others the fully-connected layer's
//
// z is kept in fp32 in every type, so that the derivative sees what the activation saw. dz is rounded to the 16-bit type once,
// as the products' operand: in two parts each, dx and dW would cost twice the matrix work for one rounding among as
// many as there are products' operands. db is summed before that rounding. fp16 has not the range of dz, which is a product of three
// numbers: there dz is held times a power of two that brings its largest finite value into [2^14, 2^15), so what vanishes is 2^-39 of that
// at most, and the products' sums are taken back by the same power (gate_dz_peak_kernel).
#include "gemm16.h"
#include "gemm_x3.h"

namespace tdh {

namespace {

constexpr int GF_NT = 256;

// s = 1 / (1 + exp(-x)); the two instructions are off by an ulp each. rest: 1 - s, from the exponential, as a difference it has nothing
// left where s is next to 1 (the derivative of a sigmoid gate at 17 and more would be 0).
__device__ __forceinline__ float logistic(const float x, float *rest) {
  const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * __builtin_fabsf(x)), big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  *rest = x < 0.0f ? big : small;
  return x < 0.0f ? small : big;
}

// the gate's activation, and its derivative
template <int KIND>
__device__ __forceinline__ float gate_act(const float g, float *slope) {
  if constexpr (KIND == TDH_GATE_SILU) {
    float rest;
    const float s = logistic(g, &rest);
    *slope = s * (1.0f + g * rest);
    return g * s;
  } else if constexpr (KIND == TDH_GATE_GELU) {
    // Beside zero cdf(-|g|) = erfc(x) / 2, x = |g| / sqrt(2), falls like exp(-x^2), and so that h keeps its figures there, the fit is one of
    // erfc(x) exp(x^2) / 2, a polynomial in t = 1 / (1 + 0.38 x) without a constant term, off by 2.7e-8 of the value at most for 0 <= x <= 14.2
    // (fitted for the least relative error), and g^2 brings its rounding along. In fp32 h is off by 7 half-ulps at most for
    // -13 <= g <= 8, the derivative by 7 of cdf + |g| pdf, beside an ulp each of the machine's exponential and reciprocal. 20 us of 2294 more
    // than a fit good to 1.5e-7 of one (4096 x 4096 -> 2 x 12288 in bf16 there and back).
    const float c = __builtin_amdgcn_fmed3f(g, -20.0f, 20.0f);   // (exp(-200) is 0, and the square stays finite)
    const float q = c * c, a = -0.72134752044448170f * q;
    const float lo = __builtin_fmaf(q, -0.72134752044448170f, -a) - 0.72134752044448170f * __builtin_fmaf(c, c, -q) - 9.6298e-9f * q;
    const float e0 = __builtin_amdgcn_exp2f(a), e = __builtin_fmaf(e0, 0.69314718055994531f * lo, e0);
    const float t  = __builtin_amdgcn_rcpf(__builtin_fmaf(0.26870057f, __builtin_fabsf(c), 1.0f));
    constexpr float fit[9] = {0.10720470547676086f, 0.10697626322507858f, 0.10180984437465668f, 0.06998414546251297f, 0.1132340133190155f,
                              -0.07782156765460968f, 0.1790992021560669f, -0.12963144481182098f, 0.029144831001758575f};
    float r = fit[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) r = __builtin_fmaf(r, t, fit[i]);
    const float tail = e * (t * r), cdf = g < 0.0f ? tail : 1.0f - tail;   // (NaN stays)
    *slope = cdf + g * (0.39894228040143268f * e);
    return g * cdf;
  } else if constexpr (KIND == TDH_GATE_GELU_TANH) {
    // 0.5 (1 + tanh(y)) = 1 / (1 + exp(-2 y)), y = sqrt(2/pi) (g + 0.044715 g^3); beyond 16 it is 0 or 1, and the
    // square in the derivative would overflow where its factor is 0
    const float c = __builtin_amdgcn_fmed3f(g, -16.0f, 16.0f);
    float rest;
    const float s = logistic(1.5957691216057308f * (c + 0.044715f * c * c * c), &rest);
    *slope = s + g * s * rest * (1.5957691216057308f * (1.0f + 0.134145f * c * c));
    return g * s;
  } else if constexpr (KIND == TDH_GATE_SIGMOID) {
    float rest;
    const float s = logistic(g, &rest);
    *slope = s * rest;
    return s;
  } else if constexpr (KIND == TDH_GATE_RELU) {
    *slope = g > 0.0f ? 1.0f : 0.0f;
    return g > 0.0f ? g : g != g ? g : 0.0f;
  } else {
    *slope = 1.0f;
    return g;
  }
}
// f with the kind as a constant: one branch around a loop, not one in every turn
template <class F>
__device__ __forceinline__ void with_gate(const int act, const F &f) {
  switch (act) {
    case TDH_GATE_SILU: return f(std::integral_constant<int, TDH_GATE_SILU>());
    case TDH_GATE_GELU: return f(std::integral_constant<int, TDH_GATE_GELU>());
    case TDH_GATE_GELU_TANH: return f(std::integral_constant<int, TDH_GATE_GELU_TANH>());
    case TDH_GATE_SIGMOID: return f(std::integral_constant<int, TDH_GATE_SIGMOID>());
    case TDH_GATE_RELU: return f(std::integral_constant<int, TDH_GATE_RELU>());
    default: return f(std::integral_constant<int, TDH_GATE_NONE>());
  }
}

// h of z, for the products that are the fully-connected layer's. Bound by memory: 12 bytes an element.
__global__ void __launch_bounds__(GF_NT)
gate_fwd_kernel(const float *__restrict__ z, float *__restrict__ h, const int hidden, const size_t total, const int act) {
  const size_t i = static_cast<size_t>(blockIdx.x) * GF_NT + threadIdx.x;
  if (i >= total) return;
  const size_t row = i / hidden, c = i - row * hidden;
  with_gate(act, [&](auto kind) {
    float slope;
    const float a = gate_act<decltype(kind)::value>(z[row * 2 * hidden + c], &slope);
    h[i] = a * z[row * 2 * hidden + hidden + c];
  });
}

// dst = src in another type, an element a thread: 67 M elements from fp32 to bf16 134 us, 3.0 TB/s, bound by accesses of two bytes a lane.
template <class D, class S>
__global__ void __launch_bounds__(GF_NT)
cast_kernel(const S *__restrict__ src, D *__restrict__ dst, const size_t n) {
  const size_t stride = static_cast<size_t>(gridDim.x) * GF_NT;
  for (size_t i = static_cast<size_t>(blockIdx.x) * GF_NT + threadIdx.x; i < n; i += stride) dst[i] = from_f32<D>(to_f32(src[i]));
}

template <class D, class S>
int launch_cast(const S *src, D *dst, size_t n) {
  if (!n) return TDH_OK;
  ProfScope prof("cast", static_cast<double>(n) * (sizeof(D) + sizeof(S)), WORK_BYTE);
  TDH_LAUNCH((cast_kernel<D, S>), dim3(static_cast<unsigned>(std::min<size_t>(ceil_div_sz(n, GF_NT), GRID_X_MAX))),
             dim3(GF_NT), 0, ctx().stream, src, dst, n);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

template <class T>
int take(size_t n, T **out) {
  void *p = nullptr;
  TDH_TRY(ws_take(n * sizeof(T), &p));
  *out = static_cast<T *>(p);
  return TDH_OK;
}

// ------------------------------------------------------------ 16-bit types
// What leaves the products. Columns of z, w and dz come in two halves of `half` columns, of which the first `hidden`
// are in use (half is hidden rounded up to a multiple of 8 where a packed copy is read).

// forward: h, and z where it is kept
template <class T>
struct EpiGate {
  T *h;
  float *z;            // or null
  const T *bias;       // or null
  float *partial;      // slices of z, [split][rows][2 half], that a sum of them reads
  int rows, hidden, half, act;
  // g and u at (m, n) to h; writes z
  template <int KIND>
  __device__ __forceinline__ float one(const size_t m, const int n, const float g, const float u) const {
    if (z) {   // (read in the backward pass, after much else: past the caches)
      __builtin_nontemporal_store(g, z + m * 2 * hidden + n);
      __builtin_nontemporal_store(u, z + m * 2 * hidden + hidden + n);
    }
    float slope;
    return gate_act<KIND>(g, &slope) * u;
  }
  // the whole sums of (m, n), without the bias
  __device__ __forceinline__ void finish(const size_t m, const int n, float g, float u) const {
    if (bias) {
      g += to_f32(bias[n]);
      u += to_f32(bias[hidden + n]);
    }
    with_gate(act, [&](auto kind) { h[m * hidden + n] = from_f32<T>(one<decltype(kind)::value>(m, n, g, u)); });
  }
  template <int TM, int TN>
  __device__ __forceinline__ void done(const g16_f32x16 (&acc)[TM][TN], const int m0, const int n0, const int lane, const int,
                                       float *lds) const {
    const int n = n0 + (lane & 31), m = m0 + 4 * (lane >> 5);
    float bg[TN / 2], bu[TN / 2];
#pragma unroll
    for (int j = 0; j < TN / 2; ++j) {
      const bool in = bias && n + 32 * j < hidden;
      bg[j] = in ? to_f32(bias[n + 32 * j]) : 0.0f;
      bu[j] = in ? to_f32(bias[hidden + n + 32 * j]) : 0.0f;
    }
    with_gate(act, [&](auto kind) {
      const G16Turn<16 * TN> turn{lds};
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN / 2; ++j)
          turn.put(lane, j, [&](int r) {
            const int row = m + 32 * i + 8 * (r >> 2) + (r & 3);
            if (row >= rows || n + 32 * j >= hidden) return 0.0f;
            return one<decltype(kind)::value>(row, n + 32 * j, acc[i][2 * j][r] + bg[j], acc[i][2 * j + 1][r] + bu[j]);
          });
        turn.rows(lane, [&](int row, int col, const float (&v)[8]) {
          if (m0 + 32 * i + row >= rows) return;
          T *p = h + static_cast<size_t>(m0 + 32 * i + row) * hidden + n0 + col;
          if (n0 + col + 8 <= hidden) return store8(p, v);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n0 + col + e < hidden) p[e] = from_f32<T>(v[e]);
        });
      }
    });
  }
};

// a gradient: out (+)= C
template <class T>
struct EpiGrad {
  T *out;
  float *partial;      // slices instead, [split][rows][cols]
  int rows, cols;      // of C
  int hidden, half;    // two halves of columns, as above (one: both are cols)
  int accumulate;
  const float *unscale = nullptr;   // fp16: what C has to be multiplied with (device memory; null: nothing)
  __device__ __forceinline__ float factor() const {
    if constexpr (std::is_same<T, f16>::value) return unscale ? *unscale : 1.0f;
    return 1.0f;
  }
  // where column n of C's row m goes (n is in use)
  __device__ __forceinline__ T *at(const size_t m, const int n) const {
    return out + m * (cols > half ? 2 * hidden : hidden) + (n < half ? n : n - half + hidden);
  }
  __device__ __forceinline__ void one(const size_t m, const int n, float v) const {
    if ((n < half ? n : n - half) >= hidden) return;
    T *p = at(m, n);
    if (accumulate) v += to_f32(*p);
    *p = from_f32<T>(v);
  }
  template <int TM, int TN>
  __device__ __forceinline__ void done(const g16_f32x16 (&acc)[TM][TN], const int m0, const int n0, const int lane, const int split,
                                       float *lds) const {
    if (partial) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int m = m0 + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const int n = n0 + 32 * j + (lane & 31);
            if (m < rows && n < cols) partial[(static_cast<size_t>(split) * rows + m) * cols + n] = acc[i][j][r];
          }
        }
      return;
    }
    const G16Turn<32 * TN> turn{lds};
    const float f = factor();
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) turn.put(lane, j, [&](int r) { return f * acc[i][j][r]; });
      turn.rows(lane, [&](int row, int col, const float (&v)[8]) {
        const int m = m0 + 32 * i + row, n = n0 + col;
        if (m >= rows) return;
        if (n < cols && (n < half ? n : n - half) + 8 <= hidden) {   // (half is a multiple of eight, or all there is)
          T *p = at(m, n);
          if (!accumulate) return store8(p, v);
          float o[8];
          load8(p, o);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] += v[e];
          store8(p, o);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < cols) one(m, n + e, v[e]);
        }
      });
    }
  }
};

// slices added up, in their order; bound by reading them (three of 2000 x 5280: 31 us, 4.1 TB/s; 16 of one row of 24576: 4.0, a launch,
// with workgroups of 64 threads, so that more compute units have one)
template <class T>
__global__ void __launch_bounds__(GF_NT)
gate_reduce_kernel(const EpiGate<T> epi, const int splits) {
  const size_t i = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= static_cast<size_t>(epi.rows) * epi.hidden) return;
  const size_t m = i / epi.hidden, slice = static_cast<size_t>(epi.rows) * 2 * epi.half;
  const int n = static_cast<int>(i - m * epi.hidden);
  const float *p = epi.partial + m * 2 * epi.half + n;
  float g = 0.0f, u = 0.0f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    g += p[s * slice];
    u += p[s * slice + epi.half];
  }
  epi.finish(m, n, g, u);
}
template <class T>
int launch_gate_reduce(const EpiGate<T> &epi, int splits) {
  const size_t total = static_cast<size_t>(epi.rows) * epi.hidden;
  const int threads  = total < 32768 ? 64 : GF_NT;
  ProfScope prof("gated_ff_fwd_reduce", 8.0 * splits * total, WORK_BYTE);
  TDH_LAUNCH((gate_reduce_kernel<T>), dim3(static_cast<unsigned>(ceil_div_sz(total, threads))), dim3(threads), 0, ctx().stream, epi, splits);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}
template <class T>
__global__ void __launch_bounds__(GF_NT)
grad_reduce_kernel(const EpiGrad<T> epi, const int splits) {
  const size_t total = static_cast<size_t>(epi.rows) * epi.cols, i = static_cast<size_t>(blockIdx.x) * GF_NT + threadIdx.x;
  if (i >= total) return;
  const size_t m = i / epi.cols;
  float v = 0.0f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) v += epi.partial[s * total + i];
  epi.one(m, static_cast<int>(i - m * epi.cols), epi.factor() * v);
}

template <class T>
int launch_grad_reduce(const EpiGrad<T> &epi, int splits) {
  const size_t total = static_cast<size_t>(epi.rows) * epi.cols;
  ProfScope prof("gated_ff_bwd_reduce", 4.0 * splits * total, WORK_BYTE);
  TDH_LAUNCH((grad_reduce_kernel<T>), dim3(static_cast<unsigned>(ceil_div_sz(total, GF_NT))), dim3(GF_NT), 0, ctx().stream, epi, splits);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

// Matrices copied to padded ones: columns in one or two halves of `used` values, `half` (a multiple of 8) apart in the copy;
// what is behind a half is zero. A thread writes eight values as a word. (1001 -> 2 x 2731 and 77 samples in fp16, 11 MB: 8.7 us. Products that
// read unaligned rows would do without, but loads straight into LDS are of whole 16-byte words.)
template <class T>
struct PackJobs {
  struct Job {
    const T *src;
    T *dst;
    int used, half, halves;
    unsigned blocks;
    size_t words;
  } job[2];
};
template <class T>
__global__ void __launch_bounds__(GF_NT)
pack_kernel(const PackJobs<T> jobs) {
  const bool second = blockIdx.x >= jobs.job[0].blocks;
  const typename PackJobs<T>::Job &j = jobs.job[second];
  const size_t i = static_cast<size_t>(blockIdx.x - (second ? jobs.job[0].blocks : 0)) * GF_NT + threadIdx.x;
  if (i >= j.words) return;
  const int per = j.half / 8;   // words of a half
  const size_t row = i / (per * j.halves);
  int c = static_cast<int>(i - row * (per * j.halves)), h = c >= per ? 1 : 0;
  c = (c - h * per) * 8;
  const T *p = j.src + (row * j.halves + h) * j.used + c;
  uint4 v;
  if (c + 8 <= j.used) {
    v = load_word(p).raw;
  } else {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c + e < j.used ? to_f32(p[e]) : 0.0f;
    v = Word<T>::from(f).raw;
  }
  *reinterpret_cast<uint4 *>(j.dst + i * 8) = v;
}

// dz of the columns n .. of a word of T, row by row: take(m, dg, du), zero behind `hidden`
template <class T, class F>
__device__ __forceinline__ void gate_dz_rows(const float *__restrict__ z, const T *__restrict__ dh, const int n, const int hidden, const int act,
                                             const int first, const int end, const F &take) {
  constexpr int E  = Word<T>::N;
  const bool whole = n + E <= hidden;
  with_gate(act, [&](auto kind) {
#pragma unroll 2
    for (int m = first; m < end; ++m) {
      float g[E], u[E], d[E], dg[E], du[E];
      const float *zr = z + static_cast<size_t>(m) * 2 * hidden + n;
      const T *dr     = dh + static_cast<size_t>(m) * hidden + n;
      if (whole) {
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
          const Word<float> gq = load_word(zr + 4 * q), uq = load_word(zr + hidden + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            g[4 * q + e] = gq[e];
            u[4 * q + e] = uq[e];
          }
        }
        const Word<T> w = load_word(dr);
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = w[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool in = n + e < hidden;
          g[e] = in ? zr[e] : 0.0f;
          u[e] = in ? zr[hidden + e] : 0.0f;
          d[e] = in ? to_f32(dr[e]) : 0.0f;
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float slope;
        const float a = gate_act<decltype(kind)::value>(g[e], &slope);
        dg[e] = d[e] * u[e] * slope;
        du[e] = d[e] * a;
        if (!whole && n + e >= hidden) dg[e] = du[e] = 0.0f;
      }
      take(m, dg, du);
    }
  });
}

// The largest finite |dz| of a workgroup's part, in front of gate_dz_kernel: which power of two fp16 holds dz times. It reads what that pass
// reads, as dz is known only then: 4096 x 12288 105-114 us (4.4-4.7 TB/s) of a step of 2480, 300 x 1000 4, a launch. About 1024 workgroups (or
// as many as a row of columns has), as every workgroup of the next pass reads all their peaks.
template <class T>
__global__ void __launch_bounds__(GF_NT)
gate_dz_peak_kernel(const float *__restrict__ z, const T *__restrict__ dh, float *__restrict__ peaks, const int rows, const int hidden,
                    const int act, const int blocks_n, const int band_rows) {
  constexpr int E = Word<T>::N;
  __shared__ float part[GF_NT / 64];
  const int n = (blockIdx.x % blocks_n * GF_NT + threadIdx.x) * E, first = blockIdx.x / blocks_n * band_rows;
  float peak = 0.0f;
  if (n < hidden)
    gate_dz_rows(z, dh, n, hidden, act, first, min(rows, first + band_rows), [&](int, const float (&dg)[E], const float (&du)[E]) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float a = __builtin_fabsf(dg[e]), b = __builtin_fabsf(du[e]);
        if (a < INFINITY) peak = fmaxf(peak, a);
        if (b < INFINITY) peak = fmaxf(peak, b);
      }
    });
#pragma unroll
  for (int o = 32; o; o >>= 1) peak = fmaxf(peak, __shfl_xor(peak, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = peak;
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int w = 1; w < GF_NT / 64; ++w) peak = fmaxf(peak, part[w]);
  peaks[blockIdx.x] = peak;
}
// 2^k that brings the largest of n peaks into [2^14, 2^15) (as far as 2^126 does), the same in every thread of the workgroup
__device__ __forceinline__ float gate_dz_scale(const float *__restrict__ peaks, const int n) {
  __shared__ float part[GF_NT / 64];
  float peak = 0.0f;
  for (int i = threadIdx.x; i < n; i += GF_NT) peak = fmaxf(peak, peaks[i]);
#pragma unroll
  for (int o = 32; o; o >>= 1) peak = fmaxf(peak, __shfl_xor(peak, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = peak;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < GF_NT / 64; ++w) peak = fmaxf(peak, part[w]);
  // (exponents as they are held: the scale's is 127 + 14 - (peak's - 127))
  return __uint_as_float(min(268u - (__float_as_uint(peak) >> 23), 253u) << 23);
}
// the peaks of a call, and where the inverse of the scale is left for the products (null: dz is not scaled)
struct DzPeaks {
  const float *peaks;
  int n;
  float *unscale;
};

// dz as the products read it (type Z), [rows][2 half], zero behind each half; and with `bias_part` the sums of dz over the rows of this
// workgroup's band (in fp32, before the rounding). A thread takes a word of T's columns. Bound by memory: 4096 x 12288 in bf16 136-142 us,
// 5.0 TB/s (z is 8 of its 14 bytes an element; read past the caches 142). A pass of its own: as a part of the products it would read
// z and dh once a tile of columns, and dW reads dz with the other fast index.
template <class T, class Z>
__global__ void __launch_bounds__(GF_NT)
gate_dz_kernel(const float *__restrict__ z, const T *__restrict__ dh, Z *__restrict__ dz, float *__restrict__ bias_part,
               const int rows, const int hidden, const int half, const int act, const int blocks_n, const int band_rows, const DzPeaks peaks) {
  constexpr int E = Word<T>::N;
  float scale     = 1.0f;
  if constexpr (std::is_same<Z, f16>::value)
    if (peaks.unscale) {
      scale = gate_dz_scale(peaks.peaks, peaks.n);
      if (blockIdx.x == 0 && threadIdx.x == 0) *peaks.unscale = __uint_as_float((254u << 23) - __float_as_uint(scale));
    }
  const int n = (blockIdx.x % blocks_n * GF_NT + threadIdx.x) * E, band = blockIdx.x / blocks_n;
  if (n >= half) return;
  float sg[E] = {}, su[E] = {};
  gate_dz_rows(z, dh, n, hidden, act, band * band_rows, min(rows, (band + 1) * band_rows), [&](int m, const float (&dg)[E], const float (&du)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      sg[e] += dg[e];
      su[e] += du[e];
    }
    if (!dz) return;
    Z *o = dz + static_cast<size_t>(m) * 2 * half + n;
    if (n + E <= half) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float(&v)[E] = s ? du : dg;
#pragma unroll
        for (int q = 0; q < E / Word<Z>::N; ++q) {
          float w[Word<Z>::N];
#pragma unroll
          for (int e = 0; e < Word<Z>::N; ++e) w[e] = scale * v[q * Word<Z>::N + e];
          store_word(o + s * half + q * Word<Z>::N, Word<Z>::from(w).raw);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (n + e < half) {
          o[e]        = from_f32<Z>(scale * dg[e]);
          o[half + e] = from_f32<Z>(scale * du[e]);
        }
    }
  });
  if (bias_part) {
    float *p = bias_part + static_cast<size_t>(band) * 2 * hidden + n;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (n + e < hidden) {
        p[e]          = sg[e];
        p[hidden + e] = su[e];
      }
  }
}
// rows of a band: 32, or as few as it takes for four workgroups a compute unit (bias sums: no more than 128 bands up to 4096 samples)
struct DzPlan {
  int blocks_n, band_rows, bands;
};
template <class T>
DzPlan dz_plan(int half, int batch, bool sums) {
  DzPlan p;
  p.blocks_n  = ceil_div(half, Word<T>::N * GF_NT);
  p.band_rows = std::max(1, std::min<int>(32, static_cast<long>(batch) * p.blocks_n / 1024));
  if (sums) p.band_rows = std::max(p.band_rows, std::min(32, ceil_div(batch, 128)));
  p.bands = ceil_div(batch, p.band_rows);
  return p;
}
// ... of the pass for the largest dz: four workgroups a compute unit at most, where a row of columns has no more
template <class T>
DzPlan dz_peak_plan(int hidden, int batch) {
  DzPlan p;
  p.blocks_n  = ceil_div(hidden, Word<T>::N * GF_NT);
  p.band_rows = std::max(1, static_cast<int>((static_cast<long>(batch) * p.blocks_n + 1023) / 1024));
  p.bands     = ceil_div(batch, p.band_rows);
  return p;
}
template <class T, class Z>
int launch_dz(const DzPlan &p, int act, int hidden, int half, int batch, const float *z, const T *dh, Z *dz, float *bias_part,
              const DzPeaks &peaks = DzPeaks{}) {
  ProfScope prof("gated_ff_dz", (8.0 + 3 * sizeof(T)) * batch * hidden, WORK_BYTE);
  TDH_LAUNCH((gate_dz_kernel<T, Z>), dim3(p.blocks_n * p.bands), dim3(GF_NT), 0, ctx().stream, z, dh, dz, bias_part, batch, hidden, half,
             act, p.blocks_n, p.band_rows, peaks);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}
template <class T>
int launch_dz_peak(const DzPlan &p, int act, int hidden, int batch, const float *z, const T *dh, float *peaks) {
  ProfScope prof("gated_ff_dz_peak", (8.0 + sizeof(T)) * batch * hidden, WORK_BYTE);
  TDH_LAUNCH((gate_dz_peak_kernel<T>), dim3(p.blocks_n * p.bands), dim3(GF_NT), 0, ctx().stream, z, dh, peaks, batch, hidden, act, p.blocks_n,
             p.band_rows);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}
// db (+)= the bands' sums: 32 columns a workgroup, 32 groups of bands, their sums in order (128 bands of 8192 columns 4.1 us, a launch;
// a thread a column, all bands in turn: 45)
constexpr int BS_GROUPS = 32;
template <class T>
__global__ void __launch_bounds__(32 * BS_GROUPS)
bias_sum_kernel(const float *__restrict__ part, T *__restrict__ db, const int bands, const int cols, const int accumulate) {
  __shared__ float lds[BS_GROUPS][32];
  const int c = threadIdx.x & 31, group = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
  float s = 0.0f;
  if (n < cols) {
#pragma unroll 4
    for (int b = group; b < bands; b += BS_GROUPS) s += part[static_cast<size_t>(b) * cols + n];
  }
  lds[group][c] = s;
  __syncthreads();
  if (group || n >= cols) return;
#pragma unroll
  for (int g = 1; g < BS_GROUPS; ++g) s += lds[g][c];
  if (accumulate) s += to_f32(db[n]);
  db[n] = from_f32<T>(s);
}
template <class T>
int launch_db(const float *part, T *db, int bands, int hidden, int accumulate) {
  ProfScope prof("gated_ff_db", 8.0 * bands * hidden, WORK_BYTE);
  TDH_LAUNCH((bias_sum_kernel<T>), dim3(ceil_div(2 * hidden, 32)), dim3(32 * BS_GROUPS), 0, ctx().stream, part, db, bands, 2 * hidden,
             accumulate);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

// ------------------------------------------------------------ a few rows, any type
// Up to FEW_ROWS samples: the weights are read once, in words, straight into the vector units; bound by that read (and
// the write of dW).
constexpr int FEW_ROWS = 4, FEW_NT = 512;

// Forward. A unit of work is a strip of LANES words along the columns and `rows` of the k; its threads are LANES lanes along
// the columns times 512 / LANES along k, x lies in LDS in slices, and the sums of the waves meet in LDS at the end. Long
// rows matter more than anything: 1 KB of a row at a time reaches 6.4 TB/s, 128 bytes of many rows 4.1 to 4.4. So
// large matrices are split along k, gate and up columns apart, and their slices added up by a launch of its own (BOTH =
// false); where a strip is small a workgroup takes the gate's columns and the up columns that belong to them, and
// finishes (BOTH = true). 4096 -> 2 x 12288 in bf16, one row: 31.5 us and 2.5 for the sum of 16 slices; through the caches
// 35.6.
constexpr int FEW_X = 8192;   // values of x in LDS
template <class T, int M, int LANES, bool BOTH, bool ONCE>
__global__ void __launch_bounds__(FEW_NT)
few_fwd_kernel(const T *__restrict__ x, const T *__restrict__ w, const EpiGate<T> epi, const int in, const int strips, const int split_rows) {
  constexpr int E = Word<T>::N, COLS = LANES * E, KG = FEW_NT / LANES, H = BOTH ? 2 : 1;
  constexpr int SLICE = FEW_X / M, SUMS = FEW_NT / 64 * H * COLS;
  __shared__ float lds[FEW_X > SUMS ? FEW_X : SUMS];
  const int tid = threadIdx.x, lc = tid % LANES, kg = tid / LANES, hidden = epi.hidden;
  const int id    = xcd_compact_id(blockIdx.x, gridDim.x);
  const int strip = id % strips, split = BOTH ? 0 : id / strips / 2, half = BOTH ? 0 : id / strips % 2;
  const int first = strip * COLS, n = first + lc * E;
  const int kend = min(in, (split + 1) * split_rows);
  const size_t ld = 2 * static_cast<size_t>(hidden);
  float acc[M][H][E] = {};
  for (int k0 = split * split_rows; k0 < kend; k0 += SLICE) {
    const int len = min(SLICE, kend - k0);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m)
      for (int k = tid; k < len; k += FEW_NT) lds[m * SLICE + k] = m < epi.rows ? to_f32(x[static_cast<size_t>(m) * in + k0 + k]) : 0.0f;
    __syncthreads();
    const T *wp = w + static_cast<size_t>(k0 + kg) * ld + half * hidden + n;
    auto add = [&](int k, const float (&v)[H][E]) {
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float xv = lds[m * SLICE + k];
#pragma unroll
        for (int s = 0; s < H; ++s)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[m][s][e] = __builtin_fmaf(xv, v[s][e], acc[m][s][e]);
      }
    };
    if (n + E <= hidden) {
#pragma unroll 8
      for (int k = kg; k < len; k += KG, wp += KG * ld) {
        float v[H][E];
#pragma unroll
        for (int s = 0; s < H; ++s) {
          const Word<T> word = load_word<T, ONCE>(wp + s * hidden);
#pragma unroll
          for (int e = 0; e < E; ++e) v[s][e] = word[e];
        }
        add(k, v);
      }
    } else if (n < hidden) {   // (the lane that has the last columns)
      for (int k = kg; k < len; k += KG, wp += KG * ld) {
        float v[H][E];
#pragma unroll
        for (int s = 0; s < H; ++s)
#pragma unroll
          for (int e = 0; e < E; ++e) v[s][e] = n + e < hidden ? to_f32(wp[s * hidden + e]) : 0.0f;
        add(k, v);
      }
    }
  }
#pragma unroll
  for (int o = LANES; o < 64; o <<= 1)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int s = 0; s < H; ++s)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[m][s][e] += __shfl_xor(acc[m][s][e], o);
#pragma unroll
  for (int m = 0; m < M; ++m) {
    if (m >= epi.rows) break;
    __syncthreads();
    if ((tid & 63) < LANES) {
#pragma unroll
      for (int s = 0; s < H; ++s)
#pragma unroll
        for (int e = 0; e < E; ++e) lds[(tid / 64 * H + s) * COLS + lc * E + e] = acc[m][s][e];
    }
    __syncthreads();
    for (int c = tid; c < COLS; c += FEW_NT) {
      const int col = first + c;
      if (col >= hidden) break;
      float v[H] = {};
#pragma unroll
      for (int q = 0; q < FEW_NT / 64; ++q)
#pragma unroll
        for (int s = 0; s < H; ++s) v[s] += lds[(q * H + s) * COLS + c];
      if constexpr (BOTH)
        epi.finish(m, col, v[0], v[1]);
      else
        epi.partial[(static_cast<size_t>(split) * epi.rows + m) * 2 * hidden + half * hidden + col] = v[0];
    }
  }
}

// Backward, bound by w and dw: dx[m][i] = sum_c dz[m][c] w[i][c] and dw[i][c] (+)= sum_m x[m][i] dz[m][c] in one pass over c: a workgroup has
// FEW_I rows of w and dw, its four waves take turns along c. dz is in fp32 (there is little of it). 4096 -> 2 x 12288 in bf16, one
// sample: 77 us, 5.2 TB/s; four: 118, their sums beside the memory. dx null: only dw, and w is not read; dw null: only dx.
constexpr int FEW_I = 4;
template <class T, int M, bool ONCE>
__global__ void __launch_bounds__(256)
few_bwd_kernel(const T *__restrict__ x, const T *__restrict__ w, const float *__restrict__ dz, T *__restrict__ dx, T *__restrict__ dw,
               const int in, const int cols, const int batch, const int accumulate) {
  constexpr int E = Word<T>::N;
  __shared__ float sums[4][M * FEW_I];
  const int tid = threadIdx.x, lane = tid & 63, i0 = blockIdx.x * FEW_I;
  float xv[M][FEW_I], acc[M][FEW_I] = {};
  size_t row[FEW_I];   // (rows past the end: the last one again, and nothing of it is kept)
#pragma unroll
  for (int i = 0; i < FEW_I; ++i) {
    row[i] = static_cast<size_t>(min(i0 + i, in - 1));
#pragma unroll
    for (int m = 0; m < M; ++m) xv[m][i] = dw && m < batch ? to_f32(x[m * static_cast<size_t>(in) + row[i]]) : 0.0f;
  }
  // the columns c .. c + E - 1, of which `n` are in use (WHOLE: all)
  auto chunk = [&](const int c, auto all, const int n) {
    constexpr bool WHOLE = decltype(all)::value;
    float d[M][E], wv[FEW_I][E];
#pragma unroll
    for (int i = 0; i < FEW_I; ++i) {
      if (!dx) break;
      const T *p = w + row[i] * cols + c;
      if constexpr (WHOLE) {
        const Word<T> v = load_word<T, ONCE>(p);
#pragma unroll
        for (int e = 0; e < E; ++e) wv[i][e] = v[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) wv[i][e] = e < n ? to_f32(p[e]) : 0.0f;
      }
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const float *p = dz + static_cast<size_t>(m < batch ? m : 0) * cols + c;
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        if constexpr (WHOLE) {
          const Word<float> v = load_word(p + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) d[m][4 * q + e] = m < batch ? v[e] : 0.0f;
        } else {
#pragma unroll
          for (int e = 4 * q; e < 4 * q + 4; ++e) d[m][e] = m < batch && e < n ? p[e] : 0.0f;
        }
      }
    }
    if (dx) {
#pragma unroll
      for (int i = 0; i < FEW_I; ++i)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[m][i] = __builtin_fmaf(d[m][e], wv[i][e], acc[m][i]);
    }
    if (!dw) return;
#pragma unroll
    for (int i = 0; i < FEW_I; ++i) {
      if (i0 + i >= in) break;
      T *p = dw + row[i] * cols + c;
      float o[E] = {};
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = m < batch ? __builtin_fmaf(xv[m][i], d[m][e], o[e]) : o[e];
      if constexpr (WHOLE) {
        if (accumulate) {
          const Word<T> was = load_word<T, ONCE>(p);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += was[e];
        }
        store_word<ONCE>(p, Word<T>::from(o).raw);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e < n) p[e] = from_f32<T>(accumulate ? o[e] + to_f32(p[e]) : o[e]);
      }
    }
  };
  int c = tid * E;
#pragma unroll 2
  for (; c + E <= cols; c += 256 * E) chunk(c, std::true_type(), E);
  if (c < cols) chunk(c, std::false_type(), cols - c);
  if (!dx) return;
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int i = 0; i < FEW_I; ++i) {
      float v = acc[m][i];
#pragma unroll
      for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
      if (lane == 0) sums[tid >> 6][m * FEW_I + i] = v;
    }
  __syncthreads();
  if (tid < M * FEW_I) {
    const int m = tid / FEW_I, i = tid % FEW_I;
    if (m < batch && i0 + i < in)
      dx[static_cast<size_t>(m) * in + i0 + i] = from_f32<T>(sums[0][tid] + sums[1][tid] + sums[2][tid] + sums[3][tid]);
  }
}

// f with the rows rounded up to a power of two as a constant
template <class F>
int with_rows(int batch, const F &f) {
  if (batch <= 1) return f(std::integral_constant<int, 1>());
  if (batch <= 2) return f(std::integral_constant<int, 2>());
  return f(std::integral_constant<int, 4>());
}
// matrices that the L2 caches (8 x 4 MB) do not hold are read past them
constexpr size_t FEW_ONCE_BYTES = 32u << 20;

template <class T>
int few_fwd(int act, int in, int hidden, int batch, const T *x, const T *w, const T *b, T *h, float *z) {
  const bool wide = hidden >= 256;
  const size_t bytes = sizeof(T) * static_cast<size_t>(in) * 2 * hidden;
  const int cols = (wide ? 64 : 16) * Word<T>::N, strips = ceil_div(hidden, cols);
  // a workgroup reads 256 KB at most, or an equal part of one of 768
  const long want  = std::min<long>(768, static_cast<long>(bytes >> 17));
  const bool both  = bytes / strips <= (256u << 10);
  const int most   = std::max(1, in / 32), splits = both ? 1 : static_cast<int>(std::min<long>(most, std::max(1L, (want + 2 * strips - 1) / (2 * strips))));
  const int rows_s = ceil_div(in, splits), used = ceil_div(in, rows_s);
  const size_t part = static_cast<size_t>(batch) * 2 * hidden;
  EpiGate<T> epi{h, z, b, nullptr, batch, hidden, hidden, act};
  if (!both) {
    TDH_TRY(ws_begin(ws_align(4 * part * used)));
    TDH_TRY(take(part * used, &epi.partial));
  }
  const bool once = bytes > FEW_ONCE_BYTES;
  TDH_TRY(with_rows(batch, [&](auto rows) {
    constexpr int M = decltype(rows)::value;
    ProfScope prof("gated_ff_few_fwd", static_cast<double>(bytes), WORK_BYTE);
    auto go = [&](auto kernel) {
      TDH_LAUNCH(kernel, dim3(both ? strips : 2 * strips * used), dim3(FEW_NT), 0, ctx().stream, x, w, epi, in, strips, rows_s);
      TDH_LAUNCH_CHECK();
      return static_cast<int>(TDH_OK);
    };
    if (both) return wide ? go(few_fwd_kernel<T, M, 64, true, false>) : go(few_fwd_kernel<T, M, 16, true, false>);
    if (!wide) return go(few_fwd_kernel<T, M, 16, false, false>);
    return once ? go(few_fwd_kernel<T, M, 64, false, true>) : go(few_fwd_kernel<T, M, 64, false, false>);
  }));
  return both ? static_cast<int>(TDH_OK) : launch_gate_reduce(epi, used);
}

template <class T>
int few_bwd(int act, int in, int hidden, int batch, const T *x, const T *w, const float *z, const T *dh, T *dx, T *dw, T *db,
            int accumulate) {
  const int cols = 2 * hidden;
  const DzPlan pz = dz_plan<T>(hidden, batch, db != nullptr);
  TDH_TRY(ws_begin(ws_align(sizeof(float) * batch * cols) + ws_align(4 * static_cast<size_t>(pz.bands) * cols)));
  float *dz = nullptr, *bias_part = nullptr;
  if (dx || dw) TDH_TRY(take(static_cast<size_t>(batch) * cols, &dz));
  if (db) TDH_TRY(take(static_cast<size_t>(pz.bands) * cols, &bias_part));
  TDH_TRY(launch_dz(pz, act, hidden, hidden, batch, z, dh, dz, bias_part));
  if (db) TDH_TRY(launch_db(bias_part, db, pz.bands, hidden, accumulate));
  if (!dx && !dw) return TDH_OK;
  ProfScope prof("gated_ff_few_bwd", sizeof(T) * static_cast<double>(in) * cols * ((dx ? 1 : 0) + (dw ? 1 : 0)), WORK_BYTE);
  return with_rows(batch, [&](auto rows) {
    constexpr int M = decltype(rows)::value;
    auto go = [&](auto kernel) {
      TDH_LAUNCH(kernel, dim3(ceil_div(in, FEW_I)), dim3(256), 0, ctx().stream, x, w, dz, dx, dw, in, cols, batch, accumulate);
      TDH_LAUNCH_CHECK();
      return static_cast<int>(TDH_OK);
    };
    return sizeof(T) * static_cast<size_t>(in) * cols > FEW_ONCE_BYTES ? go(few_bwd_kernel<T, M, true>) : go(few_bwd_kernel<T, M, false>);
  });
}

// ---- plans
// A tile shape: the workgroups that a compute unit holds, us of a tile of 64 reduction indices with one, two, ... of them on a
// compute unit (all of them take that long), us of a round of workgroups beside that, and of the launch. Measured on
// products of 256 to 1024 tiles with k of 64 to 2048; 256 x 256 reaches 1100 TFLOP/s there, 128 x 128 990, 64 x 128 760,
// 64 x 64 650, 32 x 256 620.
struct FfTile {
  int bm, bn, bufs, per_cu;
  double us[4], round_us, launch_us;
};
constexpr FfTile FF_TILES[] = {{256, 256, 2, 1, {1.65}, 5.0, 5.0},
                               {128, 128, 2, 2, {0.77, 0.92}, 3.0, 3.0},
                               {64, 128, 3, 2, {0.39, 0.64}, 1.7, 2.5},
                               {64, 64, 2, 4, {0.37, 0.45, 0.60, 0.78}, 1.0, 2.7},
                               {32, 256, 2, 2, {0.80, 0.78}, 2.0, 2.5}};

// The tile shape and the split along k that take the least by these figures, round of workgroups by round. What a round reads
// comes no faster than the bytes in flight allow: 3.3 TB/s with 3.5 MB of them, 4.5 with 7, 5.4 with 14 and more
// (a product of 32 rows with 200 MB of weights, 32 x 256: 78 us unsplit, 39 in 5 slices that are just resident, 50 in
// 11), and of rows of 64 or 128 bytes 0.4 or 0.6 of that (pair: an unsplit tile takes half of its columns from either half of
// the matrix; the product above, 64 x 128: 64 us, 39 if its columns lie together). A split's slices are written and
// read once and its sum is another launch.
}  // namespace
FfPlan ff_plan(int M, int N, int K, bool pair) {
  const long cus    = ctx().compute_units > 0 ? ctx().compute_units : 256;
  const int ktiles  = std::max(1, ceil_div(K, G16_BK));
  const double read = 2.0 * (static_cast<double>(M) + N) * K;
  FfPlan best{0, 1, ktiles * G16_BK};
  double best_us = 1e30;
  for (int c = 0; c < 5; ++c) {
    const FfTile &t  = FF_TILES[c];
    const long tiles = static_cast<long>(ceil_div(M, t.bm)) * ceil_div(N, t.bn), slots = cus * t.per_cu;
    int last = 0;
    for (int want = 1; want <= 64 && want <= ktiles; want += want < 8 ? 1 : want / 4) {
      const int per = ceil_div(ktiles, want), splits = ceil_div(ktiles, per);
      if (splits == last) continue;
      last = splits;
      const long groups = tiles * splits;
      auto round = [&](long n) {
        const double flight = n * (t.bufs - 1) * (t.bm + t.bn) * 128.0, scatter = !pair || splits > 1 || t.bn >= 256 ? 1.0 : t.bn == 128 ? 0.6 : 0.4,
                     speed = scatter * std::min(5.4e6, 7.0e6 * flight / (flight + 4e6));
        return std::max(per * t.us[(n - 1) / cus], read * n / groups / speed) + t.round_us;
      };
      double us = t.launch_us + (groups / slots) * round(slots);
      if (groups % slots) us += round(groups % slots);
      if (splits > 1) us += 3.0 + 8.0 * splits * M * N / 8e6;
      if (us < best_us) {
        best_us = us;
        best    = FfPlan{c, splits, per * G16_BK};
      }
    }
  }
  return best;
}
namespace {
size_t ff_partial_bytes(const FfPlan &p, size_t elements) { return p.splits > 1 ? ws_align(4 * p.splits * elements) : 0; }

// N: the columns of B in use (PAIR: both halves)
template <class T, bool A_KC, bool B_KC, bool PAIR, class Epi>
int ff_gemm(const FfPlan &p, const G16Matrix &A, const G16Matrix &B, const Epi &epi, int M, int N, int K, const char *tag) {
  ProfScope prof(tag, M, N, K);
  const FfTile &t   = FF_TILES[p.cfg];
  const int tiles_m = ceil_div(M, t.bm), tiles_n = PAIR ? ceil_div(N / 2, t.bn / 2) : ceil_div(N, t.bn);
  const dim3 grid(static_cast<unsigned>(tiles_m) * tiles_n * p.splits);
  auto go = [&](auto kernel, int threads) {
    TDH_LAUNCH(kernel, grid, dim3(threads), 0, ctx().stream, A, B, epi, tiles_m, tiles_n, K, p.k_per_split);
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  };
  switch (p.cfg) {
    case 0: return go(gemm16_kernel<T, 2, 4, 4, 2, 2, A_KC, B_KC, PAIR, Epi>, 512);
    case 1: return go(gemm16_kernel<T, 2, 2, 2, 2, 2, A_KC, B_KC, PAIR, Epi>, 256);
    case 2: return go(gemm16_kernel<T, 2, 2, 1, 2, 3, A_KC, B_KC, PAIR, Epi>, 256);
    case 3: return go(gemm16_kernel<T, 2, 1, 1, 2, 2, A_KC, B_KC, PAIR, Epi>, 128);
    default: return go(gemm16_kernel<T, 1, 4, 1, 2, 2, A_KC, B_KC, PAIR, Epi>, 256);
  }
}

// `src` as the products read it: itself where it lies on 16-byte boundaries, else a padded copy out of the scratch
int padded(int n) { return (n + 7) & ~7; }
template <class T>
bool fits(const T *p, int cols) { return cols % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
template <class T>
size_t pack_bytes(const T *p, int rows, int used, int halves) {
  return fits(p, used) ? 0 : ws_align(static_cast<size_t>(rows) * halves * padded(used) * sizeof(T));
}
template <class T>
struct Packer {
  PackJobs<T> jobs{};
  int n = 0;
  // notes the copy, if one is needed; run() makes them all
  int add(const T *src, int rows, int used, int halves, G16Matrix *out) {
    const int half = padded(used);
    *out = G16Matrix{src, static_cast<long>(halves) * half, rows, halves * half};
    if (fits(src, used)) return TDH_OK;
    typename PackJobs<T>::Job &j = jobs.job[n++];
    j = {src, nullptr, used, half, halves, 0, static_cast<size_t>(rows) * halves * half / 8};
    j.blocks = static_cast<unsigned>(ceil_div_sz(j.words, GF_NT));
    TDH_TRY(take(j.words * 8, &j.dst));
    out->p = j.dst;
    return TDH_OK;
  }
  int run() {
    if (!n) return TDH_OK;
    const size_t words = jobs.job[0].words + jobs.job[1].words;
    ProfScope prof("ff_pack", 32.0 * words, WORK_BYTE);
    TDH_LAUNCH((pack_kernel<T>), dim3(jobs.job[0].blocks + jobs.job[1].blocks), dim3(GF_NT), 0, ctx().stream, jobs);
    TDH_LAUNCH_CHECK();
    return TDH_OK;
  }
};

template <class T>
int ff_fwd_16(int act, int in, int hidden, int batch, const T *x, const T *w, const T *b, T *h, float *z) {
  const int half    = padded(hidden);
  const FfPlan plan = ff_plan(batch, 2 * half, in, /*pair=*/true);
  const size_t part = static_cast<size_t>(batch) * 2 * half;
  TDH_TRY(ws_begin(pack_bytes(x, batch, in, 1) + pack_bytes(w, in, hidden, 2) + ff_partial_bytes(plan, part)));
  G16Matrix A, B;
  Packer<T> packer;
  TDH_TRY(packer.add(x, batch, in, 1, &A));
  TDH_TRY(packer.add(w, in, hidden, 2, &B));
  TDH_TRY(packer.run());
  EpiGate<T> epi{h, z, b, nullptr, batch, hidden, half, act};
  if (plan.splits == 1) return ff_gemm<T, true, false, true>(plan, A, B, epi, batch, 2 * half, in, "gated_ff_fwd");
  TDH_TRY(take(plan.splits * part, &epi.partial));
  const EpiGrad<T> slices{nullptr, epi.partial, batch, 2 * half, hidden, half, 0};
  TDH_TRY((ff_gemm<T, true, false, false>(plan, A, B, slices, batch, 2 * half, in, "gated_ff_fwd")));
  return launch_gate_reduce(epi, plan.splits);
}

template <class T, bool A_KC, bool B_KC>
int ff_grad(const FfPlan &plan, const G16Matrix &A, const G16Matrix &B, EpiGrad<T> epi, int K, const char *tag) {
  if (plan.splits > 1) TDH_TRY(take(plan.splits * static_cast<size_t>(epi.rows) * epi.cols, &epi.partial));
  TDH_TRY((ff_gemm<T, A_KC, B_KC, false>(plan, A, B, epi, epi.rows, epi.cols, K, tag)));
  return plan.splits > 1 ? launch_grad_reduce(epi, plan.splits) : static_cast<int>(TDH_OK);
}

template <class T>
int ff_bwd_16(int act, int in, int hidden, int batch, const T *x, const T *w, const float *z, const T *dh, T *dx, T *dw, T *db,
              int accumulate) {
  const int half = padded(hidden);
  const DzPlan pz = dz_plan<T>(half, batch, db != nullptr);
  const int bands = pz.bands;
  const FfPlan px = ff_plan(batch, in, 2 * half, false), pw = ff_plan(in, 2 * half, batch, false);
  const size_t nx = static_cast<size_t>(batch) * in, nw = static_cast<size_t>(in) * 2 * half;
  const bool scaled = std::is_same<T, f16>::value && (dx || dw);
  const DzPlan pp   = dz_peak_plan<T>(hidden, batch);
  DzPeaks peaks{nullptr, pp.blocks_n * pp.bands, nullptr};
  TDH_TRY(ws_begin((scaled ? ws_align(4 * (static_cast<size_t>(peaks.n) + 1)) : 0) +
                   ws_align(sizeof(T) * batch * 2 * half) + ws_align(4 * static_cast<size_t>(bands) * 2 * hidden) +
                   (dx ? pack_bytes(w, in, hidden, 2) + ff_partial_bytes(px, nx) : 0) +
                   (dw ? pack_bytes(x, batch, in, 1) + ff_partial_bytes(pw, nw) : 0)));
  T *dz = nullptr;
  float *bias_part = nullptr;
  if (dx || dw) TDH_TRY(take(static_cast<size_t>(batch) * 2 * half, &dz));
  if (db) TDH_TRY(take(static_cast<size_t>(bands) * 2 * hidden, &bias_part));
  if (scaled) {
    float *p = nullptr;
    TDH_TRY(take(static_cast<size_t>(peaks.n) + 1, &p));
    peaks.peaks   = p;
    peaks.unscale = p + peaks.n;
    TDH_TRY(launch_dz_peak(pp, act, hidden, batch, z, dh, p));
  }
  TDH_TRY(launch_dz(pz, act, hidden, half, batch, z, dh, dz, bias_part, peaks));
  if (db) TDH_TRY(launch_db(bias_part, db, bands, hidden, accumulate));
  const G16Matrix Z{dz, 2L * half, batch, 2 * half};
  G16Matrix W, X;   // w: [in][2 half], of which the rows are the product's columns
  Packer<T> packer;
  if (dx) TDH_TRY(packer.add(w, in, hidden, 2, &W));
  if (dw) TDH_TRY(packer.add(x, batch, in, 1, &X));
  TDH_TRY(packer.run());
  if (dx) {
    TDH_TRY((ff_grad<T, true, true>(px, Z, W, EpiGrad<T>{dx, nullptr, batch, in, in, in, 0, peaks.unscale}, 2 * half, "gated_ff_dx")));
  }
  if (dw) {
    TDH_TRY((ff_grad<T, false, false>(pw, X, Z, EpiGrad<T>{dw, nullptr, in, 2 * half, hidden, half, accumulate, peaks.unscale}, batch, "gated_ff_dw")));
  }
  return TDH_OK;
}

// ------------------------------------------------------------------- fp32
// Products of many samples on operands that are split in three parts by a pass of their own (gemm_x3.h); the others are the
// fully-connected layer's.

// fp32 matrices to their three planes, a thread eight neighbours. sign: 1 turns every other group of 32 rows, 2 of columns.
// Bound by memory, 4 bytes in and 6 out (1344 -> 2 x 2640 and 2000 samples, three launches of a step: 54 us, 5.6 TB/s). A pass of its own:
// within a product the split would be made again by every tile that reads the element, on the vector units beside its products.
// Columns come in one or two halves of `used` values, `half` (a multiple of 8) apart in the planes, zero behind a half.
struct SplitJobs {
  struct Job {
    const float *src;
    uint16_t *dst;   // planes, 8 * words elements each
    int used, half, halves, sign;
    unsigned blocks;
    size_t words;    // of eight elements
  } job[2];
};
__global__ void __launch_bounds__(GF_NT)
split_kernel(const SplitJobs jobs) {
  const bool second = blockIdx.x >= jobs.job[0].blocks;
  const SplitJobs::Job &j = jobs.job[second];
  const size_t i = static_cast<size_t>(blockIdx.x - (second ? jobs.job[0].blocks : 0)) * GF_NT + threadIdx.x;
  if (i >= j.words) return;
  const int per = j.half / 8;   // words of a half
  const size_t row = i / (per * j.halves);
  const int col = static_cast<int>(i - row * (per * j.halves)) * 8, h = col >= j.half ? 1 : 0, c0 = col - h * j.half;
  const bool turn  = j.sign == 1 ? (row / X3P_BK) & 1 : j.sign == 2 ? (col / X3P_BK) & 1 : false;
  const float scale = turn ? -X3_SCALE : X3_SCALE;
  const float *p = j.src + (row * j.halves + h) * j.used + c0;
  float v[8];
  if (c0 + 8 <= j.used) {
    load8(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c0 + e < j.used ? p[e] : 0.0f;
  }
  uint4 out[X3_PARTS];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t part[X3_PARTS];
    split_pair(scale * v[2 * c], scale * v[2 * c + 1], part);
#pragma unroll
    for (int q = 0; q < X3_PARTS; ++q) (&out[q].x)[c] = part[q];
  }
#pragma unroll
  for (int q = 0; q < X3_PARTS; ++q) reinterpret_cast<uint4 *>(j.dst)[q * j.words + i] = out[q];
}
struct Splitter {
  SplitJobs jobs{};
  int n = 0;
  static size_t bytes(size_t rows, int used, int halves) { return ws_align(6 * rows * halves * padded(used)); }
  int add(const float *src, int rows, int used, int halves, int sign, G16Matrix *out) {
    const int half = padded(used);
    SplitJobs::Job &j = jobs.job[n++];
    j = {src, nullptr, used, half, halves, sign, 0, static_cast<size_t>(rows) * halves * half / 8};
    j.blocks = static_cast<unsigned>(ceil_div_sz(j.words, GF_NT));
    TDH_TRY(take(j.words * 24, &j.dst));
    *out = G16Matrix{j.dst, static_cast<long>(halves) * half, rows, halves * half};
    return TDH_OK;
  }
  int run() {
    const size_t words = jobs.job[0].words + jobs.job[1].words;
    ProfScope prof("ff_split", 80.0 * words, WORK_BYTE);
    TDH_LAUNCH(split_kernel, dim3(jobs.job[0].blocks + jobs.job[1].blocks), dim3(GF_NT), 0, ctx().stream, jobs);
    TDH_LAUNCH_CHECK();
    return TDH_OK;
  }
};

// Tiles of 128 x 128, split along k where they do not fill the compute units: 2.55 us a tile of 32 indices with two workgroups a
// compute unit, 2.3 with one (whose loads nothing covers), and 5 a round.
constexpr int X3P_TILE = 128;
FfPlan x3_plan(int M, int N, int K) {
  const long cus   = ctx().compute_units > 0 ? ctx().compute_units : 256, tiles = static_cast<long>(ceil_div(M, X3P_TILE)) * ceil_div(N, X3P_TILE);
  const int ktiles = std::max(1, ceil_div(K, X3P_BK));
  FfPlan best{0, 1, ktiles * X3P_BK};
  double best_us = 1e30;
  for (int want = 1; want <= 16 && want <= ktiles; ++want) {
    const int per = ceil_div(ktiles, want), splits = ceil_div(ktiles, per);
    const long groups = tiles * splits, rest = groups % (2 * cus);
    double us = static_cast<double>(groups / (2 * cus)) * (per * 2.55 + 5.0);
    if (rest) us += per * (rest > cus ? 2.55 : 2.3) + 5.0;
    if (splits > 1) us += 3.0 + 8.0 * splits * M * N / 8e6;
    if (us < best_us) {
      best_us = us;
      best    = FfPlan{0, splits, per * X3P_BK};
    }
  }
  return best;
}
template <bool A_KC, bool B_KC, bool PAIR, bool ON_THE_WAY, class Epi>
int x3_gemm(const FfPlan &p, const G16Matrix &A, const G16Matrix &B, const X3Source &src, const Epi &epi, int K, const char *tag) {
  ProfScope prof(tag, src.rows, src.cols, K);
  const int tiles_m = ceil_div(src.rows, X3P_TILE), tiles_n = PAIR ? ceil_div(src.cols / 2, X3P_TILE / 2) : ceil_div(src.cols, X3P_TILE);
  TDH_LAUNCH((gemm_x3_kernel<A_KC, B_KC, PAIR, ON_THE_WAY, Epi>), dim3(static_cast<unsigned>(tiles_m) * tiles_n * p.splits), dim3(256), 0,
             ctx().stream, A, B, static_cast<long>(A.rows) * A.cols, static_cast<long>(B.rows) * B.cols, src, epi, tiles_m, tiles_n, K,
             p.k_per_split);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}
template <bool A_KC, bool B_KC, bool ON_THE_WAY>
int x3_grad(const G16Matrix &A, const G16Matrix &B, const X3Source &src, EpiGrad<float> epi, int K, const char *tag) {
  const FfPlan plan  = x3_plan(src.rows, src.cols, K);
  const size_t total = static_cast<size_t>(src.rows) * src.cols;
  if (plan.splits > 1) TDH_TRY(take(plan.splits * total, &epi.partial));
  TDH_TRY((x3_gemm<A_KC, B_KC, false, ON_THE_WAY>(plan, A, B, src, epi, K, tag)));
  return plan.splits > 1 ? launch_grad_reduce(epi, plan.splits) : static_cast<int>(TDH_OK);
}

// Whether the weights' planes pay for themselves (they are made anew in every call), and whether those of x and dz do: the pass that
// writes planes grows with in + 2 hidden, what the product gains by them with in * hidden. us of a training step with all three products
// on planes, dW alone, and none (the fully-connected layer's products): 1024 -> 2 x 2048, 256 samples 105 / 95 / 104, 1200 266 / 266 /
// 262, 4000 658 / 695 / 686; 1344 -> 2 x 2640, 200 samples 135 / 110 / 129, 2000 632 / 652 / 654; 4096 -> 2 x 4096, 256 samples 472 / 358 /
// 396; 2000 -> 2 x 200, 8000 samples 378 / 363 / 344; 128 -> 2 x 2000, 20000 samples 818 / 945 / 798.
// Sizes that are no multiple of four the layer's own three-part products do not take, and its others read element by element: 1023 ->
// 2 x 2047, 128 samples 85 / - / 79, 200 105 / - / 122, 801 202 / - / 377; 4097 -> 2 x 4099, 33 samples 227 / - / 198, 65 244 / - / 330, 257 543 / -
// / 1034; 331 -> 2 x 333, 1501 samples 85 / 96 / 98; 61 -> 2 x 1999, 20001 samples 838 / 962 / 895; 1999 -> 2 x 50 505 / 520 / 493, 2 x 61 496 /
// 563 / 550.
constexpr int X3P_BATCH = 2000, X3P_DW_BATCH = 128, X3P_BATCH_ODD = 160, X3P_BATCH_ODD_LARGE = 65, X3P_SIZE = 400, X3P_SIZE_ODD = 40;
constexpr double X3P_FLOP = 6e8, X3P_FLOP_LARGE = 4e9;   // below the first the products are short
bool x3_pays(int in, int hidden, int batch, int from) {
  const bool odd    = batch % 4 || in % 4 || hidden % 2;
  const double flop = 4.0 * batch * in * hidden;
  return batch >= (!odd ? from : flop >= X3P_FLOP_LARGE ? X3P_BATCH_ODD_LARGE : X3P_BATCH_ODD) && flop >= X3P_FLOP &&
         static_cast<double>(in) * hidden >= (odd ? X3P_SIZE_ODD : X3P_SIZE) * (in + 2.0 * hidden);
}
// Up to so many samples few tiles read a weight, and the forward product and dX split it on the way into LDS: 4097 -> 2 x 4099, 257
// samples 543, with planes 598; 701 -> 2 x 703, 501 samples 87 / 91; 1023 -> 2 x 2047, 801 samples 215 / 202.
constexpr int X3P_ON_THE_WAY = 512;
bool x3_weights(int in, int hidden, int batch) { return x3_pays(in, hidden, batch, X3P_BATCH); }
bool x3_dw(int in, int hidden, int batch) { return x3_pays(in, hidden, batch, X3P_DW_BATCH); }

constexpr int FF_OWN_DB = 512;
int ff_fwd_f32(int act, int in, int hidden, int batch, const float *x, const float *w, const float *b, float *h, float *z) {
  const size_t nz = static_cast<size_t>(batch) * 2 * hidden;
  if (x3_weights(in, hidden, batch)) {
    const int half    = padded(hidden);
    const size_t part = static_cast<size_t>(batch) * 2 * half;
    const FfPlan plan = x3_plan(batch, 2 * half, in);
    const bool way    = batch <= X3P_ON_THE_WAY;
    TDH_TRY(ws_begin(Splitter::bytes(batch, in, 1) + (way ? 0 : Splitter::bytes(in, hidden, 2)) + ff_partial_bytes(plan, part)));
    Splitter split;
    G16Matrix X, W{};
    TDH_TRY(split.add(x, batch, in, 1, way ? 0 : 2, &X));
    if (!way) TDH_TRY(split.add(w, in, hidden, 2, 0, &W));
    TDH_TRY(split.run());
    const X3Source src{x, w, in, 1, 2L * hidden, 1, batch, 2 * half, {in, in}, {hidden, half}};
    EpiGate<float> epi{h, z, b, nullptr, batch, hidden, half, act};
    if (plan.splits == 1)
      return way ? x3_gemm<true, false, true, true>(plan, X, W, src, epi, in, "gated_ff_fwd_x3")
                 : x3_gemm<true, false, true, false>(plan, X, W, src, epi, in, "gated_ff_fwd_x3");
    TDH_TRY(take(plan.splits * part, &epi.partial));
    const EpiGrad<float> slices{nullptr, epi.partial, batch, 2 * half, hidden, half, 0};
    if (way)
      TDH_TRY((x3_gemm<true, false, false, true>(plan, X, W, src, slices, in, "gated_ff_fwd_x3")));
    else
      TDH_TRY((x3_gemm<true, false, false, false>(plan, X, W, src, slices, in, "gated_ff_fwd_x3")));
    return launch_gate_reduce(epi, plan.splits);
  }
  TDH_TRY(ws_begin(fc_workspace_bytes(in, 2 * hidden, batch) + (z ? 0 : ws_align(4 * nz))));
  if (!z) TDH_TRY(take(nz, &z));
  TDH_TRY(fc_fwd(in, 2 * hidden, b != nullptr, batch, x, w, b, z));
  const size_t total = nz / 2;
  ProfScope prof("gate_fwd", 12.0 * total, WORK_BYTE);
  TDH_LAUNCH(gate_fwd_kernel, dim3(static_cast<unsigned>(ceil_div_sz(total, GF_NT))), dim3(GF_NT), 0, ctx().stream, z, h, hidden, total, act);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}
int ff_bwd_f32(int act, int in, int hidden, int batch, const float *x, const float *w, const float *z, const float *dh, float *dx,
               float *dw, float *db, int accumulate) {
  const int cols = 2 * hidden, half = padded(hidden);
  const bool planes_x = dx && x3_weights(in, hidden, batch), planes_w = dw && x3_dw(in, hidden, batch), way = batch <= X3P_ON_THE_WAY;
  // db by the bands of the dz pass, 4 us; without planes the layer's column sums, which ride along with dw's launch or take 5 us at
  // 500 samples, 24 at 4000, 540 at 100000
  const bool own_db   = db && (planes_w || batch > FF_OWN_DB);
  const DzPlan pz     = dz_plan<float>(hidden, batch, own_db);
  const size_t nz = static_cast<size_t>(batch) * cols, nx = static_cast<size_t>(batch) * in, nw = static_cast<size_t>(in) * 2 * half;
  TDH_TRY(ws_begin(ws_align(4 * nz) + (own_db ? ws_align(4 * static_cast<size_t>(pz.bands) * cols) : 0) +
                   (planes_x || planes_w ? Splitter::bytes(batch, hidden, 2) : 0) +
                   (planes_x ? (way ? 0 : Splitter::bytes(in, hidden, 2)) + ff_partial_bytes(x3_plan(batch, in, 2 * half), nx) : 0) +
                   (planes_w ? Splitter::bytes(batch, in, 1) + ff_partial_bytes(x3_plan(in, 2 * half, batch), nw) : 0) +
                   (planes_x && planes_w ? 0 : fc_workspace_bytes(in, cols, batch))));
  float *dz = nullptr, *bias_part = nullptr;
  TDH_TRY(take(nz, &dz));
  if (own_db) TDH_TRY(take(static_cast<size_t>(pz.bands) * cols, &bias_part));
  TDH_TRY(launch_dz(pz, act, hidden, hidden, batch, z, dh, dz, bias_part));
  if (own_db) TDH_TRY(launch_db(bias_part, db, pz.bands, hidden, accumulate));
  if (planes_x || planes_w) {
    G16Matrix Z, X, W{};
    Splitter split, weights;
    TDH_TRY(split.add(dz, batch, hidden, 2, 0, &Z));
    if (planes_w) TDH_TRY(split.add(x, batch, in, 1, 1, &X));
    TDH_TRY(split.run());
    if (planes_w)
      TDH_TRY((x3_grad<false, false, false>(X, Z, X3Source{x, dz, 1, in, cols, 1, in, 2 * half, {batch, batch}, {hidden, half}},
                                     EpiGrad<float>{dw, nullptr, in, 2 * half, hidden, half, accumulate}, batch, "gated_ff_dw_x3")));
    if (planes_x) {
      const X3Source src{dz, w, cols, 1, 1, cols, batch, in, {hidden, half}, {in, in}};
      const EpiGrad<float> epi{dx, nullptr, batch, in, in, in, 0};
      if (way) {
        TDH_TRY((x3_grad<true, true, true>(Z, W, src, epi, 2 * half, "gated_ff_dx_x3")));
      } else {
        TDH_TRY(weights.add(w, in, hidden, 2, 2, &W));
        TDH_TRY(weights.run());
        TDH_TRY((x3_grad<true, true, false>(Z, W, src, epi, 2 * half, "gated_ff_dx_x3")));
      }
    }
  }
  if ((dx && !planes_x) || (dw && !planes_w) || (db && !own_db))
    return fc_bwd(in, cols, db && !own_db, batch, x, w, dz, planes_x ? nullptr : dx, planes_w ? nullptr : dw, own_db ? nullptr : db,
                  accumulate, ActGrad());
  return TDH_OK;
}

// the gradients of no samples
template <class T>
int no_rows(int in, int hidden, T *dw, T *db) {
  if (dw) TDH_TRY(launch_grad_reduce(EpiGrad<T>{dw, nullptr, in, 2 * hidden, hidden, hidden, 0}, 0));
  return db ? launch_db<T>(nullptr, db, 0, hidden, 0) : static_cast<int>(TDH_OK);
}

int check_ff(const char *who, int dtype, int act, int in, int hidden, int batch) {
  TDH_CHECK_ARG(dtype_known(dtype), "%s: element type %d", who, dtype);
  TDH_CHECK_ARG(act >= TDH_GATE_SILU && act <= TDH_GATE_NONE, "%s: gate activation %d", who, act);
  TDH_CHECK_ARG(in > 0 && hidden > 0 && batch >= 0, "%s: bad shape %d->2*%d batch %d", who, in, hidden, batch);
  TDH_CHECK_ARG(2L * in * hidden < (1L << 31) && static_cast<long>(batch) * in < (1L << 31) && 2L * batch * hidden < (1L << 31),
                "%s: tensor exceeds 2^31 elements", who);
  // (offsets within a tile of 256 rows are 32 bits, a launch has fewer than 2^24 workgroups, and the fully-connected layer's products,
  // in fp32, fewer than 2^16 tiles of rows)
  const int most = dtype == TDH_F32 ? 1 << 20 : 1 << 24;
  TDH_CHECK_ARG(in <= (1 << 21) && hidden <= (1 << 20) && batch <= most, "%s: %d->2*%d batch %d is beyond 2^21->2*2^20 batch %d", who,
                in, hidden, batch, most);
  return TDH_OK;
}
int check_aligned(const char *who, int dtype, std::initializer_list<const void *> tensors) {
  for (const void *p : tensors)
    TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) == 0, "%s: a tensor that is not aligned to its elements", who);
  return TDH_OK;
}

}  // namespace
}  // namespace tdh

using namespace tdh;

extern "C" {

int tdh_gated_ff_fwd(int dtype, int act, int in, int hidden, int has_bias, int batch, const void *x, const void *w,
                     const void *b, void *h, float *z) {
  TDH_TRY(check_ff("tdh_gated_ff_fwd", dtype, act, in, hidden, batch));
  TDH_CHECK_ARG(batch == 0 || (x && w && h), "tdh_gated_ff_fwd: null tensor");
  TDH_CHECK_ARG(batch == 0 || !has_bias || b, "tdh_gated_ff_fwd: has_bias set but b is null");
  TDH_TRY(check_aligned("tdh_gated_ff_fwd", dtype, {x, w, b, h}));
  TDH_TRY(check_aligned("tdh_gated_ff_fwd", TDH_F32, {z}));
  const size_t e = dtype_size(dtype), nx = static_cast<size_t>(batch) * in, nh = static_cast<size_t>(batch) * hidden, nw = 2 * static_cast<size_t>(in) * hidden;
  TDH_TRY(check_apart("tdh_gated_ff_fwd", {{h, e * nh}, {z, 8 * nh}}, {{x, e * nx}, {w, e * nw}, {has_bias ? b : nullptr, 2 * e * hidden}}));
  TDH_REQUIRE_INIT();
  if (batch == 0) return TDH_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T *xt = static_cast<const T *>(x), *wt = static_cast<const T *>(w), *bt = has_bias ? static_cast<const T *>(b) : nullptr;
    if (batch <= FEW_ROWS) return few_fwd<T>(act, in, hidden, batch, xt, wt, bt, static_cast<T *>(h), z);
    if constexpr (sizeof(T) == 4)
      return ff_fwd_f32(act, in, hidden, batch, xt, wt, bt, static_cast<T *>(h), z);
    else
      return ff_fwd_16<T>(act, in, hidden, batch, xt, wt, bt, static_cast<T *>(h), z);
  });
}

int tdh_gated_ff_bwd(int dtype, int act, int in, int hidden, int has_bias, int batch, const void *x, const void *w,
                     const float *z, const void *dh, void *dx, void *dw, void *db, int accumulate) {
  TDH_TRY(check_ff("tdh_gated_ff_bwd", dtype, act, in, hidden, batch));
  TDH_CHECK_ARG(batch == 0 || (x && w && z && dh), "tdh_gated_ff_bwd: null tensor");
  TDH_TRY(check_aligned("tdh_gated_ff_bwd", dtype, {x, w, dh, dx, dw, db}));
  TDH_TRY(check_aligned("tdh_gated_ff_bwd", TDH_F32, {z}));
  const size_t e = dtype_size(dtype), nx = static_cast<size_t>(batch) * in, nh = static_cast<size_t>(batch) * hidden, nw = 2 * static_cast<size_t>(in) * hidden;
  TDH_TRY(check_apart("tdh_gated_ff_bwd", {{dx, e * nx}, {dw, e * nw}, {has_bias ? db : nullptr, 2 * e * hidden}},
                      {{x, e * nx}, {batch ? w : nullptr, e * nw}, {z, 8 * nh}, {dh, e * nh}}));
  TDH_REQUIRE_INIT();
  if (batch == 0 && accumulate) return TDH_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T *xt = static_cast<const T *>(x), *wt = static_cast<const T *>(w), *dt = static_cast<const T *>(dh);
    T *dbt = has_bias ? static_cast<T *>(db) : nullptr;
    if (batch == 0) return no_rows<T>(in, hidden, static_cast<T *>(dw), dbt);
    if (batch <= FEW_ROWS) return few_bwd<T>(act, in, hidden, batch, xt, wt, z, dt, static_cast<T *>(dx), static_cast<T *>(dw), dbt, accumulate);
    if constexpr (sizeof(T) == 4)
      return ff_bwd_f32(act, in, hidden, batch, xt, wt, z, dt, static_cast<T *>(dx), static_cast<T *>(dw), dbt, accumulate);
    else
      return ff_bwd_16<T>(act, in, hidden, batch, xt, wt, z, dt, static_cast<T *>(dx), static_cast<T *>(dw), dbt, accumulate);
  });
}

int tdh_cast(int dst_dtype, int src_dtype, size_t n, const void *src, void *dst) {
  TDH_CHECK_ARG(dtype_known(dst_dtype) && dtype_known(src_dtype), "tdh_cast: element type %d to %d", src_dtype, dst_dtype);
  TDH_CHECK_ARG(n == 0 || (src && dst), "tdh_cast: null tensor");
  TDH_CHECK_ARG(n <= SIZE_MAX / 8, "tdh_cast: %zu elements", n);
  TDH_TRY(check_aligned("tdh_cast", src_dtype, {src}));
  TDH_TRY(check_aligned("tdh_cast", dst_dtype, {dst}));
  const uintptr_t s = reinterpret_cast<uintptr_t>(src), d = reinterpret_cast<uintptr_t>(dst);
  TDH_CHECK_ARG(s + n * dtype_size(src_dtype) <= d || d + n * dtype_size(dst_dtype) <= s, "tdh_cast: source and destination overlap");
  TDH_REQUIRE_INIT();
  if (n == 0) return TDH_OK;
  return with_dtype(dst_dtype, [&](auto to) {
    return with_dtype(src_dtype, [&](auto from) {
      using D = decltype(to);
      using S = decltype(from);
      return launch_cast<D, S>(static_cast<const S *>(src), static_cast<D *>(dst), n);
    });
  });
}

}  // extern "C"
