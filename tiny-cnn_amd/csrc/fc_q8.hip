// fc_q8.hip — a fully-connected layer whose weights are held in 8 bits with a scale for each output, and whose samples are brought to 8 bits with a scale
// for each sample.
//
//   scale = max |x| / 127, q = round(x / scale); y[m][n] = (sum_k q[m][k] wq[n][k]) scale[m] wscale[n] + b[n]
//
// The sum is one of whole numbers and exact (in up to 2^17: below 2^31), so it may be split and joined in any order.
//
//   up to Q8_FEW samples   one launch: every workgroup brings the samples to 8 bits for itself and streams its rows of weights through the vector
//                          units' four-fold products; bound by reading the weights with one sample; eight take three times as long
//   more                   a pass that writes q and the scales, and the products of gemm16.h, pairs of bytes in the place of 16-bit elements; the matrix
//                          units are busy for 53% of a long prompt's
//
// bf16, 4096 -> 12288: 1 sample 9.8 us with the same 50 MB of weights again and again, which the memory-side cache holds, 12.3 with eight such matrices in turns, 4.1 TB/s. In
// the same order 2 samples 13.1 and 15.7, 4 19.4 and 21.8, 8 30.9 and 33.0; the other way 9 samples 18.1 and 20.3, 16 17.3 and 19.7, 64 20.5 and 25.1, so the border is too far up
// for this layer. 4096 samples 13.8 us and 201 us, 2050 TOPS (tiles of 256 x 256; of 128 x 128 225 us). Packing, which reads w twice: 129 and 169 of bf16, 127 and 170 of fp32.
#include "gemm16.h"

#include <cfloat>

namespace tdh {

namespace {

// q of eight values and a scale, as packed bytes. The quotient is fp32's, rounded to nearest, ties to even, as the product's definition has it; a product with
// the reciprocal is within 2^-15 of it and rounds to the same number, unless it lies beside a half (one in some thousands), where it is
// divided. 4096 x 4096 in bf16: 13.8 us, all of them divided 15.3.
__device__ __forceinline__ uint2 quantized(const float (&v)[8], const float scale, const float inverse) {
  uint2 o = make_uint2(0, 0);
  if (!(scale > 0.0f)) return o;   // (all zero, or NaN)
  float r[8], near = scale < 0x1p-100f ? 1.0f : 0.0f;   // (whose reciprocal is no number, or has few figures)
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = v[e] * inverse;
    r[e] = __builtin_rintf(t);
    near = fmaxf(near, __builtin_fabsf(t - r[e]));
  }
  if (near > 0.4999f)
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = __builtin_rintf(v[e] / scale);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int q = static_cast<int>(__builtin_amdgcn_fmed3f(r[e], -127.0f, 127.0f));
    (&o.x)[e / 4] |= static_cast<uint32_t>(q & 255) << (8 * (e & 3));
  }
  return o;
}
// eight values of a row from k on, zero behind its `len` elements
template <class T>
__device__ __forceinline__ void row8(const T *p, const int k, const int len, float (&v)[8]) {
  if (k + 8 <= len) return load8(p + k, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = k + e < len ? to_f32(p[k + e]) : 0.0f;
}
// the larger, or NaN
__device__ __forceinline__ float most_of(const float a, const float b) { return a != a || b <= a ? a : b; }
__device__ __forceinline__ float most_of(const float (&v)[8], float most) {
#pragma unroll
  for (int e = 0; e < 8; ++e) most = most_of(most, __builtin_fabsf(v[e]));
  return most;
}
__device__ __forceinline__ float scale_of(const float most) { return most <= FLT_MAX ? most / 127.0f : __builtin_nanf(""); }

// A scale as f 2^e, f in [1/2, 1): a product of the two scales alone, or of one and the sum, may leave fp32's range where the result does not. NaN stays
// in f.
struct Scale {
  float f;
  int e;
};
__device__ __forceinline__ Scale scale_parts(const float s) { return Scale{__builtin_amdgcn_frexp_mantf(s), __builtin_amdgcn_frexp_expf(s)}; }
__device__ __forceinline__ float scaled(const int sum, const Scale s, const Scale w, const float b) {
  return __builtin_ldexpf(static_cast<float>(sum) * (s.f * w.f), s.e + w.e) + b;
}

// LANES lanes a row, W eights a lane in registers (W = 0: any number, the row is read twice)
template <class T, int LANES, int W>
__global__ void __launch_bounds__(256)
quantize_kernel(const T *__restrict__ x, int8_t *__restrict__ q, float *__restrict__ scale, const int rows, const int len, const int ld) {
  __shared__ float part[4];
  const int lane = threadIdx.x % LANES, eights = ld / 8;   // (those behind len are written as zeros)
  const long row = static_cast<long>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  const bool live = row < rows;
  const T *p = x + (live ? row : 0) * len;
  float held[W ? W : 1][8], most = 0.0f;
  if constexpr (W > 0) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (lane + i * LANES < eights) {
        row8(p, 8 * (lane + i * LANES), len, held[i]);
        most = most_of(held[i], most);
      }
  } else {
    for (int k = lane; k < eights; k += LANES) {
      float v[8];
      row8(p, 8 * k, len, v);
      most = most_of(v, most);
    }
  }
#pragma unroll
  for (int o = (LANES < 64 ? LANES : 64) / 2; o; o >>= 1) most = most_of(most, __shfl_xor(most, o));
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    most = most_of(most_of(part[0], part[1]), most_of(part[2], part[3]));
  }
  if (!live) return;
  const float s = scale_of(most), inverse = 1.0f / s;
  if (lane == 0) scale[row] = s;
  uint2 *out = reinterpret_cast<uint2 *>(q + row * ld);
  if constexpr (W > 0) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (lane + i * LANES < eights) out[lane + i * LANES] = quantized(held[i], s, inverse);
  } else {
    for (int k = lane; k < eights; k += LANES) {
      float v[8];
      row8(p, 8 * k, len, v);
      out[k] = quantized(v, s, inverse);
    }
  }
}
template <class T>
int launch_quantize(const T *x, int8_t *q, float *scale, int rows, int len, int ld) {
  ProfScope prof("q8_quantize", (sizeof(T) + 1.0) * rows * len, WORK_BYTE);
  auto go = [&](auto kernel, int lanes) {
    TDH_LAUNCH(kernel, dim3(ceil_div(rows, 256 / lanes)), dim3(256), 0, ctx().stream, x, q, scale, rows, len, ld);
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  };
  const int eights = ld / 8;
  if (eights <= 64) return go(quantize_kernel<T, 64, 1>, 64);
  if (eights <= 256) return go(quantize_kernel<T, 64, 4>, 64);
  if (eights <= 512 && rows > 1024) return go(quantize_kernel<T, 64, 8>, 64);
  if (eights <= 1024) return go(quantize_kernel<T, 256, 4>, 256);
  return go(quantize_kernel<T, 256, 0>, 256);
}

// --------------------------------------------------------------- many samples
template <class T>
struct EpiQ8 {
  T *y;
  const float *scale, *wscale;
  const T *bias;      // or null
  int *partial;       // slices instead, [split][rows][cols]
  int rows, cols;
  __device__ __forceinline__ float one(const int sum, const float s, const int n) const {
    return scaled(sum, scale_parts(s), scale_parts(wscale[n]), bias ? to_f32(bias[n]) : 0.0f);
  }
  template <int TM, int TN>
  __device__ __forceinline__ void done(const g16_f32x16 (&acc)[TM][TN], const int m0, const int n0, const int lane, const int split, float *lds) const {
    if (partial) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int m = m0 + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const int n = n0 + 32 * j + (lane & 31);
            if (m < rows && n < cols) partial[(static_cast<size_t>(split) * rows + m) * cols + n] = __float_as_int(acc[i][j][r]);
          }
        }
      return;
    }
    const G16Turn<32 * TN> turn{lds};
    // a lane has the same eight columns in all of its rows
    const int n = n0 + lane % (4 * TN) * 8;
    Scale w[8];
    float b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = min(n + e, cols - 1);
      w[e] = scale_parts(wscale[c]);
      b[e] = bias ? to_f32(bias[c]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) turn.put(lane, j, [&](int r) { return acc[i][j][r]; });
      turn.rows(lane, [&](int row, int, const float (&v)[8]) {
        const int m = m0 + 32 * i + row;
        if (m >= rows || n >= cols) return;
        const Scale s = scale_parts(scale[m]);
        T *p = y + static_cast<size_t>(m) * cols + n;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = scaled(__float_as_int(v[e]), s, w[e], b[e]);
        if (n + 8 <= cols) return store8(p, o);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < cols) p[e] = from_f32<T>(o[e]);
      });
    }
  }
};
template <class T>
__global__ void __launch_bounds__(256)
q8_reduce_kernel(const EpiQ8<T> epi, const int splits) {
  const size_t total = static_cast<size_t>(epi.rows) * epi.cols, i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int m = static_cast<int>(i / epi.cols), n = static_cast<int>(i - static_cast<size_t>(m) * epi.cols);
  int v = 0;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) v += epi.partial[s * total + i];
  epi.y[i] = from_f32<T>(epi.one(v, epi.scale[m], n));
}
template <class T>
int q8_many(int in, int out, int batch, const T *x, const int8_t *wq, const float *wscale, const T *b, T *y) {
  const int ld      = static_cast<int>(tdh_q8_row(in)), pairs = ld / 2;
  const FfPlan plan = ff_plan(batch, out, pairs, false);
  const size_t part = plan.splits > 1 ? static_cast<size_t>(plan.splits) * batch * out : 0;
  TDH_TRY(ws_begin(ws_align(static_cast<size_t>(batch) * ld) + ws_align(4 * static_cast<size_t>(batch)) + ws_align(4 * part)));
  void *q = nullptr, *scale = nullptr, *partial = nullptr;
  TDH_TRY(ws_take(static_cast<size_t>(batch) * ld, &q));
  TDH_TRY(ws_take(4 * static_cast<size_t>(batch), &scale));
  if (part) TDH_TRY(ws_take(4 * part, &partial));
  TDH_TRY(launch_quantize(x, static_cast<int8_t *>(q), static_cast<float *>(scale), batch, in, ld));
  const G16Matrix A{q, pairs, batch, pairs}, B{wq, pairs, out, pairs};
  using Epi = EpiQ8<T>;
  const Epi epi{y, static_cast<const float *>(scale), wscale, b, static_cast<int *>(partial), batch, out};
  {
    ProfScope prof("q8_product", batch, out, in);
    auto go = [&](auto kernel, int bm, int bn, int threads) {
      const int tm = ceil_div(batch, bm), tn = ceil_div(out, bn);
      TDH_LAUNCH(kernel, dim3(static_cast<unsigned>(tm) * tn * plan.splits), dim3(threads), 0, ctx().stream, A, B, epi, tm, tn, pairs, plan.k_per_split);
      TDH_LAUNCH_CHECK();
      return static_cast<int>(TDH_OK);
    };
    switch (plan.cfg) {
      case 0: TDH_TRY(go(gemm16_kernel<i8x2, 2, 4, 4, 2, 2, true, true, false, Epi>, 256, 256, 512)); break;
      case 1: TDH_TRY(go(gemm16_kernel<i8x2, 2, 2, 2, 2, 2, true, true, false, Epi>, 128, 128, 256)); break;
      case 2: TDH_TRY(go(gemm16_kernel<i8x2, 2, 2, 1, 2, 3, true, true, false, Epi>, 64, 128, 256)); break;
      case 3: TDH_TRY(go(gemm16_kernel<i8x2, 2, 1, 1, 2, 2, true, true, false, Epi>, 64, 64, 128)); break;
      default: TDH_TRY(go(gemm16_kernel<i8x2, 1, 4, 1, 2, 2, true, true, false, Epi>, 32, 256, 256)); break;
    }
  }
  if (!part) return TDH_OK;
  ProfScope prof("q8_reduce", 4.0 * part, WORK_BYTE);
  TDH_LAUNCH((q8_reduce_kernel<T>), dim3(static_cast<unsigned>(ceil_div_sz(static_cast<size_t>(batch) * out, 256))), dim3(256), 0, ctx().stream, epi,
             plan.splits);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

// ------------------------------------------------------------------ a few samples
constexpr int Q8_FEW = 8, Q8_FEW_BYTES = 48 << 10, Q8_NT = 512;
// the sum over a wave, in its last lane
__device__ __forceinline__ int last_lane_sum(int v) {
  auto add = [&](auto ctrl, auto rows) { v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false); };
  using I = std::integral_constant<int, 0xf>;
  add(std::integral_constant<int, 0x111>(), I());   // from 1, 2, 4 and 8 lanes before, within rows of 16
  add(std::integral_constant<int, 0x112>(), I());
  add(std::integral_constant<int, 0x114>(), I());
  add(std::integral_constant<int, 0x118>(), I());
  add(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());   // the last lane of a row to the next one
  add(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());   // ... of the second row to the two behind it
  return v;
}
// M samples in LDS (q, in rows of `ld`). A wave goes through its outputs' rows of weights two at a time, 4 KB of either, with the next two such pieces on
// their way; the first three are asked for before the samples are looked at, and arrive while those are brought to 8 bits.
template <class T, int M>
__global__ void __launch_bounds__(Q8_NT)
q8_few_kernel(const T *__restrict__ x, const int8_t *__restrict__ wq, const float *__restrict__ wscale, const T *__restrict__ bias, T *__restrict__ y,
              const int in, const int ld, const int out, const int batch, const int per_wave) {
  constexpr int R = 2, K = 4, AHEAD = M <= 4 ? 3 : 2;
  extern __shared__ uint4 lds[];
  __shared__ float part[M][Q8_NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, eights = ld / 8, words = ld / 16;
  const int first = (blockIdx.x * (Q8_NT / 64) + wave) * per_wave, last = min(out, first + per_wave);
  const int blocks = (words + 64 * K - 1) / (64 * K), pieces = first < last ? (last - first + R - 1) / R * blocks : 0;
  uint4 w[AHEAD][R][K];
  auto fetch = [&](uint4 (&to)[R][K], const int piece) {
    const int n = first + piece / blocks * R, k0 = piece % blocks * 64 * K + lane;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int at = min(k0 + 64 * k, words - 1);   // (behind the row: nothing is made of it)
        const any_word t = __builtin_nontemporal_load(reinterpret_cast<const any_word *>(wq + static_cast<size_t>(min(n + i, out - 1)) * ld) + at);
        to[i][k] = __builtin_bit_cast(uint4, t);
      }
  };
#pragma unroll
  for (int a = 0; a < AHEAD; ++a)
    if (a < pieces) fetch(w[a], a);
  __builtin_amdgcn_sched_barrier(0);

  float most[M] = {};
#pragma unroll
  for (int m = 0; m < M; ++m) {
    if (m >= batch) break;
    for (int k = tid; k < eights; k += Q8_NT) {
      float v[8];
      row8(x + static_cast<size_t>(m) * in, 8 * k, in, v);
      most[m] = most_of(v, most[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll
    for (int o = 32; o; o >>= 1) most[m] = most_of(most[m], __shfl_xor(most[m], o));
    if (lane == 0) part[m][wave] = most[m];
  }
  __syncthreads();
  float scale[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    float v = part[m][0];
#pragma unroll
    for (int i = 1; i < Q8_NT / 64; ++i) v = most_of(v, part[m][i]);
    scale[m] = scale_of(v);
    if (m >= batch) continue;
    uint2 *q = reinterpret_cast<uint2 *>(lds) + static_cast<size_t>(m) * eights;
    const float inverse = 1.0f / scale[m];
    for (int k = tid; k < eights; k += Q8_NT) {
      float e[8];
      row8(x + static_cast<size_t>(m) * in, 8 * k, in, e);
      q[k] = quantized(e, scale[m], inverse);
    }
  }
  __syncthreads();
  int sum[M][R] = {};
  auto use = [&](const uint4 (&v)[R][K], const int piece) {
    const int block = piece % blocks, n = first + piece / blocks * R;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int at = block * 64 * K + lane + 64 * k;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (at < words && m < batch) q = lds[m * words + at];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[m][i] = __builtin_amdgcn_sdot4(static_cast<int>((&q.x)[e]), static_cast<int>((&v[i][k].x)[e]), sum[m][i], false);
      }
    }
    if (block + 1 < blocks) return;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int total = last_lane_sum(sum[m][i]);
        sum[m][i] = 0;
        if (lane == 63 && n + i < last && m < batch)
          y[static_cast<size_t>(m) * out + n + i] =
              from_f32<T>(scaled(total, scale_parts(scale[m]), scale_parts(wscale[n + i]), bias ? to_f32(bias[n + i]) : 0.0f));
      }
  };
#pragma unroll 1
  for (int p = 0; p < pieces; p += AHEAD) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (p + a >= pieces) break;
      use(w[a], p + a);
      if (p + a + AHEAD < pieces) fetch(w[a], p + a + AHEAD);
    }
  }
}
template <class T>
int q8_few(int in, int out, int batch, const T *x, const int8_t *wq, const float *wscale, const T *b, T *y) {
  const int ld = static_cast<int>(tdh_q8_row(in)), cus = std::max(1, ctx().compute_units), waves = Q8_NT / 64;
  // as many workgroups as compute units, each wave pairs of outputs
  const int per_wave = ceil_div(ceil_div(out, cus * waves), 2) * 2, grid = ceil_div(out, per_wave * waves);
  ProfScope prof("q8_few", static_cast<double>(ld) * out, WORK_BYTE);
  auto go = [&](auto kernel) {
    TDH_LAUNCH(kernel, dim3(grid), dim3(Q8_NT), static_cast<size_t>(batch) * ld, ctx().stream, x, wq, wscale, b, y, in, ld, out, batch, per_wave);
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  };
  if (batch <= 1) return go(q8_few_kernel<T, 1>);
  if (batch <= 2) return go(q8_few_kernel<T, 2>);
  if (batch <= 4) return go(q8_few_kernel<T, 4>);
  return go(q8_few_kernel<T, 8>);
}

// ---------------------------------------------------------------- weights, once
// wscale of 64 columns a workgroup
template <class T>
__global__ void __launch_bounds__(1024)
q8_wscale_kernel(const T *__restrict__ w, float *__restrict__ wscale, const int in, const int out) {
  __shared__ float part[16][64];
  const int c = threadIdx.x & 63, g = threadIdx.x >> 6, col = blockIdx.x * 64 + c;
  float most = 0.0f;
  if (col < out)
    for (int k = g; k < in; k += 16) most = most_of(most, __builtin_fabsf(to_f32(w[static_cast<size_t>(k) * out + col])));
  part[g][c] = most;
  __syncthreads();
  if (g || col >= out) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) most = most_of(most, part[i][c]);
  wscale[col] = scale_of(most);
}
// 64 x 64 values through LDS
template <class T>
__global__ void __launch_bounds__(256)
q8_pack_kernel(const T *__restrict__ w, const float *__restrict__ wscale, int8_t *__restrict__ wq, const int in, const int out, const int ld) {
  __shared__ float tile[64][65];
  const int k0 = blockIdx.y * 64, n0 = blockIdx.x * 64, c = threadIdx.x & 63, g = threadIdx.x >> 6;
#pragma unroll 4
  for (int i = g; i < 64; i += 4)
    tile[i][c] = k0 + i < in && n0 + c < out ? to_f32(w[static_cast<size_t>(k0 + i) * out + n0 + c]) : 0.0f;
  __syncthreads();
  const int n = threadIdx.x >> 2, k = (threadIdx.x & 3) * 16;
  if (n0 + n >= out || k0 + k >= ld) return;
  const float s = wscale[n0 + n];
  uint2 o[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[k + 8 * h + e][n];
    o[h] = quantized(v, s, 1.0f / s);
  }
  *reinterpret_cast<uint4 *>(wq + static_cast<size_t>(n0 + n) * ld + k0 + k) = make_uint4(o[0].x, o[0].y, o[1].x, o[1].y);
}

constexpr int Q8_IN = 1 << 17, Q8_OUT = 1 << 20, Q8_BATCH = 1 << 24;
int check_q8(const char *who, int dtype, int in, int out) {
  TDH_CHECK_ARG(dtype_known(dtype), "%s: element type %d", who, dtype);
  TDH_CHECK_ARG(in > 0 && out > 0, "%s: bad shape %d -> %d", who, in, out);
  TDH_CHECK_ARG(in <= Q8_IN && out <= Q8_OUT, "%s: %d -> %d is beyond 2^17 -> 2^20", who, in, out);
  TDH_CHECK_ARG(static_cast<double>(tdh_q8_row(in)) * out < 2147483648.0, "%s: weights of 2^31 bytes or more", who);
  return TDH_OK;
}

}  // namespace
}  // namespace tdh

using namespace tdh;

extern "C" {

size_t tdh_q8_row(int in) { return in > 0 ? (static_cast<size_t>(in) + 15) & ~static_cast<size_t>(15) : 0; }

int tdh_fc_q8_pack(int dtype, int in, int out, const void *w, int8_t *wq, float *wscale) {
  const char *who = "tdh_fc_q8_pack";
  TDH_TRY(check_q8(who, dtype, in, out));
  TDH_CHECK_ARG(w && wq && wscale, "%s: null tensor", who);
  TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(wq) & 15) == 0, "%s: 8-bit weights not on a 16-byte boundary", who);
  TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(w) & (dtype_size(dtype) - 1)) == 0 && (reinterpret_cast<uintptr_t>(wscale) & 3) == 0,
                "%s: a tensor that is not aligned to its elements", who);
  const int ld = static_cast<int>(tdh_q8_row(in));
  TDH_TRY(check_apart(who, {{wq, static_cast<size_t>(ld) * out}, {wscale, 4 * static_cast<size_t>(out)}}, {{w, dtype_size(dtype) * in * out}}));
  TDH_REQUIRE_INIT();
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T *src = static_cast<const T *>(w);
    {
      ProfScope prof("q8_wscale", static_cast<double>(sizeof(T)) * in * out, WORK_BYTE);
      TDH_LAUNCH((q8_wscale_kernel<T>), dim3(ceil_div(out, 64)), dim3(1024), 0, ctx().stream, src, wscale, in, out);
      TDH_LAUNCH_CHECK();
    }
    ProfScope prof("q8_pack", (sizeof(T) + 1.0) * in * out, WORK_BYTE);
    TDH_LAUNCH((q8_pack_kernel<T>), dim3(ceil_div(out, 64), ceil_div(ld, 64)), dim3(256), 0, ctx().stream, src, wscale, wq, in, out, ld);
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  });
}

int tdh_fc_q8_fwd(int dtype, int in, int out, int has_bias, int batch, const void *x, const int8_t *wq, const float *wscale, const void *b, void *y) {
  const char *who = "tdh_fc_q8_fwd";
  TDH_TRY(check_q8(who, dtype, in, out));
  TDH_CHECK_ARG(batch >= 0 && batch <= Q8_BATCH, "%s: %d samples", who, batch);
  TDH_CHECK_ARG(static_cast<double>(batch) * tdh_q8_row(in) < 2147483648.0 && static_cast<double>(batch) * out < 2147483648.0,
                "%s: a tensor of 2^31 elements or more", who);
  TDH_CHECK_ARG(batch == 0 || (x && wq && wscale && y), "%s: null tensor", who);
  TDH_CHECK_ARG(!has_bias || b, "%s: has_bias set but no bias", who);
  const size_t size = dtype_size(dtype);
  TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(wq) & 15) == 0, "%s: 8-bit weights not on a 16-byte boundary", who);
  TDH_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(y)) & (size - 1)) == 0 &&
                    (reinterpret_cast<uintptr_t>(wscale) & 3) == 0,
                "%s: a tensor that is not aligned to its elements", who);
  TDH_TRY(check_apart(who, {{y, size * batch * out}}, {{x, size * batch * in}, {wq, tdh_q8_row(in) * out}, {wscale, 4 * static_cast<size_t>(out)},
                                                     {has_bias ? b : nullptr, size * out}}));
  TDH_REQUIRE_INIT();
  if (batch == 0) return TDH_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T *xs = static_cast<const T *>(x), *bs = has_bias ? static_cast<const T *>(b) : nullptr;
    if (batch <= Q8_FEW && batch * tdh_q8_row(in) <= Q8_FEW_BYTES) return q8_few(in, out, batch, xs, wq, wscale, bs, static_cast<T *>(y));
    return q8_many(in, out, batch, xs, wq, wscale, bs, static_cast<T *>(y));
  });
}

}  // extern "C"
