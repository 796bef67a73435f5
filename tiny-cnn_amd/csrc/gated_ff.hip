// gated_ff.hip — the gated feed-forward block: z = x W + b with W = [in][2 hidden], gate columns first, and
// h = act(z_gate) * z_up; on the way back dz = (dh * z_up * act'(z_gate), dh * act(z_gate)),
// dx = dz W^T, dW = x^T dz, db = the column sums of dz.
#include "lm_types.h"

namespace tdh {

namespace {

constexpr int GF_NT = 256;

// the gate's activation, and its derivative
__device__ __forceinline__ float gate_act(const int kind, const float g, float *slope) {
  switch (kind) {
    case TDH_GATE_SILU: {
      const float s = 1.0f / (1.0f + expf(-g));
      *slope = s * (1.0f + g * (1.0f - s));
      return g * s;
    }
    case TDH_GATE_GELU: {
      const float cdf = 0.5f * erfcf(-0.70710678118654752f * g);
      *slope = cdf + g * (0.39894228040143268f * expf(-0.5f * g * g));
      return g * cdf;
    }
    case TDH_GATE_GELU_TANH: {
      // 0.5 (1 + tanh(y)) = 1 / (1 + exp(-2 y)), y = sqrt(2/pi) (g + 0.044715 g^3)
      const float y2 = 1.5957691216057308f * (g + 0.044715f * g * g * g);
      const float s  = 1.0f / (1.0f + expf(-y2));
      *slope = s + g * s * (1.0f - s) * (1.5957691216057308f * (1.0f + 0.134145f * g * g));
      return g * s;
    }
    case TDH_GATE_SIGMOID: {
      const float s = 1.0f / (1.0f + expf(-g));
      *slope = s * (1.0f - s);
      return s;
    }
    case TDH_GATE_RELU: *slope = g > 0.0f ? 1.0f : 0.0f; return g > 0.0f ? g : 0.0f;
    default: *slope = 1.0f; return g;
  }
}

template <class T>
__global__ void __launch_bounds__(GF_NT)
gate_fwd_kernel(const float *__restrict__ z, T *__restrict__ h, const int hidden, const size_t total, const int act) {
  const size_t i = static_cast<size_t>(blockIdx.x) * GF_NT + threadIdx.x;
  if (i >= total) return;
  const size_t row = i / hidden, c = i - row * hidden;
  float slope;
  const float a = gate_act(act, z[row * 2 * hidden + c], &slope);
  h[i] = from_f32<T>(a * z[row * 2 * hidden + hidden + c]);
}

template <class T>
__global__ void __launch_bounds__(GF_NT)
gate_bwd_kernel(const float *__restrict__ z, const T *__restrict__ dh, float *__restrict__ dz, const int hidden,
                const size_t total, const int act) {
  const size_t i = static_cast<size_t>(blockIdx.x) * GF_NT + threadIdx.x;
  if (i >= total) return;
  const size_t row = i / hidden, c = i - row * hidden;
  float slope;
  const float a = gate_act(act, z[row * 2 * hidden + c], &slope), d = to_f32(dh[i]);
  dz[row * 2 * hidden + c]          = d * z[row * 2 * hidden + hidden + c] * slope;
  dz[row * 2 * hidden + hidden + c] = d * a;
}

// dst (+)= src in another type
template <class D, class S, bool ADD>
__global__ void __launch_bounds__(GF_NT)
cast_kernel(const S *__restrict__ src, D *__restrict__ dst, const size_t n) {
  const size_t stride = static_cast<size_t>(gridDim.x) * GF_NT;
  for (size_t i = static_cast<size_t>(blockIdx.x) * GF_NT + threadIdx.x; i < n; i += stride)
    dst[i] = from_f32<D>(to_f32(src[i]) + (ADD ? to_f32(dst[i]) : 0.0f));
}

template <class D, class S, bool ADD = false>
int launch_cast(const S *src, D *dst, size_t n) {
  if (!n) return TDH_OK;
  ProfScope prof("cast", static_cast<double>(n) * (sizeof(D) + sizeof(S)), WORK_BYTE);
  TDH_LAUNCH((cast_kernel<D, S, ADD>), dim3(static_cast<unsigned>(std::min<size_t>(ceil_div_sz(n, GF_NT), GRID_X_MAX))),
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

template <class T>
int ff_fwd(int act, int in, int hidden, int batch, const T *x, const T *w, const T *b, T *h, float *z) {
  const size_t nx = static_cast<size_t>(batch) * in, nw = static_cast<size_t>(in) * 2 * hidden, nz = static_cast<size_t>(batch) * 2 * hidden;
  constexpr bool cast = sizeof(T) == 2;
  TDH_TRY(ws_begin(fc_workspace_bytes(in, 2 * hidden, batch) + (z ? 0 : ws_align(4 * nz)) +
                   (cast ? ws_align(4 * nx) + ws_align(4 * nw) + ws_align(8 * hidden) : 0)));
  const float *xf = reinterpret_cast<const float *>(x), *wf = reinterpret_cast<const float *>(w), *bf = reinterpret_cast<const float *>(b);
  if (!z) TDH_TRY(take(nz, &z));
  if (cast) {
    float *p;
    TDH_TRY(take(nx, &p));
    TDH_TRY((launch_cast<float, T>(x, p, nx)));
    xf = p;
    TDH_TRY(take(nw, &p));
    TDH_TRY((launch_cast<float, T>(w, p, nw)));
    wf = p;
    if (b) {
      TDH_TRY(take(2 * static_cast<size_t>(hidden), &p));
      TDH_TRY((launch_cast<float, T>(b, p, 2 * static_cast<size_t>(hidden))));
      bf = p;
    }
  }
  TDH_TRY(fc_fwd(in, 2 * hidden, b != nullptr, batch, xf, wf, bf, z));
  const size_t total = nz / 2;
  ProfScope prof("gate_fwd", (8.0 + sizeof(T)) * total, WORK_BYTE);
  TDH_LAUNCH((gate_fwd_kernel<T>), dim3(static_cast<unsigned>(ceil_div_sz(total, GF_NT))), dim3(GF_NT), 0, ctx().stream, z, h,
             hidden, total, act);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

template <class T>
int ff_bwd(int act, int in, int hidden, int batch, const T *x, const T *w, const float *z, const T *dh, T *dx, T *dw, T *db,
           int accumulate) {
  const size_t nx = static_cast<size_t>(batch) * in, nw = static_cast<size_t>(in) * 2 * hidden, nz = static_cast<size_t>(batch) * 2 * hidden,
               nb = 2 * static_cast<size_t>(hidden);
  constexpr bool cast = sizeof(T) == 2;
  TDH_TRY(ws_begin(fc_workspace_bytes(in, 2 * hidden, batch) + ws_align(4 * nz) +
                   (cast ? 2 * ws_align(4 * nx) + 2 * ws_align(4 * nw) + ws_align(4 * nb) : 0)));
  float *dz;
  TDH_TRY(take(nz, &dz));
  const size_t total = nz / 2;
  {
    ProfScope prof("gate_bwd", (16.0 + sizeof(T)) * total, WORK_BYTE);
    TDH_LAUNCH((gate_bwd_kernel<T>), dim3(static_cast<unsigned>(ceil_div_sz(total, GF_NT))), dim3(GF_NT), 0, ctx().stream, z, dh,
               dz, hidden, total, act);
    TDH_LAUNCH_CHECK();
  }
  if constexpr (!cast) {
    return fc_bwd(in, 2 * hidden, db != nullptr, batch, reinterpret_cast<const float *>(x), reinterpret_cast<const float *>(w), dz,
                  reinterpret_cast<float *>(dx), reinterpret_cast<float *>(dw), reinterpret_cast<float *>(db), accumulate, ActGrad());
  } else {
    float *xf, *wf, *dxf, *dwf, *dbf;
    TDH_TRY(take(nx, &xf));
    TDH_TRY(take(nw, &wf));
    TDH_TRY(take(nx, &dxf));
    TDH_TRY(take(nw, &dwf));
    TDH_TRY(take(nb, &dbf));
    TDH_TRY((launch_cast<float, T>(x, xf, nx)));
    TDH_TRY((launch_cast<float, T>(w, wf, nw)));
    TDH_TRY(fc_bwd(in, 2 * hidden, db != nullptr, batch, xf, wf, dz, dx ? dxf : nullptr, dw ? dwf : nullptr, db ? dbf : nullptr, 0, ActGrad()));
    if (dx) TDH_TRY((launch_cast<T, float>(dxf, dx, nx)));
    if (dw) TDH_TRY(accumulate ? (launch_cast<T, float, true>(dwf, dw, nw)) : (launch_cast<T, float>(dwf, dw, nw)));
    if (db) TDH_TRY(accumulate ? (launch_cast<T, float, true>(dbf, db, nb)) : (launch_cast<T, float>(dbf, db, nb)));
    return TDH_OK;
  }
}

int check_ff(const char *who, int dtype, int act, int in, int hidden, int batch) {
  TDH_CHECK_ARG(dtype_known(dtype), "%s: element type %d", who, dtype);
  TDH_CHECK_ARG(act >= TDH_GATE_SILU && act <= TDH_GATE_NONE, "%s: gate activation %d", who, act);
  TDH_CHECK_ARG(in > 0 && hidden > 0 && batch >= 0, "%s: bad shape %d->2*%d batch %d", who, in, hidden, batch);
  TDH_CHECK_ARG(2L * in * hidden < (1L << 31) && static_cast<long>(batch) * in < (1L << 31) && 2L * batch * hidden < (1L << 31),
                "%s: tensor exceeds 2^31 elements", who);
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
  TDH_REQUIRE_INIT();
  if (batch == 0) return TDH_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return ff_fwd<T>(act, in, hidden, batch, static_cast<const T *>(x), static_cast<const T *>(w),
                     has_bias ? static_cast<const T *>(b) : nullptr, static_cast<T *>(h), z);
  });
}

int tdh_gated_ff_bwd(int dtype, int act, int in, int hidden, int has_bias, int batch, const void *x, const void *w,
                     const float *z, const void *dh, void *dx, void *dw, void *db, int accumulate) {
  TDH_TRY(check_ff("tdh_gated_ff_bwd", dtype, act, in, hidden, batch));
  TDH_CHECK_ARG(batch == 0 || (x && w && z && dh), "tdh_gated_ff_bwd: null tensor");
  TDH_TRY(check_aligned("tdh_gated_ff_bwd", dtype, {x, w, dh, dx, dw, db}));
  TDH_TRY(check_aligned("tdh_gated_ff_bwd", TDH_F32, {z}));
  TDH_REQUIRE_INIT();
  if (batch == 0) return TDH_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return ff_bwd<T>(act, in, hidden, batch, static_cast<const T *>(x), static_cast<const T *>(w), z, static_cast<const T *>(dh),
                     static_cast<T *>(dx), static_cast<T *>(dw), has_bias ? static_cast<T *>(db) : nullptr, accumulate);
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
