// seeded_dropout.hip — dropout whose mask is a function of the element's index and is never stored.
//
// Element i of a call under (seed, offset) has word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): counter (i / 4, offset), key seed, both low word
// first. It is kept where that word is at least floor(rate 2^32), so with a probability within 2^-32 of 1 - rate,
// and scaled by 1 / (1 - rate); the backward pass draws the same words again.
#include "lm_types.h"

namespace tdh {

namespace {

constexpr int SD_NT = 256;

__device__ __forceinline__ void philox_round(uint32_t (&c)[4], const uint32_t k0, const uint32_t k1) {
  const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c[0], b = static_cast<uint64_t>(0xCD9E8D57u) * c[2];
  // (a ^ b ^ c in one instruction)
  const uint32_t c0 = __builtin_amdgcn_bitop3_b32(static_cast<uint32_t>(b >> 32), c[1], k0, 0x96);
  const uint32_t c2 = __builtin_amdgcn_bitop3_b32(static_cast<uint32_t>(a >> 32), c[3], k1, 0x96);
  c[1] = static_cast<uint32_t>(b);
  c[3] = static_cast<uint32_t>(a);
  c[0] = c0;
  c[2] = c2;
}

// the four words of elements 4 * block .. 4 * block + 3
__device__ __forceinline__ void philox(uint32_t (&c)[4], const uint64_t block, const uint64_t offset, const uint64_t seed) {
  c[0] = static_cast<uint32_t>(block);
  c[1] = static_cast<uint32_t>(block >> 32);
  c[2] = static_cast<uint32_t>(offset);
  c[3] = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    philox_round(c, k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// y = [residual +] keep * scale * x, a 16-byte word a thread at a time. Tensors that the L2 caches do not hold go past them. Bound by
// memory with a residual (33.5 M bf16 values: 32.7 us, 6.2 TB/s; through the caches 36.8), without one by the generator's
// 64-bit products, two a round.
constexpr size_t SD_ONCE_BYTES = 32u << 20;
template <class T, bool RES, bool ONCE>
__global__ void __launch_bounds__(SD_NT)
seeded_dropout_kernel(const T *x, const T *residual, T *y, const size_t n, const uint32_t threshold, const float scale,
                      const uint64_t seed_arg, const uint64_t offset_arg, const uint64_t *__restrict__ state) {
  constexpr int E = Word<T>::N;
  const uint64_t seed = state ? state[0] : seed_arg, offset = state ? state[1] : offset_arg;
  const size_t items = (n + E - 1) / E, stride = static_cast<size_t>(gridDim.x) * SD_NT;
  for (size_t i = static_cast<size_t>(blockIdx.x) * SD_NT + threadIdx.x; i < items; i += stride) {
    const size_t at = i * E;
    uint32_t c[E / 4][4];
#pragma unroll
    for (int q = 0; q < E / 4; ++q) philox(c[q], i * (E / 4) + q, offset, seed);
    if (at + E <= n) {
      const Word<T> v = load_word<T, ONCE>(x + at), r = RES ? load_word<T, ONCE>(residual + at) : Word<T>{};
      float o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = c[e / 4][e % 4] >= threshold ? v[e] * scale : 0.0f;
        o[e] = RES ? r[e] + d : d;
      }
      store_word<ONCE>(y + at, Word<T>::from(o).raw);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (at + e >= n) break;
        const float d = c[e / 4][e % 4] >= threshold ? to_f32(x[at + e]) * scale : 0.0f;
        y[at + e] = from_f32<T>(RES ? to_f32(residual[at + e]) + d : d);
      }
    }
  }
}

__global__ void advance_kernel(uint64_t *state, const int n) {
  for (int i = threadIdx.x; i < n; i += 64) ++state[2 * i + 1];
}

}  // namespace

int seeded_dropout(int dtype, size_t n, float rate, uint64_t seed, uint64_t offset, const uint64_t *state, const void *x,
                   const void *residual, void *y, const char *tag) {
  const size_t size = dtype_size(dtype);
  ProfScope prof(tag, static_cast<double>(size) * n * (residual ? 3 : 2), WORK_BYTE);
  const uint32_t threshold = static_cast<uint32_t>(static_cast<double>(rate) * 4294967296.0);
  const float scale        = static_cast<float>(1.0 / (1.0 - static_cast<double>(rate)));
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const size_t items = ceil_div_sz(n, Word<T>::N);
    const dim3 grid(static_cast<unsigned>(std::min<size_t>(ceil_div_sz(items, SD_NT), GRID_X_MAX)));
    auto go = [&](auto kernel) {
      TDH_LAUNCH(kernel, grid, dim3(SD_NT), 0, ctx().stream, static_cast<const T *>(x), static_cast<const T *>(residual),
                 static_cast<T *>(y), n, threshold, scale, seed, offset, state);
      TDH_LAUNCH_CHECK();
      return static_cast<int>(TDH_OK);
    };
    if (size * n > SD_ONCE_BYTES) return residual ? go(seeded_dropout_kernel<T, true, true>) : go(seeded_dropout_kernel<T, false, true>);
    return residual ? go(seeded_dropout_kernel<T, true, false>) : go(seeded_dropout_kernel<T, false, false>);
  });
}

int seeded_dropout_advance(uint64_t *state, int n) {
  ProfScope prof("dropout_advance", 16.0 * n, WORK_BYTE);
  TDH_LAUNCH(advance_kernel, dim3(1), dim3(64), 0, ctx().stream, state, n);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

}  // namespace tdh

using namespace tdh;

static int check_seeded(const char *who, int dtype, size_t n, float rate, const void *in, const void *residual, const void *out) {
  TDH_CHECK_ARG(dtype_known(dtype), "%s: element type %d", who, dtype);
  TDH_CHECK_ARG(rate >= 0.0f && rate < 1.0f, "%s: dropout rate %g", who, rate);
  TDH_CHECK_ARG(n <= SIZE_MAX / 8, "%s: %zu elements", who, n);
  TDH_CHECK_ARG(n == 0 || (in && out), "%s: null tensor", who);
  const uintptr_t align = dtype_size(dtype) - 1;
  TDH_CHECK_ARG(((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(out)) & align) == 0,
                "%s: a tensor that is not aligned to its elements", who);
  const uintptr_t o = reinterpret_cast<uintptr_t>(out);
  const size_t bytes = n * dtype_size(dtype);
  for (const void *p : {in, residual}) {
    const uintptr_t q = reinterpret_cast<uintptr_t>(p);
    TDH_CHECK_ARG(!p || q == o || q + bytes <= o || o + bytes <= q, "%s: the output overlaps an input without being it", who);
  }
  return TDH_OK;
}

extern "C" {

int tdh_dropout_seeded_fwd(int dtype, size_t n, float rate, uint64_t seed, uint64_t offset, const void *x,
                           const void *residual, void *y) {
  TDH_TRY(check_seeded("tdh_dropout_seeded_fwd", dtype, n, rate, x, residual, y));
  TDH_REQUIRE_INIT();
  if (n == 0) return TDH_OK;
  return seeded_dropout(dtype, n, rate, seed, offset, nullptr, x, residual, y, "dropout_seeded_fwd");
}

int tdh_dropout_seeded_bwd(int dtype, size_t n, float rate, uint64_t seed, uint64_t offset, const void *dy, void *dx) {
  TDH_TRY(check_seeded("tdh_dropout_seeded_bwd", dtype, n, rate, dy, nullptr, dx));
  TDH_REQUIRE_INIT();
  if (n == 0) return TDH_OK;
  return seeded_dropout(dtype, n, rate, seed, offset, nullptr, dy, nullptr, dx, "dropout_seeded_bwd");
}

}  // extern "C"
