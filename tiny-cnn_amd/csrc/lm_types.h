// lm_types.h — element types of the language-model operators: what tdh_dtype names, as device types with
// their conversions to and from fp32 (to nearest, ties to even), and 16-byte words of them.
#pragma once
#include "common.h"

#include <initializer_list>

namespace tdh {

struct bf16 {
  uint16_t bits;
};
struct f16 {
  _Float16 v;
};

__device__ __forceinline__ float to_f32(const float v) { return v; }
__device__ __forceinline__ float to_f32(const bf16 v) { return __uint_as_float(static_cast<uint32_t>(v.bits) << 16); }
__device__ __forceinline__ float to_f32(const f16 v) { return static_cast<float>(v.v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(const float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(const float v) {
  return bf16{__builtin_bit_cast(uint16_t, static_cast<__bf16>(v))};
}
template <>
__device__ __forceinline__ f16 from_f32<f16>(const float v) { return f16{static_cast<_Float16>(v)}; }

// Sixteen bytes of T: element e of the word, and words put together from fp32 values.
template <class T>
struct Word {
  static constexpr int N = 16 / static_cast<int>(sizeof(T));
  uint4 raw;
  __device__ __forceinline__ float operator[](const int e) const {
    const uint32_t w = (&raw.x)[e * static_cast<int>(sizeof(T)) / 4];
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w);
    else
      return to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(e & 1 ? w >> 16 : w)));
  }
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  __device__ __forceinline__ static uint32_t pair(bf16, const float a, const float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
  }
  __device__ __forceinline__ static uint32_t pair(f16, const float a, const float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
  }
  __device__ __forceinline__ static Word from(const float (&v)[N]) {
    Word o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        (&o.raw.x)[i] = __float_as_uint(v[i]);
      else
        (&o.raw.x)[i] = pair(T(), v[2 * i], v[2 * i + 1]);   // (one instruction for the two)
    }
    return o;
  }
};

// Sixteen bytes of memory on any element's boundary (the memory instructions take them there; where rows have an odd length every
// other one starts off a 16-byte boundary). ONCE: past the caches (data larger than they are, read or written once).
typedef uint32_t any_word __attribute__((ext_vector_type(4), aligned(2)));
template <class T, bool ONCE = false>
__device__ __forceinline__ Word<T> load_word(const T *p) {
  const any_word *q = reinterpret_cast<const any_word *>(p);
  return Word<T>{__builtin_bit_cast(uint4, ONCE ? __builtin_nontemporal_load(q) : *q)};
}
template <bool ONCE = false>
__device__ __forceinline__ void store_word(void *p, const uint4 v) {
  any_word *q = static_cast<any_word *>(p);
  if constexpr (ONCE)
    __builtin_nontemporal_store(__builtin_bit_cast(any_word, v), q);
  else
    *q = __builtin_bit_cast(any_word, v);
}

// Eight neighbours.
template <class T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
#pragma unroll
  for (int q = 0; q < 8 / Word<T>::N; ++q) {
    const Word<T> w = load_word(p + q * Word<T>::N);
#pragma unroll
    for (int e = 0; e < Word<T>::N; ++e) v[q * Word<T>::N + e] = w[e];
  }
}
template <class T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
#pragma unroll
  for (int q = 0; q < 8 / Word<T>::N; ++q) {
    float w[Word<T>::N];
#pragma unroll
    for (int e = 0; e < Word<T>::N; ++e) w[e] = v[q * Word<T>::N + e];
    store_word(p + q * Word<T>::N, Word<T>::from(w).raw);
  }
}

// The N elements of word k of a row of `len`: those behind its end read as `rest`.
template <class T>
__device__ __forceinline__ Word<T> row_word(const T *p, const int k, const int len, const float rest) {
  constexpr int N = Word<T>::N;
  if (k * N + N <= len) return load_word(p + k * N);
  float v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = k * N + e < len ? to_f32(p[k * N + e]) : rest;
  return Word<T>::from(v);
}
template <class T, bool ONCE = false>
__device__ __forceinline__ void put_row_word(T *p, const int k, const int len, const float (&v)[Word<T>::N]) {
  constexpr int N = Word<T>::N;
  if (k * N + N <= len) return store_word<ONCE>(p + k * N, Word<T>::from(v).raw);
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (k * N + e < len) p[k * N + e] = from_f32<T>(v[e]);
}

inline bool dtype_known(int dtype) { return dtype == TDH_F32 || dtype == TDH_BF16 || dtype == TDH_F16; }
inline size_t dtype_size(int dtype) { return dtype == TDH_F32 ? 4 : 2; }

// No output of a call may overlap an input or another output of it.
struct Span {
  const void *p;
  size_t bytes;
};
inline int check_apart(const char *who, std::initializer_list<Span> outputs, std::initializer_list<Span> inputs) {
  auto meet = [](const Span &a, const Span &b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return x && y && a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
  };
  for (const Span &o : outputs) {
    for (const Span &i : inputs) TDH_CHECK_ARG(!meet(o, i), "%s: an output overlaps an input", who);
    for (const Span *q = &o + 1; q != outputs.end(); ++q) TDH_CHECK_ARG(!meet(o, *q), "%s: two outputs overlap", who);
  }
  return TDH_OK;
}

// Calls f with a value of the device type that `dtype` names.
template <class F>
inline int with_dtype(int dtype, const F &f) {
  switch (dtype) {
    case TDH_F32: return f(float());
    case TDH_BF16: return f(bf16());
    default: return f(f16());
  }
}

}  // namespace tdh
