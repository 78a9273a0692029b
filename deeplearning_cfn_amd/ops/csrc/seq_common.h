// Element types and vector access shared by the sequence kernels
// (embedding, document attention, Newton-Schulz).
//
// BF16 and FP16 are 16-bit storage types; arithmetic is fp32 except in the
// matrix instructions, which take 16-bit operands and add in fp32.
#pragma once

#include "dlx_common.h"

namespace dlx {

struct BF16 { uint16_t v; };
struct FP16 { uint16_t v; };

template <typename T> DLX_DEV float to_f32(T x);
template <> DLX_DEV float to_f32<float>(float x) { return x; }
template <> DLX_DEV float to_f32<BF16>(BF16 x) { return bf2f(x.v); }
template <> DLX_DEV float to_f32<FP16>(FP16 x) {
  return (float)__builtin_bit_cast(_Float16, x.v);
}

// round to nearest even
template <typename T> DLX_DEV T from_f32(float f);
template <> DLX_DEV float from_f32<float>(float f) { return f; }
template <> DLX_DEV BF16 from_f32<BF16>(float f) {
  return BF16{__builtin_bit_cast(uint16_t, (__bf16)f)};
}
template <> DLX_DEV FP16 from_f32<FP16>(float f) {
  return FP16{__builtin_bit_cast(uint16_t, (_Float16)f)};
}

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

template <typename T, int N> DLX_DEV void load_vec(const T* p, float* out) {
  const Pack<T, N> x = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = to_f32<T>(x.v[i]);
}

template <typename T, int N> DLX_DEV void store_vec(T* p, const float* in) {
  Pack<T, N> x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = from_f32<T>(in[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = x;
}

}  // namespace dlx
