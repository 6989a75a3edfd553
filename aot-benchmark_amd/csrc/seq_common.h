// What the token-sequence kernels (rope.hip, paged_attn.hip, paged_evict.hip, masked_attn.hip) share: the element types, 16-byte
// chunks of a row, and the matrix-core product of two such chunks.
#pragma once
#include "common.h"

typedef _Float16 f16;
typedef __bf16 bf16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16;

static constexpr float LOG2E = 1.44269504088896340736f;
static constexpr float NEG_INF = -__builtin_inff();

template <class T> struct Elem;
template <> struct Elem<float> { static constexpr int CE = 4; };        // elements of a 16-byte chunk
template <> struct Elem<f16> { static constexpr int CE = 8; };
template <> struct Elem<bf16> { static constexpr int CE = 8; };

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }

// two floats rounded to nearest even into one dword, low half first (one packed conversion)
template <class T> __device__ __forceinline__ unsigned pack2(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef T t2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f2{a, b}), t2));
}
template <class T> __device__ __forceinline__ float half_to_float(u16 x) {
  union { u16 u; T h; } r;
  r.u = x;
  return (float)r.h;
}

// Whether the 4-byte word holds an infinity or a NaN (of either half for the 16-bit types): all exponent bits set.
template <class T> __device__ __forceinline__ bool word_nonfinite(unsigned x) {
  if constexpr (sizeof(T) == 4) return (x & 0x7f800000u) == 0x7f800000u;
  else if constexpr (std::is_same<T, bf16>::value) return (((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
  else return (((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u) != 0;
}
// ... and the word with those elements replaced by zero
template <class T> __device__ __forceinline__ unsigned word_finite(unsigned x) {
  if constexpr (sizeof(T) == 4) return (x & 0x7f800000u) == 0x7f800000u ? 0u : x;
  else {
    const unsigned e = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
    if ((x & e) == e) x &= 0xffff0000u;
    if (((x >> 16) & e) == e) x &= 0x0000ffffu;
    return x;
  }
}

// s -> cap * tanh(s / cap) as 1 - 2 / (1 + exp(2 x)): absolute error a few 2^-24 of cap, exact limits at both ends
// (x = s * 2 log2(e) / cap on entry).  Returns the tanh.
__device__ __forceinline__ float tanh_from_exp2(float x) { return 1.f - 2.f * rcp_hw(1.f + exp2_hw(x)); }

// dtype code of the C ABI -> f(type tag); false for an unknown code
template <class F> static inline bool with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case AOT_F32: f(float{}); return true;
    case AOT_F16: f(f16{}); return true;
    case AOT_BF16: f(bf16{}); return true;
  }
  return false;
}
static inline int dtype_size(int dtype) { return dtype == AOT_F32 ? 4 : dtype == AOT_F16 || dtype == AOT_BF16 ? 2 : 0; }
static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
