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

// fp16 ends at 6e-8, above the share of a key in a long row: its probabilities are held 2^15 times as large (at most 2^15 of 65504) while they
// are rounded for a product, in the exponent they are formed with, so that none above 2^-39 of the largest is lost.
template <class T> static constexpr float LIFT = std::is_same<T, f16>::value ? 15.f : 0.f;
template <class T> static constexpr float LOWER = std::is_same<T, f16>::value ? 0x1p-15f : 1.f;

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

// The cap on a score, in powers of two: s -> cap log2(e) tanh(y), y = s scale / cap, from x = 2 log2(e) y, and the cap's derivative
// 1 - tanh^2.  With E = exp(-2 |y|) = exp2(-|x|):
//   |x| >= 1   tanh = +-(1 - E) / (1 + E) and 1 - tanh^2 = 4 E / (1 + E)^2: no cancellation that counts (1 - E is exact and at least 1/2),
//              infinities give +-1 and 0
//   |x| < 1    tanh = y (1 + z P(z)), z = x^2, P a minimax fit of (tanh(y) / y - 1) / z on [0, 1] (least squares on Chebyshev nodes, reweighted
//              until level): 0.6 2^-24 of the value.  As s log2(e) scale (1 + z P) the score's error is relative to the score whatever the cap
//              (1 - 2 / (1 + exp(2 y)) leaves a few 2^-24 of the cap: noise of the size of the scores where the cap is 1e6).
// A tile all of whose scores are small, which is the rule under the caps in use, takes the polynomial alone: 7 plain operations a
// score instead of 6 with two of quarter rate.
struct Cap {
  float mul, lin, top;                                          // s -> x; scale log2(e); cap log2(e)
  static Cap of(float scale, float cap) { return Cap{std::min(scale * 2.f * LOG2E / cap, 3.0e38f), scale * LOG2E, cap * LOG2E}; }
  __device__ __forceinline__ float bend(float x) const {        // tanh(y) / y, |x| < 1
    const float z = x * x;
    return __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -8.533986692782491e-05f, 0.0019189956365153193f), -0.04003699868917465f), 1.f);
  }
  __device__ __forceinline__ float far(float s, float E, float r) const { return __builtin_copysignf(top * ((1.f - E) * r), s); }
  __device__ __forceinline__ float operator()(float s) const {
    const float x = s * mul, E = exp2_hw(-fabsf(x)), near = s * lin * bend(x), away = far(s, E, rcp_hw(1.f + E));
    return fabsf(x) < 1.f ? near : away;                        // (both formed first: a selection, not a branch a lane)
  }
  template <int N> __device__ __forceinline__ bool small(const f32x16 (&s)[N]) const {     // of the whole wave (NaN aside)
    float a = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) a = fmaxf(a, fabsf(s[n][r]));
    return !__any(a * mul >= 1.f);
  }
  template <int N> __device__ __forceinline__ void tiles(f32x16 (&s)[N]) const {
    if (small(s)) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = s[n][r] * lin * bend(s[n][r] * mul);
    } else {
      Cap c = *this;
      asm("" : "+s"(c.mul), "+s"(c.lin));                        // (as below)
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[n][r] = c(s[n][r]);
          if (r % 2) __builtin_amdgcn_sched_barrier(0);
        }
      asm volatile("");
    }
  }
  // a tile's scores, and slope(r, the derivative) for each
  template <class F> __device__ __forceinline__ void tile(f32x16 (&s)[1], F&& slope) const {
    constexpr float HALF_LN2 = 0.34657359027997265f;
    if (small(s)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = s[0][r] * mul, w = bend(x), th = x * HALF_LN2 * w;
        s[0][r] = s[0][r] * lin * w;
        slope(r, __builtin_fmaf(-th, th, 1.f));
        if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // Registers decide here.  Without the empty statements the compiler forms what both branches begin with ahead of them and what they end
      // with behind them, for all sixteen scores, and without the fences it works on all of them side by side: 40 and more registers, spilled.
      Cap c = *this;
      asm("" : "+s"(c.mul), "+s"(c.lin));
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = s[0][r] * c.mul, E = exp2_hw(-fabsf(x)), q = rcp_hw(1.f + E), w = bend(x), th = x * HALF_LN2 * w, two = q + q;
        const float near = s[0][r] * c.lin * w, away = c.far(s[0][r], E, q), dn = __builtin_fmaf(-th, th, 1.f), da = E * two * two;
        s[0][r] = fabsf(x) < 1.f ? near : away;
        slope(r, fabsf(x) < 1.f ? dn : da);
        if (r % 2) __builtin_amdgcn_sched_barrier(0);
      }
      asm volatile("");
    }
  }
};

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
