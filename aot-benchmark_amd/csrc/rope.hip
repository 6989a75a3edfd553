// Rotary positions: every head's first `rot` elements are pairs (u, w) turned by the angle pos * freq[j],
//   (u, w) -> m (u cos - w sin, w cos + u sin)
// with pairs (j, j + rot/2) (halves) or (2j, 2j + 1) (interleaved); the rest of the head passes through.  The gradient is the turn
// by the negated angle.  The append form writes the turned keys and the values straight into their cache slots.
//
// Bound by memory: an element is read once and written once.  The angle needs 64 bits (a position of a million times a frequency of
// one is 160 000 turns: a 32-bit product has lost the fraction), so each workgroup forms the cosines and sines of its rows once,
// in shared memory -- one double product and one sincospif per (row, pair) -- and all heads of the row read them.
#include "seq_common.h"

struct RopeP {
  const char *q, *k, *v;
  char *qo, *ko, *vo;
  const int *pos, *slots;
  const double* freqs;
  long qs[3], ks[3], vs[3], qos[3], kos[3], vos[3], ps[2];   // element strides: (b, s, h); append: outputs of k / v (page, slot, head)
  long nslots;
  long rows;
  int S, H, Hk, D, rot, inter, page_shift, R, up_shift;
  float mscale, sign;
};

// VE elements a unit: a unit of a half-split head is VE elements of each half
template <class T, int VE, bool APPEND>
__global__ __launch_bounds__(256) void rope_kernel(RopeP p) {
  extern __shared__ float2 cs[];                              // [R][rot / 2]
  struct alignas(VE * sizeof(T)) Vec { T e[VE]; };
  const int half = p.rot >> 1;
  const long row0 = (long)blockIdx.x * p.R;
  const int nrow = (int)min((long)p.R, p.rows - row0);
  for (int i = threadIdx.x; i < nrow * half; i += 256) {
    const int r = i / half, j = i - r * half;
    const long row = row0 + r;
    const int b = APPEND ? 0 : (int)(row / p.S), s = APPEND ? (int)row : (int)(row - (long)b * p.S);
    const double turns = (double)p.pos[b * p.ps[0] + s * p.ps[1]] * (p.freqs[j] * 0.15915494309189533577);    // 1 / (2 pi)
    const float x = (float)(2.0 * (turns - rint(turns)));      // half turns in [-1, 1]
    float sn, c;
    sincospif(x, &sn, &c);
    cs[i] = make_float2(c * p.mscale, sn * p.sign * p.mscale);
  }
  __syncthreads();
  const int up = 1 << p.up_shift, u0 = threadIdx.x & (up - 1), h0 = threadIdx.x >> p.up_shift, hstep = 256 >> p.up_shift;
  const int na = (p.inter ? p.rot : half) / VE, n = na + (p.D - p.rot) / VE, nv = p.D / VE;
  const int heads = p.H + p.Hk, all = APPEND ? heads + p.Hk : heads;
  for (int r = 0; r < nrow; ++r) {
    const long row = row0 + r;
    const int b = APPEND ? 0 : (int)(row / p.S), s = APPEND ? (int)row : (int)(row - (long)b * p.S);
    long slot = -1;
    if (APPEND) {
      slot = p.slots[row];
      if (slot >= p.nslots) slot = -1;                          // outside the pool: not written, like a negative slot
    }
    const long pg = slot >> p.page_shift, in = slot & ((1 << p.page_shift) - 1);
    const float2* c = cs + r * half;
    for (int h = h0; h < all; h += hstep) {
      const bool isq = h < p.H, isv = h >= heads;
      const int hh = isq ? h : isv ? h - heads : h - p.H;
      if (APPEND && !isq && slot < 0) continue;
      const long* st = isq ? p.qs : isv ? p.vs : p.ks;
      const T* x = (const T*)(isq ? p.q : isv ? p.v : p.k) + b * st[0] + s * st[1] + hh * st[2];
      T* y;
      if (isq) y = (T*)p.qo + b * p.qos[0] + s * p.qos[1] + hh * p.qos[2];
      else if (APPEND) {
        const long* o = isv ? p.vos : p.kos;
        y = (T*)(isv ? p.vo : p.ko) + pg * o[0] + in * o[1] + hh * o[2];
      } else y = (T*)p.ko + b * p.kos[0] + s * p.kos[1] + hh * p.kos[2];
      for (int u = u0; u < (isv ? nv : n); u += up) {
        if (isv) {
          *(Vec*)(y + u * VE) = *(const Vec*)(x + u * VE);
        } else if (u >= na) {
          const int d = p.rot + (u - na) * VE;
          *(Vec*)(y + d) = *(const Vec*)(x + d);
        } else if (p.inter) {
          if constexpr (VE > 1) {
            Vec a = *(const Vec*)(x + u * VE), o;
#pragma unroll
            for (int e = 0; e < VE; e += 2) {
              const float2 w = c[(u * VE + e) >> 1];
              const float f = (float)a.e[e], g = (float)a.e[e + 1];
              o.e[e] = (T)(f * w.x - g * w.y);
              o.e[e + 1] = (T)(g * w.x + f * w.y);
            }
            *(Vec*)(y + u * VE) = o;
          }
        } else {
          const Vec a = *(const Vec*)(x + u * VE), z = *(const Vec*)(x + half + u * VE);
          Vec o1, o2;
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float2 w = c[u * VE + e];
            const float f = (float)a.e[e], g = (float)z.e[e];
            o1.e[e] = (T)(f * w.x - g * w.y);
            o2.e[e] = (T)(g * w.x + f * w.y);
          }
          *(Vec*)(y + u * VE) = o1;
          *(Vec*)(y + half + u * VE) = o2;
        }
      }
    }
  }
}

template <bool APPEND>
static int rope_launch(RopeP& p, int dtype, hipStream_t stream) {
  if (p.rows == 0) return AOT_OK;
  const int es = dtype_size(dtype);
  // the widest unit that divides every run a unit walks, every stride and every address
  int ve = 16 / es;
  auto fits = [&](int n) {
    const int run = p.inter ? p.rot : p.rot / 2;
    if (run % n || p.D % n || (p.D - p.rot) % n || (!p.inter && p.rot % n)) return false;
    const void* ptr[] = {p.q, p.k, p.v, p.qo, p.ko, p.vo};
    for (const void* a : ptr) if ((uintptr_t)a % (n * es)) return false;
    const long* st[] = {p.qs, p.ks, p.vs, p.qos, p.kos, p.vos};
    for (const long* a : st) for (int i = 0; i < 3; ++i) if (a[i] % n) return false;
    return true;
  };
  while (ve > (p.inter ? 2 : 1) && !fits(ve)) ve >>= 1;
  if (!fits(ve)) return AOT_ERR_BADARG;                        // interleaved pairs not aligned to a pair
  const int n = std::max((p.inter ? p.rot : p.rot / 2) / ve + (p.D - p.rot) / ve, 1);
  p.up_shift = 0;
  while ((1 << p.up_shift) < n && p.up_shift < 8) ++p.up_shift;
  // Rows a workgroup: one while that is what fills the 256 CUs, two as soon as eight workgroups a CU remain, four with sixteen a CU.  Kernel times
  // with 1 / 2 / 4 rows, 20 heads of 128 turned: 2048 rows 7.1 / 6.6 / 8.1 us, 4096 11.5 / 9.9 / 11.2, 8192 18.0 / 16.4 / 16.4, 65536 159 / 137 / 134;
  // three heads of 64: 4096 6.7 / 6.1 / 6.6, 16384 18.2 / 14.4 / 13.2; appended, 24 heads of 128: 2048 6.8 / 7.2 / 8.8, 8191 19.7 / 19.2 / 19.8.
  p.R = p.rows >= 16384 ? 4 : p.rows >= 4096 ? 2 : 1;
  const size_t lds = (size_t)p.R * (p.rot / 2) * sizeof(float2);
  const long blocks = (p.rows + p.R - 1) / p.R;
  if (blocks >= 1L << 24) return AOT_ERR_UNSUPPORTED;          // (a launch's work items are below 2^32)
  auto go = [&](auto t, auto w) {
    using T = decltype(t);
    if constexpr (decltype(w)::value * sizeof(T) <= 16) hipLaunchKernelGGL((rope_kernel<T, decltype(w)::value, APPEND>), dim3((unsigned)blocks), dim3(256), lds, stream, p);
  };
  with_dtype(dtype, [&](auto t) {
    switch (ve) {
      case 8: go(t, std::integral_constant<int, 8>{}); break;
      case 4: go(t, std::integral_constant<int, 4>{}); break;
      case 2: go(t, std::integral_constant<int, 2>{}); break;
      default: go(t, std::integral_constant<int, 1>{}); break;
    }
  });
  AOT_LAUNCH_CHECK();
}

static bool rope_args_ok(int dtype, int H, int Hk, int D, int rot) {
  return dtype_size(dtype) && H >= 0 && Hk >= 0 && H + Hk > 0 && H <= 65536 && Hk <= 65536 && D > 0 && rot >= 2 && rot <= D && rot % 2 == 0;
}

extern "C" int aot_rope(const void* q, const void* k, void* qo, void* ko, const int* pos, const double* freqs, int dtype, int B, int S,
                        int H, int Hk, int D, int rot, int interleaved, int inverse, float mscale, const long* strides, void* stream) {
  if (!rope_args_ok(dtype, H, Hk, D, rot) || B < 0 || S < 0 || !strides) return AOT_ERR_BADARG;
  if (D > 1024) return AOT_ERR_UNSUPPORTED;
  if ((long)B * S == 0) return AOT_OK;
  if (!pos || !freqs || (H && (!q || !qo)) || (Hk && (!k || !ko))) return AOT_ERR_BADARG;
  RopeP p{};
  p.q = (const char*)q; p.k = (const char*)k; p.qo = (char*)qo; p.ko = (char*)ko;
  p.pos = pos; p.freqs = freqs;
  for (int i = 0; i < 3; ++i) { p.qs[i] = strides[i]; p.ks[i] = strides[3 + i]; p.qos[i] = strides[6 + i]; p.kos[i] = strides[9 + i]; }
  p.ps[0] = strides[12]; p.ps[1] = strides[13];
  p.rows = (long)B * S; p.S = S; p.H = H; p.Hk = Hk; p.D = D; p.rot = rot; p.inter = interleaved != 0;
  p.mscale = mscale; p.sign = inverse ? -1.f : 1.f;
  return rope_launch<false>(p, dtype, (hipStream_t)stream);
}

extern "C" int aot_rope_append(const void* q, const void* k, const void* v, void* qo, void* k_pages, void* v_pages, const int* pos,
                               const int* slots, const double* freqs, int dtype, int N, int H, int Hk, int D, int rot, int interleaved,
                               float mscale, int page, long num_pages, const long* strides, void* stream) {
  if (!rope_args_ok(dtype, H, Hk, D, rot) || N < 0 || Hk < 1 || !strides || page < 1 || (page & (page - 1)) || num_pages < 0) return AOT_ERR_BADARG;
  if (D > 1024 || num_pages * page > 0x7fffffffL) return AOT_ERR_UNSUPPORTED;
  if (N == 0) return AOT_OK;
  if (!pos || !freqs || !slots || !k || !v || !k_pages || !v_pages || (H && (!q || !qo))) return AOT_ERR_BADARG;
  RopeP p{};
  p.q = (const char*)q; p.k = (const char*)k; p.v = (const char*)v;
  p.qo = (char*)qo; p.ko = (char*)k_pages; p.vo = (char*)v_pages;
  p.pos = pos; p.slots = slots; p.freqs = freqs;
  for (int i = 0; i < 2; ++i) { p.qs[1 + i] = strides[i]; p.ks[1 + i] = strides[2 + i]; p.vs[1 + i] = strides[4 + i]; p.qos[1 + i] = strides[6 + i]; }
  for (int i = 0; i < 3; ++i) { p.kos[i] = strides[8 + i]; p.vos[i] = strides[11 + i]; }
  p.ps[0] = 0; p.ps[1] = 1;
  p.nslots = num_pages * page;
  while ((1 << p.page_shift) < page) ++p.page_shift;
  p.rows = N; p.S = 1; p.H = H; p.Hk = Hk; p.D = D; p.rot = rot; p.inter = interleaved != 0;
  p.mscale = mscale; p.sign = 1.f;
  return rope_launch<true>(p, dtype, (hipStream_t)stream);
}
