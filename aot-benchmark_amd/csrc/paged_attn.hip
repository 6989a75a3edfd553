// Attention of one new token per sequence over a paged key / value cache:
//   s_t = cap tanh(scale q.k_t / cap) - slope (dist to t),   out = sum_t softmax(s)_t v_t,   weights_t += sum over the group's heads of p_t
//
// Bound by memory: K and V are read once, 4 D bytes a 16-bit entry and key head, against 4 G D operations (G query heads share a key
// head) -- 1 to 8 operations a byte.  A workgroup takes one key head of one sequence and one chunk of the cache's length; its four
// waves take blocks of 32 entries in turn, and everything a wave needs goes from global memory straight into the registers the
// matrix instructions read:
//   scores    S^T [16 entries x 16 heads] = K . Q^T on 16x16 tiles: a lane holds one entry's row (lane & 15) and a 16-byte piece of it
//             (lane >> 4), the heads' queries stay in registers.
//   values    O^T [16 rows x 16 heads] = V^T . P^T.  A tile's score registers are four consecutive entries (4 (lane >> 4) + r): taken as
//             the reduction index they make P^T the second operand as it lies, with no exchange between lanes.  V^T is loaded with
//             the same entries in the same lane -- eight rows of E consecutive elements, 16 lanes a row: whole lines -- and the rows'
//             i-th elements are gathered by byte permutes into the tile of output rows { E m + i }.
// No shared memory in the loop, no barrier: a wave's loads run ahead of its arithmetic.  The running maximum and sum are per head =
// per lane (& 15); the four waves join through shared memory and, when the length is split, leave (O, m, l) in a workspace that
// paged_join_kernel adds up in index order (no atomics: results repeat bit for bit).  Collected weights need the final maximum and
// sum, so the scores (4 bytes a head and entry, 1/64 of the cache's bytes at D = 128 and 16 bits) are left in the workspace too.
// Scores, probabilities, sums and outputs are 32-bit; a probability is rounded to the cache's type on its way into the P.V product
// (at most 2^-9 of itself for bf16, unbiased; fp16's are held 2^15 times as large meanwhile), while the sum that divides uses the
// unrounded ones.
#include "seq_common.h"

struct PagedP {
  const char *q, *k, *v;
  char* out;
  const int *table, *lengths, *key_pos;
  const float* slopes;
  float *weights, *part, *ml, *scores;
  long qs[2], os[2], ks[3], vs[3], t_s, ws[2], ps[2];
  long num_pages, S;
  int B, H, Hk, G, D, cap_len, page_shift, chunk, nsplit, osplit;
  float scale, softcap;
  Cap cap;
};

template <class T> __device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 c) {
  if constexpr (std::is_same<T, f16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else if constexpr (std::is_same<T, bf16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
}

// the row of entry t of this (sequence, head), or null past the end / on a page outside the pool
template <class T> __device__ __forceinline__ const T* entry(const char* pages, const long* st, const int* table, int t, int len, int h, const PagedP& p) {
  if (t >= len) return nullptr;
  const long pg = table[t >> p.page_shift];
  if (pg < 0 || pg >= p.num_pages) return nullptr;
  return (const T*)pages + pg * st[0] + (long)(t & ((1 << p.page_shift) - 1)) * st[1] + (long)h * st[2];
}

template <class T, int DP, bool SPLIT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (DP == 128 ? 3 : DP == 256 ? 2 : 1) : DP == 128 ? 2 : 1) void paged_attn_kernel(PagedP p) {
  constexpr int CE = Elem<T>::CE, NC = DP / (4 * CE), E = DP / 16, EW = E * sizeof(T) / 4;   // EW dwords of a row a lane holds,
  constexpr int PW = EW < 4 ? EW : 4;                                                       // PW of them a load
  __shared__ float sm[4][16], sl[4][16];
  __shared__ float so[2][16][DP + 4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const int qt = blockIdx.y / p.Hk, hk = blockIdx.y - qt * p.Hk, b = blockIdx.z, split = blockIdx.x;
  const int len = max(0, min(p.lengths[b], p.cap_len));
  const int t_begin = split * p.chunk, t_end = min(len, t_begin + p.chunk);
  if (SPLIT && t_begin >= len) return;
  const int g = qt * 16 + n;                                   // head within the group
  const bool live = g < p.G;
  const int h = hk * p.G + min(g, p.G - 1);
  const int* table = p.table + b * p.t_s;

  u32x4 qf[NC];
  {
    const T* q = (const T*)p.q + b * p.qs[0] + h * p.qs[1];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = (c * 4 + kg) * CE;
      qf[c] = live && d < p.D ? *(const u32x4*)(q + d) : u32x4{0, 0, 0, 0};
    }
  }
  const bool capped = p.softcap > 0.f;
  const Cap cap = p.cap;
  const float slope = p.slopes ? p.slopes[h] * LOG2E : 0.f;
  const int* kpos = p.key_pos ? p.key_pos + b * p.ps[0] + hk * p.ps[1] : nullptr;
  const int qpos = len > 0 ? (kpos ? kpos[len - 1] : len - 1) : 0;

  f32x4 o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = NEG_INF, l = 0.f;

  // A block's pages: one lookup for each half of 16 entries, wave-uniform; -1 where a lane-wise look at every entry is needed
  const bool coarse = p.page_shift >= 4;
  struct Pages { int a, b; };
  auto pages_of = [&](int t0) {
    Pages r{-1, -1};
    if (coarse && t0 + 32 <= len) {
      r.a = __builtin_amdgcn_readfirstlane(table[t0 >> p.page_shift]);
      r.b = __builtin_amdgcn_readfirstlane(table[(t0 + 16) >> p.page_shift]);
      if (r.a >= p.num_pages || r.b >= p.num_pages) r.a = -1;
      if (r.b < 0) r.a = -1;
    }
    return r;
  };
  struct Block { u32x4 kf[2][NC]; unsigned vf[8][EW]; unsigned ok; };
  const long in_mask = (1 << p.page_shift) - 1;
  const long k_lane = n * p.ks[1], v_lane = 4 * kg * p.vs[1];
  auto load = [&](Block& x, int t0, const Pages& pg) {
    if (pg.a >= 0) {
      x.ok = 255;
#pragma unroll
      for (int T2 = 0; T2 < 2; ++T2) {
        const long page = T2 ? pg.b : pg.a, in = (t0 + 16 * T2) & in_mask;
        const T* kb = (const T*)p.k + page * p.ks[0] + in * p.ks[1] + hk * p.ks[2];
        const T* vb = (const T*)p.v + page * p.vs[0] + in * p.vs[1] + hk * p.vs[2];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int d = (c * 4 + kg) * CE;
          x.kf[T2][c] = d < p.D ? *(const u32x4*)(kb + k_lane + d) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < EW / PW; ++i) {
            typedef unsigned piece __attribute__((ext_vector_type(PW)));
            const int d = n * E + i * PW * 4 / (int)sizeof(T);
            piece y = {};
            if (d < p.D) y = *(const piece*)(vb + r * p.vs[1] + v_lane + d);
#pragma unroll
            for (int w = 0; w < PW; ++w) x.vf[4 * T2 + r][i * PW + w] = y[w];
          }
      }
      return;
    }
    x.ok = 0;
#pragma unroll
    for (int T2 = 0; T2 < 2; ++T2) {
      const T* row = entry<T>(p.k, p.ks, table, t0 + T2 * 16 + n, len, hk, p);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = (c * 4 + kg) * CE;
        x.kf[T2][c] = row && d < p.D ? *(const u32x4*)(row + d) : u32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const T* row = entry<T>(p.v, p.vs, table, t0 + (j >> 2) * 16 + kg * 4 + (j & 3), len, hk, p);
      x.ok |= (row != nullptr) << j;
#pragma unroll
      for (int i = 0; i < EW / PW; ++i) {                       // (D is whole 16-byte pieces: none is cut)
        typedef unsigned piece __attribute__((ext_vector_type(PW)));
        const int d = n * E + i * PW * 4 / (int)sizeof(T);
        piece y = {};
        if (row && d < p.D) y = *(const piece*)(row + d);
#pragma unroll
        for (int w = 0; w < PW; ++w) x.vf[j][i * PW + w] = y[w];
      }
    }
  };
  Block blk;
  const int t_first = t_begin + wave * 32;
  Pages pg = t_first < t_end ? pages_of(t_first) : Pages{-1, -1};
  for (int t0 = t_first; t0 < t_end; t0 += 128) {
    load(blk, t0, pg);
    if (t0 + 128 < t_end) pg = pages_of(t0 + 128);
    auto& kf = blk.kf;
    auto& vf = blk.vf;
    f32x4 s[2];
#pragma unroll
    for (int T2 = 0; T2 < 2; ++T2) {
      s[T2] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) s[T2] = mfma16<T>(kf[T2][c], qf[c], s[T2]);
    }
    float x[8], mx = NEG_INF;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = t0 + (j >> 2) * 16 + kg * 4 + (j & 3);
      const float raw = s[j >> 2][j & 3];
      float y = capped ? cap(raw) : raw * cap.lin;
      if (p.slopes) y -= slope * fabsf((float)(qpos - (kpos ? (blk.ok >> j & 1 ? kpos[t] : 0) : t)));
      x[j] = blk.ok >> j & 1 ? y : NEG_INF;
      mx = fmaxf(mx, x[j]);
    }
    if (p.weights && live) {                                     // (a row of scores is whole groups of four)
      float* sc = p.scores + ((long)b * p.H + h) * p.S + t0 + kg * 4;
#pragma unroll
      for (int T2 = 0; T2 < 2; ++T2)
        if (t0 + T2 * 16 + kg * 4 < t_end) *(f32x4*)(sc + T2 * 16) = f32x4{x[4 * T2], x[4 * T2 + 1], x[4 * T2 + 2], x[4 * T2 + 3]};
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float m2 = fmaxf(m, mx), base = m2 == NEG_INF ? 0.f : m2;      // nothing seen yet: exp2(-inf - 0) = 0 everywhere
    const float f = exp2_hw(m - base), low = base - LIFT<T>;
    m = m2;
    float pr[8], add = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) { pr[j] = exp2_hw(x[j] - low); add += pr[j]; }
    l = l * f + add;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= f;
    if constexpr (sizeof(T) == 2) {
      u32x4 pf;
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[i] = pack2<T>(pr[2 * i], pr[2 * i + 1]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        u32x4 a;
#pragma unroll
        for (int i = 0; i < 4; ++i)        // element e of rows 2i and 2i + 1
          a[i] = __builtin_amdgcn_perm(vf[2 * i + 1][e >> 1], vf[2 * i][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
        o[e] = mfma16<T>(a, pf, o[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int j = 0; j < 8; ++j) o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vf[j][e]), pr[j], o[e], 0, 0, 0);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // join the four waves: common maximum, then the waves' scaled O two and two through shared memory
  if (kg == 0) { sm[wave][n] = m; sl[wave][n] = l; }
  __syncthreads();
  float M = NEG_INF, L = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w][n]);
  const float mb = M == NEG_INF ? 0.f : M;
#pragma unroll
  for (int w = 0; w < 4; ++w) L += sl[w][n] * exp2_hw(sm[w][n] - mb);
  const float f = exp2_hw(m - mb);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] *= f;
  for (int step = 2; step >= 1; step >>= 1) {                  // waves 2, 3 -> 0, 1; then 1 -> 0
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) so[wave - step][n][E * (4 * kg + r) + e] = o[e][r];
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[e][r] += so[wave][n][E * (4 * kg + r) + e];
    }
    __syncthreads();
  }
  if (wave != 0 || !live) return;
  if (SPLIT) {
    float* part = p.part + (((long)b * p.H + h) * p.nsplit + split) * p.D;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = E * (4 * kg + r) + e;
        if (d < p.D) part[d] = o[e][r];
      }
    if (kg == 0) {
      float* ml = p.ml + (((long)b * p.H + h) * p.nsplit + split) * 2;
      ml[0] = M;
      ml[1] = L;
    }
  } else {
    T* out = (T*)p.out + b * p.os[0] + h * p.os[1];
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);            // no entry: zero; a NaN stays one
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = E * (4 * kg + r) + e;
        if (d < p.D) out[d] = (T)(o[e][r] * inv);
      }
  }
}

// First B * H (* osplit) workgroups: out = sum over the splits; thread groups of D / 4 take every so-many-th split, their sums are added in a fixed
// order.  The others: weights += group sum of exp2(s - M) / L for 1024 entries of one key head, four a thread; every one forms (M, L) of its
// heads from the splits' pairs, a wave a head.
static constexpr int JOIN_KEYS = 1024;
template <class T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedP p) {
  __shared__ float fac[1024];
  __shared__ float red[8];
  __shared__ f32x4 sum[256];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const long nout = (long)p.B * p.H;
  auto live_sum = [](float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); };      // no entry: zero; a NaN stays one
  if (blockIdx.x < nout * p.osplit) {
    const int bh0 = blockIdx.x / p.osplit, cut = blockIdx.x - bh0 * p.osplit, b = bh0 / p.H, h = bh0 - b * p.H;
    const int len = max(0, min(p.lengths[b], p.cap_len)), ns = (len + p.chunk - 1) / p.chunk;
    const long at = ((long)b * p.H + h) * p.nsplit;
    const float* ml = p.ml + at * 2;
    float m = NEG_INF, l = 0.f;
    for (int i = tid; i < ns; i += 256) m = fmaxf(m, ml[2 * i]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) red[wave] = m;
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), mb = M == NEG_INF ? 0.f : M;
    for (int i = tid; i < ns; i += 256) {
      const float f = exp2_hw(ml[2 * i] - mb);
      fac[i] = f;
      l += ml[2 * i + 1] * f;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    if (lane == 0) red[4 + wave] = l;
    __syncthreads();
    const float inv = live_sum(red[4] + red[5] + red[6] + red[7]);
    const int nd = p.D / p.osplit / 4, groups = 256 / nd, g = tid / nd, d = cut * nd * 4 + (tid - g * nd) * 4;   // D is a multiple of 4, at most 256
    f32x4 a{0.f, 0.f, 0.f, 0.f};
    if (g < groups) {
#pragma unroll 4
      for (int i = g; i < ns; i += groups) a += *(const f32x4*)(p.part + (at + i) * p.D + d) * fac[i];
      sum[tid] = a;
    }
    __syncthreads();
    if (g == 0) {
      for (int i = 1; i < groups; ++i) a += sum[i * nd + tid];
      T* out = (T*)p.out + b * p.os[0] + h * p.os[1] + d;
#pragma unroll
      for (int w = 0; w < 4; ++w) out[w] = (T)(a[w] * inv);
    }
    return;
  }
  const long w = blockIdx.x - nout * p.osplit;
  const int tiles = (p.cap_len + JOIN_KEYS - 1) / JOIN_KEYS;
  const int tile = (int)(w % tiles), bh = (int)(w / tiles), b = bh / p.Hk, hk = bh - b * p.Hk;
  const int len = max(0, min(p.lengths[b], p.cap_len)), ns = (len + p.chunk - 1) / p.chunk;
  const int t0 = tile * JOIN_KEYS;
  if (t0 >= len) return;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int g0 = 0; g0 < p.G; g0 += 4) {
    const int n = min(4, p.G - g0);
    if (wave < n) {
      const float* ml = p.ml + ((long)b * p.H + hk * p.G + g0 + wave) * p.nsplit * 2;
      float m = NEG_INF, l = 0.f;
      for (int i = lane; i < ns; i += 64) m = fmaxf(m, ml[2 * i]);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
      const float mb = m == NEG_INF ? 0.f : m;
      for (int i = lane; i < ns; i += 64) l += ml[2 * i + 1] * exp2_hw(ml[2 * i] - mb);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
      if (lane == 0) { red[wave] = mb - LIFT<T>; red[4 + wave] = live_sum(l); }      // (the sums are of lifted probabilities)
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) {
      const float* sc = p.scores + ((long)b * p.H + hk * p.G + g0 + i) * p.S;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = t0 + tid + 256 * k;
        if (t < len) acc[k] += exp2_hw(sc[t] - red[i]) * red[4 + i];
      }
    }
    __syncthreads();
  }
  float* out = p.weights + b * p.ws[0] + hk * p.ws[1];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int t = t0 + tid + 256 * k;
    if (t < len) out[t] += acc[k];
  }
}

static long pow2_at_least(long x) {
  long r = 1;
  while (r < x) r <<= 1;
  return r;
}

// Entries a workgroup takes: a multiple of the waves' 4 x 32, as long as the rows alone fill the chip's 256 CUs eight deep and no row is
// cut into more than 1024; the length that counts is the table's capacity (the true ones live on the device).
static int paged_chunk(long rows, long cap) {
  const long target = 2048;
  const long want = std::max(1L, target / std::max(1L, rows));
  long chunk = (cap + want - 1) / want;
  chunk = std::max(chunk, (cap + 1023) / 1024);
  return (int)std::max(128L, pow2_at_least(chunk));             // (a capacity is at most 2^30)
}

// workspace: sums [B * H][nsplit][D], their (m, l), scores [B * H][capacity in whole groups of four]
static long score_row(long cap) { return (cap + 3) / 4 * 4; }
static long part_floats(int B, int H, int D, int nsplit) { return ((long)B * H * nsplit * (D + 2) + 3) / 4 * 4; }
static long paged_work(int B, int H, int Hk, int D, long cap, int with_weights, int* chunk, int* nsplit) {
  const int G = H / Hk, qt = (G + 15) / 16;
  *chunk = paged_chunk((long)B * Hk * qt, cap);
  *nsplit = (int)std::max(1L, (cap + *chunk - 1) / *chunk);
  if (*nsplit == 1 && !with_weights) return 0;
  return part_floats(B, H, D, *nsplit) + (with_weights ? (long)B * H * score_row(cap) : 0);
}

extern "C" int aot_paged_attn_work_floats(int B, int H, int Hk, int D, int page, int max_pages, int with_weights, long* floats) {
  if (!floats || B < 0 || Hk < 1 || H < Hk || H % Hk || D < 1 || page < 1 || max_pages < 0) return AOT_ERR_BADARG;
  if ((long)page * max_pages > (1L << 30)) return AOT_ERR_UNSUPPORTED;
  int c, n;
  *floats = paged_work(B, H, Hk, D, (long)page * max_pages, with_weights, &c, &n);
  return AOT_OK;
}

extern "C" int aot_paged_attn(const void* q, const void* k_pages, const void* v_pages, const int* table, const int* lengths, const float* slopes,
                              const int* key_pos, float* weights, void* out, float* work, long work_floats, int dtype, int B, int H, int Hk,
                              int D, int page, int max_pages, long num_pages, float scale, float softcap, const long* strides, void* stream) {
  const int es = dtype_size(dtype);
  if (!es || B < 0 || Hk < 1 || H < Hk || H % Hk || D < 1 || page < 1 || (page & (page - 1)) || max_pages < 0 || num_pages < 0 || !strides ||
      !(softcap >= 0.f && softcap < __builtin_inff()) || !(scale > 0.f && scale < __builtin_inff())) return AOT_ERR_BADARG;
  const long cap = (long)page * max_pages;
  const int G = H / Hk, qt = (G + 15) / 16;
  if (D > 256 || D * es % 16 || cap > (1L << 30) || num_pages * page > 0x7fffffffL || B > 65535 || (long)Hk * qt > 65535) return AOT_ERR_UNSUPPORTED;
  if (B == 0) return AOT_OK;
  if (!q || !lengths || !out || (cap && !table) || (num_pages && (!k_pages || !v_pages))) return AOT_ERR_BADARG;
  PagedP p{};
  p.q = (const char*)q; p.k = (const char*)k_pages; p.v = (const char*)v_pages; p.out = (char*)out;
  p.table = table; p.lengths = lengths; p.slopes = slopes; p.key_pos = key_pos; p.weights = weights;
  for (int i = 0; i < 2; ++i) { p.qs[i] = strides[i]; p.os[i] = strides[2 + i]; p.ws[i] = strides[11 + i]; p.ps[i] = strides[13 + i]; }
  for (int i = 0; i < 3; ++i) { p.ks[i] = strides[4 + i]; p.vs[i] = strides[7 + i]; }
  p.t_s = strides[10];
  const long a16 = 16 / es;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || p.qs[0] % a16 || p.qs[1] % a16) return AOT_ERR_BADARG;
  for (int i = 0; i < 3; ++i) if (p.ks[i] % a16 || p.vs[i] % a16) return AOT_ERR_BADARG;
  p.num_pages = num_pages;
  p.B = B; p.H = H; p.Hk = Hk; p.G = G; p.D = D; p.cap_len = (int)cap; p.S = score_row(cap);
  while ((1 << p.page_shift) < page) ++p.page_shift;
  p.scale = scale; p.softcap = softcap; p.cap = Cap::of(scale, softcap);
  const long need = paged_work(B, H, Hk, D, cap, weights != nullptr, &p.chunk, &p.nsplit);
  if (need && (!work || !aligned16(work) || work_floats < need)) return AOT_ERR_BADARG;
  p.part = work;
  p.ml = work + (long)B * H * p.nsplit * D;
  p.scores = work + part_floats(B, H, D, p.nsplit);
  const bool split = need > 0;
  // A head's sums by 32 columns a workgroup where they are 64 KB and more: the reading of one workgroup outweighs that of the splits' (m, l) by each.
  // Join with whole heads / by columns: D = 128, 64 splits 4.1 / 4.3 us, 128 5.4 / 4.6, 1024 8.8 / 6.0; D = 256, 64 splits 5.2 / 4.8, 1024 14.8 / 6.5.
  p.osplit = (long)p.nsplit * D >= 16384 && D % 32 == 0 ? D / 32 : 1;
  const long joins = (long)B * H * p.osplit + (weights ? (long)B * Hk * ((cap + JOIN_KEYS - 1) / JOIN_KEYS) : 0);
  if (split && joins >= 1L << 24) return AOT_ERR_UNSUPPORTED;     // (a launch's work items are below 2^32)
  const dim3 grid(p.nsplit, Hk * qt, B);
  hipStream_t st = (hipStream_t)stream;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto dp) {
      if (split) hipLaunchKernelGGL((paged_attn_kernel<T, decltype(dp)::value, true>), grid, dim3(256), 0, st, p);
      else hipLaunchKernelGGL((paged_attn_kernel<T, decltype(dp)::value, false>), grid, dim3(256), 0, st, p);
    };
    if (D <= 32) go(std::integral_constant<int, 32>{});
    else if (D <= 64) go(std::integral_constant<int, 64>{});
    else if (D <= 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (split) {
    with_dtype(dtype, [&](auto t) { hipLaunchKernelGGL((paged_join_kernel<decltype(t)>), dim3((unsigned)joins), dim3(256), 0, st, p); });
  }
  AOT_LAUNCH_CHECK();
}
