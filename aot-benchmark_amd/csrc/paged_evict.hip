// Eviction from a paged cache by accumulated attention weight.  Every (sequence, key head) row keeps `budget` of its entries: the
// first `sink`, the last `recent`, and of the others the heaviest, ties to the lower index; NaN weights count as the lightest.  The
// kept entries move, in order, into the pages of new_table, so pages that other sequences share stay as they are.
//
// Two launches.  Select: one workgroup a row; a radix select (three digits of an order-preserving key, histograms in shared memory) finds
// the weight of the last entry that stays, ballots turn the kept flags into places.  It is bound by reading the weights (rows of up
// to 16384 once, longer ones five times, from L2 after the first) and by latency.  Move: 16-byte pieces of the kept K / V rows, bound by
// memory: each kept row is read once and written once.
#include "seq_common.h"

static constexpr int SEL_T = 1024, HOLD = 16;

// larger key = heavier; -0 and +0 alike; NaN below everything
__device__ __forceinline__ unsigned weight_key(float w) {
  if (w != w) return 0u;
  const unsigned u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct EvictP {
  const int *table, *new_table, *lengths, *pos;
  const float* weights;
  int *kept, *new_lengths, *new_pos;
  float* new_weights;
  char *k, *v;
  long ks[3], vs[3], ws[2], nws[2], pss[2], nps[2], num_pages;
  long t_s, nt_s;
  int B, Hk, S, cap, budget, sink, recent, page_shift, max_pages, new_pages, es, D;
};

// exclusive prefix of x over the workgroup; total in *sum
__device__ __forceinline__ int block_scan(int x, int* lds, int* sum) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int inc = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 63) lds[w] = inc;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int i = 0; i < SEL_T / 64; ++i) {
    const int n = lds[i];
    if (i < w) base += n;
    all += n;
  }
  __syncthreads();
  *sum = all;
  return base + inc - x;
}

template <bool HELD>
__global__ __launch_bounds__(SEL_T) void evict_select_kernel(EvictP p) {
  __shared__ int hist[2048];
  __shared__ int scan[SEL_T / 64];
  __shared__ int pick[2];
  __shared__ int counts[SEL_T / 64][2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = max(0, min(p.lengths[b], p.cap));
  const float* w = p.weights + b * p.ws[0] + h * p.ws[1];
  int* kept = p.kept + ((long)b * p.Hk + h) * p.budget;
  const int keep = min(len, p.budget);
  const int lo = min(p.sink, len), hi = max(lo, len - p.recent);            // the contested middle
  const int want = keep - lo - (len - hi);                                  // how many of it stay (all of it if nothing has to go)
  // a wave owns a run of entries, 64 at a time; up to HOLD of them a lane stay in registers (HELD: the row is at most HOLD * SEL_T long),
  // so a row of 16384 is read once instead of five times: 33 us for 128 rows, 29 held
  const int per = ((len + SEL_T - 1) / SEL_T) * 64, t0 = min(wave * per, len), t1 = min(t0 + per, len), steps = per / 64;
  unsigned held[HELD ? HOLD : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      const int t = t0 + lane + 64 * i;
      held[i] = i < steps && t < t1 ? weight_key(w[t]) : 0u;
    }
  }
  auto each = [&](auto&& f) {                                               // f(entry, its key), the same order every time
    if constexpr (HELD) {
#pragma unroll
      for (int i = 0; i < HOLD; ++i)
        if (i < steps) f(t0 + lane + 64 * i, held[i]);
    } else {
      for (int t = t0 + lane; t < t0 + per; t += 64) f(t, t < t1 ? weight_key(w[t]) : 0u);
    }
  };
  unsigned thr = 0;
  int ties = 0;                                                             // of the entries equal to thr the first `ties` stay
  const bool all = keep == len;
  if (!all && want > 0) {
    // Digits of 11, 11 and 10 bits: the first holds sign, exponent and two mantissa bits, so that weights of one magnitude still spread over
    // several counters (with 8 bits a wave's 64 additions met in one or two and queued: 41 us for 128 rows of 16384, 33 with these)
    unsigned prefix = 0;
    int left = want;
#pragma unroll 1
    for (int d = 0; d < 3; ++d) {
      const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
      const unsigned digit = d == 2 ? 1023u : 2047u, above = d == 0 ? 0u : d == 1 ? ~0u << 21 : ~0u << 10;
      hist[tid] = 0;
      hist[tid + SEL_T] = 0;
      __syncthreads();
      each([&](int t, unsigned key) {
        if (t >= lo && t < min(hi, t1) && (key & above) == prefix) atomicAdd(&hist[(key >> shift) & digit], 1);
      });
      __syncthreads();
      const int c1 = hist[2047 - 2 * tid], c0 = hist[2046 - 2 * tid];       // from the heaviest digit down: where does `left` run out
      int sum;
      const int before = block_scan(c1 + c0, scan, &sum);
      if (before < left && before + c1 + c0 >= left) {
        const bool first = before + c1 >= left;
        pick[0] = first ? 2047 - 2 * tid : 2046 - 2 * tid;
        pick[1] = first ? left - before : left - before - c1;
      }
      __syncthreads();
      prefix |= (unsigned)pick[0] << shift;
      left = pick[1];
      __syncthreads();
    }
    thr = prefix;
    ties = left;
  }
  // count, exchange the waves' counts, then place the kept entries by ballots
  const unsigned long long below = (1ull << lane) - 1;
  auto kind = [&](int t, unsigned key, bool& sure, bool& tie) {
    const bool mid = !all && t >= lo && t < hi;
    sure = t < t1 && (!mid || (want > 0 && key > thr));
    tie = t < t1 && mid && want > 0 && key == thr;
  };
  int heavier = 0, equal = 0;
  each([&](int t, unsigned key) {
    bool sure, tie;
    kind(t, key, sure, tie);
    heavier += __popcll(__ballot(sure));
    equal += __popcll(__ballot(tie));
  });
  if (lane == 0) { counts[wave][0] = heavier; counts[wave][1] = equal; }
  __syncthreads();
  int at = 0, eq = 0;
  for (int i = 0; i < wave; ++i) {
    at += counts[i][0] + max(0, min(counts[i][1], ties - eq));
    eq += counts[i][1];
  }
  float* nw = p.new_weights + b * p.nws[0] + h * p.nws[1];
  const int* pos = p.pos ? p.pos + b * p.pss[0] + h * p.pss[1] : nullptr;
  int* np = p.pos ? p.new_pos + b * p.nps[0] + h * p.nps[1] : nullptr;
  each([&](int t, unsigned key) {
    bool sure, tie;
    kind(t, key, sure, tie);
    const unsigned long long teq = __ballot(tie);
    const bool stay = sure || (tie && eq + __popcll(teq & below) < ties);
    const unsigned long long go = __ballot(stay);
    if (stay) {
      const int j = at + __popcll(go & below);
      kept[j] = t;
      nw[j] = w[t];                                                         // (the weight itself: a key forgets -0 and NaN's bits)
      if (pos) np[j] = pos[t];
    }
    at += __popcll(go);
    eq += __popcll(teq);
  });
  for (int i = keep + tid; i < p.budget; i += SEL_T) kept[i] = -1;
  for (int i = keep + tid; i < p.S; i += SEL_T) {
    nw[i] = 0.f;
    if (pos) np[i] = 0;
  }
  if (h == 0 && tid == 0) p.new_lengths[b] = keep;
}

// 16-byte pieces of the kept rows: a workgroup moves ROWS places of one (b, h), K and V
static constexpr int MOVE_ROWS = 32;
template <class V>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictP p, int pieces, int up_shift) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int* kept = p.kept + ((long)b * p.Hk + h) * p.budget;
  const int up = 1 << up_shift, u0 = threadIdx.x & (up - 1), r0 = threadIdx.x >> up_shift, step = 256 >> up_shift;
  const int j0 = blockIdx.x * MOVE_ROWS;
  const int pm = (1 << p.page_shift) - 1;
  for (int j = j0 + r0; j < min(j0 + MOVE_ROWS, p.budget); j += step) {
    const int t = kept[j];
    if (t < 0) break;
    const long sp = p.table[b * p.t_s + (t >> p.page_shift)], dp = p.new_table[b * p.nt_s + (j >> p.page_shift)];
    if (sp < 0 || sp >= p.num_pages || dp < 0 || dp >= p.num_pages) continue;
    const long si = t & pm, di = j & pm;
    const V* ks = (const V*)(p.k + (sp * p.ks[0] + si * p.ks[1] + h * p.ks[2]) * p.es);
    const V* vs = (const V*)(p.v + (sp * p.vs[0] + si * p.vs[1] + h * p.vs[2]) * p.es);
    V* kd = (V*)(p.k + (dp * p.ks[0] + di * p.ks[1] + h * p.ks[2]) * p.es);
    V* vd = (V*)(p.v + (dp * p.vs[0] + di * p.vs[1] + h * p.vs[2]) * p.es);
    for (int u = u0; u < pieces; u += up) {
      const V a = ks[u], c = vs[u];
      kd[u] = a;
      vd[u] = c;
    }
  }
}

extern "C" int aot_paged_evict(void* k_pages, void* v_pages, const int* table, const int* new_table, const int* lengths, const float* weights,
                               const int* key_pos, int* kept, int* new_lengths, float* new_weights, int* new_key_pos, int dtype, int B, int Hk,
                               int D, int S, int page, int max_pages, int new_pages, long num_pages, int budget, int sink, int recent,
                               const long* strides, void* stream) {
  const int es = dtype_size(dtype);
  if (!es || B < 0 || Hk < 1 || D < 1 || S < 0 || page < 1 || (page & (page - 1)) || max_pages < 0 || new_pages < 0 || num_pages < 0 || !strides ||
      budget < 1 || sink < 0 || recent < 0 || (long)sink + recent > budget || (long)new_pages * page < budget) return AOT_ERR_BADARG;
  // (a row's entries, and the runs of them that the waves take, are counted in 32 bits; a launch's work items are below 2^32)
  if (num_pages * page > 0x7fffffffL || (long)max_pages * page > (1L << 30) || (long)new_pages * page > (1L << 30) || budget >= 1 << 29 || B > 65535 ||
      Hk > 65535) return AOT_ERR_UNSUPPORTED;
  if (B == 0) return AOT_OK;
  if (!k_pages || !v_pages || !table || !new_table || table == new_table || !lengths || !weights || !kept || !new_lengths || !new_weights ||
      new_weights == weights || lengths == new_lengths || (key_pos && (!new_key_pos || new_key_pos == key_pos))) return AOT_ERR_BADARG;
  EvictP p{};
  p.table = table; p.new_table = new_table; p.lengths = lengths; p.pos = key_pos; p.weights = weights;
  p.kept = kept; p.new_lengths = new_lengths; p.new_pos = new_key_pos; p.new_weights = new_weights;
  p.k = (char*)k_pages; p.v = (char*)v_pages;
  for (int i = 0; i < 3; ++i) { p.ks[i] = strides[i]; p.vs[i] = strides[3 + i]; }
  p.t_s = strides[6]; p.nt_s = strides[7];
  for (int i = 0; i < 2; ++i) { p.ws[i] = strides[8 + i]; p.nws[i] = strides[10 + i]; p.pss[i] = strides[12 + i]; p.nps[i] = strides[14 + i]; }
  p.num_pages = num_pages;
  p.B = B; p.Hk = Hk; p.D = D; p.S = S; p.budget = budget; p.sink = sink; p.recent = recent; p.es = es;
  p.max_pages = max_pages; p.new_pages = new_pages;
  p.cap = (int)std::min((long)S, (long)max_pages * page);
  while ((1 << p.page_shift) < page) ++p.page_shift;
  int piece = 16;
  auto fits = [&](int n) {
    if ((D * es) % n || (uintptr_t)k_pages % n || (uintptr_t)v_pages % n) return false;
    for (int i = 0; i < 3; ++i) if ((p.ks[i] * es) % n || (p.vs[i] * es) % n) return false;
    return true;
  };
  while (piece > es && !fits(piece)) piece >>= 1;
  hipStream_t st = (hipStream_t)stream;
  if (p.cap <= HOLD * SEL_T) hipLaunchKernelGGL(evict_select_kernel<true>, dim3(Hk, B), dim3(SEL_T), 0, st, p);
  else hipLaunchKernelGGL(evict_select_kernel<false>, dim3(Hk, B), dim3(SEL_T), 0, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  const int pieces = D * es / piece;
  int up = 0;
  while ((1 << up) < pieces && up < 8) ++up;
  const dim3 grid(cdiv(budget, MOVE_ROWS), Hk, B);
  if (piece == 16) hipLaunchKernelGGL(evict_move_kernel<u32x4>, grid, dim3(256), 0, st, p, pieces, up);
  else if (piece == 8) hipLaunchKernelGGL(evict_move_kernel<u32x2>, grid, dim3(256), 0, st, p, pieces, up);
  else if (piece == 4) hipLaunchKernelGGL(evict_move_kernel<unsigned>, grid, dim3(256), 0, st, p, pieces, up);
  else hipLaunchKernelGGL(evict_move_kernel<u16>, grid, dim3(256), 0, st, p, pieces, up);
  AOT_LAUNCH_CHECK();
}
