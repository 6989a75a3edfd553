// Attention under masks, forward and backward, for whole sequences of queries.  For query i of Sq (place i + off in the key sequence,
// off = Sk - Sq) and key t of Sk:
//   s = cap tanh(scale q_i.k_t / cap) - slope_h |i + off - t|          (cap = 0: no cap)
//   seen(i, t): (not causal or t <= i + off or t < prefix_b) and (no documents or doc_q[i] == doc_k[t] >= 0)
//   p = softmax of s over the seen keys, o = sum p v; a row that sees nothing is zero, with zero gradients.
// Backward, with D_i = do_i.o_i:  dv_t = sum_i p do_i;  ds = p (do_i.v_t - D_i) (1 - tanh^2);  dq_i = scale sum_t ds k_t;
// dk_t = scale sum_i ds q_i, both over the query heads that share the key head.
//
// Bound by the matrix cores and the exponentials: 4 D operations and one exponential a pair forward, 10 D backward.  Everything is
// built on 32x32 tiles whose score registers are at once the second operand of the next product:
//   a wave owns 32 columns (queries; in the key gradient's kernel: keys), one a lane; a score tile's registers run over rows
//   8 (r / 4) + 4 (lane / 32) + r % 4 of the other side.  With exactly those rows as the reduction index of the following product the
//   tile needs no exchange between lanes -- the first operand is read in the same order, transposed, from shared memory
//   (ds_read_b64_tr_b16: four rows of one column a lane; fp32: one element).
// Four waves share tiles of the other side, staged through registers into two buffers (one barrier a tile); 16-byte pieces are
// xor-swizzled by their row, so both the row reads and the transposed reads spread over the banks.
// The gradients of q and of k / v are separate kernels, each the only writer of its rows: no atomics, the result repeats bit for bit,
// for 7 products instead of 5.  Tiles that no pair of is seen in are never visited: causal bounds, and per 64 tokens the smallest and
// largest document id (doc_range_kernel), tested 64 tiles at a time by one ballot.
//
// Masked places may hold anything.  A masked score is replaced, never multiplied; where a masked row would enter a product with
// weight zero (0 * inf is NaN), infinities and NaN of a tile with a mask are replaced by zero -- forward as V is staged, backward in shared
// memory once the tile's scores, which see them, are formed; if there were any, a second walk over those tiles counts the seen ones (the
// same product, of 0 / 1 weights and small codes) and adds what they make of the sums.
//
// Scores, statistics and sums are 32-bit.  p and ds are rounded to the inputs' type for the following product (nearest even: 2^-9 of
// the value for bf16, 2^-12 for fp16), the sum that divides is not.  fp16 ends at 6e-8, so there p is held 2^15 times as large and ds by the
// power of two that its column's largest so far allows: what is lost is 2^-39 of the largest.
#include "seq_common.h"

static constexpr int AHEAD = 4;                               // fragments of a group that is read ahead of its products
static constexpr int RG = 64;                                  // tokens a document range covers

struct MaskP {
  const char *q, *k, *v, *o, *res, *d_o;
  char *out, *res_out, *dq, *dk, *dv;
  float *lse, *delta;
  const float* slopes;
  const int *doc_q, *doc_k, *prefix;
  const int4 *rq, *rk;                                         // (smallest id >= 0, largest id, 1 if any is negative, 0) of RG tokens
  long qs[3], ks[3], vs[3], os[3], dos[3], dqs[3], dks[3], dvs[3], dcs[2];
  float* part;                                                 // split key blocks: [nsplit][dv, dk][B][Sk][Hk][D]
  float *qpart, *ml;                                           // split keys: sums [qsplit][B][Sq][H][D], (m, l) [qsplit][B][Sq][H][2]
  int B, Sq, Sk, H, Hk, G, D, causal, off, nsplit, qsplit;
  float scale, softcap;
  Cap cap;
};

__global__ __launch_bounds__(256) void doc_range_kernel(const int* dq, const int* dk, int4* rq, int4* rk, int Sq, int Sk, long qs, long ks) {
  const int nq = (Sq + RG - 1) / RG, nk = (Sk + RG - 1) / RG;
  const int w = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, b = blockIdx.y;
  if (w >= nq + nk) return;
  const bool isq = w < nq;
  const int tile = isq ? w : w - nq, t = tile * RG + lane, n = isq ? Sq : Sk;
  const int id = t < n ? (isq ? dq[b * qs + t] : dk[b * ks + t]) : -1;
  int lo = id >= 0 ? id : 0x7fffffff, hi = id, neg = id < 0 && t < n;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    lo = min(lo, __shfl_xor(lo, d));
    hi = max(hi, __shfl_xor(hi, d));
    neg |= __shfl_xor(neg, d);
  }
  if (lane == 0) (isq ? rq + (long)b * nq : rk + (long)b * nk)[tile] = make_int4(lo, hi, neg, 0);
}

template <class T> __device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, f32x16 c) {
  if constexpr (std::is_same<T, f16>::value) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else if constexpr (std::is_same<T, bf16>::value) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
}

template <class T> __device__ __forceinline__ void pack_tile(const f32x16& p, u32x4 (&pk)[2]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) pk[kb][i] = pack2<T>(p[8 * kb + 2 * i], p[8 * kb + 2 * i + 1]);
  }
}

// A tile of R rows x DP columns in shared memory, in lines of 256 bytes (all 64 banks): a row is one line, a part of one, or (fp32, 128
// columns) two; the 16-byte pieces of a line are xor-swizzled by the line.  The xor is chosen for the two ways a tile is read.  Sixteen
// lanes read one column of pieces of 16 rows: the xor must differ in all of them.  A transposed read takes 4 rows x 64 bytes (fp32: 2
// rows four apart x 128 bytes): its low row bits (bit 2 of the row) must move whole 64-byte (128-byte) groups.  With the plain xor by
// row half of the time in shared memory was bank conflicts.
template <class T, int DP, int R, int NT> struct Tile {           // NT threads stage it
  static constexpr int CE = Elem<T>::CE, NCH = DP / CE, N = (R * NCH + NT - 1) / NT, ROWB = DP * (int)sizeof(T), BYTES = R * ROWB;
  static constexpr bool EVEN = R * NCH % NT == 0;                 // (else some threads have nothing to stage)
  // Byte offset of piece c of a row: its line, and a swizzled place in the line.  `place` is linear over xor in the bits of row and c,
  // so at(row + dr, c + dc) = (at(row, c) ^ place(dr, dc) * 16) + line(dr) * 256 where the bits do not overlap: a lane keeps one offset
  // for each way of reading and a read's own constants cost one xor, not a register each.
  static constexpr __device__ __forceinline__ int place(int row, int c) {
    if constexpr (NCH >= 16) return c ^ (sizeof(T) == 2 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 4) << 1) | ((row & 8) >> 1) | (row & 3));
    else if constexpr (NCH == 8) {
      const int l = row >> 1;
      return ((row & 1) * 8 + c) ^ (sizeof(T) == 2 ? ((l & 1) << 2) | ((l >> 1) & 3) : (l & 7) | ((l & 2) << 2));
    } else return ((row & 3) * 4 + c) ^ ((row >> 2) & 3);
  }
  static constexpr __device__ __forceinline__ int line(int row) { return (row * ROWB) & -(NCH >= 16 ? ROWB : 256); }
  static __device__ __forceinline__ int at(int row, int c) { return line(row) + (place(row, c) << 4); }
  static __device__ __forceinline__ int row_base() { return at(threadIdx.x & 31, (threadIdx.x >> 5) & 1); }
  static __device__ __forceinline__ int col_base() {
    const int lane = threadIdx.x & 63, i = lane & 15;
    if constexpr (sizeof(T) == 2) return at(4 * (lane >> 5) + (i >> 2), ((lane >> 4) & 1) * 2 + ((i & 3) >> 1)) + (i & 1) * 8;
    else return at(4 * (lane >> 5), (lane & 31) >> 2) + (lane & 3) * 4;
  }
  static __device__ __forceinline__ void pack(const f32x16& p, u32x4 (&pk)[2]) { pack_tile<T>(p, pk); }
  struct Regs { u32x4 r[N]; };
  // rows row0 .. of x (element stride rs), zero past nrow rows and D columns
  static __device__ __forceinline__ void load(Regs& g, const T* x, long rs, int row0, int nrow, int D) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int n = threadIdx.x + NT * i, row = row0 + n / NCH, d = (n % NCH) * CE;
      g.r[i] = row < nrow && d < D && (EVEN || n < R * NCH) ? *(const u32x4*)(x + (long)row * rs + d) : u32x4{0, 0, 0, 0};
    }
  }
  static __device__ __forceinline__ bool nonfinite(const Regs& g) {     // whether the wave has an infinity or a NaN
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) bad |= word_nonfinite<T>(g.r[i][w]);
    return __any(bad);
  }
  static __device__ __forceinline__ bool clean(Regs& g) {        // infinities and NaN to zero; whether the wave had any
    if (!nonfinite(g)) return false;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) g.r[i][w] = word_finite<T>(g.r[i][w]);
    return true;
  }
  // finite elements to 0, +inf to 1, -inf to 2^8, NaN to 2^15: sums of up to 64 of each stay apart
  // Written over the tile, one piece at a time: the rare path must not cost the common one registers.
  static __device__ __forceinline__ void encode(char* lds, const T* x, long rs, int row0, int nrow, int D) {
#pragma unroll 1
    for (int n = threadIdx.x; n < R * NCH; n += NT) {
      const int row = row0 + n / NCH, d = (n % NCH) * CE;
      u32x4 v = row < nrow && d < D ? *(const u32x4*)(x + (long)row * rs + d) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (sizeof(T) == 4) v[w] = __float_as_uint(code(__uint_as_float(v[w])));
        else v[w] = pack2<T>(code(half_to_float<T>((u16)v[w])), code(half_to_float<T>((u16)(v[w] >> 16))));
      }
      *(u32x4*)(lds + at(n / NCH, n % NCH)) = v;
    }
  }
  static __device__ __forceinline__ float code(float x) {
    return fabsf(x) < __builtin_inff() ? 0.f : x != x ? 32768.f : x > 0.f ? 1.f : 256.f;
  }
  static __device__ __forceinline__ float decode(float sum) {    // what such a sum adds to a result
    const int n = (int)sum;
    if (n == 0) return 0.f;
    const bool pos = n & 255, neg = n & 0x7f00;
    return n >= 32768 || (pos && neg) ? __builtin_nanf("") : pos ? __builtin_inff() : -__builtin_inff();
  }
  // rows 32 n .. of the tile (whole lines): infinities and NaN to zero in place
  static __device__ __forceinline__ void mend(char* lds, int n) {
    for (int i = threadIdx.x; i < 32 * ROWB / 16; i += NT) {
      u32x4* x = (u32x4*)(lds + n * 32 * ROWB) + i;
      u32x4 v = *x;
#pragma unroll
      for (int w = 0; w < 4; ++w) v[w] = word_finite<T>(v[w]);
      *x = v;
    }
  }
  static __device__ __forceinline__ void store(char* lds, const Regs& g) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int n = threadIdx.x + NT * i;
      if (EVEN || n < R * NCH) *(u32x4*)(lds + at(n / NCH, n % NCH)) = g.r[i];
    }
  }
  // first operand of a product over the columns: lane = row 32 n + (lane & 31), piece 2 c + lane / 32.  o: the tile's offset + row_base()
  // (pinned: a volatile read, which stays where it is written -- see in_groups)
  template <bool PINNED = false> static __device__ __forceinline__ u32x4 rows(const char* lds, int o, int n, int c) {
    typedef __attribute__((address_space(3))) const volatile u32x4 lds_u32x4;
    const char* x = lds + (o ^ (place(0, 2 * c) << 4)) + n * 32 * ROWB;
    if constexpr (PINNED) return *(lds_u32x4*)x;
    else return *(const u32x4*)x;
  }
  // 16-bit: first operand of a product over 16 rows (32 n + 16 kb ..) of the tile, in score-tile order: lane = column 32 db + (lane & 31).
  // o: the tile's offset + col_base()
  static __device__ __forceinline__ u32x4 col16(const char* lds, int o, int n, int db, int kb) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    u32x4 a;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + (o ^ (place(8 * s, 4 * db) << 4)) + line(8 * s) + (32 * n + 16 * kb) * ROWB));
      const u32x2 y = __builtin_bit_cast(u32x2, x);
      a[2 * s] = y[0];
      a[2 * s + 1] = y[1];
    }
    return a;
  }
  // acc[column 32 db + i][lane's own column] += sum over rows 32 n .. of tile[row][column] * p[row], p in score-tile order
  static __device__ __forceinline__ f32x16 cols(const char* lds, int o, int n, int db, const u32x4 (&pk)[2], const f32x16& p, f32x16 acc) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) acc = mfma32<T>(col16(lds, o, n, db, kb), pk[kb], acc);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int dr = mfma32_row(r & 7, 0);
        const float a = *(const float*)(lds + (o ^ (place(dr, 8 * db) << 4)) + line(dr) + (32 * n + 16 * (r >> 3)) * ROWB);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc, 0, 0, 0);
      }
    }
    return acc;
  }
};

// the lane's own row (or none), in 16-byte pieces 2 c + lane / 32
template <class T, int NP> __device__ __forceinline__ void own_row(u32x4 (&f)[NP], const T* x, bool ok, int D) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int c = 0; c < NP; ++c) {
    const int d = (2 * c + h) * Elem<T>::CE;
    f[c] = ok && d < D ? *(const u32x4*)(x + d) : u32x4{0, 0, 0, 0};
  }
}

// Tiles of the other side that this workgroup visits: [first, last), of them those whose document range meets [lo, hi]
template <int PER> struct Tiles {                                // PER tiles a document range
  const int4* r;
  int base, last, lo, hi, step, mine;
  unsigned long long mask;
  // of the tiles those with index = mine_ modulo step_
  __device__ __forceinline__ void init(const int4* ranges, int first, int last_, int lo_, int hi_, int step_ = 1, int mine_ = 0) {
    r = ranges; base = first; last = last_; lo = lo_; hi = hi_; step = step_; mine = mine_;
    if (r && hi < 0) last = first;                               // every id of ours is negative: nothing is seen
    fill();
  }
  __device__ __forceinline__ void fill() {
    const int t = base + (threadIdx.x & 63);
    bool on = t < last && (step == 1 || t % step == mine);
    if (on && r) {
      const int4 x = r[t / PER];
      on = x.y >= 0 && x.y >= lo && x.x <= hi;
    }
    mask = __ballot(on);
  }
  __device__ __forceinline__ int next() {                        // -1: none left
    while (mask == 0) {
      base += 64;
      if (base >= last) return -1;
      fill();
    }
    const int i = __builtin_ctzll(mask);
    mask &= mask - 1;
    return base + i;
  }
};

// four consecutive results of a row
template <class T> __device__ __forceinline__ void store4(T* x, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4) *(f32x4*)x = f32x4{a, b, c, d};
  else *(u32x2*)x = u32x2{pack2<T>(a, b), pack2<T>(c, d)};
}
template <int N> __device__ __forceinline__ bool any_flag(const int* f) {
  int x = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) x |= f[i];
  return __builtin_amdgcn_readfirstlane(x) != 0;
}

struct Head { int b, h, hk; };
// consecutive workgroups walk the (sequence, key head) pairs, so those that read the same keys land on the same of the 8 XCDs
__device__ __forceinline__ Head head_of(int x, const MaskP& p) {
  const int n = p.B * p.Hk, g = x / n, y = x - g * n;
  Head r;
  r.b = y / p.Hk;
  r.hk = y - r.b * p.Hk;
  r.h = r.hk * p.G + g;
  return r;
}

struct Score {
  float mul, slope;
  bool capped;
  Cap cap;
  __device__ __forceinline__ Score(const MaskP& p, int h) : mul(p.cap.lin), slope(p.slopes ? p.slopes[h] * LOG2E : 0.f), capped(p.softcap > 0.f), cap(p.cap) {}
};

// four elements e .. of an output row, and what their rounding left (for the backward pass' do.o) where it is asked for
template <class T> __device__ __forceinline__ void store_out(const MaskP& p, long at, long row, int e, const f32x4& x) {
  store4((T*)p.out + at + e, x[0], x[1], x[2], x[3]);
  if constexpr (sizeof(T) == 2)
    if (p.res_out) {
      auto left = [](float y) { return fabsf(y) < __builtin_inff() ? y - (float)(T)y : 0.f; };       // (inf - inf would be NaN)
      store4((T*)p.res_out + row * p.D + e, left(x[0]), left(x[1]), left(x[2]), left(x[3]));
    }
}

// N fragments read and used in groups of A, each group's reads issued before the products of the group ahead of it (pinned reads: left to
// itself the compiler puts every read right before its use, and a wave waits out the latency of each).  Measured at 2 x 4096 x 16 x 128 plain
// 437 -> 407 us forward, 837 -> 807 dk / dv; the dq kernel, whose registers are full, lost 4 % and does without.
template <int N, int A, class L, class U> __device__ __forceinline__ void in_groups(L&& load, U&& use) {
  u32x4 f[2][A];
#pragma unroll
  for (int i = 0; i < A; ++i) if (i < N) f[0][i] = load(i);
#pragma unroll
  for (int g = 0; g < N; g += A) {
#pragma unroll
    for (int i = 0; i < A; ++i) if (g + A + i < N) f[(g / A + 1) & 1][i] = load(g + A + i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < A; ++i) if (g + i < N) use(g + i, f[(g / A) & 1][i]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// acc[d] += the product over rows 32 n .. of the tile at o, all column blocks
template <class TL, class T, int ND> __device__ __forceinline__ void cols_all(f32x16 (&acc)[ND], const char* lds, int o, int n, const u32x4 (&pk)[2], const f32x16& p) {
  if constexpr (sizeof(T) == 2)
    in_groups<2 * ND, AHEAD>([&](int i) { return TL::col16(lds, o, n, i / 2, i % 2); },
                             [&](int i, const u32x4& a) { acc[i / 2] = mfma32<T>(a, pk[i % 2], acc[i / 2]); });
  else
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = TL::cols(lds, o, n, d, pk, p, acc[d]);
}

// acc += what the encoded tile's rows that `seen` admits add to each column; weighted: by a score gradient, which is 0 or NaN where its own row
// of q or k is not finite (a score of +-inf has weight 0, NaN, or a cap's derivative of 0), so each gives NaN
template <class TL, int R, int ND, class F> __device__ __forceinline__ void add_seen(f32x16 (&acc)[ND], const char* lds, F&& seen, bool weighted) {
  const int half = (threadIdx.x & 63) >> 5, cb = TL::col_base();
#pragma unroll 1
  for (int n = 0; n < R / 32; ++n) {
    f32x16 one;
#pragma unroll
    for (int r = 0; r < 16; ++r) one[r] = seen(n * 32 + mfma32_row(r, half)) ? 1.f : 0.f;
    u32x4 pk[2];
    TL::pack(one, pk);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      __builtin_amdgcn_sched_barrier(0);
      f32x16 z;
#pragma unroll
      for (int r = 0; r < 16; ++r) z[r] = 0.f;
      z = TL::cols(lds, cb, n, d, pk, one, z);
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] += weighted && z[r] != 0.f ? __builtin_nanf("") : TL::decode(z[r]);
    }
  }
}

// ---- forward -------------------------------------------------------------------------------------------------------------------
template <class T, int DP, int KT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (DP == 64 ? 3 : 2) : 1) void attn_masked_fwd_kernel(MaskP p) {
  using TL = Tile<T, DP, KT, 256>;
  constexpr int NP = TL::NCH / 2, ND = DP / 32, NS = KT / 32;
  __shared__ __align__(16) char smem[4 * TL::BYTES + 2 * KT * 4 + 32];      // K, V of two tiles; ids; flags of the waves
  const int rb = TL::row_base(), cb = TL::col_base();
  auto sk = [&](int buf) { return buf * TL::BYTES; };          // offsets of the tiles
  auto sv = [&](int buf) { return (2 + buf) * TL::BYTES; };
  int* const sid = (int*)(smem + 4 * TL::BYTES);                // [2][KT]
  int* const sbad = sid + 2 * KT;                               // [4]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
  const Head hd = head_of(blockIdx.x, p);
  const int q0 = (p.causal ? gridDim.y - 1 - blockIdx.y : blockIdx.y) * 128;      // the long rows of a causal mask first
  const int i = q0 + wave * 32 + (lane & 31);
  const bool iok = i < p.Sq;
  const T* K = (const T*)p.k + hd.b * p.ks[0] + hd.hk * p.ks[2];
  const T* V = (const T*)p.v + hd.b * p.vs[0] + hd.hk * p.vs[2];
  u32x4 qf[NP];
  own_row<T, NP>(qf, (const T*)p.q + hd.b * p.qs[0] + (long)i * p.qs[1] + hd.h * p.qs[2], iok, p.D);
  const Score sc(p, hd.h);
  const int prefix = p.prefix ? max(0, p.prefix[hd.b]) : 0;
  const int myid = p.doc_q ? (iok ? p.doc_q[hd.b * p.dcs[0] + i] : -1) : 0;
  const int qlast = min(q0 + 127, p.Sq - 1);
  const int4 *rk = nullptr;
  int4 qr = make_int4(0, 0, 0, 0);
  if (p.doc_q) {
    const int nq = (p.Sq + RG - 1) / RG;
    const int4* rq = p.rq + (long)hd.b * nq + q0 / RG;
    qr = rq[0];
    if (q0 / RG + 1 < nq) {
      const int4 x = rq[1];
      qr = make_int4(min(qr.x, x.x), max(qr.y, x.y), qr.z | x.z, 0);
    }
    rk = p.rk + (long)hd.b * ((p.Sk + RG - 1) / RG);
  }
  const int tend = p.causal ? min(p.Sk, max(qlast + p.off + 1, prefix)) : p.Sk;
  Tiles<RG / KT> it;
  it.init(rk, 0, (max(tend, 0) + KT - 1) / KT, qr.x, qr.y, p.qsplit, blockIdx.z);

  auto whole = [&](int t) {                                      // every pair of the tile is seen
    const int a = t * KT, z = a + KT - 1;
    if (z >= p.Sk) return false;
    if (p.causal && z > q0 + p.off && z >= prefix) return false;
    if (rk) {
      const int4 x = rk[a / RG];
      if (x.x != x.y || x.z || qr.z || qr.x != qr.y || x.x != qr.x) return false;
    }
    return true;
  };
  // the last key this lane's query sees, documents aside (none: -1)
  const int lim = myid < 0 || !iok ? -1 : p.causal ? min(p.Sk - 1, max(i + p.off, prefix - 1)) : p.Sk - 1;
  auto seen = [&](int t, int id) { return t <= lim && id == myid; };

  typename TL::Regs gk, gv;
  int gid = 0;
  bool dirty = false;
  auto fetch = [&](int t) {
    TL::load(gk, K, p.ks[1], t * KT, p.Sk, p.D);
    TL::load(gv, V, p.vs[1], t * KT, p.Sk, p.D);
    if (p.doc_k && threadIdx.x < KT) gid = t * KT + (int)threadIdx.x < p.Sk ? p.doc_k[hd.b * p.dcs[1] + t * KT + threadIdx.x] : -1;
  };
  auto put = [&](int buf, bool full) {
    if (!full) dirty |= TL::clean(gv);
    TL::store(smem + sk(buf), gk);
    TL::store(smem + sv(buf), gv);
    if (threadIdx.x < KT) sid[buf * KT + threadIdx.x] = gid;
  };

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = NEG_INF, l = 0.f;
  int t = it.next(), buf = 0;
  bool full = t >= 0 && whole(t);
  if (t >= 0) fetch(t);
  __syncthreads();
  if (t >= 0) put(0, full);
  __syncthreads();
  while (t >= 0) {
    const int tn = it.next();
    const bool fulln = tn >= 0 && whole(tn);
    if (tn >= 0) fetch(tn);
    f32x16 s[NS];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
    in_groups<NS * NP, AHEAD>([&](int i) { return TL::template rows<true>(smem, sk(buf) + rb, i / NP, i % NP); },
                              [&](int i, const u32x4& a) { s[i / NP] = mfma32<T>(a, qf[i % NP], s[i / NP]); });
    __builtin_amdgcn_s_setprio(0);
    // in powers of two: s * m0 (plain scores are left as they are, the scale goes into the exponential's argument)
    float m0 = sc.mul;
    if (sc.capped) {
      m0 = 1.f;
      sc.cap.tiles(s);
    }
    if (p.slopes) {
      const float far = (float)(i + p.off - t * KT - 4 * half);
      const int first = q0 + wave * 32 + p.off - t * KT;         // the wave's first query, from the tile's first key
      if (first >= KT - 1 || first <= -31) {                     // every key on one side of every query: two operations a pair, not three
        const float sl = first > 0 ? sc.slope : -sc.slope, c = -sl * far;
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][r] = __builtin_fmaf(s[n][r], m0, __builtin_fmaf(sl, (float)(n * 32 + mfma32_row(r, 0)), c));
      } else {
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][r] = __builtin_fmaf(s[n][r], m0, -sc.slope * fabsf(far - (float)(n * 32 + mfma32_row(r, 0))));
      }
      m0 = 1.f;
    }
    if (!full) {
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int j0 = n * 32 + 8 * r4 + 4 * half;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (j0 + w > lim - t * KT) s[n][4 * r4 + w] = NEG_INF;
          if (p.doc_k) {
            const i32x4 id = *(const i32x4*)(sid + buf * KT + j0);
#pragma unroll
            for (int w = 0; w < 4; ++w)
              if (id[w] != myid) s[n][4 * r4 + w] = NEG_INF;
          }
        }
    }
    float mx = NEG_INF;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32)) * m0;
    const float m2 = fmaxf(m, mx), base = m2 == NEG_INF ? 0.f : m2;
    const float f = exp2_hw(m - base), low = base - LIFT<T>;
    m = m2;
    l *= f;
    if (__any(f != 1.f))
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= f;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[n][r] = exp2_hw(__builtin_fmaf(s[n][r], m0, -low)); l += s[n][r]; }
      u32x4 pk[2];
      pack_tile<T>(s[n], pk);
      __builtin_amdgcn_s_setprio(1);
      cols_all<TL, T>(o, smem, sv(buf) + cb, n, pk, s[n]);
      __builtin_amdgcn_s_setprio(0);
    }
    if (tn >= 0) put(buf ^ 1, fulln);
    __syncthreads();
    buf ^= 1;
    t = tn;
    full = fulln;
  }
  // The seen infinities and NaN that staging left out, if it met any (in a masked tile): once more over the masked tiles
  if (lane == 0) sbad[wave] = dirty;
  __syncthreads();
  if (any_flag<4>(sbad)) {
    it.init(rk, 0, (max(tend, 0) + KT - 1) / KT, qr.x, qr.y, p.qsplit, blockIdx.z);
    for (t = it.next(); t >= 0; t = it.next()) {
      if (whole(t)) continue;
      __syncthreads();
      TL::encode(smem, V, p.vs[1], t * KT, p.Sk, p.D);
      if (threadIdx.x < KT) sid[threadIdx.x] = t * KT + (int)threadIdx.x < p.Sk && p.doc_k ? p.doc_k[hd.b * p.dcs[1] + t * KT + threadIdx.x] : 0;
      __syncthreads();
      add_seen<TL, KT>(o, smem, [&](int j) { return seen(t * KT + j, sid[j]); }, false);
    }
  }
  l += __shfl_xor(l, 32);
  if (!iok) return;
  const long row = ((long)hd.b * p.Sq + i) * p.H + hd.h;
  if (p.qsplit > 1) {
    const long at = blockIdx.z * (long)p.B * p.Sq * p.H + row;
    float* part = p.qpart + at * p.D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int e = d * 32 + mfma32_row(r, half);
        if (e < p.D) *(f32x4*)(part + e) = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
      }
    if (half == 0) { p.ml[2 * at] = m; p.ml[2 * at + 1] = l; }
    return;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const long at = hd.b * p.os[0] + (long)i * p.os[1] + hd.h * p.os[2];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int e = d * 32 + mfma32_row(r, half);
      if (e < p.D) store_out<T>(p, at, row, e, f32x4{o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv});
    }
  if (half == 0) p.lse[((long)hd.b * p.H + hd.h) * p.Sq + i] = l == 0.f ? NEG_INF : m + (log2f(l) - LIFT<T>);
}

// Split keys joined: four elements of a row a thread, the splits in order
template <class T>
__global__ __launch_bounds__(256) void attn_masked_join_kernel(MaskP p) {
  const int nd = p.D / 4;
  const long rows = (long)p.B * p.Sq * p.H, n = (long)blockIdx.x * 256 + threadIdx.x, row = n / nd;
  if (row >= rows) return;
  const int d = (int)(n - row * nd) * 4;
  float m = NEG_INF, l = 0.f;
  for (int s = 0; s < p.qsplit; ++s) m = fmaxf(m, p.ml[2 * (s * rows + row)]);
  const float base = m == NEG_INF ? 0.f : m;
  f32x4 a{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.qsplit; ++s) {
    const long at = s * rows + row;
    const float f = exp2_hw(p.ml[2 * at] - base);
    l += p.ml[2 * at + 1] * f;
    a += *(const f32x4*)(p.qpart + at * p.D + d) * f;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const long bi = row / p.H, h = row - bi * p.H, b = bi / p.Sq, i = bi - b * p.Sq;
  store_out<T>(p, b * p.os[0] + i * p.os[1] + h * p.os[2], row, d, a * inv);
  if (d == 0) p.lse[(b * p.H + h) * p.Sq + i] = l == 0.f ? NEG_INF : m + (log2f(l) - LIFT<T>);
}

// The largest magnitude (NaN aside) of a lane's half of its column of a score tile, and the power of two, at most `up`, by which it comes to lie in
// [2^14, 2^15); an infinity: so low that nothing finite beside it overflows
static constexpr int TOP = 60;
__device__ __forceinline__ float column_max(const f32x16& s) {
  float a = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) a = fmaxf(a, fabsf(s[r]));
  return a;
}
// x = the magnitude times 2^up.  By the whole wave, so that both halves of a column agree (an exchange for every tile would cost more than this
// does where it is rare: in a column's first tiles)
__device__ __forceinline__ int fitting(float x, int up) {
  x = fmaxf(x, __shfl_xor(x, 32));
  if (x <= 32768.f) return up;
  return x < __builtin_inff() ? min(up, up + 15 - __builtin_amdgcn_frexp_expf(x)) : min(up, -TOP);
}

// ---- gradient of the queries -----------------------------------------------------------------------------------------------------
template <class T, int DP, int KT>
__global__ __launch_bounds__(256, (sizeof(T) == 2 ? 2 : 1) + (DP == 32)) void attn_masked_dq_kernel(MaskP p) {
  using TL = Tile<T, DP, KT, 256>;
  constexpr int NP = TL::NCH / 2, ND = DP / 32, NS = KT / 32;
  __shared__ __align__(16) char smem[4 * TL::BYTES + 2 * KT * 4 + 64];
  const int rb = TL::row_base(), cb = TL::col_base();
  auto sk = [&](int buf) { return buf * TL::BYTES; };          // offsets of the tiles
  auto sv = [&](int buf) { return (2 + buf) * TL::BYTES; };
  int* const sid = (int*)(smem + 4 * TL::BYTES);
  int* const sbad = sid + 2 * KT;                               // [4]; of the two tiles [2][4]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
  const Head hd = head_of(blockIdx.x, p);
  const int q0 = (p.causal ? gridDim.y - 1 - blockIdx.y : blockIdx.y) * 128;
  const int i = q0 + wave * 32 + (lane & 31);
  const bool iok = i < p.Sq;
  const T* K = (const T*)p.k + hd.b * p.ks[0] + hd.hk * p.ks[2];
  const T* V = (const T*)p.v + hd.b * p.vs[0] + hd.hk * p.vs[2];
  u32x4 qf[NP], df[NP];
  own_row<T, NP>(qf, (const T*)p.q + hd.b * p.qs[0] + (long)i * p.qs[1] + hd.h * p.qs[2], iok, p.D);
  own_row<T, NP>(df, (const T*)p.d_o + hd.b * p.dos[0] + (long)i * p.dos[1] + hd.h * p.dos[2], iok, p.D);
  const long at = ((long)hd.b * p.H + hd.h) * p.Sq + i;
  float delta = 0.f;
  {
    u32x4 of[NP], rf[NP];                                        // the output and what its rounding left
    own_row<T, NP>(of, (const T*)p.o + hd.b * p.os[0] + (long)i * p.os[1] + hd.h * p.os[2], iok, p.D);
    own_row<T, NP>(rf, (const T*)p.res + (((long)hd.b * p.Sq + i) * p.H + hd.h) * p.D, iok && p.res, p.D);
#pragma unroll
    for (int c = 0; c < NP; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (sizeof(T) == 4) delta += __uint_as_float(of[c][w]) * __uint_as_float(df[c][w]);
        else {                                                   // (their sum first: a remainder of 0 times an infinite do is NaN)
          const unsigned o = of[c][w], x = rf[c][w], y = df[c][w];
          delta += (half_to_float<T>((u16)o) + half_to_float<T>((u16)x)) * half_to_float<T>((u16)y);
          delta += (half_to_float<T>((u16)(o >> 16)) + half_to_float<T>((u16)(x >> 16))) * half_to_float<T>((u16)(y >> 16));
        }
      }
    delta += __shfl_xor(delta, 32);
  }
  float lse = iok ? p.lse[at] : __builtin_inff();
  if (lse == NEG_INF) { lse = __builtin_inff(); delta = 0.f; }   // sees nothing: every probability is zero
  if (iok && half == 0 && blockIdx.z == 0) p.delta[at] = delta;
  const Score sc(p, hd.h);
  const int prefix = p.prefix ? max(0, p.prefix[hd.b]) : 0;
  const int myid = p.doc_q ? (iok ? p.doc_q[hd.b * p.dcs[0] + i] : -1) : 0;
  const int qlast = min(q0 + 127, p.Sq - 1);
  const int4 *rk = nullptr;
  int4 qr = make_int4(0, 0, 0, 0);
  if (p.doc_q) {
    const int nq = (p.Sq + RG - 1) / RG;
    const int4* rq = p.rq + (long)hd.b * nq + q0 / RG;
    qr = rq[0];
    if (q0 / RG + 1 < nq) {
      const int4 x = rq[1];
      qr = make_int4(min(qr.x, x.x), max(qr.y, x.y), qr.z | x.z, 0);
    }
    rk = p.rk + (long)hd.b * ((p.Sk + RG - 1) / RG);
  }
  const int tend = p.causal ? min(p.Sk, max(qlast + p.off + 1, prefix)) : p.Sk;
  Tiles<RG / KT> it;
  it.init(rk, 0, (max(tend, 0) + KT - 1) / KT, qr.x, qr.y, p.qsplit, blockIdx.z);
  auto whole = [&](int t) {
    const int a = t * KT, z = a + KT - 1;
    if (z >= p.Sk) return false;
    if (p.causal && z > q0 + p.off && z >= prefix) return false;
    if (rk) {
      const int4 x = rk[a / RG];
      if (x.x != x.y || x.z || qr.z || qr.x != qr.y || x.x != qr.x) return false;
    }
    return true;
  };
  // the last key this lane's query sees, documents aside (none: -1)
  const int lim = myid < 0 || !iok ? -1 : p.causal ? min(p.Sk - 1, max(i + p.off, prefix - 1)) : p.Sk - 1;
  auto seen = [&](int t, int id) { return t <= lim && id == myid; };
  typename TL::Regs gk, gv;
  int gid = 0;
  bool dirty = false;
  auto fetch = [&](int t) {
    TL::load(gk, K, p.ks[1], t * KT, p.Sk, p.D);
    TL::load(gv, V, p.vs[1], t * KT, p.Sk, p.D);
    if (p.doc_k && threadIdx.x < KT) gid = t * KT + (int)threadIdx.x < p.Sk ? p.doc_k[hd.b * p.dcs[1] + t * KT + threadIdx.x] : -1;
  };
  auto put = [&](int buf, bool full) {
    if (!full) {
      const bool bad = TL::nonfinite(gk);
      dirty |= bad;
      if (lane == 0) sbad[4 + 4 * buf + wave] = bad;
    }
    TL::store(smem + sk(buf), gk);
    TL::store(smem + sv(buf), gv);
    if (threadIdx.x < KT) sid[buf * KT + threadIdx.x] = gid;
  };
  // fp16: score gradients are small multiples of 1 / Sk of dout's and would be subnormal or lost; each query's are held 2^up times as large,
  // up such that its largest so far lies below 2^15 (lowered, with the sums, when a larger one comes; part of the exponent otherwise).  With
  // dout of 1e-3 at 4096 keys dq was off by 5e-3 of itself, eight times its own rounding.  2 x 4096 x 16 x 64: 254 -> 300 us, dk 507 -> 550.
  constexpr bool LIFTED = std::is_same<T, f16>::value;
  int up = LIFTED ? TOP : 0;
  if constexpr (LIFTED) lse -= (float)up;
  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
  int t = it.next(), buf = 0;
  bool full = t >= 0 && whole(t);
  if (t >= 0) fetch(t);
  __syncthreads();
  if (t >= 0) put(0, full);
  __syncthreads();
  while (t >= 0) {
    const int tn = it.next();
    const bool fulln = tn >= 0 && whole(tn);
    if (tn >= 0) fetch(tn);
    const bool holes = !full && any_flag<4>(sbad + 4 + 4 * buf);   // scores from the tile as it is, the product without its infinities
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      f32x16 st[1], dp;
      f32x16& s = st[0];
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int c = 0; c < NP; ++c) s = mfma32<T>(TL::rows(smem, sk(buf) + rb, n, c), qf[c], s);
#pragma unroll
      for (int c = 0; c < NP; ++c) dp = mfma32<T>(TL::rows(smem, sv(buf) + rb, n, c), df[c], dp);
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] -= delta;
      float m0 = sc.mul;
      if (sc.capped) {
        m0 = 1.f;
        sc.cap.tile(st, [&](int r, float d) { dp[r] *= d; });
      }
      if (p.slopes) {
        const float far = (float)(i + p.off - t * KT - n * 32 - 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], m0, -sc.slope * fabsf(far - (float)mfma32_row(r, 0)));
        m0 = 1.f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = exp2_hw(__builtin_fmaf(s[r], m0, -lse)) * dp[r];
      if (!full) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int j0 = n * 32 + 8 * r4 + 4 * half;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (j0 + w > lim - t * KT) s[4 * r4 + w] = 0.f;
          if (p.doc_k) {
            const i32x4 id = *(const i32x4*)(sid + buf * KT + j0);
#pragma unroll
            for (int w = 0; w < 4; ++w)
              if (id[w] != myid) s[4 * r4 + w] = 0.f;
          }
        }
      }
      if constexpr (LIFTED) {
        const float mx = column_max(s);
        if (__any(mx > 32768.f)) {
          const int drop = up - fitting(mx, up);
          const float f = __builtin_amdgcn_ldexpf(1.f, -drop);
          up -= drop;
          lse += (float)drop;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] *= f;
#pragma unroll
          for (int d = 0; d < ND; ++d) dq[d] *= f;
        }
      }
      if (holes) {                                               // (the whole workgroup; S is formed, K is next read for its columns)
        __syncthreads();
        TL::mend(smem + sk(buf), n);
        __syncthreads();
      }
      u32x4 pk[2];
      pack_tile<T>(s, pk);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int d = 0; d < ND; ++d) dq[d] = TL::cols(smem, sk(buf) + cb, n, d, pk, s, dq[d]);
      __builtin_amdgcn_s_setprio(0);
    }
    if (tn >= 0) put(buf ^ 1, fulln);
    __syncthreads();
    buf ^= 1;
    t = tn;
    full = fulln;
  }
  // The seen infinities and NaN that the product left out, if it met any (in a masked tile): once more over the masked tiles
  if (lane == 0) sbad[wave] = dirty;
  __syncthreads();
  if (any_flag<4>(sbad)) {
    it.init(rk, 0, (max(tend, 0) + KT - 1) / KT, qr.x, qr.y, p.qsplit, blockIdx.z);
    for (t = it.next(); t >= 0; t = it.next()) {
      if (whole(t)) continue;
      __syncthreads();
      TL::encode(smem, K, p.ks[1], t * KT, p.Sk, p.D);
      if (threadIdx.x < KT) sid[threadIdx.x] = t * KT + (int)threadIdx.x < p.Sk && p.doc_k ? p.doc_k[hd.b * p.dcs[1] + t * KT + threadIdx.x] : 0;
      __syncthreads();
      add_seen<TL, KT>(dq, smem, [&](int j) { return seen(t * KT + j, sid[j]); }, true);
    }
  }
  if (!iok) return;
  T* out = (T*)p.dq + hd.b * p.dqs[0] + (long)i * p.dqs[1] + hd.h * p.dqs[2];
  float* part = p.qpart + (((long)blockIdx.z * p.B + hd.b) * p.Sq + i) * p.H * p.D + (long)hd.h * p.D;
  const float mul = __builtin_amdgcn_ldexpf(p.qsplit == 1 ? p.scale : 1.f, -up);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int e = d * 32 + mfma32_row(r, half);
      if (e >= p.D) continue;
      const f32x4 x{dq[d][r] * mul, dq[d][r + 1] * mul, dq[d][r + 2] * mul, dq[d][r + 3] * mul};
      if (p.qsplit == 1) store4(out + e, x[0], x[1], x[2], x[3]);
      else *(f32x4*)(part + e) = x;
    }
}

// ---- gradients of the keys and values ----------------------------------------------------------------------------------------------
// Eight waves own 128 keys (four own 64 where a wave of 128 fp32 columns needs all registers), two waves the same 32.  The first half of the
// waves forms S, the probabilities and dv; the second half do.v, the score gradients and dk.  A wave then needs 64 accumulators (D = 128)
// instead of 128 and two waves fit a SIMD, one's exponentials under the other's matrix work.  The probabilities (times the cap's derivative)
// go through shared memory in 32 bits, lane to lane, and the second wave uses them one tile later, so the tile's one barrier suffices: the
// tile of Q is kept a turn longer (three buffers).  One wave with both sums took 978 us for 2 x 4096 tokens and 16 heads of 128, two waves
// that both formed S 984, this 837 and 807 with the shared-memory reads a group ahead.  Where the key blocks are few, `nsplit` workgroups share the query tiles of one (every
// nsplit-th tile, so the split is even under a causal mask too); their 32-bit sums are added in order by sum_join_kernel.
template <class T, int DP, int QT, int NT>
__global__ __launch_bounds__(NT, NT / 256) void attn_masked_dkv_kernel(MaskP p) {
  using TL = Tile<T, DP, QT, NT>;
  constexpr int NW = NT / 128, KEYS = 32 * NW;                  // waves of either kind; keys of the workgroup
  constexpr int NP = TL::NCH / 2, ND = DP / 32, NS = QT / 32;
  constexpr int XB = NW * NS * 4096;                            // probabilities of a tile: [pair][half tile][4][lane][4] floats
  __shared__ __align__(16) char smem[5 * TL::BYTES + 2 * XB + 6 * QT * 4 + 128];   // dO of two tiles, Q of three; probabilities; lse, delta, ids; flags
  const int rb = TL::row_base(), cb = TL::col_base();
  auto sd = [&](int buf) { return buf * TL::BYTES; };          // offsets of the tiles
  auto sq = [&](int q3) { return (2 + q3) * TL::BYTES; };
  float* const slse = (float*)(smem + 5 * TL::BYTES + 2 * XB);  // [2][QT]
  float* const sdel = slse + 2 * QT;
  int* const sid = (int*)(sdel + 2 * QT);
  int* const sbad = sid + 2 * QT;                               // [8]; of the three tiles [3][8]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
  const bool keys = wave >= NW;                                 // this wave forms dk, else dv
  const int b = blockIdx.x / p.Hk, hk = blockIdx.x - b * p.Hk, split = blockIdx.z;
  const int k0 = blockIdx.y * KEYS;                               // (causal: the first keys are seen by most queries)
  const int t = k0 + (wave & (NW - 1)) * 32 + (lane & 31);
  const bool tok = t < p.Sk;
  u32x4 wf[NP];                                                 // the key's row of K, or (dk) of V
  {
    const long* st = keys ? p.vs : p.ks;
    own_row<T, NP>(wf, (const T*)(keys ? p.v : p.k) + b * st[0] + (long)t * st[1] + hk * st[2], tok, p.D);
  }
  auto exchange = [&](int buf, int n) { return (f32x4*)(smem + 5 * TL::BYTES + buf * XB + ((wave & (NW - 1)) * NS + n) * 4096) + lane; };
  const int prefix = p.prefix ? max(0, p.prefix[b]) : 0;
  const int myid = p.doc_k ? (tok ? p.doc_k[b * p.dcs[1] + t] : -1) : 0;
  const int klast = min(k0 + KEYS - 1, p.Sk - 1);
  const int4 *rq = nullptr;
  int4 kr = make_int4(0, 0, 0, 0);
  if (p.doc_q) {
    const int nk = (p.Sk + RG - 1) / RG;
    const int4* rk = p.rk + (long)b * nk + k0 / RG;
    kr = rk[0];
    if (KEYS > RG && k0 / RG + 1 < nk) {
      const int4 x = rk[1];
      kr = make_int4(min(kr.x, x.x), max(kr.y, x.y), kr.z | x.z, 0);
    }
    rq = p.rq + (long)b * ((p.Sq + RG - 1) / RG);
  }
  const int first = p.causal && k0 >= prefix ? max(0, k0 - p.off) / QT : 0;
  auto whole = [&](int tq) {                                     // every pair of the tile is seen (a row past Sq is not: 0 of its own meets the keys' infinities)
    const int a = tq * QT;
    if (a + QT > p.Sq) return false;
    if (p.causal && klast > a + p.off && klast >= prefix) return false;
    if (rq) {
      const int4 x = rq[a / RG];
      if (x.x != x.y || x.z || kr.z || kr.x != kr.y || x.x != kr.x) return false;
    }
    return true;
  };
  // the first query that sees this lane's key, documents aside
  const int lim = myid < 0 || !tok ? 0x7fffffff : p.causal && t >= prefix ? t - p.off : 0;
  auto seen = [&](int i, int id) { return i >= lim && i < p.Sq && id == myid; };
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  typename TL::Regs gq, gd;
  float glse = 0.f, gdel = 0.f;
  int gid = 0;
  bool dirty = false;
  const Score sc(p, hk * p.G);                                   // (its slope is the first head's: taken per tile below)
  // the tiles of all query heads that share the key head, one after the other
  Tiles<RG / QT> it;
  int g = 0;
  auto start = [&]() { it.init(rq, first, (p.Sq + QT - 1) / QT, kr.x, kr.y, p.nsplit, split); };
  auto next = [&]() {
    int x = it.next();
    while (x < 0 && ++g < p.G) {
      start();
      x = it.next();
    }
    return x;
  };
  auto fetch = [&](int tq, int g) {
    const int h = hk * p.G + g;
    TL::load(gq, (const T*)p.q + b * p.qs[0] + h * p.qs[2], p.qs[1], tq * QT, p.Sq, p.D);
    TL::load(gd, (const T*)p.d_o + b * p.dos[0] + h * p.dos[2], p.dos[1], tq * QT, p.Sq, p.D);
    if (threadIdx.x < QT) {
      const int i = tq * QT + threadIdx.x;
      const long at = ((long)b * p.H + h) * p.Sq + i;
      glse = i < p.Sq ? p.lse[at] : __builtin_inff();
      if (glse == NEG_INF) glse = __builtin_inff();              // sees nothing: every probability is zero
      glse -= LIFT<T>;
      gdel = i < p.Sq ? p.delta[at] : 0.f;
      gid = i < p.Sq ? (p.doc_q ? p.doc_q[b * p.dcs[0] + i] : 0) : -1;
    }
  };
  auto put = [&](int buf, int q3, bool full) {
    if (!full) {
      const bool badq = TL::nonfinite(gq), badd = TL::nonfinite(gd);
      dirty |= badq || badd;
      if (lane == 0) sbad[8 + 8 * q3 + wave] = badq || badd;
    }
    TL::store(smem + sq(q3), gq);
    TL::store(smem + sd(buf), gd);
    if (threadIdx.x < QT) {
      slse[buf * QT + threadIdx.x] = glse;
      sdel[buf * QT + threadIdx.x] = gdel;
      sid[buf * QT + threadIdx.x] = gid;
    }
  };
  start();
  int tq = next(), gcur = g, buf = 0, q3 = 0, qprev = 2;
  bool full = tq >= 0 && whole(tq);
  if (tq >= 0) {
    fetch(tq, gcur);
    put(0, 0, full);
  }
  for (int i = threadIdx.x; i < TL::BYTES / 16; i += NT) ((u32x4*)(smem + sq(2)))[i] = u32x4{0, 0, 0, 0};
  __syncthreads();
  constexpr bool LIFTED = std::is_same<T, f16>::value;
  int up = LIFTED && keys ? TOP : 0;                            // fp16: dk's score gradients are held 2^up times as large
  auto walk = [&](auto role) {                                 // (a loop of its own for either kind of wave: same tiles, same barriers)
    f32x16 dp[NS];                                               // dk's waves: do.v - D of the tile, until its probabilities are there
    auto finish = [&]() {                                        // dk of the tile before: its probabilities, its rows of Q
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const f32x4* x = exchange(buf ^ 1, n);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 pr = x[64 * r4];
#pragma unroll
          for (int w = 0; w < 4; ++w)                            // (-0: a masked pair, whose do.v may be anything)
            dp[n][4 * r4 + w] = __float_as_uint(pr[w]) == 0x80000000u ? 0.f : pr[w] * dp[n][4 * r4 + w];
        }
        if constexpr (LIFTED) {                                  // as in the queries' kernel, a key's column here
          const float mx = column_max(dp[n]), top = __builtin_amdgcn_ldexpf(mx, up);
          if (__any(top > 32768.f)) {
            const int to = fitting(top, up);
            const float f = __builtin_amdgcn_ldexpf(1.f, to - up);
            up = to;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] *= f;
          }
          const float f = __builtin_amdgcn_ldexpf(1.f, up);
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[n][r] *= f;
        }
        u32x4 pk[2];
        pack_tile<T>(dp[n], pk);
        __builtin_amdgcn_s_setprio(1);
        cols_all<TL, T>(acc, smem, sq(qprev) + cb, n, pk, dp[n]);
        __builtin_amdgcn_s_setprio(0);
      }
    };
    auto mend = [&](int n) {                                     // both kinds of wave: S and do.v of these rows are formed, next come their columns
      __syncthreads();
      TL::mend(smem + sq(q3), n);
      TL::mend(smem + sd(buf), n);
      __syncthreads();
    };
    if constexpr (decltype(role)::value) {                     // nothing before the first tile: probabilities of zero, rows of zero
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          exchange(1, n)[64 * r4] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < 4; ++w) dp[n][4 * r4 + w] = 0.f;
        }
    }
    for (;;) {
      if constexpr (decltype(role)::value)
        finish();
      if (tq < 0) break;
      const int tn = next(), gn = g;
      const bool fulln = tn >= 0 && whole(tn);
      if (tn >= 0) fetch(tn, gn);
      const bool holes = !full && any_flag<NT / 64>(sbad + 8 + 8 * q3);   // scores from the tiles as they are, the products without their infinities
      if constexpr (decltype(role)::value) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[n][r] = 0.f;
          __builtin_amdgcn_s_setprio(1);
          in_groups<NP, AHEAD>([&](int i) { return TL::template rows<true>(smem, sd(buf) + rb, n, i); }, [&](int i, const u32x4& a) { dp[n] = mfma32<T>(a, wf[i], dp[n]); });
          __builtin_amdgcn_s_setprio(0);
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const f32x4 de = *(const f32x4*)(sdel + buf * QT + n * 32 + 8 * r4 + 4 * half);
#pragma unroll
            for (int w = 0; w < 4; ++w) dp[n][4 * r4 + w] -= de[w];
          }
          if (holes) mend(n);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          f32x16 st[1], dcap;
          f32x16& s = st[0];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = 0.f;
          __builtin_amdgcn_s_setprio(1);
          in_groups<NP, AHEAD>([&](int i) { return TL::template rows<true>(smem, sq(q3) + rb, n, i); }, [&](int i, const u32x4& a) { s = mfma32<T>(a, wf[i], s); });
          __builtin_amdgcn_s_setprio(0);
          float m0 = sc.mul;
          if (sc.capped) {
            m0 = 1.f;
            sc.cap.tile(st, [&](int r, float d) { dcap[r] = d; });
          }
          if (p.slopes) {
            const float slope = p.slopes[hk * p.G + gcur] * LOG2E, far = (float)(tq * QT + n * 32 + 4 * half + p.off - t);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], m0, -slope * fabsf(far + (float)mfma32_row(r, 0)));
            m0 = 1.f;
          }
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const f32x4 ls = *(const f32x4*)(slse + buf * QT + n * 32 + 8 * r4 + 4 * half);
#pragma unroll
            for (int w = 0; w < 4; ++w) s[4 * r4 + w] = exp2_hw(__builtin_fmaf(s[4 * r4 + w], m0, -ls[w]));
          }
          if (!full) {
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
              const int j0 = n * 32 + 8 * r4 + 4 * half;
              const i32x4 id = *(const i32x4*)(sid + buf * QT + j0);
#pragma unroll
              for (int w = 0; w < 4; ++w)
                if (j0 + w < lim - tq * QT || id[w] != myid) { s[4 * r4 + w] = -0.f; dcap[4 * r4 + w] = 1.f; }   // (either may be NaN there)
            }
          }
          f32x4* x = exchange(buf, n);
          if (sc.capped)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
              x[64 * r4] = f32x4{s[4 * r4] * dcap[4 * r4], s[4 * r4 + 1] * dcap[4 * r4 + 1], s[4 * r4 + 2] * dcap[4 * r4 + 2], s[4 * r4 + 3] * dcap[4 * r4 + 3]};
          else
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) x[64 * r4] = f32x4{s[4 * r4], s[4 * r4 + 1], s[4 * r4 + 2], s[4 * r4 + 3]};
          u32x4 pk[2];
          pack_tile<T>(s, pk);
          if (holes) mend(n);
          __builtin_amdgcn_s_setprio(1);
          cols_all<TL, T>(acc, smem, sd(buf) + cb, n, pk, s);
          __builtin_amdgcn_s_setprio(0);
        }
      }
      const int qn = q3 == 2 ? 0 : q3 + 1;
      if (tn >= 0) put(buf ^ 1, qn, fulln);
      __syncthreads();
      buf ^= 1;
      qprev = q3;
      q3 = qn;
      tq = tn;
      gcur = gn;
      full = fulln;
    }
  };
  if (tq >= 0) {
    if (keys) walk(std::true_type{});
    else walk(std::false_type{});
  }
  if (lane == 0) sbad[wave] = dirty;
  __syncthreads();
  if (any_flag<NT / 64>(sbad)) {                                      // as in the forward kernel, over both sides' rows
    for (int g = 0; g < p.G; ++g) {
      const int h = hk * p.G + g;
      start();
      for (int tq = it.next(); tq >= 0; tq = it.next()) {
        if (whole(tq)) continue;
        __syncthreads();
        TL::encode(smem + sq(0), (const T*)p.q + b * p.qs[0] + h * p.qs[2], p.qs[1], tq * QT, p.Sq, p.D);
        TL::encode(smem + sd(0), (const T*)p.d_o + b * p.dos[0] + h * p.dos[2], p.dos[1], tq * QT, p.Sq, p.D);
        if (threadIdx.x < QT) sid[threadIdx.x] = tq * QT + (int)threadIdx.x < p.Sq && p.doc_q ? p.doc_q[b * p.dcs[0] + tq * QT + threadIdx.x] : 0;
        __syncthreads();
        add_seen<TL, QT>(acc, smem + (keys ? sq(0) : sd(0)), [&](int j) { return seen(tq * QT + j, sid[j]); }, keys);
      }
    }
  }
  if (!tok) return;
  const float mul = __builtin_amdgcn_ldexpf(keys && p.nsplit == 1 ? p.scale : 1.f, -up) * LOWER<T>;
  const long* st = keys ? p.dks : p.dvs;
  T* out = (T*)(keys ? p.dk : p.dv) + b * st[0] + (long)t * st[1] + hk * st[2];
  float* part = p.part + ((((long)split * 2 + keys) * p.B + b) * p.Sk + t) * p.Hk * p.D + (long)hk * p.D;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int e = d * 32 + mfma32_row(r, half);
      if (e >= p.D) continue;
      const f32x4 x{acc[d][r] * mul, acc[d][r + 1] * mul, acc[d][r + 2] * mul, acc[d][r + 3] * mul};
      if (p.nsplit == 1) store4(out + e, x[0], x[1], x[2], x[3]);
      else *(f32x4*)(part + e) = x;
    }
}

// out[b, t, h] = mul times the sum of the splits [n][B][S][H][D], in order; four elements a thread
struct SumP { const float* part; char* out; long st[3], next; int n, S, H, D; float mul; };
template <class T>
__global__ __launch_bounds__(256) void sum_join_kernel(SumP p, long total) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= total) return;
  f32x4 a = *(const f32x4*)(p.part + i);
  for (int s = 1; s < p.n; ++s) a += *(const f32x4*)(p.part + s * p.next + i);
  const int d = (int)(i % p.D);
  const long row = i / p.D, h = row % p.H, bt = row / p.H, t = bt % p.S, b = bt / p.S;
  store4((T*)p.out + b * p.st[0] + t * p.st[1] + h * p.st[2] + d, a[0] * p.mul, a[1] * p.mul, a[2] * p.mul, a[3] * p.mul);
}
template <class T>
static void sum_join(const float* part, char* out, const long* st, long next, int n, int B, int S, int H, int D, float mul, hipStream_t stream) {
  const long total = (long)B * S * H * D;
  hipLaunchKernelGGL(sum_join_kernel<T>, dim3(cdiv(total, 1024)), dim3(256), 0, stream, SumP{part, out, {st[0], st[1], st[2]}, next, n, S, H, D, mul}, total);
}

// ---- C entries -----------------------------------------------------------------------------------------------------------------------
static int mask_args(int dtype, int B, int Sq, int Sk, int H, int Hk, int D, float scale, float softcap, const int* doc_q, const int* doc_k, const void* ranges,
                     const long* strides) {
  const int es = dtype_size(dtype);
  if (!es || B < 0 || Sq < 0 || Sk < 0 || Hk < 1 || H < Hk || H % Hk || D < 1 || !strides || !(softcap >= 0.f && softcap < __builtin_inff()) || !(scale > 0.f && scale < __builtin_inff())) return AOT_ERR_BADARG;   // (a running maximum of unscaled scores needs a positive scale)
  if ((doc_q == nullptr) != (doc_k == nullptr) || (doc_q && !ranges)) return AOT_ERR_BADARG;
  if (D > 128 || D * es % 16 || Sq > (1 << 22) || Sk > (1 << 22) || (long)B * H * 512 > 0xffffffffL || B > 65535) return AOT_ERR_UNSUPPORTED;
  return AOT_OK;
}
static bool rows_aligned(const void* x, const long* st, int es) {
  for (int i = 0; i < 3; ++i) if (st[i] * es % 16) return false;
  return aligned16(x);
}
static void mask_common(MaskP& p, int B, int Sq, int Sk, int H, int Hk, int D, int causal, float scale, float softcap, const float* slopes,
                        const int* doc_q, const int* doc_k, const int* prefix, void* ranges) {
  p.B = B; p.Sq = Sq; p.Sk = Sk; p.H = H; p.Hk = Hk; p.G = H / Hk; p.D = D; p.causal = causal != 0; p.off = Sk - Sq;
  p.scale = scale; p.softcap = softcap; p.cap = Cap::of(scale, softcap); p.slopes = slopes; p.doc_q = doc_q; p.doc_k = doc_k; p.prefix = causal ? prefix : nullptr;
  p.rq = (const int4*)ranges;
  p.rk = p.rq + (long)B * ((Sq + RG - 1) / RG);
}
static void range_launch(const MaskP& p, hipStream_t st) {
  const int n = (p.Sq + RG - 1) / RG + (p.Sk + RG - 1) / RG;
  hipLaunchKernelGGL(doc_range_kernel, dim3((n + 3) / 4, p.B), dim3(256), 0, st, p.doc_q, p.doc_k, (int4*)p.rq, (int4*)p.rk, p.Sq, p.Sk, p.dcs[0], p.dcs[1]);
}
// f(element type, padded head width, rows of a shared-memory tile): 64 rows a tile where four of them fit 64 KB, else 32
template <class F> static void with_tile(int dtype, int D, F&& f) {
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (D <= 32) f(t, std::integral_constant<int, 32>{}, std::integral_constant<int, 64>{});
    else if (D <= 64) f(t, std::integral_constant<int, 64>{}, std::integral_constant<int, 64>{});
    else f(t, std::integral_constant<int, 128>{}, std::integral_constant<int, sizeof(T) == 4 ? 32 : 64>{});
  });
}

// Where the blocks of 128 queries (or of keys) are too few for the chip's 256 CUs twice over, several workgroups share the tiles of one
// block, every n-th tile each (even under a causal mask), a power of two of them (split keys: with at least four tiles each).  Their 32-bit sums go
// through a workspace: 8 bytes an element and split more.  Forward / backward, us, where the aim is no split, 256, 512 (taken) and 1024 workgroups,
// causal: 16 queries on 8192 keys, 8 heads of 128 225 / 340, 31 / 65, 31 / 65, 31 / 65; 2047 on 8191, 16 / 8 of 64 174 / 540, 174 / 540, 133 / 468,
// 127 / 487; 1024 on 4096, 16 of 128 124 / 270, 76 / 206, 65 / 191, 75 / 225; 2048, 16 of 128 66 / 177, 66 / 178, 63 / 148, 62 / 176; fp32 2 x 900, 8 of
// 32 46 / 143, 32 / 90, 33 / 90, 33 / 96.
static int mask_split(long blocks, int tiles) {
  int n = 1;
  while (n < 16 && blocks * n < 512 && 8 * n <= tiles) n *= 2;
  return n;
}
static int q_split(int B, int Sq, int Sk, int H) { return mask_split((long)B * H * ((Sq + 127) / 128), (Sk + 63) / 64); }
static int k_split(int B, int Sq, int Sk, int Hk) { return mask_split((long)B * Hk * ((Sk + 127) / 128), (Sq + 63) / 64 * 4); }
// Floats of scratch: forward (sums, then (m, l), of split keys); backward (delta, sums of split keys, sums of split queries)
static long fwd_floats(int B, int Sq, int Sk, int H, int D) {
  const int n = q_split(B, Sq, Sk, H);
  return n > 1 ? (long)n * B * Sq * H * (D + 2) : 0;
}
struct BwdWork { long qpart, part, all; };
static BwdWork bwd_floats(int B, int Sq, int Sk, int H, int Hk, int D) {
  const int n = q_split(B, Sq, Sk, H), m = k_split(B, Sq, Sk, Hk);
  BwdWork w;
  w.qpart = ((long)B * H * Sq + 3) / 4 * 4;
  w.part = w.qpart + (n > 1 ? (long)n * B * Sq * H * D : 0);
  w.all = w.part + (m > 1 ? 2L * m * B * Sk * Hk * D : 0);
  return w;
}
extern "C" int aot_attn_masked_floats(int B, int Sq, int Sk, int H, int Hk, int D, int backward, long* floats) {
  if (!floats || B < 0 || Sq < 0 || Sk < 0 || Hk < 1 || H < Hk || H % Hk || D < 1) return AOT_ERR_BADARG;
  *floats = backward ? bwd_floats(B, Sq, Sk, H, Hk, D).all : fwd_floats(B, Sq, Sk, H, D);
  return AOT_OK;
}

extern "C" int aot_attn_masked(const void* q, const void* k, const void* v, void* out, void* residual, float* lse, const float* slopes,
                               const int* doc_q, const int* doc_k, const int* prefix, void* ranges, float* work, long work_floats, int dtype, int B, int Sq, int Sk, int H, int Hk, int D,
                               int causal, float scale, float softcap, const long* strides, void* stream) {
  int rc = mask_args(dtype, B, Sq, Sk, H, Hk, D, scale, softcap, doc_q, doc_k, ranges, strides);
  if (rc) return rc;
  if (B == 0 || Sq == 0) return AOT_OK;
  if (!q || !out || !lse || (Sk && (!k || !v))) return AOT_ERR_BADARG;
  MaskP p{};
  p.q = (const char*)q; p.k = (const char*)k; p.v = (const char*)v; p.out = (char*)out; p.res_out = (char*)residual; p.lse = lse;
  for (int i = 0; i < 3; ++i) { p.qs[i] = strides[i]; p.ks[i] = strides[3 + i]; p.vs[i] = strides[6 + i]; p.os[i] = strides[9 + i]; }
  p.dcs[0] = strides[12]; p.dcs[1] = strides[13];
  const int es = dtype_size(dtype);
  if (!rows_aligned(q, p.qs, es) || !rows_aligned(k, p.ks, es) || !rows_aligned(v, p.vs, es) || !rows_aligned(out, p.os, es)) return AOT_ERR_BADARG;
  mask_common(p, B, Sq, Sk, H, Hk, D, causal, scale, softcap, slopes, doc_q, doc_k, prefix, ranges);
  const long need = fwd_floats(B, Sq, Sk, H, D);
  if (!aligned16(residual) || (need && (!work || !aligned16(work) || work_floats < need))) return AOT_ERR_BADARG;
  p.qsplit = q_split(B, Sq, Sk, H);
  p.qpart = work;
  p.ml = work + (long)p.qsplit * B * Sq * H * D;
  hipStream_t st = (hipStream_t)stream;
  if (doc_q) range_launch(p, st);
  const dim3 grid(B * H, cdiv(Sq, 128), p.qsplit);
  with_tile(dtype, D, [&](auto t, auto dp, auto kt) {
    hipLaunchKernelGGL((attn_masked_fwd_kernel<decltype(t), decltype(dp)::value, decltype(kt)::value>), grid, dim3(256), 0, st, p);
    if (p.qsplit > 1) hipLaunchKernelGGL(attn_masked_join_kernel<decltype(t)>, dim3(cdiv((long)B * Sq * H * (D / 4), 256)), dim3(256), 0, st, p);
  });
  AOT_LAUNCH_CHECK();
}

extern "C" int aot_attn_masked_bwd(const void* q, const void* k, const void* v, const void* out, const void* residual, const float* lse,
                                   const void* dout, void* dq, void* dk, void* dv, const float* slopes, const int* doc_q, const int* doc_k, const int* prefix, void* ranges, float* work, long work_floats,
                                   int dtype, int B, int Sq, int Sk, int H, int Hk, int D, int causal, float scale, float softcap, const long* strides,
                                   void* stream) {
  int rc = mask_args(dtype, B, Sq, Sk, H, Hk, D, scale, softcap, doc_q, doc_k, ranges, strides);
  if (rc) return rc;
  if (B == 0 || (Sq == 0 && Sk == 0)) return AOT_OK;
  if ((Sq && (!q || !out || !lse || !dout || !dq)) || (Sk && (!k || !v || !dk || !dv))) return AOT_ERR_BADARG;
  MaskP p{};
  p.q = (const char*)q; p.k = (const char*)k; p.v = (const char*)v; p.o = (const char*)out; p.res = (const char*)residual; p.d_o = (const char*)dout;
  p.lse = (float*)lse; p.dq = (char*)dq; p.dk = (char*)dk; p.dv = (char*)dv;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = strides[i]; p.ks[i] = strides[3 + i]; p.vs[i] = strides[6 + i]; p.os[i] = strides[9 + i]; p.dos[i] = strides[12 + i];
    p.dqs[i] = strides[15 + i]; p.dks[i] = strides[18 + i]; p.dvs[i] = strides[21 + i];
  }
  p.dcs[0] = strides[24]; p.dcs[1] = strides[25];
  const int es = dtype_size(dtype);
  if (!rows_aligned(q, p.qs, es) || !rows_aligned(k, p.ks, es) || !rows_aligned(v, p.vs, es) || !rows_aligned(out, p.os, es) ||
      !rows_aligned(dout, p.dos, es) || !rows_aligned(dq, p.dqs, es) || !rows_aligned(dk, p.dks, es) || !rows_aligned(dv, p.dvs, es) ||
      !aligned16(work)) return AOT_ERR_BADARG;
  const BwdWork w = bwd_floats(B, Sq, Sk, H, Hk, D);
  if (!aligned16(residual) || (w.all && (!work || work_floats < w.all))) return AOT_ERR_BADARG;
  p.delta = work;
  p.qpart = work + w.qpart;
  p.part = work + w.part;
  p.qsplit = q_split(B, Sq, Sk, H);
  p.nsplit = k_split(B, Sq, Sk, Hk);
  mask_common(p, B, Sq, Sk, H, Hk, D, causal, scale, softcap, slopes, doc_q, doc_k, prefix, ranges);
  hipStream_t st = (hipStream_t)stream;
  if (doc_q) range_launch(p, st);
  with_tile(dtype, D, [&](auto t, auto dp, auto kt) {
    constexpr int KT = decltype(dp)::value == 128 ? 32 : 64;     // (two 64-row tiles of 128 columns in flight cost spills here)
    if (Sq) {
      hipLaunchKernelGGL((attn_masked_dq_kernel<decltype(t), decltype(dp)::value, KT>), dim3(B * H, cdiv(Sq, 128), p.qsplit), dim3(256), 0, st, p);
      if (p.qsplit > 1) sum_join<decltype(t)>(p.qpart, p.dq, p.dqs, (long)B * Sq * H * D, p.qsplit, B, Sq, H, D, scale, st);
    }
    if (Sk) {
      constexpr int NT = sizeof(t) == 4 && decltype(dp)::value == 128 ? 256 : 512;
      hipLaunchKernelGGL((attn_masked_dkv_kernel<decltype(t), decltype(dp)::value, decltype(kt)::value, NT>), dim3(B * Hk, cdiv(Sk, NT / 4), p.nsplit),
                         dim3(NT), 0, st, p);
      if (p.nsplit > 1) {
        const long n = (long)B * Sk * Hk * D;
        sum_join<decltype(t)>(p.part, p.dv, p.dvs, 2 * n, p.nsplit, B, Sk, Hk, D, 1.f, st);
        sum_join<decltype(t)>(p.part + n, p.dk, p.dks, 2 * n, p.nsplit, B, Sk, Hk, D, scale, st);
      }
    }
  });
  AOT_LAUNCH_CHECK();
}
