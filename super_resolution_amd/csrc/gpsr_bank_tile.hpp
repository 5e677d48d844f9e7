// gpsr_bank_tile.hpp -- a tile of bank rows against blocks of W = 32 or 16 query columns on the matrix units.
//
// Logits are formed transposed, S^T = K Q^T (rows of the bank down, columns = queries across), with
// v_mfma_f32_32x32x16_bf16 (16x16x32 for up to 16 columns): a lane then holds logits of ONE query, 16 of 32 rows (4 of 16), so
// the softmax statistics are lane-local but for an exchange between the wave's parts, and the accumulator registers, rounded
// to bf16, are the second product's operand as they are: O^T = V^T P^T contracts over rows, and the order of a contraction is
// free as long as both operands agree, so V^T is laid out in LDS in the order in which the accumulators hold the rows.
// Held values have at most 4 significant bits: bf16 holds them exactly.  Queries are split into Terms<DT>::N bf16 terms
// (8 bits each: bf16 queries 1, f16 2, f32 3), so that the products lose nothing that the caller's type can hold.  Weights are
// not the caller's; they enter with at least twice the bits of a bf16 output (16; f32 24) wherever that costs little: few queries and
// chosen pages wait for memory (a second term took pages_image of 40 000 queries from 125 to 129 us, 12 to
// each of 8 long banks from 57 to 60, 30 to each of 4 of 256 columns from 152 to 160, small calls not measurably).  Many bf16 queries over the whole bank keep one term of 8 bits, which adds up to 2^-8 of the mean |value| to an
// output that is rounded by 2^-8 of itself: two took 65 025 queries of 5000 rows from 127 to 164 us, 40 000 of 100 000 from 1190 to 1700.
#pragma once
#include "gpsr_bank.hpp"

#include <type_traits>

// What an accumulator of W columns holds: lane = part * W + column, E values, value e of row row(part, e).  A product contracts
// over STEP indices, 8 neighbouring ones for each part; slot(r) is where row r of a STEP goes for the second product.
template <int W> struct Geo;
template <> struct Geo<32> {
  typedef f16v Acc;
  static constexpr int E = 16, STEP = 16;
  __device__ __forceinline__ static int row(int part, int e) { return 8 * (e >> 2) + 4 * part + (e & 3); }
  __device__ __forceinline__ static int slot(int r) { return ((r >> 2) & 1) * 8 + (r >> 3) * 4 + (r & 3); }   // 0-3, 8-11 | 4-7, 12-15
  __device__ __forceinline__ static Acc mul(bf8 a, bf8 b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  template <class F> __device__ __forceinline__ static float parts(float x, const F& f) { return f(x, __shfl_xor(x, 32)); }
};
template <> struct Geo<16> {
  typedef f4v Acc;
  static constexpr int E = 4, STEP = 32;
  __device__ __forceinline__ static int row(int part, int e) { return 4 * part + e; }
  __device__ __forceinline__ static int slot(int r) { return ((r >> 2) & 3) * 8 + (r >> 4) * 4 + (r & 3); }   // 0-3, 16-19 | 4-7, 20-23 | ..
  __device__ __forceinline__ static Acc mul(bf8 a, bf8 b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  template <class F> __device__ __forceinline__ static float parts(float x, const F& f) {
    x = f(x, __shfl_xor(x, 16));
    return f(x, __shfl_xor(x, 32));
  }
};
__device__ __forceinline__ float max2(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float add2(float a, float b) { return a + b; }

template <int DT> struct Terms;
template <> struct Terms<GPSR_BF16> { static constexpr int N = 1; };
template <> struct Terms<GPSR_F16> { static constexpr int N = 2; };
template <> struct Terms<GPSR_F32> { static constexpr int N = 3; };

// terms of the weights where the matrix units are not what a call waits for
static constexpr int weight_terms(int nt) { return nt < 2 ? 2 : nt; }

// registers that a wave of 32 columns and NB x 32 rows at a time needs, roughly: sums, logits, query terms, the rest
static constexpr int tile_regs(int d, int nt, int nb) { return d / 2 + 16 * nb + nt * d / 4 + 64; }
// waves per SIMD that they are budgeted for
static constexpr int tile_waves(int d, int nt, int nb) { return tile_regs(d, nt, nb) <= 128 ? 4 : tile_regs(d, nt, nb) <= 250 ? 2 : 1; }

template <int DT>
__device__ __forceinline__ typename Row<DT>::T from_f32(float y) {
  if constexpr (DT == GPSR_BF16) return bf16_rne(y); else return (typename Row<DT>::T)y;
}

// y[8] as NT bf16 terms, each the rounding of what the terms before left over.  LARGE: y may be finite and beyond the largest bf16
// number, to which its first term then stops short.
template <int NT, bool LARGE = false>
__device__ __forceinline__ void split_terms(const float* y, bf8* t) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = y[i];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[n][i] = (__bf16)(LARGE && n == 0 && fabsf(r[i]) < __builtin_inff() ? __builtin_amdgcn_fmed3f(r[i], -0x1.fep127f, 0x1.fep127f) : r[i]);
      if (n + 1 < NT) r[i] -= (float)t[n][i];
    }
}

template <int DT, int D, int W = 32>
__device__ __forceinline__ void load_query(const typename Row<DT>::T* __restrict__ p, bool wide, bool there, int part,
                                           bf8 (&qf)[Terms<DT>::N][D / Geo<W>::STEP]) {
  constexpr int NT = Terms<DT>::N;
#pragma unroll
  for (int s = 0; s < D / Geo<W>::STEP; ++s) {
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (there) load8<DT>(p + s * Geo<W>::STEP + part * 8, wide, y);
    bf8 t[NT];
    split_terms<NT, DT == GPSR_F32>(y, t);
#pragma unroll
    for (int n = 0; n < NT; ++n) qf[n][s] = t[n];
  }
}

// ---- the tile in LDS: keys [KT][D + 8], values [D][KT] (rows of the bank permuted as above), offsets [KT], marks
// The values' 16-byte granules are exchanged within each 8 by the column's number: a wave writes 8 rows x 8 columns at a time,
// 8 columns apart, and reads 8 neighbouring columns, and neither falls on the same banks (with padded rows instead, 80 % of
// the LDS cycles of 180 000 rows x 12 queries were conflicts, and the kernel, then otherwise as well slower, took 153 us and not 87).
static constexpr int tile_lds(int d, int kt) { return (kt * (d + 8) + d * kt) * 2 + kt * 4 + (kt * (d / 32) + 4) * 4; }

template <int D, int KT>
struct Tile {
  static constexpr int KS = D + 8, VS = KT;
  static constexpr int SWZ = (KT >= 64 ? 7 : KT / 8 - 1);   // granules of a row that may change places
  uint16_t *k, *v;
  float* off;
  // A value group that is NaN is held as zeros, so that it cannot reach queries that do not see its row (0 * NaN); who does
  // see it is told by its mark: mark[row][group] = the number of the tile in which it is NaN, mark[KT][0] = of the last such
  // tile.  Numbers of earlier tiles need no clearing.  mark[KT][1] = the last tile with a row that has no weight (offset -inf:
  // it does not exist, or its key is past the range): its product with a query may still be infinite or NaN.
  unsigned* mark;
  __device__ Tile(char* sm) {
    k = (uint16_t*)sm; v = k + KT * KS; off = (float*)(v + D * VS); mark = (unsigned*)(off + KT);
  }
  // where slot s of column c lies
  __device__ __forceinline__ static int at(int c, int s) { return c * VS + (s ^ (((c ^ (c >> 3)) & SWZ) << 3)); }
  __device__ void clear_marks(int tid, int threads) {
    for (int i = tid; i < KT * (D / 32) + 2; i += threads) mark[i] = 0;
  }
  __device__ __forceinline__ bool weightless(unsigned number) const {
    return __builtin_amdgcn_readfirstlane(mark[KT * (D / 32) + 1]) == (int)number;
  }
};

__device__ __forceinline__ unsigned pack_lo(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ unsigned pack_hi(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// 2 columns of a row as bf16: element pair i (0..3) of code word w (4 bits), or of the word pair (8 bits)
template <int BITS, int I>
__device__ __forceinline__ unsigned pair(unsigned w0, unsigned w1, float s) {
  bf2 r;
  if constexpr (BITS == 4) r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s, I);
  else r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(I < 2 ? w0 : w1, s, (I & 1) != 0);
  return __builtin_bit_cast(unsigned, r);
}

// ---- where the rows of a walk come from: page(v) is the physical page of row v of the walk (-1: no such row), left(v) how many
// of the rows v .. v + 3 (one page's) exist.  Row v lies at v % page_rows of its page.  A walk has at least one row (len, n > 0);
// lookups behind its end read its last entry and are then discarded, which costs less than a branch.
struct WholeBank {
  const int32_t* tab;
  int64_t pages;
  int pshift;
  unsigned len;
  __device__ __forceinline__ int page(unsigned v) const {
    const int p = tab[min(v, len - 1) >> pshift];
    return v < len && (unsigned)p < (unsigned)pages ? p : -1;
  }
  __device__ __forceinline__ int left(unsigned v) const { return v < len ? (int)min(len - v, 4u) : 0; }
};
struct PageList {   // in LDS: physical pages and how many rows each has
  const int *phys, *rows;
  int pshift;
  unsigned n;
  __device__ __forceinline__ int page(unsigned v) const {
    const int p = phys[min(v >> pshift, n - 1)];
    return left(v) > 0 ? p : -1;
  }
  __device__ __forceinline__ int left(unsigned v) const {
    const unsigned i = v >> pshift;
    const int r = rows[min(i, n - 1)] - (int)(v & ((1u << pshift) - 1));
    return i < n ? min(r, 4) : 0;
  }
};
struct OnePage {
  int phys, rows;
  __device__ __forceinline__ int page(unsigned v) const { return (int)v < rows ? phys : -1; }
  __device__ __forceinline__ int left(unsigned v) const { return min(rows - (int)v, 4); }
};

// 32 columns of a row's key to LDS; MASKED: unless `there`, zeros and an offset of -inf instead
template <int BITS, int D, int KT, bool MASKED>
__device__ __forceinline__ void store_keys(const Tile<D, KT>& tile, int r, int g, const unsigned* w, const unsigned* sc, bool there,
                                           unsigned number) {
  constexpr int CW = BITS / 4;
  u4v* dst = (u4v*)(tile.k + r * Tile<D, KT>::KS + g * 32);
  const float s = scale_of(!MASKED || there ? sc[0] : 127u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned w0 = !MASKED || there ? w[CW * j] : 0u, w1 = !MASKED || there ? w[CW * j + CW - 1] : 0u;
    dst[j] = u4v{pair<BITS, 0>(w0, w1, s), pair<BITS, 1>(w0, w1, s), pair<BITS, 2>(w0, w1, s), pair<BITS, 3>(w0, w1, s)};
  }
  if (g == 0) {
    const float o = !MASKED || there ? __uint_as_float(sc[1]) : -__builtin_inff();
    tile.off[r] = o;
    if (o == -__builtin_inff()) tile.mark[KT * (D / 32) + 1] = number;
  }
}

// 8 columns of 4 rows' values to LDS, transposed; MASKED: zeros for rows r + left and behind
template <int BITS, int D, int KT, int W, bool MASKED>
__device__ __forceinline__ void store_values(const Tile<D, KT>& tile, int r, int c, const unsigned* w, const unsigned* sc, int left,
                                             unsigned number) {
  constexpr int CW = BITS / 4;
  unsigned y[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool here = !MASKED || j < left, nan = here && sc[j] == 255u, there = here && !nan;
    if (nan) { tile.mark[(r + j) * (D / 32) + c / 4] = number; tile.mark[KT * (D / 32)] = number; }
    const float s = scale_of(there ? sc[j] : 127u);
    const unsigned w0 = there ? w[CW * j] : 0u, w1 = there ? w[CW * j + CW - 1] : 0u;
    y[j][0] = pair<BITS, 0>(w0, w1, s); y[j][1] = pair<BITS, 1>(w0, w1, s);
    y[j][2] = pair<BITS, 2>(w0, w1, s); y[j][3] = pair<BITS, 3>(w0, w1, s);
  }
  // rows r .. r + 3 of the tile are 4 neighbouring slots of a column
  const int slot = (r & ~(Geo<W>::STEP - 1)) + Geo<W>::slot(r & (Geo<W>::STEP - 1));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    *(u2v*)(tile.v + Tile<D, KT>::at(c * 8 + 2 * e, slot)) = u2v{pack_lo(y[0][e], y[1][e]), pack_lo(y[2][e], y[3][e])};
    *(u2v*)(tile.v + Tile<D, KT>::at(c * 8 + 2 * e + 1, slot)) = u2v{pack_hi(y[0][e], y[1][e]), pack_hi(y[2][e], y[3][e])};
  }
}

// ---- a tile on its way: codes are loaded a tile ahead of their use, page numbers two.  The tile is 2 U units, U of keys (32
// columns of a row each) and U of values (8 columns of 4 rows each), dealt to the threads in that order: a thread has one kind or
// the other at a time and holds both in the same registers.
template <int BITS, int D, int KT, int NTH>
struct Fetch {
  static constexpr int U = KT * D / 32, N = (2 * U + NTH - 1) / NTH;
  static constexpr int CW = BITS / 4;                    // code words of 8 columns
  static constexpr bool EVEN = 2 * U % NTH == 0;
  int page[N], left[N];                                  // of the next tile; page -1: the row does not exist
  int fpage[N], fleft[N];                                // of the tile whose codes are under way
  unsigned w[N][4 * CW], sc[N][4];                        // keys: scale byte and offset in sc[0], sc[1]

  // unit i of this thread: keys? and its number among its kind
  __device__ __forceinline__ static bool keys(int i, int tid) {
    return NTH * (i + 1) <= U ? true : NTH * i >= U ? false : tid + NTH * i < U;
  }
  __device__ __forceinline__ static int row(int i, int tid) {
    const int u = tid + NTH * i;
    return keys(i, tid) ? u / (D / 32) : (u - U) / (D / 8) * 4;
  }

  // page numbers of the rows from p0 on
  template <class Rows>
  __device__ __forceinline__ void pages(const Rows& rows, unsigned p0, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned r = p0 + row(i, tid);
      page[i] = rows.page(r);
      left[i] = rows.left(r);
    }
  }

  // codes, scales and offsets of the rows whose pages were fetched last; for a row that does not exist, some other one's
  __device__ __forceinline__ void codes(const gpsr_bank& bk, int h, int pshift, unsigned p0, int tid) {
    const unsigned mask = (1u << pshift) - 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = tid + NTH * i;
      fpage[i] = page[i]; fleft[i] = page[i] >= 0 ? left[i] : 0;
      if (!EVEN && u >= 2 * U) continue;
      const size_t at = (((size_t)max(page[i], 0) * bk.heads + h) << pshift) + ((p0 + row(i, tid)) & mask);
      if (keys(i, tid)) {
        const int g = u % (D / 32);
        const u4v* src = (const u4v*)(bk.k_codes + at * (size_t)(D * BITS / 8) + g * (4 * BITS));
#pragma unroll
        for (int j = 0; j < CW; ++j) {
          const u4v a = src[j];
          w[i][4 * j] = a.x; w[i][4 * j + 1] = a.y; w[i][4 * j + 2] = a.z; w[i][4 * j + 3] = a.w;
        }
        sc[i][0] = bk.k_scales[at * (size_t)(D / 32) + g];
        sc[i][1] = __float_as_uint(bk.offset[at]);
      } else {
        const int c = (u - U) % (D / 8);
        const uint8_t* src = bk.v_codes + at * (size_t)(D * BITS / 8) + c * BITS;
        const uint8_t* scale = bk.v_scales + at * (size_t)(D / 32) + c / 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // rows of one page: page_rows is a multiple of 16
          if constexpr (CW == 1) w[i][j] = *(const unsigned*)(src + j * (D * BITS / 8));
          else { const u2v a = *(const u2v*)(src + j * (D * BITS / 8)); w[i][2 * j] = a.x; w[i][2 * j + 1] = a.y; }
          sc[i][j] = scale[j * (D / 32)];
        }
      }
    }
  }

  // decodes them to LDS; rows that do not exist become zeros with an offset of -inf
  template <int W>
  __device__ __forceinline__ void store(const Tile<D, KT>& tile, int tid, unsigned number) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = tid + NTH * i;
      if (!EVEN && u >= 2 * U) continue;
      const int r = row(i, tid);
      if (keys(i, tid)) store_keys<BITS, D, KT, true>(tile, r, u % (D / 32), w[i], sc[i], fpage[i] >= 0, number);
      else store_values<BITS, D, KT, W, true>(tile, r, (u - U) % (D / 8), w[i], sc[i], fleft[i], number);
    }
  }
};

// ---- the same for one wave with a tile of 32 rows of its own.  Its 16-row halves lie in one page each, so page numbers and
// addresses are uniform, a lane's offsets stay the same from tile to tile, and only the bank's last tile has rows to be left out
// (with Fetch, half of the instructions of a tile were addresses and masks).
template <int BITS, int D>
struct WaveFetch {
  static constexpr int KT = 32, U = D, N = 2 * U / 64, CW = BITS / 4, RB = D * BITS / 8, G = D / 32;
  int page[2];                       // of the halves of the next tile; -1: not there
  int left;                          // rows of the tile under way that exist, if its pages do
  bool there[2];
  unsigned w[N][4 * CW], sc[N][4];

  __device__ __forceinline__ static bool keys(int i, int lane) { return 64 * (i + 1) <= U ? true : 64 * i >= U ? false : lane + 64 * i < U; }
  __device__ __forceinline__ static int row(int i, int lane) {
    const int u = lane + 64 * i;
    return keys(i, lane) ? u / G : (u - U) / (D / 8) * 4;
  }
  __device__ __forceinline__ void pages(const WholeBank& rows, unsigned p0) {
#pragma unroll
    for (int k = 0; k < 2; ++k) page[k] = __builtin_amdgcn_readfirstlane(rows.page(p0 + 16 * k));
  }
  __device__ __forceinline__ void codes(const gpsr_bank& bk, int h, int pshift, unsigned p0, unsigned len, int lane) {
    const unsigned mask = (1u << pshift) - 1;
    size_t at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      there[k] = page[k] >= 0;
      at[k] = (((size_t)max(page[k], 0) * bk.heads + h) << pshift) + ((p0 + 16 * k) & mask) - 16 * k;
    }
    left = len > p0 ? (int)min(len - p0, 32u) : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = lane + 64 * i, r = row(i, lane);
      const size_t base = r < 16 ? at[0] : at[1];
      if (keys(i, lane)) {
        const int g = u % G;
        const u4v* src = (const u4v*)(bk.k_codes + base * RB + (r * RB + g * (4 * BITS)));
#pragma unroll
        for (int j = 0; j < CW; ++j) {
          const u4v a = src[j];
          w[i][4 * j] = a.x; w[i][4 * j + 1] = a.y; w[i][4 * j + 2] = a.z; w[i][4 * j + 3] = a.w;
        }
        sc[i][0] = (bk.k_scales + base * G)[r * G + g];
        sc[i][1] = __float_as_uint((bk.offset + base)[r]);
      } else {
        const int c = (u - U) % (D / 8);
        const uint8_t* src = bk.v_codes + base * RB + (r * RB + c * BITS);
        const uint8_t* scale = bk.v_scales + base * G + (r * G + c / 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (CW == 1) w[i][j] = *(const unsigned*)(src + j * RB);
          else { const u2v a = *(const u2v*)(src + j * RB); w[i][2 * j] = a.x; w[i][2 * j + 1] = a.y; }
          sc[i][j] = scale[j * G];
        }
      }
    }
  }
  template <int W>
  __device__ __forceinline__ void store(const Tile<D, KT>& tile, int lane, unsigned number) {
    const auto all = [&](auto masked) {
      constexpr bool M = decltype(masked)::value;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int u = lane + 64 * i, r = row(i, lane);
        const bool half = r < 16 ? there[0] : there[1];
        if (keys(i, lane)) store_keys<BITS, D, KT, M>(tile, r, u % G, w[i], sc[i], half && r < left, number);
        else store_values<BITS, D, KT, W, M>(tile, r, (u - U) % (D / 8), w[i], sc[i], half ? min(left - r, 4) : 0, number);
      }
    };
    if (there[0] && there[1] && left == 32) all(std::false_type()); else all(std::true_type());
  }
};

// raw logits q.k + offset of NB x W rows (from r0 on) for a wave's W columns; weightless: rows with an offset of -inf are among the
// tile's, and their logits are -inf whatever the query holds
template <int D, int KT, int NT, int NB, int W>
__device__ __forceinline__ void tile_logits(const Tile<D, KT>& tile, int r0, int col, int part, bool weightless,
                                            const bf8 (&qf)[NT][D / Geo<W>::STEP], typename Geo<W>::Acc (&s)[NB]) {
  typedef Geo<W> X;
#pragma unroll
  for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
    for (int e = 0; e < X::E; e += 4) {
      const f4v a = *(const f4v*)(tile.off + r0 + kb * W + X::row(part, e));
#pragma unroll
      for (int j = 0; j < 4; ++j) s[kb][e + j] = a[j];
    }
    const uint16_t* base = tile.k + (r0 + kb * W + col) * Tile<D, KT>::KS + part * 8;
#pragma unroll
    for (int d = 0; d < D / X::STEP; ++d) {
      const bf8 a = *(const bf8*)(base + d * X::STEP);
#pragma unroll
      for (int t = 0; t < NT; ++t) s[kb] = X::mul(a, qf[t][d], s[kb]);
    }
  }
  if (weightless) {
    asm volatile("");        // not to be computed for the other tiles
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int e = 0; e < X::E; e += 4) {
        const f4v a = *(const f4v*)(tile.off + r0 + kb * W + X::row(part, e));
#pragma unroll
        for (int j = 0; j < 4; ++j) s[kb][e + j] = a[j] == -__builtin_inff() ? a[j] : s[kb][e + j];
      }
  }
}

// ---- running softmax of a wave's columns: m the power of two that weights are taken against (logit * log2 e; -inf: no row
// seen), l this part's sum of weights, o = sum of weights * values
template <int D, int W>
struct Soft {
  typedef Geo<W> X;
  typename X::Acc o[D / W];
  float m, l;
  unsigned nan;         // bit g: a row that the column sees is NaN in columns 32 g .. of its values
  __device__ __forceinline__ void clear() {
    m = -__builtin_inff(); l = 0.f; nan = 0;
#pragma unroll
    for (int d = 0; d < D / W; ++d)
#pragma unroll
      for (int e = 0; e < X::E; ++e) o[d][e] = 0.f;
  }
  __device__ __forceinline__ bool wants_move() const { return __ballot(m == -__builtin_inff() || l > 0x1p40f) != 0; }
  // Whether a sum came near the end of its range, or went past it (or met a NaN: then a second walk changes nothing): a weight
  // far above the reference, or values near the end of theirs.  A sum that passed it stays infinite or NaN.
  __device__ __forceinline__ bool lost() const {
    bool ok = l < 0x1p120f;
#pragma unroll
    for (int d = 0; d < D / W; ++d)
#pragma unroll
      for (int e = 0; e < X::E; ++e) ok = ok && fabsf(o[d][e]) < 0x1p120f;
    return !ok;
  }
  __device__ __forceinline__ void rescale(float a) {
    l *= a;
#pragma unroll
    for (int d = 0; d < D / W; ++d)
#pragma unroll
      for (int e = 0; e < X::E; ++e) o[d][e] *= a;
  }
  __device__ __forceinline__ void spoil() {
    if (__ballot(nan != 0))
#pragma unroll
      for (int d = 0; d < D / W; ++d)
        if (nan >> (d * W / 32) & 1)
#pragma unroll
          for (int e = 0; e < X::E; ++e) o[d][e] = __builtin_nanf("");
  }
  // divides; l becomes the whole sum
  __device__ __forceinline__ void finish() {
    l = X::parts(l, add2);
    const float r = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < D / W; ++d)
#pragma unroll
      for (int e = 0; e < X::E; ++e) o[d][e] *= r;
  }
  __device__ __forceinline__ float lse() const { return l == 0.f ? -__builtin_inff() : (log2f(l) + m) * 0.6931471805599453f; }
  // wave 0 gets the sum over WK waves that held the same columns; buf: 64 (D W / 64 + 2) floats
  template <int WK>
  __device__ __forceinline__ void join(float* buf, int wave, int lane) {
    for (int w = 1; w < WK; ++w) {
      if (wave == w) {
        buf[lane] = m; buf[64 + lane] = l;
#pragma unroll
        for (int d = 0; d < D / W; ++d)
#pragma unroll
          for (int e = 0; e < X::E; ++e) buf[(2 + d * X::E + e) * 64 + lane] = o[d][e];
      }
      __syncthreads();
      if (wave == 0) {
        const float m2 = buf[lane], mn = fmaxf(m, m2), safe = mn == -__builtin_inff() ? 0.f : mn;
        const float a = exp2f(m - safe), b = exp2f(m2 - safe);
        m = mn;
        l = l * a + buf[64 + lane] * b;
#pragma unroll
        for (int d = 0; d < D / W; ++d)
#pragma unroll
          for (int e = 0; e < X::E; ++e) o[d][e] = o[d][e] * a + buf[(2 + d * X::E + e) * 64 + lane] * b;
      }
      __syncthreads();
    }
  }
  // a lane's part of its column: 4 neighbouring dims at a time
  template <int DT>
  __device__ __forceinline__ void store(typename Row<DT>::T* __restrict__ out, int part) const {
#pragma unroll
    for (int d = 0; d < D / W; ++d)
#pragma unroll
      for (int e = 0; e < X::E; e += 4) {
        typename Row<DT>::T* p = out + d * W + X::row(part, e);
        if constexpr (DT == GPSR_F32) {
          *(f4v*)p = f4v{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
        } else {
          unsigned w[2];
#pragma unroll
          for (int j = 0; j < 2; ++j)
            w[j] = (unsigned)__builtin_bit_cast(uint16_t, from_f32<DT>(o[d][e + 2 * j])) |
                   ((unsigned)__builtin_bit_cast(uint16_t, from_f32<DT>(o[d][e + 2 * j + 1])) << 16);
          *(u2v*)p = u2v{w[0], w[1]};
        }
      }
  }
  // a partial result: sums [D], and the reference and the sum of weights
  __device__ __forceinline__ void store_partial(float* __restrict__ p, f2v* __restrict__ stat, int part) const {
    const float all = X::parts(l, add2);
#pragma unroll
    for (int d = 0; d < D / W; ++d)
#pragma unroll
      for (int e = 0; e < X::E; e += 4) *(f4v*)(p + d * W + X::row(part, e)) = f4v{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
    if (part == 0) *stat = f2v{m, all};
  }
};

// Rows of the tile that a column sees and whose values are NaN; seen(r): whether it does not skip row r of the wave's KW.
template <int D, int KT, int KW, int W, class Seen>
__device__ __forceinline__ void tile_marks(const Tile<D, KT>& tile, int wrow, unsigned number, Soft<D, W>& st, const Seen& seen) {
  if (tile.mark[KT * (D / 32)] != number) return;
#pragma unroll 1
  for (int r = 0; r < KW; ++r) {
    if (tile.off[wrow + r] == -__builtin_inff()) continue;
    unsigned bits = 0;
    for (int g = 0; g < D / 32; ++g) bits |= (tile.mark[(wrow + r) * (D / 32) + g] == number ? 1u : 0u) << g;
    st.nan |= seen(r) ? bits : 0u;
  }
}

// One step of the running softmax: logits in, weights times values added to the state.
//   MOVE: the reference becomes the maximum so far, as a power of two, and the state is rescaled: weights are at most
//     2^-above, so that fewer than 2^(above - 1) rows of any values stay in range.
//   otherwise it stays, which saves the maximum of every tile and the wait for it: bf16 and the sums have range to spare, and
//     their precision is relative.  Soft::wants_move says when it has to be moved (nothing seen yet, or a sum past 2^40); what
//     a weight far above the reference does is for the caller to look for (Soft::lost), and to walk again with MOVE only.
// WT: bf16 terms of the weights.
template <int D, int KT, int WT, int NB, int W, bool MOVE>
__device__ __forceinline__ void tile_accumulate(const Tile<D, KT>& tile, int r0, int col, int part, float c2, float above,
                                                typename Geo<W>::Acc (&s)[NB], Soft<D, W>& st) {
  typedef Geo<W> X;
  if constexpr (MOVE) {
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int e = 0; e < X::E; ++e) mx = fmaxf(mx, s[kb][e]);
    float mn = fmaxf(st.m, fmaf(X::parts(mx, max2), c2, above));
    if (X::parts(st.l, max2) > 0x1p40f) mn = fmaxf(mn, st.m + 40.f);
    st.rescale(mn == -__builtin_inff() ? 1.f : exp2f(st.m - mn));
    st.m = mn;
  }
  const float ref = st.m == -__builtin_inff() ? 0.f : -st.m;
  float sum = 0.f;
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int e = 0; e < X::E; ++e) {
      const float w = __builtin_amdgcn_exp2f(fmaf(s[kb][e], c2, ref));
      s[kb][e] = w;
      sum += w;
    }
  st.l += sum;
  constexpr int CH = NB * W / X::STEP;     // contractions of STEP rows
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    float y[8];
    if constexpr (W == 32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = s[k / 2][8 * (k % 2) + e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = s[2 * k + e / 4][e % 4];
    }
    bf8 p[WT];
    split_terms<WT>(y, p);
#pragma unroll
    for (int d = 0; d < D / W; ++d) {
      const bf8 a = *(const bf8*)(tile.v + Tile<D, KT>::at(d * W + col, r0 + k * X::STEP + part * 8));
#pragma unroll
      for (int t = 0; t < WT; ++t) st.o[d] = X::mul(a, p[t], st.o[d]);
    }
  }
}

// Joins the partial results of one column, at most 64 for each of its WJ waves (1: four columns a workgroup; 4).  First lane i weighs
// partial i, then the lanes spread over four partials or more of several rows at a time (with the weights formed along the way
// each load waited for the one before it: 30 against 9 us for 64 partials of 96 columns).  Column (t, g) of bank head bh has its n
// partials at numbers bh * per_bh + t * per_t + g * per_g + i * per_i.
template <int DT, int D, int WJ = 1>
__global__ void __launch_bounds__(256)
k_bank_join(const float* __restrict__ sums, const f2v* __restrict__ stats, int T, int G, int H, int64_t C, int n, size_t per_bh,
            size_t per_g, size_t per_t, size_t per_i, typename Row<DT>::T* __restrict__ out, float* __restrict__ lse) {
  // Weights and sums go from lane to lane through LDS, a wave's own part of it.  With permutes (ds_bpermute) the f32 form of 32 columns
  // added other lanes' values to one column in 3000, never the same ones; why is not known: its assembly reads right, and the other
  // types' forms, with as many permutes under way, never showed it.  Tests repeat every way over tens of thousands of columns.
  __shared__ float tops[4], ls[4], weight[4][64];
  __shared__ __attribute__((aligned(16))) float part[4][64][4];
  const auto sync = [] { asm volatile("" ::: "memory"); __builtin_amdgcn_wave_barrier(); };
  const int lane = threadIdx.x & 63, wave = wave_of(threadIdx.x);
  const int64_t c = WJ > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (c >= C) return;            // WJ > 1: never
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t t = c / G;
  const int g = (int)(c - t * G), hq = h * G + g;
  if (WJ > 1) n = (n - wave + 3) / 4;               // this wave's: wave, wave + 4, ..
  const size_t at = (size_t)(b * H + h) * per_bh + t * per_t + g * per_g + (WJ > 1 ? wave * per_i : 0);
  if (WJ > 1) per_i *= 4;
  const float* p = sums + at * D;
  const size_t step = per_i * D;
  float m = -__builtin_inff(), l = 0.f;
  if (lane < n) { const f2v x = stats[at + lane * per_i]; m = x.x; l = x.y; }
  const unsigned long long used = __ballot(l != 0.f);      // the others saw nothing, and their sums were not written
  float top = l != 0.f ? m : -__builtin_inff();
  top = wave_all(top, -__builtin_inff(), max2);
  if constexpr (WJ > 1) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  }
  float w = l != 0.f ? exp2f(m - (top == -__builtin_inff() ? 0.f : top)) : 0.f;
  l = l != 0.f ? l * w : 0.f;
  l = wave_all(l, 0.f, add2);
  if constexpr (WJ > 1) {
    if (lane == 0) ls[wave] = l;
    __syncthreads();
    l = (ls[0] + ls[1]) + (ls[2] + ls[3]);
  }
  w = l != 0.f ? w / l : 0.f;          // before the sums: a mean of values near the end of their range stays in it
  weight[wave][lane] = w;
  sync();
  // 4 columns a lane, R lanes a row, RP rows at a time
  constexpr int R = D / 4, RP = 64 / R;
  const int row = lane / R, c4 = (lane - row * R) * 4;
  float acc[4] = {0, 0, 0, 0};
  for (int i0 = 0; i0 < n; i0 += 4 * RP) {
    f4v y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *(const f4v*)(p + min(i0 + j * RP + row, n - 1) * step + c4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * RP + row;
      const bool use = row < RP && (used >> (i & 63) & 1) && i < n;
      const float wj = weight[wave][i & 63];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = use ? fmaf(wj, y[j][e], acc[e]) : acc[e];
    }
  }
  *(f4v*)part[wave][lane] = f4v{acc[0], acc[1], acc[2], acc[3]};
  if constexpr (WJ > 1) __syncthreads(); else sync();
  if (WJ > 1 && wave) return;
  if (lane < R)
#pragma unroll
    for (int k = 1; k < WJ * RP; ++k) {
      const f4v y = *(const f4v*)part[WJ > 1 ? k / RP : wave][lane + k % RP * R];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += y[e];
    }
  typename Row<DT>::T* o = out + (((size_t)b * T + t) * (size_t)(H * G) + hq) * D + c4;
  if (lane < R) {
    if constexpr (DT == GPSR_F32) *(f4v*)o = f4v{acc[0], acc[1], acc[2], acc[3]};
    else {
      unsigned x[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        x[j] = (unsigned)__builtin_bit_cast(uint16_t, from_f32<DT>(acc[2 * j])) | ((unsigned)__builtin_bit_cast(uint16_t, from_f32<DT>(acc[2 * j + 1])) << 16);
      *(u2v*)o = u2v{x[0], x[1]};
    }
  }
  if (lse && lane == 0) lse[((size_t)b * (H * G) + hq) * T + t] = l == 0.f ? -__builtin_inff() : (log2f(l) + top) * 0.6931471805599453f;
}

// ---- host side
static inline const char* attend_wrong(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* length,
                                       const void* q, int dtype, int q_heads, const int64_t* qst, float scale, const void* out) {
  if (const char* w = bank_wrong(bank)) return w;
  if ((!table && table_pages) || !length || !q || !qst || !out) return "bank_attend: null pointer";
  if (!type_ok(dtype)) return "bank_attend: dtype";
  if (B > 65535) return "bank_attend: more than 65535 entries";
  if (table_pages < 0) return "bank_attend: table_pages";
  if (q_heads < 1 || q_heads > 65535 || q_heads % bank->heads) return "bank_attend: query heads must be a multiple of the bank's heads, up to 65535";
  // the kernels take powers of two: scale * log2 e has to be finite too
  if (!(scale > 0.f) || scale > 2.35e38f) return "bank_attend: scale must be positive and at most 2.35e38";
  if ((uintptr_t)out & 15) return "bank_attend: out must be 16-byte aligned";
  return nullptr;
}

#define BANK_DISPATCH_D(F, DT, BITS, dim)                                        \
  switch (dim) {                                                                 \
    case 32: F(DT, BITS, 32); break;                                             \
    case 64: F(DT, BITS, 64); break;                                             \
    case 96: F(DT, BITS, 96); break;                                             \
    case 128: F(DT, BITS, 128); break;                                           \
    case 192: F(DT, BITS, 192); break;                                           \
    default: F(DT, BITS, 256); break;                                            \
  }
#define BANK_DISPATCH_B(F, DT, bits, dim)                                        \
  if ((bits) == 4) BANK_DISPATCH_D(F, DT, 4, dim) else BANK_DISPATCH_D(F, DT, 8, dim)
#define BANK_DISPATCH(F, dtype, bits, dim)                                       \
  if ((dtype) == GPSR_BF16) { BANK_DISPATCH_B(F, GPSR_BF16, bits, dim) }         \
  else if ((dtype) == GPSR_F16) { BANK_DISPATCH_B(F, GPSR_F16, bits, dim) }      \
  else { BANK_DISPATCH_B(F, GPSR_F32, bits, dim) }
