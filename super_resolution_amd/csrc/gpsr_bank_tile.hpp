// gpsr_bank_tile.hpp -- a tile of bank rows against 32-column blocks of queries on the matrix units.
//
// Logits are formed transposed, S^T = K Q^T (rows of the bank down, columns = queries across), with v_mfma_f32_32x32x16_bf16:
// a lane then holds 16 logits of ONE query for each 32 rows, so the softmax statistics are lane-local but for one exchange
// between the wave's halves, and the accumulator registers, rounded to bf16, are the second product's operand as they are:
// O^T = V^T P^T contracts over rows, and the order of a contraction is free as long as both operands agree, so V^T is laid
// out in LDS in the order in which the accumulators hold the rows (within 16 rows: 0-3, 8-11 | 4-7, 12-15).
// Held values have at most 4 significant bits: bf16 holds them exactly.  Queries and weights are split into Terms<DT>::N bf16
// terms (8 bits each: bf16 queries 1, f16 2, f32 3), so that the products lose nothing that the caller's type can hold.
#pragma once
#include "gpsr_bank.hpp"

template <int DT> struct Terms;
template <> struct Terms<GPSR_BF16> { static constexpr int N = 1; };
template <> struct Terms<GPSR_F16> { static constexpr int N = 2; };
template <> struct Terms<GPSR_F32> { static constexpr int N = 3; };

// blocks of 32 columns that a wave holds: two halve the LDS reads for a product, where the registers allow it
static constexpr int tile_nq(int d, int nt) { return nt == 1 && d <= 64 ? 2 : 1; }
// waves per SIMD that the registers are budgeted for
static constexpr int tile_waves(int d, int nt, int nq) { return (d * nq * (nt + 1)) / 4 + 32 * nq > 160 ? 1 : 2; }

template <int DT>
__device__ __forceinline__ typename Row<DT>::T from_f32(float y) {
  if constexpr (DT == GPSR_BF16) return bf16_rne(y); else return (typename Row<DT>::T)y;
}

// y[8] as NT bf16 terms, each the rounding of what the terms before left over
template <int NT>
__device__ __forceinline__ void split_terms(const float* y, bf8* t) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = y[i];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[n][i] = (__bf16)r[i];
      if (n + 1 < NT) r[i] -= (float)t[n][i];
    }
}

template <int DT, int D>
__device__ __forceinline__ void load_query(const typename Row<DT>::T* __restrict__ p, bool wide, bool there, int half,
                                           bf8 (&qf)[Terms<DT>::N][D / 16]) {
  constexpr int NT = Terms<DT>::N;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (there) load8<DT>(p + s * 16 + half * 8, wide, y);
    bf8 t[NT];
    split_terms<NT>(y, t);
#pragma unroll
    for (int n = 0; n < NT; ++n) qf[n][s] = t[n];
  }
}

// ---- the tile in LDS: keys [KT][D + 8], values [D][KT + 8] (rows permuted as above), offsets [KT], rows whose values are NaN
static constexpr int tile_lds(int d, int kt) { return (kt * (d + 8) + d * (kt + 8)) * 2 + kt * 4 + (kt * (d / 32) + 4) * 4; }

template <int D, int KT>
struct Tile {
  static constexpr int KS = D + 8, VS = KT + 8;
  uint16_t *k, *v;
  float* off;
  // A value group that is NaN is held as zeros, so that it cannot reach queries that do not see its row (0 * NaN); who does
  // see it is told by its mark: mark[row][group] = the number of the tile in which it is NaN, mark[KT][0] = of the last such
  // tile.  Numbers of earlier tiles need no clearing.
  unsigned* mark;
  __device__ Tile(char* sm) {
    k = (uint16_t*)sm; v = k + KT * KS; off = (float*)(v + D * VS); mark = (unsigned*)(off + KT);
  }
  __device__ void clear_marks(int tid) {
    for (int i = tid; i < KT * (D / 32) + 1; i += 256) mark[i] = 0;
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
// of the rows v .. v + 3 (one page's) exist.  Row v lies at v % page_rows of its page.
struct WholeBank {
  const int32_t* tab;
  int64_t pages;
  int pshift;
  unsigned len;
  __device__ __forceinline__ int page(unsigned v) const {
    const int p = v < len ? tab[v >> pshift] : -1;
    return (unsigned)p < (unsigned)pages ? p : -1;
  }
  __device__ __forceinline__ int left(unsigned v) const { return v < len ? (int)min(len - v, 4u) : 0; }
};
struct PageList {   // in LDS: physical pages and how many rows each has
  const int *phys, *rows;
  int pshift;
  unsigned n;
  __device__ __forceinline__ int page(unsigned v) const { return left(v) > 0 ? phys[v >> pshift] : -1; }
  __device__ __forceinline__ int left(unsigned v) const {
    const unsigned i = v >> pshift;
    return i < n ? min(rows[i] - (int)(v & ((1u << pshift) - 1)), 4) : 0;
  }
};
struct OnePage {
  int phys, rows;
  __device__ __forceinline__ int page(unsigned v) const { return (int)v < rows ? phys : -1; }
  __device__ __forceinline__ int left(unsigned v) const { return min(rows - (int)v, 4); }
};

// ---- a tile on its way: codes are loaded a tile ahead of their use, page numbers two
template <int BITS, int D, int KT>
struct Fetch {
  static constexpr int U = KT * D / 32;                  // units of keys (a row's 32 columns) and of values (4 rows x 8 columns)
  static constexpr int NU = (U + 255) / 256;
  static constexpr int W = BITS / 4;                     // code words of 8 columns
  int kpage[NU], vpage[NU];                              // -1: the row does not exist
  int fk[NU];
  unsigned kw[NU][4 * W], vw[NU][4][W];
  unsigned ks[NU];
  unsigned vs[NU][4];
  int vleft[NU], fleft[NU];
  float offs[NU];

  // page numbers of the rows from p0 on
  template <class Rows>
  __device__ __forceinline__ void pages(const Rows& rows, unsigned p0, int tid) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = tid + 256 * i, x = 255 - tid + 256 * i;
      const unsigned kr = p0 + u / (D / 32), vr = p0 + x / (D / 8) * 4;
      kpage[i] = u < U ? rows.page(kr) : -1;
      vpage[i] = x < U ? rows.page(vr) : -1;
      vleft[i] = rows.left(vr);
    }
  }

  // codes, scales and offsets of the rows whose pages were fetched last
  __device__ __forceinline__ void codes(const gpsr_bank& bk, int h, int pshift, unsigned p0, int tid) {
    const unsigned mask = (1u << pshift) - 1;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = tid + 256 * i, x = 255 - tid + 256 * i;
      fk[i] = kpage[i];
      if (kpage[i] >= 0) {
        const int r = u / (D / 32), g = u % (D / 32);
        const size_t row = (((size_t)kpage[i] * bk.heads + h) << pshift) + ((p0 + r) & mask);
        const u4v* src = (const u4v*)(bk.k_codes + row * (size_t)(D * BITS / 8) + g * (4 * BITS));
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const u4v a = src[j];
          kw[i][4 * j] = a.x; kw[i][4 * j + 1] = a.y; kw[i][4 * j + 2] = a.z; kw[i][4 * j + 3] = a.w;
        }
        ks[i] = bk.k_scales[row * (size_t)(D / 32) + g];
        if (g == 0) offs[i] = bk.offset[row];
      }
      fleft[i] = vpage[i] >= 0 ? vleft[i] : 0;
      if (vpage[i] >= 0) {
        const int r = x / (D / 8) * 4, c = x % (D / 8);
        const size_t row = (((size_t)vpage[i] * bk.heads + h) << pshift) + ((p0 + r) & mask);
        const uint8_t* src = bk.v_codes + row * (size_t)(D * BITS / 8) + c * BITS;
        const uint8_t* sc = bk.v_scales + row * (size_t)(D / 32) + c / 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // rows of one page: P is a multiple of 16
          if constexpr (W == 1) vw[i][j][0] = *(const unsigned*)(src + j * (D * BITS / 8));
          else { const u2v a = *(const u2v*)(src + j * (D * BITS / 8)); vw[i][j][0] = a.x; vw[i][j][1] = a.y; }
          vs[i][j] = sc[j * (D / 32)];
        }
      }
    }
  }

  // decodes them to LDS; rows that do not exist become zeros with an offset of -inf
  __device__ __forceinline__ void store(const Tile<D, KT>& tile, int tid, unsigned number) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = tid + 256 * i, x = 255 - tid + 256 * i;
      if (u < U) {
        const int r = u / (D / 32), g = u % (D / 32);
        const bool there = fk[i] >= 0;
        u4v* dst = (u4v*)(tile.k + r * Tile<D, KT>::KS + g * 32);
        const float s = scale_of(there ? ks[i] : 127u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned w0 = there ? kw[i][W * j] : 0u, w1 = there ? kw[i][W * j + W - 1] : 0u;
          dst[j] = u4v{pair<BITS, 0>(w0, w1, s), pair<BITS, 1>(w0, w1, s), pair<BITS, 2>(w0, w1, s), pair<BITS, 3>(w0, w1, s)};
        }
        if (g == 0) tile.off[r] = there ? offs[i] : -__builtin_inff();
      }
      if (x < U) {
        const int r = x / (D / 8) * 4, c = x % (D / 8);
        unsigned y[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool here = j < fleft[i], nan = here && vs[i][j] == 255u, there = here && !nan;
          if (nan) { tile.mark[(r + j) * (D / 32) + c / 4] = number; tile.mark[KT * (D / 32)] = number; }
          const float s = scale_of(there ? vs[i][j] : 127u);
          const unsigned w0 = there ? vw[i][j][0] : 0u, w1 = there ? vw[i][j][W - 1] : 0u;
          y[j][0] = pair<BITS, 0>(w0, w1, s); y[j][1] = pair<BITS, 1>(w0, w1, s);
          y[j][2] = pair<BITS, 2>(w0, w1, s); y[j][3] = pair<BITS, 3>(w0, w1, s);
        }
        // rows r .. r + 3 of the tile are 4 neighbouring slots of a column
        const int k16 = r & 15, slot = (r & ~15) + ((k16 >> 2) & 1) * 8 + (k16 >> 3) * 4;
        uint16_t* dst = tile.v + (c * 8) * Tile<D, KT>::VS + slot;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          *(u2v*)(dst + (2 * e) * Tile<D, KT>::VS) = u2v{pack_lo(y[0][e], y[1][e]), pack_lo(y[2][e], y[3][e])};
          *(u2v*)(dst + (2 * e + 1) * Tile<D, KT>::VS) = u2v{pack_hi(y[0][e], y[1][e]), pack_hi(y[2][e], y[3][e])};
        }
      }
    }
  }
};

// raw logits q.k + offset of the wave's NB x 32 rows (from wrow on) for its NQ x 32 columns
template <int D, int KT, int NT, int NQ, int NB>
__device__ __forceinline__ void tile_logits(const Tile<D, KT>& tile, int wrow, int col, int half, const bf8 (&qf)[NQ][NT][D / 16],
                                            f16v (&s)[NB][NQ]) {
#pragma unroll
  for (int kb = 0; kb < NB; ++kb) {
    f16v o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f4v a = *(const f4v*)(tile.off + wrow + kb * 32 + 8 * i + 4 * half);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[4 * i + j] = a[j];
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) s[kb][n] = o;
    const uint16_t* base = tile.k + (wrow + kb * 32 + col) * Tile<D, KT>::KS + half * 8;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const bf8 a = *(const bf8*)(base + d * 16);
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int t = 0; t < NT; ++t) s[kb][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qf[n][t][d], s[kb][n], 0, 0, 0);
    }
  }
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// ---- running softmax of a wave's columns: m the maximum raw logit, l this half's sum of weights, o = sum of weights * values
template <int D, int NQ>
struct Soft {
  f16v o[D / 32][NQ];
  float m[NQ], l[NQ];
  unsigned nan[NQ];     // bit g: a row that the column sees is NaN in columns 32 g .. of its values
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m[n] = -__builtin_inff(); l[n] = 0.f; nan[n] = 0;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][n][e] = 0.f;
    }
  }
  __device__ __forceinline__ void rescale(int n, float a) {
    l[n] *= a;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][n][e] *= a;
  }
  __device__ __forceinline__ void spoil() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const unsigned all = nan[n] | __shfl_xor(nan[n], 32);
      if (__ballot(all != 0))
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
          if (all >> d & 1)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][n][e] = __builtin_nanf("");
    }
  }
  // divides; l becomes the whole sum
  __device__ __forceinline__ void finish(int n, float c2) {
    l[n] += other_half(l[n]);
    const float r = l[n] == 0.f ? 0.f : 1.f / l[n];
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][n][e] *= r;
  }
  __device__ __forceinline__ float lse(int n, float c2) const {
    return l[n] == 0.f ? -__builtin_inff() : (log2f(l[n]) + m[n] * c2) * 0.6931471805599453f;
  }
  // wave 0 gets the sum over WK waves that held the same columns; buf: 64 x (D / 2 + 2) floats for each block of columns
  template <int WK>
  __device__ __forceinline__ void join(float* buf, int wave, int lane, float c2) {
    for (int w = 1; w < WK; ++w) {
      if (wave == w) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float* p = buf + n * 64 * (D / 2 + 2);
          p[lane] = m[n]; p[64 + lane] = l[n];
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) p[(2 + d * 16 + e) * 64 + lane] = o[d][n][e];
        }
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const float* p = buf + n * 64 * (D / 2 + 2);
          const float m2 = p[lane], mn = fmaxf(m[n], m2), safe = mn == -__builtin_inff() ? 0.f : mn;
          const float a = exp2f((m[n] - safe) * c2), b = exp2f((m2 - safe) * c2);
          m[n] = mn;
          l[n] = l[n] * a + p[64 + lane] * b;
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][n][e] = o[d][n][e] * a + p[(2 + d * 16 + e) * 64 + lane] * b;
        }
      }
      __syncthreads();
    }
  }
};

// rows that a column sees and whose values are NaN
template <int D, int KT, int NQ, int NB>
__device__ __forceinline__ void tile_marks(const Tile<D, KT>& tile, int wrow, int half, unsigned number, const f16v (&s)[NB][NQ],
                                           Soft<D, NQ>& st) {
  if (tile.mark[KT * (D / 32)] != number) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (s[kb][n][e] != -__builtin_inff())
          for (int g = 0; g < D / 32; ++g)
            if (tile.mark[(wrow + kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3)) * (D / 32) + g] == number) st.nan[n] |= 1u << g;
}

// one step of the running softmax: logits in, weights times values added to the state
template <int D, int KT, int NT, int NQ, int NB>
__device__ __forceinline__ void tile_accumulate(const Tile<D, KT>& tile, int wrow, int col, int half, float c2, f16v (&s)[NB][NQ],
                                                Soft<D, NQ>& st) {
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float mx = s[0][n][0];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][n][e]);
    mx = fmaxf(mx, other_half(mx));
    const float mn = fmaxf(st.m[n], mx);
    const float safe = mn == -__builtin_inff() ? 0.f : mn;
    // most tiles bring no new maximum once the first few have been seen
    if (__ballot(mn > st.m[n])) st.rescale(n, exp2f((st.m[n] - safe) * c2));
    st.m[n] = mn;
    const float nb = -safe * c2;
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[kb][n][e], c2, nb));
        s[kb][n][e] = w;
        sum += w;
      }
    st.l[n] += sum;
  }
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int k = 0; k < 2; ++k) {       // 16 rows
      bf8 p[NQ][NT];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = s[kb][n][8 * k + e];
        split_terms<NT>(y, p[n]);
      }
      const uint16_t* base = tile.v + col * Tile<D, KT>::VS + wrow + kb * 32 + k * 16 + half * 8;
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        const bf8 a = *(const bf8*)(base + d * 32 * Tile<D, KT>::VS);
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int t = 0; t < NT; ++t) st.o[d][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, p[n][t], st.o[d][n], 0, 0, 0);
      }
    }
}

// a lane's half of one column: 4 neighbouring dims at a time
template <int DT, int D, int NQ>
__device__ __forceinline__ void store_column(typename Row<DT>::T* __restrict__ out, int half, const f16v (&o)[D / 32][NQ], int n) {
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      typename Row<DT>::T* p = out + d * 32 + 8 * i + 4 * half;
      if constexpr (DT == GPSR_F32) {
        *(f4v*)p = f4v{o[d][n][4 * i], o[d][n][4 * i + 1], o[d][n][4 * i + 2], o[d][n][4 * i + 3]};
      } else {
        unsigned w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          w[j] = (unsigned)__builtin_bit_cast(uint16_t, from_f32<DT>(o[d][n][4 * i + 2 * j])) |
                 ((unsigned)__builtin_bit_cast(uint16_t, from_f32<DT>(o[d][n][4 * i + 2 * j + 1])) << 16);
        *(u2v*)p = u2v{w[0], w[1]};
      }
    }
}

// [D] sums, maximum raw logit, sum of weights
template <int D, int NQ>
__device__ __forceinline__ void store_partial(float* __restrict__ p, int half, Soft<D, NQ>& st, int n) {
  const float l = st.l[n] + other_half(st.l[n]);
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) p[d * 32 + 8 * i + 4 * half + j] = st.o[d][n][4 * i + j];
  if (half == 0) { p[D] = st.m[n]; p[D + 1] = l; }
}

// Joins the partial results of one column: one wave per column, lanes over the dim.  Column (t, g) of bank head bh has its n
// partials [D + 2] at bh * per_bh + t * per_t + g * per_g + i * per_i.
template <int DT, int D>
__global__ void __launch_bounds__(256)
k_bank_join(const float* __restrict__ part, int T, int G, int H, int64_t C, int n, size_t per_bh, size_t per_g, size_t per_t,
            size_t per_i, float c2, typename Row<DT>::T* __restrict__ out, float* __restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c >= C) return;
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t t = c / G;
  const int g = (int)(c - t * G), hq = h * G + g;
  const float* p = part + ((size_t)(b * H + h) * per_bh + t * per_t + g * per_g) * (D + 2);
  const size_t step = per_i * (D + 2);
  float m = -__builtin_inff();
  for (int i = lane; i < n; i += 64) if (p[i * step + D + 1] != 0.f) m = fmaxf(m, p[i * step + D]);
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float safe = m == -__builtin_inff() ? 0.f : m;
  constexpr int E = (D + 63) / 64;
  float acc[E] = {}, l = 0.f;
  for (int i = 0; i < n; ++i) {
    const float li = p[i * step + D + 1];
    if (li == 0.f) continue;             // saw nothing: its sums were not written
    const float w = exp2f((p[i * step + D] - safe) * c2);
    l = fmaf(w, li, l);
#pragma unroll
    for (int e = 0; e < E; ++e) if (e * 64 + lane < D) acc[e] = fmaf(w, p[i * step + e * 64 + lane], acc[e]);
  }
  typename Row<DT>::T* o = out + (((size_t)b * T + t) * (size_t)(H * G) + hq) * D;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e * 64 + lane < D) o[e * 64 + lane] = from_f32<DT>(l == 0.f ? 0.f : acc[e] / l);
  if (lse && lane == 0) lse[((size_t)b * (H * G) + hq) * T + t] = l == 0.f ? -__builtin_inff() : (log2f(l) + m * c2) * 0.6931471805599453f;
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
  if (!(scale > 0.f) || scale > 3.0e38f) return "bank_attend: scale must be positive and finite";
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
