// gpsr_bank_select.hip -- example bank: the best pages for each query (include/gpsr.h).
//
// The choice is defined by scores in 64 bits, but for many queries nearly all pages can be told apart with fewer:
//   prepare: each page's centroid as two bf16 terms (16 bits), its offset, and for 32 pages at a time bounds on the norms
//   screen:  scores a = q.c + offset on the matrix units, off by at most eps (below).  First pass: the pages are dealt to 128
//            groups (64 for n_sel <= 16) and each group keeps its largest a - eps; the n_sel-th largest of those, tau, is a
//            lower bound on the n_sel-th best exact score.  Second pass, the same products again: every page with a + eps >= tau
//            is a candidate.
//   pick:    where the screened scores of the n_sel-th and the next candidate differ by more than 2 eps, the choice is known;
//            otherwise exact scores of the candidates (or of all pages: few queries, few pages, or more candidates than
//            fit), sorted across a wave by (score, page).
// With Cauchy-Schwarz, and u = 2^-8 the half step of bf16: two terms of q and of c and their three larger products leave out
// at most 3 u^2 |q||c| (one exact term of q: u^2 |q||c|); the 32-bit sum of n products and the offset o adds (n + 2) 2^-23
// (|q||c| + |o|), n = 3 dim (2 dim); 1e-35 (1 + |q| + |c|) covers subnormal terms.  Norms above 1e18 are not screened: their pages
// are all candidates.  A page whose centroid is not a number is passed over, as one that does not exist: it is never chosen.
// 40 000 queries of 64 columns, 1563 pages, 16 of them: prepare 5, screen 104, pick 25 us, one after the other 125 us; one product
// at its rate in 32 bf16 terms 14; exact scores for all pages took 14 900 us.
#include "gpsr_bank_tile.hpp"

#define SE_MAX 64

struct SelectPlan { bool screen; int waves, J, blocks, slots; size_t off, bound, count, cand, bytes; };

// ---------------------------------------------------------------- prepare
// Row r of block k is page r * blocks + k: neighbouring pages, often alike, fall into different groups.  The terms lie as the
// matrix instructions take them, [16 columns][high, low][lane][8], so that a wave's load is one contiguous kilobyte (as rows,
// each load touched 32 cache lines, and the screen took 132 us instead of 94).  A workgroup has one block, 8 threads a page.
template <int D>
__global__ void __launch_bounds__(256)
k_bank_select_prepare(gpsr_bank bk, const int32_t* __restrict__ table, int J, int pshift, const int32_t* __restrict__ length, int G,
                      int blocks, __bf16* __restrict__ hl, float* __restrict__ off, f2v* __restrict__ bound) {
  __shared__ float wc[4], wo[4];
  const int k = blockIdx.x, h = blockIdx.y, b = blockIdx.z, H = bk.heads, tid = threadIdx.x, r = tid / 8, part = tid % 8;
  const int64_t lp = (int64_t)r * blocks + k;
  int64_t page = -1;
  if (lp < J && (lp << pshift) < length[b]) page = table[(size_t)b * J + lp];
  bool there = page >= 0 && page < bk.pages;
  __bf16* to = hl + ((size_t)(b * H + h) * blocks + k) * 32 * (2 * D) + r * 8;
  f4v y[D / 32];        // 4 columns at a time
  double sq = 0.0;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    y[i] = f4v{0, 0, 0, 0};
    if (there) y[i] = *(const f4v*)(bk.centroid + ((size_t)page * H + h) * D + (i * 8 + part) * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) sq = fma((double)y[i][j], (double)y[i][j], sq);
  }
  sq += __shfl_xor(sq, 1); sq += __shfl_xor(sq, 2); sq += __shfl_xor(sq, 4);
  there = there && sq == sq;      // a page that is not a number is never chosen: here as if it were not there
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int c = (i * 8 + part) * 4;
    bf2 hi[2], lo[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = there ? y[i][j] : 0.f;
      const __bf16 t = (__bf16)x;
      hi[j / 2][j % 2] = t; lo[j / 2][j % 2] = (__bf16)(x - (float)t);
    }
    const int at = (c / 16) * 1024 + (c / 8 % 2) * 256 + c % 8;
    *(u2v*)(to + at) = u2v{__builtin_bit_cast(unsigned, hi[0]), __builtin_bit_cast(unsigned, hi[1])};
    *(u2v*)(to + at + 512) = u2v{__builtin_bit_cast(unsigned, lo[0]), __builtin_bit_cast(unsigned, lo[1])};
  }
  const float o = bk.kernel_id == GPSR_KERNEL_RBF ? (float)(-0.5 * G * sq) : 0.f;
  // a norm that is too large makes the block's bound infinite
  float norm = !there ? 0.f : sq * (double)G < 1e36 ? (float)sqrt(sq) : __builtin_inff();
  float big = there && norm < __builtin_inff() ? fabsf(o) : 0.f;
  if (part == 0) off[((size_t)(b * H + h) * blocks + k) * 32 + r] = there && norm < __builtin_inff() ? o : -__builtin_inff();
  for (int d = 8; d < 64; d <<= 1) { norm = fmaxf(norm, __shfl_xor(norm, d)); big = fmaxf(big, __shfl_xor(big, d)); }
  if (tid % 64 == 0) { wc[tid / 64] = norm; wo[tid / 64] = big; }
  __syncthreads();
  if (tid == 0)
    bound[(size_t)(b * H + h) * blocks + k] = f2v{fmaxf(fmaxf(wc[0], wc[1]), fmaxf(wc[2], wc[3])), fmaxf(fmaxf(wo[0], wo[1]), fmaxf(wo[2], wo[3]))};
}

// ---------------------------------------------------------------- screen
// floats in the order of signed integers
__device__ __forceinline__ int ordered(float x) { const int i = __float_as_int(x); return i ^ ((i >> 31) & 0x7fffffff); }
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

// minimum over the wave, by moves between neighbouring lanes, rows of 16 and halves
__device__ __forceinline__ float wave_min(float x) {
#define STEP(ctrl) x = fminf(x, __int_as_float(__builtin_amdgcn_update_dpp(0x7f800000, __float_as_int(x), ctrl, 0xf, 0xf, false)))
  STEP(0x111); STEP(0x112); STEP(0x114); STEP(0x118);   // row_shr 1, 2, 4, 8
  STEP(0x142); STEP(0x143);                             // row_bcast 15, 31
#undef STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// the pages that a query skips altogether: [skipped.x, skipped.y)
__device__ __forceinline__ void skipped_pages(const int32_t* __restrict__ skip, int64_t at, int len, int pshift, int& lo, int& hi) {
  lo = hi = 0;
  if (!skip) return;
  const int a = max(skip[2 * at], 0), z = skip[2 * at + 1];
  if (z <= a) return;
  lo = (int)(((int64_t)a + (1 << pshift) - 1) >> pshift);
  hi = z >= len ? 0x7fffffff : z >> pshift;   // the last page ends with the bank
}

// A workgroup has 64 queries (32 of many columns) in blocks of 32, which every wave holds; its waves share out the blocks of
// pages and read them straight from L2 into operand registers, one block ahead, with no barrier between.  What bounds it is not
// the products (27 us of 72 for 1000 queries of 1563 pages in the first pass) but finding the hits of the second and waiting:
// three waves a SIMD 105 us, two 133, one 136 (40 000 queries; 1000 queries 72, 65, 68).
// NT: bf16 terms of the queries (1: bf16 rows taken singly, exact; 2: everything else).  SLOTS: groups of one lane in each wave
// (a column has 8 times as many); 8 halve the LDS where n_sel leaves them fine enough.
struct Candidate { int page; float a; };
// candidates that are kept for a query
static constexpr int screen_cap(int slots) { return slots * 8; }
// blocks of columns: as many as the queries' operands leave registers for
static constexpr int screen_nq(int d, int nt) { return nt * d <= 256 ? 2 : 1; }
template <int DT, int D, int NT, int SLOTS>
__global__ void __launch_bounds__(256, D * NT <= 64 ? 3 : D * NT <= 128 ? 2 : 1)
k_bank_select_screen(int H, const int32_t* __restrict__ length, int pshift, const typename Row<DT>::T* __restrict__ q, int T, int G,
                     Strides qs, bool qwide, int n_sel, const int32_t* __restrict__ skip, int J, int blocks,
                     const __bf16* __restrict__ hl, const float* __restrict__ off, const f2v* __restrict__ bound, int* __restrict__ count,
                     int32_t* __restrict__ cand, int32_t* __restrict__ sel) {
  constexpr int NQ = screen_nq(D, NT), CAP = screen_cap(SLOTS);
  __shared__ float best[4][SLOTS][NQ][64];    // each lane's own groups
  __shared__ float thr_of[NQ][32], eps_of[4][NQ][32];
  __shared__ Candidate list[32 * NQ][CAP];    // in LDS: a store to memory among the loads ahead would be waited for with them
  __shared__ int found[32 * NQ];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), half = lane >> 5, col = lane & 31;
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t t0 = (int64_t)blockIdx.x * (32 * NQ);
#pragma unroll
  for (int s = 0; s < SLOTS; ++s)
#pragma unroll
    for (int n = 0; n < NQ; ++n) best[wave][s][n][lane] = -__builtin_inff();

  // the heads that share the bank head, summed in 64 bits and rounded once
  bf8 qf[NQ][NT][D / 16];
  float qn[NQ], eps_most[NQ];
  int slo[NQ], shi[NQ];
  bool skips = false;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int64_t t = t0 + n * 32 + col;
    const bool there = t < T;
    qn[n] = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (there) {
        const typename Row<DT>::T* p = q + b * qs.b + t * qs.t + (int64_t)(h * G) * qs.h + s * 16 + half * 8;
        load8<DT>(p, qwide, y);
        if (G > 1) {
          double sum[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] = y[i];
          for (int g = 1; g < G; ++g) {
            float z[8];
            load8<DT>(p + g * qs.h, qwide, z);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += (double)z[i];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = (float)sum[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) qn[n] = fmaf(y[i], y[i], qn[n]);
      bf8 x[NT];
      split_terms<NT>(y, x);
#pragma unroll
      for (int i = 0; i < NT; ++i) qf[n][i][s] = x[i];
    }
    qn[n] += __shfl_xor(qn[n], 32);
    qn[n] = qn[n] < 1e36f ? 1.01f * sqrtf(qn[n]) : __builtin_inff();
    eps_most[n] = 0.f;
    skipped_pages(there ? skip : nullptr, (int64_t)b * T + t, length[b], pshift, slo[n], shi[n]);
    skips |= slo[n] < shi[n];
  }
  skips = __ballot(skips) != 0;

  const size_t base = (size_t)(b * H + h) * blocks;
  constexpr int ADDS = (NT + 1) * D + 2;
  const float k1 = (NT == 1 ? 1.05f : 3.1f) / 65536.f + ADDS / 8388608.f, k2 = (ADDS + 1) / 8388608.f;
  float thr[NQ];
  if (tid < 32 * NQ) found[tid] = 0;      // before the barriers between the passes
  bf8 hi[D / 16], lo[D / 16];
  f4v o4[4];
  const auto load = [&](int k) {       // behind the last block the last one again
    const __bf16* from = hl + (base + min(k, blocks - 1)) * 32 * (2 * D) + lane * 8;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) { hi[d] = *(const bf8*)(from + d * 1024); lo[d] = *(const bf8*)(from + d * 1024 + 512); }
#pragma unroll
    for (int i = 0; i < 4; ++i) o4[i] = *(const f4v*)(off + (base + min(k, blocks - 1)) * 32 + 8 * i + 4 * half);
  };
  for (int pass = 0; pass < 2; ++pass) {
    load(wave);
    for (int k = wave; k < blocks; k += 4) {
      const f2v nb = bound[base + k];
      f16v s[NQ], o;
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = o4[i / 4][i % 4];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi[d], qf[n][0][d], d ? s[n] : o, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo[d], qf[n][0][d], s[n], 0, 0, 0);
        if constexpr (NT > 1)
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi[d], qf[n][1][d], s[n], 0, 0, 0);
      }
      load(k + 4);
      if (skips) {
        asm volatile("");
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int lp = (8 * (e >> 2) + 4 * half + (e & 3)) * blocks + k;
            if (lp >= slo[n] && lp < shi[n]) s[n][e] = -__builtin_inff();
          }
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float eps = qn[n] * nb.x * k1 + nb.y * k2 + 1e-35f * (1.f + qn[n] + nb.x);
        const bool blind = !(eps < 1e37f);      // not screened: of no use as a bound, candidates all
        if (pass == 0) {
          float mx = s[n][0];
#pragma unroll
          for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[n][e]);
          float* p = &best[wave][(k >> 2) % SLOTS][n][lane];
          if (!blind) *p = fmaxf(*p, mx - eps);
          eps_most[n] = blind ? __builtin_inff() : fmaxf(eps_most[n], eps);
        } else {
          // which of the lane's 16 pages, then one of them for each lane at a time
          const float least = fmaxf(thr[n] - eps, -3.4e38f);
          unsigned hits = 0;
#pragma unroll
          for (int e = 0; e < 16; ++e) hits |= blind || s[n][e] >= least ? 1u << e : 0u;
          if (t0 + n * 32 + col >= T) hits = 0;
          while (__ballot(hits != 0)) {
            const int e = __builtin_ctz(hits | 0x10000u);
            const int lp = (8 * (e >> 2) + 4 * half + (e & 3)) * blocks + k;
            float a = 0.f;
#pragma unroll
            for (int x = 0; x < 16; ++x) a = x == e ? s[n][x] : a;
            if (hits && lp < J) {
              const int at = atomicAdd(&found[n * 32 + col], 1);
              if (at < CAP) list[n * 32 + col][at] = {lp, a};
            }
            hits &= hits - 1;
          }
        }
      }
    }
    if (pass == 0) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) if (half == 0) eps_of[wave][n][col] = eps_most[n];
      __syncthreads();
      // Wave w finds tau for block w of the columns, by bisection over the column's groups; a value a little below will do
      if (wave < NQ) {
      float v[4 * SLOTS], top = -__builtin_inff(), low = __builtin_inff(), tau = -__builtin_inff();
      int c = 0;
#pragma unroll
      for (int i = 0; i < 4 * SLOTS; ++i) {
        v[i] = best[i / SLOTS][i % SLOTS][wave][lane];
        top = fmaxf(top, v[i]);
        if (v[i] > -__builtin_inff()) { low = fminf(low, v[i]); ++c; }
      }
      c += __shfl_xor(c, 32);
      top = fmaxf(top, __shfl_xor(top, 32)); low = fminf(low, __shfl_xor(low, 32));
      int64_t a = ordered(low), z = (int64_t)ordered(top) + 1;      // at least n_sel groups are >= a, fewer >= z
      const bool enough = c >= n_sel;
      for (int i = 0; i < 20; ++i) {
        const int mid = (int)((a + z) >> 1);
        const float x = unordered(mid);
        c = 0;
#pragma unroll
        for (int s = 0; s < 4 * SLOTS; ++s) c += v[s] >= x;
        c += __shfl_xor(c, 32);
        if (c >= n_sel) a = mid; else z = mid;
      }
      if (enough) tau = unordered((int)a);
      if (half == 0) {
        thr_of[wave][col] = tau;
      }
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NQ; ++n) thr[n] = thr_of[n][col];
    }
  }
  __syncthreads();
  // Where the n_sel-th and the next best screened score are further apart than both can be off, the choice is made; count says
  // -2 for such a query, -1 for one with more candidates than were kept, and how many there are otherwise.
  for (int x = wave; x < 32 * NQ && t0 + x < T; x += 4) {
    const int64_t bth = ((int64_t)b * H + h) * T + t0 + x;
    const int n = __builtin_amdgcn_readfirstlane(found[x]), none = 0x7fffffff;
    const float eps = fmaxf(fmaxf(eps_of[0][x / 32][x % 32], eps_of[1][x / 32][x % 32]), fmaxf(eps_of[2][x / 32][x % 32], eps_of[3][x / 32][x % 32]));
    if (n <= 64 && eps < 1e37f) {
      const Candidate c = lane < n ? list[x][lane] : Candidate{none, -__builtin_inff()};
      // the few that are too many go one after the other, the smallest first
      unsigned long long chosen = n < 64 ? (1ull << n) - 1 : ~0ull;
      float most = -__builtin_inff();
      while (__popcll(chosen) > n_sel) {
        const bool in = chosen >> lane & 1;
        most = wave_min(in ? c.a : __builtin_inff());
        chosen &= ~__ballot(in && c.a == most);
      }
      const bool in = chosen >> lane & 1;
      if (n <= n_sel || (__popcll(chosen) == n_sel && wave_min(in ? c.a : __builtin_inff()) - most > 2.01f * eps)) {
        int32_t* const to = sel + (((size_t)b * T + t0 + x) * H + h) * n_sel;
        int place = 0;
        for (unsigned long long left = chosen; left; left &= left - 1) place += __builtin_amdgcn_readlane(c.page, __builtin_ctzll(left)) < c.page;
        if (in) to[place] = c.page;
        if (lane >= __popcll(chosen) && lane < n_sel) to[lane] = -1;
        if (lane == 0) count[bth] = -2;
        continue;
      }
    }
    if (lane == 0) count[bth] = n <= CAP ? n : -1;
    for (int i = lane; i < min(n, CAP); i += 64) cand[(size_t)bth * CAP + i] = list[x][i].page;
  }
}

// ---------------------------------------------------------------- pick
struct Scored { double s; int at; };      // at = INT_MAX: none
__device__ __forceinline__ bool before(const Scored& a, const Scored& b) { return a.s > b.s || (a.s == b.s && a.at < b.at); }
__device__ __forceinline__ Scored from_lane(const Scored& a, int x) { return {__shfl_xor(a.s, x), __shfl_xor(a.at, x)}; }

// lanes in the order of before(), or the other way round
// (N = 32: the first 32 lanes, where the others have none)
template <int N = 64>
__device__ __forceinline__ void sort64(Scored& a, int lane, bool best_first) {
#pragma unroll
  for (int k = 2; k <= N; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j; j >>= 1) {
      const Scored o = from_lane(a, j);
      const bool up = ((lane & k) == 0) == best_first, first = (lane & j) == 0;   // this pair's better one goes to its first lane
      if (before(o, a) == (up == first)) a = o;
    }
}
// best: 64 in order; add: 64 in the opposite order -> the best 64 of both, in order
__device__ __forceinline__ void merge64(Scored& best, const Scored& add, int lane) {
  if (before(add, best)) best = add;
#pragma unroll
  for (int j = 32; j; j >>= 1) {
    const Scored o = from_lane(best, j);
    if (before(o, best) == ((lane & j) == 0)) best = o;
  }
}

// W waves per query: 1 (four queries a workgroup; candidates from the screen, or all pages) or 16 (one query, all pages)
template <int DT, int W>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W)
k_bank_select_pick(gpsr_bank bk, const int32_t* __restrict__ table, int J, int pshift, const int32_t* __restrict__ length,
                   const typename Row<DT>::T* __restrict__ q, int T, int G, Strides qs, int n_sel, const int32_t* __restrict__ skip,
                   int cap, const int* __restrict__ count, const int32_t* __restrict__ cand, int32_t* __restrict__ sel) {
  constexpr int Q = W == 1 ? 4 : 1;
  __shared__ double qv[Q][256];
  __shared__ double ms[W == 1 ? 1 : W][64];
  __shared__ int ma[W == 1 ? 1 : W][64];
  const int D = bk.dim, H = bk.heads, tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid);
  const int slot = W == 1 ? wave : 0, h = blockIdx.y, b = blockIdx.z;
  const int64_t t = (int64_t)blockIdx.x * Q + slot;
  if (t >= T) return;              // W == 1: a whole wave, and no barrier follows; W > 1: never
  const int none = 0x7fffffff;
  const double worst = -__builtin_inf();
  const int64_t len = length[b], bth = ((int64_t)b * H + h) * T + t;
  const int64_t pages = len <= 0 ? 0 : (len + (1 << pshift) - 1) >> pshift;
  const int n_all = (int)(pages < J ? pages : J);
  int32_t* const to = sel + (((size_t)b * T + t) * H + h) * n_sel;
  int n = n_all;
  const int32_t* mine = nullptr;
  if (W == 1 && count) {
    const int c = count[bth];
    if (c == -2) return;
    if (c >= 0) { n = c; mine = cand + (size_t)bth * cap; }
  }
  for (int i = W == 1 ? lane : tid; i < D; i += W == 1 ? 64 : 64 * W) {
    double s = 0.0;
    for (int g = 0; g < G; ++g) s += (double)to_f32<DT>(q[b * qs.b + t * qs.t + (int64_t)(h * G + g) * qs.h + i]);
    qv[slot][i] = s;
  }
  if (W > 1) __syncthreads();
  int slo, shi;
  skipped_pages(skip, (int64_t)b * T + t, length[b], pshift, slo, shi);
  const bool rbf = bk.kernel_id == GPSR_KERNEL_RBF;
  Scored best = {worst, none};
  bool empty = true;
  const int part = lane & 3;
  for (int64_t i0 = (int64_t)(W == 1 ? 0 : wave) * 64; i0 < n; i0 += W == 1 ? 64 : 64 * W) {
    Scored x = {worst, none};
    // four lanes a page, 16 pages at a time; page i0 + i ends up in lane i
    int lp[4];
    const f4v* c[4];
    bool ok[4];
    const auto look_up = [&](int sub) {
      const int64_t i = i0 + sub * 16 + (lane >> 2);
      lp[sub] = i < n ? mine ? mine[i] : (int)i : none;
      const int64_t page = lp[sub] < n_all ? table[(size_t)b * J + lp[sub]] : -1;
      ok[sub] = page >= 0 && page < bk.pages && !(lp[sub] >= slo && lp[sub] < shi);
      c[sub] = (const f4v*)(bk.centroid + ((size_t)(ok[sub] ? page : 0) * H + h) * D);
    };
    const auto place = [&](int sub, double s, double sq) {
      if (rbf) s -= 0.5 * G * sq;
      s += __shfl_xor(s, 1); s += __shfl_xor(s, 2);
      Scored y = {worst, none};
      if (ok[sub] && s == s) y = {s, lp[sub]};
      y.s = __shfl(y.s, (lane & 15) * 4); y.at = __shfl(y.at, (lane & 15) * 4);
      if ((lane >> 4) == sub) x = y;
    };
    if constexpr (W > 1) {         // few waves on the chip: the look-ups of all 64 pages wait together, and 32 columns of them
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) look_up(sub);
      double dot[4] = {0, 0, 0, 0}, sq[4] = {0, 0, 0, 0};
#pragma unroll 2
      for (int g = 0; g < D / 32; ++g) {
        f4v y[4][2];
#pragma unroll
        for (int sub = 0; sub < 4; ++sub)
#pragma unroll
          for (int d = 0; d < 2; ++d) y[sub][d] = c[sub][8 * g + 4 * d + part];
#pragma unroll
        for (int sub = 0; sub < 4; ++sub)
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const double z = (double)y[sub][d][j];
              dot[sub] = fma(qv[slot][32 * g + 16 * d + 4 * part + j], z, dot[sub]);
              if (rbf) sq[sub] = fma(z, z, sq[sub]);
            }
      }
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) place(sub, dot[sub], sq[sub]);
    } else {                       // some 20 candidates: no work for pages that are not there
#pragma unroll
      for (int sub = 0; sub < 4; ++sub)
        if (i0 + sub * 16 < n) {
          look_up(sub);
          double dot[4] = {0, 0, 0, 0}, sq[4] = {0, 0, 0, 0};
          for (int g = 0; g < D / 32; ++g) {
            f4v y[2];
#pragma unroll
            for (int d = 0; d < 2; ++d) y[d] = c[sub][8 * g + 4 * d + part];
#pragma unroll
            for (int d = 0; d < 2; ++d)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const double z = (double)y[d][j];
                dot[j] = fma(qv[slot][32 * g + 16 * d + 4 * part + j], z, dot[j]);
                if (rbf) sq[j] = fma(z, z, sq[j]);
              }
          }
          place(sub, (dot[0] + dot[1]) + (dot[2] + dot[3]), (sq[0] + sq[1]) + (sq[2] + sq[3]));
        }
    }
    if (empty && n <= 32) { sort64<32>(x, lane, true); best = x; break; }
    if (empty) { sort64(x, lane, true); best = x; empty = false; continue; }
    const Scored last = {__shfl(best.s, n_sel - 1), __shfl(best.at, n_sel - 1)};
    if (!__ballot(before(x, last))) continue;
    sort64(x, lane, false);
    merge64(best, x, lane);
  }
  if constexpr (W > 1) {
    for (int step = 1; step < W; step <<= 1) {
      if ((wave & (2 * step - 1)) == step) { ms[wave][lane] = best.s; ma[wave][lane] = best.at; }
      __syncthreads();
      if ((wave & (2 * step - 1)) == 0) {
        const Scored o = {ms[wave + step][63 - lane], ma[wave + step][63 - lane]};
        merge64(best, o, lane);
      }
    }
    if (wave) return;
  }
  if (lane >= n_sel) best.at = none;
  int rank = 0;
  for (int i = 0; i < n_sel; ++i) { const int o = __shfl(best.at, i); rank += o < best.at || (o == best.at && i < lane); }
  if (lane < n_sel) to[rank] = best.at == none ? -1 : best.at;
}

// ---------------------------------------------------------------- host
static SelectPlan plan_of(const gpsr_bank* bk, int B, int table_pages, int T, int n_sel) {
  SelectPlan p = {};
  const int64_t queries = (int64_t)B * T * bk->heads;
  p.J = table_pages;
  // Exact scores for all pages take a round for each 256 queries, of 9 us and 0.8 for each 10 000 of pages x columns; the screen 55
  // and 1.2, however many they are up to some thousands (measured: 1563 pages of 64 columns 22 us a round and 82, 100 pages 9 and
  // 44, 1906 of 128 columns 30 and 95, 6000 of 256 columns 110 and 229).
  const double work = (double)table_pages * bk->dim / 10000;
  p.screen = table_pages > 64 && (double)((queries + 255) / 256) * (9 + 0.8 * work) > 55 + 1.2 * work;
  p.waves = !p.screen && table_pages > 64 ? 16 : 1;
  if (p.screen) {
    p.blocks = (table_pages + 31) / 32;
    p.slots = n_sel <= 16 ? 8 : 16;
    const size_t rows = (size_t)B * bk->heads * p.blocks * 32;
    size_t at = align256(rows * 2 * bk->dim * 2);
    p.off = at; at += align256(rows * 4);
    p.bound = at; at += align256(rows / 32 * 8);
    p.count = at; at += align256((size_t)queries * 4);
    p.cand = at; at += align256((size_t)queries * screen_cap(p.slots) * 4);
    p.bytes = at;
  }
  return p;
}

extern "C" size_t gpsr_bank_select_workspace_bytes(const gpsr_bank* bank, int B, int table_pages, int T, int q_heads, int n_sel, int dtype) {
  if (bank_wrong(bank) || B <= 0 || T <= 0 || table_pages < 0 || q_heads < 1 || q_heads % bank->heads || n_sel < 1 || n_sel > SE_MAX || !type_ok(dtype)) return 0;
  return plan_of(bank, B, table_pages, T, n_sel).bytes;
}

template <int DT, int D>
static void launch_select(const SelectPlan& p, const gpsr_bank& bk, const int32_t* table, int B, const int32_t* length, const void* q,
                          int T, int G, Strides qs, bool qwide, int n_sel, const int32_t* skip, int32_t* sel, char* ws, hipStream_t st) {
  typedef typename Row<DT>::T E;
  const int pshift = __builtin_ctz((unsigned)bk.page_rows), H = bk.heads;
  int *count = nullptr, *cand = nullptr;
  if (p.screen) {
    __bf16* hl = (__bf16*)ws;
    float* off = (float*)(ws + p.off);
    f2v* bound = (f2v*)(ws + p.bound);
    count = (int*)(ws + p.count); cand = (int*)(ws + p.cand);
    hipLaunchKernelGGL((k_bank_select_prepare<D>), dim3((unsigned)p.blocks, (unsigned)H, (unsigned)B), dim3(256), 0, st, bk, table, p.J,
                       pshift, length, G, p.blocks, hl, off, bound);
#define SCREEN(NT) if (p.slots == 8) SCREEN_(NT, 8); else SCREEN_(NT, 16)
#define SCREEN_(NT, SLOTS) hipLaunchKernelGGL((k_bank_select_screen<DT, D, NT, SLOTS>), \
    dim3((unsigned)(((int64_t)T + 32 * screen_nq(D, NT) - 1) / (32 * screen_nq(D, NT))), (unsigned)H, (unsigned)B), dim3(256), 0, st, H, length, pshift, (const E*)q, T, G, qs, \
    qwide, n_sel, skip, p.J, p.blocks, hl, off, bound, count, cand, sel)
    if constexpr (DT == GPSR_BF16) { if (G == 1) { SCREEN(1); } else { SCREEN(2); } } else { SCREEN(2); }
#undef SCREEN
#undef SCREEN_
  }
#define PICK(W, Q) hipLaunchKernelGGL((k_bank_select_pick<DT, W>), dim3((unsigned)(((int64_t)T + Q - 1) / Q), (unsigned)H, (unsigned)B), \
    dim3(W == 1 ? 256 : 64 * W), 0, st, bk, table, p.J, pshift, length, (const E*)q, T, G, qs, n_sel, skip, screen_cap(p.slots), count, cand, sel)
  if (p.waves == 1) PICK(1, 4); else PICK(16, 1);
#undef PICK
}

extern "C" int gpsr_bank_select(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* length,
                                const void* q, int dtype, int T, int q_heads, const int64_t* qst, int n_sel, const int32_t* skip,
                                int32_t* sel, void* workspace, size_t workspace_bytes, void* stream) {
  if (B <= 0 || T <= 0) return 0;
  if (const char* w = bank_wrong(bank)) return arg_fail(w);
  if ((!table && table_pages) || !length || !q || !qst || !sel) return arg_fail("bank_select: null pointer");
  if (!type_ok(dtype)) return arg_fail("bank_select: dtype");
  if (B > 65535) return arg_fail("bank_select: more than 65535 entries");
  if (table_pages > 0x7fffff00) return arg_fail("bank_select: table_pages");
  if (table_pages < 0) return arg_fail("bank_select: table_pages");
  if (q_heads < 1 || q_heads > 65535 || q_heads % bank->heads) return arg_fail("bank_select: query heads must be a multiple of the bank's heads, up to 65535");
  if (n_sel < 1 || n_sel > SE_MAX) return arg_fail("bank_select: n_sel must be in 1..64");
  if (!grid_fits(((int64_t)T + 3) / 4, 256)) return arg_fail("bank_select: too many queries for one call");
  const SelectPlan p = plan_of(bank, B, table_pages, T, n_sel);
  if (workspace_bytes < p.bytes || (p.bytes && !workspace)) return arg_fail("workspace too small");
  if (p.bytes && ((uintptr_t)workspace & 15)) return arg_fail("bank_select: workspace must be 16-byte aligned");
  const Strides qs = {qst[0], qst[1], qst[2]};
  const bool wide = rows_wide(q, qst, dtype);
  const int G = q_heads / bank->heads;
  hipStream_t st = (hipStream_t)stream;
#define SELECT(DT, BITS, D) launch_select<DT, D>(p, *bank, table, B, length, q, T, G, qs, wide, n_sel, skip, sel, (char*)workspace, st)
  if (dtype == GPSR_BF16) BANK_DISPATCH_D(SELECT, GPSR_BF16, 4, bank->dim)
  else if (dtype == GPSR_F16) BANK_DISPATCH_D(SELECT, GPSR_F16, 4, bank->dim)
  else BANK_DISPATCH_D(SELECT, GPSR_F32, 4, bank->dim)
#undef SELECT
  CHECK_LAUNCH("k_bank_select");
  return 0;
}
