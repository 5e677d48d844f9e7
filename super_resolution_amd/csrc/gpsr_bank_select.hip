// gpsr_bank_select.hip -- example bank: the best pages for each query (include/gpsr.h).
//
// The choice is defined by scores in 64 bits, but for many queries nearly all pages can be told apart with fewer:
//   prepare: each page's centroid as two bf16 terms (16 bits), its offset, and for 32 pages at a time bounds on the norms
//   screen:  scores a = q.c + offset on the matrix units, off by at most eps (below).  First pass: the pages are dealt to 128
//            groups and each group keeps its largest a - eps; the n_sel-th largest of those, tau, is a lower bound on the
//            n_sel-th best exact score.  Second pass, the same products again: every page with a + eps >= tau is a candidate.
//   pick:    exact scores of the candidates (or of all pages: few queries, few pages, or more candidates than fit), sorted
//            across a wave by (score, page).
// With Cauchy-Schwarz, and u = 2^-8 the half step of bf16: two terms of q and of c and their three larger products leave out
// at most 3 u^2 |q||c|; the 32-bit sum of 3 dim products and the offset o adds (3 dim + 2) 2^-23 (|q||c| + |o|); 1e-35 (1 +
// |q| + |c|) covers subnormal terms.  Norms above 1e18 or not finite are not screened: their pages are all candidates.
#include "gpsr_bank_tile.hpp"

#define SE_MAX 64
#define SE_SLOTS 64

struct SelectPlan { bool screen; int waves, J, blocks, cap; size_t hl, off, bound, count, cand, bytes; };

// ---------------------------------------------------------------- prepare
// Row r of block k is page r * blocks + k: neighbouring pages, often alike, fall into different groups.  A workgroup has one
// block, 8 threads a page.
template <int D>
__global__ void __launch_bounds__(256)
k_bank_select_prepare(gpsr_bank bk, const int32_t* __restrict__ table, int J, int pshift, const int32_t* __restrict__ length, int G,
                      int blocks, __bf16* __restrict__ hl, float* __restrict__ off, f2v* __restrict__ bound) {
  __shared__ float wc[4], wo[4];
  const int k = blockIdx.x, h = blockIdx.y, b = blockIdx.z, H = bk.heads, tid = threadIdx.x, r = tid / 8, part = tid % 8;
  const int64_t lp = (int64_t)r * blocks + k;
  int64_t page = -1;
  if (lp < J && (lp << pshift) < length[b]) page = table[(size_t)b * J + lp];
  const bool there = page >= 0 && page < bk.pages;
  __bf16* row = hl + (((size_t)(b * H + h) * blocks + k) * 32 + r) * (2 * D);
  double sq = 0.0;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {    // 4 columns at a time
    const int c = (i * 8 + part) * 4;
    f4v y = {0, 0, 0, 0};
    if (there) y = *(const f4v*)(bk.centroid + ((size_t)page * H + h) * D + c);
    bf2 hi[2], lo[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __bf16 t = (__bf16)y[j];
      hi[j / 2][j % 2] = t; lo[j / 2][j % 2] = (__bf16)(y[j] - (float)t);
      sq = fma((double)y[j], (double)y[j], sq);
    }
    *(u2v*)(row + c) = u2v{__builtin_bit_cast(unsigned, hi[0]), __builtin_bit_cast(unsigned, hi[1])};
    *(u2v*)(row + D + c) = u2v{__builtin_bit_cast(unsigned, lo[0]), __builtin_bit_cast(unsigned, lo[1])};
  }
  sq += __shfl_xor(sq, 1); sq += __shfl_xor(sq, 2); sq += __shfl_xor(sq, 4);
  const float o = bk.kernel_id == GPSR_KERNEL_RBF ? (float)(-0.5 * G * sq) : 0.f;
  // a norm that is too large (or NaN) makes the block's bound infinite
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

// the pages that a query skips altogether: [skipped.x, skipped.y)
__device__ __forceinline__ void skipped_pages(const int32_t* __restrict__ skip, int64_t at, int64_t len, int pshift, int64_t& lo, int64_t& hi) {
  lo = hi = 0;
  if (!skip) return;
  const int64_t P = (int64_t)1 << pshift, a = skip[2 * at] > 0 ? skip[2 * at] : 0, z = skip[2 * at + 1];
  if (z <= a) return;
  lo = (a + P - 1) >> pshift;
  hi = z >= len ? (int64_t)1 << 40 : z >> pshift;   // the last page ends with the bank
}

// NT: bf16 terms of the queries (1: bf16 rows taken singly, exact; 2: everything else)
template <int DT, int D, int NT>
__global__ void __launch_bounds__(256)
k_bank_select_screen(int H, const int32_t* __restrict__ length, int pshift, const typename Row<DT>::T* __restrict__ q, int T, int G,
                     Strides qs, bool qwide, int n_sel, const int32_t* __restrict__ skip, int J, int blocks,
                     const __bf16* __restrict__ hl, const float* __restrict__ off, const f2v* __restrict__ bound, int cap,
                     int* __restrict__ count, int* __restrict__ cand) {
  constexpr int KS = 2 * D + 8;
  __shared__ __attribute__((aligned(16))) __bf16 tile[32 * KS];
  __shared__ __attribute__((aligned(16))) float toff[32];
  __shared__ float best[SE_SLOTS][256];    // [slot][thread]: each lane's own groups
  __shared__ int found[128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t t = (int64_t)blockIdx.x * 128 + wave * 32 + col;
  const bool there = t < T;
  if (tid < 128) found[tid] = 0;
  for (int s = 0; s < SE_SLOTS; ++s) best[s][tid] = -__builtin_inff();

  // the group's heads, summed in 64 bits and rounded once
  bf8 qf[NT][D / 16];
  float qn = 0.f;
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
    for (int i = 0; i < 8; ++i) qn = fmaf(y[i], y[i], qn);
    bf8 x[NT];
    split_terms<NT>(y, x);
#pragma unroll
    for (int n = 0; n < NT; ++n) qf[n][s] = x[n];
  }
  qn += __shfl_xor(qn, 32);
  qn = qn < 1e36f ? 1.01f * sqrtf(qn) : __builtin_inff();
  int64_t slo, shi;
  skipped_pages(there ? skip : nullptr, (int64_t)b * T + t, length[b], pshift, slo, shi);
  const bool skips = __ballot(slo < shi) != 0;

  const size_t base = (size_t)(b * H + h) * blocks;
  const float k1 = 3.1f / 65536.f + (3 * D + 2) / 8388608.f, k2 = (3 * D + 3) / 8388608.f;
  float thr = 0.f;
  u4v next[D / 32];     // a block is 32 rows of 2 D bf16: D / 32 loads of 16 bytes for each thread
  float noff = 0.f;
  const auto load = [&](int k) {
    const u4v* src = (const u4v*)(hl + (base + k) * 32 * (2 * D));
#pragma unroll
    for (int i = 0; i < D / 32; ++i) next[i] = src[tid + 256 * i];
    if (tid < 32) noff = off[(base + k) * 32 + tid];
  };
  for (int pass = 0; pass < 2; ++pass) {
    load(0);
    for (int k = 0; k < blocks; ++k) {
      const f2v nb = bound[base + k];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int u = tid + 256 * i;
        *(u4v*)(tile + u / (D / 4) * KS + u % (D / 4) * 8) = next[i];
      }
      if (tid < 32) toff[tid] = noff;
      __syncthreads();
      if (k + 1 < blocks) load(k + 1);
      f16v s;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4v a = *(const f4v*)(toff + 8 * i + 4 * half);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * i + j] = a[j];
      }
      const __bf16* row = tile + col * KS + half * 8;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const bf8 hi = *(const bf8*)(row + d * 16), lo = *(const bf8*)(row + D + d * 16);
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, qf[0][d], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo, qf[0][d], s, 0, 0, 0);
        if constexpr (NT > 1) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, qf[1][d], s, 0, 0, 0);
      }
      const float eps = qn * nb.x * k1 + nb.y * k2 + 1e-35f * (1.f + qn + nb.x);
      const bool blind = !(eps < 1e37f);      // not screened: of no use as a bound, candidates all
      if (skips) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int64_t lp = (int64_t)(8 * (e >> 2) + 4 * half + (e & 3)) * blocks + k;
          if (lp >= slo && lp < shi) s[e] = -__builtin_inff();
        }
      }
      float mx = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
      if (pass == 0) {
        if (!blind) { float* p = &best[k % SE_SLOTS][tid]; *p = fmaxf(*p, mx - eps); }
      } else if (there && (blind || mx >= thr - eps)) {
        int* mine = cand + (((size_t)(b * H + h) * T) + t) * cap;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int64_t lp = (int64_t)(8 * (e >> 2) + 4 * half + (e & 3)) * blocks + k;
          if (lp < J && (blind || (s[e] > -__builtin_inff() && s[e] >= thr - eps))) {
            const int at = atomicAdd(&found[wave * 32 + col], 1);
            if (at < cap) mine[at] = (int)lp;
          }
        }
      }
    }
    if (pass == 0) {
      // tau by bisection over the lane's groups and those of its other half; a value a little below will do
      float v[SE_SLOTS], top = -__builtin_inff(), low = __builtin_inff();
      int n = 0;
#pragma unroll
      for (int s = 0; s < SE_SLOTS; ++s) {
        v[s] = best[s][tid];
        top = fmaxf(top, v[s]);
        if (v[s] > -__builtin_inff()) { low = fminf(low, v[s]); ++n; }
      }
      n += __shfl_xor(n, 32);
      top = fmaxf(top, other_half(top)); low = fminf(low, other_half(low));
      thr = -__builtin_inff();
      if (n >= n_sel) {
        int64_t a = ordered(low), z = (int64_t)ordered(top) + 1;      // at least n_sel groups are >= a, fewer >= z
        for (int i = 0; i < 20 && z - a > 1; ++i) {
          const int mid = (int)((a + z) >> 1);
          const float x = unordered(mid);
          int c = 0;
#pragma unroll
          for (int s = 0; s < SE_SLOTS; ++s) c += v[s] >= x;
          c += __shfl_xor(c, 32);
          if (c >= n_sel) a = mid; else z = mid;
        }
        thr = unordered((int)a);
      }
    }
  }
  __syncthreads();
  if (there && half == 0) count[((size_t)(b * H + h) * T) + t] = found[wave * 32 + col];
}

// ---------------------------------------------------------------- pick
struct Scored { double s; int at; };      // at = INT_MAX: none
__device__ __forceinline__ bool before(const Scored& a, const Scored& b) { return a.s > b.s || (a.s == b.s && a.at < b.at); }
__device__ __forceinline__ Scored from_lane(const Scored& a, int x) { return {__shfl_xor(a.s, x), __shfl_xor(a.at, x)}; }

// lanes in the order of before(), or the other way round
__device__ __forceinline__ void sort64(Scored& a, int lane, bool best_first) {
#pragma unroll
  for (int k = 2; k <= 64; k <<= 1)
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
                   int cap, const int* __restrict__ count, const int* __restrict__ cand, int32_t* __restrict__ sel) {
  constexpr int Q = W == 1 ? 4 : 1;
  __shared__ double qv[Q][256];
  __shared__ double ms[W == 1 ? 1 : W][64];
  __shared__ int ma[W == 1 ? 1 : W][64];
  const int D = bk.dim, H = bk.heads, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slot = W == 1 ? wave : 0, h = blockIdx.y, b = blockIdx.z;
  const int64_t t = (int64_t)blockIdx.x * Q + slot;
  const bool there = t < T;
  if (there)
    for (int i = W == 1 ? lane : tid; i < D; i += W == 1 ? 64 : 64 * W) {
      double s = 0.0;
      for (int g = 0; g < G; ++g) s += (double)to_f32<DT>(q[b * qs.b + t * qs.t + (int64_t)(h * G + g) * qs.h + i]);
      qv[slot][i] = s;
    }
  __syncthreads();
  if (!there) return;              // W == 1: a whole wave, and no barrier follows
  const int none = 0x7fffffff;
  const double worst = -__builtin_inf();
  const int64_t len = length[b], bth = ((int64_t)b * H + h) * T + t;
  const int64_t pages = len <= 0 ? 0 : (len + (1 << pshift) - 1) >> pshift;
  const int n_all = (int)(pages < J ? pages : J);
  int n = n_all;
  const int* mine = nullptr;
  if (count && count[bth] <= cap) { n = count[bth]; mine = cand + (size_t)bth * cap; }
  int64_t slo, shi;
  skipped_pages(skip, (int64_t)b * T + t, len, pshift, slo, shi);
  const bool rbf = bk.kernel_id == GPSR_KERNEL_RBF;
  Scored best = {worst, none};
  bool empty = true;
  for (int64_t i0 = (int64_t)(W == 1 ? 0 : wave) * 64; i0 < n; i0 += W == 1 ? 64 : 64 * W) {
    Scored x = {worst, none};
    const int64_t i = i0 + lane;
    if (i < n) {
      const int lp = mine ? mine[i] : (int)i;
      const int64_t page = lp < n_all ? table[(size_t)b * J + lp] : -1;
      if (page >= 0 && page < bk.pages && !(lp >= slo && lp < shi)) {
        const f4v* c = (const f4v*)(bk.centroid + ((size_t)page * H + h) * D);
        // 32 columns on their way at a time, four chains of sums
        double dot[4] = {0, 0, 0, 0}, sq[4] = {0, 0, 0, 0};
        for (int g = 0; g < D / 32; ++g) {
          f4v y[8];
#pragma unroll
          for (int d = 0; d < 8; ++d) y[d] = c[8 * g + d];
#pragma unroll
          for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const double z = (double)y[d][j];
              dot[j] = fma(qv[slot][32 * g + 4 * d + j], z, dot[j]);
              if (rbf) sq[j] = fma(z, z, sq[j]);
            }
        }
        const double all = (dot[0] + dot[1]) + (dot[2] + dot[3]);
        const double s = rbf ? all - 0.5 * G * ((sq[0] + sq[1]) + (sq[2] + sq[3])) : all;
        if (s == s) x = {s, lp};
      }
    }
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
  if (lane < n_sel) sel[(((size_t)b * T + t) * H + h) * n_sel + rank] = best.at == none ? -1 : best.at;
}

// ---------------------------------------------------------------- host
static SelectPlan plan_of(const gpsr_bank* bk, int B, int table_pages, int T, int n_sel) {
  SelectPlan p = {};
  const int64_t queries = (int64_t)B * T * bk->heads;
  p.J = table_pages;
  p.screen = table_pages > 64 && queries >= 512;
  p.waves = !p.screen && table_pages > 64 ? 16 : 1;
  if (p.screen) {
    p.blocks = (table_pages + 31) / 32;
    p.cap = 2 * n_sel + 64;
    const size_t rows = (size_t)B * bk->heads * p.blocks * 32;
    size_t at = align256(rows * 2 * bk->dim * 2);
    p.off = at; at += align256(rows * 4);
    p.bound = at; at += align256(rows / 32 * 8);
    p.count = at; at += align256((size_t)queries * 4);
    p.cand = at; at += align256((size_t)queries * p.cap * 4);
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
  const int *count = nullptr, *cand = nullptr;
  if (p.screen) {
    __bf16* hl = (__bf16*)ws;
    float* off = (float*)(ws + p.off);
    f2v* bound = (f2v*)(ws + p.bound);
    count = (const int*)(ws + p.count); cand = (const int*)(ws + p.cand);
    hipLaunchKernelGGL((k_bank_select_prepare<D>), dim3((unsigned)p.blocks, (unsigned)H, (unsigned)B), dim3(256), 0, st, bk, table, p.J,
                       pshift, length, G, p.blocks, hl, off, bound);
    const dim3 grid((unsigned)(((int64_t)T + 127) / 128), (unsigned)H, (unsigned)B);
#define SCREEN(NT) hipLaunchKernelGGL((k_bank_select_screen<DT, D, NT>), grid, dim3(256), 0, st, H, length, pshift, (const E*)q, T, G, qs, \
    qwide, n_sel, skip, p.J, p.blocks, hl, off, bound, p.cap, (int*)count, (int*)cand)
    if constexpr (DT == GPSR_BF16) { if (G == 1) SCREEN(1); else SCREEN(2); } else SCREEN(2);
#undef SCREEN
  }
#define PICK(W, Q) hipLaunchKernelGGL((k_bank_select_pick<DT, W>), dim3((unsigned)(((int64_t)T + Q - 1) / Q), (unsigned)H, (unsigned)B), \
    dim3(W == 1 ? 256 : 64 * W), 0, st, bk, table, p.J, pshift, length, (const E*)q, T, G, qs, n_sel, skip, p.cap, count, cand, sel)
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
  if (table_pages < 0) return arg_fail("bank_select: table_pages");
  if (q_heads < 1 || q_heads > 65535 || q_heads % bank->heads) return arg_fail("bank_select: query heads must be a multiple of the bank's heads, up to 65535");
  if (n_sel < 1 || n_sel > SE_MAX) return arg_fail("bank_select: n_sel must be in 1..64");
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
