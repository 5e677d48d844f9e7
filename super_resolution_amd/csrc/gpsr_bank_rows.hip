// gpsr_bank_rows.hip -- example bank: rounding rows as they are written, and reading them back (include/gpsr.h).
#include "gpsr_bank.hpp"

// ---------------------------------------------------------------- write
// One workgroup per page that the call touches: it alone rounds the page's new rows, stores them, and recomputes the
// page's centroid from all rows up to the last one, earlier ones included, so nothing is summed through atomics and a page
// gives the same bits however its rows arrived.  A thread owns 8 columns of a row (one 16- or 32-byte load, one code
// store); the 4 threads of a 32-column group share its maximum through DPP moves.
// Bound by memory: 2^20 rows of 64 bf16 columns to 4 bits 70 us, 4.9 TB/s of rows and codes.
//   scale: amax = m 2^x with m in [.5, 1); the smallest e with amax <= 6 * 2^e (E2M1) is x - 3 for m <= .75, x - 2 above
//   (E4M3: 448 = .875 * 2^9).  Dividing by 2^e is exact, so the only rounding is the conversion's own.
//   centroid and offset sums run in 64 bits, where sums of held values (<= 4 significant bits each) are exact for any
//   scales within 2^40 of each other: the order of the rows does not matter.
#define WR_THREADS 256

template <int BITS>
__device__ __forceinline__ unsigned scale_byte(float amax) {   // amax finite
  const unsigned u = __float_as_uint(amax);
  // exponent x and fraction of a normal amax; subnormal ones (x < -125) fall under the lower clamp anyway
  const int x = (int)(u >> 23) - 126;
  const unsigned frac = u & 0x7fffff;   // m = (1 + frac / 2^23) / 2
  int e = BITS == 4 ? x - 3 + (frac > 0x400000u) : x - 9 + (frac > 0x600000u);
  e = e < -110 ? -110 : e;
  const int top = BITS == 4 ? 125 : 119;
  return (unsigned)((e > top ? top : e) + 127);
}

template <int BITS>
__device__ __forceinline__ void encode8(const float* x, float s, unsigned& w0, unsigned& w1) {
  const float lim = (BITS == 4 ? 6.f : 448.f) * s;   // only a clamped scale can clip
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i], -lim, lim);
  if (BITS == 4) {
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], s, 0);
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w0, y[2], y[3], s, 1);
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w0, y[4], y[5], s, 2);
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w0, y[6], y[7], s, 3);
    w1 = 0;
  } else {
    s2v a = {0, 0}, b = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, y[0], y[1], s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, y[2], y[3], s, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, y[4], y[5], s, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, y[6], y[7], s, true);
    w0 = __builtin_bit_cast(unsigned, a); w1 = __builtin_bit_cast(unsigned, b);
  }
}

// rounds 8 columns held by this thread (the 4 threads of a group are neighbours and all here) and returns codes and scale byte
template <int BITS>
__device__ __forceinline__ unsigned quantise8(const float* x, unsigned& w0, unsigned& w1) {
  float amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(x[i]);
    bad |= !(a < __builtin_inff());
    amax = fmaxf(amax, a);
  }
  int any = bad;
  any |= __shfl_xor(any, 1); any |= __shfl_xor(any, 2);
  amax = fmaxf(amax, __shfl_xor(amax, 1)); amax = fmaxf(amax, __shfl_xor(amax, 2));
  if (any) { w0 = w1 = 0; return 255u; }
  const unsigned byte = scale_byte<BITS>(amax);
  encode8<BITS>(x, scale_of(byte), w0, w1);
  return byte;
}

// CH = dim / 8 threads per row
template <int DT, int BITS, int CH>
__global__ void __launch_bounds__(WR_THREADS)
k_bank_write(gpsr_bank bk, const int32_t* __restrict__ table, int table_pages, int pshift, const int32_t* __restrict__ start,
             const int32_t* __restrict__ count, const typename Row<DT>::T* __restrict__ k,
             const typename Row<DT>::T* __restrict__ v, int T, Strides ks, Strides vs, bool kwide, bool vwide) {
  constexpr int NR = WR_THREADS / CH;     // rows at a time; threads behind NR * CH idle (dim 96 and 192)
  constexpr int D = CH * 8;
  __shared__ double part[NR * D];         // column sums of each thread row; before, the groups' square sums of one pass
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const int P = 1 << pshift;
  const int first = start[b], n = min(count[b], T);
  if (first < 0 || n <= 0) return;
  const int64_t end = (int64_t)first + n;
  const int64_t lp = (first >> pshift) + (int64_t)blockIdx.x;   // logical page
  if (lp * P >= end || lp >= table_pages) return;
  const int64_t page = table[(size_t)b * table_pages + lp];
  if (page < 0 || page >= bk.pages) return;
  const int r0 = lp * P >= first ? 0 : (int)(first - lp * P);           // rows [r0, r1) are new, [0, r0) were there
  const int r1 = (int)(end - lp * P < P ? end - lp * P : P);
  const size_t row0 = ((size_t)page * bk.heads + h) * P;
  const int c = tid % CH, rr = tid / CH;
  const bool mine = rr < NR;
  const int64_t t0 = lp * P - first;      // t of row 0 of the page (negative before the first)
  double sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int base = 0; base < r1; base += NR) {
    const int r = base + rr;
    const bool there = mine && r < r1, fresh = there && r >= r0;
    double sq = 0.0;
    if (there) {
      unsigned w0, w1, byte;
      unsigned* codes = (unsigned*)(bk.k_codes + (row0 + r) * (D * BITS / 8)) + c * (BITS / 4);
      uint8_t* sc = bk.k_scales + (row0 + r) * (D / BK_GROUP) + c / 4;
      float x[8];
      if (fresh) {
        load8<DT>(k + b * ks.b + (t0 + r) * ks.t + h * ks.h + c * 8, kwide, x);
        byte = quantise8<BITS>(x, w0, w1);
        if (BITS == 4) codes[0] = w0; else *(u2v*)codes = u2v{w0, w1};
        if (c % 4 == 0) *sc = (uint8_t)byte;
      } else {
        w0 = codes[0]; w1 = BITS == 8 ? codes[1] : 0u; byte = *sc;
      }
      float y[8];
      decode8<BITS>(w0, w1, scale_of(byte), y);
#pragma unroll
      for (int i = 0; i < 8; ++i) { const double d = (double)y[i]; sum[i] += d; sq = fma(d, d, sq); }
      if (fresh) {
        load8<DT>(v + b * vs.b + (t0 + r) * vs.t + h * vs.h + c * 8, vwide, x);
        byte = quantise8<BITS>(x, w0, w1);
        unsigned* vc = (unsigned*)(bk.v_codes + (row0 + r) * (D * BITS / 8)) + c * (BITS / 4);
        if (BITS == 4) vc[0] = w0; else *(u2v*)vc = u2v{w0, w1};
        if (c % 4 == 0) bk.v_scales[(row0 + r) * (D / BK_GROUP) + c / 4] = (uint8_t)byte;
      }
    }
    if (bk.kernel_id == GPSR_KERNEL_RBF) {
      sq += __shfl_xor(sq, 1); sq += __shfl_xor(sq, 2);
      __syncthreads();
      if (mine && c % 4 == 0) part[rr * (CH / 4) + c / 4] = sq;
      __syncthreads();
      if (fresh && c == 0) {
        double s = 0.0;
        for (int g = 0; g < CH / 4; ++g) s += part[rr * (CH / 4) + g];
        bk.offset[row0 + r] = (float)(-0.5 * s);
      }
    } else if (fresh && c == 0) {
      bk.offset[row0 + r] = 0.f;
    }
  }
  __syncthreads();
  if (mine)
#pragma unroll
    for (int i = 0; i < 8; ++i) part[rr * D + c * 8 + i] = sum[i];
  __syncthreads();
  if (tid < D) {
    double s = 0.0;
    for (int i = 0; i < NR; ++i) s += part[i * D + tid];
    bk.centroid[((size_t)page * bk.heads + h) * D + tid] = (float)(s / (double)r1);
  }
}

template <int DT, int BITS>
static void launch_write(dim3 grid, hipStream_t st, const gpsr_bank& bk, const int32_t* table, int table_pages, int pshift,
                         const int32_t* start, const int32_t* count, const void* k, const void* v, int T, Strides ks,
                         Strides vs, bool kwide, bool vwide) {
  typedef typename Row<DT>::T E;
#define WRITE(CH) hipLaunchKernelGGL((k_bank_write<DT, BITS, CH>), grid, dim3(WR_THREADS), 0, st, bk, table, table_pages, \
                                     pshift, start, count, (const E*)k, (const E*)v, T, ks, vs, kwide, vwide)
  switch (bk.dim) {
    case 32: WRITE(4); break;
    case 64: WRITE(8); break;
    case 96: WRITE(12); break;
    case 128: WRITE(16); break;
    case 192: WRITE(24); break;
    default: WRITE(32); break;
  }
#undef WRITE
}

extern "C" int gpsr_bank_write(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* start,
                               const int32_t* count, const void* k, const void* v, int dtype, int T, const int64_t* kst,
                               const int64_t* vst, void* stream) {
  if (B <= 0 || T <= 0) return 0;
  if (const char* w = bank_wrong(bank)) return arg_fail(w);
  if (!table || !start || !count || !k || !v || !kst || !vst) return arg_fail("bank_write: null pointer");
  if (!type_ok(dtype)) return arg_fail("bank_write: dtype");
  if (B > 65535) return arg_fail("bank_write: more than 65535 entries");
  if (table_pages < 1) return arg_fail("bank_write: empty table");
  const int pshift = __builtin_ctz((unsigned)bank->page_rows);
  // a run of T rows that starts anywhere in a page touches at most this many
  int64_t touched = (((int64_t)T + bank->page_rows - 2) >> pshift) + 1;
  if (touched > table_pages) touched = table_pages;
  if (!grid_fits(touched, WR_THREADS)) return arg_fail("bank_write: too many rows for one call");
  const dim3 grid((unsigned)touched, (unsigned)bank->heads, (unsigned)B);
  const Strides ks = {kst[0], kst[1], kst[2]}, vs = {vst[0], vst[1], vst[2]};
  const bool kw = rows_wide(k, kst, dtype), vw = rows_wide(v, vst, dtype);
  hipStream_t st = (hipStream_t)stream;
#define WRITE(DT, BITS) launch_write<DT, BITS>(grid, st, *bank, table, table_pages, pshift, start, count, k, v, T, ks, vs, kw, vw)
  if (bank->bits == 4) {
    if (dtype == GPSR_BF16) WRITE(GPSR_BF16, 4); else if (dtype == GPSR_F16) WRITE(GPSR_F16, 4); else WRITE(GPSR_F32, 4);
  } else {
    if (dtype == GPSR_BF16) WRITE(GPSR_BF16, 8); else if (dtype == GPSR_F16) WRITE(GPSR_F16, 8); else WRITE(GPSR_F32, 8);
  }
#undef WRITE
  CHECK_LAUNCH("k_bank_write");
  return 0;
}

// ---------------------------------------------------------------- read
// One thread per 8 columns of a row, keys and values together; bound by the stores (4 bits: 2 bytes written per half byte read;
// 2^20 rows of 64 columns from 4 bits to bf16 61 us, 5.5 TB/s).
template <int DT, int BITS>
__global__ void __launch_bounds__(256)
k_bank_read(gpsr_bank bk, const int32_t* __restrict__ table, int table_pages, int pshift, const int32_t* __restrict__ start,
            const int32_t* __restrict__ count, typename Row<DT>::T* __restrict__ k, typename Row<DT>::T* __restrict__ v, int T) {
  const int ch = bk.dim / 8, H = bk.heads;
  const int64_t per = (int64_t)T * H * ch;                    // work items of one entry
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= per) return;
  const int b = blockIdx.y;
  const int c = (int)(item % ch);
  const int64_t th = item / ch;
  const int h = (int)(th % H);
  const int64_t t = th / H;
  const int first = start[b];
  const int64_t pos = (int64_t)first + t, lp = pos >> pshift;
  float y[8] = {0, 0, 0, 0, 0, 0, 0, 0}, z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (first >= 0 && t < count[b] && lp < table_pages) {
    const int64_t page = table[(size_t)b * table_pages + lp];
    if (page >= 0 && page < bk.pages) {
      const size_t row = (((size_t)page * H + h) << pshift) + (size_t)(pos & ((1 << pshift) - 1));
      const unsigned* kc = (const unsigned*)(bk.k_codes + row * (size_t)(bk.dim * BITS / 8)) + c * (BITS / 4);
      const unsigned* vc = (const unsigned*)(bk.v_codes + row * (size_t)(bk.dim * BITS / 8)) + c * (BITS / 4);
      const size_t g = row * (size_t)(bk.dim / BK_GROUP) + c / 4;
      decode8<BITS>(kc[0], BITS == 8 ? kc[1] : 0u, scale_of(bk.k_scales[g]), y);
      decode8<BITS>(vc[0], BITS == 8 ? vc[1] : 0u, scale_of(bk.v_scales[g]), z);
    }
  }
  const size_t at = ((size_t)b * per + item) * 8;
  store8<DT>(k + at, y);
  store8<DT>(v + at, z);
}

extern "C" int gpsr_bank_read(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* start,
                              const int32_t* count, void* k, void* v, int dtype, int T, void* stream) {
  if (B <= 0 || T <= 0) return 0;
  if (const char* w = bank_wrong(bank)) return arg_fail(w);
  if (!table || !start || !count || !k || !v) return arg_fail("bank_read: null pointer");
  if (!type_ok(dtype)) return arg_fail("bank_read: dtype");
  if (B > 65535) return arg_fail("bank_read: more than 65535 entries");
  if (table_pages < 1) return arg_fail("bank_read: empty table");
  if (((uintptr_t)k | (uintptr_t)v) & 15) return arg_fail("bank_read: k and v must be 16-byte aligned");
  const int pshift = __builtin_ctz((unsigned)bank->page_rows);
  const int64_t blocks = ((int64_t)T * bank->heads * (bank->dim / 8) + 255) / 256;
  if (!grid_fits(blocks, 256)) return arg_fail("bank_read: too many rows for one call");
  const dim3 grid((unsigned)blocks, (unsigned)B);
  hipStream_t st = (hipStream_t)stream;
#define READ(DT, BITS) hipLaunchKernelGGL((k_bank_read<DT, BITS>), grid, dim3(256), 0, st, *bank, table, table_pages, pshift, \
                                          start, count, (Row<DT>::T*)k, (Row<DT>::T*)v, T)
  if (bank->bits == 4) {
    if (dtype == GPSR_BF16) READ(GPSR_BF16, 4); else if (dtype == GPSR_F16) READ(GPSR_F16, 4); else READ(GPSR_F32, 4);
  } else {
    if (dtype == GPSR_BF16) READ(GPSR_BF16, 8); else if (dtype == GPSR_F16) READ(GPSR_F16, 8); else READ(GPSR_F32, 8);
  }
#undef READ
  CHECK_LAUNCH("k_bank_read");
  return 0;
}

// ---------------------------------------------------------------- images to rows and back
// WI_X neighbouring windows of an image row a workgroup: their pixels go through LDS once (a window shares all but a column of them
// with the next), four threads take a window's mean, then a thread makes 8 columns of a window at a time, one store.  Bound by the
// stores: 8.3 million windows of 7 x 7 pixels as 64 bf16 columns 345 us (384 without their means), 3.1 TB/s (a wave a window, two bytes
// a store, 1480 us).
#define WI_X 64
template <int DT>
__global__ void __launch_bounds__(256)
k_bank_windows(const double* __restrict__ img, int W, int side, bool centre, int wide, typename Row<DT>::T* __restrict__ out, int dim,
               bool whole) {
  constexpr int LD = WI_X + 16;
  __shared__ double px[15 * LD];
  __shared__ double mean[WI_X];
  __shared__ __attribute__((aligned(16))) uint16_t at[256];       // where a column's pixel lies behind its window's first; 0xffff: none
  const int tid = threadIdx.x, x0 = blockIdx.x * WI_X, n = min(WI_X, wide - x0), cols = side * side;
  const double* p = img + (size_t)blockIdx.y * W + x0;
  for (int i = tid; i < side * LD; i += 256) {
    const int r = i / LD, c = i - r * LD;
    if (c < n + side - 1) px[i] = p[(size_t)r * W + c];
  }
  at[tid] = tid < cols ? (uint16_t)(tid / side * LD + tid % side) : (uint16_t)0xffff;
  __syncthreads();
  const int w4 = tid >> 2;
  double sum = 0.0;
  if (centre && w4 < n)
    for (int r = tid & 3; r < side; r += 4)
      for (int c = 0; c < side; ++c) sum += px[r * LD + w4 + c];
  sum += __shfl_xor(sum, 1); sum += __shfl_xor(sum, 2);
  if ((tid & 3) == 0) mean[w4] = sum / cols;
  __syncthreads();
  const int units = (dim + 7) / 8;
  for (int u = tid; u < n * units; u += 256) {
    const int w = u / units, j = u - w * units;
    const u4v a = *(const u4v*)(at + j * 8);
    const double m = mean[w];
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned o = e % 2 ? a[e / 2] >> 16 : a[e / 2] & 0xffffu;
      y[e] = o == 0xffffu ? 0.f : (float)(px[o + w] - m);
    }
    typename Row<DT>::T* to = out + ((size_t)blockIdx.y * wide + x0 + w) * dim + j * 8;
    if (whole) store8<DT>(to, y);
    else
      for (int e = 0; e < 8 && j * 8 + e < dim; ++e) {
        if constexpr (DT == GPSR_BF16) to[e] = bf16_rne(y[e]); else to[e] = (typename Row<DT>::T)y[e];
      }
  }
}

// A workgroup has BL_X x BL_Y pixels and walks the rows of windows that reach them; each row's windows, contiguous in memory, go
// through LDS.  Thread (x, s) sums for the pixel of column x whose row is s modulo side: side neighbouring rows are being
// summed at a time, and a window row is the first of one of them and the last of another.  Every pixel's sum so runs over its
// windows in their order.  The same 8.3 million windows back to pixels 329 us, 3.2 TB/s (a thread a pixel that reads its windows
// itself, side * side cache lines for as many values, 6900 us).
#define BL_X 32
#define BL_Y 16
// elements between windows in LDS: whole 16-byte units, an odd number of them
static constexpr int blend_row(int side, int size) {
  const int u = (side * side + 7) / 8 * 8 * size / 16;
  return (u | 1) * 16 / size;
}
template <int DT>
__global__ void __launch_bounds__(512)
k_bank_blend(const double* __restrict__ img, int H, int W, int side, const typename Row<DT>::T* __restrict__ detail, int dim,
             double* __restrict__ out, bool whole) {
  typedef typename Row<DT>::T E;
  extern __shared__ __attribute__((aligned(16))) char raw[];
  E* const row = (E*)raw;
  constexpr int PU = 8 * sizeof(E) / 16;         // 16-byte pieces of a unit of 8 columns
  const int tid = threadIdx.x, threads = BL_X * side, tx = tid % BL_X, s = tid / BL_X;
  const int x0 = blockIdx.x * BL_X, y0 = blockIdx.y * BL_Y, x = x0 + tx;
  const int wide = W - side + 1, high = H - side + 1, units = (side * side + 7) / 8, ld = blend_row(side, sizeof(E));
  const int wx0 = max(x0 - side + 1, 0), nw = min(x0 + BL_X, wide) - wx0;
  const int wy0 = max(y0 - side + 1, 0), wy1 = min(y0 + BL_Y, high);
  const int xa = max(x - side + 1, 0), xz = min(x, wide - 1);
  // units of a row of windows that this thread carries: at most 3 (15 * 15 columns, 46 windows, 480 threads)
  u4v next[3][PU];
  const auto fetch = [&](int wy) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int u = tid + i * threads, w = u / units;
      if (w < nw) {
        const u4v* from = (const u4v*)(detail + ((size_t)wy * wide + wx0 + w) * dim + (u - w * units) * 8);
#pragma unroll
        for (int j = 0; j < PU; ++j) next[i][j] = from[j];
      }
    }
  };
  if (whole) fetch(wy0);
  double sum = 0.0;
  int dy = (s - wy0 % side + side) % side;       // rows between the window row and the pixel's
  for (int wy = wy0; wy < wy1; ++wy, dy = dy ? dy - 1 : side - 1) {
    __syncthreads();
    if (whole) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int u = tid + i * threads, w = u / units;
        if (w < nw)
#pragma unroll
          for (int j = 0; j < PU; ++j) ((u4v*)(row + w * ld + (u - w * units) * 8))[j] = next[i][j];
      }
    } else {
      for (int i = tid; i < nw * side * side; i += threads) {
        const int w = i / (side * side), c = i - w * (side * side);
        row[w * ld + c] = detail[((size_t)wy * wide + wx0 + w) * dim + c];
      }
    }
    __syncthreads();
    if (whole && wy + 1 < wy1) fetch(wy + 1);
    const int y = wy + dy;
    if (x < W && y >= y0 && y < y0 + BL_Y) {
      const E* from = row + (xa - wx0) * ld + dy * side + (x - xa);
      for (int wx = xa; wx <= xz; ++wx, from += ld - 1) sum += (double)to_f32<DT>(*from);
      if (wy == min(y, high - 1)) {
        const int n = (xz - xa + 1) * (wy - max(y - side + 1, 0) + 1);
        out[(size_t)y * W + x] = img[(size_t)y * W + x] + sum / n;
        sum = 0.0;
      }
    }
  }
}

static const char* windows_wrong(const double* img, int H, int W, int side, const void* rows, int dtype, int dim) {
  if (!img || !rows) return "bank_windows: null pointer";
  if (side < 3 || side > 15 || side % 2 == 0) return "bank_windows: side must be odd, 3..15";
  if (H < side || W < side) return "bank_windows: image smaller than a window";
  if (dim < side * side || dim > 256) return "bank_windows: dim must be in side * side .. 256";
  if (!type_ok(dtype)) return "bank_windows: dtype";
  if (W > (1 << 24)) return "bank_windows: more than 2^24 columns";
  if (H > 65535) return "bank_windows: more than 65535 rows";
  return nullptr;
}
extern "C" int gpsr_bank_windows(const double* img, int H, int W, int side, int centre, void* out, int dtype, int dim, void* stream) {
  if (const char* w = windows_wrong(img, H, W, side, out, dtype, dim)) return arg_fail(w);
  const int wide = W - side + 1;
  const dim3 grid((unsigned)((wide + WI_X - 1) / WI_X), (unsigned)(H - side + 1));
  const bool whole = dim % 8 == 0 && !((uintptr_t)out & 15);
  hipStream_t st = (hipStream_t)stream;
#define WINDOWS(DT) hipLaunchKernelGGL((k_bank_windows<DT>), grid, dim3(256), 0, st, img, W, side, centre != 0, wide, (Row<DT>::T*)out, dim, whole)
  if (dtype == GPSR_BF16) WINDOWS(GPSR_BF16); else if (dtype == GPSR_F16) WINDOWS(GPSR_F16); else WINDOWS(GPSR_F32);
#undef WINDOWS
  CHECK_LAUNCH("k_bank_windows");
  return 0;
}
extern "C" int gpsr_bank_blend(const double* img, int H, int W, int side, const void* detail, int dtype, int dim, double* out, void* stream) {
  if (const char* w = windows_wrong(img, H, W, side, detail, dtype, dim)) return arg_fail(w);
  if (!out) return arg_fail("bank_blend: null pointer");
  const dim3 grid((unsigned)((W + BL_X - 1) / BL_X), (unsigned)((H + BL_Y - 1) / BL_Y));
  const bool whole = dim % 8 == 0 && !((uintptr_t)detail & 15);
  const size_t lds = (size_t)(BL_X + side - 1) * blend_row(side, (int)type_size(dtype)) * type_size(dtype);
  hipStream_t st = (hipStream_t)stream;
#define BLEND(DT) hipLaunchKernelGGL((k_bank_blend<DT>), grid, dim3(BL_X * side), lds, st, img, H, W, side, (const Row<DT>::T*)detail, dim, out, whole)
  if (dtype == GPSR_BF16) BLEND(GPSR_BF16); else if (dtype == GPSR_F16) BLEND(GPSR_F16); else BLEND(GPSR_F32);
#undef BLEND
  CHECK_LAUNCH("k_bank_blend");
  return 0;
}
