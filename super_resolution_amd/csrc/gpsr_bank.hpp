// gpsr_bank.hpp -- what the example-bank kernels share: the bank's layout, its number formats, typed rows.
//
// Codes are the two element formats that gfx950 converts in hardware, E2M1 (4 bits) and E4M3 (8 bits), with one power-of-two
// scale byte per 32 columns.  v_cvt_scalef32_* multiplies by the scale while it converts, both ways, exactly (a held value
// has at most 4 significant bits, so bf16 holds it too); a scale byte of 255 gives NaN without a further instruction.
#pragma once
#include "gpsr_host.hpp"
#include "../../include/gpsr.h"

#define BK_GROUP 32   // columns that share a scale byte

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s2v __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned u2v __attribute__((ext_vector_type(2)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));

struct Strides { int64_t b, t, h; };   // elements between entries, rows, heads

// the wave's number, as the uniform value that it is: what follows from it needs no lanes and no masks
__device__ __forceinline__ int wave_of(int tid) { return __builtin_amdgcn_readfirstlane(tid >> 6); }

__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// 8 columns of a row as held: w0 (and w1 for 8 bits) are the code words, s the scale
template <int BITS>
__device__ __forceinline__ void decode8(unsigned w0, unsigned w1, float s, float* y) {
  f2v p[4];
  if (BITS == 4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w0, s, 0); p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w0, s, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w0, s, 2); p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w0, s, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w0, s, false); p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w0, s, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w1, s, false); p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w1, s, true);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) { y[2 * i] = p[i].x; y[2 * i + 1] = p[i].y; }
}

// ---- rows of the caller's type: 8 elements at p + i (elements); wide loads where the launch found every row 16-byte aligned
template <int DT> struct Row;
template <> struct Row<GPSR_BF16> { typedef uint16_t T; };
template <> struct Row<GPSR_F16> { typedef _Float16 T; };
template <> struct Row<GPSR_F32> { typedef float T; };

template <int DT>
__device__ __forceinline__ float to_f32(typename Row<DT>::T v) {
  if constexpr (DT == GPSR_BF16) return __uint_as_float((unsigned)v << 16);
  else return (float)v;
}
__device__ __forceinline__ uint16_t bf16_rne(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }

template <int DT>
__device__ __forceinline__ void load8(const typename Row<DT>::T* __restrict__ p, bool wide, float* y) {
  if (wide) {
    if constexpr (DT == GPSR_F32) {
      const f4v a = ((const f4v*)p)[0], b = ((const f4v*)p)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) { y[i] = a[i]; y[4 + i] = b[i]; }
    } else {
      const u4v a = *(const u4v*)p;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == GPSR_BF16) { y[2 * i] = __uint_as_float(a[i] << 16); y[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u); }
        else {
          y[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(a[i] & 0xffff));
          y[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(a[i] >> 16));
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_f32<DT>(p[i]);
  }
}

// rounded once; outputs are the library's own contiguous rows (dim is a multiple of 32), so stores are always wide
template <int DT>
__device__ __forceinline__ void store8(typename Row<DT>::T* __restrict__ p, const float* y) {
  if constexpr (DT == GPSR_F32) {
    f4v a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = y[i]; b[i] = y[4 + i]; }
    ((f4v*)p)[0] = a; ((f4v*)p)[1] = b;
  } else {
    u4v a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned lo, hi;
      if constexpr (DT == GPSR_BF16) { lo = bf16_rne(y[2 * i]); hi = bf16_rne(y[2 * i + 1]); }
      else { lo = __builtin_bit_cast(uint16_t, (_Float16)y[2 * i]); hi = __builtin_bit_cast(uint16_t, (_Float16)y[2 * i + 1]); }
      a[i] = lo | (hi << 16);
    }
    *(u4v*)p = a;
  }
}

// over all lanes of a wave, by moves between neighbouring lanes, rows of 16 and halves
template <class F>
__device__ __forceinline__ float wave_all(float x, float none, const F& f) {
#define STEP(ctrl) x = f(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(x), ctrl, 0xf, 0xf, false)))
  STEP(0x111); STEP(0x112); STEP(0x114); STEP(0x118);   // row_shr 1, 2, 4, 8
  STEP(0x142); STEP(0x143);                             // row_bcast 15, 31
#undef STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// ---- host side
// every bank that the kernels accept; text for arg_fail, or NULL
static inline const char* bank_wrong(const gpsr_bank* b) {
  if (!b) return "bank: null pointer";
  if (!b->k_codes || !b->k_scales || !b->v_codes || !b->v_scales || !b->offset || !b->centroid) return "bank: null pointer";
  if (b->pages < 1 || b->pages > 0x7fffffff) return "bank: pages must be in 1..2^31-1";
  if (b->heads < 1 || b->heads > 65535) return "bank: heads must be in 1..65535";
  const int P = b->page_rows, D = b->dim;
  if (P < 16 || P > 256 || (P & (P - 1))) return "bank: page_rows must be 16, 32, 64, 128 or 256";
  if (D != 32 && D != 64 && D != 96 && D != 128 && D != 192 && D != 256) return "bank: dim must be 32, 64, 96, 128, 192 or 256";
  if (b->bits != 4 && b->bits != 8) return "bank: bits must be 4 or 8";
  if (b->kernel_id != GPSR_KERNEL_RBF && b->kernel_id != GPSR_KERNEL_LINEAR) return "bank: kernel_id must be RBF or LINEAR";
  if (((uintptr_t)b->k_codes | (uintptr_t)b->v_codes | (uintptr_t)b->k_scales | (uintptr_t)b->v_scales | (uintptr_t)b->offset |
       (uintptr_t)b->centroid) & 15) return "bank: arrays must be 16-byte aligned";
  return nullptr;
}
static inline size_t type_size(int dtype) { return dtype == GPSR_F32 ? 4 : 2; }
static inline bool type_ok(int dtype) { return dtype == GPSR_BF16 || dtype == GPSR_F16 || dtype == GPSR_F32; }
// a launch can have fewer than 2^32 threads along a dimension
static inline bool grid_fits(int64_t groups, int threads) { return groups <= (int64_t)0xffffffffu / threads; }
// whether every row starts at a multiple of 16 bytes
static inline bool rows_wide(const void* p, const int64_t* st, int dtype) {
  const int64_t m = 16 / (int64_t)type_size(dtype);
  return !((uintptr_t)p & 15) && st[0] % m == 0 && st[1] % m == 0 && st[2] % m == 0;
}
