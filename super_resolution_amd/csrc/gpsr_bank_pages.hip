// gpsr_bank_pages.hip -- example bank: attention over chosen pages (include/gpsr.h).
#include "gpsr_bank_tile.hpp"

// One workgroup per query and head: 32 rows at a time are decoded to LDS, each row's logit is one thread-octet's dot product,
// the running maximum and sum rescale the output of the columns' own threads.
#define AT_ROWS 32
template <int DT, int BITS>
__global__ void __launch_bounds__(256)
k_bank_attend_pages(gpsr_bank bk, const int32_t* __restrict__ table, int table_pages, int pshift, const int32_t* __restrict__ length,
              const typename Row<DT>::T* __restrict__ q, int T, int G, Strides qs, const int32_t* __restrict__ sel, int n_sel,
              float scale, const int32_t* __restrict__ skip, typename Row<DT>::T* __restrict__ out, float* __restrict__ lse) {
  extern __shared__ float sm[];
  const int D = bk.dim, ld = D + 1, tid = threadIdx.x, P = 1 << pshift;
  float* tile = sm;                   // [AT_ROWS][D + 1]
  float* qv = tile + AT_ROWS * ld;    // [D]
  float* x = qv + D;                  // [AT_ROWS]
  const int t = blockIdx.x, hq = blockIdx.y, b = blockIdx.z, h = hq / G, H = bk.heads;
  for (int i = tid; i < D; i += 256) qv[i] = to_f32<DT>(q[b * qs.b + t * qs.t + hq * qs.h + i]);
  int64_t len = length[b];
  if (len > (int64_t)table_pages * P) len = (int64_t)table_pages * P;
  const int lo = skip ? skip[((size_t)b * T + t) * 2] : 0, hi = skip ? skip[((size_t)b * T + t) * 2 + 1] : 0;
  const int32_t* mine = sel ? sel + (((size_t)b * T + t) * H + h) * n_sel : nullptr;
  const int pages = sel ? n_sel : (int)((len + P - 1) >> pshift);
  float m = -__builtin_inff(), l = 0.f, acc = 0.f;
  const float c2 = scale * 1.4426950408889634f;
  for (int i = 0; i < pages; ++i) {
    const int lp = sel ? mine[i] : i;
    if (lp < 0 || lp >= table_pages) continue;
    bool again = false;
    if (sel) for (int j = 0; j < i; ++j) again |= mine[j] == lp;
    if (again) continue;
    const int64_t page = table[(size_t)b * table_pages + lp];
    if (page < 0 || page >= bk.pages) continue;
    const size_t row0 = ((size_t)page * H + h) << pshift;
    const int64_t pos0 = (int64_t)lp << pshift;
    for (int r0 = 0; r0 < P && pos0 + r0 < len; r0 += AT_ROWS) {
      for (int pass = 0; pass < 2; ++pass) {
        __syncthreads();
        for (int e = tid; e < AT_ROWS * (D / 8); e += 256) {
          const int r = e / (D / 8), c = e % (D / 8);
          float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          const int64_t pos = pos0 + r0 + r;
          if (r0 + r < P && pos < len && !(pos >= lo && pos < hi)) {
            const size_t row = row0 + r0 + r;
            const unsigned* w = (const unsigned*)((pass ? bk.v_codes : bk.k_codes) + row * (size_t)(D * BITS / 8)) + c * (BITS / 4);
            decode8<BITS>(w[0], BITS == 8 ? w[1] : 0u, scale_of((pass ? bk.v_scales : bk.k_scales)[row * (size_t)(D / BK_GROUP) + c / 4]), y);
          }
          for (int j = 0; j < 8; ++j) tile[r * ld + c * 8 + j] = y[j];
        }
        __syncthreads();
        if (pass == 0) {
          const int r = tid / 8, o = tid % 8;
          float s = 0.f;
          for (int i2 = o; i2 < D; i2 += 8) s = fmaf(qv[i2], tile[r * ld + i2], s);
          s += __shfl_xor(s, 1); s += __shfl_xor(s, 2); s += __shfl_xor(s, 4);
          const int64_t pos = pos0 + r0 + r;
          const bool ok = r0 + r < P && pos < len && !(pos >= lo && pos < hi);
          if (o == 0) x[r] = ok ? (s + bk.offset[row0 + r0 + r]) * c2 : -__builtin_inff();
        }
      }
      float mn = m;
      for (int r = 0; r < AT_ROWS; ++r) mn = fmaxf(mn, x[r]);
      const float safe = mn == -__builtin_inff() ? 0.f : mn;
      const float a = exp2f(m - safe);
      l *= a; acc *= a; m = mn;
      for (int r = 0; r < AT_ROWS; ++r) {
        const float p = exp2f(x[r] - safe);
        l += p;
        if (tid < D) acc = fmaf(p, tile[r * ld + tid], acc);
      }
    }
  }
  const size_t at = (((size_t)b * T + t) * (size_t)(H * G) + hq) * D;
  if (tid < D) {
    const float y = l == 0.f ? 0.f : acc / l;
    if constexpr (DT == GPSR_BF16) out[at + tid] = bf16_rne(y); else out[at + tid] = (typename Row<DT>::T)y;
  }
  if (lse && tid == 0) lse[((size_t)b * (H * G) + hq) * T + t] = l == 0.f ? -__builtin_inff() : (log2f(l) + m) * 0.6931471805599453f;
}

static int attend(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* length, const void* q,
                  int dtype, int T, int q_heads, const int64_t* qst, const int32_t* sel, int n_sel, float scale,
                  const int32_t* skip, void* out, float* lse, hipStream_t st) {
  const int pshift = __builtin_ctz((unsigned)bank->page_rows), G = q_heads / bank->heads;
  const Strides qs = {qst[0], qst[1], qst[2]};
  const dim3 grid((unsigned)T, (unsigned)q_heads, (unsigned)B);
  const size_t lds = (AT_ROWS * (bank->dim + 1) + bank->dim + AT_ROWS) * sizeof(float);
#define ATTEND(DT, BITS) hipLaunchKernelGGL((k_bank_attend_pages<DT, BITS>), grid, dim3(256), lds, st, *bank, table, table_pages, pshift, \
                                            length, (const Row<DT>::T*)q, T, G, qs, sel, n_sel, scale, skip, (Row<DT>::T*)out, lse)
  if (bank->bits == 4) {
    if (dtype == GPSR_BF16) ATTEND(GPSR_BF16, 4); else if (dtype == GPSR_F16) ATTEND(GPSR_F16, 4); else ATTEND(GPSR_F32, 4);
  } else {
    if (dtype == GPSR_BF16) ATTEND(GPSR_BF16, 8); else if (dtype == GPSR_F16) ATTEND(GPSR_F16, 8); else ATTEND(GPSR_F32, 8);
  }
#undef ATTEND
  CHECK_LAUNCH("k_bank_attend_pages");
  return 0;
}

extern "C" size_t gpsr_bank_attend_pages_workspace_bytes(const gpsr_bank* bank, int B, int table_pages, int T, int q_heads, int n_sel, int dtype) {
  return 0;
}
extern "C" int gpsr_bank_attend_pages(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* length,
                                      const void* q, int dtype, int T, int q_heads, const int64_t* qst, const int32_t* sel, int n_sel,
                                      float scale, const int32_t* skip, void* out, float* lse, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (B <= 0 || T <= 0) return 0;
  if (const char* w = attend_wrong(bank, table, B, table_pages, length, q, dtype, q_heads, qst, scale, out)) return arg_fail(w);
  if (!sel) return arg_fail("bank_attend_pages: null pointer");
  if (n_sel < 1 || n_sel > 64) return arg_fail("bank_attend_pages: n_sel must be in 1..64");
  return attend(bank, table, B, table_pages, length, q, dtype, T, q_heads, qst, sel, n_sel, scale, skip, out, lse, (hipStream_t)stream);
}
