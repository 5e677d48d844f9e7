// gpsr_bank_select.hip -- example bank: the best pages for each query (include/gpsr.h).
#include "gpsr_bank.hpp"

// One workgroup per query and bank head: 64-bit scores of 1024 pages at a time next to the best so far, n_sel rounds of arg max.
#define SE_PAGES 1024
#define SE_MAX 64
template <int DT>
__global__ void __launch_bounds__(256)
k_bank_select(gpsr_bank bk, const int32_t* __restrict__ table, int table_pages, int pshift, const int32_t* __restrict__ length,
              const typename Row<DT>::T* __restrict__ q, int T, int G, Strides qs, int n_sel, const int32_t* __restrict__ skip,
              int32_t* __restrict__ sel) {
  __shared__ double qv[256];
  __shared__ double sc[SE_PAGES + SE_MAX];
  __shared__ int id[SE_PAGES + SE_MAX];
  __shared__ double bs[4];
  __shared__ int bi[4], bp[4];
  __shared__ double keep_s[SE_MAX];
  __shared__ int keep_i[SE_MAX];
  const int D = bk.dim, tid = threadIdx.x, P = 1 << pshift, t = blockIdx.x, h = blockIdx.y, b = blockIdx.z, H = bk.heads;
  const double none = -__builtin_inf();
  for (int i = tid; i < D; i += 256) {
    double s = 0.0;
    for (int g = 0; g < G; ++g) s += (double)to_f32<DT>(q[b * qs.b + t * qs.t + (int64_t)(h * G + g) * qs.h + i]);
    qv[i] = s;
  }
  int64_t len = length[b];
  if (len > (int64_t)table_pages * P) len = (int64_t)table_pages * P;
  const int pages = len <= 0 ? 0 : (int)((len + P - 1) >> pshift);
  const int lo = skip ? skip[((size_t)b * T + t) * 2] : 0, hi = skip ? skip[((size_t)b * T + t) * 2 + 1] : 0;
  if (tid < SE_MAX) { sc[SE_PAGES + tid] = none; id[SE_PAGES + tid] = 0x7fffffff; }
  __syncthreads();
  for (int base = 0; base < pages; base += SE_PAGES) {
    for (int j = tid; j < SE_PAGES; j += 256) {
      const int lp = base + j;
      double s = none;
      if (lp < pages) {
        const int64_t page = table[(size_t)b * table_pages + lp];
        const int64_t first = (int64_t)lp * P, last = first + P < len ? first + P : len;
        if (page >= 0 && page < bk.pages && !(lo <= first && hi >= last)) {
          const float* c = bk.centroid + ((size_t)page * H + h) * D;
          double dot = 0.0, sq = 0.0;
          for (int i = 0; i < D; ++i) { const double ci = c[i]; dot = fma(qv[i], ci, dot); sq = fma(ci, ci, sq); }
          s = bk.kernel_id == GPSR_KERNEL_RBF ? dot - 0.5 * G * sq : dot;
        }
      }
      sc[j] = s; id[j] = s == none ? 0x7fffffff : lp;
    }
    __syncthreads();
    for (int k = 0; k < n_sel; ++k) {
      double s = none; int at = 0x7fffffff, place = 0;
      for (int j = tid; j < SE_PAGES + SE_MAX; j += 256)
        if (sc[j] > s || (sc[j] == s && id[j] < at)) { s = sc[j]; at = id[j]; place = j; }
      for (int o = 32; o; o >>= 1) {
        const double s2 = __shfl_xor(s, o); const int a2 = __shfl_xor(at, o), p2 = __shfl_xor(place, o);
        if (s2 > s || (s2 == s && a2 < at)) { s = s2; at = a2; place = p2; }
      }
      if (tid % 64 == 0) { bs[tid / 64] = s; bi[tid / 64] = at; bp[tid / 64] = place; }
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < 4; ++w) if (bs[w] > s || (bs[w] == s && bi[w] < at)) { s = bs[w]; at = bi[w]; place = bp[w]; }
        keep_s[k] = s; keep_i[k] = at;
        sc[place] = none; id[place] = 0x7fffffff;
      }
      __syncthreads();
    }
    if (tid < n_sel) { sc[SE_PAGES + tid] = keep_s[tid]; id[SE_PAGES + tid] = keep_i[tid]; }
    __syncthreads();
  }
  if (tid < n_sel) {
    const int mine = id[SE_PAGES + tid];
    int rank = 0;
    for (int j = 0; j < n_sel; ++j) { const int o = id[SE_PAGES + j]; rank += o < mine || (o == mine && j < tid); }
    sel[(((size_t)b * T + t) * H + h) * n_sel + rank] = mine == 0x7fffffff ? -1 : mine;
  }
}

extern "C" size_t gpsr_bank_select_workspace_bytes(const gpsr_bank* bank, int B, int table_pages, int T, int q_heads, int n_sel, int dtype) {
  return 0;
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
  const int pshift = __builtin_ctz((unsigned)bank->page_rows), G = q_heads / bank->heads;
  const Strides qs = {qst[0], qst[1], qst[2]};
  const dim3 grid((unsigned)T, (unsigned)bank->heads, (unsigned)B);
  hipStream_t st = (hipStream_t)stream;
#define SELECT(DT) hipLaunchKernelGGL((k_bank_select<DT>), grid, dim3(256), 0, st, *bank, table, table_pages, pshift, length, \
                                      (const Row<DT>::T*)q, T, G, qs, n_sel, skip, sel)
  if (dtype == GPSR_BF16) SELECT(GPSR_BF16); else if (dtype == GPSR_F16) SELECT(GPSR_F16); else SELECT(GPSR_F32);
#undef SELECT
  CHECK_LAUNCH("k_bank_select");
  return 0;
}
