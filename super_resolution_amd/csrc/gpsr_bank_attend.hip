// gpsr_bank_attend.hip -- example bank: attention over all rows (include/gpsr.h).
#include "gpsr_bank_tile.hpp"

#include <type_traits>

// ---------------------------------------------------------------- attention over the whole bank
// Columns are the (query, head) pairs that share a bank head.  A workgroup of NW waves walks the rows of its split of the
// bank, KT at a time: all threads decode the tile to LDS once, then each wave multiplies it with its own 32 columns, NB x 32
// rows at a time.
//   WK = 1: each wave has columns of its own (many queries; bound by the exponentials and the matrix units)
//   WK = NW: all have the same columns and a share of the tile's rows each (few queries; bound by reading the bank)
template <int DT, int BITS, int D, int NW, int WK, int KT, int NB>
__global__ void __launch_bounds__(64 * NW, tile_waves(D, Terms<DT>::N, 1, NB))
k_bank_attend(gpsr_bank bk, const int32_t* __restrict__ table, int table_pages, int pshift, const int32_t* __restrict__ length,
              const typename Row<DT>::T* __restrict__ q, int T, int G, Strides qs, bool qwide, float scale,
              const int32_t* __restrict__ skip, typename Row<DT>::T* __restrict__ out, float* __restrict__ lse, int splits,
              float* __restrict__ part) {
  constexpr int NT = Terms<DT>::N, KW = KT / WK;                 // rows of one wave
  constexpr int CW = (NW / WK) * 32, NQ = 1;                     // columns of the workgroup
  __shared__ __attribute__((aligned(16))) char sm[tile_lds(D, KT)];
  Tile<D, KT> tile(sm);
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), half = lane >> 5, col = lane & 31;
  const int h = blockIdx.y, b = blockIdx.z, H = bk.heads;
  const int split = blockIdx.x % splits;
  const int64_t C = (int64_t)T * G, c0 = (int64_t)(blockIdx.x / splits) * CW + (WK == 1 ? wave * 32 : 0);
  const int wrow = WK == 1 ? 0 : wave * KW;                      // first row of this wave within a tile

  unsigned len = (unsigned)max(length[b], 0);
  const int64_t most = (int64_t)table_pages << pshift;
  if ((int64_t)len > most) len = (unsigned)most;
  const unsigned tiles = (len + KT - 1) / KT;
  const unsigned per = (tiles + splits - 1) / splits;
  const unsigned i0 = min(per * split, tiles), i1 = min(i0 + per, tiles);

  // this lane's columns: query rows as operand fragments, and what they skip
  bf8 qf[NQ][NT][D / 16];
  unsigned lo[NQ], hi[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int64_t c = c0 + n * 32 + col;
    const bool there = c < C;
    const int64_t t = there ? c / G : 0;
    load_query<DT, D>(q + b * qs.b + t * qs.t + (int64_t)(h * G + (there ? c - t * G : 0)) * qs.h, qwide, there, half, qf[n]);
    lo[n] = hi[n] = 0;
    if (skip && there) {
      const int32_t* s = skip + ((size_t)b * T + t) * 2;
      lo[n] = (unsigned)max(s[0], 0); hi[n] = (unsigned)max(s[1], 0);
    }
  }
  Soft<D, NQ> st;
  const float c2 = scale * 1.4426950408889634f;

  tile.clear_marks(tid, 64 * NW);
  Fetch<BITS, D, KT, 64 * NW> f;
  const WholeBank rows = {table + (size_t)b * table_pages, bk.pages, pshift, len};
  const auto step = [&](unsigned i, auto move) {
    __syncthreads();
    f.store(tile, tid, i + 1);
    __syncthreads();
    f.codes(bk, h, pshift, (i + 1) * KT, tid);
    f.pages(rows, (i + 2) * KT, tid);
    const unsigned p0 = i * KT;
    tile_marks<D, KT, NQ, KW>(tile, wrow, i + 1, st, [&](int n, int r) { return !(p0 + wrow + r >= lo[n] && p0 + wrow + r < hi[n]); });
    bool any = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) any |= lo[n] < p0 + KT && hi[n] > p0 && lo[n] < hi[n];
    const bool skips = skip && __ballot(any);
#pragma unroll 1
    for (int r = 0; r < KW; r += 32 * NB) {
      f16v s[NB][NQ];
      tile_logits<D, KT, NT, NQ, NB>(tile, wrow + r, col, half, qf, s);
      if (skips) {
        asm volatile("");        // not to be computed for the tiles that nobody skips
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const unsigned pos = p0 + wrow + r + kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3);
              if (pos >= lo[n] && pos < hi[n]) s[kb][n][e] = -__builtin_inff();
            }
      }
      tile_accumulate<D, KT, NT, NQ, NB, decltype(move)::value>(tile, wrow + r, col, half, c2, s, st);
    }
  };
  st.clear();
  for (bool safe = WK > 1; i0 < i1; safe = true) {
    f.pages(rows, i0 * KT, tid);
    f.codes(bk, h, pshift, i0 * KT, tid);
    f.pages(rows, (i0 + 1) * KT, tid);
    // The steps without a move are a loop of their own, in which the sums never leave their registers.  The waves of a
    // workgroup may be in different ones of the two; every step has the same barriers.
    for (unsigned i = i0; i < i1;) {
      step(i++, std::true_type());
      if constexpr (WK == 1)
        while (i < i1 && !safe && !st.wants_move()) step(i++, std::false_type());
    }
    if (WK > 1 || safe || !__syncthreads_or(st.lost())) break;
    st.clear();
  }
  st.spoil();

  if constexpr (WK > 1) {   // the four waves' results, joined through LDS by wave 0
    __syncthreads();
    st.template join<WK>((float*)sm, wave, lane);
    if (wave) return;
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int64_t c = c0 + n * 32 + col;
    if (c >= C) continue;
    const int64_t t = c / G;
    const int hq = h * G + (int)(c - t * G);
    if (splits == 1) {
      st.finish(n);
      store_column<DT, D>(out + (((size_t)b * T + t) * (size_t)(H * G) + hq) * D, half, st.o, n);
      if (lse && half == 0) lse[((size_t)b * (H * G) + hq) * T + t] = st.lse(n);
    } else {
      float* p = part + (((size_t)(b * H + h) * splits + split) * C + c) * (D + 2);
      store_partial<D>(p, half, st, n);
    }
  }
}

// How one call is cut: a plan of sizes alone, so that the workspace can be asked for beforehand.
struct Plan { bool few; int cw, kt, splits; int64_t groups; };
static constexpr int many_nb(int d, int nt) { return tile_waves(d, nt, 1, 2) == tile_waves(d, nt, 1, 1) ? 2 : 1; }
static constexpr int many_nw(int d, int nt) { return tile_waves(d, nt, 1, many_nb(d, nt)) >= 2 ? 8 : 4; }
static constexpr int many_kt(int d, int nt) { return many_nw(d, nt) == 8 && tile_lds(d, 128) <= 80 * 1024 ? 128 : 64; }
static Plan plan_of(const gpsr_bank* bk, int B, int table_pages, int T, int q_heads, int dtype) {
  Plan p;
  const int64_t C = (int64_t)T * (q_heads / bk->heads);
  const int nt = dtype == GPSR_BF16 ? 1 : dtype == GPSR_F16 ? 2 : 3, nw = many_nw(bk->dim, nt);
  p.few = C <= 32;
  p.cw = p.few ? 32 : 32 * nw;
  p.kt = p.few ? 128 : many_kt(bk->dim, nt);
  p.groups = (C + p.cw - 1) / p.cw;
  const int64_t tiles = (((int64_t)table_pages * bk->page_rows) + p.kt - 1) / p.kt;
  // the splits that end soonest when `slots` workgroups run at a time, each paying for 2 tiles besides its own
  const int64_t slots = p.few ? 512 : 256 * 4 * tile_waves(bk->dim, nt, 1, many_nb(bk->dim, nt)) / nw, wgs = p.groups * bk->heads * B;
  int64_t best = -1;
  p.splits = 1;
  for (int s = 1; s <= 64 && s <= (tiles > 1 ? tiles : 1); ++s) {
    const int64_t cost = ((wgs * s + slots - 1) / slots) * ((tiles + s - 1) / s + 2) + (s > 1 ? 2 + s / 4 : 0);
    if (best < 0 || cost < best) { best = cost; p.splits = s; }
  }
  return p;
}

extern "C" size_t gpsr_bank_attend_workspace_bytes(const gpsr_bank* bank, int B, int table_pages, int T, int q_heads, int dtype) {
  if (bank_wrong(bank) || B <= 0 || T <= 0 || table_pages < 0 || q_heads < 1 || q_heads % bank->heads || !type_ok(dtype)) return 0;
  const Plan p = plan_of(bank, B, table_pages, T, q_heads, dtype);
  return p.splits == 1 ? 0 : (size_t)p.splits * B * T * q_heads * (bank->dim + 2) * sizeof(float);
}

template <int DT, int BITS, int D>
static void launch_attend(const Plan& p, const gpsr_bank& bk, const int32_t* table, int B, int table_pages, const int32_t* length,
                          const void* q, int T, int G, Strides qs, bool qwide, float scale, const int32_t* skip, void* out,
                          float* lse, float* part, hipStream_t st) {
  typedef typename Row<DT>::T E;
  constexpr int NT = Terms<DT>::N, NW = many_nw(D, NT);
  const int pshift = __builtin_ctz((unsigned)bk.page_rows);
  const dim3 grid((unsigned)(p.groups * p.splits), (unsigned)bk.heads, (unsigned)B);
#define ATTEND(NW_, WK, KT, NB) hipLaunchKernelGGL((k_bank_attend<DT, BITS, D, NW_, WK, KT, NB>), grid, dim3(64 * NW_), 0, st, bk, table, \
    table_pages, pshift, length, (const E*)q, T, G, qs, qwide, scale, skip, (E*)out, lse, p.splits, part)
  if (p.few) ATTEND(4, 4, 128, 1); else ATTEND(NW, 1, many_kt(D, NT), many_nb(D, NT));
#undef ATTEND
  if (p.splits > 1) {
    const int64_t C = (int64_t)T * G;
    hipLaunchKernelGGL((k_bank_join<DT, D>), dim3((unsigned)((C + 3) / 4), (unsigned)bk.heads, (unsigned)B), dim3(256), 0, st, part,
                       T, G, bk.heads, C, p.splits, (size_t)p.splits * C, (size_t)1, (size_t)G, (size_t)C,
                       (E*)out, lse);
  }
}

extern "C" int gpsr_bank_attend(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* length,
                                const void* q, int dtype, int T, int q_heads, const int64_t* qst, float scale,
                                const int32_t* skip, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if (B <= 0 || T <= 0) return 0;
  if (const char* w = attend_wrong(bank, table, B, table_pages, length, q, dtype, q_heads, qst, scale, out)) return arg_fail(w);
  const Plan p = plan_of(bank, B, table_pages, T, q_heads, dtype);
  if (p.groups * p.splits > 0x7fffffff) return arg_fail("bank_attend: too many queries for one call");
  const size_t need = gpsr_bank_attend_workspace_bytes(bank, B, table_pages, T, q_heads, dtype);
  if (workspace_bytes < need || (need && !workspace)) return arg_fail("workspace too small");
  if (need && ((uintptr_t)workspace & 15)) return arg_fail("bank_attend: workspace must be 16-byte aligned");
  const Strides qs = {qst[0], qst[1], qst[2]};
  const bool wide = rows_wide(q, qst, dtype);
  const int G = q_heads / bank->heads;
  hipStream_t st = (hipStream_t)stream;
#define ATTEND(DT, BITS, D) launch_attend<DT, BITS, D>(p, *bank, table, B, table_pages, length, q, T, G, qs, wide, scale, skip, \
                                                       out, lse, (float*)workspace, st)
  BANK_DISPATCH(ATTEND, dtype, bank->bits, bank->dim);
#undef ATTEND
  CHECK_LAUNCH("k_bank_attend");
  return 0;
}
