// gpsr_bank_attend.hip -- example bank: attention over all rows (include/gpsr.h).
#include "gpsr_bank_tile.hpp"

// ---------------------------------------------------------------- attention over the whole bank
// Columns are the (query, head) pairs that share a bank head.  A workgroup of NW waves walks the rows of its split of the
// bank, KT at a time, NB x W of them in one step:
//   WK = 1 (many queries): all threads decode a tile to LDS once, then each wave multiplies it with W columns of its own.
//     Bound by the exponentials and the matrix units together: 40 000 queries of 100 000 rows x 64 columns 1140 to 1200 us, 855 to
//     900 TFLOP/s, where a library's product of 8192^3 reaches 1120.
//   WK = NW (few queries): all waves have the same columns, each walks every NW-th tile in LDS of its own, so that none waits
//     for another, and the results are joined at the end.  Bound by reading the bank and waiting for it: 12 queries to each of 8
//     banks of up to 180 000 rows x 128 columns in 4 bits, 154 MB, 62 us, 2.5 TB/s; the
//     longest bank's waves walk 22 tiles where the mean is 17, since all entries of a call share one number of splits.
// AHEAD: tiles under way besides the one in LDS.
template <int DT, int BITS, int D, int W, int NW, int WK, int KT, int NB, int AHEAD>
__global__ void __launch_bounds__(64 * NW, WK > 1 ? 2 : tile_waves(D, Terms<DT>::N, NB))
k_bank_attend(gpsr_bank bk, const int32_t* __restrict__ table, int table_pages, int pshift, const int32_t* __restrict__ length,
              const typename Row<DT>::T* __restrict__ q, int T, int G, Strides qs, bool qwide, float scale,
              const int32_t* __restrict__ skip, typename Row<DT>::T* __restrict__ out, float* __restrict__ lse, int splits,
              float* __restrict__ sums, f2v* __restrict__ stats) {
  typedef Geo<W> X;
  constexpr int NT = Terms<DT>::N, CW = (NW / WK) * W;           // columns of the workgroup
  constexpr int TH = WK > 1 ? 64 : 64 * NW;                      // threads that share a tile
  __shared__ __attribute__((aligned(16))) char sm[WK * tile_lds(D, KT)];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), part = lane / W, col = lane % W;
  const int sid = WK > 1 ? lane : tid;
  Tile<D, KT> tile(sm + (WK > 1 ? wave * tile_lds(D, KT) : 0));
  const int h = blockIdx.y, b = blockIdx.z, H = bk.heads;
  const int split = blockIdx.x % splits;
  const int64_t C = (int64_t)T * G, c = (int64_t)(blockIdx.x / splits) * CW + (WK == 1 ? wave * W : 0) + col;

  unsigned len = (unsigned)max(length[b], 0);
  const int64_t most = (int64_t)table_pages << pshift;
  if ((int64_t)len > most) len = (unsigned)most;
  const unsigned tiles = (len + KT - 1) / KT;
  const unsigned per = (tiles + splits - 1) / splits;
  const unsigned i0 = min(per * split, tiles), i1 = min(i0 + per, tiles);

  // this lane's column: its query as operand fragments, and what it skips
  const bool there = c < C;
  const int64_t t = there ? c / G : 0;
  const int hq = h * G + (there ? (int)(c - t * G) : 0);
  bf8 qf[NT][D / X::STEP];
  load_query<DT, D, W>(q + b * qs.b + t * qs.t + (int64_t)hq * qs.h, qwide, there, part, qf);
  unsigned lo = 0, hi = 0;
  if (skip && there) {
    const int32_t* s = skip + ((size_t)b * T + t) * 2;
    lo = (unsigned)max(s[0], 0); hi = (unsigned)max(s[1], 0);
  }
  Soft<D, W> st;
  const float c2 = scale * 1.4426950408889634f;

  tile.clear_marks(sid, TH);
  std::conditional_t<(WK > 1), WaveFetch<BITS, D>, Fetch<BITS, D, KT, TH>> f[AHEAD];
  const WholeBank rows = {table + (size_t)b * table_pages, bk.pages, pshift, len};
  // between the accesses to a tile: LDS serves one wave in order, only the compiler has to be kept from moving them
  const auto sync = [] { if constexpr (WK > 1) { asm volatile("" ::: "memory"); __builtin_amdgcn_wave_barrier(); } else __syncthreads(); };
  const auto pages = [&](auto& f, unsigned i) { if constexpr (WK > 1) f.pages(rows, i * KT); else f.pages(rows, i * KT, sid); };
  const auto codes = [&](auto& f, unsigned i) {
    if constexpr (WK > 1) f.codes(bk, h, pshift, i * KT, len, sid); else f.codes(bk, h, pshift, i * KT, sid);
  };
  // 0, or 32 in a second walk (Soft::lost), which any 2^31 rows bear; not always 32, because products with values near 2^-100
  // would leave the range at its other end
  float above = 0.f;
  const auto step = [&](unsigned i, auto& f, auto move) {
    sync();
    f.template store<W>(tile, sid, i + 1);
    sync();
    codes(f, i + WK * AHEAD);
    pages(f, i + 2 * WK * AHEAD);
    const unsigned p0 = i * KT;
    tile_marks<D, KT, KT>(tile, 0, i + 1, st, [&](int r) { return !(p0 + r >= lo && p0 + r < hi); });
    const bool weightless = tile.weightless(i + 1);
    const bool skips = skip && __ballot(lo < p0 + KT && hi > p0 && lo < hi);
#pragma unroll 1
    for (int r = 0; r < KT; r += W * NB) {
      typename X::Acc s[NB];
      tile_logits<D, KT, NT, NB, W>(tile, r, col, part, weightless, qf, s);
      if (skips) {
        asm volatile("");        // not to be computed for the tiles that nobody skips
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int e = 0; e < X::E; ++e) {
            const unsigned pos = p0 + r + kb * W + X::row(part, e);
            if (pos >= lo && pos < hi) s[kb][e] = -__builtin_inff();
          }
      }
      tile_accumulate<D, KT, (WK > 1 ? weight_terms(NT) : NT), NB, W, decltype(move)::value>(tile, r, col, part, c2, above, s, st);
    }
  };
  st.clear();
#pragma unroll 1
  for (; i0 < i1; above = 32.f) {
    const unsigned first = i0 + (WK > 1 ? wave : 0);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      pages(f[a], first + WK * a);
      codes(f[a], first + WK * a);
      pages(f[a], first + WK * (AHEAD + a));
    }
    if constexpr (WK > 1) {
      for (unsigned i = first; i < i1; i += WK * AHEAD)
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
          if (i + WK * a < i1) step(i + WK * a, f[a], std::true_type());
      if (above != 0.f || !__ballot(st.lost())) break;
    } else {
      static_assert(AHEAD == 1, "one tile under way");
      // The steps without a move are a loop of their own, in which the sums never leave their registers.  The waves of a
      // workgroup may be in different ones of the two; every step has the same barriers.
      for (unsigned i = i0; i < i1;) {
        step(i++, f[0], std::true_type());
        while (i < i1 && above == 0.f && !st.wants_move()) step(i++, f[0], std::false_type());
      }
      if (above != 0.f || !__syncthreads_or(st.lost())) break;
    }
    st.clear();
  }
  st.spoil();

  if constexpr (WK > 1) {   // the waves' results, joined through LDS by wave 0
    __syncthreads();
    st.template join<WK>((float*)sm, wave, lane);
    if (wave) return;
  }
  if (!there) return;
  if (splits == 1) {
    st.finish();
    st.template store<DT>(out + (((size_t)b * T + t) * (size_t)(H * G) + hq) * D, part);
    if (lse && part == 0) lse[((size_t)b * (H * G) + hq) * T + t] = st.lse();
  } else {
    const size_t at = ((size_t)(b * H + h) * splits + split) * C + c;
    st.store_partial(sums + at * D, stats + at, part);
  }
}

// How one call is cut: a plan of sizes alone, so that the workspace can be asked for beforehand.
struct Plan { bool few, lone; int cw, kt, splits; int64_t groups; };
static constexpr int many_nb(int d, int nt) { return tile_waves(d, nt, 2) == tile_waves(d, nt, 1) ? 2 : 1; }
static constexpr int many_nw(int d, int nt) { return tile_waves(d, nt, many_nb(d, nt)) >= 2 ? 8 : 4; }
// 128 rows a tile where one or two workgroups of it fit a CU; 64 where the query terms leave too few registers to have more under way
// (96 columns in f16 862 against 892 us, in f32 95 against 105; 64 columns in f32 553 against 527)
static constexpr int many_kt(int d, int nt) { return many_nw(d, nt) == 8 && tile_lds(d, 128) <= 80 * 1024 && (d < 96 || nt == 1) ? 128 : 64; }
// whether there is a form with half the waves and twice the registers (plan_of says when it is taken)
static constexpr bool lone_nb(int d, int nt) { return tile_waves(d, nt, 1) == 4 && tile_waves(d, nt, 2) == 2; }
// tiles under way for up to 16 columns: two where the registers hold them (96 columns: a thread with keys and values by turns, which
// the compiler keeps in memory)
static constexpr int few_ahead(int d, int bits, int nt) { return d * bits <= 512 && d != 96 ? 2 : 1; }
static Plan plan_of(const gpsr_bank* bk, int B, int table_pages, int T, int q_heads, int dtype) {
  Plan p;
  const int64_t C = (int64_t)T * (q_heads / bk->heads);
  const int nt = dtype == GPSR_BF16 ? 1 : dtype == GPSR_F16 ? 2 : 3, nw = many_nw(bk->dim, nt);
  p.few = C <= 32;
  p.lone = false;
  p.cw = p.few ? 32 : 32 * nw;
  p.kt = p.few ? 32 : many_kt(bk->dim, nt);
  p.groups = (C + p.cw - 1) / p.cw;
  const int64_t tiles = (((int64_t)table_pages * bk->page_rows) + p.kt - 1) / p.kt;
  // The splits that end soonest when `slots` workgroups run at a time, each paying for `own` tiles besides its share, and the join
  // for some more; behind 64 of them, which one wave joins, four waves do, and the partials' way to memory and back counts (some
  // 4 MB for a tile's time): 1 query of 100 000 rows 21 us instead of 30, 256 queries 43 instead of 63.
  const int64_t wgs = p.groups * bk->heads * B;
  const int64_t slots = p.few ? 512 : 256 * 4 * tile_waves(bk->dim, nt, many_nb(bk->dim, nt)) / nw;
  const int step = p.few ? 4 : 1, own = p.few ? 4 : 2;           // tiles that a workgroup takes at once
  int64_t best = -1;
  p.splits = 1;
  for (int s = 1; s <= 256 && s * step <= (tiles > step ? tiles + step - 1 : step); s += s < 64 ? 1 : 32) {
    const int64_t join = s == 1 ? 0 : s <= 64 ? 2 + s / 4 : 5 + s / 16 + C * bk->heads * B * (s - 64) * bk->dim / 500000;
    const int64_t cost = ((wgs * s + slots - 1) / slots) * ((tiles + s * step - 1) / (s * step) + own) + join;
    if (best < 0 || cost < best) { best = cost; p.splits = s; }
  }
  // Or one workgroup on each CU with 64 rows at a time in twice the registers.  At 64 columns a tile of 128 rows takes a CU's two
  // workgroups of 4 waves a SIMD 4.4 us (and starting and ending one as much as 4 tiles), the lone one 2.95; partials cost 0.13 ns
  // a column and split, and the join 10 us.  So it pays where the columns just fill the CUs and the bank is short: 65 025 queries
  // of 5000 rows 137 us instead of 150, of 1000 rows 37 instead of 68 (but 40 000 of 100 000 rows 1470 instead of 1150).  The other form
  // that has both, 32 columns in f32, keeps their ratio: 40 000 to 131 072 queries of 1000 to 20 000 rows up to 35 % sooner at 1000 and
  // 2500 rows and within 4 % elsewhere, but for 40 000 of 2500 (98 instead of 91) and 50 000 of 5000 (189 instead of 171).
  if (!p.few && lone_nb(bk->dim, nt) && p.splits > 1) {
    const double split = ((wgs * p.splits + slots - 1) / slots) * ((tiles + p.splits - 1) / p.splits + 4) * 4.4 + 10 + 0.13e-3 * (double)C * bk->heads * B * p.splits;
    const double lone = ((wgs + 255) / 256) * (tiles + own) * 2.95;
    if (lone < split) { p.lone = true; p.splits = 1; }
  }
  return p;
}

extern "C" size_t gpsr_bank_attend_workspace_bytes(const gpsr_bank* bank, int B, int table_pages, int T, int q_heads, int dtype) {
  if (bank_wrong(bank) || B <= 0 || T <= 0 || table_pages < 0 || q_heads < 1 || q_heads % bank->heads || !type_ok(dtype)) return 0;
  const Plan p = plan_of(bank, B, table_pages, T, q_heads, dtype);
  return p.splits == 1 ? 0 : (size_t)p.splits * B * T * q_heads * (bank->dim * sizeof(float) + sizeof(f2v));
}

template <int DT, int BITS, int D>
static void launch_attend(const Plan& p, const gpsr_bank& bk, const int32_t* table, int B, int table_pages, const int32_t* length,
                          const void* q, int T, int G, Strides qs, bool qwide, float scale, const int32_t* skip, void* out,
                          float* lse, void* ws, hipStream_t st) {
  typedef typename Row<DT>::T E;
  float* sums = (float*)ws;          // every row a multiple of 128 bytes: the statistics behind them stay aligned
  f2v* stats = (f2v*)(sums + (size_t)p.splits * B * T * G * bk.heads * D);
  constexpr int NT = Terms<DT>::N, NW = many_nw(D, NT);
  const int pshift = __builtin_ctz((unsigned)bk.page_rows);
  const dim3 grid((unsigned)(p.groups * p.splits), (unsigned)bk.heads, (unsigned)B);
#define ATTEND(W, NW_, WK, KT, NB, AHEAD) hipLaunchKernelGGL((k_bank_attend<DT, BITS, D, W, NW_, WK, KT, NB, AHEAD>), grid, \
    dim3(64 * NW_), 0, st, bk, table, table_pages, pshift, length, (const E*)q, T, G, qs, qwide, scale, skip, (E*)out, lse, p.splits, sums, stats)
  if (p.few && (int64_t)T * G <= 16) ATTEND(16, 4, 4, 32, 2, few_ahead(D, BITS, NT));
  else if (p.few) ATTEND(32, 4, 4, 32, 1, 1);
  else if (!p.lone) ATTEND(32, NW, 1, many_kt(D, NT), many_nb(D, NT), 1);
  else if constexpr (lone_nb(D, NT)) ATTEND(32, NW, 1, many_kt(D, NT), 2, 1);
#undef ATTEND
  if (p.splits > 1) {
    const int64_t C = (int64_t)T * G;
#define JOIN(WJ, wgs) hipLaunchKernelGGL((k_bank_join<DT, D, WJ>), dim3((unsigned)(wgs), (unsigned)bk.heads, (unsigned)B), dim3(256), \
    0, st, sums, stats, T, G, bk.heads, C, p.splits, (size_t)p.splits * C, (size_t)1, (size_t)G, (size_t)C, (E*)out, lse)
    if (p.splits <= 64) JOIN(1, (C + 3) / 4); else JOIN(4, C);
#undef JOIN
  }
}

extern "C" int gpsr_bank_attend(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* length,
                                const void* q, int dtype, int T, int q_heads, const int64_t* qst, float scale,
                                const int32_t* skip, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if (B <= 0 || T <= 0) return 0;
  if (const char* w = attend_wrong(bank, table, B, table_pages, length, q, dtype, q_heads, qst, scale, out)) return arg_fail(w);
  const Plan p = plan_of(bank, B, table_pages, T, q_heads, dtype);
  if (!grid_fits(p.groups * p.splits, 512) || !grid_fits(((int64_t)T * (q_heads / bank->heads) + 3) / 4, 256)) return arg_fail("bank_attend: too many queries for one call");
  const size_t need = gpsr_bank_attend_workspace_bytes(bank, B, table_pages, T, q_heads, dtype);
  if (workspace_bytes < need || (need && !workspace)) return arg_fail("workspace too small");
  if (need && ((uintptr_t)workspace & 15)) return arg_fail("bank_attend: workspace must be 16-byte aligned");
  const Strides qs = {qst[0], qst[1], qst[2]};
  const bool wide = rows_wide(q, qst, dtype);
  const int G = q_heads / bank->heads;
  hipStream_t st = (hipStream_t)stream;
#define ATTEND(DT, BITS, D) launch_attend<DT, BITS, D>(p, *bank, table, B, table_pages, length, q, T, G, qs, wide, scale, skip, \
                                                       out, lse, workspace, st)
  BANK_DISPATCH(ATTEND, dtype, bank->bits, bank->dim);
#undef ATTEND
  CHECK_LAUNCH("k_bank_attend");
  return 0;
}
