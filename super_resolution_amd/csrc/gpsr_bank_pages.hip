// gpsr_bank_pages.hip -- example bank: attention over chosen pages (include/gpsr.h).
//
// Two ways through the same mathematics:
//   by query (7 us for one query and 16 pages): a workgroup per query walks that query's pages, its four waves 32 rows each against the query's heads.  Nothing
//     is shared, 31 of 32 columns of the matrix instructions idle (one head), but it takes one or two launches.
//   by page: the choices are turned over (for each page the list of queries that chose it), a workgroup takes one page and
//     128 of its queries, writes each query's partial result for that page, and a last kernel joins each query's partials.
//     Pages are decoded once per 128 queries and all columns work, at the price of writing and reading the partials: 40 000
//     queries with 16 pages each 129 us (count 14, shares 10, scan 5, fill 8, products 73, join 26), by query 4380.  Partials are
//     f32 whatever the caller's type: their sums are weighed against each other by their keys alone, and a column may be any
//     number of powers of two under its neighbours (in f16 with a power of two a row, products took 59 and the join 19 us, but
//     columns 2^-25 under the row's largest became zero).
// Within a chunk of choices the lists' order comes from counters in LDS and may differ from run to run; a partial does not depend
// on its place in a list, and the join runs in the order of the caller's numbers: results do not change.
#include "gpsr_bank_tile.hpp"

#include <cmath>

// A query's rows are at most 64 pages of 256, so with weights of at most 2^-15 sums of any values stay in float32's range, and
// products of the smallest held values (2^-111 in 4 bits) with the largest weights as well.
static constexpr float ABOVE = 15.f;

// ---------------------------------------------------------------- by query
template <int DT, int BITS, int D, int W>
__global__ void __launch_bounds__(256, 2)
k_bank_pages_query(gpsr_bank bk, const int32_t* __restrict__ table, int table_pages, int pshift, const int32_t* __restrict__ length,
                   const typename Row<DT>::T* __restrict__ q, int T, int G, Strides qs, bool qwide, const int32_t* __restrict__ sel,
                   int n_sel, float scale, const int32_t* __restrict__ skip, typename Row<DT>::T* __restrict__ out,
                   float* __restrict__ lse, int groups, int splits, float* __restrict__ sums, f2v* __restrict__ stats) {
  typedef Geo<W> X;
  constexpr int NT = Terms<DT>::N, KT = 128, NB = 32 / W;
  __shared__ __attribute__((aligned(16))) char sm[tile_lds(D, KT)];
  __shared__ int phys[64], rown[64], first[64], total;
  Tile<D, KT> tile(sm);
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), part = lane / W, col = lane % W;
  const int h = blockIdx.y, b = blockIdx.z, H = bk.heads, P = 1 << pshift;
  const int split = blockIdx.x % splits, group = blockIdx.x / splits % groups;
  const int64_t t = blockIdx.x / splits / groups;
  const int wrow = wave * 32;

  // the pages that exist, have rows, and were not named before, in the caller's order
  if (tid < 64) {
    const int64_t len = length[b];
    const int32_t* mine = sel + (((size_t)b * T + t) * H + h) * n_sel;
    const int lp = tid < n_sel ? mine[tid] : -1;
    bool ok = (unsigned)lp < (unsigned)table_pages && (int64_t)lp * P < len;
    int p = -1;
    if (ok) { p = table[(size_t)b * table_pages + lp]; ok = (unsigned)p < (unsigned)bk.pages; }
    for (int i = 0; i + 1 < n_sel; ++i) { const int o = __shfl(lp, i); ok = ok && !(i < tid && o == lp); }
    const unsigned long long all = __ballot(ok);
    if (ok) {
      const int at = __popcll(all & ((1ull << tid) - 1));
      phys[at] = p; first[at] = lp; rown[at] = (int)min((int64_t)P, len - (int64_t)lp * P);
    }
    if (tid == 0) total = __popcll(all);
  }
  tile.clear_marks(tid, 256);
  const int g = group * W + col;
  const bool there = g < G;
  bf8 qf[NT][D / X::STEP];
  load_query<DT, D, W>(q + b * qs.b + t * qs.t + (int64_t)(h * G + (there ? g : 0)) * qs.h, qwide, there, part, qf);
  const int64_t lo = skip ? skip[((size_t)b * T + t) * 2] : 0, hi = skip ? skip[((size_t)b * T + t) * 2 + 1] : 0;
  Soft<D, W> st;
  st.clear();
  const float c2 = scale * 1.4426950408889634f;
  __syncthreads();
  const PageList rows = {phys, rown, pshift, (unsigned)total};
  const unsigned tiles = (((unsigned)total << pshift) + KT - 1) / KT, per = (tiles + splits - 1) / splits;
  const unsigned i0 = min(per * split, tiles), i1 = min(i0 + per, tiles);
  Fetch<BITS, D, KT, 256> f;
  if (i0 < i1) {
    f.pages(rows, i0 * KT, tid);
    f.codes(bk, h, pshift, i0 * KT, tid);
    f.pages(rows, (i0 + 1) * KT, tid);
  }
  for (unsigned i = i0; i < i1; ++i) {
    __syncthreads();
    f.template store<W>(tile, tid, i + 1);
    __syncthreads();
    f.codes(bk, h, pshift, (i + 1) * KT, tid);
    f.pages(rows, (i + 2) * KT, tid);
    const auto skips = [&](unsigned v) {
      const unsigned slot = v >> pshift;
      const int64_t pos = slot < (unsigned)total ? (int64_t)first[slot] * P + (v & (P - 1)) : -1;
      return pos >= lo && pos < hi;
    };
    tile_marks<D, KT, 32>(tile, wrow, i + 1, st, [&](int r) { return !skips(i * KT + wrow + r); });
    typename X::Acc s[NB];
    tile_logits<D, KT, NT, NB, W>(tile, wrow, col, part, tile.weightless(i + 1), qf, s);
    if (lo < hi) {
      asm volatile("");
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int e = 0; e < X::E; ++e)
          if (skips(i * KT + wrow + kb * W + X::row(part, e))) s[kb][e] = -__builtin_inff();
    }
    tile_accumulate<D, KT, weight_terms(NT), NB, W, true>(tile, wrow, col, part, c2, ABOVE, s, st);
  }
  st.spoil();
  __syncthreads();
  st.template join<4>((float*)sm, wave, lane);
  if (wave || !there) return;
  const int hq = h * G + g;
  if (splits == 1) {
    st.finish();
    st.template store<DT>(out + (((size_t)b * T + t) * (size_t)(H * G) + hq) * D, part);
    if (lse && part == 0) lse[((size_t)b * (H * G) + hq) * T + t] = st.lse();
  } else {
    const size_t at = (((size_t)(b * H + h) * T + t) * splits + split) * G + g;
    st.store_partial(sums + at * D, stats + at, part);
  }
}

// ---------------------------------------------------------------- by page
// The choices of one entry are cut into chunks of PG_CHUNK.  A chunk counts its own in LDS (bucket: bank head and logical page)
// and writes its histogram; a choice keeps its place within its chunk's share of the list, -1 if it is passed over.  Counting
// through global atomics instead took 59 us for 640 000 choices of 1563 pages; counts 14 and shares 10 us this way.
#define PG_CHUNK 4096
#define PG_BUCKETS 16384      // of one entry: 64 KB of LDS
__global__ void __launch_bounds__(512)
k_bank_pages_count(const int32_t* __restrict__ sel, int n_sel, const int32_t* __restrict__ table, int table_pages, int64_t pages,
                   int pshift, const int32_t* __restrict__ length, int T, int H, int G, int chunks, int* __restrict__ hist,
                   int* __restrict__ rank, f2v* __restrict__ stats) {
  extern __shared__ int mine[];
  const int b = blockIdx.y, tid = threadIdx.x, buckets = H * table_pages;
  const int64_t per = (int64_t)T * H * n_sel, e0 = (int64_t)blockIdx.x * PG_CHUNK;
  for (int i = tid; i < buckets; i += 512) mine[i] = 0;
  __syncthreads();
  const int64_t len = length[b];
  const int32_t* s0 = sel + b * per;
  for (int i = tid; i < PG_CHUNK && e0 + i < per; i += 512) {
    const int64_t e = e0 + i, th = e / n_sel;
    const int s = (int)(e - th * n_sel), h = (int)(th % H);
    const int lp = s0[e];
    bool ok = (unsigned)lp < (unsigned)table_pages && ((int64_t)lp << pshift) < len;
    if (ok) ok = (uint64_t)(int64_t)table[(size_t)b * table_pages + lp] < (uint64_t)pages;
#pragma unroll 4
    for (int k = 1; k <= s; ++k) ok &= s0[e - k] != lp;      // all of them, so that the loads do not wait for each other
    rank[b * per + e] = ok ? atomicAdd(&mine[h * table_pages + lp], 1) : -1;
    if (!ok)      // the join passes over partials whose sum of weights is 0
      for (int g = 0; g < G; ++g) stats[((((size_t)b * H + h) * T + th / H) * n_sel + s) * G + g] = f2v{0.f, 0.f};
  }
  __syncthreads();
  int* to = hist + ((size_t)b * chunks + blockIdx.x) * buckets;
  for (int i = tid; i < buckets; i += 512) to[i] = mine[i];
}

// each bucket's counts become the places at which the chunks' shares start, and their sum
__global__ void __launch_bounds__(64)
k_bank_pages_shares(int* __restrict__ hist, int buckets, int chunks, int* __restrict__ count) {
  const int i = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (i >= buckets) return;
  int* p = hist + (size_t)b * chunks * buckets + i;
  int sum = 0;
  for (int c0 = 0; c0 < chunks; c0 += 32) {
    int n[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) n[j] = c0 + j < chunks ? p[(size_t)(c0 + j) * buckets] : 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      if (c0 + j < chunks) p[(size_t)(c0 + j) * buckets] = sum;
      sum += n[j];
    }
  }
  count[(size_t)b * buckets + i] = sum;
}

// exclusive sums of the counts and of the workgroups that each bucket needs, and each workgroup's bucket (found by bisection
// over the sums instead, it was a third of the product kernel's time); one workgroup
__global__ void __launch_bounds__(1024)
k_bank_pages_scan(const int* __restrict__ count, int buckets, int G, int cw, int* __restrict__ start, int* __restrict__ wgs,
                  int* __restrict__ owner) {
  __shared__ int sc[16], sw[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid);
  const int per = (buckets + 1023) / 1024;
  const int i0 = min(tid * per, buckets), i1 = min(i0 + per, buckets);
  int c = 0, w = 0;
  for (int i = i0; i < i1; ++i) { const int n = count[i]; c += n; w += (int)(((int64_t)n * G + cw - 1) / cw); }
  int pc = c, pw = w;
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(pc, o), d = __shfl_up(pw, o);
    if (lane >= o) { pc += a; pw += d; }
  }
  if (lane == 63) { sc[wave] = pc; sw[wave] = pw; }
  __syncthreads();
  for (int i = 0; i < wave; ++i) { pc += sc[i]; pw += sw[i]; }
  int oc = pc - c, ow = pw - w;
  for (int i = i0; i < i1; ++i) {
    start[i] = oc; wgs[i] = ow;
    const int n = count[i];
    oc += n;
    for (int k = (int)(((int64_t)n * G + cw - 1) / cw); k > 0; --k) owner[ow++] = i;
  }
  if (tid == 1023) { start[buckets] = pc; wgs[buckets] = pw; }
}

__global__ void __launch_bounds__(256)
k_bank_pages_fill(const int32_t* __restrict__ sel, int n_sel, int table_pages, int T, int H, int chunks, const int* __restrict__ hist,
                  const int* __restrict__ rank, const int* __restrict__ start, int* __restrict__ list) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)T * H * n_sel;
  const int b = blockIdx.y;
  if (e >= per) return;
  const int r = rank[b * per + e];
  if (r < 0) return;
  const int64_t th = e / n_sel;
  const int bucket = (int)(th % H) * table_pages + sel[b * per + e], buckets = H * table_pages;
  const int share = hist[((size_t)b * chunks + e / PG_CHUNK) * buckets + bucket];
  list[start[(size_t)b * buckets + bucket] + share + r] = (int)(th / H * n_sel + (e - th * n_sel));
}

// 32 rows at a time and three waves per SIMD: the workgroups are short and mostly wait (73 us for 40 000 queries x 16 pages of
// 64 rows of 64 columns, 144 TFLOP/s; measured with f16 partials, at 59 us, all 64 rows of a page at a time took 4 us more, two
// waves 15 more, four with spills 30 more)
template <int DT, int BITS, int D, int KT>
__global__ void __launch_bounds__(256, tile_waves(D, Terms<DT>::N, 1) > 3 ? 3 : tile_waves(D, Terms<DT>::N, 1))
k_bank_pages_page(gpsr_bank bk, const int32_t* __restrict__ table, int table_pages, int pshift, const int32_t* __restrict__ length,
                  const typename Row<DT>::T* __restrict__ q, int T, int G, Strides qs, bool qwide, int n_sel, float scale,
                  const int32_t* __restrict__ skip, const int* __restrict__ start, const int* __restrict__ wgs, int buckets,
                  const int* __restrict__ owner, const int* __restrict__ list, float* __restrict__ sums, f2v* __restrict__ stats) {
  constexpr int NT = Terms<DT>::N, NB = 1, CW = 128, W = 32;
  typedef Geo<W> X;
  __shared__ __attribute__((aligned(16))) char sm[tile_lds(D, KT)];
  Tile<D, KT> tile(sm);
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), part = lane / W, col = lane % W;
  const int w = blockIdx.x;
  const int a = owner[w];                 // of a workgroup behind the last one: whatever the memory held, and not used
  if (w >= wgs[buckets]) return;
  const int lp = a % table_pages, H = bk.heads, P = 1 << pshift;
  const int bh = a / table_pages, h = bh % H, b = bh / H;
  const int n = start[a + 1] - start[a];
  const int64_t c = (int64_t)(w - wgs[a]) * CW + wave * 32 + col;
  const bool there = c < (int64_t)n * G;
  const int id = there ? list[start[a] + (int)(c / G)] : 0, g = (int)(c % G);
  const int t = id / n_sel;
  bf8 qf[NT][D / X::STEP];
  load_query<DT, D>(q + b * qs.b + t * qs.t + (int64_t)(h * G + (there ? g : 0)) * qs.h, qwide, there, part, qf);
  int64_t lo = 0, hi = 0;
  if (skip && there) { lo = skip[((size_t)b * T + t) * 2]; hi = skip[((size_t)b * T + t) * 2 + 1]; }
  const int64_t pos0 = (int64_t)lp << pshift;
  const OnePage rows = {table[(size_t)b * table_pages + lp], (int)min((int64_t)P, length[b] - pos0)};
  Soft<D, W> st;
  st.clear();
  const float c2 = scale * 1.4426950408889634f;
  tile.clear_marks(tid, 256);
  Fetch<BITS, D, KT, 256> f;
  f.pages(rows, 0, tid);
  f.codes(bk, h, pshift, 0, tid);
  for (int v = 0; v < rows.rows; v += KT) {
    __syncthreads();
    f.template store<W>(tile, tid, v / KT + 1);
    __syncthreads();
    f.pages(rows, v + KT, tid);
    f.codes(bk, h, pshift, v + KT, tid);
    tile_marks<D, KT, KT>(tile, 0, v / KT + 1, st, [&](int r) { return !(pos0 + v + r >= lo && pos0 + v + r < hi); });
    const bool weightless = tile.weightless(v / KT + 1);
#pragma unroll 1
    for (int r = 0; r < KT; r += 32) {
      typename X::Acc s[NB];
      tile_logits<D, KT, NT, NB, W>(tile, r, col, part, weightless, qf, s);
      if (skip && __ballot(lo < pos0 + v + KT && hi > pos0 + v && lo < hi)) {
        asm volatile("");
#pragma unroll
        for (int e = 0; e < X::E; ++e) {
          const int64_t pos = pos0 + v + r + X::row(part, e);
          if (pos >= lo && pos < hi) s[0][e] = -__builtin_inff();
        }
      }
      tile_accumulate<D, KT, weight_terms(NT), NB, W, true>(tile, r, col, part, c2, ABOVE, s, st);
    }
  }
  st.spoil();
  const size_t at = ((size_t)bh * T * n_sel + id) * G + g;
  if (there) st.store_partial(sums + at * D, stats + at, part);
}

// ---------------------------------------------------------------- host
struct PagesPlan { bool by_page; int groups, splits, chunks; int64_t entries, buckets, most_wgs; size_t hist, rank, start, wgs, owner, list, stats, sums, bytes; };
static PagesPlan plan_of(const gpsr_bank* bk, int B, int table_pages, int T, int q_heads, int n_sel) {
  PagesPlan p = {};
  const int H = bk->heads, G = q_heads / H;
  p.entries = (int64_t)B * T * H * n_sel;
  p.buckets = (int64_t)B * H * table_pages;
  // By page where that is sooner.  A query (and 16 or 32 of its heads) costs 4 ns and 15 ps a row at 64 columns; by page, six
  // launches 25 us more, a page 6.5 ns and a choice 0.08 ns; more columns cost (dim / 64)^1.5 times as much.  Both sides measured for
  // 256 to 8192 queries of 4 or 16 pages, 16 or 64 rows, 32 to 6250 pages, 64 and 256 columns: 2048 queries of 16 x 64 rows
  // 49 us by query, 50 by page (1563 pages); 512 queries 20 and 44; 512 queries of 256 columns 95 and 121, 1024 190 and 125; 8192
  // queries of 16 x 16 rows of 6250 pages 72 and 86.
  const int width = G <= 16 ? 16 : 32;
  p.groups = (G + width - 1) / width;
  const double wide = bk->dim / 64.0 * sqrt(bk->dim / 64.0);
  const double by_query = wide * (double)B * T * H * p.groups * (4e-3 + 15e-6 * n_sel * bk->page_rows);
  const double by_page = 25 + wide * (6.5e-3 * (double)(p.buckets < p.entries ? p.buckets : p.entries) + 0.08e-3 * (double)p.entries * G);
  p.by_page = by_query > by_page && p.buckets > 0 && p.entries <= 0x7fffffff && (int64_t)H * table_pages <= PG_BUCKETS && p.buckets <= (1 << 24);
  if (p.by_page) {
    p.most_wgs = p.entries * G / 128 + (p.buckets < p.entries ? p.buckets : p.entries);
    p.chunks = (int)(((int64_t)T * H * n_sel + PG_CHUNK - 1) / PG_CHUNK);
    size_t at = align256((size_t)p.buckets * 4);
    p.hist = at; at += align256((size_t)p.chunks * p.buckets * 4);
    p.rank = at; at += align256((size_t)p.entries * 4);
    p.start = at; at += align256((size_t)(p.buckets + 1) * 4);
    p.wgs = at; at += align256((size_t)(p.buckets + 1) * 4);
    p.owner = at; at += align256((size_t)p.most_wgs * 4);
    p.list = at; at += align256((size_t)p.entries * 4);
    p.stats = at; at += align256((size_t)p.entries * G * sizeof(f2v));
    p.sums = at; at += (size_t)p.entries * G * bk->dim * sizeof(float);
    p.bytes = at;
  } else {
    const int64_t wgs = (int64_t)B * T * H * p.groups, tiles = ((int64_t)n_sel * bk->page_rows + 127) / 128;
    int64_t s = 512 / wgs;
    if (s < 1) s = 1;
    p.splits = (int)(s > tiles ? tiles : s);
    if (p.splits > 1) p.bytes = (size_t)p.splits * B * T * q_heads * (bk->dim * sizeof(float) + sizeof(f2v));
  }
  return p;
}

extern "C" size_t gpsr_bank_attend_pages_workspace_bytes(const gpsr_bank* bank, int B, int table_pages, int T, int q_heads, int n_sel, int dtype) {
  if (bank_wrong(bank) || B <= 0 || T <= 0 || table_pages < 0 || q_heads < 1 || q_heads % bank->heads || n_sel < 1 || n_sel > 64 || !type_ok(dtype)) return 0;
  return plan_of(bank, B, table_pages, T, q_heads, n_sel).bytes;
}

template <int DT, int BITS, int D>
static void launch_pages(const PagesPlan& p, const gpsr_bank& bk, const int32_t* table, int B, int table_pages, const int32_t* length,
                         const void* q, int T, int q_heads, Strides qs, bool qwide, const int32_t* sel, int n_sel, float scale,
                         const int32_t* skip, void* out, float* lse, char* ws, hipStream_t st) {
  typedef typename Row<DT>::T E;
  const int pshift = __builtin_ctz((unsigned)bk.page_rows), H = bk.heads, G = q_heads / H;
  const int64_t C = (int64_t)T * G;
  const dim3 join((unsigned)((C + 3) / 4), (unsigned)H, (unsigned)B);
  if (!p.by_page) {
    float* sums = (float*)ws;
    f2v* stats = (f2v*)(sums + (size_t)p.splits * B * T * q_heads * D);
#define QUERY(W) hipLaunchKernelGGL((k_bank_pages_query<DT, BITS, D, W>), dim3((unsigned)((int64_t)T * p.groups * p.splits), (unsigned)H, \
    (unsigned)B), dim3(256), 0, st, bk, table, table_pages, pshift, length, (const E*)q, T, G, qs, qwide, sel, n_sel, scale, skip, (E*)out, \
    lse, p.groups, p.splits, sums, stats)
    if (G <= 16) QUERY(16); else QUERY(32);
#undef QUERY
    if (p.splits > 1)
      hipLaunchKernelGGL((k_bank_join<DT, D>), join, dim3(256), 0, st, sums, stats, T, G, H, C, p.splits, (size_t)p.splits * C, (size_t)1,
                         (size_t)p.splits * G, (size_t)G, (E*)out, lse);
    return;
  }
  int *count = (int*)ws, *rank = (int*)(ws + p.rank), *start = (int*)(ws + p.start), *wgs = (int*)(ws + p.wgs), *list = (int*)(ws + p.list);
  float* sums = (float*)(ws + p.sums);
  f2v* stats = (f2v*)(ws + p.stats);
  int* owner = (int*)(ws + p.owner);
  const int64_t per = (int64_t)T * H * n_sel;
  const int buckets = H * table_pages;
  int* hist = (int*)(ws + p.hist);
  hipLaunchKernelGGL(k_bank_pages_count, dim3((unsigned)p.chunks, (unsigned)B), dim3(512), (size_t)buckets * 4, st, sel, n_sel, table,
                     table_pages, bk.pages, pshift, length, T, H, G, p.chunks, hist, rank, stats);
  hipLaunchKernelGGL(k_bank_pages_shares, dim3((unsigned)((buckets + 63) / 64), (unsigned)B), dim3(64), 0, st, hist, buckets, p.chunks, count);
  hipLaunchKernelGGL(k_bank_pages_scan, dim3(1), dim3(1024), 0, st, count, (int)p.buckets, G, 128, start, wgs, owner);
  hipLaunchKernelGGL(k_bank_pages_fill, dim3((unsigned)((per + 255) / 256), (unsigned)B), dim3(256), 0, st, sel, n_sel, table_pages, T,
                     H, p.chunks, hist, rank, start, list);
#define PAGE(KT) hipLaunchKernelGGL((k_bank_pages_page<DT, BITS, D, KT>), dim3((unsigned)p.most_wgs), dim3(256), 0, st, bk, table, \
    table_pages, pshift, length, (const E*)q, T, G, qs, qwide, n_sel, scale, skip, start, wgs, (int)p.buckets, owner, list, sums, stats)
  if (bk.page_rows <= 32) PAGE(32); else PAGE(64);
#undef PAGE
  hipLaunchKernelGGL((k_bank_join<DT, D>), join, dim3(256), 0, st, sums, stats, T, G, H, C, n_sel, (size_t)n_sel * C, (size_t)1,
                     (size_t)n_sel * G, (size_t)G, (E*)out, lse);
}

extern "C" int gpsr_bank_attend_pages(const gpsr_bank* bank, const int32_t* table, int B, int table_pages, const int32_t* length,
                                      const void* q, int dtype, int T, int q_heads, const int64_t* qst, const int32_t* sel, int n_sel,
                                      float scale, const int32_t* skip, void* out, float* lse, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (B <= 0 || T <= 0) return 0;
  if (const char* w = attend_wrong(bank, table, B, table_pages, length, q, dtype, q_heads, qst, scale, out)) return arg_fail(w);
  if (!sel) return arg_fail("bank_attend_pages: null pointer");
  if (n_sel < 1 || n_sel > 64) return arg_fail("bank_attend_pages: n_sel must be in 1..64");
  const PagesPlan p = plan_of(bank, B, table_pages, T, q_heads, n_sel);
  if (!grid_fits(p.by_page ? p.most_wgs : (int64_t)T * p.groups * p.splits, 256) || !grid_fits(((int64_t)T * (q_heads / bank->heads) + 3) / 4, 256))
    return arg_fail("bank_attend_pages: too many queries for one call");
  if (workspace_bytes < p.bytes || (p.bytes && !workspace)) return arg_fail("workspace too small");
  if (p.bytes && ((uintptr_t)workspace & 15)) return arg_fail("bank_attend_pages: workspace must be 16-byte aligned");
  const Strides qs = {qst[0], qst[1], qst[2]};
  const bool wide = rows_wide(q, qst, dtype);
  hipStream_t st = (hipStream_t)stream;
#define PAGES(DT, BITS, D) launch_pages<DT, BITS, D>(p, *bank, table, B, table_pages, length, q, T, q_heads, qs, wide, sel, n_sel, \
                                                     scale, skip, out, lse, (char*)workspace, st)
  BANK_DISPATCH(PAGES, dtype, bank->bits, bank->dim);
#undef PAGES
  CHECK_LAUNCH("k_bank_attend_pages");
  return 0;
}
