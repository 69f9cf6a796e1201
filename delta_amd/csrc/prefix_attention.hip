// Attention of rows that share a prefix (gfx950): the prefix's pages are read once for all its rows.
//
// Row b holds its whole page list in the CSR, the prefix's pages first; row_prefix[b] names its prefix p,
// whose (full) pages the prefix CSR lists.  The prefix applies where its tokens fit in front of the row's
// query tokens (decode: in the row at all); otherwise the row attends its pages alone, like a row of no
// prefix (row_prefix outside [0, num_prefixes)).  With (m, l, a) = (max s, sum 2^(s - m), sum 2^(s - m) v)
// over any set of tokens X, s = scale log2(e) q.k, the sets' triples combine to
//   o = sum_X a_X 2^(m_X - M) / sum_X l_X 2^(m_X - M),  lse = (M + log2 sum_X l_X 2^(m_X - M)) ln 2,
// so a row's softmax splits into its prefix and its own tokens, and each of these into any runs of pages.
//
// Work decomposition.  A segment is a prefix with the query tokens of all rows that use it (no mask: all of
// them come after it), or a row's own pages with its query tokens (causal).  Its (query token, q head of the kv head's G)
// pairs, in that order, are cut into tiles of 128, its pages into stages of 32 tokens.  The stages of
// all tiles of a kv head form one line, kTileCost more per tile for what a tile costs besides them, and
// block i of the head's `blocks` takes the i-th equal share of it: so the chip's block slots (two per CU)
// finish about together whatever the lengths are (8-13 % apart in the large cases), and a tile is cut only where a share ends.
// Only a long prompt's own tokens are shared out badly: a tile is charged its row's whole length, of which its causal mask leaves
// the first ones little (one prompt of 8000 tokens beside 31 decoding rows over 4800: 899 us, the ordinary launch 555).  The
// lengths are only on the device: every block derives the same line from the tables (build_line, 1.7-2.0 us).
//   A whole tile of a row without a prefix writes o and lse.  Any other one writes un-normalised partials
// (m, l, a): a whole tile at its token's place, a cut one into its block's two buffers (a block's first piece may
// end a cut tile, its last may begin one); the merge kernel joins them per (token, q head).  No atomics: the same call
// gives the same bits.
//
// Per block: 4 waves, each with 32 of the tile's pairs, share K and V in LDS, in stages of 32 tokens, two or three of
// them under way (64 KiB, two blocks per CU); waves without pairs only load.  MFMA
// tiles as in prefill.hip: S^T = K Q^T with lane l holding query pair l % 32 and 16 of the 32 tokens, O^T += V^T P^T, P
// rounded to the cache's type for the product as there (half a step of it per weight, and the fp32 sums l stay unrounded).
// The S of a stage are computed under the softmax of the stage before.  Tiles of up to 64 pairs (a decode row's own pages
// have G) have 16 to a wave, on 16x16 MFMA tiles.
//
// What bounds it.  Decode reads: 128 rows of 1050 own tokens over a prefix of 16384, 8 kv heads of 5: 632 MB in 144 us, 4.4
// TB/s (97 us at the 6.5 TB/s of a bare read; the ordinary launch, which reads the prefix for every row, 754); 32 rows of 530
// over 8192: 33 us against 17 and 101; the line, the pieces' beginnings (2-4 us each) and the merge (6 us with its launch) are
// the rest.  Prompts compute: 32 prompts of 34 tokens over 8192, 8 kv heads of 4: 199 us, 0.69 PFLOP/s, 1.0 in the loop
// (1.06 us a stage of two blocks; 116 us at the 1.19 of an 8192^3 product; the ordinary launch 216).  In the loop no single
// unit is the bound: without the exponentials it would take 95 % of its time, without V's fragments 94, without K's 97,
// without any of them 84.
#include "delta_common.h"
#include "mfma32.h"
#include <math.h>

namespace delta {

namespace {

constexpr int kThreads = 256;
constexpr int kStep = 32;               // kv tokens per stage, the unit of the line
constexpr int kPages = kStep / kPageSize;
constexpr int kPageB = kPageSize * 256; // bytes of a page's K (or V) of one head
constexpr int kStageB = 4 * kPageB;     // a stage: 32 tokens' K, then their V
constexpr int kStages = 4;              // stages in LDS
constexpr int kQ = 128;                 // (token, head) pairs of a tile, at most
constexpr int kMaxRows = 1024;          // rows, and prefixes, of a call (the tables: 41 KiB)
constexpr int kSlots = 512;             // blocks the chip holds (two per CU)
// Stages that a tile costs besides its own, and those of a share, at least: geometric means over 25 batches against units
// of 64 tokens, tile cost 2, shares of 2: (5, 6) -0.5 %, (5, 4) -0.4, (4, 4) +0.3, (6, 6) +0.2, (7, 6) +1.0, (3, 4) +1.6.
constexpr int kTileCost = 5;
constexpr int kMinShare = 6;

struct PrefixArgs {
  const uint16_t *q;
  int64_t q_stride_t, q_stride_h;
  const uint16_t *kv;
  int64_t num_pages;
  const int32_t *qo_indptr;  // null: one query token per row
  const int32_t *kv_indptr;
  const int32_t *kv_indices;
  int64_t kv_indices_len;
  const int32_t *last_page_len;
  const int32_t *row_prefix;
  const int32_t *prefix_indptr;
  const int32_t *prefix_indices;
  int64_t prefix_indices_len;
  int num_prefixes;
  uint16_t *o;
  int64_t o_stride_t, o_stride_h;
  float *lse;
  // Partials: rows (prefix 0 / own 1, token, q head) of whole tiles, then (kv head, block, ends 0 / begins 1 a cut tile,
  // pair) of cut ones.
  float *part_ml;   // [row][2]
  float *part_acc;  // [row][128]
  int2 *runs;       // [prefix / own][token][head of the kv head's]: first block of its tile, runs | pair in the tile << 16
  int batch, tokens, hq, hkv;
  int blocks;       // per kv head
  float sm_scale;
};

// Pages [first, first + n) of CSR entry i, clamped to the index array.
struct Pages {
  int first, n;
};
__device__ __forceinline__ Pages csr_pages(const int32_t *indptr, int len, int i) {
  int p0 = ld_scalar(indptr, i), p1 = ld_scalar(indptr, i + 1);
  p0 = min(max(p0, 0), len);
  p1 = min(max(p1, p0), len);
  return Pages{p0, p1 - p0};
}

struct Row {
  int kv0, pages, len;  // its pages in kv_indices and its tokens, the prefix's included
  int q0, qn;           // query tokens
};
__device__ __forceinline__ Row row_of(const PrefixArgs &a, int r) {
  Row x;
  const Pages p = csr_pages(a.kv_indptr, (int)a.kv_indices_len, r);
  int last = ld_scalar(a.last_page_len, r);
  last = min(max(last, 0), kPageSize);
  x.kv0 = p.first;
  x.pages = p.n;
  x.len = p.n > 0 ? (p.n - 1) * kPageSize + last : 0;
  x.q0 = r;
  x.qn = 1;
  if (a.qo_indptr) {
    int q0 = ld_scalar(a.qo_indptr, r), q1 = ld_scalar(a.qo_indptr, r + 1);
    q0 = min(max(q0, 0), a.tokens);
    q1 = min(max(q1, q0), a.tokens);
    x.q0 = q0;
    x.qn = q1 - q0;
  }
  return x;
}
// Whether a prefix of n pages applies to the row.
__device__ __forceinline__ bool prefix_fits(const PrefixArgs &a, const Row &x, int n) {
  return n > 0 && n <= x.pages && n * kPageSize <= x.len - (a.qo_indptr ? x.qn : 0);
}

__device__ __forceinline__ int div_up(int a, int b) { return (a + b - 1) / b; }

// Tiles of n query tokens.
template <int G>
__device__ __forceinline__ int tiles_of(int n) {
  return div_up(n * G, kQ);
}

// Whether a row's query tokens leave at most an eighth of its tiles idle: such a row shares no tiles with the others of
// its prefix, but sweeps the prefix's pages with its own, from one tile's start to its end (the pages come from the L2
// either way, and nothing has to be joined).
template <int G>
__device__ __forceinline__ bool fills_tiles(int qn) {
  return 9 * qn * G >= 8 * kQ * tiles_of<G>(qn);
}

// A pointer that is the same in every lane, in scalar registers.
template <typename T>
__device__ __forceinline__ T *uniform_ptr(T *p) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  return (T *)(uintptr_t)((uint64_t)(uint32_t)uniform((int)(uint32_t)x) |
                          (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// Exclusive sum over the block's threads, saturating; *total: the block's sum.  `sums` holds 4 ints, free again on return.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *sums, uint32_t *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t incl = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t x = __shfl_up(incl, off, 64);
    if (lane >= off) incl = add_sat(incl, x);
  }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    before = add_sat(before, w < wave ? sums[w] : 0);
    all = add_sat(all, sums[w]);
  }
  __syncthreads();
  *total = all;
  return add_sat(before, incl) - v;
}

// The tables and the line of a kv head's work, in LDS behind the stages.
struct Line {
  int *toks;         // [kQ + 4] query tokens of a prefix's tile
  uint32_t *sums;    // [4]
  int *at;           // [prefixes + rows + 1] where each segment begins (the prefixes, then the rows), and the end
  int *prefix_toks;  // [prefixes] query tokens
  int *prefix_ids;   // [prefixes] first page in prefix_indices
  int *prefix_pages; // [prefixes]
  int *row_prefix;   // [rows] the prefix that applies, -1: none
  int *row_ids;      // [rows] first own page in kv_indices
  int *row_len;      // [rows] own tokens
  int *row_q0, *row_qn;  // [rows] query tokens
  __device__ __forceinline__ Line(int *lds, int prefixes, int rows)
      : toks(lds), sums(reinterpret_cast<uint32_t *>(toks + kQ + 4)), at(toks + kQ + 8), prefix_toks(at + prefixes + rows + 1),
        prefix_ids(prefix_toks + prefixes), prefix_pages(prefix_ids + prefixes), row_prefix(prefix_pages + prefixes),
        row_ids(row_prefix + rows), row_len(row_ids + rows), row_q0(row_len + rows), row_qn(row_q0 + rows) {}
  static size_t bytes(int prefixes, int rows) {
    return ((size_t)kQ + 8 + 4 * (size_t)prefixes + 6 * (size_t)rows + 1) * sizeof(int);
  }
};

// The line's length; 0 where it would pass 2^30 (only rows that overlap, in tables that do not ascend, come to that).
template <int G>
__device__ __forceinline__ int build_line(const PrefixArgs &a, const Line &line) {
  const int tid = threadIdx.x, P = a.num_prefixes, B = a.batch;
#pragma unroll 1
  for (int r0 = 0; r0 < B; r0 += kThreads) {
    const int r = r0 + tid;
    const Row x = row_of(a, r < B ? r : 0);
    const int want = a.row_prefix[r < B ? r : 0];
    if (r0 == 0) {  // (the rows' tables are asked for before the prefixes' have come)
      for (int p = tid; p < P; p += kThreads) {
        const Pages pages = csr_pages(a.prefix_indptr, (int)a.prefix_indices_len, p);
        line.prefix_toks[p] = 0;
        line.prefix_ids[p] = pages.first;
        line.prefix_pages[p] = pages.n;
      }
      __syncthreads();
    }
    if (r >= B) continue;
    const bool named = want >= 0 && want < P;
    const int n = named ? line.prefix_pages[want] : 0;
    const bool fits = named && !fills_tiles<G>(x.qn) && prefix_fits(a, x, n);
    if (fits) atomicAdd(&line.prefix_toks[want], x.qn);
    const int own = x.len - (fits ? n * kPageSize : 0);
    line.row_prefix[r] = fits ? want : -1;
    line.row_ids[r] = x.kv0 + (fits ? n : 0);
    line.row_len[r] = own;
    line.row_q0[r] = x.q0;
    line.row_qn[r] = x.qn;
  }
  __syncthreads();
  uint32_t end = 0;
  for (int i0 = 0; i0 < P + B; i0 += kThreads) {
    const int i = i0 + tid;
    uint64_t cost = 0;
    uint32_t total;
    if (i < P) {
      const int toks = min(line.prefix_toks[i], a.tokens);
      line.prefix_toks[i] = toks;
      cost = (uint64_t)(uint32_t)tiles_of<G>(toks) * (uint32_t)(div_up(line.prefix_pages[i], kPages) + kTileCost);
    } else if (i < P + B) {
      cost = (uint64_t)(uint32_t)tiles_of<G>(line.row_qn[i - P]) * (uint32_t)(div_up(line.row_len[i - P], kStep) + kTileCost);
    }
    const uint32_t before = block_scan((uint32_t)(cost < UINT32_MAX ? cost : UINT32_MAX), line.sums, &total);
    if (i < P + B) line.at[i] = (int)add_sat(end, before);
    end = add_sat(end, total);
  }
  if (tid == 0) line.at[P + B] = (int)end;
  __syncthreads();
  return end <= 1u << 30 ? (int)end : 0;
}

template <int DT, int G>
__global__ void __launch_bounds__(kThreads, 2) prefix_attention_kernel(PrefixArgs a) {
#pragma clang fp contract(off)
  using MF = Mfma32<DT>;
  using E = Elem<DT>;
  // A ring of stages, each the K tile, then the V tile (swizzled rows).
  extern __shared__ __attribute__((aligned(1024))) char tiles[];
  const Line line(reinterpret_cast<int *>(tiles + kStages * kStageB), a.num_prefixes, a.batch);

  const int wv = uniform((int)(threadIdx.x >> 6));
  const int h = blockIdx.x, blk = blockIdx.y;
  const int total = uniform(build_line<G>(a, line));
  int share = uniform(div_up(total, a.blocks));
  share = share < kMinShare ? kMinShare : share;
  int pos = blk * share;  // (total <= 2^30: build_line)
  const int end = min(total, pos + share);

  // Loads: K and V rows go straight to LDS, 1 KiB (4 rows of this head) per load.  16-byte chunk ch of K row r sits at
  // slot ch ^ (r % 16) and of V row r at ch ^ 4 (r % 4), so that the fragment reads cover the banks once.
  const uint32_t row_bytes = (uint32_t)a.hkv * kHeadDim * 2;
  const uint32_t page_bytes = 2 * kPageSize * row_bytes;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)&tiles[0];
  const char *const kvh = reinterpret_cast<const char *>(a.kv) + (int64_t)h * (kHeadDim * 2);
  const uint32_t num_pages = a.num_pages < INT32_MAX ? (uint32_t)a.num_pages : (uint32_t)INT32_MAX;
  const float scale2 = a.sm_scale == 0.f ? 1.f : fabsf(a.sm_scale) * kLog2e;
  int item = 0;
  while (pos < end) {
    // The lane, hidden from the compiler: it would keep every offset that follows from it in registers over all pieces.
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int lrow = lane >> 4, lch = lane & 15;
    // ---- The piece at pos: segment, tile, stages [s0, s1).
    const int items = a.num_prefixes + a.batch;
    for (;; item += 64) {  // the first segment that ends past pos
      const int i = item + lane;
      const uint64_t past = __ballot(i < items && line.at[i < items ? i + 1 : items] > pos);
      if (past) {
        item = uniform(item + __builtin_ctzll(past));
        break;
      }
    }
    const bool of_prefix = item < a.num_prefixes;
    const int32_t *ids;  // the segment's page ids
    int np, len, seg_toks, q0 = 0, px = -1;
    if (of_prefix) {
      ids = a.prefix_indices + uniform(line.prefix_ids[item]);
      np = uniform(line.prefix_pages[item]);
      len = np * kPageSize;
      seg_toks = uniform(line.prefix_toks[item]);
    } else {
      const int r = item - a.num_prefixes;
      px = uniform(line.row_prefix[r]);
      ids = a.kv_indices + uniform(line.row_ids[r]);
      len = uniform(line.row_len[r]);
      np = div_up(len, kPageSize);
      seg_toks = uniform(line.row_qn[r]);
      q0 = uniform(line.row_q0[r]);
    }
    const int cost = div_up(len, kStep) + kTileCost;
    const int seg_at = uniform(line.at[item]);
    const int tile = uniform((pos - seg_at) / cost), tile_at = seg_at + tile * cost;
    const int stop = min(end, tile_at + cost);
    const int s0 = max(0, pos - tile_at - kTileCost);
    int s1 = max(0, stop - tile_at - kTileCost);
    const int first_blk = uniform(tile_at / share), runs = uniform((tile_at + cost - 1) / share) - first_blk + 1;
    const int run = blk - first_blk;
    pos = stop;
    // The tile's pairs, and the query tokens [t0, t0 + ntok) of the segment that they belong to (where G does not divide
    // 128 a token's heads may lie in two tiles).
    const int pairs0 = tile * kQ, pairs = min(kQ, seg_toks * G - pairs0);
    const int t0 = pairs0 / G, ntok = (pairs0 + pairs - 1) / G + 1 - t0, skew = pairs0 - t0 * G;
    // Segment position of query token t0 + i of a row: first_pos + i; a prefix's tokens come behind all of it.
    const int first_pos = of_prefix ? len : len - seg_toks + t0;
    if (!of_prefix) {
      const int reach = first_pos + ntok;  // tokens that the tile's last query token attends
      s1 = min(s1, reach > 0 ? div_up(min(reach, len), kStep) : 0);
    }
    if (of_prefix) {
      // The tile's tokens out of those of the prefix's rows, row by row.
      uint32_t before = 0, sum;
      const int upto = t0 + ntok;
      for (int r0 = 0; r0 < a.batch; r0 += kThreads) {
        const int r = r0 + threadIdx.x;
        const bool mine = r < a.batch && line.row_prefix[r] == item;
        const int qn = mine ? line.row_qn[r] : 0, rq0 = mine ? line.row_q0[r] : 0;
        const int at = (int)min(add_sat(before, block_scan(qn, line.sums, &sum)), (uint32_t)upto);
        for (int k = t0 > at ? t0 - at : 0; k < qn && at + k < upto; ++k) line.toks[at + k - t0] = rq0 + k;
        before = add_sat(before, sum);
        if (before >= (uint32_t)upto) break;
      }
    }
    __syncthreads();  // the tile's tokens are listed, the piece before is done with the buffers

    // Loads: wave w loads rows 4 w .. + 3 of both of a stage's pages, K and V.  Page ids, 64 per register (lane i: page
    // 64 w + i of the piece); bit i of *bad: outside the cache.
    const uint32_t wlds = lds0 + wv * 1024;
    const uint32_t koff = (4 * wv + lrow) * row_bytes + 16 * (lch ^ (4 * wv + lrow));
    const uint32_t voff = (kPageSize + 4 * wv + lrow) * row_bytes + 16 * (lch ^ (4 * lrow));
    const int p0 = kPages * s0, count = min(np, kPages * s1) - p0;  // <= 0: no page
    const int nst = count > 0 ? (count + 1) >> 1 : 0;
    auto load_ids = [&](int w, uint64_t *bad) {
      const int i = 64 * w + lane;
      const int id = i < count ? ids[p0 + i] : 0;
      const bool ok = (uint32_t)id < num_pages;
      *bad = __ballot(!ok);
      return ok ? id : 0;
    };
    uint64_t bad = 0, bad_next = 0;
    int idv = 0;
    auto first_loads = [&]() { idv = load_ids(0, &bad); };
    auto issue = [&](int j) {  // stage j of the piece; a page past it is page 0 of the cache (masked later)
      const uint32_t dst = wlds + (uint32_t)(j & (kStages - 1)) * kStageB;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const char *pg = uniform_ptr(kvh + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(idv, (2 * j + i) & 63) * page_bytes);
        if (of_prefix || a.qo_indptr) {
          load_lds_1k(dst + i * kPageB, pg, koff);
          load_lds_1k(dst + 2 * kPageB + i * kPageB, pg, voff);
        } else {  // read once
          load_lds_1k<true>(dst + i * kPageB, pg, koff);
          load_lds_1k<true>(dst + 2 * kPageB + i * kPageB, pg, voff);
        }
      }
    };
    auto start = [&]() {
      bad_next = bad;
      for (int j = 0; j < 3 && j < nst; ++j) issue(j);
    };
    auto bad_of = [&](int j) { return (uint32_t)(bad >> ((2 * j) & 63)) & 3u; };  // bit i: page i of stage j
    // V rows past the segment and of pages outside the cache meet p = 0 but may hold NaN/Inf: zeros.
    auto clear_v = [&](int j, uint32_t sbad) {
      const int kv0 = s0 * kStep + 32 * j;
      if (kv0 + 32 <= len && sbad == 0) return;
      const int r = (int)threadIdx.x >> 3;
      if (kv0 + r >= len || ((sbad >> (r >> 4)) & 1u)) {
        char *vr = &tiles[(j & (kStages - 1)) * kStageB + 2 * kPageB] + r * 256 + 32 * ((int)threadIdx.x & 7);
#pragma unroll
        for (int i = 0; i < 2; ++i) st128(vr + 16 * i, u32x4{0u, 0u, 0u, 0u});
      }
    };

    auto enter = [&]() {  // the first stage has landed
      if (nst > 2)
        wait_loads<8>();
      else if (nst > 1)
        wait_loads<4>();
      else
        wait_loads<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (nst > 0) clear_v(0, bad_of(0));
    };
    auto step = [&](int j) {  // stage j + 1 has landed, stage j - 1 is left by every wave; returns bad_of(j)
      if (j + 2 < nst)
        wait_loads<4>();
      else
        wait_loads<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const uint32_t sbad = bad_of(j);
      if (((j + 1) & 31) == 0) bad = bad_next;
      if (j + 3 < nst) {
        if (((j + 3) & 31) == 0) idv = load_ids((j + 3) >> 5, &bad_next);
        issue(j + 3);
      }
      if (j + 1 < nst) clear_v(j + 1, bad_of(j + 1));
      return sbad;
    };
    const bool whole = runs == 1 && !of_prefix && px < 0;
    // Results of a pair from the lanes that hold it: 4 outputs from d(k) on in v(k), k < N; `one` of the lanes also
    // writes the statistics.
    auto put = [&](auto count, int pair, bool one, float m, float l, auto &&v, auto &&d) {
      constexpr int N = decltype(count)::value;
      const int pt = (skew + pair) / G, hq = h * G + skew + pair - pt * G;
      const int t = of_prefix ? line.toks[pt] : q0 + t0 + pt;
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t *op = a.o + (int64_t)t * a.o_stride_t + (int64_t)hq * a.o_stride_h;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const f32x4 x = v(k);
          uint32_t *w = reinterpret_cast<uint32_t *>(op + d(k));
          w[0] = pack2<DT>(x[0] * inv, x[1] * inv);
          w[1] = pack2<DT>(x[2] * inv, x[3] * inv);
        }
        if (a.lse && one) a.lse[(int64_t)t * a.hq + hq] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
      } else {
        const int64_t at = runs == 1 ? ((int64_t)(of_prefix ? 0 : a.tokens) + t) * a.hq + hq
                                     : (int64_t)2 * a.tokens * a.hq +
                                           (((int64_t)h * a.blocks + blk) * 2 + (run == 0 ? 1 : 0)) * kQ + pair;
        float *op = a.part_acc + at * kHeadDim;
#pragma unroll
        for (int k = 0; k < N; ++k) *reinterpret_cast<f32x4 *>(op + d(k)) = v(k);
        if (one) *reinterpret_cast<float2 *>(a.part_ml + at * 2) = float2{m, l};
      }
    };

    if (pairs <= 64) {
      // ---- 16 pairs per wave, on 16x16 tiles: half the MFMA time and half the scores per lane of the 32x32 ones, and more
      // of the SIMDs at work (a decode row's own pages, one wave: 0.93 us a stage on 32x32 tiles, 0.85 here; us for 64 prompts of 5
      // tokens behind up to 1500 own, 25 pairs, 81.3 / 78.0; for 8 rows of 7 heads over 16384, 56 pairs, 23.8 / 22.7).
      // Lane (c, n) = (lane / 16, lane % 16): pair n; scores of tokens 4 c + i and 16 + 4 c + i; outputs d = 16 dt + 4 c + i.
      const int c = lane >> 4, n = lane & 15;
      const int qsub = (wv + blk) & 3, pair = 16 * qsub + n;
      const bool active = 16 * qsub < pairs, ok = pair < pairs;
      const int pt = ok ? (skew + pair) / G : 0, t = of_prefix ? line.toks[pt] : q0 + t0 + pt;
      const int lim = of_prefix ? len - 1 : min(len - 1, first_pos + pt);
      const int wpos = of_prefix ? len - 1 : min(len - 1, first_pos + (skew + 16 * qsub) / G);
      u32x4 qf[4];  // B operand of S^T: d = 32 ks + 8 c + [0, 8)
      const uint16_t *qp = a.q + (int64_t)t * a.q_stride_t + (int64_t)(h * G + (ok ? skew + pair - pt * G : 0)) * a.q_stride_h + 8 * c;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) qf[ks] = ok ? ld128(qp + 32 * ks) : u32x4{0u, 0u, 0u, 0u};
      first_loads();
      // Settles q with the page ids: inside the loop its wait would also drain the stages under way.
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) asm volatile("" : "+v"(qf[ks]));
      start();
      const uint32_t kfo = (uint32_t)(n * 256 + 16 * (c ^ n));  // K fragment: row n (+ 16), chunk 4 ks + c (64 ks by xor)
      // V^T fragment of d tile dt: rows 4 c .. + 3 (+ 16) at columns 16 dt + [0, 16) (32 dt by xor)
      const uint32_t vfo = (uint32_t)((4 * c + (n >> 2)) * 256 + 16 * (((n & 3) >> 1) ^ (4 * (n >> 2))) + 8 * (n & 1));
      float m = -INFINITY, l = 0.f;
      f32x4 acc[8], S[2];
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
      auto scores = [&](int j) {
        const char *tk = &tiles[(j & (kStages - 1)) * kStageB];
        S[0] = S[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            S[u] = E::mfma(*reinterpret_cast<const u32x4 *>(tk + (kfo ^ (64u * ks)) + u * 4096), qf[ks], S[u]);
      };
      enter();
      if (active && nst > 0) scores(0);
      for (int j = 0; j < nst; ++j) {
        const uint32_t sbad = step(j);
        if (!active) continue;
        const int kv0 = s0 * kStep + 32 * j;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = S[i >> 2][i & 3];
        if (!(a.sm_scale > 0.f)) {  // (the scale below is positive)
          const float sign = a.sm_scale == 0.f ? 0.f : -1.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= sign;
        }
        if (kv0 + 31 > wpos || sbad) {
          const int last = lim - kv0 - 4 * c;
          uint32_t b = sbad;  // (in a vector register: selects, not a branch for each value)
          asm volatile("" : "+v"(b));
#pragma unroll
          for (int i = 0; i < 8; ++i)
            x[i] = 16 * (i >> 2) + (i & 3) <= last && !((b >> (i >> 2)) & 1u) ? x[i] : -INFINITY;
        }
        scores(j + 1);  // (of no use behind the last stage) under the softmax
        float pm = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) pm = fmaxf(pm, x[i]);
        // (the reference maximum as below)
        const float smax = rows4_max(pm) * scale2;
        const bool moves = smax > m + 8.f;
        const float alpha = moves ? fast_exp2(m - smax) : 1.f;
        m = moves ? smax : m;
        const float nm = m == -INFINITY ? 0.f : -m;
        float ps = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = fast_exp2(fmaf(x[i], scale2, nm));
          ps += x[i];
        }
        l = l * alpha + ps;  // this lane's tokens; joined once at the end
        const u32x4 pc = {pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7])};
        if (__ballot(moves)) {
#pragma unroll
          for (int dt = 0; dt < 8; ++dt) acc[dt] *= alpha;
        }
        const char *tv = &tiles[(j & (kStages - 1)) * kStageB + 2 * kPageB];
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
          const char *rd = tv + (vfo ^ (32u * dt));
          const ps4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ps4_t *)rd);
          const ps4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ps4_t *)(rd + 4096));
          const uint2 lo = __builtin_bit_cast(uint2, v0), hi = __builtin_bit_cast(uint2, v1);
          acc[dt] = E::mfma(u32x4{lo.x, lo.y, hi.x, hi.y}, pc, acc[dt]);
        }
      }
      l = rows4_sum(l);
      if (ok)
        put(std::integral_constant<int, 8>(), pair, c == 0, m, l, [&](int k) { return acc[k]; },
            [&](int k) { return 16 * k + 4 * c; });
    } else {
      // ---- The wave's pairs: 32 from 32 qsub on.
      const int n = lane & 31, hl = lane >> 5, qsub = (wv + blk) & 3;  // (a short tile keeps some SIMDs at work)
      const bool active = 32 * qsub < pairs;
      const int pair = 32 * qsub + n;
      const bool row_ok = pair < pairs;
      const int pt = row_ok ? (skew + pair) / G : 0, g = row_ok ? (skew + pair) % G : 0;
      const int t = of_prefix ? line.toks[pt] : q0 + t0 + pt;
      const int lim = of_prefix ? len - 1 : min(len - 1, first_pos + pt);  // the last position that the lane's pair attends
      // Stages that end at or below the position of the wave's first token need no mask.
      const int wpos = of_prefix ? len - 1 : min(len - 1, first_pos + (skew + 32 * qsub) / G);
      u32x4 qf[8];  // B operand of S^T = K Q^T: d = 16 ks + 8 hl + [0, 8)
      {
        const uint16_t *qp = a.q + (int64_t)t * a.q_stride_t + (int64_t)(h * G + g) * a.q_stride_h + 8 * hl;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qf[ks] = row_ok ? ld128(qp + 16 * ks) : u32x4{0u, 0u, 0u, 0u};
      }
      first_loads();
      // (see above)
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) asm volatile("" : "+v"(qf[ks]));
      start();
      // K fragment of k-slice ks: row n, chunk 2 ks + hl (32 ks comes in by xor: the bits above it are the row's).
      const uint32_t kfo = (uint32_t)(n * 256 + 16 * (hl ^ (n & 15)));
      // ds_read_b64_tr_b16 of V^T: 16-lane group q16 = lane / 16, t16 = lane % 16 reads rows (kv) base + t16 / 4 at columns
      // 32 dt + 16 (q16 % 2) + 4 (t16 % 4), and receives its column's four rows (64 dt by xor).
      const int q16 = lane >> 4, t16 = lane & 15;
      const uint32_t vfo = (uint32_t)((4 * hl + (t16 >> 2)) * 256 +
                                      16 * ((2 * (q16 & 1) + ((t16 & 3) >> 1)) ^ (4 * (t16 >> 2))) + 8 * (t16 & 1));
      float m = -INFINITY, l = 0.f;
      f32x16 acc[4];
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;

      // S^T of the first stage.
      auto scores = [&](f32x16 &S) {
#pragma unroll
        for (int i = 0; i < 16; ++i) S[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) S = MF::run(*reinterpret_cast<const u32x4 *>(tiles + (kfo ^ (32u * ks))), qf[ks], S);
      };
      f32x16 S;  // of the stage worked on
      enter();
      if (active && nst > 0) scores(S);
      for (int j = 0; j < nst; ++j) {
        const uint32_t sbad = step(j);
        if (!active) continue;
        const int kv0 = s0 * kStep + 32 * j;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = S[i];
        if (!(a.sm_scale > 0.f)) {  // (the scale below is positive)
          const float sign = a.sm_scale == 0.f ? 0.f : -1.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= sign;
        }
        auto tok = [&](int i) { return 8 * (i >> 2) + (i & 3); };  // of x[i], from kv0 + 4 hl on
        if (kv0 + 31 > wpos) {
          const int last = lim - kv0 - 4 * hl;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = tok(i) <= last ? x[i] : -INFINITY;
        }
        if (sbad) {
          uint32_t b = sbad;  // (in a vector register: selects, not a branch for each value)
          asm volatile("" : "+v"(b));
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = (b >> (i >> 3)) & 1u ? -INFINITY : x[i];
        }
        // The next stage's S (of no use behind the last stage), an MFMA at a time between pieces of this one's softmax:
        // each piece runs while its MFMA does.  The fences keep that order.
        const char *tk = &tiles[((j + 1) & (kStages - 1)) * kStageB];
        auto kfrag = [&](int ks) { return *reinterpret_cast<const u32x4 *>(tk + (kfo ^ (32u * ks))); };
        u32x4 kq[4];
#pragma unroll
        for (int ks = 0; ks < 3; ++ks) kq[ks] = kfrag(ks);
#pragma unroll
        for (int i = 0; i < 16; ++i) S[i] = 0.f;
        auto mfma_s = [&](int ks) {
          if (ks + 3 < 8) kq[(ks + 3) & 3] = kfrag(ks + 3);
          S = MF::run(kq[ks & 3], qf[ks], S);
          __builtin_amdgcn_sched_barrier(0);
        };
        float pm = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) pm = fmaxf(pm, x[i]);
        __builtin_amdgcn_sched_barrier(0);
        mfma_s(0);
        // m is a reference maximum: it moves only when a score exceeds it by more than 8 (log2), so the exponentials
        // stay <= 256 and the accumulators are rescaled on few stages.
        const float smax = halves_max(pm) * scale2;
        const bool moves = smax > m + 8.f;  // also the first finite score (m = -inf)
        const float alpha = moves ? fast_exp2(m - smax) : 1.f;
        m = moves ? smax : m;
        const float nm = m == -INFINITY ? 0.f : -m;
        __builtin_amdgcn_sched_barrier(0);
        mfma_s(1);
        const char *tv = &tiles[(j & (kStages - 1)) * kStageB + 2 * kPageB];
        auto vfrag = [&](int i) {  // V^T fragment of 16-token chunk i / 4, d tile i % 4
          const char *rd = tv + (vfo ^ (64u * (i % 4))) + (i / 4) * 4096;
          const ps4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ps4_t *)rd);
          const ps4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ps4_t *)(rd + 2048));
          const uint2 lo = __builtin_bit_cast(uint2, v0), hi = __builtin_bit_cast(uint2, v1);
          return u32x4{lo.x, lo.y, hi.x, hi.y};
        };
        constexpr int kAhead = 4;
        u32x4 vq[kAhead + 1];
        float ps = 0.f;
        u32x4 pc[2];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          x[2 * c] = fast_exp2(fmaf(x[2 * c], scale2, nm));
          x[2 * c + 1] = fast_exp2(fmaf(x[2 * c + 1], scale2, nm));
          if (c > 0) {
            ps += x[2 * c - 2] + x[2 * c - 1];
            pc[(c - 1) >> 2][(c - 1) & 3] = pack2<DT>(x[2 * c - 2], x[2 * c - 1]);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (c < 6) mfma_s(c + 2);
          if (c >= 4) vq[c - 4] = vfrag(c - 4);
        }
        ps += x[14] + x[15];
        pc[1][3] = pack2<DT>(x[14], x[15]);
        l = l * alpha + ps;  // this half-wave's tokens; joined once at the end
        // (used here, or the compiler moves the exponentials behind the rescaling branch, away from the MFMAs)
        asm volatile("" : "+v"(pc[0]), "+v"(pc[1]), "+v"(l));
        if (__ballot(alpha != 1.f)) {
#pragma unroll
          for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i + kAhead < 8) vq[(i + kAhead) % (kAhead + 1)] = vfrag(i + kAhead);
          acc[i % 4] = MF::run(vq[i % (kAhead + 1)], pc[i / 4], acc[i % 4]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      l = halves_sum(l);
      // (the lane's pair worked out again: held over the stages it would cost registers)
      asm volatile("" : "+v"(lane));
      const int wpair = 32 * qsub + (lane & 31);
      if (wpair < pairs)
        put(std::integral_constant<int, 16>(), wpair, (lane >> 5) == 0, m, l,
            [&](int k) {
              return f32x4{acc[k >> 2][4 * (k & 3)], acc[k >> 2][4 * (k & 3) + 1], acc[k >> 2][4 * (k & 3) + 2],
                           acc[k >> 2][4 * (k & 3) + 3]};
            },
            [&](int k) { return 32 * (k >> 2) + 8 * (k & 3) + 4 * (lane >> 5); });
    }
    if (h == 0 && run == 0 && (int)threadIdx.x < pairs) {
      const int pair = threadIdx.x, pt = (skew + pair) / G, g = skew + pair - pt * G;
      const int ti = of_prefix ? line.toks[pt] : q0 + t0 + pt;
      a.runs[((of_prefix ? 0 : a.tokens) + ti) * G + g] = int2{first_blk, runs | pair << 16};
      if (!of_prefix && px < 0) a.runs[ti * G + g] = int2{0, 0};
    }
    __syncthreads();  // the next piece lists its tokens and loads its pages
  }
}

// The runs of (token t, q head hq): entry e's row in the partials, the prefix's runs first, then the own tile's.
struct Runs {
  int first[2], count[2], pair[2], t, hq, h;
  bool skip;  // left as they are: a query token of no row, and one whose tile wrote it
};
__device__ __forceinline__ Runs runs_of(const PrefixArgs &a, int64_t row) {
  Runs x;
  const bool in = row < (int64_t)a.tokens * a.hq;
  x.t = (int)((in ? row : 0) / a.hq);
  x.hq = (int)((in ? row : 0) - (int64_t)x.t * a.hq);
  const int G = a.hq / a.hkv;
  x.h = x.hq / G;
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {  // (the limits keep a table that is no CSR inside the partials)
    const int2 r = a.runs[(kind * a.tokens + x.t) * G + x.hq - x.h * G];
    x.first[kind] = min(max(r.x, 0), a.blocks - 1);
    x.count[kind] = min(r.y & 0xffff, a.blocks - x.first[kind]);
    x.pair[kind] = min((r.y >> 16) & 0xffff, kQ - 1);
  }
  x.skip = !in || (a.qo_indptr && (x.t < a.qo_indptr[0] || x.t >= a.qo_indptr[a.batch])) ||
           (x.count[0] == 0 && x.count[1] == 1);
  if (x.skip) x.count[0] = x.count[1] = 0;
  return x;
}
// (e >= the runs' number: some row of the partials)
__device__ __forceinline__ int entry_row(const PrefixArgs &a, const Runs &x, int e) {
  const bool own = e >= x.count[0];
  const int kind = own ? 1 : 0, r = min(own ? e - x.count[0] : e, max(x.count[kind] - 1, 0));
  return x.count[kind] <= 1 ? (kind * a.tokens + x.t) * a.hq + x.hq
                            : 2 * a.tokens * a.hq + ((x.h * a.blocks + x.first[kind] + r) * 2 + (r == 0)) * kQ + x.pair[kind];
}
template <int DT>
__device__ __forceinline__ void merged(const PrefixArgs &a, const Runs &x, int d, f32x4 A, float M, float L) {
  using E = Elem<DT>;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint32_t *op = reinterpret_cast<uint32_t *>(a.o + (int64_t)x.t * a.o_stride_t + (int64_t)x.hq * a.o_stride_h + d);
  op[0] = E::from_float(A[0] * inv) | (E::from_float(A[1] * inv) << 16);
  op[1] = E::from_float(A[2] * inv) | (E::from_float(A[3] * inv) << 16);
  if (d == 0 && a.lse) a.lse[(int64_t)x.t * a.hq + x.hq] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// Joins the runs of each (token, q head), W half-waves each (W = 1: two rows to a wave): lane e of half-wave w holds the
// row and (m, l) of entry e W + w, then sums four of the 128 outputs over its half-wave's entries; W half-waves are joined
// in LDS.  A chain of two loads (the runs; partials and statistics together), so what counts is how many are under way.
template <int DT, int W>
__global__ void __launch_bounds__(kThreads, 6) prefix_merge_kernel(PrefixArgs a) {
  constexpr int kHalves = kThreads / 32, kRows = kHalves / W;
  __shared__ float s_m[kHalves], s_l[kHalves];
  __shared__ f32x4 s_a[kHalves][32];
  const int lane = threadIdx.x & 31, half = threadIdx.x >> 5, w0 = half % W;
  const Runs x = runs_of(a, (int64_t)blockIdx.x * kRows + half / W);
  const int n = x.count[0] + x.count[1], mine = n > w0 ? (n - w0 + W - 1) / W : 0;  // entries of this half-wave
  float M = -INFINITY, L = 0.f;
  f32x4 A = {0.f, 0.f, 0.f, 0.f};
  const int base = threadIdx.x & 32;  // the half-wave's first lane
  for (int e0 = 0; __ballot(e0 < mine) != 0; e0 += 32) {
    const bool have = e0 + lane < mine;
    const int at = entry_row(a, x, (e0 + lane) * W + w0);
    const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + (int64_t)at * 2);
    auto load = [&](int i) {
      const int64_t from = __builtin_amdgcn_ds_bpermute((base + i) << 2, at);
      return *reinterpret_cast<const f32x4 *>(a.part_acc + from * kHeadDim + 4 * lane);
    };
    f32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = load(k);  // under the weights' arithmetic
    const float ms = have ? ml.x : -INFINITY;
    float cm = fmaxf(M, ms);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) cm = fmaxf(cm, shfl_xor(cm, off));
    const float ref = cm == -INFINITY ? 0.f : cm, al = fast_exp2(M - ref);
    const float w = have ? fast_exp2(ms - ref) : 0.f;  // 0 where nothing was attended
    float s = have ? ml.y * w : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += shfl_xor(s, off);
    L = L * al + s;
    A *= al;
    M = cm;
    const int most = min(32, mine - e0);
    for (int i0 = 0;;) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float ws = shfl(w, base + i0 + k);
        if (i0 + k < most) A += v[k] * ws;
      }
      i0 += 4;
      if (__ballot(i0 < most) == 0) break;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = load(i0 + k);
    }
  }
  if constexpr (W > 1) {
    s_a[half][lane] = A;
    if (lane == 0) {
      s_m[half] = M;
      s_l[half] = L;
    }
    __syncthreads();
    if (w0 != 0) return;
    M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, s_m[half + w]);
    const float ref = M == -INFINITY ? 0.f : M;
    L = 0.f;
    A = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float sc = fast_exp2(s_m[half + w] - ref);
      L = fmaf(s_l[half + w], sc, L);
      A += s_a[half + w][lane] * sc;
    }
  }
  if (!x.skip) merged<DT>(a, x, 4 * lane, A, M, L);
}

// Blocks per kv head: as many as the chip holds, or as the longest line of `tokens` query tokens over rows of
// `max_pages` fills with kMinShare stages each.
int plan_blocks(int64_t tokens, int hkv, int64_t max_pages, int slots) {
  const int64_t fill = slots / hkv > 0 ? slots / hkv : 1;
  const int64_t steps = ceil_div(max_pages, kPages) + kTileCost;
  if (steps >= fill * kMinShare || 2 * tokens >= fill * kMinShare) return (int)fill;
  const int64_t n = ceil_div(2 * tokens * steps, kMinShare);
  return (int)(n < fill ? n : fill);
}

// Blocks the chip holds: two per CU where their LDS (160 KiB per CU) allows.
int resident_blocks(int prefixes, int rows) {
  return 2 * (kStages * kStageB + Line::bytes(prefixes, rows)) <= 160 * 1024 ? kSlots : kSlots / 2;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t partial_rows(int64_t tokens, int hq, int hkv, int blocks) {
  return (size_t)2 * tokens * hq + (size_t)hkv * blocks * 2 * kQ;
}

size_t workspace_bytes_for(int64_t tokens, int hq, int hkv, int blocks) {
  const size_t rows = partial_rows(tokens, hq, hkv, blocks);
  return align256(rows * 2 * sizeof(float)) + align256(rows * kHeadDim * sizeof(float)) +
         align256((size_t)2 * tokens * (hq / hkv) * sizeof(int2));
}

template <int DT, int G>
void launch_g(const PrefixArgs &a, hipStream_t stream) {
  hipLaunchKernelGGL((prefix_attention_kernel<DT, G>), dim3((unsigned)a.hkv, (unsigned)a.blocks), dim3(kThreads),
                     kStages * kStageB + Line::bytes(a.num_prefixes, a.batch), stream, a);
}

template <int DT, int W>
void launch_merge(const PrefixArgs &a, int64_t rows, hipStream_t stream) {
  constexpr int kRows = kThreads / 32 / W;
  hipLaunchKernelGGL((prefix_merge_kernel<DT, W>), dim3((unsigned)ceil_div(rows, kRows)), dim3(kThreads), 0, stream, a);
}

template <int DT>
void launch(const PrefixArgs &a, int G, hipStream_t stream) {
  switch (G) {
    case 1: launch_g<DT, 1>(a, stream); break;
    case 2: launch_g<DT, 2>(a, stream); break;
    case 3: launch_g<DT, 3>(a, stream); break;
    case 4: launch_g<DT, 4>(a, stream); break;
    case 5: launch_g<DT, 5>(a, stream); break;
    case 6: launch_g<DT, 6>(a, stream); break;
    case 7: launch_g<DT, 7>(a, stream); break;
    default: launch_g<DT, 8>(a, stream); break;
  }
  // Where all tokens share a prefix a row has as many runs as blocks share its tile, about 512 * 128 / rows: about four of
  // them to a half-wave.
  const int64_t rows = (int64_t)a.tokens * a.hq, each = ceil_div((int64_t)kSlots * kQ, rows);
  if (each > 16)
    launch_merge<DT, 8>(a, rows, stream);
  else if (each > 8)
    launch_merge<DT, 4>(a, rows, stream);
  else if (each > 4)
    launch_merge<DT, 2>(a, rows, stream);
  else
    launch_merge<DT, 1>(a, rows, stream);
}

// Whether a decode batch is too small for sharing to pay: one row, or rows that are read in the time that the launches here take
// besides their work (the line, the merge, and a piece's beginning for every row's own pages: 8 us for few rows, 20 for 1024 (row,
// kv head) pairs).  The ordinary launch reads every row, pages that rows share mostly from the L2 and the Infinity Cache.  What
// the rows share is known on the device only, so the rule goes by all that they may read, planned; us here / ordinary at rows
// that share four fifths of it, bf16, the line at 8192 page-heads (of 8 KiB) up to 32 pairs, 18.3 k for 128, 41 k for 512:
//   8 kv heads of 4: 8 rows, 8 k 15.4 / 14.4, 16 k 17.8 / 19.2; 16 rows, 16 k 18.1 / 18.1, 33 k 22.1 / 29.9; 32 rows, 16 k 20.8 /
//   15.5, 33 k 24.9 / 26.9; 64 rows, 8 k 24.6 / 8.8, 33 k 28.8 / 23.0, 49 k 33.5 / 32.7, 66 k 37.0 / 41.9; 128 rows, 49 k 39.1 /
//   33.3, 66 k 41.5 / 42.5; 2 of 6: 16 rows, 8 k 17.7 / 14.7, 16 k 20.2 / 21.3; 64 rows, 16 k 22.5 / 19.0, 33 k 26.9 / 32.1; 256
//   rows, 33 k 33.9 / 26.7, 66 k 40.8 / 45.4; 8 of 1: 64 rows, 16 k 17.6 / 12.3, 33 k 20.3 / 21.1.
// (The ordinary launch takes at most 16 kv heads.)
bool decode_alone(int64_t rows, int hkv, int64_t max_pages) {
  if (hkv > 16 || rows > kMaxRows) return false;
  const double pairs = (double)(rows * hkv);
  return rows == 1 || pairs * (double)max_pages <= 8192.0 * pow(pairs > 32 ? pairs / 32 : 1.0, 0.58);
}
// And a prompt step: the ordinary launch has one block sweep a row's pages for each of its tiles, 6 us and 0.3 a page whatever the
// number of rows, the launches here take 15-50 us whatever the pages.  The host knows the rows' pages in all only, so a single row
// of up to 32, several of up to 64 together (us here / ordinary, 8 kv heads of 4, 7 new tokens: one row of 30 pages 15.4 / 14.6, of
// 40 15.6 / 17.0, of 62 15.8 / 24.2; 2 rows of 31 16.4 / 14.6, 3 of 21 18.1 / 12.3, 4 of 16 19.3 / 9.8; past 64 two rows of 46 15.7 /
// 19.4, but 32 of 20 31.1 / 11.3: who knows that the longest row is that short takes delta_paged_prefill).
bool prefill_alone(int64_t pages, int batch) { return pages <= (batch == 1 ? 32 : 64); }

size_t prefix_workspace_bytes(int64_t tokens, int hq, int hkv, int64_t max_pages) {
  const size_t n = workspace_bytes_for(tokens, hq, hkv, plan_blocks(tokens, hkv, max_pages, kSlots));
  if (!decode_alone(tokens, hkv, max_pages)) return n;
  const size_t alone = delta_paged_decode_workspace_bytes((int)tokens, hq, hkv, (int)max_pages);
  return n > alone ? n : alone;
}

int check_prefix(const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *kv_cache, int64_t num_pages,
                 const int32_t *kv_indptr, const int32_t *kv_indices, int64_t kv_indices_len,
                 const int32_t *kv_last_page_len, const delta_shared_prefix_t *px, const void *o, int64_t o_stride_t,
                 int64_t o_stride_h, int batch, int64_t tokens, int hq, int hkv, int head_dim, int dtype, int64_t max_pages,
                 const void *workspace, size_t workspace_bytes, const char *who) {
  clear_error();
  if (batch <= 0 || tokens <= 0) return DELTA_OK;
  if (head_dim != kHeadDim) return set_error(DELTA_ERR_INVALID, "%s: head_dim must be 128", who);
  if (hkv <= 0 || hq <= 0 || hq % hkv)
    return set_error(DELTA_ERR_INVALID, "%s: num_qo_heads must be a multiple of num_kv_heads", who);
  const int G = hq / hkv;
  if (G > kMaxGroup) return set_error(DELTA_ERR_INVALID, "%s: group size %d > %d unsupported", who, G, kMaxGroup);
  if (dtype != DELTA_BF16 && dtype != DELTA_FP16) return set_error(DELTA_ERR_INVALID, "%s: bad dtype", who);
  if (!px) return set_error(DELTA_ERR_INVALID, "%s: null prefix", who);
  if (batch > kMaxRows || px->num_prefixes > kMaxRows || px->num_prefixes < 0)
    return set_error(DELTA_ERR_INVALID, "%s: at most %d rows and prefixes (got %d, %d)", who, kMaxRows, batch,
                     px->num_prefixes);
  if (!q || !kv_cache || !kv_indptr || !kv_indices || !kv_last_page_len || !o || !px->row_prefix ||
      (px->num_prefixes > 0 && !px->indptr) || (px->indices_len > 0 && !px->indices))
    return set_error(DELTA_ERR_INVALID, "%s: null pointer", who);
  if (((uintptr_t)q | (uintptr_t)kv_cache) & 15u || (q_stride_t % 8) || (q_stride_h % 8))
    return set_error(DELTA_ERR_INVALID, "%s: q and kv_cache 16-byte aligned, q strides multiples of 8", who);
  if (((uintptr_t)o & 3u) || (o_stride_t % 2) || (o_stride_h % 2))
    return set_error(DELTA_ERR_INVALID, "%s: o 4-byte aligned with even strides", who);
  if (num_pages <= 0 || kv_indices_len < 0 || px->indices_len < 0 || kv_indices_len > INT32_MAX / kPageSize ||
      px->indices_len > INT32_MAX / kPageSize)
    return set_error(DELTA_ERR_INVALID, "%s: empty cache or bad table lengths", who);
  // The line's length (each segment's tiles, at most all tokens', times its stages) and the partials' rows stay below 2^30.
  const int64_t steps = ceil_div(kv_indices_len, kPages) + ceil_div(px->indices_len, kPages) +
                        (kTileCost + 1) * ((int64_t)batch + px->num_prefixes);
  if (tokens > 1 << 23 || (ceil_div(tokens * G, kQ) + 1) * steps > 1 << 30 || partial_rows(tokens, hq, hkv, kSlots) > 1 << 30)
    return set_error(DELTA_ERR_INVALID, "%s: too many query tokens", who);
  const size_t need = prefix_workspace_bytes(tokens, hq, hkv, max_pages);
  if (!workspace || workspace_bytes < need)
    return set_error(DELTA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
  if ((uintptr_t)workspace & 255u) return set_error(DELTA_ERR_INVALID, "%s: workspace must be 256-byte aligned", who);
  return DELTA_OK;
}

// Arguments checked by check_prefix.
int run_prefix(const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *kv_cache, int64_t num_pages,
               const int32_t *qo_indptr, const int32_t *kv_indptr, const int32_t *kv_indices, int64_t kv_indices_len,
               const int32_t *kv_last_page_len, const delta_shared_prefix_t *px, void *o, int64_t o_stride_t,
               int64_t o_stride_h, float *lse, int batch, int64_t tokens, int hq, int hkv, int dtype, float sm_scale,
               int64_t max_pages, void *workspace, delta_stream_t stream, const char *who) {
  const int G = hq / hkv;
  PrefixArgs a;
  a.q = (const uint16_t *)q;
  a.q_stride_t = q_stride_t;
  a.q_stride_h = q_stride_h;
  a.kv = (const uint16_t *)kv_cache;
  a.num_pages = num_pages;
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.kv_indices = kv_indices;
  a.kv_indices_len = kv_indices_len;
  a.last_page_len = kv_last_page_len;
  a.row_prefix = px->row_prefix;
  a.prefix_indptr = px->indptr;
  a.prefix_indices = px->indices;
  a.prefix_indices_len = px->indices_len;
  a.num_prefixes = px->num_prefixes;
  a.o = (uint16_t *)o;
  a.o_stride_t = o_stride_t;
  a.o_stride_h = o_stride_h;
  a.lse = lse;
  a.batch = batch;
  a.tokens = (int)tokens;
  a.hq = hq;
  a.hkv = hkv;
  a.blocks = plan_blocks(tokens, hkv, max_pages, resident_blocks(px->num_prefixes, batch));
  a.sm_scale = sm_scale;
  const size_t rows = partial_rows(tokens, hq, hkv, a.blocks);
  char *ws = (char *)workspace;
  a.part_ml = (float *)ws;
  ws += align256(rows * 2 * sizeof(float));
  a.part_acc = (float *)ws;
  ws += align256(rows * kHeadDim * sizeof(float));
  a.runs = (int2 *)ws;
  if (dtype == DELTA_BF16)
    launch<DELTA_BF16>(a, G, (hipStream_t)stream);
  else
    launch<DELTA_FP16>(a, G, (hipStream_t)stream);
  return check_launch(who);
}

}  // namespace
}  // namespace delta

extern "C" DELTA_EXPORT size_t delta_prefix_attention_workspace_bytes(int64_t tokens, int num_qo_heads,
                                                                      int num_kv_heads, int64_t max_pages) {
  if (tokens <= 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || num_qo_heads % num_kv_heads || max_pages < 0 ||
      max_pages > INT32_MAX || tokens > INT32_MAX)
    return 0;
  return delta::prefix_workspace_bytes(tokens, num_qo_heads, num_kv_heads, max_pages > 1 ? max_pages : 1);
}

extern "C" DELTA_EXPORT int delta_paged_decode_prefix(
    const delta_shared_prefix_t *prefix, const void *q, int64_t q_stride_b, int64_t q_stride_h, const void *kv_cache,
    int64_t num_pages, const int32_t *kv_indptr, const int32_t *kv_indices, int64_t kv_indices_len,
    const int32_t *kv_last_page_len, void *o, int64_t o_stride_b, int64_t o_stride_h, float *lse, int batch,
    int num_qo_heads, int num_kv_heads, int head_dim, int dtype, float sm_scale, int max_pages_per_row,
    void *workspace, size_t workspace_bytes, delta_stream_t stream) {
  const char *who = "delta_paged_decode_prefix";
  if (max_pages_per_row <= 0) max_pages_per_row = 1;
  const int rc = delta::check_prefix(q, q_stride_b, q_stride_h, kv_cache, num_pages, kv_indptr, kv_indices, kv_indices_len,
                                     kv_last_page_len, prefix, o, o_stride_b, o_stride_h, batch, batch, num_qo_heads,
                                     num_kv_heads, head_dim, dtype, max_pages_per_row, workspace, workspace_bytes, who);
  if (rc != DELTA_OK || batch <= 0) return rc;
  if (delta::decode_alone(batch, num_kv_heads, max_pages_per_row))
    return delta_paged_decode(q, q_stride_b, q_stride_h, kv_cache, num_pages, kv_indptr, kv_indices, kv_indices_len,
                              kv_last_page_len, o, o_stride_b, o_stride_h, lse, nullptr, 0, 0, batch, num_qo_heads,
                              num_kv_heads, head_dim, dtype, sm_scale, max_pages_per_row, workspace, workspace_bytes,
                              stream);
  return delta::run_prefix(q, q_stride_b, q_stride_h, kv_cache, num_pages, nullptr, kv_indptr, kv_indices,
                           kv_indices_len, kv_last_page_len, prefix, o, o_stride_b, o_stride_h, lse, batch, batch,
                           num_qo_heads, num_kv_heads, dtype, sm_scale, max_pages_per_row, workspace, stream, who);
}

extern "C" DELTA_EXPORT int delta_paged_prefill_prefix(
    const delta_shared_prefix_t *prefix, const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *kv_cache,
    int64_t num_pages, const int32_t *qo_indptr, const int32_t *kv_indptr, const int32_t *kv_indices,
    int64_t kv_indices_len, const int32_t *kv_last_page_len, void *o, int64_t o_stride_t, int64_t o_stride_h,
    float *lse, int batch, int64_t num_tokens, int max_qo_len, int num_qo_heads, int num_kv_heads, int head_dim, int dtype,
    float sm_scale, void *workspace, size_t workspace_bytes, delta_stream_t stream) {
  const char *who = "delta_paged_prefill_prefix";
  if (max_qo_len <= 0) num_tokens = 0;
  if (batch > 0 && num_tokens > 0 && !qo_indptr) {
    delta::clear_error();
    return delta::set_error(DELTA_ERR_INVALID, "%s: null pointer", who);
  }
  const int rc = delta::check_prefix(q, q_stride_t, q_stride_h, kv_cache, num_pages, kv_indptr, kv_indices, kv_indices_len,
                                     kv_last_page_len, prefix, o, o_stride_t, o_stride_h, batch, num_tokens, num_qo_heads,
                                     num_kv_heads, head_dim, dtype, kv_indices_len > 1 ? kv_indices_len : 1, workspace,
                                     workspace_bytes, who);
  if (rc != DELTA_OK || batch <= 0 || num_tokens <= 0) return rc;
  if (delta::prefill_alone(kv_indices_len, batch) && !((uintptr_t)o & 7u) && o_stride_t % 4 == 0 && o_stride_h % 4 == 0)
    return delta_paged_prefill_rows(q, q_stride_t, q_stride_h, kv_cache, num_pages, qo_indptr, kv_indptr, kv_indices,
                                    kv_indices_len, kv_last_page_len, o, o_stride_t, o_stride_h, lse, batch, num_qo_heads,
                                    num_kv_heads, head_dim, dtype, sm_scale, max_qo_len, num_tokens, 0, 0, 0, nullptr, 0,
                                    stream);
  return delta::run_prefix(q, q_stride_t, q_stride_h, kv_cache, num_pages, qo_indptr, kv_indptr, kv_indices,
                           kv_indices_len, kv_last_page_len, prefix, o, o_stride_t, o_stride_h, lse, batch, num_tokens,
                           num_qo_heads, num_kv_heads, dtype, sm_scale, kv_indices_len > 1 ? kv_indices_len : 1, workspace, stream,
                           who);
}
