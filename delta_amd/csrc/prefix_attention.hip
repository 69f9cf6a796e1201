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
// them come after it), or a row's own pages with its query tokens (causal).  Its (query token, q head of the
// kv head's G) pairs are cut into tiles of 128, its pages into runs of `chunk` steps of 64 tokens; a block of
// 4 waves takes one (kv head, segment, tile, run) and writes un-normalised partials (m, l, a), which the
// merge kernel joins per (token, q head).  The rows' lengths are only on the device, so every block derives
// the same plan from the tables (plan_unit): it counts the steps of all segments, sets the runs so that
// they fill the chip's block slots about once, and finds its own unit.
//
// Per block: 4 waves, a 64-token step (four pages) of K and V in LDS, the next one in flight (64 KiB, two
// blocks per CU).  With more than 64 pairs in the tile every wave owns 32 of them and sweeps the whole step;
// with 33-64 two waves share 32 pairs and take 32 tokens of the step each; with up to 32 (one decode row's
// own pages) two waves split the step and the others only load.  Waves that share pairs are joined in LDS.
// MFMA tiles as in prefill.hip: S^T = K Q^T with lane l holding query row l % 32 and 16 tokens per 32,
// O^T += V^T P^T, P rounded to the cache's type for the product as there (the sums l stay unrounded fp32).
#include <type_traits>

#include "delta_common.h"
#include "mfma32.h"

namespace delta {

namespace {

constexpr int kThreads = 256;
constexpr int kStep = 64;               // kv tokens per step
constexpr int kPages = kStep / kPageSize;
constexpr int kTileB = kStep * 256;     // bytes of a step's K (or V) tile: 64 rows of 256 bytes
constexpr int kQ = 128;                 // (token, head) pairs of a tile
constexpr int kMaxRows = 1024;          // rows, and prefixes, of a call (plan_unit's tables)
constexpr int kMaxSplits = 32;          // runs of a segment
constexpr int kMinChunk = 2;            // steps of a run, at least
constexpr int kSlots = 512;             // blocks the chip holds (two per CU)

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
  float *part_ml;      // [slot][token][q head][2]
  float *part_acc;     // [slot][token][q head][128]; slots [0, splits): prefix runs, then as many: own runs
  int32_t *tok_runs;   // [token] runs of its prefix | runs of its own tile << 16
  int batch, tokens, hq, hkv;
  int splits;          // slots of a kind
  int target;          // units per kv head that fill the chip
  float sm_scale;
};

struct RowTable {  // the plan's view of a row
  int prefix;      // -1: none applies
  int kv0, pages;  // own pages: first index in kv_indices, count
  int len;         // own tokens
  int q0, qn;      // query tokens
};

// Pages [first, first + n) of CSR entry i, clamped to the index array.
__device__ __forceinline__ void csr_pages(const int32_t *indptr, int64_t len, int i, int *first, int *n) {
  int64_t p0 = indptr[i], p1 = indptr[i + 1];
  p0 = p0 < 0 ? 0 : (p0 > len ? len : p0);
  p1 = p1 < p0 ? p0 : (p1 > len ? len : p1);
  *first = (int)p0;
  *n = (int)(p1 - p0);
}

__device__ __forceinline__ RowTable row_table(const PrefixArgs &a, int r) {
  RowTable x;
  csr_pages(a.kv_indptr, a.kv_indices_len, r, &x.kv0, &x.pages);
  int last = a.last_page_len[r];
  last = last < 0 ? 0 : (last > kPageSize ? kPageSize : last);
  x.len = x.pages > 0 ? (x.pages - 1) * kPageSize + last : 0;
  x.q0 = r;
  x.qn = 1;
  int behind = 0;  // query tokens that the prefix has to leave room for
  if (a.qo_indptr) {
    int q0 = a.qo_indptr[r], q1 = a.qo_indptr[r + 1];
    q0 = q0 < 0 ? 0 : (q0 > a.tokens ? a.tokens : q0);
    q1 = q1 < q0 ? q0 : (q1 > a.tokens ? a.tokens : q1);
    x.q0 = q0;
    behind = x.qn = q1 - q0;
  }
  x.prefix = -1;
  const int p = a.row_prefix[r];
  if (p >= 0 && p < a.num_prefixes) {
    int first, n;
    csr_pages(a.prefix_indptr, a.prefix_indices_len, p, &first, &n);
    if (n > 0 && n <= x.pages && n * kPageSize <= x.len - behind) {
      x.prefix = p;
      x.kv0 += n;
      x.pages -= n;
      x.len -= n * kPageSize;
    }
  }
  return x;
}

__device__ __forceinline__ int div_up(int a, int b) { return (a + b - 1) / b; }

// Steps of a run in a segment of `steps` steps: the plan's, unless that takes more runs than there are slots.
__device__ __forceinline__ int run_steps(int steps, int chunk, int splits) {
  const int least = div_up(steps, splits);
  return least > chunk ? least : chunk;
}

// A pointer that is the same in every lane, in scalar registers.
template <typename T>
__device__ __forceinline__ T *uniform_ptr(T *p) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  return (T *)(uintptr_t)((uint64_t)(uint32_t)uniform((int)(uint32_t)x) |
                          (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

// What a block works on.
struct Unit {
  const int32_t *ids;  // the segment's page ids
  int pages, len;      // its pages and tokens
  int pairs0, pairs;   // first (token, head) pair of the tile and how many it has
  int first_pos;       // segment position of the segment's first query token; >= len: a prefix, no mask
  int s0, s1;          // steps [s0, s1)
  int slot;            // partial slot
};

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int x = __shfl_up(v, off, 64);
    if (lane >= off) v += x;
  }
  return v;
}

// Exclusive sum over the block's threads; *total: the block's sum.  `sums` holds 4 ints; ends with a barrier
// before it is written again.
__device__ __forceinline__ int block_scan(int v, int *sums, int *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int incl = wave_scan(v, lane);
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  __syncthreads();
  *total = all;
  return before + incl - v;
}

constexpr int kPlanInts = 6 * kMaxRows + 16;

// Finds unit u; false past the last one.  `sc` (kPlanInts ints of LDS) is free again on return, toks[i] holds the
// query token of pair index (pairs0 / G + i) * G.  Writes tok_runs for the tokens of a row's first run (head 0).
template <int G>
__device__ bool plan_unit(const PrefixArgs &a, int u, bool head0, int *sc, int *toks, Unit *unit) {
  int *const cnt = sc;                    // [prefix] query tokens
  int *const psteps = sc + kMaxRows;      // [prefix] steps
  int *const rprefix = sc + 2 * kMaxRows; // [row]
  int *const rsteps = sc + 3 * kMaxRows;
  int *const rq0 = sc + 4 * kMaxRows;
  int *const rqn = sc + 5 * kMaxRows;
  int *const sums = sc + 6 * kMaxRows;    // [4]
  int *const found = sums + 4;            // item, unit within it
  const int tid = threadIdx.x;
  const int P = a.num_prefixes, B = a.batch;
  for (int p = tid; p < P; p += kThreads) cnt[p] = 0;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  int work = 0;
  for (int r = tid; r < B; r += kThreads) {
    const RowTable x = row_table(a, r);
    const int steps = div_up(x.len, kStep);
    rprefix[r] = x.prefix;
    rsteps[r] = steps;
    rq0[r] = x.q0;
    rqn[r] = x.qn;
    if (x.prefix >= 0) atomicAdd(&cnt[x.prefix], x.qn);
    work += div_up(x.qn * G, kQ) * (steps > 1 ? steps : 1);
  }
  __syncthreads();
  for (int p = tid; p < P; p += kThreads) {
    int first, n;
    csr_pages(a.prefix_indptr, a.prefix_indices_len, p, &first, &n);
    psteps[p] = div_up(n, kPages);
    work += div_up(cnt[p] * G, kQ) * psteps[p];
  }
  int total;
  block_scan(work, sums, &total);
  int chunk = div_up(total, a.target);
  chunk = chunk < kMinChunk ? kMinChunk : chunk;
  // Items: the prefixes, then the rows.
  auto tiles_of = [&](int i) { return div_up((i < P ? cnt[i] : rqn[i - P]) * G, kQ); };
  auto steps_of = [&](int i) { return i < P ? psteps[i] : (rsteps[i - P] > 1 ? rsteps[i - P] : 1); };
  auto runs_of = [&](int steps) { return div_up(steps, run_steps(steps, chunk, a.splits)); };
  int base = 0;
  for (int i0 = 0; i0 < P + B; i0 += kThreads) {
    const int i = i0 + tid;
    const int n = i < P + B ? tiles_of(i) * runs_of(steps_of(i)) : 0;
    const int at = base + block_scan(n, sums, &total);
    if (u >= at && u < at + n) {
      found[0] = i;
      found[1] = u - at;
    }
    base += total;
    if (u < base) break;
  }
  __syncthreads();
  const int item = uniform(found[0]), v = uniform(found[1]);  // (read as scalars: the compiler cannot see it)
  if (item < 0) return false;
  const int tiles = tiles_of(item), steps = steps_of(item), each = run_steps(steps, chunk, a.splits);
  const int run = v / tiles, tile = tiles - 1 - (v - run * tiles);  // a row's last tile attends the most
  const int nq = (item < P ? cnt[item] : rqn[item - P]) * G;
  unit->pairs0 = tile * kQ;
  unit->pairs = min(kQ, nq - tile * kQ);
  unit->s0 = run * each;
  unit->s1 = min(steps, unit->s0 + each);
  const int t0 = unit->pairs0 / G, t1 = (unit->pairs0 + unit->pairs - 1) / G + 1;  // tokens of the tile
  if (item < P) {
    int first, n;
    csr_pages(a.prefix_indptr, a.prefix_indices_len, item, &first, &n);
    unit->ids = a.prefix_indices + first;
    unit->pages = n;
    unit->len = n * kPageSize;
    unit->first_pos = unit->len;
    unit->slot = run;
    // The tile's tokens out of those of the prefix's rows, row by row.
    int before = 0;
    for (int r0 = 0; r0 < B; r0 += kThreads) {
      const int r = r0 + tid;
      const int n_r = r < B && rprefix[r] == item ? rqn[r] : 0;
      const int at = before + block_scan(n_r, sums, &total);
      for (int k = t0 > at ? t0 - at : 0; k < n_r && at + k < t1; ++k) toks[at + k - t0] = rq0[r] + k;
      before += total;
      if (before >= t1) break;
    }
  } else {
    const int r = item - P;
    const RowTable x = row_table(a, r);
    unit->ids = a.kv_indices + x.kv0;
    unit->pages = x.pages;
    unit->len = x.len;
    unit->first_pos = x.len - x.qn;
    const int reach = unit->first_pos + t1;  // tokens that the tile's last query token attends
    unit->s1 = min(unit->s1, reach > 0 ? div_up(min(reach, x.len), kStep) : 0);
    unit->slot = a.splits + run;
    const int pruns = x.prefix >= 0 ? runs_of(psteps[x.prefix]) : 0;
    for (int k = tid; k < t1 - t0; k += kThreads) {
      toks[k] = x.q0 + t0 + k;
      if (head0 && run == 0) a.tok_runs[x.q0 + t0 + k] = pruns | (runs_of(steps) << 16);
    }
  }
  __syncthreads();
  return true;
}

template <int DT, int G>
__global__ void __launch_bounds__(kThreads, 2) prefix_attention_kernel(PrefixArgs a) {
#pragma clang fp contract(off)
  using MF = Mfma32<DT>;
  // Step buffers, each the K tile, then the V tile (swizzled rows), shared by the block's waves; the plan's tables
  // before the first step, the joined waves' accumulators after the last.
  __shared__ __attribute__((aligned(1024))) char tiles[2][2 * kTileB];
  __shared__ int toks[kQ + 2];
  static_assert(kPlanInts * sizeof(int) <= sizeof(tiles), "the plan's tables lie in the step buffers");

  const int lane = threadIdx.x & 63, hl = lane >> 5, n = lane & 31;
  const int wv = uniform((int)(threadIdx.x >> 6));
  const int h = blockIdx.x;
  Unit un;
  if (!plan_unit<G>(a, (int)(blockIdx.z * gridDim.y + blockIdx.y), h == 0, reinterpret_cast<int *>(&tiles[0][0]), toks,
                    &un))
    return;  // whole block
  const int np = uniform(un.pages), len = uniform(un.len), s0 = uniform(un.s0), s1 = uniform(un.s1);
  const int pairs = uniform(un.pairs);

  // The wave's pairs (32 from 32 qsub on) and 32-token halves of each step.
  const int groups = pairs > 64 ? 4 : (pairs > 32 ? 2 : 1);
  const int qsub = wv & (groups - 1);
  const int half = groups == 4 ? 0 : wv / groups;  // the wave's half (groups 4: both)
  const bool active = half < 2 && 32 * qsub < pairs;

  // This lane's pair: token and head, and the last position of the segment that it attends.
  const int pair = 32 * qsub + n;
  const bool row_ok = active && pair < pairs;
  const int pt = (un.pairs0 + (row_ok ? pair : 0)) / G, g = (un.pairs0 + (row_ok ? pair : 0)) % G;
  const int t = toks[pt - un.pairs0 / G];
  const int lim = un.first_pos >= len ? len - 1 : un.first_pos + pt;
  u32x4 qf[8];  // B operand of S^T = K Q^T: d = 16 ks + 8 hl + [0, 8)
  if (row_ok) {
    // A negative scale flips q's signs, scale 0 clears q: the scale below is then positive.
    const uint32_t flip = a.sm_scale < 0.f ? 0x80008000u : 0u, keep = a.sm_scale == 0.f ? 0u : 0xffffffffu;
    const uint16_t *qp = a.q + (int64_t)t * a.q_stride_t + (int64_t)(h * G + g) * a.q_stride_h + 8 * hl;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
      qf[ks] = (ld128(qp + 16 * ks) ^ u32x4{flip, flip, flip, flip}) & u32x4{keep, keep, keep, keep};
  } else {
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qf[ks] = u32x4{0u, 0u, 0u, 0u};
  }
  const float scale2 = a.sm_scale == 0.f ? 1.f : fabsf(a.sm_scale) * kLog2e;
  // Steps that end at or below the position of the wave's first token need no causal mask.
  const int wpos = un.first_pos >= len ? len - 1 : un.first_pos + (un.pairs0 + 32 * qsub) / G;

  // Step loads: K and V rows go straight to LDS, 1 KiB (4 rows of this head) per load: wave w loads rows 4 w .. + 3 of
  // each of the step's four pages, K and V.  16-byte chunk ch of K row r sits at slot ch ^ (r % 16) and of V row r at
  // ch ^ 4 (r % 4), so that the fragment reads cover the banks once.
  const uint32_t row_bytes = (uint32_t)a.hkv * kHeadDim * 2;
  const uint32_t page_bytes = 2 * kPageSize * row_bytes;
  const int lrow = lane >> 4, lch = lane & 15;
  const uint32_t koff = (4 * wv + lrow) * row_bytes + 16 * (lch ^ (4 * wv + lrow));
  const uint32_t voff = (kPageSize + 4 * wv + lrow) * row_bytes + 16 * (lch ^ (4 * lrow));
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)&tiles[0][0] + wv * 1024;
  const char *const kvh = reinterpret_cast<const char *>(a.kv) + (int64_t)h * (kHeadDim * 2);
  const int32_t *const ids = uniform_ptr(un.ids);
  auto page_bad = [&](int pid) { return pid < 0 || (int64_t)pid >= a.num_pages; };
  // Page ids outside the cache are looked for once, over the run's pages.
  bool run_bad = false;
  for (int i = s0 * kPages; i < s1 * kPages && i < np; i += 64)
    run_bad |= __ballot(i + lane < np && i + lane < s1 * kPages && page_bad(ids[i + lane < np ? i + lane : 0])) != 0;
  // The step's page ids by scalar loads (their waits leave the tile loads in flight), a step ahead; pages past the
  // segment repeat its last one (masked later).
  int id[kPages];
  auto load_ids = [&](int j) {
#pragma unroll
    for (int i = 0; i < kPages; ++i) {
      const int pg = kPages * j + i;
      id[i] = ld_scalar(ids, pg < np ? pg : np - 1);
    }
  };
  auto bad_of = [&](int j) {  // bit i: page i of step j lies outside the cache
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < kPages; ++i) {
      const int pg = kPages * j + i;
      r |= (pg < np && page_bad(ld_scalar(ids, pg < np ? pg : np - 1)) ? 1u : 0u) << i;
    }
    return r;
  };
  auto issue = [&](int j) {  // step j's loads, then the ids of step j + 1
#pragma unroll
    for (int i = 0; i < kPages; ++i) {
      const char *pbase = uniform_ptr(kvh + (uint64_t)(uint32_t)(run_bad && page_bad(id[i]) ? 0 : id[i]) * page_bytes);
      const uint32_t dst = lds0 + (uint32_t)(j & 1) * (2 * kTileB) + i * 4096;
      load_lds_1k(dst, pbase, koff);
      load_lds_1k(dst + kTileB, pbase, voff);
    }
    load_ids(j + 1);
  };
  if (s0 < s1) {
    load_ids(s0);
    issue(s0);
  }

  float m = -INFINITY, l = 0.f;
  f32x16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
  uint32_t kfo[8];  // K fragment of k-slice ks: row n, chunk 2 ks + hl
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) kfo[ks] = (uint32_t)(n * 256 + 16 * ((2 * ks + hl) ^ (n & 15)));
  // ds_read_b64_tr_b16 of V^T: 16-lane group q16 = lane / 16, t16 = lane % 16 reads rows (kv) base + t16 / 4 at columns
  // 32 dt + 16 (q16 % 2) + 4 (t16 % 4), and receives its column's four rows.
  const int q16 = lane >> 4, t16 = lane & 15;
  uint32_t vfo[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
    vfo[dt] = (uint32_t)(kTileB + (4 * hl + (t16 >> 2)) * 256 +
                         16 * ((4 * dt + 2 * (q16 & 1) + ((t16 & 3) >> 1)) ^ (4 * (t16 >> 2))) + 8 * (t16 & 1));

  // 32-token halves [h0, h0 + NS) of step j (tile tk): scores, online softmax, P.V.
  auto sweep = [&](auto ns, int j, const char *tk, int h0, uint32_t bad) {
    constexpr int NS = decltype(ns)::value;
    f32x16 S[NS];
#pragma unroll
    for (int sb = 0; sb < NS; ++sb)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[sb][i] = 0.f;
    const char *tkh = tk + h0 * 8192;
    auto kfrag = [&](int sb, int ks) { return *reinterpret_cast<const u32x4 *>(tkh + kfo[ks] + sb * 8192); };
    u32x4 kq[4][NS];
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
      for (int sb = 0; sb < NS; ++sb) kq[s][sb] = kfrag(sb, s);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      if (ks + 3 < 8) {
#pragma unroll
        for (int sb = 0; sb < NS; ++sb) kq[(ks + 3) % 4][sb] = kfrag(sb, ks + 3);
      }
#pragma unroll
      for (int sb = 0; sb < NS; ++sb) S[sb] = MF::run(kq[ks % 4][sb], qf[ks], S[sb]);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int kv0 = j * kStep + 32 * h0;
    constexpr int NX = 16 * NS;
    const bool full = kv0 + 32 * NS - 1 <= wpos && kv0 + 32 * NS <= len && bad == 0;
    float x[NX];
    float pm = -INFINITY;
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      x[i] = S[i >> 4][i & 15];
      if (!full) {
        const int mm = 32 * (i >> 4) + 8 * ((i & 15) >> 2) + 4 * hl + (i & 3);
        const int tk_i = kv0 + mm;
        const bool pg_ok = ((bad >> (2 * h0 + (mm >> 4))) & 1u) == 0;
        x[i] = pg_ok && tk_i <= lim && tk_i < len ? x[i] : -INFINITY;
      }
      pm = fmaxf(pm, x[i]);
    }
    // m is a reference maximum: it moves only when a score exceeds it by more than 8 (log2), so the exponentials
    // stay <= 256 and the accumulators are rescaled on few steps.
    const float smax = halves_max(pm) * scale2;
    float alpha = 1.f;
    if (smax > m + 8.f) {  // also the first finite score (m = -inf)
      alpha = fast_exp2(m - smax);
      m = smax;
    }
    const float nm = m == -INFINITY ? 0.f : -m;
    float ps = 0.f;
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      x[i] = fast_exp2(fmaf(x[i], scale2, nm));
      ps += x[i];
    }
    l = l * alpha + ps;  // this half-wave's tokens; joined once at the end
    if (__ballot(alpha != 1.f)) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
    }
    u32x4 pc[2 * NS];
#pragma unroll
    for (int cc = 0; cc < 2 * NS; ++cc)
#pragma unroll
      for (int w = 0; w < 4; ++w) pc[cc][w] = pack2<DT>(x[8 * cc + 2 * w], x[8 * cc + 2 * w + 1]);
    auto vfrag = [&](int i) {  // V^T fragment of 16-token chunk i / 4, d tile i % 4
      const char *rd = tkh + vfo[i % 4] + (i / 4) * 4096;
      const ps4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ps4_t *)rd);
      const ps4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ps4_t *)(rd + 2048));
      const uint2 lo = __builtin_bit_cast(uint2, v0), hi = __builtin_bit_cast(uint2, v1);
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
    constexpr int kAhead = 4;
    u32x4 vq[kAhead + 1];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vq[i] = vfrag(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8 * NS; ++i) {
      if (i + kAhead < 8 * NS) vq[(i + kAhead) % (kAhead + 1)] = vfrag(i + kAhead);
      acc[i % 4] = MF::run(vq[i % (kAhead + 1)], pc[i / 4], acc[i % 4]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  for (int j = s0; j < s1; ++j) {
    wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint32_t bad = run_bad ? bad_of(j) : 0u;
    if (j + 1 < s1) issue(j + 1);
    if ((j + 1) * kStep > len || bad != 0) {
      // V rows past the segment and of pages outside the cache meet p = 0 but may hold NaN/Inf: zeros.
      const int r = (int)threadIdx.x >> 2;
      if (j * kStep + r >= len || ((bad >> (r >> 4)) & 1u)) {
        char *vr = &tiles[j & 1][kTileB + r * 256 + 64 * ((int)threadIdx.x & 3)];
#pragma unroll
        for (int i = 0; i < 4; ++i) st128(vr + 16 * i, u32x4{0u, 0u, 0u, 0u});
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    if (active) {
      const char *tk = &tiles[j & 1][0];
      if (groups == 4)
        sweep(std::integral_constant<int, 2>(), j, tk, 0, bad);
      else
        sweep(std::integral_constant<int, 1>(), j, tk, half, bad);
    }
  }

  l = halves_sum(l);
  if (groups < 4) {
    // Join the waves that took the two halves: the second's (m, l, acc) through LDS.
    float *const buf = reinterpret_cast<float *>(&tiles[0][0]) + qsub * (66 * 64) + lane;
    __syncthreads();
    if (half == 1 && active) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) buf[64 * (16 * dt + i)] = acc[dt][i];
      buf[64 * 64] = m;
      buf[64 * 65] = l;
    }
    __syncthreads();
    if (half == 0 && active) {
      const float m2 = buf[64 * 64], l2 = buf[64 * 65];
      const float M = fmaxf(m, m2), ref = M == -INFINITY ? 0.f : M;
      const float w1 = fast_exp2(m - ref), w2 = fast_exp2(m2 - ref);
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] = acc[dt][i] * w1 + buf[64 * (16 * dt + i)] * w2;
      l = l * w1 + l2 * w2;
      m = M;
    }
  }
  if (row_ok && half == 0) {
    const int64_t at = ((int64_t)un.slot * a.tokens + t) * a.hq + h * G + g;
    float *op = a.part_acc + at * kHeadDim + 4 * hl;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<f32x4 *>(op + 32 * dt + 8 * q4) =
            f32x4{acc[dt][4 * q4], acc[dt][4 * q4 + 1], acc[dt][4 * q4 + 2], acc[dt][4 * q4 + 3]};
    if (hl == 0) *reinterpret_cast<float2 *>(a.part_ml + at * 2) = float2{m, l};
  }
}

// Joins the runs of each (token, q head): one wave each, lane i reading slot i's (m, l) (the prefix's runs from lane
// 0 on, the row's own from lane kMaxSplits on), then two of the 128 outputs per lane over all runs.
template <int DT>
__global__ void __launch_bounds__(kThreads) prefix_merge_kernel(PrefixArgs a) {
  using E = Elem<DT>;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (row >= (int64_t)a.tokens * a.hq) return;
  const int t = uniform((int)(row / a.hq)), hq = uniform((int)(row % a.hq));
  const int lane = threadIdx.x & 63;
  // (a query token of no row is left as it was; the limits keep a table that is no CSR inside the slots)
  if (a.qo_indptr && (t < a.qo_indptr[0] || t >= a.qo_indptr[a.batch])) return;
  const int runs = uniform(a.tok_runs[t]);
  const int np = min(runs & 0xffff, a.splits), no = min((runs >> 16) & 0xffff, a.splits);
  const int64_t stride = (int64_t)a.tokens * a.hq, at = (int64_t)t * a.hq + hq;
  const bool own = lane >= kMaxSplits;
  const int s = own ? lane - kMaxSplits : lane;
  const bool have = s < (own ? no : np);
  float ms = -INFINITY, ls = 0.f;
  if (have) {
    const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + ((own ? a.splits + s : s) * stride + at) * 2);
    ms = ml.x;
    ls = ml.y;
  }
  float M = ms;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, shfl_xor(M, off));
  const float w = fast_exp2(ms - (M == -INFINITY ? 0.f : M));  // 0 where nothing was attended
  float L = ls * w;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) L += shfl_xor(L, off);
  float2 A = {0.f, 0.f};
  auto add = [&](int slot, int from) {
    const float2 x = *reinterpret_cast<const float2 *>(a.part_acc + (slot * stride + at) * kHeadDim + 2 * lane);
    const float ws = readlane(w, from);
    A.x = fmaf(x.x, ws, A.x);
    A.y = fmaf(x.y, ws, A.y);
  };
  for (int i = 0; i < np; ++i) add(i, i);
  for (int i = 0; i < no; ++i) add(a.splits + i, kMaxSplits + i);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint32_t *op = reinterpret_cast<uint32_t *>(a.o + (int64_t)t * a.o_stride_t + (int64_t)hq * a.o_stride_h);
  op[lane] = E::from_float(A.x * inv) | (E::from_float(A.y * inv) << 16);
  if (lane == 0 && a.lse) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// Runs per segment that can be useful: as many as fill the chip when the tokens share one prefix, none shorter than
// kMinChunk steps.
int plan_splits(int64_t tokens, int hq, int hkv, int64_t max_pages) {
  const int64_t tiles = ceil_div(tokens * (hq / hkv), kQ);
  int64_t n = ceil_div(ceil_div(kSlots, hkv), tiles > 0 ? tiles : 1);
  const int64_t most = ceil_div(ceil_div(max_pages, kPages), kMinChunk);
  n = n < most ? n : most;
  return (int)(n < 1 ? 1 : (n > kMaxSplits ? kMaxSplits : n));
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t workspace_bytes_for(int64_t tokens, int hq, int splits) {
  const size_t rows = (size_t)2 * splits * tokens * hq;
  return align256(rows * 2 * sizeof(float)) + align256(rows * kHeadDim * sizeof(float)) +
         align256((size_t)tokens * sizeof(int32_t));
}

template <int DT, int G>
void launch_g(const PrefixArgs &a, hipStream_t stream) {
  // Every unit of plan_unit: at most total / chunk (<= target) and one per (segment, tile).
  const int64_t tiles = ceil_div((int64_t)a.tokens * G, kQ);
  const int64_t units = a.target + 2 * tiles + a.batch + (a.num_prefixes < a.batch ? a.num_prefixes : a.batch);
  const int64_t y = units < 32768 ? units : 32768;
  hipLaunchKernelGGL((prefix_attention_kernel<DT, G>), dim3((unsigned)a.hkv, (unsigned)y, (unsigned)ceil_div(units, y)),
                     dim3(kThreads), 0, stream, a);
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
  const int64_t rows = (int64_t)a.tokens * a.hq;
  hipLaunchKernelGGL((prefix_merge_kernel<DT>), dim3((unsigned)ceil_div(rows, kThreads / 64)), dim3(kThreads), 0, stream, a);
}

int run_prefix(const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *kv_cache, int64_t num_pages,
               const int32_t *qo_indptr, const int32_t *kv_indptr, const int32_t *kv_indices, int64_t kv_indices_len,
               const int32_t *kv_last_page_len, const delta_shared_prefix_t *px, void *o, int64_t o_stride_t,
               int64_t o_stride_h, float *lse, int batch, int64_t tokens, int hq, int hkv, int head_dim, int dtype,
               float sm_scale, int64_t max_pages, void *workspace, size_t workspace_bytes, delta_stream_t stream,
               const char *who) {
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
  if (tokens * G > INT32_MAX / 2) return set_error(DELTA_ERR_INVALID, "%s: too many query tokens", who);
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
  a.splits = plan_splits(tokens, hq, hkv, max_pages);
  a.target = (int)ceil_div(kSlots, hkv);
  a.sm_scale = sm_scale;
  const size_t need = workspace_bytes_for(tokens, hq, a.splits);
  if (!workspace || workspace_bytes < need)
    return set_error(DELTA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
  if ((uintptr_t)workspace & 255u) return set_error(DELTA_ERR_INVALID, "%s: workspace must be 256-byte aligned", who);
  const size_t rows = (size_t)2 * a.splits * tokens * hq;
  char *ws = (char *)workspace;
  a.part_ml = (float *)ws;
  ws += align256(rows * 2 * sizeof(float));
  a.part_acc = (float *)ws;
  ws += align256(rows * kHeadDim * sizeof(float));
  a.tok_runs = (int32_t *)ws;
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
  if (tokens <= 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || num_qo_heads % num_kv_heads || max_pages < 0) return 0;
  return delta::workspace_bytes_for(tokens, num_qo_heads,
                                    delta::plan_splits(tokens, num_qo_heads, num_kv_heads, max_pages));
}

extern "C" DELTA_EXPORT int delta_paged_decode_prefix(
    const delta_shared_prefix_t *prefix, const void *q, int64_t q_stride_b, int64_t q_stride_h, const void *kv_cache,
    int64_t num_pages, const int32_t *kv_indptr, const int32_t *kv_indices, int64_t kv_indices_len,
    const int32_t *kv_last_page_len, void *o, int64_t o_stride_b, int64_t o_stride_h, float *lse, int batch,
    int num_qo_heads, int num_kv_heads, int head_dim, int dtype, float sm_scale, int max_pages_per_row,
    void *workspace, size_t workspace_bytes, delta_stream_t stream) {
  return delta::run_prefix(q, q_stride_b, q_stride_h, kv_cache, num_pages, nullptr, kv_indptr, kv_indices,
                           kv_indices_len, kv_last_page_len, prefix, o, o_stride_b, o_stride_h, lse, batch, batch,
                           num_qo_heads, num_kv_heads, head_dim, dtype, sm_scale, max_pages_per_row, workspace,
                           workspace_bytes, stream, "delta_paged_decode_prefix");
}

extern "C" DELTA_EXPORT int delta_paged_prefill_prefix(
    const delta_shared_prefix_t *prefix, const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *kv_cache,
    int64_t num_pages, const int32_t *qo_indptr, const int32_t *kv_indptr, const int32_t *kv_indices,
    int64_t kv_indices_len, const int32_t *kv_last_page_len, void *o, int64_t o_stride_t, int64_t o_stride_h,
    float *lse, int batch, int64_t num_tokens, int num_qo_heads, int num_kv_heads, int head_dim, int dtype,
    float sm_scale, void *workspace, size_t workspace_bytes, delta_stream_t stream) {
  const char *who = "delta_paged_prefill_prefix";
  if (batch > 0 && num_tokens > 0 && !qo_indptr) {
    delta::clear_error();
    return delta::set_error(DELTA_ERR_INVALID, "%s: null pointer", who);
  }
  return delta::run_prefix(q, q_stride_t, q_stride_h, kv_cache, num_pages, qo_indptr, kv_indptr, kv_indices,
                           kv_indices_len, kv_last_page_len, prefix, o, o_stride_t, o_stride_h, lse, batch, num_tokens,
                           num_qo_heads, num_kv_heads, head_dim, dtype, sm_scale, kv_indices_len, workspace,
                           workspace_bytes, stream, who);
}
