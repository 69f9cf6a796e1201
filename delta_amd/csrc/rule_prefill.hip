// Attention of several new tokens a row over the paged cache under a score rule (score_rule.h): scores capped by a tanh, a
// bias that falls with the distance, and of each query token's keys a range [lo, hi) only (causal, a window, packed
// documents, a prefix seen as a whole).  The cache already holds the new tokens; query i of row b sits at position
// kv_len_b - qo_len_b + i.
//
// Work decomposition, on the 32x32 MFMA tiles of the causal prompt kernel (prefill.hip): a block is PW waves of one (row, kv
// head) and a run of query tokens; each wave owns 32 query rows, the (token, q head) pairs of TW = 32 / G tokens, with its q
// in registers.  The block sweeps the keys that any of its tokens sees, 64 at a time from the first one's step to the last
// one's; K and V go from global memory straight to LDS.  Per wave and step S^T = K Q^T, the rule on the scores in registers,
// the online softmax, O^T += V^T P^T.  Steps that all the wave's rows see whole take no masks, steps that none of them sees
// are left out.
//
// Calls of a few hundred blocks run them with two sets of four waves, every other step each (TWO, two_sided).
//
// Few tokens over a long cache are too few blocks: the tile's steps are cut into parts, each a block of its own that writes
// its sums (acc, m, l) to the workspace, and a second launch joins them.  How many parts is a matter of all rows' lengths,
// which only the device knows: every block adds up the call's work W (tiles x steps), and with C = W hkv / kTargetBlocks
// steps (at least kMinSteps; up to kLoneSteps twice as many) a row of s steps is cut into s / C parts (row_parts).  So a
// decode row beside short prompts is cut, equal long prompts are not, and the cut rows' parts are kTargetBlocks blocks at
// most.
//
// A key that a mask leaves out has no part in the result, whatever it holds.  Its score is replaced and its p is 0, but 0
// times a V of infinity or NaN is NaN in the product of the whole tile, so a row that ends with sums that are not finite is
// summed again key by key over its own keys alone, beside their maximum (slow_row): nothing for finite caches.
//
// What bounds it: the card's power for long prompts.  8192 tokens of 32 + 8 heads under a cap of 50 take 612 us in a replayed
// graph, 0.90 PFLOP/s (an 8192^3 product 1.22; no rule 522, slopes 573; the cap in fp16 671, of 55 to 64 in bf16 662, with slopes 765, of
// 100 723): the clock falls to 1.86 GHz where matrix and ordinary instructions
// run together (1.7 the former alone, 2.3 the latter), so fewer idle cycles bring little: waves that interleave one
// sub-tile's MFMAs with another's softmax took 623-632.  Page ids by vector loads and readlane (scalar loads in flight make
// every LDS wait a full one): 666 -> 630.  A block's start, four dependent loads, is 3 us, its step 1.5 us alone on a CU and
// 2.4 beside another: what is left above the steps in short documents and windows.
#include <type_traits>

#include "delta_common.h"
#include "mfma32.h"
#include "score_rule.h"

namespace delta {
namespace {

constexpr int kSub = 2;                // 32-token sub-tiles per step
constexpr int kKvStep = 32 * kSub;     // keys per step
constexpr int kPgStep = kKvStep / 16;  // pages per step
constexpr int kTileB = kKvStep * 256;  // bytes of a step's K (or V) tile: 64 rows of 256 bytes
constexpr int kTargetBlocks = 512;     // two 4-wave blocks for each CU (TWO: half as many)
constexpr int kMinSteps = 4;           // a part's steps, at least
constexpr int kLoneSteps = 8;          // up to so many, one block for each CU
constexpr int kMaxParts = 1024;
constexpr int kJoin = 16;              // parts whose sums the join loads together
constexpr int kTwoFrom = 128, kTwoTo = 450;  // blocks of a call that are TWO (two_sided)
constexpr int kSplitWaves = 4;         // waves of a block where rows may be cut

// What the rule does to the scores, a kernel each (a branch in the step costs the instructions that the compiler moves out
// of it): nothing, a cap alone, slopes alone, anything.  kCappedRef: a cap alone, and the exponents' reference is a
// constant.
enum ScoreMode { kPlain = 0, kCapped = 1, kCappedRef = 2, kLeaning = 3, kAny = 4 };

// A cap c alone: c tanh(y), y = x s / c, in log2 units is xs r + xo with r = -1 / (1 + e^(2 y)), xs = 2 c log2 e and
// xo = c log2 e; off by 2^-22 c, so for caps up to kQuickCap (1.5e-5) and smaller ones alone.  (tanh as a polynomial of x,
// one multiply-add a degree, took 739 us where this takes 670: a step's exponentials and reciprocals cost two issue slots
// each, no more.)
constexpr float kQuickCap = 64.f;
struct CapArgs {
  float k, xs, xo;  // k = 2 log2 e s / c
  float ref;        // kCappedRef: the reference, log2 units
};

struct RulePrefillArgs {
  const uint16_t *q;
  int64_t q_stride_t, q_stride_h;
  const uint16_t *kv;
  int64_t num_pages;
  const int32_t *qo_indptr, *kv_indptr, *kv_indices;
  int64_t kv_indices_len;
  const int32_t *last_page_len;
  uint16_t *o;
  int64_t o_stride_t, o_stride_h;
  float *lse;
  int batch, hq, hkv, G;
  int token_limit;  // query tokens of all rows
  int row_tiles;    // the most tiles a row has (of max_qo_len tokens)
  int max_cut;      // units of cut rows that the workspace holds, 0: no row is cut
  bool two;         // blocks are TWO
  float sm_scale;
  RuleArgs rule;
  CapArgs cap;
  float2 *part_ml;  // [unit][hkv][wave][32 rows]
  float *part_le;   // likewise
  int *any_cut;     // whether any row is: else the join has nothing to do
  f32x4 *part_acc;  // [unit][hkv][wave][16][64 lanes], the accumulators as the lanes hold them
};

// Parts of a row of s steps, `longer`: than 1.5 times the call's mean.  A step takes about 1.5 us in a block with a CU of its own and
// 2.4 in each of two, a cut's end and join 8 us: three parts gain from 14 steps on.  Two parts of like rows (that fill 2/3 of
// the CUs uncut) gain nothing: 192 blocks of 32 steps 55 us, 384 of 16 65.
__host__ __device__ __forceinline__ int row_parts(int s, int C, bool longer) {
  const int p = s / C;
  return s < 14 || p < 2 || (p == 2 && (s < 24 || !longer)) ? 1 : p < kMaxParts ? p : kMaxParts;
}

struct RowBounds {
  int q0, q1, p0, np, kv_len;
};
__device__ __forceinline__ RowBounds row_bounds(const RulePrefillArgs &a, int r) {
  if (r >= a.batch) return RowBounds{0, 0, 0, 0, 0};
  RowBounds x;
  x.q0 = min(max(a.qo_indptr[r], 0), a.token_limit);
  x.q1 = min(max(a.qo_indptr[r + 1], 0), a.token_limit);
  const int64_t ilen = a.kv_indices_len;
  int64_t p0 = a.kv_indptr[r], p1 = a.kv_indptr[r + 1];
  p0 = p0 < 0 ? 0 : (p0 > ilen ? ilen : p0);
  p1 = p1 < p0 ? p0 : (p1 > ilen ? ilen : p1);
  int lp = a.last_page_len[r];
  lp = lp < 0 ? 0 : (lp > kPageSize ? kPageSize : lp);
  x.p0 = (int)p0;
  x.np = (int)(p1 - p0);
  x.kv_len = x.np > 0 ? (x.np - 1) * kPageSize + lp : 0;
  return x;
}
__device__ __forceinline__ RowBounds bounds_of_lane(const RowBounds &x, int l) {
  return RowBounds{__builtin_amdgcn_readlane(x.q0, l), __builtin_amdgcn_readlane(x.q1, l),
                   __builtin_amdgcn_readlane(x.p0, l), __builtin_amdgcn_readlane(x.np, l),
                   __builtin_amdgcn_readlane(x.kv_len, l)};
}

// Over a wave: the 16-lane rows by DPP, the four rows by permlane swaps.
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
  v += (uint32_t)dpp_i<0xB1>((int)v);
  v += (uint32_t)dpp_i<0x4E>((int)v);
  v += (uint32_t)dpp_i<0x141>((int)v);
  v += (uint32_t)dpp_i<0x140>((int)v);
  auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = a[0] + a[1];
  auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (uint32_t)uniform((int)(b[0] + b[1]));
}

// One block's work: part `part` of `parts` of a row's tile.
struct Unit {
  RowBounds row;
  int h, tile, part, parts;
  int slot;  // of a cut row's unit in the workspace
};

// Unit (u, h) of the launch, h the kv head: the cut rows' first, then the others' tiles row by row, a row's last tile first
// (in a causal row it sees the most keys); false past the last one.  Consecutive blocks go to the eight XCDs in turn, so a
// cut row's blocks are dealt out in groups of eight (part, head) pairs, whose tiles follow one another eight blocks apart: the
// tiles of a part read its keys from one L2 (groups of 7 over 65548 keys: 48 tokens fetch 142 MB, not 381; 32 tokens 63 us, not
// 67).
__device__ __forceinline__ bool find_unit(const RulePrefillArgs &a, int BT, int u, int h, int lane, Unit *unit) {
  auto tiles_of = [&](const RowBounds &x) {
    const int qn = x.q1 - x.q0;
    return qn <= 0 ? 0 : min((qn + BT - 1) / BT, a.row_tiles);
  };
  auto steps_of = [&](const RowBounds &x) {  // of one tile, at most
    const int span = a.rule.window > 0 && a.rule.window < x.kv_len - BT ? a.rule.window + BT : x.kv_len;
    return (span + kKvStep - 1) / kKvStep;
  };
  const int lanes = a.batch > 32 ? 64 : a.batch > 8 ? 32 : a.batch > 2 ? 8 : 2;  // that hold rows (prefix sums stop there)
  const RowBounds head = row_bounds(a, lane);  // (of most calls all rows: loaded once)
  auto rows_at = [&](int r0) { return r0 == 0 ? head : row_bounds(a, r0 + lane); };
  // Whole numbers, up to 2^47 tile steps: the kernel and its join, each block of both, cut alike.
  int C = 0;
  uint64_t w = 0;
  uint32_t t = 0;
  if (a.max_cut > 0) {
    for (int r0 = 0; r0 < a.batch; r0 += 64) {
      const RowBounds x = rows_at(r0);
      t += (uint32_t)tiles_of(x);
      w += (uint64_t)tiles_of(x) * (uint32_t)steps_of(x);
    }
    // (64 lanes' lower 26 bits add up below 2^32)
    w = ((uint64_t)wave_sum((uint32_t)(w >> 26)) << 26) + wave_sum((uint32_t)w & 0x3ffffffu);
    t = wave_sum(t);
    const uint64_t wh = w * (uint32_t)a.hkv, one = (wh + kTargetBlocks - 1) / kTargetBlocks;
    const uint64_t two = (2 * wh + kTargetBlocks - 1) / kTargetBlocks;
    const uint64_t lone = kLoneSteps, least = kMinSteps;
    const uint64_t c = a.two ? max(two, lone) : max(max(one, min(two, lone)), least);
    C = c > 100000000 ? 100000000 : (int)c;
  }
  auto parts_of = [&](const RowBounds &x) {
    const int s = steps_of(x);
    return C > 0 ? row_parts(s, C, 2 * (uint64_t)(uint32_t)s * t > 3 * w) : 1;
  };
  int base = 0;
  for (int pass = C > 0 ? 0 : 1; pass < 2; ++pass) {
    for (int r0 = 0; r0 < a.batch; r0 += 64) {
      const RowBounds mine = rows_at(r0);
      const int parts = parts_of(mine), tiles = tiles_of(mine);
      const int n = (parts > 1) == (pass == 0) ? tiles * parts : 0;
      if (__ballot(n > 0) == 0) continue;
      int incl = n;
      for (int off = 1; off < lanes; off <<= 1) {
        const int v = __shfl_up(incl, off, 64);
        if (lane >= off) incl += v;
      }
      const uint64_t m = __ballot(base + incl > u);  // (the first such lane is a row's)
      if (m != 0) {
        const int l = __builtin_ctzll(m);
        unit->row = bounds_of_lane(mine, l);
        unit->parts = __builtin_amdgcn_readlane(parts, l);
        const int nt = __builtin_amdgcn_readlane(tiles, l), end = base + __builtin_amdgcn_readlane(incl, l);
        unit->h = h;
        unit->tile = end - 1 - u;  // from the row's last
        unit->part = unit->slot = 0;
        if (unit->parts > 1) {
          const int start = end - nt * unit->parts;
          unit->tile = 0;
          unit->part = u - start;
          if (nt > 1) {
            const int rel = (u - start) * a.hkv + h, group = rel / (8 * nt), r = rel - group * 8 * nt;
            const int wide = min(8, unit->parts * a.hkv - 8 * group);
            unit->tile = r / wide;
            const int pair = 8 * group + r - unit->tile * wide;
            unit->part = pair / a.hkv;
            unit->h = pair - unit->part * a.hkv;
          }
          unit->slot = start + unit->tile * unit->parts + unit->part;
        }
        return true;
      }
      base += __builtin_amdgcn_readlane(incl, lanes - 1);
    }
  }
  return false;
}

// c + the sum of two packed 16-bit values, in fp32
template <int DT>
__device__ __forceinline__ float add2(uint32_t v, float c) {
  if constexpr (DT == DELTA_BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, v), __builtin_bit_cast(b2, 0x3f803f80u), c, false);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, v), __builtin_bit_cast(h2, 0x3c003c00u), c, false);
  }
}

// Likewise the largest or least value.
template <bool MAX>
__device__ __forceinline__ int wave_extreme(int v) {
  auto pick = [](int a, int b) { return MAX ? max(a, b) : min(a, b); };
  v = pick(v, dpp_i<0xB1>(v));
  v = pick(v, dpp_i<0x4E>(v));
  v = pick(v, dpp_i<0x141>(v));
  v = pick(v, dpp_i<0x140>(v));
  auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = pick((int)a[0], (int)a[1]);
  auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return uniform(pick((int)b[0], (int)b[1]));
}

template <int DT, int PW, bool TWO, int SM>
__global__ void __launch_bounds__(PW * (TWO ? 128 : 64), 2) paged_prefill_rule_kernel(RulePrefillArgs a) {
#pragma clang fp contract(off)
  static_assert(!TWO || PW == 4, "TWO: 4-wave tiles");
  using E = Elem<DT>;
  using MF = Mfma32<DT>;
  constexpr bool kLate = PW == 8;   // the second wave of each SIMD runs half a step behind
  constexpr int kBufs = kLate ? 4 : 2;
  constexpr int kPgWave = 16 / PW;  // pages a wave loads rows of, per step
  constexpr int kStride = TWO ? 2 : 1;
  __shared__ __attribute__((aligned(1024))) char lds[kStride * kBufs][2 * kTileB];

  const int G = a.G, TW = 32 / G, BT = PW * TW;
  const int wave = (threadIdx.x >> 6) & (PW - 1), lane = threadIdx.x & 63;
  const int side = TWO ? uniform((int)(threadIdx.x >> 8)) : 0;  // TWO: the block's first or second four waves
  const int hl = lane >> 5, n = lane & 31;
  const int u = (int)(blockIdx.z * gridDim.y + blockIdx.y);
  Unit un;
  const bool work = find_unit(a, BT, u, (int)blockIdx.x, lane, &un);
  if (a.max_cut > 0 && u == 0 && blockIdx.x == 0 && threadIdx.x == 0) *a.any_cut = work && un.parts > 1;  // (cut rows come first)
  if (!work) return;  // whole block
  const int h = un.h;
  const int64_t q0 = un.row.q0;
  const int qn = un.row.q1 - un.row.q0, np = un.row.np, kv_len = un.row.kv_len;
  const int btok0 = un.tile * BT;
  const int tok0 = __builtin_amdgcn_readfirstlane(btok0 + wave * TW);

  // This lane's query row n = (token tt, head g) and its keys [lo, hi).
  const int tt = n / G, g = n - tt * G;
  const bool row_ok = n < TW * G && tok0 + tt < qn;
  const int qpos = kv_len - qn + tok0 + tt;
  u32x4 qf[8];  // B operand of S^T = K Q^T: d = 16 ks + 8 hl + [0, 8)
  if (row_ok) {
    const uint16_t *qp = a.q + (q0 + tok0 + tt) * a.q_stride_t + (int64_t)(h * G + g) * a.q_stride_h + 8 * hl;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qf[ks] = ld128(qp + 16 * ks);
  } else {
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qf[ks] = u32x4{0u, 0u, 0u, 0u};
  }
  int lo = 0, hi = 0;
  if (row_ok) {
    key_range(a.rule, q0 + tok0 + tt, qpos, kv_len, &lo, &hi);
    if (hi <= lo) lo = hi = 0;
  }
  // The wave's rows together: the first and last key any of them sees, and the keys that all of them see; and the block's
  // tokens together.  Without bounds of their own the tokens' ranges move up with them: the first and last one's say it all.
  const int wtok1 = min(tok0 + TW, qn), btok1 = min(btok0 + BT, qn);
  int any0, any1, all0, all1, blo, bhi;
  if (!a.rule.kv_begin && !a.rule.kv_end) {
    int unused;
    key_range(a.rule, 0, kv_len - qn + tok0, kv_len, &any0, &all1);
    key_range(a.rule, 0, kv_len - qn + wtok1 - 1, kv_len, &all0, &any1);
    if (wtok1 <= tok0) any1 = 0;
    key_range(a.rule, 0, kv_len - qn + btok0, kv_len, &blo, &unused);
    key_range(a.rule, 0, kv_len - qn + btok1 - 1, kv_len, &unused, &bhi);
  } else {
    any0 = wave_extreme<false>(hi > lo ? lo : INT32_MAX);
    any1 = wave_extreme<true>(hi);
    all0 = wave_extreme<true>(row_ok ? lo : 0);
    all1 = wave_extreme<false>(row_ok ? hi : INT32_MAX);
    blo = INT32_MAX;
    bhi = 0;
    for (int t0 = btok0; t0 < btok1; t0 += 64) {
      const int tk = t0 + lane;
      if (tk < btok1) {
        int l2, h2;
        key_range(a.rule, q0 + tk, kv_len - qn + tk, kv_len, &l2, &h2);
        if (h2 > l2) {
          blo = min(blo, l2);
          bhi = max(bhi, h2);
        }
      }
    }
    blo = wave_extreme<false>(blo);
    bhi = wave_extreme<true>(bhi);
  }
  // The block's steps [s0, s1) (its part of them) and the wave's.
  int s0 = 0, s1 = 0;
  if (bhi > blo) {
    s0 = blo / kKvStep;
    s1 = (bhi + kKvStep - 1) / kKvStep;
    if (un.parts > 1) {
      const int per = (s1 - s0 + un.parts - 1) / un.parts;
      s0 += un.part * per;
      s1 = min(s1, s0 + per);
    }
  }
  const int w0 = any1 > 0 ? max(s0, any0 / kKvStep) : 0, w1 = any1 > 0 ? min(s1, (any1 + kKvStep - 1) / kKvStep) : 0;

  // Step loads (as in prefill.hip): 1 KiB a load, 4 rows of this head; 16-byte chunk ch of K row r at slot ch ^ (r % 16),
  // of V row r at ch ^ 4 (r % 4).
  const uint32_t row_bytes = (uint32_t)a.hkv * kHeadDim * 2;
  const uint32_t page_bytes = 2 * kPageSize * row_bytes;
  const int wv = uniform(wave);
  const int lrow = lane >> 4, lch = lane & 15;
  const uint32_t koff = (4 * (wv & 3) + lrow) * row_bytes + 16 * (lch ^ (4 * (wv & 3) + lrow));
  const uint32_t voff = (kPageSize + 4 * (wv & 3) + lrow) * row_bytes + 16 * (lch ^ (4 * lrow));
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)&lds[side * kBufs][0] + wv * 1024;
  const char *const kvh = reinterpret_cast<const char *>(a.kv) + (int64_t)h * (kHeadDim * 2);
  const int32_t *const row_ids = a.kv_indices + un.row.p0;
  auto page_bad = [&](int pid) { return pid < 0 || (int64_t)pid >= a.num_pages; };
  auto bad_of = [&](int j) {  // bit i: page i of step j lies outside the cache
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < kPgStep; ++i) {
      const int pg = kPgStep * j + i;
      r |= (pg < np && page_bad(ld_scalar(row_ids, pg < np ? pg : np - 1)) ? 1u : 0u) << i;
    }
    return r;
  };
  const uint32_t last_pg = (uint32_t)(np - 1);  // (steps exist only where pages do)
  uint32_t id[kPgWave];                         // of the step issued next; pages past the row repeat its last one
  int next_ids = 0;
  auto load_ids = [&](int j) { next_ids = row_ids[min((uint32_t)(kPgStep * j + (lane & 3)), last_pg)]; };
  auto take_ids = [&]() {
    const int v = page_bad(next_ids) ? 0 : next_ids;
#pragma unroll
    for (int i = 0; i < kPgWave; ++i) id[i] = (uint32_t)__builtin_amdgcn_readlane(v, i * (PW / 4) + (wv >> 2));
  };
  auto buf = [&](int j) { return (uint32_t)(j / kStride & (kBufs - 1)); };  // of the side's buffers
  auto tile = [&](int j) { return &lds[side * kBufs + buf(j)][0]; };
  auto issue = [&](int j, int i) {
    const uint32_t dst = lds0 + buf(j) * (2 * kTileB) + i * (PW / 4) * 4096;
    const char *pg = kvh + (uint64_t)id[i] * page_bytes;
    load_lds_1k(dst, pg, koff);
    load_lds_1k(dst + kTileB, pg, voff);
  };
  auto issue_step = [&](int j) {  // step j's loads, then the ids of step j + 1
#pragma unroll
    for (int i = 0; i < kPgWave; ++i) issue(j, i);
  };
  if (s0 + side < s1) {
    load_ids(s0 + side);
    take_ids();
    load_ids(s0 + side + kStride);
    issue_step(s0 + side);
    if (kLate && s0 + 1 < s1) {
      take_ids();
      load_ids(s0 + 2);
      issue_step(s0 + 1);
    }
  }
  // With a negative scale q's signs are flipped (the scale below is then positive).  The xor also makes q's loads, in flight
  // beside the first keys', complete here, before the kv loop.
  const uint32_t flip = a.sm_scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) qf[ks] ^= u32x4{flip, flip, flip, flip};
  // Ids outside the cache are looked for once over the part's pages; steps of a row without any take its ids as they are.
  bool row_bad = false;
  for (int i = s0 * kPgStep; i < s1 * kPgStep && i < np; i += 64)
    row_bad |= __ballot(i + lane < np && i + lane < s1 * kPgStep && page_bad(row_ids[i + lane < np ? i + lane : 0])) != 0;
  uint32_t bad = 0;  // bad_of(j)

  // p is rounded to 16 bits for its product with V.  A row is divided by l, which in steps with masks adds up the rounded
  // p: a row of one key is that key's v, and a few keys' weights add up to 1.  Over whole steps the roundings of 64 keys and
  // more average out, and l takes the fp32 p as le does, the sum for the lse (rounded ones there as well took 8192 tokens
  // with a cap from 613 to 627 us).
  float m = SM == kCappedRef ? a.cap.ref : -INFINITY, l = 0.f, le = 0.f;
  f32x16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
  const float scale = fabsf(a.sm_scale), scale2 = scale * kLog2e;
  const bool capped = a.rule.softcap > 0.f, leaning = a.rule.slopes != nullptr;
  // Scores leave the rule in log2 units but for kPlain, which keeps the scale for the exponent's fma.
  const float xs = SM == kPlain || SM == kLeaning ? scale2 : SM == kAny ? 1.f : a.cap.xs;
  float xo = SM == kCapped || SM == kCappedRef ? a.cap.xo : 0.f;  // (kLeaning: of the step)
  const int first_pos = kv_len - qn + tok0;  // the wave's first query's position
  const float slope2 = leaning && row_ok ? a.rule.slopes[h * G + g] * kLog2e : 0.f;
  const float lean = slope2 / scale2;  // kLeaning: the slope in units of the unscaled scores
  uint32_t kfo[8];  // K fragment of k-slice ks: row 32 sb + n, chunk 2 ks + hl
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) kfo[ks] = (uint32_t)(n * 256 + 16 * ((2 * ks + hl) ^ (n & 15)));
  const int q16 = lane >> 4, t16 = lane & 15;
  uint32_t vfo[4];  // transposed V reads
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
    vfo[dt] = (uint32_t)(kTileB + (4 * hl + (t16 >> 2)) * 256 +
                         16 * ((4 * dt + 2 * (q16 & 1) + ((t16 & 3) >> 1)) ^ (4 * (t16 >> 2))) + 8 * (t16 & 1));

  // One step for the wave: S^T = K Q^T, the rule, the online softmax and P^T packed into pc.
  auto score_step = [&](int j, const char *tk, u32x4 (&pc)[2 * kSub]) {
    f32x16 S[kSub];
#pragma unroll
    for (int sb = 0; sb < kSub; ++sb)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[sb][i] = 0.f;
    auto kfrag = [&](int sb, int ks) { return *reinterpret_cast<const u32x4 *>(tk + kfo[ks] + sb * 8192); };
    u32x4 kq[4][kSub];  // three k-slices ahead of the MFMAs; the fences keep the reads from sinking to their uses
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
      for (int sb = 0; sb < kSub; ++sb) kq[s][sb] = kfrag(sb, s);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      if (ks + 3 < 8) {
#pragma unroll
        for (int sb = 0; sb < kSub; ++sb) kq[(ks + 3) % 4][sb] = kfrag(sb, ks + 3);
      }
#pragma unroll
      for (int sb = 0; sb < kSub; ++sb) S[sb] = MF::run(kq[ks % 4][sb], qf[ks], S[sb]);
      if (!kLate && ks < kPgWave && j + kStride < s1) issue(j + kStride, ks);  // the next step's loads go out under the MFMAs
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    const int kv0 = j * kKvStep;
    const bool full = kv0 >= all0 && kv0 + kKvStep <= all1 && bad == 0;
    constexpr int NX = 16 * kSub;
    float x[NX];
#pragma unroll
    for (int i = 0; i < NX; ++i) x[i] = S[i >> 4][i & 15];
    auto key = [&](int i) { return 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3); };  // + kv0 + 4 hl
    if constexpr (SM == kCapped || SM == kCappedRef) {
#pragma unroll
      for (int i = 0; i < NX; ++i) x[i] = __builtin_amdgcn_rcpf(-1.f - fast_exp2(x[i] * a.cap.k));
    } else if constexpr (SM == kLeaning) {
      const float d0 = (float)(qpos - kv0 - 4 * hl);
      if (kv0 + kKvStep - 1 <= first_pos) {  // no key behind a query: -lean (d0 - key), its -lean d0 a constant of the row
#pragma unroll
        for (int i = 0; i < NX; ++i) x[i] = fmaf(lean, (float)key(i), x[i]);
        xo = -slope2 * d0;
      } else {
#pragma unroll
        for (int i = 0; i < NX; ++i) x[i] = fmaf(-lean, fabsf(d0 - (float)key(i)), x[i]);
        xo = 0.f;
      }
    } else if constexpr (SM == kAny) {
      if (a.cap.k > 0.f) {  // a cap up to kQuickCap
#pragma unroll
        for (int i = 0; i < NX; ++i) x[i] = fmaf(a.cap.xs, __builtin_amdgcn_rcpf(-1.f - fast_exp2(x[i] * a.cap.k)), a.cap.xo);
      } else if (capped) {
        cap_scores(x, a.rule, scale, kLog2e);
      } else {
#pragma unroll
        for (int i = 0; i < NX; ++i) x[i] *= scale2;
      }
      if (leaning) {
        const float d0 = (float)(qpos - kv0 - 4 * hl);
#pragma unroll
        for (int i = 0; i < NX; ++i) x[i] = fmaf(-slope2, fabsf(d0 - (float)key(i)), x[i]);
      }
    }
    float pm = -INFINITY;
    if (!full) {
      const int l0 = lo - kv0 - 4 * hl, h0 = hi - kv0 - 4 * hl;
#pragma unroll
      for (int i = 0; i < NX; ++i)
        x[i] = key(i) >= l0 && key(i) < h0 && ((bad >> (2 * (i >> 4) + ((i & 15) >> 3))) & 1u) == 0 ? x[i] : -INFINITY;
    }
    float alpha = 1.f, pe = 0.f;
    if constexpr (SM == kCappedRef) {
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        x[i] = fast_exp2(fmaf(x[i], xs, xo - m));
        pe += x[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NX; ++i) pm = fmaxf(pm, x[i]);
      // m is the row's reference maximum: it moves only when a score exceeds it by more than 8 (a factor of 2^8).
      const float smax = halves_max(fmaf(pm, xs, xo));
      if (smax > m + 8.f) {  // also the first finite score of the row (m = -inf)
        alpha = fast_exp2(m - smax);
        m = smax;
      }
      const float nm = m == -INFINITY ? 0.f : xo - m;
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        x[i] = fast_exp2(fmaf(x[i], xs, nm));
        pe += x[i];
      }
      if (__ballot(alpha != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
      }
    }
#pragma unroll
    for (int cc = 0; cc < 2 * kSub; ++cc)
#pragma unroll
      for (int w = 0; w < 4; ++w) pc[cc][w] = pack2<DT>(x[8 * cc + 2 * w], x[8 * cc + 2 * w + 1]);
    float ps = pe;
    if (!full) {
      ps = 0.f;
#pragma unroll
      for (int cc = 0; cc < 2 * kSub; ++cc)
#pragma unroll
        for (int w = 0; w < 4; ++w) ps = add2<DT>(pc[cc][w], ps);
    }
    l = l * alpha + ps;  // this half's keys; the halves are summed once at the end
    le = le * alpha + pe;
  };
  // O^T += V^T P^T of a step whose P^T is in pc.
  auto pv_step = [&](const char *tk, const u32x4 (&pc)[2 * kSub]) {
    auto vfrag = [&](int i) {  // V^T fragment of chunk i / 4, d tile i % 4
      const char *rd = tk + vfo[i % 4] + (i / 4) * 4096;
      const ps4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ps4_t *)rd);
      const ps4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ps4_t *)(rd + 2048));
      u32x4 va;
      va[0] = (uint32_t)(uint16_t)v0[0] | ((uint32_t)(uint16_t)v0[1] << 16);
      va[1] = (uint32_t)(uint16_t)v0[2] | ((uint32_t)(uint16_t)v0[3] << 16);
      va[2] = (uint32_t)(uint16_t)v1[0] | ((uint32_t)(uint16_t)v1[1] << 16);
      va[3] = (uint32_t)(uint16_t)v1[2] | ((uint32_t)(uint16_t)v1[3] << 16);
      return va;
    };
    constexpr int kAhead = 4;  // fragments read ahead of their MFMAs
    u32x4 vq[kAhead + 1];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vq[i] = vfrag(i);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 8 * kSub; ++i) {
      if (i + kAhead < 8 * kSub) vq[(i + kAhead) % (kAhead + 1)] = vfrag(i + kAhead);
      acc[i % 4] = MF::run(vq[i % (kAhead + 1)], pc[i / 4], acc[i % 4]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  const bool late = kLate && wave >= PW / 2;
  u32x4 pcar[2 * kSub];
  for (int j0 = s0; s0 < s1 && j0 < s1 + (kLate ? 1 : 0); j0 += kStride) {
    const int j = j0 + side;
    // Step j's loads have landed when at most the next step's (kLate: four, and an id load in front of them) are pending.  (kLate:
    // take_ids below waits for these too, the compiler counting the id load behind loads that it does not see: the second
    // stage is under way during the barrier alone.)
    if (kLate && j + 1 < s1)
      wait_loads<2 * kPgWave + 1>();
    else
      wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    uint32_t bad0 = 0;  // of the block's step or two
    if (row_bad) {
      bad = j < s1 ? bad_of(j) : 0u;
      bad0 = TWO ? bad_of(j0) | bad_of(j0 + 1) : bad;
    }
    if (j0 < s1 && (j0 * kKvStep < blo || (j0 + kStride) * kKvStep > bhi || bad0 != 0)) {
      // V rows that no token of the block sees, and of pages outside the cache, meet p = 0 but may hold NaN/Inf: zeros.
      constexpr int kTpr = PW;  // threads per row
      const int t = (int)threadIdx.x & (PW * 64 - 1), r = t / kTpr, at = j * kKvStep + r;
      if (j < s1 && (at < blo || at >= bhi || ((bad >> (r >> 4)) & 1u))) {
        char *vr = tile(j) + kTileB + r * 256 + 256 / kTpr * (t % kTpr);
#pragma unroll
        for (int i = 0; i < 16 / kTpr; ++i) st128(vr + 16 * i, u32x4{0u, 0u, 0u, 0u});
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    const bool mine = j >= w0 && j < w1;
    constexpr int kNext = kLate ? 2 : kStride;  // the step whose loads go out
    if (j + kNext < s1) {
      take_ids();
      load_ids(j + kNext + kStride);
      if (kLate || !mine) issue_step(j + kNext);
    }
    if (late) {
      if (j - 1 >= w0 && j - 1 < w1) pv_step(tile(j - 1), pcar);
      if (mine) score_step(j, tile(j), pcar);
    } else if (mine) {
      u32x4 pc[2 * kSub];
      score_step(j, tile(j), pc);
      pv_step(tile(j), pc);
    }
  }

  l = halves_sum(l);
  le = halves_sum(le);
  if constexpr (TWO) {  // the second four waves' sums, through the LDS that held the tiles, to the first four's
    f32x4 *const xa = reinterpret_cast<f32x4 *>(&lds[0][0]);   // [wave][16][64 lanes]
    float *const xs = reinterpret_cast<float *>(xa + PW * 16 * 64);  // [wave][3][64 lanes]
    __syncthreads();
    if (side == 1) {
#pragma unroll
      for (int c = 0; c < 16; ++c)
        xa[(wave * 16 + c) * 64 + lane] = f32x4{acc[c >> 2][4 * (c & 3)], acc[c >> 2][4 * (c & 3) + 1],
                                                acc[c >> 2][4 * (c & 3) + 2], acc[c >> 2][4 * (c & 3) + 3]};
      xs[(wave * 3 + 0) * 64 + lane] = m;
      xs[(wave * 3 + 1) * 64 + lane] = l;
      xs[(wave * 3 + 2) * 64 + lane] = le;
    }
    __syncthreads();
    if (side == 1) return;
    const float m1 = xs[(wave * 3 + 0) * 64 + lane], top = fmaxf(m, m1), ref = top == -INFINITY ? 0.f : top;
    const float f0 = fast_exp2(m - ref), f1 = fast_exp2(m1 - ref);
    l = l * f0 + xs[(wave * 3 + 1) * 64 + lane] * f1;
    le = le * f0 + xs[(wave * 3 + 2) * 64 + lane] * f1;
    m = top;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const f32x4 v = xa[(wave * 16 + c) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[c >> 2][4 * (c & 3) + i] = acc[c >> 2][4 * (c & 3) + i] * f0 + v[i] * f1;
    }
  }
  // Rows whose sums are not finite though their scores are: slow_row's.  (Among them rows without a key, l = 0, whose sums are 0 times
  // values that their wave's other rows saw: nothing to add up there, and 0.)
  bool odd = false;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) odd |= !(fabsf(acc[dt][i]) < INFINITY);
  const uint64_t om = __ballot(odd && row_ok && l < INFINITY);
  const uint32_t odd_rows = (uint32_t)om | (uint32_t)(om >> 32);
  const bool sums_ok = ((odd_rows >> n) & 1u) == 0;
  const int64_t pslot = ((int64_t)un.slot * a.hkv + h) * PW + wave;
  if (un.parts > 1 && un.slot >= a.max_cut) return;  // (no call's cut rows are that many)
  uint16_t *const orow = a.o + (q0 + tok0 + tt) * a.o_stride_t + (int64_t)(h * G + g) * a.o_stride_h;
  if (un.parts > 1) {
    if (hl == 0) a.part_ml[pslot * 32 + n] = float2{m, l};
    if (a.lse && hl == 0) a.part_le[pslot * 32 + n] = le;
    if (w0 < w1 && sums_ok) {  // (l = 0 of a wave without steps: the join takes no sums)
#pragma unroll
      for (int c = 0; c < 16; ++c)
        a.part_acc[(pslot * 16 + c) * 64 + lane] = f32x4{acc[c >> 2][4 * (c & 3)], acc[c >> 2][4 * (c & 3) + 1],
                                                         acc[c >> 2][4 * (c & 3) + 2], acc[c >> 2][4 * (c & 3) + 3]};
    }
  } else if (row_ok) {
    // Normalise and write: lane l holds O[row l%32][32 dt + 8 (i / 4) + 4 hl + i % 4].  (l is NaN where a score is.)
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < 16 && sums_ok; ++c) {
      uint2 w;
      w.x = pack2<DT>(acc[c >> 2][4 * (c & 3)] * inv, acc[c >> 2][4 * (c & 3) + 1] * inv);
      w.y = pack2<DT>(acc[c >> 2][4 * (c & 3) + 2] * inv, acc[c >> 2][4 * (c & 3) + 3] * inv);
      *reinterpret_cast<uint2 *>(orow + 4 * hl + 32 * (c >> 2) + 8 * (c & 3)) = w;
    }
    if (a.lse && hl == 0) a.lse[(q0 + tok0 + tt) * a.hq + h * G + g] = l != 0.f ? (m + log2f(le)) * kLn2 : -INFINITY;
  }

  // slow_row: the sums again, key by key, over the row's own keys, beside their own maximum.
  for (uint32_t rows = odd_rows; rows != 0; rows &= rows - 1) {
    const int rn = __builtin_ctz(rows);
    const int rlo = max(__builtin_amdgcn_readlane(lo, rn), s0 * kKvStep), rhi = min(__builtin_amdgcn_readlane(hi, rn), s1 * kKvStep);
    const float rs = readlane(slope2, rn);
    const int rt = rn / G, rg = rn - rt * G, rpos = __builtin_amdgcn_readlane(qpos, rn);
    const uint16_t *qp = a.q + (q0 + tok0 + rt) * a.q_stride_t + (int64_t)(h * G + rg) * a.q_stride_h;
    float rm = -INFINITY, rl = 0.f, o0 = 0.f, o1 = 0.f;  // d = 2 lane, 2 lane + 1
    for (int c0 = rlo; c0 < rhi; c0 += 64) {
      const int k = c0 + lane;
      int pid = k < rhi && k / kPageSize < np ? row_ids[k / kPageSize] : -1;
      if (page_bad(pid)) pid = -1;
      float x[1] = {0.f};
      if (pid >= 0) {
        const uint32_t *kp = reinterpret_cast<const uint32_t *>(kvh + (uint64_t)pid * page_bytes + (k % kPageSize) * row_bytes);
        for (int d = 0; d < 64; ++d) {
          const uint32_t kw = kp[d], qw = reinterpret_cast<const uint32_t *>(qp)[d];
          x[0] = fmaf(E::lo(kw), E::lo(qw), x[0]);
          x[0] = fmaf(E::hi(kw), E::hi(qw), x[0]);
        }
      }
      if (capped)
        cap_scores(x, a.rule, a.sm_scale, kLog2e);
      else
        x[0] *= a.sm_scale * kLog2e;
      if (leaning) x[0] = fmaf(-rs, fabsf((float)(rpos - k)), x[0]);
      const float top = fmaxf(rm, rows4_max(row16_max(pid >= 0 ? x[0] : -INFINITY)));
      if (top > rm) {
        const float al = fast_exp2(rm - top);
        rl *= al;
        o0 *= al;
        o1 *= al;
        rm = top;
      }
      const float p = fast_exp2(x[0] - (rm == -INFINITY ? 0.f : rm));
      for (uint64_t keys = __ballot(pid >= 0); keys != 0; keys &= keys - 1) {
        const int kl = __builtin_ctzll(keys);
        const float pk = readlane(p, kl);
        rl += pk;
        const uint64_t kpid = (uint32_t)__builtin_amdgcn_readlane(pid, kl);
        const uint32_t vw = reinterpret_cast<const uint32_t *>(kvh + kpid * page_bytes +
                                                               (uint32_t)(kPageSize + (c0 + kl) % kPageSize) * row_bytes)[lane];
        o0 = fmaf(pk, E::lo(vw), o0);
        o1 = fmaf(pk, E::hi(vw), o1);
      }
    }
    if (un.parts > 1) {
      // element d of the row: chunk d / 8, lane 32 ((d % 8) / 4) + n, component d % 4
      const int d = 2 * lane;
      float *dst = reinterpret_cast<float *>(a.part_acc + (pslot * 16 + d / 8) * 64 + 32 * (d % 8 / 4) + rn) + d % 4;
      dst[0] = o0;
      dst[1] = o1;
      if (lane == 0) a.part_ml[pslot * 32 + rn] = float2{rm, rl};
      if (a.lse && lane == 0) a.part_le[pslot * 32 + rn] = rl;
    } else {
      const float inv = rl != 0.f ? 1.f / rl : 0.f;
      uint32_t *dst = reinterpret_cast<uint32_t *>(a.o + (q0 + tok0 + rt) * a.o_stride_t + (int64_t)(h * G + rg) * a.o_stride_h);
      dst[lane] = pack2<DT>(o0 * inv, o1 * inv);
    }
  }
}

// Joins the parts of cut rows: the blocks of a tile's parts share its (wave, chunk) pairs, a wave each, whose lanes hold
// the rows as the accumulators did.
template <int DT>
__global__ void __launch_bounds__(kSplitWaves * 64) rule_join_kernel(RulePrefillArgs a) {
  if (*a.any_cut == 0) return;
  constexpr int PW = kSplitWaves;
  const int G = a.G, TW = 32 / G, BT = PW * TW;
  const int lane = threadIdx.x & 63, hl = lane >> 5, n = lane & 31;
  const int u = (int)(blockIdx.z * gridDim.y + blockIdx.y);
  Unit un;
  if (!find_unit(a, BT, u, (int)blockIdx.x, lane, &un) || un.parts == 1) return;
  const int h = un.h;
  const int qn = un.row.q1 - un.row.q0, btok0 = un.tile * BT;
  const int waves = min(PW, (qn - btok0 + TW - 1) / TW);
  const int64_t first = un.slot - un.part;
  for (int task = un.part * PW + uniform((int)(threadIdx.x >> 6)); task < waves * 16; task += un.parts * PW) {
    const int w = task >> 4, c = task & 15;
    const bool want_lse = a.lse && c == 0;
    float M = -INFINITY, L = 0.f, LE = 0.f;
    f32x4 A = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < un.parts; s0 += kJoin) {
      float2 ml[kJoin];
      float le[kJoin];
      f32x4 av[kJoin];
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        const int64_t at = ((first + min(s0 + i, un.parts - 1)) * a.hkv + h) * PW + w;
        ml[i] = a.part_ml[at * 32 + n];
        le[i] = want_lse ? a.part_le[at * 32 + n] : 0.f;
        av[i] = a.part_acc[(at * 16 + c) * 64 + lane];
      }
      float top = M;  // the largest part's m + log2 l: no part's sums weigh more than its values
#pragma unroll
      for (int i = 0; i < kJoin; ++i) top = fmaxf(top, ml[i].y != 0.f ? ml[i].x + __builtin_amdgcn_logf(ml[i].y) : -INFINITY);
      const float ref = top == -INFINITY ? 0.f : top, al = fast_exp2(M - ref);
      L *= al;
      LE *= al;
      A = A * al;
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        if (s0 + i < un.parts && ml[i].y != 0.f) {  // (a part without keys wrote no sums)
          const float sc = fast_exp2(ml[i].x - ref);
          L = fmaf(ml[i].y, sc, L);
          LE = fmaf(le[i], sc, LE);
#pragma unroll
          for (int e = 0; e < 4; ++e) A[e] = fmaf(av[i][e], sc, A[e]);
        }
      }
      M = top;
    }
    const int tt = n / G, g = n - tt * G, tok = btok0 + w * TW + tt;
    if (n < TW * G && tok < qn) {
      const int64_t t = un.row.q0 + tok;
      const float inv = L != 0.f ? 1.f / L : 0.f;
      uint2 o;
      o.x = pack2<DT>(A[0] * inv, A[1] * inv);
      o.y = pack2<DT>(A[2] * inv, A[3] * inv);
      *reinterpret_cast<uint2 *>(a.o + t * a.o_stride_t + (int64_t)(h * G + g) * a.o_stride_h + 4 * hl + 8 * c) = o;
      if (want_lse && hl == 0) a.lse[t * a.hq + h * G + g] = L != 0.f ? (M + log2f(LE)) * kLn2 : -INFINITY;
    }
  }
}

// Tiles of BT tokens that rows of num_tokens tokens in all, max_qo_len each at most, have at most.
int64_t tiles_bound(int64_t num_tokens, int batch, int max_qo_len, int BT) {
  const int64_t slots = (int64_t)batch * ceil_div(max_qo_len, BT);
  const int64_t most = (num_tokens + (int64_t)batch * (BT - 1)) / BT;
  return slots < most ? slots : most;
}

// Calls whose blocks have a CU each, or nearly, and are too many to be cut are bound by the longest one's steps: there a
// block's keys are swept by two sets of four waves, every other step each, whose sums are added at the end (us one set / two;
// prompts of 8 kv heads of 4: 512 tokens, 128 blocks 19.9 / 19.1, 1024 34 / 29, 1536, 384 blocks 48 / 40, 1800, 452 55 / 52; of 8
// of 5: 1200, 400 blocks 41 / 38, 1536, 512 48 / 50; 24 rows of 24 tokens over 4096, 192 blocks 110 / 100).  The two cross
// between 450 and 512 blocks, in groups of 4 and 5; others were not measured.  Fewer blocks are better cut (16 tokens over
// 1600, 8 blocks 20.4 / 22.3), a single step is quicker with one set (9.6 / 11.1).
bool two_sided(int64_t num_tokens, int batch, int hkv, int G, int max_qo_len) {
  const int64_t blocks = tiles_bound(num_tokens, batch, max_qo_len, kSplitWaves * (32 / G)) * hkv;
  return blocks >= kTwoFrom && blocks <= kTwoTo;
}

// Units of cut rows (a kv head's), at most; 0 where no row can be cut, or, in a call of whole prompts, none would gain: there the
// page table has room for the new tokens and the rest of the rows' last pages, and no row is longer than max_qo_len (12 prompts of
// 166 tokens of 8 kv heads of 5 30.6 us with the join's launch, 27.4 without).  Of num_tokens, which may be padded, at
// most max_qo_len a row are new ones: padding alone does not make a call one of whole prompts.
int64_t cut_bound(int64_t num_tokens, int batch, int hkv, int G, int max_qo_len, int64_t kv_indices_len, int window) {
  const int BT = kSplitWaves * (32 / G);
  const bool two = two_sided(num_tokens, batch, hkv, G, max_qo_len);
  const int target = two ? kTargetBlocks / 2 : kTargetBlocks, least = two ? kLoneSteps : kMinSteps;
  const int64_t keys = kv_indices_len * kPageSize, span = window > 0 && window + (int64_t)BT < keys ? window + (int64_t)BT : keys;
  const int64_t steps = ceil_div(span, kKvStep), most = (int64_t)batch * max_qo_len;
  const int64_t room = keys - (num_tokens < most ? num_tokens : most);
  if (room >= 0 && room <= (int64_t)batch * (kPageSize - 1)) {
    const int64_t longest = max_qo_len + room < span ? max_qo_len + room : span;
    if (row_parts((int)ceil_div(longest, kKvStep), least, true) == 1) return 0;
  }
  if (row_parts((int)steps, least, true) == 1) return 0;
  const int64_t tiles = tiles_bound(num_tokens, batch, max_qo_len, BT);
  if (batch == 1 && tiles * hkv >= target) return 0;  // C >= steps
  const int64_t by_work = target / hkv + 1;             // (C hkv parts <= W hkv <= C target)
  const int64_t by_size = tiles * (steps / least);
  return by_work < by_size ? by_work : by_size;
}

// How the kernel treats the scores, and for a cap alone its constants.
int score_mode(RulePrefillArgs &a, int dtype) {
  const double scale = fabs((double)a.sm_scale);
  if (!(scale > 0)) return kAny;
  if (!(a.rule.softcap > 0.f)) return !a.rule.slopes ? kPlain : scale > 1e-10 ? kLeaning : kAny;
  if (a.rule.softcap > kQuickCap) return kAny;
  const double c2 = a.rule.softcap * 1.4426950408889634;
  const float k = (float)(2 * 1.4426950408889634 * scale / a.rule.softcap);
  if (!(k < INFINITY)) return kAny;
  a.cap.k = k;
  a.cap.xs = (float)(2 * c2);
  a.cap.xo = (float)c2;
  if (a.rule.slopes) return kAny;
  // Scores lie within c2 of 0, so with p = 2^(score - ref) in [2^-64, 2^92] (caps up to 54) no maximum is needed: every p is a
  // normal number of fp32 and bf16, and so are its products with values of 2^-40 to 2^20 and their sums (the matrix unit drops
  // smaller products; rows whose sums overflow are slow_row's).  Larger caps take the running maximum.
  const double top = 2 * c2 - 64 > 0 ? 2 * c2 - 64 : 0;
  a.cap.ref = (float)(c2 - top);
  return dtype == DELTA_BF16 && top <= 92 ? kCappedRef : kCapped;
}

size_t part_bytes(int64_t units, int hkv) {
  const size_t per = (size_t)kSplitWaves * 32 * (sizeof(float2) + sizeof(float) + kHeadDim * sizeof(float));
  return (units * hkv * per + sizeof(int) + 255) & ~(size_t)255;
}

template <int DT>
int launch_rule(RulePrefillArgs a, int64_t num_tokens, int max_qo_len, hipStream_t stream, const char *who) {
  const int TW = 32 / a.G;
  // Whole prompts that fill the chip nearly twice over in 4-wave blocks run 8-wave ones (prefill.hip, wide_blocks).
  a.two = two_sided(num_tokens, a.batch, a.hkv, a.G, max_qo_len);
  const bool wide = !a.two && a.max_cut == 0 && a.hkv * ceil_div(max_qo_len, 4 * TW) >= 850;
  const int BT = TW * (wide ? 8 : 4);
  a.row_tiles = (int)ceil_div(max_qo_len, BT);
  const int64_t units = a.max_cut + tiles_bound(num_tokens, a.batch, max_qo_len, BT), y = units < 32768 ? units : 32768;
  const dim3 grid((unsigned)a.hkv, (unsigned)y, (unsigned)ceil_div(units, y));
  auto launch = [&](auto sm) {
    constexpr int SM = decltype(sm)::value;
    if (wide)
      hipLaunchKernelGGL((paged_prefill_rule_kernel<DT, 8, false, SM>), grid, dim3(512), 0, stream, a);
    else if (a.two)
      hipLaunchKernelGGL((paged_prefill_rule_kernel<DT, 4, true, SM>), grid, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL((paged_prefill_rule_kernel<DT, 4, false, SM>), grid, dim3(256), 0, stream, a);
  };
  switch (score_mode(a, DT)) {
    case kPlain: launch(std::integral_constant<int, kPlain>()); break;
    case kCapped: launch(std::integral_constant<int, kCapped>()); break;
    case kCappedRef: if constexpr (DT == DELTA_BF16) launch(std::integral_constant<int, kCappedRef>()); break;
    case kLeaning: launch(std::integral_constant<int, kLeaning>()); break;
    default: launch(std::integral_constant<int, kAny>()); break;
  }
  const int rc = check_launch(who);
  if (rc || a.max_cut == 0) return rc;
  hipLaunchKernelGGL((rule_join_kernel<DT>), dim3((unsigned)a.hkv, (unsigned)a.max_cut), dim3(kSplitWaves * 64), 0, stream, a);
  return check_launch(who);
}

}  // namespace
}  // namespace delta

extern "C" DELTA_EXPORT size_t delta_paged_prefill_rule_workspace_bytes(int64_t num_tokens, int batch, int num_qo_heads,
                                                                        int num_kv_heads, int max_qo_len,
                                                                        int64_t kv_indices_len, int window) {
  using namespace delta;
  if (num_tokens <= 0 || batch <= 0 || max_qo_len <= 0 || num_kv_heads <= 0 || num_qo_heads < num_kv_heads ||
      num_qo_heads % num_kv_heads || num_qo_heads / num_kv_heads > kMaxGroup || kv_indices_len <= 0)
    return 0;
  const int64_t units = cut_bound(num_tokens, batch, num_kv_heads, num_qo_heads / num_kv_heads, max_qo_len, kv_indices_len, window);
  return units > 0 ? part_bytes(units, num_kv_heads) : 0;
}

extern "C" DELTA_EXPORT int delta_paged_prefill_rule(const delta_score_rule_t *rule, const void *q, int64_t q_stride_t,
                                                     int64_t q_stride_h, const void *kv_cache, int64_t num_pages,
                                                     const int32_t *qo_indptr, const int32_t *kv_indptr,
                                                     const int32_t *kv_indices, int64_t kv_indices_len,
                                                     const int32_t *kv_last_page_len, void *o, int64_t o_stride_t,
                                                     int64_t o_stride_h, float *lse, int batch, int64_t num_tokens,
                                                     int max_qo_len, int num_qo_heads, int num_kv_heads, int head_dim,
                                                     int dtype, float sm_scale, void *workspace, size_t workspace_bytes,
                                                     delta_stream_t stream) {
  using namespace delta;
  clear_error();
  const char *who = "delta_paged_prefill_rule";
  if (batch <= 0 || num_tokens <= 0 || max_qo_len <= 0) return DELTA_OK;
  if (head_dim != kHeadDim) return set_error(DELTA_ERR_INVALID, "%s: head_dim must be 128", who);
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads)
    return set_error(DELTA_ERR_INVALID, "%s: num_qo_heads must be a multiple of num_kv_heads", who);
  const int G = num_qo_heads / num_kv_heads;
  if (G > kMaxGroup) return set_error(DELTA_ERR_INVALID, "%s: group size %d > %d unsupported", who, G, kMaxGroup);
  if (dtype != DELTA_BF16 && dtype != DELTA_FP16) return set_error(DELTA_ERR_INVALID, "%s: bad dtype", who);
  RulePrefillArgs a = {};
  const int rc = rule_args(rule, &a.rule, who);
  if (rc) return rc;
  if (!q || !kv_cache || !qo_indptr || !kv_indptr || (!kv_indices && kv_indices_len > 0) || !kv_last_page_len || !o)
    return set_error(DELTA_ERR_INVALID, "%s: null pointer", who);
  if (((uintptr_t)q | (uintptr_t)kv_cache) & 15u || (q_stride_t % 8) || (q_stride_h % 8))
    return set_error(DELTA_ERR_INVALID, "%s: q and kv_cache 16-byte aligned, q strides multiples of 8", who);
  if (((uintptr_t)o & 7u) || (o_stride_t % 4) || (o_stride_h % 4))
    return set_error(DELTA_ERR_INVALID, "%s: o 8-byte aligned with strides in multiples of 4", who);
  if (num_pages <= 0 || kv_indices_len < 0) return set_error(DELTA_ERR_INVALID, "%s: empty cache", who);
  if (num_tokens > 1 << 23 || batch > 1 << 20 || num_kv_heads > 1 << 12 || kv_indices_len > 1 << 26)
    return set_error(DELTA_ERR_INVALID, "%s: more than 2^23 tokens, 2^20 rows, 2^12 kv heads or 2^26 pages", who);
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
  a.o = (uint16_t *)o;
  a.o_stride_t = o_stride_t;
  a.o_stride_h = o_stride_h;
  a.lse = lse;
  a.batch = batch;
  a.hq = num_qo_heads;
  a.hkv = num_kv_heads;
  a.G = G;
  a.token_limit = (int)num_tokens;
  a.sm_scale = sm_scale;
  const int64_t cut = cut_bound(num_tokens, batch, num_kv_heads, G, max_qo_len, kv_indices_len, a.rule.window);
  if (cut > 0) {
    const size_t need = part_bytes(cut, num_kv_heads);
    if (!workspace || workspace_bytes < need)
      return set_error(DELTA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
    if ((uintptr_t)workspace & 255u) return set_error(DELTA_ERR_INVALID, "%s: workspace must be 256-byte aligned", who);
    a.max_cut = (int)cut;
    a.part_acc = (f32x4 *)workspace;
    a.part_ml = (float2 *)(a.part_acc + (size_t)cut * num_kv_heads * kSplitWaves * 16 * 64);
    a.part_le = (float *)(a.part_ml + (size_t)cut * num_kv_heads * kSplitWaves * 32);
    a.any_cut = (int *)(a.part_le + (size_t)cut * num_kv_heads * kSplitWaves * 32);
  }
  if (dtype == DELTA_BF16) return launch_rule<DELTA_BF16>(a, num_tokens, max_qo_len, (hipStream_t)stream, who);
  return launch_rule<DELTA_FP16>(a, num_tokens, max_qo_len, (hipStream_t)stream, who);
}
