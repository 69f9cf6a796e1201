// What a score rule (delta_score_rule_t) does to the scores x = q.k sm_scale of one query token, for the attention kernels:
//   x <- c tanh(x / c)                      softcap c
//   x <- x - slope_h |pos - key|            slopes, by the distance of the key's position to the query's
//   keys lo <= key < hi only:               lo = max(0, kv_begin, pos - window + 1),
//                                           hi = min(kv_len, kv_end, or without kv_end pos + 1)
#pragma once

#include "delta_common.h"

namespace delta {

struct RuleArgs {
  float softcap, rcp_cap;  // 0: none
  const float *slopes;
  int window;              // 0: none
  const int32_t *kv_begin, *kv_end;
};

// The keys that query token `tok` at position pos of a row of kv_len tokens sees: [*lo, *hi), 0 <= *lo.  hi <= lo: none.
__device__ __forceinline__ void key_range(const RuleArgs &r, int64_t tok, int pos, int kv_len, int *lo, int *hi) {
  int l = 0, h = pos + 1;
  if (r.window > 0 && pos >= r.window) l = pos - r.window + 1;
  if (r.kv_begin) l = max(l, r.kv_begin[tok]);
  if (r.kv_end) h = r.kv_end[tok];
  *lo = l;
  *hi = min(h, kv_len);
}

// tanh(y) / y for |y| <= 0.5, a polynomial in y^2 interpolated at Chebyshev nodes (off by 2^-23 of the value in fp32).
__device__ __forceinline__ float tanh_ratio(float u) {
  float p = fmaf(u, -0.0066158641f, 0.0212762337f);
  p = fmaf(u, p, -0.0538937524f);
  p = fmaf(u, p, 0.1333290488f);
  p = fmaf(u, p, -0.3333332539f);
  return fmaf(u, p, 1.f);
}

// x <- unit c tanh(x in / c) for a wave's N scores a lane (in: the scale that x still lacks; unit: log2 e for scores in
// log2 units, else 1).  c - 2 c / (1 + e^(2 y)) is off by 2^-22 c, whatever the score: it is for scores past c / 2, and the
// polynomial, whose error is relative to the score, for the others, so a cap far above the scores costs them nothing.  Each
// score's form is its own matter, since those beside it may be hidden keys'; where no score of the wave's passes c / 2 the first
// form is left out.
template <int N>
__device__ __forceinline__ void cap_scores(float (&x)[N], const RuleArgs &r, float in, float unit) {
  const float ky = in * r.rcp_cap, kx = in * unit;
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) big = fmaxf(big, fabsf(x[i]));
  if (__ballot(big * fabsf(ky) > 0.5f) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = x[i] * ky;
      x[i] = (x[i] * kx) * tanh_ratio(y * y);
    }
  } else {
    const float k2 = 2.f * kLog2e * ky, c = r.softcap * unit;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // (what both branches compute alike stays in each: moved in front of them it takes a register a score)
      asm volatile("" : "+v"(x[i]));
      const float y = x[i] * ky, near = (x[i] * kx) * tanh_ratio(y * y);
      const float far = fmaf(-2.f * c, __builtin_amdgcn_rcpf(1.f + fast_exp2(x[i] * k2)), c);
      x[i] = fabsf(y) > 0.5f ? far : near;
    }
  }
}

// Checks a caller's rule and sets the kernels' form of it (host).
inline int rule_args(const delta_score_rule_t *rule, RuleArgs *a, const char *who) {
  *a = RuleArgs{};
  if (!rule) return set_error(DELTA_ERR_INVALID, "%s: null score rule", who);
  if (!(rule->softcap >= 0.f) || rule->softcap > 1e30f)
    return set_error(DELTA_ERR_INVALID, "%s: softcap must be 0 (none) or positive and finite", who);
  if (rule->softcap > 0.f && rule->softcap < 1e-30f) return set_error(DELTA_ERR_INVALID, "%s: softcap too small", who);
  if (rule->window < 0) return set_error(DELTA_ERR_INVALID, "%s: window must be 0 (none) or positive", who);
  if (((uintptr_t)rule->slopes | (uintptr_t)rule->kv_begin | (uintptr_t)rule->kv_end) & 3u)
    return set_error(DELTA_ERR_INVALID, "%s: slopes, kv_begin and kv_end must be 4-byte aligned", who);
  a->softcap = rule->softcap;
  a->rcp_cap = rule->softcap > 0.f ? 1.f / rule->softcap : 0.f;
  a->slopes = rule->slopes;
  a->window = rule->window;
  a->kv_begin = rule->kv_begin;
  a->kv_end = rule->kv_end;
  return DELTA_OK;
}

// The most pages that one query token's keys lie in, of rows of at most max_pages pages.
inline int rule_pages(int window, int max_pages) {
  if (window <= 0) return max_pages;
  const int64_t p = ((int64_t)window + 14) / kPageSize + 1;
  return p < max_pages ? (int)p : max_pages;
}

}  // namespace delta
