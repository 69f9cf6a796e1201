// Per-head RMS norms of queries and keys, the position rotation in either pair layout, and the KV append, in one pass.
//
//   y = x rsqrt(mean(x^2) + eps) w            per head of 128, q and k with weights of their own (or no norm)
//   (a, b) -> f (a cos t - b sin t, b cos t + a sin t)   for the pairs j < R / 2 of the head's first R elements, which
//             are (2j, 2j + 1) (interleaved) or (j, j + R / 2) (half); the other elements pass
//   t = pos F_j                               F_j in turns per position, a 64-bit fraction: pos F_j mod 2^64 is the
//             angle's turn, exact for every 32-bit position, so that far positions cost no bits (an fp32 angle is off by
//             half a step of pos F_j: 0.004 rad at position 131072, a bf16 step of the result)
// All in fp32, rounded once.  k goes to k_out, or with v into the token's page slot (found as delta_append_kv does).
//
// A 16-lane group holds a head, 8 elements (16 bytes) a lane: the norm is one DPP sum over the group, interleaved pairs
// are in the lane, half pairs R / 16 lanes away (where R / 2 is no multiple of 8, an element's partner is read again).
// A wave finds the token's row by a ballot over the row bounds, its lane j computes pair j's (cos, sin) and the group
// takes the pairs of its elements by lane permutes: no LDS and no barrier, every wave runs on its own.
// What bounds it: memory for prompts (q, k, v read once and written once: 8192 tokens of 32 + 8 heads 46.8 us from and to
// HBM, 4.3 TB/s where a copy reaches 5.1; 44 us in a replayed graph, part of its inputs still in the caches); for a decode
// step the chain row bounds -> position and page -> store (one token 3.6 us, 128 tokens 4.4).  At six waves a SIMD the interleaved
// layout takes 43 us where it took 50, at eight the half layout spills.
#include "delta_common.h"
#include "mfma32.h"

namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 16;  // heads of a block's pass
constexpr int kPre = 4;                 // passes whose loads go out before the row is known

// q, k and v as they come in are read here for the last time: past the caches, which keeps what is written in them for the
// attention behind (with it, 8 rows of 512 tokens 74.3 us, 75.2 with ordinary loads; stores past the caches as well make
// this kernel 10% faster and the two together 3% slower).
__device__ __forceinline__ u32x4 ld_once(const uint16_t *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
}

struct NormRopeArgs {
  const uint16_t *q, *k, *v;  // v NULL: no append
  int64_t q_stride, k_stride, v_stride;
  uint16_t *q_out, *k_out;
  int64_t q_out_stride, k_out_stride;
  const uint16_t *q_weight, *k_weight;  // NULL: no norm
  float eps;
  const uint64_t *turns;
  int pairs;  // R / 2
  float factor;
  const int32_t *indptr, *offsets;
  uint16_t *cache;
  int64_t num_pages;
  const int32_t *kv_indices;
  int64_t kv_indices_len;
  const int32_t *kv_indptr, *last_page_len;
  int batch, hq, hkv;
};

template <int DT, bool INTER>
__global__ void __launch_bounds__(kThreads, 6) norm_rope_kernel(NormRopeArgs a) {
  using E = Elem<DT>;
  const int i = blockIdx.x;
  const int lane = threadIdx.x & 63, t = lane & 15;
  const int nh = a.hq + a.hkv + (a.v ? a.hkv : 0);
  const int first = blockIdx.y * kGroups + (threadIdx.x >> 4), step = gridDim.y * kGroups;
  auto src = [&](int h) {
    return h < a.hq           ? a.q + (int64_t)i * a.q_stride + (int64_t)h * kHeadDim
           : h < a.hq + a.hkv ? a.k + (int64_t)i * a.k_stride + (int64_t)(h - a.hq) * kHeadDim
                              : a.v + (int64_t)i * a.v_stride + (int64_t)(h - a.hq - a.hkv) * kHeadDim;
  };
  u32x4 pre[kPre];
#pragma unroll
  for (int p = 0; p < kPre; ++p)
    if (first + p * step < nh) pre[p] = ld_once(src(first + p * step) + 8 * t);
  const uint64_t turn = lane < a.pairs ? a.turns[lane] : 0;

  // The token's row; a token behind the last row is left alone.
  int row = -1;
  for (int r0 = 0; r0 < a.batch && row < 0; r0 += 64) {
    const int r = r0 + lane;
    const uint64_t m = __ballot(r < a.batch && a.indptr[r < a.batch ? r : 0] <= i && i < a.indptr[r < a.batch ? r + 1 : 0]);
    if (m) row = r0 + __builtin_ctzll(m);
  }
  if (row < 0) return;
  row = uniform(row);
  const int at = i - a.indptr[row];
  const int64_t pos = (int64_t)a.offsets[row] + at;

  // Slot of the append (delta_append_kv's checks; a token without one appends nothing).
  int pid = -1, slot = 0;
  if (a.v) {
    const int64_t p0 = a.kv_indptr[row], p1 = a.kv_indptr[row + 1];
    int lp = a.last_page_len[row];
    lp = lp < 0 ? 0 : (lp > kPageSize ? kPageSize : lp);
    if (p0 >= 0 && p1 >= p0 && p1 <= a.kv_indices_len) {
      const int np = (int)(p1 - p0);
      const int64_t len = np > 0 ? (int64_t)(np - 1) * kPageSize + lp : 0;
      const int64_t apos = len - (a.indptr[row + 1] - a.indptr[row]) + at;
      if (apos >= 0 && apos / kPageSize < np) {
        const int p = a.kv_indices[p0 + apos / kPageSize];
        if (p >= 0 && (int64_t)p < a.num_pages) {
          pid = p;
          slot = (int)(apos % kPageSize);
        }
      }
    }
  }

  // Pair `lane`: the turn's upper 32 bits as a signed fraction, in half turns.
  float cs = 1.f, sn = 0.f;
  if (lane < a.pairs) {
    const int32_t frac = (int32_t)(((uint64_t)pos * turn) >> 32);
    sincospif((float)frac * 0x1p-31f, &sn, &cs);
    cs *= a.factor;
    sn *= a.factor;
  }
  // (cos, +-sin) of this lane's elements; elements past R keep (1, 0).
  const int P = a.pairs;
  float ce[8], se[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = 8 * t + e;
    const int j = INTER ? d >> 1 : (d < P ? d : d - P);
    const bool turned = INTER ? j < P : d < 2 * P;
    const bool minus = INTER ? (d & 1) == 0 : d < P;
    const float c = shfl(cs, turned ? j : 0), s = shfl(sn, turned ? j : 0);
    ce[e] = turned ? c : 1.f;
    se[e] = turned ? (minus ? -s : s) : 0.f;
  }
  const bool shuffled = (P & 7) == 0;
  const int partner = lane + (8 * t < P ? P >> 3 : -(P >> 3));  // (half, lanes of the first R elements)

  auto one = [&](int h, u32x4 raw) {
    const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
    float x[8], y[8], w[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = E::lo(raw[e]);
      x[2 * e + 1] = E::hi(raw[e]);
    }
    const uint16_t *wp = is_q ? a.q_weight : a.k_weight;
    float inv = 1.f;
    if (a.q_weight) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(x[e], x[e], s);
      inv = rsqrtf(row16_sum(s) * (1.f / kHeadDim) + a.eps);
      const u32x4 wr = ld128(wp + 8 * t);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[2 * e] = E::lo(wr[e]);
        w[2 * e + 1] = E::hi(wr[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * w[e];
    }
    if (INTER) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(x[e], ce[e], x[e ^ 1] * se[e]);
    } else if (shuffled) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float o = shfl(x[e], partner);
        y[e] = 8 * t < 2 * P ? fmaf(x[e], ce[e], o * se[e]) : x[e];
      }
    } else {
      const uint16_t *sp = src(h);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 8 * t + e, o = d < P ? d + P : d - P;
        y[e] = x[e];
        if (d < 2 * P) {
          float z = E::lo(sp[o]);
          if (a.q_weight) z = z * inv * E::lo(wp[o]);
          y[e] = fmaf(x[e], ce[e], z * se[e]);
        }
      }
    }
    u32x4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = is_v ? raw[e] : pack2<DT>(y[2 * e], y[2 * e + 1]);
    if (is_q) {
      st128(a.q_out + (int64_t)i * a.q_out_stride + (int64_t)h * kHeadDim + 8 * t, out);
    } else if (!a.v) {
      st128(a.k_out + (int64_t)i * a.k_out_stride + (int64_t)(h - a.hq) * kHeadDim + 8 * t, out);
    } else if (pid >= 0) {
      const int hk = is_v ? h - a.hq - a.hkv : h - a.hq;
      st128(a.cache + ((((int64_t)pid * 2 + is_v) * kPageSize + slot) * a.hkv + hk) * kHeadDim + 8 * t, out);
    }
  };
#pragma unroll
  for (int p = 0; p < kPre; ++p)
    if (first + p * step < nh) one(first + p * step, pre[p]);
  for (int h = first + kPre * step; h < nh; h += step) one(h, ld_once(src(h) + 8 * t));
}

// Blocks over a token's heads: one pass each until the chip's block slots are filled, then one block a token, whose
// passes share its row search and angles.
int launch(NormRopeArgs &a, int nnz, int interleaved, int dtype, hipStream_t stream, const char *who) {
  const int groups = (int)ceil_div(a.hq + a.hkv + (a.v ? a.hkv : 0), kGroups);
  const dim3 grid((unsigned)nnz, (unsigned)((int64_t)nnz * groups <= 1024 ? groups : 1)), block(kThreads);
  if (dtype == DELTA_BF16) {
    if (interleaved)
      hipLaunchKernelGGL((norm_rope_kernel<DELTA_BF16, true>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((norm_rope_kernel<DELTA_BF16, false>), grid, block, 0, stream, a);
  } else {
    if (interleaved)
      hipLaunchKernelGGL((norm_rope_kernel<DELTA_FP16, true>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((norm_rope_kernel<DELTA_FP16, false>), grid, block, 0, stream, a);
  }
  return check_launch(who);
}

// What both entry points check and set.
int common(NormRopeArgs &a, const delta_rotary_t *rotary, const delta_head_norm_t *norm, const void *q, int64_t q_stride,
           const void *k, int64_t k_stride, void *q_out, int64_t q_out_stride, const int32_t *indptr,
           const int32_t *offsets, int nnz, int batch, int hq, int hkv, int head_dim, int dtype, const char *who) {
  if (head_dim != kHeadDim) return set_error(DELTA_ERR_INVALID, "%s: head_dim must be 128", who);
  if (dtype != DELTA_BF16 && dtype != DELTA_FP16) return set_error(DELTA_ERR_INVALID, "%s: bad dtype", who);
  if (hq <= 0 || hkv <= 0 || hq > 1 << 16 || hkv > 1 << 16) return set_error(DELTA_ERR_INVALID, "%s: bad head counts", who);
  if (nnz > 1 << 23) return set_error(DELTA_ERR_INVALID, "%s: more than 2^23 tokens", who);
  if (!q || !k || !q_out || !indptr || !offsets) return set_error(DELTA_ERR_INVALID, "%s: null pointer", who);
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out) & 15u) || (q_stride % 8) || (k_stride % 8) || (q_out_stride % 8))
    return set_error(DELTA_ERR_INVALID, "%s: q, k and outputs 16-byte aligned with strides in multiples of 8", who);
  a = NormRopeArgs{};
  if (rotary && rotary->rotary_dim != 0) {
    if (rotary->rotary_dim < 0 || rotary->rotary_dim > kHeadDim || rotary->rotary_dim % 2)
      return set_error(DELTA_ERR_INVALID, "%s: rotary_dim must be even and at most 128", who);
    if (!rotary->turns || ((uintptr_t)rotary->turns & 7u))
      return set_error(DELTA_ERR_INVALID, "%s: rotary turns null or not 8-byte aligned", who);
    a.turns = rotary->turns;
    a.pairs = rotary->rotary_dim / 2;
    a.factor = rotary->factor;
  }
  if (norm) {
    if (!norm->q_weight || !norm->k_weight || (((uintptr_t)norm->q_weight | (uintptr_t)norm->k_weight) & 15u))
      return set_error(DELTA_ERR_INVALID, "%s: norm weights null or not 16-byte aligned", who);
    if (!(norm->eps >= 0.f)) return set_error(DELTA_ERR_INVALID, "%s: bad eps", who);
    a.q_weight = (const uint16_t *)norm->q_weight;
    a.k_weight = (const uint16_t *)norm->k_weight;
    a.eps = norm->eps;
  }
  a.q = (const uint16_t *)q;
  a.q_stride = q_stride;
  a.k = (const uint16_t *)k;
  a.k_stride = k_stride;
  a.q_out = (uint16_t *)q_out;
  a.q_out_stride = q_out_stride;
  a.indptr = indptr;
  a.offsets = offsets;
  a.batch = batch;
  a.hq = hq;
  a.hkv = hkv;
  return DELTA_OK;
}

}  // namespace
}  // namespace delta

extern "C" DELTA_EXPORT int delta_qk_norm_rope(const delta_rotary_t *rotary, const delta_head_norm_t *norm, const void *q,
                                               int64_t q_stride, const void *k, int64_t k_stride, void *q_out,
                                               int64_t q_out_stride, void *k_out, int64_t k_out_stride,
                                               const int32_t *indptr, const int32_t *offsets, int nnz, int batch,
                                               int num_qo_heads, int num_kv_heads, int head_dim, int dtype,
                                               delta_stream_t stream) {
  using namespace delta;
  clear_error();
  const char *who = "delta_qk_norm_rope";
  if (nnz <= 0 || batch <= 0) return DELTA_OK;
  NormRopeArgs a;
  const int rc = common(a, rotary, norm, q, q_stride, k, k_stride, q_out, q_out_stride, indptr, offsets, nnz, batch,
                        num_qo_heads, num_kv_heads, head_dim, dtype, who);
  if (rc) return rc;
  if (!k_out || ((uintptr_t)k_out & 15u) || (k_out_stride % 8))
    return set_error(DELTA_ERR_INVALID, "%s: k_out null or not 16-byte aligned", who);
  a.k_out = (uint16_t *)k_out;
  a.k_out_stride = k_out_stride;
  return launch(a, nnz, rotary && rotary->interleaved, dtype, (hipStream_t)stream, who);
}

extern "C" DELTA_EXPORT int delta_qk_norm_rope_append(const delta_rotary_t *rotary, const delta_head_norm_t *norm,
                                                      const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                                                      const void *v, int64_t v_stride, void *q_out, int64_t q_out_stride,
                                                      const int32_t *kv_append_indptr, const int32_t *offsets,
                                                      void *kv_cache, int64_t num_pages, const int32_t *kv_indices,
                                                      int64_t kv_indices_len, const int32_t *kv_indptr,
                                                      const int32_t *kv_last_page_len, int nnz, int batch,
                                                      int num_qo_heads, int num_kv_heads, int head_dim, int dtype,
                                                      delta_stream_t stream) {
  using namespace delta;
  clear_error();
  const char *who = "delta_qk_norm_rope_append";
  if (nnz <= 0 || batch <= 0) return DELTA_OK;
  NormRopeArgs a;
  const int rc = common(a, rotary, norm, q, q_stride, k, k_stride, q_out, q_out_stride, kv_append_indptr, offsets, nnz,
                        batch, num_qo_heads, num_kv_heads, head_dim, dtype, who);
  if (rc) return rc;
  if (!v || !kv_cache || (!kv_indices && kv_indices_len > 0) || !kv_indptr || !kv_last_page_len)
    return set_error(DELTA_ERR_INVALID, "%s: null pointer", who);
  if ((((uintptr_t)v | (uintptr_t)kv_cache) & 15u) || (v_stride % 8))
    return set_error(DELTA_ERR_INVALID, "%s: v and kv_cache 16-byte aligned, v stride a multiple of 8", who);
  if (num_pages <= 0 || kv_indices_len < 0) return set_error(DELTA_ERR_INVALID, "%s: empty cache", who);
  a.v = (const uint16_t *)v;
  a.v_stride = v_stride;
  a.cache = (uint16_t *)kv_cache;
  a.num_pages = num_pages;
  a.kv_indices = kv_indices;
  a.kv_indices_len = kv_indices_len;
  a.kv_indptr = kv_indptr;
  a.last_page_len = kv_last_page_len;
  return launch(a, nnz, rotary && rotary->interleaved, dtype, (hipStream_t)stream, who);
}
