// Page copies in every layer's paged cache (gfx950): forked sequences and moved pages.
//
// Entry i copies the first tokens[i] tokens' K and V of page src[i] to page dst[i], in each of the caches.  A page is
// [2, 16, Hkv, 128]: its K and its V are contiguous, and so are their first tokens.  A block copies the K or the V of
// one (entry, cache), up to 16 * Hkv * 256 bytes, 16 bytes per thread and load, all of a thread's loads issued before
// its stores.  Bound by HBM: every byte is read and written once (4000 pages of 64 KiB in each of 4 caches: 2.1 GB in 414 us, 5.1
// TB/s, against 4.85 of a plain copy of 2 GiB; 64 pages in each of 32: 23 us), and by the launch for a single fork (2.9 us).
#include "delta_common.h"

namespace delta {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxCaches = 128;  // per launch: their addresses travel in the launch's arguments

struct CopyArgs {
  char *caches[kMaxCaches];
  const int32_t *src, *dst, *tokens;  // tokens null: whole pages
  int64_t num_pages;
  uint32_t token_bytes;  // of one token's K
};

__global__ void __launch_bounds__(kThreads) copy_pages_kernel(CopyArgs a) {
  const int64_t i = blockIdx.x;
  const int64_t src = a.src[i], dst = a.dst[i];
  int n = a.tokens ? a.tokens[i] : kPageSize;
  n = n < 0 ? 0 : (n > kPageSize ? kPageSize : n);
  if (src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages || src == dst) return;
  const uint32_t half = kPageSize * a.token_bytes;
  char *const cache = a.caches[blockIdx.y >> 1] + (blockIdx.y & 1) * (int64_t)half;
  const char *from = cache + src * 2 * half;
  char *to = cache + dst * 2 * half;
  const uint32_t bytes = n * a.token_bytes;
  constexpr uint32_t kBatch = 8;
  for (uint32_t at = threadIdx.x * 16; at < bytes; at += kThreads * 16 * kBatch) {
    u32x4 v[kBatch];
#pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k)
      if (at + k * kThreads * 16 < bytes) v[k] = ld128(from + at + k * kThreads * 16);
#pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k)
      if (at + k * kThreads * 16 < bytes) st128(to + at + k * kThreads * 16, v[k]);
  }
}

}  // namespace
}  // namespace delta

extern "C" DELTA_EXPORT int delta_copy_pages(void *const *caches, int num_caches, int64_t num_pages, int num_kv_heads,
                                             int head_dim, int dtype, const int32_t *src, const int32_t *dst,
                                             const int32_t *tokens, int64_t num_copies, delta_stream_t stream) {
  using namespace delta;
  const char *who = "delta_copy_pages";
  clear_error();
  if (num_copies <= 0 || num_caches <= 0) return DELTA_OK;
  if (head_dim != kHeadDim) return set_error(DELTA_ERR_INVALID, "%s: head_dim must be 128", who);
  if (dtype != DELTA_BF16 && dtype != DELTA_FP16) return set_error(DELTA_ERR_INVALID, "%s: bad dtype", who);
  if (num_kv_heads <= 0 || num_kv_heads > 4096 || num_pages <= 0)
    return set_error(DELTA_ERR_INVALID, "%s: bad num_kv_heads or num_pages", who);
  if (num_copies > 1 << 23) return set_error(DELTA_ERR_INVALID, "%s: more than 2^23 entries", who);
  if (!caches || !src || !dst) return set_error(DELTA_ERR_INVALID, "%s: null pointer", who);
  for (int c = 0; c < num_caches; ++c)
    if (!caches[c] || ((uintptr_t)caches[c] & 15u))
      return set_error(DELTA_ERR_INVALID, "%s: cache %d null or not 16-byte aligned", who, c);
  CopyArgs a;
  a.src = src;
  a.dst = dst;
  a.tokens = tokens;
  a.num_pages = num_pages;
  a.token_bytes = (uint32_t)num_kv_heads * kHeadDim * 2;
  for (int c0 = 0; c0 < num_caches; c0 += kMaxCaches) {
    const int n = num_caches - c0 < kMaxCaches ? num_caches - c0 : kMaxCaches;
    for (int c = 0; c < n; ++c) a.caches[c] = (char *)caches[c0 + c];
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)num_copies, (unsigned)(2 * n)), dim3(kThreads), 0,
                       (hipStream_t)stream, a);
    const int rc = check_launch(who);
    if (rc) return rc;
  }
  return DELTA_OK;
}
