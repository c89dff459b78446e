// Page arithmetic of the paged cache, shared by the kernels and plain C++ (the
// CPU tests compile this file alone).
#pragma once
#include <stdint.h>
#if defined(__HIP__) || defined(__HIPCC__)
#define KV_FN __host__ __device__ __forceinline__
#else
#define KV_FN static inline
#endif

// Pages that n positions cover.
KV_FN int kv_cover(int n, int page) { return (n + page - 1) / page; }
// Whether n more positions behind len fit a sequence of max_pages pages; len
// and n as they come from memory.
KV_FN bool kv_fits(int len, int n, int page, int max_pages) {
  return len >= 0 && n >= 0 && (int64_t)len + n <= (int64_t)max_pages * page;
}
// Pages that a cut of a sequence of `cur` positions to `to` leaves of its `held` ones, or -1
// when it cannot be made: `cur` may claim more than the pages hold.
KV_FN int kv_cut(int to, int cur, int held, int page) {
  return to > cur || !kv_fits(to, 0, page, held) ? -1 : kv_cover(to, page);
}
// A table entry as an index that is safe to use; *bad when it is none.
KV_FN int kv_page_ok(int entry, int n_pages, bool *bad) {
  if ((unsigned)entry < (unsigned)n_pages) return entry;
  *bad = true;
  return 0;
}
// Pages a sequence holds, as an index bound: an invalid count holds none.
KV_FN int kv_held_ok(int held, int max_pages, bool *bad) {
  if (held >= 0 && held <= max_pages) return held;
  *bad = true;
  return 0;
}
// Positions that a reader may touch of a sequence that claims `len` cached and
// `extra` behind them: no more than its pages hold.
KV_FN int kv_readable(int len, int extra, int held, int page, int max_pages, bool *bad) {
  const int h = kv_held_ok(held, max_pages, bad);
  if (len < 0) {
    *bad = true;
    return 0;
  }
  const int64_t want = (int64_t)len + extra, most = (int64_t)h * page;
  if (want <= most) return (int)want;
  *bad = true;
  return (int)most;
}
// The part of a claimed length that lies below the `keys` positions of kv_readable, so that
// 0 <= keys - kv_cached <= extra whatever the state claims.
KV_FN int kv_cached(int len, int keys) { return len < 0 ? 0 : len < keys ? len : keys; }
// The element offset of (layer, page, head, row) of the pools.
KV_FN int64_t kv_at(int layer, int pg, int head, int row, int n_pages, int n_kv_head, int page, int head_dim) {
  return ((((int64_t)layer * n_pages + pg) * n_kv_head + head) * page + row) * head_dim;
}
// Lines of the tree attention's keys (one for each row tile of a group) when a group has `tiles` of
// them at most and there are `pieces` workgroups: as many as tiles, or one.  With fewer lines than
// tiles, groups of unequal tiles could add up to what equal ones do.
KV_FN int tree_levels(int64_t tiles, int pieces) { return tiles <= pieces ? (int)tiles : 1; }
