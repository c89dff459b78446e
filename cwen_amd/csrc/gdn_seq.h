// Packed sequences over a pool's slots, on the device.
#pragma once
#include "cwen_internal.h"
#include "gdn_table.h"

struct GdnSeq {
  int first, n;       // its rows that the call takes
  int src, dst;       // -1: none
  bool ok;
};

__device__ __forceinline__ GdnSeq gdn_seq(const GdnSeqs &a, int s) {
  GdnSeq q;
  q.first = gdn_border(a.cu[s], a.total);
  q.n = gdn_rows(q.first, gdn_border(a.cu[s + 1], a.total));
  q.src = a.src ? a.src[s] : -1;
  q.dst = a.dst ? a.dst[s] : -1;
  q.ok = gdn_slot_ok(q.src, a.n_slots) && gdn_slot_ok(q.dst, a.n_slots);
  if (a.count) {
    const int c = a.count[s];
    q.ok = q.ok && gdn_count_ok(c, q.n);
    q.n = q.ok ? c : 0;
  }
  if (!q.ok) q.src = q.dst = -1;
  return q;
}
// Whether another sequence names the slot that sequence s ends in; all lanes of the wave take part.
__device__ __forceinline__ bool gdn_taken(const GdnSeqs &a, int s, int dst) {
  if (dst < 0 || a.n_seq == 1) return false;
  bool bad = false;
  for (int j = threadIdx.x & 63; j < a.n_seq; j += 64)
    bad |= j != s && gdn_clash(dst, a.src ? a.src[j] : -1, a.dst[j]);
  return __any(bad);
}
__device__ __forceinline__ void gdn_raise(const GdnSeqs &a) {
  if ((threadIdx.x & 63) == 0) __hip_atomic_fetch_or(a.status, CWEN_GDN_ARG, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The sequence of piece z (gdn_piece0) of N rows, or -1; the wave's lanes look at 64 borders at a time.
__device__ __forceinline__ int gdn_find(const GdnSeqs &a, int z, int N) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = a.n_seq;
  do {
    const int step = (hi - lo + 63) >> 6, s = lo + lane * step;
    const int n = __builtin_popcountll(__ballot(s < hi && gdn_piece0(gdn_border(a.cu[min(s, hi - 1)], a.total), s, N) <= z));
    if (n == 0) return -1;
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  } while (hi - lo > 1);
  return __builtin_amdgcn_readfirstlane(lo);
}
