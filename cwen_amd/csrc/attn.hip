// Attention of packed prompts and of drafted trees over the paged cache.
#include <math.h>
#include <algorithm>
#include "cwen_internal.h"
#include "kv_table.h"
#include "attn_core.h"

namespace {

constexpr float LN2 = 0.69314718055994530942f, LOG2E = 1.44269504088896340736f;

// One row over the keys begin .. end - 1 by a whole wave, key after key: what the
// tiles cannot do, leave a hidden key out whatever it holds.  Lane l holds dims
// E l .. of the query, of each key and of the output, E = D / 64.  m and l as
// AttnWave keeps them; sees: whether the row sees any key.
template <typename T, int D> struct AttnRow {
  static constexpr int E = D / 64;
  float acc[E], m, l;
  bool sees;
  template <typename SEES, typename ROWS>
  __device__ __forceinline__ void run(const typename T::elem *q, int begin, int end, float c, SEES see, ROWS rows) {
    const int lane = threadIdx.x & 63;
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] = (float)q[lane * E + e];
      acc[e] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
    sees = false;
    for (int j = begin; j < end; ++j) {
      if (!see(j)) continue;
      sees = true;
      const typename T::elem *k, *v;
      rows(j, &k, &v);
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(x[e], (float)k[lane * E + e], s);
      s = sum64(s) * c;
      const float mn = fmaxf(m, s), a = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      const float p = __builtin_amdgcn_exp2f(s - (mn == -INFINITY ? 0.f : mn));
      l = fmaf(l, a, p);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], a, p * (float)v[lane * E + e]);
      m = mn;
    }
  }
  __device__ __forceinline__ void store(typename T::elem *o, float *lse) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < E; ++e) o[lane * E + e] = (typename T::elem)(sees ? acc[e] / l : 0.f);
    if (lse && lane == 0) *lse = LN2 * (m + __builtin_amdgcn_logf(l));
  }
};

// ---- packed prompts ----
// Sequence and tile of item `it`: the sequences' tiles of BM queries, counted
// one after the other.  Every wave finds it by itself (64 sequences at a time).
struct Item {
  int seq, tile;      // seq < 0: past the last one
};
__device__ __forceinline__ int span(const int *cu, int s, int total, int *first) {
  const int a = min(max(cu[s], 0), total), b = min(max(cu[s + 1], 0), total);
  *first = a;
  return max(b - a, 0);
}
// The same for a wave's one sequence, in scalar registers.
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int span1(const int *cu, int s, int total, int *first) {
  const int n = scalar(span(cu, s, total, first));
  *first = scalar(*first);
  return n;
}
template <int BM> __device__ __forceinline__ Item find_item(const int *cu, int n_seq, int total, int it) {
  const int lane = threadIdx.x & 63;
  for (int s0 = 0; s0 < n_seq; s0 += 64) {
    int first, v = s0 + lane < n_seq ? (span(cu, s0 + lane, total, &first) + BM - 1) / BM : 0, inc = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int u = __shfl_up(inc, d);
      if (lane >= d) inc += u;
    }
    const unsigned long long past = __ballot(inc > it);
    if (past) {
      const int w = __builtin_ctzll(past);
      return {s0 + w, it - __builtin_amdgcn_readlane(inc - v, w)};
    }
    it -= __builtin_amdgcn_readlane(inc, 63);
  }
  return {-1, 0};
}

// NW waves of 32 QB queries of one head share double-buffered tiles of BN keys.
template <typename T, int D, int NW, int BN, int QB, int OCC> __global__ __launch_bounds__(64 * NW, OCC) void prompt_kernel(PromptArgs a) {
  typedef typename T::elem elem;
  constexpr int WM = 32 * QB, BM = WM * NW;
  __shared__ __align__(1024) elem K0[BN * D], K1[BN * D], V0[BN * D], V1[BN * D];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = a.nh / a.nkv;
  // Blocks of one kv head go to one or two XCDs (block b runs on XCD b % 8), long rows first.
  const int hh = blockIdx.x % a.nh, h = (hh % a.nkv) * g + hh / a.nkv, hkv = hh % a.nkv;
  const int items = gridDim.x / a.nh;
  const Item item = find_item<BM>(a.cu_q, a.n_seq, a.total_q, items - 1 - (int)(blockIdx.x / a.nh));
  if (item.seq < 0) return;
  int q0, k0;
  const int nq = span1(a.cu_q, item.seq, a.total_q, &q0), nk = span1(a.cu_k, item.seq, a.total_k, &k0), off = nk - nq;
  const int first = item.tile * BM, w0 = first + wave * WM;      // the workgroup's and this wave's first query
  AttnWave<T, D, BN, QB> w;
  int limit[QB];                                                 // the last key of this lane's queries
#pragma unroll
  for (int y = 0; y < QB; ++y) {
    const int row = w0 + 32 * y + n;
    limit[y] = row < nq ? row + off : -1;
    w.start(y, row < nq ? (const elem *)a.q + (long long)(q0 + row) * a.qs + h * D : nullptr);
  }
  const elem *kp = (const elem *)a.k + (long long)k0 * a.ks + hkv * D, *vp = (const elem *)a.v + (long long)k0 * a.vs + hkv * D;
  const int kend = min(min(first + BM, nq) + off, nk);           // keys that the workgroup's rows see
  const int wend = min(min(w0 + WM, nq) + off, nk);              // and this wave's
  const float c = a.scale * LOG2E;
  auto land = [&](elem *Kd, elem *Vd, int t0) __attribute__((always_inline)) {
    land_rows<D, BN, false, NW>(Kd, wave, t0, nk - 1, (uint32_t)a.ks * 2, [&](int, int j) { return kp + j * a.ks; });
    land_rows<D, BN, true, NW>(Vd, wave, t0, nk - 1, (uint32_t)a.vs * 2, [&](int, int j) { return vp + j * a.vs; });
  };
  auto ready = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    asm volatile("" ::: "memory");
  };
  // Tiles that every row sees whole come first, two per turn; what is left has
  // its keys compared with each row's last.
  const int full = max(min(first + off + 1, nk), 0) / (2 * BN) * (2 * BN);
  if (kend > 0) land(K0, V0, 0);
  int t0 = 0;
  for (; t0 < full; t0 += 2 * BN) {
    ready();
    land(K1, V1, t0 + BN);
    w.template tile<false>(K0, V0, c, [](int, int) { return false; });
    ready();
    if (t0 + 2 * BN < kend) land(K0, V0, t0 + 2 * BN);
    w.template tile<false>(K1, V1, c, [](int, int) { return false; });
  }
  for (; t0 < kend; t0 += 2 * BN) {
    ready();
    if (t0 + BN < kend) land(K1, V1, t0 + BN);
    if (t0 < wend) w.template tile<true>(K0, V0, c, [&](int y, int j) { return t0 + j > limit[y]; });
    if (t0 + BN >= kend) break;
    ready();
    if (t0 + 2 * BN < kend) land(K0, V0, t0 + 2 * BN);
    if (t0 + BN < wend) w.template tile<true>(K1, V1, c, [&](int y, int j) { return t0 + BN + j > limit[y]; });
  }
  if (__any(w.odd != w.odd)) {   // a hidden value may have leaked: these rows one by one
    for (int i = 0; i < WM && w0 + i < nq; ++i) {
      const long long t = q0 + w0 + i;
      AttnRow<T, D> x;
      x.run((const elem *)a.q + t * a.qs + h * D, 0, min(nk, w0 + i + off + 1), c, [](int) { return true; },
            [&](int j, const elem **k, const elem **v) {
              *k = kp + j * a.ks;
              *v = vp + j * a.vs;
            });
      x.store((elem *)a.o + t * a.os + h * D, a.lse ? a.lse + t * a.nh + h : nullptr);
    }
    return;
  }
#pragma unroll
  for (int y = 0; y < QB; ++y) {
    const int row = w0 + 32 * y + n;
    const float l = w.sum(y), inv = limit[y] < 0 ? 0.f : 1.f / l;
    if (row >= nq) continue;
    elem *orow = (elem *)a.o + (long long)(q0 + row) * a.os + h * D;
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typename AttnOps<T>::vec4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (elem)(limit[y] < 0 ? 0.f : w.o[y][b][4 * i + j] * inv);
        *(typename AttnOps<T>::vec4 *)(orow + 32 * b + 8 * i + 4 * (lane >> 5)) = v;
      }
    if (a.lse && lane < 32) a.lse[(long long)(q0 + row) * a.nh + h] = LN2 * (w.m[y] + __builtin_amdgcn_logf(l));
  }
}

// ---- trees over the paged cache ----
// Row r of group s and a kv head is head r % g of node r / g: the query heads
// that share the kv head's keys lie side by side, so a group's n nodes are n g
// rows against one stream of pages.  Few rows leave the work bound by that
// stream, many by the matrix cores, and both want it cut along the keys, since
// groups are few: row tiles of RT rows are cut into chunks of whole tiles of
// keys, as many that about `target` items per kv head arise over all groups
// (so that a long sequence among short ones does not set the time).  Nothing of
// this is known on the host: every workgroup finds its item from the lengths on the
// device, 64 groups at a time.
struct TreeSeq {
  int c0, nodes, len, keys, id;     // first node, nodes, cached positions, keys in all, sequence (0 when invalid)
  bool bad;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs &a, int s) {
  TreeSeq q;
  q.nodes = min(span(a.cu, s, a.total, &q.c0), a.max_nodes);
  q.id = a.seqs[s];
  q.bad = (unsigned)q.id >= (unsigned)a.kv.max_seqs;
  if (q.bad) {
    q.id = q.len = q.keys = 0;
  } else {
    q.len = a.kv.len[q.id];
    q.keys = kv_readable(q.len, q.nodes, a.kv.held[q.id], a.kv.page, a.kv.max_pages, &q.bad);
  }
  return q;
}
__device__ __forceinline__ TreeSeq tree_seq1(const TreeArgs &a, int s) {     // in scalar registers
  const TreeSeq q = tree_seq(a, s);
  return {scalar(q.c0), scalar(q.nodes), scalar(q.len), scalar(q.keys), scalar(q.id), scalar(q.bad) != 0};
}
struct TreeItem {
  int s, tile, split, nsplit;   // group (< 0: none), row tile, key chunk and their number
  int slot;                     // the row tile's first partial
  int chunk;                    // keys of a chunk
};
// The item `it`, or with `node` the group whose nodes hold token `it` (tile and split 0).
__device__ __forceinline__ TreeItem tree_find(const TreeArgs &a, int it, bool node, int rt, int unit, int target) {
  const int lane = threadIdx.x & 63, g = a.nh / a.kv.n_kv_head;
  auto at = [&](int s, int *tiles, int *units, TreeSeq *q) {
    *tiles = *units = 0;
    if (s >= a.n_seq) return;
    *q = tree_seq(a, s);
    *tiles = (q->nodes * g + rt - 1) / rt;
    *units = (q->keys + unit - 1) / unit;
  };
  auto scan = [&](int v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int u = __shfl_up(v, d);
      if (lane >= d) v += u;
    }
    return v;
  };
  TreeSeq q = {};
  int tiles, units;
  long long work = 0;
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    at(s0 + lane, &tiles, &units, &q);
    long long v = (long long)tiles * units;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    work += v;
  }
  // units of a chunk; target 0: every row tile one chunk
  const int per = (int)min(target ? max((work + target - 1) / target, 1ll) : 1ll << 30, (1ll << 30) / unit);
  int slot = 0;
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    if (a.n_seq > 64) at(s0 + lane, &tiles, &units, &q);     // with up to 64 groups the values are still there
    const int ns = max((units + per - 1) / per, 1), items = tiles * ns, parts = ns > 1 ? items : 0;
    const int inc = scan(items), pinc = scan(parts);
    const bool mine = node ? s0 + lane < a.n_seq && it >= q.c0 && it < q.c0 + q.nodes : inc > it;
    const unsigned long long hit = __ballot(mine);
    if (hit) {
      const int w = __builtin_ctzll(hit);
      const int nsplit = __builtin_amdgcn_readlane(ns, w), r = node ? 0 : it - __builtin_amdgcn_readlane(inc - items, w);
      const int tile = r / nsplit;
      return {s0 + w, tile, r - tile * nsplit, nsplit, slot + __builtin_amdgcn_readlane(pinc - parts, w) + tile * nsplit, per * unit};
    }
    if (!node) it -= __builtin_amdgcn_readlane(inc, 63);
    slot += __builtin_amdgcn_readlane(pinc, 63);
  }
  return {-1, 0, 0, 1, 0, 0};
}
__device__ __forceinline__ TreeItem tree_item(const TreeArgs &a, int it, int rt, int unit, int target) {   // in scalar registers
  const TreeItem x = tree_find(a, it, false, rt, unit, target);
  return {scalar(x.s), scalar(x.tile), scalar(x.split), scalar(x.nsplit), scalar(x.slot), scalar(x.chunk)};
}
// Bit j: whether node i's row sees key u0 + j of the drafted ones (u0 < 0: a
// cached position, seen), j < 32; n nodes.
__device__ __forceinline__ uint32_t tree_sees(const unsigned long long *row, int mw, int i, int n, int u0) {
  if (u0 <= -32) return ~0u;
  const int u = max(u0, 0), before = u - u0;      // before: cached positions of the 32
  unsigned long long w;
  if (u >= n) {
    w = 0;
  } else if (!row) {
    w = i < u ? 0 : i - u >= 63 ? ~0ull : (2ull << (i - u)) - 1;
  } else {
    const int k = u >> 6, b = u & 63;
    w = row[k] >> b;
    if (b && k + 1 < mw) w |= row[k + 1] << (64 - b);
  }
  if (n - u < 64 && n > u) w &= (1ull << (n - u)) - 1;
  return (uint32_t)(w << before) | (uint32_t)((1ull << before) - 1);
}

struct TreeLaunch {
  int target;                   // items per kv head
  float *po;                    // partial outputs [kv head][slot][row][D]
  float2 *ml;                   // and their maxima and sums [kv head][slot][row]
  int slots;
};

// One group's rows against the pages: what both forms share.
template <typename T, int D> struct TreeRows {
  typedef typename T::elem elem;
  const TreeArgs &a;
  const TreeSeq &q;
  int hkv, g, shift;                // shift: log2 of the page size
  // The sequence's pages, as constant memory: no kernel that reads them writes
  // them, and with a uniform index the entry is a scalar load.
  const __attribute__((address_space(4))) int *tab;
  __device__ __forceinline__ TreeRows(const TreeArgs &a, const TreeSeq &q, int hkv)
      : a(a), q(q), hkv(hkv), g(a.nh / a.kv.n_kv_head), shift(__builtin_ctz(a.kv.page)),
        tab((const __attribute__((address_space(4))) int *)(a.kv.table + (size_t)q.id * a.kv.max_pages)) {}
  // The page that holds key j (past the last: the last).
  __device__ __forceinline__ int page(int j) const { return tab[min(j, q.keys - 1) >> shift]; }
  // Key j of that page.
  __device__ __forceinline__ const elem *row(const void *pool, int page, int j, bool *bad) const {
    const int pg = kv_page_ok(page, a.kv.n_pages, bad);
    return (const elem *)pool + kv_at(a.layer, pg, hkv, j & (a.kv.page - 1), a.kv.n_pages, a.kv.n_kv_head, a.kv.page, D);
  }
  __device__ __forceinline__ const elem *query(int r) const {
    return (const elem *)a.q + (long long)(q.c0 + r / g) * a.qs + (hkv * g + r % g) * D;
  }
  __device__ __forceinline__ elem *out(int r) const {
    return (elem *)a.o + (long long)(q.c0 + r / g) * a.os + (hkv * g + r % g) * D;
  }
  __device__ __forceinline__ float *lse(int r) const {
    return a.lse ? a.lse + (long long)(q.c0 + r / g) * a.nh + hkv * g + r % g : nullptr;
  }
  __device__ __forceinline__ const unsigned long long *mask(int r) const {
    return a.mask ? a.mask + (long long)(q.c0 + r / g) * a.mw : nullptr;
  }
  // Row r alone over the keys begin .. end - 1; po, ml: its partial, or null.
  __device__ __forceinline__ void plain(int r, int begin, int end, float *po, float2 *ml) const {
    const unsigned long long *mk = mask(r);
    const int i = r / g, lane = threadIdx.x & 63;
    AttnRow<T, D> x;
    x.run(query(r), begin, end, a.scale * LOG2E,
          [&](int j) {
            const int u = j - q.len;
            return u < 0 || (mk ? (mk[u >> 6] >> (u & 63)) & 1 : u <= i);
          },
          [&](int j, const elem **k, const elem **v) {
            bool bad = false;
            *k = row(a.kv.k, page(j), j, &bad);
            *v = row(a.kv.v, page(j), j, &bad);
          });
    if (!po) {
      x.store(out(r), lse(r));
      return;
    }
#pragma unroll
    for (int e = 0; e < D / 64; ++e) po[lane * (D / 64) + e] = x.acc[e];
    if (lane == 0) *ml = make_float2(x.m, x.sees && x.l == 0.f ? NAN : x.l);
  }
};

// Few rows: one tile of 32, the chunk's keys dealt to 4 waves 32 at a time.  A wave
// has its own K and V rows in LDS and no barrier in its loop: the next K rows
// are requested when the scores are done, the next V rows after the outputs, so
// that half of its LDS and more is always under way.  The waves' sums meet at the
// end.
template <typename T, int D> __global__ __launch_bounds__(256, 1) void tree_few_kernel(TreeArgs a, TreeLaunch p) {
  typedef typename T::elem elem;
  constexpr int BN = 32, NW = 4, UNIT = BN * NW, PC = D / 4;      // PC: 16-byte pieces of an f32 row
  __shared__ __align__(1024) elem Ks[NW * BN * D], Vs[NW * BN * D];
  __shared__ float2 s_ml[NW][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nkv = a.kv.n_kv_head, hkv = blockIdx.x % nkv, n = lane & 31, hi = lane >> 5;
  const TreeItem item = tree_item(a, blockIdx.x / nkv, 32, UNIT, p.target);
  if (item.s < 0) return;
  const TreeSeq q = tree_seq1(a, item.s);
  if (q.bad && tid == 0) kv_raise(a.kv, CWEN_KV_PAGE);
  const TreeRows<T, D> rows(a, q, hkv);
  const int base = item.tile * 32, R = min(q.nodes * rows.g - base, 32), r = base + n;
  const bool live = n < R;
  const int begin = item.split * item.chunk, end = min(begin + item.chunk, q.keys);
  elem *Kw = Ks + wave * BN * D, *Vw = Vs + wave * BN * D;
  bool bad = false;
  int t0 = begin + wave * BN;
  AttnWave<T, D, BN, 1> w;
  // 16 rows never straddle a page: two lookups a tile, for the tile after the current one.
  int pg[2];
  auto land = [&](elem *dst, const void *pool, auto isv) __attribute__((always_inline)) {
    constexpr int half = 16 / (64 / (D / 8));       // loads of 16 rows
    land_rows<D, BN, decltype(isv)::value, 1>(dst, 0, t0, q.keys - 1, D * 2,
                                              [&](int i, int j) { return rows.row(pool, pg[i / half], j, &bad); });
  };
  auto pages = [&]() __attribute__((always_inline)) {
    pg[0] = rows.page(t0);
    pg[1] = rows.page(t0 + 16);
  };
  if (t0 < end) {
    pages();
    land(Kw, a.kv.k, std::false_type{});
    land(Vw, a.kv.v, std::true_type{});
  }
  w.start(0, live ? rows.query(r) : nullptr);
  const float c = a.scale * LOG2E;
  const unsigned long long *mask = live ? rows.mask(r) : nullptr;
  const int node = r / rows.g;
  bool saw = false;
  while (t0 < end) {
    const int u0 = t0 - q.len;
    t0 += UNIT;
    if (t0 < end) pages();
    f32x16_t s[1][1];
    typename AttnWave<T, D, BN, 1>::vec8 pr[1][2];
    w.scores(Kw, s);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // its rows are read
    if (t0 < end) land(Kw, a.kv.k, std::false_type{});
    if (u0 + BN > 0) {
      const uint32_t see = tree_sees(mask, a.mw, node, q.keys - q.len, u0);
      saw |= see != 0;
      w.template soft<true>(s, c, [&](int, int j) { return !((see >> j) & 1); }, pr);
      w.template outputs<true>(Vw, pr);
    } else {
      saw = true;
      w.template soft<false>(s, c, [](int, int) { return false; }, pr);
      w.template outputs<false>(Vw, pr);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t0 < end) land(Vw, a.kv.v, std::true_type{});
  }
  if (bad) kv_raise(a.kv, CWEN_KV_PAGE);
  const float l = w.sum(0);
  if (lane < 32) s_ml[wave][n] = make_float2(w.m[0], saw && l == 0.f ? NAN : l);
  const bool whole = item.nsplit == 1;
  const size_t slot = ((size_t)hkv * p.slots + item.slot + item.split) * 32;
  if (__syncthreads_or(w.odd != w.odd)) {        // a hidden value may have leaked: the rows one by one
    for (int x = wave; x < R; x += NW)
      rows.plain(base + x, begin, end, whole ? nullptr : p.po + (slot + x) * D, whole ? nullptr : p.ml + slot + x);
    return;
  }
  // Each wave's outputs against the row's common maximum, through LDS (rows of D
  // floats, their pieces permuted by the row), then summed in the waves' order.
  float M = -INFINITY;
#pragma unroll
  for (int x = 0; x < NW; ++x) M = fmaxf(M, s_ml[x][n].x);
  const float f = w.m[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m[0] - M);
  auto area = [&](int x) { return (float *)(x < 2 ? Ks : Vs) + (x & 1) * 32 * D; };
  float *mine = area(wave);
#pragma unroll
  for (int b = 0; b < D / 32; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(float4 *)(mine + n * D + 4 * ((8 * b + 2 * i + hi) ^ (n & 15))) =
          make_float4(w.o[0][b][4 * i] * f, w.o[0][b][4 * i + 1] * f, w.o[0][b][4 * i + 2] * f, w.o[0][b][4 * i + 3] * f);
  __syncthreads();
  for (int x = tid; x < R * PC; x += 256) {
    const int y = x / PC, pc = x - y * PC;
    float Mr = -INFINITY, L = 0.f;
#pragma unroll
    for (int u = 0; u < NW; ++u) Mr = fmaxf(Mr, s_ml[u][y].x);
#pragma unroll
    for (int u = 0; u < NW; ++u) L += s_ml[u][y].x == -INFINITY ? s_ml[u][y].y : s_ml[u][y].y * __builtin_amdgcn_exp2f(s_ml[u][y].x - Mr);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float4 v = *(const float4 *)(area(u) + y * D + 4 * (pc ^ (y & 15)));
      o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
    }
    if (whole) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const typename AttnOps<T>::vec4 e = {(elem)(o.x * inv), (elem)(o.y * inv), (elem)(o.z * inv), (elem)(o.w * inv)};
      *(typename AttnOps<T>::vec4 *)(rows.out(base + y) + 4 * pc) = e;
      if (pc == 0 && a.lse) *rows.lse(base + y) = LN2 * (Mr + __builtin_amdgcn_logf(L));
    } else {
      *(float4 *)(p.po + (slot + y) * D + 4 * pc) = o;
      if (pc == 0) p.ml[slot + y] = make_float2(Mr, L);
    }
  }
}

// Many rows: NW waves of 32 QB rows share double-buffered tiles of BN keys.
template <typename T, int D, int NW, int BN, int QB, int OCC>
__global__ __launch_bounds__(64 * NW, OCC) void tree_many_kernel(TreeArgs a, TreeLaunch p) {
  typedef typename T::elem elem;
  constexpr int WM = 32 * QB, RT = WM * NW, PER = BN * D / 8 / (64 * NW);
  __shared__ __align__(1024) elem K0[BN * D], K1[BN * D], V0[BN * D], V1[BN * D];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nkv = a.kv.n_kv_head, hkv = blockIdx.x % nkv, n = lane & 31, hi = lane >> 5;
  const TreeItem item = tree_item(a, blockIdx.x / nkv, RT, BN, p.target);
  if (item.s < 0) return;
  const TreeSeq q = tree_seq1(a, item.s);
  if (q.bad && tid == 0) kv_raise(a.kv, CWEN_KV_PAGE);
  const TreeRows<T, D> rows(a, q, hkv);
  const int base = item.tile * RT + wave * WM, R = min(q.nodes * rows.g - base, WM);   // R <= 0: no rows here
  const int begin = item.split * item.chunk, end = min(begin + item.chunk, q.keys);
  bool bad = false;
  const float c = a.scale * LOG2E;
  // The page of each piece that this wave lands (its rows lie in one page), a tile ahead.
  int pg[PER];
  auto pages = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) pg[i] = rows.page(t0 + (i * NW + wave) * 64 / (D / 8));
  };
  auto land = [&](elem *Kd, elem *Vd, int t0) __attribute__((always_inline)) {
    land_rows<D, BN, false, NW>(Kd, wave, t0, q.keys - 1, D * 2, [&](int i, int j) { return rows.row(a.kv.k, pg[i], j, &bad); });
    land_rows<D, BN, true, NW>(Vd, wave, t0, q.keys - 1, D * 2, [&](int i, int j) { return rows.row(a.kv.v, pg[i], j, &bad); });
    if (t0 + BN < end) pages(t0 + BN);
    __builtin_amdgcn_sched_barrier(0);              // the addresses' registers are free again before the tile
  };
  auto ready = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    asm volatile("" ::: "memory");
  };
  if (begin < end) {
    pages(begin);
    land(K0, V0, begin);
  }
  int t0 = begin;
  if (R <= 0) {                                     // a wave without rows lands its share and does no more
    for (bool one = true; t0 < end; t0 += BN, one = !one) {
      ready();
      if (t0 + BN < end) land(one ? K1 : K0, one ? V1 : V0, t0 + BN);
    }
    if (bad) kv_raise(a.kv, CWEN_KV_PAGE);
    return;
  }
  AttnWave<T, D, BN, QB> w;
#pragma unroll
  for (int y = 0; y < QB; ++y) w.start(y, 32 * y + n < R ? rows.query(base + 32 * y + n) : nullptr);
  const int full = begin + max(min(end, q.len) - begin, 0) / (2 * BN) * (2 * BN);   // whole tiles of cached positions
  uint32_t saw[QB];
#pragma unroll
  for (int y = 0; y < QB; ++y) saw[y] = full > begin;
  auto part = [&](const elem *Kb, const elem *Vb, int t0) __attribute__((always_inline)) {
    uint32_t see[QB][BN / 32];
#pragma unroll
    for (int y = 0; y < QB; ++y) {
      const int r = base + 32 * y + n;
      const unsigned long long *mask = 32 * y + n < R ? rows.mask(r) : nullptr;
#pragma unroll
      for (int b = 0; b < BN / 32; ++b)
        saw[y] |= see[y][b] = tree_sees(mask, a.mw, r / rows.g, q.keys - q.len, t0 + 32 * b - q.len);
    }
    w.template tile<true>(Kb, Vb, c, [&](int y, int j) { return !((see[y][j >> 5] >> (j & 31)) & 1); });
  };
  for (; t0 < full; t0 += 2 * BN) {
    ready();
    land(K1, V1, t0 + BN);
    w.template tile<false>(K0, V0, c, [](int, int) { return false; });
    ready();
    if (t0 + 2 * BN < end) land(K0, V0, t0 + 2 * BN);
    w.template tile<false>(K1, V1, c, [](int, int) { return false; });
  }
  for (; t0 < end; t0 += 2 * BN) {
    ready();
    if (t0 + BN < end) land(K1, V1, t0 + BN);
    part(K0, V0, t0);
    if (t0 + BN >= end) break;
    ready();
    if (t0 + 2 * BN < end) land(K0, V0, t0 + 2 * BN);
    part(K1, V1, t0 + BN);
  }
  if (bad) kv_raise(a.kv, CWEN_KV_PAGE);
  const bool whole = item.nsplit == 1;
  const size_t slot = ((size_t)hkv * p.slots + item.slot + item.split) * RT + wave * WM;
  if (__any(w.odd != w.odd)) {
    for (int x = 0; x < R; ++x)
      rows.plain(base + x, begin, end, whole ? nullptr : p.po + (slot + x) * D, whole ? nullptr : p.ml + slot + x);
    return;
  }
#pragma unroll
  for (int y = 0; y < QB; ++y) {
    const int x = 32 * y + n;
    const float l = w.sum(y), ls = saw[y] && l == 0.f ? NAN : l, inv = whole ? (ls == 0.f ? 0.f : 1.f / ls) : 1.f;
    if (x >= R) continue;
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = make_float4(w.o[y][b][4 * i] * inv, w.o[y][b][4 * i + 1] * inv, w.o[y][b][4 * i + 2] * inv,
                                     w.o[y][b][4 * i + 3] * inv);
        const int d = 32 * b + 8 * i + 4 * hi;
        if (whole) {
          const typename AttnOps<T>::vec4 e = {(elem)v.x, (elem)v.y, (elem)v.z, (elem)v.w};
          *(typename AttnOps<T>::vec4 *)(rows.out(base + x) + d) = e;
        } else {
          *(float4 *)(p.po + (slot + x) * D + d) = v;
        }
      }
    if (lane < 32) {
      if (!whole) p.ml[slot + x] = make_float2(w.m[y], ls);
      else if (a.lse) *rows.lse(base + x) = LN2 * (w.m[y] + __builtin_amdgcn_logf(l));
    }
  }
}

// The chunks of a row joined: one workgroup per (node, head), each of its waves a
// contiguous quarter of the chunks in order, the quarters then added in order.
template <typename T, int D> __global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, TreeLaunch p, int rt, int unit) {
  typedef typename T::elem elem;
  constexpr int E = D / 64;
  __shared__ float s_o[4][D], s_m[4], s_l[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x % a.nh, g = a.nh / a.kv.n_kv_head, hkv = h / g;
  const int t = blockIdx.x / a.nh;
  const TreeItem item = tree_find(a, t, true, rt, unit, p.target);
  if (item.s < 0 || item.nsplit == 1) return;
  int c0;
  span(a.cu, item.s, a.total, &c0);
  const int r = (t - c0) * g + h % g, tile = r / rt;
  const size_t first = ((size_t)hkv * p.slots + item.slot + tile * item.nsplit) * rt + r % rt;    // chunk x: first + x * rt
  float M = -INFINITY;
  for (int x = lane; x < item.nsplit; x += 64) M = fmaxf(M, p.ml[first + (size_t)x * rt].x);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) M = fmaxf(M, __shfl_xor(M, d));
  const int per = (item.nsplit + 3) / 4, x0 = wave * per, x1 = min(x0 + per, item.nsplit);
  float L = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int x = x0; x < x1; ++x) {
    const size_t at = first + (size_t)x * rt;
    const float2 ml = p.ml[at];
    const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : ml.y) : __builtin_amdgcn_exp2f(ml.x - M);   // NaN stays
    L += ml.x == -INFINITY ? f : ml.y * f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(p.po[at * D + lane * E + e], f, o[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[wave][lane * E + e] = o[e];
  if (lane == 0) s_l[wave] = L;
  __syncthreads();
  (void)s_m;
  L = s_l[0] + s_l[1] + s_l[2] + s_l[3];
  const float inv = L == 0.f ? 0.f : 1.f / L;
  for (int d = tid; d < D; d += 256)
    ((elem *)a.o)[(long long)t * a.os + h * D + d] = (elem)((s_o[0][d] + s_o[1][d] + s_o[2][d] + s_o[3][d]) * inv);
  if (a.lse && tid == 0) a.lse[(long long)t * a.nh + h] = LN2 * (M + __builtin_amdgcn_logf(L));
}

template <typename F> int by_type(int type, int D, F f) {
  if (type == CWEN_T_F16) {
    if (D == 64) f(TypeF16{}, std::integral_constant<int, 64>{});
    else if (D == 128) f(TypeF16{}, std::integral_constant<int, 128>{});
    else f(TypeF16{}, std::integral_constant<int, 256>{});
  } else {
    if (D == 64) f(TypeBF16{}, std::integral_constant<int, 64>{});
    else if (D == 128) f(TypeBF16{}, std::integral_constant<int, 128>{});
    else f(TypeBF16{}, std::integral_constant<int, 256>{});
  }
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}

}  // namespace

int attn_prompt_launch(const cwen_ctx *, int type, int D, const PromptArgs &a, hipStream_t st) {
  const int BM = D == 256 ? 128 : 256;
  const long long items = (a.total_q + BM - 1) / BM + a.n_seq;
  if (items * a.nh > INT32_MAX) return CWEN_EINVAL;
  return by_type(type, D, [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int dim = decltype(d)::value;
    const dim3 grid((unsigned)(items * a.nh));
    if constexpr (dim == 256) hipLaunchKernelGGL((prompt_kernel<T, dim, 4, 32, 1, 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((prompt_kernel<T, dim, 8, 64, 1, 2>), grid, dim3(512), 0, st, a);
  });
}
int attn_tree_launch(const cwen_ctx *ctx, const TreeArgs &a, hipStream_t st) {
  const int nkv = a.kv.n_kv_head, g = a.nh / nkv, D = a.kv.head_dim;
  const long long rows = (long long)a.max_nodes * g;
  const int form = rows <= 32 ? 1 : 4;                           // row tiles of 32 of a workgroup
  const int rt = 32 * form, unit = form == 1 ? 128 : D == 256 ? 32 : 64;
  const long long tiles = (rows + rt - 1) / rt;                  // of one group at most
  const long long room = (long long)ctx->attn_floats / ((D + 2ll) * rt * nkv);   // slots that the scratch holds
  TreeLaunch p;
  long long want = std::max(1ll, 2ll * ctx->ncu / nkv);
  p.target = (int)std::max(1ll, std::min(want, room / 2));
  if (2ll * p.target > room) return CWEN_ESCRATCH;
  if (a.max_len + a.max_nodes <= unit) p.target = 0;             // no chunks worth joining
  p.slots = 2 * p.target;
  p.ml = (float2 *)ctx->attn_part;
  p.po = ctx->attn_part + (((size_t)nkv * p.slots * rt * 2 + 3) & ~(size_t)3);
  const long long items = p.target + a.n_seq * tiles;            // at most
  if (items * nkv > INT32_MAX || (long long)a.total * a.nh > INT32_MAX) return CWEN_EINVAL;
  const dim3 grid((unsigned)(items * nkv));
  int rc = by_type(a.kv.type, D, [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int dim = decltype(d)::value, BN = dim == 256 ? 32 : 64;
    if (form == 1) hipLaunchKernelGGL((tree_few_kernel<T, dim>), grid, dim3(256), 0, st, a, p);
    else if constexpr (dim == 256) hipLaunchKernelGGL((tree_many_kernel<T, dim, 4, BN, 1, 2>), grid, dim3(256), 0, st, a, p);
    else hipLaunchKernelGGL((tree_many_kernel<T, dim, 4, BN, 1, 2>), grid, dim3(256), 0, st, a, p);
  });
  if (rc || !p.target) return rc;
  return by_type(a.kv.type, D, [&](auto t, auto d) {
    hipLaunchKernelGGL((tree_join_kernel<decltype(t), decltype(d)::value>), dim3((unsigned)a.total * a.nh), dim3(256), 0, st, a, p,
                       rt, unit);
  });
}
