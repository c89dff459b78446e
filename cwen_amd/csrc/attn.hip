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
    int lane = threadIdx.x & 63;    // opaque: what follows from it is not kept through the tiles
    asm volatile("" : "+v"(lane));
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
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int e = 0; e < E; ++e) o[lane * E + e] = (typename T::elem)(sees ? acc[e] / l : 0.f);
    if (lse && lane == 0) *lse = LN2 * (m + __builtin_amdgcn_logf(l));
  }
};

// Inclusive sum over the wave's lanes (row shifts, then row broadcasts).
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ int scan64(int v) {
  v = dpp_add<0x111, 0xF>(v);
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);
  return dpp_add<0x143, 0xC>(v);
}
__device__ __forceinline__ int lane_of(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ int max64(int v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = max(v, __shfl_xor(v, d));
  return v;
}

// ---- packed prompts ----
// Sequence and tile of item `it` of the sequences' tiles of BM queries.  Every wave
// finds it by itself.
struct Item {
  int seq, tile;      // seq < 0: past the last one
  int q0, nq, k0, nk; // the sequence's first query, queries, first key, keys
};
__device__ __forceinline__ int span(const int *cu, int s, int total, int *first) {
  const int a = min(max(cu[s], 0), total), b = min(max(cu[s + 1], 0), total);
  *first = a;
  return max(b - a, 0);
}
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Long tiles first: the sequences' last tiles, then those before, all that have as
// many keys behind each other (up to 64 sequences; past them sequence by sequence
// from the last).  In the sequences' own order a long one's last tiles may start when the
// others are done.
template <int BM> __device__ __forceinline__ Item find_item(const PromptArgs &a, int it) {
  const int lane = threadIdx.x & 63;
  int q0 = 0, nq = 0, k0 = 0, nk = 0;
  auto load = [&](int s) {
    nq = nk = 0;
    if (s >= a.n_seq) return;
    nq = span(a.cu_q, s, a.total_q, &q0);
    nk = span(a.cu_k, s, a.total_k, &k0);
  };
  auto item = [&](int s0, int w, int tile) {
    return Item{scalar(s0 + w), scalar(tile), lane_of(q0, w), lane_of(nq, w), lane_of(k0, w), lane_of(nk, w)};
  };
  load(lane);
  int tiles = (nq + BM - 1) / BM;
  if (a.n_seq <= 64) {
    // The level: the largest tile index i such that more than `it` tiles have an index >= i.
    if (lane_of(scan64(tiles), 63) <= it) return {-1};
    int lo = 0, hi = lane_of(max64(tiles), 0);            // tiles of an index >= hi: none
    while (lo + 1 < hi) {
      const int mid = (lo + hi) >> 1;
      if (lane_of(scan64(max(tiles - mid, 0)), 63) > it) lo = mid;
      else hi = mid;
    }
    it -= lane_of(scan64(max(tiles - lo - 1, 0)), 63);     // which of the level's sequences
    const unsigned long long have = __ballot(tiles > lo);
    const int rank = __builtin_popcountll(have & ((1ull << lane) - 1));
    return item(0, __builtin_ctzll(__ballot(tiles > lo && rank == it)), lo);
  }
  // From the last sequence's last tile on: the total first.
  int all = lane_of(scan64(tiles), 63);
  for (int s0 = 64; s0 < a.n_seq; s0 += 64) {
    load(s0 + lane);
    all += lane_of(scan64((nq + BM - 1) / BM), 63);
  }
  it = all - 1 - it;
  if (it < 0) return {-1};
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    load(s0 + lane);
    tiles = (nq + BM - 1) / BM;
    const int inc = scan64(tiles);
    const unsigned long long past = __ballot(inc > it);
    if (past) {
      const int w = __builtin_ctzll(past);
      return item(s0, w, it - lane_of(inc - tiles, w));
    }
    it -= lane_of(inc, 63);
  }
  return {-1};
}

// Bound by the matrix cores, and there by power: 32768 tokens of 32/8 heads of 128 in bf16 take
// 7.55 to 7.9 ms, 1.11 to 1.17 PFLOP/s with the matrix pipes 57 % busy at 1.94 GHz (a product of
// 8192^3 reaches 1.2 to 1.38); 9 prompts of 16301 tokens in all 334 to 355 us (0.87 to 0.92), 4096 tokens
// of 24/4 heads of 256 in f16 225 to 231 us (0.89 to 0.92: the longest row sets the time).
// RW KW waves share double-buffered tiles of KW BN keys: RW of them have 32 queries
// of one head each, and with KW = 2 the first RW take one half of every tile's keys, the
// others, for the same queries, the other; their sums meet at the end.
template <typename T, int D, int RW, int KW, int BN, int OCC>
__global__ __launch_bounds__(64 * RW * KW, OCC) void prompt_kernel(PromptArgs a) {
  typedef typename T::elem elem;
  constexpr int NW = RW * KW, WM = 32, BM = WM * RW, BT = KW * BN;
  __shared__ __align__(1024) elem K0[BT * D], K1[BT * D], V0[BT * D], V1[BT * D];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = a.nh / a.nkv;
  // Blocks of one kv head go to one or two XCDs (block b runs on XCD b % 8), long rows first.
  const int hh = blockIdx.x % a.nh, h = (hh % a.nkv) * g + hh / a.nkv, hkv = hh % a.nkv;
  const Item item = find_item<BM>(a, blockIdx.x / a.nh);
  if (item.seq < 0) return;
  const int tile = item.tile, q0 = item.q0, nq = item.nq, k0 = item.k0, nk = item.nk, off = nk - nq;
  const int rw = wave % RW, kw = wave / RW;
  const int first = tile * BM, w0 = first + rw * WM;        // the workgroup's and this wave's first query
  const elem *kp = (const elem *)a.k + (long long)k0 * a.ks + hkv * D, *vp = (const elem *)a.v + (long long)k0 * a.vs + hkv * D;
  const int kend = min(min(first + BM, nq) + off, nk);           // keys that the workgroup's rows see
  const int wend = min(min(w0 + WM, nq) + off, nk);              // and this wave's
  const float c = a.scale * LOG2E;
  auto land = [&](elem *Kd, elem *Vd, int t0) __attribute__((always_inline)) {
    land_rows<D, BT, false, NW>(Kd, wave, t0, nk - 1, (uint32_t)a.ks * 2, [&](int, int j) { return kp + j * a.ks; });
    land_rows<D, BT, true, NW>(Vd, wave, t0, nk - 1, (uint32_t)a.vs * 2, [&](int, int j) { return vp + j * a.vs; });
  };
  auto ready = [&]() __attribute__((always_inline)) {
    wait_loads<0>();
    lds_barrier();
    asm volatile("" ::: "memory");
  };
  // Tiles that every row sees whole come first, two per turn; what is left has
  // its keys compared with each row's last.
  const int full = max(min(first + off + 1, nk), 0) / (2 * BT) * (2 * BT);
  if (kend > 0) land(K0, V0, 0);
  AttnWave<T, D, BN> w;
  const int row = w0 + n, limit = row < nq ? row + off : -1;     // this lane's query and its last key
  w.start(row < nq ? (const elem *)a.q + (long long)(q0 + row) * a.qs + h * D : nullptr);
  const int k0w = kw * BN, at = k0w * D;                         // this wave's keys of a tile
  int t0 = 0;
  for (; t0 < full; t0 += 2 * BT) {
    ready();
    land(K1, V1, t0 + BT);
    w.template tile<false>(K0 + at, V0 + at, c, [](int) { return false; });
    ready();
    if (t0 + 2 * BT < kend) land(K0, V0, t0 + 2 * BT);
    w.template tile<false>(K1 + at, V1 + at, c, [](int) { return false; });
  }
  for (; t0 < kend; t0 += 2 * BT) {
    ready();
    if (t0 + BT < kend) land(K1, V1, t0 + BT);
    if (t0 + k0w < wend) w.template tile<true>(K0 + at, V0 + at, c, [&](int j) { return t0 + k0w + j + 4 * (lane >> 5) > limit; });
    if (t0 + BT >= kend) break;
    ready();
    if (t0 + 2 * BT < kend) land(K0, V0, t0 + 2 * BT);
    if (t0 + BT + k0w < wend) w.template tile<true>(K1 + at, V1 + at, c, [&](int j) { return t0 + BT + k0w + j + 4 * (lane >> 5) > limit; });
  }
  lds_barrier();                 // every wave is through with the tiles
  elem *mine = (rw * 4 / RW == 0 ? K0 : rw * 4 / RW == 1 ? K1 : rw * 4 / RW == 2 ? V0 : V1) + rw % (RW / 4) * (4 * BT * D / RW);
  if constexpr (KW == 2) {       // the second half's sums, lane by lane as they lie in registers
    static_assert(RW == 4 && BT * sizeof(elem) >= 32 * sizeof(float), "a wave's outputs fill an array");
    __shared__ float s_ml[RW][3][64];
    float4 *x = (float4 *)mine + lane;
    if (kw) {
#pragma unroll
      for (int b = 0; b < D / 32; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[64 * (4 * b + i)] = make_float4(w.o[b][4 * i], w.o[b][4 * i + 1], w.o[b][4 * i + 2], w.o[b][4 * i + 3]);
      s_ml[rw][0][lane] = w.m;
      s_ml[rw][1][lane] = w.l;
      s_ml[rw][2][lane] = w.odd;
    }
    lds_barrier();
    if (kw) return;
    const float m = s_ml[rw][0][lane], M = fmaxf(w.m, m);
    const float f0 = w.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m - M), f1 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
    w.m = M;
    w.l = w.l * f0 + s_ml[rw][1][lane] * f1;
    w.odd += s_ml[rw][2][lane];
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = x[64 * (4 * b + i)];
        w.o[b][4 * i] = w.o[b][4 * i] * f0 + v.x * f1;
        w.o[b][4 * i + 1] = w.o[b][4 * i + 1] * f0 + v.y * f1;
        w.o[b][4 * i + 2] = w.o[b][4 * i + 2] * f0 + v.z * f1;
        w.o[b][4 * i + 3] = w.o[b][4 * i + 3] * f0 + v.w * f1;
      }
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
  const float l = w.sum(), inv = limit < 0 ? 0.f : 1.f / l;
  if (a.lse && row < nq && lane < 32) a.lse[(long long)(q0 + row) * a.nh + h] = LN2 * (w.m + __builtin_amdgcn_logf(l));
  // The outputs through LDS, DC columns of a wave's rows at a time, so that a store takes whole
  // rows.  From the registers it takes 32 rows, 16 bytes of each, whose distance often puts them
  // all in one channel of the L2: 1.5 % of a prompt of 4096 tokens with heads of 256, 2.5 % of 40
  // prompts of 125 with heads of 64.
  constexpr int DC = BT * D / (8 * RW) < D ? BT * D / (8 * RW) : D, PC = DC / 8, RPI = 64 / PC, IN = 32 / RPI, XOR = PC < 16 ? PC - 1 : 15;
  int me = lane;                 // opaque: its addresses are not kept through the tiles
  asm volatile("" : "+v"(me));
  const int x = me & 31, half = me >> 5, pc = me % PC, y0 = me / PC;
  elem *to = (elem *)a.o + (long long)(q0 + w0 + y0) * a.os + h * D + 8 * pc;
#pragma unroll
  for (int d0 = 0; d0 < D; d0 += DC) {
#pragma unroll
    for (int b = d0 / 32; b < (d0 + DC) / 32; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typename AttnOps<T>::vec4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (elem)(limit < 0 ? 0.f : w.o[b][4 * i + j] * inv);
        *(typename AttnOps<T>::vec4 *)(mine + x * DC + 8 * ((4 * (b - d0 / 32) + i) ^ (x & XOR)) + 4 * half) = v;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    typename AttnOps<T>::vec8 v[IN];
#pragma unroll
    for (int u = 0; u < IN; ++u) {
      const int y = y0 + u * RPI;
      v[u] = *(const typename AttnOps<T>::vec8 *)(mine + y * DC + 8 * (pc ^ (y & XOR)));
    }
#pragma unroll
    for (int u = 0; u < IN; ++u)
      if (w0 + y0 + u * RPI < nq) *(typename AttnOps<T>::vec8 *)(to + (long long)u * RPI * a.os + d0) = v[u];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- trees over the paged cache ----
// Row r of group s and a kv head is head r % g of node r / g: the query heads
// that share the kv head's keys lie side by side, so a group's n nodes are n g
// rows against one stream of pages.  Few rows leave the work bound by that
// stream, many by the matrix cores, and both want it cut along the keys, since
// groups are few.  All row tiles (RT rows) of all groups are laid end to end, each
// as long as its keys (in units of 128), and the line is cut into `lines`
// equal pieces, one workgroup each: no long sequence sets the time, and a piece that
// begins or ends inside a row tile leaves a partial result, at most two a
// workgroup.  Nothing of this is known on the host: every workgroup finds
// its pieces from the lengths on the device, 64 groups at a time.
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
    const int len = a.kv.len[q.id];
    q.keys = kv_readable(len, q.nodes, a.kv.held[q.id], a.kv.page, a.kv.max_pages, &q.bad);
    q.len = kv_cached(len, q.keys);       // what the masks' words are counted by
  }
  return q;
}
struct TreeTile {
  int s, tile;              // group (< 0: none) and row tile of it
  int units;                // its length without the `extra` behind it
  int at;                   // where it begins on the line
};
// Where every group has the same number of row tiles (`levels`, more than one of
// them for many rows), each level has a line of its own, as long as the groups'
// keys, cut alike: the workgroups that read the same keys for different rows then
// run at the same time on the same XCD and find them in its L2.  On one line, 288
// rows behind 32000 positions read every key from memory three times (106 us
// against 89 with lines that happened to be cut alike).
// A row tile takes longer than its keys: its pages are looked up, its outputs leave, its drafted
// keys are slower.  `extra` units behind its keys, with no work in them, stand for that, so a piece
// that holds the end of one gets fewer keys: 48 trees behind up to 12000 positions (32/8 heads of
// 128) 131 us against 147 without, behind 2000 32 against 42.
// Pieces shorter than 128 keys leave more partials than they save time: 288 rows of 256 behind
// 2000 positions 31 us, cut by 64 keys 38 (behind 300 26 and 25).
constexpr int UNIT = 128;
struct TreePlan {
  int rt, extra, levels, lines;   // levels 1: one line for all (or one row tile a group)
  int total;                     // a line's length; the launch has made sure that the sums fit 32 bits
  // A lane's group: its sequence, row tiles and units.
  struct Mine {
    TreeSeq q;
    int tiles, units;
  };
  __device__ __forceinline__ Mine load(const TreeArgs &a, int s0) const {
    const int s = s0 + (int)(threadIdx.x & 63);
    Mine m = {};
    if (s >= a.n_seq) return m;
    m.q = tree_seq(a, s);
    m.tiles = (m.q.nodes * (a.nh / a.kv.n_kv_head) + rt - 1) / rt;
    m.units = max((m.q.keys + UNIT - 1) / UNIT, 1) + extra;  // rows without keys are work too
    return m;
  }
  // m: load(a, 0)
  __device__ __forceinline__ TreePlan(int rt, int extra) : rt(rt), extra(extra) {}
  __device__ __forceinline__ void lay(const TreeArgs &a, Mine m, int want, int most) {
    int sum = 0, one = 0;
    for (int s0 = 0;;) {
      sum += lane_of(scan64(m.tiles * m.units), 63);
      if (want > 1) one += lane_of(scan64(m.tiles ? m.units : 0), 63);
      if ((s0 += 64) >= a.n_seq) break;
      m = load(a, s0);
    }
    levels = want > 1 && sum == one * want ? want : 1;   // no group has more than `want`: all have as many
    total = levels > 1 ? one : sum;
    lines = min(most / levels, total);
  }
  // Where piece w begins, and the piece that holds position u.
  __device__ __forceinline__ int begin(int w) const { return total / lines * w + total % lines * w / lines; }
  __device__ __forceinline__ int piece(int u) const { return (int)(((long long)(u + 1) * lines - 1) / total); }
  // The row tile at position u of a level's line; or, with node >= 0, the first one of
  // the group that holds it.  q: the group's sequence.
  __device__ __forceinline__ TreeTile find(const TreeArgs &a, Mine m, int level, int u, int node, TreeSeq *q) const {
    int at = 0;
    for (int s0 = 0; s0 < a.n_seq;) {
      const int mine = (levels > 1 ? m.tiles > 0 : m.tiles) * m.units, inc = at + scan64(mine);
      const unsigned long long hit = __ballot(node >= 0 ? node >= m.q.c0 && node < m.q.c0 + m.q.nodes : inc > u);
      if (hit) {
        const int w = __builtin_ctzll(hit), n = lane_of(m.units, w), first = lane_of(inc - mine, w);
        const int tile = node >= 0 ? 0 : (u - first) / n;
        *q = {lane_of(m.q.c0, w), lane_of(m.q.nodes, w), lane_of(m.q.len, w), lane_of(m.q.keys, w), lane_of(m.q.id, w),
              lane_of(m.q.bad, w) != 0};
        return {scalar(s0 + w), scalar(levels > 1 ? level : tile), n - extra, scalar(first + tile * n)};
      }
      at = lane_of(inc, 63);
      if ((s0 += 64) < a.n_seq) m = load(a, s0);
    }
    return {-1, 0, 0, 0};
  }
};
// The level, piece and kv head of a workgroup: blocks run on XCD b % 8, and a
// piece's levels follow each other there.
struct TreeBlock {
  int level, piece, hkv;
};
__device__ __forceinline__ TreeBlock tree_block(const TreePlan &p, int nkv) {
  const int b = blockIdx.x, q = b >> 3, pair = q / p.levels * 8 + (b & 7);
  return {q % p.levels, pair / nkv, pair % nkv};
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

// A share of a row's keys leaves its maximum and sum {m, l}; the score that set a finite maximum adds
// about 1 to the sum (the maximum's own rounding away).  With a maximum of -inf, l is 0 where the row saw
// none of the keys, LOWEST where all that it saw have scores of -inf, and NaN.  Such keys weigh
// nothing beside others, and 2^-100 is lost in their sum; a row that sees no others, whose
// sum is then that of up to 1024 shares, is NaN (0 / 0), its lse -inf.
constexpr float LOWEST = 0x1p-100f;
__device__ __forceinline__ float share_sum(bool saw, float l) { return saw && l == 0.f ? LOWEST : l; }
// How a share's sums count against the row's maximum M (NaN stays), and what it adds to the row's sum.
__device__ __forceinline__ float chunk_weight(float2 ml, float M, float *sum) {
  const float f = ml.x == -INFINITY ? 0.f * ml.y : __builtin_amdgcn_exp2f(ml.x - M);
  *sum += ml.x == -INFINITY ? ml.y : ml.y * f;
  return f;
}
// What a row's sums are multiplied by.
__device__ __forceinline__ float row_scale(float l) { return l == 0.f ? 0.f : l < 0x1p-80f ? NAN : 1.f / l; }

struct TreeLaunch {
  int lines, levels;            // pieces of a kv head, of all levels; row tiles of a group at most, or 1
  int extra;                    // units that a row tile counts beyond its keys
  float *po;                    // partial outputs [kv head][2 lines][row][D]: piece w's first row tile, its last
  float2 *ml;                   // and their maxima and sums [kv head][2 lines][row]
  int *count;                   // few rows: arrivals per (kv head, group), zero between launches; null: joined by a launch
};

// One group's rows against the pages: what both forms share.
template <typename T, int D> struct TreeRows {
  typedef typename T::elem elem;
  const TreeArgs &a;
  const TreeSeq &q;
  int hkv, g;
  const elem *kb, *vb;              // the layer's rows of the kv head in page 0
  int64_t step;                     // elements from page to page
  int shift, last, n_pages;         // log2 of the page size, the last key
  // The sequence's pages, as constant memory: no kernel that reads them writes
  // them, and with a uniform index the entry is a scalar load.
  const __attribute__((address_space(4))) int *tab;
  __device__ __forceinline__ TreeRows(const TreeArgs &a, const TreeSeq &q, int hkv)
      : a(a), q(q), hkv(hkv), g(a.nh / a.kv.n_kv_head), step((int64_t)a.kv.n_kv_head * a.kv.page * D),
        shift(__builtin_ctz(a.kv.page)), last(q.keys - 1), n_pages(a.kv.n_pages),
        tab((const __attribute__((address_space(4))) int *)(a.kv.table + (size_t)q.id * a.kv.max_pages)) {
    const int64_t first = kv_at(a.layer, 0, hkv, 0, a.kv.n_pages, a.kv.n_kv_head, a.kv.page, D);
    kb = (const elem *)a.kv.k + first;
    vb = (const elem *)a.kv.v + first;
  }
  // The page that holds key j (past the last: the last).
  __device__ __forceinline__ int page(int j) const { return tab[min(j, last) >> shift]; }
  // Key j of that page.
  __device__ __forceinline__ const elem *row(const elem *pool, int page, int j, bool *bad) const {
    return pool + kv_page_ok(page, n_pages, bad) * step + (j & ((1 << shift) - 1)) * D;
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
    const int i = r / g;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    AttnRow<T, D> x;
    x.run(query(r), begin, end, a.scale * LOG2E,
          [&](int j) {
            const int u = j - q.len;
            return u < 0 || (mk ? (mk[u >> 6] >> (u & 63)) & 1 : u <= i);
          },
          [&](int j, const elem **k, const elem **v) {
            bool bad = false;
            *k = row(kb, page(j), j, &bad);
            *v = row(vb, page(j), j, &bad);
          });
    if (!po) {
      x.store(out(r), lse(r));
      return;
    }
#pragma unroll
    for (int e = 0; e < D / 64; ++e) po[lane * (D / 64) + e] = x.acc[e];
    if (lane == 0) *ml = make_float2(x.m, share_sum(x.sees, x.l));
  }
};

// Values that other workgroups of this launch wrote: at the device's coherence point.
__device__ __forceinline__ void put2(void *p, float x, float y) {
  __hip_atomic_store((uint64_t *)p, __builtin_bit_cast(uint64_t, make_float2(x, y)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const void *p) {
  return __builtin_bit_cast(float2, __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ float max64(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// Bound by a chain of six trips to memory, then by the pages' bytes: one node of 24/4 heads of 256
// behind 4096 positions 9.7 to 10.8 us (16.8 MB), 64 of them behind up to 8000 102 us, 48 of 32/8 heads
// of 128 behind up to 12000 218 us (1.2 GB, 5.5 TB/s).
// Few rows: one tile of 32, the chunk's keys dealt to 4 waves 32 at a time.  A wave
// has its own K and V rows in LDS and no barrier in its loop: the next K rows
// are requested when the scores are done, the next V rows after the outputs, so
// that half of its LDS and more is always under way.  The waves' sums meet at the
// end.  Where the chunks of a group are few, the last workgroup to leave one joins
// them in the same launch.
template <typename T, int D> __global__ __launch_bounds__(256, 1) __attribute__((amdgpu_num_vgpr(256))) void tree_few_kernel(TreeArgs a, TreeLaunch p) {
  typedef typename T::elem elem;
  constexpr int BN = 32, NW = 4, PC = D / 4;      // PC: 16-byte pieces of an f32 row
  constexpr int LOADS = BN * D / 8 / 64;                          // of one tile of K or V, by one wave
  constexpr int JOIN = 16;
  __shared__ __align__(1024) elem Ks[NW * BN * D], Vs[NW * BN * D];
  __shared__ float2 s_ml[NW][32];
  __shared__ int s_end;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nkv = a.kv.n_kv_head, n = lane & 31, hi = lane >> 5;
  TreePlan plan(32, p.extra);
  TreePlan::Mine groups = plan.load(a, 0);
  plan.lay(a, groups, p.levels, p.lines);
  const TreeBlock me = tree_block(plan, nkv);
  const int piece = scalar(me.piece), hkv = scalar(me.hkv);
  if (piece >= plan.lines) return;
  const int stop = scalar(plan.begin(piece + 1));
  bool first = true;
  for (int u = scalar(plan.begin(piece)); u < stop; first = false) {
    if (!first) groups = plan.load(a, 0);          // not kept through the tiles
    TreeSeq q;
    const TreeTile item = plan.find(a, groups, me.level, u, -1, &q);
    const int skip = u - item.at, count = min(item.at + item.units, stop) - u;
    u = min(item.at + item.units + plan.extra, stop);
    if (count <= 0) continue;
    if (q.bad && tid == 0) kv_raise(a.kv, CWEN_KV_PAGE);
    const TreeRows<T, D> rows(a, q, hkv);
    const int base = item.tile * 32, R = min(q.nodes * rows.g - base, 32), r = base + n;
    const bool live = n < R;
    const int begin = skip * UNIT, end = min(begin + count * UNIT, q.keys);
    elem *Kw = Ks + wave * BN * D, *Vw = Vs + wave * BN * D;
    bool bad = false;
    int t0 = begin + wave * BN;
    AttnWave<T, D, BN> w;
    // 16 rows never straddle a page: two lookups a tile, for the tile after the current one.
    int pg[2];
    auto land = [&](elem *dst, const elem *pool, auto isv) __attribute__((always_inline)) {
      constexpr int half = 16 / (64 / (D / 8));       // loads of 16 rows
      land_rows<D, BN, decltype(isv)::value, 1>(dst, 0, t0, rows.last, D * 2,
                                                [&](int i, int j) { return rows.row(pool, pg[i / half], j, &bad); });
    };
    auto pages = [&]() __attribute__((always_inline)) {
      pg[0] = rows.page(t0);
      pg[1] = rows.page(t0 + 16);
    };
    if (t0 < end) {
      pages();
      land(Kw, rows.kb, std::false_type{});
      land(Vw, rows.vb, std::true_type{});
    }
    w.start(live ? rows.query(r) : nullptr);
    const float c = a.scale * LOG2E;
    const unsigned long long *mask = live ? rows.mask(r) : nullptr;
    const int node = r / rows.g;
    uint32_t saw = 0;
    auto step = [&](auto hide) __attribute__((always_inline)) {
      constexpr bool H = decltype(hide)::value;
      const int u0 = t0 - q.len;
      t0 += UNIT;
      if (t0 < end) pages();
      f32x16_t s[1];
      typename AttnWave<T, D, BN>::vec8 pr[2];
      // Loads land in the order of their requests: K's are there when no more
      // than V's are still under way, V's when no more than the next K's.
      wait_loads<LOADS>();
      w.scores(Kw, s);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // its rows are read
      if (t0 < end) land(Kw, rows.kb, std::false_type{});
      const uint32_t see = H ? tree_sees(mask, a.mw, node, q.keys - q.len, u0) : ~0u;
      saw |= see;
      const uint32_t mine = see >> 4 * hi;
      w.template soft<H>(s, c, [&](int j) { return !((mine >> j) & 1); }, pr);
      if (t0 < end) wait_loads<LOADS>();
      else wait_loads<0>();
      w.template outputs<H>(Vw, pr);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (t0 < end) land(Vw, rows.vb, std::true_type{});
    };
    while (t0 < min(end, q.len - BN + 1)) step(std::false_type{});  // tiles of cached positions
    while (t0 < end) step(std::true_type{});
    if (bad) kv_raise(a.kv, CWEN_KV_PAGE);
    const float l = w.sum();
    if (lane < 32) s_ml[wave][n] = make_float2(w.m, share_sum(saw != 0, l));
    const bool whole = count == item.units;
    const size_t slot = ((size_t)hkv * 2 * p.lines + 2 * (piece * plan.levels + me.level) + !first) * 32;
    auto join = [&]() __attribute__((always_inline)) {
      const int at0 = item.at, p0 = plan.piece(at0), nsplit = plan.piece(at0 + item.units - 1) - p0 + 1;
      int *count = p.count + hkv * a.n_seq + item.s;
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");    // the partial has arrived
      __syncthreads();
      if (tid == 0) s_end = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nsplit - 1;
      __syncthreads();
      if (!s_end) return;
      const size_t first0 = ((size_t)hkv * p.lines + p0) * 2 * 32, odd0 = plan.begin(p0) < at0 ? 32 : 0;
      auto place = [&](int x, int y) { return first0 + (size_t)x * 64 + (x ? 0 : odd0) + y; };
      // The chunks' weights of as many rows as LDS holds, then 16 bytes a thread of
      // their outputs, JOIN chunks under way at a time: each round is a trip to memory.
      float *weight = (float *)Ks;
      const int batch = min(R, NW * BN * D / 2 / nsplit);
      for (int y0 = 0; y0 < R; y0 += batch) {
        const int y1 = min(y0 + batch, R);
        for (int y = y0 + wave; y < y1; y += NW) {
          float M = -INFINITY, L = 0.f;
          for (int x = lane; x < nsplit; x += 64) M = fmaxf(M, get2(p.ml + place(x, y)).x);
          M = max64(M);
          for (int x = lane; x < nsplit; x += 64) weight[(y - y0) * nsplit + x] = chunk_weight(get2(p.ml + place(x, y)), M, &L);
          L = sum64(L);
          if (lane == 0) s_ml[0][y] = make_float2(M, L);
        }
        __syncthreads();
        for (int z = tid; z < (y1 - y0) * PC; z += 256) {
          const int y = y0 + z / PC, pc = z % PC;
          const float *wy = weight + (y - y0) * nsplit;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int x = 0; x < nsplit; x += JOIN) {
            float2 v[JOIN][2];
#pragma unroll
            for (int u = 0; u < JOIN; ++u) {
              const float *po = p.po + place(min(x + u, nsplit - 1), y) * D + 4 * pc;
              v[u][0] = get2(po);
              v[u][1] = get2(po + 2);
            }
#pragma unroll
            for (int u = 0; u < JOIN; ++u) {
              if (x + u >= nsplit) break;
              const float f = wy[x + u];
              o.x = fmaf(v[u][0].x, f, o.x); o.y = fmaf(v[u][0].y, f, o.y);
              o.z = fmaf(v[u][1].x, f, o.z); o.w = fmaf(v[u][1].y, f, o.w);
            }
          }
          const float2 ml = s_ml[0][y];
          const float inv = row_scale(ml.y);
          const typename AttnOps<T>::vec4 e = {(elem)(o.x * inv), (elem)(o.y * inv), (elem)(o.z * inv), (elem)(o.w * inv)};
          *(typename AttnOps<T>::vec4 *)(rows.out(base + y) + 4 * pc) = e;
          if (pc == 0 && a.lse) *rows.lse(base + y) = LN2 * (ml.x + __builtin_amdgcn_logf(ml.y));
        }
        __syncthreads();
      }
      if (tid == 0) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    if (__syncthreads_or(w.odd != w.odd)) {        // a hidden value may have leaked: the rows one by one
      for (int x = wave; x < R; x += NW)
        rows.plain(base + x, begin, end, whole ? nullptr : p.po + (slot + x) * D, whole ? nullptr : p.ml + slot + x);
      if (!whole && p.count) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
        join();
      }
      __syncthreads();
      continue;
    }
    // Each wave's outputs against the row's common maximum, through LDS (rows of D
    // floats, their pieces permuted by the row), then summed in the waves' order.
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) M = fmaxf(M, s_ml[x][n].x);
    const float f = w.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m - M);
    auto area = [&](int x) { return (float *)(x < 2 ? Ks : Vs) + (x & 1) * 32 * D; };
    float *mine = area(wave);
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(float4 *)(mine + n * D + 4 * ((8 * b + 2 * i + hi) ^ (n & 15))) =
            make_float4(w.o[b][4 * i] * f, w.o[b][4 * i + 1] * f, w.o[b][4 * i + 2] * f, w.o[b][4 * i + 3] * f);
    __syncthreads();
    for (int x = tid; x < R * PC; x += 256) {
      const int y = x / PC, pc = x - y * PC;
      float Mr = -INFINITY, L = 0.f;
#pragma unroll
      for (int u = 0; u < NW; ++u) Mr = fmaxf(Mr, s_ml[u][y].x);
#pragma unroll
      for (int u = 0; u < NW; ++u) chunk_weight(s_ml[u][y], Mr, &L);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < NW; ++u) {
        const float4 v = *(const float4 *)(area(u) + y * D + 4 * (pc ^ (y & 15)));
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
      }
      if (whole) {
        const float inv = row_scale(L);
        const typename AttnOps<T>::vec4 e = {(elem)(o.x * inv), (elem)(o.y * inv), (elem)(o.z * inv), (elem)(o.w * inv)};
        *(typename AttnOps<T>::vec4 *)(rows.out(base + y) + 4 * pc) = e;
        if (pc == 0 && a.lse) *rows.lse(base + y) = LN2 * (Mr + __builtin_amdgcn_logf(L));
      } else if (p.count) {
        float *po = p.po + (slot + y) * D + 4 * pc;
        put2(po, o.x, o.y);
        put2(po + 2, o.z, o.w);
        if (pc == 0) put2(p.ml + slot + y, Mr, L);
      } else {
        *(float4 *)(p.po + (slot + y) * D + 4 * pc) = o;
        if (pc == 0) p.ml[slot + y] = make_float2(Mr, L);
      }
    }
    if (!whole && p.count) join();
    __syncthreads();                               // LDS is free for the next row tile
  }
}

// Bound by the pages' bytes while rows are few (48 trees of up to 24 nodes behind up to 12000
// positions, 32/8 heads of 128: 128 to 130 us, 617 MB, 4.8 TB/s), by matrix work and the partials with
// more (48 nodes of 24/4 heads of 256 behind 32000: 64 us).
// Many rows: 4 waves of 32 rows share double-buffered tiles of BN keys.
template <typename T, int D, int BN>
__global__ __launch_bounds__(256, 2) void tree_many_kernel(TreeArgs a, TreeLaunch p) {
  typedef typename T::elem elem;
  constexpr int NW = 4, RT = 32 * NW, PER = BN * D / 8 / (64 * NW);
  __shared__ __align__(1024) elem K0[BN * D], K1[BN * D], V0[BN * D], V1[BN * D];
  constexpr int WORDS = CWEN_TREE_MAX / 32;
  __shared__ uint32_t s_see[NW][WORDS][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nkv = a.kv.n_kv_head, n = lane & 31, hi = lane >> 5;
  TreePlan plan(RT, p.extra);
  TreePlan::Mine groups = plan.load(a, 0);
  plan.lay(a, groups, p.levels, p.lines);
  const TreeBlock me = tree_block(plan, nkv);
  const int piece = scalar(me.piece), hkv = scalar(me.hkv);
  if (piece >= plan.lines) return;
  const int stop = scalar(plan.begin(piece + 1));
  bool first = true;
  for (int u = scalar(plan.begin(piece)); u < stop; first = false) {
    if (!first) groups = plan.load(a, 0);          // not kept through the tiles
    TreeSeq q;
    const TreeTile item = plan.find(a, groups, me.level, u, -1, &q);
    const int skip = u - item.at, count = min(item.at + item.units, stop) - u;
    u = min(item.at + item.units + plan.extra, stop);
    if (count <= 0) continue;
    if (q.bad && tid == 0) kv_raise(a.kv, CWEN_KV_PAGE);
    const TreeRows<T, D> rows(a, q, hkv);
    const int base = item.tile * RT + wave * 32, R = min(q.nodes * rows.g - base, 32);   // R <= 0: no rows here
    const int begin = skip * UNIT, end = min(begin + count * UNIT, q.keys);
    bool bad = false;
    const float c = a.scale * LOG2E;
    // The page of each load's rows (they lie in one page), a tile ahead.
    int pg[PER];
    auto pages = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < PER; ++i) pg[i] = rows.page(t0 + (i * NW + wave) * 64 / (D / 8));
    };
    auto land = [&](elem *Kd, elem *Vd, int t0) __attribute__((always_inline)) {
      land_rows<D, BN, false, NW>(Kd, wave, t0, rows.last, D * 2, [&](int i, int j) { return rows.row(rows.kb, pg[i], j, &bad); });
      land_rows<D, BN, true, NW>(Vd, wave, t0, rows.last, D * 2, [&](int i, int j) { return rows.row(rows.vb, pg[i], j, &bad); });
      if (t0 + BN < end) pages(t0 + BN);
      __builtin_amdgcn_sched_barrier(0);              // the addresses' registers are free again before the tile
    };
    auto ready = [&]() __attribute__((always_inline)) {
      wait_loads<0>();
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
      lds_barrier();
      lds_barrier();
      continue;
    }
    // What the rows see of the drafted nodes, before the tiles need the registers.
    const int words = (q.keys - q.len + 31) / 32;
    if (end > q.len) {
      const unsigned long long *mask = n < R ? rows.mask(base + n) : nullptr;
      for (int k = hi; k < words; k += 2) s_see[wave][k][n] = tree_sees(mask, a.mw, (base + n) / rows.g, q.keys - q.len, 32 * k);
    }
    AttnWave<T, D, BN> w;
    w.start(n < R ? rows.query(base + n) : nullptr);
    const int full = begin + max(min(end, q.len) - begin, 0) / (2 * BN) * (2 * BN);   // whole tiles of cached positions
    uint32_t saw = full > begin;
    auto part = [&](const elem *Kb, const elem *Vb, int t0) __attribute__((always_inline)) {
      uint32_t see[BN / 32];
#pragma unroll
      for (int b = 0; b < BN / 32; ++b) {
        const int u0 = t0 + 32 * b - q.len, k = u0 >> 5;              // 32 bits across two words
        const uint32_t lo = k < 0 ? ~0u : k < words ? s_see[wave][k][n] : 0;
        const uint32_t up = k < -1 ? ~0u : k + 1 < words ? s_see[wave][k + 1][n] : 0;
        see[b] = __builtin_amdgcn_alignbit(up, lo, u0 & 31);
        saw |= see[b];
        see[b] >>= 4 * hi;
      }
      w.template tile<true>(Kb, Vb, c, [&](int j) { return !((see[j >> 5] >> (j & 31)) & 1); });
    };
    for (; t0 < full; t0 += 2 * BN) {
      ready();
      land(K1, V1, t0 + BN);
      w.template tile<false>(K0, V0, c, [](int) { return false; });
      ready();
      if (t0 + 2 * BN < end) land(K0, V0, t0 + 2 * BN);
      w.template tile<false>(K1, V1, c, [](int) { return false; });
    }
    for (bool one = false; t0 < end; t0 += BN, one = !one) {
      ready();
      if (t0 + BN < end) land(one ? K0 : K1, one ? V0 : V1, t0 + BN);
      part(one ? K1 : K0, one ? V1 : V0, t0);
    }
    if (bad) kv_raise(a.kv, CWEN_KV_PAGE);
    const bool whole = count == item.units;
    const size_t slot = ((size_t)hkv * 2 * p.lines + 2 * (piece * plan.levels + me.level) + !first) * RT + wave * 32;
    lds_barrier();                                    // every wave is through with the tiles
    if (__any(w.odd != w.odd)) {
      for (int x = 0; x < R; ++x)
        rows.plain(base + x, begin, end, whole ? nullptr : p.po + (slot + x) * D, whole ? nullptr : p.ml + slot + x);
      lds_barrier();
      continue;
    }
    constexpr int DC = BN * D / 64, PC = DC / 4, RPI = 64 / PC;   // columns, 16-byte pieces and rows of a load
    int me_lane = lane;                               // opaque: its addresses are not kept through the tiles
    asm volatile("" : "+v"(me_lane));
    const int row = me_lane & 31, half = me_lane >> 5, pc = me_lane % PC;
    const float l = share_sum(saw != 0, w.sum()), inv = whole ? row_scale(l) : 1.f;
    if (me_lane < min(R, 32)) {
      if (!whole) p.ml[slot + row] = make_float2(w.m, l);
      else if (a.lse) *rows.lse(base + row) = LN2 * (w.m + __builtin_amdgcn_logf(l));
    }
    // The outputs through LDS, DC columns of a wave's rows at a time, so that lanes side by side
    // store what lies side by side: from the registers a store touches 32 rows, 32 bytes of each
    // (48 nodes behind 32000 positions, heads of 256: 70 us so, 66 through LDS).
    float *mine = (float *)(wave == 0 ? K0 : wave == 1 ? K1 : wave == 2 ? V0 : V1);
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += DC) {
#pragma unroll
      for (int b = d0 / 32; b < (d0 + DC) / 32; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(float4 *)(mine + row * DC + 4 * ((8 * (b - d0 / 32) + 2 * i + half) ^ (row & 15))) =
              make_float4(w.o[b][4 * i] * inv, w.o[b][4 * i + 1] * inv, w.o[b][4 * i + 2] * inv, w.o[b][4 * i + 3] * inv);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      for (int x = me_lane / PC; x < R; x += RPI) {
        const float4 v = *(const float4 *)(mine + x * DC + 4 * (pc ^ (x & 15)));
        if (whole) {
          const typename AttnOps<T>::vec4 e = {(elem)v.x, (elem)v.y, (elem)v.z, (elem)v.w};
          *(typename AttnOps<T>::vec4 *)(rows.out(base + x) + d0 + 4 * pc) = e;
        } else {
          *(float4 *)(p.po + (slot + x) * D + d0 + 4 * pc) = v;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    lds_barrier();                                 // LDS is free for the next row tile
  }
}

// The chunks of rows joined: a workgroup takes `hpw` heads of a node.  LR lanes find
// a row's chunks and their weights, into LDS; then each thread adds 16 bytes of a
// row's outputs, or, with fewer of those than threads, a share of its chunks. So
// the trips to memory are few however many rows a workgroup has: one after the
// other they took 28 us of a batch of 580 nodes, now 12; 33 chunks of one node take 6.4.
constexpr int JOIN_HEADS = 32;
template <typename T, int D, int LR>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, TreeLaunch p, int rt, int hpw) {
  typedef typename T::elem elem;
  constexpr int PC = D / 4, CAP = 4096, U = 8, Z = 2, C = 4;
  __shared__ float s_w[CAP];
  __shared__ float2 s_ml[JOIN_HEADS];
  __shared__ long long s_first[JOIN_HEADS];
  __shared__ int s_n[JOIN_HEADS], s_odd[JOIN_HEADS];
  __shared__ float4 s_o[256];
  const int tid = threadIdx.x, blocks = (a.nh + hpw - 1) / hpw, t = blockIdx.x / blocks, h0 = (blockIdx.x - t * blocks) * hpw;
  TreePlan plan(rt, p.extra);
  const TreePlan::Mine groups = plan.load(a, 0);
  plan.lay(a, groups, p.levels, p.lines);
  TreeSeq q;
  const TreeTile group = plan.find(a, groups, 0, 0, t, &q);
  if (group.s < 0 || plan.lines == 1) return;
  const int g = a.nh / a.kv.n_kv_head, rows = min(hpw, a.nh - h0), step = 2 * plan.levels * rt;
  const int batch = min(rows, CAP / plan.lines);                  // at most 4 workgroups a CU: lines <= 1024 <= CAP
  for (int y0 = 0; y0 < rows; y0 += batch) {
    const int nb = min(batch, rows - y0);
    for (int i = tid / LR; i < nb; i += 256 / LR) {
      const int h = h0 + y0 + i, hkv = h / g, r = (t - q.c0) * g + h - hkv * g, tile = r / rt, level = plan.levels > 1 ? tile : 0;
      const int at0 = group.at + (tile - level) * (group.units + p.extra), w0 = plan.piece(at0);
      const int n = plan.piece(at0 + group.units - 1) - w0 + 1, l = tid % LR;
      // Chunk x is piece w0 + x's: its first row tile's, but for chunk 0 if the piece began before this tile.
      const long long first = ((long long)hkv * 2 * p.lines + 2 * (w0 * plan.levels + level)) * rt + r % rt;
      const int odd = plan.begin(w0) < at0 ? rt : 0;
      float M = -INFINITY, L = 0.f;
      if (n > 1) {
        auto ml = [&](int x) { return p.ml[first + (long long)x * step + (x ? 0 : odd)]; };
        const float2 mine = ml(min(l, n - 1));
        if (l < n) M = mine.x;
        for (int x = l + LR; x < n; x += LR) M = fmaxf(M, ml(x).x);
#pragma unroll
        for (int d = 1; d < LR; d *= 2) M = fmaxf(M, __shfl_xor(M, d));
        for (int x = l; x < n; x += LR) s_w[i * plan.lines + x] = chunk_weight(x == l ? mine : ml(x), M, &L);
#pragma unroll
        for (int d = 1; d < LR; d *= 2) L += __shfl_xor(L, d);
      }
      if (l == 0) {
        s_n[i] = n;
        s_first[i] = first;
        s_odd[i] = odd;
        s_ml[i] = make_float2(M, L);
      }
    }
    __syncthreads();
    auto chunk = [&](int i, int pc, int x) {
      return *(const float4 *)(p.po + (s_first[i] + (long long)x * step + (x ? 0 : s_odd[i])) * D + 4 * pc);
    };
    auto add = [&](float4 &o, float4 v, float f) {
      o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y);
      o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    };
    auto leave = [&](int i, int pc, float4 o) {
      const int h = h0 + y0 + i;
      const float2 ml = s_ml[i];
      const float inv = row_scale(ml.y);
      const typename AttnOps<T>::vec4 e = {(elem)(o.x * inv), (elem)(o.y * inv), (elem)(o.z * inv), (elem)(o.w * inv)};
      *(typename AttnOps<T>::vec4 *)((elem *)a.o + (long long)t * a.os + h * D + 4 * pc) = e;
      if (a.lse && pc == 0) a.lse[(long long)t * a.nh + h] = LN2 * (ml.x + __builtin_amdgcn_logf(ml.y));
    };
    const int items = nb * PC;
    // Z pieces a thread, C chunks of each under way at a time (16 trees of 16 nodes, heads of 256: 12.0 us;
    // 4 pieces cost the registers that hold a fifth workgroup on the CU: 17.0; 1 piece of 8 chunks 13.8).
    if (items >= 256) {
      for (int z0 = tid; z0 < items; z0 += 256 * Z) {
        float4 o[Z];
        int n[Z], most = 0;
#pragma unroll
        for (int k = 0; k < Z; ++k) {
          o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          n[k] = z0 + 256 * k < items ? s_n[(z0 + 256 * k) / PC] : 0;
          if (n[k] == 1) n[k] = 0;
          most = max(most, n[k]);
        }
        for (int x = 0; x < most; x += C) {
          float4 v[Z][C];
#pragma unroll
          for (int k = 0; k < Z; ++k)
#pragma unroll
            for (int u = 0; u < C; ++u) {
              const int z = min(z0 + 256 * k, items - 1);
              v[k][u] = chunk(z / PC, z % PC, min(x + u, max(n[k] - 1, 0)));
            }
#pragma unroll
          for (int k = 0; k < Z; ++k)
#pragma unroll
            for (int u = 0; u < C; ++u)
              if (x + u < n[k]) add(o[k], v[k][u], s_w[(z0 + 256 * k) / PC * plan.lines + x + u]);
        }
#pragma unroll
        for (int k = 0; k < Z; ++k)
          if (n[k]) leave((z0 + 256 * k) / PC, (z0 + 256 * k) % PC, o[k]);
      }
    } else {                     // a share of a row's chunks each
      const int shares = 256 / items, z = tid % items, share = tid / items, i = z / PC, pc = z % PC;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      if (share < shares) {
        const int n = s_n[i] > 1 ? s_n[i] : 0, per = (n + shares - 1) / shares, x1 = min((share + 1) * per, n);
        for (int x = share * per; x < x1; x += U) {
          float4 v[U];
#pragma unroll
          for (int u = 0; u < U; ++u) v[u] = chunk(i, pc, min(x + u, x1 - 1));
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (x + u < x1) add(o, v[u], s_w[i * plan.lines + x + u]);
        }
      }
      s_o[tid] = o;
      __syncthreads();
      if (share == 0 && s_n[i] > 1) {
        for (int u = 1; u < shares; ++u) {
          const float4 v = s_o[tid + u * items];
          o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
        }
        leave(i, pc, o);
      }
    }
    __syncthreads();
  }
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

int attn_prompt_launch(const cwen_ctx *ctx, int type, int D, const PromptArgs &a, hipStream_t st) {
  const long long tiles = (a.total_q + 127) / 128 + a.n_seq;      // of 128 rows, at most
  // Up to 2.5 workgroups per CU (heads of 64: 4.5) the longest row sets the time, so its keys
  // go to two halves of a workgroup: heads of 128, 32/8: 2048 tokens 48 us against 56 (2560: 76 against
  // 74, 4096: 159 against 144); of 256, 24/4: 2048 73 against 101 (4096 241 against 238); of 64, 16/4: 2048
  // 26 against 36, 8192 178 against 184 (40 prompts of 125 14.4 against 11.3).
  const bool split = 2 * tiles * a.nh <= (D == 64 ? 9ll : 5ll) * ctx->ncu;
  // Sequences of 4096 tokens and more on average: workgroups of 8 waves read K and V half as often as
  // those of 4, which leave fewer waves idle in short sequences and more workgroups to a CU (heads of 128,
  // 32/8: one prompt of 4096 140 us against 144, of 32768 7.77 ms against 7.98, 9 of 1811 345 us against 297; at
  // the line the sides differ by 2 %, 4 prompts of 4096 the other way, 556 against 545; of 256, 24/4: 4096
  // 229 us against 238, 16384 2.99 ms against 3.19).  Heads of 64, 32/8, are not built so: 4096 106 us against 101,
  // 32768 4.80 ms against 5.11.
  const bool wide = !split && D != 64 && a.total_q >= 4096ll * a.n_seq;
  const int BM = wide ? 256 : 128;
  const long long items = (a.total_q + BM - 1) / BM + a.n_seq;    // items * nh fits a launch (the entry point has checked)
  return by_type(type, D, [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int dim = decltype(d)::value;
    const dim3 grid((unsigned)(items * a.nh));
    if (split) hipLaunchKernelGGL((prompt_kernel<T, dim, 4, 2, 32, 2>), grid, dim3(512), 0, st, a);
    else if (!wide) hipLaunchKernelGGL((prompt_kernel<T, dim, 4, 1, 32, dim == 256 ? 2 : 3>), grid, dim3(256), 0, st, a);
    else if constexpr (dim != 64) hipLaunchKernelGGL((prompt_kernel<T, dim, 8, 1, dim == 256 ? 32 : 64, 2>), grid, dim3(512), 0, st, a);
  });
}
int attn_tree_launch(const cwen_ctx *ctx, const TreeArgs &a, hipStream_t st) {
  const int nkv = a.kv.n_kv_head, g = a.nh / nkv, D = a.kv.head_dim;
  const long long rows = (long long)a.max_nodes * g;
  const int form = rows <= 32 ? 1 : 4;                           // row tiles of 32 of a workgroup
  const int rt = 32 * form;
  const long long room = (long long)ctx->attn_floats / ((D + 2ll) * rt * nkv * 2);   // pieces whose partials the scratch holds
  const int per_cu = form == 1 ? 256 / D : D == 64 ? 3 : 2;      // workgroups that a CU holds at once
  TreeLaunch p;
  p.extra = D == 256 ? 1 : 2;                                    // the units of 256 take twice as long
  // One piece a KV head at least: it holds whole rows and leaves no partials, so it needs no room.
  p.lines = (int)std::max(1ll, std::min((long long)per_cu * ctx->ncu / nkv, room));
  p.ml = (float2 *)ctx->attn_part;
  // Up to 96 (row, chunk) partials of a group are joined in the launch: one token of 6 heads behind 1000
  // positions 14.6 us so, 16.1 in two launches; behind 2600 17.1 and 16.0.  Of many groups one is taken
  // to hold at most twice its share of the pieces: 48 tokens of 32/8 heads behind up to 12000
  // positions 113 us and 117; with 6 nodes each (24 rows) 164 and 162.
  const long long share = 2ll * ((p.lines + a.n_seq - 1) / a.n_seq) + 1;
  const long long chunks = std::min({(long long)p.lines, share, ((long long)a.max_len + a.max_nodes + UNIT - 1) / UNIT});
  p.count = form == 1 && chunks * rows <= 96 && (long long)nkv * a.n_seq <= ctx->ncounters ? ctx->counters : nullptr;
  p.po = ctx->attn_part + (((size_t)nkv * p.lines * 2 * rt * 2 + 3) & ~(size_t)3);
  const long long tiles = (rows + rt - 1) / rt;                  // of one group at most
  p.levels = tree_levels(tiles, p.lines);
  const long long blocks = 8ll * std::max((long long)p.levels * (((long long)nkv * (p.lines / p.levels) + 7) / 8),
                                          ((long long)nkv * p.lines + 7) / 8);
  // Every line's positions fit 32 bits.
  const long long units = ((long long)a.kv.max_pages * a.kv.page + UNIT - 1) / UNIT + 1 + p.extra;
  if ((a.n_seq + 64ll) * tiles * units > INT32_MAX) return CWEN_EINVAL;
  if (blocks > INT32_MAX || (long long)a.total * a.nh > INT32_MAX) return CWEN_EINVAL;
  const dim3 grid((unsigned)blocks);
  int rc = by_type(a.kv.type, D, [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int dim = decltype(d)::value, BN = dim == 256 ? 32 : 64;
    if (form == 1) hipLaunchKernelGGL((tree_few_kernel<T, dim>), grid, dim3(256), 0, st, a, p);
    else hipLaunchKernelGGL((tree_many_kernel<T, dim, BN>), grid, dim3(256), 0, st, a, p);
  });
  if (rc || p.lines == 1 || p.count) return rc;
  // Up to 4 rows per CU: a workgroup each; past them as many heads to a workgroup as leave 2 per CU.
  const long long all = (long long)a.total * a.nh;
  int hpw = 1;
  if (all > 4ll * ctx->ncu) hpw = (int)std::min<long long>(std::min(a.nh, JOIN_HEADS), std::max(2ll, all / (2ll * ctx->ncu)));
  return by_type(a.kv.type, D, [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int dim = decltype(d)::value;
    const dim3 grid((unsigned)(a.total * ((a.nh + hpw - 1) / hpw)));
    if (hpw <= 4) hipLaunchKernelGGL((tree_join_kernel<T, dim, 64>), grid, dim3(256), 0, st, a, p, rt, hpw);
    else hipLaunchKernelGGL((tree_join_kernel<T, dim, 16>), grid, dim3(256), 0, st, a, p, rt, hpw);
  });
}
