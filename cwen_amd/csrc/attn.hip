// Attention of packed prompts and of drafted trees over the paged cache.
#include <math.h>
#include "cwen_internal.h"
#include "kv_table.h"
#include "attn_core.h"

namespace {

// ---- one wave per (token, head), the plain loop over its keys ----
// Lane l holds dims E l .. of the query, of each key and of the output, E = D /
// 64; the running maximum and sum of the softmax in f32.
template <typename T, int D, typename SEES, typename ROWS>
__device__ __forceinline__ void row_plain(const typename T::elem *q, typename T::elem *o, float *lse, int n, float scale,
                                          SEES sees, ROWS rows) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  float x[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = (float)q[lane * E + e];
    acc[e] = 0.f;
  }
  for (int j = 0; j < n; ++j) {
    if (!sees(j)) continue;
    const typename T::elem *k, *v;
    rows(j, &k, &v);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(x[e], (float)k[lane * E + e], s);
    s = sum64(s) * scale;
    const float mn = fmaxf(m, s), a = m == mn ? 1.f : expf(m - mn), p = expf(s - mn);
    l = fmaf(l, a, p);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], a, p * (float)v[lane * E + e]);
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) o[lane * E + e] = (typename T::elem)(l == 0.f ? 0.f : acc[e] / l);
  if (lse && lane == 0) *lse = l == 0.f ? -INFINITY : m + logf(l);
}

template <typename T, int D> __global__ __launch_bounds__(256) void tree_plain_kernel(TreeArgs a) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y, g = a.nh / a.kv.n_kv_head;
  if (t >= a.total) return;
  int s = 0;
  while (s < a.n_seq && !(a.cu[s] <= t && t < a.cu[s + 1])) ++s;
  if (s == a.n_seq) return;
  const int c0 = max(a.cu[s], 0), i = t - c0, nodes = min(min(a.cu[s + 1], a.total) - c0, a.max_nodes), id = a.seqs[s];
  if (i >= nodes) return;
  bool bad = (unsigned)id >= (unsigned)a.kv.max_seqs;
  const int sid = bad ? 0 : id;
  const int len = a.kv.len[sid];
  const int n = bad ? 0 : kv_readable(len, nodes, a.kv.held[sid], a.kv.page, a.kv.max_pages, &bad);
  const int *tab = a.kv.table + (size_t)sid * a.kv.max_pages;
  const unsigned long long *mask = a.mask ? a.mask + (size_t)t * a.mw : nullptr;
  row_plain<T, D>((const typename T::elem *)a.q + (long long)t * a.qs + h * D,
                  (typename T::elem *)a.o + (long long)t * a.os + h * D, a.lse ? a.lse + (long long)t * a.nh + h : nullptr, n,
                  a.scale,
                  [&](int j) {
                    const int u = j - len;
                    return u < 0 || (mask ? (mask[u >> 6] >> (u & 63)) & 1 : u <= i);
                  },
                  [&](int j, const typename T::elem **k, const typename T::elem **v) {
                    const int pg = kv_page_ok(tab[j / a.kv.page], a.kv.n_pages, &bad);
                    const int64_t at = kv_at(a.layer, pg, h / g, j % a.kv.page, a.kv.n_pages, a.kv.n_kv_head, a.kv.page, D);
                    *k = (const typename T::elem *)a.kv.k + at;
                    *v = (const typename T::elem *)a.kv.v + at;
                  });
  if (bad) kv_raise(a.kv, CWEN_KV_PAGE);
}

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

template <typename T, int D, int NW, int BN> __global__ __launch_bounds__(64 * NW, 2) void prompt_kernel(PromptArgs a) {
  typedef typename T::elem elem;
  constexpr int BM = 32 * NW;
  __shared__ __align__(1024) elem K0[BN * D], K1[BN * D], V0[BN * D], V1[BN * D];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = a.nh / a.nkv;
  // Blocks of one kv head go to one or two XCDs (block b runs on XCD b % 8), long rows first.
  const int hh = blockIdx.x % a.nh, h = (hh % a.nkv) * g + hh / a.nkv, hkv = hh % a.nkv;
  const int items = gridDim.x / a.nh;
  const Item item = find_item<BM>(a.cu_q, a.n_seq, a.total_q, items - 1 - (int)(blockIdx.x / a.nh));
  if (item.seq < 0) return;
  int q0, k0;
  const int nq = span(a.cu_q, item.seq, a.total_q, &q0), nk = span(a.cu_k, item.seq, a.total_k, &k0), off = nk - nq;
  const int w0 = item.tile * BM + wave * 32, n = lane & 31;
  const int row = w0 + n;                                        // this lane's query of the sequence
  const bool live = row < nq;
  const int limit = live ? row + off : -1;                       // its last key
  AttnWave<T, D, BN> w;
  w.start(live ? (const elem *)a.q + (long long)(q0 + row) * a.qs + h * D : nullptr);
  const elem *kp = (const elem *)a.k + (long long)k0 * a.ks + hkv * D, *vp = (const elem *)a.v + (long long)k0 * a.vs + hkv * D;
  const int kend = min(min(item.tile * BM + BM, nq) + off, nk);  // keys that the workgroup's rows see
  const int wend = min(min(w0 + 32, nq) + off, nk);              // and this wave's
  const float c = a.scale * 1.44269504088896340736f;
  auto land = [&](elem *Kd, elem *Vd, int t0) __attribute__((always_inline)) {
    land_rows<D, BN, false, NW>(Kd, wave, [&](int r) { return kp + min(t0 + r, nk - 1) * a.ks; });
    land_rows<D, BN, true, NW>(Vd, wave, [&](int r) { return vp + min(t0 + r, nk - 1) * a.vs; });
  };
  auto ready = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    asm volatile("" ::: "memory");
  };
  // Tiles that every row sees whole come first, two per turn; what is left has
  // its keys compared with each row's last.
  const int full = max(min(item.tile * BM + off + 1, nk), 0) / (2 * BN) * (2 * BN);
  if (kend > 0) land(K0, V0, 0);
  int t0 = 0;
  for (; t0 < full; t0 += 2 * BN) {
    ready();
    land(K1, V1, t0 + BN);
    w.template tile<false>(K0, V0, c, [](int) { return false; });
    ready();
    if (t0 + 2 * BN < kend) land(K0, V0, t0 + 2 * BN);
    w.template tile<false>(K1, V1, c, [](int) { return false; });
  }
  for (; t0 < kend; t0 += 2 * BN) {
    ready();
    if (t0 + BN < kend) land(K1, V1, t0 + BN);
    if (t0 < wend) w.template tile<true>(K0, V0, c, [&](int j) { return t0 + j > limit; });
    if (t0 + BN >= kend) break;
    ready();
    if (t0 + 2 * BN < kend) land(K0, V0, t0 + 2 * BN);
    if (t0 + BN < wend) w.template tile<true>(K1, V1, c, [&](int j) { return t0 + BN + j > limit; });
  }
  const float l = w.sum();
  elem *orow = (elem *)a.o + (long long)(q0 + row) * a.os + h * D;
  if (__any(w.odd != w.odd)) {   // a hidden value may have leaked: these rows one by one
    for (int i = 0; i < 32 && w0 + i < nq; ++i)
      row_plain<T, D>((const elem *)a.q + (long long)(q0 + w0 + i) * a.qs + h * D, (elem *)a.o + (long long)(q0 + w0 + i) * a.os + h * D,
                      a.lse ? a.lse + (long long)(q0 + w0 + i) * a.nh + h : nullptr, min(nk, w0 + i + off + 1), a.scale,
                      [](int) { return true; },
                      [&](int j, const elem **k, const elem **v) {
                        *k = kp + j * a.ks;
                        *v = vp + j * a.vs;
                      });
    return;
  }
  if (!live) return;
  const float inv = limit < 0 ? 0.f : 1.f / l;
#pragma unroll
  for (int b = 0; b < D / 32; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      typename AttnOps<T>::vec4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (elem)(limit < 0 ? 0.f : w.o[b][4 * i + j] * inv);
      *(typename AttnOps<T>::vec4 *)(orow + 32 * b + 8 * i + 4 * (lane >> 5)) = v;
    }
  if (a.lse && lane < 32)
    a.lse[(long long)(q0 + row) * a.nh + h] = limit < 0 ? -INFINITY : 0.69314718055994530942f * (w.m + __builtin_amdgcn_logf(l));
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
  constexpr int NW = 8;
  const long long items = (a.total_q + 32 * NW - 1) / (32 * NW) + a.n_seq;
  if (items * a.nh > INT32_MAX) return CWEN_EINVAL;
  return by_type(type, D, [&](auto t, auto d) {
    constexpr int dim = decltype(d)::value;
    hipLaunchKernelGGL((prompt_kernel<decltype(t), dim, NW, dim == 256 ? 32 : 64>), dim3((unsigned)(items * a.nh)),
                       dim3(64 * NW), 0, st, a);
  });
}
int attn_tree_launch(const cwen_ctx *, const TreeArgs &a, hipStream_t st) {
  return by_type(a.kv.type, a.kv.head_dim, [&](auto t, auto d) {
    hipLaunchKernelGGL((tree_plain_kernel<decltype(t), decltype(d)::value>), dim3((a.total + 3) / 4, a.nh), dim3(256), 0, st,
                       a);
  });
}
