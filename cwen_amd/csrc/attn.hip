// Attention of packed prompts and of drafted trees over the paged cache.
#include <math.h>
#include "cwen_internal.h"
#include "kv_table.h"

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

template <typename T, int D> __global__ __launch_bounds__(256) void prompt_plain_kernel(PromptArgs a) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y, g = a.nh / a.nkv;
  if (t >= a.total_q) return;
  int s = 0;
  while (s < a.n_seq && !(a.cu_q[s] <= t && t < a.cu_q[s + 1])) ++s;
  if (s == a.n_seq) return;
  const int q0 = max(a.cu_q[s], 0), q1 = min(a.cu_q[s + 1], a.total_q);
  const int k0 = max(a.cu_k[s], 0), k1 = min(a.cu_k[s + 1], a.total_k), nk = max(k1 - k0, 0);
  const typename T::elem *K = (const typename T::elem *)a.k + (long long)k0 * a.ks + (h / g) * D;
  const typename T::elem *V = (const typename T::elem *)a.v + (long long)k0 * a.vs + (h / g) * D;
  const int n = min(nk, t - q0 + nk - (q1 - q0) + 1);
  row_plain<T, D>((const typename T::elem *)a.q + (long long)t * a.qs + h * D,
                  (typename T::elem *)a.o + (long long)t * a.os + h * D, a.lse ? a.lse + (long long)t * a.nh + h : nullptr, n,
                  a.scale, [](int) { return true; },
                  [&](int j, const typename T::elem **k, const typename T::elem **v) {
                    *k = K + j * a.ks;
                    *v = V + j * a.vs;
                  });
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
  return by_type(type, D, [&](auto t, auto d) {
    hipLaunchKernelGGL((prompt_plain_kernel<decltype(t), decltype(d)::value>), dim3((a.total_q + 3) / 4, a.nh), dim3(256), 0,
                       st, a);
  });
}
int attn_tree_launch(const cwen_ctx *, const TreeArgs &a, hipStream_t st) {
  return by_type(a.kv.type, a.kv.head_dim, [&](auto t, auto d) {
    hipLaunchKernelGGL((tree_plain_kernel<decltype(t), decltype(d)::value>), dim3((a.total + 3) / 4, a.nh), dim3(256), 0, st,
                       a);
  });
}
