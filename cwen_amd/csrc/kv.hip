// The paged cache's bookkeeping on the device: fork, reserve (with its copies
// of shared pages), keep (an accepted branch's rows) and truncate.
//
// All state is in device memory and every decision is taken there, so a step
// needs no host round trip and can be captured.  A free page is one with ref 0;
// pages are taken lowest id first and the counts only ever change by atomic
// adds whose order does not matter, so the result does not depend on timing.
// The bookkeeping is latency (a few dependent loads per launch); the rows that
// move are bandwidth.
#include "cwen_internal.h"
#include "kv_table.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Inclusive sum over the wave's lanes below and at this one.
__device__ __forceinline__ int scan64(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d);
    if (lane >= d) v += u;
  }
  return v;
}
// Exclusive sum over the workgroup; *total its whole sum.  red: one int per wave.
template <int N> __device__ __forceinline__ int scan_block(int v, int *red, int *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int inc = scan64(v);
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) {
    const int x = red[w];
    if (w < wave) before += x;
    all += x;
  }
  __syncthreads();
  *total = all;
  return before + inc - v;
}

__global__ __launch_bounds__(256) void kv_reset_kernel(cwen_kv kv) {
  const long long n = (long long)kv.max_seqs * kv.max_pages;
  const long long i0 = blockIdx.x * 256ll + threadIdx.x, step = gridDim.x * 256ll;
  for (long long i = i0; i < n; i += step) kv.table[i] = -1;
  for (long long i = i0; i < kv.n_pages; i += step) kv.ref[i] = 0;
  for (long long i = i0; i < kv.max_seqs; i += step) kv.len[i] = kv.held[i] = 0;
  if (i0 == 0) *kv.status = 0;
}
__global__ void kv_take_status_kernel(int *status, int *out) { *out = atomicExch(status, 0); }

// Whether seqs[i] is out of range or named again by another request (the whole
// workgroup asks; the result is uniform).
template <int N> __device__ __forceinline__ bool bad_request(const int *seqs, int i, int n, int max_seqs) {
  const int s = seqs[i];
  bool bad = (unsigned)s >= (unsigned)max_seqs;
  for (int j = threadIdx.x; j < n; j += N) bad |= j != i && seqs[j] == s;
  return __syncthreads_or(bad);
}

// Give back the pages `from` .. held - 1 of sequence s (one workgroup).
template <int N> __device__ __forceinline__ void release_from(const cwen_kv &kv, int s, int from, int held) {
  bool bad = false;
  for (int i = from + (int)threadIdx.x; i < held; i += N) {
    int *e = kv.table + (size_t)s * kv.max_pages + i;
    bool b = false;
    const int pg = kv_page_ok(*e, kv.n_pages, &b);
    if (!b) atomicSub(kv.ref + pg, 1);
    bad |= b;
    *e = -1;
  }
  if (bad) kv_raise(kv, CWEN_KV_PAGE);
}

// One workgroup per request.
__global__ __launch_bounds__(256) void kv_truncate_kernel(cwen_kv kv, const int *seqs, const int *len, int n) {
  const int i = blockIdx.x;
  if (bad_request<256>(seqs, i, n, kv.max_seqs)) {
    if (threadIdx.x == 0) kv_raise(kv, CWEN_KV_ARG);
    return;
  }
  const int s = seqs[i], to = len ? len[i] : 0, cur = kv.len[s];
  bool bad = to < 0 || to > cur;
  const int held = kv_held_ok(kv.held[s], kv.max_pages, &bad);
  __syncthreads();                               // every thread has read len and held
  if (bad) {
    if (threadIdx.x == 0) kv_raise(kv, CWEN_KV_ARG);
    return;
  }
  const int pages = kv_cover(to, kv.page);
  release_from<256>(kv, s, pages, held);
  if (threadIdx.x == 0) {
    kv.len[s] = to;
    kv.held[s] = min(pages, held);
  }
}

// One workgroup per request.
__global__ __launch_bounds__(256) void kv_fork_kernel(cwen_kv kv, const int *src, const int *dst, int n) {
  const int i = blockIdx.x, a = src[i], b = dst[i];
  bool bad = (unsigned)a >= (unsigned)kv.max_seqs || (unsigned)b >= (unsigned)kv.max_seqs || a == b;
  for (int j = threadIdx.x; j < n; j += 256) bad |= (j != i && dst[j] == b) || src[j] == b || dst[j] == a;
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) kv_raise(kv, CWEN_KV_ARG);
    return;
  }
  const int len = kv.len[a];
  bad = kv.len[b] != 0 || kv.held[b] != 0;
  const int held = kv_held_ok(kv.held[a], kv.max_pages, &bad);
  if (!kv_fits(len, 0, kv.page, held)) bad = true;   // a length past its pages
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0) kv_raise(kv, CWEN_KV_ARG);
    return;
  }
  const int pages = kv_cover(len, kv.page);
  const int *from = kv.table + (size_t)a * kv.max_pages;
  int *to = kv.table + (size_t)b * kv.max_pages;
  bool badpage = false;
  for (int k = threadIdx.x; k < pages; k += 256) {
    const int e = from[k];
    bool bp = false;
    const int pg = kv_page_ok(e, kv.n_pages, &bp);
    if (!bp) atomicAdd(kv.ref + pg, 1);
    badpage |= bp;
    to[k] = e;
  }
  if (badpage) kv_raise(kv, CWEN_KV_PAGE);
  if (threadIdx.x == 0) {
    kv.len[b] = len;
    kv.held[b] = pages;
  }
}

// The plan of a reserve: one workgroup.  work: the free pages found, then per
// request the copy to make, {old, new, rows, -} (old < 0: none).
constexpr int RES = 1024;
__global__ __launch_bounds__(RES) void kv_reserve_kernel(cwen_kv kv, const int *seqs, const int *grow, int n) {
  __shared__ int s_first[CWEN_KV_REQ_MAX + 1];     // pages taken by the requests before
  __shared__ int s_last[CWEN_KV_REQ_MAX];          // the shared page that a request would write to, or -1
  __shared__ uint32_t s_seen[65536 / 32];
  __shared__ int red[RES / 64];
  const int tid = threadIdx.x;
  int *jobs = kv.work + ((kv.n_pages + 3) & ~3);
  for (int i = tid; i < (kv.max_seqs + 31) / 32; i += RES) s_seen[i] = 0;
  __syncthreads();
  bool bad = false, badpage = false;
  for (int i = tid; i < n; i += RES) {
    const int s = seqs[i], g = grow[i];
    int need = 0, last = -1;
    if ((unsigned)s >= (unsigned)kv.max_seqs) {
      bad = true;
    } else {
      bad |= (atomicOr(&s_seen[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1;
      const int len = kv.len[s], held = kv_held_ok(kv.held[s], kv.max_pages, &bad);
      if (!kv_fits(len, g, kv.page, kv.max_pages) || !kv_fits(len, 0, kv.page, held)) {
        bad = true;
      } else {
        need = max(kv_cover(len + g, kv.page) - held, 0);
        if (g > 0 && len % kv.page) {
          const int pg = kv_page_ok(kv.table[(size_t)s * kv.max_pages + len / kv.page], kv.n_pages, &badpage);
          if (kv.ref[pg] > 1) last = pg;
        }
      }
    }
    s_first[i] = need;
    s_last[i] = last;
  }
  if (__syncthreads_or(bad | badpage)) {
    for (int i = tid; i < n; i += RES) jobs[4 * i] = -1;
    if (bad) kv_raise(kv, CWEN_KV_ARG);
    if (badpage) kv_raise(kv, CWEN_KV_PAGE);
    return;
  }
  // Of the requests that share a page each but the last holder copies it.
  for (int i = tid; i < n; i += RES) {
    const int last = s_last[i];
    int copy = 0;
    if (last >= 0) {
      int earlier = 0;
      for (int j = 0; j < i; ++j) earlier += s_last[j] == last;
      copy = kv.ref[last] - earlier > 1;
    }
    jobs[4 * i] = copy ? last : -1;
    s_first[i] += copy;                            // own entry only; s_last stays for the others
  }
  __syncthreads();
  // Exclusive sums, each thread a run of requests.
  const int run = (n + RES - 1) / RES, r0 = min(tid * run, n), r1 = min(r0 + run, n);
  int mine = 0, total;
  for (int i = r0; i < r1; ++i) mine += s_first[i];
  int at = scan_block<RES>(mine, red, &total);
  for (int i = r0; i < r1; ++i) {
    const int need = s_first[i];
    s_first[i] = at;
    at += need;
  }
  if (tid == 0) s_first[n] = total;
  __syncthreads();
  // The `total` lowest free pages.
  int found = 0;
  for (int p0 = 0; p0 < kv.n_pages && found < total; p0 += 4 * RES) {
    const int p = p0 + 4 * tid;
    int f[4], m = 0;
    if (p + 3 < kv.n_pages) {
      const int4 r = *(const int4 *)(kv.ref + p);
      f[0] = r.x == 0; f[1] = r.y == 0; f[2] = r.z == 0; f[3] = r.w == 0;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = p + j < kv.n_pages && kv.ref[p + j] == 0;
    }
    m = f[0] + f[1] + f[2] + f[3];
    int all, o = found + scan_block<RES>(m, red, &all);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (f[j]) {
        if (o < total) kv.work[o] = p + j;
        ++o;
      }
    found += all;
  }
  __syncthreads();
  if (found < total) {
    for (int i = tid; i < n; i += RES) jobs[4 * i] = -1;
    if (tid == 0) kv_raise(kv, CWEN_KV_FULL);
    return;
  }
  // Page f of the list belongs to the last request whose first page is <= f
  // among those that take any: found by bisection.
  for (int f = tid; f < total; f += RES) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_first[mid] <= f) lo = mid;
      else hi = mid - 1;
    }
    const int i = lo, k = f - s_first[i], pg = kv.work[f], s = seqs[i], old = jobs[4 * i];
    int *row = kv.table + (size_t)s * kv.max_pages;
    kv.ref[pg] = 1;
    if (old >= 0 && k == 0) {
      row[kv.len[s] / kv.page] = pg;
      jobs[4 * i + 1] = pg;
      jobs[4 * i + 2] = kv.len[s] % kv.page;
      atomicSub(kv.ref + old, 1);
    } else {
      row[kv.held[s] + k - (old >= 0)] = pg;
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += RES) kv.held[seqs[i]] += s_first[i + 1] - s_first[i] - (jobs[4 * i] >= 0);
}

// The filled rows of the shared pages that a reserve replaced.  Grid (requests,
// layers, k and v); a head's rows are contiguous in both pages.
__global__ __launch_bounds__(256) void kv_copy_kernel(cwen_kv kv) {
  const int *job = kv.work + ((kv.n_pages + 3) & ~3) + 4 * blockIdx.x;
  const int old = job[0];
  if (old < 0) return;
  const int pg = job[1], n16 = job[2] * kv.head_dim / 8;    // 16-byte pieces of one head
  uint16_t *pool = (uint16_t *)(blockIdx.z ? kv.v : kv.k);
  const uint16_t *a = pool + kv_at(blockIdx.y, old, 0, 0, kv.n_pages, kv.n_kv_head, kv.page, kv.head_dim);
  uint16_t *b = pool + kv_at(blockIdx.y, pg, 0, 0, kv.n_pages, kv.n_kv_head, kv.page, kv.head_dim);
  for (int h = 0; h < kv.n_kv_head; ++h)
    for (int i = threadIdx.x; i < n16; i += 256) {
      const size_t o = (size_t)h * kv.page * kv.head_dim + 8 * (size_t)i;
      *(u32x4_t *)(b + o) = *(const u32x4_t *)(a + o);
    }
}

// Whether request i of a keep can be met (workgroup-uniform).  len and held
// are the sequence's.
template <int N>
__device__ __forceinline__ bool keep_ok(const cwen_kv &kv, const int *seqs, const int *count, const int *path, int ps, int i,
                                        int n, int *len, int *held) {
  if (bad_request<N>(seqs, i, n, kv.max_seqs)) return false;
  const int s = seqs[i], c = count[i];
  bool bad = false;
  *len = kv.len[s];
  *held = kv_held_ok(kv.held[s], kv.max_pages, &bad);
  bad |= !kv_fits(*len, c, kv.page, *held) || (path && c > ps);
  if (path && !bad) {
    const int *row = path + (size_t)i * ps;
    for (int j = threadIdx.x; j < c; j += N) {
      const int r = row[j], before = j ? row[j - 1] : -1;
      bad |= r <= before || !kv_fits(*len, r, kv.page, *held) || *len + r >= *held * kv.page;
      if (!bad && r != j) {                         // a row that moves: into pages held alone
        bool bp = false;
        const int pg = kv_page_ok(kv.table[(size_t)s * kv.max_pages + (*len + j) / kv.page], kv.n_pages, &bp);
        bad |= bp || kv.ref[pg] != 1;
      }
    }
  }
  return !__syncthreads_or(bad);
}

// The rows of an accepted branch.  Grid (requests, layers, k and v).  A thread
// owns 16 bytes of the row (all heads side by side) and takes the branch's rows in
// order, KEEP at a time: a destination never lies behind a later source, so
// nothing is overwritten before it is read, and no thread depends on another.
constexpr int KEEP = 8;
__global__ __launch_bounds__(256) void kv_keep_kernel(cwen_kv kv, const int *seqs, const int *count, const int *path, int ps,
                                                      int n) {
  const int i = blockIdx.x;
  int len, held;
  if (!keep_ok<256>(kv, seqs, count, path, ps, i, n, &len, &held)) return;   // kv_keep_end_kernel raises the flag
  const int c = count[i], *row = path + (size_t)i * ps;
  const int *tab = kv.table + (size_t)seqs[i] * kv.max_pages;
  uint16_t *pool = (uint16_t *)(blockIdx.z ? kv.v : kv.k);
  const int per = kv.head_dim / 8;                 // 16-byte pieces of one head's row
  auto at = [&](int pos, int h, int d) {
    bool bad = false;
    const int pg = kv_page_ok(tab[pos / kv.page], kv.n_pages, &bad);
    return kv_at(blockIdx.y, pg, h, pos % kv.page, kv.n_pages, kv.n_kv_head, kv.page, kv.head_dim) + 8 * d;
  };
  for (int x = threadIdx.x; x < per * kv.n_kv_head; x += 256) {
    const int h = x / per, d = x - h * per;
    for (int j0 = 0; j0 < c; j0 += KEEP) {
      u32x4_t v[KEEP];
#pragma unroll
      for (int u = 0; u < KEEP; ++u)
        if (j0 + u < c) v[u] = *(const u32x4_t *)(pool + at(len + row[j0 + u], h, d));
#pragma unroll
      for (int u = 0; u < KEEP; ++u)
        if (j0 + u < c) *(u32x4_t *)(pool + at(len + j0 + u, h, d)) = v[u];
    }
  }
}
// The new lengths, and the pages behind them given back.
__global__ __launch_bounds__(256) void kv_keep_end_kernel(cwen_kv kv, const int *seqs, const int *count, const int *path,
                                                          int ps, int n) {
  const int i = blockIdx.x;
  int len, held;
  if (!keep_ok<256>(kv, seqs, count, path, ps, i, n, &len, &held)) {
    if (threadIdx.x == 0) kv_raise(kv, CWEN_KV_ARG);
    return;
  }
  const int s = seqs[i], pages = kv_cover(len + count[i], kv.page);
  release_from<256>(kv, s, pages, held);
  if (threadIdx.x == 0) {
    kv.len[s] = len + count[i];
    kv.held[s] = pages;
  }
}

}  // namespace

int kv_reset_launch(const cwen_kv &kv, hipStream_t st) {
  hipLaunchKernelGGL(kv_reset_kernel, dim3(256), dim3(256), 0, st, kv);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
int kv_take_status_launch(const cwen_kv &kv, int *out, hipStream_t st) {
  hipLaunchKernelGGL(kv_take_status_kernel, dim3(1), dim3(1), 0, st, kv.status, out);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
int kv_reserve_launch(const cwen_kv &kv, const int *seqs, const int *n, int n_req, hipStream_t st) {
  hipLaunchKernelGGL(kv_reserve_kernel, dim3(1), dim3(RES), 0, st, kv, seqs, n, n_req);
  CWEN_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(kv_copy_kernel, dim3(n_req, kv.n_layers, 2), dim3(256), 0, st, kv);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
int kv_fork_launch(const cwen_kv &kv, const int *src, const int *dst, int n_req, hipStream_t st) {
  hipLaunchKernelGGL(kv_fork_kernel, dim3(n_req), dim3(256), 0, st, kv, src, dst, n_req);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
int kv_keep_launch(const cwen_kv &kv, const int *seqs, const int *count, const int *path, int ps, int n_req,
                   hipStream_t st) {
  if (path) {
    hipLaunchKernelGGL(kv_keep_kernel, dim3(n_req, kv.n_layers, 2), dim3(256), 0, st, kv, seqs, count, path, ps, n_req);
    CWEN_HIP_TRY(hipGetLastError());
  }
  hipLaunchKernelGGL(kv_keep_end_kernel, dim3(n_req), dim3(256), 0, st, kv, seqs, count, path, ps, n_req);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
int kv_truncate_launch(const cwen_kv &kv, const int *seqs, const int *len, int n_req, hipStream_t st) {
  hipLaunchKernelGGL(kv_truncate_kernel, dim3(n_req), dim3(256), 0, st, kv, seqs, len, n_req);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
