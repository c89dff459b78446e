// The paged cache's bookkeeping on the device: fork, reserve (with its copies
// of shared pages), keep (an accepted branch's rows) and truncate.
//
// All state is in device memory and every decision is taken there, so a step
// needs no host round trip and can be captured.  A free page is one with ref 0;
// pages are taken lowest id first and the counts only ever change by atomic
// adds whose order does not matter, so the result does not depend on timing.
// The bookkeeping is latency: a launch is a chain of dependent loads of 0.5 to 1 us
// each (truncate and fork 2.1 to 4.4 us, reserve 8 to 9 in pools of up to some 20000 pages: it
// looks for free ones from page 0, 4096 a round, so that behind 200000 held pages it takes 40 us
// more and behind 1000000 220).  The rows that move are
// bandwidth behind such a chain: 64 children, 16 layers, 44 MB of shared pages copied in
// 11.1 us and 36 MB of kept rows in 13.8 (read and written).
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
  const int s = seqs[i], to = len ? len[i] : 0;
  bool bad = false;
  const int held = kv_held_ok(kv.held[s], kv.max_pages, &bad), pages = kv_cut(to, kv.len[s], held, kv.page);
  __syncthreads();                               // every thread has read len and held
  if (bad || pages < 0) {
    if (threadIdx.x == 0) kv_raise(kv, CWEN_KV_ARG);
    return;
  }
  release_from<256>(kv, s, pages, held);
  if (threadIdx.x == 0) {
    kv.len[s] = to;
    kv.held[s] = pages;
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

// The filled rows of a shared page that a reserve replaced, in the slices l0 .. l1 - 1 (slice
// 2 l: layer l's keys, 2 l + 1: its values), by the workgroup's N threads; a head's
// rows are contiguous in both pages.  job: {old, new, rows, -} (old < 0: none).
template <int N> __device__ __forceinline__ void copy_page(const cwen_kv &kv, const int *job, int l0, int l1) {
  const int old = job[0];
  if (old < 0) return;
  const int pg = job[1], n16 = job[2] * kv.head_dim / 8;    // 16-byte pieces of one head
  const int slice = n16 * kv.n_kv_head;
  for (int x = threadIdx.x; x < slice * (l1 - l0); x += N) {
    const int l = l0 + x / slice, y = x % slice, h = y / n16;
    uint16_t *pool = (uint16_t *)(l & 1 ? kv.v : kv.k);
    const size_t o = (size_t)h * kv.page * kv.head_dim + 8 * (size_t)(y - h * n16);
    *(u32x4_t *)(pool + kv_at(l >> 1, pg, 0, 0, kv.n_pages, kv.n_kv_head, kv.page, kv.head_dim) + o) =
        *(const u32x4_t *)(pool + kv_at(l >> 1, old, 0, 0, kv.n_pages, kv.n_kv_head, kv.page, kv.head_dim) + o);
  }
}

// The plan of a reserve: one workgroup.  work: the free pages found, then per
// request the copy to make, {old, new, rows, -} (old < 0: none).
// With `copy` it makes the copies too (few and small ones: a launch saved).
constexpr int RES = 1024;
__global__ __launch_bounds__(RES) void kv_reserve_kernel(cwen_kv kv, const int *seqs, const int *grow, int n, int copy) {
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
  if (copy)
    for (int i = 0; i < n; ++i) copy_page<RES>(kv, jobs + 4 * i, 0, 2 * kv.n_layers);
}
// Grid (requests, slices).
__global__ __launch_bounds__(256) void kv_copy_kernel(cwen_kv kv) {
  copy_page<256>(kv, kv.work + ((kv.n_pages + 3) & ~3) + 4 * blockIdx.x, blockIdx.y, blockIdx.y + 1);
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
        const int *tab = kv.table + (size_t)s * kv.max_pages;
        const int pg = kv_page_ok(tab[(*len + j) / kv.page], kv.n_pages, &bp);
        kv_page_ok(tab[(*len + r) / kv.page], kv.n_pages, &bp);
        bad |= bp || kv.ref[pg] != 1;
      }
    }
  }
  return !__syncthreads_or(bad);
}

// The rows of an accepted branch, layers l0 .. l1 - 1.  Those that stay where they
// are come first (the path increases), and only the others are touched: 256 of them
// at a time have their places worked out in LDS, then a thread owns 16 bytes of the row (k
// and v, all heads side by side) and takes the rows in order, KEEP at a time.  A
// destination never lies behind a later source, so nothing is overwritten before
// it is read, and no thread depends on another.  With every place looked up by
// every thread, and every row moved, 64 branches of 32 rows in 16 layers took 44 us.
constexpr int KEEP = 8;
__device__ __forceinline__ void keep_rows(const cwen_kv &kv, int s, int len, int c, const int *row, int l0, int l1) {
  __shared__ long long s_src[256], s_dst[256];
  const int *tab = kv.table + (size_t)s * kv.max_pages;
  const int tid = threadIdx.x, per = kv.head_dim / 8, pieces = per * kv.n_kv_head;
  int first = 0;
  for (int j0 = 0; j0 < c; j0 += 256) first += __syncthreads_count(j0 + tid < c && row[j0 + tid] == j0 + tid);
  auto at = [&](int pos) {
    bool bad = false;
    const int pg = kv_page_ok(tab[pos / kv.page], kv.n_pages, &bad);
    return kv_at(0, pg, 0, pos % kv.page, kv.n_pages, kv.n_kv_head, kv.page, kv.head_dim);
  };
  const long long layer = (long long)kv.n_pages * kv.n_kv_head * kv.page * kv.head_dim;
  for (int j0 = first; j0 < c; j0 += 256) {
    const int n = min(256, c - j0);
    if (tid < n) {
      s_src[tid] = at(len + row[j0 + tid]);
      s_dst[tid] = at(len + j0 + tid);
    }
    __syncthreads();
    for (int x = tid; x < 2 * pieces * (l1 - l0); x += 256) {
      const int l = l0 + x / (2 * pieces), y = x % (2 * pieces), v = y >= pieces, z = y - v * pieces, h = z / per;
      uint16_t *pool = (uint16_t *)(v ? kv.v : kv.k) + l * layer + (long long)h * kv.page * kv.head_dim + 8 * (z - h * per);
      for (int u0 = 0; u0 < n; u0 += KEEP) {
        u32x4_t val[KEEP];
#pragma unroll
        for (int u = 0; u < KEEP; ++u) val[u] = *(const u32x4_t *)(pool + s_src[min(u0 + u, n - 1)]);
#pragma unroll
        for (int u = 0; u < KEEP; ++u)
          if (u0 + u < n) *(u32x4_t *)(pool + s_dst[u0 + u]) = val[u];
      }
    }
    __syncthreads();
  }
}
// Grid (requests, layers).
__global__ __launch_bounds__(256) void kv_keep_kernel(cwen_kv kv, const int *seqs, const int *count, const int *path, int ps,
                                                      int n) {
  const int i = blockIdx.x;
  int len, held;
  if (!keep_ok<256>(kv, seqs, count, path, ps, i, n, &len, &held)) return;   // kv_keep_end_kernel raises the flag
  keep_rows(kv, seqs[i], len, count[i], path + (size_t)i * ps, blockIdx.y, blockIdx.y + 1);
}
// The new lengths, and the pages behind them given back; with `rows` (few layers
// and requests: a launch saved) the rows first.  Grid: requests.
__global__ __launch_bounds__(256) void kv_keep_end_kernel(cwen_kv kv, const int *seqs, const int *count, const int *path,
                                                          int ps, int n, int rows) {
  const int i = blockIdx.x;
  int len, held;
  if (!keep_ok<256>(kv, seqs, count, path, ps, i, n, &len, &held)) {
    if (threadIdx.x == 0) kv_raise(kv, CWEN_KV_ARG);
    return;
  }
  const int s = seqs[i], c = count[i], pages = kv_cover(len + c, kv.page);
  if (rows) keep_rows(kv, s, len, c, path + (size_t)i * ps, 0, kv.n_layers);
  release_from<256>(kv, s, pages, held);
  if (threadIdx.x == 0) {
    kv.len[s] = len + c;
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
// Whether one workgroup per request moves a request's rows of every layer in about the time of a launch.
static bool few_rows(const cwen_kv &kv, int n_req, int rows) {
  return (long long)n_req * kv.n_layers * rows * kv.n_kv_head * kv.head_dim <= 1 << 17;
}
int kv_reserve_launch(const cwen_kv &kv, const int *seqs, const int *n, int n_req, hipStream_t st) {
  const bool few = few_rows(kv, n_req, kv.page);
  hipLaunchKernelGGL(kv_reserve_kernel, dim3(1), dim3(RES), 0, st, kv, seqs, n, n_req, (int)few);
  CWEN_HIP_TRY(hipGetLastError());
  if (few) return CWEN_OK;
  hipLaunchKernelGGL(kv_copy_kernel, dim3(n_req, 2 * kv.n_layers), dim3(256), 0, st, kv);
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
  const bool few = path && few_rows(kv, 1, ps);
  if (path && !few) {
    hipLaunchKernelGGL(kv_keep_kernel, dim3(n_req, kv.n_layers), dim3(256), 0, st, kv, seqs, count, path, ps, n_req);
    CWEN_HIP_TRY(hipGetLastError());
  }
  hipLaunchKernelGGL(kv_keep_end_kernel, dim3(n_req), dim3(256), 0, st, kv, seqs, count, path, ps, n_req, (int)few);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
int kv_truncate_launch(const cwen_kv &kv, const int *seqs, const int *len, int n_req, hipStream_t st) {
  hipLaunchKernelGGL(kv_truncate_kernel, dim3(n_req), dim3(256), 0, st, kv, seqs, len, n_req);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
