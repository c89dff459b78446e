// Log probabilities of given tokens, their ranks, entropies and the largest
// logits, in one pass over the logits.
//
// A thread keeps m, s = sum e^(x - m) and t = sum e^(x - m) (x - m) of its
// logits; then lse = m + ln s and the entropy is ln s - t / s.  The reference m
// is renewed only when a logit outgrows it by more than LAG: s stays below
// e^LAG times the number of logits.
//
// A wave keeps the 64 largest logits seen, one a lane, sorted by value and then
// by index.  A logit that comes before the last of the wanted ones goes into a
// queue in LDS; when 64 wait there they are sorted and merged into the list, so
// that few logits cost more than a comparison.
#include <math.h>
#include <algorithm>
#include "cwen_internal.h"

namespace {

constexpr int THREADS = 256, WAVES = 4, LIST = CWEN_LOGPROBS_TOP, SPLITS = 64;
constexpr float LAG = 8.f, LOG2E = 1.44269504088896340736f;
constexpr int NONE = 0x7fffffff;            // index of a list entry that is none

// ---- sums
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }
// With another reference, not below the present one.
__device__ __forceinline__ void renew(Sums &a, float m) {
  const float d = a.m == -INFINITY ? 0.f : a.m - m, e = a.m == -INFINITY ? 0.f : exp_of(d);
  a.t = e * fmaf(a.s, fmaxf(d, -200.f), a.t);     // e is 0 there, and the product must not be infinite
  a.s *= e;
  a.m = m;
}
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  if (m != -INFINITY) {
    renew(a, m);
    renew(b, m);
  }
  return {m, a.s + b.s, a.t + b.t};
}

// ---- lists: one entry a lane
struct Entry {
  float v;
  int i;
};
__device__ __forceinline__ bool before(Entry a, Entry b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
__device__ __forceinline__ Entry of_lane(Entry a, int l) { return {__shfl(a.v, l), __shfl(a.i, l)}; }
// The bitonic step between lanes x apart; down: the lower lane keeps the entry that comes first.
__device__ __forceinline__ Entry step(Entry a, int x, bool down) {
  const int lane = threadIdx.x & 63;
  const Entry b = {__shfl_xor(a.v, x), __shfl_xor(a.i, x)};
  const bool first = ((lane & x) == 0) == down;
  return before(b, a) == first ? b : a;
}
__device__ __forceinline__ Entry sorted(Entry a) {
  const int lane = threadIdx.x & 63;
  for (int k = 2; k <= 64; k *= 2)
    for (int x = k / 2; x > 0; x /= 2) a = step(a, x, (lane & k) == 0);
  return a;
}
// The 64 first of two sorted lists.
__device__ __forceinline__ Entry merged(Entry a, Entry b) {
  b = of_lane(b, 63 - (threadIdx.x & 63));
  a = before(b, a) ? b : a;
  for (int x = 32; x > 0; x /= 2) a = step(a, x, true);
  return a;
}

struct Best {
  Entry mine, last;         // this lane's entry; the last one wanted
  float *qv;                // the wave's queue
  int *qi;
  int n, top;               // entries waiting, entries wanted
  __device__ __forceinline__ void start(float *v, int *i, int wanted) {
    mine = last = {-INFINITY, NONE};
    qv = v;
    qi = i;
    n = 0;
    top = wanted;
  }
  __device__ __forceinline__ static void settle() {     // the wave's LDS writes are done
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  __device__ __forceinline__ void flush() {
    const int lane = threadIdx.x & 63;
    settle();
    const Entry a = lane < n ? Entry{qv[lane], qi[lane]} : Entry{-INFINITY, NONE};
    const Entry rest = 64 + lane < n ? Entry{qv[64 + lane], qi[64 + lane]} : Entry{-INFINITY, NONE};
    mine = merged(mine, sorted(a));
    last = of_lane(mine, top - 1);
    settle();
    qv[lane] = rest.v;
    qi[lane] = rest.i;
    n = max(n - 64, 0);
  }
  __device__ __forceinline__ void offer(float v, int i) {
    const bool in = before({v, i}, last);
    const unsigned long long who = __ballot(in);
    if (!who) return;
    if (in) {
      const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
      qv[at] = v;
      qi[at] = i;
    }
    n += __builtin_popcountll(who);
    if (n >= 64) flush();
  }
};

// Words of one part's result: m, s, t, count, then the list.
__host__ __device__ constexpr int part_words(int top) { return 4 + 2 * ((top + 1) & ~1); }

struct Split {
  int n;              // parts of a row
  int vecs;           // 16-byte pieces of a part
};

__device__ __forceinline__ void finish(const LogprobArgs &a, int row, Sums r, int before_it, float xt, Entry e) {
  const int lane = threadIdx.x & 63;
  const float ls = (float)log((double)r.s);
  if (lane == 0) {
    const int tok = a.tokens ? a.tokens[row] : -1;
    const bool there = tok >= 0 && tok < a.V && xt == xt;
    if (a.lse) a.lse[row] = r.m == -INFINITY && r.s == 0.f ? -INFINITY : (float)((double)r.m + log((double)r.s));
    if (a.entropy) a.entropy[row] = r.m == -INFINITY ? NAN : (float)(log((double)r.s) - (double)r.t / (double)r.s);
    if (a.logprob) a.logprob[row] = there ? (xt - r.m) - ls : NAN;
    if (a.rank) a.rank[row] = there ? before_it : -1;
  }
  if (lane < a.top) {
    if (a.top_ids) a.top_ids[(long long)row * a.top + lane] = e.i == NONE ? -1 : e.i;
    if (a.top_lp) a.top_lp[(long long)row * a.top + lane] = e.i == NONE ? -INFINITY : (e.v - r.m) - ls;
  }
}

template <typename T> __device__ __forceinline__ float token_logit(const LogprobArgs &a, int row) {
  const int tok = a.tokens ? a.tokens[row] : -1;
  return tok >= 0 && tok < a.V ? (float)((const T *)a.x)[row * a.ls + tok] : NAN;
}

template <typename T> __global__ __launch_bounds__(THREADS) void part_kernel(LogprobArgs a, Split sp) {
  constexpr int E = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
  __shared__ float s_qv[WAVES][128], s_sums[WAVES][3];
  __shared__ int s_qi[WAVES][128], s_cnt[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x / sp.n, part = blockIdx.x - row * sp.n;
  const T *x = (const T *)a.x + row * a.ls;
  // Whole 16-byte pieces lie behind `head` logits; the first part takes those too, the last one the row's end.
  const int head = min((int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T), a.V), nvec = (a.V - head) / E;
  const int tok = a.rank && a.tokens ? a.tokens[row] : -1;
  const float xt = a.rank ? token_logit<T>(a, row) : NAN;
  Sums r = {-INFINITY, 0.f, 0.f};
  int cnt = 0;
  Best best;
  best.start(s_qv[wave], s_qi[wave], max(a.top, 1));
  auto one = [&](float v, int i, bool in) {       // all lanes; in: there is one
    v = in ? v : -INFINITY;
    if (__any(v > r.m + LAG)) renew(r, fmaxf(r.m, v));
    const float d = fmaxf(v - (r.m == -INFINITY ? 0.f : r.m), -1e30f), e = exp_of(d);
    r.s += v != v ? v : e;
    r.t = fmaf(e, d, r.t);
    cnt += in && (v > xt || (v == xt && i < tok)) ? 1 : 0;
    if (a.top) best.offer(in ? v : -INFINITY, in ? i : NONE);
  };
  const int v0 = part * sp.vecs, v1 = min(nvec, v0 + sp.vecs);
  if (part == 0)
    for (int i = 0; i < head; i += THREADS) one(i + (int)threadIdx.x < head ? (float)x[i + threadIdx.x] : 0.f, i + threadIdx.x, i + (int)threadIdx.x < head);
  for (int u = v0; u < v1; u += THREADS) {
    const int p = u + threadIdx.x;
    const bool in = p < v1;
    vec w = {};
    if (in) w = *(const vec *)(x + head + (long long)p * E);
    for (int e = 0; e < E; ++e) one((float)w[e], head + p * E + e, in);
  }
  if (part == sp.n - 1) {
    const int t0 = head + nvec * E;
    one(t0 + (int)threadIdx.x < a.V ? (float)x[t0 + threadIdx.x] : 0.f, t0 + threadIdx.x, t0 + (int)threadIdx.x < a.V);
  }
  if (a.top) best.flush();
  for (int d = 32; d > 0; d /= 2) r = joined(r, {__shfl_xor(r.m, d), __shfl_xor(r.s, d), __shfl_xor(r.t, d)});
  for (int d = 32; d > 0; d /= 2) cnt += __shfl_xor(cnt, d);
  Best::settle();
  s_qv[wave][lane] = best.mine.v;
  s_qi[wave][lane] = best.mine.i;
  if (lane == 0) {
    s_sums[wave][0] = r.m; s_sums[wave][1] = r.s; s_sums[wave][2] = r.t;
    s_cnt[wave] = cnt;
  }
  __syncthreads();
  if (wave) return;
  Entry l = best.mine;
  for (int w = 1; w < WAVES; ++w) {
    r = joined(r, {s_sums[w][0], s_sums[w][1], s_sums[w][2]});
    cnt += s_cnt[w];
    if (a.top) l = merged(l, {s_qv[w][lane], s_qi[w][lane]});
  }
  if (sp.n == 1) {
    finish(a, row, r, cnt, token_logit<T>(a, row), l);
    return;
  }
  float *o = a.work + (long long)blockIdx.x * part_words(a.top);
  if (lane == 0) *(float4 *)o = make_float4(r.m, r.s, r.t, __builtin_bit_cast(float, cnt));
  if (lane < a.top) *(float2 *)(o + 4 + 2 * lane) = make_float2(l.v, __builtin_bit_cast(float, l.i));
}

template <typename T> __global__ __launch_bounds__(64) void join_kernel(LogprobArgs a, int parts) {
  const int lane = threadIdx.x & 63, row = blockIdx.x, words = part_words(a.top);
  const float *w = a.work + (long long)row * parts * words;
  Sums r = {-INFINITY, 0.f, 0.f};
  int cnt = 0;
  if (lane < parts) {
    const float4 f = *(const float4 *)(w + lane * words);
    r = {f.x, f.y, f.z};
    cnt = __builtin_bit_cast(int, f.w);
  }
  for (int d = 32; d > 0; d /= 2) r = joined(r, {__shfl_xor(r.m, d), __shfl_xor(r.s, d), __shfl_xor(r.t, d)});
  for (int d = 32; d > 0; d /= 2) cnt += __shfl_xor(cnt, d);
  Entry l = {-INFINITY, NONE};
  if (a.top)
    for (int p = 0; p < parts; ++p) {
      Entry e = {-INFINITY, NONE};
      if (lane < a.top) {
        const float2 f = *(const float2 *)(w + p * words + 4 + 2 * lane);
        e = {f.x, __builtin_bit_cast(int, f.y)};
      }
      l = merged(l, e);
    }
  finish(a, row, r, cnt, token_logit<T>(a, row), l);
}

// Parts of a row: enough workgroups for the card, 4096 logits or more each.
int parts_of(int rows, int V) { return std::max(1, std::min({SPLITS, (1024 + rows - 1) / std::max(rows, 1), V / 4096})); }

template <typename T> void launch(const LogprobArgs &a, hipStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const int n = parts_of(a.rows, a.V);
  const Split sp = {n, (a.V / E + n - 1) / n};
  hipLaunchKernelGGL((part_kernel<T>), dim3((unsigned)(a.rows * n)), dim3(THREADS), 0, st, a, sp);
  if (n > 1) hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)a.rows), dim3(64), 0, st, a, n);
}

}  // namespace

size_t logprobs_bytes(int rows, int V, int top) {
  const int n = parts_of(rows, V);
  return n > 1 ? (size_t)rows * n * part_words(top) * sizeof(float) : 0;
}

int logprobs_launch(int type, const LogprobArgs &a, hipStream_t st) {
  if (type == CWEN_T_F32) launch<float>(a, st);
  else if (type == CWEN_T_F16) launch<TypeF16::elem>(a, st);
  else launch<TypeBF16::elem>(a, st);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
