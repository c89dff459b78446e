// Log probabilities of given tokens, their ranks, entropies and the largest
// logits, in one pass over the logits.
//
// A thread keeps m, its largest logit, s = sum e^(x - m) and t = sum e^(x - m)
// (x - m); then lse = m + ln s and the entropy is ln s - t / s.  The largest one's
// own term is exactly 1, so that a token near certainty keeps its digits, and the 16
// terms of a turn are summed by themselves first, so that many small ones are not
// lost one by one beside a large sum.
//
// A wave keeps the 64 largest logits seen, one a lane, sorted by value and then
// by index.  A logit that comes before the last of the wanted ones goes into a
// queue in LDS; when 64 wait there they are sorted and merged into the list, so
// that few logits cost more than a comparison.
//
// Bound by memory where rows are many (1500 rows of 248320 in f32, the best one:
// 274 us, 5.4 TB/s), by the lists and the join where they are few (96 rows of bf16,
// the best 20: 38 us for 48 MB).
#include <math.h>
#include <algorithm>
#include "cwen_internal.h"
#include "logprobs_table.h"

namespace {

constexpr int THREADS = LP_THREADS, WAVES = 4, SPLITS = LP_SPLITS;
constexpr float LOG2E = 1.44269504088896340736f;
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
__device__ __forceinline__ Entry of_lane(Entry a, int l) {
  return {__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, a.v), l)), __builtin_amdgcn_readlane(a.i, l)};
}
// The value of the lane X apart (lane ^ X), by row permutes and swaps: a shuffle through LDS takes 100 cycles.
template <int X> __device__ __forceinline__ int apart(int v) {
  auto perm = [](int x, auto ctrl) { return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xF, 0xF, false); };
  if constexpr (X == 1) return perm(v, std::integral_constant<int, 0xB1>{});
  else if constexpr (X == 2) return perm(v, std::integral_constant<int, 0x4E>{});
  else if constexpr (X == 4) return perm(perm(v, std::integral_constant<int, 0x141>{}), std::integral_constant<int, 0x1B>{});
  else if constexpr (X == 8) return perm(v, std::integral_constant<int, 0x128>{});
  else if constexpr (X == 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __builtin_amdgcn_inverse_ballot_w64(0xFFFF0000FFFF0000ull) ? (int)p[0] : (int)p[1];
  } else {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_inverse_ballot_w64(0xFFFFFFFF00000000ull) ? (int)p[0] : (int)p[1];
  }
}
template <int X> __device__ __forceinline__ float apart(float v) { return __builtin_bit_cast(float, apart<X>(__builtin_bit_cast(int, v))); }
template <int X> __device__ __forceinline__ Entry apart(Entry a) { return {apart<X>(a.v), apart<X>(a.i)}; }
// The lanes whose bit X is clear, and of those and the others (in blocks of K) the ones that keep the entry that comes first.
constexpr unsigned long long lanes_clear(int x) {
  unsigned long long m = 0;
  for (int l = 0; l < 64; ++l)
    if (!(l & x)) m |= 1ull << l;
  return m;
}
constexpr unsigned long long keep_first(int x, int k) {
  unsigned long long m = 0;
  for (int l = 0; l < 64; ++l)
    if (!(l & x) == !(l & k)) m |= 1ull << l;
  return m;
}
// Bitonic steps X, X / 2, .. 1; in every other block of K lanes the other way round.
template <int X, int K> __device__ __forceinline__ Entry steps(Entry a) {
  const Entry b = apart<X>(a);
  const bool first = __builtin_amdgcn_inverse_ballot_w64(K < 64 ? keep_first(X, K) : lanes_clear(X));
  a = before(b, a) == first ? b : a;
  if constexpr (X > 1) return steps<X / 2, K>(a);
  else return a;
}
__device__ __forceinline__ Entry sorted(Entry a) {
  return steps<32, 64>(steps<16, 32>(steps<8, 16>(steps<4, 8>(steps<2, 4>(steps<1, 2>(a))))));
}
// The other way round: lane 63 - l.
__device__ __forceinline__ Entry turned(Entry a) { return apart<32>(apart<16>(apart<8>(apart<4>(apart<2>(apart<1>(a)))))); }
// The 64 first of two sorted lists.
__device__ __forceinline__ Entry merged(Entry a, Entry b) {
  b = turned(b);
  return steps<32, 64>(before(b, a) ? b : a);
}
// Over the wave.
__device__ __forceinline__ Sums joined(Sums r) {
  r = joined(r, {apart<1>(r.m), apart<1>(r.s), apart<1>(r.t)});
  r = joined(r, {apart<2>(r.m), apart<2>(r.s), apart<2>(r.t)});
  r = joined(r, {apart<4>(r.m), apart<4>(r.s), apart<4>(r.t)});
  r = joined(r, {apart<8>(r.m), apart<8>(r.s), apart<8>(r.t)});
  r = joined(r, {apart<16>(r.m), apart<16>(r.s), apart<16>(r.t)});
  return joined(r, {apart<32>(r.m), apart<32>(r.s), apart<32>(r.t)});
}
__device__ __forceinline__ int added(int c) {
  c += apart<1>(c);
  c += apart<2>(c);
  c += apart<4>(c);
  c += apart<8>(c);
  c += apart<16>(c);
  return c + apart<32>(c);
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
  // The lanes' largest of several logits each: as many logits as are wanted are not below the last of so many lanes.
  __device__ __forceinline__ void hint(float most) { last.v = of_lane(sorted({most, NONE}), top - 1).v; }
  __device__ __forceinline__ void offer(float v, int i) {
    if (!__any(v >= last.v)) return;
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

// One wanted entry: each lane's own, its indexes coming in their order.
struct Most {
  Entry mine, last;
  __device__ __forceinline__ void start(float *, int *, int) { mine = last = {-INFINITY, NONE}; }
  __device__ __forceinline__ void hint(float) {}
  __device__ __forceinline__ void offer(float v, int i) {
    if (before({v, i}, mine)) mine = {v, i};
  }
  __device__ __forceinline__ void flush() {
    auto step = [&](Entry b) { mine = before(b, mine) ? b : mine; };
    step(apart<1>(mine));
    step(apart<2>(mine));
    step(apart<4>(mine));
    step(apart<8>(mine));
    step(apart<16>(mine));
    step(apart<32>(mine));
    if (threadIdx.x & 63) mine = {-INFINITY, NONE};
  }
};

// Words of one part's result: m, s, t, count, then the list.
__host__ __device__ constexpr int part_words(int top) { return 4 + 2 * ((top + 1) & ~1); }
static_assert(LP_WORKGROUPS * part_words(CWEN_LOGPROBS_TOP) * 4 == CWEN_LOGPROBS_WORK_MAX, "scratch that serves every call");

__device__ __forceinline__ void finish(const LogprobArgs &a, int row, Sums r, int before_it, float xt, Entry e) {
  const int lane = threadIdx.x & 63;
  const double ls = log((double)r.s);
  if (lane == 0) {
    const int tok = a.tokens ? a.tokens[row] : -1;
    const bool there = tok >= 0 && tok < a.V && xt == xt;
    if (a.lse) a.lse[row] = r.m == -INFINITY && r.s == 0.f ? -INFINITY : (float)((double)r.m + ls);
    if (a.entropy) a.entropy[row] = r.m == -INFINITY ? NAN : (float)(ls - (double)r.t / (double)r.s);
    if (a.logprob) a.logprob[row] = there ? (float)((double)xt - r.m - ls) : NAN;
    if (a.rank) a.rank[row] = there ? before_it : -1;
  }
  if (lane < a.top) {
    if (a.top_ids) a.top_ids[(long long)row * a.top + lane] = e.i == NONE ? -1 : e.i;
    if (a.top_lp) a.top_lp[(long long)row * a.top + lane] = e.i == NONE ? -INFINITY : (float)((double)e.v - r.m - ls);
  }
}

template <typename T> __device__ __forceinline__ float token_logit(const LogprobArgs &a, int row) {
  const int tok = a.tokens ? a.tokens[row] : -1;
  return tok >= 0 && tok < a.V ? (float)((const T *)a.x)[row * a.ls + tok] : NAN;
}

// TOP: 0 no largest logits are wanted, 1 one, 2 more.  RANK: whether ranks are.
template <typename T, int TOP, bool RANK> __global__ __launch_bounds__(THREADS) void part_kernel(LogprobArgs a, lp_split sp) {
  constexpr int E = 16 / sizeof(T), VECS = LP_LOGITS / E;
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
  __shared__ float s_qv[WAVES][128], s_sums[WAVES][3];
  __shared__ int s_qi[WAVES][128], s_cnt[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x / sp.n, part = blockIdx.x - row * sp.n;
  const T *x = (const T *)a.x + row * a.ls;
  // Whole 16-byte pieces lie behind `head` logits; the first part takes those too, the last one the row's end.
  const int head = min((int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T), a.V), nvec = (a.V - head) / E;
  const int tok = RANK ? a.tokens[row] : -1;
  // What comes before the token: from its logit on at lower indexes, from the next float on at higher ones.
  const float xt = RANK ? token_logit<T>(a, row) : NAN;
  const float above = __builtin_bit_cast(float, lp_above(__builtin_bit_cast(unsigned, xt)));
  Sums r = {-INFINITY, 0.f, 0.f};
  float ref = 0.f;                    // r.m, or 0 before there is one
  int cnt = 0;
  typename std::conditional<TOP == 2, Best, Most>::type best;
  best.start(s_qv[wave], s_qi[wave], a.top);
  auto grow = [&](float v) {          // all lanes
    if (__any(v > r.m)) {
      renew(r, fmaxf(r.m, v));
      ref = r.m == -INFINITY ? 0.f : r.m;
    }
  };
  auto add = [&](float v) {
    const float d = v - ref, e = exp_of(d);
    r.s += e;
    r.t = fmaf(e, fmaxf(d, -200.f), r.t);
  };
  auto one = [&](float v, int i, bool in) {       // all lanes; in: there is one
    v = in ? v : -INFINITY;
    grow(v);
    add(v);
    if (RANK) cnt += in && v >= (i < tok ? xt : above) ? 1 : 0;
    if (TOP) best.offer(v, in ? i : NONE);
  };
  const int v0 = part * sp.vecs, v1 = part == sp.n - 1 ? nvec : min(nvec, v0 + sp.vecs);
  if (part == 0) one((int)threadIdx.x < head ? (float)x[threadIdx.x] : 0.f, threadIdx.x, (int)threadIdx.x < head);
  const int tokvec = RANK ? lp_piece(tok, head, E) : -1;
  int u = v0;
  for (; u + THREADS * VECS <= v1; u += THREADS * VECS) {
    vec w[VECS];
#pragma unroll
    for (int k = 0; k < VECS; ++k) w[k] = *(const vec *)(x + head + (long long)(u + THREADS * k + threadIdx.x) * E);
    float f[VECS][E], most = -INFINITY;
#pragma unroll
    for (int k = 0; k < VECS; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f[k][e] = (float)w[k][e];
        most = fmaxf(most, f[k][e]);
      }
    grow(most);
    float s4[4] = {}, t4[4] = {};
#pragma unroll
    for (int k = 0; k < VECS; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = f[k][e] - ref, x = exp_of(d);
        s4[e & 3] += x;
        t4[e & 3] = fmaf(x, fmaxf(d, -200.f), t4[e & 3]);       // x is 0 there, and 0 times -infinity is not
      }
    r.s += (s4[0] + s4[1]) + (s4[2] + s4[3]);
    r.t += (t4[0] + t4[1]) + (t4[2] + t4[3]);
    if (RANK) {
#pragma unroll
      for (int k = 0; k < VECS; ++k) {
        const int p = u + THREADS * k + threadIdx.x;
        const float from = p < tokvec ? xt : above;
#pragma unroll
        for (int e = 0; e < E; ++e) cnt += f[k][e] >= from ? 1 : 0;
        if (p == tokvec)
          for (int e = 0; e < E; ++e) cnt += (float)w[k][e] == xt && head + p * E + e < tok ? 1 : 0;
      }
    }
    if (TOP == 2 && u == v0) best.hint(most);
    if (TOP && __any(most >= (TOP == 1 ? best.mine.v : best.last.v))) {
#pragma unroll
      for (int k = 0; k < VECS; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) best.offer(f[k][e], head + (u + THREADS * k + (int)threadIdx.x) * E + e);
    }
  }
  for (; u < v1; u += THREADS) {
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
  if (TOP) best.flush();
  r = joined(r);
  cnt = added(cnt);
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
    if (TOP) l = merged(l, {s_qv[w][lane], s_qi[w][lane]});
  }
  if (sp.n == 1) {
    finish(a, row, r, cnt, token_logit<T>(a, row), l);
    return;
  }
  float *o = a.work + (long long)blockIdx.x * part_words(a.top);
  if (lane == 0) *(float4 *)o = make_float4(r.m, r.s, r.t, __builtin_bit_cast(float, cnt));
  if (lane < a.top) *(float2 *)(o + 4 + 2 * lane) = make_float2(l.v, __builtin_bit_cast(float, l.i));
}

// The parts of a row together: every wave asks for all of its lists at once, and merges those that can
// still matter.
template <typename T> __global__ __launch_bounds__(THREADS) void join_kernel(LogprobArgs a, int parts) {
  __shared__ float s_v[WAVES][64];
  __shared__ int s_i[WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x, words = part_words(a.top);
  const float *w = a.work + (long long)row * parts * words;
  Sums r = {-INFINITY, 0.f, 0.f};
  int cnt = 0;
  if (lane < parts) {
    const float4 f = *(const float4 *)(w + lane * words);
    r = {f.x, f.y, f.z};
    cnt = __builtin_bit_cast(int, f.w);
  }
  const float xt = token_logit<T>(a, row);
  Entry l = {-INFINITY, NONE};
  if (a.top) {
    constexpr int LISTS = SPLITS / WAVES;
    float2 e[LISTS];
#pragma unroll
    for (int k = 0; k < LISTS; ++k) {
      const int p = k * WAVES + wave;
      e[k] = make_float2(-INFINITY, __builtin_bit_cast(float, NONE));
      if (p < parts && lane < a.top) e[k] = *(const float2 *)(w + p * words + 4 + 2 * lane);
    }
#pragma unroll
    for (int k = 0; k < LISTS; ++k) {
      const Entry b = {e[k].x, __builtin_bit_cast(int, e[k].y)};
      if (k == 0) l = b;
      else if (__any(before(b, of_lane(l, a.top - 1)))) l = merged(l, b);
    }
    s_v[wave][lane] = l.v;
    s_i[wave][lane] = l.i;
    __syncthreads();
  }
  if (wave) return;
  if (a.top)
    for (int k = 1; k < WAVES; ++k) {
      const Entry b = {s_v[k][lane], s_i[k][lane]};
      if (__any(before(b, of_lane(l, a.top - 1)))) l = merged(l, b);
    }
  r = joined(r);
  cnt = added(cnt);
  finish(a, row, r, cnt, xt, l);
}

template <typename T, int TOP> void launch_parts(const LogprobArgs &a, const lp_split &sp, hipStream_t st) {
  const dim3 grid((unsigned)(a.rows * sp.n));
  if (a.rank) hipLaunchKernelGGL((part_kernel<T, TOP, true>), grid, dim3(THREADS), 0, st, a, sp);
  else hipLaunchKernelGGL((part_kernel<T, TOP, false>), grid, dim3(THREADS), 0, st, a, sp);
}
template <typename T> void launch(const LogprobArgs &a, hipStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const lp_split sp = lp_divide(a.rows, a.V, E);
  const int n = sp.n;
  if (a.top == 0) launch_parts<T, 0>(a, sp, st);
  else if (a.top == 1) launch_parts<T, 1>(a, sp, st);
  else launch_parts<T, 2>(a, sp, st);
  if (n > 1) hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)a.rows), dim3(THREADS), 0, st, a, n);
}

}  // namespace

size_t logprobs_bytes(int rows, int V, int top) {
  const int n = std::max(lp_divide(rows, V, 4).n, lp_divide(rows, V, 8).n);
  return n > 1 ? (size_t)rows * n * part_words(top) * sizeof(float) : 0;
}

int logprobs_launch(int type, const LogprobArgs &a, hipStream_t st) {
  if (type == CWEN_T_F32) launch<float>(a, st);
  else if (type == CWEN_T_F16) launch<TypeF16::elem>(a, st);
  else launch<TypeBF16::elem>(a, st);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
