// The gated delta rule over packed prompts, in chunks of 32 rows.
//
// With G_i the log decays of a chunk's rows summed up to row i, D_ij = exp(G_i -
// G_j) and S the state before the chunk, the rows' updates d_i solve
//   (1 + L) d = r,  L_ij = beta_i D_ij k_i.k_j (j < i),  r_i = beta_i (v_i - e^G_i S^T k_i)
// and   o_i = (e^G_i S^T q_i + sum_(j <= i) D_ij q_i.k_j d_j) / sqrt(D)
//       S  <- e^G_31 S + sum_i e^(G_31 - G_i) k_i d_i^T.
// T = (1 + L)^-1 and the scores A_ij = D_ij q_i.k_j / sqrt(D) do not depend on
// the state: a first launch forms them for all chunks side by side, a second
// one runs over the chunks of each sequence and head, S in registers.
//
// The second launch is a chain of products per chunk, column by column of S:
// X = K S, d = T r, S += K^T d.  A wave has 16 columns.  On 16x16x32 MFMA a
// product's result holds rows 4 g + i (g = lane >> 4) of column lane & 15, and an
// operand 8 values of that column; the sum's order is free as long as both
// operands agree, so the results of two 16-row tiles are the next product's
// operand as they stand (operand slot (g, j) is row 4 g + j, or 16 + 4 g + j - 4):
// the chain never leaves the registers and needs no exchange between lanes or
// waves.  K and Q are laid out in that order by the first launch.
//
// Precision: f32 values enter a product as two f16 values, x s = hi + lo with a
// power of two s, 21 bits and more below the column's largest.  One s serves a
// chunk's S, r and d: with the largest |S| and |v| of a column at 2^8 .. 2^9,
// |S^T k| <= sqrt(128) 2^9, and r and d (which the rule does not enlarge) stay
// below 2^15.  Keys and queries of 16 bits are exact f16 values after a power of
// two; what is left of their length (rho, 1 .. 2) goes into the rows' factors.  f32
// ones are normalised and split.
#include <math.h>
#include "gdn_seq.h"
#include "attn_core.h"

namespace {

constexpr int N = 32;                       // rows of a chunk

// A chunk's record of a key head: K hi [, K lo], Q hi [, Q lo] as operands:
// row 16 mt + m, dims 32 u + 4 g + j and 32 u + 16 + 4 g + j (j < 4) at half
// ((mt U + u) 64 + 16 g + m) 8, U = D / 32.  Of a value head: T hi, T lo, A hi
// [, A lo] as operands (rows mt, the chunk's rows as dims), then the factors.
template <int D, bool KL, bool OF> struct Rec {
  static constexpr int U = D / 32;
  static constexpr int OP = N * D * 2;                       // bytes of an operand
  static constexpr int K = 0, KLO = OP, Q = KL ? 2 * OP : OP, QLO = 3 * OP, KEY = KL ? 4 * OP : 2 * OP;
  static constexpr int T = 0, TLO = 2048, A = 4096, ALO = 6144, F = OF ? 8192 : 6144, HEAD = F + 1024;
};
// The factors: per row beta, beta e^G rho, rho e^(G_31 - G), e^G sigma; then e^G_31.  The scores
// and the last of the rows' factors are in units of O_UNIT, so that the low halves of small scores are no
// subnormals, and without 1 / sqrt(D).
constexpr float O_UNIT = 1.f / 64;
enum { F_BETA = 0, F_X = 32, F_D = 64, F_O = 96, F_END = 128 };

// Whether the outputs are formed with both halves of S, A and d.  Single ones are
// off by 2^-12 of S, A and d: beside the rounding to bf16 (2^-9) that does not show,
// beside the one to f16 it would.
template <typename TX, typename TO> constexpr bool full_out() { return sizeof(TX) == 4 || !std::is_same<TO, TypeBF16::elem>::value; }

struct PromptWork {
  char *key, *head;          // [piece][key head], [piece][value head]
};

__device__ __forceinline__ int operand_at(int row, int d, int U) {       // half index
  return (((row >> 4) * U + (d >> 5)) * 64 + ((d & 15) >> 2) * 16 + (row & 15)) * 8 + (d & 3) + ((d >> 4) & 1) * 4;
}
// x as an f16 value, subnormals kept.  The opaque copy keeps the compiler from
// folding a product or sum into the conversion: v_fma_mixlo_f16 gives 0 for
// subnormal results, which the low halves of values around 1 are.
__device__ __forceinline__ _Float16 f16_of(float x) { return (_Float16)f32_of(x); }
__device__ __forceinline__ floatx4_t mma(half8_t a, half8_t b, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ int value_head(const GdnRuleArgs &a, int hk, int r) { return a.group ? hk * a.group + r : hk + a.nkh * r; }

// ---- first launch: a workgroup has one chunk of one key head ----
constexpr int PREP_WAVES = 2;

template <typename TX, int D, bool OF> __global__ __launch_bounds__(64 * PREP_WAVES) void prep_kernel(GdnRuleArgs a, PromptWork w) {
  constexpr bool KL = sizeof(TX) == 4;
  typedef Rec<D, KL, OF> R;
  constexpr int U = R::U, GS = 33, HEADS = 2 * PREP_WAVES;               // HEADS value heads at a time
  __shared__ __align__(16) char s_key[R::KEY];
  __shared__ float s_G[N * GS], s_P[N * GS], s_rho[N], s_sig[N];
  // L of a head, then its T hi, T lo, A operands (rows of L are read 4 floats at a time)
  __shared__ __align__(16) char s_head[HEADS][R::F + 64];
  __shared__ float2 s_gb[HEADS][N];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int z = blockIdx.x / a.nkh, hk = blockIdx.x - z * a.nkh;
  const int s = gdn_find(a.s, z, N);
  if (s < 0) return;
  const GdnSeq q = gdn_seq(a.s, s);
  const int t0 = (z - gdn_piece0(q.first, s, N)) * N, rows = min(q.n - t0, N);
  if (t0 < 0 || rows <= 0) return;
  const long long first = (long long)q.first + t0;

  // K and Q into LDS as operands: 8 threads a row
  constexpr int PER = D / 8;
#pragma unroll
  for (int op = 0; op < 2; ++op)
    for (int row = tid >> 3; row < N; row += 8 * PREP_WAVES) {
      const TX *p = (const TX *)(op ? a.q : a.k) + (first + min(row, rows - 1)) * (op ? a.qs : a.ks) + hk * D + (tid & 7) * PER;
      float x[PER], ss = 0.f;
#pragma unroll
      for (int i = 0; i < PER; i += 8) Io<TX>::load(p + i, *(float(*)[8])&x[i]);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (row >= rows) x[i] = 0.f;
        ss = fmaf(x[i], x[i], ss);
      }
      ss += dpp<0xB1>(ss);
      ss += dpp<0x4E>(ss);
      ss += dpp<0x141>(ss);
      const float inv = 1.f / sqrtf(ss + 1e-6f);
      // 16 bits: the power of two below 1 / length, exact; the rest is a factor of the row
      const float f = KL ? inv : __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, inv) & 0x7f800000u);
      if ((tid & 7) == 0) (op ? s_sig : s_rho)[row] = KL || f == 0.f ? 1.f : inv / f;
      _Float16 *hi = (_Float16 *)(s_key + (op ? R::Q : R::K)), *lo = (_Float16 *)(s_key + (op ? R::QLO : R::KLO));
#pragma unroll
      for (int i = 0; i < PER; i += 4) {
        typedef _Float16 half4 __attribute__((ext_vector_type(4)));
        half4 h, l;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float y = x[i + j] * f;
          h[j] = f16_of(y);
          l[j] = f16_of(y - (float)h[j]);
        }
        const int at = operand_at(row, (tid & 7) * PER + i, U);
        *(half4 *)(hi + at) = h;
        if (KL) *(half4 *)(lo + at) = l;
      }
    }
  __syncthreads();
  {
    char *out = w.key + ((long long)z * a.nkh + hk) * R::KEY;
    for (int i = tid * 16; i < R::KEY; i += 64 * PREP_WAVES * 16) *(uint4 *)(out + i) = *(const uint4 *)(s_key + i);
  }
  // k_i.k_j and q_i.k_j: the waves take the rows' halves
  for (int mt = wave; mt < 2; mt += PREP_WAVES) {
    floatx4_t g[2] = {}, p[2] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      auto op = [&](int base, int m) { return *(const half8_t *)(s_key + base + ((m * U + u) * 64 + lane) * 16); };
      const half8_t km = op(R::K, mt), qm = op(R::Q, mt);
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const half8_t kn = op(R::K, nt);
        g[nt] = mma(km, kn, g[nt]);
        p[nt] = mma(qm, kn, p[nt]);
        if (KL) {
          const half8_t kl = op(R::KLO, nt);
          g[nt] = mma(km, kl, mma(op(R::KLO, mt), kn, g[nt]));
          p[nt] = mma(qm, kl, mma(op(R::QLO, mt), kn, p[nt]));
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * mt + 4 * (lane >> 4) + i, col = 16 * nt + (lane & 15);
        s_G[row * GS + col] = g[nt][i];
        s_P[row * GS + col] = p[nt][i];
      }
  }
  __syncthreads();

  // The value heads: 32 lanes each, lane n the column n of L, T and A.
  const int n = lane & 31, sub = 2 * wave + (lane >> 5), grp = a.nvh / a.nkh;
  const float rho = s_rho[n], sig = s_sig[n];
  for (int r0 = 0; r0 < grp; r0 += HEADS) {
    const int r = r0 + sub;
    const bool have = r < grp;
    const int hv = value_head(a, hk, have ? r : 0);
    float g = 0.f, beta = 0.f;
    if (have && n < rows) {
      g = a.a[(first + n) * a.gs + hv];
      beta = a.b[(first + n) * a.gs + hv];
      if (a.A) {
        const float y = g + a.dt[hv];
        g = a.A[hv] * (y > 20.f ? y : log1pf(expf(y)));
        beta = 1.f / (1.f + expf(-beta));
      }
    }
    s_gb[sub][n] = make_float2(g, beta);
    float *L = (float *)s_head[sub];
    _Float16 *op = (_Float16 *)s_head[sub];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // Decays from n to i, added up from n on: no difference of sums that are far larger.
    float acc = 0.f, pre = 0.f, dec = 1.f;
    float A[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 gb = s_gb[sub][i];
      acc = i > n ? acc + gb.x : 0.f;
      pre += i <= n ? gb.x : 0.f;
      dec = i > n ? expf(acc) : 1.f;
      L[i * N + n] = i > n ? gb.y * s_rho[i] * rho * dec * s_G[i * GS + n] : 0.f;
      A[i] = i >= n ? s_sig[i] * rho * dec * s_P[i * GS + n] / O_UNIT : 0.f;
    }
    if (have) {
      float *F = (float *)(w.head + ((long long)z * a.nvh + hv) * R::HEAD + R::F);
      const float e = expf(pre);
      F[F_BETA + n] = beta;
      F[F_X + n] = beta * e * rho;
      F[F_D + n] = rho * dec;
      F[F_O + n] = e * sig / O_UNIT;
      if (n == N - 1) F[F_END] = e;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // T column by column: T_in = [i = n] - sum_(j < i) L_ij T_jn
    float T[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = i == n ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; j += 4) {
        const float4 l = *(const float4 *)(L + i * N + j);
        t = fmaf(-l.x, T[j], t);
        if (j + 1 < i) t = fmaf(-l.y, T[j + 1], t);
        if (j + 2 < i) t = fmaf(-l.z, T[j + 2], t);
        if (j + 3 < i) t = fmaf(-l.w, T[j + 3], t);
      }
      T[i] = t;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = operand_at(i, n, 1);
      const _Float16 h = f16_of(T[i]), x = f16_of(A[i]);
      op[R::T / 2 + at] = h;
      op[R::TLO / 2 + at] = f16_of(T[i] - (float)h);
      op[R::A / 2 + at] = x;
      if (OF) op[R::ALO / 2 + at] = f16_of(A[i] - (float)x);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (have) {
      char *out = w.head + ((long long)z * a.nvh + hv) * R::HEAD;
#pragma unroll
      for (int i = 0; i < R::F; i += 512) *(uint4 *)(out + i + n * 16) = *(const uint4 *)(s_head[sub] + i + n * 16);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- second launch: NW waves of 16 columns of one head's state, over a sequence's chunks ----
// The column's largest over the 4 lanes that share it.
__device__ __forceinline__ float max_groups(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  return max_halves(fmaxf(__builtin_bit_cast(float, (int)p[0]), __builtin_bit_cast(float, (int)p[1])));
}
// x f, f a power of two, as two f16 values (below 2^-14 as 0, 2^-22 of the column's largest).
__device__ __forceinline__ void split(float x, float f, _Float16 &hi, _Float16 &lo) {
  hi = (_Float16)(x * f);
  lo = (_Float16)fmaf(x, f, -(float)hi);
}
// Any value.  The opaque copy makes its high half one value: left to itself, the
// compiler folds the product or sum before it into one of the half's two uses,
// where it is rounded once instead of twice and now and then is another.
__device__ __forceinline__ void split(float x, _Float16 &hi, _Float16 &lo) {
  x = f32_of(x);
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

template <typename TX, typename TO, int D, int NW> __global__ __launch_bounds__(64 * NW) void chain_kernel(GdnRuleArgs a, PromptWork w) {
  constexpr bool KL = sizeof(TX) == 4, OF = full_out<TX, TO>();
  typedef Rec<D, KL, OF> R;
  constexpr int U = R::U, DT = D / 16, SL = D / (16 * NW), KB = (R::KEY + R::HEAD) / 1024;
  __shared__ __align__(1024) char s_buf[2][R::KEY + R::HEAD];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  const int per = a.nvh * SL, s = blockIdx.x / per, i0 = blockIdx.x - s * per, grp = a.nvh / a.nkh;
  // Workgroups of one key head share its operands: on one XCD (block b runs on XCD b % 8).
  int hk, rest;
  if (a.nkh % 8 == 0) {
    const int j = i0 >> 3;
    hk = (i0 & 7) + 8 * (j / (grp * SL));
    rest = j % (grp * SL);
  } else {
    hk = i0 / (grp * SL);
    rest = i0 - hk * (grp * SL);
  }
  const int hv = value_head(a, hk, rest / SL), slice = rest % SL;
  const GdnSeq q = gdn_seq(a.s, s);
  if (!q.ok || gdn_taken(a.s, s, q.dst)) {
    gdn_raise(a.s);
    return;
  }
  if (q.n == 0 && (q.dst < 0 || q.dst == q.src)) return;
  const int col = slice * 16 * NW + wave * 16 + n, chunks = (q.n + N - 1) / N;
  const long long z0 = gdn_piece0(q.first, s, N);
  const char *key = w.key + (z0 * a.nkh + hk) * R::KEY, *head = w.head + (z0 * a.nvh + hv) * R::HEAD;
  const long long key_step = (long long)a.nkh * R::KEY, head_step = (long long)a.nvh * R::HEAD;
  auto land = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < (KB + NW - 1) / NW; ++p) {
      const int kb = p * NW + wave;
      if (kb < KB) {
        const char *from = kb < R::KEY / 1024 ? key + c * key_step + kb * 1024 : head + c * head_step + (kb * 1024 - R::KEY);
        __builtin_amdgcn_global_load_lds((attn_glb_t *)(from + lane * 16), (attn_lds_t *)(s_buf[c & 1] + kb * 1024), 16, 0, 0);
      }
    }
  };
  const TX *vp = (const TX *)a.v + (long long)q.first * a.vs + hv * D + col;
  TX vr[8];
  auto load_v = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vr[e] = vp[(long long)min(c * N + (e >> 2) * 16 + 4 * g + (e & 3), q.n - 1) * a.vs];
  };
  floatx4_t S[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) S[t] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
  const long long slot = (long long)a.nvh * D * D, at = (long long)hv * D * D + 4 * g * D + col;
  if (chunks) {
    land(0);
    load_v(0);
  }
  if (q.src >= 0) {
    const float *p = a.state + q.src * slot + at;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[t][i] = p[(16 * t + i) * D];
  }
  float unit = 1.f;             // S holds the state divided by it
  float o[8];                   // the last chunk's outputs
  auto store_o = [&](int c) __attribute__((always_inline)) {
    TO *p = (TO *)a.o + (long long)q.first * a.os + hv * D + col;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int row = c * N + (e >> 2) * 16 + 4 * g + (e & 3);
      if (row < q.n) p[(long long)row * a.os] = (TO)o[e];
    }
  };
  for (int c = 0; c < chunks; ++c) {
    const char *b = s_buf[c & 1], *h = b + R::KEY;
    wait_loads<0>();
    lds_barrier();
    asm volatile("" ::: "memory");
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c * N + (e >> 2) * 16 + 4 * g + (e & 3) < q.n ? (float)vr[e] : 0.f;
    // The last outputs leave here, so that the wait above never meets a store that has just begun.
    if (a.o && c) store_o(c - 1);
    if (c + 1 < chunks) {
      land(c + 1);
      load_v(c + 1);
    }
    auto op = [&](int base, int i) __attribute__((always_inline)) { return *(const half8_t *)(b + base + (i * 64 + lane) * 16); };
    // the new unit: the largest at 2^8 .. 2^9
    float mx = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) mx = fmaxf(fmaxf(fmaxf(mx, fabsf(S[t][0])), fmaxf(fabsf(S[t][1]), fabsf(S[t][2]))), fabsf(S[t][3]));
    mx *= unit;
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[e]));
    mx = max_groups(mx);
    const int ex = min(max((int)(__builtin_bit_cast(uint32_t, mx) >> 23) - 8, 1), 253);
    const float new_unit = __builtin_bit_cast(float, ex << 23), per_unit = __builtin_bit_cast(float, (254 - ex) << 23);
    // (a column that fell further than 2^100 within a chunk holds nothing beside what it held)
    const float ratio = fminf(unit * per_unit, 0x1p100f);
    unit = new_unit;
    half8_t hi[U], lo[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        _Float16 x, y;
        split(S[2 * u + (j >> 2)][j & 3], ratio, x, y);
        hi[u][j] = x;
        lo[u][j] = y;
      }
    floatx4_t X[2] = {}, Y[2] = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const half8_t k = op(R::K, mt * U + u);
        X[mt] = mma(k, lo[u], X[mt]);
        X[mt] = mma(k, hi[u], X[mt]);
        if (KL) X[mt] = mma(op(R::KLO, mt * U + u), hi[u], X[mt]);
      }
    if (a.o) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const half8_t x = op(R::Q, mt * U + u);
          Y[mt] = mma(x, hi[u], Y[mt]);
          if (OF) Y[mt] = mma(x, lo[u], Y[mt]);
          if (KL) Y[mt] = mma(op(R::QLO, mt * U + u), hi[u], Y[mt]);
        }
    }
    const float *F = (const float *)(h + R::F);
    auto rows4 = [&](int f, int mt) __attribute__((always_inline)) { return *(const floatx4_t *)(F + f + 16 * mt + 4 * g); };
    half8_t rh, rl;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const floatx4_t fb = rows4(F_BETA, mt), fx = rows4(F_X, mt);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        _Float16 x, y;
        split(fmaf(fb[i], v[4 * mt + i] * per_unit, -fx[i] * X[mt][i]), x, y);
        rh[4 * mt + i] = x;
        rl[4 * mt + i] = y;
      }
    }
    floatx4_t d[2] = {};
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const half8_t th = op(R::KEY + R::T, mt);
      d[mt] = mma(th, rh, mma(th, rl, mma(op(R::KEY + R::TLO, mt), rh, d[mt])));
    }
    half8_t dh, dl;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const floatx4_t fd = rows4(F_D, mt);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        _Float16 x, y;
        split(d[mt][i] * fd[i], x, y);
        dh[4 * mt + i] = x;
        dl[4 * mt + i] = y;
      }
    }
    const float end = F[F_END] * ratio;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      // lane i of 16: rows 4 g + i / 4, dims 4 (i % 4) ..; it gets dim i of the four rows
      auto kt = [&](int base) __attribute__((always_inline)) {
        const char *p = b + base + ((t >> 1) * 64 + (n & 3) * 16 + 4 * g + (n >> 2)) * 16 + (t & 1) * 8;
        const auto x = AttnOps<TypeF16>::tr(p), y = AttnOps<TypeF16>::tr(p + U * 1024);
        return (half8_t){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) S[t][i] *= end;
      const half8_t k = kt(R::K);
      S[t] = mma(k, dh, mma(k, dl, S[t]));
      if (KL) S[t] = mma(kt(R::KLO), dh, S[t]);
    }
    if (a.o) {
      half8_t oh, ol;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          _Float16 x, y;
          split(d[mt][i], x, y);
          oh[4 * mt + i] = x;
          ol[4 * mt + i] = y;
        }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const floatx4_t fo = rows4(F_O, mt);
        floatx4_t y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = fo[i] * Y[mt][i];
        const half8_t A = op(R::KEY + R::A, mt);
        y = mma(A, oh, y);
        if (OF) y = mma(A, ol, mma(op(R::KEY + R::ALO, mt), oh, y));
#pragma unroll
        for (int i = 0; i < 4; ++i) o[4 * mt + i] = y[i] * (unit * O_UNIT / sqrtf((float)D));
      }
    }
  }
  if (a.o && chunks) store_o(chunks - 1);
  if (q.dst >= 0) {
    float *p = a.state + q.dst * slot + at;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[(16 * t + i) * D] = S[t][i] * unit;
  }
}

template <bool KL, bool OF> void sizes(int D, size_t *key, size_t *head) {
  *key = D == 128 ? Rec<128, KL, OF>::KEY : Rec<64, KL, OF>::KEY;
  *head = Rec<128, KL, OF>::HEAD;
}
void sizes_of(int xtype, int otype, int D, size_t *key, size_t *head) {
  if (xtype == CWEN_T_F32) sizes<true, true>(D, key, head);
  else if (otype == CWEN_T_BF16) sizes<false, false>(D, key, head);
  else sizes<false, true>(D, key, head);
}

template <typename TX, typename TO, int D> void launch(const GdnRuleArgs &a, const PromptWork &w, hipStream_t st) {
  constexpr bool OF = full_out<TX, TO>();
  constexpr int NW = 4;
  const long long pieces = gdn_pieces(a.s.total, a.s.n_seq, N);
  hipLaunchKernelGGL((prep_kernel<TX, D, OF>), dim3((unsigned)(pieces * a.nkh)), dim3(64 * PREP_WAVES), 0, st, a, w);
  hipLaunchKernelGGL((chain_kernel<TX, TO, D, NW>), dim3((unsigned)((long long)a.s.n_seq * a.nvh * (D / (16 * NW)))), dim3(64 * NW), 0, st, a, w);
}
template <typename TX, typename TO> void launch_d(int D, const GdnRuleArgs &a, const PromptWork &w, hipStream_t st) {
  if (D == 128) launch<TX, TO, 128>(a, w, st);
  else launch<TX, TO, 64>(a, w, st);
}
template <typename TX> void launch_o(int otype, int D, const GdnRuleArgs &a, const PromptWork &w, hipStream_t st) {
  if (otype == CWEN_T_F32) launch_d<TX, float>(D, a, w, st);
  else if (otype == CWEN_T_F16) launch_d<TX, TypeF16::elem>(D, a, w, st);
  else launch_d<TX, TypeBF16::elem>(D, a, w, st);
}

}  // namespace

size_t gdn_prompt_bytes(int xtype, int otype, int D, int nkh, int nvh, int n_seq, int total) {
  size_t key, head;
  sizes_of(xtype, otype, D, &key, &head);
  return (size_t)gdn_pieces(total, n_seq, N) * (nkh * key + nvh * head);
}

int gdn_prompt_launch(int xtype, int otype, int D, const GdnRuleArgs &a, void *work, hipStream_t st) {
  size_t key, head;
  sizes_of(xtype, otype, D, &key, &head);
  const PromptWork w = {(char *)work, (char *)work + (size_t)gdn_pieces(a.s.total, a.s.n_seq, N) * a.nkh * key};
  if (xtype == CWEN_T_F32) launch_o<float>(otype, D, a, w, st);
  else if (xtype == CWEN_T_F16) launch_o<TypeF16::elem>(otype, D, a, w, st);
  else launch_o<TypeBF16::elem>(otype, D, a, w, st);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
