// The gated delta rule over packed prompts, in chunks of 32 rows.
//
// With G_i the log decays of a chunk's rows summed up to row i, D_ij = exp(G_i -
// G_j) and S the state before the chunk, the rows' updates d_i solve
//   (1 + L) d = beta r,  L_ij = beta_i D_ij k_i.k_j (j < i),  r_i = v_i - e^G_i S^T k_i
// and   o_i = (e^G_i S^T q_i + sum_(j <= i) D_ij q_i.k_j d_j) / sqrt(D)
//       S  <- e^G_31 S + sum_i e^(G_31 - G_i) k_i d_i^T.
// T = (1 + L)^-1 beta and the scores A_ij = D_ij q_i.k_j do not depend on
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
// power of two s per column: 22 bits, and down to 2^-25 of a unit.  What counts beside
// |S| is beta |v|: T, whose columns have beta as a factor, is divided by a power of two
// of the chunk and head, its scale, that is not below the betas (1 for betas above 1/4),
// and r is multiplied by it, v and S^T k each.  The unit is taken anew, the larger of
// |S| and scale |v| at 1 .. 2, every 8 chunks and whenever a chunk's largest scale |v|
// is outside 1/8 .. 16 units.  A row lengthens a column of S by beta |v| < 32 units
// at most, from 2 sqrt(D) before the 9 chunks that a unit can have to go through: |S|,
// |S^T k| and r stay below 9300 units, d = beta (v - S^T k) below 18600, and with rho
// below 37200, where f16 ends at 65504.  Keys and queries of 16 bits are exact
// f16 values after a power of two; what is left of their length (rho, 1 .. 2) goes into
// the rows' factors.  f32 ones are normalised and split.
#include <math.h>
#include "gdn_seq.h"
#include "attn_core.h"

namespace {

constexpr int N = 32;                       // rows of a chunk

// A chunk's record of a key head: K hi [, K lo], Q hi [, Q lo] as operands:
// row 16 mt + m, dims 32 u + 4 g + j and 32 u + 16 + 4 g + j (j < 4) at half
// ((mt U + u) 64 + 16 g + m) 8, U = D / 32.  Of a value head: T hi, T lo, A hi,
// A lo as operands (rows mt, the chunk's rows as dims), then the factors.
template <int D, bool KL> struct Rec {
  static constexpr int U = D / 32;
  static constexpr int OP = N * D * 2;                       // bytes of an operand
  static constexpr int K = 0, KLO = OP, Q = KL ? 2 * OP : OP, QLO = 3 * OP, KEY = KL ? 4 * OP : 2 * OP;
  static constexpr int T = 0, TLO = 2048, A = 4096, ALO = 6144, F = 8192, HEAD = F + 512;
};
// The factors: per row scale e^G rho, rho e^(G_31 - G), e^G sigma; then e^G_31, the scale and the next chunk's (beta is in
// T's columns).  The scores
// and the last of the rows' factors are in units of O_UNIT, so that the low halves of small scores are no
// subnormals, and without 1 / sqrt(D).
constexpr float O_UNIT = 1.f / 64;
enum { F_X = 0, F_D = 32, F_O = 64, F_END = 96, F_SCALE = 97, F_NEXT = 98 };

struct PromptWork {
  char *key, *head;          // [piece][key head], [piece][value head]
};

__device__ __forceinline__ int operand_at(int row, int d, int U) {       // half index
  return (((row >> 4) * U + (d >> 5)) * 64 + ((d & 15) >> 2) * 16 + (row & 15)) * 8 + (d & 3) + ((d >> 4) & 1) * 4;
}
// x as an f16 value.  The opaque copy gives it one rounding to f32 first: left to
// itself, the compiler folds the product or sum before the conversion into one of
// the value's uses and not into another (v_fma_mixlo_f16), and now and then the
// two are different values; their difference is lost then.
__device__ __forceinline__ _Float16 f16_of(float x) { return (_Float16)f32_of(x); }
__device__ __forceinline__ floatx4_t mma(half8_t a, half8_t b, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ int value_head(const GdnRuleArgs &a, int hk, int r) { return a.group ? hk * a.group + r : hk + a.nkh * r; }

// The scale of a chunk and head, from its rows' betas in 32 lanes; one that is no number does not count.
__device__ __forceinline__ float scale_of(float beta) {
  float x = fmaxf(beta, 0.f);
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  x = fmaxf(x, dpp<0x141>(x));
  x = fmaxf(x, dpp<0x140>(x));
  const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  x = fmaxf(__builtin_bit_cast(float, (int)p[0]), __builtin_bit_cast(float, (int)p[1]));
  const float up = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, fminf(x, 1.f)) + 0x7fffffu) & 0x7f800000u);
  return x > 0.25f ? 1.f : fmaxf(up, 0x1p-60f);
}
// The value that the wave's lower (e = 0) or upper 32 lanes have in common.
__device__ __forceinline__ float of_half(float x, int e) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 32 * e));
}

// ---- first launch: a workgroup has one chunk of one key head ----
// Bound by the trips to memory and the steps of the solve, not by its bytes or operations: all loads stand at the
// start, and LDS is used twice.  Three workgroups share a CU, by their registers and by LDS (16301 rows of 16/48 heads of
// 128 in bf16: 143 us, 3.7 TB/s).
constexpr int PREP_WAVES = 4;

template <typename TX, int D> __global__ __launch_bounds__(64 * PREP_WAVES) void prep_kernel(GdnRuleArgs a, PromptWork w) {
  constexpr bool KL = sizeof(TX) == 4;
  typedef Rec<D, KL> R;
  constexpr int U = R::U, GS = 33, LS = N, HEADS = 4, HB = R::F + 64;     // HEADS value heads at a time, two a wave
  constexpr int BYTES = R::KEY > HEADS * HB ? R::KEY : HEADS * HB;
  // First K and Q; then, for a head, the rows of L (read 4 floats at a time), then its T hi, T lo, A operands.
  __shared__ __align__(16) char s_mem[BYTES];
  __shared__ float s_G[N * GS], s_P[N * GS], s_rho[N], s_sig[N];
  __shared__ float2 s_gb[HEADS][N];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int z = blockIdx.x / a.nkh, hk = blockIdx.x - z * a.nkh;
  const int s = gdn_find(a.s, z, N);
  if (s < 0) return;
  const GdnSeq q = gdn_seq(a.s, s);
  const int t0 = (z - gdn_piece0(q.first, s, N)) * N, rows = min(q.n - t0, N);
  if (t0 < 0 || rows <= 0) return;
  const long long first = (long long)q.first + t0;
  const int n = lane & 31, sub = 2 * wave + (lane >> 5), grp = a.nvh / a.nkh;
  // The gates of value head r0 + sub, row n, and the next chunk's beta there.
  const int rows_next = q.n - t0 - N;
  auto gate = [&](int r0, float &g, float &beta, float &beta_next, int &hv) {
    const int r = r0 + sub;
    const bool have = sub < HEADS && r < grp;
    hv = have ? value_head(a, hk, r) : -1;
    g = beta = beta_next = 0.f;
    if (have && n < rows) {
      g = a.a[(first + n) * a.gs + hv];
      beta = a.b[(first + n) * a.gs + hv];
    }
    if (have && n < rows_next) beta_next = a.b[(first + N + n) * a.gs + hv];
  };

  // K and Q into LDS as operands: 8 threads a row
  constexpr int PER = D / 8;
  const int row = tid >> 3;
  float x[2][PER], g, beta, beta_next;
  int hv;
#pragma unroll
  for (int op = 0; op < 2; ++op) {
    const TX *p = (const TX *)(op ? a.q : a.k) + (first + min(row, rows - 1)) * (op ? a.qs : a.ks) + hk * D + (tid & 7) * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 8) Io<TX>::load(p + i, *(float(*)[8])&x[op][i]);
  }
  gate(0, g, beta, beta_next, hv);
#pragma unroll
  for (int op = 0; op < 2; ++op) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (row >= rows) x[op][i] = 0.f;
      ss = fmaf(x[op][i], x[op][i], ss);
    }
    ss += dpp<0xB1>(ss);
    ss += dpp<0x4E>(ss);
    ss += dpp<0x141>(ss);
    const float inv = 1.f / sqrtf(ss + 1e-6f);
    // 16 bits: the power of two below 1 / length, exact; the rest is a factor of the row
    const float f = KL ? inv : __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, inv) & 0x7f800000u);
    if ((tid & 7) == 0) (op ? s_sig : s_rho)[row] = KL || f == 0.f ? 1.f : inv / f;
    _Float16 *hi = (_Float16 *)(s_mem + (op ? R::Q : R::K)), *lo = (_Float16 *)(s_mem + (op ? R::QLO : R::KLO));
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      typedef _Float16 half4 __attribute__((ext_vector_type(4)));
      half4 h, l;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = x[op][i + j] * f;
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
#pragma unroll
    for (int i = 0; i < R::KEY; i += 64 * PREP_WAVES * 16) *(uint4 *)(out + i + tid * 16) = *(const uint4 *)(s_mem + i + tid * 16);
  }
  // k_i.k_j (waves 0, 1) and q_i.k_j (2, 3), 16 rows i each
  {
    const int mt = wave & 1;
    const bool isq = wave >> 1;
    floatx4_t c[2] = {};
    auto op = [&](int base, int m, int u) { return *(const half8_t *)(s_mem + base + ((m * U + u) * 64 + lane) * 16); };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const half8_t m = op(isq ? R::Q : R::K, mt, u);
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const half8_t kn = op(R::K, nt, u);
        c[nt] = mma(m, kn, c[nt]);
        if (KL) c[nt] = mma(m, op(R::KLO, nt, u), mma(op(isq ? R::QLO : R::KLO, mt, u), kn, c[nt]));
      }
    }
    float *to = isq ? s_P : s_G;
    const float *len = isq ? s_sig : s_rho;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * mt + 4 * (lane >> 4) + i, k = 16 * nt + (lane & 15);
        to[r * GS + k] = c[nt][i] * (len[r] * s_rho[k] * (isq ? 1.f / O_UNIT : 1.f));
      }
  }
  __syncthreads();

  // The value heads: 32 lanes each, lane n the column n of L, T and A.
  if (wave >= HEADS / 2) return;
  const float rho = s_rho[n], sig = s_sig[n];
  for (int r0 = 0; r0 < grp; r0 += HEADS) {
    if (r0) gate(r0, g, beta, beta_next, hv);
    if (a.A && hv >= 0 && n < rows) {
      const float y = g + a.dt[hv];
      g = a.A[hv] * (y > 20.f ? y : log1pf(expf(y)));
      beta = 1.f / (1.f + expf(-beta));
    }
    if (a.A && hv >= 0 && n < rows_next) beta_next = 1.f / (1.f + expf(-beta_next));
    const float scale = scale_of(beta), per_scale = __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(uint32_t, scale));
    const float eg = expf(g);
    s_gb[sub][n] = make_float2(eg, beta);
    float *L = (float *)(s_mem + sub * HB);
    _Float16 *op = (_Float16 *)L;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // Decays from n to i and up to n, multiplied up: no difference of sums that are far larger.
    float dec = 0.f, pre = 1.f;
    float A[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 gb = s_gb[sub][i];
      dec = i == n ? 1.f : dec * gb.x;
      pre *= i <= n ? gb.x : 1.f;
      L[i * LS + n] = gb.y * dec * s_G[i * GS + n];             // (only i > n is read)
      A[i] = i >= n ? dec * s_P[i * GS + n] : 0.f;
    }
    const float next = scale_of(beta_next);
    char *out = w.head + ((long long)z * a.nvh + max(hv, 0)) * R::HEAD;
    if (hv >= 0) {
      float *F = (float *)(out + R::F);
      F[F_X + n] = pre * rho * scale;
      F[F_D + n] = rho * dec;
      F[F_O + n] = pre * sig / O_UNIT;
      if (n == N - 1) {
        F[F_END] = pre;
        F[F_SCALE] = scale;
        F[F_NEXT] = next;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // (1 + L)^-1 in blocks of 16 rows: the two on the diagonal column by column, T_in = [i = n] - sum_(j < i) L_ij T_jn,
    // both at once; the third is -T22 (L21 T11), on the matrix cores in f32.
    float T[16];
    {
      const int h = n >> 4, m = n & 15;
      const float *Lh = L + 16 * h * LS + 16 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float t = i == m ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; j += 4) {
          const float4 l = *(const float4 *)(Lh + i * LS + j);
          t = fmaf(-l.x, T[j], t);
          if (j + 1 < i) t = fmaf(-l.y, T[j + 1], t);
          if (j + 2 < i) t = fmaf(-l.z, T[j + 2], t);
          if (j + 3 < i) t = fmaf(-l.w, T[j + 3], t);
        }
        T[i] = t;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < 16; ++i) L[(16 * h + i) * LS + 16 * h + m] = T[i];      // over L11 and L22
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    floatx4_t T21[2];                  // of the wave's two heads: rows 16 + 4 g + i, column m
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float *Lw = (const float *)(s_mem + (2 * wave + e) * HB);
      const int m = lane & 15, g4 = lane >> 4;
      floatx4_t M = {}, t = {};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        M = __builtin_amdgcn_mfma_f32_16x16x4f32(Lw[(16 + m) * LS + 4 * g4 + k], Lw[(4 * g4 + k) * LS + m], M, 0, 0, 0);
      // (a row of M that is not finite makes the rows from it on so, and must not reach those before it)
      int clear = 16;
      if (__any(!(fabsf(M[0]) + fabsf(M[1]) + fabsf(M[2]) + fabsf(M[3]) < INFINITY))) {
#pragma unroll
        for (int k = 15; k >= 0; --k)
          if (__any(4 * g4 == (k & 12) && !(fabsf(M[k & 3]) < INFINITY))) clear = k;
#pragma unroll
        for (int k = 0; k < 4; ++k) M[k] = 4 * g4 + k < clear ? M[k] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float T22 = m >= 4 * g4 + k ? Lw[(16 + m) * LS + 16 + 4 * g4 + k] : 0.f;
        t = __builtin_amdgcn_mfma_f32_16x16x4f32(T22, -M[k], t, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) T21[e][k] = 4 * g4 + k < clear ? t[k] : NAN;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    auto put = [&](_Float16 *to, int i, int col, float t) {
      const int at = operand_at(i, col, 1);
      const _Float16 h = f16_of(t);
      to[R::T / 2 + at] = h;
      to[R::TLO / 2 + at] = f16_of(t - (float)h);
    };
#pragma unroll
    for (int i = 0; i < 16; ++i) put(op, 16 * (n >> 4) + i, n, i >= (n & 15) ? T[i] * (beta * per_scale) : 0.f);   // (beta may be NaN)
    // rows 0 .. 15 of the later columns: nothing (zeros of the earlier lanes' blocks)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (n >= 16) put(op, i, n, 0.f);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int m = lane & 15;
      const float b = s_gb[2 * wave + e][m].y * of_half(per_scale, e);
#pragma unroll
      for (int i = 0; i < 4; ++i) put((_Float16 *)(s_mem + (2 * wave + e) * HB), 16 + 4 * (lane >> 4) + i, m, T21[e][i] * b);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = operand_at(i, n, 1);
      const _Float16 x = f16_of(A[i]);
      op[R::A / 2 + at] = x;
      op[R::ALO / 2 + at] = f16_of(A[i] - (float)x);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (hv >= 0) {
#pragma unroll
      for (int i = 0; i < R::F; i += 512) *(uint4 *)(out + i + n * 16) = *(const uint4 *)(s_mem + sub * HB + i + n * 16);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- second launch: NW waves of 16 columns of one head's state, over a sequence's chunks ----
// One more wave of the workgroup brings the records into LDS, two chunks ahead: the loads take the time of
// their bytes to issue, which a wave of the chain would wait out.
// The column's largest over the 4 lanes that share it.
__device__ __forceinline__ float max_groups(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  return max_halves(fmaxf(__builtin_bit_cast(float, (int)p[0]), __builtin_bit_cast(float, (int)p[1])));
}
// Two operands whose sum is x, one multiply-add that rounds to f16 for each low half (the compiler takes two
// instructions and a half).  The block reads x behind the conversions that gave h0 .. h3, so a matrix result in x is
// complete.  Its first instruction is the wait that a matrix instruction's addend needs before it may be overwritten (7
// cycles here), its last the one that a vector result needs before a matrix instruction reads it: the compiler puts
// neither in front of or behind assembly.
__device__ __forceinline__ void split8(const float (&x)[8], half8_t &hi, half8_t &lo) {
  half2_t h0 = {(_Float16)x[0], (_Float16)x[1]}, h1 = {(_Float16)x[2], (_Float16)x[3]};
  half2_t h2 = {(_Float16)x[4], (_Float16)x[5]}, h3 = {(_Float16)x[6], (_Float16)x[7]}, l0, l1, l2, l3;
  asm("s_nop 7\n"
      "v_fma_mixlo_f16 %0, %8, 1.0, -%4 op_sel_hi:[0,0,1]\n"
      "v_fma_mixlo_f16 %1, %10, 1.0, -%5 op_sel_hi:[0,0,1]\n"
      "v_fma_mixlo_f16 %2, %12, 1.0, -%6 op_sel_hi:[0,0,1]\n"
      "v_fma_mixlo_f16 %3, %14, 1.0, -%7 op_sel_hi:[0,0,1]\n"
      "v_fma_mixhi_f16 %0, %9, 1.0, -%4 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n"
      "v_fma_mixhi_f16 %1, %11, 1.0, -%5 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n"
      "v_fma_mixhi_f16 %2, %13, 1.0, -%6 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n"
      "v_fma_mixhi_f16 %3, %15, 1.0, -%7 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n"
      "s_nop 1"
      : "=&v"(l0), "=&v"(l1), "=&v"(l2), "=&v"(l3), "+v"(h0), "+v"(h1), "+v"(h2), "+v"(h3)
      : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]));
  hi = (half8_t){h0[0], h0[1], h1[0], h1[1], h2[0], h2[1], h3[0], h3[1]};
  lo = (half8_t){l0[0], l0[1], l1[0], l1[1], l2[0], l2[1], l3[0], l3[1]};
}
// The high one alone.
__device__ __forceinline__ half8_t high8(const float (&x)[8]) {
  return (half8_t){(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3], (_Float16)x[4], (_Float16)x[5], (_Float16)x[6], (_Float16)x[7]};
}

template <typename TX, typename TO, int D, int NW> struct Chain {
  static constexpr bool KL = sizeof(TX) == 4;
  typedef Rec<D, KL> R;
  static constexpr int U = R::U, DT = D / 16, KB = R::KEY / 1024 + R::HEAD / 1024 + 1, XS = sizeof(TX), OS = sizeof(TO);
  static constexpr int VP = XS / 2, OP = OS / 2;     // a wave's loads and stores of a chunk
  // Of two waves each has another one that forms its outputs, a chunk later, from S's and d's halves in LDS: what a chunk
  // takes is one wave's products and instructions, one after the other (8192 rows of 48 heads of 128 in bf16, both launches:
  // 406 us, with the outputs among them 449).  f32 heads of 128 have no room for that and a fourth record.
  static constexpr bool SPLIT = NW == 2 && (XS == 2 || D == 64);
  static constexpr int EX = 2 * (U + 1) * 1024 + 512, NV = SPLIT ? 4 : 3;
  typedef char Buf[R::KEY + R::HEAD];

  int lane, n, g;
  // the sequence
  long long v_chunk, o_chunk;        // bytes of a chunk's rows
  const char *v0;
  char *o0;
  int rows;
  uint32_t v_row, o_row;             // bytes of a row
  uint32_t v_at[VP], o_at[OP];
  char *s_io;                        // the wave's columns of a chunk, row by row: values, then outputs, of which the
                                     // values are read before outputs are written, and outputs before the next values
  float out_unit;
  // the state, divided by the column's unit, and the present chunk's values, with its scale
  floatx4_t S[DT];
  float unit, per_unit, v[8], vmax, scale;
  uint4 vr[NV][VP];                  // values on their way: chunk c's in vr[c % NV]
  float far[XS == 4 ? 8 : 4];    // the chunk's after that, by columns (16 bits: two a float)

  // A chunk's rows of v and o as buffers that end with the sequence: loads past it give 0, stores past it (and to no o)
  // do nothing, so no row needs a comparison.  A lane takes 16 bytes at a time; LDS turns rows into columns.
  __device__ __forceinline__ uint32_t bytes_of(int c, uint32_t row, int es) const {
    const int left = min(rows - c * N, N);
    return c >= 0 && left > 0 ? (uint32_t)(left - 1) * row + D * es : 0u;
  }
  __device__ __forceinline__ void load_v(int c, uint4 (&to)[VP]) const {
    const auto r = make_rsrc(v0 + c * v_chunk, bytes_of(c, v_row, XS));
#pragma unroll
    for (int i = 0; i < VP; ++i) to[i] = bload16(r, v_at[i]);
  }
  __device__ __forceinline__ void turn_v(const uint4 (&from)[VP]) {
    typedef typename std::conditional<std::is_same<TX, TypeBF16::elem>::value, TypeBF16, TypeF16>::type Type;
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < VP; ++i) *(uint4 *)(s_io + (i * 64 + lane) * 16) = from[i];
    asm volatile("" ::: "memory");
    if constexpr (XS == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) far[e] = ((const float *)s_io)[((e >> 2) * 16 + 4 * g + (e & 3)) * 16 + n];
    } else {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 x = __builtin_bit_cast(f2, AttnOps<Type>::tr(s_io + (mt * 16 + 4 * g + (n >> 2)) * 32 + (n & 3) * 8));
        far[2 * mt] = x[0];
        far[2 * mt + 1] = x[1];
      }
    }
    asm volatile("" ::: "memory");
  }
  // The turned values become the present ones; vmax: their column's largest, times their scale.
  __device__ __forceinline__ void take_v() {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (XS == 4) {
        v[e] = far[e];
      } else {
        const uint32_t x = __builtin_bit_cast(uint32_t, far[e >> 1]);
        if constexpr (std::is_same<TX, TypeBF16::elem>::value) v[e] = __builtin_bit_cast(float, e & 1 ? x & 0xffff0000u : x << 16);
        else v[e] = (float)__builtin_bit_cast(half2_t, x)[e & 1];
      }
    }
    vmax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) vmax = fmaxf(vmax, fabsf(v[e]));
    vmax = max_groups(vmax) * scale;
  }
  // Of the finite ones: an infinite value is no measure for the rows before it.
  __device__ __forceinline__ void finite_vmax() {
    vmax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) vmax = fmaxf(vmax, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
    vmax = max_groups(vmax) * scale;
  }
  // The unit for the larger of |S| and `most` (a scaled |v|) to lie in 1 .. 2, in the columns that call for it: what a column
  // gets does not depend on its neighbours.  Returns what S has to be multiplied by.
  __device__ __forceinline__ float renew(float most, bool call) {
    float mx = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fabsf(S[t][i]));
    mx = fmaxf(max_groups(mx) * unit, most);
    const int ex = min(max((int)(__builtin_bit_cast(uint32_t, mx) >> 23), 1), 253);
    const float old = unit;
    unit = call ? __builtin_bit_cast(float, ex << 23) : unit;
    per_unit = call ? __builtin_bit_cast(float, (254 - ex) << 23) : per_unit;
    // (a column that fell further than 2^100 since holds nothing beside what it held)
    return fminf(old * per_unit, 0x1p100f);
  }
  // The first of a column's rows that is not finite, or N, less 4 g (value e of a lane is row at(e) + 4 g).
  static __device__ constexpr int at(int e) { return (e >> 2) * 16 + (e & 3); }
  __device__ __forceinline__ int first_odd(const float (&x)[8]) const {
    int first = N;
#pragma unroll
    for (int e = 7; e >= 0; --e) first = fabsf(x[e]) < INFINITY ? first : at(e);
    return -(int)max_groups(-(float)min(first + 4 * g, N)) - 4 * g;
  }
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  __device__ __forceinline__ void read_o(u32x4 (&x)[OP]) const {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < OP; ++i) x[i] = *(const u32x4 *)(s_io + (i * 64 + lane) * 16);
    asm volatile("" ::: "memory");
  }
  __device__ __forceinline__ void store_o(int c, const u32x4 (&x)[OP]) const {
    const auto r = make_rsrc(o0 + c * o_chunk, o0 ? bytes_of(c, o_row, OS) : 0u);
#pragma unroll
    for (int i = 0; i < OP; ++i) __builtin_amdgcn_raw_buffer_store_b128(x[i], r, o_at[i], 0, 0);
  }

  // Chunk c, whose record is in `b` behind the barrier.  v holds its values, `far` those of c + 1, vr_2 those of c + 2;
  // vr_4 takes c + 4's.
  __device__ __forceinline__ void chunk(int c, Buf &b, const uint4 (&vr_2)[VP], uint4 (&vr_4)[VP], char *ex) {
    const float *F = (const float *)(b + R::KEY + R::F);
    u32x4 o_last[OP];
    if (!SPLIT) read_o(o_last);
    asm volatile("" ::: "memory");
    lds_barrier();
    asm volatile("" ::: "memory");
    auto op = [&](int base, int i) __attribute__((always_inline)) { return *(const half8_t *)(b + base + (i * 64 + lane) * 16); };
    auto rows4 = [&](int f, int mt) __attribute__((always_inline)) { return *(const floatx4_t *)(F + f + 16 * mt + 4 * g); };
    // lane i of 16: rows 4 g + i / 4, dims 4 (i % 4) ..; it gets dim i of the four rows
    auto kt = [&](int base, int t) __attribute__((always_inline)) {
      const char *p = b + base + ((t >> 1) * 64 + (n & 3) * 16 + 4 * g + (n >> 2)) * 16 + (t & 1) * 8;
      const auto x = AttnOps<TypeF16>::tr(p), y = AttnOps<TypeF16>::tr(p + U * 1024);
      return (half8_t){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };
    // Operands are asked for a stage before the product that takes them (stages do not mix): left to itself the
    // compiler reads each one just ahead of its product, and the wave, alone on its SIMD, waits for LDS 30 times a chunk.
    const float scale_next = F[F_NEXT];
    half8_t K[2 * U], KL_[2 * U];
#pragma unroll
    for (int i = 0; i < 2 * U; ++i) {
      K[i] = op(R::K, i);
      if (KL) KL_[i] = op(R::KLO, i);
    }
    floatx4_t fx[2], fd[2], fo[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) fx[mt] = rows4(F_X, mt);
    // The present values, scaled, in units, and whether the next ones call for new units in the chunks to come: at least
    // every 8, and where their scaled |v| leaves what the present one is good for.
    float w[8], ratio = 1.f;
    const float vmax_here = vmax, unit_here = unit, to_units = per_unit * scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = v[e] * to_units;
    scale = scale_next;
    take_v();
    auto stay = [&]() __attribute__((always_inline)) {
      const float vu = vmax * per_unit;
      return (c & 7) != 7 && vu < 16.f && vu >= 0.125f;
    };
    if (!__all(stay())) {
      if (__any(vmax == INFINITY)) finite_vmax();
      ratio = renew(fmaxf(vmax_here, vmax), !stay());
    }
    if (!SPLIT) store_o(c - 1, o_last);
    load_v(c + 4, vr_4);
    half8_t hi[U], lo[U];
    floatx4_t X[2] = {}, Y[2] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = S[2 * u + (j >> 2)][j & 3];
      split8(x, hi[u], lo[u]);
      if (SPLIT) {
        *(half8_t *)(ex + (u * 64 + lane) * 16) = hi[u];
        *(half8_t *)(ex + ((U + 1 + u) * 64 + lane) * 16) = lo[u];
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) X[mt] = mma(K[mt * U + u], lo[u], X[mt]);
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) X[mt] = mma(K[mt * U + u], hi[u], X[mt]);
      if (KL)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) X[mt] = mma(KL_[mt * U + u], hi[u], X[mt]);
    }
    __builtin_amdgcn_sched_barrier(0);
    half8_t T[2], TL[2], Q[2 * U], QL[2 * U];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) T[mt] = op(R::KEY + R::T, mt), TL[mt] = op(R::KEY + R::TLO, mt);
    if (!SPLIT)
#pragma unroll
      for (int i = 0; i < 2 * U; ++i) {
        Q[i] = op(R::Q, i);
        if (KL) QL[i] = op(R::QLO, i);
      }
    half8_t rh, rl;
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = fmaf(-fx[e >> 2][e & 3], X[e >> 2][e & 3], w[e]);
    split8(r, rh, rl);
    if (!SPLIT)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          Y[mt] = mma(Q[mt * U + u], hi[u], Y[mt]);
          Y[mt] = mma(Q[mt * U + u], lo[u], Y[mt]);
          if (KL) Y[mt] = mma(QL[mt * U + u], hi[u], Y[mt]);
        }
    __builtin_amdgcn_sched_barrier(0);
    half8_t KT[DT], KTL[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      KT[t] = kt(R::K, t);
      if (KL) KTL[t] = kt(R::KLO, t);
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) fd[mt] = rows4(F_D, mt);
    const float end = F[F_END];
    // (two waves have registers for these as well by now; of more, three share a SIMD's)
    half8_t A[2], AL[2];
    auto ask_a = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        fo[mt] = rows4(F_O, mt);
        A[mt] = op(R::KEY + R::A, mt);
        AL[mt] = op(R::KEY + R::ALO, mt);
      }
    };
    if (NW <= 2 && !SPLIT) ask_a();
    floatx4_t d[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) d[mt] = mma(T[mt], rh, mma(TL[mt], rh, mma(T[mt], rl, (floatx4_t){0.f, 0.f, 0.f, 0.f})));
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[t][i] *= end * ratio;
    __builtin_amdgcn_sched_barrier(0);
    turn_v(vr_2);
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = d[e >> 2][e & 3];
      y[e] = x[e] * (fd[e >> 2][e & 3] * ratio);
    }
    // A row of d that is not finite leaves nothing finite in its column of S.  But it must not reach the outputs of the rows
    // before it, whose products with it are 0 times that, neither here nor in d: there those rows are solved anew.
    float odd = 0.f;
    half8_t oh = high8(x), ol;
#pragma unroll
    for (int e = 0; e < 8; e += 2) odd = __builtin_amdgcn_fdot2((half2_t){oh[e], oh[e + 1]}, (half2_t){0, 0}, odd, false);
    const bool is_odd = __any(odd != 0.f);        // (0 or NaN)
    half8_t dh, dl;
    split8(y, dh, dl);
#pragma unroll
    for (int t = 0; t < DT; ++t) S[t] = mma(KT[t], dl, S[t]);
#pragma unroll
    for (int t = 0; t < DT; ++t) S[t] = mma(KT[t], dh, S[t]);
    if (KL)
#pragma unroll
      for (int t = 0; t < DT; ++t) S[t] = mma(KTL[t], dh, S[t]);
    if (NW > 2) {
      __builtin_amdgcn_sched_barrier(0);
      ask_a();
    }
    int clear = N;                // (less 4 g)
    if (is_odd) {                 // (behind the state's products: ahead of them its values would not fit the registers)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)rh[e];
      clear = first_odd(x);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at(e) >= clear) rh[e] = rl[e] = (_Float16)0.f;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const half8_t t = op(R::KEY + R::T, mt), u = op(R::KEY + R::TLO, mt);
        d[mt] = mma(t, rh, mma(u, rh, mma(t, rl, (floatx4_t){0.f, 0.f, 0.f, 0.f})));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = d[e >> 2][e & 3];
      clear = min(clear, first_odd(x));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = at(e) < clear ? x[e] : 0.f;
        if (at(e) >= clear) Y[e >> 2][e & 3] = NAN;
      }
    }
    split8(x, oh, ol);
    if constexpr (SPLIT) {
      *(half8_t *)(ex + (U * 64 + lane) * 16) = oh;
      *(half8_t *)(ex + ((2 * U + 1) * 64 + lane) * 16) = ol;
      *(float2 *)(ex + 2 * (U + 1) * 1024 + lane * 8) = make_float2(unit_here, __builtin_bit_cast(float, clear));
      return;
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      floatx4_t y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = fo[mt][i] * Y[mt][i];
      y = mma(A[mt], ol, mma(AL[mt], oh, mma(A[mt], oh, y)));
#pragma unroll
      for (int i = 0; i < 4; ++i) ((TO *)s_io)[(16 * mt + 4 * g + i) * 16 + n] = (TO)(y[i] * (unit_here * out_unit));
    }
  }

  // The other wave's part of chunk c, behind the barrier of chunk c + 1.
  __device__ __forceinline__ void outputs(int c, Buf &b, const char *ex) {
    asm volatile("" ::: "memory");
    lds_barrier();
    asm volatile("" ::: "memory");
    if (!o0) return;
    const float *F = (const float *)(b + R::KEY + R::F);
    auto op = [&](const char *from, int i) __attribute__((always_inline)) { return *(const half8_t *)(from + (i * 64 + lane) * 16); };
    half8_t Q[2 * U], QL[2 * U], hi[U], lo[U], A[2], AL[2], oh, ol;
    floatx4_t Y[2] = {}, fo[2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      hi[u] = op(ex, u);
      lo[u] = op(ex, U + 1 + u);
    }
#pragma unroll
    for (int i = 0; i < 2 * U; ++i) {
      Q[i] = op(b + R::Q, i);
      if (KL) QL[i] = op(b + R::QLO, i);
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      fo[mt] = *(const floatx4_t *)(F + F_O + 16 * mt + 4 * g);
      A[mt] = op(b + R::KEY + R::A, mt);
      AL[mt] = op(b + R::KEY + R::ALO, mt);
    }
    oh = op(ex, U);
    ol = op(ex, 2 * U + 1);
    const float2 column = *(const float2 *)(ex + 2 * (U + 1) * 1024 + lane * 8);       // its unit; its first row that is not finite
    const int clear = __builtin_bit_cast(int, column.y);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        Y[mt] = mma(Q[mt * U + u], hi[u], Y[mt]);
        Y[mt] = mma(Q[mt * U + u], lo[u], Y[mt]);
        if (KL) Y[mt] = mma(QL[mt * U + u], hi[u], Y[mt]);
      }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      floatx4_t y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = 16 * mt + i < clear ? fo[mt][i] * Y[mt][i] : NAN;
      y = mma(A[mt], ol, mma(AL[mt], oh, mma(A[mt], oh, y)));
#pragma unroll
      for (int i = 0; i < 4; ++i) ((TO *)s_io)[(16 * mt + 4 * g + i) * 16 + n] = (TO)(y[i] * (column.x * out_unit));
    }
    u32x4 o[OP];
    read_o(o);
    store_o(c, o);
  }
};

// The nth longest sequence (of up to 64; more stay in their order), so that no long one starts when the others are done.
__device__ __forceinline__ int nth_longest(const GdnSeqs &a, int nth) {
  if (a.n_seq == 1 || a.n_seq > 64) return nth;
  const int lane = threadIdx.x & 63, n = lane < a.n_seq ? gdn_seq(a, lane).n : -1;
  int rank = 0;
  for (int j = 0; j < a.n_seq; ++j) {
    const int m = __builtin_amdgcn_readlane(n, j);
    rank += m > n || (m == n && j < lane) ? 1 : 0;
  }
  return __builtin_ctzll(__ballot(lane < a.n_seq && rank == nth));
}

// Three records in LDS, an array each: in one, the compiler would wait for the loads into one record
// before it reads another.
template <typename TX, typename TO, int D, int NW>
__global__ __launch_bounds__(64 * (Chain<TX, TO, D, NW>::SPLIT ? 2 * NW + 1 : NW + 1), NW >= 4 && sizeof(TX) == 2 ? 3 : 1)
void chain_kernel(GdnRuleArgs a, PromptWork w) {
  typedef Chain<TX, TO, D, NW> C;
  typedef typename C::R R;
  constexpr bool SPLIT = C::SPLIT;
  constexpr int SL = D / (16 * NW), OUT = SPLIT ? NW : 0;        // waves of outputs, before those of the chain
  __shared__ __align__(1024) typename C::Buf b0, b1, b2;
  __shared__ __align__(1024) char b3_[SPLIT ? sizeof(typename C::Buf) : 16];
  __shared__ __align__(16) char s_io[OUT + NW][N * 16 * (C::XS > C::OS ? C::XS : C::OS)];
  __shared__ __align__(16) char s_ex[SPLIT ? 2 : 1][SPLIT ? NW : 1][SPLIT ? C::EX : 16];
  typename C::Buf &b3 = (typename C::Buf &)b3_;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = a.nvh * SL, nth = blockIdx.x / per, i0 = blockIdx.x - nth * per, grp = a.nvh / a.nkh;
  const int s = nth_longest(a.s, nth);
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
  const int chunks = (q.n + N - 1) / N;
  if (wave == OUT + NW) {
    if (!chunks) return;
    const long long z0 = gdn_piece0(q.first, s, N), key_step = (long long)a.nkh * R::KEY, head_step = (long long)a.nvh * R::HEAD;
    const char *key = w.key + (z0 * a.nkh + hk) * R::KEY + lane * 16, *head = w.head + (z0 * a.nvh + hv) * R::HEAD + lane * 16;
    // The next record, in order; past the last one that one again, so that there is always one to count.
    int c = 0;
    auto land = [&](typename C::Buf &to) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < R::KEY / 1024; ++i)
        __builtin_amdgcn_global_load_lds((attn_glb_t *)(key + i * 1024), (attn_lds_t *)(to + i * 1024), 16, 0, 0);
#pragma unroll
      for (int i = 0; i < R::HEAD / 1024; ++i)
        __builtin_amdgcn_global_load_lds((attn_glb_t *)(head + i * 1024), (attn_lds_t *)(to + R::KEY + i * 1024), 16, 0, 0);
      constexpr int most = R::HEAD / 1024 * 1024;
      static_assert(R::KEY % 1024 == 0 && R::HEAD - most == 512, "a record ends in half a load");
      if (lane < 32)
        __builtin_amdgcn_global_load_lds((attn_glb_t *)(head + most), (attn_lds_t *)(to + R::KEY + most), 16, 0, 0);
      if (++c < chunks) key += key_step, head += head_step;
    };
    // Buffer c % 3 is read until the barrier of chunk c + 1, behind which chunk c + 3 goes there (SPLIT: c % 4, c + 2, c + 4).
    auto next = [&](typename C::Buf &to) __attribute__((always_inline)) {
      wait_loads<C::KB>();
      lds_barrier();
      asm volatile("" ::: "memory");
      land(to);
    };
    land(b0);
    land(b1);
    for (int i = 0;;) {
      next(b2);
      if (++i == chunks) break;
      if (SPLIT) {
        next(b3);
        if (++i == chunks) break;
      }
      next(b0);
      if (++i == chunks) break;
      next(b1);
      if (++i == chunks) break;
    }
    if (SPLIT) lds_barrier();
    wait_loads<0>();            // what was asked for past the end lands before the LDS is given up
    return;
  }
  C p;
  p.lane = lane;
  p.n = lane & 15;
  p.g = lane >> 4;
  const int part = SPLIT && wave >= NW ? wave - NW : wave, c0 = (slice * NW + part) * 16;             // the wave's first column
  p.rows = q.n;
  p.o0 = a.o ? (char *)a.o + (q.first * a.os + hv * D) * C::OS : nullptr;
  p.o_row = (uint32_t)a.os * C::OS;
  p.o_chunk = a.os * C::OS * N;
#pragma unroll
  for (int i = 0; i < C::OP; ++i) p.o_at[i] = (i * 64 + lane) / C::OS * p.o_row + c0 * C::OS + lane % C::OS * 16;
  p.s_io = s_io[wave];
  p.out_unit = O_UNIT / sqrtf((float)D);
  if constexpr (SPLIT) {
    if (wave < NW) {
      if (!chunks) return;
      lds_barrier();                                   // of chunk 0
      for (int c = 0;;) {
        p.outputs(c, b0, s_ex[0][part]);
        if (++c == chunks) break;
        p.outputs(c, b1, s_ex[1][part]);
        if (++c == chunks) break;
        p.outputs(c, b2, s_ex[0][part]);
        if (++c == chunks) break;
        p.outputs(c, b3, s_ex[1][part]);
        if (++c == chunks) break;
      }
      return;
    }
  }
  const long long slot = (long long)a.nvh * D * D, at = (long long)hv * D * D + 4 * p.g * D + c0 + p.n;
#pragma unroll
  for (int t = 0; t < C::DT; ++t) p.S[t] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
  if (q.src >= 0) {
    const float *from = a.state + q.src * slot + at;
#pragma unroll
    for (int t = 0; t < C::DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) p.S[t][i] = from[(16 * t + i) * D];
  }
  p.unit = p.per_unit = p.scale = 1.f;
  if (chunks) {
    p.scale = *(const float *)(w.head + ((long long)gdn_piece0(q.first, s, N) * a.nvh + hv) * R::HEAD + R::F + 4 * F_SCALE);
    p.v0 = (const char *)a.v + (q.first * a.vs + hv * D) * C::XS;
    p.v_row = (uint32_t)a.vs * C::XS;
    p.v_chunk = a.vs * C::XS * N;
#pragma unroll
    for (int i = 0; i < C::VP; ++i) p.v_at[i] = (i * 64 + p.lane) / C::XS * p.v_row + c0 * C::XS + p.lane % C::XS * 16;
    p.load_v(0, p.vr[0]);
    p.load_v(1, p.vr[1]);
    p.load_v(2, p.vr[2]);
    p.turn_v(p.vr[0]);
    p.take_v();
    p.finite_vmax();
    p.turn_v(p.vr[1]);
    p.load_v(3, p.vr[3 % C::NV]);
    const float ratio = p.renew(p.vmax, true);
#pragma unroll
    for (int t = 0; t < C::DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) p.S[t][i] *= ratio;
    if constexpr (SPLIT) {
      for (int c = 0;;) {
        p.chunk(c, b0, p.vr[2], p.vr[0], s_ex[0][part]);
        if (++c == chunks) break;
        p.chunk(c, b1, p.vr[3], p.vr[1], s_ex[1][part]);
        if (++c == chunks) break;
        p.chunk(c, b2, p.vr[0], p.vr[2], s_ex[0][part]);
        if (++c == chunks) break;
        p.chunk(c, b3, p.vr[1], p.vr[3], s_ex[1][part]);
        if (++c == chunks) break;
      }
      asm volatile("" ::: "memory");
      lds_barrier();
    } else {
      for (int c = 0;;) {
        p.chunk(c, b0, p.vr[2], p.vr[1], nullptr);
        if (++c == chunks) break;
        p.chunk(c, b1, p.vr[0], p.vr[2], nullptr);
        if (++c == chunks) break;
        p.chunk(c, b2, p.vr[1], p.vr[0], nullptr);
        if (++c == chunks) break;
      }
      typename C::u32x4 o_last[C::OP];
      p.read_o(o_last);
      p.store_o(chunks - 1, o_last);
    }
  }
  if (q.dst >= 0) {
    float *to = a.state + q.dst * slot + at;
#pragma unroll
    for (int t = 0; t < C::DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) to[(16 * t + i) * D] = p.S[t][i] * p.unit;
  }
}

void sizes_of(int xtype, int D, size_t *key, size_t *head) {
  if (xtype == CWEN_T_F32) *key = D == 128 ? Rec<128, true>::KEY : Rec<64, true>::KEY;
  else *key = D == 128 ? Rec<128, false>::KEY : Rec<64, false>::KEY;
  *head = Rec<128, true>::HEAD;             // of every form
}

template <typename TX, typename TO, int D, int NW> void launch_chain(const GdnRuleArgs &a, const PromptWork &w, hipStream_t st) {
  constexpr int SL = D / (16 * NW);
  hipLaunchKernelGGL((chain_kernel<TX, TO, D, NW>), dim3((unsigned)((long long)a.s.n_seq * a.nvh * SL)), dim3(64 * (Chain<TX, TO, D, NW>::SPLIT ? 2 * NW + 1 : NW + 1)), 0, st, a, w);
}
template <typename TX, typename TO, int D> void launch(const GdnRuleArgs &a, const PromptWork &w, hipStream_t st) {
  const long long pieces = gdn_pieces(a.s.total, a.s.n_seq, N);
  hipLaunchKernelGGL((prep_kernel<TX, D>), dim3((unsigned)(pieces * a.nkh)), dim3(64 * PREP_WAVES), 0, st, a, w);
  // Waves of a workgroup: the fewest with which the workgroups have a CU each.  Few waves beside each other are faster
  // (1024 rows of 48 heads of 128 in bf16, both launches: 63 us with two, 71 with four, 91 with eight), two workgroups on a
  // CU are not (two such sequences: 116, 82, 104).  Past that all of a head's columns: a record then comes once, and two of
  // the chain's waves share a SIMD (four: 177, 147, 119; 48: 2058, 1365, 1179).  Short sequences are the same: 8 of 64 rows
  // 54, 38, 37; 40 of 16 rows 194, 103, 92; 40 of 256 rows 564, 359, 315.  (Workgroups of eight have a CU each, so one head
  // more than there are CUs is a second round: five sequences 133, six 212.)  Eight waves of f32 operands do not fit the
  // registers.
  constexpr int MANY = D == 128 && sizeof(TX) == 2 ? 8 : 4, CUS = 256;
  const long long heads = (long long)a.s.n_seq * a.nvh;
  if (heads * (D / 32) <= CUS) launch_chain<TX, TO, D, 2>(a, w, st);
  else if (heads * (D / 64) <= CUS) launch_chain<TX, TO, D, 4>(a, w, st);
  else launch_chain<TX, TO, D, MANY>(a, w, st);
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

size_t gdn_prompt_bytes(int xtype, int D, int nkh, int nvh, int n_seq, int total) {
  size_t key, head;
  sizes_of(xtype, D, &key, &head);
  return (size_t)gdn_pieces(total, n_seq, N) * (nkh * key + nvh * head);
}

int gdn_prompt_launch(int xtype, int otype, int D, const GdnRuleArgs &a, void *work, hipStream_t st) {
  size_t key, head;
  sizes_of(xtype, D, &key, &head);
  const PromptWork w = {(char *)work, (char *)work + (size_t)gdn_pieces(a.s.total, a.s.n_seq, N) * a.nkh * key};
  if (xtype == CWEN_T_F32) launch_o<float>(otype, D, a, w, st);
  else if (xtype == CWEN_T_F16) launch_o<TypeF16::elem>(otype, D, a, w, st);
  else launch_o<TypeBF16::elem>(otype, D, a, w, st);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
