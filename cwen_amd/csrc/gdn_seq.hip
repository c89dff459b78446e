// The GatedDeltaNet layers of many sequences: the causal convolution over packed
// rows, and the delta rule row after row.
#include "gdn_seq.h"

namespace {

// x / (1 + exp(-x)) with the hardware's exp2 and reciprocal, each off by an ulp.  With the exact division the
// convolution is bound by its instructions (8192 rows of 10240 channels in bf16: 108 us instead of 84).
__device__ __forceinline__ float silu_near(float x) {
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * x));
}

// ---- convolution ----
// A thread has 8 channels of the TB rows of one piece, the last three inputs
// and the taps in registers, so that a row is read once by its own piece and the
// three before it by the next.  Bound by memory (8192 rows of 10240 channels
// in bf16: 84 us, 4.0 TB/s).  The first piece also moves
// the history: the thread that reads the old one writes the new one, after it.
constexpr int CONV_TB = 32, CONV_THREADS = 128;

template <typename TX, typename TY> __global__ __launch_bounds__(CONV_THREADS) void conv_kernel(GdnConvArgs a) {
  const int c = (blockIdx.y * CONV_THREADS + threadIdx.x) * 8;
  const int s = gdn_find(a.s, blockIdx.x, CONV_TB);
  if (s < 0) return;
  GdnSeq q = gdn_seq(a.s, s);
  const int t0 = ((int)blockIdx.x - gdn_piece0(q.first, s, CONV_TB)) * CONV_TB;
  if (t0 < 0 || (t0 > 0 && t0 >= q.n)) return;
  if (!q.ok || gdn_taken(a.s, s, q.dst)) {
    gdn_raise(a.s);
    return;
  }
  if (c >= a.C) return;
  const TX *x = (const TX *)a.x + (long long)q.first * a.xs + c;
  const float *h0 = q.src >= 0 ? a.hist + ((long long)q.src * a.C + c) * 3 : nullptr;
  float past[24];           // [channel][input]: the history
#pragma unroll
  for (int i = 0; i < 24; ++i) past[i] = 0.f;
  if (h0 && t0 == 0) {
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const float4 f = *(const float4 *)(h0 + 4 * i);
      past[4 * i] = f.x; past[4 * i + 1] = f.y; past[4 * i + 2] = f.z; past[4 * i + 3] = f.w;
    }
  }
  if (a.y) {
    float in[3][8];
    float4 w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = *(const float4 *)(a.kw + (long long)(c + e) * 4);
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      if (t0) {
        Io<TX>::load(x + (long long)(t0 - 3 + j) * a.xs, in[j]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) in[j][e] = past[3 * e + j];
      }
    }
    TY *y = (TY *)a.y + (long long)q.first * a.ys + c;
    const int end = min(t0 + CONV_TB, q.n);
#pragma unroll 4
    for (int t = t0; t < end; ++t) {
      float cur[8], out[8];
      Io<TX>::load(x + (long long)t * a.xs, cur);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        out[e] = silu_near(conv4(in[0][e], in[1][e], in[2][e], cur[e], w[e]));
        in[0][e] = in[1][e];
        in[1][e] = in[2][e];
        in[2][e] = cur[e];
      }
      Io<TY>::store(y + (long long)t * a.ys, out);
    }
  }
  if (t0 == 0 && q.dst >= 0) {
    float last[3][8];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int t = q.n - 3 + j;
      if (t >= 0) {
        Io<TX>::load(x + (long long)t * a.xs, last[j]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) last[j][e] = t == -3 ? past[3 * e] : t == -2 ? past[3 * e + 1] : past[3 * e + 2];
      }
    }
    float *h1 = a.hist + ((long long)q.dst * a.C + c) * 3;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      float f[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) f[u] = last[(4 * i + u) % 3][(4 * i + u) / 3];
      *(float4 *)(h1 + 4 * i) = make_float4(f[0], f[1], f[2], f[3]);
    }
  }
}

// ---- delta rule ----
// A wave has 32 columns of one value head's state; the rule is local to a
// column.  Lane (rg = lane >> 3, cg = lane & 7) holds rows rg R .. of 4 columns
// (R = D / 8), so a load takes whole 128-byte lines and a column's sum is over 8
// lanes 8 apart.  With u = S^T k and w = S^T q of the state before the row,
//   d = beta (v - g u),  o = (g w + (k.q) d) / sqrt(D),  S = g S + k d^T:
// both sums are under way together.  Bound by memory (the state in and out)
// while sequences have a row each (128 of 48 heads of 128: 159 us, 5.1 TB/s), by
// the rows' trips and sums otherwise (24 sequences of 9 rows: 42 us).
__device__ __forceinline__ float sum_rows(float x) {
  x += dpp<0x128>(x);                                            // 8 lanes on, within 16
  const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  x = __builtin_bit_cast(float, (int)p[0]) + __builtin_bit_cast(float, (int)p[1]);
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  return __builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]);
}

template <typename TX, typename TO, int D> __global__ __launch_bounds__(256) void step_kernel(GdnRuleArgs a) {
  constexpr int R = D / 8, SL = D / 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x * 4 + wave, s = item / (SL * a.nvh), rest = item - s * (SL * a.nvh);
  if (s >= a.s.n_seq) return;
  const int hv = rest / SL, slice = rest - hv * SL, hk = a.group ? hv / a.group : hv % a.nkh;
  const int rg = lane >> 3, cg = lane & 7, i0 = rg * R, j0 = slice * 32 + cg * 4;
  GdnSeq q = gdn_seq(a.s, s);
  const bool ok = q.ok && !gdn_taken(a.s, s, q.dst);
  if (!ok) {
    gdn_raise(a.s);
    return;
  }
  if (q.n == 0 && (q.dst < 0 || q.dst == q.src)) return;
  const long long head = (long long)hv * D * D + i0 * D + j0, slot = (long long)a.nvh * D * D;
  float4 S[R];
#pragma unroll
  for (int r = 0; r < R; ++r) S[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (q.src >= 0) {
    const float *p = a.state + q.src * slot + head;
#pragma unroll
    for (int r = 0; r < R; ++r) S[r] = *(const float4 *)(p + r * D);
  }
  const TX *qp = (const TX *)a.q + (long long)q.first * a.qs + hk * D + i0;
  const TX *kp = (const TX *)a.k + (long long)q.first * a.ks + hk * D + i0;
  const TX *vp = (const TX *)a.v + (long long)q.first * a.vs + hv * D + j0;
  const float *ap = a.a + (long long)q.first * a.gs + hv, *bp = a.b + (long long)q.first * a.gs + hv;
  const float scale = 1.f / sqrtf((float)D);
  typedef TX vec4 __attribute__((ext_vector_type(4)));
  // A row's operands are asked for while the row before is computed, its gates with those of 64 rows, one a lane.
  float k1[R], x1[R];
  vec4 v1 = {};
  float g64 = 0.f, beta64 = 0.f;
  auto ask = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < R; r += 8) {
      Io<TX>::load(kp + t * a.ks + r, *(float(*)[8])&k1[r]);
      Io<TX>::load(qp + t * a.qs + r, *(float(*)[8])&x1[r]);
    }
    v1 = *(const vec4 *)(vp + t * a.vs);
  };
  if (q.n) ask(0);
  for (int t = 0; t < q.n; ++t) {
    if ((t & 63) == 0) {
      const int u = min(t + lane, q.n - 1);
      g64 = ap[u * a.gs];
      beta64 = bp[u * a.gs];
      if (a.A) {
        const float y = g64 + a.dt[hv];
        g64 = a.A[hv] * (y > 20.f ? y : log1pf(expf(y)));
        beta64 = 1.f / (1.f + expf(-beta64));
      }
      g64 = expf(g64);
    }
    const float g = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, g64), t & 63));
    const float beta = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, beta64), t & 63));
    float k[R], x[R];
    const vec4 v = v1;
#pragma unroll
    for (int r = 0; r < R; ++r) k[r] = k1[r], x[r] = x1[r];
    if (t + 1 < q.n) ask(t + 1);
    float kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      kk = fmaf(k[r], k[r], kk);
      qq = fmaf(x[r], x[r], qq);
      kq = fmaf(k[r], x[r], kq);
    }
    const float kn = 1.f / sqrtf(sum_rows(kk) + 1e-6f);
    float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      u.x = fmaf(S[r].x, k[r], u.x); u.y = fmaf(S[r].y, k[r], u.y); u.z = fmaf(S[r].z, k[r], u.z); u.w = fmaf(S[r].w, k[r], u.w);
    }
    const float gk = g * kn;
    float4 d;
    d.x = beta * ((float)v[0] - gk * sum_rows(u.x)); d.y = beta * ((float)v[1] - gk * sum_rows(u.y));
    d.z = beta * ((float)v[2] - gk * sum_rows(u.z)); d.w = beta * ((float)v[3] - gk * sum_rows(u.w));
    if (a.o) {
      float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        w.x = fmaf(S[r].x, x[r], w.x); w.y = fmaf(S[r].y, x[r], w.y); w.z = fmaf(S[r].z, x[r], w.z); w.w = fmaf(S[r].w, x[r], w.w);
      }
      const float qn = 1.f / sqrtf(sum_rows(qq) + 1e-6f), gq = g * qn, c = sum_rows(kq) * kn * qn;
      w = make_float4(sum_rows(w.x), sum_rows(w.y), sum_rows(w.z), sum_rows(w.w));
      if (rg == 0) {
        typedef TO out4 __attribute__((ext_vector_type(4)));
        *(out4 *)((TO *)a.o + (long long)(q.first + t) * a.os + hv * D + j0) =
            (out4){(TO)(scale * fmaf(gq, w.x, c * d.x)), (TO)(scale * fmaf(gq, w.y, c * d.y)),
                   (TO)(scale * fmaf(gq, w.z, c * d.z)), (TO)(scale * fmaf(gq, w.w, c * d.w))};
      }
    }
    if (t + 1 == q.n && q.dst < 0) return;          // the last row's state is nobody's
    d.x *= kn; d.y *= kn; d.z *= kn; d.w *= kn;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      S[r].x = fmaf(k[r], d.x, g * S[r].x); S[r].y = fmaf(k[r], d.y, g * S[r].y);
      S[r].z = fmaf(k[r], d.z, g * S[r].z); S[r].w = fmaf(k[r], d.w, g * S[r].w);
    }
  }
  if (q.dst >= 0) {
    float *p = a.state + q.dst * slot + head;
#pragma unroll
    for (int r = 0; r < R; ++r) *(float4 *)(p + r * D) = S[r];
  }
}

template <typename TX, typename TO> void launch_conv(const GdnConvArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)gdn_pieces(a.s.total, a.s.n_seq, CONV_TB), (unsigned)((a.C / 8 + CONV_THREADS - 1) / CONV_THREADS));
  hipLaunchKernelGGL((conv_kernel<TX, TO>), grid, dim3(CONV_THREADS), 0, st, a);
}
template <typename TX, typename TO> void launch_step(int D, const GdnRuleArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)(((long long)a.s.n_seq * a.nvh * (D / 32) + 3) / 4));
  if (D == 128) hipLaunchKernelGGL((step_kernel<TX, TO, 128>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((step_kernel<TX, TO, 64>), grid, dim3(256), 0, st, a);
}

typedef TypeF16::elem f16;
typedef TypeBF16::elem bf16;

// f(X{}, Y{}) with the element types of two CWEN_T_* (checked before).
template <typename TX, typename F> void with_out(int t, F f) {
  if (t == CWEN_T_F32) f(TX{}, float{});
  else if (t == CWEN_T_F16) f(TX{}, f16{});
  else f(TX{}, bf16{});
}
template <typename F> void with_types(int x, int y, F f) {
  if (x == CWEN_T_F32) with_out<float>(y, f);
  else if (x == CWEN_T_F16) with_out<f16>(y, f);
  else with_out<bf16>(y, f);
}

}  // namespace

int gdn_conv_launch(int xtype, int ytype, const GdnConvArgs &a, hipStream_t st) {
  with_types(xtype, ytype, [&](auto x, auto y) { launch_conv<decltype(x), decltype(y)>(a, st); });
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}

int gdn_step_launch(int xtype, int otype, int D, const GdnRuleArgs &a, hipStream_t st) {
  with_types(xtype, otype, [&](auto x, auto o) { launch_step<decltype(x), decltype(o)>(D, a, st); });
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
