// The tile of prompt and tree attention: one wave's query rows against BN
// keys whose K and V rows lie in LDS.
//
// The scores are taken transposed, S^T = K Q^T (v_mfma_f32_32x32x16, K the
// left operand): lane (n = lane & 31, hi = lane >> 5) then holds 16 scores of
// query n per 32 keys, namely of the keys 8 i + 4 hi + j (i, j < 4).  So the
// softmax's maximum and sum run over a lane's own registers with one exchange
// between the wave's halves, and the probabilities are already where the next
// product wants them: O^T = V^T P^T, P^T the right operand, whose lane (n, hi)
// supplies 8 keys of query n.  A product's keys may be taken in any order as
// long as both operands agree; V^T's lanes read the matching keys, 4 and 4,
// with transposing LDS reads (ds_read_b64_tr_b16).
//
// Rows in LDS are D elements without padding (they arrive by loads that land
// there directly); their 16-byte pieces are permuted instead, so that lanes that
// read the same piece of different rows hit different banks.
#pragma once
#include <math.h>
#include "cwen_internal.h"

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void attn_lds_t;
typedef const __attribute__((address_space(1))) void attn_glb_t;

template <typename T> struct AttnOps;
template <> struct AttnOps<TypeF16> {
  typedef TypeF16::vec8 vec8;
  typedef _Float16 vec4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x16_t mma(vec8 a, vec8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ vec4 tr(const void *p) {
    typedef __fp16 v4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(
        vec4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) v4 *)(attn_lds_t *)const_cast<void *>(p)));
  }
  // NaN when an element is not finite (times 0).
  static __device__ __forceinline__ float probe(vec8 v, float acc) {
    const half2_t z = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2) acc = __builtin_amdgcn_fdot2((half2_t){v[i], v[i + 1]}, z, acc, false);
    return acc;
  }
};
template <> struct AttnOps<TypeBF16> {
  typedef TypeBF16::vec8 vec8;
  typedef __bf16 vec4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x16_t mma(vec8 a, vec8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ vec4 tr(const void *p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) vec4 *)(attn_lds_t *)const_cast<void *>(p));
  }
  static __device__ __forceinline__ float probe(vec8 v, float acc) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    const v2 z = {(__bf16)0.f, (__bf16)0.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) acc = __builtin_amdgcn_fdot2_f32_bf16((v2){v[i], v[i + 1]}, z, acc, false);
    return acc;
  }
};

// Wait until at most N of the wave's loads are under way.  The builtin and not
// asm: the compiler then knows that the older ones have landed and adds no
// wait of its own before it reads them from LDS (vmcnt(0) there, which would
// also wait for the next tile, took a third of the tree attention's time).
template <int N> __device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 0x70 | 0xF00 | (N >> 4) << 14);   // gfx9 encoding: vmcnt(N), the others unchanged
  asm volatile("" ::: "memory");
}

// Pieces (16 bytes) of a row, and where piece c of row r is kept.
template <int D> __device__ __forceinline__ constexpr int k_piece(int r, int c) { return c ^ (r & (D >= 128 ? 15 : 7)); }
template <int D> __device__ __forceinline__ constexpr int v_piece(int r, int c) {
  return c ^ (D >= 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2);
}

__device__ __forceinline__ float max_halves(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (int)p[0]), __builtin_bit_cast(float, (int)p[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  return __builtin_bit_cast(float, (int)p[0]) + __builtin_bit_cast(float, (int)p[1]);
}

// The maximum a row's exponents are taken against is renewed only when a row
// outgrew it by more than 2^8: the probabilities stay below 2^8 (f16 holds
// 65504), and most tiles then leave the output sums alone.
constexpr float ATTN_SLACK = 8.f;

// A wave holds 32 query rows.  64 of them, which would read each fragment from LDS half as
// often, do not fit the registers with heads of 256 and gain nothing with shorter ones: the
// reads are hidden behind the products.
template <typename T, int D, int BN> struct AttnWave {
  typedef typename T::elem elem;
  typedef typename AttnOps<T>::vec8 vec8;
  typedef typename AttnOps<T>::vec4 vec4;
  static constexpr int QS = D / 16, OB = D / 32, KB = BN / 32;

  vec8 q[QS];            // dims 16 s + 8 hi .. + 7 of query n
  f32x16_t o[OB];        // [i]: output dims 32 b + 8 (i / 4) + 4 hi + i % 4 of query n
  float m, l;            // maximum (in powers of two) and this lane's part of the sum
  float odd;             // NaN once a partly hidden tile held a value that is not finite

  // row: the elements of query n, null for a row that does not exist
  __device__ __forceinline__ void start(const elem *row) {
    const int hi = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int s = 0; s < QS; ++s) q[s] = row ? *(const vec8 *)(row + 16 * s + 8 * hi) : vec8{};
#pragma unroll
    for (int b = 0; b < OB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.f;
    m = -INFINITY;
    l = odd = 0.f;
  }

  // The scores of one tile, K the LDS array of its BN rows.
  __device__ __forceinline__ void scores(const elem *K, f32x16_t (&s)[KB]) {
    const int lane = threadIdx.x & 63, n = lane & 31, hi = lane >> 5;
    // Byte of piece hi of row n; piece 2 k + hi is an exclusive or away (k_piece).
    // Opaque, so that the addresses are formed when they are used: kept, they
    // would cost the registers that hold fragments on their way.
    uint32_t at = (uint32_t)(n * D * 2 + 16 * k_piece<D>(n, hi));
    asm("" : "+v"(at));
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
    for (int k = 0; k < QS; ++k)
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const vec8 kf = *(const vec8 *)((const char *)K + (at ^ (32u * (k & 7))) + 256 * (k >> 3) + b * 64 * D);
        s[b] = AttnOps<T>::mma(kf, q[k], s[b]);
      }
  }
  // Their softmax against the row's maximum so far.  c: scale * log2(e).  HIDE:
  // hide(j) tells whether this lane's query does not see key j + 4 hi of
  // the tile (j is a constant then: with 4 hi in it the compiler kept 16 masks in registers).
  template <bool HIDE, typename F>
  __device__ __forceinline__ void soft(f32x16_t (&s)[KB], float c, F hide, vec8 (&p)[2 * KB]) {
    if (HIDE) {
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (hide(b * 32 + 8 * (i >> 2) + (i & 3))) s[b][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
    mx = max_halves(mx) * c;
    if (__any(mx > m + ATTN_SLACK)) {
      const float mn = fmaxf(m, mx), a = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= a;
#pragma unroll
      for (int b = 0; b < OB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= a;
      m = mn;
    }
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, -ms));
        l += e;
        p[2 * b + (i >> 3)][i & 7] = (elem)e;     // half a step; the sum keeps all of it
      }
  }
  // The outputs' sums, V the LDS array of the tile's rows.  Lane i of a group of
  // 16 addresses the 4 keys' rows 4 g + i / 4 and gets column i of all 4.
  template <bool HIDE> __device__ __forceinline__ void outputs(const elem *V, const vec8 (&p)[2 * KB]) {
    const int lane = threadIdx.x & 63, hi = lane >> 5;
    const int vi = lane & 15, vr = 4 * hi + (vi >> 2), vc = ((lane >> 4) & 1) * 2 + ((vi & 3) >> 1), ve = (vi & 1) * 4;
    uint32_t at = (uint32_t)(vr * D * 2 + 16 * v_piece<D>(vr, vc) + 2 * ve);
    asm("" : "+v"(at));
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
      for (int b = 0; b < OB; ++b) {
        const char *r = (const char *)V + (at ^ (64u * (b & 3))) + 256 * (b >> 2) + 32 * t * D;
        const vec4 a = AttnOps<T>::tr(r), d = AttnOps<T>::tr(r + 16 * D);
        const vec8 vf = {a[0], a[1], a[2], a[3], d[0], d[1], d[2], d[3]};
        if (HIDE) odd = AttnOps<T>::probe(vf, odd);
        o[b] = AttnOps<T>::mma(vf, p[t], o[b]);
      }
  }
  template <bool HIDE, typename F> __device__ __forceinline__ void tile(const elem *K, const elem *V, float c, F hide) {
    f32x16_t s[KB];
    vec8 p[2 * KB];
    scores(K, s);
    soft<HIDE>(s, c, hide, p);
    outputs<HIDE>(V, p);
  }

  // The whole row's sum.
  __device__ __forceinline__ float sum() const { return sum_halves(l); }
};

// Rows t0 .. t0 + BN - 1 into LDS, by NW waves; rows past `last` are copies of
// it (never what lies behind them).  A wave's load takes 64 / (D / 8) rows that
// follow each other at `stride` bytes in memory and lie one after the other in
// LDS; row(i, j) gives the address of row j, the first of the wave's i-th load, the same for all
// lanes: it stays in scalar registers, and a lane adds 32 bits of its own.
template <int D, int BN, bool ISV, int NW, typename elem, typename F>
__device__ __forceinline__ void land_rows(elem *dst, int wave, int t0, int last, uint32_t stride, F row) {
  constexpr int C = D / 8, RI = 64 / C;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < BN / (RI * NW); ++i) {
    const int x0 = (i * NW + wave) * RI, j = min(t0 + x0, last);
    const char *base = (const char *)row(i, j);
    const int x = x0 + lane / C, p = lane % C;
    const uint32_t off = (uint32_t)min(lane / C, last - j) * stride + 16u * (ISV ? v_piece<D>(x, p) : k_piece<D>(x, p));
    __builtin_amdgcn_global_load_lds((attn_glb_t *)(base + off), (attn_lds_t *)(dst + x0 * D), 16, 0, 0);
  }
}
