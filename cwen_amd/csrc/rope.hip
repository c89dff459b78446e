// Rotary positions: one tensor's heads, or a step's queries, keys and values
// with the write into the paged cache.
//
// The turn of pair i at position p is p * turns[i] whole circles.  The product
// is taken and reduced to (-1/2, 1/2] in f64 (at p = 2^31 the reduced angle
// still holds 2^-22 of a circle), the sine and cosine in f32.  A workgroup
// computes them once per token into LDS and turns every head with them; an f64
// product per head instead would cost as much as the head's memory traffic.
// Memory bound past a few hundred tokens: every element is read and written
// once, 8 at a time.
#include "cwen_internal.h"
#include "kv_table.h"

namespace {

constexpr int THREADS = 256;

struct RopeTab {
  double turns[128];
  float mscale;
  int D, n_rot;
};

template <typename T> struct Io;
template <> struct Io<float> {
  static __device__ __forceinline__ void load(const float *p, float (&x)[8]) {
    const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  static __device__ __forceinline__ void store(float *p, const float (&x)[8]) {
    *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
    *(float4 *)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  }
};
template <typename T, typename V> struct Io16 {
  static __device__ __forceinline__ void load(const T *p, float (&x)[8]) {
    const V a = *(const V *)p;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)a[j];
  }
  static __device__ __forceinline__ void store(T *p, const float (&x)[8]) {
    V a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = (T)x[j];
    *(V *)p = a;
  }
};
template <> struct Io<TypeF16::elem> : Io16<TypeF16::elem, TypeF16::vec8> {};
template <> struct Io<TypeBF16::elem> : Io16<TypeBF16::elem, TypeBF16::vec8> {};

__device__ __forceinline__ void turn(float &x, float &y, float2 cs) {
  const float a = x * cs.x - y * cs.y;
  y = x * cs.y + y * cs.x;
  x = a;
}

// Grid (tokens, row groups).  A row is one head of the token: its work items are
// 8 elements of the passed-through tail or of the turned part, with HALVES two
// times 8 (both ends of 8 pairs).  One token to a workgroup and its heads over as
// many as give every thread one item.  A decode step of 32 heads takes 3.0 us, a launch's
// own length; 8192 tokens of 32/8 heads of 128 in bf16 38 us (201 MB, 5.2 TB/s: a large
// copy reaches 4.8).  With several tokens to a workgroup the divisions cost 10 us there.
template <typename TX, typename TY, bool HALVES>
__global__ __launch_bounds__(THREADS) void rope_kernel(RopeParams p, RopeTab tab) {
  __shared__ float2 s_cs[128];
  const int np = tab.n_rot / 2, D = tab.D, t = blockIdx.x;
  if (threadIdx.x < np) {
    const double a = (double)p.pos[t] * tab.turns[threadIdx.x];
    float sn, cs;
    sincospif(2.f * (float)(a - rint(a)), &sn, &cs);
    s_cs[threadIdx.x] = make_float2(cs * tab.mscale, (p.inverse ? -sn : sn) * tab.mscale);
  }
  long long row = -1;            // element offset of the token's cache row of head 0; < 0: none
  if (p.k) {
    const int s = p.seq[t], slot = p.slot[t];
    if (slot >= 0) {
      bool bad = (unsigned)s >= (unsigned)p.kv.max_seqs;
      if (!bad) {
        const int i = slot / p.kv.page;
        bad = i >= kv_held_ok(p.kv.held[s], p.kv.max_pages, &bad);
        if (!bad) {
          const int pg = kv_page_ok(p.kv.table[(size_t)s * p.kv.max_pages + i], p.kv.n_pages, &bad);
          if (p.kv.ref[pg] != 1) bad = true;
          row = kv_at(p.layer, pg, 0, slot - i * p.kv.page, p.kv.n_pages, p.kv.n_kv_head, p.kv.page, D);
        }
      }
      if (bad) {
        row = -1;
        if (blockIdx.y == 0 && threadIdx.x == 0) kv_raise(p.kv, CWEN_KV_ARG);
      }
    }
  }
  __syncthreads();

  const int n_kv = p.k ? p.kv.n_kv_head : 0, H = p.nh + 2 * n_kv;
  const int turned = HALVES ? tab.n_rot / 16 : tab.n_rot / 8;
  const int items = turned + (D - tab.n_rot) / 8;          // of one row
  const int per = THREADS / items;                          // rows side by side
  const int c = threadIdx.x % items;
  for (int h = blockIdx.y * per + threadIdx.x / items; h < H; h += gridDim.y * per) {
    if ((int)threadIdx.x >= per * items) break;
    const TX *src;
    TY *dst;
    bool rot = c < turned;
    if (h < p.nh) {
      src = (const TX *)p.q + t * p.q_ts + h * p.q_hs;
      dst = (TY *)p.qo + t * p.qo_ts + h * p.qo_hs;
    } else {
      if (row < 0) continue;
      const bool isv = h >= p.nh + n_kv;
      const int hk = h - p.nh - (isv ? n_kv : 0);
      src = isv ? (const TX *)p.v + t * p.v_ts + (long long)hk * D : (const TX *)p.k + t * p.k_ts + (long long)hk * D;
      dst = (TY *)(isv ? p.kv.v : p.kv.k) + row + (long long)hk * p.kv.page * D;
      rot = rot && !isv;
    }
    float x[8];
    if (HALVES) {
      if (c < turned) {
        float y[8];
        Io<TX>::load(src + 8 * c, x);
        Io<TX>::load(src + np + 8 * c, y);
        if (rot)
#pragma unroll
          for (int j = 0; j < 8; ++j) turn(x[j], y[j], s_cs[8 * c + j]);
        Io<TY>::store(dst + 8 * c, x);
        Io<TY>::store(dst + np + 8 * c, y);
      } else {
        const int d = tab.n_rot + 8 * (c - turned);
        Io<TX>::load(src + d, x);
        Io<TY>::store(dst + d, x);
      }
    } else {
      Io<TX>::load(src + 8 * c, x);
      if (rot)
#pragma unroll
        for (int j = 0; j < 4; ++j) turn(x[2 * j], x[2 * j + 1], s_cs[4 * c + j]);
      Io<TY>::store(dst + 8 * c, x);
    }
  }
}

template <typename TX, typename TY>
void launch(bool halves, dim3 g, const RopeParams &p, const RopeTab &t, hipStream_t st) {
  if (halves) hipLaunchKernelGGL((rope_kernel<TX, TY, true>), g, dim3(THREADS), 0, st, p, t);
  else hipLaunchKernelGGL((rope_kernel<TX, TY, false>), g, dim3(THREADS), 0, st, p, t);
}
template <typename TX>
void launch_y(int ytype, bool halves, dim3 g, const RopeParams &p, const RopeTab &t, hipStream_t st) {
  if (ytype == CWEN_T_F32) launch<TX, float>(halves, g, p, t, st);
  else if (ytype == CWEN_T_F16) launch<TX, TypeF16::elem>(halves, g, p, t, st);
  else launch<TX, TypeBF16::elem>(halves, g, p, t, st);
}

}  // namespace

int rope_launch(const cwen_rope *r, int xtype, int ytype, const RopeParams &p, hipStream_t st) {
  RopeTab t;
  for (int i = 0; i < r->n_rot / 2; ++i) t.turns[i] = r->turns[i];
  t.mscale = r->mscale;
  t.D = r->head_dim;
  t.n_rot = r->n_rot;
  const int rows = p.nh + (p.k ? 2 * p.kv.n_kv_head : 0);
  const int per = THREADS * 8 / r->head_dim;
  const dim3 g((unsigned)p.T, (unsigned)((rows + per - 1) / per));
  const bool halves = r->layout == CWEN_ROPE_HALVES;
  if (xtype == CWEN_T_F32) launch_y<float>(ytype, halves, g, p, t, st);
  else if (xtype == CWEN_T_F16) launch_y<TypeF16::elem>(ytype, halves, g, p, t, st);
  else launch_y<TypeBF16::elem>(ytype, halves, g, p, t, st);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
