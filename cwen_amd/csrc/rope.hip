// Rotary positions: one tensor's heads, or a step's queries, keys and values
// with the write into the paged cache.
//
// The turn of pair i at position p is p * turns[i] whole circles.  The product
// is taken and reduced to (-1/2, 1/2] in f64, the sine and cosine in f32.  turns[i] <=
// 1 / 2 pi carries about a dozen roundings of 2^-53 (its power, scaling, division) and the
// product one: p 2^-52 of a circle at most, 2^-21 at the last position, and less than the
// rounding to f32 (2^-26 of a circle) up to position 2^26.  A workgroup
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
  int tok;                       // tokens of a workgroup
};

__device__ __forceinline__ void turn(float &x, float &y, float2 cs) {
  const float a = x * cs.x - y * cs.y;
  y = x * cs.y + y * cs.x;
  x = a;
}

// Work items of a row, one head of a token: 8 elements of the passed-through tail or
// of the turned part, with HALVES two times 8 (both ends of 8 pairs).
__host__ __device__ constexpr int rope_items(int D, int n_rot, bool halves) { return (D - n_rot) / 8 + n_rot / (halves ? 16 : 8); }

// A thread has one item.  Grid (tokens, row groups), or, where the rows of three tokens and
// more fit a workgroup, (groups of tok tokens, 1): about one workgroup starts a ns, so 8192
// tokens of 5/1 heads of 128 take 9.3 us instead of 13.6, 100000 of one head of 64 12 instead
// of 56 (two tokens to a workgroup lose to one in f32: 16 heads of 64 15 against 12.5).  A
// decode step of 32 heads takes 3.2 us, a launch's own length; 8192 tokens of 32/8
// heads of 128 in bf16 32 us (201 MB, 6.3 TB/s: a copy of 256 MiB reaches 5.4, a plain kernel 6.2).
template <typename TX, typename TY, bool HALVES, bool GROUP>
__global__ __launch_bounds__(THREADS) void rope_kernel(RopeParams p, RopeTab tab) {
  __shared__ float2 s_cs[GROUP ? 2048 : 128];   // tok n_rot / 2 <= 256 / items * 8 items
  const int np = tab.n_rot / 2, D = tab.D, tok = GROUP ? tab.tok : 1, t0 = blockIdx.x * tok, nt = min(tok, p.T - t0);
  const int items = rope_items(D, tab.n_rot, HALVES), per = THREADS / items, turned = tab.n_rot / (HALVES ? 16 : 8);
  const int n_kv = p.k ? p.kv.n_kv_head : 0, H = p.nh + 2 * n_kv;
  const int r = threadIdx.x / items, c = threadIdx.x - r * items, lt = GROUP ? r / H : 0, t = t0 + lt;
  const int h = GROUP ? r - lt * H : blockIdx.y * per + r;
  const bool live = (int)threadIdx.x < per * items && h < H && lt < nt, both = HALVES && c < turned;
  const int d = HALVES && !both ? tab.n_rot + 8 * (c - turned) : 8 * c;      // the first element
  float x[8], y[8];
  auto load = [&]() {
    const int hk = h - p.nh;
    const TX *src = hk < 0 ? (const TX *)p.q + t * p.q_ts + h * p.q_hs
                    : hk < n_kv ? (const TX *)p.k + t * p.k_ts + (long long)hk * D : (const TX *)p.v + t * p.v_ts + (long long)(hk - n_kv) * D;
    Io<TX>::load(src + d, x);
    if (both) Io<TX>::load(src + np + d, y);
  };
  if (GROUP && live) load();
  for (int i = threadIdx.x; i < nt * np; i += THREADS) {
    const int u = GROUP ? i / np : 0;
    const double a = (double)p.pos[t0 + u] * tab.turns[i - u * np];
    float sn, cs;
    sincospif(2.f * (float)(a - rint(a)), &sn, &cs);
    s_cs[i] = make_float2(cs * tab.mscale, (p.inverse ? -sn : sn) * tab.mscale);
  }
  long long row = -1;            // element offset of the token's cache row of head 0; < 0: none
  if (p.k && live) {
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
        if (h == 0 && c == 0) kv_raise(p.kv, CWEN_KV_ARG);
      }
    }
  }
  __syncthreads();
  if (!live || (h >= p.nh && row < 0)) return;
  if (!GROUP) load();
  const int hk = h - p.nh;
  const bool isv = hk >= n_kv;
  TY *dst = hk < 0 ? (TY *)p.qo + t * p.qo_ts + h * p.qo_hs
                   : (TY *)(isv ? p.kv.v : p.kv.k) + row + (long long)(hk - (isv ? n_kv : 0)) * p.kv.page * D;
  if (c < turned && !(hk >= 0 && isv)) {
    if (HALVES)
#pragma unroll
      for (int j = 0; j < 8; ++j) turn(x[j], y[j], s_cs[lt * np + 8 * c + j]);
    else
#pragma unroll
      for (int j = 0; j < 4; ++j) turn(x[2 * j], x[2 * j + 1], s_cs[lt * np + 4 * c + j]);
  }
  Io<TY>::store(dst + d, x);
  if (both) Io<TY>::store(dst + np + d, y);
}

template <typename TX, typename TY>
void launch(bool halves, dim3 g, const RopeParams &p, const RopeTab &t, hipStream_t st) {
  if (halves) {
    if (t.tok > 1) hipLaunchKernelGGL((rope_kernel<TX, TY, true, true>), g, dim3(THREADS), 0, st, p, t);
    else hipLaunchKernelGGL((rope_kernel<TX, TY, true, false>), g, dim3(THREADS), 0, st, p, t);
  } else {
    if (t.tok > 1) hipLaunchKernelGGL((rope_kernel<TX, TY, false, true>), g, dim3(THREADS), 0, st, p, t);
    else hipLaunchKernelGGL((rope_kernel<TX, TY, false, false>), g, dim3(THREADS), 0, st, p, t);
  }
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
  const int per = THREADS / rope_items(r->head_dim, r->n_rot, r->layout == CWEN_ROPE_HALVES);
  t.tok = per / rows >= 3 ? per / rows : 1;
  const dim3 g((unsigned)((p.T + t.tok - 1) / t.tok), (unsigned)((rows + per - 1) / per));
  const bool halves = r->layout == CWEN_ROPE_HALVES;
  if (xtype == CWEN_T_F32) launch_y<float>(ytype, halves, g, p, t, st);
  else if (xtype == CWEN_T_F16) launch_y<TypeF16::elem>(ytype, halves, g, p, t, st);
  else launch_y<TypeBF16::elem>(ytype, halves, g, p, t, st);
  CWEN_HIP_TRY(hipGetLastError());
  return CWEN_OK;
}
