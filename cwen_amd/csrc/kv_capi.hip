// C ABI entry points of the serving operators: rotary positions, the paged
// cache, prompt and tree attention.  Argument checks; nothing here touches the
// GPU before they have passed.
#include <math.h>
#include <stdlib.h>
#include "capi_checks.h"

namespace {

int check_kv(const cwen_kv *kv) {
  if (!kv) return CWEN_EINVAL;
  if (kv->type != CWEN_T_F16 && kv->type != CWEN_T_BF16) return CWEN_ETYPE;
  if (kv->n_layers < 1 || kv->n_layers > 32767 || kv->n_kv_head < 1 || kv->n_kv_head > 65535) return CWEN_EINVAL;
  if (kv->head_dim < 8 || kv->head_dim > 512 || kv->head_dim % 8) return CWEN_EINVAL;
  if (kv->page < 16 || kv->page > 256 || (kv->page & (kv->page - 1))) return CWEN_EINVAL;
  if (kv->n_pages < 1 || kv->n_pages > (1 << 24) || kv->max_seqs < 1 || kv->max_seqs > 65536) return CWEN_EINVAL;
  if (kv->max_pages < 1 || (long long)kv->max_pages * kv->page >= 1ll << 30) return CWEN_EINVAL;
  if ((long long)kv->max_pages * kv->max_seqs > INT32_MAX) return CWEN_EINVAL;
  if (!kv->k || !kv->v || !aligned16(kv->k) || !aligned16(kv->v)) return CWEN_EINVAL;
  if (!kv->table || !kv->len || !kv->held || !kv->ref || !kv->work || !kv->status) return CWEN_EINVAL;
  if (!aligned16(kv->ref) || !aligned4(kv->table) || !aligned4(kv->len) || !aligned4(kv->held) || !aligned4(kv->work) ||
      !aligned4(kv->status))
    return CWEN_EINVAL;
  return CWEN_OK;
}
// n_req requests over `a` (and `b`): an empty call is CWEN_OK without a launch.
int check_req(const cwen_ctx *ctx, const cwen_kv *kv, const void *a, const void *b, int n_req) {
  if (!ctx) return CWEN_EINVAL;
  const int rc = check_kv(kv);
  if (rc) return rc;
  if (n_req < 0 || n_req > CWEN_KV_REQ_MAX || n_req > kv->max_seqs) return CWEN_EINVAL;
  if (n_req && (!a || !b || !aligned4(a) || !aligned4(b))) return CWEN_EINVAL;
  return CWEN_OK;
}

}  // namespace

extern "C" {

// ------------------------------------------------------------ rotary positions
int cwen_rope_create(const cwen_rope_cfg *c, cwen_rope **out) {
  if (!out) return CWEN_EINVAL;
  *out = nullptr;
  if (!c) return CWEN_EINVAL;
  if (c->layout != CWEN_ROPE_PAIRS && c->layout != CWEN_ROPE_HALVES) return CWEN_EINVAL;
  if (c->scaling < CWEN_ROPE_PLAIN || c->scaling > CWEN_ROPE_YARN) return CWEN_EINVAL;
  if (c->head_dim < 8 || c->head_dim > 512 || c->head_dim % 8) return CWEN_EINVAL;
  if (c->n_rot < 8 || c->n_rot > 256 || c->n_rot > c->head_dim || c->n_rot % (c->layout == CWEN_ROPE_HALVES ? 16 : 8))
    return CWEN_EINVAL;
  if (c->freq_dim < 0 || !(c->theta > 1) || !isfinite(c->theta) || !(c->mscale >= 0) || !isfinite(c->mscale)) return CWEN_EINVAL;
  if (c->scaling != CWEN_ROPE_PLAIN && (!(c->factor >= 1) || !isfinite(c->factor))) return CWEN_EINVAL;
  const double d = c->freq_dim ? c->freq_dim : c->n_rot, two_pi = 6.283185307179586476925;
  double low = 0, high = 0;
  if (c->scaling == CWEN_ROPE_YARN) {
    if (!(c->orig_ctx > 0) || !isfinite(c->orig_ctx) || !(c->beta_slow > 0) || !(c->beta_fast >= c->beta_slow) ||
        !isfinite(c->beta_fast))
      return CWEN_EINVAL;
    low = fmax(floor(d * log(c->orig_ctx / (two_pi * c->beta_fast)) / (2 * log(c->theta))), 0.);
    high = fmin(ceil(d * log(c->orig_ctx / (two_pi * c->beta_slow)) / (2 * log(c->theta))), d - 1);
    if (high == low) high += 0.001;
  }
  cwen_rope *r = (cwen_rope *)calloc(1, sizeof(cwen_rope));
  if (!r) return CWEN_ENOMEM;
  r->head_dim = c->head_dim;
  r->n_rot = c->n_rot;
  r->layout = c->layout;
  r->mscale = c->mscale > 0 ? (float)c->mscale : c->scaling == CWEN_ROPE_YARN ? (float)(0.1 * log(c->factor) + 1) : 1.f;
  for (int i = 0; i < c->n_rot / 2; ++i) {
    double f = pow(c->theta, -2.0 * i / d);
    if (c->scaling == CWEN_ROPE_LINEAR) f /= c->factor;
    if (c->scaling == CWEN_ROPE_YARN) {
      const double ramp = fmin(fmax((i - low) / (high - low), 0.), 1.);
      f = f * (1 - ramp) + f / c->factor * ramp;
    }
    r->turns[i] = f / two_pi;
  }
  *out = r;
  return CWEN_OK;
}
int cwen_rope_free(cwen_rope *r) {
  if (!r) return CWEN_EINVAL;
  free(r);
  return CWEN_OK;
}

int cwen_rope_apply(cwen_ctx *ctx, const cwen_rope *r, int xtype, const void *x, long long x_ts, long long x_hs, int ytype,
                    void *y, long long y_ts, long long y_hs, const int *pos, int T, int n_head, int inverse, void *stream) {
  if (!ctx || !r || T < 0 || T >= 1 << 24 || n_head < 1 || n_head > 65535) return CWEN_EINVAL;
  const int xe = elem_size(xtype), ye = elem_size(ytype);
  if (!xe || !ye) return CWEN_ETYPE;
  if (T == 0) return CWEN_OK;
  if (!x || !y || !pos || !aligned16(x) || !aligned16(y) || !aligned4(pos)) return CWEN_EINVAL;
  if (x_ts % 8 || x_hs % 8 || y_ts % 8 || y_hs % 8 || x_ts < 0 || x_hs < 0 || y_ts < 0 || y_hs < 0) return CWEN_EINVAL;
  // Rows of the output must not share memory with each other: one of the two
  // strides steps over all that the other spans.
  const long long D = r->head_dim, ys = (n_head - 1) * y_hs + D, yt = (T - 1) * y_ts + D;
  if ((n_head > 1 && y_hs < D) || (T > 1 && y_ts < D)) return CWEN_EINVAL;
  if (T > 1 && n_head > 1 && y_ts < ys && y_hs < yt) return CWEN_EINVAL;
  const bool same = x == y && xtype == ytype && (T == 1 || x_ts == y_ts) && (n_head == 1 || x_hs == y_hs);
  if (!same && overlap(x, ((T - 1) * x_ts + (n_head - 1) * x_hs + D) * xe, y, ((T - 1) * y_ts + (n_head - 1) * y_hs + D) * ye))
    return CWEN_EINVAL;
  OnDevice dev(ctx->device);
  if (dev.rc) return dev.rc;
  RopeParams p = {};
  p.q = x; p.q_ts = x_ts; p.q_hs = x_hs;
  p.qo = y; p.qo_ts = y_ts; p.qo_hs = y_hs;
  p.pos = pos; p.T = T; p.nh = n_head; p.inverse = inverse != 0;
  return rope_launch(r, xtype, ytype, p, (hipStream_t)stream);
}

int cwen_rope_kv(cwen_ctx *ctx, const cwen_rope *r, int xtype, const void *q, long long q_ts, const void *k, long long k_ts,
                 const void *v, long long v_ts, void *qo, long long qo_ts, const cwen_kv *kv, int layer, const int *seq,
                 const int *slot, const int *pos, int T, int n_head, void *stream) {
  if (!ctx || !r || T < 0 || T >= 1 << 24 || n_head < 1 || n_head > 65535) return CWEN_EINVAL;
  const int rc = check_kv(kv);
  if (rc) return rc;
  const int xe = elem_size(xtype);
  if (!xe) return CWEN_ETYPE;
  if (kv->head_dim != r->head_dim || layer < 0 || layer >= kv->n_layers) return CWEN_EINVAL;
  if (T == 0) return CWEN_OK;
  const long long D = r->head_dim, qr = n_head * D, kr = kv->n_kv_head * D;
  if (!ok_rows(q, q_ts, T > 1 ? qr : 0) || !ok_rows(k, k_ts, T > 1 ? kr : 0) || !ok_rows(v, v_ts, T > 1 ? kr : 0) ||
      !ok_rows(qo, qo_ts, T > 1 ? qr : 0))
    return CWEN_EINVAL;
  if (!seq || !slot || !pos || !aligned4(seq) || !aligned4(slot) || !aligned4(pos)) return CWEN_EINVAL;
  const bool same = q == qo && xtype == kv->type && (T == 1 || q_ts == qo_ts);
  const long long qo_bytes = ((T - 1) * qo_ts + qr) * 2;
  if (!same && overlap(q, ((T - 1) * q_ts + qr) * xe, qo, qo_bytes)) return CWEN_EINVAL;
  if (!clear_of(k, k_ts * xe, kr * xe, qo, qo_ts * 2, qr * 2, T, same)) return CWEN_EINVAL;
  if (!clear_of(v, v_ts * xe, kr * xe, qo, qo_ts * 2, qr * 2, T, same)) return CWEN_EINVAL;
  OnDevice dev(ctx->device);
  if (dev.rc) return dev.rc;
  RopeParams p = {};
  p.q = q; p.q_ts = q_ts; p.q_hs = D;
  p.qo = qo; p.qo_ts = qo_ts; p.qo_hs = D;
  p.k = k; p.k_ts = k_ts; p.v = v; p.v_ts = v_ts;
  p.kv = *kv; p.layer = layer;
  p.seq = seq; p.slot = slot; p.pos = pos; p.T = T; p.nh = n_head;
  return rope_launch(r, xtype, kv->type, p, (hipStream_t)stream);
}

// ------------------------------------------------------------ paged cache
int cwen_kv_reset(cwen_ctx *ctx, const cwen_kv *kv, void *stream) {
  if (!ctx) return CWEN_EINVAL;
  const int rc = check_kv(kv);
  if (rc) return rc;
  OnDevice dev(ctx->device);
  return dev.rc ? dev.rc : kv_reset_launch(*kv, (hipStream_t)stream);
}
int cwen_kv_reserve(cwen_ctx *ctx, const cwen_kv *kv, const int *seqs, const int *n, int n_req, void *stream) {
  const int rc = check_req(ctx, kv, seqs, n, n_req);
  if (rc || !n_req) return rc;
  OnDevice dev(ctx->device);
  return dev.rc ? dev.rc : kv_reserve_launch(*kv, seqs, n, n_req, (hipStream_t)stream);
}
int cwen_kv_fork(cwen_ctx *ctx, const cwen_kv *kv, const int *src, const int *dst, int n_req, void *stream) {
  const int rc = check_req(ctx, kv, src, dst, n_req);
  if (rc || !n_req) return rc;
  OnDevice dev(ctx->device);
  return dev.rc ? dev.rc : kv_fork_launch(*kv, src, dst, n_req, (hipStream_t)stream);
}
int cwen_kv_keep(cwen_ctx *ctx, const cwen_kv *kv, const int *seqs, const int *count, const int *path, int ps, int n_req,
                 void *stream) {
  const int rc = check_req(ctx, kv, seqs, count, n_req);
  if (rc) return rc;
  if (path && (ps < 1 || !aligned4(path))) return CWEN_EINVAL;
  if (!n_req) return CWEN_OK;
  OnDevice dev(ctx->device);
  return dev.rc ? dev.rc : kv_keep_launch(*kv, seqs, count, path, ps, n_req, (hipStream_t)stream);
}
int cwen_kv_truncate(cwen_ctx *ctx, const cwen_kv *kv, const int *seqs, const int *len, int n_req, void *stream) {
  const int rc = check_req(ctx, kv, seqs, len ? len : seqs, n_req);
  if (rc || !n_req) return rc;
  OnDevice dev(ctx->device);
  return dev.rc ? dev.rc : kv_truncate_launch(*kv, seqs, len, n_req, (hipStream_t)stream);
}
int cwen_kv_status(cwen_ctx *ctx, const cwen_kv *kv, int *bits, void *stream) {
  if (!ctx || !bits) return CWEN_EINVAL;
  int rc = check_kv(kv);
  if (rc) return rc;
  OnDevice dev(ctx->device);
  if (dev.rc) return dev.rc;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  CWEN_HIP_TRY(hipStreamIsCapturing((hipStream_t)stream, &cap));
  if (cap != hipStreamCaptureStatusNone) return CWEN_EINVAL;
  rc = kv_take_status_launch(*kv, ctx->res, (hipStream_t)stream);
  if (rc) return rc;
  CWEN_HIP_TRY(hipMemcpyAsync(bits, ctx->res, sizeof(int), hipMemcpyDeviceToHost, (hipStream_t)stream));
  CWEN_HIP_TRY(hipStreamSynchronize((hipStream_t)stream));
  return CWEN_OK;
}

// ------------------------------------------------------------ attention
constexpr long long launch_max = 1 << 24;       // workgroups of 256: a launch has less than 2^32 threads
static int check_heads(int nh, int nkv, int D, float scale) {
  if (nh < 1 || nkv < 1 || nh > 65535 || nh % nkv || (D != 64 && D != 128 && D != 256)) return CWEN_EINVAL;
  return scale > 0 && isfinite(scale * 1.44269504f) ? CWEN_OK : CWEN_EINVAL;     // exponents are powers of two
}

int cwen_attn_prompt(cwen_ctx *ctx, int type, const void *q, long long q_ts, const void *k, long long k_ts, const void *v,
                     long long v_ts, void *o, long long o_ts, float *lse, const int *cu_q, const int *cu_k, int n_seq,
                     int total_q, int total_k, int n_head, int n_kv_head, int head_dim, float scale, void *stream) {
  if (!ctx) return CWEN_EINVAL;
  if (type != CWEN_T_F16 && type != CWEN_T_BF16) return CWEN_ETYPE;
  int rc = check_heads(n_head, n_kv_head, head_dim, scale);
  if (rc) return rc;
  if (n_seq < 0 || n_seq > 65536 || total_q < 0 || total_k < 0 || total_q >= 1 << 30 || total_k >= 1 << 30) return CWEN_EINVAL;
  if (!cu_k && total_q != total_k) return CWEN_EINVAL;
  if (n_seq == 0 || total_q == 0) return CWEN_OK;
  if (((total_q + 127ll) / 128 + n_seq) * n_head >= launch_max) return CWEN_EINVAL;
  const long long qr = (long long)n_head * head_dim, kr = (long long)n_kv_head * head_dim;
  if (!ok_rows(q, q_ts, qr) || !ok_rows(o, o_ts, qr) || !cu_q || !aligned4(cu_q) || !aligned4(cu_k) || !aligned4(lse))
    return CWEN_EINVAL;
  if (total_k && (!ok_rows(k, k_ts, kr) || !ok_rows(v, v_ts, kr) || k_ts >= 1 << 27 || v_ts >= 1 << 27)) return CWEN_EINVAL;
  const long long ob = ((total_q - 1) * o_ts + qr) * 2;
  if (overlap(q, ((total_q - 1) * q_ts + qr) * 2, o, ob)) return CWEN_EINVAL;
  if (total_k && (overlap(k, ((total_k - 1) * k_ts + kr) * 2, o, ob) || overlap(v, ((total_k - 1) * v_ts + kr) * 2, o, ob)))
    return CWEN_EINVAL;
  OnDevice dev(ctx->device);
  if (dev.rc) return dev.rc;
  const PromptArgs a = {q, k, v, o, q_ts, k_ts, v_ts, o_ts, lse, cu_q, cu_k ? cu_k : cu_q, n_seq, total_q, total_k, n_head,
                        n_kv_head, scale};
  return attn_prompt_launch(ctx, type, head_dim, a, (hipStream_t)stream);
}

int cwen_attn_tree(cwen_ctx *ctx, const cwen_kv *kv, int layer, const void *q, long long q_ts, void *o, long long o_ts,
                   float *lse, const int *seqs, const int *cu, const unsigned long long *mask, int mw, int n_seq, int total,
                   int max_nodes, int max_len, int n_head, float scale, void *stream) {
  if (!ctx) return CWEN_EINVAL;
  int rc = check_kv(kv);
  if (!rc) rc = check_heads(n_head, kv->n_kv_head, kv->head_dim, scale);
  if (rc) return rc;
  if (layer < 0 || layer >= kv->n_layers || n_seq < 0 || n_seq > kv->max_seqs || total < 0 || total >= 1 << 24) return CWEN_EINVAL;
  if (max_nodes < 0 || max_nodes > CWEN_TREE_MAX || max_len < 0) return CWEN_EINVAL;
  if (mask && ((uintptr_t)mask % 8 || mw < 1 || mw > CWEN_TREE_MAX / 64 || max_nodes > 64 * mw)) return CWEN_EINVAL;
  if (n_seq == 0 || total == 0 || max_nodes == 0) return CWEN_OK;
  if ((n_head + 31ll) / 32 * total >= launch_max) return CWEN_EINVAL;
  const long long qr = (long long)n_head * kv->head_dim;
  if (!ok_rows(q, q_ts, qr) || !ok_rows(o, o_ts, qr) || !seqs || !cu || !aligned4(seqs) || !aligned4(cu) || !aligned4(lse))
    return CWEN_EINVAL;
  if (overlap(q, ((total - 1) * q_ts + qr) * 2, o, ((total - 1) * o_ts + qr) * 2)) return CWEN_EINVAL;
  OnDevice dev(ctx->device);
  if (dev.rc) return dev.rc;
  const TreeArgs a = {*kv, layer, q, o, q_ts, o_ts, lse, seqs, cu, mask, mw, n_seq, total, max_nodes, max_len, n_head, scale};
  return attn_tree_launch(ctx, a, (hipStream_t)stream);
}

}  // extern "C"
