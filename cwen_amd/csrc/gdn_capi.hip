// C ABI entry points of the GatedDeltaNet layers of many sequences and of the
// log probabilities.  Argument checks; nothing here touches the GPU before they
// have passed.
#include "capi_checks.h"
#include "gdn_table.h"

namespace {

constexpr long long launch_max = 1 << 24;       // workgroups of 256: a launch has less than 2^32 threads

int check_pool(const cwen_gdn_pool *p) {
  if (!p || p->n_layers < 1 || p->n_layers > 32767 || p->n_slots < 1 || p->n_slots > 65536) return CWEN_EINVAL;
  if (p->nkh < 1 || p->nvh < 1 || p->nvh > 4096 || p->nvh % p->nkh || (p->dk != 64 && p->dk != 128)) return CWEN_EINVAL;
  if (p->key_head != CWEN_GDN_MOD && p->key_head != CWEN_GDN_GROUP) return CWEN_EINVAL;
  if (!aligned16(p->state) || !aligned16(p->hist) || !p->status || !aligned4(p->status)) return CWEN_EINVAL;
  return CWEN_OK;
}
int channels(const cwen_gdn_pool *p) { return (2 * p->nkh + p->nvh) * p->dk; }
int check_seqs(const cwen_ctx *ctx, const cwen_gdn_pool *p, int layer, const int *cu, const int *count, const int *src,
               const int *dst, int n_seq, int total) {
  if (!ctx) return CWEN_EINVAL;
  const int rc = check_pool(p);
  if (rc) return rc;
  if (layer < 0 || layer >= p->n_layers || n_seq < 0 || n_seq > CWEN_GDN_SEQ_MAX || total < 0 || total >= 1 << 30) return CWEN_EINVAL;
  if (n_seq && (!cu || !aligned4(cu) || !aligned4(count) || !aligned4(src) || !aligned4(dst))) return CWEN_EINVAL;
  return CWEN_OK;
}
// Rows of `row` elements of `es` bytes; with no rows the address does not matter.
bool ok_part(const void *p, long long ts, long long row, int total) { return !total || ok_rows(p, ts, total > 1 ? row : 0); }

// What step and prompt have in common; *none: nothing to do.
int check_rule(const cwen_ctx *ctx, const cwen_gdn_pool *pool, int layer, int xtype, const void *q, long long q_ts, const void *k,
               long long k_ts, const void *v, long long v_ts, const float *a, const float *b, long long g_ts, const float *A,
               const float *dt, int otype, void *o, long long o_ts, const int *cu, const int *count, const int *src, const int *dst,
               int n_seq, int total, GdnRuleArgs *out, bool *none) {
  const int rc = check_seqs(ctx, pool, layer, cu, count, src, dst, n_seq, total);
  if (rc) return rc;
  const int xe = elem_size(xtype), oe = elem_size(otype);
  if (!xe || !oe) return CWEN_ETYPE;
  if (!pool->state || (A == nullptr) != (dt == nullptr) || !aligned4(A) || !aligned4(dt)) return CWEN_EINVAL;
  const long long D = pool->dk, kr = pool->nkh * D, vr = pool->nvh * D;
  if (!ok_part(q, q_ts, kr, total) || !ok_part(k, k_ts, kr, total) || !ok_part(v, v_ts, vr, total)) return CWEN_EINVAL;
  if (total && (!a || !b || !aligned4(a) || !aligned4(b) || (total > 1 && g_ts < pool->nvh))) return CWEN_EINVAL;
  if (o && total) {
    if (!ok_part(o, o_ts, vr, total)) return CWEN_EINVAL;
    const long long ob = o_ts * oe, orow = vr * oe;
    if (!clear_of(q, q_ts * xe, kr * xe, o, ob, orow, total, true) || !clear_of(k, k_ts * xe, kr * xe, o, ob, orow, total, true) ||
        !clear_of(v, v_ts * xe, vr * xe, o, ob, orow, total, true))
      return CWEN_EINVAL;
  }
  *none = n_seq == 0;
  const long long layer_floats = (long long)pool->n_slots * pool->nvh * D * D;
  if (total == 1) q_ts = k_ts = kr, v_ts = o_ts = vr, g_ts = pool->nvh;       // strides of nothing
  *out = {{cu, count, src, dst, n_seq, total, pool->n_slots, pool->status}, q, k, v, o, q_ts, k_ts, v_ts, o_ts, g_ts, a, b, A, dt,
          pool->state + layer * layer_floats, pool->nkh, pool->nvh, pool->key_head == CWEN_GDN_GROUP ? pool->nvh / pool->nkh : 0};
  return CWEN_OK;
}

}  // namespace

extern "C" {

int cwen_gdn_status(cwen_ctx *ctx, const cwen_gdn_pool *pool, int *bits, void *stream) {
  if (!ctx || !bits) return CWEN_EINVAL;
  int rc = check_pool(pool);
  if (rc) return rc;
  OnDevice dev(ctx->device);
  if (dev.rc) return dev.rc;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  CWEN_HIP_TRY(hipStreamIsCapturing((hipStream_t)stream, &cap));
  if (cap != hipStreamCaptureStatusNone) return CWEN_EINVAL;
  cwen_kv kv = {};
  kv.status = pool->status;
  rc = kv_take_status_launch(kv, ctx->res, (hipStream_t)stream);
  if (rc) return rc;
  CWEN_HIP_TRY(hipMemcpyAsync(bits, ctx->res, sizeof(int), hipMemcpyDeviceToHost, (hipStream_t)stream));
  CWEN_HIP_TRY(hipStreamSynchronize((hipStream_t)stream));
  return CWEN_OK;
}

int cwen_gdn_conv(cwen_ctx *ctx, const cwen_gdn_pool *pool, int layer, int xtype, const void *x, long long x_ts, const float *kw,
                  int ytype, void *y, long long y_ts, const int *cu, const int *count, const int *src, const int *dst, int n_seq,
                  int total, void *stream) {
  const int rc = check_seqs(ctx, pool, layer, cu, count, src, dst, n_seq, total);
  if (rc) return rc;
  const int xe = elem_size(xtype), ye = elem_size(ytype);
  if (!xe || !ye) return CWEN_ETYPE;
  const int C = channels(pool);
  if (!pool->hist || !ok_part(x, x_ts, C, total) || !kw || !aligned16(kw)) return CWEN_EINVAL;
  if (y && total) {
    if (!ok_part(y, y_ts, C, total)) return CWEN_EINVAL;
    if (!clear_of(x, x_ts * xe, (long long)C * xe, y, y_ts * ye, (long long)C * ye, total, true)) return CWEN_EINVAL;
  }
  if (n_seq == 0) return CWEN_OK;
  if (gdn_pieces(total, n_seq, 32) >= 2 * launch_max) return CWEN_EINVAL;      // workgroups of 128
  OnDevice dev(ctx->device);
  if (dev.rc) return dev.rc;
  const GdnConvArgs a = {{cu, count, src, dst, n_seq, total, pool->n_slots, pool->status}, x, y, x_ts, y_ts, kw,
                         pool->hist + (long long)layer * pool->n_slots * C * 3, C};
  return gdn_conv_launch(xtype, ytype, a, (hipStream_t)stream);
}

int cwen_gdn_step(cwen_ctx *ctx, const cwen_gdn_pool *pool, int layer, int xtype, const void *q, long long q_ts, const void *k,
                  long long k_ts, const void *v, long long v_ts, const float *a, const float *b, long long g_ts, const float *A,
                  const float *dt, int otype, void *o, long long o_ts, const int *cu, const int *count, const int *src, const int *dst,
                  int n_seq, int total, void *stream) {
  GdnRuleArgs args;
  bool none = false;
  const int rc = check_rule(ctx, pool, layer, xtype, q, q_ts, k, k_ts, v, v_ts, a, b, g_ts, A, dt, otype, o, o_ts, cu, count, src, dst,
                            n_seq, total, &args, &none);
  if (rc || none) return rc;
  if ((long long)n_seq * pool->nvh >= launch_max) return CWEN_EINVAL;
  OnDevice dev(ctx->device);
  return dev.rc ? dev.rc : gdn_step_launch(xtype, otype, pool->dk, args, (hipStream_t)stream);
}

int cwen_gdn_prompt_work(const cwen_gdn_pool *pool, int xtype, int otype, int n_seq, int total, size_t *bytes) {
  if (!bytes) return CWEN_EINVAL;
  *bytes = 0;
  const int rc = check_pool(pool);
  if (rc) return rc;
  if (!elem_size(xtype) || !elem_size(otype)) return CWEN_ETYPE;
  if (n_seq < 0 || n_seq > CWEN_GDN_SEQ_MAX || total < 0 || total >= 1 << 30) return CWEN_EINVAL;
  if (n_seq) *bytes = gdn_prompt_bytes(xtype, pool->dk, pool->nkh, pool->nvh, n_seq, total);
  return CWEN_OK;
}

int cwen_gdn_prompt(cwen_ctx *ctx, const cwen_gdn_pool *pool, int layer, int xtype, const void *q, long long q_ts, const void *k,
                    long long k_ts, const void *v, long long v_ts, const float *a, const float *b, long long g_ts, const float *A,
                    const float *dt, int otype, void *o, long long o_ts, const int *cu, const int *count, const int *src,
                    const int *dst, int n_seq, int total, void *work, size_t work_bytes, void *stream) {
  GdnRuleArgs args;
  bool none = false;
  const int rc = check_rule(ctx, pool, layer, xtype, q, q_ts, k, k_ts, v, v_ts, a, b, g_ts, A, dt, otype, o, o_ts, cu, count, src, dst,
                            n_seq, total, &args, &none);
  if (rc || none) return rc;
  // (the second launch has up to 640 threads a sequence and head)
  if (gdn_pieces(total, n_seq, 32) * pool->nvh * 2 >= launch_max || (long long)n_seq * pool->nvh * 4 >= launch_max) return CWEN_EINVAL;
  if (total > 1 && (v_ts >= 1 << 24 || (o && o_ts >= 1 << 24))) return CWEN_EINVAL;      // a chunk's rows by 32-bit offsets
  const size_t need = gdn_prompt_bytes(xtype, pool->dk, pool->nkh, pool->nvh, n_seq, total);
  if (need && (!work || ((uintptr_t)work & 255u))) return CWEN_EINVAL;
  if (work_bytes < need) return CWEN_ESCRATCH;
  OnDevice dev(ctx->device);
  return dev.rc ? dev.rc : gdn_prompt_launch(xtype, otype, pool->dk, args, work, (hipStream_t)stream);
}

// ------------------------------------------------------------ log probabilities
static int check_logprobs(int rows, int V, int top) {
  return rows < 0 || rows >= launch_max / 64 || V < 1 || V > 1 << 30 || top < 0 || top > CWEN_LOGPROBS_TOP ? CWEN_EINVAL : CWEN_OK;
}
int cwen_logprobs_work(int rows, int V, int top, size_t *bytes) {
  if (!bytes) return CWEN_EINVAL;
  *bytes = 0;
  const int rc = check_logprobs(rows, V, top);
  if (!rc) *bytes = logprobs_bytes(rows, V, top);
  return rc;
}
int cwen_logprobs(cwen_ctx *ctx, int type, const void *logits, long long ls, int V, int rows, const int *tokens, float *logprob,
                  int *rank, float *entropy, float *lse, int top, int *top_ids, float *top_logprobs, void *work, size_t work_bytes,
                  void *stream) {
  if (!ctx) return CWEN_EINVAL;
  const int rc = check_logprobs(rows, V, top), es = elem_size(type);
  if (rc) return rc;
  if (!es) return CWEN_ETYPE;
  if ((logprob || rank) && !tokens) return CWEN_EINVAL;
  if (!aligned4(tokens) || !aligned4(logprob) || !aligned4(rank) || !aligned4(entropy) || !aligned4(lse) || !aligned4(top_ids) ||
      !aligned4(top_logprobs))
    return CWEN_EINVAL;
  if (rows == 0) return CWEN_OK;
  if (!logits || (uintptr_t)logits % es || (rows > 1 && ls < V)) return CWEN_EINVAL;
  if (!top_ids && !top_logprobs) top = 0;
  const size_t need = logprobs_bytes(rows, V, top);
  if (need && (!work || !aligned16(work))) return CWEN_EINVAL;
  if (work_bytes < need) return CWEN_ESCRATCH;
  OnDevice dev(ctx->device);
  if (dev.rc) return dev.rc;
  const LogprobArgs a = {logits, ls, V, rows, top, tokens, logprob, entropy, lse, top_logprobs, rank, top_ids, (float *)work};
  return logprobs_launch(type, a, (hipStream_t)stream);
}

}  // extern "C"
