/* Losses on logits for tuning a language model: the clipped policy loss with a KL term and the preference loss
 * (include/nc_ext.h says what they compute). They stand beside cross_entropy and nll_loss: i32 labels, checked
 * on the host when their host copy is current and by the kernel otherwise, a scalar loss, sums in 64 bits in a
 * fixed order. newch has neither. */
#include "nc_internal.h"

#include <cuda_runtime_api.h>
#include <math.h>

/* The inputs of a node: the logits, then those of a fixed list that were given (bit i of p.i[0]). */
enum { LAB = 1, OLD = 2, REF = 4, ADV = 8, MASK = 16 };
enum { P_HAS, P_MORE }; /* p.i[P_MORE]: the header of the second result, made before the op (0: not asked for) */

static nc_tensor *input(const nc_node *n, int which) {
    if (!(n->p.i[P_HAS] & which)) return NULL;
    int k = 1;
    for (int w = LAB; w < which; w <<= 1) k += (n->p.i[P_HAS] & w) != 0;
    return n->in[k];
}

typedef struct {
    float *stat, *coef, *scale;
} loss_saved;

static int refuse(nc_ctx *ctx, nc_status code, const char *op, const char *what) {
    nc__error(ctx, code, "%s: %s", op, what);
    return 0;
}

/* Checks what every input is before anything is made. `given` lists the inputs in the order of the bits. */
static int inputs_ok(const char *op, nc_tensor *z, nc_tensor *const given[5]) {
    static const char *const names[5] = {"labels", "old_logp", "ref_logp", "advantages", "mask"};
    nc_ctx *ctx = z->ctx;
    for (int i = -1; i < 5; i++) {
        const nc_tensor *t = i < 0 ? z : given[i];
        if (t && nc__is_released(t)) return refuse(ctx, NC_ERR_STATE, op, "an input was released");
    }
    if (z->dtype != NC_F32) return refuse(ctx, NC_ERR_DTYPE, op, "logits must be f32");
    if ((z->ndim != 2 && z->ndim != 3) || z->shape[z->ndim - 1] < 1 || z->shape[z->ndim - 1] > INT32_MAX)
        return refuse(ctx, NC_ERR_SHAPE, op, "logits must be [rows, vocab] or [batch, tokens, vocab], 1 <= vocab < 2^31");
    for (int i = 0; i < 5; i++) {
        const nc_tensor *t = given[i];
        if (!t) continue;
        const int whole = i == 0 || i == 4;
        if (t->ctx != ctx) return refuse(ctx, NC_ERR_ARG, op, "inputs belong to different contexts");
        if (whole ? t->dtype != NC_I32 : t->dtype != NC_F32) {
            nc__error(ctx, NC_ERR_DTYPE, "%s: %s must be %s, got %s", op, names[i], whole ? "i32" : "f32",
                      nc__dtype_name(t->dtype));
            return 0;
        }
        if (ctx->grad_enabled && nc__needs_grad(t)) {
            nc__error(ctx, NC_ERR_ARG, "%s: %s is a constant and must not require grad (detach it)", op, names[i]);
            return 0;
        }
    }
    return 1;
}

static int leading_shape(const char *op, const nc_tensor *z, const nc_tensor *t, const char *name) {
    int ok = t->ndim == z->ndim - 1;
    for (int i = 0; ok && i < t->ndim; i++) ok = t->shape[i] == z->shape[i];
    if (!ok) {
        char sz[96], st[96];
        nc__error(z->ctx, NC_ERR_SHAPE, "%s: %s %s does not have the leading shape of logits %s", op, name,
                  nc__shape_str(t->ndim, t->shape, st, sizeof st), nc__shape_str(z->ndim, z->shape, sz, sizeof sz));
    }
    return ok;
}

/* counted labels against [0, vocab), when the host has current copies of them (and of the mask) */
static int labels_ok(const char *op, nc_tensor *lab, nc_tensor *mask, int64_t V) {
    const int32_t *h = (const int32_t *)nc__host_view(lab);
    const int32_t *m = mask ? (const int32_t *)nc__host_view(mask) : NULL;
    if (!h || (mask && !m)) return 1;
    for (int64_t i = 0, N = nc_numel(lab); i < N; i++)
        if ((!m || m[i]) && (h[i] < 0 || h[i] >= V)) {
            nc__error(lab->ctx, NC_ERR_ARG, "%s: label %d at row %lld outside [0, %lld)", op, h[i], (long long)i, (long long)V);
            return 0;
        }
    return 1;
}

static nc_status loss_infer(nc_node *n, nc_dtype *dt, int *nd, int64_t *shape) {
    (void)n, (void)shape;
    *dt = NC_F32;
    *nd = 0;
    return NC_OK;
}

/* The kernels' description of the logits; 0 on failure. */
static int rows_of(const nc_node *n, nck_rows *q) {
    nc_tensor *z = n->in[0], *lab = input(n, LAB), *mask = input(n, MASK);
    const int k = z->ndim - 1;
    memset(q, 0, sizeof *q);
    q->V = z->shape[k];
    q->N = nc_numel(z) / q->V;
    q->T = k == 2 ? z->shape[1] : q->N;
    if (z->stride[k] == 1 || q->V == 1) {
        q->z = (const float *)nc__dev(z);
        q->st = z->stride[k - 1];
        q->sb = k == 2 ? z->stride[0] : 0;
        if (k == 2 && q->sb == q->st * q->T) q->T = q->N; /* rows one stride apart */
    } else {
        q->z = nc__contig_f32(z);
        q->T = q->N, q->st = q->V;
    }
    if (q->T < 1) q->T = 1;
    q->lab = (const int32_t *)nc__contig(lab);
    q->mask = mask ? (const int32_t *)nc__contig(mask) : NULL;
    return q->z && q->lab && (!mask || q->mask);
}

/* What backward needs of the rows, when the op is recorded. */
static loss_saved *keep(nc_node *n, nck_rows *q, int64_t coefs) {
    nc_ctx *ctx = n->out->ctx;
    loss_saved *sv = (loss_saved *)nc__meta_alloc(ctx, sizeof(loss_saved), 0);
    float *stat = (float *)nc__arena_alloc(ctx, (size_t)(q->N * 2 + 2) * sizeof(float));
    float *coef = (float *)nc__arena_alloc(ctx, (size_t)(coefs + 1) * sizeof(float));
    if (!sv || !stat || !coef) return NULL;
    sv->stat = q->stat = stat;
    sv->coef = coef;
    sv->scale = coef + coefs;
    n->saved = sv;
    return sv;
}

static void loss_bwd(nc_node *n, int64_t per_coef, int scaled) {
    nc_tensor *z = n->in[0];
    const loss_saved *sv = (const loss_saved *)n->saved;
    nck_rows q;
    if (!rows_of(n, &q)) return;
    q.stat = sv->stat;
    nck_rows_grad g;
    memset(&g, 0, sizeof g);
    nc_tensor *gz = nc__grad_buf_set(z, &g.acc);
    if (!gz) return;
    g.up = (const float *)n->out->grad->data;
    g.scale = scaled ? sv->scale : NULL;
    g.coef = sv->coef;
    g.per_coef = per_coef;
    g.dz = (float *)gz->data;
    nck_rows_bwd(nc__k(z->ctx), &q, &g);
}

static float *more_data(const nc_node *n) {
    nc_tensor *t = (nc_tensor *)(intptr_t)n->p.i[P_MORE];
    return t ? (float *)t->data : NULL;
}

/* the second result, not on the tape */
static nc_tensor *make_more(nc_ctx *ctx, int nd, const int64_t *shape) {
    return nc__tensor_new(ctx, NC_F32, nd, shape, nc__is_persistent_mode(ctx));
}

/* ---- policy loss -------------------------------------------------------------------------------- */

static nc_status policy_fwd(nc_node *n) {
    nc_tensor *ref = input(n, REF);
    nck_rows q;
    nck_policy p;
    memset(&p, 0, sizeof p);
    if (!rows_of(n, &q)) return NC_ERR_OOM;
    p.old = nc__contig_f32(input(n, OLD));
    p.adv = nc__contig_f32(input(n, ADV));
    p.ref = ref ? nc__contig_f32(ref) : NULL;
    if (!p.old || !p.adv || (ref && !p.ref)) return NC_ERR_OOM;
    p.clip_low = n->p.f[0], p.clip_high = n->p.f[1], p.kl = n->p.f[2];
    p.loss = (float *)n->out->data;
    q.lp32 = more_data(n);
    if (n->out->ctx->fwd_on_tape) {
        loss_saved *sv = keep(n, &q, q.N);
        if (!sv) return NC_ERR_OOM;
        p.coef = sv->coef, p.scale = sv->scale;
    }
    nck_rows_logp(nc__k(n->out->ctx), &q, &p);
    return NC_OK;
}

static void policy_bwd(nc_node *n) { loss_bwd(n, 1, 1); }

const nc_op_def nc_op_policy_loss = {"policy_loss", 0, 0, loss_infer, NULL, policy_fwd, policy_bwd};

/* a mask of another integer type becomes i32, as masked_fill's does (a released one is refused with the rest) */
static nc_tensor *as_mask(nc_tensor *mask) {
    return mask && !nc__is_released(mask) && (mask->dtype == NC_I8 || mask->dtype == NC_U8) ? nc_to_dtype(mask, NC_I32) : mask;
}

nc_tensor *nc_ext_policy_loss(nc_tensor *logits, nc_tensor *actions, nc_tensor *old_logp, nc_tensor *ref_logp,
                              nc_tensor *advantages, nc_tensor *mask, const nc_ext_policy_opts *opts, nc_tensor **logp) {
    static const char *const op = "policy_loss";
    if (logp) *logp = NULL;
    if (!logits || !actions || !old_logp || !advantages) return NULL;
    nc_ctx *ctx = logits->ctx;
    if (ctx->status != NC_OK) return NULL;
    if (!opts) return refuse(ctx, NC_ERR_ARG, op, "opts must not be NULL"), NULL;
    nc_tensor *const asked = mask;
    mask = as_mask(mask);
    if (asked && !mask) return NULL;
    nc_tensor *const given[5] = {actions, old_logp, ref_logp, advantages, mask};
    if (!inputs_ok(op, logits, given) || !leading_shape(op, logits, actions, "labels") ||
        !leading_shape(op, logits, old_logp, "old_logp") || (ref_logp && !leading_shape(op, logits, ref_logp, "ref_logp")) ||
        !leading_shape(op, logits, advantages, "advantages") || (mask && !leading_shape(op, logits, mask, "mask")))
        return NULL;
    if (!(opts->clip_low >= 0.0f && opts->clip_low <= 1.0f) || !(opts->clip_high >= 0.0f) || !isfinite(opts->clip_high))
        return refuse(ctx, NC_ERR_ARG, op, "clip_low must lie in [0, 1] and clip_high be at least 0"), NULL;
    if (!isfinite(opts->kl_coef)) return refuse(ctx, NC_ERR_ARG, op, "kl_coef must be finite"), NULL;
    if (opts->kl_coef != 0.0f && !ref_logp) return refuse(ctx, NC_ERR_ARG, op, "a KL term needs ref_logp"), NULL;
    if (!labels_ok(op, actions, mask, logits->shape[logits->ndim - 1])) return NULL;
    nc_tensor *more = NULL;
    if (logp && !(more = make_more(ctx, logits->ndim - 1, logits->shape))) return NULL;
    nc_op_params p;
    memset(&p, 0, sizeof p);
    nc_tensor *in[6] = {logits};
    int k = 1;
    for (int i = 0; i < 5; i++)
        if (given[i]) in[k++] = given[i], p.i[P_HAS] |= 1 << i;
    p.i[P_MORE] = (int64_t)(intptr_t)more;
    p.f[0] = opts->clip_low, p.f[1] = opts->clip_high, p.f[2] = opts->kl_coef;
    nc_tensor *loss = nc__apply(&nc_op_policy_loss, in, k, &p);
    if (loss && logp) *logp = more;
    else nc_release(more);
    return loss;
}

/* ---- preference loss ---------------------------------------------------------------------------- */

static nc_status pref_fwd(nc_node *n) {
    nc_ctx *ctx = n->out->ctx;
    nc_tensor *z = n->in[0], *ref = input(n, REF);
    nck_rows q;
    nck_pairs p;
    memset(&p, 0, sizeof p);
    if (!rows_of(n, &q)) return NC_ERR_OOM;
    p.P = z->shape[0] / 2, p.T = z->shape[1];
    p.ref = ref ? nc__contig_f32(ref) : NULL;
    p.beta = n->p.f[0], p.smoothing = n->p.f[1];
    p.seq = more_data(n);
    p.loss = (float *)n->out->data;
    q.lp64 = (double *)nc__arena_alloc(ctx, (size_t)(q.N + 1) * sizeof(double));
    p.term = (double *)nc__arena_alloc(ctx, (size_t)p.P * sizeof(double));
    if (!q.lp64 || !p.term || (ref && !p.ref)) return NC_ERR_OOM;
    if (ctx->fwd_on_tape) {
        loss_saved *sv = keep(n, &q, 2 * p.P);
        if (!sv) return NC_ERR_OOM;
        p.coef = sv->coef;
    }
    if (q.N) nck_rows_logp(nc__k(ctx), &q, NULL);
    nck_pref_pairs(nc__k(ctx), &p, q.lp64);
    return NC_OK;
}

static void pref_bwd(nc_node *n) { loss_bwd(n, n->in[0]->shape[1], 0); }

const nc_op_def nc_op_preference_loss = {"preference_loss", 0, 0, loss_infer, NULL, pref_fwd, pref_bwd};

nc_tensor *nc_ext_preference_loss(nc_tensor *logits, nc_tensor *labels, nc_tensor *ref_logp, nc_tensor *mask, float beta,
                                  float label_smoothing, nc_tensor **seq_logp) {
    static const char *const op = "preference_loss";
    if (seq_logp) *seq_logp = NULL;
    if (!logits || !labels) return NULL;
    nc_ctx *ctx = logits->ctx;
    if (ctx->status != NC_OK) return NULL;
    nc_tensor *const asked = mask;
    mask = as_mask(mask);
    if (asked && !mask) return NULL;
    nc_tensor *const given[5] = {labels, NULL, ref_logp, NULL, mask};
    if (!inputs_ok(op, logits, given)) return NULL;
    if (logits->ndim != 3 || logits->shape[0] < 2 || (logits->shape[0] & 1) || logits->shape[0] / 2 > INT32_MAX)
        return refuse(ctx, NC_ERR_SHAPE, op, "logits must be [2 pairs, tokens, vocab] with at least one pair"), NULL;
    if (!leading_shape(op, logits, labels, "labels") || (mask && !leading_shape(op, logits, mask, "mask"))) return NULL;
    if (ref_logp && (ref_logp->ndim != 1 || ref_logp->shape[0] != logits->shape[0]))
        return refuse(ctx, NC_ERR_SHAPE, op, "ref_logp must be [2 pairs]"), NULL;
    if (!(beta > 0.0f) || !isfinite(beta)) return refuse(ctx, NC_ERR_ARG, op, "beta must be positive"), NULL;
    if (!(label_smoothing >= 0.0f && label_smoothing <= 0.5f))
        return refuse(ctx, NC_ERR_ARG, op, "label_smoothing must lie in [0, 0.5]"), NULL;
    if (!labels_ok(op, labels, mask, logits->shape[2])) return NULL;
    nc_tensor *more = NULL;
    if (seq_logp && !(more = make_more(ctx, 1, logits->shape))) return NULL;
    nc_op_params p;
    memset(&p, 0, sizeof p);
    nc_tensor *in[4] = {logits};
    int k = 1;
    for (int i = 0; i < 5; i++)
        if (given[i]) in[k++] = given[i], p.i[P_HAS] |= 1 << i;
    p.i[P_MORE] = (int64_t)(intptr_t)more;
    p.f[0] = beta, p.f[1] = label_smoothing;
    nc_tensor *loss = nc__apply(&nc_op_preference_loss, in, k, &p);
    if (loss && seq_logp) *seq_logp = more;
    else nc_release(more);
    return loss;
}
