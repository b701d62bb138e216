/* Query and key norms with rotary positions: one op over the heads of a projection, forward and backward
 * (nc_ext_qk_norm_rope in include/nc_ext.h says what it computes). newch's transformer has neither; the op
 * follows the conventions of layer_norm: weights are inputs, NULL for none. */
#include "nc_internal.h"

#include <cuda_runtime_api.h>
#include <math.h>

enum { P_QHEADS, P_AXES, P_SECTION, P_FLAGS = P_SECTION + 3, P_HAS }; /* node parameters p.i */
enum { HAS_WQ = 1, HAS_WK = 2, HAS_POS = 4 };

static nc_tensor *input(const nc_node *n, int which) {
    if (!(n->p.i[P_HAS] & which)) return NULL;
    int k = 1;
    for (int w = HAS_WQ; w < which; w <<= 1) k += (n->p.i[P_HAS] & w) != 0;
    return n->in[k];
}

static nc_status refuse(nc_ctx *ctx, nc_status code, const char *what) {
    nc__error(ctx, code, "qk_norm_rope: %s", what);
    return code;
}

static nc_status rope_infer(nc_node *n, nc_dtype *dt, int *nd, int64_t *shape) {
    nc_tensor *x = n->in[0];
    nc_ctx *ctx = x->ctx;
    for (int i = 0; i < n->n_in; i++)
        if (nc__is_released(n->in[i])) return refuse(ctx, NC_ERR_STATE, "an input was released");
    if (!nc__expect_f32(n, 0)) return NC_ERR_DTYPE;
    if (x->ndim != 4) return refuse(ctx, NC_ERR_SHAPE, "x must be [batch, tokens, heads, dim]");
    const int64_t H = x->shape[2], D = x->shape[3], A = n->p.i[P_AXES];
    if (D < 2 || D > NCK_ROPE_MAX_DIM || (D & 1)) return refuse(ctx, NC_ERR_SHAPE, "the head size must be even, 2 to 256");
    if (H > 65535 || x->shape[0] * x->shape[1] > INT32_MAX - 64)
        return refuse(ctx, NC_ERR_SHAPE, "more than 65535 heads, or batch * tokens above 2^31 - 65");
    if (n->p.i[P_QHEADS] < 0 || n->p.i[P_QHEADS] > H) return refuse(ctx, NC_ERR_ARG, "q_heads must lie in [0, heads]");
    if (A < 1 || A > 3) return refuse(ctx, NC_ERR_ARG, "n_axes must be 1, 2 or 3");
    int64_t pairs = 0;
    for (int a = 0; a < A; a++) {
        if (n->p.i[P_SECTION + a] < 0) return refuse(ctx, NC_ERR_ARG, "a section must not be negative");
        pairs += n->p.i[P_SECTION + a];
    }
    if (pairs > D / 2) return refuse(ctx, NC_ERR_ARG, "the sections hold more pairs than dim / 2");
    if (!(n->p.f[0] > 0.0f) || !isfinite(n->p.f[0])) return refuse(ctx, NC_ERR_ARG, "base must be positive");
    if (!(n->p.f[1] >= 0.0f) || !isfinite(n->p.f[1])) return refuse(ctx, NC_ERR_ARG, "eps must not be negative");
    if (n->p.i[P_FLAGS] & ~(int64_t)(NC_EXT_ROPE_INTERLEAVED | NC_EXT_ROPE_AXIS_FREQ | NC_EXT_ROPE_NO_NORM))
        return refuse(ctx, NC_ERR_ARG, "unknown flags");
    for (int w = HAS_WQ; w <= HAS_WK; w <<= 1) {
        const nc_tensor *t = input(n, w);
        if (!t) continue;
        if (t->dtype != NC_F32) return refuse(ctx, NC_ERR_DTYPE, "weights must be f32");
        if (t->ndim != 1 || t->shape[0] != D) return refuse(ctx, NC_ERR_SHAPE, "weights must be [dim]");
    }
    const nc_tensor *pos = input(n, HAS_POS);
    if (pos) {
        if (pos->dtype != NC_I32) return refuse(ctx, NC_ERR_DTYPE, "positions must be i32");
        const int k = pos->ndim - 2; /* 0: [tokens, axes], 1: [batch, tokens, axes] */
        if ((k != 0 && k != 1) || pos->shape[k + 1] != A || pos->shape[k] != x->shape[1] || (k && pos->shape[0] != x->shape[0]))
            return refuse(ctx, NC_ERR_SHAPE, "positions must be [tokens, n_axes] or [batch, tokens, n_axes]");
    } else if (A != 1) {
        return refuse(ctx, NC_ERR_ARG, "several axes need positions");
    }
    *dt = NC_F32;
    *nd = 4;
    memcpy(shape, x->shape, sizeof(int64_t) * 4);
    return NC_OK;
}

/* The kernels' description of the node; 0 on failure. */
static int rope_of(const nc_node *n, nck_rope *q) {
    nc_tensor *x = n->in[0], *wq = input(n, HAS_WQ), *wk = input(n, HAS_WK), *pos = input(n, HAS_POS);
    memset(q, 0, sizeof *q);
    q->B = x->shape[0], q->T = x->shape[1], q->H = (int)x->shape[2], q->D = (int)x->shape[3];
    q->HQ = (int)n->p.i[P_QHEADS];
    q->n_axes = (int)n->p.i[P_AXES];
    q->eps = n->p.f[1];
    q->norm = !(n->p.i[P_FLAGS] & NC_EXT_ROPE_NO_NORM);
    q->interleaved = (n->p.i[P_FLAGS] & NC_EXT_ROPE_INTERLEAVED) != 0;
    if (x->stride[3] == 1) { /* any layout of whole rows is read in place */
        q->x = (const float *)nc__dev(x);
        q->sb = x->stride[0], q->st = x->stride[1], q->sh = x->stride[2];
    } else {
        q->x = nc__contig_f32(x);
        q->sh = q->D, q->st = q->sh * q->H, q->sb = q->st * q->T;
    }
    q->wq = wq ? nc__contig_f32(wq) : NULL;
    q->wk = wk ? nc__contig_f32(wk) : NULL;
    q->pos = pos ? (const int32_t *)nc__contig(pos) : NULL;
    q->pos_t = q->n_axes;
    q->pos_b = pos && pos->ndim == 3 ? q->T * q->n_axes : 0;
    if (!q->x || (wq && !q->wq) || (wk && !q->wk) || (pos && !q->pos)) return 0;
    /* Turns of pair i per step, base^-(i / half) / 2 pi, as fractions of 2^64: the first one times the ratio of
     * neighbours again and again, in 64 by 64 bits. A product adds half a unit, and the ratio's own error (a unit or
     * two of 2^-64) at most a sixth of it for each, so 128 pairs are off by less than 2^-57 at worst; replayed against
     * 60 digits for bases from 1.0000001 to 1e30 and 1 to 128 pairs it is 9 units of 2^-64 at most, 3 for a base of
     * 10000. In long double for a base of 1 or less, whose turns grow past whole ones: off by 2^-58 for a base of 0.5
     * (128 pairs), and in proportion to the largest turn below that. With AXIS_FREQ i counts from the start of its
     * section and half is the section's length. */
    const long double unit = 0.159154943091895335768883763372514362L, two64 = 0x1p64L, ln_base = logl((long double)n->p.f[0]);
    const int half = q->D / 2, by_axis = (n->p.i[P_FLAGS] & NC_EXT_ROPE_AXIS_FREQ) != 0;
    const uint64_t first = (uint64_t)(unit * two64);
    long double f = unit, step = expl(-ln_base / half);
    uint64_t turn = first, ratio = step < 1.0L ? (uint64_t)(step * two64) : 0;
    for (int a = 0, i = 0; a < q->n_axes; a++) {
        const int len = (int)n->p.i[P_SECTION + a];
        if (by_axis && len) {
            f = unit, step = expl(-ln_base / len);
            turn = first, ratio = step < 1.0L ? (uint64_t)(step * two64) : 0;
        }
        for (int j = 0; j < len; j++, i++) {
            q->axis[i] = (unsigned char)a;
            if (ratio) {
                q->turns[i] = turn;
                turn = (uint64_t)(((unsigned __int128)turn * ratio + ((uint64_t)1 << 63)) >> 64);
            } else {
                q->turns[i] = (uint64_t)((f - floorl(f)) * two64);
                f *= step;
            }
        }
    }
    return 1;
}

static nc_status rope_fwd(nc_node *n) {
    nck_rope q;
    if (!rope_of(n, &q)) return NC_ERR_OOM;
    nck_rope_fwd(nc__k(n->out->ctx), &q, (float *)n->out->data);
    return NC_OK;
}

static void rope_bwd(nc_node *n) {
    nck_rope q;
    nc_tensor *in[3] = {n->in[0], input(n, HAS_WQ), input(n, HAS_WK)};
    float *g[3] = {NULL, NULL, NULL};
    int acc[3] = {1, 1, 1};
    if (!rope_of(n, &q)) return;
    for (int k = 0; k < 3; k++) {
        if (!in[k] || !nc__needs_grad(in[k])) continue;
        if (k == 2 && in[2] == in[1]) {
            g[2] = g[1];
            continue;
        }
        nc_tensor *t = nc__grad_buf_set(in[k], &acc[k]);
        if (!t) return;
        g[k] = (float *)t->data;
    }
    if (g[2] && g[2] == g[1]) { /* one weight for all heads: its two sums are added one after the other */
        nck_rope_bwd(nc__k(n->out->ctx), &q, (const float *)n->out->grad->data, g[0], acc[0], g[1], acc[1], NULL, 1);
        nck_rope_bwd(nc__k(n->out->ctx), &q, (const float *)n->out->grad->data, NULL, 1, NULL, 1, g[2], 1);
        return;
    }
    nck_rope_bwd(nc__k(n->out->ctx), &q, (const float *)n->out->grad->data, g[0], acc[0], g[1], acc[1], g[2], acc[2]);
}

const nc_op_def nc_op_qk_norm_rope = {"qk_norm_rope", 0, 0, rope_infer, NULL, rope_fwd, rope_bwd};

nc_tensor *nc_ext_qk_norm_rope(nc_tensor *x, nc_tensor *q_weight, nc_tensor *k_weight, nc_tensor *positions,
                               const nc_ext_rope_opts *opts) {
    if (!x) return NULL;
    if (!opts) {
        nc__error(x->ctx, NC_ERR_ARG, "qk_norm_rope: opts must not be NULL");
        return NULL;
    }
    nc_tensor *in[4] = {x, NULL, NULL, NULL};
    nc_tensor *more[3] = {q_weight, k_weight, positions};
    nc_op_params p;
    memset(&p, 0, sizeof p);
    int k = 1;
    for (int i = 0; i < 3; i++)
        if (more[i]) in[k++] = more[i], p.i[P_HAS] |= 1 << i;
    p.i[P_QHEADS] = opts->q_heads;
    p.i[P_AXES] = opts->n_axes;
    for (int a = 0; a < 3; a++) p.i[P_SECTION + a] = opts->sections[a];
    p.i[P_FLAGS] = opts->flags;
    p.f[0] = opts->base;
    p.f[1] = opts->eps;
    return nc__apply(&nc_op_qk_norm_rope, in, k, &p);
}
