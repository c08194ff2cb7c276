/*
 * Layer norm over the last dimension: the calls on tensors of the caller
 * (pg_amd_layernorm, pg_amd_layernorm_backward) and the autograd node
 * (pg_ag_layernorm).
 */
#include "internal.h"

#include <math.h>
#include <stdlib.h>

/* x's rows and their length; false with the error set */
static bool rows_of(const char *what, const pg_tensor *x, size_t *m, size_t *d)
{
    if (!x || !x->ndim || !x->shape[x->ndim - 1] || x->shape[x->ndim - 1] > PGK_NORM_MAX_D) {
        pga_set_err("%s: needs x [.., D] with D from 1 to 2^28", what);
        return false;
    }
    *d = x->shape[x->ndim - 1];
    *m = x->numel / *d;
    if (*m > 0x7fffffff) {
        pga_set_err("%s: more than 2^31 - 1 rows", what);
        return false;
    }
    return true;
}

static bool weights_ok(const char *what, const pg_tensor *w, const pg_tensor *b, size_t d)
{
    if ((w && (w->dtype != PG_DTYPE_F32 || w->numel != d)) || (b && (b->dtype != PG_DTYPE_F32 || b->numel != d))) {
        pga_set_err("%s: weight and bias must be f32 [D]", what);
        return false;
    }
    return true;
}

static bool eps_ok(const char *what, float eps)
{
    if (eps >= 0.0f && isfinite(eps))
        return true;
    pga_set_err("%s: eps must be finite and at least 0", what);
    return false;
}

static bool same_shape(const pg_tensor *a, const pg_tensor *b)
{
    return a && pg_shape_equal(a->ndim, a->shape, b->ndim, b->shape);
}

static bool device(const char *what)
{
    if (pgd_ok())
        return true;
    pga_set_err("%s: no device", what);
    return false;
}

/* a launch with its workspace, which is freed in stream order */
static bool run(const char *what, const pgk_norm_args *a, bool backward)
{
    const size_t wb = backward ? pgk_norm_bwd_workspace(a->dtype, a->m, a->d, a->dw || a->db)
                               : pgk_norm_workspace(a->dtype, a->m, a->d);
    pgk_stream st = pgd_stream();
    void *ws = wb ? pgd_malloc(wb) : NULL;
    const bool ok = (ws || !wb) && pgd_check(backward ? pgk_norm_bwd(a, ws, st) : pgk_norm(a, ws, st), what);
    if (ws)
        pgd_free(ws, wb);
    if (!ok)
        pga_set_err("%s: %s", what, pg_amd_last_error());
    return ok;
}

/* ---------------------------------------------------------------- on tensors */

bool pg_amd_layernorm(const pg_tensor *x, const pg_tensor *w, const pg_tensor *b, float eps, pg_tensor *y,
                      pg_tensor *stats)
{
    static const char *const what = "pg_amd_layernorm";
    size_t m, d;
    if (!rows_of(what, x, &m, &d) || !weights_ok(what, w, b, d) || !eps_ok(what, eps))
        return false;
    if (!same_shape(y, x) || (y->dtype != x->dtype && y->dtype != PG_DTYPE_F32) ||
        (stats && (stats->dtype != PG_DTYPE_F32 || stats->numel != 2 * m))) {
        pga_set_err("%s: y must have x's shape and its dtype or f32, stats f32 [M, 2]", what);
        return false;
    }
    if (!device(what))
        return false;
    /* y may take x's place */
    const bool inplace = y->dev == x->dev && y->dtype == x->dtype && pgt_is_contiguous(x);
    const pg_tensor *in[4] = {w, b, stats, x}, *sin[4] = {w, b, x, y};
    if (!pgo_output_ok(what, y, in, inplace ? 3 : 4) || (stats && !pgo_output_ok(what, stats, sin, 4)))
        return false;
    if (!m)
        return true;
    pg_tensor *own[3] = {NULL, NULL, NULL};
    const pg_tensor *xc = pgo_input(what, x, &own[0]), *wc = xc && w ? pgo_input(what, w, &own[1]) : NULL;
    const pg_tensor *bc = xc && b ? pgo_input(what, b, &own[2]) : NULL;
    bool ok = xc && (wc || !w) && (bc || !b);
    if (ok) {
        pgo_output(y);
        if (stats)
            pgo_output(stats);
        const pgk_norm_args a = {.x = xc->dev, .dtype = (int)x->dtype, .m = m, .d = d, .w = wc ? wc->dev : NULL,
                                 .b = bc ? bc->dev : NULL, .eps = eps, .y = y->dev, .y_dtype = (int)y->dtype,
                                 .stats = stats ? stats->dev : NULL};
        ok = run(what, &a, false);
    }
    for (int i = 0; i < 3; i++)
        pg_tensor_free(own[i]);
    return ok;
}

bool pg_amd_layernorm_backward(const pg_tensor *x, const pg_tensor *w, const pg_tensor *stats, const pg_tensor *dy,
                               pg_tensor *dx, pg_tensor *dw, pg_tensor *db)
{
    static const char *const what = "pg_amd_layernorm_backward";
    size_t m, d;
    if (!rows_of(what, x, &m, &d) || !weights_ok(what, w, NULL, d))
        return false;
    if (!stats || stats->dtype != PG_DTYPE_F32 || stats->numel != 2 * m || !same_shape(dy, x) ||
        (dy->dtype != x->dtype && dy->dtype != PG_DTYPE_F32)) {
        pga_set_err("%s: needs stats f32 [M, 2] and dy of x's shape and its dtype or f32", what);
        return false;
    }
    if ((dx && (!same_shape(dx, x) || (dx->dtype != x->dtype && dx->dtype != PG_DTYPE_F32))) ||
        (dw && (dw->dtype != PG_DTYPE_F32 || dw->numel != d)) || (db && (db->dtype != PG_DTYPE_F32 || db->numel != d))) {
        pga_set_err("%s: dx must have x's shape and its dtype or f32, dw and db f32 [D]", what);
        return false;
    }
    if (!device(what))
        return false;
    const pg_tensor *in[7] = {x, w, stats, dy, dx, dw, db};
    if ((db && !pgo_output_ok(what, db, in, 6)) || (dw && !pgo_output_ok(what, dw, in, 5)) ||
        (dx && !pgo_output_ok(what, dx, in, 4)))
        return false;
    pg_tensor *outs[3] = {dx, dw, db}, *own[4] = {NULL, NULL, NULL, NULL};
    if (!m || !(dx || dw || db)) { /* sums over nothing, or nothing wanted */
        for (int i = 1; i < 3; i++)
            if (outs[i]) {
                pgo_output(outs[i]);
                pg_tensor_fill(outs[i], 0.0f);
            }
        return true;
    }
    const pg_tensor *xc = pgo_input(what, x, &own[0]), *wc = xc && w ? pgo_input(what, w, &own[1]) : NULL;
    const pg_tensor *sc = xc ? pgo_input(what, stats, &own[2]) : NULL, *gc = sc ? pgo_input(what, dy, &own[3]) : NULL;
    bool ok = gc && (wc || !w);
    if (ok) {
        for (int i = 0; i < 3; i++)
            if (outs[i])
                pgo_output(outs[i]);
        const pgk_norm_args a = {.x = xc->dev, .dtype = (int)x->dtype, .m = m, .d = d, .w = wc ? wc->dev : NULL,
                                 .stats = sc->dev, .dy = gc->dev, .dy_dtype = (int)dy->dtype, .dx = dx ? dx->dev : NULL,
                                 .dx_dtype = dx ? (int)dx->dtype : PG_DTYPE_F32, .dw = dw ? dw->dev : NULL,
                                 .db = db ? db->dev : NULL};
        ok = run(what, &a, true);
    }
    for (int i = 0; i < 4; i++)
        pg_tensor_free(own[i]);
    return ok;
}

/* ---------------------------------------------------------------- node */

typedef struct {
    pg_tensor *stats; /* NULL when no grad is needed */
    bool has_w, has_b; /* parents: x, then the weight, then the bias */
} norm_ctx;

void pgo_layernorm_free_ctx(void *ctx)
{
    norm_ctx *cx = ctx;
    if (cx)
        pg_tensor_free(cx->stats);
    free(cx);
}

void pgo_layernorm_backward(pg_node *n)
{
    static const char *const what = "layernorm backward";
    const norm_ctx *cx = n->ctx;
    pg_node *px = n->parents[0], *pw = cx->has_w ? n->parents[1] : NULL, *pb = cx->has_b ? n->parents[1 + cx->has_w] : NULL;
    size_t m, d;
    if (!cx->stats || !rows_of(what, px->value, &m, &d) || !m)
        return;
    pgt_materialize(px->value);
    if (pw)
        pgt_materialize(pw->value);
    pgt_materialize(n->grad);
    pgk_norm_args a = {.x = px->value->dev, .m = m, .d = d, .w = pw ? pw->value->dev : NULL, .stats = cx->stats->dev,
                       .dy = n->grad->dev};
    pg_tensor *gx = px->requires_grad ? pga_grad_for_write(px, &a.beta_x) : NULL;
    pg_tensor *gw = pw && pw->requires_grad ? pga_grad_for_write(pw, &a.beta_w) : NULL;
    pg_tensor *gb = pb && pb->requires_grad ? pga_grad_for_write(pb, &a.beta_b) : NULL;
    /* a node that is two of them takes its parts in calls of their own, one after
     * the other: within a call dx and the sums may be written at the same time */
    const bool w_apart = gw && pw == px, b_apart = gb && (pb == px || pb == pw);
    a.dx = gx ? gx->dev : NULL;
    a.dw = gw && !w_apart ? gw->dev : NULL;
    a.db = gb && !b_apart ? gb->dev : NULL;
    if ((a.dx || a.dw || a.db) && !run(what, &a, true))
        return;
    a.dx = a.db = NULL;
    a.dw = w_apart ? gw->dev : NULL;
    if (a.dw && !run(what, &a, true))
        return;
    a.dw = NULL;
    a.db = b_apart ? gb->dev : NULL;
    if (a.db)
        run(what, &a, true);
}

/* a node's value as an operand: f32, contiguous, its elements current */
static bool operand(const char *what, const pg_node *n)
{
    if (!n || !n->value || !n->value->dev || n->value->dtype != PG_DTYPE_F32 || !pgt_is_contiguous(n->value)) {
        pga_set_err("%s: operands must be contiguous f32 nodes", what);
        return false;
    }
    return true;
}

pg_node *pg_ag_layernorm(pg_node *x, pg_node *weight, pg_node *bias, float eps)
{
    static const char *const what = "pg_ag_layernorm";
    size_t m, d;
    if (!operand(what, x) || (weight && !operand(what, weight)) || (bias && !operand(what, bias)) ||
        !rows_of(what, x->value, &m, &d) ||
        !weights_ok(what, weight ? weight->value : NULL, bias ? bias->value : NULL, d) || !eps_ok(what, eps) || !device(what))
        return NULL;
    const bool grad = pg_autograd_is_grad_enabled() && (x->requires_grad || (weight && weight->requires_grad) ||
                                                        (bias && bias->requires_grad));
    pg_tensor *y = pgt_alloc(PG_DTYPE_F32, x->value->ndim, x->value->shape);
    pg_tensor *stats = grad && y ? pgt_alloc(PG_DTYPE_F32, 2, (size_t[]){m, 2}) : NULL;
    norm_ctx *cx = calloc(1, sizeof *cx);
    bool ok = y && cx && (stats || !grad);
    if (!ok)
        pga_set_err("%s: out of memory", what);
    if (ok && m) {
        pgt_materialize(x->value);
        if (weight)
            pgt_materialize(weight->value);
        if (bias)
            pgt_materialize(bias->value);
        const pgk_norm_args a = {.x = x->value->dev, .m = m, .d = d, .w = weight ? weight->value->dev : NULL,
                                 .b = bias ? bias->value->dev : NULL, .eps = eps, .y = y->dev,
                                 .stats = stats ? stats->dev : NULL};
        ok = run(what, &a, false);
    }
    if (!ok) {
        pg_tensor_free(y);
        pg_tensor_free(stats);
        free(cx);
        return NULL;
    }
    *cx = (norm_ctx){stats, weight != NULL, bias != NULL};
    pg_node *parents[3] = {x};
    size_t np = 1;
    if (weight)
        parents[np++] = weight;
    if (bias)
        parents[np++] = bias;
    pg_node *n = pga_attach(y, np, parents, pgo_layernorm_backward, NULL, PG_AG_OP_LAYERNORM);
    if (n && n->backward)
        n->ctx = cx;
    else
        pgo_layernorm_free_ctx(cx);
    return n;
}
