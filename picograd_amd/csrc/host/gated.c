/*
 * Gated feed-forward layer h = act(x Wg + bg) * (x Wu + bu): the calls on
 * tensors of the caller (pg_amd_gated, pg_amd_gated_backward) and the autograd
 * node (pg_amd_ag_gated16).  W = [Wg | Wu] [K, 2F] is one matrix, so the two
 * products of the backward are one dgrad and one wgrad over [dg | du].
 *
 * The 16-bit operands have rows of whole 16-byte pieces: x as [M, K8], W as
 * [K8, 2, F8] (K8, F8: K, F rounded up to 8, zeros between), dz as [M, 2, F8].
 */
#include "internal.h"

#include <stdlib.h>

static size_t up8(size_t x) { return (x + 7) & ~(size_t)7; }

typedef struct {
    size_t M, K, F, K8, F8;
} gated_dims;

static bool act_ok(int act) { return act >= PGK_ACT_NONE && act <= PGK_ACT_SIGMOID; }

static bool dims_ok(const pg_tensor *x, const pg_tensor *w, const pg_tensor *b, gated_dims *d)
{
    if (x->ndim != 2 || w->ndim != 2 || x->shape[1] != w->shape[0] || w->shape[1] % 2 ||
        (b && b->numel != w->shape[1]))
        return false;
    *d = (gated_dims){x->shape[0], x->shape[1], w->shape[1] / 2, up8(x->shape[1]), up8(w->shape[1] / 2)};
    return d->M <= 0x7fffff00 && d->K <= 0x3fffffff && d->F <= 0x1fffffff;
}

/* z (when given) and h of the layer; h in f32 (h32) and / or 16 bits (h16) */
static bool forward(const char *what, int dt, const gated_dims *d, int act, const uint16_t *x16, const uint16_t *w16,
                    const float *bias, float *z, float *h32, uint16_t *h16)
{
    int tk = pgd_tbegin(PGD_T_GEMM16);
    const int rc = pgk_gated_forward(dt, act, d->M, d->F, d->K8, x16, d->K8, w16, d->F8, bias, z, h32, h16, pgd_stream());
    pgd_tend(tk);
    return pgd_check(rc, what);
}

/* an output of a product: f32 (beta: added to) or 16 bits, at p with leading
 * dim ld; p NULL: not wanted */
typedef struct {
    void *p;
    bool is16;
    int beta;
} gated_out;

static bool product(const char *what, int dt, int t, size_t m, size_t n, size_t k, const uint16_t *a, size_t lda,
                    size_t aext, const uint16_t *b, size_t ldb, size_t bext, const gated_out *o, size_t ldc)
{
    if (!o->is16)
        return pgm_gemm16x(dt, t, t, m, n, k, a, lda, 0, aext, b, ldb, 0, bext, o->p, ldc, 0, 1, o->beta, NULL, what);
    const pgk_epi epi = {.act = PGK_ACT_NONE, .c16 = o->p, .dtype16 = dt, .skip_out = 1};
    return pgm_gemm16x(dt, t, t, m, n, k, a, lda, 0, aext, b, ldb, 0, bext, NULL, ldc, 0, 1, 0, &epi, what);
}

/* both grads in one launch; false: not for these sizes (nothing launched) or an
 * error, which the products alone then meet again */
static bool both_grads(int dt, const pgk_gemm_desc *dd, uint16_t *d16, const pgk_gemm_desc *dw, uint16_t *w16)
{
    const size_t wb = pgk_gemm16_grads_workspace(dd, dw);
    void *ws = wb ? pgd_malloc(wb) : NULL;
    if (wb && !ws)
        return false;
    int tk = pgd_tbegin(PGD_T_GEMM16);
    const int rc = pgk_gemm16_grads(dt, dd, d16, dw, w16, ws, pgd_stream());
    pgd_tend(tk);
    if (ws)
        pgd_free(ws, wb);
    return rc == 0;
}

/* dx = dz W^T and dW = x^T dz from dz16 [M, 2, F8]; M, K, F > 0.  An odd F's dW
 * is a batch of two halves, F apart in its rows. */
static bool grads(const char *what, int dt, const gated_dims *d, const uint16_t *x16, const uint16_t *w16,
                  const uint16_t *dz16, const gated_out *dx, const gated_out *dw)
{
    const size_t N = 2 * d->F, N8 = 2 * d->F8, halves = N == N8 ? 1 : 2, n = N / halves, n8 = N8 / halves;
    if (dx->p && dw->p && dx->p != dw->p) {
        const pgk_gemm_desc dd = {d->M, d->K, N8, dz16, N8, 0, d->M, w16, N8, 0, d->K, dx->is16 ? NULL : dx->p, d->K, 0, 1,
                                  dx->beta};
        const pgk_gemm_desc dg = {d->K, n, d->M, x16, d->K8, 0, d->K8, dz16, N8, n8, n8, dw->is16 ? NULL : dw->p, N, n, halves,
                                  dw->beta};
        const bool f32 = !dx->is16 && !dw->is16 && halves == 1;
        if ((f32 && pgm_pair_ks(dt, &dd, &dg, what)) ||
            both_grads(dt, &dd, dx->is16 ? dx->p : NULL, &dg, dw->is16 ? dw->p : NULL) ||
            (f32 && pgm_pair_full(dt, &dd, &dg, what)))
            return true;
    }
    bool ok = true;
    if (dx->p)
        ok = product(what, dt, 0, d->M, d->K, N8, dz16, N8, d->M, w16, N8, d->K, dx, d->K);
    if (dw->p && halves == 1) {
        ok = ok && product(what, dt, 1, d->K, N, d->M, x16, d->K8, d->K8, dz16, N8, N8, dw, N);
    } else if (ok && dw->p) {
        const pgk_epi epi = {.act = PGK_ACT_NONE, .c16 = dw->p, .dtype16 = dt, .skip_out = 1};
        ok = pgm_gemm16x(dt, 1, 1, d->K, n, d->M, x16, d->K8, 0, d->K8, dz16, N8, n8, n8, dw->is16 ? NULL : dw->p, N, n, 2,
                         dw->is16 ? 0 : dw->beta, dw->is16 ? &epi : NULL, what);
    }
    return ok;
}

/* dz16 (allocated, M * 2 * F8) and db from dh and z */
static uint16_t *make_dz(const char *what, int dt, const gated_dims *d, int act, const pg_tensor *dh, const float *z,
                         float *db, int db_beta)
{
    const size_t bytes = d->M * 2 * d->F8 * 2, wb = db ? pgk_gated_bwd_workspace(d->M, d->F) : 0;
    uint16_t *dz = pgd_malloc(bytes);
    void *ws = wb ? pgd_malloc(wb) : NULL;
    bool ok = dz && (ws || !wb) &&
              pgd_check(pgk_gated_bwd(act, dh->dev, (int)dh->dtype, z, d->M, d->F, dz, dt, db, db_beta, ws,
                                      pgd_stream()),
                        what);
    if (ws)
        pgd_free(ws, wb);
    if (!ok && dz)
        pgd_free(dz, bytes);
    return ok ? dz : NULL;
}

/* few rows (pgk_gated_few_grads_ok): all grads from f32 dz, x and W as they lie (x
 * rows ldx apart, W's halves `half`) */
static bool few_rows(const char *what, int dt, const gated_dims *d, int act, const pg_tensor *dh, const float *z, float *db,
                     int db_beta, const uint16_t *x, size_t ldx, const uint16_t *w, size_t half, const gated_out *dx,
                     const gated_out *dw)
{
    const size_t bytes = d->M * 2 * d->F * sizeof(float);
    const size_t wb = dx->p ? pgk_gated_few_grads_workspace(d->M, d->K, d->F) : 0;
    float *dz = pgd_malloc(bytes);
    void *ws = wb ? pgd_malloc(wb) : NULL;
    pgk_stream st = pgd_stream();
    int tk = pgd_tbegin(PGD_T_GEMM16);
    bool ok = dz && (ws || !wb) &&
              pgd_check(pgk_gated_few_dz(act, dh->dev, (int)dh->dtype, z, d->M, d->F, dz, db, db_beta, st), what);
    /* x and W in one storage: its grads one after the other */
    const bool apart = dx->p && dx->p == dw->p;
    for (int i = apart ? 0 : 1; ok && i < 2 && (dx->p || dw->p); i++)
        ok = pgd_check(pgk_gated_few_grads(dt, dz, d->M, d->K, d->F, x, ldx, w, half, apart && i ? NULL : dx->p,
                                           dx->is16 ? dt : 0, dx->beta, apart && !i ? NULL : dw->p, dw->is16 ? dt : 0,
                                           dw->beta, ws, st),
                       what);
    pgd_tend(tk);
    if (ws)
        pgd_free(ws, wb);
    if (dz)
        pgd_free(dz, bytes);
    return ok;
}

/* ---------------------------------------------------------------- on tensors */

static bool aligned16(const void *p) { return !((uintptr_t)p & 15); }

/* x [M, K8] and W [K8, 2, F8]: where they lie, or padded copies */
typedef struct {
    const uint16_t *x, *w;
    uint16_t *ox, *ow;
    size_t bx, bw;
} gated_ops;

static bool stage(const gated_dims *d, const pg_tensor *x, const pg_tensor *w, gated_ops *o)
{
    *o = (gated_ops){x->dev, w->dev, NULL, NULL, 0, 0};
    if (!d->K)
        return true;
    if (d->K != d->K8 || !aligned16(x->dev)) {
        o->bx = d->M * d->K8 * 2;
        o->x = o->ox = pgd_malloc(o->bx);
        if (!o->x)
            return false;
    }
    if (d->K != d->K8 || d->F != d->F8 || !aligned16(w->dev)) {
        o->bw = d->K8 * 2 * d->F8 * 2;
        o->w = o->ow = pgd_malloc(o->bw);
        if (!o->w)
            return false;
    }
    return !(o->ox || o->ow) ||
           pgd_check(pgk_gated_pad(x->dev, d->M, d->K, o->ox, w->dev, d->F, o->ow, pgd_stream()), "gated operands");
}

static void unstage(const gated_ops *o)
{
    if (o->ox)
        pgd_free(o->ox, o->bx);
    if (o->ow)
        pgd_free(o->ow, o->bw);
}

static bool shape_is(const pg_tensor *t, size_t a, size_t b)
{
    return t->ndim == 2 && t->shape[0] == a && t->shape[1] == b;
}

/* the checks that both calls share */
static bool call_ok(const char *what, const pg_tensor *x, const pg_tensor *w, const pg_tensor *b, int act, gated_dims *d)
{
    if (!x || !w) {
        pga_set_err("%s: null operand", what);
        return false;
    }
    if (!act_ok(act)) {
        pga_set_err("%s: act must be one of PG_ACT_* (0 to 4)", what);
        return false;
    }
    if ((x->dtype != PG_DTYPE_F16 && x->dtype != PG_DTYPE_BF16) || w->dtype != x->dtype ||
        (b && b->dtype != PG_DTYPE_F32)) {
        pga_set_err("%s: x and w must share a 16-bit dtype, b must be f32", what);
        return false;
    }
    if (!dims_ok(x, w, b, d)) {
        pga_set_err("%s: needs x [M, K], w [K, 2F] and b [2F]", what);
        return false;
    }
    if (!pgd_ok()) {
        pga_set_err("%s: no device", what);
        return false;
    }
    return true;
}

/* a device error as the autograd error too */
static bool done(const char *what, bool ok)
{
    if (!ok)
        pga_set_err("%s: %s", what, pg_amd_last_error());
    return ok;
}

bool pg_amd_gated(const pg_tensor *x, const pg_tensor *w, const pg_tensor *b, int act, pg_tensor *h, pg_tensor *z)
{
    static const char *const what = "pg_amd_gated";
    gated_dims d;
    if (!call_ok(what, x, w, b, act, &d))
        return false;
    if (!h || !shape_is(h, d.M, d.F) || (h->dtype != x->dtype && h->dtype != PG_DTYPE_F32) ||
        (z && (!shape_is(z, d.M, 2 * d.F) || z->dtype != PG_DTYPE_F32))) {
        pga_set_err("%s: h must be [M, F] of x's dtype or f32, z f32 [M, 2F]", what);
        return false;
    }
    const pg_tensor *in[4] = {x, w, b, z};
    if (!pgo_output_ok(what, h, in, 4) || (z && !pgo_output_ok(what, z, in, 3)))
        return false;
    if (!d.M || !d.F)
        return true;
    pg_tensor *own[3] = {NULL, NULL, NULL};
    const pg_tensor *xc = pgo_input(what, x, &own[0]), *wc = xc ? pgo_input(what, w, &own[1]) : NULL;
    const pg_tensor *bc = wc && b ? pgo_input(what, b, &own[2]) : NULL;
    bool ok = wc && (bc || !b);
    if (ok) {
        gated_ops o;
        pgo_output(h);
        if (z)
            pgo_output(z);
        ok = done(what, stage(&d, xc, wc, &o) &&
                            forward(what, (int)x->dtype, &d, act, o.x, o.w, bc ? bc->dev : NULL, z ? z->dev : NULL,
                                    h->dtype == PG_DTYPE_F32 ? h->dev : NULL,
                                    h->dtype == PG_DTYPE_F32 ? NULL : h->dev));
        unstage(&o);
    }
    for (int i = 0; i < 3; i++)
        pg_tensor_free(own[i]);
    return ok;
}

bool pg_amd_gated_backward(const pg_tensor *x, const pg_tensor *w, const pg_tensor *z, const pg_tensor *dh, int act,
                           pg_tensor *dx, pg_tensor *dw, pg_tensor *db)
{
    static const char *const what = "pg_amd_gated_backward";
    gated_dims d;
    if (!call_ok(what, x, w, NULL, act, &d))
        return false;
    if (!z || !dh || !shape_is(z, d.M, 2 * d.F) || z->dtype != PG_DTYPE_F32 || !shape_is(dh, d.M, d.F) ||
        (dh->dtype != x->dtype && dh->dtype != PG_DTYPE_F32)) {
        pga_set_err("%s: needs z f32 [M, 2F] and dh [M, F] of x's dtype or f32", what);
        return false;
    }
    if ((dx && (!shape_is(dx, d.M, d.K) || (dx->dtype != x->dtype && dx->dtype != PG_DTYPE_F32))) ||
        (dw && (!shape_is(dw, d.K, 2 * d.F) || (dw->dtype != x->dtype && dw->dtype != PG_DTYPE_F32))) ||
        (db && (db->numel != 2 * d.F || db->dtype != PG_DTYPE_F32))) {
        pga_set_err("%s: dx must be [M, K] and dw [K, 2F], of x's dtype or f32, db f32 [2F]", what);
        return false;
    }
    const pg_tensor *in[7] = {x, w, z, dh, dx, dw, db};
    if ((db && !pgo_output_ok(what, db, in, 6)) || (dw && !pgo_output_ok(what, dw, in, 5)) ||
        (dx && !pgo_output_ok(what, dx, in, 4)))
        return false;
    pg_tensor *outs[3] = {dx, dw, db};
    for (int i = 0; i < 3; i++)
        if (outs[i] && outs[i]->numel)
            pgo_output(outs[i]);
    if (!d.M || !d.F) { /* sums over nothing */
        for (int i = 0; i < 3; i++)
            if (outs[i] && outs[i]->numel)
                pg_tensor_fill(outs[i], 0.0f);
        return true;
    }
    pg_tensor *own[4] = {NULL, NULL, NULL, NULL};
    const pg_tensor *xc = pgo_input(what, x, &own[0]), *wc = xc ? pgo_input(what, w, &own[1]) : NULL;
    const pg_tensor *zc = wc ? pgo_input(what, z, &own[2]) : NULL, *hc = zc ? pgo_input(what, dh, &own[3]) : NULL;
    bool ok = hc != NULL;
    if (ok) {
        const int dt = (int)x->dtype;
        float *const b = db ? db->dev : NULL;
        const gated_out ox = {dx && d.K ? dx->dev : NULL, dx && dx->dtype != PG_DTYPE_F32, 0};
        const gated_out ow = {dw && d.K ? dw->dev : NULL, dw && dw->dtype != PG_DTYPE_F32, 0};
        if (pgk_gated_few_grads_ok(d.M, d.K, d.F)) {
            ok = few_rows(what, dt, &d, act, hc, zc->dev, b, 0, xc->dev, d.K, wc->dev, d.F, &ox, &ow);
        } else {
            gated_ops o = {0};
            uint16_t *dz = make_dz(what, dt, &d, act, hc, zc->dev, b, 0);
            ok = dz && stage(&d, xc, wc, &o) && grads(what, dt, &d, o.x, o.w, dz, &ox, &ow);
            unstage(&o);
            if (dz)
                pgd_free(dz, d.M * 2 * d.F8 * 2);
        }
        done(what, ok);
    }
    for (int i = 0; i < 4; i++)
        pg_tensor_free(own[i]);
    return ok;
}

/* ---------------------------------------------------------------- node */

typedef struct {
    int dt, act;
    pg_tensor *z; /* pre-activations [g | u], NULL when no grad is needed */
} gated_ctx;

void pgo_gated_free_ctx(void *ctx)
{
    gated_ctx *cx = ctx;
    if (cx)
        pg_tensor_free(cx->z);
    free(cx);
}

/* q(x) and q(W): the copies kept with their storages where those have the
 * layout, else staged ones; with x and W in one storage W's is always staged
 * (the two would share the one kept copy) */
static bool operands(const gated_dims *d, int dt, pg_tensor *x, pg_tensor *w, bool want_x, bool want_w, gated_ops *o)
{
    *o = (gated_ops){0};
    if (want_x && !(o->x = pgm_operand16(x, dt, d->M, d->K, d->M, d->K8, &o->ox, &o->bx)))
        return false;
    if (!want_w)
        return true;
    if (x->data_ref == w->data_ref) {
        pgt_materialize(w);
        o->w = o->ow = pgm_stage16(dt, 0, w->dev, 2 * d->K, d->F, d->F, 2 * d->K8, d->F8, 1, 0, &o->bw);
    } else if (d->F == d->F8) {
        o->w = pgm_operand16(w, dt, d->K, 2 * d->F, d->K8, 2 * d->F, &o->ow, &o->bw);
    } else {
        o->w = pgm_operand16(w, dt, 2 * d->K, d->F, 2 * d->K8, d->F8, &o->ow, &o->bw);
    }
    return o->w != NULL;
}

void pgo_gated_backward(pg_node *n)
{
    static const char *const what = "gated16 backward";
    pg_node *px = n->parents[0], *pw = n->parents[1], *pb = n->nparents > 2 ? n->parents[2] : NULL;
    const gated_ctx *cx = n->ctx;
    gated_dims d;
    if (!dims_ok(px->value, pw->value, NULL, &d) || !d.M || !d.F || !cx->z)
        return;
    pgt_materialize(n->grad);
    int bb = 0, bx = 0, bw = 0;
    pg_tensor *gb = pb && pb->requires_grad ? pga_grad_for_write(pb, &bb) : NULL;
    float *const db = gb ? gb->dev : NULL;
    const bool few = pgk_gated_few_grads_ok(d.M, d.K, d.F);
    uint16_t *dz = few ? NULL : make_dz(what, cx->dt, &d, cx->act, n->grad, cx->z->dev, db, bb);
    if (!dz && !few)
        return;
    pg_tensor *gx = d.K && px->requires_grad ? pga_grad_for_write(px, &bx) : NULL;
    pg_tensor *gw = d.K && pw->requires_grad ? pga_grad_for_write(pw, &bw) : NULL;
    gated_ops o;
    if (operands(&d, cx->dt, px->value, pw->value, gw != NULL, gx != NULL, &o)) {
        const gated_out ox = {gx ? gx->dev : NULL, false, bx}, ow = {gw ? gw->dev : NULL, false, bw};
        if (few)
            few_rows(what, cx->dt, &d, cx->act, n->grad, cx->z->dev, db, bb, o.x, d.K8, o.w, d.F8, &ox, &ow);
        else
            grads(what, cx->dt, &d, o.x, o.w, dz, &ox, &ow);
    }
    unstage(&o);
    if (dz)
        pgd_free(dz, d.M * 2 * d.F8 * 2);
}

pg_node *pg_amd_ag_gated16(pg_node *x, pg_node *w, pg_node *b, int act, pg_dtype dtype)
{
    static const char *const what = "gated16";
    if (!x || !w || !x->value || !w->value || (b && !b->value)) {
        pga_set_err("%s: null operand", what);
        return NULL;
    }
    if (dtype != PG_DTYPE_F16 && dtype != PG_DTYPE_BF16) {
        pga_set_err("%s: dtype must be PG_DTYPE_F16 or PG_DTYPE_BF16", what);
        return NULL;
    }
    if (!act_ok(act)) {
        pga_set_err("%s: act must be one of PG_ACT_* (0 to 4)", what);
        return NULL;
    }
    pg_tensor *xv = x->value, *wv = w->value, *bv = b ? b->value : NULL;
    gated_dims d;
    if (xv->dtype != PG_DTYPE_F32 || wv->dtype != PG_DTYPE_F32 || !pgt_is_contiguous(xv) || !pgt_is_contiguous(wv) ||
        (bv && (bv->dtype != PG_DTYPE_F32 || !pgt_is_contiguous(bv)))) {
        pga_set_err("%s: operands must be contiguous f32", what);
        return NULL;
    }
    if (!dims_ok(xv, wv, bv, &d)) {
        pga_set_err("%s: needs x [M, K], W [K, 2F] and b [2F]", what);
        return NULL;
    }
    if (!pgd_ok()) {
        pga_set_err("%s: no device", what);
        return NULL;
    }
    /* x's and W's f32 elements are read only to make a 16-bit copy */
    if (xv->pg_flags & PG_TENSOR_ZERO_PENDING)
        pgt_materialize(xv);
    if (wv->pg_flags & PG_TENSOR_ZERO_PENDING)
        pgt_materialize(wv);
    if (bv)
        pgt_materialize(bv);
    const int dt = (int)dtype;
    const bool grad = pg_autograd_is_grad_enabled() &&
                      (x->requires_grad || w->requires_grad || (b && b->requires_grad));
    pg_tensor *out = pgt_alloc(PG_DTYPE_F32, 2, (size_t[]){d.M, d.F});
    pg_tensor *z = grad ? pgt_alloc(PG_DTYPE_F32, 2, (size_t[]){d.M, 2 * d.F}) : NULL;
    gated_ctx *cx = calloc(1, sizeof *cx);
    bool ok = out && cx && (z || !grad);
    /* h's 16-bit copy, kept as its shadow for the next layer */
    if (ok && d.F % 8 == 0 && d.M * d.F) {
        pg_data_ref *r = out->data_ref;
        r->shadow = pgd_malloc(d.M * d.F * 2);
        r->shadow_bytes = d.M * d.F * 2;
        r->shadow_dtype = dt;
        r->shadow_stale = true;
        ok = r->shadow != NULL;
    }
    if (ok && d.M && d.F) {
        gated_ops o = {0};
        ok = (!d.K || operands(&d, dt, xv, wv, true, true, &o)) &&
             forward(what, dt, &d, act, o.x, o.w, bv ? bv->dev : NULL, z ? z->dev : NULL, out->dev,
                     out->data_ref->shadow);
        unstage(&o);
        if (ok && out->data_ref->shadow)
            out->data_ref->shadow_stale = false;
    }
    if (!ok) {
        done(what, false);
        pg_tensor_free(out);
        pg_tensor_free(z);
        free(cx);
        return NULL;
    }
    *cx = (gated_ctx){dt, act, z};
    pg_node *n = pga_attach(out, b ? 3 : 2, (pg_node *[]){x, w, b}, pgo_gated_backward, NULL, PG_AG_OP_MATMUL);
    if (n && n->backward)
        n->ctx = cx;
    else
        pgo_gated_free_ctx(cx);
    return n;
}
