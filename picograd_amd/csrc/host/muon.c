/*
 * Orthogonal factors of matrices (pg_amd_orthogonalise) and the optimiser that
 * steps along those of the momentum (pg_amd_muon_*), around pgk_muon.  The
 * reference's optimisers are SGD and Adam (opt/sgd.c, opt/adam.c); registration,
 * zero_grad and the state's file format follow theirs.
 */
#define _POSIX_C_SOURCE 200809L
#include "internal.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>

#define MOST_STEPS 100
/* matrices share launches up to this much workspace */
#define MOST_WORKSPACE ((size_t)8 << 30)

static bool sides_ok(const pg_tensor *t)
{
    return t->ndim == 2 && t->shape[0] && t->shape[1] && t->shape[0] <= PGK_MUON_MAX_SIDE &&
           t->shape[1] <= PGK_MUON_MAX_SIDE;
}

/* the matrices in groups of what one launch and the workspace hold */
static bool run(const char *what, const pgk_muon_seg *segs, size_t n, float mu, bool nesterov, int steps)
{
    for (size_t i = 0; i < n;) {
        size_t k = 1, wb = pgk_muon_workspace(segs + i, 1);
        while (i + k < n && k < PGK_MUON_MAX) {
            const size_t more = pgk_muon_workspace(segs + i, (int)k + 1);
            if (more > MOST_WORKSPACE)
                break;
            wb = more;
            k++;
        }
        pgk_stream st = pgd_stream();
        void *ws = wb ? pgd_malloc(wb) : NULL;
        const bool ok = (ws || !wb) && pgd_check(pgk_muon(segs + i, (int)k, mu, nesterov, steps, ws, st), what);
        if (ws)
            pgd_free(ws, wb); /* in stream order */
        if (!ok) {
            pga_set_err("%s: %s", what, pg_amd_last_error());
            return false;
        }
        i += k;
    }
    return true;
}

bool pg_amd_orthogonalise(const pg_tensor *g, int steps, pg_tensor *out)
{
    static const char *const what = "pg_amd_orthogonalise";
    if (!g || !sides_ok(g) || !out || !pg_shape_equal(out->ndim, out->shape, g->ndim, g->shape) ||
        !pg_dtype_is_float(out->dtype)) {
        pga_set_err("%s: needs a matrix with sides of 1 to 2^16 and an output of its shape", what);
        return false;
    }
    if (steps < 1 || steps > MOST_STEPS) {
        pga_set_err("%s: steps must be 1 to %d", what, MOST_STEPS);
        return false;
    }
    if (!pgd_ok()) {
        pga_set_err("%s: no device", what);
        return false;
    }
    /* out may take g's place */
    const bool inplace = out->dev == g->dev && out->dtype == g->dtype && pgt_is_contiguous(g);
    const pg_tensor *in[1] = {inplace ? NULL : g};
    if (!pgo_output_ok(what, out, in, 1))
        return false;
    pg_tensor *own;
    const pg_tensor *c = pgo_input(what, g, &own);
    if (!c)
        return false;
    pgo_output(out);
    const pgk_muon_seg seg = {.rows = g->shape[0], .cols = g->shape[1], .g = c->dev, .g_dtype = (int)g->dtype,
                              .out = out->dev, .out_dtype = (int)out->dtype};
    const bool ok = run(what, &seg, 1, 0.0f, false, steps);
    pg_tensor_free(own);
    return ok;
}

/* ---------------------------------------------------------------- optimiser */

typedef struct {
    pg_node *param;
    pg_tensor *buf; /* NULL without momentum */
} muon_state;

struct pg_amd_muon {
    pg_amd_muon_cfg cfg;
    muon_state *st;
    size_t n, cap;
};

pg_amd_muon_cfg pg_amd_muon_cfg_default(void)
{
    const pg_amd_muon_cfg c = {.lr = 0.02f, .momentum = 0.95f, .weight_decay = 0.0f, .rms = 0.0f, .steps = 5, .nesterov = true};
    return c;
}

static bool at_least_0(float v) { return v >= 0.0f && isfinite(v); }

pg_amd_muon *pg_amd_muon_new(const pg_amd_muon_cfg *cfg)
{
    const pg_amd_muon_cfg c = cfg ? *cfg : pg_amd_muon_cfg_default();
    if (!at_least_0(c.lr) || !at_least_0(c.momentum) || !at_least_0(c.weight_decay) || !at_least_0(c.rms) || c.steps < 1 ||
        c.steps > MOST_STEPS) {
        pga_set_err("pg_amd_muon_new: needs finite values of at least 0 and 1 to %d steps", MOST_STEPS);
        return NULL;
    }
    pg_amd_muon *o = calloc(1, sizeof *o);
    if (o)
        o->cfg = c;
    else
        pga_set_err("pg_amd_muon_new: out of memory");
    return o;
}

void pg_amd_muon_free(pg_amd_muon *opt)
{
    if (!opt)
        return;
    for (size_t i = 0; i < opt->n; i++) {
        pg_node_free(opt->st[i].param);
        pg_tensor_free(opt->st[i].buf);
    }
    free(opt->st);
    free(opt);
}

static bool value_ok(const pg_tensor *v)
{
    return v && v->dev && v->dtype == PG_DTYPE_F32 && sides_ok(v) && pgt_is_contiguous(v);
}

/* whether v shares memory with one of the first n parameters' values (with_grad: of
 * those that have a grad) */
static bool taken(const pg_amd_muon *opt, size_t n, const pg_tensor *v, bool with_grad)
{
    const char *lo = v->dev, *hi = lo + v->numel * 4;
    for (size_t i = 0; i < n; i++) {
        const pg_node *p = opt->st[i].param;
        const pg_tensor *o = p->value;
        if ((p->grad || !with_grad) && (const char *)o->dev < hi && lo < (const char *)o->dev + o->numel * 4)
            return true;
    }
    return false;
}

int pg_amd_muon_add_param(pg_amd_muon *opt, pg_node *param)
{
    static const char *const what = "pg_amd_muon_add_param";
    if (!opt || !param || !param->requires_grad || !value_ok(param->value)) {
        pga_set_err("%s: needs a contiguous f32 matrix node that requires grads, with sides of 1 to 2^16", what);
        return -1;
    }
    if (taken(opt, opt->n, param->value, false)) {
        pga_set_err("%s: the matrix is a parameter already", what);
        return -1;
    }
    if (opt->n == opt->cap) {
        const size_t nc = opt->cap ? opt->cap * 2 : 8;
        muon_state *p = realloc(opt->st, nc * sizeof *p);
        if (!p) {
            pga_set_err("%s: out of memory", what);
            return -1;
        }
        opt->st = p;
        opt->cap = nc;
    }
    pg_tensor *buf = NULL;
    if (opt->cfg.momentum != 0.0f && !(buf = pg_tensor_zeros(2, param->value->shape))) {
        pga_set_err("%s: %s", what, pg_amd_last_error());
        return -1;
    }
    opt->st[opt->n++] = (muon_state){pg_node_retain(param), buf};
    return 0;
}

size_t pg_amd_muon_num_params(const pg_amd_muon *opt) { return opt ? opt->n : 0; }

pg_tensor *pg_amd_muon_buffer(pg_amd_muon *opt, size_t i) { return opt && i < opt->n ? opt->st[i].buf : NULL; }

bool pg_amd_muon_set_lr(pg_amd_muon *opt, float lr)
{
    if (!opt || !at_least_0(lr)) {
        pga_set_err("pg_amd_muon_set_lr: needs an optimiser and a finite rate of at least 0");
        return false;
    }
    opt->cfg.lr = lr;
    return true;
}

float pg_amd_muon_get_lr(const pg_amd_muon *opt) { return opt ? opt->cfg.lr : 0.0f; }

void pg_amd_muon_zero_grad(pg_amd_muon *opt)
{
    for (size_t i = 0; opt && i < opt->n; i++) {
        pg_node *p = opt->st[i].param;
        pg_tensor_free(p->grad);
        p->grad = NULL;
    }
}

bool pg_amd_muon_step(pg_amd_muon *opt)
{
    static const char *const what = "pg_amd_muon_step";
    if (!opt || !pgd_ok()) {
        pga_set_err("%s: %s", what, opt ? "no device" : "null optimiser");
        return false;
    }
    const pg_amd_muon_cfg c = opt->cfg;
    /* a node's value may have been replaced since it was added */
    for (size_t i = 0; i < opt->n; i++) {
        const pg_tensor *v = opt->st[i].param->value, *g = opt->st[i].param->grad, *m = opt->st[i].buf;
        if (g && (!value_ok(v) || g->dtype != PG_DTYPE_F32 || !pgt_is_contiguous(g) ||
                  !pg_shape_equal(g->ndim, g->shape, v->ndim, v->shape))) {
            pga_set_err("%s: parameters and grads must be contiguous f32 of one shape", what);
            return false;
        }
        if (g && m && !pg_shape_equal(m->ndim, m->shape, v->ndim, v->shape)) {
            pga_set_err("%s: a parameter has another shape than its momentum", what);
            return false;
        }
        if (g && taken(opt, i, v, true)) {
            pga_set_err("%s: two parameters' matrices overlap", what);
            return false;
        }
    }
    pgk_muon_seg *segs = calloc(opt->n ? opt->n : 1, sizeof *segs);
    if (!segs) {
        pga_set_err("%s: out of memory", what);
        return false;
    }
    size_t ns = 0;
    for (size_t i = 0; i < opt->n; i++) {
        pg_tensor *v = opt->st[i].param->value, *g = opt->st[i].param->grad, *m = opt->st[i].buf;
        if (!g)
            continue;
        /* a pending clip scale is applied as the grad is read (and stays pending
         * for its other readers); what else is pending is written first */
        pg_data_ref *gr = g->data_ref, *r = v->data_ref;
        const bool clip = gr && gr->clip_pending && !gr->act_pending && !gr->narrow && !(g->pg_flags & PG_TENSOR_ZERO_PENDING);
        if (!clip)
            pgt_materialize(g);
        pgt_materialize(v);
        const double k = (double)v->shape[0], n = (double)v->shape[1];
        const double size = c.rms > 0.0f ? c.rms * sqrt(k > n ? k : n) : sqrt(n > k ? n / k : 1.0);
        pgk_muon_seg *q = &segs[ns++];
        *q = (pgk_muon_seg){.rows = v->shape[0], .cols = v->shape[1], .g = g->dev, .gclip = clip,
                            .gmul = clip ? gr->clip_mul : 1.0f, .ginv = clip ? gr->clip_inv : 1.0f, .m = m ? m->dev : NULL,
                            .w = v->dev, .decay = (float)(1.0 - (double)c.lr * c.weight_decay),
                            .step = (float)((double)c.lr * size)};
        if (m) {
            pgt_materialize(m);
            pgt_touch(m);
        }
        /* a 16-bit copy of the parameter kept for the products is rewritten with it */
        if (r && r->shadow && v->dev == r->ptr && v->numel * 4 == r->nbytes) {
            q->shadow = r->shadow;
            q->shadow_dtype = r->shadow_dtype;
            q->shadow_cols = r->shadow_cols;
            q->shadow_ld = r->shadow_ld;
            r->shadow_stale = false;
        } else {
            pgt_touch(v);
        }
    }
    const bool ok = run(what, segs, ns, c.momentum, c.nesterov, c.steps);
    for (size_t i = 0; !ok && i < opt->n; i++) /* copies of what was not written */
        pgt_touch(opt->st[i].param->value);
    free(segs);
    return ok;
}

/* ---------------------------------------------------------------- momentum checkpoint ("PGMU") */

bool pg_amd_muon_save_fp(const pg_amd_muon *opt, FILE *fp)
{
    if (!opt || !fp)
        return false;
    const uint32_t ver = 1;
    const uint64_t n = (uint64_t)opt->n;
    if (fwrite("PGMU", 1, 4, fp) != 4 || fwrite(&ver, 4, 1, fp) != 1 || fwrite(&n, 8, 1, fp) != 1)
        return false;
    for (size_t i = 0; i < opt->n; i++) {
        const uint32_t has = opt->st[i].buf ? 1u : 0u;
        if (fwrite(&has, 4, 1, fp) != 1 || (has && !pg_tensor_save_fp(opt->st[i].buf, fp)))
            return false;
    }
    return true;
}

bool pg_amd_muon_save(const pg_amd_muon *opt, const char *path)
{
    FILE *fp = path ? fopen(path, "wb") : NULL;
    if (!fp)
        return false;
    const bool ok = pg_amd_muon_save_fp(opt, fp);
    return fclose(fp) == 0 && ok;
}

bool pg_amd_muon_load_into_fp(pg_amd_muon *opt, FILE *fp)
{
    if (!opt || !fp)
        return false;
    char magic[4];
    uint32_t ver = 0;
    uint64_t n = 0;
    if (fread(magic, 1, 4, fp) != 4 || memcmp(magic, "PGMU", 4) != 0 || fread(&ver, 4, 1, fp) != 1 || ver != 1 ||
        fread(&n, 8, 1, fp) != 1 || n != (uint64_t)opt->n)
        return false;
    for (size_t i = 0; i < opt->n; i++) {
        uint32_t has = 0;
        if (fread(&has, 4, 1, fp) != 1 || has > 1)
            return false;
        pg_tensor *buf = opt->st[i].buf;
        if (has && (!buf || !pgc_load_into(buf, fp))) /* without momentum there is nowhere to load it */
            return false;
        if (!has && buf)
            pg_tensor_fill(buf, 0.0f);
    }
    return true;
}

bool pg_amd_muon_load_into(pg_amd_muon *opt, const char *path)
{
    FILE *fp = path ? fopen(path, "rb") : NULL;
    if (!fp)
        return false;
    const bool ok = pg_amd_muon_load_into_fp(opt, fp);
    fclose(fp);
    return ok;
}
