/*
 * Distillation of a student's logits from a teacher's top logits
 * (pg_amd_distill, pg_amd_ag_distill): argument checks and the autograd node
 * around pgk_distill.  The reference has no such loss; its cross entropy
 * (autograd.h:131) is the case without a teacher.
 */
#include "internal.h"

#include <math.h>
#include <stdlib.h>

static const char *const WHAT = "pg_amd_distill";

/* the checks of the inputs' types and shapes; false with the error set */
static bool inputs_ok(const pg_tensor *logits, const pg_tensor *top, const pg_tensor *idx, const pg_tensor *labels,
                      const pg_amd_distill_cfg *cfg)
{
    if (!logits || !top || !idx || !cfg) {
        pga_set_err("%s: null operand", WHAT);
        return false;
    }
    if (logits->ndim != 2 || top->ndim != 2 || idx->ndim != 2 || top->shape[0] != logits->shape[0] ||
        idx->shape[0] != top->shape[0] || idx->shape[1] != top->shape[1] ||
        (labels && labels->numel != logits->shape[0])) {
        pga_set_err("%s: needs logits [N, V], top and top_idx [N, k] and labels [N]", WHAT);
        return false;
    }
    if (!logits->shape[1] || logits->shape[1] > PGK_DISTILL_MAX_V || !top->shape[1] ||
        top->shape[1] > PGK_DISTILL_TOP || logits->shape[0] > 0x7fffffff) {
        pga_set_err("%s: V must be 1 to 2^24 and k 1 to %d", WHAT, PGK_DISTILL_TOP);
        return false;
    }
    if (idx->dtype != PG_DTYPE_F32 || (labels && labels->dtype != PG_DTYPE_F32)) {
        pga_set_err("%s: indices and labels are whole numbers held as f32", WHAT);
        return false;
    }
    if (!(cfg->temperature > 0.0f) || !isfinite(cfg->temperature) || !(cfg->alpha >= 0.0f && cfg->alpha <= 1.0f) ||
        !isfinite(cfg->scale)) {
        pga_set_err("%s: needs a finite temperature > 0, alpha in [0, 1] and a finite scale", WHAT);
        return false;
    }
    if (!pgd_ok()) {
        pga_set_err("%s: no device", WHAT);
        return false;
    }
    return true;
}

/* one launch over checked operands; loss and ds are device addresses */
static bool launch(const pg_tensor *logits, const pg_tensor *top, const pg_tensor *idx, const pg_tensor *labels,
                   const pg_amd_distill_cfg *cfg, const float *up, float *loss, void *ds, pg_dtype ds_dtype, int beta)
{
    pgk_distill_args a = {.s = logits->dev, .dtype = (int)logits->dtype, .n = logits->shape[0], .v = logits->shape[1],
                          .t = top->dev, .top_dtype = (int)top->dtype, .idx = idx->dev,
                          .label = labels ? labels->dev : NULL, .top = (int)top->shape[1],
                          .temperature = cfg->temperature, .alpha = cfg->alpha, .scale = cfg->scale, .up = up,
                          .loss = loss, .ds = ds, .ds_dtype = (int)ds_dtype, .beta = beta};
    const size_t wb = pgk_distill_workspace(&a);
    void *ws = wb ? pgd_malloc(wb) : NULL; /* freed in stream order */
    const bool ok = (ws || !wb) && pgd_check(pgk_distill(&a, ws, pgd_stream()), WHAT);
    if (ws)
        pgd_free(ws, wb);
    if (ok)
        return true;
    pga_set_err("%s", pg_amd_last_error());
    return false;
}

bool pg_amd_distill(const pg_tensor *logits, const pg_tensor *top, const pg_tensor *top_idx, const pg_tensor *labels,
                    const pg_amd_distill_cfg *cfg, pg_tensor *loss, pg_tensor *dlogits)
{
    if (!inputs_ok(logits, top, top_idx, labels, cfg))
        return false;
    if (!loss || loss->dtype != PG_DTYPE_F32 || loss->numel != logits->shape[0]) {
        pga_set_err("%s: loss must be f32 [N]", WHAT);
        return false;
    }
    if (dlogits && (dlogits->ndim != 2 || dlogits->shape[0] != logits->shape[0] ||
                    dlogits->shape[1] != logits->shape[1] ||
                    (dlogits->dtype != logits->dtype && dlogits->dtype != PG_DTYPE_F32))) {
        pga_set_err("%s: dlogits must be [N, V], of the logits' dtype or f32", WHAT);
        return false;
    }
    /* the grad may take the logits' own place */
    const bool inplace = dlogits && dlogits->dev == logits->dev && dlogits->dtype == logits->dtype &&
                         pgt_is_contiguous(logits);
    const pg_tensor *in[5] = {top, top_idx, labels, logits, dlogits};
    if (!pgo_output_ok(WHAT, loss, in, 5) || (dlogits && !pgo_output_ok(WHAT, dlogits, in, inplace ? 3 : 4)))
        return false;
    pg_tensor *own[4] = {NULL, NULL, NULL, NULL};
    const pg_tensor *s = pgo_input(WHAT, logits, &own[0]);
    const pg_tensor *t = s ? pgo_input(WHAT, top, &own[1]) : NULL;
    const pg_tensor *i = t ? pgo_input(WHAT, top_idx, &own[2]) : NULL;
    const pg_tensor *l = i && labels ? pgo_input(WHAT, labels, &own[3]) : NULL;
    bool ok = i && (l || !labels);
    if (ok && s->numel) {
        pgo_output(loss);
        if (dlogits)
            pgo_output(dlogits);
        ok = launch(s, t, i, l, cfg, NULL, loss->dev, dlogits ? dlogits->dev : NULL,
                    dlogits ? dlogits->dtype : PG_DTYPE_F32, 0);
    }
    for (int k = 0; k < 4; k++)
        pg_tensor_free(own[k]);
    return ok;
}

/* ---------------------------------------------------------------- node */

typedef struct {
    pg_tensor *top, *idx, *labels; /* views or copies of the caller's, held */
    pg_amd_distill_cfg cfg;
} distill_ctx;

void pgo_distill_free_ctx(void *ctx)
{
    distill_ctx *cx = ctx;
    if (cx) {
        pg_tensor_free(cx->top);
        pg_tensor_free(cx->idx);
        pg_tensor_free(cx->labels);
    }
    free(cx);
}

void pgo_distill_backward(pg_node *n)
{
    const distill_ctx *cx = n->ctx;
    pg_node *p = n->parents[0];
    if (!p->requires_grad || !p->value->numel)
        return;
    pgt_materialize(p->value);
    pgt_materialize(n->grad);
    int beta = 0;
    pg_tensor *g = pga_grad_for_write(p, &beta);
    if (g)
        launch(p->value, cx->top, cx->idx, cx->labels, &cx->cfg, n->grad->dev, NULL, g->dev, PG_DTYPE_F32, beta);
}

/* t's elements in row-major order, held past the caller's own reference */
static pg_tensor *hold(const pg_tensor *t)
{
    pg_tensor *own = NULL;
    const pg_tensor *c = pgo_input("pg_amd_ag_distill", t, &own);
    if (!c)
        return NULL;
    if (own)
        return own;
    pg_tensor *v = pg_tensor_view(c);
    if (v) {
        v->view_parent = NULL; /* the view outlives the tensor it was made from */
    }
    return v;
}

pg_node *pg_amd_ag_distill(pg_node *logits, const pg_tensor *top, const pg_tensor *top_idx, const pg_tensor *labels,
                           const pg_amd_distill_cfg *cfg)
{
    const pg_tensor *s = logits ? logits->value : NULL;
    if (!inputs_ok(s, top, top_idx, labels, cfg))
        return NULL;
    if (s->dtype != PG_DTYPE_F32 || !pgt_is_contiguous(s)) {
        pga_set_err("pg_amd_ag_distill: logits must be a contiguous f32 node");
        return NULL;
    }
    pgt_materialize(logits->value);
    const size_t N = s->shape[0];
    distill_ctx *cx = calloc(1, sizeof *cx);
    pg_tensor *rows = pgt_alloc(PG_DTYPE_F32, 1, (size_t[]){N});
    pg_tensor *value = pgt_alloc(PG_DTYPE_F32, 1, (size_t[]){1});
    bool ok = cx && rows && value;
    if (ok) {
        cx->cfg = *cfg;
        cx->top = hold(top);
        cx->idx = hold(top_idx);
        cx->labels = labels ? hold(labels) : NULL;
        ok = cx->top && cx->idx && (cx->labels || !labels);
    }
    if (ok && N)
        ok = launch(s, cx->top, cx->idx, cx->labels, cfg, NULL, rows->dev, NULL, PG_DTYPE_F32, 0);
    if (ok) /* in a fixed order */
        ok = pgd_check(N ? pgk_sum_vec_f32(rows->dev, value->dev, N, 1.0f, pgd_stream())
                         : pgk_fill_f32(value->dev, 1, 0.0f, pgd_stream()),
                       "pg_amd_ag_distill");
    pg_tensor_free(rows);
    if (!ok) {
        pg_tensor_free(value);
        pgo_distill_free_ctx(cx);
        return NULL;
    }
    pg_node *n = pga_attach(value, 1, &logits, pgo_distill_backward, NULL, PG_AG_OP_CROSS_ENTROPY);
    if (n && n->backward)
        n->ctx = cx;
    else
        pgo_distill_free_ctx(cx);
    return n;
}
