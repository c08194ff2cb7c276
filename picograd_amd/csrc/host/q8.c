/*
 * Matrices held in 8 bits with a scale per line along the reduction
 * (pg_amd_q8_*): their storage, argument checks and the product of a rounded
 * tensor with one.
 */
#include "internal.h"

#include <stdlib.h>

struct pg_amd_q8 {
    pgk_q8 q;
    size_t code_bytes, scale_bytes;
    int axis; /* the source's dimension that the lines run along */
};

static void release(pg_amd_q8 *m)
{
    if (m->q.codes)
        pgd_free(m->q.codes, m->code_bytes);
    if (m->q.scale)
        pgd_free(m->q.scale, m->scale_bytes);
    m->q.codes = NULL;
    m->q.scale = NULL;
}

static bool reserve(pg_amd_q8 *m, size_t rows, size_t cols)
{
    pgk_q8_shape(&m->q, rows, cols, &m->code_bytes, &m->scale_bytes);
    m->q.codes = pgd_malloc(m->code_bytes);
    m->q.scale = pgd_malloc(m->scale_bytes);
    if (m->q.codes && m->q.scale)
        return true;
    release(m);
    return false;
}

/* rounds dense elements into m's storage; the workspace is freed in stream order */
static bool quantize(const char *what, const pg_amd_q8 *m, const pg_tensor *c, int trans)
{
    const size_t wb = pgk_q8_workspace(&m->q, trans);
    void *ws = wb ? pgd_malloc(wb) : NULL;
    const bool ok = (ws || !wb) && pgd_check(pgk_q8_quantize(&m->q, c->dev, (int)c->dtype, trans, ws, pgd_stream()), what);
    if (ws)
        pgd_free(ws, wb);
    return ok;
}

/* what the kernels' sums and indices hold */
static bool fits(size_t rows, size_t cols) { return rows && cols && rows <= 0x3fffffff && cols <= PGK_Q8_MAX_K; }

pg_amd_q8 *pg_amd_q8_quantize(const pg_tensor *t, int axis)
{
    static const char *const what = "pg_amd_q8_quantize";
    if (!t || t->ndim != 2 || (axis != 0 && axis != 1) || !fits(t->shape[1 - axis], t->shape[axis])) {
        pga_set_err("%s: needs a matrix that is not empty, of up to 2^17 along axis 0 or 1", what);
        return NULL;
    }
    if (!pgd_ok()) {
        pga_set_err("%s: no device", what);
        return NULL;
    }
    pg_tensor *own;
    const pg_tensor *c = pgo_input(what, t, &own);
    if (!c)
        return NULL;
    pg_amd_q8 *m = calloc(1, sizeof *m);
    const bool ok = m && reserve(m, t->shape[1 - axis], t->shape[axis]) && quantize(what, m, c, axis == 0);
    pg_tensor_free(own);
    if (!ok) {
        pga_set_err("%s: %s", what, m ? pg_amd_last_error() : "out of memory");
        pg_amd_q8_free(m);
        return NULL;
    }
    m->axis = axis;
    return m;
}

void pg_amd_q8_free(pg_amd_q8 *q)
{
    if (q)
        release(q);
    free(q);
}

size_t pg_amd_q8_bytes(const pg_amd_q8 *q) { return q ? q->code_bytes + q->scale_bytes : 0; }

bool pg_amd_q8_dequantize(const pg_amd_q8 *q, pg_tensor *out)
{
    static const char *const what = "pg_amd_q8_dequantize";
    if (!q || !out || out->ndim != 2 || out->shape[q->axis] != q->q.cols || out->shape[1 - q->axis] != q->q.rows ||
        !pg_dtype_is_float(out->dtype)) {
        pga_set_err("%s: needs a matrix of the source's shape", what);
        return false;
    }
    if (!pgo_output_ok(what, out, NULL, 0))
        return false;
    pgo_output(out);
    if (pgd_check(pgk_q8_dequantize(&q->q, out->dev, (int)out->dtype, q->axis == 0, pgd_stream()), what))
        return true;
    pga_set_err("%s", pg_amd_last_error());
    return false;
}

bool pg_amd_q8_matmul(const pg_tensor *x, const pg_amd_q8 *w, pg_tensor *y)
{
    static const char *const what = "pg_amd_q8_matmul";
    if (!x || !w || !y || x->ndim != 2 || y->ndim != 2 || w->axis != 0 || x->shape[1] != w->q.cols ||
        y->shape[0] != x->shape[0] || y->shape[1] != w->q.rows || !pg_dtype_is_float(y->dtype) ||
        x->shape[0] > 0x3fffffff) {
        pga_set_err("%s: needs x [M, K], W [K, N] with its scales for the columns and y [M, N]", what);
        return false;
    }
    const pg_tensor *in[1] = {x};
    if (!pgo_output_ok(what, y, in, 1))
        return false;
    if (!x->shape[0])
        return true;
    pg_tensor *own;
    const pg_tensor *c = pgo_input(what, x, &own);
    if (!c)
        return false;
    pgo_output(y);
    const size_t M = x->shape[0];
    const bool few = pgk_q8_few_rows(M), fused = few && pgk_q8_few_fused(M, x->shape[1]);
    pg_amd_q8 t = {0}; /* x in 8 bits, freed in stream order */
    bool ok = fused || (reserve(&t, M, x->shape[1]) && quantize(what, &t, c, 0));
    if (ok) {
        pgk_stream st = pgd_stream();
        ok = pgd_check(few ? pgk_q8_matmul_few(c->dev, (int)c->dtype, fused ? NULL : &t.q, M, &w->q, y->dev, (int)y->dtype, st)
                           : pgk_q8_matmul(&t.q, &w->q, y->dev, (int)y->dtype, st),
                       what);
    }
    release(&t);
    pg_tensor_free(own);
    if (!ok)
        pga_set_err("%s: %s", what, pg_amd_last_error());
    return ok;
}
