/*
 * Matrices held in 4 bits with a power of two per 32 values (pg_amd_mx4_*):
 * their storage, argument checks and the product of a rounded tensor with one.
 */
#include "internal.h"

#include <stdlib.h>

struct pg_amd_mx4 {
    pgk_mx4 q;
    size_t code_bytes, power_bytes;
    int axis; /* the source's dimension that the blocks run along */
};

static void release(pg_amd_mx4 *m)
{
    if (m->q.codes)
        pgd_free(m->q.codes, m->code_bytes);
    if (m->q.powers)
        pgd_free(m->q.powers, m->power_bytes);
    m->q.codes = m->q.powers = NULL;
}

static bool reserve(pg_amd_mx4 *m, size_t rows, size_t cols)
{
    pgk_mx4_shape(&m->q, rows, cols, &m->code_bytes, &m->power_bytes);
    m->q.codes = pgd_malloc(m->code_bytes);
    m->q.powers = pgd_malloc(m->power_bytes);
    if (m->q.codes && m->q.powers)
        return true;
    release(m);
    return false;
}

/* sizes that the kernels' 32-bit indices hold */
static bool fits(size_t rows, size_t cols) { return rows && cols && rows <= 0x3fffffff && cols <= (size_t)1 << 24; }

pg_amd_mx4 *pg_amd_mx4_quantize(const pg_tensor *t, int axis)
{
    static const char *const what = "pg_amd_mx4_quantize";
    if (!t || t->ndim != 2 || (axis != 0 && axis != 1) || !fits(t->shape[1 - axis], t->shape[axis])) {
        pga_set_err("%s: needs a matrix that is not empty, of up to 2^24 along axis 0 or 1", what);
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
    pg_amd_mx4 *m = calloc(1, sizeof *m);
    bool ok = m && reserve(m, t->shape[1 - axis], t->shape[axis]) &&
              pgd_check(pgk_mx4_quantize(&m->q, c->dev, (int)c->dtype, axis == 0, pgd_stream()), what);
    pg_tensor_free(own);
    if (!ok) {
        pga_set_err("%s: %s", what, m ? pg_amd_last_error() : "out of memory");
        pg_amd_mx4_free(m);
        return NULL;
    }
    m->axis = axis;
    return m;
}

void pg_amd_mx4_free(pg_amd_mx4 *q)
{
    if (q)
        release(q);
    free(q);
}

size_t pg_amd_mx4_bytes(const pg_amd_mx4 *q) { return q ? q->code_bytes + q->power_bytes : 0; }

bool pg_amd_mx4_dequantize(const pg_amd_mx4 *q, pg_tensor *out)
{
    static const char *const what = "pg_amd_mx4_dequantize";
    if (!q || !out || out->ndim != 2 || out->shape[q->axis] != q->q.cols || out->shape[1 - q->axis] != q->q.rows ||
        !pg_dtype_is_float(out->dtype)) {
        pga_set_err("%s: needs a matrix of the source's shape", what);
        return false;
    }
    if (!pgo_output_ok(what, out, NULL, 0))
        return false;
    pgo_output(out);
    if (pgd_check(pgk_mx4_dequantize(&q->q, out->dev, (int)out->dtype, q->axis == 0, pgd_stream()), what))
        return true;
    pga_set_err("%s", pg_amd_last_error());
    return false;
}

bool pg_amd_mx4_matmul(const pg_tensor *x, const pg_amd_mx4 *w, pg_tensor *y)
{
    static const char *const what = "pg_amd_mx4_matmul";
    if (!x || !w || !y || x->ndim != 2 || y->ndim != 2 || w->axis != 0 || x->shape[1] != w->q.cols ||
        y->shape[0] != x->shape[0] || y->shape[1] != w->q.rows || !pg_dtype_is_float(y->dtype) ||
        x->shape[0] > 0x3fffffff) {
        pga_set_err("%s: needs x [M, K], W [K, N] with its blocks along K and y [M, N]", what);
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
    pg_amd_mx4 t = {0}; /* x in 4 bits, freed in stream order */
    bool ok;
    if (pgk_mx4_few_rows(x->shape[0]))
        ok = pgd_check(pgk_mx4_matmul_few(c->dev, (int)c->dtype, x->shape[0], &w->q, y->dev, (int)y->dtype,
                                          pgd_stream()),
                       what);
    else
        ok = reserve(&t, x->shape[0], x->shape[1]) &&
             pgd_check(pgk_mx4_quantize(&t.q, c->dev, (int)c->dtype, 0, pgd_stream()), what) &&
             pgd_check(pgk_mx4_matmul(&t.q, &w->q, y->dev, (int)y->dtype, pgd_stream()), what);
    release(&t);
    pg_tensor_free(own);
    if (!ok)
        pga_set_err("%s: %s", what, pg_amd_last_error());
    return ok;
}
