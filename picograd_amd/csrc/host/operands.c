/*
 * Operands of the calls that write into tensors of the caller
 * (pg_amd_distill, pg_amd_gated, pg_amd_mx4_*): inputs may be strided views,
 * outputs are contiguous and may not overlap what the call reads.
 */
#include "internal.h"

const pg_tensor *pgo_input(const char *what, const pg_tensor *t, pg_tensor **owned)
{
    *owned = NULL;
    if (!t || (!t->dev && t->numel) || !pg_dtype_is_float(t->dtype)) {
        pga_set_err("%s: null tensor", what);
        return NULL;
    }
    pgt_materialize((pg_tensor *)t);
    const pg_tensor *c = pgt_contiguous(t, owned);
    if (!c)
        pga_set_err("%s: %s", what, pg_amd_last_error());
    return c;
}

/* the bytes from t's first to its last element */
static void span(const pg_tensor *t, const char **lo, const char **hi)
{
    size_t last = 0;
    for (size_t d = 0; d < t->ndim; d++)
        last += t->shape[d] ? (t->shape[d] - 1) * t->stride[d] : 0;
    *lo = t->dev;
    *hi = *lo + (t->numel ? (last + 1) * t->elem_size : 0);
}

bool pgo_output_ok(const char *what, const pg_tensor *t, const pg_tensor *const *in, size_t nin)
{
    if (!t || (!t->dev && t->numel) || !pgt_is_contiguous(t)) {
        pga_set_err("%s: an output must be a contiguous tensor", what);
        return false;
    }
    const char *lo, *hi, *a, *b;
    span(t, &lo, &hi);
    for (size_t i = 0; i < nin; i++) {
        if (!in[i])
            continue;
        span(in[i], &a, &b);
        if (a < hi && lo < b) {
            pga_set_err("%s: an output overlaps another operand", what);
            return false;
        }
    }
    return true;
}

void pgo_output(pg_tensor *t)
{
    pgm_colsum_flush_for(t); /* a deferred write of its own lands first */
    pgt_overwrite(t);
    t->pg_flags &= ~PG_TENSOR_ZERO_PENDING;
    pgt_touch(t);
}
