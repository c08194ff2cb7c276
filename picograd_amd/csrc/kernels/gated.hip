// Gated feed-forward layer: h = act(g) u over z = x W + b = [g | u], and the
// backward of that product.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "convert16.h"
#include "gate_act.h"
#include "launch.h"

namespace {

__global__ void __launch_bounds__(256) k_gated_act(int act, const float *__restrict__ z, size_t m, size_t f, float *h32,
                                                   uint16_t *h16, int dtype)
{
    const size_t n = m * f;
    gate_switch(act, [&](auto code) {
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
            const size_t r = i / f, c = i - r * f;
            const float h = gate_f<decltype(code)::value>(z[r * 2 * f + c]) * z[r * 2 * f + f + c];
            if (h32)
                h32[i] = h;
            if (h16)
                h16[i] = to16(dtype, h);
        }
    });
}

// dz over a strip of 64 columns of f and a run of rows per block; its four
// waves take every fourth row each and keep the strip's column sums, joined
// through LDS in wave order into the block's row of part
__global__ void __launch_bounds__(256)
    k_gated_bwd(int act, const void *__restrict__ dh, int dh_dtype, const float *__restrict__ z, size_t m, size_t f,
                size_t f8, uint16_t *__restrict__ dz, int dtype, float *__restrict__ part, int rows)
{
    __shared__ float sums[4][2][64];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const size_t c = (size_t)blockIdx.x * 64 + lane;
    const size_t r0 = (size_t)blockIdx.y * rows, r1 = r0 + rows < m ? r0 + rows : m;
    float sg = 0.0f, su = 0.0f;
    gate_switch(act, [&](auto code) {
        for (size_t r = r0 + wave; r < r1; r += 4) {
            float dg = 0.0f, du = 0.0f;
            if (c < f) {
                const float d = dh_dtype == 0 ? ((const float *)dh)[r * f + c]
                                              : from16(dh_dtype, ((const uint16_t *)dh)[r * f + c]);
                float da;
                const float a = gate_fd<decltype(code)::value>(z[r * 2 * f + c], da);
                dg = d * z[r * 2 * f + f + c] * da;
                du = d * a;
                sg += dg;
                su += du;
            }
            if (c < f8) {
                dz[r * 2 * f8 + c] = to16(dtype, dg);
                dz[r * 2 * f8 + f8 + c] = to16(dtype, du);
            }
        }
    });
    if (!part)
        return;
    sums[wave][0][lane] = sg;
    sums[wave][1][lane] = su;
    __syncthreads();
    if (wave < 2 && c < f)
        part[(size_t)blockIdx.y * 2 * f + wave * f + c] =
            sums[0][wave][lane] + sums[1][wave][lane] + sums[2][wave][lane] + sums[3][wave][lane];
}

// rows per block: about 2048 blocks, at most 256 of them along the rows (the
// partial column sums)
struct bwd_plan {
    unsigned gx, gy;
    int rows;
};
bwd_plan plan_bwd(size_t m, size_t f)
{
    const size_t gx = (f + 63) / 64;
    size_t gy = 2048 / gx ? 2048 / gx : 1;
    gy = gy > 256 ? 256 : gy;
    size_t rows = (m + gy - 1) / gy;
    rows = (rows + 3) / 4 * 4;
    return {(unsigned)gx, (unsigned)((m + rows - 1) / rows), (int)rows};
}

} // namespace

extern "C" int pgk_gated_act(int act, const float *z, size_t m, size_t f, float *h32, uint16_t *h16, int dtype,
                             pgk_stream s)
{
    const size_t n = m * f;
    if (!n)
        return 0;
    const unsigned g = (unsigned)((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096);
    hipLaunchKernelGGL(k_gated_act, dim3(g), dim3(256), 0, (hipStream_t)s, act, z, m, f, h32, h16, dtype);
    return (int)hipGetLastError();
}

extern "C" size_t pgk_gated_bwd_workspace(size_t m, size_t f) { return m && f ? plan_bwd(m, f).gy * 2 * f * sizeof(float) : 0; }

extern "C" int pgk_gated_bwd(int act, const void *dh, int dh_dtype, const float *z, size_t m, size_t f, uint16_t *dz16,
                             int dtype, float *db, int db_beta, void *ws, pgk_stream s)
{
    if (!m || !f)
        return 0;
    if (m > 0x7fffffff || f > 0x3fffffff || (db && !ws))
        return (int)hipErrorInvalidValue;
    const bwd_plan p = plan_bwd(m, f);
    hipLaunchKernelGGL(k_gated_bwd, dim3(p.gx, p.gy), dim3(256), 0, (hipStream_t)s, act, dh, dh_dtype, z, m, f,
                       (f + 7) & ~(size_t)7, dz16, dtype, db ? (float *)ws : nullptr, p.rows);
    const int rc = (int)hipGetLastError();
    if (rc || !db)
        return rc;
    const pgk_colsum_job job = {(const float *)ws, p.gy, 2 * f, db, db_beta};
    return pgk_colsum_run(&job, s);
}
