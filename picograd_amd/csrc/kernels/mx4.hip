// Matrices in 4 bits: e2m1 values (0, .5, 1, 1.5, 2, 3, 4, 6 and their
// negatives) with one power of two for each 32 along the reduction, and their
// product on the block-scaled matrix instructions.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "convert16.h"
#include "launch.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kBlock = 32; // values under one power of two

__device__ __forceinline__ float ld_any(int dtype, const void *p, size_t i)
{
    return dtype == 0 ? ((const float *)p)[i] : dtype == 1 ? (float)((const _Float16 *)p)[i] : (float)((const __bf16 *)p)[i];
}
__device__ __forceinline__ void st_any(int dtype, void *p, size_t i, float v)
{
    if (dtype == 0)
        ((float *)p)[i] = v;
    else
        ((uint16_t *)p)[i] = to16(dtype, v);
}

// The block's exponent byte for its largest magnitude, given as the bits of
// |v| (whose order is that of the magnitudes, infinities and NaN last):
// floor(log2) - 2 with the bias, 0 at least; 255 for a block with either.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top)
{
    const uint32_t e = top >> 23;
    return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
__device__ __forceinline__ float scale_of(uint32_t byte)
{
    return byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u); // 2^-127 is subnormal
}

// eight values in 4 bits each, the first in the low bits; the hardware
// conversion rounds v / scale to nearest even and past 6 to 6
__device__ __forceinline__ uint32_t pack8(const float *v, float scale)
{
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
    return r;
}

__device__ __forceinline__ uint8_t *scale_at(const pgk_mx4 &q, size_t row, size_t blk)
{
    return q.scales + ((blk >> 3) * q.rows_p + row) * 8 + (blk & 7);
}

// One thread per block of 32 values.
__global__ void __launch_bounds__(256) k_mx4_quantize(pgk_mx4 q, const void *__restrict__ src, int dtype, int trans)
{
    const size_t nb = q.pitch / 16, n = nb * q.rows;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        // along the source's contiguous dimension
        const size_t row = trans ? i % q.rows : i / nb, blk = trans ? i / q.rows : i % nb;
        float v[kBlock];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < kBlock; ++j) {
            const size_t c = blk * kBlock + j;
            v[j] = c < q.cols ? ld_any(dtype, src, trans ? c * q.rows + row : row * q.cols + c) : 0.0f;
            const uint32_t a = __float_as_uint(v[j]) & 0x7fffffffu;
            top = a > top ? a : top;
        }
        const uint32_t b = scale_byte(top);
        uint4 w = make_uint4(0, 0, 0, 0);
        if (b != 255) {
            const float s = scale_of(b);
            w = make_uint4(pack8(v, s), pack8(v + 8, s), pack8(v + 16, s), pack8(v + 24, s));
        }
        *(uint4 *)(q.codes + row * q.pitch + blk * 16) = w;
        *scale_at(q, row, blk) = (uint8_t)b;
    }
}

__device__ __forceinline__ float value_of(uint32_t code, uint32_t byte)
{
    const uint32_t m = code & 7;
    // e2m1: 0, .5, then (1 + m0 / 2) 2^(e - 1)
    const float a = m < 2 ? 0.5f * (float)m : (float)(2 + (m & 1)) * (float)(1 << (m >> 1)) * 0.25f;
    const float s = byte == 255 ? __uint_as_float(0x7fc00000u) : scale_of(byte);
    return (code & 8 ? -a : a) * s;
}

__global__ void __launch_bounds__(256) k_mx4_dequantize(pgk_mx4 q, void *__restrict__ dst, int dtype, int trans)
{
    const size_t n = q.rows * q.cols;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t row = trans ? i % q.rows : i / q.cols, c = trans ? i / q.rows : i % q.cols;
        const uint32_t code = q.codes[row * q.pitch + c / 2] >> (4 * (c & 1));
        st_any(dtype, dst, i, value_of(code & 15, *scale_at(q, row, c / kBlock)));
    }
}

// One wave per 32 x 32 tile of y, the operands straight from memory: lane l
// gives row l % 32 and the block l / 32 of each pair of blocks.
__global__ void __launch_bounds__(64) k_mx4_tile32(pgk_mx4 x, pgk_mx4 w, void *__restrict__ y, int y_dtype)
{
    const int lane = (int)threadIdx.x, lr = lane & 31, lk = lane >> 5;
    const size_t m0 = (size_t)blockIdx.y * 32, n0 = (size_t)blockIdx.x * 32;
    const size_t rx = m0 + lr < x.rows ? m0 + lr : x.rows - 1, rw = n0 + lr < w.rows ? n0 + lr : w.rows - 1;
    const size_t nb = x.pitch / 16;
    f32x16 acc = {};
    for (size_t b0 = 0; b0 < nb; b0 += 2) {
        const size_t b = b0 + lk;
        uint4 a = make_uint4(0, 0, 0, 0), c = a;
        int sa = 127, sc = 127;
        if (b < nb) {
            a = *(const uint4 *)(x.codes + rx * x.pitch + b * 16);
            c = *(const uint4 *)(w.codes + rw * w.pitch + b * 16);
            sa = *scale_at(x, rx, b);
            sc = *scale_at(w, rw, b);
        }
        const v8i va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
        const v8i vc = {(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0};
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vc, acc, 4, 4, 0, sa, 0, sc);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const size_t m = m0 + (e >> 2) * 8 + lk * 4 + (e & 3), n = n0 + lr;
        if (m < x.rows && n < w.rows)
            st_any(y_dtype, y, m * w.rows + n, acc[e]);
    }
}

unsigned blocks_for(size_t n) { return (unsigned)((n + 255) / 256 < 8192 ? (n + 255) / 256 : 8192); }

} // namespace

extern "C" void pgk_mx4_shape(pgk_mx4 *q, size_t rows, size_t cols, size_t *code_bytes, size_t *scale_bytes)
{
    const size_t nb = (cols + kBlock - 1) / kBlock;
    q->rows = rows;
    q->cols = cols;
    q->pitch = nb * 16;
    q->rows_p = (rows + 15) & ~(size_t)15;
    *code_bytes = rows * q->pitch;
    *scale_bytes = (nb + 7) / 8 * q->rows_p * 8;
}

extern "C" int pgk_mx4_quantize(const pgk_mx4 *q, const void *src, int dtype, int trans, pgk_stream s)
{
    hipLaunchKernelGGL(k_mx4_quantize, dim3(blocks_for(q->rows * (q->pitch / 16))), dim3(256), 0, (hipStream_t)s, *q,
                       src, dtype, trans);
    return (int)hipGetLastError();
}

extern "C" int pgk_mx4_dequantize(const pgk_mx4 *q, void *dst, int dtype, int trans, pgk_stream s)
{
    hipLaunchKernelGGL(k_mx4_dequantize, dim3(blocks_for(q->rows * q->cols)), dim3(256), 0, (hipStream_t)s, *q, dst,
                       dtype, trans);
    return (int)hipGetLastError();
}

extern "C" int pgk_mx4_matmul(const pgk_mx4 *x, const pgk_mx4 *w, void *y, int y_dtype, pgk_stream s)
{
    if (x->cols != w->cols || x->rows > 65535 * (size_t)32)
        return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(k_mx4_tile32, dim3((unsigned)((w->rows + 31) / 32), (unsigned)((x->rows + 31) / 32)), dim3(64), 0,
                       (hipStream_t)s, *x, *w, y, y_dtype);
    return (int)hipGetLastError();
}
