// Matrices in 8 bits: whole numbers of -127 .. 127 with a scale for each row along
// the reduction, and their product on the integer matrix instructions.
//
// A row's scale is s = max |v| / 127 in f32, its codes v / s to nearest, ties to
// even.  y = (sum qx qw) sx sw: the sums are exact (32 bits hold 2^17 products), y
// is rounded once from three f32 factors.  A row that holds a NaN or an infinity
// has scale NaN.
//
// Codes lie as rows at a pitch of whole 128-byte pieces with zeros behind the end,
// so no product checks bounds along the reduction.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include <type_traits>

#include "launch.h"
#include "piece_tile.h"

namespace {

constexpr size_t kMostBlocks = (size_t)1 << 20; // of a grid; kernels loop past it

// ---------------------------------------------------------------- rounding

// A code from 1 / s: fma with 1.5 2^23 rounds v / s to a whole number in the low
// bits of the sum.  What is left over, v - q s, is exact in f32; where it reaches
// s / 2 (a tie, or 1 / s on the wrong side of one) or s is next to the subnormals
// the quotient is taken in 64 bits, which separates every quotient of two f32 from
// a tie.
constexpr float kRound = 12582912.0f;
constexpr float kLeastScale = 0x1p-120f;

__device__ __forceinline__ uint32_t code_exact(float v, float s)
{
    const double q = rint((double)v / (double)s);
    return (uint32_t)(int)fmin(fmax(q, -127.0), 127.0);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return lo | hi << 16;
}
// 16 values under scale s, inv = 1 / s; s 0 or NaN: zeros
__device__ __forceinline__ uint4 codes16(const float (&v)[16], float s, float inv)
{
    uint32_t b[16];
    if (!(s > 0.0f))
        return make_uint4(0, 0, 0, 0);
    float worst = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float t = fmaf(v[i], inv, kRound);
        worst = fmaxf(worst, fabsf(fmaf(kRound - t, s, v[i])));
        b[i] = __float_as_uint(t);
    }
    if (!(worst < 0.5f * s) || s < kLeastScale) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            b[i] = code_exact(v[i], s);
    }
    return make_uint4(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]), pack4(b[8], b[9], b[10], b[11]),
                      pack4(b[12], b[13], b[14], b[15]));
}
// a row's scale from the bits of its largest magnitude
__device__ __forceinline__ float scale_of(uint32_t top)
{
    return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(top) / 127.0f;
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t wave_top(uint32_t v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t a = (uint32_t)__shfl_xor((int)v, o);
        v = a > v ? a : v;
    }
    return v;
}

// elements 16 c .. of the row p [k], at any alignment; past the end: 0
template <class T>
__device__ __forceinline__ void load16(const T *p, size_t c, size_t k, float (&v)[16])
{
    constexpr int E = 16 / sizeof(T);
    typedef T tv __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    const size_t at = c * 16;
    if (at + 16 <= k) {
#pragma unroll
        for (int i = 0; i < 16 / E; ++i) {
            const tv q = *(const tv *)(p + at + i * E);
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[i * E + e] = (float)q[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            v[i] = at + i < k ? (float)p[at + i] : 0.0f;
    }
}
__device__ __forceinline__ uint32_t top16(const float (&v)[16], uint32_t top)
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t a = magnitude(v[i]);
        top = a > top ? a : top;
    }
    return top;
}

// Rows: TPR threads per row, two chunks of 16 values each held between the
// search for the largest and the rounding; LONG rows are read again.
template <class T, int TPR, bool LONG>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_q8_rows(pgk_q8 q, const T *__restrict__ src)
{
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1, R = 2;
    __shared__ uint32_t tops[2][TPR > 64 ? TPR / 64 : 1];
    const int tid = (int)threadIdx.x, lane = tid % TPR;
    const size_t nc = q.ld / 16;
    int turn = 0;
    for (size_t r0 = (size_t)blockIdx.x * RPB; r0 < q.rows; r0 += (size_t)gridDim.x * RPB, turn ^= 1) {
        const size_t row = r0 + tid / TPR;
        const bool in = row < q.rows;
        const T *p = src + (in ? row : 0) * q.cols;
        float v[R][16];
        uint32_t top = 0;
        if constexpr (LONG) {
            for (size_t c = lane; c < nc; c += TPR) {
                load16(p, c, q.cols, v[0]);
                top = top16(v[0], top);
            }
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if ((size_t)(lane + i * TPR) < nc)
                    load16(p, lane + i * TPR, q.cols, v[i]);
                else
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        v[i][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i)
                top = top16(v[i], top);
        }
        top = wave_top(top);
        if constexpr (TPR > 64) {
            if ((tid & 63) == 0)
                tops[turn][tid >> 6] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < TPR / 64; ++w)
                top = tops[turn][w] > top ? tops[turn][w] : top;
        }
        const float s = scale_of(top), inv = 1.0f / s;
        if (!in)
            continue;
        if (lane == 0)
            q.scale[row] = s;
        uint4 *out = (uint4 *)(q.codes + row * q.ld);
        if constexpr (LONG) {
            for (size_t c = lane; c < nc; c += TPR) {
                load16(p, c, q.cols, v[0]);
                out[c] = codes16(v[0], s, inv);
            }
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if ((size_t)(lane + i * TPR) < nc)
                    out[lane + i * TPR] = codes16(v[i], s, inv);
        }
    }
}

// Columns of src [cols, rows].  The largest of each, over a slab of kSlab of the
// reduction: 64 columns by four threads a block.
constexpr int kSlab = 256;

template <class T>
__global__ void __launch_bounds__(256) k_q8_tops(pgk_q8 q, const T *__restrict__ src, uint32_t *__restrict__ part,
                                                 size_t nx, size_t ny)
{
    __shared__ uint32_t s[4][64];
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
    for (size_t job = blockIdx.x; job < nx * ny; job += gridDim.x) {
        const size_t slab = job / nx, col = (job - slab * nx) * 64 + lane;
        const size_t k0 = slab * kSlab, end = k0 + kSlab < q.cols ? k0 + kSlab : q.cols;
        uint32_t top = 0;
        if (col < q.rows)
#pragma unroll 8
            for (size_t k = k0 + w; k < end; k += 4) {
                const uint32_t a = magnitude((float)src[k * q.rows + col]);
                top = a > top ? a : top;
            }
        s[w][lane] = top;
        __syncthreads();
        if (w == 0 && col < q.rows) {
#pragma unroll
            for (int i = 1; i < 4; ++i)
                top = s[i][lane] > top ? s[i][lane] : top;
            part[slab * q.rows + col] = top;
        }
        __syncthreads();
    }
}

// Codes of 64 columns by kSlab of the reduction: a thread rounds 64 values down a
// column, LDS turns them into pieces of the column's row.
template <class T>
__global__ void __launch_bounds__(256) k_q8_columns(pgk_q8 q, const T *__restrict__ src, const uint32_t *__restrict__ part,
                                                    int slabs, size_t nx, size_t ny)
{
    constexpr int PITCH = kSlab + 16;
    __shared__ uint4 piece[64 * PITCH / 16];
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
    for (size_t job = blockIdx.x; job < nx * ny; job += gridDim.x) {
        const size_t slab = job / nx, c0 = (job - slab * nx) * 64, col = c0 + lane, k0 = slab * kSlab;
        uint32_t top = 0;
        if (col < q.rows)
            for (int i = 0; i < slabs; ++i) {
                const uint32_t a = part[(size_t)i * q.rows + col];
                top = a > top ? a : top;
            }
        const float s = scale_of(top), inv = 1.0f / s;
        if (slab == 0 && w == 0 && col < q.rows)
            q.scale[col] = s;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const size_t k = k0 + w * 64 + i * 16 + e;
                v[e] = col < q.rows && k < q.cols ? (float)src[k * q.rows + col] : 0.0f;
            }
            piece[(lane * PITCH + w * 64) / 16 + i] = codes16(v, s, inv);
        }
        __syncthreads();
#pragma unroll
        for (int i = (int)threadIdx.x; i < 64 * (kSlab / 16); i += 256) {
            const int r = i / (kSlab / 16), c = i % (kSlab / 16);
            if (c0 + r < q.rows && k0 + c * 16 < q.ld)
                *(uint4 *)(q.codes + (c0 + r) * q.ld + k0 + c * 16) = piece[r * PITCH / 16 + c];
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- reading back

__device__ __forceinline__ float value_of(uint32_t word, int byte, float s)
{
    return (float)(int8_t)(word >> (8 * byte)) * s;
}

// Rows: four values a thread.
template <class O>
__global__ void __launch_bounds__(256) k_q8_back_rows(pgk_q8 q, O *__restrict__ dst)
{
    const size_t per = (q.cols + 3) / 4, n = per * q.rows;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t row = i / per, c = (i - row * per) * 4;
        const uint32_t w = *(const uint32_t *)(q.codes + row * q.ld + c);
        const float s = q.scale[row];
        O *p = dst + row * q.cols + c;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < q.cols)
                p[e] = (O)value_of(w, e, s);
    }
}

// Columns, as k_q8_columns takes them.
template <class O>
__global__ void __launch_bounds__(256) k_q8_back_columns(pgk_q8 q, O *__restrict__ dst, size_t nx, size_t ny)
{
    constexpr int PITCH = kSlab + 16;
    __shared__ uint4 piece[64 * PITCH / 16];
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
    for (size_t job = blockIdx.x; job < nx * ny; job += gridDim.x) {
        const size_t slab = job / nx, c0 = (job - slab * nx) * 64, col = c0 + lane, k0 = slab * kSlab;
#pragma unroll
        for (int i = (int)threadIdx.x; i < 64 * (kSlab / 16); i += 256) {
            const int r = i / (kSlab / 16), c = i % (kSlab / 16);
            if (c0 + r < q.rows && k0 + c * 16 < q.ld)
                piece[r * PITCH / 16 + c] = *(const uint4 *)(q.codes + (c0 + r) * q.ld + k0 + c * 16);
        }
        __syncthreads();
        const float s = col < q.rows ? q.scale[col] : 0.0f;
        if (col < q.rows)
#pragma unroll 4
            for (int i = 0; i < 16; ++i) {
                const uint32_t word = ((const uint32_t *)piece)[(lane * PITCH + w * 64) / 4 + i];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const size_t k = k0 + w * 64 + i * 4 + e;
                    if (k < q.cols)
                        dst[k * q.rows + col] = (O)value_of(word, e, s);
                }
            }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- products

// 16 x 16 over 64: a lane holds 16 values of row (column) lane % 16; lane l gets
// column l % 16 of rows 4 (l / 16) .. + 3
__device__ __forceinline__ i32x4 mma16(const uint4 &a, const uint4 &b, const i32x4 &c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// `n` neighbours of a row of y, at most four
template <class O>
__device__ __forceinline__ void put4(O *p, const float (&v)[4], int n)
{
    typedef O o4 __attribute__((ext_vector_type(4), aligned(sizeof(O))));
    if (n >= 4) {
        o4 q;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            q[e] = (O)v[e];
        *(o4 *)p = q;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n)
            p[e] = (O)v[e];
}

// Up to 16 rows of x: a thread block owns 16 columns of y and its waves split the
// reduction, so the weights stream past once.  FUSED: every block finds the rows'
// scales and rounds x by itself, no other launch; else xq holds them.  Bound by
// the loads' latency and the launch.
constexpr int kFewWaves = 8;

template <class T, class O, bool FUSED>
__global__ void __launch_bounds__(kFewWaves * 64, 1)
    k_q8_few(const T *__restrict__ x, pgk_q8 xq, int m, pgk_q8 w, O *__restrict__ y, size_t tiles)
{
    constexpr int U = 4; // steps of 64 in flight
    __shared__ int part[kFewWaves][16][17];
    __shared__ uint32_t tops[kFewWaves][16];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const size_t steps = w.ld / 64, k = w.cols;
    for (size_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const size_t n0 = tile * 16, wr = n0 + r < w.rows ? n0 + r : w.rows - 1;
        const uint8_t *const pw = (const uint8_t *)w.codes + wr * w.ld + g * 16;
        float s = 0.0f, inv = 0.0f;
        if constexpr (FUSED) {
            uint32_t top = 0;
            if (r < m)
                for (size_t st = wave; st < steps; st += kFewWaves) {
                    float v[16];
                    load16(x + r * k, st * 4 + g, k, v);
                    top = top16(v, top);
                }
#pragma unroll
            for (int o = 16; o < 64; o <<= 1) {
                const uint32_t a = (uint32_t)__shfl_xor((int)top, o);
                top = a > top ? a : top;
            }
            if (g == 0)
                tops[wave][r] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kFewWaves; ++i)
                top = tops[i][r] > top ? tops[i][r] : top;
            s = scale_of(top);
            inv = 1.0f / s;
        }
        i32x4 acc = {0, 0, 0, 0};
        for (size_t s0 = (size_t)wave * U; s0 < steps; s0 += kFewWaves * U) {
            uint4 b[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s0 + u < steps)
                    b[u] = *(const uint4 *)(pw + (s0 + u) * 64);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (s0 + u >= steps)
                    break;
                uint4 a = make_uint4(0, 0, 0, 0);
                if (r < m) {
                    if constexpr (FUSED) {
                        float v[16];
                        load16(x + r * k, (s0 + u) * 4 + g, k, v);
                        a = codes16(v, s, inv);
                    } else {
                        a = *(const uint4 *)(xq.codes + r * xq.ld + (s0 + u) * 64 + g * 16);
                    }
                }
                acc = mma16(a, b[u], acc);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            part[wave][4 * g + e][r] = acc[e];
        // (lanes of the first wave with g == 0 hold the rows' scales)
        __shared__ float scales[16];
        if (FUSED && wave == 0 && g == 0)
            scales[r] = s;
        __syncthreads();
        const int row = tid >> 4, col = tid & 15;
        if (row < m && row < 16 && n0 + col < w.rows) {
            int sum = 0;
#pragma unroll
            for (int i = 0; i < kFewWaves; ++i)
                sum += part[i][row][col];
            const float sx = FUSED ? scales[row] : xq.scale[row];
            y[(size_t)row * w.rows + n0 + col] = (O)((float)sum * sx * w.scale[n0 + col]);
        }
        __syncthreads();
    }
}

// Products that the tiles below would not spread over the chip: a thread block owns
// FM x FN tiles of 16 and its KG waves split the reduction, wave v taking the
// pairs of steps v, v + KG, ... straight from memory into registers, the next
// pair's loads in flight.  LDS only for the exact sum of the partial tiles.
template <int FM, int FN>
struct pair_of_steps {
    uint4 a[2][FM], b[2][FN];
    __device__ __forceinline__ void load(const uint8_t *const (&pa)[FM], const uint8_t *const (&pb)[FN], size_t s)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
                a[h][i] = *(const uint4 *)(pa[i] + (s + h) * 64);
#pragma unroll
            for (int j = 0; j < FN; ++j)
                b[h][j] = *(const uint4 *)(pb[j] + (s + h) * 64);
        }
    }
    __device__ __forceinline__ void multiply(i32x4 (&acc)[FM][FN]) const
    {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = mma16(a[h][i], b[h][j], acc[i][j]);
    }
};

template <int FM, int FN, int KG, class O>
__global__ void __launch_bounds__(KG * 64, 1) k_q8_split(pgk_q8 x, pgk_q8 w, O *__restrict__ y)
{
    constexpr int TM = 16 * FM, TN = 16 * FN, RS = TN + 4;
    __shared__ int part[KG / 2][TM * RS];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, lg = lane >> 4;
    const int tiles_n = (int)((w.rows + TN - 1) / TN);
    const int pid = xcd_tile((int)blockIdx.x, (int)gridDim.x);
    const size_t m0 = (size_t)(pid / tiles_n) * TM, n0 = (size_t)(pid % tiles_n) * TN;
    const size_t steps = x.ld / 64; // an even number
    const uint8_t *pa[FM], *pb[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const size_t r = m0 + i * 16 + lr;
        pa[i] = (const uint8_t *)x.codes + (r < x.rows ? r : x.rows - 1) * x.ld + lg * 16;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const size_t r = n0 + j * 16 + lr;
        pb[j] = (const uint8_t *)w.codes + (r < w.rows ? r : w.rows - 1) * w.ld + lg * 16;
    }
    i32x4 acc[FM][FN] = {};
    pair_of_steps<FM, FN> cur, next;
    size_t s = wave * 2;
    if (s < steps)
        cur.load(pa, pb, s);
    for (; s < steps; s += 2 * KG) {
        const size_t ahead = s + 2 * KG;
        if (ahead < steps)
            next.load(pa, pb, ahead);
        cur.multiply(acc);
        cur = next;
    }
    auto at = [&](int slot, int i, int j, int e) -> int & { return part[slot][(i * 16 + 4 * lg + e) * RS + j * 16 + lr]; };
    if (wave >= KG / 2)
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    at(wave - KG / 2, i, j, e) = acc[i][j][e];
    __syncthreads();
    if (wave < KG / 2) // each in its own slot
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    at(wave, i, j, e) += acc[i][j][e];
    __syncthreads();
    const size_t M = x.rows, N = w.rows;
#pragma unroll 1
    for (int i = tid; i < TM * TN / 4; i += KG * 64) {
        const int row = i / (TN / 4), c4 = i % (TN / 4) * 4;
        const size_t gm = m0 + row, gn = n0 + c4;
        if (gm >= M || gn >= N)
            continue;
        i32x4 v = *(const i32x4 *)&part[0][row * RS + c4];
#pragma unroll
        for (int p = 1; p < KG / 2; ++p)
            v += *(const i32x4 *)&part[p][row * RS + c4];
        const float sx = x.scale[gm];
        const int n = N - gn < 4 ? (int)(N - gn) : 4;
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            o[e] = e < n ? (float)v[e] * sx * w.scale[gn + e] : 0.0f;
        put4(y + gm * N + gn, o, n);
    }
}

// Large products on the tiles of piece_loop.
template <class CF, class O>
__global__ void __launch_bounds__(CF::NT, 1) k_q8_tiles(pgk_q8 x, pgk_q8 w, O *__restrict__ y)
{
    __shared__ uint4 smem[CF::LDS_U4];
    LDS uint4 *const lds = (LDS uint4 *)smem;
    const int M = (int)x.rows, N = (int)w.rows;
    const int tiles_m = (M + CF::BM - 1) / CF::BM, tiles_n = (N + CF::BN - 1) / CF::BN;
    // neighbouring tiles on one XCD, eight tile-rows at a time
    const int pid = xcd_tile((int)blockIdx.x, (int)gridDim.x);
    const int per_group = 8 * tiles_n, group = pid / per_group, first = group * 8;
    const int gsz = tiles_m - first < 8 ? tiles_m - first : 8, in = pid - group * per_group;
    const int m0 = (first + in % gsz) * CF::BM, n0 = in / gsz * CF::BN;
    i32x16 acc[CF::FM][CF::FN];
    piece_loop<CF>({(const uint16_t *)x.codes, x.ld / 2, 0, M}, {(const uint16_t *)w.codes, w.ld / 2, 0, N}, 0, (int)(x.ld / 2),
                   m0, n0, lds, acc);
    piece_out<CF, i32x4>(acc, m0, n0, M, N, lds, false, [&](int row, int col, const i32x4 &v, bool) {
        const float sx = x.scale[row];
        const int n = N - col < 4 ? N - col : 4;
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            o[e] = e < n ? (float)v[e] * sx * w.scale[col + e] : 0.0f;
        put4(y + (size_t)row * N + col, o, n);
    });
}

// ---------------------------------------------------------------- launches

unsigned grid_of(size_t n) { return (unsigned)(n < kMostBlocks ? n : kMostBlocks); }
size_t slabs_of(const pgk_q8 *q) { return (q->cols + kSlab - 1) / kSlab; }
size_t ld_of(size_t cols) { return (cols + 127) & ~(size_t)127; }

template <class FN>
int by_type(int dtype, FN fn)
{
    return dtype == 0 ? fn((float *)nullptr) : dtype == 1 ? fn((_Float16 *)nullptr) : fn((__bf16 *)nullptr);
}

template <class T>
int quantize_rows(const pgk_q8 &q, const T *src, hipStream_t st)
{
    const size_t nc = q.ld / 16;
    auto go = [&](auto tpr, auto lng) {
        constexpr int TPR = decltype(tpr)::value, NT = TPR < 256 ? 256 : TPR;
        hipLaunchKernelGGL((k_q8_rows<T, TPR, decltype(lng)::value>), dim3(grid_of((q.rows + NT / TPR - 1) / (NT / TPR))),
                           dim3(NT), 0, st, q, src);
    };
    if (nc <= 128)
        go(std::integral_constant<int, 64>{}, std::false_type{});
    else if (nc <= 512)
        go(std::integral_constant<int, 256>{}, std::false_type{});
    else
        go(std::integral_constant<int, 1024>{}, std::true_type{});
    return (int)hipGetLastError();
}

template <class T>
int quantize_columns(const pgk_q8 &q, const T *src, uint32_t *ws, hipStream_t st)
{
    const size_t nx = (q.rows + 63) / 64, ny = slabs_of(&q);
    hipLaunchKernelGGL(k_q8_tops<T>, dim3(grid_of(nx * ny)), dim3(256), 0, st, q, src, ws, nx, ny);
    if (const int rc = (int)hipGetLastError())
        return rc;
    hipLaunchKernelGGL(k_q8_columns<T>, dim3(grid_of(nx * ny)), dim3(256), 0, st, q, src, ws, (int)ny, nx, ny);
    return (int)hipGetLastError();
}

template <int FM, int FN, int KG, class O>
void split(const pgk_q8 &x, const pgk_q8 &w, O *y, hipStream_t st)
{
    const size_t blocks = (x.rows + 16 * FM - 1) / (16 * FM) * ((w.rows + 16 * FN - 1) / (16 * FN));
    hipLaunchKernelGGL((k_q8_split<FM, FN, KG, O>), dim3((unsigned)blocks), dim3(KG * 64), 0, st, x, w, y);
}

template <class O>
int product(const pgk_q8 &x, const pgk_q8 &w, O *y, hipStream_t st)
{
    auto tiles = [&](size_t bm, size_t bn) { return (x.rows + bm - 1) / bm * ((w.rows + bn - 1) / bn); };
    if (tiles(128, 128) >> 22) { // a grid holds under 2^32 threads: the rows in two halves
        if (x.rows <= 256) // over 2^28 columns
            return (int)hipErrorInvalidValue;
        pgk_q8 a = x, b = x;
        a.rows = (x.rows / 2 + 255) & ~(size_t)255;
        b.rows -= a.rows;
        b.codes += a.rows * x.ld;
        b.scale += a.rows;
        const int rc = product(a, w, y, st);
        return rc ? rc : product(b, w, y + a.rows * w.rows, st);
    }
    using T128 = pcfg<i32x16, 1, 128, 128, 2, 2, false, 64, 2>;
    using T256 = pcfg<i32x16, 1, 256, 256, 2, 4, false, 64, 2>;
    if (tiles(32, 32) <= 256)
        split<2, 2, 8>(x, w, y, st);
    else if (tiles(64, 32) <= 256)
        split<4, 2, 8>(x, w, y, st);
    else if (tiles(64, 64) <= 256)
        split<4, 4, 8>(x, w, y, st);
    else if (tiles(64, 64) <= 512)
        split<4, 4, 4>(x, w, y, st);
    else if (tiles(256, 256) < 192)
        hipLaunchKernelGGL((k_q8_tiles<T128, O>), dim3((unsigned)tiles(128, 128)), dim3(T128::NT), 0, st, x, w, y);
    else
        hipLaunchKernelGGL((k_q8_tiles<T256, O>), dim3((unsigned)tiles(256, 256)), dim3(T256::NT), 0, st, x, w, y);
    return (int)hipGetLastError();
}

bool fits(const pgk_q8 *q) { return q->rows && q->rows <= 0x3fffffff && q->cols && q->cols <= PGK_Q8_MAX_K; }

} // namespace

extern "C" void pgk_q8_shape(pgk_q8 *q, size_t rows, size_t cols, size_t *code_bytes, size_t *scale_bytes)
{
    q->rows = rows;
    q->cols = cols;
    q->ld = ld_of(cols);
    *code_bytes = rows * q->ld;
    *scale_bytes = rows * sizeof(float);
}

extern "C" size_t pgk_q8_workspace(const pgk_q8 *q, int trans) { return trans ? slabs_of(q) * q->rows * sizeof(uint32_t) : 0; }

extern "C" int pgk_q8_quantize(const pgk_q8 *q, const void *src, int dtype, int trans, void *ws, pgk_stream s)
{
    if (!fits(q))
        return (int)hipErrorInvalidValue;
    return by_type(dtype, [&](auto t) {
        using T = const std::remove_pointer_t<decltype(t)>;
        return trans ? quantize_columns(*q, (T *)src, (uint32_t *)ws, (hipStream_t)s) : quantize_rows(*q, (T *)src, (hipStream_t)s);
    });
}

extern "C" int pgk_q8_dequantize(const pgk_q8 *q, void *dst, int dtype, int trans, pgk_stream s)
{
    if (!fits(q))
        return (int)hipErrorInvalidValue;
    return by_type(dtype, [&](auto t) {
        using O = std::remove_pointer_t<decltype(t)>;
        const hipStream_t st = (hipStream_t)s;
        const size_t nx = (q->rows + 63) / 64, ny = slabs_of(q);
        if (trans)
            hipLaunchKernelGGL(k_q8_back_columns<O>, dim3(grid_of(nx * ny)), dim3(256), 0, st, *q, (O *)dst, nx, ny);
        else
            hipLaunchKernelGGL(k_q8_back_rows<O>, dim3(grid_of((q->rows * ((q->cols + 3) / 4) + 255) / 256)), dim3(256), 0, st,
                               *q, (O *)dst);
        return (int)hipGetLastError();
    });
}

extern "C" int pgk_q8_few_rows(size_t m) { return m <= 16; }
extern "C" int pgk_q8_few_fused(size_t m, size_t k) { return m * k <= 16384; }

extern "C" int pgk_q8_matmul_few(const void *x, int dtype, const pgk_q8 *xq, size_t m, const pgk_q8 *w, void *y, int y_dtype,
                                 pgk_stream s)
{
    if (!pgk_q8_few_rows(m) || !fits(w))
        return (int)hipErrorInvalidValue;
    const size_t tiles = (w->rows + 15) / 16;
    const dim3 grid(grid_of(tiles)), block(kFewWaves * 64);
    return by_type(y_dtype, [&](auto o) {
        using O = std::remove_pointer_t<decltype(o)>;
        if (xq) {
            hipLaunchKernelGGL((k_q8_few<float, O, false>), grid, block, 0, (hipStream_t)s, (const float *)nullptr, *xq, (int)m, *w,
                               (O *)y, tiles);
            return (int)hipGetLastError();
        }
        return by_type(dtype, [&](auto t) {
            using T = std::remove_pointer_t<decltype(t)>;
            hipLaunchKernelGGL((k_q8_few<T, O, true>), grid, block, 0, (hipStream_t)s, (const T *)x, pgk_q8{}, (int)m, *w, (O *)y,
                               tiles);
            return (int)hipGetLastError();
        });
    });
}

extern "C" int pgk_q8_matmul(const pgk_q8 *x, const pgk_q8 *w, void *y, int y_dtype, pgk_stream s)
{
    if (x->cols != w->cols || !fits(x) || !fits(w))
        return (int)hipErrorInvalidValue;
    return by_type(y_dtype, [&](auto o) { return product(*x, *w, (decltype(o))y, (hipStream_t)s); });
}
