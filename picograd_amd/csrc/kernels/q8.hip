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

// A code from 1 / s: fma with 1.5 2^23 rounds v / s to a whole number q in the low
// bits of the sum.  What is left over, v - q s, is exact in f32 (a multiple of half
// the last place of s, below s / 2 but for some units of it).  Where it reaches s / 2,
// a tie or 1 / s on the wrong side of one, q moves by one towards v or to the even
// one.  A scale next to the subnormals is taken with its values times 2^100; one
// rounded there may leave v / s past 127.
constexpr float kRound = 12582912.0f;
constexpr float kLeastScale = 0x1p-120f;

// the code from v, s and t, the sum with kRound
__device__ __forceinline__ uint32_t code_exact(float v, float s, float t)
{
    float q = t - kRound;
    const float r = fmaf(-q, s, v), a = fabsf(r), half = 0.5f * s;
    const bool away = (a > half) | ((a == half) & (bool)(__float_as_uint(t) & 1));
    q += away ? copysignf(1.0f, r) : 0.0f;
    return (uint32_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
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
        const float unit = s < kLeastScale ? 0x1p100f : 1.0f, su = s * unit, iu = s < kLeastScale ? 1.0f / su : inv;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            b[i] = code_exact(v[i] * unit, su, fmaf(v[i] * unit, iu, kRound));
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

// Codes of columns: a thread takes C neighbours of 16 neighbouring rows of src, so that
// it has a whole piece of each of its columns' codes; 16 / C lanes side by side, the
// others down a wave, the waves below each other.  HELD: a block holds its 16 columns
// whole (kHeld long) and finds their scales by itself, src is read once; else the
// tops are there.  C is four, of 16-bit columns past 4096 eight (shorter ones' blocks
// would have half the waves).  Bound by the stream of the source: 4096 x 4096 in f32, 84
// MB with the codes, 22 us; the search and the rounding in passes of their own took 28.
constexpr int kColumns = 16; // of a block
template <int C>
constexpr int kHeld = 64 / (kColumns / C) * 16 * 16; // rows of 16 waves

template <class T, int C, bool HELD>
__global__ void __launch_bounds__(1024, 1) k_q8_columns(pgk_q8 q, const T *__restrict__ src, const uint32_t *__restrict__ part,
                                                        int slabs, size_t nx, size_t ny)
{
    constexpr int A = kColumns / C; // lanes side by side
    typedef T tv __attribute__((ext_vector_type(C), aligned(sizeof(T))));
    __shared__ uint32_t tops[2][kColumns];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lc = lane % A * C, lrow = (wave * (64 / A) + lane / A) * 16;
    if (tid < kColumns)
        tops[0][tid] = 0;
    __syncthreads();
    int turn = 0;
    for (size_t job = blockIdx.x; job < nx * ny; job += gridDim.x, turn ^= 1) {
        // neighbouring columns share lines: on one XCD
        const size_t at = gridDim.x == nx * ny ? (size_t)xcd_tile((int)job, (int)gridDim.x) : job, x = at % nx;
        const size_t col = x * kColumns + lc, k0 = at / nx * kHeld<C> + lrow;
        const int left = col < q.rows ? (int)(q.rows - col < C ? q.rows - col : C) : 0;
        tv raw[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const size_t k = k0 + i;
            raw[i] = tv{};
            if (k < q.cols) {
                const T *const p = src + k * q.rows + col;
                if (left == C)
                    raw[i] = *(const tv *)p;
                else if constexpr (sizeof(T) == 4) { // without conditions: 1000 x 2049 in 6.8 us, with them 11
                    if (left)
#pragma unroll
                        for (int e = 0; e < C; ++e) {
                            const T one = p[e < left ? e : 0];
                            raw[i][e] = e < left ? one : 0.0f;
                        }
                } else { // two to a register: 2045 x 197 in 9.0 us, without conditions 10.3
#pragma unroll
                    for (int e = 0; e < C; ++e)
                        if (e < left)
                            raw[i][e] = p[e];
                }
            }
        }
        if constexpr (HELD) {
            // magnitudes order as their bits do, in the source's own width
            using B = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
            typedef B bits __attribute__((ext_vector_type(C)));
            bits top = {};
#pragma unroll
            for (int i = 0; i < 16; ++i)
                top = __builtin_elementwise_max(top, __builtin_bit_cast(bits, raw[i]) & (B)((B)~0u >> 1));
#pragma unroll
            for (int o = A; o < 64; o <<= 1) {
                typedef int words __attribute__((ext_vector_type(sizeof(bits) / 4)));
                words w = __builtin_bit_cast(words, top);
#pragma unroll
                for (int i = 0; i < (int)(sizeof(bits) / 4); ++i)
                    w[i] = __shfl_xor(w[i], o);
                top = __builtin_elementwise_max(top, __builtin_bit_cast(bits, w));
            }
            if (lane < A)
#pragma unroll
                for (int e = 0; e < C; ++e) {
                    const B one = top[e];
                    atomicMax(&tops[turn][lc + e], magnitude((float)__builtin_bit_cast(T, one)));
                }
        } else if (tid < kColumns) {
            uint32_t top = 0;
            if (x * kColumns + tid < q.rows)
                for (int i = 0; i < slabs; ++i) {
                    const uint32_t a = part[(size_t)i * q.rows + x * kColumns + tid];
                    top = a > top ? a : top;
                }
            tops[turn][tid] = top;
        }
        __syncthreads();
        if (HELD && tid < kColumns)
            tops[turn ^ 1][tid] = 0; // (read before the barrier above, filled behind the one below)
#pragma unroll
        for (int e = 0; e < C; ++e) {
            if (e >= left)
                break;
            const float s = scale_of(tops[turn][lc + e]);
            if (k0 == 0)
                q.scale[col + e] = s;
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
                v[i] = (float)raw[i][e];
            if (k0 < q.ld)
                *(uint4 *)(q.codes + (col + e) * q.ld + k0) = codes16(v, s, 1.0f / s);
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

// N sums under both scales.  Under a scale of x outside these bounds the first product
// may leave f32 where the second comes back into it (x of 1e33 under weights of
// 1e-10): then 64 bits hold all three.
template <int N, class V>
__device__ __forceinline__ void scaled(const V &sum, float sx, const float (&sw)[N], float (&y)[N])
{
    if (sx < 0x1p90f && sx > 0x1p-90f)
#pragma unroll
        for (int e = 0; e < N; ++e)
            y[e] = (float)sum[e] * sx * sw[e];
    else
#pragma unroll
        for (int e = 0; e < N; ++e)
            y[e] = (float)((double)sum[e] * (double)sx * (double)sw[e]);
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
// reduction, so the weights stream past once.  FUSED: every block rounds x into LDS by
// itself while its first weights are on their way, no other launch; else xq holds
// it.  Bound by the loads' latency and the launch.
constexpr int kFewWaves = 8, kFewFused = 16384; // values of x that every block rounds

template <class T, class O, bool FUSED>
__global__ void __launch_bounds__(kFewWaves * 64, 1)
    k_q8_few(const T *__restrict__ x, pgk_q8 xq, int m, pgk_q8 w, O *__restrict__ y, size_t tiles)
{
    constexpr int U = 8, MOST = FUSED ? kFewFused / 16 + 16 * 8 : 1; // steps of 64 in flight; pieces of x
    constexpr int PER = (MOST + kFewWaves * 64 - 1) / (kFewWaves * 64);
    __shared__ int part[kFewWaves][16][17];
    __shared__ uint4 xs[MOST];
    __shared__ uint32_t tops[16];
    // (the wave's number is uniform to the compiler: a matrix instruction heeds no mask)
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const size_t steps = w.ld / 64, k = w.cols;
    const int nc = (int)(w.ld / 16), xr = r < m ? r : m - 1; // (rows past the last give sums that no one takes)
    for (size_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const size_t n0 = tile * 16, wr = n0 + r < w.rows ? n0 + r : w.rows - 1;
        const uint8_t *const pw = (const uint8_t *)w.codes + wr * w.ld + g * 16;
        uint4 b[U];
        auto load = [&](size_t s0) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s0 + u < steps)
                    b[u] = *(const uint4 *)(pw + (s0 + u) * 64);
        };
        size_t s0 = (size_t)wave * U;
        load(s0);
        if (FUSED && tile == blockIdx.x) {
            if (tid < 16)
                tops[tid] = 0;
            float v[PER][16];
            uint32_t top[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = tid + i * kFewWaves * 64, row = c / nc;
                top[i] = 0;
                if (row < m) {
                    load16(x + row * k, c - row * nc, k, v[i]);
                    top[i] = top16(v[i], 0);
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = tid + i * kFewWaves * 64, row = c / nc;
                // a wave within one row has one largest
                if (__all(row == __builtin_amdgcn_readfirstlane(row))) {
                    const uint32_t t = wave_top(top[i]);
                    if (lane == 0 && row < m)
                        atomicMax(&tops[row], t);
                } else if (row < m) {
                    atomicMax(&tops[row], top[i]);
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = tid + i * kFewWaves * 64, row = c / nc;
                if (row < m) {
                    const float s = scale_of(tops[row]);
                    xs[c] = codes16(v[i], s, 1.0f / s);
                }
            }
            __syncthreads();
        }
        i32x4 acc = {0, 0, 0, 0};
        while (s0 < steps) {
            uint4 a[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s0 + u < steps) {
                    if constexpr (FUSED)
                        a[u] = xs[xr * nc + (s0 + u) * 4 + g];
                    else
                        a[u] = *(const uint4 *)(xq.codes + xr * xq.ld + (s0 + u) * 64 + g * 16);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s0 + u < steps)
                    acc = mma16(a[u], b[u], acc);
            s0 += kFewWaves * U;
            load(s0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            part[wave][4 * g + e][r] = acc[e];
        __syncthreads();
        const int row = tid >> 4, col = tid & 15;
        if (row < m && row < 16 && n0 + col < w.rows) {
            int sum[1] = {0};
#pragma unroll
            for (int i = 0; i < kFewWaves; ++i)
                sum[0] += part[i][row][col];
            const float sx = FUSED ? scale_of(tops[row]) : xq.scale[row];
            const float sw[1] = {w.scale[n0 + col]};
            float o[1];
            scaled(sum, sx, sw, o);
            y[(size_t)row * w.rows + n0 + col] = (O)o[0];
        }
        __syncthreads();
    }
}

// More rows on the tiles of piece_loop: bound by loads' latency where there are few
// tiles, by LDS and the matrix units where there are many (8192 x 4096 x 4096: 131 us,
// 2.1 POP/s; along the reduction alone 2.7 of the 3.0 that the instruction reaches).
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
    // a lane's columns are the same in every strip
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    const int col0 = n0 + wave % CF::WGN * CF::WN + lane % (CF::WN / 4) * 4;
    float sw[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        sw[e] = col0 + e < N ? w.scale[col0 + e] : 0.0f;
#pragma unroll
    for (int i = 0; i < CF::FM; ++i)
        piece_out_strip<CF, i32x4>(
            acc[i], i, m0, n0, M, N, lds, false, [&](int row, int) { return x.scale[row]; },
            [&](int row, int col, const i32x4 &v, float sx, bool) {
                float o[4];
                scaled(v, sx, sw, o);
                put4(y + (size_t)row * N + col, o, N - col < 4 ? N - col : 4);
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
    const size_t nx = (q.rows + kColumns - 1) / kColumns;
    auto held = [&](auto c) {
        constexpr int C = decltype(c)::value;
        constexpr size_t per = kHeld<C> / 16; // rows of a wave
        hipLaunchKernelGGL((k_q8_columns<T, C, true>), dim3(grid_of(nx)), dim3((unsigned)((q.ld + per - 1) / per) * 64), 0, st, q,
                           src, (const uint32_t *)nullptr, 0, nx, (size_t)1);
        return (int)hipGetLastError();
    };
    if (q.ld <= kHeld<4>)
        return held(std::integral_constant<int, 4>{});
    if constexpr (sizeof(T) == 2)
        if (q.ld <= kHeld<8>)
            return held(std::integral_constant<int, 8>{});
    constexpr int C = 16 / sizeof(T);
    const size_t sx = (q.rows + 63) / 64, slabs = slabs_of(&q), ny = (q.ld + kHeld<C> - 1) / kHeld<C>;
    hipLaunchKernelGGL(k_q8_tops<T>, dim3(grid_of(sx * slabs)), dim3(256), 0, st, q, src, ws, sx, slabs);
    if (const int rc = (int)hipGetLastError())
        return rc;
    hipLaunchKernelGGL((k_q8_columns<T, C, false>), dim3(grid_of(nx * ny)), dim3(1024), 0, st, q, src, ws, (int)slabs, nx, ny);
    return (int)hipGetLastError();
}

template <class O>
int product(const pgk_q8 &x, const pgk_q8 &w, O *y, hipStream_t st)
{
    auto tiles = [&](size_t bm, size_t bn) { return (x.rows + bm - 1) / bm * ((w.rows + bn - 1) / bn); };
    // a grid holds under 2^32 threads: the rows in two halves (up to 256 of them by 2^30
    // columns are 2^23 of the larger tiles at most, 2^31 threads)
    if (x.rows > 256 && tiles(64, 64) >> 24) {
        pgk_q8 a = x, b = x;
        a.rows = (x.rows / 2 + 255) & ~(size_t)255;
        b.rows -= a.rows;
        b.codes += a.rows * x.ld;
        b.scale += a.rows;
        const int rc = product(a, w, y, st);
        return rc ? rc : product(b, w, y + a.rows * w.rows, st);
    }
    using T64 = pcfg<i32x16, 1, 64, 64, 2, 2, false, 64, 4>;
    using T128 = pcfg<i32x16, 1, 128, 128, 4, 2, false, 64, 4>;
    using TWO = pcfg<i32x16, 1, 128, 128, 2, 2, false, 64, 2>; // of 128 x 128 to a CU
    using TALL = pcfg<i32x16, 1, 256, 128, 4, 2, false, 64, 3>;
    using T256 = pcfg<i32x16, 1, 256, 256, 2, 4, false, 64, 2>;
    auto go = [&](auto cf) {
        using CF = decltype(cf);
        hipLaunchKernelGGL((k_q8_tiles<CF, O>), dim3((unsigned)tiles(CF::BM, CF::BN)), dim3(CF::NT), 0, st, x, w, y);
    };
    // The largest tile that fills the chip; over K = N = 4096 with M rows, in us:
    //   M       512    1000   1024   1500   2048   3000   4096   5000
    //   64     15.8     29   29.6     43     57     83    110    141
    //   128    17.6     23   23.4     39     46     66     89    108
    //   TALL   25.8     29   29.6     33     39     65     76    102
    //   TWO    23.4     28   27.8     37     42     66     77     98
    //   256    43.1     47   47.5     50     53     57     68    109
    // Past those: whole rounds of 256-tiles against half rounds of two 128-tiles a
    // CU, each 0.68 of one.
    const size_t big = (tiles(256, 256) + 255) / 256, half = (tiles(128, 128) + 255) / 256;
    if (tiles(128, 128) <= 128)
        go(T64{});
    else if (tiles(128, 128) <= 256)
        go(T128{});
    else if (tiles(256, 128) <= 256)
        go(TALL{});
    else if ((double)big <= 0.34 * (double)half)
        go(T256{});
    else
        go(TWO{});
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

extern "C" size_t pgk_q8_workspace(const pgk_q8 *q, int trans)
{
    return trans && q->ld > kHeld<4> ? slabs_of(q) * q->rows * sizeof(uint32_t) : 0;
}

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
extern "C" int pgk_q8_few_fused(size_t m, size_t k) { return m * k <= kFewFused; }

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
