// Matrices in 4 bits: e2m1 values (0, .5, 1, 1.5, 2, 3, 4, 6 and their
// negatives) with one power of two for each 32 along the reduction, and their
// product on the block-scaled matrix instruction
// (v_mfma_scale_f32_16x16x128_f8f6f4, four times the rate of the 16-bit ones).
//
// The block's power is 2^(floor(log2 max |v|) - 2), so the largest magnitude
// lies in [4, 8) units; what is past 6 becomes 6, the rest is rounded to
// nearest, ties to the even code.  y = Q(x) Q(W)^T over both operands' rows: the
// products of two 4-bit values are exact, their sums f32, y is rounded once.
//
// Both operands are held in the instruction's own order (pgk_mx4), so a wave
// loads a 16-row operand of 128 values as 1 KiB in a row, to registers or to LDS,
// with no padding, swizzle or bounds check along the reduction.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include <type_traits>

#include "gemm_tile.h"
#include "launch.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

#define INLINE __attribute__((always_inline)) // of a lambda

constexpr int kBlock = 32; // values under one power of two

// A launch holds under 2^32 threads in x and 65536 blocks in y: longer grids are
// several launches, each told the first block of its own (a loop over the blocks
// within the kernels costs a 4096 x 4096 matrix taken to 4 bits and back 11 us of 30).
constexpr size_t kMostX = (size_t)1 << 22, kMostY = 65535;

// the bytes of step s of tile t, and of its powers (of the pair of steps s / 2)
__device__ __forceinline__ uint8_t *codes_at(const pgk_mx4 &q, size_t t, size_t s)
{
    return q.codes + (t * q.steps + s) * 1024;
}
__device__ __forceinline__ uint16_t *powers_at(const pgk_mx4 &q, size_t t, size_t s)
{
    return (uint16_t *)(q.powers + (t * (q.steps / 2) + s / 2) * 128);
}

// ---------------------------------------------------------------- rounding

// The block's exponent byte for its largest magnitude, given as the bits of
// |v| (whose order is that of the magnitudes, infinities and NaN last):
// floor(log2) - 2 with the bias, 0 at least; 255 for a block with either.
__device__ __forceinline__ uint32_t power_byte(uint32_t top)
{
    const uint32_t e = top >> 23;
    return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
__device__ __forceinline__ float power_of(uint32_t byte)
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
// a block of 32 values in 4 bits, and its exponent byte
__device__ __forceinline__ uint4 round_block(const float *v, uint32_t &byte)
{
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kBlock; ++i) {
        const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
        top = a > top ? a : top;
    }
    byte = power_byte(top);
    if (byte == 255)
        return make_uint4(0, 0, 0, 0);
    const float s = power_of(byte);
    return make_uint4(pack8(v, s), pack8(v + 8, s), pack8(v + 16, s), pack8(v + 24, s));
}

// a block of a row as f32: 16-byte loads (VEC: p is aligned) or one by one;
// values at and past `left` are 0
template <class T, bool VEC>
__device__ __forceinline__ void load_block(const T *p, int left, float *v)
{
    if (VEC && left >= kBlock) {
        constexpr int E = 16 / sizeof(T);
        typedef T tv __attribute__((ext_vector_type(E)));
#pragma unroll
        for (int i = 0; i < kBlock / E; ++i) {
            const tv q = ((const tv *)p)[i];
#pragma unroll
            for (int j = 0; j < E; ++j)
                v[i * E + j] = (float)q[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kBlock; ++i)
            v[i] = i < left ? (float)p[i] : 0.0f;
    }
}

// Blocks along the source's rows: a wave makes two steps of one tile, lane l
// the blocks that are entry l of each, so a lane rounds a block by itself and
// the codes leave as whole kilobytes.  Bound by the stream of the source (8192 x
// 4096 in bf16, 84 MB with the codes: 14 us, 6 TB/s with a part still cached).
template <class T, bool VEC>
__global__ void __launch_bounds__(256) k_mx4_rows(pgk_mx4 q, const T *__restrict__ src)
{
    const int lane = (int)threadIdx.x & 63;
    const size_t pairs = q.steps / 2, n = q.tiles * pairs;
    for (size_t i = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (size_t)gridDim.x * 4) {
        const size_t t = i / pairs, s = (i - t * pairs) * 2, row = t * 16 + (lane & 15);
        uint32_t both = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const size_t c = (s + h) * 128 + (size_t)(lane >> 4) * kBlock;
            float v[kBlock];
            const bool in = row < q.rows && c < q.cols;
            load_block<T, VEC>(src + (in ? row * q.cols + c : 0), in ? (int)(q.cols - c < kBlock ? q.cols - c : kBlock) : 0, v);
            uint32_t byte;
            ((uint4 *)codes_at(q, t, s + h))[lane] = round_block(v, byte);
            both |= byte << (8 * h);
        }
        powers_at(q, t, s)[lane] = (uint16_t)both;
    }
}

// Blocks down the source's columns ([cols, rows]): a thread takes block `wave`
// of two steps of one column, so that a wave reads whole row pieces of 64
// columns (four tiles).  Bound by the stream of the source (4096 x 4096 in f32,
// 76 MB with the codes: 13.9 us).
template <class T>
__global__ void __launch_bounds__(256) k_mx4_columns(pgk_mx4 q, const T *__restrict__ src, size_t x0, size_t y0)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const size_t row = (x0 + blockIdx.x) * 64 + lane, s = (y0 + blockIdx.y) * 2, t = row >> 4;
    if (t >= q.tiles)
        return;
    const int entry = wave * 16 + (lane & 15);
    uint32_t both = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const size_t c0 = (s + h) * 128 + (size_t)wave * kBlock;
        float v[kBlock];
#pragma unroll
        for (int j = 0; j < kBlock; ++j)
            v[j] = row < q.rows && c0 + j < q.cols ? (float)__builtin_nontemporal_load(src + (c0 + j) * q.rows + row) : 0.0f;
        uint32_t byte;
        ((uint4 *)codes_at(q, t, s + h))[entry] = round_block(v, byte);
        both |= byte << (8 * h);
    }
    powers_at(q, t, s)[entry] = (uint16_t)both;
}

// ---------------------------------------------------------------- reading back

// the eight values of a dword of codes
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t byte, float *v)
{
    const float s = power_of(byte), bad = __uint_as_float(0x7fc00000u);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
    const float q[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = byte == 255 ? bad : q[i];
}

// Rows back: four lanes per block, eight values each, along the row.
template <class O>
__global__ void __launch_bounds__(256) k_mx4_back_rows(pgk_mx4 q, O *__restrict__ dst)
{
    const size_t per = (q.cols + 7) / 8, n = per * q.rows;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t row = i / per, part = i - row * per, c = part * 8, s = c / 128;
        const int entry = (int)(c / kBlock & 3) * 16 + (int)(row & 15);
        float v[8];
        unpack8(((const uint32_t *)codes_at(q, row >> 4, s))[entry * 4 + (part & 3)],
                powers_at(q, row >> 4, s)[entry] >> (8 * (s & 1)) & 255, v);
        O *p = dst + row * q.cols + c;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < q.cols)
                p[j] = (O)v[j];
    }
}

// Columns back, as k_mx4_columns reads them.
template <class O>
__global__ void __launch_bounds__(256) k_mx4_back_columns(pgk_mx4 q, O *__restrict__ dst, size_t x0, size_t y0)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const size_t row = (x0 + blockIdx.x) * 64 + lane, s = (y0 + blockIdx.y) * 2, t = row >> 4;
    if (row >= q.rows)
        return;
    const int entry = wave * 16 + (lane & 15);
    const uint32_t both = powers_at(q, t, s)[entry];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint4 w = ((const uint4 *)codes_at(q, t, s + h))[entry];
        const uint32_t d[4] = {w.x, w.y, w.z, w.w};
        const size_t c0 = (s + h) * 128 + (size_t)wave * kBlock;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v[8];
            unpack8(d[j], both >> (8 * h) & 255, v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + j * 8 + e < q.cols)
                    __builtin_nontemporal_store((O)v[e], dst + (c0 + j * 8 + e) * q.rows + row);
        }
    }
}

// ---------------------------------------------------------------- products

// 16 x 16 over a step of 128: the powers of the lanes' entries in byte H of sa
// and sb; lane l gets column l % 16 of rows 4 (l / 16) .. + 3
template <int H>
__device__ __forceinline__ f32x4 mfma4(const uint4 &a, const uint4 &b, const f32x4 &c, uint32_t sa, uint32_t sb)
{
    const v8i va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
    const v8i vb = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, H, (int)sa, H, (int)sb);
}

// `n` neighbours of a row of y, at most four; v4: whole rows keep the alignment
// of four; PAST: past the caches
template <bool PAST = false, class O>
__device__ __forceinline__ void store4(O *p, const f32x4 &v, int n, bool v4)
{
    typedef O o4 __attribute__((ext_vector_type(4)));
    if (v4 && n >= 4) {
        if constexpr (PAST)
            __builtin_nontemporal_store(__builtin_convertvector(v, o4), (o4 *)p);
        else
            *(o4 *)p = __builtin_convertvector(v, o4);
        return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (q < n)
            p[q] = (O)v[q];
}
template <class O>
__device__ __forceinline__ bool rows_keep_four(const O *y, size_t n)
{
    return (n & 3) == 0 && (((uintptr_t)y) & (4 * sizeof(O) - 1)) == 0;
}

// Up to 16 rows of x: a thread block owns 16 columns of y and its waves split
// the reduction, so the weights stream past once.  A lane rounds its own blocks of x
// on the way (entry l of a step is one block of one row): no other launch.  The
// waves' partial tiles are added through LDS in wave order.  Bound by the loads'
// latency and the launch: one row by 4096 x 4096, 8.9 MB, 4.7 us.
constexpr int kFewWaves = 8;

template <class T, class O, bool VEC>
__global__ void __launch_bounds__(kFewWaves * 64, 1)
    k_mx4_few(const T *__restrict__ x, int m, pgk_mx4 w, O *__restrict__ y, int t0)
{
    constexpr int U = 4; // steps in flight
    __shared__ float part[kFewWaves][16][17];
    // (the wave's number is uniform to the compiler: a matrix instruction heeds no mask)
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int t = t0 + xcd_tile((int)blockIdx.x, (int)gridDim.x), steps = (int)w.steps, k = (int)w.cols;
    // runs of U neighbouring steps, dealt to the waves in turn
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = wave * U; s0 < steps; s0 += kFewWaves * U) {
        uint4 b[U];
        uint32_t sb[U / 2];
#pragma unroll
        for (int u = 0; u < U; u += 2) {
            const int s = s0 + u < steps ? s0 + u : s0; // an even number of steps
            b[u] = ((const uint4 *)codes_at(w, t, s))[lane];
            b[u + 1] = ((const uint4 *)codes_at(w, t, s + 1))[lane];
            sb[u / 2] = powers_at(w, t, s)[lane];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = (s0 + u) * 128 + g * kBlock;
            uint4 a = make_uint4(0, 0, 0, 0);
            uint32_t sa = 127;
            if (r < m && c < k) { // (steps past the end have no column)
                float v[kBlock];
                load_block<T, VEC>(x + (size_t)r * k + c, k - c, v);
                a = round_block(v, sa);
            }
            // a step past the end repeats one of the weights, whose powers may be NaN
            if (s0 + u < steps)
                acc = u & 1 ? mfma4<1>(a, b[u], acc, sa << 8, sb[u / 2]) : mfma4<0>(a, b[u], acc, sa, sb[u / 2]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        part[wave][4 * g + e][r] = acc[e];
    __syncthreads();
    const int row = tid >> 4, col = tid & 15;
    const size_t n = (size_t)t * 16 + col;
    if (row < m && row < 16 && n < w.rows) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < kFewWaves; ++i)
            v += part[i][row][col];
        y[(size_t)row * w.rows + n] = (O)v;
    }
}

// Products that the tiles below would not spread over the chip: a thread block
// owns FM x FN tiles of 16 and its KG waves split the reduction, wave v taking the
// pairs of steps v, v + KG, ... straight from memory into registers, the next
// pair's loads in flight.  LDS only for the sum of the partial tiles: the upper
// half of the waves leaves its own, the lower half adds them and leaves the
// sums, which are added in wave order.  Bound by the loads' latency: 333 x 1000 x
// 2049 takes 5.9 us, 0.23 PFLOP/s, beside 4.9 for rounding x.
template <int FM, int FN>
struct pair_of_steps {
    uint4 a[2][FM], b[2][FN];
    uint32_t sa[FM], sb[FN];
    __device__ __forceinline__ void load(const pgk_mx4 &x, const pgk_mx4 &w, const size_t (&tx)[FM], const size_t (&tw)[FN],
                                         int s, int lane)
    {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const uint4 *p = (const uint4 *)codes_at(x, tx[i], s);
            a[0][i] = p[lane];
            a[1][i] = p[64 + lane];
            sa[i] = powers_at(x, tx[i], s)[lane];
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const uint4 *p = (const uint4 *)codes_at(w, tw[j], s);
            b[0][j] = p[lane];
            b[1][j] = p[64 + lane];
            sb[j] = powers_at(w, tw[j], s)[lane];
        }
    }
    __device__ __forceinline__ void multiply(f32x4 (&acc)[FM][FN]) const
    {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = mfma4<0>(a[0][i], b[0][j], acc[i][j], sa[i], sb[j]);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = mfma4<1>(a[1][i], b[1][j], acc[i][j], sa[i], sb[j]);
    }
};

template <int FM, int FN, int KG, class O>
__global__ void __launch_bounds__(KG * 64, 1) k_mx4_split(pgk_mx4 x, pgk_mx4 w, O *__restrict__ y)
{
    constexpr int TM = 16 * FM, TN = 16 * FN, RS = TN + 4;
    __shared__ float part[KG / 2][TM * RS];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, lg = lane >> 4;
    const int tiles_n = (int)((w.tiles + FN - 1) / FN);
    const int pid = xcd_tile((int)blockIdx.x, (int)gridDim.x);
    const size_t m0 = (size_t)(pid / tiles_n) * FM, n0 = (size_t)(pid % tiles_n) * FN; // in tiles of 16
    const int steps = (int)x.steps;
    size_t tx[FM], tw[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
        tx[i] = m0 + i < x.tiles ? m0 + i : x.tiles - 1;
#pragma unroll
    for (int j = 0; j < FN; ++j)
        tw[j] = n0 + j < w.tiles ? n0 + j : w.tiles - 1;
    f32x4 acc[FM][FN] = {};
    pair_of_steps<FM, FN> cur, next;
    int s = wave * 2;
    if (s < steps)
        cur.load(x, w, tx, tw, s, lane);
    for (; s < steps; s += 2 * KG) {
        const int ahead = s + 2 * KG;
        if (ahead < steps)
            next.load(x, w, tx, tw, ahead, lane);
        cur.multiply(acc);
        cur = next;
    }
    auto at = [&](int slot, int i, int j, int e) -> float & {
        return part[slot][(i * 16 + 4 * lg + e) * RS + j * 16 + lr];
    };
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
    const bool v4 = rows_keep_four(y, N);
#pragma unroll 1
    for (int i = tid; i < TM * TN / 4; i += KG * 64) {
        const int row = i / (TN / 4), c4 = i % (TN / 4) * 4;
        const size_t gm = m0 * 16 + row, gn = n0 * 16 + c4;
        if (gm >= M || gn >= N)
            continue;
        f32x4 v = *(const f32x4 *)&part[0][row * RS + c4];
#pragma unroll
        for (int p = 1; p < KG / 2; ++p)
            v += *(const f32x4 *)&part[p][row * RS + c4];
        store4(y + gm * N + gn, v, N - gn < 4 ? (int)(N - gn) : 4, v4);
    }
}

// Large products: BM x BN tiles of y on WGM x WGN waves, the operands staged through
// LDS by direct loads in four stages of one step (128 values), their powers
// beside them.  A step's operands are read during the step before: x's each as
// soon as the products with the one it replaces are issued, w's into a second
// set.  A stage is refilled during the step that follows its last read, behind
// the step's one barrier, so its loads have three steps to land.  Tiles of
// 128 x 128 on four waves, two blocks to a CU, of which one computes while the
// other waits at its barrier.  8192 x 4096 x 4096 takes 75 us and the
// rounding of x 14, 3.7 PFLOP/s of the product where the matrix
// units alone reach 6.0 on random codes; two stages of two steps take 109 and
// 256 x 256 tiles, whose eight waves run out of registers, 90 to 111.  Bound by
// LDS: a wave's 64 x 64 reads 8 KB for 16 matrix instructions.
template <int BM, int BN, int WGM, int WGN, class O>
__global__ void __launch_bounds__(64 * WGM *WGN, 1) k_mx4_tiles(pgk_mx4 x, pgk_mx4 w, O *__restrict__ y)
{
    constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, FM = WM / 16, FN = WN / 16, S = 4;
    // a stage: A's tiles [BM / 16][64], B's, then their powers ([tile][64][two
    // steps], a kilobyte per eight tiles)
    constexpr int TA = BM / 16, TB = BN / 16, QA = TA / NW, QB = TB / NW; // kilobytes, and per wave
    constexpr int WPA = TA / 8, WPB = TB / 8, STAGE = (TA + TB + WPA + WPB) * 64;
    static_assert(TA % NW == 0 && TB % NW == 0 && NW % (WPA + WPB) == 0, "whole loads per wave");
    __shared__ uint4 smem[S * STAGE];
    LDS uint4 *const lds = (LDS uint4 *)smem;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    const int tiles_m = (int)((x.rows + BM - 1) / BM), tiles_n = (int)((w.rows + BN - 1) / BN);
    const int pid = xcd_tile((int)blockIdx.x, (int)gridDim.x);
    const int per_group = 8 * tiles_n, group = pid / per_group, first = group * 8;
    const int gsz = tiles_m - first < 8 ? tiles_m - first : 8, in = pid - group * per_group;
    const int m0 = (first + in % gsz) * BM, n0 = in / gsz * BN;
    const int steps = (int)x.steps, tx = (int)x.tiles, tw = (int)w.tiles;

    // this wave's loads of a stage: kilobytes wave Q + q of A and of B, as byte
    // offsets from the block's first tile; the base advances by a step a stage
    const uint8_t *const baseA = codes_at(x, m0 / 16, 0), *const baseB = codes_at(w, n0 / 16, 0);
    uint32_t off[QA + QB];
#pragma unroll
    for (int q = 0; q < QA + QB; ++q) {
        const int p = q < QA ? wave * QA + q : wave * QB + q - QA;
        const int last = (q < QA ? tx - m0 / 16 : tw - n0 / 16) - 1, t = p < last ? p : last;
        off[q] = (uint32_t)(t * steps * 1024 + lane * 16);
    }
    // a kilobyte of powers: eight tiles, eight lanes each; waves past those that
    // there are bring the same ones again, to the same place
    const int pw = wave % (WPA + WPB);
    const bool of_b = pw >= WPA;
    int pt = (of_b ? n0 / 16 + (pw - WPA) * 8 : m0 / 16 + pw * 8) + (lane >> 3);
    pt = pt < (of_b ? tw : tx) ? pt : (of_b ? tw : tx) - 1;
    const uint8_t *psrc = (const uint8_t *)powers_at(of_b ? w : x, pt, 0) + (lane & 7) * 16;
    constexpr int LPT = QA + QB + 1;
    static_assert((S - 1) * LPT < 64, "the loads in flight fit the vmcnt counter");
    auto dma = [&](int q, int t, int st) INLINE {
        const int tt = t < steps ? t : steps - 1; // stages past the end are read by none
        LDS uint4 *base = lds + st * STAGE;
        if (q < QA)
            dma16s(off[q], baseA + (size_t)tt * 1024, base + (wave * QA + q) * 64);
        else if (q < QA + QB)
            dma16s(off[q], baseB + (size_t)tt * 1024, base + (TA + wave * QB + q - QA) * 64);
        else
            dma16(psrc + (size_t)(tt >> 1) * 128, base + (TA + TB + pw) * 64);
    };
    auto sync_stage = [&](auto newer) INLINE { // all but the newest stages' loads have landed
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(decltype(newer)::value * LPT));
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
    };
    auto frag = [&](int st, int tile) INLINE { // of A's tiles, then B's
        return __builtin_bit_cast(uint4, ((const LDS u32x4 *)(lds + st * STAGE))[tile * 64 + lane]);
    };
    auto power = [&](int st, int tile) INLINE {
        return (uint32_t)((const LDS uint16_t *)(lds + st * STAGE + (TA + TB) * 64))[tile * 64 + lane];
    };
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    uint4 fa[FM], fb[2][FN];
    uint32_t pa[FM], pb[2][FN]; // powers of a pair of steps; w's of the next pair too
    // the step in stage u; `next`: the operands of the step behind it are read and
    // the stage takes step `reload`
    auto step = [&](auto uu, bool next, int reload) INLINE {
        constexpr int u = decltype(uu)::value, h = u & 1, nu = (u + 1) % S, pair = u >> 1 & 1;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                acc[i][j] = mfma4<h>(fa[i], fb[h][j], acc[i][j], pa[i], pb[pair][j]);
                const int g = i * FN + j;
                if (next) {
                    if (i == 0) { // w's are needed first
                        fb[h ^ 1][j] = frag(nu, TA + wn * FN + j);
                        if (h)
                            pb[pair ^ 1][j] = power(nu, TA + wn * FN + j);
                    }
                    if (j == FN - 1) {
                        fa[i] = frag(nu, wm * FM + i);
                        if (h)
                            pa[i] = power(nu, wm * FM + i);
                    }
#pragma unroll
                    for (int q = g * LPT / (FM * FN); q < (g + 1) * LPT / (FM * FN); ++q)
                        dma(q, reload, u);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
#pragma unroll
    for (int t = 0; t < S; ++t)
#pragma unroll
        for (int q = 0; q < LPT; ++q)
            dma(q, t, t);
    sync_stage(std::integral_constant<int, S - 1>{});
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        fa[i] = frag(0, wm * FM + i);
        pa[i] = power(0, wm * FM + i);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        fb[0][j] = frag(0, TA + wn * FN + j);
        pb[0][j] = power(0, TA + wn * FN + j);
    }
    // each step but the last behind a barrier: the next stage has landed (two
    // newer ones may be in flight) and every wave has read this one
    int t = 0;
    auto link = [&](auto u) INLINE {
        sync_stage(std::integral_constant<int, S - 2>{});
        step(u, true, t + S);
        ++t;
    };
    using U0 = std::integral_constant<int, 0>;
    using U1 = std::integral_constant<int, 1>;
    using U2 = std::integral_constant<int, 2>;
    using U3 = std::integral_constant<int, 3>;
    while (t + S < steps) {
        link(U0{});
        link(U1{});
        link(U2{});
        link(U3{});
    }
    link(U0{}); // two or four steps are left
    if (t + 1 < steps) {
        link(U1{});
        link(U2{});
        step(U3{}, false, 0);
    } else {
        step(U1{}, false, 0);
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0)); // the loads past the end land before the LDS is used anew

    // 32 rows of the wave's tile at a time through LDS, four columns a lane; whole
    // lines past the caches (8192 x 4096 x 4096 over inputs that change 90 : 113 us)
    constexpr int RS = WN + 4, CL = WN / 4; // lanes of a row
    static_assert(CL == 16 || CL == 32, "whole rows per pass");
    static_assert(NW * 32 * RS * 4 <= S * STAGE * 16, "the regions fit the stages");
    LDS float *reg = (LDS float *)lds + wave * 32 * RS;
    const int c4 = (lane & (CL - 1)) * 4, lg = lane >> 4, M = (int)x.rows, N = (int)w.rows;
    const int col = n0 + wn * WN + c4;
    const bool v4 = rows_keep_four(y, w.rows);
#pragma unroll
    for (int i = 0; i < FM; i += 2) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    reg[(k * 16 + 4 * lg + e) * RS + j * 16 + (lane & 15)] = acc[i + k][j][e];
        __syncthreads();
#pragma unroll 1
        for (int row = lane / CL; row < 32; row += 64 / CL) {
            const int grow = m0 + wm * WM + i * 16 + row;
            if (grow < M && col < N)
                store4<true>(y + (size_t)grow * N + col, f32x4(*(const LDS f32x4 *)(reg + row * RS + c4)), N - col, v4);
        }
    }
}

// ---------------------------------------------------------------- launches

unsigned blocks_for(size_t n) { return (unsigned)((n + 255) / 256 < 8192 ? (n + 255) / 256 : 8192); }

template <class T>
bool vector_rows(const T *p, size_t cols)
{
    return ((uintptr_t)p & 15) == 0 && cols * sizeof(T) % 16 == 0;
}

// fn(grid, first x, first y) for parts of an x by y grid
template <class FN>
int by_parts(size_t x, size_t y, FN fn)
{
    for (size_t x0 = 0; x0 < x; x0 += kMostX)
        for (size_t y0 = 0; y0 < y; y0 += kMostY) {
            const size_t nx = x - x0 < kMostX ? x - x0 : kMostX, ny = y - y0 < kMostY ? y - y0 : kMostY;
            fn(dim3((unsigned)nx, (unsigned)ny), x0, y0);
            const int rc = (int)hipGetLastError();
            if (rc)
                return rc;
        }
    return 0;
}

template <class T>
int quantize(const pgk_mx4 &q, const T *src, int trans, hipStream_t st)
{
    if (trans)
        return by_parts((q.tiles + 3) / 4, q.steps / 2, [&](const dim3 &grid, size_t x0, size_t y0) {
            hipLaunchKernelGGL(k_mx4_columns<T>, grid, dim3(256), 0, st, q, src, x0, y0);
        });
    const dim3 grid(blocks_for(q.tiles * q.steps / 2 * 64));
    if (vector_rows(src, q.cols))
        hipLaunchKernelGGL((k_mx4_rows<T, true>), grid, dim3(256), 0, st, q, src);
    else
        hipLaunchKernelGGL((k_mx4_rows<T, false>), grid, dim3(256), 0, st, q, src);
    return (int)hipGetLastError();
}

template <class O>
int dequantize(const pgk_mx4 &q, O *dst, int trans, hipStream_t st)
{
    if (trans)
        return by_parts((q.tiles + 3) / 4, q.steps / 2, [&](const dim3 &grid, size_t x0, size_t y0) {
            hipLaunchKernelGGL(k_mx4_back_columns<O>, grid, dim3(256), 0, st, q, dst, x0, y0);
        });
    hipLaunchKernelGGL(k_mx4_back_rows<O>, dim3(blocks_for(q.rows * ((q.cols + 7) / 8))), dim3(256), 0, st, q, dst);
    return (int)hipGetLastError();
}

template <class T, class O>
int few(const T *x, size_t m, const pgk_mx4 &w, O *y, hipStream_t st)
{
    return by_parts(w.tiles, 1, [&](const dim3 &grid, size_t t0, size_t) {
        if (vector_rows(x, w.cols))
            hipLaunchKernelGGL((k_mx4_few<T, O, true>), grid, dim3(kFewWaves * 64), 0, st, x, (int)m, w, y, (int)t0);
        else
            hipLaunchKernelGGL((k_mx4_few<T, O, false>), grid, dim3(kFewWaves * 64), 0, st, x, (int)m, w, y, (int)t0);
    });
}

template <int FM, int FN, int KG, class O>
void split(const pgk_mx4 &x, const pgk_mx4 &w, O *y, hipStream_t st)
{
    const size_t blocks = (x.tiles + FM - 1) / FM * ((w.tiles + FN - 1) / FN);
    hipLaunchKernelGGL((k_mx4_split<FM, FN, KG, O>), dim3((unsigned)blocks), dim3(KG * 64), 0, st, x, w, y);
}

template <class O>
int product(const pgk_mx4 &x, const pgk_mx4 &w, O *y, hipStream_t st)
{
    auto tiles = [&](size_t bm, size_t bn) { return (x.rows + bm - 1) / bm * ((w.rows + bn - 1) / bn); };
    if (tiles(128, 128) >> 24) // 2^32 threads
        return (int)hipErrorInvalidValue;
    if (tiles(32, 32) <= 256)
        split<2, 2, 8>(x, w, y, st);
    else if (tiles(64, 32) <= 256)
        split<4, 2, 8>(x, w, y, st);
    else if (tiles(64, 64) <= 256)
        split<4, 4, 8>(x, w, y, st);
    else if (tiles(64, 64) <= 512)
        split<4, 4, 4>(x, w, y, st);
    else
        hipLaunchKernelGGL((k_mx4_tiles<128, 128, 2, 2, O>), dim3((unsigned)tiles(128, 128)), dim3(256), 0, st, x, w, y);
    return (int)hipGetLastError();
}

// fn with a null pointer of the type that a dtype code names
template <class FN>
int by_type(int dtype, FN fn)
{
    return dtype == 0 ? fn((float *)nullptr) : dtype == 1 ? fn((_Float16 *)nullptr) : fn((__bf16 *)nullptr);
}

} // namespace

extern "C" void pgk_mx4_shape(pgk_mx4 *q, size_t rows, size_t cols, size_t *code_bytes, size_t *power_bytes)
{
    q->rows = rows;
    q->cols = cols;
    q->tiles = (rows + 15) / 16;
    q->steps = (cols + 255) / 256 * 2;
    *code_bytes = q->tiles * q->steps * 1024;
    *power_bytes = q->tiles * q->steps * 64;
}

extern "C" int pgk_mx4_quantize(const pgk_mx4 *q, const void *src, int dtype, int trans, pgk_stream s)
{
    return by_type(dtype, [&](auto t) { return quantize(*q, (decltype(t))src, trans, (hipStream_t)s); });
}

extern "C" int pgk_mx4_dequantize(const pgk_mx4 *q, void *dst, int dtype, int trans, pgk_stream s)
{
    return by_type(dtype, [&](auto t) { return dequantize(*q, (decltype(t))dst, trans, (hipStream_t)s); });
}

extern "C" int pgk_mx4_few_rows(size_t m) { return m <= 16; }

extern "C" int pgk_mx4_matmul_few(const void *x, int dtype, size_t m, const pgk_mx4 *w, void *y, int y_dtype, pgk_stream s)
{
    if (!pgk_mx4_few_rows(m) || w->rows > 0x3fffffff || w->cols > (size_t)1 << 24)
        return (int)hipErrorInvalidValue;
    return by_type(dtype, [&](auto t) {
        return by_type(y_dtype, [&](auto o) {
            return few((const std::remove_pointer_t<decltype(t)> *)x, m, *w, (decltype(o))y, (hipStream_t)s);
        });
    });
}

extern "C" int pgk_mx4_matmul(const pgk_mx4 *x, const pgk_mx4 *w, void *y, int y_dtype, pgk_stream s)
{
    // (the offsets within a block's 16 tiles fit 32 bits)
    if (x->cols != w->cols || x->rows > 0x3fffffff || w->rows > 0x3fffffff || x->cols > (size_t)1 << 24)
        return (int)hipErrorInvalidValue;
    return by_type(y_dtype, [&](auto o) { return product(*x, *w, (decltype(o))y, (hipStream_t)s); });
}
