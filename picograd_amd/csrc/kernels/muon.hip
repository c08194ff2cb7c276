// Orthogonal factors by Newton-Schulz products, and the optimiser step made of
// them, for a list of matrices at once.
//
//   u = g, or with momentum m <- mu m + g and u = m (nesterov: g + mu m)
//   X = u / ||u||_F, of the shorter side m as rows (a tall u transposed)
//   `steps` times: S = X X^T, B = b S + c S S, X <- a X + B X
//   out = X, or W <- decay W - step X
//
// The singular values s of X follow s <- a s + b s^3 + c s^5; with (a, b, c) =
// (3.4445, -4.7750, 2.0315) those over 1/660 come to 0.68 .. 1.203 in five steps, and
// none passes 1.203 in any, so no entry of X, S or B passes 2.9.
//
// An error in an early X grows as the small singular values do, by up to a a
// step, so f32 is held throughout: X, S and B are kept as two f16 pieces each,
// high and low (22 to 23 bits), times 4096 to keep the low ones from the f16
// subnormals, and a product is three on the f16 matrix units, hh + hl + lh, in
// f32 sums.  Against 64 bits the result is as near as f32 products' (2.8e-6
// against 2.5e-6 of 512 x 512 with singular values over 3.5 decades; measured to
// sides of 4500).  Entries under 2^-15, such as X's before the first step past sides of
// some 2^15, have low pieces among the subnormals and are held to 2^-37 itself.
// a X is added apart from B X: a on the diagonal of B would round it with each
// entry and triples the error.
//
// S and S S are symmetric: tiles below the diagonal, each written twice.
//
// How a product is cut depends on all matrices of a launch, and with it the order of
// its sums: a matrix's last bits may differ with the others beside it, never from one
// call to the next.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "launch.h"
#include "piece_tile.h"

namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kUnit = 4096.0f; // the pieces hold values times this

constexpr int kMostParts = 512; // of a matrix's sum of squares
constexpr int kMost = PGK_MUON_MAX;

// A matrix on its way: X [mp, np] in two pieces, np mp places apart, and so S and
// B [mp, mp]; m, n its own sizes, mp, np those rounded up to 64 with zeros between
struct ns_prob {
    uint16_t *x, *to, *s, *b;
    double *part;
    int m, n, mp, np, parts;
    uint32_t per_part; // elements
};
// Tiles are numbered through all matrices; those from `whole` on are split along
// the reduction in z slices, whose sums go to partial and are joined by a launch of
// their own
struct ns_table {
    int n, whole, z;
    float *partial;
    int first[kMost + 1]; // blocks
    ns_prob p[kMost];
};
struct seg_table {
    int n, whole, z;
    float *partial;
    int first[kMost + 1];
    float mu;
    int nesterov;
    pgk_muon_seg seg[kMost];
    ns_prob p[kMost];
};

template <class TAB>
__device__ __forceinline__ int which(const TAB &t, int block)
{
    int i = 0;
    while (i + 1 < t.n && block >= t.first[i + 1])
        ++i;
    return i;
}

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// n (1 to 4) neighbours of the grad from element i
__device__ __forceinline__ void grad4(const pgk_muon_seg &s, size_t i, int n, float (&g)[4])
{
    auto from = [&](auto *p) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        typedef T v4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        if (n == 4) {
            const v4 v = *(const v4 *)(p + i);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                g[e] = (float)v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                g[e] = e < n ? (float)p[i + e] : 0.0f;
        }
    };
    if (s.g_dtype == 1)
        from((const _Float16 *)s.g);
    else if (s.g_dtype == 2)
        from((const __bf16 *)s.g);
    else
        from((const float *)s.g);
    if (s.gclip)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            g[e] = g[e] * s.gmul * s.ginv; // as a pending scale is written
}
__device__ __forceinline__ void momentum4(const float *p, int n, float (&m)[4])
{
    if (n == 4) {
        const f32x4u v = *(const f32x4u *)p;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            m[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            m[e] = e < n ? p[e] : 0.0f;
    }
}

// The momentum, and the blocks' sums of u's squares in 64 bits.
__global__ void __launch_bounds__(256) k_ns_size(seg_table t)
{
    __shared__ double sums[4];
    const int k = which(t, (int)blockIdx.x), part = (int)blockIdx.x - t.first[k], tid = (int)threadIdx.x;
    const pgk_muon_seg &s = t.seg[k];
    const ns_prob &p = t.p[k];
    const size_t n = s.rows * s.cols, begin = (size_t)part * p.per_part;
    const size_t end = begin + p.per_part < n ? begin + p.per_part : n;
    double sum = 0.0;
#pragma unroll 2
    for (size_t i = begin + tid * 4; i < end; i += 1024) {
        const int some = end - i < 4 ? (int)(end - i) : 4;
        float u[4], m[4];
        grad4(s, i, some, u);
        if (s.m) {
            momentum4(s.m + i, some, m);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = t.mu * m[e] + u[e];
                u[e] = t.nesterov ? u[e] + t.mu * m[e] : m[e];
            }
            if (some == 4)
                *(f32x4u *)(s.m + i) = f32x4u{m[0], m[1], m[2], m[3]};
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < some)
                        s.m[i + e] = m[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            sum += (double)u[e] * (double)u[e];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0)
        sums[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0)
        p.part[part] = sums[0] + sums[1] + sums[2] + sums[3];
}

__device__ __forceinline__ void pieces(float v, uint16_t &hi, uint16_t &lo)
{
    const _Float16 h = (_Float16)v, l = (_Float16)(v - (float)h);
    hi = __builtin_bit_cast(uint16_t, h);
    lo = __builtin_bit_cast(uint16_t, l);
}
__device__ __forceinline__ float whole(uint16_t hi, uint16_t lo)
{
    return (float)__builtin_bit_cast(_Float16, hi) + (float)__builtin_bit_cast(_Float16, lo);
}

// X from u, 64 x 64 of it a block, through LDS where u is tall.
__global__ void __launch_bounds__(256) k_ns_start(seg_table t)
{
    __shared__ double sums[4];
    __shared__ float tile[64][65];
    const int k = which(t, (int)blockIdx.x), tid = (int)threadIdx.x;
    const pgk_muon_seg &s = t.seg[k];
    const ns_prob &p = t.p[k];
    const int at = (int)blockIdx.x - t.first[k], across = p.np / 64, i0 = at / across * 64, j0 = at % across * 64;
    double sum = 0.0;
    for (int i = tid; i < p.parts; i += 256)
        sum += p.part[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0)
        sums[tid >> 6] = sum;
    __syncthreads();
    sum = sums[0] + sums[1] + sums[2] + sums[3];
    const double scale = sum == 0.0 ? 0.0 : (double)kUnit / sqrt(sum);
    const bool tall = s.rows > s.cols;
    const size_t plane = (size_t)p.mp * p.np;
    auto put = [&](int r, int c4, const float (&x)[4]) { // four neighbours of X
        uint16_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            pieces(x[e], h[e], l[e]);
        uint16_t *const d = p.x + (size_t)(i0 + r) * p.np + j0 + c4;
        *(uint2 *)d = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
        *(uint2 *)(d + plane) = make_uint2(l[0] | (uint32_t)l[1] << 16, l[2] | (uint32_t)l[3] << 16);
    };
    const int c4 = (tid & 15) * 4;
#pragma unroll
    for (int r = tid >> 4; r < 64; r += 16) {
        // row and columns of u
        const int row = (tall ? j0 : i0) + r, col = (tall ? i0 : j0) + c4;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if ((size_t)row < s.rows && (size_t)col < s.cols) {
            const size_t i = (size_t)row * s.cols + col;
            const int some = s.cols - col < 4 ? (int)(s.cols - col) : 4;
            float m[4];
            if (!s.m || t.nesterov)
                grad4(s, i, some, x);
            if (s.m) {
                momentum4(s.m + i, some, m);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = t.nesterov ? x[e] + t.mu * m[e] : m[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = (float)((double)x[e] * scale);
        }
        if (tall)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                tile[c4 + e][r] = x[e];
        else
            put(r, c4, x);
    }
    if (!tall)
        return;
    __syncthreads();
#pragma unroll
    for (int r = tid >> 4; r < 64; r += 16) {
        const float x[4] = {tile[r][c4], tile[r][c4 + 1], tile[r][c4 + 2], tile[r][c4 + 3]};
        put(r, c4, x);
    }
}

// four neighbours in two pieces
struct pieces4 {
    uint2 h, l;
    __device__ __forceinline__ void values(float (&v)[4]) const
    {
        v[0] = whole((uint16_t)h.x, (uint16_t)l.x);
        v[1] = whole((uint16_t)(h.x >> 16), (uint16_t)(l.x >> 16));
        v[2] = whole((uint16_t)h.y, (uint16_t)l.y);
        v[3] = whole((uint16_t)(h.y >> 16), (uint16_t)(l.y >> 16));
    }
};
__device__ __forceinline__ pieces4 raw4(const uint16_t *p, size_t plane)
{
    return {*(const uint2 *)p, *(const uint2 *)(p + plane)};
}
__device__ __forceinline__ void load4(const uint16_t *p, size_t plane, float (&v)[4]) { raw4(p, plane).values(v); }
__device__ __forceinline__ void store4(uint16_t *p, size_t plane, const f32x4 &v)
{
    uint16_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        pieces(v[e], h[e], l[e]);
    *(uint2 *)p = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    *(uint2 *)(p + plane) = make_uint2(l[0] | (uint32_t)l[1] << 16, l[2] | (uint32_t)l[3] << 16);
}

// n (1 to 4) neighbours of w from element i; of an output without w nothing is read
__device__ __forceinline__ f32x4 weights4(const pgk_muon_seg &s, size_t i, int n)
{
    f32x4 w = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!s.w)
        return w;
    if (n == 4) {
        const f32x4u v = *(const f32x4u *)(s.w + i);
        return f32x4{v[0], v[1], v[2], v[3]};
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n)
            w[e] = s.w[i + e];
    return w;
}
// what becomes of them, from the last X times kUnit
__device__ __forceinline__ void finish4(const pgk_muon_seg &s, size_t i, const f32x4 &w, const f32x4 &x, int n)
{
    typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(2)));
    f32x4 o = x * (1.0f / kUnit);
    if (s.w)
        o = s.decay * w - s.step * o;
    float *const wide = s.w ? s.w : s.out_dtype == 0 ? (float *)s.out : nullptr;
    if (wide) {
        if (n == 4)
            *(f32x4u *)(wide + i) = f32x4u{o[0], o[1], o[2], o[3]};
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n)
                    wide[i + e] = o[e];
    }
    uint16_t *const narrow = s.w ? s.shadow : (uint16_t *)s.out;
    const int dt = s.w ? s.shadow_dtype : s.out_dtype;
    if (!narrow || dt == 0)
        return;
    if (n == 4 && !s.shadow_cols) {
        *(u32x2u *)(narrow + i) = u32x2u{to16x2(dt, o[0], o[1]), to16x2(dt, o[2], o[3])};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) {
            const size_t j = i + e;
            narrow[s.shadow_cols ? j / s.shadow_cols * s.shadow_ld + j % s.shadow_cols : j] = to16(dt, o[e]);
        }
}

// the same of one
__device__ __forceinline__ void finish1(const pgk_muon_seg &s, uint32_t i, float x)
{
    const float o = s.w ? s.decay * s.w[i] - s.step * (x * (1.0f / kUnit)) : x * (1.0f / kUnit);
    if (s.w)
        s.w[i] = o;
    else if (s.out_dtype == 0)
        ((float *)s.out)[i] = o;
    uint16_t *const narrow = s.w ? s.shadow : (uint16_t *)s.out;
    const int dt = s.w ? s.shadow_dtype : s.out_dtype;
    if (narrow && dt != 0) {
        const uint32_t c = (uint32_t)s.shadow_cols;
        narrow[c ? i / c * s.shadow_ld + i % c : i] = to16(dt, o);
    }
}

enum { NS_S = 0, NS_B = 1, NS_X = 2, NS_LAST = 3 };

// row and column of tile i of a lower triangle, row by row
__device__ __forceinline__ void triangle(int i, int &r, int &c)
{
    r = (int)((sqrtf(8.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
    while (r * (r + 1) / 2 > i)
        --r;
    while ((r + 1) * (r + 2) / 2 <= i)
        ++r;
    c = i - r * (r + 1) / 2;
}

// tile `at` of a matrix: its first row and column
template <class CF, int WHAT>
__device__ __forceinline__ void tile_of(const ns_prob &p, int at, int &m0, int &n0)
{
    if constexpr (WHAT == NS_S || WHAT == NS_B) {
        triangle(at, m0, n0);
        m0 *= CF::BM;
        n0 *= CF::BN;
    } else { // eight tile-rows at a time
        const int tiles_m = (p.mp + CF::BM - 1) / CF::BM, tiles_n = (p.np + CF::BN - 1) / CF::BN;
        const int per_group = 8 * tiles_n, group = at / per_group, first = group * 8;
        const int gsz = tiles_m - first < 8 ? tiles_m - first : 8, in = at - group * per_group;
        m0 = (first + in % gsz) * CF::BM;
        n0 = in / gsz * CF::BN;
    }
}

// the reduction of a product
template <int WHAT>
__device__ __forceinline__ int depth_of(const ns_prob &p)
{
    return WHAT == NS_S ? p.np : p.mp;
}

// strip i of the tile at (m0, n0): what becomes of the sums
template <class CF, int WHAT, class TAB>
__device__ __forceinline__ void strip_out(const TAB &t, int k, f32x16 (&acc)[CF::FN], int i, int m0, int n0,
                                          LDS uint4 *const lds)
{
    const ns_prob &p = t.p[k];
    const size_t px = (size_t)p.mp * p.np, ps = (size_t)p.mp * p.mp;
    if constexpr (WHAT == NS_S || WHAT == NS_B) {
        uint16_t *const to = WHAT == NS_S ? p.s : p.b;
        piece_out_strip<CF, f32x4>(
            acc, i, m0, n0, p.mp, p.mp, lds, m0 != n0,
            [&](int row, int col) {
                if constexpr (WHAT == NS_B)
                    return raw4(p.s + (size_t)row * p.mp + col, ps);
                else
                    return 0;
            },
            [&](int row, int col, f32x4 &v, const auto &with, bool mirror) {
                if (mirror) {
                    store4(to + (size_t)col * p.mp + row, ps, v);
                    return;
                }
                v *= 1.0f / kUnit;
                if constexpr (WHAT == NS_B) {
                    float x[4];
                    with.values(x);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] = kB * x[e] + kC * v[e];
                }
                store4(to + (size_t)row * p.mp + col, ps, v);
            });
    } else if constexpr (WHAT == NS_X) {
        piece_out_strip<CF, f32x4>(
            acc, i, m0, n0, p.mp, p.np, lds, false,
            [&](int row, int col) { return raw4(p.x + (size_t)row * p.np + col, px); },
            [&](int row, int col, f32x4 &v, const pieces4 &with, bool) {
                float x[4];
                with.values(x);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = kA * x[e] + v[e] * (1.0f / kUnit);
                store4(p.to + (size_t)row * p.np + col, px, v);
            });
    } else { // as u lies
        const pgk_muon_seg &s = t.seg[k];
        const bool tall = s.rows > s.cols;
        struct from4 {
            pieces4 x;
            f32x4 w;
        };
        piece_out_strip<CF, f32x4, 2>(
            acc, i, m0, n0, p.mp, p.np, lds, tall,
            [&](int row, int col) {
                from4 q = {raw4(p.x + (size_t)row * p.np + col, px), {}};
                if (!tall && row < p.m && col < p.n)
                    q.w = weights4(s, (size_t)row * p.n + col, p.n - col < 4 ? p.n - col : 4);
                return q;
            },
            [&](int row, int col, f32x4 &v, const from4 &with, bool mirror) {
                if (!mirror) {
                    float x[4];
                    with.x.values(x);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] = kA * x[e] + v[e] * (1.0f / kUnit);
                }
                if (mirror != tall || row >= p.m || col >= p.n)
                    return;
                const int left = tall ? p.m - row : p.n - col, n = left < 4 ? left : 4;
                const size_t at = tall ? (size_t)col * p.m + row : (size_t)row * p.n + col;
                finish4(s, at, tall ? weights4(s, at, n) : with.w, v, n);
            });
    }
}

// a slice's part of a tile's sums, in the order in which the lanes hold them
template <class CF>
__device__ __forceinline__ f32x4 *partial_at(float *p, size_t unit, int i, int j)
{
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    return (f32x4 *)p + ((unit * (CF::NT / 64) + wave) * (CF::FM * CF::FN) + i * CF::FN + j) * 256 + lane;
}

// One product for every matrix: S, B, the next X or the last.  The 256 x 256 tiles of
// 4096 x 4096 run at 1300 TFLOP/s of the three f16 products, where a large f16
// product alone reaches 1060 on the same card: a k-step's three products share
// the operands of two, so less is moved for each.  Bound by the matrix units at the
// clock that they hold.
template <class CF, int WHAT, class TAB>
__global__ void __launch_bounds__(CF::NT, 1) k_ns_product(TAB t)
{
    __shared__ uint4 smem[CF::LDS_U4];
    LDS uint4 *const lds = (LDS uint4 *)smem;
    int tile = (int)blockIdx.x, slice = 0;
    const bool split = tile >= t.whole;
    if (split) {
        const int r = tile - t.whole;
        tile = t.whole + r / t.z;
        slice = r % t.z;
    } else { // neighbours on one XCD, within what the chip runs at a time
        constexpr int round = CF::BM == 64 ? 512 : 256;
        const int first = tile / round * round, left = t.whole - first;
        tile = first + xcd_tile(tile - first, left < round ? left : round);
    }
    const int k = which(t, tile);
    const ns_prob &p = t.p[k];
    const size_t px = (size_t)p.mp * p.np, ps = (size_t)p.mp * p.mp;
    int m0, n0;
    tile_of<CF, WHAT>(p, tile - t.first[k], m0, n0);
    int begin = 0, end = depth_of<WHAT>(p);
    if (split) {
        const int kt = end / CF::KB;
        begin = kt * slice / t.z * CF::KB;
        end = kt * (slice + 1) / t.z * CF::KB;
        if (begin == end) // fewer tiles of the reduction than slices
            return;
    }
    f32x16 acc[CF::FM][CF::FN];
    if constexpr (WHAT == NS_S)
        piece_loop<CF>({p.x, (size_t)p.np, px, p.mp}, {p.x, (size_t)p.np, px, p.mp}, begin, end - begin, m0, n0, lds, acc);
    else if constexpr (WHAT == NS_B)
        piece_loop<CF>({p.s, (size_t)p.mp, ps, p.mp}, {p.s, (size_t)p.mp, ps, p.mp}, begin, end - begin, m0, n0, lds, acc);
    else
        piece_loop<CF>({p.b, (size_t)p.mp, ps, p.mp}, {p.x, (size_t)p.np, px, p.np}, begin, end - begin, m0, n0, lds, acc);
    if (split) {
        const size_t unit = blockIdx.x - t.whole;
#pragma unroll
        for (int i = 0; i < CF::FM; ++i)
#pragma unroll
            for (int j = 0; j < CF::FN; ++j) {
                f32x4 *const to = partial_at<CF>(t.partial, unit, i, j);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    to[q * 64] = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < CF::FM; ++i)
        strip_out<CF, WHAT>(t, k, acc[i], i, m0, n0, lds);
}

// The slices of split tiles joined in their order, a strip a block.
template <class CF, int WHAT, class TAB>
__global__ void __launch_bounds__(CF::NT, 1) k_ns_join(TAB t)
{
    __shared__ uint4 smem[CF::OUT_U4];
    LDS uint4 *const lds = (LDS uint4 *)smem;
    const int r = (int)blockIdx.x / CF::FM, i = (int)blockIdx.x % CF::FM, tile = t.whole + r, k = which(t, tile);
    const ns_prob &p = t.p[k];
    int m0, n0;
    tile_of<CF, WHAT>(p, tile - t.first[k], m0, n0);
    const int kt = depth_of<WHAT>(p) / CF::KB;
    f32x16 acc[CF::FN];
#pragma unroll
    for (int j = 0; j < CF::FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            acc[j][e] = 0.0f;
#pragma unroll 2
    for (int s = 0; s < t.z; ++s) {
        if (kt * s / t.z == kt * (s + 1) / t.z)
            continue;
#pragma unroll
        for (int j = 0; j < CF::FN; ++j) {
            const f32x4 *const from = partial_at<CF>(t.partial, (size_t)r * t.z + s, i, j);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 v = from[q * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[j][4 * q + e] += v[e];
            }
        }
    }
    strip_out<CF, WHAT>(t, k, acc, i, m0, n0, lds);
}

// ---------------------------------------------------------------- small matrices, a block each

// Short sides of up to 64, long ones of up to NP: everything in LDS, X as rows of
// both sides so that each product's operands lie along its reduction.  Sixteen
// waves, one 16 x 16 tile of S and B each, which keep their tiles of S and X in f32
// beside the pieces that the others read; tiles and parts of the reduction past the
// matrix's own sizes are left out.  Bound by the chain of dependent products: 64 x 64
// in five steps takes 15 of them, 16.4 us, where launches of their own take 4 us each.
constexpr int kSmallM = 64, kSmallN = 256;

__device__ __forceinline__ f32x4 mma16(const uint4 &a, const uint4 &b, const f32x4 &c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int NP>
__global__ void __launch_bounds__(1024, 1) k_ns_small(seg_table t, int steps)
{
    constexpr int M = kSmallM, PX = NP + 8, PM = M + 8, T = NP / 64; // pitches; tiles of X per wave
    constexpr int XP = M * PX, YP = NP * PM, SP = M * PM;            // a piece of X, of its transpose, of S
    __shared__ uint4 mem[(2 * XP + 2 * YP + 2 * SP) / 8];
    __shared__ double sums[16];
    uint16_t *const X = (uint16_t *)mem, *const Y = X + 2 * XP, *const S = Y + 2 * YP;
    const pgk_muon_seg &s = t.seg[blockIdx.x];
    const int tid = (int)threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6); // (uniform to the compiler: matrix instructions heed no mask)
    const int rows = (int)s.rows, cols = (int)s.cols;
    const bool tall = rows > cols;
    const int sm = tall ? cols : rows, sn = tall ? rows : cols;
    for (int i = tid; i < (2 * XP + 2 * YP + 2 * SP) / 8; i += 1024)
        mem[i] = make_uint4(0, 0, 0, 0);
    // up to Q pieces of four values a thread
    constexpr int Q = M * NP / 4096;
    const int per = (cols + 3) / 4;
    float u[Q][4];
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int at = tid + q * 1024, row = at / per, col = (at - row * per) * 4;
        if (row >= rows)
            break;
        const size_t i = (size_t)row * cols + col;
        const int some = cols - col < 4 ? cols - col : 4;
        grad4(s, i, some, u[q]);
        if (s.m) {
            float m[4];
            momentum4(s.m + i, some, m);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = t.mu * m[e] + u[q][e];
                u[q][e] = t.nesterov ? u[q][e] + t.mu * m[e] : m[e];
                if (e < some)
                    s.m[i + e] = m[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            sum += (double)u[q][e] * (double)u[q][e];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        sum += __shfl_xor(sum, o);
    if (lane == 0)
        sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < 16; ++w)
        sum += sums[w];
    const double scale = sum == 0.0 ? 0.0 : (double)kUnit / sqrt(sum);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int at = tid + q * 1024, row = at / per, col = (at - row * per) * 4;
        if (row >= rows)
            break;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < cols) {
                const int i = tall ? col + e : row, j = tall ? row : col + e;
                uint16_t h, l;
                pieces((float)((double)u[q][e] * scale), h, l);
                X[i * PX + j] = h;
                X[XP + i * PX + j] = l;
                Y[j * PM + i] = h;
                Y[YP + j * PM + i] = l;
            }
    }
    __syncthreads();
    // the sums over k <= MOST of rows a0 + lr of A and b0 + lr of B: lane gets column lr
    // of rows 4 lg .. + 3
    auto product = [&](const uint16_t *A, int pa, int planeA, int a0, const uint16_t *B, int pb, int planeB, int b0, auto most,
                       int k) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        const uint16_t *const a = A + (a0 + lr) * pa + lg * 8, *const b = B + (b0 + lr) * pb + lg * 8;
#pragma unroll
        for (int i = 0; i < decltype(most)::value; i += 32) {
            if (i >= k)
                break;
            const uint4 ah = *(const uint4 *)(a + i), al = *(const uint4 *)(a + planeA + i);
            const uint4 bh = *(const uint4 *)(b + i), bl = *(const uint4 *)(b + planeB + i);
            acc = mma16(ah, bh, acc);
            acc = mma16(ah, bl, acc);
            acc = mma16(al, bh, acc);
        }
        return acc;
    };
    const std::integral_constant<int, M> along_m;
    const std::integral_constant<int, NP> along_n;
    const int ti = wave >> 2 << 4, tj = (wave & 3) << 4;
    const bool has_s = ti < sm && tj < sm; // a tile of S
    auto has_x = [&](int j0) { return ti < sm && j0 < sn; };
    uint16_t *const mine = S + (tj + lr) * PM + ti + 4 * lg; // S and B are symmetric: down a column is along a row
    f32x4 x[T];
#pragma unroll
    for (int q = 0; q < T; ++q) {
        float v[4];
        load4(Y + (q * 64 + tj + lr) * PM + ti + 4 * lg, YP, v);
        x[q] = f32x4{v[0], v[1], v[2], v[3]};
    }
    for (int step = 0; step < steps; ++step) {
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (has_s) {
            v = product(X, PX, XP, ti, X, PX, XP, tj, along_n, sn) * (1.0f / kUnit);
            store4(mine, SP, v);
        }
        __syncthreads();
        if (has_s)
            v = kB * v + product(S, PM, SP, ti, S, PM, SP, tj, along_m, sm) * (kC / kUnit);
        __syncthreads(); // S is read
        if (has_s)
            store4(mine, SP, v);
        __syncthreads();
#pragma unroll
        for (int q = 0; q < T; ++q) {
            const int j0 = q * 64 + tj;
            if (has_x(j0))
                x[q] = kA * x[q] + product(S, PM, SP, ti, Y, PM, YP, j0, along_m, sm) * (1.0f / kUnit);
        }
        if (step + 1 == steps) {
#pragma unroll
            for (int q = 0; q < T; ++q) {
                const int i = ti + 4 * lg, j = q * 64 + tj + lr;
                if (i >= sm || j >= sn)
                    continue;
                if (tall) {
                    const size_t at = (size_t)j * sm + i;
                    const int some = sm - i < 4 ? sm - i : 4;
                    finish4(s, at, weights4(s, at, some), x[q], some);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (i + e < sm) {
                            const size_t at = (size_t)(i + e) * sn + j;
                            finish4(s, at, weights4(s, at, 1), f32x4{x[q][e], 0.0f, 0.0f, 0.0f}, 1);
                        }
                }
            }
            break;
        }
        __syncthreads(); // X is read
#pragma unroll
        for (int q = 0; q < T; ++q) {
            const int j0 = q * 64 + tj, j = j0 + lr, i = ti + 4 * lg;
            if (!has_x(j0))
                continue;
            uint16_t h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pieces(x[q][e], h[e], l[e]);
                X[(i + e) * PX + j] = h[e];
                X[XP + (i + e) * PX + j] = l[e];
            }
            store4(Y + j * PM + i, YP, x[q]);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- thin matrices, a block each

// Short sides of up to 16 MB (MB 1 or 2), long ones of up to 256 SW: X stays in
// registers, of the long kinds (16 and 2 x 8 blocks a wave) but for some 100 of them that
// the compiler spills (356 and 404 bytes a lane).  A wave owns strips of 16 columns; a lane holds column lane % 16 of rows
// 4 (lane / 16) .. + 3 of each 16 x 16 block, as the 16 x 16 x 16 products give their
// sums and as they take an operand whose reduction runs along those rows.  So
//   B X takes X as it lies, and leaves it so;
//   X X^T takes X turned, which is its pieces' product with the unit matrix (exact);
//   S, symmetric, serves as either operand as it lies.
// Only the waves' parts of S pass through LDS, joined in the waves' order; B each wave
// works out by itself.  Bound by one CU: the conversions between f32 and pieces and, of
// the long kinds, the spills' way (five steps of 16 x 4096, 16 strips a wave, 74 us, and of
// 4096 x 16 113; in launches of their own 137 and 139), of a few strips the two barriers
// of a step (1 x 64: 7.0 us).
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

struct halves4 {
    f16x4 h, l;
    __device__ __forceinline__ halves4() {}
    __device__ __forceinline__ explicit halves4(const f32x4 &v)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            h[e] = (_Float16)v[e];
            l[e] = (_Float16)(v[e] - (float)h[e]);
        }
    }
};
__device__ __forceinline__ f32x4 mma4(const f16x4 &a, const f16x4 &b, const f32x4 &c)
{
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma4(const halves4 &a, const halves4 &b, f32x4 c)
{
    c = mma4(a.h, b.h, c);
    c = mma4(a.h, b.l, c);
    return mma4(a.l, b.h, c);
}

// with what both pieces leave over, all of f32's bits
struct thirds4 : halves4 {
    f16x4 r;
    __device__ __forceinline__ thirds4() {}
    __device__ __forceinline__ explicit thirds4(const f32x4 &v) : halves4(v)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            r[e] = (_Float16)(v[e] - (float)h[e] - (float)l[e]);
    }
};
// the products beside that of the high pieces
__device__ __forceinline__ f32x4 rest4(const thirds4 &a, const halves4 &b)
{
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return mma4(a.l, b.h, mma4(a.h, b.l, mma4(a.l, b.l, mma4(a.r, b.h, zero))));
}
__device__ __forceinline__ f32x4 rest4(const thirds4 &a, const thirds4 &b)
{
    return rest4(a, (const halves4 &)b) + mma4(a.h, b.r, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
}

template <int MB, int SW>
__global__ void __launch_bounds__(1024, 1) k_ns_thin(seg_table t, int steps)
{
    constexpr int SIZE = MB * MB * 256;
    // FINE, one strip a wave: products with B and of S with itself take all of f32's bits, and
    // what cancels between a X and B X (b S and c S S) does so in the high pieces' products,
    // before the others are added.  The errors of S and B are shared by whole rows of X
    // and average out over many rows only: over 64 inputs each of 1 x 7 to 4 x 60 those of two
    // pieces are 1.6 to 2.4 times f32 products' in the root mean square, these 0.7 to 1.2.
    constexpr bool FINE = SW == 1;
    static_assert(!FINE || MB == 1, "one block");
    using whole4 = std::conditional_t<FINE, thirds4, halves4>;
    __shared__ float parts[16][SIZE], joined[SIZE];
    __shared__ double sums[16];
    const pgk_muon_seg s = t.seg[blockIdx.x];
    const int tid = (int)threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6); // (uniform to the compiler: matrix instructions heed no mask)
    const int rows = (int)s.rows, cols = (int)s.cols;
    const bool tall = rows > cols;
    const int m = tall ? cols : rows, n = tall ? rows : cols, strips = (n + 15) / 16, waves = strips < 16 ? strips : 16;
    // neighbours of a lane lie `along` apart
    const uint32_t along = tall ? 1 : n;
    auto place = [&](int q, int b) { // of the first
        const uint32_t i = b * 16 + 4 * lg, j = (q * 16 + wave) * 16 + lr;
        return tall ? j * m + i : i * n + j;
    };
    auto some = [&](int q, int b) { // how many there are
        const int left = m - (b * 16 + 4 * lg);
        return (q * 16 + wave) * 16 + lr < n && left > 0 ? left < 4 ? left : 4 : 0;
    };
    f32x4 x[SW][MB];
    auto fetch = [&](auto *p) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        T raw[SW][MB][4];
#pragma unroll
        for (int q = 0; q < SW; ++q)
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                __builtin_amdgcn_sched_barrier(0); // (all addresses at once would not fit the registers)
                const uint32_t at = place(q, b);
                const int k = some(q, b);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    raw[q][b][e] = p[e < k ? at + e * along : 0];
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < SW; ++q)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[q][b][e] = e < some(q, b) ? (float)raw[q][b][e] : 0.0f;
    };
    if (s.g_dtype == 1)
        fetch((const _Float16 *)s.g);
    else if (s.g_dtype == 2)
        fetch((const __bf16 *)s.g);
    else
        fetch((const float *)s.g);
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < SW; ++q)
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            f32x4 &u = x[q][b];
            if (s.gclip)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    u[e] = u[e] * s.gmul * s.ginv; // as a pending scale is written
            __builtin_amdgcn_sched_barrier(0);
            if (s.m) {
                const uint32_t at = place(q, b);
                const int k = some(q, b);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = s.m[e < k ? at + e * along : 0];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < k) {
                        v[e] = t.mu * v[e] + u[e];
                        s.m[at + e * along] = v[e];
                        u[e] = t.nesterov ? u[e] + t.mu * v[e] : v[e];
                    }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sum += (double)u[e] * (double)u[e];
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        sum += __shfl_xor(sum, o);
    if (lane == 0)
        sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < 16; ++w)
        sum += sums[w];
    const double scale = sum == 0.0 ? 0.0 : (double)kUnit / sqrt(sum);
#pragma unroll
    for (int q = 0; q < SW; ++q)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[q][b][e] = (float)((double)x[q][b][e] * scale);
    f16x4 unit;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        unit[e] = (_Float16)(4 * lg + e == lr ? 1.0f : 0.0f);
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int step = 0; step < steps; ++step) {
        f32x4 g[MB][MB];
#pragma unroll
        for (int r = 0; r < MB; ++r)
#pragma unroll
            for (int c = 0; c < MB; ++c)
                g[r][c] = zero;
#pragma unroll
        for (int q = 0; q < SW; ++q) {
            if (q * 16 + wave >= strips)
                break;
            halves4 turned[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                const halves4 v(x[q][b]);
                const f32x4 h = mma4(v.h, unit, zero), l = mma4(v.l, unit, zero);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    turned[b].h[e] = (_Float16)h[e];
                    turned[b].l[e] = (_Float16)l[e];
                }
            }
            if constexpr (FINE) {
                const halves4 &t0 = turned[0];
                g[0][0] = mma4(t0.l, t0.h, mma4(t0.h, t0.l, mma4(t0.l, t0.l, zero))) + mma4(t0.h, t0.h, zero);
                break;
            }
#pragma unroll
            for (int r = 0; r < MB; ++r)
#pragma unroll
                for (int c = 0; c < MB; ++c)
                    g[r][c] = mma4(turned[r], turned[c], g[r][c]);
        }
        if (wave < waves)
#pragma unroll
            for (int r = 0; r < MB; ++r)
#pragma unroll
                for (int c = 0; c < MB; ++c)
                    *(f32x4 *)&parts[wave][(r * MB + c) * 256 + lane * 4] = g[r][c];
        __syncthreads();
        if (tid < SIZE) {
            float v = 0.0f;
            for (int w = 0; w < waves; ++w)
                v += parts[w][tid];
            joined[tid] = v * (1.0f / kUnit);
        }
        __syncthreads();
        if (wave >= waves)
            continue;
        // blocks [r][c] of S and B: rows of r, a column of c; by symmetry a row of c along r
        f32x4 f[MB][MB];
        whole4 a[MB][MB];
#pragma unroll
        for (int r = 0; r < MB; ++r)
#pragma unroll
            for (int c = 0; c < MB; ++c) {
                f[r][c] = *(const f32x4 *)&joined[(r * MB + c) * 256 + lane * 4];
                a[r][c] = whole4(f[r][c]);
            }
#pragma unroll
        for (int r = 0; r < MB; ++r)
#pragma unroll
            for (int c = 0; c < MB; ++c) {
                if constexpr (FINE) {
                    f[0][0] = kB * f[0][0] + mma4(a[0][0].h, a[0][0].h, zero) * (kC / kUnit);
                    f[0][0] += rest4(a[0][0], a[0][0]) * (kC / kUnit);
                    break;
                }
                f32x4 v = zero;
#pragma unroll
                for (int k = 0; k < MB; ++k)
                    v = mma4(a[k][r], a[k][c], v);
                f[r][c] = kB * f[r][c] + v * (kC / kUnit);
            }
#pragma unroll
        for (int r = 0; r < MB; ++r)
#pragma unroll
            for (int c = 0; c < MB; ++c)
                a[r][c] = whole4(f[r][c]);
#pragma unroll
        for (int q = 0; q < SW; ++q) {
            if (q * 16 + wave >= strips)
                break;
            whole4 v[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b)
                v[b] = whole4(x[q][b]);
#pragma unroll
            for (int r = 0; r < MB; ++r) {
                if constexpr (FINE) {
                    x[q][0] = kA * x[q][0] + mma4(a[0][0].h, v[0].h, zero) * (1.0f / kUnit);
                    x[q][0] += rest4(a[0][0], v[0]) * (1.0f / kUnit);
                    break;
                }
                f32x4 y = zero;
#pragma unroll
                for (int k = 0; k < MB; ++k)
                    y = mma4(a[k][r], v[k], y);
                x[q][r] = kA * x[q][r] + y * (1.0f / kUnit);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < SW; ++q)
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            __builtin_amdgcn_sched_barrier(0);
            const uint32_t at = place(q, b);
            const int k = some(q, b);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < k)
                    finish1(s, at + e * along, x[q][b][e]);
        }
}

// ---------------------------------------------------------------- launches

template <bool TB>
using T256 = pcfg<f32x16, 2, 256, 256, 2, 4, TB, 32, 2>;
template <bool TB>
using T128 = pcfg<f32x16, 2, 128, 128, 4, 2, TB, 32, 4>;
template <bool TB>
using T64 = pcfg<f32x16, 2, 64, 64, 2, 2, TB, 64, 2>;
template <bool TB>
using ONE64 = pcfg<f32x16, 2, 64, 64, 2, 2, TB, 32, 4>; // for one to a CU: more stages on their way

size_t up64(size_t v) { return (v + 63) & ~(size_t)63; }

void shape(const pgk_muon_seg &s, ns_prob *p)
{
    const size_t m = s.rows < s.cols ? s.rows : s.cols, n = s.rows < s.cols ? s.cols : s.rows, all = m * n;
    size_t per = (all + kMostParts - 1) / kMostParts;
    per = per < 4096 ? 4096 : per;
    *p = {};
    p->m = (int)m;
    p->n = (int)n;
    p->mp = (int)up64(m);
    p->np = (int)up64(n);
    p->per_part = (uint32_t)per;
    p->parts = (int)((all + per - 1) / per);
}
template <class TAB, class FN>
int number(TAB &t, FN blocks)
{
    int all = 0;
    for (int i = 0; i < t.n; ++i) {
        t.first[i] = all;
        all += blocks(t.p[i]);
    }
    t.first[t.n] = all;
    return all;
}

// tiles of a side: below the diagonal, or all of X
int tiles_of(const ns_prob &p, int what, int side)
{
    const int r = (p.mp + side - 1) / side;
    return what == NS_S || what == NS_B ? r * (r + 1) / 2 : r * ((p.np + side - 1) / side);
}

// How a product of all matrices is cut.  Whole rounds of tiles over the chip run
// as they are; what is left, less than a round, is split along the reduction
// where that is faster.  The time of 32 along the reduction was measured with few
// blocks and with as many as fit (two on a CU of 64, else one), in us: 1.7 and 2.4
// for a side of 256, 0.5 and 0.75 for 128, 0.36 and 0.44 for 64, 0.25 and 0.29 for 64 one
// to a CU; a joining launch takes some 5 us and the partial sums' way at 3.5 TB/s.
struct ns_plan {
    int side, kind, whole, z, tiles;
};
enum { KIND256, KIND128, KIND64, KIND_ONE64 };
ns_plan plan_of(const ns_prob *p, int n, int what)
{
    static const struct {
        int side, blocks;
        double alone, full;
    } kinds[4] = {{256, 1, 1.7, 2.4}, {128, 1, 0.5, 0.75}, {64, 2, 0.36, 0.44}, {64, 1, 0.25, 0.29}};
    ns_plan best = {};
    double least = 0.0;
    for (const auto &c : kinds) {
        int tiles = 0;
        double work = 0.0; // of the reduction, in 32s
        for (int i = 0; i < n; ++i) {
            tiles += tiles_of(p[i], what, c.side);
            work += (double)tiles_of(p[i], what, c.side) * ((what == NS_S ? p[i].np : p[i].mp) / 32);
        }
        const int slots = 256 * c.blocks, whole = tiles / slots * slots, rest = tiles - whole;
        // the longest reduction among the last tiles
        int depth = 0;
        double left = 0.0;
        for (int i = n - 1, seen = 0; i >= 0 && seen < rest; --i) {
            const int t = tiles_of(p[i], what, c.side), d = (what == NS_S ? p[i].np : p[i].mp) / 32;
            left += (double)(t < rest - seen ? t : rest - seen) * d;
            depth = d > depth ? d : depth;
            seen += t;
        }
        for (int z = 1; rest ? z <= 16 && rest * z <= slots && (z == 1 || depth / z >= 4) : z == 1; ++z) {
            const int units = rest * z;
            const double steps = (double)((depth + z - 1) / z);
            double time = (work - left) / slots * c.full;
            if (rest)
                time += 2.0 + steps * (units <= 256 ? c.alone + (c.full / c.blocks - c.alone) * (c.blocks == 1 ? units / 256.0 : 0.0)
                                                    : c.full);
            if (z > 1)
                time += 5.0 + units * (double)c.side * c.side * 8.0 / 3.5e6;
            if (!best.side || time < least) {
                least = time;
                best = {c.side, (int)(&c - kinds), z == 1 ? tiles : whole, z, tiles};
            }
        }
    }
    return best;
}
size_t partial_bytes(const ns_plan &q) { return (size_t)(q.tiles - q.whole) * q.z * q.side * q.side * sizeof(float); }

template <template <bool> class TILE, int WHAT, class TAB>
int launch(TAB &t, const ns_plan &q, hipStream_t st)
{
    using CF = TILE<(WHAT == NS_X || WHAT == NS_LAST)>;
    number(t, [&](const ns_prob &p) { return tiles_of(p, WHAT, q.side); });
    t.whole = q.whole;
    t.z = q.z;
    const int rest = q.tiles - q.whole;
    hipLaunchKernelGGL((k_ns_product<CF, WHAT, TAB>), dim3((unsigned)(q.whole + rest * q.z)), dim3(CF::NT), 0, st, t);
    if (rest)
        hipLaunchKernelGGL((k_ns_join<CF, WHAT, TAB>), dim3((unsigned)(rest * CF::FM)), dim3(CF::NT), 0, st, t);
    return (int)hipGetLastError();
}

template <int WHAT, class TAB>
int product(TAB &t, hipStream_t st)
{
    const ns_plan q = plan_of(t.p, t.n, WHAT);
    return q.kind == KIND256   ? launch<T256, WHAT>(t, q, st)
           : q.kind == KIND128 ? launch<T128, WHAT>(t, q, st)
           : q.kind == KIND64  ? launch<T64, WHAT>(t, q, st)
                               : launch<ONE64, WHAT>(t, q, st);
}

// the matrices' own places and the partial sums'
size_t places(ns_prob *p, int n, char *at, float **partial)
{
    char *const begin = at;
    size_t most = 0;
    for (int what = NS_S; what <= NS_X; ++what) {
        const size_t b = partial_bytes(plan_of(p, n, what));
        most = b > most ? b : most;
    }
    *partial = (float *)at;
    at += most;
    for (int i = 0; i < n; ++i) {
        const size_t px = (size_t)p[i].mp * p[i].np * 4, ps = (size_t)p[i].mp * p[i].mp * 4;
        p[i].x = (uint16_t *)at;
        p[i].to = (uint16_t *)(at + px);
        p[i].s = (uint16_t *)(at + 2 * px);
        p[i].b = (uint16_t *)(at + 2 * px + ps);
        p[i].part = (double *)(at + 2 * px + 2 * ps);
        at += 2 * px + 2 * ps + kMostParts * sizeof(double);
    }
    return (size_t)(at - begin);
}

// the largest first, so that the tiles left over are the shortest
void order(ns_prob *p, pgk_muon_seg *seg, int n)
{
    for (int i = 1; i < n; ++i)
        for (int j = i; j > 0 && (size_t)p[j].mp * p[j].np > (size_t)p[j - 1].mp * p[j - 1].np; --j) {
            std::swap(p[j], p[j - 1]);
            if (seg)
                std::swap(seg[j], seg[j - 1]);
        }
}

bool fits(const pgk_muon_seg &s)
{
    return s.rows && s.cols && s.rows <= PGK_MUON_MAX_SIDE && s.cols <= PGK_MUON_MAX_SIDE;
}

// matrices that a block holds, by its kernel; FINE where it costs nothing (16 x 64: 7.5 us, in
// two pieces 7.7; 16 x 256 11.3 and 10.2) and for few rows, which need it
enum { LARGE = -1, SMALL64, SMALL256, THIN16_FINE, THIN16, THIN16_LONG, THIN32, THIN32_LONG, KINDS };
int kind_of(const pgk_muon_seg &s)
{
    const size_t lo = s.rows < s.cols ? s.rows : s.cols, hi = s.rows < s.cols ? s.cols : s.rows;
    if (lo <= 16)
        return hi <= (lo <= 4 ? 256 : 64) ? THIN16_FINE : hi <= 1024 ? THIN16 : hi <= 4096 ? THIN16_LONG : LARGE;
    if (lo <= 32)
        return hi <= 512 ? THIN32 : hi <= 2048 ? THIN32_LONG : LARGE;
    return lo > kSmallM || hi > kSmallN ? LARGE : hi <= 64 ? SMALL64 : SMALL256;
}

// Long thin ones beside a large one take their tiles in its launches: 4096 x 10 costs
// 81 us on a CU of its own before them, next to nothing in 7.4 ms of theirs.
void kinds_of(const pgk_muon_seg *segs, int n, int (&kind)[kMost])
{
    bool large = false;
    for (int i = 0; i < n; ++i) {
        kind[i] = kind_of(segs[i]);
        large |= kind[i] == LARGE;
    }
    for (int i = 0; i < n; ++i)
        if (large && (kind[i] == THIN16_LONG || kind[i] == THIN32_LONG))
            kind[i] = LARGE;
}

} // namespace

extern "C" size_t pgk_muon_workspace(const pgk_muon_seg *segs, int n)
{
    ns_prob p[kMost];
    int k = 0, kind[kMost];
    n = n < kMost ? n : kMost;
    kinds_of(segs, n, kind);
    for (int i = 0; i < n; ++i)
        if (kind[i] == LARGE)
            shape(segs[i], &p[k++]);
    order(p, NULL, k);
    float *partial;
    return k ? places(p, k, NULL, &partial) : 0;
}

extern "C" int pgk_muon(const pgk_muon_seg *segs, int n, float mu, int nesterov, int steps, void *ws, pgk_stream s)
{
    if (n < 1 || n > kMost || steps < 1)
        return (int)hipErrorInvalidValue;
    static_assert(sizeof(seg_table) <= 4096, "the table fits the kernels' arguments");
    const hipStream_t st = (hipStream_t)s;
    seg_table t = {};
    t.mu = mu;
    t.nesterov = nesterov;
    for (int i = 0; i < n; ++i)
        if (!fits(segs[i]))
            return (int)hipErrorInvalidValue;
    int kinds[kMost];
    kinds_of(segs, n, kinds);
    for (int kind = 0; kind < KINDS; ++kind) {
        t.n = 0;
        for (int i = 0; i < n; ++i)
            if (kinds[i] == kind)
                t.seg[t.n++] = segs[i];
        if (!t.n)
            continue;
        const dim3 grid((unsigned)t.n), block(1024);
        if (kind == SMALL64)
            hipLaunchKernelGGL(k_ns_small<64>, grid, block, 0, st, t, steps);
        else if (kind == SMALL256)
            hipLaunchKernelGGL(k_ns_small<kSmallN>, grid, block, 0, st, t, steps);
        else if (kind == THIN16_FINE)
            hipLaunchKernelGGL((k_ns_thin<1, 1>), grid, block, 0, st, t, steps);
        else if (kind == THIN16)
            hipLaunchKernelGGL((k_ns_thin<1, 4>), grid, block, 0, st, t, steps);
        else if (kind == THIN16_LONG)
            hipLaunchKernelGGL((k_ns_thin<1, 16>), grid, block, 0, st, t, steps);
        else if (kind == THIN32)
            hipLaunchKernelGGL((k_ns_thin<2, 2>), grid, block, 0, st, t, steps);
        else
            hipLaunchKernelGGL((k_ns_thin<2, 8>), grid, block, 0, st, t, steps);
        if (const int rc = (int)hipGetLastError())
            return rc;
    }
    t.n = 0;
    for (int i = 0; i < n; ++i)
        if (kinds[i] == LARGE) {
            t.seg[t.n] = segs[i];
            shape(segs[i], &t.p[t.n++]);
        }
    if (!(n = t.n))
        return 0;
    order(t.p, t.seg, n);
    places(t.p, n, (char *)ws, &t.partial);
    int blocks = number(t, [](const ns_prob &p) { return p.parts; });
    hipLaunchKernelGGL(k_ns_size, dim3((unsigned)blocks), dim3(256), 0, st, t);
    if (const int rc = (int)hipGetLastError())
        return rc;
    blocks = number(t, [](const ns_prob &p) { return p.mp / 64 * (p.np / 64); });
    hipLaunchKernelGGL(k_ns_start, dim3((unsigned)blocks), dim3(256), 0, st, t);
    if (const int rc = (int)hipGetLastError())
        return rc;
    ns_table q = {};
    q.n = n;
    q.partial = t.partial;
    for (int i = 0; i < n; ++i)
        q.p[i] = t.p[i];
    for (int k = 0; k < steps; ++k) {
        int rc = product<NS_S>(q, st);
        rc = rc ? rc : product<NS_B>(q, st);
        if (rc)
            return rc;
        if (k + 1 < steps) {
            if ((rc = product<NS_X>(q, st)))
                return rc;
            for (int i = 0; i < n; ++i) {
                uint16_t *const x = q.p[i].x;
                q.p[i].x = q.p[i].to;
                q.p[i].to = x;
            }
        }
    }
    for (int i = 0; i < n; ++i)
        t.p[i] = q.p[i];
    return product<NS_LAST>(t, st);
}
