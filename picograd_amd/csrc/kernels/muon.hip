// Orthogonal factors by Newton-Schulz products, and the optimiser step made of
// them, for a list of matrices at once.
//
//   u = g, or with momentum m <- mu m + g and u = m (nesterov: g + mu m)
//   X = u / ||u||_F, of the shorter side m as rows (a tall u transposed)
//   `steps` times: S = X X^T, B = b S + c S S, X <- a X + B X
//   out = X, or W <- decay W - step X
//
// The singular values s of X follow s <- a s + b s^3 + c s^5; with (a, b, c) =
// (3.4445, -4.7750, 2.0315) all but the smallest come to 0.7 .. 1.2 in five steps,
// and none passes 1.21, so no entry of X, S or B passes 2.9.
//
// An error in an early X grows as the small singular values do, by up to a a
// step, so f32 is held throughout: X, S and B are kept as two f16 pieces each,
// high and low (22 to 23 bits), times 4096 to keep the low ones from the f16
// subnormals, and a product is three on the f16 matrix units, hh + hl + lh, in
// f32 sums.  Against 64 bits the result is as near as f32 products' (2.8e-6
// against 2.5e-6 of 512 x 512 with singular values over 3.5 decades).  a X is
// added apart from B X: a on the diagonal of B would round it with each entry
// and triples the error.
//
// S and S S are symmetric: tiles below the diagonal, each written twice.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include <type_traits>

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
struct ns_table {
    int n;
    int first[kMost + 1]; // blocks
    ns_prob p[kMost];
};
struct seg_table {
    int n;
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

__device__ __forceinline__ float grad_at(const pgk_muon_seg &s, size_t i)
{
    if (s.g_dtype == 1)
        return (float)((const _Float16 *)s.g)[i];
    if (s.g_dtype == 2)
        return (float)((const __bf16 *)s.g)[i];
    const float g = ((const float *)s.g)[i];
    return s.gclip ? g * s.gmul * s.ginv : g;
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
    for (size_t i = begin + tid; i < end; i += 256) {
        float u = grad_at(s, i);
        if (s.m) {
            const float g = u, m = t.mu * s.m[i] + g;
            s.m[i] = m;
            u = t.nesterov ? g + t.mu * m : m;
        }
        sum += (double)u * (double)u;
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
    const int c = tid & 63;
#pragma unroll 4
    for (int r = tid >> 6; r < 64; r += 4) {
        // row and column of u
        const int row = (tall ? j0 : i0) + r, col = (tall ? i0 : j0) + c;
        float x = 0.0f;
        if ((size_t)row < s.rows && (size_t)col < s.cols) {
            const size_t i = (size_t)row * s.cols + col;
            float u;
            if (s.m)
                u = t.nesterov ? grad_at(s, i) + t.mu * s.m[i] : s.m[i];
            else
                u = grad_at(s, i);
            x = (float)((double)u * scale);
        }
        tile[tall ? c : r][tall ? r : c] = x;
    }
    __syncthreads();
    const size_t plane = (size_t)p.mp * p.np;
#pragma unroll
    for (int r = tid >> 4; r < 64; r += 16) {
        const int c4 = (tid & 15) * 4;
        uint16_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            pieces(tile[r][c4 + e], h[e], l[e]);
        uint16_t *const d = p.x + (size_t)(i0 + r) * p.np + j0 + c4;
        *(uint2 *)d = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
        *(uint2 *)(d + plane) = make_uint2(l[0] | (uint32_t)l[1] << 16, l[2] | (uint32_t)l[3] << 16);
    }
}

__device__ __forceinline__ void load4(const uint16_t *p, size_t plane, float (&v)[4])
{
    const uint2 h = *(const uint2 *)p, l = *(const uint2 *)(p + plane);
    v[0] = whole((uint16_t)h.x, (uint16_t)l.x);
    v[1] = whole((uint16_t)(h.x >> 16), (uint16_t)(l.x >> 16));
    v[2] = whole((uint16_t)h.y, (uint16_t)l.y);
    v[3] = whole((uint16_t)(h.y >> 16), (uint16_t)(l.y >> 16));
}
__device__ __forceinline__ void store4(uint16_t *p, size_t plane, const f32x4 &v)
{
    uint16_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        pieces(v[e], h[e], l[e]);
    *(uint2 *)p = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    *(uint2 *)(p + plane) = make_uint2(l[0] | (uint32_t)l[1] << 16, l[2] | (uint32_t)l[3] << 16);
}

// four neighbours of the result, X times kUnit, at element i of the matrix
__device__ __forceinline__ void finish4(const pgk_muon_seg &s, size_t i, const f32x4 &x, int n)
{
    float o[4];
    if (s.w) {
        const float step = s.step / kUnit;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) {
                o[e] = s.decay * s.w[i + e] - step * x[e];
                s.w[i + e] = o[e];
                if (s.shadow) {
                    const size_t j = i + e;
                    s.shadow[s.shadow_cols ? j / s.shadow_cols * s.shadow_ld + j % s.shadow_cols : j] =
                        to16(s.shadow_dtype, o[e]);
                }
            }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) {
            const float v = x[e] / kUnit;
            if (s.out_dtype == 0)
                ((float *)s.out)[i + e] = v;
            else
                ((uint16_t *)s.out)[i + e] = to16(s.out_dtype, v);
        }
}

enum { NS_S = 0, NS_B = 1, NS_X = 2 };

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

// One product for every matrix: S, B or the next X.
template <class CF, int WHAT>
__global__ void __launch_bounds__(CF::NT, 1) k_ns_product(ns_table t)
{
    __shared__ uint4 smem[CF::LDS_U4];
    LDS uint4 *const lds = (LDS uint4 *)smem;
    const int pid = xcd_tile((int)blockIdx.x, (int)gridDim.x);
    const ns_prob &p = t.p[which(t, pid)];
    const int at = pid - t.first[which(t, pid)];
    const size_t px = (size_t)p.mp * p.np, ps = (size_t)p.mp * p.mp;
    f32x16 acc[CF::FM][CF::FN];
    if constexpr (WHAT == NS_X) {
        const int tiles_m = (p.mp + CF::BM - 1) / CF::BM, tiles_n = (p.np + CF::BN - 1) / CF::BN;
        const int per_group = 8 * tiles_n, group = at / per_group, first = group * 8;
        const int gsz = tiles_m - first < 8 ? tiles_m - first : 8, in = at - group * per_group;
        const int m0 = (first + in % gsz) * CF::BM, n0 = in / gsz * CF::BN;
        piece_loop<CF>({p.b, (size_t)p.mp, ps, p.mp}, {p.x, (size_t)p.np, px, p.np}, p.mp, m0, n0, lds, acc);
        piece_out<CF, f32x4>(acc, m0, n0, p.mp, p.np, lds, false, [&](int row, int col, f32x4 &v, bool) {
            float x[4];
            load4(p.x + (size_t)row * p.np + col, px, x);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = kA * x[e] + v[e] * (1.0f / kUnit);
            store4(p.to + (size_t)row * p.np + col, px, v);
        });
    } else {
        int r, c;
        triangle(at, r, c);
        const int m0 = r * CF::BM, n0 = c * CF::BN;
        if constexpr (WHAT == NS_S)
            piece_loop<CF>({p.x, (size_t)p.np, px, p.mp}, {p.x, (size_t)p.np, px, p.mp}, p.np, m0, n0, lds, acc);
        else
            piece_loop<CF>({p.s, (size_t)p.mp, ps, p.mp}, {p.s, (size_t)p.mp, ps, p.mp}, p.mp, m0, n0, lds, acc);
        uint16_t *const to = WHAT == NS_S ? p.s : p.b;
        piece_out<CF, f32x4>(acc, m0, n0, p.mp, p.mp, lds, r != c, [&](int row, int col, f32x4 &v, bool mirror) {
            if (mirror) {
                store4(to + (size_t)col * p.mp + row, ps, v);
                return;
            }
            v *= 1.0f / kUnit;
            if constexpr (WHAT == NS_B) {
                float x[4];
                load4(p.s + (size_t)row * p.mp + col, ps, x);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = kB * x[e] + kC * v[e];
            }
            store4(to + (size_t)row * p.mp + col, ps, v);
        });
    }
}

// The last X, straight to where it goes.
template <class CF>
__global__ void __launch_bounds__(CF::NT, 1) k_ns_last(seg_table t)
{
    __shared__ uint4 smem[CF::LDS_U4];
    LDS uint4 *const lds = (LDS uint4 *)smem;
    const int pid = xcd_tile((int)blockIdx.x, (int)gridDim.x), k = which(t, pid), at = pid - t.first[k];
    const ns_prob &p = t.p[k];
    const pgk_muon_seg &s = t.seg[k];
    const size_t px = (size_t)p.mp * p.np, ps = (size_t)p.mp * p.mp;
    const int tiles_m = (p.mp + CF::BM - 1) / CF::BM, tiles_n = (p.np + CF::BN - 1) / CF::BN;
    const int per_group = 8 * tiles_n, group = at / per_group, first = group * 8;
    const int gsz = tiles_m - first < 8 ? tiles_m - first : 8, in = at - group * per_group;
    const int m0 = (first + in % gsz) * CF::BM, n0 = in / gsz * CF::BN;
    const bool tall = s.rows > s.cols;
    f32x16 acc[CF::FM][CF::FN];
    piece_loop<CF>({p.b, (size_t)p.mp, ps, p.mp}, {p.x, (size_t)p.np, px, p.np}, p.mp, m0, n0, lds, acc);
    piece_out<CF, f32x4>(acc, m0, n0, p.mp, p.np, lds, tall, [&](int row, int col, f32x4 &v, bool mirror) {
        if (!mirror) {
            float x[4];
            load4(p.x + (size_t)row * p.np + col, px, x);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = kA * x[e] + v[e] * (1.0f / kUnit);
        }
        if (mirror != tall || row >= p.m || col >= p.n)
            return;
        const int left = tall ? p.m - row : p.n - col;
        finish4(s, tall ? (size_t)col * p.m + row : (size_t)row * p.n + col, v, left < 4 ? left : 4);
    });
}

// ---------------------------------------------------------------- launches

template <bool TB>
using T128 = pcfg<f32x16, 2, 128, 128, 2, 2, TB, 32, 2>;
template <bool TB>
using T64 = pcfg<f32x16, 2, 64, 64, 2, 2, TB, 32, 2>;

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
size_t bytes_of(const ns_prob &p)
{
    return ((size_t)p.mp * p.np * 2 + (size_t)p.mp * p.mp * 2) * 4 + kMostParts * sizeof(double);
}

// tiles of a side: below the diagonal, or all of X
template <class CF>
int tiles(const ns_prob &p, bool sym)
{
    const int r = (p.mp + CF::BM - 1) / CF::BM;
    return sym ? r * (r + 1) / 2 : r * ((p.np + CF::BN - 1) / CF::BN);
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

template <class TAB, template <bool> class CF, bool TB>
int total(TAB &t, bool sym)
{
    return number(t, [&](const ns_prob &p) { return tiles<CF<TB>>(p, sym); });
}

template <int WHAT>
int product(ns_table &t, hipStream_t st)
{
    constexpr bool TB = WHAT == NS_X, sym = !TB;
    const int big = total<ns_table, T128, TB>(t, sym);
    if (big >= 256) {
        hipLaunchKernelGGL((k_ns_product<T128<TB>, WHAT>), dim3((unsigned)big), dim3(T128<TB>::NT), 0, st, t);
    } else {
        const int n = total<ns_table, T64, TB>(t, sym);
        hipLaunchKernelGGL((k_ns_product<T64<TB>, WHAT>), dim3((unsigned)n), dim3(T64<TB>::NT), 0, st, t);
    }
    return (int)hipGetLastError();
}

int last(seg_table &t, hipStream_t st)
{
    const int big = total<seg_table, T128, true>(t, false);
    if (big >= 256) {
        hipLaunchKernelGGL((k_ns_last<T128<true>>), dim3((unsigned)big), dim3(T128<true>::NT), 0, st, t);
    } else {
        const int n = total<seg_table, T64, true>(t, false);
        hipLaunchKernelGGL((k_ns_last<T64<true>>), dim3((unsigned)n), dim3(T64<true>::NT), 0, st, t);
    }
    return (int)hipGetLastError();
}

bool fits(const pgk_muon_seg &s)
{
    return s.rows && s.cols && s.rows <= PGK_MUON_MAX_SIDE && s.cols <= PGK_MUON_MAX_SIDE;
}

} // namespace

extern "C" size_t pgk_muon_workspace(const pgk_muon_seg *segs, int n)
{
    size_t all = 0;
    for (int i = 0; i < n; ++i) {
        ns_prob p;
        shape(segs[i], &p);
        all += bytes_of(p);
    }
    return all;
}

extern "C" int pgk_muon(const pgk_muon_seg *segs, int n, float mu, int nesterov, int steps, void *ws, pgk_stream s)
{
    if (n < 1 || n > kMost || steps < 1)
        return (int)hipErrorInvalidValue;
    static_assert(sizeof(seg_table) <= 4096, "the table fits the kernels' arguments");
    const hipStream_t st = (hipStream_t)s;
    seg_table t = {};
    t.n = n;
    t.mu = mu;
    t.nesterov = nesterov;
    char *at = (char *)ws;
    for (int i = 0; i < n; ++i) {
        if (!fits(segs[i]))
            return (int)hipErrorInvalidValue;
        t.seg[i] = segs[i];
        ns_prob &p = t.p[i];
        shape(segs[i], &p);
        const size_t px = (size_t)p.mp * p.np * 4, ps = (size_t)p.mp * p.mp * 4;
        p.x = (uint16_t *)at;
        p.to = (uint16_t *)(at + px);
        p.s = (uint16_t *)(at + 2 * px);
        p.b = (uint16_t *)(at + 2 * px + ps);
        p.part = (double *)(at + 2 * px + 2 * ps);
        at += bytes_of(p);
    }
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
    return last(t, st);
}
