// Gated feed-forward layer: h = act(g) u over z = x W + b = [g | u] in one launch,
// and the backward of the gate (the two products of the layer's backward are
// ordinary GEMMs over [dg | du]).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "convert16.h"
#include "gate_act.h"
#include "gemm_tile.h"
#include "launch.h"

namespace {

// ---------------------------------------------------------------- operands

// Two matrices of 16-bit values with their rows padded by zeros to whole 16-byte
// pieces, in one launch: eight values a thread, a whole piece as one load at
// whatever address it has, the last piece of a row one by one.
struct pad_job {
    const uint16_t *src;
    uint16_t *dst;
    size_t rows, cols, rows_pad, cols8; // cols8: pieces of a padded row
};
__global__ void __launch_bounds__(256) k_gated_pad(pad_job a, pad_job b, size_t na, size_t n)
{
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const bool second = i >= na;
        const pad_job &j = second ? b : a;
        const size_t k = second ? i - na : i, r = k / j.cols8, c = (k - r * j.cols8) * 8;
        const uint16_t *p = j.src + r * j.cols + c;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (r < j.rows && c + 8 <= j.cols) {
            __builtin_memcpy(&q, p, sizeof(q));
        } else if (r < j.rows) {
            uint16_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = c + e < j.cols ? p[e] : (uint16_t)0;
            __builtin_memcpy(&q, v, sizeof(q));
        }
        ((uint4 *)j.dst)[k] = q;
    }
}

// ---------------------------------------------------------------- forward

// A tile of the product holds columns of Wg beside the same columns of Wu
// (TileGate), so its epilogue has g and u of each output and z need not be
// read back; z itself is written only for a backward.  Tiles and k-loops are
// the 16-bit GEMM's, and what bounds it is what bounds that: in rounds of full
// tiles the matrix units (4096 x 4096 x 8192 in bf16 509 us, 1.08 PFLOP/s, z's 268 MB
// among them), with one round the loads' latency and the epilogue (512 x 1024 x
// 4096 17 us, 0.5 PFLOP/s).
template <class CF>
__global__ void __launch_bounds__(CF::NT, 1) k_gated(gemm_kargs g)
{
    __shared__ uint4 smem[CF::LDS_U4];
    gemm16_block<CF>(g, (int)blockIdx.x, (int)gridDim.x, true, 0, (LDS uint4 *)smem);
}
template <class CF>
__global__ void __launch_bounds__(CF::NT, CF::KG == 4 ? 2 : 1) k_gated_ks(gemm_kargs g)
{
    __shared__ uint4 smem[CF::LDS_U4];
    ks_block<CF>(g, 1, (int)blockIdx.x, (int)gridDim.x, true, 0, (LDS uint4 *)smem);
}

// Up to 16 rows: a block owns 16 outputs, whose 32 columns of W it streams past
// once, its four waves splitting the reduction, each with a ring of two 64-deep
// chunks of its own and no block barrier until the waves' partial tiles (16 x 16,
// one of g and one of u) are added through LDS in wave order.  Bound by W's
// stream; the block being small, the chip fills at few outputs.  One row, k x f,
// this kernel against the tiles below: 1024 x 1024 4.5 : 6.1 us, 1024 x 4096
// 7.2 : 8.4, 4096 x 4096 18.7 : 20.9 (3.6 TB/s of W); 4096 x 8192, whose
// blocks come in two rounds, 50.4 : 35.5, so it is taken up to
// 256 blocks.  Eight waves and three chunks: 8.0, 19.2 and 52.3 us.
typedef float f32x4m __attribute__((ext_vector_type(4)));
template <bool F16>
__device__ __forceinline__ f32x4m mfma16(const uint4 &a, const uint4 &b, const f32x4m &c)
{
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
}
constexpr int kFewWaves = 4, kFewStages = 2, kFewK = 64;
constexpr int kFewBlocks = 256;
constexpr int kFewA = 16 * kFewK / 8, kFewB = kFewK * 32 / 8; // uint4 of one A and one B stage

template <bool F16>
__global__ void __launch_bounds__(kFewWaves * 64, 2) k_gated_few(gemm_kargs g)
{
    __shared__ uint4 smem[kFewWaves * kFewStages * (kFewA + kFewB)];
    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // neighbouring blocks share each 128-byte line of a row: on one XCD
    const int n0 = xcd_tile((int)blockIdx.x, (int)gridDim.x) * 16;
    LDS uint4 *const ring = (LDS uint4 *)smem + wave * kFewStages * (kFewA + kFewB);
    using TK = TileK<16, 64, kFewK>;
    static_assert(TK::NQ == 2 && kFewB == 256, "two loads of A and four of B per stage");
    constexpr int LPT = 6;
    const int nct = (g.K + kFewK - 1) / kFewK, nc = nct > wave ? (nct - wave + kFewWaves - 1) / kFewWaves : 0;
    // this wave's chunk c (chunk c * waves + wave of the reduction) into stage
    // st; k at or past K reads the zero page
    auto load = [&](int c, int st) {
        const int ch = c * kFewWaves + wave, k0 = ch < nct ? ch * kFewK : g.K;
        LDS uint4 *sa = ring + st * (kFewA + kFewB), *sb = sa + kFewA;
#pragma unroll
        for (int q = 0; q < 4; ++q) { // [64 k][16 of g, 16 of u]: four 16-byte chunks per k row
            const int slot = q * 64 + lane, k = slot >> 2, half = slot >> 1 & 1;
            int col = n0 + (slot & 1) * 8;
            col = (col < g.b_extent ? col : g.b_extent - 8) + half * g.b_extent;
            const void *src = k0 + k < g.K ? (const void *)(g.B + (size_t)(k0 + k) * g.ldb + col) : (const void *)&g_zero16;
            dma16(src, sb + q * 64);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
            TK::load_q(q, g.A, g.lda, 0, g.a_extent, k0, g.K, sa, lane);
    };
    const int grp = lane >> 4, q16 = lane & 15;
    f32x4m acc[2] = {};
    if (nc > 0) {
#pragma unroll
        for (int s = 0; s < kFewStages; ++s)
            load(s, s);
        int st = 0;
        for (int c = 0; c < nc; ++c) {
            const LDS uint4 *sa = ring + st * (kFewA + kFewB), *sb = sa + kFewA;
            // chunk c landed (the newest kFewStages - 1 chunks may be in flight)
            __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((kFewStages - 1) * LPT));
            __asm__ volatile("" ::: "memory");
            // 16-lane group grp holds k = 32 s + 8 grp .. + 7 of row (A) or
            // column (B) lane % 16; B from two transposing reads
            uint4 fa[2], fb[2][2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const u32x4 v = ((const LDS u32x4 *)sa)[q16 * TK::CH + TK::swz(4 * s + grp, q16)];
                fa[s] = __builtin_bit_cast(uint4, v);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint2 h2[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int k = 32 * s + 8 * grp + 4 * h + (q16 >> 2);
                        h2[h] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                              (LDS v4s *)((const LDS char *)sb + k * 64 + t * 32 + (q16 & 3) * 8)));
                    }
                    fb[s][t] = make_uint4(h2[0].x, h2[0].y, h2[1].x, h2[1].y);
                }
            }
            // the stage's reads are done before its refill
            __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(63));
            __asm__ volatile("" ::: "memory");
            load(c + kFewStages, st);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    acc[t] = mfma16<F16>(fa[s], fb[s][t], acc[t]);
            st = st + 1 == kFewStages ? 0 : st + 1;
        }
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0));
    }
    __syncthreads(); // the rings are done: the waves' partials through LDS, added in wave order
    constexpr int RP = 36;
    LDS float *part = (LDS float *)smem;
    static_assert(kFewWaves * 16 * RP * 4 <= (int)sizeof(smem), "partials fit the rings");
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) // lane holds column lane % 16 of rows 4 (lane / 16) + e
            part[(wave * 16 + 4 * grp + e) * RP + t * 16 + q16] = acc[t][e];
    __syncthreads();
    const int row = (int)threadIdx.x >> 2, c4 = ((int)threadIdx.x & 3) * 4;
    if (row < 16 && row < g.M && n0 + c4 < g.N) {
        f32x4 gv = {0.0f, 0.0f, 0.0f, 0.0f}, uv = gv;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) {
            gv += *(const LDS f32x4 *)(part + (w * 16 + row) * RP + c4);
            uv += *(const LDS f32x4 *)(part + (w * 16 + row) * RP + 16 + c4);
        }
        if (gate_whole(g.epi, g.C, g.N)) {
            gate_store4(g.epi, g.C, g.N, row, n0 + c4, gv, uv);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (n0 + c4 + q < g.N)
                    gate_store1(g.epi, g.C, g.N, row, n0 + c4 + q, gv[q], uv[q]);
        }
    }
}

template <class CF>
int launch_tiles(gemm_kargs g, hipStream_t s)
{
    g.tiles_m = (g.M + CF::BM - 1) / CF::BM, g.tiles_n = (g.N + CF::BN / 2 - 1) / (CF::BN / 2);
    hipLaunchKernelGGL(k_gated<CF>, dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(CF::NT), 0, s, g);
    return (int)hipGetLastError();
}
template <class CF>
int launch_split(gemm_kargs g, hipStream_t s)
{
    g.tiles_m = (g.M + CF::TM - 1) / CF::TM, g.tiles_n = (g.N + CF::TN / 2 - 1) / (CF::TN / 2);
    hipLaunchKernelGGL(k_gated_ks<CF>, dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(CF::NT), 0, s, g);
    return (int)hipGetLastError();
}

template <bool F16>
int launch_forward(int tile, const gemm_kargs &g, hipStream_t s)
{
    if (g.M <= 16 && (g.N + 15) / 16 <= kFewBlocks) {
        hipLaunchKernelGGL(k_gated_few<F16>, dim3((unsigned)((g.N + 15) / 16)), dim3(kFewWaves * 64), 0, s, g);
        return (int)hipGetLastError();
    }
    switch (tile) {
    // four stages of 32 rather than the plain product's two of 64: 512 x 1024 x
    // 4096 18.6 : 19.8 us, 200 x 4096 x 4096 35.9 : 43.4
    case 1: return launch_tiles<gcfg<128, 128, 2, 2, false, true, F16, true, 32, 4, true>>(g, s);
    case 2: return launch_tiles<gcfg<256, 256, 2, 4, false, true, F16, true, 32, 4, true>>(g, s);
    case 3: return launch_tiles<gcfg<128, 256, 2, 4, false, true, F16, true, 32, 4, true>>(g, s);
    case 5: return launch_split<kscfg<32, 32, 8, 64, 2, false, true, F16, true>>(g, s);
    case 6: return launch_split<kscfg<32, 64, 8, 32, 3, false, true, F16, true>>(g, s);
    case 7: return launch_split<kscfg<64, 64, 4, 32, 2, false, true, F16, true>>(g, s);
    default: return launch_split<kscfg<64, 64, 8, 32, 2, false, true, F16, true>>(g, s);
    }
}

// ---------------------------------------------------------------- backward

// The gate's backward over a strip of 256 columns of f and a run of rows per
// block: its four waves take every fourth row each, four neighbouring columns a
// lane, and keep the strip's column sums, joined through LDS in wave order into
// the block's row of part.  dz is rounded to the operands' 16 bits, in which both
// products take it (in f32 the matrix units run at an eighth of the rate, and a dz
// split into two halves doubles the products); the sums take it before.  Bound by the stream of z and dh in
// and dz out (4096 x 8192 in bf16: 470 MB in 90 us, 5.2 TB/s).  A piece of four is one load at
// whatever address an odd f gives it (1023 x 2049: one value a lane took 11 us).
constexpr int kBwdV = 4;
template <bool WHOLE, class T>
__device__ __forceinline__ void load_piece(const T *p, size_t left, float *v)
{
    typedef T tv __attribute__((ext_vector_type(kBwdV), aligned(sizeof(T))));
    if constexpr (WHOLE) {
        const tv q = __builtin_nontemporal_load((const tv *)p); // read once
#pragma unroll
        for (int i = 0; i < kBwdV; ++i)
            v[i] = (float)q[i];
    } else {
#pragma unroll
        for (int i = 0; i < kBwdV; ++i)
            v[i] = i < left ? (float)p[i] : 0.0f;
    }
}

template <int ACT, class D>
__global__ void __launch_bounds__(256)
    k_gated_bwd(const D *__restrict__ dh, const float *__restrict__ z, size_t m, size_t f, size_t f8,
                uint16_t *__restrict__ dz, int dtype, float *__restrict__ part, int rows)
{
    constexpr int V = kBwdV;
    __shared__ float sums[4][2][64 * V];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const size_t c = ((size_t)blockIdx.x * 64 + lane) * V;
    const size_t r0 = (size_t)blockIdx.y * rows, r1 = r0 + rows < m ? r0 + rows : m;
    float sg[V] = {}, su[V] = {};
    // the rows of a lane whose piece lies within f, or of f's last columns (past
    // them zeros, whose grads are zeros)
    auto run = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        const size_t left = f - c;
#pragma unroll WHOLE ? 4 : 1
        for (size_t r = r0 + wave; r < r1; r += 4) {
            float d[V], g[V], u[V], dg[V], du[V];
            load_piece<WHOLE>(dh + r * f + c, left, d);
            load_piece<WHOLE>(z + r * 2 * f + c, left, g);
            load_piece<WHOLE>(z + r * 2 * f + f + c, left, u);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float da;
                const float a = gate_fd<ACT>(g[i], da);
                dg[i] = d[i] * u[i] * da;
                du[i] = d[i] * a;
                sg[i] += dg[i];
                su[i] += du[i];
            }
            uint16_t *p = dz + r * 2 * f8 + c;
            *(uint2 *)p = make_uint2(to16x2(dtype, dg[0], dg[1]), to16x2(dtype, dg[2], dg[3]));
            *(uint2 *)(p + f8) = make_uint2(to16x2(dtype, du[0], du[1]), to16x2(dtype, du[2], du[3]));
        }
    };
    if (c + V <= f)
        run(std::true_type{});
    else if (c < f)
        run(std::false_type{});
    else if (c < f8) // the zeros past an odd f
        for (size_t r = r0 + wave; r < r1; r += 4)
            *(uint2 *)(dz + r * 2 * f8 + c) = *(uint2 *)(dz + r * 2 * f8 + f8 + c) = make_uint2(0, 0);
    if (!part)
        return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        sums[wave][0][lane * V + i] = sg[i];
        sums[wave][1][lane * V + i] = su[i];
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < 2 * 64 * V; i += 256) {
        const int half = i / (64 * V), j = i % (64 * V);
        const size_t col = (size_t)blockIdx.x * 64 * V + j;
        if (col < f)
            part[(size_t)blockIdx.y * 2 * f + half * f + col] =
                sums[0][half][j] + sums[1][half][j] + sums[2][half][j] + sums[3][half][j];
    }
}

// The blocks of rows: enough to fill the chip, at most 64 where they leave
// partial column sums, which one more launch adds one after the other.
struct bwd_plan {
    unsigned gx, gy;
    int rows;
};
bwd_plan plan_bwd(size_t m, size_t f, bool sums)
{
    const size_t gx = (f + 64 * kBwdV - 1) / (64 * kBwdV);
    size_t gy = (sums ? 2048 : 4096) / gx;
    gy = gy < 1 ? 1 : sums && gy > 64 ? 64 : gy > 16384 ? 16384 : gy;
    size_t rows = (m + gy - 1) / gy;
    rows = (rows + 3) / 4 * 4;
    return {(unsigned)gx, (unsigned)((m + rows - 1) / rows), (int)rows};
}

struct bwd_args {
    const void *dh;
    const float *z;
    size_t m, f;
    uint16_t *dz;
    int dtype;
    float *part;
};
template <int ACT, class D>
void launch_bwd(const bwd_args &a, const bwd_plan &p, hipStream_t s)
{
    hipLaunchKernelGGL((k_gated_bwd<ACT, D>), dim3(p.gx, p.gy), dim3(256), 0, s, (const D *)a.dh, a.z, a.m, a.f,
                       (a.f + 7) & ~(size_t)7, a.dz, a.dtype, a.part, p.rows);
}
template <int ACT>
void launch_bwd(const bwd_args &a, int dh_dtype, const bwd_plan &p, hipStream_t s)
{
    dh_dtype == 0 ? launch_bwd<ACT, float>(a, p, s)
                  : dh_dtype == 1 ? launch_bwd<ACT, _Float16>(a, p, s) : launch_bwd<ACT, __bf16>(a, p, s);
}

// Few rows (pgk_gated_few_grads_ok): dz stays in f32 (rounded to 16 bits it is half of the error of so
// few sums) and both grads are one launch over the matrices where they lie.
// One thread per column of f: dz and, over the rows in turn, db.
template <int ACT, class D>
__global__ void __launch_bounds__(64)
    k_gated_few_dz(const D *__restrict__ dh, const float *__restrict__ z, int m, size_t f, float *__restrict__ dz,
                   float *__restrict__ db, int db_beta)
{
    const size_t c = (size_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= f)
        return;
    float sg = 0.0f, su = 0.0f;
#pragma unroll 4
    for (int r = 0; r < m; ++r) {
        const float d = (float)dh[r * f + c], g = z[r * 2 * f + c], u = z[r * 2 * f + f + c];
        float da;
        const float a = gate_fd<ACT>(g, da), dg = d * u * da, du = d * a;
        dz[r * 2 * f + c] = dg;
        dz[r * 2 * f + f + c] = du;
        sg += dg;
        su += du;
    }
    if (db) {
        db[c] = db_beta ? db[c] + sg : sg;
        db[f + c] = db_beta ? db[f + c] + su : su;
    }
}

// dx[:, k] = dz W[k, :] and dW[k, :] = x[:, k] dz for 16 rows k of W and a part of
// its columns per block, by 16 x 16 x 4 products in f32 (W and x widened).  A wave
// takes every eighth piece of 64 columns: W's piece once, in the order of dx's
// product (lane l: row l % 16, columns 8 (l / 16) .. + 7), dz in that order and again
// in dW's (rows 4 s + l / 16, columns 4 (l % 16) .. + 3) from the caches; the waves'
// sums of dx are joined through LDS in wave order, the parts' in one more small
// launch.  Bound by the latency of a piece's loads, then by dz from the caches
// (loads a piece ahead cost more in registers than they hid, two and four row
// groups a wave gained at 4096 x 8192 alone).
constexpr int kFgWaves = 8;
struct few_grads {
    const uint16_t *x, *w;
    size_t ldx, ldw, half; // of W: a row, and from g's columns to u's in it
    const float *dz;
    int m;
    size_t k, f, first; // the launch's first 16 rows of W
    void *dx, *dw; // NULL: not wanted
    int dx_dtype, dw_dtype, dx_beta, dw_beta;
    float *part; // [parts, m, k] of dx where the columns are in more than one part
};

// the parts of the columns: a block for each CU, a piece a wave at least
unsigned few_parts(size_t k, size_t f)
{
    const size_t rows = (k + 15) / 16, pieces = 2 * ((f + 63) / 64), most = pieces / kFgWaves;
    const size_t want = 256 / rows, n = want < most ? want : most;
    return n > 1 ? (unsigned)n : 1;
}

template <bool F16>
__device__ __forceinline__ float widened(uint32_t bits)
{
    if constexpr (F16)
        return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
    else
        return __builtin_bit_cast(float, bits << 16);
}

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4h __attribute__((ext_vector_type(4), aligned(2)));

// N values at p, those at or past `left` and of an absent row as zeros (p is then
// another row's)
template <int N>
__device__ __forceinline__ void load_f32(const float *p, long left, bool row, float *v)
{
    if (left >= N) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4u q = *(const f32x4u *)(p + i);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[i + e] = row ? q[e] : 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = row && i < left ? p[i] : 0.0f;
    }
}

// v as the output type at p[i], or added to an f32 there
__device__ __forceinline__ void put(void *p, int dtype, int beta, size_t i, float v)
{
    if (dtype == 0) {
        float *const q = (float *)p + i;
        *q = beta ? *q + v : v;
    } else {
        ((uint16_t *)p)[i] = to16(dtype, v);
    }
}

template <bool F16>
__global__ void __launch_bounds__(kFgWaves * 64, 2) k_gated_few_grads(few_grads a)
{
    __shared__ float sums[kFgWaves][16][17];
    const int lane = (int)threadIdx.x & 63, q = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const size_t k0 = (a.first + blockIdx.x) * 16, kr = k0 + q < a.k ? k0 + q : a.k - 1;
    const size_t per = (a.f + 63) / 64, pieces = 2 * per;
    float xv[4]; // x[4 s + l / 16][k0 + l % 16]
#pragma unroll
    for (int s = 0; s < 4; ++s)
        xv[s] = a.dw && 4 * s + grp < a.m ? widened<F16>(a.x[(4 * s + grp) * a.ldx + kr]) : 0.0f;
    f32x4m acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (size_t p = blockIdx.y * kFgWaves + wave; p < pieces; p += (size_t)kFgWaves * gridDim.y) {
        const size_t h = p >= per, c0 = (p - h * per) * 64;
        const float *dz = a.dz + h * a.f + c0;
        const long left = (long)(a.f - c0);
        u32x4 w[2];    // W's row kr at columns 8 grp .. + 7 of both halves
        float da[2][8]; // dz of row q there
        float db[4][4]; // dz of rows 4 s + grp at columns 4 q .. + 3
        if (a.dx) {
            const uint16_t *src = a.w + kr * a.ldw + h * a.half + c0;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int c = 32 * t + 8 * grp;
                if (left - c >= 8) {
                    w[t] = __builtin_bit_cast(u32x4, *(const u32x4h *)(src + c));
                } else {
                    uint16_t e16[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        e16[e] = c + e < left ? src[c + e] : (uint16_t)0;
                    __builtin_memcpy(&w[t], e16, 16);
                }
                load_f32<8>(dz + (size_t)(q < a.m ? q : 0) * 2 * a.f + c, left - c, q < a.m, da[t]);
            }
        }
        if (a.dw)
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (4 * s < a.m) {
                    const int m = 4 * s + grp;
                    load_f32<4>(dz + (size_t)(m < a.m ? m : 0) * 2 * a.f + 4 * q, left - 4 * q, m < a.m, db[s]);
                }
        if (a.dx)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(da[t][e], widened<F16>(w[t][e >> 1] >> 16 * (e & 1) & 0xffffu), acc,
                                                               0, 0, 0);
        if (!a.dw)
            continue;
        f32x4m o[4] = {};
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (4 * s < a.m)
#pragma unroll
                for (int e = 0; e < 4; ++e) // columns 4 q + e of rows k
                    o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[s], db[s][e], o[e], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) { // lane: rows 4 grp + r
            const size_t row = k0 + 4 * grp + r, at = row * 2 * a.f + h * a.f + c0 + 4 * q;
            if (row >= a.k)
                continue;
            const float v[4] = {o[0][r], o[1][r], o[2][r], o[3][r]};
            if (left >= 4 * q + 4 && !a.dw_beta) {
                if (a.dw_dtype == 0) {
                    *(f32x4u *)((float *)a.dw + at) = f32x4u{v[0], v[1], v[2], v[3]};
                } else {
                    typedef uint32_t u32x2h __attribute__((ext_vector_type(2), aligned(2)));
                    *(u32x2h *)((uint16_t *)a.dw + at) = u32x2h{to16x2(a.dw_dtype, v[0], v[1]), to16x2(a.dw_dtype, v[2], v[3])};
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * q + e < left)
                        put(a.dw, a.dw_dtype, a.dw_beta, at + e, v[e]);
            }
        }
    }
    if (!a.dx)
        return;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        sums[wave][4 * grp + r][q] = acc[r]; // row of x, row of W
    __syncthreads();
    const int row = (int)threadIdx.x >> 4, col = (int)threadIdx.x & 15;
    if (row < a.m && k0 + col < a.k) {
        float v = 0.0f;
#pragma unroll
        for (int t = 0; t < kFgWaves; ++t)
            v += sums[t][row][col];
        const size_t at = (size_t)row * a.k + k0 + col;
        if (a.part)
            a.part[(size_t)blockIdx.y * a.m * a.k + at] = v;
        else
            put(a.dx, a.dx_dtype, a.dx_beta, at, v);
    }
}
// the parts of dx, added in their order
__global__ void __launch_bounds__(256) k_gated_few_join(few_grads a, unsigned parts)
{
    const size_t n = (size_t)a.m * a.k, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n)
        return;
    float v = 0.0f;
    for (unsigned t = 0; t < parts; ++t)
        v += a.part[t * n + i];
    put(a.dx, a.dx_dtype, a.dx_beta, i, v);
}

} // namespace

extern "C" int pgk_gated_pad(const uint16_t *x, size_t m, size_t k, uint16_t *x16, const uint16_t *w, size_t f, uint16_t *w16,
                             pgk_stream s)
{
    const size_t k8 = (k + 7) / 8, f8 = (f + 7) / 8;
    const pad_job a = {x, x16, m, k, m, k8}, b = {w, w16, 2 * k, f, 16 * k8, f8};
    const size_t na = x16 ? a.rows_pad * a.cols8 : 0, n = na + (w16 ? b.rows_pad * b.cols8 : 0);
    if (!n)
        return 0;
    const size_t blocks = (n + 255) / 256;
    hipLaunchKernelGGL(k_gated_pad, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, (hipStream_t)s, a, b, na,
                       n);
    return (int)hipGetLastError();
}

extern "C" int pgk_gated_forward(int dtype, int act, size_t m, size_t f, size_t k8, const uint16_t *x, size_t ldx,
                                 const uint16_t *w, size_t f8, const float *bias, float *z, float *h32, uint16_t *h16,
                                 pgk_stream s)
{
    if (!m || !f)
        return 0;
    if (m > 0x7fffffff || f > 0x1fffffff || k8 > 0x7fff0000 || (k8 & 7) || (ldx & 7) || (f8 & 7) || f8 < f || ldx < k8 ||
        ((((uintptr_t)x) | (uintptr_t)w) & 15) || (dtype != 1 && dtype != 2))
        return (int)hipErrorInvalidValue;
    if (((m + 127) / 128) * ((f + 63) / 64) >> 24) // a launch holds under 2^32 threads, a tile has 256
        return (int)hipErrorInvalidValue;
    gemm_kargs g = {};
    g.A = x, g.lda = ldx, g.a_extent = (int)m;
    g.B = w, g.ldb = 2 * f8, g.b_extent = (int)f8;
    g.C = h32, g.ldc = f;
    g.M = (int)m, g.N = (int)f, g.K = g.k_total = (int)k8;
    g.epi.bias = bias, g.epi.act = act, g.epi.z = z, g.epi.c16 = h16, g.epi.dtype16 = dtype, g.epi.skip_out = !h32;
    g.fast_ok = ldx < kFastLd && 2 * f8 < kFastLd;
    const int tile = pgk_gemm16_whole_tile(m, 2 * f, k8);
    return dtype == 1 ? launch_forward<true>(tile, g, (hipStream_t)s) : launch_forward<false>(tile, g, (hipStream_t)s);
}

extern "C" size_t pgk_gated_bwd_workspace(size_t m, size_t f)
{
    if (!m || !f)
        return 0;
    return plan_bwd(m, f, true).gy * 2 * f * sizeof(float);
}

extern "C" int pgk_gated_bwd(int act, const void *dh, int dh_dtype, const float *z, size_t m, size_t f, uint16_t *dz16,
                             int dtype, float *db, int db_beta, void *ws, pgk_stream s)
{
    if (!m || !f)
        return 0;
    if (m > 0x7fffffff || f > 0x1fffffff || (db && !ws) || ((uintptr_t)dz16 & 15) || act < 0 || act > PGK_ACT_SIGMOID)
        return (int)hipErrorInvalidValue;
    const bwd_plan p = plan_bwd(m, f, db != nullptr);
    const bwd_args a = {dh, z, m, f, dz16, dtype, db ? (float *)ws : nullptr};
    hipStream_t st = (hipStream_t)s;
    switch (act) {
    case PGK_ACT_RELU: launch_bwd<PGK_ACT_RELU>(a, dh_dtype, p, st); break;
    case PGK_ACT_GELU: launch_bwd<PGK_ACT_GELU>(a, dh_dtype, p, st); break;
    case PGK_ACT_SILU: launch_bwd<PGK_ACT_SILU>(a, dh_dtype, p, st); break;
    case PGK_ACT_SIGMOID: launch_bwd<PGK_ACT_SIGMOID>(a, dh_dtype, p, st); break;
    default: launch_bwd<PGK_ACT_NONE>(a, dh_dtype, p, st); break;
    }
    const int rc = (int)hipGetLastError();
    if (rc || !db)
        return rc;
    const pgk_colsum_job job = {(const float *)ws, p.gy, 2 * f, db, db_beta};
    return pgk_colsum_run(&job, s);
}

// Against the 16-bit products, us for k x f in bf16 with 1, 4, 16 rows (those:
// 17): 64 x 64 6.1, 6.2, 7.5 (10.5), 64 x 8192 16, 16, 19 (36), 1024 x 4096 20, 21,
// 29 (28), 4096 x 8192 107, 110, 159 (103).  Up to four rows it is taken at the last
// sizes too, for the error of so few sums.
extern "C" int pgk_gated_few_grads_ok(size_t m, size_t k, size_t f)
{
    return m <= 4 || (m <= 16 && (!k || f <= ((size_t)1 << 22) / k));
}

extern "C" size_t pgk_gated_few_grads_workspace(size_t m, size_t k, size_t f)
{
    const unsigned parts = k && f ? few_parts(k, f) : 1;
    return parts > 1 ? parts * m * k * sizeof(float) : 0;
}

namespace {
template <int ACT>
void launch_few_dz(const void *dh, int dh_dtype, const float *z, int m, size_t f, float *dz, float *db, int db_beta, hipStream_t s)
{
    const dim3 grid((unsigned)((f + 63) / 64));
    if (dh_dtype == 0)
        hipLaunchKernelGGL((k_gated_few_dz<ACT, float>), grid, dim3(64), 0, s, (const float *)dh, z, m, f, dz, db, db_beta);
    else if (dh_dtype == 1)
        hipLaunchKernelGGL((k_gated_few_dz<ACT, _Float16>), grid, dim3(64), 0, s, (const _Float16 *)dh, z, m, f, dz, db, db_beta);
    else
        hipLaunchKernelGGL((k_gated_few_dz<ACT, __bf16>), grid, dim3(64), 0, s, (const __bf16 *)dh, z, m, f, dz, db, db_beta);
}
} // namespace

extern "C" int pgk_gated_few_dz(int act, const void *dh, int dh_dtype, const float *z, size_t m, size_t f, float *dz, float *db,
                                int db_beta, pgk_stream s)
{
    if (m > 16 || !f || f > 0x1fffffff)
        return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)s;
    switch (act) {
    case PGK_ACT_RELU: launch_few_dz<PGK_ACT_RELU>(dh, dh_dtype, z, (int)m, f, dz, db, db_beta, st); break;
    case PGK_ACT_GELU: launch_few_dz<PGK_ACT_GELU>(dh, dh_dtype, z, (int)m, f, dz, db, db_beta, st); break;
    case PGK_ACT_SILU: launch_few_dz<PGK_ACT_SILU>(dh, dh_dtype, z, (int)m, f, dz, db, db_beta, st); break;
    case PGK_ACT_SIGMOID: launch_few_dz<PGK_ACT_SIGMOID>(dh, dh_dtype, z, (int)m, f, dz, db, db_beta, st); break;
    default: launch_few_dz<PGK_ACT_NONE>(dh, dh_dtype, z, (int)m, f, dz, db, db_beta, st); break;
    }
    return (int)hipGetLastError();
}

extern "C" int pgk_gated_few_grads(int dtype, const float *dz, size_t m, size_t k, size_t f, const uint16_t *x, size_t ldx,
                                   const uint16_t *w, size_t half, void *dx, int dx_dtype, int dx_beta, void *dw, int dw_dtype,
                                   int dw_beta, void *ws, pgk_stream s)
{
    if (!m || m > 16 || !k || k > 0x3fffffff || !f || f > 0x1fffffff || (dtype != 1 && dtype != 2) || (dx_beta && dx_dtype) ||
        (dw_beta && dw_dtype) || half < f || (dw && ldx < k) ||
        (dx && !ws && few_parts(k, f) > 1))
        return (int)hipErrorInvalidValue;
    few_grads a = {x, w, ldx, 2 * half, half, dz, (int)m, k, f, 0, dx, dw, dx_dtype, dw_dtype, dx_beta, dw_beta,
                   few_parts(k, f) > 1 ? (float *)ws : nullptr};
    // a launch holds under 2^32 threads
    const size_t blocks = (k + 15) / 16, most = (size_t)1 << 22;
    const unsigned parts = few_parts(k, f);
    for (; a.first < blocks; a.first += most) {
        const dim3 grid((unsigned)(blocks - a.first < most ? blocks - a.first : most), parts);
        if (dtype == 1)
            hipLaunchKernelGGL(k_gated_few_grads<true>, grid, dim3(kFgWaves * 64), 0, (hipStream_t)s, a);
        else
            hipLaunchKernelGGL(k_gated_few_grads<false>, grid, dim3(kFgWaves * 64), 0, (hipStream_t)s, a);
    }
    if (dx && parts > 1)
        hipLaunchKernelGGL(k_gated_few_join, dim3((unsigned)((m * k + 255) / 256)), dim3(256), 0, (hipStream_t)s, a, parts);
    return (int)hipGetLastError();
}
