// GEMM kernels for gfx950.
//
// k_gemm16: C[b][i, j] (beta ? += : =) sum_p A(i, p) B(p, j) with f16/bf16
// operands, f32 accumulation in MFMA (v_mfma_f32_32x32x16_{bf16,f16}) and
// f32 output.  Each operand is either "K-contiguous" (its reduction dim is
// contiguous: A(i, p) = a[i * lda + p], B(p, j) = b[j * ldb + p]) or
// "MN-contiguous" (A(i, p) = a[p * lda + i], B(p, j) = b[p * ldb + j]), so
// dgrad (dC . W^T), wgrad (A^T . dC) and the forward product (A . W) all
// read their operands where they lie, with no transposed copies.
//
// Data path, per block tile BM x BN x KB (KB = 32 or 64):
//  - global -> LDS directly (global_load_lds_dwordx4: 64 lanes x 16 bytes
//    per instruction, no staging registers) into an S-stage LDS ring; the
//    next S - 1 k-tiles' loads are in flight while one is computed;
//  - K-contiguous tiles sit in LDS as [rows][64] with 16-byte chunks
//    XOR-swizzled by (r ^ r >> 3) & 7 and reach the MFMA with ds_read_b128;
//    MN-contiguous tiles sit as [64][rows] with chunks swizzled by
//    4 (k & 3) and reach it with ds_read_b64_tr_b16, the gfx950 transposing
//    LDS read (within each 16-lane group, lane i of the result takes element
//    i % 4 of the 8 bytes lane 4p + i / 4 addressed, for slot p);
//  - fragment reads for the next 16-wide k step are issued one per MFMA of
//    the current one, and the k-loop has no branches between two barriers,
//    so each MFMA waits only for its own fragments;
//  - tiles are remapped so the blocks that share operand panels run on one
//    XCD (and its L2), grouped 8 tile-rows at a time.
// A partial last k-tile loads zeros past K: its out-of-range chunks (K % 8
// == 0 for a K-contiguous operand) or k-rows (MN-contiguous) are DMA'd from
// a 16-byte zero page.  Otherwise the host runs the last K % 64 columns as
// one more launch over zero-padded copies (beta = 1).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include <initializer_list>
#include <type_traits>

#include "convert16.h"
#include "gemm_tile.h"
#include "launch.h"
#include "pgmath.h"

namespace {

template <class CF>
__global__ void __launch_bounds__(CF::NT, 1) k_gemm16(gemm_kargs g)
{
    __shared__ uint4 smem[CF::LDS_U4];
    gemm16_block<CF>(g, (int)blockIdx.x, (int)gridDim.x, true, (int)blockIdx.z, (LDS uint4 *)smem);
}

// Two problems in one launch (the dgrad and wgrad of one matmul when each
// alone leaves CUs idle): blocks [0, n1) take problem 1 (tile b % nb1 of
// slice / batch entry b / nb1), the rest problem 2; one LDS ring, sized for
// the larger configuration.  Both configurations have the same thread
// count.  Problem 2's tiles are regrouped by XCD only when n1 % 8 == 0.
template <class C1, class C2>
__global__ void __launch_bounds__(C1::NT, 1) k_gemm16_pair(gemm_kargs g1, gemm_kargs g2, int nb1, int n1, int nb2)
{
    static_assert(C1::NT == C2::NT, "one block size");
    __shared__ uint4 smem[C1::LDS_U4 > C2::LDS_U4 ? C1::LDS_U4 : C2::LDS_U4];
    const int b = (int)blockIdx.x;
    if (b < n1)
        gemm16_block<C1>(g1, b % nb1, nb1, true, b / nb1, (LDS uint4 *)smem);
    else
        gemm16_block<C2>(g2, (b - n1) % nb2, nb2, (n1 & 7) == 0, (b - n1) / nb2, (LDS uint4 *)smem);
}

// Skinny product: C[m, n] (+)= A . B for n <= 16 with B MN-contiguous
// (b[p * ldb + j]), A K-contiguous (TA false: the forward x . W of a narrow
// layer) or MN-contiguous (TA true: a narrow layer's weight grad x^T . dz).
// Such a product streams A once, so split-K's partials and summing launch
// dominated it.  A block owns 16 rows of C (256 blocks for 4096 rows: every
// CU streams) and its eight waves split the reduction into runs of 64-deep
// chunks, each wave with a three-stage ring of its own in LDS (no block
// barrier in the k-loop: a wave waits only on its own loads; two chunks
// ahead measured faster than four).  The 32 x 32 x 16 MFMA holds the 16 rows and 16
// columns in a quarter of its outputs: its other rows and columns read
// duplicates or zeros and are never stored.  The waves' partial products
// are added through LDS in wave order, then each element goes through the
// plain store (beta) or the forward epilogue.
constexpr int kSkWaves = 8, kSkStages = 3, kSkRows = 16;
constexpr int kSkA = kSkRows * 64 / 8, kSkB = 64 * 16 / 8; // uint4 of one A and one B stage

template <bool TA, bool F16>
__global__ void __launch_bounds__(kSkWaves * 64, 1)
    k_skinny(const uint16_t *__restrict__ A, size_t lda, int a_extent, const uint16_t *__restrict__ B, size_t ldb,
             int b_extent, float *__restrict__ C, size_t ldc, int m, int n, int k, int beta, pgk_epi epi, int has_epi)
{
    __shared__ uint4 smem[kSkWaves * kSkStages * (kSkA + kSkB)];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // consecutive row tiles on one XCD: with A MN-contiguous four tiles
    // share each 128-byte line of a row
    int pid = (int)blockIdx.x;
    const int nb = (int)gridDim.x;
    if ((nb & 7) == 0)
        pid = (pid & 7) * (nb >> 3) + (pid >> 3);
    const int r0 = pid * kSkRows;
    LDS uint4 *const ring = (LDS uint4 *)smem + wave * kSkStages * (kSkA + kSkB);
    // this wave's run of chunks; loads at k >= kend read the zero page
    const int nct = (k + 63) / 64, cpw = (nct + kSkWaves - 1) / kSkWaves, c0 = wave * cpw;
    const int nc = nct - c0 < cpw ? (nct - c0 > 0 ? nct - c0 : 0) : cpw;
    const int kend = (c0 + nc) * 64 < k ? (c0 + nc) * 64 : k;
    using TK = TileK<kSkRows, 64, 64>;
    static_assert(TK::NQ == 2, "two loads of 8 rows x 128 bytes per A stage");
    constexpr int LPT = 4; // loads per chunk: two of A, two of B
    auto load = [&](int c, int st) {
        LDS uint4 *sa = ring + st * (kSkA + kSkB), *sb = sa + kSkA;
        const int k0 = (c0 + c) * 64;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if constexpr (!TA) {
                TK::load_q(q, A, lda, r0, a_extent, k0, kend, sa, lane);
            } else {
                // [64 p][16 i]: two 16-byte chunks per p-row
                const int slot = q * 64 + lane, p = slot >> 1;
                int i = r0 + (slot & 1) * 8;
                i = i < a_extent ? i : a_extent - 8;
                const void *src = k0 + p < kend ? (const void *)(A + (size_t)(k0 + p) * lda + i) : (const void *)&g_zero16;
                dma16(src, sa + q * 64);
            }
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            // [64 p][16 j]: two 16-byte chunks per p-row
            const int slot = q * 64 + lane, p = slot >> 1, j = (slot & 1) * 8;
            const void *src =
                k0 + p < kend && j < b_extent ? (const void *)(B + (size_t)(k0 + p) * ldb + j) : (const void *)&g_zero16;
            dma16(src, sb + q * 64);
        }
    };
    // ds_read_b64_tr_b16 pair over a [64][16] tile (32-byte rows): in 16-lane
    // group g, source lane q points at [k0 + q / 4][4 (q % 4)] and result lane
    // i holds column i, k = k0 .. k0 + 7 (k0 = 16 s + 8 (g >> 1))
    auto tr_frag = [&](const LDS uint4 *st, int s) {
        const int g = (lane >> 4) & 3, q = lane & 15;
        uint2 h2[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int p = 16 * s + 8 * (g >> 1) + 4 * h + (q >> 2);
            h2[h] = __builtin_bit_cast(
                uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS v4s *)((const LDS char *)st + p * 32 + (q & 3) * 8)));
        }
        return make_uint4(h2[0].x, h2[0].y, h2[1].x, h2[1].y);
    };
    // lanes of B columns 0 .. 15 (the rest hold columns 16 .. 31: zero)
    const bool bcol = ((lane >> 4) & 1) == 0;
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e)
        acc[e] = 0.0f;
    if (nc > 0) {
#pragma unroll
        for (int s = 0; s < kSkStages; ++s)
            load(s, s);
        for (int c = 0; c < nc; ++c) {
            const int st = c % kSkStages;
            const LDS uint4 *sa = ring + st * (kSkA + kSkB), *sb = sa + kSkA;
            // chunk c landed (the newest kSkStages - 1 chunks may be in flight)
            __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((kSkStages - 1) * LPT));
            __asm__ volatile("" ::: "memory");
            uint4 af[4], bf[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if constexpr (!TA) {
                    // rows lane % 16 (lanes 16 .. 31 of each half repeat them)
                    const int r = lane & 15;
                    const u32x4 v = ((const LDS u32x4 *)sa)[r * TK::CH + TK::swz(2 * s + (lane >> 5), r)];
                    af[s] = __builtin_bit_cast(uint4, v);
                } else {
                    af[s] = tr_frag(sa, s);
                }
                const uint4 b = tr_frag(sb, s);
                bf[s] = bcol ? b : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
                acc = mfma32<F16>(af[s], bf[s], acc);
            // the stage's reads are done before its refill
            __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(63));
            __asm__ volatile("" ::: "memory");
            load(c + kSkStages, st);
        }
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0));
    }
    // the waves' partials through LDS (the rings are done), added in wave
    // order; output rows 8 (e / 4) + 4 (lane / 32) + e % 4 < 16 are e < 8
    __syncthreads();
    constexpr int RP = 17;
    LDS float *red = (LDS float *)smem;
    static_assert(kSkWaves * kSkRows * RP * 4 <= (int)sizeof(smem), "partials fit the rings");
    const int col = lane & 31, lk = lane >> 5;
    if (col < 16) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            red[(wave * kSkRows + (e >> 2) * 8 + lk * 4 + (e & 3)) * RP + col] = acc[e];
    }
    __syncthreads();
    static_assert(kSkWaves * 64 >= kSkRows * 16, "a thread per element of the block's rows");
    const int t = (int)threadIdx.x, row = t >> 4, j = t & 15, gr = r0 + row;
    if (row < kSkRows && gr < m && j < n) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kSkWaves; ++w)
            v += red[(w * kSkRows + row) * RP + j];
        const size_t off = (size_t)gr * ldc + j;
        if (has_epi)
            epi_store(epi, C, off, j, v);
        else
            C[off] = beta ? C[off] + v : v;
    }
}

// four-wave blocks stay within two waves per SIMD, so two blocks share a CU
template <class CF>
__global__ void __launch_bounds__(CF::NT, CF::KG == 4 ? 2 : 1) k_gemm16_ks(gemm_kargs g, int has_epi)
{
    __shared__ uint4 smem[CF::LDS_U4];
    ks_block<CF>(g, has_epi, (int)blockIdx.x, (int)gridDim.x, true, (int)blockIdx.z, (LDS uint4 *)smem);
}

// a matmul's dgrad (blocks [0, n1)) and wgrad in one launch, each nb tiles
// per batch entry, on one tile shape
template <class C1, class C2>
__global__ void __launch_bounds__(C1::NT, C1::KG == 4 ? 2 : 1) k_gemm16_ks_pair(gemm_kargs g1, gemm_kargs g2, int nb1, int n1, int nb2)
{
    static_assert(C1::NT == C2::NT && C1::LDS_U4 == C2::LDS_U4, "one tile shape");
    __shared__ uint4 smem[C1::LDS_U4];
    const int b = (int)blockIdx.x;
    if (b < n1)
        ks_block<C1>(g1, 0, b % nb1, nb1, true, b / nb1, (LDS uint4 *)smem);
    else
        ks_block<C2>(g2, 0, (b - n1) % nb2, nb2, (n1 & 7) == 0, (b - n1) / nb2, (LDS uint4 *)smem);
}

// Few rows: C[m, n] (+)= A . B with A K-contiguous and B MN-contiguous, m <= 16
// (a forward over a handful of inputs; up to 64 for at most 16 columns).  Such
// a product streams B once, so a block owns 16 columns of one 16-row tile (256
// blocks for 4096 columns: every CU streams) and its eight waves split the
// reduction as k_gemm16_ks's do, each with a three-stage ring of 64-deep
// chunks of its own.  Tiles of 16 x 16 (v_mfma_f32_16x16x32) halve what A costs
// the 32-row ones.  Bound by the stream of 32-byte row pieces: 16 x 4096 x 4096
// takes 11.4 us back to back (2.9 TB/s; 10.8 in the kernel, 3.1; 64-column
// pieces would take 8.8 without the sum across blocks that they need), against
// 14.3 on 32 x 32 tiles and 18.3 for split-K and its sum; 16 columns of the
// same take 5.9 us against 12.9.  Two or four stages, sixteen waves and 32 columns a block measured the same or slower.
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

constexpr int kFrWaves = 8, kFrStages = 3, kFrTile = 16, kFrK = 64;
constexpr int kFrA = kFrTile * kFrK / 8, kFrB = kFrK * kFrTile / 8; // uint4 of one A and one B stage

template <bool F16>
__global__ void __launch_bounds__(kFrWaves * 64, 1) k_few_rows(gemm_kargs g, int has_epi)
{
    __shared__ uint4 smem[kFrWaves * kFrStages * (kFrA + kFrB)];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // neighbouring column tiles share each 128-byte line of a row: on one XCD
    // (9 x 4032 at k = 7232, 252 blocks: 33 us as dealt, 15 grouped)
    const int pid = xcd_tile((int)blockIdx.x, (int)gridDim.x);
    const int n0 = pid * kFrTile, m0 = (int)blockIdx.y * kFrTile;
    LDS uint4 *const ring = (LDS uint4 *)smem + wave * kFrStages * (kFrA + kFrB);
    using TK = TileK<kFrTile, 64, kFrK>;
    static_assert(TK::NQ == 2 && kFrB == 128, "two loads of A and two of B per stage");
    constexpr int LPT = 4;
    const int nct = (g.K + kFrK - 1) / kFrK, nc = nct > wave ? (nct - wave + kFrWaves - 1) / kFrWaves : 0;
    // this wave's chunk c (chunk c * waves + wave of the reduction) into stage
    // st; k at or past K reads the zero page
    auto load = [&](int c, int st) {
        const int ch = c * kFrWaves + wave, k0 = ch < nct ? ch * kFrK : g.K;
        LDS uint4 *sa = ring + st * (kFrA + kFrB), *sb = sa + kFrA;
#pragma unroll
        for (int q = 0; q < 2; ++q)
            TK::load_q(q, g.A, g.lda, m0, g.a_extent, k0, g.K, sa, lane);
#pragma unroll
        for (int q = 0; q < 2; ++q) { // [64 k][16 columns]: two 16-byte chunks per k row
            const int slot = q * 64 + lane, k = slot >> 1;
            int col = n0 + (slot & 1) * 8;
            col = col < g.b_extent ? col : g.b_extent - 8;
            const void *src = k0 + k < g.K ? (const void *)(g.B + (size_t)(k0 + k) * g.ldb + col) : (const void *)&g_zero16;
            dma16(src, sb + q * 64);
        }
    };
    const int grp = lane >> 4, q16 = lane & 15;
    f32x4m acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (nc > 0) {
#pragma unroll
        for (int s = 0; s < kFrStages; ++s)
            load(s, s);
        int st = 0;
        for (int c = 0; c < nc; ++c) {
            const LDS uint4 *sa = ring + st * (kFrA + kFrB), *sb = sa + kFrA;
            // chunk c landed (the newest kFrStages - 1 chunks may be in flight)
            __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((kFrStages - 1) * LPT));
            __asm__ volatile("" ::: "memory");
            // 16-lane group grp holds k = 32 s + 8 grp .. + 7 of row (A) or
            // column (B) lane % 16; B from two transposing reads
            uint4 fa[2], fb[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const u32x4 v = ((const LDS u32x4 *)sa)[q16 * TK::CH + TK::swz(4 * s + grp, q16)];
                fa[s] = __builtin_bit_cast(uint4, v);
                uint2 h2[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = 32 * s + 8 * grp + 4 * h + (q16 >> 2);
                    h2[h] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                          (LDS v4s *)((const LDS char *)sb + k * 32 + (q16 & 3) * 8)));
                }
                fb[s] = make_uint4(h2[0].x, h2[0].y, h2[1].x, h2[1].y);
            }
            // the stage's reads are done before its refill
            __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(63));
            __asm__ volatile("" ::: "memory");
            load(c + kFrStages, st);
#pragma unroll
            for (int s = 0; s < 2; ++s)
                acc = mfma16<F16>(fa[s], fb[s], acc);
            st = st + 1 == kFrStages ? 0 : st + 1;
        }
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0));
    }
    __syncthreads(); // the rings are done: the waves' partials through LDS, added in wave order
    constexpr int RP = kFrTile + 1;
    LDS float *part = (LDS float *)smem;
    static_assert(kFrWaves * kFrTile * RP * 4 <= (int)sizeof(smem), "partials fit the rings");
#pragma unroll
    for (int e = 0; e < 4; ++e) // lane holds column lane % 16 of rows 4 (lane / 16) + e
        part[(wave * kFrTile + 4 * grp + e) * RP + q16] = acc[e];
    __syncthreads();
    const int t = (int)threadIdx.x, row = t >> 4, col = t & 15;
    if (row < kFrTile && m0 + row < g.M && n0 + col < g.N) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kFrWaves; ++w)
            v += part[(w * kFrTile + row) * RP + col];
        const size_t off = (size_t)(m0 + row) * g.ldc + n0 + col;
        if (has_epi)
            epi_store(g.epi, g.C, off, n0 + col, v);
        else
            g.C[off] = g.beta ? g.C[off] + v : v;
    }
}

// the same epilogue as a pass over a finished C (k-tail runs)
__global__ void __launch_bounds__(256) k_bias_act(float *__restrict__ c, size_t ldc, int m, int n, pgk_epi epi)
{
    const size_t mn = (size_t)m * n;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < mn; i += (size_t)gridDim.x * blockDim.x) {
        const size_t r = i / n, col = i - r * n, off = r * ldc + col;
        epi_store(epi, c, off, (int)col, c[off]);
    }
}

// zero-padded copy of the k-slab [k0, k0 + kn) of an operand, kn <= 64:
// K-contiguous -> dst[r * 64 + c], MN-contiguous -> dst[c * rows_pad + r]
__global__ void __launch_bounds__(256) k_pack_slab(int mn_major, const uint16_t *__restrict__ src, size_t ld,
                                                   size_t sstride, int rows, int rows_pad, int k0, int kn,
                                                   uint16_t *__restrict__ dst, size_t dstride)
{
    const uint16_t *s = src + (size_t)blockIdx.z * sstride;
    uint16_t *d = dst + (size_t)blockIdx.z * dstride;
    const size_t total = (size_t)rows_pad * 64;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        int r, c;
        if (mn_major) {
            c = (int)(i / rows_pad);
            r = (int)(i % rows_pad);
        } else {
            r = (int)(i / 64);
            c = (int)(i % 64);
        }
        uint16_t v = 0;
        if (r < rows && c < kn)
            v = mn_major ? s[(size_t)(k0 + c) * ld + r] : s[(size_t)r * ld + k0 + c];
        d[i] = v;
    }
}

// split-K finish of up to two problems (grid z picks one; a problem with
// splits = 0 is absent): C = (beta ? C : 0) + sum over the `splits` partial
// products (each m x n, dense), added in split order, then with `epi` the
// GEMM's epilogue on that value (k_bias_act's arithmetic, in the same
// pass).  With n and ldc allowing 16-byte accesses, rows run along grid y
// (stride gridDim.y) and columns along x, four per thread; otherwise
// (narrow outputs such as n = 10) one element per thread over the
// flattened m x n, indexed with a 32-bit division when m n fits
struct splitk_desc {
    const float *part;
    int splits, m, n;
    float *c;
    size_t ldc;
    int beta, v4, has_epi;
    pgk_epi epi;
};

splitk_desc splitk_of(const float *part, int splits, size_t m, size_t n, float *c, size_t ldc, int beta,
                      const pgk_epi *epi = nullptr)
{
    int v4 = ((n | (ldc & 3)) & 3) == 0 && (((uintptr_t)c | (uintptr_t)part) & 15) == 0;
    if (epi)
        v4 = v4 && ((((uintptr_t)epi->z) | ((uintptr_t)epi->bias)) & 15) == 0 && (((uintptr_t)epi->c16) & 7) == 0;
    return splitk_desc{part, splits, (int)m, (int)n, c, ldc, beta, v4, epi != nullptr, epi ? *epi : pgk_epi{}};
}

dim3 splitk_grid(const splitk_desc &a, const splitk_desc &b)
{
    unsigned gx = 1, gy = 1;
    for (const splitk_desc *d : {&a, &b}) {
        if (!d->splits)
            continue;
        const size_t mn = (size_t)d->m * d->n;
        const unsigned x = d->v4 ? (unsigned)((d->n / 4 + 255) / 256) : (unsigned)((mn + 255) / 256 < 2048 ? (mn + 255) / 256 : 2048);
        const unsigned y = d->v4 ? (unsigned)(d->m < 65535 ? d->m : 65535) : 1u;
        gx = x > gx ? x : gx;
        gy = y > gy ? y : gy;
    }
    return dim3(gx, gy, &a == &b || !b.splits ? 1u : 2u);
}

__global__ void __launch_bounds__(256) k_splitk_sum(splitk_desc d0, splitk_desc d1)
{
    const splitk_desc &d = blockIdx.z ? d1 : d0;
    if (!d.splits)
        return;
    const float *__restrict__ part = d.part;
    float *__restrict__ c = d.c;
    const int m = d.m, n = d.n, splits = d.splits, beta = d.beta;
    const size_t ldc = d.ldc;
    const size_t mn = (size_t)m * n;
    if (d.v4) {
        const int j = blockIdx.x * blockDim.x + threadIdx.x;
        if (j >= n >> 2)
            return;
        for (int r = blockIdx.y; r < m; r += gridDim.y) {
            const float *p = part + (size_t)r * n + 4 * j;
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int z = 0; z < splits; ++z)
                acc += __builtin_nontemporal_load((const f32x4 *)(p + (size_t)z * mn)); // read once
            f32x4 *q = (f32x4 *)(c + (size_t)r * ldc + 4 * j);
            const f32x4 v = beta ? *q + acc : acc;
            if (!d.has_epi) {
                *q = v;
                continue;
            }
            const pgk_epi &epi = d.epi;
            const size_t off = (size_t)r * ldc + 4 * j;
            f32x4 zv = v, o;
            if (epi.bias)
                zv += *(const f32x4 *)(epi.bias + 4 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[e] = act_f(epi.act, zv[e]);
            if (!epi.skip_out)
                *q = o;
            if (epi.z)
                *(f32x4 *)(epi.z + off) = zv;
            if (epi.c16)
                *(uint2 *)(epi.c16 + off) = make_uint2(to16x2(epi.dtype16, o[0], o[1]), to16x2(epi.dtype16, o[2], o[3]));
        }
        return;
    }
    if (blockIdx.y)
        return;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < mn; i += (size_t)gridDim.x * blockDim.x) {
        size_t r, col;
        if (mn <= 0xffffffffu) {
            r = (uint32_t)i / (uint32_t)n;
            col = (uint32_t)i - (uint32_t)r * (uint32_t)n;
        } else {
            r = i / n;
            col = i - r * n;
        }
        float acc = 0.0f;
        for (int z = 0; z < splits; ++z)
            acc += part[(size_t)z * mn + i];
        const size_t off = r * ldc + col;
        const float v = beta ? c[off] + acc : acc;
        if (d.has_epi)
            epi_store(d.epi, c, off, (int)col, v);
        else
            c[off] = v;
    }
}

// C rows of an empty reduction: zeros
__global__ void __launch_bounds__(256) k_zero_rows(float *__restrict__ c, size_t ldc, size_t sc, int m, int n)
{
    float *cb = c + (size_t)blockIdx.z * sc;
    const size_t mn = (size_t)m * n;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < mn; i += (size_t)gridDim.x * blockDim.x) {
        const size_t r = i / n, col = i - r * n;
        cb[r * ldc + col] = 0.0f;
    }
}

struct gemm_args {
    const uint16_t *a;
    size_t lda, sa;
    int a_extent;
    const uint16_t *b;
    size_t ldb, sb;
    int b_extent;
    float *c;
    size_t ldc, sc;
    int m, n, k, beta;
    unsigned batch;
    int tile = 0;     // 2: 256 x 256 tiles, 1: 128 x 128, 0: by tile count
    // split-K: slice z reduces [z kz_step, min(k_total, (z+1) kz_step));
    // k_total = 0: no split
    int k_total = 0, kz_step = 0;
};

template <class CF>
gemm_kargs make_kargs(const gemm_args &g, const pgk_epi &epi)
{
    gemm_kargs k;
    k.A = g.a, k.lda = g.lda, k.sA = g.sa, k.a_extent = g.a_extent;
    k.B = g.b, k.ldb = g.ldb, k.sB = g.sb, k.b_extent = g.b_extent;
    k.C = g.c, k.ldc = g.ldc, k.sC = g.sc;
    k.M = g.m, k.N = g.n, k.K = g.k, k.beta = g.beta;
    k.tiles_m = (g.m + CF::BM - 1) / CF::BM, k.tiles_n = (g.n + CF::BN - 1) / CF::BN;
    k.epi = epi;
    k.k_total = g.k_total ? g.k_total : g.k, k.kz_step = g.kz_step;
    k.fast_ok = (int)(g.lda < kFastLd && g.ldb < kFastLd);
    return k;
}

template <int BM, int BN, int WGM, int WGN, bool TA, bool TB, bool F16, bool EPI, int KB = 64, int S = 2>
int launch_tile(const gemm_args &g, const pgk_epi &epi, hipStream_t s)
{
    using CF = gcfg<BM, BN, WGM, WGN, TA, TB, F16, EPI, KB, S>;
    const gemm_kargs k = make_kargs<CF>(g, epi);
    hipLaunchKernelGGL(k_gemm16<CF>, dim3((unsigned)(k.tiles_m * k.tiles_n), 1, g.batch), dim3(CF::NT), 0, s, k);
    return (int)hipGetLastError();
}

// the split-over-waves tiles of the planner: 5 is 32 x 32 with eight waves, 6
// 32 x 64 with eight, 7 64 x 64 with four (two blocks per CU), 8 64 x 64 with
// eight.  Deeper rings measured slower.
template <int TILE, bool TA, bool TB, bool F16>
using ks_cfg = typename std::conditional<
    TILE == 5, kscfg<32, 32, 8, 64, 2, TA, TB, F16>,
    typename std::conditional<TILE == 6, kscfg<32, 64, 8, 32, 3, TA, TB, F16>,
                              kscfg<64, 64, TILE == 8 ? 8 : 4, 32, 2, TA, TB, F16>>::type>::type;

template <class CF>
gemm_kargs ks_kargs(const gemm_args &g, const pgk_epi &epi)
{
    return make_kargs<gcfg<CF::TM, CF::TN, 1, 1, CF::TA, CF::TB, CF::F16, false, 64, 2>>(g, epi);
}

template <class CF>
int launch_ks(const gemm_args &g, const pgk_epi &epi, int has_epi, hipStream_t s)
{
    const gemm_kargs k = ks_kargs<CF>(g, epi);
    hipLaunchKernelGGL(k_gemm16_ks<CF>, dim3((unsigned)(k.tiles_m * k.tiles_n), 1, g.batch), dim3(CF::NT), 0, s, k,
                       has_epi);
    return (int)hipGetLastError();
}

template <bool TA, bool TB, bool F16>
int launch_ks_tile(const gemm_args &g, const pgk_epi &epi, int has_epi, hipStream_t s)
{
    switch (g.tile) {
    case 5: return launch_ks<ks_cfg<5, TA, TB, F16>>(g, epi, has_epi, s);
    case 6: return launch_ks<ks_cfg<6, TA, TB, F16>>(g, epi, has_epi, s);
    case 8: return launch_ks<ks_cfg<8, TA, TB, F16>>(g, epi, has_epi, s);
    default: return launch_ks<ks_cfg<7, TA, TB, F16>>(g, epi, has_epi, s);
    }
}

int launch_ks_any(int f16, int ta, int tb, const gemm_args &g, const pgk_epi &epi, int has_epi, hipStream_t s)
{
    const int sel = (f16 ? 4 : 0) | (ta ? 2 : 0) | (tb ? 1 : 0);
    switch (sel) {
    case 0: return launch_ks_tile<false, false, false>(g, epi, has_epi, s);
    case 1: return launch_ks_tile<false, true, false>(g, epi, has_epi, s);
    case 2: return launch_ks_tile<true, false, false>(g, epi, has_epi, s);
    case 3: return launch_ks_tile<true, true, false>(g, epi, has_epi, s);
    case 4: return launch_ks_tile<false, false, true>(g, epi, has_epi, s);
    case 5: return launch_ks_tile<false, true, true>(g, epi, has_epi, s);
    case 6: return launch_ks_tile<true, false, true>(g, epi, has_epi, s);
    default: return launch_ks_tile<true, true, true>(g, epi, has_epi, s);
    }
}

template <bool F16, int TILE>
int launch_ks_pair(const gemm_args &gd, const gemm_args &gw, hipStream_t s)
{
    using CD = ks_cfg<TILE, false, false, F16>;
    using CW = ks_cfg<TILE, true, true, F16>;
    const gemm_kargs kd = ks_kargs<CD>(gd, pgk_epi{}), kw = ks_kargs<CW>(gw, pgk_epi{});
    const int nb1 = kd.tiles_m * kd.tiles_n, nb2 = kw.tiles_m * kw.tiles_n;
    const int n1 = nb1 * (int)gd.batch, n2 = nb2 * (int)gw.batch;
    hipLaunchKernelGGL((k_gemm16_ks_pair<CD, CW>), dim3((unsigned)(n1 + n2)), dim3(CD::NT), 0, s, kd, kw, nb1, n1, nb2);
    return (int)hipGetLastError();
}

template <bool F16>
int launch_ks_pair_tile(int tile, const gemm_args &gd, const gemm_args &gw, hipStream_t s)
{
    switch (tile) {
    case 5: return launch_ks_pair<F16, 5>(gd, gw, s);
    case 6: return launch_ks_pair<F16, 6>(gd, gw, s);
    case 8: return launch_ks_pair<F16, 8>(gd, gw, s);
    default: return launch_ks_pair<F16, 7>(gd, gw, s);
    }
}

// The configurations launch_layout picks from (the planner's tile ids):
//  - 2: 256 x 256 tiles, eight waves of 128 x 64; k-tiles of 32 in a
//    four-stage ring (128 KiB of LDS), except with both operands
//    K-contiguous: there a k-tile of 32 covers half of each 128-byte row
//    segment per load, and k-tiles of 64 in two stages measure faster;
//  - 3: 128 x 256 tiles, eight waves of 64 x 64: twice the tiles of 2 for
//    grids 2 leaves short of the chip, without split-K's partials; k-tiles
//    of 64 in three stages (144 KiB) with both operands K-contiguous, else
//    of 32 in four stages (96 KiB);
//  - 1: 128 x 128 tiles, four waves of 64 x 64; k-tiles of 64, two stages.
// An unplanned launch (tile 0) takes 2 when that still gives most CUs a
// tile, else 1.
inline int tile_of(const gemm_args &g)
{
    if (g.tile)
        return g.tile;
    const size_t big = (size_t)((g.m + 255) / 256) * ((g.n + 255) / 256) * g.batch;
    return big >= 128 ? 2 : 1;
}

template <bool TA, bool TB, bool F16, bool EPI, int TILE>
using layout_cfg = typename std::conditional<
    TILE == 2,
    typename std::conditional<!TA && !TB, gcfg<256, 256, 2, 4, TA, TB, F16, EPI, 64, 2>,
                              gcfg<256, 256, 2, 4, TA, TB, F16, EPI, 32, 4>>::type,
    typename std::conditional<
        TILE == 3,
        typename std::conditional<!TA && !TB, gcfg<128, 256, 2, 4, TA, TB, F16, EPI, 64, 3>,
                                  gcfg<128, 256, 2, 4, TA, TB, F16, EPI, 32, 4>>::type,
        gcfg<128, 128, 2, 2, TA, TB, F16, EPI, 64, 2>>::type>::type;

template <class CF>
int launch_cfg(const gemm_args &g, const pgk_epi &epi, hipStream_t s)
{
    return launch_tile<CF::BM, CF::BN, CF::WGM, CF::WGN, CF::TA, CF::TB, CF::F16, CF::EPI, CF::KB, CF::S>(g, epi, s);
}

template <bool TA, bool TB, bool F16, bool EPI = false>
int launch_layout(const gemm_args &g, hipStream_t s, const pgk_epi &epi = pgk_epi{})
{
    switch (tile_of(g)) {
    case 2: return launch_cfg<layout_cfg<TA, TB, F16, EPI, 2>>(g, epi, s);
    case 3: return launch_cfg<layout_cfg<TA, TB, F16, EPI, 3>>(g, epi, s);
    default: return launch_cfg<layout_cfg<TA, TB, F16, EPI, 1>>(g, epi, s);
    }
}

// dgrad (both operands K-contiguous, tile TD) and wgrad (both MN-contiguous,
// tile TW) of one matmul in one launch
template <bool F16, int TD, int TW>
int launch_pair_dw(const gemm_args &gd, const gemm_args &gw, hipStream_t s)
{
    using CD = layout_cfg<false, false, F16, false, TD>;
    using CW = layout_cfg<true, true, F16, false, TW>;
    const gemm_kargs kd = make_kargs<CD>(gd, pgk_epi{}), kw = make_kargs<CW>(gw, pgk_epi{});
    const int nb1 = kd.tiles_m * kd.tiles_n, nb2 = kw.tiles_m * kw.tiles_n;
    const int n1 = nb1 * (int)gd.batch, n2 = nb2 * (int)gw.batch;
    hipLaunchKernelGGL((k_gemm16_pair<CD, CW>), dim3((unsigned)(n1 + n2)), dim3(CD::NT), 0, s, kd, kw, nb1, n1, nb2);
    return (int)hipGetLastError();
}

// A dgrad in `splits` slices of its reduction and a wgrad, each finished by an
// epilogue (or, in slices, left as dense f32 partials), in one launch on 128 x
// 256 tiles.  A slice's blocks, and neighbouring tiles of the wgrad, go to one
// XCD: with every slice on every XCD each L2 would read the whole of both
// operands.
template <class C1, class C2>
__global__ void __launch_bounds__(C1::NT, 1) k_gemm16_grads(gemm_kargs g1, gemm_kargs g2, int nb1, int n1, int n2)
{
    static_assert(C1::NT == C2::NT, "one block size");
    __shared__ uint4 smem[C1::LDS_U4 > C2::LDS_U4 ? C1::LDS_U4 : C2::LDS_U4];
    const int b = (int)blockIdx.x;
    if (b < n1) {
        const int t = xcd_tile(b, n1);
        gemm16_block<C1>(g1, t % nb1, nb1, false, t / nb1, (LDS uint4 *)smem);
    } else {
        const int t = xcd_tile(b - n1, n2), nb2 = g2.tiles_m * g2.tiles_n;
        gemm16_block<C2>(g2, t % nb2, nb2, false, t / nb2, (LDS uint4 *)smem);
    }
}

template <bool F16>
int launch_grads(const gemm_args &gd, const pgk_epi &ed, const gemm_args &gw, const pgk_epi &ew, hipStream_t s)
{
    using CD = layout_cfg<false, false, F16, true, 3>;
    using CW = layout_cfg<true, true, F16, true, 3>;
    const gemm_kargs kd = make_kargs<CD>(gd, ed), kw = make_kargs<CW>(gw, ew);
    const int nb1 = kd.tiles_m * kd.tiles_n, n1 = nb1 * (int)gd.batch, n2 = kw.tiles_m * kw.tiles_n * (int)gw.batch;
    hipLaunchKernelGGL((k_gemm16_grads<CD, CW>), dim3((unsigned)(n1 + n2)), dim3(CD::NT), 0, s, kd, kw, nb1, n1, n2);
    return (int)hipGetLastError();
}

// both problems on tile `tile`
template <bool F16>
int launch_pair_tiles(int tile, const gemm_args &gd, const gemm_args &gw, hipStream_t s)
{
    switch (tile) {
    case 2: return launch_pair_dw<F16, 2, 2>(gd, gw, s);
    case 3: return launch_pair_dw<F16, 3, 3>(gd, gw, s);
    default: return launch_pair_dw<F16, 1, 1>(gd, gw, s);
    }
}

int launch_any(int f16, int ta, int tb, const gemm_args &g, hipStream_t s)
{
    const int sel = (f16 ? 4 : 0) | (ta ? 2 : 0) | (tb ? 1 : 0);
    switch (sel) {
    case 0: return launch_layout<false, false, false>(g, s);
    case 1: return launch_layout<false, true, false>(g, s);
    case 2: return launch_layout<true, false, false>(g, s);
    case 3: return launch_layout<true, true, false>(g, s);
    case 4: return launch_layout<false, false, true>(g, s);
    case 5: return launch_layout<false, true, true>(g, s);
    case 6: return launch_layout<true, false, true>(g, s);
    default: return launch_layout<true, true, true>(g, s);
    }
}

// ---------------------------------------------------------------- MFMA probe
// The attainable MFMA rate of this chip, for the roofline: eight waves per
// CU run back-to-back v_mfma_f32_32x32x16_bf16 on 4 x 2 fragment tiles,
// either from registers (lds = 0) or read from LDS one k-step ahead as the
// GEMM's inner loop does (lds = 1).  The operands are bf16 values of
// magnitude 0.5 .. 2 with pseudo-random signs and mantissas: the matrix
// units draw more power, and the chip clocks lower, on such data than on
// constant patterns.
__global__ void __launch_bounds__(512, 1) k_mfma_probe(float *sink, int iters, int lds)
{
    __shared__ uint4 sm[8192];
    for (int i = threadIdx.x; i < 8192; i += blockDim.x) {
        uint32_t v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t h = (uint32_t)(i * 4 + q + 1) * 2654435761u;
            h ^= h >> 15;
            h *= 2246822519u;
            h ^= h >> 13;
            const uint32_t lo = (h & 0x7Fu) | ((h >> 9) & 1u ? 0x3F80u : 0x3F00u) | ((h & 0x100u) << 7);
            const uint32_t hi = ((h >> 16) & 0x7Fu) | ((h >> 25) & 1u ? 0x3F80u : 0x3F00u) | ((h >> 9) & 0x8000u);
            v[q] = lo | (hi << 16);
        }
        sm[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
    __syncthreads();
    f32x16 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[i][j][e] = 0.0f;
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint4 fa[2][4], fb[2][2];
    auto rd = [&](int it, uint4(&xa)[4], uint4(&xb)[2]) {
        const int base = lds ? (it & 7) * 512 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            xa[i] = sm[((w * 8 + i) * 64 + l + base) & 8191];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            xb[j] = sm[((w * 8 + 4 + j) * 64 + l + base) & 8191];
    };
    rd(0, fa[0], fb[0]);
    rd(1, fa[1], fb[1]);
    for (int it = 0; it < iters; it += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (lds)
                rd(it + u + 2, fa[u ^ 1], fb[u ^ 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = mfma32<false>(fa[u][i], fb[u][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                sum += acc[i][j][e];
    sink[(size_t)blockIdx.x * blockDim.x + threadIdx.x] = sum;
}

} // namespace


// Launch plan of one GEMM: the tile (256 x 256 with eight waves, or
// 128 x 128 with four) and a split-K factor, from a small cost model of
// this chip.  A launch takes ceil(blocks / 256 CUs) rounds of one block's
// time, that block running at the per-CU rate measured for its tile
// (~4.4 and ~2.6 TFLOP/s); split-K (slices of the reduction run as a
// batch into dense partials that k_splitk_sum adds in slice order, so the
// result is deterministic) adds a pass over sp + 1 copies of C at ~5 TB/s.
// Ragged shapes such as M = 4097 (33 rows of 128-tiles) and weight grads
// with a short output dim are where it matters.
typedef struct {
    int tile; // 2 = 256 x 256, 3 = 128 x 256, 1 = 128 x 128, 5 - 8: ks_tile
    int sp;   // split-K factor, 1 = none
} gemm_plan;

// `cu_budget` is the number of CUs the launch may occupy (another launch
// runs beside it on the rest), 0 for the whole chip.
static constexpr int kCUs = 256;

// The split-over-waves tile for `problems` problems run as one launch, 0 when
// none: the smallest tile whose blocks all run at once, one per CU (two for
// the 64 x 64 tile), up to the longest reduction at which it still wins.
// Blocks: each tile beats the larger ones up to its count (32 x 32 at 256
// blocks 3.7 - 13 against 7.2 - 20 us; 64 x 64 at 512 blocks 7.1 - 33 against
// 7.5 - 36 us, k 128 to 2816) and loses past it (64 x 64 at 1024 blocks 12 - 21
// against 7.6 - 17 us).
// Reductions: a block's waves stream its operands through one CU where
// split-K's eight slices have eight, so long ones are the split's (700 shapes,
// other inputs in every launch).  Alone, a 32 x 32 tile is 0.95 - 2.5 times as
// fast up to k = 10240 and with both operands MN-contiguous, whose every k row
// is a 64-byte piece, 0.92 - 2 times up to 6144 (0.67 - 1 from 8192; 512 x 512 at
// 65536: 175 against 93 us), 32 x 64 to 5632 (0.77 - 0.99 from 6144), 64 x 64 to
// 4608 with one block on a CU and to 2816 with two (0.73 - 1.1 at 2816 - 4096;
// 2048 x 1024 at 65536: 659 against 236 us).  A pair saves launches too and holds
// to 8192 on tiles of 32 rows (1.2 - 2.4 times the two apart), on 64 x 64 to 7168
// with one block on a CU and to 4096 with two: past it the long wgrad is a few
// blocks of a tile larger than its own (f16 matmul with grads of 8192 x 128 x
// 1024 52 against 43 us, 16384 x 64 x 64 65 against 39).
// 64 x 64 tiles take eight waves in place of four for a long reduction that
// leaves one block per CU: the same time (8.4 and 8.5 us at 1024^3), with a
// shorter chain of sums per wave.  plan_gemm keeps products of at most 16
// columns from these tiles (more than half would be padding); in a pair they
// are welcome (rows 6928, 16 x 88: 16 us in one launch, 22 in two).
struct ks_size {
    size_t m, n, batch, k;
};
static int ks_tile(std::initializer_list<ks_size> problems, bool mn, bool any_k = false)
{
    static const struct {
        int tile;
        size_t tm, tn, most, k_most, k_mn, k_pair; // k_mn: both operands MN-contiguous
    } shapes[4] = {{5, 32, 32, 256, 10240, 6144, 8192}, {6, 32, 64, 256, 5632, 5632, 8192},
                   {8, 64, 64, 256, 4608, 4608, 7168}, {7, 64, 64, 512, 2816, 2816, 4096}};
    for (const auto &sh : shapes) {
        size_t blocks = 0, k = 0;
        for (const ks_size &q : problems) {
            blocks += ((q.m + sh.tm - 1) / sh.tm) * ((q.n + sh.tn - 1) / sh.tn) * q.batch;
            k = q.k > k ? q.k : k;
        }
        if (blocks > sh.most)
            continue;
        if (!any_k && k > (problems.size() > 1 ? sh.k_pair : mn ? sh.k_mn : sh.k_most))
            return 0;
        return sh.tile == 8 && k < 1024 ? 7 : sh.tile;
    }
    return 0;
}

// its time, from the same measurements: a launch and a rate per k
static double ks_time(int tile, size_t m, size_t n, size_t k, size_t batch)
{
    const double kk = (double)k / 1024.0;
    if (tile == 5)
        return (3.4 + 1.8 * kk) * 1e-6;
    if (tile == 6)
        return (3.8 + 2.6 * kk) * 1e-6;
    const size_t blocks = ((m + 63) / 64) * ((n + 63) / 64) * batch;
    return (blocks <= 256 ? 4.6 + 3.5 * kk : 6.0 + 6.8 * kk) * 1e-6;
}

// Time model: rounds of one block per CU, each block at its tile's rate
// per CU (measured under a loaded chip), plus for a split its partials:
// the slices write sp - 1 more tiles of C than one launch would, the sum
// reads sp and writes one, at ~5 TB/s, and one more launch.  A split must
// still win by 8 % over the best plan without one: its partials also cost
// HBM capacity.
static gemm_plan plan_gemm(int ta, int tb, size_t m, size_t n, size_t kin, size_t batch, int cu_budget = 0,
                           double *time = nullptr, bool whole_k = false)
{
    const bool whole = !(cu_budget > 0 && cu_budget < kCUs);
    const double cus = whole ? (double)kCUs : (double)cu_budget;
    const int ks = whole && n > 16 && kin ? ks_tile({{m, n, batch, kin}}, ta && tb) : 0;
    if (ks) {
        if (time)
            *time = ks_time(ks, m, n, kin, batch);
        return {ks, 1};
    }
    struct shape {
        int tile;
        size_t bm, bn;
        double rate;
    };
    static const shape shapes[3] = {{2, 256, 256, 4.4e12}, {3, 128, 256, 3.75e12}, {1, 128, 128, 2.0e12}};
    const double bw = 5.0e12, launch = 5e-6;
    gemm_plan best = {2, 1};
    double best_t = 1e300;
    for (const shape &sh : shapes) {
        const size_t tiles = ((m + sh.bm - 1) / sh.bm) * ((n + sh.bn - 1) / sh.bn) * batch;
        const int max_sp = batch == 1 && kin >= 1024 && !whole_k ? 8 : 1;
        for (int sp = 1; sp <= max_sp; ++sp) {
            const size_t ks = ((kin + sp - 1) / sp + BK - 1) / BK * BK;
            if (sp > 1 && ks * (size_t)(sp - 1) >= kin)
                break; // the last slice would be empty
            const double rounds = ceil((double)(tiles * sp) / cus);
            double t = rounds * 2.0 * (double)sh.bm * (double)sh.bn * (double)(sp > 1 ? ks : kin) / sh.rate;
            if (sp > 1)
                t += 2.0 * (double)sp * (double)m * (double)n * 4.0 / bw + launch;
            if (t < best_t * (sp > 1 && best.sp == 1 ? 0.92 : 1.0)) {
                best_t = t;
                best.tile = sh.tile;
                best.sp = sp;
            }
        }
    }
    if (time)
        *time = best_t;
    return best;
}

// the k the main kernel covers: all of it when both operands are
// MN-contiguous (a partial last k-tile reads zero rows past k) or k % 8 == 0
// (zero chunks past k), else the 64-aligned part, the rest going through
// zero-padded slabs in one more launch
static size_t k_inkernel(int ta, int tb, size_t k) { return (ta && tb) || k % 8 == 0 ? k : k - k % BK; }

// k_skinny's products: at most 16 columns of C from an MN-contiguous B, one
// problem, a reduction it covers whole (any k with both operands
// MN-contiguous, k % 8 == 0 with A K-contiguous), and rows enough for 64 of
// its 16-row blocks; the rest keep the tiled plans (split-K among them)
static bool skinny_ok(int ta, int tb, size_t m, size_t n, size_t k, size_t batch)
{
    // (a launch holds under 2^32 threads, a block has 512)
    return tb && n <= 16 && batch == 1 && k && (ta || k % 8 == 0) && (m + 15) / 16 >= 64 &&
           (m + 15) / 16 < (size_t)1 << 23;
}

// k_few_rows's products: one 16-row tile with a block per CU at most (past
// 4096 columns the wider tiles stream faster: 22.5 against 37.5 us at 11008),
// or a few such tiles of one column tile.  Reductions as above: up to 12288 it
// is 0.95 - 2.8 times as fast as the split, from there 0.74 - 1.07, and up to
// 32768 for one column tile (8 at 33296: 24 against 34 us)
static bool few_rows_ok(int ta, int tb, size_t m, size_t n, size_t k, size_t batch)
{
    return !ta && tb && batch == 1 && k && k % 8 == 0 && ((m <= 16 && n <= 4096) || (m <= 64 && n <= 16)) &&
           (k <= 12288 || (k <= 32768 && n <= 16));
}

static size_t tail_ws(int ta, int tb, size_t m, size_t n, size_t k, size_t batch)
{
    if (k_inkernel(ta, tb, k) == k)
        return 0;
    const size_t ma = (m + 7) & ~(size_t)7, nb = (n + 7) & ~(size_t)7;
    const size_t a = (ta ? 64 * (ma < 8 ? 8 : ma) : 64 * m) * batch;
    const size_t b = (tb ? 64 * (nb < 8 ? 8 : nb) : 64 * n) * batch;
    return (a + 64 + b) * sizeof(uint16_t);
}

// the checks of pgk_gemm16_cu's operands
int check_gemm_args(int ta, int tb, size_t m, size_t n, size_t k, const uint16_t *a, size_t lda, size_t stride_a,
                    size_t a_extent, const uint16_t *b, size_t ldb, size_t stride_b, size_t b_extent, size_t batch)
{
    // k leaves headroom for the k offsets of the tiles the kernel loads
    // past the end (from the zero page) to stay within int
    if (m > 0x7fffffff || n > 0x7fffffff || k > 0x7fff0000 || batch > 65535)
        return (int)hipErrorInvalidValue;
    // a launch holds under 2^32 threads (more of them wrap with no error), a
    // 128 x 128 tile has 256
    if (((m + 127) / 128) * ((n + 127) / 128) >> 24)
        return (int)hipErrorInvalidValue;
    // 16-byte global loads: aligned bases, leading dims and batch strides
    if ((((uintptr_t)a | (uintptr_t)b) & 15) || (lda & 7) || (ldb & 7) || (stride_a & 7) || (stride_b & 7))
        return (int)hipErrorInvalidValue;
    // the clamped loads stay inside [0, extent) of each operand
    if (!a_extent || !b_extent || (ta && ((a_extent & 7) || a_extent < m)) || (tb && ((b_extent & 7) || b_extent < n)) ||
        (!ta && a_extent < m) || (!tb && b_extent < n) || a_extent > 0x7fffffff || b_extent > 0x7fffffff)
        return (int)hipErrorInvalidValue;
    return 0;
}

extern "C" size_t pgk_gemm16_workspace_cu(int ta, int tb, size_t m, size_t n, size_t k, size_t batch, int cu_budget)
{
    if (skinny_ok(ta, tb, m, n, k, batch) || few_rows_ok(ta, tb, m, n, k, batch))
        return 0;
    const gemm_plan pl = plan_gemm(ta, tb, m, n, k_inkernel(ta, tb, k), batch, cu_budget);
    const size_t part = pl.sp > 1 ? (((size_t)pl.sp * m * n * sizeof(float) + 255) & ~(size_t)255) : 0;
    return part + tail_ws(ta, tb, m, n, k, batch);
}

extern "C" size_t pgk_gemm16_workspace(int ta, int tb, size_t m, size_t n, size_t k, size_t batch)
{
    return pgk_gemm16_workspace_cu(ta, tb, m, n, k, batch, 0);
}

extern "C" int pgk_gemm16_plan(int ta, int tb, size_t m, size_t n, size_t k, size_t batch, int cu_budget, int *splits)
{
    if (skinny_ok(ta, tb, m, n, k, batch) || few_rows_ok(ta, tb, m, n, k, batch)) {
        if (splits)
            *splits = 1;
        return skinny_ok(ta, tb, m, n, k, batch) ? 4 : 9;
    }
    const gemm_plan pl = plan_gemm(ta, tb, m, n, k_inkernel(ta, tb, k), batch, cu_budget);
    if (splits)
        *splits = pl.sp;
    return pl.tile;
}

extern "C" int pgk_gemm16_whole_tile(size_t m, size_t n, size_t k)
{
    return plan_gemm(0, 1, m, n, k, 1, 0, nullptr, true).tile;
}

extern "C" double pgk_gemm16_time(int ta, int tb, size_t m, size_t n, size_t k, size_t batch, int cu_budget)
{
    if (skinny_ok(ta, tb, m, n, k, batch)) // A streamed once at ~5 TB/s, one launch
        return (double)(m * k * 2 + k * 32 + m * n * 4) / 5.0e12 + 5e-6;
    if (few_rows_ok(ta, tb, m, n, k, batch)) // B streamed once
        return (double)(n * k * 2) / 3.7e12 + 3.5e-6;
    double t = 0.0;
    plan_gemm(ta, tb, m, n, k_inkernel(ta, tb, k), batch, cu_budget, &t);
    return t;
}

extern "C" int pgk_gemm16(int dtype, int ta, int tb, size_t m, size_t n, size_t k, const uint16_t *a, size_t lda,
                          size_t stride_a, size_t a_extent, const uint16_t *b, size_t ldb, size_t stride_b,
                          size_t b_extent, float *c, size_t ldc, size_t stride_c, size_t batch, int beta,
                          const pgk_epi *epi, void *ws, pgk_stream s)
{
    return pgk_gemm16_cu(dtype, ta, tb, m, n, k, a, lda, stride_a, a_extent, b, ldb, stride_b, b_extent, c, ldc,
                         stride_c, batch, beta, epi, ws, 0, s);
}

extern "C" int pgk_gemm16_cu(int dtype, int ta, int tb, size_t m, size_t n, size_t k, const uint16_t *a, size_t lda,
                             size_t stride_a, size_t a_extent, const uint16_t *b, size_t ldb, size_t stride_b,
                             size_t b_extent, float *c, size_t ldc, size_t stride_c, size_t batch, int beta,
                             const pgk_epi *epi, void *ws, int cu_budget, pgk_stream s)
{
    if (!m || !n || !batch)
        return 0;
    const bool has_epi = epi && (epi->bias || epi->act != PGK_ACT_NONE || epi->z || epi->c16);
    // of a batch only the 16-bit form, where one launch finishes it
    const bool only16 = has_epi && epi->c16 && epi->skip_out && !epi->bias && epi->act == PGK_ACT_NONE && !epi->z;
    if (has_epi && (beta || (batch != 1 && !only16) || (epi->c16 && epi->dtype16 != 1 && epi->dtype16 != 2)))
        return (int)hipErrorInvalidValue;
    // an unwritten C needs the epilogue on the GEMM or the split-K sum: the
    // k-tail and empty-k paths apply it over C's accumulated values
    if (has_epi && epi->skip_out && (!k || k_inkernel(ta, tb, k) != k))
        return (int)hipErrorInvalidValue;
    const int bad = check_gemm_args(ta, tb, m, n, k, a, lda, stride_a, a_extent, b, ldb, stride_b, b_extent, batch);
    if (bad)
        return bad;
    hipStream_t st = (hipStream_t)s;
    const int f16 = dtype == 1;
    const size_t kmain = k_inkernel(ta, tb, k), ktail = k - kmain;
    const size_t mn = m * n;
    const unsigned gmn = (unsigned)((mn + 255) / 256 < 2048 ? (mn + 255) / 256 : 2048);
    if (!k) { // empty reduction: C = beta ? C : 0
        if (!beta)
            hipLaunchKernelGGL(k_zero_rows, dim3(gmn, 1, (unsigned)batch), dim3(256), 0, st, c, ldc, stride_c,
                               (int)m, (int)n);
        if (has_epi)
            hipLaunchKernelGGL(k_bias_act, dim3(gmn), dim3(256), 0, st, c, ldc, (int)m, (int)n, *epi);
        return (int)hipGetLastError();
    }
    if (skinny_ok(ta, tb, m, n, k, batch)) {
        const dim3 grid((unsigned)((m + 15) / 16));
        const pgk_epi e = has_epi ? *epi : pgk_epi{};
        const int he = has_epi ? 1 : 0;
        if (ta) {
            if (f16)
                hipLaunchKernelGGL((k_skinny<true, true>), grid, dim3(kSkWaves * 64), 0, st, a, lda, (int)a_extent, b, ldb,
                                   (int)b_extent, c, ldc, (int)m, (int)n, (int)k, beta, e, he);
            else
                hipLaunchKernelGGL((k_skinny<true, false>), grid, dim3(kSkWaves * 64), 0, st, a, lda, (int)a_extent, b, ldb,
                                   (int)b_extent, c, ldc, (int)m, (int)n, (int)k, beta, e, he);
        } else {
            if (f16)
                hipLaunchKernelGGL((k_skinny<false, true>), grid, dim3(kSkWaves * 64), 0, st, a, lda, (int)a_extent, b, ldb,
                                   (int)b_extent, c, ldc, (int)m, (int)n, (int)k, beta, e, he);
            else
                hipLaunchKernelGGL((k_skinny<false, false>), grid, dim3(kSkWaves * 64), 0, st, a, lda, (int)a_extent, b, ldb,
                                   (int)b_extent, c, ldc, (int)m, (int)n, (int)k, beta, e, he);
        }
        return (int)hipGetLastError();
    }
    if (few_rows_ok(ta, tb, m, n, k, batch)) {
        gemm_args g = {a, lda, 0, (int)a_extent, b, ldb, 0, (int)b_extent, c, ldc, 0, (int)m, (int)n, (int)k, beta, 1u};
        const gemm_kargs kg = make_kargs<gcfg<64, 64, 1, 1, false, true, false, false, 64, 2>>(g, has_epi ? *epi : pgk_epi{});
        const dim3 grid((unsigned)((n + kFrTile - 1) / kFrTile), (unsigned)((m + kFrTile - 1) / kFrTile));
        if (f16)
            hipLaunchKernelGGL(k_few_rows<true>, grid, dim3(kFrWaves * 64), 0, st, kg, (int)has_epi);
        else
            hipLaunchKernelGGL(k_few_rows<false>, grid, dim3(kFrWaves * 64), 0, st, kg, (int)has_epi);
        return (int)hipGetLastError();
    }
    const gemm_plan pl = plan_gemm(ta, tb, m, n, kmain, batch, cu_budget);
    const int sp = pl.sp > 1 ? pl.sp : 0;
    // the epilogue rides on the GEMM when one launch of the forward layout
    // finishes C, on the split-K sum when that finishes C, otherwise it is
    // a pass over C afterwards
    if ((sp || ktail) && !ws)
        return (int)hipErrorInvalidValue;
    if (pl.tile >= 5 && kmain) {
        const bool fused = has_epi && !ktail;
        gemm_args g = {a, lda, stride_a, (int)a_extent, b, ldb, stride_b, (int)b_extent, c, ldc, stride_c,
                       (int)m, (int)n, (int)kmain, beta, (unsigned)batch, pl.tile};
        const int rc = launch_ks_any(f16, ta, tb, g, fused ? *epi : pgk_epi{}, fused, st);
        if (rc || fused || (!ktail && !has_epi))
            return rc;
    } else if (has_epi && !sp && !ktail && (tb || !ta)) {
        // a forward product's epilogue, or a grad's rounded to 16 bits
        gemm_args g = {a, lda, stride_a, (int)a_extent, b, ldb, stride_b, (int)b_extent, c, ldc, stride_c,
                       (int)m, (int)n, (int)kmain, 0, (unsigned)batch, pl.tile};
        if (!tb)
            return f16 ? launch_layout<false, false, true, true>(g, st, *epi)
                       : launch_layout<false, false, false, true>(g, st, *epi);
        if (ta)
            return f16 ? launch_layout<true, true, true, true>(g, st, *epi)
                       : launch_layout<true, true, false, true>(g, st, *epi);
        return f16 ? launch_layout<false, true, true, true>(g, st, *epi)
                   : launch_layout<false, true, false, true>(g, st, *epi);
    }
    const size_t part_bytes = sp ? (((size_t)sp * m * n * sizeof(float) + 255) & ~(size_t)255) : 0;
    int rc = 0;
    if (pl.tile >= 5) {
        // queued above; a k tail and its epilogue follow
    } else if (kmain && sp) {
        // slice z covers k in [z * ks, min(kmain, (z + 1) * ks)): operand
        // offsets along the reduction, dense [m, n] partials
        const size_t ks = ((kmain + sp - 1) / sp + BK - 1) / BK * BK;
        float *part = (float *)ws;
        gemm_args g = {a, lda, ta ? ks * lda : ks, (int)a_extent, b, ldb, tb ? ks * ldb : ks, (int)b_extent, part, n,
                       m * n, (int)m, (int)n, (int)ks, 0, (unsigned)sp, pl.tile, (int)kmain, (int)ks};
        rc = launch_any(f16, ta, tb, g, st);
        if (rc)
            return rc;
        // the epilogue rides on the sum when nothing is added to C after it
        const splitk_desc sd = splitk_of(part, sp, m, n, c, ldc, beta, has_epi && !ktail ? epi : nullptr);
        hipLaunchKernelGGL(k_splitk_sum, splitk_grid(sd, sd), dim3(256), 0, st, sd, sd);
        rc = (int)hipGetLastError();
        if (rc || (has_epi && !ktail))
            return rc;
    } else if (kmain) {
        gemm_args g = {a, lda, stride_a, (int)a_extent, b, ldb, stride_b, (int)b_extent, c, ldc, stride_c,
                       (int)m, (int)n, (int)kmain, beta, (unsigned)batch, pl.tile};
        rc = launch_any(f16, ta, tb, g, st);
        if (rc)
            return rc;
    }
    if (ktail) {
        // (k % 8 != 0) last k-slab of each operand, zero-padded to 64 (and to
        // a multiple of 8 columns for an MN-contiguous copy), then one more
        // launch
        const size_t ma = ta ? (((m + 7) & ~(size_t)7) < 8 ? 8 : ((m + 7) & ~(size_t)7)) : m;
        const size_t nbp = tb ? (((n + 7) & ~(size_t)7) < 8 ? 8 : ((n + 7) & ~(size_t)7)) : n;
        uint16_t *pa = (uint16_t *)((char *)ws + part_bytes);
        const size_t asz = 64 * ma;
        uint16_t *pb = pa + ((asz * batch + 63) & ~(size_t)63);
        const size_t bsz = 64 * nbp;
        const unsigned ga = (unsigned)((asz + 255) / 256 < 4096 ? (asz + 255) / 256 : 4096);
        const unsigned gb = (unsigned)((bsz + 255) / 256 < 4096 ? (bsz + 255) / 256 : 4096);
        hipLaunchKernelGGL(k_pack_slab, dim3(ga, 1, (unsigned)batch), dim3(256), 0, st, ta, a, lda, stride_a, (int)m,
                           (int)ma, (int)kmain, (int)ktail, pa, asz);
        hipLaunchKernelGGL(k_pack_slab, dim3(gb, 1, (unsigned)batch), dim3(256), 0, st, tb, b, ldb, stride_b, (int)n,
                           (int)nbp, (int)kmain, (int)ktail, pb, bsz);
        rc = (int)hipGetLastError();
        if (rc)
            return rc;
        gemm_args g = {pa, ta ? ma : (size_t)64, asz, (int)(ta ? ma : m), pb, tb ? nbp : (size_t)64, bsz,
                       (int)(tb ? nbp : n), c, ldc, stride_c, (int)m, (int)n, BK, kmain ? 1 : beta,
                       (unsigned)batch};
        rc = launch_any(f16, ta, tb, g, st);
        if (rc)
            return rc;
    }
    if (has_epi) {
        hipLaunchKernelGGL(k_bias_act, dim3(gmn), dim3(256), 0, st, c, ldc, (int)m, (int)n, *epi);
        return (int)hipGetLastError();
    }
    return 0;
}

// Without a workspace: the split-over-waves tile by its block count alone, for
// a caller whose fixed workspace cannot hold the faster plan's partials
extern "C" int pgk_gemm16_lean_tile(int ta, int tb, size_t m, size_t n, size_t k, size_t batch)
{
    return m && n && batch && k && k_inkernel(ta, tb, k) == k ? ks_tile({{m, n, batch, k}}, ta && tb, true) : 0;
}

extern "C" int pgk_gemm16_lean(int dtype, int ta, int tb, size_t m, size_t n, size_t k, const uint16_t *a, size_t lda,
                               size_t stride_a, size_t a_extent, const uint16_t *b, size_t ldb, size_t stride_b,
                               size_t b_extent, float *c, size_t ldc, size_t stride_c, size_t batch, int beta,
                               pgk_stream s)
{
    const int tile = pgk_gemm16_lean_tile(ta, tb, m, n, k, batch);
    const int bad = check_gemm_args(ta, tb, m, n, k, a, lda, stride_a, a_extent, b, ldb, stride_b, b_extent, batch);
    if (!tile || bad)
        return bad ? bad : (int)hipErrorInvalidValue;
    const gemm_args g = {a, lda, stride_a, (int)a_extent, b, ldb, stride_b, (int)b_extent, c, ldc, stride_c,
                         (int)m, (int)n, (int)k, beta, (unsigned)batch, tile};
    return launch_ks_any(dtype == 1, ta, tb, g, pgk_epi{}, 0, (hipStream_t)s);
}

extern "C" size_t pgk_gemm16_pair_dw_workspace(const pgk_gemm_desc *d, const pgk_gemm_desc *w, int cu_d, size_t *off_w)
{
    const size_t wd = pgk_gemm16_workspace_cu(0, 0, d->m, d->n, d->k, d->batch, cu_d);
    *off_w = (wd + 255) & ~(size_t)255;
    return *off_w + pgk_gemm16_workspace_cu(1, 1, w->m, w->n, w->k, w->batch, kCUs - cu_d);
}

extern "C" int pgk_gemm16_pair_dw(int dtype, const pgk_gemm_desc *d, const pgk_gemm_desc *w, int cu_d, void *ws,
                                  pgk_stream s)
{
    if (cu_d < 0 || cu_d >= kCUs || !d->m || !d->n || !d->batch || !w->m || !w->n || !w->batch || !d->k || !w->k)
        return PGK_GEMM_NOT_PAIRED;
    int bad = check_gemm_args(0, 0, d->m, d->n, d->k, d->a, d->lda, d->stride_a, d->a_extent, d->b, d->ldb,
                              d->stride_b, d->b_extent, d->batch);
    if (!bad)
        bad = check_gemm_args(1, 1, w->m, w->n, w->k, w->a, w->lda, w->stride_a, w->a_extent, w->b, w->ldb,
                              w->stride_b, w->b_extent, w->batch);
    if (bad)
        return bad;
    // one launch covers each problem: no k tail, one tile size for both (a
    // skinny wgrad runs alone)
    if (k_inkernel(0, 0, d->k) != d->k || k_inkernel(1, 1, w->k) != w->k ||
        skinny_ok(1, 1, w->m, w->n, w->k, w->batch))
        return PGK_GEMM_NOT_PAIRED;
    const gemm_plan pd = plan_gemm(0, 0, d->m, d->n, d->k, d->batch, cu_d), pw = plan_gemm(1, 1, w->m, w->n, w->k, w->batch,
                                                                                      kCUs - cu_d);
    if (pd.tile != pw.tile || pd.tile >= 5)
        return PGK_GEMM_NOT_PAIRED;
    size_t off_w = 0;
    pgk_gemm16_pair_dw_workspace(d, w, cu_d, &off_w);
    if ((pd.sp > 1 || pw.sp > 1) && !ws)
        return (int)hipErrorInvalidValue;
    // a split problem writes its slices' partials to its workspace part;
    // one summing launch then adds both problems' slices in order
    auto args = [&](const pgk_gemm_desc *x, int ta, int tb, const gemm_plan &pl, float *part) {
        gemm_args g = {x->a, x->lda, x->stride_a, (int)x->a_extent, x->b, x->ldb, x->stride_b, (int)x->b_extent,
                       x->c, x->ldc, x->stride_c, (int)x->m, (int)x->n, (int)x->k, x->beta, (unsigned)x->batch,
                       pl.tile};
        if (pl.sp > 1) {
            const size_t ks = ((x->k + pl.sp - 1) / pl.sp + BK - 1) / BK * BK;
            g.sa = ta ? ks * x->lda : ks, g.sb = tb ? ks * x->ldb : ks;
            g.c = part, g.ldc = x->n, g.sc = x->m * x->n, g.k = (int)ks, g.beta = 0, g.batch = (unsigned)pl.sp;
            g.k_total = (int)x->k, g.kz_step = (int)ks;
        }
        return g;
    };
    float *part_d = (float *)ws, *part_w = (float *)((char *)ws + off_w);
    const gemm_args gd = args(d, 0, 0, pd, part_d), gw = args(w, 1, 1, pw, part_w);
    hipStream_t st = (hipStream_t)s;
    int rc = dtype == 1 ? launch_pair_tiles<true>(pd.tile, gd, gw, st) : launch_pair_tiles<false>(pd.tile, gd, gw, st);
    if (rc || (pd.sp <= 1 && pw.sp <= 1))
        return rc;
    const splitk_desc s1 = pd.sp > 1 ? splitk_of(part_d, pd.sp, d->m, d->n, d->c, d->ldc, d->beta) : splitk_desc{};
    const splitk_desc s2 = pw.sp > 1 ? splitk_of(part_w, pw.sp, w->m, w->n, w->c, w->ldc, w->beta) : splitk_desc{};
    hipLaunchKernelGGL(k_splitk_sum, splitk_grid(s1, s2), dim3(256), 0, st, s1, s2);
    return (int)hipGetLastError();
}

// The slices of the dgrad in k_gemm16_grads, 0 when the two products are better
// alone.  Depths in the reduction, a block costing its own and some 800 of
// start and epilogue; the dgrad's blocks run first, the wgrad's fill the CUs
// that they leave; a launch takes some 8 us per 1024 of its longest CU and 10
// more per 1024 of the mean, a sum 5 us and its bytes at 5 TB/s.  Together
// against alone, M x K x F (dgrad of depth 2F, wgrad of depth M), us:
//   512 x 1024 x 4096   36 : 46      1024 x 768 x 2048   28 : 40
//   1023 x 777 x 2049   37 : 51      2048 x 1024 x 2048  46 : 66
//   256 x 2048 x 4096   44 : 51      512 x 4096 x 1024   34 : 43
//   2048 x 2048 x 2048  75 : 92      4096 x 1024 x 4096 157 : 178
//   20 x 1024 x 8192    35 : 50      1000 x 1000 x 3001  46 : 66
// and with more work than the last the larger tiles of the products alone
// gain on it (2048 x 2048 x 4096 172 : 168); with few tiles of either, or where
// both are small enough for the split-over-waves tiles, it loses (100 x 512 x
// 2048 23 : 17, 512 x 512 x 2048 24 : 20, 8192 x 256 x 512 83 : 37).
static int grads_plan(const pgk_gemm_desc *d, const pgk_gemm_desc *w)
{
    const size_t nd = ((d->m + 127) / 128) * ((d->n + 255) / 256);
    const size_t nw = ((w->m + 127) / 128) * ((w->n + 255) / 256) * w->batch;
    if (d->batch != 1 || nd < 4 || nw < 64 || nd * d->k + nw * w->k > (size_t)8192 * kCUs ||
        (ks_tile({{d->m, d->n, 1, d->k}}, false) && ks_tile({{w->m, w->n, w->batch, w->k}}, true)))
        return 0;
    int best = 0;
    double best_t = 1e300;
    for (int sp : {1, 2, 3, 4, 6, 8}) {
        const size_t ks = ((d->k + sp - 1) / sp + BK - 1) / BK * BK, n1 = nd * sp;
        if (ks * (size_t)(sp - 1) >= d->k)
            break; // the last slice would be empty
        const double a = (double)ks + 800, b = (double)w->k + 800;
        // CUs with one dgrad block more than the rest, and the time at which
        // all the wgrad's blocks have had their place
        const double r = (double)(n1 / kCUs), more = (double)(n1 % kCUs), la = (r + (more > 0 ? 1 : 0)) * a, lb = r * a;
        double ca = la, cb = lb + ceil((la - lb) / b) * b, t = la;
        while (more * floor((t - la) / b) + (kCUs - more) * floor((t - lb) / b) < (double)nw) {
            (ca <= cb ? ca : cb) += b;
            t = ca < cb ? ca : cb;
        }
        t = (t * 8e-6 + ((double)n1 * a + (double)nw * b) / kCUs * 10e-6) / 1024;
        if (sp > 1)
            t += 5e-6 + 2.0 * sp * (double)d->m * (double)d->n * 4.0 / 5.0e12;
        if (t < best_t) {
            best_t = t;
            best = sp;
        }
    }
    return nd * best < 32 ? 0 : best;
}

extern "C" size_t pgk_gemm16_grads_workspace(const pgk_gemm_desc *d, const pgk_gemm_desc *w)
{
    const int sp = grads_plan(d, w);
    return sp > 1 ? (size_t)sp * d->m * d->n * sizeof(float) : 0;
}

extern "C" int pgk_gemm16_grads(int dtype, const pgk_gemm_desc *d, uint16_t *d16, const pgk_gemm_desc *w, uint16_t *w16,
                                void *ws, pgk_stream s)
{
    if (d->beta || w->beta || !d->m || !d->n || !d->k || !w->m || !w->n || !w->k || !w->batch || d->k % 8)
        return PGK_GEMM_NOT_PAIRED;
    const int sp = grads_plan(d, w);
    if (!sp)
        return PGK_GEMM_NOT_PAIRED;
    int bad = check_gemm_args(0, 0, d->m, d->n, d->k, d->a, d->lda, d->stride_a, d->a_extent, d->b, d->ldb,
                              d->stride_b, d->b_extent, d->batch);
    if (!bad)
        bad = check_gemm_args(1, 1, w->m, w->n, w->k, w->a, w->lda, w->stride_a, w->a_extent, w->b, w->ldb,
                              w->stride_b, w->b_extent, w->batch);
    if (bad || (sp > 1 && !ws))
        return bad ? bad : (int)hipErrorInvalidValue;
    pgk_epi ed = {}, ew = {};
    if (w16)
        ew.c16 = w16, ew.dtype16 = dtype, ew.skip_out = 1;
    if (d16)
        ed.c16 = d16, ed.dtype16 = dtype, ed.skip_out = 1;
    const gemm_args gw = {w->a, w->lda, w->stride_a, (int)w->a_extent, w->b, w->ldb, w->stride_b, (int)w->b_extent, w->c,
                          w->ldc, w->stride_c, (int)w->m, (int)w->n, (int)w->k, 0, (unsigned)w->batch, 3};
    gemm_args gd = {d->a, d->lda, 0, (int)d->a_extent, d->b, d->ldb, 0, (int)d->b_extent, d->c, d->ldc, 0, (int)d->m,
                    (int)d->n, (int)d->k, 0, 1u, 3};
    hipStream_t st = (hipStream_t)s;
    float *const part = (float *)ws;
    if (sp > 1) {
        const size_t ks = ((d->k + sp - 1) / sp + BK - 1) / BK * BK;
        gd.sa = gd.sb = ks, gd.c = part, gd.ldc = d->n, gd.sc = d->m * d->n, gd.k = (int)ks, gd.batch = (unsigned)sp;
        gd.k_total = (int)d->k, gd.kz_step = (int)ks;
    }
    const pgk_epi e1 = sp > 1 ? pgk_epi{} : ed;
    int rc = dtype == 1 ? launch_grads<true>(gd, e1, gw, ew, st) : launch_grads<false>(gd, e1, gw, ew, st);
    if (rc || sp == 1)
        return rc;
    const splitk_desc sd = splitk_of(part, sp, d->m, d->n, d->c, d->ldc, 0, d16 ? &ed : nullptr);
    hipLaunchKernelGGL(k_splitk_sum, splitk_grid(sd, sd), dim3(256), 0, st, sd, sd);
    return (int)hipGetLastError();
}

extern "C" int pgk_gemm16_ks_pair_tile(const pgk_gemm_desc *d, const pgk_gemm_desc *w)
{
    if (!d->m || !d->n || !d->k || !d->batch || !w->m || !w->n || !w->k || !w->batch || d->k % 8 ||
        skinny_ok(1, 1, w->m, w->n, w->k, w->batch))
        return 0;
    return ks_tile({{d->m, d->n, d->batch, d->k}, {w->m, w->n, w->batch, w->k}}, false);
}

extern "C" int pgk_gemm16_ks_pair(int dtype, const pgk_gemm_desc *d, const pgk_gemm_desc *w, pgk_stream s)
{
    const int tile = pgk_gemm16_ks_pair_tile(d, w);
    if (!tile)
        return PGK_GEMM_NOT_PAIRED;
    int bad = check_gemm_args(0, 0, d->m, d->n, d->k, d->a, d->lda, d->stride_a, d->a_extent, d->b, d->ldb,
                              d->stride_b, d->b_extent, d->batch);
    if (!bad)
        bad = check_gemm_args(1, 1, w->m, w->n, w->k, w->a, w->lda, w->stride_a, w->a_extent, w->b, w->ldb,
                              w->stride_b, w->b_extent, w->batch);
    if (bad)
        return bad;
    auto args = [&](const pgk_gemm_desc *x) {
        return gemm_args{x->a, x->lda, x->stride_a, (int)x->a_extent, x->b, x->ldb, x->stride_b, (int)x->b_extent,
                         x->c, x->ldc, x->stride_c, (int)x->m, (int)x->n, (int)x->k, x->beta, (unsigned)x->batch, tile};
    };
    const gemm_args gd = args(d), gw = args(w);
    return dtype == 1 ? launch_ks_pair_tile<true>(tile, gd, gw, (hipStream_t)s)
                      : launch_ks_pair_tile<false>(tile, gd, gw, (hipStream_t)s);
}

extern "C" int pgk_mfma_probe(int lds, float *sink, size_t sink_floats, int blocks, int iters, pgk_stream s)
{
    if (blocks < 1 || iters < 2 || (iters & 1) || sink_floats < (size_t)blocks * 512)
        return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(k_mfma_probe, dim3((unsigned)blocks), dim3(512), 0, (hipStream_t)s, sink, iters, lds);
    return (int)hipGetLastError();
}
