// The tiled products' device code, shared by the kernel files: operand tiles
// (TileK, TileMN), the block of the LDS-ring GEMM (gemm16_block) and the
// block of the split-over-waves GEMM (ks_block).  The data path is described
// at the top of gemm.hip.
#ifndef PGK_GEMM_TILE_H
#define PGK_GEMM_TILE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include <initializer_list>
#include <type_traits>

#include "convert16.h"
#include "gate_act.h"
#include "launch.h"
#include "pgmath.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
#define LDS __attribute__((address_space(3)))

// alignment of split-K slices and of the zero-padded k-tail slabs: a
// multiple of every kernel k-tile depth (32 and 64)
constexpr int BK = 64;

__device__ __forceinline__ float act_f(int act, float v)
{
    if (act == PGK_ACT_RELU)
        return v > 0.0f ? v : 0.0f;
    if (act == PGK_ACT_GELU)
        return pgm_gelu(v);
    return v;
}

// s_waitcnt immediate waiting for vmcnt <= n and lgkmcnt == 0 (gfx9
// encoding: vmcnt in bits 3:0 and 15:14, expcnt 6:4 left at its maximum,
// lgkmcnt 11:8)
constexpr int vmcnt_lgkm0_imm(int n) { return (n & 0xF) | 0x70 | (((n >> 4) & 3) << 14); }

template <bool F16>
__device__ __forceinline__ f32x16 mfma32(const uint4 &a, const uint4 &b, const f32x16 &c)
{
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// One wave's 64 x 16-byte global -> LDS copy: lane i's bytes land at
// M0 + 16 i.  Issued as asm so the compiler's wait insertion does not
// track it (it would otherwise drain every such load before the next LDS
// read); the k-loop waits on these loads explicitly.  M0 is reserved to
// the compiler, which therefore ignores a clobber of it: the GEMM kernels
// below generate no other M0 use (checked on their gfx950 assembly), so
// writing it here disturbs nothing.  An SALU write of M0 needs one wait
// state before an LDS DMA reads it (a gfx9 hazard the compiler's hazard
// recognizer cannot see inside asm): the s_nop.
__device__ __forceinline__ void dma16(const void *src, LDS uint4 *dst)
{
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}

// The same copy from a wave-uniform base address in SGPRs plus a 32-bit
// per-lane byte offset: the form for k-tiles that lie wholly below the end
// of the reduction dim, whose per-lane offsets stay fixed from tile to tile
// (only the scalar base moves), so the loop spends no vector ALU work on
// addresses.  `sbase` must be wave-uniform and the compiler must keep it in
// SGPRs: if a change to the kernel leads it to compute the base in VGPRs,
// the assembler rejects the instruction and the build fails.  (Forcing it
// with v_readfirstlane costs two VALU ops per load in the k-loop; when doing
// so, zero-extend each 32-bit half: the builtin returns a signed int.)
__device__ __forceinline__ void dma16s(uint32_t voff, const void *sbase, LDS uint4 *dst)
{
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(voff), "s"(sbase)
                     : "memory");
}

// 16 zero bytes in global memory: the DMA source of every chunk past the
// end of the reduction dim, so a partial last k-tile lands zero-filled
__device__ const uint4 g_zero16 = {0u, 0u, 0u, 0u};

// leading dims under this take the fast loads below: their 32-bit lane
// offsets span at most 16 rows
constexpr size_t kFastLd = (size_t)1 << 26;

// K-contiguous operand tile: ROWS x KB (KB = 64 or 32), rows of KB / 8
// 16-byte chunks.  Load instruction q of wave w fills chunk slots
// (w NQ + q) 64 .. + 63.  Chunks are XOR-swizzled within a row so the 16
// lanes of each ds_read_b128 pass hit 16 different bank groups: by
// (r ^ r >> 3) & 7 for 8-chunk rows, by (r >> 2) & 3 for 4-chunk rows (four
// 64-byte rows share a 256-byte bank window).
template <int ROWS, int NT, int KB>
struct TileK {
    static constexpr int CH = KB / 8;
    static constexpr int NQ = ROWS * CH / NT;
    static_assert(ROWS * CH % NT == 0, "tile slots must divide by the thread count");
    static_assert(KB == 64 || KB == 32, "k depth");
    __device__ __forceinline__ static int swz(int chunk, int row)
    {
        return CH == 8 ? chunk ^ ((row ^ (row >> 3)) & 7) : chunk ^ ((row >> 2) & 3);
    }

    // rows past `extent` are clamped to its last row (their results are
    // never stored); 1 <= extent
    // chunks at k >= kend read zeros (kend % 8 == 0)
    __device__ __forceinline__ static void load_q(int q, const uint16_t *__restrict__ p, size_t ld, int row0,
                                                  int extent, int k0, int kend, LDS uint4 *dst, int tid)
    {
        const int lane = tid & 63, wave = tid >> 6;
        const int base = (wave * NQ + q) * 64;
        const int slot = base + lane;
        const int row = slot / CH;
        const int logical = swz(slot % CH, row);
        int gr = row0 + row;
        gr = gr < extent ? gr : extent - 1;
        const int kc = k0 + logical * 8;
        const void *src = kc < kend ? (const void *)(p + (size_t)gr * ld + kc) : (const void *)&g_zero16;
        dma16(src, dst + base);
    }
    // Fast form of load q (k-tiles below kend): the scalar base is row
    // `srow` (the first row load q touches, clamped like the rows) and each
    // lane's offset is (its clamped row - srow) ld + its chunk, in bytes;
    // the 64 lanes span 64 / CH rows, so the offset fits 32 bits for
    // ld < kFastLd.  `wave` must be wave-uniform.
    struct Fast {
        uint32_t voff;
        int srow;
    };
    __device__ __forceinline__ static Fast fast_q(int q, size_t ld, int row0, int extent, int wave, int lane)
    {
        const int base = (wave * NQ + q) * 64;
        const int qrow = row0 + base / CH;
        const int srow = qrow < extent ? qrow : extent - 1;
        const int slot = base + lane;
        const int row = slot / CH;
        const int logical = swz(slot % CH, row);
        int gr = row0 + row;
        gr = gr < extent ? gr : extent - 1;
        return {(uint32_t)((size_t)(gr - srow) * ld * 2 + (size_t)logical * 16), srow};
    }
    __device__ __forceinline__ static void load_fast(int q, const Fast &f, const uint16_t *__restrict__ p, size_t ld,
                                                     int /*row0*/, int k0, LDS uint4 *dst, int wave)
    {
        dma16s(f.voff, p + (size_t)f.srow * ld + k0, dst + (wave * NQ + q) * 64);
    }

    // MFMA operand fragment: rows r0 + lane % 32, k = 16 s + 8 (lane / 32) .. + 7
    __device__ __forceinline__ static uint4 frag(const LDS uint4 *sm, int r0, int s, int lane)
    {
        const int r = r0 + (lane & 31);
        const u32x4 v = ((const LDS u32x4 *)sm)[r * CH + swz(2 * s + (lane >> 5), r)];
        return __builtin_bit_cast(uint4, v);
    }
};

// MN-contiguous operand tile: held as [KB][ROWS] (k-major rows of ROWS
// values), 16-byte chunks swizzled by 4 (k & 3) so the k-rows one
// transposing read touches fall in distinct banks.
template <int ROWS, int NT, int KB>
struct TileMN {
    static constexpr int CPR = ROWS / 8;
    static constexpr int NQ = KB * CPR / NT;
    static_assert(KB * CPR % NT == 0, "tile slots must divide by the thread count");
    static_assert(CPR >= 16 || CPR == 8 || CPR == 4, "the swizzle permutes the 64-byte windows of a row");
    // chunk swizzle of row k: the 64-byte windows of rows k = 0..3 (mod 4)
    // land on four different quarters of the 64 banks, so the 8 rows x 64
    // bytes one ds_read_b64_tr_b16 touches take the minimum two passes (two
    // rows of 128 bytes, or four of 64, already span the banks)
    __device__ __forceinline__ static int fk(int k)
    {
        return CPR >= 16 ? (k & 3) << 2 : CPR == 8 ? (k >> 1 & 1) << 2 : 0;
    }

    // columns past `extent` are clamped to its last 8 (never stored);
    // extent % 8 == 0, extent >= 8
    // k-rows at k >= kend read zeros
    __device__ __forceinline__ static void load_q(int q, const uint16_t *__restrict__ p, size_t ld, int row0,
                                                  int extent, int k0, int kend, LDS uint4 *dst, int tid)
    {
        const int lane = tid & 63, wave = tid >> 6;
        const int base = (wave * NQ + q) * 64;
        const int slot = base + lane;
        const int k = slot / CPR;
        const int logical = (slot % CPR) ^ fk(k);
        int mn = row0 + logical * 8;
        mn = mn < extent ? mn : extent - 8;
        const void *src =
            k0 + k < kend ? (const void *)(p + (size_t)(k0 + k) * ld + mn) : (const void *)&g_zero16;
        dma16(src, dst + base);
    }
    // Fast form of load q (k-tiles below kend): the scalar base is k-row
    // k0 + kq (the first k-row load q touches), column row0, and each lane's
    // offset is (its k-row - kq) ld + (its clamped column - row0), in bytes;
    // the 64 lanes span 64 / CPR k-rows, at most 16, so leading dims under
    // kFastLd keep it within 32 bits.  `wave` must be wave-uniform.
    static_assert((uint64_t)(64 / CPR > 1 ? 64 / CPR - 1 : 1) * kFastLd * 2 + ROWS * 2 < ((uint64_t)1 << 32),
                  "a load's lane offsets fit 32 bits");
    struct Fast {
        uint32_t voff;
        int srow;
    };
    __device__ __forceinline__ static Fast fast_q(int q, size_t ld, int row0, int extent, int wave, int lane)
    {
        const int base = (wave * NQ + q) * 64;
        const int kq = base / CPR;
        const int slot = base + lane;
        const int k = slot / CPR;
        const int logical = (slot % CPR) ^ fk(k);
        int mn = row0 + logical * 8;
        mn = mn < extent ? mn : extent - 8;
        return {(uint32_t)(((size_t)(k - kq) * ld + (size_t)(mn - row0)) * 2), kq};
    }
    __device__ __forceinline__ static void load_fast(int q, const Fast &f, const uint16_t *__restrict__ p, size_t ld,
                                                     int row0, int k0, LDS uint4 *dst, int wave)
    {
        dma16s(f.voff, p + (size_t)(k0 + f.srow) * ld + row0, dst + (wave * NQ + q) * 64);
    }

    // MFMA operand fragment from two ds_read_b64_tr_b16: in 16-lane group g
    // source lane q points at [k0 + q / 4][R0 + 4 (q % 4)] and result lane i
    // holds rows R0 + i, k = k0 .. k0 + 3 (R0 = r0 + 16 (g & 1),
    // k0 = 16 s + 8 (g >> 1) + 4 h for half h)
    __device__ __forceinline__ static uint4 frag(const LDS uint4 *sm, int r0, int s, int lane)
    {
        const int g = (lane >> 4) & 3, q = lane & 15;
        const int mn = r0 + 16 * (g & 1) + 4 * (q & 3);
        uint2 h2[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 16 * s + 8 * (g >> 1) + 4 * h + (q >> 2);
            const int byte = k * ROWS * 2 + (((mn >> 3) ^ fk(k)) << 4) + (mn & 7) * 2;
            h2[h] = __builtin_bit_cast(
                uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS v4s *)((const LDS char *)sm + byte)));
        }
        return make_uint4(h2[0].x, h2[0].y, h2[1].x, h2[1].y);
    }
};

// MN-contiguous tile of a gated layer's W = [Wg | Wu] [K, 2, extent]: groups of G
// columns of Wg, each beside the same G columns of Wu, so that a block
// holds g and u of the same outputs.  Fragments are TileMN's; column row0 counts
// within either half.
template <int ROWS, int NT, int KB, int G>
struct TileGate : TileMN<ROWS, NT, KB> {
    using Base = TileMN<ROWS, NT, KB>;
    static_assert(G % 8 == 0 && ROWS % (2 * G) == 0, "whole chunks, whole pairs of groups");
    // the column of W that tile column c (a multiple of 8) is; columns past
    // `extent` of a half are clamped to its last 8 (never stored)
    __device__ __forceinline__ static int column(int c, int row0, int extent)
    {
        const int f = row0 + c / (2 * G) * G + c % G;
        return (c / G & 1) * extent + (f < extent ? f : extent - 8);
    }
    __device__ __forceinline__ static void load_q(int q, const uint16_t *__restrict__ p, size_t ld, int row0,
                                                  int extent, int k0, int kend, LDS uint4 *dst, int tid)
    {
        const int lane = tid & 63, wave = tid >> 6;
        const int base = (wave * Base::NQ + q) * 64;
        const int slot = base + lane, k = slot / Base::CPR, logical = (slot % Base::CPR) ^ Base::fk(k);
        const int mn = column(logical * 8, row0, extent);
        const void *src = k0 + k < kend ? (const void *)(p + (size_t)(k0 + k) * ld + mn) : (const void *)&g_zero16;
        dma16(src, dst + base);
    }
    using Fast = typename Base::Fast;
    // the offset is from column 0 of the k-row, within a row of W for leading
    // dims under kFastLd
    __device__ __forceinline__ static Fast fast_q(int q, size_t ld, int row0, int extent, int wave, int lane)
    {
        const int base = (wave * Base::NQ + q) * 64, kq = base / Base::CPR;
        const int slot = base + lane, k = slot / Base::CPR, logical = (slot % Base::CPR) ^ Base::fk(k);
        return {(uint32_t)(((size_t)(k - kq) * ld + (size_t)column(logical * 8, row0, extent)) * 2), kq};
    }
    __device__ __forceinline__ static void load_fast(int q, const Fast &f, const uint16_t *__restrict__ p, size_t ld,
                                                     int /*row0*/, int k0, LDS uint4 *dst, int wave)
    {
        dma16s(f.voff, p + (size_t)(k0 + f.srow) * ld, dst + (wave * Base::NQ + q) * 64);
    }
};

// A GEMM launch's arguments (one problem; a paired launch takes two).
struct gemm_kargs {
    const uint16_t *A;
    size_t lda, sA;
    int a_extent;
    const uint16_t *B;
    size_t ldb, sB;
    int b_extent;
    float *C;
    size_t ldc, sC;
    int M, N, K, beta, tiles_m, tiles_n;
    pgk_epi epi;
    int k_total, kz_step, fast_ok;
};

// one kernel configuration: block tile BM x BN on WGM x WGN waves, operand
// layouts TA / TB, f16 or bf16, fused epilogue, k-tile depth KB, S stages
// GATE: the forward of a gated layer (TB, EPI; N, b_extent and n0 count the
// columns of one half of W, a tile holds BN / 2 of them; epi.z [M, 2 N])
template <int BM_, int BN_, int WGM_, int WGN_, bool TA_, bool TB_, bool F16_, bool EPI_, int KB_, int S_, bool GATE_ = false>
struct gcfg {
    static constexpr bool GATE = GATE_;
    static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, KB = KB_, S = S_;
    static constexpr bool TA = TA_, TB = TB_, F16 = F16_, EPI = EPI_;
    static constexpr int NT = 64 * WGM * WGN;
    static constexpr int LDS_U4 = S * (BM * KB / 8 + BN * KB / 8); // uint4 of LDS
};

// Outputs of a gated layer: z = [g | u] (biases added here) and h = act(g) u, in
// f32 (c) unless skip_out and in 16 bits.  gate_store4: columns col .. col + 3 of
// the n (a multiple of 4) of row `row`, whole pieces; gate_store1: one column.
__device__ __forceinline__ bool gate_whole(const pgk_epi &epi, const float *c, int n)
{
    return (n & 3) == 0 && ((((uintptr_t)c) | (uintptr_t)epi.z) & 15) == 0 && (((uintptr_t)epi.c16) & 7) == 0;
}
__device__ __forceinline__ void gate_store4(const pgk_epi &epi, float *c, int n, int row, int col, f32x4 gv, f32x4 uv)
{
    const size_t h = (size_t)row * n + col, zg = (size_t)row * 2 * n + col;
    f32x4 o;
    if (epi.bias)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            gv[q] += epi.bias[col + q];
            uv[q] += epi.bias[n + col + q];
        }
    gate_switch(epi.act, [&](auto code) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            o[q] = gate_f<decltype(code)::value>(gv[q]) * uv[q];
    });
    if (epi.z) { // read again only by the backward, much later
        __builtin_nontemporal_store(gv, (f32x4 *)(epi.z + zg));
        __builtin_nontemporal_store(uv, (f32x4 *)(epi.z + zg + n));
    }
    if (!epi.skip_out)
        *(f32x4 *)(c + h) = o;
    if (epi.c16)
        *(uint2 *)(epi.c16 + h) = make_uint2(to16x2(epi.dtype16, o[0], o[1]), to16x2(epi.dtype16, o[2], o[3]));
}
__device__ __forceinline__ void gate_store1(const pgk_epi &epi, float *c, int n, int row, int col, float gv, float uv)
{
    const size_t h = (size_t)row * n + col, zg = (size_t)row * 2 * n + col;
    if (epi.bias) {
        gv += epi.bias[col];
        uv += epi.bias[n + col];
    }
    float o = 0.0f;
    gate_switch(epi.act, [&](auto code) { o = gate_f<decltype(code)::value>(gv) * uv; });
    if (epi.z) {
        epi.z[zg] = gv;
        epi.z[zg + n] = uv;
    }
    if (!epi.skip_out)
        c[h] = o;
    if (epi.c16)
        epi.c16[h] = to16(epi.dtype16, o);
}

// One block tile of problem g: tile pid of the nb tiles of batch entry (or
// split-K slice) z, with the LDS ring at lds.  remap: block ids were dealt
// to the 8 XCDs round-robin with pid % 8 naming the XCD.
template <class CF>
__device__ __forceinline__ void gemm16_block(const gemm_kargs &g, int pid, int nb, bool remap, int z,
                                             LDS uint4 *const lds)
{
    constexpr int BM = CF::BM, BN = CF::BN, WGM = CF::WGM, WGN = CF::WGN, KB = CF::KB, S = CF::S;
    constexpr bool TA = CF::TA, TB = CF::TB, F16 = CF::F16, EPI = CF::EPI;
    const uint16_t *__restrict__ A = g.A;
    const uint16_t *__restrict__ B = g.B;
    float *__restrict__ C = g.C;
    const size_t lda = g.lda, sA = g.sA, ldb = g.ldb, sB = g.sB, ldc = g.ldc, sC = g.sC;
    const int a_extent = g.a_extent, b_extent = g.b_extent, M = g.M, N = g.N, K = g.K, beta = g.beta;
    const int tiles_m = g.tiles_m, tiles_n = g.tiles_n, k_total = g.k_total, kz_step = g.kz_step;
    const int fast_ok = g.fast_ok;
    const pgk_epi &epi = g.epi;
    constexpr int NT = 64 * WGM * WGN;
    constexpr int WM = BM / WGM, WN = BN / WGN;
    constexpr int FM = WM / 32, FN = WN / 32;
    using OA = typename std::conditional<TA, TileMN<BM, NT, KB>, TileK<BM, NT, KB>>::type;
    constexpr bool GATE = CF::GATE;
    using OB = typename std::conditional<
        GATE, TileGate<BN, NT, KB, 32>,
        typename std::conditional<TB, TileMN<BN, NT, KB>, TileK<BN, NT, KB>>::type>::type;
    // S-stage ring of A and B tiles in one LDS block; the k-loop below is
    // unrolled by S, so every stage index is a compile-time constant
    constexpr int SA = BM * KB / 8, SB = BN * KB / 8; // uint4 per stage
    auto stA = [&](int st) { return lds + st * SA; };
    auto stB = [&](int st) { return lds + S * SA + st * SB; };

    // tile order: XCD-aware (block ids dealt round-robin to the 8 XCDs are
    // regrouped so consecutive ids share an XCD), then 8 tile-rows at a time
    if (remap && (nb & 7) == 0)
        pid = (pid & 7) * (nb >> 3) + (pid >> 3);
    const int GM = 8;
    const int per_group = GM * tiles_n;
    const int group = pid / per_group;
    const int first_m = group * GM;
    const int gsz = tiles_m - first_m < GM ? tiles_m - first_m : GM;
    const int in_group = pid - group * per_group;
    const int m0 = (first_m + in_group % gsz) * BM, n0 = (in_group / gsz) * (GATE ? BN / 2 : BN);

    const uint16_t *Ab = A + (size_t)z * sA;
    const uint16_t *Bb = B + (size_t)z * sB;
    float *Cb = C + (size_t)z * sC;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WGN, wn = wave % WGN;
    const int wave_u = __builtin_amdgcn_readfirstlane(wave);

    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[i][j][e] = 0.0f;

    // valid reduction length of this batch entry: K, or for split-K slice z
    // the rest of k_total from z * kz_step; the last partial tile reads
    // zeros past it (kend % 8 == 0)
    const int krem = k_total - z * kz_step;
    const int kend = krem < K ? krem : K;
    const int KT = (kend + KB - 1) / KB;
    // S-stage ring, tile t in stage t % S.  Between two barriers the
    // k-loop is straight-line code, so the compiler's LDS wait counts stay
    // exact: at a control-flow merge it falls back to waiting for every
    // outstanding LDS read, which would stall each wave on the fragment
    // reads it has just issued for the next k-step.
    //  - k-step s of a tile runs its MFMAs on the fragments read one step
    //    earlier and reads those of step s + 1 between them;
    //  - a tile's last k-step ("tail") starts with the one barrier per tile:
    //    every wave has then read the whole stage (its last fragments are in
    //    registers), so the stage is refilled with tile t + S during that
    //    step's MFMAs and the next tile's first fragments are read while
    //    they run -- the matrix units do not drain at the barrier;
    //  - a "link" is the tail of tile t and the other k-steps ("head") of
    //    tile t + 1, so each link starts at the barrier, whose explicit wait
    //    leaves no LDS read outstanding, and the branches between links
    //    (S per loop iteration, for constant stage offsets) cost no waits;
    //  - tiles 0 .. S-1 are in flight before the first tile and tile t + S
    //    is loaded during tile t's tail also when t + S >= KT: such tiles lie
    //    past kend and every chunk comes from the zero page (never read: no
    //    stage is read after the last tile).
    static_assert(S >= 2 && (KB / 16) % 2 == 0, "two or more stages, an even number of k-steps per tile");
    constexpr int LPT = OA::NQ + OB::NQ; // DMA instructions per thread per tile
    static_assert((S - 1) * LPT < 64, "the loads in flight fit the vmcnt counter");
    constexpr int KS = KB / 16, NM = FM * FN;
    const int links = KT > 1 ? KT - 1 : 0;
    auto dma = [&](int q, int t, LDS uint4 *dA, LDS uint4 *dB) {
        if (q < OA::NQ)
            OA::load_q(q, Ab, lda, m0, a_extent, t * KB, kend, dA, tid);
        else
            OB::load_q(q - OA::NQ, Bb, ldb, n0, b_extent, t * KB, kend, dB, tid);
    };
    // per-lane offsets of the fast form (tiles wholly below kend, leading
    // dims under kFastLd: fast_ok), fixed for the whole k-loop
    typename OA::Fast fA[OA::NQ];
    typename OB::Fast fB[OB::NQ];
#pragma unroll
    for (int q = 0; q < OA::NQ; ++q)
        fA[q] = OA::fast_q(q, lda, m0, a_extent, wave_u, lane);
#pragma unroll
    for (int q = 0; q < OB::NQ; ++q)
        fB[q] = OB::fast_q(q, ldb, n0, b_extent, wave_u, lane);
    auto dma_fast = [&](int q, int t, LDS uint4 *dA, LDS uint4 *dB) {
        if (q < OA::NQ)
            OA::load_fast(q, fA[q], Ab, lda, m0, t * KB, dA, wave_u);
        else
            OB::load_fast(q - OA::NQ, fB[q - OA::NQ], Bb, ldb, n0, t * KB, dB, wave_u);
    };
    // a bare s_barrier after an explicit wait on this wave's loads (all but
    // the newest NEWER tiles' landed in LDS) and on its LDS reads: the
    // fence of __syncthreads() would drain every outstanding memory
    // operation; the empty asm statements keep LDS accesses from moving
    // across it
    auto sync_tile = [&](auto newer) {
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(decltype(newer)::value * LPT));
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
    };
    uint4 fa[2][FM], fb[2][FN];
    auto rd = [&](const LDS uint4 *cA, const LDS uint4 *cB, int s, uint4(&xa)[FM], uint4(&xb)[FN]) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
            xa[i] = OA::frag(cA, wm * WM + i * 32, s, lane);
#pragma unroll
        for (int j = 0; j < FN; ++j)
            xb[j] = OB::frag(cB, wn * WN + j * 32, s, lane);
    };
    // MFMAs of k-step s; in a tail, tile `reload` goes into stage (dA, dB),
    // a few loads per MFMA rather than one burst at the vector-memory queue,
    // in the fast form when FAST (a compile-time tag).  With `next`, the
    // fragments of k-step ns of the tile in stage (nA, nB) are read into the
    // other fragment buffer one per MFMA, so the LDS reads spread over the
    // step instead of arriving in one burst ahead of it (wgrad's
    // transposing reads, two per fragment, gain the most).  `next` is a
    // flag rather than a null test of nA: LDS address 0 is a valid stage.
    auto mfmas = [&](int s, bool tail, int reload, LDS uint4 *dA, LDS uint4 *dB, auto fast, bool next,
                     const LDS uint4 *nA, const LDS uint4 *nB, int ns) {
        // keep the reads and loads placed here in their slots between the
        // MFMAs: left alone, the scheduler sinks each read to just before
        // its first use and the LDS latency shows at every step
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                acc[i][j] = mfma32<F16>(fa[s & 1][i], fb[s & 1][j], acc[i][j]);
                if (next) {
                    const int g = i * FN + j;
                    static_assert(FM * FN >= FM + FN, "one fragment read per MFMA at most");
                    if (g < FM)
                        fa[(s + 1) & 1][g] = OA::frag(nA, wm * WM + g * 32, ns, lane);
                    else if (g < FM + FN)
                        fb[(s + 1) & 1][g - FM] = OB::frag(nB, wn * WN + (g - FM) * 32, ns, lane);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (tail) {
                    const int g = i * FN + j;
#pragma unroll
                    for (int q = g * LPT / NM; q < (g + 1) * LPT / NM; ++q) {
                        if constexpr (decltype(fast)::value)
                            dma_fast(q, reload, dA, dB);
                        else
                            dma(q, reload, dA, dB);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    // k-steps 0 .. KS-2 of the tile in stage (cA, cB); step 0's fragments
    // are in fa[0], fb[0]
    auto head = [&](const LDS uint4 *cA, const LDS uint4 *cB) {
#pragma unroll
        for (int s = 0; s < KS - 1; ++s)
            mfmas(s, false, 0, nullptr, nullptr, std::false_type{}, true, cA, cB, s + 1);
    };
    // the tail of tile t (stage cA, cB) and the head of tile t + 1 (oA, oB)
    auto link = [&](int t, LDS uint4 *cA, LDS uint4 *cB, LDS uint4 *oA, LDS uint4 *oB, auto fast) {
        // tile t + 1 landed; tiles t + 2 .. t + S - 1 may be in flight
        sync_tile(std::integral_constant<int, S - 2>{});
        mfmas(KS - 1, true, t + S, cA, cB, fast, true, oA, oB, 0);
        head(oA, oB);
    };
#pragma unroll
    for (int t = 0; t < S; ++t)
#pragma unroll
        for (int q = 0; q < LPT; ++q)
            dma(q, t, stA(t), stB(t));
    sync_tile(std::integral_constant<int, S - 1>{}); // tile 0 landed
    rd(stA(0), stB(0), 0, fa[0], fb[0]);
    head(stA(0), stB(0));
    // link t reloads tile t + S: in the fast form while that tile lies
    // wholly below kend, for whole groups of S links (so the second loop
    // starts at stage 0), then the general form
    const int full_tiles = kend / KB;
    int fast_links = full_tiles > S ? full_tiles - S : 0;
    fast_links = fast_ok ? (fast_links < links ? fast_links : links) / S * S : 0;
    int t = 0;
    for (; t < fast_links; t += S) {
#pragma unroll
        for (int u = 0; u < S; ++u)
            link(t + u, stA(u), stB(u), stA((u + 1) % S), stB((u + 1) % S), std::true_type{});
    }
    for (; t < links; t += S) {
#pragma unroll
        for (int u = 0; u < S; ++u)
            if (t + u < links)
                link(t + u, stA(u), stB(u), stA((u + 1) % S), stB((u + 1) % S), std::false_type{});
    }
    mfmas(KS - 1, false, 0, nullptr, nullptr, std::false_type{}, false, nullptr, nullptr, 0); // the last tail
    // the loads of the tiles past the end land before the LDS is reused
    // (the epilogue's staging, or the next block on this CU)
    __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0));

    // epilogue: lane holds column lane % 32 of rows (e/4)*8 + (lane/32)*4 + e%4
    const int lrow = lane & 31, lk = lane >> 5;
    if constexpr (GATE) {
        // through LDS as below: the wave's first 32 columns are g, the others u of
        // the same 32 outputs; four outputs a lane, or one where rows of n do
        // not keep whole pieces (then neighbouring lanes store neighbours)
        static_assert(WN == 64 && EPI && TB && !TA, "one group of g and one of u per wave");
        constexpr int RS = WN + 8;
        LDS float *reg = (LDS float *)((LDS char *)lds + wave * (32 * RS * 4));
        const bool v4 = gate_whole(epi, g.C, N);
        const int cl = v4 ? (lane & 7) * 4 : lrow, col = n0 + wn * 32 + cl;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    reg[((e >> 2) * 8 + lk * 4 + (e & 3)) * RS + j * 32 + lrow] = acc[i][j][e];
            __syncthreads();
            const int grow0 = m0 + wm * WM + i * 32;
            if (col >= N)
                continue;
            if (v4) {
#pragma unroll 1
                for (int row = lane >> 3; row < 32 && grow0 + row < M; row += 8)
                    gate_store4(epi, g.C, N, grow0 + row, col, *(const LDS f32x4 *)(reg + row * RS + cl),
                                *(const LDS f32x4 *)(reg + row * RS + 32 + cl));
            } else {
#pragma unroll 1
                for (int row = lk; row < 32 && grow0 + row < M; row += 2)
                    gate_store1(epi, g.C, N, grow0 + row, col, reg[row * RS + cl], reg[row * RS + 32 + cl]);
            }
        }
    } else if constexpr (EPI) {
        // Through LDS, 32 rows of the wave's WM x WN tile at a time: the
        // accumulators land row-major in a per-wave [32][WN + 8] f32 region
        // (in the operand stages, free after the k-loop) and come back as
        // float4 along a row, so bias, activation and the three stores (out,
        // pre-activation, 16-bit out) run 4 columns per lane with 16-byte
        // (8-byte for 16-bit) stores.  Every index into acc stays static.
        static_assert(WN == 64, "one lane group of 16 x 4 columns per row");
        constexpr int RS = WN + 8;
        static_assert(WGM * WGN * 32 * RS * 4 <= S * (SA + SB) * 16, "epilogue regions fit the stages");
        LDS float *reg = (LDS float *)((LDS char *)lds + wave * (32 * RS * 4));
        const int c4 = (lane & 15) * 4;
        const int gcol = n0 + wn * WN + c4;
        float bias4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            bias4[q] = (epi.bias && gcol + q < N) ? epi.bias[gcol + q] : 0.0f;
        uint16_t *const c16 = epi.c16 ? epi.c16 + (size_t)z * sC : nullptr;
        const bool v4 = gcol + 3 < N; // at any alignment: rows of an odd width start anywhere
        typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
        typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(2)));
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            __syncthreads(); // the k-loop's (or the previous pass') LDS reads are done
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    reg[((e >> 2) * 8 + lk * 4 + (e & 3)) * RS + j * 32 + lrow] = acc[i][j][e];
            __syncthreads();
            for (int t = 0; t < 8; ++t) {
                const int row = (lane >> 4) + 4 * t;
                const int grow = m0 + wm * WM + i * 32 + row;
                if (grow >= M || gcol >= N)
                    continue;
                const f32x4 a4 = *(const LDS f32x4 *)(reg + row * RS + c4);
                const float zv[4] = {a4[0] + bias4[0], a4[1] + bias4[1], a4[2] + bias4[2], a4[3] + bias4[3]};
                float o[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    o[q] = act_f(epi.act, zv[q]);
                const size_t off = (size_t)grow * ldc + gcol;
                if (v4) {
                    if (!epi.skip_out)
                        *reinterpret_cast<f32x4u *>(Cb + off) = f32x4u{o[0], o[1], o[2], o[3]};
                    if (epi.z) { // read again only by the backward, much later
                        const f32x4u zz = {zv[0], zv[1], zv[2], zv[3]};
                        __builtin_nontemporal_store(zz, reinterpret_cast<f32x4u *>(epi.z + off));
                    }
                    if (c16) {
                        const u32x2u q2 = {to16x2(epi.dtype16, o[0], o[1]), to16x2(epi.dtype16, o[2], o[3])};
                        if constexpr (TA == TB) // a grad: past the caches, as below
                            __builtin_nontemporal_store(q2, reinterpret_cast<u32x2u *>(c16 + off));
                        else
                            *reinterpret_cast<u32x2u *>(c16 + off) = q2;
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (gcol + q >= N)
                            break;
                        if (!epi.skip_out)
                            Cb[off + q] = o[q];
                        if (epi.z)
                            epi.z[off + q] = zv[q];
                        if (c16)
                            c16[off + q] = to16(epi.dtype16, o[q]);
                    }
                }
            }
        }
    } else {
        // dgrad and wgrad outputs take non-temporal stores: the write burst
        // passes the caches by (config 3's GEMM pair 213 -> 210 us and the
        // cast pass after it faster, config 5 +1.6 %); a forward product
        // (A K-contiguous, B MN-contiguous) keeps ordinary stores, as the
        // next kernel reads it (config 5's unfused graph +1.3 %)
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int col = n0 + wn * WN + j * 32 + lrow;
                if (col >= N)
                    continue;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = m0 + wm * WM + i * 32 + (e >> 2) * 8 + lk * 4 + (e & 3);
                    if (row < M) {
                        float *p = Cb + (size_t)row * ldc + col;
                        if constexpr (!TA && TB)
                            *p = beta ? *p + acc[i][j][e] : acc[i][j][e];
                        else
                            __builtin_nontemporal_store(beta ? *p + acc[i][j][e] : acc[i][j][e], p);
                    }
                }
            }
        }
    }
}

// the epilogue of one element: C = act(v + bias), the pre-activation and
// the 16-bit copy beside it (gemm16_block's EPI path applies it from LDS)
__device__ __forceinline__ void epi_store(const pgk_epi &epi, float *c, size_t off, int col, float v)
{
    const float zv = v + (epi.bias ? epi.bias[col] : 0.0f);
    const float o = act_f(epi.act, zv);
    if (!epi.skip_out)
        c[off] = o;
    if (epi.z)
        epi.z[off] = zv;
    if (epi.c16)
        epi.c16[off] = to16(epi.dtype16, o);
}

// Middle-sized product: a block owns a TM x TN tile of C (32 or 64 a side) and
// its KG waves split the reduction, wave w taking the KB-deep chunks w,
// w + KG, ...  Each wave computes the whole tile over its chunks from an
// S-stage DMA ring of its own, so the k-loop has no block barrier and the
// waves' load latencies overlap; their partial tiles are then added through
// LDS in wave order and every thread finishes whole 16-byte pieces of rows
// (beta, or the forward epilogue).  One launch fills the chip where 128-tiles
// do not, without split-K's partials in memory and its summing launch.
// Bound by the loads' latency and the launch itself at these sizes.  Measured
// back to back against the 128-tile plans (split-K where they split):
// 512 x 1024 x 4096 dgrad 20.0 -> 14.4 us, 1024^3 20.1 -> 8.4 us, a
// 512 x 4096 x 1024 gelu layer 22.8 -> 17.1 us, 256 x 256 x 512 9.5 -> 4.5 us.
// GATE: as gcfg's
template <int TM_, int TN_, int KG_, int KB_, int S_, bool TA_, bool TB_, bool F16_, bool GATE_ = false>
struct kscfg {
    static constexpr bool GATE = GATE_;
    static constexpr int TM = TM_, TN = TN_, KG = KG_, KB = KB_, S = S_;
    static constexpr bool TA = TA_, TB = TB_, F16 = F16_;
    static constexpr int NT = 64 * KG, RS = TN + 4; // floats of a partial tile's row
    static constexpr int STAGE = (TM + TN) * KB / 8, RING = KG * S * STAGE;
    static constexpr int PART = KG * TM * RS / 4;
    static constexpr int LDS_U4 = RING > PART ? RING : PART;
};

// block id -> tile: ids are dealt to the 8 XCDs round-robin (from any first
// one), so consecutive tiles, which share lines and panels of the operands, are
// regrouped onto one XCD and its L2; the last nb % 8 stay where they are
__device__ __forceinline__ int xcd_tile(int pid, int nb)
{
    const int q = nb >> 3;
    return pid < (q << 3) ? (pid & 7) * q + (pid >> 3) : pid;
}

template <class CF>
__device__ __forceinline__ void ks_block(const gemm_kargs &g, int has_epi, int pid, int nb, bool remap, int z,
                                         LDS uint4 *const lds)
{
    constexpr int TM = CF::TM, TN = CF::TN, KG = CF::KG, KB = CF::KB, S = CF::S, FM = TM / 32, FN = TN / 32;
    constexpr bool F16 = CF::F16;
    using OA = typename std::conditional<CF::TA, TileMN<TM, 64, KB>, TileK<TM, 64, KB>>::type;
    using OB = typename std::conditional<
        CF::GATE, TileGate<TN, 64, KB, TN / 2>,
        typename std::conditional<CF::TB, TileMN<TN, 64, KB>, TileK<TN, 64, KB>>::type>::type;
    constexpr int LPT = OA::NQ + OB::NQ, SA = TM * KB / 8, KS = KB / 16;
    static_assert((S - 1) * LPT < 64, "the loads in flight fit the vmcnt counter");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // tile order as the tiled kernel's: consecutive tiles on one XCD, 8
    // tile-rows at a time.  Also for counts that 8 does not divide where the
    // output is wider than tall: as dealt, every XCD fetches each line of the
    // wide operand (98 x 3720 at k = 3008, 236 blocks: 26 us as dealt, 14
    // grouped; 51 such shapes 0.99 - 1.7 times as fast, 95 tall ones 0.75 - 1.2)
    if (g.tiles_n > g.tiles_m || (remap && (nb & 7) == 0))
        pid = xcd_tile(pid, nb);
    const int group = pid / (8 * g.tiles_n), first = group * 8;
    const int gsz = g.tiles_m - first < 8 ? g.tiles_m - first : 8, in = pid - group * 8 * g.tiles_n;
    const int m0 = (first + in % gsz) * TM, n0 = in / gsz * (CF::GATE ? TN / 2 : TN);
    const uint16_t *A = g.A + (size_t)z * g.sA, *B = g.B + (size_t)z * g.sB;
    LDS uint4 *const ring = lds + wave * S * CF::STAGE;
    const int nct = (g.K + KB - 1) / KB, nc = nct > wave ? (nct - wave + KG - 1) / KG : 0;
    const int whole = g.fast_ok ? g.K / KB : 0; // chunks wholly below K
    typename OA::Fast fA[OA::NQ];
    typename OB::Fast fB[OB::NQ];
#pragma unroll
    for (int q = 0; q < OA::NQ; ++q)
        fA[q] = OA::fast_q(q, g.lda, m0, g.a_extent, 0, lane);
#pragma unroll
    for (int q = 0; q < OB::NQ; ++q)
        fB[q] = OB::fast_q(q, g.ldb, n0, g.b_extent, 0, lane);
    // this wave's chunk c into stage st; chunks past the end read the zero page
    auto load = [&](int c, int st) {
        LDS uint4 *sa = ring + st * CF::STAGE, *sb = sa + SA;
        const int ch = c * KG + wave;
        if (ch < whole) {
#pragma unroll
            for (int q = 0; q < OA::NQ; ++q)
                OA::load_fast(q, fA[q], A, g.lda, m0, ch * KB, sa, 0);
#pragma unroll
            for (int q = 0; q < OB::NQ; ++q)
                OB::load_fast(q, fB[q], B, g.ldb, n0, ch * KB, sb, 0);
        } else {
            const int k0 = ch < nct ? ch * KB : g.K;
#pragma unroll
            for (int q = 0; q < OA::NQ; ++q)
                OA::load_q(q, A, g.lda, m0, g.a_extent, k0, g.K, sa, lane);
#pragma unroll
            for (int q = 0; q < OB::NQ; ++q)
                OB::load_q(q, B, g.ldb, n0, g.b_extent, k0, g.K, sb, lane);
        }
    };
    // Four waves keep two sums each, their even and odd chunks': eight partial
    // sums of a reduction, as many as eight waves or the split-K plan have, so
    // the error against 64 bits is no larger than theirs (dW of 2048 x 512 x 512:
    // 1.02e-7, with one sum per wave 1.32e-7)
    constexpr int NA = KG == 4 ? 2 : 1;
    f32x16 acc[NA][FM][FN];
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    acc[a][i][j][e] = 0.0f;
    if (nc > 0) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            load(s, s);
        int st = 0;
        auto chunk = [&](int c, f32x16(&sum)[FM][FN]) {
            const LDS uint4 *sa = ring + st * CF::STAGE, *sb = sa + SA;
            // chunk c landed (the newest S - 1 chunks may be in flight)
            __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((S - 1) * LPT));
            __asm__ volatile("" ::: "memory");
            uint4 fa[KS][FM], fb[KS][FN];
#pragma unroll
            for (int s = 0; s < KS; ++s) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    fa[s][i] = OA::frag(sa, i * 32, s, lane);
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    fb[s][j] = OB::frag(sb, j * 32, s, lane);
            }
            // the stage's reads are done before its refill
            __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(63));
            __asm__ volatile("" ::: "memory");
            load(c + S, st);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        sum[i][j] = mfma32<F16>(fa[s][i], fb[s][j], sum[i][j]);
            st = st + 1 == S ? 0 : st + 1;
        };
        int c = 0;
        for (; c + NA <= nc; c += NA)
#pragma unroll
            for (int a = 0; a < NA; ++a)
                chunk(c + a, acc[a]);
        if (c < nc) // NA == 2: the last even chunk
            chunk(c, acc[0]);
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0));
    }
#pragma unroll
    for (int a = 1; a < NA; ++a)
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[0][i][j] += acc[a][i][j];
    __syncthreads(); // the rings are done
    LDS float *part = (LDS float *)lds;
    const int lrow = lane & 31, lk = lane >> 5;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                part[(wave * TM + i * 32 + (e >> 2) * 8 + lk * 4 + (e & 3)) * CF::RS + j * 32 + lrow] = acc[0][i][j][e];
    __syncthreads();
    if constexpr (CF::GATE) {
        if (gate_whole(g.epi, g.C, g.N)) {
#pragma unroll 1
            for (int i = (int)threadIdx.x; i < TM * TN / 8; i += CF::NT) {
                const int row = i / (TN / 8), c4 = i % (TN / 8) * 4, gr = m0 + row, gc = n0 + c4;
                if (gr >= g.M || gc >= g.N)
                    continue;
                f32x4 gv = {0.0f, 0.0f, 0.0f, 0.0f}, uv = gv;
#pragma unroll
                for (int w = 0; w < KG; ++w) {
                    gv += *(const LDS f32x4 *)(part + (w * TM + row) * CF::RS + c4);
                    uv += *(const LDS f32x4 *)(part + (w * TM + row) * CF::RS + TN / 2 + c4);
                }
                gate_store4(g.epi, g.C, g.N, gr, gc, gv, uv);
            }
        } else {
#pragma unroll 1
            for (int i = (int)threadIdx.x; i < TM * TN / 2; i += CF::NT) {
                const int row = i / (TN / 2), c = i % (TN / 2), gr = m0 + row, gc = n0 + c;
                if (gr >= g.M || gc >= g.N)
                    continue;
                float gv = 0.0f, uv = 0.0f;
#pragma unroll
                for (int w = 0; w < KG; ++w) {
                    gv += part[(w * TM + row) * CF::RS + c];
                    uv += part[(w * TM + row) * CF::RS + TN / 2 + c];
                }
                gate_store1(g.epi, g.C, g.N, gr, gc, gv, uv);
            }
        }
        return;
    }
    float *C = g.C + (size_t)z * g.sC;
    pgk_epi epi = g.epi;
    if (epi.c16)
        epi.c16 += (size_t)z * g.sC;
    const bool v4 = (g.ldc & 3) == 0 && (((uintptr_t)C | (uintptr_t)epi.z) & 15) == 0 && (((uintptr_t)epi.c16) & 7) == 0;
#pragma unroll
    for (int i = (int)threadIdx.x; i < TM * TN / 4; i += CF::NT) {
        const int row = i / (TN / 4), c4 = i % (TN / 4) * 4;
        const int gr = m0 + row, gc = n0 + c4;
        if (gr >= g.M || gc >= g.N)
            continue;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < KG; ++w)
            v += *(const LDS f32x4 *)(part + (w * TM + row) * CF::RS + c4);
        const size_t off = (size_t)gr * g.ldc + gc;
        if (!v4 || gc + 3 >= g.N) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (gc + q >= g.N)
                    break;
                if (has_epi)
                    epi_store(epi, C, off + q, gc + q, v[q]);
                else
                    C[off + q] = g.beta ? C[off + q] + v[q] : v[q];
            }
        } else if (has_epi) {
            f32x4 zv = v, o;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                zv[q] += epi.bias ? epi.bias[gc + q] : 0.0f;
                o[q] = act_f(epi.act, zv[q]);
            }
            if (!epi.skip_out)
                *(f32x4 *)(C + off) = o;
            if (epi.z)
                *(f32x4 *)(epi.z + off) = zv;
            if (epi.c16)
                *(uint2 *)(epi.c16 + off) = make_uint2(to16x2(epi.dtype16, o[0], o[1]), to16x2(epi.dtype16, o[2], o[3]));
        } else {
            *(f32x4 *)(C + off) = g.beta ? *(const f32x4 *)(C + off) + v : v;
        }
    }
}

} // namespace

#endif
