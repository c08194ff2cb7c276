// Block tiles of products whose operands are padded: rows at a pitch of whole
// 128-byte pieces, the reduction a whole number of tiles with zeros behind its
// end.  An operand may come in two pieces, high and low, whose sum it is: then
//   A B = Ah Bh + Ah Bl + Al Bh
// in one accumulator (Al Bl lies below the pieces' own rounding).  Signed bytes
// are taken two to a 16-bit place, so every size along the reduction counts pairs.
#ifndef PGK_PIECE_TILE_H
#define PGK_PIECE_TILE_H

#include "gemm_tile.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// 32 x 32 products of f16 (over 16) and of signed bytes (over 32, exact); a lane
// holds row (column) lane % 32 of an operand, and column lane % 32 of rows
// (e / 4) 8 + (lane / 32) 4 + e % 4 of the sums
__device__ __forceinline__ f32x16 piece_mma(const uint4 &a, const uint4 &b, const f32x16 &c) { return mfma32<true>(a, b, c); }
__device__ __forceinline__ i32x16 piece_mma(const uint4 &a, const uint4 &b, const i32x16 &c)
{
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// ACC f32x16 (f16 operands) or i32x16 (signed bytes); P pieces per operand; BM x BN
// tile on WGM x WGN waves; A rows K-contiguous, B's too, or with TB k-rows of N;
// stages of KB along the reduction, S of them
template <class ACC_, int P_, int BM_, int BN_, int WGM_, int WGN_, bool TB_, int KB_, int S_>
struct pcfg {
    using ACC = ACC_;
    static constexpr int P = P_, BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, KB = KB_, S = S_;
    static constexpr bool TB = TB_;
    static constexpr int NT = 64 * WGM * WGN, WM = BM / WGM, WN = BN / WGN, FM = WM / 32, FN = WN / 32;
    static constexpr int SA = BM * KB / 8, SB = BN * KB / 8, STAGE = P * (SA + SB), RS = WN + 4;
    static constexpr int OUT_U4 = WGM * WGN * 32 * RS / 4; // the sums' way out, 32 rows a wave
    static constexpr int LDS_U4 = S * STAGE > OUT_U4 ? S * STAGE : OUT_U4;
};

// piece p of an operand starts p * plane places behind the first; ext: its rows (with
// TB columns, a multiple of 8), at least 1; ld < kFastLd
struct piece_operand {
    const uint16_t *p;
    size_t ld, plane;
    int ext;
};

// The sums of the tile at (m0, n0) over [k0, k0 + K), both multiples of KB, K
// positive.  The ring of S stages works as the 16-bit products' (gemm16_block): one
// barrier a tile, behind which the stage that every wave has read is refilled and
// the next tile's first operands are read, in slots between the matrix
// instructions.  LDS is free again afterwards (behind a barrier).
//
// One piece: a k-step's operands are read a step ahead into a second set.  Two
// pieces: its three products run one after the other, Ah Bh beside which Al is read,
// Ah Bl, Al Bh, and the next step's Bh, Ah and Bl are read as soon as the last
// product with the ones that they replace is issued; only Bh has a second set.  In
// a tile's last step the barrier stands behind the first product.
template <class CF>
__device__ __forceinline__ void piece_loop(const piece_operand &A, const piece_operand &B, int k0, int K, int m0, int n0,
                                           LDS uint4 *const lds, typename CF::ACC (&acc)[CF::FM][CF::FN])
{
    constexpr int P = CF::P, BM = CF::BM, BN = CF::BN, WM = CF::WM, WN = CF::WN, KB = CF::KB, S = CF::S, NT = CF::NT;
    constexpr int FM = CF::FM, FN = CF::FN, SA = CF::SA, SB = CF::SB;
    using OA = TileK<BM, NT, KB>;
    using OB = typename std::conditional<CF::TB, TileMN<BN, NT, KB>, TileK<BN, NT, KB>>::type;
    constexpr int LPT = P * (OA::NQ + OB::NQ), KS = KB / 16, NM = FM * FN;
    static_assert(P == 1 || P == 2, "one piece or two");
    static_assert(S >= 2 && KS % 2 == 0, "two or more stages, an even number of k-steps per tile");
    static_assert((S - 1) * LPT < 64, "the loads in flight fit the vmcnt counter");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / CF::WGN, wn = wave % CF::WGN;
    const int KT = K / KB;
    auto stA = [&](int st, int p) { return lds + st * CF::STAGE + p * SA; };
    auto stB = [&](int st, int p) { return lds + st * CF::STAGE + P * SA + p * SB; };
    typename OA::Fast fA[OA::NQ];
    typename OB::Fast fB[OB::NQ];
#pragma unroll
    for (int q = 0; q < OA::NQ; ++q)
        fA[q] = OA::fast_q(q, A.ld, m0, A.ext, wave, lane);
#pragma unroll
    for (int q = 0; q < OB::NQ; ++q)
        fB[q] = OB::fast_q(q, B.ld, n0, B.ext, wave, lane);
    auto dma = [&](int q, int t, int st) {
        const int k = k0 + (t < KT ? t : KT - 1) * KB; // stages past the end are read by none
        if (q < P * OA::NQ) {
            const int p = q / OA::NQ, i = q % OA::NQ;
            OA::load_fast(i, fA[i], A.p + p * A.plane, A.ld, m0, k, stA(st, p), wave);
        } else {
            const int p = (q - P * OA::NQ) / OB::NQ, i = (q - P * OA::NQ) % OB::NQ;
            OB::load_fast(i, fB[i], B.p + p * B.plane, B.ld, n0, k, stB(st, p), wave);
        }
    };
    auto sync_tile = [&](auto newer) { // all but the newest tiles' loads have landed, every wave has read its operands
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(decltype(newer)::value * LPT));
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
    };
    auto fragA = [&](int st, int p, int i, int s) { return OA::frag(stA(st, p), wm * WM + i * 32, s, lane); };
    auto fragB = [&](int st, int p, int j, int s) { return OB::frag(stB(st, p), wn * WN + j * 32, s, lane); };
    // part g of n of `all` things, in slots between the matrix instructions
    auto slots = [&](int g, int n, int all, auto f) {
#pragma unroll
        for (int r = g * all / n; r < (g + 1) * all / n; ++r)
            f(r);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[i][j][e] = 0;
#pragma unroll
    for (int t = 0; t < S; ++t)
#pragma unroll
        for (int q = 0; q < LPT; ++q)
            dma(q, t, t);
    sync_tile(std::integral_constant<int, S - 1>{});
    // ah, al: A's pieces; bh: B's high piece of even and odd steps (with one piece,
    // ah and al those of even and odd steps); bl: B's low piece
    uint4 ah[FM], al[FM], bh[2][FN], bl[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
        ah[i] = fragA(0, 0, i, 0);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        bh[0][j] = fragB(0, 0, j, 0);
        if constexpr (P == 2)
            bl[j] = fragB(0, 1, j, 0);
    }
    // k-step s of the tile in stage st; `next`: the operands of step ns of the tile in
    // stage nst are read beside it; `tail`: its barrier, and tile `reload` to stage st
    auto step = [&](int s, int st, bool next, int nst, int ns, bool tail, int reload) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (P == 1) {
            if (tail)
                sync_tile(std::integral_constant<int, S - 2>{});
            uint4(&a)[FM] = s & 1 ? al : ah;
            uint4(&na)[FM] = s & 1 ? ah : al;
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    acc[i][j] = piece_mma(a[i], bh[s & 1][j], acc[i][j]);
                    if (next)
                        slots(i * FN + j, NM, FM + FN, [&](int r) {
                            if (r < FM)
                                na[r] = fragA(nst, 0, r, ns);
                            else
                                bh[s + 1 & 1][r - FM] = fragB(nst, 0, r - FM, ns);
                        });
                    if (tail)
                        slots(i * FN + j, NM, LPT, [&](int q) { dma(q, reload, st); });
                }
        } else {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    acc[i][j] = piece_mma(ah[i], bh[s & 1][j], acc[i][j]);
                    slots(i * FN + j, NM, FM, [&](int r) { al[r] = fragA(st, 1, r, s); });
                }
            if (tail)
                sync_tile(std::integral_constant<int, S - 2>{});
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    acc[i][j] = piece_mma(ah[i], bl[j], acc[i][j]);
                    const int g = i * FN + j;
                    if (next)
                        slots(g, NM, FN, [&](int r) { bh[s + 1 & 1][r] = fragB(nst, 0, r, ns); });
                    if (tail)
                        slots(g, 2 * NM, LPT, [&](int q) { dma(q, reload, st); });
                }
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    acc[i][j] = piece_mma(al[i], bh[s & 1][j], acc[i][j]);
                    const int g = i * FN + j;
                    if (next)
                        slots(g, NM, FM + FN, [&](int r) {
                            if (r < FM)
                                ah[r] = fragA(nst, 0, r, ns);
                            else
                                bl[r - FM] = fragB(nst, 1, r - FM, ns);
                        });
                    if (tail)
                        slots(NM + g, 2 * NM, LPT, [&](int q) { dma(q, reload, st); });
                }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto head = [&](int st) {
#pragma unroll
        for (int s = 0; s < KS - 1; ++s)
            step(s, st, true, st, s + 1, false, 0);
    };
    head(0);
    // the last step of tile t in stage u and the others of tile t + 1
    auto link = [&](int t, int u) {
        step(KS - 1, u, true, (u + 1) % S, 0, true, t + S);
        head((u + 1) % S);
    };
    int t = 0;
    for (; t + S <= KT - 1; t += S)
#pragma unroll
        for (int u = 0; u < S; ++u)
            link(t + u, u);
#pragma unroll
    for (int u = 0; u < S - 1; ++u)
        if (t + u < KT - 1)
            link(t + u, u);
    step(KS - 1, (KT - 1) % S, false, 0, 0, false, 0);
    __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0)); // the loads past the end land before the LDS is used anew
}

// The way out of strip i of the sums, 32 rows of each wave's tile, through LDS.
// f(row, column, v, from(row, column), false) takes four neighbouring sums of a
// row, for every row < M and column < N (a multiple of 4 behind n0), and may change
// them; `from` is asked for all of a thread's places before the first f, so that
// its loads wait for none of f's stores (f loading what it needs by itself took 26 us
// of each round of 256 x 256 tiles, now 11); U > 0: of U places at a time.  With
// `down` f(row, column, v, {}, true) then takes what it left, four down a column.
template <class CF, class V4, int U_ = 0, class FROM, class FN_>
__device__ __forceinline__ void piece_out_strip(typename CF::ACC (&acc)[CF::FN], int i, int m0, int n0, int M, int N,
                                                LDS uint4 *const lds, bool down, FROM from, FN_ f)
{
    constexpr int RS = CF::RS, WN = CF::WN, CL = WN / 4, STEP = 64 / CL, NR = 32 / STEP;
    constexpr int U = U_ && U_ < NR ? U_ : NR;
    static_assert(NR % U == 0, "whole groups of places");
    typedef LDS int *lds_int;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / CF::WGN, wn = wave % CF::WGN;
    const int lrow = lane & 31, lk = lane >> 5;
    const lds_int reg = (lds_int)lds + wave * 32 * RS;
    const int col0 = n0 + wn * WN, row0 = m0 + wm * CF::WM + i * 32, r0 = lane / CL, c4 = (lane % CL) * 4;
    decltype(from(0, 0)) with[U] = {};
    auto ask = [&](int r1) {
#pragma unroll
        for (int r = 0; r < U; ++r)
            if (row0 + r0 + (r1 + r) * STEP < M && col0 + c4 < N)
                with[r] = from(row0 + r0 + (r1 + r) * STEP, col0 + c4);
    };
    ask(0);
    __syncthreads(); // the stages' (or the previous strip's) reads are done
#pragma unroll
    for (int j = 0; j < CF::FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const auto one = acc[j][e]; // (a bit cast of a vector's element itself takes its first)
            reg[((e >> 2) * 8 + lk * 4 + (e & 3)) * RS + j * 32 + lrow] = __builtin_bit_cast(int, one);
        }
    __syncthreads();
#pragma unroll 1
    for (int r1 = 0; r1 < NR; r1 += U) {
        if (r1)
            ask(r1);
#pragma unroll
        for (int r = 0; r < U; ++r) {
            const int row = r0 + (r1 + r) * STEP;
            if (row0 + row >= M || col0 + c4 >= N)
                continue;
            LDS i32x4 *const at = (LDS i32x4 *)(reg + row * RS + c4);
            V4 v = __builtin_bit_cast(V4, *at);
            f(row0 + row, col0 + c4, v, with[r], false);
            if (down)
                *at = __builtin_bit_cast(i32x4, v);
        }
    }
    if (down) {
        __syncthreads();
        const int r4 = (lane & 7) * 4;
#pragma unroll 4
        for (int c = lane >> 3; c < WN; c += 8) {
            if (row0 + r4 >= M || col0 + c >= N)
                continue;
            const i32x4 q = {reg[r4 * RS + c], reg[(r4 + 1) * RS + c], reg[(r4 + 2) * RS + c], reg[(r4 + 3) * RS + c]};
            V4 v = __builtin_bit_cast(V4, q);
            f(row0 + r4, col0 + c, v, decltype(from(0, 0)){}, true);
        }
    }
}

} // namespace

#endif
