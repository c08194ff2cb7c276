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

// The sums of the tile at (m0, n0) over K, a positive multiple of KB.  The ring of
// S stages works as the 16-bit products' (gemm16_block): a tile's last k-step
// starts behind the one barrier of the tile, refills the stage that every wave
// has read and reads the next tile's first operands, in slots between the
// matrix instructions.  LDS is free again afterwards (behind a barrier).
template <class CF>
__device__ __forceinline__ void piece_loop(const piece_operand &A, const piece_operand &B, int K, int m0, int n0,
                                           LDS uint4 *const lds, typename CF::ACC (&acc)[CF::FM][CF::FN])
{
    constexpr int P = CF::P, BM = CF::BM, BN = CF::BN, WM = CF::WM, WN = CF::WN, KB = CF::KB, S = CF::S, NT = CF::NT;
    constexpr int FM = CF::FM, FN = CF::FN, SA = CF::SA, SB = CF::SB;
    using OA = TileK<BM, NT, KB>;
    using OB = typename std::conditional<CF::TB, TileMN<BN, NT, KB>, TileK<BN, NT, KB>>::type;
    constexpr int LPT = P * (OA::NQ + OB::NQ), KS = KB / 16;
    constexpr int NP = P == 1 ? 1 : 3, NM = NP * FM * FN, NF = P * (FM + FN); // products and operands of a k-step
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
        const int k0 = (t < KT ? t : KT - 1) * KB; // stages past the end are read by none
        if (q < P * OA::NQ) {
            const int p = q / OA::NQ, i = q % OA::NQ;
            OA::load_fast(i, fA[i], A.p + p * A.plane, A.ld, m0, k0, stA(st, p), wave);
        } else {
            const int p = (q - P * OA::NQ) / OB::NQ, i = (q - P * OA::NQ) % OB::NQ;
            OB::load_fast(i, fB[i], B.p + p * B.plane, B.ld, n0, k0, stB(st, p), wave);
        }
    };
    auto sync_tile = [&](auto newer) { // all but the newest tiles' loads have landed, every wave has read its operands
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(decltype(newer)::value * LPT));
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
    };
    uint4 fa[2][P][FM], fb[2][P][FN];
    // operand r of k-step s of the tile in stage st
    auto read = [&](int r, int st, int s, int to) {
        if (r < P * FM)
            fa[to][r / FM][r % FM] = OA::frag(stA(st, r / FM), wm * WM + (r % FM) * 32, s, lane);
        else
            fb[to][(r - P * FM) / FN][(r - P * FM) % FN] =
                OB::frag(stB(st, (r - P * FM) / FN), wn * WN + ((r - P * FM) % FN) * 32, s, lane);
    };
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[i][j][e] = 0;
    // k-step s; `next`: k-step ns of the tile in stage nst is read beside it;
    // `tail`: tile `reload` goes to stage rst
    auto step = [&](int s, bool next, int nst, int ns, bool tail, int reload, int rst) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int pr = 0; pr < NP; ++pr)
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    acc[i][j] = piece_mma(fa[s & 1][pr == 2][i], fb[s & 1][pr == 1][j], acc[i][j]);
                    const int g = (pr * FM + i) * FN + j;
                    if (next) {
#pragma unroll
                        for (int r = g * NF / NM; r < (g + 1) * NF / NM; ++r)
                            read(r, nst, ns, (s + 1) & 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (tail) {
#pragma unroll
                        for (int q = g * LPT / NM; q < (g + 1) * LPT / NM; ++q)
                            dma(q, reload, rst);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto head = [&](int st) {
#pragma unroll
        for (int s = 0; s < KS - 1; ++s)
            step(s, true, st, s + 1, false, 0, 0);
    };
#pragma unroll
    for (int t = 0; t < S; ++t)
#pragma unroll
        for (int q = 0; q < LPT; ++q)
            dma(q, t, t);
    sync_tile(std::integral_constant<int, S - 1>{});
#pragma unroll
    for (int r = 0; r < NF; ++r)
        read(r, 0, 0, 0);
    head(0);
    // the tail of tile t in stage u and the head of tile t + 1
    auto link = [&](int t, int u) {
        sync_tile(std::integral_constant<int, S - 2>{});
        step(KS - 1, true, (u + 1) % S, 0, true, t + S, u);
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
    step(KS - 1, false, 0, 0, false, 0, 0);
    __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0)); // the loads past the end land before the LDS is used anew
}

// The sums' way out: 32 rows of each wave's tile at a time through LDS.  f(row,
// column, v, false) takes four neighbouring sums of a row, for every row < M and
// column < N (a multiple of 4 behind n0), and may change them; with `down`
// f(row, column, v, true) then takes what it left, four down a column.
template <class CF, class V4, class FN_>
__device__ __forceinline__ void piece_out(typename CF::ACC (&acc)[CF::FM][CF::FN], int m0, int n0, int M, int N,
                                          LDS uint4 *const lds, bool down, FN_ f)
{
    constexpr int RS = CF::RS, WN = CF::WN, CL = WN / 4;
    typedef LDS int *lds_int;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / CF::WGN, wn = wave % CF::WGN;
    const int lrow = lane & 31, lk = lane >> 5;
    const lds_int reg = (lds_int)lds + wave * 32 * RS;
    const int col0 = n0 + wn * WN;
#pragma unroll
    for (int i = 0; i < CF::FM; ++i) {
        __syncthreads(); // the stages' (or the previous pass's) reads are done
#pragma unroll
        for (int j = 0; j < CF::FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const auto one = acc[i][j][e]; // (a bit cast of a vector's element itself takes its first)
                reg[((e >> 2) * 8 + lk * 4 + (e & 3)) * RS + j * 32 + lrow] = __builtin_bit_cast(int, one);
            }
        __syncthreads();
        const int row0 = m0 + wm * CF::WM + i * 32, c4 = (lane % CL) * 4;
#pragma unroll 1
        for (int r = lane / CL; r < 32; r += 64 / CL)
            if (row0 + r < M && col0 + c4 < N) {
                LDS i32x4 *const at = (LDS i32x4 *)(reg + r * RS + c4);
                V4 v = __builtin_bit_cast(V4, *at);
                f(row0 + r, col0 + c4, v, false);
                if (down)
                    *at = __builtin_bit_cast(i32x4, v);
            }
        if (down) {
            __syncthreads();
            const int r4 = (lane & 7) * 4;
#pragma unroll 1
            for (int c = lane >> 3; c < WN; c += 8) {
                if (row0 + r4 >= M || col0 + c >= N)
                    continue;
                const i32x4 q = {reg[r4 * RS + c], reg[(r4 + 1) * RS + c], reg[(r4 + 2) * RS + c], reg[(r4 + 3) * RS + c]};
                V4 v = __builtin_bit_cast(V4, q);
                f(row0 + r4, col0 + c, v, true);
            }
        }
    }
}

} // namespace

#endif
