// Layer norm over the rows of x [m, d] and its backward.
//
//   n = (x - mean) rstd, mean = sum x / d, rstd = 1 / sqrt(sum (x - mean)^2 / d + eps)
//   y = n w + b
//   h = dy w: dx = rstd (h - sum h / d - n sum (h n) / d), dw = sum over rows of dy n, db = of dy
//
// Statistics and sums are f32 from values held in registers; y and dx round once.  The
// variance is of differences, not of squares: those from a first mean, whose own mean
// then corrects both (settled), so that a row of equal values has its value as mean
// and no variance.  A row that a block holds is read once; longer ones are cut into
// slices for blocks of their own and read twice.  Bound by the stream of the rows: HBM for large calls
// (8192 x 8192 in bf16: forward 54 to 57 us, 4.8 TB/s, backward 92 to 95, 4.3 TB/s, where a
// copy reaches 5.2), the launches and a row's loads for small ones (1 x 4096: 2.9 us;
// 33 x 50001 in f16 with its backward, four launches: 19).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include <type_traits>

#include "launch.h"

namespace {

constexpr int kChunks = 2; // of 16 bytes of x, per thread of a slice
constexpr unsigned kMostBlocks = 1u << 20; // of a grid; kernels loop past it

// Chunk c of E of a row of d: its place, and which of the E there are its own.  The last
// one of a row lies over its neighbour, so that it is loaded as the others are (its
// elements one by one held up the row's whole block: 8192 x 4095 in bf16, backward,
// 96 us against 43 of 4096).  Of a slice of a longer row the neighbour may be the
// slice before; with SHORT a row of less than a chunk has one of d.
template <int E, bool SHORT = false>
struct spot {
    int at, lo, hi;
    __device__ __forceinline__ spot(int c, int d)
    {
        const int over = (c + 1) * E - d;
        lo = over > 0 ? over : 0;
        at = c * E - lo;
        hi = E;
        if (SHORT && d < E) {
            lo = at = 0;
            hi = d;
        }
    }
    __device__ __forceinline__ bool full() const { return !SHORT || hi == E; }
    __device__ __forceinline__ bool whole() const { return full() && lo == 0; }
    __device__ __forceinline__ bool has(int e) const { return e >= lo && (!SHORT || e < hi); }
};

// as many values of S as 16 bytes hold of T, at any alignment of an element
template <class T, class S>
struct piece {
    static constexpr int E = 16 / sizeof(T);
    typedef S sv __attribute__((ext_vector_type(E), aligned(sizeof(S))));
    sv q;
    // of the row p; past a short row's end: 0
    template <bool SHORT>
    __device__ __forceinline__ void load(const S *p, const spot<E, SHORT> &c)
    {
        if (c.full()) {
            q = *(const sv *)(p + c.at);
        } else {
            q = sv{};
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < c.hi)
                    q[e] = p[e];
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return (float)q[e]; }
    // 0 for the neighbour's
    template <bool SHORT>
    __device__ __forceinline__ void own(const spot<E, SHORT> &c)
    {
        if (c.lo)
#pragma unroll
            for (int e = 0; e < E; ++e)
                q[e] = e < c.lo ? (S)0.0f : q[e];
    }
    // new to the compiler: the values read from here on are converted anew, where
    // those converted before would be kept in twice the registers
    __device__ __forceinline__ void again()
    {
        typedef uint32_t words __attribute__((ext_vector_type(sizeof(sv) / 4)));
        words v = __builtin_bit_cast(words, q);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(sv) / 4); ++i) {
            uint32_t one = v[i];
            __asm__("" : "+v"(one));
            v[i] = one;
        }
        q = __builtin_bit_cast(sv, v);
    }
};

// the same as f32
template <class T>
struct chunk {
    static constexpr int E = 16 / sizeof(T);
    float v[E];
    template <bool SHORT, class S>
    __device__ __forceinline__ void load(const S *p, const spot<E, SHORT> &c)
    {
        piece<T, S> q;
        q.load(p, c);
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] = q[e];
    }
    // (of its own)
    template <bool SHORT, class O>
    __device__ __forceinline__ void store(O *p, const spot<E, SHORT> &c) const
    {
        typedef O ov __attribute__((ext_vector_type(E), aligned(sizeof(O))));
        if (c.whole()) {
            ov q;
#pragma unroll
            for (int e = 0; e < E; ++e)
                q[e] = (O)v[e];
            *(ov *)(p + c.at) = q;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (c.has(e))
                    p[c.at + e] = (O)v[e];
        }
    }
    __device__ __forceinline__ void fill(float f)
    {
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] = f;
    }
};

// s of a lane and of lane ^ O, for O from 32 down one after the other (so that O = 4 finds
// a period of eight lanes, as a rotation in 16 needs it), without LDS (f32 4096 x 1024,
// forward: 9.5 us, with shuffles 11.2)
template <int O>
__device__ __forceinline__ float with_xor(float s)
{
    const uint32_t v = __float_as_uint(s);
    if constexpr (O >= 16) { // both halves of the wave, or of 32 lanes
        const auto both = O == 32 ? __builtin_amdgcn_permlane32_swap(v, v, false, false)
                                  : __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return __uint_as_float(both[0]) + __uint_as_float(both[1]);
    } else { // rotations by 8 and 4 in 16 lanes, exchanges in 4
        constexpr int how = O == 8 ? 0x128 : O == 4 ? 0x124 : O == 2 ? 0x4e : 0xb1;
        return s + __uint_as_float(__builtin_amdgcn_update_dpp(0, v, how, 0xf, 0xf, true));
    }
}

// sums over the TPR threads that share a row, in a fixed order.  TPR over 64:
// through `red` [waves of a row], which the caller does not reuse before the
// next barrier but one; the waves' sums are read ON at a time
template <int TPR, int ON = TPR / 64, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float (*red)[N], int tid)
{
    static_assert(TPR == 8 || TPR >= 64, "eight lanes or whole waves");
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (TPR == 8)
            s[i] += __shfl_xor(s[i], 4);
        else
            s[i] = with_xor<4>(with_xor<8>(with_xor<16>(with_xor<32>(s[i]))));
        s[i] = with_xor<1>(with_xor<2>(s[i]));
    }
    if constexpr (TPR > 64) {
        if ((tid & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i)
                red[tid >> 6][i] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i)
            s[i] = 0.0f;
#pragma unroll ON
        for (int w = 0; w < TPR / 64; ++w)
#pragma unroll
            for (int i = 0; i < N; ++i)
                s[i] += red[w][i];
    }
}

// The mean and the sum of the squares of what differs from it, from a first mean, which
// is off by the roundings of its sum (some 80 half units of its last place at most).
// sums(mean, s, k): those of the differences c = x - mean and of their squares, the k'th
// time (0, 1).  With D = sum c / d the mean is D further and the squares about it are
// sum c^2 - D sum c.  Where D is what carries the squares (a row of values that differ by
// a few of those units, or not at all), the difference would be mostly rounding: both
// sums are taken once more, about the moved mean.
template <class FN>
__device__ __forceinline__ float settled(float &mean, float inv, FN sums)
{
    float s[2];
    sums(mean, s, 0);
    float off = s[0] * inv;
    mean += off;
    if (off != 0.0f && !(s[0] * off < 0.25f * s[1])) { // (also where the squares leave f32)
        sums(mean, s, 1);
        off = s[0] * inv;
        mean += off;
    }
    const float squares = s[1] - s[0] * off;
    return squares < 0.0f ? 0.0f : squares; // (a NaN stays)
}

// ---------------------------------------------------------------- rows that a block holds

// TPR threads per row, R chunks each; a block of 256 threads takes 256 / TPR rows at a
// time, one of 1024 threads one.  The next rows are on their way while a row is
// worked on; HOLD: the weights stay in registers.
template <class T, class O, int TPR, int R, bool HOLD>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_norm(const T *x, const float *__restrict__ w,
                                                                const float *__restrict__ b, float eps, size_t m, int d,
                                                                O *y, float *__restrict__ stats)
{
    using ch = chunk<T>;
    using at = spot<ch::E, TPR == 8>;
    constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
    constexpr int W = TPR > 64 ? TPR / 64 : 1;
    __shared__ float first[2][W][1], about[3][W][2];
    const int tid = (int)threadIdx.x, lane = tid % TPR;
    const int nc = (d + ch::E - 1) / ch::E;
    const float inv = 1.0f / (float)d;
    ch wv[HOLD ? R : 1], bv[HOLD ? R : 1];
    auto weights = [&](int i, ch &wi, ch &bi) {
        const int c = lane + i * TPR;
        if (w && c < nc)
            wi.load(w, at(c, d));
        else
            wi.fill(1.0f);
        if (b && c < nc)
            bi.load(b, at(c, d));
        else
            bi.fill(0.0f);
    };
    // as if new to the compiler: what follows from it for R chunks is worked out anew,
    // not kept in registers
    auto anew = [&] {
        int l = lane;
        if constexpr (R > 2)
            __asm__("" : "+v"(l));
        return l;
    };
    piece<T, T> cur[R];
    auto ask = [&](size_t row, piece<T, T>(&q)[R]) {
        const T *p = x + row * d;
        const int l = anew();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            q[i].q = {};
            if (row < m && l + i * TPR < nc)
                q[i].load(p, at(l + i * TPR, d));
        }
    };
    const size_t step = (size_t)gridDim.x * RPB;
    size_t row = (size_t)blockIdx.x * RPB + tid / TPR;
    ask(row, cur);
    if constexpr (HOLD)
#pragma unroll
        for (int i = 0; i < R; ++i)
            weights(i, wv[i], bv[i]);
    int turn = 0;
    for (size_t r0 = (size_t)blockIdx.x * RPB; r0 < m; r0 += step, row += step, turn ^= 1) {
        piece<T, T> next[R];
        if (r0 + step < m)
            ask(row + step, next);
        float one[1] = {0.0f};
        int l = anew();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (l + i * TPR < nc)
                cur[i].own(at(l + i * TPR, d));
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                one[0] = fmaf(cur[i][e], inv, one[0]); // (the values' sum may leave f32)
        }
        row_sum<TPR, 8>(one, first[turn], tid);
        float mean = one[0];
        const float sum = settled(mean, inv, [&](float mu, float (&t)[2], int again) {
            t[0] = t[1] = 0.0f;
            const int q = anew();
#pragma unroll
            for (int i = 0; i < R; ++i) {
                cur[i].again();
                const at k(q + i * TPR, d);
                const bool in = q + i * TPR < nc, whole = k.whole();
#pragma unroll
                for (int e = 0; e < ch::E; ++e) {
                    const float c = in && (whole || k.has(e)) ? cur[i][e] - mu : 0.0f;
                    t[0] += c;
                    t[1] += c * c;
                }
            }
            // (of more waves two at a time: no more registers are left beside the next row's)
            row_sum<TPR, (TPR <= 256 ? 4 : 2)>(t, about[again ? 2 : turn], tid);
        });
        const float rstd = 1.0f / sqrtf(sum * inv + eps);
        if (row < m) {
            if (stats && lane == 0)
                *(float2 *)(stats + row * 2) = make_float2(mean, rstd);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int c = anew() + i * TPR;
                if (c >= nc)
                    break;
                if constexpr (!HOLD)
                    weights(i, wv[0], bv[0]);
                cur[i].again();
                ch o;
#pragma unroll
                for (int e = 0; e < ch::E; ++e)
                    o.v[e] = (cur[i][e] - mean) * rstd * wv[HOLD ? i : 0].v[e] + bv[HOLD ? i : 0].v[e];
                o.store(y + row * d, at(c, d));
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
            cur[i] = next[i];
    }
}

// The grads of a block's rows: dx, and the block's own sums of dw and db to part
// [blocks][2][d] (NULL: not wanted), each thread those of its own columns.  The
// next rows are on their way while a row is worked on.
template <class T, class G, class O, int TPR, int R>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_norm_bwd(const T *__restrict__ x, const float *__restrict__ w,
                                                     const float *__restrict__ stats, const G *__restrict__ dy, size_t m,
                                                     int d, O *__restrict__ dx, int beta, float *__restrict__ part)
{
    using ch = chunk<T>;
    using at = spot<ch::E, TPR == 8>;
    constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR, COLS = TPR * R * ch::E;
    __shared__ float red[2][TPR > 64 ? TPR / 64 : 1][2];
    __shared__ float sums[RPB > 1 ? RPB : 1][RPB > 1 ? COLS : 1];
    const int tid = (int)threadIdx.x, lane = tid % TPR, group = tid / TPR;
    const int nc = (d + ch::E - 1) / ch::E;
    const float inv = 1.0f / (float)d;
    ch gw[R], gb[R], wv[R];
    struct rows {
        piece<T, T> x[R];
        piece<T, G> dy[R];
        float2 st;
    } cur;
    auto ask = [&](size_t row, rows &q) { // (past the end of a row and of all rows dy is 0)
        const size_t first = row * d;
        q.st = row < m ? *(const float2 *)(stats + row * 2) : make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = lane + i * TPR;
            q.x[i].q = {};
            q.dy[i].q = {};
            if (row < m && c < nc) {
                q.x[i].load(x + first, at(c, d));
                q.dy[i].load(dy + first, at(c, d));
            }
        }
    };
    const size_t step = (size_t)gridDim.x * RPB;
    size_t row = (size_t)blockIdx.x * RPB + group;
    ask(row, cur);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        gw[i].fill(0.0f);
        gb[i].fill(0.0f);
        if (w && lane + i * TPR < nc)
            wv[i].load(w, at(lane + i * TPR, d));
        else
            wv[i].fill(1.0f);
    }
    int turn = 0;
    for (size_t r0 = (size_t)blockIdx.x * RPB; r0 < m; r0 += step, row += step, turn ^= 1) {
        rows next;
        if (r0 + step < m)
            ask(row + step, next);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (lane + i * TPR < nc)
                cur.dy[i].own(at(lane + i * TPR, d));
#pragma unroll
            for (int e = 0; e < ch::E; ++e) {
                const float g = cur.dy[i][e], h = g * wv[i].v[e];
                const float n = (cur.x[i][e] - cur.st.x) * cur.st.y; // (beside a g of 0 if not its own)
                gw[i].v[e] += g * n;
                gb[i].v[e] += g;
                s[0] += h;
                s[1] += h * n;
            }
        }
        row_sum<TPR>(s, red[turn], tid);
        if (dx && row < m) {
            const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int c = lane + i * TPR;
                if (c >= nc)
                    break;
                cur.x[i].again();
                cur.dy[i].again();
                ch o;
                if (beta)
                    o.load(dx + row * d, at(c, d));
                else
                    o.fill(0.0f);
#pragma unroll
                for (int e = 0; e < ch::E; ++e)
                    o.v[e] += cur.st.y * (cur.dy[i][e] * wv[i].v[e] - c1 - (cur.x[i][e] - cur.st.x) * cur.st.y * c2);
                o.store(dx + row * d, at(c, d));
            }
        }
        cur = next;
    }
    if (!part)
        return;
    // the groups' sums of a column in the groups' order
    auto leave = [&](ch(&g)[R], float *out) {
        if constexpr (RPB == 1) {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (lane + i * TPR < nc)
                    g[i].store(out, at(lane + i * TPR, d));
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const at k(lane + i * TPR, d);
#pragma unroll
                for (int e = 0; e < ch::E; ++e)
                    if (lane + i * TPR < nc && k.has(e))
                        sums[group][k.at + e] = g[i].v[e];
            }
            __syncthreads();
            for (int c = tid; c < d; c += NT) {
                float t = 0.0f;
#pragma unroll 4
                for (int r = 0; r < RPB; ++r)
                    t += sums[r][c];
                out[c] = t;
            }
        }
    };
    float *out = part + (size_t)blockIdx.x * 2 * d;
    leave(gw, out);
    leave(gb, out + d);
}

// dw and db (either NULL) from the blocks' sums [blocks][2][d], in a fixed order: 64
// columns of one of them a job, NT / 64 threads taking every (NT / 64)'th block's
template <int NT>
__device__ __forceinline__ void join_sums(const float *__restrict__ part, int blocks, int d, int job, float *dw, int beta_w,
                                          float *db, int beta_b)
{
    constexpr int K = NT / 64;
    __shared__ float s[K][64];
    const int across = (d + 63) / 64, col = job % across * 64 + ((int)threadIdx.x & 63), k = (int)threadIdx.x >> 6;
    const bool second = job >= across;
    float *out = second ? db : dw;
    const int beta = second ? beta_b : beta_w;
    if (!out)
        return;
    float t = 0.0f;
    if (col < d) {
        const float *p = part + (second ? d : 0) + col;
#pragma unroll 16
        for (int i = k; i < blocks; i += K)
            t += p[(size_t)i * 2 * d];
    }
    s[k][threadIdx.x & 63] = t;
    __syncthreads();
    if (k || col >= d)
        return;
    t = 0.0f;
#pragma unroll
    for (int i = 0; i < K; ++i)
        t += s[i][threadIdx.x];
    out[col] = beta ? out[col] + t : t;
}
__global__ void __launch_bounds__(1024) k_norm_fin(const float *__restrict__ part, int blocks, int d, float *dw, int beta_w,
                                                   float *db, int beta_b)
{
    join_sums<1024>(part, blocks, d, (int)blockIdx.x, dw, beta_w, db, beta_b);
}

// ---------------------------------------------------------------- longer rows, in slices

// A slice is what 256 threads hold.  Statistics: each slice's mean and sum of
// squared differences from it, joined (in a fixed order) by
//   n = n1 + n2, q = m2 - m1: mean = m1 + q n2 / n, sum = s1 + s2 + q^2 n1 n2 / n
template <class T>
constexpr int kSlice = 256 * kChunks * chunk<T>::E;

// a wave's two sums over the k pairs of floats of a row's slices
__device__ __forceinline__ float2 slice_sums(const float2 *p, int k, int lane)
{
    float a = 0.0f, b = 0.0f;
    for (int i = lane; i < k; i += 64) {
        a += p[i].x;
        b += p[i].y;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        a += __shfl_xor(a, o);
        b += __shfl_xor(b, o);
    }
    return make_float2(a, b);
}

struct moments {
    float n, mean, sum;
    __device__ __forceinline__ void join(float n2, float m2, float s2)
    {
        const float all = n + n2, q = m2 - mean, f = all > 0.0f ? n2 / all : 0.0f;
        mean += q * f;
        sum += s2 + q * (n * f) * q; // (beside nothing q is a mean, whose square may leave f32)
        n = all;
    }
};

template <class T>
__global__ void __launch_bounds__(256) k_norm_slices(const T *__restrict__ x, size_t m, int d, int slices,
                                                     float2 *__restrict__ part)
{
    using ch = chunk<T>;
    using at = spot<ch::E>;
    __shared__ float sums[2][4][1], about[3][4][2];
    const int tid = (int)threadIdx.x;
    int turn = 0;
    for (size_t job = blockIdx.x; job < m * slices; job += gridDim.x, turn ^= 1) {
        const size_t row = job / slices;
        const int first = (int)(job - row * slices) * kSlice<T>, len = d - first < kSlice<T> ? d - first : kSlice<T>;
        const T *p = x + row * d + first;
        const int nc = (len + ch::E - 1) / ch::E;
        const float inv = 1.0f / (float)len;
        ch v[kChunks];
        float one[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
            if (tid + i * 256 < nc)
                v[i].load(p, at(tid + i * 256, len));
            else
                v[i].fill(0.0f);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const at k(tid + i * 256, len);
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                one[0] = fmaf(e >= k.lo ? v[i].v[e] : 0.0f, inv, one[0]); // (0 past a short row)
        }
        row_sum<256>(one, sums[turn], tid);
        float mean = one[0];
        const float sum = settled(mean, inv, [&](float mu, float (&t)[2], int again) {
            t[0] = t[1] = 0.0f;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const at k(tid + i * 256, len);
#pragma unroll
                for (int e = 0; e < ch::E; ++e) {
                    const float c = tid + i * 256 < nc && k.has(e) ? v[i].v[e] - mu : 0.0f;
                    t[0] += c;
                    t[1] += c * c;
                }
            }
            row_sum<256>(t, about[again ? 2 : turn], tid);
        });
        if (tid == 0)
            part[job] = make_float2(mean, sum);
    }
}

template <class T, class O>
__global__ void __launch_bounds__(256) k_norm_long(const T *x, const float *__restrict__ w, const float *__restrict__ b,
                                                   float eps, size_t m, int d, int slices,
                                                   const float2 *__restrict__ part, O *y, float *__restrict__ stats)
{
    using ch = chunk<T>;
    using at = spot<ch::E>;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    for (size_t job = blockIdx.x; job < m * slices; job += gridDim.x) {
        const size_t row = job / slices;
        const int k = (int)(job - row * slices), first = k * kSlice<T>;
        const int len = d - first < kSlice<T> ? d - first : kSlice<T>, nc = (len + ch::E - 1) / ch::E;
        const size_t from = row * d + first;
        ch v[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
            if (tid + i * 256 < nc)
                v[i].load(x + from, at(tid + i * 256, len));
        // every wave joins the row's slices by itself
        moments a = {0.0f, 0.0f, 0.0f};
        for (int i = lane; i < slices; i += 64) {
            const float2 q = part[row * slices + i];
            a.join((float)(i + 1 < slices ? kSlice<T> : d - i * kSlice<T>), q.x, q.y);
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            // lower lanes first, on both sides of the exchange
            moments p = {__shfl_xor(a.n, o), __shfl_xor(a.mean, o), __shfl_xor(a.sum, o)};
            if (lane & o) {
                p.join(a.n, a.mean, a.sum);
                a = p;
            } else {
                a.join(p.n, p.mean, p.sum);
            }
        }
        const float mean = a.mean, rstd = 1.0f / sqrtf(a.sum / (float)d + eps);
        if (stats && k == 0 && tid == 0)
            *(float2 *)(stats + row * 2) = make_float2(mean, rstd);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = tid + i * 256;
            if (c >= nc)
                break;
            ch wv, bv;
            if (w)
                wv.load(w + first, at(c, len));
            else
                wv.fill(1.0f);
            if (b)
                bv.load(b + first, at(c, len));
            else
                bv.fill(0.0f);
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                v[i].v[e] = (v[i].v[e] - mean) * rstd * wv.v[e] + bv.v[e];
            v[i].store(y + from, at(c, len));
        }
    }
}

// What the backward sums: a block owns 256 chunks of columns and every gridDim.y'th row,
// four of them on their way at a time.  Each row's sums of h and h n over these
// columns go to rows [m][gridDim.x], the block's own of dw and db (unless NULL) to
// part [gridDim.y][2][d].
template <class T, class G>
__global__ void __launch_bounds__(256) k_norm_sums(const T *__restrict__ x, const float *__restrict__ w,
                                                   const float *__restrict__ stats, const G *__restrict__ dy, size_t m, int d,
                                                   float2 *__restrict__ rows, float *__restrict__ part)
{
    using ch = chunk<T>;
    using at = spot<ch::E>;
    constexpr int U = 4;
    __shared__ float red[2][4][2 * U];
    const int tid = (int)threadIdx.x, c = (int)blockIdx.x * 256 + tid;
    ch gw, gb, wv;
    gw.fill(0.0f);
    gb.fill(0.0f);
    wv.fill(1.0f);
    const at k(c, d);
    const bool in = c * ch::E < d;
    if (w && in)
        wv.load(w, k);
    int turn = 0;
    for (size_t r0 = blockIdx.y; r0 < m; r0 += (size_t)gridDim.y * U, turn ^= 1) {
        piece<T, T> n[U];
        piece<T, G> g[U];
        float2 st[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t row = r0 + (size_t)u * gridDim.y;
            n[u].q = {};
            g[u].q = {};
            st[u] = make_float2(0.0f, 0.0f);
            if (row < m && in) {
                n[u].load(x + row * d, k);
                g[u].load(dy + row * d, k);
                st[u] = *(const float2 *)(stats + row * 2);
            }
        }
        float s[2 * U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[2 * u] = s[2 * u + 1] = 0.0f;
            if (in)
                g[u].own(k);
#pragma unroll
            for (int e = 0; e < ch::E; ++e) {
                const float f = (n[u][e] - st[u].x) * st[u].y, h = g[u][e] * wv.v[e]; // (beside a g of 0 if not its own)
                gw.v[e] += g[u][e] * f;
                gb.v[e] += g[u][e];
                s[2 * u] += h;
                s[2 * u + 1] += h * f;
            }
        }
        row_sum<256>(s, red[turn], tid);
        if (tid < U) {
            const size_t row = r0 + (size_t)tid * gridDim.y;
            if (row < m) {
                float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u == tid)
                        v = make_float2(s[2 * u], s[2 * u + 1]);
                rows[row * gridDim.x + blockIdx.x] = v;
            }
        }
    }
    if (part && in) {
        float *out = part + (size_t)blockIdx.y * 2 * d;
        gw.store(out, k);
        gb.store(out + d, k);
    }
}

// dx of a slice, and behind the slices' blocks the joining of dw and db
template <class T, class G, class O>
__global__ void __launch_bounds__(256) k_norm_bwd_long(const T *__restrict__ x, const float *__restrict__ w,
                                                       const float *__restrict__ stats, const G *__restrict__ dy, size_t m,
                                                       int d, int slices, int blocks, const float2 *__restrict__ rows,
                                                       int across, O *__restrict__ dx, int beta,
                                                       const float *__restrict__ part, int parts, float *dw, int beta_w,
                                                       float *db, int beta_b)
{
    using ch = chunk<T>;
    using at = spot<ch::E>;
    if ((int)blockIdx.x >= blocks) {
        join_sums<256>(part, parts, d, (int)blockIdx.x - blocks, dw, beta_w, db, beta_b);
        return;
    }
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const float inv = 1.0f / (float)d;
    for (size_t job = blockIdx.x; job < m * slices; job += blocks) {
        const size_t row = job / slices;
        const int first = (int)(job - row * slices) * kSlice<T>, len = d - first < kSlice<T> ? d - first : kSlice<T>;
        const size_t from = row * d + first;
        const int nc = (len + ch::E - 1) / ch::E;
        piece<T, T> n[kChunks];
        piece<T, G> g[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
            if (tid + i * 256 < nc) {
                n[i].load(x + from, at(tid + i * 256, len));
                g[i].load(dy + from, at(tid + i * 256, len));
            }
        const float2 st = *(const float2 *)(stats + row * 2), s = slice_sums(rows + row * across, across, lane);
        const float c1 = s.x * inv, c2 = s.y * inv;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = tid + i * 256;
            if (c >= nc)
                break;
            ch wv, o;
            if (w)
                wv.load(w + first, at(c, len));
            else
                wv.fill(1.0f);
            if (beta)
                o.load(dx + from, at(c, len));
            else
                o.fill(0.0f);
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                o.v[e] += st.y * (g[i][e] * wv.v[e] - c1 - (n[i][e] - st.x) * st.y * c2);
            o.store(dx + from, at(c, len));
        }
    }
}

// ---------------------------------------------------------------- launches

int elements(int dtype) { return dtype == 0 ? 4 : 8; } // of a chunk
size_t chunks(int dtype, size_t d) { return (d + elements(dtype) - 1) / elements(dtype); }
size_t slices_of(int dtype, size_t d) { return (chunks(dtype, d) + 256 * kChunks - 1) / (256 * kChunks); }

unsigned grid_of(size_t n) { return (unsigned)(n < kMostBlocks ? n : kMostBlocks); }

// Threads per row, of two chunks each (more would not leave registers for the next
// row), as the row's c chunks need them; 1024 of up to eight each for many longer rows
// of the forward (a block's row of 50000 takes 15 us, so that slices of it on every CU
// are faster for few).  0: slices.
int threads_per_row(size_t m, size_t c, bool backward)
{
    return c <= 8 * 2 ? 8 : c <= 64 * 2 ? 64 : c <= 256 * 2 ? 256 : c <= 512 * 2 ? 512 : !backward && c <= 1024 * 8 && m >= 256 ? 1024 : 0;
}
template <class FN>
void by_row(int tpr, FN fn)
{
    using std::integral_constant;
    if (tpr == 8)
        fn(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else if (tpr == 64)
        fn(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (tpr == 256)
        fn(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else
        fn(integral_constant<int, 512>{}, integral_constant<int, 2>{});
}

// Blocks of the backward, each of which leaves its sums of 2 d floats: two per CU, of
// the longest rows one (8192 x 8192 in bf16: 94 us, with two 101, with four 115)
size_t bwd_blocks(size_t m, int tpr)
{
    const size_t rows = tpr < 256 ? 256 / tpr : 1, n = (m + rows - 1) / rows, most = tpr == 512 ? 256 : 512;
    return n < most ? n : most;
}
// row groups of the sums of longer rows: some 512 blocks, four rows each at least
size_t across_of(int dtype, size_t d) { return (chunks(dtype, d) + 255) / 256; }
size_t long_groups(int dtype, size_t m, size_t d)
{
    const size_t a = across_of(dtype, d), n = a < 512 ? 512 / a : 1, most = (m + 3) / 4;
    return most < n ? most : n;
}

template <class FN>
int by_type(int dtype, FN fn)
{
    return dtype == 0 ? fn((float *)nullptr) : dtype == 1 ? fn((_Float16 *)nullptr) : fn((__bf16 *)nullptr);
}
// the type itself, or f32
template <class T, class FN>
int type_or_f32(int dtype, FN fn)
{
    return dtype == 0 ? fn((float *)nullptr) : fn((T *)nullptr);
}

template <class T, class O>
int forward(const pgk_norm_args &a, const T *x, O *y, float2 *ws, hipStream_t st)
{
    const size_t c = chunks(a.dtype, a.d);
    const int tpr = threads_per_row(a.m, c, false);
    if (tpr) {
        const int nt = tpr < 256 ? 256 : tpr;
        // a few rows to a block, so that the weights are read less often than x
        const size_t blocks = (a.m + nt / tpr - 1) / (nt / tpr), most = 2048 * 256 / nt;
        const dim3 grid((unsigned)(blocks < most ? blocks : most));
        auto go = [&](auto n, auto r) {
            constexpr int TPR = decltype(n)::value, R = decltype(r)::value;
            hipLaunchKernelGGL((k_norm<T, O, TPR, R, (TPR < 1024)>), grid, dim3(nt), 0, st, x, a.w, a.b, a.eps, a.m, (int)a.d, y,
                               a.stats);
        };
        if (tpr < 1024)
            by_row(tpr, go);
        else if (c <= 1024 * 4)
            go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
        else
            go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 8>{});
        return (int)hipGetLastError();
    }
    const size_t slices = slices_of(a.dtype, a.d);
    const dim3 grid(grid_of(a.m * slices));
    hipLaunchKernelGGL(k_norm_slices<T>, grid, dim3(256), 0, st, x, a.m, (int)a.d, (int)slices, ws);
    if (const int rc = (int)hipGetLastError())
        return rc;
    hipLaunchKernelGGL((k_norm_long<T, O>), grid, dim3(256), 0, st, x, a.w, a.b, a.eps, a.m, (int)a.d, (int)slices, ws, y,
                       a.stats);
    return (int)hipGetLastError();
}

template <class T, class G, class O>
int backward(const pgk_norm_args &a, const T *x, const G *dy, O *dx, void *ws, hipStream_t st)
{
    const int tpr = threads_per_row(a.m, chunks(a.dtype, a.d), true);
    const bool sums = a.dw || a.db;
    const int fin = sums ? 2 * (int)((a.d + 63) / 64) : 0;
    if (tpr) {
        const size_t parts = bwd_blocks(a.m, tpr);
        float *const part = sums ? (float *)ws : NULL;
        by_row(tpr, [&](auto n, auto r) {
            hipLaunchKernelGGL((k_norm_bwd<T, G, O, decltype(n)::value, decltype(r)::value>), dim3((unsigned)parts),
                               dim3(tpr < 256 ? 256 : tpr), 0, st, x, a.w, a.stats, dy, a.m, (int)a.d, dx, a.beta_x, part);
        });
        if (const int rc = (int)hipGetLastError())
            return rc;
        if (sums)
            hipLaunchKernelGGL(k_norm_fin, dim3((unsigned)fin), dim3(1024), 0, st, part, (int)parts, (int)a.d, a.dw, a.beta_w,
                               a.db, a.beta_b);
        return (int)hipGetLastError();
    }
    const size_t slices = slices_of(a.dtype, a.d), across = across_of(a.dtype, a.d), groups = long_groups(a.dtype, a.m, a.d);
    float2 *const rows = (float2 *)ws;
    float *const part = sums ? (float *)(rows + a.m * across) : NULL;
    hipLaunchKernelGGL((k_norm_sums<T, G>), dim3((unsigned)across, (unsigned)groups), dim3(256), 0, st, x, a.w, a.stats, dy, a.m,
                       (int)a.d, rows, part);
    if (const int rc = (int)hipGetLastError())
        return rc;
    const unsigned blocks = dx ? grid_of(a.m * slices) : 0;
    hipLaunchKernelGGL((k_norm_bwd_long<T, G, O>), dim3(blocks + (unsigned)fin), dim3(256), 0, st, x, a.w, a.stats, dy, a.m,
                       (int)a.d, (int)slices, (int)blocks, rows, (int)across, dx, a.beta_x, part, (int)groups, a.dw, a.beta_w,
                       a.db, a.beta_b);
    return (int)hipGetLastError();
}

bool fits(const pgk_norm_args *a) { return a->m && a->m <= 0x7fffffff && a->d && a->d <= PGK_NORM_MAX_D; }

} // namespace

extern "C" size_t pgk_norm_workspace(int dtype, size_t m, size_t d)
{
    return threads_per_row(m, chunks(dtype, d), false) ? 0 : m * slices_of(dtype, d) * sizeof(float2);
}

extern "C" int pgk_norm(const pgk_norm_args *a, void *ws, pgk_stream s)
{
    if (!fits(a))
        return (int)hipErrorInvalidValue;
    return by_type(a->dtype, [&](auto t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return type_or_f32<T>(a->y_dtype, [&](auto o) {
            return forward(*a, (const T *)a->x, (decltype(o))a->y, (float2 *)ws, (hipStream_t)s);
        });
    });
}

extern "C" size_t pgk_norm_bwd_workspace(int dtype, size_t m, size_t d, int sums)
{
    const int tpr = threads_per_row(m, chunks(dtype, d), true);
    if (tpr)
        return sums ? bwd_blocks(m, tpr) * 2 * d * sizeof(float) : 0;
    return m * across_of(dtype, d) * sizeof(float2) + (sums ? long_groups(dtype, m, d) * 2 * d * sizeof(float) : 0);
}

extern "C" int pgk_norm_bwd(const pgk_norm_args *a, void *ws, pgk_stream s)
{
    if (!fits(a))
        return (int)hipErrorInvalidValue;
    return by_type(a->dtype, [&](auto t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return type_or_f32<T>(a->dy_dtype, [&](auto g) {
            using G = std::remove_pointer_t<decltype(g)>;
            return type_or_f32<T>(a->dx_dtype, [&](auto o) {
                return backward(*a, (const T *)a->x, (const G *)a->dy, (decltype(o))a->dx, ws, (hipStream_t)s);
            });
        });
    });
}
