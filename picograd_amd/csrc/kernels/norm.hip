// Layer norm over the rows of x [m, d] and its backward.
//
//   n = (x - mean) rstd, mean = sum x / d, rstd = 1 / sqrt(sum (x - mean)^2 / d + eps)
//   y = n w + b
//   h = dy w: dx = rstd (h - sum h / d - n sum (h n) / d), dw = sum over rows of dy n, db = of dy
//
// Statistics and sums are f32 from values held in registers (the variance is of
// the differences from the mean, not of squares); y and dx round once.  A row
// that a block holds is read once; longer ones are cut into slices for blocks of
// their own and read twice.  Bound by the stream of the rows: HBM for large
// calls, the launch and a row's loads for small ones.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include <type_traits>

#include "launch.h"

namespace {

constexpr int kChunks = 4;            // of 16 bytes of x, per thread
constexpr unsigned kMostBlocks = 1u << 20; // of a grid; kernels loop past it

// 16 bytes of x's type, at any alignment of an element
template <class T>
struct chunk {
    static constexpr int E = 16 / sizeof(T);
    float v[E];
    template <class S> // elements c E .. of the row p [d]; past the end: 0
    __device__ __forceinline__ void load(const S *p, int c, int d)
    {
        typedef S sv __attribute__((ext_vector_type(E), aligned(sizeof(S))));
        const int at = c * E, left = d - at;
        if (left >= E) {
            const sv q = *(const sv *)(p + at);
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[e] = (float)q[e];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[e] = e < left ? (float)p[at + e] : 0.0f;
        }
    }
    template <class O>
    __device__ __forceinline__ void store(O *p, int c, int d) const
    {
        typedef O ov __attribute__((ext_vector_type(E), aligned(sizeof(O))));
        const int at = c * E, left = d - at;
        if (left >= E) {
            ov q;
#pragma unroll
            for (int e = 0; e < E; ++e)
                q[e] = (O)v[e];
            *(ov *)(p + at) = q;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < left)
                    p[at + e] = (O)v[e];
        }
    }
    __device__ __forceinline__ void fill(float f)
    {
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] = f;
    }
};

// sums over the TPR threads that share a row, in a fixed order.  TPR over 64:
// through `red` [waves of a row], which the caller does not reuse before the
// next barrier but one
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float (*red)[N], int tid)
{
#pragma unroll
    for (int o = TPR < 64 ? TPR / 2 : 32; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i)
            s[i] += __shfl_xor(s[i], o);
    if constexpr (TPR > 64) {
        if ((tid & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i)
                red[tid >> 6][i] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < TPR / 64; ++w)
                s[i] += red[w][i];
        }
    }
}

// ---------------------------------------------------------------- rows that a block holds

// TPR threads per row, kChunks chunks each; a block of 256 threads takes 256 / TPR
// rows, one of 1024 threads one.
template <class T, class O, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_norm(const T *x, const float *__restrict__ w,
                                                                const float *__restrict__ b, float eps, size_t m, int d,
                                                                O *y, float *__restrict__ stats)
{
    using ch = chunk<T>;
    constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
    __shared__ float red[4][TPR > 64 ? TPR / 64 : 1][1];
    const int tid = (int)threadIdx.x, lane = tid % TPR;
    const int nc = (d + ch::E - 1) / ch::E;
    int turn = 0;
    for (size_t r0 = (size_t)blockIdx.x * RPB; r0 < m; r0 += (size_t)gridDim.x * RPB, turn ^= 2) {
        const size_t row = r0 + tid / TPR;
        const bool in = row < m;
        const T *p = x + (in ? row : 0) * d;
        ch v[kChunks];
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
            if (lane + i * TPR < nc)
                v[i].load(p, lane + i * TPR, d);
            else
                v[i].fill(0.0f);
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                s[0] += v[i].v[e];
        row_sum<TPR>(s, red[turn], tid);
        const float mean = s[0] / (float)d;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
            for (int e = 0; e < ch::E; ++e) {
                const float c = v[i].v[e] - mean;
                s[0] += (lane + i * TPR) * ch::E + e < d ? c * c : 0.0f;
            }
        row_sum<TPR>(s, red[turn + 1], tid);
        const float rstd = 1.0f / sqrtf(s[0] / (float)d + eps);
        if (!in)
            continue;
        if (stats && lane == 0)
            *(float2 *)(stats + row * 2) = make_float2(mean, rstd);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = lane + i * TPR;
            if (c >= nc)
                break;
            ch wv, bv;
            if (w)
                wv.load(w, c, d);
            else
                wv.fill(1.0f);
            if (b)
                bv.load(b, c, d);
            else
                bv.fill(0.0f);
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                v[i].v[e] = (v[i].v[e] - mean) * rstd * wv.v[e] + bv.v[e];
            v[i].store(y + row * d, c, d);
        }
    }
}

// The grads of a block's rows: dx, and the block's own sums of dw and db to part
// [blocks][2][d] (NULL: not wanted), each thread those of its own columns.
template <class T, class G, class O, int TPR>
__global__ void __launch_bounds__(256) k_norm_bwd(const T *__restrict__ x, const float *__restrict__ w,
                                                  const float *__restrict__ stats, const G *__restrict__ dy, size_t m,
                                                  int d, O *__restrict__ dx, int beta, float *__restrict__ part)
{
    using ch = chunk<T>;
    constexpr int RPB = 256 / TPR, COLS = TPR * kChunks * ch::E;
    __shared__ float red[2][TPR > 64 ? TPR / 64 : 1][2];
    __shared__ float sums[RPB > 1 ? RPB : 1][RPB > 1 ? COLS : 1];
    const int tid = (int)threadIdx.x, lane = tid % TPR, group = tid / TPR;
    const int nc = (d + ch::E - 1) / ch::E;
    const float inv = 1.0f / (float)d;
    ch gw[kChunks], gb[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        gw[i].fill(0.0f);
        gb[i].fill(0.0f);
    }
    int turn = 0;
    for (size_t r0 = (size_t)blockIdx.x * RPB; r0 < m; r0 += (size_t)gridDim.x * RPB, turn ^= 1) {
        const size_t row = r0 + group;
        const bool in = row < m;
        const size_t at = (in ? row : 0) * d;
        const float2 st = in ? *(const float2 *)(stats + row * 2) : make_float2(0.0f, 0.0f);
        ch n[kChunks], h[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = lane + i * TPR;
            if (in && c < nc) {
                n[i].load(x + at, c, d);
                h[i].load(dy + at, c, d);
            } else {
                n[i].fill(st.x);
                h[i].fill(0.0f);
            }
        }
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = lane + i * TPR;
            ch wv;
            if (w && c < nc)
                wv.load(w, c, d);
            else
                wv.fill(1.0f);
#pragma unroll
            for (int e = 0; e < ch::E; ++e) {
                // (past the end of a row dy is 0 and n is never stored)
                const float g = h[i].v[e];
                n[i].v[e] = c * ch::E + e < d ? (n[i].v[e] - st.x) * st.y : 0.0f;
                gw[i].v[e] += g * n[i].v[e];
                gb[i].v[e] += g;
                h[i].v[e] = g * wv.v[e];
                s[0] += h[i].v[e];
                s[1] += h[i].v[e] * n[i].v[e];
            }
        }
        row_sum<TPR>(s, red[turn], tid);
        if (!dx || !in)
            continue;
        const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = lane + i * TPR;
            if (c >= nc)
                break;
            ch o;
            if (beta)
                o.load(dx + at, c, d);
            else
                o.fill(0.0f);
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                o.v[e] += st.y * (h[i].v[e] - c1 - n[i].v[e] * c2);
            o.store(dx + at, c, d);
        }
    }
    if (!part)
        return;
    // the groups' sums of a column in the groups' order
    auto leave = [&](ch(&g)[kChunks], float *out) {
        if constexpr (RPB == 1) {
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
                if (lane + i * TPR < nc)
                    g[i].store(out, lane + i * TPR, d);
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
#pragma unroll
                for (int e = 0; e < ch::E; ++e)
                    sums[group][(lane + i * TPR) * ch::E + e] = g[i].v[e];
            __syncthreads();
            for (int c = tid; c < d; c += 256) {
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

// dw and db (either NULL) from the blocks' sums, in a fixed order: 16 threads
// take every 16th block's of a column
__global__ void __launch_bounds__(1024) k_norm_fin(const float *__restrict__ part, int blocks, int d, float *dw, int beta_w,
                                                   float *db, int beta_b)
{
    __shared__ float s[16][64];
    const int col = (int)blockIdx.x * 64 + ((int)threadIdx.x & 63), k = (int)threadIdx.x >> 6;
    const bool second = blockIdx.y != 0;
    float *out = second ? db : dw;
    const int beta = second ? beta_b : beta_w;
    if (!out)
        return;
    float t = 0.0f;
    if (col < d) {
        const float *p = part + (second ? d : 0) + col;
#pragma unroll 4
        for (int i = k; i < blocks; i += 16)
            t += p[(size_t)i * 2 * d];
    }
    s[k][threadIdx.x & 63] = t;
    __syncthreads();
    if (k || col >= d)
        return;
    t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        t += s[i][threadIdx.x];
    out[col] = beta ? out[col] + t : t;
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
        sum += s2 + (q * n) * (q * f);
        n = all;
    }
};

template <class T>
__global__ void __launch_bounds__(256) k_norm_slices(const T *__restrict__ x, size_t m, int d, int slices,
                                                     float2 *__restrict__ part)
{
    using ch = chunk<T>;
    __shared__ float red[4][4][1];
    const int tid = (int)threadIdx.x;
    int turn = 0;
    for (size_t job = blockIdx.x; job < m * slices; job += gridDim.x, turn ^= 2) {
        const size_t row = job / slices;
        const int first = (int)(job - row * slices) * kSlice<T>, len = d - first < kSlice<T> ? d - first : kSlice<T>;
        const T *p = x + row * d + first;
        const int nc = (len + ch::E - 1) / ch::E;
        ch v[kChunks];
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
            if (tid + i * 256 < nc)
                v[i].load(p, tid + i * 256, len);
            else
                v[i].fill(0.0f);
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                s[0] += v[i].v[e];
        row_sum<256>(s, red[turn], tid);
        const float mean = s[0] / (float)len;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
            for (int e = 0; e < ch::E; ++e) {
                const float c = v[i].v[e] - mean;
                s[0] += (tid + i * 256) * ch::E + e < len ? c * c : 0.0f;
            }
        row_sum<256>(s, red[turn + 1], tid);
        if (tid == 0)
            part[job] = make_float2(mean, s[0]);
    }
}

template <class T, class O>
__global__ void __launch_bounds__(256) k_norm_long(const T *x, const float *__restrict__ w, const float *__restrict__ b,
                                                   float eps, size_t m, int d, int slices,
                                                   const float2 *__restrict__ part, O *y, float *__restrict__ stats)
{
    using ch = chunk<T>;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    for (size_t job = blockIdx.x; job < m * slices; job += gridDim.x) {
        const size_t row = job / slices;
        const int k = (int)(job - row * slices), first = k * kSlice<T>;
        const int len = d - first < kSlice<T> ? d - first : kSlice<T>, nc = (len + ch::E - 1) / ch::E;
        const size_t at = row * d + first;
        ch v[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
            if (tid + i * 256 < nc)
                v[i].load(x + at, tid + i * 256, len);
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
                wv.load(w + first, c, len);
            else
                wv.fill(1.0f);
            if (b)
                bv.load(b + first, c, len);
            else
                bv.fill(0.0f);
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                v[i].v[e] = (v[i].v[e] - mean) * rstd * wv.v[e] + bv.v[e];
            v[i].store(y + at, c, len);
        }
    }
}

// each slice's sums of h and h n
template <class T, class G>
__global__ void __launch_bounds__(256) k_norm_bwd_slices(const T *__restrict__ x, const float *__restrict__ w,
                                                         const float *__restrict__ stats, const G *__restrict__ dy,
                                                         size_t m, int d, int slices, float2 *__restrict__ part)
{
    using ch = chunk<T>;
    __shared__ float red[2][4][2];
    const int tid = (int)threadIdx.x;
    int turn = 0;
    for (size_t job = blockIdx.x; job < m * slices; job += gridDim.x, turn ^= 1) {
        const size_t row = job / slices;
        const int first = (int)(job - row * slices) * kSlice<T>, len = d - first < kSlice<T> ? d - first : kSlice<T>;
        const size_t at = row * d + first;
        const int nc = (len + ch::E - 1) / ch::E;
        const float2 st = *(const float2 *)(stats + row * 2);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = tid + i * 256;
            if (c >= nc)
                break;
            ch n, h, wv;
            n.load(x + at, c, len);
            h.load(dy + at, c, len);
            if (w)
                wv.load(w + first, c, len);
            else
                wv.fill(1.0f);
#pragma unroll
            for (int e = 0; e < ch::E; ++e)
                if (c * ch::E + e < len) {
                    const float f = h.v[e] * wv.v[e];
                    s[0] += f;
                    s[1] += f * ((n.v[e] - st.x) * st.y);
                }
        }
        row_sum<256>(s, red[turn], tid);
        if (tid == 0)
            part[job] = make_float2(s[0], s[1]);
    }
}

// A block owns a slice's columns and every gridDim.y'th row; its sums of dw and db
// to part [gridDim.y][2][d].
template <class T, class G, class O>
__global__ void __launch_bounds__(256) k_norm_bwd_long(const T *__restrict__ x, const float *__restrict__ w,
                                                       const float *__restrict__ stats, const G *__restrict__ dy, size_t m,
                                                       int d, int slices, const float2 *__restrict__ sums,
                                                       O *__restrict__ dx, int beta, float *__restrict__ part)
{
    using ch = chunk<T>;
    const int tid = (int)threadIdx.x, lane = tid & 63, first = (int)blockIdx.x * kSlice<T>;
    const int len = d - first < kSlice<T> ? d - first : kSlice<T>, nc = (len + ch::E - 1) / ch::E;
    const float inv = 1.0f / (float)d;
    ch gw[kChunks], gb[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        gw[i].fill(0.0f);
        gb[i].fill(0.0f);
    }
    for (size_t row = blockIdx.y; row < m; row += gridDim.y) {
        const size_t at = row * d + first;
        const float2 st = *(const float2 *)(stats + row * 2);
        float2 s = make_float2(0.0f, 0.0f);
        if (dx)
            s = slice_sums(sums + row * slices, slices, lane);
        const float c1 = s.x * inv, c2 = s.y * inv;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = tid + i * 256;
            if (c >= nc)
                break;
            ch n, h, wv, o;
            n.load(x + at, c, len);
            h.load(dy + at, c, len);
            if (w)
                wv.load(w + first, c, len);
            else
                wv.fill(1.0f);
            if (dx && beta)
                o.load(dx + at, c, len);
            else
                o.fill(0.0f);
#pragma unroll
            for (int e = 0; e < ch::E; ++e) {
                const float f = (n.v[e] - st.x) * st.y, g = h.v[e];
                gw[i].v[e] += g * f;
                gb[i].v[e] += g;
                o.v[e] += st.y * (g * wv.v[e] - c1 - f * c2);
            }
            if (dx)
                o.store(dx + at, c, len);
        }
    }
    if (!part)
        return;
    float *out = part + (size_t)blockIdx.y * 2 * d + first;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
        if (tid + i * 256 < nc) {
            gw[i].store(out, tid + i * 256, len);
            gb[i].store(out + d, tid + i * 256, len);
        }
}

// ---------------------------------------------------------------- launches

int elements(int dtype) { return dtype == 0 ? 4 : 8; } // of a chunk
size_t chunks(int dtype, size_t d) { return (d + elements(dtype) - 1) / elements(dtype); }
size_t slices_of(int dtype, size_t d) { return (chunks(dtype, d) + 256 * kChunks - 1) / (256 * kChunks); }

unsigned grid_of(size_t n) { return (unsigned)(n < kMostBlocks ? n : kMostBlocks); }

// threads per row, of the rows that 1024 (forward) or 256 threads (backward)
// hold; 0: longer
int threads_per_row(size_t c, bool backward)
{
    return c <= 8 * kChunks ? 8 : c <= 64 * kChunks ? 64 : c <= 256 * kChunks ? 256 : !backward && c <= 1024 * kChunks ? 1024 : 0;
}

// blocks of the backward: each leaves its sums of 2 d floats, so no more than two per CU
size_t bwd_blocks(size_t m, int tpr)
{
    const size_t rows = 256 / tpr, n = (m + rows - 1) / rows;
    return n < 512 ? n : 512;
}
// row groups of the backward of long rows: some 1024 blocks
size_t long_groups(size_t m, size_t slices)
{
    const size_t n = slices < 1024 ? 1024 / slices : 1;
    return m < n ? m : n;
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
    const int tpr = threads_per_row(chunks(a.dtype, a.d), false);
    if (tpr) {
        const int nt = tpr < 256 ? 256 : tpr;
        const dim3 grid(grid_of((a.m + nt / tpr - 1) / (nt / tpr)));
        auto go = [&](auto n) {
            hipLaunchKernelGGL((k_norm<T, O, decltype(n)::value>), grid, dim3(nt), 0, st, x, a.w, a.b, a.eps, a.m, (int)a.d, y,
                               a.stats);
        };
        if (tpr == 8)
            go(std::integral_constant<int, 8>{});
        else if (tpr == 64)
            go(std::integral_constant<int, 64>{});
        else if (tpr == 256)
            go(std::integral_constant<int, 256>{});
        else
            go(std::integral_constant<int, 1024>{});
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
    const int tpr = threads_per_row(chunks(a.dtype, a.d), true);
    const bool sums = a.dw || a.db;
    size_t parts;
    float *part = NULL;
    if (tpr) {
        parts = bwd_blocks(a.m, tpr);
        part = sums ? (float *)ws : NULL;
        auto go = [&](auto n) {
            hipLaunchKernelGGL((k_norm_bwd<T, G, O, decltype(n)::value>), dim3((unsigned)parts), dim3(256), 0, st, x, a.w,
                               a.stats, dy, a.m, (int)a.d, dx, a.beta_x, part);
        };
        if (tpr == 8)
            go(std::integral_constant<int, 8>{});
        else if (tpr == 64)
            go(std::integral_constant<int, 64>{});
        else
            go(std::integral_constant<int, 256>{});
    } else {
        const size_t slices = slices_of(a.dtype, a.d);
        float2 *const s = (float2 *)ws;
        parts = long_groups(a.m, slices);
        part = sums ? (float *)(s + a.m * slices) : NULL;
        if (dx)
            hipLaunchKernelGGL((k_norm_bwd_slices<T, G>), dim3(grid_of(a.m * slices)), dim3(256), 0, st, x, a.w, a.stats, dy,
                               a.m, (int)a.d, (int)slices, s);
        if (const int rc = (int)hipGetLastError())
            return rc;
        hipLaunchKernelGGL((k_norm_bwd_long<T, G, O>), dim3((unsigned)slices, (unsigned)parts), dim3(256), 0, st, x, a.w,
                           a.stats, dy, a.m, (int)a.d, (int)slices, s, dx, a.beta_x, part);
    }
    if (const int rc = (int)hipGetLastError())
        return rc;
    if (sums)
        hipLaunchKernelGGL(k_norm_fin, dim3((unsigned)((a.d + 63) / 64), 2), dim3(1024), 0, st, part, (int)parts, (int)a.d,
                           a.dw, a.beta_w, a.db, a.beta_b);
    return (int)hipGetLastError();
}

bool fits(const pgk_norm_args *a) { return a->m && a->m <= 0x7fffffff && a->d && a->d <= PGK_NORM_MAX_D; }

} // namespace

extern "C" size_t pgk_norm_workspace(int dtype, size_t m, size_t d)
{
    return threads_per_row(chunks(dtype, d), false) ? 0 : m * slices_of(dtype, d) * sizeof(float2);
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
    const int tpr = threads_per_row(chunks(dtype, d), true);
    if (tpr)
        return sums ? bwd_blocks(m, tpr) * 2 * d * sizeof(float) : 0;
    const size_t slices = slices_of(dtype, d);
    return m * slices * sizeof(float2) + (sums ? long_groups(m, slices) * 2 * d * sizeof(float) : 0);
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
