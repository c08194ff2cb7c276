// Distillation of a student's logits from a teacher's top logits, with the
// grad of the logits.
//
// Per row s [v] with the teacher's logits t_k at the indices i_k (an index
// outside [0, v) is padding) and a label (outside: none):
//   p = softmax(t / T) over the entries, q = softmax(s / T), r = softmax(s)
//   loss = scale (alpha T^2 sum_k p_k (log p_k - log q_{i_k}) + (1 - alpha) (-log r_label))
//   ds_j = scale up (alpha T (q_j - sum_{k: i_k = j} p_k) + (1 - alpha) (r_j - [j = label]))
// A row without entries (all padding, or all at -inf) has no first part, one
// without a label no second; a row with neither has loss and grad 0, whatever
// its logits hold.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <math.h>

#include "convert16.h"
#include "launch.h"
#include "pgmath.h"

namespace {

constexpr float kLog2e = 1.44269504089f;

template <class T>
__device__ __forceinline__ float ld(const void *p, size_t i)
{
    return (float)((const T *)p)[i];
}
__device__ __forceinline__ float ld_any(int dtype, const void *p, size_t i)
{
    return dtype == 0 ? ld<float>(p, i) : dtype == 1 ? ld<_Float16>(p, i) : ld<__bf16>(p, i);
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1)
        v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1)
        v += __shfl_xor(v, o);
    return v;
}

// What a row's teacher and label say, in LDS: entry e < n has index idx[e]
// (< 0: padding), probability p[e] and its logarithm; entry k is the label.
struct row_head {
    int idx[PGK_DISTILL_TOP + 1];
    float p[PGK_DISTILL_TOP + 1], logp[PGK_DISTILL_TOP + 1];
    int some, has;
};

// filled by the block's first wave
__device__ __forceinline__ void load_head(const pgk_distill_args &a, size_t row, row_head *h, int lane)
{
    const float inv_t = 1.0f / a.temperature;
    float tmax = -INFINITY;
    int some = 0;
    float t[PGK_DISTILL_TOP / 64];
#pragma unroll
    for (int q = 0; q < PGK_DISTILL_TOP / 64; ++q) {
        const int e = q * 64 + lane;
        t[q] = -INFINITY;
        if (e < a.top) {
            const float f = a.idx[row * a.top + e];
            const bool there = f >= 0.0f && f < (float)a.v;
            h->idx[e] = there ? (int)f : -1;
            if (there)
                t[q] = ld_any(a.top_dtype, a.t, row * a.top + e) * inv_t;
            some |= !(t[q] == -INFINITY);
            tmax = fmaxf(tmax, t[q]);
        }
    }
    tmax = wave_max(tmax);
    some = __any(some) && a.alpha > 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < PGK_DISTILL_TOP / 64; ++q)
        sum += t[q] == -INFINITY ? 0.0f : expf(t[q] - tmax);
    sum = wave_sum(sum);
    const float lsum = logf(sum);
#pragma unroll
    for (int q = 0; q < PGK_DISTILL_TOP / 64; ++q) {
        const int e = q * 64 + lane;
        if (e < a.top) {
            const bool zero = !some || t[q] == -INFINITY;
            h->p[e] = zero ? 0.0f : expf(t[q] - tmax) / sum;
            h->logp[e] = zero ? 0.0f : t[q] - tmax - lsum;
        }
    }
    if (lane == 0) {
        int lab = -1;
        if (a.label && a.alpha < 1.0f) {
            const float f = a.label[row];
            lab = f >= 0.0f && f < (float)a.v ? (int)f : -1;
        }
        h->idx[a.top] = lab;
        h->p[a.top] = 0.0f;
        h->some = some;
        h->has = lab >= 0;
    }
}

// The row's loss, by the block's first wave: zt and z1 are the sums of
// exp((s - m) / T) and exp(s - m).
template <class T>
__device__ __forceinline__ void store_loss(const pgk_distill_args &a, size_t row, const T *s, const row_head *h, float m,
                                           float zt, float z1, int lane)
{
    float kl = 0.0f;
    if (h->some) {
        const float inv_t = 1.0f / a.temperature, lz = logf(zt);
        for (int e = lane; e < a.top; e += 64) {
            const float p = h->p[e];
            if (h->idx[e] >= 0 && !(p == 0.0f))
                kl += p * (h->logp[e] - (((float)s[h->idx[e]] - m) * inv_t - lz));
        }
        kl = wave_sum(kl) * a.alpha * a.temperature * a.temperature;
    }
    if (lane == 0) {
        if (h->has)
            kl += (1.0f - a.alpha) * (logf(z1) - ((float)s[h->idx[a.top]] - m));
        a.loss[row] = a.scale * kl;
    }
}

// Grad entry e of the row (e == top: the label) where it is the first of its
// index: the whole grad of that logit, rounded once.
template <class T, class O>
__device__ __forceinline__ void fix_entry(const pgk_distill_args &a, const row_head *h, int e, float s, O *ds, float m,
                                          float ct, float wt, float w1, float c1, float c2)
{
    const int j = h->idx[e];
    float p = h->p[e];
    for (int i = e + 1; i < a.top; ++i)
        p += h->idx[i] == j ? h->p[i] : 0.0f;
    float v = -c1 * p;
    if (h->has && h->idx[a.top] == j)
        v -= c2;
    if (a.beta) { // the softmaxes have been added already
        ds[j] = (O)((float)ds[j] + v);
        return;
    }
    v += wt * PGM_EXP2((s - m) * ct);
    if (h->has)
        v += w1 * PGM_EXP2((s - m) * kLog2e);
    ds[j] = (O)v;
}

constexpr int kStreamThreads = 1024;

// One block per row, the row read twice (its maximum, its sums) and once more
// for the grad.
template <class T, class O>
__global__ void __launch_bounds__(kStreamThreads) k_distill_stream(pgk_distill_args a)
{
    __shared__ row_head h;
    __shared__ float red[3][kStreamThreads / 64];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x;
    const T *s = (const T *)a.s + row * a.v;
    O *ds = a.ds ? (O *)a.ds + row * a.v : nullptr;
    if (wave == 0)
        load_head(a, row, &h, lane);
    float m = -INFINITY;
    for (size_t i = tid; i < a.v; i += kStreamThreads)
        m = fmaxf(m, (float)s[i]);
    m = wave_max(m);
    if (lane == 0)
        red[0][wave] = m;
    __syncthreads();
    m = red[0][0];
    for (int w = 1; w < kStreamThreads / 64; ++w)
        m = fmaxf(m, red[0][w]);
    const bool some = h.some, has = h.has;
    if (!some && !has) {
        if (tid == 0 && a.loss)
            a.loss[row] = 0.0f;
        if (ds && !a.beta)
            for (size_t i = tid; i < a.v; i += kStreamThreads)
                ds[i] = (O)0.0f;
        return;
    }
    const float ct = kLog2e / a.temperature;
    float zt = 0.0f, z1 = 0.0f;
    for (size_t i = tid; i < a.v; i += kStreamThreads) {
        const float d = (float)s[i] - m;
        zt += some ? PGM_EXP2(d * ct) : 0.0f;
        z1 += has ? PGM_EXP2(d * kLog2e) : 0.0f;
    }
    zt = wave_sum(zt);
    z1 = wave_sum(z1);
    if (lane == 0) {
        red[1][wave] = zt;
        red[2][wave] = z1;
    }
    __syncthreads();
    zt = z1 = 0.0f;
    for (int w = 0; w < kStreamThreads / 64; ++w) {
        zt += red[1][w];
        z1 += red[2][w];
    }
    if (a.loss && wave == 0)
        store_loss<T>(a, row, s, &h, m, zt, z1, lane);
    if (!ds)
        return;
    const float up = a.up ? a.up[0] : 1.0f;
    const float c1 = some ? a.scale * up * a.alpha * a.temperature : 0.0f, c2 = has ? a.scale * up * (1.0f - a.alpha) : 0.0f;
    const float wt = some ? c1 / zt : 0.0f, w1 = has ? c2 / z1 : 0.0f;
    // the entries' logits, before a grad written in place of the logits covers them
    float mine = 0.0f;
    bool fix = tid <= a.top && h.idx[tid] >= 0;
    if (fix) {
        for (int e = 0; e < tid; ++e)
            fix = fix && h.idx[e] != h.idx[tid];
        mine = (float)s[h.idx[tid]];
    }
    __syncthreads();
    for (size_t i = tid; i < a.v; i += kStreamThreads) {
        const float d = (float)s[i] - m;
        float v = some ? wt * PGM_EXP2(d * ct) : 0.0f;
        v += has ? w1 * PGM_EXP2(d * kLog2e) : 0.0f;
        ds[i] = (O)(a.beta ? (float)ds[i] + v : v);
    }
    __syncthreads();
    if (fix)
        fix_entry<T, O>(a, &h, tid, mine, ds, m, ct, wt, w1, c1, c2);
}

template <class T, class O>
int launch(const pgk_distill_args &a, hipStream_t st)
{
    hipLaunchKernelGGL((k_distill_stream<T, O>), dim3((unsigned)a.n), dim3(kStreamThreads), 0, st, a);
    return (int)hipGetLastError();
}

} // namespace

extern "C" int pgk_distill(const pgk_distill_args *a, pgk_stream s)
{
    if (!a->n || !a->v)
        return 0;
    if (a->n > 0x7fffffff || a->v > PGK_DISTILL_MAX_V || a->top < 1 || a->top > PGK_DISTILL_TOP ||
        (a->ds && a->ds_dtype != a->dtype && a->ds_dtype != 0))
        return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)s;
    const bool wide = !a->ds || a->ds_dtype == 0;
    if (a->dtype == 0)
        return launch<float, float>(*a, st);
    if (a->dtype == 1)
        return wide ? launch<_Float16, float>(*a, st) : launch<_Float16, _Float16>(*a, st);
    return wide ? launch<__bf16, float>(*a, st) : launch<__bf16, __bf16>(*a, st);
}
