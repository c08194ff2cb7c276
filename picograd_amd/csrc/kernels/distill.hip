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

// A wave's maximum and sum, uniform: within rows of 16 lanes by shifts, then
// across the rows, the last lane has it.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float none, float v)
{
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(none), __float_as_uint(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float last_lane(float v)
{
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}
__device__ __forceinline__ float wave_max(float v)
{
    const float low = -INFINITY;
    v = fmaxf(v, dpp<0x111, 0xf>(low, v)); // row_shr 1, 2, 4, 8
    v = fmaxf(v, dpp<0x112, 0xf>(low, v));
    v = fmaxf(v, dpp<0x114, 0xf>(low, v));
    v = fmaxf(v, dpp<0x118, 0xf>(low, v));
    v = fmaxf(v, dpp<0x142, 0xa>(low, v)); // row_bcast 15, 31
    v = fmaxf(v, dpp<0x143, 0xc>(low, v));
    return last_lane(v);
}
__device__ __forceinline__ float wave_sum(float v)
{
    v += dpp<0x111, 0xf>(0.0f, v);
    v += dpp<0x112, 0xf>(0.0f, v);
    v += dpp<0x114, 0xf>(0.0f, v);
    v += dpp<0x118, 0xf>(0.0f, v);
    v += dpp<0x142, 0xa>(0.0f, v);
    v += dpp<0x143, 0xc>(0.0f, v);
    return last_lane(v);
}

// ---------------------------------------------------------------- a row's entries

// What a row's teacher and label say, in LDS: entry e < top has index idx[e]
// (< 0: padding), the teacher's logit over T and the student's logit s[e];
// entry `top` is the label.  Each of the first waves makes 64 entries and leaves
// their maximum and sum of exponentials.
constexpr int kHeadWaves = PGK_DISTILL_TOP / 64;
struct alignas(16) row_head {
    int idx[PGK_DISTILL_TOP + 4]; // read four at a time
    float t[PGK_DISTILL_TOP], s[PGK_DISTILL_TOP + 1];
    float tmax[kHeadWaves], tsum[kHeadWaves];
    int some[kHeadWaves], has;
};
// the threads that make it
__device__ __forceinline__ int head_threads(const pgk_distill_args &a) { return (a.top + 63) & ~63; }

// the teacher's softmax over the entries
struct teacher {
    float tmax, sum, lsum;
    bool some;
    __device__ teacher(const pgk_distill_args &a, const row_head &h)
    {
        tmax = -INFINITY, sum = 0.0f;
        int any = 0;
        const int n = head_threads(a) / 64;
        for (int i = 0; i < n; ++i) {
            tmax = fmaxf(tmax, h.tmax[i]);
            any |= h.some[i];
        }
        some = any && a.alpha > 0.0f;
        for (int i = 0; i < n; ++i)
            sum += h.tmax[i] == -INFINITY ? h.tsum[i] : h.tsum[i] * expf(h.tmax[i] - tmax);
        lsum = logf(sum);
    }
    __device__ float p(const row_head &h, int e) const
    {
        return !some || h.t[e] == -INFINITY ? 0.0f : expf(h.t[e] - tmax) / sum;
    }
    __device__ float logp(const row_head &h, int e) const { return h.t[e] - tmax - lsum; }
};

// An entry per thread of the first waves, in three steps so that the loads of
// the row proper are in flight between the indices' arrival and the logits
// they point to.
struct entry_loads {
    float f, t, label, s, slabel;
    __device__ __forceinline__ void begin(const pgk_distill_args &a, size_t row, int tid)
    {
        f = -1.0f, t = -INFINITY, label = -1.0f;
        if (tid < a.top) {
            f = a.idx[row * a.top + tid];
            t = ld_any(a.top_dtype, a.t, row * a.top + tid);
        }
        if (tid == 0 && a.label && a.alpha < 1.0f)
            label = a.label[row];
    }
    // (no row: its logits are elsewhere)
    template <class T>
    __device__ __forceinline__ void gather(const pgk_distill_args &a, const T *row, row_head &h, int tid)
    {
        const bool there = f >= 0.0f && f < (float)a.v;
        t = there ? t / a.temperature : -INFINITY;
        s = slabel = 0.0f;
        if (tid < a.top) {
            h.idx[tid] = there ? (int)f : -1;
            if (there && row)
                s = (float)row[(int)f];
        }
        if (tid == 0) {
            const bool has = label >= 0.0f && label < (float)a.v;
            if (has && row)
                slabel = (float)row[(int)label];
            h.idx[a.top] = has ? (int)label : -1;
            h.has = has;
        }
    }
    __device__ __forceinline__ void finish(const pgk_distill_args &a, row_head &h, int tid)
    {
        if (tid < a.top) {
            h.t[tid] = t;
            h.s[tid] = s;
        }
        const float m = wave_max(t);
        const float sum = wave_sum(t == -INFINITY ? 0.0f : expf(t - m));
        const bool some = __any(!(t == -INFINITY));
        if ((tid & 63) == 0) {
            h.tmax[tid >> 6] = m;
            h.tsum[tid >> 6] = sum;
            h.some[tid >> 6] = some;
        }
        if (tid == 0)
            h.s[a.top] = slabel;
    }
};

// ---------------------------------------------------------------- a row's softmaxes

// Reference of a running softmax: exponents are taken against it, and 0 stands
// in while every value seen is -inf, whose exponentials are then 0.
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }

// what a launch sums: exp((s - m) / T) and exp(s - m), one sum for both at T = 1
struct wants {
    bool zt, z1;
    float ct;
    __device__ explicit wants(const pgk_distill_args &a)
    {
        const bool one = a.temperature == 1.0f, first = a.alpha > 0.0f, second = a.label && a.alpha < 1.0f;
        zt = first || (one && second);
        z1 = second && !one;
        ct = kLog2e / a.temperature;
    }
};

// maximum and the two sums
struct stats {
    float m, zt, z1;
    __device__ float sum1(const wants &w) const { return w.z1 ? z1 : zt; }
};
__device__ __forceinline__ void join(stats &a, const stats &b, const wants &w)
{
    const float m = fmaxf(a.m, b.m), r = finite_ref(m);
    if (w.zt)
        a.zt = a.zt * PGM_EXP2((a.m - r) * w.ct) + b.zt * PGM_EXP2((b.m - r) * w.ct);
    if (w.z1)
        a.z1 = a.z1 * PGM_EXP2((a.m - r) * kLog2e) + b.z1 * PGM_EXP2((b.m - r) * kLog2e);
    a.m = m;
}
// of one value; a NaN shows in the sums
__device__ __forceinline__ stats stats_of(float v)
{
    if (v != v)
        return {-INFINITY, v, v};
    const float one = v == -INFINITY ? 0.0f : 1.0f;
    return {v, one, one};
}

// A barrier for LDS alone: loads and stores of memory stay in flight.
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_s_waitcnt(0xc07f); // lgkmcnt 0, vmcnt and expcnt at their maximum
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

// over a wave, then over the block by way of LDS; every LDS write of the
// block's threads before it is seen after it
__device__ __forceinline__ stats wave_join(const stats &st, const wants &w)
{
    const float m = wave_max(st.m), d = st.m - finite_ref(m);
    return {m, w.zt ? wave_sum(st.zt * PGM_EXP2(d * w.ct)) : 0.0f, w.z1 ? wave_sum(st.z1 * PGM_EXP2(d * kLog2e)) : 0.0f};
}
template <int NT>
__device__ __forceinline__ stats block_join(stats st, const wants &w, stats *red, int tid)
{
    st = wave_join(st, w);
    if ((tid & 63) == 0)
        red[tid >> 6] = st;
    lds_barrier();
    const int lane = tid & 63;
    st = {-INFINITY, 0.0f, 0.0f};
    if (lane < NT / 64)
        st = red[lane];
    return wave_join(st, w);
}

// The row's loss, by one wave.
__device__ __forceinline__ void store_loss(const pgk_distill_args &a, size_t row, const row_head &h, const stats &st,
                                           const wants &w, int lane)
{
    const teacher t(a, h);
    float kl = 0.0f;
    if (t.some) {
        const float inv_t = 1.0f / a.temperature, lz = logf(st.zt);
        for (int e = lane; e < a.top; e += 64) {
            const float p = t.p(h, e);
            if (!(p == 0.0f))
                kl += p * (t.logp(h, e) - ((h.s[e] - st.m) * inv_t - lz));
        }
        kl = wave_sum(kl) * a.alpha * a.temperature * a.temperature;
    }
    if (lane == 0) {
        if (h.has)
            kl += (1.0f - a.alpha) * (logf(st.sum1(w)) - (h.s[a.top] - st.m));
        a.loss[row] = a.scale * kl;
    }
}

// The coefficients of a row's grad: ds = wt exp((s - m) / T) + w1 exp(s - m),
// less c1 p and c2 at the entries and the label.  any: the row has a target;
// one: the second exponential is there (at T = 1 the first stands for both).
struct coefs {
    float m, ct, wt, w1, c1, c2;
    bool any, one;
    __device__ coefs() {}
    __device__ coefs(const pgk_distill_args &a, const row_head &h, const stats &st, const wants &w) : m(st.m), ct(w.ct)
    {
        int some = 0;
        for (int i = 0; i < head_threads(a) / 64; ++i)
            some |= h.some[i];
        some = __builtin_amdgcn_readfirstlane(some) && a.alpha > 0.0f;
        const bool has = __builtin_amdgcn_readfirstlane(h.has);
        const float up = a.scale * (a.up ? a.up[0] : 1.0f);
        any = some || has;
        one = has && a.temperature != 1.0f;
        c1 = some ? up * a.alpha * a.temperature : 0.0f;
        c2 = has ? up * (1.0f - a.alpha) : 0.0f;
        wt = some ? c1 / st.zt : 0.0f;
        w1 = has ? c2 / st.sum1(w) : 0.0f;
        if (a.temperature == 1.0f)
            wt += w1;
    }
    template <bool ONE>
    __device__ __forceinline__ float at(float s) const
    {
        const float d = s - m;
        const float v = wt * PGM_EXP2(d * ct);
        return ONE ? v + w1 * PGM_EXP2(d * kLog2e) : v;
    }
    __device__ float at(float s) const { return one ? at<true>(s) : at<false>(s); }
};

// Grad entry e of the row (e == top: the label), where it is the first of its
// index: the whole grad of that logit, rounded once.
template <class O>
__device__ __forceinline__ void fix_entry(const pgk_distill_args &a, const row_head &h, int e, O *ds, const coefs &c)
{
    const int j = h.idx[e];
    if (j < 0)
        return;
    int same = 0, before = 0;
    for (int i = 0; i < a.top; i += 4) {
        const int4 q = *(const int4 *)&h.idx[i];
        const int s0 = q.x == j, s1 = q.y == j && i + 1 < a.top, s2 = q.z == j && i + 2 < a.top, s3 = q.w == j && i + 3 < a.top;
        same += s0 + s1 + s2 + s3;
        before |= (s0 && i < e) | (s1 && i + 1 < e) | (s2 && i + 2 < e) | (s3 && i + 3 < e);
    }
    if (before)
        return;
    const teacher t(a, h);
    float p = 0.0f;
    if (same == 1 && e < a.top)
        p = t.p(h, e);
    else if (same)
        for (int i = 0; i < a.top; ++i)
            p += h.idx[i] == j ? t.p(h, i) : 0.0f;
    float v = -c.c1 * p;
    if (h.idx[a.top] == j)
        v -= c.c2;
    // an added grad has the softmaxes already
    ds[j] = (O)(a.beta ? (float)ds[j] + v : v + c.at(h.s[e]));
}

// ---------------------------------------------------------------- rows held in registers

template <class T>
struct chunk_of; // 16 bytes of T
template <>
struct chunk_of<float> {
    static constexpr int N = 4;
    static constexpr uint32_t kLow = 0xff800000u; // -inf
    __device__ static void get(const uint4 &c, float *v)
    {
        v[0] = __uint_as_float(c.x), v[1] = __uint_as_float(c.y), v[2] = __uint_as_float(c.z), v[3] = __uint_as_float(c.w);
    }
    __device__ static uint4 put(const float *v)
    {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <>
struct chunk_of<_Float16> {
    static constexpr int N = 8;
    static constexpr uint32_t kLow = 0xfc00fc00u;
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    __device__ static void get(const uint4 &c, float *v)
    {
        const h8 h = __builtin_bit_cast(h8, c);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = (float)h[i];
    }
    __device__ static uint4 put(const float *v)
    {
        h8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            h[i] = (_Float16)v[i];
        return __builtin_bit_cast(uint4, h);
    }
};
template <>
struct chunk_of<__bf16> {
    static constexpr int N = 8;
    static constexpr uint32_t kLow = 0xff80ff80u;
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 h2 __attribute__((ext_vector_type(2)));
    __device__ static void get(const uint4 &c, float *v)
    {
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ static uint4 put(const float *v)
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{v[2 * i], v[2 * i + 1]}), h2));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// The rows pass by the caches: each is read once and written once (4096 x
// 131072 bf16 in 505 us with ordinary accesses, 487 with these).
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load_once(const uint4 *p)
{
    return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const u32x4 *)p));
}
__device__ __forceinline__ void store_once(uint4 *p, const uint4 &v)
{
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4 *)p);
}

// A row as the threads of a block hold it: whole 16-byte chunks, chunk
// i * NT + tid in register i, and at the ends up to one element per thread that
// no whole chunk covers.
template <class T>
struct span {
    const T *s;
    int chunks;     // whole chunks
    int head, tail; // elements before the first and behind the last
    __device__ span(const T *row, size_t n) : s(row)
    {
        constexpr int V = chunk_of<T>::N;
        const int over = (int)(((uintptr_t)row & 15) / sizeof(T));
        head = over ? V - over : 0;
        head = (size_t)head < n ? head : (int)n;
        chunks = (int)((n - head) / V);
        tail = (int)(n - head - (size_t)chunks * V);
    }
    __device__ int edge(int tid) const { return tid < head ? tid : chunks * chunk_of<T>::N + tid; }
    __device__ float load_edge(int tid) const { return tid < head + tail ? (float)s[edge(tid)] : -INFINITY; }
    // chunk k0 + tid, or -inf past the first `lim`; k0 is uniform, so that the
    // addresses take no vector registers of their own
    __device__ __forceinline__ uint4 load(int k0, int tid, int lim) const
    {
        constexpr uint32_t low = chunk_of<T>::kLow;
        const uint4 *p = (const uint4 *)(s + head) + k0;
        uint4 c = make_uint4(low, low, low, low);
        if (tid < lim - k0)
            c = load_once(p + tid);
        return c;
    }
};

// The stats of what a thread holds, folded in groups as the loads land: one
// maximum and one rescaling per group.  after(i): register i has been read for
// the last time.
template <class T, int PER, class FN>
__device__ __forceinline__ stats fold(const uint4 (&r)[PER], float edge, const wants &w, FN after)
{
    constexpr int V = chunk_of<T>::N, G = PER < 16 / V ? PER : 16 / V;
    stats st = stats_of(edge);
#pragma unroll
    for (int g = 0; g < PER; g += G) {
        float v[G][V], m = st.m;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            chunk_of<T>::get(r[g + i], v[i]);
#pragma unroll
            for (int j = 0; j < V; ++j)
                m = fmaxf(m, v[i][j]);
        }
        const float ref = finite_ref(m);
        auto add = [&](float z, float c) {
            z *= PGM_EXP2((st.m - ref) * c);
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    z += PGM_EXP2((v[i][j] - ref) * c);
            return z;
        };
        if (w.zt)
            st.zt = add(st.zt, w.ct);
        if (w.z1)
            st.z1 = add(st.z1, kLog2e);
        st.m = m;
#pragma unroll
        for (int i = 0; i < G; ++i)
            after(g + i);
        __builtin_amdgcn_sched_barrier(0); // one group's values at a time in registers
    }
    return st;
}

// The grad of what a thread holds, each value rounded once.
template <class T, class O, int PER, int NT, bool ONE, class FN>
__device__ __forceinline__ void store_chunks(const span<T> &sp, const uint4 (&r)[PER], O *ds, const coefs &c, int tid,
                                             FN after)
{
    constexpr int V = chunk_of<T>::N, VO = chunk_of<O>::N, K = V / VO;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        float v[V];
        chunk_of<T>::get(r[i], v);
#pragma unroll
        for (int j = 0; j < V; ++j)
            v[j] = c.at<ONE>(v[j]);
        uint4 *p = (uint4 *)(ds + sp.head) + (size_t)(i * NT) * K;
        if (tid < sp.chunks - i * NT)
#pragma unroll
            for (int j = 0; j < K; ++j)
                store_once(p + tid * K + j, chunk_of<O>::put(v + j * VO));
        after(i);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// One block per row, the row held in registers from its one read to its
// grad's store.  A block takes every gridDim-th row, and each register is
// refilled from the next row as soon as it has been read for the last time, so
// that loads are in flight while the grad (or, for the loss alone, the sums)
// is computed.  The entries of a row are put right one row later, behind that
// row's barrier: a block's accesses pass its CU's L1 in the order of their issue,
// so the row's stores, issued before the barrier by any wave, land before these.
// ONE: the second exponential may be there.  Bound by the stream of the rows in
// and out: 4096 x 131072 bf16 467 us, 4.6 TB/s, 1000 x 50001 f32 91 us, 4.4 TB/s.
template <class T, class O, int NT, int PER, bool GRAD, bool ONE>
__global__ void __launch_bounds__(NT, 4) k_distill_rows(pgk_distill_args a)
{
    static_assert(NT >= PGK_DISTILL_TOP, "a thread per entry");
    __shared__ row_head heads[3]; // this row's, the last one's, and one that a slower wave may still read
    __shared__ stats red[2][NT / 64];
    const int tid = (int)threadIdx.x, nh = head_threads(a);
    const wants w(a);
    size_t row = blockIdx.x;
    span<T> sp((const T *)a.s + row * a.v, a.v);
    entry_loads e;
    if (tid < nh)
        e.begin(a, row, tid);
    uint4 r[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
        r[i] = sp.load(i * NT, tid, sp.chunks);
    float edge = sp.load_edge(tid);
    coefs last;
    last.any = false;
    for (int it = 0;; it = it == 5 ? 0 : it + 1) {
        const size_t next = row + gridDim.x;
        const bool more = next < a.n;
        row_head &h = heads[it % 3];
        const span<T> sn((const T *)a.s + (more ? next : row) * a.v, a.v);
        const int lim = more ? sn.chunks : 0;
        auto refill = [&](int i) { r[i] = sn.load(i * NT, tid, lim); };
        if (tid < nh)
            e.gather(a, sp.s, h, tid);
        stats st = fold<T, PER>(r, edge, w, [&](int i) {
            if constexpr (!GRAD)
                refill(i);
        });
        if (tid < nh) {
            e.finish(a, h, tid);
            if (more)
                e.begin(a, next, tid);
        }
        st = block_join<NT>(st, w, red[it & 1], tid);
        if constexpr (GRAD) {
            const coefs before = last;
            last = coefs(a, h, st, w);
            if (!last.any) { // exp(-inf) is the 0 of such a row
                constexpr uint32_t low = chunk_of<T>::kLow;
                last.m = last.wt = last.w1 = 0.0f;
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    r[i] = make_uint4(low, low, low, low);
                edge = -INFINITY;
            }
            // the grad widens the held values anew: keeping the widened ones
            // from the sums would take twice the registers
#pragma unroll
            for (int i = 0; i < PER; ++i)
                __asm__("" : "+v"(r[i].x), "+v"(r[i].y), "+v"(r[i].z), "+v"(r[i].w));
            O *const ds = (O *)a.ds + row * a.v;
            store_chunks<T, O, PER, NT, ONE>(sp, r, ds, last, tid, refill);
            if (tid < sp.head + sp.tail)
                ds[sp.edge(tid)] = (O)last.at<ONE>(edge);
            if (before.any)
                for (int i = tid; i <= a.top; i += NT)
                    fix_entry<O>(a, heads[(it + 2) % 3], i, (O *)a.ds + (row - gridDim.x) * a.v, before);
        }
        if (a.loss && tid >= NT - 64)
            store_loss(a, row, h, st, w, tid - (NT - 64));
        if (!more) {
            if (GRAD && last.any) {
                __syncthreads();
                for (int i = tid; i <= a.top; i += NT)
                    fix_entry<O>(a, h, i, (O *)a.ds + row * a.v, last);
            }
            return;
        }
        edge = sn.load_edge(tid);
        sp = sn;
        row = next;
    }
}

// ---------------------------------------------------------------- rows split over blocks

// Few long rows, and rows past what a block holds: part blockIdx.x of a row is
// kPartChunks of its chunks (part 0 has its edges too).  One launch leaves every
// part's stats and, once per row, the logits at its entries in memory (the
// grad may take the logits' place in the second); the next joins them and
// writes the loss and the part's grad.
constexpr int kPartThreads = 256, kPartPer = 4, kPartChunks = kPartThreads * kPartPer;

// a row's workspace: the parts' stats, then the logits at its entries and label
__host__ __device__ __forceinline__ size_t part_floats(size_t parts, int top) { return parts * 3 + top + 1; }

template <class T>
__global__ void __launch_bounds__(kPartThreads) k_distill_parts(pgk_distill_args a, float *ws)
{
    __shared__ stats red[kPartThreads / 64];
    const int tid = (int)threadIdx.x, part = (int)blockIdx.x;
    const size_t row = blockIdx.y;
    const span<T> sp((const T *)a.s + row * a.v, a.v);
    const wants w(a);
    float *const mine = ws + row * part_floats(gridDim.x, a.top);
    uint4 r[kPartPer];
#pragma unroll
    for (int i = 0; i < kPartPer; ++i)
        r[i] = sp.load(part * kPartChunks + i * kPartThreads, tid, sp.chunks);
    if (part == 0)
        for (int e = tid; e <= a.top; e += kPartThreads) {
            const float f = e < a.top ? a.idx[row * a.top + e] : a.label ? a.label[row] : -1.0f;
            mine[gridDim.x * 3 + e] = f >= 0.0f && f < (float)a.v ? (float)sp.s[(int)f] : 0.0f;
        }
    stats st = fold<T, kPartPer>(r, part == 0 ? sp.load_edge(tid) : -INFINITY, w, [](int) {});
    st = block_join<kPartThreads>(st, w, red, tid);
    if (tid == 0) {
        mine[part * 3] = st.m;
        mine[part * 3 + 1] = st.zt;
        mine[part * 3 + 2] = st.z1;
    }
}

template <class T, class O, bool GRAD, bool ONE>
__global__ void __launch_bounds__(kPartThreads) k_distill_finish(pgk_distill_args a, const float *ws, int parts)
{
    __shared__ row_head h;
    const int tid = (int)threadIdx.x, lane = tid & 63, part = (int)blockIdx.x;
    const size_t row = blockIdx.y;
    const span<T> sp((const T *)a.s + row * a.v, a.v);
    const wants w(a);
    const float *const mine = ws + row * part_floats(parts, a.top);
    uint4 r[kPartPer];
    float edge = -INFINITY;
    if constexpr (GRAD) {
#pragma unroll
        for (int i = 0; i < kPartPer; ++i)
            r[i] = sp.load(part * kPartChunks + i * kPartThreads, tid, sp.chunks);
        edge = part == 0 ? sp.load_edge(tid) : -INFINITY;
    }
    if (tid < head_threads(a)) {
        entry_loads e;
        e.begin(a, row, tid);
        e.gather(a, (const T *)nullptr, h, tid);
        e.s = tid < a.top ? mine[parts * 3 + tid] : 0.0f;
        e.slabel = mine[parts * 3 + a.top];
        e.finish(a, h, tid);
    }
    stats st = {-INFINITY, 0.0f, 0.0f};
    for (int p = lane; p < parts; p += 64)
        join(st, stats{mine[p * 3], mine[p * 3 + 1], mine[p * 3 + 2]}, w);
    st = wave_join(st, w);
    __syncthreads();
    if (a.loss && part == 0 && tid < 64)
        store_loss(a, row, h, st, w, tid);
    if constexpr (GRAD) {
        coefs c(a, h, st, w);
        if (!c.any) {
            constexpr uint32_t low = chunk_of<T>::kLow;
            c.m = c.wt = c.w1 = 0.0f;
#pragma unroll
            for (int i = 0; i < kPartPer; ++i)
                r[i] = make_uint4(low, low, low, low);
            edge = -INFINITY;
        }
        O *ds = (O *)a.ds + row * a.v;
        span<T> own = sp; // its chunks from the part's first on
        own.s += (size_t)part * kPartChunks * chunk_of<T>::N;
        own.chunks -= part * kPartChunks;
        O *const dsp = ds + (size_t)part * kPartChunks * chunk_of<T>::N;
        store_chunks<T, O, kPartPer, kPartThreads, ONE>(own, r, dsp, c, tid, [](int) {});
        if (part == 0 && tid < sp.head + sp.tail)
            ds[sp.edge(tid)] = (O)c.at<ONE>(edge);
        __syncthreads();
        // the entries in what the block wrote: its chunks, and for part 0 the edges
        const int lo = sp.head + part * kPartChunks * chunk_of<T>::N;
        const int hi = sp.head + min(sp.chunks, (part + 1) * kPartChunks) * chunk_of<T>::N;
        const int end = sp.head + sp.chunks * chunk_of<T>::N;
        for (int i = tid; c.any && i <= a.top; i += kPartThreads) {
            const int j = h.idx[i];
            if ((j >= lo && j < hi) || (part == 0 && (j < sp.head || j >= end)))
                fix_entry<O>(a, h, i, ds, c);
        }
    }
}

// ---------------------------------------------------------------- rows streamed

constexpr int kStreamThreads = 1024;

// Logits and a grad whose 16-byte chunks do not fall together (tensors that start
// inside their storage), a grad that is added to, and more than 65535 rows past what a
// block holds: one block per row, value by value, the row read once for its stats and
// once for the grad.
template <class T, class O>
__global__ void __launch_bounds__(kStreamThreads) k_distill_stream(pgk_distill_args a)
{
    __shared__ row_head h;
    __shared__ stats red[kStreamThreads / 64];
    const int tid = (int)threadIdx.x;
    const size_t row = blockIdx.x;
    const T *s = (const T *)a.s + row * a.v;
    if (tid < head_threads(a)) {
        entry_loads e;
        e.begin(a, row, tid);
        e.gather(a, s, h, tid);
        e.finish(a, h, tid);
    }
    const wants w(a);
    stats st = stats_of(-INFINITY);
    for (size_t i = tid; i < a.v; i += kStreamThreads)
        join(st, stats_of((float)s[i]), w);
    st = block_join<kStreamThreads>(st, w, red, tid);
    if (a.loss && tid < 64)
        store_loss(a, row, h, st, w, tid);
    if (!a.ds)
        return;
    O *ds = (O *)a.ds + row * a.v;
    const coefs c(a, h, st, w);
    if (!c.any && a.beta)
        return;
    for (size_t i = tid; i < a.v; i += kStreamThreads) {
        const float v = c.any ? c.at((float)s[i]) : 0.0f;
        ds[i] = (O)(a.beta ? (float)ds[i] + v : v);
    }
    __syncthreads();
    for (int i = tid; c.any && i <= a.top; i += kStreamThreads)
        fix_entry<O>(a, h, i, ds, c);
}

// ---------------------------------------------------------------- short rows

// Rows of at most 4 G values and G entries, G lanes per row: everything in
// registers, joined by shuffles among the G lanes, the entries handed round.
// Bound by the launch itself (4096 x 10 with four entries: 4.3 us).
template <class T, class O, int G>
__global__ void __launch_bounds__(256) k_distill_short(pgk_distill_args a)
{
    constexpr int PER = 4;
    const int tid = (int)threadIdx.x, lane = tid & (G - 1);
    const size_t row = (size_t)blockIdx.x * (256 / G) + tid / G;
    if (row >= a.n) // whole groups of lanes
        return;
    const int v = (int)a.v;
    const T *s = (const T *)a.s + row * v;
    const wants w(a);
    const float f = lane < a.top ? a.idx[row * a.top + lane] : -1.0f;
    float t = lane < a.top ? ld_any(a.top_dtype, a.t, row * a.top + lane) : 0.0f;
    const float fl = a.label && a.alpha < 1.0f ? a.label[row] : -1.0f;
    float x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = i * G + lane;
        x[i] = j < v ? (float)s[j] : -INFINITY;
    }
    const bool there = f >= 0.0f && f < (float)v, has = fl >= 0.0f && fl < (float)v;
    const int idx = there ? (int)f : -1, lab = has ? (int)fl : -1;
    const float se = there ? (float)s[idx] : 0.0f, sl = has ? (float)s[lab] : 0.0f;
    t = there ? t / a.temperature : -INFINITY;
    auto gmax = [](float q) {
#pragma unroll
        for (int o = G / 2; o; o >>= 1)
            q = fmaxf(q, __shfl_xor(q, o, G));
        return q;
    };
    auto gsum = [](float q) {
#pragma unroll
        for (int o = G / 2; o; o >>= 1)
            q += __shfl_xor(q, o, G);
        return q;
    };
    // the softmaxes
    stats st = stats_of(x[0]);
#pragma unroll
    for (int i = 1; i < PER; ++i)
        join(st, stats_of(x[i]), w);
    const float m = gmax(st.m), d = st.m - finite_ref(m);
    st = {m, w.zt ? gsum(st.zt * PGM_EXP2(d * w.ct)) : 0.0f, w.z1 ? gsum(st.z1 * PGM_EXP2(d * kLog2e)) : 0.0f};
    // the teacher's
    const bool some = gmax(t == -INFINITY ? 0.0f : 1.0f) > 0.0f && a.alpha > 0.0f;
    const float tmax = gmax(t), e = t == -INFINITY ? 0.0f : expf(t - tmax), sum = gsum(e);
    const float p = some ? e / sum : 0.0f;
    float kl = 0.0f;
    if (some && there && !(p == 0.0f))
        kl = p * (t - tmax - logf(sum) - ((se - m) / a.temperature - logf(st.zt)));
    kl = gsum(kl) * a.alpha * a.temperature * a.temperature;
    if (has)
        kl += (1.0f - a.alpha) * (logf(st.sum1(w)) - (sl - m));
    if (a.loss && lane == 0)
        a.loss[row] = some || has ? a.scale * kl : 0.0f;
    if (!a.ds)
        return;
    O *ds = (O *)a.ds + row * v;
    const float up = a.scale * (a.up ? a.up[0] : 1.0f);
    const float c1 = some ? up * a.alpha * a.temperature : 0.0f, c2 = has ? up * (1.0f - a.alpha) : 0.0f;
    const float wt = some ? c1 / st.zt : 0.0f, w1 = has ? c2 / st.sum1(w) : 0.0f;
    float g[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const float dx = x[i] - m;
        g[i] = some ? wt * PGM_EXP2(dx * w.ct) : 0.0f;
        g[i] += has ? w1 * PGM_EXP2(dx * kLog2e) : 0.0f;
        g[i] -= has && i * G + lane == lab ? c2 : 0.0f;
    }
    for (int k = 0; k < a.top; ++k) {
        const int jk = __shfl(idx, k, G);
        const float pk = c1 * __shfl(p, k, G);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            g[i] -= some && i * G + lane == jk ? pk : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = i * G + lane;
        if (j < v)
            ds[j] = (O)(a.beta ? (float)ds[j] + g[i] : g[i]);
    }
}

// ---------------------------------------------------------------- launches

// whether every whole 16-byte chunk of the logits is one (or two) of the grad
template <class T, class O>
bool chunks_match(const pgk_distill_args &a)
{
    return !a.ds || ((uintptr_t)a.ds / sizeof(O) - (uintptr_t)a.s / sizeof(T)) % (16 / sizeof(O)) == 0;
}

template <class T, class O, int NT, int PER>
void launch_rows(const pgk_distill_args &a, int per_cu, hipStream_t st)
{
    const size_t most = (size_t)256 * per_cu;
    const dim3 grid((unsigned)(a.n < most ? a.n : most));
    if (!a.ds)
        hipLaunchKernelGGL((k_distill_rows<T, O, NT, PER, false, false>), grid, dim3(NT), 0, st, a);
    else if (a.label && a.alpha < 1.0f && a.temperature != 1.0f)
        hipLaunchKernelGGL((k_distill_rows<T, O, NT, PER, true, true>), grid, dim3(NT), 0, st, a);
    else
        hipLaunchKernelGGL((k_distill_rows<T, O, NT, PER, true, false>), grid, dim3(NT), 0, st, a);
}

template <class T>
size_t parts_of(const pgk_distill_args &a)
{
    return (a.v / chunk_of<T>::N + kPartChunks - 1) / kPartChunks;
}

// A launch holds under 2^32 threads: fn(args of a run of rows) for runs of at most
// `most`.
template <class FN>
void by_runs(const pgk_distill_args &a, size_t most, FN fn)
{
    auto size = [](int dtype) { return dtype == 0 ? (size_t)4 : (size_t)2; };
    for (size_t r = 0; r < a.n; r += most) {
        pgk_distill_args b = a;
        b.n = a.n - r < most ? a.n - r : most;
        b.s = (const char *)a.s + r * a.v * size(a.dtype);
        b.t = (const char *)a.t + r * a.top * size(a.top_dtype);
        b.idx = a.idx + r * a.top;
        b.label = a.label ? a.label + r : nullptr;
        b.loss = a.loss ? a.loss + r : nullptr;
        b.ds = a.ds ? (char *)a.ds + r * a.v * size(a.ds_dtype) : nullptr;
        fn(b);
    }
}

template <class T, class O, int G>
void launch_short(const pgk_distill_args &all, hipStream_t st)
{
    constexpr size_t R = 256 / G; // rows of a block
    by_runs(all, R << 22, [&](const pgk_distill_args &a) {
        hipLaunchKernelGGL((k_distill_short<T, O, G>), dim3((unsigned)((a.n + R - 1) / R)), dim3(256), 0, st, a);
    });
}

template <class T, class O>
void launch_stream(const pgk_distill_args &all, hipStream_t st)
{
    by_runs(all, (size_t)1 << 21, [&](const pgk_distill_args &a) {
        hipLaunchKernelGGL((k_distill_stream<T, O>), dim3((unsigned)a.n), dim3(kStreamThreads), 0, st, a);
    });
}

// The rows' blocks would leave most of the chip idle, or cannot hold a row.  Up
// to 2^21 chunks of 16 bytes in all the two reads of a split row cost less than
// the idle CUs: 16 rows of 131072 f16 take 9.9 us split and 28.0 whole, 128 26.9
// and 32.6, 200 38.6 and 36.9; 256 rows of 32768 17.7 and 22.2.
template <class T>
bool split(const pgk_distill_args &a)
{
    const size_t chunks = a.v / chunk_of<T>::N;
    return !a.beta && a.n <= 65535 && (chunks > 16384 || (chunks >= 2048 && a.n <= 256 && a.n * chunks <= (size_t)1 << 21));
}

template <class T, class O>
int launch(const pgk_distill_args &a, float *ws, hipStream_t st)
{
    const size_t chunks = a.v / chunk_of<T>::N;
    const bool one = a.label && a.alpha < 1.0f && a.temperature != 1.0f;
    if (a.v <= 64 && a.top <= 16) {
        launch_short<T, O, 16>(a, st);
    } else if (a.v <= 256 && a.top <= 64) {
        launch_short<T, O, 64>(a, st);
    } else if (!chunks_match<T, O>(a) || a.beta) {
        launch_stream<T, O>(a, st);
    } else if (split<T>(a)) {
        const int parts = (int)parts_of<T>(a);
        const dim3 grid((unsigned)parts, (unsigned)a.n);
        hipLaunchKernelGGL(k_distill_parts<T>, grid, dim3(kPartThreads), 0, st, a, ws);
        if (!a.ds)
            hipLaunchKernelGGL((k_distill_finish<T, O, false, false>), dim3(1, grid.y), dim3(kPartThreads), 0, st, a, ws, parts);
        else if (one)
            hipLaunchKernelGGL((k_distill_finish<T, O, true, true>), grid, dim3(kPartThreads), 0, st, a, ws, parts);
        else
            hipLaunchKernelGGL((k_distill_finish<T, O, true, false>), grid, dim3(kPartThreads), 0, st, a, ws, parts);
    } else if (chunks > 16384) {
        launch_stream<T, O>(a, st);
    } else if (chunks > 8192) {
        launch_rows<T, O, 1024, 16>(a, 1, st);
    } else if (chunks > 4096) {
        launch_rows<T, O, 512, 16>(a, 2, st);
    } else if (chunks > 1024) {
        launch_rows<T, O, 256, 16>(a, 4, st);
    } else if (chunks > 256) {
        launch_rows<T, O, 256, 4>(a, 6, st);
    } else {
        launch_rows<T, O, 256, 1>(a, 7, st);
    }
    return (int)hipGetLastError();
}

template <class T>
size_t workspace(const pgk_distill_args &a)
{
    return split<T>(a) ? a.n * part_floats(parts_of<T>(a), a.top) * sizeof(float) : 0;
}

} // namespace

extern "C" size_t pgk_distill_workspace(const pgk_distill_args *a)
{
    return a->dtype == 0 ? workspace<float>(*a) : a->dtype == 1 ? workspace<_Float16>(*a) : workspace<__bf16>(*a);
}

extern "C" int pgk_distill(const pgk_distill_args *a, void *ws, pgk_stream s)
{
    if (!a->n || !a->v)
        return 0;
    if (a->n > 0x7fffffff || a->v > PGK_DISTILL_MAX_V || a->top < 1 || a->top > PGK_DISTILL_TOP ||
        (a->ds && a->ds_dtype != a->dtype && a->ds_dtype != 0) || (!ws && pgk_distill_workspace(a)))
        return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)s;
    float *w = (float *)ws;
    const bool wide = !a->ds || a->ds_dtype == 0;
    if (a->dtype == 0)
        return launch<float, float>(*a, w, st);
    if (a->dtype == 1)
        return wide ? launch<_Float16, float>(*a, w, st) : launch<_Float16, _Float16>(*a, w, st);
    return wide ? launch<__bf16, float>(*a, w, st) : launch<__bf16, __bf16>(*a, w, st);
}
