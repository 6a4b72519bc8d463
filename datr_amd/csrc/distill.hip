// distill.hip -- distillation from a teacher of whom each row's top logits were kept (gfx950).
//
//   p_j  = softmax over the row's valid slots j of teacher[j] / tau         (a slot whose index is outside [0, V) is not valid)
//   q_v  = softmax over all V columns of z[v] / tau
//   loss = tau^2 sum_j p_j (log p_j - log q_{i_j}),      d loss / d z_v = tau (q_v - sum over {j : i_j = v} p_j)
//
// A row without a valid slot, or with nothing but -inf in them, has loss 0 and gradient 0; a NaN in a valid slot is the teacher's answer
// and makes p, the loss and the kept columns' gradient NaN.  Bound by memory: forward reads z once, with the running maximum M
// and the sum S of exp((z - M) / tau) in fp32; backward reads z again and writes dz, with M, S and the teacher's two from the
// forward pass.  M and S are kept apart rather than as one log-sum-exp: q = exp((z - M) / tau) / S keeps its relative error
// for logits of any size.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "datr_hip.h"
#include "elem.h"

namespace {

constexpr int kMaxSlots = 1024;                     // as many as datr_topk_rows_f32 selects
constexpr float kLog2e = 1.44269504088896340736f;

// Who works on a row (us for both passes, fp32):
//   V <= 64       16 lanes, an element each and step: 16 384 rows of 9 take 7.5 (a wave a row: 25), of 64 take 16 (25)
//   V <= 2048,    a wave, 16-byte accesses: 8192 rows of 2048 take 40 (a workgroup a row: 81), 2000 rows of 8000 take 39 (45); 64 rows of
//   or <= 8192    2048 are no different, and longer rows lose (16 000 columns, 8192 rows: 314 against 287)
//   and R >= 1024
//   else          a workgroup, and several where few rows would leave the chip idle: forward parts are joined by a second
//                 launch, backward parts need no join.  4096 rows of 128 000 bf16: 585 us for both passes over 3.15 GB = 5.4 TB/s;
//                 1000 rows of 50 257 fp32: 108 us = 5.6 TB/s (a large copy on this card: 4.7).  dz goes out by streaming stores:
//                 kept in the caches it costs 25 % more at 1000 x 50 257, where z would still be there for backward
constexpr int kGroupThreads = 256;
constexpr int kRowThreads = 512;
constexpr int kTinyV = 64;

bool by_wave(int64_t R, int64_t V) { return V <= 2048 || (V <= 8192 && R >= 1024); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float teacher_at(int dtype, const void *t, int64_t i) {
    if (dtype == DATR_FP32) return ((const float *)t)[i];
    if (dtype == DATR_FP16) return (float)((const _Float16 *)t)[i];
    return (float)((const __bf16 *)t)[i];
}

// the sum s of exp((x - m) / tau), m = -inf: nothing yet
struct Soft {
    float m, s;
};

// whether the teacher's softmax has terms: NaN never raises the maximum, so the sum has to say that one was there
__device__ __forceinline__ bool kept_any(float m, float s) { return m != -INFINITY || s != 0.f; }

__device__ __forceinline__ float shift(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ Soft join(Soft a, Soft b, float c) {
    Soft r;
    r.m = fmaxf(a.m, b.m);
    const float m = shift(r.m);
    r.s = a.s * exp2_fast((a.m - m) * c) + b.s * exp2_fast((b.m - m) * c);
    return r;
}

template <int N>
__device__ __forceinline__ void add(Soft &a, const float (&f)[N], float c) {
    float top = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, f[i]);
    if (top > a.m) {
        a.s *= exp2_fast((a.m - top) * c);
        a.m = top;
    }
    const float m = shift(a.m);
#pragma unroll
    for (int i = 0; i < N; ++i) a.s += exp2_fast((f[i] - m) * c);
}

// joined over the G threads of a row (G <= 64: lanes of one wave; more: the whole workgroup)
template <int G>
__device__ __forceinline__ Soft join_row(Soft a, float c, Soft *lds) {
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) a = join(a, Soft{__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64)}, c);
    if constexpr (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
        __syncthreads();
        a = lds[0];
        for (int w = 1; w < G / 64; ++w) a = join(a, lds[w], c);
    }
    return a;
}

struct Slots {
    const void *teacher;
    const int64_t *index;
    int dtype, k;
};

// thread x of the row's G: the teacher's softmax over the row's slots, then the loss; `live` is false for threads without a row
template <class T, int G>
__device__ __forceinline__ void finish(bool live, int64_t r, int x, const T *row, int64_t V, const Slots &sl, float tau, Soft a, Soft *lds,
                                       float *__restrict__ loss, float4 *__restrict__ stats) {
    const float c = kLog2e / tau;
    Soft t{-INFINITY, 0.f};
    if (live)
        for (int j = x; j < sl.k; j += G) {
            const int64_t i = sl.index[r * sl.k + j];
            const float f[1] = {teacher_at(sl.dtype, sl.teacher, r * sl.k + j)};
            if (i >= 0 && i < V) add<1>(t, f, c);
        }
    t = join_row<G>(t, c, lds);
    float sum = 0.f;
    if (live && kept_any(t.m, t.s)) {
        // tau goes once into the logarithms beside the logits' differences and once into the sum: tau^2 and quotients by tau leave fp32
        // long before the loss does
        const float log_s = tau * logf(a.s), log_t = tau * logf(t.s);
        for (int j = x; j < sl.k; j += G) {
            const int64_t i = sl.index[r * sl.k + j];
            if (i < 0 || i >= V) continue;
            const float d = teacher_at(sl.dtype, sl.teacher, r * sl.k + j) - t.m;
            const float p = exp2_fast(d * c) / t.s;
            if (p != 0.f) sum += p * ((d - log_t) - (((float)row[i] - a.m) - log_s));
        }
    }
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if constexpr (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6].s = sum;
        __syncthreads();
        if (x == 0)
            for (int w = 1; w < G / 64; ++w) sum += lds[w].s;
    }
    if (live && x == 0) {
        loss[r] = tau * sum;
        stats[r] = make_float4(a.m, a.s, t.m, t.s);
    }
}

// G threads a row; parts > 1 (G == TH only): `parts` workgroups a row that leave their sums in `partial`
template <class T, int G, int TH>
__global__ __launch_bounds__(TH) void distill_fwd(const T *__restrict__ z, int64_t ldz, int64_t R, int64_t V, Slots sl, float tau, int parts,
                                                  float2 *__restrict__ partial, float *__restrict__ loss, float4 *__restrict__ stats) {
    constexpr int N = elem::Vec16<T>::N;
    __shared__ Soft lds[TH / 64];
    const float c = kLog2e / tau;
    const int x = threadIdx.x % G;
    const int64_t r = G < TH ? (int64_t)blockIdx.x * (TH / G) + threadIdx.x / G : blockIdx.x / parts;
    const bool live = r < R;
    const T *row = z + (live ? r : 0) * ldz;
    Soft a{-INFINITY, 0.f};
    if constexpr (G < 64) {
        if (live)
            for (int64_t i = x; i < V; i += G) {
                const float f[1] = {(float)row[i]};
                add<1>(a, f, c);
            }
    } else if (live) {
        const int64_t vectors = V / N, per = (vectors + parts - 1) / parts;
        const int64_t part = G < TH ? 0 : blockIdx.x % parts, hi = min((part + 1) * per, vectors);
        int64_t i = part * per + x;
        constexpr int U = 8;                        // 4: 3 % slower over 128 000 columns of bf16
        for (; i + (U - 1) * G < hi; i += U * G) {
            typename elem::Vec16<T>::type v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = elem::load(row + (i + u * G) * N, N);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[N];
                elem::to_float<T>(v[u], f);
                add<N>(a, f, c);
            }
        }
        for (; i < hi; i += G) {
            float f[N];
            elem::to_float<T>(elem::load(row + i * N, N), f);
            add<N>(a, f, c);
        }
        if (part == parts - 1 && vectors * N + x < V) {
            const float f[1] = {(float)row[vectors * N + x]};
            add<1>(a, f, c);
        }
    }
    a = join_row<G>(a, c, lds);
    if (G == TH && parts > 1) {
        if (x == 0) partial[blockIdx.x] = make_float2(a.m, a.s);
        return;
    }
    finish<T, G>(live, r, x, row, V, sl, tau, a, lds, loss, stats);
}

template <class T>
__global__ __launch_bounds__(kGroupThreads) void distill_fwd_join(const T *__restrict__ z, int64_t ldz, int64_t V, Slots sl, float tau, int parts,
                                                                  const float2 *__restrict__ partial, float *__restrict__ loss,
                                                                  float4 *__restrict__ stats) {
    __shared__ Soft lds[kGroupThreads / 64];
    const float c = kLog2e / tau;
    const int64_t r = blockIdx.x;
    Soft a{-INFINITY, 0.f};
    for (int i = threadIdx.x; i < parts; i += kGroupThreads) {
        const float2 p = partial[r * parts + i];
        a = join(a, Soft{p.x, p.y}, c);
    }
    a = join_row<kGroupThreads>(a, c, lds);
    finish<T, kGroupThreads>(true, r, threadIdx.x, z + r * ldz, V, sl, tau, a, lds, loss, stats);
}

// Rows of at most kTinyV: every lane sums its column's slots itself.
template <class T, int G, int TH>
__global__ __launch_bounds__(TH) void distill_bwd_tiny(const T *__restrict__ z, int64_t ldz, int64_t R, int64_t V, Slots sl, float tau,
                                                       const float4 *__restrict__ stats, const float *__restrict__ upstream, T *__restrict__ dz) {
    const float c = kLog2e / tau;
    const int64_t r = (int64_t)blockIdx.x * (TH / G) + threadIdx.x / G;
    if (r >= R) return;
    const float4 st = stats[r];
    const bool any = kept_any(st.z, st.w);
    const float g = upstream[r] * tau, inv = 1.f / st.y, t_inv = 1.f / st.w;
    for (int64_t i = threadIdx.x % G; i < V; i += G) {
        float p = 0.f;
        if (any)
            for (int j = 0; j < sl.k; ++j)
                if (sl.index[r * sl.k + j] == i) p += exp2_fast((teacher_at(sl.dtype, sl.teacher, r * sl.k + j) - st.z) * c) * t_inv;
        dz[r * V + i] = (T)(any ? g * (exp2_fast(((float)z[r * ldz + i] - st.x) * c) * inv - p) : 0.f);
    }
}

// G threads a row, or `parts` workgroups: all columns as if the teacher kept none, then the kept ones again.
template <class T, int G, int TH>
__global__ __launch_bounds__(TH) void distill_bwd(const T *__restrict__ z, int64_t ldz, int64_t R, int64_t V, Slots sl, float tau, int parts,
                                                  bool reverse, const float4 *__restrict__ stats, const float *__restrict__ upstream,
                                                  T *__restrict__ dz) {
    constexpr int N = elem::Vec16<T>::N;
    __shared__ int at[TH / G][kMaxSlots];
    __shared__ float p[TH / G][kMaxSlots];
    const float c = kLog2e / tau;
    const int x = threadIdx.x % G, own = threadIdx.x / G;
    const int64_t r = G < TH ? (int64_t)blockIdx.x * (TH / G) + own : reverse ? R - 1 - blockIdx.x / parts : blockIdx.x / parts;
    const bool live = r < R;
    const T *row = z + (live ? r : 0) * ldz;
    T *out = dz + (live ? r : 0) * V;
    const float4 st = stats[live ? r : 0];
    const bool any = live && kept_any(st.z, st.w);
    const float g = live ? upstream[r] * tau : 0.f, inv = 1.f / st.y;
    const int64_t vectors = V / N, per = (vectors + parts - 1) / parts;
    const int64_t part = G < TH ? 0 : blockIdx.x % parts, lo = part * per, hi = min(lo + per, vectors);
    const int64_t first = lo * N, end = part == parts - 1 ? V : hi * N;
    auto value = [&](float f) { return any ? g * (exp2_fast((f - st.x) * c) * inv) : 0.f; };
    if (live) {
        int64_t i = lo + x;
        constexpr int U = 4;
        for (; i + (U - 1) * G < hi; i += U * G) {
            typename elem::Vec16<T>::type v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = elem::load(row + (i + u * G) * N, N);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[N];
                elem::to_float<T>(v[u], f);
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] = value(f[e]);
                elem::store<true>(out + (i + u * G) * N, f, N);
            }
        }
        for (; i < hi; i += G) {
            float f[N];
            elem::to_float<T>(elem::load(row + i * N, N), f);
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = value(f[e]);
            elem::store<true>(out + i * N, f, N);
        }
        if (part == parts - 1 && vectors * N + x < V) out[vectors * N + x] = (T)value((float)row[vectors * N + x]);
    }
    for (int j = x; j < sl.k; j += G) {
        const int64_t i = any ? sl.index[r * sl.k + j] : -1;
        const bool in = i >= first && i < end;
        at[own][j] = in ? (int)i : -1;
        p[own][j] = in ? exp2_fast((teacher_at(sl.dtype, sl.teacher, r * sl.k + j) - st.z) * c) / st.w : 0.f;
    }
    // the stores above are at the L2 before another wave writes one of their columns again
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int j = x; j < sl.k; j += G) {
        const int i = at[own][j];
        if (i < 0) continue;
        float sum = 0.f;
        bool earliest = true;                       // a column named by several slots is written by the first of them
        for (int o = 0; o < sl.k; ++o) {
            if (at[own][o] != i) continue;
            earliest = earliest && o >= j;
            sum += p[own][o];
        }
        if (earliest) out[i] = (T)(g * (exp2_fast(((float)row[i] - st.x) * c) * inv - sum));
    }
}

// workgroups a row: `target` over all rows, none with fewer than two rounds of its threads
int parts_of(int dtype, int64_t R, int64_t V, int target) {
    if (by_wave(R, V)) return 1;
    const int64_t rounds = V * elem::bytes(dtype) / 16 / (2 * kRowThreads), want = (target + R - 1) / R;
    const int64_t p = rounds < want ? rounds : want;
    return (int)(p < 1 ? 1 : p);
}

template <class T>
int forward(const void *z, int64_t ldz, const Slots &sl, int64_t R, int64_t V, float tau, int parts, float *partial, float *loss, float *stats,
            hipStream_t st) {
    float4 *s4 = (float4 *)stats;
    float2 *p2 = (float2 *)partial;
    const T *zt = (const T *)z;
    auto blocks = [&](int rows) { return dim3((unsigned)((R + rows - 1) / rows)); };
    if (V <= kTinyV) {
        hipLaunchKernelGGL((distill_fwd<T, 16, kGroupThreads>), blocks(kGroupThreads / 16), dim3(kGroupThreads), 0, st, zt, ldz, R, V, sl, tau, 1, p2, loss, s4);
    } else if (by_wave(R, V)) {
        hipLaunchKernelGGL((distill_fwd<T, 64, kGroupThreads>), blocks(kGroupThreads / 64), dim3(kGroupThreads), 0, st, zt, ldz, R, V, sl, tau, 1, p2, loss, s4);
    } else {
        hipLaunchKernelGGL((distill_fwd<T, kRowThreads, kRowThreads>), dim3((unsigned)(R * parts)), dim3(kRowThreads), 0, st, zt, ldz, R, V, sl, tau, parts, p2, loss, s4);
        if (parts > 1) hipLaunchKernelGGL(distill_fwd_join<T>, dim3((unsigned)R), dim3(kGroupThreads), 0, st, zt, ldz, V, sl, tau, parts, p2, loss, s4);
    }
    return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
}

template <class T>
int backward(const void *z, int64_t ldz, const Slots &sl, int64_t R, int64_t V, float tau, int parts, const float *stats, const float *upstream,
             void *dz, hipStream_t st) {
    const float4 *s4 = (const float4 *)stats;
    const T *zt = (const T *)z;
    T *dt = (T *)dz;
    // forward has just read the rows in ascending order: where they pass the 256 MB of the last cache, the last ones are still there
    const bool reverse = R * V * (int64_t)sizeof(T) > 256LL << 20;
    auto blocks = [&](int rows) { return dim3((unsigned)((R + rows - 1) / rows)); };
    if (V <= kTinyV)
        hipLaunchKernelGGL((distill_bwd_tiny<T, 16, kGroupThreads>), blocks(kGroupThreads / 16), dim3(kGroupThreads), 0, st, zt, ldz, R, V, sl, tau, s4, upstream, dt);
    else if (by_wave(R, V))
        hipLaunchKernelGGL((distill_bwd<T, 64, kGroupThreads>), blocks(kGroupThreads / 64), dim3(kGroupThreads), 0, st, zt, ldz, R, V, sl, tau, 1, false, s4, upstream, dt);
    else
        hipLaunchKernelGGL((distill_bwd<T, kRowThreads, kRowThreads>), dim3((unsigned)(R * parts)), dim3(kRowThreads), 0, st, zt, ldz, R, V, sl, tau, parts, reverse, s4, upstream, dt);
    return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
}

constexpr int kTarget = 512;                        // workgroups of 512 threads for forward: two on each of the 256 CUs; twice as many for backward

bool sizes_fit(int64_t R, int64_t V, int64_t k) { return R < (V <= 2048 ? 1LL << 25 : 1LL << 22) && V < (1LL << 31) && k <= kMaxSlots; }

// up to where tau^2 log V is an fp32 number
bool tau_fits(float tau) { return tau >= 1e-30f && tau <= 1e18f; }

}  // namespace

extern "C" {

int64_t datr_topk_distill_workspace_floats(int dtype, int64_t R, int64_t V) {
    if (!elem::known(dtype) || R < 1 || V < 1) return 0;
    const int64_t parts = parts_of(dtype, R, V, kTarget);
    return parts > 1 ? 2 * R * parts : 0;
}

int datr_topk_distill_forward(int dtype, const void *z, int64_t ldz, int teacher_dtype, const void *teacher, const int64_t *index,
                              int64_t R, int64_t V, int64_t k, float tau, float *loss, float *stats, float *workspace,
                              int64_t workspace_floats, void *stream) {
    if (!elem::known(dtype) || !elem::known(teacher_dtype) || R < 0 || V < 1 || k < 0 || ldz < V || !tau_fits(tau)) return DATR_EINVAL;
    if (R == 0) return DATR_OK;
    if (!sizes_fit(R, V, k)) return DATR_EUNSUPPORTED;
    if (!z || !loss || !stats || !elem::aligned16(stats) || (k > 0 && (!teacher || !index))) return DATR_EINVAL;
    const int64_t need = datr_topk_distill_workspace_floats(dtype, R, V);
    if (workspace_floats < need || (need > 0 && !workspace)) return DATR_EINVAL;
    const Slots sl = {teacher, index, teacher_dtype, (int)k};
    const int parts = parts_of(dtype, R, V, kTarget);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case DATR_FP32: return forward<float>(z, ldz, sl, R, V, tau, parts, workspace, loss, stats, st);
        case DATR_FP16: return forward<_Float16>(z, ldz, sl, R, V, tau, parts, workspace, loss, stats, st);
        default: return forward<__bf16>(z, ldz, sl, R, V, tau, parts, workspace, loss, stats, st);
    }
}

int datr_topk_distill_backward(int dtype, const void *z, int64_t ldz, int teacher_dtype, const void *teacher, const int64_t *index,
                               int64_t R, int64_t V, int64_t k, float tau, const float *stats, const float *upstream, void *dz,
                               void *stream) {
    if (!elem::known(dtype) || !elem::known(teacher_dtype) || R < 0 || V < 1 || k < 0 || ldz < V || !tau_fits(tau)) return DATR_EINVAL;
    if (R == 0) return DATR_OK;
    if (!sizes_fit(R, V, k)) return DATR_EUNSUPPORTED;
    if (!z || !stats || !elem::aligned16(stats) || !upstream || !dz || (k > 0 && (!teacher || !index))) return DATR_EINVAL;
    const Slots sl = {teacher, index, teacher_dtype, (int)k};
    const int parts = parts_of(dtype, R, V, 2 * kTarget);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case DATR_FP32: return backward<float>(z, ldz, sl, R, V, tau, parts, stats, upstream, dz, st);
        case DATR_FP16: return backward<_Float16>(z, ldz, sl, R, V, tau, parts, stats, upstream, dz, st);
        default: return backward<__bf16>(z, ldz, sl, R, V, tau, parts, stats, upstream, dz, st);
    }
}

}  // extern "C"
