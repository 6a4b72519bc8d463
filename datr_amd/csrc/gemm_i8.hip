// gemm_i8.hip -- a linear layer in 8-bit integers with one scale for each token and one for each output channel (gfx950).
//
//   s_m    = max_k |x[m, k]| / 127,       q[m, k] = x[m, k] / s_m rounded to nearest, ties to even
//   y[m,n] = relu?( sum_k q[m, k] W[n, k] * s_m * w_n + bias[n] )          W int8 [N, K] with scales w_n, sums in 32-bit integers
//
// The integer sum is exact (|sum| <= 127 * 128 * K < 2^31 for K <= 131072), so y does not depend on tiles or on the order of sums.
//
// Two launches (one for a single token): the rows of x are quantised (bound by memory: x once, q once; 88 892 x 2048 fp32: 147 us on
// average, 136 at best = 6.2 and 6.7 TB/s), then multiplied.  The product's W is the matrix instruction's first operand: a lane then
// holds four consecutive channels of one token, which leave as one 8- or 16-byte piece.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "datr_hip.h"
#include "elem.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
typedef __attribute__((address_space(3))) float lds_float;
typedef __attribute__((address_space(3))) void lds_void;

constexpr int64_t kMaxK = 131072;
constexpr int kRowBytes = 128;                                   // of K in a step of the tile kernel
constexpr int kFewBytes = 256;                                   // of the kernel for few tokens; q's rows are whole numbers of these,
                                                                 // with zeros behind column K

// ---- quantisation ---------------------------------------------------------------------------------------------------------
// Adding 1.5 * 2^23 to x * (127 / top) in one fused operation leaves the rounded product in the sum's low bits.  The product is off by
// less than 127 * 2^-24 < 1e-5 (127 / top is rounded), so away from a border m + 1/2 the integer is the exact quotient's, and next
// to one the product's integer part is m.  There (m + 1/2) top is compared with 127 |x| in fp64, where both are exact (33 and 31
// bits).  Rows whose largest magnitude is so small that 127 / top leaves fp32 are lifted by a power of two first.
constexpr float kNearBorder = 0.4999f, kRounder = 12582912.f;
constexpr float kSmallTop = 0x1p-90f, kLift = 0x1p100f;

// q of N elements, four to a word; top >= 2^-90, inv = 127 / top
template <int N>
__device__ __forceinline__ void quantize(const float (&f)[N], float top, float inv, unsigned (&out)[N / 4]) {
    unsigned q[N];
    float away = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float r = fmaf(f[i], inv, kRounder);
        away = fmaxf(away, fabsf(fmaf(f[i], inv, kRounder - r)));
        q[i] = __float_as_uint(r);
    }
    if (away > kNearBorder) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float n = __uint_as_float(q[i]) - kRounder;
            if (fabsf(fmaf(f[i], inv, -n)) <= kNearBorder) continue;
            const int m = (int)fabsf(f[i] * inv);
            const double u = 127.0 * fabs((double)f[i]), border = ((double)m + 0.5) * (double)top;
            const int exact = u > border || (u == border && (m & 1)) ? m + 1 : m;
            q[i] = (unsigned)(f[i] < 0.f ? -exact : exact);
        }
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i)                              // the low bytes side by side
        out[i] = __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0C0C0400u) | __builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x04000C0Cu);
}

// What a row's largest magnitude says (as an integer: so magnitudes compare, NaN above infinity).  A row with an infinity or a NaN
// has no scale: it takes NaN, and with it every output of the row.
struct RowScale {
    float top, lift, lifted, inv;
    bool usable, finite;
    __device__ __forceinline__ explicit RowScale(unsigned most)
        : top(__uint_as_float(most)), lift(top < kSmallTop ? kLift : 1.f), lifted(top * lift), inv(127.f / lifted),
          usable(most > 0 && most < 0x7F800000u), finite(most < 0x7F800000u) {}
    __device__ __forceinline__ float scale() const { return finite ? top / 127.f : NAN; }
    template <int N>
    __device__ __forceinline__ void row(float (&f)[N], unsigned (&out)[N / 4]) const {
        if (lift != 1.f) {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] *= lift;
        }
        quantize<N>(f, lifted, inv, out);
    }
};

// G threads a row (G = 64: four rows a workgroup), which keep R 16-byte vectors each: one pass over x.  R == 0: longer rows, read
// twice.  kStream: x is past what the last cache holds; passed by it, it leaves q there for the product (88 892 x 2048 fp32: 235 ->
// 219 us for the layer; an x that fits is 5 % slower so).
constexpr int kQuantThreads = 256;

template <class T, int G, int R, bool kStream>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows(const T *__restrict__ x, int64_t rows, int64_t K, int64_t ldx,
                                                               int8_t *__restrict__ q, int64_t ldq, float *__restrict__ scale) {
    constexpr int N = elem::Vec16<T>::N;
    __shared__ unsigned wave_top[kQuantThreads / 64];
    const int64_t r = (int64_t)blockIdx.x * (kQuantThreads / G) + threadIdx.x / G;
    const int t = threadIdx.x % G;
    const bool live = r < rows;
    const T *row = x + (live ? r : 0) * ldx;
    typename elem::Vec16<T>::type v[R > 0 ? R : 1];
    unsigned top = 0;                                            // magnitudes compare as integers, NaN above infinity
    auto look = [&](const typename elem::Vec16<T>::type &a) {
        float f[N];
        elem::to_float<T>(a, f);
#pragma unroll
        for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t c = ((int64_t)i * G + t) * N;
            v[i] = c < K && live ? elem::load<kStream>(row + c, K - c) : typename elem::Vec16<T>::type{};
        }
#pragma unroll
        for (int i = 0; i < R; ++i) look(v[i]);
    } else {
        for (int64_t c = t * N; c < K; c += G * N) look(elem::load(row + c, K - c));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    if constexpr (G > 64) {
        if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
        __syncthreads();
        for (int w = 0; w < G / 64; ++w) top = max(top, wave_top[w]);
    }
    if (!live) return;
    const RowScale rs(top);
    auto put = [&](int64_t c, const typename elem::Vec16<T>::type &a) {
        float f[N];
        unsigned w[N / 4] = {};
        elem::to_float<T>(a, f);
        if (rs.usable) rs.template row<N>(f, w);
        if constexpr (N == 8) *reinterpret_cast<uint2 *>(q + r * ldq + c) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<unsigned *>(q + r * ldq + c) = w[0];
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t c = ((int64_t)i * G + t) * N;
            if (c < ldq) put(c, v[i]);
        }
    } else {
        for (int64_t c = t * N; c < ldq; c += G * N) put(c, c < K ? elem::load(row + c, K - c) : typename elem::Vec16<T>::type{});
    }
    if (t == 0) scale[r] = rs.scale();
}

template <class T>
int quantize_launch(const void *x, int64_t rows, int64_t K, int64_t ldx, int8_t *q, int64_t ldq, float *scale, hipStream_t st) {
    const int64_t vectors = ldq / elem::Vec16<T>::N;
    const T *xt = (const T *)x;
    const dim3 block(kQuantThreads), by4((unsigned)((rows + 3) / 4)), by1((unsigned)rows);
    const bool stream = rows * K * (int64_t)sizeof(T) > 256LL << 20;
    if (vectors <= 64 * 2) hipLaunchKernelGGL((quantize_rows<T, 64, 2, false>), by4, block, 0, st, xt, rows, K, ldx, q, ldq, scale);
    else if (vectors <= 256 * 2 && stream) hipLaunchKernelGGL((quantize_rows<T, 256, 2, true>), by1, block, 0, st, xt, rows, K, ldx, q, ldq, scale);
    else if (vectors <= 256 * 2) hipLaunchKernelGGL((quantize_rows<T, 256, 2, false>), by1, block, 0, st, xt, rows, K, ldx, q, ldq, scale);
    else if (vectors <= 256 * 8 && stream) hipLaunchKernelGGL((quantize_rows<T, 256, 8, true>), by1, block, 0, st, xt, rows, K, ldx, q, ldq, scale);
    else if (vectors <= 256 * 8) hipLaunchKernelGGL((quantize_rows<T, 256, 8, false>), by1, block, 0, st, xt, rows, K, ldx, q, ldq, scale);
    else hipLaunchKernelGGL((quantize_rows<T, 256, 0, false>), by1, block, 0, st, xt, rows, K, ldx, q, ldq, scale);
    return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
}

int quantize_any(int dtype, const void *x, int64_t rows, int64_t K, int64_t ldx, int8_t *q, int64_t ldq, float *scale, hipStream_t st) {
    switch (dtype) {
        case DATR_FP32: return quantize_launch<float>(x, rows, K, ldx, q, ldq, scale, st);
        case DATR_FP16: return quantize_launch<_Float16>(x, rows, K, ldx, q, ldq, scale, st);
        default: return quantize_launch<__bf16>(x, rows, K, ldx, q, ldq, scale, st);
    }
}

// ---- product --------------------------------------------------------------------------------------------------------------
struct Product {
    const int8_t *a;                                             // q [M, lda]
    const float *a_scale;
    const int8_t *w;
    const float *w_scale, *bias;
    void *y;
    int64_t M, N, K, lda, ldw, ldy;
    int relu;
};

// The sum meets the token's scale first and the channel's in one fused operation with the bias: the two scales' product by itself may
// leave fp32 where the result does not.  |sum| < 2^31, so a token scale up to 2^96 keeps the first product finite; a larger one
// (at most 2^121.02) gives 2^25 to the channel's scale, which stays finite for a sum of 0's sake.
constexpr float kLargeScale = 0x1p96f, kGive = 0x1p25f, kFinite = 0x1.fffffep127f;

__device__ __forceinline__ float token_part(float s) { return s > kLargeScale ? s * (1.f / kGive) : s; }
__device__ __forceinline__ float channel_part_large(float ws) {
    return fabsf(ws) <= kFinite ? fminf(fmaxf(ws * kGive, -kFinite), kFinite) : ws;
}

// s and ws: the parts above
__device__ __forceinline__ float finish(const Product &p, int acc, float s, float ws, float b) {
    const float v = (float)acc * s * ws + b;
    return p.relu && v < 0.f ? 0.f : v;                          // a NaN stays one
}

// one result of a row whose scale is s
__device__ __forceinline__ float finish_one(const Product &p, int acc, float s, int64_t n) {
    const float ws = p.w_scale[n];
    return finish(p, acc, token_part(s), s > kLargeScale ? channel_part_large(ws) : ws, p.bias ? p.bias[n] : 0.f);
}

// rows from row0 on, as a buffer whose range check gives zeros behind the last row's K columns (rounded up to a word)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const int8_t *base, int64_t row0, int64_t rows, int64_t most, int64_t ld, int64_t K) {
    const int64_t n = min(rows - row0, most);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(base + row0 * ld), 0, (int)((n - 1) * ld + ((K + 3) & ~3LL)), 0x00020000);
}

// Tile kernel: WN x WM waves, each with TN x TM tiles of 32 channels x 32 tokens (v_mfma_i32_32x32x32_i8), K in steps of 128
// bytes.  Both operands go from memory to LDS without registers (buffer_load ... lds), a ring of S stages: step k + S - 1 is
// requested right behind the barrier that publishes step k.  A row of a step is one 128-byte line of eight 16-byte pieces, piece c of row r at
// place c ^ ((r >> 1) & 7) -- by permuting the source addresses, the LDS side being lane-linear -- so that a fragment's
// ds_read_b128 meets every bank once.
//
// 8192 x 4096 x 14336, launches of a trace: 534 us on average, 469 at best = 1.8 and 2.05 P op/s; bound by power: the matrix pipes are
// busy 52 % of the time at 1.73 GHz, where a library product of the same size (1.94 P op/s) has them busy 66 % at 1.44 GHz.  Steps
// of 64 bytes in four stages take 4 % longer.
template <class T, int TN, int TM, int WN, int WM, int S>
__global__ __launch_bounds__(64 * WN * WM) void gemm_tile(Product p, int tiles_n, int tiles_m) {
    constexpr int BN = 32 * TN * WN, BM = 32 * TM * WM, WAVES = WN * WM, STAGE = (BN + BM) * kRowBytes;
    constexpr int LOADS_W = BN / 8 / WAVES, LOADS_A = BM / 8 / WAVES;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, half = lane >> 5;
    // workgroup b runs on XCD b % 8: each XCD takes consecutive tiles, in blocks of up to 8 token tiles, channel tile outermost
    const int b = blockIdx.x, total = tiles_n * tiles_m, per = total / 8, rest = total % 8, xcd = b % 8;
    const int t = xcd * per + min(xcd, rest) + b / 8;
    const int block = t / (8 * tiles_n), high = min(8, tiles_m - block * 8), in = t - block * 8 * tiles_n;
    const int64_t m0 = (int64_t)(block * 8 + in % high) * BM, n0 = (int64_t)(in / high) * BN;

    const __amdgpu_buffer_rsrc_t wr = rows_of(p.w, n0, p.N, BN, p.ldw, p.K);
    const __amdgpu_buffer_rsrc_t ar = rows_of(p.a, m0, p.M, BM, p.lda, p.lda);
    unsigned from_w[LOADS_W], from_a[LOADS_A];
    auto source = [&](int q, int64_t ld) {                       // of this lane's piece of the 8 rows that instruction q loads
        const int row = q * 8 + (lane >> 3);
        return (unsigned)(row * ld + (((lane & 7) ^ ((row >> 1) & 7)) << 4));
    };
#pragma unroll
    for (int u = 0; u < LOADS_W; ++u) from_w[u] = source(wave * LOADS_W + u, p.ldw);
#pragma unroll
    for (int u = 0; u < LOADS_A; ++u) from_a[u] = source(wave * LOADS_A + u, p.lda);
    const int steps = (int)((p.K + kRowBytes - 1) / kRowBytes);
    auto issue = [&](int step, int stage) {                      // steps behind the last load nothing but keep the count
        const unsigned k = step < steps ? (unsigned)step * kRowBytes : 1u << 31, base = (unsigned)stage * STAGE;
#pragma unroll
        for (int u = 0; u < LOADS_W; ++u)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, reinterpret_cast<lds_void *>((uintptr_t)(base + (wave * LOADS_W + u) * 1024u)), 16,
                                                     (int)(from_w[u] + k), 0, 0, 0);
#pragma unroll
        for (int u = 0; u < LOADS_A; ++u)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ar, reinterpret_cast<lds_void *>((uintptr_t)(base + BN * kRowBytes + (wave * LOADS_A + u) * 1024u)), 16,
                                                     (int)(from_a[u] + k), 0, 0, 0);
    };

    const int wn = wave % WN, wm = wave / WN;
    // the channels' scales, biases and scales for tokens of a large one wait behind the operands' LDS, the tokens' scales in registers
    constexpr unsigned SCALES = S * STAGE;
    for (int c = threadIdx.x; c < BN; c += 64 * WAVES) {
        const bool in = n0 + c < p.N;
        const float ws = in ? p.w_scale[n0 + c] : 0.f;
        *reinterpret_cast<lds_float *>((uintptr_t)(SCALES + c * 4u)) = ws;
        *reinterpret_cast<lds_float *>((uintptr_t)(SCALES + (BN + c) * 4u)) = in && p.bias ? p.bias[n0 + c] : 0.f;
        *reinterpret_cast<lds_float *>((uintptr_t)(SCALES + (2 * BN + c) * 4u)) = channel_part_large(ws);
    }
    float token_scale[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) token_scale[j] = p.a_scale[min(m0 + (wm * TM + j) * 32 + l31, p.M - 1)];
#pragma unroll
    for (int k = 0; k < S - 1; ++k) issue(k, k);
    i32x16 acc[TN][TM] = {};
    const unsigned swizzle = (l31 >> 1) & 7;
    const unsigned row_w = (wn * TN * 32 + l31) * kRowBytes, row_a = BN * kRowBytes + (wm * TM * 32 + l31) * kRowBytes;
    int stage = 0;
    for (int k = 0; k < steps; ++k) {
        // this wave's share of step k has landed (only the S - 2 steps behind it may be outstanding), everybody's behind the barrier;
        // the readers of the stage that is requested next are past it too
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * (LOADS_W + LOADS_A)) : "memory");
        issue(k + S - 1, stage == 0 ? S - 1 : stage - 1);
        const unsigned base = (unsigned)stage * STAGE;
        stage = stage == S - 1 ? 0 : stage + 1;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const unsigned place = ((2 * s + half) ^ swizzle) << 4;
            i32x4 fw[TN], fa[TM];
#pragma unroll
            for (int i = 0; i < TN; ++i) fw[i] = *reinterpret_cast<const lds_i32x4 *>((uintptr_t)(base + row_w + i * 32 * kRowBytes + place));
#pragma unroll
            for (int j = 0; j < TM; ++j) fa[j] = *reinterpret_cast<const lds_i32x4 *>((uintptr_t)(base + row_a + j * 32 * kRowBytes + place));
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[i], fa[j], acc[i][j], 0, 0, 0);
        }
    }

    // y goes through LDS, 32 tokens of a wave at a time and no barrier between waves: a lane writes four channels of its token, then
    // reads 16 bytes of a row, so that a row's 32 TN channels leave side by side.  16-byte piece c of row r lies at c ^ (r % pieces).
    constexpr int PIECES = TN * 32 * (int)sizeof(T) / 16, ROW = PIECES * 16, N16 = 16 / (int)sizeof(T);
    static_assert(32 * ROW * WAVES <= S * STAGE, "the staging rows fit the operands' LDS");
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const unsigned mine = (unsigned)wave * 32 * ROW;
    const int64_t n_wave = n0 + wn * TN * 32;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int64_t m_first = m0 + (wm * TM + j) * 32;
        const float s = token_part(token_scale[j]);
        const unsigned scales = SCALES + (token_scale[j] > kLargeScale ? 2 * BN * 4u : 0u);
#pragma unroll
        for (int i = 0; i < TN; ++i) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = i * 32 + 8 * g + 4 * half;
                const f32x4 ws = *reinterpret_cast<const lds_f32x4 *>((uintptr_t)(scales + (wn * TN * 32 + c) * 4u));
                const f32x4 bias = *reinterpret_cast<const lds_f32x4 *>((uintptr_t)(SCALES + (BN + wn * TN * 32 + c) * 4u));
                T out[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = (T)finish(p, acc[i][j][4 * g + e], s, ws[e], bias[e]);
                const unsigned bytes = c * (unsigned)sizeof(T), to = mine + l31 * ROW + (((bytes >> 4) ^ (l31 % PIECES)) << 4) + (bytes & 15);
                typedef T T4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) T4 lds_T4;
                *reinterpret_cast<lds_T4 *>((uintptr_t)to) = T4{out[0], out[1], out[2], out[3]};
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        constexpr int AT_ONCE = 64 / PIECES;
        const int piece = lane % PIECES;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
            const int r = r0 + lane / PIECES;
            const i32x4 v = *reinterpret_cast<const lds_i32x4 *>((uintptr_t)(mine + r * ROW + ((piece ^ (r % PIECES)) << 4)));
            const int64_t n = n_wave + piece * N16, m = m_first + r;
            if (m >= p.M || n >= p.N) continue;
            T *to = (T *)p.y + m * p.ldy + n;
            typedef typename elem::Vec16<T>::type V;
            const V o = __builtin_bit_cast(V, v);
            if (p.N - n >= N16) {
                *reinterpret_cast<typename elem::Vec16<T>::loose *>(to) = o;
            } else {
#pragma unroll
                for (int e = 0; e < N16 - 1; ++e)
                    if (n + e < p.N) to[e] = o[e];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// Few tokens: bound by reading W once.  A workgroup takes 16 TN channels and 16 TM tokens, K in steps of 256 bytes through a ring
// of S stages in LDS (whole lines of both operands, S - 1 steps in flight, no registers); of each step its four waves take 64 bytes
// each (v_mfma_i32_16x16x64_i8), and their integer sums meet in LDS.  Piece c of row r lies at place c ^ r.  Straight from memory
// into registers -- 16 rows' half lines an instruction -- 45 MB of W took 20.9 us at 32 tokens, this way 13.6 on average and 12.1 at best.
constexpr int kFewWaves = 4;

template <class T, int TN, int TM, int S>
__global__ __launch_bounds__(64 * kFewWaves) void gemm_few(Product p) {
    constexpr int BLOCK = 16 * kFewBytes, STAGE = (TN + TM) * BLOCK, LOADS = TN + TM;     // LOADS of a wave and step
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n0 = (int64_t)blockIdx.x * 16 * TN, m0 = (int64_t)blockIdx.y * 16 * TM;
    const __amdgpu_buffer_rsrc_t wr = rows_of(p.w, n0, p.N, 16 * TN, p.ldw, p.K);
    const __amdgpu_buffer_rsrc_t ar = rows_of(p.a, m0, p.M, 16 * TM, p.lda, p.lda);
    const int steps = (int)(p.lda / kFewBytes);
    // the wave loads four of a block's 16 rows: this lane's piece of them, and the blocks' distances
    const int row = wave * 4 + (lane >> 4);
    const unsigned piece = ((lane & 15) ^ row) << 4;
    const unsigned from_w = (unsigned)(row * p.ldw) + piece, from_a = (unsigned)(row * p.lda) + piece;
    auto issue = [&](int step, int stage) {                      // steps behind the last load nothing but keep the count
        const unsigned k = step < steps ? (unsigned)step * kFewBytes : 1u << 31, to = (unsigned)stage * STAGE + wave * 1024u;
#pragma unroll
        for (int i = 0; i < TN; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, reinterpret_cast<lds_void *>((uintptr_t)(to + i * BLOCK)), 16,
                                                     (int)(from_w + i * 16 * (unsigned)p.ldw + k), 0, 0, 0);
#pragma unroll
        for (int j = 0; j < TM; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ar, reinterpret_cast<lds_void *>((uintptr_t)(to + (TN + j) * BLOCK)), 16,
                                                     (int)(from_a + j * 16 * (unsigned)p.lda + k), 0, 0, 0);
    };
#pragma unroll
    for (int k = 0; k < S - 1; ++k) issue(k, k);
    i32x4 acc[TN][TM] = {};
    const unsigned place = (lane & 15) * kFewBytes + (((wave * 4 + (lane >> 4)) ^ (lane & 15)) << 4);
    int stage = 0;
    for (int k = 0; k < steps; ++k) {
        // step k has landed: of this wave's loads only those of the S - 2 steps behind it may be outstanding
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * LOADS) : "memory");
        issue(k + S - 1, stage == 0 ? S - 1 : stage - 1);
        const unsigned base = (unsigned)stage * STAGE + place;
        i32x4 fw[TN], fa[TM];
#pragma unroll
        for (int i = 0; i < TN; ++i) fw[i] = *reinterpret_cast<const lds_i32x4 *>((uintptr_t)(base + i * BLOCK));
#pragma unroll
        for (int j = 0; j < TM; ++j) fa[j] = *reinterpret_cast<const lds_i32x4 *>((uintptr_t)(base + (TN + j) * BLOCK));
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fa[j], acc[i][j], 0, 0, 0);
        stage = stage == S - 1 ? 0 : stage + 1;
    }
    static_assert(kFewWaves * TN * TM * 1024 <= S * STAGE, "the partial sums fit the ring");
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
            *reinterpret_cast<lds_i32x4 *>((uintptr_t)(((i * TM + j) * kFewWaves + wave) * 1024u + lane * 16u)) = acc[i][j];
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    for (int t = wave; t < TN * TM; t += kFewWaves) {
        i32x4 sum = {};
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) sum += *reinterpret_cast<const lds_i32x4 *>((uintptr_t)((t * kFewWaves + w) * 1024u + lane * 16u));
        const int64_t m = m0 + t % TM * 16 + (lane & 15), n = n0 + t / TM * 16 + (lane >> 4) * 4;
        if (m >= p.M) continue;
        const float s = p.a_scale[m];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < p.N) ((T *)p.y)[m * p.ldy + n + e] = (T)finish_one(p, sum[e], s, n + e);
    }
}

// One token: the same product in one launch.  Every workgroup quantises the token for itself, up to 64 elements a thread, while its
// first steps of W are on their way.  (1 x 4096 x 4096: 7.2 us instead of 9.7.)
constexpr int kOneElements = 16384;
constexpr int kOneStages = 8;

template <class X, class T>
__global__ __launch_bounds__(64 * kFewWaves) void gemm_one(Product p, const X *__restrict__ x) {
    constexpr int S = kOneStages, N = elem::Vec16<X>::N, R = kOneElements / (64 * kFewWaves * N), STAGE = 16 * kFewBytes;
    constexpr unsigned ROW = S * STAGE, TOPS = ROW + kOneElements;          // q, then the waves' largest magnitudes
    typedef __attribute__((address_space(3))) unsigned lds_unsigned;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, width = (int)p.lda;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    typename elem::Vec16<X>::type v[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int c = (i * 64 * kFewWaves + tid) * N;
        v[i] = c < p.K ? elem::load(x + c, p.K - c) : typename elem::Vec16<X>::type{};
    }
    const __amdgpu_buffer_rsrc_t wr = rows_of(p.w, n0, p.N, 16, p.ldw, p.K);
    const int steps = width / kFewBytes, row = wave * 4 + (lane >> 4);
    const unsigned from_w = (unsigned)(row * p.ldw) + (((lane & 15) ^ row) << 4);
    auto issue = [&](int step, int stage) {
        const unsigned k = step < steps ? (unsigned)step * kFewBytes : 1u << 31;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, reinterpret_cast<lds_void *>((uintptr_t)((unsigned)stage * STAGE + wave * 1024u)), 16,
                                                 (int)(from_w + k), 0, 0, 0);
    };
#pragma unroll
    for (int k = 0; k < S - 1; ++k) issue(k, k);
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float f[N];
        elem::to_float<X>(v[i], f);
#pragma unroll
        for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    *reinterpret_cast<lds_unsigned *>((uintptr_t)(TOPS + wave * 4u)) = top;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) top = max(top, *reinterpret_cast<const lds_unsigned *>((uintptr_t)(TOPS + w * 4u)));
    const RowScale rs(top);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int c = (i * 64 * kFewWaves + tid) * N;
        if (c < width) {
            float f[N];
            unsigned w[N / 4] = {};
            elem::to_float<X>(v[i], f);
            if (rs.usable) rs.template row<N>(f, w);
#pragma unroll
            for (int e = 0; e < N / 4; ++e) *reinterpret_cast<lds_unsigned *>((uintptr_t)(ROW + c + 4 * e)) = w[e];
        }
    }
    i32x4 acc = {};
    const int piece = wave * 4 + (lane >> 4);
    const unsigned place = (lane & 15) * kFewBytes + ((piece ^ (lane & 15)) << 4), place_a = ROW + (piece << 4);
    int stage = 0;
    for (int k = 0; k < steps; ++k) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(S - 2) : "memory");
        issue(k + S - 1, stage == 0 ? S - 1 : stage - 1);
        const i32x4 fw = *reinterpret_cast<const lds_i32x4 *>((uintptr_t)((unsigned)stage * STAGE + place));
        const i32x4 fa = *reinterpret_cast<const lds_i32x4 *>((uintptr_t)(place_a + k * (unsigned)kFewBytes));
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw, fa, acc, 0, 0, 0);          // 16 equal columns: the token
        stage = stage == S - 1 ? 0 : stage + 1;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    *reinterpret_cast<lds_i32x4 *>((uintptr_t)(wave * 1024u + lane * 16u)) = acc;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (wave || (lane & 15)) return;
    i32x4 sum = {};
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) sum += *reinterpret_cast<const lds_i32x4 *>((uintptr_t)(w * 1024u + lane * 16u));
    const int64_t n = n0 + (lane >> 4) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < p.N) ((T *)p.y)[n + e] = (T)finish_one(p, sum[e], rs.scale(), n + e);
}

template <class T, int TN, int TM, int WN, int WM, int S>
int launch_tile(const Product &p, hipStream_t st) {
    constexpr int BN = 32 * TN * WN, BM = 32 * TM * WM;
    const int64_t tn = (p.N + BN - 1) / BN, tm = (p.M + BM - 1) / BM;
    if (tn * tm * 64 * WN * WM >= (1LL << 32)) return DATR_EUNSUPPORTED;
    constexpr int lds = S * (BN + BM) * kRowBytes + BN * 12;
    auto kernel = gemm_tile<T, TN, TM, WN, WM, S>;
    if (lds > 65536 && hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return DATR_ELAUNCH;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tn * tm)), dim3(64 * WN * WM), lds, st, p, (int)tn, (int)tm);
    return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
}

template <class T, int TN, int TM, int S>
int launch_few(const Product &p, hipStream_t st) {
    constexpr int lds = S * (TN + TM) * 16 * kFewBytes;
    auto kernel = gemm_few<T, TN, TM, S>;
    if (lds > 65536 && hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return DATR_ELAUNCH;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((p.N + 16 * TN - 1) / (16 * TN)), (unsigned)((p.M + 16 * TM - 1) / (16 * TM))), dim3(64 * kFewWaves), lds,
                       st, p);
    return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
}

template <class X, class T>
int launch_one(const Product &p, const void *x, hipStream_t st) {
    constexpr int lds = kOneStages * 16 * kFewBytes + kOneElements + 4 * kFewWaves;
    static_assert(lds <= 65536, "the default limit");
    hipLaunchKernelGGL((gemm_one<X, T>), dim3((unsigned)((p.N + 15) / 16)), dim3(64 * kFewWaves), lds, st, p, (const X *)x);
    return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
}

template <class T>
int launch_one(const Product &p, int dtype, const void *x, hipStream_t st) {
    switch (dtype) {
        case DATR_FP32: return launch_one<float, T>(p, x, st);
        case DATR_FP16: return launch_one<_Float16, T>(p, x, st);
        default: return launch_one<__bf16, T>(p, x, st);
    }
}

template <class T>
int launch(const Product &p, hipStream_t st) {
    // Few tokens: 16 channels a workgroup, 32 where those still give every CU one (32 tokens, K = 4096, us with the quantisation:
    // 21.2 -> 19.1 for 11 008 channels, 11.7 -> 12.1 for 4096).  From 33 tokens on the tiles below are as good where channels are many
    // (48 tokens: 19.6 -> 16.2 for 11 008 channels, 14.3 -> 15.2 for 7000, 11.6 -> 14.6 for 4096).
    const bool wide = p.N >= 8192;
    if (p.M <= 16) return wide ? launch_few<T, 2, 1, 5>(p, st) : launch_few<T, 1, 1, 8>(p, st);
    if (p.M <= 32) return wide ? launch_few<T, 2, 2, 4>(p, st) : launch_few<T, 1, 2, 5>(p, st);
    if (p.M <= 64 && !wide) return launch_few<T, 1, 4, 4>(p, st);
    auto tiles = [&](int bn, int bm) { return (p.N + bn - 1) / bn * ((p.M + bm - 1) / bm); };
    // Larger tiles read less, smaller ones fill the chip and keep more steps in flight.  Measured (bf16, us, with the quantisation; the
    // four tiles in the order below):   4400 x 256 x 2048     18    17    23    20
    //                                   1000 x 4096 x 4096    58    32    37    36
    //                                   512 x 4096 x 4096     56    29    22    22
    //                                   100 x 4096 x 4096     52    26    19    15
    //                                   8192 x 4096 x 14336   465   552   798   769
    if (tiles(256, 256) >= 256) return launch_tile<T, 4, 2, 2, 4, 2>(p, st);
    if (tiles(128, 128) >= 224) return launch_tile<T, 2, 2, 2, 2, 2>(p, st);
    if (tiles(128, 64) >= 128) return launch_tile<T, 2, 1, 2, 2, 4>(p, st);
    return launch_tile<T, 1, 1, 2, 2, 4>(p, st);
}

}  // namespace

extern "C" {

int64_t datr_quantized_row_bytes(int64_t K) { return K < 1 ? 0 : (K + kFewBytes - 1) / kFewBytes * kFewBytes; }

int datr_quantize_rows_i8(int dtype, const void *x, int64_t rows, int64_t K, int64_t ldx, int8_t *q, int64_t ldq, float *scale,
                          void *stream) {
    if (!elem::known(dtype) || rows < 0 || K < 1 || ldx < K || ldq != datr_quantized_row_bytes(K)) return DATR_EINVAL;
    if (rows == 0) return DATR_OK;
    if (rows >= (1LL << 24) || K > kMaxK) return DATR_EUNSUPPORTED;
    if (!x || !q || !scale || !elem::aligned16(q)) return DATR_EINVAL;
    return quantize_any(dtype, x, rows, K, ldx, q, ldq, scale, (hipStream_t)stream);
}

// q, then one scale per row; one token is quantised where it is multiplied
int64_t datr_linear_i8_workspace_bytes(int64_t M, int64_t K) {
    if (M == 1 && datr_quantized_row_bytes(K) <= kOneElements) return 0;
    return M < 1 || K < 1 || K > kMaxK ? 0 : M * datr_quantized_row_bytes(K) + (M * 4 + 127) / 128 * 128;
}

int datr_linear_i8(int dtype, const void *x, int64_t ldx, const int8_t *w, int64_t ldw, const float *w_scale, const float *bias,
                   int64_t M, int64_t N, int64_t K, int relu, int y_dtype, void *y, int64_t ldy, void *workspace,
                   int64_t workspace_bytes, void *stream) {
    if (!elem::known(dtype) || !elem::known(y_dtype) || M < 0 || N < 0 || K < 1 || ldx < K || ldw < K || ldy < N) return DATR_EINVAL;
    if (M == 0 || N == 0) return DATR_OK;
    if (K > kMaxK || M >= (1LL << 24) || N >= (1LL << 24) || ldw % 16 || ldw >= (1LL << 22)) return DATR_EUNSUPPORTED;
    if (!x || !w || !w_scale || !y || !elem::aligned16(w)) return DATR_EINVAL;
    const int64_t need = datr_linear_i8_workspace_bytes(M, K);
    if (workspace_bytes < need || (need > 0 && (!workspace || !elem::aligned16(workspace)))) return DATR_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    const int64_t lda = datr_quantized_row_bytes(K);
    int8_t *q = (int8_t *)workspace;
    float *scale = (float *)(q + M * lda);
    const Product p = {q, scale, w, w_scale, bias, y, M, N, K, lda, ldw, ldy, relu};
    if (M == 1 && lda <= kOneElements) {
        switch (y_dtype) {
            case DATR_FP32: return launch_one<float>(p, dtype, x, st);
            case DATR_FP16: return launch_one<_Float16>(p, dtype, x, st);
            default: return launch_one<__bf16>(p, dtype, x, st);
        }
    }
    const int rc = quantize_any(dtype, x, M, K, ldx, q, lda, scale, st);
    if (rc != DATR_OK) return rc;
    switch (y_dtype) {
        case DATR_FP32: return launch<float>(p, st);
        case DATR_FP16: return launch<_Float16>(p, st);
        default: return launch<__bf16>(p, st);
    }
}

}  // extern "C"
