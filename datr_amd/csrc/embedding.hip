// embedding.hip -- rows of a table by token, scaled, and the table's gradient (gfx950).
//
//   forward    y[t, :]  = scale * W[id_t, :]                        (an id outside [0, V): a row of zeros)
//   backward   dW[v, :] = scale * sum over {t : id_t = v} dy[t, :]  in the tokens' order, held in fp32 and rounded once
//              to the table's type; rows without a token, and the padding row, are zeros.
//
// Both are bound by memory: forward reads min(T, V) rows and writes T, backward reads T rows of dy and writes all V rows
// of dW.  No atomics: every row of dW has one owner that adds its tokens in ascending order.
//
// 32 768 tokens of 128 000 rows x 4096 bf16: 356 us for both directions over 1.85 GB = 5.2 TB/s (a large copy on this card: 4.7).  In
// a kernel trace, which adds a little to each: forward 93, the sort with the zeros beside it 175, sums 82, their join 9.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <utility>

#include "datr_hip.h"
#include "elem.h"

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxTokens = 1LL << 27;

// `per_row` threads (a power of two) share a row
template <class T>
__global__ __launch_bounds__(kThreads) void embedding_fwd(const int64_t *__restrict__ ids, const T *__restrict__ table, int64_t tokens,
                                                          int64_t V, int D, int64_t ld, float scale, int per_row,
                                                          T *__restrict__ out) {
    constexpr int N = elem::Vec16<T>::N;
    const int rows = kThreads / per_row;
    for (int64_t t = (int64_t)blockIdx.x * rows + threadIdx.x / per_row; t < tokens; t += (int64_t)gridDim.x * rows) {
        const int64_t id = ids[t];
        const bool in = id >= 0 && id < V;
        const T *src = table + (in ? id : 0) * ld;
        T *dst = out + t * D;
#pragma unroll 4
        for (int c = (threadIdx.x % per_row) * N; c < D; c += per_row * N) {
            float f[N] = {};
            if (in) elem::to_float<T>(elem::load(src + c, D - c), f);
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] *= scale;
            elem::store(dst + c, f, D - c);
        }
    }
}

// ---- gradient, few tokens and rows: one workgroup per row of the table looks through all ids itself -------------------
// One launch instead of three.  A row's tokens are one workgroup's, so only while all of them together are short: the label table's
// 400 tokens and 10 rows of 256 take 5.3 us (three launches: 9.8), 2000 tokens and 200 rows of 256 take 8.8 (11.6); but 2000 tokens
// and 10 rows of 4096 would take 249 (18.9), 400 tokens and 10 rows of 4096 38.7 (10.6).
constexpr int kScanThreads = 512;
constexpr int kScanTokens = 2048;
constexpr int kScanRows = 1024;
constexpr int64_t kScanElements = 1 << 19;

template <class T>
__global__ __launch_bounds__(kScanThreads) void embedding_bwd_scan(const int64_t *__restrict__ ids, const T *__restrict__ dy, int tokens,
                                                                   int D, int64_t ld, float scale, int64_t padding,
                                                                   int across, T *__restrict__ dW) {
    constexpr int N = elem::Vec16<T>::N;
    __shared__ unsigned short list[kScanTokens];
    __shared__ int wave_n[kScanThreads / 64];
    __shared__ float part[kScanThreads * N];
    const int64_t v = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int n = 0;
    if (v != padding) {
        for (int base = 0; base < tokens; base += kScanThreads) {
            const bool hit = base + tid < tokens && ids[base + tid] == v;
            const unsigned long long m = __ballot(hit);
            if (lane == 0) wave_n[wave] = __popcll(m);
            __syncthreads();
            int at = n;
            for (int w = 0; w < kScanThreads / 64; ++w) {
                if (w < wave) at += wave_n[w];
                n += wave_n[w];
            }
            if (hit) list[at + __popcll(m & ((1ull << lane) - 1))] = (unsigned short)(base + tid);
            __syncthreads();
        }
    }
    // `across` threads (a power of two) side by side on a row; the groups take consecutive parts of the list, joined in order
    const int groups = kScanThreads / across, g = tid / across, x = tid % across;
    const int share = (n + groups - 1) / groups;
    const int lo = min(g * share, n), hi = min(lo + share, n);
    for (int c0 = 0; c0 < D; c0 += across * N) {
        const int c = c0 + x * N;
        float acc[N] = {};
        if (c < D) {
#pragma unroll 4
            for (int j = lo; j < hi; ++j) {
                float f[N];
                elem::to_float<T>(elem::load(dy + list[j] * ld + c, D - c), f);
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] += f[i];
            }
        }
        if (n > 1) {                                          // uniform over the workgroup
#pragma unroll
            for (int i = 0; i < N; ++i) part[i * kScanThreads + tid] = acc[i];
            __syncthreads();
            if (g == 0)
                for (int o = 1; o < groups && o * share < n; ++o)
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[i] += part[i * kScanThreads + o * across + x];
            __syncthreads();
        }
        if (g == 0 && c < D) {
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] *= scale;
            elem::store(dW + v * D + c, acc, D - c);
        }
    }
}

// ---- gradient, general: the tokens are sorted by id (stable, so a row's tokens stay in ascending order), then cut into
// chunks of equal length whatever their ids -- a frequent token's row is shared by many waves, a rare one's costs its own
// bytes.  A run of one id inside a chunk is a finished row of dW; runs that pass a chunk's border leave fp32 partial sums
// that a second kernel adds in the chunks' order.
//
// Ids that take no gradient (padding, outside the table) have the key V and sort to the end.  No atomic decides an order:
//   * up to 8192 tokens: a token's place is the number of smaller (key, position) pairs, counted against all others, T^2
//     comparisons spread over the chip in one launch (5000 tokens: 15.7 us for a radix sort in one workgroup's LDS -> 7.5);
//   * more: a radix sort by digits of up to 9 bits, least significant first, whose ranks come from ballots over the digit's
//     bits, wave by wave in token order.
//
// The radix sort is a chain of short dependent kernels (4-6 us each for 32 768 tokens) that leaves the chip idle, and most rows
// of a large table take no token: so the zeros of those rows are written by further workgroups of the sort's own launches, in
// equal shares.  (32 768 tokens x 4096, 128 000 rows, bf16: 329 -> 280 us for the gradient.)
constexpr int kRankThreads = 1024;
constexpr int kRankTokens = 8192;
constexpr int kRankShare = 32;                                   // tokens placed by one workgroup
constexpr int kPassThreads = 256;                                // a tile of the radix sort: 2048 tokens
constexpr int kItems = 8;
constexpr int kPassTile = kPassThreads * kItems;
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;

__device__ __forceinline__ unsigned key_of(int64_t id, int64_t V, int64_t padding) {
    return id >= 0 && id < V && id != padding ? (unsigned)id : (unsigned)V;
}

// rows v0 .. v0 + rows - 1 of dW that `empty` names become zeros: as many threads side by side as a row has 16-byte pieces
template <class F>
__device__ __forceinline__ void zero_rows(void *dW, int64_t v0, int rows, int64_t row_bytes, F empty) {
    int across = 1;
    while (across < (int)blockDim.x && across * 16 < row_bytes) across *= 2;
    const int x = threadIdx.x % across;
    for (int r = threadIdx.x / across; r < rows; r += blockDim.x / across) {
        if (!empty(r)) continue;
        char *row = (char *)dW + (v0 + r) * row_bytes;
        const int64_t head = min((int64_t)(-(intptr_t)row & 15), row_bytes), body = (row_bytes - head) & ~15LL;
        for (int64_t c = x * 16; c < body; c += across * 16) *reinterpret_cast<uint4 *>(row + head + c) = make_uint4(0, 0, 0, 0);
        for (int64_t c = x * 2; c < head; c += across * 2) *reinterpret_cast<unsigned short *>(row + c) = 0;
        for (int64_t c = head + body + x * 2; c < row_bytes; c += across * 2) *reinterpret_cast<unsigned short *>(row + c) = 0;
    }
}

// rows [from, to) of dW, `rows` a workgroup: zeros where present[] (nullptr: everywhere) has none
struct Zeros {
    void *dW;
    const unsigned char *present;
    int64_t from, to, row_bytes;
    int rows;
};

__device__ __forceinline__ void write_zeros(const Zeros &z, int64_t block) {
    const int64_t v0 = z.from + block * z.rows;
    const int rows = (int)min((int64_t)z.rows, z.to - v0);
    if (!z.present) return zero_rows((char *)z.dW + v0 * z.row_bytes, 0, 1, rows * z.row_bytes, [](int) { return true; });
    zero_rows(z.dW, v0, rows, z.row_bytes, [&](int r) { return !z.present[v0 + r]; });
}

template <int TH>
struct RankScratch {
    unsigned short count[TH / 64][kDigits];          // a wave's items of a digit; then the ones of the waves before it
    unsigned total[kDigits];
    unsigned wave_total[kDigits / 64];
};

// rank[i] = how many earlier items of this wave share item i's digit.  Item i of lane l of wave w is number
// (w * kItems + i) * 64 + l of the tile.  On return count[w][d] holds the items of digit d in the waves before w, total[d]
// those of the whole tile.
template <int TH>
__device__ __forceinline__ void rank_tile(const unsigned (&digit)[kItems], int bits, RankScratch<TH> &s, unsigned (&rank)[kItems]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < TH / 64 * kDigits / 2; i += TH) reinterpret_cast<unsigned *>(&s.count[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        unsigned long long peers = ~0ull;
        for (int b = 0; b < bits; ++b) {
            const bool one = (digit[i] >> b) & 1;
            const unsigned long long m = __ballot(one);
            peers &= one ? m : ~m;
        }
        const unsigned before = __popcll(peers & ((1ull << lane) - 1));
        const unsigned base = s.count[wave][digit[i]];
        rank[i] = base + before;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (before == 0) s.count[wave][digit[i]] = (unsigned short)(base + __popcll(peers));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (int d = tid; d < kDigits; d += TH) {
        unsigned n[TH / 64], sum = 0;
#pragma unroll
        for (int w = 0; w < TH / 64; ++w) n[w] = s.count[w][d];
#pragma unroll
        for (int w = 0; w < TH / 64; ++w) {
            s.count[w][d] = (unsigned short)sum;
            sum += n[w];
        }
        s.total[d] = sum;
    }
    __syncthreads();
}

// s.total[d] becomes the sum over the digits below d
template <int TH>
__device__ __forceinline__ void scan_totals(RankScratch<TH> &s) {
    const int tid = threadIdx.x, lane = tid & 63;
    for (int d = tid; d < kDigits; d += TH) {                    // whole waves: a wave's 64 digits at a time
        const unsigned own = s.total[d];
        unsigned sum = own;
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = __shfl_up(sum, o, 64);
            if (lane >= o) sum += t;
        }
        if (lane == 63) s.wave_total[d >> 6] = sum;
        s.total[d] = sum - own;
    }
    __syncthreads();
    for (int d = tid; d < kDigits; d += TH) {
        unsigned sum = s.total[d];
        for (int w = 0; w < (d >> 6); ++w) sum += s.wave_total[w];
        s.total[d] = sum;
    }
    __syncthreads();
}

// up to 8192 tokens, a key and a position in 32 bits; the workgroups behind the tokens' write zeros
__global__ __launch_bounds__(kRankThreads) void sort_rank(const int64_t *__restrict__ ids, int tokens, int64_t V, int64_t padding,
                                                          int position_bits, int blocks, unsigned *__restrict__ keys,
                                                          unsigned *__restrict__ order, Zeros zeros) {
    if ((int)blockIdx.x >= blocks) return write_zeros(zeros, blockIdx.x - blocks);
    // lane l of a wave counts for token t0 + l % 32, over one of kGroups equal parts of the tokens
    constexpr int kGroups = kRankThreads / kRankShare;
    __shared__ unsigned e[kRankTokens];
    __shared__ unsigned count[kGroups / 2][kRankShare];
    const int tid = threadIdx.x, x = tid % kRankShare, group = tid / kRankShare, t0 = blockIdx.x * kRankShare;
    const int part = ((tokens + kGroups - 1) / kGroups + 3) & ~3;
    for (int t = tid; t < part * kGroups; t += kRankThreads)
        e[t] = t < tokens ? key_of(ids[t], V, padding) << position_bits | (unsigned)t : ~0u;      // ~0: smaller than none
    __syncthreads();
    const unsigned own = t0 + x < tokens ? e[t0 + x] : 0;
    unsigned n = 0;
    for (int j = group * part; j < (group + 1) * part; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4 *>(e + j);
        n += (o.x < own) + (o.y < own) + (o.z < own) + (o.w < own);
    }
    n += __shfl_xor(n, kRankShare, 64);
    if ((group & 1) == 0) count[group / 2][x] = n;
    __syncthreads();
    if (tid < kRankShare && t0 + tid < tokens) {
        unsigned to = 0;
        for (int g = 0; g < kGroups / 2; ++g) to += count[g][tid];
        keys[to] = own >> position_bits;
        order[to] = own & ((1u << position_bits) - 1);
    }
}

// one pass of the sort of more tokens; ids: the first pass' input, then nullptr and keys / order
struct Pass {
    const int64_t *ids;
    const unsigned *keys, *order;
    unsigned *keys_out, *order_out, *hist, *totals;
    int64_t V, padding;
    int tokens, shift, bits, tiles;
};

__device__ __forceinline__ unsigned key_at(const Pass &p, int t) {
    if (t >= p.tokens) return ~0u;
    return p.ids ? key_of(p.ids[t], p.V, p.padding) : p.keys[t];
}

// per digit, the tiles' histograms; the first pass' further workgroups clear `present`, 16 bytes a thread, ...
__global__ __launch_bounds__(kPassThreads) void sort_count(Pass p, uint4 *clear, int64_t clear_n, Zeros zeros) {
    const int tid = threadIdx.x;
    if ((int)blockIdx.x >= p.tiles) {
        const int64_t block = blockIdx.x - p.tiles;
        if (clear) {
            if (block * kPassThreads + tid < clear_n) clear[block * kPassThreads + tid] = make_uint4(0, 0, 0, 0);
            return;
        }
        return write_zeros(zeros, block);
    }
    __shared__ unsigned count[kDigits];
    for (int d = tid; d < kDigits; d += kPassThreads) count[d] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) atomicAdd(&count[(key_at(p, blockIdx.x * kPassTile + i * kPassThreads + tid) >> p.shift) & ((1u << p.bits) - 1)], 1u);
    __syncthreads();
    for (int d = tid; d < 1 << p.bits; d += kPassThreads) p.hist[(int64_t)d * p.tiles + blockIdx.x] = count[d];
}

// ... their sums over the tiles before, one workgroup per digit; the first pass' further workgroups mark the rows that have a
// token (all write the same value), ...
__global__ __launch_bounds__(kPassThreads) void sort_scan(Pass p, unsigned char *mark, Zeros zeros) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if ((int)blockIdx.x >= 1 << p.bits) {
        const int64_t block = blockIdx.x - (1 << p.bits);
        if (mark) {
            const int64_t t = block * kPassThreads + tid;
            const unsigned k = t < p.tokens ? key_at(p, (int)t) : (unsigned)p.V;
            if (k < p.V) mark[k] = 1;
            return;
        }
        return write_zeros(zeros, block);
    }
    __shared__ unsigned wave_sum[kPassThreads / 64];
    unsigned *row = p.hist + (int64_t)blockIdx.x * p.tiles;
    unsigned carry = 0;
    for (int base = 0; base < p.tiles; base += kPassThreads) {
        const unsigned own = base + tid < p.tiles ? row[base + tid] : 0;
        unsigned sum = own;
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = __shfl_up(sum, o, 64);
            if (lane >= o) sum += t;
        }
        if (lane == 63) wave_sum[wave] = sum;
        __syncthreads();
        unsigned all = 0;
        for (int w = 0; w < kPassThreads / 64; ++w) {
            if (w < wave) sum += wave_sum[w];
            all += wave_sum[w];
        }
        if (base + tid < p.tiles) row[base + tid] = carry + sum - own;
        carry += all;
        __syncthreads();
    }
    if (tid == 0) p.totals[blockIdx.x] = carry;
}

// ... and every item to its place
__global__ __launch_bounds__(kPassThreads) void sort_place(Pass p, Zeros zeros) {
    if ((int)blockIdx.x >= p.tiles) return write_zeros(zeros, blockIdx.x - p.tiles);
    __shared__ RankScratch<kPassThreads> s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned key[kItems], digit[kItems], rank[kItems], before[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        key[i] = key_at(p, blockIdx.x * kPassTile + (wave * kItems + i) * 64 + lane);
        digit[i] = (key[i] >> p.shift) & ((1u << p.bits) - 1);
        before[i] = p.hist[(int64_t)digit[i] * p.tiles + blockIdx.x];
    }
    rank_tile(digit, p.bits, s, rank);
    for (int d = tid; d < kDigits; d += kPassThreads) s.total[d] = d < 1 << p.bits ? p.totals[d] : 0;
    __syncthreads();
    scan_totals(s);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int t = blockIdx.x * kPassTile + (wave * kItems + i) * 64 + lane;
        const unsigned to = s.total[digit[i]] + before[i] + s.count[wave][digit[i]] + rank[i];
        if (t < p.tokens) {
            p.keys_out[to] = key[i];
            p.order_out[to] = p.ids ? (unsigned)t : p.order[t];
        }
    }
}

template <int N>
__device__ __forceinline__ void store_partial(float *p, const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
}

template <int N>
__device__ __forceinline__ void add_partial(const float *p, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 q = *reinterpret_cast<const float4 *>(p + i);
        f[i] += q.x, f[i + 1] += q.y, f[i + 2] += q.z, f[i + 3] += q.w;
    }
}

// One wave per (chunk, column tile).
// partial [chunks][2][Dp]: slot 0 a run that began before the chunk, slot 1 one that begins in it and goes on behind it.
template <class T>
__global__ __launch_bounds__(kThreads) void embedding_bwd_runs(const unsigned *__restrict__ keys, const unsigned *__restrict__ order,
                                                               const T *__restrict__ dy, int tokens, int64_t V, int D, int64_t ld,
                                                               float scale, int chunk, int tiles, int64_t units, int64_t Dp, float *__restrict__ partial,
                                                               T *__restrict__ dW) {
    constexpr int N = elem::Vec16<T>::N;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (unit >= units) return;
    const int64_t ch = unit / tiles;
    const int c = (int)(unit - ch * tiles) * 64 * N + lane * N;
    const int lo = (int)(ch * chunk), n = min(chunk, tokens - lo);
    const int key = lane < n ? (int)keys[lo + lane] : -1;
    const int at = lane < n ? (int)order[lo + lane] : 0;
    const int before = lo > 0 ? (int)keys[lo - 1] : -1, behind = lo + n < tokens ? (int)keys[lo + n] : -1;
    const int live = __popcll(__ballot(lane < n && key < V));    // ids without a gradient are the last
    if (live == 0) return;
    constexpr int U = 8;                                         // rows in flight
    // dy's rows are read once, past the caches: 5 % of both directions of that batch
    auto row = [&](int j) { return c < D ? elem::load<true>(dy + (int64_t)__builtin_amdgcn_readlane(at, min(j, live - 1)) * ld + c, D - c)
                                         : typename elem::Vec16<T>::type{}; };
    typename elem::Vec16<T>::type next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = row(u);
    float acc[N] = {};
    int cur = __builtin_amdgcn_readlane(key, 0);
    bool began_before = cur == before;
    auto flush = [&](bool goes_on) {
        if (began_before || goes_on) {
            if (c < D) store_partial<N>(partial + (ch * 2 + (began_before ? 0 : 1)) * Dp + c, acc);
        } else if (c < D) {
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] *= scale;
            elem::store(dW + (int64_t)cur * D + c, acc, D - c);
        }
        began_before = false;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
    };
    for (int j = 0; j < live; j += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (j + u >= live) break;
            float f[N];
            elem::to_float<T>(next[u], f);
            next[u] = row(j + u + U);
            const int k = __builtin_amdgcn_readlane(key, j + u);
            if (k != cur) {
                flush(false);
                cur = k;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += f[i];
        }
    }
    flush(live == n && cur == behind);
}

// One workgroup per (chunk, column tile) in which a run begins that goes on behind the chunk: its waves add consecutive parts of
// the run's partial sums, joined in order.
constexpr int kJoinThreads = 512;

template <class T>
__global__ __launch_bounds__(kJoinThreads) void embedding_bwd_join(const unsigned *__restrict__ keys, int tokens, int64_t V, int D,
                                                                   float scale, int chunk, int tiles, int64_t Dp,
                                                                   const float *__restrict__ partial, T *__restrict__ dW) {
    constexpr int N = elem::Vec16<T>::N, W = kJoinThreads / 64;
    __shared__ float part[N][kJoinThreads];
    const int64_t ch = blockIdx.x / tiles;
    const int lo = (int)(ch * chunk), hi = min(lo + chunk, tokens);
    if (hi >= tokens) return;
    const unsigned k = keys[hi - 1];
    if (k >= V || keys[hi] != k || (keys[lo] == k && lo > 0 && keys[lo - 1] == k)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = (int)(blockIdx.x - ch * tiles) * 64 * N + lane * N;
    // chunks behind this one that the run reaches: those whose first key is k
    const int chunks = (tokens + chunk - 1) / chunk;
    int reach = 0;
    for (int o = (int)ch + 1;; o += 64) {
        const bool in = o + lane < chunks && keys[(int64_t)(o + lane) * chunk] == k;
        const unsigned long long out = ~__ballot(in);
        if (out) {
            reach += __ffsll((unsigned long long)out) - 1;
            break;
        }
        reach += 64;
    }
    const int n = reach + 1, share = (n + W - 1) / W;
    const int a = min(wave * share, n), b = min(a + share, n);
    float acc[N] = {};
    if (c < D) {
#pragma unroll 4
        for (int j = a; j < b; ++j) add_partial<N>(partial + ((ch + j) * 2 + (j == 0 ? 1 : 0)) * Dp + c, acc);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) part[i][threadIdx.x] = acc[i];
    __syncthreads();
    if (wave || c >= D) return;
    for (int w = 1; w < W && w * share < n; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += part[i][w * 64 + lane];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= scale;
    elem::store(dW + (int64_t)k * D + c, acc, D - c);
}

template <class T>
int forward(const int64_t *ids, const void *table, int64_t tokens, int64_t V, int64_t D, int64_t ld, float scale, void *out,
            hipStream_t st) {
    // as many threads on a row as are busy seven times out of eight, 16 at least
    const int64_t vectors = (D + elem::Vec16<T>::N - 1) / elem::Vec16<T>::N;
    int per_row = kThreads;
    while (per_row > 16 && vectors * 8 < (vectors + per_row - 1) / per_row * per_row * 7) per_row /= 2;
    int64_t blocks = (tokens + kThreads / per_row - 1) / (kThreads / per_row);
    if (blocks > 1 << 20) blocks = 1 << 20;
    hipLaunchKernelGGL(embedding_fwd<T>, dim3((unsigned)blocks), dim3(kThreads), 0, st, ids, (const T *)table, tokens, V,
                       (int)D, ld, scale, per_row, (T *)out);
    return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
}

// how the gradient of `tokens` tokens is computed, and where its parts lie in the workspace
struct Plan {
    bool scan;                                                   // the one-launch kernel
    bool rank;                                                   // sorted by counting, else by digits
    int position_bits, passes, bits, tiles, chunk;
    int64_t chunks, Dp, keys, order, keys2, order2, hist, totals, present, partial, bytes;
};

Plan plan_of(int64_t tokens, int64_t V, int64_t D) {
    Plan p = {};
    p.scan = tokens <= kScanTokens && V <= kScanRows && tokens * D <= kScanElements;
    if (p.scan) return p;
    int need = 1;
    while ((V >> need) != 0) ++need;                             // keys 0 .. V
    p.passes = (need + kDigitBits - 1) / kDigitBits;
    p.bits = (need + p.passes - 1) / p.passes;
    while (tokens > 1LL << p.position_bits) ++p.position_bits;
    p.rank = tokens <= kRankTokens && need + p.position_bits <= 32;
    // (beside the ranking every row is zeroed, and the few with tokens are written again: looking the others up in the sorted keys
    // afterwards takes 48 us instead of 41 at 8000 tokens of 30 000 rows x 1024)
    p.tiles = (int)((tokens + kPassTile - 1) / kPassTile);
    // 64 tokens a wave where that gives the chip enough waves
    p.chunk = 64;
    while (p.chunk > 8 && tokens / p.chunk * ((D + 255) / 256) < 2048) p.chunk /= 2;
    p.chunks = (tokens + p.chunk - 1) / p.chunk;
    p.Dp = (D + 7) / 8 * 8;
    int64_t at = 0;
    auto take = [&](int64_t n) {
        const int64_t here = at;
        at += (n * 4 + 255) / 256 * 256;
        return here;
    };
    p.keys = take(tokens);
    p.order = take(tokens);
    if (!p.rank) {
        p.keys2 = take(tokens);
        p.order2 = take(tokens);
        p.hist = take((int64_t)kDigits * p.tiles);
        p.totals = take(kDigits);
        p.present = take((V + 3) / 4);
    }
    p.partial = take(p.chunks * 2 * p.Dp);
    p.bytes = at;
    return p;
}

template <class T>
int backward(const int64_t *ids, const void *dy, int64_t tokens, int64_t V, int64_t D, int64_t ld, float scale, int64_t padding,
             void *dW, char *ws, hipStream_t st) {
    const Plan p = plan_of(tokens, V, D);
    if (p.scan) {
        int across = 16;
        while (across < kScanThreads && across * elem::Vec16<T>::N < D) across *= 2;
        hipLaunchKernelGGL(embedding_bwd_scan<T>, dim3((unsigned)V), dim3(kScanThreads), 0, st, ids, (const T *)dy, (int)tokens, (int)D,
                           ld, scale, padding, across, (T *)dW);
        return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
    }
    const int n = (int)tokens;
    unsigned *keys = (unsigned *)(ws + p.keys), *order = (unsigned *)(ws + p.order);
    // zeros: 64 bytes a thread and workgroup (32 768 tokens, 128 000 rows of 8 KB: 64 KB a workgroup of 256 is 3 % slower)
    int rows = (int)((p.rank ? 64 * kRankThreads : 64 * kPassThreads) / (D * (int64_t)sizeof(T)));
    rows = rows < 1 ? 1 : rows > kThreads ? kThreads : rows;
    Zeros zeros = {dW, nullptr, 0, V, D * (int64_t)sizeof(T), rows};
    auto blocks_of = [&](const Zeros &z) { return (z.to - z.from + rows - 1) / rows; };
    const int tiles = (int)((D + 64 * elem::Vec16<T>::N - 1) / (64 * elem::Vec16<T>::N));
    const int64_t units = p.chunks * tiles, blocks = (units + kThreads / 64 - 1) / (kThreads / 64);
    if ((blocks_of(zeros) + kRankTokens) * kRankThreads >= (1LL << 32) || blocks * kThreads >= (1LL << 32) || units * kJoinThreads >= (1LL << 32))
        return DATR_EUNSUPPORTED;
    if (p.rank) {
        const int rank_blocks = (n + kRankShare - 1) / kRankShare;
        if (rank_blocks + blocks_of(zeros) > 0)
            hipLaunchKernelGGL(sort_rank, dim3((unsigned)(rank_blocks + blocks_of(zeros))), dim3(kRankThreads), 0, st, ids, n, V, padding,
                               p.position_bits, rank_blocks, keys, order, zeros);
    } else {
        Pass pass = {ids, nullptr, nullptr, (unsigned *)(ws + p.keys2), (unsigned *)(ws + p.order2), (unsigned *)(ws + p.hist),
                     (unsigned *)(ws + p.totals), V, padding, n, 0, p.bits, p.tiles};
        zeros.present = (unsigned char *)(ws + p.present);
        const int64_t shares = 1 + 3 * (p.passes - 1), share = (V + shares - 1) / shares;
        zeros.to = 0;
        auto next = [&] {                                        // the rows of one launch
            zeros.from = zeros.to;
            zeros.to = zeros.to + share < V ? zeros.to + share : V;
            return (unsigned)blocks_of(zeros);
        };
        const int64_t clear_n = (V + 15) / 16;
        for (int i = 0; i < p.passes; ++i) {
            pass.shift = i * p.bits;
            const unsigned more_count = i ? next() : (unsigned)((clear_n + kPassThreads - 1) / kPassThreads);
            hipLaunchKernelGGL(sort_count, dim3(p.tiles + more_count), dim3(kPassThreads), 0, st, pass,
                               i ? nullptr : (uint4 *)(ws + p.present), clear_n, zeros);
            const unsigned more_scan = i ? next() : (unsigned)((n + kPassThreads - 1) / kPassThreads);
            hipLaunchKernelGGL(sort_scan, dim3((1u << p.bits) + more_scan), dim3(kPassThreads), 0, st, pass,
                               i ? nullptr : (unsigned char *)(ws + p.present), zeros);
            const unsigned more_place = next();
            hipLaunchKernelGGL(sort_place, dim3(p.tiles + more_place), dim3(kPassThreads), 0, st, pass, zeros);
            keys = pass.keys_out, order = pass.order_out;
            pass.keys_out = (unsigned *)(ws + (i & 1 ? p.keys2 : p.keys));
            pass.order_out = (unsigned *)(ws + (i & 1 ? p.order2 : p.order));
            pass.ids = nullptr, pass.keys = keys, pass.order = order;
        }
    }
    float *partial = (float *)(ws + p.partial);
    if (blocks == 0) return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
    hipLaunchKernelGGL(embedding_bwd_runs<T>, dim3((unsigned)blocks), dim3(kThreads), 0, st, keys, order, (const T *)dy, n, V, (int)D, ld,
                       scale, p.chunk, tiles, units, p.Dp, partial, (T *)dW);
    if (p.chunks > 1)
        hipLaunchKernelGGL(embedding_bwd_join<T>, dim3((unsigned)units), dim3(kJoinThreads), 0, st, keys, n, V, (int)D, scale, p.chunk, tiles,
                           p.Dp, partial, (T *)dW);
    return hipGetLastError() == hipSuccess ? DATR_OK : DATR_ELAUNCH;
}

}  // namespace

extern "C" {

int datr_embedding_forward(int dtype, const int64_t *ids, const void *table, int64_t tokens, int64_t V, int64_t D, int64_t ld,
                           float scale, void *out, void *stream) {
    if (!elem::known(dtype) || tokens < 0 || V < 0 || D < 0 || ld < D) return DATR_EINVAL;
    if (tokens == 0 || D == 0) return DATR_OK;
    if (tokens >= (1LL << 31) || V >= (1LL << 31) || D >= (1LL << 24)) return DATR_EUNSUPPORTED;
    if (!ids || !out || (!table && V > 0)) return DATR_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case DATR_FP32: return forward<float>(ids, table, tokens, V, D, ld, scale, out, st);
        case DATR_FP16: return forward<_Float16>(ids, table, tokens, V, D, ld, scale, out, st);
        default: return forward<__bf16>(ids, table, tokens, V, D, ld, scale, out, st);
    }
}

int64_t datr_embedding_backward_workspace_bytes(int64_t tokens, int64_t V, int64_t D) {
    if (tokens < 0 || V < 0 || D < 0 || tokens > kMaxTokens || V >= (1LL << 31) - 1 || D >= (1LL << 24)) return 0;
    return plan_of(tokens, V, D).bytes;
}

int datr_embedding_backward(int dtype, const int64_t *ids, const void *dy, int64_t tokens, int64_t V, int64_t D, int64_t ld,
                            float scale, int64_t padding, void *dW, void *workspace, int64_t workspace_bytes, void *stream) {
    if (!elem::known(dtype) || tokens < 0 || V < 0 || D < 0 || ld < 0) return DATR_EINVAL;
    if (V == 0 || D == 0) return DATR_OK;
    if (tokens > kMaxTokens || V >= (1LL << 31) - 1 || D >= (1LL << 24)) return DATR_EUNSUPPORTED;
    if (workspace_bytes < plan_of(tokens, V, D).bytes || (workspace_bytes > 0 && !workspace)) return DATR_EINVAL;
    if (!dW || (tokens > 0 && (!ids || !dy))) return DATR_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case DATR_FP32: return backward<float>(ids, dy, tokens, V, D, ld, scale, padding, dW, (char *)workspace, st);
        case DATR_FP16: return backward<_Float16>(ids, dy, tokens, V, D, ld, scale, padding, dW, (char *)workspace, st);
        default: return backward<__bf16>(ids, dy, tokens, V, D, ld, scale, padding, dW, (char *)workspace, st);
    }
}

}  // extern "C"
