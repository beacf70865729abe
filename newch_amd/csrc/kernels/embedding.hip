// Rows of a table looked up by token and scaled, and the table's gradient: y[i] = s W[t_i], gW[v] (+)= s sum over t_i = v of g[i].  No
// counterpart in the reference on the device (its index_select copies rows on the host).
//
// The gradient sums in a fixed order without atomics.  Of few tokens a workgroup for each sums its token's rows (k_embed_few).  Positions of
// more are sorted by (token, position); blocks of 8 or 32 sorted positions are summed by a lane for every four columns.  A token whose
// positions lie within one block has its row written there; one that goes over blocks leaves a part with each (at most two a block: one
// of a token that began before it, one of a token that goes on behind it), which a second kernel adds in the blocks' order, in fp64.
// Rows of tokens that do not occur are cleared by workgroups of the same launch, so a stored gradient is written once.
//
// Bound by memory: reads 4 N D bytes of g, writes 4 V D (what is stored) or reads and writes the rows that occur (what is added).
#include "common.hpp"

#include <algorithm>

namespace nchip {

constexpr int kEmbB = 256;
constexpr int kClearMost = 32768;  // words of the table that one workgroup clears, at most
constexpr int kClearFew = 4096;    // and, always as many, without a sort
constexpr int kRankB = 1024, kRankMost = 8192;  // tokens whose places are counted, at most
constexpr int kFewMost = 2560;                  // tokens whose rows are summed without a sort, at most
constexpr int kDigitBits = 10, kChunk = 1024;   // of the others' sort
constexpr int kSumChunks = 256;  // chunks whose counts each workgroup adds up itself, at most; more are summed by a launch of its own
constexpr int64_t kMaxTokens = int64_t(1) << 30;
constexpr int64_t kMaxRows = int64_t(1) << 31;

// A workgroup's lanes over a matrix: `lanes` (a power of two up to kEmbB) of them side by side over four columns each, kEmbB / lanes rows.
struct Lay {
    int64_t D;
    int shift;  // log2 of the lanes of a row
    int pieces() const { return (int)((D + 3) / 4); }
    int slices() const { return (pieces() + (1 << shift) - 1) >> shift; }
    int rows() const { return kEmbB >> shift; }
};

static Lay lay_of(int64_t D) {
    Lay l{D, 0};
    while ((1 << l.shift) < kEmbB && (1 << l.shift) < l.pieces()) l.shift++;
    return l;
}

// How rows are read and written: by aligned 16 bytes; by 16 bytes anywhere; rows of less than 16 bytes.
enum { ROWS_SHORT, ROWS_ANYWHERE, ROWS_ALIGNED };

// Four columns of a row from c on: loaded without a branch, since a lane that waits for a row's end of its own waits for each row, and behind
// the last four columns moved from those, by a step of its own that comes after the loads of all rows (885 tokens of 774 columns, both ways:
// 34 us by branches, 22 moved at once, 13 so).  What lies behind the row's end is anything.
template <int M>
__device__ __forceinline__ f4 load4(const float *row, int64_t c, int64_t D) {
    if (M == ROWS_ALIGNED) return *(const f4 *)(row + c);
    if (M == ROWS_SHORT) return f4{row[0], row[min(int64_t(1), D - 1)], row[D - 1], 0.0f};
    return *(const f4u *)(row + min(c, D - 4));
}

template <int M>
__device__ __forceinline__ f4 moved(f4 v, int64_t c, int64_t D) {
    if (M != ROWS_ANYWHERE || c <= D - 4) return v;
    const int by = (int)(c - (D - 4));
    return by == 1 ? f4{v[1], v[2], v[3], 0.0f} : by == 2 ? f4{v[2], v[3], 0.0f, 0.0f} : f4{v[3], 0.0f, 0.0f, 0.0f};
}

template <int M>
__device__ __forceinline__ void put(float *row, int64_t c, int64_t D, f4 v) {
    if (M == ROWS_ALIGNED) __builtin_nontemporal_store(v, (f4 *)(row + c));
    else if (c + 4 <= D) *(f4u *)(row + c) = v;
    else
        for (int e = 0; e < (int)(D - c); e++) row[c + e] = v[e];
}

// runs a call made for each of the three
template <class F>
static void by_rows(bool al, int64_t D, F run) {
    if (al) run(std::integral_constant<int, ROWS_ALIGNED>{});
    else if (D >= 4) run(std::integral_constant<int, ROWS_ANYWHERE>{});
    else run(std::integral_constant<int, ROWS_SHORT>{});
}

// ---- forward ------------------------------------------------------------------------------------------------
// tokens outside the table give rows of zeros
template <int M, int U>
__global__ __launch_bounds__(kEmbB) void k_embed(const float *__restrict__ w, int64_t ldw, const int32_t *__restrict__ tokens, float scale,
                                                 float *__restrict__ y, int64_t N, int64_t V, Lay l) {
    const int64_t c = 4 * (((int64_t)blockIdx.y << l.shift) + (threadIdx.x & ((1 << l.shift) - 1)));
    if (c >= l.D) return;
    const int rows = kEmbB >> l.shift;
    const int64_t i0 = (int64_t)blockIdx.x * rows * U + (threadIdx.x >> l.shift);
    int32_t t[U];
    f4 v[U];
#pragma unroll
    for (int u = 0; u < U; u++) t[u] = i0 + u * rows < N ? tokens[i0 + u * rows] : -1;
#pragma unroll
    for (int u = 0; u < U; u++) v[u] = (uint32_t)t[u] < V ? load4<M>(w + t[u] * ldw, c, l.D) : f4{};
#pragma unroll
    for (int u = 0; u < U; u++)
        if (i0 + u * rows < N) put<M>(y + (i0 + u * rows) * l.D, c, l.D, moved<M>(v[u], c, l.D) * scale);
}

// the first token outside the table as (position << 32) | token, or all ones
__global__ __launch_bounds__(1024) void k_embed_check(const int32_t *__restrict__ tokens, int64_t N, int64_t V,
                                                      unsigned long long *__restrict__ bad) {
    __shared__ unsigned long long sh[1024 / kWave];
    constexpr int U = 8;  // asked for together: 65536 tokens in 5 us, 2^20 in 100
    unsigned long long k = ~0ull;
    for (int64_t i0 = threadIdx.x; i0 < N; i0 += 1024 * U) {
        uint32_t t[U];
#pragma unroll
        for (int u = 0; u < U; u++) t[u] = i0 + u * 1024 < N ? (uint32_t)tokens[i0 + u * 1024] : 0;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + u * 1024 < N && t[u] >= V && k == ~0ull) k = ((unsigned long long)(i0 + u * 1024) << 32) | t[u];
    }
    k = wave_min_u64(k);
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = k;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 1024 / kWave; i++) k = sh[i] < k ? sh[i] : k;
        // at system scope: *bad may be host memory that the host watches while the kernel runs
        __hip_atomic_store(bad, k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
}

// ---- the order of the positions -----------------------------------------------------------------------------
// A position's place is the number of those that come before it by (token, position).  Tokens compare as unsigned, so those outside the
// table come last, in whatever order.
//
// Few tokens: every place by counting, in one launch.  A workgroup has 32 positions, all tokens in LDS, and counts with each half of its
// 16 waves over a thirty-second of them: 8192 tokens take two instructions a pair, 7 us.
__device__ __forceinline__ uint32_t sort_key(int32_t t) { return min((uint32_t)t, 0xfffffffeu); }  // a key has one above it

__global__ __launch_bounds__(kRankB) void k_embed_rank(const int32_t *__restrict__ tokens, int N, uint32_t *__restrict__ sorted,
                                                       int32_t *__restrict__ from) {
    __shared__ __attribute__((aligned(16))) uint32_t keys[kRankMost];
    __shared__ int counts[kRankB / 32][32];
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const int padded = (N + 127) / 128 * 128;  // a multiple of four keys for each of the 32 groups
    for (int j = threadIdx.x; j < padded; j += kRankB) keys[j] = j < N ? sort_key(tokens[j]) : 0xffffffffu;  // behind all others
    __syncthreads();
    const int col = threadIdx.x & 31, group = threadIdx.x / 32;
    const int first = blockIdx.x * 32, i = first + col;
    const uint32_t t = i < N ? keys[i] : 0;
    const int per = padded / 32, a = group * per, b = a + per;
    auto count = [&](int from_j, int to_j, uint32_t bound) {
        int n = 0;
#pragma unroll 4
        for (int j = from_j; j < to_j; j += 4) {
            const u4 k = *(const u4 *)(keys + j);
            n += (k.x < bound) + (k.y < bound) + (k.z < bound) + (k.w < bound);
        }
        return n;
    };
    int n = count(a, min(b, first), t + 1);                      // equal ones before the workgroup's positions come first,
    for (int j = max(a, first); j < min(b, first + 32); j++) n += keys[j] < t + (j < i);
    n += count(max(a, first + 32), b, t);                        // those behind them do not
    counts[group][col] = n;
    __syncthreads();
    if (group == 0 && i < N) {
        n = 0;
#pragma unroll
        for (int k = 0; k < kRankB / 32; k++) n += counts[k][col];
        sorted[n] = t;
        from[n] = i;
    }
}

// Many: digits of up to kDigitBits from the last to the first, two launches each.  A workgroup has kChunk positions in order.
struct Digits {
    const uint32_t *key_in;  // or none: the tokens themselves, and positions as they lie
    const int32_t *tokens, *from_in;
    uint32_t *key_out;
    int32_t *from_out;
    int *counts;  // [chunks][bins]; summed: of the chunks before, and of all in one more row
    bool summed;
    int N, chunks, bins, shift;
    uint32_t top;  // the key of all tokens outside the table: the number of its rows

    __device__ __forceinline__ uint32_t key(int i) const { return key_in ? key_in[i] : min((uint32_t)tokens[i], top); }
    __device__ __forceinline__ int digit(uint32_t k) const { return (int)(k >> shift) & (bins - 1); }
};

__global__ __launch_bounds__(kEmbB) void k_embed_digits(Digits p) {
    __shared__ int bin[1 << kDigitBits];
    for (int b = threadIdx.x; b < p.bins; b += kEmbB) bin[b] = 0;
    __syncthreads();
    const int i0 = blockIdx.x * kChunk;
#pragma unroll
    for (int u = 0; u < kChunk / kEmbB; u++) {
        const int i = i0 + u * kEmbB + threadIdx.x;
        if (i < p.N) atomicAdd(&bin[p.digit(p.key(i))], 1);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < p.bins; b += kEmbB) p.counts[(int64_t)blockIdx.x * p.bins + b] = bin[b];
}

// counts of the chunks before each, and of all
__global__ __launch_bounds__(kWave) void k_embed_sum(Digits p) {
    constexpr int U = 16;
    const int b = blockIdx.x * kWave + threadIdx.x;
    if (b >= p.bins) return;
    int sum = 0;
    for (int c0 = 0; c0 < p.chunks; c0 += U) {
        int n[U];
#pragma unroll
        for (int u = 0; u < U; u++) n[u] = c0 + u < p.chunks ? p.counts[(int64_t)(c0 + u) * p.bins + b] : 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c0 + u < p.chunks) p.counts[(int64_t)(c0 + u) * p.bins + b] = sum;
            sum += n[u];
        }
    }
    p.counts[(int64_t)p.chunks * p.bins + b] = sum;
}

// Each wave has a quarter of the chunk, in order: its positions of a digit go behind those of smaller digits, of earlier chunks and of
// the waves before it, and among themselves in their order.
__global__ __launch_bounds__(kEmbB) void k_embed_place(Digits p) {
    constexpr int kWaves = kEmbB / kWave, kEach = kChunk / kWaves, kBinsEach = (1 << kDigitBits) / kEmbB;
    __shared__ int at[kWaves][1 << kDigitBits];
    __shared__ int wave_total[kWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int b = threadIdx.x; b < kWaves << kDigitBits; b += kEmbB) (&at[0][0])[b] = 0;
    __syncthreads();
    const int i0 = blockIdx.x * kChunk + wave * kEach;
    uint32_t key[kEach / kWave];
    int from[kEach / kWave];
#pragma unroll
    for (int u = 0; u < kEach / kWave; u++) {
        const int i = i0 + u * kWave + lane;
        key[u] = i < p.N ? p.key(i) : 0;
        from[u] = i < p.N ? (p.key_in ? p.from_in[i] : i) : -1;
        if (from[u] >= 0) atomicAdd(&at[wave][p.digit(key[u])], 1);
    }
    __syncthreads();
    // this lane's kBinsEach digits, one after the other: how many in all, and in chunks before this one
    int total[kBinsEach], before[kBinsEach], sum = 0;
#pragma unroll
    for (int e = 0; e < kBinsEach; e++) {
        const int b = threadIdx.x * kBinsEach + e;
        total[e] = before[e] = 0;
        if (b < p.bins && p.summed) {
            before[e] = p.counts[(int64_t)blockIdx.x * p.bins + b];
            total[e] = p.counts[(int64_t)p.chunks * p.bins + b];
        } else if (b < p.bins)
#pragma unroll 8
            for (int c = 0; c < p.chunks; c++) {
                const int n = p.counts[(int64_t)c * p.bins + b];
                total[e] += n;
                before[e] += c < (int)blockIdx.x ? n : 0;
            }
        sum += total[e];
    }
    int up = sum;  // of this lane and those below it in the wave
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int v = __shfl_up(up, d);
        if (lane >= d) up += v;
    }
    if (lane == kWave - 1) wave_total[wave] = up;
    __syncthreads();
    int start = up - sum;
    for (int w = 0; w < wave; w++) start += wave_total[w];
#pragma unroll
    for (int e = 0; e < kBinsEach; e++) {
        const int b = threadIdx.x * kBinsEach + e;
        if (b < p.bins) {
            int here = start + before[e];
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const int n = at[w][b];
                at[w][b] = here;
                here += n;
            }
        }
        start += total[e];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kEach / kWave; u++) {
        const bool on = from[u] >= 0;
        const int d = p.digit(key[u]);
        unsigned long long same = __ballot(on);
        for (int bit = 0; (1 << bit) < p.bins; bit++) {
            const unsigned long long m = __ballot((d >> bit) & 1);
            same &= (d >> bit) & 1 ? m : ~m;
        }
        if (on) {
            const int to = at[wave][d] + __popcll(same & ((1ull << lane) - 1));
            p.key_out[to] = key[u];
            p.from_out[to] = from[u];
            // the digit's last lane moves its place on; the wave's lanes have read it
            if (same >> lane == 1) at[wave][d] = to + 1;
        }
    }
}

// ---- the gradient ---------------------------------------------------------------------------------------------
struct EmbGrad {
    const uint32_t *sorted;
    const int32_t *from;
    const float *g;
    float *gw, *parts;  // parts: [blocks][2][4 pieces]
    int64_t N, V;
    int64_t blocks;      // of S sorted positions
    unsigned sum_groups;  // workgroups that sum; the others clear
    uint32_t padding;    // a token without a gradient (>= V: none)
    float scale;
    int acc;
    int clear_words;     // of a workgroup that clears, a multiple of 4 kEmbB
    int clear_shift;     // words by which gw lies behind a 16-byte boundary
    Lay l;

    __device__ __forceinline__ bool counts(uint32_t t) const { return t < V && t != padding; }
};

template <int M>
__device__ __forceinline__ void put_row(const EmbGrad &p, uint32_t t, int64_t c, f4 sum) {
    float *row = p.gw + (int64_t)t * p.l.D;
    if (p.acc) {
        const f4 old = moved<M>(load4<M>(row, c, p.l.D), c, p.l.D);
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = fma_(p.scale, sum[e], old[e]);
        put<M>(row, c, p.l.D, v);
    } else {
        put<M>(row, c, p.l.D, sum * p.scale);
    }
}

__device__ __forceinline__ float *part_at(const EmbGrad &p, int64_t block, int slot, int64_t c) {
    return p.parts + (block * 2 + slot) * ((p.l.D + 3) / 4 * 4) + c;
}

template <int M, int S>
__device__ __forceinline__ void sum_block(const EmbGrad &p, int64_t block, int64_t c) {
    constexpr int U = 8;
    const int64_t k0 = block * S, k1 = min(p.N, k0 + S);
    uint32_t cur = p.sorted[k0];
    bool before = k0 > 0 && p.sorted[k0 - 1] == cur;  // the token began before this block
    f4 sum = {};
    auto flush = [&](bool goes_on) {
        if (!p.counts(cur)) return;
        if (before) *(f4 *)part_at(p, block, 0, c) = sum;
        else if (goes_on) *(f4 *)part_at(p, block, 1, c) = sum;
        else put_row<M>(p, cur, c, sum);
    };
    for (int64_t k = k0; k < k1; k += U) {
        uint32_t t[U];
        f4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) t[u] = k + u < k1 ? p.sorted[k + u] : ~0u;
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = k + u < k1 && p.counts(t[u]) ? load4<M>(p.g + p.from[k + u] * p.l.D, c, p.l.D) : f4{};
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (k + u >= k1) break;
            if (t[u] != cur) {
                flush(false);
                cur = t[u], before = false, sum = f4{};
            }
            sum = sum + moved<M>(v[u], c, p.l.D);
        }
    }
    flush(k1 < p.N && p.sorted[k1] == cur);
}

// A workgroup's words of the table, whatever rows they are of: cleared where the row's token does not occur.  By whole 16 bytes at their
// boundaries, since rows of odd lengths begin anywhere (84 tokens of 90560 x 2889, both ways: 306 us with rows stored as they begin, 180
// so).  Without a sort a workgroup clears 4096 words, since 32768 leave the memory idle at the end (213 us).  `find` marks the tokens that occur among rows r0 to r1.
template <class F>
__device__ __forceinline__ void clear_words(const EmbGrad &p, F find) {
    __shared__ uint32_t used[kClearMost / 32 + 1];
    __shared__ int any;
    const int64_t D = p.l.D, all = p.V * D;
    const int64_t chunk = (int64_t)blockIdx.y * (gridDim.x - p.sum_groups) + (blockIdx.x - p.sum_groups);
    const int64_t first = chunk * p.clear_words - p.clear_shift;  // 16-byte aligned, and before the table for the first chunk
    const int64_t f0 = max(first, int64_t(0)), f1 = min(first + p.clear_words, all);
    if (f0 >= f1) return;
    const int64_t r0 = f0 / D, r1 = (f1 - 1) / D;
    for (int k = threadIdx.x; k <= (int)(r1 - r0) / 32; k += kEmbB) used[k] = 0;
    if (threadIdx.x == 0) any = 0;
    __syncthreads();
    find(r0, r1, [&](uint32_t t) {
        const int k = (int)((int64_t)t - r0);
        atomicOr(used + k / 32, 1u << (k & 31));
        any = 1;
    });
    __syncthreads();
    const bool some = any;
    const float per = 1.0f / (float)D;
    const int64_t start = r0 * D;
    for (int k = threadIdx.x * 4; k < p.clear_words; k += 4 * kEmbB) {
        const int64_t i = first + k;
        if (i >= f0 && i + 4 <= f1 && !some) {
            __builtin_nontemporal_store(f4{}, (f4 *)(p.gw + i));
            continue;
        }
        if (i + 4 <= f0 || i >= f1) continue;
        const int64_t from = max(i, f0), rel = from - start;
        int r = (int)((float)rel * per);  // at most one off
        r += (int64_t)(r + 1) * D <= rel ? 1 : (int64_t)r * D > rel ? -1 : 0;
        const bool left = (int64_t)(r + 1) * D < i + 4 - start || i < f0 || i + 4 > f1;  // more than one row, or not whole
        if (!left) {
            if (!(used[r / 32] >> (r & 31) & 1)) __builtin_nontemporal_store(f4{}, (f4 *)(p.gw + i));
            continue;
        }
        int64_t next = (int64_t)(r + 1) * D;
        for (int64_t j = from; j < min(i + 4, f1); j++) {
            if (j - start >= next) r++, next += D;
            if (!(used[r / 32] >> (r & 31) & 1)) p.gw[j] = 0.0f;
        }
    }
}

// clear_words by the sorted tokens: 64 places at a time for the first of row r0 or later
__device__ __forceinline__ void clear_sorted(const EmbGrad &p) {
    clear_words(p, [&](int64_t r0, int64_t r1, auto mark) {
        int64_t lo = 0, hi = p.N;
        while (lo < hi) {
            const int64_t step = (hi - lo + kWave - 1) / kWave, k = lo + (int64_t)(threadIdx.x & (kWave - 1)) * step;
            const int less = __popcll(__ballot(k < hi && p.sorted[min(k, hi - 1)] < r0));
            hi = min(hi, lo + less * step);
            if (less) lo += (less - 1) * step + 1;
        }
        for (int64_t k = lo + threadIdx.x; k < p.N; k += kEmbB) {
            const uint32_t t = p.sorted[k];
            if (t > r1) break;
            if (p.counts(t)) mark(t);
        }
    });
}

template <int M, int S>
__global__ __launch_bounds__(kEmbB) void k_embed_grad(EmbGrad p) {
    const int64_t c = 4 * (((int64_t)blockIdx.y << p.l.shift) + (threadIdx.x & ((1 << p.l.shift) - 1)));
    if (blockIdx.x >= p.sum_groups) {
        clear_sorted(p);
        return;
    }
    const int64_t block = (int64_t)blockIdx.x * (kEmbB >> p.l.shift) + (threadIdx.x >> p.l.shift);
    if (c < p.l.D && block < p.blocks) sum_block<M, S>(p, block, c);
}

// Few tokens, in one launch and unsorted: a workgroup for every position, which goes on if its token has none earlier, lists the token's
// positions and sums their rows, 8 at a time and these in fp64; the workgroups behind them clear rows.
template <int M, int MOST>
__global__ __launch_bounds__(kEmbB) void k_embed_few(EmbGrad p, const int32_t *__restrict__ tokens) {
    constexpr int U = 8;
    // the tokens, and behind the last look at them the groups' sums: 2000 tokens of 512 columns 21.5 -> 18.9 us by the room it leaves
    __shared__ __attribute__((aligned(16))) uint32_t token[MOST > 8 * kEmbB ? MOST : 8 * kEmbB];
    double(*part)[kEmbB] = (double(*)[kEmbB])token;
    __shared__ uint16_t list[MOST];
    __shared__ unsigned long long masks[MOST / kWave];
    const int N = (int)p.N, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t c = 4 * (((int64_t)blockIdx.y << p.l.shift) + (threadIdx.x & ((1 << p.l.shift) - 1)));
    const int R = kEmbB >> p.l.shift, group = threadIdx.x >> p.l.shift;
    if (blockIdx.x >= p.sum_groups) {
        clear_words(p, [&](int64_t r0, int64_t r1, auto mark) {
#pragma unroll 4
            for (int j = threadIdx.x; j < N; j += kEmbB) {
                const uint32_t t = (uint32_t)tokens[j];
                if (p.counts(t) && t >= r0 && t <= r1) mark(t);
            }
        });
        return;
    }
#pragma unroll
    for (int u = 0; u < MOST / kEmbB; u++) {
        const int j = u * kEmbB + threadIdx.x;
        token[j] = j < N ? (uint32_t)tokens[j] : ~0u;
    }
    __syncthreads();
    const uint32_t t = token[blockIdx.x];
    if (!p.counts(t)) return;
#pragma unroll
    for (int u = 0; u < MOST / kEmbB; u++) {
        const unsigned long long m = __ballot(token[u * kEmbB + threadIdx.x] == t);
        if (lane == 0) masks[u * (kEmbB / kWave) + wave] = m;
    }
    __syncthreads();
    const unsigned long long mine = lane < MOST / kWave ? masks[lane] : 0;
    int upto = __popcll(mine);  // the token's positions up to this lane's mask
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int below = __shfl_up(upto, d);
        if (lane >= d) upto += below;
    }
    const int count = __shfl(upto, kWave - 1), k_first = __builtin_ctzll(__ballot(mine != 0));
    if (k_first * kWave + __builtin_ctzll(masks[k_first]) != (int)blockIdx.x) return;
#pragma unroll
    for (int u = 0; u < MOST / kEmbB; u++) {
        const int k = u * (kEmbB / kWave) + wave, before = __shfl(upto, k);
        const unsigned long long m = masks[k];
        if (m >> lane & 1) list[before - __popcll(m >> lane)] = (uint16_t)(k * kWave + lane);
    }
    __syncthreads();
    double sum[4] = {};
    if (c < p.l.D)
        for (int k0 = group; k0 < count; k0 += U * R) {
            f4 v[U];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = k0 + u * R < count ? load4<M>(p.g + (int64_t)list[k0 + u * R] * p.l.D, c, p.l.D) : f4{};
#pragma unroll
            for (int d = 1; d < U; d *= 2)
#pragma unroll
                for (int u = 0; u < U; u += 2 * d) v[u] = v[u] + v[u + d];
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] += (double)moved<M>(v[0], c, p.l.D)[e];
        }
    if (R > 1) {
#pragma unroll
        for (int e = 0; e < 4; e++) part[e][threadIdx.x] = sum[e];
        __syncthreads();
        if (group > 0) return;
        for (int r = 1; r < min(R, count); r++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] += part[e][(r << p.l.shift) + threadIdx.x];
    }
    if (c < p.l.D) put_row<M>(p, t, c, f4{(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]});
}

// The rows of tokens that go over blocks, where each begins.
template <int M, int S>
__global__ __launch_bounds__(kEmbB) void k_embed_join(EmbGrad p) {
    constexpr int U = 16;
    const int64_t c = 4 * (((int64_t)blockIdx.y << p.l.shift) + (threadIdx.x & ((1 << p.l.shift) - 1)));
    const int64_t block = (int64_t)blockIdx.x * (kEmbB >> p.l.shift) + (threadIdx.x >> p.l.shift);
    const int64_t end = (block + 1) * S;
    if (c >= p.l.D || end >= p.N) return;
    const uint32_t t = p.sorted[end];
    if (!p.counts(t) || p.sorted[end - 1] != t) return;
    const int64_t begin = block * S;
    if (begin > 0 && p.sorted[begin - 1] == t) return;  // it began before
    int64_t last = block + 1, step = 1;  // the block it ends in: in steps that double, then in halves
    auto holds = [&](int64_t b) { return b * S < p.N && p.sorted[b * S] == t; };
    while (holds(last + step)) last += step, step *= 2;
    for (; step > 0; step /= 2)
        if (holds(last + step)) last += step;
    const f4 head = *(const f4 *)part_at(p, block, 1, c);
    double sum[4] = {head[0], head[1], head[2], head[3]};
    for (int64_t b = block + 1; b <= last; b += U) {
        f4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = b + u <= last ? *(const f4 *)part_at(p, b + u, 0, c) : f4{};
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] += (double)v[u][e];
    }
    put_row<M>(p, t, c, f4{(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]});
}

static size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// Without a sort: 17 -> 12 us at 800 tokens of 100 columns, 19 -> 13 at 2331 of 256.  Every workgroup looks at all tokens, so its lead
// is gone from some number of them on, which depends on the words (us, unsorted : sorted; 10007 and 50000 rows): even ones over rows of 250
// and 256 columns 1536 14 : 17, 2304 18 : 18, 2560 23 : 21, 4096 31 : 23; of 16 to 128 columns 2560 14 : 16, 3088 15 : 16, 3584 17 : 17, 4096
// 20 : 17; frequencies as one over their rank 2560 16 : 23, 3584 29 : 28, 4096 33 : 30.  2560 lies between.  A token that all positions have
// is one workgroup's and slice's, so long rows of many tokens are sorted all the same (1024 times the same of 2048: 27 us sorted, 91
// unsorted; of 512: 47 unsorted, 2331 times of 256: 33 sorted, 50 unsorted).
static bool sums_unsorted(int64_t N, int64_t D) { return N <= kFewMost && N * D <= int64_t(1) << 20; }

// Sorted positions of a block: 8 where blocks of 32 would leave most of the chip idle (4378 tokens of 254 columns 46 -> 34 us, 4300 of 736
// 57 -> 54, 16245 of 256 alike), but of many tokens 32, since those that occur often go over many blocks (words' frequencies as one over
// their rank; 17000 of 64: 48 -> 46, 65536 of 64: 112 -> 78; 64 at a time take 97 with 100000 words, 76 with 300).
static int sorted_block(int64_t N, int64_t D) { return N < 16384 && (N + 31) / 32 * ((D + 3) / 4) < 65536 ? 8 : 32; }

// the workspace: [tokens in order][their positions], where digits are sorted the same again and the digits' counts, [parts]
struct SortPlan {
    int passes, bits, chunks;
    size_t list, counts, parts;
};
static SortPlan sort_plan(int64_t N, int64_t V) {
    SortPlan s{};
    s.list = round16((size_t)N * 4);
    if (N > kRankMost) {
        int bits = 1;
        while (bits < 31 && (int64_t(1) << bits) <= V) bits++;  // V itself is a key
        s.passes = (bits + kDigitBits - 1) / kDigitBits;
        s.bits = (bits + s.passes - 1) / s.passes;
        s.chunks = (int)((N + kChunk - 1) / kChunk);
        s.counts = 4 * s.list;
        s.parts = s.counts + round16(((size_t)(s.chunks + 1) << s.bits) * 4);
    } else {
        s.parts = 2 * s.list;
    }
    return s;
}

static const char *size_error(int64_t N, int64_t V, int64_t D) {
    if (N < 0 || N > kMaxTokens) return "0 to 2^30 tokens";
    if (V < 0 || V >= kMaxRows) return "0 to 2^31 - 1 rows";
    if (D < 1 || D > int64_t(1) << 24) return "1 to 2^24 columns";
    return nullptr;
}

}  // namespace nchip

using namespace nchip;

extern "C" NC_HIP_API int nc_hip_embedding_fwd(int64_t N, int64_t V, int64_t D, const float *w, int64_t ldw, const int32_t *tokens,
                                               float scale, float *y, uint64_t *bad, void *stream) {
    const char *what = "nc_hip_embedding_fwd";
    if (const char *e = size_error(N, V, D)) return set_error(NC_HIP_ERR_ARG, "%s: bad size, %s", what, e);
    if (N > 0 && (!tokens || !y || (V > 0 && !w))) return set_error(NC_HIP_ERR_ARG, "%s: NULL pointer", what);
    if (V > 1 && ldw < D) return set_error(NC_HIP_ERR_ARG, "%s: rows closer than their %lld columns", what, (long long)D);
    if (((uintptr_t)bad & 7u) != 0) return set_error(NC_HIP_ERR_ARG, "%s: bad is not 8-byte aligned", what);
    hipStream_t st = as_stream(stream);
    if (bad) hipLaunchKernelGGL(k_embed_check, 1, 1024, 0, st, tokens, N, V, (unsigned long long *)bad);
    if (N > 0) {
        const Lay l = lay_of(D);
        const bool al = D % 4 == 0 && ldw % 4 == 0 && aligned16(w) && aligned16(y);
        // four rows a lane where that leaves the chip full
        const int U = N * l.pieces() >= int64_t(1) << 20 ? 4 : 1;
        const int64_t per = (int64_t)l.rows() * U;
        const int64_t groups = (N + per - 1) / per;
        if (groups * l.slices() * kEmbB > kMaxLanes) return set_error(NC_HIP_ERR_ARG, "%s: bad size, no launch holds it", what);
        const dim3 grid((unsigned)groups, (unsigned)l.slices());
        auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, kEmbB, 0, st, w, ldw, tokens, scale, y, N, V, l); };
        by_rows(al, D, [&](auto m) {
            constexpr int M = decltype(m)::value;
            U == 4 ? run(k_embed<M, 4>) : run(k_embed<M, 1>);
        });
    }
    return check_launch(what);
}

extern "C" NC_HIP_API size_t nc_hip_embedding_bwd_workspace(int64_t N, int64_t V, int64_t D) {
    if (size_error(N, V, D) || sums_unsorted(N, D)) return 0;
    const int S = sorted_block(N, D);
    return sort_plan(N, V).parts + (size_t)((N + S - 1) / S) * 2 * (size_t)((D + 3) / 4 * 4) * sizeof(float);
}

extern "C" NC_HIP_API int nc_hip_embedding_bwd(int64_t N, int64_t V, int64_t D, const int32_t *tokens, int32_t padding, float scale,
                                               const float *g, float *gw, int accumulate, void *ws, size_t ws_bytes, void *stream) {
    const char *what = "nc_hip_embedding_bwd";
    if (const char *e = size_error(N, V, D)) return set_error(NC_HIP_ERR_ARG, "%s: bad size, %s", what, e);
    if (V == 0 || (N == 0 && accumulate)) return NC_HIP_OK;
    if (!gw || (N > 0 && (!tokens || !g))) return set_error(NC_HIP_ERR_ARG, "%s: NULL pointer", what);
    const size_t need = nc_hip_embedding_bwd_workspace(N, V, D);
    if (need && (!ws || ws_bytes < need)) return set_error(NC_HIP_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, need);
    if (((uintptr_t)ws & 15u) != 0) return set_error(NC_HIP_ERR_ARG, "%s: the workspace is not 16-byte aligned", what);
    hipStream_t st = as_stream(stream);
    EmbGrad p{};
    p.l = lay_of(D);
    const SortPlan sp = sort_plan(N, V);
    const int S = sorted_block(N, D);
    uint32_t *sorted = (uint32_t *)ws;
    int32_t *from = (int32_t *)((char *)ws + sp.list);
    p.sorted = sorted, p.from = from, p.parts = (float *)((char *)ws + sp.parts);
    p.g = g, p.gw = gw, p.N = N, p.V = V, p.scale = scale, p.acc = accumulate != 0;
    p.padding = padding >= 0 ? (uint32_t)padding : ~0u;
    p.blocks = (N + S - 1) / S;
    const bool few = sums_unsorted(N, D);
    const int64_t groups = few ? N : (p.blocks + p.l.rows() - 1) / p.l.rows();
    p.sum_groups = (unsigned)groups;
    const int64_t slices = p.l.slices(), words = V * D;
    p.clear_words = few ? kClearFew : (int)std::max<int64_t>(4 * kEmbB, std::min<int64_t>(kClearMost, words / 4096 / (4 * kEmbB) * (4 * kEmbB)));
    p.clear_shift = (int)((uintptr_t)gw / 4 & 3u);
    const int64_t chunks = (words + p.clear_shift + p.clear_words - 1) / p.clear_words;
    const int64_t clear = accumulate ? 0 : (chunks + slices - 1) / slices;
    if ((groups + clear) * slices * kEmbB > kMaxLanes)
        return set_error(NC_HIP_ERR_ARG, "%s: bad size, no launch holds it", what);
    const bool al = D % 4 == 0 && aligned16(g) && aligned16(gw);
    const dim3 grid((unsigned)(groups + clear), (unsigned)slices), joins((unsigned)groups, (unsigned)slices);
    if (few) {
        auto sum = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, kEmbB, 0, st, p, tokens); };
        by_rows(al, D, [&](auto m) {
            constexpr int M = decltype(m)::value;
            N <= 1024 ? sum(k_embed_few<M, 1024>) : sum(k_embed_few<M, kFewMost>);
        });
        return check_launch(what);
    }
    if (N > kRankMost) {
        // the last digit's places are the workspace's first lists: an odd number of digits starts there, an even one in the others
        uint32_t *keys[2] = {sorted, (uint32_t *)((char *)ws + 2 * sp.list)};
        int32_t *places[2] = {from, (int32_t *)((char *)ws + 3 * sp.list)};
        Digits d{nullptr, tokens, nullptr, nullptr, nullptr, (int *)((char *)ws + sp.counts), sp.chunks > kSumChunks, (int)N, sp.chunks, 1 << sp.bits, 0, (uint32_t)V};
        for (int i = 0; i < sp.passes; i++) {
            const int to = (sp.passes - 1 - i) & 1;
            d.key_out = keys[to], d.from_out = places[to], d.shift = i * sp.bits;
            hipLaunchKernelGGL(k_embed_digits, (unsigned)sp.chunks, kEmbB, 0, st, d);
            if (d.summed) hipLaunchKernelGGL(k_embed_sum, (unsigned)((d.bins + kWave - 1) / kWave), kWave, 0, st, d);
            hipLaunchKernelGGL(k_embed_place, (unsigned)sp.chunks, kEmbB, 0, st, d);
            d.key_in = d.key_out, d.from_in = d.from_out;
        }
    } else {
        hipLaunchKernelGGL(k_embed_rank, (unsigned)((N + 31) / 32), kRankB, 0, st, tokens, (int)N, sorted, from);
    }
    auto run = [&](auto kernel, dim3 g) { hipLaunchKernelGGL(kernel, g, kEmbB, 0, st, p); };
    by_rows(al, D, [&](auto m) {
        constexpr int M = decltype(m)::value;
        S == 8 ? run(k_embed_grad<M, 8>, grid) : run(k_embed_grad<M, 32>, grid);
        if (p.blocks > 1) S == 8 ? run(k_embed_join<M, 8>, joins) : run(k_embed_join<M, 32>, joins);
    });
    return check_launch(what);
}
