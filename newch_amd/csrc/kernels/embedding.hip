// Rows of a table looked up by token and scaled, and the table's gradient: y[i] = s W[t_i], gW[v] (+)= s sum over t_i = v of g[i].  No
// counterpart in the reference on the device (its index_select copies rows on the host).
//
// The gradient sums in a fixed order without atomics.  Positions are sorted by (token, position); blocks of kSortedBlock sorted
// positions are summed by a lane for every four columns.  A token whose positions lie within one block has its row written there; one
// that goes over blocks leaves a part with each (at most two a block: one of a token that began before it, one of a token that goes on
// behind it), which a second kernel adds in the blocks' order, in fp64.  Rows of tokens that do not occur are cleared by workgroups of
// the same launch that look their rows up in the sorted tokens, so a stored gradient is written once.
//
// Bound by memory: reads 4 N D bytes of g, writes 4 V D (what is stored) or reads and writes the rows that occur (what is added).
#include "common.hpp"

#include <algorithm>

namespace nchip {

constexpr int kEmbB = 256;
constexpr int kSortedBlock = 32;  // sorted positions that one workgroup's lane sums
constexpr int kClearRows = 32;    // rows of the table that one workgroup clears, or as many as it has side by side
constexpr int kRankB = 1024, kRankWaves = kRankB / kWave;
constexpr int64_t kMaxTokens = int64_t(1) << 30;
constexpr int64_t kMaxRows = int64_t(1) << 31;

// A workgroup's lanes over a matrix: `lanes` (a power of two up to kEmbB) of them side by side over four columns each, kEmbB / lanes rows.
struct Lay {
    int64_t D;
    int shift;  // log2 of the lanes of a row
    int pieces() const { return (int)((D + 3) / 4); }
    int slices() const { return (pieces() + (1 << shift) - 1) >> shift; }
    int rows() const { return kEmbB >> shift; }
    int clear_rows() const { return rows() > kClearRows ? rows() : kClearRows; }
};

static Lay lay_of(int64_t D) {
    Lay l{D, 0};
    while ((1 << l.shift) < kEmbB && (1 << l.shift) < l.pieces()) l.shift++;
    return l;
}

template <bool AL>
__device__ __forceinline__ f4 piece(const float *row, int64_t c, int64_t D) {
    if (AL || c + 4 <= D) return AL ? *(const f4 *)(row + c) : (f4) * (const f4u *)(row + c);
    f4 v = {};
    for (int e = 0; e < (int)(D - c); e++) v[e] = row[c + e];
    return v;
}

template <bool AL>
__device__ __forceinline__ void put(float *row, int64_t c, int64_t D, f4 v) {
    if (AL) *(f4 *)(row + c) = v;
    else if (c + 4 <= D) *(f4u *)(row + c) = v;
    else
        for (int e = 0; e < (int)(D - c); e++) row[c + e] = v[e];
}

// ---- forward ------------------------------------------------------------------------------------------------
// tokens outside the table give rows of zeros
template <bool AL, int U>
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
    for (int u = 0; u < U; u++) v[u] = (uint32_t)t[u] < V ? piece<AL>(w + t[u] * ldw, c, l.D) : f4{};
#pragma unroll
    for (int u = 0; u < U; u++)
        if (i0 + u * rows < N) put<AL>(y + (i0 + u * rows) * l.D, c, l.D, v[u] * scale);
}

// the first token outside the table as (position << 32) | token, or all ones
__global__ __launch_bounds__(1024) void k_embed_check(const int32_t *__restrict__ tokens, int64_t N, int64_t V,
                                                      unsigned long long *__restrict__ bad) {
    __shared__ unsigned long long sh[1024 / kWave];
    unsigned long long k = ~0ull;
    for (int64_t i = threadIdx.x; i < N; i += 1024) {
        const uint32_t t = (uint32_t)tokens[i];
        if (t >= V && k == ~0ull) k = ((unsigned long long)i << 32) | t;
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
// A position's place is the number of those before it: tokens that are less, and equal ones at earlier positions.  A workgroup
// counts for 64 positions, a sixteenth of all tokens in each wave.  Tokens compare as unsigned, so those in the table come first.
__global__ __launch_bounds__(kRankB) void k_embed_rank(const uint32_t *__restrict__ tokens, int N, uint32_t *__restrict__ sorted,
                                                       int32_t *__restrict__ from) {
    __shared__ int counts[kRankWaves][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int first = blockIdx.x * kWave, i = first + lane;
    const uint32_t t = i < N ? tokens[i] : 0;
    const int per = (N + kRankWaves - 1) / kRankWaves;
    const int a = min(N, wave * per), b = min(N, a + per);
    int n = 0;
    for (int j = a; j < min(b, first); j++) n += tokens[j] <= t;
    for (int j = max(a, first); j < min(b, first + kWave); j++) n += tokens[j] < t || (tokens[j] == t && j < i);
    for (int j = max(a, first + kWave); j < b; j++) n += tokens[j] < t;
    counts[wave][lane] = n;
    __syncthreads();
    if (wave == 0 && i < N) {
        n = 0;
#pragma unroll
        for (int k = 0; k < kRankWaves; k++) n += counts[k][lane];
        sorted[n] = t;
        from[n] = i;
    }
}

// ---- the gradient ---------------------------------------------------------------------------------------------
struct EmbGrad {
    const uint32_t *sorted;
    const int32_t *from;
    const float *g;
    float *gw, *parts;  // parts: [blocks][2][4 pieces]
    int64_t N, V;
    int64_t blocks;      // of sorted positions
    unsigned sum_groups;  // workgroups that sum; the others clear
    uint32_t padding;    // a token without a gradient (>= V: none)
    float scale;
    int acc;
    int clear_rows;      // of a workgroup that clears
    Lay l;

    __device__ __forceinline__ bool counts(uint32_t t) const { return t < V && t != padding; }
};

template <bool AL>
__device__ __forceinline__ void put_row(const EmbGrad &p, uint32_t t, int64_t c, f4 sum) {
    float *row = p.gw + (int64_t)t * p.l.D;
    if (p.acc) {
        const f4 old = piece<AL>(row, c, p.l.D);
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = fma_(p.scale, sum[e], old[e]);
        put<AL>(row, c, p.l.D, v);
    } else {
        put<AL>(row, c, p.l.D, sum * p.scale);
    }
}

__device__ __forceinline__ float *part_at(const EmbGrad &p, int64_t block, int slot, int64_t c) {
    return p.parts + (block * 2 + slot) * ((p.l.D + 3) / 4 * 4) + c;
}

template <bool AL>
__device__ __forceinline__ void sum_block(const EmbGrad &p, int64_t block, int64_t c) {
    constexpr int U = 8;
    const int64_t k0 = block * kSortedBlock, k1 = min(p.N, k0 + kSortedBlock);
    uint32_t cur = p.sorted[k0];
    bool before = k0 > 0 && p.sorted[k0 - 1] == cur;  // the token began before this block
    f4 sum = {};
    auto flush = [&](bool goes_on) {
        if (!p.counts(cur)) return;
        if (before) *(f4 *)part_at(p, block, 0, c) = sum;
        else if (goes_on) *(f4 *)part_at(p, block, 1, c) = sum;
        else put_row<AL>(p, cur, c, sum);
    };
    for (int64_t k = k0; k < k1; k += U) {
        uint32_t t[U];
        f4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) t[u] = k + u < k1 ? p.sorted[k + u] : ~0u;
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = k + u < k1 && p.counts(t[u]) ? piece<AL>(p.g + p.from[k + u] * p.l.D, c, p.l.D) : f4{};
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (k + u >= k1) break;
            if (t[u] != cur) {
                flush(false);
                cur = t[u], before = false, sum = f4{};
            }
            sum = sum + v[u];
        }
    }
    flush(k1 < p.N && p.sorted[k1] == cur);
}

// of `count` rows of the table from r0 on, those whose tokens do not occur
template <bool AL>
__device__ __forceinline__ void clear_rows(const EmbGrad &p, int64_t r0, int count, int64_t c) {
    __shared__ int used[kEmbB];
    used[threadIdx.x] = 0;
    int64_t lo = 0, hi = p.N;  // the first sorted position of row r0 or later
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (p.sorted[mid] < r0) lo = mid + 1;
        else hi = mid;
    }
    __syncthreads();
    for (int64_t k = lo + threadIdx.x; k < p.N; k += kEmbB) {
        const uint32_t t = p.sorted[k];
        if (t >= r0 + count) break;
        if (p.counts(t)) used[t - r0] = 1;
    }
    __syncthreads();
    if (c >= p.l.D) return;
    for (int r = threadIdx.x >> p.l.shift; r < count; r += kEmbB >> p.l.shift)
        if (r0 + r < p.V && !used[r]) put<AL>(p.gw + (r0 + r) * p.l.D, c, p.l.D, f4{});
}

template <bool AL>
__global__ __launch_bounds__(kEmbB) void k_embed_grad(EmbGrad p) {
    const int64_t c = 4 * (((int64_t)blockIdx.y << p.l.shift) + (threadIdx.x & ((1 << p.l.shift) - 1)));
    if (blockIdx.x >= p.sum_groups) {
        clear_rows<AL>(p, (int64_t)(blockIdx.x - p.sum_groups) * p.clear_rows, p.clear_rows, c);
        return;
    }
    const int64_t block = (int64_t)blockIdx.x * (kEmbB >> p.l.shift) + (threadIdx.x >> p.l.shift);
    if (c < p.l.D && block < p.blocks) sum_block<AL>(p, block, c);
}

// The rows of tokens that go over blocks, where each begins.
template <bool AL>
__global__ __launch_bounds__(kEmbB) void k_embed_join(EmbGrad p) {
    constexpr int U = 8;
    const int64_t c = 4 * (((int64_t)blockIdx.y << p.l.shift) + (threadIdx.x & ((1 << p.l.shift) - 1)));
    const int64_t block = (int64_t)blockIdx.x * (kEmbB >> p.l.shift) + (threadIdx.x >> p.l.shift);
    const int64_t end = (block + 1) * kSortedBlock;
    if (c >= p.l.D || end >= p.N) return;
    const uint32_t t = p.sorted[end];
    if (!p.counts(t) || p.sorted[end - 1] != t) return;
    const int64_t begin = block * kSortedBlock;
    if (begin > 0 && p.sorted[begin - 1] == t) return;  // it began before
    int64_t last = block + 1;  // the block it ends in
    while ((last + 1) * kSortedBlock < p.N && p.sorted[(last + 1) * kSortedBlock] == t) last++;
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
    put_row<AL>(p, t, c, f4{(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]});
}

static size_t round16(size_t n) { return (n + 15) / 16 * 16; }

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
        if (U == 4) al ? run(k_embed<true, 4>) : run(k_embed<false, 4>);
        else al ? run(k_embed<true, 1>) : run(k_embed<false, 1>);
    }
    return check_launch(what);
}

extern "C" NC_HIP_API size_t nc_hip_embedding_bwd_workspace(int64_t N, int64_t V, int64_t D) {
    if (size_error(N, V, D) || N == 0) return 0;
    const int64_t blocks = (N + kSortedBlock - 1) / kSortedBlock;
    return 2 * round16((size_t)N * 4) + (size_t)blocks * 2 * (size_t)((D + 3) / 4 * 4) * sizeof(float);
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
    p.sorted = (uint32_t *)ws;
    p.from = (int32_t *)((char *)ws + round16((size_t)N * 4));
    p.parts = (float *)((char *)ws + 2 * round16((size_t)N * 4));
    p.g = g, p.gw = gw, p.N = N, p.V = V, p.scale = scale, p.acc = accumulate != 0;
    p.padding = padding >= 0 ? (uint32_t)padding : ~0u;
    p.blocks = (N + kSortedBlock - 1) / kSortedBlock;
    const int64_t groups = (p.blocks + p.l.rows() - 1) / p.l.rows();
    p.sum_groups = (unsigned)groups;
    p.clear_rows = p.l.clear_rows();
    const int64_t clear = accumulate ? 0 : (V + p.clear_rows - 1) / p.clear_rows;
    if ((groups + clear) * p.l.slices() * kEmbB > kMaxLanes || N * kRankWaves > kMaxLanes)
        return set_error(NC_HIP_ERR_ARG, "%s: bad size, no launch holds it", what);
    const bool al = D % 4 == 0 && aligned16(g) && aligned16(gw);
    if (N > 0)
        hipLaunchKernelGGL(k_embed_rank, (unsigned)((N + kWave - 1) / kWave), kRankB, 0, st, (const uint32_t *)tokens, (int)N,
                           (uint32_t *)p.sorted, (int32_t *)p.from);
    const dim3 grid((unsigned)(groups + clear), (unsigned)p.l.slices());
    if (al) hipLaunchKernelGGL(k_embed_grad<true>, grid, kEmbB, 0, st, p);
    else hipLaunchKernelGGL(k_embed_grad<false>, grid, kEmbB, 0, st, p);
    if (p.blocks > 1) {
        const dim3 joins((unsigned)groups, (unsigned)p.l.slices());
        if (al) hipLaunchKernelGGL(k_embed_join<true>, joins, kEmbB, 0, st, p);
        else hipLaunchKernelGGL(k_embed_join<false>, joins, kEmbB, 0, st, p);
    }
    return check_launch(what);
}
