// Cross entropy of z = x W^T + b against labels, with its gradients, z held for a piece of the rows at a time.  The reference multiplies
// and takes the loss of stored logits [N, V] (linear, ops_linalg.c:255-330; cross_entropy, ops_nn.c:83-156), which come to gigabytes for
// a language model's vocabulary.
//
// Row i counts where its label is not `ignore`: loss_i = log sum_v exp z_iv - z_il, loss = their mean (or sum).  The gradients follow from
// G = softmax(z) - onehot(l), scaled by 1 / count and by the loss's own gradient: gx = G W, gW = G^T x, gb = column sums of G; rows that
// do not count have none, and what their x holds counts nowhere.
//
// A row's own entry of G is -(1 - p_l) = -others / (others + e_l), with the exponentials of the other words summed by
// themselves: p_l - 1 would lose the bits of a word that is all but certain.
#include "vocab_loss.hpp"

namespace nchip {

constexpr size_t kVlPiece = size_t(1) << 30;  // bytes of z held at a time
constexpr int64_t kVlRows = 32768;            // and rows

// Rows whose count the workgroup of every short row takes for itself, at most, in place of a launch: 64 and 256 rows over 1000 words are
// 1.6 us faster by it, 2000 no more, 4000 to 8000 4 to 20 us slower.
constexpr int64_t kVlCountMost = 1024;
constexpr int kVlChunk = 2048;  // words of a row that a workgroup takes, where a row is shared by several
constexpr int kVlShort = 4096;  // words of a row that one workgroup takes alone, at most

struct VlArgs {
    int64_t N, V, ldz;
    int64_t row0, rows;  // the rows of this piece
    int chunks;          // of a row
    const int32_t *labels;
    int32_t ignore;
    int sum;
    bool count_here;  // the rows that count are counted here, not by k_vl_count
    VlHead *head;
    unsigned long long *bad;
    const float *gout;
    const float *x;
    int64_t ldx, D;
    float *clean;      // [N][D], x with zeros for the rows that do not count, or none
    float *z;          // [rows][ldz]: the products, then G
    f2 *part;          // [rows][chunks] {maximum, sum of exponentials}, the label's left out of the sum
    float *label_z;    // [rows]
    double *row_loss;  // [N]
    float *row_out;    // [N] or none
};

// Rows that count, and, SAY, for the head and the caller, the first label that is neither a word nor `ignore`, as (row << 32) | label, or
// all ones.
template <int B, bool SAY>
__device__ __forceinline__ int64_t vl_count(const VlArgs &p, double *sh) {
    __shared__ unsigned long long shk[B / kWave];
    unsigned long long k = ~0ull;
    double n = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < p.N; i += B) {
        const int32_t l = p.labels[i];
        if (vl_counts(l, p.ignore, p.V)) n += 1.0;
        else if (SAY && l != p.ignore && k == ~0ull) k = ((unsigned long long)i << 32) | (uint32_t)l;
    }
    if (SAY) {
        k = wave_min_u64(k);
        if ((threadIdx.x & (kWave - 1)) == 0) shk[threadIdx.x / kWave] = k;
    }
    n = vl_wg_sum(n, sh);
    if (SAY && threadIdx.x == 0) {
        for (int i = 1; i < B / kWave; i++) k = shk[i] < k ? shk[i] : k;
        p.head->count = (int64_t)n;
        // at system scope: *bad may be host memory that the host watches while the kernel runs
        if (p.bad) __hip_atomic_store(p.bad, k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
    return (int64_t)n;
}

__global__ __launch_bounds__(1024) void k_vl_count(VlArgs p) {
    __shared__ double sh[1024 / kWave];
    vl_count<1024, true>(p, sh);
}

// this workgroup's share, part of parts, of row i of the x that gW takes
__device__ __forceinline__ void vl_clean(const VlArgs &p, int64_t i, bool on, int part, int parts) {
    if (p.clean)
        for (int64_t d = (int64_t)part * kVlB + threadIdx.x; d < p.D; d += (int64_t)parts * kVlB)
            p.clean[i * p.D + d] = on ? p.x[i * p.ldx + d] : 0.0f;
}

// what a row's G is made from
struct VlStat {
    float m, ls, own, coef;
};

__device__ __forceinline__ VlStat vl_stat(const VlArgs &p, int64_t i, float m, double others, float zl, int64_t count, bool first) {
    const double own = (double)exp8_nonpos(zl), total = others + own;
    const double ls = zl == 0.0f ? log1p(others) : log(total);
    if (first) {
        const double loss = ls - (double)zl;
        p.row_loss[i] = loss;
        if (p.row_out) p.row_out[i] = (float)loss;
    }
    const float c = p.gout ? *p.gout : 1.0f;
    return {m, (float)ls, (float)(-others / total), p.sum ? c : c / (float)count};
}

__device__ __forceinline__ float vl_entry(float z, int64_t v, int32_t label, const VlStat &s) {
    return (v == label ? s.own : exp8_nonpos((z - s.m) - s.ls)) * s.coef;
}

// A workgroup's row of up to kVlShort words, in registers: its statistics, its loss, and, GRAD, its row of G in place of z.
template <bool GRAD>
__global__ __launch_bounds__(kVlB) void k_vl_softmax(VlArgs p) {
    constexpr int kEach = kVlShort / kVlB;
    __shared__ double sh[kVlB / kWave];
    __shared__ float shm[kVlB / kWave], own;
    const int64_t r = blockIdx.x, i = p.row0 + r;
    const int V = (int)p.V;
    float *z = p.z + r * p.ldz;
    const int32_t l = p.labels[i];
    const bool on = vl_counts(l, p.ignore, p.V);
    if (GRAD) vl_clean(p, i, on, 0, 1);
    if (p.count_here && r == 0) vl_count<kVlB, true>(p, sh);
    if (!on) {
        if (threadIdx.x == 0) {
            p.row_loss[i] = 0.0;
            if (p.row_out) p.row_out[i] = 0.0f;
        }
        if (GRAD)
            for (int v = threadIdx.x; v < V; v += kVlB) z[v] = 0.0f;
        return;
    }
    float x[kEach], m = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < kEach; k++) x[k] = k * kVlB + (int)threadIdx.x < V ? z[k * kVlB + threadIdx.x] : -__builtin_inff();
    const int64_t count = !GRAD || p.sum ? 0 : p.count_here ? vl_count<kVlB, false>(p, sh) : p.head->count;
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        m = __builtin_fmaxf(m, x[k]);
        if (k * kVlB + (int)threadIdx.x == l) own = x[k];
    }
    m = wave_max_nan_skip(m);
    if ((threadIdx.x & (kWave - 1)) == 0) shm[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVlB / kWave; k++) m = __builtin_fmaxf(m, shm[k]);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kEach; k++)
        if (k * kVlB < V) s += k * kVlB + (int)threadIdx.x == l || k * kVlB + (int)threadIdx.x >= V ? 0.0 : (double)exp_sum_term(x[k] - m);
    const double others = vl_wg_sum(s, sh);
    const VlStat st = vl_stat(p, i, m, others, own - m, count, threadIdx.x == 0);
    if (GRAD)
#pragma unroll
        for (int k = 0; k < kEach; k++)
            if (k * kVlB + (int)threadIdx.x < V) z[k * kVlB + threadIdx.x] = vl_entry(x[k], k * kVlB + threadIdx.x, l, st);
}

// The same of long rows, whose chunks are workgroups of their own: first each chunk's maximum and sum, and, by one workgroup behind
// them, the count,
__global__ __launch_bounds__(kVlB) void k_vl_part(VlArgs p) {
    constexpr int kEach = kVlChunk / kVlB;
    __shared__ double sh[kVlB / kWave];
    __shared__ float shm[kVlB / kWave];
    const int64_t r = blockIdx.y, v0 = (int64_t)blockIdx.x * kVlChunk;
    if (r == p.rows) {
        if (blockIdx.x == 0) vl_count<kVlB, true>(p, sh);
        return;
    }
    const int32_t l = p.labels[p.row0 + r];
    if (!vl_counts(l, p.ignore, p.V)) return;
    const float *z = p.z + r * p.ldz;
    float x[kEach], m = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const int64_t v = v0 + k * kVlB + threadIdx.x;
        x[k] = v < p.V ? z[v] : -__builtin_inff();
        m = __builtin_fmaxf(m, x[k]);
        if (v == l) {
            p.label_z[r] = x[k];
            x[k] = -__builtin_inff();
        }
    }
    m = wave_max_nan_skip(m);
    if ((threadIdx.x & (kWave - 1)) == 0) shm[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVlB / kWave; k++) m = __builtin_fmaxf(m, shm[k]);
    double s = 0.0;
    const float base = m == -__builtin_inff() ? 0.0f : m;  // words that are all -inf have no part in the row's sum
#pragma unroll
    for (int k = 0; k < kEach; k++) s += (double)exp_sum_term(x[k] - base);
    s = vl_wg_sum(s, sh);
    if (threadIdx.x == 0) p.part[r * p.chunks + blockIdx.x] = f2{m, (float)s};
}

// then, from those of its row, a chunk of G.
template <bool GRAD>
__global__ __launch_bounds__(kVlB) void k_vl_chunk(VlArgs p) {
    __shared__ double sh[kVlB / kWave];
    __shared__ float shm[kVlB / kWave];
    const int64_t r = blockIdx.y, i = p.row0 + r, v0 = (int64_t)blockIdx.x * kVlChunk;
    const int32_t l = p.labels[i];
    float *z = p.z + r * p.ldz;
    const bool on = vl_counts(l, p.ignore, p.V);
    if (GRAD) vl_clean(p, i, on, blockIdx.x, p.chunks);
    if (!on) {
        if (threadIdx.x == 0 && blockIdx.x == 0) {
            p.row_loss[i] = 0.0;
            if (p.row_out) p.row_out[i] = 0.0f;
        }
        if (GRAD)
            for (int64_t v = v0 + threadIdx.x; v < min(p.V, v0 + kVlChunk); v += kVlB) z[v] = 0.0f;
        return;
    }
    const f2 *part = p.part + r * p.chunks;
    float m = -__builtin_inff();
    for (int k = threadIdx.x; k < p.chunks; k += kVlB) m = __builtin_fmaxf(m, part[k].x);
    m = wave_max_nan_skip(m);
    if ((threadIdx.x & (kWave - 1)) == 0) shm[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVlB / kWave; k++) m = __builtin_fmaxf(m, shm[k]);
    double s = 0.0;
    for (int k = threadIdx.x; k < p.chunks; k += kVlB) s += (double)part[k].y * (double)(part[k].x == m ? 1.0f : exp8_nonpos(part[k].x - m));
    const double others = vl_wg_sum(s, sh);
    const VlStat st = vl_stat(p, i, m, others, p.label_z[r] - m, GRAD && !p.sum ? p.head->count : 0, blockIdx.x == 0 && threadIdx.x == 0);
    if (GRAD)
        for (int64_t v = v0 + threadIdx.x; v < min(p.V, v0 + kVlChunk); v += kVlB) z[v] = vl_entry(z[v], v, l, st);
}

// What is left of a piece, in one launch: gx (+)= the sum of its parts; gb (+)= the column sums of G, 64 columns a workgroup, a quarter
// of the rows in each wave; and at the last the loss, which of no rows is NaN, as a mean over nothing is (a sum: 0).
struct VlTail {
    const float *parts;
    int slices;
    int64_t n;  // words of a part
    float *gx;
    int acc_x;
    unsigned joins, columns;  // workgroups
    const float *g;
    int64_t ldz, rows, V;
    float *gb;
    int acc_b;
    const double *row_loss;
    int64_t N;
    const VlHead *head;
    int sum;
    float *loss;
};

__global__ __launch_bounds__(kVlB) void k_vl_tail(VlTail p) {
    constexpr int kWaves = kVlB / kWave;
    __shared__ double sh[kWaves * kWave];
    if (blockIdx.x < p.joins) {
        for (int64_t i = (int64_t)blockIdx.x * kVlB + threadIdx.x; i < p.n; i += (int64_t)p.joins * kVlB) {
            double s = p.acc_x ? (double)p.gx[i] : 0.0;
#pragma unroll 8
            for (int k = 0; k < p.slices; k++) s += (double)p.parts[k * p.n + i];
            p.gx[i] = (float)s;
        }
    } else if (blockIdx.x - p.joins < p.columns) {
        const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
        const int64_t v = (int64_t)(blockIdx.x - p.joins) * kWave + lane;
        double s = 0.0;
        if (v < p.V)
#pragma unroll 8
            for (int64_t r = wave; r < p.rows; r += kWaves) s += (double)p.g[r * p.ldz + v];
        sh[threadIdx.x] = s;
        __syncthreads();
        if (wave != 0 || v >= p.V) return;
#pragma unroll
        for (int w = 1; w < kWaves; w++) s += sh[w * kWave + lane];
        p.gb[v] = (float)(p.acc_b ? (double)p.gb[v] + s : s);
    } else {
        const double t = vl_wg_sum(vl_lane_sum(p.row_loss, p.N), sh);
        if (threadIdx.x == 0) *p.loss = p.sum ? (float)t : p.head->count ? (float)(t / (double)p.head->count) : __builtin_nanf("");
    }
}

__global__ __launch_bounds__(kVlB) void k_vl_zero(float *__restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * kVlB + threadIdx.x; i < n; i += (int64_t)gridDim.x * kVlB) p[i] = 0.0f;
}

// the workspace: [head][row losses][labels' products][chunks' statistics][x without the rows that do not count][z of a piece][parts of gx]
struct VlPlan {
    int64_t ldz, piece;
    int chunks, slices;
    int64_t slice;  // words of a part of gx
    bool few_x, few_w;  // gx and gW by vocab_few.hip
    size_t losses, label_z, part, rows, z, parts, total;
};

// Whether gx and gW are vocab_few.hip's (rows over words x columns, us without : with): 23 over 54997 x 1712 389 : 283, 8 over 4000 x 1024
// 38 : 31, 23 over 4000 x 256 31 : 31, 1000 x 1024 24 : 31; gW alone, 60 over 54997 x 1712 517 : 440; gx of more than 32 rows takes longer
// (60: 163 : 188).  Rows that are no whole 16 bytes are written at half the rate.
static bool vl_few_pays(int64_t D, int64_t V) { return D % 4 == 0 && D >= 128 && V * D >= int64_t(1) << 21; }

static VlPlan vl_plan(int64_t N, int64_t D, int64_t V, bool want_x, bool want_w) {
    VlPlan p{};
    p.ldz = (V + 15) / 16 * 16;
    const int64_t most = std::max<int64_t>(64, (int64_t)(kVlPiece / 4) / p.ldz / 64 * 64);
    p.piece = std::min(std::min(N, most), vl_piece_rows(kVlRows));
    p.chunks = V > kVlShort ? (int)((V + kVlChunk - 1) / kVlChunk) : 1;
    // gx of few rows: its words in parts, as many as give the chip's CUs two tiles of 64 x 64 each, of at least 512 words
    const int64_t tiles = (p.piece + 63) / 64 * ((D + 63) / 64);
    const int64_t cut = std::max<int64_t>(1, std::min((2 * kPlanCUs + tiles - 1) / std::max<int64_t>(tiles, 1), V / 512));
    const bool few = vl_few_pays(D, V) && p.piece == N;
    p.few_x = few && N <= 32, p.few_w = few && N <= 64;
    p.slice = p.few_x ? vl_few_slice(D, V) : cut > 1 ? ((V + cut - 1) / cut + 31) / 32 * 32 : V;
    p.slices = (int)((V + p.slice - 1) / p.slice);
    p.losses = 256;
    p.label_z = p.losses + vl_round256((size_t)N * 8);
    p.part = p.label_z + vl_round256((size_t)p.piece * 4);
    p.rows = p.part + vl_round256((size_t)p.piece * p.chunks * sizeof(f2));
    p.z = p.rows + (want_w ? vl_round256((size_t)(N * D) * 4) : 0);
    p.parts = p.z + vl_round256((size_t)(p.piece * p.ldz) * 4);
    p.total = p.parts + (want_x && (p.few_x || p.slices > 1) ? (size_t)p.slices * p.piece * D * 4 : 0);
    return p;
}

static const char *vl_size_error(int64_t N, int64_t D, int64_t V) {
    if (N < 0 || N >= int64_t(1) << 31) return "0 to 2^31 - 1 rows";
    if (D < 1 || D > int64_t(1) << 20) return "1 to 2^20 columns";
    if (V < 1 || V > int64_t(1) << 26) return "1 to 2^26 words";
    return nullptr;
}

}  // namespace nchip

using namespace nchip;

extern "C" NC_HIP_API size_t nc_hip_linear_cross_entropy_workspace(int64_t N, int64_t D, int64_t V, int want_x, int want_w, int want_b) {
    if (vl_size_error(N, D, V)) return 0;
    if (vl_split_pays(N, D, V, want_x || want_w || want_b)) return vl_split_workspace(N, D, V, want_x != 0, want_w != 0, want_b != 0);
    return vl_plan(N, D, V, want_x != 0, want_w != 0).total;
}

extern "C" NC_HIP_API int nc_hip_linear_cross_entropy(int64_t N, int64_t D, int64_t V, const float *x, int64_t ldx, const float *w,
                                                      int64_t ldw, const float *bias, const int32_t *labels, int32_t ignore, int sum,
                                                      const float *gout, float *loss, float *row_loss, uint64_t *bad, float *gx,
                                                      float *gw, float *gb, int acc_x, int acc_w, int acc_b, void *ws, size_t ws_bytes,
                                                      void *stream) {
    const char *what = "nc_hip_linear_cross_entropy";
    if (const char *e = vl_size_error(N, D, V)) return set_error(NC_HIP_ERR_ARG, "%s: bad size, %s", what, e);
    if (!loss || !w || (N > 0 && (!x || !labels))) return set_error(NC_HIP_ERR_ARG, "%s: NULL pointer", what);
    if (ldx < D || ldw < D) return set_error(NC_HIP_ERR_ARG, "%s: rows closer than their %lld columns", what, (long long)D);
    if (((uintptr_t)bad & 7u) != 0) return set_error(NC_HIP_ERR_ARG, "%s: bad is not 8-byte aligned", what);
    const size_t need = nc_hip_linear_cross_entropy_workspace(N, D, V, gx != nullptr, gw != nullptr, gb != nullptr);
    if (!ws || ws_bytes < need) return set_error(NC_HIP_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, need);
    if (((uintptr_t)ws & 15u) != 0) return set_error(NC_HIP_ERR_ARG, "%s: the workspace is not 16-byte aligned", what);
    hipStream_t st = as_stream(stream);
    const bool grad = gx || gw || gb;
    if (vl_split_pays(N, D, V, grad))
        return vl_split_run({N, D, V, x, ldx, w, ldw, bias, labels, ignore, sum, gout, loss, row_loss, (unsigned long long *)bad, gx, gw, gb,
                             acc_x, acc_w, acc_b, (char *)ws, st}, what);
    const VlPlan plan = vl_plan(N, D, V, gx != nullptr, gw != nullptr);
    char *base = (char *)ws;
    VlHead *head = (VlHead *)base;
    double *losses = (double *)(base + plan.losses);
    float *clean = (float *)(base + plan.rows), *z = (float *)(base + plan.z), *parts = (float *)(base + plan.parts);
    VlArgs a{};
    a.N = N, a.V = V, a.ldz = plan.ldz, a.chunks = plan.chunks, a.labels = labels, a.ignore = ignore, a.sum = sum;
    a.head = head, a.bad = (unsigned long long *)bad, a.gout = gout, a.x = x, a.ldx = ldx, a.D = D, a.clean = gw ? clean : nullptr;
    a.z = z, a.part = (f2 *)(base + plan.part), a.label_z = (float *)(base + plan.label_z), a.row_loss = losses, a.row_out = row_loss;
    VlTail t{};
    t.parts = parts, t.slices = plan.slices, t.acc_x = acc_x, t.g = z, t.ldz = plan.ldz, t.V = V, t.gb = gb;
    t.row_loss = losses, t.N = N, t.head = head, t.sum = sum, t.loss = loss;
    const bool count_here = N > 0 && (plan.chunks > 1 || N <= kVlCountMost);
    if (!count_here) hipLaunchKernelGGL(k_vl_count, 1, 1024, 0, st, a);
    for (int64_t r0 = 0; r0 < N; r0 += plan.piece) {
        a.row0 = r0, a.rows = std::min(plan.piece, N - r0), a.count_here = count_here && r0 == 0;
        const VlFew few{N, D, V, w, ldw, z, plan.ldz, clean, parts, plan.slice, gw, acc_w};
        int rc = nc_hip_gemm_f32_bias(0, 1, a.rows, V, D, 1.0f, x + r0 * ldx, ldx, w, ldw, bias, z, plan.ldz, stream);
        if (rc) return rc;
        if (plan.chunks > 1) {
            const dim3 grid((unsigned)plan.chunks, (unsigned)a.rows);
            hipLaunchKernelGGL(k_vl_part, dim3(grid.x, grid.y + a.count_here), kVlB, 0, st, a);
            if (grad) hipLaunchKernelGGL(k_vl_chunk<true>, grid, kVlB, 0, st, a);
            else hipLaunchKernelGGL(k_vl_chunk<false>, dim3(1, grid.y), kVlB, 0, st, a);
        } else if (grad) {
            hipLaunchKernelGGL(k_vl_softmax<true>, (unsigned)a.rows, kVlB, 0, st, a);
        } else {
            hipLaunchKernelGGL(k_vl_softmax<false>, (unsigned)a.rows, kVlB, 0, st, a);
        }
        const bool cut = gx && (plan.few_x || plan.slices > 1);
        if (plan.few_x && gx) {
            vl_few_gx(few, st);
        } else if (cut) {
            const int64_t whole = V / plan.slice, rest = V - whole * plan.slice, part = a.rows * D;
            const int64_t shape = whole, sa = plan.slice, sb = plan.slice * ldw;
            rc = nc_hip_gemm_f32_bmm(0, 0, a.rows, D, plan.slice, z, plan.ldz, w, ldw, 0.0f, parts, D, 1, &shape, &sa, &sb, &part, nullptr, 0, stream);
            if (!rc && rest)
                rc = nc_hip_gemm_f32(0, 0, a.rows, D, rest, 1.0f, z + whole * plan.slice, plan.ldz, w + whole * sb, ldw, 0.0f,
                                     parts + whole * part, D, stream);
        } else if (gx) {
            rc = nc_hip_gemm_f32(0, 0, a.rows, D, V, 1.0f, z, plan.ldz, w, ldw, acc_x ? 1.0f : 0.0f, gx + r0 * D, D, stream);
        }
        if (gw && plan.few_w && aligned16(gw)) vl_few_gw(few, st);
        else if (!rc && gw)
            rc = nc_hip_gemm_f32(1, 0, V, D, a.rows, 1.0f, z, plan.ldz, clean + r0 * D, D, acc_w || r0 ? 1.0f : 0.0f, gw, D, stream);
        if (rc) return rc;
        t.rows = a.rows, t.n = a.rows * D, t.gx = cut ? gx + r0 * D : nullptr, t.acc_b = acc_b || r0;
        t.joins = cut ? stream_grid(t.n, kVlB) : 0, t.columns = gb ? (unsigned)((V + kWave - 1) / kWave) : 0;
        const unsigned last = r0 + a.rows == N;
        if (t.joins + t.columns + last) hipLaunchKernelGGL(k_vl_tail, t.joins + t.columns + last, kVlB, 0, st, t);
    }
    if (N == 0) {
        if (gw && !acc_w) hipLaunchKernelGGL(k_vl_zero, stream_grid(V * D, kVlB), kVlB, 0, st, gw, V * D);
        if (gb && !acc_b) hipLaunchKernelGGL(k_vl_zero, stream_grid(V, kVlB), kVlB, 0, st, gb, V);
        hipLaunchKernelGGL(k_vl_tail, 1, kVlB, 0, st, t);
    }
    return check_launch(what);
}
