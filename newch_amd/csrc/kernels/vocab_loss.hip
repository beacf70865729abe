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

struct VlArgs {
    int64_t N, V, ldz;
    int64_t row0, rows;  // the rows of this piece
    const int32_t *labels;
    int32_t ignore;
    int sum;
    const VlHead *head;
    const float *gout;
    float *z;         // [rows][ldz]: the products, then G
    double *row_loss;  // [N]
    float *row_out;   // [N] or none
};

// rows that count, and the first label that is neither a word nor `ignore`, as (row << 32) | label, or all ones
__global__ __launch_bounds__(1024) void k_vl_count(const int32_t *__restrict__ labels, int64_t N, int64_t V, int32_t ignore, VlHead *head,
                                                   unsigned long long *bad) {
    __shared__ unsigned long long shk[1024 / kWave];
    __shared__ double shn[1024 / kWave];
    unsigned long long k = ~0ull;
    double n = 0.0;
    for (int64_t i = threadIdx.x; i < N; i += 1024) {
        const int32_t l = labels[i];
        if (l == ignore) continue;
        if (l >= 0 && l < V) n += 1.0;
        else if (k == ~0ull) k = ((unsigned long long)i << 32) | (uint32_t)l;
    }
    k = wave_min_u64(k);
    n = wave_sum(n);
    if ((threadIdx.x & (kWave - 1)) == 0) shk[threadIdx.x / kWave] = k, shn[threadIdx.x / kWave] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 1024 / kWave; i++) {
            k = shk[i] < k ? shk[i] : k;
            n += shn[i];
        }
        head->count = (int64_t)n;
        // at system scope: *bad may be host memory that the host watches while the kernel runs
        if (bad) __hip_atomic_store(bad, k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
}

// x with zeros for the rows that do not count
__global__ __launch_bounds__(kVlB) void k_vl_rows(const float *__restrict__ x, int64_t ldx, const int32_t *__restrict__ labels, int32_t ignore,
                                                  int64_t N, int64_t D, int64_t V, float *__restrict__ out) {
    for (int64_t i = blockIdx.x; i < N; i += gridDim.x) {
        const bool on = vl_counts(labels[i], ignore, V);
        for (int64_t d = threadIdx.x; d < D; d += kVlB) out[i * D + d] = on ? x[i * ldx + d] : 0.0f;
    }
}

// A workgroup's row: its statistics, its loss, and, GRAD, its row of G in place of z.
template <bool GRAD>
__global__ __launch_bounds__(kVlB) void k_vl_softmax(VlArgs p) {
    __shared__ double sh[kVlB / kWave];
    __shared__ float shm[kVlB / kWave];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const int64_t i = p.row0 + r;
        float *z = p.z + r * p.ldz;
        const int32_t l = p.labels[i];
        if (!vl_counts(l, p.ignore, p.V)) {
            if (threadIdx.x == 0) {
                p.row_loss[i] = 0.0;
                if (p.row_out) p.row_out[i] = 0.0f;
            }
            if (GRAD)
                for (int64_t v = threadIdx.x; v < p.V; v += kVlB) z[v] = 0.0f;
            continue;
        }
        float m = -__builtin_inff();
        for (int64_t v = threadIdx.x; v < p.V; v += kVlB) m = __builtin_fmaxf(m, z[v]);
        m = wave_max_nan_skip(m);
        __syncthreads();
        if ((threadIdx.x & (kWave - 1)) == 0) shm[threadIdx.x / kWave] = m;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kVlB / kWave; k++) m = __builtin_fmaxf(m, shm[k]);
        double s = 0.0;
        for (int64_t v = threadIdx.x; v < p.V; v += kVlB) s += v == l ? 0.0 : (double)exp_sum_term(z[v] - m);
        const double others = vl_wg_sum(s, sh);
        const float zl = z[l] - m;
        const double own = (double)exp8_nonpos(zl), total = others + own;
        const double ls = zl == 0.0f ? log1p(others) : log(total);
        if (threadIdx.x == 0) {
            const double loss = ls - (double)zl;
            p.row_loss[i] = loss;
            if (p.row_out) p.row_out[i] = (float)loss;
        }
        if (GRAD) {
            float c = p.gout ? *p.gout : 1.0f;
            if (!p.sum) c = c / (float)p.head->count;
            const float g_own = (float)(-others / total), lf = (float)ls;
            __syncthreads();  // z[l] has been read
            for (int64_t v = threadIdx.x; v < p.V; v += kVlB) z[v] = (v == l ? g_own : exp8_nonpos((z[v] - m) - lf)) * c;
        }
    }
}

// gb (+)= column sums of G, rows in order
__global__ __launch_bounds__(kVlB) void k_vl_columns(const float *__restrict__ g, int64_t ldz, int64_t rows, int64_t V, float *gb, int acc) {
    const int64_t v = (int64_t)blockIdx.x * kVlB + threadIdx.x;
    if (v >= V) return;
    double s = acc ? (double)gb[v] : 0.0;
    for (int64_t r = 0; r < rows; r++) s += (double)g[r * ldz + v];
    gb[v] = (float)s;
}

// the loss of no rows is NaN, as a mean over nothing is (a sum: 0)
__global__ __launch_bounds__(kVlB) void k_vl_finish(const double *__restrict__ row_loss, int64_t N, const VlHead *__restrict__ head, int sum,
                                                    float *__restrict__ loss) {
    __shared__ double sh[kVlB / kWave];
    double t = 0.0;
    for (int64_t i = threadIdx.x; i < N; i += kVlB) t += row_loss[i];
    t = vl_wg_sum(t, sh);
    if (threadIdx.x == 0) *loss = sum ? (float)t : head->count ? (float)(t / (double)head->count) : __builtin_nanf("");
}

__global__ __launch_bounds__(kVlB) void k_vl_zero(float *__restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * kVlB + threadIdx.x; i < n; i += (int64_t)gridDim.x * kVlB) p[i] = 0.0f;
}

// the workspace: [head][row losses][x without the rows that do not count][z of a piece]
struct VlPlan {
    int64_t ldz, piece;
    size_t losses, rows, z, total;
};

static VlPlan vl_plan(int64_t N, int64_t D, int64_t V, bool want_w) {
    VlPlan p{};
    p.ldz = (V + 15) / 16 * 16;
    const int64_t most = std::max<int64_t>(64, (int64_t)(kVlPiece / 4) / p.ldz / 64 * 64);
    p.piece = std::min(N, most);
    p.losses = 256;
    p.rows = p.losses + vl_round256((size_t)N * 8);
    p.z = p.rows + (want_w ? vl_round256((size_t)(N * D) * 4) : 0);
    p.total = p.z + (size_t)(p.piece * p.ldz) * 4;
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
    return vl_plan(N, D, V, want_w != 0).total;
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
    const VlPlan plan = vl_plan(N, D, V, gw != nullptr);
    char *base = (char *)ws;
    VlHead *head = (VlHead *)base;
    double *losses = (double *)(base + plan.losses);
    float *clean = (float *)(base + plan.rows), *z = (float *)(base + plan.z);
    hipLaunchKernelGGL(k_vl_count, 1, 1024, 0, st, labels, N, V, ignore, head, (unsigned long long *)bad);
    if (N > 0 && gw) hipLaunchKernelGGL(k_vl_rows, (unsigned)std::min<int64_t>(N, 1 << 16), kVlB, 0, st, x, ldx, labels, ignore, N, D, V, clean);
    for (int64_t r0 = 0; r0 < N; r0 += plan.piece) {
        VlArgs a{N, V, plan.ldz, r0, std::min(plan.piece, N - r0), labels, ignore, sum, head, gout, z, losses, row_loss};
        int rc = nc_hip_gemm_f32_bias(0, 1, a.rows, V, D, 1.0f, x + r0 * ldx, ldx, w, ldw, bias, z, plan.ldz, stream);
        if (rc) return rc;
        const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 1 << 16);
        if (grad) hipLaunchKernelGGL(k_vl_softmax<true>, grid, kVlB, 0, st, a);
        else hipLaunchKernelGGL(k_vl_softmax<false>, grid, kVlB, 0, st, a);
        if (gx) rc = nc_hip_gemm_f32(0, 0, a.rows, D, V, 1.0f, z, plan.ldz, w, ldw, acc_x ? 1.0f : 0.0f, gx + r0 * D, D, stream);
        if (!rc && gw)
            rc = nc_hip_gemm_f32(1, 0, V, D, a.rows, 1.0f, z, plan.ldz, clean + r0 * D, D, acc_w || r0 ? 1.0f : 0.0f, gw, D, stream);
        if (rc) return rc;
        if (gb) hipLaunchKernelGGL(k_vl_columns, (unsigned)((V + kVlB - 1) / kVlB), kVlB, 0, st, z, plan.ldz, a.rows, V, gb, acc_b || r0);
    }
    if (N == 0) {
        if (gw && !acc_w) hipLaunchKernelGGL(k_vl_zero, stream_grid(V * D, kVlB), kVlB, 0, st, gw, V * D);
        if (gb && !acc_b) hipLaunchKernelGGL(k_vl_zero, stream_grid(V, kVlB), kVlB, 0, st, gb, V);
    }
    hipLaunchKernelGGL(k_vl_finish, 1, kVlB, 0, st, losses, N, head, sum, loss);
    return check_launch(what);
}
