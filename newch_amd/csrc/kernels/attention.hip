// Attention of queries to keys and values of another length (cross attention; self attention without a mask is the case of
// equal lengths), forward and backward.  q [B, Lq, Hq, D], k and v [B, Lk, Hkv, D], any strides with unit columns; query head
// h reads the keys of head h / (Hq / Hkv); key_len [B] (or none) cuts each sequence's keys.
//
//     s = scale q . k,  p = softmax(s) over the sequence's keys,  o = p v,  lse = log sum exp(s)
//     dp = go . v,  ds = p (dp - go . o) scale,  gq = ds k,  gk = ds^T q,  gv = p^T go
//
// A sequence without keys gives o = 0, lse = -inf and no gradient.  Keys and values past a sequence's length are not read.
#include "common.hpp"

#include <math.h>

namespace nchip {

constexpr int kAttnD = 256;
constexpr int kAttnB = 256;

struct AttnArgs {
    int64_t B, Lq, Lk, Hq, Hkv, D, G;  // G: query heads of a key head
    int64_t sq[3], sk[3], sv[3];
    float scale;
};

__device__ __forceinline__ int64_t attn_keys(const AttnArgs &a, const int *key_len, int64_t b) {
    if (!key_len) return a.Lk;
    const int64_t n = key_len[b];
    return n < 0 ? 0 : n < a.Lk ? n : a.Lk;
}

__device__ __forceinline__ float dot_row(const float *a, const float *b, int D) {
    float s = 0.0f;
    for (int d = 0; d < D; d++) s = fma_(a[d], b[d], s);
    return s;
}

// value of all the workgroup's lanes
__device__ __forceinline__ float wg_reduce(float v, float *red, bool max) {
    v = max ? wave_max_nan_skip(v) : wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return max ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
}

// a workgroup a query row, a lane a key
__global__ __launch_bounds__(kAttnB) void k_attn_fwd_row(AttnArgs a, const float *q, const float *k, const float *v,
                                                         const int *key_len, float *o, float *lse) {
    __shared__ float qs[kAttnD], ps[kAttnB], red[4];
    const int64_t rows = a.B * a.Lq * a.Hq;
    const int t = threadIdx.x, D = (int)a.D;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int64_t h = r % a.Hq, i = r / a.Hq % a.Lq, b = r / a.Hq / a.Lq, u = h / a.G, n = attn_keys(a, key_len, b);
        const float *kb = k + b * a.sk[0] + u * a.sk[2], *vb = v + b * a.sv[0] + u * a.sv[2];
        __syncthreads();
        if (t < D) qs[t] = q[b * a.sq[0] + i * a.sq[1] + h * a.sq[2] + t];
        float m = -INFINITY, l = 0.0f, acc = 0.0f;
        for (int64_t j0 = 0; j0 < n; j0 += kAttnB) {
            const int c = (int)min((int64_t)kAttnB, n - j0);
            __syncthreads();
            const float s = t < c ? a.scale * dot_row(qs, kb + (j0 + t) * a.sk[1], D) : -INFINITY;
            const float mn = fmaxf(m, wg_reduce(s, red, true));
            const float p = t < c ? (mn == -INFINITY ? 0.0f : expf(s - mn)) : 0.0f;
            const float w = m == mn ? 1.0f : expf(m - mn);
            ps[t] = p;
            l = l * w + wg_reduce(p, red, false);
            acc *= w;
            m = mn;
            if (t < D)
                for (int j = 0; j < c; j++) acc = fma_(ps[j], vb[(j0 + j) * a.sv[1] + t], acc);
        }
        if (t < D) o[r * D + t] = n ? acc / l : 0.0f;
        if (lse && t == 0) lse[(b * a.Hq + h) * a.Lq + i] = n ? m + logf(l) : -INFINITY;
    }
}

__global__ __launch_bounds__(kAttnB) void k_attn_dq_row(AttnArgs a, const float *q, const float *k, const float *v,
                                                        const int *key_len, const float *o, const float *lse, const float *go,
                                                        float *gq, int acc_q) {
    __shared__ float qs[kAttnD], gs[kAttnD], ps[kAttnB], red[4];
    const int64_t rows = a.B * a.Lq * a.Hq;
    const int t = threadIdx.x, D = (int)a.D;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int64_t h = r % a.Hq, i = r / a.Hq % a.Lq, b = r / a.Hq / a.Lq, u = h / a.G, n = attn_keys(a, key_len, b);
        const float *kb = k + b * a.sk[0] + u * a.sk[2], *vb = v + b * a.sv[0] + u * a.sv[2];
        __syncthreads();
        if (t < D) qs[t] = q[b * a.sq[0] + i * a.sq[1] + h * a.sq[2] + t], gs[t] = go[r * D + t];
        const float delta = wg_reduce(t < D ? go[r * D + t] * o[r * D + t] : 0.0f, red, false);
        const float ls = lse[(b * a.Hq + h) * a.Lq + i];
        float acc = 0.0f;
        for (int64_t j0 = 0; j0 < n; j0 += kAttnB) {
            const int c = (int)min((int64_t)kAttnB, n - j0);
            __syncthreads();
            if (t < c) {
                const float p = expf(a.scale * dot_row(qs, kb + (j0 + t) * a.sk[1], D) - ls);
                ps[t] = p * (dot_row(gs, vb + (j0 + t) * a.sv[1], D) - delta) * a.scale;
            }
            __syncthreads();
            if (t < D)
                for (int j = 0; j < c; j++) acc = fma_(ps[j], kb[(j0 + j) * a.sk[1] + t], acc);
        }
        if (t < D) gq[r * D + t] = (acc_q ? gq[r * D + t] : 0.0f) + acc;
    }
}

// a workgroup a key, a lane a query row
__global__ __launch_bounds__(kAttnB) void k_attn_dkv_row(AttnArgs a, const float *q, const float *k, const float *v,
                                                         const int *key_len, const float *o, const float *lse,
                                                         const float *go, float *gk, float *gv, int acc_k, int acc_v) {
    __shared__ float ks[kAttnD], vs[kAttnD], ps[kAttnB], ds[kAttnB];
    const int64_t rows = a.B * a.Lk * a.Hkv, nq = a.G * a.Lq;
    const int t = threadIdx.x, D = (int)a.D;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int64_t u = r % a.Hkv, j = r / a.Hkv % a.Lk, b = r / a.Hkv / a.Lk, n = attn_keys(a, key_len, b);
        __syncthreads();
        float sk = 0.0f, sv = 0.0f;
        if (j < n) {
            if (t < D) ks[t] = k[b * a.sk[0] + j * a.sk[1] + u * a.sk[2] + t], vs[t] = v[b * a.sv[0] + j * a.sv[1] + u * a.sv[2] + t];
            for (int64_t i0 = 0; i0 < nq; i0 += kAttnB) {
                const int c = (int)min((int64_t)kAttnB, nq - i0);
                __syncthreads();
                if (t < c) {
                    const int64_t i = (i0 + t) / a.G, h = u * a.G + (i0 + t) % a.G;
                    const float *gr = go + ((b * a.Lq + i) * a.Hq + h) * D, *orow = o + ((b * a.Lq + i) * a.Hq + h) * D;
                    const float p = expf(a.scale * dot_row(ks, q + b * a.sq[0] + i * a.sq[1] + h * a.sq[2], D) - lse[(b * a.Hq + h) * a.Lq + i]);
                    ps[t] = p;
                    ds[t] = p * (dot_row(vs, gr, D) - dot_row(gr, orow, D)) * a.scale;
                }
                __syncthreads();
                if (t < D)
                    for (int x = 0; x < c; x++) {
                        const int64_t i = (i0 + x) / a.G, h = u * a.G + (i0 + x) % a.G;
                        sv = fma_(ps[x], go[((b * a.Lq + i) * a.Hq + h) * D + t], sv);
                        sk = fma_(ds[x], q[b * a.sq[0] + i * a.sq[1] + h * a.sq[2] + t], sk);
                    }
            }
        }
        if (t < D) {
            if (gk) gk[r * D + t] = (acc_k ? gk[r * D + t] : 0.0f) + sk;
            if (gv) gv[r * D + t] = (acc_v ? gv[r * D + t] : 0.0f) + sv;
        }
    }
}

static int attn_args(const char *what, AttnArgs &a, int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv, int64_t D,
                     float scale, const int64_t *sq, const int64_t *sk, const int64_t *sv) {
    if (B < 0 || Lq < 0 || Lk < 0 || Hq < 1 || Hkv < 1 || D < 1 || D > kAttnD)
        return set_error(NC_HIP_ERR_ARG, "%s: bad size (heads of 1 to %d columns)", what, kAttnD);
    if (Hq % Hkv) return set_error(NC_HIP_ERR_ARG, "%s: %lld query heads cannot share %lld heads of keys", what, (long long)Hq, (long long)Hkv);
    if (Lq > INT32_MAX || Lk > INT32_MAX || Hq > INT32_MAX || B > INT32_MAX) return set_error(NC_HIP_ERR_ARG, "%s: sizes past 2^31", what);
    if (!isfinite(scale)) return set_error(NC_HIP_ERR_ARG, "%s: the scale must be finite", what);
    if (!sq || !sk || !sv) return set_error(NC_HIP_ERR_ARG, "%s: strides are needed", what);
    a = {B, Lq, Lk, Hq, Hkv, D, Hq / Hkv, {sq[0], sq[1], sq[2]}, {sk[0], sk[1], sk[2]}, {sv[0], sv[1], sv[2]}, scale};
    return NC_HIP_OK;
}

static unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

}  // namespace nchip

using namespace nchip;

extern "C" NC_HIP_API size_t nc_hip_cross_attention_fwd_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv,
                                                                  int64_t D) {
    (void)B, (void)Lq, (void)Lk, (void)Hq, (void)Hkv, (void)D;
    return 0;
}

extern "C" NC_HIP_API int nc_hip_cross_attention_fwd(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv, int64_t D,
                                                     float scale, const float *q, const int64_t *sq, const float *k,
                                                     const int64_t *sk, const float *v, const int64_t *sv,
                                                     const int32_t *key_len, float *o, float *lse, void *ws,
                                                     size_t ws_bytes, void *stream) {
    const char *what = "nc_hip_cross_attention_fwd";
    AttnArgs a;
    if (const int rc = attn_args(what, a, B, Lq, Lk, Hq, Hkv, D, scale, sq, sk, sv)) return rc;
    if (B == 0 || Lq == 0) return NC_HIP_OK;
    if (!q || !o || (Lk && (!k || !v))) return set_error(NC_HIP_ERR_ARG, "%s: q, k, v and o are needed", what);
    (void)ws, (void)ws_bytes;
    hipLaunchKernelGGL(k_attn_fwd_row, dim3(row_grid(B * Lq * Hq)), kAttnB, 0, as_stream(stream), a, q, k, v, key_len, o, lse);
    return check_launch(what);
}

extern "C" NC_HIP_API size_t nc_hip_cross_attention_bwd_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv,
                                                                  int64_t D) {
    (void)B, (void)Lq, (void)Lk, (void)Hq, (void)Hkv, (void)D;
    return 0;
}

extern "C" NC_HIP_API int nc_hip_cross_attention_bwd(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv, int64_t D,
                                                     float scale, const float *q, const int64_t *sq, const float *k,
                                                     const int64_t *sk, const float *v, const int64_t *sv,
                                                     const int32_t *key_len, const float *o, const float *lse,
                                                     const float *go, float *gq, float *gk, float *gv, int acc_q, int acc_k,
                                                     int acc_v, void *ws, size_t ws_bytes, void *stream) {
    const char *what = "nc_hip_cross_attention_bwd";
    AttnArgs a;
    if (const int rc = attn_args(what, a, B, Lq, Lk, Hq, Hkv, D, scale, sq, sk, sv)) return rc;
    if (B == 0) return NC_HIP_OK;
    if ((Lq && (!q || !o || !lse || !go)) || (Lk && (!k || !v)))
        return set_error(NC_HIP_ERR_ARG, "%s: q, k, v, o, lse and go are needed", what);
    (void)ws, (void)ws_bytes;
    hipStream_t st = as_stream(stream);
    if (gq && Lq) hipLaunchKernelGGL(k_attn_dq_row, dim3(row_grid(B * Lq * Hq)), kAttnB, 0, st, a, q, k, v, key_len, o, lse, go, gq, acc_q);
    if ((gk || gv) && Lk)
        hipLaunchKernelGGL(k_attn_dkv_row, dim3(row_grid(B * Lk * Hkv)), kAttnB, 0, st, a, q, k, v, key_len, o, lse, go, gk, gv, acc_k, acc_v);
    return check_launch(what);
}
