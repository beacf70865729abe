// Rotary positions of several axes, and the per-head RMS norm of queries and keys with the rotation in the same pass.
//
// A row is one head of one token, D floats.  Its first columns are cut into sections, one per position axis: section a of
// d_a columns holds d_a / 2 pairs, (i, i + d_a / 2) or side by side (2 i, 2 i + 1); pair i is turned by the angle
// pos[token][a] * base^(-2 i / d_a).  The columns past the sections stay.  With the norm the row is first scaled by
// r = 1 / sqrt(mean(x^2) + eps) and by its head's weights.
//
//     forward   n = x r,  h = n w,  (y1, y2) = (h1 c - h2 s, h2 c + h1 s)
//     backward  g = the inverse rotation of gy,  gw += sum over rows of g n,  h = g w,  gx = r (h - n mean(h n))
//
// Both directions are bound by memory (8 and 12 bytes a value).  The cosines and sines of a group of tokens are computed
// once, into LDS, for all of its heads: angles in turns in fp64 (a position of 2^31 keeps 2^-22 of a turn), reduced to an
// eighth of a turn exactly and only then rounded to fp32.  A row is held by 8 to 32 lanes, units of V pairs a lane: V = 4
// where every section's columns fall into whole 16-byte pieces, else up to 8 single pairs.  Lanes keep their unit for all rows, so
// that the weights and the weights' gradients stay in registers.
//
// Measured, beside a copy of 1 GiB at 4.8 TB/s: rotation of [8, 1024, 16, 64], two axes, 13 us each way (5.2 TB/s); of [1, 16384, 32,
// 128], three axes, 96 us (5.6 TB/s); norm and rotation of [4, 2048, 20, 128] 33 us (5.1 TB/s), back 45 us (5.6 TB/s) and 4.6 for
// joining the weights' gradients; of [3, 777, 10, 80] with odd sections, by single pairs, 10 and 15 us, which is latency.
#include "common.hpp"
#include "intdiv.hpp"

#include <math.h>

namespace nchip {

constexpr int kRopeB = 256;
constexpr int kRopeAxes = 4;
constexpr int kRopeD = 256;
constexpr int kRopeTable = 2048;    // (cos, sin) pairs of a token group in LDS, 16 KiB
constexpr int kRopeBlocks = 1024;   // workgroups wanted, and the weights' gradients' partials at most

struct RopeArgs {
    int D, H, q_heads;
    int64_t tokens, L;         // B * L, L
    int64_t sb, sl, sh;        // x's strides
    int axes, inter, batched;  // position axes, pairs side by side, positions for every sequence
    int col0[kRopeAxes + 1], pair0[kRopeAxes + 1];  // first column and pair of each section; [axes]: of the rest
    int group, chunk, chunks;  // tokens of a group, heads a workgroup takes of them, such parts
    int64_t items;             // groups * chunks
    IntDiv heads;              // by the heads of a part
    float eps;
    int acc, acc_wq, acc_wk;
    double turn[kRopeD / 2];   // turns per position of each pair
};

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
    v += dpp_f32<kDppXor1>(v, 0.0f);
    v += dpp_f32<kDppXor2>(v, 0.0f);
    v += dpp_f32<kDppHalfMirror>(v, 0.0f);
    if constexpr (LPR >= 16) v += dpp_f32<kDppMirror>(v, 0.0f);
    if constexpr (LPR >= 32) v += __shfl_xor(v, 16);
    return v;
}

// a lane's unit: V pairs; first table entry (-1: not rotated), columns of its two halves (-1: none)
struct RopeUnit {
    int pair, c1, c2;
};

template <int V>
__device__ __forceinline__ RopeUnit rope_unit(const RopeArgs &a, int u) {
    RopeUnit r = {-1, -1, -1};
    for (int x = 0; x < a.axes; x++) {
        const int half = a.pair0[x + 1] - a.pair0[x], n = half / V;
        if (u < n) {
            r.pair = a.pair0[x] + V * u;
            r.c1 = a.col0[x] + (a.inter ? 2 * V * u : V * u);
            r.c2 = a.inter ? r.c1 + V : r.c1 + half;
            return r;
        }
        u -= n;
    }
    const int c = a.col0[a.axes] + 2 * V * u;
    if (c < a.D) {
        r.c1 = c;
        if (c + V < a.D) r.c2 = c + V;
    }
    return r;
}

template <int V>
__device__ __forceinline__ void rope_get(const float *row, const RopeUnit &u, float *e) {
#pragma unroll
    for (int i = 0; i < 2 * V; i++) e[i] = 0.0f;
    if constexpr (V == 4) {
        f4 p = {0.f, 0.f, 0.f, 0.f}, q = p;
        if (u.c1 >= 0) p = *(const f4u *)(row + u.c1);
        if (u.c2 >= 0) q = *(const f4u *)(row + u.c2);
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = p[i], e[4 + i] = q[i];
    } else {
        if (u.c1 >= 0) e[0] = row[u.c1];
        if (u.c2 >= 0) e[1] = row[u.c2];
    }
}

template <int V>
__device__ __forceinline__ void rope_put(float *row, const RopeUnit &u, const float *e, int acc) {
    float o[2 * V];
    if (acc) {
        rope_get<V>(row, u, o);
#pragma unroll
        for (int i = 0; i < 2 * V; i++) o[i] += e[i];
    } else {
#pragma unroll
        for (int i = 0; i < 2 * V; i++) o[i] = e[i];
    }
    if constexpr (V == 4) {
        if (u.c1 >= 0) *(f4u *)(row + u.c1) = f4{o[0], o[1], o[2], o[3]};
        if (u.c2 >= 0) *(f4u *)(row + u.c2) = f4{o[4], o[5], o[6], o[7]};
    } else {
        if (u.c1 >= 0) row[u.c1] = o[0];
        if (u.c2 >= 0) row[u.c2] = o[1];
    }
}

// the pairs of e turned by the table's angles, backwards where sign is -1
template <int V>
__device__ __forceinline__ void rope_turn(float *e, const float2 *cs, const RopeUnit &u, int inter, float sign) {
    if (u.pair < 0) return;
    auto turn = [&](float2 t, float &p, float &q) {
        const float c = t.x, s = sign * t.y, a = p, b = q;
        p = fma_(a, c, -(b * s));
        q = fma_(b, c, a * s);
    };
    if (inter) {
#pragma unroll
        for (int i = 0; i < V; i++) turn(cs[u.pair + i], e[2 * i], e[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) turn(cs[u.pair + i], e[i], e[V + i]);
    }
}

// rows in flight: about 64 bytes of each tensor a lane
constexpr int rope_rows(int mode, int v, int upl) { return (mode == 2 ? 2 : 4) / (v == 1 && upl > 4 ? 2 : 1); }

// MODE 0: rotation of x (sign 1) or of gy back (sign -1); 1: norm and rotation; 2: their gradient
template <int V, int LPR, int UPL, int MODE>
__global__ __launch_bounds__(kRopeB) void k_rope(const RopeArgs a, const float *__restrict__ x,
                                                 const float *__restrict__ wq, const float *__restrict__ wk,
                                                 const int *__restrict__ pos, const float *__restrict__ gy,
                                                 float *__restrict__ y, double *__restrict__ part, float sign) {
    constexpr int slots = kRopeB / LPR;
    constexpr int U = rope_rows(MODE, V, UPL);  // rows a slot holds at once
    __shared__ float2 table[kRopeTable];
    __shared__ float red[MODE == 2 ? kRopeB * 2 * V : 1];
    const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const int P = a.pair0[a.axes];
    RopeUnit un[UPL];
    float w[2][UPL][2 * V], gw[2][UPL][2 * V];
#pragma unroll
    for (int k = 0; k < UPL; k++) {
        un[k] = rope_unit<V>(a, lane + k * LPR);
        if constexpr (MODE != 0) {
#pragma unroll
            for (int i = 0; i < 2 * V; i++) w[0][k][i] = w[1][k][i] = 1.0f, gw[0][k][i] = gw[1][k][i] = 0.0f;
            if (wq) rope_get<V>(wq, un[k], w[0][k]);
            if (wk) rope_get<V>(wk, un[k], w[1][k]);
        }
    }
    for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t grp = item / a.chunks;
        const int h0 = (int)(item - grp * a.chunks) * a.chunk;
        const int heads = min(a.chunk, a.H - h0);
        const int64_t t0 = grp * a.group;
        const int n = (int)min((int64_t)a.group, a.tokens - t0);
        const int64_t b0 = t0 / a.L;
        const uint32_t l0 = (uint32_t)(t0 - b0 * a.L), L = (uint32_t)a.L;
        const int rows = n * heads;
        for (int r0 = 0; r0 < rows; r0 += slots * U) {  // every lane takes part in the rows' sums
            float e[U][UPL][2 * V], g[MODE == 2 ? U : 1][UPL][2 * V];
            int tok[U], head[U];
#pragma unroll
            for (int k = 0; k < U; k++) {  // all loads first, and before the table
                if (r0 + k * slots >= rows) break;
                const int r = min(r0 + k * slots + slot, rows - 1);
                const int t = heads == a.chunk ? (int)a.heads.div31(r) : r / heads, h = h0 + r - t * heads;
                tok[k] = t, head[k] = h;
                int64_t b = b0;
                uint32_t l = l0 + t;
                if (l >= L) {
                    b += l / L;
                    l %= L;
                }
                const float *xr = x + b * a.sb + (int64_t)l * a.sl + h * a.sh;
#pragma unroll
                for (int i = 0; i < UPL; i++) rope_get<V>(xr, un[i], e[k][i]);
                if constexpr (MODE == 2) {
                    const float *gr = gy + ((t0 + t) * a.H + h) * a.D;
#pragma unroll
                    for (int i = 0; i < UPL; i++) rope_get<V>(gr, un[i], g[k][i]);
                }
            }
            if (r0 == 0) {
                __syncthreads();  // the last group's table has been read
                for (int j = threadIdx.x; j < n * P; j += kRopeB) {
                    const int t = j / P, p = j - t * P;
                    int ax = 0;
                    while (ax + 1 < a.axes && p >= a.pair0[ax + 1]) ax++;
                    const uint32_t l = l0 + t;
                    const int64_t at = a.batched ? t0 + t : (int64_t)(l < L ? l : l % L);
                    const double turns = (double)pos[at * a.axes + ax] * a.turn[p];
                    const double r = turns - rint(turns);   // -1/2 .. 1/2, exact
                    const double quarter = rint(4.0 * r);   // nearest quarter turn
                    float s, c;
                    sincospif((float)(2.0 * (r - 0.25 * quarter)), &s, &c);  // at most an eighth of a turn
                    const int k = (int)quarter & 3;
                    const float cc = k & 1 ? s : c, ss = k & 1 ? c : s;
                    table[j] = float2{k == 1 || k == 2 ? -cc : cc, k >= 2 ? -ss : ss};
                }
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < U; k++) {
                if (r0 + k * slots >= rows) break;
                const bool live = r0 + k * slots + slot < rows;
                float *yr = y + ((t0 + tok[k]) * a.H + head[k]) * a.D;
                const float2 *cs = table + tok[k] * P;
                if constexpr (MODE == 0) {
#pragma unroll
                    for (int i = 0; i < UPL; i++) {
                        rope_turn<V>(e[k][i], cs, un[i], a.inter, sign);
                        if (live) rope_put<V>(yr, un[i], e[k][i], a.acc);
                    }
                } else {
                    const bool key = head[k] >= a.q_heads;
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < UPL; i++)
#pragma unroll
                        for (int c = 0; c < 2 * V; c++) ss = fma_(e[k][i][c], e[k][i][c], ss);
                    const float rn = 1.0f / sqrtf(group_sum<LPR>(ss) / (float)a.D + a.eps);
                    if constexpr (MODE == 1) {
#pragma unroll
                        for (int i = 0; i < UPL; i++) {
#pragma unroll
                            for (int c = 0; c < 2 * V; c++) e[k][i][c] = e[k][i][c] * rn * (key ? w[1][i][c] : w[0][i][c]);
                            rope_turn<V>(e[k][i], cs, un[i], a.inter, 1.0f);
                            if (live) rope_put<V>(yr, un[i], e[k][i], 0);
                        }
                    } else {
                        float dot = 0.0f;
#pragma unroll
                        for (int i = 0; i < UPL; i++) {
                            rope_turn<V>(g[k][i], cs, un[i], a.inter, -1.0f);
#pragma unroll
                            for (int c = 0; c < 2 * V; c++)
                                dot = fma_(g[k][i][c] * (key ? w[1][i][c] : w[0][i][c]), e[k][i][c], dot);
                        }
                        const float m = group_sum<LPR>(dot) * rn / (float)a.D;
#pragma unroll
                        for (int i = 0; i < UPL; i++) {
                            float o[2 * V];
#pragma unroll
                            for (int c = 0; c < 2 * V; c++) {
                                const float nv = e[k][i][c] * rn, term = live ? g[k][i][c] * nv : 0.0f;
                                gw[0][i][c] += key ? 0.0f : term;
                                gw[1][i][c] += key ? term : 0.0f;
                                o[c] = rn * fma_(-nv, m, g[k][i][c] * (key ? w[1][i][c] : w[0][i][c]));
                            }
                            if (live) rope_put<V>(yr, un[i], o, a.acc);
                        }
                    }
                }
            }
        }
    }
    if constexpr (MODE == 2) {
        if (!part) return;
        // the slots' sums in slot order, in fp64: this workgroup's partial [2][D]
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int k = 0; k < UPL; k++) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 2 * V; i++) red[threadIdx.x * 2 * V + i] = gw[q][k][i];
                __syncthreads();
                for (int j = threadIdx.x; j < LPR * 2 * V; j += kRopeB) {
                    const RopeUnit u = rope_unit<V>(a, j / (2 * V) + k * LPR);
                    const int i = j % (2 * V), col = i < V ? u.c1 : u.c2;
                    if (col < 0) continue;
                    double s = 0.0;
                    for (int t = 0; t < slots; t++) s += (double)red[t * LPR * 2 * V + j];
                    part[((int64_t)blockIdx.x * 2 + q) * a.D + col + i % V] = s;
                }
            }
    }
}

// gwq and gwk: the workgroups' partials in a fixed order, 16 columns and 64 runs of partials a workgroup
__global__ __launch_bounds__(1024) void k_rope_weights(const double *__restrict__ part, int n, int D, float *gwq, float *gwk,
                                                       int acc_q, int acc_k) {
    __shared__ double red[64][17];
    const int c = threadIdx.x % 16, run = threadIdx.x / 16, col = blockIdx.x * 16 + c, q = blockIdx.y;
    float *out = q ? gwk : gwq;
    if (!out) return;
    double s = 0.0;
    if (col < D) {
#pragma unroll 8
        for (int i = run; i < n; i += 64) s += part[((int64_t)i * 2 + q) * D + col];
    }
    red[run][c] = s;
    __syncthreads();
    for (int h = 32; h; h /= 2) {
        if (run < h) red[run][c] += red[run + h][c];
        __syncthreads();
    }
    if (run == 0 && col < D) {
        const int acc = q ? acc_k : acc_q;
        out[col] = (acc ? out[col] : 0.0f) + (float)red[0][c];
    }
}

// how a call's rows go to lanes and workgroups
struct RopePlan {
    int v, lpr, upl, group, chunk, chunks;
    int64_t items;
    unsigned blocks;
};

static RopePlan rope_plan(int64_t tokens, int H, int D, int P, bool wide) {
    RopePlan p{};
    p.v = wide ? 4 : 1;
    const int units = (D + 2 * p.v - 1) / (2 * p.v);  // an upper bound: sections end on whole units, the rest on one
    p.lpr = wide ? 8 : 16;
    while (wide && p.lpr < units) p.lpr *= 2;
    p.upl = (units + p.lpr - 1) / p.lpr;
    const int slots = kRopeB / p.lpr;
    // four rounds of rows a group, fewer where the tokens would not make kRopeBlocks groups
    int64_t g = 4 * slots / H;
    if (P && g > kRopeTable / P) g = kRopeTable / P;
    if (g > tokens / kRopeBlocks) g = tokens / kRopeBlocks;
    p.group = (int)(g < 1 ? 1 : g);
    const int64_t groups = (tokens + p.group - 1) / p.group;
    const int rounds = (H + slots - 1) / slots;
    int64_t parts = groups < kRopeBlocks ? kRopeBlocks / groups : 1;
    if (parts > rounds) parts = rounds;
    p.chunk = (int)((rounds + parts - 1) / parts) * slots;
    if (p.chunk > H) p.chunk = H;
    p.chunks = (H + p.chunk - 1) / p.chunk;
    p.items = groups * p.chunks;
    p.blocks = (unsigned)(p.items < (1 << 20) ? p.items : (1 << 20));
    return p;
}

template <int MODE>
static int rope_launch(const RopePlan &p, const RopeArgs &a, const float *x, const float *wq, const float *wk, const int *pos,
                       const float *gy, float *y, double *part, float sign, hipStream_t st, const char *what) {
#define NC_ROPE(V_, LPR_, UPL_) \
    hipLaunchKernelGGL((k_rope<V_, LPR_, UPL_, MODE>), dim3(p.blocks), kRopeB, 0, st, a, x, wq, wk, pos, gy, y, part, sign)
    if (p.v == 4) {
        if (p.lpr == 8) NC_ROPE(4, 8, 1);
        else if (p.lpr == 16) NC_ROPE(4, 16, 1);
        else NC_ROPE(4, 32, 1);
    } else if (p.upl == 1) NC_ROPE(1, 16, 1);
    else if (p.upl == 2) NC_ROPE(1, 16, 2);
    else if (p.upl == 3) NC_ROPE(1, 16, 3);
    else if (p.upl == 4) NC_ROPE(1, 16, 4);
    else NC_ROPE(1, 16, 8);
#undef NC_ROPE
    return check_launch(what);
}

// the arguments all calls share; rows of n x 4 bytes are cut into whole 16-byte pieces where `wide` comes back true
static int rope_args(const char *what, RopeArgs &a, bool &wide, int64_t B, int64_t L, int64_t H, int64_t D, const int64_t *sx,
                     const int32_t *pos, int batched, int n_axes, const int64_t *axis_dims, float base, int inter) {
    if (B < 0 || L < 0 || H < 0 || D < 1 || D > kRopeD)
        return set_error(NC_HIP_ERR_ARG, "%s: bad size (heads of 1 to %d columns)", what, kRopeD);
    if (H > INT32_MAX / 64 || L > INT32_MAX || (L && B > (INT64_MAX >> 24) / L))
        return set_error(NC_HIP_ERR_ARG, "%s: too many heads or tokens", what);
    if (n_axes < 0 || n_axes > kRopeAxes || (n_axes > 0 && (!axis_dims || !pos)))
        return set_error(NC_HIP_ERR_ARG, "%s: 0 to %d position axes, with their columns and positions", what, kRopeAxes);
    if (n_axes > 0 && !(base > 0.0f && isfinite(base)))
        return set_error(NC_HIP_ERR_ARG, "%s: the base must be positive and finite", what);
    a.D = (int)D;
    a.H = (int)H;
    a.tokens = B * L;
    a.L = L;
    a.axes = n_axes;
    a.inter = inter != 0;
    a.batched = batched != 0;
    if (sx) a.sb = sx[0], a.sl = sx[1], a.sh = sx[2];
    int64_t col = 0;
    wide = true;
    for (int x = 0; x < n_axes; x++) {
        const int64_t d = axis_dims[x];
        if (d < 2 || d % 2 || d > D - col)
            return set_error(NC_HIP_ERR_ARG, "%s: axis %d has %lld columns (even, at least 2, %lld left in the head)", what, x,
                             (long long)d, (long long)(D - col));
        a.col0[x] = (int)col;
        a.pair0[x] = (int)(col / 2);
        for (int64_t i = 0; i < d / 2; i++)
            a.turn[col / 2 + i] = pow((double)base, -2.0 * (double)i / (double)d) / (2.0 * M_PI);
        wide = wide && d % 8 == 0;
        col += d;
    }
    a.col0[n_axes] = (int)col;
    a.pair0[n_axes] = (int)(col / 2);
    wide = wide && (D - col) % 4 == 0;
    return NC_HIP_OK;
}

static RopePlan rope_finish(RopeArgs &a, bool wide) {
    const RopePlan p = rope_plan(a.tokens, a.H, a.D, a.pair0[a.axes], wide);
    a.group = p.group;
    a.chunk = p.chunk;
    a.chunks = p.chunks;
    a.items = p.items;
    a.heads = IntDiv((uint32_t)p.chunk);
    return p;
}

static unsigned rope_partials(const RopePlan &p) { return p.blocks < kRopeBlocks ? p.blocks : kRopeBlocks; }

}  // namespace nchip

using namespace nchip;

extern "C" NC_HIP_API int nc_hip_rope_fwd(int64_t B, int64_t L, int64_t H, int64_t D, const float *x, const int64_t *sx,
                                          const int32_t *pos, int pos_batched, int n_axes, const int64_t *axis_dims,
                                          float base, int interleaved, float *y, void *stream) {
    RopeArgs a{};
    bool wide;
    if (const int rc = rope_args("nc_hip_rope_fwd", a, wide, B, L, H, D, sx, pos, pos_batched, n_axes, axis_dims, base, interleaved)) return rc;
    if (a.tokens == 0 || H == 0) return NC_HIP_OK;
    if (n_axes < 1 || !x || !sx || !y) return set_error(NC_HIP_ERR_ARG, "nc_hip_rope_fwd: an axis and x, sx, y are needed");
    const RopePlan p = rope_finish(a, wide);
    return rope_launch<0>(p, a, x, nullptr, nullptr, pos, nullptr, y, nullptr, 1.0f, as_stream(stream), "nc_hip_rope_fwd");
}

extern "C" NC_HIP_API int nc_hip_rope_bwd(int64_t B, int64_t L, int64_t H, int64_t D, const float *gy, const int32_t *pos,
                                          int pos_batched, int n_axes, const int64_t *axis_dims, float base,
                                          int interleaved, float *gx, int accumulate, void *stream) {
    RopeArgs a{};
    bool wide;
    if (const int rc = rope_args("nc_hip_rope_bwd", a, wide, B, L, H, D, nullptr, pos, pos_batched, n_axes, axis_dims, base, interleaved)) return rc;
    if (a.tokens == 0 || H == 0) return NC_HIP_OK;
    if (n_axes < 1 || !gy || !gx) return set_error(NC_HIP_ERR_ARG, "nc_hip_rope_bwd: an axis and gy, gx are needed");
    a.acc = accumulate != 0;
    a.sh = D, a.sl = H * D, a.sb = L * a.sl;
    const RopePlan p = rope_finish(a, wide);
    return rope_launch<0>(p, a, gy, nullptr, nullptr, pos, nullptr, gx, nullptr, -1.0f, as_stream(stream), "nc_hip_rope_bwd");
}

static int norm_args(const char *what, int64_t H, int64_t q_heads, float eps) {
    if (q_heads < 0 || q_heads > H)
        return set_error(NC_HIP_ERR_ARG, "%s: %lld query heads of %lld", what, (long long)q_heads, (long long)H);
    if (!(eps >= 0.0f && isfinite(eps))) return set_error(NC_HIP_ERR_ARG, "%s: eps must be finite and not negative", what);
    return NC_HIP_OK;
}

extern "C" NC_HIP_API int nc_hip_qk_norm_rope_fwd(int64_t B, int64_t L, int64_t H, int64_t D, int64_t q_heads, const float *x,
                                                  const int64_t *sx, const float *wq, const float *wk, float eps,
                                                  const int32_t *pos, int pos_batched, int n_axes,
                                                  const int64_t *axis_dims, float base, int interleaved, float *y,
                                                  void *stream) {
    RopeArgs a{};
    bool wide;
    const char *what = "nc_hip_qk_norm_rope_fwd";
    if (const int rc = rope_args(what, a, wide, B, L, H, D, sx, pos, pos_batched, n_axes, axis_dims, base, interleaved)) return rc;
    if (const int rc = norm_args(what, H, q_heads, eps)) return rc;
    if (a.tokens == 0 || H == 0) return NC_HIP_OK;
    if (!x || !sx || !y) return set_error(NC_HIP_ERR_ARG, "%s: x, sx and y are needed", what);
    a.q_heads = (int)q_heads;
    a.eps = eps;
    const RopePlan p = rope_finish(a, wide);
    return rope_launch<1>(p, a, x, wq, wk, pos, nullptr, y, nullptr, 1.0f, as_stream(stream), what);
}

extern "C" NC_HIP_API size_t nc_hip_qk_norm_rope_bwd_workspace(int64_t B, int64_t L, int64_t H, int64_t D) {
    if (B <= 0 || L <= 0 || H <= 0 || D <= 0) return 0;
    return (size_t)kRopeBlocks * 2 * (size_t)D * sizeof(double);
}

extern "C" NC_HIP_API int nc_hip_qk_norm_rope_bwd(int64_t B, int64_t L, int64_t H, int64_t D, int64_t q_heads, const float *x,
                                                  const int64_t *sx, const float *wq, const float *wk, float eps,
                                                  const int32_t *pos, int pos_batched, int n_axes,
                                                  const int64_t *axis_dims, float base, int interleaved, const float *gy,
                                                  float *gx, float *gwq, float *gwk, int acc_x, int acc_wq, int acc_wk,
                                                  void *ws, size_t ws_bytes, void *stream) {
    RopeArgs a{};
    bool wide;
    const char *what = "nc_hip_qk_norm_rope_bwd";
    if (const int rc = rope_args(what, a, wide, B, L, H, D, sx, pos, pos_batched, n_axes, axis_dims, base, interleaved)) return rc;
    if (const int rc = norm_args(what, H, q_heads, eps)) return rc;
    hipStream_t st = as_stream(stream);
    const bool cols = gwq || gwk, empty = a.tokens == 0 || H == 0;
    if (!empty && (!x || !sx || !gy || !gx)) return set_error(NC_HIP_ERR_ARG, "%s: x, sx, gy and gx are needed", what);
    const size_t need = cols ? nc_hip_qk_norm_rope_bwd_workspace(B, L, H, D) : 0;
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
        return set_error(NC_HIP_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, 16-byte aligned", what, need);
    int n = 0;
    if (!empty) {
        a.q_heads = (int)q_heads;
        a.eps = eps;
        a.acc = acc_x != 0;
        RopePlan p = rope_finish(a, wide);
        n = (int)(p.blocks = rope_partials(p));
        if (const int rc = rope_launch<2>(p, a, x, wq, wk, pos, gy, gx, cols ? (double *)ws : nullptr, 1.0f, st, what)) return rc;
    }
    if (!cols) return NC_HIP_OK;
    hipLaunchKernelGGL(k_rope_weights, dim3((unsigned)((D + 15) / 16), 2), 1024, 0, st, (const double *)ws, n, (int)D, gwq, gwk,
                       acc_wq, acc_wk);
    return check_launch(what);
}
