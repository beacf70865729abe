// Attention to few keys (a padded text, the patches of a small image): a head's keys fit a workgroup, which splits them itself
// instead of reading them packed.  D padded to DP columns, at most 16384 / DP keys forward; one tile of 32 keys a wave, four waves
// or eight, backward.
#include "attention.hpp"
#include "attention_short.hpp"

#include <math.h>

namespace nchip {

// A wave splits 32 rows of `src` (from `row0` on, n in all, `step` floats apart) into a tile in LDS; returns the tile's exponent.
template <int DP>
__device__ __forceinline__ float wave_tile(const float *src, int64_t step, int row0, int n, int D, char *tile) {
    constexpr int PER = DP / 16;  // chunks of a lane
    const int lane = threadIdx.x & 63, half = lane >> 5, r = lane & 31;
    const bool live = row0 + r < n;
    const float *row = src + (live ? row0 + r : 0) * step;
    float x[PER][8], most = 0.0f;
    load_chunks(row, 8 * half, 16, D, x);
#pragma unroll
    for (int k = 0; k < PER; k++) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[k][e] = live ? x[k][e] : 0.0f;
        most = abs_max(x[k], most);
    }
    const int ex = tile_exponent(wave_max_nan_skip(most));
    const float inv = pow2i(-ex);
    char *out = tile + row_at(lane);
#pragma unroll
    for (int k = 0; k < PER; k++) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[k][e] *= inv;
        const Split8 s = split8(x[k]);
        *(h8 *)(out + 1024 * k) = s.hi;
        *(h8 *)(out + 64 * DP + 1024 * k) = s.lo;
    }
    return (float)ex;
}

// Forward: keys and values of a pair stay in LDS, and each wave goes over tiles of queries by itself.
template <int DP, int W, int OCC>
__global__ __launch_bounds__(W *kWave, OCC) void k_attn_short_fwd(const ShortFwd f) {
    constexpr int TB = 128 * DP;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float *const exps = (float *)(smem + 2 * f.tiles * TB);
    for (int64_t w = blockIdx.x; w < f.units; w += gridDim.x) {
        const int64_t pair = w / f.splits, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int split = (int)(w - pair * f.splits);
        const int n = (int)keys_of(a.Lk, f.key_len, b), nt = (n + kTile - 1) / kTile;
        const int64_t t0 = f.qtiles * split / f.splits, t1 = f.qtiles * (split + 1) / f.splits;
        __syncthreads();  // the last unit's keys have been read
        for (int t = wave; t < 2 * nt; t += W) {
            const bool val = t >= nt;
            const int k = val ? t - nt : t;
            const float *src = val ? f.v + b * a.sv[0] + u * a.sv[2] : f.k + b * a.sk[0] + u * a.sk[2];
            const float e = wave_tile<DP>(src, val ? a.sv[1] : a.sk[1], k * kTile, n, (int)a.D, smem + (val ? f.tiles + k : k) * TB);
            if (lane == 0) exps[val ? f.tiles + k : k] = e;
        }
        __syncthreads();
        for (int64_t qt = t0 + wave; qt < t1; qt += W) {
            const int64_t R = qt * kTile + (lane & 31);
            const bool live = R < f.rows;
            int64_t i, g;
            a.row(live ? R : 0, i, g);
            const int64_t h = u * a.G + g;
            Query<DP> q;
            load_query(q, f.q + b * a.sq[0] + i * a.sq[1] + h * a.sq[2], live, a.scale, half, (int)a.D);
            Sums<DP> sum;
            sum.clear();
            const char *kt = smem + row_at(lane), *vt = smem + f.tiles * TB + col_at(lane);
            for (int t = 0; t < nt; t++)
                attend(sum, q, kt + t * TB, vt + t * TB, exps[t], exps[f.tiles + t], t + 1 == nt, min(n - t * kTile, kTile) - 4 * half);
            const float l = halves_sum(sum.l);
            if (live) {
                store_column<false>(f.o + ((b * a.Lq + i) * a.Hq + h) * a.D, sum.o, true, l != 0.0f ? pow2i((int)sum.E) / l : 0.0f, half, (int)a.D, 0);
                if (f.lse && half == 0)
                    f.lse[(b * a.Hq + h) * a.Lq + i] = nt ? fma_(sum.m - kPShift, kLn2, logf(l)) : -INFINITY;
            }
        }
    }
}

// Backward in one pass over the queries: every wave holds 32 keys, the workgroup splits a tile of queries and output gradients
// (the next one's on their way meanwhile), and each wave takes its part of gk and gv as k_attn_dkv does, then turns its ds in LDS
// and multiplies it with its keys; the waves' parts of gq are added in wave order.
template <int DP, int W>
__global__ __launch_bounds__(W *kWave, 2) void k_attn_short_bwd(const ShortBwd f) {
    constexpr int KS = DP / 16, NT = DP / 32, TB = 128 * DP, LO = 64 * DP;
    constexpr int THREADS = W * kWave, UNITS = 4 * DP, PER = (UNITS + THREADS - 1) / THREADS;  // 8-column pieces of a tile
    constexpr int LD = DP + 4, PART = 32 * LD * 4;  // a wave's part of gq: 32 rows, which also holds ds turned, and at first a tile
    constexpr int LDS_DS = 36;
    static_assert(PART >= TB && PART >= 32 * LDS_DS * 4, "a wave's part holds a tile and a turned ds");
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // q's tile, go's tile, the waves' parts, then small tables
    char *const qs = smem, *const gs = smem + TB, *const parts = smem + 2 * TB;
    float *const small = (float *)(parts + W * PART);
    float *const stats = small, *const dots = small + 64, *const red = dots + (DP / 8) * 32;  // [64], [DP / 8][32], [2][W]
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ra = row_at(lane), ca = col_at(lane), D = (int)a.D;
    for (int64_t w = blockIdx.x; w < f.units; w += gridDim.x) {
        const int64_t pair = w / f.splits, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int split = (int)(w - pair * f.splits);
        const int n = (int)keys_of(a.Lk, f.key_len, b), nt = (n + kTile - 1) / kTile;
        const int64_t t0 = f.qtiles * split / f.splits, t1 = f.qtiles * (split + 1) / f.splits;
        // workgroups that share a CU give the first tiles of keys (the only ones of a short sequence) to other waves, so to other SIMDs
        const int kw = (wave + (int)(w >> 8) * (W / 2)) & (W - 1), key = kw * kTile + (lane & 31);
        char *const part = parts + kw * PART;
        const bool mine = kw < nt, live = key < n;

        // the next tile's pieces: piece p is columns 8 (p / 32) .. + 7 of row p % 32
        float nq[PER][8], ng[PER][8], no[PER][8], nl = INFINITY;
        auto fetch = [&](int64_t t) {
#pragma unroll
            for (int k = 0; k < PER; k++) {
                const int p = threadIdx.x + k * THREADS;
                const int64_t R = t * kTile + (p & 31);
                const bool in = p < UNITS && R < f.rows;
                int64_t i, g;
                a.row(in ? R : 0, i, g);
                const int64_t h = u * a.G + g;
                const int64_t at = ((b * a.Lq + i) * a.Hq + h) * D;
                const int d = in ? 8 * (p >> 5) : D;  // nothing is read from column D on
                load8(f.q + b * a.sq[0] + i * a.sq[1] + h * a.sq[2], d, D, nq[k]);
                load8(f.go + at, d, D, ng[k]);
                load8(f.o + at, d, D, no[k]);
                if (k == 0) nl = p < 32 && in ? f.lse[(b * a.Hq + h) * a.Lq + i] * kLog2e : INFINITY;
            }
        };
        __syncthreads();  // the last unit's parts have been read
        if (t0 < t1) fetch(t0);
        h8 kh[KS], kl[KS], vh[KS], vl[KS], ch[2][NT], cl[2][NT];
        float ek = 0.0f, ev = 0.0f;
        if (mine) {  // this wave's keys and values, through its part of LDS
            ek = wave_tile<DP>(f.k + b * a.sk[0] + u * a.sk[2], a.sk[1], kw * kTile, n, D, part);
#pragma unroll
            for (int s = 0; s < KS; s++) kh[s] = row_frag(part + ra, s), kl[s] = row_frag(part + ra + LO, s);
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int t = 0; t < NT; t++) ch[s][t] = col_frag(part + ca, s, t), cl[s][t] = col_frag(part + ca + LO, s, t);
            ev = wave_tile<DP>(f.v + b * a.sv[0] + u * a.sv[2], a.sv[1], kw * kTile, n, D, part);
#pragma unroll
            for (int s = 0; s < KS; s++) vh[s] = row_frag(part + ra, s), vl[s] = row_frag(part + ra + LO, s);
        }
        f16x dk[NT], dv[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) dk[t][r] = dv[t][r] = 0.0f;
        float F = 0x1p100f, E = -1000.0f;
        const float ck = pow2i((int)ek) * a.scale * kLog2e, cv = pow2i((int)ev);
        for (int64_t t = t0; t < t1; t++) {
            // the tile's scales and the rows' go . o
            float mq = 0.0f, mg = 0.0f;
#pragma unroll
            for (int k = 0; k < PER; k++) {
                const int p = threadIdx.x + k * THREADS;
                float dot = 0.0f;
                mq = abs_max(nq[k], mq), mg = abs_max(ng[k], mg);
#pragma unroll
                for (int e = 0; e < 8; e++) dot = fma_(ng[k][e], no[k][e], dot);
                if (p < UNITS) dots[p] = dot;
            }
            mq = wave_max_nan_skip(mq), mg = wave_max_nan_skip(mg);
            if (lane == 0) red[wave] = mq, red[W + wave] = mg;
            __syncthreads();
            mq = red[0], mg = red[W];
#pragma unroll
            for (int x = 1; x < W; x++) mq = __builtin_fmaxf(mq, red[x]), mg = __builtin_fmaxf(mg, red[W + x]);
            const int eq = tile_exponent(mq), eg = tile_exponent(mg);
            const float iq = pow2i(-eq), ig = pow2i(-eg);
#pragma unroll
            for (int k = 0; k < PER; k++) {
                const int p = threadIdx.x + k * THREADS, c = p >> 5;
                if (p >= UNITS) continue;
#pragma unroll
                for (int e = 0; e < 8; e++) nq[k][e] *= iq, ng[k][e] *= ig;
                const int at = 16 * (32 * c + ((p & 31) ^ (4 * (c & 1))));
                const Split8 x = split8(nq[k]), y = split8(ng[k]);
                *(h8 *)(qs + at) = x.hi, *(h8 *)(qs + LO + at) = x.lo;
                *(h8 *)(gs + at) = y.hi, *(h8 *)(gs + LO + at) = y.lo;
            }
            if (threadIdx.x < 32) {
                float d = dots[threadIdx.x];
#pragma unroll
                for (int c = 1; c < DP / 8; c++) d += dots[32 * c + threadIdx.x];
                stats[threadIdx.x] = nl;
                stats[32 + threadIdx.x] = d;
            }
            __syncthreads();
            if (t + 1 < t1) fetch(t + 1);
            if (mine) {
                const char *qt = qs + ra, *gt = gs + ra, *qc = qs + ca, *gc = gs + ca;
                const f4 *rows = (const f4 *)stats + half;
                f16x s, dp;
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = dp[r] = 0.0f;
                steps<2 * KS>([&](int k) { return k % 2 ? Pieces{row_frag(gt, k / 2), row_frag(gt + LO, k / 2)} : Pieces{row_frag(qt, k / 2), row_frag(qt + LO, k / 2)}; },
                              [&](int k, const Pieces &x) {
                                  if (k % 2) dp = mfma3(x.hi, x.lo, vh[k / 2], vl[k / 2], dp);
                                  else s = mfma3(x.hi, x.lo, kh[k / 2], kl[k / 2], s);
                              });
                const float ex = (float)eg;
                if (ex > E) {
                    scale_acc(dv, __builtin_amdgcn_exp2f(E - ex));
                    E = ex;
                }
                const float sh = 14.0f + __builtin_fmaxf(ex - E, -60.0f), base = live ? sh : -INFINITY;
                const float c = ck * pow2i(eq), c2 = cv * pow2i(eg);
                float most = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f4 ls = rows[2 * j], de = rows[8 + 2 * j];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = 4 * j + e;
                        s[r] = __builtin_amdgcn_exp2f(fma_(s[r], c, base - ls[e]));
                        dp[r] = s[r] * fma_(dp[r], c2, -de[e]);
                        most = __builtin_fmaxf(most, __builtin_fabsf(dp[r]));
                    }
                }
                // ds, 2^-sh times: for gq as it is, one row of queries after another
                float *turned = (float *)part + (lane & 31);
#pragma unroll
                for (int r = 0; r < 16; r++) turned[(8 * (r / 4) + 4 * half + r % 4) * LDS_DS] = dp[r];
                const float kap = __builtin_amdgcn_exp2f((float)eq - sh);
                float by;
                if (column_scale(halves_max(most) * kap, F, by)) scale_acc(dk, by);
                const float kF = kap * F;
#pragma unroll
                for (int r = 0; r < 16; r++) dp[r] *= kF;
                const Split8 ps[2] = {split_regs(s, 0), split_regs(s, 8)}, ds[2] = {split_regs(dp, 0), split_regs(dp, 8)};
                // steps of 2 NT: go's fragment (s, t), then q's
                steps<4 * NT>([&](int k) {
                                  const char *c = k % 2 ? qc : gc;
                                  return Pieces{col_frag(c, k / 2 / NT, k / 2 % NT), col_frag(c + LO, k / 2 / NT, k / 2 % NT)};
                              },
                              [&](int k, const Pieces &x) {
                                  const int r = k / 2 / NT, d = k / 2 % NT;
                                  if (k % 2) dk[d] = mfma3(x.hi, x.lo, ds[r].hi, ds[r].lo, dk[d]);
                                  else dv[d] = mfma3(x.hi, x.lo, ps[r].hi, ps[r].lo, dv[d]);
                              });
                // gq^T of this wave's keys: k^T ds^T, a lane a row of queries
                float x[2][8], top = 0.0f;
                const float *row = (const float *)part + (lane & 31) * LDS_DS + 4 * half;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const f4 lo = *(const f4 *)(row + 16 * k), hi = *(const f4 *)(row + 16 * k + 8);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[k][e] = lo[e], x[k][4 + e] = hi[e];
                        top = __builtin_fmaxf(top, __builtin_fmaxf(__builtin_fabsf(lo[e]), __builtin_fabsf(hi[e])));
                    }
                }
                float Fq = 0x1p100f, by_q;
                column_scale(halves_max(top), Fq, by_q);
                f16x dq[NT];
#pragma unroll
                for (int d = 0; d < NT; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++) dq[d][r] = 0.0f;
#pragma unroll
                for (int k = 0; k < 2; k++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[k][e] *= Fq;
                    const Split8 y = split8(x[k]);
#pragma unroll
                    for (int d = 0; d < NT; d++) dq[d] = mfma3(ch[k][d], cl[k][d], y.hi, y.lo, dq[d]);
                }
                const float back = __builtin_amdgcn_exp2f(ek - sh) / Fq * a.scale;
                float *mypart = (float *)part + (lane & 31) * LD + 4 * half;
#pragma unroll
                for (int d = 0; d < NT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        *(f4 *)(mypart + 32 * d + 8 * j) = f4{dq[d][4 * j] * back, dq[d][4 * j + 1] * back, dq[d][4 * j + 2] * back, dq[d][4 * j + 3] * back};
            }
            __syncthreads();
            if (f.gq) {
                for (int p = threadIdx.x; p < 32 * DP / 4; p += THREADS) {
                    const int r = p / (DP / 4), d = 4 * (p - r * (DP / 4));
                    const int64_t R = t * kTile + r;
                    if (R >= f.rows || d >= D) continue;
                    f4 sum = {0.f, 0.f, 0.f, 0.f};
                    for (int x = 0; x < nt; x++) sum += *(const f4 *)((const float *)(parts + x * PART) + r * LD + d);
                    int64_t i, g;
                    a.row(R, i, g);
                    const int64_t h = u * a.G + g;
                    store4(f.gq + ((b * a.Lq + i) * a.Hq + h) * D, d, D, sum, f.acc_q);
                }
            }
        }
        if (key < a.Lk) {
            const int64_t at = ((b * a.Lk + key) * a.Hkv + u) * D;
            const bool some = live && t0 < t1;
            if (f.gk) store_column<true>(f.gk + split * f.part_k + at, dk, some, a.scale / F, half, D, f.acc_k);
            if (f.gv) store_column<true>(f.gv + split * f.part_k + at, dv, some, __builtin_amdgcn_exp2f(E - 14.0f), half, D, f.acc_v);
        }
    }
}

int short_keys_fwd(int DP) { return DP <= 128 ? 16384 / DP : -1; }
int short_keys_bwd(int DP) { return DP <= 64 ? 256 : -1; }

template <class F, class A>
static void launch(F *kernel, int64_t units, int threads, size_t lds, hipStream_t st, const A &args) {
    if (lds > 65536) (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(units < kAttnGrid ? units : kAttnGrid)), dim3(threads), lds, st, args);
}

void short_fwd(const ShortFwd &f, int DP, hipStream_t st) {
    const size_t lds = (size_t)f.tiles * 2 * tile_bytes(DP) + 2 * f.tiles * sizeof(float);
    if (DP == 32) launch(&k_attn_short_fwd<32, 8, 4>, f.units, 512, lds, st, f);
    else if (DP == 64) launch(&k_attn_short_fwd<64, 8, 2>, f.units, 512, lds, st, f);
    else if (DP == 96) launch(&k_attn_short_fwd<96, 8, 2>, f.units, 512, lds, st, f);
    else launch(&k_attn_short_fwd<128, 8, 2>, f.units, 512, lds, st, f);
}

template <int DP, int W>
static void bwd_launch(const ShortBwd &f, hipStream_t st) {
    const size_t lds = 2 * 128 * DP + (size_t)W * 32 * (DP + 4) * 4 + (64 + DP / 8 * 32 + 2 * W) * sizeof(float);
    launch(&k_attn_short_bwd<DP, W>, f.units, W * kWave, lds, st, f);
}

void short_bwd(const ShortBwd &f, int DP, hipStream_t st) {
    const bool four = f.a.Lk <= 4 * kTile;
    if (DP == 32) four ? bwd_launch<32, 4>(f, st) : bwd_launch<32, 8>(f, st);
    else four ? bwd_launch<64, 4>(f, st) : bwd_launch<64, 8>(f, st);
}

}  // namespace nchip
