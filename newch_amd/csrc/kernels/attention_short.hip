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

// Forward: keys and values of a pair stay in LDS, and each wave goes over tiles of queries by itself.  4096 x at most 77, 4 x 16
// heads of 64: 43 to 46 us for 136 MB (3.1 TB/s) -- a wave reads its rows, multiplies and stores in turn, and two waves a SIMD
// do not cover all of it.
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

// A lane's place in a packed tile for fragments of the 16x16x32 product whose rows are summed over: 16 lanes take rows 8 (l / 16)
// .. + 3 and, at the place ^ 64, the next four, of 16 columns (tile t: + 1024 t), without bank conflicts.
__device__ __forceinline__ int turned_at(int lane) {
    const int i = lane & 15, odd = (i >> 1) & 1;
    return 512 * odd + 16 * ((8 * (lane >> 4) + i / 4) ^ (4 * odd)) + 8 * (i & 1);
}
__device__ __forceinline__ h8 turned16(const char *first, const char *second) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)first);
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)second);
    return __builtin_bit_cast(h8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

constexpr int kDsTile = 4096;  // bytes of a packed tile of 32 columns

// Backward in one pass over the queries: every wave holds 32 keys, the workgroup splits a tile of queries and output gradients
// (the next one's on their way meanwhile), and each wave takes its part of gk and gv as k_attn_dkv does.  It leaves its ds in LDS,
// and the waves share the blocks of gq^T = k^T ds^T over all keys.  The same sizes: 100 to 105 us, and 120 to 125 with every
// wave's part of gq added in LDS; memory would take 57.  A tile's steps follow each other (read, split, scores, gradients, store), two
// workgroups a CU, by the registers, and heads of more than 64 columns do not fit them.
template <int DP, int W>
__global__ __launch_bounds__(W *kWave, 2) void k_attn_short_bwd(const ShortBwd f) {
    constexpr int KS = DP / 16, NT = DP / 32, TB = 128 * DP, LO = 64 * DP;
    constexpr int THREADS = W * kWave, UNITS = 4 * DP, PER = (UNITS + THREADS - 1) / THREADS;  // 8-column pieces of a tile
    constexpr int BLOCKS = DP / 8, PW = (BLOCKS + W - 1) / W;  // 16 x 16 blocks of a tile's gq, of a wave
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // q's tile, go's tile, the waves' keys, their ds, then small tables
    char *const qs = smem, *const gs = smem + TB, *const keys = smem + 2 * TB, *const dss = keys + W * TB;
    float *const small = (float *)(dss + W * kDsTile);
    float *const stats = small, *const dots = small + 64, *const red = dots + (DP / 8) * 32;  // [64], [DP / 8][32], [2][W]
    f2 *const dsx = (f2 *)(red + 2 * W);  // [W]: the scales of the waves' ds, and of their keys
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ra = row_at(lane), ca = col_at(lane), ta = turned_at(lane), D = (int)a.D;
    for (int64_t w = blockIdx.x; w < f.units; w += gridDim.x) {
        const int64_t pair = w / f.splits, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int split = (int)(w - pair * f.splits);
        const int n = (int)keys_of(a.Lk, f.key_len, b), nt = (n + kTile - 1) / kTile;
        const int64_t t0 = f.qtiles * split / f.splits, t1 = f.qtiles * (split + 1) / f.splits;
        // workgroups that share a CU give the first tiles of keys (the only ones of a short sequence) to other waves, so to other SIMDs
        const int kw = (wave + (int)(w >> 8) * (W / 2)) & (W - 1), key = kw * kTile + (lane & 31);
        char *const kt = keys + kw * TB, *const mine_ds = dss + kw * kDsTile;
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
        __syncthreads();  // the last unit's keys have been read
        if (t0 < t1) fetch(t0);
        h8 kh[KS], kl[KS], vh[KS], vl[KS];
        float ek = 0.0f, ev = 0.0f;
        if (mine) {  // this wave's values, through the place of its keys, and its keys, which stay
            ev = wave_tile<DP>(f.v + b * a.sv[0] + u * a.sv[2], a.sv[1], kw * kTile, n, D, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) vh[s] = row_frag(kt + ra, s), vl[s] = row_frag(kt + ra + LO, s);
            ek = wave_tile<DP>(f.k + b * a.sk[0] + u * a.sk[2], a.sk[1], kw * kTile, n, D, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) kh[s] = row_frag(kt + ra, s), kl[s] = row_frag(kt + ra + LO, s);
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
                // ds for gq, in two pieces: a tile of 32 rows of keys, its columns the rows of queries
                float finite = most;
                if (__builtin_expect(most == INFINITY, 0)) {  // a row of queries with an infinity leaves the others their scale
                    finite = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; r++) finite = __builtin_fmaxf(finite, __builtin_fabsf(dp[r]) < INFINITY ? __builtin_fabsf(dp[r]) : 0.0f);
                }
                const int ed = tile_exponent(wave_max_nan_skip(finite));
                const float id = pow2i(-ed);
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = dp[4 * j + e] * id;
                    const Split8 x = split8(y);
                    char *const at = mine_ds + 512 * j + 8 * half;
                    const int r0 = 16 * (lane & 31), r1 = r0 ^ 64;
                    *(h4 *)(at + r0) = x.hi.lo, *(h4 *)(at + 512 + r1) = x.hi.hi;
                    *(h4 *)(at + 2048 + r0) = x.lo.lo, *(h4 *)(at + 2560 + r1) = x.lo.hi;
                }
                if (lane == 0) dsx[kw] = f2{__builtin_amdgcn_exp2f((float)ed - sh), pow2i((int)ek) * a.scale};
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
            }
            __syncthreads();
            if (f.gq) {  // gq^T = k^T ds^T over all keys, blocks of 16 columns and 16 rows of queries
                f4 sum[PW];
#pragma unroll
                for (int x = 0; x < PW; x++) sum[x] = f4{0.f, 0.f, 0.f, 0.f};
                for (int y = 0; y < nt; y++) {
                    const f2 by = dsx[y];
#pragma unroll
                    for (int x = 0; x < PW; x++) {
                        const int block = wave + x * W, c = block % (DP / 16), r = block / (DP / 16);
                        if (BLOCKS % W && block >= BLOCKS) break;
                        const char *const kc = keys + y * TB + 1024 * c + ta, *const dc = dss + y * kDsTile + 1024 * r + ta;
                        const char *const kc2 = keys + y * TB + 1024 * c + (ta ^ 64), *const dc2 = dss + y * kDsTile + 1024 * r + (ta ^ 64);
                        const h8 ah = turned16(kc, kc2), al = turned16(kc + LO, kc2 + LO), bh = turned16(dc, dc2), bl = turned16(dc + 2048, dc2 + 2048);
                        f4 v = {0.f, 0.f, 0.f, 0.f};
                        v = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, v, 0, 0, 0);
                        v = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, v, 0, 0, 0);
                        v = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, v, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; e++) sum[x][e] = fma_(v[e] * by.x, by.y, sum[x][e]);
                    }
                }
#pragma unroll
                for (int x = 0; x < PW; x++) {
                    const int block = wave + x * W, c = block % (DP / 16), r = block / (DP / 16);
                    const int64_t R = t * kTile + 16 * r + (lane & 15);
                    if (block >= BLOCKS || R >= f.rows) continue;
                    int64_t i, g;
                    a.row(R, i, g);
                    store4(f.gq + ((b * a.Lq + i) * a.Hq + u * a.G + g) * D, 16 * c + 4 * (lane >> 4), D, sum[x], f.acc_q);
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
    const size_t lds = 2 * 128 * DP + (size_t)W * (128 * DP + kDsTile) + (64 + DP / 8 * 32 + 4 * W) * sizeof(float);
    launch(&k_attn_short_bwd<DP, W>, f.units, W * kWave, lds, st, f);
}

void short_bwd(const ShortBwd &f, int DP, hipStream_t st) {
    const bool four = f.a.Lk <= 4 * kTile;
    if (DP == 32) four ? bwd_launch<32, 4>(f, st) : bwd_launch<32, 8>(f, st);
    else four ? bwd_launch<64, 4>(f, st) : bwd_launch<64, 8>(f, st);
}

}  // namespace nchip
