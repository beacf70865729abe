// Attention to few keys (a padded text, the patches of a small image): a head's keys fit a workgroup, which splits them itself
// instead of reading them packed.  D padded to DP columns, at most 16384 / DP keys forward; backward at most 256 in heads of up to
// 64 columns and 128 in heads of up to 128.
#include "attention.hpp"
#include "attention_short.hpp"

#include <math.h>

namespace nchip {

// A wave reads 32 rows of `src` (from `row0` on, n in all, `step` floats apart): the tile's exponent, with kOwnRows added where its rows
// have their own (wanted: own is given, this lane's row's); and splits them into LDS.
template <int DP>
__device__ __forceinline__ int tile_load(const float *src, int64_t step, int row0, int n, int D, float (&x)[DP / 16][8], int *own = nullptr) {
    const int lane = threadIdx.x & 63, half = lane >> 5, r = lane & 31;
    const bool live = row0 + r < n;
    float most = 0.0f;
    load_chunks(src + (live ? row0 + r : 0) * step, 8 * half, 16, D, x);
#pragma unroll
    for (int k = 0; k < DP / 16; k++) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[k][e] = live ? x[k][e] : 0.0f;
        most = abs_max(x[k], most);
    }
    const float top = wave_max_nan_skip(most);
    const int ex = tile_exponent(top);
    if (!own) return ex;
    most = halves_max(most);
    const bool unlike = rows_unlike(most, top);
    *own = unlike ? row_exponent(most, ex) : ex;
    return unlike ? ex + kOwnRows : ex;
}
template <int DP>
__device__ __forceinline__ void tile_split(float (&x)[DP / 16][8], int ex, char *tile) {
    const float inv = pow2i(-ex);
    char *out = tile + row_at(threadIdx.x & 63);
#pragma unroll
    for (int k = 0; k < DP / 16; k++) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[k][e] *= inv;
        const Split8 s = split8(x[k]);
        *(h8 *)(out + 1024 * k) = s.hi;
        *(h8 *)(out + 64 * DP + 1024 * k) = s.lo;
    }
}

// Forward: keys and values of a pair stay in LDS, and each wave goes over tiles of queries by itself.  4096 x at most 77, 4 x 16
// heads of 64: 42 to 44 us for 136 MB (3.2 TB/s) -- a wave reads its rows, multiplies and stores in turn, and the three
// waves of a SIMD do not cover all of it.
template <int DP, int W, int OCC>
__global__ __launch_bounds__(W *kWave, OCC) void k_attn_short_fwd(const ShortFwd f) {
    constexpr int TB = 128 * DP;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float *const rows = (float *)(smem + 2 * f.tiles * TB);  // [2][tiles][32], then the tiles' exponents
    int *const exps = (int *)(rows + 2 * f.tiles * kTile);
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
            float x[DP / 16][8];
            int er;
            const int at = val ? f.tiles + k : k, e = tile_load<DP>(src, val ? a.sv[1] : a.sk[1], k * kTile, n, (int)a.D, x, &er);
            tile_split<DP>(x, er, smem + at * TB);
            if (lane == 0) exps[at] = e;
            if (own_rows(e) && half == 0) rows[at * kTile + lane] = (float)(er - exponent_of(e));
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
                attend(sum, q, kt + t * TB, vt + t * TB, __builtin_amdgcn_readfirstlane(exps[t]), __builtin_amdgcn_readfirstlane(exps[f.tiles + t]),
                       rows + t * kTile + 4 * half, rows + (f.tiles + t) * kTile + 4 * half, t + 1 == nt, min(n - t * kTile, kTile) - 4 * half);
            const float l = halves_sum(sum.l);
            if (live) {
                store_column<false>(f.o + ((b * a.Lq + i) * a.Hq + h) * a.D, sum.o, true, l != 0.0f ? unit_of(sum.U) / l : 0.0f, half, (int)a.D, 0);
                if (f.lse && half == 0)
                    f.lse[(b * a.Hq + h) * a.Lq + i] = nt ? fma_(sum.m, kLn2, logf(l)) : -INFINITY;
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

// The backward's way in: the workgroup's W waves read a tile of 32 rows of queries, output gradients and outputs, one tile ahead,
// and split it.  Piece p is columns 8 (p / 32) .. + 7 of row p % 32.
template <int DP, int W>
struct Feed {
    static constexpr int THREADS = W * kWave, UNITS = 4 * DP, PER = (UNITS + THREADS - 1) / THREADS;
    float q[PER][8], go[PER][8], o[PER][8], lse;

    __device__ __forceinline__ void fetch(const ShortBwd &f, int64_t b, int64_t u, int64_t t) {
        const AttnArgs &a = f.a;
        const int D = (int)a.D;
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
            load8(f.q + b * a.sq[0] + i * a.sq[1] + h * a.sq[2], d, D, q[k]);
            load8(f.go + at, d, D, go[k]);
            load8(f.o + at, d, D, o[k]);
            if (k == 0) lse = p < 32 && in ? f.lse[(b * a.Hq + h) * a.Lq + i] * kLog2e : INFINITY;
        }
    }

    // into the tiles qs and gs, with stats[64]: the rows' log2-sum-exps and go . o; dots [DP / 8][32] and red [2][W] are scratch
    __device__ __forceinline__ void split(char *qs, char *gs, float *stats, float *dots, float *red, int &eq, int &eg) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        float mq = 0.0f, mg = 0.0f;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const int p = threadIdx.x + k * THREADS;
            float dot = 0.0f;
            mq = abs_max(q[k], mq), mg = abs_max(go[k], mg);
#pragma unroll
            for (int e = 0; e < 8; e++) dot = fma_(go[k][e], o[k][e], dot);
            if (p < UNITS) dots[p] = dot;
        }
        mq = wave_max_nan_skip(mq), mg = wave_max_nan_skip(mg);
        if (lane == 0) red[wave] = mq, red[W + wave] = mg;
        __syncthreads();
        mq = red[0], mg = red[W];
#pragma unroll
        for (int x = 1; x < W; x++) mq = __builtin_fmaxf(mq, red[x]), mg = __builtin_fmaxf(mg, red[W + x]);
        eq = tile_exponent(mq), eg = tile_exponent(mg);
        const float iq = pow2i(-eq), ig = pow2i(-eg);
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const int p = threadIdx.x + k * THREADS, c = p >> 5;
            if (p >= UNITS) continue;
#pragma unroll
            for (int e = 0; e < 8; e++) q[k][e] *= iq, go[k][e] *= ig;
            const int at = 16 * (32 * c + ((p & 31) ^ (4 * (c & 1))));
            const Split8 x = split8(q[k]), y = split8(go[k]);
            *(h8 *)(qs + at) = x.hi, *(h8 *)(qs + 64 * DP + at) = x.lo;
            *(h8 *)(gs + at) = y.hi, *(h8 *)(gs + 64 * DP + at) = y.lo;
        }
        if (threadIdx.x < 32) {
            float d = dots[threadIdx.x];
#pragma unroll
            for (int c = 1; c < DP / 8; c++) d += dots[32 * c + threadIdx.x];
            stats[threadIdx.x] = lse;
            stats[32 + threadIdx.x] = d;
        }
        __syncthreads();
    }
};

// A wave's ds (32 rows of queries as a result's rows, its keys the columns; `most` its lane's largest) in two pieces as a packed
// tile of 32 rows of keys, whose columns are the rows of queries; returns the tile's exponent.
__device__ __forceinline__ int put_ds(const f16x &ds, float most, char *tile) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    float finite = most;
    if (__builtin_expect(most == INFINITY, 0)) {  // a row of queries with an infinity leaves the others their scale
        finite = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r++) finite = __builtin_fmaxf(finite, __builtin_fabsf(ds[r]) < INFINITY ? __builtin_fabsf(ds[r]) : 0.0f);
    }
    const int ed = tile_exponent(wave_max_nan_skip(finite));
    const float id = pow2i(-ed);
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = ds[4 * j + e] * id;
        const Split8 x = split8(y);
        char *const at = tile + 512 * j + 8 * half;
        const int r0 = 16 * (lane & 31), r1 = r0 ^ 64;
        *(h4 *)(at + r0) = x.hi.lo, *(h4 *)(at + 512 + r1) = x.hi.hi;
        *(h4 *)(at + 2048 + r0) = x.lo.lo, *(h4 *)(at + 2560 + r1) = x.lo.hi;
    }
    return ed;
}

// gq^T = k^T ds^T over all nt tiles of keys, blocks of 16 columns and 16 rows of queries dealt over the W waves; scale[y]: the
// scales of tile y's ds, and of its keys
template <int DP, int W>
__device__ __forceinline__ void gq_blocks(const ShortBwd &f, int64_t b, int64_t u, int64_t t, int nt, const char *keys, const char *dss, const f2 *scale) {
    constexpr int TB = 128 * DP, LO = 64 * DP, BLOCKS = DP / 8, PW = (BLOCKS + W - 1) / W;
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ta = turned_at(lane);
    f4 sum[PW];
#pragma unroll
    for (int x = 0; x < PW; x++) sum[x] = f4{0.f, 0.f, 0.f, 0.f};
    for (int y = 0; y < nt; y++) {
        const f2 by = scale[y];
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
        store4(f.gq + ((b * a.Lq + i) * a.Hq + u * a.G + g) * a.D, 16 * c + 4 * (lane >> 4), (int)a.D, sum[x], f.acc_q);
    }
}

// Backward in one pass over the queries: every wave holds 32 keys, the workgroup splits a tile of queries and output gradients
// (the next one's on their way meanwhile), and each wave takes its part of gk and gv as k_attn_dkv does.  It leaves its ds in LDS,
// and the waves share the blocks of gq^T = k^T ds^T over all keys.  The same sizes: 97 to 104 us, and 120 to 125 with every
// wave's part of gq added in LDS; memory would take 57.  A tile's steps follow each other (read, split, scores, gradients, store), two
// workgroups a CU, by the registers, which hold heads of 64 columns and no more.
template <int DP, int W>
__global__ __launch_bounds__(W *kWave, 2) void k_attn_short_bwd(const ShortBwd f) {
    constexpr int KS = DP / 16, NT = DP / 32, TB = 128 * DP, LO = 64 * DP;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // q's tile, go's tile, the waves' keys, their ds, then small tables
    char *const qs = smem, *const gs = smem + TB, *const keys = smem + 2 * TB, *const dss = keys + W * TB;
    float *const small = (float *)(dss + W * kDsTile);
    float *const stats = small, *const dots = small + 64, *const red = dots + (DP / 8) * 32;  // [64], [DP / 8][32], [2][W]
    f2 *const dsx = (f2 *)(red + 2 * W);  // [W]: the scales of the waves' ds, and of their keys
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
        char *const kt = keys + kw * TB, *const mine_ds = dss + kw * kDsTile;
        const bool mine = kw < nt, live = key < n;

        Feed<DP, W> next;
        __syncthreads();  // the last unit's keys have been read
        if (t0 < t1) next.fetch(f, b, u, t0);
        h8 kh[KS], kl[KS], vh[KS], vl[KS];
        float ek = 0.0f, ev = 0.0f;
        if (mine) {  // this wave's values, through the place of its keys, and its keys, which stay
            float x[KS][8];
            ev = (float)tile_load<DP>(f.v + b * a.sv[0] + u * a.sv[2], a.sv[1], kw * kTile, n, D, x);
            tile_split<DP>(x, (int)ev, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) vh[s] = row_frag(kt + ra, s), vl[s] = row_frag(kt + ra + LO, s);
            ek = (float)tile_load<DP>(f.k + b * a.sk[0] + u * a.sk[2], a.sk[1], kw * kTile, n, D, x);
            tile_split<DP>(x, (int)ek, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) kh[s] = row_frag(kt + ra, s), kl[s] = row_frag(kt + ra + LO, s);
        }
        f16x dk[NT], dv[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) dk[t][r] = dv[t][r] = 0.0f;
        float F = 0x1p100f, E = -1000.0f;
        const ScaleParts parts(a.scale);
        const float ck = pow2i((int)ek) * a.scale * kLog2e, cv = pow2i((int)ev);
        for (int64_t t = t0; t < t1; t++) {
            int eq, eg;
            next.split(qs, gs, stats, dots, red, eq, eg);
            if (t + 1 < t1) next.fetch(f, b, u, t + 1);
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
                const int ed = put_ds(dp, most, mine_ds);
                if (lane == 0) dsx[kw] = f2{__builtin_amdgcn_exp2f((float)ed - sh), pow2i((int)ek) * a.scale};
                const float kap = parts.times((float)eq - sh);
                float by;
                if (column_scale(halves_max(most) * __builtin_fabsf(kap), F, by)) scale_acc(dk, by);
                const float kF = finite_product(kap, F);
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
            if (f.gq) gq_blocks<DP, W>(f, b, u, t, nt, keys, dss, dsx);
        }
        if (key < a.Lk) {
            const int64_t at = ((b * a.Lk + key) * a.Hkv + u) * D;
            const bool some = live && t0 < t1;
            if (f.gk) store_column<true>(f.gk + split * f.part_k + at, dk, some, 1.0f / F, half, D, f.acc_k);
            if (f.gv) store_column<true>(f.gv + split * f.part_k + at, dv, some, __builtin_amdgcn_exp2f(E - 14.0f), half, D, f.acc_v);
        }
    }
}

// Backward in one pass over the queries: two waves share 32 keys, and the workgroup splits a tile of queries and output gradients
// (the next one's on their way meanwhile).  As in k_attn_dkv one wave takes the scores, p and gv, the other makes ds of p and takes
// gk; it leaves ds in LDS, and all waves share the blocks of gq^T = k^T ds^T over all keys.  Half the registers for each wave's
// keys: heads of up to 128 columns, a workgroup a CU.  4096 x 77, 4 x 16 heads, forward and backward: of 128 columns 320 us, and 487
// through packed tiles and k_attn_dkv, k_attn_dq; of 80, 258 and 319; of 64, 204 where the kernel above takes 150.
template <int DP, int KT>
__global__ __launch_bounds__(2 * KT *kWave, 2) void k_attn_short_bwd_pairs(const ShortBwd f) {
    constexpr int KS = DP / 16, NT = DP / 32, TB = 128 * DP, LO = 64 * DP, W = 2 * KT;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // q's tile, go's tile, the tiles of keys, p and then ds of each, then small tables
    char *const qs = smem, *const gs = smem + TB, *const keys = smem + 2 * TB, *const dss = keys + KT * TB;
    float *const small = (float *)(dss + KT * kDsTile);
    float *const stats = small, *const dots = small + 64, *const red = dots + (DP / 8) * 32;  // [64], [DP / 8][32], [2][W]
    f2 *const dsx = (f2 *)(red + 2 * W);  // [KT]: the scales of the tiles' ds, and of their keys
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ra = row_at(lane), ca = col_at(lane), D = (int)a.D;
    const int ds_wave = wave / KT;  // 0: p and gv, 1: ds and gk
    for (int64_t w = blockIdx.x; w < f.units; w += gridDim.x) {
        const int64_t pair = w / f.splits, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int split = (int)(w - pair * f.splits);
        const int n = (int)keys_of(a.Lk, f.key_len, b), nt = (n + kTile - 1) / kTile;
        const int64_t t0 = f.qtiles * split / f.splits, t1 = f.qtiles * (split + 1) / f.splits;
        // workgroups that share a CU give the first tiles of keys (the only ones of a short sequence) to other waves, so to other SIMDs
        const int kw = (wave + (int)(w >> 8) * (KT / 2)) & (KT - 1), key = kw * kTile + (lane & 31);
        char *const kt = keys + kw * TB, *const hand = dss + kw * kDsTile;
        const bool mine = kw < nt, live = key < n;

        Feed<DP, W> next;
        __syncthreads();  // the last unit's keys have been read
        // this wave's keys or values as row fragments: the values go through the place of the keys, which stay there
        h8 kh[KS], kl[KS];
        int ek = 0;
        if (mine && ds_wave) {
            float x[KS][8];
            ek = tile_load<DP>(f.v + b * a.sv[0] + u * a.sv[2], a.sv[1], kw * kTile, n, D, x);
            tile_split<DP>(x, ek, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) kh[s] = row_frag(kt + ra, s), kl[s] = row_frag(kt + ra + LO, s);
        }
        __syncthreads();
        if (mine && !ds_wave) {
            float x[KS][8];
            ek = tile_load<DP>(f.k + b * a.sk[0] + u * a.sk[2], a.sk[1], kw * kTile, n, D, x);
            tile_split<DP>(x, ek, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) kh[s] = row_frag(kt + ra, s), kl[s] = row_frag(kt + ra + LO, s);
            if (lane == 0) dsx[kw].y = pow2i(ek) * a.scale;
        }
        if (t0 < t1) next.fetch(f, b, u, t0);
        f16x acc[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[t][r] = 0.0f;
        float F = 0x1p100f, E = -1000.0f;
        const ScaleParts parts(a.scale);
        const float ck = ds_wave ? pow2i(ek) : pow2i(ek) * a.scale * kLog2e;
        for (int64_t t = t0; t < t1; t++) {
            int eq, eg;
            next.split(qs, gs, stats, dots, red, eq, eg);
            if (t + 1 < t1) next.fetch(f, b, u, t + 1);
            const f4 *const rows = (const f4 *)stats + half;
            f4 *const ph = (f4 *)hand + lane;  // p's registers 4 j .. 4 j + 3 at 64 j
            // p as 2^14 p, less for tiles of smaller gradients (no less than 2^-60 times: below what gv can show)
            const float ex = (float)eg, En = __builtin_fmaxf(E, ex), sh = 14.0f + __builtin_fmaxf(ex - En, -60.0f);
            f16x s;
            if (mine) {
                const char *rt = (ds_wave ? gs : qs) + ra;
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = 0.0f;
                steps<KS>([&](int k) { return Pieces{row_frag(rt, k), row_frag(rt + LO, k)}; },
                          [&](int k, const Pieces &x) { s = mfma3(x.hi, x.lo, kh[k], kl[k], s); });
                if (!ds_wave) {
                    if (ex > E) scale_acc(acc, __builtin_amdgcn_exp2f(E - ex));
                    const float c = ck * pow2i(eq), base = live ? sh : -INFINITY;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const f4 ls = rows[2 * j];
#pragma unroll
                        for (int e = 0; e < 4; e++) s[4 * j + e] = __builtin_amdgcn_exp2f(fma_(s[4 * j + e], c, base - ls[e]));
                        ph[64 * j] = f4{s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]};
                    }
                }
            }
            E = En;
            lds_barrier();  // p is there
            if (mine) {
                if (ds_wave) {
                    const float c = ck * pow2i(eg), kap = parts.times((float)eq - sh);
                    float most = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const f4 p = ph[64 * j], de = rows[8 + 2 * j];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int r = 4 * j + e;
                            s[r] = p[e] * fma_(s[r], c, -de[e]);
                            most = __builtin_fmaxf(most, __builtin_fabsf(s[r]));
                        }
                    }
                    const int ed = put_ds(s, most, hand);  // where p was
                    if (lane == 0) dsx[kw].x = __builtin_amdgcn_exp2f((float)ed - sh);
                    float by;
                    if (column_scale(halves_max(most) * __builtin_fabsf(kap), F, by)) scale_acc(acc, by);
                    const float kF = finite_product(kap, F);
#pragma unroll
                    for (int r = 0; r < 16; r++) s[r] *= kF;
                }
                const char *ct = (ds_wave ? qs : gs) + ca;
                const Split8 y[2] = {split_regs(s, 0), split_regs(s, 8)};
                steps<2 * NT>([&](int k) { return Pieces{col_frag(ct, k / NT, k % NT), col_frag(ct + LO, k / NT, k % NT)}; },
                              [&](int k, const Pieces &v) { acc[k % NT] = mfma3(v.hi, v.lo, y[k / NT].hi, y[k / NT].lo, acc[k % NT]); });
            }
            lds_barrier();
            if (f.gq) gq_blocks<DP, W>(f, b, u, t, nt, keys, dss, dsx);
        }
        float *const out = ds_wave ? f.gk : f.gv;
        if (out && key < a.Lk)
            store_column<true>(out + split * f.part_k + ((b * a.Lk + key) * a.Hkv + u) * D, acc, live && t0 < t1,
                               ds_wave ? 1.0f / F : __builtin_amdgcn_exp2f(E - 14.0f), half, D, ds_wave ? f.acc_k : f.acc_v);
    }
}

int short_keys_fwd(int DP) { return DP <= 128 ? 16384 / DP : -1; }
int short_keys_bwd(int DP) { return DP <= 64 ? 256 : DP <= 128 ? 128 : -1; }

template <class F, class A>
static void launch(F *kernel, int64_t units, int threads, size_t lds, hipStream_t st, const A &args) {
    if (lds > 65536) (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(units < kAttnGrid ? units : kAttnGrid)), dim3(threads), lds, st, args);
}

void short_fwd(const ShortFwd &f, int DP, hipStream_t st) {
    const size_t lds = (size_t)f.tiles * 2 * (tile_bytes(DP) + (kTile + 1) * sizeof(float));
    if (DP == 32) launch(&k_attn_short_fwd<32, 8, 4>, f.units, 512, lds, st, f);
    // three workgroups of four waves a CU where their keys fit its LDS, else eight waves over one copy (heads of 64, both ways: 4096
    // x 77, 4 x 16 heads 147 us with four and 153 with eight, 64 x 64, 64 x 8 35 and 39; 197 x 197, 8 x 12 heads 60 and 58)
    else if (DP == 64 && 3 * lds <= 160 * 1024) launch(&k_attn_short_fwd<64, 4, 3>, f.units, 256, lds, st, f);
    else if (DP == 64) launch(&k_attn_short_fwd<64, 8, 2>, f.units, 512, lds, st, f);
    else if (DP == 96) launch(&k_attn_short_fwd<96, 8, 2>, f.units, 512, lds, st, f);
    else launch(&k_attn_short_fwd<128, 8, 2>, f.units, 512, lds, st, f);
}

template <int DP, int W, int KT, class F>
static void bwd_launch(F *kernel, const ShortBwd &f, hipStream_t st) {  // W waves, KT tiles of keys
    const size_t lds = 2 * 128 * DP + (size_t)KT * (128 * DP + kDsTile) + (64 + DP / 8 * 32 + 2 * W + 2 * KT) * sizeof(float);
    launch(kernel, f.units, W * kWave, lds, st, f);
}

void short_bwd(const ShortBwd &f, int DP, hipStream_t st) {
    const bool four = f.a.Lk <= 4 * kTile;
    if (DP == 32) four ? bwd_launch<32, 4, 4>(&k_attn_short_bwd<32, 4>, f, st) : bwd_launch<32, 8, 8>(&k_attn_short_bwd<32, 8>, f, st);
    else if (DP == 64) four ? bwd_launch<64, 4, 4>(&k_attn_short_bwd<64, 4>, f, st) : bwd_launch<64, 8, 8>(&k_attn_short_bwd<64, 8>, f, st);
    else if (DP == 96) bwd_launch<96, 8, 4>(&k_attn_short_bwd_pairs<96, 4>, f, st);
    else bwd_launch<128, 8, 4>(&k_attn_short_bwd_pairs<128, 4>, f, st);
}

}  // namespace nchip
