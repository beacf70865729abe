// Attention of queries to keys and values of another length (cross attention; self attention without a mask is the case of
// equal lengths), forward and backward.  q [B, Lq, Hq, D], k and v [B, Lk, Hkv, D], any strides with unit columns; query head
// h reads the keys of head h / (Hq / Hkv); key_len [B] (or none) cuts each sequence's keys.
//
//     s = scale q . k,  p = softmax(s) over the sequence's keys,  o = p v,  lse = log sum exp(s)
//     dp = go . v,  ds = p (dp - go . o) scale,  gq = ds k,  gk = ds^T q,  gv = p^T go
//
// A sequence without keys gives o = 0, lse = -inf and no gradient.  Keys and values past a sequence's length are not read.
//
// A value that counts and is not finite makes the results that meet it NaN: pieces of an infinity are NaN (inf - inf), and the
// kernel that reads plain fp32 (k_attn_token) looks at the operands of scores that are not finite.
//
// The products run on the fp16 matrix cores with operands in two pieces (attention.hpp), packed once into a workspace, where
// they bound the time: three products for one reach at most a third of a library's fp16 product of 8192^3, 1.23 PFLOP/s, which
// is 2.7 times what its fp32 product reaches.  Few rows of queries (k_attn_token) are bound by reading the keys, few keys
// (attention_short.hip) by the chain of one tile's steps.
#include "attention.hpp"
#include "attention_short.hpp"

#include <math.h>

#include <algorithm>

namespace nchip {

// ------------------------------------------------------------------------------------------------
// packing: a workgroup a tile of 32 rows; bound by memory (8192 keys and values of 16 heads of 128, 134 MB each way: 58 us, 4.6 TB/s)
// ------------------------------------------------------------------------------------------------
// Rows of a (sequence, head of keys) pair: queries' row R is token R / G of query head u G + R % G, keys' are tokens.
struct PackJob {
    const float *src;
    int64_t sb, sl, sh;
    int64_t len, tiles;    // rows and tiles of a pair, before key_len
    int by_len;            // keys: rows are cut by key_len; else queries
    char *out;             // [pair][tile][128 DP]
    int *exps;             // [pair][tile] exponents of the scales, kOwnRows added where `rows` counts, or with stats where a row is `loose`
    float *rows;           // [pair][tile][32] rows' exponents below it, where they have their own; none: they are in stats
    int64_t first;         // the job's first workgroup
    const float *o, *lse;  // the output gradient's job: o (laid out as src), the rows' log-sum-exps [B, Hq, Lq]
    // [pair][tile][64]: log2-sum-exps (infinite past the rows), src . o of the tile's rows.  Where the rows have their own exponents,
    // d below the tile's (d <= 0), log2-sum-exps less d, and 2^-d src . o: the scores' gradients p (go . v - go . o) come out
    // of p 2^d and the row's pieces' products with v as if the rows had the tile's.
    float *stats;
};
struct PackArgs {
    PackJob job[4];
    int jobs;
    AttnArgs a;
    int64_t total;
    const int *key_len;
};

template <int DP>
__global__ __launch_bounds__(kAttnB) void k_attn_pack(const PackArgs a) {
    constexpr int C = DP / 8, PER = (C + 7) / 8;  // chunks of a row; of a lane
    __shared__ float tops[8][kTile], dots[8][kTile];
    const int t = threadIdx.x, row = t & 31, cl = t >> 5;
    for (int64_t w = blockIdx.x; w < a.total; w += gridDim.x) {
        int jx = 0;
        while (jx + 1 < a.jobs && w >= a.job[jx + 1].first) jx++;
        const PackJob &j = a.job[jx];
        const int64_t pair = (w - j.first) / j.tiles, tl = (w - j.first) - pair * j.tiles;
        const int64_t b = pair / a.a.Hkv, u = pair - b * a.a.Hkv;
        const int64_t n = j.by_len ? keys_of(a.a.Lk, a.key_len, b) : j.len;
        const int64_t R = tl * kTile + row;
        if (tl * kTile >= n) continue;  // no workgroup reads this tile
        const bool live = R < n;
        int64_t i = live ? R : 0, g = 0;
        if (!j.by_len) a.a.row(i, i, g);
        const int64_t h = j.by_len ? u : u * a.a.G + g, off = b * j.sb + i * j.sl + h * j.sh;
        const float *src = j.src + off;
        float x[PER][8], most = 0.0f, dot = 0.0f;
#pragma unroll
        for (int k = 0; k < PER; k++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[k][e] = 0.0f;
            const int c = cl + 8 * k;
            if (live && c < C) load8(src, 8 * c, (int)a.a.D, x[k]);
            most = abs_max(x[k], most);
            if (j.stats && live && c < C) {
                float y[8];
                load8(j.o + off, 8 * c, (int)a.a.D, y);
#pragma unroll
                for (int e = 0; e < 8; e++) dot = fma_(x[k][e], y[e], dot);
            }
        }
        __syncthreads();  // the last tile has been read
        if (j.stats) dots[cl][row] = dot;
        tops[cl][row] = most;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; e++) most = __builtin_fmaxf(most, tops[e][row]);
        const float top = wave_max_nan_skip(most);
        const int ex = tile_exponent(top);
        const bool own = rows_unlike(most, top);
        const int er = own ? row_exponent(most, ex) : ex;
        const float inv = pow2i(-er);
        const int64_t at = pair * j.tiles + tl;
        float log_sum = INFINITY;
        if (j.stats && live) log_sum = j.lse[(b * a.a.Hq + h) * a.a.Lq + i] * kLog2e;
        const bool marked = (own && j.rows) || __any(loose(log_sum));
        if (t == 0) j.exps[at] = marked ? ex + kOwnRows : ex;
        if (own && j.rows && t < kTile) j.rows[at * kTile + t] = (float)(er - ex);
        if (j.stats && t < kTile) {
            float d = dots[0][t];
#pragma unroll
            for (int e = 1; e < 8; e++) d += dots[e][t];
            j.stats[at * 64 + t] = log_sum - (float)(er - ex);
            j.stats[at * 64 + 32 + t] = d * pow2i(ex - er);
        }
        char *out = j.out + at * tile_bytes(DP);
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const int c = cl + 8 * k;
            if (c >= C) continue;
#pragma unroll
            for (int e = 0; e < 8; e++) x[k][e] *= inv;
            const Split8 s = split8(x[k]);
            h8 *o = (h8 *)out + c * 32 + (row ^ (4 * (c & 1)));
            o[0] = s.hi;
            o[4 * DP] = s.lo;
        }
    }
}

// ------------------------------------------------------------------------------------------------
// stages of tiles in LDS
// ------------------------------------------------------------------------------------------------
// blocks of 1 KiB dealt over the workgroup's waves, copied straight to LDS; nothing waits for them here
template <int WAVES = kAttnWaves>
__device__ __forceinline__ void stage_copy(const char *src, uint32_t lds, int blocks) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    for (int i = wave; i < blocks; i += WAVES) dma16(src + i * 1024 + lane * 16, lds + i * 1024);
}
__device__ __forceinline__ void stage_wait() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // this wave's copies and LDS reads
    __builtin_amdgcn_s_barrier();                                // everyone's
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}

// A value that the launch does not write, through the scalar cache: a vector load here would wait behind the next stage's
// copies, which share its counter.
__device__ __forceinline__ int scalar_load(const int *p) { return *(const __attribute__((address_space(4))) int *)(uintptr_t)p; }

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
struct FwdArgs {
    AttnArgs a;
    const float *q;
    const char *kp, *vp;         // packed keys and values
    const int *kx, *vx;          // their exponents
    const float *kr, *vr;        // and their rows'
    const int *key_len;
    float *o, *lse;
    float *po;                   // splits: [split][pair][row][D] sums, and {reference, sum} of each row
    f2 *pm;
    int64_t rows, tiles, units;  // rows of a pair (G Lq), tiles of keys of a pair at most, workgroups' units
    int qtiles, splits;          // groups of 128 rows of a pair, parts its keys are cut into
};

// A workgroup's waves hold 32 rows of queries each, so that a stage of TPS tiles of keys and values comes from L2 once for 128
// rows, the next one on its way meanwhile.  Two waves a SIMD (what the registers allow) run one's exponentials beside the other's
// products: from two workgroups, or from KG = 2 groups of waves of one, which take every other stage (key_groups below).  8192 x
// 8192, 16 heads of 128: 1.45 to 1.54 ms from card to card, 1.07 to 1.14 PFLOP/s of fp16 products.  Heads of up to 128 columns hold
// everything in registers; those of 129 to 256 spill 78.
template <int DP, int TPS, int OCC, int KG>
__global__ __launch_bounds__(KG *kAttnB, OCC) void k_attn_fwd(const FwdArgs f) {
    constexpr int TB = 128 * DP, TS = KG * TPS, STAGE = 2 * TS * TB;  // bytes of a packed tile; tiles and bytes of a stage
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = wave_all & (kAttnWaves - 1), kg = wave_all / kAttnWaves;  // tile of queries, group of keys
    const int ra = row_at(lane), ca = col_at(lane);
    const uint32_t lds = lds_address(smem);
    for (int64_t w = blockIdx.x; w < f.units; w += gridDim.x) {
        const int64_t unit = xcd_unit(w, f.units);
        const int64_t rest = unit / f.qtiles;
        const int qt = (int)(unit - rest * f.qtiles);
        const int64_t pair = rest / f.splits, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int split = (int)(rest - pair * f.splits);
        const int64_t n = keys_of(a.Lk, f.key_len, b), nt = (n + kTile - 1) / kTile;
        const int64_t t0 = nt * split / f.splits, t1 = nt * (split + 1) / f.splits;
        const char *kp = f.kp + pair * f.tiles * TB, *vp = f.vp + pair * f.tiles * TB;
        const int *kx = f.kx + pair * f.tiles, *vx = f.vx + pair * f.tiles;
        const float *kr = f.kr + pair * f.tiles * kTile, *vr = f.vr + pair * f.tiles * kTile;

        auto copy = [&](int64_t t, int buf) {
            const int c = (int)min((int64_t)TS, t1 - t) * (TB / 1024);
            const uint32_t at = __builtin_amdgcn_readfirstlane(lds + buf * STAGE);
            stage_copy<KG * kAttnWaves>(kp + t * TB, at, c);
            stage_copy<KG * kAttnWaves>(vp + t * TB, at + TS * TB, c);
        };
        __syncthreads();  // the last unit's stages have been read
        if (t0 < t1) copy(t0, 0);

        // this lane's row of queries, times scale log2(e), as the second operand
        const int64_t R = ((int64_t)qt * kAttnWaves + wave) * kTile + (lane & 31);
        const bool live = R < f.rows;
        int64_t i, g;
        a.row(live ? R : 0, i, g);
        const int64_t h = u * a.G + g;
        Query<DP> q;
        load_query(q, f.q + b * a.sq[0] + i * a.sq[1] + h * a.sq[2], live, a.scale, half, (int)a.D);
        Sums<DP> sum;
        sum.clear();
        for (int64_t t = t0, buf = 0; t < t1; t += TS, buf ^= 1) {
            const int64_t tg = t + kg * TPS;  // this group's first tile
            int ek[TPS], ev[TPS];
#pragma unroll
            for (int x = 0; x < TPS; x++) ek[x] = scalar_load(kx + min(tg + x, t1 - 1)), ev[x] = scalar_load(vx + min(tg + x, t1 - 1));
            stage_wait();
            if (t + TS < t1) copy(t + TS, (int)buf ^ 1);
            const char *st = smem + buf * STAGE + kg * TPS * TB;
#pragma unroll
            for (int x = 0; x < TPS; x++) {
                if (tg + x >= t1) break;
                attend(sum, q, st + x * TB + ra, st + (TS + x) * TB + ca, ek[x], ev[x], kr + (tg + x) * kTile, vr + (tg + x) * kTile,
                       tg + x + 1 == nt, (int)min(n - (tg + x) * kTile, (int64_t)kTile) - 4 * half);
            }
        }
        if constexpr (KG > 1) {  // the second group's sums join the first's through LDS
            f4 *const hand = (f4 *)smem + wave * (4 * (DP / 32) + 1) * kWave + lane;
            __syncthreads();  // the last stage has been read
            if (kg) put(sum, hand);
            __syncthreads();
            if (kg) continue;
            join(sum, hand);
        }
        const float l = halves_sum(sum.l);
        if (live && f.splits == 1) {
            // no keys: o is zero
            store_column<false>(f.o + ((b * a.Lq + i) * a.Hq + h) * a.D, sum.o, true, l != 0.0f ? unit_of(sum.U) / l : 0.0f, half, (int)a.D, 0);
            if (f.lse && half == 0)
                f.lse[(b * a.Hq + h) * a.Lq + i] = nt ? fma_(sum.m, kLn2, logf(l)) : -INFINITY;
        } else if (live) {
            const int64_t pr = ((int64_t)split * a.B * a.Hkv + pair) * f.rows + R;
            store_column<true>(f.po + pr * a.D, sum.o, t0 < t1, unit_of(sum.U), half, (int)a.D, 0);
            if (half == 0) f.pm[pr] = f2{t0 < t1 ? sum.m : -INFINITY, l};
        }
    }
}

// ------------------------------------------------------------------------------------------------
// forward of a few rows: single tokens against long caches
// ------------------------------------------------------------------------------------------------
// Bound by reading keys and values once.  LPK lanes hold a key's columns, two 16-byte pieces each, for NR rows of queries at once
// (the query heads that share the keys); each group of LPK lanes keeps its own running maximum, sum and o over the keys that it
// sees, U of them in flight, and the groups, waves and parts are joined at the end.  All in fp32 on the vector unit: 8 rows of
// 128 columns still take less time than the keys' way from memory.  1500 keys, 8 x 12 heads of 64: 16 us (4.5 TB/s) and 4 for the
// join; up to 16384 keys, 16 x 8 heads of 128, four rows: 203 to 206 us (5.5 TB/s).
template <int LPK>
__device__ __forceinline__ float lanes_sum(float v) {  // over LPK neighbours
    v += dpp_f32<kDppXor1>(v, 0.0f);
    v += dpp_f32<kDppXor2>(v, 0.0f);
    if constexpr (LPK >= 8) v += dpp_f32<kDppHalfMirror>(v, 0.0f);
    if constexpr (LPK >= 16) v += dpp_f32<kDppMirror>(v, 0.0f);
    if constexpr (LPK >= 32) v += __shfl_xor(v, 16);
    return v;
}

// piece c of a row: four columns, from the row's first where the piece lies past its end; D4: no piece is cut short
template <bool D4>
__device__ __forceinline__ f4 row_piece(const float *row, int c, int D) {
    if constexpr (D4) {
        return *(const f4u *)(row + (4 * c < D ? 4 * c : 0));
    } else {
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = row[4 * c + e < D ? 4 * c + e : 0];
        return v;
    }
}

// a row whose probabilities sum to zero: without keys `none`, else all its scores are -inf
__device__ __forceinline__ float without_sum(int64_t keys, float none = 0.0f) { return keys ? NAN : none; }
__device__ __forceinline__ float nan_if_infinite(float v) { return v + (v - v); }

template <int NR, int LPK, int U, bool D4>
__global__ __launch_bounds__(kAttnB) void k_attn_token(const FwdArgs f, const float *k, const float *v) {
    constexpr int NG = kWave / LPK, KEYS = kAttnWaves * U * NG;  // groups of a wave; keys of a round
    __shared__ float part[kAttnWaves][NR][8 * LPK];
    __shared__ f2 ml[kAttnWaves][NR];
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane % LPK, grp = lane / LPK, D = (int)a.D;
    for (int64_t w = blockIdx.x; w < f.units; w += gridDim.x) {
        const int64_t pair = w / f.splits, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int split = (int)(w - pair * f.splits);
        const int64_t n = keys_of(a.Lk, f.key_len, b), nt = (n + kTile - 1) / kTile;
        const int64_t j0 = nt * split / f.splits * kTile, j1 = min(n, nt * (split + 1) / f.splits * kTile);
        const float *kb = k + b * a.sk[0] + u * a.sk[2], *vb = v + b * a.sv[0] + u * a.sv[2];
        f4 q[NR][2], o[NR][2];
        float m[NR], l[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            int64_t i, g;
            a.row(r < f.rows ? r : 0, i, g);
            const int64_t h = u * a.G + g;
            const float *row = f.q + b * a.sq[0] + i * a.sq[1] + h * a.sq[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                q[r][x] = row_piece<D4>(row, ln + x * LPK, D) * (a.scale * kLog2e);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * (ln + x * LPK) + e >= D) q[r][x][e] = 0.0f;
                o[r][x] = f4{0.f, 0.f, 0.f, 0.f};
            }
            m[r] = -INFINITY, l[r] = 0.0f;
        }
        float low = 0.0f;  // -inf where a score was: it would count nothing (other scores that are not finite give NaN by themselves)
        for (int64_t j = j0; j < j1; j += KEYS) {
            f4 kk[U][2], vv[U][2];
#pragma unroll
            for (int x = 0; x < U; x++) {
                const int64_t key = min(j + (wave * U + x) * NG + grp, j1 - 1);
                const float *kr = kb + key * a.sk[1], *vr = vb + key * a.sv[1];
#pragma unroll
                for (int y = 0; y < 2; y++) kk[x][y] = row_piece<D4>(kr, ln + y * LPK, D), vv[x][y] = row_piece<D4>(vr, ln + y * LPK, D);
            }
            __builtin_amdgcn_sched_barrier(0);  // all loads are on their way before the first is waited for
            float s[NR][U];
#pragma unroll
            for (int x = 0; x < U; x++) {
                const bool in = j + (wave * U + x) * NG + grp < j1;
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    float t = 0.0f;
#pragma unroll
                    for (int y = 0; y < 2; y++)
#pragma unroll
                        for (int e = 0; e < 4; e++) t = fma_(q[r][y][e], kk[x][y][e], t);
                    t = lanes_sum<LPK>(t);
                    low = __builtin_fminf(low, t);
                    s[r][x] = in ? t : -INFINITY;
                }
            }
#pragma unroll
            for (int r = 0; r < NR; r++) {
                float top = m[r];
#pragma unroll
                for (int x = 0; x < U; x++) top = __builtin_fmaxf(top, s[r][x]);
                // no key yet: the reference stays, and every p is 0
                const float ref = top == -INFINITY ? 0.0f : top, al = __builtin_amdgcn_exp2f(m[r] - ref);
                m[r] = top;
                l[r] *= al;
                o[r][0] *= al;
                o[r][1] *= al;
#pragma unroll
                for (int x = 0; x < U; x++) {
                    const float p = __builtin_amdgcn_exp2f(s[r][x] - ref);
                    l[r] += p;
#pragma unroll
                    for (int y = 0; y < 2; y++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[r][y][e] = fma_(p, vv[x][y][e], o[r][y][e]);
                }
            }
        }
        if (__builtin_expect(__any(low == -INFINITY), 0)) {
            // NaN where a key or the query is not finite; finite ones' scores are what they are (below a float's range: they count
            // nothing).  The wave reads its keys again: a branch in the loop costs every call (1500 keys, 8 x 12 heads of 64: 17.9
            // us, and 15.9).
            for (int64_t j = j0 + wave * U * NG + grp; j < j1; j += KEYS)
                for (int64_t key = j; key < min(j + U * NG, j1); key += NG) {
                    float z = 0.0f;
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const f4 again = row_piece<D4>(kb + key * a.sk[1], ln + y * LPK, D);
#pragma unroll
                        for (int e = 0; e < 4; e++) z = fma_(again[e], 0.0f, z);
                    }
#pragma unroll
                    for (int r = 0; r < NR; r++) l[r] += z;
                }
#pragma unroll
            for (int r = 0; r < NR; r++) {
                float z = 0.0f;
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int e = 0; e < 4; e++) z = fma_(q[r][y][e], 0.0f, z);
                l[r] = lanes_sum<LPK>(l[r] + z) * (1.0f / LPK);  // the group's lanes hold one l: NaN in one of them is all of theirs
            }
        }
        // the wave's groups, then the waves
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float top = m[r];
#pragma unroll
            for (int x = LPK; x < kWave; x *= 2) {
                const float t = __shfl_xor(top, x);
                top = top >= t || top != top ? top : t;  // a NaN stays
            }
            const float al = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[r] - top);
            l[r] *= al;
            o[r][0] *= al;
            o[r][1] *= al;
#pragma unroll
            for (int x = LPK; x < kWave; x *= 2) {
                l[r] += __shfl_xor(l[r], x);
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[r][y][e] += __shfl_xor(o[r][y][e], x);
            }
            m[r] = top;
        }
        __syncthreads();  // the last unit's parts have been read
#pragma unroll
        for (int r = 0; r < NR; r++) {
            if (grp == 0) {
                *(f4 *)&part[wave][r][4 * ln] = o[r][0];
                *(f4 *)&part[wave][r][4 * (ln + LPK)] = o[r][1];
            }
            if (lane == 0) ml[wave][r] = f2{m[r], l[r]};
        }
        __syncthreads();
        for (int x = threadIdx.x; x < NR * 8 * LPK; x += kAttnB) {
            const int r = x / (8 * LPK), d = x - r * 8 * LPK;
            if (r >= f.rows || d >= D) continue;
            float top = -INFINITY;
#pragma unroll
            for (int y = 0; y < kAttnWaves; y++) {
                const float t = ml[y][r].x;
                top = top >= t || top != top ? top : t;
            }
            float sum = 0.0f, total = 0.0f;
#pragma unroll
            for (int y = 0; y < kAttnWaves; y++) {
                const f2 t = ml[y][r];
                const float al = t.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(t.x - top);
                sum = fma_(al, part[y][r][d], sum);
                total = fma_(al, t.y, total);
            }
            if (f.splits == 1) {
                int64_t i, g;
                a.row(r, i, g);
                const int64_t h = u * a.G + g;
                f.o[((b * a.Lq + i) * a.Hq + h) * a.D + d] = nan_if_infinite(total != 0.0f ? sum / total : without_sum(n));
                if (f.lse && d == 0)
                    f.lse[(b * a.Hq + h) * a.Lq + i] = total != 0.0f ? fma_(top, kLn2, logf(total)) : without_sum(n, -INFINITY);
            } else {
                const int64_t pr = ((int64_t)split * a.B * a.Hkv + pair) * f.rows + r;
                f.po[pr * D + d] = sum;
                if (d == 0) f.pm[pr] = f2{top, total};
            }
        }
    }
}

// The splits' parts of a row joined: a part counts by 2^(its reference - the largest).  A wave a row, where there are few: lane s
// has part s's reference and sum, then every lane 64th column.
__global__ __launch_bounds__(kAttnB) void k_attn_join_rows(const AttnArgs a, int64_t rows, int splits, const float *po, const f2 *pm,
                                                      const int *key_len, float *o, float *lse) {
    const int64_t all = a.B * a.Hkv * rows;
    const int lane = threadIdx.x & 63;
    for (int64_t pr = (int64_t)blockIdx.x * kAttnWaves + (threadIdx.x >> 6); pr < all; pr += (int64_t)gridDim.x * kAttnWaves) {
        const int64_t pair = pr / rows, R = pr - pair * rows, b = pair / a.Hkv, u = pair - b * a.Hkv;
        int64_t i, g;
        a.row(R, i, g);
        const int64_t h = u * a.G + g;
        const f2 ml = lane < splits ? pm[lane * all + pr] : f2{-INFINITY, 0.0f};
        const bool nan = __any(ml.x != ml.x);
        const float M = wave_max_nan_skip(ml.x);
        const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
        const float l = wave_sum(w * ml.y);
        const int64_t n = keys_of(a.Lk, key_len, b);
        const float wn = nan ? NAN : l != 0.0f ? w / l : without_sum(n);
        for (int64_t d0 = 0; d0 < a.D; d0 += kWave) {
            const int64_t d = d0 + lane;
            const float *p = po + pr * a.D + (d < a.D ? d : 0);
            float sum = 0.0f;
            for (int s0 = 0; s0 < splits; s0 += 8) {
                float x[8];
#pragma unroll
                for (int s = 0; s < 8; s++) x[s] = p[min(s0 + s, splits - 1) * all * a.D];
#pragma unroll
                for (int s = 0; s < 8; s++) {  // a lane past the parts has weight 0; parts without keys hold nothing that counts
                    const float ws = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wn), s0 + s));
                    sum = ws != 0.0f ? fma_(ws, x[s], sum) : sum;
                }
            }
            if (d < a.D) o[((b * a.Lq + i) * a.Hq + h) * a.D + d] = nan_if_infinite(sum);
        }
        if (lse && lane == 0) lse[(b * a.Hq + h) * a.Lq + i] = l == 0.0f ? without_sum(n, -INFINITY) : fma_(M, kLn2, logf(l));
    }
}

// the same for many rows in up to eight parts: a lane four columns of a row
__global__ __launch_bounds__(kAttnB) void k_attn_join(const AttnArgs a, int64_t rows, int splits, const float *po, const f2 *pm,
                                                      const int *key_len, float *o, float *lse) {
    const int64_t all = a.B * a.Hkv * rows, D4 = (a.D + 3) / 4;
    for (int64_t x = (int64_t)blockIdx.x * kAttnB + threadIdx.x; x < all * D4; x += (int64_t)gridDim.x * kAttnB) {
        const int64_t pr = x / D4, pair = pr / rows, R = pr - pair * rows, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int d = (int)(x - pr * D4) * 4;
        int64_t i, g;
        a.row(R, i, g);
        const int64_t h = u * a.G + g;
        f2 ml[8];
        f4 p[8];
        float M = -INFINITY, l = 0.0f;
        bool nan = false;
#pragma unroll
        for (int s = 0; s < 8; s++) {
            ml[s] = f2{-INFINITY, 0.0f};
            if (s >= splits) continue;
            const int64_t at = s * all + pr;
            ml[s] = pm[at];
            p[s] = a.D >= 4 ? last4(po + at * a.D, d, (int)a.D) : f4{po[at * a.D], po[at * a.D + (a.D > 1)], po[at * a.D + a.D - 1], 0.0f};
        }
#pragma unroll
        for (int s = 0; s < 8; s++) {
            nan = nan || ml[s].x != ml[s].x;
            M = __builtin_fmaxf(M, ml[s].x);
        }
        f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 8; s++) {
            if (ml[s].y == 0.0f) continue;  // a part without keys; scores of NaN leave a NaN as their sum
            const float w = __builtin_amdgcn_exp2f(ml[s].x - M);
            l = fma_(w, ml[s].y, l);
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] = fma_(w, p[s][e], sum[e]);
        }
        const int64_t n = keys_of(a.Lk, key_len, b);
        const float inv = nan ? NAN : l != 0.0f ? 1.0f / l : without_sum(n);
#pragma unroll
        for (int e = 0; e < 4; e++) sum[e] = nan_if_infinite(sum[e] * inv);
        store4(o + ((b * a.Lq + i) * a.Hq + h) * a.D, d, (int)a.D, sum, 0);
        if (lse && d == 0) lse[(b * a.Hq + h) * a.Lq + i] = l == 0.0f ? without_sum(n, -INFINITY) : fma_(M, kLn2, logf(l));
    }
}

// ------------------------------------------------------------------------------------------------
// backward: two kernels, each with its own recomputed scores, so that every gradient is summed in one place and order
// ------------------------------------------------------------------------------------------------
// 2^ the exponent of this lane's row of a packed tile
__device__ __forceinline__ float column_exponent(const int *exps, const float *rows, int64_t tile) {
    const int e = exps[tile];
    return pow2i(own_rows(e) ? exponent_of(e) + (int)rows[tile * kTile + (threadIdx.x & 31)] : e);
}

struct BwdArgs {
    AttnArgs a;
    const char *kp, *vp, *qp, *gp;                 // packed
    const int *kx, *vx, *qx, *gx;                  // their exponents
    const float *kr, *vr, *qr;                     // and their rows'
    const float *stats;
    const int *key_len;
    float *gq, *gk, *gv;                           // the gradients, or the splits' parts [split][...] where there are any
    int64_t rows, qtiles, ktiles, units, part_q, part_k;  // rows of a pair, tiles, units; floats of a part
    int groups, splits;                            // groups of four tiles of a pair, parts the other side is cut into
    int acc_q, acc_k, acc_v;
};

// gk and gv: two waves share 32 keys as columns and go over the tiles of queries.  One takes s = q k^T and p, whose rows are queries,
// hands p over through LDS and sums gv^T += go^T p; the other takes dp = go v^T, makes ds of it and sums gk^T += q^T ds.  Each keeps
// half of the fragments and of the sums, so that two waves fit a SIMD: one's exponentials run under the other's products (128
// columns, 2 x 16 heads on 4, 2048 x 4096: 0.77 ms, and 0.90 with one wave that does both, before the fragments were read ahead; since
// then 0.72 to 0.77 ms from card to card, 1.07 to 1.15 PFLOP/s).  Heads of 33 to 64 columns, four waves a SIMD, spill 37 registers, of
// up to 32 two, of 129 to 256 17.  Padded rows of queries have an infinite log-sum-exp: p = 0.  gv's unit follows p times the gradients' size, as o's
// does in the forward.
template <int DP, int OCC>
__global__ __launch_bounds__(2 * kAttnB, OCC) void k_attn_dkv(const BwdArgs f) {
    constexpr int KS = DP / 16, NT = DP / 32, TB = 128 * DP, LO = 64 * DP, STAGE = 2 * TB + 256;
    constexpr bool REG = DP <= 128;  // keys or values stay in registers, else they are read again for every tile
    // the last products' first fragments are read before p is there, but where that spills (2048 x 2048, 16 heads of 64: 542 us, and 570)
    constexpr bool EARLY = OCC == 2 && DP <= 128;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int which = wave & (kAttnWaves - 1), ds_wave = wave / kAttnWaves;  // tile of keys; 0: p and gv, 1: ds and gk
    const int ra = row_at(lane), ca = col_at(lane);
    const uint32_t lds = lds_address(smem);
    f4 *const hand = (f4 *)(smem + 2 * STAGE) + which * 320 + lane;  // p's registers 4 j .. 4 j + 3 at 64 j
    for (int64_t w = blockIdx.x; w < f.units; w += gridDim.x) {
        const int64_t unit = xcd_unit(w, f.units);
        const int64_t rest = unit / f.groups;
        const int kg = (int)(unit - rest * f.groups);
        const int64_t pair = rest / f.splits, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int split = (int)(rest - pair * f.splits);
        const int64_t n = keys_of(a.Lk, f.key_len, b);
        const int64_t k0 = (int64_t)kg * kAttnWaves + which, key = k0 * kTile + (lane & 31);
        const bool any = (int64_t)kg * kAttnWaves * kTile < n, mine = k0 * kTile < n, live = key < n;
        const int64_t t0 = any ? f.qtiles * split / f.splits : 0, t1 = any ? f.qtiles * (split + 1) / f.splits : 0;
        const int64_t q0 = pair * f.qtiles;
        auto copy = [&](int64_t t, int buf) {
            const uint32_t at = __builtin_amdgcn_readfirstlane(lds + buf * STAGE);
            const int64_t x = (q0 + t) * TB;
            stage_copy<2 * kAttnWaves>(f.qp + x, at, TB / 1024);
            stage_copy<2 * kAttnWaves>(f.gp + x, at + TB, TB / 1024);
            if (threadIdx.x < 16) dma16(f.stats + (q0 + t) * 64 + threadIdx.x * 4, at + 2 * TB);
        };
        __syncthreads();  // the last unit's stages have been read
        if (t0 < t1) copy(t0, 0);
        const int64_t tile = pair * f.ktiles + (mine ? k0 : 0);
        const char *kt = (ds_wave ? f.vp : f.kp) + tile * TB + ra;
        h8 kh[REG ? KS : 1], kl[REG ? KS : 1];
        float ck = 0.0f;
        if (mine) {
            ck = column_exponent(ds_wave ? f.vx : f.kx, ds_wave ? f.vr : f.kr, tile);
            if (!ds_wave) ck *= a.scale * kLog2e;
            if constexpr (REG) {
#pragma unroll
                for (int s = 0; s < KS; s++) kh[s] = row_frag(kt, s), kl[s] = row_frag(kt + LO, s);
            }
        }
        f16x acc[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[t][r] = 0.0f;
        float scale = ds_wave ? 0x1p100f : live ? kNoUnit : -kNoUnit;
        const ScaleParts parts(a.scale);
        for (int64_t t = t0, buf = 0; t < t1; t++, buf ^= 1) {
            const int eg = scalar_load(f.gx + q0 + t), eq = scalar_load(f.qx + q0 + t);
            stage_wait();
            if (t + 1 < t1) copy(t + 1, (int)buf ^ 1);
            const char *st = smem + buf * STAGE;
            const f4 *rows = (const f4 *)(st + 2 * TB) + half;
            const float *qr = f.qr + (q0 + t) * kTile;
            const int xq = exponent_of(eq), xg = exponent_of(eg);
            f16x s;
            if (mine) {
                const char *rt = st + ds_wave * TB + ra;
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = 0.0f;
                steps<KS>([&](int k) { return Pieces{row_frag(rt, k), row_frag(rt + LO, k)}; },
                          [&](int k, const Pieces &x) {
                              s = mfma3(x.hi, x.lo, REG ? kh[k] : row_frag(kt, k), REG ? kl[k] : row_frag(kt + LO, k), s);
                          });
                if (!ds_wave) {
                    if (own_rows(eq)) scale_rows(s, qr);
                    const float c = ck * pow2i(xq), off = live ? first_shift((float)xg, scale) : -INFINITY;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const f4 ls = rows[2 * j];
#pragma unroll
                        for (int e = 0; e < 4; e++) s[4 * j + e] = __builtin_amdgcn_exp2f(fma_(s[4 * j + e], c, off - ls[e]));
                    }
                    hand[256].x = column_unit(s, (float)xg, own_rows(eg), scale, acc);
#pragma unroll
                    for (int j = 0; j < 4; j++) hand[64 * j] = f4{s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]};
                }
            }
            const char *ct = st + (ds_wave ? 0 : TB) + ca;
            const auto turned = [&](int k) { return Pieces{col_frag(ct, k / NT, k % NT), col_frag(ct + LO, k / NT, k % NT)}; };
            Pieces x[3];
            if constexpr (EARLY) x[0] = turned(0), x[1] = turned(1);
            lds_barrier();  // p is there (the next stage's copies stay on their way)
            if (!mine) continue;
            if (ds_wave) {
                const float c = ck * pow2i(xg), kap = parts.times((float)xq - hand[256].x);
                float most = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f4 p = hand[64 * j], de = rows[8 + 2 * j];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = 4 * j + e;
                        s[r] = p[e] * fma_(s[r], c, -de[e]);
                        most = __builtin_fmaxf(most, __builtin_fabsf(s[r]));
                    }
                }
                if (own_rows(eq)) {
                    scale_rows(s, qr);
                    most = largest(s);
                }
                float by;
                if (column_scale(halves_max(most) * __builtin_fabsf(kap), scale, by)) scale_acc(acc, by);
                const float kF = finite_product(kap, scale);
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] *= kF;
            }
            const Split8 y[2] = {split_regs(s, 0), split_regs(s, 8)};
            if constexpr (!EARLY) x[0] = turned(0), x[1] = turned(1);
            steps<2 * NT>(x, turned, [&](int k, const Pieces &v) { acc[k % NT] = mfma3(v.hi, v.lo, y[k / NT].hi, y[k / NT].lo, acc[k % NT]); });
        }
        float *const out = ds_wave ? f.gk : f.gv;
        if (out && key < a.Lk)
            store_column<true>(out + split * f.part_k + ((b * a.Lk + key) * a.Hkv + u) * a.D, acc, live && t0 < t1,
                               ds_wave ? 1.0f / scale : unit_of(scale), half, (int)a.D, ds_wave ? f.acc_k : f.acc_v);
    }
}

// gq: a wave holds 32 rows of queries as columns, as the forward does, and goes over the tiles of keys: s^T = k q^T and
// dp^T = v go^T, then gq^T += k^T ds^T.  The same sizes: 0.61 to 0.64 ms, 0.97 to 1.02 PFLOP/s (the queries' and gradients' fragments
// fill the registers: heads of 97 to 128 columns spill 34, of 129 to 256 113, so fewer reads are ahead than in k_attn_dkv).
template <int DP, int OCC, int KG>
__global__ __launch_bounds__(KG *kAttnB, OCC) void k_attn_dq(const BwdArgs f) {
    constexpr int KS = DP / 16, NT = DP / 32, TB = 128 * DP, LO = 64 * DP, STAGE = 2 * KG * TB;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = wave_all & (kAttnWaves - 1), kg = wave_all / kAttnWaves;  // tile of queries, group of keys
    const int ra = row_at(lane), ca = col_at(lane);
    const uint32_t lds = lds_address(smem);
    for (int64_t w = blockIdx.x; w < f.units; w += gridDim.x) {
        const int64_t unit = xcd_unit(w, f.units);
        const int64_t rest = unit / f.groups;
        const int qg = (int)(unit - rest * f.groups);
        const int64_t pair = rest / f.splits, b = pair / a.Hkv, u = pair - b * a.Hkv;
        const int split = (int)(rest - pair * f.splits);
        const int64_t n = keys_of(a.Lk, f.key_len, b), nt = (n + kTile - 1) / kTile;
        const int64_t t0 = nt * split / f.splits, t1 = nt * (split + 1) / f.splits;
        const int64_t qt = (int64_t)qg * kAttnWaves + wave, R = qt * kTile + (lane & 31);
        const bool mine = qt < f.qtiles;
        const int64_t k0 = pair * f.ktiles;
        auto copy = [&](int64_t t, int buf) {
            const uint32_t at = __builtin_amdgcn_readfirstlane(lds + buf * STAGE);
            const int64_t x = (k0 + t) * TB;
            const int c = (int)min((int64_t)KG, t1 - t) * (TB / 1024);
            stage_copy<KG * kAttnWaves>(f.kp + x, at, c);
            stage_copy<KG * kAttnWaves>(f.vp + x, at + KG * TB, c);
        };
        __syncthreads();  // the last unit's stages have been read
        if (t0 < t1) copy(t0, 0);
        const int64_t tile = pair * f.qtiles + (mine ? qt : 0);
        const char *qp = f.qp + tile * TB + ra, *gp = f.gp + tile * TB + ra;
        h8 qh[KS], ql[KS], gh[KS], gl[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) {
            qh[s] = row_frag(qp, s), ql[s] = row_frag(qp + LO, s);
            gh[s] = row_frag(gp, s), gl[s] = row_frag(gp + LO, s);
        }
        const float cq = column_exponent(f.qx, f.qr, tile) * a.scale * kLog2e, cg = pow2i(exponent_of(f.gx[tile]));
        const float ls = f.stats[tile * 64 + (lane & 31)], de = f.stats[tile * 64 + 32 + (lane & 31)];
        f16x dq[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) dq[t][r] = 0.0f;
        float F = 0x1p100f;
        const ScaleParts parts(a.scale);
        for (int64_t ts = t0, buf = 0; ts < t1; ts += KG, buf ^= 1) {
            const int64_t t = ts + kg;
            const int ek = scalar_load(f.kx + k0 + min(t, t1 - 1)), ev = scalar_load(f.vx + k0 + min(t, t1 - 1));
            stage_wait();
            if (ts + KG < t1) copy(ts + KG, (int)buf ^ 1);
            const char *st = smem + buf * STAGE + kg * TB;
            if (!mine || t >= t1) continue;
            const char *kt = st + ra, *vt = st + KG * TB + ra, *kc = st + ca;
            f16x s, dp;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = dp[r] = 0.0f;
            steps<2 * KS>([&](int k) { return k % 2 ? Pieces{row_frag(vt, k / 2), row_frag(vt + LO, k / 2)} : Pieces{row_frag(kt, k / 2), row_frag(kt + LO, k / 2)}; },
                          [&](int k, const Pieces &x) {
                              if (k % 2) dp = mfma3(x.hi, x.lo, gh[k / 2], gl[k / 2], dp);
                              else s = mfma3(x.hi, x.lo, qh[k / 2], ql[k / 2], s);
                          });
            const auto turned = [&](int k) { return Pieces{col_frag(kc, k / NT, k % NT), col_frag(kc + LO, k / NT, k % NT)}; };
            Pieces x[3];
            if constexpr (DP <= 128) x[0] = turned(0), x[1] = turned(1);  // wider: 1024 x 1024, 8 heads of 256 152 us, and 190 with the spills
            const float *kr = f.kr + (k0 + t) * kTile;
            if (own_rows(max(ek, ev))) {
                if (own_rows(ek)) scale_rows(s, kr);
                if (own_rows(ev)) scale_rows(dp, f.vr + (k0 + t) * kTile);
            }
            const float c = cq * pow2i(exponent_of(ek)), c2 = cg * pow2i(exponent_of(ev));
            const int left = (int)min(n - t * kTile, (int64_t)kTile) - 4 * half;
            float most = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                // roundings of large scores and of their sum may put p above 1: far above, it is held there (a NaN shows in o, so in de)
                float p = __builtin_amdgcn_exp2f(__builtin_fminf(fma_(s[r], c, -ls), 0.0f));
                p = 8 * (r / 4) + r % 4 < left ? p : 0.0f;
                dp[r] = p * fma_(dp[r], c2, -de);
                most = __builtin_fmaxf(most, __builtin_fabsf(dp[r]));
            }
            if (own_rows(ek)) {
                scale_rows(dp, kr);
                most = largest(dp);
            }
            const float kap = parts.times((float)exponent_of(ek));
            float step;
            if (column_scale(halves_max(most) * __builtin_fabsf(kap), F, step)) scale_acc(dq, step);
            const float kF = finite_product(kap, F);
#pragma unroll
            for (int r = 0; r < 16; r++) dp[r] *= kF;
            const Split8 y[2] = {split_regs(dp, 0), split_regs(dp, 8)};
            if constexpr (DP > 128) x[0] = turned(0), x[1] = turned(1);
            steps<2 * NT>(x, turned, [&](int k, const Pieces &v) { dq[k % NT] = mfma3(v.hi, v.lo, y[k / NT].hi, y[k / NT].lo, dq[k % NT]); });
        }
        float by = 1.0f / F;
        if constexpr (KG > 1) {  // the second group's sums are added through LDS
            f4 *const hand = (f4 *)smem + wave * 4 * NT * kWave + lane;
            __syncthreads();  // the last stage has been read
            if (kg) {
#pragma unroll
                for (int d = 0; d < NT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++) hand[(4 * d + j) * kWave] = f4{dq[d][4 * j], dq[d][4 * j + 1], dq[d][4 * j + 2], dq[d][4 * j + 3]} * by;
            }
            __syncthreads();
            if (kg) continue;
#pragma unroll
            for (int d = 0; d < NT; d++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f4 v = hand[(4 * d + j) * kWave];
#pragma unroll
                    for (int e = 0; e < 4; e++) dq[d][4 * j + e] = fma_(dq[d][4 * j + e], by, v[e]);
                }
            by = 1.0f;
        }
        if (R < f.rows) {
            int64_t i, g;
            a.row(R, i, g);
            const int64_t h = u * a.G + g;
            store_column<true>(f.gq + split * f.part_q + ((b * a.Lq + i) * a.Hq + h) * a.D, dq, t0 < t1, by, half, (int)a.D, f.acc_q);
        }
    }
}

// out (+)= the splits' parts [split][n], in order; one or two tensors of one size.  Bound by memory (two parts of 2 x 1.2 million
// floats: 7 us, 4.1 TB/s).
struct SumArgs {
    const float *part[2];
    float *out[2];
    int acc[2];
    int64_t n;
    int splits;
};
__global__ __launch_bounds__(kAttnB) void k_attn_sum(const SumArgs a) {
    const float *part = a.part[blockIdx.y];
    float *out = a.out[blockIdx.y];
    for (int64_t i = (int64_t)blockIdx.x * kAttnB + threadIdx.x; i < a.n; i += (int64_t)gridDim.x * kAttnB) {
        float s = 0.0f;
        for (int k = 0; k < a.splits; k += 8) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = k + e < a.splits ? part[(k + e) * a.n + i] : 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) s += x[e];
        }
        out[i] = a.acc[blockIdx.y] ? out[i] + s : s;
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
    const int64_t G = Hq / Hkv;
    a = {B, Lq, Lk, Hq, Hkv, D, G, {sq[0], sq[1], sq[2]}, {sk[0], sk[1], sk[2]}, {sv[0], sv[1], sv[2]}, scale, G * Lq <= INT32_MAX, IntDiv((uint32_t)G)};
    return NC_HIP_OK;
}

}  // namespace nchip

using namespace nchip;

namespace nchip {

static int padded(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256; }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// dispatch over the padded columns
#define NC_ATTN_DP(dp, ...)                                  \
    do {                                                     \
        if ((dp) == 32) { constexpr int DP = 32; __VA_ARGS__; }         \
        else if ((dp) == 64) { constexpr int DP = 64; __VA_ARGS__; }    \
        else if ((dp) == 96) { constexpr int DP = 96; __VA_ARGS__; }    \
        else if ((dp) == 128) { constexpr int DP = 128; __VA_ARGS__; }  \
        else { constexpr int DP = 256; __VA_ARGS__; }                   \
    } while (0)

// Parts so that there are `want` workgroups, 64 parts at most, of at least four tiles each, or sixteen where the whole ones already
// fill half the CUs: joining costs as much as it gains there, or more (1024 rows, 16 heads of 128, forward, whole and in two parts:
// against 300 keys 33 and 41 us, 600 keys 46 both, 1000 keys 55 both; 1000 x 400, 4 x 6 heads of 256 77 and 110).
static int attn_splits(int64_t whole, int64_t tiles, int64_t want) {
    int64_t s = whole ? want / whole : 1;
    s = std::min(s, tiles / (whole >= kPlanCUs / 2 ? 16 : 4));
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

// Two groups of waves that share a workgroup's rows and take every other tile of keys, joined through LDS: where workgroups of four
// waves would leave most SIMDs with one wave or none.  (1024 x 1024, 32 heads of 128: forward 78 us, and 90 with one group, forward
// and backward 300 and 335; 8 heads of 64: 95 and 99.)
static bool key_groups(int64_t whole, int64_t tiles, int DP) { return DP <= 128 && whole <= kPlanCUs && tiles >= 4; }

// Rows of a pair that k_attn_token takes; more go through the pack, which costs the keys' bytes twice more.  8 x 8 heads of keys of 128
// columns, four rows, eight, and 9 to 32: 4096 keys 61, 78 and 169 us, 16384 keys 204, 220 and 652 (four and eight rows packed: 169
// and 647).
constexpr int64_t kTokenRows = 8;

struct FwdPlan {
    bool token, few;  // k_attn_token; few keys
    int DP, qtiles, splits, kg;  // kg: groups of waves that share a workgroup's keys
    int64_t rows, tiles, pairs, units;
    size_t kp, vp, kx, vx, kr, vr, po, pm, total;  // offsets into the workspace
};

static FwdPlan fwd_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv, int64_t D) {
    FwdPlan p{};
    p.DP = padded(D);
    p.rows = Hq / Hkv * Lq;
    p.pairs = B * Hkv;
    p.tiles = (Lk + kTile - 1) / kTile;
    p.qtiles = (int)((p.rows + kAttnWaves * kTile - 1) / (kAttnWaves * kTile));
    p.token = p.rows <= kTokenRows;
    p.few = !p.token && Lk <= short_keys_fwd(p.DP);
    if (p.few) {
        // two workgroups a CU with a tile of queries for each of their eight waves, or one a CU with two tiles at least (58 rows x
        // 2 heads against 96 keys, heads of 128, four sequences: 30 us with eight tiles a workgroup, 20 with two)
        const int64_t tiles = (p.rows + kTile - 1) / kTile;
        const auto cut = [&](int64_t units, int64_t least) { return std::min(p.pairs ? units / p.pairs : 1, tiles / least); };
        const int64_t parts = std::max(cut(2 * kPlanCUs, 8), cut(kPlanCUs, 2));
        p.splits = (int)(parts < 1 ? 1 : parts);
        p.units = p.pairs * p.splits;
        return p;
    }
    if (p.token) p.qtiles = 1;
    const int64_t whole = p.pairs * p.qtiles;
    p.kg = !p.token && key_groups(whole, p.tiles, p.DP);
    p.splits = attn_splits(whole, p.tiles, (p.token ? 8 : p.kg ? 1 : 2) * kPlanCUs);
    p.units = whole * p.splits;
    const size_t pt = (size_t)(p.pairs * p.tiles);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up256(bytes);
        return here;
    };
    if (!p.token) {
        p.kp = take(pt * tile_bytes(p.DP));
        p.vp = take(pt * tile_bytes(p.DP));
        p.kx = take(pt * 4);
        p.vx = take(pt * 4);
        p.kr = take(pt * 4 * kTile);
        p.vr = take(pt * 4 * kTile);
    }
    if (p.splits > 1) {
        p.po = take((size_t)p.splits * p.pairs * p.rows * D * 4);
        p.pm = take((size_t)p.splits * p.pairs * p.rows * 8);
    }
    p.total = at;
    return p;
}

static unsigned attn_grid(int64_t units) { return (unsigned)(units < kAttnGrid ? units : kAttnGrid); }

template <class F, class A>
static void attn_launch(F *kernel, int64_t units, size_t lds, hipStream_t st, const A &args, int threads = kAttnB) {
    if (lds > 65536) (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL(kernel, dim3(attn_grid(units)), dim3(threads), lds, st, args);
}

template <int NR, int LPK>
static void token_launch2(const FwdArgs &f, const float *k, const float *v, hipStream_t st) {
    constexpr int U = NR <= 4 ? 4 : 2;
    if (f.a.D % 4 == 0) hipLaunchKernelGGL((k_attn_token<NR, LPK, U, true>), dim3(attn_grid(f.units)), dim3(kAttnB), 0, st, f, k, v);
    else hipLaunchKernelGGL((k_attn_token<NR, LPK, U, false>), dim3(attn_grid(f.units)), dim3(kAttnB), 0, st, f, k, v);
}
template <int NR>
static void token_launch1(const FwdArgs &f, const float *k, const float *v, hipStream_t st) {
    if (f.a.D <= 32) token_launch2<NR, 4>(f, k, v, st);
    else if (f.a.D <= 64) token_launch2<NR, 8>(f, k, v, st);
    else if (f.a.D <= 128) token_launch2<NR, 16>(f, k, v, st);
    else token_launch2<NR, 32>(f, k, v, st);
}
static void token_launch(const FwdArgs &f, const float *k, const float *v, hipStream_t st) {
    if (f.rows == 1) token_launch1<1>(f, k, v, st);
    else if (f.rows == 2) token_launch1<2>(f, k, v, st);
    else if (f.rows <= 4) token_launch1<4>(f, k, v, st);
    else token_launch1<8>(f, k, v, st);
}

static void pack_launch(PackArgs &p, int64_t pairs, int DP, hipStream_t st) {
    p.total = 0;
    for (int j = 0; j < p.jobs; j++) {
        p.job[j].first = p.total;
        p.total += pairs * p.job[j].tiles;
    }
    if (!p.total) return;
    NC_ATTN_DP(DP, hipLaunchKernelGGL((k_attn_pack<DP>), dim3(attn_grid(p.total)), dim3(kAttnB), 0, st, p));
}

}  // namespace nchip

extern "C" NC_HIP_API size_t nc_hip_cross_attention_fwd_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv,
                                                                  int64_t D) {
    if (B <= 0 || Lq <= 0 || Lk < 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
    return fwd_plan(B, Lq, Lk, Hq, Hkv, D).total;
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
    const FwdPlan p = fwd_plan(B, Lq, Lk, Hq, Hkv, D);
    if (p.total && (!ws || ws_bytes < p.total || (uintptr_t)ws % 16))
        return set_error(NC_HIP_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, 16-byte aligned", what, p.total);
    hipStream_t st = as_stream(stream);
    char *const w = (char *)ws;
    if (p.few) {
        const ShortFwd f{a, q, k, v, key_len, o, lse, p.rows, (p.rows + kTile - 1) / kTile, p.units, (int)p.tiles, p.splits};
        short_fwd(f, p.DP, st);
        return check_launch(what);
    }
    if (Lk && !p.token) {
        PackArgs pk{};
        pk.a = a, pk.key_len = key_len, pk.jobs = 2;
        pk.job[0] = {k, sk[0], sk[1], sk[2], Lk, p.tiles, 1, w + p.kp, (int *)(w + p.kx), (float *)(w + p.kr), 0, nullptr, nullptr, nullptr};
        pk.job[1] = {v, sv[0], sv[1], sv[2], Lk, p.tiles, 1, w + p.vp, (int *)(w + p.vx), (float *)(w + p.vr), 0, nullptr, nullptr, nullptr};
        pack_launch(pk, p.pairs, p.DP, st);
    }
    FwdArgs f{a, q, w + p.kp, w + p.vp, (int *)(w + p.kx), (int *)(w + p.vx), (float *)(w + p.kr), (float *)(w + p.vr), key_len, o, lse, (float *)(w + p.po), (f2 *)(w + p.pm),
              p.rows, p.tiles, p.units, p.qtiles, p.splits};
    if (p.token)
        token_launch(f, k, v, st);
    else
        NC_ATTN_DP(p.DP, constexpr int TPS = DP <= 64 ? 2 : 1; constexpr int OCC = DP <= 128 ? 2 : 1; constexpr int KG = DP <= 128 ? 2 : 1;
                   if (p.kg) attn_launch(&k_attn_fwd<DP, 1, OCC, KG>, p.units, 2 * 2 * KG * 128 * DP, st, f, KG * kAttnB);
                   else attn_launch(&k_attn_fwd<DP, TPS, OCC, 1>, p.units, 2 * 2 * TPS * 128 * DP, st, f));
    // a wave a row while that fills the chip at most twice over, or for more than eight parts
    const int64_t all = p.pairs * p.rows, pieces = all * ((D + 3) / 4);
    if (p.splits > 8 || (p.splits > 1 && all <= 16 * kPlanCUs))
        hipLaunchKernelGGL(k_attn_join_rows, dim3(attn_grid((all + kAttnWaves - 1) / kAttnWaves)), dim3(kAttnB), 0, st, a, p.rows, p.splits, f.po, f.pm, key_len, o, lse);
    else if (p.splits > 1)
        hipLaunchKernelGGL(k_attn_join, dim3(attn_grid((pieces + kAttnB - 1) / kAttnB)), dim3(kAttnB), 0, st, a, p.rows, p.splits, f.po, f.pm, key_len, o, lse);
    return check_launch(what);
}

namespace nchip {

struct BwdPlan {
    bool few, kg;  // few keys; two groups of waves share a workgroup's keys for gq
    int DP, qgroups, kgroups, qsplits, ksplits;  // splits of the keys for gq, of the queries for gk and gv
    int64_t rows, qtiles, ktiles, pairs, nq, nk;
    size_t kp, vp, qp, gp, kx, vx, qx, gx, kr, vr, qr, stats, pq, pk, pv, total;
};

static BwdPlan bwd_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv, int64_t D) {
    BwdPlan p{};
    p.DP = padded(D);
    p.rows = Hq / Hkv * Lq;
    p.pairs = B * Hkv;
    p.qtiles = (p.rows + kTile - 1) / kTile;
    p.ktiles = (Lk + kTile - 1) / kTile;
    p.qgroups = (int)((p.qtiles + kAttnWaves - 1) / kAttnWaves);
    p.kgroups = (int)((p.ktiles + kAttnWaves - 1) / kAttnWaves);
    p.kg = key_groups(p.pairs * p.qgroups, p.ktiles, p.DP);
    p.qsplits = attn_splits(p.pairs * p.qgroups, p.ktiles, kPlanCUs * (p.DP <= 128 && !p.kg ? 2 : 1));
    p.ksplits = attn_splits(p.pairs * p.kgroups, p.qtiles, kPlanCUs * (p.DP <= 64 ? 2 : 1));
    p.nq = B * Lq * Hq * D;
    p.nk = B * Lk * Hkv * D;
    p.few = Lk <= short_keys_bwd(p.DP);
    if (p.few) {  // a workgroup of eight waves a CU, or two of four, with two tiles of queries at least
        int64_t parts = p.pairs ? (p.ktiles <= 4 && p.DP <= 64 ? 2 : 1) * kPlanCUs / p.pairs : 1;
        if (parts > p.qtiles / 2) parts = p.qtiles / 2;
        p.ksplits = (int)(parts < 1 ? 1 : parts);
    }
    size_t at = 0;
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += up256((size_t)bytes);
        return here;
    };
    const int64_t q = p.few ? 0 : p.pairs * p.qtiles, k = p.few ? 0 : p.pairs * p.ktiles, tb = tile_bytes(p.DP);
    p.kp = take(k * tb), p.vp = take(k * tb), p.qp = take(q * tb), p.gp = take(q * tb);
    p.kx = take(k * 4), p.vx = take(k * 4), p.qx = take(q * 4), p.gx = take(q * 4), p.stats = take(q * 256);
    p.kr = take(k * 4 * kTile), p.vr = take(k * 4 * kTile), p.qr = take(q * 4 * kTile);
    if (p.qsplits > 1 && !p.few) p.pq = take(p.qsplits * p.nq * 4);
    if (p.ksplits > 1) p.pk = take(p.ksplits * p.nk * 4), p.pv = take(p.ksplits * p.nk * 4);
    p.total = at;
    return p;
}

static void sum_launch(int64_t n, int splits, const float *p0, float *o0, int acc0, const float *p1, float *o1, int acc1, hipStream_t st) {
    SumArgs s{{o0 ? p0 : p1, p1}, {o0 ? o0 : o1, o1}, {o0 ? acc0 : acc1, acc1}, n, splits};
    hipLaunchKernelGGL(k_attn_sum, dim3(attn_grid((n + kAttnB - 1) / kAttnB), o0 && o1 ? 2 : 1), dim3(kAttnB), 0, st, s);
}

}  // namespace nchip

extern "C" NC_HIP_API size_t nc_hip_cross_attention_bwd_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv,
                                                                  int64_t D) {
    if (B <= 0 || Lq < 0 || Lk < 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
    return bwd_plan(B, Lq, Lk, Hq, Hkv, D).total;
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
    const bool want_q = gq && Lq, want_k = (gk || gv) && Lk;
    if (!want_q && !want_k) return NC_HIP_OK;
    const BwdPlan p = bwd_plan(B, Lq, Lk, Hq, Hkv, D);
    if (p.total && (!ws || ws_bytes < p.total || (uintptr_t)ws % 16))
        return set_error(NC_HIP_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, 16-byte aligned", what, p.total);
    hipStream_t st = as_stream(stream);
    char *const w = (char *)ws;
    if (p.few) {
        const bool cut = p.ksplits > 1;
        ShortBwd f{a, q, k, v, key_len, o, lse, go, want_q ? gq : nullptr, cut && gk ? (float *)(w + p.pk) : gk, cut && gv ? (float *)(w + p.pv) : gv,
                   p.rows, p.qtiles, p.pairs * p.ksplits, p.nk, p.ksplits, acc_q, cut ? 0 : acc_k, cut ? 0 : acc_v};
        short_bwd(f, p.DP, st);
        if (cut && want_k) sum_launch(p.nk, p.ksplits, f.gk, gk, acc_k, f.gv, gv, acc_v, st);
        return check_launch(what);
    }
    BwdArgs f{};
    f.a = a;
    f.kp = w + p.kp, f.vp = w + p.vp, f.qp = w + p.qp, f.gp = w + p.gp;
    f.kx = (int *)(w + p.kx), f.vx = (int *)(w + p.vx), f.qx = (int *)(w + p.qx), f.gx = (int *)(w + p.gx);
    f.kr = (float *)(w + p.kr), f.vr = (float *)(w + p.vr), f.qr = (float *)(w + p.qr);
    f.stats = (float *)(w + p.stats);
    f.key_len = key_len;
    f.rows = p.rows, f.qtiles = p.qtiles, f.ktiles = p.ktiles;
    PackArgs pk{};
    pk.a = a, pk.key_len = key_len;
    if (Lk) {
        pk.job[pk.jobs++] = {k, sk[0], sk[1], sk[2], Lk, p.ktiles, 1, w + p.kp, (int *)(w + p.kx), (float *)(w + p.kr), 0, nullptr, nullptr, nullptr};
        pk.job[pk.jobs++] = {v, sv[0], sv[1], sv[2], Lk, p.ktiles, 1, w + p.vp, (int *)(w + p.vx), (float *)(w + p.vr), 0, nullptr, nullptr, nullptr};
    }
    if (Lq) {
        pk.job[pk.jobs++] = {q, sq[0], sq[1], sq[2], p.rows, p.qtiles, 0, w + p.qp, (int *)(w + p.qx), (float *)(w + p.qr), 0, nullptr, nullptr, nullptr};
        pk.job[pk.jobs++] = {go, Lq * Hq * D, Hq * D, D, p.rows, p.qtiles, 0, w + p.gp, (int *)(w + p.gx), nullptr, 0, o, lse, (float *)(w + p.stats)};
    }
    pack_launch(pk, p.pairs, p.DP, st);
    if (want_q) {
        const bool cut = p.qsplits > 1;
        f.gq = cut ? (float *)(w + p.pq) : gq;
        f.acc_q = cut ? 0 : acc_q;
        f.part_q = p.nq, f.groups = p.qgroups, f.splits = p.qsplits;
        f.units = p.pairs * p.qgroups * p.qsplits;
        NC_ATTN_DP(p.DP, constexpr int OCC = DP <= 128 ? 2 : 1; constexpr int KG = DP <= 128 ? 2 : 1;
                   if (p.kg) attn_launch(&k_attn_dq<DP, OCC, KG>, f.units, 2 * 2 * KG * 128 * DP, st, f, KG * kAttnB);
                   else attn_launch(&k_attn_dq<DP, OCC, 1>, f.units, 2 * 2 * 128 * DP, st, f));
        if (cut) sum_launch(p.nq, p.qsplits, f.gq, gq, acc_q, nullptr, nullptr, 0, st);
    }
    if (want_k) {
        const bool cut = p.ksplits > 1;
        f.gk = cut && gk ? (float *)(w + p.pk) : gk;
        f.gv = cut && gv ? (float *)(w + p.pv) : gv;
        f.acc_k = cut ? 0 : acc_k;
        f.acc_v = cut ? 0 : acc_v;
        f.part_k = p.nk, f.groups = p.kgroups, f.splits = p.ksplits;
        f.units = p.pairs * p.kgroups * p.ksplits;
        NC_ATTN_DP(p.DP, constexpr int OCC = DP <= 64 ? 4 : 2;
                   attn_launch(&k_attn_dkv<DP, OCC>, f.units, 2 * (2 * 128 * DP + 256) + 4 * 320 * 16, st, f, 2 * kAttnB));
        if (cut) sum_launch(p.nk, p.ksplits, f.gk, gk, acc_k, f.gv, gv, acc_v, st);
    }
    return check_launch(what);
}
