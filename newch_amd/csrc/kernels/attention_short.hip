// Attention to few keys (a padded text, the patches of a small image): a head's keys fit a workgroup, which splits them itself
// instead of reading them packed.  D padded to DP columns, at most 16384 / DP keys forward; backward at most 256 in heads of up to
// 64 columns and 128 in heads of up to 128.
#include "attention.hpp"
#include "attention_short.hpp"

#include <math.h>

namespace nchip {

// A wave reads 32 rows of `src` (from `row0` on, n in all, `step` floats apart): the tile's exponent, with kOwnRows added where its rows
// have their own, and this lane's row's; and splits them into LDS.
template <int DP>
__device__ __forceinline__ int tile_load(const float *src, int64_t step, int row0, int n, int D, float (&x)[DP / 16][8], int &own) {
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
    most = halves_max(most);
    const bool unlike = rows_unlike(most, top);
    own = unlike ? row_exponent(most, ex) : ex;
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
// heads of 64: 38 to 43 us for 136 MB (3.2 to 3.6 TB/s) -- a wave reads its rows, multiplies and stores in turn, and the three
// waves of a SIMD do not cover all of it.  Heads of 97 to 128 columns spill seven registers.
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
            const int at = val ? f.tiles + k : k, e = tile_load<DP>(src, val ? a.sv[1] : a.sk[1], k * kTile, n, (int)a.D, x, er);
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
                       rows + t * kTile, rows + (f.tiles + t) * kTile, t + 1 == nt, min(n - t * kTile, kTile) - 4 * half);
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
// and split it, a piece a lane: piece p is columns 8 (p / 32) .. + 7 of row p % 32.  Gradients of unlike rows have a scale for each row,
// which goes into the rows' statistics as in PackJob; queries of unlike rows are taken in several passes, each with rows that are alike and
// zeros in the others' places.
template <int DP, int W>
struct FeedTables {  // in LDS
    float stats[64];                // the rows' log2-sum-exps (infinite: not in this pass) and go . o, as in PackJob
    float dots[DP / 8][kTile];      // scratch
    float tops[2][DP / 8][kTile];   // the largest of the pieces of queries, of gradients
    float red[2][W];
    int several[4];                 // a row is loose, rows are unlike
};
struct FeedPass {
    int eq, eg;       // exponents of the tile's queries and gradients
    uint32_t rows;    // that are in this pass; none: rows are unlike, or one is loose
    bool last, hold;  // the tile's last; a row may be loose
};
template <int DP, int W>
struct Feed {
    static constexpr int UNITS = 4 * DP;
    static_assert(UNITS <= W * kWave, "a piece a lane");
    float q[8], go[8], o[8], lse;

    __device__ __forceinline__ void fetch(const ShortBwd &f, int64_t b, int64_t u, int64_t t) {
        const AttnArgs &a = f.a;
        const int D = (int)a.D, p = threadIdx.x;
        const int64_t R = t * kTile + (p & 31);
        const bool in = p < UNITS && R < f.rows;
        int64_t i, g;
        a.row(in ? R : 0, i, g);
        const int64_t h = u * a.G + g;
        const int64_t at = ((b * a.Lq + i) * a.Hq + h) * D;
        const int d = in ? 8 * (p >> 5) : D;  // nothing is read from column D on
        load8(f.q + b * a.sq[0] + i * a.sq[1] + h * a.sq[2], d, D, q);
        load8(f.go + at, d, D, go);
        load8(f.o + at, d, D, o);
        lse = p < 32 && in ? f.lse[(b * a.Hq + h) * a.Lq + i] * kLog2e : INFINITY;
    }

    // this lane's piece under 2^ex, or zeros
    static __device__ __forceinline__ void put(const float (&x)[8], int ex, bool in, char *tile) {
        const int p = threadIdx.x, c = p >> 5, at = 16 * (32 * c + ((p & 31) ^ (4 * (c & 1))));
        if (p >= UNITS) return;
        const float by = pow2i(-ex);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = in ? x[e] * by : 0.0f;
        const Split8 s = split8(y);
        *(h8 *)(tile + at) = s.hi, *(h8 *)(tile + 64 * DP + at) = s.lo;
    }
    // the largest of this lane's row; all lanes of the workgroup
    static __device__ __forceinline__ float of_row(float piece, FeedTables<DP, W> &t) {
        const int p = threadIdx.x;
        __syncthreads();  // dots have been read
        if (p < UNITS) t.dots[p >> 5][p & 31] = piece;
        __syncthreads();
        float most = t.dots[0][p & 31];
        for (int c = 1; c < DP / 8; c++) most = __builtin_fmaxf(most, t.dots[c][p & 31]);
        return most;
    }

    // into the tiles qs and gs, and the tables
    __device__ __forceinline__ FeedPass split(char *qs, char *gs, FeedTables<DP, W> &t) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), p = threadIdx.x;
        const float mq = abs_max(q, 0.0f), mg = abs_max(go, 0.0f);
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) dot = fma_(go[e], o[e], dot);
        if (p < UNITS) t.dots[p >> 5][p & 31] = dot, t.tops[0][p >> 5][p & 31] = mq, t.tops[1][p >> 5][p & 31] = mg;
        float tq = wave_max_nan_skip(mq), tg = wave_max_nan_skip(mg);
        if (lane == 0) t.red[0][wave] = tq, t.red[1][wave] = tg;
        __syncthreads();
        tq = t.red[0][0], tg = t.red[1][0];
#pragma unroll
        for (int x = 1; x < W; x++) tq = __builtin_fmaxf(tq, t.red[0][x]), tg = __builtin_fmaxf(tg, t.red[1][x]);
        const int eq = tile_exponent(tq), eg = tile_exponent(tg);
        // the first wave sums the rows' pieces of go . o, the second takes the rows' largest: queries' in the one half, gradients' in the other
        float row[DP / 8];
        if (wave < 2) {
            const float *const from = (wave == 0 ? t.dots[0] : t.tops[lane >> 5][0]) + (lane & 31);
#pragma unroll
            for (int c = 0; c < DP / 8; c++) row[c] = from[c * kTile];
        }
        put(q, eq, true, qs);
        put(go, eg, true, gs);
        if (wave == 0) {
            float d = row[0];
#pragma unroll
            for (int c = 1; c < DP / 8; c++) d += row[c];
            if (lane < kTile) t.stats[lane] = lse, t.stats[32 + lane] = d;
            const bool some = __any(loose(lse));
            if (lane == 0) t.several[0] = some;
        } else if (wave == 1) {
            float most = row[0];
#pragma unroll
            for (int c = 1; c < DP / 8; c++) most = __builtin_fmaxf(most, row[c]);
            const bool some = rows_unlike(most, lane < kTile ? tq : tg);
            if (lane == 0) t.several[1] = some;
        }
        __syncthreads();
        const int several = __builtin_amdgcn_readfirstlane(t.several[0] | t.several[1]);
        return {eq, eg, several ? 0u : ~0u, true, false};
    }

    // the same for those rows of `todo` whose queries are like the largest, gradients by their rows' own scales
    __device__ __forceinline__ FeedPass split_rows(char *qs, char *gs, FeedTables<DP, W> &t, uint32_t todo) {
        const int p = threadIdx.x;
        const float row_q = of_row(abs_max(q, 0.0f), t), row_g = of_row(abs_max(go, 0.0f), t);
        bool in = (todo >> (p & 31)) & 1;
        const float tq = wave_max_nan_skip(in ? row_q : 0.0f);
        in = in && (row_q == 0.0f || row_q >= tq * kAlike);
        const int eq = tile_exponent(tq), eg = tile_exponent(wave_max_nan_skip(in ? row_g : 0.0f)), own = row_exponent(row_g, eg);
        const uint32_t rows = (uint32_t)__ballot(in);
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) dot = fma_(go[e], o[e], dot);
        __syncthreads();  // dots have been read
        if (p < UNITS) t.dots[p >> 5][p & 31] = dot;
        put(q, eq, in, qs);
        put(go, own, in, gs);
        __syncthreads();
        if (p < kTile) {
            float d = t.dots[0][p];
            for (int c = 1; c < DP / 8; c++) d += t.dots[c][p];
            t.stats[p] = in ? lse - (float)(own - eg) : INFINITY;
            t.stats[32 + p] = in ? d * pow2i(eg - own) : 0.0f;
        }
        __syncthreads();
        return {eq, eg, rows, (todo & ~rows) == 0, true};
    }

    // The next pass, of tile t, with the next tile's rows on their way.  The rows of a tile that is cut again are read again: kept, they would
    // hold up the next tile's (4096 x 77, 4 x 16 heads of 64, rows alike: 136 us, and 148), or cost the passes' registers.
    __device__ __forceinline__ FeedPass pass(const ShortBwd &f, int64_t b, int64_t u, int64_t &t, int64_t t1, uint32_t &todo, char *qs, char *gs,
                                             FeedTables<DP, W> &tables) {
        FeedPass r;
        r.rows = 0;
        if (todo == ~0u) {
            r = split(qs, gs, tables);
            if (t + 1 < t1) fetch(f, b, u, t + 1);
        }
        if (__builtin_expect(r.rows == 0, 0)) {
            fetch(f, b, u, t);
            r = split_rows(qs, gs, tables, todo);
            todo = r.last ? ~0u : todo & ~r.rows;
            if (r.last && t + 1 < t1) fetch(f, b, u, t + 1);
        }
        t += r.last;
        return r;
    }
};

// The largest of each of a result's 16 rows over its 32 columns, a lane's times f, in magnitude: lane l gets register (l / 2) % 16's.
// Each step halves the registers and the lanes that have to be joined.
__device__ __forceinline__ float largest_of_rows(const f16x &x, float f) {
    const int lane = threadIdx.x & 63;
    float a[8];
#pragma unroll
    for (int r = 0; r < 8; r++) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_int(x[r] * f), __float_as_int(x[r + 8] * f), false, false);
        a[r] = __builtin_fmaxf(__builtin_fabsf(__int_as_float(s[0])), __builtin_fabsf(__int_as_float(s[1])));
    }
    const auto halve = [&](int n, bool upper, auto from) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (r >= n) break;
            const float keep = upper ? a[r + n] : a[r], give = upper ? a[r] : a[r + n];
            a[r] = __builtin_fmaxf(keep, from(give));
        }
    };
    halve(4, lane & 8, [](float v) { return dpp_f32<kDppRor8>(v, 0.0f); });
    halve(2, lane & 4, [](float v) { return dpp_f32<kDppHalfMirror>(v, 0.0f); });
    halve(1, lane & 2, [](float v) { return dpp_f32<kDppXor2>(v, 0.0f); });
    return __builtin_fmaxf(a[0], dpp_f32<kDppXor1>(a[0], 0.0f));
}

// A wave's ds (32 rows of queries as a result's rows, its keys the columns), a lane's times f, in two pieces as a packed tile of 32 rows
// of keys, whose columns are the rows of queries.  Each row of queries has a scale of its own, its gradients being small or large with
// the values and gradients that it meets: scale [2][32], 2^(its exponent - 14), and its inverse less the 14.
__device__ __forceinline__ void put_ds(const f16x &ds, float f, char *tile, float *scale) {
    const int lane = threadIdx.x & 63, half = lane >> 5, r = (lane >> 1) & 15;
    const int er = tile_exponent(largest_of_rows(ds, f)), at = 8 * (r / 4) + 4 * half + r % 4;
    scale[at] = pow2i(max(er - 14, -126));
    scale[kTile + at] = pow2i(-er);
    asm volatile("" ::: "memory");  // a wave's LDS accesses are in order
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        float y[8];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const f4 inv = *(const f4 *)(scale + kTile + 4 * half + 8 * (j + h));
#pragma unroll
            for (int e = 0; e < 4; e++) y[4 * h + e] = ds[4 * (j + h) + e] * f * inv[e];
        }
        const Split8 s = split8(y);
        char *const to = tile + 512 * j + 8 * half;
        const int r0 = 16 * (lane & 31), r1 = r0 ^ 64;
        *(h4 *)(to + r0) = s.hi.lo, *(h4 *)(to + 512 + r1) = s.hi.hi;
        *(h4 *)(to + 2048 + r0) = s.lo.lo, *(h4 *)(to + 2560 + r1) = s.lo.hi;
    }
}

// gq^T = k^T ds^T over all nt tiles of keys, blocks of 16 columns and 16 rows of queries dealt over the W waves; rows
// [nt][2][32] and keys_by [nt]: the scales of a tile's ds, and of its keys; in: the rows of queries that are stored
template <int DP, int W>
__device__ __forceinline__ void gq_blocks(const ShortBwd &f, int64_t b, int64_t u, int64_t t, int nt, const char *keys, const char *dss, const float *rows,
                                          const float *keys_by, uint32_t in) {
    constexpr int TB = 128 * DP, LO = 64 * DP, BLOCKS = DP / 8, PW = (BLOCKS + W - 1) / W;
    const AttnArgs &a = f.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ta = turned_at(lane);
    f4 sum[PW];
#pragma unroll
    for (int x = 0; x < PW; x++) sum[x] = f4{0.f, 0.f, 0.f, 0.f};
    for (int y = 0; y < nt; y++) {
        const float by_keys = keys_by[y];
#pragma unroll
        for (int x = 0; x < PW; x++) {
            const int block = wave + x * W, c = block % (DP / 16), r = block / (DP / 16);
            if (BLOCKS % W && block >= BLOCKS) break;
            const char *const kc = keys + y * TB + 1024 * c + ta, *const dc = dss + y * kDsTile + 1024 * r + ta;
            const char *const kc2 = keys + y * TB + 1024 * c + (ta ^ 64), *const dc2 = dss + y * kDsTile + 1024 * r + (ta ^ 64);
            const h8 ah = turned16(kc, kc2), al = turned16(kc + LO, kc2 + LO), bh = turned16(dc, dc2), bl = turned16(dc + 2048, dc2 + 2048);
            const float by = rows[2 * y * kTile + 16 * r + (lane & 15)];
            f4 v = {0.f, 0.f, 0.f, 0.f};
            v = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, v, 0, 0, 0);
            v = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, v, 0, 0, 0);
            v = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, v, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) sum[x][e] = fma_(v[e] * by, by_keys, sum[x][e]);
        }
    }
#pragma unroll
    for (int x = 0; x < PW; x++) {
        const int block = wave + x * W, c = block % (DP / 16), r = block / (DP / 16);
        const int64_t R = t * kTile + 16 * r + (lane & 15);
        if (block >= BLOCKS || R >= f.rows || !((in >> (16 * r + (lane & 15))) & 1)) continue;
        int64_t i, g;
        a.row(R, i, g);
        store4(f.gq + ((b * a.Lq + i) * a.Hq + u * a.G + g) * a.D, 16 * c + 4 * (lane >> 4), (int)a.D, sum[x], f.acc_q);
    }
}

// Backward in one pass over the queries: every wave holds 32 keys, the workgroup splits a tile of queries and output gradients
// (the next one's on their way meanwhile), and each wave takes its part of gk and gv as k_attn_dkv does.  It leaves its ds in LDS,
// and the waves share the blocks of gq^T = k^T ds^T over all keys.  The same sizes: 105 to 108 us, of which the look
// at the rows, the units of gv's columns and the scales of ds's rows are 8, and 23 more with every wave's part of gq added in LDS; memory
// would take 57.  A tile's steps follow each other (read, split, scores, gradients, store), two
// workgroups a CU, by the registers, which hold heads of 64 columns and no more.
template <int DP, int W>
__global__ __launch_bounds__(W *kWave, 2) void k_attn_short_bwd(const ShortBwd f) {
    constexpr int KS = DP / 16, NT = DP / 32, TB = 128 * DP, LO = 64 * DP;
    constexpr bool REG = DP <= 32;  // keys stay in registers, else they are read from LDS for every tile, where they are anyway
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // q's tile, go's tile, the waves' keys, their ds, then small tables
    char *const qs = smem, *const gs = smem + TB, *const keys = smem + 2 * TB, *const dss = keys + W * TB;
    FeedTables<DP, W> &tables = *(FeedTables<DP, W> *)(dss + W * kDsTile);
    float *const ds_by = (float *)(&tables + 1), *const keys_by = ds_by + 2 * W * kTile;  // [W][2][32], [W]: the scales of the waves' ds and of their keys
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
        h8 kh[REG ? KS : 1], kl[REG ? KS : 1], vh[KS], vl[KS];
        int ek = 0, own_k = 0, own_v = 0;  // the keys' tile's exponent, this lane's key's and value's
        if (mine) {  // this wave's values, through the place of its keys, and its keys, which stay
            float x[KS][8];
            (void)tile_load<DP>(f.v + b * a.sv[0] + u * a.sv[2], a.sv[1], kw * kTile, n, D, x, own_v);
            tile_split<DP>(x, own_v, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) vh[s] = row_frag(kt + ra, s), vl[s] = row_frag(kt + ra + LO, s);
            ek = exponent_of(tile_load<DP>(f.k + b * a.sk[0] + u * a.sk[2], a.sk[1], kw * kTile, n, D, x, own_k));
            tile_split<DP>(x, own_k, kt);
            if constexpr (REG) {
#pragma unroll
                for (int s = 0; s < KS; s++) kh[s] = row_frag(kt + ra, s), kl[s] = row_frag(kt + ra + LO, s);
            }
            if (lane == 0) keys_by[kw] = pow2i(ek) * a.scale;
        }
        f16x dk[NT], dv[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) dk[t][r] = dv[t][r] = 0.0f;
        float F = 0x1p100f, U = live ? kNoUnit : -kNoUnit;
        const ScaleParts parts(a.scale);
        const float ck = pow2i(own_k) * a.scale * kLog2e, cv = pow2i(own_v), key_below = (float)(own_k - ek);
        uint32_t todo = ~0u;  // rows of a tile that no pass had
        for (int64_t t = t0, tn = t0; t < t1; t = tn) {
            const FeedPass pass = next.pass(f, b, u, tn, t1, todo, qs, gs, tables);
            if (mine) {
                const char *qt = qs + ra, *gt = gs + ra, *qc = qs + ca, *gc = gs + ca;
                const f4 *rows = (const f4 *)tables.stats + half;
                f16x s, dp;
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = dp[r] = 0.0f;
                steps<2 * KS>([&](int k) { return k % 2 ? Pieces{row_frag(gt, k / 2), row_frag(gt + LO, k / 2)} : Pieces{row_frag(qt, k / 2), row_frag(qt + LO, k / 2)}; },
                              [&](int k, const Pieces &x) {
                                  if (k % 2) dp = mfma3(x.hi, x.lo, vh[k / 2], vl[k / 2], dp);
                                  else s = mfma3(x.hi, x.lo, REG ? kh[k / 2] : row_frag(kt + ra, k / 2), REG ? kl[k / 2] : row_frag(kt + ra + LO, k / 2), s);
                              });
                const float c = ck * pow2i(pass.eq), c2 = cv * pow2i(pass.eg), xg = (float)pass.eg, off = live ? first_shift(xg, U) : -INFINITY;
                float most = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f4 ls = rows[2 * j];
#pragma unroll
                    for (int e = 0; e < 4; e++) s[4 * j + e] = __builtin_amdgcn_exp2f(fma_(s[4 * j + e], c, off - ls[e]));
                }
                const float sh = column_unit(s, xg, pass.hold, U, dv);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f4 de = rows[8 + 2 * j];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = 4 * j + e;
                        dp[r] = s[r] * fma_(dp[r], c2, -de[e]);
                        most = __builtin_fmaxf(most, __builtin_fabsf(dp[r]));
                    }
                }
                put_ds(dp, __builtin_amdgcn_exp2f(key_below + 14.0f - sh), mine_ds, ds_by + 2 * kw * kTile);
                const float kap = parts.times((float)pass.eq - sh);
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
            if (f.gq) gq_blocks<DP, W>(f, b, u, t, nt, keys, dss, ds_by, keys_by, pass.rows);
        }
        if (key < a.Lk) {
            const int64_t at = ((b * a.Lk + key) * a.Hkv + u) * D;
            const bool some = live && t0 < t1;
            if (f.gk) store_column<true>(f.gk + split * f.part_k + at, dk, some, 1.0f / F, half, D, f.acc_k);
            if (f.gv) store_column<true>(f.gv + split * f.part_k + at, dv, some, unit_of(U), half, D, f.acc_v);
        }
    }
}

// Backward in one pass over the queries: two waves share 32 keys, and the workgroup splits a tile of queries and output gradients
// (the next one's on their way meanwhile).  As in k_attn_dkv one wave takes the scores, p and gv, the other makes ds of p and takes
// gk; it leaves ds in LDS, and all waves share the blocks of gq^T = k^T ds^T over all keys.  Half the registers for each wave's
// keys: heads of up to 128 columns, a workgroup a CU.  4096 x 77, 4 x 16 heads, forward and backward: of 128 columns 332 us (39
// registers spill), and 491 through packed tiles and k_attn_dkv, k_attn_dq; of 80, 268 and 326; of 64, 216 where the kernel above takes 161.
template <int DP, int KT>
__global__ __launch_bounds__(2 * KT *kWave, 2) void k_attn_short_bwd_pairs(const ShortBwd f) {
    constexpr int KS = DP / 16, NT = DP / 32, TB = 128 * DP, LO = 64 * DP, W = 2 * KT;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // q's tile, go's tile, the tiles of keys, p and then ds of each, then small tables
    char *const qs = smem, *const gs = smem + TB, *const keys = smem + 2 * TB, *const dss = keys + KT * TB;
    FeedTables<DP, W> &tables = *(FeedTables<DP, W> *)(dss + KT * kDsTile);
    float *const ds_by = (float *)(&tables + 1), *const keys_by = ds_by + 2 * KT * kTile;  // [KT][2][32], [KT]: the scales of the tiles' ds and of their keys
    float *const shift = keys_by + KT, *const below = shift + KT * kWave;  // [KT][64]: p is handed over as 2^shift p; the keys' own exponents
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
        int own = 0;  // this lane's key's or value's exponent
        if (mine && ds_wave) {
            float x[KS][8];
            (void)tile_load<DP>(f.v + b * a.sv[0] + u * a.sv[2], a.sv[1], kw * kTile, n, D, x, own);
            tile_split<DP>(x, own, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) kh[s] = row_frag(kt + ra, s), kl[s] = row_frag(kt + ra + LO, s);
        }
        __syncthreads();
        if (mine && !ds_wave) {
            float x[KS][8];
            const int ek = exponent_of(tile_load<DP>(f.k + b * a.sk[0] + u * a.sk[2], a.sk[1], kw * kTile, n, D, x, own));
            tile_split<DP>(x, own, kt);
#pragma unroll
            for (int s = 0; s < KS; s++) kh[s] = row_frag(kt + ra, s), kl[s] = row_frag(kt + ra + LO, s);
            if (lane == 0) keys_by[kw] = pow2i(ek) * a.scale;
            below[kw * kWave + lane] = (float)(own - ek);
        }
        if (t0 < t1) next.fetch(f, b, u, t0);
        f16x acc[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[t][r] = 0.0f;
        float F = 0x1p100f, U = live ? kNoUnit : -kNoUnit;
        const ScaleParts parts(a.scale);
        const float ck = ds_wave ? pow2i(own) : pow2i(own) * a.scale * kLog2e;
        uint32_t todo = ~0u;  // rows of a tile that no pass had
        for (int64_t t = t0, tn = t0; t < t1; t = tn) {
            const FeedPass pass = next.pass(f, b, u, tn, t1, todo, qs, gs, tables);
            const f4 *const rows = (const f4 *)tables.stats + half;
            f4 *const ph = (f4 *)hand + lane;  // p's registers 4 j .. 4 j + 3 at 64 j
            const float xg = (float)pass.eg;
            f16x s;
            if (mine) {
                const char *rt = (ds_wave ? gs : qs) + ra;
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = 0.0f;
                steps<KS>([&](int k) { return Pieces{row_frag(rt, k), row_frag(rt + LO, k)}; },
                          [&](int k, const Pieces &x) { s = mfma3(x.hi, x.lo, kh[k], kl[k], s); });
                if (!ds_wave) {
                    const float c = ck * pow2i(pass.eq), off = live ? first_shift(xg, U) : -INFINITY;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const f4 ls = rows[2 * j];
#pragma unroll
                        for (int e = 0; e < 4; e++) s[4 * j + e] = __builtin_amdgcn_exp2f(fma_(s[4 * j + e], c, off - ls[e]));
                    }
                    shift[kw * kWave + lane] = column_unit(s, xg, pass.hold, U, acc);
#pragma unroll
                    for (int j = 0; j < 4; j++) ph[64 * j] = f4{s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]};
                }
            }
            lds_barrier();  // p is there
            if (mine) {
                if (ds_wave) {
                    const float sh = shift[kw * kWave + lane], c = ck * pow2i(pass.eg), kap = parts.times((float)pass.eq - sh);
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
                    put_ds(s, __builtin_amdgcn_exp2f(below[kw * kWave + lane] + 14.0f - sh), hand, ds_by + 2 * kw * kTile);  // where p was
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
            if (f.gq) gq_blocks<DP, W>(f, b, u, t, nt, keys, dss, ds_by, keys_by, pass.rows);
        }
        float *const out = ds_wave ? f.gk : f.gv;
        if (out && key < a.Lk)
            store_column<true>(out + split * f.part_k + ((b * a.Lk + key) * a.Hkv + u) * D, acc, live && t0 < t1,
                               ds_wave ? 1.0f / F : unit_of(U), half, D, ds_wave ? f.acc_k : f.acc_v);
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
    // x 77, 4 x 16 heads 161 us with four and 165 with eight, 64 x 64, 64 x 8 38 and 42; 197 x 197, 8 x 12 heads 65 and 63)
    else if (DP == 64 && 3 * lds <= 160 * 1024) launch(&k_attn_short_fwd<64, 4, 3>, f.units, 256, lds, st, f);
    else if (DP == 64) launch(&k_attn_short_fwd<64, 8, 2>, f.units, 512, lds, st, f);
    else if (DP == 96) launch(&k_attn_short_fwd<96, 8, 2>, f.units, 512, lds, st, f);
    else launch(&k_attn_short_fwd<128, 8, 2>, f.units, 512, lds, st, f);
}

template <int DP, int W, int KT, class F>
static void bwd_launch(F *kernel, const ShortBwd &f, hipStream_t st) {  // W waves, KT tiles of keys
    const size_t lds = 2 * 128 * DP + (size_t)KT * (128 * DP + kDsTile) + sizeof(FeedTables<DP, W>) +
                       KT * (2 * kTile + 1 + (W > KT ? 2 * kWave : 0)) * sizeof(float);
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
