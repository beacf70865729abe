// Shared pieces of the attention kernels (attention.hip): fp32 operands as pairs of fp16 on the matrix cores.
//
// A 32-row tile of an operand is scaled by a power of two that puts its largest finite value into [2^14, 2^15), or, where its rows are
// unlike (kOwnRows), each row by one of its own; and every value is cut into x = hi + lo, fp16 each (rounded to nearest: |x - hi| <=
// 2^-11 |x|, |x - hi - lo| <= 2^-22 |x|).  A product is hi hi + hi lo + lo hi on v_mfma_f32_32x32x16_f16, which sums in fp32: the
// part left out, lo lo, is at most 2^-22 of it.  Values 2^-17 of what they are scaled by and up have their 22 bits, smaller ones
// an absolute error of 2^-40 of it, so no more than 2^-28 of their row's largest.  Where rows are summed over, the other operand takes
// the rows' powers of two, and its own scale follows the products' size, not that of the tiles.  Three products at the fp16 rate cost
// three eighths of v_mfma_f32_32x32x2_f32's one.
//
// Fragments: lane l of the 32x32x16 product holds row (of A) or column (of B) l % 32 and eight k, those of half l / 32; the
// result's column l % 32 in rows 8 (r / 4) + 4 (l / 32) + r % 4, r < 16.  A tile holds the 16 bytes of columns 8 c .. 8 c + 7 of row
// r at 16 (32 c + (r ^ 4 (c & 1))), first of all hi, then of all lo: 128 DP bytes, DP the columns padded to 32, 64, 96, 128 or
// 256 with zeros.  From LDS it gives both operands without bank conflicts:
//   row fragments (the columns are summed over), one 16-byte read: columns 16 s + 8 (l / 32) .. + 7 of row l % 32;
//   column fragments (the rows are summed over), two transposing 8-byte reads: rows 16 s + 4 (l / 32) + {0, 1, 2, 3, 8, 9, 10, 11}
//   of column 32 t + l % 32 -- the order in which a result's registers 8 s .. 8 s + 7 hold their rows, so that probabilities
//   are the next product's operand without leaving their lanes.
#pragma once

#include "common.hpp"
#include "intdiv.hpp"

namespace nchip {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16x __attribute__((ext_vector_type(16)));

constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;

struct AttnArgs {
    int64_t B, Lq, Lk, Hq, Hkv, D, G;  // G: query heads of a key head
    int64_t sq[3], sk[3], sv[3];
    float scale;
    bool narrow;   // fewer than 2^31 rows of a pair
    IntDiv by_g;

    // row R of a pair: token and, among the heads that share the pair's keys, head
    __device__ __forceinline__ void row(int64_t R, int64_t &i, int64_t &g) const {
        if (G == 1) {
            i = R, g = 0;
        } else if (narrow) {
            const uint32_t q = by_g.div31((uint32_t)R);
            i = q, g = (uint32_t)R - q * (uint32_t)G;
        } else {
            i = R / G, g = R - i * G;
        }
    }
};

constexpr int kAttnD = 256;       // columns at most
constexpr int kAttnB = 256;       // lanes of a workgroup
constexpr int kAttnWaves = 4;
constexpr int kTile = 32;         // rows of a tile
constexpr int64_t kAttnGrid = 1 << 22;  // workgroups of a launch at most

__host__ __device__ constexpr int64_t tile_bytes(int DP) { return 128 * (int64_t)DP; }  // one layout

struct Split8 {
    h8 hi, lo;
};

__device__ __forceinline__ Split8 split8(const float *x) {
    Split8 r;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const h2 h = __builtin_convertvector(f2{x[i], x[i + 1]}, h2);
        const h2 l = __builtin_convertvector(f2{x[i] - (float)h.x, x[i + 1] - (float)h.y}, h2);
        r.hi[i] = h.x, r.hi[i + 1] = h.y;
        r.lo[i] = l.x, r.lo[i + 1] = l.y;
    }
    return r;
}

// a lane's byte offset in a tile for row fragment 0 (s: + 1024 s; lo: + 64 DP), and for column fragment (0, 0)
__device__ __forceinline__ int row_at(int lane) {
    const int half = lane >> 5, r = lane & 31;
    return half * 512 + (r ^ (4 * half)) * 16;
}
__device__ __forceinline__ int col_at(int lane) {
    const int i = lane & 15, g = lane >> 4, b = (i >> 1) & 1;
    return (2 * (g & 1) + b) * 512 + (((g >> 1) ^ b) * 4 + i / 4) * 16 + 8 * (i & 1);
}
__device__ __forceinline__ h8 row_frag(const char *tile, int s) { return *(const h8 *)(tile + 1024 * s); }
// 16 lanes read four rows of 16 columns, four columns a lane, and get four rows of one column each
__device__ __forceinline__ h8 col_frag(const char *tile, int s, int t) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const char *p = tile + 2048 * t + 256 * s;
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p));
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 128));
    typedef short s8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(h8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

// a result's registers r0 .. r0 + 7 as the next product's operand
__device__ __forceinline__ Split8 split_regs(const f16x &s, int r0) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = s[r0 + e];
    return split8(y);
}

__device__ __forceinline__ f16x mfma3(const h8 &ah, const h8 &al, const h8 &bh, const h8 &bl, f16x c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, c, 0, 0, 0);
}

// the other half-wave's value of the same column, combined
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __builtin_fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// The largest |x| of n values that is finite: NaNs do not count, and where an infinity is met the values are looked at again.
template <int N>
__device__ __forceinline__ float abs_max(const float (&x)[N], float most) {
    float m = most;
#pragma unroll
    for (int i = 0; i < N; i++) m = __builtin_fmaxf(m, __builtin_fabsf(x[i]));
    if (__builtin_expect(m == INFINITY, 0)) {
        m = most;
#pragma unroll
        for (int i = 0; i < N; i++) m = __builtin_fmaxf(m, __builtin_fabsf(x[i]) < INFINITY ? __builtin_fabsf(x[i]) : 0.0f);
    }
    return m;
}

// the exponent e of a scale 2^e that puts `most` (finite, >= 0) into [2^14, 2^15) when values are divided by it
__device__ __forceinline__ int tile_exponent(float most) {
    const int e = (int)(__float_as_uint(most) >> 23) - 127 - 14;
    return e < -120 ? -120 : e;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// A tile whose rows are unlike -- the largest of one, zeros aside, below 2^-12 of the tile's -- is scaled row by row: rows above keep 22
// bits of values down to 2^-5 of their own largest.  (A limit of 2^-6 was met by gradients of 2^(2 N(0, 1)): with few keys, where unlike
// rows cost another pass, 287 us where 145 do, 4096 x 77, 4 x 16 heads of 64.)  The tile's exponent, the largest row's, is stored with kOwnRows added, and how far each row's lies below it (0 to -100) beside it.
constexpr int kOwnRows = 1024;
constexpr float kAlike = 0x1p-12f;
__device__ __forceinline__ bool own_rows(int code) { return code >= kOwnRows / 2; }
__device__ __forceinline__ int exponent_of(int code) { return own_rows(code) ? code - kOwnRows : code; }
__device__ __forceinline__ bool rows_unlike(float row_most, float tile_most) {  // of a wave that has all rows
    return __any(row_most > 0.0f && row_most < tile_most * kAlike);
}
__device__ __forceinline__ int row_exponent(float row_most, int tile_ex) {
    return row_most > 0.0f ? max(tile_exponent(row_most), tile_ex - 100) : tile_ex;
}

__device__ __forceinline__ f4 moved4(f4 v, int by) {  // down by `by` places
    if (by & 1) v = f4{v[1], v[2], v[3], 0.0f};
    if (by & 2) v = f4{v[2], v[3], 0.0f, 0.0f};
    if (by & ~3) v = f4{0.0f, 0.0f, 0.0f, 0.0f};
    return v;
}

// four columns of a row of D >= 4 from d on, zeros from column D on: the row's last four, moved down, where it ends among them
__device__ __forceinline__ f4 last4(const float *row, int d, int D) {
    const int o = min(d, D - 4);
    return moved4(*(const f4u *)(row + o), d - o);
}

// eight columns of a row from d on, zeros from column D on
__device__ __forceinline__ void load8(const float *row, int d, int D, float *x) {
    f4 p = {0.0f, 0.0f, 0.0f, 0.0f}, q = p;
    if (d + 8 <= D) {
        p = *(const f4u *)(row + d);
        q = *(const f4u *)(row + d + 4);
    } else if (d < D && D >= 4) {
        p = last4(row, d, D);
        q = last4(row, d + 4, D);
    } else if (d < D) {  // a row of one to three columns
        p[0] = row[0];
        if (D > 1) p[1] = row[1];
        if (D > 2) p[2] = row[2];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = p[i], x[4 + i] = q[i];
}

// N times eight columns of a row, from d0, d0 + step, ... on, zeros from column D on.  All loads are on their way before the first
// is waited for: addresses are held inside the row rather than branched on (with load8 a wave waits for each in turn: 4096 x 77,
// 4 x 16 heads of 64, forward: 46 us, and 55 with it).
template <int N>
__device__ __forceinline__ void load_chunks(const float *row, int d0, int step, int D, float (&x)[N][8]) {
    if (D < 4) {  // at most the first chunk's first three
#pragma unroll
        for (int k = 0; k < N; k++) load8(row, d0 + k * step, D, x[k]);
        return;
    }
    f4 v[N][2];
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
        for (int h = 0; h < 2; h++) v[k][h] = *(const f4u *)(row + min(d0 + k * step + 4 * h, D - 4));
    if (D % 4 == 0) {
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[k][e] = d0 + k * step + 4 * (e / 4) < D ? v[k][e / 4][e % 4] : 0.0f;
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int d = d0 + k * step + 4 * h;
                const f4 m = moved4(v[k][h], d - min(d, D - 4));
#pragma unroll
                for (int e = 0; e < 4; e++) x[k][4 * h + e] = m[e];
            }
    }
}

// four columns of a contiguous row from d on, stored or added
__device__ __forceinline__ void store4(float *row, int d, int D, f4 v, int acc) {
    if (d + 4 <= D) {
        if (acc) v += *(const f4u *)(row + d);
        *(f4u *)(row + d) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (d + i < D) row[d + i] = acc ? row[d + i] + v[i] : v[i];
    }
}

__device__ __forceinline__ int64_t keys_of(int64_t Lk, const int *key_len, int64_t b) {
    if (!key_len) return Lk;
    const int64_t n = key_len[b];
    return n < 0 ? 0 : n < Lk ? n : Lk;
}

// A block of N steps, each with two fragments from LDS (read(k): its hi and lo) and three products (step(k, pieces)): the
// fragments are read two steps ahead of their products, which the compiler on its own does not do -- it saves registers and waits
// for LDS in every step.  `first`: the steps 0 and 1, where they are read earlier still.
struct Pieces {
    h8 hi, lo;
};
__device__ __forceinline__ void keep_order() {  // LDS reads and products stay where they are; all else may pass
    __builtin_amdgcn_sched_barrier(0x0002 | 0x0004 | 0x0010 | 0x0020 | 0x0040);
}
template <int N, class Read, class Step>
__device__ __forceinline__ void steps(Pieces (&f)[3], Read &&read, Step &&step) {
    keep_order();
#pragma unroll
    for (int k = 0; k < N; k++) {
        if (k + 2 < N) f[(k + 2) % 3] = read(k + 2);
        step(k, f[k % 3]);
        keep_order();
    }
}
template <int N, class Read, class Step>
__device__ __forceinline__ void steps(Read &&read, Step &&step) {
    Pieces f[3];
    f[0] = read(0);
    f[1] = read(1);
    steps<N>(f, read, step);
}

// Workgroups are dealt round robin over the 8 XCDs: consecutive units of a launch go to one XCD, which then keeps their
// keys in its L2.
__device__ __forceinline__ int64_t xcd_unit(int64_t w, int64_t units) {
    const int64_t each = units / 8, rest = units % 8, x = w % 8, k = w / 8;
    return x * each + (x < rest ? x : rest) + k;
}

// The gradients of the scores have no bound to scale them by beforehand: a lane's column (a key, or a query's row) has a power of
// two F of its own that puts its largest |x| into [2^11, 2^12) when it first shows or passes 2^15, and its sums are brought along.
__device__ __forceinline__ bool column_scale(float most, float &F, float &by) {
    by = 1.0f;
    const bool over = most * F > 32768.0f;
    if (over) {
        int e = (int)(__float_as_uint(most) >> 23);
        e = e < 12 ? 12 : e;
        const float f = __uint_as_float((uint32_t)(127 + 11 + 127 - e) << 23);
        by = f / F;
        F = f;
    }
    return __any(over);
}

// a result's rows 8 (r / 4) + 4 (lane / 32) + r % 4 times 2^ the exponents of a tile's 32 rows
__device__ __forceinline__ void scale_rows(f16x &s, const float *rows) {
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const f4 e = *(const f4 *)(rows + 4 * half + 8 * j);
#pragma unroll
        for (int x = 0; x < 4; x++) s[4 * j + x] *= __builtin_amdgcn_exp2f(e[x]);
    }
}
__device__ __forceinline__ float largest(const f16x &s) {
    float most = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r++) most = __builtin_fmaxf(most, __builtin_fabsf(s[r]));
    return most;
}

// gv's sums: a lane's column (a key) has a unit 2^U of its own, for products of probabilities and gradients of 2^e.  Probabilities
// are taken as p 2^first_shift; where one of 1 would pass 2^14 in the unit, or the tile is `loose`, column_unit looks at the column's
// largest: the unit is raised so that 1 is 2^14 where the key is counted by 2^-16 and up, else so that this largest product is 2^10.
// So a tile of large gradients whose rows do not count a key leaves it its bits, and a key that is hardly counted by any row has
// its own.  Returns the shift of the probabilities as they are left, e - U.
constexpr float kPTop = 10.0f, kPSlack = 4.0f, kNoUnit = -1000.0f;
__device__ __forceinline__ float first_shift(float e, float U) {  // no less than -60: far below what gv can show
    return __builtin_fminf(__builtin_fmaxf(e - U, -60.0f), kPTop + kPSlack);
}
template <int NT>
__device__ __forceinline__ float column_unit(f16x &p, float e, bool loose, float &U, f16x (&acc)[NT]) {
    constexpr float most = kPTop + kPSlack;
    float shift = first_shift(e, U);
    if (__any(e - U > most) || loose) {
        float top = 0.0f;
        const float one = __builtin_amdgcn_ldexpf(1.0f, (int)shift);
#pragma unroll
        for (int r = 0; r < 16; r++) p[r] = p[r] > one ? one : p[r], top = __builtin_fmaxf(top, p[r]);
        top = halves_max(top);
        const float log_top = (float)((int)(__float_as_uint(top) >> 23) - 126) - shift;  // rounded up; far below where there is none
        const float need = log_top >= -16.0f ? e - most : __builtin_fmaxf(log_top + (e - kPTop), e - 100.0f);
        const float Un = e - U > most ? __builtin_fmaxf(U, need) : U, left = __builtin_fmaxf(e - Un, -60.0f);
        const float by = __builtin_amdgcn_exp2f(U - Un), to = __builtin_amdgcn_exp2f(left - shift);
        U = Un;
        shift = left;
#pragma unroll
        for (int r = 0; r < 16; r++) p[r] *= to;
#pragma unroll
        for (int d = 0; d < NT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[d][r] *= by;
    }
    return shift;
}
// A probability taken from scores and their sum past 2^20 may come out above 1, far past 2^24: a tile with such rows is marked.
__device__ __forceinline__ bool loose(float log_sum) { return __builtin_fabsf(log_sum) > 0x1p20f && log_sum < INFINITY; }
__device__ __forceinline__ float unit_of(float U) { return __builtin_amdgcn_ldexpf(1.0f, (int)__builtin_fmaxf(U, -1000.0f)); }

// The scale of the scores times 2^e, e far outside a float's exponents where the scale is: it goes into the scores' gradients before
// their column scale, which would lose them else.
struct ScaleParts {
    float m, k;  // m 2^k
    __device__ __forceinline__ explicit ScaleParts(float scale) {
        const int e = (int)((__float_as_uint(scale) >> 23) & 255) - 127;
        k = (float)e;
        m = e > 126 ? scale * 0.5f * pow2i(1 - e) : scale * pow2i(-e);
    }
    __device__ __forceinline__ float times(float e) const { return m * __builtin_amdgcn_exp2f(e + k); }
};
// kap F, held finite: where it is not, every gradient of the tile is zero, or past a float's range
__device__ __forceinline__ float finite_product(float kap, float F) { return __builtin_fminf(__builtin_fmaxf(kap * F, -0x1p127f), 0x1p127f); }

template <int NT>
__device__ __forceinline__ void scale_acc(f16x (&acc)[NT], float by) {
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[d][r] *= by;
}

// a lane's column as a row of the output, `by` times; CHECK: zeros where it holds nothing that counts
template <bool CHECK, int NT>
__device__ __forceinline__ void store_column(float *row, const f16x (&acc)[NT], bool some, float by, int half, int D, int add) {
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            f4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = !CHECK || some ? acc[d][4 * j + e] * by : 0.0f;
            store4(row, 32 * d + 8 * j + 4 * half, D, v, add);
        }
}

// ------------------------------------------------------------------------------------------------
// forward: a wave's 32 rows of queries against a tile of keys
// ------------------------------------------------------------------------------------------------
// A wave holds 32 rows of queries as columns: s^T = k q^T (A: 32 keys), so that a row's scores lie in the registers of two lanes
// and its maximum, sum and scale are theirs; p^T is then the operand of o^T = v^T p^T as it lies.  One pass over the keys.  p = 2^(s - m)
// for a reference m, a whole number that moves when a score passes it by 2^4.  What is cut into pieces is p 2^(e - U): e the
// exponent of the tile's values, U that of o's unit, a row's own, which is raised so that its largest product -- p and value
// together -- lies at 2^10 when it passes 2^14, and falls as m rises.  So a value that is large and does not count leaves the
// others their bits, and a product below 2^-24 of a row's largest loses low bits against an absolute 2^-35 of it.
template <int DP>
struct Query {  // the rows times scale log2(e), as the second operand: column fragments of q^T
    h8 hi[DP / 16], lo[DP / 16];
    float c;  // 2^ its exponent
};

template <int DP>
__device__ __forceinline__ void load_query(Query<DP> &q, const float *row, bool live, float scale, int half, int D) {
    const float c = live ? scale * kLog2e : 0.0f;
    float most = 0.0f, x[DP / 16][8];
    load_chunks(row, 8 * half, 16, D, x);
#pragma unroll
    for (int s = 0; s < DP / 16; s++) most = abs_max(x[s], most);
    // c 2^-e stays finite where the row is all but zero
    const int e = max(tile_exponent(halves_max(most) * __builtin_fabsf(c)), tile_exponent(__builtin_fabsf(c)) - 98);
    const float by = c * pow2i(-e);
    q.c = pow2i(e);
#pragma unroll
    for (int s = 0; s < DP / 16; s++) {
#pragma unroll
        for (int k = 0; k < 8; k++) x[s][k] *= by;
        const Split8 p = split8(x[s]);
        q.hi[s] = p.hi, q.lo[s] = p.lo;
    }
}

template <int DP>
struct Sums {
    f16x o[DP / 32];
    float m, l, U;  // reference, sum of p, exponent of o's unit
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < DP / 32; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[t][r] = 0.0f;
        m = -INFINITY, l = 0.0f, U = -INFINITY;
    }
};

// a wave's sums handed to another one through LDS, lane by lane, and joined there to its own
template <int DP>
__device__ __forceinline__ void put(const Sums<DP> &a, f4 *to) {
#pragma unroll
    for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int j = 0; j < 4; j++) to[(4 * d + j) * kWave] = f4{a.o[d][4 * j], a.o[d][4 * j + 1], a.o[d][4 * j + 2], a.o[d][4 * j + 3]};
    to[DP / 8 * kWave] = f4{a.m, a.l, a.U, 0.0f};
}
template <int DP>
__device__ __forceinline__ void join(Sums<DP> &a, const f4 *from) {
    const f4 b = from[DP / 8 * kWave];
    const float m = __builtin_fmaxf(a.m, b[0]), da = a.m == m ? 0.0f : a.m - m, db = b[0] == m ? 0.0f : b[0] - m;
    const float ua = a.U + da, ub = b[2] + db, U = __builtin_fmaxf(ua, ub);
    const float oa = ua == U ? 1.0f : __builtin_amdgcn_exp2f(ua - U), ob = ub == U ? 1.0f : __builtin_amdgcn_exp2f(ub - U);
#pragma unroll
    for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const f4 v = from[(4 * d + j) * kWave];
#pragma unroll
            for (int e = 0; e < 4; e++) a.o[d][4 * j + e] = fma_(a.o[d][4 * j + e], oa, v[e] * ob);
        }
    a.l = fma_(a.l, __builtin_amdgcn_exp2f(da), b[1] * __builtin_amdgcn_exp2f(db));
    a.m = m, a.U = U;
}

// kt, vt: the tile's keys and values in LDS, at this lane's row_at and col_at; ek, ev: their exponents; kr, vr: their rows', read where
// they have their own; left: keys of the tile that count (32 but in the last one), less 4 half
template <int DP>
__device__ __forceinline__ void attend(Sums<DP> &a, const Query<DP> &q, const char *kt, const char *vt, int ek, int ev, const float *kr,
                                       const float *vr, bool cut, int left) {
    constexpr int KS = DP / 16, NT = DP / 32, LO = 64 * DP;
    f16x s;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = 0.0f;
    steps<KS>([&](int k) { return Pieces{row_frag(kt, k), row_frag(kt + LO, k)}; },
              [&](int k, const Pieces &f) { s = mfma3(f.hi, f.lo, q.hi[k], q.lo[k], s); });
    const auto value = [&](int k) { return Pieces{col_frag(vt, k / NT, k % NT), col_frag(vt + LO, k / NT, k % NT)}; };
    Pieces f[3];
    f[0] = value(0);
    f[1] = value(1);
    float c = __builtin_fmaxf(q.c * pow2i(exponent_of(ek)), 0x1p-126f);  // -inf * c stays -inf
    if (cut || own_rows(ek)) {
        if (own_rows(ek)) scale_rows(s, kr);
        if (cut) {
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (8 * (r / 4) + r % 4 >= left) s[r] = -INFINITY;
        }
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; r++) top = __builtin_fmaxf(top, s[r]);
    top = halves_max(top) * c;
    const float e = (float)exponent_of(ev);
    const bool own = own_rows(ev);
    float dv = e - a.U;
    if (__any(top - a.m > kPSlack || top - a.m + dv > kPTop + kPSlack) || own) {
        const float mn = top - a.m > kPSlack ? __builtin_rintf(top) : a.m, down = a.m == mn ? 0.0f : a.m - mn;
        a.l *= __builtin_amdgcn_exp2f(down);
        a.U += down;
        a.m = mn;
        if (own) {  // p's sum, then p times 2^ its value's own exponent in p's place
            const int half = (threadIdx.x >> 5) & 1;
            float sum = 0.0f;
            top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f4 er = *(const f4 *)(vr + 4 * half + 8 * j);
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int r = 4 * j + x;
                    sum += __builtin_amdgcn_exp2f(fma_(s[r], c, -mn));
                    s[r] = fma_(s[r], c, er[x]);
                    top = __builtin_fmaxf(top, s[r]);
                }
            }
            top = halves_max(top);
            c = 1.0f;
            a.l += sum;
        }
        const float over = top - mn;
        const float Un = over + (e - a.U) > kPTop + kPSlack ? __builtin_ceilf(over) + (e - kPTop) : a.U;
        const float by = a.U == Un ? 1.0f : __builtin_amdgcn_exp2f(a.U - Un);
        a.U = Un;
        dv = e - Un;
#pragma unroll
        for (int d = 0; d < NT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) a.o[d][r] *= by;
    }
    // no smaller than 2^-60: far below what o can show, and p's sum keeps its bits
    dv = __builtin_fmaxf(dv, -60.0f);
    const float off = dv - a.m;
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r++) {
        s[r] = __builtin_amdgcn_exp2f(fma_(s[r], c, off));
        sum += s[r];
    }
    a.l = fma_(sum, own ? 0.0f : __builtin_amdgcn_exp2f(-dv), a.l);
    const Split8 p[2] = {split_regs(s, 0), split_regs(s, 8)};
    steps<2 * NT>(f, value, [&](int k, const Pieces &v) { a.o[k % NT] = mfma3(v.hi, v.lo, p[k / NT].hi, p[k / NT].lo, a.o[k % NT]); });
}

}  // namespace nchip
