// Shared pieces of the attention kernels (attention.hip): fp32 operands as pairs of fp16 on the matrix cores.
//
// A 32-row tile of an operand is scaled by a power of two that puts its largest finite value into [2^14, 2^15), and every value
// is cut into x = hi + lo, fp16 each (rounded to nearest: |x - hi| <= 2^-11 |x|, |x - hi - lo| <= 2^-22 |x|).  A product is
// hi hi + hi lo + lo hi on v_mfma_f32_32x32x16_f16, which sums in fp32: the part left out, lo lo, is at most 2^-22 of it.  The
// scale keeps the whole exponent range: values 2^-17 of their tile's largest and up have their 22 bits, smaller ones an absolute
// error of 2^-40 of that largest.  Three products at the fp16 rate cost a fifth of v_mfma_f32_32x32x2_f32's one.
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

namespace nchip {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16x __attribute__((ext_vector_type(16)));

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

__device__ __forceinline__ float finite_abs(float x) {
    const float a = __builtin_fabsf(x);
    return a < INFINITY ? a : 0.0f;  // NaN too
}

// the exponent e of a scale 2^e that puts `most` (finite, >= 0) into [2^14, 2^15) when values are divided by it
__device__ __forceinline__ int tile_exponent(float most) {
    const int e = (int)(__float_as_uint(most) >> 23) - 127 - 14;
    return e < -120 ? -120 : e;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// eight columns of a row from d on, zeros from column D on
__device__ __forceinline__ void load8(const float *row, int d, int D, float *x) {
    if (d + 8 <= D) {
        const f4 p = *(const f4u *)(row + d), q = *(const f4u *)(row + d + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = p[i], x[4 + i] = q[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = row[d + i < D ? d + i : D - 1];
            x[i] = d + i < D ? v : 0.0f;
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

}  // namespace nchip
