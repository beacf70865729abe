// The vocabulary loss with its three products on the fp16 matrix cores: z = x W^T, gx = G W, gW = G^T x.
//
// A library's fp32 product of 8192^3 reaches an eighth of what its fp16 one does, so every operand is cut into two fp16 pieces under
// a power of two of its row (the index that is not summed over): x = 2^e (hi + lo), the row's largest finite value in [2^14, 2^15)
// after the scaling, hi and lo rounded to nearest: 22 bits of every value down to 2^-17 of its row's largest, an absolute error of
// 2^-40 of that below.  A product is hi hi + hi lo + lo hi, summed in fp32; lo lo, at most 2^-22 of a term, is left out.
//
// Packed operands.  A block of 32 rows by 16 k is 2 KiB: its hi pieces, then its lo pieces, each as a wave holds them for
// v_mfma_f32_32x32x16_f16 -- lane l has row l % 32 and eight k of half l / 32 in 16 bytes.  So a block is loaded into LDS as it lies, a
// KiB an instruction, and read from there as it lies, without bank conflicts.  z is left by the first product in the registers' order,
// 4 KiB a block of 32 rows n by 32 words v: lane l has n = l % 32 and v = 8 q + 4 (l / 32) + e, q and e < 4.  Quads 2 s and 2 s + 1 are then
// eight k of a block of 16 words, in the order 4 (l / 32) + {0, 1, 2, 3, 8, 9, 10, 11}, which the packed W that they meet has too.
//
// Steps of a call: labels that count are listed (rows that do not count take part in nothing); x and W are packed, by rows and by
// columns; then for pieces of the rows z (with each row's maximum and sum of exponentials over every 128 words), the rows' statistics,
// G's largest entry of every word, G in pieces for both products (in z's place, and turned for gW), gx in parts over the words and their
// sum, gW.  Scoring ends with the rows' statistics and leaves no z.
#include "vocab_loss.hpp"

namespace nchip {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16x __attribute__((ext_vector_type(16)));
typedef int i4v __attribute__((ext_vector_type(4)));

constexpr int kTile = 256;       // rows and columns of a workgroup's product
constexpr int kMmB = 512;        // its lanes: 8 waves, 2 over the rows and 4 over the columns
constexpr int kStages = 4;       // blocks of 16 k in LDS
constexpr int kStage = 2 * kTile * 16 * 4;  // bytes of one: both operands' 256 rows, two pieces
constexpr size_t kMmLds = (size_t)kStages * kStage;
constexpr int64_t kZBytes = int64_t(4) << 30;  // of z and of the turned G, both together, held at a time
constexpr int64_t kScored = int64_t(1) << 36;  // products of a launch that leaves no z
constexpr int64_t kPieceRows = 1 << 20;
constexpr int kStatWords = 128;  // words of one partial statistic

struct VlRow {
    float m, ls;  // the row's maximum and log sum exp(z - m)
    float own;    // p_l - 1, the largest of its row of G
    int label;
};

// the exponent e that puts `most` (finite, >= 0) into [2^14, 2^15) when values are divided by 2^e
__device__ __forceinline__ int piece_exponent(float most) {
    const int e = (int)(__float_as_uint(most) >> 23) - 127 - 14;
    return e < -120 ? -120 : e;
}
__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ float finite_abs(float x) {
    const float a = __builtin_fabsf(x);
    return a < __builtin_inff() ? a : 0.0f;
}

struct Pieces {
    h8 hi, lo;
};
__device__ __forceinline__ Pieces cut(const float (&x)[8], float scale) {
    Pieces r;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = x[i] * scale;
        const _Float16 h = (_Float16)v;
        r.hi[i] = h;
        r.lo[i] = (_Float16)(v - (float)h);
    }
    return r;
}

// ---- the product ------------------------------------------------------------------------------------------------------
enum { MM_Z = 0, MM_GX = 1, MM_GW = 2 };

struct MmArgs {
    const char *A, *B;      // packed; blocks of a row block follow each other
    int64_t step_a, step_b;  // bytes from a row block to the next
    int tiles_m, tiles_n, slices;
    int kblocks;            // of 16 k, all slices together: an even number, as each slice's is
    const VlHead *head;
    int64_t row0;           // of this piece, among the rows that count
    int64_t V, D;
    // MM_Z: A the words, B the rows
    const int *ew, *ex;
    const float *bias;
    const int32_t *labels;  // of this piece's rows
    float *z;               // or none
    int64_t zwords;         // blocks of 32 words of a row block
    f2 *part;               // [words / kStatWords][rows]
    float *label_z;         // [rows]
    int64_t rows;           // of a piece, padded
    // MM_GX: A the rows, B the columns
    float *parts;           // [slices][rows][columns]
    int64_t cols;           // columns, padded
    // MM_GW: A the words, B the columns
    const float *most_a, *most_b;
    const float *gout;
    float *out;
    int sum, acc;
};

struct Frags {
    h8 a[4][2], b[2][2];
};

__device__ __forceinline__ float vl_coef(const VlHead *head, const float *gout, int sum) {
    const float c = gout ? *gout : 1.0f;
    return sum ? c : c / (float)head->count;
}

// The wave's 128 words by 64 rows of z, out of its accumulators.
__device__ __forceinline__ void z_out(const MmArgs &p, f16x (&acc)[4][2], int64_t v0, int64_t n0, int lane) {
    const int half = lane >> 5;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int64_t n = n0 + 32 * j + (lane & 31);
        const int ex = p.ex[n];
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int64_t v = v0 + 32 * i + 8 * q + 4 * half;
                const i4v ew = *(const i4v *)(p.ew + v);
                f4 z;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float b = p.bias && v + e < p.V ? p.bias[v + e] : 0.0f;
                    z[e] = __builtin_amdgcn_ldexpf(acc[i][j][4 * q + e], ew[e] + ex) + b;
                    z[e] = v + e < p.V ? z[e] : -__builtin_inff();
                    acc[i][j][4 * q + e] = z[e];
                }
                if (p.z) *(f4 *)(p.z + ((n0 / 32 + j) * p.zwords + v0 / 32 + i) * 1024 + q * 256 + lane * 4) = z;
            }
        }
        float m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) m = __builtin_fmaxf(m, acc[i][j][r]);
        m = __builtin_fmaxf(m, __shfl_xor(m, 32));
        const int label = p.labels[n];  // -1 where no row is
        const int64_t at = (int64_t)label - v0;
        if (__any(label >= 0 && at >= 0 && at < kStatWords)) {  // the label's own term is kept apart
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (at == 32 * i + 8 * (r / 4) + 4 * half + r % 4) {
                        p.label_z[n] = acc[i][j][r];
                        acc[i][j][r] = -__builtin_inff();
                    }
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) s += exp_sum_term(acc[i][j][r] - m);
        if (m == -__builtin_inff()) s = s == s ? s : 0.0f;
        s += __shfl_xor(s, 32);
        if (half == 0) p.part[(v0 / kStatWords) * p.rows + n] = f2{m, s};
    }
}

template <int WHAT>
__global__ __launch_bounds__(kMmB, 2) void k_vl_product(MmArgs p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave & 1, wn = wave >> 1;
    // XCD x runs the workgroups b with b % 8 == x: it gets the x-th of 8 runs of tiles, in groups of 8 tile rows
    const uint32_t nblk = gridDim.x, xcd = blockIdx.x & 7, per = nblk >> 3, rem = nblk & 7;
    const uint32_t id = xcd * per + min(xcd, rem) + (blockIdx.x >> 3);
    const uint32_t tiles = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n;
    const int slice = (int)(id / tiles), tile = (int)(id % tiles);
    const int per_group = 8 * p.tiles_n, group = tile / per_group, in_group = tile % per_group;
    const int gsize = min(p.tiles_m - group * 8, 8);
    const int tm = group * 8 + in_group % gsize, tn = in_group / gsize;

    const int64_t left = p.head->count - p.row0;  // rows of this piece and behind it
    int k0 = 0, k1 = p.kblocks;
    if (WHAT == MM_Z && (int64_t)tn * kTile >= left) return;
    if (WHAT == MM_GX) {
        if ((int64_t)tm * kTile >= left) return;
        const int64_t pairs = p.kblocks / 2;
        k0 = 2 * (int)(pairs * slice / p.slices), k1 = 2 * (int)(pairs * (slice + 1) / p.slices);
    }
    if (WHAT == MM_GW) {
        k1 = (int)min((int64_t)p.kblocks, left > 0 ? (left + 31) / 32 * 2 : 0);
        if (k1 == 0 && p.acc) return;
    }
    const int nk = k1 - k0;

    // wave w brings four of a stage's 32 KiB: pieces of row blocks 2 (w % 4) and the next, of A (w < 4) or B
    const char *src;
    int64_t next;
    {
        const bool b = wave >= 4;
        const int64_t rb = (int64_t)(b ? tn : tm) * (kTile / 32) + 2 * (wave & 3);
        next = b ? p.step_b : p.step_a;
        src = (b ? p.B : p.A) + rb * next + (int64_t)k0 * 2048 + lane * 16;
    }
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const uint32_t to = base + (uint32_t)wave * 4096;
    auto bring = [&](int kt) {
        const uint32_t at = __builtin_amdgcn_readfirstlane(to + (uint32_t)(kt & (kStages - 1)) * kStage);
        const char *s = src + (int64_t)kt * 2048;
        dma16(s, at);
        dma16(s + 1024, at + 1024);
        dma16(s + next, at + 2048);
        dma16(s + next + 1024, at + 3072);
    };
    auto fetch = [&](int kt, Frags &f) {
        const char *s = lds + (kt & (kStages - 1)) * kStage + lane * 16;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f.a[i][0] = *(const h8 *)(s + (4 * wm + i) * 2048);
            f.a[i][1] = *(const h8 *)(s + (4 * wm + i) * 2048 + 1024);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            f.b[j][0] = *(const h8 *)(s + kStage / 2 + (2 * wn + j) * 2048);
            f.b[j][1] = *(const h8 *)(s + kStage / 2 + (2 * wn + j) * 2048 + 1024);
        }
    };
    f16x acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = f16x{};
    auto multiply = [&](const Frags &f) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.a[i][1], f.b[j][0], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.a[i][0], f.b[j][1], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.a[i][0], f.b[j][0], acc[i][j], 0, 0, 0);
    };
    // At the barrier before block kt every wave's share of block kt + 1 is in LDS, and every wave has read block kt and with it left block
    // kt - 1, whose stage then takes block kt + 3.  A wave reads block kt + 1 into registers while it multiplies block kt.
    auto wait = [&](int kt) {  // this wave's loads of block kt + 1 have landed; those of kt + 2 may be on their way
        if (kt + 2 < nk) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
    };
    if (nk > 0) {
        for (int kt = 0; kt < 3 && kt < nk; kt++) bring(kt);
        if (nk >= 3) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
        Frags f0, f1;
        fetch(0, f0);
        for (int kt = 0; kt < nk; kt += 2) {  // behind the last block a stage is read again, for nothing
            wait(kt);
            if (kt + 3 < nk) bring(kt + 3);
            fetch(kt + 1, f1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(f0);
            wait(kt + 1);
            if (kt + 4 < nk) bring(kt + 4);
            fetch(kt + 2, f0);
            __builtin_amdgcn_sched_barrier(0);
            multiply(f1);
        }
    }

    // what the results need is computed behind the products, whose registers it would take
    int at = lane;
    asm volatile("" : "+v"(at)::"memory");
    const int64_t m0 = (int64_t)tm * kTile + 128 * wm, n0 = (int64_t)tn * kTile + 64 * wn;
    if constexpr (WHAT == MM_Z) {
        z_out(p, acc, m0, n0, at);
    } else if constexpr (WHAT == MM_GX) {
        // a store instruction writes 32 columns of two rows
        float *out = p.parts + ((int64_t)slice * p.rows + m0 + 4 * (at >> 5)) * p.cols + n0 + (at & 31);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int r = 0; r < 16; r++)
#pragma unroll
                for (int j = 0; j < 2; j++) out[(32 * i + 8 * (r / 4) + r % 4) * p.cols + 32 * j] = acc[i][j][r];
    } else {
        const float c = nk > 0 ? vl_coef(p.head, p.gout, p.sum) : 0.0f;
        const int64_t m1 = m0 + 4 * (at >> 5), d = n0 + (at & 31);
        float *out = p.out + m1 * p.D + d;
        const bool in0 = d < p.D, in1 = d + 32 < p.D;
        const int ed0 = piece_exponent(in0 ? p.most_b[d] : 0.0f), ed1 = piece_exponent(in1 ? p.most_b[d + 32] : 0.0f);
        auto put = [&](float *o, float v, int e) {
            v = __builtin_amdgcn_ldexpf(v, e);
            *o = p.acc ? fma_(v, c, *o) : v * c;
        };
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int dm = 32 * i + 8 * (r / 4) + r % 4;
                if (m1 + dm >= p.V) continue;
                const int em = piece_exponent(p.most_a[m1 + dm]);
                float *o = out + (int64_t)dm * p.D;
                if (in0) put(o, acc[i][0][r], ed0 + em);
                if (in1) put(o + 32, acc[i][1][r], ed1 + em);
            }
    }
}

// ---- which rows count ----------------------------------------------------------------------------------------------------
// Lists the rows that count and their labels (-1 behind the last), and looks for the first label that is neither a word nor `ignore`.
__global__ __launch_bounds__(1024) void k_vl_list(const int32_t *__restrict__ labels, int64_t N, int64_t padded, int64_t V, int32_t ignore,
                                                  VlHead *head, int32_t *__restrict__ from, int32_t *__restrict__ list, unsigned long long *bad) {
    constexpr int kWaves = 1024 / kWave;
    __shared__ unsigned long long shk[kWaves];
    __shared__ int shn[kWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    unsigned long long k = ~0ull;
    int64_t count = 0;
    for (int64_t i0 = 0; i0 < N; i0 += 1024) {
        const int64_t i = i0 + threadIdx.x;
        const int32_t l = i < N ? labels[i] : ignore;
        const bool on = i < N && vl_counts(l, ignore, V);
        if (i < N && !on && l != ignore && k == ~0ull) k = ((unsigned long long)i << 32) | (uint32_t)l;
        const unsigned long long mask = __ballot(on);
        __syncthreads();
        if (lane == 0) shn[wave] = __popcll(mask);
        __syncthreads();
        int64_t at = count;
        for (int w = 0; w < kWaves; w++) {
            if (w < wave) at += shn[w];
            count += shn[w];
        }
        if (on) {
            at += __popcll(mask & ((1ull << lane) - 1));
            from[at] = (int32_t)i;
            list[at] = l;
        }
    }
    for (int64_t i = count + threadIdx.x; i < padded; i += 1024) {
        from[i] = -1;
        list[i] = -1;
    }
    k = wave_min_u64(k);
    if (lane == 0) shk[wave] = k;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWaves; w++) k = shk[w] < k ? shk[w] : k;
        head->count = count;
        // at system scope: *bad may be host memory that the host watches while the kernel runs
        if (bad) __hip_atomic_store(bad, k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
}

// no loss and no gradient for the rows that do not count
__global__ __launch_bounds__(kVlB) void k_vl_off(const int32_t *__restrict__ labels, int64_t N, int64_t D, int64_t V, int32_t ignore,
                                                 float *__restrict__ row_loss, float *__restrict__ gx) {
    for (int64_t i = blockIdx.x; i < N; i += gridDim.x) {
        if (vl_counts(labels[i], ignore, V)) continue;
        if (row_loss && threadIdx.x == 0) row_loss[i] = 0.0f;
        if (gx)
            for (int64_t d = threadIdx.x; d < D; d += kVlB) gx[i * D + d] = 0.0f;
    }
}

__global__ __launch_bounds__(kVlB) void k_vl_clear(float *__restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * kVlB + threadIdx.x; i < n; i += (int64_t)gridDim.x * kVlB) p[i] = 0.0f;
}

// ---- operands in pieces ----------------------------------------------------------------------------------------------------
struct PackArgs {
    const float *s;
    int64_t ld, rows, cols;
    const int32_t *from;  // the rows' places, or none: as they lie
    const VlHead *head;   // counts the rows where they are listed
    char *out;
    int64_t step;         // bytes from a row block to the next
    int kblocks;
    int *e;               // by rows: their exponents
    int64_t slice;        // rows of a workgroup that looks for the columns' largest
    float *most;          // by columns: their largest sizes
};

// A workgroup's 32 rows, summed over by columns: each row's exponent, then its pieces.
__global__ __launch_bounds__(kVlB) void k_vl_pack_rows(PackArgs p) {
    __shared__ float sh[kVlB / 32][32];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, half = lane >> 5;
    const int64_t rb = blockIdx.x, r = rb * 32 + (lane & 31);
    const int64_t rows = p.from ? p.head->count : p.rows;
    const bool on = r < rows;
    const float *row = p.s + (on ? (p.from ? (int64_t)p.from[r] : r) : 0) * p.ld;
    auto load = [&](int kb, float (&x)[8]) {
        const int64_t k = 16 * (int64_t)kb + 8 * half;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = 0.0f;
        if (!on || k >= p.cols) return;
        if (k + 8 <= p.cols) {
            const f4 a = *(const f4u *)(row + k), b = *(const f4u *)(row + k + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = a[e], x[4 + e] = b[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (k + e < p.cols) x[e] = row[k + e];
        }
    };
    float most = 0.0f, x[8];
    for (int kb = wave; kb < p.kblocks; kb += kVlB / kWave) {
        load(kb, x);
#pragma unroll
        for (int e = 0; e < 8; e++) most = __builtin_fmaxf(most, finite_abs(x[e]));
    }
    sh[threadIdx.x / 32][lane & 31] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kVlB / 32; i++) most = __builtin_fmaxf(most, sh[i][lane & 31]);
    const int ex = piece_exponent(most);
    if (threadIdx.x < 32) p.e[r] = ex;
    const float scale = power(-ex);
    for (int kb = wave; kb < p.kblocks; kb += kVlB / kWave) {
        load(kb, x);
        const Pieces c = cut(x, scale);
        char *o = p.out + rb * p.step + (int64_t)kb * 2048 + lane * 16;
        *(h8 *)o = c.hi;
        *(h8 *)(o + 1024) = c.lo;
    }
}

// the columns' largest sizes
__global__ __launch_bounds__(kVlB) void k_vl_most(PackArgs p) {
    const int64_t d = (int64_t)blockIdx.x * kVlB + threadIdx.x;
    const int64_t rows = p.from ? p.head->count : p.rows;
    const int64_t r0 = (int64_t)blockIdx.y * p.slice, r1 = min(rows, r0 + p.slice);
    if (d >= p.cols || r0 >= r1) return;
    float most = 0.0f;
    for (int64_t r = r0; r < r1; r++) most = __builtin_fmaxf(most, finite_abs(p.s[(p.from ? (int64_t)p.from[r] : r) * p.ld + d]));
    atomicMax((unsigned int *)p.most + d, __float_as_uint(most));
}

// Columns as rows, summed over by rows; a wave's block of 32 columns by 16 rows.  TURNED: the k in the order that z's registers have.
template <bool TURNED>
__global__ __launch_bounds__(kVlB) void k_vl_pack_columns(PackArgs p) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, half = lane >> 5;
    const int64_t db = (int64_t)blockIdx.y * (kVlB / kWave) + wave, d = db * 32 + (lane & 31);
    const int64_t rows = p.from ? p.head->count : p.rows;
    if (db * 32 >= p.cols) return;
    const float scale = d < p.cols ? power(-piece_exponent(p.most[d])) : 0.0f;
    for (int kb = blockIdx.x; kb < p.kblocks; kb += gridDim.x) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int64_t k = 16 * (int64_t)kb + (TURNED ? 4 * half + (e & 3) + 8 * (e >> 2) : 8 * half + e);
            x[e] = d < p.cols && k < rows ? p.s[(p.from ? (int64_t)p.from[k] : k) * p.ld + d] : 0.0f;
        }
        const Pieces c = cut(x, scale);
        char *o = p.out + db * p.step + (int64_t)kb * 2048 + lane * 16;
        *(h8 *)o = c.hi;
        *(h8 *)(o + 1024) = c.lo;
    }
}

// ---- the rows' statistics and G ---------------------------------------------------------------------------------------------
struct GradArgs {
    const VlHead *head;
    int64_t row0, rows;  // of this piece: the first, how many (padded)
    int64_t V, words;    // words, padded
    const f2 *part;
    const float *label_z;
    const int32_t *labels, *from;  // of this piece's rows
    VlRow *row;
    double *losses;      // by place in the list
    float *row_loss;
    float *z;
    char *turned;
    int64_t turned_step;
    float *most;         // of every word of this piece
    double *column;      // [slices][words], or none
    int slices;
};

// lanes over 32 rows, eight of them over the partial statistics of each
__global__ __launch_bounds__(kVlB) void k_vl_stats(GradArgs p) {
    __shared__ double sh[kVlB / 32][32];
    __shared__ float shm[kVlB / 32][32];
    const int sub = threadIdx.x / 32, col = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * 32 + col;
    const int64_t parts = p.words / kStatWords;
    float m = -__builtin_inff();
    for (int64_t i = sub; i < parts; i += kVlB / 32) m = __builtin_fmaxf(m, p.part[i * p.rows + n].x);
    shm[sub][col] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kVlB / 32; i++) m = __builtin_fmaxf(m, shm[i][col]);
    double s = 0.0;
    for (int64_t i = sub; i < parts; i += kVlB / 32) {
        const f2 v = p.part[i * p.rows + n];
        s += (double)v.y * (double)(v.x == m ? 1.0f : exp8_nonpos(v.x - m));
    }
    sh[sub][col] = s;
    __syncthreads();
    if (sub != 0) return;
    double others = 0.0;
#pragma unroll
    for (int i = 0; i < kVlB / 32; i++) others += sh[i][col];
    const int label = p.labels[n];
    VlRow row = {0.0f, 0.0f, 0.0f, -1};
    if (p.row0 + n < p.head->count) {
        const float zl = p.label_z[n] - m;
        const double total = others + (double)exp8_nonpos(zl);
        const double ls = zl == 0.0f ? log1p(others) : log(total), loss = ls - (double)zl;
        p.losses[p.row0 + n] = loss;
        if (p.row_loss) p.row_loss[p.from[n]] = (float)loss;
        row = {m, (float)ls, (float)(-others / total), label};
    }
    p.row[n] = row;
}

// a lane's entry of G: word v of its row
__device__ __forceinline__ float g_entry(float z, int64_t v, const VlRow &row) {
    const float p = exp8_nonpos((z - row.m) - row.ls);
    return v == row.label ? row.own : p;
}

// Every word's largest entry of G in this piece and, SUM, the sum of them.  A wave takes 32 words and goes over its slice of the rows.
template <bool SUM>
__global__ __launch_bounds__(kVlB) void k_vl_words(GradArgs p) {
    const int lane = threadIdx.x & (kWave - 1), half = lane >> 5;
    const int64_t vb = (int64_t)blockIdx.x * (kVlB / kWave) + threadIdx.x / kWave, zwords = p.words / 32;
    const int64_t left = min(p.rows, p.head->count - p.row0), blocks = left > 0 ? (left + 31) / 32 : 0;
    const int64_t b0 = blocks * blockIdx.y / p.slices, b1 = blocks * (blockIdx.y + 1) / p.slices;
    float most[16];
    double sum[SUM ? 16 : 1];
#pragma unroll
    for (int r = 0; r < 16; r++) most[r] = -__builtin_inff();
#pragma unroll
    for (int r = 0; r < (SUM ? 16 : 1); r++) sum[r] = 0.0;
    for (int64_t nb = b0; nb < b1; nb++) {
        const VlRow row = p.row[nb * 32 + (lane & 31)];
        const float *z = p.z + (nb * zwords + vb) * 1024 + lane * 4;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const f4 v = *(const f4 *)(z + q * 256);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool own = vb * 32 + 8 * q + 4 * half + e == row.label;
                if constexpr (SUM) {
                    const float g = row.label < 0 ? 0.0f : g_entry(v[e], vb * 32 + 8 * q + 4 * half + e, row);
                    most[4 * q + e] = __builtin_fmaxf(most[4 * q + e], __builtin_fabsf(g));
                    sum[4 * q + e] += (double)g;
                } else {
                    // logarithms: the exponential of the largest is the largest
                    const float t = own ? 0.0f : (v[e] - row.m) - row.ls;
                    most[4 * q + e] = __builtin_fmaxf(most[4 * q + e], row.label < 0 ? -__builtin_inff() : t);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 16; r++) {
        float m = most[r];
        m = __builtin_fmaxf(m, __shfl_xor(m, 1));
        m = __builtin_fmaxf(m, __shfl_xor(m, 2));
        m = __builtin_fmaxf(m, __shfl_xor(m, 4));
        m = __builtin_fmaxf(m, __shfl_xor(m, 8));
        m = __builtin_fmaxf(m, __shfl_xor(m, 16));
        const int64_t v = vb * 32 + 8 * (r / 4) + 4 * half + r % 4;
        if (!SUM) m = exp8_nonpos(m);
        else m = m > 0.0f ? m : 0.0f;
        if ((lane & 31) == 0) atomicMax((unsigned int *)p.most + v, __float_as_uint(m));
        if constexpr (SUM) {
            double s = sum[r];
            for (int d = 1; d < 32; d *= 2) s += __shfl_xor(s, d);
            if ((lane & 31) == 0) p.column[(int64_t)blockIdx.y * p.words + v] = s;
        }
    }
}

// gb (+)= the slices' sums
__global__ __launch_bounds__(kVlB) void k_vl_bias(const double *__restrict__ column, int slices, int64_t words, int64_t V, const VlHead *head,
                                                  const float *gout, int sum, float *__restrict__ gb, int acc) {
    const int64_t v = (int64_t)blockIdx.x * kVlB + threadIdx.x;
    if (v >= V) return;
    double s = 0.0;
    for (int i = 0; i < slices; i++) s += column[(int64_t)i * words + v];
    const float c = vl_coef(head, gout, sum);
    gb[v] = head->count == 0 ? (acc ? gb[v] : 0.0f) : (acc ? fma_((float)s, c, gb[v]) : (float)s * c);
}

// G of a block of 32 rows by 32 words, in pieces: under the rows' exponents in z's place (X), and turned, under the words' (W).
template <bool X, bool W>
__global__ __launch_bounds__(kVlB) void k_vl_grad(GradArgs p) {
    __shared__ float turn[W ? kVlB / kWave : 1][32][33];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, half = lane >> 5, col = lane & 31;
    const int64_t vb = (int64_t)blockIdx.x * (kVlB / kWave) + wave, nb = blockIdx.y, zwords = p.words / 32;
    if (p.row0 + nb * 32 >= p.head->count) {
        return;  // gW does not read what lies behind the rows' last 32
    }
    const VlRow row = p.row[nb * 32 + col];
    float *z = p.z + (nb * zwords + vb) * 1024;
    float g[16];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const f4 v = *(const f4 *)(z + q * 256 + lane * 4);
#pragma unroll
        for (int e = 0; e < 4; e++) g[4 * q + e] = row.label < 0 ? 0.0f : g_entry(v[e], vb * 32 + 8 * q + 4 * half + e, row);
    }
    if constexpr (X) {
        const float scale = power(-piece_exponent(finite_abs(row.own)));
#pragma unroll
        for (int s = 0; s < 2; s++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = g[8 * s + e];
            const Pieces c = cut(x, scale);
            char *o = (char *)z + s * 2048 + lane * 16;
            *(h8 *)o = c.hi;
            *(h8 *)(o + 1024) = c.lo;
        }
    }
    if constexpr (W) {
#pragma unroll
        for (int r = 0; r < 16; r++) turn[wave][8 * (r / 4) + 4 * half + r % 4][col] = g[r];
        // the wave's own part of LDS: it reads what it wrote
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const float scale = power(-piece_exponent(p.most[vb * 32 + col]));
#pragma unroll
        for (int s = 0; s < 2; s++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = turn[wave][col][16 * s + 8 * half + e];
            const Pieces c = cut(x, scale);
            char *o = p.turned + vb * p.turned_step + (nb * 2 + s) * 2048 + lane * 16;
            *(h8 *)o = c.hi;
            *(h8 *)(o + 1024) = c.lo;
        }
    }
}

// gx (+)= the parts' sum, at the rows' places
__global__ __launch_bounds__(kVlB) void k_vl_gx(const float *__restrict__ parts, int slices, int64_t rows, int64_t cols, const VlHead *head,
                                                int64_t row0, const int32_t *__restrict__ from, const VlRow *__restrict__ row,
                                                const float *__restrict__ most, int64_t D, const float *gout, int sum, float *__restrict__ gx,
                                                int acc) {
    const int64_t left = min(rows, head->count - row0);
    const float c = vl_coef(head, gout, sum);
    for (int64_t n = blockIdx.x; n < left; n += gridDim.x) {
        const int en = piece_exponent(finite_abs(row[n].own));
        float *out = gx + (int64_t)from[n] * D;
        for (int64_t d = threadIdx.x; d < D; d += kVlB) {
            double s = 0.0;
            for (int i = 0; i < slices; i++) s += (double)parts[((int64_t)i * rows + n) * cols + d];
            const float v = __builtin_amdgcn_ldexpf((float)s, en + piece_exponent(most[d]));
            out[d] = acc ? fma_(v, c, out[d]) : v * c;
        }
    }
}

// the loss of no rows is NaN, as a mean over nothing is (a sum: 0)
__global__ __launch_bounds__(1024) void k_vl_total(const double *__restrict__ losses, const VlHead *__restrict__ head, int sum,
                                                   float *__restrict__ loss) {
    __shared__ double sh[1024 / kWave];
    double t = 0.0;
    for (int64_t i = threadIdx.x; i < head->count; i += 1024) t += losses[i];
    t = vl_wg_sum(t, sh);
    if (threadIdx.x == 0) *loss = sum ? (float)t : head->count ? (float)(t / (double)head->count) : __builtin_nanf("");
}

// ---- one call -----------------------------------------------------------------------------------------------------------------
struct SplitPlan {
    int64_t n, d, v;   // rows, columns and words, padded to tiles
    int64_t dk;        // columns, padded to two blocks of k
    int64_t piece;     // rows of a piece, padded
    int slices;        // of the words in gx
    int columns;       // slices of the rows in gb and the words' largest
    size_t from, list, losses, row, label_z, part, ew, ex, most_w, most_x, most_g, column, x1, x3, w1, w2, z, turned, parts, total;
};

static int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

static SplitPlan split_plan(int64_t N, int64_t D, int64_t V, bool want_x, bool want_w, bool want_b) {
    SplitPlan p{};
    const bool grad = want_x || want_w || want_b;
    p.n = up_to(N, kTile), p.d = up_to(D, kTile), p.v = up_to(V, kTile), p.dk = up_to(D, 32);
    const int64_t most = grad ? kZBytes / (8 * p.v) : kScored / p.v;
    p.piece = std::max<int64_t>(kTile, std::min(std::min(p.n, kPieceRows), most / kTile * kTile));
    // enough parts of gx for four rounds of workgroups, none with fewer than 64 blocks of k
    const int64_t tiles = p.piece / kTile * (p.d / kTile);
    p.slices = (int)std::max<int64_t>(1, std::min((4 * kPlanCUs + tiles - 1) / tiles, p.v / 16 / 64));
    p.columns = (int)std::max<int64_t>(1, std::min(p.piece / 32, (4096 + p.v / 32 - 1) / (p.v / 32)));
    size_t at = 256;
    auto take = [&](bool wanted, int64_t bytes) {
        const size_t here = at;
        if (wanted) at += vl_round256((size_t)bytes);
        return here;
    };
    p.from = take(true, p.n * 4);
    p.list = take(true, p.n * 4);
    p.losses = take(true, p.n * 8);
    p.row = take(true, p.piece * (int64_t)sizeof(VlRow));
    p.label_z = take(true, p.piece * 4);
    p.part = take(true, p.v / kStatWords * p.piece * 8);
    p.ew = take(true, p.v * 4);
    p.ex = take(true, p.n * 4);
    p.most_w = take(want_x, p.d * 4);
    p.most_x = take(want_w, p.d * 4);
    p.most_g = take(want_w || want_b, p.v * 4);
    p.column = take(want_b, p.columns * p.v * 8);
    p.x1 = take(true, p.n * p.dk * 4);
    p.x3 = take(want_w, p.d * p.n * 4);
    p.w1 = take(true, p.v * p.dk * 4);
    p.w2 = take(want_x, p.d * p.v * 4);
    p.z = take(grad, p.piece * p.v * 4);
    p.turned = take(want_w, p.piece * p.v * 4);
    p.parts = take(want_x, p.slices * p.piece * p.d * 4);
    p.total = at;
    return p;
}

bool vl_split_pays(int64_t N, int64_t D, int64_t V, bool grads) {
    (void)grads;
    return N >= 256 && N <= kPieceRows * 16 && D >= 64 && V >= 1024;
}

size_t vl_split_workspace(int64_t N, int64_t D, int64_t V, bool want_x, bool want_w, bool want_b) {
    return split_plan(N, D, V, want_x, want_w, want_b).total;
}

int vl_split_run(const VlCall &c, const char *what) {
    const SplitPlan pl = split_plan(c.N, c.D, c.V, c.gx, c.gw, c.gb);
    const bool grad = c.gx || c.gw || c.gb;
    auto at = [&](size_t off) { return c.ws + off; };
    VlHead *head = (VlHead *)c.ws;
    int32_t *from = (int32_t *)at(pl.from), *list = (int32_t *)at(pl.list);
    double *losses = (double *)at(pl.losses);
    hipLaunchKernelGGL(k_vl_list, 1, 1024, 0, c.st, c.labels, c.N, pl.n, c.V, c.ignore, head, from, list, c.bad);
    if (c.row_loss || (c.gx && !c.acc_x))
        hipLaunchKernelGGL(k_vl_off, (unsigned)std::min<int64_t>(c.N, 1 << 14), kVlB, 0, c.st, c.labels, c.N, c.D, c.V, c.ignore, c.row_loss,
                           c.acc_x ? nullptr : c.gx);

    PackArgs x{c.x, c.ldx, c.N, c.D, from, head, at(pl.x1), pl.dk * 128, (int)(pl.dk / 16), (int *)at(pl.ex), 0, nullptr};
    PackArgs w{c.w, c.ldw, c.V, c.D, nullptr, head, at(pl.w1), pl.dk * 128, (int)(pl.dk / 16), (int *)at(pl.ew), 0, nullptr};
    hipLaunchKernelGGL(k_vl_pack_rows, (unsigned)(pl.n / 32), kVlB, 0, c.st, x);
    hipLaunchKernelGGL(k_vl_pack_rows, (unsigned)(pl.v / 32), kVlB, 0, c.st, w);
    auto columns = [&](PackArgs a, size_t most, size_t out, int64_t k, bool turned) {
        a.most = (float *)at(most), a.out = at(out), a.step = k * 128, a.kblocks = (int)(k / 16);
        hipLaunchKernelGGL(k_vl_clear, (unsigned)((pl.d + kVlB - 1) / kVlB), kVlB, 0, c.st, a.most, pl.d);
        a.slice = std::max<int64_t>(256, (a.rows + 4095) / 4096);
        const dim3 g1((unsigned)((c.D + kVlB - 1) / kVlB), (unsigned)((a.rows + a.slice - 1) / a.slice));
        hipLaunchKernelGGL(k_vl_most, g1, kVlB, 0, c.st, a);
        const dim3 g2((unsigned)std::min<int64_t>(k / 16, 1 << 16), (unsigned)((c.D + 127) / 128));
        if (turned) hipLaunchKernelGGL(k_vl_pack_columns<true>, g2, kVlB, 0, c.st, a);
        else hipLaunchKernelGGL(k_vl_pack_columns<false>, g2, kVlB, 0, c.st, a);
    };
    if (c.gw) columns(x, pl.most_x, pl.x3, pl.n, false);
    if (c.gx) columns(w, pl.most_w, pl.w2, pl.v, true);

    auto product = [&](auto kernel, const MmArgs &m) {
        (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kMmLds);
        hipLaunchKernelGGL(kernel, (unsigned)(m.tiles_m * m.tiles_n * m.slices), kMmB, kMmLds, c.st, m);
    };
    for (int64_t r0 = 0; r0 < pl.n; r0 += pl.piece) {
        const int64_t rows = std::min(pl.piece, pl.n - r0);
        MmArgs m{};
        m.A = at(pl.w1), m.step_a = pl.dk * 128, m.B = at(pl.x1) + r0 / 32 * (pl.dk * 128), m.step_b = pl.dk * 128;
        m.tiles_m = (int)(pl.v / kTile), m.tiles_n = (int)(rows / kTile), m.slices = 1, m.kblocks = (int)(pl.dk / 16);
        m.head = head, m.row0 = r0, m.V = c.V, m.D = c.D;
        m.ew = (const int *)at(pl.ew), m.ex = (const int *)at(pl.ex) + r0, m.bias = c.bias, m.labels = list + r0;
        m.z = grad ? (float *)at(pl.z) : nullptr, m.zwords = pl.v / 32, m.part = (f2 *)at(pl.part), m.label_z = (float *)at(pl.label_z);
        m.rows = pl.piece;
        product(k_vl_product<MM_Z>, m);

        GradArgs g{};
        g.head = head, g.row0 = r0, g.rows = pl.piece, g.V = c.V, g.words = pl.v, g.part = m.part, g.label_z = m.label_z;
        g.labels = list + r0, g.from = from + r0, g.row = (VlRow *)at(pl.row), g.losses = losses, g.row_loss = c.row_loss;
        g.z = m.z, g.turned = at(pl.turned), g.turned_step = pl.piece * 128, g.most = (float *)at(pl.most_g), g.column = (double *)at(pl.column);
        g.slices = pl.columns;
        hipLaunchKernelGGL(k_vl_stats, (unsigned)(rows / 32), kVlB, 0, c.st, g);
        if (!grad) continue;
        if (c.gw || c.gb) {
            hipLaunchKernelGGL(k_vl_clear, (unsigned)((pl.v + kVlB - 1) / kVlB), kVlB, 0, c.st, g.most, pl.v);
            const dim3 gw((unsigned)(pl.v / 32 / (kVlB / kWave)), (unsigned)pl.columns);
            if (c.gb) hipLaunchKernelGGL(k_vl_words<true>, gw, kVlB, 0, c.st, g);
            else hipLaunchKernelGGL(k_vl_words<false>, gw, kVlB, 0, c.st, g);
            if (c.gb)
                hipLaunchKernelGGL(k_vl_bias, (unsigned)((c.V + kVlB - 1) / kVlB), kVlB, 0, c.st, g.column, pl.columns, pl.v, c.V, head, c.gout,
                                   c.sum, c.gb, c.acc_b || r0);
        }
        const dim3 gg((unsigned)(pl.v / 32 / (kVlB / kWave)), (unsigned)(rows / 32));
        if (c.gx && c.gw) hipLaunchKernelGGL((k_vl_grad<true, true>), gg, kVlB, 0, c.st, g);
        else if (c.gx) hipLaunchKernelGGL((k_vl_grad<true, false>), gg, kVlB, 0, c.st, g);
        else if (c.gw) hipLaunchKernelGGL((k_vl_grad<false, true>), gg, kVlB, 0, c.st, g);
        if (c.gx) {
            MmArgs a = m;
            a.A = (const char *)m.z, a.step_a = pl.v * 128, a.B = at(pl.w2), a.step_b = pl.v * 128;
            a.tiles_m = (int)(rows / kTile), a.tiles_n = (int)(pl.d / kTile), a.slices = pl.slices, a.kblocks = (int)(pl.v / 16);
            a.parts = (float *)at(pl.parts), a.cols = pl.d;
            product(k_vl_product<MM_GX>, a);
            hipLaunchKernelGGL(k_vl_gx, (unsigned)std::min<int64_t>(rows, 1 << 14), kVlB, 0, c.st, a.parts, pl.slices, pl.piece, pl.d, head, r0,
                               from + r0, g.row, (const float *)at(pl.most_w), c.D, c.gout, c.sum, c.gx, c.acc_x);
        }
        if (c.gw) {
            MmArgs a = m;
            a.A = g.turned, a.step_a = g.turned_step, a.B = at(pl.x3) + r0 / 16 * 2048, a.step_b = pl.n * 128;
            a.tiles_m = (int)(pl.v / kTile), a.tiles_n = (int)(pl.d / kTile), a.kblocks = (int)(rows / 16);
            a.most_a = g.most, a.most_b = (const float *)at(pl.most_x), a.gout = c.gout, a.out = c.gw, a.sum = c.sum, a.acc = c.acc_w || r0;
            product(k_vl_product<MM_GW>, a);
        }
    }
    hipLaunchKernelGGL(k_vl_total, 1, 1024, 0, c.st, losses, head, c.sum, c.loss);
    return check_launch(what);
}

}  // namespace nchip
