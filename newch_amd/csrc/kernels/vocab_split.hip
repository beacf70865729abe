// The vocabulary loss with its three products on the fp16 matrix cores: z = x W^T, gx = G W, gW = G^T x.
//
// A library's fp32 product of 8192^3 reaches an eighth of what its fp16 one does, so operands are cut into two fp16 pieces under a
// power of two of their row: x = 2^e (hi + lo), the row's largest finite value in [2^14, 2^15) after the scaling, hi and lo rounded to
// nearest.  A product is hi hi + hi lo + lo hi, summed in fp32; lo lo, at most 2^-22 of a term, is left out.
//
// fp16 has its 11 bits down to 2^-14 only, and steps of 2^-24 below.  So x and W keep lo as 2^11 lo, and the factors 2^-11 that their
// products then need are taken out of fragments in registers.  gx and gW: out of G's hi, so that every value of W and x has its 22 bits down to
// 2^-28 of its row's largest (an absolute error of 2^-50 of that below), and a column that is small in all rows its gradient's bits.  z:
// halves of it out of all four pieces, 22 bits down to 2^-22 and 2^-44 below, so that columns which x and W scale oppositely cost
// nothing.  G's own lo is kept as it is: what is below 2^-17 of the largest term of a sum, and so held to 2^-39 of it, is lost in that sum.
//
// x and W are packed once, by rows.  gx and gW sum over those rows, so G takes their powers of two: gx_n = sum_v (G_nv 2^e_v) pieces of W_v,
// where the row n of G 2^e has the power of its own largest entry, which is that of the largest term that gx_n sums; gW in
// the same way.  So rows of x or W far larger than those that a result counts leave those their bits.
//
// A packed block, 32 rows by 16 k, is 2 KiB: for each half of the rows 256 bytes of hi of k 0 .. 7, of hi of k 8 .. 15, and of lo of both;
// a row's eight k are 16 bytes, at place r % 16 ^ 8 (k / 8).  Blocks go into LDS as they lie, a KiB an instruction, and give
// v_mfma_f32_32x32x16_f16's fragments from there: rows that are not summed over by one 16-byte read of a lane (row l % 32, k of half
// l / 32), rows that are by two transposing 8-byte reads (column l % 32 of 32, rows 4 (l / 32) + {0, 1, 2, 3, 8, 9, 10, 11} of a half).
// That is the order in which a result's registers hold rows, so z's blocks are left as the registers hold them -- 32 rows n by 32 words v
// in 4 KiB, lane l with n = l % 32 and v = 8 q + 4 (l / 32) + e, q and e < 4 -- and G's pieces take z's place without leaving their lanes.
//
// Steps of a call: labels that count are listed (rows that do not count take part in nothing); x and W are packed; then for pieces of the
// rows z, with each row's maximum, sum of exponentials and largest term of gx over every 128 words; the rows' statistics; the largest
// terms of gW of every word; G in pieces for both products (in z's place, and turned for gW); gx in parts over the words and their
// sum; gW.  Scoring ends with the rows' statistics and leaves no z.
#include "vocab_loss.hpp"

namespace nchip {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16x __attribute__((ext_vector_type(16)));
typedef int i4v __attribute__((ext_vector_type(4)));

// A workgroup's product: 256 rows by 64 columns for each of its WN pairs of waves, WN 2 or 4; kStages blocks of 16 k in LDS.
constexpr int kTileM = 256, kTileMost = 256;
constexpr int kStages = 3;
template <int WN>
struct Tile {
    static constexpr int kN = 64 * WN, kLanes = 128 * WN;
    static constexpr uint32_t kStageA = kTileM * 16 * 4, kStage = (kTileM + kN) * 16 * 4;  // bytes: the rows of A, all
    static constexpr int kLds = kStages * kStage;
    static constexpr int kA = 4 / WN;                // row blocks of A that a wave brings, besides one of B
    static constexpr int kLoads = 2 * (kA + 1);      // and the KiB that these are
};
constexpr int64_t kZBytes = int64_t(4) << 30;  // of z and of the turned G, both together, held at a time
constexpr int64_t kPieceRows = 1 << 20;
constexpr int64_t kPartBytes = int64_t(512) << 20;  // of the parts of gx; of those of gW; of the statistics where no z is held
constexpr int kStatWords = 128;  // words of one partial statistic

constexpr float kLog2e = 1.44269504088896341f;

struct VlRow {
    float m, ls;  // the row's maximum and log sum exp(z - m)
    float own;    // p_l - 1
    int label;    // -1: no row
    int e;        // the power of two of its row of G 2^e_v
    int ex;       // of its row of x
    int pad[2];
};
// of 128 words of a row: the maximum, the sum of exponentials from there, the largest term of gx (a base-2 logarithm from there)
struct VlPart {
    float m, s, c;
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

// The largest of a word's or a row's terms is kept as the whole part of its base-2 logarithm; kNoTerm: there is none.
constexpr int kNoTerm = -400;
__device__ __forceinline__ int term_exponent(float log2) { return log2 > (float)kNoTerm ? (int)__builtin_floorf(__builtin_fminf(log2, 400.0f)) : kNoTerm; }
__device__ __forceinline__ int word_exponent(int term) { return term - 14; }

struct Pieces {
    h8 hi, lo;
};
constexpr int kLow = 11;  // x and W keep 2^kLow lo
template <int LOW>
__device__ __forceinline__ Pieces cut(const float (&x)[8], float scale) {
    Pieces r;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = x[i] * scale;
        const _Float16 h = (_Float16)v;
        r.hi[i] = h;
        r.lo[i] = (_Float16)((v - (float)h) * (float)(1 << LOW));
    }
    return r;
}

// a lane's place in a packed block: row l % 32, k of half l / 32
__device__ __forceinline__ int block_at(int lane) {
    const int half = lane >> 5, r = lane & 31;
    return (r >> 4) * 1024 + half * 256 + ((r & 15) ^ (8 * half)) * 16;
}
__device__ __forceinline__ void store_block(char *block, int lane, const Pieces &c) {
    char *o = block + block_at(lane);
    *(h8 *)o = c.hi;
    *(h8 *)(o + 512) = c.lo;
}

// ---- the product ------------------------------------------------------------------------------------------------------
enum { MM_Z = 0, MM_GX = 1, MM_GW = 2, MM_GW_PARTS = 3, MM_SCORE = 4 };  // MM_SCORE: z, not kept

struct MmArgs {
    const char *A, *B;      // packed; blocks of a row block follow each other
    int64_t step_a, step_b;  // bytes from a row block to the next
    int tiles_m, tiles_n;   // at most
    int kblocks;            // of 16 k: an even number, as each slice's is
    const VlHead *head;
    int64_t row0;           // of this piece, among the rows that count
    int64_t V, D;
    // MM_Z: A the words, B the rows
    const int *ew, *ex;
    const float *bias;
    const int32_t *labels;  // of this piece's rows
    float *z;               // MM_Z
    int64_t zwords;         // blocks of 32 words of a row block
    VlPart *part;           // [words / kStatWords][rows]
    float *label_z;         // [rows]
    int64_t rows;           // of a piece, padded
    // MM_GX: A the rows, B the words; MM_GW: A the words, B the rows; of B the columns, `blocks` of 16
    int blocks;
    float *parts;           // MM_GX, MM_GW_PARTS: [slices][rows or words][columns]
    int64_t part_rows, cols;  // rows or words, and columns, padded
    const int *eg;          // MM_GW: the largest terms' exponents of the words
    const float *gout;
    float *out;
    int sum, acc;
};

struct Frags {
    h8 a[4][2], b[2][2];
};

// What the sums of gx, gW and gb are multiplied by, as m 2^e with 1 <= |m| < 2: the sums are in pieces' powers, and with 2^e taken
// into those no step passes a float's range unless the result does (gW sums N rows, of which the mean may be all that is a float).
struct VlCoef {
    float m;
    int e;
};
__device__ __forceinline__ VlCoef vl_coef(const VlHead *head, const float *gout, int sum) {
    const float c = gout ? *gout : 1.0f, v = sum ? c : c / (float)head->count;
    return {2.0f * __builtin_amdgcn_frexp_mantf(v), __builtin_amdgcn_frexp_expf(v) - 1};
}

// The wave's 128 words by 64 rows of z, out of its accumulators.
template <bool KEEP>
__device__ __forceinline__ void z_out(const MmArgs &p, f16x (&acc)[4][2], int64_t v0, int64_t n0, int lane) {
    const int half = lane >> 5, ex[2] = {p.ex[n0 + (lane & 31)], p.ex[n0 + 32 + (lane & 31)]};
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int64_t v = v0 + 32 * i + 8 * q + 4 * half;
            const i4v ew = *(const i4v *)(p.ew + v);
            f4 b = {};
            if (p.bias) {
                if (v + 4 <= p.V) b = *(const f4u *)(p.bias + v);
                else
                    for (int e = 0; e < 3; e++)
                        if (v + e < p.V) b[e] = p.bias[v + e];
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                f4 z;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    z[e] = __builtin_amdgcn_ldexpf(acc[i][j][4 * q + e], ew[e] + ex[j]) + b[e];
                    z[e] = v + e < p.V ? z[e] : -__builtin_inff();
                    acc[i][j][4 * q + e] = z[e];
                }
                if (KEEP) *(f4 *)(p.z + ((n0 / 32 + j) * p.zwords + v0 / 32 + i) * 1024 + q * 256 + lane * 4) = z;
            }
        }
        // a block of words at a time: the accumulators leave no registers to load ahead
        asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1])::"memory");
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int64_t n = n0 + 32 * j + (lane & 31);
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
        float s = 0.0f, c = -__builtin_inff();
        const float base = m == -__builtin_inff() ? 0.0f : m;  // words that are all -inf have no part in the row's sum
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                i4v ew = {};
                if (KEEP) ew = *(const i4v *)(p.ew + v0 + 32 * i + 8 * q + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float t = (acc[i][j][4 * q + e] - base) * kLog2e;
                    s += __builtin_amdgcn_exp2f(t);
                    if (KEEP) c = __builtin_fmaxf(c, t + (float)ew[e]);
                }
            }
        s += __shfl_xor(s, 32);
        c = __builtin_fmaxf(c, __shfl_xor(c, 32));
        if (half == 0) p.part[(v0 / kStatWords) * p.rows + n] = {m, s, c};
    }
}

// How many parts a sum is cut into, of 64 at most: of few tiles' products, as many as make the rounds of workgroups full.  A wave's lanes
// try one number each.  In units of a block of 16 k of a tile: a round costs its blocks and some 24 to start and to leave, and a part of a
// tile an eighth of one on its way through memory.
__device__ __forceinline__ int parts_of(int64_t tiles, int kblocks, int most, int at_once) {
    const int s = (int)(threadIdx.x & (kWave - 1)) + 1;
    const int64_t rounds = (tiles * s + at_once - 1) / at_once;
    const int64_t cost = rounds * ((kblocks + s - 1) / s + 24) + tiles * s * kPlanCUs / (8 * at_once);
    const unsigned long long key = s <= most ? (unsigned long long)cost << 8 | (unsigned)s : ~0ull;
    return (int)max(1ull, wave_min_u64(key) & 0xff) & 0x7f;
}

// WN 2: two workgroups a CU, so that one multiplies while the other starts or leaves, and fewer that wait for the last.  WN 4: one, which
// brings three quarters as much for a product.
template <int WHAT, int WN>
__global__ __launch_bounds__(Tile<WN>::kLanes, 2) void k_vl_product(MmArgs p) {
    using T = Tile<WN>;
    constexpr uint32_t kStage = T::kStage;
    constexpr bool kZ = WHAT == MM_Z || WHAT == MM_SCORE;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave & 1, wn = wave >> 1;
    const int64_t left = p.head->count - p.row0;  // rows of this piece and behind it
    const int slices = WHAT == MM_GX ? p.head->slices_x : WHAT == MM_GW_PARTS ? p.head->slices_w : 1;
    const uint32_t tiles_m = WHAT == MM_GX ? (uint32_t)(left > 0 ? (min(left, p.rows) + kTileM - 1) / kTileM : 0) : (uint32_t)p.tiles_m;
    const uint32_t tiles_n = kZ ? (uint32_t)(left > 0 ? (min(left, p.rows) + T::kN - 1) / T::kN : 0) : (uint32_t)p.tiles_n;
    const uint32_t tiles = tiles_m * tiles_n, nblk = tiles * (uint32_t)slices;
    if (blockIdx.x >= nblk) return;
    // XCD x runs the workgroups b with b % 8 == x: it gets the x-th of 8 runs of tiles, in groups of 8 tile rows
    const uint32_t xcd = blockIdx.x & 7, per = nblk >> 3, rem = nblk & 7;
    const uint32_t id = xcd * per + min(xcd, rem) + (blockIdx.x >> 3);
    const int slice = (int)(id / tiles), tile = (int)(id % tiles);
    const int per_group = 8 * (int)tiles_n, group = tile / per_group, in_group = tile % per_group;
    const int gsize = min((int)tiles_m - group * 8, 8);
    const int tm = group * 8 + in_group % gsize, tn = in_group / gsize;
    int k0 = 0, k1 = p.kblocks;
    if (WHAT == MM_GW || WHAT == MM_GW_PARTS) k1 = (int)min((int64_t)p.kblocks, left > 0 ? (left + 31) / 32 * 2 : 0);
    if (WHAT == MM_GW && k1 == 0 && p.acc) return;
    if (WHAT == MM_GX || WHAT == MM_GW_PARTS) {
        const int64_t pairs = k1 / 2;
        k0 = 2 * (int)(pairs * slice / slices), k1 = 2 * (int)(pairs * (slice + 1) / slices);
    }
    const int nk = k1 - k0;
    const int64_t m0 = (int64_t)tm * kTileM + 128 * wm, n0 = (int64_t)tn * T::kN + 64 * wn;
    // a wave whose columns no result has only brings its share
    const bool works = n0 < (kZ ? left : p.D);

    // each wave brings its share of a stage: the pieces of kA row blocks of A and of one of B
    const char *src_a = p.A + ((int64_t)tm * (kTileM / 32) + T::kA * wave) * p.step_a + (int64_t)k0 * 2048 + lane * 16;
    // of B: its row block's 2 KiB, or, where B's rows are summed over, half a block, 16 rows, of two blocks of columns (behind the
    // last columns the last block again)
    constexpr bool kTurned = !kZ;
    const int db = min(p.blocks - 1, tn * (T::kN / 16) + 2 * wave), db1 = min(p.blocks - 1, db + 1);
    const char *src_b = kTurned ? p.B + k0 / 2 * p.step_b + db * 2048 + lane * 16
                                : p.B + ((int64_t)tn * (T::kN / 32) + wave) * p.step_b + (int64_t)k0 * 2048 + lane * 16;
    const int next_b = kTurned ? (db1 - db) * 2048 : 1024;
    const int64_t odd_b = kTurned ? p.step_b - 1024 : 2048, even_b = kTurned ? 1024 : 2048;
    int brought = 0;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const uint32_t to_a = base + (uint32_t)wave * (2048 * T::kA), to_b = base + T::kStageA + (uint32_t)wave * 2048;
    auto bring = [&](uint32_t stage) {
        const uint32_t a = __builtin_amdgcn_readfirstlane(to_a + stage), b = __builtin_amdgcn_readfirstlane(to_b + stage);
#pragma unroll
        for (int i = 0; i < T::kA; i++) {
            dma16(src_a + i * p.step_a, a + 2048 * i);
            dma16(src_a + i * p.step_a + 1024, a + 2048 * i + 1024);
        }
        dma16(src_b, b);
        dma16(src_b + next_b, b + 1024);
        src_a += 2048, src_b += brought++ & 1 ? odd_b : even_b;
    };
    const char *const my_a = lds + wm * 8192 + block_at(lane), *const my_b = lds + T::kStageA + wn * 4096;
    // the transposing reads' places: 16 lanes bring four rows of 16 columns, four columns a lane
    const int u = (lane >> 1) & 1, row = 4 * (lane >> 5) + (lane & 15) / 4;
    const int turned = ((lane >> 4) & 1) * 1024 + u * 256 + (row + 8 * u) * 16 + 8 * (lane & 1);
    auto fetch = [&](uint32_t stage, Frags &f) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f.a[i][0] = *(const h8 *)(my_a + stage + i * 2048);
            f.a[i][1] = *(const h8 *)(my_a + stage + i * 2048 + 512);
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                if constexpr (kTurned) {
                    typedef short s4 __attribute__((ext_vector_type(4)));
                    typedef short s8 __attribute__((ext_vector_type(8)));
                    typedef __attribute__((address_space(3))) s4 lds_s4;
                    const char *q = my_b + stage + j * 2048 + t * 512 + turned;
                    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(q));
                    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(q + 128 - 256 * u));
                    f.b[j][t] = __builtin_bit_cast(h8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
                } else {
                    f.b[j][t] = *(const h8 *)(my_b + stage + j * 2048 + t * 512 + block_at(lane));
                }
            }
    };
    f16x acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = f16x{};
    // hi hi, then the pieces scaled in place, then hi lo and lo hi
    auto product = [&](const Frags &f, int a, int b) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.a[i][a], f.b[j][b], acc[i][j], 0, 0, 0);
    };
    auto multiply = [&](Frags &f) {
        constexpr _Float16 kHalf = (_Float16)(1.0f / (1 << kLow / 2)), kRest = (_Float16)(1.0f / (1 << (kLow - kLow / 2)));
        product(f, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f.a[i][0] *= kZ ? kHalf : (_Float16)(1.0f / (1 << kLow));
            if (kZ) f.a[i][1] *= kRest;
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
            if (kZ) f.b[j][0] *= kHalf, f.b[j][1] *= kRest;
        product(f, 0, 1);
        product(f, 1, 0);
    };
    // At the barrier before block kt every wave's share of block kt + 1 is in LDS and every wave holds block kt in registers, so its
    // stage takes block kt + 3.  A wave reads block kt + 1 into registers while it multiplies block kt.
    auto wait = [&](int kt) {  // this wave's loads of block kt + 1 have landed; those of kt + 2 may be on their way
        if (kt + 2 < nk) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
    };
    if (nk > 0) {
        bring(0);
        bring(kStage);
        if (nk > 2) bring(2 * kStage);
        if (nk > 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * T::kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
        Frags f0, f1;
        uint32_t here = 0;  // the stage of block kt
        auto after = [](uint32_t stage) { return stage == 2 * kStage ? 0u : stage + kStage; };
        if (works) {
            fetch(0, f0);
            for (int kt = 0; kt < nk; kt += 2) {  // behind the last block a stage is read again, for nothing
                const uint32_t next = after(here), next2 = after(next);
                wait(kt);
                if (kt + 3 < nk) bring(here);
                fetch(next, f1);
                __builtin_amdgcn_sched_barrier(0);
                multiply(f0);
                wait(kt + 1);
                if (kt + 4 < nk) bring(next);
                fetch(next2, f0);
                __builtin_amdgcn_sched_barrier(0);
                multiply(f1);
                here = next2;
            }
        } else {
            for (int kt = 0; kt < nk; kt++) {
                wait(kt);
                if (kt + 3 < nk) bring(here);
                here = after(here);
            }
        }
    }
    if (!works) return;

    // what the results need is computed behind the products, whose registers it would take
    int at = lane;
    asm volatile("" : "+v"(at)::"memory");
    if constexpr (kZ) {
        z_out<WHAT == MM_Z>(p, acc, m0, n0, at);
    } else if constexpr (WHAT == MM_GX || WHAT == MM_GW_PARTS) {
        // a store instruction writes 32 columns of two rows
        float *out = p.parts + ((int64_t)slice * p.part_rows + m0 + 4 * (at >> 5)) * p.cols + n0 + (at & 31);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int r = 0; r < 16; r++)
#pragma unroll
                for (int j = 0; j < 2; j++) out[(32 * i + 8 * (r / 4) + r % 4) * p.cols + 32 * j] = acc[i][j][r];
    } else {
        const VlCoef c = nk > 0 ? vl_coef(p.head, p.gout, p.sum) : VlCoef{0.0f, 0};
        const int64_t m1 = m0 + 4 * (at >> 5), d = n0 + (at & 31);
        float *out = p.out + m1 * p.D + d;
        const bool in0 = d < p.D, in1 = d + 32 < p.D;
        // the old values of 16 rows are asked for together
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float old[2][16];
            if (p.acc) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int dm = 32 * i + 8 * (r / 4) + r % 4;
                    const float *o = out + (int64_t)dm * p.D;
                    old[0][r] = m1 + dm < p.V && in0 ? o[0] : 0.0f;
                    old[1][r] = m1 + dm < p.V && in1 ? o[32] : 0.0f;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int dm = 32 * i + 8 * (r / 4) + r % 4;
                if (m1 + dm >= p.V) continue;
                const int em = word_exponent(p.eg[m1 + dm]) + c.e;
                float *o = out + (int64_t)dm * p.D;
                const float v0 = __builtin_amdgcn_ldexpf(acc[i][0][r], em), v1 = __builtin_amdgcn_ldexpf(acc[i][1][r], em);
                if (in0) o[0] = p.acc ? fma_(v0, c.m, old[0][r]) : v0 * c.m;
                if (in1) o[32] = p.acc ? fma_(v1, c.m, old[1][r]) : v1 * c.m;
            }
        }
    }
}

// ---- which rows count ----------------------------------------------------------------------------------------------------
// Workgroup 0 lists the rows that count and their labels (-1 behind the last), and looks for the first label that is neither a word
// nor `ignore`; the others set what grows from nothing: the words' largest terms, the losses and gradients of the rows that do not count.
__global__ __launch_bounds__(1024) void k_vl_begin(const int32_t *__restrict__ labels, int64_t N, int64_t padded, int64_t D, int64_t V,
                                                   int32_t ignore, VlHead *head, int32_t *__restrict__ from, int32_t *__restrict__ list,
                                                   unsigned long long *bad, int *__restrict__ terms, int64_t n_terms,
                                                   float *__restrict__ row_loss, float *__restrict__ gx) {
    constexpr int kB = 1024, kWaves = kB / kWave;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    if (blockIdx.x > 0) {
        const int64_t block = blockIdx.x - 1, blocks = gridDim.x - 1;
        for (int64_t i = block * kB + threadIdx.x; i < n_terms; i += blocks * kB) terms[i] = kNoTerm;
        for (int64_t i = block * kWaves + wave; i < N; i += blocks * kWaves) {
            if (vl_counts(labels[i], ignore, V)) continue;
            if (row_loss && lane == 0) row_loss[i] = 0.0f;
            if (gx)
                for (int64_t d = lane; d < D; d += kWave) gx[i * D + d] = 0.0f;
        }
        return;
    }
    __shared__ unsigned long long shk[kWaves];
    __shared__ int shn[kWaves];
    unsigned long long k = ~0ull;
    int64_t count = 0;
    for (int64_t i0 = 0; i0 < N; i0 += kB) {
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
    for (int64_t i = count + threadIdx.x; i < padded; i += kB) {
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

// ---- operands in pieces ----------------------------------------------------------------------------------------------------
struct PackArgs {
    const float *s;
    int64_t ld, rows, cols;
    const int32_t *from;  // the rows' places, or none: as they lie
    const VlHead *head;   // counts the rows where they are listed
    int *e;               // the rows' exponents
    char *out;
    int groups;           // of 32 rows, padded
};
struct PackPair {
    PackArgs a[2];  // x, W
    int kblocks;
};

// A workgroup's 32 rows.  A lane has eight k of its row in every eighth block, up to NB of them in registers (NB 0: more, read again once
// the rows' largest values are known).
template <int NB>
__global__ __launch_bounds__(512) void k_vl_pack(PackPair pp) {
    constexpr int kWaves = 8, kHold = NB ? NB : 4;
    __shared__ float sh[2 * kWaves][32];
    const bool second = (int)blockIdx.x >= pp.a[0].groups;
    const PackArgs &p = pp.a[second];
    const int64_t rb = blockIdx.x - (second ? pp.a[0].groups : 0);
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, half = lane >> 5, col = lane & 31;
    const int64_t r = rb * 32 + col;
    const bool on = r < (p.from ? p.head->count : p.rows);
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
    float x[kHold][8], most = 0.0f;
    for (int k0 = 0; k0 < (NB ? 1 : pp.kblocks); k0 += kHold * kWaves) {
#pragma unroll
        for (int i = 0; i < kHold; i++) load(k0 + wave + i * kWaves, x[i]);
#pragma unroll
        for (int i = 0; i < kHold; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) most = __builtin_fmaxf(most, finite_abs(x[i][e]));
    }
    sh[threadIdx.x / 32][col] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * kWaves; i++) most = __builtin_fmaxf(most, sh[i][col]);
    const int ex = piece_exponent(most);
    if (threadIdx.x < 32) p.e[r] = ex;
    const float scale = power(-ex);
    char *out = p.out + rb * pp.kblocks * 2048;
    for (int k0 = 0; k0 < (NB ? 1 : pp.kblocks); k0 += kHold * kWaves) {
#pragma unroll
        for (int i = 0; i < kHold; i++) {
            const int kb = k0 + wave + i * kWaves;
            if (kb >= pp.kblocks) break;
            if (!NB) load(kb, x[i]);
            store_block(out + (int64_t)kb * 2048, lane, cut<kLow>(x[i], scale));
        }
    }
}

// ---- the rows' statistics and G ---------------------------------------------------------------------------------------------
// of a product whose sum is cut: tiles over the columns, parts at most, workgroups that the chip holds
struct PartPlan {
    int tiles_n, most, at_once;
};

struct GradArgs {
    VlHead *head;
    int64_t row0, rows;  // of this piece: the first, how many (padded)
    int64_t V, words;    // words, padded
    const VlPart *part;
    const float *label_z;
    const int32_t *labels, *from;  // of this piece's rows
    const int *ex, *ew;  // the exponents of this piece's rows, of the words
    VlRow *row;
    double *losses;      // by place in the list
    float *row_loss;
    float *z;
    char *turned;
    int64_t turned_step;
    int *term;           // of every word of this piece, or none
    float *column;       // [rows / 32][words], or none
    int slices;          // of the rows where the words' largest are looked for
    PartPlan of_x, of_w;
};

// lanes over 32 rows, 32 of them over the partial statistics of each; and what the next steps of this piece need
__global__ __launch_bounds__(1024) void k_vl_stats(GradArgs p) {
    constexpr int kSubs = 1024 / 32;
    __shared__ double sh[kSubs][32];
    __shared__ float shm[kSubs][32];
    if (p.term && p.row0 > 0)  // the first piece finds them set
        for (int64_t v = (int64_t)blockIdx.x * 1024 + threadIdx.x; v < p.words; v += (int64_t)gridDim.x * 1024) p.term[v] = kNoTerm;
    const int64_t left = p.head->count - p.row0;
    if (blockIdx.x == 0 && threadIdx.x < 2 * kWave) {
        const bool w = threadIdx.x >= kWave;
        const int64_t here = max(int64_t(0), min(p.rows, left));
        const PartPlan &q = w ? p.of_w : p.of_x;
        const int64_t tiles_m = w ? p.words / kTileM : (here + kTileM - 1) / kTileM;
        const int64_t kblocks = w ? (here + 31) / 32 * 2 : p.words / 16;
        const int n = parts_of(tiles_m * q.tiles_n, (int)kblocks, q.most, q.at_once);
        if ((threadIdx.x & (kWave - 1)) == 0) (w ? p.head->slices_w : p.head->slices_x) = n;
    }
    const int sub = threadIdx.x / 32, col = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * 32 + col;
    const int64_t parts = p.words / kStatWords;
    float m = -__builtin_inff();
#pragma unroll 4
    for (int64_t i = sub; i < parts; i += kSubs) m = __builtin_fmaxf(m, p.part[i * p.rows + n].m);
    shm[sub][col] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSubs; i++) m = __builtin_fmaxf(m, shm[i][col]);
    double s = 0.0;
    float c = -__builtin_inff();
#pragma unroll 4
    for (int64_t i = sub; i < parts; i += kSubs) {
        const VlPart v = p.part[i * p.rows + n];
        s += (double)v.s * (double)(v.m == m ? 1.0f : exp8_nonpos(v.m - m));
        c = __builtin_fmaxf(c, v.m == m ? v.c : v.c + (v.m - m) * kLog2e);
    }
    __syncthreads();
    sh[sub][col] = s;
    shm[sub][col] = c;
    __syncthreads();
    if (sub != 0) return;
    double others = 0.0;
#pragma unroll
    for (int i = 0; i < kSubs; i++) {
        others += sh[i][col];
        c = __builtin_fmaxf(c, shm[i][col]);
    }
    const int label = p.labels[n];
    VlRow row = {0.0f, 0.0f, 0.0f, -1, 0, p.ex[n], {}};
    if (n < left) {
        const float zl = p.label_z[n] - m;
        const double total = others + (double)exp8_nonpos(zl);
        const double ls = zl == 0.0f ? log1p(others) : log(total), loss = ls - (double)zl;
        p.losses[p.row0 + n] = loss;
        if (p.row_loss) p.row_loss[p.from[n]] = (float)loss;
        row.m = m, row.ls = (float)ls, row.own = (float)(-others / total), row.label = label;
        const float term = __builtin_fmaxf(c - row.ls * kLog2e, __builtin_log2f(__builtin_fabsf(row.own)) + (float)p.ew[label]);
        row.e = word_exponent(term_exponent(term));
    }
    p.row[n] = row;
}

// a lane's entry of G: word v of its row
__device__ __forceinline__ float g_entry(float z, int64_t v, const VlRow &row) {
    const float p = exp8_nonpos((z - row.m) - row.ls);
    return v == row.label ? row.own : p;
}

// Every word's largest term of gW in this piece.  A wave takes 32 words and goes over its slice of the rows.
__global__ __launch_bounds__(kVlB) void k_vl_words(GradArgs p) {
    const int lane = threadIdx.x & (kWave - 1), half = lane >> 5;
    const int64_t vb = (int64_t)blockIdx.x * (kVlB / kWave) + threadIdx.x / kWave, zwords = p.words / 32;
    const int64_t left = min(p.rows, p.head->count - p.row0), blocks = left > 0 ? (left + 31) / 32 : 0;
    const int64_t b0 = blocks * blockIdx.y / p.slices, b1 = blocks * (blockIdx.y + 1) / p.slices;
    float most[16];  // logarithms of the terms' sizes
#pragma unroll
    for (int r = 0; r < 16; r++) most[r] = -__builtin_inff();
    for (int64_t nb = b0; nb < b1; nb++) {
        const VlRow row = p.row[nb * 32 + (lane & 31)];
        const float *z = p.z + (nb * zwords + vb) * 1024 + lane * 4;
        const float e = row.label < 0 ? -__builtin_inff() : (float)row.ex;
        const float of_own = __builtin_log2f(__builtin_fabsf(row.own));
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const f4 v = *(const f4 *)(z + q * 256);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float t = ((v[k] - row.m) - row.ls) * kLog2e;
                most[4 * q + k] = __builtin_fmaxf(most[4 * q + k], (vb * 32 + 8 * q + 4 * half + k == row.label ? of_own : t) + e);
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
        if ((lane & 31) == 0) atomicMax(p.term + v, term_exponent(m));
    }
}

// G of a block of 32 rows by 32 words, in pieces: under the rows' powers in z's place (X), and turned, under the words' (W),
// with the sums of its columns where gb wants them.
template <bool X, bool W>
__global__ __launch_bounds__(kVlB) void k_vl_grad(GradArgs p) {
    __shared__ float turn[W ? kVlB / kWave : 1][32][33];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, half = lane >> 5, col = lane & 31;
    const int64_t vb = (int64_t)blockIdx.x * (kVlB / kWave) + wave, nb = blockIdx.y, zwords = p.words / 32;
    if (p.row0 + nb * 32 >= p.head->count) {
        return;  // gW does not read what lies behind the rows' last 32
    }
    __shared__ int exs[W ? kVlB / kWave : 1][32];
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
#pragma unroll
        for (int s = 0; s < 2; s++) {
            float x[8];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const i4v ew = *(const i4v *)(p.ew + vb * 32 + 8 * (2 * s + t) + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; e++) x[4 * t + e] = __builtin_amdgcn_ldexpf(g[8 * s + 4 * t + e], ew[e] - row.e);
            }
            store_block((char *)z + s * 2048, lane, cut<0>(x, 1.0f));
        }
    }
    if constexpr (W) {
#pragma unroll
        for (int r = 0; r < 16; r++) turn[wave][8 * (r / 4) + 4 * half + r % 4][col] = g[r];
        if (half == 0) exs[wave][col] = row.ex;
        // the wave's own part of LDS: it reads what it wrote
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int ev = word_exponent(p.term[vb * 32 + col]);
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int k = 16 * s + 4 * half + (e & 3) + 8 * (e >> 2);
                const float v = turn[wave][col][k];
                sum += v;
                x[e] = __builtin_amdgcn_ldexpf(v, exs[wave][k] - ev);
            }
            store_block(p.turned + vb * p.turned_step + (nb * 2 + s) * 2048, lane, cut<0>(x, 1.0f));
        }
        if (p.column) {
            sum += __shfl_xor(sum, 32);
            if (half == 0) p.column[nb * p.words + vb * 32 + col] = sum;
        }
    }
}

// What is left of a piece, in one launch: gx (+)= its parts' sum, at the rows' places; gW (+)= its parts' sum; gb (+)= the sums of the
// columns of G, which k_vl_grad left for every 32 rows; and at the last the loss, which of no rows is NaN, as a mean over nothing is
// (a sum: 0).
struct TailArgs {
    unsigned gx, gw, gb;  // workgroups
    VlHead *head;
    const float *gout;
    int sum;
    int64_t row0, rows, V, D, words, cols;
    const int32_t *from;  // of this piece's rows
    const VlRow *row;
    const int *term;
    const float *parts_x, *parts_w, *column;
    float *out_x, *out_w, *out_b;
    int acc_x, acc_w, acc_b;
    const double *losses;
    float *loss;
};

__global__ __launch_bounds__(kVlB) void k_vl_ends(TailArgs p) {
    __shared__ double sh[kVlB / kWave];
    const int64_t count = p.head->count, left = min(p.rows, count - p.row0);
    const VlCoef c = count ? vl_coef(p.head, p.gout, p.sum) : VlCoef{0.0f, 0};
    unsigned b = blockIdx.x;
    if (b < p.gx) {
        const int slices = p.head->slices_x;
        for (int64_t n = b; n < left; n += p.gx) {
            const int en = p.row[n].e + c.e;
            float *out = p.out_x + (int64_t)p.from[n] * p.D;
            for (int64_t d = threadIdx.x; d < p.D; d += kVlB) {
                double s = 0.0;
#pragma unroll 8
                for (int i = 0; i < slices; i++) s += (double)p.parts_x[((int64_t)i * p.rows + n) * p.cols + d];
                const float v = __builtin_amdgcn_ldexpf((float)s, en);
                out[d] = p.acc_x ? fma_(v, c.m, out[d]) : v * c.m;
            }
        }
    } else if ((b -= p.gx) < p.gw) {
        const int slices = p.head->slices_w;
        for (int64_t v = b; v < p.V; v += p.gw) {
            const int ev = word_exponent(p.term[v]) + c.e;
            for (int64_t d = threadIdx.x; d < p.D; d += kVlB) {
                double s = 0.0;
#pragma unroll 8
                for (int i = 0; i < slices; i++) s += (double)p.parts_w[((int64_t)i * p.words + v) * p.cols + d];
                const float x = __builtin_amdgcn_ldexpf((float)s, ev);
                float *o = p.out_w + v * p.D + d;
                *o = p.acc_w ? fma_(x, c.m, *o) : x * c.m;
            }
        }
    } else if ((b -= p.gw) < p.gb) {
        const int64_t v = (int64_t)b * kVlB + threadIdx.x, blocks = left > 0 ? (left + 31) / 32 : 0;
        if (v >= p.V) return;
        double s = 0.0;
#pragma unroll 8
        for (int64_t i = 0; i < blocks; i++) s += (double)p.column[i * p.words + v];
        const float x = __builtin_amdgcn_ldexpf((float)s, c.e);
        p.out_b[v] = p.acc_b ? fma_(x, c.m, p.out_b[v]) : x * c.m;
    } else {
        const double t = vl_wg_sum(vl_lane_sum(p.losses, count), sh);
        if (threadIdx.x == 0) *p.loss = p.sum ? (float)t : count ? (float)(t / (double)count) : __builtin_nanf("");
    }
}

// ---- one call -----------------------------------------------------------------------------------------------------------------
struct SplitPlan {
    int64_t n, d, v;   // rows, columns and words, padded to tiles
    int64_t dk;        // columns, padded to two blocks of k
    int64_t piece;     // rows of a piece, padded
    int slices, slices_w;  // parts of gx and of gW, at most; 0: gW is not cut
    int columns;       // slices of the rows where the words' largest are looked for
    size_t from, list, losses, row, label_z, part, ew, ex, term, column, x, w, z, turned, parts_x, parts_w, total;
};

static int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

static SplitPlan split_plan(int64_t N, int64_t D, int64_t V, bool want_x, bool want_w, bool want_b) {
    SplitPlan p{};
    const bool grad = want_x || want_w || want_b;
    p.n = up_to(N, kTileM), p.d = up_to(D, kTileMost), p.v = up_to(V, kTileM), p.dk = up_to(D, 32);
    int64_t most = grad ? kZBytes / (8 * p.v) : kPartBytes / (p.v / kStatWords * (int64_t)sizeof(VlPart));
    if (want_x) most = std::min(most, kPartBytes / (p.d * 4));
    p.piece = std::max<int64_t>(kTileM, std::min(std::min(p.n, up_to(vl_piece_rows(kPieceRows), kTileM)), most / kTileM * kTileM));
    p.slices = (int)std::max<int64_t>(1, std::min<int64_t>(64, kPartBytes / (p.piece * p.d * 4)));
    // gW: where its tiles would leave the chip's CUs idle
    if (p.v / kTileM * ((D + 127) / 128) < kPlanCUs) p.slices_w = (int)std::max<int64_t>(1, std::min<int64_t>(64, kPartBytes / (p.v * p.d * 4)));
    p.columns = (int)std::max<int64_t>(1, std::min<int64_t>(16, std::min(p.piece / 32, (4096 + p.v / 32 - 1) / (p.v / 32))));
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
    p.part = take(true, p.v / kStatWords * p.piece * (int64_t)sizeof(VlPart));
    p.ew = take(true, p.v * 4);
    p.ex = take(true, p.n * 4);
    p.term = take(want_w || want_b, p.v * 4);
    p.column = take(want_b, p.piece / 32 * p.v * 4);
    p.x = take(true, p.n * p.dk * 4);
    p.w = take(true, p.v * p.dk * 4);
    p.z = take(grad, p.piece * p.v * 4);
    p.turned = take(want_w || want_b, p.piece * p.v * 4);
    p.parts_x = take(want_x, p.slices * p.piece * p.d * 4);
    p.parts_w = take(want_w && p.slices_w, p.slices_w * p.v * p.d * 4);
    p.total = at;
    return p;
}

// The two forms' times by what they do, in us.  fp32 products start at once and run at 115 TFLOP/s; pieces have x and W read and written
// first, whole tiles of rows, and some 370 TFLOP/s.  Both sides measured (us, fp32 products : pieces): 128000 x 2048 with gradients, 64
// rows 1172 : 1418, 256 3632 : 1865; 32000 x 1024, 64 rows 172 : 265, 128 300 : 288, 4096 7284 : 2542; 2000 x 256, 1024 rows 73 : 96, 4096
// 192 : 136; scored, 32000 x 1024, 64 rows 55 : 102, 128 88 : 106, 256 165 : 115; 5000 x 64, 512 rows 23 : 28, 1024 34 : 29.  Over the 400
// sizes that the numbers are fitted to (1 to 4096 rows, 64 to 2048 columns, 500 to 128000 words) what it chooses takes 0.1% longer in the
// mean than the better one, 11% at most.
bool vl_split_pays(int64_t N, int64_t D, int64_t V, bool grads) {
    if (N == 0 || N > kPieceRows * 16) return false;
    if (const char *form = getenv("NC_HIP_VOCAB_FORM")) return form[0] == 's';
    const double d = (double)D, vd = (double)V * d, nv = (double)N * (double)V, nvd = nv * d;
    const double fp32 = grads ? 30 + 2e-6 * vd + 4.5e-6 * nv + 5.2e-8 * nvd : 17 + 0.75e-6 * vd + 1.4e-6 * nv + 1.6e-8 * nvd;
    const double split = grads ? 52 + 0.043 * d + 0.8e-3 * (double)V + 4e-6 * vd + 4e-6 * nv + 1e-8 * nvd
                               : 20 + 0.036 * d + 2.1e-6 * vd + 0.4e-6 * nv + 3.5e-9 * nvd;
    return split < fp32;
}

size_t vl_split_workspace(int64_t N, int64_t D, int64_t V, bool want_x, bool want_w, bool want_b) {
    return split_plan(N, D, V, want_x, want_w, want_b).total;
}

// Whether a product runs on tiles of 256 columns, one a CU, rather than of 128, two a CU: by the rounds that they take, where a last round
// of 128s that finds a CU each takes half.  At the same number those are 4% slower (gW of 128000 x 4096 x 2048: 5.5 ms, 6.3 with tiles of
// 128; 50021 x 700 x 770, 4 rounds for 3: 257 us, 239).  A sum that is cut fills the rounds by itself: where more than 128 columns are there.
static bool wide_tiles(int64_t tiles_m, int64_t cols, bool cut) {
    if (cut) return cols > 128;
    const int64_t wide = tiles_m * ((cols + 255) / 256), narrow = tiles_m * ((cols + 127) / 128), last = narrow % (2 * kPlanCUs);
    const int64_t halves = narrow / (2 * kPlanCUs) * 2 + (last > kPlanCUs ? 2 : last > 0 ? 1 : 0);
    return 25 * 2 * ((wide + kPlanCUs - 1) / kPlanCUs) <= 26 * halves;
}

int vl_split_run(const VlCall &c, const char *what) {
    const SplitPlan pl = split_plan(c.N, c.D, c.V, c.gx, c.gw, c.gb);
    const bool grad = c.gx || c.gw || c.gb;
    auto at = [&](size_t off) { return c.ws + off; };
    VlHead *head = (VlHead *)c.ws;
    int32_t *from = (int32_t *)at(pl.from), *list = (int32_t *)at(pl.list);
    double *losses = (double *)at(pl.losses);
    float *const gx_off = c.acc_x ? nullptr : c.gx;
    const int64_t terms = c.gw || c.gb ? pl.v : 0;
    const int64_t helpers = std::min<int64_t>(1024, (std::max(terms / 4, c.row_loss || gx_off ? c.N : 0) + 255) / 256);
    hipLaunchKernelGGL(k_vl_begin, (unsigned)(1 + helpers), 1024, 0, c.st, c.labels, c.N, pl.n, c.D, c.V, c.ignore, head, from, list, c.bad,
                       (int *)at(pl.term), terms, c.row_loss, gx_off);
    PackPair pp{};
    pp.a[0] = {c.x, c.ldx, c.N, c.D, from, head, (int *)at(pl.ex), at(pl.x), (int)(pl.n / 32)};
    pp.a[1] = {c.w, c.ldw, c.V, c.D, nullptr, head, (int *)at(pl.ew), at(pl.w), (int)(pl.v / 32)};
    pp.kblocks = (int)(pl.dk / 16);
    const unsigned packing = (unsigned)(pp.a[0].groups + pp.a[1].groups);
    if (pp.kblocks <= 32) hipLaunchKernelGGL(k_vl_pack<4>, packing, 512, 0, c.st, pp);
    else if (pp.kblocks <= 64) hipLaunchKernelGGL(k_vl_pack<8>, packing, 512, 0, c.st, pp);
    else if (pp.kblocks <= 128) hipLaunchKernelGGL(k_vl_pack<16>, packing, 512, 0, c.st, pp);
    else hipLaunchKernelGGL(k_vl_pack<0>, packing, 512, 0, c.st, pp);

    auto launch = [&](auto kernel, int lanes, int lds, int64_t groups, const MmArgs &m) {
        (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        hipLaunchKernelGGL(kernel, (unsigned)groups, lanes, lds, c.st, m);
    };
    auto product = [&](auto what, MmArgs m, int64_t cols, int slices) {
        constexpr int W = decltype(what)::value;
        const bool wide = wide_tiles(m.tiles_m, cols, W == MM_GX || W == MM_GW_PARTS);
        m.tiles_n = (int)((cols + (wide ? 255 : 127)) / (wide ? 256 : 128));
        const int64_t groups = (int64_t)m.tiles_m * m.tiles_n * slices;
        if (wide) launch(k_vl_product<W, 4>, Tile<4>::kLanes, Tile<4>::kLds, groups, m);
        else launch(k_vl_product<W, 2>, Tile<2>::kLanes, Tile<2>::kLds, groups, m);
    };
    for (int64_t r0 = 0; r0 < pl.n; r0 += pl.piece) {
        const int64_t rows = std::min(pl.piece, pl.n - r0);
        MmArgs m{};
        m.A = at(pl.w), m.step_a = pl.dk * 128, m.B = at(pl.x) + r0 / 32 * (pl.dk * 128), m.step_b = pl.dk * 128;
        m.tiles_m = (int)(pl.v / kTileM), m.kblocks = (int)(pl.dk / 16);
        m.head = head, m.row0 = r0, m.V = c.V, m.D = c.D;
        m.ew = (const int *)at(pl.ew), m.ex = (const int *)at(pl.ex) + r0, m.bias = c.bias, m.labels = list + r0;
        m.z = grad ? (float *)at(pl.z) : nullptr, m.zwords = pl.v / 32, m.part = (VlPart *)at(pl.part), m.label_z = (float *)at(pl.label_z);
        m.rows = pl.piece, m.blocks = (int)(pl.dk / 16);
        if (grad) product(std::integral_constant<int, MM_Z>{}, m, rows, 1);
        else product(std::integral_constant<int, MM_SCORE>{}, m, rows, 1);

        GradArgs g{};
        g.head = head, g.row0 = r0, g.rows = pl.piece, g.V = c.V, g.words = pl.v, g.part = m.part, g.label_z = m.label_z;
        g.labels = list + r0, g.from = from + r0, g.row = (VlRow *)at(pl.row), g.losses = losses, g.row_loss = c.row_loss;
        g.z = m.z, g.turned = at(pl.turned), g.turned_step = pl.piece * 128, g.term = c.gw || c.gb ? (int *)at(pl.term) : nullptr, g.column = c.gb ? (float *)at(pl.column) : nullptr;
        g.slices = pl.columns;
        const bool wide = wide_tiles(0, c.D, true);
        g.of_x = {(int)((c.D + (wide ? 255 : 127)) / (wide ? 256 : 128)), pl.slices, wide ? kPlanCUs : 2 * kPlanCUs};
        g.of_w = {g.of_x.tiles_n, pl.slices_w, g.of_x.at_once};
        g.ex = m.ex, g.ew = m.ew;
        hipLaunchKernelGGL(k_vl_stats, (unsigned)(rows / 32), 1024, 0, c.st, g);
        const bool turn = c.gw || c.gb;
        if (turn) {
            const dim3 gw((unsigned)(pl.v / 32 / (kVlB / kWave)), (unsigned)pl.columns);
            hipLaunchKernelGGL(k_vl_words, gw, kVlB, 0, c.st, g);
        }
        const dim3 gg((unsigned)(pl.v / 32 / (kVlB / kWave)), (unsigned)(rows / 32));
        if (c.gx && turn) hipLaunchKernelGGL((k_vl_grad<true, true>), gg, kVlB, 0, c.st, g);
        else if (c.gx) hipLaunchKernelGGL((k_vl_grad<true, false>), gg, kVlB, 0, c.st, g);
        else if (turn) hipLaunchKernelGGL((k_vl_grad<false, true>), gg, kVlB, 0, c.st, g);
        TailArgs t{};
        t.head = head, t.gout = c.gout, t.sum = c.sum, t.row0 = r0, t.rows = pl.piece, t.V = c.V, t.D = c.D, t.words = pl.v, t.cols = pl.d;
        t.from = g.from, t.row = g.row, t.term = g.term, t.column = g.column, t.losses = losses, t.loss = c.loss;
        t.parts_x = (float *)at(pl.parts_x), t.parts_w = (float *)at(pl.parts_w), t.out_x = c.gx, t.out_w = c.gw, t.out_b = c.gb;
        t.acc_x = c.acc_x, t.acc_w = c.acc_w || r0, t.acc_b = c.acc_b || r0;
        t.gb = c.gb ? (unsigned)((c.V + kVlB - 1) / kVlB) : 0;
        if (c.gx) {
            MmArgs a = m;
            a.A = (const char *)m.z, a.step_a = pl.v * 128, a.B = at(pl.w), a.step_b = pl.dk * 128;
            a.tiles_m = (int)(rows / kTileM), a.kblocks = (int)(pl.v / 16);
            a.parts = (float *)at(pl.parts_x), a.part_rows = pl.piece, a.cols = pl.d;
            product(std::integral_constant<int, MM_GX>{}, a, c.D, pl.slices);
            t.gx = (unsigned)std::min<int64_t>(rows, 1 << 14);
        }
        if (c.gw) {
            MmArgs a = m;
            a.A = g.turned, a.step_a = g.turned_step;
            a.tiles_m = (int)(pl.v / kTileM), a.kblocks = (int)(rows / 16);
            a.eg = g.term, a.gout = c.gout, a.out = c.gw, a.sum = c.sum, a.acc = c.acc_w || r0;
            if (pl.slices_w) {
                a.parts = (float *)at(pl.parts_w), a.part_rows = pl.v, a.cols = pl.d;
                product(std::integral_constant<int, MM_GW_PARTS>{}, a, c.D, pl.slices_w);
                t.gw = (unsigned)std::min<int64_t>(c.V, 1 << 14);
            } else {
                product(std::integral_constant<int, MM_GW>{}, a, c.D, 1);
            }
        }
        const unsigned last = r0 + pl.piece >= pl.n;
        const unsigned groups = t.gx + t.gw + t.gb + last;
        if (groups) hipLaunchKernelGGL(k_vl_ends, groups, kVlB, 0, c.st, t);
    }
    return check_launch(what);
}

}  // namespace nchip
