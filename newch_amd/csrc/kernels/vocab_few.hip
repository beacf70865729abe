// Vocabulary loss: the gradients of few rows with a large table, which are bound by reading W for gx and writing gW.  Waves take their
// operands from memory straight into registers and multiply on the fp32 matrix cores (32 x 32 x 2).  A lane has four consecutive columns,
// one in each of four tiles, so that loads and stores of W, x and gW are of 16 bytes; and four consecutive words of G, used in four
// steps, each of which adds one word from the lower half of the wave and one from the upper.
//
// 32 rows: 64 cycles of a SIMD for 256 bytes of W, 9.8 TB/s over the chip.  Measured over 73424 words of 2048 columns, 23 rows: gx 110 to
// 144 us (5.5 to 4.2 TB/s), gW 133 to 169; the products of the other sizes take 170 and 284 for them.
#include "vocab_loss.hpp"

namespace nchip {

typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kFewWaves = kVlB / kWave;

// where a lane's results of a 32 x 32 tile lie: column lane & 31, row
__device__ __forceinline__ int few_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

// parts of gx = G W: a workgroup has a slice of the words and 128 columns; its waves share the words, 16 at a time
__global__ __launch_bounds__(kVlB) void k_vl_few_gx(VlFew p) {
    constexpr int U = 2;
    __shared__ float sh[2][64][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, half = lane >> 5, col = lane & 31;
    const int64_t c = (int64_t)blockIdx.x * 128 + 4 * col, v0 = (int64_t)blockIdx.y * p.slice, v1 = min(p.V, v0 + p.slice);
    const float *g = p.z + min((int64_t)col, p.N - 1) * p.ldz, *w = p.w + min(c, p.D - 4);
    f16v acc[4] = {};
    f4 a[2][U], b[2][U][4];
    auto load = [&](int i, int64_t k0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t k = k0 + 8 * u + 4 * half;
#pragma unroll
            for (int e = 0; e < 4; e++) b[i][u][e] = *(const f4u *)(w + min(k + e, v1 - 1) * p.ldw);
            a[i][u] = *(const f4 *)(g + min(k, p.ldz - 4));
        }
    };
    auto add = [&](int i, int64_t k0) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = k0 + 8 * u + 4 * half + e < v1 ? a[i][u][e] : 0.0f;
#pragma unroll
                for (int q = 0; q < 4; q++) acc[q] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, b[i][u][e][q], acc[q], 0, 0, 0);
            }
    };
    constexpr int64_t step = 8 * U * kFewWaves;
    int64_t k0 = v0 + 8 * U * wave;
    load(0, k0);
    for (; k0 < v1; k0 += 2 * step) {
        load(1, k0 + step);
        __builtin_amdgcn_sched_barrier(0);
        add(0, k0);
        load(0, k0 + 2 * step);
        __builtin_amdgcn_sched_barrier(0);
        add(1, k0 + step);
    }
    // the waves' sums: 2 and 3 to 0 and 1, then 1 to 0
#pragma unroll
    for (int from = 2; from > 0; from /= 2) {
        if (wave >= from && wave < 2 * from)
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int r = 0; r < 16; r++) sh[wave - from][q * 16 + r][lane] = acc[q][r];
        __syncthreads();
        if (wave < from)
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int r = 0; r < 16; r++) acc[q][r] += sh[wave][q * 16 + r][lane];
        __syncthreads();
    }
    if (wave > 0 || c >= p.D) return;
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int64_t n = few_row(r, half);
        if (n < p.N) *(f4 *)(p.parts + ((int64_t)blockIdx.y * p.N + n) * p.D + c) = f4{acc[0][r], acc[1][r], acc[2][r], acc[3][r]};
    }
}

// gW (+)= G^T x, x without the rows that do not count: a wave has 32 words and 128 columns
__global__ __launch_bounds__(kVlB) void k_vl_few_gw(VlFew p) {
    constexpr int U = 4;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, half = lane >> 5, col = lane & 31;
    const unsigned blocks = (unsigned)((p.D + 127) / 128);
    const int64_t c = (int64_t)(blockIdx.x % blocks) * 128 + 4 * col, v0 = ((int64_t)(blockIdx.x / blocks) * kFewWaves + wave) * 32;
    if (v0 >= p.V) return;
    const float *x = p.clean + min(c, p.D - 4), *g = p.z + min(v0 + col, p.V - 1);
    const int last = (int)p.N - 1;
    f16v acc[4] = {};
    f4 b[2][U];
    float a[2][U];
    auto load = [&](int i, int n0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int n = min(n0 + 2 * u + half, last);
            b[i][u] = *(const f4 *)(x + n * p.D);
            a[i][u] = g[n * p.ldz];
        }
    };
    auto add = [&](int i, int n0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool on = n0 + 2 * u + half <= last;
            const float s = on ? a[i][u] : 0.0f;
            const f4 y = on ? b[i][u] : f4{};
#pragma unroll
            for (int q = 0; q < 4; q++) acc[q] = __builtin_amdgcn_mfma_f32_32x32x2f32(s, y[q], acc[q], 0, 0, 0);
        }
    };
    load(0, 0);
    for (int n0 = 0; n0 <= last; n0 += 4 * U) {
        load(1, n0 + 2 * U);
        __builtin_amdgcn_sched_barrier(0);
        add(0, n0);
        load(0, n0 + 4 * U);
        __builtin_amdgcn_sched_barrier(0);
        add(1, n0 + 2 * U);
    }
    if (c >= p.D) return;
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int64_t v = v0 + few_row(r, half);
        if (v >= p.V) continue;
        float *out = p.gw + v * p.D + c;
        f4 s = {acc[0][r], acc[1][r], acc[2][r], acc[3][r]};
        if (p.acc_w) s = s + *(const f4 *)out;
        __builtin_nontemporal_store(s, (f4 *)out);
    }
}

// words of a part of gx: four workgroups a CU, of at least 256 words
int64_t vl_few_slice(int64_t D, int64_t V) {
    const int64_t blocks = (D + 127) / 128, want = (4 * kPlanCUs + blocks - 1) / blocks;
    return std::max<int64_t>(256, ((V + want - 1) / want + 63) / 64 * 64);
}

void vl_few_gx(const VlFew &p, hipStream_t st) {
    const dim3 grid((unsigned)((p.D + 127) / 128), (unsigned)((p.V + p.slice - 1) / p.slice));
    hipLaunchKernelGGL(k_vl_few_gx, grid, kVlB, 0, st, p);
}

void vl_few_gw(const VlFew &p, hipStream_t st) {
    const int64_t groups = (p.D + 127) / 128 * ((p.V + 32 * kFewWaves - 1) / (32 * kFewWaves));
    hipLaunchKernelGGL(k_vl_few_gw, (unsigned)groups, kVlB, 0, st, p);
}

}  // namespace nchip
