// Shared pieces of the vocabulary loss: vocab_loss.hip (entry points, the form on fp32 products) and vocab_split.hip (the form whose
// products run on the fp16 matrix cores).
#pragma once

#include "common.hpp"

#include <algorithm>

namespace nchip {

constexpr int kVlB = 256;

// the head of the workspace
struct VlHead {
    int64_t count;  // rows that count
    int slices_x, slices_w;  // parts of gx and gW
};

// one call's arguments
struct VlCall {
    int64_t N, D, V;
    const float *x;
    int64_t ldx;
    const float *w;
    int64_t ldw;
    const float *bias;
    const int32_t *labels;
    int32_t ignore;
    int sum;
    const float *gout;
    float *loss, *row_loss;
    unsigned long long *bad;
    float *gx, *gw, *gb;
    int acc_x, acc_w, acc_b;
    char *ws;
    hipStream_t st;
};

__device__ __forceinline__ bool vl_counts(int32_t label, int32_t ignore, int64_t V) { return label != ignore && label >= 0 && label < V; }

__device__ __forceinline__ double vl_wg_sum(double v, double *sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < (int)blockDim.x / kWave; i++) t += sh[i];
    return t;
}

// a lane's share of v[0 .. n) for workgroups of kVlB, eight asked for at a time, the last ones' too (4000 rows: 1.5 us less than by a
// loop that the compiler unrolls, whose remainder waits for each)
__device__ __forceinline__ double vl_lane_sum(const double *v, int64_t n) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 8 * kVlB) {
        double x[8];
#pragma unroll
        for (int u = 0; u < 8; u++) x[u] = v[min(i + u * kVlB, n - 1)];
#pragma unroll
        for (int u = 0; u < 8; u++) s += i + u * kVlB < n ? x[u] : 0.0;
    }
    return s;
}

inline size_t vl_round256(size_t n) { return (n + 255) / 256 * 256; }

// rows of a piece at most: `most`, or what the test hook NC_HIP_VOCAB_ROWS says
inline int64_t vl_piece_rows(int64_t most) {
    if (const char *e = getenv("NC_HIP_VOCAB_ROWS")) {
        const long long v = atoll(e);
        if (v > 0 && v < most) return v;
    }
    return most;
}

// gx and gW of few rows (vocab_few.hip); D a multiple of 4, gw and z's rows 16-byte aligned
struct VlFew {
    int64_t N, D, V;
    const float *w;
    int64_t ldw;
    const float *z;  // G [N][ldz]
    int64_t ldz;
    const float *clean;  // [N][D]
    float *parts;   // [slices][N][D]
    int64_t slice;  // words of a part of gx
    float *gw;
    int acc_w;
};
int64_t vl_few_slice(int64_t D, int64_t V);
void vl_few_gx(const VlFew &p, hipStream_t st);
void vl_few_gw(const VlFew &p, hipStream_t st);

// whether the products of a call are worth cutting into pieces, the workspace that takes, and the call itself
bool vl_split_pays(int64_t N, int64_t D, int64_t V, bool grads);
size_t vl_split_workspace(int64_t N, int64_t D, int64_t V, bool want_x, bool want_w, bool want_b);
int vl_split_run(const VlCall &c, const char *what);

}  // namespace nchip
