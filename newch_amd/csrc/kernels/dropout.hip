// Dropout whose mask is never stored: value i of a call stays where word i % 4 of a counter-based generator's block i / 4 is at least
// p 2^32, so the backward (or a replay) makes the same mask again from the call's seed and offset.  No counterpart in the reference,
// whose dropout draws the mask from the context's sequential generator and keeps it.
//
// The generator is Philox 4x32 with 10 rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// key = the seed's 64 bits, counter = (i / 4, offset), 64 bits each.  A round is two products of 32 x 32 -> 64 bits and four xors;
// twenty products for four values.
//
// A stream of 8 bytes a value (12 with a residual or where a gradient is added to): one lane makes the four words of one
// block and moves the four values they belong to, one 16-byte access each, at any 4-byte alignment.
#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace nchip {

constexpr int kDropB = 256;
constexpr int64_t kDropBlocks = int64_t(1) << 30;  // generator blocks (lanes) of a launch at most

struct DropArgs {
    int64_t n, base;  // values; the first generator block of this launch
    uint64_t seed, offset;
    const uint64_t *offset_dev;  // added to the offset where set
    uint32_t last;               // the largest word that drops its value
    bool any;                    // whether one does
    float scale;
    const float *x, *r;
    float *y;
};

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t block, uint64_t offset, uint64_t seed) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// y = keep x scale (+ r): a value that is dropped counts as 0, be it infinite or NaN.  r is the residual of the forward or the old
// gradient of a backward that adds.
template <bool ADD>
__global__ __launch_bounds__(kDropB) void k_dropout(DropArgs p) {
    const int64_t b = p.base + (int64_t)blockIdx.x * kDropB + threadIdx.x;
    const int64_t i = 4 * b;
    if (i >= p.n) return;
    const bool whole = i + 4 <= p.n;
    f4 x = {}, r = {};
    if (whole) {
        x = __builtin_nontemporal_load((const f4u *)(p.x + i));
        if (ADD) r = __builtin_nontemporal_load((const f4u *)(p.r + i));
    } else {
        for (int e = 0; e < (int)(p.n - i); e++) {
            x[e] = p.x[i + e];
            if (ADD) r[e] = p.r[i + e];
        }
    }
    const Words w = philox((uint64_t)b, p.offset + (p.offset_dev ? *p.offset_dev : 0), p.seed);
    f4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const bool dropped = p.any && w.w[e] <= p.last;
        y[e] = ADD ? (dropped ? r[e] : fma_(x[e], p.scale, r[e])) : (dropped ? 0.0f : x[e] * p.scale);
    }
    if (whole) {
        __builtin_nontemporal_store((f4u)y, (f4u *)(p.y + i));
    } else {
        for (int e = 0; e < (int)(p.n - i); e++) p.y[i + e] = y[e];
    }
}

static int dropout(const char *what, int64_t n, double prob, uint64_t seed, uint64_t offset, const uint64_t *offset_dev, const float *x,
                   const float *r, float *y, void *stream) {
    if (n < 0 || n > int64_t(1) << 60) return set_error(NC_HIP_ERR_ARG, "%s: bad size %lld", what, (long long)n);
    if (!(prob >= 0.0 && prob <= 1.0)) return set_error(NC_HIP_ERR_ARG, "%s: p must be in [0, 1], got %g", what, prob);
    if (((uintptr_t)offset_dev & 7u) != 0) return set_error(NC_HIP_ERR_ARG, "%s: the offset is not 8-byte aligned", what);
    if (n == 0) return NC_HIP_OK;
    if (!x || !y) return set_error(NC_HIP_ERR_ARG, "%s: NULL pointer", what);
    const uint64_t below = (uint64_t)std::llrint(prob * 4294967296.0);  // words that drop a value, 0 .. 2^32
    DropArgs p{};
    p.n = n, p.seed = seed, p.offset = offset, p.offset_dev = offset_dev;
    p.any = below > 0, p.last = (uint32_t)(below - 1);
    p.scale = prob < 1.0 ? (float)(1.0 / (1.0 - prob)) : 0.0f;
    p.x = x, p.r = r, p.y = y;
    const int64_t blocks = (n - 1) / 4 + 1;
    for (; p.base < blocks; p.base += kDropBlocks) {
        const unsigned grid = (unsigned)((std::min(blocks - p.base, kDropBlocks) + kDropB - 1) / kDropB);
        if (r) hipLaunchKernelGGL(k_dropout<true>, grid, kDropB, 0, as_stream(stream), p);
        else hipLaunchKernelGGL(k_dropout<false>, grid, kDropB, 0, as_stream(stream), p);
    }
    return check_launch(what);
}

}  // namespace nchip

using namespace nchip;

extern "C" NC_HIP_API int nc_hip_dropout_fwd(int64_t n, double p, uint64_t seed, uint64_t offset, const uint64_t *offset_dev,
                                             const float *x, const float *residual, float *y, void *stream) {
    return dropout("nc_hip_dropout_fwd", n, p, seed, offset, offset_dev, x, residual, y, stream);
}

extern "C" NC_HIP_API int nc_hip_dropout_bwd(int64_t n, double p, uint64_t seed, uint64_t offset, const uint64_t *offset_dev,
                                             const float *gy, float *gx, int accumulate, void *stream) {
    return dropout("nc_hip_dropout_bwd", n, p, seed, offset, offset_dev, gy, accumulate ? gx : nullptr, gx, stream);
}
