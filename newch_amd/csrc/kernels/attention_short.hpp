// Launches of the kernels for few keys (attention_short.hip).
#pragma once

#include "attention.hpp"

namespace nchip {

struct ShortFwd {
    AttnArgs a;
    const float *q, *k, *v;
    const int *key_len;
    float *o, *lse;
    int64_t rows, qtiles, units;  // rows of a pair, their tiles, pairs times parts
    int tiles, splits;            // tiles of keys, parts the tiles of queries are cut into
};

struct ShortBwd {
    AttnArgs a;
    const float *q, *k, *v;
    const int *key_len;
    const float *o, *lse, *go;
    float *gq, *gk, *gv;  // gk and gv: the parts' [split][...] where there are several
    int64_t rows, qtiles, units, part_k;
    int splits, acc_q, acc_k, acc_v;
};

// keys that the kernels take at most
int short_keys_fwd(int DP);
int short_keys_bwd(int DP);
void short_fwd(const ShortFwd &f, int DP, hipStream_t st);
void short_bwd(const ShortBwd &f, int DP, hipStream_t st);

}  // namespace nchip
