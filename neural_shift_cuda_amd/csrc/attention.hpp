// attention.hpp -- what the attention kernels share: their arguments as the
// device takes them, a query's position and a pair's visibility, and the
// score's cap and biases.
#pragma once

#include "nsh_common.hpp"

namespace nsh {

// The C arguments, narrowed and with the constants the kernels use.
struct Att {
    const void *q, *k, *v;
    int B, Hq, Hk, Lq, Lk, D, per;  // per = Hq / Hk query heads share a key head
    int64_t qs[3], ks[3], vs[3], os[3];
    const int32_t *lengths, *prefix, *documents, *buckets;
    const float* slopes;
    const void* table;
    int num_buckets, reach;
    float scale, cap;
    int causal;
    void* out;
    float* degree;
    const void* go;
    const float* gdegree;
    int64_t gos[3], gqs[3], gks[3], gvs[3];
    void *gq, *gk, *gv, *gtable;
};

__device__ __forceinline__ int filled_keys(const Att& a, int b) {
    if (!a.lengths) return a.Lk;
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n > a.Lk ? a.Lk : n);
}

}  // namespace nsh
