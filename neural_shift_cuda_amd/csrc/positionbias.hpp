// positionbias.hpp -- limits of the bucketed position bias, and the last step
// of its gradient, which the attention's bias shares.
#pragma once

#include "nsh_common.hpp"

namespace nsh {

constexpr int kMaxReach = 2048;      // relative positions -2048 .. 2048: 16 KiB of LDS
constexpr int kTableThreads = 1024;  // of the gradient's last step

// The starts of the runs that one of `blocks` workgroups takes, in turns.  In 64
// bits: a turn of 2^21 workgroups of 2048 places is 2^32 long, and in 32 its next
// start would be the first again.
struct Turns {
    uint64_t at, step;
    static __host__ __device__ __forceinline__ Turns of(uint32_t block, uint32_t blocks, uint32_t run) {
        return Turns{static_cast<uint64_t>(block) * run, static_cast<uint64_t>(blocks) * run};
    }
};

// grad_table (num_buckets, H) from sums per relative position,
// partial[(h * chunks + c) * (2 R + 1) + rel + R], added over c in order.
int table_gradient(const float* partial, const int32_t* buckets, int64_t H, int64_t chunks,
                   int64_t num_buckets, int64_t R, int dtype, void* grad_table, hipStream_t stream);

}  // namespace nsh
