// attention_rows.hpp -- query rows as the attention kernels cut them up: the
// lane's row, what the rows of a wave have in common, and which keys they see.
#pragma once

#include "attention_tiles.hpp"

namespace nsh {

// Rows of a wave: where lane row l % 32 of a row block stands.
struct LaneRow {
    int i, h;
    bool live;
    Row r;
};

__device__ __forceinline__ LaneRow lane_row(const Att& a, int b, int group, int row, int n) {
    const int R = a.Lq * a.pack;
    LaneRow x;
    x.live = row < R;
    row = min(row, R - 1);
    x.i = a.pack == 1 ? row : row / a.pack;
    x.h = group * a.pack + (a.pack == 1 ? 0 : row - x.i * a.pack);
    x.r = row_of(a, b, x.i, n);
    return x;
}

// The end of the keys that rows up to `row` of a batch see by order.
__device__ __forceinline__ int keys_end(const Att& a, int b, int last_row, int n) {
    if (!a.causal) return n;
    const int i = min(last_row, a.Lq * a.pack - 1) / a.pack;
    return min(n, max(i + n - a.Lq + 1, a.prefix ? a.prefix[b] : 0));
}

// Lowest and highest document of rows [r0, r0 + count) of the group.
__device__ __forceinline__ int2 row_documents(const Att& a, int b, int r0, int count, int n) {
    int lo = 0x7fffffff, hi = -1;
    for (int r = r0 + (threadIdx.x & 63); r < r0 + count; r += 64) {
        const int i = min(r, a.Lq * a.pack - 1) / a.pack, p = i + n - a.Lq;
        const int d = p >= 0 && p < n ? a.documents[static_cast<int64_t>(b) * a.Lk + p] : -1;
        if (d >= 0) lo = min(lo, d), hi = max(hi, d);
    }
    return make_int2(wave_min(lo), wave_max(hi));
}

// What a wave's rows have in common.
struct WaveRows {
    int least, most;      // of the rows' key ends
    int first, last;      // of their positions
};

__device__ __forceinline__ WaveRows wave_rows(const LaneRow& x) {
    WaveRows w;
    w.least = __builtin_amdgcn_readfirstlane(wave_min(x.r.lim));
    w.most = __builtin_amdgcn_readfirstlane(wave_max(x.r.lim));
    w.first = __builtin_amdgcn_readfirstlane(wave_min(x.r.p));
    w.last = __builtin_amdgcn_readfirstlane(wave_max(x.r.p));
    return w;
}

__device__ __forceinline__ Bias lane_bias(const Att& a, int h, const float* line) {
    return Bias{a.slopes ? a.slopes[h] * kLog2e : 0.f, line};
}

// Not seen -> -inf, for 32 keys from j0 (kd: their documents, in LDS).
__device__ __forceinline__ f32x16 mask_keys(const Att& a, const Row& x, int j0, const int* kd, int l,
                                            f32x16 s) {
    const int left = here(x.lim - j0 - 4 * (l >> 5));
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = el(r) < left ? s[r] : -INFINITY;
    if (a.documents) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const i32x4 d = *reinterpret_cast<const i32x4*>(kd + 8 * c + 4 * (l >> 5));
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * c + e] = d[e] == x.doc ? s[4 * c + e] : -INFINITY;
        }
    }
    return s;
}

}  // namespace nsh
