// attention_fwd.hpp -- the forward kernels of the biased attention.
//
// One pass over the keys with a running maximum and sum.  A wave owns 32 query
// rows, one to a lane pair (l, l + 32): the scores of a tile are K q^T, so a
// lane has its row's scores in its own registers, the maximum and sum need one
// exchange of lane halves, and the rounded weights feed V^T p as they lie.
//   SPLIT false: a workgroup owns 128 rows; K and V tiles are shared by its
//     four waves, double buffered, loaded straight to LDS.
//   SPLIT true: the four waves own the same 32 rows and a part of the keys
//     each, with tiles of their own and no barrier; several workgroups may
//     share a row block's keys (`splits`), and a second launch joins them.
//
// What bounds them (times: medians of many launches with inputs in turn): the
// vector work of a score (an exp2, with a cap another and a reciprocal, and 6 to 10
// more instructions) takes more issue than its products (at width 128, capped: 60%
// of the time and 34%), and the two overlap only as far as the two waves of a SIMD
// are out of step.  2 x 16 heads, 4 of keys, 4096 tokens, width 128, causal, capped,
// bf16: 176 us, 780 TFLOP/s of the 1223 that a large library product reaches; 16
// heads, 8 of keys, 8192 tokens, width 96, a quarter of them a prefix: 231 us, 950.
// One token over 16 caches of up to 8192, 32 heads, 8 of keys: 78 + 5 us, 5.2 TB/s,
// near what a copy reaches.  With a learned bias (4 x 12 heads, 1024 tokens, width 64:
// 40 us) or documents (2 x 12 heads, rows of 2500: 38 us) neither is busy: vector 32%
// and 23%, products 11% and 5%, with one wave to a SIMD or less.
#pragma once

#include "attention_rows.hpp"

namespace nsh {

// The weights' running state of a lane's row.
template <int ND>
struct Running {
    f32x16 o[ND];
    float m, z;  // maximum (units of log 2), the lane half's sum
};

// Tiles whose maximum grows the running one by less than 2^8 leave it: the
// weights then reach 2^8 and the sums' rescaling is skipped.  In fp16 the running
// one is kept 7 below, so that weights reach 2^15 and the small ones, which a long
// row may have by the hundred thousand, stay normal numbers down to 2^-21 of the
// largest (140,000 keys 14.5 below one of them: the row is off by 5.5e-2 without, by
// 4e-4 with, its own rounding).
constexpr float kLazy = 8.f;
template <typename T> constexpr float kBelow = kNarrow<T> ? 7.f : 0.f;

template <typename T, int DP, int NB, Kind KIND>
__device__ __forceinline__ void attend(const Att& a, const Cap& cap, const Bias& bs, const Row& x,
                                       const WaveRows& wr, const typename Eight<T>::V (&q)[DP / 16],
                                       const char* K, const char* V, int by_row, int by_col, const int* kd, int j0,
                                       int l, Running<DP / 32>& st) {
    f32x16 s[NB];
    {
        RowFragments<T, DP> f[NB];
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) f[kb].read(K, by_row, kb * 32);
        // a product issues in 4 cycles and takes 32: ahead of the other wave's vector
        // work, which fills the rest (first dozen launches, 2 x 16 heads of 4096, causal,
        // capped: 212 us without, 204 with, 219 the other way round; prompt of 8192:
        // 262, 250, 267)
        priority<1>();
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) s[kb] = f[kb].products(q);
        priority<0>();
    }
    ColumnFragments<T, DP> f;
    const bool whole = j0 + NB * 32 <= wr.least && !(KIND == kGeneral && a.documents);
    if (KIND != kGeneral) {
        f.read(V, by_col);
        settle<T>();
        if (!whole) {
            const int left = here(x.lim - j0 - 4 * (l >> 5));
#pragma unroll
            for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kb][r] = kb * 32 + el(r) < left ? s[kb][r] : -INFINITY;
        }
    } else {
        settle<T>();
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            s[kb] = cap_scores<false>(cap, s[kb]).s;
            const int rel0 = j0 + kb * 32 + 4 * (l >> 5) - x.p;
            s[kb] = add_bias<1>(a, bs, rel0, j0 + kb * 32 - wr.last, j0 + kb * 32 + 31 - wr.first, s[kb]);
            if (!whole) s[kb] = mask_keys(a, x, j0 + kb * 32, kd + kb * 32, l, s[kb]);
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
    top = halves_max(top);
    // the maximum so far is of raw products
    if (KIND == kPlain) top *= cap.c;
    if (KIND == kCapped)
        top = top == -INFINITY ? top : fma_acc(quick_r(top, cap.k), -2.f * cap.top, cap.top);
    const bool grow = top > st.m + (kLazy + kBelow<T>);
    if (__any(grow)) {
        const float keep = grow ? __builtin_amdgcn_exp2f(st.m - (top - kBelow<T>)) : 1.f;
        st.m = grow ? top - kBelow<T> : st.m;
        st.z *= keep;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) st.o[d] *= keep;
    }
    const float m = st.m == -INFINITY ? 0.f : st.m;
    const float up = cap.top - m;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float y = KIND == kPlain    ? fma_acc(s[kb][r], cap.c, -m)
                            : KIND == kCapped ? fma_acc(quick_r(s[kb][r], cap.k), -2.f * cap.top, up)
                                              : s[kb][r] - m;
            s[kb][r] = __builtin_amdgcn_exp2f(y);
        }
    if (KIND == kCapped && !whole) {  // the cap of -inf is finite
        const int left = here(x.lim - j0 - 4 * (l >> 5));
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] = kb * 32 + el(r) < left ? s[kb][r] : 0.f;
    }
    float z0 = 0.f, z1 = 0.f;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; r += 2) z0 += s[kb][r], z1 += s[kb][r + 1];
    st.z += z0 + z1;
    order();
    if (KIND == kGeneral) f.read(V, by_col);
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
        ColumnFragments<T, DP> ahead;
        if (kb + 1 < NB) ahead.read(V, by_col, kb * 32 + 32);
        priority<1>();
        f.weigh(st.o, s[kb]);
        priority<0>();
        order();
        if (kb + 1 < NB) f = ahead;
    }
    settle<T>();
}

// Rows whose result is no number are computed again pair by pair.
template <typename T, int ND>
__device__ __forceinline__ void recompute_bad(const Att& a, int b, const LaneRow& x, const f32x16 (&o)[ND]) {
    float bad = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = fma_acc(o[d][r], 0.f, bad);
    unsigned long long rows = __ballot(bad != 0.f);
    rows = (rows | rows >> 32) & 0xffffffffull & __ballot(x.live);
#pragma unroll 1
    for (; rows; rows &= rows - 1) {
        const int t = __builtin_ctzll(rows);
        exact_row<T>(a, b, __shfl(x.h, t), __shfl(x.i, t));
    }
}

template <typename T, int DP>
struct FwdShape {
    using L = Tile<T, DP>;
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32;       // keys of a shared tile
    static constexpr int NBUF = L::ROW > 256 ? 1 : 2;         // of a wave's own 32-key tile
    static constexpr int kShared = 2 * 2 * KT * L::ROW;       // two buffers of K and V
    static constexpr int kOwn = kAttWaves * NBUF * 2 * 32 * L::ROW;
};

template <typename T, int DP, Kind KIND>
__global__ __launch_bounds__(kAttThreads, DP * sizeof(T) > 384 ? 1 : 2) void att_fwd_kernel(Att a) {
    using S = FwdShape<T, DP>;
    using L = Tile<T, DP>;
    constexpr int KT = S::KT, NB = KT / 32, HALF = KT * L::ROW;
    // two buffers under names of their own: reads of one then do not wait for
    // the loads under way into the other
    __shared__ __attribute__((aligned(1024))) char tiles0[2][HALF];
    __shared__ __attribute__((aligned(1024))) char tiles1[2][HALF];
    __shared__ __attribute__((aligned(256))) int docs0[64], docs1[64];
    extern __shared__ float line[];
    const int l = threadIdx.x & 63, wave = wave_id();
    const int G = a.Hq / a.pack;
    int bg, rest;
    place(blockIdx.x, a.B * G, bg, rest);
    const int b = bg / G, group = bg - b * G, rb = a.rblocks - 1 - rest;
    const int n = filled_keys(a, b), hk = group * a.pack / a.per;
    const LaneRow x = lane_row(a, b, group, rb * 128 + wave * 32 + (l & 31), n);
    const WaveRows wr = wave_rows(x);
    const Cap cap = cap_of<T, KIND>(a, false);
    if (KIND == kGeneral && a.table) stage_line<T>(a, group, line);  // read after the first barrier
    const Bias bs = lane_bias(a, x.h, line);
    typename Eight<T>::V q[L::NS];
    load_row<T, DP>(q, row_at<T>(a.q, a.qs, b, x.h, x.i), a.D, l);
    if (a.scale < 0.f)
        for (int s = 0; s < L::NS; ++s) q[s] = Eight<T>::negate(q[s]);

    Loader<T, DP, KT, kAttWaves> lk, lv;
    lk.init(threadIdx.x, a.ks[2], a.D);
    lv.init(threadIdx.x, a.vs[2], a.D);
    const T* kbase = row_at<T>(a.k, a.ks, b, hk, 0);
    const T* vbase = row_at<T>(a.v, a.vs, b, hk, 0);
    const int32_t* dbase = KIND == kGeneral && a.documents ? a.documents + static_cast<int64_t>(b) * a.Lk : nullptr;
    auto load = [&](int t, char (&tiles)[2][HALF], int (&docs)[64]) {
        lk.load(tiles[0], kbase, a.ks[2], t * KT, n, a.D, wave);
        lv.load(tiles[1], vbase, a.vs[2], t * KT, n, a.D, wave);
        if (dbase && wave == 0) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<int32_t*>(dbase + t * KT), static_cast<short>(0),
                static_cast<int>(min(n - t * KT, 64) * 4), 0x00020000);
            to_lds<4>(rs, docs, l * 4);
        }
    };
    const int end = (keys_end(a, b, rb * 128 + 127, n) + KT - 1) / KT;
    const int2 own = KIND == kGeneral && a.documents ? row_documents(a, b, rb * 128, 128, n) : make_int2(0, 0);
    auto wanted = [&](int t) {
        if (KIND != kGeneral || !a.documents) return true;
        const int e = t * KT / kRangeKeys;
        if (e >= a.nranges) return false;
        const int2 r = a.ranges[b * a.nranges + e];
        return r.x <= own.y && own.x <= r.y;
    };
    Needed<decltype(wanted)> need{wanted};
    Running<L::ND> st{};
    st.m = -INFINITY;
    int t = need.next(0, end);
    const int by_row = L::row_base(0, l), by_col = L::col_base(0, l);
    auto step = [&](char (&tiles)[2][HALF], int (&docs)[64], char (&ahead)[2][HALF], int (&docs_ahead)[64]) {
        const int tn = KIND == kGeneral && a.documents ? need.next(t + 1, end) : t + 1;
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the tile has landed
        __syncthreads();
        if (tn < end) load(tn, ahead, docs_ahead);
        if (t * KT < wr.most)
            attend<T, DP, NB, KIND>(a, cap, bs, x.r, wr, q, tiles[0], tiles[1], by_row, by_col, docs, t * KT, l, st);
        t = tn;
    };
    if (t < end) load(t, tiles0, docs0);
    while (t < end) {
        step(tiles0, docs0, tiles1, docs1);
        if (t < end) step(tiles1, docs1, tiles0, docs0);
    }
    const float z = halves_sum(st.z);
    const float inv = z == 0.f ? 0.f : 1.f / z;
#pragma unroll
    for (int d = 0; d < L::ND; ++d) st.o[d] *= inv;
    if (x.live) {
        T* out = const_cast<T*>(row_at<T>(a.out, a.os, b, x.h, x.i));
#pragma unroll
        for (int d = 0; d < L::ND; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int at = d * 32 + 8 * c + 4 * (l >> 5);
                if (at < a.D)
                    store4<T>(out + at, f32x4{st.o[d][4 * c], st.o[d][4 * c + 1], st.o[d][4 * c + 2], st.o[d][4 * c + 3]});
            }
        if (a.rest) {
            T* rest = rest_at<T>(a, b, x.h, x.i);
#pragma unroll
            for (int d = 0; d < L::ND; ++d)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int at = d * 32 + 8 * c + 4 * (l >> 5);
                    if (at < a.D)
                        store4_rest<T>(rest + at, f32x4{st.o[d][4 * c], st.o[d][4 * c + 1], st.o[d][4 * c + 2], st.o[d][4 * c + 3]});
                }
        }
        if (l < 32) put_stats(a, (static_cast<int64_t>(b) * a.Hq + x.h) * a.Lq + x.i, st.m, z);
    }
    recompute_bad<T, L::ND>(a, b, x, st.o);
}

// The waves split the keys.
template <typename T, int DP, Kind KIND>
__global__ __launch_bounds__(kAttThreads, 1) void att_fwd_split_kernel(Att a) {
    using S = FwdShape<T, DP>;
    using L = Tile<T, DP>;
    constexpr int HALF = 32 * L::ROW;
    __shared__ __attribute__((aligned(1024))) char tiles0[kAttWaves][2][HALF];
    __shared__ __attribute__((aligned(1024))) char tiles1[S::NBUF == 2 ? kAttWaves : 1][2][S::NBUF == 2 ? HALF : 16];
    __shared__ __attribute__((aligned(256))) int docs0[kAttWaves][64], docs1[kAttWaves][64];
    __shared__ float stat[kAttWaves][2][32];
    extern __shared__ float line[];
    static_assert(sizeof(tiles0) >= kAttWaves * 32 * DP * 4, "the waves' sums take the tiles' place");
    const int l = threadIdx.x & 63, wave = wave_id();
    const int G = a.Hq / a.pack;
    int bg, rest;
    place(blockIdx.x, a.B * G, bg, rest);
    const int b = bg / G, group = bg - b * G, split = rest % a.splits, rb = a.rblocks - 1 - rest / a.splits;
    const int n = filled_keys(a, b), hk = group * a.pack / a.per;
    const LaneRow x = lane_row(a, b, group, rb * 32 + (l & 31), n);
    const WaveRows wr = wave_rows(x);
    const Cap cap = cap_of<T, KIND>(a, false);
    if (KIND == kGeneral && a.table) {
        stage_line<T>(a, group, line);
        __syncthreads();
    }
    const Bias bs = lane_bias(a, x.h, line);

    Loader<T, DP, 32, 1> lk, lv;
    lk.init(l, a.ks[2], a.D);
    lv.init(l, a.vs[2], a.D);
    const T* kbase = row_at<T>(a.k, a.ks, b, hk, 0);
    const T* vbase = row_at<T>(a.v, a.vs, b, hk, 0);
    const int32_t* dbase = KIND == kGeneral && a.documents ? a.documents + static_cast<int64_t>(b) * a.Lk : nullptr;
    auto load = [&](int t, char* tile, int* docs) {
        lk.load(tile, kbase, a.ks[2], t * 32, n, a.D, 0);
        lv.load(tile + HALF, vbase, a.vs[2], t * 32, n, a.D, 0);
        if (dbase) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<int32_t*>(dbase + t * 32), static_cast<short>(0),
                static_cast<int>(min(n - t * 32, 64) * 4), 0x00020000);
            to_lds<4>(rs, docs, l * 4);
        }
    };
    const int64_t tiles_all = (keys_end(a, b, rb * 32 + 31, n) + 31) / 32;
    const int unit = split * kAttWaves + wave, units = a.splits * kAttWaves;
    const int begin = static_cast<int>(tiles_all * unit / units), end = static_cast<int>(tiles_all * (unit + 1) / units);
    const int2 own = KIND == kGeneral && a.documents ? row_documents(a, b, rb * 32, 32, n) : make_int2(0, 0);
    auto wanted = [&](int t) {
        if (KIND != kGeneral || !a.documents) return true;
        const int e = t * 32 / kRangeKeys;
        if (e >= a.nranges) return false;
        const int2 r = a.ranges[b * a.nranges + e];
        return r.x <= own.y && own.x <= r.y;
    };
    Needed<decltype(wanted)> need{wanted};
    Running<L::ND> st{};
    st.m = -INFINITY;
    int t = need.next(begin, end);
    if (t < end) load(t, tiles0[wave][0], docs0[wave]);
    typename Eight<T>::V q[L::NS];
    load_row<T, DP>(q, row_at<T>(a.q, a.qs, b, x.h, x.i), a.D, l);
    if (a.scale < 0.f)
        for (int s = 0; s < L::NS; ++s) q[s] = Eight<T>::negate(q[s]);
    const int by_row = L::row_base(0, l), by_col = L::col_base(0, l);
    auto step = [&](char* tile, int* docs, char* ahead, int* docs_ahead) {
        const int tn = KIND == kGeneral && a.documents ? need.next(t + 1, end) : t + 1;
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the tile has landed
        if (S::NBUF == 2 && tn < end) load(tn, ahead, docs_ahead);
        attend<T, DP, 1, KIND>(a, cap, bs, x.r, wr, q, tile, tile + HALF, by_row, by_col, docs, t * 32, l, st);
        if (S::NBUF == 1 && tn < end) {
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the tile has been read
            load(tn, tile, docs);
        }
        t = tn;
    };
    while (t < end) {
        step(tiles0[wave][0], docs0[wave], tiles1[S::NBUF == 2 ? wave : 0][0], docs1[wave]);
        if (S::NBUF == 2 && t < end) step(tiles1[S::NBUF == 2 ? wave : 0][0], docs1[wave], tiles0[wave][0], docs0[wave]);
    }
    // the waves' sums, to one maximum, in their order
    const float z = halves_sum(st.z);
    if (l < 32) stat[wave][0][l] = st.m, stat[wave][1][l] = z;
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kAttWaves; ++w) top = fmaxf(top, stat[w][0][l & 31]);
    const float zero = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kAttWaves; ++w)
        total += stat[w][1][l & 31] * __builtin_amdgcn_exp2f(stat[w][0][l & 31] - zero);
    const bool last = a.splits == 1;
    const float mine = __builtin_amdgcn_exp2f(st.m - zero) * (!last ? 1.f : total == 0.f ? 0.f : 1.f / total);
    float* sums = reinterpret_cast<float*>(&tiles0[0][0][0]);  // [wave][column][row]
#pragma unroll
    for (int d = 0; d < L::ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            sums[(wave * DP + d * 32 + el(r) + 4 * (l >> 5)) * 32 + (l & 31)] = st.o[d][r] * mine;
    __syncthreads();
    // [row][split][D], then [row][split][maximum, sum]
    const int64_t at = (static_cast<int64_t>(b) * a.Hq + x.h) * a.Lq + x.i;
    float* const stats = a.part + static_cast<int64_t>(a.B) * a.Hq * a.Lq * a.splits * a.D;
    const int row = threadIdx.x & 31;
    float bad = 0.f;
    for (int d = (threadIdx.x >> 5) * 4; d < a.D; d += kAttThreads / 32 * 4) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = sums[(d + e) * 32 + row];
#pragma unroll
            for (int w = 1; w < kAttWaves; ++w) v[e] += sums[(w * DP + d + e) * 32 + row];
            bad = fma_acc(v[e], 0.f, bad);
        }
        if (!x.live) continue;
        if (last) {
            store4<T>(const_cast<T*>(row_at<T>(a.out, a.os, b, x.h, x.i)) + d, v);
            if (a.rest) store4_rest<T>(rest_at<T>(a, b, x.h, x.i) + d, v);
        } else
            *reinterpret_cast<f32x4*>(a.part + (at * a.splits + split) * a.D + d) = v;
    }
    if (wave == 0 && l < 32 && x.live) {
        if (!last) {
            stats[(at * a.splits + split) * 2] = top;
            stats[(at * a.splits + split) * 2 + 1] = total;
        } else {
            put_stats(a, at, top, total);
        }
    }
    if (!last) return;
    if (!__syncthreads_or(bad != 0.f)) return;
    // some row is no number: its columns lie with several threads
    float* rows = &stat[0][0][0];
    if (threadIdx.x < 32) rows[threadIdx.x] = 0.f;
    __syncthreads();
    if (bad != 0.f) rows[row] = 1.f;
    __syncthreads();
    for (int r = wave; r < 32; r += kAttWaves)
        if (rows[r] != 0.f && __shfl(static_cast<int>(x.live), r)) exact_row<T>(a, b, __shfl(x.h, r), __shfl(x.i, r));
}

// Joins the workgroups that shared a row's keys: one wave per row.
template <typename T>
__global__ __launch_bounds__(kAttThreads) void att_join_kernel(Att a) {
    const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Lq;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kAttWaves + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int l = threadIdx.x & 63, S = a.splits;
    const float* stat = a.part + rows * S * a.D + row * S * 2;
    const float* sums = a.part + row * S * a.D;
    float top = -INFINITY, z = 0.f, o[2] = {};
    for (int s = 0; s < S; ++s) top = fmaxf(top, stat[2 * s]);
    const float zero = top == -INFINITY ? 0.f : top;
#pragma unroll 4
    for (int s = 0; s < S; ++s) {
        const float w = __builtin_amdgcn_exp2f(stat[2 * s] - zero);
        z = fma_acc(w, stat[2 * s + 1], z);
#pragma unroll
        for (int c = 0; c < 2; ++c)
            if (l + c * 64 < a.D) o[c] = fma_acc(w, sums[s * a.D + l + c * 64], o[c]);
    }
    const int i = static_cast<int>(row % a.Lq), h = static_cast<int>(row / a.Lq % a.Hq),
              b = static_cast<int>(row / a.Lq / a.Hq);
    T* out = const_cast<T*>(row_at<T>(a.out, a.os, b, h, i));
    float bad = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c)
        if (l + c * 64 < a.D) {
            const float v = z == 0.f ? 0.f : o[c] / z;
            bad = fma_acc(v, 0.f, bad);
            out[l + c * 64] = from_acc<T>(v);
            if (a.rest) rest_at<T>(a, b, h, i)[l + c * 64] = from_acc<T>(rounded_off<T>(v));
        }
    if (l == 0) put_stats(a, row, top, z);
    if (__any(bad != 0.f)) exact_row<T>(a, b, h, i);
}

template <typename T, int DP, Kind KIND>
static void forward_kind(const Att& a, hipStream_t st) {
    const unsigned lds = a.table ? (2 * a.reach + 1) * 4 : 0;
    const int64_t blocks = static_cast<int64_t>(a.B) * (a.Hq / a.pack) * a.rblocks;
    if (a.splits == 0)
        att_fwd_kernel<T, DP, KIND><<<static_cast<unsigned>(blocks), kAttThreads, lds, st>>>(a);
    else
        att_fwd_split_kernel<T, DP, KIND><<<static_cast<unsigned>(blocks * a.splits), kAttThreads, lds, st>>>(a);
}

template <typename T, int DP>
static void forward_width(const Att& a, hipStream_t st) {
    const Kind kind = kind_of<T>(a);
    if constexpr (sizeof(T) == 2)  // fp32 has no quick cap
        if (kind == kCapped) return forward_kind<T, DP, kCapped>(a, st);
    if (kind == kPlain) forward_kind<T, DP, kPlain>(a, st);
    else forward_kind<T, DP, kGeneral>(a, st);
}

template <typename T>
int attention_forward_launch(const Att& a, hipStream_t st) {
    if (a.D <= 32) forward_width<T, 32>(a, st);
    else if (a.D <= 64) forward_width<T, 64>(a, st);
    else if (a.D <= 96) forward_width<T, 96>(a, st);
    else forward_width<T, 128>(a, st);
    if (int rc = nsh_host::check_launch("attention_forward")) return rc;
    if (a.splits > 1) {
        const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Lq;
        att_join_kernel<T><<<static_cast<unsigned>(nsh_host::ceil_div(rows, kAttWaves)), kAttThreads, 0, st>>>(a);
        return nsh_host::check_launch("attention_join");
    }
    return NSH_OK;
}

}  // namespace nsh
