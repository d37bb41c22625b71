// attention_bwd.hpp -- the gradients of the biased attention.
//
//   p = exp(s) / degree          dS = p (dO v - delta)    delta = dO out - ddegree
//   dv = p^T dO    dx = dS (1 - tanh^2) scale    dq = dx k    dk = dx^T q
//   dtable[bucket] = the sum of dS over the bucket's pairs
//
// Two launches that form the scores anew, rather than one that adds up dq
// between workgroups: every sum has one owner and one order, for seven matrix
// products instead of five.
//   1. by query rows, as the forward (a wave has 32 rows, one to a lane pair):
//      delta, dq, and the table's sums per relative position.
//   2. by keys (a wave has 32 keys): walks the queries of all heads of its key
//      head; dk and dv stay in registers.  Where that leaves the card short of
//      workgroups, or their loads uneven, `parts` workgroups share a key
//      block's queries and a third launch adds their sums.
//
// What bounds them (times as in the forward): by rows as there the vector work of a
// score next to its products, 60% and 40% of the time: 2 x 16 heads, 4 of keys, 4096
// tokens, width 128, causal, capped, bf16: 231 us, 890 TFLOP/s.  By keys, 324 us, 850,
// and 17 for the join, vector work is 44%, products 34%, LDS reads 30% (2.3 for each
// product: K and V come from there again for every 32 rows), and the waves wait 28% of
// their time: no one unit is full.  The accumulators fill half of the registers at
// width 128, which leaves one wave to a SIMD; by keys, two fit with K and V in LDS
// instead (`kPaired`).  4 x 12 heads, 1024 tokens, width 64 with a learned bias, bf16:
// 58 and 70 us, and 7 for the table; documents in rows of 2500, 2 x 12 heads, fp16: 55
// and 59: waves wait 40 to 47% of their time, one to a SIMD on average.
#pragma once

#include "attention_rows.hpp"
#include "positionbias.hpp"

namespace nsh {

// The table's sums per relative position, of one wave.  A tile's 63 diagonals
// are lined up in LDS, one to a lane's run of 32 places (a place that no pair
// of a tile falls on stays zero).  Keys come in ascending order and a diagonal
// crosses two tiles at most, so after a tile the lower 32 are complete and go
// out; the upper 31 wait for the next.  Positions beyond the reach are sums in
// registers.
struct TableSums {
    float* lines;  // in LDS, zero at first
    float* out;    // by relative position + reach, zero at first
    float carry;   // lane l < 31: relative position next - 31 + l
    int next;      // the tile (key less the wave's first row) that the carry waits for
    float low, high;
};

__device__ __forceinline__ void table_out(const Att& a, TableSums& ts, int rel, float s) {
    if (rel <= -a.reach) ts.low += s;
    else if (rel >= a.reach) ts.high += s;
    else ts.out[rel + a.reach] = s;
}

__device__ __forceinline__ void table_flush(const Att& a, TableSums& ts, int l) {
    if (l < 31) table_out(a, ts, ts.next - 31 + l, ts.carry);
    ts.carry = 0.f;
}

__device__ __forceinline__ void add_table(const Att& a, TableSums& ts, int rel0, int least, int most, int l,
                                          const f32x16& ds) {
    if (most <= -a.reach || least >= a.reach) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) s += ds[r];
        if (least >= a.reach) ts.high += s; else ts.low += s;
        return;
    }
    // diagonal key - row + 31, place row
    float* at = ts.lines + (4 * (l >> 5) - (l & 31) + 31) * kDiagonal + (l & 31);
#pragma unroll
    for (int r = 0; r < 16; ++r) at[el(r) * kDiagonal] = ds[r];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x4 v = {};
    if (l < 63) {
#pragma unroll
        for (int c = 0; c < 8; ++c) v += *reinterpret_cast<const f32x4*>(ts.lines + l * kDiagonal + 4 * c);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    float s = (v[0] + v[1]) + (v[2] + v[3]);
    if (rel0 != ts.next && ts.next != -0x40000000) table_flush(a, ts, l);
    if (l < 31) s += ts.carry;
    if (l < 32) table_out(a, ts, rel0 - 31 + l, s);
    ts.carry = __shfl_down(s, 32);
    ts.next = rel0 + 32;
}

// The gradients by keys of a plain 16-bit call have 1 / sum in the exponent next to
// the maximum.  A row whose two come to less than this is off by less than 2^-15 of
// its weights, a sixteenth of an fp16 weight's own half step; the launch by rows
// notes, wave by wave, where some row is beyond.
constexpr float kNear = 1024.f;
template <typename T, Kind KIND> constexpr bool kNotes = KIND == kPlain && sizeof(T) == 2;

template <typename T, int DP>
struct BwdShape {
    using L = Tile<T, DP>;
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32;
    static constexpr int NBUF = L::ROW > 256 ? 1 : 2;
};

// 32 keys' part of the wave's dq, and of the table's sums.
template <typename T, int DP, Kind KIND>
__device__ __forceinline__ void row_gradient(const Att& a, const Cap& cap, const Bias& bs, const Row& x,
                                             const WaveRows& wr, const typename Eight<T>::V (&q)[DP / 16],
                                             const typename Eight<T>::V (&go)[DP / 16], float2 stat, float delta,
                                             const char* K, const char* V, int by_row, int by_col, const int* kd, int j0, int l,
                                             TableSums* ts, float& by, f32x16 (&dq)[DP / 32]) {
    f32x16 s, dp;
    {
        RowFragments<T, DP> fk, fv;
        fk.read(K, by_row), fv.read(V, by_row);
        // here the vector work goes ahead of the other wave's products (first dozen
        // launches, 2 x 16 heads of 4096, causal, capped: 291 us without, 267 with, 287
        // the other way round, as the forward has it; by keys neither changes anything)
        priority<0>();
        s = fk.products(q), dp = fv.products(go);
        priority<1>();
    }
    ColumnFragments<T, DP> f;
    f.read(K, by_col);
    if (KIND != kGeneral) {
        order();
        // 1 / sum goes to the other factor: in the exponent, next to a maximum of
        // thousands, it would lose its last places
        const float up = (KIND == kCapped ? cap.top : 0.f) - stat.x;
        const float y = kNarrow<T> ? stat.y * by : stat.y, d = delta * y;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (KIND == kPlain) {
                dp[r] = __builtin_amdgcn_exp2f(fma_acc(s[r], cap.c, up)) * fma_acc(dp[r], y, -d);
            } else {
                const float c = quick_r(s[r], cap.k);
                dp[r] = __builtin_amdgcn_exp2f(fma_acc(c, -2.f * cap.top, up)) * fma_acc(dp[r], y, -d) *
                        (4.f * fma_acc(-c, c, c));
            }
        }
        if (j0 + 32 > wr.least) {  // 0 times what an unseen pair holds is not always 0
            const int left = here(x.lim - j0 - 4 * (l >> 5));
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = el(r) < left ? dp[r] : 0.f;
        }
    } else {
        settle<T>();
        const Scores y = cap_scores<true>(cap, s);
        const int rel0 = j0 + 4 * (l >> 5) - x.p, least = j0 - wr.last, most = j0 + 31 - wr.first;
        s = add_bias<1>(a, bs, rel0, least, most, y.s);
        const bool whole = j0 + 32 <= wr.least && !a.documents;
        if (!whole) s = mask_keys(a, x, j0, kd, l, s);
        const float w = kNarrow<T> ? stat.y * by : stat.y, d = delta * w;
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = __builtin_amdgcn_exp2f(s[r] - stat.x) * fma_acc(dp[r], w, -d);
        if (!whole) {
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = s[r] == -INFINITY ? 0.f : dp[r];
        }
        if (ts) add_table(a, *ts, j0 - wr.first, least, most, l, kNarrow<T> ? dp * (1.f / by) : dp);
        if (cap.mode != 0) dp *= y.w;
    }
    dp = fit<T>(by, dp, dq);
    priority<0>();
    f.weigh_fine(dq, dp);
    priority<1>();
    settle<T>();
}

template <typename T, int DP, bool SPLIT, Kind KIND>
__global__ __launch_bounds__(kAttThreads, SPLIT || DP * sizeof(T) > (KIND == kGeneral ? 192 : 256) ? 1 : 2) void att_bwd_row_kernel(Att a) {
    using L = Tile<T, DP>;
    using S = BwdShape<T, DP>;
    constexpr int KT = SPLIT ? 32 : S::KT, NB = KT / 32, HALF = KT * L::ROW;
    constexpr int ROWS = SPLIT ? 32 : 128, OWN = SPLIT ? kAttWaves : 1;
    constexpr int NBUF = SPLIT ? S::NBUF : 2;
    // K and V tiles, one buffer after the other, under names of their own:
    // reads of one do not wait for the loads under way into the other
    __shared__ __attribute__((aligned(1024))) char tiles0[OWN][2][HALF];
    __shared__ __attribute__((aligned(1024))) char tiles1[NBUF == 2 ? OWN : 1][2][NBUF == 2 ? HALF : 16];
    __shared__ __attribute__((aligned(256))) int docs0[OWN][64], docs1[OWN][64];
    extern __shared__ __attribute__((aligned(16))) float room[];  // line, then the table's sums
    const int l = threadIdx.x & 63, wave = wave_id();
    int bh, rest;
    place(blockIdx.x, a.B * a.Hq, bh, rest);
    const int b = bh / a.Hq, h = bh - b * a.Hq, rb = a.rblocks - 1 - rest;
    const int n = filled_keys(a, b), hk = h / a.per;
    const LaneRow x = lane_row(a, b, h, rb * ROWS + (SPLIT ? 0 : wave * 32) + (l & 31), n);
    const WaveRows wr = wave_rows(x);
    const Cap cap = cap_of<T, KIND>(a, true);
    if (KIND == kGeneral && a.table) stage_line<T>(a, h, room);
    const Bias bs = lane_bias(a, h, room);
    TableSums sums{};
    if (KIND == kGeneral && a.gtable) {
        const int n2 = 2 * a.reach + 1;
        sums.lines = room + ((n2 + 3) & ~3) + wave * kDiagonals;
        sums.out = a.bins + (((static_cast<int64_t>(h) * a.B + b) * a.rblocks + rb) * kAttWaves + wave) * n2;
        for (int i = l; i < kDiagonals; i += 64) sums.lines[i] = 0.f;
        for (int i = l; i < n2; i += 64) sums.out[i] = 0.f;
        sums.next = -0x40000000;
    }
    if (KIND == kGeneral && a.table) __syncthreads();

    const int64_t at = (static_cast<int64_t>(b) * a.Hq + h) * a.Lq + x.i;
    typename Eight<T>::V q[L::NS], go[L::NS];
    load_row<T, DP>(q, row_at<T>(a.out, a.os, b, h, x.i), a.D, l);
    load_row<T, DP>(go, row_at<T>(a.go, a.gos, b, h, x.i), a.D, l);
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < L::NS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fma_acc(static_cast<float>(q[s][e]), static_cast<float>(go[s][e]), delta);
    if (a.rest) {
        load_row<T, DP>(q, rest_at<T>(a, b, h, x.i), a.D, l);
#pragma unroll
        for (int s = 0; s < L::NS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fma_acc(static_cast<float>(q[s][e]), static_cast<float>(go[s][e]), delta);
    }
    delta = halves_sum(delta) - (a.gdegree ? a.gdegree[at] : 0.f);
    if (x.live && l < 32 && (!SPLIT || wave == 0)) a.delta[at] = delta;
    load_row<T, DP>(q, row_at<T>(a.q, a.qs, b, h, x.i), a.D, l);
    // rows that see nothing, and lanes that stand in for no row, weigh nothing
    float2 stat = get_stats(a, at);
    if (!x.live) stat.y = 0.f;
    if constexpr (kNotes<T, KIND>) {
        const int beyond = __any(stat.y != 0.f && fabsf(__builtin_amdgcn_logf(stat.y * kRoom<T>) - stat.x) > kNear);
        if (l == 0) a.far[((static_cast<int64_t>(b) * a.Hq + h) * a.rblocks + rb) * kAttWaves + wave] = beyond;
    }

    Loader<T, DP, KT, SPLIT ? 1 : kAttWaves> lk, lv;
    lk.init(SPLIT ? l : threadIdx.x, a.ks[2], a.D);
    lv.init(SPLIT ? l : threadIdx.x, a.vs[2], a.D);
    const T* kbase = row_at<T>(a.k, a.ks, b, hk, 0);
    const T* vbase = row_at<T>(a.v, a.vs, b, hk, 0);
    const int32_t* dbase = KIND == kGeneral && a.documents ? a.documents + static_cast<int64_t>(b) * a.Lk : nullptr;
    auto load = [&](int t, char* tile, int* docs) {
        lk.load(tile, kbase, a.ks[2], t * KT, n, a.D, SPLIT ? 0 : wave);
        lv.load(tile + HALF, vbase, a.vs[2], t * KT, n, a.D, SPLIT ? 0 : wave);
        if (dbase && (SPLIT || wave == 0)) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<int32_t*>(dbase + t * KT), static_cast<short>(0),
                static_cast<int>(min(n - t * KT, 64) * 4), 0x00020000);
            to_lds<4>(rs, docs, l * 4);
        }
    };
    const int64_t tiles_all = (keys_end(a, b, rb * ROWS + ROWS - 1, n) + KT - 1) / KT;
    const int begin = SPLIT ? static_cast<int>(tiles_all * wave / kAttWaves) : 0;
    const int end = SPLIT ? static_cast<int>(tiles_all * (wave + 1) / kAttWaves) : static_cast<int>(tiles_all);
    const int2 own = KIND == kGeneral && a.documents ? row_documents(a, b, rb * ROWS, ROWS, n) : make_int2(0, 0);
    auto wanted = [&](int t) {
        if (KIND != kGeneral || !a.documents) return true;
        const int e = t * KT / kRangeKeys;
        if (e >= a.nranges) return false;
        const int2 r = a.ranges[b * a.nranges + e];
        return r.x <= own.y && own.x <= r.y;
    };
    Needed<decltype(wanted)> need{wanted};
    f32x16 dq[L::ND] = {};
    float by = kFitFirst;  // what dq's weights are times
    int t = need.next(begin, end);
    TableSums* const ts = KIND == kGeneral && a.gtable ? &sums : nullptr;
    const int by_row = L::row_base(0, l), by_col = L::col_base(0, l);
    auto compute = [&](const char* tile, const int* docs) {
#pragma unroll 1
        for (int kb = 0; kb < NB; ++kb)
        {
            const int j0 = t * KT + kb * 32;
            if (j0 >= wr.most) break;
            row_gradient<T, DP, KIND>(a, cap, bs, x.r, wr, q, go, stat, delta, tile + kb * 32 * L::ROW,
                                      tile + HALF + kb * 32 * L::ROW, by_row, by_col, docs + kb * 32, j0, l, ts, by, dq);
        }
    };
    auto step = [&](char* tile, int* docs, char* ahead, int* docs_ahead) {
        const int tn = KIND == kGeneral && a.documents ? need.next(t + 1, end) : t + 1;
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the tile has landed
        if (!SPLIT) __syncthreads();
        if (NBUF == 2 && tn < end) load(tn, ahead, docs_ahead);
        compute(tile, docs);
        if (NBUF == 1 && tn < end) {
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the tile has been read
            load(tn, tile, docs);
        }
        t = tn;
    };
    const int mine = SPLIT ? wave : 0;
    if (t < end) load(t, tiles0[mine][0], docs0[mine]);
    while (t < end) {
        step(tiles0[mine][0], docs0[mine], tiles1[NBUF == 2 ? mine : 0][0], docs1[mine]);
        if (NBUF == 2 && t < end) step(tiles1[NBUF == 2 ? mine : 0][0], docs1[mine], tiles0[mine][0], docs0[mine]);
    }
    float bad = 0.f;
    const float last = kNarrow<T> ? a.scale / by : a.scale;
#pragma unroll
    for (int d = 0; d < L::ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[d][r] *= last, bad = fma_acc(dq[d][r], 0.f, bad);
    if constexpr (SPLIT) {
        // the waves' sums in their order, half of the columns at a time
        float* part = reinterpret_cast<float*>(&tiles0[0][0][0]);  // [wave][column][row]
        static_assert(sizeof(tiles0) >= kAttWaves * 32 * DP * 2, "half of the waves' sums take the tiles' place");
        constexpr int HALVES = sizeof(tiles0) >= kAttWaves * 32 * DP * 4 ? 1 : L::ND;
        constexpr int NDH = L::ND / HALVES;
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < NDH; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    part[(wave * NDH * 32 + d * 32 + el(r) + 4 * (l >> 5)) * 32 + (l & 31)] = dq[half * NDH + d][r];
            __syncthreads();
            for (int d = (threadIdx.x >> 5) * 4; d < NDH * 32 && half * NDH * 32 + d < a.D; d += kAttThreads / 32 * 4) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = part[(d + e) * 32 + (l & 31)];
#pragma unroll
                    for (int w = 1; w < kAttWaves; ++w) v[e] += part[((w * NDH * 32) + d + e) * 32 + (l & 31)];
                }
                if (x.live)
                    store4<T>(const_cast<T*>(row_at<T>(a.gq, a.gqs, b, h, x.i)) + half * NDH * 32 + d, v);
            }
        }
        // all waves have the same rows: a bad one in any wave is bad
        __syncthreads();
        int* flags = reinterpret_cast<int*>(part);
        if (threadIdx.x < 32) flags[threadIdx.x] = 0;
        __syncthreads();
        if (bad != 0.f) flags[l & 31] = 1;
        __syncthreads();
        unsigned long long rows = __ballot(flags[l & 31] && x.live) & 0xffffffffull;
        for (int c = 0; rows; rows &= rows - 1, ++c) {
            const int u = __builtin_ctzll(rows);
            if (c % kAttWaves == wave) exact_row_gradient<T>(a, b, h, __shfl(x.i, u), __shfl(delta, u));
        }
    } else {
        if (x.live) {
            T* out = const_cast<T*>(row_at<T>(a.gq, a.gqs, b, h, x.i));
#pragma unroll
            for (int d = 0; d < L::ND; ++d)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int col = d * 32 + 8 * c + 4 * (l >> 5);
                    if (col < a.D)
                        store4<T>(out + col, f32x4{dq[d][4 * c], dq[d][4 * c + 1], dq[d][4 * c + 2], dq[d][4 * c + 3]});
                }
        }
        unsigned long long rows = __ballot(bad != 0.f);
        rows = (rows | rows >> 32) & 0xffffffffull & __ballot(x.live);
#pragma unroll 1
        for (; rows; rows &= rows - 1) {
            const int u = __builtin_ctzll(rows);
            exact_row_gradient<T>(a, b, h, __shfl(x.i, u), __shfl(delta, u));
        }
    }
    if (KIND != kGeneral || !a.gtable) return;
    if (sums.next != -0x40000000) table_flush(a, sums, l);
    sums.low = wave_sum(sums.low), sums.high = wave_sum(sums.high);
    if (l == 0) {
        sums.out[0] = a.reach ? sums.low : sums.low + sums.high;
        if (a.reach) sums.out[2 * a.reach] = sums.high;
    }
}

// How the waves share a workgroup's work: KG groups of 32 keys, and QP waves to
// a group, one for each half of a 64-row tile; the second waves' sums join the
// first's at the end.
//   kAlone   4 x 1
//   kTwin    2 x 2: for heads up to 64 wide, twice the workgroups of half the
//            length each
//   kPaired  4 x 2, with K and V in LDS rather than in registers: of those, the
//            sums of wider heads leave too few for two waves to a SIMD otherwise,
//            and one wave waits for its own products
enum Share { kAlone, kTwin, kPaired };


template <typename T, int DP, Kind KIND, Share SHARE>
__global__ __launch_bounds__(SHARE == kPaired ? 512 : kAttThreads, SHARE != kPaired && DP * sizeof(T) < 256 ? 2 : 1)
void att_bwd_key_kernel(Att a) {
    constexpr int KG = SHARE == kTwin ? 2 : 4, QP = SHARE == kAlone ? 1 : 2;
    constexpr bool PAIRED = SHARE == kPaired;
    // fp32 results show the places that 1 / sum loses in the exponent from the first
    // score on: there it is a factor of its own
    constexpr bool kApart = sizeof(T) == 4;
    using L = Tile<T, DP>;
    constexpr int QT = BwdShape<T, DP>::KT, NB = QT / 32, HALF = QT * L::ROW;
    constexpr int KV = PAIRED ? 128 * L::ROW : 16;
    __shared__ __attribute__((aligned(1024))) char kv[2][KV];
    __shared__ __attribute__((aligned(1024))) char tiles0[2][HALF];
    __shared__ __attribute__((aligned(1024))) char tiles1[2][HALF];
    // log 2 of weight over score, maximum, 1 / sum (without a bias: what that log 2
    // leaves of it), delta, key end, document
    __shared__ __attribute__((aligned(256))) float info[2][6][QT];
    extern __shared__ float line[];
    const int l = threadIdx.x & 63, wave = wave_id(), g = l >> 5, kw = wave % KG;
    int bg, rest;
    place(blockIdx.x, a.B * a.Hk, bg, rest);
    const int b = bg / a.Hk, hk = bg - b * a.Hk, part = rest % a.parts, kb = rest / a.parts;
    const int n = filled_keys(a, b), off = n - a.Lq;
    const int j0 = kb * KG * 32 + kw * 32, j = j0 + (l & 31);
    const Cap cap = cap_of<T, KIND>(a, true);
    const int prefix = a.prefix ? a.prefix[b] : 0;
    const int doc = a.documents && j < n ? a.documents[static_cast<int64_t>(b) * a.Lk + j] : 0;

    using V = typename Eight<T>::V;
    V k[L::NS], v[L::NS];
#pragma unroll
    for (int s = 0; s < L::NS; ++s) k[s] = V{}, v[s] = V{};
    const bool second = PAIRED && wave >= 4;  // these waves load the tiles' second tensor
    if (PAIRED) {
        const int64_t stride = second ? a.vs[2] : a.ks[2];
        const T* base = second ? row_at<T>(a.v, a.vs, b, hk, 0) : row_at<T>(a.k, a.ks, b, hk, 0);
        Loader<T, DP, PAIRED ? 128 : QT, 4> lk;
        lk.init(threadIdx.x & 255, stride, a.D);
        lk.load(second ? kv[1] : kv[0], base, stride, kb * 128, n, a.D, kw);
    } else if (j < n) {
        load_row<T, DP>(k, row_at<T>(a.k, a.ks, b, hk, j), a.D, l);
        load_row<T, DP>(v, row_at<T>(a.v, a.vs, b, hk, j), a.D, l);
    }

    // Whether some row of these heads is far (kNear): asked for here, the first of
    // the answers looked at with the first rows' own values.
    bool far = false;
    constexpr int kAsk = 8;
    const int notes = kNotes<T, KIND> ? a.per * a.rblocks * kAttWaves : 0;
    const int* const note = a.far + static_cast<int64_t>(b * a.Hq + hk * a.per) * a.rblocks * kAttWaves;
    int noted[kAsk];
#pragma unroll
    for (int c = 0; c < kAsk; ++c) noted[c] = c * 64 + l < notes ? note[c * 64 + l] : 0;

    // the queries that see any of the block's keys: all of them, or those from
    // the first key's position on
    const int jb = kb * KG * 32;
    int t0 = 0, t1 = jb < n ? (a.Lq + QT - 1) / QT : 0;
    if (a.causal && jb >= prefix) t0 = max(0, jb - off) / QT;
    t0 = min(t0, t1);
    const int64_t units = static_cast<int64_t>(t1 - t0) * a.per;
    const int u0 = static_cast<int>(units * part / a.parts), u1 = static_cast<int>(units * (part + 1) / a.parts);
    int2 own = make_int2(0, 0);
    if (KIND == kGeneral && a.documents && jb < n) {
        const int e = jb / kRangeKeys;
        own = a.ranges[b * a.nranges + e];
        if (KG == 4 && e + 1 < a.nranges) {
            const int2 r = a.ranges[b * a.nranges + e + 1];
            own.x = min(own.x, r.x), own.y = max(own.y, r.y);
        }
    }
    // `t` counts the key block's units: a head's query tiles, then the next's
    auto wanted = [&](int u) {
        if (KIND != kGeneral || !a.documents) return true;
        if (u >= u1) return false;
        const int i0 = (t0 + u % (t1 - t0)) * QT;
        const int p0 = max(0, i0 + off), p1 = min(n, min(a.Lq, i0 + QT) + off) - 1;
        for (int e = p0 / kRangeKeys; p0 <= p1 && e <= p1 / kRangeKeys; ++e) {
            const int2 r = a.ranges[b * a.nranges + e];
            if (r.x <= own.y && own.x <= r.y) return true;
        }
        return false;
    };
    Needed<decltype(wanted)> need{wanted};

    Loader<T, DP, QT, 4, PAIRED> lq, lg;
    lq.init(threadIdx.x & 255, second ? a.gos[2] : a.qs[2], a.D);
    if (!PAIRED) lg.init(threadIdx.x, a.gos[2], a.D);
    // a unit's head and first row, kept up by addition
    struct Unit {
        int u, h, i0;
    };
    auto onward = [&](Unit x) {
        const int u = KIND == kGeneral && a.documents ? need.next(x.u + 1, u1) : x.u + 1;
        int64_t i0 = x.i0 + static_cast<int64_t>(u - x.u) * QT;
        if (u < u1)
            while (i0 >= static_cast<int64_t>(t1) * QT) i0 -= static_cast<int64_t>(t1 - t0) * QT, ++x.h;
        x.u = u, x.i0 = static_cast<int>(i0);
        return x;
    };
    auto load = [&](const Unit& x, char* tile) {
        const int h = x.h, i0 = x.i0;
        if (PAIRED) {
            const T* base = second ? row_at<T>(a.go, a.gos, b, h, 0) : row_at<T>(a.q, a.qs, b, h, 0);
            lq.load(tile + (second ? HALF : 0), base, second ? a.gos[2] : a.qs[2], i0, a.Lq, a.D, kw);
        } else {
            lq.load(tile, row_at<T>(a.q, a.qs, b, h, 0), a.qs[2], i0, a.Lq, a.D, wave);
            lg.load(tile + HALF, row_at<T>(a.go, a.gos, b, h, 0), a.gos[2], i0, a.Lq, a.D, wave);
        }
    };
    // row values of a unit, in registers until its tile is the next
    float2 r_stat{};
    float r_delta = 0.f;
    int r_lim = 0, r_doc = -1;
    auto fetch = [&](const Unit& y) {
        const int x = threadIdx.x;
        if (x >= QT) return;
        const int i = y.i0 + x;
        // a row past the end has a maximum that no bias comes near: exp2 of its scores is 0
        r_stat = make_float2(__FLT_MAX__, 0.f), r_delta = 0.f, r_lim = 0, r_doc = -1;
        if (i < a.Lq) {
            const int64_t at = (static_cast<int64_t>(b) * a.Hq + y.h) * a.Lq + i;
            const Row r = row_of(a, b, i, n, prefix);
            r_stat = get_stats(a, at), r_delta = a.delta[at], r_lim = r.lim;
            if (KIND == kGeneral) r_doc = r.doc;
        }
    };
    auto put = [&](int buf) {
        const int x = threadIdx.x;
        if (x >= QT) return;
        if (KIND == kGeneral) {
            info[buf][1][x] = r_stat.x, info[buf][2][x] = r_stat.y * kRoom<T>;
        } else {
            // 1 / sum joins the exponent; next to a large maximum that loses its last
            // places, and the weights take what it lost as a factor
            const float y = r_stat.y * kRoom<T>, up = __builtin_amdgcn_logf(y) - r_stat.x;
            info[buf][0][x] = kApart ? -r_stat.x : up + (KIND == kCapped ? cap.top : 0.f);
            if (kApart) info[buf][2][x] = y;
            if (far) info[buf][2][x] = y == 0.f ? y : y * __builtin_amdgcn_exp2f(-r_stat.x - up);
        }
        info[buf][3][x] = r_delta;
        info[buf][4][x] = __int_as_float(r_lim);
        if (KIND == kGeneral) info[buf][5][x] = __int_as_float(r_doc);
    };
    f32x16 dk[L::ND] = {}, dv[L::ND] = {};
    float by = kFitFirst / kRoom<T>;  // what dk's weights are times, besides kRoom
    Unit now{need.next(u0, u1), 0, 0};
    if (now.u < u1) now.h = hk * a.per + now.u / (t1 - t0), now.i0 = (t0 + now.u % (t1 - t0)) * QT;
    int staged = -1;
    Bias bs{0.f, line};
    // a wave's places in a tile (its half of one, if paired) and among the keys
    const int half = QP == 2 ? wave / KG * 32 : 0;
    const int by_row = L::row_base(half, l), by_col = L::col_base(half, l);
    const int key_off = (kw * 32 - half) * L::ROW;  // from a row's place to the keys'
    // one 32-row part of a tile, whatever it holds
    auto general = [&](const char* tile, int buf, int qb, int pf, bool whole) {
        const char* part = QP == 2 ? tile : tile + qb * 32 * L::ROW;
        const float* rows = &info[buf][0][qb * 32 + 4 * g];
        RowFragments<T, DP> fq, fg;
        fq.read(part, by_row), fg.read(part + HALF, by_row);
        order();
        const f32x16 xs = fq.products(k);
        f32x16 dp = fg.products(v);
        ColumnFragments<T, DP> cg, cq;
        if (DP <= 64) cg.read(part + HALF, by_col);
        settle<T>();
        const Scores y = cap_scores<true>(cap, xs);
        f32x16 s = add_bias<-1>(a, bs, j - pf - 4 * g, j0 - pf - 31, j0 + 31 - pf, y.s);
        if (!whole) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const i32x4 m = *reinterpret_cast<const i32x4*>(rows + 4 * QT + 8 * c);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * c + e] = j < m[e] ? s[4 * c + e] : -INFINITY;
            }
            if (a.documents) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const i32x4 d = *reinterpret_cast<const i32x4*>(rows + 5 * QT + 8 * c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[4 * c + e] = d[e] == doc ? s[4 * c + e] : -INFINITY;
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const f32x4 top = *reinterpret_cast<const f32x4*>(rows + QT + 8 * c);
            const f32x4 inv = *reinterpret_cast<const f32x4*>(rows + 2 * QT + 8 * c);
            const f32x4 del = *reinterpret_cast<const f32x4*>(rows + 3 * QT + 8 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * c + e;
                const float w = __builtin_amdgcn_exp2f(s[r] - top[e]) * inv[e];
                dp[r] = w * (dp[r] - del[e]);
                s[r] = w;
            }
        }
        if (cap.mode != 0) dp *= y.w;
        if (kNarrow<T>) dp *= by;
        if (!whole) {  // 0 times what an unseen pair holds is not always 0
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = s[r] == 0.f ? 0.f : dp[r];
        }
        order();
        if (DP > 64) cg.read(part + HALF, by_col);
        if (DP <= 64) cq.read(part, by_col);
        dp = fit<T>(by, dp, dk);
        cg.weigh(dv, s);
        if (DP > 64) cq.read(part, by_col);
        cq.weigh_fine(dk, dp);
        settle<T>();
    };
    // The weights p (in place of the products s) and dx, without a bias.
    struct RowInfo {
        f32x4 up[4], del[4], inv[kApart ? 4 : 1];
    };
    auto row_info = [&](int buf, int qb) {
        const float* rows = &info[buf][0][qb * 32 + 4 * g];
        RowInfo x;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            x.up[c] = *reinterpret_cast<const f32x4*>(rows + 8 * c);
            x.del[c] = *reinterpret_cast<const f32x4*>(rows + 3 * QT + 8 * c);
            if (kApart) x.inv[c] = *reinterpret_cast<const f32x4*>(rows + 2 * QT + 8 * c);
        }
        return x;
    };
    auto weights = [&](const RowInfo& x, f32x16& s, f32x16& dp) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if constexpr (KIND == kPlain) {
                s[r] = __builtin_amdgcn_exp2f(fma_acc(s[r], cap.c, x.up[r / 4][r % 4]));
                if constexpr (kApart) s[r] *= x.inv[r / 4][r % 4];
                dp[r] = s[r] * (dp[r] - x.del[r / 4][r % 4]);
                if constexpr (kNarrow<T>) dp[r] *= by;
            } else {
                const float q = quick_r(s[r], cap.k);
                s[r] = __builtin_amdgcn_exp2f(fma_acc(q, -2.f * cap.top, x.up[r / 4][r % 4]));
                dp[r] = s[r] * (dp[r] - x.del[r / 4][r % 4]) * ((kNarrow<T> ? 4.f * by : 4.f) * fma_acc(-q, q, q));
            }
        }
    };
    // Unseen pairs to 0, and far rows' weights to their last places.
    auto mend = [&](int buf, int qb, f32x16& s, f32x16& dp) {
        const float* rows = &info[buf][4][qb * 32 + 4 * g];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const i32x4 lim = *reinterpret_cast<const i32x4*>(rows + 8 * c);
            f32x4 fix = {1.f, 1.f, 1.f, 1.f};
            if (far) fix = *reinterpret_cast<const f32x4*>(rows - 2 * QT + 8 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * c + e;
                s[r] = j < lim[e] ? s[r] * fix[e] : 0.f, dp[r] = j < lim[e] ? dp[r] * fix[e] : 0.f;
            }
        }
    };
    auto simple = [&](const char* tile, int buf, int qb, bool whole) {
        const char* part = QP == 2 ? tile : tile + qb * 32 * L::ROW;
        RowFragments<T, DP> fq, fg;
        fq.read(part, by_row), fg.read(part + HALF, by_row);
        order();
        f32x16 s = fq.products(k), dp = fg.products(v);
        ColumnFragments<T, DP> cg, cq;
        cg.read(part + HALF, by_col);
        const RowInfo x = row_info(buf, qb);
        settle<T>();
        weights(x, s, dp);
        if (!whole) mend(buf, qb, s, dp);
        cq.read(part, by_col);
        dp = fit<T>(by, dp, dk);
        order();
        cg.weigh(dv, s);
        cq.weigh_fine(dk, dp);
        settle<T>();
    };
    auto paired = [&](const char* tile, int buf, int qb, bool whole) {
        // formed anew for each tile: kept, the reads' addresses would be spilled
        const int rows = here(by_row), cols = here(by_col), keys = rows + key_off;
        f32x16 s, dp;
        {
            RowFragments<T, DP> f, key;
            f.read(tile, rows), key.read(kv[0], keys);
            order();
            s = f.products(key.f);
        }
        {
            RowFragments<T, DP> f, key;
            f.read(tile + HALF, rows), key.read(kv[1], keys);
            order();
            dp = f.products(key.f);
        }
        settle<T>();
        weights(row_info(buf, qb), s, dp);
        ColumnFragments<T, DP> cg, cq;
        cg.read(tile + HALF, cols);
        if (!whole) mend(buf, qb, s, dp);
        cq.read(tile, cols);
        dp = fit<T>(by, dp, dk);
        order();
        cg.weigh(dv, s);
        cq.weigh_fine(dk, dp);
        settle<T>();
    };
    auto compute = [&](const char* tile, int buf) {
        const int i0 = now.i0, p0 = i0 + off;
        // the rows' key ends rise with their position
        auto ends = [&](int p) { return a.causal ? min(n, max(p + 1, prefix)) : n; };
        if constexpr (QP == 2) {
            const int qb = wave / KG, pf = p0 + qb * 32, count = min(a.Lq - i0 - qb * 32, 32);
            if (count <= 0 || j0 >= ends(pf + count - 1)) return;
            const bool whole = j0 + 32 <= ends(pf) && !(KIND == kGeneral && a.documents) && !far;
            if constexpr (KIND == kGeneral) general(tile, buf, qb, pf, whole);
            else if constexpr (PAIRED) paired(tile, buf, qb, whole);
            else simple(tile, buf, qb, whole);
        } else {
#pragma unroll 1
            for (int qb = 0; qb < NB; ++qb) {
                const int pf = p0 + qb * 32, count = min(a.Lq - i0 - qb * 32, 32);
                if (count <= 0) break;
                if (j0 >= ends(pf + count - 1)) continue;
                const bool whole = j0 + 32 <= ends(pf) && !(KIND == kGeneral && a.documents);
                if constexpr (KIND == kGeneral) general(tile, buf, qb, pf, whole);
                else simple(tile, buf, qb, whole);
            }
        }
    };
    auto step = [&](char* tile, char* ahead, int buf) {
        const Unit then = onward(now);
        if (KIND == kGeneral && (a.table || a.slopes) && now.h != staged) {
            staged = now.h;
            if (a.table) {
                __syncthreads();
                stage_line<T>(a, staged, line);
            }
            bs = lane_bias(a, staged, line);
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the tile has landed
        __syncthreads();
        if (then.u < u1) {
            fetch(then);
            load(then, ahead);
        }
        compute(tile, buf);
        if (then.u < u1) put(buf ^ 1);
        now = then;
    };
    if (now.u < u1) {
        fetch(now);
        load(now, tiles0[0]);
        if constexpr (kNotes<T, KIND>) {
            int any = 0;
#pragma unroll
            for (int c = 0; c < kAsk; ++c) any |= noted[c];
            for (int i = kAsk * 64 + l; i < notes; i += 64) any |= note[i];
            far = __any(any);
        }
        put(0);
    }
    while (now.u < u1) {
        step(tiles0[0], tiles1[0], 0);
        if (now.u < u1) step(tiles1[0], tiles0[0], 1);
    }
    if constexpr (kNarrow<T>) {
        const float back = 1.f / (by * kRoom<T>);
#pragma unroll
        for (int d = 0; d < L::ND; ++d) dk[d] *= back, dv[d] *= 1.f / kRoom<T>;
    }
    if constexpr (QP == 2) {  // the second waves' sums join the first's
        // a part without a unit (late keys of a causal call have few) has not waited
        // for its K and V, whose place the sums take
        if (PAIRED) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        float* const room = reinterpret_cast<float*>(PAIRED ? &kv[0][0] : &tiles0[0][0]);
        float* sums = room + (kw * DP + 4 * g) * 32 + (l & 31);  // [keys][column][key]
        static_assert((PAIRED ? sizeof(kv) : sizeof(tiles0)) >= KG * DP * 32 * 4, "the sums of dk take the tiles' place");
        auto join = [&](f32x16 (&acc)[L::ND]) {
            __syncthreads();
            if (wave >= KG) {
#pragma unroll
                for (int d = 0; d < L::ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sums[(d * 32 + el(r)) * 32] = acc[d][r];
            }
            __syncthreads();
            if (wave < KG) {
#pragma unroll
                for (int d = 0; d < L::ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] += sums[(d * 32 + el(r)) * 32];
            }
        };
        join(dk);
        join(dv);
        if (wave >= KG) return;
    }
    float bad = 0.f;
#pragma unroll
    for (int d = 0; d < L::ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dk[d][r] *= a.scale;
            bad = fma_acc(dk[d][r], 0.f, fma_acc(dv[d][r], 0.f, bad));
        }
    const bool live = j < a.Lk;
    if (a.parts > 1) {
        // [k, v][part][b, hk, j][D], added by the next launch
        if (!live) return;
        const int64_t rows = static_cast<int64_t>(a.B) * a.Hk * a.Lk, row = (static_cast<int64_t>(b) * a.Hk + hk) * a.Lk + j;
        float* pk = a.part + (static_cast<int64_t>(part) * rows + row) * a.D;
        float* pv = pk + a.parts * rows * a.D;
#pragma unroll
        for (int d = 0; d < L::ND; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int col = d * 32 + 8 * c + 4 * g;
                if (col >= a.D) continue;
                *reinterpret_cast<f32x4*>(pk + col) = f32x4{dk[d][4 * c], dk[d][4 * c + 1], dk[d][4 * c + 2], dk[d][4 * c + 3]};
                *reinterpret_cast<f32x4*>(pv + col) = f32x4{dv[d][4 * c], dv[d][4 * c + 1], dv[d][4 * c + 2], dv[d][4 * c + 3]};
            }
        return;
    }
    if (live) {
        T* ok = const_cast<T*>(row_at<T>(a.gk, a.gks, b, hk, j));
        T* ov = const_cast<T*>(row_at<T>(a.gv, a.gvs, b, hk, j));
#pragma unroll
        for (int d = 0; d < L::ND; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int col = d * 32 + 8 * c + 4 * g;
                if (col >= a.D) continue;
                store4<T>(ok + col, f32x4{dk[d][4 * c], dk[d][4 * c + 1], dk[d][4 * c + 2], dk[d][4 * c + 3]});
                store4<T>(ov + col, f32x4{dv[d][4 * c], dv[d][4 * c + 1], dv[d][4 * c + 2], dv[d][4 * c + 3]});
            }
    }
    unsigned long long rows = __ballot(bad != 0.f);
    rows = (rows | rows >> 32) & 0xffffffffull & __ballot(live);
#pragma unroll 1
    for (; rows; rows &= rows - 1) exact_key_gradient<T>(a, b, hk, j0 + __builtin_ctzll(rows));
}

// Adds the parts of dk and dv: one wave per key.
template <typename T>
__global__ __launch_bounds__(kAttThreads) void att_bwd_join_kernel(Att a) {
    const int64_t rows = static_cast<int64_t>(a.B) * a.Hk * a.Lk;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kAttWaves + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int l = threadIdx.x & 63;
    const int j = static_cast<int>(row % a.Lk), hk = static_cast<int>(row / a.Lk % a.Hk),
              b = static_cast<int>(row / a.Lk / a.Hk);
    // a lane takes four columns of dk (first half of the wave) or dv
    const int c = (l & 31) * 4;
    float bad = 0.f;
    if (c < a.D) {
        const float* p = a.part + ((l >> 5) * a.parts * rows + row) * a.D + c;
        f32x4 s = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 4
        for (int i = 1; i < a.parts; ++i) s += *reinterpret_cast<const f32x4*>(p + i * rows * a.D);
        bad = fma_acc(s[0], 0.f, fma_acc(s[1], 0.f, fma_acc(s[2], 0.f, s[3] * 0.f)));
        T* out = const_cast<T*>(l < 32 ? row_at<T>(a.gk, a.gks, b, hk, j) : row_at<T>(a.gv, a.gvs, b, hk, j));
        store4<T>(out + c, s);
    }
    if (__any(bad != 0.f)) exact_key_gradient<T>(a, b, hk, j);
}

template <typename T, int DP, Kind KIND>
static void backward_kind(const Att& a, hipStream_t st) {
    const unsigned line = a.table ? ((2 * a.reach + 4) & ~3) * 4 : 0;
    const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.rblocks;
    if (a.splits)
        att_bwd_row_kernel<T, DP, true, KIND><<<static_cast<unsigned>(rows), kAttThreads, attention_row_lds(a), st>>>(a);
    else
        att_bwd_row_kernel<T, DP, false, KIND><<<static_cast<unsigned>(rows), kAttThreads, attention_row_lds(a), st>>>(a);
    const int64_t keys = static_cast<int64_t>(a.B) * a.Hk * a.kblocks * a.parts;
    constexpr Share share = sizeof(T) == 4 ? kAlone : DP <= 64 ? kTwin : KIND != kGeneral ? kPaired : kAlone;
    static_assert((share == kTwin) == (key_block(sizeof(T), DP) == 64), "the cut agrees");
    att_bwd_key_kernel<T, DP, KIND, share>
        <<<static_cast<unsigned>(keys), share == kPaired ? 512 : kAttThreads, line, st>>>(a);
}

template <typename T, int DP>
static void backward_width(const Att& a, hipStream_t st) {
    const Kind kind = kind_of<T>(a);
    if constexpr (sizeof(T) == 2)  // fp32 has no quick cap
        if (kind == kCapped) return backward_kind<T, DP, kCapped>(a, st);
    if (kind == kPlain) backward_kind<T, DP, kPlain>(a, st);
    else backward_kind<T, DP, kGeneral>(a, st);
}

template <typename T>
int attention_backward_launch(const Att& a, hipStream_t st) {
    if (a.D <= 32) backward_width<T, 32>(a, st);
    else if (a.D <= 64) backward_width<T, 64>(a, st);
    else if (a.D <= 96) backward_width<T, 96>(a, st);
    else backward_width<T, 128>(a, st);
    if (int rc = nsh_host::check_launch("attention_backward")) return rc;
    if (a.parts > 1) {
        const int64_t rows = static_cast<int64_t>(a.B) * a.Hk * a.Lk;
        att_bwd_join_kernel<T><<<static_cast<unsigned>(nsh_host::ceil_div(rows, kAttWaves)), kAttThreads, 0, st>>>(a);
        if (int rc = nsh_host::check_launch("attention_backward_join")) return rc;
    }
    if (a.gtable) {
        constexpr int code = sizeof(T) == 4 ? NSH_DTYPE_FLOAT32 : __is_same(T, f16) ? NSH_DTYPE_FLOAT16 : NSH_DTYPE_BFLOAT16;
        return table_gradient(a.bins, a.buckets, a.Hq, static_cast<int64_t>(a.B) * a.rblocks * kAttWaves, a.num_buckets, a.reach,
                              code, a.gtable, st);
    }
    return NSH_OK;
}

}  // namespace nsh
