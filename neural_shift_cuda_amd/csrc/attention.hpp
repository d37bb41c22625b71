// attention.hpp -- what the attention kernels share: their arguments as the
// device takes them, how a call is cut into workgroups, and the exact row by
// row computation that stands behind the tiles.
#pragma once

#include "nsh_common.hpp"

namespace nsh {

constexpr int kAttThreads = 256;
constexpr int kAttWaves = 4;
constexpr int kRangeKeys = 64;  // keys of one document range
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;

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
    float* stats;  // of every row: maximum in units of log 2, 1 / sum of exp2(score - maximum)
    void* rest;    // (B, Hq, Lq, D): what out's rounding left
    const float* gdegree;
    int64_t gos[3], gqs[3], gks[3], gvs[3];
    void *gq, *gk, *gv, *gtable;
    int wide;  // fp32
    // the cut
    int pack;      // query heads whose rows stand side by side (1 or per)
    int rblocks;   // row blocks of a head group
    int splits;    // workgroups that share a row block's keys
    int kblocks;   // key blocks of the k and v gradients
    int parts;     // workgroups that share a key block's queries
    int nranges;   // document ranges of a batch
    const int2* ranges;
    float *part, *delta, *bins;
    int* far;      // by row block and wave of the gradients by rows: some row's weights need care
};

__device__ __forceinline__ int filled_keys(const Att& a, int b) {
    if (!a.lengths) return a.Lk;
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n > a.Lk ? a.Lk : n);
}

template <typename T>
__device__ __forceinline__ const T* row_at(const void* base, const int64_t (&s)[3], int b, int h,
                                           int i) {
    return static_cast<const T*>(base) + b * s[0] + h * s[1] + i * s[2];
}

// The gradients take delta = dO . out once for a whole row, so out's rounding
// would be an error that all of the row's pairs share: over the thousands of
// pairs of one bucket of the bias it adds up as their count, where the pairs'
// own roundings add up as its root.  A 16-bit forward that trains therefore
// leaves what the rounding took off beside out, 0 where that is no number.
// (4 x 12 heads, 1024 tokens, width 64, bf16: the table's gradient is off by
// 0.0032 without it, where its own rounding is 0.0017 to 0.0023; dq and dk of 4 heads,
// 1024 tokens, width 128, causal, by 0.00255 and with it by 0.00238.)
template <typename T>
__device__ __forceinline__ T* rest_at(const Att& a, int b, int h, int i) {
    return static_cast<T*>(a.rest) + ((static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i) * a.D;
}
template <typename T>
__device__ __forceinline__ float rounded_off(float y) {
    const float r = y - to_acc(from_acc<T>(y));
    return fabsf(r) < INFINITY ? r : 0.f;
}

// What a query row needs for its scores: its position, the end of the keys
// that order lets it see, its document.
struct Row {
    int p, lim, doc;
};

__device__ __forceinline__ Row row_of(const Att& a, int b, int i, int n, int prefix) {
    Row r;
    r.p = i + n - a.Lq;
    r.lim = a.causal ? min(n, max(r.p + 1, prefix)) : n;
    r.doc = 0;
    if (a.documents) {
        r.doc = r.p >= 0 && r.p < n ? a.documents[static_cast<int64_t>(b) * a.Lk + r.p] : -1;
        if (r.doc < 0) r.lim = 0;
    }
    return r;
}
__device__ __forceinline__ Row row_of(const Att& a, int b, int i, int n) {
    return row_of(a, b, i, n, a.prefix ? a.prefix[b] : 0);
}

__device__ __forceinline__ bool sees(const Att& a, const Row& r, int b, int j) {
    return j < r.lim && (!a.documents || a.documents[static_cast<int64_t>(b) * a.Lk + j] == r.doc);
}

// The table's value of a relative position, in units of log 2 (NaN for a
// bucket it lacks; the type's lowest value stays a number).
template <typename T>
__device__ __forceinline__ float table_value(const Att& a, int h, int rel) {
    rel = rel < -a.reach ? -a.reach : (rel > a.reach ? a.reach : rel);
    const int w = a.buckets[rel + a.reach];
    if (w < 0 || w >= a.num_buckets) return __builtin_nanf("");
    const float v = to_acc(static_cast<const T*>(a.table)[static_cast<int64_t>(w) * a.Hq + h]);
    const float y = v * kLog2e;
    return fabsf(v) <= __FLT_MAX__ && fabsf(y) > __FLT_MAX__ ? copysignf(__FLT_MAX__, v) : y;
}

// A row's maximum and sum as the two numbers that the gradients weigh pairs
// with, p = exp2(s - x) y, and its log degree.  The sum is kept apart: added to
// a maximum of 1e9 (a bias that stands for "never", in every place of a row) it
// would be lost.  A row that sees nothing weighs nothing.
__device__ __forceinline__ void put_stats(const Att& a, int64_t row, float m, float z) {
    if (a.stats) a.stats[2 * row] = z == 0.f ? 0.f : m, a.stats[2 * row + 1] = z == 0.f ? 0.f : 1.f / z;
    if (a.degree)
        a.degree[row] = z == 0.f ? -INFINITY : m == -__FLT_MAX__ ? m : kLn2 * (m + __builtin_amdgcn_logf(z));
}
__device__ __forceinline__ float2 get_stats(const Att& a, int64_t row) {
    if (a.stats) return make_float2(a.stats[2 * row], a.stats[2 * row + 1]);
    const float d = a.degree[row];
    return d == -INFINITY ? make_float2(0.f, 0.f) : make_float2(d * kLog2e, 1.f);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int k = 32; k; k >>= 1) v += __shfl_xor(v, k);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int k = 32; k; k >>= 1) v = fmaxf(v, __shfl_xor(v, k));
    return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int k = 32; k; k >>= 1) v = min(v, __shfl_xor(v, k));
    return v;
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int k = 32; k; k >>= 1) v = max(v, __shfl_xor(v, k));
    return v;
}

// ---------------------------------------------------------------------------
// One row by one wave, pair by pair: a pair that is not seen takes part in
// nothing.  The matrix products of the tiles give such a pair the weight 0,
// which is no help against an infinity or a NaN in the other factor, so a row
// whose tiles end in one of those is computed again here.  Data without them, and
// whose sums fp32 holds, never come this way (it takes some fifty times as long).
// ---------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ float pair_dot(const T* x, const T* y, int D) {
    float s = 0.f;
#pragma unroll 1
    for (int d = 0; d < D; ++d) s = fma_acc(to_acc(x[d]), to_acc(y[d]), s);
    return s;
}

// The biased score of a product in units of log 2, and the cap's derivative.
template <typename T>
__device__ __forceinline__ float pair_score(const Att& a, const Row& r, int h, int j, float x,
                                            float& slope) {
    x *= a.scale;
    slope = 1.f;
    if (a.cap > 0.f) {
        const float t = tanhf(x / a.cap);
        x = a.cap * t;
        slope = 1.f - t * t;
    }
    const int rel = j - r.p;
    x *= kLog2e;
    if (a.slopes) x -= a.slopes[h] * kLog2e * fabsf(static_cast<float>(rel));
    if (a.table) x += table_value<T>(a, h, rel);
    return x;
}

template <typename T>
__device__ __forceinline__ void exact_row(const Att& a, int b, int h, int i) {
    const int l = threadIdx.x & 63, n = filled_keys(a, b);
    const T* q = row_at<T>(a.q, a.qs, b, h, i);
    const Row r = row_of(a, b, i, n);
    float m = -INFINITY, z = 0.f, o[2] = {};
#pragma unroll 1
    for (int j0 = 0; j0 < r.lim; j0 += 64) {
        const int j = j0 + l;
        float s = -INFINITY, unused;
        if (sees(a, r, b, j))
            s = pair_score<T>(a, r, h, j, pair_dot(row_at<T>(a.k, a.ks, b, h / a.per, j), q, a.D), unused);
        const float top = fmaxf(wave_max(s), m);
        const bool see = s != -INFINITY;  // a score of -inf excludes the key
        const float e = see ? __builtin_amdgcn_exp2f(s - (top == -INFINITY ? 0.f : top)) : 0.f;
        const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        z = z * keep + wave_sum(e);
        m = top;
        unsigned long long seen = __ballot(see);
        o[0] *= keep, o[1] *= keep;
#pragma unroll 1
        for (; seen; seen &= seen - 1) {
            const int t = __builtin_ctzll(seen);
            const T* v = row_at<T>(a.v, a.vs, b, h / a.per, j0 + t);
            const float w = __shfl(e, t);
            for (int c = 0; c < 2; ++c)
                if (l + c * 64 < a.D) o[c] = fma_acc(w, to_acc(v[l + c * 64]), o[c]);
        }
    }
    const bool empty = m == -INFINITY && z == 0.f;
    T* out = const_cast<T*>(row_at<T>(a.out, a.os, b, h, i));
    for (int c = 0; c < 2; ++c)
        if (l + c * 64 < a.D) {
            const float y = empty ? 0.f : o[c] / z;
            out[l + c * 64] = from_acc<T>(y);
            if (a.rest) rest_at<T>(a, b, h, i)[l + c * 64] = from_acc<T>(rounded_off<T>(y));
        }
    if (l == 0) put_stats(a, (static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i, m, empty ? 0.f : z);
}

template <typename T>
__device__ __forceinline__ void exact_row_gradient(const Att& a, int b, int h, int i, float delta) {
    const int l = threadIdx.x & 63, n = filled_keys(a, b);
    const T* q = row_at<T>(a.q, a.qs, b, h, i);
    const T* go = row_at<T>(a.go, a.gos, b, h, i);
    const Row r = row_of(a, b, i, n);
    const float2 st = get_stats(a, (static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i);
    float g[2] = {};
#pragma unroll 1
    for (int j0 = 0; j0 < r.lim; j0 += 64) {
        const int j = j0 + l;
        float ds = 0.f, t;
        bool see = sees(a, r, b, j) && st.y != 0.f;
        if (see) {
            const float s = pair_score<T>(a, r, h, j, pair_dot(row_at<T>(a.k, a.ks, b, h / a.per, j), q, a.D), t);
            see = s != -INFINITY;
            if (see)
                ds = __builtin_amdgcn_exp2f(s - st.x) * st.y *
                     (pair_dot(row_at<T>(a.v, a.vs, b, h / a.per, j), go, a.D) - delta) * t * a.scale;
        }
        unsigned long long seen = __ballot(see);
#pragma unroll 1
        for (; seen; seen &= seen - 1) {
            const int u = __builtin_ctzll(seen);
            const T* k = row_at<T>(a.k, a.ks, b, h / a.per, j0 + u);
            const float w = __shfl(ds, u);
            for (int c = 0; c < 2; ++c)
                if (l + c * 64 < a.D) g[c] = fma_acc(w, to_acc(k[l + c * 64]), g[c]);
        }
    }
    T* gq = const_cast<T*>(row_at<T>(a.gq, a.gqs, b, h, i));
    for (int c = 0; c < 2; ++c)
        if (l + c * 64 < a.D) gq[l + c * 64] = from_acc<T>(g[c]);
}

template <typename T>
__device__ __forceinline__ void exact_key_gradient(const Att& a, int b, int hk, int j) {
    const int l = threadIdx.x & 63, n = filled_keys(a, b);
    const T* k = row_at<T>(a.k, a.ks, b, hk, j);
    const T* v = row_at<T>(a.v, a.vs, b, hk, j);
    float gk[2] = {}, gv[2] = {};
#pragma unroll 1
    for (int h = hk * a.per; h < (hk + 1) * a.per; ++h)
#pragma unroll 1
        for (int i0 = 0; i0 < a.Lq; i0 += 64) {
            const int i = i0 + l;
            float p = 0.f, ds = 0.f, t;
            bool see = false;
            if (i < a.Lq) {
                const Row r = row_of(a, b, i, n);
                const int64_t at = (static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i;
                const float2 st = get_stats(a, at);
                see = sees(a, r, b, j) && st.y != 0.f;
                if (see) {
                    const float s = pair_score<T>(a, r, h, j, pair_dot(row_at<T>(a.q, a.qs, b, h, i), k, a.D), t);
                    see = s != -INFINITY;
                    if (see) {
                        p = __builtin_amdgcn_exp2f(s - st.x) * st.y;
                        ds = p * (pair_dot(row_at<T>(a.go, a.gos, b, h, i), v, a.D) - a.delta[at]) * t * a.scale;
                    }
                }
            }
            unsigned long long seen = __ballot(see);
#pragma unroll 1
            for (; seen; seen &= seen - 1) {
                const int u = __builtin_ctzll(seen);
                const T* q = row_at<T>(a.q, a.qs, b, h, i0 + u);
                const T* go = row_at<T>(a.go, a.gos, b, h, i0 + u);
                const float w = __shfl(ds, u), x = __shfl(p, u);
                for (int c = 0; c < 2; ++c)
                    if (l + c * 64 < a.D) {
                        gk[c] = fma_acc(w, to_acc(q[l + c * 64]), gk[c]);
                        gv[c] = fma_acc(x, to_acc(go[l + c * 64]), gv[c]);
                    }
            }
        }
    T* ok = const_cast<T*>(row_at<T>(a.gk, a.gks, b, hk, j));
    T* ov = const_cast<T*>(row_at<T>(a.gv, a.gvs, b, hk, j));
    for (int c = 0; c < 2; ++c)
        if (l + c * 64 < a.D) ok[l + c * 64] = from_acc<T>(gk[c]), ov[l + c * 64] = from_acc<T>(gv[c]);
}

// cap * tanh(x |scale| / cap) is 1 - 2 / (1 + exp) in three cheap steps, off by
// some 2^-22 of the cap; with fp32 results, or a cap above 256 (2^-14, where a
// 16-bit weight's half step is 2^-12), small arguments take the series.
constexpr float kQuickCap = 256.f;

// Keys of a workgroup of the gradients by keys.  16-bit heads up to 64 wide take
// 64, two waves to a group of 32 keys, each with one half of a query tile: rows
// of 2500 tokens in documents, 2 x 12 heads, fp16, 57 us as the rule was set (59 now),
// and 76 with 128 keys, one wave to each 32.
constexpr int key_block(int bytes, int D) { return bytes == 2 && D <= 64 ? 64 : 128; }

// Launches of one type's kernels (attention_fwd_*.hip, attention_bwd_*.hip).
template <typename T> int attention_forward_launch(const Att& a, hipStream_t st);
template <typename T> int attention_backward_launch(const Att& a, hipStream_t st);

// LDS of the row gradients whose waves split the keys: their tiles, and for a
// bias table its line and the lined-up diagonals.
constexpr int kDiagonal = 36;  // places of a diagonal, with room against bank conflicts
constexpr int kDiagonals = 63 * kDiagonal;
inline int attention_row_lds(const Att& a) {
    return (a.table ? ((2 * a.reach + 4) & ~3) * 4 : 0) + (a.gtable ? kAttWaves * kDiagonals * 4 : 0);
}
inline bool attention_split_fits(const Att& a) {
    const int row = (a.D + 31) / 32 * 32 * (a.wide ? 4 : 2), buffers = row > 256 ? 1 : 2;
    return kAttWaves * (buffers * 64 * row + 512) + attention_row_lds(a) <= 160 * 1024;
}

}  // namespace nsh
