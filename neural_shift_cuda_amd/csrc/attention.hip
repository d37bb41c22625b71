// attention.hip -- attention over tokens with capped scores, distance biases
// and masks, forward and backward.
//
// One wave owns one query row (forward, gradient of q) or one key row
// (gradients of k and v) and walks the other side 64 rows at a time: a lane
// forms one pair's score, then the lanes turn to the columns.
#include <cmath>

#include "attention.hpp"

namespace nsh {

constexpr int kAttLanes = 64;
constexpr int kAttCols = 2;  // columns of a row per lane: D <= 128

struct Row {  // what a query row needs for its scores
    int p, n, prefix, doc;
    float slope;
};

__device__ __forceinline__ Row row_of(const Att& a, int b, int h, int i) {
    Row r;
    r.n = filled_keys(a, b);
    r.p = i + r.n - a.Lq;
    r.prefix = a.prefix ? a.prefix[b] : 0;
    r.slope = a.slopes ? a.slopes[h] : 0.f;
    r.doc = a.documents && r.p >= 0 ? a.documents[static_cast<int64_t>(b) * a.Lk + r.p] : -1;
    return r;
}

__device__ __forceinline__ bool sees(const Att& a, const Row& r, int b, int j) {
    if (j >= r.n) return false;
    if (a.causal && j > r.p && j >= r.prefix) return false;
    if (a.documents && (r.doc < 0 || a.documents[static_cast<int64_t>(b) * a.Lk + j] != r.doc))
        return false;
    return true;
}

__device__ __forceinline__ int bucket_of(const Att& a, int rel) {
    rel = rel < -a.reach ? -a.reach : (rel > a.reach ? a.reach : rel);
    return a.buckets[rel + a.reach];
}

// The biased score of a product, and the cap's derivative.
template <typename T>
__device__ __forceinline__ float score(const Att& a, const Row& r, int h, int j, float x,
                                       float& slope) {
    x *= a.scale;
    slope = 1.f;
    if (a.cap > 0.f) {
        const float t = tanhf(x / a.cap);
        x = a.cap * t;
        slope = 1.f - t * t;
    }
    const int rel = j - r.p;
    if (a.slopes) x -= r.slope * static_cast<float>(rel < 0 ? -rel : rel);
    if (a.table) {
        const int w = bucket_of(a, rel);
        x += w >= 0 && w < a.num_buckets
                 ? to_acc(static_cast<const T*>(a.table)[static_cast<int64_t>(w) * a.Hq + h])
                 : __builtin_nanf("");
    }
    return x;
}

template <typename T>
__device__ __forceinline__ const T* row_at(const void* base, const int64_t (&s)[3], int b, int h,
                                           int i) {
    return static_cast<const T*>(base) + b * s[0] + h * s[1] + i * s[2];
}

template <typename T>
__device__ __forceinline__ float dot(const T* x, const float* y, int D) {
    float s = 0.f;
    for (int d = 0; d < D; ++d) s = fma_acc(to_acc(x[d]), y[d], s);
    return s;
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

template <typename T>
__global__ __launch_bounds__(kAttLanes) void att_fwd_kernel(Att a) {
    __shared__ float qrow[128], prob[kAttLanes];
    const int64_t row = blockIdx.x;
    const int i = static_cast<int>(row % a.Lq), h = static_cast<int>(row / a.Lq % a.Hq),
              b = static_cast<int>(row / a.Lq / a.Hq), l = threadIdx.x;
    const T* q = row_at<T>(a.q, a.qs, b, h, i);
    for (int d = l; d < a.D; d += kAttLanes) qrow[d] = to_acc(q[d]);
    __syncthreads();
    const Row r = row_of(a, b, h, i);
    float m = -INFINITY, z = 0.f, o[kAttCols] = {};
    for (int j0 = 0; j0 < r.n; j0 += kAttLanes) {
        const int j = j0 + l;
        const bool see = sees(a, r, b, j);
        float s = -INFINITY, unused;
        if (see) s = score<T>(a, r, h, j, dot(row_at<T>(a.k, a.ks, b, h / a.per, j), qrow, a.D), unused);
        float top = wave_max(s);
        top = fmaxf(top, m);
        // a NaN score stays one; a row with nothing seen yet keeps its -inf
        const float e = see ? __expf(s - (top == -INFINITY ? 0.f : top)) : 0.f;
        const float keep = m == -INFINITY ? 0.f : __expf(m - top);
        z = z * keep + wave_sum(e);
        m = top;
        prob[l] = e;
        __syncthreads();
        const unsigned long long seen = __ballot(see);
        for (int c = 0; c < kAttCols; ++c) {
            const int d = l + c * kAttLanes;
            if (d >= a.D) break;
            o[c] *= keep;
            for (int t = 0; t < kAttLanes; ++t)
                if (seen >> t & 1)
                    o[c] = fma_acc(prob[t], to_acc(row_at<T>(a.v, a.vs, b, h / a.per, j0 + t)[d]), o[c]);
        }
        __syncthreads();
    }
    const bool empty = m == -INFINITY && z == 0.f;
    T* out = const_cast<T*>(row_at<T>(a.out, a.os, b, h, i));
    for (int c = 0; c < kAttCols; ++c) {
        const int d = l + c * kAttLanes;
        if (d < a.D) out[d] = from_acc<T>(empty ? 0.f : o[c] / z);
    }
    if (a.degree && l == 0) a.degree[row] = empty ? -INFINITY : m + __logf(z);
}

// One wave per query row: gradient of q, and the row's share of the table's.
template <typename T>
__global__ __launch_bounds__(kAttLanes) void att_bwd_q_kernel(Att a, float* delta, float* rows) {
    __shared__ float qrow[128], gorow[128], ds[kAttLanes];
    const int64_t row = blockIdx.x;
    const int i = static_cast<int>(row % a.Lq), h = static_cast<int>(row / a.Lq % a.Hq),
              b = static_cast<int>(row / a.Lq / a.Hq), l = threadIdx.x;
    const T* q = row_at<T>(a.q, a.qs, b, h, i);
    const T* go = row_at<T>(a.go, a.gos, b, h, i);
    const T* out = row_at<T>(a.out, a.os, b, h, i);
    float dl = 0.f;
    for (int d = l; d < a.D; d += kAttLanes) {
        qrow[d] = to_acc(q[d]);
        gorow[d] = to_acc(go[d]);
        dl += gorow[d] * to_acc(out[d]);
    }
    __syncthreads();
    dl = wave_sum(dl) - (a.gdegree ? a.gdegree[row] : 0.f);
    if (l == 0) delta[row] = dl;
    const Row r = row_of(a, b, h, i);
    const float degree = a.degree[row];
    float g[kAttCols] = {};
    for (int j0 = 0; j0 < r.n; j0 += kAttLanes) {
        const int j = j0 + l;
        const bool see = sees(a, r, b, j) && degree != -INFINITY;
        float x = 0.f, t = 0.f;
        if (see) {
            const float s = score<T>(a, r, h, j, dot(row_at<T>(a.k, a.ks, b, h / a.per, j), qrow, a.D), t);
            x = __expf(s - degree) * (dot(row_at<T>(a.v, a.vs, b, h / a.per, j), gorow, a.D) - dl);
        }
        if (rows && j < r.n) rows[(row * a.Lk) + j] = x;
        ds[l] = x * t * a.scale;
        __syncthreads();
        const unsigned long long seen = __ballot(see);
        for (int c = 0; c < kAttCols; ++c) {
            const int d = l + c * kAttLanes;
            if (d >= a.D) break;
            for (int u = 0; u < kAttLanes; ++u)
                if (seen >> u & 1)
                    g[c] = fma_acc(ds[u], to_acc(row_at<T>(a.k, a.ks, b, h / a.per, j0 + u)[d]), g[c]);
        }
        __syncthreads();
    }
    T* gq = const_cast<T*>(row_at<T>(a.gq, a.gqs, b, h, i));
    for (int c = 0; c < kAttCols; ++c) {
        const int d = l + c * kAttLanes;
        if (d < a.D) gq[d] = from_acc<T>(g[c]);
    }
}

// One wave per key row and key head: gradients of k and v.
template <typename T>
__global__ __launch_bounds__(kAttLanes) void att_bwd_kv_kernel(Att a, const float* delta) {
    __shared__ float krow[128], vrow[128], ds[kAttLanes], ps[kAttLanes];
    const int64_t row = blockIdx.x;
    const int j = static_cast<int>(row % a.Lk), hk = static_cast<int>(row / a.Lk % a.Hk),
              b = static_cast<int>(row / a.Lk / a.Hk), l = threadIdx.x;
    const T* k = row_at<T>(a.k, a.ks, b, hk, j);
    const T* v = row_at<T>(a.v, a.vs, b, hk, j);
    for (int d = l; d < a.D; d += kAttLanes) krow[d] = to_acc(k[d]), vrow[d] = to_acc(v[d]);
    __syncthreads();
    float gk[kAttCols] = {}, gv[kAttCols] = {};
    for (int h = hk * a.per; h < (hk + 1) * a.per; ++h)
        for (int i0 = 0; i0 < a.Lq; i0 += kAttLanes) {
            const int i = i0 + l;
            bool see = false;
            float p = 0.f, x = 0.f, t = 0.f;
            if (i < a.Lq) {
                const Row r = row_of(a, b, h, i);
                const int64_t at = (static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i;
                see = sees(a, r, b, j) && a.degree[at] != -INFINITY;
                if (see) {
                    const float s = score<T>(a, r, h, j, dot(row_at<T>(a.q, a.qs, b, h, i), krow, a.D), t);
                    p = __expf(s - a.degree[at]);
                    x = p * (dot(row_at<T>(a.go, a.gos, b, h, i), vrow, a.D) - delta[at]);
                }
            }
            ds[l] = x * t * a.scale;
            ps[l] = p;
            __syncthreads();
            const unsigned long long seen = __ballot(see);
            for (int c = 0; c < kAttCols; ++c) {
                const int d = l + c * kAttLanes;
                if (d >= a.D) break;
                for (int u = 0; u < kAttLanes; ++u)
                    if (seen >> u & 1) {
                        gk[c] = fma_acc(ds[u], to_acc(row_at<T>(a.q, a.qs, b, h, i0 + u)[d]), gk[c]);
                        gv[c] = fma_acc(ps[u], to_acc(row_at<T>(a.go, a.gos, b, h, i0 + u)[d]), gv[c]);
                    }
            }
            __syncthreads();
        }
    T* ok = const_cast<T*>(row_at<T>(a.gk, a.gks, b, hk, j));
    T* ov = const_cast<T*>(row_at<T>(a.gv, a.gvs, b, hk, j));
    for (int c = 0; c < kAttCols; ++c) {
        const int d = l + c * kAttLanes;
        if (d < a.D) ok[d] = from_acc<T>(gk[c]), ov[d] = from_acc<T>(gv[c]);
    }
}

// One workgroup per bucket and head: the table's gradient from the rows.
template <typename T>
__global__ __launch_bounds__(256) void att_bwd_table_kernel(Att a, const float* rows) {
    __shared__ float part[256];
    const int w = blockIdx.x, h = blockIdx.y;
    float s = 0.f;
    for (int b = 0; b < a.B; ++b) {
        const int n = filled_keys(a, b);
        for (int i = 0; i < a.Lq; ++i) {
            const float* at = rows + ((static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i) * a.Lk;
            for (int j = threadIdx.x; j < n; j += 256)
                if (bucket_of(a, j - (i + n - a.Lq)) == w) s += at[j];
        }
    }
    part[threadIdx.x] = s;
    __syncthreads();
    for (int k = 128; k; k >>= 1) {
        if (static_cast<int>(threadIdx.x) < k) part[threadIdx.x] += part[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0)
        static_cast<T*>(a.gtable)[static_cast<int64_t>(w) * a.Hq + h] = from_acc<T>(part[0]);
}

}  // namespace nsh

using nsh_host::check_launch;
using nsh_host::fail;

static bool rows_aligned(const void* p, const int64_t (&s)[3], int64_t bytes) {
    return nsh_host::aligned(p, 16) && s[0] * bytes % 16 == 0 && s[1] * bytes % 16 == 0 &&
           s[2] * bytes % 16 == 0;
}

static void take(int64_t (&to)[3], const int64_t (&from)[3]) {
    for (int i = 0; i < 3; ++i) to[i] = from[i];
}

static int attention_check(const char* op, const nsh_attention_args* g, nsh::Att* a) {
    if (!g) return fail(NSH_ERR_INVALID, "%s: null arguments", op);
    if (g->dtype < NSH_DTYPE_FLOAT16 || g->dtype > NSH_DTYPE_FLOAT32)
        return fail(NSH_ERR_INVALID, "%s: unsupported dtype code %d", op, g->dtype);
    constexpr int64_t kMost = int64_t(1) << 30;
    if (g->B < 1 || g->Hq < 1 || g->Hk < 1 || g->Lq < 1 || g->Lk < 1)
        return fail(NSH_ERR_INVALID, "%s: empty tensor", op);
    if (g->B > kMost || g->Hq > kMost || g->Lq > kMost || g->Lk > kMost ||
        g->B * g->Hq > kMost || g->B * g->Hq * g->Lq > 2 * kMost - 1 ||
        g->B * g->Hk * g->Lk > 2 * kMost - 1)
        return fail(NSH_ERR_INVALID, "%s: a size exceeds 2^30", op);
    if (g->Hq % g->Hk) return fail(NSH_ERR_INVALID, "%s: query heads must be a multiple of key heads", op);
    if (g->D < 8 || g->D > 128 || g->D % 8)
        return fail(NSH_ERR_INVALID, "%s: the head width must be a multiple of 8 up to 128", op);
    if (!(g->cap >= 0.0) || !std::isfinite(g->cap) || !std::isfinite(g->scale))
        return fail(NSH_ERR_INVALID, "%s: scale and cap must be finite, cap not negative", op);
    if (g->prefix && !g->causal) return fail(NSH_ERR_INVALID, "%s: a prefix needs causal", op);
    if (g->bias_table &&
        (!g->buckets || g->reach < 0 || g->reach > 2048 || g->num_buckets < 1 || g->num_buckets > 4097))
        return fail(NSH_ERR_INVALID, "%s: a bias table needs buckets, reach <= 2048 and 1..4097 buckets", op);
    if (!g->q || !g->k || !g->v || !g->out) return fail(NSH_ERR_INVALID, "%s: null pointer argument", op);
    const int64_t bytes = g->dtype == NSH_DTYPE_FLOAT32 ? 4 : 2;
    if (!rows_aligned(g->q, g->q_stride, bytes) || !rows_aligned(g->k, g->k_stride, bytes) ||
        !rows_aligned(g->v, g->v_stride, bytes) || !rows_aligned(g->out, g->out_stride, bytes))
        return fail(NSH_ERR_INVALID, "%s: rows must start on 16 bytes", op);
    *a = nsh::Att{};
    a->q = g->q, a->k = g->k, a->v = g->v;
    a->B = static_cast<int>(g->B), a->Hq = static_cast<int>(g->Hq), a->Hk = static_cast<int>(g->Hk);
    a->Lq = static_cast<int>(g->Lq), a->Lk = static_cast<int>(g->Lk), a->D = static_cast<int>(g->D);
    a->per = a->Hq / a->Hk;
    take(a->qs, g->q_stride), take(a->ks, g->k_stride), take(a->vs, g->v_stride), take(a->os, g->out_stride);
    a->lengths = g->lengths, a->prefix = g->prefix, a->documents = g->documents;
    a->slopes = g->slopes, a->table = g->bias_table, a->buckets = g->buckets;
    a->num_buckets = static_cast<int>(g->num_buckets), a->reach = static_cast<int>(g->reach);
    a->scale = static_cast<float>(g->scale), a->cap = static_cast<float>(g->cap);
    a->causal = g->causal != 0;
    a->out = g->out, a->degree = g->log_degree;
    return NSH_OK;
}

static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

extern "C" int64_t nsh_attention_workspace_bytes(const nsh_attention_args* g, int backward) {
    if (!g || g->B < 1 || g->Hq < 1 || g->Lq < 1 || g->Lk < 1) return -1;
    if (!backward) return 0;
    const int64_t rows = g->B * g->Hq * g->Lq;
    return up256(rows * 4) + (g->bias_table ? rows * g->Lk * 4 : 0);
}

#define NSH_ATT_TYPES(...)                                          \
    switch (g->dtype) {                                            \
        case NSH_DTYPE_FLOAT16: { using T = nsh::f16; __VA_ARGS__ } break;   \
        case NSH_DTYPE_BFLOAT16: { using T = nsh::bf16; __VA_ARGS__ } break; \
        default: { using T = float; __VA_ARGS__ } break;                  \
    }

extern "C" int nsh_attention_forward(const nsh_attention_args* g, void* stream) {
    nsh::Att a;
    if (int rc = attention_check("attention_forward", g, &a)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(g->B * g->Hq * g->Lq);
    NSH_ATT_TYPES(nsh::att_fwd_kernel<T><<<grid, nsh::kAttLanes, 0, st>>>(a);)
    return check_launch("attention_forward");
}

extern "C" int nsh_attention_backward(const nsh_attention_args* g, void* stream) {
    nsh::Att a;
    if (int rc = attention_check("attention_backward", g, &a)) return rc;
    if (!g->log_degree || !g->grad_out || !g->grad_q || !g->grad_k || !g->grad_v ||
        (g->grad_bias_table && !g->bias_table))
        return fail(NSH_ERR_INVALID, "attention_backward: null pointer argument");
    const int64_t bytes = g->dtype == NSH_DTYPE_FLOAT32 ? 4 : 2;
    if (!rows_aligned(g->grad_out, g->go_stride, bytes) || !rows_aligned(g->grad_q, g->gq_stride, bytes) ||
        !rows_aligned(g->grad_k, g->gk_stride, bytes) || !rows_aligned(g->grad_v, g->gv_stride, bytes))
        return fail(NSH_ERR_INVALID, "attention_backward: rows must start on 16 bytes");
    if (!g->workspace || g->workspace_bytes < nsh_attention_workspace_bytes(g, 1))
        return fail(NSH_ERR_INVALID, "attention_backward: workspace smaller than nsh_attention_workspace_bytes");
    a.go = g->grad_out, a.gdegree = g->grad_log_degree;
    take(a.gos, g->go_stride), take(a.gqs, g->gq_stride), take(a.gks, g->gk_stride), take(a.gvs, g->gv_stride);
    a.gq = g->grad_q, a.gk = g->grad_k, a.gv = g->grad_v, a.gtable = g->grad_bias_table;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t nq = g->B * g->Hq * g->Lq, nk = g->B * g->Hk * g->Lk;
    float* delta = static_cast<float*>(g->workspace);
    float* rows = a.gtable ? delta + up256(nq * 4) / 4 : nullptr;
    NSH_ATT_TYPES(
        nsh::att_bwd_q_kernel<T><<<static_cast<unsigned>(nq), nsh::kAttLanes, 0, st>>>(a, delta, rows);
        nsh::att_bwd_kv_kernel<T><<<static_cast<unsigned>(nk), nsh::kAttLanes, 0, st>>>(a, delta);
        if (rows)
            nsh::att_bwd_table_kernel<T><<<dim3(a.num_buckets, a.Hq), 256, 0, st>>>(a, rows);)
    return check_launch("attention_backward");
}
