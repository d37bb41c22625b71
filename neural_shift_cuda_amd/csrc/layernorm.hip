// layernorm.hip -- layer norm of rows, alone or of their sum with a residual
// stream, and its gradients, on gfx950.
//
//   s = x + residual (rounded to the type, and written)     h = (s - mean) / sqrt(var + eps)
//   y = h w + b
//   g' = gy w,  gx = gs + (g' - mean(g') - h mean(g' h)) / sqrt(var + eps)
//   gw = sum gy h,  gb = sum gy
//
// HBM streams: every input is read and every output written once.  A row belongs
// to a group of lanes that holds it whole in registers, 16 bytes a lane and part:
// up to 64 lanes of a wave, then a workgroup of 256 or 512.  So mean and variance
// are two sums over the same registers, the variance about the mean (as a
// difference of squares it would lose what the mean is larger than the deviations).
// Rows wider than a workgroup holds are read again for each sum.  Bound by memory: 16384 x
// 2048 bf16 with a residual, forward 268 MB in 45.5 us (5.9 TB/s), backward as much in 44.5;
// 3000 x 16384 fp16 forward 197 MB in 39 (5.0), backward 295 in 64 (4.6: a CU's registers hold
// one workgroup, whose loads and sums overlap by one row).
//
// gw and gb: a lane adds up its own columns over the rows that its group walks, the
// groups of a workgroup add in order, and a second launch adds the workgroups'
// sums in order (512 of them, 2048 columns: 4 us; 256, 16384 columns: 7.5).
#include <algorithm>
#include <cmath>

#include "rows.hpp"

namespace nsh {

struct LayerNormArgs {
    const void *x, *residual, *weight, *bias, *grad_y, *grad_s;
    int64_t x_stride, residual_stride, gy_stride, gs_stride;
    void *y, *s, *gx, *gw, *gb;
    float* stats;    // (rows, 2): mean and 1 / sqrt(var + eps), or NULL
    float* partial;  // (blocks, 2, N)
    int64_t rows;
    int n, blocks;
    float eps, inv_n;
};

// Groups of G lanes; several waves meet through LDS, `turn` telling two sums in a
// row apart.
template <int G>
struct Group {
    static constexpr int kThreads = G > 64 ? G : 256;
    static constexpr int kGroups = kThreads / G;
    static constexpr int kWaves = G > 64 ? G / 64 : 1;
    float* lds;  // 2 turns of two values a wave
    int turn = 0;

    __device__ __forceinline__ void sum(float& a, float& b) {
        a = lanes_sum<(G < 64 ? G : 64)>(a);
        b = lanes_sum<(G < 64 ? G : 64)>(b);
        if constexpr (kWaves > 1) {
            float* at = lds + turn * 2 * kWaves;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) {
                at[threadIdx.x / 64] = a;
                at[kWaves + threadIdx.x / 64] = b;
            }
            lds_barrier();
            a = b = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) a += at[w], b += at[kWaves + w];
        }
    }
    __device__ __forceinline__ float sum(float a) {
        float b = 0.f;
        if constexpr (kWaves > 1) {
            sum(a, b);
        } else {
            a = lanes_sum<G>(a);
        }
        return a;
    }
};

// sum / n: times 1 / n, and what that leaves.  (The product alone would be rounded only
// together with what it is taken from, and be off by 1 / n's rounding.)  So the deviations of a
// row of one value are all the same, and whole steps of the value's last place, their sums are
// exact, and what is left of them and of the variance is 0.
__device__ __forceinline__ float mean_of(float sum, const LayerNormArgs& a) {
    const float mean = sum * a.inv_n;
    return fma_acc(fma_acc(-mean, static_cast<float>(a.n), sum), a.inv_n, mean);
}

// 1 / sqrt(v).  The instruction takes subnormal numbers for 0: rows of 1e-20 would be infinite.
__device__ __forceinline__ float root_below(float v) {
    const bool small = v < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p100f : v);
    return small ? r * 0x1p50f : r;
}

// Of a row's deviations from its mean as first summed: 1 / sqrt(var + eps), and their own
// mean, what that sum's rounding left (rows of one value would otherwise come out as its
// last place over sqrt(eps)).
template <typename Gr>
__device__ __forceinline__ float variance(Gr& group, float square, float off, const LayerNormArgs& a, float& by) {
    group.sum(square, off);
    const float rest = mean_of(off, a);
    float var = square * a.inv_n;
    // (squares beyond fp32 leave infinity, and a row of zeros, as the formula does)
    if (var < INFINITY) var = mean_of(square, a) - rest * rest;
    // (the difference may round below 0; what is no number stays so)
    by = root_below((var < 0.f ? 0.f : var) + a.eps);
    return rest;
}

// Whole vectors need nothing but a mask, which keeps registers free where no row is loaded
// ahead (16384 x 2048 bf16, forward: 46 us, 52 by kNear); others (backward, by elements and
// by kNear: 16384 x 2047 bf16 65 and 42 us, 16384 x 333 25 and 13).
constexpr Reach reach_of(int lanes, bool ahead, bool whole) {
    return whole && !ahead ? kMasked : lanes == 8 ? kShort : kNear;
}

template <typename T, int G, int NV, bool WHOLE>
__global__ __launch_bounds__(Group<G>::kThreads) void layer_norm_forward_kernel(LayerNormArgs a) {
    using Gr = Group<G>;
    constexpr int V = kVec<T>;
    __shared__ float meet[Gr::kWaves > 1 ? 4 * Gr::kWaves : 1];
    Gr group{meet};
    // Groups of a wave keep the weights for all their rows; a workgroup of 256 has one row, and
    // reads them at its end: registers for more workgroups at once instead.  One of 512 walks
    // rows, and has the next one's loads under way (3000 x 16384 fp16: 48 us with a row each, 38
    // so).
    constexpr bool AHEAD = G == 512, KEEP = G <= 64 || AHEAD;
    constexpr Reach REACH = reach_of(G, AHEAD, WHOLE);
    const int lane = threadIdx.x % G, own = threadIdx.x / G;
    ux4 w[KEEP ? NV : 1], b[KEEP ? NV : 1];
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            if (a.weight) w[i] = load_near<T, REACH>(static_cast<const T*>(a.weight), c, a.n);
            if (a.bias) b[i] = load_near<T, REACH>(static_cast<const T*>(a.bias), c, a.n);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            if (a.weight) in_place<T, REACH, WHOLE>(w[i], c, a.n);
            if (a.bias) in_place<T, REACH, WHOLE>(b[i], c, a.n);
        }
    }
    struct Row {
        ux4 x[NV], more[NV];
    };
    const int64_t step = static_cast<int64_t>(a.blocks) * Gr::kGroups;
    auto fetch = [&](int64_t r0, Row& f) {
        const int64_t row = r0 + own < a.rows ? r0 + own : 0;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) f.x[i] = load_near<T, REACH>(x, (i * G + lane) * V, a.n);
        if (a.residual) {
            const T* r = static_cast<const T*>(a.residual) + row * a.residual_stride;
#pragma unroll
            for (int i = 0; i < NV; ++i) f.more[i] = load_near<T, REACH>(r, (i * G + lane) * V, a.n);
        }
    };
    // every lane of the workgroup takes every turn: the groups meet in lane exchanges
    auto norm = [&](int64_t r0, Row& cur, Row& next) {
        const bool live = r0 + own < a.rows;
        const int64_t row = live ? r0 + own : 0;
        if constexpr (AHEAD)
            fetch(r0 + step < a.rows ? r0 + step : r0, next);
        else
            fetch(r0, cur);
        float v[NV][V], total = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            in_place<T, REACH, WHOLE>(cur.x[i], c, a.n);
            unpack<T>(cur.x[i], v[i]);
            if (a.residual) {
                float m[V];
                in_place<T, REACH, WHOLE>(cur.more[i], c, a.n);
                unpack<T>(cur.more[i], m);
#pragma unroll
                for (int k = 0; k < V; ++k) v[i][k] += m[k];
                cur.x[i] = pack<T>(v[i]);
                unpack<T>(cur.x[i], v[i]);
                if (live) store_bits<T, WHOLE>(static_cast<T*>(a.s) + row * a.n, c, a.n, cur.x[i]);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) total += v[i][k];
        }
        const float mean = mean_of(group.sum(total), a);
        float square = 0.f, off = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[i][k] = (WHOLE ? c : c + k) < a.n ? v[i][k] - mean : 0.f;
                square = fma_acc(v[i][k], v[i][k], square);
                off += v[i][k];
            }
        }
        float by;
        const float rest = variance(group, square, off, a, by);
        if (!live) return;
        if (a.stats && lane == 0) a.stats[2 * row] = mean + rest, a.stats[2 * row + 1] = by;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            float m[V];
#pragma unroll
            for (int k = 0; k < V; ++k) v[i][k] = (v[i][k] - rest) * by;
            if (a.weight) {
                unpack<T>(KEEP ? w[KEEP ? i : 0] : load_row<T, REACH, WHOLE>(static_cast<const T*>(a.weight), c, a.n), m);
#pragma unroll
                for (int k = 0; k < V; ++k) v[i][k] *= m[k];
            }
            if (a.bias) {
                unpack<T>(KEEP ? b[KEEP ? i : 0] : load_row<T, REACH, WHOLE>(static_cast<const T*>(a.bias), c, a.n), m);
#pragma unroll
                for (int k = 0; k < V; ++k) v[i][k] += m[k];
            }
            store_bits<T, WHOLE>(static_cast<T*>(a.y) + row * a.n, c, a.n, pack<T>(v[i]));
        }
    };
    int64_t r0 = static_cast<int64_t>(blockIdx.x) * Gr::kGroups;
    Row even, odd;
    if constexpr (AHEAD) {
        fetch(r0, even);
        for (;;) {
            norm(r0, even, odd);
            if ((r0 += step) >= a.rows) break;
            norm(r0, odd, even);
            if ((r0 += step) >= a.rows) break;
        }
    } else {
        for (; r0 < a.rows; r0 += step) norm(r0, even, even);
    }
}

// A lane's sums of d h and d over its columns, in LDS: four at a time, the lanes side by
// side.  `at` of `all` parts.
template <int V>
__device__ __forceinline__ void add_columns(float* lds, int at, int all, const float (&h)[V], const float (&d)[V]) {
    fx4* sums = reinterpret_cast<fx4*>(lds);
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        fx4 &w = sums[q * all + at], &b = sums[(V / 4 + q) * all + at];
        fx4 x = w, y = b;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = fma_acc(d[4 * q + e], h[4 * q + e], x[e]);
            y[e] += d[4 * q + e];
        }
        w = x, b = y;
    }
}

// A lane's columns side by side (by elements, each a store 32 bytes off the next lane's:
// 3000 x 16384 fp16 77 us instead of 64).
template <int V>
__device__ __forceinline__ void store_sums(const float (&sum)[V], float* to, int c, int n) {
    if (c + V <= n) {
        __builtin_memcpy(to + c, sum, sizeof(sum));
        return;
    }
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (c + k < n) to[c + k] = sum[k];
}

// Sums over the rows of a workgroup's groups, in their order, to its partial sums.
template <int G, int NV, int V>
__device__ __forceinline__ void add_groups(const float (&sum)[NV][V], float* to, int n, float* lds) {
    using Gr = Group<G>;
    if constexpr (Gr::kGroups == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) store_sums(sum[i], to, (i * G + static_cast<int>(threadIdx.x)) * V, n);
    } else {
        const int lane = threadIdx.x % G, own = threadIdx.x / G;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) lds[own * (G * NV * V) + (i * G + lane) * V + k] = sum[i][k];
        __syncthreads();
        for (int c = threadIdx.x; c < n; c += Gr::kThreads) {
            float s = 0.f;
            for (int i = 0; i < Gr::kGroups; ++i) s += lds[i * (G * NV * V) + c];
            to[c] = s;
        }
    }
}

template <typename T, int G, int NV, bool WHOLE>
__global__ __launch_bounds__(Group<G>::kThreads) void layer_norm_backward_kernel(LayerNormArgs a) {
    using Gr = Group<G>;
    constexpr int V = kVec<T>;
    // A workgroup's registers leave one or two of them to a CU: the next row's loads are
    // under way during this one's sums.  (Where its columns past a whole vector let it: 32 a
    // lane would spill.)
    constexpr bool AHEAD = G >= 256 && (WHOLE || NV * V < 32);
    constexpr Reach REACH = reach_of(G, AHEAD, WHOLE);
    // 32 columns a lane: their sums are in LDS, and leave the next row its registers (3000
    // x 16384 fp16: 104 us with the sums in registers and no row ahead, 85 so, before the
// loads were unconditional and the sums stored side by side: 64)
    constexpr bool IN_LDS = NV * V == 32 && G > 64;
    __shared__ float lds[Gr::kGroups > 1 ? Gr::kThreads * NV * V : 4 * Gr::kWaves];
    __shared__ __attribute__((aligned(16))) float sums[IN_LDS ? 2 * Gr::kThreads * NV * V : 1];
    Gr group{lds};
    const int lane = threadIdx.x % G, own = threadIdx.x / G;
    ux4 w[NV];
    float gw[NV][V], gb[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (a.weight) w[i] = load_near<T, REACH>(static_cast<const T*>(a.weight), (i * G + lane) * V, a.n);
#pragma unroll
        for (int k = 0; k < V; ++k) gw[i][k] = gb[i][k] = 0.f;
        if constexpr (IN_LDS) {
#pragma unroll
            for (int q = 0; q < V / 2; ++q) reinterpret_cast<fx4*>(sums)[q * NV * G + i * G + lane] = fx4{0.f, 0.f, 0.f, 0.f};
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (a.weight) in_place<T, REACH, WHOLE>(w[i], (i * G + lane) * V, a.n);
    struct Row {
        ux4 x[NV], g[NV];
        float mean, by;
    };
    const int64_t step = static_cast<int64_t>(a.blocks) * Gr::kGroups;
    auto fetch = [&](int64_t r0, Row& f) {
        const int64_t row = r0 + own < a.rows ? r0 + own : 0;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* g = static_cast<const T*>(a.grad_y) + row * a.gy_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            f.x[i] = load_near<T, REACH>(x, (i * G + lane) * V, a.n);
            f.g[i] = load_near<T, REACH>(g, (i * G + lane) * V, a.n);
        }
        f.mean = a.stats[2 * row], f.by = a.stats[2 * row + 1];
    };
    auto gradients = [&](int64_t r0, Row& cur, Row& next) {
        const bool live = r0 + own < a.rows;
        const int64_t row = live ? r0 + own : 0;
        if constexpr (!AHEAD) fetch(r0, cur);
        ux4 more[NV];
        if (a.grad_s) {
            const T* s = static_cast<const T*>(a.grad_s) + row * a.gs_stride;
#pragma unroll
            for (int i = 0; i < NV; ++i) more[i] = load_near<T, REACH>(s, (i * G + lane) * V, a.n);
        }
        // (behind the last row this one once more)
        if constexpr (AHEAD) fetch(r0 + step < a.rows ? r0 + step : r0, next);
        const float mean = cur.mean, by = cur.by;
        float h[NV][V], d[NV][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            float m[V];
            in_place<T, REACH, WHOLE>(cur.x[i], c, a.n);
            in_place<T, REACH, WHOLE>(cur.g[i], c, a.n);
            unpack<T>(cur.x[i], h[i]);
            unpack<T>(cur.g[i], d[i]);
            if (a.weight) unpack<T>(w[i], m);
#pragma unroll
            for (int k = 0; k < V; ++k)
                // past the row's end nothing: there x is 0, and less the mean no number
                // that 0 would take away where the mean is none
                h[i][k] = (WHOLE ? c : c + k) < a.n ? (h[i][k] - mean) * by : 0.f;
            if constexpr (IN_LDS) {
                add_columns<V>(sums, i * G + lane, NV * G, h[i], d[i]);
            } else if (live) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    gw[i][k] = fma_acc(d[i][k], h[i][k], gw[i][k]);
                    gb[i][k] += d[i][k];
                }
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if (a.weight) d[i][k] *= m[k];
                s1 += d[i][k];
                s2 = fma_acc(d[i][k], h[i][k], s2);
            }
        }
        group.sum(s1, s2);
        s1 *= a.inv_n, s2 *= a.inv_n;
        if (live && a.gx) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float m[V];
                if (a.grad_s) {
                    in_place<T, REACH, WHOLE>(more[i], (i * G + lane) * V, a.n);
                    unpack<T>(more[i], m);
                }
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    d[i][k] = (d[i][k] - s1 - h[i][k] * s2) * by;
                    if (a.grad_s) d[i][k] += m[k];
                }
                store_bits<T, WHOLE>(static_cast<T*>(a.gx) + row * a.n, (i * G + lane) * V, a.n, pack<T>(d[i]));
            }
        }
    };
    int64_t r0 = static_cast<int64_t>(blockIdx.x) * Gr::kGroups;
    Row even, odd;
    if constexpr (AHEAD) {  // (r0 < a.rows: there are no more workgroups than rows)
        fetch(r0, even);
        for (;;) {
            gradients(r0, even, odd);
            if ((r0 += step) >= a.rows) break;
            gradients(r0, odd, even);
            if ((r0 += step) >= a.rows) break;
        }
    } else {
        for (; r0 < a.rows; r0 += step) gradients(r0, even, even);
    }
    if (!a.partial) return;
    float* to = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.n;
    if constexpr (IN_LDS) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int q = 0; q < V / 4; ++q) {
                const fx4 x = reinterpret_cast<fx4*>(sums)[q * NV * G + i * G + lane];
                const fx4 y = reinterpret_cast<fx4*>(sums)[(V / 4 + q) * NV * G + i * G + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) gw[i][4 * q + e] = x[e], gb[i][4 * q + e] = y[e];
            }
    }
    add_groups<G, NV, V>(gw, to, a.n, lds);
    add_groups<G, NV, V>(gb, to + a.n, a.n, lds);
}

// ---------------------------------------------------------------------------
// Rows wider than a workgroup holds
// ---------------------------------------------------------------------------

constexpr int kWideThreads = 1024;
using WideGroup = Group<kWideThreads>;

template <typename T>
__device__ __forceinline__ void wide_values(const LayerNormArgs& a, int64_t row, int c, bool summed, float (&v)[kVec<T>]) {
    unpack<T>(load_row<T, kNear>(static_cast<const T*>(a.x) + row * a.x_stride, c, a.n), v);
    if (summed && a.residual) {
        float m[kVec<T>];
        unpack<T>(load_row<T, kNear>(static_cast<const T*>(a.residual) + row * a.residual_stride, c, a.n), m);
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) v[k] += m[k];
        unpack<T>(pack<T>(v), v);
    }
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void layer_norm_wide_forward_kernel(LayerNormArgs a) {
    constexpr int V = kVec<T>, kStep = kWideThreads * V;
    __shared__ float meet[4 * WideGroup::kWaves];
    WideGroup group{meet};
    for (int64_t row = blockIdx.x; row < a.rows; row += a.blocks) {
        float v[V], m[V], total = 0.f, square = 0.f, off = 0.f;
        for (int c = threadIdx.x * V; c < a.n; c += kStep) {
            wide_values<T>(a, row, c, true, v);
            if (a.residual) store_bits(static_cast<T*>(a.s) + row * a.n, c, a.n, pack<T>(v));
#pragma unroll
            for (int k = 0; k < V; ++k) total += v[k];
        }
        const float mean = mean_of(group.sum(total), a);
        for (int c = threadIdx.x * V; c < a.n; c += kStep) {
            wide_values<T>(a, row, c, true, v);
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (c + k < a.n) square = fma_acc(v[k] - mean, v[k] - mean, square), off += v[k] - mean;
        }
        float by;
        const float rest = variance(group, square, off, a, by);
        if (a.stats && threadIdx.x == 0) a.stats[2 * row] = mean + rest, a.stats[2 * row + 1] = by;
        for (int c = threadIdx.x * V; c < a.n; c += kStep) {
            wide_values<T>(a, row, c, true, v);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = (v[k] - mean - rest) * by;
            if (a.weight) {
                unpack<T>(load_row<T, kNear>(static_cast<const T*>(a.weight), c, a.n), m);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] *= m[k];
            }
            if (a.bias) {
                unpack<T>(load_row<T, kNear>(static_cast<const T*>(a.bias), c, a.n), m);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] += m[k];
            }
            store_bits(static_cast<T*>(a.y) + row * a.n, c, a.n, pack<T>(v));
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void layer_norm_wide_backward_kernel(LayerNormArgs a) {
    constexpr int V = kVec<T>, kStep = kWideThreads * V;
    __shared__ float meet[4 * WideGroup::kWaves];
    WideGroup group{meet};
    for (int64_t row = blockIdx.x; row < a.rows; row += a.blocks) {
        const float mean = a.stats[2 * row], by = a.stats[2 * row + 1];
        const T* g = static_cast<const T*>(a.grad_y) + row * a.gy_stride;
        float h[V], d[V], m[V], s1 = 0.f, s2 = 0.f;
        for (int turn = 0; turn < 2; ++turn) {
            for (int c = threadIdx.x * V; c < a.n; c += kStep) {
                wide_values<T>(a, row, c, false, h);
                unpack<T>(load_row<T, kNear>(g, c, a.n), d);
                if (a.weight) {
                    unpack<T>(load_row<T, kNear>(static_cast<const T*>(a.weight), c, a.n), m);
#pragma unroll
                    for (int k = 0; k < V; ++k) d[k] *= m[k];
                }
#pragma unroll
                for (int k = 0; k < V; ++k) h[k] = c + k < a.n ? (h[k] - mean) * by : 0.f;
                if (turn == 0) {
#pragma unroll
                    for (int k = 0; k < V; ++k) s1 += d[k], s2 = fma_acc(d[k], h[k], s2);
                    continue;
                }
#pragma unroll
                for (int k = 0; k < V; ++k) d[k] = (d[k] - s1 - h[k] * s2) * by;
                if (a.grad_s) {
                    unpack<T>(load_row<T, kNear>(static_cast<const T*>(a.grad_s) + row * a.gs_stride, c, a.n), m);
#pragma unroll
                    for (int k = 0; k < V; ++k) d[k] += m[k];
                }
                store_bits(static_cast<T*>(a.gx) + row * a.n, c, a.n, pack<T>(d));
            }
            if (turn == 0) {
                group.sum(s1, s2);
                s1 *= a.inv_n, s2 *= a.inv_n;
            }
        }
    }
}

// 512 columns (256 in fp32) of every gridDim.y-th row for each wave.
template <typename T>
__global__ __launch_bounds__(64) void layer_norm_columns_kernel(LayerNormArgs a) {
    constexpr int V = kVec<T>;
    const int c = (blockIdx.x * 64 + threadIdx.x) * V;
    float gw[V] = {}, gb[V] = {};
#pragma unroll 4
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float mean = a.stats[2 * row], by = a.stats[2 * row + 1];
        float h[V], d[V];
        wide_values<T>(a, row, c, false, h);
        unpack<T>(load_row<T, kNear>(static_cast<const T*>(a.grad_y) + row * a.gy_stride, c, a.n), d);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            gw[k] = fma_acc(d[k], (h[k] - mean) * by, gw[k]);
            gb[k] += d[k];
        }
    }
    float* to = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.n;
    store_sums(gw, to, c, a.n);
    store_sums(gb, to + a.n, c, a.n);
}

// 32 columns per workgroup, 32 runs of blocks each: gw (blockIdx.y 0) or gb.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_weights_kernel(LayerNormArgs a) {
    __shared__ float part[32][32];
    void* out = blockIdx.y ? a.gb : a.gw;
    if (!out) return;
    const int col = threadIdx.x % 32, run = threadIdx.x / 32;
    const float* at = a.partial + (blockIdx.y ? a.n : 0);
    const int len = (a.blocks + 31) / 32, end = min(a.blocks, (run + 1) * len);
    for (int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + col; c - col < a.n; c += static_cast<int64_t>(gridDim.x) * 32) {
        float s = 0.f;
        if (c < a.n) {
#pragma unroll 8
            for (int i = run * len; i < end; ++i) s += at[static_cast<int64_t>(i) * 2 * a.n + c];
        }
        part[run][col] = s;
        __syncthreads();
        if (run == 0 && c < a.n) {
            for (int i = 1; i < 32; ++i) s += part[i][col];
            static_cast<T*>(out)[c] = from_acc<T>(s);
        }
        __syncthreads();
    }
}

// Lanes a row and parts of 16 bytes a lane; 0 lanes: rows that are read again for each sum.
struct NormForm {
    int lanes, parts;
};

// As few lanes as hold a row in one part each, up to a wave with four parts; then a workgroup
// (16384 x 2048 bf16 by waves 46 us forward and 45 backward, by workgroups 47 and 55; 16384 x
// 1040 18 and 27, 23 and 35).  Up to a row for each CU, the workgroup takes rows that a wave would
// hold (64 x 2000 fp16: 3.4 and 4.1 us, by waves 4.0 and 6.2).
static NormForm norm_form(int64_t rows, int64_t n, int vec) {
    const int64_t parts = nsh_host::ceil_div(n, vec);
    if (parts <= 64) return {parts <= 8 ? 8 : parts <= 16 ? 16 : parts <= 32 ? 32 : 64, 1};
    if (parts <= 256 && rows <= nsh_host::compute_units()) return {256, 1};
    if (parts <= 256) return {64, parts <= 128 ? 2 : 4};
    if (parts <= 512) return {256, 2};
    if (parts <= 2048) return {512, parts <= 1024 ? 2 : 4};
    return {0, 0};
}

// Workgroups that walk the rows: enough to fill the card.
static int norm_row_blocks(int64_t rows, int per, int64_t each) {
    return static_cast<int>(std::min(nsh_host::ceil_div(rows, per), nsh_host::compute_units() * each));
}

// In the backward few enough that their sums of the weights' gradients, one set a workgroup,
// stay small next to the rows (two a CU: 16384 x 2048 bf16 44.5 us and 4.0 for the sums, four:
// 49 and 4.6); 512 lanes' registers leave one workgroup to a CU.
constexpr int kMostNormBlocks = 2;

static int64_t wide_columns_across(int64_t n, int vec) { return nsh_host::ceil_div(n, 64 * vec); }

// Sets of such sums, which the workspace holds and the launches write.
static int norm_sums(int64_t rows, int64_t n, int vec) {
    const NormForm f = norm_form(rows, n, vec);
    if (f.lanes) return norm_row_blocks(rows, f.lanes < 256 ? 256 / f.lanes : 1, f.lanes == 512 ? 1 : kMostNormBlocks);
    // 16 waves a CU, no more than there is room for (600 x 40000 bf16: 18 us, and 108 with
    // 512 of them down the rows, whose sums are more than the rows)
    return static_cast<int>(std::min<int64_t>(norm_row_blocks(rows, 1, kMostNormBlocks),
                                              nsh_host::ceil_div(16 * nsh_host::compute_units(), wide_columns_across(n, vec))));
}

// (a launch takes less than 2^32 threads)
template <typename T>
static void layer_norm_weights(const LayerNormArgs& a, hipStream_t st) {
    const int blocks = std::min((a.n + 31) / 32, 1 << 20);
    layer_norm_weights_kernel<T><<<dim3(blocks, 2), 1024, 0, st>>>(a);
}

template <typename T, int G, int NV, bool WHOLE>
static int layer_norm_rows(LayerNormArgs a, bool bwd, hipStream_t st) {
    using Gr = Group<G>;
    // (forward, rows of a workgroup: one each, as far as a launch's 2^32 threads go)
    a.blocks = bwd ? norm_sums(a.rows, a.n, kVec<T>) : norm_row_blocks(a.rows, Gr::kGroups, G == 512 ? 2 : G > 64 ? 1 << 13 : 8);
    if (!bwd) {
        layer_norm_forward_kernel<T, G, NV, WHOLE><<<a.blocks, Gr::kThreads, 0, st>>>(a);
        return nsh_host::check_launch("layer_norm_forward");
    }
    layer_norm_backward_kernel<T, G, NV, WHOLE><<<a.blocks, Gr::kThreads, 0, st>>>(a);
    if (a.partial) layer_norm_weights<T>(a, st);
    return nsh_host::check_launch("layer_norm_backward");
}

template <typename T, int G, int NV>
static int layer_norm_launch(const LayerNormArgs& a, bool bwd, hipStream_t st) {
    return a.n % kVec<T> ? layer_norm_rows<T, G, NV, false>(a, bwd, st) : layer_norm_rows<T, G, NV, true>(a, bwd, st);
}

template <typename T>
static int layer_norm_wide(LayerNormArgs a, bool bwd, hipStream_t st) {
    a.blocks = norm_row_blocks(a.rows, 1, bwd ? kMostNormBlocks : 8);
    if (!bwd) {
        layer_norm_wide_forward_kernel<T><<<a.blocks, kWideThreads, 0, st>>>(a);
        return nsh_host::check_launch("layer_norm_forward");
    }
    if (a.gx) layer_norm_wide_backward_kernel<T><<<a.blocks, kWideThreads, 0, st>>>(a);
    if (a.partial) {
        a.blocks = norm_sums(a.rows, a.n, kVec<T>);
        const unsigned across = static_cast<unsigned>(wide_columns_across(a.n, kVec<T>));
        layer_norm_columns_kernel<T><<<dim3(across, a.blocks), 64, 0, st>>>(a);
        layer_norm_weights<T>(a, st);
    }
    return nsh_host::check_launch("layer_norm_backward");
}

template <typename T>
static int layer_norm_dispatch(const LayerNormArgs& a, bool bwd, hipStream_t st) {
    const NormForm f = norm_form(a.rows, a.n, kVec<T>);
    switch (f.lanes) {
        case 8: return layer_norm_launch<T, 8, 1>(a, bwd, st);
        case 16: return layer_norm_launch<T, 16, 1>(a, bwd, st);
        case 32: return layer_norm_launch<T, 32, 1>(a, bwd, st);
        case 64:
            if (f.parts == 1) return layer_norm_launch<T, 64, 1>(a, bwd, st);
            return f.parts == 2 ? layer_norm_launch<T, 64, 2>(a, bwd, st) : layer_norm_launch<T, 64, 4>(a, bwd, st);
        case 256: return f.parts == 1 ? layer_norm_launch<T, 256, 1>(a, bwd, st) : layer_norm_launch<T, 256, 2>(a, bwd, st);
        case 512: return f.parts == 2 ? layer_norm_launch<T, 512, 2>(a, bwd, st) : layer_norm_launch<T, 512, 4>(a, bwd, st);
        default: return layer_norm_wide<T>(a, bwd, st);
    }
}

}  // namespace nsh

using nsh_host::fail;

extern "C" int64_t nsh_layer_norm_workspace_bytes(const nsh_layer_norm_args* g) {
    if (!g || g->rows < 1 || g->n < 1 || g->dtype < NSH_DTYPE_FLOAT16 || g->dtype > NSH_DTYPE_FLOAT32) return -1;
    const int vec = g->dtype == NSH_DTYPE_FLOAT32 ? 4 : 8;
    return static_cast<int64_t>(nsh::norm_sums(g->rows, g->n, vec)) * 2 * g->n * 4;
}

static int layer_norm(const char* op, const nsh_layer_norm_args* g, bool bwd, void* stream) {
    if (!g) return fail(NSH_ERR_INVALID, "%s: null arguments", op);
    if (g->dtype < NSH_DTYPE_FLOAT16 || g->dtype > NSH_DTYPE_FLOAT32)
        return fail(NSH_ERR_INVALID, "%s: unsupported dtype code %d", op, g->dtype);
    if (g->rows < 1 || g->n < 1) return fail(NSH_ERR_INVALID, "%s: empty tensor", op);
    if (g->n > (int64_t(1) << 30) || g->rows > (int64_t(1) << 40))
        return fail(NSH_ERR_INVALID, "%s: rows wider than 2^30 or more than 2^40", op);
    if (!(g->eps >= 0) || std::isinf(g->eps)) return fail(NSH_ERR_INVALID, "%s: eps must be finite and not negative", op);
    if (bwd ? !g->x || !g->grad_y || !g->stats || (!g->grad_x && !g->grad_weight && !g->grad_bias)
            : !g->x || !g->y || !g->residual != !g->s)
        return fail(NSH_ERR_INVALID, "%s: null pointer argument", op);
    nsh::LayerNormArgs a{};
    a.x = g->x, a.weight = g->weight, a.x_stride = g->x_stride;
    a.stats = g->stats, a.rows = g->rows, a.n = static_cast<int>(g->n);
    a.eps = static_cast<float>(g->eps), a.inv_n = 1.f / static_cast<float>(a.n);
    if (bwd) {
        a.grad_y = g->grad_y, a.gy_stride = g->gy_stride, a.grad_s = g->grad_s, a.gs_stride = g->gs_stride;
        a.gx = g->grad_x, a.gw = g->grad_weight, a.gb = g->grad_bias;
        if (a.gw || a.gb) {
            if (!g->workspace || g->workspace_bytes < nsh_layer_norm_workspace_bytes(g))
                return fail(NSH_ERR_INVALID, "%s: workspace smaller than nsh_layer_norm_workspace_bytes", op);
            if (!nsh_host::aligned(g->workspace, 4)) return fail(NSH_ERR_INVALID, "%s: misaligned workspace", op);
            a.partial = static_cast<float*>(g->workspace);
        }
    } else {
        a.residual = g->residual, a.residual_stride = g->residual_stride, a.bias = g->bias;
        a.y = g->y, a.s = g->s;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (g->dtype) {
        case NSH_DTYPE_FLOAT16: return nsh::layer_norm_dispatch<nsh::f16>(a, bwd, st);
        case NSH_DTYPE_BFLOAT16: return nsh::layer_norm_dispatch<nsh::bf16>(a, bwd, st);
        default: return nsh::layer_norm_dispatch<float>(a, bwd, st);
    }
}

extern "C" int nsh_layer_norm_forward(const nsh_layer_norm_args* g, void* stream) {
    return layer_norm("layer_norm_forward", g, false, stream);
}

extern "C" int nsh_layer_norm_backward(const nsh_layer_norm_args* g, void* stream) {
    return layer_norm("layer_norm_backward", g, true, stream);
}
