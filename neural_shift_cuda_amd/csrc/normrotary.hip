// normrotary.hip -- norm of queries and keys for each head with the rotation
// by position, in one pass, on gfx950.
//
//   r = (mean(x^2) + eps)^(-1/2),  y = x r w,  out = rotation(y)
//   g' = rotation^T(g),  gx = r (g' w - x r^2 mean(g' w x)),  gw = sum g' x r
//
// HBM streams: forward reads and writes every element once, backward reads x
// and g and writes gx.  A row (one head of one token) belongs to a group of
// lanes that holds it whole in registers, 16 bytes a lane where the rows allow
// it.  The sum of squares meets in the group, and a rotated pair's other half
// comes from its lane, by DPP and row swaps: through LDS (shuffles) the forward
// of 4 x 20 heads of 4096 tokens, width 128, bf16 took 51.5 us instead of 35 and
// waited on LDS, not on memory.  A row's head, token and batch come from
// multiplications by reciprocals.  Rows run with the heads fastest, so a token's
// cos and sin stay in the caches for all its heads.  Queries and keys share the
// launch.  gw: each lane adds up its own columns over the rows it walks, the
// groups of a workgroup add in order, and a second launch adds the workgroups'
// sums in order.
//
// At that size: forward 40 us (84 + 84 MB, 4.2 TB/s; 35 where the inputs are the
// same each time and the memory side cache has some of them), backward 59 us (168 +
// 84 MB, 4.3 TB/s), the weights' sums 5 us; a copy of 84 MB runs at 7.0 TB/s from that
// cache and at 5.1 without.  What bounds them is memory latency behind a position's:
// its table rows can be asked for only then.  The root is the reciprocal square root
// instruction's, off by 2^-23 of the row (fp32 errors 1.4e-7 to 2.0e-7).
#include <algorithm>
#include <cmath>

#include "divisor.hpp"

namespace nsh {

constexpr int kNormThreads = 256;
constexpr int kNormMaxD = 512;

// One of the two tensors, as the kernels take it.
struct NormSide {
    const void *x, *w, *g;
    int64_t xs[3], gs[3];
    void *out, *gw;
    int H, blocks;
    Divisor by_h;
};

struct NormArgs {
    NormSide side[2];
    const float *cos, *sin;
    const int32_t* positions;
    int64_t pos_stride;
    int L, D, half, interleaved;
    int full;         // the row's two halves are its lanes' two halves
    float inv_d;      // 1 / D
    uint32_t tokens;  // B * L
    Divisor by_l;
    int64_t rows;
    float eps;
    float* partial;  // (blocks of both, D)
};

template <typename T, int VEC>
__device__ __forceinline__ void load_cols(const T* p, int d0, int D, float (&o)[VEC]) {
    if constexpr (VEC == 1) {
        o[0] = d0 < D ? to_acc(p[d0]) : 0.f;
    } else {
        if (d0 < D) {
            load_acc<T, VEC>(p + d0, o);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) o[k] = 0.f;
        }
    }
}

typedef float fx8 __attribute__((ext_vector_type(8)));
typedef float fx4 __attribute__((ext_vector_type(4)));

// Rounded to nearest even by the conversion instructions.
template <typename T, int VEC>
__device__ __forceinline__ void store_cols(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 8 && __is_same(T, bf16)) {
        typedef __bf16 V __attribute__((ext_vector_type(8)));
        *reinterpret_cast<V*>(p) = __builtin_convertvector((fx8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}), V);
    } else if constexpr (VEC == 8 && __is_same(T, f16)) {
        typedef _Float16 V __attribute__((ext_vector_type(8)));
        *reinterpret_cast<V*>(p) = __builtin_convertvector((fx8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}), V);
    } else if constexpr (VEC == 4 && __is_same(T, float)) {
        *reinterpret_cast<fx4*>(p) = fx4{v[0], v[1], v[2], v[3]};
    } else {
        store_acc<T, VEC>(p, v, false);
    }
}

// Lane exchanges within a group without LDS: DPP in rows of 16 lanes, swaps of
// rows beyond.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum_rows(float v) {  // with the row of 16 lanes next to it
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The value of lane ^ (G / 2).
template <int G>
__device__ __forceinline__ float across(float v) {
    const uint32_t x = __float_as_uint(v);
    if constexpr (G == 8) {
        // lanes 4 b .. 4 b + 3 of a row of 16: even b from four lanes on, odd from four before
        int t = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x104, 0xf, 0x5, true);
        t = __builtin_amdgcn_update_dpp(t, static_cast<int>(x), 0x114, 0xf, 0xa, false);
        return __int_as_float(t);
    } else if constexpr (G == 16) {
        return dpp<0x128>(v);  // rotation by 8
    } else if constexpr (G == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return __uint_as_float(threadIdx.x & 16 ? r[0] : r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return __uint_as_float(threadIdx.x & 32 ? r[0] : r[1]);
    }
}

// A lane holds N parts of VEC columns: part n starts at (n * G + lane) * VEC.
// VEC > 1 has N == 1, whole vectors inside the row, and pairs that lie in one
// lane (interleaved) or a whole number of lanes apart.  SIGN -1 is the
// transposed rotation.
template <int VEC, int N, int G>
__device__ __forceinline__ void rotate(float (&y)[N][VEC], const NormArgs& a, int lane,
                                       const float* cs, const float* sn, bool ok, float sign,
                                       float* lds) {
    const int rot = 2 * a.half;
    if constexpr (VEC > 1) {
        const int d0 = lane * VEC;
        if (a.interleaved) {
#pragma unroll
            for (int k = 0; k < VEC; k += 2) {
                const int d = d0 + k;
                if (d < rot) {
                    const float c = ok ? cs[d / 2] : __builtin_nanf("");
                    const float s = ok ? sn[d / 2] * sign : 0.f;
                    const float u = y[0][k], v = y[0][k + 1];
                    y[0][k] = u * c - v * s;
                    y[0][k + 1] = u * s + v * c;
                }
            }
        } else {
            const bool first = d0 < a.half;
            const int other = first ? lane + a.half / VEC : lane - a.half / VEC;
            const int base = (threadIdx.x & 63 & ~(G - 1)) + (other & (G - 1));
            float z[VEC];
            if (a.full) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) z[k] = across<G>(y[0][k]);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) z[k] = __shfl(y[0][k], base);
            }
            if (d0 < rot) {
                const int e = first ? d0 : d0 - a.half;
                float c[VEC], s[VEC];
                if (ok) {
#pragma unroll
                    for (int k = 0; k < VEC; k += 4) {
                        load_acc<float, 4>(cs + e + k, *reinterpret_cast<float(*)[4]>(&c[k]));
                        load_acc<float, 4>(sn + e + k, *reinterpret_cast<float(*)[4]>(&s[k]));
                    }
                }
                const float sg = first ? -sign : sign;
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    y[0][k] = ok ? y[0][k] * c[k] + sg * s[k] * z[k] : __builtin_nanf("");
            }
        }
    } else {
        // any width: the row goes through LDS (the workgroup is one wave)
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (n * G + lane < a.D) lds[n * G + lane] = y[n][0];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int d = n * G + lane;
            if (d >= rot) continue;
            const bool first = a.interleaved ? !(d & 1) : d < a.half;
            const int e = a.interleaved ? d / 2 : first ? d : d - a.half;
            const int o = a.interleaved ? d ^ 1 : first ? d + a.half : d - a.half;
            const float c = ok ? cs[e] : __builtin_nanf(""), s = ok ? sn[e] : 0.f;
            y[n][0] = y[n][0] * c + (first ? -sign : sign) * s * lds[o];
        }
        __syncthreads();
    }
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
    v += dpp<0xB1>(v);   // lane ^ 1
    v += dpp<0x4E>(v);   // lane ^ 2
    v += dpp<0x141>(v);  // mirrored in eight lanes, whose fours agree
    if constexpr (G >= 16) v += dpp<0x140>(v);  // mirrored in 16
    if constexpr (G >= 32) v = sum_rows(v);
    if constexpr (G >= 64) v = sum_halves(v);
    return v;
}

// ROWS rows of a group go at once, all their loads first: a row's loads hang on
// its position's, and one row a group leaves too few bytes under way.
template <typename T, int VEC, int N, int G, int THREADS, bool BWD, int ROWS>
__global__ __launch_bounds__(THREADS) void norm_rotary_kernel(NormArgs a) {
    __shared__ float lds[VEC == 1 || BWD ? (VEC == 1 ? kNormMaxD : THREADS * VEC) : 1];
    const bool key = static_cast<int>(blockIdx.x) >= a.side[0].blocks;
    const NormSide& sd = a.side[key];
    const int block = key ? blockIdx.x - a.side[0].blocks : blockIdx.x;
    constexpr int kRows = THREADS / G * ROWS;
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const int64_t total = static_cast<int64_t>(a.tokens) * sd.H;
    float w[N][VEC], gw[N][VEC];
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[n][k] = 1.f, gw[n][k] = 0.f;
        if (sd.w) load_cols<T, VEC>(static_cast<const T*>(sd.w), (n * G + lane) * VEC, a.D, w[n]);
    }
    // every lane of the workgroup takes every turn: the groups meet in shuffles
    for (int64_t r0 = static_cast<int64_t>(block) * kRows; r0 < total;
         r0 += static_cast<int64_t>(sd.blocks) * kRows) {
        float v[ROWS][N][VEC], g[BWD ? ROWS : 1][N][VEC];
        bool live[ROWS], ok[ROWS];
        int64_t pos[ROWS];
        T* out[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const int64_t r = r0 + group * ROWS + u;
            live[u] = r < total;
            const uint32_t rr = live[u] ? static_cast<uint32_t>(r) : 0u;
            const uint32_t token = sd.by_h(rr), h = rr - token * sd.H;
            const uint32_t b = a.by_l(token), t = token - b * a.L;
            pos[u] = a.positions ? a.positions[b * a.pos_stride + t] : t;
            const T* x = static_cast<const T*>(sd.x) + b * sd.xs[0] + h * sd.xs[1] + t * sd.xs[2];
            out[u] = static_cast<T*>(sd.out) + ((static_cast<int64_t>(b) * sd.H + h) * a.L + t) * a.D;
#pragma unroll
            for (int n = 0; n < N; ++n) load_cols<T, VEC>(x, (n * G + lane) * VEC, a.D, v[u][n]);
            if constexpr (BWD) {
                const T* gp = static_cast<const T*>(sd.g) + b * sd.gs[0] + h * sd.gs[1] + t * sd.gs[2];
#pragma unroll
                for (int n = 0; n < N; ++n) load_cols<T, VEC>(gp, (n * G + lane) * VEC, a.D, g[u][n]);
            }
        }
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            ok[u] = pos[u] >= 0 && pos[u] < a.rows;
            const float* cs = a.cos + (ok[u] ? pos[u] : 0) * a.half;
            const float* sn = a.sin + (ok[u] ? pos[u] : 0) * a.half;
            float sq = 0.f;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < VEC; ++k) sq = fma_acc(v[u][n][k], v[u][n][k], sq);
            const float rs = __builtin_amdgcn_rsqf(fma_acc(group_sum<G>(sq), a.inv_d, a.eps));
            if constexpr (!BWD) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) v[u][n][k] = v[u][n][k] * rs * w[n][k];
                rotate<VEC, N, G>(v[u], a, lane, cs, sn, ok[u], 1.f, lds);
            } else {
                rotate<VEC, N, G>(g[u], a, lane, cs, sn, ok[u], -1.f, lds);
                float dot = 0.f;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        if (live[u]) gw[n][k] = fma_acc(g[u][n][k] * rs, v[u][n][k], gw[n][k]);
                        g[u][n][k] *= w[n][k];
                        dot = fma_acc(g[u][n][k], v[u][n][k], dot);
                    }
                dot = group_sum<G>(dot) * a.inv_d * rs * rs;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) v[u][n][k] = rs * (g[u][n][k] - v[u][n][k] * dot);
            }
            if (live[u]) {
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int d0 = (n * G + lane) * VEC;
                    if (d0 < a.D) store_cols<T, VEC>(out[u] + d0, v[u][n]);
                }
            }
        }
    }
    if constexpr (BWD) {
        if (!a.partial) return;
        float* part = a.partial + static_cast<int64_t>(blockIdx.x) * a.D;
        if constexpr (VEC == 1) {
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (n * G + lane < a.D) part[n * G + lane] = gw[n][0];
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) lds[(group * G + lane) * VEC + k] = gw[0][k];
            __syncthreads();
            for (int d = threadIdx.x; d < a.D; d += THREADS) {
                float s = 0.f;
                for (int i = 0; i < THREADS / G; ++i) s += lds[i * G * VEC + d];
                part[d] = s;
            }
        }
    }
}

// 32 columns of one side per workgroup, 32 runs of blocks each.
template <typename T>
__global__ __launch_bounds__(1024) void norm_weight_kernel(NormArgs a) {
    __shared__ float part[32][32];
    const NormSide& sd = a.side[blockIdx.y];
    if (!sd.gw) return;
    const int c = threadIdx.x % 32, run = threadIdx.x / 32, d = blockIdx.x * 32 + c;
    const float* at = a.partial + (blockIdx.y ? static_cast<int64_t>(a.side[0].blocks) * a.D : 0);
    const int len = (sd.blocks + 31) / 32, end = min(sd.blocks, (run + 1) * len);
    float s = 0.f;
    if (d < a.D) {
#pragma unroll 16
        for (int i = run * len; i < end; ++i) s += at[static_cast<int64_t>(i) * a.D + d];
    }
    part[run][c] = s;
    __syncthreads();
    if (run == 0 && d < a.D) {
        for (int i = 1; i < 32; ++i) s += part[i][c];
        static_cast<T*>(sd.gw)[d] = from_acc<T>(s);
    }
}

static bool norm_vectors(const nsh_norm_rotary_args* g, bool bwd) {
    const int64_t bytes = g->dtype == NSH_DTYPE_FLOAT32 ? 4 : 2, vec = 16 / bytes;
    if (g->D % vec || (!g->interleaved && g->half % vec) || g->half % 4) return false;
    auto good = [&](const void* p, const int64_t* s) {
        return !p || (nsh_host::aligned(p, 16) && s[0] % vec == 0 && s[1] % vec == 0 && s[2] % vec == 0);
    };
    static const int64_t none[3] = {0, 0, 0};
    return good(g->q, g->q_stride) && good(g->k, g->k_stride) && good(g->q_weight, none) &&
           good(g->k_weight, none) && good(g->cos, none) && good(g->sin, none) &&
           (bwd ? good(g->grad_q_out, g->gq_stride) && good(g->grad_k_out, g->gk_stride) &&
                      good(g->grad_q, none) && good(g->grad_k, none)
                : good(g->q_out, none) && good(g->k_out, none));
}

// Workgroups of a side: enough to fill the card, few enough that their sums of
// the weight gradient stay small.
static int norm_blocks(int64_t rows, int per, bool bwd) {
    const int64_t most = static_cast<int64_t>(nsh_host::compute_units()) * (bwd ? 8 : 16);
    return static_cast<int>(std::min(nsh_host::ceil_div(rows, per), most));
}

template <typename T, int VEC, int N, int G, int THREADS, int ROWS>
static int norm_launch(NormArgs a, bool bwd, hipStream_t st) {
    for (auto& sd : a.side)
        sd.blocks = norm_blocks(static_cast<int64_t>(a.tokens) * sd.H, THREADS / G * ROWS, bwd);
    a.full = VEC > 1 && !a.interleaved && 2 * a.half == G * VEC;
    const unsigned grid = a.side[0].blocks + a.side[1].blocks;
    if (bwd) {
        norm_rotary_kernel<T, VEC, N, G, THREADS, true, ROWS><<<grid, THREADS, 0, st>>>(a);
        if (a.partial)
            norm_weight_kernel<T><<<dim3((a.D + 31) / 32, 2), 1024, 0, st>>>(a);
    } else {
        norm_rotary_kernel<T, VEC, N, G, THREADS, false, ROWS><<<grid, THREADS, 0, st>>>(a);
    }
    return nsh_host::check_launch(bwd ? "norm_rotary_backward" : "norm_rotary_forward");
}

// Two rows at once, forward, where that leaves no CU without work (4 x 20 heads
// of 4096 tokens, bf16, the same inputs each time: 38.7 us with one, 35.1 with two,
// 40.1 with four).  The backward has two tensors' loads under way with one (60.5 us,
// 67.9 with two).
template <typename T, int G>
static int norm_rows(const NormArgs& a, bool bwd, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int64_t rows = static_cast<int64_t>(a.tokens) * (a.side[0].H + a.side[1].H);
    const bool many = rows * G >= static_cast<int64_t>(nsh_host::compute_units()) * kNormThreads * 8;
    return many && !bwd ? norm_launch<T, V, 1, G, kNormThreads, 2>(a, bwd, st)
                        : norm_launch<T, V, 1, G, kNormThreads, 1>(a, bwd, st);
}

template <typename T>
static int norm_dispatch(const NormArgs& a, bool vectors, bool bwd, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (!vectors) return norm_launch<T, 1, kNormMaxD / 64, 64, 64, 1>(a, bwd, st);
    const int lanes = a.D / V;
    if (lanes <= 8) return norm_rows<T, 8>(a, bwd, st);
    if (lanes <= 16) return norm_rows<T, 16>(a, bwd, st);
    if (lanes <= 32) return norm_rows<T, 32>(a, bwd, st);
    if (lanes <= 64) return norm_rows<T, 64>(a, bwd, st);
    return norm_launch<T, 1, kNormMaxD / 64, 64, 64, 1>(a, bwd, st);
}

}  // namespace nsh

using nsh_host::fail;

extern "C" int64_t nsh_norm_rotary_workspace_bytes(const nsh_norm_rotary_args* g) {
    if (!g || g->B < 1 || g->L < 1 || g->D < 1) return -1;
    // at least one row a workgroup, whichever lanes the rows take
    const int64_t blocks = static_cast<int64_t>(nsh::norm_blocks(g->B * g->L * g->Hq, 1, true)) +
                           nsh::norm_blocks(g->B * g->L * g->Hk, 1, true);
    return blocks * g->D * 4;
}

static int norm_rotary(const char* op, const nsh_norm_rotary_args* g, bool bwd, void* stream) {
    if (!g) return fail(NSH_ERR_INVALID, "%s: null arguments", op);
    if (g->dtype < NSH_DTYPE_FLOAT16 || g->dtype > NSH_DTYPE_FLOAT32)
        return fail(NSH_ERR_INVALID, "%s: unsupported dtype code %d", op, g->dtype);
    if (g->B < 1 || g->L < 1 || g->Hq < 0 || g->Hk < 0 || g->Hq + g->Hk < 1)
        return fail(NSH_ERR_INVALID, "%s: empty tensor", op);
    constexpr int64_t kMost = int64_t(1) << 30;
    if (g->B > kMost || g->L > kMost || g->Hq > kMost || g->Hk > kMost || g->B * g->L > kMost ||
        g->B * g->L * std::max(g->Hq, g->Hk) > 2 * kMost - 1)
        return fail(NSH_ERR_INVALID, "%s: more than 2^31 rows", op);
    if (g->D < 1 || g->D > nsh::kNormMaxD || g->half < 0 || 2 * g->half > g->D)
        return fail(NSH_ERR_INVALID, "%s: the width must be 1..512 and hold the rotated pairs", op);
    if (g->rows < 0 || (g->half && (!g->cos || !g->sin)))
        return fail(NSH_ERR_INVALID, "%s: rotation without cos and sin", op);
    if ((g->Hq && !g->q) || (g->Hk && !g->k) ||
        (bwd ? (g->Hq && (!g->grad_q_out || !g->grad_q)) || (g->Hk && (!g->grad_k_out || !g->grad_k))
             : (g->Hq && !g->q_out) || (g->Hk && !g->k_out)))
        return fail(NSH_ERR_INVALID, "%s: null pointer argument", op);
    nsh::NormArgs a{};
    a.cos = g->cos, a.sin = g->sin, a.positions = g->positions, a.pos_stride = g->position_stride;
    a.L = static_cast<int>(g->L), a.D = static_cast<int>(g->D), a.half = static_cast<int>(g->half);
    a.interleaved = g->interleaved != 0;
    a.tokens = static_cast<uint32_t>(g->B * g->L);
    a.inv_d = 1.f / static_cast<float>(a.D), a.by_l = nsh::Divisor::of(static_cast<uint32_t>(g->L));
    a.rows = g->rows, a.eps = static_cast<float>(g->eps);
    nsh::NormSide &q = a.side[0], &k = a.side[1];
    q.x = g->q, q.w = g->q_weight, q.H = static_cast<int>(g->Hq);
    k.x = g->k, k.w = g->k_weight, k.H = static_cast<int>(g->Hk);
    for (auto& sd : a.side) sd.by_h = nsh::Divisor::of(static_cast<uint32_t>(std::max(sd.H, 1)));
    for (int i = 0; i < 3; ++i) q.xs[i] = g->q_stride[i], k.xs[i] = g->k_stride[i];
    if (bwd) {
        q.g = g->grad_q_out, k.g = g->grad_k_out, q.out = g->grad_q, k.out = g->grad_k;
        q.gw = g->grad_q_weight, k.gw = g->grad_k_weight;
        for (int i = 0; i < 3; ++i) q.gs[i] = g->gq_stride[i], k.gs[i] = g->gk_stride[i];
        if (q.gw || k.gw) {
            if (!g->workspace || g->workspace_bytes < nsh_norm_rotary_workspace_bytes(g))
                return fail(NSH_ERR_INVALID, "%s: workspace smaller than nsh_norm_rotary_workspace_bytes", op);
            a.partial = static_cast<float*>(g->workspace);
        }
    } else {
        q.out = g->q_out, k.out = g->k_out;
    }
    const bool vectors = nsh::norm_vectors(g, bwd);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (g->dtype) {
        case NSH_DTYPE_FLOAT16: return nsh::norm_dispatch<nsh::f16>(a, vectors, bwd, st);
        case NSH_DTYPE_BFLOAT16: return nsh::norm_dispatch<nsh::bf16>(a, vectors, bwd, st);
        default: return nsh::norm_dispatch<float>(a, vectors, bwd, st);
    }
}

extern "C" int nsh_norm_rotary_forward(const nsh_norm_rotary_args* g, void* stream) {
    return norm_rotary("norm_rotary_forward", g, false, stream);
}

extern "C" int nsh_norm_rotary_backward(const nsh_norm_rotary_args* g, void* stream) {
    return norm_rotary("norm_rotary_backward", g, true, stream);
}
