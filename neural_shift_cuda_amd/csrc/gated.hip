// gated.hip -- the gated projections' entries: checks, workspaces, and the passes
// around the products of gated.hpp (copies of rows that do not start on 16 bytes,
// dg and du with fp16's factor, the join of split sums).
#include <algorithm>
#include <cmath>

#include "gated.hpp"

namespace nsh {

NSH_GATED_ENTRIES(extern, f16, false)
NSH_GATED_ENTRIES(extern, bf16, false)
NSH_GATED_ENTRIES(extern, float, false)
NSH_GATED_ENTRIES(extern, float, true)
NSH_GATED_FEW_ROWS(extern, f16)
NSH_GATED_FEW_ROWS(extern, bf16)
NSH_GATED_FEW_ROWS(extern, float)

constexpr int kPassThreads = 256;

// Rows copied to a length of whole 16 bytes, zeros behind them: up to three matrices (1025 x 1001
// and two of 2731 x 1001 bf16, 13 MB each way: 6.7 us).
struct CopyArgs {
    struct Side {
        const void* from;
        void* to;
        int64_t rows, stride;  // stride in elements
    } side[3];
    int n, np;
};

template <typename T>
__global__ __launch_bounds__(kPassThreads) void gated_copy_kernel(CopyArgs a) {
    const CopyArgs::Side& s = a.side[blockIdx.y];
    const int each = a.np / kVec<T>;
    const int64_t all = s.rows * each, step = static_cast<int64_t>(gridDim.x) * kPassThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kPassThreads + threadIdx.x; i < all; i += step) {
        const int64_t row = i / each;
        const int c = static_cast<int>(i - row * each) * kVec<T>;
        const ux4 v = load_row<T, kShort>(static_cast<const T*>(s.from) + row * s.stride, c, a.n);
        *reinterpret_cast<ux4*>(static_cast<T*>(s.to) + row * a.np + c) = v;
    }
}

// The same into three planes of bf16 (2048 x 1024 and two of 2816 x 1024, 31 MB to 47: 15.4 us, 5.1
// TB/s).
__global__ __launch_bounds__(kPassThreads) void gated_split_kernel(CopyArgs a) {
    const CopyArgs::Side& s = a.side[blockIdx.y];
    const int each = a.np / 8;
    const int64_t all = s.rows * each, step = static_cast<int64_t>(gridDim.x) * kPassThreads, plane = s.rows * a.np;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kPassThreads + threadIdx.x; i < all; i += step) {
        const int64_t row = i / each;
        const int c = static_cast<int>(i - row * each) * 8;
        const float* from = static_cast<const float*>(s.from) + row * s.stride;
        float x[8], part[3][8];
        unpack<float>(load_row<float, kShort>(from, c, a.n), *reinterpret_cast<float(*)[4]>(&x[0]));
        unpack<float>(load_row<float, kShort>(from, c + 4, a.n), *reinterpret_cast<float(*)[4]>(&x[4]));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float p[3];
            split(x[e], p);
#pragma unroll
            for (int k = 0; k < 3; ++k) part[k][e] = p[k];
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)
            *reinterpret_cast<ux4*>(static_cast<bf16*>(s.to) + k * plane + row * a.np + c) = pack<bf16>(part[k]);
    }
}

struct SlopeArgs {
    const void* gh;
    int64_t gh_stride, first, rows, dgu_stride, dgu_plane;  // elements; rows from the first on
    char* kept;
    void* dgu;
    int F, Fp;
    uint32_t across;  // workgroups a row of blocks
    const float* scale;
};

// dg and du: a wave has 32 rows and 128 bytes of each, blocks of what was kept.  A stream: 8192 x
// 8192 bf16, 420 MB read and 268 written, 139 us, 4.9 TB/s; 4096 x 4096 fp16 37 us, 5.4.
template <typename T, bool PARTS>
__global__ __launch_bounds__(kPassThreads) void gated_slope_kernel(SlopeArgs a) {
    using E = typename Parts<T, PARTS>::E;
    constexpr int COLS = 128 / sizeof(T), BLOCKS = COLS / 32;
    using S = Stage<T, 32, COLS>;
    __shared__ __attribute__((aligned(256))) char stages[kPassThreads / 64][S::BYTES];
    char* stage = stages[wave_id()];
    const uint32_t down = blockIdx.x / a.across, across = blockIdx.x - down * a.across;
    const int c0 = (across * (kPassThreads / 64) + wave_id()) * COLS;
    if (c0 >= a.Fp) return;
    const float by = __is_same(T, f16) && a.scale ? a.scale[0] : 1.f;
    const int64_t m0 = a.first + static_cast<int64_t>(down) * 32, rows = a.rows - m0;
    Kept<T> k[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
        if (c0 + 32 * b < a.F) k[b].load(Kept<T>::block(a.kept, m0, c0 + 32 * b, a.F));
    S::load(stage, static_cast<const T*>(a.gh) + m0 * a.gh_stride + c0, a.gh_stride, rows, a.F - c0);
    wave_exchange();
    f32x16 d[BLOCKS], x[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) d[b] = S::get(stage, 0, b) * by;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const int left = a.F - c0 - 32 * b;
            x[b] = left > 0 ? d[b] * k[b].factor(side) : f32x16{};
            // (dh past F is 0, but the factors kept there are those of a product of x with
            // zeros, no numbers where x is infinite)
            if (left > 0 && left < 32) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r / 4) + 4 * static_cast<int>((threadIdx.x & 63) >> 5) + r % 4 >= left) x[b][r] = 0.f;
            }
        }
        using To = Stage<E, 32, COLS>;
        E* to = static_cast<E*>(a.dgu) + m0 * a.dgu_stride + side * a.Fp + c0;
        f32x16 parts[PARTS ? 3 : 1];
        if constexpr (PARTS) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float p[3];
                split(x[0][r], p);
                parts[0][r] = p[0], parts[1][r] = p[1], parts[2][r] = p[2];
            }
        }
#pragma unroll
        for (int n = 0; n < (PARTS ? 3 : 1); ++n) {
            wave_exchange();
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) To::put(stage, 0, b, PARTS ? parts[n] : x[b]);
            wave_exchange();
            To::store(stage, to + n * a.dgu_plane, a.dgu_stride, rows, COLS);
        }
    }
}

// fp16's numbers end at 2^-24 and lose bits from 2^-14 down, where the gradients of a
// mean loss are.  dg and du are multiplied by a power of two that brings the largest dh times
// the largest factor to 2^13 .. 2^15, and that the sums are divided by: what is rounded off,
// where it is not half a step, is then at most 2^-38 of that product, which may be far above
// the largest dg or du (a row of large factors whose dh is 0).
constexpr int kMostBlocks = 2048;

// Over rows of n, four parts of 16 bytes a lane at once (4096 x 4096: 10.4 us, 3.2 TB/s).
__global__ __launch_bounds__(kPassThreads) void gated_most_kernel(const f16* gh, int64_t stride, int64_t rows, int64_t n,
                                                                  float* out) {
    constexpr int kParts = 4;
    __shared__ float lds[kPassThreads / 64];
    float most = 0.f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y)
        for (int64_t c = static_cast<int64_t>(blockIdx.x) * (kPassThreads * 8 * kParts) + threadIdx.x * 8; c < n;
             c += static_cast<int64_t>(gridDim.x) * (kPassThreads * 8 * kParts)) {
            ux4 v[kParts];
            // (past the end the last numbers once more)
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const int64_t at = c + i * kPassThreads * 8;
                if (n < 8)
                    v[i] = load_bits(gh + row * stride, 0, static_cast<int>(n));
                else
                    __builtin_memcpy(&v[i], gh + row * stride + min(at, n - 8), 16);
            }
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                float d[8];
                unpack<f16>(v[i], d);
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(d[e]) < INFINITY ? fabsf(d[e]) : 0.f);
            }
        }
    most = workgroup_max<kPassThreads>(most, lds);
    if (threadIdx.x == 0) out[blockIdx.y * gridDim.x + blockIdx.x] = most;
}

__global__ __launch_bounds__(kPassThreads) void gated_scale_kernel(const float* gh, int n, const float* kept, int nk,
                                                                   float* scale) {
    __shared__ float lds[kPassThreads / 64];
    float x = 0.f, y = 0.f;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += kPassThreads) x = fmaxf(x, gh[i]);
#pragma unroll 8
    for (int i = threadIdx.x; i < nk; i += kPassThreads) y = fmaxf(y, kept[i]);
    x = workgroup_max<kPassThreads>(x, lds);
    y = workgroup_max<kPassThreads>(y, lds);
    if (threadIdx.x) return;
    int e = 0;
    if (x > 0.f && y > 0.f) {
        int ex, ey;
        frexpf(x, &ex);
        frexpf(y, &ey);  // x < 2^ex, y < 2^ey
        e = min(max(15 - ex - ey, -100), 100);
    }
    scale[0] = ldexpf(1.f, e);
    scale[1] = ldexpf(1.f, -e);
}

// The workgroups' sums, in order, four places of a row a lane, all of them asked for before
// the first is waited for (4096 x 1024 fp16 of two sums: 8.2 us, 5.1 TB/s).
template <typename T, int SPLITS>
__global__ __launch_bounds__(kPassThreads) void gated_join_kernel(const float* part, int64_t rows, int K, int Kq, T* out) {
    const int c = (blockIdx.x * kPassThreads + threadIdx.x) * 4;
    if (c >= K) return;
    for (int64_t m = blockIdx.y; m < rows; m += gridDim.y) {
        float s[4] = {}, v[SPLITS][4];
#pragma unroll
        for (int k = 0; k < SPLITS; ++k) load_acc<float, 4>(part + (k * rows + m) * Kq + c, v[k]);
#pragma unroll
        for (int k = 0; k < SPLITS; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[k][e];
        T e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = from_acc<T>(s[k]);
        if (c + 4 <= K) {
            __builtin_memcpy(out + m * K + c, e, sizeof(e));
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (c + k < K) out[m * K + c + k] = e[k];
        }
    }
}

template <typename T>
int gated_join(const GatedArgs& a, int splits, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(nsh_host::ceil_div(a.K, 4 * kPassThreads)),
                    static_cast<unsigned>(std::min<int64_t>(a.rows, 32768)));
    auto go = [&](auto n) {
        gated_join_kernel<T, decltype(n)::value><<<grid, kPassThreads, 0, st>>>(a.part, a.rows, a.K, a.Kq, static_cast<T*>(a.dx));
    };
    switch (splits) {
        case 2: go(std::integral_constant<int, 2>{}); break;
        case 3: go(std::integral_constant<int, 3>{}); break;
        case 4: go(std::integral_constant<int, 4>{}); break;
        case 6: go(std::integral_constant<int, 6>{}); break;
        case 8: go(std::integral_constant<int, 8>{}); break;
        case 12: go(std::integral_constant<int, 12>{}); break;
        case 16: go(std::integral_constant<int, 16>{}); break;
        default: return nsh_host::fail(NSH_ERR_INVALID, "gated_linear_backward: no join of %d sums", splits);
    }
    return nsh_host::check_launch("gated_linear_backward");
}

}  // namespace nsh

using nsh_host::ceil_div;
using nsh_host::fail;

namespace {

constexpr int64_t kWidest = int64_t(1) << 20;
constexpr int64_t kStep = int64_t(1) << 23;  // bytes from a row to the next that a panel's 32-bit offsets take

struct Plan {
    bool few, parts;       // up to 64 rows; fp32 by bf16 products
    int64_t esz, Kp, Fp;   // esz: bytes of the products' elements
    bool copy[3];          // x, gate, up
    int64_t copies[3];     // offsets in the workspace
    int64_t planes;        // bytes of dgu's parts
    int64_t dgu, scale, most, part, bytes;
    nsh::Cut cut;
};

int64_t up(int64_t v, int64_t to) { return ceil_div(v, to) * to; }

nsh::Cut cut_of(const nsh_gated_linear_args* g, bool bwd, nsh::Means by) {
    return bwd ? nsh::gradient_cut(g->rows, g->K, g->F, by, g->grad_x != nullptr, g->grad_gate || g->grad_up)
               : nsh::forward_cut(g->rows, g->F, g->K, by);
}

Plan plan_of(const nsh_gated_linear_args* g, bool bwd) {
    Plan p{};
    const bool wide = g->dtype == NSH_DTYPE_FLOAT32;
    p.few = !bwd && !g->kept && g->rows <= nsh::kFewRows;
    if (!p.few) p.cut = cut_of(g, bwd, {wide, 1});
    if (wide && !p.few) {
        // against the time of taking the parts: 4 bytes read, 6 written and read once more
        nsh::Cut parts = cut_of(g, bwd, {false, 6});
        const double taken = parts.time + 4 + static_cast<double>((g->rows + 2 * g->F) * g->K) * 10 / 3.5e6;
        p.parts = parts.time > 0 && (p.cut.time == 0 || taken < p.cut.time);
        if (p.parts) p.cut = parts;
    }
    p.esz = wide && !p.parts ? 4 : 2;
    const int64_t vec = 16 / p.esz;
    p.Kp = up(g->K, vec), p.Fp = up(g->F, 64);
    const void* at[3] = {g->x, g->gate_weight, g->up_weight};
    const int64_t stride[3] = {g->x_stride, g->gate_stride, g->up_stride}, rows[3] = {g->rows, g->F, g->F};
    for (int i = 0; i < 3; ++i) {
        // (a single row has no step to the next)
        const bool steps = rows[i] == 1 || (stride[i] % vec == 0 && stride[i] >= g->K && stride[i] * p.esz <= kStep);
        p.copy[i] = p.parts || g->K % vec != 0 || !nsh_host::aligned(at[i], 16) || !steps;
        p.copies[i] = p.bytes;
        if (p.copy[i]) p.bytes += up(rows[i] * p.Kp * p.esz * (p.parts ? 3 : 1), 256);
    }
    if (!bwd) return p;
    p.dgu = p.bytes;
    p.planes = g->rows * (2 * p.Fp * p.esz + 128);
    p.bytes += up(p.planes * (p.parts ? 3 : 1), 256);
    p.scale = p.bytes, p.bytes += 256;
    p.most = p.bytes, p.bytes += up(nsh::kMostBlocks * 4, 256);
    p.part = p.bytes;
    if (p.cut.splits > 1) p.bytes += up(p.cut.splits * g->rows * up(g->K, 4) * 4, 256);
    return p;
}

// (fp16: of the forward that keeps what the backward needs)
int64_t forward_blocks(const nsh_gated_linear_args* g) { return cut_of(g, false, {false, 1}).tiles(); }

int64_t kept_blocks(const nsh_gated_linear_args* g) {
    const int64_t each = g->dtype == NSH_DTYPE_FLOAT32    ? nsh::Kept<float>::BYTES
                         : g->dtype == NSH_DTYPE_BFLOAT16 ? nsh::Kept<nsh::bf16>::BYTES
                                                          : nsh::Kept<nsh::f16>::BYTES;
    return ceil_div(g->rows, 32) * ceil_div(g->F, 32) * each;
}

int check(const char* op, const nsh_gated_linear_args* g, bool bwd) {
    if (!g) return fail(NSH_ERR_INVALID, "%s: null arguments", op);
    if (g->dtype < NSH_DTYPE_FLOAT16 || g->dtype > NSH_DTYPE_FLOAT32)
        return fail(NSH_ERR_INVALID, "%s: unsupported dtype code %d", op, g->dtype);
    if (g->rows < 1 || g->K < 1 || g->F < 1) return fail(NSH_ERR_INVALID, "%s: empty tensor", op);
    if (g->K > kWidest || g->F > kWidest || g->rows > (int64_t(1) << 30))
        return fail(NSH_ERR_INVALID, "%s: width or hidden size above 2^20, or more than 2^30 rows", op);
    if (g->activation < NSH_ACTIVATION_SILU || g->activation > NSH_ACTIVATION_SIGMOID)
        return fail(NSH_ERR_INVALID, "%s: unknown activation code %d", op, g->activation);
    if (!g->x || !g->gate_weight || !g->up_weight ||
        (bwd ? !g->kept || !g->grad_h || (!g->grad_x && !g->grad_gate && !g->grad_up) : !g->h))
        return fail(NSH_ERR_INVALID, "%s: null pointer argument", op);
    if (g->kept && !nsh_host::aligned(g->kept, 16)) return fail(NSH_ERR_INVALID, "%s: misaligned kept", op);
    return NSH_OK;
}

template <typename T>
int copy_rows(const nsh_gated_linear_args* g, const Plan& p, nsh::GatedArgs& a, char* ws, hipStream_t st) {
    nsh::CopyArgs c{};
    int n = 0;
    int64_t most = 0;
    const void** at[3] = {&a.x, &a.wg, &a.wu};
    uint32_t* stride[3] = {&a.x_stride, &a.wg_stride, &a.wu_stride};
    int64_t* plane[3] = {&a.x_plane, &a.wg_plane, &a.wu_plane};
    const int64_t steps[3] = {g->x_stride, g->gate_stride, g->up_stride}, rows[3] = {g->rows, g->F, g->F};
    for (int i = 0; i < 3; ++i) {
        *stride[i] = static_cast<uint32_t>(rows[i] == 1 ? p.Kp * p.esz : steps[i] * p.esz);
        if (!p.copy[i]) continue;
        c.side[n++] = {*at[i], ws + p.copies[i], rows[i], steps[i]};
        *at[i] = ws + p.copies[i];
        *stride[i] = static_cast<uint32_t>(p.Kp * p.esz);
        *plane[i] = rows[i] * p.Kp * p.esz;
        most = std::max(most, rows[i] * (p.Kp * p.esz / 16));
    }
    if (!n) return NSH_OK;
    c.n = static_cast<int>(g->K), c.np = static_cast<int>(p.Kp);
    const int64_t blocks = std::min<int64_t>(ceil_div(most, nsh::kPassThreads), nsh_host::compute_units() * 16);
    const dim3 grid(static_cast<unsigned>(blocks), n);
    if (p.parts)
        nsh::gated_split_kernel<<<grid, nsh::kPassThreads, 0, st>>>(c);
    else
        nsh::gated_copy_kernel<T><<<grid, nsh::kPassThreads, 0, st>>>(c);
    return nsh_host::check_launch("gated_linear");
}

template <typename T, bool PARTS>
int backward(const nsh_gated_linear_args* g, const Plan& p, nsh::GatedArgs a, char* ws, hipStream_t st) {
    float* scale = nullptr;
    if constexpr (__is_same(T, nsh::f16)) {
        scale = reinterpret_cast<float*>(ws + p.scale);
        float* most = reinterpret_cast<float*>(ws + p.most);
        const bool flat = g->gh_stride == g->F;
        const int64_t rows = flat ? 1 : g->rows, cols = flat ? g->rows * g->F : g->F;
        const int64_t x = std::min<int64_t>(ceil_div(cols, nsh::kPassThreads * 32), nsh::kMostBlocks);
        const int64_t y = std::min<int64_t>(rows, nsh::kMostBlocks / x), n = x * y;
        nsh::gated_most_kernel<<<dim3(static_cast<unsigned>(x), static_cast<unsigned>(y)), nsh::kPassThreads, 0, st>>>(
            static_cast<const nsh::f16*>(g->grad_h), g->gh_stride, rows, cols, most);
        nsh::gated_scale_kernel<<<1, nsh::kPassThreads, 0, st>>>(most, static_cast<int>(n),
                                                                 reinterpret_cast<const float*>(a.kept + kept_blocks(g)),
                                                                 static_cast<int>(forward_blocks(g)), scale);
    }
    a.scale = scale, a.dgu = ws + p.dgu;
    a.dgu_plane = p.planes;
    const uint32_t across = static_cast<uint32_t>(ceil_div(a.Fp, nsh::kPassThreads / 64 * 128 / sizeof(T)));
    nsh::SlopeArgs s{g->grad_h, g->gh_stride, 0, g->rows, 2 * p.Fp + 128 / p.esz, p.planes / p.esz, a.kept, a.dgu, a.F, a.Fp, across, scale};
    const int64_t most = std::max((1 << 20) / across, 1u);  // rows of blocks a launch
    for (; s.first < g->rows; s.first += most * 32) {
        const int64_t downs = std::min(ceil_div(g->rows - s.first, 32), most);
        nsh::gated_slope_kernel<T, PARTS><<<static_cast<unsigned>(across * downs), nsh::kPassThreads, 0, st>>>(s);
    }
    a.Kq = static_cast<int>(up(g->K, 4));
    a.part = p.cut.splits > 1 ? reinterpret_cast<float*>(ws + p.part) : nullptr;
    const int rc = nsh::gated_gradients<T, PARTS>(a, p.cut, st);
    if (rc != NSH_OK || !a.part) return rc;
    return nsh::gated_join<T>(a, p.cut.splits, st);
}

template <typename T>
int run(const nsh_gated_linear_args* g, const Plan& p, bool bwd, hipStream_t st) {
    nsh::GatedArgs a{};
    char* ws = static_cast<char*>(g->workspace);
    a.x = g->x, a.wg = g->gate_weight, a.wu = g->up_weight;
    a.rows = g->rows, a.K = static_cast<int>(g->K), a.F = static_cast<int>(g->F);
    a.Kp = static_cast<int>(p.Kp), a.Fp = static_cast<int>(p.Fp);
    a.activation = g->activation - NSH_ACTIVATION_SILU;
    a.h = g->h, a.dx = g->grad_x, a.dwg = g->grad_gate, a.dwu = g->grad_up;
    const int rc = copy_rows<T>(g, p, a, ws, st);
    if (rc != NSH_OK) return rc;
    a.kept = static_cast<char*>(g->kept);
    if constexpr (sizeof(T) == 4)
        if (p.parts) return bwd ? backward<T, true>(g, p, a, ws, st) : nsh::gated_forward<T, true>(a, p.cut, st);
    if (bwd) return backward<T, false>(g, p, a, ws, st);
    if (p.few) return nsh::gated_few_rows<T>(a, st);
    if (__is_same(T, nsh::f16) && a.kept) a.most = reinterpret_cast<float*>(a.kept + kept_blocks(g));
    return nsh::gated_forward<T, false>(a, p.cut, st);
}

int gated_linear(const char* op, const nsh_gated_linear_args* g, bool bwd, void* stream) {
    const int rc = check(op, g, bwd);
    if (rc != NSH_OK) return rc;
    const Plan p = plan_of(g, bwd);
    if (!p.few && p.cut.time == 0) return fail(NSH_ERR_INVALID, "%s: more tiles than one launch takes", op);
    if (p.bytes > 0 && (!g->workspace || g->workspace_bytes < p.bytes))
        return fail(NSH_ERR_INVALID, "%s: workspace smaller than nsh_gated_linear_workspace_bytes", op);
    if (p.bytes > 0 && !nsh_host::aligned(g->workspace, 16)) return fail(NSH_ERR_INVALID, "%s: misaligned workspace", op);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (g->dtype) {
        case NSH_DTYPE_FLOAT16: return run<nsh::f16>(g, p, bwd, st);
        case NSH_DTYPE_BFLOAT16: return run<nsh::bf16>(g, p, bwd, st);
        default: return run<float>(g, p, bwd, st);
    }
}

}  // namespace

extern "C" int64_t nsh_gated_linear_workspace_bytes(const nsh_gated_linear_args* g, int backward) {
    if (!g || g->rows < 1 || g->K < 1 || g->F < 1) return -1;
    return plan_of(g, backward != 0).bytes;
}

extern "C" int64_t nsh_gated_linear_kept_bytes(const nsh_gated_linear_args* g) {
    if (!g || g->rows < 1 || g->K < 1 || g->F < 1) return -1;
    return kept_blocks(g) + (g->dtype == NSH_DTYPE_FLOAT16 ? forward_blocks(g) * 4 : 0);
}

extern "C" int nsh_gated_linear_forward(const nsh_gated_linear_args* g, void* stream) {
    return gated_linear("gated_linear_forward", g, false, stream);
}

extern "C" int nsh_gated_linear_backward(const nsh_gated_linear_args* g, void* stream) {
    return gated_linear("gated_linear_backward", g, true, stream);
}
