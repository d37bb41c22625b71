// gated.hpp -- the gated projections of a feed-forward and their gradients.
//
//   g = x Wg^T,  u = x Wu^T,  h = act(g) u
//   dg = dh u act'(g),  du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// Three products over panels (panels.hpp).  Forward: both weights' rows stand side by
// side in one panel, so a lane has g and u of the same place and the activation and
// the product never leave its registers.  Training keeps u act'(g) and act(g), the
// factors that dh takes, finer than the type (struct Kept): rounded to it they would bring
// a third rounding next to dg's and the result's (errors of the gradients 1.7 times the
// result's own rounding instead of 1.4).  Backward: one pass forms dg and du, as one matrix
// (rows, 2, Fp) of the operands' type (a matrix instruction takes no other; each is off by
// half a step, of the size of the result's own rounding and not shared by a sum's
// terms), then dx takes both in one sum over 2 F, and one product gives both weights'
// gradients.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "panels.hpp"

namespace nsh {

struct GatedArgs {
    const void *x, *wg, *wu;
    uint32_t x_stride, wg_stride, wu_stride;  // bytes from row to row
    int64_t x_plane, wg_plane, wu_plane, dgu_plane;  // bytes from a part to the next (struct Parts)
    int64_t rows;
    int K, F, Kp, Fp;     // Kp: columns of x and the weights as they lie; Fp: F in whole panels
    int activation;
    void* h;
    char* kept;            // blocks of 32 x 32 (struct Kept), or NULL
    float* most;           // fp16 training: largest factor of every workgroup
    void* dgu;             // (rows, 2, Fp) and a panel's width of nothing
    const float* scale;    // fp16: what dgu was multiplied by, and its inverse
    void *dx, *dwg, *dwu;
    float* part;           // (splits, rows, Kq): sums of dx that a second launch joins, Kq a multiple of 4
    int Kq;
    int tiles_m, tiles_n;  // of h, or of dx
    int splits;            // workgroups that share a tile of dx
    int weight_m, weight_n;  // tiles of the weights' gradients, both sides
    int first;             // workgroups of the part that comes first
    bool weights_first;
};

enum Activation { kSilu, kGelu, kGeluTanh, kRelu, kSigmoid };

// The activation at g and its slope there, by instructions of one place in the last or so, a
// third of the library functions' time.  An exponential's argument is rounded once: the result
// is off by 2^-24 of the argument's size, 1e-6 of itself for silu at -20, where the sums'
// roundings are as much.
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * x));
}
template <Activation KIND>
__device__ __forceinline__ float2 activate(float g) {
    if constexpr (KIND == kSilu) {
        const float s = sigmoid(g);
        return make_float2(g * s, s * fma_acc(g, 1.f - s, 1.f));
    } else if constexpr (KIND == kGelu) {
        // Phi(-|g|) = exp(-g^2 / 2) erfcx(|g| / sqrt 2) / 2, whose small values keep their
        // places; erfcx(z) / t as a polynomial in t = 1 / (1 + 0.4 z), by least squares with
        // weights towards the smallest largest error: 4e-8 of it, 1e-7 with fp32's roundings
        const float z = fabsf(g), t = __builtin_amdgcn_rcpf(fma_acc(0.28284271247461901f, z, 1.f));
        const float e = __builtin_amdgcn_exp2f(z * z * (-0.5f * kLog2e));
        float p = -0.0292149931f;
        p = fma_acc(p, t, 0.140446082f);
        p = fma_acc(p, t, -0.235525861f);
        p = fma_acc(p, t, 0.137559712f);
        p = fma_acc(p, t, -0.0468939133f);
        p = fma_acc(p, t, 0.0839158222f);
        p = fma_acc(p, t, 0.119008467f);
        p = fma_acc(p, t, 0.17173925f);
        p = fma_acc(p, t, 0.207613736f);
        p = fma_acc(p, t, 0.225675866f);
        p = fma_acc(p, t, 0.225675836f);
        const float tail = 0.5f * e * (p * t), below = g > 0.f ? 1.f - tail : tail;
        return make_float2(g * below, fma_acc(g * 0.3989422804014327f, e, below));
    } else if constexpr (KIND == kGeluTanh) {
        constexpr float a = 1.5957691216057308f, b = 0.044715f;  // 2 sqrt(2 / pi)
        const float s = sigmoid(a * g * fma_acc(b * g, g, 1.f));
        // (beyond 20 either way s is 1 or 0 to the last place; g's square would be infinite, and 0
        // times it no number)
        const float near = fminf(fmaxf(g, -20.f), 20.f);
        return make_float2(g * s, fma_acc(near * s * (1.f - s), a * fma_acc(3.f * b * near, near, 1.f), s));
    } else if constexpr (KIND == kRelu) {
        return g > 0.f ? make_float2(g, 1.f) : make_float2(g == g ? 0.f : g, 0.f);
    } else {
        // (by -|g|: 1 - s would be nothing but the last place of s where that is near 1)
        const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(g)), r = __builtin_amdgcn_rcpf(1.f + e);
        return make_float2(g < 0.f ? e * r : r, e * r * r);
    }
}

// v and slope of N places.
template <int N, typename V>
__device__ __forceinline__ void activate(int kind, const V& g, V& v, V& slope) {
    auto all = [&](auto one) {
#pragma unroll
        for (int r = 0; r < N; ++r) {
            const float2 f = one(g[r]);
            v[r] = f.x, slope[r] = f.y;
        }
    };
    switch (kind) {
        case kSilu: return all([](float x) { return activate<kSilu>(x); });
        case kGelu: return all([](float x) { return activate<kGelu>(x); });
        case kGeluTanh: return all([](float x) { return activate<kGeluTanh>(x); });
        case kRelu: return all([](float x) { return activate<kRelu>(x); });
        default: return all([](float x) { return activate<kSigmoid>(x); });
    }
}

// The largest magnitude of a lane's 16 numbers: an infinity says nothing of the others.
__device__ __forceinline__ float largest(const f32x16& v) {
    float most = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(v[r]));
    if (!(most < INFINITY)) {
        most = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(v[r]) < INFINITY ? fabsf(v[r]) : 0.f);
    }
    return most;
}

// What training keeps of a block of 32 x 32 places: the two factors as the lanes have
// them, so that every store and load is 1 KB in one piece (rows of their own, 16 bytes a
// lane apart, took the forward 8192 x 2048 -> 8192 from 480 to 1017 us).
//   bf16: fp16 times a power of two of each lane's largest, which leaves 11 bits of all
//     that is not below 2^-28 of it, and of the rest what is 2^-39 of it
//   fp16: the upper 24 bits of fp32
//   fp32: itself
template <typename T>
struct Kept {
    static constexpr int BYTES = sizeof(T) == 4 ? 8192 : __is_same(T, bf16) ? 4096 + 256 : 6144;

    static __device__ __forceinline__ char* block(char* kept, int64_t m, int c, int F) {
        return kept + ((m >> 5) * ((F + 31) >> 5) + (c >> 5)) * BYTES;
    }
    static __device__ __forceinline__ ux4* part(char* at, int n) {
        return reinterpret_cast<ux4*>(at + n * 1024) + (threadIdx.x & 63);
    }

    // The exponent field of the largest number of a lane's 16 (15 at the least).
    static __device__ __forceinline__ uint32_t field(const f32x16& v) { return max(__float_as_uint(largest(v)) >> 23, 15u); }

    static __device__ __forceinline__ void store(char* at, const f32x16& s, const f32x16& h) {
        const f32x16* both[2] = {&s, &h};
        uint32_t fields[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const f32x16& v = *both[n];
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *part(at, 4 * n + q) = __builtin_bit_cast(ux4, (f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]}));
            } else if constexpr (__is_same(T, bf16)) {
                fields[n] = field(v);
                const f32x16 x = v * __uint_as_float((268u - fields[n]) << 23);  // to 2^14 .. 2^15
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const f32x8 y = {x[8 * q], x[8 * q + 1], x[8 * q + 2], x[8 * q + 3],
                                     x[8 * q + 4], x[8 * q + 5], x[8 * q + 6], x[8 * q + 7]};
                    *part(at, 2 * n + q) = __builtin_bit_cast(ux4, __builtin_convertvector(y, f16x8));
                }
            } else {
                uint32_t b[16];
#pragma unroll
                for (int r = 0; r < 16; ++r)  // (no carry out of what is no number)
                    b[r] = v[r] == v[r] ? __float_as_uint(v[r]) + 0x80u : 0x7fc00000u;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    ux4 x;  // upper halves of two
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __builtin_amdgcn_perm(b[8 * q + 2 * e + 1], b[8 * q + 2 * e], 0x07060302);
                    *part(at, 2 * n + q) = x;
                }
                ux4 x;  // second bytes of four
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[4 * e + 3], b[4 * e + 2], 0x05010501),
                                                 __builtin_amdgcn_perm(b[4 * e + 1], b[4 * e], 0x05010501), 0x05040100);
                *part(at, 4 + n) = x;
            }
        }
        if constexpr (__is_same(T, bf16))
            reinterpret_cast<uint32_t*>(at + 4096)[threadIdx.x & 63] = fields[0] | fields[1] << 16;
    }

    // As loaded, and its numbers.
    ux4 bits[BYTES / 1024];
    uint32_t fields;
    __device__ __forceinline__ void load(char* at) {
#pragma unroll
        for (int n = 0; n < BYTES / 1024; ++n) bits[n] = *part(at, n);
        if constexpr (__is_same(T, bf16)) fields = reinterpret_cast<const uint32_t*>(at + 4096)[threadIdx.x & 63];
    }
    __device__ __forceinline__ f32x16 factor(int n) const {
        f32x16 v;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] = __uint_as_float(bits[4 * n + r / 4][r % 4]);
        } else if constexpr (__is_same(T, bf16)) {
            const uint32_t f = n ? fields >> 16 : fields & 0xffffu;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const f32x8 x = __builtin_convertvector(__builtin_bit_cast(f16x8, bits[2 * n + q]), f32x8);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * q + e] = x[e];
            }
            v *= __uint_as_float((f - 14u) << 23);
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t hi = bits[2 * n + r / 8][r / 2 % 4], lo = bits[4 + n][r / 4] >> 8 * (r % 4) & 0xffu;
                v[r] = __uint_as_float((r % 2 ? hi & 0xffff0000u : hi << 16) | lo << 8);
            }
        }
        return v;
    }
};

// h of the lane's 16 places from column c on, and what the gradients need.
template <typename T>
__device__ __forceinline__ f32x16 gate_block(const GatedArgs& a, int64_t m, int c, const f32x16& g, const f32x16& u, float& most) {
    f32x16 h, s;
    activate<16>(a.activation, g, h, s);
    if (a.kept && (m & ~int64_t(31)) < a.rows && c < a.F) {
        s *= u;
        Kept<T>::store(Kept<T>::block(a.kept, m, c, a.F), s, h);
        if constexpr (__is_same(T, f16)) most = fmaxf(most, fmaxf(largest(s), largest(h)));
    }
    return h * u;
}

// fp32 by bf16 products: a number is the sum of three of bf16, 24 bits in all, and six of the
// products of parts are summed, the smallest first, by the same panels and six times as many.
// What is left out, a second part by a third and a third by a third, is 4e-8 of a product on
// average and below 2^-21 at most.  A product of fp32 matrices takes 16 times as long as one
// of bf16.  (2048 x 1024 -> 2816: forward 138 us, 219 by fp32 products, gradients 266, 407; the
// matrix units are busy for 46 and 49%, with 176 and 216 tiles for 256 CUs.)
template <typename T, bool PARTS>
struct Parts {
    using E = std::conditional_t<PARTS, bf16, T>;
    static constexpr int N = PARTS ? 6 : 1;
    // which parts (0: the largest) of the two sides the n-th product takes
    static __device__ __forceinline__ int first(int n) { return PARTS ? 0x052 >> 2 * n & 3 : 0; }
    static __device__ __forceinline__ int second(int n) { return PARTS ? 0x118 >> 2 * n & 3 : 0; }
};

// x as such a sum, eight bits at a time and all of x's sign, so that six products of parts have
// the sign of the whole: what is beyond fp32 is one infinity, as in fp32.  (Rounded, the parts
// leave out 6e-9, but a second one may have the other sign, and infinities of both make a NaN of
// a finite 1e30 * 1e12.)  What is no number is in the last part, which meets the other side's
// first alone: 1 for an infinity there, with its sign.
__device__ __forceinline__ void split(float x, float (&part)[3]) {
    const bool number = fabsf(x) < INFINITY;
    const float v = number ? x : copysignf(1.f, x);
    const auto upper = [](float y) { return __uint_as_float(__float_as_uint(y) & 0xffff0000u); };
    part[0] = upper(v);
    const float rest = v - part[0];
    part[1] = upper(rest);
    part[2] = number ? rest - part[1] : x;
}

// Bytes of a row of dgu: not a power of two, which would have every row's same place in
// one channel of the caches.
template <typename E>
__device__ __forceinline__ uint32_t dgu_stride(const GatedArgs& a) {
    return 2 * a.Fp * static_cast<uint32_t>(sizeof(E)) + 128;
}

template <typename T, bool PARTS, int BM, int BN, int WAVES_M, int WAVES_N, int KB>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void gated_forward_kernel(GatedArgs a) {
    using Of = Parts<T, PARTS>;
    using E = typename Of::E;
    using P = Product<E, BM, BN, WAVES_M, WAVES_N, KB, kAlong, kAlong, true>;
    // (panels of 24 KB: a third leaves room for two workgroups a CU; 100 rows, 2048 -> 5504: 30
    // us with two, 23 with three)
    constexpr bool THREE = BM < 128;
    __shared__ __attribute__((aligned(1024))) char b0[P::BYTES], b1[P::BYTES], b2[THREE ? P::BYTES : 1];
    const TileOrder t(blockIdx.x, gridDim.x, a.tiles_m, a.tiles_n, 8);
    const int64_t m0 = static_cast<int64_t>(t.m) * BM;
    const int c0 = t.n * (BN / 2), wave = wave_id();
    typename P::FirstPanel gate, up;
    typename P::SecondPanel rows;
    gate.init(a.wg_stride);
    up.init(a.wu_stride);
    rows.init(a.x_stride);
    const char* x = static_cast<const char*>(a.x) + m0 * a.x_stride;
    const char* wg = static_cast<const char*>(a.wg) + static_cast<int64_t>(c0) * a.wg_stride;
    const char* wu = static_cast<const char*>(a.wu) + static_cast<int64_t>(c0) * a.wu_stride;
    const int64_t wide = static_cast<int64_t>(a.Kp) * sizeof(E);
    const int left_m = static_cast<int>(min(a.rows - m0, int64_t(BM)));
    P p;
    p.init();
    const int n = (a.Kp + P::BK - 1) / P::BK * Of::N;
    const auto load = [&](int i, char* f, char* s) {
        const int block = i / Of::N, term = i % Of::N;
        const int64_t at = static_cast<int64_t>(block) * KB;
        const int left_f = i < n ? a.F - c0 : 0;
        gate.load(f, wg + Of::first(term) * a.wg_plane + at, a.wg_stride, left_f, wide - at, wave);
        up.load(f + P::FIRST_BYTES / 2, wu + Of::first(term) * a.wu_plane + at, a.wu_stride, left_f, wide - at, wave);
        rows.load(s, x + Of::second(term) * a.x_plane + at, a.x_stride, i < n ? left_m : 0, wide - at, wave);
    };
    if constexpr (THREE)
        p.run(n, b0, b1, b2, load);
    else
        p.run(n, b0, b1, load);
    float most = 0.f;
    const int64_t m = m0 + P::wave_m() * P::WM;
    const int c = c0 + P::column(0);
    __syncthreads();  // the panels' place is free
    store_tile<T, P::WM, P::WN / 2>(P::stage(b0, b1), static_cast<T*>(a.h) + m * a.F + c, a.F, a.rows - m, a.F - c,
                                    [&](int i, int b) {
                                        return gate_block<T>(a, m0 + P::row(i), c0 + P::column(b), p.acc[i][b],
                                                             p.acc[i][b + P::NB / 2], most);
                                    });
    if constexpr (__is_same(T, f16)) {
        if (!a.most) return;
        __syncthreads();
        most = workgroup_max<P::NT>(most, reinterpret_cast<float*>(b0));
        if (threadIdx.x == 0) a.most[blockIdx.x] = most;
    }
}

// dx: over the hidden columns of dg, then of du.
template <typename T, typename Of, typename P>
__device__ __forceinline__ void input_gradient(const GatedArgs& a, uint32_t id, char (&b0)[P::BYTES], char (&b1)[P::BYTES]) {
    using E = typename P::T;
    const uint32_t tiles = static_cast<uint32_t>(a.tiles_m) * a.tiles_n;
    const int split = TileOrder::uniform(id / tiles);
    const TileOrder t(id - split * tiles, tiles, a.tiles_m, a.tiles_n, 8);
    const int64_t m0 = static_cast<int64_t>(t.m) * P::BM;
    const int64_t c0 = static_cast<int64_t>(t.n) * P::BN;
    const int wave = wave_id();
    typename P::FirstPanel gate, up;
    typename P::SecondPanel rows;
    gate.init(a.wg_stride);
    up.init(a.wu_stride);
    const uint32_t stride = dgu_stride<E>(a);
    rows.init(stride);
    const char* d = static_cast<const char*>(a.dgu) + m0 * stride;
    const char* wg = static_cast<const char*>(a.wg) + c0 * static_cast<int64_t>(sizeof(E));
    const char* wu = static_cast<const char*>(a.wu) + c0 * static_cast<int64_t>(sizeof(E));
    const int left_m = static_cast<int>(min(a.rows - m0, int64_t(P::BM)));
    const int64_t left_c = (a.Kp - c0) * static_cast<int64_t>(sizeof(E));
    const int half = a.Fp / P::BK, all = 2 * half * Of::N;
    const int begin = TileOrder::uniform(all * static_cast<uint32_t>(split) / a.splits);
    const int end = TileOrder::uniform(all * static_cast<uint32_t>(split + 1) / a.splits);
    P p;
    p.init();
    p.run(end - begin, b0, b1, [&](int i, char* f, char* s) {
        const int block = (begin + i) / Of::N, term = (begin + i) % Of::N;
        const bool one = block < half;
        const int64_t row = static_cast<int64_t>(one ? block : block - half) * P::BK;
        const uint32_t step = one ? a.wg_stride : a.wu_stride;
        const int64_t plane = Of::first(term) * (one ? a.wg_plane : a.wu_plane);
        P::FirstPanel::either(one, gate, up).load(f, (one ? wg : wu) + plane + row * step, step, a.F - static_cast<int>(row), left_c, wave);
        rows.load(s, d + Of::second(term) * a.dgu_plane + static_cast<int64_t>(block) * P::KB, stride, left_m, P::KB, wave);
    });
    const float by = __is_same(T, f16) && a.scale ? a.scale[1] : 1.f;
    const int64_t m = m0 + P::wave_m() * P::WM, c = c0 + P::column(0);
    __syncthreads();  // the panels' place is free
    char* stage = P::stage(b0, b1);
    const auto value = [&](int i, int b) { return p.acc[i][b] * by; };
    if (a.part)
        store_tile<float, P::WM, P::WN>(stage, a.part + (split * a.rows + m) * a.Kq + c, a.Kq, a.rows - m, a.K - c, value);
    else
        store_tile<T, P::WM, P::WN>(stage, static_cast<T*>(a.dx) + m * a.K + c, a.K, a.rows - m, a.K - c, value);
}

// Both weights' gradients: tiles of hidden rows of the one, then of the other.
template <typename T, typename Of, typename P>
__device__ __forceinline__ void weight_gradient(const GatedArgs& a, uint32_t id, char (&b0)[P::BYTES], char (&b1)[P::BYTES]) {
    using E = typename P::T;
    const int each = a.weight_m / 2;
    const TileOrder t(id, static_cast<uint32_t>(a.weight_m) * a.weight_n, a.weight_m, a.weight_n, 8);
    const int side = t.m >= each;
    T* out = static_cast<T*>(side ? a.dwu : a.dwg);
    if (!out) return;
    const int f_first = (side ? t.m - each : t.m) * P::BM;
    const int64_t c0 = static_cast<int64_t>(t.n) * P::BN;
    const int wave = wave_id();
    typename P::FirstPanel in;
    typename P::SecondPanel d;
    in.init(a.x_stride);
    const uint32_t stride = dgu_stride<E>(a);
    d.init(stride);
    const char* x = static_cast<const char*>(a.x) + c0 * static_cast<int64_t>(sizeof(E));
    const char* dgu = static_cast<const char*>(a.dgu) + (static_cast<int64_t>(side) * a.Fp + f_first) * static_cast<int64_t>(sizeof(E));
    const int64_t left_c = (a.Kp - c0) * static_cast<int64_t>(sizeof(E));
    const int64_t left_f = (static_cast<int64_t>(a.Fp) - f_first) * static_cast<int64_t>(sizeof(E));
    P p;
    p.init();
    p.run(static_cast<int>((a.rows + P::BK - 1) / P::BK) * Of::N, b0, b1, [&](int i, char* f, char* s) {
        const int64_t at = static_cast<int64_t>(i / Of::N) * P::BK;
        const int term = i % Of::N, left = static_cast<int>(min(a.rows - at, int64_t(P::BK)));
        in.load(f, x + Of::first(term) * a.x_plane + at * a.x_stride, a.x_stride, left, left_c, wave);
        d.load(s, dgu + Of::second(term) * a.dgu_plane + at * stride, stride, left, left_f, wave);
    });
    const float by = __is_same(T, f16) && a.scale ? a.scale[1] : 1.f;
    const int64_t f = f_first + P::wave_m() * P::WM, c = c0 + P::column(0);
    __syncthreads();  // the panels' place is free
    store_tile<T, P::WM, P::WN>(P::stage(b0, b1), out + f * a.K + c, a.K, a.F - f, a.K - c,
                                [&](int i, int b) { return p.acc[i][b] * by; });
}

// Both, in one launch: neither alone fills the card but for large calls.  Whichever has the
// longer workgroups comes first.
template <typename T, bool PARTS, int BM, int BN, int WAVES_M, int WAVES_N, int KB>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void gated_gradients_kernel(GatedArgs a) {
    using Of = Parts<T, PARTS>;
    using E = typename Of::E;
    using In = Product<E, BM, BN, WAVES_M, WAVES_N, KB, kAcross, kAlong, false>;
    using Weights = Product<E, BM, BN, WAVES_M, WAVES_N, KB, kAcross, kAcross, false>;
    __shared__ __attribute__((aligned(1024))) char b0[In::BYTES], b1[In::BYTES];
    const uint32_t first = a.first;
    const bool second = blockIdx.x >= first;
    const uint32_t id = second ? blockIdx.x - first : blockIdx.x;
    if (second == a.weights_first)
        input_gradient<T, Of, In>(a, id, b0, b1);
    else
        weight_gradient<T, Of, Weights>(a, id, b0, b1);
}

// ---------------------------------------------------------------------------
// Few rows: the weights are read once, past the LDS
// ---------------------------------------------------------------------------

// Four contraction steps of 16 x 16 products: 16 bytes a lane.
template <typename T>
__device__ __forceinline__ f32x4 multiply16(ux4 first, ux4 second, f32x4 c) {
    if constexpr (__is_same(T, f16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, first), __builtin_bit_cast(f16x8, second), c, 0, 0, 0);
    } else if constexpr (__is_same(T, bf16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, first), __builtin_bit_cast(bf16x8, second), c, 0, 0, 0);
    } else {
        const f32x4 x = __builtin_bit_cast(f32x4, first), y = __builtin_bit_cast(f32x4, second);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
}

// 16 hidden columns and MG groups of 16 rows a workgroup, whose waves take turns in KB
// bytes of the contraction, each with panels of its own in LDS and no barrier.  (Straight to
// registers a lane would load 16 bytes of its own row, and lanes side by side other
// rows: 45 rows, 4096 -> 11000, took 65 us, four times the caches' requests.)  Bound by the
// weights' stream: that call 43 us, 4.2 TB/s, and 1 row, 2048 -> 8192 bf16 11.7 us, 5.7.
template <typename T, int MG, int WAVES, int KB>
__global__ __launch_bounds__(64 * WAVES) void gated_rows_kernel(GatedArgs a) {
    using L = Tile<T, KB / sizeof(T)>;
    constexpr int SIZE = 16 * KB, NI = KB / 64, STEPS = KB / 64, LOADS = NI * (2 + MG);
    __shared__ __attribute__((aligned(1024))) char panels0[WAVES][(2 + MG) * SIZE], panels1[WAVES][(2 + MG) * SIZE];
    static_assert(sizeof(panels0) >= WAVES * MG * 1024, "the waves' sums take the panels' place");
    const int l = threadIdx.x & 63, wave = wave_id(), f0 = blockIdx.x * 16;
    const int row_bytes = a.Kp * static_cast<int>(sizeof(T));
    const int left = min(a.F - f0, 16), rows = static_cast<int>(a.rows);
    auto matrix = [&](const void* base, uint32_t stride, int64_t first, int n) {
        return __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(static_cast<const char*>(base) + first * stride), static_cast<short>(0),
            static_cast<int>((n - 1) * stride + row_bytes), 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t rg = matrix(a.wg, a.wg_stride, f0, left), ru = matrix(a.wu, a.wu_stride, f0, left);
    const __amdgpu_buffer_rsrc_t rx = matrix(a.x, a.x_stride, 0, rows);
    // the chunk that the lane loads of its row, and where that row starts (a row that is none
    // lies past any buffer: zeros)
    uint32_t og[NI], ou[NI], ox[MG][NI];
    int chunk[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int x = i * 64 + l, r = x / L::NC;
        chunk[i] = ((x % L::NC) ^ L::turn(r)) * 16;
        og[i] = r < left ? r * a.wg_stride + chunk[i] : 0x80000000u;
        ou[i] = r < left ? r * a.wu_stride + chunk[i] : 0x80000000u;
#pragma unroll
        for (int j = 0; j < MG; ++j) ox[j][i] = 16 * j + r < rows ? (16 * j + r) * a.x_stride + chunk[i] : 0x80000000u;
    }
    auto load = [&](char* to, int k) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const bool past = k + chunk[i] >= row_bytes;
            to_lds<16>(rg, to + i * 1024, past ? 0x80000000u : og[i] + k);
            to_lds<16>(ru, to + SIZE + i * 1024, past ? 0x80000000u : ou[i] + k);
#pragma unroll
            for (int j = 0; j < MG; ++j) to_lds<16>(rx, to + (2 + j) * SIZE + i * 1024, past ? 0x80000000u : ox[j][i] + k);
        }
    };
    f32x4 acc[MG][2] = {};
    auto multiply = [&](const char* from) {
        ux4 v[STEPS][2 + MG];
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int n = 0; n < 2 + MG; ++n)
                v[s][n] = *reinterpret_cast<const ux4*>(from + n * SIZE + L::at(l & 15, s * 4 + (l >> 4)));
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int j = 0; j < MG; ++j) {
                acc[j][0] = multiply16<T>(v[s][0], v[s][2 + j], acc[j][0]);
                acc[j][1] = multiply16<T>(v[s][1], v[s][2 + j], acc[j][1]);
            }
    };
    char *p = panels0[wave], *q = panels1[wave];
    const int turns = (row_bytes + WAVES * KB - 1) / (WAVES * KB);
    auto place = [&](int i) { return (i * WAVES + wave) * KB; };
    // (turns past the end load zeros, and nothing from memory)
    load(p, place(0));
    load(q, place(1));
    for (int i = 0; i < turns; i += 2) {
        __builtin_amdgcn_s_waitcnt(0x0f70 | LOADS);  // all but the other panels'
        order();
        multiply(p);
        order();
        load(p, place(i + 2));
        __builtin_amdgcn_s_waitcnt(0x0f70 | LOADS);
        order();
        multiply(q);
        order();
        load(q, place(i + 3));
    }
    settle<float>();
    __builtin_amdgcn_s_waitcnt(0x0f70);  // the zeros have landed, and the panels' place is free
    __syncthreads();
    f32x4 *meet_g = reinterpret_cast<f32x4*>(panels0), *meet_u = reinterpret_cast<f32x4*>(panels1);  // (wave, group, lane)
#pragma unroll
    for (int j = 0; j < MG; ++j) meet_g[(wave * MG + j) * 64 + l] = acc[j][0], meet_u[(wave * MG + j) * 64 + l] = acc[j][1];
    __syncthreads();
    for (int j = wave; j < MG; j += WAVES) {
        const int m = 16 * j + (l & 15), f = f0 + 4 * (l >> 4);
        f32x4 g = {}, u = {};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) g += meet_g[(w * MG + j) * 64 + l], u += meet_u[(w * MG + j) * 64 + l];
        if (m >= rows || f >= a.F) continue;
        T* out = static_cast<T*>(a.h) + static_cast<int64_t>(m) * a.F + f;
        f32x4 h, slope;
        activate<4>(a.activation, g, h, slope);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f + e < a.F) out[e] = from_acc<T>(h[e] * u[e]);
    }
}

// ---------------------------------------------------------------------------
// Which workgroups a call takes
// ---------------------------------------------------------------------------

// Up to here the weights are read past the tiles (48 rows, 2048 -> 8192 bf16: 15.5 us, 22.8 by
// tiles; 64 rows: 18.7 and 23.0; 64 rows, 4096 -> 11000 fp16: 52.1 and 52.5, where the panels leave
// one workgroup to a CU).
constexpr int kFewRows = 64;

// Workgroup tiles, and the microseconds that a panel takes where one, two or three of
// them share a CU (measured at sizes that leave the clock alone; 0: they do not fit);
// `setup`: what a workgroup takes besides, in panels.  The bytes of what is written are in no
// term: a choice between tiles, not a forecast (128 rows, 4096 -> 11000: 41 us by these, 66
// measured; a training forward of 4096 x 1024 -> 4096 60 and 93; the gradients of 1025 x 1001 ->
// 2731 44 and 33).
struct Shape {
    int bm, bn;
    float along[3], across[3], wide[3];
    float setup;
};
constexpr Shape kShapes[3] = {{256, 256, {1.42f}, {1.5f}, {}, 5.f},
                              {128, 128, {0.72f, 1.12f}, {0.73f, 1.15f}, {1.9f, 3.5f}, 5.f},
                              {64, 128, {0.5f, 0.6f}, {0.57f, 0.9f, 1.25f}, {0.98f, 1.8f}, 5.f}};

// n workgroups of `length` panels, on as many CUs as there are.
struct Part {
    int64_t n, length;
};

// Panels until the last of two parts' workgroups is done, the longer ones first.
inline double panels_until_done(Part a, Part b, double setup, int64_t slots) {
    if (a.length < b.length) std::swap(a, b);
    const int64_t turns = a.n / slots, over = a.n % slots;
    const double la = static_cast<double>(a.length) + setup, lb = static_cast<double>(b.length) + setup;
    const double late = static_cast<double>(turns + 1) * la, early = static_cast<double>(turns) * la;
    double done = over ? late : early;
    if (!b.n) return done;
    auto room = [&](double t) {
        return (t > late ? over * static_cast<int64_t>((t - late) / lb) : 0) +
               (t > early ? (slots - over) * static_cast<int64_t>((t - early) / lb) : 0);
    };
    double t = (static_cast<double>(a.n) * la + static_cast<double>(b.n) * lb) / static_cast<double>(slots);
    while (room(t) < b.n) t += lb / 8;
    return std::max(done, t);
}

struct Cut {
    int shape, tiles_m, tiles_n, splits, weight_m, weight_n;
    double time;
    int64_t tiles() const { return static_cast<int64_t>(tiles_m) * tiles_n; }
    int64_t weights() const { return static_cast<int64_t>(weight_m) * weight_n; }
};

// How a call's products are formed: of fp32 numbers, or of `terms` products of 16 bits.
struct Means {
    bool wide;
    int terms;
    int64_t panels(int64_t length) const { return nsh_host::ceil_div(length, wide ? 32 : 64) * terms; }
};

// (0: no launch takes as many)
inline double time_of(const Shape& s, const float (&rate)[3], Part a, Part b, int64_t cus) {
    if ((a.n + b.n) * (s.bm == 256 ? 512 : 256) >> 32) return 0;
    int share = 1;
    while (share < 3 && rate[share] > 0 && share * cus < a.n + b.n) ++share;
    return panels_until_done(a, b, s.setup, cus * share) * rate[share - 1];
}

inline Cut forward_cut(int64_t rows, int64_t F, int64_t K, Means by) {
    const int64_t cus = nsh_host::compute_units();
    Cut best{};
    for (int i = by.wide ? 1 : 0; i < 3; ++i) {
        const Shape& s = kShapes[i];
        Cut c{i, static_cast<int>(nsh_host::ceil_div(rows, s.bm)), static_cast<int>(nsh_host::ceil_div(F, s.bn / 2)), 1, 0, 0, 0};
        c.time = time_of(s, by.wide ? s.wide : s.along, {c.tiles(), by.panels(K)}, {0, 0}, cus);
        if (c.time > 0 && (best.time == 0 || c.time < best.time)) best = c;
    }
    return best;
}

// Of dx, of the weights' gradients, or of both in one launch: with few tiles of dx,
// workgroups share a tile's sum over the hidden columns, and another launch joins them
// (4 us, and their sums' bytes at 3.5 TB/s).
inline Cut gradient_cut(int64_t rows, int64_t K, int64_t F, Means by, bool input, bool weights) {
    const int64_t cus = nsh_host::compute_units();
    Cut best{};
    for (int i = by.wide ? 1 : 0; i < 3; ++i) {
        const Shape& s = kShapes[i];
        Cut c{i, 0, 0, 1, 0, 0, 0};
        if (input) c.tiles_m = static_cast<int>(nsh_host::ceil_div(rows, s.bm)), c.tiles_n = static_cast<int>(nsh_host::ceil_div(K, s.bn));
        if (weights) c.weight_m = 2 * static_cast<int>(nsh_host::ceil_div(F, s.bm)), c.weight_n = static_cast<int>(nsh_host::ceil_div(K, s.bn));
        const int64_t panels = 2 * by.panels(F);
        for (const int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {  // (those that the join knows)
            if (splits > 1 && (!input || panels / splits < 4)) break;
            c.splits = splits;
            c.time = time_of(s, by.wide ? s.wide : s.across, {c.tiles() * splits, nsh_host::ceil_div(panels, splits)},
                             {c.weights(), by.panels(rows)}, cus);
            if (c.time == 0) break;
            if (splits > 1) c.time += 4 + static_cast<double>(splits * rows * K) * 4 / 3.5e6;
            if (best.time == 0 || c.time < best.time) best = c;
        }
    }
    return best;
}

template <typename T>
int gated_few_rows(GatedArgs a, hipStream_t st) {
    const unsigned grid = (a.F + 15) / 16;
    // One group of rows and workgroups for a part of the CUs: twice the waves (4 rows, 8192 -> 1024
    // bf16: 10.5 us, 11.9 with four; with a workgroup on every CU, 16 rows, 2048 -> 5504: 13.0
    // and 12.3).  More groups leave eight waves panels of 64 bytes a row (40 rows, 4096 -> 2048
    // fp16: 12.4 and 10.9; 45 rows, 4096 -> 11000: 58 us by 64 bytes, 43 by 128).
    if (a.rows <= 16 && grid < static_cast<unsigned>(nsh_host::compute_units()))
        gated_rows_kernel<T, 1, 8, 128><<<grid, 512, 0, st>>>(a);
    else if (a.rows <= 16)
        gated_rows_kernel<T, 1, 4, 128><<<grid, 256, 0, st>>>(a);
    else if (a.rows <= 32)
        gated_rows_kernel<T, 2, 4, 128><<<grid, 256, 0, st>>>(a);
    else if (a.rows <= 48)
        gated_rows_kernel<T, 3, 4, 128><<<grid, 256, 0, st>>>(a);
    else
        gated_rows_kernel<T, 4, 4, 128><<<grid, 256, 0, st>>>(a);
    return nsh_host::check_launch("gated_linear_forward");
}

template <typename T, bool PARTS>
int gated_forward(GatedArgs a, const Cut& c, hipStream_t st) {
    a.tiles_m = c.tiles_m, a.tiles_n = c.tiles_n;
    const unsigned grid = static_cast<unsigned>(c.tiles());
    if constexpr (sizeof(T) == 2 || PARTS)
        if (c.shape == 0) gated_forward_kernel<T, PARTS, 256, 256, 4, 2, 128><<<grid, 512, 0, st>>>(a);
    if (c.shape == 1) gated_forward_kernel<T, PARTS, 128, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    if (c.shape == 2) gated_forward_kernel<T, PARTS, 64, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    return nsh_host::check_launch("gated_linear_forward");
}

template <typename T, bool PARTS>
int gated_gradients(GatedArgs a, const Cut& c, hipStream_t st) {
    a.tiles_m = c.tiles_m, a.tiles_n = c.tiles_n, a.splits = c.splits, a.weight_m = c.weight_m, a.weight_n = c.weight_n;
    const int64_t in = c.tiles() * c.splits, all = in + c.weights();
    a.weights_first = 2 * a.Fp / c.splits < a.rows;
    a.first = static_cast<int>(a.weights_first ? c.weights() : in);
    const unsigned grid = static_cast<unsigned>(all);
    if constexpr (sizeof(T) == 2 || PARTS)
        if (c.shape == 0) gated_gradients_kernel<T, PARTS, 256, 256, 4, 2, 128><<<grid, 512, 0, st>>>(a);
    if (c.shape == 1) gated_gradients_kernel<T, PARTS, 128, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    if (c.shape == 2) gated_gradients_kernel<T, PARTS, 64, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    return nsh_host::check_launch("gated_linear_backward");
}

#define NSH_GATED_ENTRIES(EXTERN, T, PARTS)                                        \
    EXTERN template int gated_forward<T, PARTS>(GatedArgs, const Cut&, hipStream_t); \
    EXTERN template int gated_gradients<T, PARTS>(GatedArgs, const Cut&, hipStream_t);
#define NSH_GATED_FEW_ROWS(EXTERN, T) EXTERN template int gated_few_rows<T>(GatedArgs, hipStream_t);

}  // namespace nsh
