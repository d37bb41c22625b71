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

#include "panels.hpp"

namespace nsh {

struct GatedArgs {
    const void *x, *wg, *wu;
    uint32_t x_stride, wg_stride, wu_stride;  // bytes from row to row
    int64_t rows;
    int K, F, Kp, Fp;     // Kp: columns of x and the weights as they lie; Fp: F in whole panels
    int activation;
    void* h;
    char* kept;            // blocks of 32 x 32 (struct Kept), or NULL
    float* most;           // fp16 training: largest factor of every workgroup
    void* dgu;             // (rows, 2, Fp) and a panel's width of nothing
    const float* scale;    // fp16: what dgu was multiplied by, and its inverse
    void *dx, *dwg, *dwu;
    float* part;           // (splits, rows, K): sums of dx that a second launch joins
    int tiles_m, tiles_n, splits;
};

enum Activation { kSilu, kGelu, kGeluTanh, kRelu, kSigmoid };

// The activation at g and its slope there, by instructions of one place in the last or so:
// next to the sums' roundings nothing, and a third of the library functions' time.
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
        // weights towards the smallest largest error: 6e-9 of it, 1e-7 with fp32's roundings
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
        return make_float2(g * s, fma_acc(g * s * (1.f - s), a * fma_acc(3.f * b * g, g, 1.f), s));
    } else if constexpr (KIND == kRelu) {
        return g > 0.f ? make_float2(g, 1.f) : make_float2(g == g ? 0.f : g, 0.f);
    } else {
        const float s = sigmoid(g);
        return make_float2(s, s * (1.f - s));
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

// What training keeps of a block of 32 x 32 places: the two factors as the lanes have
// them, so that every store and load is 1 KB in one piece (rows of their own, 16 bytes a
// lane apart, took the forward 8192 x 2048 -> 8192 from 480 to 1017 us).
//   bf16: fp16 times a power of two of each lane's largest, which leaves 11 bits of all
//     that is not below 2^-29 of it, and 2^-40 of it of the rest
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
    static __device__ __forceinline__ uint32_t field(const f32x16& v) {
        float most = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(v[r]));
        if (!(most < INFINITY)) {  // an infinity says nothing of the others
            most = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(v[r]) < INFINITY ? fabsf(v[r]) : 0.f);
        }
        return max(__float_as_uint(most) >> 23, 15u);
    }

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
                for (int r = 0; r < 16; ++r) b[r] = __float_as_uint(v[r]) + 0x80u;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    ux4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = b[8 * q + 2 * e] >> 16 | (b[8 * q + 2 * e + 1] & 0xffff0000u);
                    *part(at, 2 * n + q) = x;
                }
                ux4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = (b[4 * e] >> 8 & 0xffu) | (b[4 * e + 1] & 0xff00u) | (b[4 * e + 2] & 0xff00u) << 8 |
                           (b[4 * e + 3] & 0xff00u) << 16;
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
        if constexpr (__is_same(T, f16)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                // (numbers only: an infinity says nothing of the others)
                const float x = fabsf(s[r]), y = fabsf(h[r]);
                most = fmaxf(most, fmaxf(x < INFINITY ? x : 0.f, y < INFINITY ? y : 0.f));
            }
        }
    }
    return h * u;
}

// Bytes of a row of dgu: not a power of two, which would have every row's same place in
// one channel of the caches.
template <typename T>
__device__ __forceinline__ uint32_t dgu_stride(const GatedArgs& a) {
    return 2 * a.Fp * static_cast<uint32_t>(sizeof(T)) + 128;
}

template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, int KB>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void gated_forward_kernel(GatedArgs a) {
    using P = Product<T, BM, BN, WAVES_M, WAVES_N, KB, kAlong, kAlong, true>;
    __shared__ __attribute__((aligned(1024))) char f0[P::FIRST_BYTES], s0[P::SECOND_BYTES];
    __shared__ __attribute__((aligned(1024))) char f1[P::FIRST_BYTES], s1[P::SECOND_BYTES];
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
    const int64_t wide = static_cast<int64_t>(a.Kp) * sizeof(T);
    const int left_m = static_cast<int>(min(a.rows - m0, int64_t(BM)));
    P p;
    p.init();
    const int n = (a.Kp + P::BK - 1) / P::BK;
    p.run(n, f0, s0, f1, s1, [&](int i, char* f, char* s) {
        const int64_t at = static_cast<int64_t>(i) * KB;
        const int left_f = i < n ? a.F - c0 : 0;
        gate.load(f, wg + at, a.wg_stride, left_f, wide - at, wave);
        up.load(f + P::FIRST_BYTES / 2, wu + at, a.wu_stride, left_f, wide - at, wave);
        rows.load(s, x + at, a.x_stride, i < n ? left_m : 0, wide - at, wave);
    });
    float most = 0.f;
    const int64_t m = m0 + P::wave_m() * P::WM;
    const int c = c0 + P::column(0);
    __syncthreads();  // the panels' place is free
    store_tile<T, P::WM, P::WN / 2>(P::stage(f0, s0, f1, s1), static_cast<T*>(a.h) + m * a.F + c, a.F, a.rows - m, a.F - c,
                                    [&](int i, int b) {
                                        return gate_block<T>(a, m0 + P::row(i), c0 + P::column(b), p.acc[i][b],
                                                             p.acc[i][b + P::NB / 2], most);
                                    });
    if constexpr (__is_same(T, f16)) {
        if (!a.most) return;
        float* meet = reinterpret_cast<float*>(f0);
        __syncthreads();
        meet[threadIdx.x] = most;
        __syncthreads();
        for (int n = P::NT / 2; n >= 1; n /= 2) {
            if (static_cast<int>(threadIdx.x) < n) meet[threadIdx.x] = fmaxf(meet[threadIdx.x], meet[threadIdx.x + n]);
            __syncthreads();
        }
        if (threadIdx.x == 0) a.most[blockIdx.x] = meet[0];
    }
}

// dx: over the hidden columns of dg, then of du.
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, int KB>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void gated_input_gradient_kernel(GatedArgs a) {
    using P = Product<T, BM, BN, WAVES_M, WAVES_N, KB, kAcross, kAlong, false>;
    __shared__ __attribute__((aligned(1024))) char f0[P::FIRST_BYTES], s0[P::SECOND_BYTES];
    __shared__ __attribute__((aligned(1024))) char f1[P::FIRST_BYTES], s1[P::SECOND_BYTES];
    const uint32_t tiles = static_cast<uint32_t>(a.tiles_m) * a.tiles_n;
    const int split = TileOrder::uniform(blockIdx.x / tiles);
    const TileOrder t(blockIdx.x - split * tiles, tiles, a.tiles_m, a.tiles_n, 8);
    const int64_t m0 = static_cast<int64_t>(t.m) * BM;
    const int64_t c0 = static_cast<int64_t>(t.n) * BN;
    const int wave = wave_id();
    typename P::FirstPanel gate, up;
    typename P::SecondPanel rows;
    gate.init(a.wg_stride);
    up.init(a.wu_stride);
    const uint32_t stride = dgu_stride<T>(a);
    rows.init(stride);
    const char* d = static_cast<const char*>(a.dgu) + m0 * stride;
    const char* wg = static_cast<const char*>(a.wg) + c0 * static_cast<int64_t>(sizeof(T));
    const char* wu = static_cast<const char*>(a.wu) + c0 * static_cast<int64_t>(sizeof(T));
    const int left_m = static_cast<int>(min(a.rows - m0, int64_t(BM)));
    const int64_t left_c = (a.Kp - c0) * static_cast<int64_t>(sizeof(T));
    const int half = a.Fp / P::BK, all = 2 * half;
    const int begin = TileOrder::uniform(all * static_cast<uint32_t>(split) / a.splits);
    const int end = TileOrder::uniform(all * static_cast<uint32_t>(split + 1) / a.splits);
    P p;
    p.init();
    p.run(end - begin, f0, s0, f1, s1, [&](int i, char* f, char* s) {
        const int at = begin + i, in = at < half ? at : at - half;
        const bool one = at < half;
        const uint32_t step = one ? a.wg_stride : a.wu_stride;
        P::FirstPanel::either(one, gate, up).load(f, (one ? wg : wu) + static_cast<int64_t>(in) * P::BK * step, step,
                                                  at < end ? a.F - in * P::BK : 0, left_c, wave);
        rows.load(s, d + static_cast<int64_t>(at) * KB, stride, at < end ? left_m : 0, KB, wave);
    });
    const float by = __is_same(T, f16) && a.scale ? a.scale[1] : 1.f;
    const int64_t m = m0 + P::wave_m() * P::WM, c = c0 + P::column(0);
    __syncthreads();  // the panels' place is free
    char* stage = P::stage(f0, s0, f1, s1);
    const auto value = [&](int i, int b) { return p.acc[i][b] * by; };
    if (a.part)
        store_tile<float, P::WM, P::WN>(stage, a.part + (split * a.rows + m) * a.K + c, a.K, a.rows - m, a.K - c, value);
    else
        store_tile<T, P::WM, P::WN>(stage, static_cast<T*>(a.dx) + m * a.K + c, a.K, a.rows - m, a.K - c, value);
}

// Both weights' gradients: tiles of hidden rows of the one, then of the other.
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, int KB>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void gated_weight_gradient_kernel(GatedArgs a) {
    using P = Product<T, BM, BN, WAVES_M, WAVES_N, KB, kAcross, kAcross, false>;
    __shared__ __attribute__((aligned(1024))) char f0[P::FIRST_BYTES], s0[P::SECOND_BYTES];
    __shared__ __attribute__((aligned(1024))) char f1[P::FIRST_BYTES], s1[P::SECOND_BYTES];
    const int each = a.tiles_m / 2;
    const TileOrder t(blockIdx.x, gridDim.x, a.tiles_m, a.tiles_n, 8);
    const int side = t.m >= each;
    T* out = static_cast<T*>(side ? a.dwu : a.dwg);
    if (!out) return;
    const int f_first = (side ? t.m - each : t.m) * BM;
    const int64_t c0 = static_cast<int64_t>(t.n) * BN;
    const int wave = wave_id();
    typename P::FirstPanel in;
    typename P::SecondPanel d;
    in.init(a.x_stride);
    const uint32_t stride = dgu_stride<T>(a);
    d.init(stride);
    const char* x = static_cast<const char*>(a.x) + c0 * static_cast<int64_t>(sizeof(T));
    const char* dgu = static_cast<const char*>(a.dgu) + (static_cast<int64_t>(side) * a.Fp + f_first) * static_cast<int64_t>(sizeof(T));
    const int64_t left_c = (a.Kp - c0) * static_cast<int64_t>(sizeof(T));
    const int64_t left_f = (static_cast<int64_t>(a.Fp) - f_first) * static_cast<int64_t>(sizeof(T));
    P p;
    p.init();
    p.run(static_cast<int>((a.rows + P::BK - 1) / P::BK), f0, s0, f1, s1, [&](int i, char* f, char* s) {
        const int64_t at = static_cast<int64_t>(i) * P::BK;
        const int left = static_cast<int>(max(min(a.rows - at, int64_t(P::BK)), int64_t(0)));
        in.load(f, x + at * a.x_stride, a.x_stride, left, left_c, wave);
        d.load(s, dgu + at * stride, stride, left, left_f, wave);
    });
    const float by = __is_same(T, f16) && a.scale ? a.scale[1] : 1.f;
    const int64_t f = f_first + P::wave_m() * P::WM, c = c0 + P::column(0);
    __syncthreads();  // the panels' place is free
    store_tile<T, P::WM, P::WN>(P::stage(f0, s0, f1, s1), out + f * a.K + c, a.K, a.F - f, a.K - c,
                                [&](int i, int b) { return p.acc[i][b] * by; });
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

// FG groups of 16 hidden columns and MG of 16 rows a workgroup, whose four waves take
// turns in 256 bytes of the contraction: a lane (row l % 16) reads 16 bytes of each 64.
template <typename T, int FG, int MG>
__global__ __launch_bounds__(256) void gated_rows_kernel(GatedArgs a) {
    constexpr int kBlock = 256, kSteps = 4;
    __shared__ f32x4 meet[4][FG][MG][2][64];
    const int l = threadIdx.x & 63, wave = wave_id(), f0 = blockIdx.x * (16 * FG);
    const int row_bytes = a.Kp * static_cast<int>(sizeof(T));
    auto matrix = [&](const void* base, uint32_t stride, int64_t first, int rows) {
        return __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(static_cast<const char*>(base) + first * stride), static_cast<short>(0),
            static_cast<int>((rows - 1) * stride + row_bytes), 0x00020000);
    };
    const int left = min(a.F - f0, 16 * FG), rows = static_cast<int>(a.rows);
    const __amdgpu_buffer_rsrc_t rg = matrix(a.wg, a.wg_stride, f0, left), ru = matrix(a.wu, a.wu_stride, f0, left);
    const __amdgpu_buffer_rsrc_t rx = matrix(a.x, a.x_stride, 0, rows);
    struct Block {
        ux4 g[FG][kSteps], u[FG][kSteps], x[MG][kSteps];
    };
    const int r = l & 15, part = (l >> 4) * 16;
    auto read = [&](Block& b, int k) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int at = k + s * 64 + part;
            const bool in = at < row_bytes;
            auto get = [&](__amdgpu_buffer_rsrc_t rs, int row, int most, uint32_t stride) {
                const uint32_t off = in && row < most ? static_cast<uint32_t>(row) * stride + at : 0x80000000u;
                return __builtin_bit_cast(ux4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
            };
#pragma unroll
            for (int i = 0; i < FG; ++i) {
                b.g[i][s] = get(rg, 16 * i + r, left, a.wg_stride);
                b.u[i][s] = get(ru, 16 * i + r, left, a.wu_stride);
            }
#pragma unroll
            for (int i = 0; i < MG; ++i) b.x[i][s] = get(rx, 16 * i + r, rows, a.x_stride);
        }
    };
    f32x4 acc[FG][MG][2] = {};
    auto multiply = [&](const Block& b) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int i = 0; i < FG; ++i)
#pragma unroll
                for (int j = 0; j < MG; ++j) {
                    acc[i][j][0] = multiply16<T>(b.g[i][s], b.x[j][s], acc[i][j][0]);
                    acc[i][j][1] = multiply16<T>(b.u[i][s], b.x[j][s], acc[i][j][1]);
                }
    };
    Block p, q;
    int k = wave * kBlock;
    if (k < row_bytes) read(p, k);
    while (k < row_bytes) {
        const int next = k + 4 * kBlock, after = k + 8 * kBlock;
        if (next < row_bytes) read(q, next);
        multiply(p);
        if (next >= row_bytes) break;
        if (after < row_bytes) read(p, after);
        multiply(q);
        k = after;
    }
    settle<float>();
#pragma unroll
    for (int i = 0; i < FG; ++i)
#pragma unroll
        for (int j = 0; j < MG; ++j) meet[wave][i][j][0][l] = acc[i][j][0], meet[wave][i][j][1][l] = acc[i][j][1];
    __syncthreads();
    for (int n = wave; n < FG * MG; n += 4) {
        const int i = n / MG, j = n % MG, m = 16 * j + r, f = f0 + 16 * i + 4 * (l >> 4);
        f32x4 g = {}, u = {};
#pragma unroll
        for (int w = 0; w < 4; ++w) g += meet[w][i][j][0][l], u += meet[w][i][j][1][l];
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

constexpr int kFewRows = 64;

struct Cut {
    int bm, bn;  // of the result
    int tiles_m, tiles_n;
    int64_t tiles() const { return static_cast<int64_t>(tiles_m) * tiles_n; }
};

// Tiles of 256 x 256 where they fill the card, of 128 x 128, or of 64 x 128 (`paired`: a
// tile has half as many columns, of both matrices).
inline Cut cut_of(int64_t rows, int64_t cols, bool wide, bool paired, int sides) {
    static constexpr int kSizes[3][2] = {{256, 256}, {128, 128}, {64, 128}};
    const int cus = nsh_host::compute_units();
    Cut c{};
    for (int i = wide ? 1 : 0; i < 3; ++i) {
        c.bm = kSizes[i][0], c.bn = kSizes[i][1];
        c.tiles_m = static_cast<int>(nsh_host::ceil_div(rows, c.bm)) * sides;
        c.tiles_n = static_cast<int>(nsh_host::ceil_div(cols, paired ? c.bn / 2 : c.bn));
        if (c.tiles() >= (i == 0 ? cus * 3 / 4 : cus)) break;
    }
    return c;
}

template <typename T>
int gated_forward(GatedArgs a, hipStream_t st) {
    if (a.rows <= kFewRows && !a.kept) {
        const unsigned one = (a.F + 15) / 16, two = (a.F + 31) / 32;
        if (a.rows <= 16)
            gated_rows_kernel<T, 1, 1><<<one, 256, 0, st>>>(a);
        else if (a.rows <= 32)
            gated_rows_kernel<T, 2, 2><<<two, 256, 0, st>>>(a);
        else
            gated_rows_kernel<T, 2, 4><<<two, 256, 0, st>>>(a);
        return nsh_host::check_launch("gated_linear_forward");
    }
    const Cut c = cut_of(a.rows, a.F, sizeof(T) == 4, true, 1);
    a.tiles_m = c.tiles_m, a.tiles_n = c.tiles_n;
    const unsigned grid = static_cast<unsigned>(c.tiles());
    if constexpr (sizeof(T) == 2)
        if (c.bm == 256) gated_forward_kernel<T, 256, 256, 4, 2, 128><<<grid, 512, 0, st>>>(a);
    if (c.bm == 128) gated_forward_kernel<T, 128, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    if (c.bm == 64) gated_forward_kernel<T, 64, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    return nsh_host::check_launch("gated_linear_forward");
}

template <typename T>
int gated_input_gradient(GatedArgs a, const Cut& c, hipStream_t st) {
    a.tiles_m = c.tiles_m, a.tiles_n = c.tiles_n;
    const unsigned grid = static_cast<unsigned>(c.tiles() * a.splits);
    if constexpr (sizeof(T) == 2)
        if (c.bm == 256) gated_input_gradient_kernel<T, 256, 256, 4, 2, 128><<<grid, 512, 0, st>>>(a);
    if (c.bm == 128) gated_input_gradient_kernel<T, 128, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    if (c.bm == 64) gated_input_gradient_kernel<T, 64, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    return nsh_host::check_launch("gated_linear_backward");
}

template <typename T>
int gated_weight_gradient(GatedArgs a, hipStream_t st) {
    const Cut c = cut_of(a.F, a.K, sizeof(T) == 4, false, 2);
    a.tiles_m = c.tiles_m, a.tiles_n = c.tiles_n;
    const unsigned grid = static_cast<unsigned>(c.tiles());
    if constexpr (sizeof(T) == 2)
        if (c.bm == 256) gated_weight_gradient_kernel<T, 256, 256, 4, 2, 128><<<grid, 512, 0, st>>>(a);
    if (c.bm == 128) gated_weight_gradient_kernel<T, 128, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    if (c.bm == 64) gated_weight_gradient_kernel<T, 64, 128, 2, 2, 128><<<grid, 256, 0, st>>>(a);
    return nsh_host::check_launch("gated_linear_backward");
}

#define NSH_GATED_ENTRIES(EXTERN, T)                                                       \
    EXTERN template int gated_forward<T>(GatedArgs, hipStream_t);                          \
    EXTERN template int gated_input_gradient<T>(GatedArgs, const Cut&, hipStream_t);       \
    EXTERN template int gated_weight_gradient<T>(GatedArgs, hipStream_t);

}  // namespace nsh
