// attention_tiles.hpp -- tiles of rows in LDS and the 32 x 32 matrix products
// over them, for fp16, bf16 and fp32 alike.
//
// A wave's products have the rows of an LDS tile on their first side and 32
// rows held in registers, one to a lane (lane l: row l % 32), on their second;
// lane halves (g = l / 32) share a row's contraction.  The result leaves every
// lane with 16 of the tile's 32 rows for its own row,
//     element r <-> tile row 8 (r / 4) + 4 g + r % 4,
// which is also the order in which the second product (weights times the
// tile's rows, contracted over those) wants its second side: it needs no
// exchange of lanes, only the tile read by columns in the same order.
#pragma once

#include "attention.hpp"

namespace nsh {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

#define NSH_LDS __attribute__((address_space(3)))

// Eight contraction steps of a lane half: what one row contributes to 16.
template <typename T> struct Eight;
template <> struct Eight<f16> {
    using V = f16x8;
    static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ V pack(f32x8 v) { return __builtin_convertvector(v, f16x8); }
    static __device__ __forceinline__ V negate(V v) { return -v; }
};
template <> struct Eight<bf16> {
    using V = bf16x8;
    static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ V pack(f32x8 v) { return __builtin_convertvector(v, bf16x8); }
    static __device__ __forceinline__ V negate(V v) {
        return __builtin_bit_cast(V, __builtin_bit_cast(s16x8, v) ^ static_cast<short>(0x8000));
    }
};
template <> struct Eight<float> {
    using V = f32x8;
    static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ V pack(f32x8 v) { return v; }
    static __device__ __forceinline__ V negate(V v) { return -v; }
};

// Four results rounded to T, stored together.
template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<f32x4*>(p) = v;
    else if constexpr (__is_same(T, f16))
        *reinterpret_cast<f16x4*>(p) = __builtin_convertvector(v, f16x4);
    else
        *reinterpret_cast<bf16x4*>(p) = __builtin_convertvector(v, bf16x4);
}

// What store4 rounds off, stored in its place beside out.
template <typename T>
__device__ __forceinline__ void store4_rest(T* p, f32x4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = rounded_off<T>(v[e]);
    store4<T>(p, v);
}

// Tile row of result element r, less the lane half's 4 g.
__device__ __forceinline__ constexpr int el(int r) { return 8 * (r / 4) + r % 4; }

// The other lane half's value joined to one's own.
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Rows of DP elements in LDS, 16-byte chunks.  A row's chunks are permuted by
// turn(row): LDS serves 256 bytes a cycle from 64 banks, and 16 rows read at
// one chunk, as well as four rows read at 64 bytes by columns, then fall on
// every bank once.
template <typename T, int DP>
struct Tile {
    static constexpr int CE = 16 / sizeof(T), NC = DP / CE, ROW = DP * sizeof(T);
    static constexpr int NS = DP / 16, ND = DP / 32;
    using V = typename Eight<T>::V;

    // turn() only moves bits of the row about, so that a place's address is one
    // of the lane's with constants joined by exclusive or, within FIELD bytes,
    // and by addition beyond.
    static constexpr int FIELD = NC % 16 == 0 ? 256 : NC % 8 == 0 ? 128 : 64;
    static __host__ __device__ __forceinline__ constexpr int turn(int r) {
        if constexpr (NC % 16 == 0 && sizeof(T) == 2)
            return (r & 3) << 2 | (r >> 2 & 3);
        else if constexpr (NC % 16 == 0)  // by columns, rows r and r + 4 are read at 128 bytes
            return (r >> 2 & 1) << 3 | (r & 3) << 1 | (r >> 3 & 1);
        else if constexpr (NC % 8 == 0)
            return (r >> 1 & 1) << 2 | (r >> 2 & 3);
        else
            return r >> 2 & 3;
    }
    static __device__ __forceinline__ int at(int r, int c) { return r * ROW + ((c ^ turn(r)) * 16); }
    static __device__ __forceinline__ int moved(int base, int bytes, int row) {
        return (base ^ (bytes % FIELD) ^ turn(row) * 16) + bytes / FIELD * FIELD + row * ROW;
    }

    // The lane's place in row r0 + l % 32 (r0 a multiple of 32), and by columns.
    static __device__ __forceinline__ int row_base(int r0, int l) {
        return at(r0 + (l & 31), (l >> 5) * (sizeof(T) / 2));
    }
    static __device__ __forceinline__ int col_base(int r0, int l) {
        if constexpr (sizeof(T) == 2) {
            // a transposing read takes four rows by 16 columns from 16 lanes
            const int i = l & 15, d = (l & 16) + 4 * (i & 3);
            return at(r0 + 4 * (l >> 5) + (i >> 2), d / 8) + (d & 7) * 2;
        } else {
            const int d = l & 31;
            return at(r0 + 4 * (l >> 5), d / 4) + (d & 3) * 4;
        }
    }

    // Steps s of the lane's row, `row` rows on (a multiple of 32).
    static __device__ __forceinline__ V row(const char* lds, int base, int row, int s) {
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const V*>(lds + moved(base, 32 * s, row));
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4*>(lds + moved(base, 64 * s, row));
            const f32x4 b = *reinterpret_cast<const f32x4*>(lds + moved(base, 64 * s + 16, row));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // Column 32 db + l % 32 of 16 rows, `row` rows on (a multiple of 16), in the
    // order of result elements.
    static __device__ __forceinline__ V col(const char* lds, int base, int row, int db) {
        if constexpr (sizeof(T) == 2) {
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NSH_LDS s16x4*)(lds + moved(base, 64 * db, row)));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NSH_LDS s16x4*)(lds + moved(base, 64 * db, row + 8)));
            return __builtin_bit_cast(V, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            V v;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = *reinterpret_cast<const float*>(lds + moved(base, 128 * db, row + el(e)));
            return v;
        }
    }
};

// v, and nothing formed of it ahead of here: what only a branch needs is
// otherwise computed in front of it.
__device__ __forceinline__ int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// BYTES a lane from its offset in the buffer to LDS, the lanes side by side
// from `lds` on; nothing passes through registers.
template <int BYTES>
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t rs, void* lds, uint32_t off) {
#ifdef __HIP_DEVICE_COMPILE__  // the host's parse of this header knows no 16-byte form
    if constexpr (BYTES == 16)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (NSH_LDS void*)(lds), 16, off, 0, 0, 0);
    else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (NSH_LDS void*)(lds), 4, off, 0, 0, 0);
#endif
}

// Tile rows [0, ROWS) of a tensor from global memory straight into LDS by NW
// waves.  Rows past the tensor's end, and columns past D, arrive as zeros (the
// buffer's range check): nothing behind a cache's filled part is read.
//
// LEAN keeps one offset in a register and forms the others of it at each load,
// where an instruction covers whole sets of 16 rows, whose chunks' order repeats.
template <typename T, int DP, int ROWS, int NW, bool LEAN = false>
struct Loader {
    using L = Tile<T, DP>;
    static constexpr int NI = ROWS * L::NC / (NW * 64);
    static_assert(NI * NW * 64 == ROWS * L::NC, "whole instructions");
    static constexpr bool kOne = LEAN && NW * 64 % (16 * L::NC) == 0;
    uint32_t off[kOne ? 1 : NI];

    __device__ __forceinline__ void init(int id, int64_t stride, int D) {
#pragma unroll
        for (int i = 0; i < (kOne ? 1 : NI); ++i) {
            const int x = i * NW * 64 + id, r = x / L::NC, c = (x % L::NC) ^ L::turn(r);
            off[i] = c * L::CE < D ? static_cast<uint32_t>(r) * static_cast<uint32_t>(stride * sizeof(T)) + c * 16 : 0x80000000u;
        }
    }
    // base: the tensor's row 0; bytes: from row to row (2^24 at most); first: the
    // tile's first row; rows: the tensor's end.
    __device__ __forceinline__ void load(char* lds, const T* base, int64_t stride, int first, int rows,
                                         int D, int wave) const {
        const uint32_t bytes = static_cast<uint32_t>(stride) * sizeof(T);
        const uint32_t left = static_cast<uint32_t>(max(min(rows - first, ROWS), 0));  // rows past the tile are not asked for
        const uint32_t size = left ? (left - 1) * bytes + D * static_cast<uint32_t>(sizeof(T)) : 0u;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(reinterpret_cast<const char*>(base) + static_cast<uint64_t>(static_cast<uint32_t>(first)) * bytes),
            static_cast<short>(0), static_cast<int>(size), 0x00020000);
        // (columns past D are at 2^31, and 112 rows of 2^24 bytes on past any size still)
        const uint32_t one = kOne ? static_cast<uint32_t>(here(static_cast<int>(off[0]))) : 0u;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            to_lds<16>(rs, lds + (i * NW + wave) * 1024, kOne ? one + i * (NW * 64 / L::NC) * bytes : off[i]);
    }
};

// The lane's row, as the second side of the products (zeros past D).
template <typename T, int DP>
__device__ __forceinline__ void load_row(typename Eight<T>::V (&v)[DP / 16], const T* row, int D, int l) {
    using V = typename Eight<T>::V;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = s * 16 + (l >> 5) * 8;
        if constexpr (sizeof(T) == 2) {
            i32x4 x = {};
            if (d < D) x = *reinterpret_cast<const i32x4*>(row + d);
            v[s] = __builtin_bit_cast(V, x);
        } else {
            f32x4 x = {}, y = {};
            if (d < D) {
                x = *reinterpret_cast<const f32x4*>(row + d);
                y = *reinterpret_cast<const f32x4*>(row + d + 4);
            }
            v[s] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
}

// Reads from LDS take some hundred cycles.  They go out together, ahead of the
// products that use them; order() keeps the compiler from moving them back to
// their uses, one read and one wait at a time.
__device__ __forceinline__ void order() { __builtin_amdgcn_sched_barrier(0); }

// Which of a SIMD's waves issues first, from here on.  Without it the older wave
// goes on with whatever it does, and the two tend to do the same.
template <int P>
__device__ __forceinline__ void priority() {
    order();
    __builtin_amdgcn_s_setprio(P);
    order();
}

// Ends a run of products ahead of a branch.  Their results may be read 12 wait
// states (18 for the fp32 products) after the last one at the earliest, and the
// hardware does not wait by itself; the compiler counts the states, but has
// been seen to miss a read in another block (a copy of the sums behind a loop's
// exit took their last two rows too early).
template <typename T>
__device__ __forceinline__ void settle() {
    order();
    if constexpr (sizeof(T) == 4)
        asm volatile("s_nop 15\n\ts_nop 1");
    else
        asm volatile("s_nop 11");
    order();
}

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Kinds of call, each with kernels of its own: no bias, no documents and a scale, without
// a cap (kPlain) or with the quick one (kCapped), whose tiles take no branch; or
// whatever a call may hold (kGeneral), at a cost in registers.
enum Kind { kPlain, kCapped, kGeneral };

template <typename T, int DP>
struct RowFragments {  // 32 tile rows, `row` rows on from the base's
    typename Eight<T>::V f[DP / 16];
    __device__ __forceinline__ void read(const char* lds, int base, int row = 0) {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) f[s] = Tile<T, DP>::row(lds, base, row, s);
    }
    // their products with the lane's row
    __device__ __forceinline__ f32x16 products(const typename Eight<T>::V (&v)[DP / 16]) const {
        f32x16 c = {};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) c = Eight<T>::mma(f[s], v[s], c);
        return c;
    }
};

template <typename T, int DP>
struct ColumnFragments {  // 32 tile rows, `row` rows on from the base's, by columns
    typename Eight<T>::V f[DP / 32][2];
    __device__ __forceinline__ void read(const char* lds, int base, int row = 0) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
            f[d][0] = Tile<T, DP>::col(lds, base, row, d), f[d][1] = Tile<T, DP>::col(lds, base, row + 16, d);
    }
    // acc += their columns times the weights w, rounded to T as the matrix
    // instructions want them: in 16 bits half a step of each weight, of the size of
    // the result's own rounding and not shared by a row's pairs (errors 0.0017 to
    // 0.0024 of the whole in bf16, 2.1e-4 to 2.9e-4 in fp16; a second product for what
    // the rounding left would take that away for half as much matrix time again)
    __device__ __forceinline__ void weigh(f32x16 (&acc)[DP / 32], const f32x16& w) const {
        const typename Eight<T>::V lo = Eight<T>::pack(__builtin_shufflevector(w, w, 0, 1, 2, 3, 4, 5, 6, 7));
        const typename Eight<T>::V hi = Eight<T>::pack(__builtin_shufflevector(w, w, 8, 9, 10, 11, 12, 13, 14, 15));
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Eight<T>::mma(f[d][0], lo, acc[d]);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Eight<T>::mma(f[d][1], hi, acc[d]);
    }
    // The same for the gradients of q and k, whose weights dx take both signs and
    // cancel: in fp16, which is chosen for its 11 bits, w goes in two parts, what
    // the type takes of it and of the rest (errors of those gradients 3.4e-4 to
    // 2.9e-4 at 2500 tokens of width 64, where the result's own rounding makes
    // 2.1e-4; 5% of the gradients' time), brought into its range by fit().  In
    // bf16 one part's rounding, at most 2^-9 of every dx, is of the size of the
    // results' own; two would cost 15%.
    __device__ __forceinline__ void weigh_fine(f32x16 (&acc)[DP / 32], const f32x16& w) const {
        if constexpr (!__is_same(T, f16)) return weigh(acc, w);
        using V = typename Eight<T>::V;
        const f32x8 a = __builtin_shufflevector(w, w, 0, 1, 2, 3, 4, 5, 6, 7);
        const f32x8 b = __builtin_shufflevector(w, w, 8, 9, 10, 11, 12, 13, 14, 15);
        const V lo = Eight<T>::pack(a), hi = Eight<T>::pack(b);
        const V lo2 = Eight<T>::pack(a - __builtin_convertvector(lo, f32x8));
        const V hi2 = Eight<T>::pack(b - __builtin_convertvector(hi, f32x8));
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Eight<T>::mma(f[d][0], lo, acc[d]);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Eight<T>::mma(f[d][1], hi, acc[d]);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Eight<T>::mma(f[d][0], lo2, acc[d]);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Eight<T>::mma(f[d][1], hi2, acc[d]);
    }
};

// fp16 has its 11 bits from 2^-14 to 2^16 alone, where the gradients' weights lie
// anywhere: a mean loss sends dO of 1e-5, and p is 1 / count.  The products take
// both times powers of two, which the sums are rid of at the end: p (1 at most)
// times kRoom, dx times a factor of the lane's own row or key, kept as the running
// maximum of a softmax is: a tile whose largest dx passes kFitMost brings that
// down to kFitTo, and the sums with it.  It starts where the smallest dx that an
// fp16 result can show is still a normal number.  (2500 tokens, width 64, causal,
// dO of 2^-10: dq and dk off by 2.8e-4 and 3.0e-4, their own rounding, and 1.1e-3
// without; by keys at 2 x 16 heads, 4096 tokens, width 128: 339 us without, 357 with.)
template <typename T> constexpr bool kNarrow = __is_same(T, f16);
template <typename T> constexpr float kRoom = kNarrow<T> ? 32768.f : 1.f;
constexpr float kFitMost = 32768.f, kFitFirst = 1.0995116e12f;  // 2^40
constexpr int kFitTo = 8;                                       // the largest below 2^8

template <typename T, int ND>
__device__ __forceinline__ f32x16 fit(float& by, f32x16 dx, f32x16 (&acc)[ND]) {
    if constexpr (!kNarrow<T>) return dx;
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(dx[r]));
    top = halves_max(top);
    if (__any(top > kFitMost)) {
        const float down = top > kFitMost ? ldexpf(1.f, kFitTo - __builtin_amdgcn_frexp_expf(top)) : 1.f;
        by *= down;
        dx *= down;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= down;
    }
    return dx;
}

// ---------------------------------------------------------------------------
// Scores, in units of log 2.
// ---------------------------------------------------------------------------

struct Cap {
    int mode;      // 0: none, 1: quick, 2: accurate
    float c;       // scale log2 e
    float k;       // 2 log2 e scale / cap
    float top;     // cap log2 e
    float inv;     // scale / cap
};

template <typename T>
inline Kind kind_of(const Att& a) {
    // a scale of 0 too: the others mask their products ahead of it, and -inf times 0 is none
    if (a.slopes || a.table || a.documents || a.scale == 0.f) return kGeneral;
    return a.cap <= 0.f ? kPlain : sizeof(T) == 2 && a.cap <= kQuickCap ? kCapped : kGeneral;
}

// (The forward has its rows' signs turned where the scale is negative, for the
// largest product to be the largest score; the gradients take it as it is.)
template <typename T, Kind KIND>
__device__ __forceinline__ Cap cap_of(const Att& a, bool backward) {
    Cap c;
    const float s = backward ? a.scale : fabsf(a.scale);
    c.mode = KIND == kPlain ? 0 : KIND == kCapped ? 1 : a.cap <= 0.f ? 0 : sizeof(T) == 2 && a.cap <= kQuickCap ? 1 : 2;
    c.c = s * kLog2e;
    c.inv = a.cap > 0.f ? s / a.cap : 0.f;
    c.k = 2.f * kLog2e * c.inv;
    c.top = a.cap * kLog2e;
    return c;
}

__device__ __forceinline__ float quick_r(float x, float k) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * k));
}

// tanh with a small relative error everywhere: its series up to x^11 below
// 0.3 (the next term is 2e-9 of it).
__device__ __forceinline__ float tanh_rel(float x) {
    const float y = x * x;
    float p = fma_acc(y, -1382.f / 155925.f, 62.f / 2835.f);
    p = fma_acc(y, p, -17.f / 315.f);
    p = fma_acc(y, p, 2.f / 15.f);
    p = fma_acc(y, p, -1.f / 3.f);
    p = fma_acc(y * x, p, x);
    const float q = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.f * kLog2e * fabsf(x)));
    return fabsf(x) < 0.3f ? p : copysignf(q, x);
}

// Raw products to scores, and the cap's derivative.  (Vectors go by value here
// and below: through references they have ended in scratch memory.)
struct Scores {
    f32x16 s, w;
};

// (w is left open without a cap: nothing reads it.)
template <bool SLOPE>
__device__ __forceinline__ Scores cap_scores(const Cap& c, f32x16 s) {
    Scores x;
    if (c.mode == 0) {
        x.s = s * c.c;
    } else if (c.mode == 1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float q = quick_r(s[r], c.k);
            x.s[r] = fma_acc(q, -2.f * c.top, c.top);
            if (SLOPE) x.w[r] = 4.f * fma_acc(-q, q, q);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float t = tanh_rel(s[r] * c.inv);
            x.s[r] = c.top * t;
            if (SLOPE) x.w[r] = fma_acc(-t, t, 1.f);
        }
    }
    return x;
}

// The bias of a lane's 16 pairs with relative positions rel0 + sign * el(r).
struct Bias {
    float slope;        // the lane's, in units of log 2
    const float* line;  // the table by relative position + reach, in LDS
};

template <int SIGN>
__device__ __forceinline__ f32x16 add_bias(const Att& a, const Bias& bs, int rel0, int least, int most,
                                           f32x16 s) {
    if (a.slopes) {
        const float f = static_cast<float>(rel0);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fma_acc(-bs.slope, fabsf(f + SIGN * el(r)), s[r]);
    }
    if (!a.table) return s;
    if (most <= -a.reach || least >= a.reach) {  // the tile's extremes: one value
        const float far = bs.line[least >= a.reach ? 2 * a.reach : 0];
        s += far;
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            int rel = rel0 + SIGN * el(r);
            rel = min(max(rel, -a.reach), a.reach);
            s[r] += bs.line[rel + a.reach];
        }
    }
    return s;
}

// The head's table by relative position, in units of log 2, by all threads.
template <typename T>
__device__ __forceinline__ void stage_line(const Att& a, int h, float* line) {
    for (int r = threadIdx.x; r <= 2 * a.reach; r += kAttThreads)
        line[r] = table_value<T>(a, h, r - a.reach);
}

// ---------------------------------------------------------------------------
// Which workgroup does what.  Workgroups are dealt to the eight XCDs in turn;
// where the head groups divide among them, an XCD keeps its groups, whose keys
// then stay in its L2.  Late rows of a causal call see the most: they go first.
// ---------------------------------------------------------------------------

__device__ __forceinline__ void place(int n, int groups, int& group, int& rest) {
    const int x = n % groups;
    rest = n / groups;
    group = groups % 8 == 0 ? (x % 8) * (groups / 8) + x / 8 : x;
}

// Which of a run of tiles are needed, 64 at a time.
template <typename F>
struct Needed {
    F f;
    unsigned long long bits = 0;
    int w = -1;
    __device__ __forceinline__ bool operator()(int t) {
        if (t >> 6 != w) {
            w = t >> 6;
            bits = __ballot(f((w << 6) + (threadIdx.x & 63)));
        }
        return bits >> (t & 63) & 1;
    }
    // The first needed tile from t on, or end.
    __device__ __forceinline__ int next(int t, int end) {
        while (t < end) {
            (*this)(t);
            const unsigned long long left = bits >> (t & 63);
            if (left) {
                t += __builtin_ctzll(left);
                return t < end ? t : end;
            }
            t = ((t >> 6) + 1) << 6;
        }
        return end;
    }
};

}  // namespace nsh
