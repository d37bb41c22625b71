// rows.hpp -- 16 bytes of a row at a time, whatever it is aligned to, and sums
// over groups of lanes.
#pragma once

#include "nsh_common.hpp"

namespace nsh {

typedef float fx8 __attribute__((ext_vector_type(8)));
typedef float fx4 __attribute__((ext_vector_type(4)));
typedef uint32_t ux4 __attribute__((ext_vector_type(4)));

template <typename T> constexpr int kVec = 16 / sizeof(T);

// Columns c .. c + kVec - 1 of a row of n, those past its end as zeros.  Rows need
// no alignment beyond an element's: gfx950 splits a load that crosses a line.
// WHOLE: n is a multiple of kVec (the path by elements costs a kernel up to a hundred
// registers).
template <typename T, bool WHOLE = false>
__device__ __forceinline__ ux4 load_bits(const T* row, int c, int n) {
    ux4 r = {0, 0, 0, 0};
    if constexpr (WHOLE) {
        if (c < n) __builtin_memcpy(&r, row + c, 16);
    } else if (c + kVec<T> <= n) {
        __builtin_memcpy(&r, row + c, 16);
    } else if (c < n) {
        T e[kVec<T>] = {};
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k)
            if (c + k < n) e[k] = row[c + k];
        __builtin_memcpy(&r, e, 16);
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void unpack(ux4 r, float (&o)[kVec<T>]) {
    const Pack<T, kVec<T>> v = __builtin_bit_cast(Pack<T, kVec<T>>, r);
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k) o[k] = to_acc(v.e[k]);
}

// Rounded to nearest even by the conversion instructions.
template <typename T>
__device__ __forceinline__ ux4 pack(const float (&v)[kVec<T>]) {
    if constexpr (__is_same(T, float)) {
        return __builtin_bit_cast(ux4, (fx4{v[0], v[1], v[2], v[3]}));
    } else {
        const fx8 f = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
        if constexpr (__is_same(T, bf16)) {
            typedef __bf16 V __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(ux4, __builtin_convertvector(f, V));
        } else {
            typedef _Float16 V __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(ux4, __builtin_convertvector(f, V));
        }
    }
}

template <typename T, bool WHOLE = false>
__device__ __forceinline__ void store_bits(T* row, int c, int n, ux4 r) {
    if constexpr (WHOLE) {
        if (c < n) __builtin_memcpy(row + c, &r, 16);
    } else if (c + kVec<T> <= n) {
        __builtin_memcpy(row + c, &r, 16);
    } else if (c < n) {
        T e[kVec<T>];
        __builtin_memcpy(e, &r, 16);
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k)
            if (c + k < n) row[c + k] = e[k];
    }
}

// How a lane past a row's end, or with less than kVec columns left, loads.
//   kMasked: not at all (rows of whole vectors)
//   kNear: the row's last kVec, which in_place() brings to where they belong, zeros behind
//     them.  Every lane loads: a load that may not be there has the compiler wait for all that
//     are under way, and single elements would be loads of their own, one after the other.
//   kShort: so, and by elements where the row has less than kVec.
enum Reach { kMasked, kNear, kShort };

template <typename T, Reach REACH>
__device__ __forceinline__ ux4 load_near(const T* row, int c, int n) {
    if constexpr (REACH == kMasked) return load_bits<T, true>(row, c, n);
    if (REACH == kShort && n < kVec<T>) return load_bits(row, c, n);
    ux4 r;
    __builtin_memcpy(&r, row + min(c, n - kVec<T>), 16);
    return r;
}
template <typename T, Reach REACH, bool WHOLE = false>
__device__ __forceinline__ void in_place(ux4& r, int c, int n) {
    if constexpr (REACH == kMasked) return;
    const int past = c + kVec<T> - n;
    if (REACH == kShort && n < kVec<T>) return;
    if (WHOLE ? past > 0 : past >= kVec<T>)
        r = ux4{0, 0, 0, 0};
    else if (!WHOLE && past > 0)
        r = __builtin_bit_cast(ux4, __builtin_bit_cast(unsigned __int128, r) >> (past * 8 * static_cast<int>(sizeof(T))));
}
template <typename T, Reach REACH, bool WHOLE = false>
__device__ __forceinline__ ux4 load_row(const T* row, int c, int n) {
    ux4 r = load_near<T, REACH>(row, c, n);
    in_place<T, REACH, WHOLE>(r, c, n);
    return r;
}

template <int CTRL>
__device__ __forceinline__ float lane_moved(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}

// Over G lanes that stand side by side, in every one of them (no LDS).
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
    v += lane_moved<0xB1>(v);   // lane ^ 1
    v += lane_moved<0x4E>(v);   // lane ^ 2
    v += lane_moved<0x141>(v);  // mirrored in eight lanes, whose fours agree
    if constexpr (G >= 16) v += lane_moved<0x140>(v);  // mirrored in 16
    if constexpr (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// The largest of a workgroup's THREADS numbers, in all of them; lds: one for each wave.
template <int THREADS>
__device__ __forceinline__ float workgroup_max(float v, float* lds) {
    v = fmaxf(v, lane_moved<0xB1>(v));
    v = fmaxf(v, lane_moved<0x4E>(v));
    v = fmaxf(v, lane_moved<0x141>(v));
    v = fmaxf(v, lane_moved<0x140>(v));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v = fmaxf(v, lds[w]);
    __syncthreads();
    return v;
}

}  // namespace nsh
