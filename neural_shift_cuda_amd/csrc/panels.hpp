// panels.hpp -- products of two matrices by panels in LDS, for fp16, bf16 and
// fp32, whichever way each of them runs in memory.
//
//   out[m][n] = sum_k second[m][k] first[n][k]
//
// A workgroup owns BM x BN of the result.  Of both matrices it takes KB bytes of the
// contraction at a time (BK elements) straight from memory to LDS, one panel ahead of the
// products (two in the smallest tiles): with the contraction running along the rows (`kAlong`, one LDS row
// for each row of the result) or across them (`kAcross`, one LDS row for each
// contraction step, read by columns).  The chunk order within an LDS row is
// attention_tiles.hpp's, free of bank conflicts both ways.
//
// A wave has WM x WN of the result in 32 x 32 products with `first` on their first
// side, so a lane holds one row m and, of every 32 columns n, four times four next to
// each other.  The operands of a step are read while the products of the step before
// run, those of a panel's first step too: the panels change hands (one barrier) ahead
// of a panel's last products.
#pragma once

#include "attention_tiles.hpp"
#include "rows.hpp"

namespace nsh {

enum Run { kAlong, kAcross };

// How the lane's operands lie in a panel: DP is the LDS row's length.
template <typename T, int DP, Run RUN>
struct Operand {
    using L = Tile<T, DP>;
    using V = typename Eight<T>::V;
    static constexpr int READS = RUN == kAlong ? sizeof(T) / 2 : sizeof(T) == 2 ? 2 : 8;  // instructions of a read()

    // first: the wave's first row (or column) of the panel, a multiple of 32 (of
    // the wave's own width, if across)
    static __device__ __forceinline__ int base(int first, int l) {
        if constexpr (RUN == kAlong) {
            return L::at(first + (l & 31), (l >> 5));
        } else if constexpr (sizeof(T) == 2) {
            // a transposing read takes four rows by 16 columns from 16 lanes; a lane
            // half has eight contraction steps in a row, as along
            const int i = l & 15, d = first + (l & 16) + 4 * (i & 3);
            return L::at(8 * (l >> 5) + (i >> 2), d / 8) + (d & 7) * 2;
        } else {
            const int d = first + (l & 31);
            return L::at(4 * (l >> 5), d / 4) + (d & 3) * 4;
        }
    }

    // Step s (16 of the contraction) of the 32 rows or columns `on` further.
    static __device__ __forceinline__ V read(const char* lds, int base, int on, int s) {
        if constexpr (RUN == kAlong && sizeof(T) == 2) {
            return *reinterpret_cast<const V*>(lds + L::moved(base, 32 * s, on));
        } else if constexpr (RUN == kAlong) {  // steps 4 g .. and 8 + 4 g .., as across
            const f32x4 a = *reinterpret_cast<const f32x4*>(lds + L::moved(base, 64 * s, on));
            const f32x4 b = *reinterpret_cast<const f32x4*>(lds + L::moved(base, 64 * s + 32, on));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else if constexpr (sizeof(T) == 2) {
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NSH_LDS s16x4*)(lds + L::moved(base, on * 2, 16 * s)));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NSH_LDS s16x4*)(lds + L::moved(base, on * 2, 16 * s + 4)));
            return __builtin_bit_cast(V, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return L::col(lds, base, 16 * s, on / 32);
        }
    }
};

// A matrix's panel, from memory straight to LDS by NT lanes.  Rows past the matrix's end
// arrive as zeros (the buffer's range check), and along, columns past its end too.
template <typename T, int ROWS, int DP, int NT, Run RUN>
struct Panel {
    using L = Tile<T, DP>;
    static constexpr int NI = ROWS * L::NC / NT;
    static_assert(NI * NT == ROWS * L::NC, "whole instructions");
    // along, a lane has the same chunk of every row it loads
    static_assert(RUN == kAcross || (NT / L::NC) % 16 == 0, "whole sets of 16 rows");
    uint32_t off[NI];
    int chunk;

    __device__ __forceinline__ void init(uint32_t stride) {
        chunk = ((threadIdx.x % L::NC) ^ L::turn(threadIdx.x / L::NC)) * 16;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int x = i * NT + threadIdx.x, r = x / L::NC;
            off[i] = static_cast<uint32_t>(r) * stride + ((x % L::NC) ^ L::turn(r)) * 16;
        }
    }
    static __device__ __forceinline__ Panel either(bool first, const Panel& a, const Panel& b) {
        Panel p;
        p.chunk = a.chunk;
#pragma unroll
        for (int i = 0; i < NI; ++i) p.off[i] = first ? a.off[i] : b.off[i];
        return p;
    }
    // from: the panel's first row; rows: how many are left, from there (none: nothing is
    // read); left: bytes left of a row
    __device__ __forceinline__ void load(char* lds, const char* from, uint32_t stride, int rows, int64_t left, int wave) const {
        const uint32_t n = static_cast<uint32_t>(max(min(rows, ROWS), 0));
        const uint32_t last = static_cast<uint32_t>(min(left, static_cast<int64_t>(DP * sizeof(T))));
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(from), static_cast<short>(0), static_cast<int>(n ? (n - 1) * stride + last : 0u), 0x00020000);
        const bool past = RUN == kAlong && chunk >= static_cast<int>(last);
#pragma unroll
        for (int i = 0; i < NI; ++i) to_lds<16>(rs, lds + (i * (NT / 64) + wave) * 1024, past ? 0x80000000u : off[i]);
    }
};

// PAIRED: the wave's columns come in equal parts from the two halves of BN.
template <typename T_, int BM_, int BN_, int WAVES_M, int WAVES_N, int KB_, Run FIRST, Run SECOND, bool PAIRED_>
struct Product {
    using T = T_;
    using V = typename Eight<T>::V;
    static constexpr int BM = BM_, BN = BN_, KB = KB_, BK = KB / sizeof(T), STEPS = BK / 16;
    static constexpr int NT = 64 * WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N;
    static constexpr int MT = WM / 32, NB = WN / 32;
    static constexpr bool PAIRED = PAIRED_;
    using First = Operand<T, FIRST == kAlong ? BK : BN, FIRST>;
    using Second = Operand<T, SECOND == kAlong ? BK : BM, SECOND>;
    using FirstPanel = Panel<T, FIRST == kAlong ? (PAIRED ? BN / 2 : BN) : BK, FIRST == kAlong ? BK : BN, NT, FIRST>;
    using SecondPanel = Panel<T, SECOND == kAlong ? BM : BK, SECOND == kAlong ? BK : BM, NT, SECOND>;
    static constexpr int FIRST_BYTES = BN * KB, SECOND_BYTES = BM * KB, BYTES = FIRST_BYTES + SECOND_BYTES;
    static_assert(STEPS % 2 == 0 && (!PAIRED || (FIRST == kAlong && NB % 2 == 0)), "");

    // fp32: the sums of a chain of panels, 16 or 15, 512 of the contraction, are added to `whole`
    // and start anew.  (In one chain of 4096 the roundings of h came to 1.7e-6 of it, twice a
    // library's that shares a sum between workgroups.)
    static constexpr bool FOLD = sizeof(T) == 4;
    static constexpr int CHAIN2 = 16, CHAIN3 = 15;
    f32x16 acc[MT][NB], whole[FOLD ? MT : 1][FOLD ? NB : 1];
    int by_first, by_second;
    struct Step {
        V f[NB], s[MT];
    };

    static __device__ __forceinline__ int wave_m() { return wave_id() % WAVES_M; }
    static __device__ __forceinline__ int wave_n() { return wave_id() / WAVES_M; }
    // Where the wave's columns b start in the tile (PAIRED: b < NB / 2, in each half).
    static __device__ __forceinline__ int column(int b) { return wave_n() * (PAIRED ? WN / 2 : WN) + b * 32; }
    // The lane's row of block i.
    static __device__ __forceinline__ int row(int i) { return wave_m() * WM + i * 32 + (threadIdx.x & 31); }

    __device__ __forceinline__ void init() {
        const int l = threadIdx.x & 63;
        by_first = First::base(column(0), l);
        by_second = Second::base(wave_m() * WM, l);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[i][b] = f32x16{};
        if constexpr (FOLD) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b) whole[i][b] = f32x16{};
        }
    }
    // acc added to `whole`, and started anew or, LAST, with all of it.
    template <bool LAST>
    __device__ __forceinline__ void fold() {
        settle<T>();
        if constexpr (FOLD) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    whole[i][b] += acc[i][b];
                    acc[i][b] = LAST ? whole[i][b] : f32x16{};
                }
            order();
        }
    }
    __device__ __forceinline__ void read(Step& x, const char* panel, int s) const {
#pragma unroll
        for (int b = 0; b < NB; ++b)
            x.f[b] = First::read(panel, by_first, PAIRED && b >= NB / 2 ? BN / 2 + (b - NB / 2) * 32 : b * 32, s);
#pragma unroll
        for (int i = 0; i < MT; ++i) x.s[i] = Second::read(panel + FIRST_BYTES, by_second, i * 32, s);
    }
    template <int FROM, int TO>
    __device__ __forceinline__ void multiply(const Step& x) {
#pragma unroll
        for (int i = FROM; i < TO; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[i][b] = Eight<T>::mma(x.f[b], x.s[i], acc[i][b]);
    }

    static constexpr int LOADS = BYTES / (NT * 16);  // of a panel, a lane
    static constexpr int READS = NB * First::READS + MT * Second::READS;    // of a step
    static constexpr int ROW = NB * (sizeof(T) == 4 ? 8 : 1);               // products of 32 rows

    // The region's products with reads between them: a product issues in 4 cycles and
    // takes 32, and what stands in front of a run of them keeps it waiting.
    template <int ALL, int READS>
    static __device__ __forceinline__ void mix() {
#pragma unroll
        for (int i = 0; i < ALL; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            constexpr int R = (READS + ALL - 1) / ALL;
            if (i * R < READS) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
        }
        order();
    }

    // A panel's products but the last step's, which is read.
    __device__ __forceinline__ void steps(Step& x, Step& y, const char* b) {
#pragma unroll
        for (int st = 0; st + 1 < STEPS; ++st) {
            read(st % 2 ? x : y, b, st + 1);
            multiply<0, MT>(st % 2 ? y : x);
            mix<MT * ROW, READS>();
        }
    }
    // The panels change hands: the next one is there (but the loads of LATER others may be
    // under way) and everyone past this one's reads; its first step is read, and `ahead` asks
    // for the one that takes this one's place, during the last step's products.
    template <int LATER, typename Ahead>
    __device__ __forceinline__ void turn(Step& x, Step& y, const char* next, const Ahead& ahead) {
        landed<LATER>();
        read(x, next, 0);  // (behind the last panel nothing that is used)
        multiply<0, (MT + 1) / 2>(y);
        mix<(MT + 1) / 2 * ROW, READS>();
        ahead();
        order();
        multiply<(MT + 1) / 2, MT>(y);
        order();
    }

    // All n panels (n >= 1); load(i, first, second) asks for panel i.
    template <typename Load>
    __device__ __forceinline__ void run(int n, char (&b0)[BYTES], char (&b1)[BYTES], const Load& load) {
        Step x, y;
        load(0, b0, b0 + FIRST_BYTES);
        landed<0>();
        if (n > 1) load(1, b1, b1 + FIRST_BYTES);
        read(x, b0, 0);
        order();
        int first = 0;
        if constexpr (FOLD) {
            for (; first + CHAIN2 < n; first += CHAIN2) {
                for (int i = first; i < first + CHAIN2; i += 2) {
                    steps(x, y, b0);
                    turn<0>(x, y, b1, [&] { load(i + 2, b0, b0 + FIRST_BYTES); });
                    steps(x, y, b1);
                    turn<0>(x, y, b0, [&] { if (i + 3 < n) load(i + 3, b1, b1 + FIRST_BYTES); });
                }
                fold<false>();
            }
        }
        for (int i = first; i < n; i += 2) {
            steps(x, y, b0);
            turn<0>(x, y, b1, [&] { if (i + 2 < n) load(i + 2, b0, b0 + FIRST_BYTES); });
            if (i + 1 < n) {
                steps(x, y, b1);
                turn<0>(x, y, b0, [&] { if (i + 3 < n) load(i + 3, b1, b1 + FIRST_BYTES); });
            }
        }
        fold<true>();
    }

    // The same with two panels ahead.  From n on load() asks for nothing (a buffer of no
    // bytes): the compiler tells loads under way apart by their number, and a load that may
    // not be there would have it wait for all of them (as it does at the loop's head).
    template <typename Load>
    __device__ __forceinline__ void run(int n, char (&b0)[BYTES], char (&b1)[BYTES], char (&b2)[BYTES], const Load& load) {
        Step x, y;
        load(0, b0, b0 + FIRST_BYTES);
        load(1, b1, b1 + FIRST_BYTES);
        load(2, b2, b2 + FIRST_BYTES);
        landed<2 * LOADS>();
        read(x, b0, 0);
        order();
        int first = 0;
        if constexpr (FOLD) {
            for (; first + CHAIN3 < n; first += CHAIN3) {
                for (int i = first; i < first + CHAIN3; i += 3) {
                    steps(x, y, b0);
                    turn<LOADS>(x, y, b1, [&] { load(i + 3, b0, b0 + FIRST_BYTES); });
                    steps(x, y, b1);
                    turn<LOADS>(x, y, b2, [&] { load(i + 4, b1, b1 + FIRST_BYTES); });
                    steps(x, y, b2);
                    turn<LOADS>(x, y, b0, [&] { load(i + 5, b2, b2 + FIRST_BYTES); });
                }
                fold<false>();
            }
        }
        for (int i = first;; i += 3) {
            steps(x, y, b0);
            turn<LOADS>(x, y, b1, [&] { load(i + 3, b0, b0 + FIRST_BYTES); });
            if (i + 1 >= n) break;
            steps(x, y, b1);
            turn<LOADS>(x, y, b2, [&] { load(i + 4, b1, b1 + FIRST_BYTES); });
            if (i + 2 >= n) break;
            steps(x, y, b2);
            turn<LOADS>(x, y, b0, [&] { load(i + 5, b2, b2 + FIRST_BYTES); });
            if (i + 3 >= n) break;
        }
        fold<true>();
        landed<0>();  // what was asked for past the end has no place in what follows
    }

    // A place of the wave's own in the panels, for 32 x 64 in fp32.
    static __device__ __forceinline__ char* stage(char (&b0)[BYTES], char (&b1)[BYTES]) {
        constexpr int SIZE = 32 * 64 * 4, EACH = BYTES / SIZE;
        static_assert(2 * EACH >= NT / 64, "a place for every wave");
        const int w = wave_id();
        return w < EACH ? b0 + w * SIZE : b1 + (w - EACH) * SIZE;
    }

    // Every wave's loads but its last LATER ones have landed, and every wave has read what
    // it needs of the panel before.
    template <int LATER>
    static __device__ __forceinline__ void landed() {
        static_assert(LATER < 16, "");
        __builtin_amdgcn_s_waitcnt(0x0070 | LATER);  // vmcnt, lgkmcnt(0)
        if constexpr (LATER == 0)
            __syncthreads();
        else
            __builtin_amdgcn_s_barrier();
        order();
    }
};

// The order of result tiles: every XCD has a run of its own, in which `rows` rows of
// tiles advance together, so that its L2 serves both matrices.
struct TileOrder {
    int m, n;
    __device__ __forceinline__ TileOrder(uint32_t id, uint32_t count, int tiles_m, int tiles_n, int rows) {
        const uint32_t xcd = id % kXcds, local = id / kXcds, per = count / kXcds, rem = count % kXcds;
        const uint32_t t = xcd * per + min(xcd, rem) + local, band = static_cast<uint32_t>(rows) * tiles_n;
        const uint32_t group = t / band, in = t - group * band;
        const uint32_t first = group * rows, deep = min(static_cast<uint32_t>(tiles_m) - first, static_cast<uint32_t>(rows));
        n = uniform(in / deep);
        m = uniform(first + in % deep);
    }
    // (divisions come out of vector registers, and a load's buffer has to be in scalar ones)
    static __device__ __forceinline__ int uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
};

// Lanes that wrote to LDS and read what others of their wave wrote.
__device__ __forceinline__ void wave_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ROWS x COLS of a wave in LDS, between the products' order (a lane: row l % 32 of 32, and
// of 32 columns four times four) and rows of memory, 16 bytes a lane and as much of a row
// side by side as there is: stored from the products' order, 32 rows are 32 pieces of 32
// bytes.  The chunks of a row are permuted so that no bank is asked twice either way.
template <typename T, int ROWS, int COLS>
struct Stage {
    static constexpr int CHUNKS = COLS * sizeof(T) / 16, ROW = CHUNKS * 16, BYTES = ROWS * ROW;
    static constexpr int PER = CHUNKS < 16 ? 16 / CHUNKS : 1;  // rows that share 256 bytes
    static constexpr int TURNS = ROWS * CHUNKS / 64;
    static_assert(TURNS * 64 == ROWS * CHUNKS && CHUNKS >= 4, "whole instructions");

    static __device__ __forceinline__ int at(int row, int chunk) {
        return row * ROW + ((chunk ^ (row / PER % (CHUNKS < 16 ? CHUNKS : 16))) * 16);
    }
    // Block (i, b) of 32 x 32.
    static __device__ __forceinline__ void put(char* lds, int i, int b, const f32x16& v) {
        const int l = threadIdx.x & 63, row = i * 32 + (l & 31);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 x = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            if constexpr (sizeof(T) == 4)
                *reinterpret_cast<f32x4*>(lds + at(row, b * 8 + 2 * q + (l >> 5))) = x;
            else
                store4<T>(reinterpret_cast<T*>(lds + at(row, b * 4 + q) + (l >> 5) * 8), x);
        }
    }
    static __device__ __forceinline__ f32x16 get(const char* lds, int i, int b) {
        const int l = threadIdx.x & 63, row = i * 32 + (l & 31);
        f32x16 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (sizeof(T) == 4) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(lds + at(row, b * 8 + 2 * q + (l >> 5)));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * q + e] = x[e];
            } else {
                float x[4];
                load_acc<T, 4>(reinterpret_cast<const T*>(lds + at(row, b * 4 + q) + (l >> 5) * 8), x);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * q + e] = x[e];
            }
        }
        return v;
    }
    // To and from memory: `rows` rows of `cols` columns (more than there are, or none).
    static __device__ __forceinline__ void store(const char* lds, T* to, int64_t stride, int64_t rows, int64_t cols) {
        const int l = threadIdx.x & 63, n = static_cast<int>(min(cols, int64_t(COLS)));
#pragma unroll
        for (int t = 0; t < TURNS; ++t) {
            const int x = t * 64 + l, row = x / CHUNKS, chunk = x % CHUNKS;
            const ux4 v = *reinterpret_cast<const ux4*>(lds + at(row, chunk));
            if (row < rows) store_bits(to + row * stride, chunk * kVec<T>, n, v);
        }
    }
    static __device__ __forceinline__ void load(char* lds, const T* from, int64_t stride, int64_t rows, int64_t cols) {
        const int l = threadIdx.x & 63, n = static_cast<int>(min(cols, int64_t(COLS)));
        ux4 v[TURNS];
#pragma unroll
        for (int t = 0; t < TURNS; ++t) {
            const int x = t * 64 + l, row = x / CHUNKS, c = x % CHUNKS * kVec<T>;
            v[t] = ux4{0, 0, 0, 0};
            if (row < rows) v[t] = load_near<T, kShort>(from + row * stride, c, n);
        }
#pragma unroll
        for (int t = 0; t < TURNS; ++t) {
            const int x = t * 64 + l;
            in_place<T, kShort>(v[t], x % CHUNKS * kVec<T>, n);
            *reinterpret_cast<ux4*>(lds + at(x / CHUNKS, x % CHUNKS)) = v[t];
        }
    }
};

// A wave's tile to memory, 32 rows and 64 columns of it at a time through LDS.
template <typename T, int ROWS, int COLS, typename Value>
__device__ __forceinline__ void store_tile(char* lds, T* to, int64_t stride, int64_t rows, int64_t cols, const Value& value) {
    constexpr int PART = COLS < 64 ? COLS : 64;
    using S = Stage<T, 32, PART>;
#pragma unroll
    for (int i = 0; i < ROWS / 32; ++i)
#pragma unroll
        for (int c = 0; c < COLS; c += PART) {
#pragma unroll
            for (int b = 0; b < PART / 32; ++b) S::put(lds, 0, b, value(i, c / 32 + b));
            wave_exchange();
            S::store(lds, to + i * 32 * stride + c, stride, rows - i * 32, cols - c);
            wave_exchange();
        }
}

}  // namespace nsh
