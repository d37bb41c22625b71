// positionbias.hip -- a learned relative position bias by buckets, written out
// for every head, query and key, and its gradient, on gfx950.
//
//   out[h, i, j] = table[buckets[clamp(j - (i + Lk - Lq), -R, R) + R], h]
//   gtable[w, h] = sum of gout[h, i, j] over the places of bucket w
//
// Forward: a stream of 16-byte stores.  A workgroup stages its head's value of
// each of the 2R + 1 relative positions in LDS and writes a run of the head's
// places; a vector whose places are all beyond R takes one value.
// Backward: a read of every element once.  A workgroup takes kBiasRows rows of
// a head, which are one run of memory: 16 bytes a lane, for the two far ends of
// every row, one relative position each.  Within the reach, a thread then owns
// relative positions and walks the rows along its diagonals (neighbouring lanes
// read neighbouring elements), which are in the caches by then.  The
// sums per relative position go to a workspace, and one workgroup per head adds
// them, first over the workgroups, then over each bucket's relative positions:
// all in a fixed order.
//
// 16 heads, 2048 x 2048, fp32 (268 MB): forward 51 us (5.3 TB/s), backward 72
// (3.7 TB/s; 54 where the upstream gradient is the same each time and the memory
// side cache has some of it) and 6.5 for the table's sums; a copy of 268 MB runs at
// 5.4 TB/s, a library sum over as much at 3.6, a plain read at 6.2.  Both are bound by
// memory; the backward's second reads, along the diagonals, cost it the rest.  Its
// sums are fp32 throughout (off by 1.8e-7 of the whole, where rounding the result
// alone makes 2.2e-8).
#include <algorithm>

#include "divisor.hpp"
#include "positionbias.hpp"

namespace nsh {

constexpr int kBiasThreads = 256;
constexpr int kBiasVectors = 8;  // vectors of the output per thread
constexpr int kBiasRows = 16;    // rows per workgroup of the backward

// STREAM: stores past the caches, for an output that they do not hold anyhow:
// kept there, its lines are written out while the next kernel reads (16 heads,
// 2048 x 2048, fp32, 268 MB: forward 42 us, and the backward after it 104;
// streamed 52 and 64).
constexpr int64_t kStreamBytes = int64_t(128) << 20;

template <typename T, int VEC, bool STREAM>
__global__ __launch_bounds__(kBiasThreads) void bias_fwd_kernel(
    const T* __restrict__ table, const int32_t* __restrict__ buckets, int H, int Lq, int Lk,
    int nb, int R, T* __restrict__ out) {
    __shared__ T line[2 * kMaxReach + 1];
    const int h = blockIdx.y;
    for (int r = threadIdx.x; r <= 2 * R; r += kBiasThreads) {
        const int w = buckets[r];
        line[r] = w >= 0 && w < nb ? table[static_cast<int64_t>(w) * H + h]
                                   : from_acc<T>(__builtin_nanf(""));
    }
    __syncthreads();
    const int64_t n = static_cast<int64_t>(Lq) * Lk;
    T* o = out + h * n;
    // the head's first whole vector of the output
    const int lead = static_cast<int>((VEC - (h * n) % VEC) % VEC);
    const int64_t e0 = lead + static_cast<int64_t>(blockIdx.x) * (kBiasThreads * kBiasVectors * VEC);
    const int off = Lk - Lq;
    auto value = [&](int i, int j) {
        int rel = j - i - off;
        rel = rel < -R ? -R : (rel > R ? R : rel);
        return line[rel + R];
    };
    if (blockIdx.x == 0 && static_cast<int>(threadIdx.x) < lead && threadIdx.x < n) {
        const int e = threadIdx.x;
        o[e] = value(e / Lk, e % Lk);
    }
    const int64_t base_i = e0 / Lk;
    const int base_j = static_cast<int>(e0 - base_i * Lk);
#pragma unroll
    for (int t = 0; t < kBiasVectors; ++t) {
        const int x = (t * kBiasThreads + threadIdx.x) * VEC;
        const int64_t e = e0 + x;
        if (e >= n) break;
        const unsigned jj = static_cast<unsigned>(base_j) + x;
        const unsigned down = jj / static_cast<unsigned>(Lk);
        int i = static_cast<int>(base_i) + static_cast<int>(down);
        int j = static_cast<int>(jj - down * static_cast<unsigned>(Lk));
        if (e + VEC <= n) {
            Pack<T, VEC> v;
            const int first = j - i - off;
            if (j + VEC <= Lk && (first >= R || first + VEC - 1 <= -R)) {
                const T far = line[first >= R ? 2 * R : 0];
#pragma unroll
                for (int k = 0; k < VEC; ++k) v.e[k] = far;
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    v.e[k] = value(i, j);
                    if (++j == Lk) j = 0, ++i;
                }
            }
            if constexpr (STREAM) store_pack_nt<T, VEC>(o + e, v);
            else store_pack<T, VEC>(o + e, v);
        } else {
            for (int k = 0; e + k < n; ++k) {
                o[e + k] = value(i, j);
                if (++j == Lk) j = 0, ++i;
            }
        }
    }
}

// This workgroup's share of a head's far sums: 16 bytes a lane, eight loads
// under way, in turns with the head's other workgroups, so that at any time
// they read one stretch of memory.  A vector across a border of the reach, or of
// a row, is taken apart.
constexpr int kWay = 8;

template <typename T, int VEC>
__device__ __forceinline__ void far_sums(const T* g, uint32_t n, int Lk, Divisor by_lk, int first, int off, int R,
                                         float& low, float& high) {
    const uint32_t cut = static_cast<uint32_t>((VEC - reinterpret_cast<uintptr_t>(g) / sizeof(T) % VEC) % VEC);
    const uint32_t lead = cut < n ? cut : n, whole = (n - lead) / VEC;
    auto one = [&](uint32_t e) {
        const uint32_t row = by_lk(e);
        const int rel = static_cast<int>(e - row * Lk) - (first + static_cast<int>(row) + off);
        const float v = to_acc(g[e]);
        if (rel <= -R) low += v;
        else if (rel >= R) high += v;
    };
    auto take = [&](uint32_t k, const float (&v)[VEC]) {
        const uint32_t e = lead + k * VEC;
        const uint32_t row = by_lk(e);
        int j = static_cast<int>(e - row * Lk), rel = j - (first + static_cast<int>(row) + off);
        const bool split = j + VEC > Lk;
        float u = v[0];
#pragma unroll
        for (int c = 1; c < VEC; ++c) u += v[c];
        if (!split && (rel + VEC - 1 <= -R || rel >= R)) {
            (rel >= R ? high : low) += u;
        } else if (split || rel <= -R || rel + VEC - 1 >= R) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                if (rel <= -R) low += v[c];
                else if (rel >= R) high += v[c];
                ++rel;
                if (++j == Lk) j = 0, rel -= Lk + 1;
            }
        }
    };
    for (Turns turn = Turns::of(blockIdx.x, gridDim.x, kWay * kBiasThreads); turn.at < whole; turn.at += turn.step) {
        const uint32_t at = static_cast<uint32_t>(turn.at), k = at + threadIdx.x;
        if (at + kWay * kBiasThreads <= whole) {
            Pack<T, VEC> p[kWay];
#pragma unroll
            for (int w = 0; w < kWay; ++w) p[w] = load_pack<T, VEC>(g + lead + (k + w * kBiasThreads) * VEC);
#pragma unroll
            for (int w = 0; w < kWay; ++w) {
                float v[VEC];
#pragma unroll
                for (int c = 0; c < VEC; ++c) v[c] = to_acc(p[w].e[c]);
                take(k + w * kBiasThreads, v);
            }
        } else {
            for (uint32_t x = k; x < whole; x += kBiasThreads) {
                float v[VEC];
                load_acc<T, VEC>(g + lead + x * VEC, v);
                take(x, v);
            }
        }
    }
    if (blockIdx.x) return;
    if (threadIdx.x < lead) one(threadIdx.x);
    const uint32_t tail = lead + whole * VEC + threadIdx.x;
    if (tail < n) one(tail);
}

template <typename T, int VEC>
__global__ __launch_bounds__(kBiasThreads) void bias_bwd_kernel(const T* __restrict__ go, int Lq,
                                                                int Lk, Divisor by_lk, int R,
                                                                float* __restrict__ partial) {
    __shared__ float ends[2][kBiasThreads / 64];
    const int h = blockIdx.y, i0 = blockIdx.x * kBiasRows, i1 = min(Lq, i0 + kBiasRows);
    const int off = Lk - Lq, t = threadIdx.x;
    const T* g = go + static_cast<int64_t>(h) * Lq * Lk;
    float* part = partial + (static_cast<int64_t>(h) * gridDim.x + blockIdx.x) * (2 * R + 1);
    float low = 0.f, high = 0.f;
    const int most = static_cast<int>(min(static_cast<int64_t>(Lq), (int64_t(1) << 30) / Lk));  // rows with 31-bit places
    for (int i = 0; i < Lq; i += most)
        far_sums<T, VEC>(g + static_cast<int64_t>(i) * Lk, static_cast<uint32_t>(min(most, Lq - i)) * Lk, Lk, by_lk,
                         i, off, R, low, high);
    for (int r = t - R + 1; r < R; r += kBiasThreads) {  // of what the far sums have just brought in
        float s = 0.f;
#pragma unroll 8
        for (int i = i0; i < i1; ++i) {
            const int j = r + i + off;
            if (j >= 0 && j < Lk) s += to_acc(g[static_cast<int64_t>(i) * Lk + j]);
        }
        part[r + R] = s;
    }
    const int wave = t / 64, lane = t % 64;
#pragma unroll
    for (int k = 32; k; k >>= 1) low += __shfl_xor(low, k), high += __shfl_xor(high, k);
    if (lane == 0) ends[0][wave] = low, ends[1][wave] = high;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < kBiasThreads / 64; ++w) low += ends[0][w], high += ends[1][w];
        if (R == 0)
            part[0] = low + high;
        else
            part[0] = low, part[2 * R] = high;
    }
}

template <typename T>
__global__ __launch_bounds__(kTableThreads) void table_gradient_kernel(
    const float* __restrict__ partial, const int32_t* __restrict__ buckets, int H, int64_t chunks,
    int nb, int R, T* __restrict__ out) {
    __shared__ float sum[2 * kMaxReach + 1];
    __shared__ int id[2 * kMaxReach + 1];
    __shared__ float run_sum[kTableThreads];
    const int h = blockIdx.x, n = 2 * R + 1;
    const float* p = partial + h * chunks * n;
    // several runs of chunks at once where the positions leave threads over
    const int runs = n < kTableThreads ? kTableThreads / n : 1, run = threadIdx.x / n;
    const int64_t len = (chunks + runs - 1) / runs, c0 = runs > 1 ? run * len : 0;
    const int64_t c1 = c0 + len < chunks ? c0 + len : chunks;
    for (int r = runs > 1 ? threadIdx.x - run * n : threadIdx.x; r < n && (runs == 1 || run < runs); r += kTableThreads) {
        float s = 0.f;
#pragma unroll 8
        for (int64_t c = c0; c < c1; ++c) s += p[c * n + r];
        if (runs > 1) run_sum[threadIdx.x] = s;
        else sum[r] = s;
    }
    for (int r = threadIdx.x; r < n; r += kTableThreads) id[r] = buckets[r];
    __syncthreads();
    if (runs > 1) {
        if (static_cast<int>(threadIdx.x) < n) {
            float s = 0.f;
            for (int i = 0; i < runs; ++i) s += run_sum[i * n + threadIdx.x];
            sum[threadIdx.x] = s;
        }
        __syncthreads();
    }
    const int lane = threadIdx.x % 64;
    for (int w = threadIdx.x / 64; w < nb; w += kTableThreads / 64) {
        float s = 0.f;
        for (int r = lane; r < n; r += 64) s += id[r] == w ? sum[r] : 0.f;
#pragma unroll
        for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
        if (lane == 0) out[static_cast<int64_t>(w) * H + h] = from_acc<T>(s);
    }
}

int table_gradient(const float* partial, const int32_t* buckets, int64_t H, int64_t chunks,
                   int64_t nb, int64_t R, int dtype, void* out, hipStream_t st) {
    const int n = static_cast<int>(nb), r = static_cast<int>(R), heads = static_cast<int>(H);
    const unsigned grid = static_cast<unsigned>(H);
    if (dtype == NSH_DTYPE_FLOAT16)
        table_gradient_kernel<f16><<<grid, kTableThreads, 0, st>>>(partial, buckets, heads, chunks, n, r, static_cast<f16*>(out));
    else if (dtype == NSH_DTYPE_BFLOAT16)
        table_gradient_kernel<bf16><<<grid, kTableThreads, 0, st>>>(partial, buckets, heads, chunks, n, r, static_cast<bf16*>(out));
    else
        table_gradient_kernel<float><<<grid, kTableThreads, 0, st>>>(partial, buckets, heads, chunks, n, r, static_cast<float*>(out));
    return nsh_host::check_launch("table_gradient");
}

static int bias_check(const char* op, int64_t H, int64_t Lq, int64_t Lk, int64_t nb, int64_t R,
                      int dtype) {
    if (H < 1 || Lq < 1 || Lk < 1 || nb < 1) return nsh_host::fail(NSH_ERR_INVALID, "%s: empty tensor", op);
    if (H > 65535 || Lq > (1 << 28) || Lk > (1 << 28))
        return nsh_host::fail(NSH_ERR_INVALID, "%s: up to 65535 heads and 2^28 rows and columns are served", op);
    if (R < 0 || R > kMaxReach || nb > 2 * kMaxReach + 1)
        return nsh_host::fail(NSH_ERR_INVALID, "%s: reach must be 0..%d, with up to %d buckets", op, kMaxReach,
                              2 * kMaxReach + 1);
    if (dtype < NSH_DTYPE_FLOAT16 || dtype > NSH_DTYPE_FLOAT32)
        return nsh_host::fail(NSH_ERR_INVALID, "%s: unsupported dtype code %d", op, dtype);
    return NSH_OK;
}

template <typename T>
static int bias_forward(const void* table, const int32_t* buckets, int64_t H, int64_t Lq,
                        int64_t Lk, int64_t nb, int64_t R, void* out, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const dim3 grid(static_cast<unsigned>(
                        nsh_host::ceil_div(Lq * Lk, static_cast<int64_t>(kBiasThreads) * kBiasVectors * V)),
                    static_cast<unsigned>(H));
    const auto kernel = H * Lq * Lk * static_cast<int64_t>(sizeof(T)) >= kStreamBytes ? bias_fwd_kernel<T, V, true>
                                                                                     : bias_fwd_kernel<T, V, false>;
    kernel<<<grid, kBiasThreads, 0, st>>>(
        static_cast<const T*>(table), buckets, static_cast<int>(H), static_cast<int>(Lq),
        static_cast<int>(Lk), static_cast<int>(nb), static_cast<int>(R), static_cast<T*>(out));
    return nsh_host::check_launch("position_bias_forward");
}

template <typename T>
static int bias_backward(const void* go, const int32_t* buckets, int64_t H, int64_t Lq, int64_t Lk,
                         int64_t nb, int64_t R, int dtype, void* gt, float* partial,
                         hipStream_t st) {
    const int64_t chunks = nsh_host::ceil_div(Lq, kBiasRows);
    bias_bwd_kernel<T, 16 / sizeof(T)>
        <<<dim3(static_cast<unsigned>(chunks), static_cast<unsigned>(H)), kBiasThreads, 0, st>>>(
            static_cast<const T*>(go), static_cast<int>(Lq), static_cast<int>(Lk),
            Divisor::of(static_cast<uint32_t>(Lk)), static_cast<int>(R), partial);
    if (int rc = nsh_host::check_launch("position_bias_backward")) return rc;
    return table_gradient(partial, buckets, H, chunks, nb, R, dtype, gt, st);
}

}  // namespace nsh

using nsh_host::fail;

extern "C" int nsh_position_bias_forward(const void* table, const int32_t* buckets, int64_t H,
                                         int64_t Lq, int64_t Lk, int64_t num_buckets, int64_t reach,
                                         int dtype, void* out, void* stream) {
    if (int rc = nsh::bias_check("position_bias_forward", H, Lq, Lk, num_buckets, reach, dtype)) return rc;
    if (!table || !buckets || !out || !nsh_host::aligned(out, 16))
        return fail(NSH_ERR_INVALID, "position_bias_forward: null pointer argument, or out not on 16 bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case NSH_DTYPE_FLOAT16: return nsh::bias_forward<nsh::f16>(table, buckets, H, Lq, Lk, num_buckets, reach, out, st);
        case NSH_DTYPE_BFLOAT16: return nsh::bias_forward<nsh::bf16>(table, buckets, H, Lq, Lk, num_buckets, reach, out, st);
        default: return nsh::bias_forward<float>(table, buckets, H, Lq, Lk, num_buckets, reach, out, st);
    }
}

extern "C" int64_t nsh_position_bias_workspace_bytes(int64_t H, int64_t Lq, int64_t Lk, int64_t reach) {
    if (H < 1 || Lq < 1 || Lk < 1 || reach < 0 || reach > nsh::kMaxReach) return -1;
    return H * nsh_host::ceil_div(Lq, nsh::kBiasRows) * (2 * reach + 1) * 4;
}

extern "C" int nsh_position_bias_backward(const void* grad_out, const int32_t* buckets, int64_t H,
                                          int64_t Lq, int64_t Lk, int64_t num_buckets,
                                          int64_t reach, int dtype, void* grad_table,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = nsh::bias_check("position_bias_backward", H, Lq, Lk, num_buckets, reach, dtype)) return rc;
    if (!grad_out || !buckets || !grad_table || !workspace)
        return fail(NSH_ERR_INVALID, "position_bias_backward: null pointer argument");
    if (workspace_bytes < nsh_position_bias_workspace_bytes(H, Lq, Lk, reach))
        return fail(NSH_ERR_INVALID, "position_bias_backward: workspace smaller than "
                    "nsh_position_bias_workspace_bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(workspace);
    switch (dtype) {
        case NSH_DTYPE_FLOAT16: return nsh::bias_backward<nsh::f16>(grad_out, buckets, H, Lq, Lk, num_buckets, reach, dtype, grad_table, ws, st);
        case NSH_DTYPE_BFLOAT16: return nsh::bias_backward<nsh::bf16>(grad_out, buckets, H, Lq, Lk, num_buckets, reach, dtype, grad_table, ws, st);
        default: return nsh::bias_backward<float>(grad_out, buckets, H, Lq, Lk, num_buckets, reach, dtype, grad_table, ws, st);
    }
}
