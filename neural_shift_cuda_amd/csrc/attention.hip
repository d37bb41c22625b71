// attention.hip -- attention over tokens with capped scores, distance biases
// and masks: the entries' checks, how a call is cut into workgroups, and the
// document ranges by which tiles are passed over.
#include <algorithm>
#include <cmath>

#include "attention.hpp"
#include "positionbias.hpp"

namespace nsh {

// Lowest and highest document of every kRangeKeys keys (padding left out):
// one wave per range.
__global__ __launch_bounds__(kAttThreads) void att_ranges_kernel(Att a, int2* out) {
    const int e = blockIdx.x * kAttWaves + (threadIdx.x >> 6), b = blockIdx.y;
    if (e >= a.nranges) return;
    const int j = e * kRangeKeys + (threadIdx.x & 63);
    const int d = j < a.Lk ? a.documents[static_cast<int64_t>(b) * a.Lk + j] : -1;
    const int lo = wave_min(d >= 0 ? d : 0x7fffffff), hi = wave_max(d);
    if ((threadIdx.x & 63) == 0) out[static_cast<int64_t>(b) * a.nranges + e] = make_int2(lo, hi);
}

static int ranges_launch(const Att& a, hipStream_t st) {
    for (int b = 0; b < a.B; b += 65535) {  // the grid's second side
        Att c = a;
        c.documents += static_cast<int64_t>(b) * a.Lk;
        att_ranges_kernel<<<dim3(nsh_host::ceil_div(a.nranges, kAttWaves), std::min(a.B - b, 65535)), kAttThreads, 0, st>>>(
            c, const_cast<int2*>(a.ranges) + static_cast<int64_t>(b) * a.nranges);
    }
    return nsh_host::check_launch("attention_ranges");
}

// Document numbers of any 64-bit size as int32: each becomes the place where it
// first stands in its row, so equal ones stay equal, the rising numbers of packed
// rows stay rising, and the ranges above stay narrow; negative ones become -1.  A
// wave takes 64 places and looks up their numbers, one after the other, from the
// row's start on, 256 places a step.
constexpr int kLookups = 4;  // loads under way
__global__ __launch_bounds__(kAttThreads) void document_ids_kernel(const int64_t* __restrict__ ids, int64_t B, int64_t L,
                                                                   int64_t waves, int32_t* __restrict__ out) {
    const int l = threadIdx.x & 63;
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * kAttWaves + (threadIdx.x >> 6); w < B * waves;
         w += static_cast<int64_t>(gridDim.x) * kAttWaves) {
        const int64_t b = w / waves, j = (w - b * waves) * 64 + l;
        const int64_t* row = ids + b * L;
        const int64_t mine = j < L ? row[j] : -1;
        int64_t first = -1;
        for (unsigned long long open = __ballot(mine >= 0); open;) {
            const int64_t id = __shfl(mine, __builtin_ctzll(open));
            const unsigned long long same = __ballot(mine == id);
            int64_t at = -1;
            for (int64_t i0 = 0; at < 0; i0 += 64 * kLookups) {  // its own place ends the search
                int64_t v[kLookups];
#pragma unroll
                for (int c = 0; c < kLookups; ++c) v[c] = i0 + c * 64 + l < L ? row[i0 + c * 64 + l] : -1;
#pragma unroll
                for (int c = 0; c < kLookups; ++c) {
                    const unsigned long long hit = __ballot(v[c] == id);
                    if (hit && at < 0) at = i0 + c * 64 + __builtin_ctzll(hit);
                }
                if (i0 > L) break;
            }
            if (same >> l & 1) first = at;
            open &= ~same;
        }
        if (j < L) out[b * L + j] = static_cast<int32_t>(first);
    }
}

// The cut of a call, from its sizes alone (workspace sizes come from here too).
//
// Rows go 128 to a workgroup where that gives every CU one; otherwise 32, and
// the workgroup's waves split the keys.  (4 x 12 heads, 1024 tokens, width 64,
// bf16, a learned bias, 384 workgroups of 128: forward 43 us, gradients by rows 65;
// split 55 and 129.)  A forward short of workgroups even so
// (single tokens over a cache) shares a row block's keys among `splits` more,
// up to what the CUs hold at once (one of these workgroups where its tiles take
// most of the LDS, or two), as long as a wave keeps four tiles of 32 keys, or
// two in fp32, whose products take 16 times as long.  16 x 32 heads, 8 of keys,
// one token over 8192, bf16: 82 us in all with two workgroups for every CU,
// 77 with one; 2 x 5 heads, 333 over 517 tokens, fp32: 34 us with four tiles
// kept, 30 with two; 8 heads, one token over 500, fp16: 10.8 with four, 11.4
// with two.
// Fewer rows than a wave holds (32) take the rows of all the heads of a key head
// side by side, which then reads its keys once; a bias table is staged for one
// head, and keeps to one.
static void cut_rows(Att& a, bool backward) {
    const int64_t cus = nsh_host::compute_units();
    a.pack = !backward && a.Lq < 32 && !a.table ? a.per : 1;
    const int64_t rows = static_cast<int64_t>(a.Lq) * a.pack, groups = static_cast<int64_t>(a.B) * (a.Hq / a.pack);
    a.splits = 0;
    a.rblocks = static_cast<int>(nsh_host::ceil_div(rows, int64_t(128)));
    if (groups * a.rblocks >= cus) return;
    if (backward && a.gtable && !attention_split_fits(a)) return;
    a.rblocks = static_cast<int>(nsh_host::ceil_div(rows, int64_t(32)));
    a.splits = 1;
    if (backward) return;
    const int64_t blocks = groups * a.rblocks, keep = (a.wide ? 2 : 4) * kAttWaves;
    const int64_t room = cus * (a.D * (a.wide ? 4 : 2) > 128 ? 1 : 2);
    a.splits = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>({room / blocks, nsh_host::ceil_div(a.Lk, 32) / keep, 64})));
}

// Keys go key_block() to a workgroup.  `parts` workgroups share a key block's queries
// where there are too few of them to go round, as long as each keeps two query
// tiles; the third launch that adds up their sums costs more than it brings from
// five workgroups to four CUs on.  As the rule was set: 4 x 12 heads, 1024 tokens,
// width 64, bf16 (384 workgroups, then of 128 keys): 86 us alone, 92 + 16 with two
// parts; 2 x 16 heads, 4 of keys, 4096 tokens, width 128, causal (256): 791 alone,
// 500 + 18 (now 324 + 17); 2 x 5 heads, 333 over 517 tokens, fp32: 60 + 5 with four
// tiles kept, 38 + 5 with two, 48 + 8 with one.
static void cut_keys(Att& a) {
    const int64_t cus = nsh_host::compute_units(), tile = a.wide ? 32 : 64;
    a.kblocks = static_cast<int>(nsh_host::ceil_div(a.Lk, key_block(a.wide ? 4 : 2, a.D)));
    const int64_t blocks = static_cast<int64_t>(a.B) * a.Hk * a.kblocks;
    const int64_t units = nsh_host::ceil_div(a.Lq, tile) * a.per;
    a.parts = 1;
    if (4 * blocks < 5 * cus)
        a.parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({nsh_host::ceil_div(2 * cus, blocks), units / 2, 64})));
}

}  // namespace nsh

using nsh_host::check_launch;
using nsh_host::fail;

static bool rows_aligned(const void* p, const int64_t (&s)[3], int64_t bytes) {
    return nsh_host::aligned(p, 16) && s[0] * bytes % 16 == 0 && s[1] * bytes % 16 == 0 &&
           s[2] * bytes % 16 == 0;
}

// Tiles are read with 32-bit offsets from their first row.
static bool rows_near(const int64_t (&s)[3], int64_t bytes) {
    return s[2] >= 0 && s[2] * bytes <= (int64_t(1) << 24);
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
    // the kernels hold both in fp32, with the cap's reciprocal
    if (!std::isfinite(static_cast<float>(g->scale)) ||
        (g->cap != 0.0 && (g->cap < std::ldexp(1.0, -60) || g->cap > std::ldexp(1.0, 60))))
        return fail(NSH_ERR_INVALID, "%s: a scale within fp32 and a cap of 2^-60 to 2^60, or none, are served", op);
    if (g->prefix && !g->causal) return fail(NSH_ERR_INVALID, "%s: a prefix needs causal", op);
    if (g->bias_table &&
        (!g->buckets || g->reach < 0 || g->reach > 2048 || g->num_buckets < 1 || g->num_buckets > 4097))
        return fail(NSH_ERR_INVALID, "%s: a bias table needs buckets, reach <= 2048 and 1..4097 buckets", op);
    if (!g->q || !g->k || !g->v || !g->out) return fail(NSH_ERR_INVALID, "%s: null pointer argument", op);
    const int64_t bytes = g->dtype == NSH_DTYPE_FLOAT32 ? 4 : 2;
    if (!rows_aligned(g->q, g->q_stride, bytes) || !rows_aligned(g->k, g->k_stride, bytes) ||
        !rows_aligned(g->v, g->v_stride, bytes) || !rows_aligned(g->out, g->out_stride, bytes))
        return fail(NSH_ERR_INVALID, "%s: rows must start on 16 bytes", op);
    if (g->out_rest && !nsh_host::aligned(g->out_rest, 16))
        return fail(NSH_ERR_INVALID, "%s: out_rest must start on 16 bytes", op);
    if (!rows_near(g->q_stride, bytes) || !rows_near(g->k_stride, bytes) || !rows_near(g->v_stride, bytes))
        return fail(NSH_ERR_INVALID, "%s: token strides of 0 to 2^24 bytes are served", op);
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
    a->wide = g->dtype == NSH_DTYPE_FLOAT32;
    a->out = g->out, a->degree = g->log_degree, a->stats = g->row_stats, a->rest = g->out_rest;
    return NSH_OK;
}

static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// The cut, and where a call's workspace holds what; returns its bytes.
static int64_t plan(nsh::Att& a, bool backward, char* ws) {
    int64_t at = 0;
    auto take_bytes = [&](int64_t n) {
        char* p = ws + at;
        at += up256(n);
        return p;
    };
    const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Lq;
    nsh::cut_rows(a, backward);
    a.nranges = a.documents ? nsh_host::ceil_div(a.Lk, nsh::kRangeKeys) : 0;
    if (a.documents) a.ranges = reinterpret_cast<const int2*>(take_bytes(static_cast<int64_t>(a.B) * a.nranges * 8));
    if (!backward) {
        if (a.splits > 1) a.part = reinterpret_cast<float*>(take_bytes(rows * a.splits * (2 + a.D) * 4));
        return at;
    }
    nsh::cut_keys(a);
    a.delta = reinterpret_cast<float*>(take_bytes(rows * 4));
    a.far = reinterpret_cast<int*>(take_bytes(static_cast<int64_t>(a.B) * a.Hq * a.rblocks * nsh::kAttWaves * 4));
    if (a.parts > 1)
        a.part = reinterpret_cast<float*>(take_bytes(2 * a.parts * static_cast<int64_t>(a.B) * a.Hk * a.Lk * a.D * 4));
    if (a.gtable)
        a.bins = reinterpret_cast<float*>(
            take_bytes(static_cast<int64_t>(a.B) * a.Hq * a.rblocks * nsh::kAttWaves * (2 * a.reach + 1) * 4));
    return at;
}

extern "C" int64_t nsh_attention_workspace_bytes(const nsh_attention_args* g, int backward) {
    nsh::Att a;
    if (attention_check("attention_workspace_bytes", g, &a)) return -1;
    a.gtable = backward ? g->grad_bias_table : nullptr;
    return plan(a, backward != 0, nullptr);
}

#define NSH_ATT_TYPES(...)                                                   \
    switch (g->dtype) {                                                      \
        case NSH_DTYPE_FLOAT16: { using T = nsh::f16; __VA_ARGS__ } break;   \
        case NSH_DTYPE_BFLOAT16: { using T = nsh::bf16; __VA_ARGS__ } break; \
        default: { using T = float; __VA_ARGS__ } break;                     \
    }

extern "C" int nsh_document_ids(const int64_t* documents, int64_t B, int64_t L, int32_t* out, void* stream) {
    constexpr int64_t kMost = int64_t(1) << 30;
    if (B < 1 || L < 1) return fail(NSH_ERR_INVALID, "document_ids: empty tensor");
    if (B > kMost || L > kMost) return fail(NSH_ERR_INVALID, "document_ids: a size exceeds 2^30");
    if (!documents || !out) return fail(NSH_ERR_INVALID, "document_ids: null pointer argument");
    const int64_t waves = nsh_host::ceil_div(L, 64);
    const int64_t blocks = std::min<int64_t>(nsh_host::ceil_div(B * waves, nsh::kAttWaves), 1 << 20);
    nsh::document_ids_kernel<<<static_cast<unsigned>(blocks), nsh::kAttThreads, 0, static_cast<hipStream_t>(stream)>>>(
        documents, B, L, waves, out);
    return check_launch("document_ids");
}

extern "C" int nsh_attention_forward(const nsh_attention_args* g, void* stream) {
    nsh::Att a;
    if (int rc = attention_check("attention_forward", g, &a)) return rc;
    const int64_t need = plan(a, false, static_cast<char*>(g->workspace));
    if (need && (!g->workspace || !nsh_host::aligned(g->workspace, 16) || g->workspace_bytes < need))
        return fail(NSH_ERR_INVALID, "attention_forward: workspace smaller than nsh_attention_workspace_bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.documents)
        if (int rc = nsh::ranges_launch(a, st)) return rc;
    NSH_ATT_TYPES(return nsh::attention_forward_launch<T>(a, st);)
}

extern "C" int nsh_attention_backward(const nsh_attention_args* g, void* stream) {
    nsh::Att a;
    if (int rc = attention_check("attention_backward", g, &a)) return rc;
    if ((!g->log_degree && !g->row_stats) || !g->grad_out || !g->grad_q || !g->grad_k || !g->grad_v ||
        (g->grad_bias_table && !g->bias_table))
        return fail(NSH_ERR_INVALID, "attention_backward: null pointer argument");
    const int64_t bytes = g->dtype == NSH_DTYPE_FLOAT32 ? 4 : 2;
    if (!rows_aligned(g->grad_out, g->go_stride, bytes) || !rows_aligned(g->grad_q, g->gq_stride, bytes) ||
        !rows_aligned(g->grad_k, g->gk_stride, bytes) || !rows_aligned(g->grad_v, g->gv_stride, bytes))
        return fail(NSH_ERR_INVALID, "attention_backward: rows must start on 16 bytes");
    if (!rows_near(g->go_stride, bytes))
        return fail(NSH_ERR_INVALID, "attention_backward: token strides of 0 to 2^24 bytes are served");
    a.go = g->grad_out, a.gdegree = g->grad_log_degree;
    take(a.gos, g->go_stride), take(a.gqs, g->gq_stride), take(a.gks, g->gk_stride), take(a.gvs, g->gv_stride);
    a.gq = g->grad_q, a.gk = g->grad_k, a.gv = g->grad_v, a.gtable = g->grad_bias_table;
    const int64_t need = plan(a, true, static_cast<char*>(g->workspace));
    if (!g->workspace || !nsh_host::aligned(g->workspace, 16) || g->workspace_bytes < need)
        return fail(NSH_ERR_INVALID, "attention_backward: workspace smaller than nsh_attention_workspace_bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.documents)
        if (int rc = nsh::ranges_launch(a, st)) return rc;
    NSH_ATT_TYPES(return nsh::attention_backward_launch<T>(a, st);)
}
