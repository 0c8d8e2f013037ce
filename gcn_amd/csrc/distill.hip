// Distillation from a teacher's top logits, masked as the reference's loss is (gcn/metrics.py:85-92), and its gradient.
//
//   p = softmax over the listed logits t_j / T of a row (an index outside [0, c) is no entry),  q = softmax(s / T)
//   row loss = w T^2 sum_j p_j (log p_j - log q_idx_j),   w = mask / mean(mask)
//   d(mean over the n rows) / ds_c = (q_c - P_c) T w / n,   P_c = the p_j listed at class c, added up
//   agreement = w where argmax s (ties: the lowest class) is the class of the largest listed logit (ties: the first listed)
//
// Bound by memory: the logits are read once and their gradient is written once, the exponentials of a row staying in
// registers between the two; rows outside the mask are not read at all.  Rows of up to 256 classes belong to G lanes
// with four consecutive classes each, so that a wave holds 64 / G rows and the eight reductions a row needs are shared
// by them; wider ones to a wave or a workgroup, up to 65,536 classes; beyond that the row is read a second time for
// its gradient.
#include <algorithm>
#include <hip/hip_fp16.h>

#include "common.h"
#include "lanes.h"
#include "row_vectors.h"

namespace gcn {

constexpr int kDistillMaxK = 256;

struct DistillArgs {
    int64_t n;                // rows of this launch
    float per_row;            // 1 / rows of the whole call
    int c;
    const float* logits;
    int64_t ldx;
    const void* values;       // teacher's logits, `type` says in which form
    int type;
    int64_t ldv;
    const int32_t* indices;
    int64_t ldi;
    int k;
    const int32_t* mask;      // may be null: all ones
    float inv_mask_mean, inv_t, t;
    float* stats;             // [n x 2] or null
    float* grad;              // [n x c] or null
    int64_t ldg;
    const float* upstream;    // device scalar the gradient is multiplied by, or null
};

__device__ __forceinline__ float teacher_value(const DistillArgs& a, int64_t row, int j) {
    const int64_t at = row * a.ldv + j;
    if (a.type == GCN_F32) return static_cast<const float*>(a.values)[at];
    if (a.type == GCN_F16) return __half2float(static_cast<const __half*>(a.values)[at]);
    return __uint_as_float((uint32_t) static_cast<const uint16_t*>(a.values)[at] << 16);
}

// One entry of the teacher's list: its logit over the temperature, -inf where it is no entry.
struct Entry {
    float t;
    int at;
};
__device__ __forceinline__ Entry teacher_entry(const DistillArgs& a, int64_t row, int j) {
    Entry e = {-INFINITY, -1};
    if (j < a.k) {
        const int at = a.indices[row * a.ldi + j];
        if (at >= 0 && at < a.c) {
            e.t = teacher_value(a, row, j) * a.inv_t;
            e.at = at;
        }
    }
    return e;
}

// the loss row from its parts: tsum = sum e_j, tdot = sum e_j (t_j - tmax), qdot = sum p_j log q_j.  Without an entry: 0.
__device__ __forceinline__ float row_loss(float tsum, float tdot, float qdot, float t2w) {
    return (tdot / tsum - logf(tsum) - qdot) * t2w;
}

// ------------------------------------------------------------------------------------------------
// c <= 4 G: G lanes a row
// ------------------------------------------------------------------------------------------------
template <int G>
__global__ __launch_bounds__(256) void distill_group_kernel(DistillArgs a, int tile) {
    constexpr int kRows = 256 / G;
    const int sub = threadIdx.x % G, c0 = 4 * sub;
    const float up = (a.upstream ? *a.upstream : 1.0f) * a.t * a.per_row;
    const int64_t base = (int64_t)blockIdx.x * tile * kRows;
    for (int t = 0; t < tile; ++t) {
        const int64_t i = base + (int64_t)t * kRows + threadIdx.x / G;
        if (base + (int64_t)t * kRows >= a.n) break;
        const bool live = i < a.n;
        const int m = live ? (a.mask ? a.mask[i] : 1) : 0;
        const float w = (float)m * a.inv_mask_mean;
        if (live && m == 0) {
            const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (a.grad && c0 < a.c) store_cols(a.grad + i * a.ldg, c0, a.c, zero);
            if (a.stats && sub == 0) *reinterpret_cast<float2*>(a.stats + 2 * i) = make_float2(0.0f, 0.0f);
        }
        if (m == 0) continue;                            // the lanes of a row agree; reductions stay inside the row
        float x[4], p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        load_cols(a.logits + i * a.ldx, c0 < a.c ? c0 : 0, a.c, x);
        // the teacher's entries, G at a time; lists of at most G entries are read once
        Entry e = teacher_entry(a, i, sub);
        float tmax = e.t;
        for (int j = G; j < a.k; j += G) tmax = fmaxf(tmax, teacher_entry(a, i, j + sub).t);
        tmax = lanes_reduce<G, OpMax>(tmax);
        const float tref = tmax > -INFINITY ? tmax : 0.0f;
        float xm = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (c0 + q < a.c) xm = fmaxf(xm, x[q]);
        xm = lanes_reduce<G, OpMax>(xm);
        int first = 0x7fffffff;
#pragma unroll
        for (int q = 3; q >= 0; --q)
            if (c0 + q < a.c && x[q] == xm) first = c0 + q;
        float s = 0.0f, z[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            z[q] = (x[q] - xm) * a.inv_t;
            x[q] = c0 + q < a.c ? expf(z[q]) : 0.0f;
            s += x[q];
        }
        s = lanes_reduce<G, OpAdd>(s);
        float tsum = 0.0f, tdot = 0.0f;
        int top = 0x7fffffff;
        for (int j = 0; j < a.k; j += G) {
            if (j > 0) e = teacher_entry(a, i, j + sub);
            const float d = e.t - tref, ex = e.at >= 0 ? expf(d) : 0.0f;
            tsum += ex;
            if (ex > 0.0f) tdot = fmaf(ex, d, tdot);
            if (e.at >= 0 && e.t == tmax) top = min(top, j + sub);
            const int here = min(G, a.k - j);
            for (int b = 0; b < here; ++b) {
                const float exb = __shfl(ex, b, G);
                const int at = __shfl(e.at, b, G) - c0;
#pragma unroll
                for (int q = 0; q < 4; ++q) p[q] += at == q ? exb : 0.0f;
            }
        }
        tsum = lanes_reduce<G, OpAdd>(tsum);
        const bool any = tmax > -INFINITY || !(tsum == 0.0f);       // a NaN logit of the teacher is an entry
        const float pscale = any ? 1.0f / tsum : 0.0f;
        const float logs = logf(s);
        float qdot = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            p[q] *= pscale;
            if (!(p[q] == 0.0f)) qdot = fmaf(p[q], z[q] - logs, qdot);
        }
        if (a.stats) {
            tdot = lanes_reduce<G, OpAdd>(tdot);
            qdot = lanes_reduce<G, OpAdd>(qdot);
            first = __float_as_int(lanes_reduce<G, OpMinInt>(__int_as_float(first)));
            top = __float_as_int(lanes_reduce<G, OpMinInt>(__int_as_float(top)));
            if (sub == 0) {
                const int best = top < a.k ? a.indices[i * a.ldi + top] : -1;
                *reinterpret_cast<float2*>(a.stats + 2 * i) =
                    make_float2(any ? row_loss(tsum, tdot, qdot, w * a.t * a.t) : 0.0f, any && first == best ? w : 0.0f);
            }
        }
        if (a.grad && c0 < a.c) {
            const float scale = w * up, qs = 1.0f / s;
            float g[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) g[q] = any ? (x[q] * qs - p[q]) * scale : 0.0f;
            store_cols(a.grad + i * a.ldg, c0, a.c, g);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// wider rows: a wave (G = 64, four rows a workgroup) or a workgroup (G = BLOCK) a row
// ------------------------------------------------------------------------------------------------
template <int G, class Op>
__device__ __forceinline__ float wide_reduce(float v, float* lds) {
    v = lanes_reduce<64, Op>(v);
    if (G > 64) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < G / 64; ++w) v = Op::f(v, lds[w]);
    }
    return v;
}

// The list of a row, one wave: entries (e_j = exp(t_j - tmax), class) in LDS and the sums over them.
struct Listed {
    float tsum, tdot;
    int top;         // class of the largest listed logit, -1 without one
    bool any;
};
__device__ __forceinline__ Listed list_entries(const DistillArgs& a, int64_t i, int lane, float2* list) {
    float tmax = -INFINITY;
    Entry e[kDistillMaxK / 64];
#pragma unroll
    for (int b = 0; b < kDistillMaxK / 64; ++b) {
        e[b] = 64 * b < a.k ? teacher_entry(a, i, 64 * b + lane) : Entry{-INFINITY, -1};
        tmax = fmaxf(tmax, e[b].t);
    }
    tmax = lanes_reduce<64, OpMax>(tmax);
    const float tref = tmax > -INFINITY ? tmax : 0.0f;
    Listed l = {0.0f, 0.0f, 0x7fffffff, false};
#pragma unroll
    for (int b = 0; b < kDistillMaxK / 64; ++b) {
        const float d = e[b].t - tref, ex = e[b].at >= 0 ? expf(d) : 0.0f;
        l.tsum += ex;
        if (ex > 0.0f) l.tdot = fmaf(ex, d, l.tdot);
        if (e[b].at >= 0 && e[b].t == tmax) l.top = min(l.top, 64 * b + lane);
        if (64 * b + lane < a.k) list[64 * b + lane] = make_float2(ex, __int_as_float(e[b].at));
    }
    l.tsum = lanes_reduce<64, OpAdd>(l.tsum);
    l.tdot = lanes_reduce<64, OpAdd>(l.tdot);
    l.top = __float_as_int(lanes_reduce<64, OpMinInt>(__int_as_float(l.top)));
    l.any = tmax > -INFINITY || !(l.tsum == 0.0f);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the list is read by other lanes of this wave
    __builtin_amdgcn_wave_barrier();
    l.top = l.top < a.k ? __float_as_int(list[l.top].y) : -1;
    return l;
}

// Entry j of the list (one lane each): the e added up over all entries of its class in list order -- every entry of a
// class forms the same sum, and the first one is the one that uses it -- so a class listed twice needs no atomics.
__device__ __forceinline__ bool sum_of_class(const float2* list, int k, int j, int at, float* sum) {
    float s = 0.0f;
    bool first = at >= 0;
    for (int o = 0; o < k; ++o) {
        const float2 v = list[o];
        if (__float_as_int(v.y) == at) {
            s += v.x;
            if (o < j) first = false;
        }
    }
    *sum = s;
    return first;
}

// sum_j p_j log q_j of the list, by one wave (the logits of the listed classes come from memory, which the row's loads
// have just brought near)
__device__ __forceinline__ float listed_log_q(const DistillArgs& a, int64_t i, int lane, const float2* list, float xm,
                                              float logs, float pscale) {
    float qdot = 0.0f;
    for (int j = lane; j < a.k; j += 64) {
        const float2 v = list[j];
        if (__float_as_int(v.y) >= 0 && !(v.x == 0.0f))
            qdot = fmaf(v.x * pscale, (a.logits[i * a.ldx + __float_as_int(v.y)] - xm) * a.inv_t - logs, qdot);
    }
    return lanes_reduce<64, OpAdd>(qdot);
}

__device__ __forceinline__ void listed_grad(const DistillArgs& a, int64_t i, int lane, const float2* list, float xm, float qs,
                                            float pscale, float scale) {
    for (int j = lane; j < a.k; j += 64) {
        const int at = __float_as_int(list[j].y);
        float sum;
        if (sum_of_class(list, a.k, j, at, &sum)) {
            const float q = expf((a.logits[i * a.ldx + at] - xm) * a.inv_t) * qs;
            a.grad[i * a.ldg + at] = (q - sum * pscale) * scale;
        }
    }
}

template <int G, int VPL, int BLOCK>
__global__ __launch_bounds__(BLOCK) void distill_row_kernel(DistillArgs a) {
    constexpr int kRows = BLOCK / G;
    __shared__ float lds[3][16];
    __shared__ float2 lists[kRows][kDistillMaxK];
    __shared__ Listed shared_list[kRows];
    const int sub = threadIdx.x % G, slot = threadIdx.x / G, lane = threadIdx.x & 63;
    const bool lister = sub < 64;                        // the wave that reads the teacher's list
    const int64_t i = (int64_t)blockIdx.x * kRows + slot;
    if (i >= a.n) return;                                // G == BLOCK: uniform; G == 64: no barriers below
    const int m = a.mask ? a.mask[i] : 1;
    const float w = (float)m * a.inv_mask_mean;
    const float* xr = a.logits + i * a.ldx;
    float* gr = a.grad ? a.grad + i * a.ldg : nullptr;
    float2* list = lists[slot];
    if (m == 0) {
        if (gr)
            for (int c = 4 * sub; c < a.c; c += 4 * G) {
                const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                store_cols(gr, c, a.c, zero);
            }
        if (a.stats && sub == 0) *reinterpret_cast<float2*>(a.stats + 2 * i) = make_float2(0.0f, 0.0f);
        return;
    }
    float x[VPL][4];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int c = 4 * (sub + G * j);
        load_cols(xr, c < a.c ? c : 0, a.c, x[j]);
    }
    Listed l;
    if (lister) {
        l = list_entries(a, i, lane, list);
        if (G > 64 && lane == 0) shared_list[slot] = l;
    }
    float xm = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (4 * (sub + G * j) + q < a.c) xm = fmaxf(xm, x[j][q]);
    xm = wide_reduce<G, OpMax>(xm, lds[0]);
    if (G > 64) l = shared_list[slot];
    int first = 0x7fffffff;
    float s = 0.0f;
#pragma unroll
    for (int j = VPL - 1; j >= 0; --j)
#pragma unroll
        for (int q = 3; q >= 0; --q) {
            const int c = 4 * (sub + G * j) + q;
            if (c < a.c && x[j][q] == xm) first = c;
            x[j][q] = c < a.c ? expf((x[j][q] - xm) * a.inv_t) : 0.0f;
            s += x[j][q];
        }
    s = wide_reduce<G, OpAdd>(s, lds[1]);
    const float pscale = l.any ? 1.0f / l.tsum : 0.0f;
    // a NaN among the listed logits makes the whole row NaN, as it does where P covers every class
    const float scale = l.tsum == l.tsum ? w * (a.upstream ? *a.upstream : 1.0f) * a.t * a.per_row : NAN;
    const float qs = 1.0f / s;
    if (gr) {
        const float all = l.any ? qs * scale : 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int c = 4 * (sub + G * j);
            float g[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) g[q] = l.any ? x[j][q] * all : 0.0f;
            if (c < a.c) store_cols(gr, c, a.c, g);
        }
    }
    if (a.stats) {
        first = __float_as_int(wide_reduce<G, OpMinInt>(__int_as_float(first), lds[2]));
        if (lister) {
            const float qdot = listed_log_q(a, i, lane, list, xm, logf(s), pscale);
            if (lane == 0)
                *reinterpret_cast<float2*>(a.stats + 2 * i) =
                    make_float2(l.any ? row_loss(l.tsum, l.tdot, qdot, w * a.t * a.t) : 0.0f,
                                l.any && first == l.top ? w : 0.0f);
        }
    }
    if (!gr || !l.any) return;
    // the listed classes, over what the row's lanes have just written there: those stores come first
    if (G > 64)
        __syncthreads();
    else
        __threadfence_block();
    if (lister) listed_grad(a, i, lane, list, xm, qs, pscale, scale);
}

// any number of classes: the row is read twice, the second time for its gradient
__global__ __launch_bounds__(1024) void distill_long_kernel(DistillArgs a) {
    constexpr int G = 1024;
    __shared__ float lds[3][16];
    __shared__ float2 list[kDistillMaxK];
    __shared__ Listed shared_list;
    const int64_t i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63;
    const int m = a.mask ? a.mask[i] : 1;
    const float w = (float)m * a.inv_mask_mean;
    const float* xr = a.logits + i * a.ldx;
    float* gr = a.grad ? a.grad + i * a.ldg : nullptr;
    if (m == 0) {
        if (gr)
            for (int64_t c = tid; c < a.c; c += G) gr[c] = 0.0f;
        if (a.stats && tid == 0) *reinterpret_cast<float2*>(a.stats + 2 * i) = make_float2(0.0f, 0.0f);
        return;
    }
    if (tid < 64) {
        const Listed l = list_entries(a, i, lane, list);
        if (lane == 0) shared_list = l;
    }
    // running maximum and the sum relative to it, per lane; NaN ends up in the sum
    float run = -INFINITY, s = 0.0f;
    int first = 0x7fffffff;
    for (int64_t c = tid; c < a.c; c += G) {
        const float v = xr[c];
        if (v > run) {
            s *= expf((run - v) * a.inv_t);
            run = v;
            first = (int)c;
        }
        s += v == -INFINITY ? 0.0f : expf((v - run) * a.inv_t);
    }
    const float xm = wide_reduce<G, OpMax>(run, lds[0]);
    const Listed l = shared_list;
    if (run != xm) first = 0x7fffffff;
    s = run == -INFINITY && s == 0.0f ? (xm == -INFINITY ? NAN : 0.0f) : s * expf((run - xm) * a.inv_t);
    s = wide_reduce<G, OpAdd>(s, lds[1]);
    const float pscale = l.any ? 1.0f / l.tsum : 0.0f;
    // a NaN among the listed logits makes the whole row NaN, as it does where P covers every class
    const float scale = l.tsum == l.tsum ? w * (a.upstream ? *a.upstream : 1.0f) * a.t * a.per_row : NAN;
    const float qs = 1.0f / s;
    if (gr)
        for (int64_t c = tid; c < a.c; c += G) gr[c] = l.any ? expf((xr[c] - xm) * a.inv_t) * (qs * scale) : 0.0f;
    if (a.stats) {
        first = __float_as_int(wide_reduce<G, OpMinInt>(__int_as_float(first), lds[2]));
        if (tid < 64) {
            const float qdot = listed_log_q(a, i, lane, list, xm, logf(s), pscale);
            if (lane == 0)
                *reinterpret_cast<float2*>(a.stats + 2 * i) =
                    make_float2(l.any ? row_loss(l.tsum, l.tdot, qdot, w * a.t * a.t) : 0.0f,
                                l.any && first == l.top ? w : 0.0f);
        }
    }
    if (!gr || !l.any) return;
    __syncthreads();
    if (tid < 64) listed_grad(a, i, lane, list, xm, qs, pscale, scale);
}

template <int G>
static void launch_group(const DistillArgs& a, hipStream_t st) {
    constexpr int kRows = 256 / G;
    // one group of rows a workgroup until there are 16 workgroups for every compute unit
    const int tile = (int)std::min<int64_t>(8, std::max<int64_t>(1, ceil_div(a.n, (int64_t)kRows) / 4096));
    distill_group_kernel<G><<<(unsigned)ceil_div(a.n, (int64_t)kRows * tile), 256, 0, st>>>(a, tile);
}

template <int G, int VPL, int BLOCK>
static void launch_row(const DistillArgs& a, hipStream_t st) {
    distill_row_kernel<G, VPL, BLOCK><<<(unsigned)ceil_div(a.n, (int64_t)(BLOCK / G)), BLOCK, 0, st>>>(a);
}

static void launch_distill(const DistillArgs& a, hipStream_t st) {
    if (a.c <= 4) launch_group<1>(a, st);
    else if (a.c <= 8) launch_group<2>(a, st);
    else if (a.c <= 16) launch_group<4>(a, st);
    else if (a.c <= 32) launch_group<8>(a, st);
    else if (a.c <= 64) launch_group<16>(a, st);
    else if (a.c <= 128) launch_group<32>(a, st);
    else if (a.c <= 256) launch_group<64>(a, st);
    else if (a.c <= 512) launch_row<64, 2, 256>(a, st);
    else if (a.c <= 1024) launch_row<64, 4, 256>(a, st);
    else if (a.c <= 4096) launch_row<256, 4, 256>(a, st);
    else if (a.c <= 8192) launch_row<256, 8, 256>(a, st);
    else if (a.c <= 16384) launch_row<1024, 4, 1024>(a, st);
    else if (a.c <= 32768) launch_row<1024, 8, 1024>(a, st);
    else if (a.c <= 65536) launch_row<1024, 16, 1024>(a, st);
    else distill_long_kernel<<<(unsigned)a.n, 1024, 0, st>>>(a);
}

}  // namespace gcn

using namespace gcn;

extern "C" {

int gcn_distill_topk_f32(int64_t n, int64_t c, const float* logits, int64_t ldx, const void* values, int value_type,
                         int64_t ldv, const int32_t* indices, int64_t ldi, int64_t k, const int32_t* mask, float mask_mean,
                         float temperature, const float* upstream, float* row_stats, float* dlogits, int64_t ldd,
                         void* stream) {
    if (n < 0 || c < 1 || c > INT32_MAX - 4096 || ldx < c || (dlogits && ldd < c))
        return fail(GCN_ERR_BAD_ARG, "bad shape: n=%lld c=%lld", (long long)n, (long long)c);
    if (k < 1 || k > kDistillMaxK || ldv < k || ldi < k)
        return fail(GCN_ERR_BAD_ARG, "the teacher lists 1 to %d classes a row: k=%lld", kDistillMaxK, (long long)k);
    if (value_type != GCN_F32 && value_type != GCN_F16 && value_type != GCN_BF16)
        return fail(GCN_ERR_BAD_ARG, "unknown type %d of the teacher's logits", value_type);
    if (!(mask_mean > 0.0f)) return fail(GCN_ERR_BAD_ARG, "mask_mean must be positive (an empty mask has no loss)");
    if (!(temperature > 0.0f) || !(temperature < INFINITY)) return fail(GCN_ERR_BAD_ARG, "the temperature must be positive");
    if (n == 0) return GCN_OK;
    if (!logits || !values || !indices) return fail(GCN_ERR_BAD_ARG, "null pointer");
    if (row_stats && ((uintptr_t)row_stats & 7)) return fail(GCN_ERR_BAD_ARG, "row_stats must be 8-byte aligned");
    if (!row_stats && !dlogits) return GCN_OK;
    // a launch counts its threads in 32 bits: 2^22 - 1 rows of up to 1024 threads at a time
    constexpr int64_t kSlice = ((int64_t)1 << 22) - 1;
    const int64_t value_size = value_type == GCN_F32 ? 4 : 2;
    for (int64_t r = 0; r < n; r += kSlice) {
        const DistillArgs a = {std::min(kSlice, n - r), 1.0f / (float)n, (int)c, logits + r * ldx, ldx,
                               (const char*)values + r * ldv * value_size, value_type, ldv, indices + r * ldi, ldi, (int)k,
                               mask ? mask + r : nullptr, 1.0f / mask_mean, 1.0f / temperature, temperature,
                               row_stats ? row_stats + 2 * r : nullptr, dlogits ? dlogits + r * ldd : nullptr, ldd, upstream};
        launch_distill(a, (hipStream_t)stream);
        GCN_LAUNCH_CHECK();
    }
    return GCN_OK;
}

}  // extern "C"
