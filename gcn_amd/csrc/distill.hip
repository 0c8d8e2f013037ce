// Distillation from a teacher's top logits, masked as the reference's loss is (gcn/metrics.py:85-92), and its gradient.
//
//   p = softmax over the listed logits t_j / T of a row (an index outside [0, c) is no entry),  q = softmax(s / T)
//   row loss = w T^2 sum_j p_j (log p_j - log q_idx_j),   w = mask / mean(mask)
//   d(mean over the n rows) / ds_c = (q_c - P_c) T w / n,   P_c = the p_j listed at class c, added up
//   agreement = w where argmax s (ties: the lowest class) is the class of the largest listed logit (ties: the first listed)
//
// Bound by memory: the logits are read once and their gradient is written once, the exponentials of a row staying in
// registers between the two; rows outside the mask are not read at all.  Rows of up to 256 classes belong to G lanes with
// four or eight classes each, so that a wave holds 64 / G rows and the reductions a row needs are shared by them; wider
// ones to a wave or a workgroup, up to 32,768 classes; beyond that the row is read a second time for its gradient.
// Measured, compulsory bytes over time (a large copy: 4.7 TB/s): 4 M x 47 classes, 5 listed: 390 us, 4.5 TB/s;
// 4 M x 7, 3 listed: 90 us, 4.0; 1 M x 200, 20 listed: 354 to 389 us, 4.7 (546 where nearly every list names a class twice); 8,192 x 32,768, 32 listed: 416 us, 5.2;
// read twice, 2,048 x 65,536: 292 us, 3.7 (held in registers, which then spill, 426 us); 8,192 x 32,768 read twice: 497 us.
#include <algorithm>
#include <hip/hip_fp16.h>

#include "common.h"
#include "lanes.h"
#include "operands.h"
#include "row_vectors.h"

namespace gcn {

constexpr int kDistillMaxK = 256;
constexpr int kWaveRowC = 1024;          // wider rows belong to a workgroup each

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
    float inv_mask_mean, t, to_log2;      // t: the temperature; to_log2: log2(e) / t
    float* stats;             // [n x 2] or null
    float* grad;              // [n x c] or null
    int64_t ldg;
    const float* upstream;    // device scalar the gradient is multiplied by, or null
};

// One entry of the teacher's list: its logit, -inf and no class where it is no entry.
struct Entry {
    float t;
    int at;
};
// The same as loaded: the 32-bit word that holds the logit (of a 16-bit logit the whole aligned word, inside the
// allocation whatever its address), where in it, and the class.  Nothing here depends on a loaded value and nothing branches
// on the type, so that a list can be fetched ahead of its use.
struct RawEntry {
    uint32_t word;
    int shift, at;
};
__device__ __forceinline__ RawEntry fetch_entry(const DistillArgs& a, int64_t row, int j) {
    RawEntry r = {0u, 0, -1};
    if (j < a.k) {
        const uintptr_t where = (uintptr_t)a.values + ((uint64_t)(row * a.ldv + j) << (a.type == GCN_F32 ? 2 : 1));
        r.word = *reinterpret_cast<const uint32_t*>(where & ~(uintptr_t)3);
        r.shift = (int)(where & 2) * 8;
        r.at = a.indices[row * a.ldi + j];
    }
    return r;
}
__device__ __forceinline__ Entry entry_of(const DistillArgs& a, const RawEntry& r) {
    const uint32_t half = (r.word >> r.shift) & 0xffffu;
    const float f16 = __half2float(__builtin_bit_cast(__half, (uint16_t)half));
    const float t = a.type == GCN_F32 ? __uint_as_float(r.word) : a.type == GCN_F16 ? f16 : __uint_as_float(half << 16);
    const bool in = r.at >= 0 && r.at < a.c;
    return {in ? t : -INFINITY, in ? r.at : -1};
}
__device__ __forceinline__ Entry teacher_entry(const DistillArgs& a, int64_t row, int j) {
    return entry_of(a, fetch_entry(a, row, j));
}

// LDS accesses of one wave stay in program order; this keeps the compiler to it.
__device__ __forceinline__ void lds_in_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Exponents and logarithms are base 2 (one instruction each): a logit's exponent is (s - max) log2(e) / T.
// The loss row from its parts: tsum = sum 2^d_j, tdot = sum 2^d_j d_j (d_j: the exponents of the list), qdot = sum p_j log2 q_j.
__device__ __forceinline__ float row_loss(const DistillArgs& a, float tsum, float tdot, float qdot, float w) {
    const float kLn2 = 0.6931471805599453f;
    return (tdot * __builtin_amdgcn_rcpf(tsum) - __builtin_amdgcn_logf(tsum) - qdot) * (kLn2 * a.t * a.t * w);
}

// ------------------------------------------------------------------------------------------------
// c <= 4 G VPL: G lanes a row, 64 / G rows a wave
// ------------------------------------------------------------------------------------------------
// The rows of a group are a pipeline: the mask is fetched two rows ahead and the logits and the list one row ahead of the
// row in work, nothing of the fetch depending on a loaded value.  A row outside the
// mask is a row without entries whose logits are not loaded: it takes the same way and ends as zeros.
// P, the teacher's probabilities by class, is made in LDS: every entry writes its number at its class and reads it back;
// if all find their own, no class is listed twice and they write their exponentials there.  Otherwise the wave adds the
// entries one by one in list order.
// A lane holds NE entries of the list in registers (G NE of them a row); MORE: longer lists, whose other entries are read
// again by every pass over the list (17 entries on 47 classes: 1.13 ms against 0.48 in registers).
template <int G, int VPL, int NE, bool MORE>
__global__ __launch_bounds__(256) void distill_group_kernel(DistillArgs a, int tile) {
    constexpr int kRows = 256 / G;
    __shared__ __attribute__((aligned(16))) float by_class[kRows][4 * G * VPL];
    const int sub = threadIdx.x % G, group = threadIdx.x / G;
    float* const mine = by_class[group];
    const float up = (a.upstream ? *a.upstream : 1.0f) * a.t * a.per_row;
    const int64_t base = (int64_t)blockIdx.x * tile * kRows + group;
    const int rows = (int)(base >= a.n ? 0 : std::min<int64_t>(tile, (a.n - base + kRows - 1) / kRows));   // of this group
    const int left = a.c - 4 * sub;                  // columns from the lane's first one on
    auto load_mask = [&](int t) { return t < rows ? (a.mask ? a.mask[base + (int64_t)t * kRows] : 1) : 0; };
    auto fetch_row = [&](int t, int m, float (&x)[VPL][4], RawEntry (&e)[NE]) {
#pragma unroll
        for (int u = 0; u < NE; ++u) e[u] = {0u, 0, -1};
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int q = 0; q < 4; ++q) x[v][q] = 0.0f;
        if (m != 0) {
            const int64_t i = base + (int64_t)t * kRows;
            load_row<G, VPL>(a.logits + i * a.ldx, sub, a.c, i == a.n - 1, x);
#pragma unroll
            for (int u = 0; u < NE; ++u) e[u] = fetch_entry(a, i, G * u + sub);
        }
    };
    float nx[VPL][4];
    RawEntry ne[NE];
    int nm = load_mask(0);
    fetch_row(0, nm, nx, ne);
    int nnm = load_mask(1);
    for (int t = 0; t < tile; ++t) {
        if ((int64_t)blockIdx.x * tile * kRows + (int64_t)t * kRows >= a.n) break;      // uniform in the workgroup
        const int64_t i = base + (int64_t)t * kRows;
        const bool live = t < rows;
        const int m = nm;
        Entry e0[NE];
#pragma unroll
        for (int u = 0; u < NE; ++u) e0[u] = entry_of(a, ne[u]);
        // calls f(entry, its number) for the lane's entries, in list order
        auto entries = [&](auto f) {
#pragma unroll
            for (int u = 0; u < NE; ++u) f(e0[u], G * u + sub);
            if (MORE)
                for (int j = G * NE; j < a.k; j += G) f(m != 0 ? teacher_entry(a, i, j + sub) : Entry{-INFINITY, -1}, j + sub);
        };
        float x[VPL][4], xm = -INFINITY;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                x[v][q] = 4 * G * v + q < left ? nx[v][q] : -INFINITY;
                xm = fmaxf(xm, x[v][q]);
            }
        nm = nnm;
        fetch_row(t + 1, nm, nx, ne);
        nnm = load_mask(t + 2);
        const float w = (float)m * a.inv_mask_mean;
        xm = lanes_reduce<G, OpMax>(xm);
        float tmax = -INFINITY;
        entries([&](const Entry& e, int) { tmax = fmaxf(tmax, e.t); });
        tmax = lanes_reduce<G, OpMax>(tmax);
        const float tref = tmax > -INFINITY ? tmax : 0.0f;
        // the list: its sums, its first maximum, P
#pragma unroll
        for (int v = 0; v < VPL; ++v)
            *reinterpret_cast<float4*>(mine + 4 * (sub + G * v)) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        lds_in_order();
        entries([&](const Entry& e, int number) {
            if (e.at >= 0) mine[e.at] = __int_as_float(number + 1);
        });
        lds_in_order();
        float tsum = 0.0f, tdot = 0.0f;
        int top = 0x7fffffff, top_at = -1;
        bool twice = false;
        entries([&](const Entry& e, int number) {
            const int found = __float_as_int(mine[max(e.at, 0)]);
            twice = twice || (e.at >= 0 && found != number + 1);
            const float d = (e.t - tref) * a.to_log2, ex = e.at >= 0 ? __builtin_amdgcn_exp2f(d) : 0.0f;
            tsum += ex;
            tdot = fmaf(ex, ex > 0.0f ? d : 0.0f, tdot);
            const bool here = e.at >= 0 && e.t == tmax && top_at < 0;
            top = here ? number : top;
            top_at = here ? e.at : top_at;
        });
        lds_in_order();
        float p[VPL][4];
        if (__any(twice)) {
#pragma unroll
            for (int v = 0; v < VPL; ++v)
#pragma unroll
                for (int q = 0; q < 4; ++q) p[v][q] = 0.0f;
            entries([&](const Entry& e, int number) {
                const float ex = e.at >= 0 ? __builtin_amdgcn_exp2f((e.t - tref) * a.to_log2) : 0.0f;
                const int here = min(G, a.k - (number - sub));           // the entries the row's lanes hold now
                for (int b = 0; b < here; ++b) {
                    const float exb = __shfl(ex, b, G);
                    const int at = __shfl(e.at, b, G) - 4 * sub;
#pragma unroll
                    for (int v = 0; v < VPL; ++v)
#pragma unroll
                        for (int q = 0; q < 4; ++q) p[v][q] += at == 4 * G * v + q ? exb : 0.0f;
                }
            });
        } else {
            entries([&](const Entry& e, int) {
                if (e.at >= 0) mine[e.at] = __builtin_amdgcn_exp2f((e.t - tref) * a.to_log2);
            });
            lds_in_order();
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const float4 f = *reinterpret_cast<const float4*>(mine + 4 * (sub + G * v));
                p[v][0] = f.x;
                p[v][1] = f.y;
                p[v][2] = f.z;
                p[v][3] = f.w;
            }
        }
        lds_in_order();
        tsum = lanes_reduce<G, OpAdd>(tsum);
        const bool any = tmax > -INFINITY || !(tsum == 0.0f);       // a NaN logit of the teacher is an entry
        const float pscale = any ? __builtin_amdgcn_rcpf(tsum) : 0.0f;
        // the student; columns past the end are -inf and add nothing
        int first = 0x7fffffff;
        float s = 0.0f, dot = 0.0f;
#pragma unroll
        for (int v = VPL - 1; v >= 0; --v)
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                first = x[v][q] == xm ? 4 * (sub + G * v) + q : first;
                const float z = (x[v][q] - xm) * a.to_log2;
                x[v][q] = __builtin_amdgcn_exp2f(z);
                s += x[v][q];
                p[v][q] *= pscale;
                dot = fmaf(p[v][q], p[v][q] == 0.0f ? 0.0f : z, dot);
            }
        s = lanes_reduce<G, OpAdd>(s);
        if (a.stats) {
            tdot = lanes_reduce<G, OpAdd>(tdot);
            dot = lanes_reduce<G, OpAdd>(dot);
            first = __float_as_int(lanes_reduce<G, OpMinInt>(__int_as_float(first)));
            const int best = __float_as_int(lanes_reduce<G, OpMinInt>(__int_as_float(top)));
            // sum p log q = sum p z - log2(s): the p add up to 1
            const float hit = lanes_reduce<G, OpMax>(top_at >= 0 && top == best && top_at == first ? w : 0.0f);
            const float loss = row_loss(a, tsum, tdot, dot - __builtin_amdgcn_logf(s), w);
            if (live && sub == 0)
                *reinterpret_cast<float2*>(a.stats + 2 * i) = make_float2(any ? loss : 0.0f, any ? hit : 0.0f);
        }
        if (a.grad) {
            const float scale = w * up, qs = __builtin_amdgcn_rcpf(s);
#pragma unroll
            for (int v = 0; v < VPL; ++v)
#pragma unroll
                for (int q = 0; q < 4; ++q) x[v][q] = any ? (x[v][q] * qs - p[v][q]) * scale : 0.0f;
            if (live) store_row<G, VPL>(a.grad + i * a.ldg, sub, a.c, x);
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
        const float d = (e[b].t - tref) * a.to_log2, ex = e[b].at >= 0 ? __builtin_amdgcn_exp2f(d) : 0.0f;
        l.tsum += ex;
        if (ex > 0.0f) l.tdot = fmaf(ex, d, l.tdot);
        if (e[b].at >= 0 && e[b].t == tmax) l.top = min(l.top, 64 * b + lane);
        if (64 * b + lane < a.k) list[64 * b + lane] = make_float2(ex, __int_as_float(e[b].at));
    }
    l.tsum = lanes_reduce<64, OpAdd>(l.tsum);
    l.tdot = lanes_reduce<64, OpAdd>(l.tdot);
    l.top = __float_as_int(lanes_reduce<64, OpMinInt>(__int_as_float(l.top)));
    l.any = tmax > -INFINITY || !(l.tsum == 0.0f);
    lds_in_order();                                              // the list is read by other lanes of this wave
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
            qdot = fmaf(v.x * pscale, (a.logits[i * a.ldx + __float_as_int(v.y)] - xm) * a.to_log2 - logs, qdot);
    }
    return lanes_reduce<64, OpAdd>(qdot);
}

__device__ __forceinline__ void listed_grad(const DistillArgs& a, int64_t i, int lane, const float2* list, float xm, float qs,
                                            float pscale, float scale) {
    for (int j = lane; j < a.k; j += 64) {
        const int at = __float_as_int(list[j].y);
        float sum;
        if (sum_of_class(list, a.k, j, at, &sum)) {
            const float q = __builtin_amdgcn_exp2f((a.logits[i * a.ldx + at] - xm) * a.to_log2) * qs;
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
    load_row<G, VPL>(xr, sub, a.c, i == a.n - 1, x);
    Listed l;
    if (lister) {
        l = list_entries(a, i, lane, list);
        if (G > 64 && lane == 0) shared_list[slot] = l;
    }
    // columns past the end are -inf and add nothing
    const int left = a.c - 4 * sub;
    float xm = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            x[j][q] = 4 * G * j + q < left ? x[j][q] : -INFINITY;
            xm = fmaxf(xm, x[j][q]);
        }
    xm = wide_reduce<G, OpMax>(xm, lds[0]);
    if (G > 64) l = shared_list[slot];
    int first = 0x7fffffff;
    float s = 0.0f;
#pragma unroll
    for (int j = VPL - 1; j >= 0; --j)
#pragma unroll
        for (int q = 3; q >= 0; --q) {
            first = x[j][q] == xm ? 4 * (sub + G * j) + q : first;
            x[j][q] = __builtin_amdgcn_exp2f((x[j][q] - xm) * a.to_log2);
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
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) x[j][q] = l.any ? x[j][q] * all : 0.0f;
        store_row<G, VPL>(gr, sub, a.c, x);
    }
    if (a.stats) {
        first = __float_as_int(wide_reduce<G, OpMinInt>(__int_as_float(first), lds[2]));
        if (lister) {
            const float qdot = listed_log_q(a, i, lane, list, xm, __builtin_amdgcn_logf(s), pscale);
            if (lane == 0)
                *reinterpret_cast<float2*>(a.stats + 2 * i) =
                    make_float2(l.any ? row_loss(a, l.tsum, l.tdot, qdot, w) : 0.0f,
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

// Calls use(column, values) for the lane's vectors of a row of any length, kDepth of them in flight.
template <int G, class F>
__device__ __forceinline__ void walk_row(const float* __restrict__ row, int sub, int c, F use) {
    constexpr int kDepth = 4;
    for (int64_t c0 = 4 * sub; c0 < c; c0 += 4 * G * kDepth) {
        float v[kDepth][4];
#pragma unroll
        for (int u = 0; u < kDepth; ++u) load_cols(row, c0 + 4 * G * u < c ? (int)c0 + 4 * G * u : 4 * sub, c, v[u]);
#pragma unroll
        for (int u = 0; u < kDepth; ++u)
            if (c0 + 4 * G * u < c) use((int)c0 + 4 * G * u, v[u]);
    }
}

// any number of classes: the row is read twice, the second time, from the caches, for its gradient
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
            for (int64_t c = 4 * tid; c < a.c; c += 4 * G) {
                const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                store_cols(gr, (int)c, a.c, zero);
            }
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
    walk_row<G>(xr, tid, a.c, [&](int c, const float (&v)[4]) {
        float most = -INFINITY;
        int at = 0;
#pragma unroll
        for (int e = 3; e >= 0; --e)
            if (c + e < a.c && v[e] >= most) {
                most = v[e];
                at = c + e;
            }
        if (most > run) {
            s *= __builtin_amdgcn_exp2f((run - most) * a.to_log2);
            run = most;
            first = at;
        }
        const float ref = run > -INFINITY ? run : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) s += c + e < a.c ? __builtin_amdgcn_exp2f((v[e] - ref) * a.to_log2) : 0.0f;
    });
    const float xm = wide_reduce<G, OpMax>(run, lds[0]);
    const Listed l = shared_list;
    if (run != xm) first = 0x7fffffff;
    s = run == -INFINITY && s == 0.0f ? (xm == -INFINITY ? NAN : 0.0f) : s * __builtin_amdgcn_exp2f((run - xm) * a.to_log2);
    s = wide_reduce<G, OpAdd>(s, lds[1]);
    const float pscale = l.any ? 1.0f / l.tsum : 0.0f;
    // a NaN among the listed logits makes the whole row NaN, as it does where P covers every class
    const float scale = l.tsum == l.tsum ? w * (a.upstream ? *a.upstream : 1.0f) * a.t * a.per_row : NAN;
    const float qs = 1.0f / s;
    if (gr)
        walk_row<G>(xr, tid, a.c, [&](int c, const float (&v)[4]) {
            float g[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = l.any ? __builtin_amdgcn_exp2f((v[e] - xm) * a.to_log2) * (qs * scale) : 0.0f;
            store_cols(gr, c, a.c, g);
        });
    if (a.stats) {
        first = __float_as_int(wide_reduce<G, OpMinInt>(__int_as_float(first), lds[2]));
        if (tid < 64) {
            const float qdot = listed_log_q(a, i, lane, list, xm, __builtin_amdgcn_logf(s), pscale);
            if (lane == 0)
                *reinterpret_cast<float2*>(a.stats + 2 * i) =
                    make_float2(l.any ? row_loss(a, l.tsum, l.tdot, qdot, w) : 0.0f,
                                l.any && first == l.top ? w : 0.0f);
        }
    }
    if (!gr || !l.any) return;
    __syncthreads();
    if (tid < 64) listed_grad(a, i, lane, list, xm, qs, pscale, scale);
}

template <int G, int VPL>
static void launch_group(const DistillArgs& a, hipStream_t st) {
    constexpr int kRows = 256 / G;
    // one group of rows a workgroup until there are 16 workgroups for every compute unit
    const int tile = (int)std::min<int64_t>(8, std::max<int64_t>(1, ceil_div(a.n, (int64_t)kRows) / 4096));
    const unsigned blocks = (unsigned)ceil_div(a.n, (int64_t)kRows * tile);
    if (a.k <= G)
        distill_group_kernel<G, VPL, 1, false><<<blocks, 256, 0, st>>>(a, tile);
    else if (a.k <= 2 * G)
        distill_group_kernel<G, VPL, 2, false><<<blocks, 256, 0, st>>>(a, tile);
    else if (a.k <= 4 * G)
        distill_group_kernel<G, VPL, 4, false><<<blocks, 256, 0, st>>>(a, tile);
    else
        distill_group_kernel<G, VPL, 4, true><<<blocks, 256, 0, st>>>(a, tile);
}

template <int G, int VPL, int BLOCK>
static void launch_row(const DistillArgs& a, hipStream_t st) {
    distill_row_kernel<G, VPL, BLOCK><<<(unsigned)ceil_div(a.n, (int64_t)(BLOCK / G)), BLOCK, 0, st>>>(a);
}

// Lanes and vectors a row.  Two vectors a lane from 17 classes on: half the reductions a row (25 classes: 232 us against 261
// with one; 47 classes: 390 against 478, and 412 with four); below, the longer pipelines of entries cost more than that.
static void launch_distill(const DistillArgs& a, hipStream_t st) {
    if (a.c <= 4) launch_group<1, 1>(a, st);
    else if (a.c <= 8) launch_group<2, 1>(a, st);
    else if (a.c <= 16) launch_group<4, 1>(a, st);
    else if (a.c <= 32) launch_group<4, 2>(a, st);
    else if (a.c <= 64) launch_group<8, 2>(a, st);
    else if (a.c <= 128) launch_group<16, 2>(a, st);
    else if (a.c <= 256) launch_group<32, 2>(a, st);
    else if (a.c <= 512) launch_row<64, 2, 256>(a, st);
    else if (a.c <= kWaveRowC) launch_row<64, 4, 256>(a, st);
    else if (a.c <= 4096) launch_row<256, 4, 256>(a, st);
    else if (a.c <= 8192) launch_row<256, 8, 256>(a, st);
    else if (a.c <= 16384) launch_row<1024, 4, 1024>(a, st);
    else if (a.c <= 32768) launch_row<1024, 8, 1024>(a, st);
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
    if (!(temperature > 0.0f) || !(temperature < INFINITY) || !(1.4426950408889634f / temperature < INFINITY))
        return fail(GCN_ERR_BAD_ARG, "the temperature must be positive, and its inverse a float32 number");
    if (n == 0) return GCN_OK;
    if (!logits || !values || !indices) return fail(GCN_ERR_BAD_ARG, "null pointer");
    if (row_stats && ((uintptr_t)row_stats & 7)) return fail(GCN_ERR_BAD_ARG, "row_stats must be 8-byte aligned");
    if (!row_stats && !dlogits) return GCN_OK;
    const int64_t value_size = value_type == GCN_F32 ? 4 : 2;
    const Place out_d = place(dlogits, n, c, ldd), out_s = place(row_stats, n, 2, 2);
    const Place in[] = {place(logits, n, c, ldx), place((const char*)values, n, k * value_size, ldv * value_size),
                        place(indices, n, k, ldi), place(mask, n), place(upstream, 1)};
    for (const Place& operand : in)
        if (share_memory(out_d, operand) || share_memory(out_s, operand))
            return fail(GCN_ERR_BAD_ARG, "an output lies over an operand: it needs memory of its own, the operands are read after its first stores");
    if (share_memory(out_d, out_s)) return fail(GCN_ERR_BAD_ARG, "two outputs share memory: each needs its own");
    // a launch counts its threads in 32 bits: rows of at most 64 threads, or of up to 1024
    const int64_t slice = (c <= kWaveRowC ? (int64_t)1 << 26 : (int64_t)1 << 22) - 4;
    for (int64_t r = 0; r < n; r += slice) {
        const DistillArgs a = {std::min(slice, n - r), 1.0f / (float)n, (int)c, logits + r * ldx, ldx,
                               (const char*)values + r * ldv * value_size, value_type, ldv, indices + r * ldi, ldi, (int)k,
                               mask ? mask + r : nullptr, 1.0f / mask_mean, temperature, 1.4426950408889634f / temperature,
                               row_stats ? row_stats + 2 * r : nullptr, dlogits ? dlogits + r * ldd : nullptr, ldd, upstream};
        launch_distill(a, (hipStream_t)stream);
        GCN_LAUNCH_CHECK();
    }
    return GCN_OK;
}

}  // extern "C"
