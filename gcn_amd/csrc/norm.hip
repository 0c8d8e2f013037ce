// Root-mean-square norm of the rows of a layer's activations, with the residual's addition in front of it, its
// output as float32 or as 8-bit rows with a scale each (the operand gcn_spmm_csr_quant_f32 gathers), and its
// gradients.  The reference has no normalisation layer; the operators stand in front of its propagation step
// (gcn/layers.py:198-202).
//
//   h = x + residual            inv = 1 / sqrt(mean_c h_c^2 + eps)            y_c = h_c inv w_c
//   8 bits: scale = max(max_c |y_c| / 448, 2^-120),  q_c = e4m3(y_c / scale)       (448: the largest e4m3 value)
//   g = w dy:  dx_c = dh_c + inv (g_c - h_c inv^2 mean_c(g h)),   dw_c = sum over rows of dy_c h_c inv
//
// Both directions are bound by memory: a row is read once, lives in registers between the reduction and the use of
// its result, and is written once.  A row of f columns belongs to G lanes (G a power of two; a wave holds 64 / G
// rows) or, past 1024 columns, to a whole workgroup; lane l holds the columns 4 (l + G j) .. + 3, so that an
// instruction of a group reads 16 G consecutive bytes.  Sums, the maximum and the weight's gradient are float32.
// Measured, compulsory bytes over time (a large copy: 4.7 TB/s), rows of 1 GB: 8-bit output with residual 4.9 to 5.4 TB/s at
// 16, 64, 256, 500, 1433, 2048, 8192, 9000, 12,000 and 16,384 columns (100: 4.0, whose 112 of 128 bytes a row are partial
// lines), float32 output 4.9 to 5.7, gradients 4.4 to 5.1 up to 8192 columns and 3.4 (9000) to 4.4 (16,384) up to 16,384, where
// the kernel spills 11 registers; past that 3.6 to 5.2 forward, and the gradient, which reads its rows twice there,
// 2.5 to 3.3 (1.4 with everything in registers).
// A wave a row at 1433 columns (eight vectors a lane, two waves a SIMD) ran the gradient at 2.6 instead of 4.7.
#include <algorithm>

#include "common.h"
#include "operands.h"
#include "quant_rows.h"
#include "row_vectors.h"

namespace gcn {

constexpr int kNormMaxF = 32768;
constexpr int kWaveRowF = 1024;          // wider rows belong to a workgroup each
// the larger of two magnitudes, by their bits: a NaN is larger than everything
__device__ __forceinline__ float larger(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}
// sum or largest magnitude over the G lanes of a row (G <= 64: lanes of one wave; more: the workgroup, through `lds`)
template <int G, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* lds) {
    constexpr int W = G < 64 ? G : 64;
#pragma unroll
    for (int d = W / 2; d > 0; d >>= 1) {
        const float o = __shfl_xor(v, d);
        v = MAX ? larger(v, o) : v + o;
    }
    if (G > 64) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < G / 64; ++w) v = MAX ? larger(v, lds[w]) : v + lds[w];
    }
    return v;
}

struct NormArgs {
    int64_t n;
    int f;
    const float* x;
    int64_t ldx;
    const float* residual;   // may be null
    int64_t ldr;
    const float* w;          // may be null: all ones
    float eps;
    float* h;                // x + residual; null without a residual
    int64_t ldh;
    float* inv;              // [n]
    float* y;                // float32 output, or null
    int64_t ldy;
    uint8_t* q;              // 8-bit output, or null
    int64_t ldq;
    float* scales;           // [n], with q
};

template <int G, int VPL, int BLOCK>
__global__ __launch_bounds__(BLOCK) void rms_norm_kernel(NormArgs a, int tile) {
    constexpr int kRows = BLOCK / G;                 // rows a workgroup holds at a time
    __shared__ float lds[4][16];                     // two reductions a row, two rows before a slot is used again
    const int sub = threadIdx.x % G;
    const int f = a.f;
    float w[VPL][4];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int c = 4 * (sub + G * j);
        if (a.w && c < f) {
            load_cols(a.w, c, f, w[j]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[j][e] = 1.0f;
        }
    }
    const float inv_f = 1.0f / (float)f;
    const int left = f - 4 * sub;                    // columns from the lane's first one on
    const int64_t base = (int64_t)blockIdx.x * tile * kRows;
    for (int t = 0; t < tile; ++t) {
        const int64_t i = base + (int64_t)t * kRows + threadIdx.x / G;
        if (base + (int64_t)t * kRows >= a.n) break;                         // uniform in the workgroup
        const bool live = i < a.n;
        float v[VPL][4], sum = 0.0f;
        const int64_t row = live ? i : a.n - 1;
        const bool last = row == a.n - 1;
        load_row<G, VPL>(a.x + row * a.ldx, sub, f, last, v);
        if (a.residual) {
            float r[VPL][4];
            load_row<G, VPL>(a.residual + row * a.ldr, sub, f, last, r);
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] += r[j][e];
            if (live) store_row<G, VPL>(a.h + i * a.ldh, sub, f, v);
        }
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[j][e] = 4 * G * j + e < left ? v[j][e] : 0.0f;
                sum = fmaf(v[j][e], v[j][e], sum);
            }
        sum = row_reduce<G, false>(sum, lds[2 * (t & 1)]);
        const float ms = sum * inv_f;
        const float inv = rsqrtf(ms + a.eps);
        if (live && sub == 0) a.inv[i] = inv;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = v[j][e] * inv * w[j][e];
        if (!a.q) {
            if (live) store_row<G, VPL>(a.y + i * a.ldy, sub, f, v);
            continue;
        }
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = larger(most, fabsf(v[j][e]));      // 0 past the row's end
        most = row_reduce<G, true>(most, lds[2 * (t & 1) + 1]);
        // Quotients, not products with a rounded inverse: those put the scale of six rows in ten one step off and now and
        // then a byte on the wrong side of the middle of two.  Within 1 % of the products' time up to 16,384 columns, where
        // the memory hides them; past that, a workgroup a compute unit, 8 % (8192 x 32,768: 773 -> 836 us).
        float scale = fmaxf(most / kE4m3Max, kQuantScaleMin);
        // a row whose mean square or maximum is not finite has no scale: it stands for NaN as a whole
        if (!(ms < INFINITY) || !(most < INFINITY)) scale = NAN;
        if (live && sub == 0) a.scales[i] = scale;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int c = 4 * (sub + G * j);
            // the bytes from f to the next multiple of 16 are part of the row and zero
            if (live && c < ((f + 15) & ~15))
                *reinterpret_cast<uint32_t*>(a.q + i * a.ldq + c) =
                    e4m3_pack4(v[j][0] / scale, v[j][1] / scale, v[j][2] / scale, v[j][3] / scale, f - c);
        }
    }
}

struct NormGradArgs {
    int64_t n;
    int f;
    const float* dy;
    int64_t lddy;
    const float* h;
    int64_t ldh;
    const float* w;          // may be null: all ones
    const float* inv;        // [n]
    const float* dh;         // gradient that reaches h from elsewhere; may be null
    int64_t lddh;
    float* dx;               // may be null
    int64_t lddx;
    float* part;             // [workgroups x f] partial sums of the weight's gradient, or null
};

template <int G, int VPL, int BLOCK>
__global__ __launch_bounds__(BLOCK) void rms_norm_grad_kernel(NormGradArgs a, int tile) {
    constexpr int kRows = BLOCK / G;
    __shared__ float lds[2][16];
    __shared__ float cols[G < 256 ? (kRows - 1) * G * VPL * 4 + 1 : 1];      // weight gradients of the groups but the first
    const int sub = threadIdx.x % G, group = threadIdx.x / G;
    const int f = a.f;
    float w[VPL][4], dw[VPL][4];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int c = 4 * (sub + G * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[j][e] = 1.0f;
            dw[j][e] = 0.0f;
        }
        if (a.w && c < f) load_cols(a.w, c, f, w[j]);
    }
    const float inv_f = 1.0f / (float)f;
    const int left = f - 4 * sub;                    // columns from the lane's first one on
    const int64_t base = (int64_t)blockIdx.x * tile * kRows;
    for (int t = 0; t < tile; ++t) {
        const int64_t i = base + (int64_t)t * kRows + group;
        if (base + (int64_t)t * kRows >= a.n) break;                         // uniform in the workgroup
        const bool live = i < a.n;
        const int64_t row = live ? i : a.n - 1;
        const bool last = row == a.n - 1;
        const float inv = a.inv[row];
        float dy[VPL][4], h[VPL][4];
        load_row<G, VPL>(a.dy + row * a.lddy, sub, f, last, dy);
        load_row<G, VPL>(a.h + row * a.ldh, sub, f, last, h);
        float along = 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = 4 * G * j + e < left;
                dy[j][e] = in && live ? dy[j][e] : 0.0f;
                h[j][e] = in ? h[j][e] : 0.0f;
                along = fmaf(dy[j][e] * w[j][e], h[j][e], along);
                dw[j][e] = fmaf(dy[j][e], h[j][e] * inv, dw[j][e]);
            }
        along = row_reduce<G, false>(along, lds[t & 1]);
        const float back = along * inv_f * inv * inv;
        if (a.dx) {
            float u[VPL][4];
            if (a.dh) load_row<G, VPL>(a.dh + row * a.lddh, sub, f, last, u);
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float o = inv * (dy[j][e] * w[j][e] - h[j][e] * back);
                    dy[j][e] = a.dh ? o + u[j][e] : o;
                }
            if (live) store_row<G, VPL>(a.dx + i * a.lddx, sub, f, dy);
        }
    }
    if (!a.part) return;
    // the groups of the workgroup in order, then one row of partial sums: no atomics, the same bits every time
    if (G < 256 && kRows > 1) {
        if (group > 0) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) cols[((group - 1) * VPL + j) * G * 4 + e * G + sub] = dw[j][e];
        }
        __syncthreads();
        if (group > 0) return;
        for (int g = 0; g < kRows - 1; ++g)
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) dw[j][e] += cols[(g * VPL + j) * G * 4 + e * G + sub];
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int c = 4 * (sub + G * j);
        if (c < f) store_cols(a.part + (int64_t)blockIdx.x * f, c, f, dw[j]);
    }
}

// Rows past 16,384 columns, a workgroup a row: two of its operands, the weight and its gradient do not fit the 128 registers
// of a lane among 1024 (the kernel above spilled 338 of them).  The weight's gradient stays in LDS, every lane at its own
// columns, and the row is read a second time, from the caches, for dx.  (The two operands alone would be 64 registers a lane:
// a form that keeps them has not been built.)
__global__ __launch_bounds__(1024) void rms_norm_grad_wide_kernel(NormGradArgs a, int tile) {
    constexpr int G = 1024, kDepth = 4;
    __shared__ float lds[2][16];
    __shared__ __attribute__((aligned(16))) float dw[kNormMaxF];
    const int sub = threadIdx.x, f = a.f;
    const float inv_f = 1.0f / (float)f;
    for (int c = 4 * sub; c < f; c += 4 * G) *reinterpret_cast<float4*>(dw + c) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // calls use(column, g, h) for the lane's vectors of a row, kDepth of them in flight; g = dy without the weight
    auto walk = [&](const float* dy, const float* h, auto use) {
        for (int c0 = 4 * sub; c0 < f; c0 += 4 * G * kDepth) {
            float g[kDepth][4], x[kDepth][4], w[kDepth][4];
#pragma unroll
            for (int u = 0; u < kDepth; ++u) {
                const int c = c0 + 4 * G * u < f ? c0 + 4 * G * u : 4 * sub;
                load_cols(dy, c, f, g[u]);
                load_cols(h, c, f, x[u]);
                if (a.w) {
                    load_cols(a.w, c, f, w[u]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[u][e] = 1.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < kDepth; ++u)
                if (c0 + 4 * G * u < f) use(c0 + 4 * G * u, g[u], x[u], w[u]);
        }
    };
    for (int t = 0; t < tile; ++t) {
        const int64_t i = (int64_t)blockIdx.x * tile + t;
        if (i >= a.n) break;                                                  // uniform in the workgroup
        const float *dy = a.dy + i * a.lddy, *h = a.h + i * a.ldh;
        const float inv = a.inv[i];
        float along = 0.0f;
        walk(dy, h, [&](int c, const float (&g)[4], const float (&x)[4], const float (&w)[4]) {
            float4 s = *reinterpret_cast<float4*>(dw + c);
            s.x = fmaf(g[0], x[0] * inv, s.x);
            s.y = fmaf(g[1], x[1] * inv, s.y);
            s.z = fmaf(g[2], x[2] * inv, s.z);
            s.w = fmaf(g[3], x[3] * inv, s.w);
            *reinterpret_cast<float4*>(dw + c) = s;
#pragma unroll
            for (int e = 0; e < 4; ++e) along = fmaf(g[e] * w[e], x[e], along);
        });
        if (!a.dx) continue;
        along = row_reduce<G, false>(along, lds[t & 1]);
        const float back = along * inv_f * inv * inv;
        walk(dy, h, [&](int c, const float (&g)[4], const float (&x)[4], const float (&w)[4]) {
            float u[4] = {0.0f, 0.0f, 0.0f, 0.0f}, o[4];
            if (a.dh) load_cols(a.dh + i * a.lddh, c, f, u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[e] = inv * (g[e] * w[e] - x[e] * back);
                if (a.dh) o[e] += u[e];
            }
            store_cols(a.dx + i * a.lddx, c, f, o);
        });
    }
    if (!a.part) return;
    for (int c = 4 * sub; c < f; c += 4 * G) {
        const float4 s = *reinterpret_cast<const float4*>(dw + c);
        const float v[4] = {s.x, s.y, s.z, s.w};
        store_cols(a.part + (int64_t)blockIdx.x * f, c, f, v);
    }
}

// out[c] = sum over the rows of part [rows x f]: 16 columns a workgroup, 64 strided sums a column, eight of their rows in
// flight, added pairwise in a fixed tree.  (64 columns a workgroup and one row in flight: 38 us for 1974 x 256, 50 us for
// 1924 x 1433; this form: 7 and 9 us.)
__global__ __launch_bounds__(1024) void column_sums_kernel(int64_t rows, int f, const float* __restrict__ part,
                                                           float* __restrict__ out) {
    constexpr int kSlices = 64, kDepth = 8;
    __shared__ float lds[kSlices][16];
    const int col = threadIdx.x & 15, slice = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + col;
    float s = 0.0f;
    if (c < f) {
        int64_t r = slice;
        for (; r + (kDepth - 1) * kSlices < rows; r += kDepth * kSlices) {
            float v[kDepth];
#pragma unroll
            for (int u = 0; u < kDepth; ++u) v[u] = part[(r + u * kSlices) * f + c];
#pragma unroll
            for (int u = 0; u < kDepth; ++u) s += v[u];
        }
        for (; r < rows; r += kSlices) s += part[r * f + c];
    }
    lds[slice][col] = s;
#pragma unroll
    for (int half = kSlices / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (slice < half) lds[slice][col] += lds[slice + half][col];
    }
    if (slice == 0 && c < f) out[c] = lds[0][col];
}

int launch_column_sums(int64_t rows, int64_t f, const float* part, float* out, hipStream_t st) {
    column_sums_kernel<<<(unsigned)ceil_div(f, (int64_t)16), 1024, 0, st>>>(rows, (int)f, part, out);
    GCN_LAUNCH_CHECK();
    return GCN_OK;
}

// rows a workgroup holds at a time for rows of f columns (the G, VPL and BLOCK of the launchers below)
static inline int norm_rows(int64_t f) {
    const int64_t vecs = ceil_div(f, (int64_t)4);
    int g = 4;
    while (g < 64 && g < vecs) g <<= 1;
    return f <= kWaveRowF ? 256 / g : 1;
}

#define GCN_NORM_BY_WIDTH(LAUNCH)              \
    if (f <= 16) { LAUNCH(4, 1, 256); }        \
    else if (f <= 32) { LAUNCH(8, 1, 256); }   \
    else if (f <= 64) { LAUNCH(16, 1, 256); }  \
    else if (f <= 128) { LAUNCH(32, 1, 256); } \
    else if (f <= 256) { LAUNCH(64, 1, 256); } \
    else if (f <= 512) { LAUNCH(64, 2, 256); } \
    else if (f <= 1024) { LAUNCH(64, 4, 256); } \
    else if (f <= 2048) { LAUNCH(256, 2, 256); } \
    else if (f <= 4096) { LAUNCH(256, 4, 256); } \
    else if (f <= 8192) { LAUNCH(256, 8, 256); } \
    else if (f <= 16384) { LAUNCH(1024, 4, 1024); }

// row groups a workgroup walks one after the other: one until there are workgroups for every compute unit's slots
static inline int norm_tile(int64_t n, int64_t f) {
    return (int)std::min<int64_t>(8, std::max<int64_t>(1, ceil_div(n, (int64_t)norm_rows(f)) / 4096));
}

// The gradient's workgroups: at most 2048, so that the partial sums of the weight's gradient stay small (2 MB at 256
// columns) and their addition short.
static inline int64_t norm_grad_tile(int64_t n, int64_t f) {
    return std::max<int64_t>(1, ceil_div(ceil_div(n, (int64_t)norm_rows(f)), (int64_t)2048));
}
static inline int64_t norm_grad_blocks(int64_t n, int64_t f) {
    return ceil_div(n, norm_rows(f) * norm_grad_tile(n, f));
}

static int norm_shape(int64_t n, int64_t f) {
    if (n < 0 || f < 1 || f > kNormMaxF)
        return fail(GCN_ERR_BAD_ARG, "bad shape: n=%lld f=%lld (a row holds 1 to %d columns)", (long long)n, (long long)f,
                    kNormMaxF);
    if (n > ((int64_t)1 << 32)) return fail(GCN_ERR_BAD_ARG, "more than 2^32 rows in one launch");
    return GCN_OK;
}

}  // namespace gcn

using namespace gcn;

extern "C" {

int gcn_quant_pitch(int64_t f, int64_t* pitch_bytes) {
    if (!pitch_bytes || f < 1 || f > kNormMaxF) return fail(GCN_ERR_BAD_ARG, "a row holds 1 to %d columns", kNormMaxF);
    *pitch_bytes = quant_pitch(f);
    return GCN_OK;
}

int gcn_rms_norm_f32(int64_t n, int64_t f, const float* x, int64_t ldx, const float* residual, int64_t ldr,
                     const float* weight, float eps, float* h, int64_t ldh, float* inv, float* y, int64_t ldy,
                     uint8_t* q, int64_t ldq, float* scales, void* stream) {
    if (int rc = norm_shape(n, f)) return rc;
    if (!(eps >= 0.0f)) return fail(GCN_ERR_BAD_ARG, "eps must not be negative");
    if (ldx < f || (residual && (ldr < f || ldh < f)) || (y && ldy < f))
        return fail(GCN_ERR_BAD_ARG, "a leading dimension is shorter than the row");
    if (q && (ldq < (f + 15) / 16 * 16 || ldq % 16 != 0 || ((uintptr_t)q & 15) || !scales))
        return fail(GCN_ERR_BAD_ARG, "8-bit rows want scales, a 16-byte aligned address and a pitch that is a multiple of 16 "
                                     "not below the width: pitch %lld", (long long)ldq);
    if (n == 0) return GCN_OK;
    if ((y != nullptr) == (q != nullptr)) return fail(GCN_ERR_BAD_ARG, "one of the outputs y and q is wanted");
    if (!x || !inv || (residual && !h)) return fail(GCN_ERR_BAD_ARG, "null pointer");
    const Place in_x = place(x, n, f, ldx), in_r = place(residual, n, f, ldr), in_w = place(weight, f);
    const Place out_h = place(residual ? h : nullptr, n, f, ldh), out_y = place(y, n, f, ldy);
    const Place out_q = place(q, n, (f + 15) / 16 * 16, ldq), out_i = place(inv, n), out_s = place(q ? scales : nullptr, n);
    for (const Place& out : {out_h, out_y})
        if (lies_across(out, in_x) || lies_across(out, in_r) || share_memory(out, in_w))
            return fail(GCN_ERR_BAD_ARG, "an output lies across x, the residual or the weight: it may be x or the residual itself");
    for (const Place& out : {out_q, out_i, out_s})
        if (share_memory(out, in_x) || share_memory(out, in_r) || share_memory(out, in_w))
            return fail(GCN_ERR_BAD_ARG, "inv, q or the scales lie over an operand");
    const Place outs[] = {out_h, out_y, out_q, out_i, out_s};
    for (int i = 0; i < 5; ++i)
        for (int j = 0; j < i; ++j)
            if (share_memory(outs[i], outs[j]))
                return fail(GCN_ERR_BAD_ARG, "two outputs share memory: each needs its own");
    NormArgs a = {n, (int)f, x, ldx, residual, ldr, weight, eps, h, ldh, inv, y, ldy, q, ldq, scales};
    const int tile = norm_tile(n, f);
    const int64_t blocks = ceil_div(n, (int64_t)norm_rows(f) * tile);
    if (blocks >= (int64_t)1 << 22) return fail(GCN_ERR_BAD_ARG, "too many rows for one launch");   // threads count in 32 bits
#define GCN_LAUNCH_NORM(G, VPL, BLOCK) \
    rms_norm_kernel<G, VPL, BLOCK><<<(unsigned)blocks, BLOCK, 0, (hipStream_t)stream>>>(a, tile)
    GCN_NORM_BY_WIDTH(GCN_LAUNCH_NORM)
    else { GCN_LAUNCH_NORM(1024, 8, 1024); }
#undef GCN_LAUNCH_NORM
    GCN_LAUNCH_CHECK();
    return GCN_OK;
}

int gcn_rms_norm_grad_workspace_bytes(int64_t n, int64_t f, size_t* bytes) {
    if (!bytes) return fail(GCN_ERR_BAD_ARG, "null pointer");
    if (int rc = norm_shape(n, f)) return rc;
    *bytes = n ? (size_t)norm_grad_blocks(n, f) * (size_t)f * sizeof(float) : 0;
    return GCN_OK;
}

int gcn_rms_norm_grad_f32(int64_t n, int64_t f, const float* dy, int64_t lddy, const float* h, int64_t ldh,
                          const float* weight, const float* inv, const float* dh, int64_t lddh, float* dx, int64_t lddx,
                          float* dweight, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = norm_shape(n, f)) return rc;
    if (lddy < f || ldh < f || (dh && lddh < f) || (dx && lddx < f))
        return fail(GCN_ERR_BAD_ARG, "a leading dimension is shorter than the row");
    hipStream_t st = (hipStream_t)stream;
    if (n == 0) return dweight ? launch_column_sums(0, f, nullptr, dweight, st) : GCN_OK;
    if (!dy || !h || !inv) return fail(GCN_ERR_BAD_ARG, "null pointer");
    if (!dx && !dweight) return GCN_OK;
    const int64_t blocks = norm_grad_blocks(n, f);
    if (dweight) {
        const size_t need = (size_t)blocks * (size_t)f * sizeof(float);
        if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
            return fail(GCN_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed (16-byte aligned)", workspace_bytes, need);
    }
    const Place out = place(dx, n, f, lddx);
    if (lies_across(out, place(dy, n, f, lddy)) || lies_across(out, place(h, n, f, ldh)) || lies_across(out, place(dh, n, f, lddh)) ||
        share_memory(out, place(weight, f)) || share_memory(out, place(inv, n)) || share_memory(out, place(dweight, f)))
        return fail(GCN_ERR_BAD_ARG, "dx lies across an operand or dweight: it may be dy, dh or h itself");
    NormGradArgs a = {n, (int)f, dy, lddy, h, ldh, weight, inv, dh, lddh, dx, lddx, dweight ? (float*)workspace : nullptr};
    const int tile = (int)norm_grad_tile(n, f);
#define GCN_LAUNCH_NORM(G, VPL, BLOCK) \
    rms_norm_grad_kernel<G, VPL, BLOCK><<<(unsigned)blocks, BLOCK, 0, st>>>(a, tile)
    GCN_NORM_BY_WIDTH(GCN_LAUNCH_NORM)
    else rms_norm_grad_wide_kernel<<<(unsigned)blocks, 1024, 0, st>>>(a, tile);
#undef GCN_LAUNCH_NORM
    GCN_LAUNCH_CHECK();
    return dweight ? launch_column_sums(blocks, f, (const float*)workspace, dweight, st) : GCN_OK;
}

}  // extern "C"
