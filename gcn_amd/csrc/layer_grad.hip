// What the backward pass of a dense layer adds to its two products (gcn_gemm_f32 with trans_b and gcn_gemm_tn_f32): the
// gradient of the pre-activation and of the bias in one pass,
//   dz = dout act'(pre),   dbias_c = sum over rows of dz,
// and the join of a product whose k was cut, sum over the cuts in order + bias, activation, residual.
// Both are bound by memory; a workgroup walks consecutive rows, its column sums stay in registers and end as one row of
// partial sums, which are added in a fixed order.
#include <algorithm>

#include "activations.h"
#include "common.h"
#include "operands.h"
#include "row_vectors.h"

namespace gcn {

constexpr int kTileCols = 256;           // columns of a workgroup; wider matrices take more of them (grid y)

// dz may be dout or pre itself (no __restrict__ on the three): a lane reads its columns of a row before it stores them, and
// what a shifted load of a row's last columns takes besides them is replaced.
template <int G>
__global__ __launch_bounds__(256) void act_grad_kernel(int64_t m, int n, int act, const float* dout, int64_t ldo,
                                                       const float* pre, int64_t ldp, float* dz, int64_t ldz,
                                                       float* __restrict__ part, int64_t tile) {
    constexpr int kRows = 256 / G;
    __shared__ float cols[kRows > 1 ? (kRows - 1) * G * 4 : 1];
    const int sub = threadIdx.x % G, group = threadIdx.x / G;
    const int c = (int)blockIdx.y * kTileCols + 4 * sub;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t base = (int64_t)blockIdx.x * tile * kRows;
    if (c < n)
        with_act(act, [&](auto which) {
            constexpr int ACT = decltype(which)::value;
            for (int64_t t = 0; t < tile; ++t) {
                const int64_t i = base + t * kRows + group;
                if (i >= m) break;
                float g[4], z[4];
                load_cols(dout + i * ldo, c, n, g);
                if (ACT != GCN_ACT_NONE) {
                    load_cols(pre + i * ldp, c, n, z);
#pragma unroll
                    for (int e = 0; e < 4; ++e) g[e] *= act_slope<ACT>(z[e]);
                }
                if (dz) store_cols(dz + i * ldz, c, n, g);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += c + e < n ? g[e] : 0.0f;
            }
        });
    if (!part) return;
    if (kRows > 1) {
        if (group > 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) cols[(group - 1) * G * 4 + e * G + sub] = sum[e];
        }
        __syncthreads();
        if (group > 0) return;
        for (int g = 0; g < kRows - 1; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += cols[g * G * 4 + e * G + sub];
    }
    if (c < n) store_cols(part + (int64_t)blockIdx.x * n, c, n, sum);
}

static inline int act_grad_lanes(int64_t n) {
    int g = 1;
    while (g < 64 && 4 * g < n) g <<= 1;
    return g;
}
// rows of a lane group: one until the columns' workgroups number 2048
static inline int64_t act_grad_tile(int64_t m, int64_t n) {
    const int64_t groups = ceil_div(m, (int64_t)(256 / act_grad_lanes(n)));
    return std::max<int64_t>(1, ceil_div(groups, std::max<int64_t>(1, 2048 / ceil_div(n, (int64_t)kTileCols))));
}
static inline int64_t act_grad_blocks(int64_t m, int64_t n) {
    return ceil_div(m, 256 / act_grad_lanes(n) * act_grad_tile(m, n));
}

// C = act(sum over the cuts of part [splits][m x n], in order, + bias) + residual
__global__ __launch_bounds__(256) void join_splits_kernel(int64_t m, int n, int splits, const float* __restrict__ part,
                                                          const float* __restrict__ bias, int act,
                                                          const float* residual, int64_t ldr, float* __restrict__ pre,
                                                          int64_t ldp, float* c, int64_t ldc) {
    const int64_t total = m * n;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / n;
        const int col = (int)(i - r * n);
        float z = part[i];
        for (int s = 1; s < splits; ++s) z += part[(int64_t)s * total + i];
        if (bias) z += bias[col];
        if (pre) pre[r * ldp + col] = z;
        with_act(act, [&](auto which) { z = act_value<decltype(which)::value>(z); });
        if (residual) z += residual[r * ldr + col];
        c[r * ldc + col] = z;
    }
}

int launch_join_splits(int64_t m, int64_t n, int64_t splits, const float* part, const EpiArgs& ep, float* c, int64_t ldc,
                       hipStream_t st) {
    const int64_t blocks = std::min<int64_t>(ceil_div(m * n, (int64_t)256), 1 << 16);
    join_splits_kernel<<<(unsigned)blocks, 256, 0, st>>>(m, (int)n, (int)splits, part, ep.bias, ep.act, ep.residual, ep.ldr,
                                                         ep.pre, ep.ldp, c, ldc);
    GCN_LAUNCH_CHECK();
    return GCN_OK;
}

}  // namespace gcn

using namespace gcn;

extern "C" {

int gcn_act_grad_workspace_bytes(int64_t m, int64_t n, size_t* bytes) {
    if (!bytes || m < 0 || n < 0 || n > INT32_MAX - 1024) return fail(GCN_ERR_BAD_ARG, "bad argument");
    *bytes = m && n ? (size_t)act_grad_blocks(m, n) * (size_t)n * sizeof(float) : 0;
    return GCN_OK;
}

int gcn_act_grad_f32(int64_t m, int64_t n, int act, const float* dout, int64_t ldo, const float* pre, int64_t ldp, float* dz,
                     int64_t ldz, float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    if (m < 0 || n < 0 || n > INT32_MAX - 1024) return fail(GCN_ERR_BAD_ARG, "bad shape: m=%lld n=%lld", (long long)m, (long long)n);
    if (act < GCN_ACT_NONE || act > GCN_ACT_SILU) return fail(GCN_ERR_BAD_ARG, "unknown activation %d", act);
    if (ldo < n || (act != GCN_ACT_NONE && ldp < n) || (dz && ldz < n))
        return fail(GCN_ERR_BAD_ARG, "leading dimension too small");
    if (n == 0) return GCN_OK;
    hipStream_t st = (hipStream_t)stream;
    if (m == 0) return dbias ? launch_column_sums(0, n, nullptr, dbias, st) : GCN_OK;
    if (!dout || (act != GCN_ACT_NONE && !pre)) return fail(GCN_ERR_BAD_ARG, "null pointer");
    if (!dz && !dbias) return GCN_OK;
    const int64_t blocks = act_grad_blocks(m, n);
    if (dbias) {
        const size_t need = (size_t)blocks * (size_t)n * sizeof(float);
        if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
            return fail(GCN_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed (16-byte aligned)", workspace_bytes, need);
    }
    const Place out = place(dz, m, n, ldz);
    if (lies_across(out, place(dout, m, n, ldo)) || (act != GCN_ACT_NONE && lies_across(out, place(pre, m, n, ldp))) ||
        share_memory(out, place(dbias, n)))
        return fail(GCN_ERR_BAD_ARG, "dz lies across dout, pre or dbias: it may be dout or pre itself");
    const dim3 grid((unsigned)blocks, (unsigned)ceil_div(n, (int64_t)kTileCols));
    if (grid.y > 65535) return fail(GCN_ERR_BAD_ARG, "too many columns for one launch");
#define GCN_ACT_GO(G)                                                                                                       \
    act_grad_kernel<G><<<grid, 256, 0, st>>>(m, (int)n, act, dout, ldo, pre, ldp, dz, ldz, dbias ? (float*)workspace : nullptr, \
                                             act_grad_tile(m, n))
    switch (act_grad_lanes(n)) {
        case 1: GCN_ACT_GO(1); break;
        case 2: GCN_ACT_GO(2); break;
        case 4: GCN_ACT_GO(4); break;
        case 8: GCN_ACT_GO(8); break;
        case 16: GCN_ACT_GO(16); break;
        case 32: GCN_ACT_GO(32); break;
        default: GCN_ACT_GO(64);
    }
#undef GCN_ACT_GO
    GCN_LAUNCH_CHECK();
    return dbias ? launch_column_sums(blocks, n, (const float*)workspace, dbias, st) : GCN_OK;
}

}  // extern "C"
