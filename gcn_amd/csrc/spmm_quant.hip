// CSR x 8-bit rows (quant_rows.h): C = act(A . B) with B[r, c] = scales[r] e4m3(q[r, c]), the propagation step
// dot(support, ., sparse=True) of a layer (gcn/layers.py:202) on an operand a quarter as wide.
//
//   C[i, :] = act(sum_e (a_e s[col_e]) q[col_e, :])        float32 sums, one fused multiply-add an element
//
// The ReLU keeps a NaN (the float32 product's makes it 0): a row of B that stands for NaN as a whole stays visible.
//
// The product is bound by the rows it gathers: at 256 columns 256 bytes an entry (two 128-byte lines) and the entry's
// scale, instead of the 1024 bytes of float32 rows.  A wave takes a strip of the rows the plan cut.  L lanes hold 16 columns
// each (one 16-byte load a row), so 64 / L entries are gathered by one instruction; each lane group adds its entries, and at
// the end of a row the groups are added by exchanging halves: after the exchange over lane distance 32 a lane is left with
// 8 of its 16 columns, then 4, 2, 1.  Long rows are cut at the chunks of the wide dense product and joined in chunk order.
// Measured (R-MAT, 32 entries a row; rows gathered + compulsory bytes over time; random row gathers end at 7.5 TB/s):
// 2^20 nodes x 256: 1.29 ms, 7.5 TB/s (float32 rows: 3.92 ms); x 512: 2.54 (8.34); x 128: 0.81 (1.93); x 16: 0.58 (0.56).
// 2^24 nodes x 256: 28.5 ms (74.6), x 128: 18.9 (39.0), x 64: 18.2 (20.1), x 32: 17.5 (11.1), x 16: 16.8 (10.7): there the
// 64 MB of scales no longer stay in the L2s and every entry pays a line for its scale, so rows of 32 columns and fewer are for
// graphs of up to about 2^20 nodes (2^22 x 32: 3.4 ms against 2.5, x 64: 3.8 against 4.5).
// At six waves a SIMD the kernel spills 3 to 13 registers where rows of 33 to 128 or more than 256 columns are gathered.
// Steps tried on 2^20 x 256 / 2^24 x 256: a row after the other, every row's loads drained before the next row's
// 1.62 / 33.8 ms; the stream below with 4 steps in flight 1.38 / 28.8, with 8 (4 waves a SIMD) 1.55 / 30.3, with 2 and 6 waves
// a SIMD 1.29 / 28.5; non-temporal row loads 1.95 / 32.3 (the hubs' rows leave the L2).
#include <algorithm>

#include "common.h"
#include "operands.h"
#include "quant_rows.h"
#include "spmm_plan.h"

namespace gcn {

constexpr int kBlock = 256;

typedef float f32x2 __attribute__((ext_vector_type(2)));

// acc += w * (the 16 values of a 16-byte piece)
__device__ __forceinline__ void add_piece(const uint4& raw, float w, float (&acc)[16]) {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)words[i], false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)words[i], true);
        acc[4 * i] = fmaf(w, lo.x, acc[4 * i]);
        acc[4 * i + 1] = fmaf(w, lo.y, acc[4 * i + 1]);
        acc[4 * i + 2] = fmaf(w, hi.x, acc[4 * i + 2]);
        acc[4 * i + 3] = fmaf(w, hi.y, acc[4 * i + 3]);
    }
}

// Adds the lane groups of L lanes: the lane is left with kLeft(L) sums of its 16 columns, from column `offset` on.
constexpr int left_of(int L) { return L >= 64 ? 16 : L == 32 ? 8 : L == 16 ? 4 : L == 8 ? 2 : 1; }
template <int L>
__device__ __forceinline__ int add_groups(float (&acc)[16], int lane) {
    int offset = 0;
    if (L <= 32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i]), __float_as_uint(acc[i + 8]), false, false);
            acc[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
        }
        offset += (lane & 32) ? 8 : 0;
    }
    if (L <= 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i]), __float_as_uint(acc[i + 4]), false, false);
            acc[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
        }
        offset += (lane & 16) ? 4 : 0;
    }
    if (L <= 8) {
        const bool up = lane & 8;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float give = up ? acc[i] : acc[i + 2], keep = up ? acc[i + 2] : acc[i];
            acc[i] = keep + __shfl_xor(give, 8);
        }
        offset += up ? 2 : 0;
    }
    if (L <= 4) {
        const bool up = lane & 4;
        const float give = up ? acc[0] : acc[1], keep = up ? acc[1] : acc[0];
        acc[0] = keep + __shfl_xor(give, 4);
        offset += up ? 1 : 0;
    }
    if (L <= 2) acc[0] += __shfl_xor(acc[0], 2);
    if (L <= 1) acc[0] += __shfl_xor(acc[0], 1);
    return offset;
}

// A run of `total` consecutive entries from k0 on, holding whole rows one after the other: row number x of the run ends
// before entry row_end(x) of it (non-decreasing, the last one `total`); finish(x) takes the sums of row x out of acc.
// The entries are one stream, whatever rows they belong to: lane l holds (column, weight) of entry 64 b + l of batch b, the
// pairs are fetched two batches and the scales one batch ahead, and step s of a batch gathers entries s P .. s P + P - 1, one
// a lane group, U steps in flight while the U before are added.  A step that a row ends in is added once for every row it
// touches, the pieces and weights of other rows replaced by zeros (not multiplied by zero: they may be NaN).
template <int L, int U, class RowEnd, class Finish>
__device__ __forceinline__ void stream_quant(int64_t k0, int total, const int32_t* __restrict__ indices,
                                             const float* __restrict__ vals, const uint8_t* __restrict__ q, uint32_t ldq,
                                             const float* __restrict__ scales, int lane, int64_t piece, int rows,
                                             RowEnd row_end, Finish finish, float (&acc)[16]) {
    constexpr int P = 64 / L, C = L / U;
    const int group = lane / L;
    int row = 0, begin = 0, end = row_end(0);            // the row in work: entries begin .. end - 1
    if (total > 0) {
        auto entry = [&](int t) { return k0 + (t < total ? t : total - 1); };      // past the end: the last one again
        auto gather = [&](uint4 (&raw)[U], int32_t col, int chunk) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t c = (uint32_t)__shfl(col, (chunk * U + u) * P + group);
                raw[u] = *reinterpret_cast<const uint4*>(q + (uint64_t)c * ldq + piece);
            }
        };
        int32_t col = indices[entry(lane)], col1 = indices[entry(64 + lane)];
        float val1 = vals[entry(64 + lane)];
        float w = vals[entry(lane)] * scales[col];
        uint4 raw[U];
        gather(raw, col, 0);
        for (int t0 = 0; t0 < total; t0 += 64) {
            const float scale1 = scales[col1];
            const int32_t col2 = indices[entry(t0 + 128 + lane)];
            const float val2 = vals[entry(t0 + 128 + lane)];
#pragma unroll 1
            for (int c = 0; c < C; ++c) {
                uint4 next[U];
                const int t1 = t0 + (c + 1) * U * P;                 // first entry of the next chunk
                if (t1 < total) gather(next, c + 1 < C ? col : col1, c + 1 < C ? c + 1 : 0);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int from = t0 + (c * U + u) * P, to = from + P;
                    const float ws = __shfl(w, (c * U + u) * P + group);
                    if (from < total) {
                        if (begin <= from && end > to) {
                            add_piece(raw[u], ws, acc);
                        } else {
                            const int idx = from + group;
                            for (;;) {
                                if (end > begin && end > from) {
                                    const bool in = idx >= begin && idx < end;
                                    const uint4 mine = {in ? raw[u].x : 0u, in ? raw[u].y : 0u, in ? raw[u].z : 0u, in ? raw[u].w : 0u};
                                    add_piece(mine, in ? ws : 0.0f, acc);
                                }
                                if (end > to || row == rows) break;
                                finish(row);
                                begin = end;
                                ++row;
                                if (row < rows) end = row_end(row);
                                if (row == rows || begin >= to) break;
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = next[u];
            }
            col = col1;
            w = val1 * scale1;
            col1 = col2;
            val1 = val2;
        }
    }
    for (; row < rows; ++row) finish(row);               // empty rows at the end
}

template <int L, int U>
__global__ __launch_bounds__(kBlock, 6) void spmm_quant_kernel(PlanView pv, const int64_t* __restrict__ indptr,
                                                            const int32_t* __restrict__ indices,
                                                            const float* __restrict__ vals, int f,
                                                            const uint8_t* __restrict__ q, uint32_t ldq,
                                                            const float* __restrict__ scales, float* __restrict__ c,
                                                            int64_t ldc, int c_vec, float* __restrict__ part, int64_t ldp,
                                                            int relu) {
    constexpr int kLeft = left_of(L);
    const int lane = threadIdx.x & 63, sub = lane % L;
    const int col0 = (int)blockIdx.y * 16 * L + 16 * sub;           // this lane's columns
    const int64_t piece = col0 < f ? col0 : (int64_t)blockIdx.y * 16 * L;
    const int64_t block = blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    auto store = [&](float (&acc)[16], float* row, bool vec, bool act) {
        const int at = col0 + add_groups<L>(acc, lane);
        if (!(L < 4 && (lane & 3 & ~(L - 1)))) {                    // L = 1, 2: the groups past the fourth hold the same sum
#pragma unroll
            for (int i = 0; i < kLeft; ++i)
                if (act) acc[i] = acc[i] <= 0.0f ? 0.0f : acc[i];      // a NaN stays one
#pragma unroll
            for (int i = 0; i < kLeft; i += 4) {
                if (kLeft >= 4 && vec && at + i + 4 <= f) {
                    *reinterpret_cast<float4*>(row + at + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4 && i + e < kLeft; ++e)
                        if (at + i + e < f) row[at + i + e] = acc[i + e];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    };
    float acc[16] = {};
    if (block < pv.chunk_blocks) {
        const int64_t chunk = block * (kBlock / 64) + wave;
        if (chunk >= pv.n_chunks) return;
        const int li = pv.chunk_long[chunk];
        const int r = pv.long_row[li];
        const int64_t k0 = indptr[r] + (chunk - pv.long_chunk[li]) * (int64_t)pv.chunk_len;
        const int64_t row_end = indptr[r + 1];
        const int total = (int)(k0 + pv.chunk_len < row_end ? pv.chunk_len : row_end - k0);
        // partial rows: 16-byte aligned, pitch a multiple of 4
        stream_quant<L, U>(k0, total, indices, vals, q, ldq, scales, lane, piece, 1, [&](int) { return total; },
                           [&](int) { store(acc, part + chunk * ldp, true, false); }, acc);
        return;
    }
    const int64_t strip = (block - pv.chunk_blocks) * (kBlock / 64) + wave;
    if (strip >= pv.n_strips) return;
    // A strip has at most 64 rows: lane l keeps the end of row r_lo + l,
    // counted from the strip's first entry.  Rows that are summed chunk-wise cut the strip's entries into runs.
    static_assert(kStripNnz / kRowCost <= 64, "a strip's rows are held one a lane");
    const int r_lo = pv.strip_row[strip], n_rows = pv.strip_row[strip + 1] - r_lo;
    if (n_rows == 0) return;
    const int64_t base = indptr[r_lo];
    const int mine = lane < n_rows ? lane : n_rows - 1;
    const int64_t len = indptr[r_lo + mine + 1] - indptr[r_lo + mine];
    const int ends = (int)min(indptr[r_lo + mine + 1] - base, (int64_t)0x7fffffff);
    uint64_t cut = __ballot(lane < n_rows && len > pv.split);
    for (int first = 0; first < n_rows;) {
        const int next = cut ? __builtin_ctzll(cut) : n_rows;      // the next row that is summed chunk-wise
        if (next > first) {
            const int at = first ? __builtin_amdgcn_readlane(ends, first - 1) : 0;
            const int total = __builtin_amdgcn_readlane(ends, next - 1) - at;
            stream_quant<L, U>(base + at, total, indices, vals, q, ldq, scales, lane, piece, next - first,
                               [&](int x) { return __builtin_amdgcn_readlane(ends, first + x) - at; },
                               [&](int x) { store(acc, c + (int64_t)(r_lo + first + x) * ldc, c_vec != 0, relu != 0); }, acc);
        }
        first = next + 1;
        cut &= cut - 1;
    }
}

// y <- the float32 values an 8-bit matrix stands for, four columns a thread: 2^20 x 256 494 us, 2.7 TB/s (single stores, a
// division for the row)
__global__ __launch_bounds__(kBlock) void quant_dense_kernel(int64_t n_rows, int f, const uint8_t* __restrict__ q, int64_t ldq,
                                                             const float* __restrict__ scales, float* __restrict__ y,
                                                             int64_t ldy) {
    const int64_t per_row = (f + 3) / 4, total = n_rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < total; i += (int64_t)gridDim.x * kBlock) {
        const int64_t r = i / per_row;
        const int c = 4 * (int)(i - r * per_row);
        const int word = *reinterpret_cast<const int*>(q + r * ldq + c);
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
        const float s = scales[r], v[4] = {s * lo.x, s * lo.y, s * hi.x, s * hi.y};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < f) y[r * ldy + c + e] = v[e];
    }
}

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace gcn

using namespace gcn;

extern "C" {

int gcn_quant_dense_f32(int64_t n_rows, int64_t f, const uint8_t* q, int64_t ldq, const float* scales, float* y, int64_t ldy,
                        void* stream) {
    if (n_rows < 0 || f < 1 || f > 32768) return fail(GCN_ERR_BAD_ARG, "an 8-bit row holds 1 to 32768 columns: f=%lld", (long long)f);
    if (ldy < f || ldq < (f + 15) / 16 * 16 || ldq % 16 != 0) return fail(GCN_ERR_BAD_ARG, "bad pitch");
    if (n_rows == 0) return GCN_OK;
    if (!q || !scales || !y) return fail(GCN_ERR_BAD_ARG, "null pointer");
    if (!aligned16(q)) return fail(GCN_ERR_BAD_ARG, "8-bit rows must be 16-byte aligned");
    if (share_memory(place(y, n_rows, f, ldy), place(q, n_rows, (f + 15) / 16 * 16, ldq)) ||
        share_memory(place(y, n_rows, f, ldy), place(scales, n_rows)))
        return fail(GCN_ERR_BAD_ARG, "y lies over the 8-bit rows or their scales");
    const int64_t blocks = std::min<int64_t>(ceil_div(n_rows * ((f + 3) / 4), (int64_t)kBlock), 1 << 16);
    quant_dense_kernel<<<(unsigned)blocks, kBlock, 0, (hipStream_t)stream>>>(n_rows, (int)f, q, ldq, scales, y, ldy);
    GCN_LAUNCH_CHECK();
    return GCN_OK;
}

int gcn_spmm_csr_quant_f32(const gcn_spmm_plan* plan, const int64_t* indptr, const int32_t* indices, const float* vals,
                           int64_t f, const uint8_t* q, int64_t ldq, const float* scales, float* c, int64_t ldc, int flags,
                           void* workspace, size_t workspace_bytes, void* stream) {
    if (!plan) return fail(GCN_ERR_BAD_ARG, "plan is null");
    if (f < 1 || f > 32768) return fail(GCN_ERR_BAD_ARG, "an 8-bit row holds 1 to 32768 columns: f=%lld", (long long)f);
    if (ldc < f || ldq < (f + 15) / 16 * 16 || ldq % 16 != 0 || ldq > INT32_MAX)
        return fail(GCN_ERR_BAD_ARG, "bad pitch: ldc=%lld, 8-bit pitch %lld", (long long)ldc, (long long)ldq);
    if (!indptr || (plan->nnz > 0 && (!indices || !vals))) return fail(GCN_ERR_BAD_ARG, "null CSR pointer");
    if (flags & ~GCN_RELU) return fail(GCN_ERR_BAD_ARG, "unknown flag bits 0x%x", flags);
    if (plan->n_rows == 0) return GCN_OK;
    if (!c || (plan->nnz > 0 && (!q || !scales))) return fail(GCN_ERR_BAD_ARG, "null dense pointer");
    if (!aligned16(q)) return fail(GCN_ERR_BAD_ARG, "8-bit rows must be 16-byte aligned");
    const gcn_spmm_plan::LongTable& lt = plan->table[1];            // the cut points of the wide dense product
    constexpr int kWaves = kBlock / 64;
    PlanView pv;
    pv.n_strips = plan->n_strips;
    pv.nnz = plan->nnz;
    pv.n_chunks = lt.n_chunks;
    pv.chunk_blocks = ceil_div(lt.n_chunks, kWaves);
    pv.split = plan->split[1];
    pv.chunk_len = plan->chunk_len ? plan->chunk_len : pv.split;
    pv.hot_cols = 0;
    pv.lds_hub_rows = 0;
    pv.strip_row = plan->strip_row;
    pv.chunk_long = lt.chunk_long;
    pv.long_row = lt.long_row;
    pv.long_chunk = lt.long_chunk;
    float* part = nullptr;
    const int64_t ldp = (f + 3) / 4 * 4;
    if (lt.n_chunks > 0) {
        const size_t need = (size_t)lt.n_chunks * (size_t)ldp * sizeof(float);
        if (!workspace || workspace_bytes < need)
            return fail(GCN_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
        if (!aligned16(workspace)) return fail(GCN_ERR_BAD_ARG, "workspace must be 16-byte aligned");
        part = (float*)workspace;
    }
    const int64_t grid = pv.chunk_blocks + ceil_div(plan->n_strips, kWaves);
    if (grid >= (int64_t)1 << 24) return fail(GCN_ERR_BAD_ARG, "matrix too large for one launch");   // threads count in 32 bits
    const Place out = place(c, plan->n_rows, f, ldc);
    if (share_memory(out, place(q, plan->n_cols, (f + 15) / 16 * 16, ldq)) || share_memory(out, place(scales, plan->n_cols)))
        return fail(GCN_ERR_BAD_ARG, "the result lies over the 8-bit rows or their scales");
    hipStream_t st = (hipStream_t)stream;
    const int relu = (flags & GCN_RELU) ? 1 : 0;
    const int c_vec = (ldc % 4 == 0 && aligned16(c)) ? 1 : 0;
    if (plan->timing) GCN_HIP_TRY(hipEventRecord(plan->ev[0], st));
#define GCN_QUANT_GO(L, U)                                                                                                \
    spmm_quant_kernel<L, U><<<dim3((unsigned)grid, (unsigned)ceil_div(f, (int64_t)16 * L)), kBlock, 0, st>>>(               \
        pv, indptr, indices, vals, (int)f, q, (uint32_t)ldq, scales, c, ldc, c_vec, part, ldp, relu)
    if (f <= 16) GCN_QUANT_GO(1, 1);
    else if (f <= 32) GCN_QUANT_GO(2, 1);
    else if (f <= 64) GCN_QUANT_GO(4, 2);
    else if (f <= 128) GCN_QUANT_GO(8, 2);
    else if (f <= 256) GCN_QUANT_GO(16, 2);
    else if (f <= 512) GCN_QUANT_GO(32, 2);
    else GCN_QUANT_GO(64, 2);                                           // wider rows: ranges of 1024 columns
#undef GCN_QUANT_GO
    GCN_LAUNCH_CHECK();
    if (plan->timing) GCN_HIP_TRY(hipEventRecord(plan->ev[1], st));
    if (lt.n_chunks > 0)
        if (int rc = launch_long_reduce(lt, f, part, ldp, c, ldc, relu ? kReluKeepNan : 0, c_vec && f % 4 == 0, st)) return rc;
    if (plan->timing) GCN_HIP_TRY(hipEventRecord(plan->ev[2], st));
    return GCN_OK;
}

}  // extern "C"
