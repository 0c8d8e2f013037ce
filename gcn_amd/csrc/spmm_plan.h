// The product plan and what the product kernels see of it.
#pragma once

#include "common.h"

struct gcn_spmm_plan {
    int64_t n_rows, n_cols, nnz;
    int64_t n_strips;
    int strip_nnz;       // entries per strip
    int chunk_len;       // entries per chunk of a long row; 0: the split threshold itself
    int split[2];        // rows longer than this are summed chunk-wise (narrow / wide dense operands)
    int device;
    int32_t* strip_row;  // [n_strips + 1] first row starting in each strip
    // rows longer than the split threshold, cut in chunks of that many entries; table 0 serves narrow
    // dense operands (threshold kSplitNarrow), table 1 wide ones (kSplitWide)
    struct LongTable {
        int64_t n_long, n_chunks;
        int32_t* long_row;    // [n_long] ascending
        int64_t* long_chunk;  // [n_long + 1] first chunk of each long row
        int32_t* chunk_long;  // [n_chunks] long-row slot of each chunk
    } table[2];
    // columns >= hot_cols are loaded with the non-temporal hint by the wave-per-row instances (0: off).
    // After a degree-descending relabel the first columns are the hub rows of B: the rows worth caching.
    int64_t hot_cols;
    // narrow products stage the first lds_hub_rows rows of B in LDS, once per workgroup, and entries whose
    // column is below that number read them from there (0: off).  For a degree-ordered matrix those are the
    // hub rows: the "LDS-staged row-block" form of the product.
    int64_t lds_hub_rows;
    int timing;           // record events around the kernels of every product
    hipEvent_t ev[3];     // start, after the row kernel, after the long-row reduction
};

namespace gcn {

constexpr int kStripNnz = 256;       // entries per strip on a matrix large enough to fill the chip with such strips
constexpr int kRowCost = 4;          // a row's fixed cost (pointer loads, store) in units of one entry

struct PlanView {
    int64_t n_strips, n_chunks, chunk_blocks, nnz;
    int split;
    int chunk_len;
    uint32_t hot_cols;
    uint32_t lds_hub_rows;
    const int32_t* strip_row;
    const int32_t* chunk_long;
    const int32_t* long_row;
    const int64_t* long_chunk;
};

constexpr int kReluKeepNan = 2;      // launch_long_reduce's ReLU: 1 maps a NaN to 0, this one keeps it

// the partial rows of the long rows of a table, added in chunk order into c (spmm.hip)
int launch_long_reduce(const gcn_spmm_plan::LongTable& lt, int64_t f, const float* part, int64_t ldp, float* c, int64_t ldc,
                       int relu, int vec_c, hipStream_t st);

}  // namespace gcn
