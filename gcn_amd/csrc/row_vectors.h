// Rows of float32 in vectors of four, at any alignment and any length.
#pragma once

#include <hip/hip_runtime.h>

namespace gcn {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // 128-bit accesses at any element

// columns c .. c + 3 of a row of f columns, zero past its end.  The address is moved back inside the row instead of
// a branch around the load, so that the loads of a row stay in flight together.
__device__ __forceinline__ void load_cols(const float* __restrict__ row, int c, int f, float (&v)[4]) {
    if (f >= 4) {
        const int from = c + 4 <= f ? c : f - 4;
        const f4u t = *reinterpret_cast<const f4u*>(row + from);
        const int gone = c - from;                 // columns of t that belong to the vector before this one
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        if (gone > 0) {
            v[0] = gone == 1 ? t.y : gone == 2 ? t.z : gone == 3 ? t.w : 0.0f;
            v[1] = gone == 1 ? t.z : gone == 2 ? t.w : 0.0f;
            v[2] = gone == 1 ? t.w : 0.0f;
            v[3] = 0.0f;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < f ? row[c + e] : 0.0f;
    }
}
__device__ __forceinline__ void store_cols(float* __restrict__ row, int c, int f, const float (&v)[4]) {
    if (c + 4 <= f) {
        f4u t = {v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f4u*>(row + c) = t;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (c + e < f) row[c + e] = v[e];
    }
}

// out[c] = sum over the rows of part [rows x f], in a fixed order (norm.hip)
int launch_column_sums(int64_t rows, int64_t f, const float* part, float* out, hipStream_t st);

}  // namespace gcn
