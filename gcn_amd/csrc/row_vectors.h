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

// A row of f columns in G lanes, VPL vectors a lane: lane `sub` holds the columns 4 (sub + G v) .. + 3.  What lies past the
// row's end is NOT zero after load_row (a value of the next row, or of column 0): the caller replaces it, knowing that
// element (v, q) is a column of the row where 4 G v + q < f - 4 sub.  `last`: the row is the matrix's last one.
template <int G, int VPL>
__device__ __forceinline__ void load_row(const float* __restrict__ row, int sub, int f, bool last, float (&x)[VPL][4]) {
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        // a vector that begins in the row may end in the next one, whose values are replaced below; behind the last
        // row there may be nothing, and rows of one column may end less than a vector behind this one
        const int at = 4 * (sub + G * v);
        if ((!last && f >= 2) || at + 4 <= f) {
            const f4u t = *reinterpret_cast<const f4u*>(row + (at < f ? at : 0));
            x[v][0] = t.x;
            x[v][1] = t.y;
            x[v][2] = t.z;
            x[v][3] = t.w;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) x[v][q] = at + q < f ? row[at + q] : 0.0f;
        }
    }
}
// the row's columns; the one vector that the row's end cuts is stored by one instruction of its length
template <int G, int VPL>
__device__ __forceinline__ void store_row(float* __restrict__ row, int sub, int f, const float (&g)[VPL][4]) {
    const int cut = f & 3;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        const int at = 4 * (sub + G * v);
        if (at + 4 <= f) *reinterpret_cast<f4u*>(row + at) = f4u{g[v][0], g[v][1], g[v][2], g[v][3]};
        if (cut != 0 && at < f && at + 4 > f) {
            typedef float f2u __attribute__((ext_vector_type(2), aligned(4)));
            typedef float f3u __attribute__((ext_vector_type(3), aligned(4)));
            if (cut == 1) row[at] = g[v][0];
            else if (cut == 2) *reinterpret_cast<f2u*>(row + at) = f2u{g[v][0], g[v][1]};
            else *reinterpret_cast<f3u*>(row + at) = f3u{g[v][0], g[v][1], g[v][2]};
        }
    }
}

// out[c] = sum over the rows of part [rows x f], in a fixed order (norm.hip)
int launch_column_sums(int64_t rows, int64_t f, const float* part, float* out, hipStream_t st);

}  // namespace gcn
