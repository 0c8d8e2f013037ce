// All-reductions over G neighbouring lanes of a wave (G a power of two up to 64) on the vector ALU: the partners at
// distance 1 and 2 by quad permutes, 4 and 8 by the mirrored half row and row (the quads, then the halves, are uniform
// by then, so the mirror image holds the partner's value), 16 and 32 by the lane-swap instructions.  A shuffle through
// LDS costs a round trip there and occupies the pipe that all waves of a compute unit share.
#pragma once

#include <hip/hip_runtime.h>

namespace gcn {

struct OpAdd {
    static __device__ __forceinline__ float f(float a, float b) { return a + b; }
};
struct OpMax {
    static __device__ __forceinline__ float f(float a, float b) { return fmaxf(a, b); }
};
struct OpMinInt {      // on the bits: a non-negative int carried in a float register
    static __device__ __forceinline__ float f(float a, float b) {
        const int x = __float_as_int(a), y = __float_as_int(b);
        return __int_as_float(x < y ? x : y);
    }
};

template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}

template <int G, class Op>
__device__ __forceinline__ float lanes_reduce(float v) {
    if (G >= 2) v = Op::f(v, dpp_move<0xB1>(v));       // quad_perm [1,0,3,2]
    if (G >= 4) v = Op::f(v, dpp_move<0x4E>(v));       // quad_perm [2,3,0,1]
    if (G >= 8) v = Op::f(v, dpp_move<0x141>(v));      // row_half_mirror
    if (G >= 16) v = Op::f(v, dpp_move<0x140>(v));     // row_mirror
    if (G >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = Op::f(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    if (G >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = Op::f(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    return v;
}

}  // namespace gcn
