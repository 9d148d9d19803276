// Warp-level bf16 matrix product for the kernels that are bound by memory and
// have too few rows for a tcgen05 tile (one query per sequence, a few tokens
// per weight matrix): D[16,8] += A[16,16] B[16,8] with f32 accumulation.
//
// Lane l = 4 g + t (g 0..7, t 0..3) holds
//   A: a[0] = rows g, columns 2t, 2t+1; a[1] = row g+8, same columns;
//      a[2] = row g, columns 2t+8, 2t+9; a[3] = row g+8, columns 2t+8, 2t+9
//   B: b0 = rows 2t, 2t+1 of column g; b1 = rows 2t+8, 2t+9 of column g
//   D: d[0], d[1] = row g, columns 2t, 2t+1; d[2], d[3] = row g+8
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace hx {

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transposes an 8 x 8 matrix of 16-bit elements held one row per 4 lanes.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// (low halves of x and y) and (high halves), x in the lower half.
__device__ __forceinline__ uint32_t pair_lo(uint32_t x, uint32_t y) { return __byte_perm(x, y, 0x5410); }
__device__ __forceinline__ uint32_t pair_hi(uint32_t x, uint32_t y) { return __byte_perm(x, y, 0x7632); }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

}  // namespace hx
