// f32 values as sums of bf16 ones, which the matrix cores multiply exactly and sum in f32.
#pragma once

#include "kernels/device_common.h"

namespace dlk {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// The first 8 bits of each of eight values, cut off (no finite value becomes infinite), and the rest: three parts hold all 24.
__device__ __forceinline__ u32x4 cut(float (&v)[8]) {
    u32x4 part;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(v[2 * i]), b = __float_as_uint(v[2 * i + 1]);
        part[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        v[2 * i] -= __uint_as_float(a & 0xffff0000u);
        v[2 * i + 1] -= __uint_as_float(b & 0xffff0000u);
    }
    return part;
}
__device__ __forceinline__ uint16_t cut(float& v) {
    const uint32_t a = __float_as_uint(v);
    v -= __uint_as_float(a & 0xffff0000u);
    return static_cast<uint16_t>(a >> 16);
}

// 16 rows by 16 columns: lane l holds 8 entries of row (of `a`) and column (of `b`) l % 16, those of the sum's index from
// 8 (l / 16) on, and the sum's column l % 16, rows 4 (l / 16) to + 3.
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), sum, 0, 0, 0);
}
// The same of f32: lane l holds one entry of row and column l % 16, at index l / 16 of four.
__device__ __forceinline__ f32x4 product(float a, float b, f32x4 sum) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, sum, 0, 0, 0);
}

} // namespace dlk
