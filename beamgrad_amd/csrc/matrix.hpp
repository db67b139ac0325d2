// SPDX-License-Identifier: MIT
//
// Products of 16 x 16 blocks by the matrix instructions, of each type of a
// cache. A lane (lane % 16, lane / 16) gives row lane % 16 of either operand, 16
// bytes of it for each step: the products' terms are summed in whatever order, so
// that the same bytes of both rows meet is all that counts. It gets column
// lane % 16 (of the second operand's rows), rows 4 * (lane / 16) + i.
#pragma once

#include <hip/hip_runtime.h>

#include "dbs_cuda.h"

namespace dbs_hip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <int DTYPE>
struct Elem;
template <>
struct Elem<DBS_CUDA_DTYPE_BF16> {
    using T = __bf16;
    using Frag = bf16x8;
    using Quad = bf16x4;
    static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Elem<DBS_CUDA_DTYPE_F16> {
    using T = _Float16;
    using Frag = f16x8;
    using Quad = f16x4;
    static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Elem<DBS_CUDA_DTYPE_F32> {
    using T = float;
    using Frag = f32x4;
    using Quad = f32x4;
    static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

}  // namespace dbs_hip
