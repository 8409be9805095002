// Rows of floats as operands of the float matrix cores, in the order in which the plain kernels add a dot product up
// (attention_f32.hip, attention_weighed.hip).
#pragma once

#include "common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Lane (r, g) = 16 g + r holds elements 4 g .. 4 g + 3 of its row; afterwards element e of it is element 4 e + g of the row: the order in which
// four steps of the matrix instruction take them.  And the other way round.
__device__ __forceinline__ void across_groups(f32x4& x) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const u32x2 v = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[e]), __float_as_uint(x[e + 2]), false, false);
        x[e] = __uint_as_float(v[0]), x[e + 2] = __uint_as_float(v[1]);
    }
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
        const u32x2 v = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[e]), __float_as_uint(x[e + 1]), false, false);
        x[e] = __uint_as_float(v[0]), x[e + 1] = __uint_as_float(v[1]);
    }
}
