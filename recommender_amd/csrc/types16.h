// Element types of the lookup and loss operators: 32-bit floats and the two 16-bit formats, all arithmetic on them in 32 bits.
#pragma once
#include "reco_common.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// N consecutive values of T moved as one access (N * sizeof(T) a power of two up to 16)
template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// A sum of many values and what rounding has put into it too much: its error does not grow with their number.  MAY_BE_INFINITE: an infinite
// sum stays so, as a plain one does (else it is NaN from the next value on).
struct Sum {
    float s = 0.f, over = 0.f;
    template <bool MAY_BE_INFINITE> __device__ __forceinline__ void add(float v)
    {
        const float part = v - over, total = s + part;
        over = !MAY_BE_INFINITE || fabsf(total) < INFINITY ? (total - s) - part : 0.f;
        s = total;
    }
    __device__ __forceinline__ void scale(float f)
    {
        s *= f;
        over *= f;
    }
};

// Calls fn with a value of the element type that `dtype` (RECO_DT_*) names; fn returns the call's status.
template <typename F> static int reco_with_type(int dtype, F&& fn)
{
    switch (dtype) {
    case RECO_DT_F32: return fn(float());
    case RECO_DT_BF16: return fn(__bf16());
    case RECO_DT_F16: return fn(_Float16());
    default: reco_set_error("unknown element type %d", dtype); return RECO_EINVAL;
    }
}
