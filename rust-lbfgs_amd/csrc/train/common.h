// rust-lbfgs_amd/csrc/train/common.h -- what the units of liblbfgs_train.so share: element types, unaligned vector loads,
// wave reductions, the error text of a refused call.  Not installed, not part of the ABI (include/lbfgs_train.h).
#pragma once
#include "../../../include/lbfgs_train.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#define LT_INTERNAL __attribute__((visibility("hidden")))

LT_INTERNAL int lt_fail(int code, const char* fmt, ...);  // (losses.hip) keeps the text for lbfgs_train_last_error
LT_INTERNAL int lt_launched(const char* what);            // the launch error of the kernels just enqueued, if any

namespace lt {

typedef __bf16 bf16;
typedef _Float16 f16;

// An element type and the type its arithmetic is done in: 32 bits or more.
template <class T>
struct Num {
    typedef float acc;
};
template <>
struct Num<double> {
    typedef double acc;
};

constexpr int WAVE = 64;

// N consecutive elements as one load / store of up to 16 bytes at the element's own alignment: global memory is byte
// addressable for vector accesses on gfx950, so odd row lengths and shifted views need no scalar path of their own
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[N];
};
template <class T>
constexpr int vec_len() {
    return 16 / (int)sizeof(T);
}

template <class A>
__device__ __forceinline__ A shfl_xor(A v, int o) {
    return __shfl_xor(v, o, WAVE);
}
template <class A>
__device__ __forceinline__ A wave_sum(A v) {
#pragma unroll
    for (int o = WAVE / 2; o; o >>= 1) v += shfl_xor(v, o);
    return v;
}
template <class A>
__device__ __forceinline__ A wave_max(A v) {
#pragma unroll
    for (int o = WAVE / 2; o; o >>= 1) {
        const A w = shfl_xor(v, o);
        v = w > v ? w : v;
    }
    return v;
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double exp2_of(double x) { return exp2(x); }

}  // namespace lt
