// rust-lbfgs_amd/csrc/train/orthogonal.h -- what the units of the orthogonalised update share: values in two parts of 16 bits, and what
// orthogonal.hip hands to orthogonal_short.hip (a short side up to 64) and orthogonal_panel.hip (up to 128, the long one not much more).
#pragma once
#include "common.h"

namespace lt {

typedef f16 half8 __attribute__((ext_vector_type(8)));
typedef f16 half2 __attribute__((ext_vector_type(2)));
typedef f16 half4 __attribute__((ext_vector_type(4)));
typedef float float4_ __attribute__((ext_vector_type(4)));

constexpr int NORM_BLOCKS = 256;  // workgroups of a matrix's norm, each leaving a part of the sum of squares

// (by value: halves of a vector are no lvalues to refer to)
struct Halves {
    f16 hi, lo;
};
__device__ __forceinline__ Halves split(float v) {
    // One value for both: a product that v comes from may otherwise be made anew for hi, and rounded to f16 at once there (an
    // instruction that multiplies and converts), while lo is what is left of its 32-bit rounding: near ties, in one of 2^13
    // values, the two then are off by a step of hi.
    asm("" : "+v"(v));
    const f16 hi = (f16)v;
    return {hi, (f16)(v - (float)hi)};
}

constexpr int SHORT = 64;

struct Short {
    const void* update;
    void *out, *workspace;  // (aligned to 32 bytes, short_workspace() bytes)
    int m, n, tall, batch, steps;  // m <= n; tall: the matrices are n x m
    double a, b, c;
};
LT_INTERNAL uint64_t short_workspace(int64_t batch, int m, int n);
template <class T>
LT_INTERNAL void short_orthogonalize(const Short& p, hipStream_t s);

struct Panel {
    const void* update;
    void *out, *workspace;  // (aligned to 32 bytes, panel_workspace() bytes; it begins with the parts of the norms, NORM_BLOCKS a matrix)
    int m, n, tall, batch, steps;
    double a, b, c, sx, ss, sp;  // ... what X, S and P are multiplied by
    int norms;                   // parts of a norm there are
};
LT_INTERNAL bool panel_fits(int dtype, int64_t batch, int m, int n);
LT_INTERNAL uint64_t panel_workspace(int64_t batch, int m, int n);
template <class T>
LT_INTERNAL void panel_orthogonalize(const Panel& p, hipStream_t s);

}  // namespace lt
