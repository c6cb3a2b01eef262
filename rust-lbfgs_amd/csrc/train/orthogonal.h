// rust-lbfgs_amd/csrc/train/orthogonal.h -- what orthogonal.hip hands to orthogonal_short.hip: updates of a short side up to SHORT.
#pragma once
#include "common.h"

namespace lt {

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

}  // namespace lt
