"""Directions for matrix parameters, beside the optimiser's own for vectors (the two-loop recursion, the orthant projection).

    d = directions.orthogonalize(-gradient.view(rows, cols).float())      # every singular value brought near 1

The optimiser's gradients are float64, an orthogonalised update is not: it is a step of a descent of its own over matrices, and the polynomial
leaves singular values tens of percent apart.

Kernels: rust-lbfgs_amd/csrc/train/orthogonal.hip behind include/lbfgs_train.h.
"""
from __future__ import annotations

import torch

from . import _train

# a s + b s^3 + c s^5, the published constants of K. Jordan and others ("Muon: an optimizer for hidden layers in neural networks", 2024): tuned
# for a steep start, not for 1; the values that have grown stay within 0.68 .. 1.21
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(update, *, steps=5, coefficients=COEFFICIENTS):
    """`update` [..., rows, cols] (float32, bfloat16, float16) with its singular values brought near each other.

    Each matrix is divided by its Frobenius norm (zeros stay zeros); then, `steps` times, every singular value s becomes
    a s + b s^3 + c s^5 while the singular vectors stay: X <- (a I + b S + c S S) X with S = X X^T of the shorter side.  With the
    default coefficients five steps bring all but the smallest (below 1/650 of the norm) into 0.68 .. 1.21.
    Products have 32-bit precision or more for all types, and the result is rounded once; for 16-bit types the last steps are
    taken together, which adds at most half of that rounding's bound (2^-10 of the result's norm in bfloat16, 2^-13 in float16).
    Coefficients that lead singular values of [0, 1] beyond 64, or multiply one by 128 or more in a step, are refused.
    A direction, not a part of the loss: nothing is recorded for autograd.
    A matrix that holds a NaN or an infinity gives NaN, the others of its batch are not touched by it."""
    done = _train.calls().orthogonalize(update, steps, *coefficients) if len(coefficients) == 3 else None
    if done is not None:
        return _train.results(done)[0]
    _train.floating("update", update)
    if update.dtype == torch.float64:
        raise TypeError("update must be float32, bfloat16 or float16: the polynomial itself leaves singular values 20 % apart, "
                        "64 bits have nothing to hold (convert it)")
    if update.dim() < 2:
        raise ValueError(f"update must be [..., rows, cols], not {tuple(update.shape)}")
    if len(coefficients) != 3:
        raise ValueError(f"coefficients are (a, b, c), not {coefficients!r}")
    steps = _train.whole("steps", steps, 32)
    dev = _train.on_gpu("update", update)
    L = _train.load()
    g = update if update.is_contiguous() else update.detach().contiguous()
    out = g.new_empty(g.shape)
    rows, cols = g.shape[-2:]
    batch = g.numel() // (rows * cols) if rows and cols else 0
    size = L.lbfgs_train_orthogonalize_workspace(_train.DTYPES[g.dtype], batch, rows, cols)
    ws = g.new_empty(size, dtype=torch.uint8) if size else None
    _train.enqueue(L.lbfgs_train_orthogonalize, dev, _train.DTYPES[g.dtype], batch, rows, cols, g.data_ptr(), out.data_ptr(), steps, *coefficients,
                   _train.ptr(ws), size)
    return out
