"""Losses of language-model tuning with their gradients: the inside of an `evaluate` closure whose f is such a loss.

    logps, lse = losses.token_logprobs_with_lse(logits, targets)         # one pass over the logits
    r = losses.preference(logps, ref_logps, offsets=offsets)             # r.f, r.rewards, r.grad = df/dlogps
    dlogits = losses.token_logprobs_grad(logits, targets, lse, r.grad)   # -> back through the model, into g

A loss gives its value and its gradient in one call, as an objective of this package does; nothing is copied to the host.
`token_logprobs`, `preference_loss` and `policy_loss` are the same operators for torch's autograd.

Sequences: with `offsets` [S + 1] (int32 or int64, not decreasing) the tensors over tokens are one-dimensional and sequence
s is [offsets[s], offsets[s + 1]); without, they are a padded batch [S, L].  `mask` (bool, the same shape) says which tokens
count; what is masked, or belongs to no sequence, is not looked at and gets the gradient 0.

Kernels: rust-lbfgs_amd/csrc/train/{logprobs,losses}.hip behind include/lbfgs_train.h.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _train

KINDS = {"logistic": 0, "hinge": 1, "squared": 2}
REDUCTIONS = {"tokens": 0, "sequences": 1}


# ------------------------------------------------------------------------------------ token log-probabilities
def _rows(logits, targets, ignore_index):
    """-> (Rows, what keeps its memory alive).  A view without its last positions ([:, :-1]) is read as it is."""
    _train.floating("logits", logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., vocabulary] with at least one entry, not {tuple(logits.shape)}")
    if not isinstance(targets, torch.Tensor) or targets.dtype != torch.int64:
        raise TypeError(f"targets must be an int64 tensor, not {getattr(targets, 'dtype', type(targets).__name__)}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(logits.shape[:-1])}, one for each row of logits, not {tuple(targets.shape)}")
    _train.on_gpu(("logits", logits), targets=targets)
    targets = targets.contiguous()
    x = logits.detach()
    if x.dim() > 3:
        x = x.flatten(0, -3)  # (a copy only if the leading dimensions have no common stride)
    while x.dim() < 3:
        x = x.unsqueeze(0)
    if (x.shape[-1] > 1 and x.stride(-1) != 1) or any(n > 1 and st < 0 for n, st in zip(x.shape, x.stride())):
        x = x.contiguous()
    r = _train.Rows(x.data_ptr(), targets.data_ptr(), _train.DTYPES[x.dtype], 0, x.shape[0], x.shape[1], x.shape[2], x.stride(0), x.stride(1),
                    int(ignore_index))
    return r, (x, targets)


def token_logprobs_with_lse(logits, targets, temperature=1.0, ignore_index=-100):
    """log softmax(logits / temperature) at the targets, and what its gradient needs again.

    logits [..., V] (float64, float32, bfloat16, float16; the last dimension adjacent, or it is copied), targets [...] int64
    -> (logps [...] in float64 for float64 logits, else float32; lse [..., 2] float64: each row's largest logit m and
    log sum exp((logits - m) / temperature), the two parts of its log-sum-exp m / temperature + that).  A target `ignore_index` gives 0 and its
    row is not read; any other target outside [0, V) gives NaN.  Masked logits may be -inf or the type's lowest value."""
    rows, keep = _rows(logits, targets, ignore_index)
    L, dev = _train.load(), logits.device
    with _train.current(dev):
        logps = torch.empty(targets.shape, dtype=_train.wide(logits.dtype), device=dev)
        lse = torch.empty((*targets.shape, 2), dtype=torch.float64, device=dev)
        size = L.lbfgs_train_token_logprobs_workspace(rows.dtype, targets.numel(), rows.vocab)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _train.check(L.lbfgs_train_token_logprobs(C.byref(rows), temperature, logps.data_ptr(), lse.data_ptr(), _train.ptr(ws), size,
                                                  _train.stream_of(dev)))
    del keep
    return logps, lse


def token_logprobs_grad(logits, targets, lse, grad, temperature=1.0, ignore_index=-100):
    """The gradient of the logits: grad/temperature * (onehot(target) - softmax(logits/temperature)), [..., V] in the logits' type.

    `lse` and the other arguments are those of token_logprobs_with_lse; `grad` [...] is df/dlogps in its type.  Rows whose
    grad is 0 are not read."""
    rows, keep = _rows(logits, targets, ignore_index)
    _train.like("lse", lse, "the logits", logits, torch.float64, (*targets.shape, 2))
    _train.like("grad", grad, "the logits", logits, _train.wide(logits.dtype), targets.shape)
    dev = _train.on_gpu(("logits", logits), lse=lse, grad=grad)
    L = _train.load()
    with _train.current(dev):
        lse, grad = lse.contiguous(), grad.contiguous()
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        _train.check(L.lbfgs_train_token_logprobs_grad(C.byref(rows), temperature, lse.data_ptr(), grad.data_ptr(), out.data_ptr(),
                                                       _train.stream_of(dev)))
    del keep
    return out


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature, ignore_index):
        logps, lse = token_logprobs_with_lse(logits, targets, temperature, ignore_index)
        ctx.save_for_backward(logits, targets, lse)
        ctx.extra = temperature, ignore_index
        return logps

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        logits, targets, lse = ctx.saved_tensors
        return token_logprobs_grad(logits, targets, lse, grad, *ctx.extra), None, None, None


def token_logprobs(logits, targets, temperature=1.0, ignore_index=-100):
    """log softmax(logits / temperature) at the targets; differentiable in the logits.  See token_logprobs_with_lse."""
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        if logits.is_cuda:
            _train.refuse_capture("token_logprobs", "token_logprobs_with_lse and token_logprobs_grad")
        return _TokenLogprobs.apply(logits, targets, temperature, ignore_index)
    return token_logprobs_with_lse(logits, targets, temperature, ignore_index)[0]


# ------------------------------------------------------------------------------------ losses over sequences
def _sequences(logps, offsets, mask, others):
    """-> (Sequences, number of them, the tensors, dense, in the order logps, mask, offsets, others)."""
    _train.floating("logps", logps)
    for name, t in others.items():
        if t is not None:
            _train.like(name, t, "logps", logps)
    if mask is not None:
        _train.like("mask", mask, "logps", logps, torch.bool)
    if offsets is None:
        if logps.dim() != 2 or logps.shape[0] < 1:
            raise ValueError(f"without offsets logps must be a padded batch [sequences, tokens], not {tuple(logps.shape)}")
        count = logps.shape[0]
    else:
        if not isinstance(offsets, torch.Tensor) or offsets.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"offsets must be an int32 or int64 tensor, not {getattr(offsets, 'dtype', type(offsets).__name__)}")
        if offsets.dim() != 1 or offsets.shape[0] < 2:
            raise ValueError(f"offsets must be [sequences + 1], not {tuple(offsets.shape)}")
        if logps.dim() != 1:
            raise ValueError(f"with offsets logps must be one-dimensional, not {tuple(logps.shape)}")
        count = offsets.shape[0] - 1
    dense = [t if t is None else t.detach().contiguous() for t in (logps, mask, offsets, *others.values())]
    bits = 0 if offsets is None else 32 if offsets.dtype == torch.int32 else 64
    q = _train.Sequences(_train.ptr(dense[2]), _train.ptr(dense[1]), bits, _train.DTYPES[logps.dtype], logps.numel(), count)
    return q, count, dense


class Preference(NamedTuple):
    f: torch.Tensor         # the mean loss over the pairs
    rewards: torch.Tensor   # [2 P]: beta times each sequence's log ratio
    grad: torch.Tensor      # df/dlogps


def preference(logps, ref_logps=None, *, offsets=None, mask=None, beta=0.1, kind="logistic", label_smoothing=0.0, normalize_lengths=False):
    """Loss of paired log ratios, value and gradient.

    2 P sequences: i is preferred to i + P.  With R the sum over a sequence's tokens of logps - ref_logps (ref_logps None:
    of logps; normalize_lengths: divided by their number) and h = beta (R_i - R_{i+P}), the loss of a pair is
        logistic  -(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h)
        hinge     max(0, 1 - h)                  squared   (h / beta - 1 / (2 beta))^2
    All sums are taken in 64 bits.  -> Preference(f, rewards, grad); f and rewards in float64 for float64 data, else float32."""
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {', '.join(KINDS)}, not {kind!r}")
    q, count, (x, m, o, ref) = _sequences(logps, offsets, mask, {"ref_logps": ref_logps})
    dev = _train.on_gpu(("logps", logps), offsets=offsets, mask=mask, ref_logps=ref_logps)
    L = _train.load()
    with _train.current(dev):
        out = _train.wide(x.dtype)
        f, rewards = torch.empty((), dtype=out, device=dev), torch.empty(count, dtype=out, device=dev)
        grad = torch.empty_like(x)
        size = L.lbfgs_train_sequences_workspace(q.tokens, count)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        _train.check(L.lbfgs_train_preference(C.byref(q), x.data_ptr(), _train.ptr(ref), beta, label_smoothing, KINDS[kind], int(normalize_lengths),
                                              f.data_ptr(), rewards.data_ptr(), grad.data_ptr(), ws.data_ptr(), size, _train.stream_of(dev)))
    return Preference(f, rewards, grad)


class Policy(NamedTuple):
    f: torch.Tensor              # the loss
    kl: torch.Tensor             # mean of exp(q) - 1 - q, q = ref_logps - logps, over the tokens that count
    clip_fraction: torch.Tensor  # share of them whose ratio is clipped
    grad: torch.Tensor           # df/dlogps


def policy(logps, old_logps, advantages, *, ref_logps=None, offsets=None, mask=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="tokens"):
    """Clipped policy loss with a KL term, value and gradient.

    With r = exp(logps - old_logps), q = ref_logps - logps and a token's advantage A (advantages like logps, or [S, 1]: one for
    each sequence), a token's loss is -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(q) - 1 - q); f is the
    mean over all tokens ("tokens"), or over the sequences that have any of their own means ("sequences").  clip_high may be
    infinite.  -> Policy(f, kl, clip_fraction, grad); the scalars in float64 for float64 data, else float32."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(REDUCTIONS)}, not {reduction!r}")
    if kl_coef != 0 and ref_logps is None:
        raise ValueError("a KL term needs ref_logps")
    q, count, (x, m, o, old, ref) = _sequences(logps, offsets, mask, {"old_logps": old_logps, "ref_logps": ref_logps})
    per_token = not (isinstance(advantages, torch.Tensor) and tuple(advantages.shape) == (count, 1))
    _train.like("advantages", advantages, "logps (or [sequences, 1])", logps, shape=None if per_token else (count, 1))
    dev = _train.on_gpu(("logps", logps), offsets=offsets, mask=mask, old_logps=old_logps, advantages=advantages, ref_logps=ref_logps)
    L = _train.load()
    with _train.current(dev):
        adv = advantages.detach().contiguous()
        f, kl, clipped = torch.empty(3, dtype=_train.wide(x.dtype), device=dev).unbind()
        grad = torch.empty_like(x)
        size = L.lbfgs_train_sequences_workspace(q.tokens, count)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        _train.check(L.lbfgs_train_policy(C.byref(q), x.data_ptr(), old.data_ptr(), _train.ptr(ref), adv.data_ptr(), int(per_token), clip_low, clip_high,
                                          kl_coef, REDUCTIONS[reduction], f.data_ptr(), kl.data_ptr(), clipped.data_ptr(), grad.data_ptr(), ws.data_ptr(),
                                          size, _train.stream_of(dev)))
    return Policy(f, kl, clipped, grad)


class _ValueAndGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, result):
        ctx.save_for_backward(result.grad)
        return result.f

    @staticmethod
    @once_differentiable
    def backward(ctx, up):
        return ctx.saved_tensors[0] * up.to(ctx.saved_tensors[0].dtype), None


def _differentiable(name, logps, result):
    if logps.requires_grad and torch.is_grad_enabled():
        _train.refuse_capture(name + "_loss", name)
        return _ValueAndGrad.apply(logps, result)
    return result.f


def preference_loss(logps, ref_logps=None, **options):
    """`preference(...).f`, differentiable in logps (the reference is a constant)."""
    return _differentiable("preference", logps, preference(logps, ref_logps, **options))


def policy_loss(logps, old_logps, advantages, **options):
    """`policy(...).f`, differentiable in logps (old and reference log-probabilities and advantages are constants)."""
    return _differentiable("policy", logps, policy(logps, old_logps, advantages, **options))
