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
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _train

KINDS = {"logistic": 0, "hinge": 1, "squared": 2}
REDUCTIONS = {"tokens": 0, "sequences": 1}


# ------------------------------------------------------------------------------------ token log-probabilities
def _rows(logits, targets, ignore_index):
    """-> (Rows, device, what keeps its memory alive).  A view without its last positions ([:, :-1]) is read as it is."""
    _train.floating("logits", logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., vocabulary] with at least one entry, not {tuple(logits.shape)}")
    if not isinstance(targets, torch.Tensor) or targets.dtype != torch.int64:
        raise TypeError(f"targets must be an int64 tensor, not {getattr(targets, 'dtype', type(targets).__name__)}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(logits.shape[:-1])}, one for each row of logits, not {tuple(targets.shape)}")
    ignore_index = _train.whole("ignore_index", ignore_index, 64)
    dev = _train.on_gpu("logits", logits, (("targets", targets),))
    if not targets.is_contiguous():
        targets = targets.contiguous()
    x = logits
    if x.is_contiguous():
        v = x.shape[-1]
        return _train.Rows(x.data_ptr(), targets.data_ptr(), _train.DTYPES[x.dtype], 0, 1, targets.numel(), v, 0, v, ignore_index), dev, (x, targets)
    n = x.dim()
    if n > 3:
        x = x.detach().flatten(0, -3)  # (a copy only if the leading dimensions have no common stride)
        n = 3
    shape, strides = x.shape, x.stride()
    if shape[-1] > 1 and strides[-1] != 1:
        x = x.detach().contiguous()
        strides = x.stride()
    outer, outer_stride = (shape[0], strides[0]) if n == 3 else (1, 0)
    inner, inner_stride = (shape[-2], strides[-2]) if n > 1 else (1, 0)
    r = _train.Rows(x.data_ptr(), targets.data_ptr(), _train.DTYPES[x.dtype], 0, outer, inner, shape[-1], outer_stride, inner_stride, ignore_index)
    return r, dev, (x, targets)


def token_logprobs_with_lse(logits, targets, temperature=1.0, ignore_index=-100):
    """log softmax(logits / temperature) at the targets, and what its gradient needs again.

    logits [..., V] (float64, float32, bfloat16, float16; the last dimension adjacent, or it is copied), targets [...] int64
    -> (logps [...] in float64 for float64 logits, else float32; lse [..., 2] float64: each row's largest logit m and
    log sum exp((logits - m) / temperature), the two parts of its log-sum-exp m / temperature + that).  A target `ignore_index` gives 0 and its
    row is not read; any other target outside [0, V) gives NaN.  Masked logits may be -inf or the type's lowest value."""
    done = _train.calls().logprobs(logits, targets, temperature, ignore_index)
    if done is not None:
        return _train.results(done)
    rows, dev, keep = _rows(logits, targets, ignore_index)
    L = _train.load()
    logps = torch.empty_like(keep[1], dtype=_train.wide(logits.dtype))  # (the targets, dense)
    lse = logits.new_empty((*targets.shape, 2), dtype=torch.float64)
    size = L.lbfgs_train_token_logprobs_workspace(rows.dtype, rows.outer * rows.inner, rows.vocab)
    ws = logits.new_empty(size, dtype=torch.uint8) if size else None
    _train.enqueue(L.lbfgs_train_token_logprobs, dev, C.byref(rows), temperature, logps.data_ptr(), lse.data_ptr(), _train.ptr(ws), size)
    del keep
    return logps, lse


def token_logprobs_grad(logits, targets, lse, grad, temperature=1.0, ignore_index=-100):
    """The gradient of the logits: grad/temperature * (onehot(target) - softmax(logits/temperature)), [..., V] in the logits' type.

    `lse` and the other arguments are those of token_logprobs_with_lse; `grad` [...] is df/dlogps in its type.  Rows whose
    grad is 0 are not read."""
    done = _train.calls().logprobs_grad(logits, targets, lse, grad, temperature, ignore_index)
    if done is not None:
        return _train.results(done)[0]
    rows, dev, keep = _rows(logits, targets, ignore_index)
    _train.like("lse", lse, "logits", torch.float64, (*targets.shape, 2))
    _train.like("grad", grad, "logits", _train.wide(logits.dtype), targets.shape)
    _train.on_gpu("logits", logits, (("lse", lse), ("grad", grad)))
    L = _train.load()
    lse, grad = lse.contiguous(), grad.contiguous()
    out = logits.new_empty(logits.shape)
    _train.enqueue(L.lbfgs_train_token_logprobs_grad, dev, C.byref(rows), temperature, lse.data_ptr(), grad.data_ptr(), out.data_ptr())
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
        _train.refuse_capture("the backward pass of token_logprobs", "token_logprobs_grad")
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
def _dense(t):
    return t if t is None or t.is_contiguous() else t.detach().contiguous()


def _sequences(logps, offsets, mask, others, wide_grad):
    """-> (Sequences, number of them, the tensors, dense, in the order logps, mask, offsets, others)."""
    _train.floating("logps", logps)
    shape, dtype = logps.shape, logps.dtype
    for name, t in others:
        if t is not None:
            _train.like(name, t, "logps", dtype, shape)
    if mask is not None:
        _train.like("mask", mask, "logps", torch.bool, shape)
    if offsets is None:
        if len(shape) != 2 or shape[0] < 1:
            raise ValueError(f"without offsets logps must be a padded batch [sequences, tokens], not {tuple(shape)}")
        count, bits = shape[0], 0
    else:
        if not isinstance(offsets, torch.Tensor) or offsets.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"offsets must be an int32 or int64 tensor, not {getattr(offsets, 'dtype', type(offsets).__name__)}")
        if offsets.dim() != 1 or offsets.shape[0] < 2:
            raise ValueError(f"offsets must be [sequences + 1], not {tuple(offsets.shape)}")
        if len(shape) != 1:
            raise ValueError(f"with offsets logps must be one-dimensional, not {tuple(shape)}")
        count, bits = offsets.shape[0] - 1, 32 if offsets.dtype == torch.int32 else 64
    x, m, o = _dense(logps), _dense(mask), _dense(offsets)
    q = _train.Sequences(_train.ptr(o), _train.ptr(m), bits, _train.DTYPES[dtype] | (_train.WIDE_GRAD if wide_grad else 0), x.numel(), count)
    return q, count, (x, m, o, *[_dense(t) for _, t in others])


class Preference(NamedTuple):
    f: torch.Tensor         # the mean loss over the pairs
    rewards: torch.Tensor   # [2 P]: beta times each sequence's log ratio
    grad: torch.Tensor      # df/dlogps


def preference(logps, ref_logps=None, *, offsets=None, mask=None, beta=0.1, kind="logistic", label_smoothing=0.0, normalize_lengths=False, wide_grad=False):
    """Loss of paired log ratios, value and gradient.

    2 P sequences: i is preferred to i + P.  With R the sum over a sequence's tokens of logps - ref_logps (ref_logps None:
    of logps; normalize_lengths: divided by their number) and h = beta (R_i - R_{i+P}), the loss of a pair is
        logistic  -(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h)
        hinge     max(0, 1 - h)                  squared   (h / beta - 1 / (2 beta))^2
    All sums are taken in 64 bits.  -> Preference(f, rewards, grad); f and rewards in float64 for float64 data, else float32.
    The gradient is in the type of logps.  In 16 bits that rounds slopes of 1/pairs and 1/length before anything is multiplied into them,
    and float16 has fewer bits for them below 6e-5 and none below 6e-8: wide_grad gives them in float32."""
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {', '.join(KINDS)}, not {kind!r}")
    calls = _train.calls()
    done = (calls.preference_wide if wide_grad else calls.preference)(logps, ref_logps, offsets, mask, beta, label_smoothing, KINDS[kind], normalize_lengths)
    if done is not None:
        return Preference._make(_train.results(done))
    others = (("ref_logps", ref_logps),)
    q, count, (x, m, o, ref) = _sequences(logps, offsets, mask, others, wide_grad)
    dev = _train.on_gpu("logps", logps, (("offsets", offsets), ("mask", mask), *others))
    L, out = _train.load(), _train.wide(x.dtype)
    f, rewards = x.new_empty((), dtype=out), x.new_empty(count, dtype=out)
    grad = torch.empty_like(x, dtype=out if wide_grad else x.dtype)
    size = L.lbfgs_train_sequences_workspace(q.tokens, count)
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    _train.enqueue(L.lbfgs_train_preference, dev, C.byref(q), x.data_ptr(), _train.ptr(ref), beta, label_smoothing, KINDS[kind], bool(normalize_lengths),
                   f.data_ptr(), rewards.data_ptr(), grad.data_ptr(), _train.ptr(ws), size)
    return Preference(f, rewards, grad)


class Policy(NamedTuple):
    f: torch.Tensor              # the loss
    kl: torch.Tensor             # mean of exp(q) - 1 - q, q = ref_logps - logps, over the tokens that count; 0 without a KL term in f
    clip_fraction: torch.Tensor  # share of them whose ratio is clipped
    grad: torch.Tensor           # df/dlogps


def policy(logps, old_logps, advantages, *, ref_logps=None, offsets=None, mask=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="tokens",
           wide_grad=False):
    """Clipped policy loss with a KL term, value and gradient.

    With r = exp(logps - old_logps), q = ref_logps - logps and a token's advantage A (advantages like logps, or [S, 1]: one for
    each sequence), a token's loss is -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(q) - 1 - q); f is the
    mean over all tokens ("tokens"), or over the sequences that have any of their own means ("sequences").  clip_high may be
    infinite.  -> Policy(f, kl, clip_fraction, grad); the scalars in float64 for float64 data, else float32.  The gradient is in the
    type of logps; wide_grad as in preference: in float16 slopes of 1/tokens lose bits from some 10^4 tokens on."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(REDUCTIONS)}, not {reduction!r}")
    if kl_coef != 0 and ref_logps is None:
        raise ValueError("a KL term needs ref_logps")
    calls = _train.calls()
    done = (calls.policy_wide if wide_grad else calls.policy)(logps, old_logps, advantages, ref_logps, offsets, mask, clip_low, clip_high, kl_coef, REDUCTIONS[reduction])
    if done is not None:
        return Policy._make(_train.results(done))
    others = (("old_logps", old_logps), ("ref_logps", ref_logps))
    q, count, (x, m, o, old, ref) = _sequences(logps, offsets, mask, others, wide_grad)
    per_token = not (isinstance(advantages, torch.Tensor) and advantages.shape == (count, 1))
    _train.like("advantages", advantages, "logps (or [sequences, 1])", x.dtype, x.shape if per_token else (count, 1))
    dev = _train.on_gpu("logps", logps, (("offsets", offsets), ("mask", mask), ("advantages", advantages), *others))
    L, adv, out = _train.load(), _dense(advantages), _train.wide(x.dtype)
    f, kl, clipped = x.new_empty(3, dtype=out).unbind()
    grad = torch.empty_like(x, dtype=out if wide_grad else x.dtype)
    size = L.lbfgs_train_sequences_workspace(q.tokens, count)
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    _train.enqueue(L.lbfgs_train_policy, dev, C.byref(q), x.data_ptr(), old.data_ptr(), _train.ptr(ref), adv.data_ptr(), per_token, clip_low, clip_high, kl_coef,
                   REDUCTIONS[reduction], f.data_ptr(), kl.data_ptr(), clipped.data_ptr(), grad.data_ptr(), _train.ptr(ws), size)
    return Policy(f, kl, clipped, grad)


class _ValueAndGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, result):
        ctx.save_for_backward(result.grad)
        ctx.dtype = logps.dtype
        return result.f

    @staticmethod
    @once_differentiable
    def backward(ctx, up):
        _train.refuse_capture("the backward pass of a loss", "preference or policy")
        (grad,) = ctx.saved_tensors  # (in 32 bits or more, as what comes in: the product is rounded, once)
        return (grad * up).to(ctx.dtype), None


def _differentiable(name, function, logps, *others, **options):
    wanted = isinstance(logps, torch.Tensor) and logps.requires_grad and torch.is_grad_enabled()
    result = function(logps, *others, wide_grad=wanted, **options)
    if not wanted:
        return result.f
    _train.refuse_capture(name + "_loss", name)
    return _ValueAndGrad.apply(logps, result)


def preference_loss(logps, ref_logps=None, **options):
    """`preference(...).f`, differentiable in logps (the reference is a constant)."""
    return _differentiable("preference", preference, logps, ref_logps, **options)


def policy_loss(logps, old_logps, advantages, **options):
    """`policy(...).f`, differentiable in logps (old and reference log-probabilities and advantages are constants)."""
    return _differentiable("policy", policy, logps, old_logps, advantages, **options)
