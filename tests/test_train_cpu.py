"""The loss and update operators without a GPU: the library's exports against its header, and every refusal -- of the C entry
points (before anything touches a device) and of the Python functions."""
import ctypes as C
import math
import os
import re

import pytest
import torch

import rust_lbfgs_amd as R
from rust_lbfgs_amd import _build, _ffi, _train, directions, losses

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG = _ffi.HIP_ERR_ARG
P = 4096  # a pointer that is not null; no refused call looks at it


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_build.TRAIN_LIB):
        _build.build_train()
    if not os.path.exists(_build.CALLS_LIB):
        _build.build_calls()
    return _train.load()


def header():
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "lbfgs_train.h")).read(), flags=re.S)


def test_exports_are_the_headers(lib):
    names = sorted(set(re.findall(r"\b(lbfgs_train_\w+)\s*\(", header())))
    assert names == sorted(_train.SIGNATURES) and len(names) >= 11
    raw = C.CDLL(_build.TRAIN_LIB)
    assert all(hasattr(raw, n) for n in names)
    want = int(re.search(r"#define LBFGS_TRAIN_ABI_VERSION (\d+)", header()).group(1))
    assert lib.lbfgs_train_abi_version() == want == _train.ABI_VERSION
    assert lib.lbfgs_train_build_id().decode() == _build.train_build_id() == _build.embedded_id(_build.TRAIN_LIB, "LBFGS_TRAIN_BUILD_ID")


def test_structs_match_the_header(tmp_path):
    import subprocess

    structs = {"lbfgs_train_rows": _train.Rows, "lbfgs_train_sequences": _train.Sequences}
    lines = ["#include <stdio.h>", '#include "lbfgs_train.h"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    for ln in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, val = ln.split()
        assert int(val) == (C.sizeof(structs[name]) if field == "size" else getattr(structs[name], field).offset), ln


def test_no_kernel_uses_scratch_memory(lib):
    txt = open(_build.TRAIN_RESOURCES).read()
    sizes = re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", txt)
    assert len(sizes) >= 40 and set(sizes) == {"0"}


def test_inline_assembly_names_the_special_registers_it_writes():
    """What the compiler is not told of it may keep something in."""
    found = 0
    for unit in _build.TRAIN_SRCS:
        for text in re.findall(r"\basm\b\s*(?:volatile)?\s*\((.*?)\);", open(unit).read(), flags=re.S):
            clobbers = text.rsplit(":", 1)[1] if text.count(":") >= 3 else ""
            for instruction in re.split(r"\\n|;", text.split(":")[0].replace("\\t", " ").replace('"', " ")):
                for register in ("m0", "vcc", "exec", "scc"):
                    if re.match(r"\s*\w+ " + register + r"\b", instruction):
                        found += 1
                        assert f'"{register}"' in clobbers, (unit, text)
    assert found  # the copies to LDS


def test_the_library_is_rebuilt_when_its_sources_differ(lib, monkeypatch):
    monkeypatch.setattr(_build, "train_build_id", lambda: "0" * 16)
    monkeypatch.setattr(_train, "_LIB", None)
    with pytest.raises(ImportError, match="build id"):
        _train.load()


# ------------------------------------------------------------------------------------ C entry points
def rows(**kw):
    v = dict(logits=P, targets=P, dtype=1, _pad=0, outer=1, inner=2, vocab=8, outer_stride=16, inner_stride=8, ignore_index=-100) | kw
    return C.byref(_train.Rows(*[v[f] for f, _ in _train.Rows._fields_]))


def seqs(**kw):
    v = dict(offsets=P, mask=None, offset_bits=64, dtype=1, tokens=10, count=4) | kw
    return C.byref(_train.Sequences(*[v[f] for f, _ in _train.Sequences._fields_]))


def refused(rc, text):
    assert rc == ARG
    assert text in _train.load().lbfgs_train_last_error().decode()


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=4), "element type"), (dict(dtype=-1), "element type"), (dict(vocab=0), "rows of 0 logits"), (dict(outer=-1), "rows of"),
    (dict(outer=1 << 40, inner=1 << 40), "rows of"), (dict(logits=None), "are needed"), (dict(targets=None), "are needed")])
def test_c_rows_refusals(lib, kw, text):
    refused(lib.lbfgs_train_token_logprobs(rows(**kw), 1.0, P, P, P, 1 << 30, None), text)
    refused(lib.lbfgs_train_token_logprobs_grad(rows(**kw), 1.0, P, P, P, None), text)


def test_c_logprobs_refusals(lib):
    for t in (0.0, -1.0, math.nan, math.inf):
        refused(lib.lbfgs_train_token_logprobs(rows(), t, P, P, P, 1 << 30, None), "temperature")
        refused(lib.lbfgs_train_token_logprobs_grad(rows(), t, P, P, P, None), "temperature")
    for dtype, values in ((0, (1e-301, 1e301)), (1, (1e-38, 1e38)), (2, (1e-38, 1e38)), (3, (1e-38, 1e38))):
        for t in values:
            refused(lib.lbfgs_train_token_logprobs(rows(dtype=dtype), t, P, P, P, 1 << 30, None), "out of range")
            refused(lib.lbfgs_train_token_logprobs_grad(rows(dtype=dtype), t, P, P, P, None), "out of range")
    refused(lib.lbfgs_train_token_logprobs(None, 1.0, P, P, P, 0, None), "no rows")
    refused(lib.lbfgs_train_token_logprobs(rows(), 1.0, None, P, P, 0, None), "are needed")
    refused(lib.lbfgs_train_token_logprobs(rows(), 1.0, P, None, P, 0, None), "are needed")
    refused(lib.lbfgs_train_token_logprobs_grad(rows(), 1.0, P, P, None, None), "are needed")
    need = lib.lbfgs_train_token_logprobs_workspace(2, 2, 400000)
    assert need > 0 and lib.lbfgs_train_token_logprobs_workspace(2, 100000, 400000) == 0
    refused(lib.lbfgs_train_token_logprobs(rows(dtype=2, vocab=400000), 1.0, P, P, P, need - 1, None), "workspace")
    refused(lib.lbfgs_train_token_logprobs(rows(dtype=2, vocab=400000), 1.0, P, P, None, need, None), "workspace")
    refused(lib.lbfgs_train_token_logprobs(rows(dtype=2, vocab=400000), 1.0, P, P, P + 128, 1 << 30, None), "aligned")
    assert lib.lbfgs_train_token_logprobs(rows(outer=0), 1.0, None, None, None, 0, None) == 0  # no rows: nothing to do


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=4), "element type"), (dict(tokens=-1), "tokens in"), (dict(count=0), "tokens in"), (dict(offset_bits=16), "offsets of 16 bits"),
    (dict(offsets=None, tokens=10, count=4), "no padded batch")])
def test_c_sequences_refusals(lib, kw, text):
    refused(lib.lbfgs_train_preference(seqs(**kw), P, P, 0.1, 0.0, 0, 0, P, P, P, P, 1 << 30, None), text)
    refused(lib.lbfgs_train_policy(seqs(**kw), P, P, P, P, 1, 0.2, 0.2, 0.0, 0, P, P, P, P, P, 1 << 30, None), text)


def test_c_preference_refusals(lib):
    def call(s=None, logps=P, beta=0.1, smoothing=0.0, kind=0, f=P, rewards=P, grad=P, ws=P, size=1 << 30):
        return lib.lbfgs_train_preference(s or seqs(), logps, P, beta, smoothing, kind, 0, f, rewards, grad, ws, size, None)

    refused(call(seqs(count=3)), "no pairs")
    for beta in (0.0, -0.1, math.nan, math.inf):
        refused(call(beta=beta), "beta")
    for e in (-0.1, 0.5, math.nan):
        refused(call(smoothing=e), "label_smoothing")
    refused(call(smoothing=0.1, kind=1), "logistic")
    refused(call(kind=3), "kind")
    for name in ("logps", "f", "rewards", "grad"):
        refused(call(**{name: None}), "are needed")
    assert lib.lbfgs_train_sequences_workspace(10, 4) == 0 and call(seqs(count=3), ws=None, size=0) == ARG
    need = lib.lbfgs_train_sequences_workspace(100000, 4)
    refused(call(seqs(tokens=100000), size=need - 1), "workspace")
    refused(call(seqs(tokens=100000), ws=None), "workspace")
    refused(call(seqs(tokens=100000), ws=P + 8), "aligned")


def test_c_policy_refusals(lib):
    def call(s=None, logps=P, old=P, ref=P, adv=P, per_token=1, low=0.2, high=0.2, kl_coef=0.1, f=P, kl=P, clip=P, grad=P, size=1 << 30):
        return lib.lbfgs_train_policy(s or seqs(), logps, old, ref, adv, per_token, low, high, kl_coef, 0, f, kl, clip, grad, P, size, None)

    for low in (-0.1, 1.1, math.nan):
        refused(call(low=low), "clip_low")
    for high in (-0.1, math.nan):
        refused(call(high=high), "clip_high")
    refused(call(kl_coef=math.inf), "kl_coef")
    refused(call(ref=None), "ref_logps")
    for name in ("logps", "old", "adv", "f", "kl", "clip", "grad"):
        refused(call(**{name: None}), "are needed")
    refused(call(seqs(tokens=100000), size=10), "workspace")


def test_c_orthogonalize_refusals(lib):
    def call(dtype=1, batch=1, m=4, n=4, g=P, out=P, steps=5, abc=directions.COEFFICIENTS, ws=P, size=1 << 40):
        return lib.lbfgs_train_orthogonalize(dtype, batch, m, n, g, out, steps, *abc, ws, size, None)

    for dtype in (0, 4):
        refused(call(dtype=dtype), "element type")
    refused(call(batch=32768), "matrices of")
    refused(call(m=-1), "matrices of")
    refused(call(n=(1 << 20) + 1), "matrices of")
    for steps in (0, 65):
        refused(call(steps=steps), "steps")
    refused(call(abc=(math.nan, 0, 0)), "coefficients")
    refused(call(abc=(4.0, 0.0, 0.0)), "out of range")        # grows by 4 in each of five steps
    refused(call(abc=(-8.0, 0.0, 4000.0)), "out of range")
    refused(call(g=None), "are needed")
    refused(call(ws=None), "workspace")
    refused(call(ws=P + 64), "aligned")
    refused(call(size=lib.lbfgs_train_orthogonalize_workspace(1, 1, 4, 4) - 1), "workspace")
    assert lib.lbfgs_train_orthogonalize_workspace(1, 0, 4, 4) == lib.lbfgs_train_orthogonalize_workspace(0, 1, 4, 4) == 0
    assert call(batch=0, g=None, out=None, ws=None) == 0 and call(m=0, g=None, out=None, ws=None) == 0


def test_the_flag_of_a_wide_gradient(lib):
    assert int(re.search(r"LBFGS_TRAIN_WIDE_GRAD = (\d+)", header()).group(1)) == _train.WIDE_GRAD
    for dtype in (4, -1, 255, 512):
        s = seqs(dtype=dtype | _train.WIDE_GRAD)
        refused(lib.lbfgs_train_preference(s, P, P, 0.1, 0.0, 0, 0, P, P, P, P, 1 << 30, None), "element type")
        refused(lib.lbfgs_train_policy(s, P, P, P, P, 1, 0.2, 0.2, 0.0, 0, P, P, P, P, P, 1 << 30, None), "element type")
    for dtype in (0, 1, 2, 3):  # offered: what is wrong then is something else
        s = seqs(dtype=dtype | _train.WIDE_GRAD)
        refused(lib.lbfgs_train_preference(s, None, P, 0.1, 0.0, 0, 0, P, P, P, P, 1 << 30, None), "are needed")
        refused(lib.lbfgs_train_policy(s, None, P, P, P, 1, 0.2, 0.2, 0.0, 0, P, P, P, P, P, 1 << 30, None), "are needed")
    c = _train.calls()
    for f, n in ((c.preference_wide, 8), (c.policy_wide, 10)):
        with pytest.raises(TypeError, match=f"{n} are taken"):
            f(*[0] * (n - 1))
    x = torch.zeros(2, 8)
    assert c.preference_wide(x, x, None, None, 0.1, 0.0, 0, False) is None and c.policy_wide(x, x, x, None, None, None, 0.2, 0.2, 0.0, 0) is None


# ------------------------------------------------------------------------------------ Python functions
def test_logprobs_refusals(lib):
    x, y = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    for fn in (losses.token_logprobs, losses.token_logprobs_with_lse):
        with pytest.raises(TypeError, match="no CPU fallback"):
            fn(x, y)
        with pytest.raises(TypeError, match="float64, float32"):
            fn(x.long(), y)
        with pytest.raises(TypeError, match="torch tensor"):
            fn([[0.0]], y)
        with pytest.raises(TypeError, match="int64"):
            fn(x, y.int())
        with pytest.raises(ValueError, match="one for each row"):
            fn(x, torch.zeros(3, dtype=torch.int64))
        with pytest.raises(ValueError, match="vocabulary"):
            fn(torch.zeros(2, 0), y)
    lse, g = torch.zeros(2, 2, dtype=torch.float64), torch.zeros(2)
    meta = torch.device("meta")
    with pytest.raises(TypeError, match="no CPU fallback"):
        losses.token_logprobs_grad(x, y, lse, g)
    with pytest.raises(TypeError, match="no CPU fallback"):
        losses.token_logprobs(x.to(meta).requires_grad_(), y.to(meta))


def test_sequence_refusals(lib):
    lp, off = torch.zeros(6), torch.tensor([0, 3, 6])
    calls = [lambda x, **kw: losses.preference(x, **kw), lambda x, **kw: losses.policy(x, x, x, **kw)]
    for call in calls:
        with pytest.raises(TypeError, match="no CPU fallback"):
            call(lp, offsets=off)
        with pytest.raises(TypeError, match="int32 or int64"):
            call(lp, offsets=off.float())
        with pytest.raises(ValueError, match="sequences \\+ 1"):
            call(lp, offsets=off[:1])
        with pytest.raises(ValueError, match="one-dimensional"):
            call(torch.zeros(2, 3), offsets=off)
        with pytest.raises(ValueError, match="padded batch"):
            call(lp)
        with pytest.raises(ValueError, match="padded batch"):
            call(torch.zeros(0, 3))
        with pytest.raises(TypeError, match="mask"):
            call(lp, offsets=off, mask=torch.zeros(6))
        with pytest.raises(ValueError, match="mask"):
            call(lp, offsets=off, mask=torch.zeros(5, dtype=torch.bool))
        with pytest.raises(TypeError, match="float64, float32"):
            call(lp.int(), offsets=off)
    with pytest.raises(ValueError, match="kind"):
        losses.preference(lp, offsets=off, kind="other")
    with pytest.raises(TypeError, match="ref_logps"):
        losses.preference(lp, lp.double(), offsets=off)
    with pytest.raises(ValueError, match="reduction"):
        losses.policy(lp, lp, lp, offsets=off, reduction="sum")
    with pytest.raises(ValueError, match="KL term"):
        losses.policy(lp, lp, lp, offsets=off, kl_coef=0.1)
    with pytest.raises(ValueError, match="old_logps"):
        losses.policy(lp, lp[:5], lp, offsets=off)
    with pytest.raises(ValueError, match="advantages"):
        losses.policy(lp, lp, lp[:2], offsets=off)  # one for each sequence is [2, 1]
    with pytest.raises(TypeError, match="advantages"):
        losses.policy(lp, lp, lp[:2, None].double(), offsets=off)


def test_orthogonalize_refusals(lib):
    with pytest.raises(TypeError, match="no CPU fallback"):
        directions.orthogonalize(torch.zeros(2, 3))
    with pytest.raises(TypeError, match="64 bits"):
        directions.orthogonalize(torch.zeros(2, 3, dtype=torch.float64))
    with pytest.raises(ValueError, match="rows, cols"):
        directions.orthogonalize(torch.zeros(3))
    with pytest.raises(ValueError, match="coefficients"):
        directions.orthogonalize(torch.zeros(2, 3), coefficients=(1.0, 2.0))


def test_the_example_of_a_direction_takes_the_optimisers_gradients(lib):
    """float64, as every gradient that the optimiser has; with one of the CPU what is wrong is the device alone."""
    example = re.search(r"    d = (directions\.orthogonalize\(.*\))  ", directions.__doc__).group(1)
    names = dict(directions=directions, gradient=torch.ones(6, dtype=torch.float64), rows=2, cols=3)
    with pytest.raises(TypeError, match="no CPU fallback"):
        eval(example, names)


def test_what_is_said_of_the_default_coefficients():
    smallest, low, high = re.search(r"below 1/(\d+) of the norm\) into ([0-9.]+) \.\. ([0-9.]+)\.\n", directions.orthogonalize.__doc__).groups()
    s = torch.linspace(1 / int(smallest), 1, 1000001, dtype=torch.float64)
    a, b, c = directions.COEFFICIENTS
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    assert float(low) <= float(s.min()) < float(low) + 0.01 and float(high) - 0.01 < float(s.max()) <= float(high)


def test_views_with_a_sign_to_come_are_refused(lib):
    lazy = torch.view_as_complex(torch.ones(6, 2)).conj().imag
    assert lazy.is_neg()
    off = torch.tensor([0, 2, 6])
    for call in (lambda: losses.token_logprobs(lazy, torch.tensor(0)), lambda: losses.preference(lazy, offsets=off), lambda: losses.preference(torch.ones(6), lazy, offsets=off),
                 lambda: losses.policy(torch.ones(6), torch.ones(6), lazy, offsets=off), lambda: directions.orthogonalize(lazy.view(2, 3))):
        with pytest.raises(TypeError, match="resolve_neg"):
            call()


@pytest.mark.parametrize("value", [1 << 70, 2 ** 64, 2 ** 64 + 5, 1 << 63, -(1 << 63) - 1, -2 ** 64 - 100])
def test_whole_numbers_that_do_not_fit_are_refused(lib, value):
    """Their low bits alone would be another number that is offered: 0, 5, ..."""
    x, y = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: losses.token_logprobs(x, y, ignore_index=value), lambda: losses.token_logprobs(x.clone().requires_grad_(), y, ignore_index=value),
                 lambda: losses.token_logprobs_with_lse(x, y, ignore_index=value), lambda: losses.token_logprobs_with_lse(torch.zeros(2, 9)[:, :8], y, ignore_index=value),
                 lambda: losses.token_logprobs_grad(x, y, torch.zeros(2, 2, dtype=torch.float64), torch.zeros(2), ignore_index=value)):
        with pytest.raises(ValueError, match="ignore_index must fit 64 bits"):
            call()
    for steps in (value, 2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31):
        with pytest.raises(ValueError, match="steps must fit 32 bits"):
            directions.orthogonalize(torch.zeros(2, 3), steps=steps)
    with pytest.raises(TypeError):
        losses.token_logprobs(x, y, ignore_index=1.5)
    with pytest.raises(TypeError):
        directions.orthogonalize(torch.zeros(2, 3), steps=5.5)


def test_forward_mode_derivatives_are_refused(lib):
    """A dual tensor has requires_grad False: taken as it is, its tangent would be lost and read as a derivative of 0."""
    from torch.autograd import forward_ad

    x, y, off = torch.zeros(6), torch.zeros((), dtype=torch.int64), torch.tensor([0, 2, 6])
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones(6))
        view = d.view(2, 3)
        for call in (lambda: losses.token_logprobs(d, y), lambda: losses.token_logprobs_with_lse(d, y), lambda: losses.token_logprobs_grad(d, y, x, x),
                     lambda: losses.preference(d, offsets=off), lambda: losses.preference_loss(view), lambda: losses.preference_loss(x, d, offsets=off),
                     lambda: losses.policy_loss(d, x, x, offsets=off), lambda: losses.policy(x, d, x, offsets=off), lambda: losses.policy(x, x, d, offsets=off),
                     lambda: losses.policy(x, x, x, ref_logps=d, kl_coef=0.1, offsets=off), lambda: directions.orthogonalize(view)):
            with pytest.raises(TypeError, match="forward-mode derivative"):
                call()


def test_native_calls_decline_what_is_not_ordinary(lib):
    """Tensors that are elsewhere, of other types or shapes, or no tensors at all: None, and nothing done."""
    c = _train.calls()
    x, y, g = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    for a in ((x, y, 1.0, -100), (None, y, 1.0, -100), (x, 3, 1.0, -100), (x, y, "1", -100), (x, y, 1.0, 1 << 70), ("x", y, 1, -100)):
        assert c.logprobs(*a) is None
    assert c.logprobs_grad(x, y, torch.zeros(2, 2, dtype=torch.float64), g, 1.0, -100) is None
    for off, mask in ((None, None), (torch.tensor([0, 1]), None), (7, x), ("a", 1)):
        assert c.preference(x, x, off, mask, 0.1, 0.0, 0, False) is None
        assert c.policy(x, x, x, None, off, mask, 0.2, 0.2, 0.0, 0) is None
    assert c.orthogonalize(x, 5, 1.0, 2.0, 3.0) is None and c.orthogonalize(None, 5, 1.0, 2.0, 3.0) is None
    assert c.orthogonalize(x.to_sparse(), 5, 1.0, 2.0, 3.0) is None and c.orthogonalize(torch.zeros(2, 3, device="meta"), 5, 1.0, 2.0, 3.0) is None
    for f, n in ((c.logprobs, 4), (c.logprobs_grad, 6), (c.preference, 8), (c.policy, 10), (c.orthogonalize, 5), (c.bind, 9)):
        for k in (0, n - 1, n + 1):
            with pytest.raises(TypeError, match=f"{n} are taken"):
                f(*[x] * k)


def test_the_native_calls_are_rebuilt_when_sources_or_torch_differ(lib, monkeypatch):
    assert _build.embedded_id(_build.CALLS_LIB, "LBFGS_TRAIN_CALLS_BUILD_ID") == _build.calls_build_id()
    assert _build._torch()[1] == torch.__version__
    before = _build.calls_build_id()
    monkeypatch.setattr(_build, "_torch", lambda: (os.path.dirname(torch.__file__), "0.0"))
    assert _build.calls_build_id() != before
    monkeypatch.setattr(_train, "_CALLS", None)
    with pytest.raises(ImportError, match="build id"):
        _train.calls()
    monkeypatch.setattr(_build, "CALLS_LIB", "/nowhere.so")
    with pytest.raises(ImportError, match="missing"):
        _train.calls()


def test_modules_are_reached_from_the_package():
    assert R.losses is losses and R.directions is directions
