"""The block-scaled operators and the rms norm seen from between autograd and the
kernels: fake tensors, dispatch modes, tracing. No kernel may run there."""

import collections.abc
import os

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from vilbert_multi_task_amd.ops import functional as F_ops

gpu = pytest.mark.gpu
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
EPS = 1e-6

if not F_ops.extension_available():
    pytest.skip("the extension is not built", allow_module_level=True)


def _args(device, rows=(3, 5), k=200, n=130, scales=BF):
    x = torch.ones(*rows, k, device=device)
    w, b = torch.ones(k, device=device), torch.zeros(k, device=device)
    wide = torch.ones(n, k, device=device)
    x8 = torch.ones(*rows, k, device=device).to(E4)
    xs = torch.ones(*rows, -(-k // 128), device=device, dtype=scales)
    w8 = torch.ones(n, k, device=device).to(E4)
    ws = torch.ones(-(-n // 128), -(-k // 128), device=device, dtype=scales)
    return x, w, b, wide, (x8, xs, w8, ws)


def _all(device, scales=BF):
    """Every entry point's results by name."""
    x, w, b, wide, p = _args(device, scales=scales)
    t = x.clone()
    return {
        "rms": F_ops.rms_norm(x, w, EPS),
        "rms_res": F_ops.rms_norm(x, w, EPS, residual=t),
        "rms8": F_ops.rms_norm_fp8_block(x, w, EPS, scale_dtype=scales),
        "rms8_res": F_ops.rms_norm_fp8_block(x, w, EPS, residual=t, scale_dtype=scales),
        "layer8": F_ops.layer_norm_fp8_block(x, w, b, EPS, residual=t, scale_dtype=scales),
        "quant": F_ops.quantize_fp8_block(x, scale_dtype=scales),
        "weight": F_ops.quantize_fp8_block_weight(wide, scale_dtype=scales),
        "linear": F_ops.fp8_block_linear(*p, gelu=True),
        "linear_f32": F_ops.fp8_block_linear(*p, out_dtype=F32),
        "linear8": F_ops.fp8_block_linear_fp8(*p),
    }


def _leaves(v):
    return [v] if isinstance(v, torch.Tensor) else list(v)


@pytest.mark.parametrize("scales", [BF, F32])
def test_fake_tensors_come_back_with_their_sizes(scales):
    real = _all("cpu", scales)
    with FakeTensorMode():
        fake = _all("cuda", scales)
    for name, want in real.items():
        got = _leaves(fake[name])
        assert len(got) == len(_leaves(want))
        for g, t in zip(got, _leaves(want)):
            assert isinstance(g, FakeTensor) and g.device.type == "cuda", name
            assert g.shape == t.shape and g.dtype == t.dtype, name
        if got[0].dtype == E4:  # rows at multiples of 16 bytes, as the kernels lay them out
            assert got[0].stride(-2) % 16 == 0


class _Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.add(func.name())
        return func(*args, **(kwargs or {}))


def test_modes_see_every_operator():
    with FakeTensorMode(), _Seen() as seen:
        with torch.no_grad():
            _all("cuda")
        x, w, *_ = _args("cuda")
        y, t = F_ops.rms_norm(x.clone().requires_grad_(), w, EPS, residual=x)
        assert y.requires_grad and t.requires_grad
        rstd = torch.ones(15, device="cuda")
        gx, gw = F_ops._require_extension().rms_bwd(x, None, x, rstd, w)
        assert gx.shape == x.shape and gw.shape == w.shape
    assert {
        "vilbert_amd::" + name for name in (
            "rms_norm", "rms_norm_residual", "rms_fwd_train", "rms_bwd", "rms_norm_fp8_block",
            "layer_norm_fp8_block", "quantize_fp8_block", "quantize_fp8_block_weight",
            "fp8_block_linear", "fp8_block_linear_fp8")
    } <= seen.names


@gpu  # torch's engine asks for a device, also where all tensors are fake
@pytest.mark.parametrize("with_res", [False, True])
def test_fake_gradients(with_res):
    with FakeTensorMode():
        for dtype in (BF, F32):
            x, r = (torch.ones(4, 6, 96, device="cuda", dtype=dtype, requires_grad=True) for _ in range(2))
            w = torch.ones(96, device="cuda", dtype=dtype, requires_grad=True)
            y = F_ops.rms_norm(x, w, EPS, residual=r if with_res else None)
            leaves = (x, w, r) if with_res else (x, w)
            grads = torch.autograd.grad(sum(t.sum() for t in _leaves(y)), leaves)
            for g, t in zip(grads, leaves):
                assert g.shape == t.shape and g.dtype == t.dtype and g.device == t.device


def test_tracing_with_symbolic_sizes():
    def step(*tensors):  # moved here, where moving is traced too
        x, w, w8, ws = (t.to("cuda") for t in tensors)
        q, s = F_ops.rms_norm_fp8_block(x, w, EPS)
        q, s = F_ops.fp8_block_linear_fp8(q, s, w8, ws, gelu=True)
        return q, s

    x, w, _, _, (_, _, w8, ws) = _args("cpu", rows=(7,))
    with torch.no_grad():
        traced = make_fx(step, tracing_mode="symbolic")(x, w, w8, ws)
    called = [n.target.name() for n in traced.graph.nodes if isinstance(n.target, torch._ops.OpOverload)]
    assert "vilbert_amd::rms_norm_fp8_block" in called and "vilbert_amd::fp8_block_linear_fp8" in called
    sizes = next(n for n in traced.graph.nodes if n.op == "placeholder").meta["val"].shape
    assert not isinstance(sizes[0], int)


def test_refusals_of_fake_tensors():
    with FakeTensorMode():
        x, w, b, wide, p = _args("cuda")
        with pytest.raises(RuntimeError, match="rms_norm"):
            F_ops.rms_norm(x, w[:7], EPS)
        for t in (x.half(), x.double()):  # 64 bits: the plain form alone
            with pytest.raises(RuntimeError, match="quantize_fp8_block"):
                F_ops.quantize_fp8_block(t)
            for res in (None, t):
                with pytest.raises(RuntimeError, match="rms_norm"):
                    F_ops.rms_norm(t, w.to(t.dtype), EPS, residual=res)
        with pytest.raises(RuntimeError, match="fp8_block_linear"):
            F_ops.fp8_block_linear(*p[:3], p[3][:1])
        with pytest.raises(RuntimeError, match="no gradient"):
            F_ops.quantize_fp8_block(x.requires_grad_())


def _calls_with_tangents(device):
    x, w, b, wide, p = _args(device)
    one = torch.ones_like

    def dual(t):
        return fwAD.make_dual(t, one(t))

    d, dw = dual(x), dual(w)
    bias = dual(torch.zeros(130, device=device))
    return x, d, {
        "rms_norm_fp8_block": [
            lambda: F_ops.rms_norm_fp8_block(d, w, EPS), lambda: F_ops.rms_norm_fp8_block(x, dw, EPS),
            lambda: F_ops.rms_norm_fp8_block(x, w, EPS, residual=d)],
        "layer_norm_fp8_block": [
            lambda: F_ops.layer_norm_fp8_block(d, w, b, EPS), lambda: F_ops.layer_norm_fp8_block(x, w, dw, EPS)],
        "quantize_fp8_block": [lambda: F_ops.quantize_fp8_block(d)],
        "quantize_fp8_block_weight": [lambda: F_ops.quantize_fp8_block_weight(dual(wide))],
        "fp8_block_linear": [lambda: F_ops.fp8_block_linear(*p, bias)],
        "fp8_block_linear_fp8": [
            lambda: F_ops.fp8_block_linear_fp8(*p, bias),
            lambda: F_ops.fp8_block_linear_fp8(p[0], dual(p[1]), *p[2:])],
    }


def _refuses_tangents(calls):
    for name, fs in calls.items():
        for f in fs:
            for grad in (True, False):  # no_grad is about the backward pass
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match=name + " has no forward-mode"):
                    f()


def test_tangents_are_refused_not_dropped():
    with fwAD.dual_level():
        x, d, calls = _calls_with_tangents("cpu")
        _refuses_tangents(calls)
        # the plain norm has its derivative
        w = torch.ones(200)
        assert fwAD.unpack_dual(F_ops.rms_norm(d, w, EPS)).tangent is not None
    with FakeTensorMode(), fwAD.dual_level():
        x, d, calls = _calls_with_tangents("cuda")
        _refuses_tangents(calls)
        w = torch.ones(200, device="cuda")
        dw = fwAD.make_dual(w, torch.ones_like(w))
        calls = {"rms_norm": [
            lambda: F_ops.rms_norm(d, w, EPS), lambda: F_ops.rms_norm(x, dw, EPS),
            lambda: F_ops.rms_norm(x, w, EPS, residual=d), lambda: F_ops.rms_norm(d, w, EPS, residual=x)]}
        _refuses_tangents(calls)
        assert F_ops.rms_norm(x, w, EPS).shape == x.shape  # without one, as ever


@gpu
def test_tangents_are_refused_on_the_gpu():
    with fwAD.dual_level():
        x, d, calls = _calls_with_tangents("cuda")
        w = torch.ones(200, device="cuda")
        calls["rms_norm"] = [lambda: F_ops.rms_norm(d, w, EPS), lambda: F_ops.rms_norm(x, w, EPS, residual=d)]
        _refuses_tangents(calls)


@gpu
@pytest.mark.parametrize("scales", [BF, F32])
def test_fake_and_real_agree(scales):
    real = _all("cuda", scales)
    with FakeTensorMode():
        fake = _all("cuda", scales)
    for name, want in real.items():
        for g, t in zip(_leaves(fake[name]), _leaves(want)):
            assert g.shape == t.shape and g.dtype == t.dtype and g.stride() == t.stride(), name


@gpu
def test_modes_see_the_kernels_calls():
    with _Seen() as seen:
        got = _all("cuda")
    want = _all("cuda")
    assert "vilbert_amd::quantize_fp8_block" in seen.names and "vilbert_amd::rms_norm" in seen.names
    for name in want:
        for g, t in zip(_leaves(got[name]), _leaves(want[name])):
            assert torch.equal(g.float(), t.float()), name


@gpu
def test_compiled_training_step_gives_the_same_bits():
    x, r = (torch.randn(40, 300, generator=torch.Generator().manual_seed(s)).cuda() for s in (1, 2))
    w = torch.linspace(0.5, 1.5, 300, device="cuda")

    def step(x, w, r):
        y, t = F_ops.rms_norm(x, w, EPS, residual=r)
        return (y * y).sum() + t.sum()

    results = []
    for f in (step, torch.compile(step, backend="aot_eager")):
        leaves = [t.clone().requires_grad_() for t in (x, w, r)]
        f(*leaves).backward()
        results.append([t.grad for t in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@gpu
def test_backward_operator_checks_what_it_is_given():
    ext = F_ops._require_extension()
    t, w = torch.ones(4, 32, device="cuda"), torch.ones(32, device="cuda")
    rstd = torch.ones(4, device="cuda")
    for bad in (
        (t[:3], None, t, rstd, w), (t, t[:3], t, rstd, w), (t, None, t, rstd[:3], w),
        (t, None, t, rstd.double(), w), (t, None, t, rstd, w[:31]), (t.to(BF), None, t, rstd, w),
        (t, None, t, rstd.cpu(), w), (t, None, t, torch.ones(8, device="cuda")[::2], w),
    ):
        with pytest.raises(RuntimeError, match="rms_bwd"):
            ext.rms_bwd(*bad)


class _Environ(collections.abc.MutableMapping):
    """An environment by its public interface alone."""

    def __init__(self, values):
        self._values = dict(values)

    def __getitem__(self, name):
        return self._values[name]

    def __setitem__(self, name, value):
        self._values[name] = value

    def __delitem__(self, name):
        del self._values[name]

    def __iter__(self):
        return iter(self._values)

    def __len__(self):
        return len(self._values)


def test_switches_are_read_as_they_are_at_the_call(monkeypatch):
    env = _Environ(os.environ)
    monkeypatch.setattr(os, "environ", env)
    with FakeTensorMode(), torch.no_grad(), _Seen() as seen:
        x, w, b, wide, p = _args("cuda")
        for name, op, call in (
            ("VILBERT_AMD_FORCE_EAGER", "rms_norm", lambda: F_ops.rms_norm(x, w, EPS)),
            ("VILBERT_AMD_FORCE_EAGER", "quantize_fp8_block", lambda: F_ops.quantize_fp8_block(x)),
            ("VILBERT_AMD_FORCE_EAGER", "fp8_block_linear", lambda: F_ops.fp8_block_linear(*p)),
            ("VILBERT_AMD_EAGER_BWD", "rms_norm", lambda: torch.enable_grad()(F_ops.rms_norm)(x, w, EPS)),
        ):
            for value, own in ((None, True), ("1", False), ("0", True)):
                env.pop(name, None)
                if value is not None:
                    env[name] = value
                seen.names.clear()
                call()
                assert ("vilbert_amd::" + op in seen.names) == own, (name, value, op)
            env.pop(name)


@gpu
def test_compiled_whole():
    """Nothing in the entry points breaks a compiled graph."""
    x, w, _, _, p = _args("cuda")

    def step(x, w, *p):
        q, s = F_ops.rms_norm_fp8_block(x, w, EPS)
        y = F_ops.rms_norm(x, w, EPS)
        return q.float(), s, y, F_ops.fp8_block_linear(q, s, p[2], p[3], gelu=True), *F_ops.quantize_fp8_block(y)

    with torch.no_grad():
        want = step(x, w, *p)
        got = torch.compile(step, backend="aot_eager", fullgraph=True)(x, w, *p)
    for g, t in zip(got, want):
        assert g.dtype == t.dtype and torch.equal(g.float(), t.float())
