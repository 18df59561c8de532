"""CPU: calls of the residual norms and the AdamW step that are refused before a device is asked for."""
import ctypes as C

import pytest
import torch

from helpers import pkg


def R():
    return pkg("residual")


def test_forward_mode_differentiation_is_refused():
    """A tangent, with a leaf that requires a gradient beside it or without, in every place that it can come in by."""
    import torch.autograd.forward_ad as fw
    plain, w = torch.randn(2, 8, 4), torch.ones(8)
    spec = lambda w_, b=None: R().NormSpec("layer", w_, b)  # noqa: E731
    for grad in (False, True):
        x = plain.clone().requires_grad_(grad)
        with fw.dual_level():
            dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
            for call in (lambda: R().channel_norm(dual(x), spec(w)), lambda: R().channel_norm(x, spec(dual(w))),
                         lambda: R().channel_norm(x, spec(w, dual(w))), lambda: R().gated_residual(x, dual(x)),
                         lambda: R().gated_residual(x, x, gate=dual(w)), lambda: R().gated_residual(x, x, post=spec(dual(w))),
                         lambda: R().gated_residual(x, x, pre=spec(w, dual(w)))):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
    for transform in (lambda f: torch.func.jvp(f, (plain,), (plain,)), lambda f: torch.func.vmap(f)(plain[None]), lambda f: torch.func.grad(lambda t: f(t).sum())(plain)):
        with pytest.raises(RuntimeError):
            transform(lambda t: R().channel_norm(t, spec(w)))


def test_tracing_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = torch.randn(2, 8, 4), torch.ones(8)
    for call in (lambda t: R().channel_norm(t, R().NormSpec("rms", w)), lambda t: R().gated_residual(t, t, gate=w)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, x)
        for how in ({}, {"pre_dispatch": True}):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(call, **how)(x)
        with pytest.raises(RuntimeError, match="ROCm GPU only"):          # not traced: the next question
            call(x)


def test_a_traced_step_is_refused():
    import numpy as np
    from torch.fx.experimental.proxy_tensor import make_fx
    gather = pkg("_lib").host().gather
    lists = lambda t: gather([t], [t], np.zeros(2, np.uint64), np.zeros(1, np.uint64), np.zeros(1, np.uint8), -1)  # noqa: E731

    def call(t):
        lists(t)
        return t * 2
    for trace in (lambda: torch.jit.trace(call, torch.ones(4)), lambda: make_fx(call)(torch.ones(4))):
        with pytest.raises(RuntimeError, match="AdamW.step cannot be traced"):
            trace()
    lists(torch.ones(4))
