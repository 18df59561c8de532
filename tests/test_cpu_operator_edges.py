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


def test_workspace_is_asked_for_before_there_are_tensors():
    """The size for a descriptor of types, sizes and kinds alone is the size for the same call with its tensors, and sizes are still refused."""
    L = pkg("_lib")
    lib = L.lib()
    names = ("x", "f", "y", "h", "dy", "dh", "dx", "df", "gate", "dgate")
    for layout in (0, 1):
        for c, b, p in ((1, 1, 64), (24, 300, 1000), (64, 16, 4096), (300, 3, 1), (1000, 2, 4000), (64, 1, 1)):
            for gate_mode in (0, 1, 2, 3):
                for post, pre in ((1, 2), (2, 0), (0, 1), (0, 0)):
                    form = dict(dtype=0, layout=layout, C=c, B=b, P=p, gate_mode=gate_mode, post_kind=post, pre_kind=pre, post_eps=1e-6, pre_eps=1e-6)
                    bare = lib.srx_resnorm_ws_floats(C.byref(L.ResnormDesc(**form)))
                    there = {n: 256 for n in names}
                    full = lib.srx_resnorm_ws_floats(C.byref(L.ResnormDesc(**form, **there, **{n + "_stride": 1 << 62 for n in names}, b_post=256, db_pre=256)))
                    assert bare == full > 0, (form, lib.srx_last_error())
                    # an address without its stride, and one that a tensor could not have
                    assert lib.srx_resnorm_ws_floats(C.byref(L.ResnormDesc(**form, x=257, f=3, dx=256))) == bare
    for bad in (dict(C=0), dict(B=-1), dict(gate_mode=7), dict(pre_kind=1, pre_eps=0.0), dict(dtype=9), dict(layout=0, C=65, P=1 << 25),
                dict(gate_mode=2, B=(1 << 30) + 1)):
        assert lib.srx_resnorm_ws_floats(C.byref(L.ResnormDesc(**{**dict(dtype=0, layout=1, C=8, B=2, P=3), **bad}))) == -1, bad


def test_a_flat_gradient_off_its_alignment_is_refused():
    L = pkg("_lib")
    start = (C.c_int32 * 2)(0, 1)
    groups = (L.AdamwGroup * 1)(L.AdamwGroup(1e-3, 0.9, 0.999, 1e-8, 0.01))
    for dtype, address in ((L.F32, 66), (L.F32, 65), (L.BF16, 65)):
        d = L.AdamwDesc(state_bits=32, ntensors=1, ngroups=1, chunk_start=C.addressof(start), groups=C.addressof(groups), flat_grad=address,
                        flat_dtype=dtype, tensors=256, chunks=256, steps=256, coef=256, m=256, v=256, grad_scale=1.0)
        assert L.lib().srx_adamw_step(C.byref(d), None) == 1 and b"flat_grad is not aligned" in L.lib().srx_last_error()


def test_rounding_is_checked():
    L, p = pkg("_lib"), torch.zeros(4)
    with pytest.raises(ValueError, match="rounding must be"):
        pkg("optim").AdamW([p], state_bits=8, rounding="up")
    with pytest.raises(ValueError, match="32-bit moments"):
        pkg("optim").AdamW([p], rounding="random")
    for bits, rounding in ((32, 1), (8, 2), (8, -1)):
        assert L.lib().srx_adamw_step(C.byref(L.AdamwDesc(state_bits=bits, ntensors=1, ngroups=1, rounding=rounding)), None) == 1
        assert b"rounding" in L.lib().srx_last_error()


def test_random_bits_of_the_rounding():
    """Uniform and uncorrelated along what they depend on.  2^16 words: a mean of 2^16 uniform values is within 5 standard deviations,
    5 sqrt(1 / 12 / 2^16) = 0.0057, of 1/2, a correlation within 5 / 2^8 = 0.02 of 0, the largest distance between the distributions
    (Kolmogorov) under 2 / 2^8; over 4000 steps of one quad 0.023, 0.08 and 2 / 63."""
    import numpy as np
    from rounding_ref import word
    quads = np.arange(1 << 16, dtype=np.uint64)
    corr = lambda a, b: abs(np.corrcoef(a, b)[0, 1])  # noqa: E731
    for first in (0, 1 << 31, (1 << 33) + 5):
        q = quads + np.uint64(first)
        for step, salt in ((1, 0), (2, 3), (100000, 2)):
            w = word(q, step, salt) / 2.0 ** 32
            low = (word(q, step, salt) & np.uint32(0xFFFF)) / 2.0 ** 16
            assert abs(w.mean() - 0.5) < 0.0057 and abs(low.mean() - 0.5) < 0.0057
            assert np.abs(np.sort(w) - (np.arange(1 << 16) + 0.5) / (1 << 16)).max() < 2 / 256
            for other in (word(q, step + 1, salt), word(q, step, salt ^ 1), word(q, step, salt ^ 2), word(q + np.uint64(1), step, salt), word(q + np.uint64(64), step, salt)):
                assert corr(w, other) < 0.02
            assert corr(w, low) < 0.02
    for quad in (0, 1, 77, (1 << 33) + 5):
        w = np.array([word(np.array([quad]), t, 2)[0] for t in range(1, 4001)]) / 2.0 ** 32
        assert abs(w.mean() - 0.5) < 0.023 and corr(w[1:], w[:-1]) < 0.08 and np.abs(np.sort(w) - (np.arange(4000) + 0.5) / 4000).max() < 2 / 63


@pytest.mark.parametrize("levels", ["constant", "falling", "rising", "spike"])
def test_second_moments_of_8_bits_over_thousands_of_steps(levels):
    """v in 8 bits against v in 64 over 5000 steps, one value of each block held at 10.

    At random: each rounding has the value as its mean, so the ratio's mean over n = 16 * 255 values is 1; its spread is
    stationary, d^2 p / (2 (1 - b2)) = 0.05 with d = 0.09 between codes and p = E|g^2 / v - 1| (1 - b2) / d of the steps on which a
    code changes, up to 0.5 where v falls from far above: |mean - 1| < 5 * 0.55 / sqrt(n) = 0.043.  To nearest: what include/srx.h says of it."""
    import numpy as np
    from optim_ref import V_BASE, from8, to8
    from rounding_ref import to8_random
    level = {"constant": lambda t: 1.0, "falling": lambda t: 1.0 if t < 1000 else 0.1, "rising": lambda t: 1.0 if t < 1000 else 3.0,
             "spike": lambda t: 100.0 if t < 5 else 1.0}[levels]
    b2, n, rng = 0.999, 256 * 16, np.random.default_rng(0)
    exact, near, rand = np.zeros(n), np.zeros(n, np.float32), np.zeros(n, np.float32)
    rest = np.arange(n) % 256 > 0
    for t in range(1, 5001):
        g = rng.standard_normal(n).astype(np.float32) * np.float32(level(t))
        if levels != "spike":
            g[~rest] = 10.0
        exact = b2 * exact + (1 - b2) * g.astype(np.float64) ** 2
        new = lambda v: v * np.float32(b2) + (g * g) * np.float32(1 - b2)  # noqa: E731
        near = from8(*to8(new(near), V_BASE, 1, False), V_BASE, False)
        rand = from8(*to8_random(new(rand), V_BASE, 1, False, 0, t), V_BASE, False)
        if t % 1000 == 0:
            assert abs((rand / exact)[rest].mean() - 1) < 0.043, t
    off = np.median((near / exact)[rest])
    assert {"constant": 1.0 < off < 2, "falling": 60 < off < 76, "rising": 0.25 < off < 0.4, "spike": 0.2 < off < 0.5}[levels]
