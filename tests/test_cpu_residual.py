"""CPU: argument checks of the norms around a residual branch (C ABI and Python)."""
import ctypes as C

import pytest
import torch

from helpers import pkg


def _desc(L, **kw):
    d = L.ResnormDesc(dtype=1, layout=0, B=2, C=64, P=16, post_kind=1, pre_kind=2, gate_mode=1, scale=1.0, post_eps=1e-6, pre_eps=1e-6)
    for n in ("x", "f", "y", "h", "gate"):
        setattr(d, n, 256)
    for n in ("x", "f", "y", "h", "dy", "dh", "dx", "df", "gate", "dgate"):
        setattr(d, n + "_stride", 1024)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


REFUSED = [
    (dict(dtype=3), b"dtype"), (dict(layout=2), b"layout"), (dict(C=0), b"sizes"), (dict(B=-1), b"sizes"), (dict(P=-1), b"sizes"),
    (dict(C=1025), b"at most 1024"), (dict(layout=1, C=8193), b"at most 8192"), (dict(post_kind=3), b"norm kind"),
    (dict(pre_kind=-1), b"norm kind"), (dict(gate_mode=4), b"gate mode"), (dict(gate_act=2), b"gate mode"),
    (dict(pre_eps=0.0), b"eps"), (dict(post_eps=float("nan")), b"eps"), (dict(f=None), b"without a branch"),
    (dict(f=None, post_kind=0, gate_mode=0, pre_kind=0), b"neither"), (dict(gate=None), b"null gate"),
    (dict(x=258), b"aligned"), (dict(y_stride=1023), b"stride 1023"), (dict(x_stride=-1), b"stride"),
]


@pytest.mark.parametrize("kw,msg", REFUSED + [(dict(x=None), b"null tensor"), (dict(y=None), b"null tensor"), (dict(h=None), b"null tensor")])
def test_forward_refusals(kw, msg):
    L = pkg("_lib")
    assert L.lib().srx_resnorm_forward(C.byref(_desc(L, **kw)), None) == 1
    assert msg in L.lib().srx_last_error(), L.lib().srx_last_error()


@pytest.mark.parametrize("kw,msg", REFUSED + [(dict(), b"neither dy nor dh"), (dict(dh=256, x=None), b"and x"),
                                              (dict(dh=256, pre_kind=0), b"needs the norm"), (dict(dy=256), b"workspace"),
                                              (dict(dy=256, ws=256, dx=256, dx_stride=5), b"stride 5")])
def test_backward_refusals(kw, msg):
    L = pkg("_lib")
    assert L.lib().srx_resnorm_backward(C.byref(_desc(L, **kw)), None) == 1
    assert msg in L.lib().srx_last_error(), L.lib().srx_last_error()


def test_null_descriptors_and_workspace():
    L = pkg("_lib")
    lib = L.lib()
    assert lib.srx_resnorm_forward(None, None) == 1 and b"null descriptor" in lib.srx_last_error()
    assert lib.srx_resnorm_backward(None, None) == 1 and b"null descriptor" in lib.srx_last_error()
    assert lib.srx_resnorm_ws_floats(None) == -1 and lib.srx_resnorm_ws_floats(C.byref(_desc(L, C=0))) == -1
    assert lib.srx_resnorm_ws_floats(C.byref(_desc(L))) >= 4 * 64
    assert lib.srx_resnorm_forward(C.byref(_desc(L, B=0)), None) == 0          # nothing to do


def test_sizes_at_the_limits():
    L = pkg("_lib")
    lib = L.lib()
    far = {n + "_stride": 1 << 62 for n in ("x", "f", "y", "h", "dy", "dh", "dx", "df", "gate", "dgate")}
    floats = lambda **kw: lib.srx_resnorm_ws_floats(C.byref(_desc(L, **far, **kw)))  # noqa: E731
    # images of 2^30 and more; rows without a gate for each image are counted together
    assert floats(B=(1 << 30) + 1) == -1 and b"images" in lib.srx_last_error()
    assert floats(B=(1 << 30) + 1, layout=1, gate_mode=2) == -1 and floats(B=(1 << 31) - 1, layout=1) > 0 and floats(B=(1 << 31) - 1, P=1) > 0
    assert floats(B=1 << 30, layout=1, gate_mode=2, P=1) > 2 * 64 * (1 << 30)
    # an image of 4 GB: from 65 channels on
    assert floats(C=65, P=1 << 25) == -1 and b"4 GB" in lib.srx_last_error()
    assert floats(C=64, P=(1 << 31) - 1) > 0 and floats(C=1024, P=(1 << 20) - 1) > 0 and floats(C=1024, P=1 << 20) == -1
    # the workspace does not grow with the pixels, nor with more images than run at once, but with their gates
    assert floats(P=1 << 20) == floats(P=1 << 24)
    assert floats(B=64, P=1 << 10) <= 2 * 64 * 2 * 1024 + 1


def test_workspace_does_not_go_by_addresses():
    """Asked before the tensors are there, with weights or without, the size is enough for every form of the call."""
    L = pkg("_lib")
    lib = L.lib()
    far = {n + "_stride": 1 << 62 for n in ("x", "f", "y", "h", "dy", "dh", "dx", "df", "gate", "dgate")}
    for layout in (0, 1):
        for c in (1, 5, 8, 24, 64, 99, 300, 520, 1000):
            for b, p in ((1, 64), (16, 4096), (300, 1000), (3, 1), (2, 100000)):
                for gate_mode in (0, 1, 2, 3):
                    for kind in (1, 2):
                        base = dict(far, layout=layout, C=c, B=b, P=p, gate_mode=gate_mode, post_kind=kind, pre_kind=kind, dtype=0)
                        want = lib.srx_resnorm_ws_floats(C.byref(_desc(L, **base)))
                        for more in (dict(b_post=256), dict(b_pre=256, db_pre=256), dict(x=None, y=None, h=None), dict(dy=256, dh=256, dx=256, df=256),
                                     dict(pre_kind=0), dict(post_kind=0)):
                            assert lib.srx_resnorm_ws_floats(C.byref(_desc(L, **{**base, **more}))) == want > 0


def test_python_refusals():
    R = pkg("residual")
    x = torch.zeros(2, 8, 4, 4)
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        R.channel_norm(x, R.NormSpec("rms"))
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        R.gated_residual(x, x)
    for bad in (1e-38, 0.0, -1.0, float("nan"), float("inf"), 1e39):
        with pytest.raises(ValueError, match="eps"):
            R.channel_norm(x, R.NormSpec("rms", eps=bad))
    for bad in (float("nan"), float("inf"), -1e39):
        with pytest.raises(ValueError, match="scale"):
            R.gated_residual(x, x, scale=bad)
    with pytest.raises(ValueError, match="kind"):
        R.ChannelNorm(8, "batch")
    with pytest.raises(ValueError, match="no blocks"):
        R.GatedResidualStack([], 8)
    with pytest.raises(ValueError, match="gate must be"):
        R.GatedResidualStack([torch.nn.Identity()], 8, gate="pixel")
    with pytest.raises(ValueError, match="gate_act"):
        R.GatedResidualStack([torch.nn.Identity()], 8, gate_act="tanh")


def test_modules_parameters():
    R, O = pkg("residual"), pkg("optim")
    n = R.ChannelNorm(8)
    assert n.bias is None and n.spec.kind == "rms" and n.spec.weight is n.weight
    assert R.ChannelNorm(8, "layer").bias is not None and R.ChannelNorm(8, "layer", bias=False).bias is None
    s = R.GatedResidualStack([torch.nn.Conv2d(8, 8, 3, padding=1) for _ in range(2)], 8, "layer", gate_init=0.5)
    names = [k for k, _ in s.named_parameters()]
    assert names == [f"blocks.{i}.{w}" for i in range(2) for w in ("weight", "bias")] + \
        [f"{p}.{i}.{w}" for p in ("pre", "post") for i in range(2) for w in ("weight", "bias")] + ["gates.0", "gates.1"]
    assert [len(g["params"]) for g in O.decay_groups(s)] == [2, 12]          # norms and gates do not decay
    with pytest.raises(ValueError, match="gates"):
        s(torch.zeros(1, 8, 4, 4), [torch.zeros(8)] * 2)
