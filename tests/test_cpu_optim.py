"""CPU: argument checks of the AdamW step (C ABI and Python), parameter groups, the 8-bit moment format."""
import ctypes as C

import numpy as np
import pytest
import torch

from helpers import pkg
from optim_ref import M_BASE, V_BASE, code_values, decode, encode


def _desc(L, **kw):
    """A descriptor that passes every check, with fields replaced (the addresses are never used: the calls are refused)."""
    start = (C.c_int32 * 3)(0, 1, 2)
    groups = (L.AdamwGroup * 1)(L.AdamwGroup(1e-3, 0.9, 0.999, 1e-8, 0.01))
    grads = (C.c_void_p * 2)(16, 32)
    d = L.AdamwDesc(state_bits=32, ntensors=2, ngroups=1)
    d.tensors = d.chunks = d.steps = d.coef = d.m = d.v = d.partial = d.norm = 256
    d.chunk_start, d.groups, d.grads = C.addressof(start), C.addressof(groups), C.addressof(grads)
    d.grad_scale = 1.0
    d.keep = (start, groups, grads)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,msg", [
    (dict(state_bits=16), b"state_bits"), (dict(ntensors=0), b"ntensors"), (dict(ngroups=0), b"groups"),
    (dict(ngroups=33), b"groups"), (dict(tensors=None), b"null table"), (dict(grads=None), b"either grads or flat_grad"),
    (dict(flat_grad=64), b"either grads or flat_grad"), (dict(m=None), b"null moments"), (dict(state_bits=8), b"null moments"),
    (dict(m=8), b"aligned"), (dict(max_norm=-1.0), b"max_norm"), (dict(max_norm=float("nan")), b"max_norm"),
    (dict(max_norm=1.0, partial=None), b"partial"), (dict(skip_nonfinite=1, norm=None), b"norm"),
    (dict(grad_scale=float("inf")), b"grad_scale"), (dict(grads=None, flat_grad=64, flat_dtype=5), b"flat_dtype"),
])
def test_step_refusals(kw, msg):
    L = pkg("_lib")
    assert L.lib().srx_adamw_step(C.byref(_desc(L, **kw)), None) == 1
    assert msg in L.lib().srx_last_error(), L.lib().srx_last_error()


def test_step_refuses_bad_tables():
    L = pkg("_lib")
    lib = L.lib()
    assert lib.srx_adamw_step(None, None) == 1 and b"null descriptor" in lib.srx_last_error()
    for start in ((1, 1, 2), (0, 3, 2)):
        arr = (C.c_int32 * 3)(*start)
        assert lib.srx_adamw_step(C.byref(_desc(L, chunk_start=C.addressof(arr))), None) == 1
        assert b"chunk_start" in lib.srx_last_error()
    types = (C.c_uint8 * 2)(1, 7)
    assert lib.srx_adamw_step(C.byref(_desc(L, grad_dtypes=C.addressof(types))), None) == 1
    assert b"gradient dtype 7 of tensor 1" in lib.srx_last_error()
    odd = (C.c_void_p * 2)(16, 34)
    assert lib.srx_adamw_step(C.byref(_desc(L, grads=C.addressof(odd))), None) == 1
    assert b"gradient 1 is not aligned" in lib.srx_last_error()
    for bad in ((float("nan"), .9, .999, 1e-8, 0), (1e-3, 1.0, .999, 1e-8, 0), (1e-3, .9, -.1, 1e-8, 0), (1e-3, .9, .999, -1, 0),
                (1e-3, .9, .999, 1e-8, float("inf"))):
        g = (L.AdamwGroup * 1)(L.AdamwGroup(*bad))
        assert lib.srx_adamw_step(C.byref(_desc(L, groups=C.addressof(g))), None) == 1
        assert b"hyper-parameters in group 0" in lib.srx_last_error()


def test_moment_conversion_refusals():
    L = pkg("_lib")
    lib = L.lib()
    assert lib.srx_adamw_moments_to8(None, 16, 16, 16, 16, 16, 1, None) == 1 and b"null" in lib.srx_last_error()
    assert lib.srx_adamw_moments_from8(16, 16, 16, 16, 16, 24, 1, None) == 1 and b"aligned" in lib.srx_last_error()
    assert lib.srx_adamw_moments_from8(16, 16, 16, 16, 16, 16, -1, None) == 1 and b"nblocks" in lib.srx_last_error()
    assert lib.srx_adamw_moments_to8(None, None, None, None, None, None, 0, None) == 0      # nothing to do


def test_optimizer_refuses_what_it_cannot_run():
    O = pkg("optim")
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        O.AdamW([p])
    with pytest.raises(ValueError, match="no parameters"):
        O.AdamW([])
    with pytest.raises(ValueError, match="no parameters"):
        O.AdamW([{"params": []}])
    with pytest.raises(TypeError, match="not both"):
        O.AdamW([p, {"params": [p]}])
    with pytest.raises(ValueError, match="state_bits"):
        O.AdamW([p], state_bits=4)
    with pytest.raises(ValueError, match="max_grad_norm"):
        O.AdamW([p], max_grad_norm=0.0)
    with pytest.raises(ValueError, match="unknown keys"):
        O.AdamW([{"params": [p], "momentum": 0.9}])
    with pytest.raises(ValueError, match="at most 32"):
        O.AdamW([{"params": [p]}] * 33)
    with pytest.raises(TypeError, match="not a tensor"):
        O.AdamW([None])


def test_decay_groups():
    O, G = pkg("optim"), pkg("esrgan.generator")
    g = G.GeneratorESRGAN(num_features=16, num_blocks=1)
    groups = O.decay_groups(g, 0.05)
    assert [x["weight_decay"] for x in groups] == [0.05, 0.0]
    assert all(p.dim() == 4 for p in groups[0]["params"]) and all(p.dim() == 1 for p in groups[1]["params"])
    assert {id(p) for x in groups for p in x["params"]} == {id(p) for p in g.parameters()}
    g.conv_first.bias.requires_grad_(False)
    assert len(O.decay_groups(g)[1]["params"]) == len(groups[1]["params"]) - 1


def test_code_table_of_the_8_bit_moments():
    """The values that codes stand for are the floats with 3 mantissa bits from 1 down; every value rounds to the nearest of
    them (half a step: 1/16 of its power of two at most), ties to the even code, and decoding then encoding is the identity."""
    for base, n, lowest in ((M_BASE, 127, 1.25 * 2.0 ** -16), (V_BASE, 255, 1.25 * 2.0 ** -32)):
        tab = code_values(base, n)
        assert tab[0] == 0 and tab[1] == lowest and tab[n] == 1.0 and np.all(np.diff(tab) > 0)
        assert np.array_equal(encode(tab, base, 0), np.arange(n + 1))
        rng = np.random.default_rng(0)
        t = np.exp2(rng.uniform(np.log2(lowest), 0, 20000)).astype(np.float32)
        got = tab[encode(t, base, 0)].astype(np.float64)
        best = tab[np.abs(t[:, None].astype(np.float64) - tab[None, :]).argmin(1)]
        mid = np.abs(np.abs(t - got) - np.abs(t - best)) == 0
        assert mid.all()
        assert np.abs(got / t - 1).max() <= 1 / 16
        assert list(encode(np.float32([0, lowest / 4, 1e-30]), base, 0)) == [0, 0, 0]
        assert list(encode(np.float32([0, lowest / 4, 1e-30]), base, 1)) == [0, 1, 1]
    x = decode(np.uint8([0, 1, 127, 128 + 127]), np.float32(2.0), M_BASE, True)
    assert list(x) == [0, 2.5 * 2.0 ** -16, 2.0, -2.0]
