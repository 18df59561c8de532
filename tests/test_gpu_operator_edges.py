"""GPU: unusual calls of the residual norms and the AdamW step that the documentation allows, or that are refused: what autograd is
told of a step, views with the negative bit, forward-mode differentiation and tracing, captures beside living graphs, parameters
that move under a captured step, states that are refused, second moments below the normal numbers, 8-bit moments over thousands of steps."""
import pytest
import torch

from helpers import pkg

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def R():
    return pkg("residual")


@pytest.mark.parametrize("how", ["list", "grad", "flat"])
def test_autograd_sees_that_a_step_has_written_the_parameters(how):
    """As after torch's optimizers: a graph that saved a parameter refuses a backward pass behind a step."""
    flat = torch.ones(64 + 64, device=DEV)
    w, other = (torch.nn.Parameter(torch.empty(64, device=DEV)) for _ in range(2))
    for p, t in zip((w, other), flat.split(64)):
        p.data = t                # views with counters of their own, as flatten_parameters makes them
    x = torch.randn(8, 64, device=DEV)
    opt = pkg("optim").AdamW([w, other], lr=0.1)
    h = R().channel_norm(x, R().NormSpec("rms", w))
    h.sum().backward(retain_graph=True)
    versions = w._version, other._version
    {"list": lambda: opt.step([w.grad, None]), "grad": lambda: opt.step(),
     "flat": lambda: opt.step(torch.cat([w.grad, torch.zeros_like(w)]))}[how]()
    assert w._version == versions[0] + 1 and other._version == versions[1] + (how == "flat")       # no gradient: not written
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    R().channel_norm(x, R().NormSpec("rms", w)).sum().backward()          # a new graph of the new values


def test_versions_of_masters_moments_and_inference_tensors():
    p = torch.nn.Parameter(torch.ones(300, dtype=BF16, device=DEV))
    opt = pkg("optim").AdamW([p])
    kept = [opt.master, *opt.moments()]
    versions = [t._version for t in kept]
    opt.step([None])
    assert [t._version for t in kept] == versions and p._version == 0
    opt.step([torch.ones_like(p)])
    assert [t._version for t in kept] == [v + 1 for v in versions] and p._version == 1
    with torch.inference_mode():
        q = torch.ones(300, device=DEV)
    opt = pkg("optim").AdamW([q], lr=0.5, weight_decay=0.0)
    opt.step([torch.ones(300, device=DEV)])
    # a first step of lr g / |g|, off by 12 roundings of it
    off = float((q - 0.5).abs().max())
    assert off <= 12 * 2.0 ** -24
