"""GPU: unusual calls of the residual norms and the AdamW step that the documentation allows, or that are refused: what autograd is
told of a step, views with the negative bit, forward-mode differentiation and tracing, captures beside living graphs, parameters
that move under a captured step, states that are refused, second moments below the normal numbers, 8-bit moments over thousands of steps."""
import copy

import numpy as np
import pytest
import torch

from helpers import pkg
from optim_ref import M_BASE, V_BASE, from8, moments32
from rounding_ref import to8_random

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


def negative(t):
    """t's values as a view with the negative bit: the memory holds -t."""
    n = torch._neg_view(-t.detach())
    assert n.is_neg() and torch.equal(n, t)
    return n


@pytest.mark.parametrize("shape,dim", [((2, 40, 6, 10), 1), ((3, 20, 40), 2)])
def test_negative_views_are_their_values(shape, dim):
    g = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    c = shape[dim]
    plain = [rand(*shape), rand(*shape), rand(*shape), 1 + rand(c), rand(c), 1 + rand(c), rand(c), rand(*shape), rand(*shape)]

    def run(t):
        leaves = [a.detach().requires_grad_() for a in t[:7]]
        x, f, gate, w2, b2, w1, b1 = leaves
        y, h = R().gated_residual(x, f, post=R().NormSpec("layer", w2, b2), gate=gate, gate_act="sigmoid", scale=0.5,
                                  pre=R().NormSpec("layer", w1, b1), channel_dim=dim)
        with torch.no_grad():
            serving = R().gated_residual(x, f, post=R().NormSpec("layer", w2, b2), gate=gate, gate_act="sigmoid", scale=0.5,
                                         pre=R().NormSpec("layer", w1, b1), channel_dim=dim)
        return [y, h, *serving, *torch.autograd.grad((y, h), leaves, t[7:])]
    want = run(plain)
    for i in range(9):
        got = run([negative(t) if k == i else t for k, t in enumerate(plain)])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    z = torch.view_as_real(torch.complex(plain[0], plain[1]))[..., 1]          # strides of two, no bit
    assert torch.equal(R().channel_norm(z, R().NormSpec("rms"), dim), R().channel_norm(plain[1], R().NormSpec("rms"), dim))
    z = torch.complex(plain[0], plain[1]).conj().imag
    assert z.is_neg() and torch.equal(R().channel_norm(z, R().NormSpec("rms"), dim), R().channel_norm(-plain[1], R().NormSpec("rms"), dim))


def test_negative_gates_of_images():
    x, f = torch.randn(3, 40, 9, device=DEV), torch.randn(3, 40, 9, device=DEV)
    for gate in (torch.randn(40, device=DEV), torch.randn(3, 40, device=DEV), torch.randn(3, 40, device=DEV, dtype=BF16)):
        assert torch.equal(R().gated_residual(x, f, gate=negative(gate)), R().gated_residual(x, f, gate=gate))


def test_adamw_takes_negative_gradients_for_their_values_and_refuses_such_parameters():
    p0, g = torch.randn(500, device=DEV), torch.randn(500, device=DEV)
    out = []
    for way in (lambda o: o.step([g]), lambda o: o.step([negative(g)]), lambda o: o.step(negative(g)), lambda o: o.step([negative(g.to(BF16)).float()])):
        p = torch.nn.Parameter(p0.clone())
        opt = pkg("optim").AdamW([p], max_grad_norm=1.0)
        way(opt)
        out.append((p.detach(), *opt.moments()))
    assert all(torch.equal(a, b) for k in (1, 2) for a, b in zip(out[0], out[k]))
    with pytest.raises(ValueError, match="negative view"):
        pkg("optim").AdamW([negative(p0)])
    opt = pkg("optim").AdamW([torch.nn.Parameter(p0.clone())], state_bits=8)
    m, v = opt.moments()
    opt.load_moments(negative(m + 1), negative(v + 1), 1)
    assert torch.equal(opt.moments()[0][:256], m[:256] + 1)


def freed(t):
    t = t.clone()
    t.untyped_storage().resize_(0)
    return t


def test_tensors_without_memory():
    """Zeros that are not stored count as zeros; a storage that was freed under its tensors is an error."""
    x, f, w, p0 = (torch.randn(s, device=DEV) for s in ((6, 40), (6, 40), (40,), (40,)))
    zero = torch._efficientzerotensor(6, 40, device=DEV)
    spec = R().NormSpec("rms", w)
    assert torch.equal(R().gated_residual(x, zero, post=spec), x) and not R().channel_norm(zero, spec).any()
    for call in (lambda: R().channel_norm(freed(x), spec), lambda: R().channel_norm(freed(torch.randn(40, 6, device=DEV).t()), spec), lambda: R().gated_residual(x, freed(f)),
                 lambda: R().channel_norm(x, R().NormSpec("rms", freed(w))), lambda: R().gated_residual(x, f, gate=freed(w)),
                 lambda: R().gated_residual(x, f, gate=freed(x))):
        with pytest.raises(RuntimeError, match="memory has been freed"):
            call()
    a = x.clone().requires_grad_()
    h = R().channel_norm(a, spec)
    dx, = torch.autograd.grad(h, a, zero, retain_graph=True)
    assert not dx.any()
    a.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="memory has been freed"):
        torch.autograd.grad(h, a, torch.ones_like(h))
    p = torch.nn.Parameter(p0.clone())
    opt = pkg("optim").AdamW([p], lr=0.5, weight_decay=0.5)
    for step in (lambda: opt.step([torch._efficientzerotensor(40, device=DEV)]), lambda: opt.step(torch._efficientzerotensor(40, device=DEV))):
        before = p.detach().clone()
        step()
        off = float((p.detach() - 0.75 * before).abs().max())           # a gradient of zeros: the decay alone
        assert off <= 2.0 ** -23 * 4
    assert opt.step_counts == [2]
    for step in (lambda: opt.step([freed(w)]), lambda: opt.step(freed(w))):
        with pytest.raises(ValueError, match="freed"):
            step()
    opt.step([None])
    p.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="freed"):
        opt.step([w])


def test_a_traced_backward_pass_is_refused_and_other_modes_are_not():
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    x = torch.randn(2, 40, 9, device=DEV, requires_grad=True)
    spec = R().NormSpec("rms", torch.ones(40, device=DEV))
    h = R().channel_norm(x, spec)
    dh = torch.randn_like(h)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda d: torch.autograd.grad(h, x, d, retain_graph=True)[0])(dh)
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        torch.autograd.grad(h, x, fw.make_dual(dh, dh), retain_graph=True)
    want, = torch.autograd.grad(h, x, dh, retain_graph=True)
    with FlopCounterMode(display=False):
        again = R().channel_norm(x, spec)
        got, = torch.autograd.grad(again, x, dh)
    assert torch.equal(again, h) and torch.equal(got, want)


def test_any_living_graph_of_a_leaf_on_another_stream_refuses_the_capture():
    """Autograd's accumulator of a leaf is bound to the stream of the leaf's oldest graph, not to that of each graph."""
    x = torch.randn(2, 64, 9, device=DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    call = lambda: R().channel_norm(x, R().NormSpec("rms", w))  # noqa: E731
    side = torch.cuda.Stream()

    def captured(stream, backward):
        graph = torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            z = x * 2
            if not backward:
                with pytest.raises(RuntimeError, match="recorded before this capture"):
                    call()
                return graph, z
            h = call()
            g, = torch.autograd.grad(h, w, torch.ones_like(h))
            return graph, h.detach(), g
    alive = w * 2                       # a graph of other operations
    captured(side, False)
    first = alive
    with torch.cuda.stream(side):       # a second one, on the stream of the capture, does not move the accumulator
        alive = call()
    del first
    captured(side, False)
    torch.cuda.synchronize()
    del alive
    with torch.cuda.stream(side):       # the same stream: nothing to wait for
        alive = call()
    torch.cuda.synchronize()
    graph, h, g = captured(side, True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, alive)
    del alive
    want = call()
    assert torch.equal(g, torch.autograd.grad(want, w, torch.ones_like(want))[0])


@pytest.mark.parametrize("sizes,clip", [([300, 5000, 7], None), ([300, 70000, 64] * 200, 1.0)])
def test_a_captured_step_follows_parameters_to_new_storage(sizes, clip):
    """The table of addresses that a captured step reads is the optimizer's for good: binding again writes it in place."""
    g = torch.Generator().manual_seed(1)
    start = [torch.randn(n, generator=g).to(DEV) for n in sizes]
    grads = [torch.randn(n, generator=g).to(DEV) for n in sizes]
    ps, qs = ([torch.nn.Parameter(t.clone()) for t in start] for _ in range(2))
    opt, ref = (pkg("optim").AdamW(x, lr=1e-2, state_bits=8, max_grad_norm=clip) for x in (ps, qs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grads)
    graph.replay()
    ref.step(grads)
    torch.cuda.synchronize()
    table, old = opt._tensors.data_ptr(), [p.data for p in ps]
    for p in ps:
        p.data = p.data.clone()
    opt.step(grads)
    ref.step(grads)
    kept = [t.clone() for t in old]
    fill = [torch.full((len(opt._tensors),), 255, dtype=torch.uint8, device=DEV) for _ in range(8)]      # into memory that was given back, if any was
    for _ in range(3):
        graph.replay()
        ref.step(grads)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps, qs))
    assert opt._tensors.data_ptr() == table and len(fill) == 8
    assert all(torch.equal(a, b) for a, b in zip(old, kept)) and opt.step_counts == ref.step_counts == [5] * len(sizes)


def test_a_refused_state_changes_nothing():
    p = [torch.nn.Parameter(torch.randn(300, device=DEV)), torch.nn.Parameter(torch.randn(40, device=DEV).to(BF16))]
    opt = pkg("optim").AdamW(p, lr=1e-3)
    opt.step([torch.ones_like(t) for t in p])
    good = opt.state_dict()
    opt.step([torch.ones_like(t) for t in p])

    def all_of_it():
        return ([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups], opt.step_counts,
                [t.clone() for t in (*opt.moments(), opt.master)])
    before = all_of_it()
    for where, key, value, error in (("group", "lr", -1.0, ValueError), ("group", "betas", (0.9, 1.0), ValueError), ("group", "eps", None, (TypeError, ValueError)),
                                     (0, "step", torch.tensor(-1.0), ValueError), (1, "step", torch.tensor(2.0 ** 31), ValueError),
                                     (0, "exp_avg_sq", torch.zeros(1, device=DEV), ValueError), (1, "master", torch.zeros(1, device=DEV), ValueError)):
        sd = copy.deepcopy(good)
        (sd["param_groups"][0] if where == "group" else sd["state"][where])[key] = value
        if key != "lr":
            sd["param_groups"][0]["lr"] = 0.5
        with pytest.raises(error):
            opt.load_state_dict(sd)
        after = all_of_it()
        assert after[:2] == before[:2] and all(torch.equal(a, b) for a, b in zip(after[2], before[2])), (where, key)
    with pytest.raises(ValueError, match="step"):
        opt.load_moments(*(torch.ones_like(t) for t in opt.moments()), 2 ** 31)
    assert all(torch.equal(a, b) for a, b in zip(all_of_it()[2], before[2]))
    opt.load_state_dict(good)
    assert opt.step_counts == [1, 1]


def test_a_schedule_keeps_the_groups_learning_rates_apart():
    """The trainers' epoch schedule through an optimizer whose groups differ, and through one whose groups do not."""
    OPT, T = pkg("optim"), pkg("train")
    gen = pkg("esrgan.generator").GeneratorESRGAN(num_blocks=1).to(DEV)
    disc = pkg("esrgan.discriminator").Discriminator().to(DEV)
    with pytest.warns(UserWarning):
        vgg = pkg("utils.loss").VGGLoss(device=DEV, allow_synthetic=True)

    def mk(module):
        groups = OPT.decay_groups(module, 0.1)
        if module is gen:
            groups[1]["lr"] = 5e-4
        return OPT.AdamW(groups, lr=1e-3)
    tr = T.AdversarialTrainer(gen, disc, vgg, (2, 3, 16, 16), optimizer=mk)
    lrs = lambda opt: [g["lr"] for g in opt.param_groups]  # noqa: E731
    for epoch in range(3):
        lr = T.cosine_lr(1e-3, epoch, t_max=3, eta_min=1e-7)
        tr.set_lr(lr)
        assert lrs(tr.opt_g) == [lr, lr * 0.5] and lrs(tr.opt_d) == [lr, lr]
    tr.opt_g.lr = 3e-4                  # for all, as documented
    assert lrs(tr.opt_g) == [3e-4, 3e-4]
    plain = T.AdversarialTrainer(gen, disc, vgg, (2, 3, 16, 16))
    plain.set_lr(1e-5)
    assert plain.opt_g.lr == plain.opt_d.lr == 1e-5


@pytest.mark.parametrize("eps", [1e-15, 1e-14, 1e-13, 1e-12, 1e-8])
def test_second_moments_below_the_smallest_normal_number(eps):
    """v = (1 - beta2) g^2 = 9e-39 at a first step: its root, 3e-18 with the bias correction, still counts beside eps = 1e-15."""
    p = torch.nn.Parameter(torch.zeros(600, device=DEV))
    g = torch.full((600,), 3e-18)
    opt = pkg("optim").AdamW([p], lr=1.0, weight_decay=0.0, eps=eps)
    opt.step([g.to(DEV)])
    g = float(g[0].double())
    want = -g / (g + eps)
    # v is a multiple of 2^-149 within half: 2^-150 / 9e-39 = 2^-23.6 of itself, and 12 more roundings of 2^-24 of the operations, or 2^-21 of
    # the update from the hardware's root and reciprocal
    off = float((p.detach().double() / want - 1).abs().max())
    assert off <= 2.0 ** -21 + 16 * 2.0 ** -24


@pytest.mark.parametrize("how", ["one launch", "list", "many", "flat"])
def test_random_rounding_bit_for_bit(how):
    """Three steps of every form of the call against the same operations in numpy: each stored moment, from the one before."""
    sizes = {"one launch": [1, 255, 256, 1000, 4097], "list": [1, 257, 4096, 300001], "many": [3, 700, 4097] * 320, "flat": [5, 64, 300001]}[how]
    g = torch.Generator().manual_seed(5)
    rand = lambda: [torch.randn(n, generator=g).to(DEV) * torch.exp(3 * torch.randn(n, generator=g)).to(DEV) for n in sizes]  # noqa: E731
    if how == "flat":
        buf = torch.cat(rand())
        ps = [torch.nn.Parameter(t) for t in buf.split(sizes)]
    else:
        ps = [torch.nn.Parameter(t) for t in rand()]
    # a norm that does not clip, where there are more tensors than a launch's addresses
    opt = pkg("optim").AdamW(ps, lr=1e-3, state_bits=8, rounding="random", max_grad_norm=1e30 if how == "many" else None)
    m, v = ([np.zeros(n, np.float32) for n in sizes] for _ in range(2))
    for step in (1, 2, 3):
        grads = rand()
        if step == 2 and how != "flat":
            grads[1] = None
        opt.step(torch.cat(grads) if how == "flat" else grads)
        got = [t.cpu().numpy() for t in opt.moments()]
        for i, n in enumerate(sizes):
            if grads[i] is None:
                continue
            count = step - (how != "flat" and step > 2 and i == 1)
            new = moments32(m[i], v[i], grads[i].cpu().numpy(), 1.0, 0.9, 0.999)
            at = 256 * opt._first[i]
            for mine, x, base, least, signed, all_of_it in ((m, new[0], M_BASE, 0, True, got[0]), (v, new[1], V_BASE, 1, False, got[1])):
                mine[i] = from8(*to8_random(x, base, least, signed, opt._first[i], count), base, signed)
                assert np.array_equal(all_of_it[at:at + n], mine[i]), (step, i, signed)


def test_random_rounding_in_graphs_and_state_files():
    """The random bits go by place and step count: a captured step, and an optimizer resumed from a file, give the same."""
    g = torch.Generator().manual_seed(6)
    start = [torch.randn(n, generator=g).to(DEV) for n in (300, 5000)]
    grads = [torch.randn(n, generator=g).to(DEV) for n in (300, 5000)]
    mk = lambda ps: pkg("optim").AdamW(ps, lr=1e-3, state_bits=8, rounding="random")  # noqa: E731
    ps, qs = ([torch.nn.Parameter(t.clone()) for t in start] for _ in range(2))
    opt, ref = mk(ps), mk(qs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grads)
    for _ in range(4):
        graph.replay()
        ref.step(grads)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*ps, *opt.moments()), (*qs, *ref.moments())))
    rs = [torch.nn.Parameter(q.detach().clone()) for q in qs]
    again = mk(rs)
    again.load_state_dict(ref.state_dict())
    assert torch.equal(again._m, ref._m) and torch.equal(again._v, ref._v)
    ref.step(grads)
    again.step(grads)
    assert all(torch.equal(a, b) for a, b in zip((*rs, *again.moments()), (*qs, *ref.moments())))
    near = pkg("optim").AdamW(rs, state_bits=8, rounding="nearest")
    near.load_state_dict(ref.state_dict())
    assert torch.equal(near._m, ref._m) and torch.equal(near._v, ref._v)


def test_8_bit_moments_follow_32_bit_ones_over_thousands_of_steps():
    """Gradients whose level falls tenfold, beside one of each block that keeps its own: v's mean ratio to the 32-bit one over
    n = 64 * 255 values, whose spread is 0.55 at most, is within 5 * 0.55 / sqrt(n) = 0.022 of 1; m's sum of squares, nine tenths of which turn over in 20
    steps, holds its rounding (d^2 / 6 of a value's square a step with d = 1 / 8, kept for 1 / (1 - 0.81) steps: 1.4 %) above the 32-bit one's own: within 5 %."""
    n = 256 * 64
    rest = torch.arange(n, device=DEV) % 256 > 0
    p, q = (torch.nn.Parameter(torch.zeros(n, device=DEV)) for _ in range(2))
    a = pkg("optim").AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8, rounding="random")
    b = pkg("optim").AdamW([q], lr=1e-3, weight_decay=0.0)
    gen = torch.Generator(device=DEV).manual_seed(0)
    for t in range(1, 4001):
        g = torch.randn(n, generator=gen, device=DEV) * (1.0 if t < 1000 else 0.1)
        g[~rest] = 10.0
        a.step([g])
        b.step([g])
        if t % 1000 == 0:
            (m8, v8), (m, v) = a.moments(), b.moments()
            ratio = (v8 / v)[rest].double().mean().item()
            squares = (m8[rest].double().square().sum() / m[rest].double().square().sum()).item()
            assert abs(ratio - 1) < 0.022 and abs(squares - 1) < 0.05, (t, ratio, squares)


def test_the_default_rounding_says_what_it_is():
    p = torch.nn.Parameter(torch.zeros(300, device=DEV))
    with pytest.warns(UserWarning, match="rounding='random'"):
        assert pkg("optim").AdamW([p], state_bits=8).rounding == "nearest"
    import warnings
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for k in (dict(state_bits=8, rounding="nearest"), dict(state_bits=8, rounding="random"), dict()):
            pkg("optim").AdamW([p], **k)


@pytest.mark.parametrize("shape,dim", [((2, 40, 6, 10), 1), ((3, 20, 40), 2)])
def test_inside_a_checkpoint(shape, dim):
    """Recomputation ends with an exception of its own inside the call that saves the last tensor."""
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator().manual_seed(3)
    c = shape[dim]
    leaves = [t.to(DEV).requires_grad_() for t in (torch.randn(*shape, generator=g), torch.randn(*shape, generator=g), torch.randn(c, generator=g), torch.randn(c, generator=g))]

    def run(x, f, w2, w1):
        y, h = R().gated_residual(x, f * 2, post=R().NormSpec("rms", w2), pre=R().NormSpec("layer", w1), channel_dim=dim)
        return R().channel_norm(y + h, R().NormSpec("rms", w1), dim)
    want = torch.autograd.grad(run(*leaves).square().sum(), leaves)
    for reentrant in (False, True):
        for t in leaves:
            t.grad = None
        checkpoint(run, *leaves, use_reentrant=reentrant).square().sum().backward()
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want)), reentrant


def test_exceptions_keep_their_types():
    class Stop(Exception):
        pass

    def stop(t):
        raise Stop
    x = torch.randn(4, 40, device=DEV, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(stop, lambda t: t), pytest.raises(Stop):
        R().channel_norm(x, R().NormSpec("rms"))
    wide = torch.zeros(1, 40, device=DEV).expand(1 << 22, 40)
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.001)          # of 288 GB: less than the 671 MB of one output
    try:
        with pytest.raises(torch.OutOfMemoryError):
            R().channel_norm(wide, R().NormSpec("rms"))
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


def test_sigmoid_of_far_gates():
    """y = sigmoid(q) for q over all that fp32 can hold: the gate's own bound, (1.5 |q| + 6) 2^-24 of the value, and four more
    roundings of the factors 1 around it; where it leaves the normal numbers, 2^-126."""
    q = torch.cat([torch.linspace(-87, 87, 40 * 500), torch.linspace(-2000, 2000, 40 * 10)]).view(-1, 40).to(DEV)
    x, f = torch.zeros_like(q), torch.ones_like(q)
    want = torch.sigmoid(q.double().cpu())
    for gate, out in ((q, lambda g: R().gated_residual(x, f, gate=g, gate_act="sigmoid")),
                      (q, lambda g: R().gated_residual(x[:, :, None].expand(-1, -1, 2), f[:, :, None].expand(-1, -1, 2), gate=g, gate_act="sigmoid")[..., 1])):
        got = out(gate).double().cpu()
        allowed = (1.5 * q.double().cpu().abs() + 10) * 2.0 ** -24 * want + 2.0 ** -126
        worst = float(((got - want).abs() / allowed).max())
        assert worst <= 1, worst
